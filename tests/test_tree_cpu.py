"""CPU checks of the speculative-decoding operators: the host tree layout, the refusal of bad
arguments (every refusal comes before any CUDA call, so none needs a GPU), and the verification rule itself."""
import numpy as np
import pytest

import llmdiy_b200 as L
import treemath as tm

REFUSED = r"status 1\b"  # cudaErrorInvalidValue, not the launch error of a machine without a GPU
A = 1 << 20  # a 16-byte aligned address; no refused call dereferences it


@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 200, 256])
def test_layout_matches_the_definition(n):
    rng = np.random.default_rng(n)
    parent = [-1] + [int(rng.integers(0, i)) for i in range(1, n)]
    depth, mask = L.tree_layout(parent)
    d, sees = tm.layout(parent)
    assert depth.tolist() == d
    assert np.array_equal(mask.view(np.int64), tm.mask_words(sees, n))


@pytest.mark.parametrize("parent", [[], [0], [-1, 1], [-1, -1], [-1, 0, 2], [-1, 0, 3, 0], [-1] + [0] * 256])
def test_layout_refuses_what_is_no_tree(parent):
    with pytest.raises(L.LlmdiyError, match=r"status -1\b"):
        L.tree_layout(parent)


ATTN = dict(Q=A, ldq=2048, K=A, V=A, stride=2048, slot_rows=100, num_slots=4, slot=None, lens=A, max_len=100, TK=A,
            TV=A, mask=A, tree_len=None, B=2, N=8, num_heads=16, num_kv_heads=16, O=A, ldo=2048, work=A,
            work_bytes=1 << 30)


@pytest.mark.parametrize("bad", [
    dict(Q=None), dict(Q=A + 2), dict(K=A + 8), dict(V=None), dict(TK=A + 2), dict(TV=None), dict(O=None),
    dict(lens=None), dict(mask=None), dict(work=None), dict(work=A + 4), dict(work_bytes=0),
    dict(ldq=2047), dict(ldq=2040), dict(ldo=2040), dict(ldo=2052), dict(stride=2040), dict(stride=2049), dict(B=0),
    dict(B=-1), dict(B=65536), dict(N=0), dict(N=257), dict(num_heads=0), dict(num_kv_heads=0), dict(num_kv_heads=3),
    dict(num_heads=8), dict(max_len=-1), dict(max_len=101), dict(slot_rows=0), dict(num_slots=0),
    dict(num_slots=1 << 25)])
def test_attn_refuses(bad):
    with pytest.raises(L.LlmdiyError, match=REFUSED):
        L.tree_attn(**{**ATTN, **bad})


def test_attn_work_bytes():
    full = L.tree_attn_work_bytes(16, 64, 16, 16, 4160)
    assert full >= 16
    for B, N, m in [(1, 64, 4160), (16, 1, 4160), (16, 64, 0), (16, 64, 100), (3, 17, 2048), (7, 33, 4159)]:
        assert 16 <= L.tree_attn_work_bytes(B, N, 16, 16, m) <= full, (B, N, m)
    for a in [(0, 8, 16, 16, 10), (1, 0, 16, 16, 10), (1, 257, 16, 16, 10), (1, 8, 16, 5, 10), (1, 8, 0, 1, 10),
              (1, 8, 16, 16, -1)]:
        assert L.tree_attn_work_bytes(*a) == 0, a


ROPE = dict(qkv=A, bias=None, depth=A, lens=A, tree_len=None, B=2, N=8, num_heads=16, num_kv_heads=16,
            rope_base=10000.0, Q=A, TK=A, TV=A)


@pytest.mark.parametrize("bad", [
    dict(qkv=None), dict(qkv=A + 2), dict(bias=A + 2), dict(depth=None), dict(lens=None), dict(Q=None), dict(TK=A + 4),
    dict(TV=None), dict(B=0), dict(N=0), dict(N=257), dict(num_heads=5, num_kv_heads=2), dict(num_kv_heads=0),
    dict(rope_base=0.0), dict(rope_base=-1.0), dict(rope_base=float("inf")), dict(rope_base=float("nan"))])
def test_rope_refuses(bad):
    with pytest.raises(L.LlmdiyError, match=REFUSED):
        L.tree_rope(**{**ROPE, **bad})


SOFT = dict(logits=A, ldl=100, temp=None, R=3, V=100, probs=A, ldp=100)


@pytest.mark.parametrize("bad", [dict(logits=None), dict(probs=None), dict(R=0), dict(V=0), dict(ldl=99), dict(ldp=99),
                                 dict(R=-2), dict(logits=A + 1), dict(probs=A + 2)])
def test_softmax_refuses(bad):
    with pytest.raises(L.LlmdiyError, match=REFUSED):
        L.softmax_rows(**{**SOFT, **bad})


VER = dict(target=A, ldt=100, draft=A, ldd=100, token=A, parent=A, tree_len=None, uniform=A, B=2, N=4, V=100, path=A,
           accepted=A, next_token=A)


@pytest.mark.parametrize("bad", [
    dict(target=None), dict(token=None), dict(parent=None), dict(uniform=None), dict(path=None), dict(accepted=None),
    dict(next_token=None), dict(ldt=99), dict(ldd=99), dict(B=0), dict(N=0), dict(N=257), dict(V=0),
    dict(target=A + 2), dict(draft=A + 1)])
def test_verify_refuses(bad):
    with pytest.raises(L.LlmdiyError, match=REFUSED):
        L.tree_verify(**{**VER, **bad})


COM = dict(TK=A, TV=A, tree_layer_stride=2 * 8 * 2048, K=A, V=A, layer_stride=4 * 100 * 2048, stride=2048,
           slot_rows=100, num_slots=4, slot=None, lens=A, path=A, accepted=A, B=2, N=8, num_kv_heads=16, layers=3,
           len_out=None)


@pytest.mark.parametrize("bad", [
    dict(TK=None), dict(TV=A + 2), dict(K=None), dict(V=A + 8), dict(lens=None), dict(path=None), dict(accepted=None),
    dict(len_out=A), dict(stride=2040), dict(stride=2050), dict(tree_layer_stride=2 * 8 * 2048 - 8),
    dict(tree_layer_stride=2 * 8 * 2048 + 4), dict(layer_stride=4 * 100 * 2048 - 8), dict(slot_rows=0),
    dict(num_slots=0), dict(B=0), dict(N=0), dict(num_kv_heads=0), dict(layers=0)])
def test_commit_refuses(bad):
    with pytest.raises(L.LlmdiyError, match=REFUSED):
        L.tree_commit(**{**COM, **bad})


@pytest.mark.parametrize("deterministic", [False, True])
def test_verification_rule_is_lossless(deterministic):
    """The first emitted token (the first accepted draft, or the next token) has exactly the target's
    distribution.  Two siblings under the root, V = 3: the probability of every outcome follows from the
    definition by integrating the acceptance tests (a test with ratio r succeeds with probability min(1, r)),
    and the rule as the tests use it (treemath.verify) is checked at numbers on either side of each ratio."""
    p = np.array([[0.5, 0.3, 0.2]])
    q = np.array([[0.2, 0.7, 0.1]])
    target, draft = np.vstack([p, p, p]), np.vstack([q, q, q])
    out = np.zeros(3)

    def residual(w, x):
        if deterministic:
            w = w.copy()
            w[x] = 0
        else:
            w = np.maximum(0, w - q[0])
        return w / w.sum()

    pairs = [(0, 1, 1.0)] if deterministic else [(a, b, q[0, a] * q[0, b]) for a in range(3) for b in range(3)]
    for a, b, weight in pairs:
        d = (lambda x: 1.0) if deterministic else (lambda x: q[0, x])
        ra = min(1.0, p[0, a] / d(a))
        out[a] += weight * ra
        tok, par = [0, a, b], [-1, 0, 0]
        dr = None if deterministic else draft
        if ra < 1:
            w1 = residual(p[0], a)
            rb = min(1.0, w1[b] / d(b))
            out[b] += weight * (1 - ra) * rb
            eps = 1e-9
            assert tm.verify(target, dr, tok, par, 3, [0.5, ra - eps, 0.0])[0][:1] == [1]
            if rb > 0:
                assert tm.verify(target, dr, tok, par, 3, [0.5, ra + eps, rb - eps])[0][:1] == [2]
            if rb < 1:
                w2 = residual(w1, b)
                out += weight * (1 - ra) * (1 - rb) * w2
                path, nxt = tm.verify(target, dr, tok, par, 3, [0.999999, ra + eps, rb + eps])
                assert path == [] and nxt == int(np.nonzero(w2 > 0)[0][-1])
    assert np.allclose(out, p[0], atol=1e-12)


@pytest.mark.parametrize("call,good,bad", [
    (L.tree_rope, ROPE, k) for k in (dict(depth=A + 2), dict(lens=A + 1), dict(tree_len=A + 2))] + [
    (L.softmax_rows, SOFT, k) for k in (dict(temp=A + 2), dict(V=2 ** 30 + 1, ldl=2 ** 30 + 1, ldp=2 ** 30 + 1))] + [
    (L.tree_verify, VER, k) for k in (
        dict(token=A + 2), dict(parent=A + 1), dict(tree_len=A + 2), dict(uniform=A + 2), dict(path=A + 3),
        dict(accepted=A + 2), dict(next_token=A + 2), dict(V=2 ** 30 + 1, ldt=2 ** 30 + 1, ldd=2 ** 30 + 1))] + [
    (L.tree_attn, ATTN, k) for k in (dict(slot=A + 2), dict(lens=A + 2), dict(tree_len=A + 1))] + [
    (L.tree_commit, COM, k) for k in (
        dict(slot=A + 2), dict(lens=A + 1), dict(path=A + 2), dict(accepted=A + 2), dict(len_out=A + 18))])
def test_refuses_misaligned_words_and_overlong_rows(call, good, bad):
    with pytest.raises(L.LlmdiyError, match=REFUSED):
        call(**{**good, **bad})


@pytest.mark.parametrize("sizes,path", [
    ((1, 1, 16, 16, 1023), 2), ((1, 4, 2, 2, 1000), 2), ((1, 26, 16, 16, 2047), 1), ((1, 1, 8, 1, 30000), 1),
    ((3, 100, 4, 2, 30001), 1), ((16, 64, 16, 16, 4160), 0), ((2, 48, 32, 8, 65536), 0), ((1, 1, 8, 1, 131072), 0), ((1, 64, 16, 16, 131072), 0),
    ((0, 8, 16, 16, 10), -1), ((1, 257, 16, 16, 10), -1), ((1, 8, 16, 5, 10), -1), ((1, 8, 16, 16, -1), -1)])
def test_attn_path(sizes, path):
    """The way a call takes, by its sizes (on a machine without a GPU as for 148 SMs)."""
    assert L.tree_attn_path(*sizes) == path
