"""The speculative-decoding operators (include/llmdiy_tree.h) on the GPU against plain 64-bit restatements
(treemath.py), each at the sizes, masks and values where it can go wrong, and a whole step of them together."""
import numpy as np
import pytest

import llmdiy_b200 as L
import treemath as tm
from gpu_util import torch

pytestmark = pytest.mark.gpu

D = 128


_alive = []  # every device copy of a test lives until its end: a call only holds addresses


@pytest.fixture(autouse=True)
def _free_after_the_test():
    yield
    torch().cuda.synchronize()
    _alive.clear()


def _i32(x):
    t = torch()
    _alive.append(t.tensor(np.asarray(x, np.int32), device="cuda"))
    return _alive[-1]


def _dev(a):
    t = torch()
    _alive.append(t.from_numpy(np.ascontiguousarray(a)).cuda())
    return _alive[-1]


def _ptr(x):
    return None if x is None else x.data_ptr()


def _parents(rng, n, chain=False):
    return [-1] + [i - 1 if chain else int(rng.integers(max(0, i - 9), i)) for i in range(1, n)]


# ------------------------------------------------------------------ attention
class Attn:
    """Inputs of one tree_attn call on the host (numpy) and their copies on the device."""

    def __init__(self, seed, B, N, H, KV, lens, max_len=None, tree_len=None, slots=None, num_slots=None, pad=0,
                 slot_rows=None, sees=None, scale=1.0):
        rng = np.random.default_rng(seed)
        self.B, self.N, self.H, self.KV, self.lens = B, N, H, KV, list(lens)
        self.max_len = max(lens) if max_len is None else max_len
        self.slot_rows = slot_rows or self.max_len + 3
        self.num_slots = num_slots or B
        self.slots = list(range(B)) if slots is None else list(slots)
        self.tree_len = [N] * B if tree_len is None else list(tree_len)
        self.stride, self.ldq, self.ldo = KV * D + pad, H * D + pad, H * D + 2 * pad
        f16 = lambda *s: rng.standard_normal(s, dtype=np.float32).astype(np.float16)  # noqa: E731
        self.Q = (f16(B, N, self.ldq).astype(np.float32) * scale).astype(np.float16)
        self.K, self.V = (f16(self.num_slots, self.slot_rows, self.stride) for _ in range(2))
        self.TK, self.TV = (f16(B, N, KV * D) for _ in range(2))
        self.sees = sees or [tm.layout(_parents(rng, N))[1] for _ in range(B)]
        self.give_slots = slots is not None
        self.give_tree_len = tree_len is not None

    def device(self):
        t = torch()
        self.d = {k: _dev(getattr(self, k)) for k in ("Q", "K", "V", "TK", "TV")}
        self.d["mask"] = _dev(np.stack([tm.mask_words(s, self.N) for s in self.sees]))
        self.d["len"] = _i32(self.lens)
        self.d["slot"] = _i32(self.slots) if self.give_slots else None
        self.d["tree_len"] = _i32(self.tree_len) if self.give_tree_len else None
        self.d["O"] = t.full((self.B, self.N, self.ldo), 7.0, dtype=t.float16, device="cuda")
        n = L.tree_attn_work_bytes(self.B, self.N, self.H, self.KV, self.max_len)
        self.d["work"], self.n = t.zeros((n + 3) // 4, device="cuda"), n
        return self

    def call(self, stream=None, work=None, work_bytes=None):
        d = self.d
        L.tree_attn(_ptr(d["Q"]), self.ldq, _ptr(d["K"]), _ptr(d["V"]), self.stride, self.slot_rows, self.num_slots,
                    _ptr(d["slot"]), _ptr(d["len"]), self.max_len, _ptr(d["TK"]), _ptr(d["TV"]), _ptr(d["mask"]),
                    _ptr(d["tree_len"]), self.B, self.N, self.H, self.KV, _ptr(d["O"]), self.ldo,
                    _ptr(d["work"] if work is None else work), work_bytes or self.n, stream)
        return self

    def want(self, b, i, h):
        g = h * self.KV // self.H
        cols = slice(g * D, (g + 1) * D)
        m = min(max(self.lens[b], 0), self.max_len) if 0 <= self.slots[b] < self.num_slots else 0
        js = sorted(j for j in self.sees[b][i] if j < self.tree_len[b])
        s = self.slots[b] if m else 0
        K = np.concatenate([self.K[s, :m, cols], self.TK[b, js][:, cols]])
        V = np.concatenate([self.V[s, :m, cols], self.TV[b, js][:, cols]])
        return tm.attention_row(self.Q[b, i, h * D:(h + 1) * D], K, V)

    def check(self, rows=None, status=True):
        t = torch()
        t.cuda.synchronize()
        if status:
            assert L.tree_attn_status(_ptr(self.d["work"])) == 0
        got = self.d["O"].cpu().numpy()
        assert np.all(got[..., self.H * D:] == 7.0), "columns past the heads were written"
        for b in range(self.B):
            assert np.all(got[b, max(0, self.tree_len[b]):] == 7.0), "a row past the tree was written"
        rng = np.random.default_rng(1)
        every = [(b, i, h) for b in range(self.B) for i in range(max(0, min(self.N, self.tree_len[b])))
                 for h in range(self.H)]
        if rows and len(every) > rows:
            every = [every[k] for k in rng.choice(len(every), rows, replace=False)]
        for b, i, h in every:
            o, tol = self.want(b, i, h)
            x = got[b, i, h * D:(h + 1) * D].astype(np.float64)
            bad = ~(np.abs(x - o) <= tol) & ~(np.isnan(x) & np.isnan(o)) & ~((x == o) & np.isinf(o))
            assert not bad.any(), (b, i, h, np.nonzero(bad)[0][:4], x[bad][:4], o[bad][:4], tol[bad][:4])
        return self


@pytest.mark.parametrize("B,N,H,KV,lens", [
    (1, 1, 16, 16, [1]), (1, 1, 16, 16, [1023]), (1, 1, 2, 1, [0]), (1, 8, 16, 16, [63]), (1, 8, 16, 16, [64]),
    (1, 8, 4, 4, [65]), (2, 26, 16, 16, [127, 2047]), (3, 64, 2, 2, [0, 1, 1000]), (1, 65, 2, 1, [129]),
    (2, 61, 8, 2, [700, 64]), (1, 256, 4, 2, [300]), (1, 129, 3, 1, [5]), (1, 33, 32, 2, [777]), (1, 1, 1, 1, [64]),
    (5, 3, 20, 4, [10, 0, 500, 64, 128]), (1, 100, 12, 12, [4097])])
def test_attn_matches(B, N, H, KV, lens):
    """Lengths from none, on either side of a 64-row tile, trees from one node to 256, heads grouped or not."""
    Attn(B * 1000 + N, B, N, H, KV, lens).device().call().check(rows=400)


@pytest.mark.parametrize("B,N,H,KV,lens,tree_len", [
    (1, 1, 1, 1, [0], None), (1, 1, 4, 4, [1], None), (2, 1, 2, 2, [15, 17], None), (1, 1, 3, 3, [8200], None),
    (1, 2, 4, 4, [511], None), (3, 2, 6, 3, [0, 129, 300], [2, 1, 2]), (1, 4, 2, 2, [1000], None),
    (4, 4, 2, 2, [5, 0, 64, 700], [0, 4, 3, 1]), (2, 1, 12, 4, [63, 513], None), (2, 3, 2, 2, [100, 0], [3, 9]),
    (40, 1, 16, 16, [7 * i for i in range(40)], None), (70, 1, 8, 2, [5 * i for i in range(70)], [i % 3 for i in range(70)]),
    (1, 2, 4, 2, [300], None), (1, 4, 4, 4, [2500], None), (300, 2, 2, 2, [i % 37 for i in range(300)], None)])
def test_attn_of_one_to_four_rows(B, N, H, KV, lens, tree_len):
    """Units of one to four query rows: lengths on either side of a half warp's and a CTA's share, empty trees, one CTA
    and several per unit, short and long shares, padded rows, slots in another order; the same bits again."""
    a = Attn(B * 77 + N, B, N, H, KV, lens, tree_len=tree_len, slots=list(range(B))[::-1], pad=8).device().call()
    first = a.d["O"].clone()
    a.call()
    torch().cuda.synchronize()
    assert torch().equal(a.d["O"], first)
    if tree_len:
        a.tree_len = [min(n, N) for n in tree_len]
    a.check(rows=300)


@pytest.mark.parametrize("B,N,H,KV,lens,tree_len", [
    (1, 16, 8, 2, [4096], None), (1, 8, 16, 16, [3333], None), (2, 9, 8, 4, [5000, 70], [9, 2]), (1, 70, 8, 2, [3500], None),
    (1, 16, 8, 1, [40001], None), (2, 33, 4, 1, [20000, 33], [33, 12]), (1, 1, 8, 1, [30000], None)])
def test_attn_of_few_units_with_long_caches(B, N, H, KV, lens, tree_len):
    """Clusters of 12 and 16 CTAs, and single units cut into many parts; sequences that end long before the others."""
    a = Attn(B * 31 + N, B, N, H, KV, lens, tree_len=tree_len).device().call()
    first = a.d["O"].clone()
    a.call().check(rows=60)
    assert torch().equal(a.d["O"], first)


@pytest.mark.parametrize("B,N,H,KV,lens,tree_len", [
    (4, 5, 32, 32, [280, 0, 64, 131], None), (4, 8, 16, 16, [300, 65, 128, 1], [8, 0, 5, 8]),
    (3, 20, 16, 16, [500, 499, 20], None), (5, 9, 8, 8, [700, 0, 3, 640, 128], [9, 9, 1, 4, 0]),
    (1, 101, 20, 4, [1616], None), (2, 60, 12, 12, [600, 90], [60, 33]), (3, 23, 20, 4, [35, 0, 64], None),
    (1, 64, 32, 8, [200], None), (8, 83, 3, 3, [65, 0, 1, 64, 63, 30, 10, 5], None)])
def test_attn_of_every_cluster_size(B, N, H, KV, lens, tree_len):
    """Short caches on clusters of one to eight CTAs: odd numbers of joined rows, CTAs without a tile, sequences that are
    shorter than a cluster; the same bits again."""
    a = Attn(B * 13 + N, B, N, H, KV, lens, tree_len=tree_len, pad=8).device().call()
    first = a.d["O"].clone()
    a.call().check(rows=250)
    assert torch().equal(a.d["O"], first)


def test_attn_single_tokens_captured_and_on_two_streams():
    """One row per head: a graph replayed while lengths change (down to none), beside calls on another stream."""
    t = torch()
    a, b = (Attn(70 + i, 3, 1, 8, 4, [500, 3, 200], max_len=500).device() for i in range(2))
    s1, s2 = t.cuda.Stream(), t.cuda.Stream()
    for x in (a, b):
        x.call()
    t.cuda.synchronize()
    g = t.cuda.CUDAGraph()
    with t.cuda.graph(g, stream=s1):
        a.call(stream=t.cuda.current_stream().cuda_stream)
    for lens in ([500, 3, 200], [0, 499, 1], [64, 128, 0]):
        a.lens = b.lens = lens
        for x in (a, b):
            x.d["len"].copy_(t.tensor(lens, dtype=t.int32))
            x.d["O"].fill_(7.0)
        t.cuda.synchronize()
        for _ in range(4):
            with t.cuda.stream(s1):
                g.replay()
            b.call(stream=s2.cuda_stream)
        a.check()
        b.check()


@pytest.mark.parametrize("length", [0, 30, 400])
def test_attn_of_few_rows_nothing_leaks(length):
    """Two and four rows: Inf and NaN in cache rows past the length and in tree rows that a node does not see; rows
    that see nothing give zeros; one that sees a NaN score is NaN."""
    t = torch()
    for N, H, KV in ((2, 2, 2), (4, 3, 3), (1, 4, 1)):
        sees = [[set(), {1}, {0, 1}, {3}][:N]]
        a = Attn(9 + length, 1, N, H, KV, [length], max_len=length + 60, sees=sees)
        a.K[0, length:], a.V[0, length:] = np.nan, np.inf
        a.TK[0, 0] = np.nan if N < 3 else a.TK[0, 0]
        a.TV[0, 0] = -np.inf if N < 3 else a.TV[0, 0]
        if N == 4:
            a.TV[0, 2] = a.TK[0, 2] = np.nan
        a.device().call().check()
        if length == 0:
            assert t.all(a.d["O"][0, 0, :H * D] == 0)
    a = Attn(3, 1, 2, 2, 2, [50])
    a.K[0, 49, :D] = np.nan
    a.device().call()
    t.cuda.synchronize()
    assert t.isnan(a.d["O"][0, :, :D]).all() and not t.isnan(a.d["O"][0, :, D:2 * D]).any()


def test_attn_strides_slots_and_ragged_trees():
    """Padded rows, slots of a larger pool in mixed order, trees of different sizes (one empty), lengths
    past max_len, negative lengths and slots that do not exist."""
    a = Attn(5, 6, 40, 8, 4, [90, 200, -5, 77, 1000, 30], max_len=200, tree_len=[40, 17, 3, 0, 500, 1],
             slots=[4, 0, 2, 3, 6, 99], num_slots=7, pad=24)
    a.device().call()
    a.tree_len = [40, 17, 3, 0, 40, 1]
    a.check(rows=500)


@pytest.mark.parametrize("length", [0, 40, 64, 500])
def test_attn_masks_that_leave_rows_empty(length):
    """Arbitrary masks: rows without a bit (zeros where the cache is empty too), rows that do not see
    themselves, rows that see later nodes and nodes past the tree."""
    rng = np.random.default_rng(length)
    N = 70
    sees = [[set() if i % 3 == 0 else set(np.nonzero(rng.random(N) < 0.2)[0].tolist()) for i in range(N)]
            for _ in range(2)]
    a = Attn(length, 2, N, 4, 2, [length, length], max_len=length + 1, tree_len=[70, 50], sees=sees)
    a.device().call().check(rows=400)
    if length == 0:
        assert np.all(a.d["O"].cpu().numpy()[0, 0, :4 * D] == 0.0)


@pytest.mark.parametrize("length", [3, 64, 130])
def test_attn_nothing_leaks_from_unseen_rows(length):
    """NaN and infinities in K and V rows past the length, in tree rows past the tree and in tree rows
    that only some nodes see: they reach exactly the nodes that see them."""
    N = 24
    a = Attn(length, 2, N, 4, 2, [length, length], max_len=length + 70, tree_len=[24, 20])
    for s in range(2):
        a.K[s, length:] = np.nan
        a.V[s, length:] = np.inf
        a.V[s, length + 1:] = np.nan
    a.TK[1, 20:], a.TV[1, 20:] = np.inf, np.nan
    a.TV[0, 7, 5], a.TV[0, 9, 130], a.TK[0, 11, 3] = np.nan, -np.inf, np.nan
    a.device().call()
    with np.errstate(invalid="ignore"):
        a.check()
    clean = [i for i in range(N) if not {7, 9, 11} & a.sees[0][i]]
    assert len(clean) > 5
    assert np.isfinite(a.d["O"].cpu().numpy()[0, clean, :4 * D]).all()


def test_attn_large_scores():
    """Scores of several hundred: the running maximum moves by large steps, most probabilities vanish."""
    Attn(77, 2, 30, 4, 4, [1500, 640], scale=30.0).device().call().check(rows=200)


def test_attn_long_cache():
    """A long cache, few heads: many splits of one sequence, and a short sequence beside it."""
    Attn(8, 2, 20, 4, 2, [40000, 37]).device().call().check(rows=40)


def test_attn_offsets_past_32_bits():
    """A cache whose last slot starts more than 2^31 elements after the first, and more than 2^32 bytes."""
    t = torch()
    H, N, rows, slots, m = 16, 5, 9000, 120, 200
    stride = H * D
    assert (slots - 1) * rows * stride > 2**31
    a = Attn(3, 2, N, H, H, [m, m], max_len=m, slots=[0, 1])
    a.device()
    K, V = (t.zeros((slots, rows, stride), dtype=t.float16, device="cuda") for _ in range(2))
    for x, y in ((K, a.d["K"]), (V, a.d["V"])):
        x[0, :m], x[slots - 1, :m] = y[0, :m], y[1, :m]
    d = a.d
    d["slot"] = _i32([0, slots - 1])
    L.tree_attn(_ptr(d["Q"]), a.ldq, _ptr(K), _ptr(V), stride, rows, slots, _ptr(d["slot"]), _ptr(d["len"]), m,
                _ptr(d["TK"]), _ptr(d["TV"]), _ptr(d["mask"]), None, 2, N, H, H, _ptr(d["O"]), a.ldo, _ptr(d["work"]),
                a.n)
    a.check(rows=120)


def test_attn_workspace_serves_smaller_calls_and_results_repeat():
    """One workspace for calls of different sizes back to back; the same call twice gives the same bits."""
    t = torch()
    big = Attn(1, 4, 64, 8, 8, [3000, 50, 900, 2999]).device()
    small = Attn(2, 3, 7, 8, 8, [2500, 3, 0]).device()
    for _ in range(2):
        big.call()
        small.call(work=big.d["work"], work_bytes=big.n)
    big.check(rows=150)
    small.check(rows=150)
    first = small.d["O"].clone()
    small.d["O"].fill_(7.0)
    small.call(work=big.d["work"], work_bytes=big.n)
    t.cuda.synchronize()
    assert t.equal(first, small.d["O"])


def test_attn_single_nodes_match_fd_multihead():
    """N = 1 with the node's own row is decoding: the same attention as fd_multihead over len + 1 rows."""
    t = torch()
    H, m = 16, 3000
    a = Attn(9, 1, 1, H, H, [m], slot_rows=m + 1).device().call()
    a.d["K"][0, m], a.d["V"][0, m] = a.d["TK"][0, 0], a.d["TV"][0, 0]
    nb = L.fd_mh_work_bytes(m + 1, H)
    w = t.zeros((nb + 3) // 4, device="cuda")
    O = t.zeros(H * D, dtype=t.float16, device="cuda")
    L.fd_multihead(_ptr(a.d["Q"]), _ptr(a.d["K"]), _ptr(a.d["V"]), _ptr(O), m + 1, H * D, H, _ptr(w), nb)
    t.cuda.synchronize()
    assert float((O.float() - a.d["O"].view(-1)[: H * D].float()).abs().max()) < 1e-3


# ------------------------------------------------------------------ bias + RoPE
@pytest.mark.parametrize("B,N,H,KV,lens,bias,tree_len", [
    (1, 1, 16, 16, [0], True, None), (2, 26, 16, 16, [2047, 5], True, None), (3, 9, 8, 2, [131071, 7, 0], False,
                                                                              [9, 0, 4]),
    (1, 256, 1, 1, [1000], True, None), (4, 3, 20, 4, [1, 2, 3, 1 << 20], True, [1, 2, 3, 9])])
def test_rope(B, N, H, KV, lens, bias, tree_len):
    t = torch()
    rng = np.random.default_rng(N)
    cols = (H + 2 * KV) * D
    qkv = rng.standard_normal((B, N, cols)).astype(np.float16)
    bs = rng.standard_normal(cols).astype(np.float16) if bias else None
    depth = rng.integers(0, 9, (B, N))
    dq, db, dd, dl = _dev(qkv), _dev(bs) if bias else None, _i32(depth), _i32(lens)
    tl = None if tree_len is None else _i32(tree_len)
    Q, TK, TV = (t.full((B, N, w * D), 7.0, dtype=t.float16, device="cuda") for w in (H, KV, KV))
    L.tree_rope(_ptr(dq), _ptr(db), _ptr(dd), _ptr(dl), _ptr(tl), B, N, H, KV, 10000.0, _ptr(Q), _ptr(TK), _ptr(TV))
    t.cuda.synchronize()
    Q, TK, TV = (x.cpu().numpy().astype(np.float64) for x in (Q, TK, TV))
    for b in range(B):
        n = N if tree_len is None else min(N, tree_len[b])
        for x in (Q, TK, TV):
            assert np.all(x[b, n:] == 7.0)
        for i in range(n):
            y = qkv[b, i].astype(np.float64) + (bs.astype(np.float64) if bias else 0.0)
            want = tm.rope_row(y[: (H + KV) * D].reshape(-1, D), lens[b] + depth[b, i], 10000.0)
            got = np.concatenate([Q[b, i], TK[b, i]]).reshape(-1, D)
            # fp16 rounding, and 2^-20 of the pair for the fp32 sine, cosine and products
            pair = np.abs(y[: (H + KV) * D].reshape(-1, 2, 64)).sum(1)
            tol = np.abs(want) * 2.0 ** -11 + np.concatenate([pair, pair], 1) * 2.0 ** -20 + 2.0 ** -25
            assert np.all(np.abs(got - want) <= tol), (b, i)
            v = y[(H + KV) * D:]
            assert np.all(np.abs(TV[b, i] - v) <= np.abs(v) * (2.0 ** -11 + 2.0 ** -23) + 2.0 ** -25), (b, i)


def test_rope_of_a_chain_is_the_decode_rope():
    """The root at position p turns as llmdiy_fused_qkv_rope_cache turns a decoded token (whose angles are
    fast-math fp32: |error| at most p * 2^-20 there, so p = 100 keeps it under 1e-3 of the pair)."""
    t = torch()
    rng = np.random.default_rng(2)
    H, p = 16, 100
    qkv = rng.standard_normal((1, 1, 3 * H * D)).astype(np.float16)
    d1, d2 = _dev(qkv), _dev(qkv)
    K, V = (t.zeros((p + 1, H * D), dtype=t.float16, device="cuda") for _ in range(2))
    L.fused_qkv_rope_cache(_ptr(d1), _ptr(K), _ptr(V), p, p + 1, H, D)
    Q, TK, TV = (t.zeros((H * D,), dtype=t.float16, device="cuda") for _ in range(3))
    L.tree_rope(_ptr(d2), None, _ptr(_i32([0])), _ptr(_i32([p])), None, 1, 1, H, H, 10000.0, _ptr(Q), _ptr(TK), _ptr(TV))
    t.cuda.synchronize()
    for x, y in ((Q, d1.view(-1)[: H * D]), (TK, K[p]), (TV, V[p])):
        assert float((x.float() - y.float()).abs().max()) < 8e-3
    assert t.equal(TV, V[p]) and t.equal(d2, _dev(qkv))


# ------------------------------------------------------------------ probabilities
@pytest.mark.parametrize("R,V,pad", [(1, 1, 0), (3, 7, 1), (5, 1000, 0), (4, 1001, 3), (2, 151936, 0), (3, 151935, 1),
                                     (2, 8192, 8), (9, 20000, 4), (1, 500009, 7), (700, 33, 0)])
def test_softmax(R, V, pad):
    t = torch()
    rng = np.random.default_rng(V)
    x = (rng.standard_normal((R, V + pad)) * 3).astype(np.float16)
    x[0, : V // 3] = -np.inf
    if R > 1:
        x[1, :V] = -np.inf  # nothing above -inf
    if R > 2:
        x[2, :V] = np.float16(-65504.0)  # the type's lowest value everywhere
        x[2, V // 2] = -np.inf
    temp = np.array([[1.0, 0.7, 0.3, 0.0, 2.5, -1.0][r % 6] for r in range(R)], np.float32)
    dx, out = _dev(x), t.full((R, V + pad), 7.0, device="cuda")
    for tmp in (temp, None):
        out.fill_(7.0)
        L.softmax_rows(_ptr(dx), V + pad, _ptr(_dev(tmp)) if tmp is not None else None, R, V, _ptr(out), V + pad)
        t.cuda.synchronize()
        got = out.cpu().numpy().astype(np.float64)
        assert np.all(got[:, V:] == 7.0)
        for r in range(R):
            want = tm.softmax_row(x[r, :V], 1.0 if tmp is None else float(tmp[r]))
            # exponent (v - m) / t in fp32: two roundings of 2^-24 each; exp, sum and quotient: 2^-20
            big = np.abs(np.log(np.maximum(want, 1e-45)))
            tol = want * (big * 2.0 ** -22 + 2.0 ** -20) + 2.0 ** -126
            assert np.all(np.abs(got[r, :V] - want) <= tol), (r, np.abs(got[r, :V] - want).max())


def test_softmax_nan_and_inf():
    """A NaN makes its row NaN, +inf too (inf - inf), as softmax does; other rows are untouched by it."""
    t = torch()
    x = np.zeros((4, 40), np.float16)
    x[0, 3], x[2, 5] = np.nan, np.inf
    out = t.zeros((4, 40), device="cuda")
    L.softmax_rows(_ptr(_dev(x)), 40, None, 4, 40, _ptr(out), 40)
    t.cuda.synchronize()
    got = out.cpu().numpy()
    assert np.isnan(got[0]).all() and np.isnan(got[2, 5])
    assert np.all(got[1] == np.float32(1 / 40)) and np.all(got[3] == np.float32(1 / 40))


def test_softmax_extreme_temperatures():
    """The largest and smallest temperatures, infinity and NaN: entries of -inf stay 0 and no NaN appears."""
    t = torch()
    V, temps = 300, [np.inf, 3e38, 1e30, 1e-30, 1e-44, np.nan, -np.inf]
    rng = np.random.default_rng(11)
    x = np.tile((rng.standard_normal(V) * 4).astype(np.float16), (len(temps), 1))
    x[:, 5::7] = -np.inf
    top = x[0] == x[0].max()
    out = t.zeros((len(temps), V), device="cuda")
    L.softmax_rows(_ptr(_dev(x)), V, _ptr(_dev(np.array(temps, np.float32))), len(temps), V, _ptr(out), V)
    t.cuda.synchronize()
    got = out.cpu().numpy().astype(np.float64)
    flat = np.where(np.isinf(x[0]), 0.0, 1.0 / np.isfinite(x[0]).sum())
    sharp = np.where(top, 1.0 / top.sum(), 0.0)
    for r, want in enumerate([flat] * 3 + [sharp] * 4):
        # equal shares but for the quotient's and the exponential's roundings; exponents below 2^-20 vanish
        assert np.all(np.abs(got[r] - want) <= want * 2.0 ** -20), (r, temps[r])


# ------------------------------------------------------------------ verification
def _verify(target, draft, token, parent, u, tree_len=None, pad=0):
    t = torch()
    B, N, V = target.shape
    if pad:
        target = np.concatenate([target, np.full((B, N, pad), 9.0, np.float32)], 2)
        draft = None if draft is None else np.concatenate([draft, np.full((B, N, pad), 9.0, np.float32)], 2)
    dt, dd = _dev(target), None if draft is None else _dev(draft)
    path, acc, nxt = _i32(np.full((B, N), 5)), _i32(np.full(B, 5)), _i32(np.full(B, 5))
    L.tree_verify(_ptr(dt), V + pad, _ptr(dd), V + pad, _ptr(_i32(token)), _ptr(_i32(parent)),
                  None if tree_len is None else _ptr(_i32(tree_len)), _ptr(_dev(u)), B, N, V, _ptr(path), _ptr(acc),
                  _ptr(nxt))
    t.cuda.synchronize()
    return path.cpu().numpy(), acc.cpu().numpy(), nxt.cpu().numpy()


def _soft(x):
    e = np.exp(x - x.max(-1, keepdims=True))
    return (e / e.sum(-1, keepdims=True)).astype(np.float32)


def _draws(rng, B, N, V, spread, with_draft, chain=False, sharp=3.0):
    x = rng.standard_normal((B, N, V)) * sharp
    target, draft = _soft(x), _soft(x + spread * rng.standard_normal((B, N, V)))
    parent = np.array([_parents(rng, N, chain) for _ in range(B)])
    token = np.zeros((B, N), np.int64)
    for b in range(B):
        for i in range(1, N):
            q = draft[b, parent[b, i]].astype(np.float64)
            token[b, i] = rng.choice(V, p=q / q.sum()) if with_draft else np.argsort(-q)[int((parent[b, :i] ==
                                                                                            parent[b, i]).sum()) % V]
    return target, draft if with_draft else None, token, parent, rng.random((B, N)).astype(np.float32)


def _same(got, target, draft, token, parent, u, tree_len=None):
    path, acc, nxt = got
    some = 0
    for b in range(len(target)):
        n = target.shape[1] if tree_len is None else max(0, min(target.shape[1], tree_len[b]))
        want = tm.verify(target[b], None if draft is None else draft[b], token[b], parent[b], n, u[b])
        if want is None:
            assert acc[b] == -1 and nxt[b] == -1 and np.all(path[b] == -1)
            continue
        assert acc[b] == len(want[0]) and nxt[b] == want[1], (b, acc[b], nxt[b], want)
        assert path[b].tolist() == want[0] + [-1] * (path.shape[1] - len(want[0]))
        some += len(want[0])
    return some


@pytest.mark.parametrize("with_draft", [True, False])
@pytest.mark.parametrize("B,N,V,spread,pad", [(1, 1, 100, 1.0, 0), (40, 8, 37, 1.0, 0), (64, 32, 500, 0.7, 1),
                                              (9, 64, 1000, 2.0, 4), (3, 256, 64, 0.3, 0), (2, 6, 151936, 0.8, 0),
                                              (2, 6, 151935, 0.8, 0), (200, 5, 1, 1.0, 0), (30, 12, 129, 1.0, 3)])
def test_verify(B, N, V, spread, pad, with_draft):
    rng = np.random.default_rng(B + V)
    case = _draws(rng, B, N, V, spread, with_draft)
    _same(_verify(*case, pad=pad), *case)


def test_verify_edges():
    """Bad tokens and parents are never tried, empty trees, numbers at 0 and just under 1, distributions
    with zeros, NaN, negatives, all zero, and drafts equal to the target (nothing left after a refusal)."""
    rng = np.random.default_rng(4)
    B, N, V = 12, 7, 50
    target, draft, token, parent, u = _draws(rng, B, N, V, 1.0, True)
    token[0, 1:3], token[1, 1] = -1, V
    parent[2, 3], parent[2, 4], parent[2, 5] = 3, 6, -7
    u[3], u[4] = 0.0, np.nextafter(np.float32(1), np.float32(0))
    target[5], draft[5] = 0.0, 0.0
    target[6, :, ::2], draft[6, :, 1::2] = np.nan, -0.5
    target[7, :, 3:] = 0.0
    draft[8] = target[8]
    target[9, :, 10] = 0.0
    target[9, :, 20:] = 0.0
    u[9, 0] = 1.0 - 2.0 ** -24
    lens = [7, 7, 7, 7, 7, 7, 7, 7, 7, 7, 0, -3]
    _same(_verify(target, draft, token, parent, u, lens), target, draft, token, parent, u, lens)
    _same(_verify(target, None, token, parent, u, lens), target, None, token, parent, u, lens)


def test_verify_repeated_siblings():
    """The same token several times under one node."""
    rng = np.random.default_rng(6)
    target, draft, token, parent, u = _draws(rng, 64, 6, 4, 1.5, True, sharp=0.5)
    parent[:] = [-1, 0, 0, 0, 0, 0]
    token[:, 1:] = rng.integers(0, 2, (64, 5))
    u[:, 1:] = 0.6 + 0.39 * u[:, 1:]
    for d in (draft, None):
        _same(_verify(target, d, token, parent, u), target, d, token, parent, u)


def test_verify_is_distributed_as_the_target():
    """20000 sequences with the same distributions and fresh draws: the first emitted token follows the
    target's distribution.  Each frequency has standard deviation sqrt(p (1 - p) / n): five of them."""
    rng = np.random.default_rng(8)
    n, V = 20000, 8
    p, q = _soft(rng.standard_normal((1, V))), _soft(rng.standard_normal((1, V)))
    target, draft = np.broadcast_to(p, (n, 4, V)).copy(), np.broadcast_to(q, (n, 4, V)).copy()
    parent = np.broadcast_to([-1, 0, 0, 1], (n, 4)).copy()
    qq = q[0].astype(np.float64)
    token = rng.choice(V, size=(n, 4), p=qq / qq.sum())
    path, acc, nxt = _verify(target, draft, token, parent, rng.random((n, 4)).astype(np.float32))
    first = np.where(acc > 0, token[np.arange(n), np.maximum(path[:, 0], 0)], nxt)
    f = np.bincount(first, minlength=V) / n
    assert np.all(np.abs(f - p[0]) < 5 * np.sqrt(p[0] * (1 - p[0]) / n)), (f, p)


# ------------------------------------------------------------------ commit
@pytest.mark.parametrize("layers,KV,pad", [(1, 16, 0), (3, 2, 16)])
def test_commit(layers, KV, pad):
    t = torch()
    rng = np.random.default_rng(layers)
    B, N, rows, slots = 8, 20, 30, 9
    cols = KV * D
    stride = cols + pad
    f16 = lambda *s: rng.standard_normal(s).astype(np.float16)  # noqa: E731
    TK, TV = f16(layers, B, N, cols), f16(layers, B, N, cols)
    K, V = f16(layers, slots, rows, stride), f16(layers, slots, rows, stride)
    slot, lens = [8, 0, 3, 2, 5, 99, 6, 7], [0, 5, 26, 30, 29, 3, 31, 4]
    acc = [3, 0, 7, 2, 4, 2, 2, -1]
    path = np.full((B, N), -1)
    for b in range(B):
        path[b, :max(acc[b], 0)] = np.sort(1 + rng.permutation(N - 1)[:max(acc[b], 0)])
    path[0, 1] = 400  # outside the tree: its row stays
    wk, wv, wl = K.copy(), V.copy(), list(lens)
    for b in range(B):
        if acc[b] < 0 or not 0 <= slot[b] < slots or lens[b] > rows:
            continue
        for r in range(min(1 + acc[b], rows - lens[b])):
            node = path[b, r - 1] if r else 0
            if 0 <= node < N:
                wk[:, slot[b], lens[b] + r, :cols], wv[:, slot[b], lens[b] + r, :cols] = TK[:, b, node], TV[:, b, node]
            wl[b] += 1
    d = [_dev(x) for x in (TK, TV, K, V)]
    out, dl = _i32([7] * B), _i32(lens)
    args = (_ptr(d[0]), _ptr(d[1]), B * N * cols, _ptr(d[2]), _ptr(d[3]), slots * rows * stride, stride, rows, slots,
            _ptr(_i32(slot)), _ptr(dl), _ptr(_i32(path)), _ptr(_i32(acc)), B, N, KV, layers)
    keep = [_i32(slot), _i32(path), _i32(acc)]
    L.tree_commit(*args[:9], _ptr(keep[0]), _ptr(dl), _ptr(keep[1]), _ptr(keep[2]), B, N, KV, layers, _ptr(out))
    t.cuda.synchronize()
    assert np.array_equal(d[2].cpu().numpy().view(np.int16), wk.view(np.int16))
    assert np.array_equal(d[3].cpu().numpy().view(np.int16), wv.view(np.int16))
    assert out.tolist() == wl and dl.tolist() == lens
    L.tree_commit(*args[:9], _ptr(keep[0]), _ptr(dl), _ptr(keep[1]), _ptr(keep[2]), B, N, KV, layers, None)
    t.cuda.synchronize()  # the same call again: the same caches
    assert np.array_equal(d[2].cpu().numpy().view(np.int16), wk.view(np.int16))


# ------------------------------------------------------------------ together
class Step:
    """A step of speculative decoding for B sequences: one attention layer whose output is projected to
    logits (gemm_tc), then probabilities, verification and commit."""

    def __init__(self, seed, B, N, H, lens, V, room):
        t = torch()
        rng = np.random.default_rng(seed)
        self.B, self.N, self.H, self.V, self.rows = B, N, H, V, room
        W = H * D
        parents = [_parents(rng, N) for _ in range(B)]
        lay = [L.tree_layout(p) for p in parents]
        f16 = lambda *s: _dev(rng.standard_normal(s).astype(np.float16))  # noqa: E731
        self.qkv, self.bias = f16(B, N, 3 * W), f16(3 * W)
        self.K, self.V_ = f16(B, room, W), f16(B, room, W)
        self.head = _dev((rng.standard_normal((V, W)) * 0.3).astype(np.float16))
        self.depth, self.mask = _i32([d for d, _ in lay]), _dev(np.stack([m.view(np.int64) for _, m in lay]))
        self.parent, self.lens, self.parents = _i32(parents), _i32(lens), parents
        self.token, self.u = _i32(rng.integers(0, V, (B, N))), _dev(rng.random((B, N)).astype(np.float32))
        z = lambda *s, dt=t.float16: t.zeros(s, dtype=dt, device="cuda")  # noqa: E731
        self.Q, self.TK, self.TV, self.O = z(B, N, W), z(B, N, W), z(B, N, W), z(B, N, W)
        self.logits, self.probs = z(B * N, V), z(B * N, V, dt=t.float32)
        self.temp = t.full((B * N,), 0.8, device="cuda")
        self.path, self.acc, self.next, self.len_out = (z(*s, dt=t.int32) for s in ((B, N), (B,), (B,), (B,)))
        self.nb = L.tree_attn_work_bytes(B, N, H, H, room)
        self.work = z((self.nb + 3) // 4, dt=t.float32)

    def run(self, stream=None):
        B, N, H, V, W = self.B, self.N, self.H, self.V, self.H * D
        L.tree_rope(_ptr(self.qkv), _ptr(self.bias), _ptr(self.depth), _ptr(self.lens), None, B, N, H, H, 10000.0,
                    _ptr(self.Q), _ptr(self.TK), _ptr(self.TV), stream)
        L.tree_attn(_ptr(self.Q), W, _ptr(self.K), _ptr(self.V_), W, self.rows, B, None, _ptr(self.lens), self.rows,
                    _ptr(self.TK), _ptr(self.TV), _ptr(self.mask), None, B, N, H, H, _ptr(self.O), W, _ptr(self.work),
                    self.nb, stream)
        L.gemm_tc(_ptr(self.O), _ptr(self.head), _ptr(self.logits), B * N, V, W, stream)
        L.softmax_rows(_ptr(self.logits), V, _ptr(self.temp), B * N, V, _ptr(self.probs), V, stream)
        L.tree_verify(_ptr(self.probs), V, None, 0, _ptr(self.token), _ptr(self.parent), None, _ptr(self.u), B, N, V,
                      _ptr(self.path), _ptr(self.acc), _ptr(self.next), stream)
        L.tree_commit(_ptr(self.TK), _ptr(self.TV), 0, _ptr(self.K), _ptr(self.V_), 0, W, self.rows, B, None,
                      _ptr(self.lens), _ptr(self.path), _ptr(self.acc), B, N, H, 1, _ptr(self.len_out), stream)
        return self


def test_a_whole_step_equals_sequential_decoding():
    """Rope, attention, logits, probabilities, verification and commit in a row; afterwards plain flash decoding
    (llmdiy_fd_multihead) over the committed cache, one accepted node after the other, gives the attention
    that the tree gave, and the verified path is the definition's."""
    t = torch()
    B, N, H, V, room = 3, 12, 16, 24, 800
    s = Step(11, B, N, H, [500, 0, 63], V, room)
    # every node's token among the likely ones, so that some are accepted
    s.run()
    t.cuda.synchronize()
    s.token.copy_(s.probs.view(B, N, V)[t.arange(B, device="cuda")[:, None], s.parent.clamp(min=0).long()].argmax(-1))
    s.run()
    t.cuda.synchronize()
    assert L.tree_attn_status(_ptr(s.work)) == 0 and L.gemm_tc_status() == 0
    probs = s.probs.view(B, N, V).cpu().numpy()
    accepted = _same((s.path.cpu().numpy(), s.acc.cpu().numpy(), s.next.cpu().numpy()), probs, None,
                     s.token.cpu().numpy(), s.parent.cpu().numpy(), s.u.cpu().numpy())
    assert accepted > 0
    lens = s.lens.tolist()
    for b in range(B):
        rows = [0] + s.path[b, : int(s.acc[b])].tolist()
        assert int(s.len_out[b]) == lens[b] + len(rows)
        for r, node in enumerate(rows):
            m = lens[b] + r + 1
            assert t.equal(s.K[b, m - 1], s.TK[b, node])
            nb = L.fd_mh_work_bytes(m, H)
            w, O = t.zeros((nb + 3) // 4, device="cuda"), t.zeros(H * D, dtype=t.float16, device="cuda")
            L.fd_multihead(_ptr(s.Q[b, node]), _ptr(s.K[b]), _ptr(s.V_[b]), _ptr(O), m, H * D, H, _ptr(w), nb)
            t.cuda.synchronize()
            assert float((O.float() - s.O[b, node].float()).abs().max()) < 2e-3, (b, r)


def test_a_step_captured_and_replayed_on_another_stream():
    """The step captured once into a graph and replayed on another stream with other lengths and numbers gives
    what calling it gives; two steps with workspaces of their own run on two streams at once."""
    t = torch()
    a, b = (Step(21, 2, 9, 16, [100, 300], 1000, 600) for _ in range(2))
    for s in (a, b):  # what a first call sets is set outside the capture; both commit the same rows
        s.run()
    t.cuda.synchronize()
    st = t.cuda.Stream()
    g = t.cuda.CUDAGraph()
    with t.cuda.graph(g, stream=st):
        a.run(st.cuda_stream)
    for lens, seed in (([0, 591], 1), ([64, 1], 2)):
        u = t.rand((2, 9), generator=t.Generator(device="cuda").manual_seed(seed), device="cuda")
        for s in (a, b):
            s.lens.copy_(_i32(lens))
            s.u.copy_(u)
        t.cuda.synchronize()
        with t.cuda.stream(st):
            g.replay()
        other = t.cuda.Stream()
        b.run(other.cuda_stream)
        t.cuda.synchronize()
        for x in ("Q", "TK", "TV", "O", "logits", "probs", "path", "acc", "next", "len_out", "K", "V_"):
            assert t.equal(getattr(a, x), getattr(b, x)), x


# ------------------------------------------------------------------ long and many
# Long caches of several sequences go in equal ranges over all SMs (flat), the others a cluster to a unit (direct):
# the tests above are mostly direct, these are flat.
@pytest.mark.parametrize("length", [40000, 26000 + 63])
def test_attn_nothing_leaks_in_a_long_cache(length):
    N = 24
    a = Attn(length, 2, N, 4, 2, [length, length], max_len=length + 70, tree_len=[24, 20])
    for s in range(2):
        a.K[s, length:] = np.nan
        a.V[s, length:] = np.inf
        a.V[s, length + 1:] = np.nan
    a.TK[1, 20:], a.TV[1, 20:] = np.inf, np.nan
    a.TV[0, 7, 5], a.TV[0, 9, 130], a.TK[0, 11, 3] = np.nan, -np.inf, np.nan
    a.device().call()
    with np.errstate(invalid="ignore"):
        a.check(rows=150)
    clean = [i for i in range(N) if not {7, 9, 11} & a.sees[0][i]]
    assert np.isfinite(a.d["O"].cpu().numpy()[0, clean, :4 * D]).all()


def test_attn_long_cache_with_empty_rows_and_two_tree_tiles():
    rng = np.random.default_rng(5)
    N = 100
    sees = [[set() if i % 3 == 0 else set(np.nonzero(rng.random(N) < 0.2)[0].tolist()) for i in range(N)]
            for _ in range(3)]
    a = Attn(6, 3, N, 4, 2, [30000, 0, 511], max_len=30001, tree_len=[100, 70, 30], sees=sees, pad=8)
    a.device().call().check(rows=200)
    assert np.all(a.d["O"].cpu().numpy()[1, 0, :4 * D] == 0.0)


def test_attn_many_sequences_of_all_lengths():
    """More sequences than a warp has lanes, several of them reading one slot, lengths from none to 13000."""
    rng = np.random.default_rng(12)
    B = 70
    lens = [int(x) for x in np.exp(rng.uniform(0, np.log(13000), B))]
    lens[3], lens[40], lens[69] = 0, 13000, 12999
    tl = [int(x) for x in rng.integers(0, 6, B)]
    a = Attn(13, B, 5, 2, 1, lens, max_len=13000, tree_len=tl, slots=[b % 3 for b in range(B)], num_slots=3)
    a.device().call().check(rows=400)


def test_attn_many_short_sequences():
    rng = np.random.default_rng(14)
    B = 300
    a = Attn(15, B, 4, 4, 2, [int(x) for x in rng.integers(0, 130, B)], max_len=130)
    a.device().call().check(rows=400)


def test_attn_long_captured_and_on_two_streams():
    """A flat call (two launches) captured, replayed with other lengths, beside an eager one on another stream."""
    t = torch()
    a, b = (Attn(31, 2, 20, 4, 2, [40000, 31000], max_len=40000).device() for _ in range(2))
    a.call()
    t.cuda.synchronize()
    st, other = t.cuda.Stream(), t.cuda.Stream()
    g = t.cuda.CUDAGraph()
    with t.cuda.graph(g, stream=st):
        a.call(st.cuda_stream)
        a.call(st.cuda_stream)  # the second in a row on one workspace
    for lens in ([39999, 64], [1, 40000], [0, 0]):
        a.lens = b.lens = lens
        for x in (a, b):
            x.d["len"].copy_(_i32(lens))
            x.d["O"].fill_(7.0)
        t.cuda.synchronize()
        with t.cuda.stream(st):
            g.replay()
        b.call(other.cuda_stream)
        t.cuda.synchronize()
        assert t.equal(a.d["O"], b.d["O"])
        a.check(rows=20)


def test_softmax_many_rows_of_odd_length():
    """More rows than clusters run at once, each starting at another alignment: no row sees its neighbours."""
    t = torch()
    for R, V in ((80, 151935), (900, 1001)):
        g = t.Generator(device="cuda").manual_seed(R)
        x = t.randn(R, V, generator=g, device="cuda", dtype=t.float16) * 3
        x[::3] += 20  # neighbours of other sizes
        x[1::7, : V // 2] = -float("inf")
        out = t.zeros(R, V, device="cuda")
        L.softmax_rows(_ptr(x), V, None, R, V, _ptr(out), V)
        want = t.softmax(x.double(), 1)
        big = want.clamp(min=1e-45).log().abs()
        tol = want * (big * 2.0 ** -22 + 2.0 ** -20) + 2.0 ** -126
        assert bool(((out.double() - want).abs() <= tol).all()), (R, V)


def test_softmax_and_verify_past_32_bit_offsets():
    """Rows that begin more than 2^31 entries after the first."""
    t = torch()
    N, V, B = 256, 151936, 57
    assert (B * N - 1) * V > 2 ** 31
    logits = t.zeros(B * N, V, dtype=t.float16, device="cuda")
    g = t.Generator(device="cuda").manual_seed(3)
    logits[-N:] = t.randn(N, V, generator=g, device="cuda", dtype=t.float16) * 3
    probs = t.empty(B * N, V, device="cuda")
    L.softmax_rows(_ptr(logits), V, None, B * N, V, _ptr(probs), V)
    t.cuda.synchronize()
    for r in (B * N - 1, B * N - N, B * N - N - 1):
        want = t.softmax(logits[r].double(), 0)
        tol = want * (want.log().abs() * 2.0 ** -22 + 2.0 ** -20)
        assert bool(((probs[r].double() - want).abs() <= tol).all()), r
    rng = np.random.default_rng(2)
    parent = np.array([_parents(rng, N)] * B)
    token = np.zeros((B, N), np.int64)
    last = probs[-N:].cpu().numpy()
    token[-1] = last.argmax(1)[np.maximum(parent[-1], 0)]
    u = rng.random((B, N)).astype(np.float32)
    path, acc, nxt = _i32(np.zeros((B, N))), _i32(np.zeros(B)), _i32(np.zeros(B))
    L.tree_verify(_ptr(probs), V, None, 0, _ptr(_i32(token)), _ptr(_i32(parent)), None, _ptr(_dev(u)), B, N, V, _ptr(path),
                  _ptr(acc), _ptr(nxt))
    t.cuda.synchronize()
    want = tm.verify(last, None, token[-1], parent[-1], N, u[-1])
    assert int(acc[-1]) == len(want[0]) and int(nxt[-1]) == want[1]
    assert path[-1, : len(want[0])].tolist() == want[0]
