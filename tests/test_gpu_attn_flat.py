"""Tree attention (llmdiy_tree_attn, include/llmdiy_tree.h) in the flat order: all units' keys dealt in equal ranges over
the SMs, cut units joined by a second launch. Every case asserts that it takes this way."""
import numpy as np
import pytest

import llmdiy_b200 as L
import treemath as tm
from gpu_util import torch
from test_gpu_tree import Attn, D, _free_after_the_test, _i32, _parents  # noqa: F401

pytestmark = pytest.mark.gpu


def _flat(a):
    assert L.tree_attn_path(a.B, a.N, a.H, a.KV, a.max_len) == 0
    return a


def _twice(a, rows):
    """The call, checked, and the same bits again."""
    a.call()
    first = a.d["O"].clone()
    a.call()
    if a.give_tree_len:
        a.tree_len = [min(max(n, 0), a.N) for n in a.tree_len]
    a.check(rows=rows)
    assert torch().equal(first, a.d["O"])


@pytest.mark.parametrize("B,N,H,KV,lens,max_len,tree_len", [
    (1, 20, 8, 1, [33000], None, None), (2, 40, 8, 1, [33000, 64], None, [40, 10]), (2, 70, 1, 1, [33000, 17], None, None),
    (3, 100, 8, 1, [13000, 500, 0], None, [100, 7, 17]), (1, 200, 4, 1, [32999], 33000, None),
    (6, 256, 8, 1, [6000, 1, 0, 5999, 64, 3000], None, [256, 255, 16, 0, 65, 900]),
    (8, 200, 8, 1, [6000, 100, 4000, 6000, 0, 65, 1, 129], None, [1, 200, 129, 3, 128, 0, 64, -4]),
    (1, 1, 8, 1, [131072], None, None), (1, 1, 8, 1, [63], 131072, None), (3, 90, 8, 2, [0, 0, 0], 20000, [90, 2, 0])])
def test_flat_matches(B, N, H, KV, lens, max_len, tree_len):
    """Trees of one M tile and of up to sixteen, some of them ending before the later tiles; one to four tiles of tree rows;
    caches from none to the longest, and all of them far shorter than max_len."""
    _twice(_flat(Attn(B * 91 + N, B, N, H, KV, lens, max_len=max_len, tree_len=tree_len, pad=8)).device(), 120)


def test_flat_masks_that_leave_rows_empty():
    """M tiles side by side, masks of any pattern; rows that see nothing of an empty cache are zeros."""
    rng = np.random.default_rng(7)
    N = 100
    sees = [[set() if i % 3 == 0 else set(np.nonzero(rng.random(N) < 0.2)[0].tolist()) for i in range(N)]
            for _ in range(3)]
    a = _flat(Attn(16, 3, N, 8, 1, [13000, 0, 511], max_len=13001, tree_len=[100, 70, 20], sees=sees, pad=8)).device()
    _twice(a, 250)
    got = a.d["O"].cpu().numpy()
    assert all(np.all(got[1, i, :8 * D] == 0.0) for i in range(0, 70, 3))


@pytest.mark.parametrize("length", [12936, 13000])
def test_flat_nothing_leaks_from_unseen_rows(length):
    """NaN and infinities past the lengths, past the trees and in tree rows of both tiles that only some nodes see."""
    N = 100
    a = _flat(Attn(length, 3, N, 8, 1, [length, 70, 0], max_len=13100, tree_len=[100, 80, 17]))
    for b in range(3):
        a.K[b, a.lens[b]:], a.V[b, a.lens[b]:] = np.nan, np.inf
        a.V[b, a.lens[b] + 1:] = np.nan
        a.TK[b, a.tree_len[b]:], a.TV[b, a.tree_len[b]:] = np.inf, np.nan
        a.TV[b, 9, 5], a.TK[b, 11, 3] = np.nan, np.nan
    a.TV[0, 70, 100], a.TV[1, 65, 0] = -np.inf, np.nan
    a.device().call()
    with np.errstate(invalid="ignore"):
        a.check(rows=400)
    got = a.d["O"].cpu().numpy()
    for b in range(3):
        clean = [i for i in range(a.tree_len[b]) if not {9, 11, 65, 70} & a.sees[b][i]]
        assert len(clean) > 5 and np.isfinite(got[b, clean, :8 * D]).all()


def test_flat_workspace_serves_smaller_calls():
    """One workspace, sized for the largest, for calls of other sizes back to back: partials of both are written."""
    big = _flat(Attn(1, 4, 64, 8, 1, [50000, 50, 900, 49999])).device()
    few = _flat(Attn(2, 2, 7, 8, 1, [33000, 3])).device()
    for other in (few, _flat(Attn(3, 2, 40, 8, 1, [33000, 3], tree_len=[40, 9])).device()):
        assert other.n <= big.n
        for _ in range(2):
            big.call()
            other.call(work=big.d["work"], work_bytes=big.n)
        big.check(rows=100)
        other.check(rows=100)


def test_flat_captured_with_other_trees_and_lengths():
    """A graph of two calls on one workspace, M tiles side by side, replayed while lengths, trees and masks change, beside
    eager calls on another stream."""
    t = torch()
    N = 100
    a, b = (_flat(Attn(31, 3, N, 8, 1, [13000, 12000, 0], tree_len=[100, 1, 30])).device() for _ in range(2))
    a.call()
    t.cuda.synchronize()
    st, other = t.cuda.Stream(), t.cuda.Stream()
    g = t.cuda.CUDAGraph()
    with t.cuda.graph(g, stream=st):
        a.call(st.cuda_stream)
        a.call(st.cuda_stream)
    rng = np.random.default_rng(3)
    for lens, trees in (([12999, 64, 5], [3, 100, 100]), ([1, 13000, 0], [64, 65, 0]), ([0, 0, 0], [100, 16, 17])):
        sees = [tm.layout(_parents(rng, N))[1] for _ in range(3)]
        mask = np.stack([tm.mask_words(s, N) for s in sees])
        for x in (a, b):
            x.lens, x.tree_len, x.sees = lens, trees, sees
            x.d["len"].copy_(_i32(lens))
            x.d["tree_len"].copy_(_i32(trees))
            x.d["mask"].copy_(t.from_numpy(mask))
            x.d["O"].fill_(7.0)
        t.cuda.synchronize()
        with t.cuda.stream(st):
            g.replay()
        b.call(other.cuda_stream)
        t.cuda.synchronize()
        assert t.equal(a.d["O"], b.d["O"])
        a.check(rows=80)
