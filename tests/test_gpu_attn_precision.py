"""Precision of the tree attention's probabilities (llmdiy_tree_attn, include/llmdiy_tree.h) where a bound per
probability shows: rows dominated by a few keys whose values are 0, so that the output is made of small probabilities
alone, and values that cancel. Scores are exact (powers of two), so the bounds hold only what the kernels round."""
import numpy as np
import pytest

import llmdiy_b200 as L
import treemath as tm
from gpu_util import torch
from test_gpu_tree import Attn, D, _free_after_the_test  # noqa: F401  (the fixture ends every test here too)

pytestmark = pytest.mark.gpu


def _score(a, rows, exponent):
    """Gives the cache rows `rows` of every slot the score -exponent * ln 2 (nearly), all others 0."""
    a.Q[...] = 0
    for i in range(a.N):
        for h in range(a.H):
            a.Q[:, i, h * D + (i + h) % 8] = 16.0  # (one dim of eight: another one for each node)
    for x in (a.K, a.TK):
        x[...] = 0
    for g in range(a.KV):
        a.K[:, rows, g * D:g * D + 8] = np.float16(-exponent * np.log(2.0) * np.sqrt(128.0) / 16.0)


def _check(a, bits):
    torch().cuda.synchronize()
    got = a.d["O"].cpu().numpy().astype(np.float64)
    for b in range(a.B):
        for i in sorted({0, a.N // 2, a.N - 1}):
            for h in sorted({0, a.H - 1}):
                cols = slice(h * a.KV // a.H * D, (h * a.KV // a.H + 1) * D)
                js, m = sorted(a.sees[b][i]), a.lens[b]
                K = np.concatenate([a.K[b, :m, cols], a.TK[b, js][:, cols]])
                V = np.concatenate([a.V[b, :m, cols], a.TV[b, js][:, cols]])
                o, tol = tm.attention_row_close(a.Q[b, i, h * D:(h + 1) * D], K, V, bits)
                err = np.abs(got[b, i, h * D:(h + 1) * D] - o)
                assert np.all(err <= tol), (b, i, h, float((err / tol).max()), float((err / np.abs(o)).max()))


# trees of one M tile and of two, one sequence and several, caches for clusters and for the flat order
SHAPES = [(1, 26, 16, 16, 2047), (4, 8, 16, 16, 1000), (1, 100, 4, 2, 1500), (1, 64, 2, 2, 500), (1, 5, 2, 1, 300),
          (2, 8, 8, 1, 33000), (3, 100, 8, 1, 13000), (1, 2, 1, 1, 1000)]


@pytest.mark.parametrize("exponent", [14.3, 18.6, 22.4, 24.6, 26.1, 30.2])
@pytest.mark.parametrize("B,N,H,KV,room", SHAPES)
def test_attn_small_probabilities_beside_dominating_keys(B, N, H, KV, room, exponent):
    """The first key of every 64 dominates and its value is 0: the output is what the small probabilities add up to."""
    m = min(room, 2047)
    a = Attn(N, B, N, H, KV, [m - 3 * b for b in range(B)], max_len=room)
    _score(a, slice(0, None, 64), -exponent)
    for x in (a.V, a.TV):
        x[...] = (1000 + 3000 * np.abs(np.sin(np.arange(x.size)))).reshape(x.shape).astype(np.float16)
    a.V[:, ::64] = 0
    # (a node sees itself: a key of score 0 with a value like the others)
    assert L.tree_attn_path(B, N, H, KV, room) == (2 if N * H // KV <= 4 else 0 if room > 3000 else 1)
    a.device().call()
    _check(a, 22)


@pytest.mark.parametrize("drop", [0.46875, 0.9140625, 1.45703125])
@pytest.mark.parametrize("B,N,H,KV,room", SHAPES + [(1, 8, 16, 16, 64), (2, 8, 16, 16, 64), (1, 1, 128, 1, 200),
                                                    (1, 100, 1, 1, 200), (2, 70, 1, 1, 33000)])
def test_attn_values_that_cancel(B, N, H, KV, room, drop):
    """Half of 64 keys has probability 1 (relative), half one that fp16 rounds by 1.7 to 1.9 quarters of its step
    2^-10, with values that cancel: what is left of the output is that rounding, whatever else is in the call."""
    a = Attn(N, B, N, H, KV, [64] * B, max_len=room, sees=[[set()] * N for _ in range(B)])
    _score(a, slice(1, None, 2), 0.0)
    p = np.exp(-16.0 * drop / np.sqrt(128.0))
    for g in range(KV):
        a.K[:, 1::2, g * D:g * D + 8] = np.float16(-drop)
    v = 1 + np.abs(np.sin(np.arange(a.V[:, ::2].size))).reshape(a.V[:, ::2].shape)
    a.V[:, ::2] = v.astype(np.float16)
    a.V[:, 1::2] = (-a.V[:, ::2][:, : a.V[:, 1::2].shape[1]].astype(np.float64) / p).astype(np.float16)
    a.device().call()
    _check(a, 22)


@pytest.mark.parametrize("size", [300.0, 3000.0, 10000.0])
@pytest.mark.parametrize("B,N,H,KV,room", [(1, 26, 16, 16, 2047), (1, 100, 4, 2, 1500), (2, 8, 8, 1, 33000),
                                           (3, 100, 8, 1, 13000), (1, 2, 1, 1, 1000)])
def test_attn_scores_of_any_size(B, N, H, KV, room, size):
    """Scores of up to 2^36 doublings: a row's largest takes all, to the last bit of the output."""
    m = min(room, 2047)
    a = Attn(N, B, N, H, KV, [m - 3 * b for b in range(B)], max_len=room)
    for x in (a.Q, a.K, a.TK):
        x[...] = (x.astype(np.float32) * size).astype(np.float16)
    a.device().call()
    torch().cuda.synchronize()
    got = a.d["O"].cpu().numpy()
    seen = 0
    for b in range(B):
        for i in range(0, N, 5):
            for h in range(H):
                cols = slice(h * KV // H * D, (h * KV // H + 1) * D)
                js = sorted(a.sees[b][i])
                K = np.concatenate([a.K[b, :a.lens[b], cols], a.TK[b, js][:, cols]]).astype(np.float64)
                V = np.concatenate([a.V[b, :a.lens[b], cols], a.TV[b, js][:, cols]])
                q = a.Q[b, i, h * D:(h + 1) * D].astype(np.float64)
                s = K @ q / np.sqrt(128.0)
                first, second = np.argsort(s)[[-1, -2]]
                # sums of 128 products, each addition within 2^-23 of the products' sizes, and 64 more doublings
                if s[first] - s[second] > (np.abs(K) @ np.abs(q)).max() * 128 * 2.0 ** -23 + 64:
                    seen += 1
                    assert np.array_equal(got[b, i, h * D:(h + 1) * D], V[first]), (b, i, h)
    assert seen >= 2 * ((N + 4) // 5) * H * B // 3
