"""Greedy verification (include/llmdiy_tree.h) where logits tie: against softmax rows of temperature 0, whose tied maxima share
the probability, and against rows that hold 1 at the winner of llmdiy_argmax, which follow the engine's greedy decoding."""
import numpy as np
import pytest

import llmdiy_b200 as L
from gpu_util import torch
from test_gpu_tree import _dev, _free_after_the_test, _parents, _ptr, _same, _verify  # noqa: F401

pytestmark = pytest.mark.gpu


def _tied_logits(rng, B, N, V):
    """fp16 logits, most rows with two to six equal maxima."""
    x = (rng.standard_normal((B, N, V)) * 2).astype(np.float16)
    top = x.max(-1)
    for b in range(B):
        for i in range(N):
            x[b, i, rng.choice(V, int(rng.integers(1, 7)), replace=False)] = top[b, i]
    return x


def _drafts(rng, x, parent):
    """Each node's token: some maximum of its parent's row, or now and then anything."""
    B, N, V = x.shape
    token = np.zeros((B, N), np.int64)
    for b in range(B):
        for i in range(1, N):
            row = x[b, parent[b, i]]
            token[b, i] = rng.choice(np.nonzero(row == row.max())[0]) if rng.random() < 0.9 else rng.integers(0, V)
    return token


@pytest.mark.parametrize("B,N,V", [(40, 9, 50), (4, 16, 32000), (2, 7, 151936)])
def test_rows_of_temperature_0_share_ties(B, N, V):
    t = torch()
    rng = np.random.default_rng(V)
    x = _tied_logits(rng, B, N, V)
    parent = np.array([_parents(rng, N) for _ in range(B)])
    token = _drafts(rng, x, parent)
    u = rng.random((B, N)).astype(np.float32)
    u[0], u[1] = 0.0, 1 - 2.0 ** -24
    probs = t.zeros(B, N, V, device="cuda")
    L.softmax_rows(_ptr(_dev(x)), V, _ptr(_dev(np.zeros(B * N, np.float32))), B * N, V, _ptr(probs), V)
    t.cuda.synchronize()
    p = probs.cpu().numpy()
    got = _verify(p, None, token, parent, u)
    assert _same(got, p, None, token, parent, u) > 0
    for b in range(B):  # every emitted token is a maximum of its row
        path, n = got[0][b], got[1][b]
        nodes = [0] + path[:n].tolist()
        for c, tok in zip(nodes, [token[b, i] for i in nodes[1:]] + [got[2][b]]):
            assert x[b, c, tok] == x[b, c].max()


@pytest.mark.parametrize("B,N,V", [(12, 9, 50), (2, 12, 32000), (2, 7, 151936)])
def test_rows_of_the_argmax_winner_follow_greedy_decoding(B, N, V):
    """Accepted is the chain of nodes whose tokens are the winners, next is the last one's winner: token for token what a
    step at a time with llmdiy_argmax gives, whatever the uniform numbers."""
    t = torch()
    rng = np.random.default_rng(V + 1)
    x = _tied_logits(rng, B, N, V)
    dx, won = _dev(x), t.zeros(B, N, dtype=t.int32, device="cuda")
    for b in range(B):
        for i in range(N):
            L.argmax(_ptr(won[b, i]), _ptr(dx[b, i]), V)
    t.cuda.synchronize()
    winner = won.cpu().numpy()
    parent = np.array([_parents(rng, N) for _ in range(B)])
    token = _drafts(rng, x, parent)
    for b in range(B):  # half of the nodes continue with the winner itself
        for i in range(1, N, 2):
            token[b, i] = winner[b, parent[b, i]]
    target = t.zeros(B, N, V, device="cuda").scatter_(2, won.long()[..., None], 1.0).cpu().numpy()
    several = 0
    for kind in (0.0, 0.5, 1 - 2.0 ** -24):
        path, acc, nxt = _verify(target, None, token, parent, np.full((B, N), kind, np.float32))
        for b in range(B):
            c, want = 0, []
            while True:
                kids = [i for i in range(1, N) if parent[b, i] == c and token[b, i] == winner[b, c]]
                if not kids:
                    break
                c = kids[0]
                want.append(c)
            assert path[b, :acc[b]].tolist() == want and nxt[b] == winner[b, c]
            several += len(want)
    assert several > 3
