"""The tree's rotary angles (llmdiy_tree_rope, include/llmdiy_tree.h) where an error of the angle shows as it is: pairs (1, 0)
and (0, 1), whose outputs are the cosine and sine, at positions where one of them nearly vanishes."""
import numpy as np
import pytest

import llmdiy_b200 as L
from gpu_util import torch
from test_gpu_tree import D, _dev, _free_after_the_test, _i32, _ptr  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("base", [10000.0, 1000000.0, 1.0, 0.25])
def test_rope_angles_at_far_positions(base):
    t = torch()
    pos = np.array([573204, 260515, 885893, 52174, 781545, 833719, 312689, 521030, 11, 22, 355, 710, 0, 1, (1 << 20) - 1,
                    1 << 20, (1 << 24) - 3, 16367173, -1, -355], np.int64)
    B = len(pos)
    for first in (1.0, 0.0):
        qkv = np.zeros((B, 1, 3 * D), np.float16)
        qkv[:, 0, :2 * D].reshape(B, 2, 2, 64)[...] = np.array([first, 1 - first], np.float16)[:, None]
        Q, TK, TV = (t.full((B, D), 7.0, dtype=t.float16, device="cuda") for _ in range(3))
        L.tree_rope(_ptr(_dev(qkv)), None, _ptr(_i32(np.full(B, 5))), _ptr(_i32(pos - 5)), None, B, 1, 1, 1, base, _ptr(Q),
                    _ptr(TK), _ptr(TV))
        t.cuda.synchronize()
        i = np.arange(64)
        a = pos[:, None].astype(np.longdouble) * np.exp2(-i.astype(np.longdouble) / 64 * np.log2(np.longdouble(base)))
        c, s = np.cos(a).astype(np.float64), np.sin(a).astype(np.float64)
        want = np.concatenate([c, s] if first else [-s, c], 1)
        # the header's 2^-21 of cosine and sine, a product and a sum in fp32 (2^-24 each), half a step of fp16
        tol = 2.0 ** -21 + 2.0 ** -22 + np.maximum(np.abs(want) * 2.0 ** -11, 2.0 ** -25)
        near = np.abs(a).astype(np.float64) <= 2.0 ** 24  # what the header gives the bound for
        near = np.concatenate([near, near], 1)
        for x in (Q, TK):
            err = np.abs(x.cpu().numpy().astype(np.float64) - want)
            assert np.all((err <= tol) | ~near), (first, np.argwhere((err > tol) & near)[:4])
        assert bool((TV == 0).all())
