"""What the speculative-decoding kernels report when a bounded wait expires: a build of them whose waits all expire at once
(_build/libllmdiy_expired.so), without a fault on the GPU. The library itself works as before afterwards."""
import ctypes
import os

import numpy as np
import pytest

import llmdiy_b200 as L
import test_gpu_tree as T
from gpu_util import torch
from test_gpu_tree import _free_after_the_test, _i32, _ptr  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.fixture
def expired(monkeypatch):
    """Calls within the test go to the build whose waits expire; returns what takes them back."""
    real = L.lib()
    small = ctypes.CDLL(os.path.join(os.path.dirname(L.LIB_PATH), "libllmdiy_expired.so"))
    for name in ("llmdiy_tree_verify", "llmdiy_tree_commit"):
        getattr(small, name).argtypes = getattr(real, name).argtypes
        getattr(small, name).restype = getattr(real, name).restype
    monkeypatch.setattr(L, "_lib", small)
    return lambda: monkeypatch.setattr(L, "_lib", real)


@pytest.mark.parametrize("B,N,V,with_draft", [(1, 5, 3000, True), (3, 8, 500, False), (200, 4, 100, True)])
def test_verify_reports_an_expired_wait(expired, B, N, V, with_draft):
    """accepted -2 and next -1, whatever the walk had come to, and a commit of that moves nothing; empty trees, which wait
    for nothing, are told as always."""
    t = torch()
    case = T._draws(np.random.default_rng(B), B, N, V, 1.0, with_draft)
    lens = [0 if b == 2 else N for b in range(B)]
    path, acc, nxt = T._verify(*case, tree_len=lens)
    assert acc.tolist() == [-1 if b == 2 else -2 for b in range(B)] and np.all(nxt == -1)
    rows = t.ones(B, N, 128, dtype=t.float16, device="cuda")
    K, V_ = (t.zeros(B, 9, 128, dtype=t.float16, device="cuda") for _ in range(2))
    out, at, a, p = _i32([7] * B), _i32([3] * B), _i32(acc), _i32(path)
    L.tree_commit(_ptr(rows), _ptr(rows), 0, _ptr(K), _ptr(V_), 0, 128, 9, B, None, _ptr(at), _ptr(p), _ptr(a), B, N, 1, 1,
                  _ptr(out))
    t.cuda.synchronize()
    assert out.tolist() == [3] * B and not K.any() and not V_.any()
    expired()
    T._same(T._verify(*case, tree_len=lens), *case, lens)
