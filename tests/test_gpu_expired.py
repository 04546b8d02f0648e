"""What the speculative-decoding kernels report when a bounded wait expires: a build of them whose waits all expire at once
(_build/libllmdiy_expired.so), without a fault on the GPU. The library itself works as before afterwards."""
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
    """Calls within the test go to the build whose waits expire; returns what takes them back to the library."""
    real, path = L.lib(), L.LIB_PATH
    monkeypatch.setattr(L, "LIB_PATH", os.path.join(os.path.dirname(path), "libllmdiy_expired.so"))
    monkeypatch.setattr(L, "_lib", None)

    def back():
        monkeypatch.setattr(L, "LIB_PATH", path)
        monkeypatch.setattr(L, "_lib", real)

    yield back
    back()


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


@pytest.mark.parametrize("B,N,H,KV,lens,max_len,path", [
    (2, 1, 4, 4, [1000, 3], None, 2), (1, 4, 2, 2, [1000], None, 2), (2, 9, 4, 2, [700, 0], None, 1),
    (1, 100, 4, 2, [1500], None, 1), (1, 8, 16, 2, [9000], None, 1), (3, 100, 8, 1, [12000, 500, 0], 13000, 0),
    (1, 20, 2, 1, [32000], 33000, 0)])
def test_attn_reports_an_expired_wait(expired, B, N, H, KV, lens, max_len, path):
    """Status -5, once; the same buffers then serve the library as if nothing had been."""
    a = T.Attn(B + N, B, N, H, KV, lens, max_len=max_len).device()
    assert L.tree_attn_path(B, N, H, KV, a.max_len) == path
    a.call()
    torch().cuda.synchronize()
    assert [L.tree_attn_status(_ptr(a.d["work"])) for _ in range(2)] == [-5, 0]
    expired()
    a.call().check(rows=100)


@pytest.mark.parametrize("R,V", [(3, 1000), (90, 40000), (5, 151936), (700, 9001), (40, 170000)])
def test_softmax_marks_what_an_expired_wait_left(expired, R, V):
    """NaN in every entry of a call none of whose waits succeeds, nothing past the rows; the library is as before."""
    t = torch()
    x = t.randn(R, V, device="cuda", dtype=t.float16, generator=t.Generator(device="cuda").manual_seed(V))
    out = t.full((R, V + 3), 7.0, device="cuda")
    L.softmax_rows(_ptr(x), V, None, R, V, _ptr(out), V + 3)
    t.cuda.synchronize()
    assert bool(t.isnan(out[:, :V]).all()) and bool((out[:, V:] == 7.0).all())
    expired()
    L.softmax_rows(_ptr(x), V, None, R, V, _ptr(out), V + 3)
    want = t.softmax(x.double(), 1)
    tol = want * (want.log().abs() * 2.0 ** -22 + 2.0 ** -20)
    assert bool(((out[:, :V].double() - want).abs() <= tol).all()) and bool((out[:, V:] == 7.0).all())
