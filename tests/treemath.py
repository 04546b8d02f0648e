"""Plain restatements of the speculative-decoding operators (include/llmdiy_tree.h) in 64 bits, written
from the definitions, one sequence and one node at a time.  numpy on the host."""
import numpy as np


def layout(parent):
    n = len(parent)
    depth, sees = [0] * n, [set() for _ in range(n)]
    for i in range(n):
        j, d = i, -1
        while j >= 0:
            sees[i].add(j)
            j, d = parent[j], d + 1
        depth[i] = d
    return depth, sees


def mask_words(sees, N):
    """[N][ceil(N/64)] int64 words of a list of sets (missing rows: 0)."""
    W = (N + 63) // 64
    out = np.zeros((N, W), np.uint64)
    for i, s in enumerate(sees):
        for j in s:
            out[i, j // 64] |= np.uint64(1) << np.uint64(j % 64)
    return out.view(np.int64)


def attention_row(q, K, V, allowed_dtype=np.float64):
    """(softmax(q K^T / sqrt(d)) V, bound on the kernel's error) for one query over rows K, V (may be none).

    The bound: probabilities are rounded to fp16 relative to a running maximum (2^-11 of each, at least
    2^-25 absolute of the largest, which is at least 1), scores carry fp32 rounding (2^-14 relative on a probability
    covers |score| up to 2^8 at 2^-23), and the output is rounded to fp16 (2^-11 relative, 2^-25 absolute)."""
    if len(K) == 0:
        z = np.zeros(V.shape[1] if V.ndim == 2 else 128)
        return z, z
    s = K.astype(np.float64) @ q.astype(np.float64) / np.sqrt(len(q))
    e = np.exp(s - s.max())
    l = e.sum()
    v = V.astype(np.float64)
    o = (e / l) @ v
    err_p = np.maximum(e * (2.0 ** -11), 2.0 ** -25) + e * 2.0 ** -14
    # the sum l is of the unrounded probabilities; 2^-14 covers its fp32 rounding
    tol = (err_p / l) @ np.abs(v) + np.abs(o) * (2.0 ** -11 + 2.0 ** -14) + 2.0 ** -25
    return o, tol


def softmax_row(x, t):
    x = x.astype(np.float64)
    m = x.max()
    if m == -np.inf:
        return np.zeros_like(x)
    if not t > 0:
        e = (x == m).astype(np.float64)
    else:
        e = np.exp((x - m) / t)
    return e / e.sum()


def rope_row(x, pos, base):
    """Heads [h][128] turned to position pos."""
    t = np.arange(64)
    a = np.float64(pos) * np.float64(base) ** (-t / 64.0)
    c, s = np.cos(a), np.sin(a)
    x1, x2 = x[:, :64], x[:, 64:]
    return np.concatenate([x1 * c - x2 * s, x2 * c + x1 * s], 1)


def verify(target, draft, token, parent, n, u):
    """One sequence: (path, next) with the residual distributions formed and normalised one by one."""
    V = target.shape[1]
    pos = lambda x: np.where(x > 0, x, 0.0)  # noqa: E731  (NaN counts as 0)
    if n == 0:
        return None
    cur, path = 0, []
    while True:
        p = pos(target[cur].astype(np.float64))
        left = p.copy()  # normalised by its sum from the first refusal on (p itself counts as normalised)
        took = -1
        scale = 1.0      # left = scale * (the normalised residual)
        for i in range(1, n):
            if parent[i] != cur or not 0 <= token[i] < V:
                continue
            x = token[i]
            if draft is None:
                if float(u[i]) * scale < left[x]:
                    took = i
                    break
                scale -= left[x]
                left[x] = 0.0
            else:
                q = pos(draft[cur].astype(np.float64))
                if float(u[i]) * q[x] < left[x]:
                    took = i
                    break
                left = pos(left - q)
                if left.sum() > 0:
                    left = left / left.sum()
        if took < 0:
            break
        path.append(took)
        cur = took
    if not left.sum() > 0:
        left = p
    if not left.sum() > 0:
        return path, -1
    run = np.cumsum(left)
    hit = np.nonzero((run > float(u[0]) * run[-1]) & (left > 0))[0]
    return path, int(hit[0]) if len(hit) else int(np.nonzero(left > 0)[0][-1])


def attention_row_close(q, K, V, bits):
    """(softmax(q K^T / sqrt(d)) V, bound on the kernel's error) for a row whose scores are exact in fp32 (few powers of
    two in q and K) and lie within 32 doublings of the largest.

    The bound, relative to the largest probability: each is rounded to `bits` significant bits (half a step 2^-bits) or by
    2^-32, whichever is more (fp16 below 2^-14 has steps of 2^-24, half of one is 2^-25, and the largest is taken as 2^7 or
    more); its exponent, up to 39, is formed with two roundings of 2^-24 (39 * 2 * 2^-24 * ln 2 < 2^-17.6; 2^-22 the
    exponential). Each product entering the fp32 sums may lose 2^-23 of the sum's largest value (n products and 64 more of
    the joins), and the sum of the probabilities n / 64 + 64 roundings of 2^-24. The output is fp16 (half a step 2^-11
    relative, 2^-25 absolute)."""
    n = len(K)
    s = K.astype(np.float64) @ q.astype(np.float64) / np.sqrt(len(q))
    e = np.exp(s - s.max())
    assert e.min() > 2.0 ** -32
    l = e.sum()
    v = V.astype(np.float64)
    o, size = (e / l) @ v, (e / l) @ np.abs(v)
    err_p = np.maximum(e * 2.0 ** -bits, 2.0 ** -32) + e * 2.0 ** -17.5
    tol = (err_p / l) @ np.abs(v) + size * (n + 64) * 2.0 ** -23 + np.abs(o) * ((n / 64 + 64) * 2.0 ** -24 + 2.0 ** -11)
    return o, tol + 2.0 ** -25
