"""Cases, plain forms and exact values of the speculative-decoding operators (include/llmdiy_tree.h).

A step of speculative decoding scores a tree of drafted tokens per sequence in one pass: the nodes'
Q/K/V get their bias and rotary positions (`rope`), attend the sequence's cache and their ancestors
(`attn`), the logits become probabilities (`softmax`), the drafts are verified against them from given
random numbers (`verify`), and the accepted nodes' K/V rows move into the caches (`commit`).

`run(state)` computes one pass in elementary torch operations, or, with `own` set, with the library's
kernels; `exact(case, seed)` computes the same from the definitions in 64 bits.
"""
import math
import os
import sys

import torch

own = False

D = 128          # head dimension
ROPE_BASE = 10000.0
VOCAB = 151936   # the engine's vocabulary


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one new token of one conversation, attending a short cache: the latency of a plain decode step
        dict(name="attn one token", op="attn", B=1, N=1, heads=16, kv=16, max_len=1023, ragged=False),
        # one conversation, a 26-node draft tree, just under 2048 rows of context
        dict(name="attn tree", op="attn", B=1, N=26, heads=16, kv=16, max_len=2047, ragged=False),
        # a batch of 16 requests of every age, 64-node trees of different sizes
        dict(name="attn batch", op="attn", B=16, N=64, heads=16, kv=16, max_len=4160, ragged=True),
        # two long documents, four query heads to a K/V head (192 query rows to a K/V row)
        dict(name="attn long grouped", op="attn", B=2, N=48, heads=32, kv=8, max_len=65536, ragged=False),
        # a chain of four drafts of one conversation, drawn from the draft model's distribution
        dict(name="verify chain", op="verify", B=1, N=5, V=VOCAB, draft=True, spread=0.5),
        # a batch of trees drawn from the draft model's distributions; siblings compete
        dict(name="verify batch", op="verify", B=24, N=32, V=VOCAB, draft=True, spread=0.9),
        # the five logits rows of that chain, each with its temperature
        dict(name="softmax chain", op="softmax", R=5, V=VOCAB),
        # the logits rows of a batch of trees
        dict(name="softmax batch", op="softmax", R=768, V=VOCAB),
        # one conversation's tree in one layer
        dict(name="rope tree", op="rope", B=1, N=26, heads=16, kv=16, max_len=2047),
        # a batch of trees in one layer, long contexts
        dict(name="rope batch", op="rope", B=24, N=64, heads=32, kv=8, max_len=131072),
        # the accepted rows of one conversation, all 24 layers
        dict(name="commit one", op="commit", B=1, N=26, kv=16, layers=24, rows=512),
        # the accepted rows of a batch, all 24 layers
        dict(name="commit batch", op="commit", B=32, N=64, kv=16, layers=24, rows=200),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attn", "attn", "attn", "verify", "verify", "softmax", "rope", "commit"])
    heads, kv = rng.choice([(16, 16), (32, 8), (12, 12), (16, 2), (20, 4), (32, 32)])
    if op == "attn":
        B, N = _log(rng, 1, 32), _log(rng, 1, 128)
        # at most the longest listed case's cache rows x heads, and its query rows x cache rows
        top = min(131072, 2 * 65536 * 8 // (B * kv), 2 * 65536 * 48 * 32 // (B * N * heads))
        return dict(op=op, B=B, N=N, heads=heads, kv=kv, max_len=_log(rng, 16, top), ragged=rng.random() < 0.7)
    if op == "verify":
        V = _log(rng, 1000, VOCAB)
        B = _log(rng, 1, 24)
        N = _log(rng, 1, min(64, 24 * 32 * VOCAB // (B * V)))
        return dict(op=op, B=B, N=N, V=V, draft=rng.random() < 0.7, spread=round(rng.uniform(0.1, 1.5), 3))
    if op == "softmax":
        V = _log(rng, 1000, VOCAB)
        return dict(op=op, R=_log(rng, 1, min(4096, 768 * VOCAB // V)), V=V)
    if op == "rope":
        N = _log(rng, 1, 256)
        return dict(op=op, B=_log(rng, 1, max(1, min(64, 1536 // N))), N=N, heads=heads, kv=kv,
                    max_len=_log(rng, 16, 131072))
    N = _log(rng, 1, 128)
    rows = _log(rng, N + 2, 400)
    layers = rng.choice([1, 12, 24, 31])
    most = max(1, min(64, 32 * 200 * 24 * 16 // (rows * layers * kv)))
    return dict(op=op, B=_log(rng, 1, most), N=N, kv=kv, layers=layers, rows=rows)


def _lens(case):
    """Committed rows of each sequence: all max_len, or spread from a few to max_len in mixed order."""
    B, M = case["B"], case["max_len"]
    if not case.get("ragged", True):
        return [M] * B
    return [max(0, M - (M * ((5 * b) % B)) // B - (3 * b) % 7) for b in range(B)]


def _tree_lens(case):
    """Nodes of each sequence's tree: N, some of them fewer."""
    N = case["N"]
    return [max(1, N - (N * (b % 4)) // 9) for b in range(case["B"])]


def _accepted(case):
    """Accepted nodes of each sequence, none to eight, as the tree and the cache leave room."""
    room = min(8, case["N"] - 1)
    return [(3 * b + 4) % (room + 1) for b in range(case["B"])]


def work(case):
    op = case["op"]
    if op == "attn":
        H, KV = case["heads"], case["kv"]
        rows = sum(_lens(case))
        nodes = sum(_tree_lens(case))
        pairs = sum(n * (m + 1) for n, m in zip(_tree_lens(case), _lens(case)))  # a node sees itself at least
        words = (case["N"] + 63) // 64
        return {"bytes": (rows + nodes) * KV * D * 4 + nodes * (H * D * 4 + 8 * words), "flops": 4 * D * H * pairs}
    if op == "verify":
        # a row of the target's (and one of the draft's) probabilities per sequence: the last token's draw
        B, N, V = case["B"], case["N"], case["V"]
        rows = 2 if case["draft"] and N > 1 else 1
        return {"bytes": B * (4 * V * rows + 12 * N), "flops": B * V * (2 * rows)}
    if op == "softmax":
        return {"bytes": case["R"] * case["V"] * 6, "flops": case["R"] * case["V"] * 4}
    if op == "rope":
        cols = (case["heads"] + 2 * case["kv"]) * D
        nodes = sum(_tree_lens(case))
        return {"bytes": nodes * (4 * cols + 4) + 2 * cols, "flops": nodes * cols * 4}
    moved = sum(1 + a for a in _accepted(case))
    return {"bytes": moved * case["kv"] * D * 2 * 2 * 2 * case["layers"], "flops": 0}


# ------------------------------------------------------------------ inputs
def _parents(case, seed):
    """Parents in breadth-first order: non-decreasing, node 0 the root (-1)."""
    import random
    r = random.Random(seed)
    out = []
    for _ in range(case["B"]):
        p = sorted(int(i * r.random() ** 0.7) for i in range(1, case["N"]))
        out.append([-1] + [min(v, i) for i, v in enumerate(p)])
    return out


def _depths(parents):
    out = []
    for p in parents:
        d = [0] * len(p)
        for i in range(1, len(p)):
            d[i] = d[p[i]] + 1
        out.append(d)
    return out


def _mask_words(parents, N):
    """Bit j of a node's words: it sees node j (itself and its ancestors)."""
    W = (N + 63) // 64
    out = []
    for p in parents:
        bits = []
        for i in range(N):
            bits.append((bits[p[i]] if i else 0) | (1 << i))
        out.append([[((b >> (64 * w)) & (2**64 - 1)) for w in range(W)] for b in bits])
    return [[[x - 2**64 if x >= 2**63 else x for x in n] for n in s] for s in out]


def _randn16(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float16)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    i32 = dict(device="cuda", dtype=torch.int32)
    op, s = case["op"], {"case": case}
    if op == "attn":
        B, N, H, KV, M = case["B"], case["N"], case["heads"], case["kv"], case["max_len"]
        s["rows"] = M + 8  # rows of a slot
        s["Q"] = _randn16(g, B, N, H * D) * 1.5
        s["K"], s["V"] = _randn16(g, B, s["rows"], KV * D), _randn16(g, B, s["rows"], KV * D)
        s["TK"], s["TV"] = _randn16(g, B, N, KV * D), _randn16(g, B, N, KV * D)
        s["mask"] = torch.tensor(_mask_words(_parents(case, seed), N), device="cuda", dtype=torch.int64)
        s["len"] = torch.tensor(_lens(case), **i32)
        s["tree_len"] = torch.tensor(_tree_lens(case), **i32)
        # slots of a pool, in another order than the sequences
        s["slot"] = torch.randperm(B, generator=g, device="cuda").to(torch.int32)
        s["O"] = torch.zeros(B, N, H * D, device="cuda", dtype=torch.float16)
        if own:
            n = _lib().tree_attn_work_bytes(B, N, H, KV, M)
            s["work"], s["work_bytes"] = torch.zeros((n + 3) // 4, device="cuda"), n
    elif op == "verify":
        B, N, V = case["B"], case["N"], case["V"]
        parents = _parents(case, seed)
        s["parent"] = torch.tensor(parents, **i32)
        # next-token distributions of a language model are peaked: a few likely tokens, a long tail
        x = torch.randn(B, N, V, generator=g, device="cuda") * 3.0
        s["target"] = torch.softmax(x, -1)
        x.add_(torch.randn(B, N, V, generator=g, device="cuda"), alpha=case["spread"])
        q = torch.softmax(x, -1)
        del x
        up = torch.tensor(parents, device="cuda").clamp(min=0)
        if case["draft"]:  # node i's token is drawn from its parent's draft distribution
            c = q.double().cumsum(-1)
            c = c.gather(1, up[:, :, None].expand(-1, -1, V))
            t = torch.rand(B, N, 1, generator=g, device="cuda", dtype=torch.float64) * c[..., -1:]
            s["token"] = torch.searchsorted(c, t, right=True).squeeze(-1).clamp(max=V - 1).to(torch.int32)
            s["draft"] = q
            del c
        else:  # deterministic drafts: siblings are their parent's likeliest tokens, in order
            rank = torch.tensor([[sum(p[j] == p[i] for j in range(1, i)) for i in range(N)] for p in parents],
                                device="cuda")
            top = q.topk(min(V, N), -1).indices
            s["token"] = top[torch.arange(B, device="cuda")[:, None], up, rank].to(torch.int32)
            s["draft"] = None
        s["tree_len"] = torch.tensor(_tree_lens(case), **i32)
        s["uniform"] = torch.rand(B, N, generator=g, device="cuda")
        s["path"] = torch.zeros(B, N, **i32)
        s["accepted"], s["next"] = torch.zeros(B, **i32), torch.zeros(B, **i32)
    elif op == "softmax":
        R, V = case["R"], case["V"]
        s["logits"] = _randn16(g, R, V) * 3.0
        # one row in four has its unlikely tokens cut off, as top-k sampling does
        cut = (torch.arange(R, device="cuda") % 4 == 1)[:, None] & (s["logits"] < 4.0)
        s["logits"][cut] = -math.inf
        s["temp"] = torch.rand(R, generator=g, device="cuda") * 1.4 + 0.1
        s["temp"][3::8] = 0.0  # greedy requests
        s["probs"] = torch.zeros(R, V, device="cuda")
    elif op == "rope":
        B, N, H, KV = case["B"], case["N"], case["heads"], case["kv"]
        s["qkv"] = _randn16(g, B, N, (H + 2 * KV) * D)
        s["bias"] = _randn16(g, (H + 2 * KV) * D) * 0.5
        s["depth"] = torch.tensor(_depths(_parents(case, seed)), **i32)
        s["len"] = torch.tensor(_lens(case), **i32)
        s["tree_len"] = torch.tensor(_tree_lens(case), **i32)
        s["Q"] = torch.zeros(B, N, H * D, device="cuda", dtype=torch.float16)
        s["TK"] = torch.zeros(B, N, KV * D, device="cuda", dtype=torch.float16)
        s["TV"] = torch.zeros(B, N, KV * D, device="cuda", dtype=torch.float16)
    else:
        B, N, KV, NL, R = case["B"], case["N"], case["kv"], case["layers"], case["rows"]
        acc = _accepted(case)
        s["K"], s["V"] = _randn16(g, NL, B, R, KV * D), _randn16(g, NL, B, R, KV * D)
        s["TK"], s["TV"] = _randn16(g, NL, B, N, KV * D), _randn16(g, NL, B, N, KV * D)
        path = torch.full((B, N), -1, dtype=torch.int32)
        cpu = torch.Generator().manual_seed(seed)
        for b in range(B):
            path[b, :acc[b]] = (1 + torch.randperm(N - 1, generator=cpu)[:acc[b]]).sort().values.to(torch.int32)
        s["path"], s["accepted"] = path.cuda(), torch.tensor(acc, **i32)
        s["len"] = torch.tensor([(R - 9) * (b + 1) // (B + 1) if R > 9 else 0 for b in range(B)], **i32)
        s["slot"] = torch.randperm(B, generator=g, device="cuda").to(torch.int32)
        s["len_out"] = torch.zeros(B, **i32)
    return s


# ------------------------------------------------------------------ one pass
_module = None


def _lib():
    global _module
    if _module is None:
        sys.path.insert(0, os.path.join(os.getcwd(), "llm-inference-diy_b200"))
        import llmdiy_b200
        _module = llmdiy_b200
    return _module


def run(state):
    op = state["case"]["op"]
    if own:
        return _OWN[op](state, _lib())
    return _PLAIN[op](state)


def _own_attn(s, L):
    c = s["case"]
    L.tree_attn(s["Q"].data_ptr(), c["heads"] * D, s["K"].data_ptr(), s["V"].data_ptr(), c["kv"] * D, s["rows"], c["B"],
                s["slot"].data_ptr(), s["len"].data_ptr(), c["max_len"], s["TK"].data_ptr(), s["TV"].data_ptr(),
                s["mask"].data_ptr(), s["tree_len"].data_ptr(), c["B"], c["N"], c["heads"], c["kv"],
                s["O"].data_ptr(), c["heads"] * D, s["work"].data_ptr(), s["work_bytes"])
    return s["O"]


def _plain_attn(s):
    c = s["case"]
    B, N, H, KV, M = c["B"], c["N"], c["heads"], c["kv"], c["max_len"]
    at = s["slot"].long()
    k = torch.cat([s["K"][at, :M], s["TK"]], 1).float().view(B, M + N, KV, D).permute(0, 2, 3, 1)
    v = torch.cat([s["V"][at, :M], s["TV"]], 1).float().view(B, M + N, KV, D).permute(0, 2, 1, 3)
    q = s["Q"].float().view(B, N, KV, H // KV, D).permute(0, 2, 1, 3, 4).reshape(B, KV, N * (H // KV), D)
    node = torch.arange(N, device="cuda")
    alive = node < s["tree_len"][:, None]
    tree = (s["mask"][:, :, node // 64] >> (node % 64)) & 1 == 1
    tree &= alive[:, None, :]
    cached = (torch.arange(M, device="cuda") < s["len"][:, None])[:, None, :].expand(B, N, M)
    seen = torch.cat([cached, tree], 2)[:, None, :, None, :]  # [B, 1, N, 1, M + N]
    x = (q @ k).view(B, KV, N, H // KV, M + N).mul_(1.0 / math.sqrt(D)).masked_fill_(~seen, -math.inf)
    x.sub_(x.amax(-1, keepdim=True).clamp_(min=-3e38)).exp_()
    total = x.sum(-1, keepdim=True)
    o = (x.view(B, KV, N * (H // KV), M + N) @ v).view(B, KV, N, H // KV, D) / total.clamp_(min=1e-38)
    o = o.permute(0, 2, 1, 3, 4).reshape(B, N, H * D)
    return torch.where(alive[:, :, None], o, 0.0).half()


def _own_verify(s, L):
    c = s["case"]
    L.tree_verify(s["target"].data_ptr(), c["V"], s["draft"].data_ptr() if c["draft"] else None, c["V"],
                  s["token"].data_ptr(), s["parent"].data_ptr(), s["tree_len"].data_ptr(), s["uniform"].data_ptr(),
                  c["B"], c["N"], c["V"], s["path"].data_ptr(), s["accepted"].data_ptr(), s["next"].data_ptr())
    return s["path"], s["accepted"], s["next"]


def _plain_verify(s):
    c = s["case"]
    B, N, V = c["B"], c["N"], c["V"]
    p, q = s["target"], s["draft"]
    each = torch.arange(B, device="cuda")
    cur = torch.zeros(B, device="cuda", dtype=torch.long)
    count = torch.zeros_like(cur)
    path = torch.full((B, N + 1), -1, device="cuda", dtype=torch.int32)
    zero = torch.zeros(B, device="cuda", dtype=torch.float64)
    one = torch.ones_like(zero)
    T, S = zero, one  # what is left of the target: max(0, p - T q), its sum S
    left = p[:, 0].double()
    for i in range(1, N):  # the walk through the tree; every step handles the whole batch
        x = s["token"][:, i].long()
        tried = (s["parent"][:, i] == cur) & (i < s["tree_len"])
        u = s["uniform"][:, i].double()
        w = left[each, x]
        qx = q[each, cur, x].double() if q is not None else one
        took = tried & (u * S * qx < w)
        lost = tried & ~took
        path[each, torch.where(took, count, N)] = i
        count = count + took
        cur = torch.where(took, i, cur)
        pc = p[each, cur].double()
        if q is not None:
            T = torch.where(took, zero, torch.where(lost, T + S, T))
            left = (pc - T[:, None] * q[each, cur].double()).clamp_(min=0.0)
            S = torch.where(took, one, torch.where(lost, left.sum(-1), S))
        else:
            left = torch.where(took[:, None], pc, left)
            S = torch.where(took, one, torch.where(lost, S - w, S))
            left[each, x] = torch.where(lost, zero, left[each, x])
    run_ = left.cumsum(-1)
    some = run_[:, -1:] > 0
    run_ = torch.where(some, run_, p[each, cur].double().cumsum(-1))
    token = (run_ <= s["uniform"][:, :1].double() * run_[:, -1:]).sum(-1).clamp(max=V - 1)
    return path[:, :N], count.int(), token.int()


def _own_softmax(s, L):
    c = s["case"]
    L.softmax_rows(s["logits"].data_ptr(), c["V"], s["temp"].data_ptr(), c["R"], c["V"], s["probs"].data_ptr(), c["V"])
    return s["probs"]


def _plain_softmax(s):
    x = s["logits"].float()
    top = x.amax(-1, keepdim=True)
    d = x - top.clamp(min=-3e38)
    t = s["temp"][:, None]
    e = torch.where(t > 0, (d / t).exp(), (d == 0).float())
    return e / e.sum(-1, keepdim=True).clamp(min=1e-38)


def _own_rope(s, L):
    c = s["case"]
    L.tree_rope(s["qkv"].data_ptr(), s["bias"].data_ptr(), s["depth"].data_ptr(), s["len"].data_ptr(),
                s["tree_len"].data_ptr(), c["B"], c["N"], c["heads"], c["kv"], ROPE_BASE,
                s["Q"].data_ptr(), s["TK"].data_ptr(), s["TV"].data_ptr())
    return s["Q"], s["TK"], s["TV"]


def _plain_rope(s):
    c = s["case"]
    B, N, H, KV = c["B"], c["N"], c["heads"], c["kv"]
    y = (s["qkv"].float() + s["bias"].float()).view(B, N, H + 2 * KV, 2, D // 2)
    t = torch.arange(D // 2, device="cuda", dtype=torch.float64)
    a = (s["len"][:, None] + s["depth"]).double()[..., None] * ROPE_BASE ** (-2.0 * t / D)
    cos, sin = a.cos().float()[:, :, None], a.sin().float()[:, :, None]
    y1, y2 = y[..., 0, :], y[..., 1, :]
    turned = torch.cat([y1 * cos - y2 * sin, y2 * cos + y1 * sin], -1)
    alive = (torch.arange(N, device="cuda") < s["tree_len"][:, None])[:, :, None, None]
    turned = torch.where(alive, turned, 0.0).half()
    tv = torch.where(alive, y[:, :, H + KV:].reshape(B, N, KV, D), 0.0).half()
    return (turned[:, :, :H].reshape(B, N, H * D), turned[:, :, H:H + KV].reshape(B, N, KV * D),
            tv.reshape(B, N, KV * D))


def _own_commit(s, L):
    c = s["case"]
    cols = c["kv"] * D
    L.tree_commit(s["TK"].data_ptr(), s["TV"].data_ptr(), c["B"] * c["N"] * cols, s["K"].data_ptr(), s["V"].data_ptr(),
                  c["B"] * c["rows"] * cols, cols, c["rows"], c["B"], s["slot"].data_ptr(), s["len"].data_ptr(),
                  s["path"].data_ptr(), s["accepted"].data_ptr(), c["B"], c["N"], c["kv"], c["layers"],
                  s["len_out"].data_ptr())
    return s["K"], s["V"], s["len_out"]


def _plain_commit(s):
    c = s["case"]
    B, N = c["B"], c["N"]
    src = torch.cat([torch.zeros(B, 1, device="cuda", dtype=torch.long), s["path"].long()], 1)[:, :N]
    place = torch.arange(N, device="cuda").expand(B, N)
    keep = place <= s["accepted"][:, None]
    # places past the accepted rows write the root's row to its own place once more
    src = torch.where(keep, src, 0)
    dst = s["len"].long()[:, None] + torch.where(keep, place, 0)
    each = torch.arange(B, device="cuda")[:, None]
    at = s["slot"].long()[:, None]
    s["K"][:, at, dst] = s["TK"][:, each, src]
    s["V"][:, at, dst] = s["TV"][:, each, src]
    return s["K"], s["V"], s["len"] + 1 + s["accepted"]


_OWN = {"attn": _own_attn, "verify": _own_verify, "softmax": _own_softmax, "rope": _own_rope, "commit": _own_commit}
_PLAIN = {"attn": _plain_attn, "verify": _plain_verify, "softmax": _plain_softmax, "rope": _plain_rope,
          "commit": _plain_commit}


# ------------------------------------------------------------------ exact values
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "attn":
        B, N, H, KV = case["B"], case["N"], case["heads"], case["kv"]
        out = torch.zeros(B, N, H, D, device="cuda", dtype=torch.float64)
        slots, lens, trees = s["slot"].tolist(), s["len"].tolist(), s["tree_len"].tolist()
        words = s["mask"].tolist()
        for b in range(B):
            m, n = lens[b], trees[b]
            seen = torch.tensor([[1 if (words[b][i][j // 64] >> (j % 64)) & 1 else 0 for j in range(n)]
                                 for i in range(n)], device="cuda").bool().view(n, n)
            for h in range(H):
                at = slice((h * KV // H) * D, (h * KV // H + 1) * D)
                q = s["Q"][b, :n, h * D:(h + 1) * D].double()
                old = q @ s["K"][slots[b], :m, at].double().T
                new = (q @ s["TK"][b, :n, at].double().T).masked_fill(~seen, -math.inf)
                x = torch.cat([old, new], 1) / math.sqrt(D)
                w = torch.exp(x - torch.logsumexp(x, 1, keepdim=True))
                out[b, :n, h] = w[:, :m] @ s["V"][slots[b], :m, at].double() + w[:, m:] @ s["TV"][b, :n, at].double()
        return out.view(B, N, H * D)
    if op == "softmax":
        x = s["logits"].double()
        out = torch.zeros_like(x)
        for r, t in enumerate(s["temp"].tolist()):
            if t == 0:
                top = x[r] == x[r].max()
                out[r] = top.double() / top.sum()
            else:
                out[r] = torch.softmax(x[r] / t, 0)
        return out
    if op == "rope":
        B, N, H, KV = case["B"], case["N"], case["heads"], case["kv"]
        z = (s["qkv"].double() + s["bias"].double()).view(B, N, H + 2 * KV, D)
        half = torch.arange(D // 2, device="cuda", dtype=torch.float64)
        angle = (s["len"].double()[:, None] + s["depth"].double())[..., None] / ROPE_BASE ** (half / (D // 2))
        z = z * (torch.arange(N, device="cuda")[None] < s["tree_len"][:, None])[..., None, None]
        w = torch.complex(z[:, :, :H + KV, :D // 2], z[:, :, :H + KV, D // 2:]) * torch.polar(
            torch.ones_like(angle), angle)[:, :, None]
        y = torch.cat([w.real, w.imag], -1)
        return (y[:, :, :H].reshape(B, N, H * D), y[:, :, H:].reshape(B, N, KV * D),
                z[:, :, H + KV:].reshape(B, N, KV * D))
    return None  # whole numbers and copies
