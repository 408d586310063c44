"""Decoding with a tree of drafted tokens, and weights of 4 bits: what is measured.

Four operators of one round in which a model checks a tree of drafted tokens a
sequence:

  tree    attention of the drafted tokens over the paged cache and their own
          ancestors (the pages' layout is that of ``perf/operators.py``)
  walk    the tree's masks and depths from its parents, and the path of nodes
          whose tokens are those that were sampled
  commit  K and V of the accepted nodes moved to their places, in every layer
  w4      few rows times weights of 4 bits with group scales

``run`` computes them in elementary torch operations, or, where ``own`` is
true, through the library's calls.

A sequence's n drafted tokens (its nodes, parents before children) are the last
of its ``len`` tokens: node i stands in slot len - n + i and at position
len - n + depth(i).  A mask is [nodes, words] int64: bit i % 64 of word i / 64
of a node's row is set where it attends to node i.

4-bit weights [N, K]: weight = scale * code + shift of its group of ``g``
neighbours along K (without shifts: scale * (code - 8)).  ``tiles`` is int32
[N / 16, K / 128, 64, 4], both rounded up: word s of lane 16 j + r holds row r's
codes of k = 128 t + 32 s + 8 j + 0 .. 7, the even ones in the nibbles of the
low half and the odd ones in those of the high half.  ``scales`` is float16
[N / 16, K / g, 16, 2] (scale, shift), or [N / 16, K / g, 16].
"""
from __future__ import annotations

import math
import random

import torch

own = False
_L = None


def listed():
    return [
        # one chat request, a small tree: latency
        dict(name="tree_one", kind="tree", cache="bf16", B=1, Hq=32, Hkv=8, D=128, page=16,
             lo=716, hi=716, nodes=16, least=16, window=0, softcap=0.0, mix=1),
        # an ordinary batch of rounds, trees and contexts of very different sizes
        dict(name="tree_batch", kind="tree", cache="bf16", B=32, Hq=32, Hkv=8, D=128, page=16,
             lo=50, hi=4096, nodes=33, least=1, window=0, softcap=0.0, mix=2),
        # wide heads over an 8-bit cache, capped scores and a sliding window, an odd batch
        dict(name="tree_window", kind="tree", cache="e4m3", B=19, Hq=16, Hkv=8, D=256, page=32,
             lo=1, hi=6000, nodes=25, least=1, window=1024, softcap=50.0, mix=3),
        # two long documents, full trees: the work is in the cache's length
        dict(name="tree_long", kind="tree", cache="bf16", B=2, Hq=32, Hkv=8, D=128, page=64,
             lo=120001, hi=131072, nodes=64, least=64, window=0, softcap=0.0, mix=4),
        # the largest: a full batch over an 8-bit cache, 256 rows a kv head
        dict(name="tree_large", kind="tree", cache="e4m3", B=64, Hq=32, Hkv=8, D=128, page=16,
             lo=500, hi=8192, nodes=64, least=64, window=0, softcap=0.0, mix=5),
        # the ends of a round: one request's tree, and a full batch of them
        dict(name="walk_one", kind="walk", B=1, nodes=26, least=26, width=8, V=32000, mix=6),
        dict(name="walk_batch", kind="walk", B=256, nodes=64, least=2, width=9, V=128256, mix=7),
        # the accepted tokens of one request, and of a batch with an 8-bit cache
        dict(name="commit_one", kind="commit", cache="bf16", B=1, L=32, Hkv=8, D=128, page=16,
             lo=90, hi=90, nodes=26, least=26, width=5, mix=8),
        dict(name="commit_batch", kind="commit", cache="e4m3", B=48, L=32, Hkv=8, D=128, page=16,
             lo=70, hi=200, nodes=64, least=20, width=9, mix=9),
        # one decoded token's projection in a layer: latency and a few MB
        dict(name="w4_token", kind="w4", M=1, N=4096, K=4096, g=128, shift=False, out="bf16"),
        # an odd number of tree nodes through a wide projection
        dict(name="w4_nodes", kind="w4", M=61, N=14336, K=4096, g=64, shift=True, out="bf16"),
        # the largest: the LM head's logits of a batch, small groups
        dict(name="w4_head", kind="w4", M=16, N=128256, K=4096, g=32, shift=True, out="f32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["tree", "tree", "tree", "walk", "commit", "w4", "w4", "w4"])
    mix = rng.randrange(1 << 30)
    if kind == "w4":
        g = rng.choice([32, 64, 128])
        K = g * max(1, round(_log(rng, 256, 14336) / g))
        return dict(kind=kind, M=_log(rng, 1, 64), N=_log(rng, 64, min(150000, 128256 * 4096 // K)),
                    K=K, g=g, shift=rng.random() < 0.5, out=rng.choice(["bf16", "f32"]))
    nodes = _log(rng, 1, 128 if kind == "walk" else 64)
    least = max(1, int(nodes * rng.choice([0.02, 0.5, 1.0])))
    if kind == "walk":
        return dict(kind=kind, B=_log(rng, 1, 256), nodes=nodes, least=least,
                    width=rng.randint(1, 12), V=_log(rng, 100, 256000), mix=mix)
    cache = rng.choice(["bf16", "bf16", "e4m3"])
    D = rng.choice([64, 128, 128, 256])
    page = rng.choice([16, 16, 32, 64, 128])
    Hkv = rng.choice([1, 2, 4, 7, 8, 8, 8, 12])
    el = 2 if cache == "bf16" else 1
    if kind == "commit":
        L = _log(rng, 1, 32)
        hi = nodes + _log(rng, 1, 400)
        most = int(1.5e9 / (L * Hkv * (hi + page) * D * 2 * el))
        return dict(kind=kind, cache=cache, B=_log(rng, 1, max(1, min(64, most))), L=L, Hkv=Hkv,
                    D=D, page=page, lo=max(nodes, hi // 3), hi=hi, nodes=nodes, least=least,
                    width=rng.randint(1, 9), mix=mix)
    Hq = Hkv * rng.choice([1, 2, 3, 4, 4, 8])
    hi = max(nodes, _log(rng, 32, 131072))
    lo = max(1, int(hi * rng.choice([0.01, 0.1, 0.5, 1.0])))
    most = min(1.0e9 / (hi * Hkv * D * 2 * el), 1.6e11 / (4.0 * hi * nodes * Hq * D))
    return dict(kind=kind, cache=cache, B=_log(rng, 1, max(1, min(256, int(most)))), Hq=Hq,
                Hkv=Hkv, D=D, page=page, lo=lo, hi=hi, nodes=nodes, least=least,
                window=rng.choice([0, 0, 0, _log(rng, 16, 4096)]),
                softcap=rng.choice([0.0, 0.0, 30.0]), mix=mix)


# ------------------------------------------------------------------ inputs
def _trees(case):
    """The sequences' lengths (drafted tokens included) and the parents of their
    nodes: part of the case, so that the work is known from it."""
    r = random.Random(case["mix"])
    lens, parents = [], []
    for _ in range(case["B"]):
        n = r.randint(case["least"], case["nodes"])
        lens.append(max(n, _log(r, case["lo"], case["hi"])) if "lo" in case else n)
        # node 0 is the last confirmed token; the others hang below recent ones
        parents.append([-1] + [r.randint(max(0, i - 9) * 2 // 3, i - 1) for i in range(1, n)])
    return lens, parents


def _words(case):
    return -(-case["nodes"] // 64)


def _masks(parents, words):
    """[nodes, words] int64 masks and the depths of one tree, as lists."""
    masks, depths = [], []
    for i, p in enumerate(parents):
        m = (masks[p] if p >= 0 else 0) | 1 << i
        masks.append(m)
        depths.append(depths[p] + 1 if p >= 0 else 0)
    split = [[m >> 64 * w & (1 << 64) - 1 for w in range(words)] for m in masks]
    return [[x - (1 << 64) if x >> 63 else x for x in m] for m in split], depths


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 7919 + 17)
    return g


def _randn(*shape, g):
    return torch.randn(*shape, generator=g, device="cuda")


def _pack_k(k, ch):
    n, H, P, D = k.shape
    return k.reshape(n, H, P, D // ch, ch).transpose(2, 3).reshape(n, H, P * D)


def _pack_v(v, ch):
    n, H, P, D = v.shape
    return v.reshape(n, H, P // ch, ch, D).transpose(3, 4).reshape(n, H, P * D)


def _pool(case, n, g):
    """One layer's pages: bf16 [n, Hkv, 2 page D], or uint8 [n, Hkv, 2 page D + 8 page]."""
    H, P, D = case["Hkv"], case["page"], case["D"]
    bf16 = case["cache"] == "bf16"
    width = 2 * P * D if bf16 else 2 * P * D + 8 * P
    pool = torch.zeros(n, H, width, dtype=torch.bfloat16 if bf16 else torch.uint8, device="cuda")
    step = max(1, (1 << 26) // (H * P * D))
    for i in range(0, n, step):
        m = min(step, n - i)
        k, v = _randn(m, H, P, D, g=g), _randn(m, H, P, D, g=g)
        part = pool[i:i + m]
        if bf16:
            part[..., :P * D] = _pack_k(k, 8)
            part[..., P * D:] = _pack_v(v, 8)
            continue
        ks, vs = k.abs().amax(3) / 448, v.abs().amax(3) / 448
        f8 = torch.float8_e4m3fn
        part[..., :P * D] = _pack_k((k / ks[..., None]).to(f8).view(torch.uint8), 16)
        part[..., P * D:2 * P * D] = _pack_v((v / vs[..., None]).to(f8).view(torch.uint8), 16)
        part[..., 2 * P * D:] = torch.cat([ks, vs], 2).view(torch.uint8)
    return pool


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _tiles(codes):
    """The tiles of codes [N, K] (both whole tiles), uint8 0 .. 15."""
    N, K = codes.shape
    x = codes.view(N // 16, 16, K // 128, 4, 4, 4, 2).int()      # [n, r, t, s, j, pair, odd]
    at = torch.tensor([[0, 16], [4, 20], [8, 24], [12, 28]], device="cuda").int()
    x = (x << at).sum((5, 6), dtype=torch.int32)                  # no two codes share a bit
    return x.permute(0, 2, 4, 1, 3).reshape(N // 16, K // 128, 64, 4).contiguous()


def prepare(case, seed):
    g = _gen(seed)
    s = dict(case)
    if case["kind"] == "w4":
        M, N, K, grp = (case[k] for k in ("M", "N", "K", "g"))
        n16, k128 = -(-N // 16) * 16, -(-K // 128) * 128
        codes = torch.zeros(n16, k128, dtype=torch.uint8, device="cuda")
        step = max(1, (1 << 27) // k128 // 16) * 16
        s["tiles"] = torch.zeros(n16 // 16, k128 // 128, 64, 4, dtype=torch.int32, device="cuda")
        for i in range(0, N, step):
            m = min(step, N - i)
            # bell-shaped weights, as a rounding to 16 levels leaves them
            codes[i:i + m, :K] = (7.5 + 2.8 * _randn(m, K, g=g)).round_().clamp_(0, 15).byte()
            s["tiles"][i // 16:(i + step) // 16] = _tiles(codes[i:i + step])
        s["codes"] = codes[:N, 0:K:2] | codes[:N, 1:K:2] << 4      # as a checkpoint holds them
        scale = (0.5 + torch.rand(N, K // grp, generator=g, device="cuda")) * (0.3 / K ** 0.5)
        scale = scale.half()
        both = scale[..., None]
        s["scale"], s["min"] = scale, None
        if case["shift"]:
            s["min"] = (-scale.float() * (7.5 + 0.5 * _randn(N, K // grp, g=g))).half()
            both = torch.stack([scale, s["min"]], 2)
        laid = torch.zeros(n16, K // grp, both.shape[2], dtype=torch.half, device="cuda")
        laid[:N] = both
        laid = laid.view(n16 // 16, 16, K // grp, -1).transpose(1, 2).contiguous()
        s["scales"] = laid if case["shift"] else laid[..., 0].contiguous()
        s["x"] = _randn(M, K, g=g).to(torch.bfloat16)
        return s
    lens, parents = _trees(case)
    new = [len(p) for p in parents]
    s["q_start"] = _i32([sum(new[:b]) for b in range(len(new) + 1)])
    if case["kind"] == "walk":
        s["parents"] = _i32([p for t in parents for p in t])
        T = sum(new)
        # two of three nodes' samples are the token of one of their children; a small
        # vocabulary has siblings that are alike
        tokens = torch.randint(0, case["V"], (T,), generator=g, device="cuda")
        s["tokens"] = tokens.int()
        start = torch.repeat_interleave(s["q_start"][:-1].long(), torch.tensor(new, device="cuda"))
        order = torch.rand(T, generator=g, device="cuda").argsort()
        child = torch.full((T + 1,), -1, device="cuda")
        up = torch.where(s["parents"] >= 0, start + s["parents"], T)
        child.scatter_reduce_(0, up, order, "amax")            # of a parent's children, one at random
        child = order.argsort()[child[:T].clamp(min=0)]
        has = torch.zeros(T + 1, dtype=torch.bool, device="cuda").index_fill_(0, up, True)[:T]
        hit = has & (torch.rand(T, generator=g, device="cuda") < 0.67)
        other = torch.randint(0, case["V"], (T,), generator=g, device="cuda")
        sampled = torch.where(hit, tokens[child], other)
        s["sampled"] = sampled.int()
        return s
    P, D, Hkv = case["page"], case["D"], case["Hkv"]
    need = [-(-x // P) for x in lens]
    M, n = max(need), sum(need) + max(1, sum(need) // 8)
    order = torch.randperm(n, generator=g, device="cuda").to(torch.int32)
    at = torch.tensor([sum(need[:b]) for b in range(len(need))], device="cuda")[:, None] + \
        torch.arange(M, device="cuda")
    held = torch.arange(M, device="cuda") < torch.tensor(need, device="cuda")[:, None]
    s["table"] = torch.where(held, order[at.clamp(max=n - 1)], -1).to(torch.int32).contiguous()
    s["kv_len"] = _i32(lens)
    if case["kind"] == "commit":
        width = 2 * P * D * (2 if case["cache"] == "bf16" else 1) + \
            (0 if case["cache"] == "bf16" else 8 * P)
        pool = torch.empty(case["L"], n, Hkv, width, dtype=torch.uint8, device="cuda")
        for x in pool:
            x.random_(0, 256, generator=g)
        s["pool"] = pool.view(torch.bfloat16) if case["cache"] == "bf16" else pool
        s["path"], s["count"] = (_i32(x) for x in _paths(case, new, seed))
        return s
    s["max_new"] = max(new)
    masks, depths = zip(*(_masks(p, _words(case)) for p in parents))
    s["mask"] = torch.tensor([m for t in masks for m in t], dtype=torch.int64, device="cuda")
    s["depth"] = _i32([d for t in depths for d in t])
    s["pool"] = _pool(case, n, g)
    # scores with a standard deviation of 2: a few tokens carry most of a row
    s["q"] = (2.0 * _randn(sum(new), case["Hq"], D, g=g)).to(torch.bfloat16)
    return s


def _paths(case, new, seed):
    """Accepted nodes and their number.  But for node 0 they lie past the slots
    that they move to, so that a round committed twice stays as it is."""
    many, r, w = random.Random(case["mix"]), random.Random(int(seed)), case["width"]
    paths, count = [], []
    for n in new:
        c = many.randint(1, min(w, n - w + 1) if n > w else n)
        p = [0] + sorted(r.sample(range(w, n), c - 1)) if n > w else list(range(c))
        paths.append(p + [-1] * (w - c))
        count.append(c)
    return paths, count


# ------------------------------------------------------------------ the operators
def _rows(s, T):
    """(sequence, place among its nodes) of every node."""
    t = torch.arange(T, device="cuda")
    b = torch.searchsorted(s["q_start"].long()[1:], t, right=True)
    return b, t - s["q_start"].long()[b]


def _bits(mask, n):
    """Masks [.., words] as truth values [.., n]."""
    i = torch.arange(n, device="cuda")
    return (mask[..., i // 64] >> i % 64 & 1).bool()


def _plain_tree(s):
    P, D, H, pool = s["page"], s["D"], s["Hkv"], s["pool"]
    q, table = s["q"], s["table"].long().clamp(min=0)
    B, M = table.shape
    T, Hq = q.shape[:2]
    G, n = Hq // H, s["max_new"]
    b, i = _rows(s, T)
    if s["cache"] == "bf16":
        ch = 8
        pages = pool[table].float()
    else:
        ch = 16
        pages = pool[table]
        sc = pages[..., 2 * P * D:].contiguous().view(torch.float32).view(B, M, H, 2, P)
        pages = pages[..., :2 * P * D].contiguous().view(torch.float8_e4m3fn).float()
    kd, vd = pages[..., :P * D], pages[..., P * D:]
    # [B, Hkv, D, tokens] and [B, Hkv, tokens, D]
    k = kd.reshape(B, M, H, D // ch, P, ch).permute(0, 2, 3, 5, 1, 4).reshape(B, H, D, M * P)
    v = vd.reshape(B, M, H, P // ch, D, ch).permute(0, 2, 1, 3, 5, 4).reshape(B, H, M * P, D)
    if s["cache"] != "bf16":
        sc = sc.permute(3, 0, 2, 1, 4).reshape(2, B, H, M * P)
        k, v = k * sc[0][:, :, None, :], v * sc[1][..., None]
    rows = torch.zeros(B, n, Hq, D, device="cuda")
    rows[b, i] = q.float()
    x = rows.view(B, n, H, G, D).permute(0, 2, 1, 3, 4).reshape(B, H, n * G, D)
    x = torch.matmul(x, k).view(B, H, n, G, M * P) * (1.0 / math.sqrt(D))
    if s["softcap"]:
        x = s["softcap"] * torch.tanh(x / s["softcap"])
    lens = s["kv_len"].long()
    base = (lens - s["q_start"].long().diff())[:, None, None]
    t = torch.arange(M * P, device="cuda")
    ok = (t < base).expand(B, n, M * P)
    if s["window"]:
        depth = torch.zeros(B, n, dtype=torch.int64, device="cuda")
        depth[b, i] = s["depth"].long()
        ok = ok & (t > base + depth[..., None] - s["window"])
    mask = torch.zeros(B, n, s["mask"].shape[1], dtype=torch.int64, device="cuda")
    mask[b, i] = s["mask"]
    node = t - base
    tree = _bits(mask, n).gather(2, node.clamp(0, n - 1).expand(B, n, M * P))
    ok = ok | tree & (node >= 0) & (t < lens[:, None, None])
    x = torch.where(ok[:, None, :, None, :], x, -torch.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True).clamp(min=-3e38))
    p = (p / p.sum(-1, keepdim=True)).view(B, H, n * G, M * P)
    held = (t < lens[:, None])[:, None, :, None]
    o = torch.matmul(p, torch.where(held, v, 0.0))
    o = o.view(B, H, n, G, D).permute(0, 2, 1, 3, 4).reshape(B, n, Hq, D)
    return o[b, i].to(torch.bfloat16)


def _plain_walk(s):
    B, T, w, n = s["B"], s["parents"].shape[0], s["width"], s["nodes"]
    b, i = _rows(s, T)
    par = torch.full((B, n), -1, dtype=torch.int64, device="cuda")
    tok, out = torch.full_like(par, -1), torch.full_like(par, -2)
    par[b, i], tok[b, i], out[b, i] = s["parents"].long(), s["tokens"].long(), s["sampled"].long()
    j = torch.arange(n, device="cuda")
    # up[b, i, j]: j is i or an ancestor of it; twice as many steps a product
    up = ((par[..., None] == j) | (j[:, None] == j)).float()
    for _ in range(max(1, (n - 1).bit_length())):
        up = (torch.matmul(up, up) > 0).float()
    depth = up.sum(2).long() - 1
    words = -(-n // 64)
    bits = torch.zeros(B, n, 64 * words, dtype=torch.int64, device="cuda")
    bits[..., :n] = up.long() << j % 64
    mask = bits.view(B, n, words, 64).sum(3)
    # a node goes on where its token is its parent's sample, and no sibling before it is
    hit = (par >= 0) & (tok == out.gather(1, par.clamp(min=0)))
    twin = (par[:, :, None] == par[:, None]) & hit[:, None] & (j < j[:, None])
    good = (hit & ~twin.any(2)) | ((j == 0) & (tok >= 0))
    on = ~((up > 0) & ~good[:, None]).any(2) & good & (up[..., 0] > 0) & (depth < w)
    path = torch.full((B, w + 1), -1, dtype=torch.int64, device="cuda")
    path.scatter_(1, torch.where(on, depth, w), torch.where(on, j.expand(B, n), -1))
    count = on.sum(1)
    last = path.gather(1, (count - 1).clamp(min=0)[:, None])
    nxt = out.gather(1, last.clamp(min=0))[:, 0]
    return dict(mask=mask[b, i], depth=depth[b, i].int(), path=path[:, :w].int(),
                count=count.int(), next=nxt.int())


def _plain_commit(s):
    P, D, H, pool = s["page"], s["D"], s["Hkv"], s["pool"]
    L, N = pool.shape[:2]
    base = s["kv_len"].long() - s["q_start"].long().diff()
    w = s["path"].shape[1]
    b, j = torch.nonzero(torch.arange(w, device="cuda") < s["count"][:, None], as_tuple=True)
    src, dst = base[b] + s["path"].long()[b, j], base[b] + j
    table = s["table"].long()
    ps, os, pd, od = table[b, src // P], src % P, table[b, dst // P], dst % P
    ch = 8 if s["cache"] == "bf16" else 16
    k = pool[..., :P * D].unflatten(3, (D // ch, P, ch))
    v = pool[..., P * D:2 * P * D].unflatten(3, (P // ch, D, ch))
    k[:, pd, :, :, od] = k[:, ps, :, :, os]
    v[:, pd, :, od // ch, :, od % ch] = v[:, ps, :, os // ch, :, os % ch]
    if s["cache"] != "bf16":
        sc = pool[..., 2 * P * D:].view(torch.float32).view(L, N, H, 2, P)
        sc[:, pd, :, :, od] = sc[:, ps, :, :, os]


def _plain_w4(s):
    N, K, g = s["N"], s["K"], s["g"]
    q = torch.stack([s["codes"] & 15, s["codes"] >> 4], 2).view(N, K // g, g).float()
    if s["min"] is None:
        w = (q - 8.0) * s["scale"].float()[..., None]
    else:
        w = q * s["scale"].float()[..., None] + s["min"].float()[..., None]
    y = torch.matmul(s["x"].float(), w.view(N, K).T)
    return y.to(torch.bfloat16) if s["out"] == "bf16" else y


def run(state):
    global _L
    s = state
    if own and _L is None:
        from chenxing_amd import _lib
        _L = _lib
    if s["kind"] == "w4":
        if own:
            return _L.w4_linear_device(s["x"], s["tiles"], s["scales"], s["N"],
                                       torch.bfloat16 if s["out"] == "bf16" else torch.float32)
        return _plain_w4(s)
    if s["kind"] == "tree":
        if own:
            return _L.tree_attention_device(s["q"], s["pool"], s["table"], s["kv_len"], s["mask"],
                                            s["q_start"], depth=s["depth"], max_new=s["max_new"],
                                            window=s["window"], softcap=s["softcap"])
        return _plain_tree(s)
    if s["kind"] == "walk":
        if own:
            mask, depth = _L.tree_masks_device(s["parents"], s["q_start"], _words(s))
            path, count, nxt = _L.tree_accept_device(s["parents"], s["tokens"], s["sampled"],
                                                     s["width"], s["q_start"])
            return dict(mask=mask, depth=depth, path=path, count=count, next=nxt)
        return _plain_walk(s)
    if own:
        _L.kv_commit_device(s["pool"], s["D"], s["table"], s["kv_len"], s["path"], s["count"],
                            s["q_start"])
    else:
        _plain_commit(s)
    if s["cache"] == "bf16":                       # bytes that are moved, not numbers
        return s["pool"].view(torch.int16)
    return s["pool"]


# ------------------------------------------------------------------ what is needed
def work(case):
    if case["kind"] == "w4":
        M, N, K, g = (case[k] for k in ("M", "N", "K", "g"))
        return dict(bytes=N * K // 2 + N * (K // g) * (4 if case["shift"] else 2) + 2 * M * K +
                    M * N * (2 if case["out"] == "bf16" else 4), flops=2 * M * N * K)
    lens, parents = _trees(case)
    T = sum(len(p) for p in parents)
    if case["kind"] == "walk":
        return dict(bytes=T * (12 + 8 * _words(case) + 4) + case["B"] * (4 * case["width"] + 12),
                    flops=0)
    P, D, H = case["page"], case["D"], case["Hkv"]
    el = 2 if case["cache"] == "bf16" else 1
    sc = 0 if case["cache"] == "bf16" else 8
    if case["kind"] == "commit":
        moved = sum(c - 1 for c, p in zip(_paths(case, [len(p) for p in parents], 0)[1], parents)
                    if len(p) > case["width"])
        return dict(bytes=2 * case["L"] * H * moved * (2 * D * el + sc) +
                    4 * case["B"] * (case["width"] + 4), flops=0)
    w = case["window"] or 1 << 40
    tokens = pairs = 0
    for n, tree in zip(lens, parents):
        m, depths = len(tree), _masks(tree, _words(case))[1]
        tokens += m + min(n - m, w - 1)
        pairs += sum(d + 1 + max(0, min(n - m, w - 1 - d)) for d in depths)
    return dict(bytes=tokens * H * (2 * D * el + sc) + T * case["Hq"] * D * 4 +
                T * (8 * _words(case) + 4) + 4 * (tokens // P + 3 * case["B"]),
                flops=4 * pairs * case["Hq"] * D)


# ------------------------------------------------------------------ the same in 64 bits
def _exact_tree(s):
    P, D, H, G = s["page"], s["D"], s["Hkv"], s["Hq"] // s["Hkv"]
    bf16 = s["cache"] == "bf16"
    ch = 8 if bf16 else 16
    flat = s["pool"].reshape(-1)
    width = s["pool"].shape[2]
    d = torch.arange(D, device="cuda")
    lens, parents = _trees(s)
    out, at = [], 0
    for b in range(s["B"]):
        n, m = lens[b], len(parents[b])
        allowed = torch.zeros(m, n, dtype=torch.bool)
        depth = []
        for i, p in enumerate(parents[b]):
            depth.append(0 if p < 0 else depth[p] + 1)
            if p >= 0:
                allowed[i, n - m:] = allowed[p, n - m:]
            allowed[i, n - m + i] = True
            first = max(0, n - m + depth[i] - s["window"] + 1) if s["window"] else 0
            allowed[i, min(first, n - m):n - m] = True
        allowed = allowed.cuda()
        t = torch.arange(n, device="cuda")
        page, off = s["table"][b].long()[t // P], t % P
        kat = ((d // ch) * P + off[:, None]) * ch + d % ch                  # [t, D]
        vat = P * D + ((off[:, None] // ch) * D + d) * ch + off[:, None] % ch
        qb = s["q"][at:at + m].double()
        ob = torch.empty(m, s["Hq"], D, dtype=torch.float64, device="cuda")
        for h in range(H):
            base = ((page * H + h) * width)[:, None]
            k, v = flat[base + kat], flat[base + vat]
            if bf16:
                k, v = k.double(), v.double()
            else:
                at4 = base + 2 * P * D + 4 * off[:, None] + torch.arange(4, device="cuda")
                ks = flat[at4].view(torch.float32).double()
                vs = flat[at4 + 4 * P].view(torch.float32).double()
                k = k.view(torch.float8_e4m3fn).double() * ks
                v = v.view(torch.float8_e4m3fn).double() * vs
            x = qb[:, h * G:(h + 1) * G].reshape(m * G, D) @ k.T.contiguous() / math.sqrt(D)
            if s["softcap"]:
                x = s["softcap"] * torch.tanh(x / s["softcap"])
            x = x.masked_fill(~allowed.repeat_interleave(G, 0), -math.inf)
            ob[:, h * G:(h + 1) * G] = (torch.softmax(x, 1) @ v).view(m, G, D)
        out.append(ob)
        at += m
    return torch.cat(out)


def _exact_w4(s):
    N, K, g = s["N"], s["K"], s["g"]
    x = s["x"].double().contiguous()
    y = torch.empty(s["M"], N, dtype=torch.float64, device="cuda")
    step = max(1, (1 << 27) // K)
    for i in range(0, N, step):
        c = s["codes"][i:i + step]
        w = torch.empty(c.shape[0], K, dtype=torch.float64, device="cuda")
        w[:, 0::2], w[:, 1::2] = (c % 16).double(), (c // 16).double()
        w = w.view(-1, K // g, g)
        f = s["scale"][i:i + step].double()[..., None]
        w = w * f + (-8 * f if s["min"] is None else s["min"][i:i + step].double()[..., None])
        y[:, i:i + step] = x @ w.view(-1, K).T.contiguous()
    return y


def exact(case, seed):
    if case["kind"] in ("walk", "commit"):
        return None                                # whole numbers, bytes: nothing is computed
    s = prepare(case, seed)
    return _exact_tree(s) if case["kind"] == "tree" else _exact_w4(s)
