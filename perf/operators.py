"""The paged KV-cache operators between two sampling calls: what is measured.

Three operators of one forward pass over a batch of running sequences:

  append   q and k normed per head and rotated, k and v written to the pages
  attend   attention of the new tokens (one of a decode step, gamma + 1 of a
           verify round) over the pages
  pages    pages copied over every layer (a fork's last page, a compaction)

``run`` computes them in elementary torch operations, or, where ``own`` is
true, through the library's calls.

A page of one layer holds ``page`` tokens of every kv head.  A head's part is
contiguous: K in 16-byte chunks [D / ch][page], then V in 16-byte chunks
[page / ch][D] whose elements are ch neighbouring tokens (ch = 8 for bf16, 16
for e4m3), then, for e4m3, one fp32 scale a token for K and one for V.
"""
from __future__ import annotations

import math
import random

import torch

own = False
_L = None

MAX_KV_BYTES = 1.0e9      # cache bytes a drawn attention case reads at most


def listed():
    return [
        # the smallest decode step: one request in the middle of a chat
        dict(name="attend_one", kind="attend", cache="bf16", B=1, Hq=32, Hkv=8, D=128, page=16,
             lo=700, hi=700, new=1, window=0, softcap=0.0, mix=1),
        # an ordinary decode batch, prompts and answers of very different lengths
        dict(name="attend_batch", kind="attend", cache="bf16", B=64, Hq=32, Hkv=8, D=128, page=16,
             lo=64, hi=8192, new=1, window=0, softcap=0.0, mix=2),
        # two long documents: few rows, the work is in the cache's length
        dict(name="attend_long", kind="attend", cache="bf16", B=2, Hq=32, Hkv=8, D=128, page=64,
             lo=120001, hi=131072, new=1, window=0, softcap=0.0, mix=3),
        # a batch of verify rounds, gamma up to 8: one to nine new tokens each
        dict(name="attend_verify", kind="attend", cache="bf16", B=32, Hq=32, Hkv=8, D=128, page=16,
             lo=50, hi=4096, new=9, window=0, softcap=0.0, mix=4),
        # wide heads, capped scores and a sliding window, an odd batch
        dict(name="attend_window", kind="attend", cache="bf16", B=37, Hq=16, Hkv=8, D=256, page=32,
             lo=1, hi=6000, new=1, window=1024, softcap=50.0, mix=5),
        # a small model without shared kv heads, narrow heads
        dict(name="attend_narrow", kind="attend", cache="bf16", B=24, Hq=12, Hkv=12, D=64, page=16,
             lo=30, hi=1500, new=1, window=0, softcap=0.0, mix=6),
        # the largest: a full decode batch over an 8-bit cache
        dict(name="attend_e4m3", kind="attend", cache="e4m3", B=256, Hq=32, Hkv=8, D=128, page=16,
             lo=500, hi=8192, new=1, window=0, softcap=0.0, mix=7),
        # one decoded token's q, k and v: latency
        dict(name="append_one", kind="append", cache="bf16", B=1, Hq=32, Hkv=8, D=128, page=16,
             lo=700, hi=700, new=1, r=128, style="half", norm=False, mix=8),
        # a full decode batch, q and k normed per head
        dict(name="append_batch", kind="append", cache="bf16", B=256, Hq=32, Hkv=8, D=128, page=16,
             lo=64, hi=8192, new=1, r=128, style="half", norm=True, mix=9),
        # prompts being prefilled into an 8-bit cache, part of each head rotated
        dict(name="append_prompt", kind="append", cache="e4m3", B=5, Hq=32, Hkv=8, D=128, page=16,
             lo=3000, hi=4096, new=2500, r=64, style="interleaved", norm=True, mix=10),
        # sixteen samples of one prompt start: each gets its own last page, in every layer
        dict(name="pages_fork", kind="pages", cache="bf16", L=32, n=256, pairs=16, Hkv=8, D=128,
             page=16, fork=True),
        # a compaction after many requests ended
        dict(name="pages_compact", kind="pages", cache="bf16", L=32, n=1000, pairs=400, Hkv=8,
             D=128, page=16, fork=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "append", "append", "pages"])
    cache = rng.choice(["bf16", "bf16", "e4m3"])
    D = rng.choice([64, 128, 128, 256])
    page = rng.choice([16, 16, 32, 64, 128])
    Hkv = rng.choice([1, 2, 3, 4, 8, 8, 8, 12])
    el = 2 if cache == "bf16" else 1
    if kind == "pages":
        L = _log(rng, 1, 32)
        most = max(2, int(1.6e9 / (L * Hkv * page * D * 2 * el)))
        n = max(2, min(_log(rng, 8, 2000), most))
        return dict(kind=kind, cache=cache, L=L, n=n, pairs=_log(rng, 1, max(1, n // 3)), Hkv=Hkv,
                    D=D, page=page, fork=rng.random() < 0.5)
    Hq = Hkv * rng.choice([1, 2, 3, 4, 4, 7, 8])
    mix = rng.randrange(1 << 30)
    if kind == "append":
        new = rng.choice([1, 1, rng.randint(2, 9), _log(rng, 16, 2048)])
        B = _log(rng, 1, max(1, min(256, 12000 // new)))
        hi = new + _log(rng, 1, 8192)
        return dict(kind=kind, cache=cache, B=B, Hq=Hq, Hkv=Hkv, D=D, page=page,
                    lo=max(new, hi // 4), hi=hi, new=new, r=rng.choice([D, D, D // 2, D // 4]),
                    style=rng.choice(["half", "half", "interleaved"]), norm=rng.random() < 0.5,
                    mix=mix)
    new = rng.choice([1, 1, 1, rng.randint(2, 9), rng.randint(2, 17)])
    hi = _log(rng, 32, 131072)
    lo = max(1, int(hi * rng.choice([0.01, 0.1, 0.5, 1.0])))
    most = int(MAX_KV_BYTES / (hi * Hkv * D * 2 * el))
    return dict(kind=kind, cache=cache, B=_log(rng, 1, max(1, min(256, most))), Hq=Hq, Hkv=Hkv,
                D=D, page=page, lo=lo, hi=hi, new=new,
                window=rng.choice([0, 0, 0, _log(rng, 16, 4096)]),
                softcap=rng.choice([0.0, 0.0, 30.0]), mix=mix)


# ------------------------------------------------------------------ inputs
def _lens(case):
    """The sequences' lengths (new tokens included) and numbers of new tokens:
    part of the case, so that the work is known from it."""
    r = random.Random(case["mix"])
    new, lens = [], []
    for _ in range(case["B"]):
        lens.append(_log(r, case["lo"], case["hi"]))
        most = min(case["new"], lens[-1])
        # verify rounds of different depths; a prompt's chunks of different sizes
        new.append(most if case["new"] == 1 else r.randint(max(1, most // 2 if most > 17 else 1),
                                                           most))
    return lens, new


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 7919 + 13)
    return g


def _randn(*shape, g):
    return torch.randn(*shape, generator=g, device="cuda")


def _pack_k(k, ch):
    n, H, P, D = k.shape
    return k.reshape(n, H, P, D // ch, ch).transpose(2, 3).reshape(n, H, P * D)


def _pack_v(v, ch):
    n, H, P, D = v.shape
    return v.reshape(n, H, P // ch, ch, D).transpose(3, 4).reshape(n, H, P * D)


def _pool(case, n, g, zero=False):
    """One layer's pages: bf16 [n, Hkv, 2 page D], or uint8 [n, Hkv, 2 page D + 8 page]."""
    H, P, D = case["Hkv"], case["page"], case["D"]
    bf16 = case["cache"] == "bf16"
    width = 2 * P * D if bf16 else 2 * P * D + 8 * P
    pool = torch.zeros(n, H, width, dtype=torch.bfloat16 if bf16 else torch.uint8, device="cuda")
    step = max(1, (1 << 26) // (H * P * D))
    for i in range(0, 0 if zero else n, step):
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


def _rope_rows(n, r):
    """fp32 [n, r]: the cosines, then the sines, of position times theta^(-2 j / r)."""
    f = 10000.0 ** (-torch.arange(r // 2, dtype=torch.float64, device="cuda") * 2 / r)
    a = torch.arange(n, dtype=torch.float64, device="cuda")[:, None] * f
    return torch.cat([a.cos(), a.sin()], 1).float()


def prepare(case, seed):
    g = _gen(seed)
    s = dict(case)
    P, D, Hkv = case["page"], case["D"], case["Hkv"]
    if case["kind"] == "pages":
        n, m = case["n"], case["pairs"]
        width = 2 * P * D * (2 if case["cache"] == "bf16" else 1) + \
            (0 if case["cache"] == "bf16" else 8 * P)
        pool = torch.empty(case["L"], n, Hkv, width, dtype=torch.uint8, device="cuda")
        for x in pool:
            x.random_(0, 256, generator=g)
        order = torch.randperm(n, generator=g, device="cuda").to(torch.int32)
        src = order[m:2 * m]
        if case["fork"]:                       # a few parents, several samples of each
            src = order[m + torch.arange(m, device="cuda") % max(1, min(m, n - m) // 4)]
        s.update(pool=pool, src=src.contiguous(), dst=order[:m].contiguous())
        return s
    lens, new = _lens(case)
    need = [-(-x // P) for x in lens]
    M, n = max(need), sum(need) + max(1, sum(need) // 8)
    order = torch.randperm(n, generator=g, device="cuda").to(torch.int32)
    at = torch.tensor([sum(need[:b]) for b in range(len(need))], device="cuda")[:, None] + \
        torch.arange(M, device="cuda")
    held = torch.arange(M, device="cuda") < torch.tensor(need, device="cuda")[:, None]
    s["table"] = torch.where(held, order[at.clamp(max=n - 1)], -1).to(torch.int32).contiguous()
    s["kv_len"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    s["max_new"] = max(new)
    s["q_start"] = None
    if s["max_new"] > 1:
        s["q_start"] = torch.tensor([sum(new[:b]) for b in range(len(new) + 1)],
                                    dtype=torch.int32, device="cuda")
    T, Hq = sum(new), case["Hq"]
    if case["kind"] == "attend":
        s["pool"] = _pool(case, n, g)
        # scores with a standard deviation of 2: a few tokens carry most of a row
        s["q"] = (2.0 * _randn(T, Hq, D, g=g)).to(torch.bfloat16)
        return s
    # one projection's output, q, k and v side by side
    qkv = _randn(T, Hq + 2 * Hkv, D, g=g).to(torch.bfloat16)
    s["q"], s["k"], s["v"] = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
    s["pool"] = _pool(case, n, g, zero=True)
    s["rope"] = _rope_rows(M * P, case["r"])
    s["q_norm"] = s["k_norm"] = None
    if case["norm"]:
        s["q_norm"] = (1 + 0.1 * _randn(D, g=g)).to(torch.bfloat16)
        s["k_norm"] = (1 + 0.1 * _randn(D, g=g)).to(torch.bfloat16)
    return s


# ------------------------------------------------------------------ the operators
def _tokens(s):
    """(sequence, place among its new tokens, number of them) of every new token."""
    T = s["q"].shape[0]
    t = torch.arange(T, device="cuda")
    if s["q_start"] is None:
        return t, torch.zeros_like(t), torch.ones_like(t)
    st = s["q_start"].long()
    b = torch.searchsorted(st[1:], t, right=True)
    return b, t - st[b], st[b + 1] - st[b]


def _plain_pages(s):
    pool = s["pool"]
    pool[:, s["dst"].long()] = pool[:, s["src"].long()]


def _plain_norm(x, w, eps=1e-6):
    x = x.float()
    if w is None:
        return x
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w.float()


def _plain_turn(x, cs, r, style):
    c, sn = cs[:, None, :r // 2], cs[:, None, r // 2:]
    y = x.clone()
    if style == "half":
        a, b = x[..., :r // 2], x[..., r // 2:r]
        y[..., :r // 2], y[..., r // 2:r] = a * c - b * sn, b * c + a * sn
    else:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        y[..., 0:r:2], y[..., 1:r:2] = a * c - b * sn, b * c + a * sn
    return y


def _plain_append(s):
    P, D, H, pool = s["page"], s["D"], s["Hkv"], s["pool"]
    b, i, n = _tokens(s)
    pos = s["kv_len"].long()[b] - n + i
    cs = s["rope"][pos]
    q = _plain_turn(_plain_norm(s["q"], s["q_norm"]), cs, s["r"], s["style"])
    k = _plain_turn(_plain_norm(s["k"], s["k_norm"]), cs, s["r"], s["style"])
    v = s["v"].float()
    page, off = s["table"].long()[b, pos // P], pos % P
    N, T = pool.shape[0], len(b)
    if s["cache"] == "bf16":
        ch = 8
        kd, vd = k.to(torch.bfloat16), v.to(torch.bfloat16)
    else:
        ch = 16
        ks, vs = k.abs().amax(2) / 448, v.abs().amax(2) / 448
        ks, vs = torch.where(ks > 0, ks, 1.0), torch.where(vs > 0, vs, 1.0)
        kd = (k / ks[..., None]).to(torch.float8_e4m3fn).view(torch.uint8)
        vd = (v / vs[..., None]).to(torch.float8_e4m3fn).view(torch.uint8)
        scales = pool[..., 2 * P * D:].view(torch.float32).view(N, H, 2, P)
        scales[page, :, 0, off] = ks
        scales[page, :, 1, off] = vs
    pool[..., :P * D].unflatten(2, (D // ch, P, ch))[page, :, :, off] = kd.view(T, H, D // ch, ch)
    pool[..., P * D:2 * P * D].unflatten(2, (P // ch, D, ch))[page, :, off // ch, :, off % ch] = vd
    return q.to(torch.bfloat16)


def _plain_attend(s):
    P, D, H, pool = s["page"], s["D"], s["Hkv"], s["pool"]
    q, table = s["q"], s["table"].long().clamp(min=0)
    B, M = table.shape
    T, Hq = q.shape[:2]
    G, n = Hq // H, s["max_new"]
    b, i, cnt = _tokens(s)
    if s["cache"] == "bf16":
        ch = 8
        pages = pool[table].float()
        kd, vd = pages[..., :P * D], pages[..., P * D:]
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
    have = torch.ones_like(lens) if s["q_start"] is None else s["q_start"].long().diff()
    pos = (lens - have)[:, None] + torch.arange(n, device="cuda")
    t = torch.arange(M * P, device="cuda")
    ok = (t <= pos[..., None]) & (t < lens[:, None, None])
    if s["window"]:
        ok &= t > pos[..., None] - s["window"]
    x = torch.where(ok[:, None, :, None, :], x, -torch.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True).clamp(min=-3e38))
    p = (p / p.sum(-1, keepdim=True)).view(B, H, n * G, M * P)
    held = (t < lens[:, None])[:, None, :, None]
    o = torch.matmul(p, torch.where(held, v, 0.0))
    o = o.view(B, H, n, G, D).permute(0, 2, 1, 3, 4).reshape(B, n, Hq, D)
    return o[b, i].to(torch.bfloat16)


def run(state):
    global _L
    s = state
    if own and _L is None:
        from chenxing_amd import _lib
        _L = _lib
    if s["kind"] == "pages":
        if own:
            _L.kv_copy_pages_device(s["pool"], s["src"], s["dst"])
        else:
            _plain_pages(s)
        return s["pool"]
    if s["kind"] == "attend":
        if own:
            return _L.paged_attention_device(s["q"], s["pool"], s["table"], s["kv_len"],
                                             s["q_start"], s["max_new"], window=s["window"],
                                             softcap=s["softcap"])
        return _plain_attend(s)
    if own:
        q = _L.kv_append_device(s["q"], s["k"], s["v"], s["pool"], s["table"], s["kv_len"],
                                s["q_start"], rope=s["rope"],
                                interleaved=s["style"] == "interleaved", q_norm=s["q_norm"],
                                k_norm=s["k_norm"])
    else:
        q = _plain_append(s)
    if s["cache"] == "bf16":
        return dict(q=q, kv=s["pool"])
    n = 2 * s["page"] * s["D"]
    return dict(q=q, codes=s["pool"][..., :n].view(torch.float8_e4m3fn),
                scales=s["pool"][..., n:].view(torch.float32))


# ------------------------------------------------------------------ what is needed
def work(case):
    P, D, H = case["page"], case["D"], case["Hkv"]
    el = 2 if case["cache"] == "bf16" else 1
    sc = 0 if case["cache"] == "bf16" else 8
    if case["kind"] == "pages":
        return dict(bytes=case["pairs"] * (2 * case["L"] * H * P * (2 * D * el + sc) + 8), flops=0)
    lens, new = _lens(case)
    T, Hq = sum(new), case["Hq"]
    if case["kind"] == "append":
        move = T * ((Hq + 2 * H) * D * 2 + Hq * D * 2 + H * (2 * D * el + sc) + 4 * case["r"])
        return dict(bytes=move + 8 * case["B"] + 4 * T, flops=6 * T * (Hq + H) * D)
    w = case["window"] or 1 << 40
    tokens = pairs = 0
    for n, m in zip(lens, new):
        tokens += n - max(0, n - m + 1 - w)
        pairs += sum(min(n - m + 1 + i, w) for i in range(m))
    return dict(bytes=tokens * H * (2 * D * el + sc) + 2 * T * Hq * D * 2 +
                4 * (tokens // P + case["B"]) + 8 * case["B"], flops=4 * pairs * Hq * D)


# ------------------------------------------------------------------ the same in 64 bits
def _exact_attend(s):
    P, D, H, G = s["page"], s["D"], s["Hkv"], s["Hq"] // s["Hkv"]
    bf16 = s["cache"] == "bf16"
    ch = 8 if bf16 else 16
    flat = s["pool"].reshape(-1)
    width = s["pool"].shape[2]
    d = torch.arange(D, device="cuda")
    lens, new = _lens(s)
    out, at = [], 0
    for b in range(s["B"]):
        n, m = lens[b], new[b]
        first = max(0, n - m + 1 - s["window"]) if s["window"] else 0
        t = torch.arange(first, n, device="cuda")
        page, off = s["table"][b].long()[t // P], t % P
        kat = ((d // ch) * P + off[:, None]) * ch + d % ch                  # [t, D]
        vat = P * D + ((off[:, None] // ch) * D + d) * ch + off[:, None] % ch
        qb = s["q"][at:at + m].double()
        pos = torch.arange(n - m, n, device="cuda")
        ok = t[None] <= pos[:, None]
        if s["window"]:
            ok &= t[None] > pos[:, None] - s["window"]
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
            x = x.masked_fill(~ok.repeat_interleave(G, 0), -math.inf)
            ob[:, h * G:(h + 1) * G] = (torch.softmax(x, 1) @ v).view(m, G, D)
        out.append(ob)
        at += m
    return torch.cat(out)


def _exact_append(s):
    P, D, H, r = s["page"], s["D"], s["Hkv"], s["r"]
    lens, new = _lens(s)
    seq = [b for b in range(s["B"]) for _ in range(new[b])]
    where = [lens[b] - new[b] + i for b in range(s["B"]) for i in range(new[b])]
    seq, pos = torch.tensor(seq, device="cuda"), torch.tensor(where, device="cuda")
    ang = s["rope"][pos].double()
    z = torch.complex(ang[:, :r // 2], ang[:, r // 2:])[:, None]

    def turned(x, w):
        x = x.double()
        if w is not None:
            x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / D + 1e-6) * w.double()
        j = torch.arange(r // 2, device="cuda")
        a, b = (j, j + r // 2) if s["style"] == "half" else (2 * j, 2 * j + 1)
        t = torch.complex(x[..., a], x[..., b]) * z
        x = x.clone()
        x[..., a], x[..., b] = t.real, t.imag
        return x

    k, v = turned(s["k"], s["k_norm"]), s["v"].double()
    ch = 8 if s["cache"] == "bf16" else 16
    page, off = s["table"][seq, pos // P].long(), pos % P
    N, n = s["pool"].shape[0], 2 * P * D
    d = torch.arange(D, device="cuda")
    row = (page[:, None] * H + torch.arange(H, device="cuda"))[..., None]     # [T, H, 1]
    kat = ((d // ch) * P + off[:, None]) * ch + d % ch
    vat = P * D + ((off[:, None] // ch) * D + d) * ch + off[:, None] % ch
    kv = torch.zeros(N * H * n, dtype=torch.float64, device="cuda")
    if s["cache"] != "bf16":
        ks, vs = k.abs().amax(2, keepdim=True) / 448, v.abs().amax(2, keepdim=True) / 448
        ks[ks == 0], vs[vs == 0] = 1, 1
        k, v = k / ks, v / vs
        sc = torch.zeros(N * H * 2 * P, dtype=torch.float64, device="cuda")
        sc[(row * 2 * P)[..., 0] + off[:, None]] = ks[..., 0]
        sc[(row * 2 * P)[..., 0] + P + off[:, None]] = vs[..., 0]
    kv[row * n + kat[:, None]] = k
    kv[row * n + vat[:, None]] = v
    q, kv = turned(s["q"], s["q_norm"]), kv.view(N, H, n)
    if s["cache"] == "bf16":
        return dict(q=q, kv=kv)
    # the codes' values before their rounding to 8 bits
    return dict(q=q, codes=kv, scales=sc.view(N, H, 2 * P))


def exact(case, seed):
    if case["kind"] == "pages":
        return None                            # bytes: nothing is computed
    s = prepare(case, seed)
    return _exact_attend(s) if case["kind"] == "attend" else _exact_append(s)
