"""The paged KV-cache operators (cx_kv_append_bf16, cx_paged_attention_bf16,
cx_kv_copy_pages) against their 64-bit restatement (oracle/paged_ref.py)."""
from __future__ import annotations

import numpy as np
import pytest

from oracle import paged_ref as R
from oracle.bf16 import bf16_bits_to_f32, f32_to_bf16_bits
import paged_cases as C

pytestmark = pytest.mark.gpu


def _values(bits):
    return bf16_bits_to_f32(bits).astype(np.float64)


# ------------------------------------------------------------------ attention
ATTEND = {
    # name: cache, Hq, Hkv, D, P, lengths, new tokens each, window, softcap
    "one_token": ("bf16", 4, 2, 64, 16, [1], [1], 0, 0.0),
    "zero_lengths": ("bf16", 4, 2, 128, 16, [0, 5, 0, 33, 0], [1, 1, 1, 1, 1], 0, 0.0),
    "page_edges": ("bf16", 8, 2, 128, 16, [15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129],
                   [1] * 12, 0, 0.0),
    "page_edges_e4m3": ("e4m3", 8, 2, 128, 16, [15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129],
                        [1] * 12, 0, 0.0),
    "big_pages": ("bf16", 6, 2, 64, 128, [1, 127, 128, 129, 1000], [1] * 5, 0, 0.0),
    "big_pages_e4m3": ("e4m3", 6, 2, 64, 256, [1, 255, 256, 257, 1000], [1] * 5, 0, 0.0),
    "wide_heads": ("bf16", 6, 3, 256, 32, [7, 300, 513], [1, 1, 1], 0, 0.0),
    "wide_heads_e4m3": ("e4m3", 6, 3, 256, 64, [7, 300, 513], [1, 1, 1], 0, 0.0),
    "narrow_e4m3": ("e4m3", 5, 5, 64, 32, [9, 200, 777], [1, 1, 1], 0, 0.0),
    "odd_group": ("bf16", 7, 1, 128, 16, [501, 250], [1, 1], 0, 0.0),
    "many_rows": ("bf16", 40, 2, 64, 16, [333, 90], [1, 1], 0, 0.0),
    "long": ("bf16", 8, 1, 128, 16, [9001], [1], 0, 0.0),
    "long_and_short": ("bf16", 8, 4, 128, 32, [6000, 3, 1, 800, 64], [1] * 5, 0, 0.0),
    "long_e4m3": ("e4m3", 4, 1, 128, 16, [12007], [1], 0, 0.0),
    "window": ("bf16", 4, 2, 128, 16, [1, 40, 100, 101, 700], [1] * 5, 100, 0.0),
    "window_one": ("bf16", 4, 2, 64, 16, [1, 17, 300], [1, 1, 1], 1, 0.0),
    "window_e4m3": ("e4m3", 8, 2, 128, 16, [5, 333, 1200], [1, 1, 3], 65, 0.0),
    "softcap": ("bf16", 4, 2, 128, 16, [3, 600], [1, 1], 0, 5.0),
    "softcap_window": ("bf16", 4, 2, 256, 32, [3, 600, 90], [2, 1, 5], 50, 30.0),
    "verify": ("bf16", 8, 2, 128, 16, [5, 40, 300, 64, 1000], [5, 1, 5, 0, 3], 0, 0.0),
    "verify_window": ("bf16", 8, 2, 128, 16, [9, 40, 300, 64], [9, 9, 7, 9], 20, 0.0),
    "verify_e4m3": ("e4m3", 8, 2, 128, 16, [5, 40, 300, 64], [5, 1, 5, 0], 0, 0.0),
    "verify_mha": ("bf16", 3, 3, 64, 16, [70, 35], [17, 16], 0, 0.0),
    "verify_wide": ("bf16", 8, 2, 256, 16, [70, 300], [9, 12], 0, 0.0),
    "verify_wide_e4m3": ("e4m3", 8, 1, 256, 16, [70, 300], [9, 12], 0, 0.0),
    "prompt": ("bf16", 4, 1, 64, 16, [150, 201], [150, 77], 0, 0.0),
    "prompt_rows": ("bf16", 24, 2, 128, 16, [50, 90], [41, 33], 0, 0.0),
    "more_new_than_tokens": ("bf16", 4, 2, 128, 16, [3, 0, 20], [5, 2, 4], 0, 0.0),
    "rows_33_narrow": ("bf16", 11, 1, 64, 16, [70, 300], [3, 3], 0, 0.0),
    "rows_20_narrow_e4m3": ("e4m3", 10, 2, 64, 16, [70, 300, 41], [4, 4, 1], 0, 0.0),
    "rows_70_e4m3": ("e4m3", 14, 1, 128, 32, [90, 300], [5, 5], 64, 0.0),
}


def _attend_inputs(name, seed=0):
    cache, Hq, Hkv, D, P, lens, new, window, cap = ATTEND[name]
    rng = np.random.default_rng(len(name) * 1009 + sum(map(ord, name)) + seed)
    table, kv_len, q_start, n = C.batch(rng, lens, new, P)
    K, V, ks, vs = C.dense_pages(rng, n, Hkv, P, D, cache)
    C.poison(K, V, ks, vs, table, lens, P)
    pages = R.pack(K, V, ks, vs)
    q = f32_to_bf16_bits(rng.normal(0, 2, (int(q_start[-1]), Hq, D)).astype(np.float32))
    return dict(q=q, pages=pages, table=table, kv_len=kv_len, q_start=q_start, P=P, D=D,
                window=window, softcap=cap, new=new)


def _widen(x):
    """A table of 4096 tokens at least: short ones are read by other means."""
    pad = max(0, 4096 // x["P"] - x["table"].shape[1])
    return dict(x, table=np.pad(x["table"], ((0, 0), (0, pad)), constant_values=-1))


def _attend(x, **kw):
    import torch
    from chenxing_amd._lib import paged_attention_device
    st = None if all(n == 1 for n in x["new"]) and kw.pop("plain", True) else C.to_gpu(x["q_start"])
    kw.setdefault("max_new", max(x["new"]))
    out = paged_attention_device(C.to_gpu(x["q"]), C.to_gpu(x["pages"]), C.to_gpu(x["table"]),
                                 C.to_gpu(x["kv_len"]), st, window=x["window"],
                                 softcap=x["softcap"], **kw)
    torch.cuda.synchronize()
    return out


def _expect(x, scale=None):
    K, V = R.unpack(x["pages"], x["D"])
    return R.attend(_values(x["q"]), K, V, x["table"], x["kv_len"], x["q_start"], x["P"],
                    x["D"] ** -0.5 if scale is None else scale, x["window"], x["softcap"])


def _check(out, want, tol):
    got = _values(C.bits_of(out))
    nan = np.isnan(want)
    assert np.array_equal(np.isnan(got), nan), (np.isnan(got).sum(), nan.sum())
    bad = ~nan & ~(np.abs(got - want) <= tol)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4], np.nanmax(np.abs(got - want)))


@pytest.mark.parametrize("name", ATTEND)
def test_attention(name):
    print(f"[gpu] attention {name}", flush=True)
    x = _attend_inputs(name)
    _check(_attend(x), *_expect(x))


@pytest.mark.parametrize("name", ATTEND)
def test_attention_wide_table(name):
    print(f"[gpu] attention {name}, wide table", flush=True)
    x = _widen(_attend_inputs(name))
    _check(_attend(x), *_expect(x))


@pytest.mark.parametrize("max_new", [1, 2, 8, 1000])
def test_attention_max_new_is_a_hint(max_new):
    print(f"[gpu] attention max_new {max_new}", flush=True)
    x = _attend_inputs("verify")
    _check(_attend(x, max_new=max_new), *_expect(x))


@pytest.mark.parametrize("max_new", [1, 3, 20, 2 ** 28])
def test_attention_max_new_below_the_rows(max_new):
    """Prompts of many row blocks under a hint of one, and a hint past any length."""
    print(f"[gpu] attention prompt rows, max_new {max_new}", flush=True)
    x = _attend_inputs("prompt_rows")
    _check(_attend(x, max_new=max_new), *_expect(x))


def test_attention_uniform_q_start_is_the_default():
    print("[gpu] attention q_start given or not", flush=True)
    import torch
    x = _attend_inputs("page_edges")
    assert torch.equal(_attend(x), _attend(x, plain=False))


def test_attention_scale():
    print("[gpu] attention scale", flush=True)
    x = _attend_inputs("long_and_short")
    _check(_attend(x, scale=0.31), *_expect(x, 0.31))


def test_attention_large_scores():
    """Scores in the hundreds: one token carries the row."""
    print("[gpu] attention large scores", flush=True)
    x = _attend_inputs("verify")
    _check(_attend(x, scale=9.0), *_expect(x, 9.0))


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
@pytest.mark.parametrize("window", [0, 3])
@pytest.mark.parametrize("wide", [False, True])
def test_attention_masked_nan_and_inf(cache, window, wide):
    """NaN and inf in the newest tokens' K or V reach the rows that attend to
    them and no other row."""
    print(f"[gpu] attention masked NaN and inf, {cache}, window {window}", flush=True)
    rng = np.random.default_rng(5)
    Hq, Hkv, D, P, lens, new = 8, 2, 128, 16, [37, 64, 90, 20], [6, 5, 9, 7]
    table, kv_len, q_start, n = C.batch(rng, lens, new, P)
    K, V, ks, vs = C.dense_pages(rng, n, Hkv, P, D, cache)
    bad = {0: 34, 1: 61, 2: 83, 3: 18}          # sequence -> position
    for b, s in bad.items():
        pg, o = table[b, s // P], s % P
        if cache == "bf16":
            x = [V, V, K, V][b]
            x[pg, :, o, 3::5] = [C.NAN16, 0x7F80, C.NAN16, 0xFF80][b]
        else:
            [vs, V, ks, V][b][pg, :, o] = [np.nan, C.NAN8, np.nan, C.NAN8][b]
    C.poison(K, V, ks, vs, table, lens, P)
    x = dict(q=f32_to_bf16_bits(rng.normal(0, 1, (sum(new), Hq, D)).astype(np.float32)),
             pages=R.pack(K, V, ks, vs), table=table, kv_len=kv_len, q_start=q_start, P=P, D=D,
             window=window, softcap=0.0, new=new)
    if wide:
        x = _widen(x)
    want, tol = _expect(x)
    got = _values(C.bits_of(_attend(x)))
    fine = np.isfinite(want)
    assert fine.any(axis=2).all(axis=1).sum() > 4 and not fine.all()
    assert (np.abs(got - want)[fine] <= tol[fine]).all()
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(got[np.isinf(want)], want[np.isinf(want)])


@pytest.mark.parametrize("wide", [False, True])
def test_attention_all_scores_minus_infinity(wide):
    """K of -inf under a positive q: a row without weight is NaN, as its
    formula; a row with one other token is that token."""
    print("[gpu] attention scores of -inf", flush=True)
    x = _attend_inputs("one_token")
    rng = np.random.default_rng(3)
    table, kv_len, q_start, n = C.batch(rng, [33, 33], [1, 1], 16)
    K, V, _, _ = C.dense_pages(rng, n, 2, 16, 64, "bf16")
    K[..., 5] = 0xFF80
    K[table[1, 1], :, 4] = 0x3F80
    q = f32_to_bf16_bits(np.abs(rng.normal(1, .1, (2, 4, 64))).astype(np.float32) + 0.1)
    x.update(q=q, pages=R.pack(K, V), table=table, kv_len=kv_len, q_start=q_start, new=[1, 1])
    if wide:
        x = _widen(x)
    got = _values(C.bits_of(_attend(x)))
    assert np.isnan(got[0]).all()
    v = _values(V[table[1, 1], :, 4])
    assert np.array_equal(got[1], np.repeat(v, 2, 0))


def test_attention_bad_table_ids_are_masked():
    """A page id outside the pool masks its tokens, wherever it stands."""
    print("[gpu] attention ids outside the pool", flush=True)
    x = _attend_inputs("long_and_short")
    x["table"] = x["table"].copy()
    x["table"][0, [0, 3, 77, 187]] = [-1, 2 ** 31 - 1, -2 ** 31, 10 ** 6]
    x["table"][1, 0] = -1
    want, tol = _expect(x)
    assert not want[1].any()
    _check(_attend(x), want, tol)


def test_attention_lengths_past_the_table():
    print("[gpu] attention lengths past the table", flush=True)
    x = _attend_inputs("page_edges")
    x["kv_len"] = x["kv_len"].copy()
    x["kv_len"][[0, 5]] = [5000, 2 ** 31 - 1]
    x["kv_len"][2] = -3
    x["table"] = np.where(x["table"] < 0, 0, x["table"] % len(x["pages"])).astype(np.int32)
    x["pages"] = R.pack(*C.dense_pages(np.random.default_rng(1), len(x["pages"]), 2, 16, 128, "bf16")[:2])
    _check(_attend(x), *_expect(x))


@pytest.mark.parametrize("window", [0, 40])
@pytest.mark.parametrize("wide", [False, True])
def test_attention_prompts_at_the_last_positions(window, wide):
    """Prompts whose positions end at 2^31 - 2, past their tables."""
    print("[gpu] attention of prompts at the last positions", flush=True)
    x = dict(_attend_inputs("prompt"), window=window)
    x["kv_len"] = np.array([2 ** 31 - 1, 2 ** 31 - 40], np.int32)
    x["table"] = np.where(x["table"] < 0, 0, x["table"] % len(x["pages"])).astype(np.int32)
    x["pages"] = R.pack(*C.dense_pages(np.random.default_rng(2), len(x["pages"]), 1, 16, 64, "bf16")[:2])
    if wide:
        x = _widen(x)
    _check(_attend(x), *_expect(x))


def test_attention_strides():
    """q with odd strides, pages inside a wider pool, a table inside a wider one."""
    print("[gpu] attention strides", flush=True)
    import torch
    from chenxing_amd._lib import paged_attention_device
    x = _attend_inputs("verify")
    want, tol = _expect(x)
    q, pages, table = (C.to_gpu(x[k]) for k in ("q", "pages", "table"))
    T, Hq, D = q.shape
    wide = torch.full((Hq, T + 3, 3 * D), float("nan"), dtype=torch.bfloat16, device="cuda")
    qv = wide[:, 1:T + 1, D:2 * D].transpose(0, 1)
    qv.copy_(q)
    pool = torch.full((pages.shape[0], 5, pages.shape[2]), float("nan"), dtype=torch.bfloat16,
                      device="cuda")[:, 1:3]
    pool.copy_(pages)
    tab = torch.full((table.shape[0], table.shape[1] + 5), -1, dtype=torch.int32,
                     device="cuda")[:, 2:2 + table.shape[1]]
    tab.copy_(table)
    out = torch.empty(T, Hq, D, dtype=torch.bfloat16, device="cuda")
    got = paged_attention_device(qv, pool, tab, C.to_gpu(x["kv_len"]), C.to_gpu(x["q_start"]),
                                 max_new=5, out=out)
    assert got is out
    _check(out, want, tol)


def _attend_torch(q, k, v, pos, scale, window):
    """R.attend for one kv head of one sequence on the GPU: q [m, D] at positions
    pos [m], k and v [t, D], fp64."""
    import torch
    t = torch.arange(k.shape[0], device=k.device)
    ok = t <= pos[:, None]
    if window:
        ok &= t > pos[:, None] - window
    x = (q @ k.T.contiguous() * scale).masked_fill(~ok, -torch.inf)
    mag = q.abs() @ k.abs().T.contiguous() * scale
    top = x.amax(1, keepdim=True)
    p = torch.softmax(x, 1)
    o = p @ v
    ds = 2 * (q.shape[1] + 64) * R.U32 * mag + 8 * R.U32 * (x.masked_fill(~ok, 0).abs() + top.abs())
    rel = 2 * ds + (2 * ok.sum(1, keepdim=True) + 64) * R.U32 + 2.0 ** -16
    a = (p * rel) @ v.abs() + o.abs() * (p * rel).sum(1, keepdim=True)
    return o, a + R.U16 * 1.01 * (o.abs() + a) + 1e-38


# the lengths spread over the shares in every way: more row blocks than workers,
# sequences past those kept in LDS, parts joined by group, wave and workgroup
MANY = {
    "short_ones": ("bf16", 8, 4, 64, 16, 700, 0, 90, 1, 0),
    "more_than_lds": ("bf16", 2, 1, 128, 16, 1300, 0, 60, 2, 0),
    "short_e4m3": ("e4m3", 4, 2, 128, 32, 400, 0, 200, 1, 0),
    "waves": ("bf16", 4, 2, 128, 16, 45, 800, 4000, 1, 0),
    "waves_narrow": ("bf16", 6, 3, 64, 32, 40, 800, 4000, 1, 0),
    "waves_wide": ("bf16", 4, 2, 256, 32, 40, 500, 3000, 1, 0),
    "groups": ("bf16", 12, 3, 128, 16, 25, 300, 4000, 7, 0),
    "groups_e4m3": ("e4m3", 12, 3, 128, 16, 25, 300, 4000, 7, 900),
    "few_long": ("bf16", 8, 2, 64, 64, 3, 20000, 50000, 3, 0),
    "one_long_e4m3": ("e4m3", 4, 1, 256, 16, 1, 30000, 30000, 1, 0),
    "window": ("bf16", 8, 4, 128, 16, 90, 1, 6000, 3, 333),
    "window_long": ("bf16", 4, 2, 128, 16, 20, 1, 9000, 4, 2345),
    "window_many": ("bf16", 8, 4, 64, 16, 600, 0, 500, 2, 33),
    "window_many_e4m3": ("e4m3", 2, 1, 256, 16, 700, 0, 300, 1, 70),
    "prompts": ("bf16", 8, 2, 128, 16, 5, 300, 3500, 1700, 0),
    "prompts_window": ("bf16", 8, 2, 128, 16, 5, 300, 3500, 1700, 500),
    "prompts_e4m3": ("e4m3", 4, 1, 128, 32, 4, 300, 5000, 1500, 0),
    "prompts_e4m3_window": ("e4m3", 6, 2, 64, 32, 4, 1000, 3000, 1500, 77),
    "prompts_wide": ("bf16", 6, 2, 256, 16, 3, 1000, 4000, 900, 700),
    "prompts_narrow": ("bf16", 14, 2, 64, 16, 3, 1000, 5000, 2000, 0),
    "short_table": ("bf16", 12, 3, 128, 32, 60, 0, 700, 4, 0),
    "short_table_e4m3": ("e4m3", 6, 3, 64, 64, 130, 0, 900, 2, 0),
}


@pytest.mark.parametrize("name", MANY)
def test_attention_many(name):
    print(f"[gpu] attention {name}", flush=True)
    _check_many(name, *MANY[name])


def test_attention_more_row_blocks_than_workers_under_a_hint_of_one():
    """Prompts told to be single tokens, heads of 64: 4160 row blocks of 16 rows in
    a sequence, 4096 workers."""
    print("[gpu] attention of a prompt, max_new 1", flush=True)
    _check_many("hint", "bf16", 64, 64, 64, 16, 1, 1030, 1030, 1030, 0, max_new=1)


def _check_many(name, cache, Hq, H, D, P, B, lo, hi, most, window, max_new=None):
    import torch
    from chenxing_amd._lib import paged_attention_device
    rng = np.random.default_rng(sum(map(ord, name)))
    lens = rng.integers(lo, hi + 1, B)
    new = np.minimum(rng.integers(1 if most == 1 else 0, most + 1, B), np.maximum(lens, 1))
    if max_new:
        new = lens
    table, kv_len, q_start, n = C.batch(rng, lens.tolist(), new.tolist(), P)
    g = torch.Generator(device="cuda")
    g.manual_seed(len(name))
    K, V = (torch.randn(n, H, P, D, generator=g, device="cuda") for _ in range(2))
    if cache == "bf16":
        pages = torch.cat([x.bfloat16().view(n, H, P, D // 8, 8).transpose(2, 3).reshape(n, H, -1)
                           if i == 0 else
                           x.bfloat16().view(n, H, P // 8, 8, D).transpose(3, 4).reshape(n, H, -1)
                           for i, x in enumerate((K, V))], 2)
        K, V = (x.bfloat16().double() for x in (K, V))
    else:
        sc = [x.abs().amax(3) / 448 for x in (K, V)]
        code = [(x / s[..., None]).to(torch.float8_e4m3fn) for x, s in zip((K, V), sc)]
        K, V = (c.double() * s[..., None].double() for c, s in zip(code, sc))
        code = [c.view(torch.uint8) for c in code]
        pages = torch.cat([code[0].view(n, H, P, D // 16, 16).transpose(2, 3).reshape(n, H, -1),
                           code[1].view(n, H, P // 16, 16, D).transpose(3, 4).reshape(n, H, -1),
                           torch.cat(sc, 2).view(torch.uint8)], 2)
    T = int(q_start[-1])
    q = (2 * torch.randn(T, Hq, D, generator=g, device="cuda")).bfloat16()
    out = paged_attention_device(q, pages, C.to_gpu(table), C.to_gpu(kv_len),
                                 C.to_gpu(q_start), max_new=max_new or most,
                                 window=window).double()
    tab, G = C.to_gpu(table).long(), Hq // H
    assert out.isfinite().all()
    for b in range(B):
        m, L = int(new[b]), int(lens[b])
        if not m:
            continue
        rows = slice(int(q_start[b]), int(q_start[b]) + m)
        if L == 0:
            assert not out[rows].any()
            continue
        pg = tab[b, :-(-L // P)]
        pos = torch.arange(L - m, L, device="cuda").repeat_interleave(G)
        for h in range(H):
            k, v = (x[pg, h].reshape(-1, D)[:L] for x in (K, V))
            qh = q[rows, h * G:(h + 1) * G].reshape(m * G, D).double()
            keep = pos >= 0
            want, tol = _attend_torch(qh[keep], k, v, pos[keep], D ** -0.5, window)
            got = out[rows, h * G:(h + 1) * G].reshape(m * G, D)
            off = (got[keep] - want).abs()
            assert (off <= tol).all(), (b, h, L, m, off.max())
            assert not got[~keep].any()


def test_attention_repeats_bit_for_bit():
    print("[gpu] attention repeats", flush=True)
    import torch
    for name in ("long_and_short", "verify", "long_e4m3"):
        x = _attend_inputs(name)
        first = _attend(x)
        for _ in range(3):
            assert torch.equal(first.view(torch.int16), _attend(x).view(torch.int16))


def test_attention_rows_do_not_depend_on_the_workspace():
    """Any contents of the workspace: NaN, then another call's."""
    print("[gpu] attention workspace contents", flush=True)
    import torch
    from chenxing_amd import _lib
    x, y = _attend_inputs("long_and_short"), _attend_inputs("long")
    first = _attend(x)
    for buf in _lib._ws_attend.bufs.values():
        buf.fill_(0xFF)
    assert torch.equal(first.view(torch.int16), _attend(x).view(torch.int16))
    _attend(y)
    assert torch.equal(first.view(torch.int16), _attend(x).view(torch.int16))


# ------------------------------------------------------------------ append
APPEND = {
    # name: cache, Hq, Hkv, D, P, lengths, new, rotary dims, interleaved, norm
    "decode": ("bf16", 4, 2, 128, 16, [1, 16, 17, 200], [1] * 4, 128, False, False),
    "decode_norm": ("bf16", 8, 2, 128, 16, [1, 16, 17, 200], [1] * 4, 128, False, True),
    "no_rope": ("bf16", 4, 2, 64, 16, [3, 20], [1, 1], 0, False, True),
    "plain": ("bf16", 3, 1, 64, 32, [3, 20], [2, 1], 0, False, False),
    "partial_half": ("bf16", 4, 4, 128, 32, [9, 33, 64], [9, 2, 3], 48, False, True),
    "partial_pairs": ("bf16", 4, 4, 256, 32, [9, 33, 64], [9, 2, 3], 80, True, False),
    "wide": ("bf16", 2, 1, 256, 128, [300, 5], [40, 5], 256, False, True),
    "narrow_pairs": ("bf16", 5, 5, 64, 16, [77, 0, 12], [33, 0, 12], 64, True, True),
    "prompt": ("bf16", 4, 2, 128, 16, [200, 131, 70], [200, 128, 3], 128, False, True),
    "prompt_small": ("bf16", 2, 2, 64, 16, [80, 90], [79, 83], 16, False, False),
    "e4m3_decode": ("e4m3", 4, 2, 128, 16, [1, 16, 17, 200], [1] * 4, 128, False, True),
    "e4m3_prompt": ("e4m3", 4, 2, 128, 16, [200, 131, 70], [200, 128, 3], 64, True, True),
    "e4m3_wide": ("e4m3", 2, 1, 256, 64, [100, 50], [61, 50], 128, False, False),
    "e4m3_narrow": ("e4m3", 3, 3, 64, 32, [100, 50], [61, 50], 64, False, True),
    "more_new_than_tokens": ("bf16", 2, 2, 64, 16, [2, 0], [5, 3], 64, False, False),
    # neighbouring tokens of many sequences, with several chunks in a tile
    "many_few": ("bf16", 2, 1, 64, 16, [3 + 7 * b % 40 for b in range(300)],
                 [1 + b % 3 for b in range(300)], 64, False, True),
    "many_some": ("bf16", 2, 1, 128, 16, [12 + 7 * b % 40 for b in range(90)],
                  [1 + b % 12 for b in range(90)], 32, True, False),
    "many_some_e4m3": ("e4m3", 2, 1, 128, 32, [20 + 7 * b % 40 for b in range(90)],
                       [b % 21 for b in range(90)], 128, False, False),
    "many_wide_e4m3": ("e4m3", 1, 1, 256, 16, [20 + 7 * b % 40 for b in range(60)],
                       [b % 21 for b in range(60)], 256, True, True),
}


def _append_inputs(name, more=1):
    cache, Hq, Hkv, D, P, lens, new, r, inter, use_norm = APPEND[name]
    Hq, Hkv = Hq * more, Hkv * more
    rng = np.random.default_rng(len(name) * 31 + sum(map(ord, name)))
    table, kv_len, q_start, n = C.batch(rng, lens, new, P)
    T = int(q_start[-1])
    x = [f32_to_bf16_bits(rng.normal(0, 1.5, (T, h, D)).astype(np.float32)) for h in (Hq, Hkv, Hkv)]
    M = table.shape[1]
    ang = np.arange(M * P)[:, None] * 100.0 ** (-np.arange(max(r, 2) // 2) * 2 / max(r, 2))
    rope = np.concatenate([np.cos(ang), np.sin(ang)], 1).astype(np.float32) if r else None
    w = [f32_to_bf16_bits(rng.normal(1, 0.2, D).astype(np.float32)) for _ in range(2)] \
        if use_norm else [None, None]
    width = 2 * P * D + (0 if cache == "bf16" else 8 * P)
    pages = rng.integers(0, 100, (n, Hkv, width)).astype(np.uint16 if cache == "bf16" else np.uint8)
    return dict(q=x[0], k=x[1], v=x[2], pages=pages, table=table, kv_len=kv_len, q_start=q_start,
                rope=rope, inter=inter, w=w, new=new, P=P, D=D, cache=cache)


def _append(x, **kw):
    import torch
    from chenxing_amd._lib import kv_append_device
    pages = C.to_gpu(x["pages"])
    st = None if all(n == 1 for n in x["new"]) else C.to_gpu(x["q_start"])
    q = kv_append_device(C.to_gpu(x["q"]), C.to_gpu(x["k"]), C.to_gpu(x["v"]), pages,
                         C.to_gpu(x["table"]), C.to_gpu(x["kv_len"]), st,
                         rope=None if x["rope"] is None else C.to_gpu(x["rope"]),
                         interleaved=x["inter"],
                         q_norm=None if x["w"][0] is None else C.to_gpu(x["w"][0]),
                         k_norm=None if x["w"][1] is None else C.to_gpu(x["w"][1]), **kw)
    torch.cuda.synchronize()
    return q, pages


def _turned(x, bits, w, pos, eps):
    """(value, bound on the fp32 result before its rounding): a handful of
    roundings of the norm (its sum over D) and of the rotation, relative to
    the pair's magnitude."""
    a = _values(bits)
    wv = None if w is None else _values(w)
    n = R.norm(a, wv, eps)
    y = R.rotate(n, pos, x["rope"], x["inter"])
    mag = np.abs(n)
    if x["rope"] is not None:
        r = x["rope"].shape[1]
        m = mag.copy()
        ia, ib = (slice(0, r, 2), slice(1, r, 2)) if x["inter"] else (slice(0, r // 2),
                                                                      slice(r // 2, r))
        m[..., ia] = m[..., ib] = mag[..., ia] + mag[..., ib]
        mag = m
    err = mag * R.U32 * (6 + (0 if w is None else x["D"] / 2 + 8))
    if w is None and x["rope"] is None:
        err = mag * 0
    elif w is None:
        err[..., x["rope"].shape[1]:] = 0
    return y, err


def _near_bf16(got_bits, want, err, where=None):
    got = _values(got_bits)
    tol = err + R.U16 * (np.abs(want) + err) * 1.0001
    assert (np.abs(got - want) <= tol).all(), np.abs(got - want).max()


@pytest.mark.parametrize("name", APPEND)
def test_append(name):
    print(f"[gpu] append {name}", flush=True)
    _check_append(_append_inputs(name))


@pytest.mark.parametrize("name", [n for n, x in APPEND.items() if sum(x[6]) >= 2 * len(x[6]) and
                                  sum(x[6]) > 10])
def test_append_many_heads(name):
    """4 million elements or more: large calls are written by other means."""
    _, Hq, Hkv, D, _, _, new = APPEND[name][:7]
    more = -(-2 ** 22 // ((Hq + 2 * Hkv) * D * sum(new)))
    print(f"[gpu] append {name}, {more} times the heads", flush=True)
    _check_append(_append_inputs(name, more))


def _check_append(x):
    eps = 1e-5
    q, pages = _append(x, eps=eps)
    P, D, n = x["P"], x["D"], len(x["pages"])
    pl = R.places(x["kv_len"], x["q_start"], P, x["table"].shape[1], x["table"], n)
    pos = np.array([p for _, p, _, _ in pl])
    held = np.array([p[2] >= 0 for p in pl])
    qw, qe = _turned(x, x["q"], x["w"][0], pos, eps)
    _near_bf16(C.bits_of(q)[held], qw[held], qe[held])
    kw, ke = _turned(x, x["k"], x["w"][1], pos, eps)
    got = C.bits_of(pages)
    # the written tokens' values, then nothing else changed
    E = 8 if x["cache"] == "bf16" else 16
    same = np.ones(got.shape, bool)
    d = np.arange(D)
    for t, (_, _, pg, o) in enumerate(pl):
        if pg < 0:
            continue
        ka, va = R._at(P, D, E, o, d)
        same[pg][:, ka] = same[pg][:, va] = False
        if x["cache"] == "bf16":
            _near_bf16(got[pg][:, ka], kw[t], ke[t])
            assert np.array_equal(got[pg][:, va], x["v"][t])
            continue
        sc = got[pg][:, 2 * P * D:].copy().view(np.float32)
        same[pg][:, 2 * P * D + 4 * o:2 * P * D + 4 * o + 4] = False
        same[pg][:, 2 * P * D + 4 * (P + o):2 * P * D + 4 * (P + o) + 4] = False
        for want, err, at, s in ((kw[t], ke[t], ka, sc[:, o]),
                                 (_values(x["v"][t]), 0 * ke[t], va, sc[:, P + o])):
            top = np.abs(want).max(1)
            assert (np.abs(s * 448.0 - top) <= top * 2 * R.U32 + err.max(1)).all()
            # a code off the exact quotient by at most half a step and the
            # quotient's own error
            v = R.E4M3[got[pg][:, at]]
            y = want / s[:, None]
            half = np.maximum(2.0 ** (np.floor(np.log2(np.maximum(np.abs(y), 2.0 ** -9))) - 4),
                              2.0 ** -10)
            off = np.abs(v - y) - err / s[:, None] - np.abs(y) * 4 * R.U32
            assert (off <= half * 1.0001).all(), off.max()
    assert np.array_equal(got[same], x["pages"][same])


def test_append_e4m3_rows_without_a_scale():
    """Zeros, denormals, inf and NaN in a row."""
    print("[gpu] append e4m3 special rows", flush=True)
    x = _append_inputs("e4m3_decode")
    x["rope"], x["w"] = None, [None, None]
    for name in ("k", "v"):
        x[name][0] = 0
        x[name][1] = 1                            # 2^-133
        x[name][2, :, 7] = 0x7F80
        x[name][3, :, 9] = C.NAN16
    q, pages = _append(x)
    K, V = R.unpack(C.bits_of(pages), 128)
    for b in range(4):
        pos = x["kv_len"][b] - 1
        pg, o = x["table"][b, pos // 16], pos % 16
        for y in (K[pg, :, o], V[pg, :, o]):
            if b < 2:
                assert (np.abs(y) <= 2.0 ** -126).all()
            else:
                assert np.isnan(y).all()


def test_append_strides_and_bad_ids():
    """q, k and v as views of one projection; a page id outside the pool and
    a position past the table write nothing."""
    print("[gpu] append strides and bad ids", flush=True)
    import torch
    from chenxing_amd._lib import kv_append_device
    x = _append_inputs("prompt")
    q0, pages0 = _append(x)
    qkv = torch.cat([C.to_gpu(x[k]) for k in ("q", "k", "v")], 1)
    Hq, H = x["q"].shape[1], x["k"].shape[1]
    n, width = len(x["pages"]), x["pages"].shape[2]
    pool = torch.zeros(n, H + 3, width, dtype=torch.bfloat16, device="cuda")
    pool[:, 1:1 + H] = C.to_gpu(x["pages"])
    table = C.to_gpu(x["table"])
    rope = C.to_gpu(x["rope"])
    w = [C.to_gpu(a) for a in x["w"]]
    args = (table, C.to_gpu(x["kv_len"]), C.to_gpu(x["q_start"]))
    q = kv_append_device(qkv[:, :Hq], qkv[:, Hq:Hq + H], qkv[:, Hq + H:], pool[:, 1:1 + H], *args,
                         rope=rope, q_norm=w[0], k_norm=w[1])
    assert torch.equal(q, q0) and torch.equal(pool[:, 1:1 + H].contiguous().view(torch.int16),
                                              pages0.view(torch.int16))
    assert not pool[:, 0].any() and not pool[:, 1 + H:].any()
    table[0, 2] = n
    table[1, 3] = -1
    lens = C.to_gpu(np.array([x["kv_len"][0], x["kv_len"][1], 10 ** 9], np.int32))
    pages1 = C.to_gpu(x["pages"])
    kv_append_device(qkv[:, :Hq], qkv[:, Hq:Hq + H], qkv[:, Hq + H:], pages1, table, lens, args[2],
                     rope=rope, q_norm=w[0], k_norm=w[1])
    skipped = [x["table"][0, 2], x["table"][1, 3],
               *x["table"][2, (x["kv_len"][2] - 3) // 16:][:1]]
    got, was, full = C.bits_of(pages1), x["pages"], C.bits_of(pages0)
    for pg in range(n):
        assert np.array_equal(got[pg], was[pg] if pg in skipped else full[pg]), pg


# ------------------------------------------------------------------ copies
@pytest.mark.parametrize("layers,n,H,width,pairs", [
    (1, 4, 1, 2 * 16 * 64, 1), (3, 40, 2, 2 * 32 * 128, 13), (2, 9, 8, 2 * 128 * 256, 4),
    (5, 33, 3, 2 * 16 * 64 + 8 * 16, 16)])
def test_copy_pages(layers, n, H, width, pairs):
    print(f"[gpu] copy {pairs} of {n} pages, {layers} layers", flush=True)
    import torch
    from chenxing_amd._lib import kv_copy_pages_device
    rng = np.random.default_rng(n)
    pool = torch.from_numpy(rng.integers(0, 256, (layers, n, H, width), np.uint8)).cuda()
    order = rng.permutation(n)
    dst = order[:pairs].astype(np.int32)
    src = order[pairs + rng.integers(0, min(pairs, n - pairs), pairs)].astype(np.int32)
    bad = np.array([[-1, 0], [n, 1], [2, -5], [3, n]], np.int32)
    ref = pool.cpu().numpy()
    ref[:, dst] = ref[:, src]
    s = torch.from_numpy(np.concatenate([src, bad[:, 0]])).cuda()
    d = torch.from_numpy(np.concatenate([dst, bad[:, 1]])).cuda()
    assert kv_copy_pages_device(pool, s, d) is pool
    assert np.array_equal(pool.cpu().numpy(), ref)
    # one layer of it, in place
    kv_copy_pages_device(pool[layers - 1], d[:1].clone(), s[:1].clone())
    ref[layers - 1, src[0]] = ref[layers - 1, dst[0]]
    assert np.array_equal(pool.cpu().numpy(), ref)
    kv_copy_pages_device(pool, s[:0], d[:0])


# ------------------------------------------------------------------ together
def test_offsets_past_32_bits():
    """A pool of 6.4 GB whose last pages are written, copied and attended."""
    print("[gpu] a pool past 4 GB", flush=True)
    import torch
    from chenxing_amd._lib import (kv_append_device, kv_copy_pages_device,
                                   paged_attention_device)
    Hq, H, D, P, n = 8, 2, 128, 16, 200_000
    pool = torch.empty(n, H, 2 * P * D, dtype=torch.bfloat16, device="cuda")
    lens = [100, 33]
    rng = np.random.default_rng(8)
    table = np.stack([n - 1 - np.arange(7), np.r_[n - 50 - np.arange(3), [0] * 4]]).astype(np.int32)
    T = sum(lens)
    x = [f32_to_bf16_bits(rng.normal(0, 1, (T, h, D)).astype(np.float32)) for h in (Hq, H, H)]
    q, k, v = (C.to_gpu(a) for a in x)
    meta = (C.to_gpu(np.array(lens, np.int32)), C.to_gpu(np.array([0, 100, 133], np.int32)))
    kv_append_device(q, k, v, pool, C.to_gpu(table), *meta)
    move = np.arange(10, 20).astype(np.int32)
    kv_copy_pages_device(pool, C.to_gpu(table.reshape(-1)[:10].copy()), C.to_gpu(move + n // 2))
    moved = table.copy()
    moved.reshape(-1)[:10] = move + n // 2
    outs = [paged_attention_device(q, pool, C.to_gpu(t), *meta, max_new=100) for t in (table, moved)]
    assert torch.equal(outs[0].view(torch.int16), outs[1].view(torch.int16))
    dense = np.zeros((2, 10, H, P, D))
    pages = np.arange(14).reshape(2, 7) % 10
    at = 0
    for b, m in enumerate(lens):
        for s in range(m):
            dense[:, pages[b, s // P], :, s % P] = [_values(x[1][at + s]), _values(x[2][at + s])]
        at += m
    want, tol = R.attend(_values(x[0]), dense[0], dense[1], pages, lens, [0, 100, 133], P,
                         D ** -0.5)
    _check(outs[0], want, tol)


def test_another_stream_and_graph_replays():
    """Append and attention on a stream of their own, then captured in a graph
    whose lengths and inputs change between replays."""
    print("[gpu] another stream, a graph", flush=True)
    import torch
    from chenxing_amd._lib import kv_append_device, paged_attention_device
    x = _append_inputs("decode")
    name = {k: C.to_gpu(x[k]) for k in ("q", "k", "v", "table", "kv_len", "rope")}
    pages = C.to_gpu(np.zeros_like(x["pages"]))
    pages.normal_()
    out = torch.empty_like(name["q"])
    qo = torch.empty_like(name["q"])

    def step():
        kv_append_device(name["q"], name["k"], name["v"], pages, name["table"], name["kv_len"],
                         rope=name["rope"], q_out=qo)
        paged_attention_device(qo, pages, name["table"], name["kv_len"], out=out)

    step()
    torch.cuda.synchronize()
    first = out.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    out.zero_()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    assert torch.equal(out, first)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        step()
        side.synchronize()
        with torch.cuda.graph(g, stream=side):
            step()
    lens = name["kv_len"].clone()
    for i in range(4):
        name["kv_len"].copy_(torch.clamp(lens - i, min=1))
        name["q"].normal_()
        name["k"].normal_()
        torch.cuda.synchronize()
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        got = out.clone()
        step()
        torch.cuda.synchronize()
        assert torch.equal(got, out) and out.abs().sum() > 0


def test_refusals():
    import torch
    from chenxing_amd._lib import (kv_append_device, kv_copy_pages_device,
                                   paged_attention_device)
    bf, i32 = torch.bfloat16, torch.int32

    def z(*shape, dtype=bf):
        return torch.zeros(*shape, dtype=dtype, device="cuda")

    q, cache, table, lens = z(2, 4, 64), z(3, 2, 2 * 16 * 64), z(2, 1, dtype=i32), z(2, dtype=i32)
    paged_attention_device(q, cache, table, lens)
    kv_append_device(q, q[:, :2], q[:, 2:], cache, table, lens)
    for bad in (dict(q=q.float()), dict(q=q.cpu()), dict(q=z(3, 4, 64)), dict(q=z(2, 3, 64)),
                dict(q=z(2, 4, 128)[..., ::2]), dict(q=z(2, 4, 32)), dict(q=z(2 * 4 * 64 + 8)[1:513].view(2, 4, 64)),
                dict(q=z(2, 4, 68)[..., :64]), dict(cache=cache.float()), dict(cache=z(3, 2, 2 * 16 * 64 + 2)),
                dict(cache=z(3, 2, 2 * 24 * 64)), dict(cache=z(3, 4, 2 * 16 * 64)[:, ::2]),
                dict(table=table.long()), dict(table=z(3, 1, dtype=i32)), dict(lens=lens.long()),
                dict(lens=lens.cpu()), dict(cache=cache.cpu())):
        a = {**dict(q=q, cache=cache, table=table, lens=lens), **bad}
        with pytest.raises(ValueError):
            paged_attention_device(a["q"], a["cache"], a["table"], a["lens"])
    for kw in (dict(max_new=0), dict(window=-1), dict(softcap=-1.0), dict(softcap=float("nan")),
               dict(scale=0.0), dict(scale=float("nan")), dict(out=z(2, 4, 128)),
               dict(out=z(2, 4, 64, dtype=torch.float32)), dict(q_start=z(2, dtype=i32)),
               dict(q_start=z(3, dtype=torch.int64))):
        with pytest.raises(ValueError):
            paged_attention_device(q, cache, table, lens, **kw)
    k = q[:, :2]
    for kw in (dict(rope=z(16, 24, dtype=torch.float32)), dict(rope=z(15, 64, dtype=torch.float32)),
               dict(rope=z(16, 80, dtype=torch.float32)), dict(rope=z(16, 64)),
               dict(q_norm=z(64, dtype=torch.float32)), dict(k_norm=z(128)), dict(eps=-1.0),
               dict(eps=float("nan")), dict(q_out=z(2, 4, 128))):
        with pytest.raises(ValueError):
            kv_append_device(q, k, k, cache, table, lens, **kw)
    with pytest.raises(ValueError):
        kv_append_device(q, q, k, cache, table, lens)
    s = z(1, dtype=i32)
    for a in ((cache, s.long(), s), (cache, s, z(2, dtype=i32)), (cache.cpu(), s, s),
              (cache, s.cpu(), s.cpu()), (z(3, 2, 7), s, s), (z(3, 4, 64)[:, ::2], s, s),
              (z(8, 64), s, s)):
        with pytest.raises(ValueError):
            kv_copy_pages_device(*a)
