"""Products with 4-bit weights against their restatement (oracle/w4_ref.py)."""
from __future__ import annotations

import numpy as np
import pytest

import paged_cases as C
from oracle import w4_ref as R
from oracle.bf16 import bf16_bits_to_f32, f32_to_bf16_bits

pytestmark = pytest.mark.gpu


def _inputs(M, N, K, group, shift, seed=0, offset=0.0):
    rng = np.random.default_rng(M * 7 + N + K + group + seed)
    codes = rng.integers(0, 16, (N, K), dtype=np.uint8)
    scale = (rng.uniform(0.5, 1.5, (N, K // group)) / 16 * rng.choice([-1, 1], (N, K // group))).astype(np.float16)
    sh = (-scale * rng.uniform(6, 9, scale.shape)).astype(np.float16) if shift else None
    x = f32_to_bf16_bits(rng.normal(offset, 1, (M, K)).astype(np.float32))
    return x, codes, scale, sh


def _check(x, codes, scale, sh, got, bf16):
    want, tol = R.linear(bf16_bits_to_f32(x).astype(np.float64), codes, scale, sh, bf16)
    got = C.bits_of(got)
    got = (bf16_bits_to_f32(got) if bf16 else got).astype(np.float64)
    off = np.abs(got - want)
    assert (off <= tol).all(), (np.argwhere(off > tol)[:4].tolist(), float((off / tol).max()))


SIZES = [(1, 16, 32, 32), (1, 1, 64, 64), (1, 17, 128, 128), (3, 100, 96, 32), (2, 33, 192, 64),
         (5, 513, 1024, 128), (16, 200, 640, 32), (17, 48, 256, 64), (32, 96, 1056, 32),
         (33, 50, 384, 128), (48, 70, 448, 64), (61, 129, 512, 128), (64, 64, 4096, 32),
         (65, 40, 256, 32), (130, 31, 320, 64), (1, 4096, 4096, 128), (1, 130, 14336, 128),
         (7, 130, 14336, 32), (4, 5001, 256, 64), (16, 20001, 128, 32), (40, 9000, 160, 32)]


@pytest.mark.parametrize("shift", [False, True])
@pytest.mark.parametrize("M,N,K,group", SIZES)
def test_linear(M, N, K, group, shift):
    import torch
    from chenxing_amd import w4
    from chenxing_amd._lib import w4_linear_device
    x, codes, scale, sh = _inputs(M, N, K, group, shift)
    tiles, scales = w4.pack(*(None if t is None else torch.from_numpy(t).cuda()
                              for t in (codes, scale, sh)))
    for dtype in (torch.float32, torch.bfloat16):
        got = w4_linear_device(C.to_gpu(x), tiles, scales, N, dtype)
        assert got.dtype == dtype and got.shape == (M, N)
        _check(x, codes, scale, sh, got, dtype == torch.bfloat16)


@pytest.mark.parametrize("M", [1, 9, 40])
def test_offset_inputs(M):
    """Inputs far from zero: the sums of x and of its products nearly cancel."""
    from chenxing_amd import w4
    import torch
    x, codes, scale, sh = _inputs(M, 77, 1024, 64, True, 1, 30.0)
    w = w4.W4Weight(*(torch.from_numpy(t).cuda() for t in (codes, scale, sh)))
    _check(x, codes, scale, sh, w(C.to_gpu(x)), False)


def test_strided_rows_and_out():
    import torch
    from chenxing_amd import w4
    x, codes, scale, sh = _inputs(5, 37, 256, 32, False, 3)
    w = w4.W4Weight(*(None if t is None else torch.from_numpy(t).cuda() for t in (codes, scale, sh)))
    wide = torch.full((5, 2, 264), float("nan"), dtype=torch.bfloat16, device="cuda")
    wide[:, 1, :256] = C.to_gpu(x)
    for dtype in (torch.float32, torch.bfloat16):
        out = torch.full((7, 41), 5.0, dtype=dtype, device="cuda")
        w(wide[:, 1, :256], out=out[1:6, 2:39])
        _check(x, codes, scale, sh, out[1:6, 2:39], dtype == torch.bfloat16)
        keep = torch.ones(7, 41, dtype=torch.bool, device="cuda")
        keep[1:6, 2:39] = False
        assert (out[keep] == 5.0).all()


def test_rows_that_are_not_finite_touch_no_other():
    import torch
    from chenxing_amd import w4
    x, codes, scale, sh = _inputs(6, 40, 256, 64, True, 4)
    w = w4.W4Weight(*(torch.from_numpy(t).cuda() for t in (codes, scale, sh)))
    bad = x.copy()
    bad[1, 7], bad[4, 255] = 0x7FC0, 0x7F80
    got = w(C.to_gpu(bad))
    assert torch.isnan(got[[1, 4]]).all()
    fine = [0, 2, 3, 5]
    _check(x[fine], codes, scale, sh, got[fine], False)


def test_zero_scales_and_extreme_codes():
    import torch
    from chenxing_amd import w4
    x, codes, scale, _ = _inputs(3, 64, 512, 128, False, 5)
    codes[:16], codes[16:32] = 0, 15
    scale[::3] = 0
    w = w4.W4Weight(*(torch.from_numpy(t).cuda() for t in (codes, scale)))
    got = w(C.to_gpu(x))
    assert (got[:, ::3] == 0).all()
    _check(x, codes, scale, None, got, False)


def test_quantized_weights_are_near():
    """Codes are the nearest of 15 steps a group: off by half a step at most (and the
    scale's and shift's roundings to 11 bits, of 15 steps and of the shift)."""
    import torch
    from chenxing_amd import w4
    g = torch.Generator().manual_seed(1)
    for group in (32, 64, 128):
        w = torch.randn(50, 256, generator=g)
        w[3], w[4, :128] = 0.25, 0.0
        codes, scale, shift = w4.quantize(w.cuda(), group)
        back = R.weights(codes.cpu().numpy(), scale.cpu().numpy(), shift.cpu().numpy())
        s = scale.float().repeat_interleave(group, 1).cpu().numpy()
        t = shift.float().abs().repeat_interleave(group, 1).cpu().numpy()
        assert (np.abs(back - w.numpy()) <= 0.5 * s * 1.01 + 2.0 ** -11 * (15 * s + t) + 1e-7).all()


def test_captured_and_replayed():
    import torch
    from chenxing_amd import w4
    x, codes, scale, sh = _inputs(9, 500, 1024, 64, True, 6)
    w = w4.W4Weight(*(torch.from_numpy(t).cuda() for t in (codes, scale, sh)))
    mine = C.to_gpu(x)
    w(mine)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = w(mine)
    for seed in range(3):
        y, *_ = _inputs(9, 500, 1024, 64, True, 10 + seed)
        mine.copy_(C.to_gpu(y))
        g.replay()
        other = w(C.to_gpu(x))
        torch.cuda.synchronize()
        _check(y, codes, scale, sh, out, False)
        _check(x, codes, scale, sh, other, False)


def test_no_rows():
    import torch
    from chenxing_amd import w4
    _, codes, scale, sh = _inputs(1, 20, 64, 32, False)
    w = w4.W4Weight(*(None if t is None else torch.from_numpy(t).cuda() for t in (codes, scale, sh)))
    assert w(torch.empty(0, 64, dtype=torch.bfloat16, device="cuda")).shape == (0, 20)


@pytest.mark.parametrize("M", [1, 16, 20, 32, 61, 64])
@pytest.mark.parametrize("N", [130, 6160, 12300, 24580, 49170, 98320])
@pytest.mark.parametrize("K,group", [(64, 32), (64, 64), (128, 128), (1056, 32), (1216, 64)])
def test_every_split(M, N, K, group):
    """Rows of W a wave and waves of a row go by N; K ends in and on a tile of 128."""
    import torch
    from chenxing_amd import w4
    from chenxing_amd._lib import w4_linear_device
    if K > 128 and N > 20000:
        K -= 1024 - 128 if N < 90000 else 1024
    shift = (M + N // 10) % 2 == 0
    g = torch.Generator(device="cuda").manual_seed(M + N + K)
    codes = torch.randint(0, 16, (N, K), generator=g, device="cuda", dtype=torch.uint8)
    scale = ((torch.rand(N, K // group, generator=g, device="cuda") + 0.5) / 16).half()
    sh = (-7.3 * scale).half() if shift else None
    x = torch.randn(M, K, generator=g, device="cuda").bfloat16()
    got = w4_linear_device(x, *w4.pack(codes, scale, sh), N, torch.float32)
    # codes and halves are exact in float64, and R.linear's bound holds for each n: checked
    # on the rows of W where tiles, waves and workgroups begin and end, all against float64
    w = codes.double() * scale.double().repeat_interleave(group, 1)
    w += (sh.double() if shift else -8 * scale.double()).repeat_interleave(group, 1)
    off = (got.double() - x.double() @ w.T).abs()
    rows = sorted({r for b in range(0, N, 16 * 64) for r in (b, b + 15, b + 16, b + 31) if r < N} | {N - 1})
    _, tol = R.linear(x.double().cpu().numpy(), codes[rows].cpu().numpy(), scale[rows].cpu().numpy(),
                      sh[rows].cpu().numpy() if shift else None, False)
    assert (off[:, rows].cpu().numpy() <= tol).all()
    # the others by the largest of their bounds
    assert (off <= 2 * float(tol.max())).all(), float(off.max())


@pytest.mark.parametrize("M", [2, 16])
def test_rows_far_apart(M):
    """Rows of x whose distances pass 32 bits."""
    import torch
    from chenxing_amd import w4
    x, codes, scale, sh = _inputs(M, 70, 192, 64, True, 8)
    w = w4.W4Weight(*(torch.from_numpy(t).cuda() for t in (codes, scale, sh)))
    for step in (1 << 26, (1 << 28) + 8):
        wide = torch.empty((M - 1) * step + 192, dtype=torch.bfloat16, device="cuda")
        rows = wide.as_strided((M, 192), (step, 1))
        rows.copy_(C.to_gpu(x))
        _check(x, codes, scale, sh, w(rows), False)
