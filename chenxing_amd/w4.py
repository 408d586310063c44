"""4-bit weights with group scales, laid out for ``_lib.w4_linear_device``.

A weight is ``scale * code + shift`` of its group of 32, 64 or 128 neighbours along
K, or ``scale * (code - 8)`` without shifts; codes are 0 .. 15, scales and shifts
float16.  (The reference's 4-bit weights are numpy formats of files,
chenxing/core/quantization.py; those with a scale and a minimum a group of 32 fit.)
"""
from __future__ import annotations

__all__ = ["pack", "quantize", "W4Weight"]


def pack(codes, scale, shift=None):
    """(tiles, scales) of codes [N, K] (uint8, 0 .. 15), scale and shift [N, K /
    group], on the codes' device: once, when a model is loaded."""
    import torch
    if codes.dim() != 2 or codes.dtype != torch.uint8:
        raise ValueError("codes must be uint8 [N, K]")
    N, K = codes.shape
    if scale.dim() != 2 or scale.shape[0] != N or scale.shape[1] < 1 or K % scale.shape[1] or \
            K // scale.shape[1] not in (32, 64, 128):
        raise ValueError("scale must be [N, K / group], group 32, 64 or 128")
    if shift is not None and shift.shape != scale.shape:
        raise ValueError("scale and shift differ in shape")
    if N and int(codes.max()) > 15:
        raise ValueError("codes must be 0 .. 15")
    n16, k128 = -(-N // 16), -(-K // 128)
    at = torch.tensor([[0, 16], [4, 20], [8, 24], [12, 28]], dtype=torch.int32, device=codes.device)
    tiles = torch.empty(n16, k128, 64, 4, dtype=torch.int32, device=codes.device)
    rows = max(1, (1 << 26) // (128 * k128) // 16) * 16           # at a time
    for i in range(0, N, rows):
        part = codes[i:i + rows]
        n = -(-part.shape[0] // 16)
        x = torch.zeros(16 * n, 128 * k128, dtype=torch.int32, device=codes.device)
        x[:part.shape[0], :K] = part
        # [tile, row, k tile, word, lane group, pair, odd]; no two codes share a bit
        x = (x.view(n, 16, k128, 4, 4, 4, 2) << at).sum((5, 6), dtype=torch.int32)
        tiles[i // 16:i // 16 + n] = x.permute(0, 2, 4, 1, 3).reshape(n, k128, 64, 4)
    both = scale.half()[..., None] if shift is None else torch.stack([scale.half(), shift.half()], 2)
    if not bool(torch.isfinite(both).all()):
        raise ValueError("scale and shift must be finite, and in the range of float16")
    laid = torch.zeros(16 * n16, *both.shape[1:], dtype=torch.float16, device=codes.device)
    laid[:N] = both
    laid = laid.view(n16, 16, *both.shape[1:]).transpose(1, 2).contiguous()
    return tiles, laid[..., 0].contiguous() if shift is None else laid


def quantize(w, group=64):
    """(codes, scale, shift) of weights [N, K]: each group's least value to its
    largest in 15 steps."""
    import torch
    N, K = w.shape
    if group not in (32, 64, 128) or K % group:
        raise ValueError("group must be 32, 64 or 128, and K a multiple of it")
    x = w.float().view(N, K // group, group)
    lo, hi = x.amin(2), x.amax(2)
    # the codes are those of the scale and shift that are kept
    shift = lo.half()
    scale = ((hi - shift.float()) / 15).half()
    if not bool(torch.isfinite(scale).all() & torch.isfinite(shift).all()):
        raise ValueError("weights must be finite, and in the range of float16")
    step = scale.float()[..., None]
    q = torch.where(step > 0, (x - shift.float()[..., None]) / step, 0.0)
    return q.round().clamp(0, 15).byte().view(N, K), scale, shift


class W4Weight:
    """A weight matrix [N, K] of 4 bits; ``weight(x)`` is ``x @ W.T``."""

    def __init__(self, codes, scale, shift=None) -> None:
        self.shape = tuple(codes.shape)
        self.tiles, self.scales = pack(codes, scale, shift)

    @classmethod
    def of(cls, w, group=64) -> "W4Weight":
        return cls(*quantize(w, group))

    def __call__(self, x, dtype=None, out=None):
        from . import _lib
        return _lib.w4_linear_device(x, self.tiles, self.scales, self.shape[0], dtype, out)
