"""8-bit block tensors, the counter-based random mask and the plain PyTorch forms of the operators around them.

The HIP kernels (``csrc/block_ops.hip``, ``csrc/fp8_gemm.hip``) and the reference path share these definitions:

* e4m3 values in blocks of 128 with one power-of-two scale ``2^e`` a block, ``e`` the smallest exponent with
  ``max|v| <= 448 * 2^e`` (0 for a block of zeros; infinities and NaN do not enter the maximum and are stored as NaN).
  e4m3 is a floating format, so a power of two costs no significand bits, and the matrix instructions apply it.
* dropout element ``n`` (row-major) takes the ``n % 8``-th 16-bit number of the Philox4x32-10 block with counter
  ``(n // 8, offset)`` and key ``seed`` (Salmon et al., "Parallel random numbers: as easy as 1, 2, 3", SC 2011): kept
  where that number is at least ``t = round(65536 p)``, and scaled by ``65536 / (65536 - t)``.
"""
from __future__ import annotations

import torch
import torch.nn.functional as F

BLOCK = 128
E4M3 = torch.float8_e4m3fn
FLOATS = (torch.bfloat16, torch.float16, torch.float32)


def padded_cols(cols: int) -> int:
    return -(-cols // BLOCK) * BLOCK


def scale_cols(cols: int) -> int:
    """Scale bytes a row: one for each block, rounded up to 4 (kernels read whole words)."""
    return -(-(-(-cols // BLOCK)) // 4) * 4


class Fp8Blocks:
    """A matrix ``[rows, cols]`` in e4m3 with one scale byte (exponent + 127) for each block of 128 columns.

    ``q``      float8_e4m3fn ``[rows, cols rounded up to 128]``; what stands behind ``cols`` counts as zeros (the
               quantisers write zeros there);
    ``scale``  uint8 ``[ceil(rows / tile), blocks rounded up to 4]``; 255 makes its block NaN; bytes behind the last
               block are not read for their value;
    ``tile``   rows that share a scale: 1 (activations) or 128 (weights).

    Made by ``quantize_fp8`` / ``quantize_fp8_weight`` / ``rms_norm_fp8``, or from a checkpoint's 8-bit weights."""

    __slots__ = ("q", "scale", "shape", "tile")

    def __init__(self, q: torch.Tensor, scale: torch.Tensor, shape, tile: int = 1):
        rows, cols = (int(s) for s in shape)
        if tile not in (1, BLOCK):
            raise ValueError(f"Fp8Blocks: tile must be 1 or {BLOCK}, got {tile}")
        if rows < 0 or cols < 1:
            raise ValueError(f"Fp8Blocks: shape {(rows, cols)}")
        if q.dtype != E4M3 or tuple(q.shape) != (rows, padded_cols(cols)) or not q.is_contiguous():
            raise ValueError(f"Fp8Blocks: q must be contiguous float8_e4m3fn {(rows, padded_cols(cols))}, "
                             f"got {q.dtype} {tuple(q.shape)}")
        want = (-(-rows // tile), scale_cols(cols))
        if scale.dtype != torch.uint8 or tuple(scale.shape) != want or not scale.is_contiguous():
            raise ValueError(f"Fp8Blocks: scale must be contiguous uint8 {want}, got {scale.dtype} {tuple(scale.shape)}")
        if q.device != scale.device:
            raise ValueError(f"Fp8Blocks: q on {q.device}, scale on {scale.device}")
        self.q, self.scale, self.shape, self.tile = q, scale, (rows, cols), tile

    @classmethod
    def _made(cls, q, scale, shape, tile):
        """Blocks that a quantiser of this package has just laid out (nothing left to check)."""
        self = cls.__new__(cls)
        self.q, self.scale, self.shape, self.tile = q, scale, shape, tile
        return self

    @property
    def device(self):
        return self.q.device

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The values this stands for, as ``dtype`` (bfloat16 and float32 hold them exactly)."""
        from . import functional as Fx
        if dtype not in FLOATS:
            raise ValueError(f"dequantize: dtype {dtype}")
        if Fx.use_hip(self.q):
            return Fx._hip().fp8_dequantize(self, dtype)
        return dequantize_ref(self).to(dtype)


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def drop_threshold(p: float) -> int:
    return min(65536, int(p * 65536 + 0.5))


def drop_scale(t: int) -> float:
    return 65536.0 / (65536 - t) if t < 65536 else 0.0


def keep_mask(n: int, t: int, seed: int, offset: int, device) -> torch.Tensor:
    """The ``n`` keep flags in row-major order."""
    low = 0xFFFFFFFF
    g = torch.arange(-(-n // 8), dtype=torch.int64, device=device)
    c0, c1 = g & low, g >> 32
    c2, c3 = torch.full_like(g, offset & low), torch.full_like(g, (offset >> 32) & low)
    k0, k1 = seed & low, (seed >> 32) & low
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # wraps past 63 bits; the words are masked out of it
        c0, c1, c2, c3 = ((p1 >> 32) & low) ^ c1 ^ k0, p1 & low, ((p0 >> 32) & low) ^ c3 ^ k1, p0 & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    halves = torch.stack([h for c in (c0, c1, c2, c3) for h in (c & 0xFFFF, c >> 16)], 1)
    return halves.reshape(-1)[:n] >= t


def drop_ref(v: torch.Tensor, t: int, seed: int, offset: int) -> torch.Tensor:
    """float32 / float64 values -> kept * scale, 0 elsewhere (also where a dropped value is infinite)."""
    keep = keep_mask(v.numel(), t, seed, offset, v.device).view(v.shape)
    return torch.where(keep, v * drop_scale(t), torch.zeros((), dtype=v.dtype, device=v.device))


def block_exponent(amax: torch.Tensor) -> torch.Tensor:
    m, ex = torch.frexp(amax.float())  # amax = m * 2^ex with 0.5 <= m < 1; 448 = 0.875 * 2^9
    e = torch.where(m <= 0.875, ex - 9, ex - 8)
    return torch.where(amax > 0, e, torch.zeros_like(e)).clamp(min=-127)


def _pow2(e: torch.Tensor) -> torch.Tensor:
    """2^e in float32, exactly, for -127 <= e <= 127; NaN for 128 (the E8M0 byte 255)."""
    normal = ((e.to(torch.int32) + 127).clamp(min=1) << 23).view(torch.float32)
    return torch.where(e < -126, normal / 2, torch.where(e > 127, torch.nan, normal))


def _finite_amax(v, dims, keepdim=True):
    return torch.where(v.isfinite(), v, torch.zeros((), dtype=v.dtype, device=v.device)).abs().amax(dims, keepdim)


def _to_e4m3(v, e):
    s = torch.where(v.isfinite(), v * _pow2(-e), torch.full((), float("nan"), device=v.device))
    return s.to(E4M3)


def quantize_rows_ref(x: torch.Tensor) -> Fp8Blocks:
    rows, cols = x.shape
    b = F.pad(x.float(), (0, padded_cols(cols) - cols)).view(rows, padded_cols(cols) // BLOCK, BLOCK)
    e = block_exponent(_finite_amax(b, 2))
    scale = torch.full((rows, scale_cols(cols)), 127, dtype=torch.uint8, device=x.device)
    scale[:, :b.shape[1]] = (e[..., 0] + 127).to(torch.uint8)
    return Fp8Blocks(_to_e4m3(b, e).reshape(rows, padded_cols(cols)), scale, (rows, cols), 1)


def quantize_tiles_ref(w: torch.Tensor) -> Fp8Blocks:
    rows, cols = w.shape
    p = F.pad(w.float(), (0, padded_cols(cols) - cols, 0, -rows % BLOCK))
    b = p.view(p.shape[0] // BLOCK, BLOCK, -1, BLOCK)
    e = block_exponent(_finite_amax(b, (1, 3)))
    scale = torch.full((b.shape[0], scale_cols(cols)), 127, dtype=torch.uint8, device=w.device)
    scale[:, :b.shape[2]] = (e[:, 0, :, 0] + 127).to(torch.uint8)
    return Fp8Blocks(_to_e4m3(b, e).view(p.shape)[:rows].contiguous(), scale, (rows, cols), BLOCK)


def dequantize_ref(b: Fp8Blocks) -> torch.Tensor:
    rows, cols = b.shape
    nb = b.q.shape[1] // BLOCK
    e = b.scale[:, :nb].to(torch.int32) - 127
    s = _pow2(e.repeat_interleave(b.tile, 0)[:rows]).repeat_interleave(BLOCK, 1)
    return (b.q.float() * s)[:, :cols]


class _RowsThrough8Bits(torch.autograd.Function):
    """y = q(x) q(w)^T + b with dx = q(dy) q(w), dw = dy^T x on bfloat16 operands, db = column sums: the linear layer of
    ``linear_fp8`` in plain torch operations."""

    @staticmethod
    def forward(ctx, x, w, b, act):
        wq = dequantize_ref(quantize_tiles_ref(w))
        y = dequantize_ref(quantize_rows_ref(x)) @ wq.t()
        if b is not None:
            y = y + b.float()
        if act == "relu":
            y = y.clamp(min=0)
        y = y.to(x.dtype)
        ctx.save_for_backward(x, w, wq, y if act == "relu" else None)
        ctx.has_b = b is not None
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, w, wq, y = ctx.saved_tensors
        g = dy.float()
        if y is not None:
            g = torch.where(y <= 0, torch.zeros_like(g), g)
        dx = (dequantize_ref(quantize_rows_ref(g)) @ wq).to(x.dtype)
        dw = (g.bfloat16().float().t() @ x.bfloat16().float()).to(w.dtype)
        return dx, dw, g.sum(0) if ctx.has_b else None, None


def linear_fp8_ref(x2, w, b, act):
    return _RowsThrough8Bits.apply(x2, w, b, act)


def _rms_parts(x, residual, eps, t, seed, offset):
    """(h in x's type, h in float32, 1 / sqrt(mean h^2 + eps))."""
    h = x
    if residual is not None or t > 0:
        h = x.float()
        if t > 0:
            h = drop_ref(h, t, seed, offset)
        if residual is not None:
            h = h + residual.float()
        h = h.to(x.dtype)
    f = h.float()
    return h, f, torch.rsqrt(f.square().mean(-1, keepdim=True) + eps)


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, eps, t, seed, offset):
        h, f, inv = _rms_parts(x, residual, eps, t, seed, offset)
        y = f * inv
        if weight is not None:
            y = y * weight.float()
        ctx.save_for_backward(h, inv, weight)
        ctx.drop = (t, seed, offset)
        ctx.res = residual is not None
        y = y.to(x.dtype)
        return (y, h) if residual is not None else y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dh=None):
        h, inv, weight = ctx.saved_tensors
        t, seed, offset = ctx.drop
        f, a = h.float(), dy.float()
        dw = None
        if weight is not None:
            dw = (a * f * inv).reshape(-1, f.shape[-1]).sum(0).to(weight.dtype)
            a = a * weight.float()
        g = inv * (a - f * inv.square() * (a * f).mean(-1, keepdim=True))
        if dh is not None:
            g = g + dh.float()
        dx = drop_ref(g, t, seed, offset) if t > 0 else g
        return dx.to(h.dtype), g.to(h.dtype) if ctx.res else None, dw, None, None, None, None


def rms_norm_ref(x, weight, eps, residual, t, seed, offset):
    """y, or (y, h): h = residual + drop(x), y = h / sqrt(mean h^2 + eps) * weight; float32 sums, one rounding each."""
    return _RmsNorm.apply(x, residual, weight, eps, t, seed, offset)


def rms_norm_fp8_ref(x, weight, eps, residual):
    """(Fp8Blocks of the float32 norm, h)."""
    h, f, inv = _rms_parts(x, residual, eps, 0, 0, 0)
    y = f * inv
    if weight is not None:
        y = y * weight.float()
    return quantize_rows_ref(y.reshape(-1, x.shape[-1])), h
