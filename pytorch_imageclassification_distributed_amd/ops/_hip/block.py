"""Counter-based dropout, root-mean-square norm with the residual's addition and 8-bit linear layers (HIP kernels
``csrc/block_ops.hip``, ``csrc/fp8_gemm.hip``).

No kernel here adds with atomics, no workspace outlives its call and nothing is read back on the host, so calls may run
on any stream, at once, and inside a captured graph.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from ..fp8_blocks import BLOCK, E4M3, Fp8Blocks, padded_cols, scale_cols
from ..grad_arena import grad_buffer
from .common import ACT, BF16, C, ws


def _dense16(t):
    """``t`` row-major and 16-byte aligned (the kernels move whole 16-byte vectors); a copy where it is not."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _f32(w):
    return None if w is None else _dense16(w.detach().float())


def _empty_blocks(rows, cols, tile, dev):
    return (torch.empty((rows, padded_cols(cols)), dtype=E4M3, device=dev),
            torch.empty((-(-rows // tile), scale_cols(cols)), dtype=torch.uint8, device=dev))


def _param_grad(p, g):
    """A float32 gradient in the parameter's own type."""
    return g if p.dtype == torch.float32 else g.to(p.dtype)


def _grad_out(p):
    """Where the float32 gradient of ``p`` goes: its arena slot / a tensor like it, row-major and dense."""
    if p.dtype == torch.float32 and p.is_contiguous():
        return grad_buffer(p, zero=False)
    return torch.empty(p.shape, dtype=torch.float32, device=p.device)


# ---------------------------------------------------------------------------
# dropout
# ---------------------------------------------------------------------------
def _drop_state(dev, seed, offset):
    """(device tensor [seed, offset] or None, seed, offset).  ``seed`` None: drawn from the device generator, on the
    device (``torch.manual_seed`` reproduces it, and a captured graph draws anew at every replay)."""
    if seed is None:
        return torch.randint(0, 2**63 - 1, (2,), device=dev, dtype=torch.int64), 0, 0
    if torch.is_tensor(seed):
        return seed, 0, 0
    return None, seed, offset


class DropoutCounterFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, t, state, seed, offset):
        x = _dense16(x)
        y = torch.empty_like(x)
        C.dropout_counter(x, None if residual is None else _dense16(residual), y, state, seed, offset, t)
        ctx.save_for_backward(state)
        ctx.args = (t, seed, offset)
        ctx.res = residual is not None
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        (state,) = ctx.saved_tensors
        t, seed, offset = ctx.args
        dx = None
        if ctx.needs_input_grad[0]:
            g16 = _dense16(g)
            dx = torch.empty_like(g16)
            C.dropout_counter(g16, None, dx, state, seed, offset, t)
        return dx, g if ctx.res else None, None, None, None, None


def dropout_counter(x, residual, t, seed, offset):
    return DropoutCounterFn.apply(x, residual, t, *_drop_state(x.device, seed, offset))


# ---------------------------------------------------------------------------
# root-mean-square norm
# ---------------------------------------------------------------------------
class RmsNormFn(torch.autograd.Function):
    """y (and h): h = residual + drop(x), y = h * rsqrt(mean h^2 + eps) * weight, one pass over x and residual; h and
    one float a row are kept for the backward pass, which makes the dropout mask again."""

    @staticmethod
    def forward(ctx, x, residual, weight, eps, t, state, seed, offset, need):
        n = x.shape[-1]
        rows = x.numel() // n
        x = _dense16(x)
        keep_h = residual is not None or (t > 0 and need)
        h = torch.empty_like(x) if keep_h else None
        y = torch.empty_like(x)
        rstd = torch.empty(rows, dtype=torch.float32, device=x.device) if need else None
        w = _f32(weight)
        C.rms_fwd(x, None if residual is None else _dense16(residual), w, h, y, rstd, rows, n, eps, state, seed, offset, t)
        ctx.set_materialize_grads(False)
        if need:
            ctx.save_for_backward(x if h is None else h, w, rstd, state)
            ctx.args = (rows, n, t, seed, offset)
            ctx.weight = weight
            ctx.res = residual is not None
        return (y, h) if residual is not None else y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dh=None):
        h, w, rstd, state = ctx.saved_tensors
        rows, n, t, seed, offset = ctx.args
        dev = h.device
        dy = torch.zeros_like(h) if dy is None else _dense16(dy)
        dh = None if dh is None else _dense16(dh)
        nx, nr, nw = ctx.needs_input_grad[:3]
        both = nx or not nr
        dx = torch.empty_like(h) if both else None
        dres = torch.empty_like(h) if nr and (t > 0 or not both) else None
        part = None
        if nw:
            part = torch.empty((C.rms_bwd_blocks(rows, n), n), dtype=torch.float32, device=dev)
        C.rms_bwd(dy, h, dh, w, rstd, dx, dres, part, rows, n, state, seed, offset, t)
        dw = None
        if nw:
            dw = _grad_out(ctx.weight)
            C.rows_sum(part, dw, part.shape[0] if rows else 0, n)
            dw = _param_grad(ctx.weight, dw)
        return (dx if nx else None, (dx if dres is None else dres) if nr else None, dw,
                None, None, None, None, None, None)


def rms_norm(x, weight, eps, residual, t, seed, offset):
    state, seed, offset = _drop_state(x.device, seed, offset) if t > 0 else (None, 0, 0)
    need = torch.is_grad_enabled() and any(v is not None and v.requires_grad for v in (x, residual, weight))
    return RmsNormFn.apply(x, residual, weight, eps, t, state, seed, offset, need)


def rms_norm_fp8(x, weight, eps, residual):
    n = x.shape[-1]
    rows = x.numel() // n
    x = _dense16(x.detach())
    h = torch.empty_like(x) if residual is not None else None
    q, sc = _empty_blocks(rows, n, 1, x.device)
    C.rms_fwd_fp8(x, None if residual is None else _dense16(residual.detach()), _f32(weight), h, q, sc, rows, n, eps)
    out = Fp8Blocks(q, sc, (rows, n), 1)
    return out if residual is None else (out, h)


# ---------------------------------------------------------------------------
# 8-bit products
# ---------------------------------------------------------------------------
def quantize_fp8(x2):
    x2 = _dense16(x2.detach())
    m, n = x2.shape
    q, sc = _empty_blocks(m, n, 1, x2.device)
    C.quant_rows(x2, None, q, sc, None, None, m, n)
    return Fp8Blocks(q, sc, (m, n), 1)


def quantize_fp8_weight(w):
    w = _dense16(w.detach())
    q, sc = _empty_blocks(w.shape[0], w.shape[1], BLOCK, w.device)
    C.quant_tiles(w, q, sc, None, None)
    return Fp8Blocks(q, sc, w.shape, BLOCK)


def fp8_dequantize(b, dtype):
    y = torch.empty(b.shape, dtype=dtype, device=b.device)
    C.fp8_dequant(b.q, b.scale, y, b.tile)
    return y


def _gemm8(a, asc, b, bsc, m, n, k, btile, dtype, bias=None, act=0):
    y = torch.empty((m, n), dtype=dtype, device=a.device)
    C.fp8_gemm(a, asc, b, bsc, y, bias, k, btile, act)
    return y


def matmul_fp8(a, b, bias, act, out_dtype):
    (m, k), n = a.shape, b.shape[0]
    return _gemm8(a.q, a.scale, b.q, b.scale, m, n, k, b.tile, out_dtype, _f32(bias), ACT[act])


def _bf16_rows_grad(dy, x, dw, m, n, k):
    """dw[n][k] = sum over the m rows of dy[row][n] x[row][k] on the framework's bf16 weight-gradient kernels (the rows
    are the pixels of a 1x1 convolution over 1x1 maps)."""
    n8, k8 = dy.shape[1], x.shape[1]
    out = dw if (n8, k8) == (n, k) else torch.empty((n8, k8), dtype=torch.float32, device=dy.device)
    out.zero_()
    if m > 0:
        stages = 7 if n8 >= 256 and k8 >= 256 else 2
        side = 256 if stages == 7 else 128
        tiles = -(-n8 // (side if n8 > 64 else 64)) * -(-k8 // side)
        splits = max(1, min(8, 512 // tiles, m // 512))  # at most 8 slabs: they are added in one ordered pass
        kps = -(-(-(-m // splits)) // 64) * 64
        splits = -(-m // kps)
        slabs = torch.empty(splits * n8 * k8, dtype=torch.float32, device=dy.device) if splits > 1 else None
        C.conv_wgrad(dy, x, out, m, n8, k8, k8, 1, 1, 1, 1, 1, 1, 0, 0, 1, 1, 1, kps, splits, ws(dy.device).zero, stages,
                     slabs, 0, xa_y=None, xa_coef=None, xf_coef=None, xf_act=0)
    if out is not dw:
        dw.copy_(out[:n, :k])


class LinearFp8Fn(torch.autograd.Function):
    """y = act(q(x) q(w)^T + b).  Backward: dx = q(dy) q(w) in 8 bits (the weights' transpose was written beside them,
    128 x 128 tiles keep their scale), db in float32, and dw = dy^T x on bf16 operands: weight gradients are summed into
    float32 masters over many steps, and the 8-bit matrix instructions cut their sums at 2^-16 where the bf16 ones keep
    float32."""

    @staticmethod
    def forward(ctx, x, weight, bias, act, need_x, need_w):
        x = _dense16(x)
        m, k = x.shape
        n = weight.shape[0]
        dev = x.device
        q, sc = _empty_blocks(m, k, 1, dev)
        copy = None
        if need_w and (x.dtype != BF16 or k % 8):
            copy = torch.empty((m, -(-k // 8) * 8), dtype=BF16, device=dev)
        C.quant_rows(x, None, q, sc, copy, None, m, k)
        wq, wsc = _empty_blocks(n, k, BLOCK, dev)
        wt, wtsc = _empty_blocks(k, n, BLOCK, dev) if need_x else (None, None)
        C.quant_tiles(_dense16(weight), wq, wsc, wt, wtsc)
        y = _gemm8(q, sc, wq, wsc, m, n, k, BLOCK, x.dtype, _f32(bias), ACT[act])
        if need_x or need_w or (bias is not None and bias.requires_grad):
            ctx.save_for_backward((x if copy is None else copy) if need_w else None, wt, wtsc, y if act == "relu" else None)
            ctx.params = (weight, bias)
            ctx.geo = (m, n, k)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        xb, wt, wtsc, y = ctx.saved_tensors
        m, n, k = ctx.geo
        weight, bias = ctx.params
        dy = _dense16(dy)
        dev = dy.device
        nx, nw, nb = ctx.needs_input_grad[:3]
        q = sc = copy = part = dx = dw = db = None
        if nx:
            q, sc = _empty_blocks(m, n, 1, dev)
        if nw and (dy.dtype != BF16 or n % 8 or y is not None):
            copy = torch.empty((m, -(-n // 8) * 8), dtype=BF16, device=dev)
        if nb:
            part = torch.empty((C.quant_rows_groups(m, n), n), dtype=torch.float32, device=dev)
        if q is not None or copy is not None or part is not None:
            C.quant_rows(dy, y, q, sc, copy, part, m, n)
        if nx:
            dx = _gemm8(q, sc, wt, wtsc, m, k, n, BLOCK, dy.dtype)
        if nw:
            dw = _grad_out(weight)
            _bf16_rows_grad(dy if copy is None else copy, xb, dw, m, n, k)
            dw = _param_grad(weight, dw)
        if nb:
            db = _grad_out(bias)
            C.rows_sum(part, db, part.shape[0], n)
            db = _param_grad(bias, db)
        return dx, dw, db, None, None, None


def linear_fp8(x2, weight, bias, act):
    grad = torch.is_grad_enabled()
    return LinearFp8Fn.apply(x2, weight, bias, act, grad and x2.requires_grad, grad and weight.requires_grad)


# names this part owns (ops/hip.py re-exports them)
_OWNED = (
    'DropoutCounterFn', 'LinearFp8Fn', 'RmsNormFn', '_bf16_rows_grad', '_dense16', '_drop_state', '_empty_blocks',
    '_f32', '_gemm8', '_grad_out', '_param_grad', 'dropout_counter', 'fp8_dequantize', 'linear_fp8', 'matmul_fp8',
    'quantize_fp8', 'quantize_fp8_weight', 'rms_norm', 'rms_norm_fp8',
)
