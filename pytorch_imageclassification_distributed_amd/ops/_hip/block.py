"""Counter-based dropout, root-mean-square norm with the residual's addition and 8-bit linear layers (HIP kernels
``csrc/block_ops.hip``, ``csrc/fp8_gemm.hip``, ``csrc/rows_grad.hip``; autograd nodes and allocation in ``csrc/block_bindings.cpp``).

No kernel here adds with atomics, no workspace outlives its call and nothing is read back on the host,
so calls may run on any stream, at once, and inside a captured graph.
"""
from __future__ import annotations

import functools
import operator

import torch

from ..fp8_blocks import BLOCK, Fp8Blocks
from ..grad_arena import grad_buffer
from .common import ACT, C


def _drop_state(dev, seed, offset):
    """(device tensor [seed, offset] or None, seed, offset).  ``seed`` None: drawn from the device generator, on the
    device (``torch.manual_seed`` reproduces it, and a captured graph draws anew at every replay)."""
    if seed is None:
        return torch.randint(0, 2**63 - 1, (2,), device=dev, dtype=torch.int64), 0, 0
    if torch.is_tensor(seed):
        return seed, 0, 0
    return None, operator.index(seed), operator.index(offset)


def _slot(p):
    """What hands out the tensor for ``p``'s float32 gradient, where ``p`` is in a gradient arena."""
    if p is None or "_imgcls_arena" not in p.__dict__ or p.dtype != torch.float32 or not p.is_contiguous():
        return None
    return functools.partial(grad_buffer, p, False)


def dropout_counter(x, residual, t, seed, offset):
    state, seed, offset = _drop_state(x.device, seed, offset)
    return C.dropout_counter(x, residual, state, seed, offset, t)


def rms_norm(x, weight, eps, residual, t, seed, offset):
    state, seed, offset = _drop_state(x.device, seed, offset) if t > 0 else (None, 0, 0)
    out = C.rms_norm(x, residual, weight, state, seed, offset, t, eps, _slot(weight))
    return out[0] if residual is None else (out[0], out[1])


def rms_norm_fp8(x, weight, eps, residual):
    n = x.shape[-1]
    q, sc, h = C.rms_norm_fp8(x, residual, weight, eps)
    out = Fp8Blocks._made(q, sc, (q.shape[0], n), 1)
    return out if residual is None else (out, h)


def quantize_fp8(x2):
    return Fp8Blocks._made(*C.quantize_fp8_rows(x2), tuple(x2.shape), 1)


def quantize_fp8_weight(w):
    return Fp8Blocks._made(*C.quantize_fp8_tiles(w), tuple(w.shape), BLOCK)


def fp8_dequantize(b, dtype):
    y = torch.empty(b.shape, dtype=dtype, device=b.device)
    C.dequantize_fp8(b.q, b.scale, y, b.tile)
    return y


def matmul_fp8(a, b, bias, act, out_dtype):
    return C.matmul_fp8(a.q, a.scale, b.q, b.scale, bias, b.shape[0], a.shape[1], b.tile, ACT[act], out_dtype)


def linear_fp8(x2, weight, bias, act):
    return C.linear_fp8(x2, weight, bias, ACT[act], _slot(weight), _slot(bias))


# names this part owns (ops/hip.py re-exports them)
_OWNED = (
    '_drop_state', '_slot', 'dropout_counter', 'fp8_dequantize', 'linear_fp8', 'matmul_fp8', 'quantize_fp8',
    'quantize_fp8_weight', 'rms_norm', 'rms_norm_fp8',
)
