"""Functional op layer the model zoo is written against.

Every model in ``models/`` expresses its forward pass with the handful of
primitives below (``conv_bn_act``, pooling, ``linear``, ``mlp``, ``se_gate``,
``drop_connect`` ...).  Each primitive has exactly two implementations:

* the **HIP path** (``ops/hip.py``): hand-written gfx950 kernels from
  ``csrc/*.hip`` operating on channels-last (NHWC) bf16 activations with fp32
  statistics/master weights.  Used for every CUDA (=HIP) tensor.
* the **reference path**: plain ATen ops in the module's own dtype.  Used on
  CPU (the unit-test oracle) and, when explicitly requested
  with ``set_backend('torch')``, on the GPU to measure the reference stack
  (PyTorch DDP + SyncBatchNorm + MIOpen) on the same box.

This mirrors what the reference computes implicitly through torchvision /
efficientnet_pytorch modules (reference nn/classifier.py:11-37) but lets the
GPU path fuse conv -> BN -> (+residual) -> activation.
"""
from __future__ import annotations

import math
import operator
import os

import torch
import torch.nn.functional as F
from torch.autograd import forward_ad

from .fp8_blocks import (FLOATS, Fp8Blocks, dequantize_ref, drop_ref, drop_threshold, linear_fp8_ref, quantize_rows_ref,
                         quantize_tiles_ref, rms_norm_fp8_ref, rms_norm_ref)

_BACKEND = os.environ.get("IMGCLS_BACKEND", "auto")  # auto | hip | torch


def set_backend(name: str) -> None:
    global _BACKEND
    if name not in ("auto", "hip", "torch"):
        raise ValueError(f"unknown backend {name!r}")
    _BACKEND = name


def get_backend() -> str:
    return _BACKEND


def use_hip(x: torch.Tensor) -> bool:
    """HIP kernels run for every GPU tensor unless the torch backend is forced."""
    if not x.is_cuda:
        if _BACKEND == "hip":
            raise RuntimeError("backend 'hip' requested for a CPU tensor")
        return False
    return _BACKEND != "torch"


_HIP = None


def _hip():
    global _HIP
    if _HIP is None:
        from . import hip  # noqa: WPS433  (lazy: loads the native extension)
        _HIP = hip
    return _HIP


# ---------------------------------------------------------------------------
# padding helpers
# ---------------------------------------------------------------------------
def conv_padding(conv, h: int, w: int):
    """Return (pad_top, pad_bottom, pad_left, pad_right) for ``conv``.

    ``conv.tf_same`` (set by the EfficientNet builder) selects TensorFlow
    "SAME" padding computed from the actual input size, as efficientnet_pytorch's
    Conv2dStaticSamePadding does for its configured image size.
    """
    kh, kw = conv.kernel_size
    sh, sw = conv.stride
    dh, dw = conv.dilation
    if getattr(conv, "tf_same", False):
        oh, ow = math.ceil(h / sh), math.ceil(w / sw)
        ph = max((oh - 1) * sh + (kh - 1) * dh + 1 - h, 0)
        pw = max((ow - 1) * sw + (kw - 1) * dw + 1 - w, 0)
        return ph // 2, ph - ph // 2, pw // 2, pw - pw // 2
    ph, pw = conv.padding
    return ph, ph, pw, pw


def _torch_conv(x, conv):
    pt, pb, pl, pr = conv_padding(conv, x.shape[-2], x.shape[-1])
    if (pt, pl) != (pb, pr):
        x = F.pad(x, (pl, pr, pt, pb))
        return F.conv2d(x, conv.weight, conv.bias, conv.stride, 0, conv.dilation, conv.groups)
    return F.conv2d(x, conv.weight, conv.bias, conv.stride, (pt, pl), conv.dilation, conv.groups)


def _act(x, act):
    if act is None:
        return x
    if act == "relu":
        return F.relu(x)
    if act == "silu":
        return F.silu(x)
    raise ValueError(act)


def _torch_bn(x, bn):
    sync = getattr(bn, "sync_group", None)
    if sync is not None and bn.training:
        from ..parallel.syncbn import sync_batch_norm
        return sync_batch_norm(x, bn, sync)
    return bn(x)


# ---------------------------------------------------------------------------
# primitives
# ---------------------------------------------------------------------------
def grad_slot(x, n: int = 2):
    """A gradient slot for a tensor with exactly ``n`` consumers that each take ``slot=`` (HIP path;
    None otherwise): their backward contributions are summed inside the consumers' own kernels."""
    if use_hip(x) and x.requires_grad and torch.is_grad_enabled():
        return _hip().GradSlot(n)
    return None


def conv_bn_act(x, conv, bn, act="relu", residual=None, x_slot=None, res_slot=None, exclusive_input=False,
                out=None, pool=None, prepool=None, defer_act=False, defer_res=False):
    """act(bn(conv(x)) [+ residual]).

    Reference equivalents: torchvision ``BasicConv2d`` (conv -> BN -> ReLU),
    ResNet ``Bottleneck``/``BasicBlock`` tails (BN -> +identity -> ReLU) and
    efficientnet_pytorch ``MBConvBlock`` (conv -> BN -> swish).
    ``pool`` = (kernel, stride, padding): a max pool follows the activation (the ResNet / Inception
    stems); the HIP path fuses it into the BN passes.
    ``prepool`` = (kernel, stride, padding): an average pool (count_include_pad) precedes the conv (the
    Inception ``branch_pool``); for a 1x1 conv the HIP path runs the conv first and pools its narrower
    output - both are linear, so conv1x1(avgpool(x)) == avgpool(conv1x1(x)).
    ``defer_act``: the caller feeds the result only to the next ``conv_bn_act`` (as its exclusive input);
    the HIP path may then skip writing act(bn(y)) and let that conv apply the BN on its operand loads.
    ``defer_res``: the result (no activation) is used only as the ``residual`` of one later ``conv_bn_act``
    (a ResNet downsample branch); the HIP path then skips writing bn(y) and that BN applies it on its loads.
    """
    if prepool is not None:
        if residual is not None or pool is not None:
            raise ValueError("conv_bn_act(prepool=...) takes a plain avgpool -> conv -> BN -> act")
        if use_hip(x):
            return _hip().pool_conv_bn_act(x, conv, bn, act, prepool, x_slot,
                                           (out[0].hip(), out[1]) if (out is not None and _hip().CONCAT_INPLACE)
                                           else None, out)
        x = F.avg_pool2d(x, *prepool)
    if pool is not None:  # stem: max_pool2d(act(bn(conv(x))), *pool) - kernel, stride, padding
        if residual is not None or x_slot is not None or out is not None:
            raise ValueError("conv_bn_act(pool=...) takes a plain conv -> BN -> act")
        if use_hip(x):
            return _hip().conv_bn_act_pool(x, conv, bn, act, pool, exclusive_input)
        return F.max_pool2d(_act(_torch_bn(_torch_conv(x, conv), bn), act), *pool)
    if use_hip(x):
        hout = (out[0].hip(), out[1]) if (out is not None and _hip().CONCAT_INPLACE) else None
        return _hip().conv_bn_act(x, conv, bn, act, residual, x_slot, res_slot, exclusive_input, hout,
                                  defer_act=defer_act, defer_res=defer_res)
    y = _torch_bn(_torch_conv(x, conv), bn)
    if residual is not None:
        y = y + residual
    return _act(y, act)


def siblings_ok(x, pairs) -> bool:
    """The HIP path can run these (conv, bn) pairs - 1x1 convs of the same ``x`` - as one GEMM
    (``conv_bn_act_siblings``); the caller then gives ``x`` one gradient-slot consumer for all of them."""
    return use_hip(x) and _hip().siblings_eligible(x, pairs)


def conv_bn_act_siblings(x, pairs, outs, act="relu", x_slot=None):
    """[act(bn(conv(x))) for (conv, bn) in pairs] as one concatenated-output GEMM (HIP path, ``siblings_ok``);
    ``outs[i]`` = (ConcatPlan, branch) writes that result into the concat output in place."""
    h = _hip()
    hout = [(o[0].hip(), o[1]) if (o is not None and h.CONCAT_INPLACE) else None for o in outs]
    res = h.conv_bn_act_siblings(x, pairs, hout, act, x_slot)
    return res


def conv(x, conv_mod):
    """Plain convolution (with optional bias), no normalisation."""
    if use_hip(x):
        return _hip().conv(x, conv_mod)
    return _torch_conv(x, conv_mod)


def max_pool2d(x, kernel_size, stride, padding=0, slot=None):
    if use_hip(x):
        return _hip().max_pool2d(x, kernel_size, stride, padding, slot)
    return F.max_pool2d(x, kernel_size, stride, padding)


def avg_pool2d(x, kernel_size, stride, padding=0, slot=None):
    """count_include_pad=True semantics (torch default, used by torchvision Inception)."""
    if use_hip(x):
        return _hip().avg_pool2d(x, kernel_size, stride, padding, slot)
    return F.avg_pool2d(x, kernel_size, stride, padding)


def global_avg_pool(x):
    """adaptive_avg_pool2d(x, 1) + flatten -> [N, C]."""
    if use_hip(x):
        return _hip().global_avg_pool(x)
    return torch.flatten(F.adaptive_avg_pool2d(x, 1), 1)


def linear(x, lin, act=None):
    if use_hip(x):
        return _hip().linear(x, lin, act)
    return _act(F.linear(x, lin.weight, lin.bias), act)


def mlp(x, seq):
    """The reference classifier head: Linear/ReLU stack (nn/classifier.py:26-34)."""
    if use_hip(x):
        return _hip().mlp(x, seq)
    return seq(x)


def dropout(x, p, training):
    if p == 0.0 or not training:
        return x
    if use_hip(x):
        return _hip().dropout(x, p)
    return F.dropout(x, p, True)


# ---------------------------------------------------------------------------
# pre-norm 8-bit linear block: counter-based dropout, root-mean-square norm, 8-bit products
# ---------------------------------------------------------------------------
def _check_floats(name, x):
    if x.dtype not in FLOATS:
        raise TypeError(f"{name}: x is {x.dtype}, expected bfloat16, float16 or float32")


def _check_like(name, what, t, x):
    if t is not None and (t.shape != x.shape or t.dtype != x.dtype or t.device != x.device):
        raise ValueError(f"{name}: {what} must match x ({x.dtype} {tuple(x.shape)} on {x.device}), "
                         f"got {t.dtype} {tuple(t.shape)} on {t.device}")


def _check_drop(name, x, p, seed, offset):
    """The drop threshold of ``p``; refuses seeds the kernels cannot take."""
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"{name}: p must be in [0, 1], got {p}")
    if torch.is_tensor(seed):
        if seed.dtype != torch.int64 or tuple(seed.shape) != (2,) or seed.device != x.device or not seed.is_contiguous():
            raise ValueError(f"{name}: a seed tensor is int64 [seed, offset] on {x.device}")
        if offset != 0:
            raise ValueError(f"{name}: a seed tensor holds the offset itself")
    elif seed is None:
        if offset != 0:
            raise ValueError(f"{name}: offset without a seed")
    elif not (0 <= operator.index(seed) < 2**64 and 0 <= operator.index(offset) < 2**64):  # (TypeError: not an integer)
        raise ValueError(f"{name}: seed and offset are 64-bit unsigned, got {seed}, {offset}")
    return drop_threshold(p)


def _seed_values(seed, offset, device):
    """Host values for the reference path."""
    if seed is None:
        seed = torch.randint(0, 2**63 - 1, (2,), dtype=torch.int64, device=device)
    if torch.is_tensor(seed):
        seed, offset = (v % 2**64 for v in seed.tolist())
    return operator.index(seed), operator.index(offset)


def dropout_counter(x, p, training=True, seed=None, offset=0, residual=None):
    """``[residual +] dropout(x, p)`` whose mask is a function of (element index, ``seed``, ``offset``) and is never
    stored: the backward pass makes it again.  The sum is rounded once, to x's type.

    ``seed``: a 64-bit integer; or an int64 tensor ``[seed, offset]`` on x's device, read when the kernels run (a captured
    graph sees the values it holds at each replay; changing it between forward and backward is an error); or None, which
    draws both from the device's generator.  Every (seed, offset) pair is an independent mask over up to 2^67 elements.
    ``p`` is rounded to a multiple of 2^-16; the kept values are scaled by 1 / (1 - that).  Elements are numbered in
    row-major order whatever the strides; the result is row-major.  A dropped infinity or NaN leaves 0.  Differentiable
    once, in reverse mode (a forward-mode tangent is refused on the GPU).
    """
    _check_floats("dropout_counter", x)
    _check_like("dropout_counter", "residual", residual, x)
    t = _check_drop("dropout_counter", x, p, seed, offset)
    if not training or t == 0:
        if residual is None:
            return x
        return _hip().dropout_counter(x, residual, 0, 0, 0) if use_hip(x) else x + residual
    if use_hip(x):
        return _hip().dropout_counter(x, residual, t, seed, offset)
    y = drop_ref(x.contiguous().float(), t, *_seed_values(seed, offset, x.device))
    return (y if residual is None else y + residual.float()).to(x.dtype)


RMS_MAX_COLS = 32768  # widest row that the HIP kernels keep in registers (csrc/block_ops.hip)


def _norm_args(name, x, norm, residual):
    _check_floats(name, x)
    _check_like(name, "residual", residual, x)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"{name}: x needs a last dimension of at least 1, got {tuple(x.shape)}")
    n = x.shape[-1]
    if isinstance(norm, torch.nn.LayerNorm) or getattr(norm, "bias", None) is not None:
        raise TypeError(f"{name}: {type(norm).__name__} is no root-mean-square norm")
    w, eps = norm.weight, norm.eps
    if w is None:
        if tuple(norm.normalized_shape) != (n,):
            raise ValueError(f"{name}: the norm is over {tuple(norm.normalized_shape)}, x's rows have {n}")
    elif w.dim() != 1 or w.shape[0] != n or w.device != x.device or w.dtype not in FLOATS:
        raise ValueError(f"{name}: weight must be [{n}] on {x.device}, got {w.dtype} {tuple(w.shape)} on {w.device}")
    if n > RMS_MAX_COLS and use_hip(x):
        raise ValueError(f"{name}: rows of at most {RMS_MAX_COLS} columns, got {n}")
    return w, eps if eps is not None else torch.finfo(x.dtype).eps


def rms_norm(x, norm, residual=None, p=0.0, training=True, seed=None, offset=0):
    """Root-mean-square norm over the last dimension (``norm``: an ``nn.RMSNorm``), with the residual's addition and the
    dropout before it in the same pass: ``h = residual + dropout_counter(x, p)``, ``y = h / sqrt(mean(h^2) + eps) * weight``.

    Returns ``y``, or ``(y, h)`` with a ``residual`` (``h``, rounded to x's type, is the next layer's residual and what
    is normalised).  ``seed`` / ``offset`` as in ``dropout_counter``.  Sums and statistics are float32.
    """
    w, eps = _norm_args("rms_norm", x, norm, residual)
    t = _check_drop("rms_norm", x, p, seed, offset) if training else 0
    if use_hip(x):
        return _hip().rms_norm(x, w, eps, residual, t, seed, offset)
    return rms_norm_ref(x.contiguous(), w, eps, residual, t, *(_seed_values(seed, offset, x.device) if t else (0, 0)))


def rms_norm_fp8(x, norm, residual=None):
    """``rms_norm`` with an 8-bit result for ``matmul_fp8``: ``Fp8Blocks`` over the flattened rows (1 x 128 blocks,
    quantised from the float32 values), or ``(Fp8Blocks, h)`` with a ``residual``.

    For inference: it has no gradient and refuses inputs that ask for one (training: ``rms_norm``, then ``linear_fp8``)."""
    w, eps = _norm_args("rms_norm_fp8", x, norm, residual)
    _refuse_grad("rms_norm_fp8", x, residual, w)
    if use_hip(x):
        return _hip().rms_norm_fp8(x, w, eps, residual)
    out, h = rms_norm_fp8_ref(x.contiguous(), w, eps, residual)
    return out if residual is None else (out, h)


def _refuse_tangent(name, *tensors):
    if forward_ad._current_level >= 0 and forward_ad._is_fwd_grad_enabled() and any(
            t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"{name} has no forward-mode derivative, and an input carries a tangent")


def _refuse_grad(name, *tensors):
    _refuse_tangent(name, *tensors)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(f"{name} has no gradient: call it under torch.no_grad(), or train through linear_fp8")


def quantize_fp8(x):
    """Activations ``[..., K]`` -> ``Fp8Blocks`` over the flattened rows, one scale for each 1 x 128 block."""
    _check_floats("quantize_fp8", x)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"quantize_fp8: x needs a last dimension of at least 1, got {tuple(x.shape)}")
    _refuse_grad("quantize_fp8", x)
    x2 = x.reshape(-1, x.shape[-1])
    return _hip().quantize_fp8(x2) if use_hip(x) else quantize_rows_ref(x2)


def quantize_fp8_weight(w):
    """A weight ``[N, K]`` -> ``Fp8Blocks`` with one scale for each 128 x 128 tile (laid out once, for serving)."""
    _check_floats("quantize_fp8_weight", w)
    if w.dim() != 2 or w.shape[0] < 1 or w.shape[1] < 1:
        raise ValueError(f"quantize_fp8_weight: a weight is [N, K], got {tuple(w.shape)}")
    _refuse_tangent("quantize_fp8_weight", w)
    w = w.detach()
    return _hip().quantize_fp8_weight(w) if use_hip(w) else quantize_tiles_ref(w)


def matmul_fp8(a, b, bias=None, act=None, out_dtype=torch.bfloat16):
    """``act(a @ b.T + bias)`` of 8-bit blocks: a ``[M, K]`` with 1 x 128 blocks, b ``[N, K]`` with 1 x 128 blocks or
    128 x 128 tiles -> ``[M, N]`` in ``out_dtype``.  ``act``: None, 'relu' or 'silu'.

    Accumulators are float32, but the matrix instructions cut each product at 2^-13 of the largest of its 8 neighbours
    (columns 8i to 8i + 7; csrc/fp8_gemm.hip), whatever ``out_dtype`` is: 1.5e-5 of the result's norm on normal data, up
    to 2^-10 of sum |a||b| on normal values that are chosen for it, and not bounded relative to a result whose terms
    cancel.  For inference: no gradient (training: ``linear_fp8``)."""
    if a.tile != 1:
        raise ValueError("matmul_fp8: a needs 1 x 128 blocks (quantize_fp8, rms_norm_fp8)")
    if a.shape[1] != b.shape[1]:
        raise ValueError(f"matmul_fp8: inner sizes differ: {a.shape} and {b.shape}")
    if a.device != b.device:
        raise ValueError(f"matmul_fp8: a on {a.device}, b on {b.device}")
    if bias is not None and (tuple(bias.shape) != (b.shape[0],) or bias.device != a.device or bias.dtype not in FLOATS):
        raise ValueError(f"matmul_fp8: bias must be [{b.shape[0]}] on {a.device}")
    if act not in (None, "relu", "silu"):
        raise ValueError(f"matmul_fp8: act {act!r}")
    if out_dtype not in FLOATS:
        raise ValueError(f"matmul_fp8: out_dtype {out_dtype}")
    _refuse_grad("matmul_fp8", bias)
    if use_hip(a.q):
        return _hip().matmul_fp8(a, b, bias, act, out_dtype)
    y = dequantize_ref(a) @ dequantize_ref(b).t()
    return _act(y if bias is None else y + bias.float(), act).to(out_dtype)


def linear_fp8(x, lin, act=None):
    """``linear`` with an 8-bit forward and data gradient (``lin``: an ``nn.Linear`` with float32, bfloat16 or float16
    parameters; the weight is quantised at every call, so an optimiser may change it in between).

    ``y = act(q(x) q(w)^T + b)`` in x's type, 1 x 128 blocks for x and dy, 128 x 128 for w; ``dx = q(dy) q(w)``;
    ``dw = dy^T x`` on x and dy rounded to bfloat16 with float32 sums; ``db`` = float32 column sums.  ``act``: None or
    'relu' (whose gradient is masked before dy is quantised)."""
    _check_floats("linear_fp8", x)
    w, b = lin.weight, lin.bias
    if act not in (None, "relu"):
        raise NotImplementedError(act)
    if x.dim() < 1 or w.dim() != 2 or x.shape[-1] != w.shape[1]:
        raise ValueError(f"linear_fp8: x {tuple(x.shape)} does not fit weight {tuple(w.shape)}")
    if w.shape[0] < 1 or w.shape[1] < 1 or w.dtype not in FLOATS:
        raise ValueError(f"linear_fp8: weight {w.dtype} {tuple(w.shape)}")
    if b is not None and (b.dtype not in FLOATS or tuple(b.shape) != (w.shape[0],)):
        raise ValueError(f"linear_fp8: bias must be [{w.shape[0]}], got {b.dtype} {tuple(b.shape)}")
    if w.device != x.device or (b is not None and b.device != x.device):
        raise ValueError(f"linear_fp8: x on {x.device}, weight on {w.device}")
    x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])  # (a reshape or view is an autograd node more, 8 us a call)
    y = _hip().linear_fp8(x2, w, b, act) if use_hip(x) else linear_fp8_ref(x2, w, b, act)
    return y if x.dim() == 2 else y.view(*x.shape[:-1], w.shape[0])


class ConcatPlan:
    """A channel concat whose branches write their outputs in place: pass ``out=(plan, i)`` to the
    branch's final ``conv_bn_act`` and ``buf=plan`` to ``cat_channels`` (HIP path: ``hip.ConcatBuffer``;
    the reference path ignores the plan and concatenates with ``torch.cat``)."""

    def __init__(self, channels):
        self.channels = list(channels)
        self._hip = None

    def hip(self):
        if self._hip is None:
            self._hip = _hip().ConcatBuffer(self.channels)
        return self._hip


def concat_buffer(channels) -> ConcatPlan:
    return ConcatPlan(channels)


def cat_channels(xs, buf=None):
    if use_hip(xs[0]):
        h = _hip()
        return h.cat_channels(xs, buf.hip() if (buf is not None and h.CONCAT_INPLACE) else None)
    return torch.cat(xs, 1)


def add(x, y):
    if use_hip(x):
        return _hip().add(x, y)
    return x + y


def se_gate(x, se_reduce, se_expand, exclusive_input=False):
    """Squeeze-and-excitation: x * sigmoid(expand(swish(reduce(avgpool(x))))).  ``exclusive_input``: the gate
    is x's only consumer (HIP path: its backward runs the backward reduce of the BN that produced x)."""
    if use_hip(x):
        return _hip().se_gate(x, se_reduce, se_expand, exclusive_input)
    s = F.adaptive_avg_pool2d(x, 1)
    s = se_expand(F.silu(se_reduce(s)))
    return torch.sigmoid(s) * x


def drop_connect(x, p, training):
    """efficientnet_pytorch utils.drop_connect: per-sample stochastic depth."""
    if not training or p == 0.0:
        return x
    if use_hip(x):
        return _hip().drop_connect(x, p)
    keep = 1.0 - p
    mask = torch.floor(keep + torch.rand([x.shape[0], 1, 1, 1], dtype=x.dtype, device=x.device))
    return x / keep * mask


def cross_entropy(logits, labels, weight=None):
    """CrossEntropyLoss(weight) with mean reduction: sum_i w_yi*nll_i / sum_i w_yi
    (reference train.py:157-158)."""
    if use_hip(logits):
        return _hip().cross_entropy(logits, labels, weight)
    return F.cross_entropy(logits.float(), labels, weight=weight)


def prepare_input(x, stem=None):
    """Move/convert a batch to the layout the active path expects.

    HIP path: channels-last bf16 (NHWC in memory); with ``stem`` (a 7x7 stride-2 first conv) the
    fp32 batch may be left for the space-to-depth stem to convert.  Reference path: unchanged.
    """
    if use_hip(x):
        return _hip().prepare_input(x, stem=stem)
    return x
