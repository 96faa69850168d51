"""Inception-E's double 3x3 branch, heads merged and not, under any choice of convolution kernels, against 64 bits.

Two correct runs may differ by far more than a rounding here.  The per-shape tuner picks kernels by timing; another tile
adds the batch norm's statistics in another order, an activation tips to its bf16 neighbour, and an element whose
pre-activation lies within a rounding of zero changes sides of the ReLU: the block's weight gradient then moves by that
element's whole share (12 % of its largest entry where g is near 1 and 100 pixels are summed).  So each run is compared
with its own mask, and the mask with 64 bits where it is not decided by a rounding."""
import random

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu
HALF = 2.0**-8  # bf16: half a step relative to the value


def _block():
    from pytorch_imageclassification_distributed_amd.models import inception as inc
    torch.manual_seed(0)
    blk = inc.InceptionE(256).to("cuda").to(memory_format=torch.channels_last).train()
    with torch.no_grad():
        for m in blk.modules():
            if isinstance(m, torch.nn.BatchNorm2d):
                m.weight.uniform_(0.5, 1.5)
                m.bias.uniform_(-0.5, 0.5)
                m.running_mean.uniform_(-0.2, 0.2)
    x = torch.randn(4, 256, 5, 5, device="cuda").to(torch.bfloat16).contiguous(memory_format=torch.channels_last)
    return blk, x


@pytest.mark.parametrize("merged", [False, True])
@pytest.mark.parametrize("choice", [None, 0, 5, 7])
def test_double_3x3_branch_against_64_bits(merged, choice, monkeypatch):
    from pytorch_imageclassification_distributed_amd.ops import hip
    from pytorch_imageclassification_distributed_amd.ops._hip import gemm
    monkeypatch.setattr(gemm, "_STAGES_TUNED", {})
    monkeypatch.setattr(gemm, "_WGRAD_TUNED", {})
    if choice is not None:  # any admissible kernel for each shape, in place of the fastest
        rng = random.Random(choice)
        monkeypatch.setattr(gemm, "_time_ms", lambda run, reps=3, trials=3: (run(), rng.random())[1])
    blk, x = _block()
    seen = {}
    blk.branch3x3dbl_2.register_forward_hook(lambda m, i, o: seen.__setitem__("bd", o.detach().double().cpu()))
    keep, hip.SIBLINGS = hip.SIBLINGS, merged
    try:
        out = blk(x.clone().requires_grad_(True))
        g = torch.linspace(-1, 1, out.numel(), device="cuda").view_as(out)
        (out.float() * g).sum().backward()
    finally:
        hip.SIBLINGS = keep
    for name, first, pad in (("branch3x3dbl_3a", 1088, (0, 1)), ("branch3x3dbl_3b", 1472, (1, 0))):
        mod = getattr(blk, name)
        bd, w = seen["bd"], mod.conv.weight.detach().to(torch.bfloat16).double().cpu()
        gamma, beta = (p.detach().double().cpu().view(1, -1, 1, 1) for p in (mod.bn.weight, mod.bn.bias))
        o = out[:, first:first + 384].detach().double().cpu()
        dz = g[:, first:first + 384].to(torch.bfloat16).double().cpu()

        def mean(v):
            return v.mean((0, 2, 3), keepdim=True)
        y = F.conv2d(bd, w, padding=pad)
        mu, inv = mean(y), 1 / torch.sqrt(y.var((0, 2, 3), unbiased=False, keepdim=True) + mod.bn.eps)
        xh = (y - mu) * inv
        z = xh * gamma + beta
        # y is stored in bf16: it, the mean and the deviation are off by at most
        ey = HALF * (y.abs() + mean(y.abs()))
        einv = inv.square() * mean((y - mu).abs() * ey)  # relative
        ex = inv * ey + einv * xh.abs()
        near = gamma.abs() * ex + 1e-4 * z.abs()
        mask = o > 0
        assert bool(((mask == (z > 0)) | (z.abs() <= near)).all()), name
        d = dz * mask * gamma
        m2 = mean(d * xh)
        dy = inv * (d - mean(d) - xh * m2)
        tol = HALF * dy.abs() + einv * dy.abs() + inv * (ex * m2.abs() + xh.abs() * mean(d.abs() * ex))
        ref = torch.nn.grad.conv2d_weight(bd, w.shape, dy, padding=pad)
        lim = torch.nn.grad.conv2d_weight(bd.abs(), w.shape, tol * (1 + HALF) + 1e-5 * dy.abs(), padding=pad)
        over = (mod.conv.weight.grad.double().cpu() - ref).abs() - lim
        assert float(over.max()) <= 0, (name, float(over.max()))
