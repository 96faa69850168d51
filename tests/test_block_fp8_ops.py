"""Counter-based dropout, root-mean-square norm with the residual's addition, and 8-bit products with block-128 scales
(ops/functional.py dropout_counter, rms_norm, rms_norm_fp8, quantize_fp8, matmul_fp8, linear_fp8).

Oracles are numpy / float64 and written here.  Tolerances count roundings: u = 2^-24 for a float32 operation, half =
finfo(T).eps / 2 for the one rounding to the output type; a float32 sum along a chain of n additions is off by at most
n u times the sum of the magnitudes.
"""
import math

import numpy as np
import pytest
import torch
import torch.nn as nn

from pytorch_imageclassification_distributed_amd.ops import functional as Fx
from pytorch_imageclassification_distributed_amd.ops import fp8_blocks as fb

U = 2.0**-24
TYPES = [torch.bfloat16, torch.float16, torch.float32]
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
gpu = pytest.mark.gpu


def half(t):
    return torch.finfo(t).eps / 2


def assert_within(got, ref, tol, what=""):
    """|got - ref| <= tol elementwise (float64 tensors on the CPU); names the worst place."""
    got, ref, tol = (torch.as_tensor(v).detach().double().cpu() for v in (got, ref, tol))
    over = (got - ref).abs() - tol.expand_as(ref)
    over = torch.where(got == ref, torch.full_like(over, -1.0), over)
    bad = ~(over <= 0)
    if bool(bad.any()):
        i = int(torch.nan_to_num(over, nan=math.inf).flatten().argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} out of tolerance; worst at flat {i}: got "
                             f"{got.flatten()[i].item()!r}, expected {ref.flatten()[i].item()!r}, "
                             f"tolerance {tol.expand_as(ref).flatten()[i].item()!r}")


def rand(shape, t, dev, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(t).to(dev)


# ---------------------------------------------------------------------------
# oracles
# ---------------------------------------------------------------------------
def philox_numbers(groups, seed, offset):
    """Philox4x32-10 in numpy uint64: the eight 16-bit numbers of each group."""
    m = np.uint64(0xFFFFFFFF)
    s = np.uint64(32)
    g = np.asarray(groups, dtype=np.uint64)
    c = [g & m, g >> s, np.full_like(g, offset & 0xFFFFFFFF), np.full_like(g, (offset >> 32) & 0xFFFFFFFF)]
    k = [seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF]
    for _ in range(10):
        p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(p1 >> s) ^ c[1] ^ np.uint64(k[0]), p1 & m, (p0 >> s) ^ c[3] ^ np.uint64(k[1]), p0 & m]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    out = np.empty((g.size, 8), np.int64)
    for j in range(4):
        out[:, 2 * j] = (c[j] & np.uint64(0xFFFF)).astype(np.int64)
        out[:, 2 * j + 1] = (c[j] >> np.uint64(16)).astype(np.int64)
    return out


def keep_oracle(shape, p, seed, offset):
    n = int(np.prod(shape))
    t = min(65536, int(math.floor(p * 65536 + 0.5)))
    keep = philox_numbers(np.arange(-(-n // 8)), seed, offset).reshape(-1)[:n] >= t
    return torch.from_numpy(keep).view(shape), (65536.0 / (65536 - t) if t < 65536 else 0.0)


def e4m3_grid():
    v = []
    for e in range(16):
        for m in range(8):
            if (e, m) != (15, 7):
                v.append((1 + m / 8) * 2.0 ** (e - 7) if e else m / 8 * 2.0**-6)
    return np.array(v)


def block_oracle(v, tile):
    """(values on the scaled e4m3 grid, exponents) of a float64 matrix: nearest, ties to the even significand, searched in
    the list of all e4m3 values."""
    grid = e4m3_grid()
    v = np.asarray(v, np.float64)
    out, exps = np.empty_like(v), np.empty((-(-v.shape[0] // tile), -(-v.shape[1] // 128)), np.int64)
    for i in range(exps.shape[0]):
        for k in range(exps.shape[1]):
            b = v[i * tile:(i + 1) * tile, k * 128:(k + 1) * 128]
            fin = np.abs(b[np.isfinite(b)])
            amax = fin.max() if fin.size else 0.0
            e = 0
            if amax > 0:
                e = -140
                while amax > 448 * 2.0**e:
                    e += 1
                e = max(e, -127)
            exps[i, k] = e
            u = np.abs(np.where(np.isfinite(b), b, 0)) * 2.0**-e
            hi = np.clip(np.searchsorted(grid, u), 1, len(grid) - 1)
            lo = hi - 1
            dl, dh = u - grid[lo], grid[hi] - u
            pick = np.where(dl < dh, lo, np.where(dl > dh, hi, np.where(lo % 2 == 0, lo, hi)))
            out[i * tile:(i + 1) * tile, k * 128:(k + 1) * 128] = np.where(
                np.isfinite(b), np.sign(b) * grid[pick] * 2.0**e, np.nan)
    return out, exps


def values_of(b):
    """Float64 values of Fp8Blocks, decoded here."""
    bits = b.q.view(torch.uint8).cpu().numpy().astype(np.int64)
    e, m = (bits >> 3) & 15, bits & 7
    v = np.where(e > 0, (1 + m / 8) * 2.0 ** (e - 7), m / 8 * 2.0**-6)
    v = np.where((bits & 127) == 127, np.nan, v) * np.where(bits >> 7, -1.0, 1.0)
    s = 2.0 ** (b.scale.cpu().numpy().astype(np.float64) - 127)
    s = s.repeat(b.tile, 0)[:b.shape[0], :b.q.shape[1] // 128].repeat(128, 1)
    return torch.from_numpy((v * s)[:, :b.shape[1]])


# ---------------------------------------------------------------------------
# dropout
# ---------------------------------------------------------------------------
def test_philox_known_answers():
    """The published test vectors of Philox4x32-10 (Random123 distribution, kat_vectors)."""
    def words(ctr, key):
        g = ctr[0] | ctr[1] << 32
        h = philox_numbers(np.array([g], np.uint64), key[0] | key[1] << 32, ctr[2] | ctr[3] << 32)[0]
        return [int(h[2 * j] | h[2 * j + 1] << 16) for j in range(4)]
    assert words([0, 0, 0, 0], [0, 0]) == [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]
    f = 0xffffffff
    assert words([f, f, f, f], [f, f]) == [0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd]
    assert words([0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344], [0xa4093822, 0x299f31d0]) == [
        0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("shape,p,res", [((1,), 0.5, False), ((7,), 0.3, True), ((4, 2048), 0.5, False),
                                         ((33, 1281), 0.1, True), ((3, 5, 64), 0.9, True), ((2, 3), 1.0, True),
                                         ((300, 1000), 1e-5, False), ((0, 8), 0.5, True)])
def test_dropout_counter(dev, t, shape, p, res):
    seed, offset = 0x9E3779B97F4A7C15, 0x1234567890
    x = rand(shape, t, dev, 1).requires_grad_(True)
    r = rand(shape, t, dev, 2, 3.0).requires_grad_(True) if res else None
    y = Fx.dropout_counter(x, p, seed=seed, offset=offset, residual=r)
    assert y.dtype == t and y.shape == x.shape
    keep, s = keep_oracle(shape, p, seed, offset)
    d = torch.where(keep, x.detach().double().cpu() * s, torch.zeros((), dtype=torch.float64))
    ref = d + (r.detach().double().cpu() if res else 0)
    # the scale, its product and the sum: three float32 roundings; one to T (subnormal steps: absolute)
    tol = half(t) * ref.abs() + 3 * U * (d.abs() + (ref - d).abs()) + torch.finfo(t).smallest_normal * torch.finfo(t).eps
    assert_within(y, ref, tol, "y")
    g = rand(shape, t, dev, 3)
    grads = torch.autograd.grad(y, (x, r) if res else (x,), g)
    dref = torch.where(keep, g.double().cpu() * s, torch.zeros((), dtype=torch.float64))
    assert_within(grads[0], dref, half(t) * dref.abs() + 3 * U * dref.abs() + torch.finfo(t).smallest_normal * torch.finfo(t).eps, "dx")
    if res:
        assert torch.equal(grads[1], g)


@pytest.mark.parametrize("dev", DEVICES)
def test_dropout_counter_orders_and_special_values(dev):
    """Elements are numbered row-major whatever the strides; a view that is not 16-byte aligned; dropped infinities."""
    base = rand((40, 66), torch.float16, dev, 4)
    for x in (base.t(), base[1:, 1:], base.flatten()[3:], base[:, ::2], base.view(2, 20, 11, 6).permute(0, 3, 1, 2)):
        y = Fx.dropout_counter(x, 0.5, seed=5)
        assert torch.equal(y, Fx.dropout_counter(x.contiguous().clone(), 0.5, seed=5))
        keep, _ = keep_oracle(tuple(x.shape), 0.5, 5, 0)
        assert torch.equal((y != 0).cpu() | (x == 0).cpu(), keep | (x == 0).cpu())
    x = torch.full((64,), float("inf"), device=dev)
    x[::3] = float("nan")
    y = Fx.dropout_counter(x, 0.5, seed=9, residual=torch.ones(64, device=dev)).cpu()
    keep, _ = keep_oracle((64,), 0.5, 9, 0)
    assert torch.equal(y[~keep], torch.ones(int((~keep).sum()))) and not bool(y[keep].isfinite().any())


@pytest.mark.parametrize("dev", DEVICES)
def test_dropout_counter_seeds(dev):
    x = torch.ones(4096, device=dev)
    a = Fx.dropout_counter(x, 0.5, seed=7, offset=3)
    assert torch.equal(a, Fx.dropout_counter(x, 0.5, seed=torch.tensor([7, 3], device=dev)))
    assert not torch.equal(a, Fx.dropout_counter(x, 0.5, seed=7, offset=4))
    assert not torch.equal(a, Fx.dropout_counter(x, 0.5, seed=8, offset=3))
    torch.manual_seed(0)
    b = Fx.dropout_counter(x, 0.5)
    c = Fx.dropout_counter(x, 0.5)
    torch.manual_seed(0)
    assert torch.equal(b, Fx.dropout_counter(x, 0.5)) and not torch.equal(b, c)
    assert Fx.dropout_counter(x, 0.5, training=False) is x
    r = torch.full_like(x, 2.0)
    assert torch.equal(Fx.dropout_counter(x, 0.5, training=False, residual=r), x + r)
    # the kept share: binomial, 6 standard deviations
    n = 1 << 20
    kept = float((Fx.dropout_counter(torch.ones(n, device=dev), 0.25, seed=1) != 0).double().mean())
    assert abs(kept - 0.75) < 6 * math.sqrt(0.25 * 0.75 / n)
    # a seed that changes between forward and backward is refused, not silently another mask
    if dev == "cuda":
        st = torch.tensor([7, 3], device=dev)
        xx = x.clone().requires_grad_(True)
        y = Fx.dropout_counter(xx, 0.5, seed=st)
        st.add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()


@gpu
def test_dropout_counter_past_32_bit_offsets():
    n = (1 << 31) + 77
    x = torch.ones(n, dtype=torch.bfloat16, device="cuda")
    y = Fx.dropout_counter(x, 0.5, seed=11)
    del x
    first = (n - 4096) // 8
    keep = philox_numbers(np.arange(first, -(-n // 8)), 11, 0).reshape(-1)[:n - first * 8] >= 32768
    assert torch.equal(y[first * 8:].cpu(), torch.from_numpy(keep).to(torch.bfloat16) * 2)
    assert torch.equal(y[:4096].cpu(), keep_oracle((4096,), 0.5, 11, 0)[0].to(torch.bfloat16) * 2)


@pytest.mark.parametrize("kw,err", [(dict(p=-0.1), ValueError), (dict(p=1.5), ValueError), (dict(p=float("nan")), ValueError),
                                    (dict(p=0.5, seed=-1), ValueError), (dict(p=0.5, seed=2**64), ValueError),
                                    (dict(p=0.5, seed=1, offset=2**64), ValueError), (dict(p=0.5, offset=1), ValueError),
                                    (dict(p=0.5, seed=torch.zeros(2)), ValueError),
                                    (dict(p=0.5, seed=torch.zeros(3, dtype=torch.int64)), ValueError),
                                    (dict(p=0.5, seed=torch.zeros(2, dtype=torch.int64), offset=1), ValueError),
                                    (dict(p=0.5, residual=torch.zeros(5)), ValueError),
                                    (dict(p=0.5, residual=torch.zeros(4, dtype=torch.float16)), ValueError)])
def test_dropout_counter_refuses(kw, err):
    with pytest.raises(err):
        Fx.dropout_counter(torch.zeros(4), **kw)
    with pytest.raises(TypeError):
        Fx.dropout_counter(torch.zeros(4, dtype=torch.int32), 0.5)


# ---------------------------------------------------------------------------
# root-mean-square norm
# ---------------------------------------------------------------------------
# additions on the longest float32 chain of a row: 8 a vector, at most 4 vectors a lane, 6 + 15 across lanes and waves;
# on the reference path torch's own row sum, at most the row's length (short rows here) in blocks of 128
CHAIN = 8 * 4 + 6 + 15


def norm_case(dev, t, rows, n, res, p, affine=True, seed=21):
    norm = nn.RMSNorm(n, eps=1e-6, elementwise_affine=affine)
    if affine:
        with torch.no_grad():
            norm.weight.copy_(rand((n,), torch.float32, "cpu", seed) * 0.3 + 1)
    norm = norm.to(dev)
    x = rand((rows, n), t, dev, seed + 1, 2.0).requires_grad_(True)
    r = rand((rows, n), t, dev, seed + 2).requires_grad_(True) if res else None
    return norm, x, r


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,n,res,p,affine", [(1, 1, True, 0.0, True), (3, 7, False, 0.0, True), (5, 512, True, 0.3, True),
                                                 (1, 2048, True, 0.0, True), (9, 1281, True, 0.25, True), (6, 1000, False, 0.5, False),
                                                 (7, 4096, False, 0.0, True), (3, 8192, True, 0.1, True), (2, 9001, True, 0.1, True),
                                                 (2, 16384, False, 0.0, True), (2, 32768, True, 0.2, True), (0, 64, True, 0.0, True),
                                                 (1500, 96, True, 0.1, True), (2100, 2560, True, 0.0, True)])
def test_rms_norm(dev, t, rows, n, res, p, affine):
    if dev == "cpu" and rows * n > 200000:
        pytest.skip("size of a kernel variant")
    norm, x, r = norm_case(dev, t, rows, n, res, p, affine)
    seed, offset = 1234567, 89
    out = Fx.rms_norm(x, norm, residual=r, p=p, seed=seed, offset=offset)
    y, h = out if res else (out, None)
    xd = x.detach().double().cpu()
    keep, s = keep_oracle((rows, n), p, seed, offset)
    hd = torch.where(keep, xd * s, torch.zeros((), dtype=torch.float64)) if p > 0 else xd
    if res:
        hd = hd + r.detach().double().cpu()
        mag = hd.abs() + 3 * (hd - r.detach().double().cpu()).abs() + r.detach().double().cpu().abs()
        assert h.dtype == t
        assert_within(h, hd, half(t) * hd.abs() + 3 * U * mag + torch.finfo(t).smallest_normal * torch.finfo(t).eps, "h")
        hd = h.detach().double().cpu()  # what is normalised
    elif p > 0:
        hd = hd.float().to(t).double()
    w = norm.weight.detach().double().cpu() if affine else torch.ones(n, dtype=torch.float64)
    inv = 1 / torch.sqrt(hd.square().mean(1, keepdim=True) + 1e-6)
    ref = hd * inv * w
    chain = CHAIN if dev == "cuda" else max(CHAIN, n)
    # half the chain's relative error in the root, then sqrt, reciprocal, division by n, eps, two products
    rel = (chain / 2 + 8) * U
    near = 1.0 + 2 * half(t)  # without a residual h itself is not returned: its float32 rounding may tip to a neighbour
    loose = 2 * half(t) if (not res and p > 0) else 0.0
    tiny = torch.finfo(t).smallest_normal * torch.finfo(t).eps
    assert_within(y, ref, (half(t) + rel + loose) * ref.abs() * near + tiny, "y")
    # gradients
    dy = rand((rows, n), t, dev, 31)
    dh = rand((rows, n), t, dev, 32) if res else None
    ins = [v for v in (x, r, norm.weight if affine else None) if v is not None]
    grads = list(torch.autograd.grad((y, h) if res else (y,), ins, (dy, dh) if res else (dy,)))
    dyd = dy.double().cpu()
    a = dyd * w
    proj = (a * hd).mean(1, keepdim=True)
    g = inv * (a - hd * inv.square() * proj)
    mag = inv * (a.abs() + hd.abs() * inv.square() * (a * hd).abs().mean(1, keepdim=True))
    if res:
        g = g + dh.double().cpu()
        mag = mag + dh.double().cpu().abs()
    tol = half(t) * g.abs() + (2 * chain + 16) * U * mag + loose * 4 * mag + tiny
    dx = torch.where(keep, g * s, torch.zeros((), dtype=torch.float64)) if p > 0 else g
    assert_within(grads[0], dx, tol * (s if p > 0 else 1) + 2 * U * dx.abs(), "dx")
    if res:
        assert_within(grads[1], g, tol, "dresidual")
    if affine:
        ref = (dyd * hd * inv).sum(0)
        mag = (dyd * hd * inv).abs().sum(0)
        assert grads[-1].dtype == torch.float32
        # per-lane sums over the rows of a block, then over the blocks; the reference sums all rows
        assert_within(grads[-1], ref, ((rows + chain / 2 + 16) * U + loose) * mag + 1e-30, "dweight")


@gpu
def test_rms_norm_gradient_against_differences():
    n, rows = 130, 4
    norm, x, r = norm_case("cuda", torch.float32, rows, n, True, 0.0)
    y, h = Fx.rms_norm(x, norm, residual=r)
    cy, ch = rand((rows, n), torch.float32, "cuda", 41), rand((rows, n), torch.float32, "cuda", 42)
    dx, dr, dw = torch.autograd.grad((y, h), (x, r, norm.weight), (cy, ch))
    xd, rd, wd, cyd, chd = (v.detach().double().cpu() for v in (x, r, norm.weight, cy, ch))

    def f(xx, rr, ww):
        hh = xx + rr
        return float((hh / torch.sqrt(hh.square().mean(1, keepdim=True) + 1e-6) * ww * cyd).sum() + (hh * chd).sum())

    g = torch.Generator().manual_seed(5)
    for name, grad, at in (("x", dx, 0), ("residual", dr, 1), ("weight", dw, 2)):
        args = [xd, rd, wd]
        v = torch.randn(args[at].shape, generator=g, dtype=torch.float64)
        eps = 1e-5
        up, down = list(args), list(args)
        up[at], down[at] = args[at] + eps * v, args[at] - eps * v
        diff = (f(*up) - f(*down)) / (2 * eps)
        got = float((grad.double().cpu() * v).sum())
        # float32 gradients of n * rows terms (1e-5 of the sum of magnitudes), differences good to ~1e-9
        assert abs(got - diff) <= 1e-5 * float((grad.double().cpu() * v).abs().sum()) + 1e-7, name


@pytest.mark.parametrize("dev", DEVICES)
def test_rms_norm_partial_gradients_and_types(dev):
    """Only some inputs ask for a gradient; only one of the two results is used; a bf16 weight; a 3-d, strided input."""
    norm, x, r = norm_case(dev, torch.bfloat16, 6, 40, True, 0.2)
    kw = dict(p=0.2, seed=3)
    y, h = Fx.rms_norm(x, norm, residual=r, **kw)
    dy = rand((6, 40), torch.bfloat16, dev, 51)
    full = torch.autograd.grad(y, (x, r, norm.weight), dy)
    for pick in ((0,), (1,), (2,), (0, 2), (1, 2)):
        ins = [x.detach().requires_grad_(0 in pick), r.detach().requires_grad_(1 in pick)]
        norm.weight.requires_grad_(2 in pick)
        y, h = Fx.rms_norm(ins[0], norm, residual=ins[1], **kw)
        src = [ins[0], ins[1], norm.weight]
        for got, i in zip(torch.autograd.grad(y, [src[i] for i in pick], dy), pick):
            assert torch.equal(got, full[i]), (pick, i)
    norm.weight.requires_grad_(True)
    y, h = Fx.rms_norm(x, norm, residual=r, **kw)
    only_h = torch.autograd.grad(h, (x, r), dy, allow_unused=True)
    keep, s = keep_oracle((6, 40), 0.2, 3, 0)
    assert torch.equal(only_h[1], dy)
    assert torch.equal(only_h[0].cpu() != 0, keep & (dy.cpu() != 0))
    nb = nn.RMSNorm(40, eps=1e-6).to(dev).to(torch.bfloat16)
    with torch.no_grad():
        nb.weight.copy_(norm.weight)
    y = Fx.rms_norm(x, nb)
    (gw,) = torch.autograd.grad(y, (nb.weight,), dy)
    assert gw.dtype == torch.bfloat16
    x3 = rand((5, 40, 6), torch.bfloat16, dev, 52).transpose(1, 2)
    assert torch.equal(Fx.rms_norm(x3, norm), Fx.rms_norm(x3.contiguous().view(-1, 40), norm).view(5, 6, 40))
    n0 = nn.RMSNorm(40).to(dev)  # eps None: the type's own, as in torch
    ref = x.detach().float() / torch.sqrt(x.detach().float().square().mean(1, keepdim=True) + torch.finfo(torch.bfloat16).eps)
    assert_within(Fx.rms_norm(x, n0), ref, half(torch.bfloat16) * ref.abs().double() + 1e-5)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("t", TYPES)
def test_results_do_not_depend_on_asking_for_gradients(dev, t):
    norm, x, r = norm_case(dev, t, 37, 264, True, 0.3)
    lin = nn.Linear(264, 40).to(dev)
    for f in (lambda: Fx.rms_norm(x, norm, p=0.3, seed=4), lambda: Fx.rms_norm(x, norm, residual=r, p=0.3, seed=4)[0],
              lambda: Fx.dropout_counter(x, 0.3, seed=4, residual=r), lambda: Fx.linear_fp8(x, lin, "relu")):
        y = f()
        with torch.no_grad():
            assert y.requires_grad and torch.equal(f(), y)


def test_rms_norm_refuses():
    x, norm = torch.zeros(3, 8), nn.RMSNorm(8)
    with pytest.raises(ValueError):
        Fx.rms_norm(x, nn.RMSNorm(9))
    with pytest.raises(ValueError):
        Fx.rms_norm(x, nn.RMSNorm(9, elementwise_affine=False))
    with pytest.raises(ValueError):
        Fx.rms_norm(x, norm, residual=torch.zeros(3, 9))
    with pytest.raises(ValueError):
        Fx.rms_norm(x, norm, residual=torch.zeros(3, 8, dtype=torch.bfloat16))
    with pytest.raises(TypeError):
        Fx.rms_norm(x.double(), norm)
    with pytest.raises(ValueError):
        Fx.rms_norm(x, norm, p=2.0)
    with pytest.raises(ValueError):
        Fx.rms_norm(torch.zeros(()), norm)
    with pytest.raises(RuntimeError, match="no gradient"):
        Fx.rms_norm_fp8(x, norm)


@gpu
def test_rms_norm_refuses_too_wide():
    with pytest.raises(ValueError, match="columns"):
        Fx.rms_norm(torch.zeros(1, 32776, device="cuda"), nn.RMSNorm(32776, device="cuda"))


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,n,res", [(1, 1, True), (3, 130, False), (5, 2048, True), (2, 1281, True), (2, 8192, False),
                                        (1, 20000, True), (0, 128, True), (700, 384, True)])
def test_rms_norm_fp8(dev, t, rows, n, res):
    norm, x, r = norm_case(dev, t, rows, n, res, 0.0)
    with torch.no_grad():
        out = Fx.rms_norm_fp8(x, norm, residual=r)
        y32 = Fx.rms_norm(x, norm, residual=r)
    b, h = out if res else (out, None)
    if res:
        assert torch.equal(h, y32[1])
    assert b.shape == (rows, n) and b.tile == 1
    hd = (h if res else x).detach().double().cpu()
    ref = hd / torch.sqrt(hd.square().mean(1, keepdim=True) + 1e-6) * norm.weight.detach().double().cpu()
    v = values_of(b)
    nb = -(-n // 128)
    e = b.scale[:, :nb].double().cpu() - 127
    amax = torch.nn.functional.pad(ref.abs(), (0, nb * 128 - n)).view(rows, nb, 128).amax(2)
    # float32 may put a maximum on the other side of 448 * 2^e when it is within 1e-5 of it
    assert bool((amax <= 448 * 2**e * (1 + 1e-5)).all()) and bool((amax * (1 + 1e-5) >= 224 * 2**e).all())
    step = 2.0 ** (torch.floor(torch.log2((ref.abs() / 2 ** e.repeat_interleave(128, 1)[:, :n]).clamp(min=2.0**-6))) - 3)
    scaled = 2 ** e.repeat_interleave(128, 1)[:, :n]
    chain = CHAIN if dev == "cuda" else max(CHAIN, n)
    assert_within(v, ref, step * scaled / 2 + (chain / 2 + 8) * U * ref.abs(), "values")
    assert bool((b.q.view(torch.uint8)[:, n:] == 0).all())


# ---------------------------------------------------------------------------
# quantisation
# ---------------------------------------------------------------------------
def tricky(rows, cols, t, seed):
    """Values across the whole range: blocks of zeros, ties, maxima on both sides of 448 * 2^e, tiny and huge blocks."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g)
    x *= 2.0 ** torch.randint(-12, 6, (rows, 1), generator=g).float()
    x[0, :min(cols, 128)] = 0
    if rows > 4:
        x[1, 0] = 448.0
        x[2, 0] = 449.0
        x[3] = torch.arange(cols).float().remainder(33) / 16  # many ties
        x[4] *= 2.0**-20
    return x.to(t)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (5, 127), (6, 128), (7, 1281), (130, 640), (257, 129)])
def test_quantize_fp8(dev, t, rows, cols):
    x = tricky(rows, cols, t, 61)
    for b, tile in ((Fx.quantize_fp8(x.to(dev)), 1), (Fx.quantize_fp8_weight(x.to(dev)), 128)):
        ref, e = block_oracle(x.double().numpy(), tile)
        assert b.tile == tile and b.shape == (rows, cols)
        assert np.array_equal(b.scale[:, :e.shape[1]].cpu().numpy().astype(np.int64) - 127, e)
        assert bool((b.scale[:, e.shape[1]:] == 127).all()) and bool((b.q.view(torch.uint8)[:, cols:] == 0).all())
        assert torch.equal(values_of(b), torch.from_numpy(ref))
        assert torch.equal(b.dequantize().double().cpu(), torch.from_numpy(ref))
        assert torch.equal(b.dequantize(torch.bfloat16).double().cpu(), torch.from_numpy(ref))


@pytest.mark.parametrize("dev", DEVICES)
def test_quantize_fp8_special_values(dev):
    x = torch.ones(3, 256)
    x[0, 5] = float("inf")
    x[0, 6] = float("-inf")
    x[1, 130] = float("nan")
    x[2, :128] = torch.finfo(torch.float32).max
    x[2, 128:] = 1e-45
    for b, tile in ((Fx.quantize_fp8(x.to(dev)), 1), (Fx.quantize_fp8_weight(x.to(dev)), 128)):
        ref, e = block_oracle(x.double().numpy(), tile)
        assert np.array_equal(b.scale[:, :2].cpu().numpy().astype(np.int64) - 127, e)
        assert torch.equal(torch.nan_to_num(values_of(b), nan=-7e7), torch.nan_to_num(torch.from_numpy(ref), nan=-7e7))
    a, w = Fx.quantize_fp8(x.to(dev)[:2]), Fx.quantize_fp8_weight(torch.eye(256, device=dev)[:64])
    y = Fx.matmul_fp8(a, w, out_dtype=torch.float32).cpu()
    assert bool(y.isnan().all())  # a NaN element makes its own row NaN
    a = Fx.quantize_fp8(torch.cat([x[:1], torch.ones(1, 256)]).to(dev))
    y = Fx.matmul_fp8(a, w, out_dtype=torch.float32).cpu()
    assert bool(y[0].isnan().all()) and torch.equal(y[1], torch.ones(64))


def test_fp8_blocks_refuses():
    q = torch.zeros(4, 256, dtype=torch.uint8).view(torch.float8_e4m3fn)
    s = torch.full((4, 4), 127, dtype=torch.uint8)
    fb.Fp8Blocks(q, s, (4, 200))
    for args in ((q, s, (4, 300), 1), (q, s, (5, 200), 1), (q, s, (4, 200), 64), (q, s[:, :2], (4, 200), 1),
                 (q, s.int(), (4, 200), 1), (q.float(), s, (4, 200), 1), (q, s, (4, 200), 128), (q, s, (4, 0), 1)):
        with pytest.raises(ValueError):
            fb.Fp8Blocks(*args)
    a = fb.Fp8Blocks(q, s, (4, 200))
    w = Fx.quantize_fp8_weight(torch.ones(3, 200))
    assert Fx.matmul_fp8(a, w).shape == (4, 3)
    with pytest.raises(ValueError):
        Fx.matmul_fp8(w, a)
    with pytest.raises(ValueError):
        Fx.matmul_fp8(a, Fx.quantize_fp8_weight(torch.ones(3, 201)))
    with pytest.raises(ValueError):
        Fx.matmul_fp8(a, w, act="gelu")
    with pytest.raises(ValueError):
        Fx.matmul_fp8(a, w, bias=torch.zeros(4))
    with pytest.raises(ValueError):
        Fx.matmul_fp8(a, w, out_dtype=torch.float64)
    with pytest.raises(RuntimeError, match="no gradient"):
        Fx.matmul_fp8(a, w, bias=torch.zeros(3, requires_grad=True))
    with pytest.raises(RuntimeError, match="no gradient"):
        Fx.quantize_fp8(torch.zeros(2, 8, requires_grad=True))
    with pytest.raises(TypeError):
        Fx.quantize_fp8(torch.zeros(2, 8, dtype=torch.float64))
    with pytest.raises(ValueError):
        Fx.quantize_fp8_weight(torch.zeros(2, 8, 2))
    lin = nn.Linear(8, 4)
    with pytest.raises(ValueError):
        Fx.linear_fp8(torch.zeros(2, 9), lin)
    with pytest.raises(NotImplementedError):
        Fx.linear_fp8(torch.zeros(2, 8), lin, act="silu")
    with pytest.raises(TypeError):
        Fx.linear_fp8(torch.zeros(2, 8, dtype=torch.float64), lin)


# ---------------------------------------------------------------------------
# products
# ---------------------------------------------------------------------------
SHAPES = [(1, 1, 1), (1, 130, 256), (2, 16, 640), (16, 33, 1281), (17, 1000, 1280), (33, 64, 2048), (65, 200, 129), (64, 513, 4096),
          (129, 257, 1000), (133, 1000, 1280), (300, 300, 896), (128, 1024, 128), (1000, 120, 512), (515, 1030, 1152),
          (0, 8, 128), (3, 2, 8192), (512, 512, 128), (769, 515, 300), (520, 1025, 1664)]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("tile", [1, 128])
def test_matmul_fp8_integers_are_exact(dev, m, n, k, tile):
    """Small integers under scales of 2^-1, 1 and 2: every product and sum is exact, so the result is too."""
    g = torch.Generator().manual_seed(m + n + k)
    kp = fb.padded_cols(k)

    def mk(rows, tl):
        v = torch.randint(-3, 4, (rows, k), generator=g).float()
        q = torch.zeros(rows, kp)
        q[:, :k] = v
        s = torch.randint(126, 129, (-(-rows // tl), fb.scale_cols(k)), generator=g).to(torch.uint8)
        b = fb.Fp8Blocks(q.to(torch.float8_e4m3fn).to(dev), s.to(dev), (rows, k), tl)
        return b, values_of(b)
    a, av = mk(m, 1)
    b, bv = mk(n, tile)
    bias = torch.randint(-5, 6, (n,), generator=g).float()
    ref = av @ bv.t()
    assert torch.equal(Fx.matmul_fp8(a, b, out_dtype=torch.float32).double().cpu(), ref)
    got = Fx.matmul_fp8(a, b, bias=bias.to(dev), act="relu", out_dtype=torch.float32)
    assert torch.equal(got.double().cpu(), (ref + bias.double()).clamp(min=0))


@gpu
@pytest.mark.parametrize("kernel", range(7))
@pytest.mark.parametrize("m,n,k", [(1, 16, 128), (5, 100, 130), (70, 130, 1000), (150, 260, 1281), (300, 515, 640), (257, 129, 2176)])
def test_matmul_fp8_every_kernel(kernel, m, n, k):
    """Each kernel at sizes that the choice by size would give to another: exact on integers, every output type."""
    from pytorch_imageclassification_distributed_amd.ops import hip
    keep = hip.C.fp8_gemm_force
    keep(kernel)
    try:
        for tile in (1, 128):
            test_matmul_fp8_integers_are_exact("cuda", m, n, k, tile)
        for t, act in ((torch.bfloat16, "silu"), (torch.float16, "relu"), (torch.float32, None)):
            test_matmul_fp8("cuda", t, m, n, k, act)
    finally:
        keep(-1)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m,n,k,act", [(1, 130, 256, "silu"), (33, 64, 2048, "relu"), (129, 257, 1000, None), (300, 300, 896, "silu"),
                                       (16, 40, 8192, None)])
def test_matmul_fp8(dev, t, m, n, k, act):
    """Real values.  The matrix instruction aligns a block's products to the largest before adding: at most 2^-12 of the
    sum of magnitudes (1.1e-4 = 2^-13 was the largest measured on values spread over the whole e4m3 range)."""
    x, w = rand((m, k), t, "cpu", 71, 2.0), rand((n, k), torch.float32, "cpu", 72, k**-0.5)
    bias = rand((n,), torch.bfloat16, "cpu", 73)
    a, b = Fx.quantize_fp8(x.to(dev)), Fx.quantize_fp8_weight(w.to(dev))
    got = Fx.matmul_fp8(a, b, bias=bias.to(dev), act=act, out_dtype=t)
    assert got.dtype == t and got.shape == (m, n)
    z = values_of(a) @ values_of(b).t() + bias.double()
    mag = values_of(a).abs() @ values_of(b).abs().t() + bias.double().abs()
    ref = z.clamp(min=0) if act == "relu" else z * torch.sigmoid(z) if act == "silu" else z
    # silu: |d silu / dz| <= 1.1; its exp and reciprocal are good to a few float32 steps
    assert_within(got, ref, half(t) * ref.abs() + 1.1 * 2.0**-12 * mag + 16 * U * z.abs(), "y")


@gpu
@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 31, 32, 33, 48, 63, 64, 65, 96, 127, 128, 129, 255, 256, 257])
def test_matmul_fp8_every_row_count(m):
    """Row counts around every tile border; the same rows give the same result whatever the count around them is, up to
    the order of the float32 sum."""
    x, w = rand((300, 1152), torch.bfloat16, "cuda", 74), rand((272, 1152), torch.float32, "cuda", 75, 0.03)
    b = Fx.quantize_fp8_weight(w)
    a = Fx.quantize_fp8(x[:m])
    got = Fx.matmul_fp8(a, b, out_dtype=torch.float32)
    va, vb = values_of(a), values_of(b)
    assert_within(got, va @ vb.t(), 2.0**-12 * (va.abs() @ vb.abs().t()), f"m={m}")
    assert torch.equal(got, Fx.matmul_fp8(a, b, out_dtype=torch.float32))


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m,k,n,act,bias", [(1, 8, 3, None, True), (5, 130, 7, "relu", True), (64, 256, 128, None, True), (200, 512, 96, "relu", True),
                                            (1024, 320, 40, None, False), (130, 1281, 257, "relu", True), (0, 64, 32, None, True),
                                            (700, 264, 520, None, True)])
def test_linear_fp8(dev, t, m, k, n, act, bias):
    lin = nn.Linear(k, n, bias=bias)
    with torch.no_grad():
        lin.weight.copy_(rand((n, k), torch.float32, "cpu", 81, k**-0.5))
    lin = lin.to(dev)
    x = rand((m, k), t, dev, 82, 1.5).requires_grad_(True)
    y = Fx.linear_fp8(x, lin, act)
    assert y.dtype == t and y.shape == (m, n)
    xq = torch.from_numpy(block_oracle(x.detach().double().cpu().numpy(), 1)[0]).view(m, k)
    wq = torch.from_numpy(block_oracle(lin.weight.detach().double().cpu().numpy(), 128)[0])
    bd = lin.bias.detach().double().cpu() if bias else torch.zeros(n, dtype=torch.float64)
    z = xq @ wq.t() + bd
    zmag = xq.abs() @ wq.abs().t() + bd.abs()
    ref = z.clamp(min=0) if act else z
    assert_within(y, ref, half(t) * ref.abs() + 2.0**-12 * zmag, "y")
    dy = rand((m, n), t, dev, 83, 1e-2)
    ins = (x, lin.weight) + ((lin.bias,) if bias else ())
    grads = torch.autograd.grad(y, ins, dy)
    g = dy.double().cpu()
    if act:
        g = torch.where(y.detach().cpu() > 0, g, torch.zeros((), dtype=torch.float64))
    gq = torch.from_numpy(block_oracle(g.numpy(), 1)[0]).view(m, n)
    assert grads[0].dtype == t
    dx = gq @ wq
    assert_within(grads[0], dx, half(t) * dx.abs() + 2.0**-12 * (gq.abs() @ wq.abs()) + torch.finfo(t).smallest_normal * torch.finfo(t).eps, "dx")
    gb, xb = g.to(torch.bfloat16).double(), x.detach().to(torch.bfloat16).double().cpu()
    assert_within(grads[1], gb.t() @ xb, (m + 16) * U * (gb.abs().t() @ xb.abs()) + 1e-30, "dweight")
    if bias:
        assert_within(grads[2], g.sum(0), (m + 16) * U * g.abs().sum(0) + 1e-30, "dbias")


@gpu
@pytest.mark.parametrize("tile", [128, 256])
@pytest.mark.parametrize("m,n,k", [(1, 5, 7), (63, 130, 129), (64, 128, 128), (65, 257, 300), (192, 100, 1281), (257, 384, 515), (320, 64, 256),
                                   (1024, 127, 640), (9000, 40, 72)])
def test_linear_fp8_weight_gradient_tiles(tile, m, n, k):
    """Both weight-gradient kernels at sizes around their tiles, stages and row splits.  Integers: every sum is exact."""
    from pytorch_imageclassification_distributed_amd.ops import hip
    g = torch.Generator().manual_seed(m + n + k)
    lin = nn.Linear(k, n).to("cuda")
    x, dy = (torch.randint(-4, 5, (m, c), generator=g).to(torch.bfloat16) for c in (k, n))
    try:
        hip.C.rows_grad_force(tile)
        (dw,) = torch.autograd.grad(Fx.linear_fp8(x.cuda(), lin), (lin.weight,), dy.cuda())
    finally:
        hip.C.rows_grad_force(0)
    assert torch.equal(dw.double().cpu(), dy.double().t() @ x.double())


@pytest.mark.parametrize("dev", DEVICES)
def test_linear_fp8_partial_gradients_shapes_and_parameter_types(dev):
    lin = nn.Linear(72, 24).to(dev)
    x = rand((2, 5, 72), torch.bfloat16, dev, 84).requires_grad_(True)
    dy = rand((2, 5, 24), torch.bfloat16, dev, 85)
    full = torch.autograd.grad(Fx.linear_fp8(x, lin, "relu"), (x, lin.weight, lin.bias), dy)
    assert full[0].shape == x.shape
    for pick in ((0,), (1,), (2,), (0, 1), (1, 2)):
        xx = x.detach().requires_grad_(0 in pick)
        lin.weight.requires_grad_(1 in pick)
        lin.bias.requires_grad_(2 in pick)
        src = (xx, lin.weight, lin.bias)
        for got, i in zip(torch.autograd.grad(Fx.linear_fp8(xx, lin, "relu"), [src[i] for i in pick], dy), pick):
            assert torch.equal(got, full[i]), (pick, i)
    lin.requires_grad_(True)
    xt = rand((72, 10), torch.bfloat16, dev, 86).t()
    assert torch.equal(Fx.linear_fp8(xt, lin), Fx.linear_fp8(xt.contiguous(), lin))
    with torch.no_grad():
        assert not Fx.linear_fp8(x, lin).requires_grad
    for t in (torch.bfloat16, torch.float16):
        low = nn.Linear(72, 24).to(dev).to(t)
        gw, gb = torch.autograd.grad(Fx.linear_fp8(x, low), (low.weight, low.bias), dy)
        assert gw.dtype == t and gb.dtype == t
    # the weight may change between calls (nothing is kept from one call for the next)
    before = Fx.linear_fp8(x, lin).detach()
    with torch.no_grad():
        lin.weight.mul_(2)
        lin.bias.mul_(2)
    assert torch.equal(Fx.linear_fp8(x, lin).detach(), before * 2)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("act", [None, "relu", "silu"])
@pytest.mark.parametrize("m,n", [(3, 40), (70, 200), (600, 520)])
def test_nan_passes_activations(dev, act, m, n):
    """A NaN or infinite input makes its row of outputs NaN through every activation, and a ReLU's backward hands such a
    row's gradient on; the other rows are as without it."""
    lin = nn.Linear(130, n)
    with torch.no_grad():
        lin.weight.copy_(rand((n, 130), torch.float32, "cpu", 87, 0.1))
    lin = lin.to(dev)
    x = rand((m, 130), torch.bfloat16, dev, 88)
    bad = x.clone()
    bad[1, 7], bad[m - 1, 129] = float("nan"), float("inf")
    rows = torch.zeros(m, dtype=torch.bool, device=dev)
    rows[1] = rows[m - 1] = True
    with torch.no_grad():
        w = Fx.quantize_fp8_weight(lin.weight)
        good, got = (Fx.matmul_fp8(Fx.quantize_fp8(v), w, bias=lin.bias, act=act) for v in (x, bad))
        assert bool(got[rows].isnan().all()) and torch.equal(got[~rows], good[~rows])
    if act != "silu":
        dy = rand((m, n), torch.bfloat16, dev, 89)
        bad.requires_grad_(True)
        y = Fx.linear_fp8(bad, lin, act)
        assert bool(y[rows].isnan().all()) and not bool(y[~rows].isnan().any())
        dx, db = torch.autograd.grad(y, (bad, lin.bias), dy)
        plain = bad.detach().requires_grad_(True)
        (through,) = torch.autograd.grad(Fx.linear_fp8(plain, lin), plain, dy)
        assert torch.equal(dx[rows], through[rows])
        g = torch.where(y <= 0, 0.0, dy.double()) if act else dy.double()
        assert_within(db, g.sum(0), (m + 16) * U * g.abs().sum(0), "dbias")


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------
class Block(nn.Module):
    """h = residual + dropout(x); y = norm(h); h + dropout(linear(relu(linear(y))))."""

    def __init__(self, d, hidden):
        super().__init__()
        self.norm, self.up, self.down = nn.RMSNorm(d, eps=1e-6), nn.Linear(d, hidden), nn.Linear(hidden, d)

    def forward(self, x, residual, p, seed):
        y, h = Fx.rms_norm(x, self.norm, residual=residual, p=p, training=self.training, seed=seed)
        z = Fx.linear_fp8(Fx.linear_fp8(y, self.up, "relu"), self.down)
        return Fx.dropout_counter(z, p, self.training, seed=seed, offset=0 if torch.is_tensor(seed) else 1, residual=h)

    @torch.no_grad()
    def serve(self, x, residual, up, down):
        a, h = Fx.rms_norm_fp8(x, self.norm, residual=residual)
        z = Fx.quantize_fp8(Fx.matmul_fp8(a, up, bias=self.up.bias, act="relu", out_dtype=x.dtype))
        return Fx.dropout_counter(Fx.matmul_fp8(z, down, bias=self.down.bias, out_dtype=x.dtype), 0.5, False, residual=h)


def make_block(d=320, hidden=520, dev="cuda"):
    torch.manual_seed(0)
    return Block(d, hidden).to(dev)


@gpu
def test_block_gpu_against_reference_path():
    """The whole block, forward and backward, against the reference path on the CPU: the same masks, and results apart by
    the 8-bit roundings that tip where a bf16 input to them differs by a bf16 step (a share of about 2^-8 / 2^-4 of the
    elements moves by up to 2^-3 of itself, three times in a row: under 2^-4 of the result's norm)."""
    d, rows = 320, 130
    net, cpu = make_block(dev="cuda"), make_block(dev="cpu")
    outs = []
    for m, dev in ((net, "cuda"), (cpu, "cpu")):
        x = rand((rows, d), torch.bfloat16, dev, 91).requires_grad_(True)
        r = rand((rows, d), torch.bfloat16, dev, 92).requires_grad_(True)
        y = m(x, r, 0.25, 77)
        y.backward(rand((rows, d), torch.bfloat16, dev, 93))
        outs.append([y.detach(), x.grad, r.grad] + [p.grad for p in m.parameters()])
    for a, b in zip(*outs):
        a, b = a.double().cpu(), b.double()
        assert float((a - b).norm() / b.norm()) < 2.0**-4
    keep, _ = keep_oracle((rows, d), 0.25, 77, 0)
    assert bool((outs[0][1].cpu()[~keep] == 0).all())


@gpu
def test_block_on_streams_and_at_once():
    """Two calls at once on two streams, neither of them the default one, equal the calls alone."""
    net = make_block()
    ins = [(rand((257, 320), torch.bfloat16, "cuda", 100 + i), rand((257, 320), torch.bfloat16, "cuda", 110 + i)) for i in range(2)]

    def step(i):
        x, r = (v.clone().requires_grad_(True) for v in ins[i])
        y = net(x, r, 0.1, 5 + i)
        return (y,) + torch.autograd.grad(y, [x, r] + list(net.parameters()), torch.ones_like(y))
    alone = [step(i) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None, None]
    for rep in range(3):
        for i, s in enumerate(streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got[i] = step(i)
        torch.cuda.synchronize()
        for a, b in zip(alone, got):
            assert all(torch.equal(u, v) for u, v in zip(a, b))


@gpu
def test_block_captured_and_replayed():
    """Serving and a training step (forward + backward, the seed in a device tensor) captured into graphs; every replay,
    with eager work between, equals the eager call on the same inputs and seed."""
    net = make_block()
    params = list(net.parameters())
    up, down = Fx.quantize_fp8_weight(net.up.weight), Fx.quantize_fp8_weight(net.down.weight)
    x, r = rand((133, 320), torch.bfloat16, "cuda", 120), rand((133, 320), torch.bfloat16, "cuda", 121)
    xg, rg = x.clone().requires_grad_(True), r.clone().requires_grad_(True)
    g = rand((133, 320), torch.bfloat16, "cuda", 122)
    state = torch.tensor([5, 0], device="cuda")

    def train():
        y = net(xg, rg, 0.1, state)
        return [y.detach()] + list(torch.autograd.grad(y, [xg, rg] + params, g))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            net.serve(x, r, up, down)
            train()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graphs = []
    for fn in (lambda: [net.serve(x, r, up, down)], train):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = fn()
        graphs.append((gr, out, fn))
    for rep in range(4):
        with torch.no_grad():
            for dst, seed in ((x, 130), (r, 140)):
                dst.copy_(rand((133, 320), torch.bfloat16, "cuda", seed + rep))
            xg.copy_(x)
            rg.copy_(r)
        state.copy_(torch.tensor([9 + rep, 3 * rep], device="cuda"))
        for gr, out, fn in graphs:
            gr.replay()
        torch.cuda.synchronize()
        for gr, out, fn in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, fn())), rep
        torch.cuda.synchronize()


@gpu
def test_block_gradients_land_in_the_arena():
    """Parameter gradients go straight into the flat gradient arena when one is armed, and accumulate otherwise."""
    from pytorch_imageclassification_distributed_amd.ops.grad_arena import GradArena
    net = make_block()
    x, r = rand((64, 320), torch.bfloat16, "cuda", 150), rand((64, 320), torch.bfloat16, "cuda", 151)
    net(x, r, 0.1, 3).sum().backward()
    plain = [p.grad.clone() for p in net.parameters()]
    for p in net.parameters():
        p.grad = None
    arena = GradArena(list(net.parameters()))
    try:
        for rep in range(2):
            for p in net.parameters():
                p.grad = None
            arena.begin()
            net(x, r, 0.1, 3).sum().backward()
            for p, g in zip(net.parameters(), plain):
                assert arena.owns(p) and torch.equal(p.grad, g)
        net(x, r, 0.1, 3).sum().backward()
        for p, g in zip(net.parameters(), plain):
            assert_within(p.grad, 2 * g.double(), 4 * U * g.double().abs())
    finally:
        arena.detach_params()


@pytest.mark.parametrize("dev", DEVICES)
def test_second_derivatives_are_refused(dev):
    x = rand((4, 64), torch.float32, dev, 170).requires_grad_(True)
    norm, lin = nn.RMSNorm(64).to(dev), nn.Linear(64, 8).to(dev)
    for f in (lambda: Fx.rms_norm(x, norm), lambda: Fx.linear_fp8(x, lin)):
        (g,) = torch.autograd.grad(f().square().sum(), (x,), create_graph=True)
        with pytest.raises(RuntimeError):
            g.sum().backward()


@gpu
def test_block_facade_and_missing_fallback():
    """The op layer's HIP part owns every name, and the operators run its kernels for GPU tensors (the torch backend gives
    the reference path)."""
    import ast
    import os
    from pytorch_imageclassification_distributed_amd.ops._hip import block
    from pytorch_imageclassification_distributed_amd.ops import hip
    names = set()
    for nd in ast.parse(open(os.path.abspath(block.__file__)).read()).body:
        if isinstance(nd, (ast.FunctionDef, ast.ClassDef)):
            names.add(nd.name)
    assert names == set(block._OWNED) and hip.matmul_fp8 is block.matmul_fp8
    x = rand((4, 64), torch.float32, "cuda", 160)
    keep = Fx.get_backend()
    try:
        Fx.set_backend("torch")
        ref = Fx.dropout_counter(x, 0.5, seed=3)
    finally:
        Fx.set_backend(keep)
    assert torch.equal(Fx.dropout_counter(x, 0.5, seed=3), ref)
