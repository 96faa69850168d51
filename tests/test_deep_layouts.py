"""Wave layouts of the prefetch-depth-2 conv kernels' table (csrc/conv_deep.hip)."""
import pytest


def test_every_deep_tile_runs_on_eight_waves():
    from pytorch_imageclassification_distributed_amd.ops import hip
    cfgs = hip.conv_deep_cfgs()
    # entry numbers are what a find-db names: the tiles and schedule variants keep their places
    assert [(c[0], c[1], c[4]) for c in cfgs] == [
        (256, 256, 0), (256, 256, 1), (256, 128, 0), (512, 64, 0), (256, 256, 8), (256, 256, 16), (256, 256, 32),
        (256, 256, 2), (256, 256, 4), (256, 256, 80), (256, 256, 144), (256, 128, 80), (256, 256, 256),
        (256, 256, 336), (256, 128, 336), (256, 256, 257)]
    for tm, bn, wm, wn, _ in cfgs:
        assert wm * wn == 8 and tm % (16 * wm) == 0 and bn % (16 * wn) == 0
        assert tm // wm * (bn // wn) // 64 <= 128  # accumulators a lane: half of the 256 registers of two waves a SIMD


@pytest.mark.gpu
def test_the_two_kinds_of_tile_give_the_same_sums():
    """The depth-2 tile and the one-tile-in-flight tile add the same products in the same order."""
    import torch
    from pytorch_imageclassification_distributed_amd.ops import hip
    g = torch.Generator().manual_seed(0)
    a = (torch.rand(1000, 640, generator=g) * 2 - 1).to(torch.bfloat16).cuda()
    b = (torch.rand(520, 640, generator=g) * 2 - 1).to(torch.bfloat16).cuda()
    zero = hip.ws(a.device).zero
    geo = (1000, 520, 640, 640, 1000, 1, 1000, 1, 1, 640, 1000, 1, 1, 0, 0, 520, 0)

    def run(cfg):
        out = torch.empty(1000, 520, device="cuda", dtype=torch.bfloat16)
        hip.C.conv_gemm(a, b.view(-1), out, None, None, *geo, [0], [0], [0], hip.G_STATS, zero, None, None, None, None,
                        None, 0, 1, 0, 0, cfg, None, None, None, None, None, None, None, 0, None, None, None, None, 0)
        return out
    ref = run(4)
    for v, c in enumerate(hip.conv_deep_cfgs()):
        if c[4] & (6 | 256) == 0:
            assert torch.equal(run(hip.DEEP_BASE + v), ref), c
