"""Channels-last GroupNorm(+SiLU), its statistics, checkpoint and gradient against 64-bit definitions."""
import pytest
import torch

from gpu_util import Guarded
from train_util import (DTYPES, K, U, assert_within, checkpoint_reference, gn_backward, gn_forward, half_step, make)

pytestmark = pytest.mark.gpu

ALL = ["float32", "float16", "bfloat16"]
EPS = 1e-5


def put(t, misalign=0):
    g = Guarded(tuple(t.shape), t.dtype, misalign)
    g.tensor.copy_(t)
    return g.tensor


def weights(C, seed):
    return make((C,), "float32", seed, 0.2, 1.0), make((C,), "float32", seed + 1, 0.3)


def inputs(shape, dtype, seed, mean=0.3):
    """Every channel with a level and a spread of its own."""
    C = shape[-1]
    x = make(shape, "float32", seed) * (0.5 + torch.rand(C, generator=torch.Generator().manual_seed(seed + 7)))
    return (x + make((C,), "float32", seed + 8, 0.5, mean)).to(DTYPES[dtype])


def check_forward(y, x, gamma, beta, G, silu, dtype, what):
    want, mean, rstd, terms = gn_forward(x, gamma, beta, G, EPS, silu)
    assert_within(y, want, half_step(want, dtype) + 1.1 * K * U * terms, what)
    return mean, rstd


def check_backward(got, dy, x, mean, rstd, gamma, beta, G, silu, dtype, what):
    want, bound = gn_backward(dy, x, mean, rstd, gamma, beta, G, silu)
    assert_within(got[0], want[0], half_step(want[0], dtype) + bound[0], what + " grad_x")
    assert_within(got[1], want[1], bound[1] + 1e-30, what + " grad_gamma")
    assert_within(got[2], want[2], bound[2] + 1e-30, what + " grad_beta")


# batch, pixels, channels, groups: one pixel, odd sizes, groups of one channel, groups that end inside a
# 16-byte vector, one group, rows of odd length, wide rows, the shapes of the UNet, many pixels
SHAPES = [(1, 1, 32, 32), (1, 1, 64, 1), (3, 1, 320, 32), (2, 5, 8, 8), (2, 37, 30, 10), (1, 63, 33, 11), (2, 64, 1280, 32),
          (2, 35, 320, 32), (1, 1024, 640, 32), (3, 47 * 13, 96, 8), (2, 130, 2560, 32), (1, 50, 5120, 1), (1, 9, 4099, 1),
          (2, 3000, 16, 4), (1, 4096, 320, 32), (2, 16384, 64, 32), (1, 70000, 32, 16), (1, 40000, 128, 32), (5, 257, 48, 3),
          (65, 17, 64, 32), (2, 1111, 1, 1), (1, 2048, 960, 32)]


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("B,P,C,G", SHAPES)
def test_forward_and_backward(sdfl, B, P, C, G, dtype):
    ops = sdfl.ops
    silu = (P + C) % 3 != 0
    x, dy = inputs((B, P, C), dtype, P + C), make((B, P, C), dtype, P + C + 50)
    gamma, beta = weights(C, C)
    dx_, dg, db = x.cuda(), gamma.cuda(), beta.cuda()
    out = Guarded((B, P, C), DTYPES[dtype])
    y, mean, rstd, kept = ops.groupnorm_channels_last_train(dx_, dg, db, G, EPS, silu, checkpoint=True, out=out.tensor)
    out.check()
    wmean, wrstd = check_forward(y, x, gamma, beta, G, silu, dtype, "forward")
    size = x.double().abs().reshape(B, P, G, C // G).mean(dim=(1, 3))
    assert_within(mean, wmean, K * U * size + 1e-30, "mean")
    # the variance's own roundings, and the mean's error squared against it
    assert_within(rstd, wrstd, wrstd * (K * U + (K * U * size * wrstd) ** 2), "rstd")
    check_forward(ops.groupnorm_channels_last(dx_, dg, db, G, EPS, silu), x, gamma, beta, G, silu, dtype, "inference")
    codes, scales, values = checkpoint_reference(x)
    assert torch.equal(kept.codes.cpu(), codes) and torch.equal(kept.scales.cpu(), scales)

    grad = Guarded((B, P, C), DTYPES[dtype])
    got = ops.groupnorm_channels_last_backward(dy.cuda(), dx_, mean, rstd, dg, db, G, silu, out=grad.tensor)
    grad.check()
    check_backward(got, dy, x, mean.cpu(), rstd.cpu(), gamma, beta, G, silu, dtype, "tensor")
    got2 = ops.groupnorm_channels_last_backward(dy.cuda(), kept, mean, rstd, dg, db, G, silu, out=grad.tensor)
    grad.check()
    check_backward(got2, dy, values, mean.cpu(), rstd.cpu(), gamma, beta, G, silu, dtype, "checkpoint")
    # the same bits again
    again = ops.groupnorm_channels_last_backward(dy.cuda(), kept, mean, rstd, dg, db, G, silu)
    assert all(torch.equal(a, b) for a, b in zip(again, got2))


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("B,P,C,G", [(2, 77, 64, 8), (1, 700, 320, 32), (1, 33000, 64, 32)])
def test_misaligned_and_in_place(sdfl, B, P, C, G, dtype):
    ops = sdfl.ops
    x, dy = inputs((B, P, C), dtype, 3), make((B, P, C), dtype, 4)
    gamma, beta = weights(C, 5)
    dg, db = gamma.cuda(), beta.cuda()
    for misalign in (0, 1):
        buf = put(x, misalign)
        y, mean, rstd, kept = ops.groupnorm_channels_last_train(buf, dg, db, G, EPS, True, checkpoint=True, out=buf)
        assert y.data_ptr() == buf.data_ptr()
        check_forward(buf, x, gamma, beta, G, True, dtype, "in place")
        codes, scales, values = checkpoint_reference(x)
        assert torch.equal(kept.codes.cpu(), codes) and torch.equal(kept.scales.cpu(), scales)
        grad = put(dy, misalign)                                          # over grad_out
        got = ops.groupnorm_channels_last_backward(grad, kept, mean, rstd, dg, db, G, True, out=grad)
        check_backward(got, dy, values, mean.cpu(), rstd.cpu(), gamma, beta, G, True, dtype, "over grad_out")
        src = put(x, misalign)                                            # over x
        got = ops.groupnorm_channels_last_backward(put(dy, misalign), src, mean, rstd, dg, db, G, True, out=src)
        check_backward(got, dy, x, mean.cpu(), rstd.cpu(), gamma, beta, G, True, dtype, "over x")


@pytest.mark.parametrize("P,C,G", [(300, 64, 8), (40000, 32, 8)])
def test_large_offset_and_outliers(sdfl, P, C, G):
    """Values far from zero (mean / spread 1000), a first pixel far from all others, a constant group."""
    gamma, beta = weights(C, 9)
    for kind in range(3):
        x = make((2, P, C), "float32", 60 + kind)
        if kind == 0:
            x = x + 1000.0
        elif kind == 1:
            x[:, 0] += 300.0
        else:
            x[:, :, :C // G] = 2.5
        y, mean, rstd, _ = sdfl.ops.groupnorm_channels_last_train(x.cuda(), gamma.cuda(), beta.cuda(), G, EPS, False)
        want, wmean, wrstd, terms = gn_forward(x, gamma, beta, G, EPS, False)
        size = x.double().abs().reshape(2, P, G, C // G).mean(dim=(1, 3))
        assert_within(mean, wmean, K * U * size, f"mean {kind}")
        assert_within(rstd, wrstd, wrstd * (K * U + (K * U * size * wrstd) ** 2), f"rstd {kind}")
        assert_within(y, want, half_step(want, "float32") + K * U * terms, f"y {kind}")


@pytest.mark.parametrize("B,P,C,G", [(2, 300, 64, 8), (2, 40000, 64, 8), (1, 33000, 512, 32), (2, 300, 30, 10)])
def test_means_whose_square_overflows(sdfl, B, P, C, G):
    """Around 2^65: the square of a value is no fp32 number, that of a deviation is."""
    gamma, beta = weights(C, 19)
    x = (make((B, P, C), "float32", 80).double() * 2.0 ** 53 + 2.0 ** 65).float()
    y, mean, rstd, _ = sdfl.ops.groupnorm_channels_last_train(x.cuda(), gamma.cuda(), beta.view(1, C).cuda(), G, EPS, False)
    want, wmean, wrstd, terms = gn_forward(x, gamma, beta, G, EPS, False)
    size = x.double().abs().reshape(B, P, G, C // G).mean(dim=(1, 3))
    assert_within(mean, wmean, K * U * size, "mean")
    assert_within(rstd, wrstd, wrstd * (K * U + (K * U * size * wrstd) ** 2), "rstd")
    assert_within(y, want, half_step(want, "float32") + K * U * terms, "y")
    dy = make((B, P, C), "float32", 81)
    got = sdfl.ops.groupnorm_channels_last_backward(dy.cuda(), x.cuda(), mean, rstd, gamma.cuda(), beta.view(1, C).cuda(), G)
    assert got[1].shape == (C,) and got[2].shape == (1, C)
    check_backward((got[0], got[1], got[2].view(C)), dy, x, mean.cpu(), rstd.cpu(), gamma, beta, G, False, "float32", "backward")


def test_gradient_against_differences(sdfl):
    B, P, C, G = 2, 30, 24, 6
    x, dy, v = (make((B, P, C), "float32", s) for s in (71, 72, 73))
    gamma, beta = weights(C, 74)
    vg, vb = make((C,), "float32", 75), make((C,), "float32", 76)
    _, mean, rstd, src = sdfl.ops.groupnorm_channels_last_train(x.cuda(), gamma.cuda(), beta.cuda(), G, EPS, True)
    gx, gg, gb = (t.cpu().double() for t in sdfl.ops.groupnorm_channels_last_backward(
        dy.cuda(), src, mean, rstd, gamma.cuda(), beta.cuda(), G, True))

    def value(t):
        y = gn_forward(x.double() + t * v.double(), gamma.double() + t * vg.double(), beta.double() + t * vb.double(),
                       G, EPS, True)[0]
        return (y * dy.double()).sum()

    h = 1e-5
    slope = (gx * v.double()).sum() + (gg * vg.double()).sum() + (gb * vb.double()).sum()
    size = (gx * v.double()).abs().sum() + (gg * vg.double()).abs().sum() + (gb * vb.double()).abs().sum()
    assert abs(slope - (value(h) - value(-h)) / (2 * h)) <= 1e-6 * size + 1e-7


def test_non_finite_values_stay_in_their_group(sdfl):
    x = inputs((2, 50, 64), "float16", 81)
    x[1, 7, 9] = float("nan")
    gamma, beta = weights(64, 82)
    y, mean, rstd, kept = sdfl.ops.groupnorm_channels_last_train(x.cuda(), gamma.cuda(), beta.cuda(), 8, EPS, True,
                                                                 checkpoint=True)
    bad = torch.zeros((2, 50, 64), dtype=torch.bool)
    bad[1, :, 8:16] = True
    assert torch.equal(torch.isnan(y.cpu()), bad)
    assert int(torch.isnan(mean).sum()) == 1 and bool(torch.isnan(mean[1, 1]))
    dy = make((2, 50, 64), "float16", 83)
    gx, gg, gb = sdfl.ops.groupnorm_channels_last_backward(dy.cuda(), x.cuda(), mean, rstd, gamma.cuda(), beta.cuda(), 8, True)
    assert torch.equal(torch.isnan(gx.cpu()), bad)
    assert torch.isnan(gg[8:16]).all() and torch.isfinite(gg[:8]).all() and torch.isfinite(gg[16:]).all()


def test_empty_tensors_and_single_gradients(sdfl):
    ops, capi = sdfl.ops, sdfl._capi
    gamma, beta = (t.cuda() for t in weights(64, 1))
    for shape in [(0, 5, 64), (2, 0, 64)]:
        x = torch.empty(shape, dtype=torch.bfloat16, device="cuda")
        y, mean, rstd, kept = ops.groupnorm_channels_last_train(x, gamma, beta, 8, checkpoint=True)
        gx, gg, gb = ops.groupnorm_channels_last_backward(y, kept, mean, rstd, gamma, beta, 8)
        assert gx.shape == shape and not gg.any() and not gb.any()
    # only one of the weight gradients, or none
    x, dy = inputs((2, 100, 64), "float32", 2).cuda(), make((2, 100, 64), "float32", 3).cuda()
    _, mean, rstd, _ = ops.groupnorm_channels_last_train(x, gamma, beta, 8)
    want = ops.groupnorm_channels_last_backward(dy, x, mean, rstd, gamma, beta, 8)
    ws = torch.empty(capi.lib.sdfl_groupnorm_channels_last_workspace_bytes(2, 64, 100, 8, 1, 0), dtype=torch.uint8, device="cuda")
    for pick in range(3):
        gx = torch.empty_like(x)
        gg, gb = torch.full((64,), 7.0, device="cuda"), torch.full((64,), 7.0, device="cuda")
        rc = capi.lib.sdfl_groupnorm_channels_last_backward(
            x.data_ptr(), None, None, dy.data_ptr(), gx.data_ptr(), gamma.data_ptr(), beta.data_ptr(), mean.data_ptr(),
            rstd.data_ptr(), gg.data_ptr() if pick == 1 else None, gb.data_ptr() if pick == 2 else None, 2, 64, 100, 8, 0, 0,
            ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream)
        assert rc == capi.OK and torch.equal(gx, want[0])
        assert torch.equal(gg, want[1]) if pick == 1 else bool((gg == 7).all())
        assert torch.equal(gb, want[2]) if pick == 2 else bool((gb == 7).all())


@pytest.mark.parametrize("B,P,C", [(2, 64, 320), (1, 4096, 320), (1, 66000, 64)])
def test_streams_and_graphs(sdfl, B, P, C):
    """An explicit stream, two graphs replayed on two streams at once, and new data in a captured graph."""
    ops = sdfl.ops
    gamma, beta = (t.cuda() for t in weights(C, 1))
    data = [(inputs((B, P, C), "bfloat16", s).cuda(), make((B, P, C), "bfloat16", s + 1).cuda()) for s in (10, 20)]

    def step(x, dy, stream=None):
        y, mean, rstd, kept = ops.groupnorm_channels_last_train(x, gamma, beta, 32, EPS, True, checkpoint=True, stream=stream)
        return (y,) + ops.groupnorm_channels_last_backward(dy, kept, mean, rstd, gamma, beta, 32, True, stream=stream)

    want = [[t.clone() for t in step(*d)] for d in data]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = step(*data[0], stream=side)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want[0]))
    graphs = []
    for k in range(2):
        x, dy = torch.zeros_like(data[0][0]), torch.zeros_like(data[0][1])
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = step(x, dy)
        graphs.append((g, x, dy, res, torch.cuda.Stream()))
    for turn in range(2):
        for k, (g, x, dy, res, s) in enumerate(graphs):
            src = data[(k + turn) % 2]
            x.copy_(src[0]), dy.copy_(src[1])
        torch.cuda.synchronize()
        for _ in range(4):
            for g, _, _, _, s in graphs:
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for k, (_, _, _, res, _) in enumerate(graphs):
            assert all(torch.equal(a, b) for a, b in zip(res, want[(k + turn) % 2]))
    assert ops.device_status() == 0


def test_block_of_a_transformer_together(sdfl):
    """Norm, projection, gate and their gradients as a training step runs them, from checkpoints alone: against
    the 64-bit chain that uses the same kept values."""
    ops = sdfl.ops
    B, P, C, G, D = 2, 333, 320, 32, 256
    x = inputs((B, P, C), "bfloat16", 90)
    gamma, beta = weights(C, 91)
    w = make((C, 2 * D), "float32", 92, C ** -0.5)
    dout = make((B, P, D), "bfloat16", 93)
    buf = x.cuda()
    h, mean, rstd, kept_x = ops.groupnorm_channels_last_train(buf, gamma.cuda(), beta.cuda(), G, EPS, True, checkpoint=True,
                                                              out=buf)
    ab = (h.float() @ w.cuda()).to(torch.bfloat16)
    y, kept_ab = ops.gelu_multiply_checkpoint(ab)
    d_ab = ops.gelu_multiply_backward(dout.cuda(), kept_ab)
    d_h = (d_ab.float() @ w.cuda().t()).to(torch.bfloat16)
    gx, gg, gb = ops.groupnorm_channels_last_backward(d_h, kept_x, mean, rstd, gamma.cuda(), beta.cuda(), G, True)
    # each stage from the stage before it as it was stored
    from train_util import geglu_backward, geglu_bound, geglu_forward
    want, _, _, terms = gn_forward(x, gamma, beta, G, EPS, True)
    assert_within(h, want, half_step(want, "bfloat16") + 1.1 * K * U * terms, "norm")
    want = geglu_forward(ab.cpu())
    assert_within(y, want, half_step(want, "bfloat16") + geglu_bound(ab.cpu(), "bfloat16"), "gate")
    want, bound = geglu_backward(dout, checkpoint_reference(ab)[2], "bfloat16")
    assert_within(d_ab, want, half_step(want, "bfloat16") + bound, "gate's gradient")
    check_backward((gx, gg, gb), d_h.cpu(), checkpoint_reference(x)[2], mean.cpu(), rstd.cpu(), gamma, beta, G, True, "bfloat16",
                   "norm's gradient")
