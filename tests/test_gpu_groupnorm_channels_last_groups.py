"""Channels-last GroupNorm: a group's results come from its own values alone, where the 16-byte vectors of a
row span groups (widths 2, 3, 4 and 10) and where they do not."""
import pytest
import torch

from test_gpu_groupnorm_channels_last import ALL, EPS, check_backward, check_forward, inputs, weights
from train_util import K, U, assert_within, checkpoint_reference, make

pytestmark = pytest.mark.gpu

# batch, pixels, channels, groups; clusters, teams, and (the last two) the launches for any shape
SHAPES = [(2, 64, 320, 32), (2, 300, 128, 32), (2, 77, 64, 32), (3, 50, 48, 16), (1, 33000, 64, 32), (2, 16384, 128, 32),
          (1, 40000, 320, 32), (2, 4096, 320, 8), (2, 300, 1032, 8), (2, 37, 30, 10)]


def same_elsewhere(got, want, group, G, what):
    """Equal bits in every channel outside the group."""
    C = want.shape[-1]
    keep = torch.ones(C, dtype=torch.bool, device=want.device)
    keep[group * (C // G):(group + 1) * (C // G)] = False
    assert torch.isfinite(want).all()
    assert torch.equal(got[..., keep], want[..., keep]), what


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("B,P,C,G", SHAPES)
def test_other_groups_keep_their_bits(sdfl, B, P, C, G, dtype):
    """One group shifted far away, or with an infinity or a NaN: the others' results do not change."""
    ops = sdfl.ops
    W = C // G
    x, dy = inputs((B, P, C), dtype, 101).cuda(), make((B, P, C), dtype, 102).cuda()
    gamma, beta = (t.cuda() for t in weights(C, 103))
    y, mean, rstd, _ = ops.groupnorm_channels_last_train(x, gamma, beta, G, EPS, True)
    kept = ops.checkpoint_pack(x)
    grads = ops.groupnorm_channels_last_backward(dy, x, mean, rstd, gamma, beta, G, True)
    kept_grads = ops.groupnorm_channels_last_backward(dy, kept, mean, rstd, gamma, beta, G, True)
    for turn, value in enumerate((1000.0, float("inf"), float("nan"))):
        k = (0, G // 2, G - 2)[turn]                  # the first group of a vector among them
        far = x.clone()
        if turn == 0:
            far[..., k * W:(k + 1) * W] += value
        else:
            far[B - 1, P // 2, k * W] = value
        out, m, r, _ = ops.groupnorm_channels_last_train(far, gamma, beta, G, EPS, True)
        same_elsewhere(out, y, k, G, f"y, {value}")
        for a, b, what in zip(ops.groupnorm_channels_last_backward(dy, far, m, r, gamma, beta, G, True), grads,
                              ("grad_x", "grad_gamma", "grad_beta")):
            same_elsewhere(a, b, k, G, f"{what}, {value}")
        # the same from a checkpoint, whose blocks are shared: here it is the group's mean that is far off
        m = mean.clone()
        m[:, k] = value
        for a, b, what in zip(ops.groupnorm_channels_last_backward(dy, kept, m, rstd, gamma, beta, G, True), kept_grads,
                              ("grad_x", "grad_gamma", "grad_beta")):
            same_elsewhere(a, b, k, G, f"{what} from a checkpoint, {value}")


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("B,P,C,G", SHAPES)
def test_levels_that_differ_from_group_to_group(sdfl, B, P, C, G, dtype):
    """Every other group a thousand spreads away from its neighbours, against the definition."""
    ops = sdfl.ops
    x = inputs((B, P, C), dtype, 111).double()
    x = (x + 1000.0 * (torch.arange(C) // (C // G) % 2)).to(x.dtype).to(getattr(torch, dtype))
    dy = make((B, P, C), dtype, 112)
    gamma, beta = weights(C, 113)
    y, mean, rstd, kept = ops.groupnorm_channels_last_train(x.cuda(), gamma.cuda(), beta.cuda(), G, EPS, False, checkpoint=True)
    wmean, wrstd = check_forward(y, x, gamma, beta, G, False, dtype, "forward")
    size = x.double().abs().reshape(B, P, G, C // G).mean(dim=(1, 3))
    assert_within(mean, wmean, K * U * size + 1e-30, "mean")
    assert_within(rstd, wrstd, wrstd * (K * U + (K * U * size * wrstd) ** 2), "rstd")
    for source, values in ((x.cuda(), x), (kept, checkpoint_reference(x)[2])):
        got = ops.groupnorm_channels_last_backward(dy.cuda(), source, mean, rstd, gamma.cuda(), beta.cuda(), G)
        check_backward(got, dy, values, mean.cpu(), rstd.cpu(), gamma, beta, G, False, dtype, "backward")
