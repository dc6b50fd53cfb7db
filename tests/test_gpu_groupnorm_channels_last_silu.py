"""SiLU and its derivative far from zero in the channels-last GroupNorm: z e^z for very negative z, 0 behind that."""
import pytest
import torch

from test_gpu_groupnorm_channels_last import ALL, EPS
from train_util import DTYPES, K, U, assert_within, gn_forward, half_step, make

pytestmark = pytest.mark.gpu

# a cluster, teams, whole vectors in several launches, single elements in several launches
SHAPES = [(2, 300, 64, 8), (1, 33000, 64, 32), (2, 60, 1032, 8), (2, 50, 30, 10)]
# 1 / (1 + e^-z) below 2^-126 counts as 0
FLUSH = 2.0 ** -125


def case(B, P, C, G, dtype, scale, seed):
    x = make((B, P, C), dtype, seed)
    gamma, beta = torch.full((C,), scale), make((C,), "float32", seed + 1)
    return x, gamma, beta


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("B,P,C,G", SHAPES)
def test_forward_tail(sdfl, B, P, C, G, dtype):
    """z down to about -150.  An error e in z changes z s(z) by at most e s (1 + |z|); exp and the reciprocal
    add K roundings of the result."""
    x, gamma, beta = case(B, P, C, G, dtype, 40.0, 121)
    y = sdfl.ops.groupnorm_channels_last(x.cuda(), gamma.cuda(), beta.cuda(), G, EPS, True)
    want, _, _, terms = gn_forward(x, gamma, beta, G, EPS, True)
    z = gn_forward(x, gamma, beta, G, EPS, False)[0]
    s = 1 / (1 + torch.exp(-z))
    bound = half_step(want, dtype) + K * U * (1.01 * terms * s * (1 + z.abs()) + want.abs()) + z.abs() * FLUSH
    assert_within(y, want, bound, "y")


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("B,P,C,G", SHAPES)
def test_backward_tail(sdfl, B, P, C, G, dtype):
    """grad_out only where z < -45, so that the sums are made of the tail alone.  |silu''| <= s (2 + |z|) there."""
    x, gamma, beta = case(B, P, C, G, dtype, 40.0, 131)
    _, mean, rstd, src = sdfl.ops.groupnorm_channels_last_train(x.cuda(), gamma.cuda(), beta.cuda(), G, EPS, True)
    per_channel = lambda t: t.cpu().double().repeat_interleave(C // G, 1)[:, None, :]
    n = (x.double() - per_channel(mean)) * per_channel(rstd)
    z = n * gamma.double() + beta.double()
    dy = make((B, P, C), dtype, 132) * (z < -45)
    s = 1 / (1 + torch.exp(-z))
    dz = dy.double() * s * (1 + z * (1 - s))
    nsize = n.abs() + per_channel(mean).abs() * per_channel(rstd) + 1
    terms = gamma.abs() * nsize + beta.abs() + 1
    err = dy.double().abs() * (K * U * 1.01 * (terms + 1) * s * (2 + z.abs()) + (1 + z.abs()) * FLUSH)
    _, gg, gb = sdfl.ops.groupnorm_channels_last_backward(dy.cuda(), src, mean, rstd, gamma.cuda(), beta.cuda(), G, True)
    assert dz.abs().sum() > 0
    assert_within(gb, dz.sum(dim=(0, 1)), (err + K * U * dz.abs()).sum(dim=(0, 1)) + 1e-37, "grad_beta")
    assert_within(gg, (dz * n).sum(dim=(0, 1)), ((err + K * U * dz.abs()) * nsize).sum(dim=(0, 1)) + 1e-37, "grad_gamma")


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("B,P,C,G", SHAPES)
def test_behind_the_tail(sdfl, B, P, C, G, dtype):
    """z of -10^29 and beyond: 0, not a multiple of z; and no gradient."""
    ops = sdfl.ops
    x, gamma, beta = case(B, P, C, G, dtype, 1e30, 141)
    y, mean, rstd, src = ops.groupnorm_channels_last_train(x.cuda(), gamma.cuda(), beta.cuda(), G, EPS, True)
    z = gn_forward(x, gamma, beta, G, EPS, False)[0]
    below = z < -1e29
    assert below.any() and not y.cpu()[below].any()
    dy = (make((B, P, C), "float32", 142) * below).to(DTYPES[dtype])
    for t in ops.groupnorm_channels_last_backward(dy.cuda(), src, mean, rstd, gamma.cuda(), beta.cuda(), G, True):
        assert not t.any()
