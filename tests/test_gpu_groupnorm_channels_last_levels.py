"""Statistics of channels-last tensors whose values lie hundreds of spreads from zero, on every launch path."""
import pytest
import torch

from test_gpu_groupnorm_channels_last import EPS, weights
from train_util import K, U, assert_within, gn_forward, half_step, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,P,C,G", [(2, 37, 30, 10), (2, 60, 1032, 8), (1, 700, 33, 11), (2, 5000, 30, 10), (2, 77, 64, 32),
                                     (2, 300, 128, 32), (1, 33000, 64, 32)])
def test_values_far_from_zero(sdfl, B, P, C, G):
    """The variance is that of the deviations: its error is roundings of itself and the square of the mean's error."""
    gamma, beta = weights(C, 171)
    c = torch.arange(C)
    # most of a group's variance comes from its channels' levels, 1 above and below the group's
    x = make((B, P, C), "float32", 172, std=0.3) + (1 - 2.0 * (c % 2)) + 400.3 * (1 + c // (C // G) % 2)
    y, mean, rstd, _ = sdfl.ops.groupnorm_channels_last_train(x.cuda(), gamma.cuda(), beta.cuda(), G, EPS)
    want, wmean, wrstd, terms = gn_forward(x, gamma, beta, G, EPS, False)
    size = x.double().abs().reshape(B, P, G, C // G).mean(dim=(1, 3))
    assert_within(mean, wmean, K * U * size, "mean")
    assert_within(rstd, wrstd, wrstd * (K * U + (K * U * size * wrstd) ** 2), "rstd")
    if C // G % 4 == 0 or C % 4:                      # elsewhere a vector spans groups
        assert_within(y, want, half_step(want, "float32") + K * U * terms, "y")
