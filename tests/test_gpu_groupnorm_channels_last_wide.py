"""Backward pass of the channels-last GroupNorm from a checkpoint with slices of 640 channels and neighbouring widths."""
import pytest
import torch

from test_gpu_groupnorm_channels_last import EPS, check_backward, inputs, weights
from train_util import checkpoint_reference, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("B,P,C,G", [(4, 4096, 640, 1), (2, 4096, 1280, 2), (1, 4096, 2560, 4), (1, 3001, 3200, 25),
                                     (1, 6000, 1920, 3), (2, 4096, 512, 1), (2, 3000, 768, 1), (2, 3000, 1024, 1)])
def test_wide_groups_from_a_checkpoint(sdfl, B, P, C, G, dtype):
    ops = sdfl.ops
    x, dy = inputs((B, P, C), dtype, 161), make((B, P, C), dtype, 162)
    gamma, beta = weights(C, 163)
    _, mean, rstd, kept = ops.groupnorm_channels_last_train(x.cuda(), gamma.cuda(), beta.cuda(), G, EPS, True, checkpoint=True)
    got = ops.groupnorm_channels_last_backward(dy.cuda(), kept, mean, rstd, gamma.cuda(), beta.cuda(), G, True)
    check_backward(got, dy, checkpoint_reference(x)[2], mean.cpu(), rstd.cpu(), gamma, beta, G, True, dtype, "checkpoint")
    got = ops.groupnorm_channels_last_backward(dy.cuda(), x.cuda(), mean, rstd, gamma.cuda(), beta.cuda(), G, True)
    check_backward(got, dy, x, mean.cpu(), rstd.cpu(), gamma, beta, G, True, dtype, "tensor")
    assert ops.device_status() == 0
