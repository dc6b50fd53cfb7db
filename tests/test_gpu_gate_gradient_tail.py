"""The gate's gradient for very negative gates, where Phi(g) is far below 1."""
import numpy as np
import pytest
import torch

from gpu_util import Guarded
from train_util import DTYPES, K, U, assert_within, checkpoint_reference, half_step, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("D", [64, 61])
def test_relative_error_in_the_tail(sdfl, D, dtype):
    """g from -2 to -12.  A relative rounding U of g/sqrt(2) changes Phi and phi by about g^2 U of themselves,
    everything else is K roundings of them."""
    rows = 50
    ab = make((rows, 2 * D), "float32", 151)
    ab[:, D:] = -(2 + 10 * torch.rand((rows, D), generator=torch.Generator().manual_seed(152)))
    ab, dy = ab.to(DTYPES[dtype]), make((rows, D), dtype, 153)
    for source, x in ((ab.cuda(), ab), (sdfl.ops.checkpoint_pack(ab.cuda()), checkpoint_reference(ab)[2])):
        out = Guarded(tuple(ab.shape), DTYPES[dtype])
        got = sdfl.ops.gelu_multiply_backward(dy.cuda(), source, out=out.tensor)
        out.check()
        a, g = x.double().chunk(2, dim=-1)
        d = dy.double()
        cdf, pdf = torch.special.erfc(-g / np.sqrt(2.0)) / 2, torch.exp(-g * g / 2) / np.sqrt(2 * np.pi)
        want = torch.cat([d * g * cdf, d * a * (cdf + g * pdf)], dim=-1)
        rel = (K + 2 * g * g) * U
        bound = torch.cat([(d * g).abs() * cdf * rel, (d * a).abs() * (cdf + g.abs() * pdf) * rel], dim=-1) + 1e-37
        assert_within(got, want, half_step(want, dtype) + bound, "gradient")
