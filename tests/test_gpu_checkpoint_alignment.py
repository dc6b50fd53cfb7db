"""Codes at any address through the C ABI: one call each of all entry points that write or read a checkpoint."""
import pytest
import torch

from gpu_util import Guarded
from test_gpu_groupnorm_channels_last import ALL, EPS, check_backward, check_forward, inputs, weights
from train_util import DTYPES, assert_within, checkpoint_reference, geglu_backward, half_step, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("shift", [1, 4, 8])
@pytest.mark.parametrize("B,P,C,G", [(2, 300, 128, 32), (1, 33000, 64, 32)])
def test_norm(sdfl, B, P, C, G, shift, dtype):
    lib, code = sdfl._capi.lib, list(DTYPES).index(dtype)
    x, dy = inputs((B, P, C), dtype, 181), make((B, P, C), dtype, 182)
    gamma, beta = weights(C, 183)
    xd, dyd, g, b = x.cuda(), dy.cuda(), gamma.cuda(), beta.cuda()
    y, dx = torch.empty_like(xd), torch.empty_like(xd)
    mean, rstd = torch.empty((B, G), device="cuda"), torch.empty((B, G), device="cuda")
    dg, db = torch.empty_like(g), torch.empty_like(b)
    codes, scales = Guarded((B * P * C,), torch.int8, shift), Guarded((B * P * C // 32,), torch.uint8, shift)
    ws = torch.empty(max(lib.sdfl_groupnorm_channels_last_workspace_bytes(B, C, P, G, k, code) for k in (0, 1)), dtype=torch.uint8,
                     device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    at = [t.data_ptr() for t in (codes.tensor, scales.tensor)]
    assert at[0] % 16 == shift
    assert lib.sdfl_groupnorm_channels_last_forward(xd.data_ptr(), y.data_ptr(), g.data_ptr(), b.data_ptr(), mean.data_ptr(),
                                                    rstd.data_ptr(), *at, B, C, P, G, EPS, 1, code, ws.data_ptr(), ws.numel(),
                                                    stream) == 0
    codes.check(), scales.check()
    check_forward(y, x, gamma, beta, G, True, dtype, "forward")
    want_codes, want_scales, values = checkpoint_reference(x)
    assert torch.equal(codes.tensor.cpu(), want_codes.flatten()) and torch.equal(scales.tensor.cpu(), want_scales.flatten())
    assert lib.sdfl_groupnorm_channels_last_backward(None, *at, dyd.data_ptr(), dx.data_ptr(), g.data_ptr(), b.data_ptr(),
                                                     mean.data_ptr(), rstd.data_ptr(), dg.data_ptr(), db.data_ptr(), B, C, P, G, 1,
                                                     code, ws.data_ptr(), ws.numel(), stream) == 0
    check_backward((dx, dg, db), dy, values, mean.cpu(), rstd.cpu(), gamma, beta, G, True, dtype, "backward")


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("shift", [1, 4, 8])
@pytest.mark.parametrize("D", [64, 40, 33])
def test_gate_and_pack(sdfl, D, shift, dtype):
    lib, code, rows = sdfl._capi.lib, list(DTYPES).index(dtype), 37
    ab, dy = make((rows, 2 * D), dtype, 191), make((rows, D), dtype, 192)
    abd, dyd = ab.cuda(), dy.cuda()
    y, dab, back = torch.empty_like(dyd), torch.empty_like(abd), torch.empty_like(abd)
    want_codes, want_scales, values = checkpoint_reference(ab)
    stream = torch.cuda.current_stream().cuda_stream
    for pack in (False, True):
        codes = Guarded((rows * 2 * D,), torch.int8, shift)
        scales = Guarded((want_scales.numel(),), torch.uint8, shift)
        at = [t.data_ptr() for t in (codes.tensor, scales.tensor)]
        if pack:
            assert lib.sdfl_checkpoint_pack(abd.data_ptr(), *at, rows, 2 * D, code, stream) == 0
        else:
            assert lib.sdfl_gelu_multiply_checkpoint(abd.data_ptr(), y.data_ptr(), *at, rows, D, code, stream) == 0
        codes.check(), scales.check()
        assert torch.equal(codes.tensor.cpu(), want_codes.flatten()) and torch.equal(scales.tensor.cpu(), want_scales.flatten())
    assert lib.sdfl_checkpoint_unpack(*at, back.data_ptr(), rows, 2 * D, code, stream) == 0
    assert torch.equal(back.cpu().double(), values)
    assert lib.sdfl_gelu_multiply_backward(None, *at, dyd.data_ptr(), dab.data_ptr(), rows, D, code, stream) == 0
    want, bound = geglu_backward(dy, values, dtype)
    assert_within(dab, want, half_step(want, dtype) + bound, "gradient")
