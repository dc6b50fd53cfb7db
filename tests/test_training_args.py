"""Refusals of the channels-last GroupNorm and checkpoint entry points: no device is touched."""
import pytest
import torch

from conftest import load_package

A, B, D, E, F, W = (1 << 24) * 1, (1 << 24) * 2, (1 << 24) * 3, (1 << 24) * 4, (1 << 24) * 5, (1 << 24) * 6
BIG = 1 << 30


def forward(**kw):
    a = dict(x=A, y=B, gamma=D, beta=D, mean=None, rstd=None, codes=None, scales=None, batch=2, channels=64, hw=100, groups=8,
             eps=1e-5, silu=1, dtype=1, ws=W, bytes=BIG)
    assert set(kw) <= set(a)
    a.update(kw)
    return load_package()._capi.lib.sdfl_groupnorm_channels_last_forward(*a.values(), None)


def backward(**kw):
    a = dict(x=A, codes=None, scales=None, dy=B, dx=E, gamma=D, beta=D, mean=F, rstd=F, dgamma=F + 4096, dbeta=F + 8192, batch=2,
             channels=64, hw=100, groups=8, silu=1, dtype=1, ws=W, bytes=BIG)
    assert set(kw) <= set(a)
    a.update(kw)
    return load_package()._capi.lib.sdfl_groupnorm_channels_last_backward(*a.values(), None)


def test_forward_refusals():
    c = load_package()._capi
    assert forward(batch=0) == c.OK and forward(hw=0) == c.OK
    for bad in (dict(dtype=3), dict(dtype=-1), dict(channels=60), dict(channels=0), dict(groups=0), dict(batch=-1), dict(hw=-1),
                dict(eps=-1.0), dict(eps=float("nan"))):
        assert forward(**bad) == c.ERR_INVALID_VALUE, bad
    for bad in (dict(x=None), dict(y=None), dict(gamma=None), dict(beta=None), dict(mean=E), dict(rstd=E), dict(codes=E),
                dict(scales=E)):
        assert forward(**bad) == c.ERR_INVALID_POINTER, bad
    for bad in (dict(y=A + 16), dict(mean=A, rstd=E), dict(mean=E, rstd=B + 64), dict(mean=E, rstd=E), dict(codes=A + 8, scales=E),
                dict(codes=E, scales=B + 1), dict(codes=E, scales=E + 1)):
        assert forward(**bad) == c.ERR_OVERLAP, bad
    for bad in (dict(ws=None), dict(bytes=0), dict(ws=W + 8), dict(bytes=16)):
        assert forward(**bad) == c.ERR_WORKSPACE, bad
    assert forward(hw=1 << 31) == c.ERR_UNSUPPORTED


def test_backward_refusals():
    c = load_package()._capi
    for bad in (dict(dtype=3), dict(channels=60), dict(groups=0), dict(batch=-1), dict(codes=W, scales=W + (1 << 23))):
        assert backward(**bad) == c.ERR_INVALID_VALUE, bad
    for bad in (dict(x=None), dict(dy=None), dict(dx=None), dict(mean=None), dict(rstd=None), dict(x=None, codes=A),
                dict(x=None, scales=A), dict(gamma=None), dict(beta=None)):
        assert backward(**bad) == c.ERR_INVALID_POINTER, bad
    for bad in (dict(dx=A + 16), dict(dx=B + 16), dict(x=None, codes=E, scales=A), dict(x=None, codes=A, scales=E + 5),
                dict(dgamma=E), dict(dbeta=B), dict(dgamma=A + 4), dict(dgamma=D), dict(dbeta=F + 4096)):
        assert backward(**bad) == c.ERR_OVERLAP, bad
    for bad in (dict(ws=None), dict(bytes=0), dict(ws=W + 4)):
        assert backward(**bad) == c.ERR_WORKSPACE, bad


def test_checkpoint_refusals():
    c = load_package()._capi
    lib = c.lib
    assert lib.sdfl_checkpoint_pack(A, B, D, 0, 64, 2, None) == c.OK
    assert lib.sdfl_checkpoint_pack(A, B, D, 4, 0, 2, None) == c.OK
    assert lib.sdfl_checkpoint_pack(A, B, D, 4, 64, 3, None) == c.ERR_INVALID_VALUE
    assert lib.sdfl_checkpoint_pack(A, B, D, -4, 64, 1, None) == c.ERR_INVALID_VALUE
    assert lib.sdfl_checkpoint_pack(A, B, D, 4, 1 << 31, 1, None) == c.ERR_UNSUPPORTED
    assert lib.sdfl_checkpoint_pack(A, None, D, 4, 64, 1, None) == c.ERR_INVALID_POINTER
    assert lib.sdfl_checkpoint_pack(A, B, None, 4, 64, 1, None) == c.ERR_INVALID_POINTER
    assert lib.sdfl_checkpoint_pack(A, A, D, 4, 64, 1, None) == c.ERR_OVERLAP
    assert lib.sdfl_checkpoint_pack(A, B, B + 255, 4, 64, 1, None) == c.ERR_OVERLAP
    assert lib.sdfl_checkpoint_unpack(B, D, None, 4, 64, 1, None) == c.ERR_INVALID_POINTER
    assert lib.sdfl_checkpoint_unpack(B, D, B, 4, 64, 1, None) == c.ERR_OVERLAP
    assert lib.sdfl_checkpoint_unpack(B, D, D - 511, 4, 64, 1, None) == c.ERR_OVERLAP
    assert lib.sdfl_gelu_multiply_checkpoint(A, B, D, None, 4, 64, 1, None) == c.ERR_INVALID_POINTER
    assert lib.sdfl_gelu_multiply_checkpoint(A, A, D, E, 4, 64, 1, None) == c.ERR_OVERLAP
    assert lib.sdfl_gelu_multiply_checkpoint(A, B, B, E, 4, 64, 1, None) == c.ERR_OVERLAP
    assert lib.sdfl_gelu_multiply_checkpoint(A, B, D, E, 4, -64, 1, None) == c.ERR_INVALID_VALUE
    assert lib.sdfl_gelu_multiply_backward(A, D, E, B, F, 4, 64, 1, None) == c.ERR_INVALID_VALUE
    assert lib.sdfl_gelu_multiply_backward(None, None, None, B, F, 4, 64, 1, None) == c.ERR_INVALID_POINTER
    assert lib.sdfl_gelu_multiply_backward(None, D, None, B, F, 4, 64, 1, None) == c.ERR_INVALID_POINTER
    assert lib.sdfl_gelu_multiply_backward(A, None, None, B, B, 4, 64, 1, None) == c.ERR_OVERLAP
    assert lib.sdfl_gelu_multiply_backward(A, None, None, B, A + 16, 4, 64, 1, None) == c.ERR_OVERLAP
    assert lib.sdfl_gelu_multiply_backward(None, D, E, B, D, 4, 64, 1, None) == c.ERR_OVERLAP


def test_bf16_stays_with_the_new_entry_points():
    c = load_package()._capi
    assert c.lib.sdfl_silu(A, B, 64, 2, None) == c.ERR_INVALID_VALUE
    assert c.lib.sdfl_groupnorm_forward(A, B, D, D, 1, 32, 64, 32, 1e-5, 1, 2, None, 0, None) == c.ERR_INVALID_VALUE


def test_workspace_query():
    q = load_package()._capi.lib.sdfl_groupnorm_channels_last_workspace_bytes
    assert q(2, 60, 100, 8, 0, 1) == 0 and q(0, 64, 100, 8, 0, 1) == 0 and q(2, 64, 100, 8, 0, 9) == 0
    assert q(2, 64, 100, 8, 1, 2) >= 0


def test_python_checks_need_no_device():
    ops = load_package().ops
    x = torch.zeros((2, 10, 64), dtype=torch.float16)
    w = torch.ones(64)
    with pytest.raises(TypeError):
        ops.groupnorm_channels_last(x, w, w, 8)
    with pytest.raises(TypeError):
        ops.checkpoint_pack(x)
    with pytest.raises(TypeError):
        ops.checkpoint_pack(x.double())
    with pytest.raises(TypeError):
        ops.Checkpoint8(x, torch.zeros((2, 10, 2), dtype=torch.uint8), torch.float16)
    with pytest.raises(TypeError):
        ops.Checkpoint8(x.to(torch.int8), torch.zeros((2, 10, 2), dtype=torch.uint8), torch.float64)
    with pytest.raises(ValueError):
        ops.Checkpoint8(x.to(torch.int8), torch.zeros((2, 10, 3), dtype=torch.uint8), torch.float16)
    kept = ops.Checkpoint8(x.to(torch.int8), torch.zeros((2, 10, 2), dtype=torch.uint8), torch.float16)
    assert kept.shape == x.shape and kept.nbytes == 2 * 10 * 66
    with pytest.raises(TypeError):
        ops.checkpoint_unpack(kept)
    with pytest.raises(TypeError):
        ops.gelu_multiply_backward(x, kept)


@pytest.mark.gpu
def test_python_refusals_on_the_device():
    ops = load_package().ops
    x = torch.zeros((2, 10, 64), dtype=torch.float16, device="cuda")
    w, w2 = torch.ones(64, device="cuda"), torch.ones(32, device="cuda")
    kept = ops.checkpoint_pack(x)
    st = torch.ones((2, 8), device="cuda")
    for call in (lambda: ops.groupnorm_channels_last(x.transpose(1, 2), w, w, 8),
                 lambda: ops.groupnorm_channels_last(x, w2, w, 8),
                 lambda: ops.groupnorm_channels_last(x, w, w, 8, out=torch.empty_like(x, dtype=torch.float32)),
                 lambda: ops.groupnorm_channels_last_train(x, w, w, 8, out=x),
                 lambda: ops.groupnorm_channels_last_backward(x, kept, st[:1], st, w, w, 8),
                 lambda: ops.groupnorm_channels_last_backward(x.float(), kept, st, st, w, w, 8),
                 lambda: ops.groupnorm_channels_last_backward(x[:1].contiguous(), x, st, st, w, w, 8),
                 lambda: ops.gelu_multiply_backward(x, kept),
                 lambda: ops.gelu_multiply_checkpoint(x[..., :33].contiguous()),
                 lambda: ops.checkpoint_unpack(kept, out=x[:1].contiguous())):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(ops.SdflError):
        ops.groupnorm_channels_last(x, w, w, 7)
    with pytest.raises(TypeError):
        ops.groupnorm_channels_last(x, w.half(), w, 8)
    with pytest.raises(TypeError):
        ops.groupnorm_channels_last(x, w.cpu(), w, 8)
