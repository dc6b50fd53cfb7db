"""Arrays that a call of the channels-last GroupNorm writes may not touch any other; no device is touched."""
import pytest

from conftest import load_package
from test_training_args import A, B, D, E, F, W, backward, forward

KEPT = dict(x=None, codes=A, scales=A + (1 << 22))


@pytest.mark.parametrize("bad", [dict(gamma=B + 64), dict(beta=B), dict(mean=D, rstd=E), dict(mean=E, rstd=D + 4),
                                 dict(codes=E, scales=F, mean=E + 128, rstd=E + (1 << 22)), dict(codes=E, scales=F, mean=F, rstd=F + 4096),
                                 dict(codes=D, scales=F), dict(codes=E, scales=D), dict(ws=A), dict(ws=B + 16), dict(ws=D),
                                 dict(mean=W, rstd=E), dict(codes=E, scales=W + 64)])
def test_forward(bad):
    assert forward(**bad) == load_package()._capi.ERR_OVERLAP, bad


@pytest.mark.parametrize("bad", [dict(mean=E), dict(rstd=E + 64), dict(gamma=E), dict(beta=E + 128), dict(dgamma=F),
                                 dict(dbeta=F + 16), dict(dgamma=F + 4096, rstd=F + 4096), dict(KEPT, dgamma=A + 4),
                                 dict(KEPT, dbeta=A + (1 << 22)), dict(ws=A), dict(ws=B), dict(ws=E), dict(ws=D), dict(ws=F),
                                 dict(ws=F + 4096), dict(KEPT, ws=A + 16), dict(KEPT, ws=A + (1 << 22))])
def test_backward(bad):
    assert backward(**bad) == load_package()._capi.ERR_OVERLAP, bad
