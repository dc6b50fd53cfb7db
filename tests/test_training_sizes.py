"""Sizes beyond what the training entry points support: refused before any arithmetic overflows; no device is touched."""
import os
import subprocess
import sys

from conftest import ROOT, load_package

A, B, D, E, W = ((1 << 24) * k for k in (1, 2, 3, 4, 6))


SHAPES = [(8, 8, 1 << 61, 8), (1 << 61, 8, 8, 8), (1, 1 << 32, 1 << 32, 1), (1 << 40, 64, 1 << 30, 8), (1, 8, 1 << 31, 1),
          (1 << 27, 8, 1, 1)]


def test_workspace_query_of_impossible_shapes():
    """In a process of its own: a division by an overflowed product would end it."""
    load_package()
    code = ("from conftest import load_package\n"
            "q = load_package()._capi.lib.sdfl_groupnorm_channels_last_workspace_bytes\n"
            f"print([q(*s, b, t) for s in {SHAPES} for b in (0, 1) for t in (0, 1, 2)])\n")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=os.path.join(ROOT, "tests"), timeout=300)
    assert r.returncode == 0, r.returncode
    assert r.stdout.strip() == str([0] * 6 * len(SHAPES))


def test_norm_of_impossible_shapes():
    c = load_package()._capi
    for batch, channels, hw, groups in [(1 << 60, 16, 1, 16), (1 << 61, 8, 8, 8), (1 << 27, 8, 1, 1)]:
        assert c.lib.sdfl_groupnorm_channels_last_forward(A, B, D, D, None, None, None, None, batch, channels, hw, groups, 1e-5, 1,
                                                          1, W, 1 << 30, None) == c.ERR_UNSUPPORTED
        assert c.lib.sdfl_groupnorm_channels_last_backward(A, None, None, B, E, D, D, D, D, None, None, batch, channels, hw,
                                                           groups, 1, 1, W, 1 << 30, None) == c.ERR_UNSUPPORTED


def test_checkpoints_of_impossible_shapes():
    c = load_package()._capi
    for rows, dim in [(1 << 39, 1 << 30), (1 << 38, 1 << 26), ((1 << 40) - 1, (1 << 31) - 1), (1 << 32, 1 << 30)]:
        for dtype in (0, 1, 2):
            assert c.lib.sdfl_checkpoint_pack(A, B, D, rows, dim, dtype, None) == c.ERR_UNSUPPORTED
            assert c.lib.sdfl_checkpoint_unpack(A, B, D, rows, dim, dtype, None) == c.ERR_UNSUPPORTED
            assert c.lib.sdfl_gelu_multiply_checkpoint(A, B, D, E, rows, dim, dtype, None) == c.ERR_UNSUPPORTED
            assert c.lib.sdfl_gelu_multiply_backward(A, None, None, B, D, rows, dim, dtype, None) == c.ERR_UNSUPPORTED
