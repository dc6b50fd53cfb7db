"""64-bit definitions and error bounds for the channels-last GroupNorm, the 8-bit checkpoints and their
gradients.

Bounds.  U = 2^-24 is half a step of fp32.  A result stored in type t is off by at most half a step of t
(finfo(t).eps / 2 relative, or half the smallest subnormal) on top of the fp32 arithmetic, which is counted as
K roundings of the terms it adds up.  A thread adds up its rows one after another, 136 at most in the shapes that
are tested here (hw / (thread blocks of a team * rows of threads) in general); the roundings of such a run have either
sign, so n of them come to about sqrt(n), 12 here.  Trees over threads, blocks and channels have 20 levels at most,
and an expression per element takes fewer than 12 operations: 44 in all, K = 64.  It is a bound for rounding
errors as they occur, not for all of them at their largest with one sign.
"""
from __future__ import annotations

import numpy as np
import torch

DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
U = 2.0 ** -24
K = 64


def make(shape, dtype: str, seed: int, std: float = 1.0, mean: float = 0.0) -> torch.Tensor:
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g, dtype=torch.float64) * std + mean).to(DTYPES[dtype])


def half_step(want: torch.Tensor, dtype: str) -> torch.Tensor:
    fi = torch.finfo(DTYPES[dtype])
    return want.abs() * (fi.eps / 2) + fi.smallest_normal * fi.eps / 2


def assert_within(got: torch.Tensor, want: torch.Tensor, bound: torch.Tensor, what: str) -> None:
    got = got.detach().cpu().double()
    want, bound = want.cpu(), bound.cpu()
    assert got.shape == want.shape, f"{what}: {tuple(got.shape)} for {tuple(want.shape)}"
    assert torch.isfinite(got).all(), f"{what}: non-finite values"
    err = (got - want).abs()
    ratio = (err / bound.clamp(min=1e-300)).max().item() if err.numel() else 0.0
    assert ratio <= 1.0, f"{what}: error {ratio:.3f} x bound (largest error {err.max().item():.3e})"


def checkpoint_reference(x: torch.Tensor):
    """(codes, scales, values) by the definition, block by block in numpy float64."""
    dim = x.shape[-1]
    rows = x.reshape(-1, dim).cpu().double().numpy()
    nb = -(-dim // 32)
    codes = np.zeros(rows.shape, np.int8)
    scales = np.zeros((rows.shape[0], nb), np.uint8)
    values = np.zeros(rows.shape, np.float64)
    for b in range(nb):
        v = rows[:, 32 * b:32 * b + 32]
        with np.errstate(invalid="ignore"):
            a = np.abs(v).max(axis=1)
        bad = ~np.isfinite(v).all(axis=1)
        a = np.where(bad, 1.0, a)
        e = np.where(a > 0, np.frexp(a)[1] - 1, -1000)          # floor(log2 a)
        p = np.maximum(e - 6, -120)
        step = np.ldexp(1.0, p)
        q = np.clip(np.rint(np.where(bad[:, None], 0.0, v) / step[:, None]), -127, 127)
        codes[:, 32 * b:32 * b + 32] = q
        scales[:, b] = np.where(bad, 255, p + 127)
        values[:, 32 * b:32 * b + 32] = np.where(bad[:, None], np.nan, q * step[:, None])
    shape = tuple(x.shape)
    return (torch.from_numpy(codes).view(shape), torch.from_numpy(scales).view(shape[:-1] + (nb,)),
            torch.from_numpy(values).view(shape))


def gn_forward(x, gamma, beta, G, eps, silu):
    """y, mean, rstd, and the size of the terms that z is made of."""
    B, C = x.shape[0], x.shape[-1]
    v = x.double().reshape(B, -1, G, C // G)
    mean = v.mean(dim=(1, 3))
    var = (v - mean[:, None, :, None]).pow(2).mean(dim=(1, 3))
    rstd = 1.0 / torch.sqrt(var + eps)
    n = ((v - mean[:, None, :, None]) * rstd[:, None, :, None]).reshape(B, -1, C)
    z = n * gamma.double() + beta.double()
    terms = gamma.double().abs() * (n.abs() + (mean.abs() * rstd).repeat_interleave(C // G, 1)[:, None, :]) \
        + beta.double().abs() + 1.0
    y = z / (1 + torch.exp(-z)) if silu else z
    return y.reshape(x.shape), mean, rstd, terms.reshape(x.shape)


def gn_backward(dy, x, mean, rstd, gamma, beta, G, silu):
    """(dx, dgamma, dbeta) and their bounds in fp32 arithmetic (without the final rounding of dx)."""
    B, C = x.shape[0], x.shape[-1]
    W = C // G
    xv, d = x.double().reshape(B, -1, C), dy.double().reshape(B, -1, C)
    P = xv.shape[1]
    g, b = gamma.double(), beta.double()
    mu = mean.double().repeat_interleave(W, 1)[:, None, :]
    rs = rstd.double().repeat_interleave(W, 1)[:, None, :]
    n = (xv - mu) * rs
    z = n * g + b
    terms = g.abs() * (n.abs() + mu.abs() * rs) + b.abs() + 1.0
    if silu:
        s = 1 / (1 + torch.exp(-z))
        dz = d * (s + z * s * (1 - s))
    else:
        dz = d
    # |act''| <= 1/2 and |act'| <= 1.1: an error U * terms in z, and the roundings of dz itself
    size = d.abs() * (1.1 + (terms if silu else 0.0))
    nsize = n.abs() + mu.abs() * rs + 1.0

    def per_group(t):
        return (t.reshape(B, P, G, W).sum(dim=(1, 3)) / (P * W)).repeat_interleave(W, 1)[:, None, :]

    m1, m2 = per_group(dz * g), per_group(dz * g * n)
    dx = rs * (dz * g - m1 - n * m2)
    bx = K * U * rs * (size * g.abs() + per_group(size * g.abs()) + nsize * per_group(size * g.abs() * nsize))
    dg, bg = (dz * n).sum(dim=(0, 1)), K * U * (size * nsize).sum(dim=(0, 1))
    db, bb = dz.sum(dim=(0, 1)), K * U * size.sum(dim=(0, 1))
    return (dx.reshape(x.shape), dg, db), (bx.reshape(x.shape), bg, bb)


def geglu_forward(ab):
    a, g = ab.double().chunk(2, dim=-1)
    return a * g * torch.special.ndtr(g)


# Half storage takes erf from a rational approximation: |error| <= 1.5e-7 (Abramowitz and Stegun 7.1.26)
# plus its own roundings, 1e-6 in all, on erf; half of that on Phi.
def geglu_bound(ab, dtype):
    a, g = ab.double().chunk(2, dim=-1)
    return a.abs() * g.abs() * (K * U + (0 if dtype == "float32" else 5e-7))


def geglu_backward(dy, ab, dtype):
    a, g = ab.double().chunk(2, dim=-1)
    d = dy.double()
    cdf = torch.special.ndtr(g)
    pdf = torch.exp(-g * g / 2) / np.sqrt(2 * np.pi)
    approx = K * U + (0 if dtype == "float32" else 5e-7)
    want = torch.cat([d * g * cdf, d * a * (cdf + g * pdf)], dim=-1)
    bound = torch.cat([(d * g).abs() * approx, (d * a).abs() * approx * (1 + g.abs())], dim=-1)
    return want, bound
