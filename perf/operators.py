"""Measured cases of the channels-last GroupNorm(+SiLU) with its gradient and of the 8-bit activation
checkpoints with the backward passes that read them.

Kinds of case (`kind`):
  gn          y = act(GroupNorm(x)), x channels last [batch, hw, channels]
  gn_bwd      gradients of x, gamma and beta from grad_out, the saved statistics and x or its checkpoint
  gn_train    forward that keeps an 8-bit checkpoint of x, then the backward pass that reads it
  checkpoint  an activation packed to 8 bits and expanded again
  geglu_train value * gelu(gate) with a checkpoint of the projection, then its gradient from that checkpoint
  geglu_bwd   the gradient of value * gelu(gate) from grad_out and the projection or its checkpoint

A checkpoint holds rows of `dim` elements in blocks of 32 along the row (the last block of a row may be
shorter): one signed byte per element and one exponent byte per block.
"""
import importlib
import math

import torch

own = False

DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
BLOCK = 32
EPS = 1e-5


def listed():
    return [
        # deepest level of the UNet, guidance pair: the smallest norm of a sampling step
        {"name": "gn_8x8x1280_f16", "kind": "gn", "batch": 2, "hw": 64, "channels": 1280, "groups": 32,
         "silu": True, "dtype": "float16"},
        # first level of the UNet, guidance pair
        {"name": "gn_64x64x320_f16", "kind": "gn", "batch": 2, "hw": 4096, "channels": 320, "groups": 32,
         "silu": True, "dtype": "float16"},
        # last level of the VAE decoder, a batch of four images
        {"name": "gn_512x512x128_f16", "kind": "gn", "batch": 4, "hw": 512 * 512, "channels": 128, "groups": 32,
         "silu": True, "dtype": "float16"},
        # norm in front of a spatial transformer (no activation) at an odd image size
        {"name": "gn_47x63x640_f32", "kind": "gn", "batch": 3, "hw": 47 * 63, "channels": 640, "groups": 32,
         "silu": False, "dtype": "float32"},
        # backward at the second level of the UNet, activations kept whole
        {"name": "gn_bwd_32x32x640_bf16", "kind": "gn_bwd", "source": "tensor", "batch": 4, "hw": 1024,
         "channels": 640, "groups": 32, "silu": True, "dtype": "bfloat16"},
        # backward at the decoder's 256 x 256 level from 8-bit checkpoints
        {"name": "gn_bwd_256x256x256_ckpt_bf16", "kind": "gn_bwd", "source": "checkpoint", "batch": 4,
         "hw": 256 * 256, "channels": 256, "groups": 32, "silu": True, "dtype": "bfloat16"},
        # a training step of one norm of the decoder's 128 x 128 level: forward with checkpoint, backward from it
        {"name": "gn_train_128x128x512_f16", "kind": "gn_train", "batch": 4, "hw": 128 * 128, "channels": 512,
         "groups": 32, "silu": True, "dtype": "float16"},
        # a transformer block's input kept in 8 bits
        {"name": "checkpoint_32768x320_bf16", "kind": "checkpoint", "rows": 8 * 4096, "dim": 320,
         "dtype": "bfloat16"},
        # rows that are not whole blocks nor whole vectors
        {"name": "checkpoint_1155x1003_f32", "kind": "checkpoint", "rows": 1155, "dim": 1003, "dtype": "float32"},
        # feed-forward gate of the UNet's first level, training step
        {"name": "geglu_train_16384x1280_f16", "kind": "geglu_train", "rows": 4 * 4096, "dim": 1280,
         "dtype": "float16"},
        # the same at the deepest level: few rows, wide
        {"name": "geglu_train_128x5120_f32", "kind": "geglu_train", "rows": 128, "dim": 5120, "dtype": "float32"},
        # backward of the gate from the whole projection, large batch
        {"name": "geglu_bwd_65536x1280_bf16", "kind": "geglu_bwd", "source": "tensor", "rows": 16 * 4096,
         "dim": 1280, "dtype": "bfloat16"},
    ]


MAX_ELEMENTS = 1 << 26          # of a drawn case's largest tensor


def draw(rng):
    kind = rng.choice(["gn", "gn", "gn_bwd", "gn_bwd", "gn_train", "checkpoint", "geglu_train", "geglu_bwd"])
    dtype = rng.choice(["float32", "float16", "bfloat16"])

    def logint(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    if kind.startswith("gn"):
        groups = rng.choice([8, 16, 32, 32])
        channels = groups * rng.choice([1, 2, 4, 8, 10, 12, 16, 20, 30, 40])
        batch = rng.randint(1, 8)
        hw = logint(16, max(17, min(512 * 512, MAX_ELEMENTS // (batch * channels))))
        case = {"kind": kind, "batch": batch, "hw": hw, "channels": channels, "groups": groups,
                "silu": rng.random() < 0.75, "dtype": dtype}
    elif kind == "checkpoint":
        dim = logint(33, 8192)
        case = {"kind": kind, "rows": logint(16, MAX_ELEMENTS // dim), "dim": dim, "dtype": dtype}
    else:
        dim = logint(64, 5120)
        dim = max(1, dim // 64) * 64 if rng.random() < 0.7 else dim     # mostly whole blocks, some odd
        case = {"kind": kind, "rows": logint(16, MAX_ELEMENTS // (2 * dim)), "dim": dim, "dtype": dtype}
    if kind in ("gn_bwd", "geglu_bwd"):
        case["source"] = rng.choice(["tensor", "checkpoint"])
    return case


# ---- inputs --------------------------------------------------------------------------------------

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(gen, shape, dtype, std=1.0):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).mul_(std).to(dtype)


def _power_of_two(exponent):
    """2^exponent as float32, exactly (exponents of normal numbers)."""
    return ((exponent.to(torch.int32) + 127) << 23).view(torch.float32)


def _pack(x):
    """Codes (int8) and exponent bytes (uint8) of a checkpoint of x, made with elementary operations."""
    dim = x.shape[-1]
    rows = x.numel() // dim
    blocks = -(-dim // BLOCK)
    padded = torch.zeros((rows, blocks * BLOCK), dtype=torch.float32, device=x.device)
    padded[:, :dim] = x.reshape(rows, dim)
    padded = padded.view(rows, blocks, BLOCK)
    amax = padded.abs().amax(dim=2)
    exponent = torch.frexp(amax).exponent - 7                # amax in [2^(k-1), 2^k): step = 2^(k-1-6)
    exponent = torch.where(amax == 0, torch.full_like(exponent, -120), exponent).clamp_(min=-120)
    step = _power_of_two(exponent)
    finite = torch.isfinite(amax)
    codes = torch.round(padded / step[..., None]).clamp_(-127, 127)
    codes = torch.where(finite[..., None], codes, torch.zeros_like(codes))
    scales = torch.where(finite, exponent + 127, torch.full_like(exponent, 255))
    codes = codes.view(rows, blocks * BLOCK)[:, :dim].to(torch.int8).contiguous()
    return codes.view(x.shape), scales.to(torch.uint8).view(*x.shape[:-1], blocks)


def _expand(codes, scales):
    """The float32 values that a checkpoint stands for."""
    dim = codes.shape[-1]
    e = scales.to(torch.int32)
    step = torch.where(e == 255, torch.full_like(e, float("nan"), dtype=torch.float32), _power_of_two(e - 127))
    return codes.float() * step.repeat_interleave(BLOCK, dim=-1)[..., :dim]


def prepare(case, seed):
    gen = _generator(seed)
    kind, dtype = case["kind"], DTYPES[case["dtype"]]
    state = {"case": case}
    if kind.startswith("gn"):
        B, P, C, G = case["batch"], case["hw"], case["channels"], case["groups"]
        # activations of a residual stream: every channel with a level and a spread of its own
        level = _normal(gen, (C,), torch.float32, 0.5)
        spread = torch.rand((C,), generator=gen, device="cuda") + 0.5
        x = _normal(gen, (B, P, C), torch.float32).mul_(spread).add_(level).to(dtype)
        state["gamma"] = 1.0 + _normal(gen, (C,), torch.float32, 0.1)
        state["beta"] = _normal(gen, (C,), torch.float32, 0.1)
        if kind != "gn":
            state["grad"] = _normal(gen, (B, P, C), dtype)
        if kind == "gn_bwd":
            v = x.view(B, P, G, C // G)
            mean = v.double().mean(dim=(1, 3))
            var = (v.double() - mean[:, None, :, None]).square().mean(dim=(1, 3))
            state["mean"] = mean.float()
            state["rstd"] = (1.0 / torch.sqrt(var + EPS)).float()
            if case["source"] == "checkpoint":
                state["codes"], state["scales"] = _pack(x)
                return state
        state["x"] = x
        return state
    if kind == "checkpoint":
        # a residual stream again, with a few channels much larger than the others
        level = _normal(gen, (case["dim"],), torch.float32, 2.0).exp_()
        state["x"] = _normal(gen, (case["rows"], case["dim"]), torch.float32).mul_(level).to(dtype)
        return state
    ab = _normal(gen, (case["rows"], 2 * case["dim"]), dtype, 1.2)
    state["grad"] = _normal(gen, (case["rows"], case["dim"]), dtype)
    if kind == "geglu_bwd" and case["source"] == "checkpoint":
        state["codes"], state["scales"] = _pack(ab)
    else:
        state["ab"] = ab
    return state


# ---- the framework's operators -------------------------------------------------------------------

def _run_own(state):
    ops = importlib.import_module("mobile-stable-diffusion_b200").ops
    case = state["case"]
    kind, dtype = case["kind"], DTYPES[case["dtype"]]
    if kind == "gn":
        return ops.groupnorm_channels_last(state["x"], state["gamma"], state["beta"], case["groups"], EPS,
                                           case["silu"])
    if kind == "gn_train":
        y, mean, rstd, kept = ops.groupnorm_channels_last_train(
            state["x"], state["gamma"], state["beta"], case["groups"], EPS, case["silu"], checkpoint=True)
        return (y,) + tuple(ops.groupnorm_channels_last_backward(
            state["grad"], kept, mean, rstd, state["gamma"], state["beta"], case["groups"], case["silu"]))
    if kind == "gn_bwd":
        kept = state["x"] if "x" in state else ops.Checkpoint8(state["codes"], state["scales"], dtype)
        return tuple(ops.groupnorm_channels_last_backward(
            state["grad"], kept, state["mean"], state["rstd"], state["gamma"], state["beta"], case["groups"],
            case["silu"]))
    if kind == "checkpoint":
        return ops.checkpoint_unpack(ops.checkpoint_pack(state["x"]))
    if kind == "geglu_train":
        y, kept = ops.gelu_multiply_checkpoint(state["ab"])
        return y, ops.gelu_multiply_backward(state["grad"], kept)
    kept = state["ab"] if "ab" in state else ops.Checkpoint8(state["codes"], state["scales"], dtype)
    return ops.gelu_multiply_backward(state["grad"], kept)


# ---- plain forms: float32, rounded once at the end --------------------------------------------------

def _sigmoid(z):
    return 1.0 / (1.0 + torch.exp(-z))


def _plain_gn_stats(x, G):
    B, P, C = x.shape
    v = x.float().view(B, P, G, C // G)
    mean = v.mean(dim=(1, 3))
    var = (v - mean[:, None, :, None]).square().mean(dim=(1, 3))
    return mean, 1.0 / torch.sqrt(var + EPS)


def _plain_gn_normalised(x, mean, rstd, G):
    B, P, C = x.shape
    v = x.float().view(B, P, G, C // G)
    return ((v - mean[:, None, :, None]) * rstd[:, None, :, None]).view(B, P, C)


def _plain_gn_backward(grad, x, mean, rstd, gamma, beta, G, silu):
    B, P, C = x.shape
    xh = _plain_gn_normalised(x, mean, rstd, G)
    dz = grad.float()
    if silu:
        z = xh * gamma + beta
        s = _sigmoid(z)
        dz = dz * (s * (1.0 + z * (1.0 - s)))
    grad_beta = dz.sum(dim=(0, 1))
    grad_gamma = (dz * xh).sum(dim=(0, 1))
    dn = (dz * gamma).view(B, P, G, C // G)
    xg = xh.view(B, P, G, C // G)
    n = P * (C // G)
    s1 = dn.sum(dim=(1, 3), keepdim=True) / n
    s2 = (dn * xg).sum(dim=(1, 3), keepdim=True) / n
    grad_x = (rstd[:, None, :, None] * (dn - s1 - xg * s2)).view(B, P, C)
    return grad_x.to(grad.dtype), grad_gamma, grad_beta


def _plain_geglu_backward(grad, ab):
    a, g = ab.float().chunk(2, dim=-1)
    cdf = 0.5 * (1.0 + torch.erf(g * 0.70710678118654752440))
    pdf = torch.exp(-0.5 * g * g) * 0.39894228040143267794
    dy = grad.float()
    return torch.cat([dy * g * cdf, dy * a * (cdf + g * pdf)], dim=-1).to(grad.dtype)


def _run_plain(state):
    case = state["case"]
    kind, dtype = case["kind"], DTYPES[case["dtype"]]
    if kind.startswith("gn"):
        G, gamma, beta = case["groups"], state["gamma"], state["beta"]
        if kind == "gn_bwd":
            x = state["x"] if "x" in state else _expand(state["codes"], state["scales"])
            return _plain_gn_backward(state["grad"], x, state["mean"], state["rstd"], gamma, beta, G, case["silu"])
        x = state["x"]
        mean, rstd = _plain_gn_stats(x, G)
        z = _plain_gn_normalised(x, mean, rstd, G) * gamma + beta
        y = (z * _sigmoid(z) if case["silu"] else z).to(dtype)
        if kind == "gn":
            return y
        del z
        kept = _expand(*_pack(x))
        return (y,) + _plain_gn_backward(state["grad"], kept, mean, rstd, gamma, beta, G, case["silu"])
    if kind == "checkpoint":
        return _expand(*_pack(state["x"])).to(dtype)
    if kind == "geglu_train":
        a, g = state["ab"].float().chunk(2, dim=-1)
        y = a * (0.5 * g * (1.0 + torch.erf(g * 0.70710678118654752440)))
        return y.to(dtype), _plain_geglu_backward(state["grad"], _expand(*_pack(state["ab"])))
    ab = state["ab"] if "ab" in state else _expand(state["codes"], state["scales"])
    return _plain_geglu_backward(state["grad"], ab)


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- what a pass cannot do without ---------------------------------------------------------------

def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    kind = case["kind"]
    if kind.startswith("gn"):
        n = case["batch"] * case["hw"] * case["channels"]
        kept = n + n // BLOCK
        act = 6 if case["silu"] else 0
        forward, backward = n * (8 + act), n * (16 + 2 * act)
        if kind == "gn":
            return {"bytes": 2 * n * size, "flops": forward}
        if kind == "gn_bwd":
            return {"bytes": 2 * n * size + (n * size if case["source"] == "tensor" else kept), "flops": backward}
        return {"bytes": 2 * n * size + 2 * n * size + 2 * kept, "flops": forward + backward + 4 * n}
    n = case["rows"] * case["dim"]
    if kind == "checkpoint":
        kept = n + case["rows"] * -(-case["dim"] // BLOCK)
        return {"bytes": 2 * n * size + 2 * kept, "flops": 5 * n}
    kept = 2 * n + case["rows"] * -(-2 * case["dim"] // BLOCK)
    if kind == "geglu_train":
        return {"bytes": 3 * n * size + 3 * n * size + 2 * kept, "flops": 60 * n}
    return {"bytes": 3 * n * size + (2 * n * size if case["source"] == "tensor" else kept), "flops": 40 * n}


# ---- the definitions in 64 bits ------------------------------------------------------------------

def _exact_kept(x):
    """Values of a checkpoint by its definition: per block of 32, steps of 2^(floor(log2 max) - 6)."""
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    dim = x.shape[-1]
    whole = dim - dim % BLOCK
    flat, dst = x.reshape(-1, dim), out.view(-1, dim)
    for lo, hi, width in ((0, whole, BLOCK), (whole, dim, dim - whole)):
        if lo == hi:
            continue
        v = flat[:, lo:hi].double().reshape(-1, (hi - lo) // width, width)
        top = v.abs().max(dim=-1, keepdim=True).values
        m, _ = torch.frexp(top)                                   # top = m * 2^k, 0.5 <= m < 1
        step = torch.where(top > 0, top / m / 128.0, torch.zeros_like(top)).clamp(min=2.0 ** -120)
        q = torch.clamp(torch.round(v / step), min=-127.0, max=127.0) * step
        dst[:, lo:hi] = q.reshape(-1, hi - lo)
    return out


def exact(case, seed):
    state = prepare(case, seed)
    kind = case["kind"]

    def phi(t):
        return torch.special.erfc(-t / math.sqrt(2.0)) / 2.0

    if kind == "checkpoint":
        return _exact_kept(state["x"])
    if kind.startswith("geglu"):
        D = case["dim"]
        if "ab" in state:
            whole = state["ab"].double()
            used = _exact_kept(state["ab"]) if kind == "geglu_train" else whole
        else:
            step = torch.exp2(state["scales"].double() - 127.0)
            used = state["codes"].double() * step[:, torch.arange(2 * D, device=step.device) // BLOCK]
        dy = state["grad"].double()
        a, g = used[:, :D], used[:, D:]
        density = torch.exp(-g.square() / 2.0) / math.sqrt(2.0 * math.pi)
        d_ab = torch.cat((dy * (g * phi(g)), dy * a * (phi(g) + g * density)), dim=1)
        if kind == "geglu_bwd":
            return d_ab
        return whole[:, :D] * whole[:, D:] * phi(whole[:, D:]), d_ab

    B, P, C, G = case["batch"], case["hw"], case["channels"], case["groups"]
    W = C // G
    gamma, beta = state["gamma"].double(), state["beta"].double()
    ys, dxs = [], []
    dgamma, dbeta = torch.zeros_like(gamma), torch.zeros_like(beta)
    for b in range(B):                                            # image by image: 64-bit copies are large
        if "x" in state:
            x = state["x"][b].double()
        else:
            step = torch.exp2(state["scales"][b].double() - 127.0)
            x = state["codes"][b].double() * step[:, torch.arange(C, device=step.device) // BLOCK]
        if kind == "gn_bwd":
            mu, rs = state["mean"][b].double(), state["rstd"][b].double()
        else:
            per_group = x.reshape(P, G, W)
            variance, mu = torch.var_mean(per_group, dim=(0, 2), correction=0)
            rs = torch.rsqrt(variance + EPS)
        mu_c, rs_c = mu.repeat_interleave(W), rs.repeat_interleave(W)
        if kind != "gn_bwd":
            z = (x - mu_c) * (rs_c * gamma) + beta
            ys.append(z / (1.0 + torch.exp(-z)) if case["silu"] else z)
        if kind == "gn":
            continue
        kept = _exact_kept(state["x"][b]) if kind == "gn_train" else x
        xh = (kept - mu_c) * rs_c
        d = state["grad"][b].double()
        if case["silu"]:
            z = xh * gamma + beta
            t = torch.exp(-z)
            d = d * (1.0 + t + z * t) / (1.0 + t).square()
        dbeta += d.sum(0)
        dgamma += (d * xh).sum(0)
        e = d * gamma
        m1 = e.sum(0).reshape(G, W).sum(1) / (P * W)
        m2 = (e * xh).sum(0).reshape(G, W).sum(1) / (P * W)
        dxs.append(rs_c * (e - m1.repeat_interleave(W) - xh * m2.repeat_interleave(W)))
    if kind == "gn":
        return torch.stack(ys)
    grads = (torch.stack(dxs), dgamma, dbeta)
    return grads if kind == "gn_bwd" else (torch.stack(ys),) + grads
