"""8-bit activation checkpoints and the GEGLU gate's forward / backward with them, on the GPU."""
import pytest
import torch

from gpu_util import Guarded
from train_util import (DTYPES, assert_within, checkpoint_reference, geglu_backward, geglu_bound, geglu_forward,
                        half_step, make)

pytestmark = pytest.mark.gpu

ALL = ["float32", "float16", "bfloat16"]


def put(t, misalign=0):
    g = Guarded(tuple(t.shape), t.dtype, misalign)
    g.tensor.copy_(t)
    return g.tensor


def spread(shape, dtype, seed):
    """Normal values times a factor per column, over several powers of two; some rows all zero."""
    x = make(shape, "float32", seed)
    f = torch.exp2(torch.arange(shape[-1]) % 11 - 5.0)
    x = (x * f).to(DTYPES[dtype])
    x.reshape(-1, shape[-1])[::7] = 0
    return x


SHAPES = [(1, 1), (3, 5), (7, 31), (4, 32), (5, 33), (9, 40), (2, 3, 320), (17, 1003), (2, 1, 64), (300, 8), (64, 4096),
          (1, 100000)]


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("misalign", [0, 1])
def test_pack_and_unpack_bit_for_bit(sdfl, shape, dtype, misalign):
    x = spread(shape, dtype, 1)
    codes, scales, values = checkpoint_reference(x)
    kept = sdfl.ops.checkpoint_pack(put(x, misalign))
    assert kept.dtype == x.dtype and kept.shape == x.shape
    assert torch.equal(kept.codes.cpu(), codes)
    assert torch.equal(kept.scales.cpu(), scales)
    for name in ALL:
        if name != "float32" and dtype == "float32":
            continue                                  # fp32 values may lie outside the narrower type
        if name == "float16" and dtype == "bfloat16":
            continue
        out = Guarded(shape, DTYPES[name], misalign)
        sdfl.ops.checkpoint_unpack(kept, out=out.tensor)
        out.check()
        assert torch.equal(out.tensor.cpu().double(), values), name


def test_pack_writes_only_its_arrays(sdfl):
    for shape in [(3, 5), (5, 40), (6, 64), (2, 1003)]:
        x = put(spread(shape, "float16", 3))
        codes = Guarded(shape, torch.int8)
        scales = Guarded((shape[0], -(-shape[1] // 32)), torch.uint8)
        lib, capi = sdfl._capi.lib, sdfl._capi
        rc = lib.sdfl_checkpoint_pack(x.data_ptr(), codes.tensor.data_ptr(), scales.tensor.data_ptr(), *shape, capi.F16,
                                      torch.cuda.current_stream().cuda_stream)
        assert rc == capi.OK
        codes.check()
        scales.check()


@pytest.mark.parametrize("dtype", ALL)
def test_extreme_values(sdfl, dtype):
    """Infinities, NaN, the largest and smallest numbers, ties, and blocks beside them that stay exact."""
    t = DTYPES[dtype]
    fi = torch.finfo(t)
    x = torch.zeros((12, 96), dtype=t)
    x[0, 3], x[1, 40], x[2, 95] = float("inf"), float("-inf"), float("nan")
    x[3:6, 0] = fi.max
    x[4, 1:32] = -fi.max
    x[6, :5] = torch.tensor([fi.smallest_normal * fi.eps, -fi.smallest_normal * fi.eps, fi.smallest_normal, 0, -0.0], dtype=t)
    x[7, :32] = torch.arange(32).to(t) * 0.5 + 64 - 0.5          # step 1: ties to even
    x[8, 32:64] = 127.5
    x[9, :] = fi.tiny
    x[10, 64:] = 1.0
    codes, scales, values = checkpoint_reference(x)
    kept = sdfl.ops.checkpoint_pack(x.cuda())
    assert torch.equal(kept.codes.cpu(), codes) and torch.equal(kept.scales.cpu(), scales)
    back = sdfl.ops.checkpoint_unpack(kept).cpu()
    assert torch.equal(torch.isnan(back), torch.isnan(values))
    assert torch.equal(torch.nan_to_num(back.double(), nan=0.0), torch.nan_to_num(values, nan=0.0))
    # the same through the element kernels
    kept2 = sdfl.ops.checkpoint_pack(put(x, 1))
    assert torch.equal(kept2.codes, kept.codes) and torch.equal(kept2.scales, kept.scales)


def test_error_of_a_value_is_within_its_step(sdfl):
    x = make((512, 320), "float32", 5, std=3.0)
    kept = sdfl.ops.checkpoint_pack(x.cuda())
    step = torch.exp2(kept.scales.cpu().double() - 127).repeat_interleave(32, 1)
    err = (sdfl.ops.checkpoint_unpack(kept).cpu().double() - x.double()).abs()
    clamped = x.double().abs() > 127.5 * step
    assert (err[~clamped] <= step[~clamped] / 2).all() and (err <= step).all()
    again = sdfl.ops.checkpoint_pack(sdfl.ops.checkpoint_unpack(kept))      # values are their own checkpoint
    assert torch.equal(again.codes, kept.codes) and torch.equal(again.scales, kept.scales)


def test_more_elements_than_31_bits(sdfl):
    """Offsets past 2^31: the last rows of a 2.2e9-element tensor."""
    rows, dim = 70000, 32000
    x = torch.zeros((rows, dim), dtype=torch.bfloat16, device="cuda")
    tail = make((4, dim), "bfloat16", 6)
    x[-4:] = tail.cuda()
    kept = sdfl.ops.checkpoint_pack(x)
    codes, scales, values = checkpoint_reference(tail)
    assert torch.equal(kept.codes[-4:].cpu(), codes) and torch.equal(kept.scales[-4:].cpu(), scales)
    del x
    back = sdfl.ops.checkpoint_unpack(kept)
    assert torch.equal(back[-4:].cpu().double(), values) and int(torch.count_nonzero(back[:-4])) == 0


def test_more_elements_than_31_bits_in_odd_rows(sdfl):
    rows, dim = 70000, 32001
    x = torch.zeros((rows, dim), dtype=torch.bfloat16, device="cuda")
    tail = make((4, dim), "bfloat16", 7)
    x[-4:] = tail.cuda()
    kept = sdfl.ops.checkpoint_pack(x)
    codes, scales, values = checkpoint_reference(tail)
    assert torch.equal(kept.codes[-4:].cpu(), codes) and torch.equal(kept.scales[-4:].cpu(), scales)
    assert int(torch.count_nonzero(kept.codes[:-4])) == 0
    del x
    back = sdfl.ops.checkpoint_unpack(kept)
    assert torch.equal(back[-4:].cpu().double(), values) and int(torch.count_nonzero(back[:-4])) == 0


def test_gate_of_more_elements_than_31_bits_in_odd_rows(sdfl):
    rows, d = 70000, 16001
    ab = torch.zeros((rows, 2 * d), dtype=torch.bfloat16, device="cuda")
    tail = make((4, 2 * d), "bfloat16", 8)
    ab[-4:] = tail.cuda()
    y, kept = sdfl.ops.gelu_multiply_checkpoint(ab)
    _, _, values = checkpoint_reference(tail)
    want = geglu_forward(tail)
    assert_within(y[-4:], want, half_step(want, "bfloat16") + geglu_bound(tail, "bfloat16"), "y")
    assert int(torch.count_nonzero(y[:-4])) == 0
    y.fill_(0.5)
    for source, x in ((kept, values), (ab, tail)):
        got = sdfl.ops.gelu_multiply_backward(y, source, out=ab)
        want, bound = geglu_backward(torch.full((4, d), 0.5), x, "bfloat16")
        assert_within(got[-4:], want, half_step(want, "bfloat16") + bound, "gradient")
        assert int(torch.count_nonzero(got[:-4])) == 0          # a = g = 0
        ab.zero_()
        ab[-4:] = tail.cuda()


GATE_SHAPES = [(1, 1), (3, 7), (5, 20), (2, 32), (77, 64), (3, 5, 96), (33, 1000), (128, 1280), (9, 5120)]


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("shape", GATE_SHAPES)
@pytest.mark.parametrize("misalign", [0, 1])
def test_gate_forward_with_checkpoint(sdfl, shape, dtype, misalign):
    D = shape[-1]
    ab = make(shape[:-1] + (2 * D,), dtype, 11, std=1.5)
    codes, scales, _ = checkpoint_reference(ab)
    out = Guarded(shape, DTYPES[dtype], misalign)
    y, kept = sdfl.ops.gelu_multiply_checkpoint(put(ab, misalign), out=out.tensor)
    out.check()
    assert torch.equal(kept.codes.cpu(), codes) and torch.equal(kept.scales.cpu(), scales)
    want = geglu_forward(ab)
    assert_within(y, want, half_step(want, dtype) + geglu_bound(ab, dtype), "gate")
    if dtype != "bfloat16":
        assert torch.equal(y, sdfl.ops.gelu_multiply(ab.cuda()))           # the bits of the plain call


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("shape", GATE_SHAPES)
@pytest.mark.parametrize("misalign", [0, 1])
def test_gate_backward_from_tensor_and_from_checkpoint(sdfl, shape, dtype, misalign):
    D = shape[-1]
    ab = make(shape[:-1] + (2 * D,), dtype, 12, std=2.0)
    dy = make(shape, dtype, 13)
    out = Guarded(tuple(ab.shape), DTYPES[dtype], misalign)
    want, bound = geglu_backward(dy, ab, dtype)
    sdfl.ops.gelu_multiply_backward(put(dy, misalign), put(ab, misalign), out=out.tensor)
    out.check()
    assert_within(out.tensor, want, half_step(want, dtype) + bound, "from the tensor")
    values = checkpoint_reference(ab)[2]
    want, bound = geglu_backward(dy, values, dtype)
    kept = sdfl.ops.checkpoint_pack(ab.cuda())
    got = sdfl.ops.gelu_multiply_backward(put(dy, misalign), kept, out=out.tensor)
    out.check()
    assert_within(got, want, half_step(want, dtype) + bound, "from the checkpoint")
    buf = put(ab, misalign)                                                # over its own input
    sdfl.ops.gelu_multiply_backward(put(dy, misalign), buf, out=buf)
    want, bound = geglu_backward(dy, ab, dtype)
    assert_within(buf, want, half_step(want, dtype) + bound, "in place")


def test_gate_gradient_against_differences(sdfl):
    ab, dy, v = make((6, 80), "float32", 21), make((6, 40), "float32", 22), make((6, 80), "float32", 23)
    got = sdfl.ops.gelu_multiply_backward(dy.cuda(), ab.cuda()).cpu().double()
    h = 1e-5
    up = (geglu_forward(ab.double() + h * v.double()) * dy.double()).sum()
    down = (geglu_forward(ab.double() - h * v.double()) * dy.double()).sum()
    slope = (got * v.double()).sum()
    # third-derivative term h^2 plus 64-bit cancellation 1e-15 / h per element, plus fp32 gradients
    assert abs(slope - (up - down) / (2 * h)) <= 1e-6 * (got * v.double()).abs().sum() + 1e-8


def test_non_finite_input_shows_in_the_gradient(sdfl):
    ab = make((4, 128), "float16", 31)
    ab[2, 5] = float("inf")
    dy = make((4, 64), "float16", 32)
    _, kept = sdfl.ops.gelu_multiply_checkpoint(ab.cuda())
    grad = sdfl.ops.gelu_multiply_backward(dy.cuda(), kept).cpu()
    # the value half's block 0 is NaN; it enters the gate half's gradient only (da = dy gelu(g))
    assert torch.isnan(grad[2, 64:96]).all()
    assert torch.isfinite(grad[[0, 1, 3]]).all() and torch.isfinite(grad[2, :64]).all() and torch.isfinite(grad[2, 96:]).all()


def test_empty_tensors(sdfl):
    for shape in [(0, 64), (3, 0)]:
        kept = sdfl.ops.checkpoint_pack(torch.empty(shape, dtype=torch.float16, device="cuda"))
        assert sdfl.ops.checkpoint_unpack(kept).shape == shape
        y, kept = sdfl.ops.gelu_multiply_checkpoint(torch.empty(shape, dtype=torch.float16, device="cuda"))
        assert y.shape == (shape[0], shape[1] // 2)
        assert sdfl.ops.gelu_multiply_backward(y, kept).shape == shape


def test_other_stream_and_graph_capture(sdfl):
    """A call on an explicit stream; two graphs, replayed on two streams at once with new data."""
    ops = sdfl.ops
    ab, dy = make((512, 2560), "bfloat16", 41).cuda(), make((512, 1280), "bfloat16", 42).cuda()
    want_y, kept = ops.gelu_multiply_checkpoint(ab)
    want_d = ops.gelu_multiply_backward(dy, kept)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    y, kept = ops.gelu_multiply_checkpoint(ab, stream=side)
    d = ops.gelu_multiply_backward(dy, kept, stream=side)
    side.synchronize()
    assert torch.equal(y, want_y) and torch.equal(d, want_d)
    graphs = []
    for k in range(2):
        bufs = [torch.zeros_like(ab), torch.zeros_like(dy)]
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y, kept = ops.gelu_multiply_checkpoint(bufs[0])
            d = ops.gelu_multiply_backward(bufs[1], kept)
        graphs.append((g, bufs, y, d, torch.cuda.Stream()))
    for g, bufs, *_ in graphs:
        bufs[0].copy_(ab), bufs[1].copy_(dy)
    torch.cuda.synchronize()
    for _ in range(3):
        for g, _, _, _, s in graphs:
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for _, _, y, d, _ in graphs:
        assert torch.equal(y, want_y) and torch.equal(d, want_d)
