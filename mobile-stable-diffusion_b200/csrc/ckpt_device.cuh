// Device side of the 8-bit activation checkpoints, shared by the kernels that write them
// (checkpoint.cu, gn_cl_*.cu) and those that read them.
//
// Format.  A tensor is [rows, dim]; a row is cut into blocks of 32 consecutive elements, the last
// one possibly shorter.  With a = max |x| over the block and e = floor(log2 a):
//     step = 2^max(e - 6, -120),   code = clamp(rne(x / step), -127, 127),   value = code * step
// stored as one signed byte per element and one byte E = 127 + log2(step) per block (row-major
// [rows, ceil(dim / 32)]).  a / step lies in [64, 128), so |value - x| <= step / 2 except that the
// clamp costs up to a whole step (1/64 of a at most) for elements above 127.5 steps; a step twice as large would
// cost the same there and double the error of everything else.  A block with an infinity or a NaN
// gets E = 255 and codes 0: 0 * inf makes every element of it NaN, so that a non-finite activation
// still shows in the gradients.
// Steps are powers of two on purpose: x / step, the rounding and code * step are then exact in
// fp32 (one correctly rounded operation gives the code), a value fits the 8 significant bits
// of bf16 and the 11 of fp16, and every kernel and plain formula that follows the definition
// gets the same bits.  The floor of 2^-120 keeps 1 / step and step normal numbers.
#pragma once

#include "common.cuh"

#include <type_traits>

namespace sdfl {

namespace {

constexpr int kCkptBlock = 32;
constexpr int kCkptNonFinite = 255;

__host__ __device__ __forceinline__ int64_t ckpt_blocks(int64_t dim) { return (dim + kCkptBlock - 1) / kCkptBlock; }

// |x| as an ordered integer: finite < inf < NaN.
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

template <int N> __device__ __forceinline__ uint32_t max_abs_bits(const float (&f)[N]) {
    uint32_t m = abs_bits(f[0]);
#pragma unroll
    for (int i = 1; i < N; ++i) m = max(m, abs_bits(f[i]));
    return m;
}

// The same of a vector as it is stored; 16-bit types two at a time, since without their signs they
// order like integers as well.
template <typename T> __device__ __forceinline__ uint32_t max_abs_bits(const uint4 &v) {
    if constexpr (sizeof(T) == 4) {
        return max(max(v.x & 0x7fffffffu, v.y & 0x7fffffffu), max(v.z & 0x7fffffffu, v.w & 0x7fffffffu));
    } else {
        const uint32_t m = __vmaxu2(__vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu),
                                    __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu));
        const uint16_t top = static_cast<uint16_t>(max(m & 0xffffu, m >> 16));
        if constexpr (std::is_same_v<T, __half>) return __float_as_uint(__half2float(__ushort_as_half(top)));
        else return static_cast<uint32_t>(top) << 16;
    }
}

struct CkptScale {
    uint32_t e;        // the scale byte
    float inv;         // 1 / step
    uint32_t keep;     // all ones, or 0 for a block with a non-finite element
    bool edge;         // the largest element is 127.5 steps or more: codes may need the clamp
};

__device__ __forceinline__ CkptScale ckpt_scale(uint32_t amax_bits) {
    const uint32_t ex = amax_bits >> 23;
    CkptScale s;
    const bool bad = ex == 255u;
    s.e = bad ? kCkptNonFinite : max(ex, 13u) - 6u;          // >= 7: step >= 2^-120
    s.inv = bad ? 0.f : __uint_as_float((254u - s.e) << 23);
    s.keep = bad ? 0u : 0xffffffffu;
    s.edge = (amax_bits & 0x7fffffu) >= 0x7f0000u;
    return s;
}

// The code in the low byte of the result.  x * inv + 1.5 * 2^23 rounds to an integer in one
// correctly rounded operation (|x * inv| < 128) whose low byte is its two's complement.
__device__ __forceinline__ uint32_t ckpt_code(float x, float inv) {
    constexpr float kMagic = 12582912.0f;
    return __float_as_uint(fminf(fmaxf(fmaf(x, inv, kMagic), kMagic - 127.0f), kMagic + 127.0f));
}

// Without the clamp: right wherever no element of the block reaches 127.5 steps, which is all but one block in
// 180 of evenly spread mantissas.  The clamp's two operations per element run on the pipe that
// bounds the packing kernels, so whole vectors go one way or the other.
__device__ __forceinline__ uint32_t ckpt_code_inside(float x, float inv) { return __float_as_uint(fmaf(x, inv, 12582912.0f)); }

template <bool CLAMP>
__device__ __forceinline__ uint32_t ckpt_code4(float a, float b, float c, float d, const CkptScale &s) {
    const auto code = [&](float x) { return CLAMP ? ckpt_code(x, s.inv) : ckpt_code_inside(x, s.inv); };
    const uint32_t lo = __byte_perm(code(a), code(b), 0x0040);
    const uint32_t hi = __byte_perm(code(c), code(d), 0x0040);
    return __byte_perm(lo, hi, 0x5410) & s.keep;
}

__device__ __forceinline__ float ckpt_step(uint8_t e) { return __uint_as_float(static_cast<uint32_t>(e) << 23); }

// Four codes to floats: the byte (offset by 128) becomes the low mantissa bits of 2^23, the
// offset is subtracted exactly, and the product with the step is exact.
__device__ __forceinline__ void ckpt_values4(uint32_t w, float step, float *f) {
    w ^= 0x80808080u;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        f[i] = (__uint_as_float(__byte_perm(w, 0x4B000000u, 0x7540u + i)) - 8388736.0f) * step;
}

__device__ __forceinline__ float ckpt_value(int8_t code, uint8_t e) { return static_cast<float>(code) * ckpt_step(e); }

// The VecOf<T>::N codes of one 16-byte vector's worth of elements.
template <int N> struct CodeVec;
template <> struct CodeVec<8> { using type = uint2; };
template <> struct CodeVec<4> { using type = uint32_t; };

__device__ __forceinline__ void ckpt_values(const uint2 &w, float step, float (&f)[8]) {
    ckpt_values4(w.x, step, f);
    ckpt_values4(w.y, step, f + 4);
}
__device__ __forceinline__ void ckpt_values(const uint32_t &w, float step, float (&f)[4]) {
    ckpt_values4(w, step, f);
}
__device__ __forceinline__ uint2 ckpt_codes(const float (&f)[8], const CkptScale &s) {
    if (s.edge)
        return make_uint2(ckpt_code4<true>(f[0], f[1], f[2], f[3], s), ckpt_code4<true>(f[4], f[5], f[6], f[7], s));
    return make_uint2(ckpt_code4<false>(f[0], f[1], f[2], f[3], s), ckpt_code4<false>(f[4], f[5], f[6], f[7], s));
}
__device__ __forceinline__ uint32_t ckpt_codes(const float (&f)[4], const CkptScale &s) {
    return s.edge ? ckpt_code4<true>(f[0], f[1], f[2], f[3], s) : ckpt_code4<false>(f[0], f[1], f[2], f[3], s);
}

// Maximum over the 32 / N neighbouring lanes that hold one block (N elements per lane, the first
// of them on a lane number that is a multiple of 32 / N).  Only these lanes have to arrive together.
template <int N> __device__ __forceinline__ uint32_t block_lanes_max(uint32_t m) {
    constexpr uint32_t L = kCkptBlock / N;
    const uint32_t mask = ((1u << L) - 1u) << (threadIdx.x & 31u & ~(L - 1u));
#pragma unroll
    for (uint32_t o = 1; o < L; o <<= 1) m = max(m, __shfl_xor_sync(mask, m, o));
    return m;
}

}  // namespace

}  // namespace sdfl
