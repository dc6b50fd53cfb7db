// Device side shared by the channels-last GroupNorm kernels: vector access (16-byte vectors or
// single elements, tensor or checkpoint), sums over the threads of one column, and the per-channel
// arithmetic of the normalise and gradient passes.
//
// Layout.  [batch, hw, channels]: a pixel is a row of `channels` elements, cut into `columns` of VEC
// elements.  A thread keeps one column and walks down the rows, so its channels' running sums sit in its registers
// and neighbouring threads read neighbouring columns; weights and statistics are read from shared memory
// (gn_cl_team.cu) or sit in registers too (gn_cl_split.cu).
//
//   forward   z = (x - mean) rstd gamma + beta,  y = z or z sigmoid(z)
//   backward  dz = dy act'(z);  per channel  B = sum dz,  A = sum dz (x - mean)
//             grad_beta = B,  grad_gamma = rstd A  (summed over the images)
//             per group (M elements)  s1 = sum gamma B / M,  s2 = sum gamma rstd A / M
//             grad_x = rstd (gamma dz - s1 - xhat s2),  xhat = (x - mean) rstd
#pragma once

#include "ckpt_device.cuh"
#include "kernels.h"

#include <type_traits>

namespace sdfl {

namespace {

// ---- one column access: VEC elements of one pixel ------------------------------------------------
template <typename T, int VEC> struct Raw { using type = uint4; };
template <typename T> struct Raw<T, 1> { using type = T; };

template <typename T, int VEC>
__device__ __forceinline__ typename Raw<T, VEC>::type raw_load(const T *p) {
    return *reinterpret_cast<const typename Raw<T, VEC>::type *>(p);
}
template <typename T, int VEC>
__device__ __forceinline__ typename Raw<T, VEC>::type raw_load_last(const T *p) {      // not needed again
    return __ldcs(reinterpret_cast<const typename Raw<T, VEC>::type *>(p));
}
template <typename T, int VEC>
__device__ __forceinline__ void raw_store(T *p, const typename Raw<T, VEC>::type &v) {
    __stcs(reinterpret_cast<typename Raw<T, VEC>::type *>(p), v);
}
template <typename T, int VEC>
__device__ __forceinline__ void raw_unpack(const typename Raw<T, VEC>::type &v, float (&f)[VEC]) {
    if constexpr (VEC == 1) f[0] = to_float<T>(v);
    else unpack<T>(v, f);
}
template <typename T, int VEC>
__device__ __forceinline__ typename Raw<T, VEC>::type raw_pack(const float (&f)[VEC]) {
    if constexpr (VEC == 1) return from_float<T>(f[0]);
    else return pack<T>(f);
}

// The normalised tensor's source in the backward pass: the tensor, or codes with their step.
template <typename T, int VEC, bool CKPT> struct Source {
    typename Raw<T, VEC>::type v;
    __device__ __forceinline__ void load(const void *x, const int8_t *, const uint8_t *, int64_t row, int64_t channels,
                                         int64_t, int channel) {
        v = raw_load<T, VEC>(static_cast<const T *>(x) + row * channels + channel);
    }
    __device__ __forceinline__ void values(float (&f)[VEC]) const { raw_unpack<T, VEC>(v, f); }
};
template <typename T, int VEC> struct Source<T, VEC, true> {
    typename CodeVec<VEC>::type c;
    uint8_t e;
    __device__ __forceinline__ void load(const void *, const int8_t *codes, const uint8_t *scales, int64_t row,
                                         int64_t channels, int64_t blocks_row, int channel) {
        c = *reinterpret_cast<const typename CodeVec<VEC>::type *>(codes + row * channels + channel);
        e = scales[row * blocks_row + channel / kCkptBlock];
    }
    __device__ __forceinline__ void values(float (&f)[VEC]) const { ckpt_values(c, ckpt_step(e), f); }
};
template <typename T> struct Source<T, 1, true> {
    int8_t c;
    uint8_t e;
    __device__ __forceinline__ void load(const void *, const int8_t *codes, const uint8_t *scales, int64_t row,
                                         int64_t channels, int64_t blocks_row, int channel) {
        c = codes[row * channels + channel];
        e = scales[row * blocks_row + channel / kCkptBlock];
    }
    __device__ __forceinline__ void values(float (&f)[1]) const { f[0] = ckpt_value(c, e); }
};

// ---- arithmetic on a column: VEC elements as VEC / 2 pairs ------------------------------------------
// The packed fp32 instructions (add, mul and fma .f32x2) do two elements per instruction; with 16 warps per SM these
// kernels take about 1.9 cycles per instruction and scheduler.  VEC = 1 uses the scalar forms.
using Pair = unsigned long long;

__device__ __forceinline__ Pair pair(float lo, float hi) {
    Pair r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void split(Pair p, float &lo, float &hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(p)); }
__device__ __forceinline__ Pair vadd(Pair a, Pair b) {
    Pair r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ Pair vmul(Pair a, Pair b) {
    Pair r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ Pair vfma(Pair a, Pair b, Pair c) {
    Pair r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ float vadd(float a, float b) { return a + b; }
__device__ __forceinline__ float vmul(float a, float b) { return a * b; }
__device__ __forceinline__ float vfma(float a, float b, float c) { return fmaf(a, b, c); }

template <int VEC> struct Column {
    using E = Pair;
    static constexpr int N = VEC / 2;
    Pair e[N];
    static __device__ __forceinline__ Pair all(float x) { return pair(x, x); }
    __device__ __forceinline__ void set(const float *f) {
#pragma unroll
        for (int i = 0; i < N; ++i) e[i] = pair(f[2 * i], f[2 * i + 1]);
    }
    __device__ __forceinline__ void get(float *f) const {
#pragma unroll
        for (int i = 0; i < N; ++i) split(e[i], f[2 * i], f[2 * i + 1]);
    }
};
template <> struct Column<1> {
    using E = float;
    static constexpr int N = 1;
    float e[1];
    static __device__ __forceinline__ float all(float x) { return x; }
    __device__ __forceinline__ void set(const float *f) { e[0] = f[0]; }
    __device__ __forceinline__ void get(float *f) const { f[0] = e[0]; }
};

// The codes of a column as whole numbers; times the step they are the values (exact either way).
__device__ __forceinline__ void codes4(uint32_t w, Pair &lo, Pair &hi) {
    const Pair offset = pair(-8388736.0f, -8388736.0f);
    w ^= 0x80808080u;
    lo = vadd(pair(__uint_as_float(__byte_perm(w, 0x4B000000u, 0x7540u)), __uint_as_float(__byte_perm(w, 0x4B000000u, 0x7541u))), offset);
    hi = vadd(pair(__uint_as_float(__byte_perm(w, 0x4B000000u, 0x7542u)), __uint_as_float(__byte_perm(w, 0x4B000000u, 0x7543u))), offset);
}

// Half h of a column (4 elements, two pairs) out of a vector of T, or out of its codes.
template <typename T> __device__ __forceinline__ void half_column(const uint4 &v, int h, Pair (&e)[2]) {
    if constexpr (sizeof(T) == 4) {
        e[0] = pair(__uint_as_float(v.x), __uint_as_float(v.y));
        e[1] = pair(__uint_as_float(v.z), __uint_as_float(v.w));
    } else {
        const uint32_t w[2] = {h ? v.z : v.x, h ? v.w : v.y};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if constexpr (std::is_same_v<T, __half>) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
                e[i] = pair(f.x, f.y);
            } else {
                e[i] = pair(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
            }
        }
    }
}
__device__ __forceinline__ void half_codes(const uint2 &w, int h, Pair (&e)[2]) { codes4(h ? w.y : w.x, e[0], e[1]); }
__device__ __forceinline__ void half_codes(uint32_t w, int, Pair (&e)[2]) { codes4(w, e[0], e[1]); }

// Two pairs back to storage: a half of a 16-bit vector, all of an fp32 one.
template <typename T> __device__ __forceinline__ void half_pack(uint4 &v, int h, const Pair (&e)[2]) {
    float f[4];
    split(e[0], f[0], f[1]);
    split(e[1], f[2], f[3]);
    if constexpr (sizeof(T) == 4) {
        v = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
    } else {
        uint32_t w[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if constexpr (std::is_same_v<T, __half>) {
                const __half2 p = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t *>(&p);
            } else {
                const __nv_bfloat162 p = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t *>(&p);
            }
        }
        (h ? v.z : v.x) = w[0];
        (h ? v.w : v.y) = w[1];
    }
}
// Four floats of shared memory as two pairs.
__device__ __forceinline__ void quad_load(const float *from, Pair (&e)[2]) {
    const float4 v = *reinterpret_cast<const float4 *>(from);
    e[0] = pair(v.x, v.y);
    e[1] = pair(v.z, v.w);
}

// VEC floats of shared memory, 16 bytes at a time (rows of a thread's column are 16-byte aligned).
template <int VEC> __device__ __forceinline__ void shared_store(float *to, const float (&f)[VEC]) {
    if constexpr (VEC == 1) to[0] = f[0];
    else
#pragma unroll
        for (int i = 0; i < VEC; i += 4)
            *reinterpret_cast<float4 *>(to + i) = make_float4(f[i], f[i + 1], f[i + 2], f[i + 3]);
}
template <int VEC> __device__ __forceinline__ void shared_load(const float *from, float (&f)[VEC]) {
    if constexpr (VEC == 1) f[0] = from[0];
    else
#pragma unroll
        for (int i = 0; i < VEC; i += 4) {
            const float4 v = *reinterpret_cast<const float4 *>(from + i);
            f[i] = v.x; f[i + 1] = v.y; f[i + 2] = v.z; f[i + 3] = v.w;
        }
}

template <int VEC> __device__ __forceinline__ void column_store(float *to, const Column<VEC> &c) {
    float f[VEC];
    c.get(f);
    shared_store<VEC>(to, f);
}

__device__ __forceinline__ float max_nan(float a, float b) {      // NaN if either is
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// s = sigmoid(z) = 1 / (1 + t) from t = exp(-z), with the SFU exp2 and reciprocal as in the other SiLU kernels
// (relative error of each about 2^-22, and |z| 2^-24 from the exponent's rounding).  Below z = -87 the
// reciprocal is 0 (subnormal), and so is z s.
__device__ __forceinline__ float sigmoid_fast(float z) {
    return rcp_approx(1.0f + ex2_approx(-1.4426950408889634f * z));
}
__device__ __forceinline__ Pair sigmoid_fast(Pair z) {
    float lo, hi;
    split(vmul(z, pair(-1.4426950408889634f, -1.4426950408889634f)), lo, hi);
    split(vadd(pair(ex2_approx(lo), ex2_approx(hi)), pair(1.0f, 1.0f)), lo, hi);
    return pair(rcp_approx(lo), rcp_approx(hi));
}

template <int ACT, typename E> __device__ __forceinline__ E act_value(E z) {
    if (ACT != kActSilu) return z;
    return vmul(z, sigmoid_fast(z));
}

// The same for results in fp16, of two elements of one group: they share one reciprocal, 1 / (a b), from which
// 1 / a = b / (a b).  Three SFU operations per pair instead of four, and at an eighth of the issue rate they bound the
// forward pass (139 -> 130 us at [4, 262144, 128]).  a b is finite because z is held at -41.5, where z e^z
// is -2^-54.5, far below half of fp16's smallest number.  fp32 and bf16 can tell z e^z from 0 down to z = -87, so there
// every element has a reciprocal of its own.  A NaN makes both elements NaN: not for pairs that span groups.
template <int ACT> __device__ __forceinline__ Pair act_value_half(Pair z) {
    if (ACT != kActSilu) return z;
    float lo, hi, a, b;
    split(z, lo, hi);
    z = pair(max_nan(lo, -41.5f), max_nan(hi, -41.5f));
    split(vmul(z, pair(-1.4426950408889634f, -1.4426950408889634f)), lo, hi);
    split(vadd(pair(ex2_approx(lo), ex2_approx(hi)), pair(1.0f, 1.0f)), a, b);
    const float r = rcp_approx(a * b);
    return vmul(z, pair(b * r, a * r));
}

// The same with w = 1 - s = t s, without the difference's cancellation.  t is held at 2^127, so that t s is 0 and
// not inf * 0 where s is 0.
__device__ __forceinline__ void sigmoid_fast(float z, float &s, float &w) {
    const float t = ex2_approx(fminf(-1.4426950408889634f * z, 127.0f));
    s = rcp_approx(1.0f + t);
    w = t * s;
}
__device__ __forceinline__ void sigmoid_fast(Pair z, Pair &s, Pair &w) {
    float lo, hi;
    split(vmul(z, pair(-1.4426950408889634f, -1.4426950408889634f)), lo, hi);
    const Pair t = pair(ex2_approx(fminf(lo, 127.0f)), ex2_approx(fminf(hi, 127.0f)));
    split(vadd(t, pair(1.0f, 1.0f)), lo, hi);
    s = pair(rcp_approx(lo), rcp_approx(hi));
    w = vmul(t, s);
}

// dy act'(z), silu'(z) = s (1 + z (1 - s)).
template <int ACT, typename E> __device__ __forceinline__ E act_grad(E dy, E z, E one) {
    if (ACT != kActSilu) return dy;
    E s, w;
    sigmoid_fast(z, s, w);
    return vmul(vmul(dy, s), vfma(z, w, one));
}

}  // namespace

}  // namespace sdfl
