// Device side shared by the channels-last GroupNorm kernels: vector access (16-byte vectors or
// single elements, tensor or checkpoint), sums over the threads of one column, and the per-channel
// arithmetic of the normalise and gradient passes.
//
// Layout.  [batch, hw, channels]: a pixel is a row of `channels` elements, cut into `columns` of VEC
// elements.  A thread keeps one column and walks down the rows, so everything that belongs to a
// channel (weights, statistics, running sums) sits in its registers, and neighbouring threads
// read neighbouring columns.
//
//   forward   z = (x - mean) rstd gamma + beta,  y = z or z sigmoid(z)
//   backward  dz = dy act'(z);  per channel  B = sum dz,  A = sum dz (x - mean)
//             grad_beta = B,  grad_gamma = rstd A  (summed over the images)
//             per group (M elements)  s1 = sum gamma B / M,  s2 = sum gamma rstd A / M
//             grad_x = rstd (gamma dz - s1 - xhat s2),  xhat = (x - mean) rstd
#pragma once

#include "ckpt_device.cuh"
#include "kernels.h"

namespace sdfl {

namespace {

inline bool cl_aligned(const void *p, unsigned a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

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

// ---- sums over the rows of a thread block ----------------------------------------------------------
// buf[row * ncols + c] summed over `rows` rows into buf[c], pairwise (error of log2(rows) roundings,
// and the same order on every run).  Synchronises before and after.
__device__ __forceinline__ void fold_rows(float *buf, int rows, int ncols) {
    __syncthreads();
    while (rows > 1) {
        const int half = (rows + 1) >> 1;
        const int n = (rows - half) * ncols;
        for (int i = threadIdx.x; i < n; i += blockDim.x) buf[i] += buf[i + half * ncols];
        rows = half;
        __syncthreads();
    }
}

// ---- running moments of a thread's column: shifted sums around the first value seen ----------------
template <int VEC> struct ColumnMoments {
    float k[VEC], s[VEC], q[VEC];
    __device__ __forceinline__ void first(const float (&f)[VEC]) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) { k[i] = f[i]; s[i] = 0.f; q[i] = 0.f; }
    }
    __device__ __forceinline__ void add(const float (&f)[VEC]) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const float d = f[i] - k[i];
            s[i] += d;
            q[i] = fmaf(d, d, q[i]);
        }
    }
};

// Moments of every column's channels over the block's rows: mean[c] and m2[c] (squared deviations from
// that mean), c < ncols, out of each thread's n values per channel.  First the means, then the
// deviations from them as M2_thread + n (mean_thread - mean)^2: only non-negative terms, nothing
// cancels.  buf: threads * VEC floats, mean: ncols floats; m2 comes back in buf.
template <int VEC>
__device__ __forceinline__ void block_moments(const ColumnMoments<VEC> &m, float n, bool active, int row, int rows,
                                              int col, int ncols, float count, float *buf, float *mean) {
    __syncthreads();                 // the buffers may still be read from the call before
    const float inv = n > 0.f ? 1.0f / n : 0.f;
    float *mine = buf + row * ncols + col * VEC;
    if (active) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) mine[i] = n > 0.f ? fmaf(n, m.k[i], m.s[i]) : 0.f;
    }
    fold_rows(buf, rows, ncols);
    for (int c = threadIdx.x; c < ncols; c += blockDim.x) mean[c] = buf[c] / count;
    __syncthreads();
    if (active) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const float t = m.s[i] * inv;
            const float d = m.k[i] + t - mean[col * VEC + i];
            mine[i] = n > 0.f ? fmaxf(fmaf(-m.s[i], t, m.q[i]), 0.f) + n * d * d : 0.f;
        }
    }
    fold_rows(buf, rows, ncols);
}

// ---- per-channel arithmetic ------------------------------------------------------------------------
// 1 / (1 + exp(-z)) with the SFU exp2 and reciprocal (relative error about 2^-22 each).
__device__ __forceinline__ float sigmoid_fast(float z) { return rcp_approx(1.0f + ex2_approx(-1.4426950408889634f * z)); }

// fp32 storage keeps (x - mean) as its own step; half storage folds the affine into one multiply-add
// (the folded constant's rounding, 2^-24 |mean| rstd, is far below half a step of the output).
template <typename T, int VEC, int ACT> struct Normalise {
    float p[VEC], q[VEC], r[VEC];       // half: z = x p + q;  fp32: z = (x - r) p + q
    __device__ __forceinline__ void set(int i, float mean, float rstd, float w, float b) {
        p[i] = w * rstd;
        if (sizeof(T) == 2) { q[i] = fmaf(-mean, p[i], b); r[i] = 0.f; }
        else { q[i] = b; r[i] = mean; }
    }
    __device__ __forceinline__ void apply(float (&f)[VEC]) const {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const float z = sizeof(T) == 2 ? fmaf(f[i], p[i], q[i]) : fmaf(f[i] - r[i], p[i], q[i]);
            f[i] = ACT == kActSilu ? z * sigmoid_fast(z) : z;
        }
    }
};

// dz = dy act'(z), silu'(z) = s + z s (1 - s) with s = sigmoid(z).
template <int ACT> __device__ __forceinline__ float act_grad(float dy, float z) {
    if (ACT != kActSilu) return dy;
    const float s = sigmoid_fast(z);
    return dy * fmaf(z * s, 1.0f - s, s);
}

}  // namespace

}  // namespace sdfl
