// Channels-last GroupNorm (+SiLU) and its gradient for any shape and alignment: statistics per
// (image, row split, channel), a merge per (image, group), and a pass that normalises (or forms the
// gradient).  Formulas and layout: gn_cl_device.cuh.
//
// The form that takes every shape: channel counts that are not whole vectors, unaligned buffers, groups wider than
// half a block's columns, and devices that do not hold a team's blocks at once.  Forward reads x twice and writes y,
// backward reads x and grad_out twice and writes grad_x; the second read comes from L2 while the tensor fits it.  With whole vectors it takes 240 us where
// the single launch of gn_cl_team.cu takes 127 ([4, 262144, 128] fp16); [4, 16384, 1032] fp16 in 8 groups, which has no other,
// takes 270 us (16 % of the measured copy bandwidth).
#include "gn_cl_device.cuh"
#include "gn_cl_internal.h"

namespace sdfl {

namespace {

constexpr int kThreads = 256;

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
// z = (x - mean) p + beta with the mean of the channel's own group: where it is far from zero compared with the
// spread, x - mean loses nothing, and a group's results do not depend on the other groups of its vectors.
template <int VEC, int ACT> struct Normalise {
    float mean[VEC], p[VEC], q[VEC];
    __device__ __forceinline__ void set(int i, float mu, float rstd, float w, float b) {
        mean[i] = mu;
        p[i] = w * rstd;
        q[i] = b;
    }
    __device__ __forceinline__ void apply(float (&f)[VEC]) const {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const float z = fmaf(f[i] - mean[i], p[i], q[i]);
            f[i] = act_value<ACT>(z);
        }
    }
};

// Columns are dealt to `col_blocks` thread blocks of `cols` columns each; a block has `rows` rows of threads.
struct Geometry {
    int vec, columns, col_blocks, cols, rows, splits;
    int64_t blocks;
};

Geometry make_geometry(const GnClShape &s, int vec) {
    Geometry g;
    g.vec = vec;
    g.columns = static_cast<int>(s.channels / vec);
    g.col_blocks = (g.columns + kThreads - 1) / kThreads;
    g.cols = (g.columns + g.col_blocks - 1) / g.col_blocks;
    g.rows = kThreads / g.cols;
    // about 4 blocks per SM in all, but at least 8 pixels per thread
    const int64_t want = (static_cast<int64_t>(sm_count()) * 4 + s.batch * g.col_blocks - 1) / (s.batch * g.col_blocks);
    const int64_t most = (s.hw + g.rows * 8 - 1) / (g.rows * 8);
    g.splits = static_cast<int>(want < most ? want : most);
    if (g.splits < 1) g.splits = 1;
    g.blocks = s.batch * g.col_blocks * g.splits;
    return g;
}

struct Where {
    int split, col, row, channel;
    int64_t image, first, end;       // pixels [first, end) of the image
    bool active;
};

__device__ __forceinline__ Where locate(const Geometry &g, int64_t hw) {
    Where w;
    w.split = static_cast<int>(blockIdx.x % g.splits);
    const int64_t t = blockIdx.x / g.splits;
    const int cb = static_cast<int>(t % g.col_blocks);
    w.image = t / g.col_blocks;
    w.row = threadIdx.x / g.cols;
    w.col = threadIdx.x - w.row * g.cols;
    w.channel = (cb * g.cols + w.col) * g.vec;
    w.active = w.row < g.rows && cb * g.cols + w.col < g.columns;
    w.first = hw * w.split / g.splits;
    w.end = hw * (w.split + 1) / g.splits;
    return w;
}

// What a group's means are counted from: its first value in the image.  Means that lie far from zero would be rounded
// at their own magnitude, and their differences, which enter the variance, by as much.
template <typename T>
__device__ __forceinline__ float group_origin(const T *x, int64_t image, int64_t group, int64_t hw, int64_t channels, int64_t width) {
    return to_float<T>(x[image * hw * channels + group * width]);
}

// partial[image][split][channel] = (mean - origin of the group, M2) over the split's pixels
template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads)
cl_moments_kernel(const T *x, float2 *partial, Geometry g, int64_t hw, int64_t channels, int64_t width) {
    __shared__ float buf[kThreads * VEC];
    __shared__ float mean[kThreads * VEC];
    const Where w = locate(g, hw);
    ColumnMoments<VEC> m;
    int n = 0;
    if (w.active) {
        const T *p = x + w.image * hw * channels + w.channel;
        for (int64_t px = w.first + w.row; px < w.end; px += g.rows, ++n) {
            float f[VEC];
            raw_unpack<T, VEC>(raw_load<T, VEC>(p + px * channels), f);
            if (n == 0) m.first(f);
            m.add(f);
        }
#pragma unroll
        for (int i = 0; i < VEC; ++i)
            m.k[i] = n > 0 ? m.k[i] - group_origin(x, w.image, (w.channel + i) / width, hw, channels, width) : 0.f;
    }
    const int ncols = g.cols * VEC;
    block_moments<VEC>(m, static_cast<float>(n), w.active || w.row < g.rows, w.row, g.rows, w.col, ncols,
                       static_cast<float>(w.end - w.first), buf, mean);
    const int first_channel = w.channel - w.col * VEC;
    for (int c = threadIdx.x; c < ncols; c += kThreads)
        if (first_channel + c < channels)
            partial[(w.image * g.splits + w.split) * channels + first_channel + c] = make_float2(mean[c], buf[c]);
}

// One block per (image, group): merge of the splits' and channels' moments.
template <typename T>
__global__ void __launch_bounds__(kThreads)
cl_statistics_kernel(const T *x, const float2 *partial, float2 *stats, float *mean_out, float *rstd_out, int splits, int64_t hw,
                     int64_t channels, int64_t groups, float eps) {
    __shared__ float scratch[33];
    const int64_t image = blockIdx.x / groups, group = blockIdx.x % groups;
    const int64_t width = channels / groups;
    const float2 *p = partial + image * splits * channels + group * width;
    const float total = static_cast<float>(hw) * static_cast<float>(width);
    float sum = 0.f;
    for (int64_t i = threadIdx.x; i < splits * width; i += kThreads) {
        const int64_t s = i / width, c = i - s * width;
        const float n = static_cast<float>(hw * (s + 1) / splits - hw * s / splits);
        sum = fmaf(n, p[s * channels + c].x, sum);
    }
    const float mean = block_sum(sum, scratch) / total;
    float m2 = 0.f;
    for (int64_t i = threadIdx.x; i < splits * width; i += kThreads) {
        const int64_t s = i / width, c = i - s * width;
        const float n = static_cast<float>(hw * (s + 1) / splits - hw * s / splits);
        const float2 v = p[s * channels + c];
        const float d = v.x - mean;
        m2 += fmaf(n * d, d, v.y);
    }
    m2 = block_sum(m2, scratch);
    if (threadIdx.x == 0) {
        const float mu = group_origin(x, image, group, hw, channels, width) + mean;
        const float rstd = 1.0f / sqrtf(m2 / total + eps);
        stats[blockIdx.x] = make_float2(mu, rstd);
        if (mean_out) { mean_out[blockIdx.x] = mu; rstd_out[blockIdx.x] = rstd; }
    }
}

template <typename T, int VEC, int ACT>
__global__ void __launch_bounds__(kThreads)
cl_normalise_kernel(const T *x, T *y, const float2 *__restrict__ stats, const float *__restrict__ gamma,
                    const float *__restrict__ beta, Geometry g, int64_t hw, int64_t channels, int64_t groups) {
    const Where w = locate(g, hw);
    if (!w.active) return;
    const int width = static_cast<int>(channels / groups);
    Normalise<VEC, ACT> a;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        const float2 st = stats[w.image * groups + (w.channel + i) / width];
        a.set(i, st.x, st.y, gamma[w.channel + i], beta[w.channel + i]);
    }
    const int64_t at = w.image * hw * channels + w.channel;
    for (int64_t px = w.first + w.row; px < w.end; px += g.rows) {
        float f[VEC];
        raw_unpack<T, VEC>(raw_load_last<T, VEC>(x + at + px * channels), f);
        a.apply(f);
        raw_store<T, VEC>(y + at + px * channels, raw_pack<T, VEC>(f));
    }
}

// ---- backward -------------------------------------------------------------------------------------
// partial[image][split][channel] = (sum dz, sum dz (x - mean))
template <typename T, int VEC, int ACT, bool CKPT>
__global__ void __launch_bounds__(kThreads)
cl_grad_sums_kernel(GnClBackward a, float2 *partial, Geometry g, int64_t hw, int64_t channels, int64_t groups) {
    __shared__ float buf[kThreads * VEC];
    const Where w = locate(g, hw);
    const int width = static_cast<int>(channels / groups);
    const int64_t blocks_row = ckpt_blocks(channels);
    float mean[VEC], p[VEC], q[VEC], s0[VEC], s1[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) { s0[i] = 0.f; s1[i] = 0.f; }
    if (w.active) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const int64_t st = w.image * groups + (w.channel + i) / width;
            mean[i] = a.mean[st];
            p[i] = a.gamma[w.channel + i] * a.rstd[st];
            q[i] = a.beta[w.channel + i];
        }
        const T *dy = static_cast<const T *>(a.grad_out);
        for (int64_t px = w.first + w.row; px < w.end; px += g.rows) {
            const int64_t row = w.image * hw + px;
            Source<T, VEC, CKPT> src;
            src.load(a.in, a.codes, a.scales, row, channels, blocks_row, w.channel);
            float x[VEC], d[VEC];
            raw_unpack<T, VEC>(raw_load<T, VEC>(dy + row * channels + w.channel), d);
            src.values(x);
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float xm = x[i] - mean[i];
                const float dz = act_grad<ACT>(d[i], fmaf(xm, p[i], q[i]), 1.0f);
                s0[i] += dz;
                s1[i] = fmaf(dz, xm, s1[i]);
            }
        }
    }
    const int ncols = g.cols * VEC;
    float2 *out = partial + (w.image * g.splits + w.split) * channels;
    const int first_channel = w.channel - w.col * VEC;
    float *mine = buf + w.row * ncols + w.col * VEC;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        __syncthreads();
        if (w.row < g.rows) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) mine[i] = half ? s1[i] : s0[i];
        }
        fold_rows(buf, g.rows, ncols);
        for (int c = threadIdx.x; c < ncols; c += kThreads)
            if (first_channel + c < channels) (half ? out[first_channel + c].y : out[first_channel + c].x) = buf[c];
    }
}

// One block per (image, group): channel totals (sum dz, sum dz xhat), and the group's s1, s2.
__global__ void __launch_bounds__(kThreads)
cl_grad_group_kernel(const float2 *partial, float2 *channel_sums, float2 *group_sums, const float *gamma,
                     const float *rstd, int splits, int64_t hw, int64_t channels, int64_t groups) {
    __shared__ float scratch[33];
    const int64_t image = blockIdx.x / groups, group = blockIdx.x % groups;
    const int64_t width = channels / groups;
    const float rs = rstd[blockIdx.x];
    const int lane = threadIdx.x & 31;
    float t1 = 0.f, t2 = 0.f;
    for (int64_t c = group * width + (threadIdx.x >> 5); c < (group + 1) * width; c += kThreads / 32) {
        float b = 0.f, a = 0.f;
        for (int s = lane; s < splits; s += 32) {
            const float2 v = partial[(image * splits + s) * channels + c];
            b += v.x;
            a += v.y;
        }
        b = warp_sum(b);
        a = warp_sum(a) * rs;
        if (lane == 0) {
            channel_sums[image * channels + c] = make_float2(b, a);
            t1 = fmaf(gamma[c], b, t1);
            t2 = fmaf(gamma[c], a, t2);
        }
    }
    t1 = block_sum(t1, scratch);
    t2 = block_sum(t2, scratch);
    if (threadIdx.x == 0) {
        const float inv = 1.0f / (static_cast<float>(hw) * static_cast<float>(width));
        group_sums[blockIdx.x] = make_float2(t1 * inv, t2 * inv);
    }
}

__global__ void __launch_bounds__(kThreads)
cl_param_grad_kernel(const float2 *channel_sums, float *grad_gamma, float *grad_beta, int64_t batch, int64_t channels) {
    const int64_t c = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
    if (c >= channels) return;
    float b = 0.f, a = 0.f;
    for (int64_t n = 0; n < batch; ++n) {
        const float2 v = channel_sums[n * channels + c];
        b += v.x;
        a += v.y;
    }
    if (grad_beta) grad_beta[c] = b;
    if (grad_gamma) grad_gamma[c] = a;
}

template <typename T, int VEC, int ACT, bool CKPT>
__global__ void __launch_bounds__(kThreads)
cl_grad_input_kernel(GnClBackward a, const float2 *__restrict__ group_sums, Geometry g, int64_t hw, int64_t channels,
                     int64_t groups) {
    const Where w = locate(g, hw);
    if (!w.active) return;
    const int width = static_cast<int>(channels / groups);
    const int64_t blocks_row = ckpt_blocks(channels);
    float mean[VEC], p[VEC], q[VEC], c0[VEC], c1[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        const int64_t st = w.image * groups + (w.channel + i) / width;
        const float rs = a.rstd[st];
        const float2 sums = group_sums[st];
        mean[i] = a.mean[st];
        p[i] = a.gamma[w.channel + i] * rs;
        q[i] = a.beta[w.channel + i];
        c0[i] = rs * sums.x;
        c1[i] = rs * rs * sums.y;
    }
    const T *dy = static_cast<const T *>(a.grad_out);
    T *dx = static_cast<T *>(a.grad_in);
    for (int64_t px = w.first + w.row; px < w.end; px += g.rows) {
        const int64_t row = w.image * hw + px;
        Source<T, VEC, CKPT> src;
        src.load(a.in, a.codes, a.scales, row, channels, blocks_row, w.channel);
        float x[VEC], d[VEC];
        raw_unpack<T, VEC>(raw_load_last<T, VEC>(dy + row * channels + w.channel), d);
        src.values(x);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const float xm = x[i] - mean[i];
            const float dz = act_grad<ACT>(d[i], fmaf(xm, p[i], q[i]), 1.0f);
            d[i] = fmaf(dz, p[i], -fmaf(xm, c1[i], c0[i]));
        }
        raw_store<T, VEC>(dx + row * channels + w.channel, raw_pack<T, VEC>(d));
    }
}

template <typename T, int VEC>
cudaError_t forward_run(const GnClShape &s, const GnClForward &a, void *ws, cudaStream_t stream) {
    const Geometry g = make_geometry(s, VEC);
    if (g.blocks >= (1ll << 31)) return cudaErrorInvalidConfiguration;
    const unsigned grid = static_cast<unsigned>(g.blocks);
    float2 *stats = static_cast<float2 *>(ws);
    float2 *partial = stats + s.batch * s.groups;
    const T *x = static_cast<const T *>(a.in);
    T *y = static_cast<T *>(a.out);
    cl_moments_kernel<T, VEC><<<grid, kThreads, 0, stream>>>(x, partial, g, s.hw, s.channels, s.channels / s.groups);
    cl_statistics_kernel<T><<<static_cast<unsigned>(s.batch * s.groups), kThreads, 0, stream>>>(
        x, partial, stats, a.mean, a.rstd, g.splits, s.hw, s.channels, s.groups, s.eps);
    if (s.act == kActSilu)
        cl_normalise_kernel<T, VEC, kActSilu><<<grid, kThreads, 0, stream>>>(x, y, stats, a.gamma, a.beta, g, s.hw,
                                                                            s.channels, s.groups);
    else
        cl_normalise_kernel<T, VEC, kActNone><<<grid, kThreads, 0, stream>>>(x, y, stats, a.gamma, a.beta, g, s.hw,
                                                                            s.channels, s.groups);
    cudaError_t err = cudaGetLastError();
    if (err == cudaSuccess) g_launches.fetch_add(3);
    return err;
}

template <typename T, int VEC, int ACT, bool CKPT>
cudaError_t backward_run(const GnClShape &s, const GnClBackward &a, void *ws, cudaStream_t stream) {
    const Geometry g = make_geometry(s, VEC);
    if (g.blocks >= (1ll << 31)) return cudaErrorInvalidConfiguration;
    const unsigned grid = static_cast<unsigned>(g.blocks);
    float2 *group_sums = static_cast<float2 *>(ws);
    float2 *channel_sums = group_sums + s.batch * s.groups;
    float2 *partial = channel_sums + s.batch * s.channels;
    cl_grad_sums_kernel<T, VEC, ACT, CKPT><<<grid, kThreads, 0, stream>>>(a, partial, g, s.hw, s.channels, s.groups);
    cl_grad_group_kernel<<<static_cast<unsigned>(s.batch * s.groups), kThreads, 0, stream>>>(
        partial, channel_sums, group_sums, a.gamma, a.rstd, g.splits, s.hw, s.channels, s.groups);
    cl_grad_input_kernel<T, VEC, ACT, CKPT><<<grid, kThreads, 0, stream>>>(a, group_sums, g, s.hw, s.channels, s.groups);
    int launches = 3;
    if (a.grad_gamma || a.grad_beta) {
        cl_param_grad_kernel<<<static_cast<unsigned>((s.channels + kThreads - 1) / kThreads), kThreads, 0, stream>>>(
            channel_sums, a.grad_gamma, a.grad_beta, s.batch, s.channels);
        ++launches;
    }
    cudaError_t err = cudaGetLastError();
    if (err == cudaSuccess) g_launches.fetch_add(launches);
    return err;
}

template <typename T, int VEC>
cudaError_t backward_pick(const GnClShape &s, const GnClBackward &a, void *ws, cudaStream_t stream) {
    if (s.act == kActSilu)
        return a.codes ? backward_run<T, VEC, kActSilu, true>(s, a, ws, stream)
                       : backward_run<T, VEC, kActSilu, false>(s, a, ws, stream);
    return a.codes ? backward_run<T, VEC, kActNone, true>(s, a, ws, stream)
                   : backward_run<T, VEC, kActNone, false>(s, a, ws, stream);
}

template <typename T> bool vectors_ok(const GnClShape &s, const void *a, const void *b, const void *c, const void *codes) {
    constexpr int VEC = VecOf<T>::N;
    return s.channels % VEC == 0 && aligned(a, 16) && aligned(b, 16) && aligned(c, 16) && aligned(codes, VEC);
}

template <typename T>
cudaError_t forward_type(const GnClShape &s, const GnClForward &a, void *ws, cudaStream_t stream) {
    return vectors_ok<T>(s, a.in, a.out, nullptr, nullptr) ? forward_run<T, VecOf<T>::N>(s, a, ws, stream)
                                                          : forward_run<T, 1>(s, a, ws, stream);
}

template <typename T>
cudaError_t backward_type(const GnClShape &s, const GnClBackward &a, void *ws, cudaStream_t stream) {
    return vectors_ok<T>(s, a.in, a.grad_out, a.grad_in, a.codes) ? backward_pick<T, VecOf<T>::N>(s, a, ws, stream)
                                                                 : backward_pick<T, 1>(s, a, ws, stream);
}

}  // namespace

size_t gn_cl_split_workspace_bytes(const GnClShape &s, bool backward) {
    int64_t splits = make_geometry(s, 1).splits;
    const int vec = s.dtype == kF32 ? 4 : 8;
    if (s.channels % vec == 0) {
        const int64_t v = make_geometry(s, vec).splits;
        if (v > splits) splits = v;
    }
    const int64_t pairs = s.batch * s.groups + s.batch * splits * s.channels + (backward ? s.batch * s.channels : 0);
    return static_cast<size_t>(pairs) * sizeof(float2);
}

cudaError_t gn_cl_split_forward(const GnClShape &s, const GnClForward &a, void *ws, cudaStream_t stream) {
    switch (s.dtype) {
        case kF16: return forward_type<__half>(s, a, ws, stream);
        case kBF16: return forward_type<__nv_bfloat16>(s, a, ws, stream);
        default: return forward_type<float>(s, a, ws, stream);
    }
}

cudaError_t gn_cl_split_backward(const GnClShape &s, const GnClBackward &a, void *ws, cudaStream_t stream) {
    switch (s.dtype) {
        case kF16: return backward_type<__half>(s, a, ws, stream);
        case kBF16: return backward_type<__nv_bfloat16>(s, a, ws, stream);
        default: return backward_type<float>(s, a, ws, stream);
    }
}

}  // namespace sdfl
