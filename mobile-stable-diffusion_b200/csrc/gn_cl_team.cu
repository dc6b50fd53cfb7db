// Channels-last GroupNorm (+SiLU) and its gradient in one persistent launch (plus a small one that adds
// up the weight gradients).  Formulas and layout: gn_cl_device.cuh.
//
// What bounds it: HBM.  The forward pass cannot do without one read and one write of the tensor, the
// backward pass without reads of x (or its checkpoint) and grad_out and one write; but both have to
// see a whole group before the first result, so every element is read twice.  The kernel keeps
// the second read inside L2.
//
// Split.  An item is a slice of an image's channels (whole groups and whole vectors, a 128-byte row or
// more where the sizes allow it) over all its pixels.  A team of M thread blocks works on one item at a
// time, each block on its own range of pixels: pass S reads and sums, the blocks' sums are exchanged, pass
// A reads again and writes.  The bytes of all teams' open items stay below kInFlight, so that the
// second read comes from L2 whatever the tensor's size.  A team with more than one item runs S of the
// next item between S and A of the current one, which hides the exchange.
//
// Loads.  Every thread owns a ring of 16-byte slots in shared memory that it fills by cp.async a few
// chunks ahead of its own use, so no barrier guards the ring.  The ring runs on over the end of a
// pass: while a block adds up its rows and waits for the others' sums, the first chunks of the next
// pass are already under way.
//
// Exchange.  A block writes its sums per group to the workspace and counts itself in; before pass A every
// block polls the count and merges all of the team's sums itself, in block order (the same bits on
// every run).  Every block of the grid is resident (cooperative launch), and every wait is
// bounded: on time-out the status word is raised and the launch finishes with an invalid result.
//
// Weight gradients: a block adds up its channels' sums over the images of its slice in shared memory and
// writes them once per slice; cl_param_sum_kernel adds the blocks' rows.
#include "gn_cl_device.cuh"
#include "gn_cl_internal.h"

#include <algorithm>
#include <numeric>

namespace sdfl {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kBlocksPerSm = 3;
constexpr int kBlocksPerSmGrad = 2;
// ring: chunks of kChunk vectors per thread, kStages chunks deep (the backward pass has two tensors)
constexpr int kChunk = 4, kStages = 3;
constexpr int kChunkGrad = 2, kStagesGrad = 4;
constexpr int kMaxCols = kThreads / 2;             // columns of a slice: keeps shared memory under 48 KB
constexpr int kMaxMembers = 512;
constexpr int kMergeLoads = kMaxMembers / 32;
constexpr int64_t kInFlight = 64ll << 20;
constexpr long long kWaitCycles = 2000000000LL;    // about a second

__device__ unsigned int g_cl_status;               // bit 0: a bounded wait ran out

struct Args {                    // one struct for both directions
    GnClForward f;
    GnClBackward b;
    GnClTeamPlan p;
    int64_t batch, hw, channels, groups;
    int width;                   // channels per group
    int share, rest;             // pixels / members, pixels % members
    float eps;
    unsigned int *arrived;       // [items]
    float2 *partial;             // [batch * groups][members]
    float2 *channel_sums;        // [slice][image_teams * members][slice channels]
};

struct Place {
    int member, slice_team, image_team, col, row, ncols, slice_groups;
    int64_t first;               // this block's pixels of every item: [first, first + pixels)
    int pixels, mine;            // of those, this thread's rows: row, row + rows, ...
    bool active;
};

__device__ __forceinline__ int member_pixels(const Args &a, int member) { return a.share + (member < a.rest ? 1 : 0); }

__device__ __forceinline__ Place place(const Args &a) {
    Place w;
    const int team = blockIdx.x / a.p.members;
    w.member = blockIdx.x - team * a.p.members;
    w.slice_team = team % a.p.slice_teams;
    w.image_team = team / a.p.slice_teams;
    w.row = threadIdx.x / a.p.cols;
    w.col = threadIdx.x - w.row * a.p.cols;
    w.active = w.row < a.p.rows;
    w.ncols = a.p.cols * a.p.vec;
    w.slice_groups = w.ncols / a.width;
    w.first = static_cast<int64_t>(w.member) * a.share + min(w.member, a.rest);
    w.pixels = member_pixels(a, w.member);
    w.mine = w.active ? (w.pixels - w.row + a.p.rows - 1) / a.p.rows : 0;
    return w;
}

// A team's items, slice by slice and image by image within a slice, and the order of their passes:
// S0, then S1 A0, S2 A1, ... and the last A (a team of one block, which has nobody to wait for: S0 A0 S1 A1 ...).
struct Items {
    int count, images, slice0, slice_step, image0, image_step;
    bool lag;
    __device__ __forceinline__ Items(const Args &a, const Place &w) {
        images = (static_cast<int>(a.batch) - w.image_team + a.p.image_teams - 1) / a.p.image_teams;
        count = images * ((a.p.slices - w.slice_team + a.p.slice_teams - 1) / a.p.slice_teams);
        slice0 = w.slice_team;
        slice_step = a.p.slice_teams;
        image0 = w.image_team;
        image_step = a.p.image_teams;
        lag = a.p.members > 1;
    }
    __device__ __forceinline__ int slice(int k) const { return slice0 + (k / images) * slice_step; }
    __device__ __forceinline__ int64_t image(int k) const { return image0 + (k % images) * image_step; }
    __device__ __forceinline__ int passes() const { return 2 * count; }
    // pass number -> item, and whether it is the second pass
    __device__ __forceinline__ int item(int pass, bool *second) const {
        if (!lag) {
            *second = pass & 1;
            return pass >> 1;
        }
        *second = pass > 0 && ((pass & 1) == 0 || pass == 2 * count - 1);
        if (!*second) return (pass + 1) >> 1;
        return pass == 2 * count - 1 ? count - 1 : (pass >> 1) - 1;
    }
};

__device__ __forceinline__ void copy_async16(void *to, const void *from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(to))), "l"(from)
                 : "memory");
}
__device__ __forceinline__ void copy_async8(void *to, const void *from) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(to))), "l"(from)
                 : "memory");
}
// 4 bytes, of which only the first `bytes` are read (the rest is zero-filled)
__device__ __forceinline__ void copy_async4(void *to, const void *from, uint32_t bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(to))),
                 "l"(from), "r"(bytes)
                 : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Counts the block in on an item; its sums were written (by any thread) before.
__device__ __forceinline__ void arrive(const Args &a, int64_t item) {
    __syncthreads();
    if (threadIdx.x == 0) {
        __threadfence();
        atomicAdd(a.arrived + item, 1u);
    }
}

// Waits until all of the team's blocks have counted themselves in.
__device__ __forceinline__ void wait_all(const Args &a, int64_t item) {
    if (threadIdx.x == 0) {
        unsigned int v;
        const long long t0 = clock64();
        for (;;) {
            asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(a.arrived + item) : "memory");
            if (v >= static_cast<unsigned>(a.p.members)) break;
            if (clock64() - t0 > kWaitCycles) {
                atomicOr(&g_cl_status, 1u);
                break;
            }
        }
    }
    __syncthreads();
}

// One group's sums of all the team's blocks, 32 per round, every load in flight at once.
__device__ __forceinline__ void load_partials(const Args &a, int64_t group, int lane, float2 (&v)[kMergeLoads]) {
    const float2 *q = a.partial + group * a.p.members;
#pragma unroll
    for (int k = 0; k < kMergeLoads; ++k) {
        v[k] = make_float2(0.f, 0.f);
        if (lane + 32 * k < a.p.members) v[k] = __ldcg(q + lane + 32 * k);
    }
}
__device__ __forceinline__ float pixels_or_none(const Args &a, int member) {
    return member < a.p.members ? static_cast<float>(member_pixels(a, member)) : 0.f;
}

// Groups of a slice are dealt to segments of L lanes, L the largest power of two up to the group's width.
struct Segments {
    int lanes, per_block, mine, lane;
    __device__ __forceinline__ explicit Segments(int width) {
        lanes = 32;
        while (lanes > width) lanes >>= 1;
        per_block = kThreads / lanes;
        mine = threadIdx.x / lanes;
        lane = threadIdx.x % lanes;
    }
    __device__ __forceinline__ float sum(float v) const {
        for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        return v;
    }
};

// ---- sums over a block's rows ----------------------------------------------------------------------
// buf[row][ncols], filled by every active thread, to buf[c] = sum over the rows, in a fixed order: each
// thread adds rows of one column, `parts` threads per column.  Synchronises before and after.
__device__ __forceinline__ void sum_rows(float *buf, int rows, int ncols) {
    __syncthreads();
    if (ncols >= kThreads) {
        for (int c = threadIdx.x; c < ncols; c += kThreads) {
            float s = buf[c];
            for (int r = 1; r < rows; ++r) s += buf[r * ncols + c];
            buf[c] = s;
        }
    } else {
        const int parts = min(kThreads / ncols, rows);
        const int part = threadIdx.x / ncols, c = threadIdx.x - part * ncols;
        float s = 0.f;
        if (part < parts) {
#pragma unroll 4
            for (int r = part; r < rows; r += parts) s += buf[r * ncols + c];
        }
        if (parts > 1) {
            __syncthreads();
            if (part > 0 && part < parts) buf[threadIdx.x] = s;
            __syncthreads();
            if (part == 0) {
                for (int k = 1; k < parts; ++k) s += buf[k * ncols + c];
                buf[c] = s;
            }
        } else if (part == 0) {
            buf[c] = s;
        }
    }
    __syncthreads();
}

// ---- forward --------------------------------------------------------------------------------------
// Statistics of a block: every thread keeps sums of d = x - (its first value) and of d^2 per channel and
// turns them into a mean and a sum of squared deviations.  The block adds up n (mean - P) and M2 + n (mean - P)^2
// with P the mean of the thread in row 0: P is close to the block's mean (it can be off by an
// outlier's share of one thread's pixels, which costs at most log2(rows) bits), so the one
// subtraction that is left, of N (block mean - P)^2, cancels next to nothing.
template <typename T, int ACT, bool PACK>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm)
cl_team_forward_kernel(const Args a) {
    constexpr int VEC = VecOf<T>::N;
    using Col = Column<VEC>;
    extern __shared__ __align__(16) unsigned char shared[];
    const Place w = place(a);
    uint4 *ring = reinterpret_cast<uint4 *>(shared) + threadIdx.x;                       // [slot][thread]
    float *buf = reinterpret_cast<float *>(shared + kChunk * kStages * kThreads * 16);   // [rows][2 ncols]
    float *cp = buf + 2 * kThreads * VEC;             // [ncols] each: P, later the scale; shift; minus the pivots
    float *cq = cp + w.ncols;
    float *pivots = cq + w.ncols;
    float2 *stat = reinterpret_cast<float2 *>(pivots + w.ncols);                         // [groups]: (mean, rstd)
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const Segments seg(a.width);
    const T *x = static_cast<const T *>(a.f.in);
    T *y = static_cast<T *>(a.f.out);
    const int64_t step = static_cast<int64_t>(a.p.rows) * a.channels;
    const int64_t mine0 = (w.first + w.row) * a.channels + w.col * VEC;                 // within an image, slice 0
    const int chunks = ((w.pixels + a.p.rows - 1) / a.p.rows + kChunk - 1) / kChunk;     // per pass
    const Items items(a, w);

    // the loading end of the ring
    const T *src = nullptr;
    int pass = -1, chunks_left = 0, left = 0, in = 0;
    auto load_chunk = [&]() {
        if (chunks_left == 0 && pass + 1 < items.passes()) {
            bool second;
            const int k = items.item(++pass, &second);
            src = x + items.image(k) * a.hw * a.channels + items.slice(k) * w.ncols + mine0;
            chunks_left = chunks;
            left = w.mine;
        }
        if (chunks_left > 0) {
#pragma unroll
            for (int k = 0; k < kChunk; ++k)
                if (k < left) copy_async16(ring + (in + k) * kThreads, src + k * step);
            src += kChunk * step;
            left -= kChunk;
            --chunks_left;
            in = in == kChunk * (kStages - 1) ? 0 : in + kChunk;
        }
        copy_commit();
    };
    int out = 0;
    auto take_chunk = [&](uint4 (&v)[kChunk]) {
        copy_wait<kStages - 1>();
#pragma unroll
        for (int k = 0; k < kChunk; ++k) v[k] = ring[(out + k) * kThreads];
        out = out == kChunk * (kStages - 1) ? 0 : out + kChunk;
        load_chunk();
    };

    auto sums = [&](int slice, int64_t image) {
        Col nk, s, q;                                 // minus the first value, sum, sum of squares
#pragma unroll
        for (int i = 0; i < Col::N; ++i) { nk.e[i] = Col::all(0.f); s.e[i] = Col::all(0.f); q.e[i] = Col::all(0.f); }
        int64_t at = image * a.hw * a.channels + slice * w.ncols + mine0;
        for (int r = 0; r < chunks * kChunk; r += kChunk, at += kChunk * step) {
            uint4 v[kChunk];
            take_chunk(v);
#pragma unroll
            for (int k = 0; k < kChunk; ++k) {
                float f[VEC];
                unpack<T>(v[k], f);
                if constexpr (PACK) {
                    // lanes past the end hold stale values of other rows, but never those of a live block
                    const CkptScale sc = ckpt_scale(block_lanes_max<VEC>(max_abs_bits<VEC>(f)));
                    if (r + k < w.mine) {
                        *reinterpret_cast<typename CodeVec<VEC>::type *>(a.f.codes + at + k * step) = ckpt_codes(f, sc);
                        if ((w.col & (kCkptBlock / VEC - 1)) == 0)
                            a.f.scales[(at + k * step) / kCkptBlock] = static_cast<uint8_t>(sc.e);
                    }
                }
                if (r + k < w.mine) {
                    if (k == 0 && r == 0) {
                        float g[VEC];
#pragma unroll
                        for (int i = 0; i < VEC; ++i) g[i] = -f[i];
                        nk.set(g);
                    }
                    Col c;
                    c.set(f);
#pragma unroll
                    for (int i = 0; i < Col::N; ++i) {
                        const Pair d = vadd(c.e[i], nk.e[i]);
                        s.e[i] = vadd(s.e[i], d);
                        q.e[i] = vfma(d, d, q.e[i]);
                    }
                }
            }
        }
        // block sums
        const float n = static_cast<float>(w.mine), inv = w.mine ? 1.0f / n : 0.f;
        float mean[VEC], m2[VEC];
        {
            float k[VEC], t[VEC], u[VEC];
            nk.get(k), s.get(t), q.get(u);
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float shift = t[i] * inv;
                mean[i] = shift - k[i];
                m2[i] = fmaxf(fmaf(-t[i], shift, u[i]), 0.f);
            }
        }
        __syncthreads();                              // the buffers may still be read by the pass before
        if (w.row == 0) shared_store<VEC>(cp + w.col * VEC, mean);
        __syncthreads();
        if (w.active) {
            float *to = buf + w.row * 2 * w.ncols + w.col * VEC;
            float head[VEC];
            shared_load<VEC>(cp + w.col * VEC, head);
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float d = w.mine ? mean[i] - head[i] : 0.f;
                mean[i] = n * d;
                m2[i] = w.mine ? fmaf(n * d, d, m2[i]) : 0.f;
            }
            shared_store<VEC>(to, mean);
            shared_store<VEC>(to + w.ncols, m2);
        }
        sum_rows(buf, a.p.rows, 2 * w.ncols);
        // channels to groups
        const int64_t group0 = image * a.groups + slice * w.slice_groups;
        const float pixels = static_cast<float>(w.pixels), inv_pixels = 1.0f / pixels;
        for (int g0 = 0; g0 < w.slice_groups; g0 += seg.per_block) {
            const int g = g0 + seg.mine;
            const int end = g < w.slice_groups ? (g + 1) * a.width : 0;
            float t = 0.f;
            for (int c = g * a.width + seg.lane; c < end; c += seg.lanes) t += fmaf(buf[c], inv_pixels, cp[c]);
            const float mu = seg.sum(t) / static_cast<float>(a.width);
            float u = 0.f;
            for (int c = g * a.width + seg.lane; c < end; c += seg.lanes) {
                const float e = buf[c] * inv_pixels, d = e + (cp[c] - mu);
                u += fmaxf(fmaf(-buf[c], e, buf[w.ncols + c]), 0.f) + pixels * d * d;
            }
            u = seg.sum(u);
            if (seg.lane == 0 && g < w.slice_groups) __stcg(a.partial + (group0 + g) * a.p.members + w.member, make_float2(mu, u));
        }
        arrive(a, image * a.p.slices + slice);
    };

    // z = (x - pivot) p + q, the pivot being the mean of the column's first channel: where the mean is far
    // from zero compared with the spread, x - pivot loses nothing, and one register serves the vector.
    auto apply = [&](int slice, int64_t image) {
        wait_all(a, image * a.p.slices + slice);
        const int64_t group0 = image * a.groups + slice * w.slice_groups;
        const float hw = static_cast<float>(a.hw), width = static_cast<float>(a.width);
        for (int g = warp; g < w.slice_groups; g += kWarps) {
            float2 v[kMergeLoads];
            load_partials(a, group0 + g, lane, v);
            float t = 0.f;
#pragma unroll
            for (int k = 0; k < kMergeLoads; ++k) t = fmaf(pixels_or_none(a, lane + 32 * k), v[k].x, t);
            const float mu = warp_sum(t) / hw;
            float u = 0.f;
#pragma unroll
            for (int k = 0; k < kMergeLoads; ++k) {
                const float d = v[k].x - mu;
                u += fmaf(pixels_or_none(a, lane + 32 * k) * width * d, d, v[k].y);
            }
            u = warp_sum(u);
            if (lane == 0) {
                const float rstd = 1.0f / sqrtf(u / (hw * width) + a.eps);
                stat[g] = make_float2(mu, rstd);
                if (w.member == 0 && a.f.mean) {
                    a.f.mean[group0 + g] = mu;
                    a.f.rstd[group0 + g] = rstd;
                }
            }
        }
        __syncthreads();
        for (int c = threadIdx.x; c < w.ncols; c += kThreads) {
            const int channel = slice * w.ncols + c;
            const float2 st = stat[c / a.width];
            const float pivot = stat[(c - c % VEC) / a.width].x;
            const float scale = a.f.gamma[channel] * st.y;
            cp[c] = scale;
            cq[c] = fmaf(pivot - st.x, scale, a.f.beta[channel]);
            pivots[c] = -pivot;
        }
        __syncthreads();
        Col cs, ch;
        column_load<VEC>(cp + w.col * VEC, cs);
        column_load<VEC>(cq + w.col * VEC, ch);
        const Pair np = Col::all(pivots[w.col * VEC]);
        T *o = y + image * a.hw * a.channels + slice * w.ncols + mine0;
        for (int r = 0; r < chunks * kChunk; r += kChunk, o += kChunk * step) {
            uint4 v[kChunk];
            take_chunk(v);
#pragma unroll
            for (int k = 0; k < kChunk; ++k)
                if (r + k < w.mine) {
                    float f[VEC];
                    unpack<T>(v[k], f);
                    Col c;
                    c.set(f);
#pragma unroll
                    for (int i = 0; i < Col::N; ++i) {
                        const Pair z = vfma(vadd(c.e[i], np), cs.e[i], ch.e[i]);
                        c.e[i] = ACT == kActSilu ? vmul(z, sigmoid_fast(z)) : z;
                    }
                    c.get(f);
                    st_stream(o + k * step, pack<T>(f));
                }
        }
    };

    for (int k = 0; k < kStages; ++k) load_chunk();
    for (int p = 0; p < items.passes(); ++p) {
        bool second;
        const int k = items.item(p, &second);
        if (second) apply(items.slice(k), items.image(k));
        else sums(items.slice(k), items.image(k));
    }
}

// ---- backward -------------------------------------------------------------------------------------
template <typename T, int ACT, bool CKPT>
__global__ void __launch_bounds__(kThreads, kBlocksPerSmGrad)
cl_team_backward_kernel(const Args a) {
    constexpr int VEC = VecOf<T>::N;
    constexpr int kSlots = kChunkGrad * kStagesGrad;
    using Col = Column<VEC>;
    using Codes = typename CodeVec<VEC>::type;
    extern __shared__ __align__(16) unsigned char shared[];
    const Place w = place(a);
    uint4 *ring = reinterpret_cast<uint4 *>(shared) + threadIdx.x;                       // grad_out, [slot][thread]
    unsigned char *ring2 = shared + kSlots * kThreads * 16;                              // x, or codes and scale words
    uint4 *ring_x = reinterpret_cast<uint4 *>(ring2) + threadIdx.x;
    Codes *ring_c = reinterpret_cast<Codes *>(ring2) + threadIdx.x;
    uint32_t *ring_s = reinterpret_cast<uint32_t *>(ring2 + kSlots * kThreads * sizeof(Codes)) + threadIdx.x;
    float *buf = reinterpret_cast<float *>(ring2 + kSlots * kThreads * 16);              // [rows][2 ncols]
    float *total = buf + 2 * kThreads * VEC;          // [2 ncols]: this slice's channel sums over the images
    float *cp = total + 2 * w.ncols;                  // [ncols] each: scale and shift of z; c0 and c1; minus the pivots
    float *cq = cp + w.ncols;
    float *c0 = cq + w.ncols;
    float *c1 = c0 + w.ncols;
    float *pivots = c1 + w.ncols;
    float2 *stat = reinterpret_cast<float2 *>(pivots + w.ncols);                         // [groups]: (s1, s2)
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const Segments seg(a.width);
    const int64_t blocks_row = ckpt_blocks(a.channels), scale_bytes = a.batch * a.hw * blocks_row;
    const T *x = static_cast<const T *>(a.b.in);
    const T *dy = static_cast<const T *>(a.b.grad_out);
    T *dx = static_cast<T *>(a.b.grad_in);
    const Pair one = Col::all(1.0f), minus_one = Col::all(-1.0f);
    const int64_t step = static_cast<int64_t>(a.p.rows) * a.channels;
    const int64_t mine0 = (w.first + w.row) * a.channels + w.col * VEC;
    const int chunks = ((w.pixels + a.p.rows - 1) / a.p.rows + kChunkGrad - 1) / kChunkGrad;
    const Items items(a, w);

    int64_t src = 0, scale_at = 0;                    // element, scale byte
    int pass = -1, chunks_left = 0, left = 0, in = 0;
    auto load_chunk = [&]() {
        if (chunks_left == 0 && pass + 1 < items.passes()) {
            bool second;
            const int k = items.item(++pass, &second);
            const int channel = items.slice(k) * w.ncols + w.col * VEC;
            src = items.image(k) * a.hw * a.channels + items.slice(k) * w.ncols + mine0;
            scale_at = (items.image(k) * a.hw + w.first + w.row) * blocks_row + channel / kCkptBlock;
            chunks_left = chunks;
            left = w.mine;
        }
        if (chunks_left > 0) {
#pragma unroll
            for (int k = 0; k < kChunkGrad; ++k)
                if (k < left) {
                    const int slot = (in + k) * kThreads;
                    copy_async16(ring + slot, dy + src + k * step);
                    if constexpr (CKPT) {
                        if constexpr (VEC == 8) copy_async8(ring_c + slot, a.b.codes + src + k * step);
                        else copy_async4(ring_c + slot, a.b.codes + src + k * step, 4);
                        // the aligned word that holds the scale byte, or what there is of it
                        const int64_t word = (scale_at + k * a.p.rows * blocks_row) & ~static_cast<int64_t>(3);
                        const int64_t rest = scale_bytes - word;
                        copy_async4(ring_s + slot, a.b.scales + word, rest < 4 ? static_cast<uint32_t>(rest) : 4u);
                    } else {
                        copy_async16(ring_x + slot, x + src + k * step);
                    }
                }
            src += kChunkGrad * step;
            scale_at += static_cast<int64_t>(kChunkGrad) * a.p.rows * blocks_row;
            left -= kChunkGrad;
            --chunks_left;
            in = in == kSlots - kChunkGrad ? 0 : in + kChunkGrad;
        }
        copy_commit();
    };
    // x and grad_out of the next chunk; `at` is the scale byte of its first row
    int out = 0;
    auto take_chunk = [&](Col (&xc)[kChunkGrad], Col (&dc)[kChunkGrad], int64_t at) {
        copy_wait<kStagesGrad - 1>();
#pragma unroll
        for (int k = 0; k < kChunkGrad; ++k) {
            const int slot = (out + k) * kThreads;
            float f[VEC];
            unpack<T>(ring[slot], f);
            dc[k].set(f);
            if constexpr (CKPT) {
                const uint32_t shift = static_cast<uint32_t>(at + k * a.p.rows * blocks_row) & 3u;
                const uint8_t e = static_cast<uint8_t>(ring_s[slot] >> (8 * shift));
                ckpt_values(ring_c[slot], ckpt_step(e), f);
            } else {
                unpack<T>(ring_x[slot], f);
            }
            xc[k].set(f);
        }
        out = out == kSlots - kChunkGrad ? 0 : out + kChunkGrad;
        load_chunk();
    };

    // z = (x - pivot) p + q as in the forward pass
    auto coefficients = [&](int slice, int64_t image, bool second) {
        __syncthreads();                              // the arrays may still be read by the pass before
        for (int c = threadIdx.x; c < w.ncols; c += kThreads) {
            const int channel = slice * w.ncols + c, head = channel - c % VEC;
            const int64_t st = image * a.groups + channel / a.width;
            const float mean = a.b.mean[st], rs = a.b.rstd[st], pivot = a.b.mean[image * a.groups + head / a.width];
            const float scale = a.b.gamma[channel] * rs;
            cp[c] = scale;
            cq[c] = fmaf(pivot - mean, scale, a.b.beta[channel]);
            pivots[c] = -pivot;
            if (second) {
                const float2 s = stat[c / a.width];
                c1[c] = -rs * rs * s.y;
                c0[c] = fmaf(pivot - mean, c1[c], -rs * s.x);
            }
        }
        __syncthreads();
    };

    auto sums = [&](int slice, int64_t image) {
        coefficients(slice, image, false);
        Col s0, s1;
#pragma unroll
        for (int i = 0; i < Col::N; ++i) { s0.e[i] = Col::all(0.f); s1.e[i] = Col::all(0.f); }
        {
            Col cs, ch;
            const int col = w.active ? w.col * VEC : 0;
            column_load<VEC>(cp + col, cs);
            column_load<VEC>(cq + col, ch);
            const Pair np = Col::all(pivots[col]);
            int64_t at = (image * a.hw + w.first + w.row) * blocks_row + (slice * w.ncols + w.col * VEC) / kCkptBlock;
            for (int r = 0; r < chunks * kChunkGrad; r += kChunkGrad, at += static_cast<int64_t>(kChunkGrad) * a.p.rows * blocks_row) {
                Col xc[kChunkGrad], dc[kChunkGrad];
                take_chunk(xc, dc, at);
#pragma unroll
                for (int k = 0; k < kChunkGrad; ++k)
                    if (r + k < w.mine) {
#pragma unroll
                        for (int i = 0; i < Col::N; ++i) {
                            const Pair xm = vadd(xc[k].e[i], np);
                            const Pair dz = act_grad<ACT>(dc[k].e[i], vfma(xm, cs.e[i], ch.e[i]), one, minus_one);
                            s0.e[i] = vadd(s0.e[i], dz);
                            s1.e[i] = vfma(dz, xm, s1.e[i]);
                        }
                    }
            }
        }
        if (w.active) {
            float *to = buf + w.row * 2 * w.ncols + w.col * VEC;
            column_store<VEC>(to, s0);
            column_store<VEC>(to + w.ncols, s1);
        }
        sum_rows(buf, a.p.rows, 2 * w.ncols);
        const int64_t group0 = image * a.groups + slice * w.slice_groups;
        for (int c = threadIdx.x; c < w.ncols; c += kThreads) {
            const int64_t st = group0 + c / a.width;
            // from sums around the pivot to sums of dz xhat
            const float t = fmaf(-pivots[c] - a.b.mean[st], buf[c], buf[w.ncols + c]) * a.b.rstd[st];
            buf[w.ncols + c] = t;
            total[c] += buf[c];
            total[w.ncols + c] += t;
        }
        __syncthreads();
        for (int g0 = 0; g0 < w.slice_groups; g0 += seg.per_block) {
            const int g = g0 + seg.mine;
            const int end = g < w.slice_groups ? (g + 1) * a.width : 0;
            float t1 = 0.f, t2 = 0.f;
            for (int c = g * a.width + seg.lane; c < end; c += seg.lanes) {
                const float gm = a.b.gamma[slice * w.ncols + c];
                t1 = fmaf(gm, buf[c], t1);
                t2 = fmaf(gm, buf[w.ncols + c], t2);
            }
            t1 = seg.sum(t1);
            t2 = seg.sum(t2);
            if (seg.lane == 0 && g < w.slice_groups) __stcg(a.partial + (group0 + g) * a.p.members + w.member, make_float2(t1, t2));
        }
        arrive(a, image * a.p.slices + slice);
    };

    auto apply = [&](int slice, int64_t image) {
        wait_all(a, image * a.p.slices + slice);
        const int64_t group0 = image * a.groups + slice * w.slice_groups;
        const float inv = 1.0f / (static_cast<float>(a.hw) * static_cast<float>(a.width));
        for (int g = warp; g < w.slice_groups; g += kWarps) {
            float2 v[kMergeLoads];
            load_partials(a, group0 + g, lane, v);
            float t1 = 0.f, t2 = 0.f;
#pragma unroll
            for (int k = 0; k < kMergeLoads; ++k) {
                t1 += v[k].x;
                t2 += v[k].y;
            }
            t1 = warp_sum(t1);
            t2 = warp_sum(t2);
            if (lane == 0) stat[g] = make_float2(t1 * inv, t2 * inv);
        }
        coefficients(slice, image, true);
        Col cs, ch, k0, k1;
        const int col = w.active ? w.col * VEC : 0;
        column_load<VEC>(cp + col, cs);
        column_load<VEC>(cq + col, ch);
        column_load<VEC>(c0 + col, k0);
        column_load<VEC>(c1 + col, k1);
        const Pair np = Col::all(pivots[col]);
        int64_t at = (image * a.hw + w.first + w.row) * blocks_row + (slice * w.ncols + w.col * VEC) / kCkptBlock;
        T *o = dx + image * a.hw * a.channels + slice * w.ncols + mine0;
        for (int r = 0; r < chunks * kChunkGrad; r += kChunkGrad, o += kChunkGrad * step,
                 at += static_cast<int64_t>(kChunkGrad) * a.p.rows * blocks_row) {
            Col xc[kChunkGrad], dc[kChunkGrad];
            take_chunk(xc, dc, at);
#pragma unroll
            for (int k = 0; k < kChunkGrad; ++k)
                if (r + k < w.mine) {
#pragma unroll
                    for (int i = 0; i < Col::N; ++i) {
                        const Pair xm = vadd(xc[k].e[i], np);
                        const Pair dz = act_grad<ACT>(dc[k].e[i], vfma(xm, cs.e[i], ch.e[i]), one, minus_one);
                        dc[k].e[i] = vfma(dz, cs.e[i], vfma(xm, k1.e[i], k0.e[i]));
                    }
                    float f[VEC];
                    dc[k].get(f);
                    st_stream(o + k * step, pack<T>(f));
                }
        }
    };

    for (int k = 0; k < kStagesGrad; ++k) load_chunk();
    for (int p = 0; p < items.passes(); ++p) {
        bool second;
        const int k = items.item(p, &second), slice = items.slice(k);
        if (second) {
            apply(slice, items.image(k));
            continue;
        }
        const bool first = k % items.images == 0, last = k % items.images == items.images - 1;
        if (first) {
            __syncthreads();
            for (int c = threadIdx.x; c < 2 * w.ncols; c += kThreads) total[c] = 0.f;
        }
        sums(slice, items.image(k));
        if (last) {
            __syncthreads();
            const int64_t entry = static_cast<int64_t>(w.image_team) * a.p.members + w.member;
            float2 *to = a.channel_sums + (static_cast<int64_t>(slice) * a.p.image_teams * a.p.members + entry) * w.ncols;
            for (int c = threadIdx.x; c < w.ncols; c += kThreads) to[c] = make_float2(total[c], total[w.ncols + c]);
        }
    }
}

// grad_beta, grad_gamma: the entries of a slice added up, 32 channels per block.
__global__ void __launch_bounds__(kThreads)
cl_param_sum_kernel(const float2 *channel_sums, float *grad_gamma, float *grad_beta, int slice_channels, int entries,
                    int64_t channels) {
    __shared__ float2 buf[kThreads];
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + (threadIdx.x & 31);
    float b = 0.f, g = 0.f;
    if (c < channels) {
        const int64_t slice = c / slice_channels;
        const float2 *p = channel_sums + slice * entries * slice_channels + (c - slice * slice_channels);
        for (int e = threadIdx.x >> 5; e < entries; e += kThreads / 32) {
            const float2 v = p[static_cast<int64_t>(e) * slice_channels];
            b += v.x;
            g += v.y;
        }
    }
    buf[threadIdx.x] = make_float2(b, g);
    __syncthreads();
    if (threadIdx.x < 32 && c < channels) {
        for (int k = 1; k < kThreads / 32; ++k) {
            b += buf[threadIdx.x + 32 * k].x;
            g += buf[threadIdx.x + 32 * k].y;
        }
        if (grad_beta) grad_beta[c] = b;
        if (grad_gamma) grad_gamma[c] = g;
    }
}

// ---- plan and launch ------------------------------------------------------------------------------
struct Layout {
    size_t partial, channel_sums, bytes;              // behind the items' counters
};

Layout layout(const GnClShape &s, const GnClTeamPlan &p, bool backward) {
    const auto up = [](size_t n) { return (n + 15) & ~static_cast<size_t>(15); };
    Layout l;
    l.partial = up(static_cast<size_t>(s.batch) * p.slices * sizeof(unsigned int));
    l.channel_sums = l.partial + up(static_cast<size_t>(s.batch) * s.groups * p.members * sizeof(float2));
    l.bytes = l.channel_sums +
              (backward ? static_cast<size_t>(p.image_teams) * p.members * s.channels * sizeof(float2) : 0);
    return l;
}

Args make_args(const GnClShape &s, const GnClTeamPlan &p, bool backward, void *ws) {
    const Layout l = layout(s, p, backward);
    char *base = static_cast<char *>(ws);
    Args a{};
    a.p = p;
    a.batch = s.batch;
    a.hw = s.hw;
    a.channels = s.channels;
    a.groups = s.groups;
    a.width = static_cast<int>(s.channels / s.groups);
    a.share = static_cast<int>(s.hw / p.members);
    a.rest = static_cast<int>(s.hw % p.members);
    a.eps = s.eps;
    a.arrived = reinterpret_cast<unsigned int *>(base);
    a.partial = reinterpret_cast<float2 *>(base + l.partial);
    a.channel_sums = reinterpret_cast<float2 *>(base + l.channel_sums);
    return a;
}

size_t shared_bytes(const GnClTeamPlan &p, bool backward) {
    const size_t ncols = static_cast<size_t>(p.cols) * p.vec;
    const size_t ring = backward ? static_cast<size_t>(kChunkGrad) * kStagesGrad * 2 : static_cast<size_t>(kChunk) * kStages;
    return ring * kThreads * 16 + (2 * static_cast<size_t>(kThreads) * p.vec + (backward ? 9 : 5) * ncols) * sizeof(float);
}

cudaError_t launch(void (*kernel)(Args), const Args &a, bool backward, cudaStream_t stream) {
    cudaError_t err = cudaMemsetAsync(a.arrived, 0, static_cast<size_t>(a.batch) * a.p.slices * sizeof(unsigned int), stream);
    if (err != cudaSuccess) return err;
    const size_t smem = shared_bytes(a.p, backward);
    err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (err != cudaSuccess) return err;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(a.p.slice_teams * a.p.image_teams * a.p.members));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeCooperative;
    attr[0].val.cooperative = 1;
    cfg.attrs = attr;
    cfg.numAttrs = a.p.members > 1 ? 1 : 0;
    err = cudaLaunchKernelEx(&cfg, kernel, a);
    if (err == cudaSuccess) g_launches.fetch_add(1);
    return err;
}

template <typename T> cudaError_t forward_type(const GnClShape &s, Args &a, cudaStream_t stream) {
    if (s.act == kActSilu)
        return a.f.codes ? launch(cl_team_forward_kernel<T, kActSilu, true>, a, false, stream)
                         : launch(cl_team_forward_kernel<T, kActSilu, false>, a, false, stream);
    return a.f.codes ? launch(cl_team_forward_kernel<T, kActNone, true>, a, false, stream)
                     : launch(cl_team_forward_kernel<T, kActNone, false>, a, false, stream);
}

template <typename T> cudaError_t backward_type(const GnClShape &s, Args &a, cudaStream_t stream) {
    if (s.act == kActSilu)
        return a.b.codes ? launch(cl_team_backward_kernel<T, kActSilu, true>, a, true, stream)
                         : launch(cl_team_backward_kernel<T, kActSilu, false>, a, true, stream);
    return a.b.codes ? launch(cl_team_backward_kernel<T, kActNone, true>, a, true, stream)
                     : launch(cl_team_backward_kernel<T, kActNone, false>, a, true, stream);
}

}  // namespace

bool gn_cl_team_plan(const GnClShape &s, bool pack, bool backward, bool ckpt, GnClTeamPlan *p) {
    const int64_t width = s.channels / s.groups;
    const int64_t esize = s.dtype == kF32 ? 4 : 2;
    p->vec = static_cast<int>(16 / esize);
    if (s.channels % p->vec != 0 || (pack && s.channels % kCkptBlock != 0)) return false;
    // the narrowest slice, in columns: whole groups, whole vectors and, when it is packed, whole blocks
    int64_t grain = std::lcm(width, static_cast<int64_t>(p->vec));
    if (pack) grain = std::lcm(grain, static_cast<int64_t>(kCkptBlock));
    if (grain > s.channels || s.channels % grain != 0) return false;
    const int64_t grains = s.channels / grain;
    grain /= p->vec;
    if (grain > kMaxCols) return false;
    const int64_t per_element = backward ? (ckpt ? 1 : esize) + esize : esize;
    const int64_t image = s.hw * s.channels * per_element;
    // slices: as many as leave rows of 128 bytes, more only where an image is too large for L2 twice
    const int64_t grain_bytes = grain * p->vec * esize;
    const int64_t want = (128 + grain_bytes - 1) / grain_bytes;                         // grains per slice
    const int64_t least = (2 * image + kInFlight - 1) / kInFlight;                      // slices
    int64_t best = 0;
    for (int64_t d = 1; d <= grains; ++d) {                                            // slices
        if (grains % d != 0 || grains / d * grain > kMaxCols) continue;
        if (best == 0 || grains / d >= want || (d >= least && best < least && grains / d * grain * p->vec * esize >= 64)) best = d;
    }
    if (best == 0) return false;
    // large images: only as many slices as the footprint asks for
    if (least > 1) {
        for (int64_t d = 1; d <= best; ++d)
            if (grains % d == 0 && grains / d * grain <= kMaxCols && d >= least) { best = d; break; }
    }
    p->slices = static_cast<int>(best);
    p->cols = static_cast<int>(grains / best * grain);
    p->rows = kThreads / p->cols;
    // what an SM holds at once: 228 KB of shared memory, 1 KB of it reserved per block
    const int64_t fit = 228 * 1024 / (static_cast<int64_t>(shared_bytes(*p, backward)) + 1024);
    const int64_t blocks = static_cast<int64_t>(sm_count()) * std::min<int64_t>(fit, backward ? kBlocksPerSmGrad : kBlocksPerSm);
    if (least > 1) {
        p->slice_teams = 1;
        p->image_teams = 1;
    } else {
        p->slice_teams = static_cast<int>(best);
        int64_t n = s.batch * image <= kInFlight ? s.batch : std::max<int64_t>(1, kInFlight / (2 * image));
        n = std::min(n, std::max<int64_t>(1, blocks / best));
        n = std::min(n, s.batch);
        n = (s.batch + (s.batch + n - 1) / n - 1) / ((s.batch + n - 1) / n);           // even rounds
        p->image_teams = static_cast<int>(n);
        if (p->slice_teams > blocks) p->slice_teams = static_cast<int>(blocks);
    }
    int64_t m = std::max<int64_t>(1, blocks / (static_cast<int64_t>(p->slice_teams) * p->image_teams));
    m = std::min(m, std::max<int64_t>(1, s.hw / (p->rows * 2)));                      // at least two pixels per thread
    p->members = static_cast<int>(std::min<int64_t>(m, kMaxMembers));
    return true;
}

size_t gn_cl_team_workspace_bytes(const GnClShape &s, const GnClTeamPlan &p, bool backward) {
    return layout(s, p, backward).bytes;
}

cudaError_t gn_cl_team_forward(const GnClShape &s, const GnClTeamPlan &p, const GnClForward &f, void *ws, cudaStream_t stream) {
    Args a = make_args(s, p, false, ws);
    a.f = f;
    switch (s.dtype) {
        case kF16: return forward_type<__half>(s, a, stream);
        case kBF16: return forward_type<__nv_bfloat16>(s, a, stream);
        default: return forward_type<float>(s, a, stream);
    }
}

cudaError_t gn_cl_team_backward(const GnClShape &s, const GnClTeamPlan &p, const GnClBackward &b, void *ws,
                                cudaStream_t stream) {
    Args a = make_args(s, p, true, ws);
    a.b = b;
    cudaError_t err;
    switch (s.dtype) {
        case kF16: err = backward_type<__half>(s, a, stream); break;
        case kBF16: err = backward_type<__nv_bfloat16>(s, a, stream); break;
        default: err = backward_type<float>(s, a, stream); break;
    }
    if (err != cudaSuccess || (!b.grad_gamma && !b.grad_beta)) return err;
    cl_param_sum_kernel<<<static_cast<unsigned>((s.channels + 31) / 32), kThreads, 0, stream>>>(
        a.channel_sums, b.grad_gamma, b.grad_beta, p.cols * p.vec, p.image_teams * p.members, s.channels);
    err = cudaGetLastError();
    if (err == cudaSuccess) g_launches.fetch_add(1);
    return err;
}

cudaError_t gn_cl_read_status(unsigned int *value, bool clear, cudaStream_t stream) {
    cudaError_t err = cudaMemcpyFromSymbolAsync(value, g_cl_status, sizeof(unsigned int), 0, cudaMemcpyDeviceToHost, stream);
    if (err != cudaSuccess) return err;
    err = cudaStreamSynchronize(stream);
    if (err != cudaSuccess) return err;
    if (clear && *value != 0) {
        const unsigned int zero = 0;
        err = cudaMemcpyToSymbolAsync(g_cl_status, &zero, sizeof(unsigned int), 0, cudaMemcpyHostToDevice, stream);
        if (err == cudaSuccess) err = cudaStreamSynchronize(stream);
    }
    return err;
}

}  // namespace sdfl
