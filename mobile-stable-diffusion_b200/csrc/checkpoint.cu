// 8-bit activation checkpoints (format: ckpt_device.cuh): packing and expanding, the GEGLU gate that
// keeps a checkpoint of its input, and the gate's backward pass from the whole input or from the
// checkpoint.  fp32, fp16 or bf16 storage, fp32 arithmetic.
//
// Every kernel is one pass, bounded by HBM: bytes per element of the input of size s are
// s + 33/32 (pack, expand), and per gate element 3 s + 2 * 33/32 (forward with checkpoint),
// 5 s or 3 s + 2 * 33/32 (backward).
//
// Vector kernels: a lane holds one 16-byte vector (8 or 4 elements), so a block of 32 is 4 or 8
// neighbouring lanes and its maximum is 2 or 3 shuffles.  They need 16-byte aligned buffers and
// rows that are whole vectors; rows that are not whole blocks are walked as if padded to whole
// blocks, the lanes beyond the row end idle.  A thread takes kVecs vectors 256 apart, all loads first:
// with one load in flight per thread the kernels reach 78 % of the copy bandwidth.
// Element kernels, for everything else: eight lanes share a block, so that what a block costs once (its row,
// its scale) is paid for four blocks at a time; a lane's four elements are eight apart, so that an access of the warp is
// four sectors.  ([65536, 1003] bf16, pack and expand: one lane per element 213 and 172 us, four elements in a row per
// lane 73 and 78, eight apart 71 and 58; aligned vectors shifted into place 89 and 81: the shifts and the ragged ends
// cost more instructions than they save accesses.  Indices are 32 bits wide where they can be: 64 bits took 89.)
//
// Measured (B200, back to back in a captured graph; share of the measured copy bandwidth):
//   pack    [262144, 320] fp16 41 us (97 %), [32768, 320] bf16 7.2 us, [65536, 1003] bf16 (element kernel) 71 us (44 %)
//   expand  the same 41 us (97 %), 6.6 us, 58 us (53 %)
//   gate with checkpoint  [65536, 1280] bf16 124 us (85 %), [16384, 1280] fp16 32 us (81 %): bound by the integer
//           operations of the maxima and the codes beside HBM
//   gate backward  [65536, 1280] bf16 from the input 130 us (100 %), from a checkpoint 112 us (94 %); element kernel
//           [8192, 1003] fp32 27 us (95 %) and 30 us (60 %), bf16 27 (47 %) and 29 us (36 %): 2-byte accesses
#include "ckpt_device.cuh"
#include "kernels.h"

namespace sdfl {

namespace {

constexpr int kCkThreads = 256;
constexpr int kVecs = 4;             // vectors per thread and round: pack, expand
constexpr int kGateVecs = 2;         // of each half: gate
// Element kernels of pack and expand: lanes per block, elements per lane, blocks of a warp, rounds of those.
constexpr int kLanes = 8, kElems = kCkptBlock / kLanes, kElemBlocks = 32 / kLanes, kElemRounds = 2;
constexpr int kGateElems = 4;        // per thread and round: element kernels of the gate

constexpr int64_t kMaxGridThreads = int64_t{1} << 22;      // of ck_grid
constexpr int64_t kMaxElementBlocks = kMaxGridThreads / 32 * kElemBlocks * kElemRounds;      // of a round of such a grid

inline unsigned ck_grid(int64_t work_items) {
    int64_t blocks = (work_items + kCkThreads - 1) / kCkThreads;
    const int64_t cap = static_cast<int64_t>(sm_count()) * 8 * 4;
    if (blocks > cap) blocks = cap;
    if (blocks > kMaxGridThreads / kCkThreads) blocks = kMaxGridThreads / kCkThreads;
    if (blocks < 1) blocks = 1;
    return static_cast<unsigned>(blocks);
}

// ---- pack ---------------------------------------------------------------------------------------
// A slot is one vector of a row padded to whole blocks.  RAGGED = false: rows are whole blocks, a slot
// is a vector of the flat tensor.
template <typename T, bool RAGGED>
__global__ void __launch_bounds__(kCkThreads)
pack_vec_kernel(const uint4 *__restrict__ src, typename CodeVec<VecOf<T>::N>::type *__restrict__ codes,
                uint8_t *__restrict__ scales, long long nslots, uint32_t slots_row, FastDiv slots_div, uint32_t vecs_row) {
    constexpr int VEC = VecOf<T>::N;
    constexpr int LANES = kCkptBlock / VEC;
    const long long stride = static_cast<long long>(gridDim.x) * kCkThreads * kVecs;
    // whole warps go round together: the shuffles need every lane
    for (long long base = static_cast<long long>(blockIdx.x) * kCkThreads * kVecs + (threadIdx.x & ~31); base < nslots;
         base += stride) {
        long long at[kVecs];
        bool live[kVecs];
        uint4 v[kVecs];
#pragma unroll
        for (int k = 0; k < kVecs; ++k) {
            const long long i = base + k * kCkThreads + (threadIdx.x & 31);
            at[k] = i;
            live[k] = i < nslots;
            if (RAGGED) {
                const uint32_t row = slots_div.div(static_cast<uint32_t>(i));
                const uint32_t col = static_cast<uint32_t>(i) - row * slots_row;
                live[k] = live[k] && col < vecs_row;
                at[k] = static_cast<long long>(row) * vecs_row + col;
            }
            v[k] = live[k] ? ld_stream(src + at[k]) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int k = 0; k < kVecs; ++k) {
            const CkptScale s = ckpt_scale(block_lanes_max<VEC>(max_abs_bits<T>(v[k])));
            if (live[k]) {
                float f[VEC];
                unpack<T>(v[k], f);
                codes[at[k]] = ckpt_codes(f, s);
                if ((threadIdx.x & (LANES - 1)) == 0)
                    scales[(base + k * kCkThreads + (threadIdx.x & 31)) / LANES] = static_cast<uint8_t>(s.e);
            }
        }
    }
}

__device__ __forceinline__ int divide(int n, int, const FastDiv &div) { return static_cast<int>(div.div(static_cast<uint32_t>(n))); }
__device__ __forceinline__ long long divide(long long n, long long by, const FastDiv &) { return n / by; }

template <typename T, typename I>
__global__ void __launch_bounds__(kCkThreads)
pack_element_kernel(const T *__restrict__ src, int8_t *__restrict__ codes, uint8_t *__restrict__ scales,
                    I nblocks, I dim, I blocks_row, FastDiv row_div) {
    const int lane = threadIdx.x & 31;
    const I step = kElemBlocks * kElemRounds;
    const I stride = static_cast<I>(gridDim.x) * (kCkThreads / 32) * step;
    for (I first = (static_cast<I>(blockIdx.x) * (kCkThreads / 32) + (threadIdx.x >> 5)) * step;
         first < nblocks; first += stride) {
        I at[kElemRounds];
        int left[kElemRounds];                        // elements inside the row from this lane's first on; may be negative
        float x[kElemRounds][kElems];
#pragma unroll
        for (int r = 0; r < kElemRounds; ++r) {
            const I b = first + r * kElemBlocks + lane / kLanes;
            const I row = divide(b, blocks_row, row_div);
            const I col = (b - row * blocks_row) * kCkptBlock + lane % kLanes;
            at[r] = row * dim + col;
            left[r] = b < nblocks ? static_cast<int>(min(dim - col, static_cast<I>(kCkptBlock))) : 0;
#pragma unroll
            for (int k = 0; k < kElems; ++k) x[r][k] = k * kLanes < left[r] ? to_float<T>(src[at[r] + k * kLanes]) : 0.f;
        }
#pragma unroll
        for (int r = 0; r < kElemRounds; ++r) {
            const I b = first + r * kElemBlocks + lane / kLanes;
            const CkptScale s = ckpt_scale(block_lanes_max<kElems>(max_abs_bits<kElems>(x[r])));
#pragma unroll
            for (int k = 0; k < kElems; ++k)
                if (k * kLanes < left[r]) codes[at[r] + k * kLanes] = static_cast<int8_t>(ckpt_code(x[r][k], s.inv) & s.keep);
            if (lane % kLanes == 0 && b < nblocks) scales[b] = static_cast<uint8_t>(s.e);
        }
    }
}

// 32-bit indices and a division by multiply-high while all elements of the padded rows, and the last round's
// overhang of every warp, fit 31 bits; 64-bit ones beyond.
inline bool narrow_blocks(int64_t nblocks) { return (nblocks + kMaxElementBlocks) * kCkptBlock < (1ll << 31); }
inline unsigned element_grid(int64_t nblocks) { return ck_grid((nblocks + kElemRounds * kElemBlocks - 1) / (kElemRounds * kElemBlocks) * 32); }

template <typename T>
cudaError_t pack_dispatch(const void *src, int8_t *codes, uint8_t *scales, int64_t rows, int64_t dim,
                          cudaStream_t stream) {
    constexpr int VEC = VecOf<T>::N;
    using CV = typename CodeVec<VEC>::type;
    const int64_t blocks_row = ckpt_blocks(dim), nblocks = rows * blocks_row;
    const int64_t slots_row = blocks_row * (kCkptBlock / VEC), nslots = rows * slots_row;
    const bool vec = dim % VEC == 0 && aligned(src, 16) && aligned(codes, VEC);
    if (vec && dim % kCkptBlock == 0) {
        pack_vec_kernel<T, false><<<ck_grid((nslots + kVecs - 1) / kVecs), kCkThreads, 0, stream>>>(
            static_cast<const uint4 *>(src), reinterpret_cast<CV *>(codes), scales, nslots, 1, FastDiv::make(1), 1);
    } else if (vec && nslots < (1ll << 31) - kVecs * kCkThreads) {
        pack_vec_kernel<T, true><<<ck_grid((nslots + kVecs - 1) / kVecs), kCkThreads, 0, stream>>>(
            static_cast<const uint4 *>(src), reinterpret_cast<CV *>(codes), scales, nslots,
            static_cast<uint32_t>(slots_row), FastDiv::make(static_cast<uint32_t>(slots_row)),
            static_cast<uint32_t>(dim / VEC));
    } else {
        if (narrow_blocks(nblocks))
            pack_element_kernel<T, int><<<element_grid(nblocks), kCkThreads, 0, stream>>>(
                static_cast<const T *>(src), codes, scales, static_cast<int>(nblocks), static_cast<int>(dim),
                static_cast<int>(blocks_row), FastDiv::make(static_cast<uint32_t>(blocks_row)));
        else
            pack_element_kernel<T, long long><<<element_grid(nblocks), kCkThreads, 0, stream>>>(
                static_cast<const T *>(src), codes, scales, nblocks, dim, blocks_row, FastDiv::make(1));
    }
    cudaError_t err = cudaGetLastError();
    if (err == cudaSuccess) g_launches.fetch_add(1);
    return err;
}

// ---- expand -------------------------------------------------------------------------------------
template <typename T, bool RAGGED>
__global__ void __launch_bounds__(kCkThreads)
unpack_vec_kernel(const typename CodeVec<VecOf<T>::N>::type *__restrict__ codes, const uint8_t *__restrict__ scales,
                  uint4 *__restrict__ dst, long long nvec, uint32_t vecs_row, FastDiv vecs_div, uint32_t blocks_row) {
    constexpr int VEC = VecOf<T>::N;
    constexpr int LANES = kCkptBlock / VEC;
    const long long stride = static_cast<long long>(gridDim.x) * kCkThreads * kVecs;
    for (long long base = static_cast<long long>(blockIdx.x) * kCkThreads * kVecs + threadIdx.x; base < nvec; base += stride) {
        typename CodeVec<VEC>::type c[kVecs];
        uint8_t e[kVecs];
#pragma unroll
        for (int k = 0; k < kVecs; ++k) {
            const long long i = base + k * kCkThreads;
            if (i >= nvec) continue;
            long long block = i / LANES;
            if (RAGGED) {
                const uint32_t row = vecs_div.div(static_cast<uint32_t>(i));
                const uint32_t col = static_cast<uint32_t>(i) - row * vecs_row;
                block = static_cast<long long>(row) * blocks_row + col / LANES;
            }
            c[k] = __ldcs(codes + i);
            e[k] = __ldg(scales + block);
        }
#pragma unroll
        for (int k = 0; k < kVecs; ++k) {
            const long long i = base + k * kCkThreads;
            if (i >= nvec) continue;
            float f[VEC];
            ckpt_values(c[k], ckpt_step(e[k]), f);
            st_stream(dst + i, pack<T>(f));
        }
    }
}

template <typename T, typename I>
__global__ void __launch_bounds__(kCkThreads)
unpack_element_kernel(const int8_t *__restrict__ codes, const uint8_t *__restrict__ scales, T *__restrict__ dst,
                      I nblocks, I dim, I blocks_row, FastDiv row_div) {
    const int lane = threadIdx.x & 31;
    const I step = kElemBlocks * kElemRounds;
    const I stride = static_cast<I>(gridDim.x) * (kCkThreads / 32) * step;
    for (I first = (static_cast<I>(blockIdx.x) * (kCkThreads / 32) + (threadIdx.x >> 5)) * step;
         first < nblocks; first += stride) {
        I at[kElemRounds];
        int left[kElemRounds];
        int8_t c[kElemRounds][kElems];
        uint8_t e[kElemRounds];
#pragma unroll
        for (int r = 0; r < kElemRounds; ++r) {
            const I b = first + r * kElemBlocks + lane / kLanes;
            const I row = divide(b, blocks_row, row_div);
            const I col = (b - row * blocks_row) * kCkptBlock + lane % kLanes;
            at[r] = row * dim + col;
            left[r] = b < nblocks ? static_cast<int>(min(dim - col, static_cast<I>(kCkptBlock))) : 0;
            e[r] = b < nblocks ? scales[b] : 0;
#pragma unroll
            for (int k = 0; k < kElems; ++k) c[r][k] = k * kLanes < left[r] ? codes[at[r] + k * kLanes] : 0;
        }
#pragma unroll
        for (int r = 0; r < kElemRounds; ++r)
#pragma unroll
            for (int k = 0; k < kElems; ++k)
                if (k * kLanes < left[r]) dst[at[r] + k * kLanes] = from_float<T>(ckpt_value(c[r][k], e[r]));
    }
}

template <typename T>
cudaError_t unpack_dispatch(const int8_t *codes, const uint8_t *scales, void *dst, int64_t rows, int64_t dim,
                            cudaStream_t stream) {
    constexpr int VEC = VecOf<T>::N;
    using CV = typename CodeVec<VEC>::type;
    const int64_t blocks_row = ckpt_blocks(dim), nblocks = rows * blocks_row;
    const int64_t vecs_row = dim / VEC, nvec = rows * vecs_row;
    const bool vec = dim % VEC == 0 && aligned(dst, 16) && aligned(codes, VEC);
    if (vec && dim % kCkptBlock == 0) {
        unpack_vec_kernel<T, false><<<ck_grid((nvec + kVecs - 1) / kVecs), kCkThreads, 0, stream>>>(
            reinterpret_cast<const CV *>(codes), scales, static_cast<uint4 *>(dst), nvec, 1, FastDiv::make(1), 1);
    } else if (vec && nvec < (1ll << 31)) {
        unpack_vec_kernel<T, true><<<ck_grid((nvec + kVecs - 1) / kVecs), kCkThreads, 0, stream>>>(
            reinterpret_cast<const CV *>(codes), scales, static_cast<uint4 *>(dst), nvec, static_cast<uint32_t>(vecs_row),
            FastDiv::make(static_cast<uint32_t>(vecs_row)), static_cast<uint32_t>(blocks_row));
    } else {
        if (narrow_blocks(nblocks))
            unpack_element_kernel<T, int><<<element_grid(nblocks), kCkThreads, 0, stream>>>(
                codes, scales, static_cast<T *>(dst), static_cast<int>(nblocks), static_cast<int>(dim),
                static_cast<int>(blocks_row), FastDiv::make(static_cast<uint32_t>(blocks_row)));
        else
            unpack_element_kernel<T, long long><<<element_grid(nblocks), kCkThreads, 0, stream>>>(
                codes, scales, static_cast<T *>(dst), nblocks, dim, blocks_row, FastDiv::make(1));
    }
    cudaError_t err = cudaGetLastError();
    if (err == cudaSuccess) g_launches.fetch_add(1);
    return err;
}

// ---- GEGLU gate with a checkpoint of its input [rows, 2 D] -----------------------------------------
// PACK: D a multiple of 32, so that no block holds elements of both halves; otherwise the gate alone, and
// pack_dispatch does the rest.  The gate itself is the arithmetic of gelu_multiply: the same bits come out.
template <typename T, bool PACK>
__global__ void __launch_bounds__(kCkThreads)
geglu_pack_kernel(const uint4 *__restrict__ ab, uint4 *__restrict__ dst,
                  typename CodeVec<VecOf<T>::N>::type *__restrict__ codes, uint8_t *__restrict__ scales,
                  long long nvec, FastDiv dvec_div, uint32_t dvec) {
    constexpr int VEC = VecOf<T>::N;
    constexpr int LANES = kCkptBlock / VEC;
    constexpr bool HALF = sizeof(T) == 2;
    const long long stride = static_cast<long long>(gridDim.x) * kCkThreads * kGateVecs;
    for (long long base = static_cast<long long>(blockIdx.x) * kCkThreads * kGateVecs + (threadIdx.x & ~31); base < nvec;
         base += stride) {
        long long at[kGateVecs];
        uint4 va[kGateVecs], vg[kGateVecs];
#pragma unroll
        for (int k = 0; k < kGateVecs; ++k) {
            const long long i = base + k * kCkThreads + (threadIdx.x & 31);
            const uint32_t n = static_cast<uint32_t>(i < nvec ? i : 0);
            const uint32_t r = dvec_div.div(n);
            at[k] = static_cast<long long>(r) * 2 * dvec + (n - r * dvec);
            va[k] = vg[k] = make_uint4(0, 0, 0, 0);
            if (i < nvec) {
                va[k] = ld_stream(ab + at[k]);
                vg[k] = ld_stream(ab + at[k] + dvec);
            }
        }
#pragma unroll
        for (int k = 0; k < kGateVecs; ++k) {
            const long long i = base + k * kCkThreads + (threadIdx.x & 31);
            float a[VEC], g[VEC];
            unpack<T>(va[k], a);
            unpack<T>(vg[k], g);
            if constexpr (PACK) {
                const CkptScale sa = ckpt_scale(block_lanes_max<VEC>(max_abs_bits<T>(va[k])));
                const CkptScale sg = ckpt_scale(block_lanes_max<VEC>(max_abs_bits<T>(vg[k])));
                if (i < nvec) {
                    codes[at[k]] = ckpt_codes(a, sa);
                    codes[at[k] + dvec] = ckpt_codes(g, sg);
                    if ((threadIdx.x & (LANES - 1)) == 0) {
                        scales[at[k] / LANES] = static_cast<uint8_t>(sa.e);
                        scales[(at[k] + dvec) / LANES] = static_cast<uint8_t>(sg.e);
                    }
                }
            }
            if (i < nvec) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) a[j] = a[j] * gelu_erf<HALF>(g[j]);
                st_stream(dst + i, pack<T>(a));
            }
        }
    }
}

// 32-bit indices as far as the input's elements and a grid's overhang go.
inline bool narrow_gate(int64_t rows, int64_t d) { return 2 * rows * d + kMaxGridThreads * kGateElems < (1ll << 31); }

// The gate alone, element by element, for rows that are not whole vectors.
template <typename T, typename I>
__global__ void __launch_bounds__(kCkThreads)
geglu_element_kernel(const T *__restrict__ ab, T *__restrict__ dst, I rows, I d, FastDiv row_div) {
    constexpr bool HALF = sizeof(T) == 2;
    const I total = rows * d, stride = static_cast<I>(gridDim.x) * kCkThreads * kGateElems;
    for (I base = static_cast<I>(blockIdx.x) * kCkThreads * kGateElems + threadIdx.x; base < total; base += stride) {
        float a[kGateElems], g[kGateElems];
#pragma unroll
        for (int k = 0; k < kGateElems; ++k) {
            const I i = base + k * kCkThreads;
            if (i >= total) continue;
            const I at = i + divide(i, d, row_div) * d;           // r * 2 d + j
            a[k] = to_float<T>(ab[at]);
            g[k] = to_float<T>(ab[at + d]);
        }
#pragma unroll
        for (int k = 0; k < kGateElems; ++k) {
            const I i = base + k * kCkThreads;
            if (i < total) dst[i] = from_float<T>(a[k] * gelu_erf<HALF>(g[k]));
        }
    }
}

template <typename T>
cudaError_t geglu_pack_dispatch(const void *ab, void *dst, int8_t *codes, uint8_t *scales, int64_t rows, int64_t d,
                                cudaStream_t stream) {
    constexpr int VEC = VecOf<T>::N;
    using CV = typename CodeVec<VEC>::type;
    const int64_t nvec = rows * (d / VEC);
    if (d % VEC == 0 && aligned(ab, 16) && aligned(dst, 16) && nvec < (1ll << 31)) {
        const uint32_t dvec = static_cast<uint32_t>(d / VEC);
        const unsigned grid = ck_grid((nvec + kGateVecs - 1) / kGateVecs);
        const bool pack = d % kCkptBlock == 0 && aligned(codes, VEC);
        if (pack)
            geglu_pack_kernel<T, true><<<grid, kCkThreads, 0, stream>>>(
                static_cast<const uint4 *>(ab), static_cast<uint4 *>(dst), reinterpret_cast<CV *>(codes), scales, nvec,
                FastDiv::make(dvec), dvec);
        else
            geglu_pack_kernel<T, false><<<grid, kCkThreads, 0, stream>>>(static_cast<const uint4 *>(ab),
                                                                        static_cast<uint4 *>(dst), nullptr, nullptr, nvec,
                                                                        FastDiv::make(dvec), dvec);
        cudaError_t err = cudaGetLastError();
        if (err != cudaSuccess) return err;
        g_launches.fetch_add(1);
        return pack ? cudaSuccess : pack_dispatch<T>(ab, codes, scales, rows, 2 * d, stream);
    }
    if (narrow_gate(rows, d))
        geglu_element_kernel<T, int><<<ck_grid((rows * d + kGateElems - 1) / kGateElems), kCkThreads, 0, stream>>>(
            static_cast<const T *>(ab), static_cast<T *>(dst), static_cast<int>(rows), static_cast<int>(d),
            FastDiv::make(static_cast<uint32_t>(d)));
    else
        geglu_element_kernel<T, long long><<<ck_grid((rows * d + kGateElems - 1) / kGateElems), kCkThreads, 0, stream>>>(
            static_cast<const T *>(ab), static_cast<T *>(dst), rows, d, FastDiv::make(1));
    cudaError_t err = cudaGetLastError();
    if (err != cudaSuccess) return err;
    g_launches.fetch_add(1);
    return pack_dispatch<T>(ab, codes, scales, rows, 2 * d, stream);
}

// ---- backward of the gate -----------------------------------------------------------------------
// y = a gelu(g), gelu(g) = g Phi(g):  da = dy g Phi(g),  dg = dy a (Phi(g) + g phi(g)).
// Phi(-|g|) = t P(t) e with e = exp(-g^2 / 2), which phi needs too, and t = 1 / (1 + q |g|): the tail without a difference
// of numbers near 1, so that it is right to a few roundings (and g^2 of them in e's exponent) however small it is.  P is
// fitted to exp(g^2 / 2) Phi(-g) / t in 64 bits on 0 <= g <= 13.5, beyond which e is 0, for the smallest relative error
// (least squares at Chebyshev nodes, weights times the error until it is level), q by a scan.  Degree 8: 2.6e-8, and 3.0e-7
// with fp32 roundings; degree 6 for 16-bit results: 6.2e-7, and 9.1e-7.  (1 + erf has no right bits left below g = -5.5;
// erfcf has, and takes 123 us from a checkpoint of [16384, 5120] in fp32 where this takes 95.)
template <bool HALF> __device__ __forceinline__ void gelu_grad(float g, float *value, float *slope) {
    const float t = rcp_approx(fmaf(HALF ? 0.265f : 0.34f, fabsf(g), 1.0f));
    float p;
    if (HALF) {
        p = fmaf(-0.0677870587f, t, 0.195273221f);
        p = fmaf(p, t, -0.066363059f);
        p = fmaf(p, t, 0.142493412f);
        p = fmaf(p, t, 0.0829465538f);
        p = fmaf(p, t, 0.107836783f);
        p = fmaf(p, t, 0.105599828f);
    } else {
        p = fmaf(-0.0263702534f, t, 0.140672088f);
        p = fmaf(p, t, -0.27546227f);
        p = fmaf(p, t, 0.204732612f);
        p = fmaf(p, t, -0.0463950336f);
        p = fmaf(p, t, 0.116034947f);
        p = fmaf(p, t, 0.115035095f);
        p = fmaf(p, t, 0.136133477f);
        p = fmaf(p, t, 0.135619342f);
    }
    const float e = ex2_approx(-0.72134752044448170368f * g * g);
    const float tail = p * t * e;
    const float cdf = g < 0.f ? tail : 1.0f - tail;
    *value = g * cdf;
    *slope = fmaf(g, e * 0.39894228040143267794f, cdf);
}

template <typename T, bool CKPT>
__global__ void __launch_bounds__(kCkThreads)
geglu_backward_vec_kernel(const uint4 *ab, const typename CodeVec<VecOf<T>::N>::type *__restrict__ codes,
                          const uint8_t *__restrict__ scales, const uint4 *dy, uint4 *dab, long long nvec,
                          FastDiv dvec_div, uint32_t dvec, uint32_t blocks_row) {
    constexpr int VEC = VecOf<T>::N;
    constexpr int LANES = kCkptBlock / VEC;
    const long long stride = static_cast<long long>(gridDim.x) * kCkThreads;
    for (long long i = static_cast<long long>(blockIdx.x) * kCkThreads + threadIdx.x; i < nvec; i += stride) {
        const uint32_t r = dvec_div.div(static_cast<uint32_t>(i));
        const uint32_t j = static_cast<uint32_t>(i) - r * dvec;
        const long long at = static_cast<long long>(r) * 2 * dvec + j;
        float a[VEC], g[VEC], d[VEC];
        if (CKPT) {
            const uint8_t *row = scales + static_cast<long long>(r) * blocks_row;
            const auto ca = __ldcs(codes + at), cg = __ldcs(codes + at + dvec);
            ckpt_values(ca, ckpt_step(__ldg(row + j / LANES)), a);
            ckpt_values(cg, ckpt_step(__ldg(row + (j + dvec) / LANES)), g);
        } else {
            const uint4 va = ld_stream(ab + at), vg = ld_stream(ab + at + dvec);
            unpack<T>(va, a);
            unpack<T>(vg, g);
        }
        unpack<T>(ld_stream(dy + i), d);
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            float value, slope;
            gelu_grad<sizeof(T) == 2>(g[k], &value, &slope);
            g[k] = d[k] * a[k] * slope;
            a[k] = d[k] * value;
        }
        st_stream(dab + at, pack<T>(a));
        st_stream(dab + at + dvec, pack<T>(g));
    }
}

template <typename T, bool CKPT, typename I>
__global__ void __launch_bounds__(kCkThreads)
geglu_backward_element_kernel(const T *ab, const int8_t *__restrict__ codes, const uint8_t *__restrict__ scales,
                              const T *dy, T *dab, I rows, I d, I blocks_row, FastDiv row_div) {
    const I total = rows * d, stride = static_cast<I>(gridDim.x) * kCkThreads * kGateElems;
    for (I base = static_cast<I>(blockIdx.x) * kCkThreads * kGateElems + threadIdx.x; base < total; base += stride) {
        I at[kGateElems];
        float a[kGateElems], g[kGateElems], grad[kGateElems];
#pragma unroll
        for (int k = 0; k < kGateElems; ++k) {
            const I i = base + k * kCkThreads;
            if (i >= total) continue;
            const I r = divide(i, d, row_div), j = i - r * d;
            at[k] = r * 2 * d + j;
            if (CKPT) {
                a[k] = ckpt_value(codes[at[k]], scales[r * blocks_row + j / kCkptBlock]);
                g[k] = ckpt_value(codes[at[k] + d], scales[r * blocks_row + (j + d) / kCkptBlock]);
            } else {
                a[k] = to_float<T>(ab[at[k]]);
                g[k] = to_float<T>(ab[at[k] + d]);
            }
            grad[k] = to_float<T>(dy[i]);
        }
#pragma unroll
        for (int k = 0; k < kGateElems; ++k) {
            if (base + k * kCkThreads >= total) continue;
            float value, slope;
            gelu_grad<sizeof(T) == 2>(g[k], &value, &slope);
            dab[at[k]] = from_float<T>(grad[k] * value);
            dab[at[k] + d] = from_float<T>(grad[k] * a[k] * slope);
        }
    }
}

template <typename T, bool CKPT>
cudaError_t geglu_backward_dispatch(const void *ab, const int8_t *codes, const uint8_t *scales, const void *dy, void *dab,
                                    int64_t rows, int64_t d, cudaStream_t stream) {
    constexpr int VEC = VecOf<T>::N;
    using CV = typename CodeVec<VEC>::type;
    const int64_t nvec = rows * (d / VEC), blocks_row = ckpt_blocks(2 * d);
    const bool src_ok = CKPT ? aligned(codes, VEC) : aligned(ab, 16);
    if (d % VEC == 0 && src_ok && aligned(dy, 16) && aligned(dab, 16) && nvec < (1ll << 31)) {
        const uint32_t dvec = static_cast<uint32_t>(d / VEC);
        geglu_backward_vec_kernel<T, CKPT><<<ck_grid(nvec), kCkThreads, 0, stream>>>(
            static_cast<const uint4 *>(ab), reinterpret_cast<const CV *>(codes), scales, static_cast<const uint4 *>(dy),
            static_cast<uint4 *>(dab), nvec, FastDiv::make(dvec), dvec, static_cast<uint32_t>(blocks_row));
    } else {
        if (narrow_gate(rows, d))
            geglu_backward_element_kernel<T, CKPT, int><<<ck_grid((rows * d + kGateElems - 1) / kGateElems), kCkThreads, 0, stream>>>(
                static_cast<const T *>(ab), codes, scales, static_cast<const T *>(dy), static_cast<T *>(dab),
                static_cast<int>(rows), static_cast<int>(d), static_cast<int>(blocks_row),
                FastDiv::make(static_cast<uint32_t>(d)));
        else
            geglu_backward_element_kernel<T, CKPT, long long><<<ck_grid((rows * d + kGateElems - 1) / kGateElems), kCkThreads, 0, stream>>>(
                static_cast<const T *>(ab), codes, scales, static_cast<const T *>(dy), static_cast<T *>(dab), rows, d,
                blocks_row, FastDiv::make(1));
    }
    cudaError_t err = cudaGetLastError();
    if (err == cudaSuccess) g_launches.fetch_add(1);
    return err;
}

template <typename T>
cudaError_t geglu_backward_source(const void *ab, const int8_t *codes, const uint8_t *scales, const void *dy, void *dab,
                                  int64_t rows, int64_t d, cudaStream_t stream) {
    return codes ? geglu_backward_dispatch<T, true>(ab, codes, scales, dy, dab, rows, d, stream)
                 : geglu_backward_dispatch<T, false>(ab, codes, scales, dy, dab, rows, d, stream);
}

}  // namespace

cudaError_t ckpt_pack_launch(const void *src, int8_t *codes, uint8_t *scales, int64_t rows, int64_t dim, int dtype,
                             cudaStream_t stream) {
    switch (dtype) {
        case kF16: return pack_dispatch<__half>(src, codes, scales, rows, dim, stream);
        case kBF16: return pack_dispatch<__nv_bfloat16>(src, codes, scales, rows, dim, stream);
        default: return pack_dispatch<float>(src, codes, scales, rows, dim, stream);
    }
}

cudaError_t ckpt_unpack_launch(const int8_t *codes, const uint8_t *scales, void *dst, int64_t rows, int64_t dim, int dtype,
                               cudaStream_t stream) {
    switch (dtype) {
        case kF16: return unpack_dispatch<__half>(codes, scales, dst, rows, dim, stream);
        case kBF16: return unpack_dispatch<__nv_bfloat16>(codes, scales, dst, rows, dim, stream);
        default: return unpack_dispatch<float>(codes, scales, dst, rows, dim, stream);
    }
}

cudaError_t geglu_pack_launch(const void *ab, void *dst, int8_t *codes, uint8_t *scales, int64_t rows, int64_t d,
                              int dtype, cudaStream_t stream) {
    switch (dtype) {
        case kF16: return geglu_pack_dispatch<__half>(ab, dst, codes, scales, rows, d, stream);
        case kBF16: return geglu_pack_dispatch<__nv_bfloat16>(ab, dst, codes, scales, rows, d, stream);
        default: return geglu_pack_dispatch<float>(ab, dst, codes, scales, rows, d, stream);
    }
}

cudaError_t geglu_backward_launch(const void *ab, const int8_t *codes, const uint8_t *scales, const void *dy, void *dab,
                                  int64_t rows, int64_t d, int dtype, cudaStream_t stream) {
    switch (dtype) {
        case kF16: return geglu_backward_source<__half>(ab, codes, scales, dy, dab, rows, d, stream);
        case kBF16: return geglu_backward_source<__nv_bfloat16>(ab, codes, scales, dy, dab, rows, d, stream);
        default: return geglu_backward_source<float>(ab, codes, scales, dy, dab, rows, d, stream);
    }
}

}  // namespace sdfl
