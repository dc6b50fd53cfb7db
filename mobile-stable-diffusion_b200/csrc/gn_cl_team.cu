// Channels-last GroupNorm (+SiLU) and its gradient in one persistent launch (plus a small one that adds
// up the weight gradients).  Formulas and layout: gn_cl_device.cuh.
//
// What it cannot do without is one read and one write of the tensor (forward), or reads of x (or its
// checkpoint) and grad_out and one write (backward); but a group's first result needs its last element,
// so every element is read twice, the second time from shared memory or from L2.  What bounds the
// forward pass is the sum of the HBM reads of pass S, the L2 reads, arithmetic and stores of pass A and the
// exchange between them ([4, 262144, 128] fp16 with SiLU, when it took 134 us: S alone 52 us, 5.1 TB/s; A's loads and the
// exchange 42; A's arithmetic and stores, which overlap, 40).  The backward pass is bound by latency: about 17
// instructions per element and pass, of which 16 consumer warps per SM issue 0.53 per cycle and scheduler; the SFU is
// its busiest pipe (51 %).
// Measured (B200, back to back in a captured graph; share of the measured copy bandwidth by the bytes above):
//   forward   [4, 262144, 128] fp16 SiLU 127 us (65 %), [4, 65536, 320] bf16 SiLU 96 us (54 %), [8, 4096, 512] fp16 25 us
//             (41 %), [3, 2961, 640] fp32 16 us (43 %), [2, 64, 1280] fp16 8.1 us; with a checkpoint [4, 16384, 512] fp16
//             47 us (56 %)
//   backward  [2, 262144, 64] fp32 113 us (55 %), [4, 65536, 320] bf16 165 us (47 %), [8, 4096, 320] bf16 32 us (31 %),
//             [4, 1024, 640] bf16 15 us; from a checkpoint [4, 65536, 256] bf16 124 us (42 %), [4, 16384, 512] fp16 68 us (39 %)
//
// Split.  An item is a slice of an image's channels (whole groups and whole vectors, a 128-byte row or
// more where the sizes allow it) over all its pixels.  A team of M thread blocks works on one item at a
// time, each block on its own range of pixels: pass S reads and sums, the blocks' sums are exchanged,
// pass A reads again and writes.
//   - Small tensors: one item per team, its share of it in a block's shared memory and read once; a team is
//     a thread-block cluster and the exchange goes through distributed shared memory: one launch, no
//     workspace.
//   - Otherwise teams of resident blocks.  If all items fit the rings at once they are read once; if not, the
//     images that are open at a time hold at most kInFlight bytes, so that the second read comes from L2
//     whatever the tensor's size.  Where that leaves two teams of one block per SM, the second starts
//     behind the first one's pass S, so that one team's reading, which waits for HBM, runs beside the
//     other's writing, which computes (134 -> 128 us).
// (Alternating the chunks of S of one item with those of A of another in the same block was tried and is
// 15 % slower: three items per team are open then, so they are smaller, and what a block spends per
// item -- about 5 us for adding up and exchanging -- is paid more often.)
//
// Loads.  A producer warp keeps a ring of chunks filled by tiled bulk copies (a chunk is kRounds rows per
// consumer thread, the box of a 2-D tensor map over [batch * hw, channels]); the consumer warps wait on
// a chunk's "full" mbarrier and release it through its "empty" one.  The ring runs on over the end of
// a pass: while a block adds up its rows and waits for the others' sums, the first chunks of the next
// pass are already under way.  The copies cost the consumers no instructions (per-thread cp.async into the same ring: 12
// more per vector).
//
// Exchange outside clusters.  A block writes its sums per group to the workspace and counts itself in (the counters are
// zeroed by a small kernel in front); before pass A one thread of a block polls the count, then
// the block merges all of the team's sums itself, in block order (the same bits on every run).  Every
// block of the grid is resident (cooperative launch), and every wait is bounded: on time-out the
// status word is raised and the launch finishes with an invalid result.
// (Sums that carry their own "written" mark, polled by all warps, save the fence and the counter but
// were 10 % slower: the polling takes issue slots and L2 bandwidth from the blocks that still compute.)
//
// Weight gradients: a block adds up its channels' sums over the images of its slice in shared memory and
// writes them once per slice; cl_param_sum_kernel adds the blocks' rows.
#include "gn_cl_device.cuh"
#include "gn_cl_internal.h"
#include "gn_device.cuh"

#include <cuda.h>

#include <algorithm>
#include <numeric>

namespace sdfl {

namespace {

constexpr int kThreads = 256;                      // consumers
constexpr int kWarps = kThreads / 32;
constexpr int kBlock = kThreads + 32;              // and the producer warp
constexpr int kBlocksPerSm = 2;
// Rows per thread and chunk, and chunks of the ring.
constexpr int kRounds = 4, kStages = 5;            // 16 KB chunks
// Backward, by the source: 16 KB of grad_out and 8 or 4 KB of codes, or 8 KB of grad_out and 8 KB of x, so that
// two blocks fit an SM either way (three chunks of 32 KB leave room for one: 35 us instead of 31 at
// [8, 4096, 320] bf16).
__host__ __device__ constexpr int rounds_grad(bool ckpt) { return ckpt ? 4 : 2; }
__host__ __device__ constexpr int stages_grad(bool ckpt) { return ckpt ? 3 : 5; }
constexpr int kMaxCols = kThreads / 2;             // columns of a slice: a box row of 2 KB
constexpr int kMergeLoads = 5;                     // a team of up to 160 blocks in one round
constexpr int64_t kInFlight = 72ll << 20;          // twice that in the backward pass
// Clusters of up to 4 start as fast as single blocks.  Clusters of 8 start 2 us later, so that [2, 4096, 320]
// fp16 takes 12.1 us in a captured graph where a cooperative grid takes 11.0, but the call is one launch
// instead of two: 13 us against 16 when calls are made one by one.  Clusters of 16 start 7 us later.
constexpr int kMaxCluster = 8;
constexpr size_t kMaxShared = 200 * 1024;
constexpr int64_t kSmShared = 228 * 1024;          // of an SM
constexpr size_t kTwoOnSm = kSmShared / 3;         // staggered teams number their blocks by two on every SM: no room for a third
constexpr int64_t kBlockShared = 1024 + 128;       // that a block takes besides its dynamic shared memory: reserved, static
constexpr int64_t kClusterPartBytes = 4096;        // shared memory for a cluster's sums
constexpr int kMaxTeamsOfSm = kBlocksPerSm;        // teams that take turns on the SMs
constexpr int kSlotWords = 1024 + kMaxTeamsOfSm;

__device__ unsigned int g_cl_status;               // bit 0: a bounded wait ran out

struct Args {                    // one struct for both directions
    GnClForward f;
    GnClBackward b;
    GnClTeamPlan p;
    int64_t batch, hw, channels, groups;
    int width;                   // channels per group
    int chunk_rows;              // pixels per chunk
    int share, rest;             // chunks of an image / members, % members
    float eps;
    unsigned int *arrived;       // [items], then kSlotWords for the placement of blocks
    long long items;
    float2 *partial;             // [batch * groups][members]
    float2 *channel_sums;        // [slice][image_teams * members][slice channels]
};

struct Place {
    int team, member, slice_team, image_team, col, row, ncols, slice_groups;
    int first, chunks, pixels;   // this block's pixels of every item: [first, first + pixels)
    bool active;
};

// A block's share of an item is whole chunks; the image's last chunk may be short.
__device__ __forceinline__ int member_first(const Args &a, int member) {
    return (member * a.share + min(member, a.rest)) * a.chunk_rows;
}
__device__ __forceinline__ int member_pixels(const Args &a, int member) {
    const int first = member_first(a, member);
    return min(static_cast<int>(a.hw) - first, (a.share + (member < a.rest ? 1 : 0)) * a.chunk_rows);
}

// Two teams that run out of step must share every SM evenly: two blocks of one team on an SM would do their
// computing at the same time and keep the rest of the team waiting (the hardware puts blocks i and
// i + #SMs together on most SMs only; 23 instead of 14 us for pass A on the others).  So a block takes its
// number from its SM: the SM's k-th block is a member of team k.
__device__ __forceinline__ int block_number(const Args &a) {
    if (!a.p.stagger) return blockIdx.x;
    __shared__ int number;
    if (threadIdx.x == 0) {
        unsigned int sm;
        asm volatile("mov.u32 %0, %smid;" : "=r"(sm));
        unsigned int *slots = a.arrived + a.items;
        const unsigned int slot = atomicAdd(slots + kMaxTeamsOfSm + sm % (kSlotWords - kMaxTeamsOfSm), 1u) % kMaxTeamsOfSm;
        number = static_cast<int>(slot * a.p.members + atomicAdd(slots + slot, 1u) % a.p.members);
    }
    __syncthreads();
    return number;
}

__device__ __forceinline__ Place place(const Args &a) {
    Place w;
    const int block = block_number(a);
    w.team = block / a.p.members;
    w.member = block - w.team * a.p.members;
    w.slice_team = w.team % a.p.slice_teams;
    w.image_team = w.team / a.p.slice_teams;
    w.row = threadIdx.x / a.p.cols;
    w.col = threadIdx.x - w.row * a.p.cols;
    w.active = w.row < a.p.rows;
    w.ncols = a.p.cols * a.p.vec;
    w.slice_groups = w.ncols / a.width;
    w.first = member_first(a, w.member);
    w.chunks = a.share + (w.member < a.rest ? 1 : 0);
    w.pixels = member_pixels(a, w.member);
    return w;
}

// A team's items, slice by slice and image by image within a slice.
struct Cursor {
    int slice, image;
    __device__ __forceinline__ void next(const Args &a, const Place &w) {
        image += a.p.image_teams;
        if (image >= static_cast<int>(a.batch)) {
            image = w.image_team;
            slice += a.p.slice_teams;
        }
    }
};

// A team's passes: S and A of an item, then the next item.
struct Passes {
    Cursor now;
    bool second;
    __device__ __forceinline__ explicit Passes(const Place &w) : now{w.slice_team, w.image_team}, second(true) {
        now.image -= 1;                               // nothing yet
    }
    // false: none left
    __device__ __forceinline__ bool next(const Args &a, const Place &w) {
        second = !second;
        if (!second) {
            if (now.image < w.image_team) now.image = w.image_team;
            else now.next(a, w);
        }
        return now.slice < a.p.slices;
    }
};

// One box of a tensor map into shared memory; x in 8-byte units (even: 16-byte aligned), y a pixel row.
__device__ __forceinline__ void box_load(uint32_t dst, const CUtensorMap *map, int x, int y, uint32_t bar, uint64_t policy) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint "
        "[%0], [%1, {%2, %3}], [%4], %5;"
        ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar), "l"(policy)
        : "memory");
}

// The ring's barriers; waits are bounded, a time-out is recorded and the block carries on.
template <int STAGES> struct Ring {
    uint32_t full, empty;        // shared addresses of STAGES mbarriers each
    int stage;
    uint32_t phase;
    long long patience;          // of a wait; short once one has run out, so that a broken launch ends soon
    __device__ __forceinline__ void init(uint64_t *bars) {
        patience = kWaitCycles;
        full = smem_addr(bars);
        empty = full + 8 * STAGES;
        stage = 0;
        phase = 0;
        if (threadIdx.x == 0) {
            for (int i = 0; i < STAGES; ++i) {
                mbar_init(full + 8 * i, 1);
                mbar_init(empty + 8 * i, kWarps);
            }
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
    }
    __device__ __forceinline__ void wait(uint32_t bar, uint32_t parity) {
        if (!mbar_wait_bounded(bar + 8 * stage, parity, patience)) {
            atomicOr(&g_cl_status, 1u);
            patience = kWaitCyclesAfterTimeout;
        }
    }
    __device__ __forceinline__ void wait_full() { wait(full, phase); }
    __device__ __forceinline__ void wait_empty() { wait(empty, phase ^ 1u); }
    // a consumer warp has read its part of the chunk
    __device__ __forceinline__ void release() {
        __syncwarp();
        if ((threadIdx.x & 31) == 0) mbar_arrive(empty + 8 * stage);
        next();
    }
    __device__ __forceinline__ void rewind() {           // to the first chunk of a ring that is never released
        stage = 0;
        phase = 0;
    }
    __device__ __forceinline__ void next() {
        if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
        }
    }
};

__device__ __forceinline__ void block_sync() { consumer_sync(kThreads); }       // the consumer warps

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// ---- exchange ---------------------------------------------------------------------------------------
// Counts the block in on an item; its sums were written (by any thread) before.
__device__ __forceinline__ void arrive(const Args &a, int64_t item) {
    block_sync();
    if (threadIdx.x == 0 && a.p.members > 1) {        // a team of one has read its own sums behind the barrier
        __threadfence();
        atomicAdd(a.arrived + item, 1u);
    }
}

__device__ __forceinline__ void wait_count(const Args &a, int64_t item, unsigned int count, unsigned int sleep,
                                           long long &patience) {
    const long long t0 = clock64();
    for (;;) {
        unsigned int v;
        asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(a.arrived + item) : "memory");
        if (v >= count) break;
        if (clock64() - t0 > patience) {
            atomicOr(&g_cl_status, 1u);
            patience = kWaitCyclesAfterTimeout;
            break;
        }
        if (sleep) __nanosleep(sleep);
    }
}

// Waits until all of the team's blocks have counted themselves in.
__device__ __forceinline__ void wait_all(const Args &a, int64_t item, long long &patience) {
    if (threadIdx.x == 0 && a.p.members > 1) wait_count(a, item, static_cast<unsigned>(a.p.members), 0, patience);
    block_sync();
}

// One group's sums of up to 32 * kMergeLoads blocks from `first` on, every load in flight at once.
__device__ __forceinline__ void load_partials(const Args &a, const float2 *sums, int first, float2 (&v)[kMergeLoads]) {
#pragma unroll
    for (int k = 0; k < kMergeLoads; ++k) {
        v[k] = make_float2(0.f, 0.f);
        if (first + 32 * k < a.p.members) v[k] = __ldcg(sums + first + 32 * k);
    }
}
__device__ __forceinline__ void load_parts(const Args &a, const float2 *sums, int lane, float2 (&v)[kMergeLoads]) {
#pragma unroll
    for (int k = 0; k < kMergeLoads; ++k) v[k] = make_float2(0.f, 0.f);
    if (lane < a.p.members) v[0] = sums[lane];
}
__device__ __forceinline__ float pixels_or_none(const Args &a, int member) {
    return member < a.p.members ? static_cast<float>(member_pixels(a, member)) : 0.f;
}

// A team that is a thread-block cluster (one item per team): its blocks put their sums into one another's
// shared memory, part[group][member], and arrive on one another's barrier.
struct ClusterExchange {
    float2 *part;
    uint32_t bar;
    __device__ __forceinline__ void init(uint64_t *b, float2 *p, int members) {
        part = p;
        bar = smem_addr(b);
        if (threadIdx.x == 0) {
            mbar_init(bar, static_cast<uint32_t>(members) * 32u);
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
    }
    // own[g]: this block's sums, behind a barrier.  Warp m serves member m (and m + 8).
    __device__ __forceinline__ void send(const Place &w, int members, const float2 *own) const {
        for (int m = threadIdx.x >> 5; m < members; m += kWarps) {
            for (int g = threadIdx.x & 31; g < w.slice_groups; g += 32)
                st_peer_f32x2(map_to_rank(smem_addr(part + g * members + w.member), m), own[g].x, own[g].y);
            mbar_arrive_peer(map_to_rank(bar, m));
        }
    }
    __device__ __forceinline__ void wait() const {
        if (!mbar_wait_cluster_bounded(bar, 0u, kWaitCycles)) atomicOr(&g_cl_status, 1u);
    }
};

// Odd teams start when half of the blocks of the team before them are through their first pass S.
__device__ __forceinline__ void stagger(const Args &a, int team, long long &patience) {
    if (!a.p.stagger || !(team & 1)) return;
    const int before = team - 1;
    wait_count(a, static_cast<int64_t>(before / a.p.slice_teams) * a.p.slices + before % a.p.slice_teams,
               static_cast<unsigned>((a.p.members + 1) / 2), 200, patience);
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
    block_sync();
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
            block_sync();
            if (part > 0 && part < parts) buf[threadIdx.x] = s;
            block_sync();
            if (part == 0) {
                for (int k = 1; k < parts; ++k) s += buf[k * ncols + c];
                buf[c] = s;
            }
        } else if (part == 0) {
            buf[c] = s;
        }
    }
    block_sync();
}

// ---- coefficients of a channel, and which channels share a mean ----------------------------------------
// z = (x - mean) p + beta: where the mean is far from zero compared with the spread, x - mean loses nothing.  It has to
// be the mean of the channel's own group: around a neighbour's, x would be rounded at that group's distance, and an
// infinity or a NaN there would reach this one.  Where groups are whole halves of vectors (four channels), the means
// of a column sit in registers; elsewhere they are read from shared memory like p and beta.
// ([4, 65536, 320] bf16 forward, ten channels to a group: 96 us, and 94 around one mean per vector.)
enum Span : int { kHalvesWhole, kPairsWhole, kAnyChannel };

// Where an array of coefficients keeps channel c of a slice: all first halves of the columns, then all second halves, so
// that neighbouring lanes read neighbouring 16 bytes (32 apart they meet in the banks: [4, 65536, 320] bf16 backward 181 us
// instead of 165).
template <int VEC> __device__ __forceinline__ int coef_slot(int c, int cols) {
    return VEC == 4 ? c : ((c >> 2) & 1) * 4 * cols + (c >> 3) * 4 + (c & 3);
}

template <typename T, int SPAN> struct Means {
    static constexpr int N = SPAN == kHalvesWhole ? VecOf<T>::N / 4 : 0;
    Pair held[N > 0 ? N : 1];
    // at: minus the means of the first half of this thread's column; `half` floats further on those of the second
    __device__ __forceinline__ explicit Means(const float *at, int half) {
#pragma unroll
        for (int i = 0; i < N; ++i) held[i] = pair(at[i * half], at[i * half]);
    }
    __device__ __forceinline__ void get(const float *at, int half, int h, Pair (&m)[2]) const {
        if constexpr (N > 0) m[0] = m[1] = held[h];
        else quad_load(at + h * half, m);
    }
};

// ---- forward --------------------------------------------------------------------------------------
// Statistics of a block: every thread keeps sums of d = x - (its first value) and of d^2 per channel and
// turns them into a mean and a sum of squared deviations.  The block adds up n (mean - P) and M2 + n (mean - P)^2
// with P the mean of the thread in row 0: P is close to the block's mean (it can be off by an
// outlier's share of one thread's pixels, which costs at most log2(rows) bits), so the one
// subtraction that is left, of N (block mean - P)^2, cancels next to nothing.
//
// SPAN: what may lie in several groups (below).
template <typename T, int ACT, bool PACK, bool CLUSTER, int SPAN>
__global__ void __launch_bounds__(kBlock, kBlocksPerSm)
cl_team_forward_kernel(const Args a, const __grid_constant__ CUtensorMap map_x) {
    constexpr int VEC = VecOf<T>::N;
    constexpr int kChunkBytes = kRounds * kThreads * 16;
    using Col = Column<VEC>;
    extern __shared__ __align__(128) unsigned char shared[];
    __shared__ uint64_t bars[2 * kStages];
    const Place w = place(a);
    float *buf = reinterpret_cast<float *>(shared + kStages * kChunkBytes);              // [rows][2 ncols]
    float *cp = buf + 2 * kThreads * VEC;             // [ncols] each: P, later the scale; beta; minus the means
    float *cq = cp + w.ncols;
    float *means = cq + w.ncols;
    float2 *stat = reinterpret_cast<float2 *>(means + w.ncols);                         // [groups]: (mean, rstd)
    int *group_of = reinterpret_cast<int *>(stat + w.ncols);                             // [ncols], within a slice
    float2 *own = reinterpret_cast<float2 *>(group_of + w.ncols);                        // cluster: [groups], then
    ClusterExchange cluster;                                                             // [groups][members]
    __shared__ uint64_t cluster_bar;
    // a team's only item that fits the ring is read once
    const bool resident = a.p.resident != 0;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    Passes passes(w);
    Ring<kStages> ring;
    ring.init(bars);
    if constexpr (CLUSTER) cluster.init(&cluster_bar, own + w.slice_groups, a.p.members);
    for (int c = threadIdx.x; c < w.ncols; c += kBlock) group_of[c] = c / a.width;
    __syncthreads();
    if constexpr (CLUSTER) cluster_arrive();          // the barriers are set up; waited for before the first store to a peer

    if (warp == kWarps) {                             // producer
        if (lane == 0) {
            stagger(a, w.team, ring.patience);
            const uint64_t done = policy_evict_first(), again = resident ? done : policy_evict_last();
            const uint32_t bytes = static_cast<uint32_t>(a.chunk_rows * w.ncols * sizeof(T));
            while (passes.next(a, w)) {
                if (passes.second && resident) break;
                const int x = static_cast<int>(passes.now.slice * w.ncols * sizeof(T) / 8);
                const int y = passes.now.image * static_cast<int>(a.hw) + w.first;
                for (int c = 0; c < w.chunks; ++c, ring.next()) {
                    ring.wait_empty();
                    mbar_expect_tx(ring.full + 8 * ring.stage, bytes);
                    box_load(smem_addr(shared) + ring.stage * kChunkBytes, &map_x, x, y + c * a.chunk_rows,
                             ring.full + 8 * ring.stage, passes.second ? done : again);
                }
            }
        }
        if constexpr (CLUSTER) {
            __syncwarp();
            cluster_wait();                           // every arrival has its wait
        }
        return;
    }

    const Segments seg(a.width);
    T *y = static_cast<T *>(a.f.out);
    const int64_t step = static_cast<int64_t>(a.p.rows) * a.channels;
    const int64_t mine0 = (w.first + w.row) * a.channels + w.col * VEC;                 // within an image, slice 0
    // this thread's vectors within a chunk, and its rows of a pass
    const uint4 *mine_in = reinterpret_cast<const uint4 *>(shared) + (w.active ? w.row * a.p.cols + w.col : 0);
    const int round = a.p.rows * a.p.cols;
    const int mine = w.active ? (w.pixels - w.row + a.p.rows - 1) / a.p.rows : 0;
    // one(vector) for each of them
    auto each = [&](bool again, auto one) {
        int left = mine;
        if (again) ring.rewind();
        for (int c = 0; c < w.chunks; ++c, left -= kRounds) {
            ring.wait_full();
            const uint4 *p = mine_in + ring.stage * (kChunkBytes / 16);
            if (left >= kRounds) {
#pragma unroll
                for (int k = 0; k < kRounds; ++k) one(p[k * round]);
            } else {
                for (int k = 0; k < left; ++k) one(p[k * round]);
            }
            if (resident) ring.next();
            else ring.release();
        }
    };

    auto sums = [&](int slice, int64_t image) {
        Col nk, s, q;                                 // minus the first value, sum, sum of squares
#pragma unroll
        for (int i = 0; i < Col::N; ++i) { nk.e[i] = Col::all(0.f); s.e[i] = Col::all(0.f); q.e[i] = Col::all(0.f); }
        if (mine) {
            ring.wait_full();
            float f[VEC];
            unpack<T>(mine_in[ring.stage * (kChunkBytes / 16)], f);
#pragma unroll
            for (int i = 0; i < VEC; ++i) f[i] = -f[i];
            nk.set(f);
        }
        int64_t at = image * a.hw * a.channels + slice * w.ncols + mine0;
        each(false, [&](const uint4 &v) {
            float f[VEC];
            unpack<T>(v, f);
            if constexpr (PACK) {
                const CkptScale sc = ckpt_scale(block_lanes_max<VEC>(max_abs_bits<T>(v)));
                *reinterpret_cast<typename CodeVec<VEC>::type *>(a.f.codes + at) = ckpt_codes(f, sc);
                if ((w.col & (kCkptBlock / VEC - 1)) == 0) a.f.scales[at / kCkptBlock] = static_cast<uint8_t>(sc.e);
                at += step;
            }
            Col c;
            c.set(f);
#pragma unroll
            for (int i = 0; i < Col::N; ++i) {
                const Pair d = vadd(c.e[i], nk.e[i]);
                s.e[i] = vadd(s.e[i], d);
                q.e[i] = vfma(d, d, q.e[i]);
            }
        });
        // block sums
        const float n = static_cast<float>(mine), inv = mine ? 1.0f / n : 0.f;
        float k[VEC], mean[VEC], m2[VEC];             // minus the first value; the mean from there on
        nk.get(k);
        {
            float t[VEC], u[VEC];
            s.get(t), q.get(u);
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                mean[i] = t[i] * inv;
                m2[i] = fmaxf(fmaf(-t[i], mean[i], u[i]), 0.f);
            }
        }
        block_sync();                              // the buffers may still be read by the pass before
        if (w.row == 0) {
            float head[VEC];
#pragma unroll
            for (int i = 0; i < VEC; ++i) head[i] = mean[i] - k[i];
            shared_store<VEC>(cp + w.col * VEC, head);
        }
        block_sync();
        if (w.active) {
            float *to = buf + w.row * 2 * w.ncols + w.col * VEC;
            float head[VEC];
            shared_load<VEC>(cp + w.col * VEC, head);
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float d = mine ? mean[i] - (k[i] + head[i]) : 0.f;       // never rounded at the mean's magnitude
                mean[i] = n * d;
                m2[i] = mine ? fmaf(n * d, d, m2[i]) : 0.f;
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
            if (seg.lane == 0 && g < w.slice_groups) {
                if constexpr (CLUSTER) own[g] = make_float2(mu, u);
                else __stcg(a.partial + (group0 + g) * a.p.members + w.member, make_float2(mu, u));
            }
        }
        if constexpr (CLUSTER) {
            block_sync();
            cluster_wait();
            cluster.send(w, a.p.members, own);
        } else {
            arrive(a, image * a.p.slices + slice);
        }
    };

    auto apply = [&](int slice, int64_t image) {
        if constexpr (CLUSTER) cluster.wait();
        else wait_all(a, image * a.p.slices + slice, ring.patience);
        const int64_t group0 = image * a.groups + slice * w.slice_groups;
        const float hw = static_cast<float>(a.hw), width = static_cast<float>(a.width);
        for (int g = warp; g < w.slice_groups; g += kWarps) {
            // Chan's merge, round by round of up to 160 blocks
            float mu = 0.f, u = 0.f, n = 0.f;
            for (int first = 0; first < a.p.members; first += 32 * kMergeLoads) {
                float2 v[kMergeLoads];
                if constexpr (CLUSTER) load_parts(a, cluster.part + g * a.p.members, lane, v);
                else load_partials(a, a.partial + (group0 + g) * a.p.members, first + lane, v);
                float t = 0.f, px = 0.f;
#pragma unroll
                for (int k = 0; k < kMergeLoads; ++k) {
                    const float c = pixels_or_none(a, first + lane + 32 * k);
                    t = fmaf(c, v[k].x, t);
                    px += c;
                }
                px = warp_sum(px);
                const float m = warp_sum(t) / px;
                float e = 0.f;
#pragma unroll
                for (int k = 0; k < kMergeLoads; ++k) {
                    const float d = v[k].x - m;
                    e += fmaf(pixels_or_none(a, first + lane + 32 * k) * width * d, d, v[k].y);
                }
                e = warp_sum(e);
                const float d = m - mu, f = px / (n + px);
                u += e + d * (d * (n * width * f));     // n is 0 in the first round, and d may be large
                mu = fmaf(d, f, mu);
                n += px;
            }
            if (lane == 0) {
                const float rstd = 1.0f / sqrtf(u / (hw * width) + a.eps);
                stat[g] = make_float2(mu, rstd);
                if (w.member == 0 && a.f.mean) {
                    a.f.mean[group0 + g] = mu;
                    a.f.rstd[group0 + g] = rstd;
                }
            }
        }
        block_sync();
        for (int c = threadIdx.x; c < w.ncols; c += kThreads) {
            const int channel = slice * w.ncols + c;
            const float2 st = stat[group_of[c]];
            const int at = coef_slot<VEC>(c, a.p.cols);
            cp[at] = a.f.gamma[channel] * st.y;
            cq[at] = a.f.beta[channel];
            means[at] = -st.x;
        }
        block_sync();
        const int col = w.active ? w.col * 4 : 0, half = 4 * a.p.cols;
        const Means<T, SPAN> minus_means(means + col, half);
        T *o = y + image * a.hw * a.channels + slice * w.ncols + mine0;
        each(resident, [&](const uint4 &v) {
            uint4 r;
#pragma unroll
            for (int h = 0; h < VEC / 4; ++h) {
                Pair e[2], p[2], q[2], m[2];
                half_column<T>(v, h, e);
                minus_means.get(means + col, half, h, m);
                quad_load(cp + col + h * half, p);
                quad_load(cq + col + h * half, q);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const Pair z = vfma(vadd(e[i], m[i]), p[i], q[i]);
                    e[i] = std::is_same_v<T, __half> && SPAN < kAnyChannel ? act_value_half<ACT>(z) : act_value<ACT>(z);
                }
                half_pack<T>(r, h, e);
            }
            st_stream(o, r);
            o += step;
        });
    };

    while (passes.next(a, w)) {
        if (passes.second) apply(passes.now.slice, passes.now.image);
        else sums(passes.now.slice, passes.now.image);
    }
}

// ---- backward -------------------------------------------------------------------------------------
template <typename T, int ACT, bool CKPT, bool CLUSTER, int SPAN>
__global__ void __launch_bounds__(kBlock, kBlocksPerSm)
cl_team_backward_kernel(const Args a, const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_dy) {
    constexpr int VEC = VecOf<T>::N;
    constexpr int kRoundsGrad = rounds_grad(CKPT), kStagesGrad = stages_grad(CKPT);
    constexpr int kBytes = kRoundsGrad * kThreads * 16;                  // grad_out's part of a chunk
    constexpr int kBytesX = CKPT ? kRoundsGrad * kThreads * VEC : kBytes;
    constexpr int kChunkBytes = kBytes + kBytesX;
    using Col = Column<VEC>;
    using X = std::conditional_t<CKPT, typename CodeVec<VEC>::type, uint4>;
    extern __shared__ __align__(128) unsigned char shared[];
    __shared__ uint64_t bars[2 * kStagesGrad];
    const Place w = place(a);
    float *buf = reinterpret_cast<float *>(shared + kStagesGrad * kChunkBytes);          // [rows][2 ncols]
    float *total = buf + 2 * kThreads * VEC;          // [2 ncols]: this slice's channel sums over the images
    float *cp = total + 2 * w.ncols;                  // [ncols] each: scale and beta; c0 and c1; minus the means
    float *cq = cp + w.ncols;
    float *c0 = cq + w.ncols;
    float *c1 = c0 + w.ncols;
    float *means = c1 + w.ncols;
    float2 *stat = reinterpret_cast<float2 *>(means + w.ncols);                         // [groups]: (s1, s2)
    int *group_of = reinterpret_cast<int *>(stat + w.ncols);                             // [ncols], within a slice
    float2 *own = reinterpret_cast<float2 *>(group_of + w.ncols);                        // cluster: [groups], then
    ClusterExchange cluster;                                                             // [groups][members]
    __shared__ uint64_t cluster_bar;
    // a team's only item that fits the ring is read once
    const bool resident = a.p.resident != 0;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    Passes passes(w);
    Ring<kStagesGrad> ring;
    ring.init(bars);
    if constexpr (CLUSTER) cluster.init(&cluster_bar, own + w.slice_groups, a.p.members);
    for (int c = threadIdx.x; c < w.ncols; c += kBlock) group_of[c] = c / a.width;
    __syncthreads();
    if constexpr (CLUSTER) cluster_arrive();          // the barriers are set up; waited for before the first store to a peer

    if (warp == kWarps) {                             // producer
        if (lane == 0) {
            stagger(a, w.team, ring.patience);
            const uint64_t done = policy_evict_first(), again = resident ? done : policy_evict_last();
            constexpr int kSizeX = CKPT ? 1 : sizeof(T);
            const uint32_t bytes = static_cast<uint32_t>(a.chunk_rows * w.ncols) * (sizeof(T) + kSizeX);
            while (passes.next(a, w)) {
                if (passes.second && resident) break;
                const int x = static_cast<int>(passes.now.slice * w.ncols * sizeof(T) / 8);
                const int xx = passes.now.slice * w.ncols * kSizeX / 8;
                const int y = passes.now.image * static_cast<int>(a.hw) + w.first;
                const uint64_t policy = passes.second ? done : again;
                for (int c = 0; c < w.chunks; ++c, ring.next()) {
                    ring.wait_empty();
                    const uint32_t bar = ring.full + 8 * ring.stage, to = smem_addr(shared) + ring.stage * kChunkBytes;
                    mbar_expect_tx(bar, bytes);
                    box_load(to, &map_dy, x, y + c * a.chunk_rows, bar, policy);
                    box_load(to + kBytes, &map_x, xx, y + c * a.chunk_rows, bar, policy);
                }
            }
        }
        if constexpr (CLUSTER) {
            __syncwarp();
            cluster_wait();                           // every arrival has its wait
        }
        return;
    }

    const Segments seg(a.width);
    const int64_t blocks_row = ckpt_blocks(a.channels), scale_step = a.p.rows * blocks_row;
    T *dx = static_cast<T *>(a.b.grad_in);
    const Pair one = Col::all(1.0f);
    const int64_t step = static_cast<int64_t>(a.p.rows) * a.channels;
    const int64_t mine0 = (w.first + w.row) * a.channels + w.col * VEC;
    // this thread's vectors within a chunk, and its rows of a pass
    const int place_in = w.active ? w.row * a.p.cols + w.col : 0;
    const int round = a.p.rows * a.p.cols;
    const int mine = w.active ? (w.pixels - w.row + a.p.rows - 1) / a.p.rows : 0;
    // The scale bytes of a checkpoint (less than 16 bytes a row) are loaded into registers one chunk ahead.
    const uint8_t *scale_at = nullptr;
    uint8_t scale[kRoundsGrad] = {};
    auto load_scales = [&](int left) {
        if constexpr (CKPT) {
#pragma unroll
            for (int k = 0; k < kRoundsGrad; ++k)
                if (k < left) scale[k] = scale_at[k * scale_step];
            scale_at += kRoundsGrad * scale_step;
        }
    };
    auto first_scales = [&](int slice, int64_t image) {
        if constexpr (CKPT) {
            scale_at = a.b.scales + (image * a.hw + w.first + w.row) * blocks_row +
                       (slice * w.ncols + w.col * VEC) / kCkptBlock;
            load_scales(mine);
        }
    };
    const int col = w.active ? w.col * 4 : 0, half = 4 * a.p.cols;                      // this column's coefficients
    // use(h, coefficients, x - mean, grad_out, vector) for both halves of each of this thread's vectors, then
    // done(vector).  The coefficients are read from shared memory where they are used: held in
    // registers they would take a third of the warps away.
    auto each = [&](bool again, auto coefficient, auto use, auto done) {
        int left = mine;
        const Means<T, SPAN> minus_means(means + col, half);
        if (again) ring.rewind();
        for (int c = 0; c < w.chunks; ++c, left -= kRoundsGrad) {
            ring.wait_full();
            const unsigned char *p = shared + ring.stage * kChunkBytes;
            uint8_t e[kRoundsGrad];
#pragma unroll
            for (int k = 0; k < kRoundsGrad; ++k) e[k] = scale[k];
            load_scales(left - kRoundsGrad);
            auto vector = [&](int k, uint8_t ek) {
                uint4 d = reinterpret_cast<const uint4 *>(p)[place_in + k * round];
                const X v = reinterpret_cast<const X *>(p + kBytes)[place_in + k * round];
#pragma unroll
                for (int h = 0; h < VEC / 4; ++h) {
                    const auto coef = coefficient(h);
                    Pair xm[2], g[2], m[2];
                    half_column<T>(d, h, g);
                    minus_means.get(means + col, half, h, m);
                    if constexpr (CKPT) {
                        half_codes(v, h, xm);
                        const Pair st = Col::all(ckpt_step(ek));
#pragma unroll
                        for (int i = 0; i < 2; ++i) xm[i] = vfma(xm[i], st, m[i]);
                    } else {
                        half_column<T>(v, h, xm);
#pragma unroll
                        for (int i = 0; i < 2; ++i) xm[i] = vadd(xm[i], m[i]);
                    }
                    use(h, coef, xm, g, d);
                }
                done(d);
            };
            if (left >= kRoundsGrad) {
#pragma unroll
                for (int k = 0; k < kRoundsGrad; ++k) vector(k, e[k]);
            } else {
#pragma unroll
                for (int k = 0; k < kRoundsGrad; ++k)
                    if (k < left) vector(k, e[k]);
            }
            if (resident) ring.next();
            else ring.release();
        }
    };
    struct Coef { Pair p[2], q[2], k0[2], k1[2]; };

    // z = (x - mean) p + beta as in the forward pass
    auto coefficients = [&](int slice, int64_t image, bool second) {
        block_sync();                              // the arrays may still be read by the pass before
        for (int c = threadIdx.x; c < w.ncols; c += kThreads) {
            const int channel = slice * w.ncols + c;
            const int64_t group0 = image * a.groups + slice * w.slice_groups;
            const int64_t st = group0 + group_of[c];
            const float rs = a.b.rstd[st];
            const int at = coef_slot<VEC>(c, a.p.cols);
            cp[at] = a.b.gamma[channel] * rs;
            cq[at] = a.b.beta[channel];
            means[at] = -a.b.mean[st];
            if (second) {
                const float2 s = stat[group_of[c]];
                c1[at] = -rs * rs * s.y;
                c0[at] = -rs * s.x;
            }
        }
        block_sync();
    };

    auto sums = [&](int slice, int64_t image) {
        first_scales(slice, image);
        coefficients(slice, image, false);
        Col s0, s1;
#pragma unroll
        for (int i = 0; i < Col::N; ++i) { s0.e[i] = Col::all(0.f); s1.e[i] = Col::all(0.f); }
        each(false,
             [&](int h) {
                 Coef c;
                 quad_load(cp + col + h * half, c.p);
                 quad_load(cq + col + h * half, c.q);
                 return c;
             },
             [&](int h, const Coef &c, const Pair (&xm)[2], const Pair (&g)[2], uint4 &) {
#pragma unroll
                 for (int i = 0; i < 2; ++i) {
                     const Pair dz = act_grad<ACT>(g[i], vfma(xm[i], c.p[i], c.q[i]), one);
                     s0.e[2 * h + i] = vadd(s0.e[2 * h + i], dz);
                     s1.e[2 * h + i] = vfma(dz, xm[i], s1.e[2 * h + i]);
                 }
             },
             [](const uint4 &) {});
        if (w.active) {
            float *to = buf + w.row * 2 * w.ncols + w.col * VEC;
            column_store<VEC>(to, s0);
            column_store<VEC>(to + w.ncols, s1);
        }
        sum_rows(buf, a.p.rows, 2 * w.ncols);
        const int64_t group0 = image * a.groups + slice * w.slice_groups;
        for (int c = threadIdx.x; c < w.ncols; c += kThreads) {
            const float t = buf[w.ncols + c] * a.b.rstd[group0 + group_of[c]];          // sum of dz xhat
            buf[w.ncols + c] = t;
            total[c] += buf[c];
            total[w.ncols + c] += t;
        }
        block_sync();
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
            if (seg.lane == 0 && g < w.slice_groups) {
                if constexpr (CLUSTER) own[g] = make_float2(t1, t2);
                else __stcg(a.partial + (group0 + g) * a.p.members + w.member, make_float2(t1, t2));
            }
        }
        if constexpr (CLUSTER) {
            block_sync();
            cluster_wait();
            cluster.send(w, a.p.members, own);
        } else {
            arrive(a, image * a.p.slices + slice);
        }
    };

    auto apply = [&](int slice, int64_t image) {
        first_scales(slice, image);
        if constexpr (CLUSTER) cluster.wait();
        else wait_all(a, image * a.p.slices + slice, ring.patience);
        const int64_t group0 = image * a.groups + slice * w.slice_groups;
        const float inv = 1.0f / (static_cast<float>(a.hw) * static_cast<float>(a.width));
        for (int g = warp; g < w.slice_groups; g += kWarps) {
            float t1 = 0.f, t2 = 0.f;
            for (int first = 0; first < a.p.members; first += 32 * kMergeLoads) {
                float2 v[kMergeLoads];
                if constexpr (CLUSTER) load_parts(a, cluster.part + g * a.p.members, lane, v);
                else load_partials(a, a.partial + (group0 + g) * a.p.members, first + lane, v);
#pragma unroll
                for (int k = 0; k < kMergeLoads; ++k) {
                    t1 += v[k].x;
                    t2 += v[k].y;
                }
            }
            t1 = warp_sum(t1);
            t2 = warp_sum(t2);
            if (lane == 0) stat[g] = make_float2(t1 * inv, t2 * inv);
        }
        coefficients(slice, image, true);
        T *o = dx + image * a.hw * a.channels + slice * w.ncols + mine0;
        each(resident,
             [&](int h) {
                 Coef c;
                 quad_load(cp + col + h * half, c.p);
                 quad_load(cq + col + h * half, c.q);
                 quad_load(c0 + col + h * half, c.k0);
                 quad_load(c1 + col + h * half, c.k1);
                 return c;
             },
             [&](int h, const Coef &c, const Pair (&xm)[2], const Pair (&g)[2], uint4 &r) {
                 Pair e[2];
#pragma unroll
                 for (int i = 0; i < 2; ++i) {
                     const Pair dz = act_grad<ACT>(g[i], vfma(xm[i], c.p[i], c.q[i]), one);
                     e[i] = vfma(dz, c.p[i], vfma(xm[i], c.k1[i], c.k0[i]));
                 }
                 half_pack<T>(r, h, e);               // over the half of grad_out that has just been used
             },
             [&](const uint4 &r) {
                 st_stream(o, r);
                 o += step;
             });
    };

    int summed = -1;                                  // the slice that `total` belongs to
    while (passes.next(a, w)) {
        const int slice = passes.now.slice;
        if (passes.second) {
            apply(slice, passes.now.image);
            continue;
        }
        if (slice != summed) {
            block_sync();
            for (int c = threadIdx.x; c < 2 * w.ncols; c += kThreads) total[c] = 0.f;
            summed = slice;
        }
        sums(slice, passes.now.image);
        if (passes.now.image + a.p.image_teams >= static_cast<int>(a.batch)) {                             // the slice's last image
            block_sync();
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

// (A memset node in front costs 3.5 us of a captured graph's time, a kernel less than 1.)
__global__ void __launch_bounds__(256) cl_clear_kernel(unsigned int *p, long long n) {
    for (long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; i < n; i += static_cast<long long>(gridDim.x) * 256)
        p[i] = 0;
}

// ---- plan and launch ------------------------------------------------------------------------------
struct Layout {
    size_t partial, channel_sums, bytes;              // behind the items' counters
};

Layout layout(const GnClShape &s, const GnClTeamPlan &p, bool backward) {
    const auto up = [](size_t n) { return (n + 15) & ~static_cast<size_t>(15); };
    Layout l;
    l.partial = p.cluster ? 0 : up((static_cast<size_t>(s.batch) * p.slices + kSlotWords) * sizeof(unsigned int));
    l.channel_sums =
        l.partial + (p.cluster ? 0 : up(static_cast<size_t>(s.batch) * s.groups * p.members * sizeof(float2)));
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
    a.chunk_rows = p.rows * p.rounds;
    const int64_t chunks = (s.hw + a.chunk_rows - 1) / a.chunk_rows;
    a.share = static_cast<int>(chunks / p.members);
    a.rest = static_cast<int>(chunks % p.members);
    a.eps = s.eps;
    a.arrived = reinterpret_cast<unsigned int *>(base);
    a.items = s.batch * p.slices;
    a.partial = reinterpret_cast<float2 *>(base + l.partial);
    a.channel_sums = reinterpret_cast<float2 *>(base + l.channel_sums);
    return a;
}

size_t shared_bytes(const GnClTeamPlan &p, bool backward, bool ckpt) {
    const size_t ncols = static_cast<size_t>(p.cols) * p.vec;
    const size_t vector = !backward ? 16 : ckpt ? 16 + p.vec : 32;
    const size_t bytes = static_cast<size_t>(backward ? stages_grad(ckpt) * rounds_grad(ckpt) : kStages * kRounds) * kThreads * vector +
           (2 * static_cast<size_t>(kThreads) * p.vec + (backward ? 10 : 6) * ncols) * sizeof(float) +
           (p.cluster ? static_cast<size_t>(p.slice_groups) * (1 + p.members) * sizeof(float2) : 0);
    return p.stagger ? std::max(bytes, kTwoOnSm) : bytes;
}

using EncodeFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                              const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// The driver's encoder, looked up once (the library does not link the driver).
EncodeFn encoder() {
    static const EncodeFn fn = [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<EncodeFn>(p);
    }();
    return fn;
}

// [rows, row_bytes] in 8-byte units; boxes of box_bytes by box_rows.  row_bytes and box_bytes are multiples
// of 16, base 16-byte aligned.
cudaError_t make_map(CUtensorMap *map, const void *base, int64_t rows, int64_t row_bytes, int box_bytes, int box_rows) {
    const EncodeFn fn = encoder();
    if (!fn) return cudaErrorNotSupported;
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(row_bytes / 8), static_cast<cuuint64_t>(rows)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(row_bytes)};
    const cuuint32_t box[2] = {static_cast<cuuint32_t>(box_bytes / 8), static_cast<cuuint32_t>(box_rows)};
    const cuuint32_t steps[2] = {1, 1};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT64, 2, const_cast<void *>(base), dims, strides, box, steps,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

// Blocks of a kernel that an SM holds; asked once per thread and change of size.
template <auto kernel> cudaError_t blocks_of_sm(int dev, size_t smem, int *blocks) {
    struct Known { int dev = -1, blocks = 0; size_t smem = 0; };
    thread_local Known known;
    if (known.dev != dev || known.smem != smem) {
        known.dev = -1;
        const cudaError_t err = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&known.blocks, kernel, kBlock, smem);
        if (err != cudaSuccess) return err;
        known.dev = dev;
        known.smem = smem;
    }
    *blocks = known.blocks;
    return cudaSuccess;
}

// A team is a cluster, or else the launch is cooperative: the blocks of a team wait for one another, so
// either all of them run or none.  A grid that the device does not hold at once is not launched at all
// (cudaErrorCooperativeLaunchTooLarge): the caller has a form without teams.
template <auto kernel, typename... Maps>
cudaError_t launch(const Args &a, size_t smem, cudaStream_t stream, const Maps &...maps) {
    cudaError_t err;
    const bool counted = !a.p.cluster && a.p.members > 1;
    const int grid = a.p.slice_teams * a.p.image_teams * a.p.members;
    // once per kernel and device, to what any of its plans may ask for
    static std::atomic<bool> prepared[kMaxDevices];
    int dev = 0;
    err = cudaGetDevice(&dev);
    if (err != cudaSuccess) return err;
    if (dev >= kMaxDevices || !prepared[dev].load(std::memory_order_relaxed)) {
        err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxShared);
        if (err != cudaSuccess) return err;
        if (dev < kMaxDevices) prepared[dev].store(true, std::memory_order_relaxed);
    }
    if (smem > kMaxShared) return cudaErrorInvalidConfiguration;
    if (counted) {
        int blocks = 0;
        err = blocks_of_sm<kernel>(dev, smem, &blocks);
        if (err != cudaSuccess) return err;
        if (grid > static_cast<int64_t>(blocks) * sm_count() || (a.p.stagger && blocks != kMaxTeamsOfSm))
            return cudaErrorCooperativeLaunchTooLarge;
        const long long words = a.items + (a.p.stagger ? kSlotWords : 0);
        cl_clear_kernel<<<static_cast<unsigned>(std::min<long long>((words + 255) / 256, 256)), 256, 0, stream>>>(a.arrived, words);
        err = cudaGetLastError();
        if (err != cudaSuccess) return err;
        g_launches.fetch_add(1);
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(grid));
    cfg.blockDim = dim3(kBlock);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    if (!counted) {
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = static_cast<unsigned>(a.p.members);
        attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = 1;
    } else {
        attr[0].id = cudaLaunchAttributeCooperative;
        attr[0].val.cooperative = 1;
    }
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    err = cudaLaunchKernelEx(&cfg, kernel, a, maps...);
    if (err == cudaSuccess) g_launches.fetch_add(1);
    return err;
}

template <typename T, bool CLUSTER, int SPAN> cudaError_t forward_run(const GnClShape &s, Args &a, cudaStream_t stream) {
    CUtensorMap x;
    const cudaError_t err = make_map(&x, a.f.in, s.batch * s.hw, s.channels * sizeof(T), a.p.cols * 16, a.chunk_rows);
    if (err != cudaSuccess) return err;
    const size_t smem = shared_bytes(a.p, false, false);
    if (s.act == kActSilu)
        return a.f.codes ? launch<cl_team_forward_kernel<T, kActSilu, true, CLUSTER, SPAN>>(a, smem, stream, x)
                         : launch<cl_team_forward_kernel<T, kActSilu, false, CLUSTER, SPAN>>(a, smem, stream, x);
    return a.f.codes ? launch<cl_team_forward_kernel<T, kActNone, true, CLUSTER, SPAN>>(a, smem, stream, x)
                     : launch<cl_team_forward_kernel<T, kActNone, false, CLUSTER, SPAN>>(a, smem, stream, x);
}

template <typename T, bool CLUSTER, int SPAN> cudaError_t backward_run(const GnClShape &s, Args &a, cudaStream_t stream) {
    const int64_t rows = s.batch * s.hw, row_bytes = s.channels * sizeof(T);
    CUtensorMap x, dy;
    cudaError_t err = make_map(&dy, a.b.grad_out, rows, row_bytes, a.p.cols * 16, a.chunk_rows);
    if (err == cudaSuccess)
        err = a.b.codes ? make_map(&x, a.b.codes, rows, s.channels, a.p.cols * a.p.vec, a.chunk_rows)
                        : make_map(&x, a.b.in, rows, row_bytes, a.p.cols * 16, a.chunk_rows);
    if (err != cudaSuccess) return err;
    const size_t smem = shared_bytes(a.p, true, a.b.codes != nullptr);
    if (s.act == kActSilu)
        return a.b.codes ? launch<cl_team_backward_kernel<T, kActSilu, true, CLUSTER, SPAN>>(a, smem, stream, x, dy)
                         : launch<cl_team_backward_kernel<T, kActSilu, false, CLUSTER, SPAN>>(a, smem, stream, x, dy);
    return a.b.codes ? launch<cl_team_backward_kernel<T, kActNone, true, CLUSTER, SPAN>>(a, smem, stream, x, dy)
                     : launch<cl_team_backward_kernel<T, kActNone, false, CLUSTER, SPAN>>(a, smem, stream, x, dy);
}

// The most special form for the width of a group; only the fp16 forward pass gains from whole pairs.
template <typename T, bool CLUSTER> cudaError_t forward_type(const GnClShape &s, Args &a, cudaStream_t stream) {
    if (a.width % 4 == 0) return forward_run<T, CLUSTER, kHalvesWhole>(s, a, stream);
    if constexpr (std::is_same_v<T, __half>)
        if (a.width % 2 == 0) return forward_run<T, CLUSTER, kPairsWhole>(s, a, stream);
    return forward_run<T, CLUSTER, kAnyChannel>(s, a, stream);
}

template <typename T, bool CLUSTER> cudaError_t backward_type(const GnClShape &s, Args &a, cudaStream_t stream) {
    if (a.width % 4 == 0) return backward_run<T, CLUSTER, kHalvesWhole>(s, a, stream);
    return backward_run<T, CLUSTER, kAnyChannel>(s, a, stream);
}

}  // namespace

bool gn_cl_team_plan(const GnClShape &s, bool pack, bool backward, bool ckpt, GnClTeamPlan *p) {
    const int64_t width = s.channels / s.groups;
    const int64_t esize = s.dtype == kF32 ? 4 : 2;
    p->vec = static_cast<int>(16 / esize);
    if (s.channels % p->vec != 0 || (pack && s.channels % kCkptBlock != 0)) return false;
    if (s.batch * s.hw >= (1ll << 31)) return false;                                  // box coordinates
    // the narrowest slice, in columns: whole groups, whole vectors, and of a checkpoint whole blocks
    // (written) or 16 bytes of codes (read)
    int64_t grain = std::lcm(width, static_cast<int64_t>(p->vec));
    if (pack) grain = std::lcm(grain, static_cast<int64_t>(kCkptBlock));
    if (ckpt) grain = std::lcm(grain, static_cast<int64_t>(16));
    if (grain > s.channels || s.channels % grain != 0) return false;
    const int64_t grains = s.channels / grain;
    grain /= p->vec;
    if (grain > kMaxCols) return false;
    const int64_t grain_bytes = grain * p->vec * esize;
    const int64_t want = (128 + grain_bytes - 1) / grain_bytes;                       // grains per slice
    p->rounds = backward ? rounds_grad(ckpt) : kRounds;
    const int stages = backward ? stages_grad(ckpt) : kStages;
    const auto allowed = [&](int64_t d) { return grains % d == 0 && grains / d * grain <= kMaxCols; };
    const auto set_slices = [&](int64_t d) {
        p->slices = static_cast<int>(d);
        p->cols = static_cast<int>(grains / d * grain);
        p->rows = std::min(kThreads / p->cols, 256 / p->rounds);                       // a box has at most 256 rows
        p->slice_groups = static_cast<int>(p->cols * p->vec / width);
        return (s.hw + p->rows * p->rounds - 1) / (p->rows * p->rounds);               // chunks of an item
    };
    p->stagger = p->resident = p->cluster = 0;
    const int64_t sms = sm_count();

    // Small tensors: one item per cluster, read once, no workspace.  Of the slices and cluster sizes that do with
    // one wave of blocks the one with the most blocks, and of those the widest rows.
    int64_t best = 0, best_slices = 0, best_members = 0;
    for (int64_t limit = kMaxCluster / 2; limit <= kMaxCluster && best == 0; limit *= 2)
        for (int64_t d = 1; d <= grains; ++d) {
            if (!allowed(d) || (d > 1 && grains / d * grain_bytes < 64)) continue;
            const int64_t n = set_slices(d);
            for (int64_t m = 1; m <= limit; m *= 2) {
                const int64_t blocks = s.batch * d * m;
                if (blocks > sms * kBlocksPerSm || m > n || (n + m - 1) / m > stages || blocks <= best ||
                    static_cast<int64_t>(p->slice_groups) * (m + 1) * 8 > kClusterPartBytes)
                    continue;
                best = blocks, best_slices = d, best_members = m;
            }
        }
    if (best > 0) {
        set_slices(best_slices);
        p->cluster = p->resident = 1;
        p->slice_teams = static_cast<int>(best_slices);
        p->image_teams = static_cast<int>(s.batch);
        p->members = static_cast<int>(best_members);
        return true;
    }

    // slices: as many as leave rows of 128 bytes, but few enough that all images that fit L2 have their teams
    const int64_t per_element = backward ? (ckpt ? 1 : esize) + esize : esize;
    const int64_t image = s.hw * s.channels * per_element;
    const int64_t in_flight = backward ? 2 * kInFlight : kInFlight;
    const int64_t images = std::min(s.batch, std::max<int64_t>(1, in_flight / image));
    int64_t slices = 0;
    for (int64_t d = 1; d <= grains; ++d)
        if (allowed(d) && (slices == 0 || (grains / d >= want && d * images <= sms * kBlocksPerSm))) slices = d;
    if (slices == 0) return false;
    const int64_t chunks = set_slices(slices);
    // what an SM holds at once
    const int64_t fit = kSmShared / (static_cast<int64_t>(shared_bytes(*p, backward, ckpt)) + kBlockShared);
    const int64_t blocks = sms * std::min<int64_t>(fit, kBlocksPerSm);
    p->slice_teams = static_cast<int>(std::min(slices, std::max<int64_t>(1, in_flight * slices / image)));
    while (slices % p->slice_teams != 0) --p->slice_teams;
    int64_t n = std::min(images, std::max<int64_t>(1, blocks / p->slice_teams));
    n = (s.batch + (s.batch + n - 1) / n - 1) / ((s.batch + n - 1) / n);               // even rounds
    p->image_teams = static_cast<int>(n);
    p->members = static_cast<int>(std::min(std::max<int64_t>(1, blocks / (p->slice_teams * n)), chunks));
    p->resident = slices == p->slice_teams && s.batch == n && (chunks + p->members - 1) / p->members <= stages;
    p->stagger = !p->resident && p->slice_teams * n == kMaxTeamsOfSm && p->members == sms && fit >= kBlocksPerSm;
    return true;
}

size_t gn_cl_team_shared_bytes(const GnClTeamPlan &p, bool backward, bool ckpt) { return shared_bytes(p, backward, ckpt); }

size_t gn_cl_team_workspace_bytes(const GnClShape &s, const GnClTeamPlan &p, bool backward) {
    return layout(s, p, backward).bytes;
}

cudaError_t gn_cl_team_forward(const GnClShape &s, const GnClTeamPlan &p, const GnClForward &f, void *ws, cudaStream_t stream) {
    Args a = make_args(s, p, false, ws);
    a.f = f;
    switch (s.dtype) {
        case kF16: return p.cluster ? forward_type<__half, true>(s, a, stream) : forward_type<__half, false>(s, a, stream);
        case kBF16: return p.cluster ? forward_type<__nv_bfloat16, true>(s, a, stream) : forward_type<__nv_bfloat16, false>(s, a, stream);
        default: return p.cluster ? forward_type<float, true>(s, a, stream) : forward_type<float, false>(s, a, stream);
    }
}

cudaError_t gn_cl_team_backward(const GnClShape &s, const GnClTeamPlan &p, const GnClBackward &b, void *ws,
                                cudaStream_t stream) {
    Args a = make_args(s, p, true, ws);
    a.b = b;
    cudaError_t err;
    switch (s.dtype) {
        case kF16: err = p.cluster ? backward_type<__half, true>(s, a, stream) : backward_type<__half, false>(s, a, stream); break;
        case kBF16: err = p.cluster ? backward_type<__nv_bfloat16, true>(s, a, stream) : backward_type<__nv_bfloat16, false>(s, a, stream); break;
        default: err = p.cluster ? backward_type<float, true>(s, a, stream) : backward_type<float, false>(s, a, stream); break;
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
