// tcgen05 kernel for the gradients of segment_mm in bfloat16, float32 sums:
//
//   da[i] = grad[i] @ b[r]^T                  (K = d2: both operands K-major)
//   db[r] = a[rows of r]^T @ grad[rows of r]  (K = rows: both M/N-major)
//
// Every operand is read as it lies in memory, 64 rows x 64 columns a TMA box;
// a box serves as K-major rows or as M/N-major columns, so the two products
// differ only in coordinates and descriptors, and no transposed copy is made.
// Two CTAs of a cluster work on one 512 x 256 tile at a time (cta_group::2): each
// holds 256 of its rows, as two 128 x 256 float32 accumulators that fill the tensor
// memory, and half of the other operand, which the tensor cores of both read.  Each
// K slice of 64 brings 32 KB + 16 KB to a CTA for 2 x 4 MMAs of 256 x 256 x 16, where
// a 256 x 256 tile of its own takes 64 KB: three quarters of the traffic from L2, and
// four slices in the ring instead of three.  32768 x 2048 x 1024 over 16 segments: 285
// us with a tile a CTA, 278 so; 500000 x 256 x 256 over 64: 228 and 222 (now 270 and
// 204).  The wide one waits for tiles for 23 % of the time and runs into the power
// limit; the narrow one is bound by memory (984 MB in 166 us in the kernel).  Taking
// da's tiles along with db's sums, 256 rows at a time, so that grad would be read from
// DRAM once, took 202 us in the kernel: the loads under way are then half L2's.
//
// One persistent launch holds both products.  Warp 10 of a pair's first CTA takes
// the next item (an atomic counter; which pair does what does not change any
// result) and publishes it to both through a four-deep queue; warp 0 of each issues
// its loads into a four-slice ring, reporting to the first CTA's barriers; warp 1 of
// the first issues the MMAs; warps 2-9 write finished tiles out (through a swizzled
// staging box and TMA stores).  What a role on the critical path tells the other CTA
// goes without a release across the cluster, which takes some 1000 cycles: where a
// thread of the second CTA passed on that its slices were there, wide took 312 us.
//
// A db slice's rows beyond the segment belong to the next one: the MMA warp
// writes zeros over those that share a 16-row MMA step with the segment's last
// rows (in both operands, so that inf and NaN of a neighbour do not get in) and
// leaves out the steps behind.  Pieces of a cut db tile go to float32 partial
// tiles, which k_grad_finish adds in order: the same bits on every run.
//
// Every mbarrier wait is bounded, with the abort protocol of grouped_mm_tc.cu.
#include "after.cuh"
#include "grouped_mm.cuh"
#include "tcgen05.cuh"

namespace bgl {
namespace {

constexpr int kStages = 4;
constexpr int kBox = kGradSlice * 128;        // 64 rows x 64 columns of bf16
constexpr int kStageBytes = 6 * kBox;         // 4 boxes of M, 2 of N
constexpr int kEpiWarps = 8;                  // two a TMEM lane quarter, 128 columns each
constexpr int kQueue = 4;
constexpr int kWarpLoad = 0, kWarpMma = 1, kWarpEpi0 = 2, kWarpNext = kWarpEpi0 + kEpiWarps;
constexpr int kThreads = 32 * (kWarpNext + 1);
constexpr int kPartial = kGradRows * kGradCols;  // values of a partial tile

struct GradArgs {
    const int64_t *off, *row_off, *item_off, *cut_off, *slot_off;
    const int32_t *order;
    int64_t *head;
    float *partial;
    __nv_bfloat16 *da, *db;
    int64_t r, n;
    int32_t cols, tiles1, tiles2, d1, d2;
    bool whole;  // no k_grad_finish follows: no sum is cut
};

// One item.  da: rows [row0, row0 + rows) of segment seg, columns from j0 on.
// db: the sum over those rows for the tile at (i0, j0) of the segment's block;
// `slot` is the partial tile it goes to, -1 where it is the whole sum.
struct Item {
    int32_t kind;  // 0: none left, 1: da, 2: db
    int32_t seg, row0, rows, i0, j0, slot;
};
constexpr int kDa = 1, kDb = 2;
constexpr size_t kSmem = 1024 + kStages * (size_t)kStageBytes + kEpiWarps * 4096 +
                         8 * (4 * kStages + 2 * kQueue + 5) + kQueue * sizeof(Item) + 16;

// Last i in [0, n) with first[i] <= at, by the whole warp (33 ways a step).
__device__ __forceinline__ int64_t warp_search(const int64_t *first, int64_t n, int64_t at) {
    const int lane = threadIdx.x & 31;
    int64_t lo = 0, hi = n;  // first[lo] <= at < first[hi]
    while (hi - lo > 1) {
        const int64_t step = (hi - lo + 32) / 33, i = lo + (lane + 1) * step;
        const unsigned below = __ballot_sync(0xffffffffu, i < hi && first[i < hi ? i : lo] <= at);
        const int64_t base = lo + (int64_t)__popc(below) * step;
        if (base + step < hi) hi = base + step;
        lo = base;
    }
    return lo;
}

// Item number `at`, on every lane of the warp.
__device__ __forceinline__ Item item_at(const GradArgs &p, int64_t at) {
    Item q = {};
    const int64_t db_items = p.head[kHeadDbItems];
    if (at >= p.head[kHeadItems]) return q;
    if (at < db_items) {
        const int64_t k = warp_search(p.item_off, p.r, at);
        q.kind = kDb;
        q.seg = p.order[k];
        const int64_t first = p.off[q.seg], len = p.off[q.seg + 1] - first;
        const GradPieces cut = grad_pieces(len, p.head[kHeadPiece]);
        const int64_t in = at - p.item_off[k], per = (int64_t)p.tiles1 * p.tiles2;
        // the tiles of one piece are neighbours: they read the same rows
        const int64_t piece = in / per, tile = in % per;
        q.i0 = (int32_t)(tile / p.tiles2) * kGradRows;
        q.j0 = (int32_t)(tile % p.tiles2) * kGradCols;
        const int64_t skip = piece * cut.slices * kGradSlice, most = cut.slices * kGradSlice;
        q.row0 = (int32_t)(first + skip);
        q.rows = (int32_t)(len - skip < most ? len - skip : most);
        q.slot = cut.count > 1 ? (int32_t)(p.slot_off[k] + tile * cut.count + piece) : -1;
    } else {
        const int64_t in = at - db_items, tile = in / p.cols;
        q.kind = kDa;
        q.seg = (int32_t)warp_search(p.row_off, p.r, tile);
        const int64_t first = p.off[q.seg] + (tile - p.row_off[q.seg]) * kGradRows;
        const int64_t left = p.off[q.seg + 1] - first;
        q.row0 = (int32_t)first;
        q.rows = (int32_t)(left < kGradRows ? left : kGradRows);
        q.j0 = (int32_t)(in % p.cols) * kGradCols;
        q.slot = -1;
    }
    return q;
}

// SWIZZLE_128B descriptor of an M- or N-major operand: 64-element runs of 128
// bytes, one a row of K; 8-row groups 1024 bytes apart (SBO), the next 64
// elements of M or N one box further on (LBO).
__device__ __forceinline__ uint64_t mn_desc(uint32_t addr) {
    return (uint64_t)((addr >> 4) & 0x3FFF) | ((uint64_t)(kBox >> 4) << 16) |
           ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

// Instruction descriptors: fp32 accumulator, bf16 operands, M = 256 over the pair,
// both operands K-major or both M/N-major.
__device__ __forceinline__ uint32_t k_instr(int n) {
    return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(256 >> 4) << 24);
}
__device__ __forceinline__ uint32_t mn_instr(int n) {
    return k_instr(n) | (1u << 15) | (1u << 16);
}

__device__ __forceinline__ void mma2(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                     uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate));
}
// Arrives on this barrier of both CTAs once the MMAs issued so far are done.
__device__ __forceinline__ void mma2_commit(uint64_t *bar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            smem_u32(bar)),
        "h"((uint16_t)3)
        : "memory");
}
// The barriers that the issuing thread uses.
struct Bars {
    uint64_t *full, *empty, *acc_full, *acc_empty;
};

// The address of a shared variable in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t in_cta(const void *p, uint32_t rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
    return r;
}
__device__ __forceinline__ void arrive_in(uint64_t *bar, uint32_t rank) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(in_cta(bar, rank)) : "memory");
}
// The same without ordering this thread's writes (a release across the cluster takes
// some 1000 cycles): for tensor memory that has been read.
__device__ __forceinline__ void signal_in(uint64_t *bar, uint32_t rank) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(in_cta(bar, rank)) : "memory");
}
// A TMA load into this CTA that reports to a barrier of either CTA of the pair.
__device__ __forceinline__ void pair_load(uint32_t dst, const CUtensorMap *map, uint32_t bar, int32_t c0, int32_t c1) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2"
        " [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1)
        : "memory");
}
__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// A waiting thread may sleep that long at a time (it wakes up when the phase is over):
// polling took a quarter of the issue slots, and power (276 -> 270 us where the power
// limit holds, 209 -> 204 for the narrow case).
constexpr uint32_t kSleepNs = 20000;

// The bounded wait for what the other CTA of the pair may have written or arrived on.
__device__ __forceinline__ bool pair_try_wait(uint64_t *bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.b32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity), "r"(kSleepNs)
        : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool pair_wait(uint64_t *bar, uint32_t parity, int code, volatile int *abort) {
    if (pair_try_wait(bar, parity)) return true;
    const unsigned long long t0 = now_ns();
    while (!pair_try_wait(bar, parity)) {
        if (abort && *abort) return false;
        if (now_ns() - t0 > kTimeoutNs) {
            atomicCAS(&g_tc_error, 0, code);
            if (abort) *abort = 1;
            return false;
        }
    }
    return true;
}

// Lane 0 waits for the whole warp.
__device__ __forceinline__ bool warp_wait(uint64_t *bar, uint32_t parity, int code,
                                          volatile int *abort) {
    int ok = 0;
    if ((threadIdx.x & 31) == 0) ok = pair_wait(bar, parity, code, abort);
    ok = __shfl_sync(0xffffffffu, ok, 0);
    __syncwarp();
    return ok != 0;
}

__device__ __forceinline__ void tma_store_3d(const CUtensorMap *map, const void *src, int32_t c0,
                                             int32_t c1, int32_t c2) {
    asm volatile(
        "cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(
            reinterpret_cast<uint64_t>(map)),
        "r"(c0), "r"(c1), "r"(c2), "r"(smem_u32(src))
        : "memory");
}

// Waits for `slices` whole K slices from number `it` on, in both CTAs, and
// multiplies them, 4 MMAs of K = 16 (STEP 16-byte units apart in both operands) for
// each 128-row half of the CTAs' rows.  The first and the last ring of slices go
// through one half and then the other, so that a finished half is read out while the
// other's MMAs run; the slices between go through both in one unrolled sequence (in
// loops over the halves with a fence each, an MMA took 240 cycles instead of 130).
template <int STEP>
__device__ __forceinline__ bool issue(const Bars &bars, uint32_t it, int64_t t, int slices, bool last, int halves,
                                      uint64_t am, uint64_t an, uint32_t idesc, uint32_t tmem,
                                      volatile int *abort) {
    int k = 0;
    auto wait = [&](int i) { return pair_wait(&bars.full[(it + i) % kStages], ((it + i) / kStages) & 1, 3, abort); };
    auto half_of = [&](int i, int h) {
        const uint32_t s = (it + i) % kStages;
        const uint64_t m = am + (s * kStageBytes + h * 2 * kBox) / 16, n = an + s * (kStageBytes / 16);
#pragma unroll
        for (int kk = 0; kk < kGradSlice / 16; ++kk)
            mma2(tmem + 256u * h, m + kk * STEP, n + kk * STEP, idesc, (i | kk) != 0);
    };
    // `count` slices (the ring holds them) through one half and then the other
    auto skewed = [&](int count) {
        const bool ends = last && k + count == slices;
        if (k == 0 && t > 0 && !pair_wait(&bars.acc_empty[0], (uint32_t)(t - 1) & 1, 5, abort)) return false;
        for (int i = k; i < k + count; ++i) {
            if (!wait(i)) return false;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            half_of(i, 0);
            if (halves == 1) mma2_commit(&bars.empty[(it + i) % kStages]);
        }
        if (ends) mma2_commit(&bars.acc_full[0]);
        if (halves == 2) {
            if (k == 0 && t > 0) {
                if (!pair_wait(&bars.acc_empty[1], (uint32_t)(t - 1) & 1, 5, abort)) return false;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            }
            for (int i = k; i < k + count; ++i) {
                half_of(i, 1);
                mma2_commit(&bars.empty[(it + i) % kStages]);
            }
            if (ends) mma2_commit(&bars.acc_full[1]);
        }
        k += count;
        return true;
    };
    if (slices > 0 && !skewed(slices < kStages ? slices : kStages)) return false;
    for (; k < slices - kStages; ++k) {
        if (!wait(k)) return false;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        half_of(k, 0);
        if (halves == 2) half_of(k, 1);
        mma2_commit(&bars.empty[(it + k) % kStages]);
    }
    return k == slices || skewed(slices - k);
}

__device__ __forceinline__ uint32_t bf16_pair(uint32_t lo, uint32_t hi) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(__uint_as_float(lo), __uint_as_float(hi));
    return *reinterpret_cast<const uint32_t *>(&p);
}

// How the roles of CTA `rank` see an item: the first of the tile's rows that it
// holds, the boxes of each operand that it loads, the K slices, and the columns of
// the pair's N operand (it loads n / 2 of them).
struct Shape {
    int first, boxes_m, boxes_n, halves, slices, n;
};
__device__ __forceinline__ Shape shape_of(const GradArgs &p, const Item &q, int rank) {
    Shape s;
    const int m = q.kind == kDa ? q.rows : p.d1 - q.i0;
    const int n = q.kind == kDa ? p.d1 - q.j0 : p.d2 - q.j0;
    const int k = q.kind == kDa ? p.d2 : q.rows;
    s.halves = m > 256 ? 2 : 1;
    s.first = rank * 128 * s.halves;
    s.boxes_m = min(2 * s.halves, max(0, (m - s.first + 63) / 64));
    s.n = min(kGradCols, (n + 31) / 32 * 32);
    const int mine = s.n / 2, left = n - rank * mine;
    // the second CTA loads a box in any case (columns behind the operand's last, which
    // no result comes from): the first does not run ahead of it in the ring
    const int need = (left + 63) / 64, least = rank == 1 && s.boxes_m == 0;
    s.boxes_n = min((mine + 63) / 64, max(least, need));
    s.slices = (k + kGradSlice - 1) / kGradSlice;
    return s;
}

// Zeroes the rows of da past the last segment; thread `at` of `threads`.
__device__ __forceinline__ void zero_behind(const GradArgs &args, int64_t at, int64_t threads) {
    uint4 *da = reinterpret_cast<uint4 *>(args.da);  // d1 is a multiple of 8
    const int64_t first = args.off[args.r] * args.d1 / 8, end = args.n * args.d1 / 8;
    for (int64_t i = first + at; i < end; i += threads) da[i] = make_uint4(0, 0, 0, 0);
}

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    k_grad_tc(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_g,
              const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_da,
              const __grid_constant__ CUtensorMap map_db, const GradArgs args) {
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = blockIdx.x & 1;  // in the pair; 0 takes items and issues the MMAs
    unsigned char *ring = reinterpret_cast<unsigned char *>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint4 *staging = reinterpret_cast<uint4 *>(ring + kStages * kStageBytes);
    uint64_t *full = reinterpret_cast<uint64_t *>(ring + kStages * kStageBytes + kEpiWarps * 4096);
    uint64_t *empty = full + kStages;           // the MMAs have read the slice, in both CTAs
    // Slices of db that are not whole, in turn (the ring holds at most kStages of them):
    uint64_t *tail = empty + kStages;  // second CTA: the rows are there
    uint64_t *peer = tail + kStages;   // first CTA: and end in zeros there
    uint64_t *next_full = peer + kStages;       // [kQueue] an item has been published
    uint64_t *next_empty = next_full + kQueue;  // [kQueue] every role has read it
    uint64_t *acc_full = next_empty + kQueue;  // [2] a half of the accumulators is finished
    uint64_t *acc_empty = acc_full + 2;  // [2] first CTA: it has been read, in both CTAs
    uint64_t *mma_done = acc_empty + 2;
    Item *queue = reinterpret_cast<Item *>(mma_done + 1);
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(queue + kQueue);
    volatile int *abort = reinterpret_cast<volatile int *>(tmem_slot + 1);

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
            mbar_init(&tail[s], 1);
            mbar_init(&peer[s], 1);
        }
        for (int s = 0; s < kQueue; ++s) {
            mbar_init(&next_full[s], 1);
            mbar_init(&next_empty[s], 2 + kEpiWarps + (rank == 0));
        }
        for (int h = 0; h < 2; ++h) {
            mbar_init(&acc_full[h], 1);
            mbar_init(&acc_empty[h], 2 * kEpiWarps);
        }
        mbar_init(mma_done, 1);
        *abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kWarpMma) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                         smem_u32(tmem_slot)),
                     "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    cluster_barrier();  // the other CTA's barriers are initialised
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = *tmem_slot;
    next_may_start();
    before_is_done();

    // Item t of this CTA, for a whole warp: false when none is left.
    auto take = [&](int64_t t, Item &q) {
        const int s = (int)(t % kQueue);
        if (!warp_wait(&next_full[s], (uint32_t)(t / kQueue) & 1, 7, abort)) return false;
        q = queue[s];
        __syncwarp();
        if (lane == 0) mbar_arrive(&next_empty[s]);
        return q.kind != 0;
    };

    if (warp == kWarpNext) {
        // Second CTA: passes on that its roles have read an item (an arrival there from
        // each of them would hold the issuing thread up for some 1000 cycles an item).
        int64_t at = blockIdx.x / 2;
        if (rank == 1 && args.whole && args.da) zero_behind(args, at * 32 + lane, (int64_t)gridDim.x / 2 * 32);
        for (int64_t t = 0;; ++t) {
            const int s = (int)(t % kQueue);
            if (rank == 1) {
                if (!warp_wait(&next_empty[s], (uint32_t)(t / kQueue) & 1, 8, abort)) break;
                const bool end = queue[s].kind == 0;
                __syncwarp();
                if (lane == 0) arrive_in(&next_empty[s], 0);
                if (end) break;
                continue;
            }
            if (t >= kQueue && !warp_wait(&next_empty[s], (uint32_t)(t / kQueue - 1) & 1, 8, abort)) break;
            const Item q = item_at(args, at);
            if (lane == 0) {
                queue[s] = q;
                mbar_arrive(&next_full[s]);
                const uint32_t there = in_cta(&queue[s], 1);
                const int32_t *word = reinterpret_cast<const int32_t *>(&q);
#pragma unroll
                for (int i = 0; i < (int)(sizeof(Item) / 4); ++i)
                    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(there + 4 * i), "r"(word[i]) : "memory");
                arrive_in(&next_full[s], 1);
            }
            if (!q.kind) break;
            if (lane == 0)
                at = (int64_t)atomicAdd(reinterpret_cast<unsigned long long *>(&args.head[kHeadNext]), 1ull);
            at = __shfl_sync(0xffffffffu, at, 0);
        }
    } else if (warp == kWarpLoad) {
        const uint32_t ring_at = in_cta(ring, rank);
        int64_t it = 0, tails = 0;
        bool ok = true;
        Item q;
        for (int64_t t = 0; ok && take(t, q); ++t) {
            const Shape sh = shape_of(args, q, rank);
            if (lane == 0) {
                const int n0 = rank * (sh.n / 2);  // this CTA's columns of N
                // da: rows of grad and of b, along K; db: rows of the sum
                const bool da = q.kind == kDa;
                const CUtensorMap *of_m = da ? &map_g : &map_a, *of_n = da ? &map_b : &map_g;
                const int32_t m0 = da ? q.row0 + sh.first : q.i0 + sh.first;
                const int32_t c0 = da ? (int32_t)(q.seg * (int64_t)args.d1) + q.j0 + n0 : q.j0 + n0;
                const Shape other = shape_of(args, q, 1);
                const uint32_t mine = (uint32_t)(sh.boxes_m + sh.boxes_n) * kBox;
                const uint32_t both = mine + (uint32_t)(other.boxes_m + other.boxes_n) * kBox;
                const int whole = !da && q.rows % kGradSlice ? sh.slices - 1 : sh.slices;
                for (int k = 0; k < sh.slices; ++k, ++it) {
                    const int s = (int)(it % kStages);
                    if (it >= kStages &&
                        !(ok = pair_wait(&empty[s], (uint32_t)((it / kStages) - 1) & 1, 1, abort)))
                        break;
                    const uint32_t m = ring_at + s * kStageBytes, n = m + 4 * kBox;
                    uint32_t bar = in_cta(&full[s], 0);
                    if (rank == 0) {
                        mbar_arrive_expect_tx(&full[s], k < whole ? both : mine);
                    } else if (k == whole) {
                        uint64_t *at = &tail[tails++ % kStages];
                        bar = in_cta(at, 1);
                        mbar_arrive_expect_tx(at, mine);
                    }
                    const int32_t at = (da ? 0 : q.row0) + kGradSlice * k;
                    for (int b = 0; b < sh.boxes_m; ++b)
                        pair_load(m + b * kBox, of_m, bar, da ? at : m0 + 64 * b, da ? m0 + 64 * b : at);
                    for (int b = 0; b < sh.boxes_n; ++b)
                        pair_load(n + b * kBox, of_n, bar, da ? at : c0 + 64 * b, da ? c0 + 64 * b : at);
                }
            }
            ok = __shfl_sync(0xffffffffu, ok, 0);
        }
        // the last issued loads (at most one per stage) have landed before exit, the
        // second CTA's among them
        if (lane == 0 && rank == 0) for (int64_t j = (it > kStages ? it - kStages : 0); j < it; ++j)
            mbar_wait(&full[j % kStages], (uint32_t)(j / kStages) & 1, 2, nullptr);
        __syncwarp();
    } else if (warp == kWarpMma) {
        // First CTA: one thread issues, in a loop of its own over an item's whole
        // slices (with the warp taking part in every slice the issue of an MMA took
        // 217 cycles, where its execution takes 128).  Second CTA: the end of a db sum.
        int64_t it = 0, tails = 0;  // slices; those of db that are not whole
        bool ok = true;
        Item q;
        for (int64_t t = 0; ok && take(t, q); ++t) {
            const Shape sh = shape_of(args, q, rank);
            const bool da = q.kind == kDa;
            const uint32_t idesc = da ? k_instr(sh.n) : mn_instr(sh.n);
            const uint32_t ring_m = smem_u32(ring), ring_n = ring_m + 4 * kBox;
            const uint64_t am = da ? smem_desc(ring_m) : mn_desc(ring_m);
            const uint64_t an = da ? smem_desc(ring_n) : mn_desc(ring_n);
            // slices that are whole; db's last one may not be
            const int whole = !da && q.rows % kGradSlice ? sh.slices - 1 : sh.slices;
            if (lane == 0 && rank == 0) {
                const Bars bars = {full, empty, acc_full, acc_empty};
                // a half that `issue` does not come to
                for (int h = whole ? sh.halves : 0; t > 0 && ok && h < 2; ++h)
                    ok = pair_wait(&acc_empty[h], (uint32_t)(t - 1) & 1, 5, abort);
                const bool last = whole == sh.slices;
                if (ok) ok = da ? issue<2>(bars, (uint32_t)it, t, whole, last, sh.halves, am, an, idesc, tmem, abort)
                                : issue<128>(bars, (uint32_t)it, t, whole, last, sh.halves, am, an, idesc, tmem, abort);
                // those whose end it does not report
                for (int h = last && whole ? sh.halves : 0; last && ok && h < 2; ++h) mma2_commit(&acc_full[h]);
            }
            ok = __shfl_sync(0xffffffffu, ok, 0);
            it += whole;
            if (ok && whole < sh.slices) {
                const int s = (int)(it % kStages);
                if (!(ok = warp_wait(rank ? &tail[tails % kStages] : &full[s], (uint32_t)((rank ? tails : it) / kStages) & 1, 3, abort))) break;
                unsigned char *m = ring + s * kStageBytes;
                const int rows = q.rows % kGradSlice, steps = (rows + 15) / 16;
                const int zero = (steps * 16 - rows) * 8;  // 16-byte pieces of a box
                for (int b = 0; b < 6; ++b) {
                    if (b < 4 ? b >= sh.boxes_m : b - 4 >= sh.boxes_n) continue;
                    uint4 *p = reinterpret_cast<uint4 *>(m + b * kBox + rows * 128);
                    for (int i = lane; i < zero; i += 32) p[i] = make_uint4(0, 0, 0, 0);
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (rank == 1) {
                    if (lane == 0) arrive_in(&peer[tails % kStages], 0);
                } else {
                    if (!(ok = warp_wait(&peer[tails % kStages], (uint32_t)(tails / kStages) & 1, 9, abort))) break;
                    if (lane == 0) {
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        for (int h = 0; h < sh.halves; ++h)
                            for (int kk = 0; kk < steps; ++kk)
                                mma2(tmem + 256u * h, am + (s * kStageBytes + h * 2 * kBox) / 16 + kk * 128,
                                     an + s * kStageBytes / 16 + kk * 128, idesc, (whole | kk) != 0);
                        mma2_commit(&empty[s]);
                        mma2_commit(&acc_full[0]);
                        mma2_commit(&acc_full[1]);
                    }
                }
                ++it;
                ++tails;
            }
            if (!ok) break;
        }
        // every MMA issued above has completed, and every arrival in the second
        // CTA has been made, before the memory is freed
        if (lane == 0) {
            if (rank == 0) mma2_commit(mma_done);
            pair_wait(mma_done, 0, 6, nullptr);
        }
        __syncwarp();
    } else {
        // warp w reads TMEM lanes [32 (w % 4), 32 (w % 4) + 32), 128 columns of them, of
        // one half and then the other
        const int quarter = warp & 3, side = (warp - kWarpEpi0) >> 2;
        const uint32_t taddr = tmem + ((uint32_t)(quarter * 32) << 16) + 128u * side;
        uint4 *stg = staging + (warp - kWarpEpi0) * 256;
        Item q;
        bool ok = true;
        for (int64_t t = 0; ok && take(t, q); ++t) {
            const bool da = q.kind == kDa;
            const Shape sh = shape_of(args, q, rank);
            const int cols = (da ? args.d1 : args.d2) - q.j0 - 128 * side;
            const bool none = !da && q.rows <= 0;
            for (int half = 0; half < 2; ++half) {
                if (!(ok = warp_wait(&acc_full[half], (uint32_t)t & 1, 4, abort))) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const int line = sh.first + half * 128 + quarter * 32;  // first row of the tile here
                // those that exist; a half that is not used has none
                const int rows = half < sh.halves ? (da ? q.rows : args.d1 - q.i0) - line : 0;
                // the values come out first, so that the accumulators are free for the
                // next tile while these are stored
                uint32_t v[2][64];
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    if (rows <= 0 || 64 * c >= cols) continue;
                    if (none) {
#pragma unroll
                        for (int i = 0; i < 64; ++i) v[c][i] = 0;
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            tmem_ld16(taddr + (uint32_t)(256 * half + 64 * c + 16 * i),
                                      *reinterpret_cast<uint32_t(*)[16]>(&v[c][16 * i]));
                    }
                }
                tmem_wait_ld();
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) signal_in(&acc_empty[half], 0);
                // a piece: float32, [CTA][half][16-byte column group][row of the half],
                // whole lines a warp
                uint4 *piece = reinterpret_cast<uint4 *>(args.partial + (int64_t)q.slot * kPartial) +
                               ((rank * 2 + half) * 64 + side * 32) * 128 + quarter * 32 + lane;
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    if (rows <= 0 || 64 * c >= cols) continue;
                    const uint32_t(&w)[64] = v[c];
                    if (q.slot >= 0) {
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            piece[(c * 16 + i) * 128] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
                        continue;
                    }
                    if (lane == 0) bulk_wait_read<0>();
                    __syncwarp();
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        stg[lane * 8 + (j ^ (lane & 7))] =
                            make_uint4(bf16_pair(w[8 * j], w[8 * j + 1]), bf16_pair(w[8 * j + 2], w[8 * j + 3]),
                                       bf16_pair(w[8 * j + 4], w[8 * j + 5]), bf16_pair(w[8 * j + 6], w[8 * j + 7]));
                    const int col0 = q.j0 + 128 * side + 64 * c;
                    if (da && rows < 32) {
                        // the segment's last rows: the next segment's must not be written
                        __syncwarp();
                        for (int i = lane; i < rows * 8; i += 32) {
                            const int row = i >> 3, j = i & 7, col = col0 + j * 8;
                            if (col < args.d1)
                                *reinterpret_cast<uint4 *>(args.da + ((int64_t)q.row0 + line + row) * args.d1 + col) =
                                    stg[row * 8 + (j ^ (row & 7))];
                        }
                        __syncwarp();
                    } else {
                        fence_proxy_async_smem();
                        __syncwarp();
                        if (lane == 0) {
                            if (da)
                                tma_store_2d(&map_da, stg, col0, q.row0 + line);
                            else  // clipped to the segment's block
                                tma_store_3d(&map_db, stg, col0, q.i0 + line, q.seg);
                            bulk_commit();
                        }
                    }
                }
            }
        }
        if (lane == 0) bulk_wait_all();
        __syncwarp();
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    // the first CTA's MMAs have read the second's shared memory, and all arrivals
    // in the other CTA have been made
    cluster_barrier();
    if (warp == kWarpMma) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
    }
}

// Adds the pieces of db's cut tiles, 16 columns a thread, and zeroes the rows of
// da past the last segment.
__global__ void __launch_bounds__(256) k_grad_finish(const GradArgs args) {
    before_is_done();
    if (args.da) zero_behind(args, (blockIdx.x + (int64_t)blockIdx.y * gridDim.x) * 256 + threadIdx.x,
                             (int64_t)gridDim.x * gridDim.y * 256);
    if (!args.db) return;
    const int64_t cuts = args.head[kHeadCut];
    for (int64_t cut = blockIdx.x; cut < cuts; cut += gridDim.x) {
        const int64_t k = warp_search(args.cut_off, args.r, cut);
        const int32_t seg = args.order[k];
        const int64_t tile = cut - args.cut_off[k];
        const int64_t count = grad_pieces(args.off[seg + 1] - args.off[seg], args.head[kHeadPiece]).count;
        // CTA, half, 16 groups of 16 columns, 128 rows
        const int idx = blockIdx.y * 256 + threadIdx.x;
        const int line = idx & 127, group = (idx >> 7) & 15, half = idx >> 11 & 1, cta = idx >> 12;
        const int32_t i0 = (int32_t)(tile / args.tiles2) * kGradRows;
        const int halves = args.d1 - i0 > 256 ? 2 : 1;
        const int32_t i = i0 + (cta * halves + half) * 128 + line;
        const int32_t j = (int32_t)(tile % args.tiles2) * kGradCols + group * 16;
        if (half >= halves || i >= args.d1 || j >= args.d2) continue;
        const float4 *src = reinterpret_cast<const float4 *>(
                                args.partial + (args.slot_off[k] + tile * count) * kPartial) +
                            ((cta * 2 + half) * 64 + group * 4) * 128 + line;
        float4 sum[4];
#pragma unroll
        for (int v = 0; v < 4; ++v) sum[v] = make_float4(0, 0, 0, 0);
        constexpr int kFlight = 4;  // pieces under way
        for (int64_t p0 = 0; p0 < count; p0 += kFlight) {
            float4 x[kFlight][4];
#pragma unroll
            for (int p = 0; p < kFlight; ++p)
#pragma unroll
                for (int v = 0; v < 4; ++v)
                    x[p][v] = p0 + p < count ? __ldcs(src + (p0 + p) * (kPartial / 4) + v * 128)
                                             : make_float4(0, 0, 0, 0);
#pragma unroll
            for (int p = 0; p < kFlight; ++p)
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    sum[v].x += x[p][v].x;
                    sum[v].y += x[p][v].y;
                    sum[v].z += x[p][v].z;
                    sum[v].w += x[p][v].w;
                }
        }
        __nv_bfloat16 *dst = args.db + (seg * (int64_t)args.d1 + i) * args.d2 + j;
#pragma unroll
        for (int v = 0; v < 2; ++v) {  // d2 is a multiple of 8
            if (j + 8 * v >= args.d2) break;
            __nv_bfloat162 o[4] = {__floats2bfloat162_rn(sum[2 * v].x, sum[2 * v].y),
                                   __floats2bfloat162_rn(sum[2 * v].z, sum[2 * v].w),
                                   __floats2bfloat162_rn(sum[2 * v + 1].x, sum[2 * v + 1].y),
                                   __floats2bfloat162_rn(sum[2 * v + 1].z, sum[2 * v + 1].w)};
            *reinterpret_cast<uint4 *>(dst + 8 * v) = *reinterpret_cast<uint4 *>(o);
        }
    }
}

// A bf16 tensor map with SWIZZLE_128B boxes of 64 columns.
int bf16_map(CUtensorMap *map, const void *ptr, int rank, const int64_t *dims, uint32_t box_rows) {
    auto fn = encode_fn();
    if (!fn) return fail(BGL_E_CUDA, "cuTensorMapEncodeTiled is not available");
    cuuint64_t size[3], stride[2];
    cuuint32_t box[3] = {64, box_rows, 1}, step[3] = {1, 1, 1};
    for (int i = 0; i < rank; ++i) size[i] = (cuuint64_t)dims[i];
    stride[0] = size[0] * 2;
    stride[1] = rank > 2 ? stride[0] * size[1] : 0;
    CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, (cuuint32_t)rank, const_cast<void *>(ptr),
                    size, stride, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(BGL_E_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
    return BGL_OK;
}

}  // namespace

// TMA wants 16-byte aligned bases and row strides, and 32-bit row numbers.
bool gmm_grad_tc_supported(const void *grad, const void *a, const void *b, const void *da,
                           const void *db, int64_t n, int64_t d1, int64_t r, int64_t d2, int dtype) {
    return dtype == BGL_BF16 && (da || db) && n > 0 && d1 > 0 && d2 > 0 && d1 % 8 == 0 &&
           d2 % 8 == 0 && n < (int64_t(1) << 31) - 1024 &&
           r * d1 < (int64_t(1) << 31) - 1024 &&
           d1 * d2 < (int64_t(1) << 39) && aligned(grad, 16) && (!da || (aligned(da, 16) && aligned(b, 16))) &&
           (!db || (aligned(db, 16) && aligned(a, 16)));
}

GradTiles gmm_grad_tiles(int64_t n, int64_t d1, int64_t r, int64_t d2) {
    GradTiles t;
    t.cols = (d1 + kGradCols - 1) / kGradCols;
    t.tiles1 = (d1 + kGradRows - 1) / kGradRows;
    t.tiles2 = (d2 + kGradCols - 1) / kGradCols;
    // no more pairs than there can be items: row tiles of da and slices of db
    const int64_t items = t.cols * (n / kGradRows + r) + t.tiles1 * t.tiles2 * (n / (kGradShortest * kGradSlice) + r);
    const int64_t most = num_sms() / 2;
    t.pairs = (int)(items < most ? (items > 0 ? items : 1) : most);
    return t;
}

int gmm_grad_tensor_core(const void *grad, const void *a, const void *b, void *da, void *db,
                         const GradLayout &l, const GradTiles &t, int64_t n, int64_t d1, int64_t r,
                         int64_t d2, cudaStream_t s) {
    CUtensorMap map_a, map_g, map_b, map_da, map_db;
    const int64_t dims_a[2] = {d1, n}, dims_g[2] = {d2, n}, dims_b[2] = {d2, r * d1},
                  dims_db[3] = {d2, d1, r};
    int rc = bf16_map(&map_g, grad, 2, dims_g, kGradSlice);
    map_a = map_b = map_da = map_db = map_g;  // not read where a gradient is not wanted
    if (!rc && da) rc = bf16_map(&map_b, b, 2, dims_b, kGradSlice);
    if (!rc && da) rc = bf16_map(&map_da, da, 2, dims_a, 32);
    if (!rc && db) rc = bf16_map(&map_a, a, 2, dims_a, kGradSlice);
    if (!rc && db) rc = bf16_map(&map_db, db, 3, dims_db, 32);
    if (rc) return rc;
    GradArgs args;
    args.off = l.off;
    args.row_off = l.row_off;
    args.item_off = l.item_off;
    args.cut_off = l.cut_off;
    args.slot_off = l.slot_off;
    args.order = l.order;
    args.head = l.head;
    args.partial = l.partial;
    args.da = static_cast<__nv_bfloat16 *>(da);
    args.db = static_cast<__nv_bfloat16 *>(db);
    args.r = r;
    args.n = n;
    args.cols = (int32_t)t.cols;
    args.tiles1 = (int32_t)t.tiles1;
    args.tiles2 = (int32_t)t.tiles2;
    args.d1 = (int32_t)d1;
    args.d2 = (int32_t)d2;
    // No sum of so few rows is cut, and the few rows behind are zeroed on the side (190
    // rows: 23.0 us with a launch for that, 21.1 us so).
    args.whole = n <= kGradShortest * kGradSlice;
    BGL_CUDA(cudaFuncSetAttribute(k_grad_tc, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmem));
    BGL_CUDA(launch_after(k_grad_tc, 2 * t.pairs, kThreads, kSmem, s, map_a, map_g, map_b, map_da, map_db, args));
    if (!args.whole) BGL_CUDA(launch_after(k_grad_finish, dim3((unsigned)t.pairs, 32), 256, 0, s, args));
    return BGL_OK;
}

cudaError_t gmm_grad_tc_error(int *code) { return take_tc_error(code); }

}  // namespace bgl
