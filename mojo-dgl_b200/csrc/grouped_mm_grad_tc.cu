// tcgen05 kernel for the gradients of segment_mm in bfloat16, float32 sums:
//
//   da[i] = grad[i] @ b[r]^T                  (K = d2: both operands K-major)
//   db[r] = a[rows of r]^T @ grad[rows of r]  (K = rows: both M/N-major)
//
// Every operand is read as it lies in memory, 64 rows x 64 columns a TMA box;
// a box serves as K-major rows or as M/N-major columns, so the two products
// differ only in coordinates and descriptors, and no transposed copy is made.
// A CTA works on one 256 x 256 tile at a time: two 128 x 256 float32
// accumulators fill the tensor memory, and each K slice of 64 (32 KB + 32 KB)
// feeds 2 x 4 MMAs, so a loaded byte meets 4/3 of the products of a 128 x 256
// tile: what bounds wide blocks is the rate at which L2 hands out tiles.
//
// One persistent launch holds both products.  Warp 10 takes the next item (an
// atomic counter; which CTA does what does not change any result) and
// publishes it through a four-deep queue, warp 0 issues the loads into a
// three-slice ring, warp 1 the MMAs, warps 2-9 write finished tiles out
// (through a swizzled staging box and TMA stores).
//
// A db slice's rows beyond the segment belong to the next one: the MMA warp
// writes zeros over those that share a 16-row MMA step with the segment's last
// rows (in both operands, so that inf and NaN of a neighbour do not get in) and
// leaves out the steps behind.  Pieces of a cut db tile go to float32 partial
// tiles, which k_grad_finish adds in order: the same bits on every run.
//
// Every mbarrier wait is bounded, with the abort protocol of grouped_mm_tc.cu.
#include "grouped_mm.cuh"
#include "tcgen05.cuh"

namespace bgl {
namespace {

constexpr int kStages = 3;
constexpr int kBox = kGradSlice * 128;        // 64 rows x 64 columns of bf16
constexpr int kStageBytes = 8 * kBox;         // 4 boxes of each operand
constexpr int kEpiWarps = 8;                  // two a TMEM lane quarter, one for each half
constexpr int kQueue = 4;
constexpr int kWarpLoad = 0, kWarpMma = 1, kWarpEpi0 = 2, kWarpNext = kWarpEpi0 + kEpiWarps;
constexpr int kThreads = 32 * (kWarpNext + 1);
constexpr int kPartial = kGradTile * kGradTile;  // values of a partial tile

struct GradArgs {
    const int64_t *off, *row_off, *item_off, *cut_off, *slot_off;
    const int32_t *order;
    int64_t *head;
    float *partial;
    __nv_bfloat16 *da, *db;
    int64_t r, n;
    int32_t tiles1, tiles2, d1, d2;
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
                         8 * (2 * kStages + 2 * kQueue + 4) + kQueue * sizeof(Item) + 16;

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
        q.i0 = (int32_t)(tile / p.tiles2) * kGradTile;
        q.j0 = (int32_t)(tile % p.tiles2) * kGradTile;
        const int64_t skip = piece * cut.slices * kGradSlice, most = cut.slices * kGradSlice;
        q.row0 = (int32_t)(first + skip);
        q.rows = (int32_t)(len - skip < most ? len - skip : most);
        q.slot = cut.count > 1 ? (int32_t)(p.slot_off[k] + tile * cut.count + piece) : -1;
    } else {
        const int64_t in = at - db_items, tile = in / p.tiles1;
        q.kind = kDa;
        q.seg = (int32_t)warp_search(p.row_off, p.r, tile);
        const int64_t first = p.off[q.seg] + (tile - p.row_off[q.seg]) * kGradTile;
        const int64_t left = p.off[q.seg + 1] - first;
        q.row0 = (int32_t)first;
        q.rows = (int32_t)(left < kGradTile ? left : kGradTile);
        q.j0 = (int32_t)(in % p.tiles1) * kGradTile;
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

// Instruction descriptors: fp32 accumulator, bf16 operands, M = 128, both
// operands K-major or both M/N-major.
__device__ __forceinline__ uint32_t k_instr(int n) {
    return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
__device__ __forceinline__ uint32_t mn_instr(int n) {
    return k_instr(n) | (1u << 15) | (1u << 16);
}

// Lane 0 waits for the whole warp.
__device__ __forceinline__ bool warp_wait(uint64_t *bar, uint32_t parity, int code,
                                          volatile int *abort) {
    int ok = 0;
    if ((threadIdx.x & 31) == 0) ok = mbar_wait(bar, parity, code, abort);
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

// Waits for `slices` whole K slices from number `it` on and multiplies them, 4 MMAs
// of K = 16 (STEP 16-byte units apart in both operands) for each 128-row half.
template <int STEP>
__device__ __forceinline__ bool issue(uint64_t *full, uint64_t *empty, int64_t it, int slices,
                                      int halves, uint64_t am, uint64_t an, uint32_t idesc,
                                      uint32_t tmem, volatile int *abort) {
    int s = (int)(it % kStages);
    uint32_t parity = (uint32_t)(it / kStages) & 1;
    for (int k = 0; k < slices; ++k) {
        if (!mbar_wait(&full[s], parity, 3, abort)) return false;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint64_t m = am + s * (kStageBytes / 16), n = an + s * (kStageBytes / 16);
#pragma unroll
        for (int kk = 0; kk < kGradSlice / 16; ++kk)
            mma<true>(tmem, m + kk * STEP, n + kk * STEP, idesc, (k | kk) != 0);
        if (halves == 2) {
#pragma unroll
            for (int kk = 0; kk < kGradSlice / 16; ++kk)
                mma<true>(tmem + 256u, m + 2 * kBox / 16 + kk * STEP, n + kk * STEP, idesc, (k | kk) != 0);
        }
        mma_commit(&empty[s]);
        if (++s == kStages) s = 0, parity ^= 1;
    }
    return true;
}

__device__ __forceinline__ uint32_t bf16_pair(uint32_t lo, uint32_t hi) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(__uint_as_float(lo), __uint_as_float(hi));
    return *reinterpret_cast<const uint32_t *>(&p);
}

// How the roles see an item: the boxes of each operand that are loaded, and the
// K slices.
struct Shape {
    int boxes_m, boxes_n, halves, slices, n;
};
__device__ __forceinline__ Shape shape_of(const GradArgs &p, const Item &q) {
    Shape s;
    const int m = q.kind == kDa ? q.rows : p.d1 - q.i0;
    const int n = q.kind == kDa ? p.d1 - q.j0 : p.d2 - q.j0;
    const int k = q.kind == kDa ? p.d2 : q.rows;
    s.boxes_m = min(4, (m + 63) / 64);
    s.boxes_n = min(4, (n + 63) / 64);
    s.halves = m > 128 ? 2 : 1;
    s.slices = (k + kGradSlice - 1) / kGradSlice;
    s.n = min(kGradTile, (n + 15) / 16 * 16);
    return s;
}

__global__ void __launch_bounds__(kThreads, 1)
    k_grad_tc(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_g,
              const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_da,
              const __grid_constant__ CUtensorMap map_db, const GradArgs args) {
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    unsigned char *ring = reinterpret_cast<unsigned char *>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint4 *staging = reinterpret_cast<uint4 *>(ring + kStages * kStageBytes);
    uint64_t *full = reinterpret_cast<uint64_t *>(ring + kStages * kStageBytes + kEpiWarps * 4096);
    uint64_t *empty = full + kStages;
    uint64_t *next_full = empty + kStages;      // [kQueue] an item has been published
    uint64_t *next_empty = next_full + kQueue;  // [kQueue] every role has read it
    uint64_t *acc_full = next_empty + kQueue;
    uint64_t *acc_empty = acc_full + 1;  // [2]: a half of the accumulators has been read
    uint64_t *mma_done = acc_empty + 2;
    Item *queue = reinterpret_cast<Item *>(mma_done + 1);
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(queue + kQueue);
    volatile int *abort = reinterpret_cast<volatile int *>(tmem_slot + 1);

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int s = 0; s < kQueue; ++s) {
            mbar_init(&next_full[s], 1);
            mbar_init(&next_empty[s], 2 + kEpiWarps);
        }
        mbar_init(acc_full, 1);
        mbar_init(&acc_empty[0], kEpiWarps / 2);
        mbar_init(&acc_empty[1], kEpiWarps / 2);
        mbar_init(mma_done, 1);
        *abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kWarpMma) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                         smem_u32(tmem_slot)),
                     "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = *tmem_slot;

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
        int64_t at = blockIdx.x;
        for (int64_t t = 0;; ++t) {
            const int s = (int)(t % kQueue);
            if (t >= kQueue && !warp_wait(&next_empty[s], (uint32_t)(t / kQueue - 1) & 1, 8, abort)) break;
            const Item q = item_at(args, at);
            if (lane == 0) {
                queue[s] = q;
                mbar_arrive(&next_full[s]);
            }
            if (!q.kind) break;
            if (lane == 0)
                at = (int64_t)atomicAdd(reinterpret_cast<unsigned long long *>(&args.head[kHeadNext]), 1ull);
            at = __shfl_sync(0xffffffffu, at, 0);
        }
    } else if (warp == kWarpLoad) {
        int64_t it = 0;
        bool ok = true;
        Item q;
        for (int64_t t = 0; ok && take(t, q); ++t) {
            const Shape sh = shape_of(args, q);
            for (int k = 0; k < sh.slices; ++k, ++it) {
                const int s = (int)(it % kStages);
                if (it >= kStages &&
                    !(ok = warp_wait(&empty[s], (uint32_t)((it / kStages) - 1) & 1, 1, abort)))
                    break;
                if (lane == 0) {
                    unsigned char *m = ring + s * kStageBytes, *n = m + 4 * kBox;
                    mbar_arrive_expect_tx(&full[s], (uint32_t)(sh.boxes_m + sh.boxes_n) * kBox);
                    if (q.kind == kDa) {
                        const int32_t row = (int32_t)(q.seg * (int64_t)args.d1) + q.j0;
                        for (int b = 0; b < sh.boxes_m; ++b)
                            tma_load_2d(m + b * kBox, &map_g, &full[s], 64 * k, q.row0 + 64 * b);
                        for (int b = 0; b < sh.boxes_n; ++b)
                            tma_load_2d(n + b * kBox, &map_b, &full[s], 64 * k, row + 64 * b);
                    } else {
                        const int32_t row = q.row0 + kGradSlice * k;
                        for (int b = 0; b < sh.boxes_m; ++b)
                            tma_load_2d(m + b * kBox, &map_a, &full[s], q.i0 + 64 * b, row);
                        for (int b = 0; b < sh.boxes_n; ++b)
                            tma_load_2d(n + b * kBox, &map_g, &full[s], q.j0 + 64 * b, row);
                    }
                }
                __syncwarp();
            }
        }
        // the last issued loads (at most one per stage) have landed before exit
        for (int64_t j = (it > kStages ? it - kStages : 0); j < it; ++j)
            mbar_wait(&full[j % kStages], (uint32_t)(j / kStages) & 1, 2, nullptr);
        __syncwarp();
    } else if (warp == kWarpMma) {
        // One thread issues, in a loop of its own over an item's whole slices: with
        // the warp taking part in every slice the issue of an MMA took 217 cycles,
        // where its execution takes 128.
        int64_t it = 0;
        bool ok = true;
        Item q;
        for (int64_t t = 0; ok && take(t, q); ++t) {
            const Shape sh = shape_of(args, q);
            const bool da = q.kind == kDa;
            const uint32_t idesc = da ? k_instr(sh.n) : mn_instr(sh.n);
            const uint32_t ring_m = smem_u32(ring), ring_n = ring_m + 4 * kBox;
            const uint64_t am = da ? smem_desc(ring_m) : mn_desc(ring_m);
            const uint64_t an = da ? smem_desc(ring_n) : mn_desc(ring_n);
            // slices that are whole; db's last one may not be
            const int whole = !da && q.rows % kGradSlice ? sh.slices - 1 : sh.slices;
            if (lane == 0) {
                for (int h = 0; t > 0 && ok && h < 2; ++h) ok = mbar_wait(&acc_empty[h], (uint32_t)(t - 1) & 1, 5, abort);
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                if (ok) ok = da ? issue<2>(full, empty, it, whole, sh.halves, am, an, idesc, tmem, abort)
                                : issue<128>(full, empty, it, whole, sh.halves, am, an, idesc, tmem, abort);
            }
            ok = __shfl_sync(0xffffffffu, ok, 0);
            it += whole;
            if (ok && whole < sh.slices) {
                const int s = (int)(it % kStages);
                if (!(ok = warp_wait(&full[s], (uint32_t)(it / kStages) & 1, 3, abort))) break;
                unsigned char *m = ring + s * kStageBytes;
                const int rows = q.rows % kGradSlice, steps = (rows + 15) / 16;
                const int zero = (steps * 16 - rows) * 8;  // 16-byte pieces of a box
                for (int b = 0; b < 8; ++b) {
                    if (b < 4 ? b >= sh.boxes_m : b - 4 >= sh.boxes_n) continue;
                    uint4 *p = reinterpret_cast<uint4 *>(m + b * kBox + rows * 128);
                    for (int i = lane; i < zero; i += 32) p[i] = make_uint4(0, 0, 0, 0);
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    for (int h = 0; h < sh.halves; ++h)
                        for (int kk = 0; kk < steps; ++kk)
                            mma<true>(tmem + 256u * h, am + (s * kStageBytes + h * 2 * kBox) / 16 + kk * 128,
                                      an + s * kStageBytes / 16 + kk * 128, idesc, (whole | kk) != 0);
                    mma_commit(&empty[s]);
                }
                ++it;
            }
            if (!ok) break;
            // (all epilogue warps have seen the tile before: they have read it)
            if (lane == 0) mma_commit(acc_full);
            __syncwarp();
        }
        // every MMA issued above has completed before the memory is freed
        if (lane == 0) {
            mma_commit(mma_done);
            mbar_wait(mma_done, 0, 6, nullptr);
        }
        __syncwarp();
    } else {
        // warp w reads TMEM lanes [32 (w % 4), 32 (w % 4) + 32) of one half
        const int quarter = warp & 3, half = (warp - kWarpEpi0) >> 2;
        const uint32_t taddr = tmem + ((uint32_t)(quarter * 32) << 16) + 256u * half;
        uint4 *stg = staging + (warp - kWarpEpi0) * 256;
        const int line = half * 128 + quarter * 32;  // first row of the tile here
        auto release = [&] {  // the accumulators have been read
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&acc_empty[half]);
        };
        Item q;
        for (int64_t t = 0; take(t, q); ++t) {
            if (!warp_wait(acc_full, (uint32_t)t & 1, 4, abort)) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const bool da = q.kind == kDa;
            const int rows = (da ? q.rows : args.d1 - q.i0) - line;  // those that exist
            const int cols = (da ? args.d1 : args.d2) - q.j0;
            const bool none = !da && q.rows <= 0;
            if (q.slot >= 0) {
                // a piece: float32, [half][16-byte column group][row of the half],
                // whole lines a warp
                for (int c = 0; rows > 0 && c < kGradTile && c < cols; c += 64) {
                    uint32_t v[64];
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        tmem_ld16(taddr + (uint32_t)(c + 16 * i),
                                  *reinterpret_cast<uint32_t(*)[16]>(&v[16 * i]));
                    tmem_wait_ld();
                    uint4 *dst = reinterpret_cast<uint4 *>(args.partial + (int64_t)q.slot * kPartial) +
                                 (half * 64 + c / 4) * 128 + quarter * 32 + lane;
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        dst[i * 128] = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
                }
                release();
                continue;
            }
            // the tile comes out as bf16 pairs first, so that the accumulators are
            // free for the next one while this one is stored
            uint4 o[4][8];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                if (rows <= 0 || 64 * c >= cols) continue;
                uint32_t v[64];
                if (none) {
#pragma unroll
                    for (int i = 0; i < 64; ++i) v[i] = 0;
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        tmem_ld16(taddr + (uint32_t)(64 * c + 16 * i),
                                  *reinterpret_cast<uint32_t(*)[16]>(&v[16 * i]));
                    tmem_wait_ld();
                }
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    o[c][j] = make_uint4(bf16_pair(v[8 * j], v[8 * j + 1]), bf16_pair(v[8 * j + 2], v[8 * j + 3]),
                                         bf16_pair(v[8 * j + 4], v[8 * j + 5]), bf16_pair(v[8 * j + 6], v[8 * j + 7]));
            }
            release();
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                if (rows <= 0 || 64 * c >= cols) continue;
                if (lane == 0) bulk_wait_read<0>();
                __syncwarp();
#pragma unroll
                for (int j = 0; j < 8; ++j) stg[lane * 8 + (j ^ (lane & 7))] = o[c][j];
                if (da && rows < 32) {
                    // the segment's last rows: the next segment's must not be written
                    __syncwarp();
                    for (int i = lane; i < rows * 8; i += 32) {
                        const int row = i >> 3, j = i & 7, col = q.j0 + 64 * c + j * 8;
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
                            tma_store_2d(&map_da, stg, q.j0 + 64 * c, q.row0 + line);
                        else  // clipped to the segment's block
                            tma_store_3d(&map_db, stg, q.j0 + 64 * c, q.i0 + line, q.seg);
                        bulk_commit();
                    }
                }
            }
        }
        if (lane == 0) bulk_wait_all();
        __syncwarp();
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == kWarpMma) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
    }
}

// Adds the pieces of db's cut tiles, 16 columns a thread, and zeroes the rows of
// da past the last segment.
__global__ void __launch_bounds__(256) k_grad_finish(const GradArgs args) {
    if (args.da) {
        const int64_t first = args.off[args.r] * args.d1 / 8, end = args.n * args.d1 / 8;
        const int64_t block = blockIdx.x + (int64_t)blockIdx.y * gridDim.x;
        uint4 *da = reinterpret_cast<uint4 *>(args.da);  // d1 is a multiple of 8
        for (int64_t i = first + block * 256 + threadIdx.x; i < end;
             i += (int64_t)gridDim.x * gridDim.y * 256)
            da[i] = make_uint4(0, 0, 0, 0);
    }
    if (!args.db) return;
    const int64_t cuts = args.head[kHeadCut];
    for (int64_t cut = blockIdx.x; cut < cuts; cut += gridDim.x) {
        const int64_t k = warp_search(args.cut_off, args.r, cut);
        const int32_t seg = args.order[k];
        const int64_t tile = cut - args.cut_off[k];
        const int64_t count = grad_pieces(args.off[seg + 1] - args.off[seg], args.head[kHeadPiece]).count;
        const int idx = blockIdx.y * 256 + threadIdx.x;  // half, 16 groups of 16 columns, 128 rows
        const int line = idx & 127, group = (idx >> 7) & 15, half = idx >> 11;
        const int32_t i = (int32_t)(tile / args.tiles2) * kGradTile + half * 128 + line;
        const int32_t j = (int32_t)(tile % args.tiles2) * kGradTile + group * 16;
        if (i >= args.d1 || j >= args.d2) continue;
        const float4 *src = reinterpret_cast<const float4 *>(
                                args.partial + (args.slot_off[k] + tile * count) * kPartial) +
                            (half * 64 + group * 4) * 128 + line;
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
    t.tiles1 = (d1 + kGradTile - 1) / kGradTile;
    t.tiles2 = (d2 + kGradTile - 1) / kGradTile;
    // no more CTAs than there can be items: row tiles of da and slices of db
    const int64_t items = t.tiles1 * (n / kGradTile + r) + t.tiles1 * t.tiles2 * (n / (8 * kGradSlice) + r);
    t.ctas = (int)(items < num_sms() ? (items > 0 ? items : 1) : num_sms());
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
    args.tiles1 = (int32_t)t.tiles1;
    args.tiles2 = (int32_t)t.tiles2;
    args.d1 = (int32_t)d1;
    args.d2 = (int32_t)d2;
    BGL_CUDA(cudaFuncSetAttribute(k_grad_tc, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmem));
    k_grad_tc<<<t.ctas, kThreads, kSmem, s>>>(map_a, map_g, map_b, map_da, map_db, args);
    BGL_LAUNCH_CHECK();
    k_grad_finish<<<dim3((unsigned)t.ctas, 16), 256, 0, s>>>(args);
    BGL_LAUNCH_CHECK();
    return BGL_OK;
}

cudaError_t gmm_grad_tc_error(int *code) { return take_tc_error(code); }

}  // namespace bgl
