// tcgen05 kernel for the weight gradient of segment_mm in bfloat16:
// db[r] = a[rows of r]^T @ grad[rows of r], float32 sums.
//
// The sum runs over rows, so both operands are read as they lie in memory, 64
// rows x 64 columns a TMA box, and are M- and N-major for the tensor cores (no
// transposed copies).  A CTA owns a 256 x 256 tile of a segment's block: two
// 128 x 256 float32 accumulators fill the tensor memory, and each 64-row slice
// of 32 KB + 32 KB feeds 2 x 4 MMAs, so a loaded byte meets twice the products
// of a 128 x 256 tile.  Warp 0 issues the loads into a three-slice ring, warp 1
// the MMAs, warps 2-9 write finished tiles out (through a swizzled staging box
// and TMA stores, clipped to the segment's block by the 3-D tensor map).
//
// A slice's rows beyond the segment belong to the next one: the MMA warp writes
// zeros over those that share a 16-row MMA step with the segment's last rows
// (in both operands, so that inf and NaN of a neighbour do not get in) and
// leaves out the steps behind.
//
// Units (one slice of one tile) are handed out as whole tiles, or split evenly
// over the CTAs (GradLayout::mode): a tile cut between CTAs then goes to float32
// partial tiles, which k_grad_join adds in order -- the same bits on every run.
//
// Every mbarrier wait is bounded, with the abort protocol of grouped_mm_tc.cu.
#include "grouped_mm.cuh"
#include "tcgen05.cuh"

namespace bgl {
namespace {

constexpr int kStages = 3;
constexpr int kBox = kGradSlice * 128;        // 64 rows x 64 columns of bf16
constexpr int kStageBytes = 8 * kBox;         // 4 boxes of a, 4 of grad
constexpr int kEpiWarps = 8;                  // two a TMEM lane quarter, one for each half
constexpr int kWarpLoad = 0, kWarpMma = 1, kWarpEpi0 = 2;
constexpr int kThreads = 32 * (kWarpEpi0 + kEpiWarps);
constexpr int kPartial = kGradTile * kGradTile;  // values of a partial tile
constexpr size_t kSmem = 1024 + kStages * (size_t)kStageBytes + kEpiWarps * 4096 + 8 * (2 * kStages + 4) + 16;

struct GradArgs {
    const int64_t *off, *unit_off, *mode;
    float *partial;
    int64_t r, per_segment;
    int32_t tiles_n, d1, d2;
};

// What a CTA does to one tile: rows [row0, row0 + rows) of segment seg, the
// tile at (i0, j0) of the segment's block; `slot` is the partial tile it goes
// to, -1 where it is the whole sum.
struct Piece {
    int64_t seg, row0, rows;
    int32_t i0, j0;
    int64_t slot;
    bool lead;  // holds the tile's first rows
};

// Walks a CTA's pieces; every role of the CTA sees the same ones.
struct Walk {
    int64_t at, end;  // tiles (whole) or units (split)
    bool split;

    __device__ __forceinline__ Walk(const GradArgs &p, int64_t cta, int64_t ctas) {
        split = *p.mode != 0;
        const int64_t units = p.unit_off[p.r];
        at = split ? units * cta / ctas : cta;
        end = split ? units * (cta + 1) / ctas : p.r * p.per_segment;
    }

    __device__ __forceinline__ bool next(const GradArgs &p, int64_t cta, int64_t ctas, Piece &q) {
        if (at >= end) return false;
        int64_t tile, k = 0, take;
        if (split) {
            int64_t lo = 0, hi = p.r - 1;  // last segment whose first unit is <= at
            while (lo < hi) {
                const int64_t mid = (lo + hi + 1) >> 1;
                if (p.unit_off[mid] <= at) lo = mid; else hi = mid - 1;
            }
            q.seg = lo;
            const int64_t slices = (p.unit_off[lo + 1] - p.unit_off[lo]) / p.per_segment;
            const int64_t in = at - p.unit_off[lo];
            tile = in / slices;
            k = in % slices;
            take = slices - k < end - at ? slices - k : end - at;
            q.lead = k == 0;
            q.slot = q.lead && take == slices ? -1 : 2 * cta + (q.lead ? 1 : 0);
            at += take;
        } else {
            q.seg = at / p.per_segment;
            tile = at % p.per_segment;
            take = INT32_MAX;
            q.lead = true;
            q.slot = -1;
            at += ctas;
        }
        const int64_t first = p.off[q.seg] + k * kGradSlice, last = p.off[q.seg + 1];
        q.row0 = first;
        q.rows = last - first < take * kGradSlice ? last - first : take * kGradSlice;
        q.i0 = (int32_t)(tile / p.tiles_n) * kGradTile;
        q.j0 = (int32_t)(tile % p.tiles_n) * kGradTile;
        return true;
    }
};

// SWIZZLE_128B descriptor of an M- or N-major operand: 64-element runs of 128
// bytes, one a row of K; 8-row groups 1024 bytes apart (SBO), the next 64
// elements of M or N one box further on (LBO).
__device__ __forceinline__ uint64_t mn_desc(uint32_t addr) {
    return (uint64_t)((addr >> 4) & 0x3FFF) | ((uint64_t)(kBox >> 4) << 16) |
           ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

// fp32 accumulator, bf16 operands, both M/N-major, M = 128.
__device__ __forceinline__ uint32_t mn_instr(int n) {
    return (1u << 4) | (1u << 7) | (1u << 10) | (1u << 15) | (1u << 16) |
           ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
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

__global__ void __launch_bounds__(kThreads, 1)
    k_grad_tc(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_g,
              const __grid_constant__ CUtensorMap map_db, const GradArgs args) {
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    unsigned char *ring = reinterpret_cast<unsigned char *>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint4 *staging = reinterpret_cast<uint4 *>(ring + kStages * kStageBytes);
    uint64_t *full = reinterpret_cast<uint64_t *>(ring + kStages * kStageBytes + kEpiWarps * 4096);
    uint64_t *empty = full + kStages;
    uint64_t *acc_full = empty + kStages;
    uint64_t *acc_empty = acc_full + 1;  // [2]: a half of the accumulators has been read
    uint64_t *mma_done = acc_empty + 2;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(mma_done + 1);
    volatile int *abort = reinterpret_cast<volatile int *>(tmem_slot + 1);

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
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
    const int64_t cta = blockIdx.x, ctas = gridDim.x;
    Walk walk(args, cta, ctas);
    Piece q;

    if (warp == kWarpLoad) {
        if (lane == 0) {
            int64_t it = 0;
            bool ok = true;
            while (ok && walk.next(args, cta, ctas, q)) {
                // boxes that lie inside the block; the others' columns are not used
                const int na = min(4, (args.d1 - q.i0 + 63) / 64), ng = min(4, (args.d2 - q.j0 + 63) / 64);
                for (int64_t k = 0; k < q.rows; k += kGradSlice, ++it) {
                    const int s = (int)(it % kStages);
                    if (it >= kStages &&
                        !(ok = mbar_wait(&empty[s], (uint32_t)((it / kStages) - 1) & 1, 1, abort)))
                        break;
                    unsigned char *stage = ring + s * kStageBytes;
                    mbar_arrive_expect_tx(&full[s], (uint32_t)(na + ng) * kBox);
                    const int32_t row = (int32_t)(q.row0 + k);
                    for (int b = 0; b < na; ++b)
                        tma_load_2d(stage + b * kBox, &map_a, &full[s], q.i0 + 64 * b, row);
                    for (int b = 0; b < ng; ++b)
                        tma_load_2d(stage + (4 + b) * kBox, &map_g, &full[s], q.j0 + 64 * b, row);
                }
            }
            // the last issued loads (at most one per stage) have landed before exit
            for (int64_t j = (it > kStages ? it - kStages : 0); j < it; ++j)
                mbar_wait(&full[j % kStages], (uint32_t)(j / kStages) & 1, 2, nullptr);
        }
    } else if (warp == kWarpMma) {
        int64_t it = 0, t = 0;
        bool ok = true;
        for (; ok && walk.next(args, cta, ctas, q); ++t) {
            const int halves = args.d1 - q.i0 > 128 ? 2 : 1;
            const int na = min(4, (args.d1 - q.i0 + 63) / 64), ng = min(4, (args.d2 - q.j0 + 63) / 64);
            const uint32_t idesc = mn_instr(min(256, (args.d2 - q.j0 + 15) / 16 * 16));
            bool waited = t == 0;  // the epilogue has read the previous tile
            for (int64_t k = 0; k < q.rows; k += kGradSlice, ++it) {
                const int s = (int)(it % kStages);
                if (!(ok = warp_wait(&full[s], (uint32_t)(it / kStages) & 1, 3, abort))) break;
                unsigned char *stage = ring + s * kStageBytes;
                const int rows = q.rows - k < kGradSlice ? (int)(q.rows - k) : kGradSlice;
                const int steps = (rows + 15) / 16;
                if (rows & 15) {
                    // 8 pieces of 16 bytes a row and box
                    const int zero = (steps * 16 - rows) * 8;
                    for (int b = 0; b < 8; ++b) {
                        if (b < 4 ? b >= na : b - 4 >= ng) continue;
                        uint4 *p = reinterpret_cast<uint4 *>(stage + b * kBox + rows * 128);
                        for (int i = lane; i < zero; i += 32) p[i] = make_uint4(0, 0, 0, 0);
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                for (int h = 0; h < halves; ++h) {
                    if (!waited && !(ok = warp_wait(&acc_empty[h], (uint32_t)(t - 1) & 1, 5, abort))) break;
                    if (!waited) asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    if (lane == 0) {
                        const uint64_t ad = mn_desc(smem_u32(stage + h * 2 * kBox));
                        const uint64_t gd = mn_desc(smem_u32(stage + 4 * kBox));
                        for (int kk = 0; kk < steps; ++kk)  // 16 rows: 2048 bytes further on
                            mma<true>(tmem + 256u * h, ad + kk * 128, gd + kk * 128, idesc,
                                      (k | kk) != 0);
                    }
                }
                if (!ok) break;
                waited = true;
                if (lane == 0) mma_commit(&empty[s]);
                __syncwarp();
            }
            // a half that this tile does not write (both, for a tile without
            // rows) takes its turn as well: acc_full moves on by one tile only
            // when every epilogue warp has seen the one before
            for (int h = waited ? halves : 0; ok && t > 0 && h < 2; ++h)
                ok = warp_wait(&acc_empty[h], (uint32_t)(t - 1) & 1, 5, abort);
            if (!ok) break;
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
        uint4 *stg = staging + (warp - kWarpEpi0) * 256;
        for (int64_t t = 0; walk.next(args, cta, ctas, q); ++t) {
            if (!warp_wait(acc_full, (uint32_t)t & 1, 4, abort)) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const int32_t i0 = q.i0 + half * 128 + quarter * 32;
            const uint32_t taddr = tmem + ((uint32_t)(quarter * 32) << 16) + 256u * half;
            const bool none = q.rows <= 0;
            if (i0 < args.d1) {
                for (int c = 0; c < 256 && q.j0 + c < args.d2; c += 64) {
                    uint32_t v[64];
                    if (none) {
#pragma unroll
                        for (int i = 0; i < 64; ++i) v[i] = 0;
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            tmem_ld16(taddr + (uint32_t)(c + 16 * i),
                                      *reinterpret_cast<uint32_t(*)[16]>(&v[16 * i]));
                        tmem_wait_ld();
                    }
                    if (q.slot >= 0) {
                        // [half][16-byte column group][row of the half]: whole lines a warp
                        uint4 *dst = reinterpret_cast<uint4 *>(args.partial + q.slot * kPartial) +
                                     (half * 64 + c / 4) * 128 + quarter * 32 + lane;
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            dst[i * 128] = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
                        continue;
                    }
                    if (lane == 0) bulk_wait_read<0>();
                    __syncwarp();
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        uint32_t o[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            __nv_bfloat162 h2 = __floats2bfloat162_rn(__uint_as_float(v[8 * j + 2 * i]),
                                                                      __uint_as_float(v[8 * j + 2 * i + 1]));
                            o[i] = *reinterpret_cast<uint32_t *>(&h2);
                        }
                        stg[lane * 8 + (j ^ (lane & 7))] = make_uint4(o[0], o[1], o[2], o[3]);
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        tma_store_3d(&map_db, stg, q.j0 + c, i0, (int32_t)q.seg);
                        bulk_commit();
                    }
                }
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&acc_empty[half]);
        }
        if (lane == 0) bulk_wait_all();
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == kWarpMma) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
    }
}

// Adds the partial tiles of the tiles that were cut: block (c, part) takes the
// tile that CTA c began and did not finish, 16 columns a thread.
__global__ void __launch_bounds__(256)
    k_grad_join(const GradArgs args, int64_t ctas, __nv_bfloat16 *__restrict__ db) {
    if (*args.mode == 0) return;
    Walk walk(args, blockIdx.x, ctas);
    Piece q, last;
    last.slot = -1;
    while (walk.next(args, blockIdx.x, ctas, q)) last = q;
    if (last.slot < 0 || !last.lead) return;
    // the CTAs that hold the rest: up to the one that ends with the segment's rows
    const int64_t seg_end = args.off[last.seg + 1];
    int64_t row = last.row0 + last.rows, more = blockIdx.x;
    while (row < seg_end && more + 1 < ctas) {
        Walk other(args, ++more, ctas);
        if (other.next(args, more, ctas, q)) row = q.row0 + q.rows;
    }
    const int idx = blockIdx.y * 256 + threadIdx.x;  // half, 16 groups of 16 columns, 128 rows
    const int line = idx & 127, group = (idx >> 7) & 15, half = idx >> 11;
    const int32_t i = last.i0 + half * 128 + line, j = last.j0 + group * 16;
    if (i >= args.d1 || j >= args.d2) return;
    float4 sum[4];
    for (int64_t c = blockIdx.x; c <= more; ++c) {
        const Walk other(args, c, ctas);
        if (other.at >= other.end) continue;  // a CTA without units
        const int64_t slot = c == blockIdx.x ? last.slot : 2 * c;
        const float4 *src = reinterpret_cast<const float4 *>(args.partial + slot * kPartial) +
                            (half * 64 + group * 4) * 128 + line;
#pragma unroll
        for (int v = 0; v < 4; ++v) {
            const float4 x = src[v * 128];
            if (c == blockIdx.x) {
                sum[v] = x;
            } else {
                sum[v].x += x.x;
                sum[v].y += x.y;
                sum[v].z += x.z;
                sum[v].w += x.w;
            }
        }
    }
    __nv_bfloat16 *dst = db + (last.seg * args.d1 + i) * (int64_t)args.d2 + j;
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

// TMA wants 16-byte aligned bases and row strides.
bool gmm_grad_tc_supported(const void *grad, const void *a, const void *db, int64_t n, int64_t d1,
                           int64_t r, int64_t d2, int dtype) {
    return dtype == BGL_BF16 && n > 0 && d1 > 0 && d2 > 0 && d1 % 8 == 0 && d2 % 8 == 0 &&
           d1 * d2 < (int64_t(1) << 39) && aligned(grad, 16) && aligned(a, 16) && aligned(db, 16);
}

GradTiles gmm_grad_tiles(int64_t n, int64_t d1, int64_t r, int64_t d2) {
    GradTiles t;
    t.tiles_n = (d2 + kGradTile - 1) / kGradTile;
    t.per_segment = t.tiles_n * ((d1 + kGradTile - 1) / kGradTile);
    // no more CTAs than there can be units
    const int64_t units = t.per_segment * (n / kGradSlice + r);
    t.ctas = (int)(units < num_sms() ? (units > 0 ? units : 1) : num_sms());
    return t;
}

int gmm_grad_tensor_core(const void *grad, const void *a, void *db, const GradLayout &l,
                         const GradTiles &t, int64_t n, int64_t d1, int64_t r, int64_t d2,
                         cudaStream_t s) {
    CUtensorMap map_a, map_g, map_db;
    const int64_t dims_a[2] = {d1, n}, dims_g[2] = {d2, n}, dims_db[3] = {d2, d1, r};
    int rc = bf16_map(&map_a, a, 2, dims_a, kGradSlice);
    if (!rc) rc = bf16_map(&map_g, grad, 2, dims_g, kGradSlice);
    if (!rc) rc = bf16_map(&map_db, db, 3, dims_db, 32);
    if (rc) return rc;
    GradArgs args;
    args.off = l.off;
    args.unit_off = l.unit_off;
    args.mode = l.mode;
    args.partial = l.partial;
    args.r = r;
    args.per_segment = t.per_segment;
    args.tiles_n = (int32_t)t.tiles_n;
    args.d1 = (int32_t)d1;
    args.d2 = (int32_t)d2;
    BGL_CUDA(cudaFuncSetAttribute(k_grad_tc, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmem));
    k_grad_tc<<<t.ctas, kThreads, kSmem, s>>>(map_a, map_g, map_db, args);
    BGL_LAUNCH_CHECK();
    k_grad_join<<<dim3((unsigned)t.ctas, 16), 256, 0, s>>>(args, t.ctas, (__nv_bfloat16 *)db);
    BGL_LAUNCH_CHECK();
    return BGL_OK;
}

cudaError_t gmm_grad_tc_error(int *code) { return take_tc_error(code); }

}  // namespace bgl
