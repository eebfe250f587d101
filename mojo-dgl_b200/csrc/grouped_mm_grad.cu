// Gradients of segment_mm, the grouped product out[i] = a[i] @ b[r(i)] over
// consecutive segments of rows:
//
//   da[i] = dout[i] @ b[r(i)]^T        db[r] = a[rows of r]^T @ dout[rows of r]
//
// Rows past the last segment have da = 0; a segment without rows has db = 0.
#include "after.cuh"
#include "grouped_mm.cuh"
#include "rows.cuh"

namespace bgl {
namespace {

constexpr int kDepth = 16;  // terms of a strip of the SIMT products

// Three sums over the block's earlier threads (exclusive), and over all of them.
struct Three {
    int64_t a, b, c;
};
__device__ __forceinline__ Three operator+(Three x, Three y) { return {x.a + y.a, x.b + y.b, x.c + y.c}; }
__device__ __forceinline__ Three operator-(Three x, Three y) { return {x.a - y.a, x.b - y.b, x.c - y.c}; }
__device__ __forceinline__ Three shfl_up(Three x, int o) {
    return {__shfl_up_sync(0xffffffffu, x.a, o), __shfl_up_sync(0xffffffffu, x.b, o), __shfl_up_sync(0xffffffffu, x.c, o)};
}
__device__ __forceinline__ Three block_scan(Three v, Three *warps, Three &total) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n = blockDim.x >> 5;
    Three sum = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const Three up = shfl_up(sum, o);
        if (lane >= o) sum = sum + up;
    }
    if (lane == 31) warps[warp] = sum;
    __syncthreads();
    if (warp == 0) {
        Three w = lane < n ? warps[lane] : Three{0, 0, 0};
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const Three up = shfl_up(w, o);
            if (lane >= o) w = w + up;
        }
        warps[lane] = w;
    }
    __syncthreads();
    total = warps[n - 1];
    const Three before = (warp ? warps[warp - 1] : Three{0, 0, 0}) + sum - v;
    __syncthreads();
    return before;
}

// First row and first 512-row tile of each segment, and db's items; one block.
// The rows are clamped as segment_mm's own schedule clamps them: negative
// lengths count as 0 and no segment runs past n.
//
// Items are taken by whichever pair of CTAs is free, db's first and its long segments
// first, da's small tiles last, so the pairs end together.  A db tile is cut
// into pieces where its sum is longer than a pair's share of all work, or three
// quarters of it where no tiles of da fill in behind; that also bounds the partial
// tiles (a sum of L slices cut into pieces of P has ceil(L / P) < 2 L / P of them
// where L > P, all sums together 2 * work / P < 3 a pair).  A tile's read-out counts
// as kTileCost slices.  Measured with pieces up to half, three quarters and the whole
// of the share: 500000 x 256 x 256 over 64 segments 224, 222, 210 us; 300000 x 256 x
// 128 over 5: 204, 160, 144; db alone, 500000 x 256 x 256: 142, 132, 149, and 32768 x
// 2048 x 1024 over 16 uneven ones: 189, 152, 148.
__global__ void __launch_bounds__(1024)
    k_grad_schedule(const int64_t *__restrict__ seglen, int64_t r, int64_t n, GradTiles t,
                    int64_t slices2, bool want_da, bool want_db, GradLayout l) {
    constexpr int64_t kTileCost = 2;
    constexpr int kSorted = 256;  // more segments than this stay in order
    __shared__ Three warps[32];
    __shared__ int64_t lens[kSorted];
    next_may_start();
    int64_t rows = 0, tiles = 0, slices = 0;
    for (int64_t i0 = 0; i0 < r; i0 += blockDim.x) {
        const int64_t i = i0 + threadIdx.x;
        int64_t len = i < r ? seglen[i] : 0;
        len = len < 0 ? 0 : len < n ? len : n;
        // (the tiles are those of the rows that there are: where lengths add up
        // to more than n, which no caller of a matching product gives, a second
        // scan counts them)
        Three total;
        Three before = block_scan({len, (len + kGradRows - 1) / kGradRows, 0}, warps, total);
        int64_t first = rows + before.a, end = first + len;
        if (rows + total.a > n) {
            first = first < n ? first : n;
            end = end < n ? end : n;
            Three clamped;
            before.b = block_scan({0, (end - first + kGradRows - 1) / kGradRows, 0}, warps, clamped).b;
            total.b = clamped.b;
        }
        int64_t mine = (end - first + kGradSlice - 1) / kGradSlice;
        if (i < r && mine == 0) mine = 1;  // a segment without rows: one piece a tile writes zeros
        if (i < r) {
            l.off[i] = first;
            l.row_off[i] = tiles + before.b;
            if (r <= kSorted) lens[i] = mine;
        }
        slices += mine;
        rows += total.a;
        tiles += total.b;
    }
    if (threadIdx.x == 0) {
        l.off[r] = rows < n ? rows : n;
        l.row_off[r] = tiles;
    }
    if (!want_da && !want_db) return;
    {
        Three total;
        block_scan({slices, 0, 0}, warps, total);
        slices = total.a;
    }
    for (int64_t i = threadIdx.x; i < r; i += blockDim.x) {
        int64_t at = i;
        if (r <= kSorted) {
            at = 0;
            for (int j = 0; j < (int)r; ++j) at += lens[j] > lens[i] || (lens[j] == lens[i] && j < i);
        }
        l.order[at] = (int32_t)i;
    }
    __syncthreads();
    const int64_t per_segment = t.tiles1 * t.tiles2;
    const int64_t da_items = want_da ? tiles * t.cols : 0;
    const int64_t da_work = da_items * (slices2 + kTileCost);
    const int64_t db_work = slices * per_segment;
    const int64_t quarters = (want_da ? 4 : 3) * (da_work + db_work);
    int64_t piece = (quarters + 4 * t.pairs - 1) / (4 * t.pairs);
    if (piece < kGradShortest) piece = kGradShortest;
    int64_t items = 0, cut = 0, slots = 0;
    for (int64_t k0 = 0; want_db && k0 < r; k0 += blockDim.x) {
        const int64_t k = k0 + threadIdx.x;
        int64_t pieces = 0;
        if (k < r) {
            const int32_t seg = l.order[k];
            const int64_t len = l.off[seg + 1] - l.off[seg];
            pieces = grad_pieces(len, piece).count;
        }
        const bool several = pieces > 1;
        Three total;
        const Three before = block_scan({pieces * per_segment, several ? per_segment : 0,
                                         several ? pieces * per_segment : 0}, warps, total);
        if (k < r) {
            l.item_off[k] = items + before.a;
            l.cut_off[k] = cut + before.b;
            l.slot_off[k] = slots + before.c;
        }
        items += total.a;
        cut += total.b;
        slots += total.c;
    }
    if (threadIdx.x == 0) {
        l.item_off[r] = items;
        l.cut_off[r] = cut;
        l.slot_off[r] = slots;
        l.head[kHeadItems] = items + da_items;
        l.head[kHeadDbItems] = items;
        l.head[kHeadPiece] = piece;
        l.head[kHeadCut] = cut;
        l.head[kHeadNext] = t.pairs;  // the first items are the pairs' own numbers
    }
}

// SIMT products, exact sums: float32 and float64, and bf16 rows that are no whole
// 16-byte pieces.  A block of 256 threads takes a square tile of outputs, 8 x 8 a
// thread (float64: 4 x 4), over strips of kDepth terms in two shared buffers: the
// next strip is under way to registers while this one is multiplied.  32768 x 2048
// x 1024 float32 over 16 segments: 7.3 ms for both gradients, of 3.8 ms that the
// FMA pipes need (12.6 ms with 4 x 4 a thread and one buffer).  A sum over a segment's
// rows is not cut here: where few segments of narrow blocks leave few tiles, db takes as
// long as a block walks its rows (1000000 rows, float32, one segment of 64 x 64: 113 ms on
// one block, five segments: 23 ms; bf16 of 60 x 60: 312 ms; bf16 of 64 x 64, on the tensor
// cores, 0.19 ms).
template <typename T>
struct Simt {
    using A = Acc<T>;
    static constexpr int kMicro = sizeof(A) == 4 ? 8 : 4, kTile = 16 * kMicro, kHalf = kTile / 2;
    static constexpr int kEach = kTile * kDepth / 256;  // values of an operand's strip a thread brings
    using Strip = A[kDepth][kTile + 4];
    A acc[kMicro][kMicro];

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < kMicro; ++i)
#pragma unroll
            for (int j = 0; j < kMicro; ++j) acc[i][j] = 0;
    }
    // thread row i of the tile: the first half of them in the tile's first half
    static __device__ __forceinline__ int place(int thread, int i) {
        return i < kMicro / 2 ? thread * (kMicro / 2) + i : kHalf + thread * (kMicro / 2) + i - kMicro / 2;
    }
    __device__ __forceinline__ void step(const Strip &left, const Strip &right) {
        const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
#pragma unroll
        for (int k = 0; k < kDepth; ++k) {
            A u[kMicro], v[kMicro];
#pragma unroll
            for (int i = 0; i < kMicro; ++i) u[i] = left[k][place(ty, i)], v[i] = right[k][place(tx, i)];
#pragma unroll
            for (int i = 0; i < kMicro; ++i)
#pragma unroll
                for (int j = 0; j < kMicro; ++j) acc[i][j] += u[i] * v[j];
        }
    }
    // A strip of rows that are contiguous along the sum: values [row + m][k + ..],
    // rows [first, end) of the array, zero elsewhere.
    static __device__ __forceinline__ void fetch_along(A (&to)[kEach], const T *from, int64_t first, int64_t end,
                                                       int64_t row, int64_t width, int64_t k0) {
        const int k = threadIdx.x % kDepth;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int64_t at = row + threadIdx.x / kDepth + i * (256 / kDepth);
            to[i] = at >= first && at < end && k0 + k < width ? to_acc(from[at * width + k0 + k]) : A(0);
        }
    }
    static __device__ __forceinline__ void put_along(const A (&from)[kEach], Strip &to) {
#pragma unroll
        for (int i = 0; i < kEach; ++i) to[threadIdx.x % kDepth][threadIdx.x / kDepth + i * (256 / kDepth)] = from[i];
    }
    // A strip of rows that are the sum's terms: values [k + ..][col + m].
    static __device__ __forceinline__ void fetch_across(A (&to)[kEach], const T *from, int64_t k0, int64_t end,
                                                        int64_t width, int64_t col) {
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int at = threadIdx.x + i * 256;
            const int64_t k = k0 + at / kTile, c = col + at % kTile;
            to[i] = k < end && c < width ? to_acc(from[k * width + c]) : A(0);
        }
    }
    static __device__ __forceinline__ void put_across(const A (&from)[kEach], Strip &to) {
#pragma unroll
        for (int i = 0; i < kEach; ++i) to[(threadIdx.x + i * 256) / kTile][(threadIdx.x + i * 256) % kTile] = from[i];
    }
};

// da: a block takes a tile of rows by columns; the rows may span segments, which
// it walks one after the other.
template <typename T>
__global__ void __launch_bounds__(256)
    k_segment_mm_da(const T *__restrict__ g, const T *__restrict__ b,
                    const int64_t *__restrict__ off, int64_t n, int64_t d1, int64_t r, int64_t d2,
                    T *__restrict__ da) {
    using S = Simt<T>;
    using A = Acc<T>;
    __shared__ typename S::Strip left[2], right[2];
    S tile;
    tile.clear();
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const int64_t row0 = (int64_t)blockIdx.x * S::kTile, col0 = (int64_t)blockIdx.y * S::kTile;
    const int64_t row_end = row0 + S::kTile < n ? row0 + S::kTile : n;
    int64_t lo = 0, hi = r;  // first segment that ends after row0
    while (lo < hi) {
        const int64_t mid = (lo + hi) >> 1;
        if (off[mid + 1] > row0) hi = mid; else lo = mid + 1;
    }
    for (int64_t seg = lo; seg < r && off[seg] < row_end; ++seg) {
        const int64_t s0 = off[seg], s1 = off[seg + 1] < row_end ? off[seg + 1] : row_end;
        if (s0 >= s1) continue;
        A u[S::kEach], v[S::kEach];
        int buffer = 0;
        auto fetch = [&](int64_t k0) {
            S::fetch_along(u, g, s0, s1, row0, d2, k0);
            S::fetch_along(v, b + seg * d1 * d2, 0, d1, col0, d2, k0);
        };
        fetch(0);
        for (int64_t k0 = 0; k0 < d2; k0 += kDepth) {
            S::put_along(u, left[buffer]);
            S::put_along(v, right[buffer]);
            __syncthreads();
            if (k0 + kDepth < d2) fetch(k0 + kDepth);
            tile.step(left[buffer], right[buffer]);
            buffer ^= 1;
        }
        __syncthreads();
        // the rows of this segment are complete: rows of others keep zeros
        // in `left`, and inf or NaN in b must not reach them
#pragma unroll
        for (int i = 0; i < S::kMicro; ++i) {
            const int64_t row = row0 + S::place(ty, i);
#pragma unroll
            for (int j = 0; j < S::kMicro; ++j) {
                const int64_t col = col0 + S::place(tx, j);
                if (row >= s0 && row < s1 && col < d1) da[row * d1 + col] = from_acc<T>(tile.acc[i][j]);
            }
        }
        tile.clear();
    }
    const int64_t covered = off[r];
#pragma unroll
    for (int i = 0; i < S::kMicro; ++i) {
        const int64_t row = row0 + S::place(ty, i);
#pragma unroll
        for (int j = 0; j < S::kMicro; ++j) {
            const int64_t col = col0 + S::place(tx, j);
            if (row >= covered && row < row_end && col < d1) da[row * d1 + col] = from_acc<T>(0);
        }
    }
}

// db: a block takes a tile of one segment's product and walks the segment's rows
// in order.
template <typename T>
__global__ void __launch_bounds__(256)
    k_segment_mm_db(const T *__restrict__ g, const T *__restrict__ a,
                    const int64_t *__restrict__ off, int64_t d1, int64_t r, int64_t d2,
                    T *__restrict__ db) {
    using S = Simt<T>;
    using A = Acc<T>;
    __shared__ typename S::Strip left[2], right[2];
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const int64_t tiles2 = (d2 + S::kTile - 1) / S::kTile;
    const int64_t i0 = (int64_t)blockIdx.x / tiles2 * S::kTile, j0 = (int64_t)blockIdx.x % tiles2 * S::kTile;
    for (int64_t seg = blockIdx.y; seg < r; seg += gridDim.y) {
        const int64_t s0 = off[seg], s1 = off[seg + 1];
        S tile;
        tile.clear();
        A u[S::kEach], v[S::kEach];
        int buffer = 0;
        auto fetch = [&](int64_t k0) {
            S::fetch_across(u, a, k0, s1, d1, i0);
            S::fetch_across(v, g, k0, s1, d2, j0);
        };
        if (s0 < s1) fetch(s0);
        for (int64_t k0 = s0; k0 < s1; k0 += kDepth) {
            S::put_across(u, left[buffer]);
            S::put_across(v, right[buffer]);
            __syncthreads();
            if (k0 + kDepth < s1) fetch(k0 + kDepth);
            tile.step(left[buffer], right[buffer]);
            buffer ^= 1;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < S::kMicro; ++i)
#pragma unroll
            for (int j = 0; j < S::kMicro; ++j) {
                const int64_t row = i0 + S::place(ty, i), col = j0 + S::place(tx, j);
                if (row < d1 && col < d2) db[(seg * d1 + row) * d2 + col] = from_acc<T>(tile.acc[i][j]);
            }
    }
}

template <typename T>
int simt(const void *g, const void *a, const void *b, const int64_t *off, int64_t n, int64_t d1,
         int64_t r, int64_t d2, void *da, void *db, cudaStream_t s) {
    constexpr int kTile = Simt<T>::kTile;
    if (da && n && d1) {
        dim3 grid((unsigned)((n + kTile - 1) / kTile), (unsigned)((d1 + kTile - 1) / kTile));
        k_segment_mm_da<T><<<grid, 256, 0, s>>>((const T *)g, (const T *)b, off, n, d1, r, d2, (T *)da);
        BGL_LAUNCH_CHECK();
    }
    if (db && r && d1 && d2) {
        const int64_t tiles = ((d1 + kTile - 1) / kTile) * ((d2 + kTile - 1) / kTile);
        dim3 grid((unsigned)tiles, (unsigned)(r < 65535 ? r : 65535));
        k_segment_mm_db<T><<<grid, 256, 0, s>>>((const T *)g, (const T *)a, off, d1, r, d2, (T *)db);
        BGL_LAUNCH_CHECK();
    }
    return BGL_OK;
}

GradLayout grad_layout(void *ws, int64_t n, int64_t d1, int64_t r, int64_t d2, int dtype) {
    const GradTiles t = gmm_grad_tiles(n, d1, r, d2);
    Carver c(ws);
    GradLayout l;
    l.off = c.take<int64_t>((size_t)r + 1);
    l.row_off = c.take<int64_t>((size_t)r + 1);
    l.order = c.take<int32_t>((size_t)r);
    l.item_off = c.take<int64_t>((size_t)r + 1);
    l.cut_off = c.take<int64_t>((size_t)r + 1);
    l.slot_off = c.take<int64_t>((size_t)r + 1);
    l.head = c.take<int64_t>(kHead);
    l.partial = nullptr;
    if (dtype == BGL_BF16 && n > kGradShortest * kGradSlice) {
        // no sum of kGradShortest slices is cut; a longer one of L has at most
        // ceil(L / kGradShortest) <= 2 (L - 1) / kGradShortest pieces
        int64_t slots = (int64_t)t.pairs * kGradSlots;
        const int64_t most = t.tiles1 * t.tiles2 * 2 * (n / kGradSlice) / kGradShortest;
        l.partial = c.take<float>((size_t)(slots < most ? slots : most) * kGradRows * kGradCols);
    }
    l.bytes = c.used + 256;
    return l;
}

}  // namespace
}  // namespace bgl

using namespace bgl;

extern "C" {

size_t bgl_segment_mm_backward_workspace_size(int64_t n, int64_t d1, int64_t r, int64_t d2,
                                              int dtype) {
    if (n < 0 || r < 0 || d1 < 0 || d2 < 0) return 0;
    return grad_layout(nullptr, n, d1, r, d2, dtype).bytes;
}

int bgl_segment_mm_backward(const void *grad, const void *a, const void *b, const int64_t *seglen,
                            int64_t n, int64_t d1, int64_t r, int64_t d2, void *da, void *db,
                            int dtype, void *workspace, size_t workspace_bytes, void *stream) {
    const char *who = "bgl_segment_mm_backward";
    if (!row_dtype(dtype)) return fail(BGL_E_UNSUPPORTED, "%s: dtype %d", who, dtype);
    if (n < 0 || d1 < 0 || r < 0 || d2 < 0) return fail(BGL_E_INVALID, "%s: negative size", who);
    if (n >= (int64_t(1) << 31) || r >= (int64_t(1) << 31) || d1 >= (1 << 21) || d2 >= (1 << 21))
        return fail(BGL_E_UNSUPPORTED, "%s: n or r >= 2^31 or a width >= 2^21", who);
    if (!da && !db) return BGL_OK;
    if (r && !seglen) return fail(BGL_E_INVALID, "%s: null seglen", who);
    if (da && n && d1 && d2 && (!grad || (r && !b))) return fail(BGL_E_INVALID, "%s: null buffer", who);
    if (db && n && r && d1 && d2 && (!grad || !a)) return fail(BGL_E_INVALID, "%s: null buffer", who);
    GradLayout l = grad_layout(workspace, n, d1, r, d2, dtype);
    if (!workspace || workspace_bytes < l.bytes)
        return fail(BGL_E_WORKSPACE, "%s: workspace too small", who);
    cudaStream_t s = as_stream(stream);
    const bool want_da = da && n && d1, want_db = db && r && d1 && d2;
    const GradTiles t = gmm_grad_tiles(n, d1, r, d2);
    const bool tc = r && gmm_grad_tc_supported(grad, a, b, want_da ? da : nullptr,
                                               want_db ? db : nullptr, n, d1, r, d2, dtype);
    const unsigned threads = r < 1024 ? (unsigned)(r + 31) / 32 * 32 : 1024;
    k_grad_schedule<<<1, threads ? threads : 32, 0, s>>>(seglen, r, n, t, (d2 + kGradSlice - 1) / kGradSlice,
                                       tc && want_da, tc && want_db, l);
    BGL_LAUNCH_CHECK();
    if (!want_da) da = nullptr;
    if (!want_db) db = nullptr;
    if (tc) return gmm_grad_tensor_core(grad, a, b, da, db, l, t, n, d1, r, d2, s);
    if (dtype == BGL_F64) return simt<double>(grad, a, b, l.off, n, d1, r, d2, da, db, s);
    if (dtype == BGL_F32) return simt<float>(grad, a, b, l.off, n, d1, r, d2, da, db, s);
    return simt<__nv_bfloat16>(grad, a, b, l.off, n, d1, r, d2, da, db, s);
}

}  // extern "C"
