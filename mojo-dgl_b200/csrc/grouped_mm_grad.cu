// Gradients of segment_mm, the grouped product out[i] = a[i] @ b[r(i)] over
// consecutive segments of rows:
//
//   da[i] = dout[i] @ b[r(i)]^T        db[r] = a[rows of r]^T @ dout[rows of r]
//
// Rows past the last segment have da = 0; a segment without rows has db = 0.
#include "rows.cuh"

namespace bgl {
namespace {

constexpr int kTile = 64, kDepth = 16;

// First row of each segment, clamped as segment_mm's own schedule clamps:
// negative lengths count as 0 and no segment runs past n.
__global__ void k_segment_offsets(const int64_t *__restrict__ seglen, int64_t r, int64_t n,
                                  int64_t *__restrict__ off) {
    if (blockIdx.x != 0 || threadIdx.x != 0) return;
    int64_t row = 0;
    off[0] = 0;
    for (int64_t i = 0; i < r; ++i) {
        int64_t len = seglen[i] < 0 ? 0 : seglen[i];
        row += len < n - row ? len : n - row;
        off[i + 1] = row;
    }
}

// 64 x 64 outputs a block of 256 threads, 4 x 4 a thread, over a shared strip
// of kDepth terms: s_left[k][i] * s_right[k][j].
template <typename A>
__device__ __forceinline__ void tile_step(const A (*left)[kTile + 1], const A (*right)[kTile + 1],
                                          A (&acc)[4][4]) {
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
#pragma unroll
    for (int k = 0; k < kDepth; ++k) {
        A u[4], v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = left[k][ty * 4 + i];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = right[k][tx * 4 + j];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] += u[i] * v[j];
    }
}

// da: a block takes 64 rows by 64 columns; the rows may span segments, which
// it walks one after the other.
template <typename T>
__global__ void __launch_bounds__(256)
    k_segment_mm_da(const T *__restrict__ g, const T *__restrict__ b,
                    const int64_t *__restrict__ off, int64_t n, int64_t d1, int64_t r, int64_t d2,
                    T *__restrict__ da) {
    using A = Acc<T>;
    __shared__ A left[kDepth][kTile + 1], right[kDepth][kTile + 1];
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const int64_t row0 = (int64_t)blockIdx.x * kTile, col0 = (int64_t)blockIdx.y * kTile;
    const int64_t row_end = row0 + kTile < n ? row0 + kTile : n;
    int64_t lo = 0, hi = r;  // first segment that ends after row0
    while (lo < hi) {
        const int64_t mid = (lo + hi) >> 1;
        if (off[mid + 1] > row0) hi = mid; else lo = mid + 1;
    }
    A acc[4][4] = {};
    for (int64_t seg = lo; seg < r && off[seg] < row_end; ++seg) {
        const int64_t s0 = off[seg], s1 = off[seg + 1];
        if (s0 == s1) continue;
        for (int64_t k0 = 0; k0 < d2; k0 += kDepth) {
            for (int i = threadIdx.x; i < kTile * kDepth; i += 256) {
                const int k = i % kDepth, m = i / kDepth;
                const int64_t row = row0 + m, col = col0 + m;
                left[k][m] = row >= s0 && row < s1 && row < row_end && k0 + k < d2
                                 ? to_acc(g[row * d2 + k0 + k]) : A(0);
                right[k][m] = col < d1 && k0 + k < d2
                                  ? to_acc(b[(seg * d1 + col) * d2 + k0 + k]) : A(0);
            }
            __syncthreads();
            tile_step<A>(left, right, acc);
            __syncthreads();
        }
        // the rows of this segment are complete: rows of others keep zeros
        // in `left`, and inf or NaN in b must not reach them
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t row = row0 + ty * 4 + i;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int64_t col = col0 + tx * 4 + j;
                if (row >= s0 && row < s1 && row < row_end && col < d1)
                    da[row * d1 + col] = from_acc<T>(acc[i][j]);
                acc[i][j] = 0;
            }
        }
    }
    const int64_t covered = off[r];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t row = row0 + ty * 4 + i;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t col = col0 + tx * 4 + j;
            if (row >= covered && row < row_end && col < d1) da[row * d1 + col] = from_acc<T>(0);
        }
    }
}

// db: a block takes a 64 x 64 tile of one segment's product and walks the
// segment's rows in order.
template <typename T>
__global__ void __launch_bounds__(256)
    k_segment_mm_db(const T *__restrict__ g, const T *__restrict__ a,
                    const int64_t *__restrict__ off, int64_t d1, int64_t r, int64_t d2,
                    T *__restrict__ db) {
    using A = Acc<T>;
    __shared__ A left[kDepth][kTile + 1], right[kDepth][kTile + 1];
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const int64_t tiles2 = (d2 + kTile - 1) / kTile;
    const int64_t i0 = (int64_t)blockIdx.x / tiles2 * kTile, j0 = (int64_t)blockIdx.x % tiles2 * kTile;
    for (int64_t seg = blockIdx.y; seg < r; seg += gridDim.y) {
        const int64_t s0 = off[seg], s1 = off[seg + 1];
        A acc[4][4] = {};
        for (int64_t k0 = s0; k0 < s1; k0 += kDepth) {
            for (int i = threadIdx.x; i < kTile * kDepth; i += 256) {
                const int m = i % kTile, k = i / kTile;
                const int64_t row = k0 + k;
                left[k][m] = row < s1 && i0 + m < d1 ? to_acc(a[row * d1 + i0 + m]) : A(0);
                right[k][m] = row < s1 && j0 + m < d2 ? to_acc(g[row * d2 + j0 + m]) : A(0);
            }
            __syncthreads();
            tile_step<A>(left, right, acc);
            __syncthreads();
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int64_t row = i0 + ty * 4 + i, col = j0 + tx * 4 + j;
                if (row < d1 && col < d2) db[(seg * d1 + row) * d2 + col] = from_acc<T>(acc[i][j]);
            }
    }
}

template <typename T>
int simt(const void *g, const void *a, const void *b, const int64_t *off, int64_t n, int64_t d1,
         int64_t r, int64_t d2, void *da, void *db, cudaStream_t s) {
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

}  // namespace
}  // namespace bgl

using namespace bgl;

extern "C" {

size_t bgl_segment_mm_backward_workspace_size(int64_t n, int64_t d1, int64_t r, int64_t d2,
                                              int dtype) {
    if (n < 0 || r < 0 || d1 < 0 || d2 < 0) return 0;
    return (size_t)(r + 1) * sizeof(int64_t) + 256;
}

int bgl_segment_mm_backward(const void *grad, const void *a, const void *b, const int64_t *seglen,
                            int64_t n, int64_t d1, int64_t r, int64_t d2, void *da, void *db,
                            int dtype, void *workspace, size_t workspace_bytes, void *stream) {
    const char *who = "bgl_segment_mm_backward";
    if (!row_dtype(dtype)) return fail(BGL_E_UNSUPPORTED, "%s: dtype %d", who, dtype);
    if (n < 0 || d1 < 0 || r < 0 || d2 < 0) return fail(BGL_E_INVALID, "%s: negative size", who);
    if (n >= (int64_t(1) << 31) || d1 >= (1 << 22) || d2 >= (1 << 22))
        return fail(BGL_E_UNSUPPORTED, "%s: n >= 2^31 or a width >= 2^22", who);
    if (!da && !db) return BGL_OK;
    if (r && !seglen) return fail(BGL_E_INVALID, "%s: null seglen", who);
    if (da && n && d1 && d2 && (!grad || (r && !b))) return fail(BGL_E_INVALID, "%s: null buffer", who);
    if (db && n && r && d1 && d2 && (!grad || !a)) return fail(BGL_E_INVALID, "%s: null buffer", who);
    if (!workspace || workspace_bytes < bgl_segment_mm_backward_workspace_size(n, d1, r, d2, dtype))
        return fail(BGL_E_WORKSPACE, "%s: workspace too small", who);
    cudaStream_t s = as_stream(stream);
    Carver c(workspace);
    int64_t *off = c.take<int64_t>((size_t)r + 1);
    k_segment_offsets<<<1, 32, 0, s>>>(seglen, r, n, off);
    BGL_LAUNCH_CHECK();
    if (dtype == BGL_F64) return simt<double>(grad, a, b, off, n, d1, r, d2, da, db, s);
    if (dtype == BGL_F32) return simt<float>(grad, a, b, off, n, d1, r, d2, da, db, s);
    return simt<__nv_bfloat16>(grad, a, b, off, n, d1, r, d2, da, db, s);
}

}  // extern "C"
