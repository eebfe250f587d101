// Layer norm over the last axis of a (rows, d) array, forward and backward.
//
//   y  = (x - mean) * rstd * w + b,    rstd = 1 / sqrt(mean((x - mean)^2) + eps)
//   v  = dy * w,  xhat = (x - mean) * rstd
//   dx = rstd * (v - mean(v) - xhat * mean(v * xhat))
//   dw = sum over rows of dy * xhat,   db = sum over rows of dy
//
// One block a row; the sums over rows for dw and db go through per-split
// partial rows that a second kernel adds in order, so results do not depend
// on the order in which blocks run.
#include "rows.cuh"

namespace bgl {
namespace {

constexpr int kSplitRows = 256;  // rows of one partial sum of dw and db, at least
constexpr int kMaxSplits = 256;

template <typename T, typename W>
__global__ void __launch_bounds__(256)
    k_layer_norm(const T *__restrict__ x, const W *__restrict__ w, const W *__restrict__ b,
                 int64_t rows, int64_t d, Acc<T> eps, T *__restrict__ y, Acc<T> *__restrict__ mean,
                 Acc<T> *__restrict__ rstd) {
    using A = Acc<T>;
    __shared__ A smem[32];
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const T *xr = x + row * d;
        A s = 0;
        for (int64_t i = threadIdx.x; i < d; i += blockDim.x) s += to_acc(xr[i]);
        const A mu = block_sum(s, smem) / A(d);
        s = 0;
        for (int64_t i = threadIdx.x; i < d; i += blockDim.x) {
            const A c = to_acc(xr[i]) - mu;
            s += c * c;
        }
        const A rs = A(1) / sqrt(block_sum(s, smem) / A(d) + eps);
        for (int64_t i = threadIdx.x; i < d; i += blockDim.x) {
            A v = (to_acc(xr[i]) - mu) * rs;
            if (w) v *= to_acc(w[i]);
            if (b) v += to_acc(b[i]);
            y[row * d + i] = from_acc<T>(v);
        }
        if (threadIdx.x == 0) {
            if (mean) mean[row] = mu;
            if (rstd) rstd[row] = rs;
        }
    }
}

template <typename T, typename W>
__global__ void __launch_bounds__(256)
    k_layer_norm_dx(const T *__restrict__ dy, const T *__restrict__ x,
                    const Acc<T> *__restrict__ mean, const Acc<T> *__restrict__ rstd,
                    const W *__restrict__ w, int64_t rows, int64_t d, T *__restrict__ dx) {
    using A = Acc<T>;
    __shared__ A smem[32];
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const A mu = mean[row], rs = rstd[row];
        A s1 = 0, s2 = 0;
        for (int64_t i = threadIdx.x; i < d; i += blockDim.x) {
            A v = to_acc(dy[row * d + i]);
            if (w) v *= to_acc(w[i]);
            s1 += v;
            s2 += v * ((to_acc(x[row * d + i]) - mu) * rs);
        }
        s1 = block_sum(s1, smem) / A(d);
        s2 = block_sum(s2, smem) / A(d);
        for (int64_t i = threadIdx.x; i < d; i += blockDim.x) {
            A v = to_acc(dy[row * d + i]);
            if (w) v *= to_acc(w[i]);
            dx[row * d + i] = from_acc<T>(rs * (v - s1 - ((to_acc(x[row * d + i]) - mu) * rs) * s2));
        }
    }
}

// partial[split][0][i] = sum of dy * xhat, partial[split][1][i] = sum of dy over the split's rows
template <typename T>
__global__ void __launch_bounds__(256)
    k_layer_norm_dw(const T *__restrict__ dy, const T *__restrict__ x,
                    const Acc<T> *__restrict__ mean, const Acc<T> *__restrict__ rstd, int64_t rows,
                    int64_t d, int64_t split_rows, Acc<T> *__restrict__ partial) {
    using A = Acc<T>;
    __shared__ A sw[8][33], sb[8][33];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const int64_t col = (int64_t)blockIdx.x * 32 + tx;
    const int64_t r0 = (int64_t)blockIdx.y * split_rows;
    const int64_t r1 = r0 + split_rows < rows ? r0 + split_rows : rows;
    A aw = 0, ab = 0;
    if (col < d)
        for (int64_t row = r0 + ty; row < r1; row += 8) {
            const A g = to_acc(dy[row * d + col]);
            ab += g;
            aw += g * ((to_acc(x[row * d + col]) - mean[row]) * rstd[row]);
        }
    sw[ty][tx] = aw;
    sb[ty][tx] = ab;
    __syncthreads();
    if (ty == 0 && col < d) {
        for (int i = 1; i < 8; ++i) {
            aw += sw[i][tx];
            ab += sb[i][tx];
        }
        partial[((int64_t)blockIdx.y * 2) * d + col] = aw;
        partial[((int64_t)blockIdx.y * 2 + 1) * d + col] = ab;
    }
}

template <typename A, typename W>
__global__ void __launch_bounds__(256)
    k_layer_norm_dw_join(const A *__restrict__ partial, int64_t splits, int64_t d,
                         W *__restrict__ dw, W *__restrict__ db) {
    for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < d;
         i += (int64_t)gridDim.x * blockDim.x) {
        A aw = 0, ab = 0;
        for (int64_t s = 0; s < splits; ++s) {
            aw += partial[(s * 2) * d + i];
            ab += partial[(s * 2 + 1) * d + i];
        }
        if (dw) dw[i] = from_acc<W>(Acc<W>(aw));
        if (db) db[i] = from_acc<W>(Acc<W>(ab));
    }
}

int64_t split_rows_of(int64_t rows) {
    int64_t per = (rows + kMaxSplits - 1) / kMaxSplits;
    return per < kSplitRows ? kSplitRows : per;
}
int64_t splits_of(int64_t rows) { return (rows + split_rows_of(rows) - 1) / split_rows_of(rows); }

int check_norm(const char *who, int64_t rows, int64_t d, int dtype, int wdtype) {
    if (!row_dtype(dtype)) return fail(BGL_E_UNSUPPORTED, "%s: dtype %d", who, dtype);
    if (wdtype != dtype && !(dtype == BGL_BF16 && wdtype == BGL_F32))
        return fail(BGL_E_UNSUPPORTED, "%s: weight dtype %d with dtype %d", who, wdtype, dtype);
    if (rows < 0 || d < 0) return fail(BGL_E_INVALID, "%s: negative size", who);
    if (d >= (int64_t(1) << 31)) return fail(BGL_E_UNSUPPORTED, "%s: d >= 2^31", who);
    return BGL_OK;
}

template <typename T, typename W>
int forward(const void *x, const void *w, const void *b, int64_t rows, int64_t d, double eps,
            void *y, void *mean, void *rstd, cudaStream_t s) {
    const int64_t cap = (int64_t)num_sms() * 8;
    k_layer_norm<T, W><<<(unsigned)(rows < cap ? rows : cap), 256, 0, s>>>(
        (const T *)x, (const W *)w, (const W *)b, rows, d, (Acc<T>)eps, (T *)y, (Acc<T> *)mean,
        (Acc<T> *)rstd);
    BGL_LAUNCH_CHECK();
    return BGL_OK;
}

template <typename T, typename W>
int backward(const void *dy, const void *x, const void *mean, const void *rstd, const void *w,
             int64_t rows, int64_t d, void *dx, void *dw, void *db, void *ws, cudaStream_t s) {
    using A = Acc<T>;
    const int64_t cap = (int64_t)num_sms() * 8;
    if (dx && rows) {
        k_layer_norm_dx<T, W><<<(unsigned)(rows < cap ? rows : cap), 256, 0, s>>>(
            (const T *)dy, (const T *)x, (const A *)mean, (const A *)rstd, (const W *)w, rows, d,
            (T *)dx);
        BGL_LAUNCH_CHECK();
    }
    if (dw || db) {
        Carver c(ws);
        A *partial = c.take<A>((size_t)(2 * splits_of(rows) * d));
        if (rows) {
            dim3 grid((unsigned)((d + 31) / 32), (unsigned)splits_of(rows));
            k_layer_norm_dw<T><<<grid, 256, 0, s>>>((const T *)dy, (const T *)x, (const A *)mean,
                                                    (const A *)rstd, rows, d, split_rows_of(rows),
                                                    partial);
            BGL_LAUNCH_CHECK();
        }
        k_layer_norm_dw_join<A, W><<<(unsigned)((d + 255) / 256), 256, 0, s>>>(
            partial, splits_of(rows), d, (W *)dw, (W *)db);
        BGL_LAUNCH_CHECK();
    }
    return BGL_OK;
}

}  // namespace
}  // namespace bgl

using namespace bgl;

extern "C" {

int bgl_layer_norm(const void *x, const void *weight, const void *bias, int64_t rows, int64_t d,
                   double eps, void *y, void *mean, void *rstd, int dtype, int wdtype,
                   void *stream) {
    int rc = check_norm("bgl_layer_norm", rows, d, dtype, wdtype);
    if (rc) return rc;
    if (!(eps >= 0)) return fail(BGL_E_INVALID, "bgl_layer_norm: eps must be >= 0");
    if (rows == 0 || d == 0) return BGL_OK;
    if (!x || !y) return fail(BGL_E_INVALID, "bgl_layer_norm: null buffer");
    cudaStream_t s = as_stream(stream);
    if (dtype == BGL_F64) return forward<double, double>(x, weight, bias, rows, d, eps, y, mean, rstd, s);
    if (dtype == BGL_F32) return forward<float, float>(x, weight, bias, rows, d, eps, y, mean, rstd, s);
    if (wdtype == BGL_F32)
        return forward<__nv_bfloat16, float>(x, weight, bias, rows, d, eps, y, mean, rstd, s);
    return forward<__nv_bfloat16, __nv_bfloat16>(x, weight, bias, rows, d, eps, y, mean, rstd, s);
}

size_t bgl_layer_norm_backward_workspace_size(int64_t rows, int64_t d, int dtype) {
    if (rows < 0 || d < 0) return 0;
    return (size_t)(2 * splits_of(rows) * d) * (dtype == BGL_F64 ? 8 : 4) + 256;
}

int bgl_layer_norm_backward(const void *grad, const void *x, const void *mean, const void *rstd,
                            const void *weight, int64_t rows, int64_t d, void *dx, void *dweight,
                            void *dbias, int dtype, int wdtype, void *workspace,
                            size_t workspace_bytes, void *stream) {
    int rc = check_norm("bgl_layer_norm_backward", rows, d, dtype, wdtype);
    if (rc) return rc;
    if (d == 0) return BGL_OK;
    if (rows && (!grad || !x || !mean || !rstd))
        return fail(BGL_E_INVALID, "bgl_layer_norm_backward: null buffer");
    if ((dweight || dbias) &&
        (!workspace || workspace_bytes < bgl_layer_norm_backward_workspace_size(rows, d, dtype)))
        return fail(BGL_E_WORKSPACE, "bgl_layer_norm_backward: workspace too small");
    cudaStream_t s = as_stream(stream);
    if (dtype == BGL_F64)
        return backward<double, double>(grad, x, mean, rstd, weight, rows, d, dx, dweight, dbias,
                                        workspace, s);
    if (dtype == BGL_F32)
        return backward<float, float>(grad, x, mean, rstd, weight, rows, d, dx, dweight, dbias,
                                      workspace, s);
    if (wdtype == BGL_F32)
        return backward<__nv_bfloat16, float>(grad, x, mean, rstd, weight, rows, d, dx, dweight,
                                              dbias, workspace, s);
    return backward<__nv_bfloat16, __nv_bfloat16>(grad, x, mean, rstd, weight, rows, d, dx, dweight,
                                                  dbias, workspace, s);
}

}  // extern "C"
