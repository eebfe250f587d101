// Sending token rows to their experts and joining what comes back.
//
// The plan is a stable counting sort of the (token, choice) pairs by expert:
// positions[t, j] is the row of pair (t, j) among all rows sorted by expert.
// Pairs without an expert come behind all others, and their position is stored
// as ~row, so that every row belongs to exactly one pair and every kernel that
// writes rows fills all of them (zeros for pairs without an expert) without
// asking how many there are.
//
//   dispatch:  rows[p] = x[t]                     combine:  y[t] = sum_j w[t, j] rows[p]
//   backward:  drows[p] = w[t, j] dy[t],  dw[t, j] = <dy[t], rows[p]>     (p = positions[t, j])
#include "rows.cuh"

namespace bgl {
namespace {

constexpr int kMaxBins = 8192;   // experts + 1: one shared-memory counter each
constexpr int kMaxChunks = 2048;

// Item i's bin: its expert, or `experts` (the last bin) for none.
__device__ __forceinline__ int bin_of(int64_t index, int experts) {
    return index >= 0 && index < experts ? (int)index : experts;
}

int64_t chunk_items(int64_t items) {
    int64_t per = (items + kMaxChunks - 1) / kMaxChunks;
    if (per < 1024) per = 1024;
    return (per + 31) / 32 * 32;
}
int64_t num_chunks(int64_t items) { return (items + chunk_items(items) - 1) / chunk_items(items); }

// bins of one chunk of consecutive items
__global__ void __launch_bounds__(256)
    k_plan_count(const int64_t *__restrict__ indices, int64_t items, int64_t per, int experts,
                 int32_t *__restrict__ chunk_bins) {
    extern __shared__ int32_t bins[];
    for (int b = threadIdx.x; b <= experts; b += blockDim.x) bins[b] = 0;
    __syncthreads();
    const int64_t i0 = blockIdx.x * per, i1 = i0 + per < items ? i0 + per : items;
    for (int64_t i = i0 + threadIdx.x; i < i1; i += blockDim.x)
        atomicAdd(&bins[bin_of(indices[i], experts)], 1);
    __syncthreads();
    for (int b = threadIdx.x; b <= experts; b += blockDim.x)
        chunk_bins[blockIdx.x * (int64_t)(experts + 1) + b] = bins[b];
}

// chunk_bins becomes the first row of each (chunk, bin); one block
__global__ void __launch_bounds__(1024)
    k_plan_scan(int32_t *__restrict__ chunk_bins, int64_t chunks, int experts,
                int64_t *__restrict__ counts) {
    extern __shared__ int32_t total[];
    for (int b = threadIdx.x; b <= experts; b += blockDim.x) {
        int32_t sum = 0;
        for (int64_t c = 0; c < chunks; ++c) {
            int32_t *p = chunk_bins + c * (experts + 1) + b;
            const int32_t n = *p;
            *p = sum;
            sum += n;
        }
        total[b] = sum;
        if (b < experts) counts[b] = sum;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        int32_t sum = 0;
        for (int b = 0; b <= experts; ++b) {
            const int32_t n = total[b];
            total[b] = sum;
            sum += n;
        }
    }
    __syncthreads();
    for (int b = threadIdx.x; b <= experts; b += blockDim.x)
        for (int64_t c = 0; c < chunks; ++c) chunk_bins[c * (experts + 1) + b] += total[b];
}

// one warp a chunk, 32 items a step in order
__global__ void __launch_bounds__(32)
    k_plan_place(const int64_t *__restrict__ indices, int64_t items, int64_t per, int experts,
                 const int32_t *__restrict__ chunk_bins, int32_t *__restrict__ positions) {
    extern __shared__ int32_t next[];
    const int lane = threadIdx.x;
    for (int b = lane; b <= experts; b += 32)
        next[b] = chunk_bins[blockIdx.x * (int64_t)(experts + 1) + b];
    __syncwarp();
    const int64_t i0 = blockIdx.x * per, i1 = i0 + per < items ? i0 + per : items;
    for (int64_t i = i0; i < i1; i += 32) {
        const bool in = i + lane < i1;
        const int bin = in ? bin_of(indices[i + lane], experts) : -1;
        const unsigned same = __match_any_sync(0xffffffffu, bin);
        const int before = __popc(same & ((1u << lane) - 1));
        const int32_t p = in ? next[bin] + before : 0;
        __syncwarp();
        if (in && before == 0) next[bin] += __popc(same);
        __syncwarp();
        if (in) positions[i + lane] = bin == experts ? ~p : p;
    }
}

// Row of a position; false where the pair has no expert.  A position outside
// [0, total) is not one of a plan's: it gives row -1, which is not touched.
__device__ __forceinline__ bool row_of(int32_t position, int64_t total, int64_t &row) {
    row = position >= 0 ? position : ~position;
    if (row >= total) row = -1;
    return position >= 0 && row >= 0;
}

template <typename T>
__global__ void __launch_bounds__(256)
    k_dispatch(const T *__restrict__ x, const int32_t *__restrict__ positions, int64_t tokens,
               int k, int64_t d, T *__restrict__ rows) {
    for (int64_t t = blockIdx.x; t < tokens; t += gridDim.x)
        for (int j = 0; j < k; ++j) {
            int64_t row;
            const bool sent = row_of(positions[t * k + j], tokens * k, row);
            if (row < 0) continue;
            for (int64_t i = threadIdx.x; i < d; i += blockDim.x)
                rows[row * d + i] = sent ? x[t * d + i] : from_acc<T>(0);
        }
}

template <typename T>
__global__ void __launch_bounds__(256)
    k_combine(const T *__restrict__ rows, const int32_t *__restrict__ positions,
              const Acc<T> *__restrict__ weights, int64_t tokens, int k, int64_t d,
              T *__restrict__ y) {
    using A = Acc<T>;
    for (int64_t t = blockIdx.x; t < tokens; t += gridDim.x)
        for (int64_t i = threadIdx.x; i < d; i += blockDim.x) {
            A sum = 0;
            for (int j = 0; j < k; ++j) {
                int64_t row;
                if (!row_of(positions[t * k + j], tokens * k, row)) continue;
                const A v = to_acc(rows[row * d + i]);
                sum += weights ? weights[t * k + j] * v : v;
            }
            y[t * d + i] = from_acc<T>(sum);
        }
}

template <typename T>
__global__ void __launch_bounds__(256)
    k_combine_backward(const T *__restrict__ dy, const T *__restrict__ rows,
                       const int32_t *__restrict__ positions, const Acc<T> *__restrict__ weights,
                       int64_t tokens, int k, int64_t d, T *__restrict__ drows,
                       Acc<T> *__restrict__ dweights) {
    using A = Acc<T>;
    __shared__ A smem[32];
    for (int64_t t = blockIdx.x; t < tokens; t += gridDim.x)
        for (int j = 0; j < k; ++j) {
            int64_t row;
            const bool sent = row_of(positions[t * k + j], tokens * k, row);
            const A w = !sent ? A(0) : weights ? weights[t * k + j] : A(1);
            A dot = 0;
            if (row >= 0)
                for (int64_t i = threadIdx.x; i < d; i += blockDim.x) {
                    const A g = sent ? to_acc(dy[t * d + i]) : A(0);
                    if (dweights && sent) dot += g * to_acc(rows[row * d + i]);
                    if (drows) drows[row * d + i] = from_acc<T>(w * g);
                }
            if (dweights) {
                dot = block_sum(dot, smem);
                if (threadIdx.x == 0) dweights[t * k + j] = dot;
            }
        }
}

int check_rows(const char *who, int64_t tokens, int64_t k, int64_t d, int dtype) {
    if (!row_dtype(dtype)) return fail(BGL_E_UNSUPPORTED, "%s: dtype %d", who, dtype);
    if (tokens < 0 || k < 0 || d < 0) return fail(BGL_E_INVALID, "%s: negative size", who);
    if (k >= (int64_t(1) << 31) || (k && tokens >= (int64_t(1) << 31) / k))
        return fail(BGL_E_UNSUPPORTED, "%s: tokens * k >= 2^31", who);
    return BGL_OK;
}

unsigned token_blocks(int64_t tokens) {
    const int64_t cap = (int64_t)num_sms() * 8;
    return (unsigned)(tokens < cap ? tokens : cap);
}

}  // namespace
}  // namespace bgl

using namespace bgl;

extern "C" {

size_t bgl_expert_plan_workspace_size(int64_t items, int64_t experts) {
    if (items < 0 || experts < 0) return 0;
    return (size_t)num_chunks(items) * (experts + 1) * sizeof(int32_t) + 256;
}

int bgl_expert_plan(const int64_t *indices, int64_t items, int64_t experts, int64_t *counts,
                    int32_t *positions, void *workspace, size_t workspace_bytes, void *stream) {
    if (items < 0 || experts < 1) return fail(BGL_E_INVALID, "bgl_expert_plan: bad size");
    if (items >= (int64_t(1) << 31)) return fail(BGL_E_UNSUPPORTED, "bgl_expert_plan: 2^31 items or more");
    if (experts >= kMaxBins)
        return fail(BGL_E_UNSUPPORTED, "bgl_expert_plan: more than %d experts", kMaxBins - 1);
    if (!counts || (items && (!indices || !positions)))
        return fail(BGL_E_INVALID, "bgl_expert_plan: null buffer");
    if (!workspace || workspace_bytes < bgl_expert_plan_workspace_size(items, experts))
        return fail(BGL_E_WORKSPACE, "bgl_expert_plan: workspace too small");
    cudaStream_t s = as_stream(stream);
    Carver c(workspace);
    const int64_t chunks = num_chunks(items), per = chunk_items(items);
    int32_t *chunk_bins = c.take<int32_t>((size_t)chunks * (experts + 1));
    const size_t smem = (size_t)(experts + 1) * sizeof(int32_t);
    if (chunks) {
        k_plan_count<<<(unsigned)chunks, 256, smem, s>>>(indices, items, per, (int)experts, chunk_bins);
        BGL_LAUNCH_CHECK();
    }
    k_plan_scan<<<1, 1024, smem, s>>>(chunk_bins, chunks, (int)experts, counts);
    BGL_LAUNCH_CHECK();
    if (chunks) {
        k_plan_place<<<(unsigned)chunks, 32, smem, s>>>(indices, items, per, (int)experts,
                                                        chunk_bins, positions);
        BGL_LAUNCH_CHECK();
    }
    return BGL_OK;
}

int bgl_dispatch_rows(const void *x, const int32_t *positions, int64_t tokens, int64_t k,
                      int64_t d, void *rows, int dtype, void *stream) {
    int rc = check_rows("bgl_dispatch_rows", tokens, k, d, dtype);
    if (rc) return rc;
    if (tokens == 0 || k == 0 || d == 0) return BGL_OK;
    if (!x || !positions || !rows) return fail(BGL_E_INVALID, "bgl_dispatch_rows: null buffer");
    cudaStream_t s = as_stream(stream);
    const unsigned grid = token_blocks(tokens);
    if (dtype == BGL_F64)
        k_dispatch<double><<<grid, 256, 0, s>>>((const double *)x, positions, tokens, (int)k, d, (double *)rows);
    else if (dtype == BGL_F32)
        k_dispatch<float><<<grid, 256, 0, s>>>((const float *)x, positions, tokens, (int)k, d, (float *)rows);
    else
        k_dispatch<__nv_bfloat16><<<grid, 256, 0, s>>>((const __nv_bfloat16 *)x, positions, tokens,
                                                       (int)k, d, (__nv_bfloat16 *)rows);
    BGL_LAUNCH_CHECK();
    return BGL_OK;
}

int bgl_combine_rows(const void *rows, const int32_t *positions, const void *weights,
                     int64_t tokens, int64_t k, int64_t d, void *y, int dtype, void *stream) {
    int rc = check_rows("bgl_combine_rows", tokens, k, d, dtype);
    if (rc) return rc;
    if (tokens == 0 || d == 0) return BGL_OK;
    if (!y || (k && (!rows || !positions))) return fail(BGL_E_INVALID, "bgl_combine_rows: null buffer");
    cudaStream_t s = as_stream(stream);
    const unsigned grid = token_blocks(tokens);
    if (dtype == BGL_F64)
        k_combine<double><<<grid, 256, 0, s>>>((const double *)rows, positions, (const double *)weights,
                                               tokens, (int)k, d, (double *)y);
    else if (dtype == BGL_F32)
        k_combine<float><<<grid, 256, 0, s>>>((const float *)rows, positions, (const float *)weights,
                                              tokens, (int)k, d, (float *)y);
    else
        k_combine<__nv_bfloat16><<<grid, 256, 0, s>>>((const __nv_bfloat16 *)rows, positions,
                                                      (const float *)weights, tokens, (int)k, d,
                                                      (__nv_bfloat16 *)y);
    BGL_LAUNCH_CHECK();
    return BGL_OK;
}

int bgl_combine_rows_backward(const void *grad, const void *rows, const int32_t *positions,
                              const void *weights, int64_t tokens, int64_t k, int64_t d,
                              void *drows, void *dweights, int dtype, void *stream) {
    int rc = check_rows("bgl_combine_rows_backward", tokens, k, d, dtype);
    if (rc) return rc;
    if (tokens == 0 || k == 0) return BGL_OK;
    if (!positions || (d && (!grad || (dweights && !rows))))
        return fail(BGL_E_INVALID, "bgl_combine_rows_backward: null buffer");
    cudaStream_t s = as_stream(stream);
    const unsigned grid = token_blocks(tokens);
    if (dtype == BGL_F64)
        k_combine_backward<double><<<grid, 256, 0, s>>>(
            (const double *)grad, (const double *)rows, positions, (const double *)weights, tokens,
            (int)k, d, (double *)drows, (double *)dweights);
    else if (dtype == BGL_F32)
        k_combine_backward<float><<<grid, 256, 0, s>>>(
            (const float *)grad, (const float *)rows, positions, (const float *)weights, tokens,
            (int)k, d, (float *)drows, (float *)dweights);
    else
        k_combine_backward<__nv_bfloat16><<<grid, 256, 0, s>>>(
            (const __nv_bfloat16 *)grad, (const __nv_bfloat16 *)rows, positions,
            (const float *)weights, tokens, (int)k, d, (__nv_bfloat16 *)drows, (float *)dweights);
    BGL_LAUNCH_CHECK();
    return BGL_OK;
}

}  // extern "C"
