// Routing of tokens to experts: scores, selection, weights, and their gradient.
//
// A warp per token.  Selection works on order-preserving integer keys of the
// selection scores, so ties, signed zeros and NaN have one order everywhere:
// NaN first, then larger scores, equal ones by the lower expert.  Key 0 is an
// expert that cannot be chosen (a logit or a biased score of -inf, or a group
// that was not kept).
#include "rows.cuh"

namespace bgl {
namespace {

constexpr int kMaxExperts = 1024, kMaxChoices = 32, kMaxGroups = 32;
constexpr int kWarps = 4;  // tokens of a block

struct RouteArgs {
    const void *logits;
    const float *bias;
    int64_t tokens;
    int experts, k, groups, topk_groups, group_top;
    bool sigmoid, renormalize, by_logit;
    float scale;
    float *weights;
    int64_t *indices;
};

// Larger scores give larger keys; -0 and +0 the same one; NaN the largest.
__device__ __forceinline__ uint32_t key_of(float c) {
    if (c != c) return 0xffffffffu;
    const uint32_t u = __float_as_uint(__fadd_rn(c, 0.0f));
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) {
    return __uint_as_float((key & 0x80000000u) ? (key ^ 0x80000000u) : ~key);
}

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// A sum of weights to divide by: the smallest normal number where all of them
// underflowed (their quotients are then 0), NaN where one of them is NaN.
__device__ __forceinline__ float at_least_tiny(float sum) {
    return sum < 1.17549435e-38f ? 1.17549435e-38f : sum;
}

// 1 / (1 + exp(-x)), every step rounded once.
__device__ __forceinline__ float sigmoid_of(float x) {
    return __fdiv_rn(1.0f, __fadd_rn(1.0f, expf(-x)));
}

template <typename T>
__global__ void __launch_bounds__(kWarps * 32) k_route_topk(const RouteArgs a) {
    extern __shared__ uint32_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t *key = smem + warp * a.experts;
    const int per_group = a.experts / a.groups;
    for (int64_t t = (int64_t)blockIdx.x * kWarps + warp; t < a.tokens;
         t += (int64_t)gridDim.x * kWarps) {
        const T *x = static_cast<const T *>(a.logits) + t * a.experts;
        float top = -INFINITY, total = 0;
        if (!a.sigmoid) {
            for (int e = lane; e < a.experts; e += 32) top = fmaxf(top, to_acc(x[e]));
            top = warp_max(top);
            if (top == -INFINITY) top = 0;
            for (int e = lane; e < a.experts; e += 32) total += expf(to_acc(x[e]) - top);
            total = warp_sum(total);
        }
        for (int e = lane; e < a.experts; e += 32) {
            const float l = to_acc(x[e]);
            float c = l;
            if (!a.by_logit) {
                c = a.sigmoid ? sigmoid_of(l) : expf(l - top) / total;
                if (a.bias) c = __fadd_rn(c, a.bias[e]);
            }
            key[e] = (l == -INFINITY || c == -INFINITY) ? 0u : key_of(c);
        }
        __syncwarp();
        if (a.groups > 1) {
            uint32_t best = 0;
            if (lane < a.groups) {
                uint32_t k1 = 0, k2 = 0;
                for (int i = 0; i < per_group; ++i) {
                    const uint32_t k = key[lane * per_group + i];
                    if (k > k1) {
                        k2 = k1;
                        k1 = k;
                    } else if (k > k2) {
                        k2 = k;
                    }
                }
                best = k1;
                if (a.group_top == 2 && k2) best = key_of(__fadd_rn(value_of(k1), value_of(k2)));
            }
            int rank = 0;
            for (int g = 0; g < a.groups; ++g) {
                const uint32_t other = __shfl_sync(0xffffffffu, best, g);
                rank += other > best || (other == best && g < lane);
            }
            if (lane < a.groups && rank >= a.topk_groups)
                for (int i = 0; i < per_group; ++i) key[lane * per_group + i] = 0;
            __syncwarp();
        }
        int mine = -1;
        for (int j = 0; j < a.k; ++j) {
            uint32_t best = 0;
            int at = a.experts;
            for (int e = lane; e < a.experts; e += 32)
                if (key[e] > best) {
                    best = key[e];
                    at = e;
                }
            const uint32_t top_key = __reduce_max_sync(0xffffffffu, best);
            if (top_key == 0) break;
            const int e = __reduce_min_sync(0xffffffffu, best == top_key ? at : a.experts);
            if (lane == j) mine = e;
            if (lane == (e & 31)) key[e] = 0;
            __syncwarp();
        }
        __syncwarp();
        const float l = mine >= 0 ? to_acc(x[mine]) : -INFINITY;
        float w = 0;
        if (a.sigmoid) {
            w = mine >= 0 ? sigmoid_of(l) : 0.0f;
            if (a.renormalize) w = w / at_least_tiny(warp_sum(w));
        } else if (a.renormalize) {
            const float m = warp_max(l);
            w = mine >= 0 ? expf(l - m) : 0.0f;
            const float sum = warp_sum(w);
            if (mine >= 0) w /= sum;
        } else if (mine >= 0) {
            w = expf(l - top) / total;
        }
        if (lane < a.k) {
            a.weights[t * a.k + lane] = mine >= 0 ? w * a.scale : 0.0f;
            a.indices[t * a.k + lane] = mine;
        }
    }
}

struct RouteGradArgs {
    const float *grad;
    const void *logits;
    const int64_t *indices;
    int64_t tokens;
    int experts, k;
    bool sigmoid, renormalize;
    float scale;
    void *dlogits;
};

template <typename T>
__global__ void __launch_bounds__(kWarps * 32) k_route_topk_backward(const RouteGradArgs a) {
    extern __shared__ float sums[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float *acc = sums + warp * a.experts;
    for (int64_t t = (int64_t)blockIdx.x * kWarps + warp; t < a.tokens;
         t += (int64_t)gridDim.x * kWarps) {
        const T *x = static_cast<const T *>(a.logits) + t * a.experts;
        T *dx = static_cast<T *>(a.dlogits) + t * a.experts;
        int64_t at = lane < a.k ? a.indices[t * a.k + lane] : -1;
        if (at >= a.experts) at = -1;
        const bool chosen = at >= 0;
        float g = chosen ? a.grad[t * a.k + lane] * a.scale : 0.0f;
        const float l = chosen ? to_acc(x[at]) : -INFINITY;
        const bool dense = !a.sigmoid && !a.renormalize;
        if (a.sigmoid) {
            const float s = chosen ? sigmoid_of(l) : 0.0f;
            if (a.renormalize) {
                const float total = at_least_tiny(warp_sum(s));
                g = (g - warp_sum(g * s) / total) / total;
            }
            g = chosen ? g * (s * sigmoid_of(-l)) : 0.0f;
        } else if (a.renormalize) {
            const float m = warp_max(l);
            const float p = chosen ? expf(l - m) : 0.0f;
            const float w = p / warp_sum(p);
            const float mean = warp_sum(chosen ? w * g : 0.0f);
            g = chosen ? w * (g - mean) : 0.0f;
        }
        for (int e = lane; e < a.experts; e += 32) acc[e] = 0;
        __syncwarp();
        // one choice after the other: indices given twice add up in order
        for (int j = 0; j < a.k; ++j) {
            if (lane == j && chosen) acc[at] += g;
            __syncwarp();
        }
        if (dense) {
            float top = -INFINITY, total = 0, dot = 0;
            for (int e = lane; e < a.experts; e += 32) top = fmaxf(top, to_acc(x[e]));
            top = warp_max(top);
            if (top == -INFINITY) top = 0;
            for (int e = lane; e < a.experts; e += 32) {
                const float p = expf(to_acc(x[e]) - top);
                total += p;
                dot += p * acc[e];
            }
            total = warp_sum(total);
            if (total == 0) total = 1;  // every expert masked: no gradient
            dot = warp_sum(dot) / total;
            for (int e = lane; e < a.experts; e += 32)
                dx[e] = from_acc<T>(expf(to_acc(x[e]) - top) / total * (acc[e] - dot));
        } else {
            for (int e = lane; e < a.experts; e += 32) dx[e] = from_acc<T>(acc[e]);
        }
        __syncwarp();
    }
}

int check_route(const char *who, int64_t tokens, int64_t experts, int64_t k, int score, int dtype) {
    if (dtype != BGL_F32 && dtype != BGL_BF16) return fail(BGL_E_UNSUPPORTED, "%s: dtype %d", who, dtype);
    if (score != BGL_SCORE_SOFTMAX && score != BGL_SCORE_SIGMOID)
        return fail(BGL_E_INVALID, "%s: score %d", who, score);
    if (tokens < 0 || experts < 1) return fail(BGL_E_INVALID, "%s: bad size", who);
    if (experts > kMaxExperts)
        return fail(BGL_E_UNSUPPORTED, "%s: more than %d experts", who, kMaxExperts);
    if (k < 1 || k > experts) return fail(BGL_E_INVALID, "%s: k must be in [1, experts]", who);
    if (k > kMaxChoices) return fail(BGL_E_UNSUPPORTED, "%s: k above %d", who, kMaxChoices);
    return BGL_OK;
}

unsigned blocks_for(int64_t tokens) {
    const int64_t want = (tokens + kWarps - 1) / kWarps, cap = (int64_t)num_sms() * 16;
    return (unsigned)(want < cap ? want : cap);
}

}  // namespace
}  // namespace bgl

using namespace bgl;

extern "C" {

int bgl_route_topk(const void *logits, const float *bias, int64_t tokens, int64_t experts,
                   int64_t k, int score, int64_t num_groups, int64_t topk_groups, int group_top,
                   int renormalize, double scale, float *weights, int64_t *indices, int dtype,
                   void *stream) {
    int rc = check_route("bgl_route_topk", tokens, experts, k, score, dtype);
    if (rc) return rc;
    if (num_groups < 1 || experts % num_groups)
        return fail(BGL_E_INVALID, "bgl_route_topk: num_groups must divide the experts");
    if (num_groups > kMaxGroups)
        return fail(BGL_E_UNSUPPORTED, "bgl_route_topk: more than %d groups", kMaxGroups);
    if (topk_groups < 1 || topk_groups > num_groups)
        return fail(BGL_E_INVALID, "bgl_route_topk: topk_groups must be in [1, num_groups]");
    if (group_top != 1 && group_top != 2)
        return fail(BGL_E_INVALID, "bgl_route_topk: group_top must be 1 or 2");
    if (k > topk_groups * (experts / num_groups))
        return fail(BGL_E_INVALID, "bgl_route_topk: k above the experts of the kept groups");
    if (tokens == 0) return BGL_OK;
    if (!logits || !weights || !indices) return fail(BGL_E_INVALID, "bgl_route_topk: null buffer");
    RouteArgs a;
    a.logits = logits;
    a.bias = bias;
    a.tokens = tokens;
    a.experts = (int)experts;
    a.k = (int)k;
    a.groups = (int)num_groups;
    a.topk_groups = (int)topk_groups;
    a.group_top = group_top;
    a.sigmoid = score == BGL_SCORE_SIGMOID;
    a.renormalize = renormalize != 0;
    // without a bias or sums of scores the order of the scores is the logits'
    a.by_logit = !bias && (num_groups == 1 || group_top == 1);
    a.scale = (float)scale;
    a.weights = weights;
    a.indices = indices;
    const size_t smem = (size_t)kWarps * experts * sizeof(uint32_t);
    if (dtype == BGL_F32)
        k_route_topk<float><<<blocks_for(tokens), kWarps * 32, smem, as_stream(stream)>>>(a);
    else
        k_route_topk<__nv_bfloat16><<<blocks_for(tokens), kWarps * 32, smem, as_stream(stream)>>>(a);
    BGL_LAUNCH_CHECK();
    return BGL_OK;
}

int bgl_route_topk_backward(const float *grad, const void *logits, const int64_t *indices,
                            int64_t tokens, int64_t experts, int64_t k, int score, int renormalize,
                            double scale, void *dlogits, int dtype, void *stream) {
    int rc = check_route("bgl_route_topk_backward", tokens, experts, k, score, dtype);
    if (rc) return rc;
    if (tokens == 0) return BGL_OK;
    if (!grad || !logits || !indices || !dlogits)
        return fail(BGL_E_INVALID, "bgl_route_topk_backward: null buffer");
    RouteGradArgs a;
    a.grad = grad;
    a.logits = logits;
    a.indices = indices;
    a.tokens = tokens;
    a.experts = (int)experts;
    a.k = (int)k;
    a.sigmoid = score == BGL_SCORE_SIGMOID;
    a.renormalize = renormalize != 0;
    a.scale = (float)scale;
    a.dlogits = dlogits;
    const size_t smem = (size_t)kWarps * experts * sizeof(float);
    if (dtype == BGL_F32)
        k_route_topk_backward<float><<<blocks_for(tokens), kWarps * 32, smem, as_stream(stream)>>>(a);
    else
        k_route_topk_backward<__nv_bfloat16>
            <<<blocks_for(tokens), kWarps * 32, smem, as_stream(stream)>>>(a);
    BGL_LAUNCH_CHECK();
    return BGL_OK;
}

}  // extern "C"
