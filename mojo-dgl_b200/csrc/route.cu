// Routing of tokens to experts: scores, selection, weights, and their gradient.
//
// Forward.  Eight lanes work on a token, four tokens a warp.  They bring the
// token's logits into shared memory in 16-byte pieces and turn them into
// selection scores there; then lane i owns the i-th eighth of the experts and
// keeps the maximum of every 8 of its scores in registers.  A round of the top-k
// is a maximum over registers and three shuffles; only the lane that holds the
// best score looks into shared memory, at 8 values, and takes it out.  Equal
// scores go to the lowest lane and the lowest place in it: the lowest expert.
// What bounds this is instructions and the length of a warp's chain of them, not
// memory.  65,536 tokens x 256 experts (sigmoid, bias, 4 of 8 groups, k = 8) took
// 172 us with a warp a token and scores rescanned every round, 92 us with 8 lanes
// and every score in unrolled registers (code beyond the instruction cache), 62 us
// with 4 lanes as below (fewest instructions, but 24 warps an SM and the last ones
// run long), 51 us so (52.4 with the question whether every sigmoid underflows).
//
// A sigmoid of float32 accuracy costs 20 instructions, an approximate one 5.
// Scores with a bias are therefore first taken from approximate sigmoids: where
// every decision (the groups kept, the order of the k best, the best of the
// rest) has more room than both scores can be off, the exact scores decide the
// same, and only the k weights need them.  Otherwise the warp selects again from
// exact scores, which is what defines the result.
//
// -inf stands for an expert that cannot be chosen.  NaN takes no part in the
// rounds (fmaxf passes over it): a row that has one picks its NaN first, in a
// loop that other rows do not enter.
//
// Backward.  The row of gradients is built in shared memory from the k chosen
// experts, the softmax's two sums run over registers.
#include "rows.cuh"

namespace bgl {
namespace {

constexpr int kMaxExperts = 1024, kMaxChoices = 32, kMaxGroups = 32;
constexpr int kLanes = 8;            // lanes of a token
constexpr int kSelect = 64;          // threads of a selecting block: two warps, so that SMs even out
constexpr int kSlots = kSelect / kLanes;  // its tokens
constexpr int kWarps = 4;            // warps of a block of the backward pass

struct RouteArgs {
    const void *logits;
    const float *bias;
    int64_t tokens;
    int experts, k, groups, topk_groups, group_top;
    bool sigmoid, renormalize, by_logit, bias_aligned;
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

// Maximum and sum over the LANES lanes of a token, on each of them.
template <int LANES>
__device__ __forceinline__ float lanes_max(float v) {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
template <int LANES>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Four logits at once.
__device__ __forceinline__ void load4(const float *p, float (&v)[4]) {
    const float4 x = __ldg(reinterpret_cast<const float4 *>(p));
    v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
}
__device__ __forceinline__ void load4(const __nv_bfloat16 *p, float (&v)[4]) {
    const uint2 x = __ldg(reinterpret_cast<const uint2 *>(p));
    v[0] = __uint_as_float(x.x << 16), v[1] = __uint_as_float(x.x & 0xffff0000u);
    v[2] = __uint_as_float(x.y << 16), v[3] = __uint_as_float(x.y & 0xffff0000u);
}
__device__ __forceinline__ void store4(float *p, const float (&v)[4]) {
    *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ void store4(__nv_bfloat16 *p, const float (&v)[4]) {
    __nv_bfloat162 o[2] = {__floats2bfloat162_rn(v[0], v[1]), __floats2bfloat162_rn(v[2], v[3])};
    *reinterpret_cast<uint2 *>(p) = *reinterpret_cast<uint2 *>(o);
}

// A sum of weights to divide by: the smallest normal number where there are none
// (their quotients are then 0), NaN where one of them is NaN.
__device__ __forceinline__ float at_least_tiny(float sum) {
    return sum < 1.17549435e-38f ? 1.17549435e-38f : sum;
}

// 1 / (1 + exp(-x)), every step rounded once.
__device__ __forceinline__ float sigmoid_of(float x) { return __frcp_rn(__fadd_rn(1.0f, expf(-x))); }

// The same from the approximate exponential and reciprocal (PTX: ex2.approx is
// off by 2 units in the last place, rcp.approx by 1).  The product of x and
// log2 e is off by 2^-23.4 |x| of an exponent, s (1 - s) |x| <= 0.224, so s is
// off by (0.17 + 0.5 + 1 + 0.5) 2^-23 at most, sigmoid_of by 1.25 * 2^-23, and
// with a bias that leaves |c| < 2 the two sums by 2^-23 each: together less
// than 6 * 2^-23.  kNear is more than twice that.
__device__ __forceinline__ float near_sigmoid(float x) {
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x * -1.4426950408889634f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
    return r;
}
constexpr float kNear = 1.0f / (1 << 19);

// NaN if either is NaN.
__device__ __forceinline__ float max_or_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// The k weights of a token whose sigmoids add up to less than kFar (`far`; the warp's
// other tokens take part).  From -88.7 on they underflow, but their shares in the sum do
// not: 1 + exp(x) is 1 there, and the sigmoids are the exponentials, which are taken
// relative to the best one's.  Apart from the kernel, so that the way past it is short
// (65536 x 256 in groups: 51.3 us without it, 52.3 so, 53.5 with a branch for each token).
constexpr float kFar = 1e-9f;
template <typename T>
__device__ __noinline__ void far_weights(const T *x, const int *pick, int k, float scale, bool far, float *weights) {
    const int own = threadIdx.x & (kLanes - 1);
    float most = -INFINITY, total = 0;
    for (int j = own; j < k; j += kLanes)
        if (pick[j] >= 0) most = fmaxf(most, to_acc(x[pick[j]]));
    most = lanes_max<kLanes>(most);
    for (int j = own; j < k; j += kLanes)
        if (pick[j] >= 0) total += expf(to_acc(x[pick[j]]) - most);
    total = lanes_sum<kLanes>(total);
    if (!far) return;
    for (int j = own; j < k; j += kLanes)
        if (pick[j] >= 0) weights[j] = expf(to_acc(x[pick[j]]) - most) / total * scale;
}

// A token's scores in shared memory: kLanes runs of subs * 8, 4 apart.
__host__ __device__ constexpr int select_row(int subs) { return kLanes * (subs * 8 + 4); }

// SUBS * 8 experts a lane; VEC: rows in 16-byte (bf16: 8-byte) pieces.
template <typename T, int SUBS, bool VEC>
__global__ void __launch_bounds__(kSelect, SUBS > 4 ? 1 : 18) k_route_topk(const RouteArgs a) {
    constexpr int kOwn = SUBS * 8;     // experts of a lane
    constexpr int kStride = kOwn + 4;  // apart in shared memory: no bank conflicts
    constexpr int kRow = select_row(SUBS);
    constexpr int kPieces = kOwn / 4;       // of four scores
    constexpr unsigned kMask = (1u << kLanes) - 1;
    extern __shared__ __align__(16) float smem[];
    const int lane = threadIdx.x & 31, own = lane & (kLanes - 1), base = lane & ~(kLanes - 1);
    const int slot = threadIdx.x / kLanes;
    float *c = smem + slot * kRow, *mine = c + own * kStride;
    int *pick = reinterpret_cast<int *>(smem + kSlots * kRow) + slot * a.k;
    uint32_t *group = reinterpret_cast<uint32_t *>(smem + kSlots * (kRow + a.k)) + slot * a.groups;
    const int experts = a.experts, per_group = experts / a.groups;
    auto at = [](int e) { return e + e / kOwn * 4; };  // expert e's place in c
    auto piece = [&](int i) {  // the i-th four scores that this lane brings in
        return reinterpret_cast<float4 *>(c + at((own + kLanes * i) * 4));
    };
    const int pieces = (experts + 4 * kLanes - 1) / (4 * kLanes);  // that have experts
    const bool need_sum = !a.sigmoid && !(a.by_logit && a.renormalize);

    // Selection from the scores of `exact` float32 arithmetic, or from nearby
    // ones: true if every decision would be the same with the exact scores.
    auto select = [&](const T *x, bool exact, float &top, float &total) {
        float nan = -INFINITY;
        top = -INFINITY, total = 1;
        if constexpr (VEC && sizeof(T) == 4) {
            // straight into shared memory, every piece in flight at once
#pragma unroll 4
            for (int i = 0; i < kPieces; ++i) {
                const int e = (own + kLanes * i) * 4;
                if (e < experts) cp_async<16>(smem_addr(piece(i)), x + e);
                else *piece(i) = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
            }
            cp_async_commit();
            cp_async_wait<0>();
        } else {
            constexpr int kFlight = kPieces < 8 ? kPieces : 8;
#pragma unroll 1
            for (int i0 = 0; i0 < kPieces; i0 += kFlight) {
                float l[kFlight][4];
#pragma unroll
                for (int i = 0; i < kFlight; ++i) {
                    const int e = (own + kLanes * (i0 + i)) * 4;
#pragma unroll
                    for (int j = 0; j < 4; ++j) l[i][j] = -INFINITY;
                    if constexpr (VEC) {
                        if (e < experts) load4(x + e, l[i]);
                    } else {
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            if (e + j < experts) l[i][j] = to_acc(x[e + j]);
                    }
                }
#pragma unroll
                for (int i = 0; i < kFlight; ++i)
                    *piece(i0 + i) = make_float4(l[i][0], l[i][1], l[i][2], l[i][3]);
            }
        }
        if (need_sum) {
            for (int i = 0; i < pieces; ++i) {
                const float4 v = *piece(i);
                top = fmaxf(fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)), top);
            }
            top = lanes_max<kLanes>(top);
            if (top == -INFINITY) top = 0;
            total = 0;
            for (int i = 0; i < pieces; ++i) {
                const float4 v = *piece(i);
                total += (expf(v.x - top) + expf(v.y - top)) + (expf(v.z - top) + expf(v.w - top));
            }
            total = lanes_sum<kLanes>(total);
        }
        // c = s + bias, in place
        auto scores_by = [&](auto score) {
#pragma unroll 2
            for (int i = 0; i < pieces; ++i) {
                const float4 q = *piece(i);
                float v[4] = {q.x, q.y, q.z, q.w};
                const int e = (own + kLanes * i) * 4;
                float b[4] = {0, 0, 0, 0};
                if (a.bias) {
                    if (VEC && e < experts && a.bias_aligned) {
                        load4(a.bias + e, b);
                    } else {
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            if (e + j < experts) b[j] = __ldg(a.bias + e + j);
                    }
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float s = __fadd_rn(score(v[j]), b[j]);
                    v[j] = v[j] == -INFINITY ? v[j] : s;
                    nan = max_or_nan(nan, v[j]);
                }
                *piece(i) = make_float4(v[0], v[1], v[2], v[3]);
            }
        };
        if (a.by_logit) {
#pragma unroll 4
            for (int i = 0; i < kPieces; ++i) {
                const float4 v = *piece(i);
                nan = max_or_nan(max_or_nan(max_or_nan(v.x, v.y), max_or_nan(v.z, v.w)), nan);
            }
        } else {
            if (!exact) scores_by([](float v) { return near_sigmoid(v); });
            else if (a.sigmoid) scores_by([](float v) { return sigmoid_of(v); });
            else scores_by([&](float v) { return expf(v - top) / total; });
        }
        const unsigned nans = __ballot_sync(0xffffffffu, nan != nan);
        if (!exact && nans) return false;
        __syncwarp();

        bool sure = true;
        if (a.groups > 1) {
            const bool fours = per_group % 4 == 0;
            for (int g = own; g < a.groups; g += kLanes) {
                float k1 = -INFINITY, k2 = -INFINITY;
                bool bad = false;
                auto see = [&](float v) {
                    k2 = fmaxf(k2, fminf(k1, v));
                    k1 = fmaxf(k1, v);
                };
                const int first = g * per_group;
                if (fours && !nans) {
#pragma unroll 2
                    for (int i = 0; i < per_group; i += 4) {
                        const float4 v = *reinterpret_cast<float4 *>(c + at(first + i));
                        see(v.x), see(v.y), see(v.z), see(v.w);
                    }
                } else {
#pragma unroll 1
                    for (int i = 0; i < per_group; ++i) {
                        const float v = c[at(first + i)];
                        if (v != v) bad = true;  // (fminf would take it for k1)
                        else see(v);
                    }
                }
                // 0: nothing to choose in this group
                uint32_t key = k1 == -INFINITY ? 0u : key_of(k1);
                if (a.group_top == 2 && k2 > -INFINITY) key = key_of(__fadd_rn(k1, k2));
                group[g] = bad ? 0xffffffffu : key;
                sure = sure && k1 < 4 && (k2 > -4 || k2 == -INFINITY);
            }
            __syncwarp();
            uint32_t least_kept = 0xffffffffu, most_left = 0;
            for (int g = own; g < a.groups; g += kLanes) {
                const uint32_t key = group[g];
                int rank = 0;
                for (int o = 0; o < a.groups; ++o) {
                    const uint32_t other = group[o];
                    rank += other > key || (other == key && o < g);
                }
                if (rank < a.topk_groups) {
                    least_kept = min(least_kept, key);
                    continue;
                }
                most_left = max(most_left, key);
                const int first = g * per_group;
                if (fours) {
                    for (int i = 0; i < per_group; i += 4)
                        *reinterpret_cast<float4 *>(c + at(first + i)) =
                            make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
                } else {
                    for (int i = 0; i < per_group; ++i) c[at(first + i)] = -INFINITY;
                }
            }
            if (!exact) {
#pragma unroll
                for (int o = kLanes / 2; o > 0; o >>= 1) {
                    least_kept = min(least_kept, __shfl_xor_sync(0xffffffffu, least_kept, o));
                    most_left = max(most_left, __shfl_xor_sync(0xffffffffu, most_left, o));
                }
                // sums of two scores: off by twice as much, and a rounding
                const float kept = value_of(least_kept), left = value_of(most_left);
                sure = most_left == 0 || (kept - left > 2 * kNear && fabsf(kept) < 4 && fabsf(left) < 4);
            }
            __syncwarp();
        }

        // the maxima of the lane's own experts, 8 by 8
        float sub[SUBS];
        auto best_of_8 = [](const float *p) {
            const float4 u = *reinterpret_cast<const float4 *>(p), v = *reinterpret_cast<const float4 *>(p + 4);
            return fmaxf(fmaxf(fmaxf(u.x, u.y), fmaxf(u.z, u.w)), fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)));
        };
#pragma unroll
        for (int s = 0; s < SUBS; ++s) sub[s] = best_of_8(mine + 8 * s);
        int first = 0;  // places taken by NaN
        if (nans) {
            if (own == 0 && (nans >> base & kMask))
                for (int e = 0; e < experts && first < a.k; ++e)
                    if (c[at(e)] != c[at(e)]) pick[first++] = e;
            first = __shfl_sync(0xffffffffu, first, base);
        }
        float before = INFINITY;
#pragma unroll 1
        for (int j = 0;; ++j) {
            if (exact && j == a.k) break;
            float best = -INFINITY;
#pragma unroll
            for (int s = 0; s < SUBS; ++s) best = fmaxf(best, sub[s]);
            const float m = lanes_max<kLanes>(best);
            // in order, and the k-th before the rest, by more than the scores may be off
            sure = sure && (m == -INFINITY || before - m > kNear) && m < 2 && (m > -2 || m == -INFINITY);
            before = m;
            if (j == a.k) break;
            const unsigned holders = __ballot_sync(0xffffffffu, best == m) >> base & kMask;
            if (j < first) continue;
            if (m == -INFINITY) {
                if (own == 0) pick[j] = -1;
            } else if (own == __ffs(holders) - 1) {
                int s = 0;
#pragma unroll
                for (int i = SUBS - 1; i >= 0; --i)
                    if (sub[i] == m) s = i;
                float *eight = mine + 8 * s;
                const float4 u = *reinterpret_cast<float4 *>(eight);
                const float4 v = *reinterpret_cast<float4 *>(eight + 4);
                int place = v.z == m ? 6 : 7;
                place = v.y == m ? 5 : place;
                place = v.x == m ? 4 : place;
                place = u.w == m ? 3 : place;
                place = u.z == m ? 2 : place;
                place = u.y == m ? 1 : place;
                place = u.x == m ? 0 : place;
                eight[place] = -INFINITY;
                pick[j] = own * kOwn + 8 * s + place;
                const float rest = best_of_8(eight);
#pragma unroll
                for (int i = 0; i < SUBS; ++i) sub[i] = i == s ? rest : sub[i];
            }
        }
        __syncwarp();
        return (bool)__all_sync(0xffffffffu, sure);
    };

    for (int64_t t0 = (int64_t)blockIdx.x * kSlots; t0 < a.tokens; t0 += (int64_t)gridDim.x * kSlots) {
        // lanes behind the last token repeat it and write nothing
        const bool live = t0 + slot < a.tokens;
        const int64_t t = live ? t0 + slot : a.tokens - 1;
        const T *x = static_cast<const T *>(a.logits) + t * experts;
        float top, total;
        bool exact = !a.sigmoid || a.by_logit;
#pragma unroll 1
        while (!select(x, exact, top, total) && !exact) exact = true;

        // weights: lane i has the choices i, i + kLanes, ...
        constexpr int kEach = kMaxChoices / kLanes;
        float w[kEach];
        float sum = 0, most = -INFINITY;
        __syncwarp();
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            if (kLanes * i >= a.k) break;
            const int j = own + kLanes * i, e = j < a.k ? pick[j] : -1;
            w[i] = e >= 0 ? to_acc(x[e]) : -INFINITY;
            most = fmaxf(most, w[i]);
        }
        if (!a.sigmoid) most = a.renormalize ? lanes_max<kLanes>(most) : top;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            if (kLanes * i >= a.k) break;
            const int j = own + kLanes * i;
            const bool chosen = j < a.k && pick[j] >= 0;
            w[i] = !chosen ? 0.0f : a.sigmoid ? sigmoid_of(w[i]) : expf(w[i] - most);
            sum += w[i];
        }
        if (a.renormalize) total = at_least_tiny(lanes_sum<kLanes>(sum));
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            if (kLanes * i >= a.k) break;
            const int j = own + kLanes * i;
            if (j >= a.k || !live) continue;
            const int e = pick[j];
            if (a.renormalize || !a.sigmoid) w[i] /= total;
            a.weights[t * a.k + j] = e >= 0 ? w[i] * a.scale : 0.0f;
            a.indices[t * a.k + j] = e;
        }
        if (a.renormalize && a.sigmoid) {
            const bool far = total < kFar && pick[0] >= 0;
            if (__any_sync(0xffffffffu, far)) far_weights(x, pick, a.k, a.scale, far && live, a.weights + t * a.k);
        }
        __syncwarp();
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

// LANES lanes a token, PER experts a lane, in pieces of four (VEC) or one.
template <typename T, int LANES, int PER, bool VEC>
__global__ void __launch_bounds__(kWarps * 32) k_route_topk_backward(const RouteGradArgs a) {
    constexpr int kSlots = kWarps * 32 / LANES;
    constexpr int kWide = VEC ? 4 : 1, kPieces = PER / kWide;
    constexpr int kEach = kMaxChoices / LANES > 0 ? kMaxChoices / LANES : 1;  // choices of a lane
    __shared__ __align__(16) float sums[kSlots][LANES * PER];
    const int lane = threadIdx.x & 31, own = lane & (LANES - 1), slot = threadIdx.x / LANES;
    const int experts = a.experts;
    const bool dense = !a.sigmoid && !a.renormalize;
    float *acc = sums[slot];
    for (int64_t t0 = (int64_t)blockIdx.x * kSlots; t0 < a.tokens; t0 += (int64_t)gridDim.x * kSlots) {
        // lanes behind the last token repeat it and write nothing
        const bool live = t0 + slot < a.tokens;
        const int64_t t = live ? t0 + slot : a.tokens - 1;
        const T *x = static_cast<const T *>(a.logits) + t * experts;
        T *dx = static_cast<T *>(a.dlogits) + t * experts;
        float l[kPieces][kWide];
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const int e = (own + LANES * i) * kWide;
#pragma unroll
            for (int j = 0; j < kWide; ++j) l[i][j] = -INFINITY;
            if (dense && e < experts) {
                if constexpr (VEC) load4(x + e, l[i]);
                else l[i][0] = to_acc(x[e]);
            }
        }
        int at[kEach];
        float g[kEach], s[kEach];
        float most = -INFINITY, total = 0, dot = 0;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int j = own + LANES * i;
            const int64_t e = j < a.k ? a.indices[t * a.k + j] : -1;
            at[i] = e >= 0 && e < experts ? (int)e : -1;
            g[i] = at[i] >= 0 ? a.grad[t * a.k + j] * a.scale : 0.0f;
            s[i] = at[i] >= 0 && !dense ? to_acc(x[at[i]]) : -INFINITY;
            most = fmaxf(most, s[i]);
        }
        if (!dense) {
            if (!a.sigmoid) {
                most = lanes_max<LANES>(most);
                if (most == -INFINITY) most = 0;  // chosen elsewhere, all of them masked: no gradient
            }
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                const float logit = s[i];
                s[i] = at[i] < 0 ? 0.0f : a.sigmoid ? sigmoid_of(logit) : expf(logit - most);
                total += s[i];
                dot += at[i] < 0 ? 0.0f : s[i] * g[i];
                if (a.sigmoid && at[i] >= 0 && !a.renormalize) g[i] *= s[i] * sigmoid_of(-logit);
                // the slope's other factor, needed again below
                if (a.sigmoid && at[i] >= 0 && a.renormalize) s[i] *= sigmoid_of(-logit);
            }
            if (a.renormalize) {
                total = lanes_sum<LANES>(total);
                if (a.sigmoid && __any_sync(0xffffffffu, total < kFar && most > -INFINITY)) {
                    // as far_weights: by the exponentials, whose slope's other factor is 1
                    const bool far = total < kFar;
                    most = lanes_max<LANES>(most);
                    float far_total = 0, far_dot = 0;
#pragma unroll
                    for (int i = 0; i < kEach; ++i) {
                        if (!far || at[i] < 0) continue;
                        s[i] = most > -INFINITY ? expf(to_acc(x[at[i]]) - most) : 0.0f;
                        far_total += s[i];
                        far_dot += s[i] * g[i];
                    }
                    far_total = lanes_sum<LANES>(far_total);
                    if (far) total = far_total, dot = far_dot;
                }
                total = at_least_tiny(total);
                dot = lanes_sum<LANES>(dot) / total;
#pragma unroll
                for (int i = 0; i < kEach; ++i)
                    if (at[i] >= 0) g[i] = s[i] / total * (g[i] - dot);
            }
        }
        // the row of the chosen experts' values, zero elsewhere
#pragma unroll
        for (int i = 0; i < PER / 4; ++i)
            *reinterpret_cast<float4 *>(acc + (own + LANES * i) * 4) = make_float4(0, 0, 0, 0);
        __syncwarp();
        // an expert that is given twice shows where the numbers of its places meet
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            if (at[i] >= 0) acc[at[i]] = __int_as_float(own + LANES * i);
        __syncwarp();
        bool twice = false;
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            twice |= at[i] >= 0 && __float_as_int(acc[at[i]]) != own + LANES * i;
        twice = __any_sync(0xffffffffu, twice);
        if (!twice) {
#pragma unroll
            for (int i = 0; i < kEach; ++i)
                if (at[i] >= 0) acc[at[i]] = g[i];
        } else {  // one place after the other: they add up in order
#pragma unroll
            for (int i = 0; i < kEach; ++i)
                if (at[i] >= 0) acc[at[i]] = 0;
            __syncwarp();
#pragma unroll
            for (int i = 0; i < kEach; ++i)
                for (int o = 0; o < LANES; ++o) {
                    if (own == o && at[i] >= 0) acc[at[i]] += g[i];
                    __syncwarp();
                }
        }
        __syncwarp();
        if (dense) {
            most = -INFINITY;
#pragma unroll
            for (int i = 0; i < kPieces; ++i)
#pragma unroll
                for (int j = 0; j < kWide; ++j) most = fmaxf(most, l[i][j]);
            most = lanes_max<LANES>(most);
            if (most == -INFINITY) most = 0;
            total = dot = 0;
#pragma unroll
            for (int i = 0; i < kPieces; ++i)
#pragma unroll
                for (int j = 0; j < kWide; ++j) {
                    l[i][j] = expf(l[i][j] - most);
                    total += l[i][j];
                    dot += l[i][j] * acc[(own + LANES * i) * kWide + j];
                }
            total = lanes_sum<LANES>(total);
            if (total == 0) total = 1;  // every expert masked: no gradient
            dot = lanes_sum<LANES>(dot) / total;
        }
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const int e = (own + LANES * i) * kWide;
            float v[kWide];
#pragma unroll
            for (int j = 0; j < kWide; ++j) {
                v[j] = acc[e + j];
                if (dense) v[j] = l[i][j] / total * (v[j] - dot);
            }
            if (e < experts && live) {
                if constexpr (VEC) store4(dx + e, v);
                else dx[e] = from_acc<T>(v[0]);
            }
        }
        __syncwarp();
    }
}

template <typename T, int SUBS, bool VEC>
int launch_topk(const RouteArgs &a, cudaStream_t s) {
    static_assert(kSlots * (select_row(SUBS) + kMaxChoices + kMaxGroups) * sizeof(float) <= 48 * 1024,
                  "shared memory that every launch may have");
    const int64_t want = (a.tokens + kSlots - 1) / kSlots;
    k_route_topk<T, SUBS, VEC><<<(unsigned)(want < (1 << 20) ? want : 1 << 20), kSelect,
                                 kSlots * (select_row(SUBS) + a.k + a.groups) * sizeof(float), s>>>(a);
    BGL_LAUNCH_CHECK();
    return BGL_OK;
}
template <typename T, int SUBS>
int launch_topk(const RouteArgs &a, cudaStream_t s) {
    const bool vec = a.experts % 4 == 0 && aligned(a.logits, 4 * sizeof(T));
    return vec ? launch_topk<T, SUBS, true>(a, s) : launch_topk<T, SUBS, false>(a, s);
}
// The fewest sets of 64 experts, doubled, that hold the row (a lane's registers grow with them).
template <typename T>
int launch_topk(const RouteArgs &a, cudaStream_t s) {
    if (a.experts <= 8 * kLanes * 1) return launch_topk<T, 1>(a, s);
    if (a.experts <= 8 * kLanes * 2) return launch_topk<T, 2>(a, s);
    if (a.experts <= 8 * kLanes * 4) return launch_topk<T, 4>(a, s);
    if (a.experts <= 8 * kLanes * 8) return launch_topk<T, 8>(a, s);
    return launch_topk<T, 16>(a, s);
}

template <typename T, int LANES, int PER>
void launch_backward(const RouteGradArgs &a, cudaStream_t s) {
    const bool vec = a.experts % 4 == 0 && aligned(a.logits, 4 * sizeof(T)) && aligned(a.dlogits, 4 * sizeof(T));
    constexpr int64_t slots = kWarps * 32 / LANES;
    const int64_t want = (a.tokens + slots - 1) / slots;
    const unsigned blocks = (unsigned)(want < (1 << 20) ? want : 1 << 20);
    if (vec) k_route_topk_backward<T, LANES, PER, true><<<blocks, kWarps * 32, 0, s>>>(a);
    else k_route_topk_backward<T, LANES, PER, false><<<blocks, kWarps * 32, 0, s>>>(a);
}
// Eight experts a lane while that leaves whole tokens to a warp.
template <typename T>
void launch_backward(const RouteGradArgs &a, cudaStream_t s) {
    if (a.experts <= 64) launch_backward<T, 8, 8>(a, s);
    else if (a.experts <= 128) launch_backward<T, 16, 8>(a, s);
    else if (a.experts <= 256) launch_backward<T, 32, 8>(a, s);
    else if (a.experts <= 512) launch_backward<T, 32, 16>(a, s);
    else launch_backward<T, 32, 32>(a, s);
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
    a.bias_aligned = aligned(bias, 16);
    a.scale = (float)scale;
    a.weights = weights;
    a.indices = indices;
    return dtype == BGL_F32 ? launch_topk<float>(a, as_stream(stream))
                            : launch_topk<__nv_bfloat16>(a, as_stream(stream));
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
    if (dtype == BGL_F32) launch_backward<float>(a, as_stream(stream));
    else launch_backward<__nv_bfloat16>(a, as_stream(stream));
    BGL_LAUNCH_CHECK();
    return BGL_OK;
}

}  // extern "C"
