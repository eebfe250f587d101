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
//
// Memory bounds the three of them: each reads a token's row once for its k
// choices, in 16-byte pieces where the row length and the addresses allow, the
// lanes of a token side by side over its row.
#include "after.cuh"
#include "rows.cuh"

namespace bgl {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxBins = 8192;  // experts + 1: shared-memory counters
constexpr int kCounters = 48 * 1024 / 4 - 32;  // of a block: 48 KB, less the sums of its warps
constexpr int kMaxChunks = 1024;

// ---------------------------------------------------------------- the plan
// Item i's bin: its expert, or `experts` (the last bin) for none.
__device__ __forceinline__ int bin_of(int64_t index, int experts) {
    return index >= 0 && index < experts ? (int)index : experts;
}

// A chunk of consecutive items goes to one block, an equal part of it to each of
// its warps, which counts and ranks 32 items a step.  As many warps as the
// counters of all of them leave room for.
struct Plan {
    int64_t items, chunks, per_warp;
    int experts, warps;
};
Plan plan_of(int64_t items, int64_t experts) {
    Plan p;
    p.items = items;
    p.experts = (int)experts;
    const int64_t room = kCounters / (experts + 1);
    p.warps = (int)(room < 8 ? room : 8);
    // 64 items a warp, more where that gave too many chunks; one chunk where 32
    // steps a warp are enough (one launch instead of three)
    int64_t steps = (items + p.warps * 32 * (int64_t)kMaxChunks - 1) / (p.warps * 32 * (int64_t)kMaxChunks);
    if (steps < 2) steps = 2;
    if (items <= p.warps * 32 * 32) steps = (items + p.warps * 32 - 1) / (p.warps * 32);
    p.per_warp = (steps > 0 ? steps : 1) * 32;
    p.chunks = (items + p.per_warp * p.warps - 1) / (p.per_warp * p.warps);
    return p;
}

// chunk_bins[bin][chunk] = items of the chunk in the bin
__global__ void __launch_bounds__(kThreads)
    k_plan_count(const Plan p, const int64_t *__restrict__ indices, int32_t *__restrict__ chunk_bins) {
    extern __shared__ int32_t bins[];
    next_may_start();
    for (int b = threadIdx.x; b <= p.experts; b += blockDim.x) bins[b] = 0;
    __syncthreads();
    const int64_t per = p.per_warp * p.warps, i0 = blockIdx.x * per;
    const int64_t i1 = i0 + per < p.items ? i0 + per : p.items;
    for (int64_t i = i0 + threadIdx.x; i < i1; i += blockDim.x)
        atomicAdd(&bins[bin_of(indices[i], p.experts)], 1);
    __syncthreads();
    for (int b = threadIdx.x; b <= p.experts; b += blockDim.x)
        chunk_bins[b * p.chunks + blockIdx.x] = bins[b];
}

// In place, for each bin the items in earlier chunks; the bin's total behind them.  A warp a bin.
__global__ void __launch_bounds__(kThreads)
    k_plan_scan(const Plan p, int32_t *__restrict__ chunk_bins, int32_t *__restrict__ totals,
                int64_t *__restrict__ counts) {
    const int lane = threadIdx.x & 31, bin = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
    next_may_start();
    before_is_done();
    if (bin > p.experts) return;
    int32_t sum = 0;
    for (int64_t c0 = 0; c0 < p.chunks; c0 += 32) {
        int32_t *at = chunk_bins + bin * p.chunks + c0 + lane;
        const int32_t n = c0 + lane < p.chunks ? *at : 0;
        int32_t scan = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int32_t up = __shfl_up_sync(0xffffffffu, scan, o);
            if (lane >= o) scan += up;
        }
        if (c0 + lane < p.chunks) *at = sum + scan - n;
        sum += __shfl_sync(0xffffffffu, scan, 31);
    }
    if (lane == 0) {
        totals[bin] = sum;
        if (bin < p.experts) counts[bin] = sum;
    }
}

// Rows of a chunk's items.  With one chunk, its own counts are the totals.
__global__ void __launch_bounds__(kThreads)
    k_plan_place(const Plan p, const int64_t *__restrict__ indices,
                 const int32_t *chunk_bins, const int32_t *totals,
                 int32_t *__restrict__ positions, int64_t *__restrict__ counts) {
    extern __shared__ int32_t next[];   // [warp][bin], at most kCounters
    __shared__ int32_t warp_sums[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, bins = p.experts + 1;
    for (int b = threadIdx.x; b < p.warps * bins; b += blockDim.x) next[b] = 0;
    __syncthreads();
    int32_t *mine = next + warp * bins;
    const int64_t i0 = (blockIdx.x * (int64_t)p.warps + warp) * p.per_warp;
    const int64_t i1 = i0 + p.per_warp < p.items ? i0 + p.per_warp : p.items;
#pragma unroll 4
    for (int64_t i = i0 + lane; i < i1; i += 32) atomicAdd(&mine[bin_of(indices[i], p.experts)], 1);
    __syncthreads();
    before_is_done();  // up to here the kernel needs no other's results
    // each bin's first row: all items of lower bins, those of its own in earlier
    // chunks, those of this chunk's earlier warps
    int32_t before = 0;
    for (int b0 = 0; b0 < bins; b0 += blockDim.x) {
        const int b = b0 + threadIdx.x;
        int32_t own = 0;
        if (b < bins) {
            for (int w = 0; w < p.warps; ++w) {
                const int32_t n = next[w * bins + b];
                next[w * bins + b] = own;
                own += n;
            }
            if (p.chunks > 1) own = totals[b];
            else if (b < p.experts) counts[b] = own;
        }
        int32_t scan = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int32_t up = __shfl_up_sync(0xffffffffu, scan, o);
            if (lane >= o) scan += up;
        }
        if (lane == 31) warp_sums[warp] = scan;
        __syncthreads();
        int32_t all = 0, lower = 0;
        for (int w = 0; w < p.warps; ++w) {
            if (w < warp) lower += warp_sums[w];
            all += warp_sums[w];
        }
        if (b < bins) {
            int32_t first = before + lower + scan - own;
            if (p.chunks > 1) first += chunk_bins[b * p.chunks + blockIdx.x];
            for (int w = 0; w < p.warps; ++w) next[w * bins + b] += first;
        }
        before += all;
        __syncthreads();
    }
    for (int64_t i = i0; i < i1; i += 32) {
        const bool in = i + lane < i1;
        const int bin = in ? bin_of(indices[i + lane], p.experts) : -1;
        const unsigned same = __match_any_sync(0xffffffffu, bin);
        const int earlier = __popc(same & ((1u << lane) - 1));
        const int32_t row = in ? mine[bin] + earlier : 0;
        __syncwarp();
        if (in && earlier == 0) mine[bin] = row + __popc(same);
        __syncwarp();
        if (in) positions[i + lane] = bin == p.experts ? ~row : row;
    }
}

// -------------------------------------------------------------------- rows
// Row of a position; false where the pair has no expert.  A position outside
// [0, total) is not one of a plan's: it gives row -1, which is not touched.
__device__ __forceinline__ bool row_of(int32_t position, int64_t total, int64_t &row) {
    row = position >= 0 ? position : ~position;
    if (row >= total) row = -1;
    return position >= 0 && row >= 0;
}

// Consecutive values of a row: 16 bytes, or one.
template <typename T, bool VEC>
struct Piece {
    static constexpr int kWide = VEC ? 16 / (int)sizeof(T) : 1;
    union {
        uint4 raw;
        T v[kWide];
    };
    __device__ Piece() {}
    __device__ __forceinline__ void load(const T *p) {
        if constexpr (VEC) raw = __ldg(reinterpret_cast<const uint4 *>(p));
        else v[0] = *p;
    }
    __device__ __forceinline__ void store(T *p) const {
        if constexpr (VEC) *reinterpret_cast<uint4 *>(p) = raw;
        else *p = v[0];
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < kWide; ++i) v[i] = from_acc<T>(0);
    }
};

// A row whose length is no multiple of 16 bytes, seen from the array it is written
// to: the aligned pieces inside it, and the values before and behind them.
template <typename T>
struct Inside {
    using P = Piece<T, true>;
    int64_t head, end, d;  // first value of the pieces, and the one behind them
    __device__ __forceinline__ Inside(int64_t row, int64_t d_) : d(d_) {
        head = (int64_t)(-(uint64_t)(row * d_) % P::kWide);
        if (head > d) head = d;
        end = head + (d - head) / P::kWide * P::kWide;
    }
    __device__ __forceinline__ int beside() const { return (int)(head + d - end); }
    __device__ __forceinline__ int64_t value(int i) const { return i < head ? i : end + i - head; }
};

// 16 bytes from any address: two aligned pieces, shifted into one once they are
// there.  `stop` is the end of the array; a piece that reached beyond it is put
// together from values.
template <typename T>
struct AnyPiece {
    uint4 lo, hi;
    unsigned shift;

    __device__ __forceinline__ void fetch(const T *from, const T *stop) {
        const uintptr_t at = reinterpret_cast<uintptr_t>(from);
        const uint4 *a = reinterpret_cast<const uint4 *>(at & ~uintptr_t(15));
        shift = (unsigned)(at & 15);
        if (reinterpret_cast<const T *>(a + 2) > stop) {
            Piece<T, true> p;
#pragma unroll
            for (int i = 0; i < Piece<T, true>::kWide; ++i) p.v[i] = from[i];
            lo = p.raw;
            shift = 0;
        } else {
            lo = __ldg(a);
            if (shift) hi = __ldg(a + 1);
        }
    }
    __device__ __forceinline__ Piece<T, true> get() const {
        Piece<T, true> p;
        uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
        if (shift & 8)
#pragma unroll
            for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
        if (shift & 4)
#pragma unroll
            for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
        if (sizeof(T) == 2) {
            const unsigned bits = (shift & 3) * 8;
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], bits);
        }
        p.raw = make_uint4(w[0], w[1], w[2], w[3]);
        return p;
    }
};
// Brings a row towards the SM before it is known which of its pieces are wanted.
template <typename T>
__device__ __forceinline__ void prefetch_row(const T *row, int64_t d, int thread, int threads) {
    for (int64_t e = thread * (128 / (int)sizeof(T)); e < d; e += threads * (128 / (int)sizeof(T)))
        asm volatile("prefetch.global.L1 [%0];" ::"l"(row + e));
}

// Rows of odd lengths (kShifted): as the kernels below, in the pieces of what is
// written; what is read lies at any shift to them.  20000 x 2 rows of 1023 bf16
// values: dispatch 81 -> 49 us, combine 84 -> 41, its gradient 88 -> 52 against
// single values.
template <typename T>
__global__ void __launch_bounds__(kThreads)
    k_dispatch_odd(const T *__restrict__ x, const int32_t *__restrict__ positions, int64_t tokens,
                   int k, int64_t d, T *__restrict__ rows) {
    using P = Piece<T, true>;
    const int64_t t = blockIdx.x * (int64_t)blockDim.y + threadIdx.y;
    if (t >= tokens) return;
    const T *from = x + t * d, *stop = x + tokens * d;
    prefetch_row(from, d, threadIdx.x, blockDim.x);
#pragma unroll 2
    for (int j = 0; j < k; ++j) {
        int64_t row;
        const bool sent = row_of(__ldg(positions + t * k + j), tokens * k, row);
        if (row < 0) continue;
        const Inside<T> in(row, d);
        T *to = rows + row * d;
        for (int64_t e = in.head + threadIdx.x * P::kWide; e < in.end; e += blockDim.x * P::kWide) {
            P v;
            v.zero();
            if (sent) {
                AnyPiece<T> any;
                any.fetch(from + e, stop);
                v = any.get();
            }
            v.store(to + e);
        }
        for (int i = threadIdx.x; i < in.beside(); i += blockDim.x)
            to[in.value(i)] = sent ? from[in.value(i)] : from_acc<T>(0);
    }
}

template <typename T, int kFlight>
__global__ void __launch_bounds__(kThreads)
    k_combine_odd(const T *__restrict__ rows, const int32_t *__restrict__ positions,
                  const Acc<T> *__restrict__ weights, int64_t tokens, int k, int64_t d,
                  T *__restrict__ y) {
    using A = Acc<T>;
    using P = Piece<T, true>;
    const int64_t t = blockIdx.x * (int64_t)blockDim.y + threadIdx.y;
    if (t >= tokens) return;
    const Inside<T> in(t, d);
    const T *stop = rows + tokens * k * d;
    T *to = y + t * d;
    // a value beside the pieces goes along with a thread's first piece (there are
    // fewer of them than threads with a piece)
    int64_t extra = (int)threadIdx.x < in.beside() ? in.value(threadIdx.x) : -1;
    for (int64_t e = in.head + threadIdx.x * P::kWide; e < in.end; e += blockDim.x * P::kWide, extra = -1) {
        A sum[P::kWide], extra_sum = 0;
#pragma unroll
        for (int i = 0; i < P::kWide; ++i) sum[i] = 0;
        for (int j0 = 0; j0 < k; j0 += kFlight) {  // rows under way
            AnyPiece<T> any[kFlight];
            T beside[kFlight];
            A w[kFlight];
            bool sent[kFlight];
#pragma unroll
            for (int j = 0; j < kFlight; ++j) {
                int64_t row;
                sent[j] = j0 + j < k && row_of(__ldg(positions + t * k + j0 + j), tokens * k, row);
                if (sent[j]) {
                    any[j].fetch(rows + row * d + e, stop);
                    if (extra >= 0) beside[j] = rows[row * d + extra];
                    w[j] = weights ? __ldg(weights + t * k + j0 + j) : A(1);
                }
            }
#pragma unroll
            for (int j = 0; j < kFlight; ++j) {
                if (!sent[j]) continue;
                const P v = any[j].get();
#pragma unroll
                for (int i = 0; i < P::kWide; ++i) sum[i] += w[j] * to_acc(v.v[i]);
                if (extra >= 0) extra_sum += w[j] * to_acc(beside[j]);
            }
        }
        P o;
#pragma unroll
        for (int i = 0; i < P::kWide; ++i) o.v[i] = from_acc<T>(sum[i]);
        o.store(to + e);
        if (extra >= 0) to[extra] = from_acc<T>(extra_sum);
    }
}

// blockDim.x threads over a row's pieces, blockDim.y tokens.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads)
    k_dispatch(const T *__restrict__ x, const int32_t *__restrict__ positions, int64_t tokens,
               int k, int64_t d, T *__restrict__ rows) {
    using P = Piece<T, VEC>;
    const int64_t t = blockIdx.x * (int64_t)blockDim.y + threadIdx.y;
    if (t >= tokens) return;
    const int32_t *pos = positions + t * k;
    P none;
    none.zero();
    for (int64_t e = threadIdx.x * P::kWide; e < d; e += blockDim.x * P::kWide) {
        P v;
        v.load(x + t * d + e);
#pragma unroll 4
        for (int j = 0; j < k; ++j) {
            int64_t row;
            const bool sent = row_of(__ldg(pos + j), tokens * k, row);
            if (row >= 0) (sent ? v : none).store(rows + row * d + e);
        }
    }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads)
    k_combine(const T *__restrict__ rows, const int32_t *__restrict__ positions,
              const Acc<T> *__restrict__ weights, int64_t tokens, int k, int64_t d,
              T *__restrict__ y) {
    using A = Acc<T>;
    using P = Piece<T, VEC>;
    constexpr int kFlight = 4;  // rows under way
    const int64_t t = blockIdx.x * (int64_t)blockDim.y + threadIdx.y;
    if (t >= tokens) return;
    const int32_t *pos = positions + t * k;
    for (int64_t e = threadIdx.x * P::kWide; e < d; e += blockDim.x * P::kWide) {
        A sum[P::kWide];
#pragma unroll
        for (int i = 0; i < P::kWide; ++i) sum[i] = 0;
        for (int j0 = 0; j0 < k; j0 += kFlight) {
            P v[kFlight];
            A w[kFlight];
            bool sent[kFlight];
#pragma unroll
            for (int j = 0; j < kFlight; ++j) {
                int64_t row;
                sent[j] = j0 + j < k && row_of(__ldg(pos + j0 + j), tokens * k, row);
                if (sent[j]) {
                    v[j].load(rows + row * d + e);
                    w[j] = weights ? __ldg(weights + t * k + j0 + j) : A(1);
                }
            }
#pragma unroll
            for (int j = 0; j < kFlight; ++j)
                if (sent[j])
#pragma unroll
                    for (int i = 0; i < P::kWide; ++i) sum[i] += w[j] * to_acc(v[j].v[i]);
        }
        P o;
#pragma unroll
        for (int i = 0; i < P::kWide; ++i) o.v[i] = from_acc<T>(sum[i]);
        o.store(y + t * d + e);
    }
}

// GROUP threads a token, `kFlight` choices at a time: dy is read once for them.
// Warps of a token need no barrier; their blocks are small, so that SMs even out.
__host__ __device__ constexpr int backward_threads(int group) { return group == 32 ? 128 : group; }

template <typename T, int GROUP, int kFlight, bool VEC>
__global__ void __launch_bounds__(backward_threads(GROUP))
    k_combine_backward(const T *__restrict__ dy, const T *__restrict__ rows,
                       const int32_t *__restrict__ positions, const Acc<T> *__restrict__ weights,
                       int64_t tokens, int k, int64_t d, T *__restrict__ drows,
                       Acc<T> *__restrict__ dweights) {
    using A = Acc<T>;
    using P = Piece<T, VEC>;
    __shared__ A smem[32];
    const int own = threadIdx.x % GROUP;
    const int64_t t = blockIdx.x * (int64_t)(backward_threads(GROUP) / GROUP) + threadIdx.x / GROUP;
    if (t >= tokens) return;  // whole groups; a group of a block is the block
    for (int j0 = 0; j0 < k; j0 += kFlight) {
        int64_t row[kFlight];
        bool sent[kFlight];
        A w[kFlight], dot[kFlight];
#pragma unroll
        for (int j = 0; j < kFlight; ++j) {
            row[j] = -1;
            sent[j] = j0 + j < k && row_of(__ldg(positions + t * k + j0 + j), tokens * k, row[j]);
            w[j] = !sent[j] ? A(0) : weights ? __ldg(weights + t * k + j0 + j) : A(1);
            dot[j] = 0;
        }
#pragma unroll 2
        for (int64_t e = own * P::kWide; e < d; e += GROUP * P::kWide) {
            P g, v[kFlight];
            g.load(dy + t * d + e);
#pragma unroll
            for (int j = 0; j < kFlight; ++j)
                if (dweights && sent[j]) v[j].load(rows + row[j] * d + e);
#pragma unroll
            for (int j = 0; j < kFlight; ++j) {
                if (row[j] < 0) continue;
                P o;
#pragma unroll
                for (int i = 0; i < P::kWide; ++i) {
                    const A gi = to_acc(g.v[i]);
                    if (dweights && sent[j]) dot[j] += gi * to_acc(v[j].v[i]);
                    o.v[i] = from_acc<T>(sent[j] ? w[j] * gi : A(0));
                }
                if (drows) o.store(drows + row[j] * d + e);
            }
        }
        if (!dweights) continue;
#pragma unroll
        for (int j = 0; j < kFlight; ++j) {
            if (j0 + j >= k) break;
            const A sum = GROUP == 32 ? warp_sum(dot[j]) : block_sum(dot[j], smem);
            if (own == 0) dweights[t * k + j0 + j] = sum;
        }
    }
}

// The same by GROUP threads a token for rows of odd lengths, a choice at a time.
template <typename T, int GROUP>
__global__ void __launch_bounds__(backward_threads(GROUP))
    k_combine_backward_odd(const T *__restrict__ dy, const T *__restrict__ rows,
                           const int32_t *__restrict__ positions, const Acc<T> *__restrict__ weights,
                           int64_t tokens, int k, int64_t d, T *__restrict__ drows,
                           Acc<T> *__restrict__ dweights) {
    using A = Acc<T>;
    using P = Piece<T, true>;
    __shared__ A smem[32];
    const int own = threadIdx.x % GROUP;
    const int64_t t = blockIdx.x * (int64_t)(backward_threads(GROUP) / GROUP) + threadIdx.x / GROUP;
    if (t >= tokens) return;  // whole groups; a group of a block is the block
    const T *from = dy + t * d, *stop = dy + tokens * d;
    prefetch_row(from, d, own, GROUP);
    for (int j = 0; j < k; ++j) {
        int64_t row;
        const bool sent = row_of(__ldg(positions + t * k + j), tokens * k, row);
        const A w = !sent ? A(0) : weights ? __ldg(weights + t * k + j) : A(1);
        const bool dots = dweights && sent;
        A dot = 0;
        if (row >= 0) {
            const Inside<T> in(row, d);
            const T *with = rows + row * d;
            T *to = drows + row * d;
            // the value beside the pieces (at most one a thread) is under way with them
            const int64_t extra = own < in.beside() ? in.value(own) : -1;
            T extra_g = from_acc<T>(0), extra_v = from_acc<T>(0);
            if (extra >= 0) {
                extra_g = from[extra];
                if (dots) extra_v = with[extra];
            }
#pragma unroll 2
            for (int64_t e = in.head + own * P::kWide; e < in.end; e += GROUP * P::kWide) {
                AnyPiece<T> any;
                any.fetch(from + e, stop);
                P v, o;
                if (dots) v.load(with + e);
                const P g = any.get();
#pragma unroll
                for (int i = 0; i < P::kWide; ++i) {
                    const A gi = to_acc(g.v[i]);
                    if (dots) dot += gi * to_acc(v.v[i]);
                    o.v[i] = from_acc<T>(sent ? w * gi : A(0));
                }
                if (drows) o.store(to + e);
            }
            if (extra >= 0) {
                const A gi = to_acc(extra_g);
                if (dots) dot += gi * to_acc(extra_v);
                if (drows) to[extra] = from_acc<T>(sent ? w * gi : A(0));
            }
        }
        if (dweights) {
            const A sum = GROUP == 32 ? warp_sum(dot) : block_sum(dot, smem);
            if (own == 0) dweights[t * k + j] = sum;
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

// Threads over a row's pieces and tokens of a block: a power of two of threads, 8
// to 256, that no row leaves mostly idle.
dim3 row_block(int64_t pieces) {
    unsigned x = 8;
    while (x < pieces && x < kThreads) x *= 2;
    return dim3(x, kThreads / x);
}
// (below 16 pieces a row, what is beside them costs more than the pieces save)
template <typename T>
RowMode row_mode(int64_t d, const void *a, const void *b, const void *c = nullptr) {
    if (!aligned(a, 16) || !aligned(b, 16) || !aligned(c, 16)) return kScalar;
    if (d * sizeof(T) % 16 == 0) return kAligned;
    return d * sizeof(T) >= 256 ? kShifted : kScalar;
}
unsigned token_blocks(int64_t tokens, unsigned per) { return (unsigned)((tokens + per - 1) / per); }

struct Rows {
    const void *in, *rows;
    const int32_t *positions;
    const void *weights;
    int64_t tokens, d;
    int k;
    void *out, *dweights;
    cudaStream_t s;
};
template <typename T>
int dispatch_as(const Rows &p) {
    const RowMode mode = row_mode<T>(p.d, p.in, p.out);
    const dim3 block = row_block(mode == kScalar ? p.d : p.d * (int64_t)sizeof(T) / 16);
    const unsigned grid = token_blocks(p.tokens, block.y);
    auto launch = [&](auto kernel) {
        kernel<<<grid, block, 0, p.s>>>((const T *)p.in, p.positions, p.tokens, p.k, p.d, (T *)p.out);
        BGL_LAUNCH_CHECK();
        return (int)BGL_OK;
    };
    return mode == kAligned ? launch(k_dispatch<T, true>) : mode == kShifted ? launch(k_dispatch_odd<T>) : launch(k_dispatch<T, false>);
}
template <typename T>
int combine_as(const Rows &p) {
    RowMode mode = row_mode<T>(p.d, p.rows, p.out);
    // values of 4 and 8 bytes move about as fast one by one as in pieces that have
    // to be shifted (float32, 6 rows of 1031 a token: 72 us against 111; bf16: 72
    // against 49)
    if (mode == kShifted && sizeof(T) > 2) mode = kScalar;
    const dim3 block = row_block(mode == kScalar ? p.d : p.d * (int64_t)sizeof(T) / 16);
    const unsigned grid = token_blocks(p.tokens, block.y);
    auto launch = [&](auto kernel) {
        kernel<<<grid, block, 0, p.s>>>((const T *)p.rows, p.positions, (const Acc<T> *)p.weights, p.tokens, p.k, p.d, (T *)p.out);
        BGL_LAUNCH_CHECK();
        return (int)BGL_OK;
    };
    if (mode == kAligned) return launch(k_combine<T, true>);
    if constexpr (sizeof(T) == 2)
        if (mode == kShifted) return p.k <= 2 ? launch(k_combine_odd<T, 2>) : launch(k_combine_odd<T, 4>);
    return launch(k_combine<T, false>);
}
template <typename T, int GROUP, int FLIGHT>
int combine_backward_as(const Rows &p) {
    constexpr int threads = backward_threads(GROUP);
    const RowMode mode = row_mode<T>(p.d, p.in, p.rows, p.out);
    const unsigned grid = token_blocks(p.tokens, threads / GROUP);
    auto launch = [&](auto kernel) {
        kernel<<<grid, threads, 0, p.s>>>((const T *)p.in, (const T *)p.rows, p.positions, (const Acc<T> *)p.weights, p.tokens,
                                          p.k, p.d, (T *)p.out, (Acc<T> *)p.dweights);
        BGL_LAUNCH_CHECK();
        return (int)BGL_OK;
    };
    if (mode == kAligned) return launch(k_combine_backward<T, GROUP, FLIGHT, true>);
    if (mode == kShifted) return launch(k_combine_backward_odd<T, GROUP>);
    return launch(k_combine_backward<T, GROUP, FLIGHT, false>);
}
template <typename T>
int combine_backward_as(const Rows &p) {
    // a warp a token, a block where there are too few tokens for that
    if (p.tokens < (int64_t)num_sms() * 16) return combine_backward_as<T, kThreads, 4>(p);
    // two choices need few registers, and more warps then fit
    return p.k <= 2 ? combine_backward_as<T, 32, 2>(p) : combine_backward_as<T, 32, 4>(p);
}

}  // namespace
}  // namespace bgl

using namespace bgl;

extern "C" {

size_t bgl_expert_plan_workspace_size(int64_t items, int64_t experts) {
    if (items < 0 || experts < 1 || experts >= kMaxBins) return 0;
    const Plan p = plan_of(items, experts);
    return p.chunks > 1 ? (size_t)(p.chunks + 1) * (experts + 1) * sizeof(int32_t) + 512 : 0;
}

int bgl_expert_plan(const int64_t *indices, int64_t items, int64_t experts, int64_t *counts,
                    int32_t *positions, void *workspace, size_t workspace_bytes, void *stream) {
    if (items < 0 || experts < 1) return fail(BGL_E_INVALID, "bgl_expert_plan: bad size");
    if (items >= (int64_t(1) << 31)) return fail(BGL_E_UNSUPPORTED, "bgl_expert_plan: 2^31 items or more");
    if (experts >= kMaxBins)
        return fail(BGL_E_UNSUPPORTED, "bgl_expert_plan: more than %d experts", kMaxBins - 1);
    if (!counts || (items && (!indices || !positions)))
        return fail(BGL_E_INVALID, "bgl_expert_plan: null buffer");
    const size_t need = bgl_expert_plan_workspace_size(items, experts);
    if (need && (!workspace || workspace_bytes < need))
        return fail(BGL_E_WORKSPACE, "bgl_expert_plan: workspace too small");
    cudaStream_t s = as_stream(stream);
    const Plan p = plan_of(items, experts);
    int32_t *chunk_bins = nullptr, *totals = nullptr;
    if (p.chunks > 1) {
        Carver c(workspace);
        chunk_bins = c.take<int32_t>((size_t)p.chunks * (experts + 1));
        totals = c.take<int32_t>((size_t)experts + 1);
        k_plan_count<<<(unsigned)p.chunks, kThreads, (experts + 1) * sizeof(int32_t), s>>>(p, indices, chunk_bins);
        BGL_LAUNCH_CHECK();
        BGL_CUDA(launch_after(k_plan_scan, (unsigned)((experts + 8) / 8), kThreads, 0, s, p, chunk_bins, totals, counts));
    }
    const unsigned chunks = (unsigned)(p.chunks > 0 ? p.chunks : 1), threads = p.warps * 32;
    const size_t smem = p.warps * (experts + 1) * sizeof(int32_t);
    if (p.chunks > 1)
        BGL_CUDA(launch_after(k_plan_place, chunks, threads, smem, s, p, indices, chunk_bins, totals, positions, counts));
    else
        k_plan_place<<<chunks, threads, smem, s>>>(p, indices, chunk_bins, totals, positions, counts);
    BGL_LAUNCH_CHECK();
    return BGL_OK;
}

int bgl_dispatch_rows(const void *x, const int32_t *positions, int64_t tokens, int64_t k,
                      int64_t d, void *rows, int dtype, void *stream) {
    int rc = check_rows("bgl_dispatch_rows", tokens, k, d, dtype);
    if (rc) return rc;
    if (tokens == 0 || k == 0 || d == 0) return BGL_OK;
    if (!x || !positions || !rows) return fail(BGL_E_INVALID, "bgl_dispatch_rows: null buffer");
    const Rows p = {x, nullptr, positions, nullptr, tokens, d, (int)k, rows, nullptr, as_stream(stream)};
    if (dtype == BGL_F64) return dispatch_as<double>(p);
    return dtype == BGL_F32 ? dispatch_as<float>(p) : dispatch_as<__nv_bfloat16>(p);
}

int bgl_combine_rows(const void *rows, const int32_t *positions, const void *weights,
                     int64_t tokens, int64_t k, int64_t d, void *y, int dtype, void *stream) {
    int rc = check_rows("bgl_combine_rows", tokens, k, d, dtype);
    if (rc) return rc;
    if (tokens == 0 || d == 0) return BGL_OK;
    if (!y || (k && (!rows || !positions))) return fail(BGL_E_INVALID, "bgl_combine_rows: null buffer");
    const Rows p = {nullptr, rows, positions, weights, tokens, d, (int)k, y, nullptr, as_stream(stream)};
    if (dtype == BGL_F64) return combine_as<double>(p);
    return dtype == BGL_F32 ? combine_as<float>(p) : combine_as<__nv_bfloat16>(p);
}

int bgl_combine_rows_backward(const void *grad, const void *rows, const int32_t *positions,
                              const void *weights, int64_t tokens, int64_t k, int64_t d,
                              void *drows, void *dweights, int dtype, void *stream) {
    int rc = check_rows("bgl_combine_rows_backward", tokens, k, d, dtype);
    if (rc) return rc;
    if (tokens == 0 || k == 0) return BGL_OK;
    if (!positions || (d && (!grad || (dweights && !rows))))
        return fail(BGL_E_INVALID, "bgl_combine_rows_backward: null buffer");
    const Rows p = {grad, rows, positions, weights, tokens, d, (int)k, drows, dweights, as_stream(stream)};
    if (dtype == BGL_F64) return combine_backward_as<double>(p);
    return dtype == BGL_F32 ? combine_backward_as<float>(p) : combine_backward_as<__nv_bfloat16>(p);
}

}  // extern "C"
