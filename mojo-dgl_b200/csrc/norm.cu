// Layer norm over the last axis of a (rows, d) array, forward and backward.
//
//   y  = (x - mean) * rstd * w + b,    rstd = 1 / sqrt(mean((x - mean)^2) + eps)
//   v  = dy * w,  xhat = (x - mean) * rstd
//   dx = rstd * (v - mean(v) - xhat * mean(v * xhat))
//   dw = sum over rows of dy * xhat,   db = sum over rows of dy
//
// Memory bounds both, so a row is read once and stays in registers: a group of
// GROUP threads holds 8 or 16 values each (GROUP * that >= d), moved in 16-byte
// pieces where the row length and the addresses allow, and the variance is that
// of the centred values in registers, not a difference of sums.  Groups walk over
// rows with the next row's loads in flight while this one is reduced and written.
//
// A mean is off by a few units in its last place.  Where that shows (kFar), what the
// centred values add up to says by how much, and they are centred again: a row of equal
// values gave y up to 4 times w without it.  That is left for the end, where the rows
// that need it are read again (8192 x 4096 bf16: 35 us a call without such rows, 61 with
// one, 136 with all).  Doing it for every row, in the reduction of the squares, took 33.3
// -> 36.6 us; asking each row whether it needs it 31.6 -> 31.8 in the kernel (65536 x 509:
// 29.5 -> 31.5, 16384 x 2047 float32, which spilled before: 54.9 -> 47.4).
//
// Backward, the thread that holds a column of this row holds it of every row it
// walks over, so dw and db add up in registers beside dx and x and dy are read
// once for all three.  At the end a block leaves one partial row of each, which
// k_layer_norm_join adds in order: the same bits on every run.
//
// Rows longer than kMostHeld go through loops that read them again (from L2).
#include "after.cuh"
#include "rows.cuh"

namespace bgl {
namespace {

constexpr int kThreads = 256;
// A block has 256 threads, or one group where that is larger.
__host__ __device__ constexpr int threads_of(int group) { return group > kThreads ? group : kThreads; }
constexpr int kMostHeld = 8192;    // values of a row that registers hold
constexpr int kSplitRows = 256;    // longer rows: rows of one partial sum, at least
constexpr int kMaxSplits = 256;

// Two values that are worked on together.  float32 pairs go through the packed
// instructions (one issue for two operations, each rounded as alone): the bf16
// kernels are bound by issue, not by memory, without them.
template <typename A>
struct Pair {
    A x, y;
};
__device__ __forceinline__ unsigned long long bits(Pair<float> p) {
    unsigned long long r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(p.x), "f"(p.y));
    return r;
}
__device__ __forceinline__ Pair<float> pair(unsigned long long b) {
    Pair<float> p;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(p.x), "=f"(p.y) : "l"(b));
    return p;
}
__device__ __forceinline__ Pair<float> operator+(Pair<float> a, Pair<float> b) {
    unsigned long long r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits(a)), "l"(bits(b)));
    return pair(r);
}
__device__ __forceinline__ Pair<float> operator*(Pair<float> a, Pair<float> b) {
    unsigned long long r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits(a)), "l"(bits(b)));
    return pair(r);
}
__device__ __forceinline__ Pair<float> fma(Pair<float> a, Pair<float> b, Pair<float> c) {
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(bits(a)), "l"(bits(b)), "l"(bits(c)));
    return pair(r);
}
__device__ __forceinline__ Pair<double> operator+(Pair<double> a, Pair<double> b) { return {a.x + b.x, a.y + b.y}; }
__device__ __forceinline__ Pair<double> operator*(Pair<double> a, Pair<double> b) { return {a.x * b.x, a.y * b.y}; }
__device__ __forceinline__ Pair<double> fma(Pair<double> a, Pair<double> b, Pair<double> c) {
    return {::fma(a.x, b.x, c.x), ::fma(a.y, b.y, c.y)};
}
template <typename A>
__device__ __forceinline__ Pair<A> both(A v) { return {v, v}; }

// Values of a row as they are in memory: pieces of 16 bytes (VEC), or of two
// values that are moved one by one; the second one of a row's last piece may lie
// behind the row (`left` values remain), and is zero then.
template <typename T, bool VEC>
struct Piece {
    static constexpr int kWide = VEC ? 16 / (int)sizeof(T) : 2;
    static constexpr int kPairs = kWide / 2;
    union {
        uint4 raw;
        T v[kWide];
    };
    __device__ Piece() {}

    __device__ __forceinline__ void load(const T *p, int64_t left) {
        if constexpr (VEC) {
            raw = __ldcs(reinterpret_cast<const uint4 *>(p));
        } else {
            v[0] = p[0];
            v[1] = left > 1 ? p[1] : from_acc<T>(0);
        }
    }
    __device__ __forceinline__ void store(T *p, int64_t left) const {
        if constexpr (VEC) {
            __stcs(reinterpret_cast<uint4 *>(p), raw);
        } else {
            p[0] = v[0];
            if (left > 1) p[1] = v[1];
        }
    }
    __device__ __forceinline__ Pair<Acc<T>> get(int i) const { return {to_acc(v[2 * i]), to_acc(v[2 * i + 1])}; }
    __device__ __forceinline__ void set(int i, Pair<Acc<T>> p) {
        v[2 * i] = from_acc<T>(p.x), v[2 * i + 1] = from_acc<T>(p.y);
    }
};
template <>
__device__ __forceinline__ void Piece<__nv_bfloat16, true>::set(int i, Pair<float> p) {
    *reinterpret_cast<__nv_bfloat162 *>(&v[2 * i]) = __floats2bfloat162_rn(p.x, p.y);
}

// The parameters of a 16-byte piece at p, 16-byte aligned.
template <typename T, typename W>
__device__ __forceinline__ void load_params(const W *p, Pair<Acc<T>> (&v)[Piece<T, true>::kPairs]) {
    using A = Acc<T>;
    constexpr int kWide = 16 / (int)sizeof(W), kLoads = Piece<T, true>::kWide / kWide;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
        union {
            uint4 raw;
            W w[kWide];
        } u;
        u.raw = __ldg(reinterpret_cast<const uint4 *>(p) + i);
#pragma unroll
        for (int j = 0; j < kWide / 2; ++j)
            v[i * (kWide / 2) + j] = {A(to_acc(u.w[2 * j])), A(to_acc(u.w[2 * j + 1]))};
    }
}

// Sums over a group of GROUP threads, on each of them.  A group of more than a
// warp meets in `smem`, whose two halves are used in turn so that one barrier of
// the block is enough.
template <int GROUP, typename A>
__device__ __forceinline__ A lanes_sum(A v) {
#pragma unroll
    for (int o = (GROUP < 32 ? GROUP : 32) / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
template <int GROUP, int K, typename A>
__device__ __forceinline__ void group_sums(A (&v)[K], A (*smem)[K * (threads_of(GROUP) / 32)], int &turn) {
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = lanes_sum<GROUP>(v[k]);
    if constexpr (GROUP > 32) {
        const int warp = threadIdx.x >> 5, first = warp / (GROUP / 32) * (GROUP / 32);
#pragma unroll
        for (int k = 0; k < K; ++k)
            if ((threadIdx.x & 31) == 0) smem[turn][K * warp + k] = v[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] = 0;
#pragma unroll
        for (int i = 0; i < GROUP / 32; ++i)
#pragma unroll
            for (int k = 0; k < K; ++k) v[k] += smem[turn][K * (first + i) + k];
        turn ^= 1;
    }
}

// The same over one of the block's groups alone; what its threads wrote before comes
// before what they write after.
template <int GROUP, typename A>
__device__ __forceinline__ A lone_sum(A v, A (*smem)[threads_of(GROUP) / 32], int &turn) {
    constexpr int kLanes = GROUP < 32 ? GROUP : 32;
    const unsigned lanes = (0xffffffffu >> (32 - kLanes)) << (threadIdx.x & 31 & ~(kLanes - 1));
    __syncwarp(lanes);
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) v += __shfl_xor_sync(lanes, v, o);
    if constexpr (GROUP > 32) {
        const int group = threadIdx.x / GROUP;
        if ((threadIdx.x & 31) == 0) smem[turn][threadIdx.x >> 5] = v;
        asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "n"(GROUP) : "memory");
        v = 0;
        for (int i = 0; i < GROUP / 32; ++i) v += smem[turn][group * (GROUP / 32) + i];
        turn ^= 1;
    }
    return v;
}

// f(column, value) over the thread's columns of a row, four loads at a time.
template <int GROUP, typename T, typename F>
__device__ __forceinline__ void walk(const T *row, int t, int d, F &&f) {
#pragma unroll 1
    for (int i = t; i < d; i += 4 * GROUP) {
        T v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (i + j * GROUP < d) v[j] = row[i + j * GROUP];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (i + j * GROUP < d) f(i + j * GROUP, to_acc(v[j]));
    }
}

// Centres rows whose mean is more than kFar + 1 times their spread a second time: a
// group's own rows, from memory, once it has written all of them.  (It looks at them
// where one passes kFar, so what becomes of a row does not depend on the others.)
constexpr int kFar = 16;
template <int GROUP, typename T, typename W>
__device__ __forceinline__ void recentre(const T *x, const W *w, const W *b, int64_t row, int64_t rows, int64_t stride,
                                         int64_t d, Acc<T> eps, T *y, Acc<T> *mean, Acc<T> *rstd,
                                         Acc<T> (*smem)[threads_of(GROUP) / 32], int turn) {
    using A = Acc<T>;
    const int t = threadIdx.x % GROUP, n = (int)d;
    for (; row < rows; row += stride) {
        const T *from = x + row * d;
        A s = 0, q = 0, e = 0;
        walk<GROUP>(from, t, n, [&](int, A v) { s += v; });
        const A mu = lone_sum<GROUP>(s, smem, turn) / A(d);
        walk<GROUP>(from, t, n, [&](int, A v) { v -= mu, q += v * v, e += v; });
        q = lone_sum<GROUP>(q, smem, turn) / A(d);
        const A off = lone_sum<GROUP>(e, smem, turn) / A(d);
        if (!(fabs(mu) > A(kFar + 1) * sqrt(q + eps))) continue;
        q = 0;
        walk<GROUP>(from, t, n, [&](int, A v) { v = v - mu - off, q += v * v; });
        const A rs = A(1) / sqrt(lone_sum<GROUP>(q, smem, turn) / A(d) + eps);
        walk<GROUP>(from, t, n, [&](int i, A v) {
            v = (v - mu - off) * rs;
            if (w) v *= to_acc(w[i]);
            if (b) v += to_acc(b[i]);
            y[row * d + i] = from_acc<T>(v);
        });
        if (t == 0) {
            if (mean) mean[row] = mu + off;
            if (rstd) rstd[row] = rs;
        }
    }
}

// Blocks an SM that the forward pass is compiled for, and the grid filled with.
__host__ __device__ constexpr int forward_resident(int group, int values, int size) {
    return (size == 8 ? 3 : values == 8 ? 5 : 4) * kThreads / threads_of(group);
}

// A thread's columns in the rows of its group: piece i holds the values from
// column(i) on.  kShifted: the pieces are the aligned ones inside the row; what is
// before and behind them goes to the group's first threads, one value each (the
// thread's `extra` column).
template <typename T, int GROUP, int MODE>
struct Columns {
    using P = Piece<T, MODE != kScalar>;
    int t, head, end;  // first column of the pieces, and the one behind them
    int extra;         // -1: none

    __device__ __forceinline__ Columns(int64_t first_row, int64_t d) : t(threadIdx.x % GROUP), head(0), end((int)d), extra(-1) {
        if (MODE == kShifted) {
            head = (int)(-(uint64_t)(first_row * d) % P::kWide);
            if (head > d) head = (int)d;
            end = head + ((int)d - head) / P::kWide * P::kWide;
            if (t < head) extra = t;
            else if (t < head + (int)d - end) extra = end + t - head;
        }
    }
    __device__ __forceinline__ int column(int i) const { return head + (t + GROUP * i) * P::kWide; }
    __device__ __forceinline__ bool some(int i) const { return column(i) < end; }
    // kScalar: the second value of a pair may lie behind the row
    __device__ __forceinline__ bool one(int i) const { return MODE == kScalar && column(i) + 1 >= end; }
    __device__ __forceinline__ bool has_extra() const { return MODE == kShifted && extra >= 0; }

    __device__ __forceinline__ void load(P &p, const T *row, int i) const { p.load(row + column(i), end - column(i)); }
    __device__ __forceinline__ void store(const P &p, T *row, int i) const { p.store(row + column(i), end - column(i)); }
    // the parameters of piece i
    template <typename W>
    __device__ __forceinline__ void params(const W *w, int i, Pair<Acc<T>> (&v)[P::kPairs]) const {
        using A = Acc<T>;
        if constexpr (MODE == kAligned) {
            load_params<T>(w + column(i), v);
        } else {
#pragma unroll
            for (int j = 0; j < P::kPairs; ++j)
                v[j] = {A(to_acc(w[column(i) + 2 * j])), one(i) ? A(0) : A(to_acc(w[column(i) + 2 * j + 1]))};
        }
    }
};

// kShifted: the parameters of a thread's columns lie in shared memory, as the
// thread will read them.
template <typename T, int GROUP, int N, int MODE>
constexpr size_t forward_smem() {
    return MODE == kShifted ? (size_t)threads_of(GROUP) * N * sizeof(Acc<T>) * 2 : 0;
}

template <typename T, typename W, int GROUP, int N, int MODE>
__global__ void __launch_bounds__(threads_of(GROUP), forward_resident(GROUP, N, sizeof(T)))
    k_layer_norm(const T *__restrict__ x, const W *__restrict__ w, const W *__restrict__ b,
                 int64_t rows, int64_t d, Acc<T> eps, T *__restrict__ y, Acc<T> *__restrict__ mean,
                 Acc<T> *__restrict__ rstd) {
    using A = Acc<T>;
    using P = Piece<T, MODE != kScalar>;
    constexpr int kThreads = threads_of(GROUP), kGroups = kThreads / GROUP, kPieces = N / P::kWide;
    __shared__ A smem[2][kThreads / 32];
    extern __shared__ __align__(16) unsigned char raw[];
    Pair<A> *params = reinterpret_cast<Pair<A> *>(raw);  // [w, b][piece][pair][thread]
    int turn = 0;
    // (kShifted: the host gives a number of groups that keeps each to one shift)
    const int64_t stride = (int64_t)gridDim.x * kGroups, first = (int64_t)blockIdx.x * kGroups;
    int64_t row = first + threadIdx.x / GROUP;
    const Columns<T, GROUP, MODE> c(row, d);
    const A inv = A(1) / A(d);
    A extra_w = 1, extra_b = 0;
    if constexpr (MODE == kShifted) {
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            if (!c.some(i)) continue;
            Pair<A> p[P::kPairs];
            for (int which = 0; which < 2; ++which) {
                const W *from = which ? b : w;
                if (!from) continue;
                c.params(from, i, p);
#pragma unroll
                for (int j = 0; j < P::kPairs; ++j)
                    params[((which * kPieces + i) * P::kPairs + j) * kThreads + threadIdx.x] = p[j];
            }
        }
        if (c.has_extra()) {
            if (w) extra_w = to_acc(w[c.extra]);
            if (b) extra_b = to_acc(b[c.extra]);
        }
    }
    auto param = [&](const W *from, int which, int i, Pair<A>(&p)[P::kPairs]) {
        if constexpr (MODE == kShifted) {
#pragma unroll
            for (int j = 0; j < P::kPairs; ++j)
                p[j] = params[((which * kPieces + i) * P::kPairs + j) * kThreads + threadIdx.x];
        } else {
            c.params(from, i, p);
        }
    };
    P next[kPieces];
    T next_extra = from_acc<T>(0);
    auto fetch = [&](int64_t r) {
        if (r >= rows) return;
#pragma unroll
        for (int i = 0; i < kPieces; ++i)
            if (c.some(i)) c.load(next[i], x + r * d, i);
        if (c.has_extra()) next_extra = x[r * d + c.extra];
    };
    fetch(row);
    // whole groups take part in the block's barriers even behind the last row
    bool far = false;
    for (int64_t r0 = first; r0 < rows; r0 += stride, row += stride) {
        const bool live = row < rows;
        Pair<A> v[kPieces][P::kPairs];
        Pair<A> s = both(A(0));
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const bool some = c.some(i) && live;
#pragma unroll
            for (int j = 0; j < P::kPairs; ++j) {
                v[i][j] = some ? next[i].get(j) : both(A(0));
                s = s + v[i][j];
            }
        }
        A extra = 0;
        if (c.has_extra() && live) s.x += extra = to_acc(next_extra);
        fetch(row + stride);
        A sum[1] = {s.x + s.y};
        group_sums<GROUP>(sum, smem, turn);
        const A mu = sum[0] * inv;
        s = both(A(0));
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
#pragma unroll
            for (int j = 0; j < P::kPairs; ++j) v[i][j] = v[i][j] + both(-mu);
            if (!c.some(i)) continue;
            if (c.one(i)) v[i][0].y = 0;
#pragma unroll
            for (int j = 0; j < P::kPairs; ++j) s = fma(v[i][j], v[i][j], s);
        }
        extra -= mu;
        if (c.has_extra()) s.x += extra * extra;
        sum[0] = s.x + s.y;
        group_sums<GROUP>(sum, smem, turn);
        const A rs = A(1) / sqrt(sum[0] * inv + eps);
        if (!live) continue;
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            if (!c.some(i)) continue;
            Pair<A> p[P::kPairs];
#pragma unroll
            for (int j = 0; j < P::kPairs; ++j) v[i][j] = v[i][j] * both(rs);
            if (w) {
                param(w, 0, i, p);
#pragma unroll
                for (int j = 0; j < P::kPairs; ++j) v[i][j] = v[i][j] * p[j];
            }
            if (b) {
                param(b, 1, i, p);
#pragma unroll
                for (int j = 0; j < P::kPairs; ++j) v[i][j] = v[i][j] + p[j];
            }
            P o;
#pragma unroll
            for (int j = 0; j < P::kPairs; ++j) o.set(j, v[i][j]);
            c.store(o, y + row * d, i);
        }
        if (c.has_extra()) y[row * d + c.extra] = from_acc<T>(extra * rs * extra_w + extra_b);
        if (c.t == 0) {
            if (mean) mean[row] = mu;
            if (rstd) rstd[row] = rs;
        }
        far |= fabs(mu) * rs > A(kFar);
    }
    if (far) recentre<GROUP>(x, w, b, first + threadIdx.x / GROUP, rows, stride, d, eps, y, mean, rstd, smem, turn);
}

// Blocks an SM that the backward pass is compiled for (16384 x 4096 bf16: 89 us with two,
// 100 us with three; 131072 x 256: 54 us with two, 49 us with three).  Rows in aligned
// pieces do so without spills; bf16 ones of 8 values a thread spill 20 to 32 bytes at
// their 80 registers in the other modes, those of 16 values 48 to 72 by single values.
__host__ __device__ constexpr int backward_resident(int group, int values, int size) {
    return group > kThreads || size == 8 ? 1 : values == 8 && size == 2 ? 3 : 2;
}

// Rows of x and dy that are under way for each group: stages of a ring in
// shared memory, as many as the blocks of an SM have room for.  A thread copies
// and reads its own pieces only, so its cp.async groups are all the
// synchronisation there is.
template <typename T, int GROUP, int N>
__host__ __device__ constexpr int ring_stages() {
    constexpr int bytes = threads_of(GROUP) * 2 * N * (int)sizeof(T);
    constexpr int n = 196608 / backward_resident(GROUP, N, sizeof(T)) / bytes;
    return n > 4 ? 4 : n;
}
// kShifted: the weights of a thread's columns lie in shared memory, as the thread
// will read them (registers are short with the extra column's values beside).
template <typename T, int GROUP, int N, int MODE>
__host__ __device__ constexpr size_t backward_weights() {
    return MODE == kShifted ? (size_t)threads_of(GROUP) * N * sizeof(Acc<T>) : 0;
}
template <typename T, int GROUP, int N, int MODE>
constexpr size_t backward_smem() {
    // the ring, or the columns where the block's groups meet at the end
    const size_t ring = MODE != kScalar ? (size_t)ring_stages<T, GROUP, N>() * threads_of(GROUP) * 2 * N * sizeof(T) : 0;
    const size_t columns = GROUP < threads_of(GROUP) ? (size_t)GROUP * N * sizeof(Acc<T>) : 0;
    return (ring > columns ? ring : columns) + backward_weights<T, GROUP, N, MODE>();
}
// kShifted: this many blocks share a run of rows, so that each group's rows have
// one shift.
template <typename T>
__host__ __device__ constexpr int shift_blocks(int groups) {
    return 16 / (int)sizeof(T) > groups ? 16 / (int)sizeof(T) / groups : 1;
}

// partial: [gridDim.x][2][d], sums of dy * xhat and of dy over the block's rows, a
// consecutive run (or every shift_blocks-th of one)
template <typename T, typename W, int GROUP, int N, int MODE>
__global__ void __launch_bounds__(threads_of(GROUP), backward_resident(GROUP, N, sizeof(T)))
    k_layer_norm_backward(const T *__restrict__ dy, const T *__restrict__ x,
                          const Acc<T> *__restrict__ mean, const Acc<T> *__restrict__ rstd,
                          const W *__restrict__ w, int64_t rows, int64_t d, T *__restrict__ dx,
                          Acc<T> *__restrict__ partial) {
    using A = Acc<T>;
    using P = Piece<T, MODE != kScalar>;
    constexpr int kThreads = threads_of(GROUP), kGroups = kThreads / GROUP, kPieces = N / P::kWide;
    constexpr int kStages = ring_stages<T, GROUP, N>();
    constexpr int kShare = MODE == kShifted ? shift_blocks<T>(kGroups) : 1, kStep = kShare * kGroups;
    __shared__ A smem[2][2 * (kThreads / 32)];
    extern __shared__ __align__(16) unsigned char raw[];
    constexpr size_t kWeights = backward_weights<T, GROUP, N, MODE>();
    Pair<A> *weights = reinterpret_cast<Pair<A> *>(raw);      // kShifted: [piece][pair][thread]
    A *columns = reinterpret_cast<A *>(raw + kWeights);       // [d], after the rows
    uint4 *ring = reinterpret_cast<uint4 *>(raw + kWeights);  // [stage][x, dy][piece][thread]
    next_may_start();
    int turn = 0;
    const int64_t run = blockIdx.x / kShare, runs = gridDim.x / kShare;
    const int64_t begin = rows * run / runs, end = rows * (run + 1) / runs;
    const int count = (int)(end - begin), lead = (int)(blockIdx.x % kShare * kGroups + threadIdx.x / GROUP);
    const int64_t mine = begin + lead;  // this thread's first row
    const Columns<T, GROUP, MODE> c(mine, d);
    Pair<A> aw[kPieces][P::kPairs], ab[kPieces][P::kPairs];
    Pair<A> wv[MODE == kShifted ? 1 : kPieces][P::kPairs];
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
#pragma unroll
        for (int j = 0; j < P::kPairs; ++j) {
            aw[i][j] = ab[i][j] = both(A(0));
            wv[MODE == kShifted ? 0 : i][j] = both(A(1));
        }
        if (w && c.some(i)) c.params(w, i, wv[MODE == kShifted ? 0 : i]);
        if constexpr (MODE == kShifted)
#pragma unroll
            for (int j = 0; j < P::kPairs; ++j) weights[(i * P::kPairs + j) * kThreads + threadIdx.x] = wv[0][j];
    }
    auto weight = [&](int i, int j) {
        return MODE == kShifted ? weights[(i * P::kPairs + j) * kThreads + threadIdx.x] : wv[MODE == kShifted ? 0 : i][j];
    };
    const A extra_w = w && c.has_extra() ? to_acc(w[c.extra]) : A(1);
    A extra_aw = 0, extra_ab = 0;
    // values to the next row to fetch, and to the row at hand
    const int64_t step = kStep * d;
    int64_t fetched = mine * d, at = fetched;
    constexpr uint32_t kStageBytes = 2 * kPieces * kThreads * 16, kRing = kStages * kStageBytes;
    const uint32_t slot0 = smem_addr(ring + threadIdx.x);
    uint32_t into = 0, from = 0;  // bytes into the ring
    auto fetch = [&](int i_row) {
        if constexpr (MODE != kScalar) {
            if (i_row < count)
#pragma unroll
                for (int i = 0; i < kPieces; ++i) {
                    if (!c.some(i)) continue;
                    const uint32_t slot = slot0 + into + i * kThreads * 16;
                    cp_async<16>(slot, x + fetched + c.column(i));
                    cp_async<16>(slot + kPieces * kThreads * 16, dy + fetched + c.column(i));
                }
            cp_async_commit();  // an empty group where there is no row: the count stays
            fetched += step;
            into = into == kRing - kStageBytes ? 0 : into + kStageBytes;
        }
    };
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) fetch(lead + i * kStep);
    const A *mu_at = mean + mine, *rs_at = rstd + mine;
    const A inv = A(1) / A(d);
    A next_mu = lead < count ? *mu_at : A(0), next_rs = lead < count ? *rs_at : A(0);
    T next_ex = from_acc<T>(0), next_eg = from_acc<T>(0);  // the extra column's x and dy
    if (c.has_extra() && lead < count) next_ex = x[at + c.extra], next_eg = dy[at + c.extra];
    for (int r0 = 0; r0 < count; r0 += kStep, at += step) {
        const bool live = r0 + lead < count;
        P hx[kPieces], hg[kPieces];
        if constexpr (MODE != kScalar) {
            fetch(r0 + lead + (kStages - 1) * kStep);  // into the stage that was read last time
            cp_async_wait<kStages - 1>();
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                const uint4 *slot = ring + from / 16 + i * kThreads + threadIdx.x;
                hx[i].raw = slot[0];
                hg[i].raw = slot[kPieces * kThreads];
            }
            from = from == kRing - kStageBytes ? 0 : from + kStageBytes;
        } else if (live) {
#pragma unroll
            for (int i = 0; i < kPieces; ++i)
                if (c.some(i)) c.load(hx[i], x + at, i), c.load(hg[i], dy + at, i);
        }
        const Pair<A> mu = both(-next_mu), rs = both(next_rs);
        mu_at += kStep, rs_at += kStep;
        const A ex = (to_acc(next_ex) - next_mu) * next_rs, eg = to_acc(next_eg), ev = eg * extra_w;
        if (r0 + lead + kStep < count) {
            next_mu = *mu_at, next_rs = *rs_at;
            if (c.has_extra()) next_ex = x[at + step + c.extra], next_eg = dy[at + step + c.extra];
        }
        Pair<A> s1 = both(A(0)), s2 = both(A(0));
        // bf16: kept as they are worked out (unpacking them again costs more
        // than the registers); else worked out again
        constexpr bool kKeep = sizeof(T) == 2;
        Pair<A> xhat[kPieces][P::kPairs], v[kPieces][P::kPairs];
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            if (!c.some(i) || !live) continue;
#pragma unroll
            for (int j = 0; j < P::kPairs; ++j) {
                const Pair<A> g = hg[i].get(j);
                xhat[i][j] = (hx[i].get(j) + mu) * rs;
                v[i][j] = g * weight(i, j);
                aw[i][j] = fma(g, xhat[i][j], aw[i][j]);
                ab[i][j] = ab[i][j] + g;
                s1 = s1 + v[i][j];
                s2 = fma(v[i][j], xhat[i][j], s2);
            }
        }
        if (c.has_extra() && live) {
            extra_aw += eg * ex;
            extra_ab += eg;
            s1.x += ev;
            s2.x += ev * ex;
        }
        A sums[2] = {s1.x + s1.y, s2.x + s2.y};
        group_sums<GROUP>(sums, smem, turn);
        s1 = both(-sums[0] * inv);
        s2 = both(-sums[1] * inv);
        if (!live || !dx) continue;
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            if (!c.some(i)) continue;
            P o;
#pragma unroll
            for (int j = 0; j < P::kPairs; ++j) {
                if constexpr (!kKeep) {
                    xhat[i][j] = (hx[i].get(j) + mu) * rs;
                    v[i][j] = hg[i].get(j) * weight(i, j);
                }
                o.set(j, rs * fma(xhat[i][j], s2, v[i][j] + s1));
            }
            c.store(o, dx + at, i);
        }
        if (c.has_extra()) dx[at + c.extra] = from_acc<T>(rs.x * (ex * s2.x + (ev + s1.x)));
    }
    if constexpr (MODE != kScalar) cp_async_wait<0>();
    if (!partial) return;
    // the block's groups one after the other (kShifted: each with columns of its
    // own, so by column), then the block's row of partials
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        Pair<A>(&a)[kPieces][P::kPairs] = which ? ab : aw;
        A *out = partial + (blockIdx.x * 2 + which) * d;
        for (int g = 0; g < kGroups; ++g) {
            if constexpr (kGroups > 1) __syncthreads();
            if (threadIdx.x / GROUP != g) continue;
            const bool last = g == kGroups - 1;
            // (loads first: the compiler cannot tell them from the stores)
            A sum[kPieces][P::kWide];
#pragma unroll
            for (int i = 0; i < kPieces; ++i)
#pragma unroll
                for (int j = 0; j < P::kWide; ++j) {
                    sum[i][j] = j & 1 ? a[i][j / 2].y : a[i][j / 2].x;
                    if (kGroups > 1 && g > 0 && c.some(i) && !(j && c.one(i))) sum[i][j] += columns[c.column(i) + j];
                }
            A *to = last ? out : columns;
            if (c.has_extra()) {
                const A mine_extra = which ? extra_ab : extra_aw;
                to[c.extra] = kGroups > 1 && g > 0 ? mine_extra + columns[c.extra] : mine_extra;
            }
#pragma unroll
            for (int i = 0; i < kPieces; ++i)
#pragma unroll
                for (int j = 0; j < P::kWide; ++j)
                    if (c.some(i) && !(j && c.one(i))) to[c.column(i) + j] = sum[i][j];
        }
    }
}

// Rows of any length: one block a row, three passes.
template <typename T, typename W>
__global__ void __launch_bounds__(kThreads)
    k_layer_norm_long(const T *__restrict__ x, const W *__restrict__ w, const W *__restrict__ b,
                      int64_t rows, int64_t d, Acc<T> eps, T *__restrict__ y,
                      Acc<T> *__restrict__ mean, Acc<T> *__restrict__ rstd) {
    using A = Acc<T>;
    __shared__ A smem[32];
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const T *xr = x + row * d;
        A s = 0;
        for (int64_t i = threadIdx.x; i < d; i += blockDim.x) s += to_acc(xr[i]);
        const A mu = block_sum(s, smem) / A(d);
        auto spread = [&](A off) {
            s = 0;
            for (int64_t i = threadIdx.x; i < d; i += blockDim.x) {
                const A c = to_acc(xr[i]) - mu - off;
                s += c * c;
            }
            return A(1) / sqrt(block_sum(s, smem) / A(d) + eps);
        };
        A off = 0, rs = spread(off);
        if (fabs(mu) * rs > A(kFar)) {
            s = 0;
            for (int64_t i = threadIdx.x; i < d; i += blockDim.x) s += to_acc(xr[i]) - mu;
            off = block_sum(s, smem) / A(d);
            rs = spread(off);
        }
        for (int64_t i = threadIdx.x; i < d; i += blockDim.x) {
            A v = (to_acc(xr[i]) - mu - off) * rs;
            if (w) v *= to_acc(w[i]);
            if (b) v += to_acc(b[i]);
            y[row * d + i] = from_acc<T>(v);
        }
        if (threadIdx.x == 0) {
            if (mean) mean[row] = mu + off;
            if (rstd) rstd[row] = rs;
        }
    }
}

template <typename T, typename W>
__global__ void __launch_bounds__(kThreads)
    k_layer_norm_dx_long(const T *__restrict__ dy, const T *__restrict__ x,
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
__global__ void __launch_bounds__(kThreads)
    k_layer_norm_dw_long(const T *__restrict__ dy, const T *__restrict__ x,
                         const Acc<T> *__restrict__ mean, const Acc<T> *__restrict__ rstd,
                         int64_t rows, int64_t d, int64_t split_rows, Acc<T> *__restrict__ partial) {
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

// Adds the partial rows: 32 columns a block, the parts 32 ways, both in a fixed
// order.  blockIdx.y: 0 dw, 1 db.
template <typename A, typename W>
__global__ void __launch_bounds__(1024)
    k_layer_norm_join(const A *partial, int64_t parts, int64_t d, W *__restrict__ dw,
                      W *__restrict__ db) {
    __shared__ A sums[32][33];
    W *out = blockIdx.y ? db : dw;
    before_is_done();
    if (!out) return;
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const int64_t col = (int64_t)blockIdx.x * 32 + tx;
    A s = 0;
    if (col < d) {
        const A *p = partial + blockIdx.y * d + col;
#pragma unroll 8
        for (int64_t i = ty; i < parts; i += 32) s += p[i * 2 * d];
    }
    sums[ty][tx] = s;
    __syncthreads();
    s = warp_sum(sums[tx][ty]);  // warp ty adds column ty
    const int64_t mine = (int64_t)blockIdx.x * 32 + ty;
    if (tx == 0 && mine < d) out[mine] = from_acc<W>(Acc<W>(s));
}

int64_t split_rows_of(int64_t rows) {
    int64_t per = (rows + kMaxSplits - 1) / kMaxSplits;
    return per < kSplitRows ? kSplitRows : per;
}
int64_t splits_of(int64_t rows) { return (rows + split_rows_of(rows) - 1) / split_rows_of(rows); }

// How a row is held: a group of threads of 8 or 16 (float64: 8) values each.  The
// fewest threads that hold it: what a row costs beside its values (reductions,
// barriers, addresses) is counted in warps.  16384 x 4096 bf16 backward: 92 us
// with 256 threads of 16, 109 us with 512 of 8 (before the packed arithmetic).
struct Shape {
    int group, values;
};
Shape shape_of(int64_t d, int dtype) {
    // (16 threads at least where up to 14 values lie beside a row's pieces)
    const bool beside = dtype == BGL_BF16 && d % 8;
    const int most = dtype == BGL_F64 ? 8 : 16;
    if (d <= 8 * 8 && !beside) return {8, 8};
    if (d <= 16 * 8) return {16, 8};
    if (d <= 32 * 8) return {32, 8};
    int group = 32;
    while ((int64_t)group * most < d) group *= 2;
    return {group, most};
}
bool is_held(int64_t d, int dtype) { return d <= (dtype == BGL_F64 ? kMostHeld / 2 : kMostHeld); }

// Blocks of the backward pass, one partial row each: resident ones, a fixed
// number for a given device so that the sums keep their order.
int64_t backward_blocks(int64_t rows, int64_t d, int dtype) {
    const Shape shape = shape_of(d, dtype);
    const int groups = threads_of(shape.group) / shape.group;
    const int resident = backward_resident(shape.group, shape.values, (int)row_elem_size(dtype));
    const int64_t want = (rows + groups - 1) / groups, most = (int64_t)num_sms() * resident;
    // whole runs of the blocks that share one (shift_blocks: at most 8)
    return want < most ? (want + 7) / 8 * 8 : most / 8 * 8;
}
int64_t parts_of(int64_t rows, int64_t d, int dtype) {
    return is_held(d, dtype) ? backward_blocks(rows, d, dtype) : splits_of(rows);
}

int check_norm(const char *who, int64_t rows, int64_t d, int dtype, int wdtype) {
    if (!row_dtype(dtype)) return fail(BGL_E_UNSUPPORTED, "%s: dtype %d", who, dtype);
    if (wdtype != dtype && !(dtype == BGL_BF16 && wdtype == BGL_F32))
        return fail(BGL_E_UNSUPPORTED, "%s: weight dtype %d with dtype %d", who, wdtype, dtype);
    if (rows < 0 || d < 0) return fail(BGL_E_INVALID, "%s: negative size", who);
    if (d >= (int64_t(1) << 31)) return fail(BGL_E_UNSUPPORTED, "%s: d >= 2^31", who);
    return BGL_OK;
}

// Calls f with the group size and the values of a thread as constants.
template <int GROUP, int N>
struct Constant {
    static constexpr int group = GROUP, values = N;
};
template <typename T, typename F>
int with_shape(Shape s, F &&f) {
    constexpr int M = sizeof(T) == 8 ? 8 : 16;
    if (s.group == 8) return f(Constant<8, 8>());
    if (s.group == 16) return f(Constant<16, 8>());
    if (s.group == 32) return s.values == 8 ? f(Constant<32, 8>()) : f(Constant<32, M>());
    if (s.group == 64) return f(Constant<64, M>());
    if (s.group == 128) return f(Constant<128, M>());
    if (s.group == 256) return f(Constant<256, M>());
    return f(Constant<512, M>());
}

// Rows of whole 16-byte pieces, of shifted ones, or (where an array does not begin
// on 16 bytes) of single values.
template <typename T>
RowMode row_mode(int64_t d, bool arrays, bool params) {
    if (!arrays) return kScalar;
    return d * sizeof(T) % 16 == 0 && params ? kAligned : kShifted;
}

struct Forward {
    const void *x, *w, *b;
    int64_t rows, d;
    double eps;
    void *y, *mean, *rstd;
    int dtype;
    cudaStream_t s;
};
template <typename T, typename W>
int forward(const Forward &p) {
    using A = Acc<T>;
    const T *x = (const T *)p.x;
    const W *w = (const W *)p.w, *b = (const W *)p.b;
    T *y = (T *)p.y;
    A *mean = (A *)p.mean, *rstd = (A *)p.rstd;
    if (!is_held(p.d, p.dtype)) {
        const int64_t cap = (int64_t)num_sms() * 8;
        k_layer_norm_long<T, W><<<(unsigned)(p.rows < cap ? p.rows : cap), kThreads, 0, p.s>>>(
            x, w, b, p.rows, p.d, (A)p.eps, y, mean, rstd);
        BGL_LAUNCH_CHECK();
        return BGL_OK;
    }
    const RowMode mode = row_mode<T>(p.d, aligned(x, 16) && aligned(y, 16), aligned(w, 16) && aligned(b, 16));
    return with_shape<T>(shape_of(p.d, p.dtype), [&](auto c) {
        constexpr int G = decltype(c)::group, N = decltype(c)::values, threads = threads_of(G), per = threads / G;
        // one wave of resident blocks (888 blocks where 592 are resident: 38 us
        // for 8192 x 4096 bf16, against 33 us)
        const int64_t want = (p.rows + per - 1) / per, cap = (int64_t)num_sms() * forward_resident(G, N, sizeof(T));
        // (a multiple of 8 blocks keeps every group to rows of one shift)
        const unsigned grid = (unsigned)(want < cap ? want : cap / 8 * 8);
        if (mode == kAligned) {
            k_layer_norm<T, W, G, N, kAligned><<<grid, threads, 0, p.s>>>(x, w, b, p.rows, p.d, (A)p.eps, y, mean, rstd);
        } else if (mode == kShifted) {
            constexpr size_t smem = forward_smem<T, G, N, kShifted>();
            if (smem > 48 * 1024)
                BGL_CUDA(cudaFuncSetAttribute(k_layer_norm<T, W, G, N, kShifted>,
                                              cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
            k_layer_norm<T, W, G, N, kShifted><<<grid, threads, smem, p.s>>>(x, w, b, p.rows, p.d, (A)p.eps, y, mean, rstd);
        } else {
            k_layer_norm<T, W, G, N, kScalar><<<grid, threads, 0, p.s>>>(x, w, b, p.rows, p.d, (A)p.eps, y, mean, rstd);
        }
        BGL_LAUNCH_CHECK();
        return (int)BGL_OK;
    });
}

struct Backward {
    const void *dy, *x, *mean, *rstd, *w;
    int64_t rows, d;
    void *dx, *dw, *db, *ws;
    int dtype;
    cudaStream_t s;
};
template <typename T, typename W>
int backward(const Backward &p) {
    using A = Acc<T>;
    const T *dy = (const T *)p.dy, *x = (const T *)p.x;
    const A *mean = (const A *)p.mean, *rstd = (const A *)p.rstd;
    const W *w = (const W *)p.w;
    T *dx = (T *)p.dx;
    const bool sums = p.dw || p.db;
    const int64_t parts = parts_of(p.rows, p.d, p.dtype);
    Carver carver(p.ws);
    A *partial = sums ? carver.take<A>((size_t)(2 * parts * p.d)) : nullptr;
    if (p.rows && !is_held(p.d, p.dtype)) {
        const int64_t cap = (int64_t)num_sms() * 8;
        if (dx) {
            k_layer_norm_dx_long<T, W><<<(unsigned)(p.rows < cap ? p.rows : cap), kThreads, 0, p.s>>>(
                dy, x, mean, rstd, w, p.rows, p.d, dx);
            BGL_LAUNCH_CHECK();
        }
        if (sums) {
            dim3 grid((unsigned)((p.d + 31) / 32), (unsigned)parts);
            k_layer_norm_dw_long<T><<<grid, kThreads, 0, p.s>>>(dy, x, mean, rstd, p.rows, p.d,
                                                                split_rows_of(p.rows), partial);
            BGL_LAUNCH_CHECK();
        }
    } else if (p.rows && (dx || sums)) {
        const RowMode mode = row_mode<T>(p.d, aligned(x, 16) && aligned(dy, 16) && aligned(dx, 16), aligned(w, 16));
        const int rc = with_shape<T>(shape_of(p.d, p.dtype), [&](auto c) {
            constexpr int G = decltype(c)::group, N = decltype(c)::values, threads = threads_of(G);
            const unsigned grid = (unsigned)parts;
            auto launch = [&](auto kernel, size_t smem) {
                if (smem > 48 * 1024)
                    BGL_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
                kernel<<<grid, threads, smem, p.s>>>(dy, x, mean, rstd, w, p.rows, p.d, dx, partial);
                BGL_LAUNCH_CHECK();
                return (int)BGL_OK;
            };
            if (mode == kAligned) return launch(k_layer_norm_backward<T, W, G, N, kAligned>, backward_smem<T, G, N, kAligned>());
            if (mode == kShifted) return launch(k_layer_norm_backward<T, W, G, N, kShifted>, backward_smem<T, G, N, kShifted>());
            return launch(k_layer_norm_backward<T, W, G, N, kScalar>, backward_smem<T, G, N, kScalar>());
        });
        if (rc) return rc;
    }
    if (sums) {
        BGL_CUDA(launch_after(k_layer_norm_join<A, W>, dim3((unsigned)((p.d + 31) / 32), 2), 1024, 0, p.s,
                              partial, parts, p.d, (W *)p.dw, (W *)p.db));
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
    const Forward p = {x, weight, bias, rows, d, eps, y, mean, rstd, dtype, as_stream(stream)};
    if (dtype == BGL_F64) return forward<double, double>(p);
    if (dtype == BGL_F32) return forward<float, float>(p);
    return wdtype == BGL_F32 ? forward<__nv_bfloat16, float>(p) : forward<__nv_bfloat16, __nv_bfloat16>(p);
}

size_t bgl_layer_norm_backward_workspace_size(int64_t rows, int64_t d, int dtype) {
    if (rows < 0 || d < 0 || !row_dtype(dtype)) return 0;
    return (size_t)(2 * parts_of(rows, d, dtype) * d) * (dtype == BGL_F64 ? 8 : 4) + 256;
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
    const Backward p = {grad, x, mean, rstd, weight, rows, d, dx, dweight, dbias, workspace, dtype, as_stream(stream)};
    if (dtype == BGL_F64) return backward<double, double>(p);
    if (dtype == BGL_F32) return backward<float, float>(p);
    return wdtype == BGL_F32 ? backward<__nv_bfloat16, float>(p) : backward<__nv_bfloat16, __nv_bfloat16>(p);
}

}  // extern "C"
