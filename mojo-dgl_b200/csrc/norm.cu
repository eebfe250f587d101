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
// Backward, the thread that holds a column of this row holds it of every row it
// walks over, so dw and db add up in registers beside dx and x and dy are read
// once for all three.  At the end a block leaves one partial row of each, which
// k_layer_norm_join adds in order: the same bits on every run.
//
// Rows longer than kMostHeld go through loops that read them again (from L2).
#include "rows.cuh"

namespace bgl {
namespace {

constexpr int kThreads = 256;
constexpr int kMostHeld = 8192;    // values of a row that registers hold
constexpr int kSplitRows = 256;    // longer rows: rows of one partial sum, at least
constexpr int kMaxSplits = 256;

// `N` values at p, 16 bytes at a time where VEC; as they are in memory, so that
// loads in flight take few registers.
template <typename T, int N, bool VEC>
struct Held {
    static constexpr int kWide = VEC ? 16 / (int)sizeof(T) : 1;
    static constexpr int kPieces = N / kWide;
    union Piece {
        uint4 raw;
        T v[kWide];
        __device__ Piece() {}
    };
    Piece p[kPieces];

    // piece i of thread t of a group: values (t + GROUP i) * kWide and on
    template <int GROUP>
    __device__ __forceinline__ void load(const T *row, int t, int64_t d) {
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const int64_t e = (int64_t)(t + GROUP * i) * kWide;
            if (e < d) {
                if constexpr (VEC) p[i].raw = __ldcs(reinterpret_cast<const uint4 *>(row + e));
                else p[i].v[0] = row[e];
            }
        }
    }
    __device__ __forceinline__ Acc<T> at(int i, int j) const { return to_acc(p[i].v[j]); }
};

// N values of the parameters at p, in 16-byte pieces where VEC.
template <typename W, int N, bool VEC, typename A>
__device__ __forceinline__ void load_params(const W *p, A (&v)[N]) {
    if constexpr (VEC) {
        constexpr int kWide = 16 / (int)sizeof(W);
        static_assert(N % kWide == 0, "whole 16-byte pieces");
#pragma unroll
        for (int i = 0; i < N / kWide; ++i) {
            union {
                uint4 raw;
                W w[kWide];
            } u;
            u.raw = __ldg(reinterpret_cast<const uint4 *>(p) + i);
#pragma unroll
            for (int j = 0; j < kWide; ++j) v[i * kWide + j] = A(to_acc(u.w[j]));
        }
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = A(to_acc(p[j]));
    }
}

// Sum over a group of GROUP threads, on each of them.  Groups of more than a
// warp are whole blocks' halves, or blocks: `smem` has two values a warp, used in
// turn so that one barrier a sum is enough.
template <int GROUP, typename A>
__device__ __forceinline__ A group_sum(A v, A (*smem)[kThreads / 32 + 1], int &turn) {
    v = warp_sum(v);
    if constexpr (GROUP > 32) {
        const int warp = threadIdx.x >> 5, first = warp / (GROUP / 32) * (GROUP / 32);
        if ((threadIdx.x & 31) == 0) smem[turn][warp] = v;
        __syncthreads();
        v = 0;
#pragma unroll
        for (int i = 0; i < GROUP / 32; ++i) v += smem[turn][first + i];
        turn ^= 1;
    }
    return v;
}

// Both sums at once, with one barrier.
template <int GROUP, typename A>
__device__ __forceinline__ void group_sums(A &u, A &v, A (*smem)[2 * (kThreads / 32)], int &turn) {
    u = warp_sum(u);
    v = warp_sum(v);
    if constexpr (GROUP > 32) {
        const int warp = threadIdx.x >> 5, first = warp / (GROUP / 32) * (GROUP / 32);
        if ((threadIdx.x & 31) == 0) smem[turn][2 * warp] = u, smem[turn][2 * warp + 1] = v;
        __syncthreads();
        u = v = 0;
#pragma unroll
        for (int i = 0; i < GROUP / 32; ++i) u += smem[turn][2 * (first + i)], v += smem[turn][2 * (first + i) + 1];
        turn ^= 1;
    }
}

template <typename T, typename W, int GROUP, int N, bool VEC>
__global__ void __launch_bounds__(kThreads)
    k_layer_norm(const T *__restrict__ x, const W *__restrict__ w, const W *__restrict__ b,
                 int64_t rows, int64_t d, Acc<T> eps, T *__restrict__ y, Acc<T> *__restrict__ mean,
                 Acc<T> *__restrict__ rstd) {
    using A = Acc<T>;
    using H = Held<T, N, VEC>;
    constexpr int kGroups = kThreads / GROUP;
    __shared__ A smem[2][kThreads / 32 + 1];
    int turn = 0;
    const int t = threadIdx.x % GROUP;
    const int64_t stride = (int64_t)gridDim.x * kGroups;
    // whole groups take part in the block's barriers even behind the last row
    const int64_t first = (int64_t)blockIdx.x * kGroups;
    H next;
    int64_t row = first + threadIdx.x / GROUP;
    if (row < rows) next.template load<GROUP>(x + row * d, t, d);
    for (int64_t r0 = first; r0 < rows; r0 += stride, row += stride) {
        const H h = next;
        if (row + stride < rows) next.template load<GROUP>(x + (row + stride) * d, t, d);
        A v[H::kPieces][H::kWide];
        A s = 0;
#pragma unroll
        for (int i = 0; i < H::kPieces; ++i) {
            const bool in = (int64_t)(t + GROUP * i) * H::kWide < d && row < rows;
#pragma unroll
            for (int j = 0; j < H::kWide; ++j) {
                v[i][j] = in ? h.at(i, j) : A(0);
                s += v[i][j];
            }
        }
        const A mu = group_sum<GROUP>(s, smem, turn) / A(d);
        s = 0;
#pragma unroll
        for (int i = 0; i < H::kPieces; ++i) {
            const bool in = (int64_t)(t + GROUP * i) * H::kWide < d;
#pragma unroll
            for (int j = 0; j < H::kWide; ++j) {
                v[i][j] -= mu;
                if (in) s += v[i][j] * v[i][j];
            }
        }
        const A rs = A(1) / sqrt(group_sum<GROUP>(s, smem, turn) / A(d) + eps);
        if (row >= rows) continue;
#pragma unroll
        for (int i = 0; i < H::kPieces; ++i) {
            const int64_t e = (int64_t)(t + GROUP * i) * H::kWide;
            if (e >= d) continue;
            A p[H::kWide];
#pragma unroll
            for (int j = 0; j < H::kWide; ++j) v[i][j] *= rs;
            if (w) {
                load_params<W, H::kWide, VEC>(w + e, p);
#pragma unroll
                for (int j = 0; j < H::kWide; ++j) v[i][j] *= p[j];
            }
            if (b) {
                load_params<W, H::kWide, VEC>(b + e, p);
#pragma unroll
                for (int j = 0; j < H::kWide; ++j) v[i][j] += p[j];
            }
            typename H::Piece o;
#pragma unroll
            for (int j = 0; j < H::kWide; ++j) o.v[j] = from_acc<T>(v[i][j]);
            if constexpr (VEC) __stcs(reinterpret_cast<uint4 *>(y + row * d + e), o.raw);
            else y[row * d + e] = o.v[0];
        }
        if (t == 0) {
            if (mean) mean[row] = mu;
            if (rstd) rstd[row] = rs;
        }
    }
}

// Rows of x and dy that are under way for each group: stages of a ring in
// shared memory, as many as two blocks an SM (one, of rows of 32 values a thread)
// have room for.  A thread copies and reads its own pieces only, so its
// cp.async groups are all the synchronisation there is.
template <typename T, int N>
__host__ __device__ constexpr int ring_stages() {
    constexpr int bytes = kThreads * 2 * N * (int)sizeof(T);
    constexpr int n = (N * (int)sizeof(T) > 64 ? 196608 : 98304) / bytes;
    return n > 4 ? 4 : n;
}
template <typename T, int GROUP, int N, bool VEC>
constexpr size_t backward_smem() {
    // the ring, or the columns where the block's groups meet at the end
    const size_t ring = VEC ? (size_t)ring_stages<T, N>() * kThreads * 2 * N * sizeof(T) : 0;
    const size_t columns = GROUP < kThreads ? (size_t)GROUP * N * sizeof(Acc<T>) : 0;
    return ring > columns ? ring : columns;
}

// partial: [gridDim.x][2][d], sums of dy * xhat and of dy over the block's rows,
// which are consecutive
template <typename T, typename W, int GROUP, int N, bool VEC>
__global__ void __launch_bounds__(kThreads)
    k_layer_norm_backward(const T *__restrict__ dy, const T *__restrict__ x,
                          const Acc<T> *__restrict__ mean, const Acc<T> *__restrict__ rstd,
                          const W *__restrict__ w, int64_t rows, int64_t d, T *__restrict__ dx,
                          Acc<T> *__restrict__ partial) {
    using A = Acc<T>;
    using H = Held<T, N, VEC>;
    constexpr int kGroups = kThreads / GROUP, kStages = ring_stages<T, N>();
    __shared__ A smem[2][2 * (kThreads / 32)];
    extern __shared__ __align__(16) unsigned char raw[];
    A *columns = reinterpret_cast<A *>(raw);  // [GROUP * N], after the rows
    uint4 *ring = reinterpret_cast<uint4 *>(raw);  // [stage][x, dy][piece][thread]
    int turn = 0;
    const int t = threadIdx.x % GROUP;
    const int64_t begin = rows * blockIdx.x / gridDim.x, end = rows * (blockIdx.x + 1) / gridDim.x;
    A aw[H::kPieces][H::kWide], ab[H::kPieces][H::kWide], wv[H::kPieces][H::kWide];
#pragma unroll
    for (int i = 0; i < H::kPieces; ++i) {
        const int64_t e = (int64_t)(t + GROUP * i) * H::kWide;
#pragma unroll
        for (int j = 0; j < H::kWide; ++j) aw[i][j] = ab[i][j] = 0, wv[i][j] = 1;
        if (w && e < d) load_params<W, H::kWide, VEC>(w + e, wv[i]);
    }
    int64_t row = begin + threadIdx.x / GROUP;
    auto fetch = [&](int64_t r, int stage) {
        if constexpr (VEC) {
            if (r < end)
#pragma unroll
                for (int i = 0; i < H::kPieces; ++i) {
                    const int64_t e = (int64_t)(t + GROUP * i) * H::kWide;
                    if (e >= d) continue;
                    uint4 *slot = ring + ((stage * 2) * H::kPieces + i) * kThreads + threadIdx.x;
                    cp_async<16>(smem_addr(slot), x + r * d + e);
                    cp_async<16>(smem_addr(slot + H::kPieces * kThreads), dy + r * d + e);
                }
            cp_async_commit();  // an empty group where there is no row: the count stays
        }
    };
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) fetch(row + i * kGroups, i);
    int stage = 0;
    A next_mu = row < end ? mean[row] : A(0), next_rs = row < end ? rstd[row] : A(0);
    for (int64_t r0 = begin; r0 < end; r0 += kGroups, row += kGroups) {
        const bool live = row < end;
        H hx, hg;
        if constexpr (VEC) {
            // into the stage that was read last time
            fetch(row + (kStages - 1) * kGroups, stage == 0 ? kStages - 1 : stage - 1);
            cp_async_wait<kStages - 1>();
#pragma unroll
            for (int i = 0; i < H::kPieces; ++i) {
                const uint4 *slot = ring + ((stage * 2) * H::kPieces + i) * kThreads + threadIdx.x;
                hx.p[i].raw = slot[0];
                hg.p[i].raw = slot[H::kPieces * kThreads];
            }
            stage = stage == kStages - 1 ? 0 : stage + 1;
        } else if (live) {
            hx.template load<GROUP>(x + row * d, t, d);
            hg.template load<GROUP>(dy + row * d, t, d);
        }
        const A mu = next_mu, rs = next_rs;
        if (row + kGroups < end) next_mu = mean[row + kGroups], next_rs = rstd[row + kGroups];
        A s1 = 0, s2 = 0;
#pragma unroll
        for (int i = 0; i < H::kPieces; ++i) {
            if ((int64_t)(t + GROUP * i) * H::kWide >= d || !live) continue;
#pragma unroll
            for (int j = 0; j < H::kWide; ++j) {
                const A g = hg.at(i, j), xhat = (hx.at(i, j) - mu) * rs, v = g * wv[i][j];
                aw[i][j] += g * xhat;
                ab[i][j] += g;
                s1 += v;
                s2 += v * xhat;
            }
        }
        group_sums<GROUP>(s1, s2, smem, turn);
        s1 /= A(d);
        s2 /= A(d);
        if (!live || !dx) continue;
#pragma unroll
        for (int i = 0; i < H::kPieces; ++i) {
            const int64_t e = (int64_t)(t + GROUP * i) * H::kWide;
            if (e >= d) continue;
            typename H::Piece o;
#pragma unroll
            for (int j = 0; j < H::kWide; ++j) {
                const A xhat = (hx.at(i, j) - mu) * rs;
                o.v[j] = from_acc<T>(rs * (hg.at(i, j) * wv[i][j] - s1 - xhat * s2));
            }
            if constexpr (VEC) __stcs(reinterpret_cast<uint4 *>(dx + row * d + e), o.raw);
            else dx[row * d + e] = o.v[0];
        }
    }
    if constexpr (VEC) cp_async_wait<0>();
    if (!partial) return;
    // the block's groups one after the other, then the block's row of partials
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        A(&a)[H::kPieces][H::kWide] = which ? ab : aw;
        if constexpr (kGroups > 1) {
            for (int g = 0; g < kGroups; ++g) {
                __syncthreads();
                if (threadIdx.x / GROUP != g) continue;
#pragma unroll
                for (int i = 0; i < H::kPieces; ++i)
#pragma unroll
                    for (int j = 0; j < H::kWide; ++j) {
                        A *c = columns + (t + GROUP * i) * H::kWide + j;
                        if (g > 0) a[i][j] += *c;
                        *c = a[i][j];
                    }
            }
            if (threadIdx.x / GROUP != kGroups - 1) continue;
        }
        A *out = partial + (blockIdx.x * 2 + which) * d;
#pragma unroll
        for (int i = 0; i < H::kPieces; ++i) {
            const int64_t e = (int64_t)(t + GROUP * i) * H::kWide;
#pragma unroll
            for (int j = 0; j < H::kWide; ++j)
                if (e + j < d) out[e + j] = a[i][j];
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
    k_layer_norm_join(const A *__restrict__ partial, int64_t parts, int64_t d, W *__restrict__ dw,
                      W *__restrict__ db) {
    __shared__ A sums[32][33];
    W *out = blockIdx.y ? db : dw;
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

// How a row is held: GROUP threads of N values.  Small rows take a warp, so that
// a block works on eight; 16 values a thread (8 of 8 bytes) keep enough bytes in
// flight with the fewest barriers.
struct Shape {
    int group, values;
};
Shape shape_of(int64_t d, int dtype) {
    const int most = dtype == BGL_F64 ? 8 : 16;
    if (d <= 32 * 8) return {32, 8};
    if (d <= 32 * most) return {32, most};
    if (d <= 128 * 8) return {128, 8};
    if (d <= 256 * 8) return {256, 8};
    if (d <= 256 * most) return {256, most};
    return {256, 2 * most};
}
int64_t most_held(int dtype) { return dtype == BGL_F64 ? kMostHeld / 2 : kMostHeld; }

// Blocks of the backward pass, one partial row each: resident ones, a fixed
// number for a given device so that the sums keep their order.
int64_t backward_blocks(int64_t rows, int64_t d, int dtype) {
    const int groups = kThreads / shape_of(d, dtype).group;
    const int64_t want = (rows + groups - 1) / groups, most = (int64_t)num_sms() * 2;
    return want < most ? want : most;
}
int64_t parts_of(int64_t rows, int64_t d, int dtype) {
    return d <= most_held(dtype) ? backward_blocks(rows, d, dtype) : splits_of(rows);
}

int check_norm(const char *who, int64_t rows, int64_t d, int dtype, int wdtype) {
    if (!row_dtype(dtype)) return fail(BGL_E_UNSUPPORTED, "%s: dtype %d", who, dtype);
    if (wdtype != dtype && !(dtype == BGL_BF16 && wdtype == BGL_F32))
        return fail(BGL_E_UNSUPPORTED, "%s: weight dtype %d with dtype %d", who, wdtype, dtype);
    if (rows < 0 || d < 0) return fail(BGL_E_INVALID, "%s: negative size", who);
    if (d >= (int64_t(1) << 31)) return fail(BGL_E_UNSUPPORTED, "%s: d >= 2^31", who);
    return BGL_OK;
}

// Calls f with the group size, the values of a thread and VEC as constants.
template <int GROUP, int N>
struct Constant {
    static constexpr int group = GROUP, values = N;
};
template <typename T, typename F>
int with_shape(Shape s, F &&f) {
    constexpr int M = sizeof(T) == 8 ? 8 : 16;
    if (s.group == 32) return s.values == 8 ? f(Constant<32, 8>()) : f(Constant<32, M>());
    if (s.group == 128) return f(Constant<128, 8>());
    if (s.values == 8) return f(Constant<256, 8>());
    if (s.values == M) return f(Constant<256, M>());
    return f(Constant<256, 2 * M>());
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
    if (p.d > most_held(p.dtype)) {
        const int64_t cap = (int64_t)num_sms() * 8;
        k_layer_norm_long<T, W><<<(unsigned)(p.rows < cap ? p.rows : cap), kThreads, 0, p.s>>>(
            x, w, b, p.rows, p.d, (A)p.eps, y, mean, rstd);
        BGL_LAUNCH_CHECK();
        return BGL_OK;
    }
    const bool vec = p.d * sizeof(T) % 16 == 0 && aligned(x, 16) && aligned(y, 16) && aligned(w, 16) && aligned(b, 16);
    return with_shape<T>(shape_of(p.d, p.dtype), [&](auto c) {
        constexpr int G = decltype(c)::group, N = decltype(c)::values, per = kThreads / G;
        const int64_t want = (p.rows + per - 1) / per, cap = (int64_t)num_sms() * 6;
        const unsigned grid = (unsigned)(want < cap ? want : cap);
        if (vec)
            k_layer_norm<T, W, G, N, true><<<grid, kThreads, 0, p.s>>>(x, w, b, p.rows, p.d, (A)p.eps, y, mean, rstd);
        else
            k_layer_norm<T, W, G, N, false><<<grid, kThreads, 0, p.s>>>(x, w, b, p.rows, p.d, (A)p.eps, y, mean, rstd);
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
    if (p.rows && p.d > most_held(p.dtype)) {
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
        const bool vec = p.d * sizeof(T) % 16 == 0 && aligned(x, 16) && aligned(dy, 16) && aligned(dx, 16) && aligned(w, 16);
        const int rc = with_shape<T>(shape_of(p.d, p.dtype), [&](auto c) {
            constexpr int G = decltype(c)::group, N = decltype(c)::values;
            const unsigned grid = (unsigned)parts;
            constexpr size_t smem = backward_smem<T, G, N, true>(), plain = backward_smem<T, G, N, false>();
            if (vec) {
                if (smem > 48 * 1024)
                    BGL_CUDA(cudaFuncSetAttribute(k_layer_norm_backward<T, W, G, N, true>,
                                                  cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
                k_layer_norm_backward<T, W, G, N, true><<<grid, kThreads, smem, p.s>>>(dy, x, mean, rstd, w, p.rows, p.d, dx, partial);
            } else {
                k_layer_norm_backward<T, W, G, N, false><<<grid, kThreads, plain, p.s>>>(dy, x, mean, rstd, w, p.rows, p.d, dx, partial);
            }
            BGL_LAUNCH_CHECK();
            return (int)BGL_OK;
        });
        if (rc) return rc;
    }
    if (sums) {
        k_layer_norm_join<A, W><<<dim3((unsigned)((p.d + 31) / 32), 2), 1024, 0, p.s>>>(
            partial, parts, p.d, (W *)p.dw, (W *)p.db);
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
