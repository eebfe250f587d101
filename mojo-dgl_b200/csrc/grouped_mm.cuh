// Shared declarations of the grouped GEMM (segment_mm / gather_mm).
#pragma once

#include "common.cuh"

namespace bgl {

// Device-side schedule of one grouped product, carved from the caller's
// workspace.  seg_off[r + 1]: first row of each segment (in the permuted order
// for gather_mm); tile_off[r + 1]: first tile of each segment; perm (gather_mm
// only): the stable sort of the row ids by idx_b.
struct GmmLayout {
    int64_t *seg_off;
    int64_t *tile_off;
    int64_t *counts;
    int32_t *keys;
    int32_t *keys_sorted;
    int32_t *iota;
    int32_t *perm;
    void *tc_b;  // tensor-core path: K-major copy of B (r x d2 x d1)
    void *sort_temp;
    size_t sort_temp_bytes;
    int64_t tile_rows;
    size_t bytes;
};

GmmLayout gmm_layout(void *ws, int64_t n, int64_t d1, int64_t r, int64_t d2, int dtype,
                     bool gather);

// tcgen05 path (grouped_mm_tc.cu).
bool gmm_tensor_core_supported(int64_t d1, int64_t d2, int dtype);
bool gmm_tensor_core_fits(int64_t n, int64_t r, int64_t d2);
int gmm_tensor_core(const void *a, const void *b, void *out, const GmmLayout &l, int64_t n,
                    int64_t d1, int64_t r, int64_t d2, int dtype, cudaStream_t s);

// Gradients of the grouped product on the tensor cores (grouped_mm_grad_tc.cu).
// Work comes in items for pairs of CTAs: 512 x 256 tiles of da, and pieces of db's
// 512 x 256 tiles (a range of the segment's 64-row slices).
constexpr int kGradSlice = 64, kGradRows = 512, kGradCols = 256;

constexpr int kGradShortest = 8;  // slices; a sum of so many is not cut

// The schedule, written by one kernel into the caller's workspace.  Segments
// are in the order of `order` in the arrays of db.
struct GradLayout {
    int64_t *off;       // [r + 1] first row of each segment
    int64_t *row_off;   // [r + 1] first 512-row tile of each segment (da)
    int32_t *order;     // [r] db's segments, long ones first
    int64_t *item_off;  // [r + 1] db's items before those of order[i]
    int64_t *cut_off;   // [r + 1] db's tiles of several pieces before those of order[i]
    int64_t *slot_off;  // [r + 1] their partial tiles
    int64_t *head;      // [kHead] see k_grad_schedule
    float *partial;     // partial tiles
    size_t bytes;
};
enum { kHeadItems = 0, kHeadDbItems = 1, kHeadPiece = 2, kHeadCut = 3, kHeadNext = 4, kHead = 5 };

// How a db tile's slices are cut: `count` pieces of `slices` each, the last
// one maybe shorter.
struct GradPieces {
    int64_t count, slices;
};
__host__ __device__ inline GradPieces grad_pieces(int64_t rows, int64_t most) {
    const int64_t all = rows > 0 ? (rows + kGradSlice - 1) / kGradSlice : 1;
    const int64_t count = (all + most - 1) / most, slices = (all + count - 1) / count;
    return {(all + slices - 1) / slices, slices};
}

struct GradTiles {
    int64_t cols;          // da: 256-column tiles of a row tile
    int64_t tiles1, tiles2;  // db: tiles of a segment's block down and across
    int pairs;
};
GradTiles gmm_grad_tiles(int64_t n, int64_t d1, int64_t r, int64_t d2);
// At most this many partial tiles a pair (k_grad_schedule's rule keeps to it).
constexpr int kGradSlots = 3;

// da or db may be null (not wanted).
bool gmm_grad_tc_supported(const void *grad, const void *a, const void *b, const void *da,
                           const void *db, int64_t n, int64_t d1, int64_t r, int64_t d2, int dtype);
int gmm_grad_tensor_core(const void *grad, const void *a, const void *b, void *da, void *db,
                         const GradLayout &l, const GradTiles &t, int64_t n, int64_t d1, int64_t r,
                         int64_t d2, cudaStream_t s);
cudaError_t gmm_grad_tc_error(int *code);

}  // namespace bgl
