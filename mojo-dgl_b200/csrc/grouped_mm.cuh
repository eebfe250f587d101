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

// tcgen05 path (grouped_mm_tc.cu).  With b == nullptr, l.tc_b already is the
// K-major B: r blocks of d2 rows of d1 values.
bool gmm_tensor_core_supported(int64_t d1, int64_t d2, int dtype);
bool gmm_tensor_core_fits(int64_t n, int64_t r, int64_t d2);
int gmm_tensor_core(const void *a, const void *b, void *out, const GmmLayout &l, int64_t n,
                    int64_t d1, int64_t r, int64_t d2, int dtype, cudaStream_t s);

// Schedule of the gradients (grouped_mm_grad.cu writes it, one kernel, in the
// caller's workspace).
struct GradLayout {
    int64_t *off;       // [r + 1] first row of each segment
    int64_t *tile_off;  // [r + 1] first 128-row tile of each segment (da)
    int64_t *unit_off;  // [r + 1] first unit of each segment (db)
    int64_t *mode;      // [1] 1: db's units are split evenly over the CTAs
    float *partial;     // db: partial tiles of split units
    size_t bytes;
};

// tcgen05 path of db (grouped_mm_grad_tc.cu).  A unit is one 64-row slice of
// one output tile's sum; a segment without rows has one unit a tile.
struct GradTiles {
    int64_t tiles_n;      // 256-column tiles of a segment's block
    int64_t per_segment;  // 256 x 256 tiles of a segment's block
    int ctas;
};
constexpr int kGradSlice = 64, kGradTile = 256;
bool gmm_grad_tc_supported(const void *grad, const void *a, const void *db, int64_t n, int64_t d1,
                           int64_t r, int64_t d2, int dtype);
GradTiles gmm_grad_tiles(int64_t n, int64_t d1, int64_t r, int64_t d2);
int gmm_grad_tensor_core(const void *grad, const void *a, void *db, const GradLayout &l,
                         const GradTiles &t, int64_t n, int64_t d1, int64_t r, int64_t d2,
                         cudaStream_t s);
cudaError_t gmm_grad_tc_error(int *code);

}  // namespace bgl
