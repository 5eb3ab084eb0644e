// Rows product with already prepared operands, for callers inside the library.
#pragma once
#include "kq_expert.cuh"

namespace kq {

// y[r] = had128(x[r] W_e^T) * svh[e] * row_scale[r] for the rows of experts 0 .. experts-1 behind `offsets`:
// x [rows x k] and W [experts][n][k] binary16 (k a multiple of 8, n of 128), svh binary16 [experts][n], y bf16 or
// fp16 with row stride ldy.
int rows_product_rotated(const uint16_t* x, const uint16_t* w, const int64_t* offsets, int64_t rows, int64_t k, int64_t n,
                         int64_t experts, const uint16_t* svh, int64_t svh_stride, const float* row_scale, void* y, int64_t ldy,
                         bool bf16_out, cudaStream_t s);

}  // namespace kq
