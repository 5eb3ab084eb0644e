// Host pieces of the rows product that its kernels share.
#pragma once
#include "kq_expert.cuh"

namespace kq {

inline int64_t round8(int64_t v) { return (v + 7) & ~(int64_t)7; }

// A 16-bit operand of `batch` matrices of `r` rows and `c` contiguous columns,
// as it is or laid out again in the workspace.
struct Operand {
    const uint16_t* base;
    int64_t batch, r, c, sb, sr;
    bool direct;
};

inline Operand operand(const void* base, int64_t batch, int64_t r, int64_t c, int64_t sb, int64_t sr) {
    Operand o{static_cast<const uint16_t*>(base), batch, r, c, sb, sr, true};
    if (r == 1) o.sr = round8(c);
    if (batch == 1) o.sb = round8(o.sr * r);
    o.direct = ((uintptr_t)base & 15) == 0 && o.sr % 8 == 0 && o.sb % 8 == 0 && o.sr >= c && o.sb >= (batch > 1 ? o.sr : 0) &&
               o.sr < ((int64_t)1 << 38) && o.sb < ((int64_t)1 << 38);
    return o;
}

inline int map_rows(CUtensorMap* m, const Operand& o, bool bf16, int box_c, int box_r, const char* what) {
    const int64_t dims[3] = {o.c, o.r, o.batch}, strides[2] = {o.sr * 2, o.sb * 2};
    const int box[3] = {box_c, box_r, 1};
    return encode_tiles(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, o.base, dims,
                        strides, box, what);
}

inline int map_rows_2d(CUtensorMap* m, const Operand& o, bool bf16, int box_c, int box_r, const char* what) {
    const int64_t dims[2] = {o.c, o.r}, strides[1] = {o.sr * 2};
    const int box[2] = {box_c, box_r};
    return encode_tiles(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, o.base, dims,
                        strides, box, what);
}

// A rows product (forward, or the gradient in z when `grad`) whose operands are laid out for TMA.
struct RowsProduct {
    Operand x, w;              // w: columns along n (mn) or along k
    const int64_t* offsets;
    const void *bias, *aux;    // aux: residual or dy
    void* out;
    void* low;                 // grad: what the rounding of dz leaves out, laid out as `out`; may be null
    int64_t bias_stride, ld_aux, ld_out;
    int64_t rows, k, n_out, experts;
    int up;                    // gated: first coordinate of the up half in W
    int act;
    bool bf16, mn, gated, grad, zero_rest;
    int* err;                  // wait_error_word
    const char* what;
};

// Few rows an expert: bound by reading W (kq_expert_few.cu).
bool few_rows(const RowsProduct& p);
int few_rows_product(const RowsProduct& p, cudaStream_t s);

// y[r] = had128(x[r] W_e^T) * svh[e] * row_scale[r] for the rows of experts first .. first + experts - 1 of all_experts
// behind `offsets`: x [rows x k] and W [experts][n][k] binary16 (k a multiple of 8, n of 128), svh binary16
// [all_experts][n], y bf16 or fp16 with row stride ldy; rows of no expert are zeroed with zero_rest (when first is 0).
int rows_product_rotated(const uint16_t* x, const uint16_t* w, const int64_t* offsets, int64_t rows, int64_t k, int64_t n,
                         int64_t all_experts, int64_t first, int64_t experts, const uint16_t* svh, int64_t svh_stride, const float* row_scale, void* y, int64_t ldy,
                         bool bf16_out, bool zero_rest, int* err, cudaStream_t s);

}  // namespace kq
