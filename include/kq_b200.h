/*
 * kq_b200.h -- C ABI of the kquant_b200 EXL3/QSRT trellis encoder for B200 (sm_100a).
 *
 * Every entry point takes plain device pointers, element counts and a
 * cudaStream_t (passed as void*).  It never allocates device memory, never
 * synchronizes the stream, and returns a KQ_* status code (0 on success).
 * kq_last_error() returns a readable message for the last failure of the
 * calling host thread.  Outputs and workspaces are caller-allocated, like the
 * reference extension's (kquant/csrc/sqg_quantize.cu:165-209).
 *
 * Layouts:
 *   tiles        float32 [n_tiles][256], 16x16 tiles already permuted to the
 *                tensor-core element order that the trellis runs along
 *                (kquant/exl3_encoder_backend.py:27-50)
 *   states       uint16  [n_tiles][256], 16-bit trellis state per element
 *   packed       uint16  [n_tiles][16*K], native EXL word order with SWAP16
 *   lut          uint8   [65536] E4M3 label bytes indexed by the 16-bit state
 *                (untransposed; kquant/sqg_e4m3.py:305-333)
 *   labels       uint16  [65536] binary16 labels indexed by state
 */
#ifndef KQ_B200_H
#define KQ_B200_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define KQ_OK 0
#define KQ_ERR_ARG (-1)        /* invalid argument (shape, K, context, pointer) */
#define KQ_ERR_WORKSPACE (-2)  /* workspace too small */
#define KQ_ERR_CUDA (-3)       /* CUDA runtime error (launch, attribute, device) */
#define KQ_ERR_ALIGN (-4)      /* pointer not aligned as the kernel requires */
#define KQ_ERR_TIMEOUT (-5)    /* an earlier kernel's internal wait ran out (kq_wait_errors) */

/* Codebook kinds, numbered like the reference's `cb` template argument
 * (kquant/csrc/qsrt_quantize_tiles_kernel.cuh:21, exl3_compat/quant/codebook.cuh). */
#define KQ_CB_3INST 0
#define KQ_CB_MCG 1
#define KQ_CB_MUL1 2
#define KQ_CB_SQG 4

/* Message describing the last non-zero status returned on this host thread. */
const char* kq_last_error(void);

/* ABI version, bumped when a signature changes. */
int kq_abi_version(void);

/*
 * Decode a codebook into 65,536 binary16 labels (one per 16-bit state).
 * kind == KQ_CB_SQG reads `lut` (device, 65,536 E4M3 bytes); other kinds
 * ignore it.
 * Replaces the per-state label decoders inlined in the reference kernel:
 * kquant/csrc/sqg_quantize.cu:17-119 (SQG) and
 * kquant/csrc/exl3_compat/quant/codebook.cuh:28-124 (MCG, MUL1, 3INST).
 */
int kq_build_labels(int kind, const uint8_t* lut, uint16_t* labels, void* stream);

/*
 * Workspace bytes that kq_viterbi_encode / kq_quantize_tiles_* need for
 * n_tiles tiles at rate K on the current device.  The figure includes the
 * 128 KiB label table that kq_quantize_tiles_* build in the workspace.
 */
size_t kq_viterbi_workspace_bytes(int K, int64_t n_tiles);

/*
 * Tail-biting Viterbi encode of n_tiles tiles against prebuilt labels.
 * out_vals[i] = label(out_states[i]) as float32.  tailbite_ctx in 1..128.
 * K in {2, 3, 4}.  Bit-exact with the reference kernel
 * kquant/csrc/qsrt_quantize_tiles_kernel.cuh:21-471 (codes and values).
 */
int kq_viterbi_encode(const float* tiles, int64_t n_tiles, int K, const uint16_t* labels,
                      int tailbite_ctx, float* out_vals, uint16_t* out_states,
                      void* workspace, size_t workspace_bytes, void* stream);

/*
 * Drop-in counterpart of the reference binding quantize_tiles_sqg
 * (kquant/csrc/sqg_quantize.cpp:23-28, sqg_quantize.cu:165-259).  It differs
 * in two ways: the LUT is the untransposed state-indexed table, and a single
 * workspace replaces the temp_costs/temp_edges pair.
 */
int kq_quantize_tiles_sqg(const float* tiles, float* out_vals, uint16_t* out_states, int64_t n_tiles,
                          const uint8_t* lut, int K, int tailbite_ctx,
                          void* workspace, size_t workspace_bytes, void* stream);

/*
 * Drop-in counterpart of quantize_tiles_procedural
 * (kquant/csrc/sqg_quantize.cpp:29-32, sqg_quantize.cu:261-342).
 * codebook: KQ_CB_MCG or KQ_CB_MUL1 (KQ_CB_3INST is also accepted).
 */
int kq_quantize_tiles_procedural(const float* tiles, float* out_vals, uint16_t* out_states,
                                 int64_t n_tiles, int K, int codebook, int tailbite_ctx,
                                 void* workspace, size_t workspace_bytes, void* stream);

/*
 * One 16-row step of the block-LDLQ traversal, fused around the Viterbi:
 * for a batch of row-major [size_k x size_n] fp32 matrices,
 *     tiles   = tensor-core-ordered 16x16 tiles of W[:, r0:r0+16] + comp
 *     What[:, r0:r0+16], enc[:, r0/16] = Viterbi(tiles)   (rows in W's layout)
 *     err[:, r0:r0+16] = W[:, r0:r0+16] - What[:, r0:r0+16]
 * comp [batch][16][size_n] is the LDLQ feedback of the step, enc
 * [batch][size_k/16][size_n/16][256] the 16-bit states.  Replaces the
 * tile gather / quantize_tiles / scatter sequence of one step of
 * kquant/exl3_encoder_backend.py:389-505 (ldlq); the arithmetic (one fp32
 * add, the Viterbi, one fp32 subtract) is the reference's.  Same labels,
 * K, context and workspace rules as kq_viterbi_encode with
 * n_tiles = batch * size_n / 16.  max_ctas > 0 caps the grid (each CTA
 * then loops over tile pairs), leaving the other SMs to concurrent work on
 * other streams; 0 uses every SM.
 */
int kq_ldlq_step_encode(const float* W, const float* comp, int64_t batch, int64_t size_k, int64_t size_n,
                        int64_t r0, int K, const uint16_t* labels, int tailbite_ctx, float* wq, float* err,
                        uint16_t* enc, int max_ctas, void* workspace, size_t workspace_bytes, void* stream);

/*
 * One LDLQ chain item: tiles [tile_col0, tile_col0 + n_tiles) of the 16-row
 * step r0 of one row-major [size_k x size_n] fp32 matrix W with its LDLQ
 * state (feedback P, error rows err, What, states enc [size_k/16][size_n/16]
 * [256]) and block-LDL factor L [size_k x size_k].  The step's feedback rows
 * are r0+16 .. end-1 (end = the end of the step's 128-row buffer).
 */
typedef struct {
    const float* W;
    const float* P;
    const float* L;
    float* err;
    float* wq;
    uint16_t* enc;
    int64_t size_k, size_n;
    int64_t r0, end;
    int64_t tile_col0, n_tiles;
    const uint16_t* labels;   /* binary16 label table of this item's codebook at rate K (kq_build_labels) */
    int32_t K;                /* 2, 3 or 4 */
    int32_t reserved;         /* 0 */
} kq_chain_item;

#define KQ_CHAIN_MAX_ITEMS 64

/*
 * One launch of LDLQ steps from up to KQ_CHAIN_MAX_ITEMS independent column
 * chains, each at its own row position:
 *     comp = P[r0:r0+16] + L[r0+16:end, r0:r0+16]^T err[r0+16:end]   (fp32)
 *     tiles = tensor-core-ordered 16x16 tiles of W[r0:r0+16] + comp
 *     What, enc = Viterbi(tiles);  err[r0:r0+16] = W - What
 * for the item's tile columns.  The feedback product is computed in the
 * kernel's tile load (one fp32 fma chain per element, in row order), so a
 * step is one launch and its result does not depend on which other items
 * share the launch.  Replaces the per-step feedback + quantize of
 * kquant/exl3_encoder_backend.py:389-505 (ldlq) / :1495-1583 (ldlq_batched);
 * the buffer-end update P[:begin] += L^T err stays with the caller.
 * Items carry their own K and label table.  When they all share both the
 * launch may hold any number of tiles.  Items of different K (or label
 * tables) share a launch when every item starts at an even tile (so each
 * tile pair has one K) and the pairs of each (K, labels) group, in runs of
 * m per CTA (m from ceil(pairs / SMs) up to 4), need at most one CTA per SM;
 * a CTA with two or more pairs hides each pair's tracebacks under another's
 * forward steps.  Workspace as
 * kq_viterbi_encode (K = 3) for the total tile count; max_ctas as
 * kq_ldlq_step_encode.
 */
int kq_ldlq_chain_step(const kq_chain_item* items, int n_items, int tailbite_ctx, int max_ctas, void* workspace,
                       size_t workspace_bytes, void* stream);

/*
 * Pack the low K bits of every state into 16*K uint16 words per tile in the
 * native EXL word order: MSB-first 16-symbol groups, then adjacent words
 * swapped (SWAP16).  Replaces ext.pack_trellis
 * (kquant/exl3_encoder_backend.py:1666-1677), whose word order
 * kquant/qsrt.py:811-833 restates.  K in 1..8.
 */
int kq_pack_trellis(const uint16_t* states, int64_t n_tiles, int K, uint16_t* packed, void* stream);

/*
 * Inverse of kq_pack_trellis, plus the cyclic state closure
 * state_i = ((state_{i-1} << K) | edge_i) & 0xFFFF.  Writes the 16-bit
 * states.  Replaces kquant/qsrt.py:836-863 (unpack_trellis_edges /
 * unpack_trellis_states) and kquant/exl3_reference.py:37-61
 * (reconstruct_trellis_states).  K in 1..8.
 */
int kq_unpack_trellis_states(const uint16_t* packed, int64_t n_tiles, int K, uint16_t* states,
                             void* stream);

/*
 * Allocation-free variant of kq_quantize_tiles_sqg for callers that cannot
 * allocate device memory themselves (a host whose allocator owns every byte
 * of the device, or code that must not trigger an allocation at an arbitrary
 * point).  No counterpart in the reference.  Same inputs, outputs and
 * results as kq_quantize_tiles_sqg, but no workspace argument: its scratch
 * (label table + decision rows, 32 MiB + 128 KiB) is a fixed __device__
 * array that every GPU loading this library holds until exit.  At most
 * KQ_NOALLOC_MAX_TILES tiles per call, a chosen bound on one call's latency
 * (not a limit of the scratch); larger counts return KQ_ERR_ARG.  The fixed
 * decision rows cap the grid at 8 CTAs (K2, K3) or 16 CTAs (K4), so a call
 * runs about 18x (K2, K3) or 9x (K4) slower than kq_quantize_tiles_sqg.
 * The first call on a device resolves the scratch address for that device
 * and caches it for the process: make that call before any stream capture,
 * and do not reset the device afterwards.  All calls share one scratch:
 * calls that overlap on the GPU (different streams, or different host
 * threads) race and corrupt each other's results; serialize them.
 */
#define KQ_NOALLOC_MAX_TILES 4096
int kq_quantize_tiles_sqg_noalloc(const float* tiles, float* out_vals, uint16_t* out_states, int64_t n_tiles,
                                  const uint8_t* lut, int K, int tailbite_ctx, void* stream);

/*
 * Fused tensor-core GEMM + trace (tcgen05 kind::tf32, TMA-fed):
 *     *out += sum_{i<M, j<N} (A B^T)[i][j] * D[i][j]
 * A [M x Kd], B [N x Kd] row-major fp32, D [M x N] with row stride ldd.
 * M % 128 == 0, N % 256 == 0, Kd % 32 == 0, 16-byte aligned rows.  Inputs
 * are rounded to TF32 by the tensor cores; accumulation is fp32, the final
 * reduction fp64.  With A = D = E^T and B = H (symmetric) this is the proxy
 * numerator tr(E^T H E) of kquant/exl3_encoder_backend.py:1466-1492
 * (block_trace).  *err is set to 1 if an internal wait timed out.
 */
int kq_trace_abt(const float* A, const float* B, const float* D, int64_t M, int64_t N, int64_t Kd, int64_t ldd,
                 double* out, int* err, void* stream);

/*
 * C = alpha * A B^T + beta * C on the tensor cores (tcgen05 kind::tf32, TMA
 * fed, TMEM accumulator).  Same shape rules as kq_trace_abt; C [M x N] with
 * row stride ldc.  The accumulator is drained into fp32 registers every
 * 128 K values, so with TF32-exact operands the result has fp32-GEMM
 * accuracy.  *err is set to 1 if an internal wait timed out.
 */
int kq_gemm_abt_tf32(const float* A, const float* B, float* C, int64_t M, int64_t N, int64_t Kd, int64_t ldc,
                     float alpha, float beta, int* err, void* stream);

/*
 * Hessian accumulation, replacing the chunk body of
 * kquant/capture.py:713-730 (_accumulate_hessian, accumulator.addmm_(x.T,
 * x * w[:, None]) in FP32):
 *     H[d x d] (row stride ldh) += x^T diag(w) x
 * for samples x [tokens x d] (row stride ldx) and weights w [tokens] (NULL:
 * all ones).  One operand kernel (transpose, weighting, TF32 hi/lo split)
 * and one tcgen05 launch over the upper-triangle tiles, mirrored, so H
 * stays exactly symmetric.  split = 3: hi*hi + hi*lo + lo*hi (fp32-grade
 * accuracy, what the FP32 addmm of the reference gives); split = 1: TF32
 * operands.  Any tokens >= 0 and dim >= 1; the workspace holds the padded
 * operands, kq_hessian_workspace_bytes(tokens, dim, split) bytes, 16-byte
 * aligned (0 = invalid arguments).
 */
size_t kq_hessian_workspace_bytes(int64_t tokens, int64_t dim, int split);
int kq_accumulate_hessian(const float* x, const float* w, int64_t tokens, int64_t dim, int64_t ldx, float* H,
                          int64_t ldh, int split, void* workspace, size_t workspace_bytes, int* err, void* stream);

/*
 * Weight load: bf16 [rows x cols] (row stride ld_src elements; HF [out, in])
 * -> fp32 [cols x rows] (EXL [in, out]), dst[c][r] = src[row_perm[r]][c]
 * (row_perm may be NULL).  Replaces the caller-side
 * source.index_select(0, perm).T.contiguous() of
 * kquant/pack/qsrt_encoder.py:554-569 (_encoder_weight) for bf16 sources.
 */
int kq_bf16_to_f32_transposed(const uint16_t* src, int64_t rows, int64_t cols, int64_t ld_src,
                              const int64_t* row_perm, float* dst, void* stream);

/*
 * Reconstruction of encoded weights in the original basis:
 *     out = had_r(had_l(wq) * su[:, None]) * sv[None, :]
 * wq, out [k x n] fp32 row-major (k, n multiples of 128; 16-byte aligned),
 * su [k], sv [n] fp32; had_l / had_r are the 128-block Sylvester Hadamards
 * normalised 1/sqrt(128).  Replaces the matmul-based reconstruction of
 * kquant/exl3_encoder_backend.py:2211-2216 and :2492-2498 (fast
 * Walsh-Hadamard transforms; equal up to fp32 rounding).
 */
int kq_reconstruct_rotated(const float* wq, const float* su, const float* sv, int64_t k, int64_t n, float* out,
                           void* stream);

/* Element types and activations of the expert-layer operators. */
#define KQ_BF16 0
#define KQ_FP16 1
#define KQ_FP32 2
#define KQ_ACT_NONE 0
#define KQ_ACT_RELU 1
#define KQ_ACT_SILU 2
#define KQ_ACT_GELU 3          /* z Phi(z), the error-function form */

/*
 * Products of rows sorted by expert with the experts' matrices (no
 * counterpart in the reference, which leaves the expert layer to its serving
 * stack).  Rows offsets[e] .. offsets[e+1] of x [rows x k] belong to expert
 * e; offsets (int64 [experts+1], non-decreasing, on the device) may be NULL
 * for one expert.  They are read by the kernels alone, so a captured call
 * follows new offsets at replay; values outside 0 .. rows are clamped.
 * W_e [k x n] is any pair of strides of which one is 1 (elements), so both
 * the EXL [in, out] and the HF [out, in] orientation are taken as stored.
 * x, W, bias, residual and y have one type (KQ_BF16 or KQ_FP16), products
 * are summed in fp32 and rounded once.  Bases and strides that are not
 * multiples of 16 bytes cost one more pass over that operand, into the
 * workspace.
 *
 *     kq_expert_linear:         y = act(x W + b) + residual
 *       gated (n = 2 n_out):    y = act(x Wg + bg) * (x Wu + bu) + residual
 *                               (Wg the first n_out columns of W)
 *     kq_expert_linear_grad_z:  dz from dy [rows x n_out] and the recomputed
 *                               z; y receives dz [rows x n]
 *     kq_expert_weight_grad:    dW_e = x_e^T dz_e, in W's strides (every
 *                               expert is written, zeros where it has no rows)
 *     kq_expert_bias_grad:      db_e = the column sums of dz_e + dz_low_e (dz_low may be NULL)
 *
 * The gradient in x is kq_expert_linear on dz with W's strides exchanged.
 * Rows of no expert are left as they were, or zeroed with zero_rest.
 * The calls after kq_expert_linear_grad_z take dz as rounded; db alone takes it
 * with what the rounding left out.
 * bias and residual may be NULL.  At most 1024 experts.
 */
typedef struct {
    const void* x;
    const void* w;
    const int64_t* offsets;
    const void* bias;          /* [experts][n], n contiguous */
    const void* residual;      /* [rows][n_out] */
    void* y;
    int64_t rows, k, n, experts;
    int64_t ldx;
    int64_t w_stride_e, w_stride_k, w_stride_n;
    int64_t bias_stride_e, ld_residual, ldy;
    int32_t dtype, activation, gated, zero_rest;
    void* y_low;                 /* kq_expert_linear_grad_z: dz - its rounding, row stride ldy; may be NULL */
} kq_expert_product;

size_t kq_expert_linear_workspace_bytes(const kq_expert_product* p);
int kq_expert_linear(const kq_expert_product* p, void* workspace, size_t workspace_bytes, void* stream);
int kq_expert_linear_grad_z(const kq_expert_product* p, const void* dy, int64_t ld_dy, void* workspace,
                            size_t workspace_bytes, void* stream);
size_t kq_expert_weight_grad_workspace_bytes(const kq_expert_product* p, const void* dz, int64_t ld_dz);
int kq_expert_weight_grad(const kq_expert_product* p, const void* dz, int64_t ld_dz, void* dw, void* workspace,
                          size_t workspace_bytes, void* stream);
int kq_expert_bias_grad(const void* dz, const void* dz_low, int64_t ld_dz, const int64_t* offsets, int64_t rows, int64_t n,
                        int64_t experts, int dtype, void* db, int64_t db_stride_e, void* stream);

/*
 * Calibration Hessians of all experts at once (kquant/capture.py:713-730,
 * _accumulate_hessian, for every expert of a layer):
 *     H_e (+)= sum_t w_t x[i_t] x[i_t]^T     den_e = sum_t w_t
 * over slots t = offsets[e] .. offsets[e+1] of `rows` slots (offsets as for
 * kq_expert_linear).  x [tokens x dim] (row stride ldx; KQ_BF16, KQ_FP16 or
 * KQ_FP32); index [rows] (int64) picks the row of each slot, NULL: slot t is
 * row t; a slot whose index is outside 0 .. tokens counts for nothing.  w
 * [rows] fp32, NULL: all ones.  H [experts][dim][dim] fp32 (strides h_stride,
 * ldh), added to when `add`, else overwritten; den [experts] fp64,
 * overwritten.  fp32 accuracy (exact 16-bit operand terms, rounded fp32
 * sums); every H_e is exactly symmetric when it starts so.  The workspace
 * (128-byte aligned) holds the gathered operand rows.
 */
size_t kq_expert_hessian_workspace_bytes(int64_t rows, int64_t dim, int64_t experts, int dtype, int weighted);
int kq_accumulate_expert_hessians(const void* x, int64_t tokens, int64_t dim, int64_t ldx, int dtype,
                                  const int64_t* index, const float* w, const int64_t* offsets, int64_t rows,
                                  int64_t experts, float* H, int64_t h_stride, int64_t ldh, int add, double* den,
                                  void* workspace, size_t workspace_bytes, void* stream);

/*
 * Products with encoded matrices, straight from the packed payload:
 *     y[r] = had(had(x[r] * suh_e) What_e) * svh_e
 * for rows grouped by expert as in kq_expert_linear, i.e. x times the weight
 * that kq_reconstruct_rotated gives (128-block Hadamards normalised
 * 1/sqrt(128), kquant/exl3_encoder_backend.py:2211-2216).  trellis
 * [experts][k/16][n/16][16 bits] words of kq_pack_trellis, every expert at
 * the same rate; suh [experts][k], svh [experts][n] binary16; x and y
 * KQ_BF16 or KQ_FP16.  codebook: KQ_CB_MCG (table NULL), KQ_CB_SQG (table:
 * 65,536 E4M3 bytes by state) or KQ_CB_LABELS (table: 65,536 binary16 labels
 * by state, kq_build_labels).  The rotated row enters the tensor cores as
 * binary16 with a power of two of its own; sums are fp32, y is rounded once.
 * Rows of no expert as in kq_expert_linear.  The workspace holds the rotated
 * rows and partial sums or decoded matrices, of the latter at most 1 GiB (or
 * one expert's, if that is more).
 */
#define KQ_CB_LABELS 5
typedef struct {
    const void* x;
    const uint16_t* trellis;
    const uint16_t* suh;
    const uint16_t* svh;
    const int64_t* offsets;
    const void* table;
    void* y;
    int64_t rows, k, n, experts;
    int64_t ldx, ldy, suh_stride_e, svh_stride_e;
    int32_t bits, codebook, dtype, zero_rest;
} kq_trellis_product;

size_t kq_trellis_linear_workspace_bytes(const kq_trellis_product* p);
int kq_trellis_linear(const kq_trellis_product* p, void* workspace, size_t workspace_bytes, void* stream);

/*
 * The internal waits of the expert-layer kernels are bounded.  When one runs
 * out the kernel ends with undefined results, and the expert-layer entry
 * points refuse every call on that device with KQ_ERR_TIMEOUT until
 * kq_wait_errors has been called.
 *
 * kq_wait_errors writes 1 to *out (device int32) if a wait ran out on this
 * device since the last call, else 0, and clears it, in stream order.
 * kq_wait_error_flag gives the address of the current device's flag in host
 * memory, for programs that look at it themselves (replayed graphs make no
 * calls): non-zero once a wait has run out.  The address stays valid.
 */
int kq_wait_errors(int32_t* out, void* stream);
int kq_wait_error_flag(int32_t** flag);

/*
 * Roofline probe (no reference counterpart): launches blocks x threads
 * threads that each issue iters*128 independent __hfma2 instructions.  Time
 * it with events on `stream`: HFMA2 rate = blocks*threads*iters*128 / time.
 * The Viterbi kernel's ALU roofline is derived from this measured rate.
 */
int kq_probe_hfma2(void* out, int iters, int blocks, int threads, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* KQ_B200_H */
