// Products of rows sorted by expert with the experts' matrices, on tcgen05.
//
//   rows:  y[r] = epilogue(x[r] W_e + b_e)     rows r of expert e
//   sums:  dW_e = x_e^T dz_e                   sum over expert e's rows
//
// Operands are bf16 or fp16, accumulation fp32 in tensor memory, one rounding
// at the end.  The epilogue of the rows product adds the bias, applies the
// activation (of the gate, times up, when gated) and adds the residual; its
// gradient form turns the recomputed pre-activation z and dy into dz.
//
// One persistent CTA per SM, 128 x 256 output tiles (gated: 128 columns of
// gate and the same 128 of up side by side).  Warp 0 issues TMA into a ring of
// 64-deep stages, warp 1 issues tcgen05.mma, warps 2..9 drain; two 256-column
// accumulators alternate, so a tile's epilogue runs under the next tile's
// products.  Both operands may be K-major or MN-major in shared memory: W is
// taken as stored ([k][n] or [n][k]), and the sums product reads x and dz as
// they are, contracting over their rows.
//
// The offsets stay on the device: every CTA scans them into shared memory and
// walks the same tile order, so a call captured into a graph follows new
// offsets at replay.  A rows tile that ends inside another expert's rows
// computes them and does not store them (a row meets only its own
// accumulators); a sums tile zeroes the rows behind its expert's last in
// shared memory before the product, because there they would be added in.
#include "kq_expert_rows.cuh"

namespace kq {
namespace {

__device__ int g_wait_error = 0;

constexpr int BM = 128, BN = 256, BK = 64, STAGES = 4;
constexpr int A_BYTES = BM * BK * 2, B_BYTES = BN * BK * 2, STAGE_BYTES = A_BYTES + B_BYTES;
constexpr int CHUNK = 64 * 128;                 // 64 rows of 128 bytes: one MN-major box
constexpr int DRAIN_WARPS = 8, THREADS = 64 + 32 * DRAIN_WARPS;
constexpr int GROUP_BYTES = (3 * kMaxExperts + 4) * 4;
constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + GROUP_BYTES + 1024;

enum { EPI_FORWARD, EPI_GRAD, EPI_SUMS, EPI_ROTATED };

struct Params {
    const int64_t* offsets;
    const void* bias;
    const void* aux;       // residual (forward), dy (gradient) or svh (rotated)
    const float* row_scale;
    void* out;
    int64_t bias_stride, ld_aux, ld_out, out_stride;   // out_stride: per expert (sums)
    int rows, experts, k_steps, m_tiles, n_tiles, m_out, n_out;
    int w_second;          // coordinate of the tile's second 128 columns, relative to its first
    int out_second;        // column of dz's up half
    int* err;
    uint32_t idesc;
    int act;
    bool a_mn, b_mn, zero_rest, vec_bias, vec_aux, vec_out;
};

struct Tile { int e, row0, count, m0, n0, k_steps; };

// Tile t of the launch.  Rows: the row tiles of an expert run fastest, so the
// CTAs that share a slice of W run together.
template <int EPI>
__device__ __forceinline__ bool tile_at(const Params& p, const int* lo, const int* cnt, const int* cum, int64_t t, Tile& o) {
    if constexpr (EPI == EPI_SUMS) {
        const int per = p.m_tiles * p.n_tiles;
        if (t >= (int64_t)per * p.experts) return false;
        o.e = (int)(t / per);
        const int l = (int)(t - (int64_t)o.e * per);
        o.m0 = (l % p.m_tiles) * BM;
        o.n0 = (l / p.m_tiles) * BN;
        o.row0 = lo[o.e];
        o.count = cnt[o.e];
        o.k_steps = (o.count + BK - 1) / BK;
    } else {
        if (t >= (int64_t)cum[p.experts] * p.n_tiles) return false;
        o.e = expert_of(cum, p.experts, (int)(t / p.n_tiles));
        const int mt = cum[o.e + 1] - cum[o.e];
        const int64_t l = t - (int64_t)cum[o.e] * p.n_tiles;
        o.m0 = (int)(l % mt) * BM;
        o.n0 = (int)(l / mt);                   // tile index; the caller scales it
        o.row0 = lo[o.e] + o.m0;
        o.count = cnt[o.e] - o.m0;
        o.k_steps = p.k_steps;
    }
    return true;
}

template <typename T, int EPI, bool GATED>
__global__ void __launch_bounds__(THREADS, 1)
expert_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const Params p) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t full_bar[STAGES], empty_bar[STAGES], acc_full[2], acc_empty[2];
    __shared__ uint32_t tmem_slot;
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    int* lo = reinterpret_cast<int*>(smem + STAGES * STAGE_BYTES);
    int* cnt = lo + kMaxExperts;
    int* cum = cnt + kMaxExperts;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int NW = GATED ? 128 : BN;        // output columns of a rows tile

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&full_bar[s], 1);
            mbar_init(&empty_bar[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&acc_full[b], 1);
            mbar_init(&acc_empty[b], DRAIN_WARPS);
        }
        mbar_init_fence();
    }
    if (warp == 1) tmem_alloc(&tmem_slot, 2 * BN);
    scan_groups(p.offsets, p.experts, p.rows, BM, lo, cnt, cum);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    bool ok = true;
    Tile t;

    if (warp == 0) {
        if (lane == 0) {
            uint32_t it = 0;
            for (int64_t i = blockIdx.x; ok && tile_at<EPI>(p, lo, cnt, cum, i, t); i += gridDim.x) {
                for (int ks = 0; ks < t.k_steps; ++ks, ++it) {
                    const int s = it % STAGES;
                    if (!(ok = mbar_wait(&empty_bar[s], ((it / STAGES) & 1) ^ 1))) break;
                    mbar_expect_tx(&full_bar[s], STAGE_BYTES);
                    uint8_t *sa = smem + s * STAGE_BYTES, *sb = sa + A_BYTES;
                    if constexpr (EPI == EPI_SUMS) {
                        const int r = t.row0 + ks * BK;
#pragma unroll
                        for (int c = 0; c < BM / 64; ++c) tma_load_2d(sa + c * CHUNK, &map_a, t.m0 + 64 * c, r, &full_bar[s]);
#pragma unroll
                        for (int c = 0; c < BN / 64; ++c) tma_load_2d(sb + c * CHUNK, &map_b, t.n0 + 64 * c, r, &full_bar[s]);
                    } else {
                        const int n0 = t.n0 * NW, n1 = n0 + p.w_second;
                        tma_load_2d(sa, &map_a, ks * BK, t.row0, &full_bar[s]);
                        if (p.b_mn) {
                            tma_load_3d(sb, &map_b, n0, ks * BK, t.e, &full_bar[s]);
                            tma_load_3d(sb + CHUNK, &map_b, n0 + 64, ks * BK, t.e, &full_bar[s]);
                            tma_load_3d(sb + 2 * CHUNK, &map_b, n1, ks * BK, t.e, &full_bar[s]);
                            tma_load_3d(sb + 3 * CHUNK, &map_b, n1 + 64, ks * BK, t.e, &full_bar[s]);
                        } else {
                            tma_load_3d(sb, &map_b, ks * BK, n0, t.e, &full_bar[s]);
                            tma_load_3d(sb + B_BYTES / 2, &map_b, ks * BK, n1, t.e, &full_bar[s]);
                        }
                    }
                }
            }
            if (!ok) report_wait_error(p.err);
        }
    } else if (warp == 1) {
        uint32_t it = 0, tile_no = 0;
        const uint32_t a_step = p.a_mn ? 128 : 2, b_step = p.b_mn ? 128 : 2;   // 16 contraction values, in 16-byte units
        for (int64_t i = blockIdx.x; ok && tile_at<EPI>(p, lo, cnt, cum, i, t); i += gridDim.x, ++tile_no) {
            const int b = tile_no & 1;
            if (!(ok = mbar_wait(&acc_empty[b], ((tile_no >> 1) & 1) ^ 1))) break;
            tc_fence_after();
            for (int ks = 0; ks < t.k_steps; ++ks, ++it) {
                const int s = it % STAGES;
                if (!(ok = mbar_wait(&full_bar[s], (it / STAGES) & 1))) break;
                uint8_t* sa = smem + s * STAGE_BYTES;
                if constexpr (EPI == EPI_SUMS) {
                    const int valid = t.count - ks * BK;
                    if (valid < BK) {           // rows of the next expert: one 128-byte line a row and chunk
                        const int lines = (BK - valid) * (STAGE_BYTES / CHUNK);
                        for (int l = lane; l < lines * 8; l += 32) {
                            const int line = l >> 3, c = line / (BK - valid), r = valid + line % (BK - valid);
                            *reinterpret_cast<uint4*>(sa + c * CHUNK + r * 128 + (l & 7) * 16) = make_uint4(0, 0, 0, 0);
                        }
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        __syncwarp();
                    }
                }
                tc_fence_after();
                if (lane == 0) {
                    const uint32_t a = smem_addr(sa);
                    const uint64_t ad = smem_desc(a, p.a_mn ? CHUNK : 16), bd = smem_desc(a + A_BYTES, p.b_mn ? CHUNK : 16);
#pragma unroll
                    for (int kk = 0; kk < BK / 16; ++kk)
                        mma_f16(tmem + b * BN, ad + a_step * kk, bd + b_step * kk, p.idesc, (ks | kk) != 0);
                    mma_commit(&empty_bar[s]);
                }
                __syncwarp();
            }
            if (ok && lane == 0) mma_commit(&acc_full[b]);
            __syncwarp();
        }
        if (!ok && lane == 0) report_wait_error(p.err);
    } else {
        const int q = warp & 3, h = (warp - 2) >> 2;    // tensor-memory lanes 32q.., column half h
        const int r = q * 32 + lane;
        uint32_t tile_no = 0;
        for (int64_t i = blockIdx.x; tile_at<EPI>(p, lo, cnt, cum, i, t); i += gridDim.x, ++tile_no) {
            const int b = tile_no & 1;
            if (!(ok = __all_sync(0xFFFFFFFFu, mbar_wait(&acc_full[b], (tile_no >> 1) & 1)))) break;
            tc_fence_after();
            const uint32_t base = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(b * BN);
            const bool live = EPI == EPI_SUMS ? t.m0 + r < p.m_out : r < t.count;
            constexpr int HALF = EPI == EPI_SUMS ? BN / 2 : NW / 2;
            const int n_base = (EPI == EPI_SUMS ? t.n0 : t.n0 * NW) + h * HALF;
            const T* bias = p.bias ? static_cast<const T*>(p.bias) + t.e * p.bias_stride : nullptr;
            T* orow;
            const T* arow = nullptr;
            if constexpr (EPI == EPI_SUMS) {
                orow = static_cast<T*>(p.out) + t.e * p.out_stride + (int64_t)(t.m0 + r) * p.ld_out;
            } else {
                orow = static_cast<T*>(p.out) + (int64_t)(t.row0 + r) * p.ld_out;
                if (EPI != EPI_ROTATED && p.aux) arow = static_cast<const T*>(p.aux) + (int64_t)(t.row0 + r) * p.ld_aux;
            }
            if constexpr (EPI == EPI_ROTATED) {
                // A thread holds one row of one 128-column Hadamard block: the transform stays in its registers.
                if (n_base < p.n_out) {
                    float z[128];
#pragma unroll
                    for (int c = 0; c < 128; c += 16) {
                        uint32_t v[16];
                        tmem_ld16(base + h * HALF + c, v);
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 16; ++e) z[c + e] = __uint_as_float(v[e]);
                    }
#pragma unroll
                    for (int d = 1; d < 128; d <<= 1)
#pragma unroll
                        for (int e = 0; e < 128; ++e)
                            if (!(e & d)) {
                                const float a = z[e], c = z[e + d];
                                z[e] = a + c;
                                z[e + d] = a - c;
                            }
                    if (live) {
                        const float scale = p.row_scale[t.row0 + r] * 0.08838834764831845f;   // 1 / sqrt(128)
                        const __half* svh = static_cast<const __half*>(p.aux) + t.e * p.ld_aux + n_base;
#pragma unroll
                        for (int c = 0; c < 128; c += 8) {
                            float a[8];
                            load8(svh + c, p.vec_aux, 8, a);
#pragma unroll
                            for (int e = 0; e < 8; ++e) a[e] *= z[c + e] * scale;
                            store8(orow + n_base + c, p.vec_out, 8, a);
                        }
                    }
                    __syncwarp();
                }
            } else {
#pragma unroll 1
            for (int c = 0; c < HALF; c += 16) {
                if (n_base + c >= p.n_out) break;
                uint32_t v[16], u[16];
                tmem_ld16(base + h * HALF + c, v);
                if constexpr (GATED) tmem_ld16(base + 128 + h * HALF + c, u);
                tmem_wait_ld();
                if (EPI == EPI_SUMS && t.k_steps == 0) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) v[e] = 0;
                }
#pragma unroll
                for (int g = 0; g < 2 && live; ++g) {
                    const int j = n_base + c + 8 * g, nv = p.n_out - j;
                    if (nv <= 0) break;
                    float z[8], w[8], a[8], d[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        z[e] = __uint_as_float(v[8 * g + e]);
                        if constexpr (GATED) w[e] = __uint_as_float(u[8 * g + e]);
                    }
                    if constexpr (EPI != EPI_SUMS) {
                        if (bias) {
                            load8(bias + j, p.vec_bias && nv >= 8, nv, a);
#pragma unroll
                            for (int e = 0; e < 8; ++e) z[e] += a[e];
                            if constexpr (GATED) {
                                load8(bias + p.n_out + j, p.vec_bias && nv >= 8, nv, a);
#pragma unroll
                                for (int e = 0; e < 8; ++e) w[e] += a[e];
                            }
                        }
                        if (arow) load8(arow + j, p.vec_aux && nv >= 8, nv, a);
                    }
                    if constexpr (EPI == EPI_FORWARD) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            z[e] = activate(p.act, z[e]);
                            if constexpr (GATED) z[e] *= w[e];
                            if (arow) z[e] += a[e];
                        }
                    }
                    if constexpr (EPI == EPI_GRAD) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            if constexpr (GATED) {
                                d[e] = a[e] * activate(p.act, z[e]);
                                z[e] = a[e] * w[e] * slope(p.act, z[e]);
                            } else {
                                z[e] = a[e] * slope(p.act, z[e]);
                            }
                        }
                        if constexpr (GATED) store8(orow + p.out_second + j, p.vec_out && nv >= 8, nv, d);
                    }
                    store8(orow + j, p.vec_out && nv >= 8, nv, z);
                }
                __syncwarp();
            }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&acc_empty[b]);
        }
        if (!ok && lane == 0) report_wait_error(p.err);
        // Rows of no expert: zero in a fresh output, untouched otherwise.
        if (EPI != EPI_SUMS && p.zero_rest && p.offsets) {
            int first, last, n;
            group_of(p.offsets, 0, p.rows, first, n);
            group_of(p.offsets, p.experts - 1, p.rows, last, n);
            last += n;
            const int width = EPI == EPI_GRAD && GATED ? p.out_second + p.n_out : p.n_out;
            for (int row = blockIdx.x; row < p.rows; row += gridDim.x) {
                if (row >= first && row < last) { continue; }
                T* o = static_cast<T*>(p.out) + (int64_t)row * p.ld_out;
                for (int j = threadIdx.x - 64; j < width; j += 32 * DRAIN_WARPS) o[j] = from_f<T>(0.f);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) tmem_free(tmem, 2 * BN);
}

// 16-bit rows [batch][r][c] -> [batch][r][cols_out]: an operand whose base or
// strides are not the multiples of 16 bytes that TMA needs is laid out once
// more.  Columns c .. cols_out are not written (no tile map reaches them, or
// only as output columns that are not stored).
__global__ void relayout_kernel(const uint16_t* __restrict__ src, int64_t sb, int64_t sr, int64_t r, int64_t c,
                                uint16_t* __restrict__ dst, int64_t db, int64_t cols_out, int64_t total) {
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
        const int64_t j = i % c, row = i / c;
        const int64_t b = row / r, y = row - b * r;
        dst[b * db + y * cols_out + j] = src[b * sb + y * sr + j];
    }
}

// Column sums of dz over every expert's rows, fp32 in row order within a
// thread: one warp per 32 columns and expert, rows split over 8 warps.
template <typename T>
__global__ void __launch_bounds__(256)
bias_grad_kernel(const T* __restrict__ dz, int64_t ld, const int64_t* __restrict__ offsets, int rows, int n, T* __restrict__ db,
                 int64_t db_stride) {
    __shared__ float part[8][32];
    const int e = blockIdx.y, lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int j = blockIdx.x * 32 + lane;
    int lo, count;
    group_of(offsets, e, rows, lo, count);
    float s = 0.f;
    if (j < n)
        for (int r = w; r < count; r += 8) s += to_f<T>(dz[(int64_t)(lo + r) * ld + j]);
    part[w][lane] = s;
    __syncthreads();
    if (w == 0 && j < n) {
        s = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) s += part[i][lane];
        db[e * db_stride + j] = from_f<T>(s);
    }
}

int64_t round8(int64_t v) { return (v + 7) & ~(int64_t)7; }

// A 16-bit operand of `batch` matrices of `r` rows and `c` contiguous columns,
// as it is or laid out again in the workspace.
struct Operand {
    const uint16_t* base;
    int64_t batch, r, c, sb, sr;
    bool direct;
};

Operand operand(const void* base, int64_t batch, int64_t r, int64_t c, int64_t sb, int64_t sr) {
    Operand o{static_cast<const uint16_t*>(base), batch, r, c, sb, sr, true};
    if (r == 1) o.sr = round8(c);
    if (batch == 1) o.sb = round8(o.sr * r);
    o.direct = ((uintptr_t)base & 15) == 0 && o.sr % 8 == 0 && o.sb % 8 == 0 && o.sr >= c && o.sb >= (batch > 1 ? o.sr : 0) &&
               o.sr < ((int64_t)1 << 38) && o.sb < ((int64_t)1 << 38);
    return o;
}

size_t relayout_bytes(const Operand& o) {
    return o.direct ? 0 : (size_t)(o.batch * o.r * round8(o.c)) * 2;
}

// `halves` = 2: the columns are two halves (gate and up) that each start on a 16-byte boundary in the copy.
int relayout(Operand& o, uint16_t*& ws, int halves, cudaStream_t s) {
    if (o.direct) return KQ_OK;
    const int64_t part = o.c / halves, pad = round8(part), cols = pad * halves;
    for (int h = 0; h < halves; ++h) {
        const int64_t total = o.batch * o.r * part;
        const int64_t blocks = (total + 1023) / 1024;
        relayout_kernel<<<(int)(blocks < 4096 ? blocks : 4096), 256, 0, s>>>(o.base + h * part, o.sb, o.sr, o.r, part, ws + h * pad,
                                                                           o.r * cols, cols, total);
        if (int rc = check_launch("relayout_kernel")) return rc;
    }
    o.base = ws;
    o.sr = cols;
    o.sb = o.r * cols;
    o.c = cols == pad ? o.c : cols;
    ws += (o.batch * o.r * cols + 7) & ~(int64_t)7;
    o.direct = true;
    return KQ_OK;
}

int map_rows(CUtensorMap* m, const Operand& o, bool bf16, int box_c, int box_r, const char* what) {
    const int64_t dims[3] = {o.c, o.r, o.batch}, strides[2] = {o.sr * 2, o.sb * 2};
    const int box[3] = {box_c, box_r, 1};
    return encode_tiles(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, o.base, dims,
                        strides, box, what);
}

int map_rows_2d(CUtensorMap* m, const Operand& o, bool bf16, int box_c, int box_r, const char* what) {
    const int64_t dims[2] = {o.c, o.r}, strides[1] = {o.sr * 2};
    const int box[2] = {box_c, box_r};
    return encode_tiles(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, o.base, dims,
                        strides, box, what);
}

template <typename T, int EPI, bool GATED>
int launch_as(const CUtensorMap& a, const CUtensorMap& b, const Params& p, int grid, cudaStream_t s) {
    cudaError_t e = cudaFuncSetAttribute(expert_kernel<T, EPI, GATED>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES);
    if (e != cudaSuccess) { set_error("cudaFuncSetAttribute: %s", cudaGetErrorString(e)); return KQ_ERR_CUDA; }
    expert_kernel<T, EPI, GATED><<<grid, THREADS, SMEM_BYTES, s>>>(a, b, p);
    return check_launch("expert_kernel");
}

template <int EPI, bool GATED>
int launch(bool bf16, const CUtensorMap& a, const CUtensorMap& b, const Params& p, int grid, cudaStream_t s) {
    return bf16 ? launch_as<__nv_bfloat16, EPI, GATED>(a, b, p, grid, s) : launch_as<__half, EPI, GATED>(a, b, p, grid, s);
}

bool vec8(const void* base, int64_t ld, int64_t ld2 = 0) {
    return ((uintptr_t)base & 15) == 0 && ld % 8 == 0 && ld2 % 8 == 0;
}

// The matrices of `p` as stored: columns contiguous along n or along k.
bool n_contiguous(const kq_expert_product& p) {
    return p.w_stride_n == 1 ? (p.w_stride_k != 1 || p.k == 1 || p.n > 1) : p.n == 1 && p.w_stride_k != 1;
}

Operand w_operand(const kq_expert_product& p, bool mn) {
    Operand o = mn ? operand(p.w, p.experts, p.k, p.n, p.w_stride_e, p.w_stride_k)
                   : operand(p.w, p.experts, p.n, p.k, p.w_stride_e, p.w_stride_n);
    // Gate and up both start at an innermost coordinate: on a 16-byte boundary.
    if (mn && p.gated && (p.n / 2) % 8) o.direct = false;
    return o;
}

size_t relayout_w_bytes(const kq_expert_product& p, const Operand& o, bool mn) {
    if (o.direct) return 0;
    return mn && p.gated ? (size_t)(o.batch * o.r * 2 * round8(p.n / 2)) * 2 : relayout_bytes(o);
}

int check_product(const kq_expert_product& p, const char* what) {
    if (p.rows < 0 || p.k <= 0 || p.n <= 0 || p.experts <= 0) {
        set_error("%s: need rows >= 0 and k, n, experts >= 1 (rows=%lld k=%lld n=%lld experts=%lld)", what, (long long)p.rows,
                  (long long)p.k, (long long)p.n, (long long)p.experts);
        return KQ_ERR_ARG;
    }
    if (p.experts > kMaxExperts) { set_error("%s: at most %d experts", what, kMaxExperts); return KQ_ERR_ARG; }
    if (p.rows > 0x7FFFFF00 || p.k > 0x7FFFFF00 || p.n > 0x7FFFFF00) { set_error("%s: problem too large", what); return KQ_ERR_ARG; }
    if (p.experts > 1 && !p.offsets) { set_error("%s: several experts need offsets", what); return KQ_ERR_ARG; }
    if (p.dtype != KQ_BF16 && p.dtype != KQ_FP16) { set_error("%s: dtype must be KQ_BF16 or KQ_FP16", what); return KQ_ERR_ARG; }
    if (p.activation < KQ_ACT_NONE || p.activation > KQ_ACT_GELU) { set_error("%s: unknown activation %d", what, p.activation); return KQ_ERR_ARG; }
    if (p.gated && p.n % 2) { set_error("%s: gated needs an even n", what); return KQ_ERR_ARG; }
    if (p.w_stride_k != 1 && p.w_stride_n != 1 && p.k > 1 && p.n > 1) {
        set_error("%s: W needs unit stride along k or n", what);
        return KQ_ERR_ARG;
    }
    if (((uintptr_t)p.x | (uintptr_t)p.w | (uintptr_t)p.y) & 1) { set_error("%s: 2-byte alignment", what); return KQ_ERR_ALIGN; }
    return KQ_OK;
}

size_t product_workspace(const kq_expert_product& p) {
    const bool mn = n_contiguous(p);
    const Operand w = w_operand(p, mn), x = operand(p.x, 1, p.rows, p.k, 0, p.ldx);
    const size_t n = relayout_w_bytes(p, w, mn) + relayout_bytes(x);
    return n ? n + 64 : 0;                      // each part is rounded up to 16 bytes
}

int rows_product(const kq_expert_product& p, const void* dy, int64_t ld_dy, void* workspace, size_t workspace_bytes,
                 cudaStream_t s, const char* what) {
    if (int rc = check_product(p, what)) return rc;
    if (p.rows == 0) return KQ_OK;
    const bool grad = dy != nullptr;
    if (!p.x || !p.w || !p.y) { set_error("%s: null pointer", what); return KQ_ERR_ARG; }
    const int64_t n_out = p.gated ? p.n / 2 : p.n;
    if (p.ldy < (grad ? p.n : n_out) && p.rows > 1) { set_error("%s: ldy too small", what); return KQ_ERR_ARG; }
    const size_t need = product_workspace(p);
    if (need && (workspace_bytes < need || !workspace)) { set_error("%s: workspace too small", what); return KQ_ERR_WORKSPACE; }
    if ((uintptr_t)workspace & 15) { set_error("%s: workspace must be 16-byte aligned", what); return KQ_ERR_ALIGN; }
    uint16_t* ws = static_cast<uint16_t*>(workspace);
    const bool bf16 = p.dtype == KQ_BF16, mn = n_contiguous(p);
    Operand x = operand(p.x, 1, p.rows, p.k, 0, p.ldx), w = w_operand(p, mn);
    const bool gated_copy = mn && p.gated && !w.direct;
    if (int rc = relayout(x, ws, 1, s)) return rc;
    if (int rc = relayout(w, ws, gated_copy ? 2 : 1, s)) return rc;
    CUtensorMap ma, mb;
    if (int rc = map_rows_2d(&ma, x, bf16, BK, BM, what)) return rc;
    if (int rc = map_rows(&mb, w, bf16, mn ? 64 : BK, mn ? BK : BN / 2, what)) return rc;
    Params q{};
    if (int rc = wait_error_word(&q.err)) return rc;
    q.offsets = p.offsets;
    q.bias = p.bias;
    q.aux = grad ? dy : p.residual;
    q.out = p.y;
    q.bias_stride = p.bias_stride_e;
    q.ld_aux = grad ? ld_dy : p.ld_residual;
    q.ld_out = p.ldy;
    q.rows = (int)p.rows;
    q.experts = (int)p.experts;
    q.k_steps = (int)((p.k + BK - 1) / BK);
    const int width = p.gated ? 128 : BN;
    q.n_tiles = (int)((n_out + width - 1) / width);
    q.n_out = (int)n_out;
    q.w_second = p.gated ? (int)(gated_copy ? round8(n_out) : n_out) : 128;
    q.out_second = (int)n_out;
    q.idesc = idesc_f16(bf16, false, mn, BM, BN);
    q.act = p.activation;
    q.b_mn = mn;
    q.zero_rest = p.zero_rest != 0;
    q.vec_bias = vec8(p.bias, p.bias_stride_e, p.gated ? n_out : 0);
    q.vec_aux = vec8(q.aux, q.ld_aux);
    q.vec_out = vec8(p.y, p.ldy, grad && p.gated ? n_out : 0);
    int sms;
    if (int rc = sm_count(&sms)) return rc;
    const int64_t most = ((p.rows + BM - 1) / BM + (p.experts < p.rows ? p.experts : p.rows)) * q.n_tiles;
    const int grid = (int)(most < sms ? most : sms);
    if (grad) return p.gated ? launch<EPI_GRAD, true>(bf16, ma, mb, q, grid, s) : launch<EPI_GRAD, false>(bf16, ma, mb, q, grid, s);
    return p.gated ? launch<EPI_FORWARD, true>(bf16, ma, mb, q, grid, s) : launch<EPI_FORWARD, false>(bf16, ma, mb, q, grid, s);
}

__global__ void take_errors_kernel(int* out) { *out = atomicExch(&g_wait_error, 0); }

}  // namespace

int rows_product_rotated(const uint16_t* x, const uint16_t* w, const int64_t* offsets, int64_t rows, int64_t k, int64_t n,
                         int64_t experts, const uint16_t* svh, int64_t svh_stride, const float* row_scale, void* y, int64_t ldy,
                         bool bf16_out, cudaStream_t s) {
    const char* what = "rows_product_rotated";
    CUtensorMap ma, mb;
    if (int rc = map_rows_2d(&ma, operand(x, 1, rows, k, 0, k), false, BK, BM, what)) return rc;
    if (int rc = map_rows(&mb, operand(w, experts, n, k, n * k, k), false, BK, BN / 2, what)) return rc;
    Params q{};
    if (int rc = wait_error_word(&q.err)) return rc;
    q.offsets = offsets;
    q.aux = svh;
    q.ld_aux = svh_stride;
    q.row_scale = row_scale;
    q.out = y;
    q.ld_out = ldy;
    q.rows = (int)rows;
    q.experts = (int)experts;
    q.k_steps = (int)((k + BK - 1) / BK);
    q.n_tiles = (int)((n + BN - 1) / BN);
    q.n_out = (int)n;
    q.w_second = 128;
    q.idesc = idesc_f16(false, false, false, BM, BN);
    q.vec_aux = vec8(svh, svh_stride);
    q.vec_out = vec8(y, ldy);
    int sms;
    if (int rc = sm_count(&sms)) return rc;
    const int64_t most = ((rows + BM - 1) / BM + (experts < rows ? experts : rows)) * q.n_tiles;
    return launch<EPI_ROTATED, false>(bf16_out, ma, mb, q, (int)(most < sms ? most : sms), s);
}

int wait_error_word(int** out) {
    void* p = nullptr;
    cudaError_t e = cudaGetSymbolAddress(&p, g_wait_error);
    if (e != cudaSuccess) { set_error("cudaGetSymbolAddress: %s", cudaGetErrorString(e)); return KQ_ERR_CUDA; }
    *out = static_cast<int*>(p);
    return KQ_OK;
}

}  // namespace kq

extern "C" size_t kq_expert_linear_workspace_bytes(const kq_expert_product* p) {
    if (!p || kq::check_product(*p, "kq_expert_linear_workspace_bytes")) return 0;
    return kq::product_workspace(*p);
}

extern "C" int kq_expert_linear(const kq_expert_product* p, void* workspace, size_t workspace_bytes, void* stream) {
    if (!p) { kq::set_error("kq_expert_linear: null pointer"); return KQ_ERR_ARG; }
    return kq::rows_product(*p, nullptr, 0, workspace, workspace_bytes, static_cast<cudaStream_t>(stream), "kq_expert_linear");
}

extern "C" int kq_expert_linear_grad_z(const kq_expert_product* p, const void* dy, int64_t ld_dy, void* workspace,
                                       size_t workspace_bytes, void* stream) {
    if (!p || (!dy && p->rows > 0)) { kq::set_error("kq_expert_linear_grad_z: null pointer"); return KQ_ERR_ARG; }
    return kq::rows_product(*p, dy, ld_dy, workspace, workspace_bytes, static_cast<cudaStream_t>(stream),
                            "kq_expert_linear_grad_z");
}

namespace kq {
namespace {

// dW as stored: rows along k (columns n contiguous) or rows along n.
struct SumsSides { Operand a, b; int64_t m, n; };

SumsSides sums_sides(const kq_expert_product& p, const void* dz, int64_t ld_dz) {
    const Operand x = operand(p.x, 1, p.rows, p.k, 0, p.ldx), z = operand(dz, 1, p.rows, p.n, 0, ld_dz);
    return n_contiguous(p) ? SumsSides{x, z, p.k, p.n} : SumsSides{z, x, p.n, p.k};
}

}  // namespace
}  // namespace kq

extern "C" size_t kq_expert_weight_grad_workspace_bytes(const kq_expert_product* p, const void* dz, int64_t ld_dz) {
    using namespace kq;
    if (!p || check_product(*p, "kq_expert_weight_grad_workspace_bytes")) return 0;
    const SumsSides o = sums_sides(*p, dz, ld_dz);
    const size_t n = relayout_bytes(o.a) + relayout_bytes(o.b);
    return n ? n + 64 : 0;
}

extern "C" int kq_expert_weight_grad(const kq_expert_product* pp, const void* dz, int64_t ld_dz, void* dw, void* workspace,
                                     size_t workspace_bytes, void* stream) {
    using namespace kq;
    const char* what = "kq_expert_weight_grad";
    if (!pp) { set_error("%s: null pointer", what); return KQ_ERR_ARG; }
    const kq_expert_product& p = *pp;
    if (int rc = check_product(p, what)) return rc;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (!dw || (p.rows > 0 && (!p.x || !dz))) { set_error("%s: null pointer", what); return KQ_ERR_ARG; }
    const bool mn = n_contiguous(p), bf16 = p.dtype == KQ_BF16;
    const int64_t ld = mn ? p.w_stride_k : p.w_stride_n, cols = mn ? p.n : p.k, lines = mn ? p.k : p.n;
    if ((lines > 1 && ld < cols) || (p.experts > 1 && p.w_stride_e < (lines - 1) * ld + cols)) {
        set_error("%s: dW's strides overlap", what);
        return KQ_ERR_ARG;
    }
    if (p.rows == 0) {                          // nothing to sum: zeros, line by line
        for (int64_t e = 0; e < p.experts; ++e) {
            cudaError_t rc = cudaMemset2DAsync(static_cast<uint16_t*>(dw) + e * p.w_stride_e, (size_t)(lines > 1 ? ld : cols) * 2, 0,
                                               (size_t)cols * 2, (size_t)lines, s);
            if (rc != cudaSuccess) { set_error("%s: %s", what, cudaGetErrorString(rc)); return KQ_ERR_CUDA; }
        }
        return KQ_OK;
    }
    const size_t need = kq_expert_weight_grad_workspace_bytes(pp, dz, ld_dz);
    if (need && (workspace_bytes < need || !workspace)) {
        set_error("%s: workspace too small", what);
        return KQ_ERR_WORKSPACE;
    }
    if ((uintptr_t)workspace & 15) { set_error("%s: workspace must be 16-byte aligned", what); return KQ_ERR_ALIGN; }
    uint16_t* ws = static_cast<uint16_t*>(workspace);
    SumsSides o = sums_sides(p, dz, ld_dz);
    if (int rc = relayout(o.a, ws, 1, s)) return rc;
    if (int rc = relayout(o.b, ws, 1, s)) return rc;
    CUtensorMap ma, mb;
    if (int rc = map_rows_2d(&ma, o.a, bf16, 64, BK, what)) return rc;
    if (int rc = map_rows_2d(&mb, o.b, bf16, 64, BK, what)) return rc;
    Params q{};
    if (int rc = wait_error_word(&q.err)) return rc;
    q.offsets = p.offsets;
    q.out = dw;
    q.ld_out = ld;
    q.out_stride = p.w_stride_e;
    q.rows = (int)p.rows;
    q.experts = (int)p.experts;
    q.m_tiles = (int)((o.m + BM - 1) / BM);
    q.n_tiles = (int)((o.n + BN - 1) / BN);
    q.m_out = (int)o.m;
    q.n_out = (int)o.n;
    q.idesc = idesc_f16(bf16, true, true, BM, BN);
    q.a_mn = q.b_mn = true;
    q.vec_out = vec8(dw, ld, p.experts > 1 ? p.w_stride_e : 0);
    if ((int64_t)q.m_tiles * q.n_tiles > 0x7FFFFFFF) { set_error("%s: problem too large", what); return KQ_ERR_ARG; }
    int sms;
    if (int rc = sm_count(&sms)) return rc;
    const int64_t tiles = (int64_t)q.m_tiles * q.n_tiles * p.experts;
    return launch<EPI_SUMS, false>(bf16, ma, mb, q, (int)(tiles < sms ? tiles : sms), s);
}

extern "C" int kq_expert_bias_grad(const void* dz, int64_t ld_dz, const int64_t* offsets, int64_t rows, int64_t n,
                                   int64_t experts, int dtype, void* db, int64_t db_stride_e, void* stream) {
    using namespace kq;
    const char* what = "kq_expert_bias_grad";
    if (!db || (rows > 0 && !dz) || rows < 0 || n <= 0 || experts <= 0 || experts > kMaxExperts || (experts > 1 && !offsets) ||
        rows > 0x7FFFFF00 || n > 0x7FFFFF00 || (dtype != KQ_BF16 && dtype != KQ_FP16)) {
        set_error("%s: bad arguments (rows=%lld n=%lld experts=%lld)", what, (long long)rows, (long long)n, (long long)experts);
        return KQ_ERR_ARG;
    }
    const dim3 grid((unsigned)((n + 31) / 32), (unsigned)experts);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (dtype == KQ_BF16)
        bias_grad_kernel<<<grid, 256, 0, s>>>(static_cast<const __nv_bfloat16*>(dz), ld_dz, offsets, (int)rows, (int)n,
                                              static_cast<__nv_bfloat16*>(db), db_stride_e);
    else
        bias_grad_kernel<<<grid, 256, 0, s>>>(static_cast<const __half*>(dz), ld_dz, offsets, (int)rows, (int)n,
                                              static_cast<__half*>(db), db_stride_e);
    return check_launch(what);
}

extern "C" int kq_wait_errors(int32_t* out, void* stream) {
    if (!out) { kq::set_error("kq_wait_errors: null pointer"); return KQ_ERR_ARG; }
    kq::take_errors_kernel<<<1, 1, 0, static_cast<cudaStream_t>(stream)>>>(out);
    return kq::check_launch("kq_wait_errors");
}
