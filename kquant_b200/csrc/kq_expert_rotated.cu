// Rows product on decoded trellis weights with the output rotation in its
// epilogue:  y[r] = had128(x'[r] What_e) * svh_e * row_scale[r].
//
// One CTA per 128 x 256 tile, persistent: rows on the M axis, so that a thread
// drains one row of one 128-column Hadamard block and the transform (7 x 64
// butterflies) stays in its registers, under the next tile's products.
#include "kq_expert_rows.cuh"

namespace kq {
namespace {

constexpr int BM = 128, BN = 256, BK = 64, STAGES = 4;
constexpr int A_BYTES = BM * BK * 2, B_BYTES = BN * BK * 2, STAGE_BYTES = A_BYTES + B_BYTES;
constexpr uint32_t kIdesc = idesc_f16(false, false, false, BM, BN);
constexpr int DRAIN_WARPS = 8, THREADS = 64 + 32 * DRAIN_WARPS;
constexpr int GROUP_BYTES = (3 * kMaxExperts + 4) * 4;
constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + GROUP_BYTES + 1024;

struct Params {
    const int64_t *offsets, *all;   // of this call's experts, and of all experts of the rows
    const __half* svh;
    const float* row_scale;
    void* out;
    int64_t svh_stride, ld_out;
    int rows, experts, all_experts, k_steps, n_tiles, n_out;
    int* err;
    bool vec_svh, vec_out, zero_rest;
};

struct Tile { int e, row0, count, n0; };

__device__ __forceinline__ bool tile_at(const Params& p, const int* lo, const int* cnt, const int* cum, int64_t t, Tile& o) {
    if (t >= (int64_t)cum[p.experts] * p.n_tiles) return false;
    o.e = expert_of(cum, p.experts, (int)(t / p.n_tiles));
    const int mt = cum[o.e + 1] - cum[o.e];
    const int64_t l = t - (int64_t)cum[o.e] * p.n_tiles;
    const int m0 = (int)(l % mt) * BM;
    o.n0 = (int)(l / mt) * BN;
    o.row0 = lo[o.e] + m0;
    o.count = cnt[o.e] - m0;
    return true;
}

template <typename T>
__global__ void __launch_bounds__(THREADS, 1)
rotated_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const Params p) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t full_bar[STAGES], empty_bar[STAGES], acc_full[2], acc_empty[2];
    __shared__ uint32_t tmem_slot;
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    int* lo = reinterpret_cast<int*>(smem + STAGES * STAGE_BYTES);
    int* cnt = lo + kMaxExperts;
    int* cum = cnt + kMaxExperts;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

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
            for (int64_t i = blockIdx.x; ok && tile_at(p, lo, cnt, cum, i, t); i += gridDim.x) {
                for (int ks = 0; ks < p.k_steps; ++ks, ++it) {
                    const int s = it % STAGES;
                    if (!(ok = mbar_wait(&empty_bar[s], ((it / STAGES) & 1) ^ 1))) break;
                    mbar_expect_tx(&full_bar[s], STAGE_BYTES);
                    uint8_t *sa = smem + s * STAGE_BYTES, *sb = sa + A_BYTES;
                    tma_load_2d(sa, &map_a, ks * BK, t.row0, &full_bar[s]);
                    tma_load_3d(sb, &map_b, ks * BK, t.n0, t.e, &full_bar[s]);
                    tma_load_3d(sb + B_BYTES / 2, &map_b, ks * BK, t.n0 + 128, t.e, &full_bar[s]);
                }
            }
            if (!ok) report_wait_error(p.err);
        }
    } else if (warp == 1) {
        uint32_t it = 0, tile_no = 0;
        for (int64_t i = blockIdx.x; ok && tile_at(p, lo, cnt, cum, i, t); i += gridDim.x, ++tile_no) {
            const int b = tile_no & 1;
            if (!(ok = mbar_wait(&acc_empty[b], ((tile_no >> 1) & 1) ^ 1))) break;
            tc_fence_after();
            for (int ks = 0; ks < p.k_steps; ++ks, ++it) {
                const int s = it % STAGES;
                if (!(ok = mbar_wait(&full_bar[s], (it / STAGES) & 1))) break;
                uint8_t* sa = smem + s * STAGE_BYTES;
                tc_fence_after();
                if (lane == 0) {
                    const uint32_t a = smem_addr(sa);
                    const uint64_t ad = smem_desc(a), bd = smem_desc(a + A_BYTES);
#pragma unroll
                    for (int kk = 0; kk < BK / 16; ++kk)
                        mma_f16(tmem + b * BN, ad + 2 * kk, bd + 2 * kk, kIdesc, (ks | kk) != 0);
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
        for (int64_t i = blockIdx.x; tile_at(p, lo, cnt, cum, i, t); i += gridDim.x, ++tile_no) {
            const int b = tile_no & 1;
            if (!(ok = __all_sync(0xFFFFFFFFu, mbar_wait(&acc_full[b], (tile_no >> 1) & 1)))) break;
            tc_fence_after();
            const uint32_t base = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(b * BN);
            const int n_base = t.n0 + h * 128;
            if (n_base < p.n_out) {
                // A thread holds one row of one 128-column Hadamard block: the transform stays in its registers.
                {
                    float z[128];
#pragma unroll
                    for (int c = 0; c < 128; c += 16) {
                        uint32_t v[16];
                        tmem_ld16(base + h * 128 + c, v);
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
                    if (r < t.count) {
                        const float scale = p.row_scale[t.row0 + r] * 0.08838834764831845f;   // 1 / sqrt(128)
                        const __half* svh = p.svh + t.e * p.svh_stride + n_base;
                        T* orow = static_cast<T*>(p.out) + (int64_t)(t.row0 + r) * p.ld_out + n_base;
#pragma unroll
                        for (int c = 0; c < 128; c += 8) {
                            float a[8];
                            load8(svh + c, p.vec_svh, 8, a);
#pragma unroll
                            for (int e = 0; e < 8; ++e) a[e] = z[c + e] * a[e] * scale;      // scale last: z * scale may be beyond fp32
                            store8(orow + c, p.vec_out, 8, a);
                        }
                    }
                    __syncwarp();
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&acc_empty[b]);
        }
        if (!ok && lane == 0) report_wait_error(p.err);
        if (p.zero_rest && p.offsets) {
            int begin, end, n;
            group_of(p.all, 0, p.rows, begin, n);
            group_of(p.all, p.all_experts - 1, p.rows, end, n);
            end += n;
            for (int row = blockIdx.x; row < p.rows; row += gridDim.x) {
                if (row >= begin && row < end) continue;
                T* o = static_cast<T*>(p.out) + (int64_t)row * p.ld_out;
                for (int j = threadIdx.x - 64; j < p.n_out; j += 32 * DRAIN_WARPS) o[j] = from_f<T>(0.f);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) tmem_free(tmem, 2 * BN);
}


template <typename T>
int launch(const CUtensorMap& a, const CUtensorMap& b, const Params& p, int grid, cudaStream_t s) {
    cudaError_t e = cudaFuncSetAttribute(rotated_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES);
    if (e != cudaSuccess) { set_error("cudaFuncSetAttribute: %s", cudaGetErrorString(e)); return KQ_ERR_CUDA; }
    rotated_kernel<T><<<grid, THREADS, SMEM_BYTES, s>>>(a, b, p);
    return check_launch("rotated_kernel");
}

}  // namespace

int rows_product_rotated(const uint16_t* x, const uint16_t* w, const int64_t* offsets, int64_t rows, int64_t k, int64_t n,
                         int64_t all_experts, int64_t first, int64_t experts, const uint16_t* svh, int64_t svh_stride, const float* row_scale, void* y, int64_t ldy,
                         bool bf16_out, bool zero_rest, int* err, cudaStream_t s) {
    const char* what = "rows_product_rotated";
    CUtensorMap ma, mb;
    const int64_t xd[2] = {k, rows}, xs[1] = {k * 2}, wd[3] = {k, n, experts}, wst[2] = {k * 2, n * k * 2};
    const int xb[2] = {BK, BM}, wb[3] = {BK, BN / 2, 1};
    if (int rc = encode_tiles(&ma, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, x, xd, xs, xb, what)) return rc;
    if (int rc = encode_tiles(&mb, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, w, wd, wst, wb, what)) return rc;
    Params q{};
    q.err = err;
    q.offsets = offsets ? offsets + first : nullptr;
    q.all = offsets;
    q.all_experts = (int)all_experts;
    q.svh = reinterpret_cast<const __half*>(svh) + first * svh_stride;
    q.svh_stride = svh_stride;
    q.row_scale = row_scale;
    q.out = y;
    q.ld_out = ldy;
    q.rows = (int)rows;
    q.experts = (int)experts;
    q.k_steps = (int)((k + BK - 1) / BK);
    q.n_tiles = (int)((n + BN - 1) / BN);
    q.n_out = (int)n;
    q.zero_rest = zero_rest && first == 0;
    q.vec_svh = ((uintptr_t)svh & 15) == 0 && svh_stride % 8 == 0;
    q.vec_out = ((uintptr_t)y & 15) == 0 && ldy % 8 == 0;
    int sms;
    if (int rc = sm_count(&sms)) return rc;
    const int64_t most = ((rows + BM - 1) / BM + (experts < rows ? experts : rows)) * q.n_tiles;
    const int grid = (int)(most < sms ? most : sms);
    return bf16_out ? launch<__nv_bfloat16>(ma, mb, q, grid, s) : launch<__half>(ma, mb, q, grid, s);
}

}  // namespace kq
