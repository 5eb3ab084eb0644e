// Product of many rows with encoded matrices, decoded on the way into the
// tensor cores:  y[r] = had128(x'[r] What_e) * svh_e * row_scale[r].
//
// A CTA takes 256 rows (two accumulators of 128 x 128) by one Hadamard block
// of columns, persistent.  Sixteen warps decode What's 64 x 128 part of each
// stage from the payload straight into the swizzled tile that the tensor core
// reads; x' comes by TMA.  What never is in memory: written and read back as
// binary16 it is 16/K times the payload twice over.  Two groups of eight warps
// take turns, a stage each, so that one waits for its words while the other
// decodes.  Rows on the M axis put a row of a Hadamard block in one thread of
// the epilogue, 32 columns at a time.
//
// Bound by the decoding's integer arithmetic (8 experts of 7168 x 4096 at 4
// bits, 32 rows each: 152 us, the ALU pipe 68% busy, HBM 9%); with more than
// 128 rows a tile the products' operands join in shared memory (256 rows: 222
// us), which E4M3 lookups already use (189 and 240 us).
#pragma once
#include "kq_expert_rows.cuh"
#include "kq_trellis_decode.cuh"

namespace kq {
namespace {

constexpr int RM = 128, RN = kBlock, RK = 64;
constexpr int R_A = RM * RK * 2, R_B = RN * RK * 2, R_STAGE = 2 * R_A + R_B;
constexpr int R_DECODE = 16, R_DRAIN = 4, R_THREADS = 32 * (2 + R_DECODE + R_DRAIN);
constexpr int R_GROUPS = (3 * kMaxExperts + 4) * 4;
constexpr int rows_stages(int dec) { return dec == DEC_MCG ? 4 : 3; }
constexpr int rows_smem(int dec) { return rows_stages(dec) * R_STAGE + table_bytes(dec) + R_GROUPS + 1024; }

struct RowsTile { int e, row0, count, n0; };

__device__ __forceinline__ bool rows_tile(const TrellisRows& p, const int* lo, const int* cnt, const int* cum, int64_t t, RowsTile& o) {
    const int nb = p.n / RN;
    if (t >= (int64_t)cum[p.experts] * nb) return false;
    o.e = expert_of(cum, p.experts, (int)(t / nb));
    const int mt = cum[o.e + 1] - cum[o.e];               // the row tiles of one column block run together
    const int64_t l = t - (int64_t)cum[o.e] * nb;
    const int m0 = (int)(l % mt) * 2 * RM;
    o.n0 = (int)(l / mt) * RN;
    o.row0 = lo[o.e] + m0;
    o.count = min(cnt[o.e] - m0, 2 * RM);
    return true;
}

template <int K, int DEC>
__global__ void __launch_bounds__(R_THREADS, 1) rows_trellis_kernel(const __grid_constant__ CUtensorMap map_x, const TrellisRows p) {
    constexpr int STAGES = rows_stages(DEC);
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t full_bar[STAGES], empty_bar[STAGES], acc_full[2], acc_empty[2];
    __shared__ uint32_t tmem_slot;
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t* table = smem + STAGES * R_STAGE;
    int* lo = reinterpret_cast<int*>(table + table_bytes(DEC));
    int* cnt = lo + kMaxExperts;
    int* cum = cnt + kMaxExperts;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, k_steps = p.k / RK;

    if (threadIdx.x == 0) {
        tma_prefetch(&map_x);
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&full_bar[s], 1 + R_DECODE / 2);
            mbar_init(&empty_bar[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&acc_full[b], 1);
            mbar_init(&acc_empty[b], R_DRAIN);
        }
        mbar_init_fence();
    }
    if (warp == 1) tmem_alloc(&tmem_slot, 512);
    load_table<DEC>(p.table, table);
    scan_groups(p.offsets, p.experts, p.rows, 2 * RM, lo, cnt, cum);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    bool ok = true;
    RowsTile t;

    if (warp == 0) {
        if (lane == 0) {
            wait_for_last();                     // x' is there
            uint32_t it = 0;
            for (int64_t i = blockIdx.x; ok && rows_tile(p, lo, cnt, cum, i, t); i += gridDim.x) {
                const bool two = t.count > RM;
                for (int ks = 0; ks < k_steps; ++ks, ++it) {
                    const int s = it % STAGES;
                    if (!(ok = mbar_wait(&empty_bar[s], ((it / STAGES) & 1) ^ 1))) break;
                    mbar_expect_tx(&full_bar[s], two ? 2 * R_A : R_A);
                    uint8_t* sa = smem + s * R_STAGE;
                    tma_load_2d(sa, &map_x, ks * RK, t.row0, &full_bar[s]);
                    if (two) tma_load_2d(sa + R_A, &map_x, ks * RK, t.row0 + RM, &full_bar[s]);
                }
            }
            if (!ok) report_wait_error(p.err);
        }
    } else if (warp == 1) {
        constexpr uint32_t idesc = idesc_f16(false, false, false, RM, RN);
        uint32_t it = 0, tile_no = 0;
        for (int64_t i = blockIdx.x; ok && rows_tile(p, lo, cnt, cum, i, t); i += gridDim.x, ++tile_no) {
            const uint32_t acc = tmem + (tile_no & 1) * 2 * RN;
            if (!(ok = mbar_wait(&acc_empty[tile_no & 1], ((tile_no >> 1) & 1) ^ 1))) break;
            tc_fence_after();
            for (int ks = 0; ks < k_steps; ++ks, ++it) {
                const int s = it % STAGES;
                if (!(ok = mbar_wait(&full_bar[s], (it / STAGES) & 1))) break;
                tc_fence_after();
                if (lane == 0) {
                    const uint32_t a = smem_addr(smem + s * R_STAGE);
                    const uint64_t bd = smem_desc(a + 2 * R_A);
                    for (int m = 0; m < (t.count > RM ? 2 : 1); ++m) {
                        const uint64_t ad = smem_desc(a + m * R_A);
#pragma unroll
                        for (int kk = 0; kk < RK / 16; ++kk)
                            mma_f16(acc + m * RN, ad + 2 * kk, bd + 2 * kk, idesc, (ks | kk) != 0);
                    }
                    mma_commit(&empty_bar[s]);
                }
                __syncwarp();
            }
            if (ok && lane == 0) mma_commit(&acc_full[tile_no & 1]);
            __syncwarp();
        }
        if (!ok && lane == 0) report_wait_error(p.err);
    } else if (warp < 2 + R_DECODE) {
        // Group g decodes the stages g, g + 2, ..; a warp 16 columns of 64 rows.  k is a multiple of 128: k_steps is even, so a
        // stage's parity is that of its place in the tile.
        const int g = (warp - 2) >> 3, col = (warp - 2) & 7, nt = p.n / 16;
        struct At { int64_t i; int ks; };
        auto source = [&](const At& at, const RowsTile& t) {
            return p.trellis + (((int64_t)t.e * (p.k / 16) + at.ks * (RK / 16)) * nt + t.n0 / 16 + col) * 8 * K;
        };
        TileWords<K> ahead[2][4];
        At next{blockIdx.x, g};                            // of the words to be fetched
        RowsTile nt_tile;
        bool more = rows_tile(p, lo, cnt, cum, next.i, nt_tile);
        auto fetch = [&](TileWords<K> (&w)[4]) {
            if (!more) return;
            const uint32_t* src = source(next, nt_tile);
#pragma unroll
            for (int a = 0; a < 4; ++a) w[a].load(src + (int64_t)a * nt * 8 * K, lane);
            if ((next.ks += 2) >= k_steps) {
                next.ks = g;
                next.i += gridDim.x;
                more = rows_tile(p, lo, cnt, cum, next.i, nt_tile);
            }
        };
        fetch(ahead[0]);
        fetch(ahead[1]);
        uint32_t it = g;
        // This lane's place in the stage: its row, chunk 0 turned by the row as the swizzle has it.
        uint32_t at = 2 * R_A + (col * 16 + (lane >> 2)) * 128 + (lane >> 2) * 16 + (lane & 3) * 4;
        asm volatile("" : "+r"(at));
        auto step = [&](TileWords<K> (&w)[4]) {
            const int s = it % STAGES;
            if (!(ok = __all_sync(0xFFFFFFFFu, mbar_wait(&empty_bar[s], ((it / STAGES) & 1) ^ 1)))) return;
            const uint32_t b = smem_addr(smem) + s * R_STAGE + at;
#pragma unroll
            for (int a = 0; a < 4; ++a) {
                uint32_t f[4];
                decode_tile<K, DEC>(w[a], lane, table, f);
                const uint32_t c0 = b ^ (a * 32), c1 = c0 ^ 16;       // 16-byte chunks 2a and 2a + 1 of the swizzled row
                asm volatile("st.shared.b32 [%0], %1;" ::"r"(c0), "r"(f[0]) : "memory");
                asm volatile("st.shared.b32 [%0], %1;" ::"r"(c1), "r"(f[1]) : "memory");
                asm volatile("st.shared.b32 [%0 + 1024], %1;" ::"r"(c0), "r"(f[2]) : "memory");
                asm volatile("st.shared.b32 [%0 + 1024], %1;" ::"r"(c1), "r"(f[3]) : "memory");
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&full_bar[s]);
            it += 2;
            fetch(w);
        };
        // Two stages a round; a tile has k_steps / 2 of each group's.
        int64_t i = blockIdx.x;
        int left = 0;
        auto begin = [&]() {
            if (left) return true;
            if (!rows_tile(p, lo, cnt, cum, i, t)) return false;
            i += gridDim.x;
            left = k_steps / 2;
            return true;
        };
        while (ok) {
            if (!begin()) break;
            step(ahead[0]);
            --left;
            if (!ok || !begin()) break;
            step(ahead[1]);
            --left;
        }
        if (!ok && lane == 0) report_wait_error(p.err);
    } else {
        const int q = warp & 3;
        uint32_t tile_no = 0;
        for (int64_t i = blockIdx.x; rows_tile(p, lo, cnt, cum, i, t); i += gridDim.x, ++tile_no) {
            const int b = tile_no & 1;
            if (!(ok = __all_sync(0xFFFFFFFFu, mbar_wait(&acc_full[b], (tile_no >> 1) & 1)))) break;
            tc_fence_after();
            wait_for_last();                     // row_scale, as this thread sees it
            const __half* svh = p.svh + t.e * p.svh_stride + t.n0;
            for (int m = 0; m < (t.count > RM ? 2 : 1); ++m) {
                const uint32_t base = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(b * 2 * RN + m * RN);
                const int r = m * RM + q * 32 + lane;
                const bool live = r < t.count;
                const float scale = (live ? p.row_scale[t.row0 + r] : 0.f) * 0.08838834764831845f;      // 1 / sqrt(128)
                const int64_t at = (int64_t)(t.row0 + (live ? r : 0)) * p.ldy + t.n0;
                // The transform of 128 is that of 4 over blocks of 32 (signs here), then that of 32 in registers.
#pragma unroll 1
                for (int o = 0; o < 4; ++o) {
                    float z[32];
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const float sign = __popc(o & c) & 1 ? -1.f : 1.f;
#pragma unroll
                        for (int h = 0; h < 32; h += 16) {
                            uint32_t v[16];
                            tmem_ld16(base + c * 32 + h, v);
                            tmem_wait_ld();
#pragma unroll
                            for (int e = 0; e < 16; ++e) z[h + e] = c ? fmaf(sign, __uint_as_float(v[e]), z[h + e]) : __uint_as_float(v[e]);
                        }
                    }
#pragma unroll
                    for (int d = 1; d < 32; d <<= 1)
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if (!(e & d)) {
                                const float a = z[e], c = z[e + d];
                                z[e] = a + c;
                                z[e + d] = a - c;
                            }
                    if (live) {
#pragma unroll
                        for (int c = 0; c < 32; c += 8) {
                            float a[8];
                            load8(svh + o * 32 + c, p.vec_svh, 8, a);
#pragma unroll
                            for (int e = 0; e < 8; ++e) a[e] = z[c + e] * a[e] * scale;      // scale last: z * scale may be beyond fp32
                            if (p.bf16) store8(static_cast<__nv_bfloat16*>(p.y) + at + o * 32 + c, p.vec_y, 8, a);
                            else store8(static_cast<__half*>(p.y) + at + o * 32 + c, p.vec_y, 8, a);
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
            group_of(p.offsets, 0, p.rows, begin, n);
            group_of(p.offsets, p.experts - 1, p.rows, end, n);
            end += n;
            for (int row = blockIdx.x; row < p.rows; row += gridDim.x) {
                if (row >= begin && row < end) continue;
                uint16_t* o = static_cast<uint16_t*>(p.y) + (int64_t)row * p.ldy;
                for (int j = threadIdx.x - 32 * (2 + R_DECODE); j < p.n; j += 32 * R_DRAIN) o[j] = 0;
            }
        }
    }
    tc_fence_before();
    wait_for_last();
    __syncthreads();
    if (warp == 1) tmem_free(tmem, 512);
}

template <int K, int DEC>
int launch_rows(const TrellisRows& p, cudaStream_t s) {
    const char* what = "rows_trellis_kernel";
    CUtensorMap map;
    const int64_t dims[2] = {p.k, p.rows}, strides[1] = {(int64_t)p.k * 2};
    const int box[2] = {RK, RM};
    if (int rc = encode_tiles(&map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, p.xr, dims, strides, box, what)) return rc;
    constexpr int smem = rows_smem(DEC);
    auto kernel = rows_trellis_kernel<K, DEC>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) { set_error("cudaFuncSetAttribute: %s", cudaGetErrorString(e)); return KQ_ERR_CUDA; }
    int sms;
    if (int rc = sm_count(&sms)) return rc;
    const int64_t busy = p.experts < p.rows ? p.experts : p.rows;
    const int64_t most = (busy + (p.rows - busy) / (2 * RM)) * (p.n / RN);
    return launch_next(kernel, dim3((unsigned)(most < sms ? most : sms)), R_THREADS, smem, s, what, map, p);
}

template <int K>
int rows_trellis(const TrellisRows& p, int dec, cudaStream_t s) {
    return dec == DEC_MCG ? launch_rows<K, DEC_MCG>(p, s) : launch_rows<K, DEC_E4M3>(p, s);
}

}  // namespace
}  // namespace kq
