// Rows product for few rows an expert, where reading W is what it costs:
//
//   y[r] = epilogue(x[r] W_e + b_e),  or dz from dy
//
// A CTA holds 128 features of W (gated: 128 of gate and the same of up) on the
// M axis of the tensor product and up to 128 rows on the N axis, so that a row
// tile costs what its rows need.  The contraction is split over the CTAs of a
// cluster: one matrix of 2048 features is 16 feature tiles, which alone would
// leave 132 SMs without a share of the reading.  Every CTA accumulates its
// range of k in tensor memory, the partial sums meet in distributed shared
// memory, and each CTA of the cluster adds up (in rank order: the same bits
// every time) and finishes its share of the features.
//
// Two CTAs share an SM with 100 KB of loads in flight each where that is at
// least three stages: the epilogue of one runs under the loads of the other.
#include "kq_expert_rows.cuh"

namespace kq {
namespace {

constexpr int BK = 64, MAX_STAGES = 8, THREADS = 128;
constexpr int SIDE = 128 * BK * 2;              // 128 features of a stage
constexpr int CHUNK = 64 * 128;
constexpr int RING_TWO = 102 * 1024, RING_ONE = 208 * 1024;   // two CTAs an SM, or one
constexpr int X_BOX = 32;                       // rows of x that one TMA box brings (16 when the tile has 16)
constexpr int PART = 32;                        // rows that are finished at a time

struct Params {
    const int64_t* offsets;
    const void *bias, *aux;
    void *out, *low;
    int64_t bias_stride, ld_aux, ld_out;
    int rows, experts, k_steps, m_out, up, nt, box, stages, splits, act;
    uint32_t idesc, tmem_cols;   // idesc without N
    int* err;
    bool mn, grad, zero_rest;
};

__device__ __forceinline__ float load_cluster(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr));
    return v;
}

__device__ __forceinline__ uint32_t rank_addr(uint32_t addr, int rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}

__device__ __forceinline__ float act_of(int act, float z) {
    switch (act) {
        case KQ_ACT_RELU: return activate<KQ_ACT_RELU>(z);
        case KQ_ACT_SILU: return activate<KQ_ACT_SILU>(z);
        case KQ_ACT_GELU: return activate<KQ_ACT_GELU>(z);
        default: return z;
    }
}

__device__ __forceinline__ float slope_of(int act, float z) {
    switch (act) {
        case KQ_ACT_RELU: return slope<KQ_ACT_RELU>(z);
        case KQ_ACT_SILU: return slope<KQ_ACT_SILU>(z);
        case KQ_ACT_GELU: return slope<KQ_ACT_GELU>(z);
        default: return 1.f;
    }
}

template <typename T, bool GATED>
__global__ void __launch_bounds__(THREADS)
few_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const Params p) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t full_bar[MAX_STAGES], empty_bar[MAX_STAGES], done_bar;
    __shared__ uint32_t tmem_slot;
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        tma_prefetch(&map_w);
        tma_prefetch(&map_x);
    }
    const int rank = p.splits > 1 ? (int)cluster_rank() : 0;
    const int m0 = (int)(blockIdx.x / p.splits) * 128;

    // The groups are needed for this tile's place alone: their scan borrows the ring before the first load.
    int* lo = reinterpret_cast<int*>(smem);
    int* cnt = lo + kMaxExperts;
    int* cum = cnt + kMaxExperts;
    scan_groups(p.offsets, p.experts, p.rows, p.nt, lo, cnt, cum);
    const int t = blockIdx.y;
    const bool mine = t < cum[p.experts];
    int e = 0, row0 = 0, count = 0;
    if (mine) {
        e = expert_of(cum, p.experts, t);
        const int r = (t - cum[e]) * p.nt;
        row0 = lo[e] + r;
        count = min(cnt[e] - r, p.nt);
    }
    if (p.zero_rest && p.offsets && rank == 0) {          // rows of no expert in a fresh output
        int end, n, begin;
        group_of(p.offsets, 0, p.rows, begin, n);
        group_of(p.offsets, p.experts - 1, p.rows, end, n);
        end += n;
        const int f = m0 + threadIdx.x;
        for (int row = t; row < p.rows; row += gridDim.y)
            if ((row < begin || row >= end) && f < p.m_out) static_cast<T*>(p.out)[(int64_t)row * p.ld_out + f] = from_f<T>(0.f);
    }
    if (!mine) return;                                    // the whole cluster, which shares blockIdx.y

    if (threadIdx.x == 0) {
        for (int s = 0; s < p.stages; ++s) {
            mbar_init(&full_bar[s], 1);
            mbar_init(&empty_bar[s], 1);
        }
        mbar_init(&done_bar, 1);
        mbar_init_fence();
    }
    __syncwarp();                                         // lane 0 was apart; what is .aligned needs its whole warp
    if (warp == 0) tmem_alloc(&tmem_slot, p.tmem_cols);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    const int k0 = (int)((int64_t)p.k_steps * rank / p.splits), k1 = (int)((int64_t)p.k_steps * (rank + 1) / p.splits);
    constexpr int W_BYTES = GATED ? 2 * SIDE : SIDE;
    const int stage_bytes = W_BYTES + p.nt * 128;
    const int boxes = (count + p.box - 1) / p.box;        // of x: the tile's rows and no more
    bool ok = true;

    if (warp == 0 && lane == 0) {
        for (int ks = k0; ks < k1; ++ks) {
            const int it = ks - k0, s = it % p.stages;
            if (!(ok = mbar_wait(&empty_bar[s], ((it / p.stages) & 1) ^ 1))) break;
            mbar_expect_tx(&full_bar[s], W_BYTES + boxes * p.box * 128);
            uint8_t* dst = smem + s * stage_bytes;
#pragma unroll
            for (int g = 0; g < (GATED ? 2 : 1); ++g) {
                const int f = m0 + (g ? p.up : 0);
                if (p.mn) {
                    tma_load_3d(dst + g * SIDE, &map_w, f, ks * BK, e, &full_bar[s]);
                    tma_load_3d(dst + g * SIDE + CHUNK, &map_w, f + 64, ks * BK, e, &full_bar[s]);
                } else {
                    tma_load_3d(dst + g * SIDE, &map_w, ks * BK, f, e, &full_bar[s]);
                }
            }
            for (int b = 0; b < boxes; ++b)
                tma_load_2d(dst + W_BYTES + b * p.box * 128, &map_x, ks * BK, row0 + b * p.box, &full_bar[s]);
        }
    } else if (warp == 1 && lane == 0) {
        const uint32_t a_step = p.mn ? 128 : 2;
        const uint32_t idesc = p.idesc | ((uint32_t)((count + 15) >> 4) << 18);      // N in units of 8, a multiple of 16
        for (int ks = k0; ks < k1; ++ks) {
            const int it = ks - k0, s = it % p.stages;
            if (!(ok = mbar_wait(&full_bar[s], (it / p.stages) & 1))) break;
            tc_fence_after();
            const uint32_t base = smem_addr(smem + s * stage_bytes);
            const uint64_t bd = smem_desc(base + W_BYTES);
#pragma unroll
            for (int g = 0; g < (GATED ? 2 : 1); ++g) {
                const uint64_t ad = smem_desc(base + g * SIDE, p.mn ? CHUNK : 16);
#pragma unroll
                for (int kk = 0; kk < BK / 16; ++kk)
                    mma_f16(tmem + g * p.nt, ad + a_step * kk, bd + 2 * kk, idesc, (it | kk) != 0);
            }
            mma_commit(&empty_bar[s]);
        }
        if (ok) mma_commit(&done_bar);
    }
    if (!ok) report_wait_error(p.err);
    __syncwarp();
    // What the epilogue reads from memory comes in under the products: the bias and the first rows of aux.
    const int width = 128 / p.splits, f0 = rank * width;
    auto load_aux = [&](float (&a)[4], int r, int step) {
        const int f = m0 + f0 + (threadIdx.x & (width - 1));
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int64_t row = row0 + min(r + u * step, count - 1);
            a[u] = p.aux && f < p.m_out ? to_f<T>(static_cast<const T*>(p.aux)[row * p.ld_aux + f]) : 0.f;
        }
    };
    float early[4], add = 0.f, add_up = 0.f;
    {
        const int shift = 31 - __clz(width), f = m0 + f0 + (threadIdx.x & (width - 1));
        load_aux(early, threadIdx.x >> shift, THREADS >> shift);
        if (p.bias && f < p.m_out) {
            const T* bias = static_cast<const T*>(p.bias) + e * p.bias_stride + f;
            add = to_f<T>(bias[0]);
            if constexpr (GATED) add_up = to_f<T>(bias[p.m_out]);
        }
    }
    if (!mbar_wait(&done_bar, 0)) {
        if (lane == 0) report_wait_error(p.err);
    }
    __syncwarp();
    tc_fence_after();

    // Partial sums [rows][128 features] (gate, then up) meet in shared memory, 32 rows at a time.
    float* part = reinterpret_cast<float*>(smem);
    const uint32_t part_addr = smem_addr(part);
    for (int c0 = 0; c0 < count; c0 += PART) {
        const int n = min(PART, count - c0);
        const uint32_t base = tmem + ((uint32_t)(warp * 32) << 16) + (uint32_t)c0;
        for (int j = 0; j < n; j += 16) {
            uint32_t v[16], u[16];
            tmem_ld16(base + j, v);
            if constexpr (GATED) tmem_ld16(base + p.nt + j, u);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                part[(j + i) * 128 + threadIdx.x] = __uint_as_float(v[i]);
                if constexpr (GATED) part[(PART + j + i) * 128 + threadIdx.x] = __uint_as_float(u[i]);
            }
        }
        if (p.splits > 1) cluster_sync();
        else __syncthreads();
        // A thread keeps its feature (128 threads are whole rows of `width` features) and takes four rows at a time.
        const int shift = 31 - __clz(width), f = f0 + (threadIdx.x & (width - 1)), step = THREADS >> shift;
        if (m0 + f < p.m_out) {
            for (int r = threadIdx.x >> shift; r < n; r += 4 * step) {
                float a[4], z[4], w[4];
                if (c0 > 0 || r >= 4 * step) load_aux(a, c0 + r, step);
                else
#pragma unroll
                    for (int u = 0; u < 4; ++u) a[u] = early[u];
#pragma unroll
                for (int u = 0; u < 4; ++u) { z[u] = 0.f; w[u] = 0.f; }
                for (int s = 0; s < p.splits; ++s) {
                    const uint32_t at = p.splits > 1 ? rank_addr(part_addr, s) : part_addr;
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const uint32_t from = at + (uint32_t)(min(r + u * step, PART - 1) * 128 + f) * 4;
                        z[u] += load_cluster(from);
                        if constexpr (GATED) w[u] += load_cluster(from + PART * 128 * 4);
                    }
                }
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    if (r + u * step >= n) break;
                    const int64_t to = (int64_t)(row0 + c0 + r + u * step) * p.ld_out + m0 + f;
                    T *o = static_cast<T*>(p.out) + to, *low = static_cast<T*>(p.low) + to;
                    const float zz = z[u] + add, ww = w[u] + add_up;
                    if (!p.grad) {
                        o[0] = from_f<T>(act_of(p.act, zz) * (GATED ? ww : 1.f) + a[u]);
                    } else if constexpr (GATED) {
                        const float dg = a[u] * ww * slope_of(p.act, zz), du = a[u] * act_of(p.act, zz);
                        o[0] = from_f<T>(dg);
                        o[p.m_out] = from_f<T>(du);
                        if (p.low) {
                            low[0] = from_f<T>(left_out<T>(dg));
                            low[p.m_out] = from_f<T>(left_out<T>(du));
                        }
                    } else {
                        const float dz = a[u] * slope_of(p.act, zz);
                        o[0] = from_f<T>(dz);
                        if (p.low) low[0] = from_f<T>(left_out<T>(dz));
                    }
                }
            }
        }
        __syncwarp();                                     // lanes without a row or feature left the loop early
        if (p.splits > 1) cluster_sync();                 // the others are done with this CTA's part
        else __syncthreads();
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) tmem_free(tmem, p.tmem_cols);
}

template <typename T, bool GATED>
int launch(const CUtensorMap& w, const CUtensorMap& x, const Params& p, int smem, dim3 grid, cudaStream_t s) {
    auto kernel = few_kernel<T, GATED>;
    // The attribute is the kernel's, for every thread of the process: always the most that a call can need.
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, RING_ONE + 1024);
    if (e != cudaSuccess) { set_error("cudaFuncSetAttribute: %s", cudaGetErrorString(e)); return KQ_ERR_CUDA; }
    cudaLaunchConfig_t c{};
    c.gridDim = grid;
    c.blockDim = dim3(THREADS);
    c.dynamicSmemBytes = (size_t)smem;
    c.stream = s;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim = {(unsigned)p.splits, 1, 1};
    c.attrs = &at;
    c.numAttrs = p.splits > 1 ? 1 : 0;
    e = cudaLaunchKernelEx(&c, kernel, w, x, p);
    if (e != cudaSuccess) { set_error("few_kernel: %s", cudaGetErrorString(e)); return KQ_ERR_CUDA; }
    return check_launch("few_kernel");
}

}  // namespace

// Up to 16 rows an expert always; up to 48 where W's rows are long enough for its reading to be what counts (8 experts of
// 7168 -> 4096 gated: 74 us against 82 us at 16 rows, 80 and 83 at 48; 1024 -> 1024: 17 and 14 us at 24).  And however many
// where the other kernel's tiles of 256 x 256 would leave most SMs without work and k is worth splitting (7168 -> 2048, 64
// rows: 21 us against 55 us; 5388 -> 39, 174 rows: 40 us against 65 us).
bool few_rows(const RowsProduct& p) {
    const int64_t busy = p.experts < p.rows ? p.experts : p.rows;
    const int64_t tiles = (p.n_out * (p.gated ? 2 : 1) + 255) / 256 * ((p.rows + 255) / 256 + busy - 1);
    return p.rows <= 16 * busy || (p.k >= 2048 && (p.rows <= 48 * busy || tiles <= 18));
}

int few_rows_product(const RowsProduct& p, cudaStream_t s) {
    const int64_t busy = p.experts < p.rows ? p.experts : p.rows, mean = (p.rows + busy - 1) / busy;
    Params q{};
    q.err = p.err;
    q.nt = mean <= 8 ? 16 : mean <= 16 ? 32 : mean <= 32 ? 64 : 128;     // twice the mean: uneven experts mostly fit one tile
    q.offsets = p.offsets;
    q.bias = p.bias;
    q.aux = p.aux;
    q.out = p.out;
    q.low = p.low;
    q.bias_stride = p.bias_stride;
    q.ld_aux = p.ld_aux;
    q.ld_out = p.ld_out;
    q.rows = (int)p.rows;
    q.experts = (int)p.experts;
    q.k_steps = (int)((p.k + BK - 1) / BK);
    q.m_out = (int)p.n_out;
    q.up = p.up;
    q.act = p.act;
    q.mn = p.mn;
    q.grad = p.grad;
    q.zero_rest = p.zero_rest;
    const int stage = (p.gated ? 2 : 1) * SIDE + q.nt * 128;
    // Two short rings on an SM hide each other's ends; where they would hold two stages only, one long ring is better.
    const int ring = RING_TWO / stage >= 3 ? RING_TWO : RING_ONE;
    q.stages = ring / stage < MAX_STAGES ? ring / stage : MAX_STAGES;
    q.box = q.nt < X_BOX ? q.nt : X_BOX;
    q.idesc = idesc_f16(p.bf16, p.mn, false, 128, 0);
    q.tmem_cols = 32;
    while ((int)q.tmem_cols < q.nt * (p.gated ? 2 : 1)) q.tmem_cols <<= 1;
    // Row tiles that the offsets can make: every busy expert's first, and one more for each nt rows beyond.
    const int64_t m_tiles = (p.n_out + 127) / 128, r_tiles = busy + (p.rows - busy) / q.nt;
    int sms;
    if (int rc = sm_count(&sms)) return rc;
    q.splits = 1;
    while (q.splits < 8 && m_tiles * r_tiles * q.splits * 2 <= 2 * sms && q.k_steps >= 4 * q.splits) q.splits *= 2;
    CUtensorMap mw, mx;
    if (int rc = map_rows(&mw, p.w, p.bf16, 64, p.mn ? 64 : 128, p.what)) return rc;
    if (int rc = map_rows_2d(&mx, p.x, p.bf16, BK, q.box, p.what)) return rc;
    if (m_tiles * q.splits > 0x7FFFFFFF || r_tiles > 65535) { set_error("%s: problem too large", p.what); return KQ_ERR_ARG; }
    const dim3 grid((unsigned)(m_tiles * q.splits), (unsigned)r_tiles);
    if (p.bf16) return p.gated ? launch<__nv_bfloat16, true>(mw, mx, q, ring + 1024, grid, s) : launch<__nv_bfloat16, false>(mw, mx, q, ring + 1024, grid, s);
    return p.gated ? launch<__half, true>(mw, mx, q, ring + 1024, grid, s) : launch<__half, false>(mw, mx, q, ring + 1024, grid, s);
}

}  // namespace kq
