// Product of few rows with packed trellis tiles: decoded in registers, used once.
//
// The trellis order of a tile is the operand order of mma.m16n8k16: the eight
// labels that a lane decodes are its two B fragments (columns 0..7 and 8..15
// of the tile), so a decoded tile goes from registers into the products of up
// to 64 rows without touching memory.  Decoding is what bounds this (the
// products of 64 rows take half of its time even on mma.sync), at three bits:
// label lookups in shared memory for the tables (E4M3: 83% of its cycles),
// integer arithmetic for MCG (8 experts of 7168 x 4096 at 4 bits, one row
// each: 104 us, ALU pipe 71%, issue slots 62%, DRAM idle for the most part).
//
// The work is dealt to a persistent grid of two CTAs an SM in equal shares of
// k tiles, wherever strips of columns end: with whole strips the last round
// of CTAs left SMs idle, with short items each began with a wait for memory.
// A CTA's warps take the k tiles of a share in turn, each with its words two
// steps ahead in registers, and add up in shared memory in a fixed order; the
// output transform adds up a strip's shares.
#pragma once
#include "kq_trellis_decode.cuh"

namespace kq {
namespace {

// Warps of a CTA: 24 an SM hide the lookups' latency where the registers allow it (16 rows), 16 with 64 rows' sums.
template <int RT> constexpr int few_warps() { return RT == 1 ? 12 : 8; }

__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// RT: row tiles of 16.
template <int RT> constexpr int few_strip() { return few_columns(RT > 1) / 16; }     // tiles of 16 columns a warp holds
template <int RT> constexpr int few_part() { return RT * 16 * (few_strip<RT>() * 16 + 8); }   // floats of a warp's sums, padded rows
template <int DEC, int RT> constexpr int few_smem() {
    return table_bytes(DEC) + few_warps<RT>() / 2 * few_part<RT>() * 4 + (kMaxExperts + 4) * 4;
}

template <int K, int DEC, int RT>
__global__ void __launch_bounds__(few_warps<RT>() * 32, DEC == DEC_F16 ? 1 : 2) few_trellis_kernel(const FewTrellis p) {
    constexpr int NT = few_strip<RT>(), COLS = NT * 16, LD = COLS + 8, WARPS = few_warps<RT>();
    extern __shared__ __align__(16) uint8_t smem[];
    float* sums = reinterpret_cast<float*>(smem + table_bytes(DEC));
    int* cum = reinterpret_cast<int*>(sums + WARPS / 2 * few_part<RT>());
    static_assert(WARPS / 2 * few_part<RT>() >= 2 * kMaxExperts, "the scan borrows the sums");
    int* first = reinterpret_cast<int*>(sums);
    let_next_start();
    load_table<DEC>(p.table, smem);
    scan_groups(p.offsets, p.experts, p.rows, RT * 16, first, first + kMaxExperts, cum);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, q = lane & 3;
    const int kt = p.k / 16, nt = p.n / 16, strips = p.n / COLS;
    const int64_t work = (int64_t)cum[p.experts] * strips * kt, per = few_share(work, gridDim.x, kt, p.parts);
    const int64_t stop = min((int64_t)(blockIdx.x + 1) * per, work);
    for (int64_t at = blockIdx.x * per; at < stop;) {
        const int64_t item = at / kt, first_cta = item * kt / per;
        const int strip = (int)(item % strips), t = (int)(item / strips), part = (int)(blockIdx.x - first_cta);
        const int e = expert_of(cum, p.experts, t), r0 = (t - cum[e]) * RT * 16;
        int lo, n_e;
        group_of(p.offsets, e, p.rows, lo, n_e);
        const int row0 = lo + r0, count = min(n_e - r0, RT * 16);
        const int ka = (int)(at - item * kt), kb = (int)min((int64_t)kt, stop - item * kt);
        at += kb - ka;
        const uint32_t* base = p.trellis + ((int64_t)e * kt * nt + strip * NT) * 8 * K;
        float acc[RT][NT][2][4] = {};
        TileWords<K> ahead[2][NT];
        auto fetch = [&](int kk, TileWords<K> (&w)[NT]) {
            if (kk >= kb) return;
#pragma unroll
            for (int j = 0; j < NT; ++j) w[j].load(base + ((int64_t)kk * nt + j) * 8 * K, lane);
        };
        fetch(ka + warp, ahead[0]);
        fetch(ka + warp + WARPS, ahead[1]);
        wait_for_last();                         // x' is there; plain loads of it, which stay behind this
        const uint16_t* xp = p.xr + (int64_t)(row0 + (lane >> 2)) * p.k + 2 * q;
        auto step = [&](int kk, TileWords<K> (&w)[NT]) {
            uint32_t a[RT][4];
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                const uint16_t* x = xp + (int64_t)r * 16 * p.k + kk * 16;
                const bool top = r * 16 + (lane >> 2) < count, low = r * 16 + 8 + (lane >> 2) < count;
                a[r][0] = top ? *reinterpret_cast<const uint32_t*>(x) : 0u;
                a[r][1] = low ? *reinterpret_cast<const uint32_t*>(x + 8 * (int64_t)p.k) : 0u;
                a[r][2] = top ? *reinterpret_cast<const uint32_t*>(x + 8) : 0u;
                a[r][3] = low ? *reinterpret_cast<const uint32_t*>(x + 8 * (int64_t)p.k + 8) : 0u;
            }
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                uint32_t f[4];
                decode_tile<K, DEC>(w[j], lane, smem, f);
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    mma16816(acc[r][j][0], a[r], f[0], f[1]);
                    mma16816(acc[r][j][1], a[r], f[2], f[3]);
                }
            }
            fetch(kk + 2 * WARPS, w);
        };
        for (int kk = ka + warp; kk < kb; kk += 2 * WARPS) {
            step(kk, ahead[0]);
            if (kk + WARPS < kb) step(kk + WARPS, ahead[1]);
        }
        // The upper half of the warps hand over, the lower half add theirs, and the block adds up the rest.
        float* mine = sums + (warp % (WARPS / 2)) * few_part<RT>();
        auto each = [&](auto f) {
#pragma unroll
            for (int r = 0; r < RT; ++r)
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int v = 0; v < 2; ++v)
                            f(reinterpret_cast<float2*>(mine + (r * 16 + v * 8 + (lane >> 2)) * LD + j * 16 + h * 8 + 2 * q),
                              acc[r][j][h][2 * v], acc[r][j][h][2 * v + 1]);
        };
        __syncthreads();                         // the last item's sums are read
        if (warp >= WARPS / 2) each([](float2* s, float x, float y) { *s = make_float2(x, y); });
        __syncthreads();
        if (warp < WARPS / 2) each([](float2* s, float x, float y) { const float2 o = *s; *s = make_float2(x + o.x, y + o.y); });
        __syncthreads();
        for (int i = threadIdx.x; i < count * COLS; i += WARPS * 32) {
            const int r = i / COLS, c = i % COLS;
            float v = 0.f;
#pragma unroll
            for (int w = 0; w < WARPS / 2; ++w) v += sums[w * few_part<RT>() + r * LD + c];
            p.partial[((int64_t)part * p.rows + row0 + r) * p.n + strip * COLS + c] = v;
        }
    }
    wait_for_last();
}

template <int K, int DEC, int RT>
int launch_few(const FewTrellis& p, cudaStream_t s) {
    constexpr int smem = few_smem<DEC, RT>();
    auto kernel = few_trellis_kernel<K, DEC, RT>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) { set_error("cudaFuncSetAttribute: %s", cudaGetErrorString(e)); return KQ_ERR_CUDA; }
    int sms;
    if (int rc = sm_count(&sms)) return rc;
    return launch_next(kernel, sms * (DEC == DEC_F16 ? 1 : 2), few_warps<RT>() * 32, smem, s, "few_trellis_kernel", p);
}

template <int K>
int few_trellis(const FewTrellis& p, int dec, bool wide, cudaStream_t s) {
    if (dec == DEC_MCG) return wide ? launch_few<K, DEC_MCG, 4>(p, s) : launch_few<K, DEC_MCG, 1>(p, s);
    if (dec == DEC_E4M3) return wide ? launch_few<K, DEC_E4M3, 4>(p, s) : launch_few<K, DEC_E4M3, 1>(p, s);
    return wide ? launch_few<K, DEC_F16, 4>(p, s) : launch_few<K, DEC_F16, 1>(p, s);
}

}  // namespace
}  // namespace kq
