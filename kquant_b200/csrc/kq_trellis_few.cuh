// Product of few rows with packed trellis tiles: decoded in registers, used once.
//
// The trellis order of a tile is the operand order of mma.m16n8k16: the eight
// labels that a lane decodes are its two B fragments (columns 0..7 and 8..15
// of the tile), so a decoded tile goes from registers into the products of up
// to 64 rows without touching memory.  Decoding is what bounds this (the
// products of 64 rows take half of its time even on mma.sync), at three bits:
// label lookups in shared memory for the tables, integer arithmetic for MCG.
//
// An item is one row tile (16 or 64 rows of an expert), a strip of columns and
// a range of k; a CTA's eight warps take the k tiles of the range in turn, each
// with its words two steps ahead in registers, and add up in shared memory in
// a fixed order.  Items are dealt to a persistent grid of two CTAs an SM, whose
// ends hide each other.
#pragma once
#include "kq_trellis_decode.cuh"

namespace kq {
namespace {

constexpr int kFewWarps = 8;

__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// RT: row tiles of 16.
template <int RT> constexpr int few_strip() { return RT == 1 ? 4 : 2; }     // tiles of 16 columns a warp holds
template <int RT> constexpr int few_part() { return RT * 16 * (few_strip<RT>() * 16 + 8); }   // floats of a warp's sums, padded rows
template <int DEC, int RT> constexpr int few_smem() {
    return table_bytes(DEC) + kFewWarps / 2 * few_part<RT>() * 4 + (kMaxExperts + 4) * 4;
}

template <int K, int DEC, int RT>
__global__ void __launch_bounds__(kFewWarps * 32, DEC == DEC_F16 ? 1 : 2) few_trellis_kernel(const FewTrellis p) {
    constexpr int NT = few_strip<RT>(), COLS = NT * 16, LD = COLS + 8;
    extern __shared__ __align__(16) uint8_t smem[];
    float* sums = reinterpret_cast<float*>(smem + table_bytes(DEC));
    int* cum = reinterpret_cast<int*>(sums + kFewWarps / 2 * few_part<RT>());
    static_assert(kFewWarps / 2 * few_part<RT>() >= 2 * kMaxExperts, "the scan borrows the sums");
    int* first = reinterpret_cast<int*>(sums);
    load_table<DEC>(p.table, smem);
    scan_groups(p.offsets, p.experts, p.rows, RT * 16, first, first + kMaxExperts, cum);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, q = lane & 3;
    const int kt = p.k / 16, nt = p.n / 16, strips = p.n / COLS;
    const int64_t items = (int64_t)cum[p.experts] * p.splits * strips;
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
        const int strip = (int)(item % strips), rest = (int)(item / strips), split = rest % p.splits, t = rest / p.splits;
        const int e = expert_of(cum, p.experts, t), r0 = (t - cum[e]) * RT * 16;
        int lo, n_e;
        group_of(p.offsets, e, p.rows, lo, n_e);
        const int row0 = lo + r0, count = min(n_e - r0, RT * 16);
        const int ka = (int)((int64_t)kt * split / p.splits), kb = (int)((int64_t)kt * (split + 1) / p.splits);
        const uint32_t* base = p.trellis + ((int64_t)e * kt * nt + strip * NT) * 8 * K;
        float acc[RT][NT][2][4] = {};
        TileWords<K> ahead[2][NT];
        auto fetch = [&](int kk, TileWords<K> (&w)[NT]) {
            if (kk >= kb) return;
#pragma unroll
            for (int j = 0; j < NT; ++j) w[j].load(base + ((int64_t)kk * nt + j) * 8 * K, lane);
        };
        fetch(ka + warp, ahead[0]);
        fetch(ka + warp + kFewWarps, ahead[1]);
        const uint16_t* xp = p.xr + (int64_t)(row0 + (lane >> 2)) * p.k + 2 * q;
        auto step = [&](int kk, TileWords<K> (&w)[NT]) {
            uint32_t a[RT][4];
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                const uint16_t* x = xp + (int64_t)r * 16 * p.k + kk * 16;
                const bool top = r * 16 + (lane >> 2) < count, low = r * 16 + 8 + (lane >> 2) < count;
                a[r][0] = top ? __ldg(reinterpret_cast<const uint32_t*>(x)) : 0u;
                a[r][1] = low ? __ldg(reinterpret_cast<const uint32_t*>(x + 8 * (int64_t)p.k)) : 0u;
                a[r][2] = top ? __ldg(reinterpret_cast<const uint32_t*>(x + 8)) : 0u;
                a[r][3] = low ? __ldg(reinterpret_cast<const uint32_t*>(x + 8 * (int64_t)p.k + 8)) : 0u;
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
            fetch(kk + 2 * kFewWarps, w);
        };
        for (int kk = ka + warp; kk < kb; kk += 2 * kFewWarps) {
            step(kk, ahead[0]);
            if (kk + kFewWarps < kb) step(kk + kFewWarps, ahead[1]);
        }
        // Warps 4..7 hand over, warps 0..3 add theirs, and the block adds up the four.
        float* mine = sums + (warp & 3) * few_part<RT>();
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
        if (warp >= 4) each([](float2* s, float x, float y) { *s = make_float2(x, y); });
        __syncthreads();
        if (warp < 4) each([](float2* s, float x, float y) { const float2 o = *s; *s = make_float2(x + o.x, y + o.y); });
        __syncthreads();
        for (int i = threadIdx.x; i < count * COLS; i += kFewWarps * 32) {
            const int r = i / COLS, c = i % COLS;
            float v = 0.f;
#pragma unroll
            for (int w = 0; w < 4; ++w) v += sums[w * few_part<RT>() + r * LD + c];
            p.partial[((int64_t)split * p.rows + row0 + r) * p.n + strip * COLS + c] = v;
        }
    }
}

template <int K, int DEC, int RT>
int launch_few(const FewTrellis& p, cudaStream_t s) {
    constexpr int smem = few_smem<DEC, RT>();
    auto kernel = few_trellis_kernel<K, DEC, RT>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) { set_error("cudaFuncSetAttribute: %s", cudaGetErrorString(e)); return KQ_ERR_CUDA; }
    int sms;
    if (int rc = sm_count(&sms)) return rc;
    kernel<<<sms * (DEC == DEC_F16 ? 1 : 2), kFewWarps * 32, smem, s>>>(p);
    return check_launch("few_trellis_kernel");
}

template <int K>
int few_trellis(const FewTrellis& p, int dec, bool wide, cudaStream_t s) {
    if (dec == DEC_MCG) return wide ? launch_few<K, DEC_MCG, 4>(p, s) : launch_few<K, DEC_MCG, 1>(p, s);
    if (dec == DEC_E4M3) return wide ? launch_few<K, DEC_E4M3, 4>(p, s) : launch_few<K, DEC_E4M3, 1>(p, s);
    return wide ? launch_few<K, DEC_F16, 4>(p, s) : launch_few<K, DEC_F16, 1>(p, s);
}

}  // namespace
}  // namespace kq
