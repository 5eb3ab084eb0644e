// Calibration Hessians of all experts at once, fp32:
//
//     H_e (+)= sum_t w_t x_i(t) x_i(t)^T,   den_e = sum_t w_t
//
// over the rows t of expert e (kquant/capture.py:713-730 for one matrix; the
// reference calls it expert by expert).  x [tokens x d] is bf16, fp16 or
// fp32, i an optional index of its rows.
//
// The products run on the 16-bit tensor pipe with exact operands: a value is
// split into 16-bit terms that add up to it, and the products of terms below
// 2^-24 of the whole are left out.
//
//     x 16-bit, no weights:  x x^T                            1 product
//     x bf16, weights:       x * (w x in 3 bf16 terms)        3 products
//     x fp16, weights:       (2 bf16 terms) * (3 terms)       5 products
//     x fp32:                (3 terms) * (3 terms)            6 products
//
// Six bf16 products cost what three TF32 products do and carry 24 bits instead
// of 22.  The operand kernel gathers the rows, applies the weights, splits, and
// pads every expert to whole 32-row stages with zeros; it writes rows as they
// are stored, since an MN-major tcgen05 operand needs no transpose.
//
// One persistent CTA per SM walks the 128 x 256 output tiles on or above the
// diagonal.  A stage holds 16 or 32 rows of every term, so each is fetched once
// for all products.  The tensor-core accumulator truncates: it holds only a few
// stages (up to 128 rows), which the drain warps add into fp32 registers with
// rounding.  Blocks above the diagonal are written twice, so H is exactly
// symmetric.  With few rows writing H is what it costs (see `whole` below).
#include "kq_expert.cuh"

namespace kq {
namespace {

constexpr int BM = 128, BN = 256;
constexpr int SLOT = 32;                        // experts are padded to whole slots of rows
constexpr int drain_warps(bool whole) { return whole ? 16 : 8; }
constexpr int threads(bool whole) { return 64 + 32 * drain_warps(whole); }
constexpr int GROUP_BYTES = (kMaxExperts + 4) * 4;
constexpr int PIECE_BYTES = 8192;               // a drain warp's 32 x 32 block of H and its mirror image, or 32 x 64 block

constexpr int products(int na, int nb) { return na == 1 ? nb : na == 2 ? 5 : 6; }
// Rows of a stage: one product needs 32 for its loads to be worth a barrier; with more terms 16 keep four stages.
constexpr int stage_rows(int na, int nb) { return products(na, nb) == 1 ? 32 : 16; }
// 64 columns of a stage: rows of 128 bytes.
constexpr int chunk_bytes(int na, int nb) { return stage_rows(na, nb) * 128; }
constexpr int stage_bytes(int na, int nb) { return (na * (BM / 64) + nb * (BN / 64)) * chunk_bytes(na, nb); }
constexpr int stages_for(int na, int nb, bool whole) {
    const int fit = (227 * 1024 - 1024 - GROUP_BYTES - drain_warps(whole) * PIECE_BYTES - 512) / stage_bytes(na, nb);
    return fit > 8 ? 8 : fit;
}
// Stages per drain: 128 rows of one product, 64 of three, 32 of more.
constexpr int seg_stages(int na, int nb) {
    return (products(na, nb) == 1 ? 128 : products(na, nb) == 3 ? 64 : 32) / stage_rows(na, nb);
}

struct Maps { CUtensorMap a[3], b[3]; };

struct Params {
    const int64_t* offsets;
    float* H;
    int* err;
    int64_t h_stride, ldh;
    int rows, experts, d, tiles, n_tiles;   // tiles per expert, and in a row of them
    uint32_t idesc;
    bool add, vec;
};

// Tile l of an expert.  On or above the diagonal: column block ni holds the row blocks 0 .. 2 ni + 1.  Whole: row by row.
template <bool WHOLE>
__device__ __forceinline__ void tile_at(int l, int n_tiles, int& m0, int& n0) {
    if constexpr (WHOLE) {
        m0 = l / n_tiles * BM;
        n0 = l % n_tiles * BN;
        return;
    }
    int ni = (int)((sqrtf(4.f * l + 1.f) - 1.f) * 0.5f);
    while (ni * (ni + 1) > l) --ni;
    while ((ni + 1) * (ni + 2) <= l) ++ni;
    m0 = (l - ni * (ni + 1)) * BM;
    n0 = ni * BN;
}

// The products of a stage, small terms first: (a term, b term) in order.
template <int NA, int NB>
__device__ __forceinline__ void product_terms(int i, int& a, int& b) {
    if constexpr (NA == 1) { a = 0; b = NB - 1 - i; }
    else if constexpr (NA == 2) { a = (0x05 >> i) & 1; b = (0x0049 >> (i * 2)) & 3; }
    else { a = (0x0052 >> (i * 2)) & 3; b = (0x0118 >> (i * 2)) & 3; }
}

// WHOLE: every tile of H, without mirror images.
template <int NA, int NB, bool WHOLE>
__global__ void __launch_bounds__(threads(WHOLE), 1)
hessian_kernel(const __grid_constant__ Maps maps, const __grid_constant__ CUtensorMap map_h, const Params p) {
    constexpr int STAGES = stages_for(NA, NB, WHOLE), STAGE = stage_bytes(NA, NB), SEG = seg_stages(NA, NB);
    constexpr int BK = stage_rows(NA, NB), PER_SLOT = SLOT / BK, CHUNK = chunk_bytes(NA, NB);
    constexpr int A_BYTES = BM / 64 * CHUNK, B_BYTES = BN / 64 * CHUNK;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t full_bar[STAGES], empty_bar[STAGES], seg_full[WHOLE ? 4 : 2], seg_empty[2];
    __shared__ uint32_t tmem_slot;
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t* out_smem = smem + STAGES * STAGE;
    int* cum = reinterpret_cast<int*>(out_smem + drain_warps(WHOLE) * PIECE_BYTES);
    int* lo = reinterpret_cast<int*>(smem);     // needed by the scan alone, before the first stage is loaded
    int* cnt = lo + kMaxExperts;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        tma_prefetch(&maps.a[0]);
        tma_prefetch(&maps.b[0]);
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&full_bar[s], 1);
            mbar_init(&empty_bar[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&seg_full[b], 1);
            if (WHOLE) mbar_init(&seg_full[2 + b], 1);
            mbar_init(&seg_empty[b], 8);
        }
        mbar_init_fence();
    }
    constexpr int DRAINS = drain_warps(WHOLE);
    if (warp == DRAINS) tmem_alloc(&tmem_slot, 2 * BN);
    scan_groups(p.offsets, p.experts, p.rows, SLOT, lo, cnt, cum);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    const int64_t all = (int64_t)p.tiles * p.experts;

    if (warp == DRAINS) {
        if (lane == 0) {
            uint32_t it = 0;
            bool ok = true;
            for (int64_t i = blockIdx.x; i < all && ok; i += gridDim.x) {
                const int e = (int)(i / p.tiles);
                int m0, n0;
                tile_at<WHOLE>((int)(i - (int64_t)e * p.tiles), p.n_tiles, m0, n0);
                for (int ks = cum[e] * PER_SLOT; ks < cum[e + 1] * PER_SLOT; ++ks, ++it) {
                    const int s = it % STAGES;
                    if (!(ok = mbar_wait(&empty_bar[s], ((it / STAGES) & 1) ^ 1))) break;
                    mbar_expect_tx(&full_bar[s], STAGE);
                    uint8_t* dst = smem + s * STAGE;
#pragma unroll
                    for (int t = 0; t < NA; ++t) tma_load_3d(dst + t * A_BYTES, &maps.a[t], 0, ks * BK, m0 / 64, &full_bar[s]);
#pragma unroll
                    for (int t = 0; t < NB; ++t)
                        tma_load_3d(dst + NA * A_BYTES + t * B_BYTES, &maps.b[t], 0, ks * BK, n0 / 64, &full_bar[s]);
                }
            }
            if (!ok) report_wait_error(p.err);
        }
    } else if (warp == DRAINS + 1) {
        if (lane == 0) {
            uint32_t it = 0, seg = 0, turn = 0;
            bool ok = true;
            for (int64_t i = blockIdx.x; i < all && ok; i += gridDim.x) {
                const int e = (int)(i / p.tiles), ks_end = cum[e + 1] * PER_SLOT;
                const int owner = WHOLE ? turn & 1 : 0;      // the group of drain warps that takes this tile
                turn += ks_end > cum[e] * PER_SLOT;
                for (int ks0 = cum[e] * PER_SLOT; ks0 < ks_end && ok; ks0 += SEG, ++seg) {
                    const int b = seg & 1;
                    if (!(ok = mbar_wait(&seg_empty[b], ((seg >> 1) & 1) ^ 1))) break;
                    tc_fence_after();
                    const int stop = min(ks_end, ks0 + SEG);
                    for (int ks = ks0; ks < stop; ++ks, ++it) {
                        const int s = it % STAGES;
                        if (!(ok = mbar_wait(&full_bar[s], (it / STAGES) & 1))) break;
                        tc_fence_after();
                        const uint32_t base = smem_addr(smem + s * STAGE);
#pragma unroll
                        for (int i2 = 0; i2 < products(NA, NB); ++i2) {
                            int ta, tb;
                            product_terms<NA, NB>(i2, ta, tb);
                            const uint64_t ad = smem_desc(base + ta * A_BYTES, CHUNK);
                            const uint64_t bd = smem_desc(base + NA * A_BYTES + tb * B_BYTES, CHUNK);
#pragma unroll
                            for (int kk = 0; kk < BK / 16; ++kk)
                                mma_f16(tmem + b * BN, ad + 128 * kk, bd + 128 * kk, p.idesc,
                                        (ks != ks0 || i2 != 0 || kk != 0) ? 1u : 0u);
                        }
                        mma_commit(&empty_bar[s]);
                    }
                    if (ok) mma_commit(&seg_full[2 * owner + b]);
                }
            }
            if (!ok) report_wait_error(p.err);
        }
    } else if constexpr (WHOLE) {
        // Two groups of eight warps take tiles in turn (four quarters of the rows, two halves of the columns): one stores
        // while the other fills its buffers.  A tile's further segments (an expert of more rows) are added to what its
        // first one wrote, by the same thread.  Each group has barriers of its own: it sees none of the other's segments, and
        // a barrier that went through a phase unseen would be taken for the one before it.
        const int q = warp & 3, h = (warp >> 2) & 1, group = warp >> 3;
        uint8_t* stage = out_smem + warp * PIECE_BYTES;          // two 32 x 32 pieces under way
        uint32_t seg = 0, turn = 0, piece_no = 0, seen = 0;                // seen: the phase of this group's two barriers
        bool ok = true;
        for (int64_t it = blockIdx.x; it < all && ok; it += gridDim.x) {
            const int e = (int)(it / p.tiles), ks_begin = cum[e] * PER_SLOT, ks_end = cum[e + 1] * PER_SLOT;
            int m0, n0;
            tile_at<WHOLE>((int)(it - (int64_t)e * p.tiles), p.n_tiles, m0, n0);
            const int i0 = m0 + q * 32, j0 = n0 + h * (BN / 2);
            // Columns j0 + c .. + 31 of this warp's 32 rows.
            auto put = [&](const uint32_t (&v)[32], int c, bool add) {
                uint8_t* piece = stage + (piece_no++ & 1) * (PIECE_BYTES / 2);
                auto unit = [&](int row, int u) { return reinterpret_cast<uint4*>(piece + row * 128 + ((u ^ (row & 7)) << 4)); };
                if (lane == 0) bulk_wait_read<1>();
                __syncwarp();
#pragma unroll
                for (int u = 0; u < 8; ++u) *unit(lane, u) = make_uint4(v[4 * u], v[4 * u + 1], v[4 * u + 2], v[4 * u + 3]);
                if (p.vec) {
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) {
                        if (i0 < p.d && j0 + c < p.d) {
                            if (add) tma_add_3d(&map_h, piece, j0 + c, i0, e);
                            else tma_store_3d(&map_h, piece, j0 + c, i0, e);
                        }
                        bulk_commit();
                    }
                    __syncwarp();                                  // the next tensor-memory load is the whole warp's
                } else {
                    __syncwarp();
                    const int j = j0 + c + lane;
                    float* dst = p.H + e * p.h_stride + (int64_t)i0 * p.ldh + j;
                    const int n = j < p.d ? p.d - i0 : 0;
#pragma unroll 16
                    for (int k = 0; k < 32; ++k, dst += p.ldh) {
                        const float x = reinterpret_cast<const float*>(unit(k, lane >> 2))[lane & 3];
                        if (k >= n) continue;
                        if (add) atomicAdd(dst, x);
                        else *dst = x;
                    }
                    __syncwarp();
                }
            };
            if (ks_begin == ks_end) {
                if (p.add || ((it / gridDim.x) & 1) != group) continue;
                const uint32_t zero[32] = {};
                for (int c = 0; c < BN / 2; c += 32) put(zero, c, false);
                continue;
            }
            const int owner = turn++ & 1;
            for (int ks0 = ks_begin; ks0 < ks_end; ks0 += SEG, ++seg) {
                if (owner != group) continue;
                ok = __all_sync(0xFFFFFFFFu, mbar_wait(&seg_full[2 * group + (seg & 1)], (seen >> (seg & 1)) & 1));
                if (!ok) break;
                seen ^= 1u << (seg & 1);
                tc_fence_after();
                if (ks0 > ks_begin && lane == 0) bulk_wait_all();      // what this adds to is there
                __syncwarp();
                const uint32_t base = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)((seg & 1) * BN + h * (BN / 2));
#pragma unroll 1
                for (int c = 0; c < BN / 2; c += 32) {
                    uint32_t v[32];
                    tmem_ld32(base + c, v);
                    tmem_wait_ld();
                    if (c + 32 == BN / 2) {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&seg_empty[seg & 1]);
                    }
                    put(v, c, p.add || ks0 > ks_begin);
                }
            }
        }
        if (lane == 0) bulk_wait_all();
        if (!ok && lane == 0) report_wait_error(p.err);
    } else {
        const int q = warp & 3, h = warp >> 2;
        uint32_t seg = 0;
        bool ok = true;
        uint8_t *piece = out_smem + warp * PIECE_BYTES, *mirror = piece + PIECE_BYTES / 2;
        for (int64_t it = blockIdx.x; it < all && ok; it += gridDim.x) {
            const int e = (int)(it / p.tiles), ks_begin = cum[e] * PER_SLOT, ks_end = cum[e + 1] * PER_SLOT;
            int m0, n0;
            tile_at<WHOLE>((int)(it - (int64_t)e * p.tiles), p.n_tiles, m0, n0);
            const int i0 = m0 + q * 32, j0 = n0 + h * (BN / 2);
            float* H = p.H + e * p.h_stride;
            // Columns j0 + c .. + 31 of this warp's 32 rows: a block above the diagonal and its mirror image, or the block
            // on it made symmetric.  Whole 128-byte lines either way: 32-byte pieces of 32 rows at a time ran at a third.
            auto put = [&](const float* v, int c) {
                const int j = j0 + c;
                if (i0 >= p.d || j >= p.d || j < i0) return;
                const bool diagonal = i0 == j;
                // Element (row, col) of a 32 x 32 block, 16-byte units swizzled by the row as the TMA map has them.
                auto at = [](uint8_t* block, int row, int col) {
                    return reinterpret_cast<float*>(block + row * 128 + (((col >> 2) ^ (row & 7)) << 4) + (col & 3) * 4);
                };
                if (!diagonal) {
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        *reinterpret_cast<float4*>(at(piece, lane, 4 * k)) = make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
#pragma unroll
                    for (int k = 0; k < 32; ++k) *at(mirror, k, lane) = v[k];
                } else {
#pragma unroll
                    for (int k = 0; k < 32; ++k) {
                        if (k >= lane) {
                            *at(piece, lane, k) = v[k];
                            *at(piece, k, lane) = v[k];
                        }
                    }
                }
                __syncwarp();
                if (p.vec && max(i0, j) + 32 <= p.d) {
                    // 16 bytes a lane, four rows an access.
                    for (int side = 0; side < (diagonal ? 1 : 2); ++side) {
                        const int row0 = (side ? j : i0) + (lane >> 3), col = (side ? i0 : j) + (lane & 7) * 4;
                        uint8_t* block = side ? mirror : piece;
                        float* dst = H + (int64_t)row0 * p.ldh + col;
#pragma unroll
                        for (int k = 0; k < 32; k += 4, dst += 4 * p.ldh) {
                            const float4 x = *reinterpret_cast<const float4*>(at(block, (lane >> 3) + k, (lane & 7) * 4));
                            if (p.add) atomicAdd(reinterpret_cast<float4*>(dst), x);
                            else __stcs(reinterpret_cast<float4*>(dst), x);
                        }
                    }
                    __syncwarp();
                } else {
                    for (int side = 0; side < (diagonal ? 1 : 2); ++side) {
                        const int row0 = side ? j : i0, col = (side ? i0 : j) + lane;
                        uint8_t* block = side ? mirror : piece;
                        float* dst = H + (int64_t)row0 * p.ldh + col;
                        const int n = col < p.d ? p.d - row0 : 0;
#pragma unroll 16
                        for (int k = 0; k < 32; ++k, dst += p.ldh) {
                            const float x = *at(block, k, lane);
                            if (k >= n) continue;
                            if (p.add) atomicAdd(dst, x);
                            else *dst = x;
                        }
                    }
                    __syncwarp();
                }
            };
            auto wait_seg = [&]() {
                ok = __all_sync(0xFFFFFFFFu, mbar_wait(&seg_full[seg & 1], (seg >> 1) & 1));
                tc_fence_after();
                return tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)((seg & 1) * BN + h * (BN / 2));
            };
            auto free_seg = [&]() {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&seg_empty[seg & 1]);
                ++seg;
            };
            if (ks_end > ks_begin && ks_end - ks_begin <= SEG) {
                // All rows in one segment: from tensor memory to H.
                const uint32_t base = wait_seg();
                if (!ok) break;
                constexpr int STEP = 32;
#pragma unroll 1
                for (int c = 0; c < BN / 2; c += STEP) {
                    uint32_t u[STEP / 32][32];
                    float v[STEP];
#pragma unroll
                    for (int k = 0; k < STEP; k += 32) tmem_ld32(base + c + k, u[k / 32]);
                    tmem_wait_ld();
                    if (c + STEP == BN / 2) free_seg();
#pragma unroll
                    for (int k = 0; k < STEP; ++k) v[k] = __uint_as_float(u[k >> 5][k & 31]);
                    put(v, c);
                }
                continue;
            }
            float r[BN / 2];
#pragma unroll
            for (int k = 0; k < BN / 2; ++k) r[k] = 0.f;
            for (int ks0 = ks_begin; ks0 < ks_end; ks0 += SEG) {
                const uint32_t base = wait_seg();
                if (!ok) break;
#pragma unroll
                for (int c0 = 0; c0 < BN / 2; c0 += 16) {
                    uint32_t v[16];
                    tmem_ld16(base + (uint32_t)c0, v);
                    tmem_wait_ld();
#pragma unroll
                    for (int k = 0; k < 16; ++k) r[c0 + k] += __uint_as_float(v[k]);
                }
                free_seg();
            }
            if (!ok) break;
            if (p.add && ks_begin == ks_end) continue;
#pragma unroll
            for (int c = 0; c < BN / 2; c += 32) put(r + c, c);
            __syncwarp();
        }
        if (!ok && lane == 0) report_wait_error(p.err);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == DRAINS) tmem_free(tmem, 2 * BN);
}

// Operand rows.  Block (t, c): slots 32 t .. of the padded rows, `block_cols`
// columns from block_cols c; the blocks behind the last row tile sum the weights of one
// expert each, in an order that depends on nothing.
struct OperandParams {
    const void* x;
    const int64_t* index;
    const float* w;
    const int64_t* offsets;
    uint16_t* terms;           // a terms, then b terms, each [slots][ld]
    double* den;
    int64_t ldx, tokens, term_stride;
    int rows, experts, d, ld, row_tiles, block_shift;   // 8 << block_shift columns a block
    bool vec;
};

__device__ __forceinline__ void split_bf16(float v, int n, uint16_t (&t)[3]) {
    float rest = v;
    const bool finite = fabsf(v) <= 3.3895313892515355e38f;
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        if (i < n) {
            const __nv_bfloat16 b = __float2bfloat16_rn(rest);
            t[i] = __bfloat16_as_ushort(b);
            rest = finite ? rest - __bfloat162float(b) : 0.f;
        }
    }
}

// NA = NB = 0: the 16-bit values themselves.
template <typename T, int NA, int NB>
__global__ void __launch_bounds__(256) operand_kernel(const OperandParams p) {
    __shared__ int lo[kMaxExperts], cnt[kMaxExperts], cum[kMaxExperts + 1];
    __shared__ double part[256];
    if ((int)blockIdx.x >= p.row_tiles) {
        if (blockIdx.y) return;
        const int e = blockIdx.x - p.row_tiles;
        int first, n;
        group_of(p.offsets, e, p.rows, first, n);
        double s = 0.0;
        for (int r = threadIdx.x; r < n; r += 256) {
            const int64_t src = p.index ? p.index[first + r] : first + r;
            if (src >= 0 && src < p.tokens) s += p.w ? (double)p.w[first + r] : 1.0;
        }
        part[threadIdx.x] = s;
        for (int d = 128; d; d >>= 1) {
            __syncthreads();
            if ((int)threadIdx.x < d) part[threadIdx.x] += part[threadIdx.x + d];
        }
        if (threadIdx.x == 0) p.den[e] = part[0];
        return;
    }
    scan_groups(p.offsets, p.experts, p.rows, SLOT, lo, cnt, cum);
    const int t = blockIdx.x;
    if (t >= cum[p.experts]) return;
    const int e = expert_of(cum, p.experts, t), first = (t - cum[e]) * SLOT;
    const int per_row = 1 << p.block_shift;
    for (int i = threadIdx.x; i < SLOT * per_row; i += 256) {    // 8 columns of one row at a time
        const int r = i >> p.block_shift, c = (blockIdx.y * per_row + (i & (per_row - 1))) * 8;
        if (c >= p.ld) continue;
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = 0.f;
        float w = 0.f;
        if (first + r < cnt[e]) {
            const int row = lo[e] + first + r;
            const int64_t src = p.index ? p.index[row] : row;
            if (src >= 0 && src < p.tokens) {
                w = p.w ? p.w[row] : 1.f;
                const T* xr = static_cast<const T*>(p.x) + src * p.ldx + c;
                const int nv = p.d - c;
                if constexpr (sizeof(T) == 4) {
                    if (p.vec && nv >= 8) {
                        *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(xr);
                        *reinterpret_cast<float4*>(v + 4) = *reinterpret_cast<const float4*>(xr + 4);
                    } else {
#pragma unroll
                        for (int k = 0; k < 8; ++k) if (k < nv) v[k] = xr[k];
                    }
                } else {
                    load8(xr, p.vec && nv >= 8, nv, v);
                }
            }
        }
        uint16_t* dst = p.terms + ((int64_t)t * SLOT + r) * p.ld + c;
        if constexpr (NA == 0) {
            T o[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) o[k] = from_f<T>(v[k]);
            *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(o);
        } else {
            uint16_t a[8][3], b[8][3];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                split_bf16(v[k], NA, a[k]);
                split_bf16(v[k] * w, NB, b[k]);
            }
#pragma unroll
            for (int q = 0; q < NA + NB; ++q) {
                uint16_t o[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) o[k] = q < NA ? a[k][q < NA ? q : 0] : b[k][q < NA ? 0 : q - NA];
                *reinterpret_cast<uint4*>(dst + q * p.term_stride) = *reinterpret_cast<const uint4*>(o);
            }
        }
    }
}

int64_t pad_width(int64_t v) { return (v + 63) & ~(int64_t)63; }

int64_t slots(int64_t rows, int64_t experts) { return ((rows + SLOT - 1) / SLOT + (experts < rows ? experts : rows)) * SLOT; }

void terms_of(int dtype, bool weighted, int& na, int& nb) {
    if (dtype == KQ_FP32) { na = 3; nb = 3; }
    else if (!weighted) { na = 0; nb = 0; }
    else if (dtype == KQ_BF16) { na = 1; nb = 3; }
    else { na = 2; nb = 3; }
}

// One set of terms for both sides where they are the 16-bit values themselves, else one for each (fp32 rows without weights too,
// whose two sets are alike).
int term_count(int dtype, bool weighted) {
    int na, nb;
    terms_of(dtype, weighted, na, nb);
    return na == 0 ? 1 : na + nb;
}

template <int NA, int NB, bool WHOLE>
int launch_hessian(const Maps& m, const CUtensorMap& h, const Params& p, int grid, cudaStream_t s) {
    constexpr int smem = stages_for(NA, NB, WHOLE) * stage_bytes(NA, NB) + drain_warps(WHOLE) * PIECE_BYTES + GROUP_BYTES + 1024;
    cudaError_t e = cudaFuncSetAttribute(hessian_kernel<NA, NB, WHOLE>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) { set_error("cudaFuncSetAttribute: %s", cudaGetErrorString(e)); return KQ_ERR_CUDA; }
    hessian_kernel<NA, NB, WHOLE><<<grid, threads(WHOLE), smem, s>>>(m, h, p);
    return check_launch("hessian_kernel");
}

bool bad_sizes(int64_t rows, int64_t tokens, int64_t d, int64_t experts, int dtype) {
    return rows < 0 || tokens < 0 || d <= 0 || experts <= 0 || experts > kMaxExperts || rows > 0x3FFFFFFF || d > (1 << 20) ||
           (dtype != KQ_BF16 && dtype != KQ_FP16 && dtype != KQ_FP32);
}

}  // namespace
}  // namespace kq

extern "C" size_t kq_expert_hessian_workspace_bytes(int64_t rows, int64_t dim, int64_t experts, int dtype, int weighted) {
    using namespace kq;
    if (bad_sizes(rows, 0, dim, experts, dtype) || rows == 0) return 0;
    return (size_t)term_count(dtype, weighted != 0) * (size_t)slots(rows, experts) * (size_t)pad_width(dim) * 2;
}

extern "C" int kq_accumulate_expert_hessians(const void* x, int64_t tokens, int64_t dim, int64_t ldx, int dtype,
                                             const int64_t* index, const float* w, const int64_t* offsets, int64_t rows,
                                             int64_t experts, float* H, int64_t h_stride, int64_t ldh, int add, double* den,
                                             void* workspace, size_t workspace_bytes, void* stream) {
    using namespace kq;
    const char* what = "kq_accumulate_expert_hessians";
    if (bad_sizes(rows, tokens, dim, experts, dtype) || (tokens > 1 && ldx < dim) || (dim > 1 && ldh < dim) ||
        (experts > 1 && h_stride < (dim - 1) * ldh + dim) || (!index && rows > tokens)) {
        set_error("%s: bad arguments (rows=%lld tokens=%lld dim=%lld experts=%lld ldx=%lld ldh=%lld dtype=%d)", what,
                  (long long)rows, (long long)tokens, (long long)dim, (long long)experts, (long long)ldx, (long long)ldh, dtype);
        return KQ_ERR_ARG;
    }
    if (experts > 1 && !offsets) { set_error("%s: several experts need offsets", what); return KQ_ERR_ARG; }
    if (!H || !den || (rows > 0 && tokens > 0 && !x)) { set_error("%s: null pointer", what); return KQ_ERR_ARG; }
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool weighted = w != nullptr;
    const size_t need = kq_expert_hessian_workspace_bytes(rows, dim, experts, dtype, weighted);
    if (need && (workspace_bytes < need || !workspace)) { set_error("%s: workspace too small", what); return KQ_ERR_WORKSPACE; }
    if ((uintptr_t)workspace & 127) { set_error("%s: workspace must be 128-byte aligned", what); return KQ_ERR_ALIGN; }
    Params q{};
    if (int rc = wait_error_word(&q.err, what)) return rc;
    const int ld = (int)pad_width(dim);
    const int64_t n_slots = slots(rows, experts);
    int na, nb;
    terms_of(dtype, weighted, na, nb);

    OperandParams o{};
    o.x = x;
    o.index = index;
    o.w = w;
    o.offsets = offsets;
    o.terms = static_cast<uint16_t*>(workspace);
    o.den = den;
    o.ldx = ldx;
    o.tokens = tokens;
    o.term_stride = n_slots * ld;
    o.rows = (int)rows;
    o.experts = (int)experts;
    o.d = (int)dim;
    o.ld = ld;
    o.row_tiles = (int)(n_slots / SLOT);
    o.vec = ((uintptr_t)x & 15) == 0 && ldx % 8 == 0;
    // Few blocks: shorter ones, for their latency.
    o.block_shift = (int64_t)o.row_tiles * ((ld + 1023) / 1024) < 296 ? 4 : 7;
    const int block_cols = 8 << o.block_shift;
    const dim3 grid((unsigned)(o.row_tiles + experts), (unsigned)((ld + block_cols - 1) / block_cols));
    if (dtype == KQ_FP32) operand_kernel<float, 3, 3><<<grid, 256, 0, s>>>(o);
    else if (dtype == KQ_BF16 && weighted) operand_kernel<__nv_bfloat16, 1, 3><<<grid, 256, 0, s>>>(o);
    else if (dtype == KQ_BF16) operand_kernel<__nv_bfloat16, 0, 0><<<grid, 256, 0, s>>>(o);
    else if (weighted) operand_kernel<__half, 2, 3><<<grid, 256, 0, s>>>(o);
    else operand_kernel<__half, 0, 0><<<grid, 256, 0, s>>>(o);
    if (int rc = check_launch("operand_kernel")) return rc;

    Maps maps{};
    const bool fp16 = dtype == KQ_FP16 && !weighted;
    // A term as [64-column slab][row][64]: one TMA instruction brings all slabs of a side (its issue bounded the loads).
    const int64_t dims[3] = {64, n_slots > 0 ? n_slots : 1, ld / 64}, strides[2] = {(int64_t)ld * 2, 128};
    const int box_rows = na ? stage_rows(na, nb) : stage_rows(1, 1);
    const int box_a[3] = {64, box_rows, BM / 64}, box_b[3] = {64, box_rows, BN / 64};
    const CUtensorMapDataType type = fp16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    for (int t = 0; t < (na ? na : 1) && rows > 0; ++t)
        if (int rc = encode_tiles(&maps.a[t], type, 3, o.terms + t * o.term_stride, dims, strides, box_a, what)) return rc;
    for (int t = 0; t < (na ? nb : 1) && rows > 0; ++t)
        if (int rc = encode_tiles(&maps.b[t], type, 3, o.terms + (na + t) * o.term_stride, dims, strides, box_b, what)) return rc;
    q.offsets = offsets;
    q.H = H;
    q.h_stride = h_stride;
    q.ldh = ldh;
    q.rows = (int)rows;
    q.experts = (int)experts;
    q.d = (int)dim;
    const int64_t nt = (dim + BN - 1) / BN;
    // One product of few rows is bound by writing H: all of it as TMA tiles takes 290 us for 512 rows of 8 experts and d
    // 7168 (222 us at the write rate of a fill), blocks above the diagonal and their mirror images 330 us.  From about 256
    // rows an expert the products of half the tiles weigh more (4096 rows: 570 us in halves, 610 us for 2048 rows whole).
    // x x^T comes out symmetric by itself, its sums being the same products in the same order on both sides.
    const bool whole = na == 0 && rows <= 128 * experts;
    q.n_tiles = (int)nt;
    q.tiles = (int)(whole ? (dim + BM - 1) / BM * nt : nt * (nt + 1));
    q.idesc = idesc_f16(!fp16, true, true, BM, BN);
    q.add = add != 0;
    const bool vec = ((uintptr_t)H & 15) == 0 && ldh % 4 == 0 && h_stride % 4 == 0;
    q.vec = vec && ldh < ((int64_t)1 << 36) && h_stride < ((int64_t)1 << 36);
    CUtensorMap map_h{};
    if (q.vec && whole) {
        const int64_t hd[3] = {dim, dim, experts}, hs[2] = {ldh * 4, (experts > 1 ? h_stride : ldh * dim) * 4};
        const int hb[3] = {32, 32, 1};
        if (int rc = encode_tiles(&map_h, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, H, hd, hs, hb, what)) return rc;
    }
    int sms;
    if (int rc = sm_count(&sms)) return rc;
    const int64_t tiles = (int64_t)q.tiles * experts;
    const int g = (int)(tiles < sms ? tiles : sms);
    if (whole) return launch_hessian<1, 1, true>(maps, map_h, q, g, s);
    if (na == 0) return launch_hessian<1, 1, false>(maps, map_h, q, g, s);
    if (na == 1) return launch_hessian<1, 3, false>(maps, map_h, q, g, s);
    if (na == 2) return launch_hessian<2, 3, false>(maps, map_h, q, g, s);
    return launch_hessian<3, 3, false>(maps, map_h, q, g, s);
}
