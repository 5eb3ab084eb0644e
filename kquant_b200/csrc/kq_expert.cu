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
// A pair of CTAs (cta_group::2) shares one output tile, persistent, one CTA
// per SM.  The M axis of the tensor product is the output's contiguous axis:
// 512 features of W in two accumulators of 256, 128 lanes of each per CTA
// (gated: 256 of gate in one and the same 256 of up in the other).  The N axis
// is the rows, 64 to 256 of them: an expert's last tile costs what its rows
// need, where row tiles of 128 or 256 on the M axis would waste 11% or 31% of
// the products of an unevenly routed prompt (8192 rows, 16 experts).  A CTA
// moves 48 KB a stage for 1024 tensor cycles; one CTA with a 128 x 256 tile
// would move the same for 512.  8192 rows without an epilogue, in a run of
// calls under the power limit: 1030 TFLOP/s at k = 1536, 1158 at 7168 (0.81
// and 0.90 of cuBLAS; 0.72 and 0.83 for single calls).
//
// Warp 0 of each CTA issues TMA into a ring of 64-deep stages; warp 1 of the
// leader issues tcgen05.mma for the pair; warps 2..17 drain.  The accumulators
// fill the tensor memory: the next tile's products into the first one start
// as soon as it is drained and run ahead of the second by up to the ring's
// stages.  Tiles of up to 128 rows take half of it, so two of them alternate.
// A thread drains one feature (TMEM lane): a warp's 2-byte access to a row is
// 64 consecutive bytes, whatever the row stride.  (Turning 8 rows in shared
// memory for 16-byte accesses takes twice the shared-memory cycles, of which
// the products leave 15%: 8% slower.)
// Both operands may be K-major or MN-major in shared memory: W is taken as
// stored ([k][n] or [n][k]), and the sums product reads x and dz as they are,
// contracting over their rows.
//
// The offsets stay on the device: every CTA scans them into shared memory and
// walks the same tile order, so a call captured into a graph follows new
// offsets at replay.  A rows tile that ends inside another expert's rows
// computes them and does not store them (a row meets only its own
// accumulators); a sums tile zeroes the rows behind its expert's last in
// shared memory before the product, because there they would be added in.
#include <atomic>
#include <cstring>
#include "kq_expert_rows.cuh"

namespace kq {
namespace {

constexpr int BK = 64, MAX_STAGES = 6;
constexpr int TILE = 256;                       // features of an accumulator pair, rows of a tile at most
constexpr int SIDE_BYTES = 128 * BK * 2;        // a CTA's share of one accumulator's A, or of B
constexpr int RING_BYTES = 12 * SIDE_BYTES;     // 4 stages with two accumulators' A, or 6 with one
constexpr int CHUNK = 64 * 128;                 // 64 rows of 128 bytes: one MN-major slab
constexpr int DRAIN_WARPS = 16, THREADS = 64 + 32 * DRAIN_WARPS;
constexpr int TR = 8, STRIDE = TR * DRAIN_WARPS / 4;   // rows that a drain warp takes at a time; the warps of a quadrant alternate
constexpr int GROUP_BYTES = (3 * kMaxExperts + 4) * 4;
constexpr int SMEM_BYTES = RING_BYTES + GROUP_BYTES + 1024;

enum { EPI_FORWARD, EPI_GRAD, EPI_SUMS };

struct Params {
    const int64_t* offsets;
    const void* bias;
    const void* aux;       // residual (forward) or dy (gradient)
    void *out, *low;       // low (gradient): what the rounding of dz leaves out, or null
    int64_t bias_stride, ld_aux, ld_out, out_stride;   // out_stride: per expert (sums)
    int rows, experts, k_steps, m_tiles, n_tiles;
    int m_out, n_out;      // output extents: features, and (sums) rows
    int span;              // features of a tile: one accumulator's or two's (gated: of gate and of up)
    int up;                // gated: first coordinate of the up half in W
    int* err;
    uint32_t idesc;        // without N
    int act;
    bool a_mn, b_mn, zero_rest;
    bool lines, wide;      // (sums) a lane drains a line of dW, not a column; its lines start on 32 bytes
};

struct Tile { int e, row0, count, m0, n0, n, k_steps, accs; };   // accs: accumulators with live features

// Tile t of the launch; m0 in features, n the extent of the tensor product's N axis.
template <int EPI, bool GATED>
__device__ __forceinline__ bool tile_at(const Params& p, const int* lo, const int* cnt, const int* cum, int64_t t, Tile& o) {
    if constexpr (EPI == EPI_SUMS) {
        const int per = p.m_tiles * p.n_tiles;
        if (t >= (int64_t)per * p.experts) return false;
        o.e = (int)(t / per);
        const int l = (int)(t - (int64_t)o.e * per);
        o.m0 = (l % p.m_tiles) * p.span;
        o.n0 = (l / p.m_tiles) * TILE;
        o.row0 = lo[o.e];
        o.count = cnt[o.e];
        o.n = p.n_out - o.n0 > 128 ? 256 : 128;
        o.k_steps = (o.count + BK - 1) / BK;
    } else {
        // The row tiles of an expert run fastest: the pairs that share a slice of W run together.
        if (t >= (int64_t)cum[p.experts] * p.m_tiles) return false;
        o.e = expert_of(cum, p.experts, (int)(t / p.m_tiles));
        const int nt = cum[o.e + 1] - cum[o.e];
        const int64_t l = t - (int64_t)cum[o.e] * p.m_tiles;
        const int r = (int)(l % nt) * TILE;
        o.m0 = (int)(l / nt) * p.span;
        o.n0 = 0;
        o.row0 = lo[o.e] + r;
        o.count = min(cnt[o.e] - r, TILE);
        o.n = (o.count + 63) & ~63;
        o.k_steps = p.k_steps;
    }
    o.accs = GATED || (p.span > TILE && p.m_out - o.m0 > TILE) ? 2 : 1;
    return true;
}

// Position in a ring of stages.
struct Ring {
    uint32_t s = 0, phase = 0;
    __device__ __forceinline__ void next(uint32_t stages) {
        if (++s == stages) { s = 0; phase ^= 1; }
    }
    __device__ __forceinline__ void skip(uint32_t n, uint32_t stages) {
        s += n;
        phase ^= (s / stages) & 1;
        s %= stages;
    }
};

// Zeroes rows valid .. 63 of a sums stage in this CTA once its loads have landed.  Whole warp.
__device__ __forceinline__ bool zero_tail(uint8_t* stage, int slabs, int valid, uint64_t* tail_bar, uint32_t parity, int lane) {
    const bool ok = mbar_wait(tail_bar, parity);
    // Eight lanes a 128-byte row.
    for (int c = 0; c < slabs; ++c)
        for (int r = valid + (lane >> 3); r < BK; r += 4)
            *reinterpret_cast<uint4*>(stage + c * CHUNK + r * 128 + (lane & 7) * 16) = make_uint4(0, 0, 0, 0);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    return ok;
}

// TR rows of one feature: pre-activations z (and up projections u) and a (residual or dy) to the results.
template <int EPI, bool GATED, int ACT>
__device__ __forceinline__ void finish(float (&z)[TR], float (&u)[TR], const float (&a)[TR]) {
#pragma unroll
    for (int j = 0; j < TR; ++j) {
        if constexpr (EPI == EPI_FORWARD) {
            z[j] = activate<ACT>(z[j]) * (GATED ? u[j] : 1.f) + a[j];
        } else if constexpr (GATED) {
            const float du = a[j] * activate<ACT>(z[j]);
            z[j] = a[j] * u[j] * slope<ACT>(z[j]);
            u[j] = du;
        } else {
            z[j] = a[j] * slope<ACT>(z[j]);
        }
    }
}

// TR rows of one feature, row stride ld: a warp's access to a row is 64 consecutive bytes.
template <typename T>
__device__ __forceinline__ void fetch_rows(T (&v)[TR], const T* src, int64_t ld, int rows) {
#pragma unroll
    for (int j = 0; j < TR; ++j) {
        v[j] = src[0];
        src += j + 1 < rows ? ld : 0;            // the last row again behind the end: no branch around a load
    }
}

template <typename T>
__device__ __forceinline__ void store_rows(T* dst, int64_t ld, int rows, const float (&v)[TR]) {
#pragma unroll
    for (int j = 0; j < TR; ++j) {
        if (j < rows) dst[0] = from_f<T>(v[j]);
        dst += ld;
    }
}

// A warp's 32 lines of dW, a line a lane, 16 columns (32 bytes) at a time; the four warps of a quadrant take turns and fill
// 128-byte lines between them.
template <typename T>
__device__ __forceinline__ void drain_lines(uint32_t tmem, T* line, bool live, int first, int step, int n, bool wide, bool zero) {
#pragma unroll 1
    for (int c = first; c < n; c += step) {
        uint32_t v[16], o[8];
        tmem_ld16(tmem + c, v);
        tmem_wait_ld();
        T* h = reinterpret_cast<T*>(o);
#pragma unroll
        for (int j = 0; j < 16; ++j) h[j] = from_f<T>(zero ? 0.f : __uint_as_float(v[j]));
        if (live) {
            if (c + 16 <= n && wide) {
                asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(line + c), "r"(o[0]), "r"(o[1]),
                             "r"(o[2]), "r"(o[3]), "r"(o[4]), "r"(o[5]), "r"(o[6]), "r"(o[7])
                             : "memory");
            } else if (c + 16 <= n) {
                reinterpret_cast<uint4*>(line + c)[0] = make_uint4(o[0], o[1], o[2], o[3]);
                reinterpret_cast<uint4*>(line + c)[1] = make_uint4(o[4], o[5], o[6], o[7]);
            } else {
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    if (c + j < n) line[c + j] = h[j];
            }
        }
        __syncwarp();                            // the next tensor-memory load is the whole warp's
    }
}

template <typename T, int EPI, bool GATED>
__global__ void __launch_bounds__(THREADS, 1)
expert_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
              const __grid_constant__ CUtensorMap map_b_full, const Params p) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t full_bar[MAX_STAGES], empty_bar[MAX_STAGES], tail_bar[MAX_STAGES], acc_full[2], acc_empty[2];
    __shared__ uint32_t tmem_slot;
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    int* lo = reinterpret_cast<int*>(smem + RING_BYTES);
    int* cnt = lo + kMaxExperts;
    int* cum = cnt + kMaxExperts;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)cluster_rank();
    const int64_t first = blockIdx.x >> 1, step = gridDim.x >> 1;
    const int a_parts = GATED || p.span > TILE ? 2 : 1;      // accumulators a stage has room for
    const uint32_t stages = 12 / (a_parts + 1), stage_bytes = (a_parts + 1) * SIDE_BYTES, b_at = a_parts * SIDE_BYTES;

    if (threadIdx.x == 0) {
        tma_prefetch(&map_a);
        tma_prefetch(&map_b);
        tma_prefetch(&map_b_full);
        for (int s = 0; s < MAX_STAGES; ++s) {
            mbar_init(&full_bar[s], 1);
            mbar_init(&empty_bar[s], 1);
            mbar_init(&tail_bar[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&acc_full[b], 1);
            mbar_init(&acc_empty[b], 2 * DRAIN_WARPS);
        }
        mbar_init_fence();
    }
    if (warp == 1) tmem2_alloc(&tmem_slot, 2 * TILE);
    scan_groups(p.offsets, p.experts, p.rows, TILE, lo, cnt, cum);
    tc_fence_before();
    __syncthreads();
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    bool ok = true;
    Tile t;

    // Halves of the tensor memory (256 columns) are used in turn.  A tile with two accumulators of more than 128 rows
    // takes two turns, any other tile one (its second accumulator at column 128).
    auto two_turns = [](const Tile& t) { return t.accs == 2 && t.n > 128; };

    if (warp == 0) {
        if (lane == 0) {
            Ring ring;
            for (int64_t i = first; ok && tile_at<EPI, GATED>(p, lo, cnt, cum, i, t); i += step) {
                const int half = t.n >> 1;
                const uint32_t bytes = t.accs * SIDE_BYTES + half * 128;
                for (int ks = 0; ks < t.k_steps; ++ks, ring.next(stages)) {
                    const uint32_t s = ring.s;
                    if (!(ok = mbar_wait(&empty_bar[s], ring.phase ^ 1))) break;
                    uint8_t *sa = smem + s * stage_bytes, *sb = sa + b_at;
                    uint32_t bar = leader_addr(&full_bar[s]);
                    const int r = t.row0 + ks * BK;
                    if (EPI == EPI_SUMS && t.count - ks * BK < BK) {   // the tail is zeroed here before it counts as loaded
                        bar = smem_addr(&tail_bar[s]);
                        mbar_expect_tx(&tail_bar[s], bytes);
                    } else if (rank == 0) {
                        mbar_expect_tx(&full_bar[s], 2 * bytes);
                    }
                    for (int a = 0; a < t.accs; ++a) {
                        const int f = t.m0 + rank * 128 + (a ? (GATED ? p.up : TILE) : 0);
                        uint8_t* dst = sa + a * SIDE_BYTES;
                        if constexpr (EPI == EPI_SUMS) {
                            tma2_load_2d(dst, &map_a, f, r, bar);
                            tma2_load_2d(dst + CHUNK, &map_a, f + 64, r, bar);
                        } else if (p.a_mn) {
                            tma2_load_3d(dst, &map_a, f, ks * BK, t.e, bar);
                            tma2_load_3d(dst + CHUNK, &map_a, f + 64, ks * BK, t.e, bar);
                        } else {
                            tma2_load_3d(dst, &map_a, ks * BK, f, t.e, bar);
                        }
                    }
                    if constexpr (EPI == EPI_SUMS) {
                        for (int c = 0; c < half; c += 64)
                            tma2_load_2d(sb + (c >> 6) * CHUNK, &map_b, t.n0 + rank * half + c, r, bar);
                    } else if (half == 128) {
                        tma2_load_2d(sb, &map_b_full, ks * BK, t.row0 + rank * half, bar);
                    } else {
                        for (int c = 0; c < half; c += 32)
                            tma2_load_2d(sb + c * 128, &map_b, ks * BK, t.row0 + rank * half + c, bar);
                    }
                }
            }
            if (!ok) report_wait_error(p.err);
        }
    } else if (warp == 1) {
        Ring at;                                // the stage of the next products into the tile's last accumulator
        uint32_t turn = 0, tails = 0;           // tails: the phase of every stage's tail_bar
        const uint32_t a_step = p.a_mn ? 128 : 2, b_step = p.b_mn ? 128 : 2;   // 16 contraction values, in 16-byte units
        for (int64_t i = first; ok && tile_at<EPI, GATED>(p, lo, cnt, cum, i, t); i += step) {
            const int tail_step = EPI == EPI_SUMS && (t.count % BK) != 0 ? t.k_steps - 1 : -1;
            const int slabs = b_at / CHUNK + (t.n >> 7);
            if (rank != 0) {                    // the leader issues for both; this CTA zeroes its own tails
                at.skip(t.k_steps, stages);
                if (tail_step >= 0) {
                    const uint32_t s = at.s ? at.s - 1 : stages - 1;
                    ok = zero_tail(smem + s * stage_bytes, slabs, t.count % BK, &tail_bar[s], (tails >> s) & 1, lane);
                    if (lane == 0) mbar_arrive_remote(leader_addr(&full_bar[s]));
                    tails ^= 1u << s;
                }
                continue;
            }
            const bool two = two_turns(t);
            const int h0 = turn & 1, h1 = (turn + 1) & 1;
            const uint32_t col[2] = {tmem + h0 * TILE, two ? tmem + h1 * TILE : tmem + h0 * TILE + 128};
            const uint32_t idesc = p.idesc | ((uint32_t)(t.n >> 3) << 17);
            auto products = [&](int a, int ks, uint32_t s) {
                if (lane == 0) {
                    const uint32_t base = smem_addr(smem + s * stage_bytes);
                    const uint64_t ad = smem_desc(base + a * SIDE_BYTES, p.a_mn ? CHUNK : 16);
                    const uint64_t bd = smem_desc(base + b_at, p.b_mn ? CHUNK : 16);
#pragma unroll
                    for (int kk = 0; kk < BK / 16; ++kk)
                        mma2_f16(col[a], ad + a_step * kk, bd + b_step * kk, idesc, (ks | kk) != 0);
                    if (a == t.accs - 1) mma2_commit(&empty_bar[s]);
                }
                __syncwarp();
            };
            auto loaded = [&](int ks, const Ring& r) {
                const uint32_t s = r.s, parity = r.phase;
                bool got = true;
                if (ks == tail_step) {          // the only arrival on full_bar is the other CTA's, for its zeroed half
                    got = zero_tail(smem + s * stage_bytes, slabs, t.count % BK, &tail_bar[s], (tails >> s) & 1, lane) &&
                          mbar_wait_cluster(&full_bar[s], parity);
                    tails ^= 1u << s;
                }
                got = got && mbar_wait(&full_bar[s], parity);
                tc_fence_after();
                return got;
            };
            if (!(ok = mbar_wait(&acc_empty[h0], ((turn >> 1) & 1) ^ 1))) break;
            tc_fence_after();
            int done0 = 0;                      // k steps issued into the first accumulator, at `lead` in the ring
            Ring lead = at;
            if (two) {
                // Until the second accumulator is drained, the first goes ahead through the stages in the ring.
                const uint32_t parity = (((turn + 1) >> 1) & 1) ^ 1;
                const int ahead = min(t.k_steps, (int)stages);
                while (done0 < ahead && ok && !__shfl_sync(0xFFFFFFFFu, (int)mbar_test(&acc_empty[h1], parity), 0)) {
                    if ((ok = loaded(done0, lead))) products(0, done0++, lead.s);
                    lead.next(stages);
                }
                if (!(ok = ok && mbar_wait(&acc_empty[h1], parity))) break;
                tc_fence_after();
            }
            for (int ks = 0; ks < t.k_steps; ++ks, at.next(stages)) {
                if (ks == done0) {
                    if (!(ok = loaded(ks, at))) break;
                    products(0, ks, at.s);
                    ++done0;
                }
                if (two && ks == t.k_steps - 1 && lane == 0) mma2_commit(&acc_full[h0]);
                if (t.accs == 2) products(1, ks, at.s);
            }
            if (ok && lane == 0) {
                if (two && t.k_steps == 0) mma2_commit(&acc_full[h0]);
                mma2_commit(&acc_full[two ? h1 : h0]);
            }
            __syncwarp();
            turn += two ? 2 : 1;
        }
        if (!ok && lane == 0) report_wait_error(p.err);
    } else {
        const int q = warp & 3, h = (warp - 2) >> 2;    // tensor-memory lanes 32q.., TR of every STRIDE columns
        uint32_t turn = 0;
        for (int64_t i = first; tile_at<EPI, GATED>(p, lo, cnt, cum, i, t); i += step) {
            const bool two = two_turns(t);
            const int h0 = turn & 1, h1 = (turn + 1) & 1;
            const uint32_t lanes = tmem + ((uint32_t)(q * 32) << 16);
            const uint32_t col[2] = {lanes + h0 * TILE, two ? lanes + h1 * TILE : lanes + h0 * TILE + 128};
            ok = mbar_wait(&acc_full[h0], (turn >> 1) & 1);
            if (GATED && two) ok = ok && mbar_wait(&acc_full[h1], ((turn + 1) >> 1) & 1);
            if (!(ok = __all_sync(0xFFFFFFFFu, ok))) break;
            tc_fence_after();
            for (int a = 0; a < (GATED ? 1 : t.accs); ++a) {
                if (a == 1 && two) {                    // the first accumulator is free before the second is looked at
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_remote(leader_addr(&acc_empty[h0]));
                    if (!(ok = __all_sync(0xFFFFFFFFu, mbar_wait(&acc_full[h1], ((turn + 1) >> 1) & 1)))) break;
                    tc_fence_after();
                }
                const uint32_t base = col[a];
                const int f0 = t.m0 + a * TILE + rank * 128 + q * 32, cols = p.m_out - f0;   // this warp's features
                if (cols <= 0) continue;
                const int n = EPI == EPI_SUMS ? min(p.n_out - t.n0, TILE) : t.count;         // rows of the output
                if constexpr (EPI == EPI_SUMS) {
                    if (p.lines) {
                        const bool live = lane < cols;
                        T* line = static_cast<T*>(p.out) + t.e * p.out_stride + (int64_t)(f0 + (live ? lane : 0)) * p.ld_out + t.n0;
                        drain_lines(base, line, live, h * 16, 4 * DRAIN_WARPS, n, p.wide, t.k_steps == 0);
                        continue;
                    }
                }
                T* out;
                const T* aux = nullptr;
                float add = 0.f, add_up = 0.f;
                if constexpr (EPI == EPI_SUMS) {
                    out = static_cast<T*>(p.out) + t.e * p.out_stride + (int64_t)t.n0 * p.ld_out + f0;
                } else {
                    out = static_cast<T*>(p.out) + (int64_t)t.row0 * p.ld_out + f0;
                    if (p.aux) aux = static_cast<const T*>(p.aux) + (int64_t)t.row0 * p.ld_aux + f0;
                    if (p.bias && lane < cols) {
                        const T* bias = static_cast<const T*>(p.bias) + t.e * p.bias_stride + f0 + lane;
                        add = to_f<T>(bias[0]);
                        if constexpr (GATED) add_up = to_f<T>(bias[p.m_out]);
                    }
                }
                const int begin = h * TR;
                const bool live = lane < cols;
                out += min(lane, cols - 1);
                if (aux) aux += min(lane, cols - 1);
                T ahead[TR];
                if (aux && begin < n) fetch_rows(ahead, aux + (int64_t)begin * p.ld_aux, p.ld_aux, n - begin);
                uint32_t v[TR], w[TR];
                __syncwarp();                           // tensor-memory loads are the whole warp's
                if (begin < n) {
                    tmem_ld8(base + begin, v);
                    if constexpr (GATED) tmem_ld8(col[1] + begin, w);
                    tmem_wait_ld();
                }
#pragma unroll 1
                for (int c = begin; c < n; c += STRIDE) {
                    float z[TR], u[TR], x[TR];
#pragma unroll
                    for (int j = 0; j < TR; ++j) {
                        x[j] = aux ? to_f<T>(ahead[j]) : 0.f;
                        z[j] = __uint_as_float(v[j]) + add;
                        if constexpr (GATED) u[j] = __uint_as_float(w[j]) + add_up;
                        if (EPI == EPI_SUMS && t.k_steps == 0) z[j] = 0.f;
                    }
                    if (c + STRIDE < n) {               // the next rows, under this chunk's arithmetic
                        if (aux) fetch_rows(ahead, aux + (int64_t)(c + STRIDE) * p.ld_aux, p.ld_aux, n - c - STRIDE);
                        tmem_ld8(base + c + STRIDE, v);
                        if constexpr (GATED) tmem_ld8(col[1] + c + STRIDE, w);
                    }
                    if constexpr (EPI != EPI_SUMS) {
                        switch (p.act) {
                            case KQ_ACT_RELU: finish<EPI, GATED, KQ_ACT_RELU>(z, u, x); break;
                            case KQ_ACT_SILU: finish<EPI, GATED, KQ_ACT_SILU>(z, u, x); break;
                            case KQ_ACT_GELU: finish<EPI, GATED, KQ_ACT_GELU>(z, u, x); break;
                            default: finish<EPI, GATED, KQ_ACT_NONE>(z, u, x);
                        }
                    }
                    store_rows(out + (int64_t)c * p.ld_out, p.ld_out, live ? n - c : 0, z);
                    if constexpr (EPI == EPI_GRAD && GATED)
                        store_rows(out + (int64_t)c * p.ld_out + p.m_out, p.ld_out, live ? n - c : 0, u);
                    if (EPI == EPI_GRAD && p.low) {
                        T* low = static_cast<T*>(p.low) + (out - static_cast<T*>(p.out)) + (int64_t)c * p.ld_out;
#pragma unroll
                        for (int j = 0; j < TR; ++j) {
                            z[j] = left_out<T>(z[j]);
                            if constexpr (GATED) u[j] = left_out<T>(u[j]);
                        }
                        store_rows(low, p.ld_out, live ? n - c : 0, z);
                        if constexpr (GATED) store_rows(low + p.m_out, p.ld_out, live ? n - c : 0, u);
                    }
                    __syncwarp();
                    tmem_wait_ld();
                }
            }
            if (!ok) break;
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive_remote(leader_addr(&acc_empty[two ? h1 : h0]));
                if (GATED && two) mbar_arrive_remote(leader_addr(&acc_empty[h0]));
            }
            turn += two ? 2 : 1;
        }
        if (!ok && lane == 0) report_wait_error(p.err);
        // Rows of no expert: zero in a fresh output, untouched otherwise.
        if (EPI != EPI_SUMS && p.zero_rest && p.offsets) {
            int begin, end, n;
            group_of(p.offsets, 0, p.rows, begin, n);
            group_of(p.offsets, p.experts - 1, p.rows, end, n);
            end += n;
            for (int row = blockIdx.x; row < p.rows; row += gridDim.x) {
                if (row >= begin && row < end) continue;
                T* o = static_cast<T*>(p.out) + (int64_t)row * p.ld_out;
                for (int j = threadIdx.x - 64; j < p.m_out; j += 32 * DRAIN_WARPS) o[j] = from_f<T>(0.f);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();                              // the pair's memory and barriers are in use until both are here
    tc_fence_after();
    if (warp == 1) tmem2_free(tmem, 2 * TILE);
}

// 16-bit rows [batch][r][c] -> [batch][r][cols_out]: an operand whose base or
// strides are not the multiples of 16 bytes that TMA needs is laid out once
// more.  Columns c .. cols_out are not written (no tile map reaches them, or
// only as output columns that are not stored).  Up to three copies in one
// launch (blockIdx.y); a warp a row at a time.
struct Copy {
    const uint16_t* src;
    uint16_t* dst;
    int64_t sb, sr, db, rows, r;       // rows = batch * r
    int c, cols_out;
};

struct Copies {
    Copy job[3];
    int n = 0;
};

__global__ void __launch_bounds__(256) relayout_kernel(const Copies copies) {
    const Copy& j = copies.job[blockIdx.y];
    const int lane = threadIdx.x & 31;
    for (int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); row < j.rows; row += (int64_t)gridDim.x * 8) {
        const int64_t b = j.r == j.rows ? 0 : row / j.r, y = row - b * j.r;
        const uint16_t* s = j.src + b * j.sb + y * j.sr;
        uint16_t* d = j.dst + b * j.db + y * j.cols_out;       // rows start on 16 bytes
        int c = lane * 2;
#pragma unroll 4
        for (; c + 1 < j.c; c += 64) *reinterpret_cast<uint32_t*>(d + c) = (uint32_t)s[c] | ((uint32_t)s[c + 1] << 16);
        if (c < j.c) d[c] = s[c];
    }
}

// Column sums of dz (and of what its rounding left out) over every expert's rows, fp32 in row order within a
// thread: one warp per 32 columns and expert, rows split over 8 warps.
template <typename T>
__global__ void __launch_bounds__(256)
bias_grad_kernel(const T* __restrict__ dz, const T* __restrict__ low, int64_t ld, const int64_t* __restrict__ offsets, int rows, int n, T* __restrict__ db,
                 int64_t db_stride) {
    __shared__ float part[8][32];
    const int e = blockIdx.y, lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int j = blockIdx.x * 32 + lane;
    int lo, count;
    group_of(offsets, e, rows, lo, count);
    float s = 0.f;
    if (j < n)
#pragma unroll 8
        for (int r = w; r < count; r += 8) {
            const int64_t at = (int64_t)(lo + r) * ld + j;
            s += to_f<T>(dz[at]) + (low ? to_f<T>(low[at]) : 0.f);
        }
    part[w][lane] = s;
    __syncthreads();
    if (w == 0 && j < n) {
        s = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) s += part[i][lane];
        db[e * db_stride + j] = from_f<T>(s);
    }
}

size_t relayout_bytes(const Operand& o) {
    return o.direct ? 0 : (size_t)(o.batch * o.r * round8(o.c)) * 2;
}

// Adds the copies that `o` needs to `jobs` and points it at them.  `halves` = 2: the columns are two halves (gate and up)
// that each start on a 16-byte boundary in the copy.
void relayout(Operand& o, uint16_t*& ws, int halves, Copies& jobs) {
    if (o.direct) return;
    const int64_t part = o.c / halves, pad = round8(part), cols = pad * halves;
    for (int h = 0; h < halves; ++h)
        jobs.job[jobs.n++] = Copy{o.base + h * part, ws + h * pad, o.sb, o.sr, o.r * cols, o.batch * o.r, o.r, (int)part, (int)cols};
    o.base = ws;
    o.sr = cols;
    o.sb = o.r * cols;
    o.c = cols == pad ? o.c : cols;
    ws += (o.batch * o.r * cols + 7) & ~(int64_t)7;
    o.direct = true;
}

int run_copies(const Copies& jobs, cudaStream_t s) {
    if (!jobs.n) return KQ_OK;
    int64_t most = 0;
    for (int i = 0; i < jobs.n; ++i) most = jobs.job[i].rows > most ? jobs.job[i].rows : most;
    const int64_t blocks = (most + 7) / 8;
    relayout_kernel<<<dim3((unsigned)(blocks < 2368 ? blocks : 2368), (unsigned)jobs.n), 256, 0, s>>>(jobs);
    return check_launch("relayout_kernel");
}

// Pairs of CTAs that run at once (every instance needs a whole SM); asked once for each device.
template <typename K>
int pairs_at_once(K kernel, int* out) {
    static int known[64] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess && dev < 64 && known[dev]) { *out = known[dev]; return KQ_OK; }
    int sms;
    if (int rc = sm_count(&sms)) return rc;
    cudaLaunchConfig_t c{};
    c.gridDim = dim3((unsigned)(sms & ~1));
    c.blockDim = dim3(THREADS);
    c.dynamicSmemBytes = SMEM_BYTES;
    cudaLaunchAttribute a{};
    a.id = cudaLaunchAttributeClusterDimension;
    a.val.clusterDim = {2, 1, 1};
    c.attrs = &a;
    c.numAttrs = 1;
    int n = 0;
    if (e == cudaSuccess) e = cudaOccupancyMaxActiveClusters(&n, kernel, &c);
    if (e != cudaSuccess || n < 1) { set_error("cudaOccupancyMaxActiveClusters: %s", cudaGetErrorString(e)); return KQ_ERR_CUDA; }
    if (dev < 64) known[dev] = n;
    *out = n;
    return KQ_OK;
}

template <typename T, int EPI, bool GATED>
int launch_as(const CUtensorMap& a, const CUtensorMap& b, const CUtensorMap& b_full, const Params& p, int64_t tiles, cudaStream_t s) {
    auto kernel = expert_kernel<T, EPI, GATED>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES);
    if (e != cudaSuccess) { set_error("cudaFuncSetAttribute: %s", cudaGetErrorString(e)); return KQ_ERR_CUDA; }
    int pairs;
    if (int rc = pairs_at_once(kernel, &pairs)) return rc;
    cudaLaunchConfig_t c{};
    c.gridDim = dim3((unsigned)(2 * (tiles < pairs ? tiles : pairs)));
    c.blockDim = dim3(THREADS);
    c.dynamicSmemBytes = SMEM_BYTES;
    c.stream = s;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim = {2, 1, 1};
    c.attrs = &at;
    c.numAttrs = 1;
    e = cudaLaunchKernelEx(&c, kernel, a, b, b_full, p);
    if (e != cudaSuccess) { set_error("expert_kernel: %s", cudaGetErrorString(e)); return KQ_ERR_CUDA; }
    return check_launch("expert_kernel");
}

template <int EPI, bool GATED>
int launch(bool bf16, const CUtensorMap& a, const CUtensorMap& b, const CUtensorMap& b_full, const Params& p, int64_t tiles,
           cudaStream_t s) {
    return bf16 ? launch_as<__nv_bfloat16, EPI, GATED>(a, b, b_full, p, tiles, s)
                : launch_as<__half, EPI, GATED>(a, b, b_full, p, tiles, s);
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

// Two accumulators a tile where that leaves at least three tiles for every pair: fewer would stand idle, which costs
// more than what the shared B tile saves (256 rows, 8192 -> 18944: 94 us with one accumulator, 145 us with two).  The
// epilogue of two is under fewer products than that of one, so a short contraction whose epilogue also reads rows takes
// one (8192 rows, 1536 -> 12288 with residual: 303 us with one, 345 us with two; 7168 -> 7168: 767 and 728).
int span_for(int64_t features, int64_t other_tiles, int64_t k, bool reads_rows, bool gated, int* span) {
    int sms;
    if (int rc = sm_count(&sms)) return rc;
    const bool enough = (features + 2 * TILE - 1) / (2 * TILE) * other_tiles >= 3 * (sms / 2);
    *span = !gated && enough && !(reads_rows && k <= 2048) ? 2 * TILE : TILE;
    return KQ_OK;
}

int many_rows_product(const RowsProduct& p, cudaStream_t s) {
    CUtensorMap ma, mb, mf;
    // Large boxes where the tile takes them whole: every TMA instruction of a stage costs issue time.
    if (int rc = map_rows(&ma, p.w, p.bf16, 64, p.mn ? 64 : 128, p.what)) return rc;
    if (int rc = map_rows_2d(&mb, p.x, p.bf16, BK, 32, p.what)) return rc;
    if (int rc = map_rows_2d(&mf, p.x, p.bf16, BK, 128, p.what)) return rc;
    Params q{};
    q.err = p.err;
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
    const int64_t r_tiles = (p.rows + TILE - 1) / TILE + (p.experts < p.rows ? p.experts : p.rows) - 1;
    if (int rc = span_for(p.n_out, r_tiles, p.k, p.aux != nullptr, p.gated, &q.span)) return rc;
    q.m_tiles = (int)((p.n_out + q.span - 1) / q.span);
    q.m_out = (int)p.n_out;
    q.up = p.up;
    q.idesc = idesc_f16(p.bf16, p.mn, false, TILE, 0);
    q.act = p.act;
    q.a_mn = p.mn;
    q.zero_rest = p.zero_rest;
    const int64_t tiles = r_tiles * q.m_tiles;
    if (p.grad)
        return p.gated ? launch<EPI_GRAD, true>(p.bf16, ma, mb, mf, q, tiles, s) : launch<EPI_GRAD, false>(p.bf16, ma, mb, mf, q, tiles, s);
    return p.gated ? launch<EPI_FORWARD, true>(p.bf16, ma, mb, mf, q, tiles, s)
                   : launch<EPI_FORWARD, false>(p.bf16, ma, mb, mf, q, tiles, s);
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
    RowsProduct r{};
    if (int rc = wait_error_word(&r.err, what)) return rc;
    const bool bf16 = p.dtype == KQ_BF16, mn = n_contiguous(p);
    Operand x = operand(p.x, 1, p.rows, p.k, 0, p.ldx), w = w_operand(p, mn);
    const bool gated_copy = mn && p.gated && !w.direct;
    Copies jobs;
    relayout(x, ws, 1, jobs);
    relayout(w, ws, gated_copy ? 2 : 1, jobs);
    if (int rc = run_copies(jobs, s)) return rc;
    r.x = x;
    r.w = w;
    r.offsets = p.offsets;
    r.bias = p.bias;
    r.aux = grad ? dy : p.residual;
    r.out = p.y;
    r.low = grad ? p.y_low : nullptr;
    r.bias_stride = p.bias_stride_e;
    r.ld_aux = grad ? ld_dy : p.ld_residual;
    r.ld_out = p.ldy;
    r.rows = p.rows;
    r.k = p.k;
    r.n_out = n_out;
    r.experts = p.experts;
    r.up = (int)(gated_copy ? round8(n_out) : n_out);
    r.act = p.activation;
    r.bf16 = bf16;
    r.mn = mn;
    r.gated = p.gated != 0;
    r.grad = grad;
    r.zero_rest = p.zero_rest != 0;
    r.what = what;
    return few_rows(r) ? few_rows_product(r, s) : many_rows_product(r, s);
}

__global__ void take_errors_kernel(volatile int* word, int* out) {
    *out = *word;
    *word = 0;
}

}  // namespace

int wait_error_flag(int** out) {
    constexpr int kDevices = 64, kApart = 32;           // a 128-byte line a device
    static std::atomic<int*> words{nullptr};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) { set_error("cudaGetDevice: %s", cudaGetErrorString(e)); return KQ_ERR_CUDA; }
    if (dev >= kDevices) { set_error("device %d: at most %d devices", dev, kDevices); return KQ_ERR_ARG; }
    int* w = words.load(std::memory_order_acquire);
    if (!w) {
        // Once in a process; the first call may be a captured one, into which this allocation does not go.
        cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
        cudaThreadExchangeStreamCaptureMode(&mode);
        void* fresh = nullptr;
        e = cudaHostAlloc(&fresh, kDevices * kApart * sizeof(int), cudaHostAllocPortable | cudaHostAllocMapped);
        cudaThreadExchangeStreamCaptureMode(&mode);
        if (e != cudaSuccess) { set_error("cudaHostAlloc: %s", cudaGetErrorString(e)); return KQ_ERR_CUDA; }
        memset(fresh, 0, kDevices * kApart * sizeof(int));
        if (words.compare_exchange_strong(w, static_cast<int*>(fresh), std::memory_order_acq_rel)) w = static_cast<int*>(fresh);
        else cudaFreeHost(fresh);                       // another thread was first, w is its memory
    }
    *out = w + dev * kApart;
    return KQ_OK;
}

int wait_error_word(int** out, const char* what) {
    if (int rc = wait_error_flag(out)) return rc;
    if (*static_cast<volatile int*>(*out)) {
        set_error("%s: an internal wait of an earlier expert-layer kernel ran out; results since the last kq_wait_errors are invalid", what);
        return KQ_ERR_TIMEOUT;
    }
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

// The sides of dW, drained by column: its contiguous axis is the tensor product's M axis (a), the other its N axis (b).
struct SumsSides { Operand a, b; };

SumsSides sums_sides(const kq_expert_product& p, const void* dz, int64_t ld_dz) {
    const Operand x = operand(p.x, 1, p.rows, p.k, 0, p.ldx), z = operand(dz, 1, p.rows, p.n, 0, ld_dz);
    return n_contiguous(p) ? SumsSides{z, x} : SumsSides{x, z};
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
    Params q{};
    if (int rc = wait_error_word(&q.err, what)) return rc;
    // A lane takes a line of dW (and stores 32 bytes at a time) where lines start on 16 bytes, else a column (2 bytes, 64 a warp):
    // dW of 7168 x 4096, 8 experts, 4096 uneven rows: 313 us against 362.
    SumsSides o = sums_sides(p, dz, ld_dz);
    const bool by_line = (((uintptr_t)dw | (uintptr_t)(ld * 2) | (uintptr_t)(p.experts > 1 ? p.w_stride_e * 2 : 0)) & 15) == 0;
    const bool wide = (((uintptr_t)dw | (uintptr_t)(ld * 2) | (uintptr_t)(p.experts > 1 ? p.w_stride_e * 2 : 0)) & 31) == 0;
    if (by_line) o = SumsSides{o.b, o.a};
    const int64_t m_out = by_line ? lines : cols, n_out = by_line ? cols : lines;
    Copies jobs;
    relayout(o.a, ws, 1, jobs);
    relayout(o.b, ws, 1, jobs);
    if (int rc = run_copies(jobs, s)) return rc;
    CUtensorMap ma, mb;
    if (int rc = map_rows_2d(&ma, o.a, bf16, 64, BK, what)) return rc;
    if (int rc = map_rows_2d(&mb, o.b, bf16, 64, BK, what)) return rc;
    q.offsets = p.offsets;
    q.out = dw;
    q.ld_out = ld;
    q.out_stride = p.w_stride_e;
    q.rows = (int)p.rows;
    q.experts = (int)p.experts;
    q.n_tiles = (int)((n_out + TILE - 1) / TILE);
    // Few rows are few products to drain under: one accumulator then, so that the two halves of the tensor memory alternate
    // (8 experts of 7168 x 4096, one / two accumulators, back to back: 263 / 298 us at 512 rows each, 305 / 326 at 640, 353 / 364
    // at 768, 442 / 435 at 1024, 822 / 744 at 2048).
    q.span = TILE;
    if (p.rows > 640 * (p.experts < p.rows ? p.experts : p.rows))
        if (int rc = span_for(m_out, (int64_t)q.n_tiles * p.experts, p.rows, false, false, &q.span)) return rc;
    q.m_tiles = (int)((m_out + q.span - 1) / q.span);
    q.m_out = (int)m_out;
    q.n_out = (int)n_out;
    q.lines = by_line;
    q.wide = wide;
    q.idesc = idesc_f16(bf16, true, true, TILE, 0);
    q.a_mn = q.b_mn = true;
    if ((int64_t)q.m_tiles * q.n_tiles > 0x7FFFFFFF) { set_error("%s: problem too large", what); return KQ_ERR_ARG; }
    return launch<EPI_SUMS, false>(bf16, ma, mb, mb, q, (int64_t)q.m_tiles * q.n_tiles * p.experts, s);
}

extern "C" int kq_expert_bias_grad(const void* dz, const void* dz_low, int64_t ld_dz, const int64_t* offsets, int64_t rows, int64_t n,
                                   int64_t experts, int dtype, void* db, int64_t db_stride_e, void* stream) {
    using namespace kq;
    const char* what = "kq_expert_bias_grad";
    if (!db || (rows > 0 && !dz) || rows < 0 || n <= 0 || experts <= 0 || experts > kMaxExperts || (experts > 1 && !offsets) ||
        rows > 0x7FFFFF00 || n > 0x7FFFFF00 || (dtype != KQ_BF16 && dtype != KQ_FP16)) {
        set_error("%s: bad arguments (rows=%lld n=%lld experts=%lld)", what, (long long)rows, (long long)n, (long long)experts);
        return KQ_ERR_ARG;
    }
    int* flag;                                  // this kernel has no waits, but dz may come from one that had
    if (int rc = wait_error_word(&flag, what)) return rc;
    const dim3 grid((unsigned)((n + 31) / 32), (unsigned)experts);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (dtype == KQ_BF16)
        bias_grad_kernel<<<grid, 256, 0, s>>>(static_cast<const __nv_bfloat16*>(dz), static_cast<const __nv_bfloat16*>(dz_low), ld_dz, offsets, (int)rows, (int)n,
                                              static_cast<__nv_bfloat16*>(db), db_stride_e);
    else
        bias_grad_kernel<<<grid, 256, 0, s>>>(static_cast<const __half*>(dz), static_cast<const __half*>(dz_low), ld_dz, offsets, (int)rows, (int)n,
                                              static_cast<__half*>(db), db_stride_e);
    return check_launch(what);
}

extern "C" int kq_wait_errors(int32_t* out, void* stream) {
    if (!out) { kq::set_error("kq_wait_errors: null pointer"); return KQ_ERR_ARG; }
    int* word;
    if (int rc = kq::wait_error_flag(&word)) return rc;
    kq::take_errors_kernel<<<1, 1, 0, static_cast<cudaStream_t>(stream)>>>(word, out);
    return kq::check_launch("kq_wait_errors");
}

extern "C" int kq_wait_error_flag(int32_t** flag) {
    if (!flag) { kq::set_error("kq_wait_error_flag: null pointer"); return KQ_ERR_ARG; }
    return kq::wait_error_flag(flag);
}
