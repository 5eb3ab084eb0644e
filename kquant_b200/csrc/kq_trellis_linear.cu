// Products with encoded matrices straight from their packed trellis payload:
//
//     y[r] = had(had(x[r] * suh_e) What_e) * svh_e       rows r of expert e
//
// which is x[r] times the reconstructed weight had_l(What) * suh, had_r, * svh
// (kquant/exl3_encoder_backend.py:2211-2216), with What decoded from the
// 16 K words of each 16 x 16 tile as it is needed.
//
// The input transform writes x' = had(x * suh) once, in binary16 with a power
// of two per row that brings its bound to 2^14 (the labels are binary16, so
// both operands of the tensor product are): 11 bits of x' against the 8 or 11
// bits of x and y.  Products are summed in fp32, the output transform runs in
// fp32, and y is rounded once.
//
// With few rows an expert, the payload is decoded in registers next to the
// product (kq_trellis_few.cuh) and partial sums over ranges of k are added up
// by the output transform.  With more it is decoded into the tensor core's
// tiles (kq_trellis_rows.cuh); with many it is decoded once, to binary16 in
// the workspace, and the tensor-core product with the rotation in its epilogue
// reads that (kq_expert_rotated.cu).
#include "kq_expert_rows.cuh"
#include "kq_trellis_decode.cuh"

namespace kq {
namespace {

// Place of one row: its expert or -1, and, counting row tiles of `tile` rows, its own and all of them.  The whole block looks
// at all offsets at once.
struct Place { int e, tile, tiles; };

__device__ __forceinline__ Place place_of_row(const int64_t* offsets, int experts, int rows, int row, int tile) {
    __shared__ int e_of, lo_of, before, all;
    if (threadIdx.x == 0) { e_of = -1; lo_of = 0; before = 0; all = 0; }
    __syncthreads();
    for (int e = threadIdx.x; e < experts; e += blockDim.x) {
        int lo, n;
        group_of(offsets, e, rows, lo, n);
        if (!n) continue;
        const int t = (n + tile - 1) / tile;
        atomicAdd(&all, t);
        if (row >= lo && row < lo + n) {
            e_of = e;
            lo_of = lo;
        } else if (lo + n <= row) {
            atomicAdd(&before, t);
        }
    }
    __syncthreads();
    return Place{e_of, before + (row - lo_of) / tile, all};
}

__device__ __forceinline__ void had128_warp(float (&v)[4], int lane) {
    const float a = v[0] + v[1], b = v[0] - v[1], c = v[2] + v[3], d = v[2] - v[3];
    v[0] = a + c; v[2] = a - c; v[1] = b + d; v[3] = b - d;
#pragma unroll
    for (int m = 1; m < 32; m <<= 1)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float o = __shfl_xor_sync(0xFFFFFFFFu, v[i], m);
            v[i] = (lane & m) ? o - v[i] : v[i] + o;
        }
}

// 4 consecutive 16-bit values, 8 bytes at once where the address allows it.
template <typename T>
__device__ __forceinline__ void load4(const T* p, float (&v)[4]) {
    if ((reinterpret_cast<uintptr_t>(p) & 7) == 0) {
        const uint2 q = __ldg(reinterpret_cast<const uint2*>(p));
        const T* h = reinterpret_cast<const T*>(&q);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = to_f<T>(h[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = to_f<T>(p[i]);
    }
}

template <typename T>
__device__ __forceinline__ void store4(T* p, const float (&v)[4]) {
    if ((reinterpret_cast<uintptr_t>(p) & 7) == 0) {
        uint2 q;
        T* h = reinterpret_cast<T*>(&q);
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = from_f<T>(v[i]);
        *reinterpret_cast<uint2*>(p) = q;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = from_f<T>(v[i]);
    }
}

// x' = had(x * suh) * 2^s in binary16 and 2^-s; one block a row, a warp a Hadamard block of 128 channels.  The row's
// largest product decides s, so it is held in registers between the two (up to HELD blocks a warp; longer rows are read
// twice).
template <typename T, int WARPS>
__global__ void __launch_bounds__(WARPS * 32) rotate_in_kernel(const T* __restrict__ x, int64_t ldx, const __half* __restrict__ suh,
                                                        int64_t suh_stride, const int64_t* __restrict__ offsets, int rows,
                                                        int experts, int k, __half* __restrict__ xr, float* __restrict__ scale) {
    constexpr int HELD = 4;
    __shared__ float most[WARPS];
    let_next_start();
    const int row = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, blocks = k / kBlock;
    const int e = place_of_row(offsets, experts, rows, row, 1).e;
    if (e < 0) return;
    const T* xp = x + (int64_t)row * ldx;
    const __half* sp = suh + e * suh_stride;
    auto fetch = [&](int blk, float (&v)[4]) {
        float s[4];
        load4(xp + blk * kBlock + lane * 4, v);
        load4(sp + blk * kBlock + lane * 4, s);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] *= s[i];
    };
    float held[HELD][4];
    float m = 0.f;
#pragma unroll
    for (int h = 0; h < HELD; ++h) {
        if (warp + h * WARPS < blocks) {
            fetch(warp + h * WARPS, held[h]);
#pragma unroll
            for (int i = 0; i < 4; ++i) m = fmaxf(m, fabsf(held[h][i]));
        }
    }
    for (int blk = warp + HELD * WARPS; blk < blocks; blk += WARPS) {
        float v[4];
        fetch(blk, v);
#pragma unroll
        for (int i = 0; i < 4; ++i) m = fmaxf(m, fabsf(v[i]));
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, d));
    if (lane == 0) most[warp] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < WARPS; ++i) m = fmaxf(m, most[i]);
    // |had(v)| <= sqrt(128) max |v| < 2^4 max |v|: the exponent that brings it to at most 2^14.
    int ex = 0;
    if (m > 0.f && m < 3.3e38f) {
        frexpf(m, &ex);                                // m < 2^ex
        ex = min(max(10 - ex, -120), 120);
    }
    // The power of two goes in first: the transform of values near the end of the fp32 range stays in it.
    const float up = ldexpf(1.f, ex), norm = 0.08838834764831845f;      // 1 / sqrt(128)
    auto emit = [&](int blk, float (&v)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] *= up;
        had128_warp(v, lane);
        __half2 o[2] = {__floats2half2_rn(v[0] * norm, v[1] * norm), __floats2half2_rn(v[2] * norm, v[3] * norm)};
        *reinterpret_cast<uint2*>(xr + (int64_t)row * k + blk * kBlock + lane * 4) = *reinterpret_cast<const uint2*>(o);
    };
#pragma unroll
    for (int h = 0; h < HELD; ++h)
        if (warp + h * WARPS < blocks) emit(warp + h * WARPS, held[h]);
    for (int blk = warp + HELD * WARPS; blk < blocks; blk += WARPS) {
        float v[4];
        fetch(blk, v);
        emit(blk, v);
    }
    if (threadIdx.x == 0) scale[row] = ldexpf(1.f, -ex);
}

// Four floats that are read once; not before wait_for_last.
__device__ __forceinline__ float4 load_once(const float* p) {
    float4 v;
    asm volatile("ld.global.cs.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p) : "memory");
    return v;
}

// y = had(sum of the partial sums) * svh * 2^-s; a warp a Hadamard block of one row.  Rows of no expert: zeros in a fresh
// output.
template <typename T>
__global__ void __launch_bounds__(256) rotate_out_kernel(const float* partial, int parts, int ctas, int kt, bool wide,
                                                         const float* scale,
                                                         const __half* __restrict__ svh, int64_t svh_stride,
                                                         const int64_t* __restrict__ offsets, int rows, int experts, int n,
                                                         T* __restrict__ y, int64_t ldy, bool zero_rest) {
    const int row = blockIdx.x, lane = threadIdx.x & 31, blk = blockIdx.y * 8 + (threadIdx.x >> 5);
    const Place at = place_of_row(offsets, experts, rows, row, wide ? kFewRows : 16);
    const int e = at.e;
    wait_for_last();
    if (blk >= n / kBlock || (e < 0 && !zero_rest)) return;
    const int j = blk * kBlock + lane * 4;
    T* o = y + (int64_t)row * ldy + j;
    if (e < 0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = from_f<T>(0.f);
        return;
    }
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    // The parts of this lane's strip: from the CTA of its first k tile to that of its last.
    const int strips = n / few_columns(wide);
    const int64_t per = few_share((int64_t)at.tiles * strips * kt, ctas, kt, parts);
    const int64_t first = ((int64_t)at.tile * strips + j / few_columns(wide)) * kt;
    const int mine = (int)((first + kt - 1) / per - first / per) + 1;
#pragma unroll 4
    for (int s = 0; s < mine; ++s) {
        const float4 q = load_once(partial + ((int64_t)s * rows + row) * n + j);
        v[0] += q.x; v[1] += q.y; v[2] += q.z; v[3] += q.w;
    }
    had128_warp(v, lane);
    const float f = scale[row] * 0.08838834764831845f;      // 1 / sqrt(128)
    float sv[4];
    load4(svh + e * svh_stride + j, sv);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = v[i] * sv[i] * f;      // f last: f * sv may be below the normal numbers
    store4(o, v);
}

// What_e as binary16 [n][k].  A block decodes 128 columns x 64 rows at a time, a warp 16 of the columns: the block reads
// 8 tiles' words in a row, and a warp turns its 64 x 16 part in shared memory and writes whole 128-byte lines.
constexpr int DN = 128, DK = 64, DPAD = 72;            // row stride of the staged tile in halves
template <int K, int DEC>
__global__ void __launch_bounds__(256) decode_kernel(const uint32_t* __restrict__ trellis, const void* __restrict__ table,
                                                     const int64_t* __restrict__ offsets, int rows, int experts, int k, int n,
                                                     __half* __restrict__ out) {
    extern __shared__ __align__(16) uint8_t smem[];
    __half* stage = reinterpret_cast<__half*>(smem + table_bytes(DEC));
    load_table<DEC>(table, smem);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int nb = n / DN, kb = k / DK, per = nb * kb, tiles_n = n / 16;
    // Block l of expert e; seek() moves on to a busy expert's (one without rows is not decoded).
    struct At { int e, l; };
    int known_e = -1, known_n = 0;
    auto seek = [&](At& at) {
        for (;; ++at.e, at.l -= per) {
            while (at.l >= per) { at.l -= per; ++at.e; }
            if (at.e >= experts) return;
            if (at.e != known_e) {
                int lo;
                group_of(offsets, at.e, rows, lo, known_n);
                known_e = at.e;
            }
            if (known_n) return;
            at.l += (per - at.l + (int)gridDim.x - 1) / (int)gridDim.x * (int)gridDim.x;   // this CTA's first one beyond it
        }
    };
    TileWords<K> w[4];
    auto fetch = [&](const At& at) {
        if (at.e >= experts) return;
        const int n0 = at.l % nb, k0 = at.l / nb;
        const uint32_t* t = trellis + (((int64_t)at.e * (k / 16) + k0 * (DK / 16)) * tiles_n + n0 * (DN / 16) + warp) * 8 * K;
#pragma unroll
        for (int a = 0; a < 4; ++a) w[a].load(t + (int64_t)a * tiles_n * 8 * K, lane);
    };
    At at{0, (int)blockIdx.x};
    seek(at);
    fetch(at);
    __syncthreads();
    while (at.e < experts) {
        const int e = at.e, n0 = at.l % nb * DN, k0 = at.l / nb * DK;
#pragma unroll
        for (int a = 0; a < 4; ++a) {
            uint32_t f[4];
            decode_tile<K, DEC>(w[a], lane, smem, f);
            uint32_t* o = reinterpret_cast<uint32_t*>(stage + (warp * 16 + (lane >> 2)) * DPAD + a * 16 + 2 * (lane & 3));
            o[0] = f[0];
            o[4] = f[1];
            o[8 * DPAD / 2] = f[2];
            o[8 * DPAD / 2 + 4] = f[3];
        }
        at.l += gridDim.x;
        seek(at);
        fetch(at);                                      // under the other warps' decoding and the stores
        // Each warp's 16 columns are its own: they leave without the rest of the block.
        __syncwarp();
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            const int r = warp * 16 + p * 4 + (lane >> 3), c = (lane & 7) * 8;
            *reinterpret_cast<uint4*>(out + ((int64_t)e * n + n0 + r) * k + k0 + c) = *reinterpret_cast<const uint4*>(stage + r * DPAD + c);
        }
        __syncwarp();
    }
    wait_for_last();
}

// Three ways, for MCG (and E4M3) at 4 bits, us by the mean of rows an expert:
//   few: in registers for mma.sync, k split over CTAs; costs what the weights' decoding costs, once per 16 or 64 rows.
//   fused: in shared memory for the tensor core, once per 256 rows; a tile of 256 rows x 128 columns takes all of k, so 64
//     tiles leave more than half of the SMs idle.
//   decoded once to the workspace, then the product; reading and writing binary16, whatever the rows.
// 8 experts of 7168 x 4096:    8 rows 113 (144) / 152 (189) / 233 (277);  16 rows 207 (220) / 152 (189) / 233 (278);
//   256 rows  - / 222 (240) / 290 (336);  384 rows  - / 405 (438) / 345 (388).
// 8 of 2048 x 7168: 8 rows 64 (81) / 92 (112) / 124 (150);  256 rows  - / 135 (149) / 158 (181).
// One of 7168 x 2048 (16 tiles): 64 rows 31 (37) / 80 (98) / 58 (62);  128 rows 46 (58) / 80 (98) / 59 (63).
// Uneven experts have more row tiles than their mean says, so the fused way ends before 256.  A binary16 table leaves no room
// for its stages; 8 of 7168 x 4096 from such a table: few 295 / 307 / 334 / 375 us at 16 / 32 / 48 / 64 rows, decoded once
// 347 to 359.
enum Way { FEW, FUSED, ONCE };

Way way_of(const kq_trellis_product& p) {
    const int64_t busy = p.experts < p.rows ? p.experts : p.rows, tiles = p.n / 128 * busy;
    if (tiles <= 64) return p.rows <= 96 * busy ? FEW : ONCE;
    if (p.codebook == KQ_CB_LABELS) return p.rows <= 40 * busy ? FEW : ONCE;
    return p.rows <= 8 * busy ? FEW : p.rows <= 192 * busy ? FUSED : ONCE;
}

int64_t align128(int64_t v) { return (v + 127) & ~(int64_t)127; }

// The decode-once way holds at most this much of What, some experts at a time: all of 384 experts of 7168 x 4096 would be
// 22 GB.  (16 such experts a round; what one expert needs if that is more.)
constexpr int64_t kDecodedBytes = (int64_t)1 << 30;

struct Plan { Way way; bool wide; int parts, together; int64_t scale, rest, bytes; };    // together: experts decoded at a time

int few_ctas(const kq_trellis_product& p, int sms) { return sms * (p.codebook == KQ_CB_LABELS ? 1 : 2); }   // a table of 128 KB leaves room for one

Plan plan(const kq_trellis_product& p) {
    Plan l{};
    const int64_t busy = p.experts < p.rows ? p.experts : p.rows;
    l.way = way_of(p);
    l.wide = p.rows > 8 * busy;
    // Parts of a strip: what an even share of a single row tile makes on 148 SMs, within 256 MB (two at least).
    const int64_t kt = p.k / 16, strips = p.n / few_columns(l.wide), one = p.rows * p.n * 4;
    const int64_t even = strips * kt / few_ctas(p, 148), share = even > 32 ? even : 32, fit = ((int64_t)1 << 28) / one;
    const int64_t most = kt / share + 2;
    l.parts = (int)(most < fit ? most : fit < 2 ? 2 : fit);
    l.scale = align128(p.rows * p.k * 2);
    l.rest = l.scale + align128(p.rows * 4);
    const int64_t expert = p.k * p.n * 2, fill = kDecodedBytes / expert;
    l.together = (int)(fill < 1 ? 1 : fill < p.experts ? fill : p.experts);
    l.bytes = l.rest + (l.way == FEW ? (int64_t)l.parts * one : l.way == FUSED ? 0 : l.together * expert);
    return l;
}

int check_trellis(const kq_trellis_product& p, const char* what) {
    if (p.rows < 0 || p.rows > 0x7FFFFF00 || p.k <= 0 || p.n <= 0 || p.k % kBlock || p.n % kBlock || p.k > (1 << 24) ||
        p.n > (1 << 24) || p.experts <= 0 || p.experts > kMaxExperts || p.bits < 1 || p.bits > 8) {
        set_error("%s: need k and n multiples of 128, 1..1024 experts, 1..8 bits (rows=%lld k=%lld n=%lld experts=%lld bits=%d)", what,
                  (long long)p.rows, (long long)p.k, (long long)p.n, (long long)p.experts, p.bits);
        return KQ_ERR_ARG;
    }
    if (p.k > (int64_t(1) << 41) / p.n) { set_error("%s: one expert's matrix has more than 2^41 elements", what); return KQ_ERR_ARG; }
    if (p.experts > 1 && !p.offsets) { set_error("%s: several experts need offsets", what); return KQ_ERR_ARG; }
    if (p.dtype != KQ_BF16 && p.dtype != KQ_FP16) { set_error("%s: dtype must be KQ_BF16 or KQ_FP16", what); return KQ_ERR_ARG; }
    if (p.codebook != KQ_CB_MCG && p.codebook != KQ_CB_SQG && p.codebook != KQ_CB_LABELS) {
        set_error("%s: codebook must be KQ_CB_MCG, KQ_CB_SQG or KQ_CB_LABELS", what);
        return KQ_ERR_ARG;
    }
    if (p.rows > 1 && (p.ldx < p.k || p.ldy < p.n)) { set_error("%s: row strides too small", what); return KQ_ERR_ARG; }
    return KQ_OK;
}

template <int K, int DEC>
int launch_decode(const kq_trellis_product& p, int64_t first, int64_t experts, __half* out, cudaStream_t s) {
    constexpr int smem = table_bytes(DEC) + DN * DPAD * 2;
    cudaError_t e = cudaFuncSetAttribute(decode_kernel<K, DEC>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) { set_error("cudaFuncSetAttribute: %s", cudaGetErrorString(e)); return KQ_ERR_CUDA; }
    int sms;
    if (int rc = sm_count(&sms)) return rc;
    const int64_t items = (p.n / DN) * (p.k / DK) * experts;
    const int per_sm = DEC == DEC_F16 ? 1 : DEC == DEC_E4M3 ? 2 : 8;
    const int grid = (int)(items < (int64_t)sms * per_sm ? items : (int64_t)sms * per_sm);
    const uint32_t* trellis = reinterpret_cast<const uint32_t*>(p.trellis) + first * (p.k / 16) * (p.n / 16) * 8 * K;
    const int64_t* offsets = p.offsets ? p.offsets + first : nullptr;
    // The first range is decoded beside the rotation of x.  A later one takes the memory of the one before it, whose products
    // have to be done: an ordinary launch.
    if (!first)
        return launch_next(decode_kernel<K, DEC>, dim3((unsigned)grid), 256, smem, s, "decode_kernel", trellis, p.table, offsets,
                           (int)p.rows, (int)experts, (int)p.k, (int)p.n, out);
    decode_kernel<K, DEC><<<grid, 256, smem, s>>>(trellis, p.table, offsets, (int)p.rows, (int)experts, (int)p.k, (int)p.n, out);
    return check_launch("decode_kernel");
}

template <int K>
int launch_decode_k(const kq_trellis_product& p, int64_t first, int64_t experts, __half* out, cudaStream_t s) {
    if (p.codebook == KQ_CB_MCG) return launch_decode<K, DEC_MCG>(p, first, experts, out, s);
    if (p.codebook == KQ_CB_SQG) return launch_decode<K, DEC_E4M3>(p, first, experts, out, s);
    return launch_decode<K, DEC_F16>(p, first, experts, out, s);
}

// What of experts first .. first + experts - 1.
int decode_range(const kq_trellis_product& p, int64_t first, int64_t experts, __half* out, cudaStream_t s) {
    switch (p.bits) {
        case 1: return launch_decode_k<1>(p, first, experts, out, s);
        case 2: return launch_decode_k<2>(p, first, experts, out, s);
        case 3: return launch_decode_k<3>(p, first, experts, out, s);
        case 4: return launch_decode_k<4>(p, first, experts, out, s);
        case 5: return launch_decode_k<5>(p, first, experts, out, s);
        case 6: return launch_decode_k<6>(p, first, experts, out, s);
        case 7: return launch_decode_k<7>(p, first, experts, out, s);
        default: return launch_decode_k<8>(p, first, experts, out, s);
    }
}

// Few rows: more warps a row, for its latency; many: enough rows an SM as it is.
template <typename T>
int rotate_in(const kq_trellis_product& p, __half* xr, float* scale, cudaStream_t s) {
    auto run = [&](auto kernel, int threads) {
        kernel<<<(unsigned)p.rows, threads, 0, s>>>(static_cast<const T*>(p.x), p.ldx, reinterpret_cast<const __half*>(p.suh),
                                                    p.suh_stride_e, p.offsets, (int)p.rows, (int)p.experts, (int)p.k, xr, scale);
    };
    if (p.rows <= 256) run(rotate_in_kernel<T, 16>, 512);
    else run(rotate_in_kernel<T, 4>, 128);
    return check_launch("rotate_in_kernel");
}

}  // namespace
}  // namespace kq

extern "C" size_t kq_trellis_linear_workspace_bytes(const kq_trellis_product* p) {
    if (!p || kq::check_trellis(*p, "kq_trellis_linear_workspace_bytes") || p->rows == 0) return 0;
    return (size_t)kq::plan(*p).bytes;
}

extern "C" int kq_trellis_linear(const kq_trellis_product* pp, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace kq;
    const char* what = "kq_trellis_linear";
    if (!pp) { set_error("%s: null pointer", what); return KQ_ERR_ARG; }
    const kq_trellis_product& p = *pp;
    if (int rc = check_trellis(p, what)) return rc;
    if (p.rows == 0) return KQ_OK;
    if (!p.x || !p.trellis || !p.suh || !p.svh || !p.y || (p.codebook != KQ_CB_MCG && !p.table)) {
        set_error("%s: null pointer", what);
        return KQ_ERR_ARG;
    }
    if (((uintptr_t)p.trellis & 15) || ((uintptr_t)p.table & 15) || (((uintptr_t)p.x | (uintptr_t)p.y | (uintptr_t)p.suh | (uintptr_t)p.svh) & 1)) {
        set_error("%s: trellis and table need 16-byte alignment", what);
        return KQ_ERR_ALIGN;
    }
    int* err;
    const Plan l = plan(p);
    if (!workspace || workspace_bytes < (size_t)l.bytes) { set_error("%s: workspace too small", what); return KQ_ERR_WORKSPACE; }
    if ((uintptr_t)workspace & 127) { set_error("%s: workspace must be 128-byte aligned", what); return KQ_ERR_ALIGN; }
    if (int rc = wait_error_word(&err, what)) return rc;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    __half* xr = reinterpret_cast<__half*>(ws);
    float* scale = reinterpret_cast<float*>(ws + l.scale);
    const bool bf16 = p.dtype == KQ_BF16;
    if (int rc = bf16 ? rotate_in<__nv_bfloat16>(p, xr, scale, s) : rotate_in<__half>(p, xr, scale, s)) return rc;
    if (l.way == FEW) {
        int sms;
        if (int rc = sm_count(&sms)) return rc;
        float* partial = reinterpret_cast<float*>(ws + l.rest);
        const FewTrellis f{reinterpret_cast<const uint32_t*>(p.trellis), p.table, p.offsets, reinterpret_cast<const uint16_t*>(xr), partial,
                           (int)p.rows, (int)p.experts, (int)p.k, (int)p.n, l.parts};
        const int dec = p.codebook == KQ_CB_MCG ? DEC_MCG : p.codebook == KQ_CB_SQG ? DEC_E4M3 : DEC_F16;
        int rc = p.bits <= 2 ? few_trellis_k12(f, p.bits, dec, l.wide, s) : p.bits <= 4 ? few_trellis_k34(f, p.bits, dec, l.wide, s)
               : p.bits <= 6 ? few_trellis_k56(f, p.bits, dec, l.wide, s) : few_trellis_k78(f, p.bits, dec, l.wide, s);
        if (rc) return rc;
        const dim3 grid((unsigned)p.rows, (unsigned)((p.n / kBlock + 7) / 8));
        const __half* svh = reinterpret_cast<const __half*>(p.svh);
        auto out = [&](auto* y) {
            return launch_next(rotate_out_kernel<std::remove_pointer_t<decltype(y)>>, grid, 256, 0, s, "rotate_out_kernel", partial, l.parts,
                               few_ctas(p, sms), (int)(p.k / 16), l.wide, scale, svh, p.svh_stride_e, p.offsets, (int)p.rows,
                               (int)p.experts, (int)p.n, y, p.ldy, p.zero_rest != 0);
        };
        return bf16 ? out(static_cast<__nv_bfloat16*>(p.y)) : out(static_cast<__half*>(p.y));
    }
    if (l.way == FUSED) {
        TrellisRows r{reinterpret_cast<const uint32_t*>(p.trellis), p.table, p.offsets, reinterpret_cast<const uint16_t*>(xr),
                      reinterpret_cast<const __half*>(p.svh), scale, p.y, p.svh_stride_e, p.ldy, (int)p.rows, (int)p.experts, (int)p.k,
                      (int)p.n, err, bf16, ((uintptr_t)p.svh & 15) == 0 && p.svh_stride_e % 8 == 0,
                      ((uintptr_t)p.y & 15) == 0 && p.ldy % 8 == 0, p.zero_rest != 0};
        const int dec = p.codebook == KQ_CB_MCG ? DEC_MCG : DEC_E4M3;
        return p.bits <= 2 ? rows_trellis_k12(r, p.bits, dec, s) : p.bits <= 4 ? rows_trellis_k34(r, p.bits, dec, s)
             : p.bits <= 6 ? rows_trellis_k56(r, p.bits, dec, s) : rows_trellis_k78(r, p.bits, dec, s);
    }
    __half* w = reinterpret_cast<__half*>(ws + l.rest);
    for (int64_t e = 0; e < p.experts; e += l.together) {
        const int64_t some = p.experts - e < l.together ? p.experts - e : l.together;
        if (int rc = decode_range(p, e, some, w, s)) return rc;
        if (int rc = rows_product_rotated(reinterpret_cast<const uint16_t*>(xr), reinterpret_cast<const uint16_t*>(w), p.offsets, p.rows,
                                          p.k, p.n, p.experts, e, some, p.svh, p.svh_stride_e, scale, p.y, p.ldy, bf16,
                                          p.zero_rest != 0, err, s))
            return rc;
    }
    return KQ_OK;
}
