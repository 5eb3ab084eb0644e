// Decoding of packed trellis tiles.
//
// State i of a tile is the 16-bit window of its cyclic bit stream
// that ends with symbol i (kq_unpack_trellis_states).  Lane m of a warp owns
// symbols 8m .. 8m+7: its eight windows lie in 7K + 16 consecutive bits, three
// (K > 6: four) 32-bit words.  Trellis position 8m + s is row 2(m%4) + (s&1) +
// 8((s>>1)&1), column m/4 + 8(s>>2) of the tile, so neighbouring symbols are
// neighbouring rows: a packed pair along the contraction axis.
// Labels: MCG is computed (a multiply, a logic op, half an add); E4M3 and
// binary16 tables are looked up in shared memory, where 32 random lookups
// take 3.5 cycles (13.1 million for the 3.76 million load instructions of 8
// experts of 7168 x 2048 at 3 bits, one row each).
#pragma once
#include "kq_expert.cuh"

namespace kq {

// The kernels of one call follow one another by programmatic launch: a kernel lets the next one start (its tables, its words of
// the payload, its first tiles), which waits for everything before it where it needs it, and at its end at the latest, so that
// a kernel's end is the end of all before it.
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_last() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <typename... P, typename... A>
int launch_next(void (*kernel)(P...), dim3 grid, int threads, int smem, cudaStream_t s, const char* what, const A&... args) {
    cudaLaunchConfig_t c{};
    c.gridDim = grid;
    c.blockDim = dim3((unsigned)threads);
    c.dynamicSmemBytes = (size_t)smem;
    c.stream = s;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    c.attrs = &at;
    c.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&c, kernel, static_cast<P>(args)...);
    if (e != cudaSuccess) { set_error("%s: %s", what, cudaGetErrorString(e)); return KQ_ERR_CUDA; }
    return check_launch(what);
}

enum { DEC_MCG, DEC_E4M3, DEC_F16 };
constexpr int kBlock = 128;    // channels of a Hadamard block

__host__ __device__ constexpr int table_bytes(int dec) { return dec == DEC_MCG ? 0 : dec == DEC_E4M3 ? 65536 : 131072; }

// Whole block: the label table into shared memory.
template <int DEC>
__device__ __forceinline__ void load_table(const void* table, uint8_t* smem) {
    if constexpr (DEC != DEC_MCG) {
        const uint4* src = static_cast<const uint4*>(table);
        for (int i = threadIdx.x; i < table_bytes(DEC) / 16; i += blockDim.x) reinterpret_cast<uint4*>(smem)[i] = __ldg(src + i);
    }
}

// Labels of two states as packed binary16.
template <int DEC>
__device__ __forceinline__ uint32_t label_pair(uint32_t s0, uint32_t s1, const uint8_t* table) {
    if constexpr (DEC == DEC_MCG) {
        const uint32_t y0 = ((s0 * 0xCBAC1FEDu) & 0x8fff8fffu) ^ 0x3b603b60u;
        const uint32_t y1 = ((s1 * 0xCBAC1FEDu) & 0x8fff8fffu) ^ 0x3b603b60u;
        const __half2 h0 = *reinterpret_cast<const __half2*>(&y0), h1 = *reinterpret_cast<const __half2*>(&y1);
        const __half2 v = __halves2half2(__hadd(__low2half(h0), __high2half(h0)), __hadd(__low2half(h1), __high2half(h1)));
        return *reinterpret_cast<const uint32_t*>(&v);
    } else if constexpr (DEC == DEC_E4M3) {
        const uint16_t b = (uint16_t)(table[s0] | (table[s1] << 8));
        uint32_t v;
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(v) : "h"(b));
        return v;
    } else {
        const uint16_t* t = reinterpret_cast<const uint16_t*>(table);
        return (uint32_t)t[s0] | ((uint32_t)t[s1] << 16);
    }
}

// A tile's words, held by the warp: lane l has words l and (K > 4) l + 32, each 32 bits of the stream, first bit on top.
template <int K>
struct TileWords {
    uint32_t w[K > 4 ? 2 : 1];
    __device__ __forceinline__ void load(const uint32_t* tile, int lane) {
        if (K >= 4 || lane < 8 * K) w[0] = __ldg(tile + lane);
        if constexpr (K > 4)
            if (lane + 32 < 8 * K) w[1] = __ldg(tile + 32 + lane);
    }
    __device__ __forceinline__ uint32_t at(int i) const {       // word i mod 8K, i in -8K .. 8K
        i = i < 0 ? i + 8 * K : i >= 8 * K ? i - 8 * K : i;
        const uint32_t a = __shfl_sync(0xFFFFFFFFu, w[0], i & 31);
        if constexpr (K > 4) {
            const uint32_t b = __shfl_sync(0xFFFFFFFFu, w[1], i & 31);
            return i >= 32 ? b : a;
        }
        return a;
    }
};

// The four fragment pairs of this lane: rows (2q, 2q+1) and (2q+8, 2q+9) of column m/4, then of column m/4 + 8.
template <int K, int DEC>
__device__ __forceinline__ void decode_tile(const TileWords<K>& t, int lane, const uint8_t* table, uint32_t (&frag)[4]) {
    const int end = 8 * K * (lane + 1), wi = end >> 5, off = end & 31;
    const uint32_t c = t.at(wi), b = t.at(wi - 1), a = t.at(wi - 2);
    // Stream bits [end-32, end), the 32 before them, and (K > 6) the 32 before those.
    const uint32_t w0 = __funnelshift_l(c, b, off), w1 = __funnelshift_l(b, a, off);
    uint32_t w2 = 0;
    if constexpr (K > 6) w2 = __funnelshift_l(a, t.at(wi - 3), off);
    // A window inside one word is shifted to its top and down again: the first shift runs as a multiply beside the ALU,
    // which is the busy pipe (a mask would be a second ALU operation).
    uint32_t s[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int sh = (7 - i) * K;
        if (sh <= 16) s[i] = (w0 << (16 - sh)) >> 16;
        else if (sh < 32) s[i] = __funnelshift_r(w0, w1, sh) & 0xFFFFu;
        else if (sh <= 48) s[i] = (w1 << (48 - sh)) >> 16;
        else s[i] = __funnelshift_r(w1, w2, sh - 32) & 0xFFFFu;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) frag[i] = label_pair<DEC>(s[2 * i], s[2 * i + 1], table);
}

// Rows product of few rows.  The work is row tiles x strips of columns x k tiles, in that order; CTA c takes the k tiles
// c * per .. of it, so a strip's sums come in up to `parts` parts, counted from the CTA that holds its first k tile:
// partial [parts][rows][n].
struct FewTrellis {
    const uint32_t* trellis;
    const void* table;
    const int64_t* offsets;
    const uint16_t* xr;        // [rows][k] binary16
    float* partial;
    int rows, experts, k, n, parts;
};

// k tiles of a CTA: an even share of `work` for `ctas`, at least 32 (a step of every warp or more), and enough that no strip is in
// more than `parts` parts.
__host__ __device__ inline int64_t few_share(int64_t work, int ctas, int kt, int parts) {
    const int64_t even = (work + ctas - 1) / ctas, least = (kt + parts - 2) / (parts - 1);
    const int64_t m = even > least ? even : least;
    return m > 32 ? m : 32;
}

constexpr int kFewRows = 64;   // rows of the larger row tile; the smaller one has 16
constexpr int few_columns(bool wide) { return wide ? 32 : 64; }     // of a strip

// Launches for the rates of one source file each; `wide`: 64 rows a tile, else 16.
int few_trellis_k12(const FewTrellis& p, int bits, int dec, bool wide, cudaStream_t s);
int few_trellis_k34(const FewTrellis& p, int bits, int dec, bool wide, cudaStream_t s);
int few_trellis_k56(const FewTrellis& p, int bits, int dec, bool wide, cudaStream_t s);
int few_trellis_k78(const FewTrellis& p, int bits, int dec, bool wide, cudaStream_t s);

// Rows product of many rows; y bf16 or fp16.
struct TrellisRows {
    const uint32_t* trellis;
    const void* table;
    const int64_t* offsets;
    const uint16_t* xr;        // [rows][k] binary16
    const __half* svh;
    const float* row_scale;
    void* y;
    int64_t svh_stride, ldy;
    int rows, experts, k, n;
    int* err;
    bool bf16, vec_svh, vec_y, zero_rest;
};

// DEC_MCG and DEC_E4M3: a binary16 table and the stages do not fit in shared memory together.
int rows_trellis_k12(const TrellisRows& p, int bits, int dec, cudaStream_t s);
int rows_trellis_k34(const TrellisRows& p, int bits, int dec, cudaStream_t s);
int rows_trellis_k56(const TrellisRows& p, int bits, int dec, cudaStream_t s);
int rows_trellis_k78(const TrellisRows& p, int bits, int dec, cudaStream_t s);

}  // namespace kq
