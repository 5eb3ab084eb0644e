// Products of many rows with tiles of 1 and 2 bits (one source file for two rates: they compile side by side).
#include "kq_trellis_rows.cuh"

int kq::rows_trellis_k12(const TrellisRows& p, int bits, int dec, cudaStream_t s) {
    return bits == 1 ? rows_trellis<1>(p, dec, s) : rows_trellis<2>(p, dec, s);
}
