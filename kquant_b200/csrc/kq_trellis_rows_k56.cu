// Products of many rows with tiles of 5 and 6 bits (one source file for two rates: they compile side by side).
#include "kq_trellis_rows.cuh"

int kq::rows_trellis_k56(const TrellisRows& p, int bits, int dec, cudaStream_t s) {
    return bits == 5 ? rows_trellis<5>(p, dec, s) : rows_trellis<6>(p, dec, s);
}
