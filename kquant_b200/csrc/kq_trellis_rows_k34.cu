// Products of many rows with tiles of 3 and 4 bits (one source file for two rates: they compile side by side).
#include "kq_trellis_rows.cuh"

int kq::rows_trellis_k34(const TrellisRows& p, int bits, int dec, cudaStream_t s) {
    return bits == 3 ? rows_trellis<3>(p, dec, s) : rows_trellis<4>(p, dec, s);
}
