// Products of many rows with tiles of 7 and 8 bits (one source file for two rates: they compile side by side).
#include "kq_trellis_rows.cuh"

int kq::rows_trellis_k78(const TrellisRows& p, int bits, int dec, cudaStream_t s) {
    return bits == 7 ? rows_trellis<7>(p, dec, s) : rows_trellis<8>(p, dec, s);
}
