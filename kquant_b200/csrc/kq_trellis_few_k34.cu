// Products of few rows with tiles of 3 and 4 bits (one source file for two rates: they compile side by side).
#include "kq_trellis_few.cuh"

int kq::few_trellis_k34(const FewTrellis& p, int bits, int dec, bool wide, cudaStream_t s) {
    return bits == 3 ? few_trellis<3>(p, dec, wide, s) : few_trellis<4>(p, dec, wide, s);
}
