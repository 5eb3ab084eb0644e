// Products of few rows with tiles of 1 and 2 bits (one source file for two rates: they compile side by side).
#include "kq_trellis_few.cuh"

int kq::few_trellis_k12(const FewTrellis& p, int bits, int dec, bool wide, cudaStream_t s) {
    return bits == 1 ? few_trellis<1>(p, dec, wide, s) : few_trellis<2>(p, dec, wide, s);
}
