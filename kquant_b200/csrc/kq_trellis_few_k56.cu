// Products of few rows with tiles of 5 and 6 bits (one source file for two rates: they compile side by side).
#include "kq_trellis_few.cuh"

int kq::few_trellis_k56(const FewTrellis& p, int bits, int dec, bool wide, cudaStream_t s) {
    return bits == 5 ? few_trellis<5>(p, dec, wide, s) : few_trellis<6>(p, dec, wide, s);
}
