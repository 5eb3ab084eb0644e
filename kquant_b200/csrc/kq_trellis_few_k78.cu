// Products of few rows with tiles of 7 and 8 bits (one source file for two rates: they compile side by side).
#include "kq_trellis_few.cuh"

int kq::few_trellis_k78(const FewTrellis& p, int bits, int dec, bool wide, cudaStream_t s) {
    return bits == 7 ? few_trellis<7>(p, dec, wide, s) : few_trellis<8>(p, dec, wide, s);
}
