// Error state and device queries shared by the C ABI.
#include <cstdarg>
#include <cstdio>
#include "kq_umma.cuh"

namespace kq {

static thread_local char g_err[512] = "";

void set_error(const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_err, sizeof(g_err), fmt, ap);
    va_end(ap);
}

const char* last_error() { return g_err; }

int sm_count(int* out) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(out, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) {
        set_error("device query: %s", cudaGetErrorString(e));
        return KQ_ERR_CUDA;
    }
    return KQ_OK;
}

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    if (!fn) {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
    }
    return fn;
}

int encode_tiles(CUtensorMap* map, CUtensorMapDataType type, int rank, const void* base, const int64_t* dims,
                 const int64_t* strides, const int* box, const char* what) {
    auto fn = encode_fn();
    if (!fn) { set_error("%s: cuTensorMapEncodeTiled unavailable", what); return KQ_ERR_CUDA; }
    cuuint64_t d[5], st[4];
    cuuint32_t b[5], es[5];
    for (int i = 0; i < rank; ++i) {
        d[i] = (cuuint64_t)dims[i];
        b[i] = (cuuint32_t)box[i];
        es[i] = 1;
        if (i) st[i - 1] = (cuuint64_t)strides[i - 1];
    }
    CUresult r = fn(map, type, (cuuint32_t)rank, const_cast<void*>(base), d, st, b, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) { set_error("%s: cuTensorMapEncodeTiled failed (%d)", what, (int)r); return KQ_ERR_CUDA; }
    return KQ_OK;
}

}  // namespace kq
