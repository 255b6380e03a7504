// Host helpers of the tensor-core products (bcjr_mm.cuh): operand maps and
// the size of a persistent grid.
#include "bcjr_mm.cuh"

#include "bcjr_kernels.h"

namespace bcjr {
namespace mm {

namespace {
typedef CUresult (*EncodeFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *,
                             const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                             const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                             CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// The driver's encoder, found through the runtime (the library does not link
// libcuda, so it loads on machines without a driver).
EncodeFn encoder() {
    static std::atomic<EncodeFn> found{nullptr};
    EncodeFn fn = found.load(std::memory_order_relaxed);
    if (!fn) {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            return nullptr;
        fn = reinterpret_cast<EncodeFn>(p);
        found.store(fn, std::memory_order_relaxed);
    }
    return fn;
}
}  // namespace

bool make_map(CUtensorMap *m, int kind, int rank, const void *base, const unsigned long long *dims,
              const unsigned long long *strides, const unsigned *box) {
    const EncodeFn fn = encoder();
    if (!fn || rank < 2 || rank > 3) return false;
    const CUtensorMapDataType type = kind == kBF16   ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                     : kind == kF16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                    : CU_TENSOR_MAP_DATA_TYPE_UINT8;
    cuuint64_t d[3], s[2];
    cuuint32_t b[3], step[3] = {1, 1, 1};
    for (int i = 0; i < rank; ++i) {
        d[i] = dims[i];
        b[i] = box[i];
        if (i + 1 < rank) s[i] = strides[i];
    }
    return fn(m, type, cuuint32_t(rank), const_cast<void *>(base), d, s, b, step,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int grid_sms(int *device) {
    static std::atomic<int> count[kMaxDevices];       // SMs, -1: not sm_100, 0: not asked yet
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return 0;
    // The map encoder wants a current context, which a thread that has made no
    // runtime call on the device yet (autograd's) does not have.
    if (cudaSetDevice(dev) != cudaSuccess) return 0;
    int n = count[dev].load(std::memory_order_relaxed);
    if (n == 0) {
        int sms = 0, major = 0;
        if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess ||
            cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev) != cudaSuccess)
            return 0;
        n = major == 10 && sms > 0 ? sms : -1;
        count[dev].store(n, std::memory_order_relaxed);
    }
    if (n < 0) return 0;
    *device = dev;
    n -= reserved_sms();
    return n > 0 ? n : 1;
}

}  // namespace mm
}  // namespace bcjr
