// tree_tc_inst.cu -- the tcgen05 tree attention kernels of one K type (CVATTN_KT).
#include <atomic>

#include "tree_tc.cuh"

namespace cvattn {
namespace tree {

template <int KT, int VT>
static cudaError_t run(cudaStream_t stream, const TcArgs& a) {
    const auto fn = tree_tc_kernel<KT, VT>;
    constexpr int smem = TcShape<KT, VT>::kBytes;
    static std::atomic<bool> allowed[64];  // dynamic shared memory granted, per device
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !allowed[dev].load(std::memory_order_relaxed)) {
        e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return e;
        if (dev < 64) allowed[dev].store(true, std::memory_order_relaxed);
    }
    return launch_overlapped(fn, dim3((unsigned)a.grid), kTcThreads, smem, stream, a);
}

template <>
cudaError_t launch_tc_for_k<CVATTN_KT>(cudaStream_t stream, const TcArgs& a) {
    switch (a.a.v_type) {
    case kF16: return run<CVATTN_KT, kF16>(stream, a);
    case kQ4_0: return run<CVATTN_KT, kQ4_0>(stream, a);
    case kQ4_1: return run<CVATTN_KT, kQ4_1>(stream, a);
    case kQ5_0: return run<CVATTN_KT, kQ5_0>(stream, a);
    case kQ5_1: return run<CVATTN_KT, kQ5_1>(stream, a);
    case kQ8_0: return run<CVATTN_KT, kQ8_0>(stream, a);
    default: return cudaErrorInvalidValue;
    }
}

}  // namespace tree
}  // namespace cvattn
