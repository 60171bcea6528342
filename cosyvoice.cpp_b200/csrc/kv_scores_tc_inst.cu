// kv_scores_tc_inst.cu -- the tcgen05 attention score kernel of one K type (CVATTN_KT).
#include <atomic>

#include "kv_scores_tc.cuh"

namespace cvattn {
namespace kvscore {

template <>
cudaError_t launch_tc_for_k<CVATTN_KT>(cudaStream_t stream, const TcArgs& a) {
    const auto fn = scores_tc_kernel<CVATTN_KT>;
    constexpr int smem = TcShape<CVATTN_KT>::kBytes;
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

}  // namespace kvscore
}  // namespace cvattn
