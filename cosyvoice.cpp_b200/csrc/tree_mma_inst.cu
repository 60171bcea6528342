// tree_mma_inst.cu -- the tree attention MMA kernels of one K type (CVATTN_KT).
#include <atomic>

#include "tree_mma.cuh"

namespace cvattn {
namespace tree {

template <int KT, int VT>
static cudaError_t run(cudaStream_t stream, const Args& a, const Shape& sh) {
    const auto fn = tree_mma_kernel<KT, VT>;
    const int smem = Smem(KT, VT, sh.stages).total;
    static std::atomic<int> allowed[64];  // dynamic shared memory granted so far, per device
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || allowed[dev].load(std::memory_order_relaxed) < smem) {
        e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return e;
        if (dev < 64) allowed[dev].store(smem, std::memory_order_relaxed);
    }
    const dim3 grid((unsigned)a.n_splits, (unsigned)(a.Hkv * sh.row_groups), (unsigned)a.n_seq);
    return launch_overlapped(fn, grid, kWarps * 32, smem, stream, a, sh);
}

template <>
cudaError_t launch_mma_for_k<CVATTN_KT>(cudaStream_t stream, const Args& a, const Shape& sh) {
    switch (a.v_type) {
    case kF16: return run<CVATTN_KT, kF16>(stream, a, sh);
    case kQ4_0: return run<CVATTN_KT, kQ4_0>(stream, a, sh);
    case kQ4_1: return run<CVATTN_KT, kQ4_1>(stream, a, sh);
    case kQ5_0: return run<CVATTN_KT, kQ5_0>(stream, a, sh);
    case kQ5_1: return run<CVATTN_KT, kQ5_1>(stream, a, sh);
    case kQ8_0: return run<CVATTN_KT, kQ8_0>(stream, a, sh);
    default: return cudaErrorInvalidValue;
    }
}

}  // namespace tree
}  // namespace cvattn
