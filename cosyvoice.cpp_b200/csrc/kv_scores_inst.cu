// kv_scores_inst.cu -- the attention score MMA kernels of one K type (CVATTN_KT).
#include <atomic>

#include "kv_scores.cuh"

namespace cvattn {
namespace kvscore {

template <int KT, int NT>
static cudaError_t run(cudaStream_t stream, const Args& a) {
    const auto fn = scores_mma_kernel<KT, NT>;
    constexpr int smem = Smem<KT, NT>::bytes, keys = Smem<KT, NT>::kKeys;
    static std::atomic<bool> allowed[64];  // dynamic shared memory granted, per device
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !allowed[dev].load(std::memory_order_relaxed)) {
        e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return e;
        if (dev < 64) allowed[dev].store(true, std::memory_order_relaxed);
    }
    return launch_overlapped(fn, dim3((unsigned)((a.max_kv_len + keys - 1) / keys), (unsigned)a.Hkv, (unsigned)a.n_seq), kThreads, smem, stream, a);
}

template <>
cudaError_t launch_mma_for_k<CVATTN_KT>(cudaStream_t stream, const Args& a) {
    // 32 keys a warp share more of each Q fragment, 16 keys fill more SMs.  us of 16 | 32 keys a warp, 14 / 2 heads, Q8_0 and f16: 64
    // tiles of 128 keys, 28 rows 4.9 | 5.7 and 4.3 | 4.6; 256 tiles, 28 rows 6.4 | 5.7 and 5.0 | 4.6, 112 rows 9.8 | 8.7 and 7.9 | 7.4;
    // 512 tiles, 28 rows 11.6 | 7.7 and 8.6 | 5.7.
    return (int64_t)a.n_seq * a.Hkv * ((a.max_kv_len + 127) / 128) > 148 ? run<CVATTN_KT, 4>(stream, a) : run<CVATTN_KT, 2>(stream, a);
}

}  // namespace kvscore
}  // namespace cvattn
