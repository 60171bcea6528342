// paged_attention.cu -- attention over a paged 8-bit cache.
#include "launch.cuh"
#include "paged.cuh"

namespace cvattn {
namespace paged {

// A warp takes one row: a lane scores a position at a time, then carries two dims of the output.
template <int F>
__global__ void __launch_bounds__(128) paged_row_kernel(const __grid_constant__ cvattn_paged_attention_params p, int* status) {
    griddep_wait();
    __shared__ float qs[4][kD];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, s = blockIdx.y;
    const int item = blockIdx.x * 4 + warp, i = item / p.n_q_heads, h = item % p.n_q_heads;
    if (i >= p.max_q) return;
    const int kvh = h / (p.n_q_heads / p.pool.n_heads), blocks = p.pool.page_size / kBlock;
    int L = p.kv_len[s], n = p.n_q ? p.n_q[s] : p.max_q;
    if (L < 0 || L > p.max_kv_len || n < 0 || n > p.max_q) {
        if (item == 0 && lane == 0) record_status(status, kStatusBadLength);
        L = n = 0;
    }
    const int end = i < n ? min(L, L - n + i + 1) : 0;
    const float* q = p.q + s * p.q_nb_seq + i * p.q_nb_tok + h * kD;
    qs[warp][lane] = q[lane] * p.scale;
    qs[warp][lane + 32] = q[lane + 32] * p.scale;
    __syncwarp();
    float m = -INFINITY, l = 0.0f, o0 = 0.0f, o1 = 0.0f;
    for (int j0 = 0; j0 < end; j0 += 32) {
        const int j = j0 + lane;
        int page = -1;
        float x = -INFINITY, vs = 0.0f;
        const uint8_t* vc = nullptr;
        if (j < end) {
            page = page_of(p.table + s * p.table_nb_seq, j / p.pool.page_size, p.pool.n_pages);
            if (page < 0) {
                record_status(status, kStatusBadPage);
            } else {
                const int in = kvh * blocks + j % p.pool.page_size / kBlock, t = j % kBlock;
                const uint8_t* kc = static_cast<const uint8_t*>(p.pool.k) + page * p.pool.nb_page + (int64_t)in * kBlockBytes + t * kD;
                vc = static_cast<const uint8_t*>(p.pool.v) + page * p.pool.nb_page + (int64_t)in * kBlockBytes;
                vs = p.pool.v_scale[page * p.pool.nb_scale + in];
                float dot = 0.0f;
                for (int d = 0; d < kD; ++d) dot = fmaf(code_value<F>(kc[d]), qs[warp][d], dot);
                x = dot * p.pool.k_scale[page * p.pool.nb_scale + in];
            }
        }
        float top = x;
        for (int w = 16; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
        top = fmaxf(top, m);
        if (top == -INFINITY) continue;
        const float f = expf(m - top), e = expf(x - top);
        float sum = e;
        for (int w = 16; w > 0; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
        l = fmaf(l, f, sum);
        m = top;
        o0 *= f;
        o1 *= f;
        for (int k = 0; k < min(32, end - j0); ++k) {
            const float w = __shfl_sync(0xffffffffu, e * vs, k);
            const uint8_t* c = reinterpret_cast<const uint8_t*>(__shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(vc), k));
            if (c == nullptr) continue;
            o0 = fmaf(w, code_value<F>(c[v_place((j0 + k) % kBlock, lane)]), o0);
            o1 = fmaf(w, code_value<F>(c[v_place((j0 + k) % kBlock, lane + 32)]), o1);
        }
    }
    float* out = p.out + s * p.out_nb_seq + i * p.out_nb_tok + h * kD;
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
    out[lane] = o0 * inv;
    out[lane + 32] = o1 * inv;
    if (p.lse && lane == 0) p.lse[((int64_t)s * p.max_q + i) * p.n_q_heads + h] = l > 0.0f ? m + logf(l) : -INFINITY;
}

}  // namespace paged

size_t paged_attention_workspace_bytes(int n_seq, int max_q, int max_kv_len, int n_q_heads, int n_kv_heads) { return 0; }

cudaError_t launch_paged_attention(cudaStream_t stream, const cvattn_paged_attention_params& p, int* status) {
    using namespace paged;
    const dim3 grid((unsigned)(((int64_t)p.max_q * p.n_q_heads + 3) / 4), (unsigned)p.n_seq);
    auto* fn = p.pool.format == kI8 ? paged_row_kernel<kI8> : paged_row_kernel<kE4M3>;
    return launch_overlapped(fn, grid, 128, 0, stream, p, status);
}

}  // namespace cvattn
