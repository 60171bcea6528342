// kv_scores.cu -- cvattn_kv_scores: the attention weight of each cached position.
#include "kv_scores_tc.cuh"

namespace cvattn {
namespace kvscore {

constexpr int kTile = 64;   // keys per CTA
constexpr int kRows = 32;   // (token, head) rows at a time
constexpr int kPad = kD + 4;

// f32 caches, on the CUDA cores: a thread owns 4 rows x 4 keys of a 32 x 64 tile.  Bound by
// FMAs, shared-memory reads and the loads of a tile, an element at a time (8 sequences of 8192,
// 64 rows of 14 heads: 381 us, from f16 the tensor cores' kernel 40; 64 of up to 4096, 4 rows:
// 146 us, from Q8_0 20).
__global__ void __launch_bounds__(128) scores_f32_kernel(const __grid_constant__ Args a) {
    __shared__ float4 qs4[kRows][kPad / 4], ks4[kTile][kPad / 4];
    __shared__ float ls[kRows], red[8][kTile];
    __shared__ int far[kRows];  // keys that the row sees
    const int tid = threadIdx.x, tr = tid >> 4, tc = tid & 15;
    const int s = blockIdx.z, kvh = blockIdx.y, p0 = blockIdx.x * kTile;
    int L, n;
    griddep_wait();
    if (!lens_of(a, s, L, n, tid == 0) || p0 >= L) return;
    const int count = min(kTile, L - p0);
    const uint8_t* kb = a.k_seq_ptrs ? reinterpret_cast<const uint8_t*>(a.k_seq_ptrs[s]) : a.k + (int64_t)s * a.k_nb2;
    float* ks = reinterpret_cast<float*>(ks4);
    float* qs = reinterpret_cast<float*>(qs4);
    const int gb = group_bytes(a.k_type);
    {
        const int key = tid >> 1, half = tid & 1;
        float* d = ks + key * kPad + half * 32;
        const uint8_t* g = kb + (int64_t)(p0 + key) * a.k_nb1 + (int64_t)(kvh * 2 + half) * gb;
        for (int e = 0; e < 32; ++e) d[e] = key < count ? dequant_elem_rt(a.k_type, g, e) : 0.0f;
    }
    float sum[4] = {};
    const int total = n * a.G;
    for (int r0 = 0; r0 < total; r0 += kRows) {
        __syncthreads();
        for (int i = tid; i < kRows; i += 128) {
            const int r = r0 + i, t = r / a.G, h = kvh * a.G + r % a.G;
            ls[i] = 0.0f;
            far[i] = 0;
            if (r < total) {
                const int at = a.rows ? a.rows[(int64_t)s * a.max_rows + t] : t;
                if (at < 0 || at >= a.n_q_rows) {
                    record_status(a.status, kStatusBadPosition);
                } else {
                    const float v = a.lse[((int64_t)s * a.n_q_rows + at) * a.Hq + h];
                    ls[i] = v * 1.4426950408889634f;
                    far[i] = v == -INFINITY ? 0 : L - n + t + 1;
                }
            }
        }
        __syncthreads();
        for (int i = tid; i < kRows * kD; i += 128) {
            const int r = r0 + i / kD, d = i % kD;
            float v = 0.0f;
            if (far[i / kD] > 0) {
                const int t = r / a.G, at = a.rows ? a.rows[(int64_t)s * a.max_rows + t] : t;
                v = a.q[(int64_t)s * a.q_nb_seq + (int64_t)at * a.q_nb_node + (kvh * a.G + r % a.G) * kD + d];
            }
            qs[(i / kD) * kPad + d] = v * a.scale_log2;
        }
        __syncthreads();
        float sc[4][4] = {};
#pragma unroll 4
        for (int d = 0; d < kD / 4; ++d) {
            float4 kk[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) kk[j] = ks4[tc + 16 * j][d];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float4 qq = qs4[tr * 4 + i][d];
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    sc[i][j] = fmaf(qq.x, kk[j].x, fmaf(qq.y, kk[j].y, fmaf(qq.z, kk[j].z, fmaf(qq.w, kk[j].w, sc[i][j]))));
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (p0 + tc + 16 * j < far[tr * 4 + i]) sum[j] += exp2f(sc[i][j] - ls[tr * 4 + i]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) red[tr][tc + 16 * j] = sum[j];
    __syncthreads();
    if (tid < count) {
        float v = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) v += red[i][tid];
        const int64_t at = (int64_t)s * a.nb_seq + (int64_t)kvh * a.nb_head + p0 + tid;
        a.out[at] = fmaf(a.decay, a.scores[at], v);
    }
}

}  // namespace kvscore

cudaError_t launch_kv_scores(cudaStream_t stream, const cvattn_kv_scores_params& p, int* status) {
    using namespace kvscore;
    Args a{};
    a.q = p.q;
    a.q_nb_node = p.q_nb_node;
    a.q_nb_seq = p.q_nb_seq;
    a.lse = p.lse;
    a.k = static_cast<const uint8_t*>(p.k.data);
    a.k_nb1 = p.k.nb1;
    a.k_nb2 = p.k.nb2;
    a.k_seq_ptrs = p.k_seq_ptrs;
    a.rows = p.rows;
    a.n_rows = p.n_rows;
    a.kv_len = p.kv_len;
    a.scores = p.scores;
    a.out = p.scores_out;
    a.nb_head = p.scores_nb_head;
    a.nb_seq = p.scores_nb_seq;
    a.k_type = p.k.type;
    a.n_seq = p.n_seq;
    a.n_q_rows = p.n_q_rows;
    a.max_rows = p.max_rows;
    a.Hq = p.n_q_heads;
    a.Hkv = p.k.n_heads;
    a.G = a.Hq / a.Hkv;
    a.max_kv_len = p.max_kv_len;
    a.scale_log2 = p.scale * 1.4426950408889634f;
    a.decay = p.decay;
    a.status = status;
    // From four 128-key tiles per SM on the persistent tcgen05 kernel, which starts later and goes through tiles faster (f16, whose
    // tiles cost the other kernel no conversion, also needs rows enough).  us of scores_mma_kernel | tcgen05, 14 / 2 heads, Q8_0
    // and f16: 16 sequences of 1000 (256 tiles), 28 rows 5.7 | 7.5 and 4.6 | 7.2; 16 of 2000 (512), 28 rows 7.7 | 8.7 and 5.7 |
    // 8.5, 112 rows 12.6 | 14.9 and 10.3 | 13.0, 448 rows 36 | 36 and 33 | 32; 64 of 1000 (1024), 7 rows 11.4 | 10.5 and 7.7 |
    // 10.4, 56 rows 17.1 | 13.7 and 13.6 | 12.4, 448 rows 69 | 47 and 63 | 41; 16 of 8192 (2048), 7 rows 20.0 | 14.6 and 13.7 |
    // 14.9, 28 rows 24.1 | 16.2 and 17.9 | 15.5.
    const int64_t entries = (int64_t)a.n_seq * a.Hkv * ((a.max_kv_len + kTcTile - 1) / kTcTile);
    const int64_t rows = (int64_t)a.max_rows * a.G;
    if (a.k_type != kF32 && entries >= 4 * 148 && entries < (int64_t)1 << 31 && (a.k_type != kF16 || entries * rows >= 1 << 15) &&
        a.n_seq <= kTcMaxSeq && rows <= kTcMaxRows) {
        TcArgs ta{};
        ta.a = a;
        ta.inv_g = (uint32_t)((65536 + a.G - 1) / a.G);
        ta.grid = 148;
        const int spare = (kTcRowTiles - (a.max_rows * a.G + 127) / 128) * 2 * kTcTileBytes;  // of the Q tiles
        const int raw = 2 * kTcTile * raw_stride(a.k_type);
        // (an even number: each producer group sees every phase of its own buffers)
        ta.raw_buffers = (2 + spare / raw < kTcRawBuffers ? 2 + spare / raw : kTcRawBuffers) & ~1;
        switch (a.k_type) {
        case kF16: return launch_tc_for_k<kF16>(stream, ta);
        case kQ4_0: return launch_tc_for_k<kQ4_0>(stream, ta);
        case kQ4_1: return launch_tc_for_k<kQ4_1>(stream, ta);
        case kQ5_0: return launch_tc_for_k<kQ5_0>(stream, ta);
        case kQ5_1: return launch_tc_for_k<kQ5_1>(stream, ta);
        case kQ8_0: return launch_tc_for_k<kQ8_0>(stream, ta);
        default: break;
        }
    }
    switch (a.k_type) {
    case kF16: return launch_mma_for_k<kF16>(stream, a);
    case kQ4_0: return launch_mma_for_k<kQ4_0>(stream, a);
    case kQ4_1: return launch_mma_for_k<kQ4_1>(stream, a);
    case kQ5_0: return launch_mma_for_k<kQ5_0>(stream, a);
    case kQ5_1: return launch_mma_for_k<kQ5_1>(stream, a);
    case kQ8_0: return launch_mma_for_k<kQ8_0>(stream, a);
    default: break;
    }
    const dim3 grid((unsigned)((a.max_kv_len + kTile - 1) / kTile), (unsigned)a.Hkv, (unsigned)a.n_seq);
    return launch_overlapped(scores_f32_kernel, grid, 128, 0, stream, a);
}

}  // namespace cvattn
