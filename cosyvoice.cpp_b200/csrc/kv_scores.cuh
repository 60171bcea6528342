// kv_scores.cuh -- the attention weight that each cached position receives:
//   s_j <- decay s_j + sum over rows (token i, query head h of the KV head) of
//          exp2(c q.k_j - lse log2 e),  c = scale log2 e.
// The rows' log-sums are known, so a key's sum needs no second pass over the keys
// and no exchange between CTAs: a CTA owns its keys and walks all rows.
// The kernel here, on mma.sync m16n8k16, is for lists too short to fill the SMs: rows are the
// M of the products, prepared as A fragments in shared memory once per CTA; each warp has its
// own keys, so a key's sum crosses 8 lanes by shuffles.  One sequence of 500 positions, 1 row
// of 14 heads, Q8_0: 4.1 us, a launch and one trip to memory and back.
#pragma once

#include "tree_mma.cuh"

namespace cvattn {
namespace kvscore {

using dmma::mma16816;
using dmma::quad_max;
using dmma::quad_sum;
using dmma::split2;
using dtc::pow2f;
using tree::convert_block;
using tree::kD;
using tree::ldsm4;
using tree::mma16816_first;
using tree::raw_stride;
using tree::store_block;

struct Args {
    const float* q;
    int64_t q_nb_node, q_nb_seq;
    const float* lse;
    const uint8_t* k;
    int64_t k_nb1, k_nb2;
    const uint64_t* k_seq_ptrs;
    const int32_t *rows, *n_rows, *kv_len;
    const float* scores;
    float* out;
    int64_t nb_head, nb_seq;
    int k_type, n_seq, n_q_rows, max_rows, Hq, Hkv, G, max_kv_len;
    float scale_log2, decay;
    int* status;
};

// The lengths of a sequence; false (and recorded) if they, or its rows' address, are out of range.
__device__ __forceinline__ bool lens_of(const Args& a, int s, int& L, int& n, bool record) {
    L = a.kv_len[s];
    n = a.n_rows ? a.n_rows[s] : a.max_rows;
    const bool odd = a.k_seq_ptrs && (a.k_seq_ptrs[s] & (a.k_type == kF32 ? 3 : 1));
    if (L >= 0 && L <= a.max_kv_len && n >= 0 && n <= a.max_rows && n <= L && !odd) return true;
    if (record) record_status(a.status, kStatusBadLength);
    return false;
}

// ------------------------------------------------------------- MMA kernel --
//
// f16 and block-quantized caches, mma.sync m16n8k16 with the exact operands of
// tree_mma.cuh (integer quants in f16, scales aside, Q in f16 hi + lo).  A CTA of 8
// warps takes 64 NT keys of one KV head; a warp keeps the K fragments of its 8 NT
// keys in registers and walks the rows, 16 at a time, whose Q fragments the CTA
// prepares 8 row tiles at a time.  The sums of a key over the rows stay in
// registers and are joined over the 8 row lanes at the end, always in the same
// order.
constexpr int kThreads = 256;
constexpr int kRowTiles = 8;  // prepared at a time

template <int KT, int NT>
struct Smem {
    static constexpr int kKeys = 64 * NT;
    static constexpr bool K_Q = KT != kF16;
    static constexpr int qf = 0;                                    // Q fragments [row tile][k-step][hi, lo][lane]
    static constexpr int info = qf + kRowTiles * 4096;              // float4 per row: factor, -log-sum, block sums of Q
    static constexpr int far = info + kRowTiles * 16 * 16;          // keys that the row sees
    static constexpr int tab = far + kRowTiles * 16 * 4;            // K scales (and mins) [block][key]
    static constexpr int tile = (tab + (K_Q ? (BlockTraits<KT>::HAS_MIN ? 4 : 2) * kKeys * 4 : 0) + 127) / 128 * 128;
    static constexpr int raw = tile + kKeys * 128;
    static constexpr int bytes = raw + (K_Q ? kKeys * raw_stride(KT) : 0);
};

template <int KT, int NT>
__global__ void __launch_bounds__(kThreads, NT == 2 ? 3 : 2) scores_mma_kernel(const __grid_constant__ Args a) {
    using S = Smem<KT, NT>;
    constexpr int kKeys = S::kKeys, slice = 2 * group_bytes(KT);
    constexpr bool K_Q = S::K_Q, K_MIN = BlockTraits<KT>::HAS_MIN;
    extern __shared__ __align__(128) uint8_t smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gid = lane >> 2, tig = lane & 3;
    const int s = blockIdx.z, kvh = blockIdx.y, p0 = blockIdx.x * kKeys;
    int L, n;
    griddep_wait();
    if (!lens_of(a, s, L, n, tid == 0) || p0 >= L) return;
    const int count = min(kKeys, L - p0), total = n * a.G;
    {   // the keys' rows: f16 straight into the tile, quants raw
        const uint8_t* kb = (a.k_seq_ptrs ? reinterpret_cast<const uint8_t*>(a.k_seq_ptrs[s]) : a.k + (int64_t)s * a.k_nb2) +
                            (int64_t)p0 * a.k_nb1 + kvh * slice;
        const uint64_t al = reinterpret_cast<uint64_t>(kb) | (uint64_t)a.k_nb1;
        const int unit = KT == kF16 && (al & 15) == 0 ? 16 : (al & 3) == 0 ? 4 : 2;
        const int w = slice / unit, per = kThreads / w, k0 = tid / w, col = (tid - k0 * w) * unit;
        const uint8_t* from = kb + (int64_t)k0 * a.k_nb1 + col;
        const int64_t step = (int64_t)per * a.k_nb1;
        if (k0 < per) {
#pragma unroll 4
            for (int key = k0; key < count; key += per, from += step) {
                uint8_t* to = K_Q ? smem + S::raw + key * raw_stride(KT) + col : smem + S::tile + key * 128 + (col ^ ((key & 7) << 4));
                if (unit == 16) tree::cp_async16(to, from, true);
                else if (unit == 4) tree::cp_async4(to, from, true);
                else *reinterpret_cast<uint16_t*>(to) = *reinterpret_cast<const uint16_t*>(from);
            }
        }
        tree::cp_async_commit();
    }
    uint4* qf = reinterpret_cast<uint4*>(smem + S::qf);
    float4* info = reinterpret_cast<float4*>(smem + S::info);
    int* far = reinterpret_cast<int*>(smem + S::far);
    const float* tab = reinterpret_cast<const float*>(smem + S::tab);
    uint32_t kf[NT][4][2];             // K fragments: [8-key tile][k-step]
    float sum[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) sum[t][0] = sum[t][1] = 0.0f;
    const int kw = warp * 8 * NT;      // this warp's first key
    // the old scores of the two keys that this lane will write (row lane t for key tile t)
    const int key_out = kw + 8 * gid + 2 * tig;
    const int64_t at_out = (int64_t)s * a.nb_seq + (int64_t)kvh * a.nb_head + p0 + key_out;
    const bool w0 = gid < NT && key_out < count, w1 = gid < NT && key_out + 1 < count;
    const float old0 = w0 ? a.scores[at_out] : 0.0f, old1 = w1 ? a.scores[at_out + 1] : 0.0f;

    for (int base = 0; base < total; base += kRowTiles * 16) {
        if (base) __syncthreads();     // every warp is done with the last rows
        // this warp's row tile of the batch
        bool left_out = false;
        if (base + warp * 16 < total) {
            uint32_t hi[4][4], lo[4][4];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int rl = warp * 16 + half * 8 + gid, r = base + rl;
                int t = r / a.G, at = t;
                const int h = kvh * a.G + r - t * a.G;
                bool real = r < total;
                float ls = -INFINITY;
                if (real) {
                    if (a.rows) at = a.rows[(int64_t)s * a.max_rows + t];
                    if (at < 0 || at >= a.n_q_rows) {
                        record_status(a.status, kStatusBadPosition);
                        real = false;
                    } else {
                        ls = a.lse[((int64_t)s * a.n_q_rows + at) * a.Hq + h];
                        real = ls != -INFINITY;
                    }
                }
                left_out |= !real;
                const float* q = a.q + (int64_t)s * a.q_nb_seq + (int64_t)at * a.q_nb_node + h * kD + 2 * tig;
                float2 e[8];  // dims 8 i + 2 tig, + 1
                float am = 0.0f, qs[2] = {0.0f, 0.0f};
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    e[i] = real ? *reinterpret_cast<const float2*>(q + 8 * i) : make_float2(0.f, 0.f);
                    am = fmaxf(am, fmaxf(fabsf(e[i].x), fabsf(e[i].y)));
                    qs[i >> 2] += e[i].x + e[i].y;
                }
                const int ex = dtc::norm_exp(quad_max(am));
                const float sc = pow2f(ex);
                if constexpr (K_MIN) {
                    qs[0] = quad_sum(qs[0]) * a.scale_log2;
                    qs[1] = quad_sum(qs[1]) * a.scale_log2;
                }
                if (tig == 0) {
                    info[rl] = make_float4(pow2f(-ex) * a.scale_log2, real ? -ls * 1.4426950408889634f : -INFINITY, qs[0], qs[1]);
                    far[rl] = real ? L - n + t + 1 : 0;
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) split2(e[i].x * sc, e[i].y * sc, hi[i >> 1][2 * (i & 1) + half], lo[i >> 1][2 * (i & 1) + half]);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                qf[((warp * 4 + k) * 2 + 0) * 32 + lane] = make_uint4(hi[k][0], hi[k][1], hi[k][2], hi[k][3]);
                qf[((warp * 4 + k) * 2 + 1) * 32 + lane] = make_uint4(lo[k][0], lo[k][1], lo[k][2], lo[k][3]);
            }
        }
        if (base == 0) {  // K: raw rows to f16 tiles and scales, then this warp's fragments
            tree::cp_async_wait<0>();
            __syncthreads();
            if constexpr (K_Q) {
                float* tb = reinterpret_cast<float*>(smem + S::tab);
#pragma unroll 1
                for (int i = tid; i < 2 * kKeys; i += kThreads) {  // a warp converts one block of 32 keys
                    const int blk = (i >> 5) & 1, key = (i >> 6) * 32 + lane;
                    if ((i >> 6) * 32 >= count) break;
                    uint32_t w[16];
                    float d, m;
                    const uint8_t* g = smem + S::raw + key * raw_stride(KT);
                    if (blk) convert_block<KT, 1>(g, w, d, m);
                    else convert_block<KT, 0>(g, w, d, m);
                    store_block(smem + S::tile, key, blk, w);
                    tb[blk * kKeys + key] = d;
                    if constexpr (K_MIN) tb[(2 + blk) * kKeys + key] = m;
                }
                __syncthreads();
            }
            const uint32_t kt = smem_addr(smem + S::tile);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const uint32_t row = lane & 7, mat = lane >> 3;
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    uint32_t r[4];
                    ldsm4(r, kt + (kw + 8 * t + row) * 128 + (((4 * half + mat) ^ row) << 4));
                    kf[t][2 * half][0] = r[0]; kf[t][2 * half][1] = r[1];
                    kf[t][2 * half + 1][0] = r[2]; kf[t][2 * half + 1][1] = r[3];
                }
            }
        }
        const bool any_out = __syncthreads_or(left_out);
        if (kw >= count) continue;
        const bool masked = any_out || p0 + kw + 8 * NT > L - n + 1;  // some (row, key) of this warp may be unseen
        const int tiles = min(kRowTiles, (total - base + 15) / 16);
#pragma unroll 1
        for (int rt = 0; rt < tiles; ++rt) {
            float acc[NT][K_Q ? 2 : 1][4];
            // low parts of Q first, while the sums are small: adds inside the tensor cores truncate
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint4 l4 = qf[((rt * 4 + k) * 2 + 1) * 32 + lane];
                const uint32_t al[4] = {l4.x, l4.y, l4.z, l4.w};
                const int b = K_Q ? k >> 1 : 0;
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    if (k == 0 || (K_Q && k == 2)) mma16816_first(acc[t][b], al, kf[t][k][0], kf[t][k][1]);
                    else mma16816(acc[t][b], al, kf[t][k][0], kf[t][k][1]);
                }
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint4 h4 = qf[((rt * 4 + k) * 2 + 0) * 32 + lane];
                const uint32_t ah[4] = {h4.x, h4.y, h4.z, h4.w};
                const int b = K_Q ? k >> 1 : 0;
#pragma unroll
                for (int t = 0; t < NT; ++t) mma16816(acc[t][b], ah, kf[t][k][0], kf[t][k][1]);
            }
            const float4 i0 = info[rt * 16 + gid], i1 = info[rt * 16 + 8 + gid];
            const int f0 = masked ? far[rt * 16 + gid] - p0 : 0, f1 = masked ? far[rt * 16 + 8 + gid] - p0 : 0;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const int c = kw + 8 * t + 2 * tig;
                float2 d0 = make_float2(1.f, 1.f), d1 = d0, m0 = make_float2(0.f, 0.f), m1 = m0;
                if constexpr (K_Q) {
                    d0 = *reinterpret_cast<const float2*>(tab + c);
                    d1 = *reinterpret_cast<const float2*>(tab + kKeys + c);
                    if constexpr (K_MIN) {
                        m0 = *reinterpret_cast<const float2*>(tab + 2 * kKeys + c);
                        m1 = *reinterpret_cast<const float2*>(tab + 3 * kKeys + c);
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float4 ri = i < 2 ? i0 : i1;
                    float v, off = ri.y;
                    if constexpr (K_Q) v = fmaf(acc[t][0][i], (i & 1) ? d0.y : d0.x, acc[t][1][i] * ((i & 1) ? d1.y : d1.x));
                    else v = acc[t][0][i];
                    if constexpr (K_MIN) off = fmaf((i & 1) ? m0.y : m0.x, ri.z, fmaf((i & 1) ? m1.y : m1.x, ri.w, off));
                    float p = fast_exp2(fmaf(v, ri.x, off));
                    if (masked && c + (i & 1) >= (i < 2 ? f0 : f1)) p = 0.0f;
                    sum[t][i & 1] += p;
                }
            }
        }
    }
    tree::cp_async_wait<0>();  // (no rows: nothing has waited for the copies)
    float v0 = 0.0f, v1 = 0.0f;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float v = sum[t][e];
            v += __shfl_xor_sync(0xffffffffu, v, 4);
            v += __shfl_xor_sync(0xffffffffu, v, 8);
            v += __shfl_xor_sync(0xffffffffu, v, 16);
            if (gid == t) (e ? v1 : v0) = v;
        }
    if (w0) a.out[at_out] = fmaf(a.decay, old0, v0);
    if (w1) a.out[at_out + 1] = fmaf(a.decay, old1, v1);
}

// Launch for K type KT (kv_scores_inst.cu, one unit per K type).
template <int KT> cudaError_t launch_mma_for_k(cudaStream_t stream, const Args& a);

}  // namespace kvscore
}  // namespace cvattn
