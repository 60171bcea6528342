// kv_evict.cu -- cvattn_kv_evict (which positions stay, and the rows that move)
// and cvattn_tree_commit (accepted drafts to the end of the cache).
#include "common.cuh"
#include "internal.h"
#include "launch.cuh"

namespace cvattn {
namespace evict {

constexpr int kThreads = 512;  // (1024 threads of 58 registers leave one CTA per SM: 31 us instead of 22 for 192 heads of 8192 slots)
constexpr int kWarps = kThreads / 32;
constexpr int kMaxKeySlots = 40 * 1024;  // 160 KB of keys
// Up to so many rows a head the selecting CTA moves them itself: one launch.  us of one | two launches, 4096 slots, Q8_0, 24 layers:
// one sequence, 64 moves 12.6 | 17.5, 256 15.6 | 17.7, 512 20.0 | 18.5; 8 sequences, 256 33.6 | 37.8, 512 50.2 | 49.6.
constexpr int kFusedMoves = 256;
constexpr int kLayersPerLaunch = 32;  // layer addresses that travel as kernel parameters

struct Args {
    uint8_t *k[kLayersPerLaunch], *v[kLayersPerLaunch];
    int64_t k_nb1, k_nb2, v_nb1, v_nb2;
    int k_slice, v_slice;  // bytes of one head in a row
    const float* scores;
    float* scores_out;
    const int32_t* pos;
    int32_t* pos_out;
    int64_t nb_head, nb_seq, nb_layer;
    const int32_t *kv_len, *kept_len, *n_tokens;
    int32_t* kv_len_out;  // null: written by a later launch
    int layers, Hkv, max_kv_len, budget, n_sink, n_recent;
    int32_t* ws;     // per (layer, seq, head): move count (padded to 4), then `moves` destinations, then sources
    int moves;       // most moves of one head
    int key_slots;   // slots whose keys fit shared memory
    bool fused;      // the selecting CTA moves the rows too
    int* status;
};

struct Seq {
    int L, kept, total;
    bool ok;
};
__device__ __forceinline__ Seq seq_of(const Args& a, int s) {
    Seq x;
    x.L = a.kv_len[s];
    x.kept = a.kept_len ? a.kept_len[s] : 0;
    x.total = a.n_tokens ? a.n_tokens[s] : x.L;
    x.ok = x.L >= 0 && x.L <= a.max_kv_len && x.kept >= 0 && x.kept <= x.L;
    return x;
}

// Order of the ranks as unsigned integers: a larger score is a larger key, -0 is
// +0, NaN is -infinity, and a protected token is above every score.
__device__ __forceinline__ uint32_t rank_key(float v, bool safe) {
    if (safe) return 0xffffffffu;
    if (v != v) v = -INFINITY;
    if (v == 0.0f) v = 0.0f;
    const uint32_t b = __float_as_uint(v);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

// K and V of one head: the rows dst[i] <- src[i], i0 <= i < i1, in units of 4 bytes where everything is aligned to them,
// else 2.  A warp takes a row, its lanes the units of the K and then of the V slice; four rows are on their way at once.
template <typename T>
__device__ __forceinline__ void move_rows(uint8_t* k, uint8_t* v, const Args& a, const int32_t* dst, const int32_t* src, int i0, int i1) {
    const int lane = threadIdx.x & 31, nw = blockDim.x >> 5;
    const int ku = a.k_slice / (int)sizeof(T), all = ku + a.v_slice / (int)sizeof(T);
    for (int u = lane; u < all; u += 32) {
        uint8_t* base = u < ku ? k + u * sizeof(T) : v + (u - ku) * sizeof(T);
        const int64_t nb1 = u < ku ? a.k_nb1 : a.v_nb1;
        for (int i = i0 + (threadIdx.x >> 5); i < i1; i += 4 * nw) {
            T x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (i + e * nw < i1) x[e] = *reinterpret_cast<const T*>(base + src[i + e * nw] * nb1);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (i + e * nw < i1) *reinterpret_cast<T*>(base + dst[i + e * nw] * nb1) = x[e];
        }
    }
}
__device__ __forceinline__ void move_head(const Args& a, int layer, int s, int kvh, const int32_t* dst, const int32_t* src, int i0, int i1) {
    uint8_t* k = a.k[layer] + (int64_t)s * a.k_nb2 + (int64_t)kvh * a.k_slice;
    uint8_t* v = a.v[layer] + (int64_t)s * a.v_nb2 + (int64_t)kvh * a.v_slice;
    // (a slice of an odd number of 2-byte units, such as one Q8_0 block, starts aligned in every second head only)
    const uint64_t all = reinterpret_cast<uint64_t>(k) | reinterpret_cast<uint64_t>(v) | (uint64_t)a.k_nb1 | (uint64_t)a.v_nb1 |
                         (uint64_t)a.k_slice | (uint64_t)a.v_slice;
    if ((all & 3) == 0) move_rows<uint32_t>(k, v, a, dst, src, i0, i1);
    else move_rows<uint16_t>(k, v, a, dst, src, i0, i1);
}

// One CTA per (head, sequence, layer).  The keys are formed once, in shared memory
// as far as they fit.  The budget-th largest is found by a radix select over 8 bits
// at a time; of the slots that equal it, the lowest stay.  Each warp owns a run of
// slots, so ranks in slot order are ballots plus one prefix over the warps.
// Latency-bound: four passes over keys in shared memory with a barrier each.  24 layers of one
// sequence, 576 slots to 512: 7.7 us, moves included; 6 layers of 16 sequences of up to 8192
// to 1024: 22 us of 31 (the moves are the rest), 1.3 TB/s of scores, tokens and rows in all.
// (Calls in a graph that repeat on the same buffers: scores and tokens come from L2.  On buffers
// that are not there the second takes 38 us.)
__global__ void __launch_bounds__(kThreads, 2) evict_select_kernel(const __grid_constant__ Args a) {
    extern __shared__ uint32_t keys[];
    __shared__ uint32_t hist[2][256];
    __shared__ uint32_t sh_prefix;
    __shared__ int sh_need, wsum[3][kWarps];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int kvh = blockIdx.x, s = blockIdx.y, layer = blockIdx.z;
    griddep_wait();
    const Seq x = seq_of(a, s);
    int32_t* ws = a.ws + (((int64_t)layer * gridDim.y + s) * gridDim.x + kvh) * (2 * (int64_t)a.moves + 4);
    if (tid == 0) {
        if (!x.ok) record_status(a.status, kStatusBadLength);
        if (a.kv_len_out && kvh == 0 && layer == 0) a.kv_len_out[s] = x.ok ? min(x.L, a.budget) : x.L;
        if (!x.ok || x.L <= a.budget) ws[0] = 0;
    }
    if (!x.ok) return;
    const int64_t base = (int64_t)layer * a.nb_layer + (int64_t)s * a.nb_seq + (int64_t)kvh * a.nb_head;
    const float* sc = a.scores + base;
    const int32_t* pos = a.pos ? a.pos + base : nullptr;
    auto token = [&](int j) { return j < x.kept ? pos[j] : x.total - x.L + j; };
    if (x.L <= a.budget) {
        for (int j = tid; j < x.L; j += kThreads) {
            a.pos_out[base + j] = token(j);
            a.scores_out[base + j] = sc[j];
        }
        return;
    }
    auto form = [&](int j) {
        const int t = token(j);
        return rank_key(sc[j], t < a.n_sink || t >= x.total - a.n_recent);
    };
    auto key_at = [&](int j) { return j < a.key_slots ? keys[j] : form(j); };
    hist[tid >> 8][tid & 255] = 0;
    __syncthreads();
    const int here = min(x.L, a.key_slots);
#pragma unroll 4
    for (int j = tid; j < here; j += kThreads) {
        const uint32_t u = form(j);
        keys[j] = u;
        atomicAdd(&hist[0][u >> 24], 1u);
    }
    for (int j = here + tid; j < x.L; j += kThreads) atomicAdd(&hist[0][form(j) >> 24], 1u);
    uint32_t prefix = 0;
    int need = a.budget;  // how many of the keys that match the prefix stay
#pragma unroll 1
    for (int shift = 24;; shift -= 8) {
        uint32_t* now = hist[(shift >> 3) & 1 ? 0 : 1];   // 24, 8: hist[0]; 16, 0: hist[1]
        uint32_t* next = hist[(shift >> 3) & 1 ? 1 : 0];
        __syncthreads();
        if (warp == 0) {
            // lane i: bins 255 - 8 i downwards; the bin in which the need-th largest key lies
            uint32_t c[8], own = 0;
#pragma unroll
            for (int b = 0; b < 8; ++b) own += c[b] = now[255 - 8 * lane - b];
            uint32_t incl = own;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t y = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += y;
            }
            uint32_t before = incl - own;
            if (before < (uint32_t)need && incl >= (uint32_t)need) {
                int b = 0;
#pragma unroll
                for (; b < 7; ++b) {
                    if (before + c[b] >= (uint32_t)need) break;
                    before += c[b];
                }
                sh_prefix = prefix | ((uint32_t)(255 - 8 * lane - b) << shift);
                sh_need = need - (int)before;
            }
        } else {
            for (int i = tid - 32; i < 256; i += kThreads - 32) next[i] = 0;
        }
        __syncthreads();
        prefix = sh_prefix;
        need = sh_need;
        if (shift == 0) break;
        const uint32_t above = 0xffffffffu << shift;
        for (int j = tid; j < x.L; j += kThreads) {
            const uint32_t u = key_at(j);
            if ((u & above) == prefix) atomicAdd(&next[(u >> (shift - 8)) & 255], 1u);
        }
    }
    // slots of this warp: [j0, j1)
    const int per = ((x.L + kWarps - 1) / kWarps + 31) & ~31;
    const int j0 = min(x.L, warp * per), j1 = min(x.L, j0 + per);
    int ties = 0;
    for (int j = j0; j < j1; j += 32) {
        const bool tie = j + lane < j1 && key_at(j + lane) == prefix;
        ties += __popc(__ballot_sync(0xffffffffu, tie));
    }
    if (lane == 0) wsum[0][warp] = ties;
    __syncthreads();
    int tie0 = 0;
    for (int w = 0; w < warp; ++w) tie0 += wsum[0][w];
    const uint32_t below = (1u << lane) - 1u;
    // kept of 32 slots, by ballot; t0 counts the ties before them
    auto kept_of = [&](int j, int& t0) {
        const uint32_t u = j + lane < j1 ? key_at(j + lane) : 0u;
        const bool tie = j + lane < j1 && u == prefix;
        const uint32_t tb = __ballot_sync(0xffffffffu, tie);
        const bool keep = j + lane < j1 && (u > prefix || (tie && t0 + __popc(tb & below) < need));
        t0 += __popc(tb);
        return keep;
    };
    int holes = 0, movers = 0, t0 = tie0;
    for (int j = j0; j < j1; j += 32) {
        const bool keep = kept_of(j, t0);
        const bool in = j + lane < j1, low = j + lane < a.budget;
        holes += __popc(__ballot_sync(0xffffffffu, in && low && !keep));
        movers += __popc(__ballot_sync(0xffffffffu, in && !low && keep));
    }
    if (lane == 0) {
        wsum[1][warp] = holes;
        wsum[2][warp] = movers;
    }
    __syncthreads();
    int h0 = 0, m0 = 0, total = 0;
    for (int w = 0; w < kWarps; ++w) {
        if (w < warp) {
            h0 += wsum[1][w];
            m0 += wsum[2][w];
        }
        total += wsum[1][w];
    }
    int32_t* dst = ws + 4;
    int32_t* src = dst + a.moves;
    if (tid == 0) ws[0] = total;
    t0 = tie0;
    for (int j = j0; j < j1; j += 32) {
        const bool keep = kept_of(j, t0);
        const bool in = j + lane < j1, low = j + lane < a.budget;
        const bool hole = in && low && !keep, mover = in && !low && keep;
        const uint32_t hb = __ballot_sync(0xffffffffu, hole), mb = __ballot_sync(0xffffffffu, mover);
        if (hole) dst[h0 + __popc(hb & below)] = j + lane;
        if (mover) src[m0 + __popc(mb & below)] = j + lane;
        h0 += __popc(hb);
        m0 += __popc(mb);
    }
    __syncthreads();
    griddep_launch_dependents();
    // the lists are complete: rows that stay, then rows that move, then the cleared tail
#pragma unroll 4
    for (int j = tid; j < a.budget; j += kThreads) {
        a.pos_out[base + j] = token(j);
        if (a.scores_out != a.scores) a.scores_out[base + j] = sc[j];
    }
    __syncthreads();
    for (int i = tid; i < total; i += kThreads) {
        a.pos_out[base + dst[i]] = token(src[i]);
        a.scores_out[base + dst[i]] = sc[src[i]];
    }
    if (a.fused) move_head(a, layer, s, kvh, dst, src, 0, total);
    __syncthreads();
    for (int j = a.budget + tid; j < x.L; j += kThreads) a.scores_out[base + j] = 0.0f;
}

constexpr int kMoveChunk = 64;  // rows of one head per CTA

// The moves of long lists, spread over CTAs of their own.  Scattered slices of 36 to 128 bytes:
// bound by the sectors that they touch; 16 sequences of 8192 to 1024, Q8_0 / Q4_0: 9 us.
__global__ void __launch_bounds__(256) evict_move_kernel(const __grid_constant__ Args a, int n_seq) {
    const int kvh = blockIdx.y % a.Hkv, s = blockIdx.y / a.Hkv, layer = blockIdx.z;
    const int32_t* ws = a.ws + (((int64_t)layer * n_seq + s) * a.Hkv + kvh) * (2 * (int64_t)a.moves + 4);
    griddep_wait();
    const int n = ws[0], i0 = blockIdx.x * kMoveChunk, i1 = min(n, i0 + kMoveChunk);
    if (i0 >= i1) return;
    const int32_t *dst = ws + 4, *src = dst + a.moves;
    move_head(a, layer, s, kvh, dst, src, i0, i1);
}

// kv_len_out that shares memory with a length read above: after every reader is done.
__global__ void evict_length_kernel(const int32_t* kv_len, const int32_t* kept, int32_t* out, int n, int most, int budget) {
    const int s = blockIdx.x * blockDim.x + threadIdx.x;
    griddep_wait();
    if (s >= n) return;
    const int L = kv_len[s], kp = kept ? kept[s] : 0;
    out[s] = L >= 0 && L <= most && kp >= 0 && kp <= L ? min(L, budget) : L;
}

}  // namespace evict

size_t kv_evict_workspace_bytes(int n_layers, int n_seq, int n_kv_heads, int max_kv_len, int budget) {
    const int64_t moves = max_kv_len > budget ? (max_kv_len - budget < budget ? max_kv_len - budget : budget) : 0;
    return (size_t)n_layers * n_seq * n_kv_heads * (2 * moves + 4) * 4;
}

cudaError_t launch_kv_evict(cudaStream_t stream, const cvattn_kv_evict_params& p, int64_t k_slice, int64_t v_slice, int* status) {
    using namespace evict;
    const bool shared_len = p.kv_len_out == p.kv_len || p.kv_len_out == p.kept_len;
    const int Hkv = p.k[0].n_heads;
    const int moves = p.max_kv_len > p.budget ? (p.max_kv_len - p.budget < p.budget ? p.max_kv_len - p.budget : p.budget) : 0;
    for (int l0 = 0; l0 < p.n_layers; l0 += kLayersPerLaunch) {
        const int n = p.n_layers - l0 < kLayersPerLaunch ? p.n_layers - l0 : kLayersPerLaunch;
        Args a{};
        for (int i = 0; i < n; ++i) {
            a.k[i] = static_cast<uint8_t*>(p.k[l0 + i].data);
            a.v[i] = static_cast<uint8_t*>(p.v[l0 + i].data);
        }
        a.k_nb1 = p.k[0].nb1; a.k_nb2 = p.k[0].nb2; a.v_nb1 = p.v[0].nb1; a.v_nb2 = p.v[0].nb2;
        a.k_slice = (int)k_slice;
        a.v_slice = (int)v_slice;
        a.scores = p.scores + l0 * p.nb_layer;
        a.scores_out = p.scores_out + l0 * p.nb_layer;
        a.pos = p.pos ? p.pos + l0 * p.nb_layer : nullptr;
        a.pos_out = p.pos_out + l0 * p.nb_layer;
        a.nb_head = p.nb_head; a.nb_seq = p.nb_seq; a.nb_layer = p.nb_layer;
        a.kv_len = p.kv_len;
        a.kept_len = p.kept_len;
        a.n_tokens = p.n_tokens;
        a.kv_len_out = shared_len || l0 ? nullptr : p.kv_len_out;
        a.layers = n;
        a.Hkv = Hkv;
        a.max_kv_len = p.max_kv_len;
        a.budget = p.budget;
        a.n_sink = p.n_sink;
        a.n_recent = p.n_recent;
        a.moves = moves;
        a.ws = static_cast<int32_t*>(p.workspace) + (int64_t)l0 * p.n_seq * Hkv * (2 * (int64_t)moves + 4);
        a.status = status;
        a.key_slots = p.max_kv_len < kMaxKeySlots ? p.max_kv_len : kMaxKeySlots;
        a.fused = moves <= kFusedMoves;
        const int smem = a.key_slots * 4;
        cudaError_t e = cudaSuccess;
        if (smem > 40 * 1024) e = cudaFuncSetAttribute(evict_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxKeySlots * 4);
        if (e != cudaSuccess) return e;
        e = launch_overlapped(evict_select_kernel, dim3((unsigned)Hkv, (unsigned)p.n_seq, (unsigned)n), kThreads, smem, stream, a);
        if (e != cudaSuccess) return e;
        if (!a.fused) {
            const dim3 grid((unsigned)((moves + kMoveChunk - 1) / kMoveChunk), (unsigned)(Hkv * p.n_seq), (unsigned)n);
            e = launch_overlapped(evict_move_kernel, grid, 256, 0, stream, a, p.n_seq);
            if (e != cudaSuccess) return e;
        }
    }
    if (shared_len) {
        return launch_overlapped(evict_length_kernel, dim3((unsigned)((p.n_seq + 255) / 256)), 256, 0, stream, p.kv_len, p.kept_len,
                                 p.kv_len_out, p.n_seq, p.max_kv_len, p.budget);
    }
    return cudaSuccess;
}

// ---------------------------------------------------------------- commit --

namespace commit {

constexpr int kTensorsPerLaunch = 48;  // 24 layers of K and V

struct Tensor {
    uint8_t* dst;
    const uint8_t* src;
    int64_t dst_nb1, dst_nb2, src_nb1, src_nb2;
    int row;  // bytes
    int unit; // bytes that every address and stride is a multiple of: 16, 8, 4 or 2
};

struct Args {
    Tensor t[kTensorsPerLaunch];
    const int32_t* accepted;
    int64_t accepted_stride;
    const int32_t *n_accepted, *kv_len;
    int32_t* kv_len_out;  // null: written by a later launch
    int n_seq, max_accepted, draft_rows;
    int64_t capacity;
    int* status;
};

template <typename T>
__device__ __forceinline__ void copy_rows(const Tensor& t, uint8_t* dst, const uint8_t* src, const int32_t* node, int n) {
    const int units = t.row / (int)sizeof(T);
    for (int i = threadIdx.x; i < n * units; i += blockDim.x) {
        const int r = i / units, u = i - r * units;
        reinterpret_cast<T*>(dst + (int64_t)r * t.dst_nb1)[u] = reinterpret_cast<const T*>(src + (int64_t)node[r] * t.src_nb1)[u];
    }
}

// Whether sequence s can be committed: lengths in range and every node a drafted row.
__device__ __forceinline__ bool fits(const Args& a, int s, int L, int n) {
    if (L < 0 || n < 0 || n > a.max_accepted || L + (int64_t)n > a.capacity) return false;
    for (int i = 0; i < n; ++i) {
        const int node = a.accepted[(int64_t)s * a.accepted_stride + i];
        if (node < 0 || node >= a.draft_rows) return false;
    }
    return true;
}

// A CTA per sequence and tensor.  Latency-bound (a launch, two dependent loads, the copy): 48
// tensors of one sequence, 4 rows 2.2 us; of 64 sequences, up to 16 rows 5.5 us for 5.6 MB
// read and written, 1.0 TB/s (in a graph; a call by itself, bound by the host, takes 5.0 and 5.4).
__global__ void __launch_bounds__(128) commit_kernel(const __grid_constant__ Args a) {
    const int s = blockIdx.x;
    const Tensor& t = a.t[blockIdx.y];
    griddep_wait();
    const int L = a.kv_len[s], n = a.n_accepted[s];
    const bool ok = fits(a, s, L, n);
    if (threadIdx.x == 0 && blockIdx.y == 0) {
        if (!ok) record_status(a.status, kStatusBadPosition);
        if (a.kv_len_out) a.kv_len_out[s] = ok ? L + n : L;
    }
    if (!ok) return;
    uint8_t* dst = t.dst + (int64_t)s * t.dst_nb2 + (int64_t)L * t.dst_nb1;
    const uint8_t* src = t.src + (int64_t)s * t.src_nb2;
    const int32_t* node = a.accepted + (int64_t)s * a.accepted_stride;
    switch (t.unit) {
    case 16: copy_rows<uint4>(t, dst, src, node, n); break;
    case 8: copy_rows<uint2>(t, dst, src, node, n); break;
    case 4: copy_rows<uint32_t>(t, dst, src, node, n); break;
    default: copy_rows<uint16_t>(t, dst, src, node, n); break;
    }
}

__global__ void commit_length_kernel(const __grid_constant__ Args a, int32_t* out) {
    const int s = blockIdx.x * blockDim.x + threadIdx.x;
    griddep_wait();
    if (s >= a.n_seq) return;
    const int L = a.kv_len[s], n = a.n_accepted[s];
    out[s] = fits(a, s, L, n) ? L + n : L;
}

}  // namespace commit

cudaError_t launch_tree_commit(cudaStream_t stream, const cvattn_tree_commit_params& p, int64_t capacity, int64_t draft_rows,
                               int* status) {
    using namespace commit;
    Args a{};
    a.accepted = p.accepted;
    a.accepted_stride = p.accepted_stride;
    a.n_accepted = p.n_accepted;
    a.kv_len = p.kv_len;
    a.n_seq = p.n_seq;
    a.max_accepted = p.max_accepted;
    a.draft_rows = (int)draft_rows;
    a.capacity = capacity;
    a.status = status;
    const bool shared_len = p.kv_len_out == p.kv_len;
    for (int t0 = 0; t0 < p.n_tensors; t0 += kTensorsPerLaunch) {
        const int n = p.n_tensors - t0 < kTensorsPerLaunch ? p.n_tensors - t0 : kTensorsPerLaunch;
        a.kv_len_out = t0 || shared_len ? nullptr : p.kv_len_out;
        for (int i = 0; i < n; ++i) {
            const cvattn_tensor &c = p.caches[t0 + i], &d = p.drafts[t0 + i];
            Tensor& t = a.t[i];
            t.dst = static_cast<uint8_t*>(c.data);
            t.src = static_cast<const uint8_t*>(d.data);
            t.dst_nb1 = c.nb1; t.dst_nb2 = c.nb2; t.src_nb1 = d.nb1; t.src_nb2 = d.nb2;
            t.row = (int)type_row_bytes(c.type, (int64_t)c.n_heads * c.head_dim);
            const uint64_t all = reinterpret_cast<uint64_t>(t.dst) | reinterpret_cast<uint64_t>(t.src) | (uint64_t)t.dst_nb1 |
                                 (uint64_t)t.dst_nb2 | (uint64_t)t.src_nb1 | (uint64_t)t.src_nb2 | (uint64_t)t.row;
            t.unit = (all & 15) == 0 ? 16 : (all & 7) == 0 ? 8 : (all & 3) == 0 ? 4 : 2;
        }
        const cudaError_t e = launch_overlapped(commit_kernel, dim3((unsigned)p.n_seq, (unsigned)n), 128, 0, stream, a);
        if (e != cudaSuccess) return e;
    }
    if (shared_len) {
        return launch_overlapped(commit_length_kernel, dim3((unsigned)((p.n_seq + 127) / 128)), 128, 0, stream, a, p.kv_len_out);
    }
    return cudaSuccess;
}

}  // namespace cvattn
