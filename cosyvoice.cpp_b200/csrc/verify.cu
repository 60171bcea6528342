// verify.cu -- drafted tokens against the target's logits, with given random numbers.
//
// verify_sums_kernel reads every row once: its largest logit m and the sum W of weights exp((l - m) / temperature), in parts
// of 2048 vectors.  verify_walk_kernel joins a sequence's parts and walks down its drafts, u q(t) W < w(t) deciding about a
// draft of token t, then finds the token that follows.
// Weights of the first kernel are f32 exponentials added up in 64 bits: a decision that they could turn has a chance of 1e-7.
// Where a draft has been refused or the path ends, there are as many borders as the vocabulary has tokens, so there the weights
// are formed in 64 bits too: 2^(n/64) from a table, the rest by its Taylor polynomial (x^4/24 < 2^-34 at x = ln 2 / 128).  The
// token that follows: sums of tiles of 32 vectors, then of the one tile that holds the border its elements in order.
//
// What bounds it, 32 chains of 8 over 151937 tokens in bf16, with draft probabilities: 42.6 us.  The sums take about 20 (78 MB in all, 12 us of
// bytes; exponentials' unit and issue slots 55 % busy each): rows that no path reaches are summed too, but a walk that sums the rows
// as it meets them, 4 of 8 here, took 87 to 107, 13 thousand cycles a node on the few SMs of one sequence.  The rest is the
// walk: a scan of a row in 64 bits for each refusal and for the token that follows (one scan for both where only one draft was refused).
// A small vocabulary is latency: 7 nodes of 6563 tokens take 11.3 to 12 us.
#include <cuda_bf16.h>

#include "common.cuh"
#include "internal.h"
#include "launch.cuh"

namespace cvattn {
namespace verify {

constexpr int kThreads = 512, kWarps = kThreads / 32;       // of the walk
constexpr int kSumThreads = 256, kSumWarps = kSumThreads / 32;
constexpr int kBF16 = CVATTN_TYPE_BF16;
constexpr int kMaxNodes = CVATTN_TREE_MAX_NODES;
constexpr int kMaxCluster = 8;
constexpr int kHeld = 8;             // vectors of a row that a thread keeps between its passes
constexpr int kSlice = kSumThreads * kHeld;
constexpr int kMaxTiles = 2048;      // of 32 vectors, per CTA

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_arrive_relaxed() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// A row of logits: `head` elements up to the first 16-byte boundary, `full` vectors of kPer elements, and the rest.
template <int T> struct Row {
    static constexpr int kSize = T == kF32 ? 4 : 2, kPer = 16 / kSize;
    const uint8_t* at;     // element 0
    int head, full, vocab;
    __device__ __forceinline__ Row(const void* logits, int64_t elements, int v) {
        at = static_cast<const uint8_t*>(logits) + elements * kSize;
        head = min(v, (int)(-reinterpret_cast<uintptr_t>(at) & 15) / kSize);
        full = (v - head) / kPer;
        vocab = v;
    }
    __device__ __forceinline__ int first(int j) const { return head + j * kPer; }  // element of vector j's place 0
    __device__ __forceinline__ uint4 load(int j) const { return __ldg(reinterpret_cast<const uint4*>(at + (int64_t)first(j) * kSize)); }
    // Elements outside the vectors, one for each lane of a warp (-1: none): the head in lanes 0 .., the rest in lanes 16 ..
    __device__ __forceinline__ int loose(int lane) const {
        const int rest = head + full * kPer;
        return lane < head ? lane : lane >= 16 && rest + lane - 16 < vocab ? rest + lane - 16 : -1;
    }
    __device__ __forceinline__ float one(int v) const {
        if constexpr (T == kF32) return __ldg(reinterpret_cast<const float*>(at) + v);
        const uint16_t h = __ldg(reinterpret_cast<const uint16_t*>(at) + v);
        return T == kF16 ? h2f(h) : __uint_as_float((uint32_t)h << 16);
    }
    static __device__ __forceinline__ void values(uint4 v, float (&x)[kPer]) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (T == kF32) {
                x[i] = __uint_as_float(w[i]);
            } else if constexpr (T == kF16) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
                x[2 * i] = f.x;
                x[2 * i + 1] = f.y;
            } else {
                x[2 * i] = __uint_as_float(w[i] << 16);
                x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            }
        }
    }
};

// The largest of a vector's elements (NaN left out), in the elements' own type.
template <int T> __device__ __forceinline__ uint4 vector_max(uint4 a, uint4 b) {
    const uint32_t x[4] = {a.x, a.y, a.z, a.w}, y[4] = {b.x, b.y, b.z, b.w};
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (T == kF32) r[i] = __float_as_uint(fmaxf(__uint_as_float(x[i]), __uint_as_float(y[i])));
        else if constexpr (T == kF16) asm("max.f16x2 %0, %1, %2;" : "=r"(r[i]) : "r"(x[i]), "r"(y[i]));
        else asm("max.bf16x2 %0, %1, %2;" : "=r"(r[i]) : "r"(x[i]), "r"(y[i]));
    }
    return make_uint4(r[0], r[1], r[2], r[3]);
}

__constant__ double kPowers[64] = {  // 2^(i / 64)
    1.0, 1.0108892860517005, 1.0218971486541166, 1.0330248790212284,
    1.0442737824274138, 1.0556451783605572, 1.0671404006768237, 1.0787607977571199,
    1.0905077326652577, 1.1023825833078409, 1.1143867425958924, 1.1265216186082418,
    1.1387886347566916, 1.1511892299529827, 1.1637248587775775, 1.1763969916502812,
    1.189207115002721, 1.2021567314527031, 1.215247359980469, 1.22848053610687,
    1.241857812073484, 1.2553807570246911, 1.2690509571917332, 1.2828700160787783,
    1.2968395546510096, 1.3109612115247644, 1.3252366431597413, 1.3396675240533029,
    1.3542555469368927, 1.3690024229745905, 1.383909881963832, 1.3989796725383112,
    1.4142135623730951, 1.42961333839197, 1.4451808069770467, 1.460917794180647,
    1.4768261459394993, 1.4929077282912648, 1.5091644275934228, 1.5255981507445384,
    1.5422108254079407, 1.5590044002378369, 1.5759808451078865, 1.593142151342267,
    1.6104903319492543, 1.6280274218573478, 1.6457554781539649, 1.6636765803267364,
    1.681792830507429, 1.7001063537185235, 1.7186192981224779, 1.7373338352737062,
    1.7562521603732995, 1.7753764925265212, 1.7947090750031072, 1.8142521755003989,
    1.8340080864093424, 1.8539791250833855, 1.8741676341103, 1.8945759815869656,
    1.9152065613971474, 1.9360617934922943, 1.9571441241754002, 1.9784560263879509,
};

// The rule at one node.
struct Node {
    float m;             // the largest logit
    float c;             // log2 e / temperature
    float reach;         // weights of logits this far below the largest: less than kNothing
    float low;           // the next number below m - reach: logits that are not above it have no weight
    double floor;        // -reach, which they count as
    double inv;          // 1 / temperature
    double u64;          // 64 / (temperature ln 2)
    int hot;             // greedy: the lowest token with logit m
    bool greedy;
    __device__ __forceinline__ void most(float l) {
        m = l;
        low = __fsub_rd(l, reach);  // (so what is above it lies within reach, however far apart numbers of that size are)
    }
};
// exp((l - m) / temperature) in 64 bits, m finite; below kNothing where l is not above x.low or a NaN.  `table`: kPowers, one entry of
// 16 apart (each lane of half a warp has a copy in banks of its own: entries are read at random, and without copies that took as long
// as the rest).
constexpr double kNothing = 1e-290;
__device__ __forceinline__ double weight64(const Node& x, float l, const double* table) {
    constexpr double magic = 6755399441055744.0;  // 1.5 * 2^52: u + magic has u's nearest integer in its low bits
    constexpr double step = 0.010830424696249145;  // ln 2 / 64
    const double d = l > x.low ? (double)l - (double)x.m : x.floor, t = fma(d, x.u64, magic), r = fma(d, x.u64, magic - t);
    const int n = __double2loint(t);
    double p = fma(r, step * step * step / 6, step * step / 2);
    p = fma(p, r, step);
    const double base = table[(n & 63) * 16];
    p = fma(p * r, base, base);
    return __hiloint2double(__double2hiint(p) + (n >> 6) * (1 << 20), __double2loint(p));
}
// Any l, m.
__device__ __forceinline__ double weight_any(const Node& x, float l, int v, const double* table) {
    if (x.greedy) return v == x.hot ? 1.0 : 0.0;
    if (l == x.m) return 1.0;
    return x.m == INFINITY || !(l > x.low) ? 0.0 : weight64(x, l, table);
}

__device__ __forceinline__ double warp_add(double x) {
#pragma unroll
    for (int w = 16; w > 0; w >>= 1) x += __shfl_xor_sync(0xffffffffu, x, w);
    return x;
}
__device__ __forceinline__ float warp_max(float x) {
#pragma unroll
    for (int w = 16; w > 0; w >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, w));
    return x;
}
__device__ __forceinline__ double positive(double x) {  // max(x, 0)
    const int hi = __double2hiint(x), lo = __double2loint(x);
    return __hiloint2double(hi < 0 ? 0 : hi, hi < 0 ? 0 : lo);
}

// Of a slice of a row: the largest logit, the sum of weights below it, and the lowest token with it (where it is asked for).
struct __align__(16) Part {
    double sum;
    float most;
    int hot;
};

__device__ __forceinline__ void set_heat(Node& x, float heat) {
    x.greedy = heat == 0.0f;
    x.inv = x.greedy ? 0.0 : 1.0 / (double)heat;
    x.u64 = x.inv * 92.332482616893656;  // 64 / ln 2
    x.c = (float)fmin(x.inv * 1.4426950408889634, 3.0e38);
    x.reach = 680.0f * heat;
    x.floor = -680.0 * (double)heat;
}

// A slice of a row stays in registers between the pass for its maximum and the one for its sum.  (8 vectors each of 256 threads, 4 of
// 256, 8 of 128: within 1.5 us of one another at 151937 tokens.)
template <int T>
__global__ void __launch_bounds__(kSumThreads) verify_sums_kernel(const __grid_constant__ cvattn_verify_params p, Part* parts) {
    using R = Row<T>;
    constexpr int kPer = R::kPer;
    __shared__ float most[kSumWarps];
    __shared__ double sums[kSumWarps];
    __shared__ int hots[kSumWarps];
    __shared__ float factor;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int slice = blockIdx.x, node = blockIdx.y, s = blockIdx.z;
    griddep_wait();
    griddep_launch_dependents();
    if (p.n_nodes && node >= p.n_nodes[s]) return;
    const float heat = p.temperature ? p.temperature[s] : 1.0f;
    const R row(p.logits, s * p.logits_nb_seq + node * p.logits_nb_node, p.vocab);
    const int j0 = slice * kSlice + tid, j1 = min(row.full, (slice + 1) * kSlice);
    uint4 held[kHeld], top;
    top.x = top.y = top.z = top.w = T == kF32 ? 0xff800000u : T == kF16 ? 0xfc00fc00u : 0xff80ff80u;
#pragma unroll
    for (int k = 0; k < kHeld; ++k) {
        held[k] = top;
        if (j0 + k * kSumThreads < j1) held[k] = row.load(j0 + k * kSumThreads);
    }
    float alone = -INFINITY;
    int loose = -1;
    if (warp == 0 && slice == 0) {
        loose = row.loose(lane);
        if (loose >= 0) alone = row.one(loose);
    }
#pragma unroll
    for (int k = 0; k < kHeld; ++k) top = vector_max<T>(top, held[k]);
    float m = fmaxf(alone, -INFINITY);  // (a NaN counts as -infinity)
    {
        float l[kPer];
        R::values(top, l);
#pragma unroll
        for (int i = 0; i < kPer; ++i) m = fmaxf(m, l[i]);
    }
    m = warp_max(m);
    if (lane == 0) most[warp] = m;
    if (tid == 0) {
        Node x;
        set_heat(x, heat);
        factor = x.c;
    }
    __syncthreads();
    m = warp_max(most[lane % kSumWarps]);
    double sum = 0.0;
    int hot = INT32_MAX;
    if (m == -INFINITY) {
    } else if (heat == 0.0f || m == INFINITY) {
        int same = 0;
#pragma unroll
        for (int k = 0; k < kHeld; ++k) {
            float l[kPer];
            R::values(held[k], l);
#pragma unroll
            for (int i = 0; i < kPer; ++i)
                if (l[i] == m) {
                    ++same;
                    hot = min(hot, row.first(j0 + k * kSumThreads) + i);
                }
        }
        if (loose >= 0 && alone == m) {
            ++same;
            hot = min(hot, loose);
        }
        sum = same;
        hot = __reduce_min_sync(0xffffffffu, hot);
    } else {
        const float c = factor;
        const float2 m2 = make_float2(-m, -m), c2 = make_float2(c, c), one = make_float2(1.0f, 1.0f);
        auto add = [&](uint4 v) {
            float l[kPer];
            R::values(v, l);
            float2 part = make_float2(0.f, 0.f);
#pragma unroll
            for (int i = 0; i < kPer; i += 2) {
                const float2 d = ffma2(make_float2(l[i], l[i + 1]), one, m2), u = ffma2(d, c2, make_float2(0.f, 0.f));
                part = ffma2(make_float2(fast_exp2(u.x), fast_exp2(u.y)), one, part);
            }
            float w = part.x + part.y;
            if (w != w) {  // NaN among them: they have no weight
                w = 0.0f;
#pragma unroll
                for (int i = 0; i < kPer; ++i) w += l[i] == l[i] ? fast_exp2((l[i] - m) * c) : 0.0f;
            }
            sum += w;
        };
#pragma unroll
        for (int k = 0; k < kHeld; ++k)
            if (j0 + k * kSumThreads < j1) add(held[k]);
        if (loose >= 0 && alone == alone) sum += fast_exp2((alone - m) * c);
    }
    sum = warp_add(sum);
    if (lane == 0) {
        sums[warp] = sum;
        hots[warp] = hot;
    }
    __syncthreads();
    if (tid == 0) {
        Part out{0.0, m, INT32_MAX};
#pragma unroll
        for (int w = 0; w < kSumWarps; ++w) {
            out.sum += sums[w];
            out.hot = min(out.hot, hots[w]);
        }
        parts[((int64_t)s * p.max_nodes + node) * gridDim.x + slice] = out;
    }
}

struct Shared {
    double table[64 * 16];
    double W[kMaxNodes];                     // of each node: sum of weights,
    float m[kMaxNodes];                      // largest logit,
    int hot[kMaxNodes];                      // lowest token with it
    int path[kMaxNodes];                     // accepted nodes, from 1 on
    float last_logit;                        // of the token that follows
    bool stands[kMaxNodes];                  // whether a draft stands where none was refused before it
    double inv_left[kMaxNodes];              // 1 / the sum of p after each refusal
    double post_sum[2][kMaxCluster], post_b[2][kMaxCluster], post_w[2][kMaxCluster];  // of the cluster's CTAs, in turn of two
    int post_found[2][kMaxCluster], post_last[2][kMaxCluster];
    int gone[kMaxNodes];                     // tokens refused
    int parent[kMaxNodes], token[kMaxNodes], first_child[kMaxNodes];
    float u[kMaxNodes];
    float logit[kMaxNodes], prob[kMaxNodes]; // of the drafts' tokens at their parents
    double weight[kMaxNodes];                // what() of them there, before any refusal
    int bad;
    double warp_w[kWarps];
    // what warp 0 has decided
    int what, at, refused, first;
    double inv_W;
};
enum { kScan = 1, kFollow = 2, kStop = 3 };  // Shared::what

template <int T>
__global__ void __launch_bounds__(kThreads, 1) verify_walk_kernel(const __grid_constant__ cvattn_verify_params p, const Part* parts,
                                                                  int n_slices, int n_tiles, int* status) {
    using R = Row<T>;
    constexpr int kPer = R::kPer;
    __shared__ Shared sh;
    extern __shared__ double tile_sum[];
    double* tile_b = tile_sum + n_tiles + 2;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    uint32_t C, rank;
    asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(C));
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    const int s = blockIdx.x / C;
    // (shared memory of another CTA may be written once it is known to have started: all wait for this before the first exchange)
    if (C > 1) cluster_arrive_relaxed();
    for (int i = tid; i < 64 * 16; i += kThreads) sh.table[i] = kPowers[i >> 4];
    const double* table = sh.table + (tid & 15);
    if (tid == 0) sh.bad = 0;
    __syncthreads();
    griddep_wait();
    const int n = p.n_nodes ? p.n_nodes[s] : p.max_nodes;
    const float heat = p.temperature ? p.temperature[s] : 1.0f;
    int32_t* accepted = p.accepted + s * p.accepted_stride;
    float* logs = p.log_probs ? p.log_probs + (int64_t)s * p.max_nodes : nullptr;
    const bool refused_all = n < 0 || n > p.max_nodes || !(heat >= 0.0f && heat < INFINITY);
    const auto row_of = [&](int node) { return R(p.logits, s * p.logits_nb_seq + node * p.logits_nb_node, p.vocab); };
    static_assert(kThreads == 2 * kMaxNodes, "a thread a node, and as many for their sums");
    if (const int i = tid; i < kMaxNodes) {
        sh.first_child[i] = kMaxNodes;
        if (i < (refused_all ? 0 : n)) {
            const int up = i == 0 ? -1 : p.parents ? p.parents[s * p.parents_nb_seq + i] : i - 1;
            const int t = p.tokens[(int64_t)s * p.max_nodes + i];
            sh.parent[i] = up;
            sh.token[i] = t;
            sh.u[i] = p.accept_u[(int64_t)s * p.max_nodes + i];
            if (i > 0) {
                if (up < 0 || up >= i || (uint32_t)t >= (uint32_t)p.vocab) {
                    sh.bad = 1;
                } else {
                    sh.logit[i] = row_of(up).one(t);
                    sh.prob[i] = p.draft_probs ? __ldg(p.draft_probs + s * p.probs_nb_seq + up * p.probs_nb_node + t) : 1.0f;
                }
            }
        }
    }
    Node x;
    set_heat(x, heat);
    // the other warps, one a node: its numbers from all slices
    if (!refused_all && tid >= kMaxNodes)
        for (int i = warp - kWarps / 2; i < n; i += kWarps / 2) {
            const Part* of = parts + ((int64_t)s * p.max_nodes + i) * n_slices;
            Part q{0.0, -INFINITY, INT32_MAX};
            for (int k = lane; k < n_slices; k += 32) {
                const Part v = of[k];
                if (v.most > q.most) {
                    x.most(v.most);
                    q.sum = v.sum + (q.sum > 0.0 && !x.greedy && v.most < INFINITY ? q.sum * weight64(x, q.most, table) : 0.0);
                    q.hot = v.hot;
                    q.most = v.most;
                } else if (v.most > -INFINITY) {
                    x.most(q.most);
                    q.sum += v.most == q.most ? v.sum : x.greedy || q.most == INFINITY ? 0.0 : v.sum * weight64(x, v.most, table);
                    if (v.most == q.most) q.hot = min(q.hot, v.hot);
                }
            }
            const float top = warp_max(q.most);
            x.most(top);
            double w = q.most == top ? 1.0 : 0.0;
            if (!x.greedy && top < INFINITY && q.most > -INFINITY && q.most < top) w = weight64(x, q.most, table);
            const double sum = warp_add(q.sum * w);
            const int hot = __reduce_min_sync(0xffffffffu, q.most == top ? q.hot : INT32_MAX);
            if (lane == 0) {
                sh.m[i] = top;
                sh.W[i] = x.greedy ? 1.0 : sum;
                sh.hot[i] = hot;
            }
        }
    if (rank == 0)
        for (int i = tid; i < p.max_nodes; i += kThreads) {
            accepted[i] = -1;
            if (logs) logs[i] = 0.0f;
        }
    __syncthreads();
    if (C > 1) cluster_wait();
    if (refused_all || sh.bad || n == 0) {
        if (rank == 0 && tid == 0) {
            if (refused_all || sh.bad) record_status(status, kStatusBadDraft);
            p.n_accepted[s] = 0;
            p.next_token[s] = -1;
        }
        return;  // (every CTA of the cluster alike)
    }
    for (int i = 1 + tid; i < n; i += kThreads) {
        const int up = sh.parent[i];
        atomicMin(&sh.first_child[up], i);
        x.most(sh.m[up]);
        x.hot = sh.hot[up];
        sh.weight[i] = weight_any(x, sh.logit[i], sh.token[i], table);
        sh.prob[i] = fmaxf(sh.prob[i], 0.0f);  // (NaN: 0)
        sh.stands[i] = (double)sh.u[i] * (double)sh.prob[i] * sh.W[up] < sh.weight[i];
    }
    __syncthreads();

    // Warp 0 posts this CTA's numbers to the slots of all CTAs, in turn of two: one is written while the other may still be
    // read.  Then every thread arrives.
    int turn = 0;
    auto exchange = [&](double sum, double sum_b, double sum_w, int found, int last) {
        if (tid < (int)C) {
            uint32_t a, b, c, d, e;
            asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_addr(&sh.post_sum[turn][rank])), "r"(tid));
            asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(b) : "r"(smem_addr(&sh.post_found[turn][rank])), "r"(tid));
            asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(c) : "r"(smem_addr(&sh.post_last[turn][rank])), "r"(tid));
            asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(d) : "r"(smem_addr(&sh.post_b[turn][rank])), "r"(tid));
            asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(e) : "r"(smem_addr(&sh.post_w[turn][rank])), "r"(tid));
            asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(a), "d"(sum) : "memory");
            asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(d), "d"(sum_b) : "memory");
            asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(e), "d"(sum_w) : "memory");
            asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(b), "r"(found) : "memory");
            asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(c), "r"(last) : "memory");
        }
        __syncwarp();
        if (warp == 0) cluster_arrive();
        else cluster_arrive_relaxed();  // (they have posted nothing)
        cluster_wait();
    };

    int at = 0, count = 1, token = -1, refused = 0;
    double inv_W = 0.0;
    R row = row_of(0);
    const float* q = nullptr;
    bool simple = false;
    // this CTA's vectors, tiles of 32 each, in order
    const int j0 = (int)rank * n_tiles * 32;
    int j1 = 0, tiles = 0;
    auto arrive_at = [&](int node) {
        at = node;
        row = row_of(node);
        q = p.draft_probs ? p.draft_probs + s * p.probs_nb_seq + node * p.probs_nb_node : nullptr;
        x.most(sh.m[node]);
        x.hot = sh.hot[node];
        simple = !x.greedy && x.m != INFINITY;
        j1 = min(j0 + n_tiles * 32, row.full);
        tiles = (j1 > j0 ? (j1 - j0 + 31) / 32 : 0) + 2;
    };
    // One token's part of p after the refusals so far, times its sum.  Weights stay as they are until the first subtraction, so
    // that equal ones add up exactly.
    auto less = [&](double w, float qv) {
        const double g = (double)fmaxf(qv, 0.0f);  // (NaN: 0)
        double r = positive(fma(w, inv_W, -g));
        if (refused > 1)
            for (int k = 1; k < refused; ++k) r = positive(fma(r, sh.inv_left[k - 1], -g));
        return r;
    };
    auto what = [&](double w, float qv, int v) {  // of a token of weight w
        if (!q)
            for (int k = 0; k < refused; ++k) w = v == sh.gone[k] ? 0.0 : w;
        else if (refused) w = less(w, qv);
        return w;
    };
    // A tile is one vector a lane: elements e, e + 1, ..  Tile 0 is the row's head (of the first CTA), the last one what its
    // vectors leave over (of the last CTA), an element a lane.
    struct Fetched {
        uint4 v;
        float g[kPer];
        int e;      // (-1: nothing)
    };
    auto fetch = [&](int t) {
        Fetched f;
        f.e = -1;
        if (t >= tiles) return f;
        if (t == 0 || t == tiles - 1) {
            const int e = row.loose(lane);
            if (e >= 0 && (t == 0 ? rank == 0 && lane < 16 : rank == C - 1 && lane >= 16)) {
                f.e = e;
                f.v.x = __float_as_uint(row.one(e));
                f.g[0] = q && refused ? __ldg(q + e) : 0.0f;
            }
            return f;
        }
        const int j = j0 + 32 * (t - 1) + lane;
        if (j < j1) {
            f.e = row.first(j);
            f.v = row.load(j);
            if (q && refused) {
#pragma unroll
                for (int i = 0; i < kPer; ++i) f.g[i] = __ldg(q + f.e + i);
            }
        }
        return f;
    };
    auto weigh = [&](int t, const Fetched& f, double (&w)[kPer]) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) w[i] = 0.0;
        if (f.e < 0) return;
        if (t == 0 || t == tiles - 1) {
            w[0] = what(weight_any(x, __uint_as_float(f.v.x), f.e, table), f.g[0], f.e);
            return;
        }
        float l[kPer];
        R::values(f.v, l);
        if (simple) {
#pragma unroll
            for (int i = 0; i < kPer; ++i) w[i] = weight64(x, l[i], table);
        } else {
#pragma unroll
            for (int i = 0; i < kPer; ++i) w[i] = (x.greedy ? f.e + i == x.hot : l[i] == x.m) ? 1.0 : 0.0;
        }
        if (!q)
            for (int k = 0; k < refused; ++k) {
                const int off = sh.gone[k] - f.e;
#pragma unroll
                for (int i = 0; i < kPer; ++i) w[i] = off == i ? 0.0 : w[i];
            }
        if (q && refused) {
#pragma unroll
            for (int i = 0; i < kPer; ++i) w[i] = positive(fma(w[i], inv_W, -(double)fmaxf(f.g[i], 0.0f)));
#pragma unroll 1
            for (int k = 1; k < refused; ++k) {
                const double by = sh.inv_left[k - 1];
#pragma unroll
                for (int i = 0; i < kPer; ++i) w[i] = positive(fma(w[i], by, -(double)fmaxf(f.g[i], 0.0f)));
            }
        }
    };
    // The first refusal against draft probabilities, in one scan: W, which the subtraction takes, is known to 1e-7 only (W~).  With S
    // the tokens of which W~ leaves something,  sum_S (w / W - q) = R + (R + B) (W~ / W - 1),  R = sum_S (w / W~ - q),  B = sum_S q.
    // (A token that the exact W would put on the other side of S has a part below 1e-7 of its own weight.)
    auto weigh_first = [&](int t, const Fetched& f, double& R1, float& B1, double& W1) {
        if (f.e < 0) return;
        if (t == 0 || t == tiles - 1) {
            const double w = weight_any(x, __uint_as_float(f.v.x), f.e, table), r = fma(w, inv_W, -(double)fmaxf(f.g[0], 0.0f));
            W1 += w;
            R1 += positive(r);
            if (r > 0.0) B1 += fmaxf(f.g[0], 0.0f);
            return;
        }
        float l[kPer];
        R::values(f.v, l);
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const double w = weight64(x, l[i], table);
            const float g = fmaxf(f.g[i], 0.0f);
            const double r = fma(w, inv_W, -(double)g);
            W1 += w;
            R1 += positive(r);
            B1 += __double2hiint(r) < 0 ? 0.0f : g;
        }
    };
    double before = 0.0, all = 0.0;    // what() over the CTAs before this one, over the vocabulary (warp 0)
    double total = 0.0, was = 0.0;     // warp 0: what()'s sum over the vocabulary, and before the last refusal
    bool known = true, exact = false;  // warp 0: whether total is that sum; whether of 64-bit weights
    bool scanned = false, first = false;
    int c = 0, order = kStop;
    auto enter = [&](int node) {       // warp 0
        at = node;
        refused = 0;
        total = sh.W[node];
        exact = x.greedy || sh.m[node] == INFINITY;
        known = true;
        c = sh.first_child[node];
    };
    if (warp == 0) enter(0);
    q = p.draft_probs;  // (whether there are any)
    for (;;) {
        if (warp == 0) {
            if (scanned) {
                known = exact = true;
                if (refused && !(all > kNothing)) {  // the last refusal left nothing: as it was
                    --refused;
                    total = was;
                    scanned = false;
                } else {
                    if (q && refused && lane == 0) sh.inv_left[refused - 1] = 1.0 / all;
                    __syncwarp();
                    total = all;
                }
            }
            order = scanned && c >= n ? kFollow : kScan;
            // first drafts that stand, one below the other
            if (!scanned) {
                bool moved = false;
                while (c < n && sh.stands[c] && sh.m[at] != -INFINITY && refused == 0) {
                    if (lane == 0) {
                        if (rank == 0) accepted[count] = c;
                        sh.path[count] = c;
                    }
                    ++count;
                    at = c;
                    c = sh.first_child[c];
                    moved = true;
                }
                if (moved) enter(at);
            }
            // drafts in turn, as long as the sum of what is left is known
            while (order == kScan) {
                if (sh.m[at] == -INFINITY) order = kStop;  // no weight anywhere
                while (c < n && sh.parent[c] != at) ++c;
                if (order == kStop || c >= n || !known) break;
                const int t = sh.token[c];
                const double pt = what(sh.weight[c], sh.prob[c], t);
                if ((double)sh.u[c] * (double)sh.prob[c] * total < pt) {
                    if (lane == 0) {
                        if (rank == 0) accepted[count] = c;
                        sh.path[count] = c;
                    }
                    ++count;
                    enter(c);
                    continue;
                }
                if (q && refused == 0) {
                    inv_W = 1.0 / total;
                    first = !exact;  // (the subtraction takes a sum of exact weights)
                }
                if (lane == 0) sh.gone[refused] = t;
                __syncwarp();
                ++refused;
                for (++c; c < n && sh.parent[c] != at;) ++c;
                was = total;
                if (q) {
                    known = false;
                } else {  // (where too little is left for a difference of such sums, they are added up anew)
                    total -= pt;
                    known = total > was * (exact ? 0x1p-10 : 0.25);
                }
            }
            if (lane == 0) {
                sh.what = order;
                sh.at = at;
                sh.refused = refused;
                sh.first = first;
                sh.inv_W = inv_W;
            }
        }
        __syncthreads();
        order = sh.what;
        if (order != kScan) break;
        arrive_at(sh.at);
        refused = sh.refused;
        first = sh.first;
        inv_W = sh.inv_W;
        // sums of tiles, of this CTA in the tiles' order, of the cluster
        double my_w = 0.0;
        Fetched f = fetch(warp);
#pragma unroll 1
        for (int t = warp; t < tiles; t += kWarps) {
            const Fetched next = fetch(t + kWarps);
            double sum = 0.0;
            if (first) {
                float b = 0.0f;
                weigh_first(t, f, sum, b, my_w);
                const double all_b = warp_add((double)b);
                if (lane == 0) tile_b[t] = all_b;
            } else {
                double w[kPer];
                weigh(t, f, w);
#pragma unroll
                for (int i = 0; i < kPer; ++i) sum += w[i];
            }
            f = next;
            sum = warp_add(sum);
            if (lane == 0) tile_sum[t] = sum;
        }
        if (first) {
            my_w = warp_add(my_w);
            if (lane == 0) sh.warp_w[warp] = my_w;
        }
        __syncthreads();
        if (warp == 0) {
            double sum = 0.0, sum_b = 0.0, sum_w = 0.0;
            for (int t = lane; t < tiles; t += 32) {
                sum += tile_sum[t];
                if (first) sum_b += tile_b[t];
            }
            all = warp_add(sum);
            if (first) {
                sum_b = warp_add(sum_b);
                sum_w = warp_add(lane < kWarps ? sh.warp_w[lane] : 0.0);
            }
            before = 0.0;
            double lead = 0.0;  // W~ / W - 1
            if (C == 1 && first) lead = 1.0 / (inv_W * sum_w) - 1.0;
            if (C > 1) exchange(all, sum_b, sum_w, 0, 0);
            if (C > 1) {
                const bool has = lane < (int)C;
                const double v = has ? sh.post_sum[turn][lane] : 0.0, v_b = has ? sh.post_b[turn][lane] : 0.0;
                if (first) {
                    sum_w = warp_add(has ? sh.post_w[turn][lane] : 0.0);
                    lead = 1.0 / (inv_W * sum_w) - 1.0;
                }
                const double u = first ? fma(v + v_b, lead, v) : v;
                before = warp_add(lane < (int)rank ? u : 0.0);
                all = warp_add(u);
            } else if (first) {
                all = fma(all + sum_b, lead, all);
            }
            if (first) {
                inv_W = 1.0 / sum_w;
                was = sum_w;
                for (int t = lane; t < tiles; t += 32) tile_sum[t] = fma(tile_sum[t] + tile_b[t], lead, tile_sum[t]);
                __syncwarp();
                first = false;
            }
        } else if (C > 1) {
            exchange(0.0, 0.0, 0.0, 0, 0);
        }
        turn ^= C > 1;
        scanned = true;
    }
    if (order == kFollow) {
        // The token that follows: the first tile whose end passes the target, and the last that has any weight (for a target
        // that rounding keeps out of reach); then its elements in order.
        int found = INT32_MAX, last = -1;
        if (warp == 0) {
            const double target = (double)p.sample_u[s] * all;
            int first = INT32_MAX, some_tile = -1;
            double run0 = before, start = 0.0;
            for (int t = 0; t < tiles && first == INT32_MAX; t += 32) {
                const double v = t + lane < tiles ? tile_sum[t + lane] : 0.0;
                double y = v;
#pragma unroll
                for (int w = 1; w < 32; w <<= 1) {
                    const double z = __shfl_up_sync(0xffffffffu, y, w);
                    if (lane >= w) y += z;
                }
                const uint32_t over = __ballot_sync(0xffffffffu, t + lane < tiles && run0 + y > target && v > kNothing);
                const uint32_t some = __ballot_sync(0xffffffffu, t + lane < tiles && v > kNothing);
                if (some) some_tile = t + 31 - __clz(some);
                if (over) {
                    const int k = __ffs(over) - 1;
                    first = t + k;
                    start = run0 + __shfl_sync(0xffffffffu, y - v, k);
                }
                run0 += __shfl_sync(0xffffffffu, y, 31);
            }
            const bool out_of_reach = first == INT32_MAX;
            const int t = out_of_reach ? some_tile : first;
            if (t >= 0) {
                const Fetched f = fetch(t);
                double w[kPer], sum = 0.0;
                weigh(t, f, w);
#pragma unroll
                for (int i = 0; i < kPer; ++i) sum += w[i];
                double y = sum;
#pragma unroll
                for (int k = 1; k < 32; k <<= 1) {
                    const double z = __shfl_up_sync(0xffffffffu, y, k);
                    if (lane >= k) y += z;
                }
                double run1 = start + (y - sum);
#pragma unroll
                for (int i = 0; i < kPer; ++i) {
                    run1 += w[i];
                    if (w[i] > kNothing) {
                        last = f.e + i;
                        if (run1 > target && found == INT32_MAX) found = f.e + i;
                    }
                }
                found = __reduce_min_sync(0xffffffffu, found);
                last = __reduce_max_sync(0xffffffffu, last);
                // (a tile whose sum passes the target while its elements, added in another order, do not: its last one)
                if (!out_of_reach && found == INT32_MAX) found = last;
                if (out_of_reach) found = INT32_MAX;
            }
        }
        if (C > 1) {
            exchange(0.0, 0.0, 0.0, found, last);
            if (warp == 0) {
                found = __reduce_min_sync(0xffffffffu, lane < (int)C ? sh.post_found[turn][lane] : INT32_MAX);
                last = __reduce_max_sync(0xffffffffu, lane < (int)C ? sh.post_last[turn][lane] : -1);
            }
        }
        if (warp == 0) {
            token = found == INT32_MAX ? last : found;
            if (lane == 0 && token >= 0) sh.last_logit = row.one(token);
        }
    }
    griddep_launch_dependents();
    if (rank == 0 && warp == 0) {
        __syncwarp();
        if (logs)
            for (int i = lane; i < count - (token < 0); i += 32) {  // of path[i + 1] at path[i], of the following token at the last
                const int from = i == 0 ? 0 : sh.path[i];
                const float l = i + 1 < count ? sh.logit[sh.path[i + 1]] : sh.last_logit, m = sh.m[from];
                logs[i] = (float)((x.greedy || l == m ? 0.0 : ((double)l - (double)m) * x.inv) - log(sh.W[from]));
            }
        if (lane == 0) {
            accepted[0] = 0;
            p.n_accepted[s] = count;
            p.next_token[s] = token;
        }
    }
    if (C > 1) {  // nobody leaves while others may post to it
        __syncwarp();
        cluster_arrive();
        cluster_wait();
    }
}

// CTAs per sequence of the walk: two tiles a warp at least, and one a SM; more where shared memory would not hold the tiles' sums.
static int cluster_of(int n_seq, int vectors) {
    int c = 1;
    while (c < kMaxCluster && vectors > c * 2 * kThreads && n_seq * c * 2 <= 148) c *= 2;
    while (c < kMaxCluster && vectors > c * kMaxTiles * 32) c *= 2;
    return c;
}

static int slices_of(int vocab, int per) { return vocab / per / kSlice + 1; }

template <int T> static cudaError_t launch_for(cudaStream_t stream, const cvattn_verify_params& p, int* status) {
    constexpr int per = Row<T>::kPer;
    Part* parts = static_cast<Part*>(p.workspace);
    const int slices = slices_of(p.vocab, per);
    cudaError_t e = cudaFuncSetAttribute(verify_walk_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (kMaxTiles + 2) * 16);
    if (e != cudaSuccess) return e;
    e = launch_overlapped(verify_sums_kernel<T>, dim3((unsigned)slices, (unsigned)p.max_nodes, (unsigned)p.n_seq), kSumThreads,
                                            0, stream, p, parts);
    if (e != cudaSuccess) return e;
    const int vectors = p.vocab / per, c = cluster_of(p.n_seq, vectors), tiles = (vectors + 32 * c - 1) / (32 * c);
    return launch_overlapped_clusters(verify_walk_kernel<T>, dim3((unsigned)(p.n_seq * c)), kThreads, (size_t)(tiles + 2) * 16, c, stream, p,
                                      (const Part*)parts, slices, tiles, status);
}

}  // namespace verify

// The longest vocabulary: a cluster's tiles of f32 vectors.
int verify_most_vocab() { return verify::kMaxCluster * verify::kMaxTiles * 32 * 4; }

size_t verify_workspace_bytes(int n_seq, int max_nodes, int vocab) {
    return (size_t)n_seq * max_nodes * verify::slices_of(vocab, 4) * sizeof(verify::Part);
}

cudaError_t launch_verify(cudaStream_t stream, const cvattn_verify_params& p, int* status) {
    using namespace verify;
    switch (p.logits_type) {
    case kF32: return launch_for<kF32>(stream, p, status);
    case kF16: return launch_for<kF16>(stream, p, status);
    default: return launch_for<kBF16>(stream, p, status);
    }
}

}  // namespace cvattn
