// verify.cu -- drafted tokens against the target's logits, with given random numbers.
#include <cuda_bf16.h>

#include "launch.cuh"
#include "common.cuh"
#include "internal.h"

namespace cvattn {
namespace verify {

constexpr int kThreads = 1024;
constexpr int kBF16 = CVATTN_TYPE_BF16;

template <int T> __device__ __forceinline__ float logit(const void* row, int v) {
    float x;
    if constexpr (T == kF32) x = static_cast<const float*>(row)[v];
    else if constexpr (T == kF16) x = __half2float(static_cast<const __half*>(row)[v]);
    else x = __bfloat162float(static_cast<const __nv_bfloat16*>(row)[v]);
    return isnan(x) ? -INFINITY : x;
}

// The target at one node: weight(v) = exp((logit - m) / temperature), their sum W.
struct Node {
    const void* row;
    const float* q;      // the drafts' probabilities there, or null
    float m;
    int hot;             // the lowest token with logit m
    double inv, W;       // 1 / temperature (0: greedy)
};
template <int T> __device__ __forceinline__ double weight(const Node& x, bool greedy, int v) {
    if (greedy) return v == x.hot ? 1.0 : 0.0;
    const float l = logit<T>(x.row, v);
    if (l == x.m) return 1.0;
    if (l == -INFINITY || x.m == INFINITY) return 0.0;
    return exp(((double)l - (double)x.m) * x.inv);
}
__device__ __forceinline__ float sane(float q) { return q > 0.0f ? q : 0.0f; }

template <class X, class F> __device__ X block_reduce(X x, F join, X* tmp) {
    for (int w = 16; w > 0; w >>= 1) x = join(x, __shfl_xor_sync(0xffffffffu, x, w));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) tmp[threadIdx.x >> 5] = x;
    __syncthreads();
    X y = tmp[0];
    for (int w = 1; w < kThreads / 32; ++w) y = join(y, tmp[w]);
    return y;
}

template <int T>
__global__ void __launch_bounds__(kThreads) verify_kernel(const __grid_constant__ cvattn_verify_params p, int* status) {
    griddep_wait();
    __shared__ double tmp[kThreads / 32];
    __shared__ float tmpf[kThreads / 32];
    __shared__ int tmpi[kThreads / 32];
    __shared__ double left_sum[CVATTN_TREE_MAX_NODES];  // of p after each refusal
    __shared__ int gone[CVATTN_TREE_MAX_NODES];         // tokens refused
    __shared__ int bad;
    const int s = blockIdx.x, tid = threadIdx.x;
    const int n = p.n_nodes ? p.n_nodes[s] : p.max_nodes;
    const float heat = p.temperature ? p.temperature[s] : 1.0f;
    const bool greedy = heat == 0.0f;
    const int32_t* tokens = p.tokens + (int64_t)s * p.max_nodes;
    const int32_t* parents = p.parents ? p.parents + s * p.parents_nb_seq : nullptr;
    const float* u = p.accept_u + (int64_t)s * p.max_nodes;
    int32_t* accepted = p.accepted + s * p.accepted_stride;
    float* logs = p.log_probs ? p.log_probs + (int64_t)s * p.max_nodes : nullptr;
    if (tid == 0) bad = n < 0 || n > p.max_nodes || !(heat >= 0.0f);
    __syncthreads();
    if (!bad)
        for (int i = 1 + tid; i < n; i += kThreads) {
            const int up = parents ? parents[i] : i - 1;
            if (up < 0 || up >= i || (uint32_t)tokens[i] >= (uint32_t)p.vocab) bad = 1;
        }
    __syncthreads();
    if (bad && tid == 0) record_status(status, kStatusBadDraft);
    for (int i = tid; i < p.max_nodes; i += kThreads) {
        accepted[i] = -1;
        if (logs) logs[i] = 0.0f;
    }
    __syncthreads();
    if (bad || n == 0) {
        if (tid == 0) {
            p.n_accepted[s] = 0;
            p.next_token[s] = -1;
        }
        return;
    }
    const auto add = [](double a, double b) { return a + b; };
    const int chunk = (p.vocab + kThreads - 1) / kThreads;
    const int v0 = min(p.vocab, tid * chunk), v1 = min(p.vocab, v0 + chunk);
    int at = 0, count = 1, token = -1;
    if (tid == 0) accepted[0] = 0;
    for (;;) {
        Node x;
        const int size = T == kF32 ? 4 : 2;
        x.row = static_cast<const uint8_t*>(p.logits) + (s * p.logits_nb_seq + at * p.logits_nb_node) * size;
        x.q = p.draft_probs ? p.draft_probs + s * p.probs_nb_seq + at * p.probs_nb_node : nullptr;
        x.inv = greedy ? 0.0 : 1.0 / (double)heat;
        float m = -INFINITY;
        for (int v = tid; v < p.vocab; v += kThreads) m = fmaxf(m, logit<T>(x.row, v));
        x.m = block_reduce(m, [](float a, float b) { return fmaxf(a, b); }, tmpf);
        if (x.m == -INFINITY) break;  // no weight anywhere
        int hot = INT32_MAX;
        for (int v = tid; v < p.vocab; v += kThreads)
            if (logit<T>(x.row, v) == x.m) hot = min(hot, v);
        x.hot = block_reduce(hot, [](int a, int b) { return min(a, b); }, tmpi);
        double w = 0.0;
        for (int v = tid; v < p.vocab; v += kThreads) w += weight<T>(x, greedy, v);
        x.W = block_reduce(w, add, tmp);
        int refused = 0;
        double total = x.W;  // of left(v)
        // p(v) after the refusals so far, times total: weights as they are until the first subtraction, so that equal ones add up exactly
        auto left = [&](int v) {
            double r = weight<T>(x, greedy, v);
            if (!x.q) {
                for (int k = 0; k < refused; ++k)
                    if (v == gone[k]) r = 0.0;
                return r;
            }
            if (refused) r /= x.W;
            for (int k = 0; k < refused; ++k) r = fmax(r - (double)sane(x.q[v]), 0.0) / left_sum[k];
            return r;
        };
        int down = -1;
        for (int c = at + 1; c < n; ++c) {
            if ((parents ? parents[c] : c - 1) != at) continue;
            const int t = tokens[c];
            const double pt = left(t), qt = x.q ? (double)sane(x.q[t]) : 1.0;
            if ((double)u[c] * qt * total < pt) {
                down = c;
                break;
            }
            double sum = 0.0;
            for (int v = tid; v < p.vocab; v += kThreads) {
                const double r = left(v);
                sum += x.q ? fmax(r / total - (double)sane(x.q[v]), 0.0) : v == t ? 0.0 : r;
            }
            sum = block_reduce(sum, add, tmp);
            if (sum > 0.0) {
                __syncthreads();
                if (tid == 0) {
                    left_sum[refused] = sum;
                    gone[refused] = t;
                }
                __syncthreads();
                ++refused;
                total = x.q ? 1.0 : sum;
            }
        }
        auto log_p = [&](int v) { return greedy ? 0.0f : (float)(log(weight<T>(x, greedy, v)) - log(x.W)); };
        if (down >= 0) {
            if (tid == 0) {
                accepted[count] = down;
                if (logs) logs[count - 1] = log_p(tokens[down]);
            }
            at = down;
            ++count;
            continue;
        }
        // the token that follows
        __shared__ double before[kThreads];
        __shared__ int found;
        double sum = 0.0;
        for (int v = v0; v < v1; ++v) sum += left(v);
        before[tid] = sum;
        if (tid == 0) found = -1;
        __syncthreads();
        if (tid == 0) {
            double all = 0.0;
            for (int i = 0; i < kThreads; ++i) {
                const double b = before[i];
                before[i] = all;
                all += b;
            }
            tmp[0] = all;
        }
        __syncthreads();
        const double target = (double)p.sample_u[s] * tmp[0];
        double c = before[tid];
        int mine = -1, last = -1;
        for (int v = v0; v < v1; ++v) {
            const double r = left(v);
            if (r > 0.0) last = v;
            c += r;
            if (mine < 0 && c > target) mine = v;
        }
        const int lowest = block_reduce(mine < 0 ? INT32_MAX : mine, [](int a, int b) { return min(a, b); }, tmpi);
        last = block_reduce(last, [](int a, int b) { return max(a, b); }, tmpi);
        token = lowest == INT32_MAX ? last : lowest;
        if (tid == 0 && logs && token >= 0) logs[count - 1] = log_p(token);
        break;
    }
    if (tid == 0) {
        p.n_accepted[s] = count;
        p.next_token[s] = token;
    }
}

}  // namespace verify

size_t verify_workspace_bytes(int n_seq, int max_nodes, int vocab) { return 0; }

cudaError_t launch_verify(cudaStream_t stream, const cvattn_verify_params& p, int* status) {
    using namespace verify;
    auto* fn = p.logits_type == kF32 ? verify_kernel<kF32> : p.logits_type == kF16 ? verify_kernel<kF16> : verify_kernel<kBF16>;
    return launch_overlapped(fn, (unsigned)p.n_seq, kThreads, 0, stream, p, status);
}

}  // namespace cvattn
