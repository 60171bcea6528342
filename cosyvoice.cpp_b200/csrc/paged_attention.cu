// paged_attention.cu -- the join of splits and the host side of attention over a paged 8-bit cache.
#include "launch.cuh"
#include "paged_tc.cuh"

namespace cvattn {
namespace paged {

// --------------------------------------------------------------- combine --
//
// 16 threads (4 dims each) follow every kLanes-th split of a row; the partial sums are joined in order.  Bound by latency: about
// 2 us behind the kernel before it, whose parts are in L2.
template <int kLanes>
__global__ void __launch_bounds__(256) paged_combine_kernel(const __grid_constant__ AttArgs a) {
    constexpr int kPer = 16 / kLanes;  // rows per CTA
    __shared__ float4 so[16][16];
    __shared__ float2 sml[16];
    griddep_wait();
    const int unit = threadIdx.x >> 4, c = threadIdx.x & 15, lane = unit % kLanes;
    const int all_rows = a.p.max_q * a.G;
    const int r = blockIdx.x * kPer + unit / kLanes, kvh = blockIdx.y, s = blockIdx.z;
    Join j;
    if (r < all_rows) {
        const int64_t slot = ((int64_t)s * a.p.pool.n_heads + kvh) * a.n_splits * all_rows + r;
        for (int k0 = lane; k0 < a.n_splits; k0 += 4 * kLanes) {
            float2 ml[4];
            float4 v[4];
            float top = j.M;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int k = k0 + u * kLanes;
                ml[u] = make_float2(-INFINITY, 0.0f);
                if (k < a.n_splits) {
                    ml[u] = *reinterpret_cast<const float2*>(a.ws_ml + (slot + (int64_t)k * all_rows) * 2);
                    v[u] = *reinterpret_cast<const float4*>(a.ws_o + (slot + (int64_t)k * all_rows) * kD + c * 4);
                }
                top = fmaxf(top, ml[u].x);
            }
            if (top == -INFINITY) continue;
            const float f = exp2f(j.M - top);
            j.M = top;
            j.l *= f;
            j.o.x *= f; j.o.y *= f; j.o.z *= f; j.o.w *= f;
#pragma unroll
            for (int u = 0; u < 4; ++u) j.add(ml[u], v[u]);
        }
    }
    if constexpr (kLanes > 1) {
        so[unit][c] = j.o;
        if (c == 0) sml[unit] = make_float2(j.M, j.l);
        __syncthreads();
        if (lane) return;
        j = Join();
#pragma unroll
        for (int k = 0; k < kLanes; ++k) j.M = fmaxf(j.M, sml[unit + k].x);
#pragma unroll
        for (int k = 0; k < kLanes; ++k) j.add(sml[unit + k], so[unit + k][c]);
    }
    if (r < all_rows) j.write(a, s, kvh, r, c);
}

// ------------------------------------------------------------------ host --

constexpr int kSms = 148;

static size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

// The tcgen05 kernel starts later (13 us in all for a single tile, where the other starts with 4), and a tile of its list costs the
// same whatever rows a unit (a sequence's tile of 128 rows for a KV head) has up to 128, a unit some more; the other's cost goes with
// rows times tiles of positions.  So: work, rows times tiles, against a constant and a share for each tile and unit.  The three numbers
// are fitted to these times, us of mma.sync | tcgen05, 14 / 2 heads, and pick the slower side of three: 1 of 65536 with 28 rows, and
// within 0.7 us 1 of 4096 with 112 and 16 of 1000 with 56.  1
// sequence of 4096, 112 rows of a KV head 16.8 | 16.1, 224 22.5 | 16.8; 1 of 65536, 14 rows 21.4 | 24.4, 28 29.9 | 25.6, 56
// 45.9 | 26.4; 4 of 2500, 56 16.8 | 17.4, 112 22.9 | 18.2; 16 of 1000, 56 19.7 | 19.3, 112 23.0 | 20.1; 16 of 8192, 28 32.5 |
// 36.1, 56 58 | 37; 64 of 1000, 28 19.7 | 27.1, 56 33.4 | 28.9; 64 of 4096, 28 49 | 56, 56 93 | 59; 256 of 500, 56 47 | 60, 112
// 78 | 65.
constexpr int64_t kTcWork = 8000, kTcPerTile = 36, kTcPerUnit = 68;

struct Plan {
    int tc_grid;   // > 0: the tcgen05 kernel on that many CTAs
    int R, row_tiles, cluster, n_splits;
};

static Plan plan_of(int n_seq, int max_q, int64_t max_kv_len, int n_q_heads, int n_kv_heads) {
    Plan p{};
    const int64_t rows = (int64_t)max_q * (n_q_heads / n_kv_heads);
    const int64_t row_tiles = (rows + kTcRows - 1) / kTcRows, units = (int64_t)n_seq * n_kv_heads * row_tiles;
    const int64_t of_unit = (max_kv_len + kTcTile - 1) / kTcTile, tiles = units * of_unit, list = tiles + kTcGap * units;
    const int64_t work = (int64_t)n_seq * n_kv_heads * of_unit * rows;
    if (tiles && work >= kTcWork + kTcPerTile * tiles + kTcPerUnit * units && n_seq <= kTcMaxSeq && list < (int64_t)1 << 30) {
        p.tc_grid = (int)(list < kSms ? list : kSms);
        p.n_splits = p.tc_grid / (int64_t)(n_seq * n_kv_heads) > 0 ? p.tc_grid / (n_seq * n_kv_heads) : 1;  // (for the combine)
        return p;
    }
    p.R = rows <= 8 ? 1 : 2;
    p.row_tiles = (int)((rows + 8 * p.R * kMmaWarps - 1) / (8 * p.R * kMmaWarps));
    const int64_t blocks = (max_kv_len + kBlock - 1) / kBlock, ctas = (int64_t)n_seq * n_kv_heads * p.row_tiles;
    int64_t want = (kSms * (p.R == 1 ? 4 : 3)) / ctas, most = blocks / kMmaWarps;
    if (want > most) want = most;
    p.cluster = 1;
    while (p.cluster < kMaxCluster && 2 * p.cluster <= want) p.cluster *= 2;
    p.n_splits = want > p.cluster ? (int)(want / p.cluster) : 1;
    return p;
}

template <int F> static cudaError_t launch_tc(cudaStream_t stream, const TcAttArgs& ta) {
    auto* fn = paged_tc_kernel<F>;
    const cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, TcSmem::kBytes);
    return e != cudaSuccess ? e : launch_overlapped(fn, dim3((unsigned)ta.grid), kTcThreads, TcSmem::kBytes, stream, ta);
}

template <int kLanes> static cudaError_t run_tc_combine(cudaStream_t stream, const TcAttArgs& ta) {
    const int rows = ta.a.p.max_q * ta.a.G;
    const dim3 grid((unsigned)((rows + 16 / kLanes - 1) / (16 / kLanes)), (unsigned)ta.a.p.pool.n_heads, (unsigned)ta.a.p.n_seq);
    return launch_overlapped(paged_tc_combine_kernel<kLanes>, grid, 256, 0, stream, ta);
}

template <int F, int R> static cudaError_t launch_mma(cudaStream_t stream, const AttArgs& a, const Plan& plan) {
    constexpr int smem = MmaSmem<R>::kBytes;
    auto* fn = paged_mma_kernel<F, R>;
    cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    const dim3 grid((unsigned)(plan.cluster * plan.n_splits), (unsigned)(a.p.pool.n_heads * plan.row_tiles), (unsigned)a.p.n_seq);
    return launch_overlapped_clusters(fn, grid, kMmaWarps * 32, smem, plan.cluster, stream, a);
}

template <int kLanes> static cudaError_t run_combine(cudaStream_t stream, const AttArgs& a) {
    const int rows = a.p.max_q * a.G;
    const dim3 grid((unsigned)((rows + 16 / kLanes - 1) / (16 / kLanes)), (unsigned)a.p.pool.n_heads, (unsigned)a.p.n_seq);
    return launch_overlapped(paged_combine_kernel<kLanes>, grid, 256, 0, stream, a);
}

}  // namespace paged

// Whether numbers of positions, and the grid, stay in range.
bool paged_attention_fits(int n_seq, int max_q, int max_kv_len, int n_q_heads, int n_kv_heads) {
    const paged::Plan p = paged::plan_of(n_seq, max_q, max_kv_len, n_q_heads, n_kv_heads);
    return max_kv_len <= 1 << 30 && (p.tc_grid || (int64_t)n_kv_heads * p.row_tiles <= 65535);
}

size_t paged_attention_workspace_bytes(int n_seq, int max_q, int max_kv_len, int n_q_heads, int n_kv_heads) {
    using namespace paged;
    const Plan p = plan_of(n_seq, max_q, max_kv_len, n_q_heads, n_kv_heads);
    if (p.tc_grid) return align256((size_t)(n_seq + 1) * 4) + (size_t)2 * p.tc_grid * kTcRows * (kD + 2) * 4;
    if (p.n_splits == 1) return 0;
    const size_t rows = (size_t)n_seq * p.n_splits * max_q * n_q_heads;
    return align256(rows * 2 * 4) + rows * kD * 4;
}

cudaError_t launch_paged_attention(cudaStream_t stream, const cvattn_paged_attention_params& p, int* status) {
    using namespace paged;
    AttArgs a{};
    a.p = p;
    a.G = p.n_q_heads / p.pool.n_heads;
    a.blocks = p.pool.page_size / kBlock;
    a.scale_log2 = p.scale * 1.4426950408889634f;
    a.status = status;
    const Plan plan = plan_of(p.n_seq, p.max_q, p.max_kv_len, p.n_q_heads, p.pool.n_heads);
    a.n_splits = plan.n_splits;
    a.by_G = inverse_of(a.G);
    a.by_parts = inverse_of(plan.tc_grid ? plan.tc_grid : plan.cluster * plan.n_splits);
    if (plan.tc_grid) {
        TcAttArgs ta{};
        ta.a = a;
        ta.grid = plan.tc_grid;
        uint8_t* ws = static_cast<uint8_t*>(p.workspace);
        ta.ws_pref = reinterpret_cast<int32_t*>(ws);
        ta.ws_o = reinterpret_cast<float*>(ws + align256((size_t)(p.n_seq + 1) * 4));
        ta.ws_ml = ta.ws_o + (size_t)2 * ta.grid * kTcRows * kD;
        const cudaError_t e = p.pool.format == kI8 ? launch_tc<kI8>(stream, ta) : launch_tc<kE4M3>(stream, ta);
        if (e != cudaSuccess) return e;
        return plan.n_splits > 24 ? run_tc_combine<16>(stream, ta) : plan.n_splits > 4 ? run_tc_combine<4>(stream, ta) : run_tc_combine<1>(stream, ta);
    }
    if (plan.n_splits > 1) {
        const size_t rows = (size_t)p.n_seq * plan.n_splits * p.max_q * p.n_q_heads;
        a.ws_ml = static_cast<float*>(p.workspace);
        a.ws_o = reinterpret_cast<float*>(static_cast<uint8_t*>(p.workspace) + align256(rows * 2 * 4));
    }
    cudaError_t e;
    if (p.pool.format == kI8) e = plan.R == 1 ? launch_mma<kI8, 1>(stream, a, plan) : launch_mma<kI8, 2>(stream, a, plan);
    else e = plan.R == 1 ? launch_mma<kE4M3, 1>(stream, a, plan) : launch_mma<kE4M3, 2>(stream, a, plan);
    if (e != cudaSuccess || plan.n_splits == 1) return e;
    return plan.n_splits > 32 ? run_combine<16>(stream, a) : plan.n_splits > 8 ? run_combine<4>(stream, a) : run_combine<1>(stream, a);
}

}  // namespace cvattn
