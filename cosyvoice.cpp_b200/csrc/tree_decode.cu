// tree_decode.cu -- kernels and host side of cvattn_tree_decode.
#include "tree_mma.cuh"
#include "tree_tc.cuh"

namespace cvattn {
namespace tree {

// ------------------------------------------------------------ f32 kernel --
//
// A CTA of 128 threads takes 32 rows of one KV head and one split.  K and V tiles
// are dequantized to f32 in shared memory; a thread owns 4 rows x 4 keys of S and
// then 4 rows x 4 dims of the output.  Rows are padded to 68 floats, so the eight
// float4s of a phase (keys apart by one row) touch different banks.  For f32 rows on either
// side, which have no two exact f16 pieces.  Bound by its FMAs, its shared-memory reads and the
// loads of a tile, an element at a time: 64 sequences of 128 to 2048, 8 nodes, f32 388 us, f32 K
// and Q8_0 V 325; 16 of 4096, 64 nodes, f32 2.2 ms.  (Q8_0 / Q4_0 on the tcgen05 kernel: 39.4.)
constexpr int kTile = 64;  // keys per tile
constexpr int kRows = 32;
constexpr int kPad = kD + 4;

__device__ __forceinline__ void load_tile(float (*dst)[kPad], int type, const uint8_t* base, int64_t nb1, int kvh, int t0,
                                          int count) {
    const int gb = group_bytes(type);
    for (int i = threadIdx.x; i < kTile * 2; i += blockDim.x) {
        const int key = i >> 1, half = i & 1;
        float* d = &dst[key][half * 32];
        if (key >= count) {
            for (int e = 0; e < 32; ++e) d[e] = 0.0f;
            continue;
        }
        const uint8_t* g = base + (int64_t)(t0 + key) * nb1 + (int64_t)(kvh * 2 + half) * gb;
        for (int e = 0; e < 32; ++e) d[e] = dequant_elem_rt(type, g, e);
    }
}

__global__ void __launch_bounds__(128) tree_f32_kernel(const __grid_constant__ Args a) {
    extern __shared__ float4 smem4[];
    float(*qs)[kPad] = reinterpret_cast<float(*)[kPad]>(smem4);
    float(*ks)[kPad] = qs + kRows;
    float(*vs)[kPad] = ks + kTile;
    float(*ps)[kPad] = vs + kTile;
    const int tid = threadIdx.x, tr = tid >> 4, tc = tid & 15;
    const int s = blockIdx.z, kvh = blockIdx.y % a.Hkv, r0 = (blockIdx.y / a.Hkv) * kRows, split = blockIdx.x;
    griddep_wait();
    const Lens x = lens_of(a, s, tid == 0 && blockIdx.x == 0 && blockIdx.y == 0);
    const int rows = x.n * a.G, all_rows = a.max_nodes * a.G;
    const int tile0 = split * a.split_tiles, tile1 = min(x.tiles, tile0 + a.split_tiles);
    const bool direct = a.n_splits == 1;
    if (!direct && (tile0 >= tile1 || r0 >= rows)) return;  // nothing that the combine would read
    const uint8_t* kb = seq_base(a.k_seq_ptrs, a.k, a.k_nb2, s);
    const uint8_t* vb = seq_base(a.v_seq_ptrs, a.v, a.v_nb2, s);
    const uint8_t* kdb = a.kd ? a.kd + (int64_t)s * a.kd_nb2 : nullptr;
    const uint8_t* vdb = a.vd ? a.vd + (int64_t)s * a.vd_nb2 : nullptr;

    for (int i = tid; i < kRows * kD; i += 128) {
        const int r = r0 + i / kD, d = i % kD;
        float v = 0.0f;
        if (r < rows) v = a.q[(int64_t)s * a.q_nb_seq + (int64_t)(r / a.G) * a.q_nb_node + (kvh * a.G + r % a.G) * kD + d];
        qs[i / kD][d] = v * a.scale_log2;
    }
    float m[4], l[4];
    float4 o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        m[i] = -INFINITY;
        l[i] = 0.0f;
        o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    for (int t = tile0; t < tile1; ++t) {
        const bool draft = t >= x.cache_tiles;
        const int p0 = (draft ? t - x.cache_tiles : t) * kTile;
        const int count = min(kTile, (draft ? x.n : x.L) - p0);
        __syncthreads();
        load_tile(ks, a.k_type, draft ? kdb : kb, draft ? a.kd_nb1 : a.k_nb1, kvh, p0, count);
        load_tile(vs, a.v_type, draft ? vdb : vb, draft ? a.vd_nb1 : a.v_nb1, kvh, p0, count);
        __syncthreads();
        float sc[4][4] = {};
#pragma unroll 4
        for (int d = 0; d < kD; d += 4) {
            float4 kk[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) kk[j] = *reinterpret_cast<const float4*>(&ks[tc + 16 * j][d]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float4 qq = *reinterpret_cast<const float4*>(&qs[tr * 4 + i][d]);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    sc[i][j] = fmaf(qq.x, kk[j].x, fmaf(qq.y, kk[j].y, fmaf(qq.z, kk[j].z, fmaf(qq.w, kk[j].w, sc[i][j]))));
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = r0 + tr * 4 + i, node = r / a.G;
            float mx = m[i];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int key = tc + 16 * j;
                const bool sees = r < rows && key < count && (!draft || node_sees(a, s, node, p0 + key));
                if (!sees) sc[i][j] = -INFINITY;
                mx = fmaxf(mx, sc[i][j]);
            }
#pragma unroll
            for (int w = 8; w > 0; w >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
            const float base = mx == -INFINITY ? 0.0f : mx;
            const float f = exp2f(m[i] - base);
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float p = exp2f(sc[i][j] - base);
                ps[tr * 4 + i][tc + 16 * j] = p;
                sum += p;
            }
#pragma unroll
            for (int w = 8; w > 0; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
            m[i] = mx;
            l[i] = fmaf(l[i], f, sum);
            o[i].x *= f; o[i].y *= f; o[i].z *= f; o[i].w *= f;
        }
        __syncwarp();  // a row's 16 threads are in one warp
#pragma unroll 4
        for (int key = 0; key < kTile; ++key) {
            const float4 vv = *reinterpret_cast<const float4*>(&vs[key][tc * 4]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float p = ps[tr * 4 + i][key];
                if (draft && p == 0.0f) continue;  // a draft that the row does not see may hold anything
                o[i].x = fmaf(p, vv.x, o[i].x); o[i].y = fmaf(p, vv.y, o[i].y);
                o[i].z = fmaf(p, vv.z, o[i].z); o[i].w = fmaf(p, vv.w, o[i].w);
            }
        }
        __syncwarp();
    }
    griddep_launch_dependents();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = r0 + tr * 4 + i;
        if (r >= all_rows) continue;
        if (direct) {
            const float inv = l[i] > 0.0f ? 1.0f / l[i] : 0.0f;
            const int node = r / a.G, h = kvh * a.G + r % a.G;
            *reinterpret_cast<float4*>(a.out + (int64_t)s * a.out_nb_seq + (int64_t)node * a.out_nb_node + h * kD + tc * 4) =
                make_float4(o[i].x * inv, o[i].y * inv, o[i].z * inv, o[i].w * inv);
            if (a.lse && tc == 0)
                a.lse[((int64_t)s * a.max_nodes + node) * a.Hq + h] = (m[i] + log2f(l[i])) * 0.69314718055994531f;
        } else if (r < rows) {
            const int64_t slot = (((int64_t)s * a.Hkv + kvh) * a.n_splits + split) * all_rows + r;
            *reinterpret_cast<float4*>(a.ws_o + slot * kD + tc * 4) = o[i];
            // (a row whose scores are all NaN has no maximum, but was seen)
            if (tc == 0) *reinterpret_cast<float2*>(a.ws_ml + slot * 2) = make_float2(m[i] == -INFINITY && l[i] != 0.0f ? 0.0f : m[i], l[i]);
        }
    }
}

// --------------------------------------------------------------- combine --
//
// out = sum_k 2^(m_k - M) o_k / sum_k 2^(m_k - M) l_k over the splits that the
// sequence has.  16 threads (4 dims each) follow every kLanes-th split of a row;
// the kLanes partial sums of a row are joined through shared memory in order.
// Latency-bound: about 2 us, started early so that its launch is hidden.
template <int kLanes>
__global__ void __launch_bounds__(256) tree_combine_kernel(const __grid_constant__ Args a) {
    constexpr int kPer = 16 / kLanes;  // rows per CTA
    __shared__ float4 so[16][16];
    __shared__ float2 sml[16];
    griddep_wait();
    const int unit = threadIdx.x >> 4, c = threadIdx.x & 15, lane = unit % kLanes;
    const int all_rows = a.max_nodes * a.G;
    const int r = blockIdx.x * kPer + unit / kLanes, kvh = blockIdx.y, s = blockIdx.z;
    const Lens x = lens_of(a, s, false);
    const int node = r / a.G, h = kvh * a.G + r % a.G;
    const int n = node < x.n ? (x.tiles + a.split_tiles - 1) / a.split_tiles : 0;  // (rows past the last: none)
    const int64_t slot = ((int64_t)s * a.Hkv + kvh) * a.n_splits * all_rows + r;
    float M = -INFINITY, l = 0.0f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k0 = lane; k0 < n; k0 += 4 * kLanes) {
        float2 ml[4];
        float4 v[4];
        float top = M;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int k = k0 + u * kLanes;
            ml[u] = make_float2(-INFINITY, 0.0f);
            if (k < n) {
                ml[u] = *reinterpret_cast<const float2*>(a.ws_ml + (slot + (int64_t)k * all_rows) * 2);
                v[u] = *reinterpret_cast<const float4*>(a.ws_o + (slot + (int64_t)k * all_rows) * kD + c * 4);
            }
            top = fmaxf(top, ml[u].x);
        }
        if (top == -INFINITY) continue;
        const float f0 = exp2f(M - top);
        M = top;
        l *= f0;
        o.x *= f0; o.y *= f0; o.z *= f0; o.w *= f0;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (ml[u].x == -INFINITY) continue;
            const float f = exp2f(ml[u].x - M);
            l = fmaf(f, ml[u].y, l);
            o.x = fmaf(f, v[u].x, o.x); o.y = fmaf(f, v[u].y, o.y); o.z = fmaf(f, v[u].z, o.z); o.w = fmaf(f, v[u].w, o.w);
        }
    }
    if constexpr (kLanes > 1) {
        so[unit][c] = o;
        if (c == 0) sml[unit] = make_float2(M, l);
        __syncthreads();
        if (lane) return;
        float top = -INFINITY;
#pragma unroll
        for (int k = 0; k < kLanes; ++k) top = fmaxf(top, sml[unit + k].x);
        l = 0.0f;
        o = make_float4(0.f, 0.f, 0.f, 0.f);
        M = top;
        if (top != -INFINITY) {
#pragma unroll
            for (int k = 0; k < kLanes; ++k) {
                if (sml[unit + k].x == -INFINITY) continue;
                const float f = exp2f(sml[unit + k].x - top);
                const float4 v = so[unit + k][c];
                l = fmaf(f, sml[unit + k].y, l);
                o.x = fmaf(f, v.x, o.x); o.y = fmaf(f, v.y, o.y); o.z = fmaf(f, v.z, o.z); o.w = fmaf(f, v.w, o.w);
            }
        }
    }
    if (r >= all_rows) return;
    const bool seen = M != -INFINITY;
    const float inv = seen ? 1.0f / l : 0.0f;
    *reinterpret_cast<float4*>(a.out + (int64_t)s * a.out_nb_seq + (int64_t)node * a.out_nb_node + h * kD + c * 4) =
        make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
    if (a.lse && c == 0) a.lse[((int64_t)s * a.max_nodes + node) * a.Hq + h] = seen ? (M + log2f(l)) * 0.69314718055994531f : -INFINITY;
}

// ------------------------------------------------------------------ host --

static size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

static bool mma_type(int t) { return t != kF32; }

// Which kernel, its shape, and how the keys are split.
struct Plan {
    bool mma;
    int tc_grid;   // > 0: the tcgen05 kernel on that many CTAs
    Shape sh;
    int tile, split_tiles, n_splits;
};

constexpr int kSms = 148;
constexpr int kSlots = 2 * kSms;  // two CTAs of tree_mma_kernel per SM
// The tcgen05 kernel starts later (10 us before the first output) and goes through tiles faster, whatever rows they have up to
// 128.  It takes over at this many 128-key tiles x rows of a KV head, and above 128 rows.  us of tree_mma_kernel | tcgen05, 14 / 2
// heads, Q8_0 and f16: one sequence of 4096 (66 tiles), 112 rows 15.4 | 15.6 and 13.4 | 15.2, 252 rows 20.0 | 17.3 and 18.4 |
// 16.3; 16 of 1000 (288), 56 rows 17.6 | 23.5 and 14.5 | 22.0, 112 rows 24.6 | 25.2 and 21.2 | 23.8; one of 65536 (1026), 28
// rows 31.8 | 29.9 and 22.4 | 24.3, 56 rows 41.6 | 30.5 and 30.8 | 25.0; 64 of 4096 (4224), 7 rows 86 | 74 and 51 | 55, 28 rows
// 108 | 75 and 69 | 55.  (One number for both kinds of cache: at 64 of 4096 with 7 rows, 29568, it keeps quants on the slower side.)
constexpr int64_t kTcMinWork = 1 << 15;

static Plan plan_of(int k_type, int v_type, int n_seq, int max_kv_len, int max_nodes, int n_q_heads, int n_kv_heads) {
    Plan p{};
    const int64_t rows = (int64_t)max_nodes * (n_q_heads / n_kv_heads);
    p.mma = mma_type(k_type) && mma_type(v_type);
    int64_t units;
    const int64_t key_tiles = (int64_t)n_seq * n_kv_heads * ((max_kv_len + kTcTile - 1) / kTcTile + (max_nodes + kTcTile - 1) / kTcTile);
    const int64_t entries = key_tiles * ((rows + kTcRows - 1) / kTcRows);
    if (p.mma && (rows > kTcRows || key_tiles * rows >= kTcMinWork) && n_seq <= kTcMaxSeq && entries < (int64_t)1 << 31) {
        p.tile = kTcTile;
        p.tc_grid = (int)(entries < kSms ? entries : kSms);
        p.n_splits = p.tc_grid / (int64_t)(n_seq * n_kv_heads) > 0 ? p.tc_grid / (n_seq * n_kv_heads) : 1;  // (for the combine)
        return p;
    }
    if (p.mma) {
        p.tile = kKeys;
        p.sh.row_groups = (int)((rows + 16 * kWarps - 1) / (16 * kWarps));
        p.sh.stages = kMaxStages;
        while (p.sh.stages > 2 && Smem(k_type, v_type, p.sh.stages).total > kHalfSm) --p.sh.stages;
        units = (int64_t)n_seq * n_kv_heads * p.sh.row_groups;
        // Few tiles: smaller ones, on more SMs.  us of 64 | 128 keys, Q8_0: one sequence of 300, 28 rows 9.9 | 10.5; 16 sequences of
        // 1000 (256 tiles), 28 rows 18.6 | 14.7.
        if (units * ((max_kv_len + kKeys - 1) / kKeys) < kSlots / 2) p.tile = kKeys / 2;
    } else {
        p.tile = kTile;
        units = (int64_t)n_seq * n_kv_heads * ((rows + kRows - 1) / kRows);
    }
    // One wave of CTAs; two where the lengths of several sequences may differ, so that short ones leave room for parts of
    // long ones.  At least two tiles per split once every slot has work.
    const int tiles = (max_kv_len + p.tile - 1) / p.tile + (max_nodes + p.tile - 1) / p.tile;
    const int64_t most = units * tiles <= kSlots ? tiles : tiles / 2;
    int64_t want = ((n_seq > 2 ? 2 : 1) * kSlots + units - 1) / units;
    if (want > most) want = most;
    if (want < 1) want = 1;
    p.split_tiles = (int)((tiles + want - 1) / want);
    p.n_splits = (tiles + p.split_tiles - 1) / p.split_tiles;
    return p;
}

template <int kLanes>
static cudaError_t run_combine(cudaStream_t stream, const Args& a) {
    const int rows = a.max_nodes * a.G;
    const dim3 grid((unsigned)((rows + 16 / kLanes - 1) / (16 / kLanes)), (unsigned)a.Hkv, (unsigned)a.n_seq);
    return launch_overlapped(tree_combine_kernel<kLanes>, grid, 256, 0, stream, a);
}

template <int kLanes>
static cudaError_t run_tc_combine(cudaStream_t stream, const TcArgs& ta) {
    const int rows = ta.a.max_nodes * ta.a.G;
    const dim3 grid((unsigned)((rows + 16 / kLanes - 1) / (16 / kLanes)), (unsigned)ta.a.Hkv, (unsigned)ta.a.n_seq);
    return launch_overlapped(tree_tc_combine_kernel<kLanes>, grid, 256, 0, stream, ta);
}

static cudaError_t launch_tc(cudaStream_t stream, const Args& a, const Plan& plan, void* workspace) {
    TcArgs ta{};
    ta.a = a;
    ta.grid = plan.tc_grid;
    ta.inv_g = (uint32_t)((65536 + a.G - 1) / a.G);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    ta.ws_pref = reinterpret_cast<int32_t*>(ws);
    ws += align256((size_t)(a.n_seq + 1) * 4);
    ta.ws_o = reinterpret_cast<float*>(ws);
    ta.ws_ml = ta.ws_o + (size_t)2 * ta.grid * kTcRows * kD;
    cudaError_t e = cudaErrorInvalidValue;
    switch (a.k_type) {
    case kF16: e = launch_tc_for_k<kF16>(stream, ta); break;
    case kQ4_0: e = launch_tc_for_k<kQ4_0>(stream, ta); break;
    case kQ4_1: e = launch_tc_for_k<kQ4_1>(stream, ta); break;
    case kQ5_0: e = launch_tc_for_k<kQ5_0>(stream, ta); break;
    case kQ5_1: e = launch_tc_for_k<kQ5_1>(stream, ta); break;
    case kQ8_0: e = launch_tc_for_k<kQ8_0>(stream, ta); break;
    default: break;
    }
    if (e != cudaSuccess) return e;
    // Lanes that share a row's parts.  us of a call with 1 | 4 | 16, 140 rows, Q8_0: 8 parts a unit (one sequence of 300) 15.1 | 13.5 |
    // 13.9, 18 (4 of 4096) 31.0 | 25.8 | 27.9, 74 (one of 4096) 35.2 | 21.0 | 17.1, 4 (16 of 4096) 50 | 51 | 66.
    return plan.n_splits > 24 ? run_tc_combine<16>(stream, ta) : plan.n_splits > 4 ? run_tc_combine<4>(stream, ta)
                                                                                   : run_tc_combine<1>(stream, ta);
}

static cudaError_t launch_combine(cudaStream_t stream, const Args& a) {
    // The same, 14 rows, Q8_0: 7 parts (one sequence of 300) 9.1 | 8.9 | 9.2, 17 (one of 1000) 11.1 | 9.5 | 9.5, 66 (one of 4096) 18.7 |
    // 12.3 | 10.8.
    return a.n_splits > 32 ? run_combine<16>(stream, a) : a.n_splits > 8 ? run_combine<4>(stream, a) : run_combine<1>(stream, a);
}

size_t workspace_bytes(int k_type, int v_type, int n_seq, int max_kv_len, int max_nodes, int n_q_heads, int n_kv_heads) {
    const Plan p = plan_of(k_type, v_type, n_seq, max_kv_len, max_nodes, n_q_heads, n_kv_heads);
    if (p.tc_grid) return align256((size_t)(n_seq + 1) * 4) + (size_t)2 * p.tc_grid * kTcRows * (kD + 2) * 4;
    if (p.n_splits == 1) return 0;
    const size_t rows = (size_t)n_seq * p.n_splits * max_nodes * n_q_heads;
    return align256(rows * 2 * 4) + rows * kD * 4;
}

}  // namespace tree

bool tree_supported(int k_type, int v_type, int head_dim, int n_q_heads, int n_kv_heads) {
    return type_known(k_type) && type_known(v_type) && head_dim == tree::kD && n_kv_heads > 0 && n_q_heads > 0 &&
           n_q_heads % n_kv_heads == 0 && n_q_heads / n_kv_heads <= 8;
}

size_t tree_workspace_bytes(int k_type, int v_type, int n_seq, int max_kv_len, int max_nodes, int n_q_heads, int n_kv_heads) {
    return tree::workspace_bytes(k_type, v_type, n_seq, max_kv_len, max_nodes, n_q_heads, n_kv_heads);
}

cudaError_t launch_tree_decode(cudaStream_t stream, const cvattn_tree_params& p, int* status) {
    using namespace tree;
    Args a{};
    a.q = p.q;
    a.q_nb_node = p.q_nb_node;
    a.q_nb_seq = p.q_nb_seq;
    a.out = p.out;
    a.out_nb_node = p.out_nb_node;
    a.out_nb_seq = p.out_nb_seq;
    a.lse = p.lse;
    a.k = static_cast<const uint8_t*>(p.k.data);
    a.v = static_cast<const uint8_t*>(p.v.data);
    a.kd = static_cast<const uint8_t*>(p.k_draft.data);
    a.vd = static_cast<const uint8_t*>(p.v_draft.data);
    a.k_nb1 = p.k.nb1; a.k_nb2 = p.k.nb2; a.v_nb1 = p.v.nb1; a.v_nb2 = p.v.nb2;
    a.kd_nb1 = p.k_draft.nb1; a.kd_nb2 = p.k_draft.nb2; a.vd_nb1 = p.v_draft.nb1; a.vd_nb2 = p.v_draft.nb2;
    a.k_seq_ptrs = p.k_seq_ptrs;
    a.v_seq_ptrs = p.v_seq_ptrs;
    a.kv_len = p.kv_len;
    a.n_nodes = p.n_nodes;
    a.mask = p.mask;
    a.mask_nb_seq = p.mask_nb_seq;
    a.mask_words = (p.max_nodes + 31) / 32;
    a.k_type = p.k.type;
    a.v_type = p.v.type;
    a.n_seq = p.n_seq;
    a.max_nodes = p.max_nodes;
    a.Hq = p.n_q_heads;
    a.Hkv = p.k.n_heads;
    a.G = a.Hq / a.Hkv;
    a.max_kv_len = p.max_kv_len;
    a.scale_log2 = p.scale * 1.4426950408889634f;
    a.status = status;
    const Plan plan = plan_of(a.k_type, a.v_type, a.n_seq, a.max_kv_len, a.max_nodes, a.Hq, a.Hkv);
    a.tile = plan.tile;
    a.split_tiles = plan.split_tiles;
    a.n_splits = plan.n_splits;
    if (plan.tc_grid) return launch_tc(stream, a, plan, p.workspace);
    if (plan.n_splits > 1) {
        const size_t rows = (size_t)a.n_seq * plan.n_splits * a.max_nodes * a.Hq;
        a.ws_ml = static_cast<float*>(p.workspace);
        a.ws_o = reinterpret_cast<float*>(static_cast<uint8_t*>(p.workspace) + align256(rows * 2 * 4));
    }
    cudaError_t e = cudaErrorInvalidValue;
    if (plan.mma) {
        switch (a.k_type) {
        case kF16: e = launch_mma_for_k<kF16>(stream, a, plan.sh); break;
        case kQ4_0: e = launch_mma_for_k<kQ4_0>(stream, a, plan.sh); break;
        case kQ4_1: e = launch_mma_for_k<kQ4_1>(stream, a, plan.sh); break;
        case kQ5_0: e = launch_mma_for_k<kQ5_0>(stream, a, plan.sh); break;
        case kQ5_1: e = launch_mma_for_k<kQ5_1>(stream, a, plan.sh); break;
        case kQ8_0: e = launch_mma_for_k<kQ8_0>(stream, a, plan.sh); break;
        default: break;
        }
    } else {
        const int rows = a.max_nodes * a.G;
        const int smem = (2 * kRows + 2 * kTile) * kPad * 4;
        e = cudaFuncSetAttribute(tree_f32_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return e;
        const dim3 grid((unsigned)plan.n_splits, (unsigned)(a.Hkv * ((rows + kRows - 1) / kRows)), (unsigned)a.n_seq);
        e = launch_overlapped(tree_f32_kernel, grid, 128, smem, stream, a);
    }
    if (e != cudaSuccess || plan.n_splits == 1) return e;
    return launch_combine(stream, a);
}

}  // namespace cvattn
