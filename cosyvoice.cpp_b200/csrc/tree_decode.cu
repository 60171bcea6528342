// tree_decode.cu -- kernels and host side of cvattn_tree_decode.
#include "tree_decode.cuh"

namespace cvattn {
namespace tree {

// ------------------------------------------------------------ f32 kernel --
//
// A CTA of 128 threads takes 32 rows of one KV head and one split.  K and V tiles
// are dequantized to f32 in shared memory; a thread owns 4 rows x 4 keys of S and
// then 4 rows x 4 dims of the output.  Rows are padded to 68 floats, so the eight
// float4s of a phase (keys apart by one row) touch different banks.
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
            if (tc == 0) *reinterpret_cast<float2*>(a.ws_ml + slot * 2) = make_float2(m[i], l[i]);
        }
    }
}

// --------------------------------------------------------------- combine --
//
// A half-warp per row joins the splits that its sequence has: out = sum_k
// 2^(m_k - M) o_k / sum_k 2^(m_k - M) l_k, in the order of the splits.
__global__ void __launch_bounds__(256) tree_combine_kernel(const __grid_constant__ Args a) {
    const int half = threadIdx.x >> 4, c = threadIdx.x & 15;
    const int all_rows = a.max_nodes * a.G;
    const int r = blockIdx.x * 16 + half, kvh = blockIdx.y, s = blockIdx.z;
    if (r >= all_rows) return;
    const Lens x = lens_of(a, s, false);
    const int node = r / a.G, h = kvh * a.G + r % a.G;
    const int n = node < x.n ? (x.tiles + a.split_tiles - 1) / a.split_tiles : 0;
    const int64_t slot = ((int64_t)s * a.Hkv + kvh) * a.n_splits * all_rows + r;
    float M = -INFINITY, l = 0.0f;
    for (int k = 0; k < n; ++k) M = fmaxf(M, a.ws_ml[(slot + (int64_t)k * all_rows) * 2]);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    if (M != -INFINITY) {
        for (int k = 0; k < n; ++k) {
            const float2 ml = *reinterpret_cast<const float2*>(a.ws_ml + (slot + (int64_t)k * all_rows) * 2);
            const float4 v = *reinterpret_cast<const float4*>(a.ws_o + (slot + (int64_t)k * all_rows) * kD + c * 4);
            const float f = exp2f(ml.x - M);
            l = fmaf(f, ml.y, l);
            o.x = fmaf(f, v.x, o.x); o.y = fmaf(f, v.y, o.y); o.z = fmaf(f, v.z, o.z); o.w = fmaf(f, v.w, o.w);
        }
    }
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
    *reinterpret_cast<float4*>(a.out + (int64_t)s * a.out_nb_seq + (int64_t)node * a.out_nb_node + h * kD + c * 4) =
        make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
    if (a.lse && c == 0) a.lse[((int64_t)s * a.max_nodes + node) * a.Hq + h] = (M + log2f(l)) * 0.69314718055994531f;
}

// ------------------------------------------------------------------ host --

static size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

// How the keys are split: about kWantCtas CTAs over (sequence, KV head, row tile, split), each with at least two tiles.
constexpr int kWantCtas = 296;

struct Plan {
    int split_tiles, n_splits;
};

static Plan plan_of(int n_seq, int max_kv_len, int max_nodes, int n_q_heads, int n_kv_heads) {
    const int tiles = (max_kv_len + kTile - 1) / kTile + (max_nodes + kTile - 1) / kTile;
    const int64_t row_tiles = ((int64_t)max_nodes * (n_q_heads / n_kv_heads) + kRows - 1) / kRows;
    const int64_t units = (int64_t)n_seq * n_kv_heads * row_tiles;
    int64_t want = (kWantCtas + units - 1) / units;
    if (want > tiles / 2) want = tiles / 2;
    if (want < 1) want = 1;
    Plan p;
    p.split_tiles = (int)((tiles + want - 1) / want);
    p.n_splits = (tiles + p.split_tiles - 1) / p.split_tiles;
    return p;
}

size_t workspace_bytes(int n_seq, int max_kv_len, int max_nodes, int n_q_heads, int n_kv_heads) {
    const Plan p = plan_of(n_seq, max_kv_len, max_nodes, n_q_heads, n_kv_heads);
    if (p.n_splits == 1) return 0;
    const size_t rows = (size_t)n_seq * p.n_splits * max_nodes * n_q_heads;
    return align256(rows * 2 * 4) + rows * kD * 4;
}

}  // namespace tree

bool tree_supported(int k_type, int v_type, int head_dim, int n_q_heads, int n_kv_heads) {
    return type_known(k_type) && type_known(v_type) && head_dim == tree::kD && n_kv_heads > 0 && n_q_heads > 0 &&
           n_q_heads % n_kv_heads == 0 && n_q_heads / n_kv_heads <= 8;
}

size_t tree_workspace_bytes(int n_seq, int max_kv_len, int max_nodes, int n_q_heads, int n_kv_heads) {
    return tree::workspace_bytes(n_seq, max_kv_len, max_nodes, n_q_heads, n_kv_heads);
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
    const Plan plan = plan_of(a.n_seq, a.max_kv_len, a.max_nodes, a.Hq, a.Hkv);
    a.split_tiles = plan.split_tiles;
    a.n_splits = plan.n_splits;
    if (plan.n_splits > 1) {
        const size_t rows = (size_t)a.n_seq * plan.n_splits * a.max_nodes * a.Hq;
        a.ws_ml = static_cast<float*>(p.workspace);
        a.ws_o = reinterpret_cast<float*>(static_cast<uint8_t*>(p.workspace) + align256(rows * 2 * 4));
    }
    const int rows = a.max_nodes * a.G;
    const int smem = (2 * kRows + 2 * kTile) * kPad * 4;
    cudaError_t e = cudaFuncSetAttribute(tree_f32_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    const dim3 grid((unsigned)plan.n_splits, (unsigned)(a.Hkv * ((rows + kRows - 1) / kRows)), (unsigned)a.n_seq);
    tree_f32_kernel<<<grid, 128, smem, stream>>>(a);
    e = cudaGetLastError();
    if (e != cudaSuccess || plan.n_splits == 1) return e;
    tree_combine_kernel<<<dim3((unsigned)((rows + 15) / 16), (unsigned)a.Hkv, (unsigned)a.n_seq), 256, 0, stream>>>(a);
    return cudaGetLastError();
}

}  // namespace cvattn
