// tree_mma.cuh -- tree attention on warp-level tensor-core MMAs (mma.sync
// m16n8k16, f16 operands, f32 accumulators) for f16 and block-quantized caches.
//
// The arithmetic is exact where the cache is: quants are integers, exact in f16,
// their block scales (and mins) stay aside in f32; Q is scaled per row by a power
// of two and split into f16 hi + lo; P' = p d_V 2^ev is split the same way.  Every
// product is then exact in the f32 accumulators and what is left out is below
// 2^-22 of the largest term.
//
// A CTA takes one split of one sequence, HC (1 or 2) neighbouring KV heads and a
// group of rows.  Its 8 warps are HC heads x WR row groups of 16 MT rows x WK
// slices of the keys.  Tiles of 128 keys arrive by cp.async into a ring of raw
// rows; a table of the tile's scales in f32 is built once for all warps.  A warp
// walks its 16-key steps: K fragments straight from the raw bytes, S in
// registers, lazy running maximum (raised when a score passes it by more than
// 2^8, with the output rescaled), P' as the A operand of P.V without leaving the
// registers, V fragments from the raw bytes.  Warps that share rows merge at the
// end through shared memory.
#pragma once

#include "decode_mma.cuh"
#include "tree_decode.cuh"

namespace cvattn {
namespace tree {

using dmma::ld_u16;
using dmma::mma16816;
using dmma::quad_max;
using dmma::quad_sum;
using dmma::split2;
using dtc::pow2f;

constexpr int kKeys = 128;    // keys per tile
constexpr int kSub = 16;      // keys per step
constexpr int kWarps = 8;
constexpr int kMaxStages = 3;
constexpr int kSmemLimit = 227 * 1024;
constexpr float kLazy = 8.0f;
constexpr int kRowInfo = 4;   // floats per row: score factor, sums of Q over the two blocks

struct Shape {
    int hc, wr, wk;    // heads, row groups, key slices: hc * wr * wk = 8
    int row_groups;    // CTAs along the rows
    int stages;        // ring slots: 3, or 2 where 3 do not fit
};

// Bytes between the keys of a tile in shared memory: 4-byte words per key odd (K), 4 mod 16 words for the byte-wide V
// of q8_0, and for f16 16 words off a multiple of 32 (K, 16-byte reads of 8 keys) or 4 words (V, 16-byte reads of 4 keys).
__host__ __device__ constexpr int k_stride(int t, int hc) {
    const int b = hc * 2 * group_bytes(t);
    if (t == kF16) return b + 64;
    return ((b / 4) | 1) * 4;
}
__host__ __device__ constexpr int v_stride(int t, int hc) {
    const int b = hc * 2 * group_bytes(t);
    if (t == kF16) return b + 16;
    if (t == kQ8_0) return b + (hc == 1 ? 12 : 8);
    return ((b / 4) | 1) * 4;
}

struct Smem {
    int q, rows, maxv, tab, tab_head, ring, k_bytes, stage, total;
    __host__ __device__ Smem(int kt, int vt, int mt, int hc, int wr, int stages) {
        int o = 0;
        q = o; o += hc * wr * mt * 4096;
        rows = o; o += hc * wr * mt * 16 * kRowInfo * 4;
        maxv = o; o += 32;
        tab = o;
        const bool km = kt == kQ4_1 || kt == kQ5_1, vm = vt == kQ4_1 || vt == kQ5_1;
        tab_head = ((kt == kF16 ? 0 : 2) + (km ? 2 : 0) + (vt == kF16 ? 0 : 2) + (vm ? 2 : 0)) * kKeys * 4;
        o += hc * tab_head;
        o = (o + 127) / 128 * 128;
        ring = o;
        k_bytes = (kKeys * k_stride(kt, hc) + 127) / 128 * 128;
        stage = k_bytes + (kKeys * v_stride(vt, hc) + 127) / 128 * 128;
        const int joined = kWarps * mt * 16 * ((kD + 4) * 4 + 8);  // the warps' outputs and (max, sum) at the end
        o += stages * stage > joined ? stages * stage : joined;
        total = o;
    }
};

// Keys [0, kKeys) of a tile, `row` bytes each, into shared memory; keys from
// count on become zeros.  unit: 16 or 4 bytes by cp.async, 2 by plain loads.
__device__ __forceinline__ void cp_async4(void* dst, const void* src, bool real) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_addr(dst)), "l"(src), "r"(real ? 4 : 0) : "memory");
}
__device__ __forceinline__ void cp_async16(void* dst, const void* src, bool real) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_addr(dst)), "l"(src), "r"(real ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void fetch_tile(uint8_t* dst, int stride, const uint8_t* src, int64_t nb1, int row, int unit, int count) {
    const int w = row / unit;
    int key = threadIdx.x / w, at = threadIdx.x - key * w;
    const int dk = (kWarps * 32) / w, da = (kWarps * 32) - dk * w;
    while (key < kKeys) {
        const bool real = key < count;
        const uint8_t* s = src + (int64_t)(real ? key : 0) * nb1 + at * unit;
        uint8_t* d = dst + key * stride + at * unit;
        if (unit == 16) cp_async16(d, s, real);
        else if (unit == 4) cp_async4(d, s, real);
        else *reinterpret_cast<uint16_t*>(d) = real ? *reinterpret_cast<const uint16_t*>(s) : (uint16_t)0;
        key += dk;
        at += da;
        if (at >= w) {
            at -= w;
            ++key;
        }
    }
}

__device__ __forceinline__ int copy_unit(int type, const uint8_t* base, int64_t nb1) {
    const uint64_t x = reinterpret_cast<uint64_t>(base) | (uint64_t)nb1;
    if (type == kF16 && (x & 15) == 0) return 16;
    return (x & 3) == 0 ? 4 : 2;
}

// K operand of one (key, block): the 8 values of thread tig (dmma::kfrag; f16: 8 consecutive values).
template <int T, int BLK>
__device__ __forceinline__ void k_frag(const uint8_t* g, int tig, uint32_t (&r)[4]) {
    if constexpr (T == kF16) {
        const uint4 w = *reinterpret_cast<const uint4*>(g + 64 * BLK + 16 * tig);
        r[0] = w.x; r[1] = w.y; r[2] = w.z; r[3] = w.w;
    } else {
        dmma::kfrag<T, BLK>(g + BLK * group_bytes(T), tig, r);
    }
}
template <int T>
__device__ __forceinline__ int k_elem(int tig, int i) {
    if constexpr (T == kF16) return 8 * tig + i;
    else return dmma::kelem<T>(tig, i);
}
// Output dim of column n of dim tile j (0..7).
template <int T>
__device__ __forceinline__ int v_dim(int n, int j) {
    if constexpr (T == kF16) return 8 * n + j;
    else return 32 * (j >> 2) + dmma::velem<T>(n, j & 3);
}

__device__ __forceinline__ bool f16x2_special(uint32_t w) {
    return (w & 0x7C00u) == 0x7C00u || (w & 0x7C000000u) == 0x7C000000u;
}

template <int KT, int VT, int MT>
__global__ void __launch_bounds__(kWarps * 32, 1) tree_mma_kernel(const __grid_constant__ Args a, const Shape sh) {
    extern __shared__ __align__(128) uint8_t smem[];
    constexpr int sliceK = 2 * group_bytes(KT), sliceV = 2 * group_bytes(VT);
    constexpr bool K_Q = KT != kF16, V_Q = VT != kF16;
    constexpr bool K_MIN = BlockTraits<KT>::HAS_MIN, V_MIN = BlockTraits<VT>::HAS_MIN;
    constexpr float kOffs = V_Q ? 0.0f : 7.0f;  // f16 V: P is kept 2^7 larger, far from f16's subnormals
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gid = lane >> 2, tig = lane & 3;
    const int s = blockIdx.z, split = blockIdx.x;
    const int n_hg = a.Hkv / sh.hc, hg = blockIdx.y % n_hg, rg = blockIdx.y / n_hg;
    const int group_rows = 16 * MT * sh.wr, r0 = rg * group_rows;
    const Lens x = lens_of(a, s, tid == 0 && blockIdx.x == 0 && blockIdx.y == 0);
    const int rows = x.n * a.G, all_rows = a.max_nodes * a.G;
    const int tile0 = split * a.split_tiles, tile1 = min(x.tiles, tile0 + a.split_tiles);
    const bool direct = a.n_splits == 1;
    if (!direct && (tile0 >= tile1 || r0 >= rows)) return;
    const Smem L(KT, VT, MT, sh.hc, sh.wr, sh.stages);
    const int strideK = k_stride(KT, sh.hc), strideV = v_stride(VT, sh.hc);
    const uint8_t* kb = seq_base(a.k_seq_ptrs, a.k, a.k_nb2, s) + (int64_t)hg * sh.hc * sliceK;
    const uint8_t* vb = seq_base(a.v_seq_ptrs, a.v, a.v_nb2, s) + (int64_t)hg * sh.hc * sliceV;
    const uint8_t* kdb = a.kd ? a.kd + (int64_t)s * a.kd_nb2 + (int64_t)hg * sh.hc * sliceK : nullptr;
    const uint8_t* vdb = a.vd ? a.vd + (int64_t)s * a.vd_nb2 + (int64_t)hg * sh.hc * sliceV : nullptr;
    const int uk = copy_unit(KT, kb, a.k_nb1), uv = copy_unit(VT, vb, a.v_nb1);
    const int ukd = copy_unit(KT, kdb, a.kd_nb1), uvd = copy_unit(VT, vdb, a.vd_nb1);

    const int n_local = r0 < rows ? max(0, tile1 - tile0) : 0;
    auto issue = [&](int t, int slot) {  // tile tile0 + t into a ring slot
        if (t < n_local) {
            const int tile = tile0 + t;
            const bool draft = tile >= x.cache_tiles;
            const int p0 = (draft ? tile - x.cache_tiles : tile) * kKeys;
            const int count = min(kKeys, (draft ? x.n : x.L) - p0);
            uint8_t* d = smem + L.ring + slot * L.stage;
            const int64_t nk = draft ? a.kd_nb1 : a.k_nb1, nv = draft ? a.vd_nb1 : a.v_nb1;
            fetch_tile(d, strideK, (draft ? kdb : kb) + (int64_t)p0 * nk, nk, sh.hc * sliceK, draft ? ukd : uk, count);
            fetch_tile(d + L.k_bytes, strideV, (draft ? vdb : vb) + (int64_t)p0 * nv, nv, sh.hc * sliceV, draft ? uvd : uv, count);
        }
        cp_async_commit();
    };
    for (int t = 0; t < sh.stages - 1; ++t) issue(t, t);

    // Q fragments of every row tile of the CTA: [head][row tile][k-step][hi, lo][lane]
    uint4* qf = reinterpret_cast<uint4*>(smem + L.q);
    float* rowinfo = reinterpret_cast<float*>(smem + L.rows);
    for (int t = warp; t < sh.hc * sh.wr * MT; t += kWarps) {
        const int hd = t / (sh.wr * MT), rt = t % (sh.wr * MT);
        uint32_t hi[4][4], lo[4][4];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int r = r0 + rt * 16 + half * 8 + gid;
            float e[2][8];
            float am = 0.0f, sum[2] = {0.0f, 0.0f};
            const bool real = r < rows;
            const float* q = a.q + (int64_t)s * a.q_nb_seq + (int64_t)(r / a.G) * a.q_nb_node +
                             ((hg * sh.hc + hd) * a.G + r % a.G) * kD;
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    e[b][i] = real ? q[32 * b + k_elem<KT>(tig, i)] : 0.0f;
                    am = fmaxf(am, fabsf(e[b][i]));
                    sum[b] += e[b][i];
                }
            am = quad_max(am);
            const int ex = dtc::norm_exp(am);
            const float sc = pow2f(ex);
            sum[0] = quad_sum(sum[0]);
            sum[1] = quad_sum(sum[1]);
            if (tig == 0) {
                float* ri = rowinfo + ((hd * sh.wr * MT + rt) * 16 + half * 8 + gid) * kRowInfo;
                ri[0] = pow2f(-ex) * a.scale_log2;
                ri[1] = sum[0] * a.scale_log2;
                ri[2] = sum[1] * a.scale_log2;
            }
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    split2(e[b][4 * j] * sc, e[b][4 * j + 1] * sc, hi[2 * b + j][half], lo[2 * b + j][half]);
                    split2(e[b][4 * j + 2] * sc, e[b][4 * j + 3] * sc, hi[2 * b + j][2 + half], lo[2 * b + j][2 + half]);
                }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            qf[((t * 4 + k) * 2 + 0) * 32 + lane] = make_uint4(hi[k][0], hi[k][1], hi[k][2], hi[k][3]);
            qf[((t * 4 + k) * 2 + 1) * 32 + lane] = make_uint4(lo[k][0], lo[k][1], lo[k][2], lo[k][3]);
        }
    }
    if (tid < 8) reinterpret_cast<uint32_t*>(smem + L.maxv)[tid] = 0u;
    __syncthreads();

    // this warp: head wh, row tiles rt0 .. rt0 + MT, key steps wk, wk + WK, ..
    const int wh = warp / (sh.wr * sh.wk), wr = warp % sh.wr, wk = (warp / sh.wr) % sh.wk;
    const int rt0 = wr * MT, t0q = wh * sh.wr * MT + rt0;
    const bool idle = r0 + rt0 * 16 >= rows;  // no row of this warp is real
    uint32_t qa[MT][4][2][4];
    float rs[MT][2], qs0[MT][2], qs1[MT][2];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint4 w = qf[(((t0q + m) * 4 + k) * 2 + h) * 32 + lane];
                qa[m][k][h][0] = w.x; qa[m][k][h][1] = w.y; qa[m][k][h][2] = w.z; qa[m][k][h][3] = w.w;
            }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float* ri = rowinfo + ((t0q + m) * 16 + h * 8 + gid) * kRowInfo;
            rs[m][h] = ri[0];
            qs0[m][h] = K_MIN ? ri[1] : 0.0f;
            qs1[m][h] = K_MIN ? ri[2] : 0.0f;
        }
    }
    float O[MT][8][4], base[MT][2], thr[MT][2], l[MT][2], om[MT][2][2];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) O[m][j][i] = 0.0f;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            base[m][h] = 0.0f;
            thr[m][h] = -INFINITY;  // nothing seen: any score raises the reference
            l[m][h] = 0.0f;
            om[m][h][0] = om[m][h][1] = 0.0f;
        }
    }
    int ev = 0;
    bool ev_set = false;

    // tables of this tile: [head][K scale, K min, V scale, V min][block][key]
    float* tab = reinterpret_cast<float*>(smem + L.tab);
    constexpr int oKm = K_Q ? 2 * kKeys : 0, oV = oKm + (K_MIN ? 2 * kKeys : 0), oVm = oV + (V_Q ? 2 * kKeys : 0);
    uint32_t* maxv = reinterpret_cast<uint32_t*>(smem + L.maxv);

    int slot = 0, free_slot = sh.stages - 1;  // of tile t, and of the tile before it, which every warp has left
    for (int t = 0; t < n_local; ++t) {
        if (sh.stages == 3) cp_async_wait<1>();
        else cp_async_wait<0>();
        __syncthreads();
        issue(t + sh.stages - 1, free_slot);
        const uint8_t* kt = smem + L.ring + slot * L.stage;
        free_slot = slot;
        slot = slot + 1 == sh.stages ? 0 : slot + 1;
        const uint8_t* vt = kt + L.k_bytes;
        const int tile = tile0 + t;
        const bool draft = tile >= x.cache_tiles;
        const int p0 = (draft ? tile - x.cache_tiles : tile) * kKeys;
        const int count = min(kKeys, (draft ? x.n : x.L) - p0);
        if constexpr (K_Q || V_Q) {
            for (int i = tid; i < sh.hc * 2 * kKeys; i += kWarps * 32) {
                const int key = i % kKeys, hb = i / kKeys;  // hb = head * 2 + block
                float* tb = tab + (hb >> 1) * (L.tab_head / 4) + (hb & 1) * kKeys + key;
                if constexpr (K_Q) {
                    const uint8_t* g = kt + key * strideK + hb * group_bytes(KT);
                    const float d = h2f((uint16_t)ld_u16(g));
                    tb[0] = d;
                    if constexpr (K_MIN) {
                        constexpr float kCentre = BlockTraits<KT>::OFF_QH >= 0 ? 16.0f : 8.0f;
                        tb[oKm] = fmaf(kCentre, d, h2f((uint16_t)ld_u16(g + BlockTraits<KT>::OFF_M)));
                    }
                }
                if constexpr (V_Q) {
                    float d, m;
                    dmma::vscale<VT>(vt + key * strideV + hb * group_bytes(VT), d, m);
                    tb[oV] = d;
                    if constexpr (V_MIN) tb[oVm] = m;
                    const uint32_t mx = __reduce_max_sync(0xffffffffu, __float_as_uint(fabsf(d)) & (isfinite(d) ? 0xffffffffu : 0u));
                    if (lane == 0 && mx) atomicMax(&maxv[(t & 1) * 2 + (hb >> 1)], mx);
                }
            }
            __syncthreads();
            if (tid < 2) maxv[((t + 1) & 1) * 2 + tid] = 0u;
        }
        if (idle) continue;
        float vf = 1.0f;  // 2^ev
        if constexpr (V_Q) {
            const float mv = __uint_as_float(maxv[(t & 1) * 2 + wh]);
            if (mv > 0.0f) {
                const int now = ev_set ? dstream::ilog2f(mv) + ev : 0;
                if (!ev_set || now < dmma::kEvMin || now > dmma::kEvMax) {
                    const int evn = dstream::v_exp_target(mv);
                    if (ev_set) {
                        const float f = pow2f(evn - ev);
#pragma unroll
                        for (int m = 0; m < MT; ++m)
#pragma unroll
                            for (int j = 0; j < 8; ++j)
#pragma unroll
                                for (int i = 0; i < 4; ++i) O[m][j][i] *= f;
                    }
                    ev = evn;
                    ev_set = true;
                }
            }
            vf = pow2f(ev);
        }
        const uint8_t* kh = kt + wh * sliceK;
        const uint8_t* vh = vt + wh * sliceV;
        const float* th = tab + wh * (L.tab_head / 4);

        auto step = [&](auto masked_tag, int sub) {
            constexpr bool kMasked = decltype(masked_tag)::value;  // some (row, key) of the step may be unseen
            float sc[MT][2][4];
            {
                float acc[MT][K_Q ? 2 : 1][2][4];
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int b = 0; b < (K_Q ? 2 : 1); ++b)
#pragma unroll
                        for (int tt = 0; tt < 2; ++tt)
#pragma unroll
                            for (int i = 0; i < 4; ++i) acc[m][b][tt][i] = 0.0f;
#pragma unroll
                for (int tt = 0; tt < 2; ++tt) {
                    const uint8_t* g = kh + (kSub * sub + 8 * tt + gid) * strideK;
                    uint32_t r[4];
                    k_frag<KT, 0>(g, tig, r);
#pragma unroll
                    for (int m = 0; m < MT; ++m) {
                        mma16816(acc[m][0][tt], qa[m][0][0], r[0], r[1]);
                        mma16816(acc[m][0][tt], qa[m][0][1], r[0], r[1]);
                        mma16816(acc[m][0][tt], qa[m][1][0], r[2], r[3]);
                        mma16816(acc[m][0][tt], qa[m][1][1], r[2], r[3]);
                    }
                    k_frag<KT, 1>(g, tig, r);
                    constexpr int b1 = K_Q ? 1 : 0;
#pragma unroll
                    for (int m = 0; m < MT; ++m) {
                        mma16816(acc[m][b1][tt], qa[m][2][0], r[0], r[1]);
                        mma16816(acc[m][b1][tt], qa[m][2][1], r[0], r[1]);
                        mma16816(acc[m][b1][tt], qa[m][3][0], r[2], r[3]);
                        mma16816(acc[m][b1][tt], qa[m][3][1], r[2], r[3]);
                    }
                }
#pragma unroll
                for (int tt = 0; tt < 2; ++tt) {
                    const int c = kSub * sub + 8 * tt + 2 * tig;
                    if constexpr (K_Q) {
                        const float2 d0 = *reinterpret_cast<const float2*>(th + c), d1 = *reinterpret_cast<const float2*>(th + kKeys + c);
                        float2 m0 = make_float2(0.f, 0.f), m1 = m0;
                        if constexpr (K_MIN) {
                            m0 = *reinterpret_cast<const float2*>(th + oKm + c);
                            m1 = *reinterpret_cast<const float2*>(th + oKm + kKeys + c);
                        }
#pragma unroll
                        for (int m = 0; m < MT; ++m)
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const int h = i >> 1;
                                const float e0 = (i & 1) ? d0.y : d0.x, e1 = (i & 1) ? d1.y : d1.x;
                                const float v = fmaf(acc[m][0][tt][i], e0, acc[m][1][tt][i] * e1);
                                float off = -base[m][h];
                                if constexpr (K_MIN)
                                    off = fmaf((i & 1) ? m0.y : m0.x, qs0[m][h], fmaf((i & 1) ? m1.y : m1.x, qs1[m][h], off));
                                sc[m][tt][i] = fmaf(v, rs[m][h], off);
                            }
                    } else {
#pragma unroll
                        for (int m = 0; m < MT; ++m)
#pragma unroll
                            for (int i = 0; i < 4; ++i) sc[m][tt][i] = fmaf(acc[m][0][tt][i], rs[m][i >> 1], -base[m][i >> 1]);
                    }
                }
            }
            if constexpr (kMasked) {
                const int j0 = p0 + kSub * sub, left = count - kSub * sub;  // keys of this step that exist
                const uint32_t exist = left >= kSub ? 0xffffu : (left <= 0 ? 0u : (1u << left) - 1u);
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int r = r0 + (rt0 + m) * 16 + h * 8 + gid;
                        uint32_t bits = r < rows ? exist : 0u;
                        if (draft && bits) {
                            const int node = r / a.G;
                            if (a.mask)
                                bits &= a.mask[(int64_t)s * a.mask_nb_seq + (int64_t)node * a.mask_words + (j0 >> 5)] >> (j0 & 31);
                            else if (node < j0 + kSub - 1)
                                bits &= node < j0 ? 0u : (2u << (node - j0)) - 1u;
                        }
#pragma unroll
                        for (int tt = 0; tt < 2; ++tt)
#pragma unroll
                            for (int e = 0; e < 2; ++e)
                                if (!((bits >> (8 * tt + 2 * tig + e)) & 1u)) sc[m][tt][2 * h + e] = -INFINITY;
                    }
            }
            float mx[MT][2];
            bool over = false;
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    mx[m][h] = fmaxf(fmaxf(sc[m][0][2 * h], sc[m][0][2 * h + 1]), fmaxf(sc[m][1][2 * h], sc[m][1][2 * h + 1]));
                    over |= mx[m][h] > thr[m][h];
                }
            if (__any_sync(0xffffffffu, over)) {
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float top = quad_max(mx[m][h]);
                        if (top > thr[m][h]) {
                            const float up = top - kOffs;
                            const float f = thr[m][h] == -INFINITY ? 0.0f : fast_exp2(-up);
                            base[m][h] += up;
                            thr[m][h] = kLazy + kOffs;
                            l[m][h] *= f;
                            om[m][h][0] *= f;
                            om[m][h][1] *= f;
#pragma unroll
                            for (int j = 0; j < 8; ++j) {
                                O[m][j][2 * h] *= f;
                                O[m][j][2 * h + 1] *= f;
                            }
#pragma unroll
                            for (int tt = 0; tt < 2; ++tt) {
                                sc[m][tt][2 * h] -= up;
                                sc[m][tt][2 * h + 1] -= up;
                            }
                        }
                    }
            }
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int tt = 0; tt < 2; ++tt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        sc[m][tt][i] = fast_exp2(sc[m][tt][i]);
                        l[m][i >> 1] += sc[m][tt][i];
                    }
            // V fragments: b0 of keys 2 tig, 2 tig + 1, b1 of the keys 8 further, for the 8 dim tiles
            const uint8_t* g0 = vh + (kSub * sub + 2 * tig) * strideV;
            const uint8_t* g1 = g0 + 8 * strideV;
            float2 dv[2][2];  // [block][8-key tile]
            if constexpr (V_Q) {
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int tt = 0; tt < 2; ++tt) {
                        dv[b][tt] = *reinterpret_cast<const float2*>(th + oV + b * kKeys + kSub * sub + 8 * tt + 2 * tig);
                        dv[b][tt].x *= vf;
                        dv[b][tt].y *= vf;
                    }
            }
            if constexpr (kMasked) {
                // Drafts hold anything where no row may look: a step whose values are not all finite is added up key by
                // key, and keys that a row does not see are left out instead of being multiplied by zero.
                bool special = false;
                if (draft) {
                    if constexpr (V_Q) {
#pragma unroll
                        for (int b = 0; b < 2; ++b)
#pragma unroll
                            for (int tt = 0; tt < 2; ++tt) special |= !isfinite(dv[b][tt].x) || !isfinite(dv[b][tt].y);
                        if constexpr (V_MIN) {
#pragma unroll
                            for (int b = 0; b < 2; ++b)
#pragma unroll
                                for (int tt = 0; tt < 2; ++tt) {
                                    const float2 vm = *reinterpret_cast<const float2*>(th + oVm + b * kKeys + kSub * sub + 8 * tt + 2 * tig);
                                    special |= !isfinite(vm.x) || !isfinite(vm.y);
                                }
                        }
                    } else {
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const uint4 w = *reinterpret_cast<const uint4*>((k & 2 ? g1 : g0) + (k & 1) * strideV + 16 * gid);
                            special |= f16x2_special(w.x) || f16x2_special(w.y) || f16x2_special(w.z) || f16x2_special(w.w);
                        }
                    }
                }
                if (__any_sync(0xffffffffu, special)) {
#pragma unroll
                    for (int tt = 0; tt < 2; ++tt)
#pragma unroll
                        for (int e = 0; e < 2; ++e)
                            for (int o = 0; o < 4; ++o) {
                                const uint8_t* g = vh + (kSub * sub + 8 * tt + 2 * o + e) * strideV;
#pragma unroll
                                for (int m = 0; m < MT; ++m) {
                                    const float pa = __shfl_sync(0xffffffffu, sc[m][tt][e], (lane & ~3) | o);
                                    const float pb = __shfl_sync(0xffffffffu, sc[m][tt][2 + e], (lane & ~3) | o);
#pragma unroll
                                    for (int j = 0; j < 8; ++j)
#pragma unroll
                                        for (int c = 0; c < 2; ++c) {
                                            const int d = v_dim<VT>(2 * tig + c, j);
                                            const float v = dequant_elem<VT>(g + (d >> 5) * group_bytes(VT), d & 31);
                                            if (pa != 0.0f) O[m][j][c] = fmaf(pa * vf, v, O[m][j][c]);
                                            if (pb != 0.0f) O[m][j][2 + c] = fmaf(pb * vf, v, O[m][j][2 + c]);
                                        }
                                }
                            }
                    return;
                }
            }
            if constexpr (V_MIN) {
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int tt = 0; tt < 2; ++tt) {
                        const float2 vm = *reinterpret_cast<const float2*>(th + oVm + b * kKeys + kSub * sub + 8 * tt + 2 * tig);
#pragma unroll
                        for (int m = 0; m < MT; ++m)
#pragma unroll
                            for (int h = 0; h < 2; ++h)
                                om[m][h][b] = fmaf(sc[m][tt][2 * h], vm.x, fmaf(sc[m][tt][2 * h + 1], vm.y, om[m][h][b]));
                    }
            }
            if constexpr (V_Q) {
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    uint32_t v0[4], v1[4];
                    if (b == 0) {
                        dmma::vfrag<VT, 0>(g0, g0 + strideV, gid, v0);
                        dmma::vfrag<VT, 0>(g1, g1 + strideV, gid, v1);
                    } else {
                        dmma::vfrag<VT, 1>(g0 + group_bytes(VT), g0 + strideV + group_bytes(VT), gid, v0);
                        dmma::vfrag<VT, 1>(g1 + group_bytes(VT), g1 + strideV + group_bytes(VT), gid, v1);
                    }
#pragma unroll
                    for (int m = 0; m < MT; ++m) {
                        uint32_t hi[4], lo[4];
#pragma unroll
                        for (int tt = 0; tt < 2; ++tt)
#pragma unroll
                            for (int h = 0; h < 2; ++h)
                                split2(sc[m][tt][2 * h] * dv[b][tt].x, sc[m][tt][2 * h + 1] * dv[b][tt].y, hi[2 * tt + h], lo[2 * tt + h]);
#pragma unroll
                        for (int jj = 0; jj < 4; ++jj) {
                            mma16816(O[m][4 * b + jj], hi, v0[jj], v1[jj]);
                            mma16816(O[m][4 * b + jj], lo, v0[jj], v1[jj]);
                        }
                    }
                }
            } else {
                const uint4 wa = *reinterpret_cast<const uint4*>(g0 + 16 * gid);
                const uint4 wb = *reinterpret_cast<const uint4*>(g0 + strideV + 16 * gid);
                const uint4 wc = *reinterpret_cast<const uint4*>(g1 + 16 * gid);
                const uint4 wd = *reinterpret_cast<const uint4*>(g1 + strideV + 16 * gid);
                const uint32_t A[4] = {wa.x, wa.y, wa.z, wa.w}, B[4] = {wb.x, wb.y, wb.z, wb.w};
                const uint32_t C[4] = {wc.x, wc.y, wc.z, wc.w}, D[4] = {wd.x, wd.y, wd.z, wd.w};
                uint32_t hi[MT][4], lo[MT][4];
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int tt = 0; tt < 2; ++tt)
#pragma unroll
                        for (int h = 0; h < 2; ++h)
                            split2(sc[m][tt][2 * h], sc[m][tt][2 * h + 1], hi[m][2 * tt + h], lo[m][2 * tt + h]);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const uint32_t pick = (j & 1) ? 0x7632u : 0x5410u;
                    const uint32_t b0 = __byte_perm(A[j >> 1], B[j >> 1], pick), b1 = __byte_perm(C[j >> 1], D[j >> 1], pick);
#pragma unroll
                    for (int m = 0; m < MT; ++m) {
                        mma16816(O[m][j], hi[m], b0, b1);
                        mma16816(O[m][j], lo[m], b0, b1);
                    }
                }
            }
        };
        const int steps = (count + kSub - 1) / kSub;
        for (int sub = wk; sub < steps; sub += sh.wk) {
            if (draft || count - sub * kSub < kSub) step(std::true_type{}, sub);
            else step(std::false_type{}, sub);
        }
    }
    cp_async_wait<0>();
    __syncthreads();
    griddep_launch_dependents();

    // every warp's rows to shared memory as (m, l) and f32 outputs, joined over the WK slices
    constexpr int kOutPad = kD + 4;
    float* ob = reinterpret_cast<float*>(smem + L.ring);
    float2* ml = reinterpret_cast<float2*>(ob + kWarps * MT * 16 * kOutPad);
    const float uf = V_Q ? pow2f(-ev) : 1.0f;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int row = (warp * MT + m) * 16 + h * 8 + gid;
            const float ls = quad_sum(l[m][h]);
            float o0 = 0.0f, o1 = 0.0f;
            if constexpr (V_MIN) {
                o0 = quad_sum(om[m][h][0]);
                o1 = quad_sum(om[m][h][1]);
            }
            if (tig == 0) ml[row] = make_float2(thr[m][h] == -INFINITY && ls == 0.0f ? -INFINITY : base[m][h], ls);  // (NaN scores raise nothing)
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int c = 0; c < 2; ++c)
                    ob[row * kOutPad + v_dim<VT>(2 * tig + c, j)] = fmaf(O[m][j][2 * h + c], uf, j < 4 ? o0 : o1);
        }
    __syncthreads();
    const int tiles_head = sh.wr * MT;
    for (int i = tid; i < sh.hc * tiles_head * 16 * 16; i += kWarps * 32) {
        const int c = i & 15, rr = i >> 4, hd = rr / (tiles_head * 16), rl = rr % (tiles_head * 16);
        const int r = r0 + rl;
        if (r >= all_rows || (!direct && r >= rows)) continue;
        // slices: warps hd * WR * WK + k * WR + (row group), tile inside the group
        const int g = rl / (16 * MT), in = rl % (16 * MT);
        float M = -INFINITY;
        for (int k = 0; k < sh.wk; ++k) M = fmaxf(M, ml[((hd * sh.wk + k) * sh.wr + g) * MT * 16 + in].x);
        float sum = 0.0f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        if (M != -INFINITY)
            for (int k = 0; k < sh.wk; ++k) {
                const int row = ((hd * sh.wk + k) * sh.wr + g) * MT * 16 + in;
                const float2 e = ml[row];
                if (e.x == -INFINITY) continue;
                const float f = exp2f(e.x - M);
                const float4 v = *reinterpret_cast<const float4*>(ob + row * kOutPad + 4 * c);
                sum = fmaf(f, e.y, sum);
                o.x = fmaf(f, v.x, o.x); o.y = fmaf(f, v.y, o.y); o.z = fmaf(f, v.z, o.z); o.w = fmaf(f, v.w, o.w);
            }
        const int kvh = hg * sh.hc + hd;
        if (direct) {
            const bool seen = M != -INFINITY && r < rows;
            const float inv = seen ? 1.0f / sum : 0.0f;
            const int node = r / a.G, h = kvh * a.G + r % a.G;
            *reinterpret_cast<float4*>(a.out + (int64_t)s * a.out_nb_seq + (int64_t)node * a.out_nb_node + h * kD + c * 4) =
                seen ? make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv) : make_float4(0.f, 0.f, 0.f, 0.f);
            if (a.lse && c == 0)
                a.lse[((int64_t)s * a.max_nodes + node) * a.Hq + h] = seen ? (M + log2f(sum)) * 0.69314718055994531f : -INFINITY;
        } else {
            const int64_t slot = (((int64_t)s * a.Hkv + kvh) * a.n_splits + split) * all_rows + r;
            *reinterpret_cast<float4*>(a.ws_o + slot * kD + c * 4) = o;
            if (c == 0) *reinterpret_cast<float2*>(a.ws_ml + slot * 2) = make_float2(M, sum);
        }
    }
}

// Launch for K type KT (tree_mma_inst.cu, one unit per K type).
template <int KT> cudaError_t launch_mma_for_k(cudaStream_t stream, const Args& a, const Shape& sh, int mt);

}  // namespace tree
}  // namespace cvattn
