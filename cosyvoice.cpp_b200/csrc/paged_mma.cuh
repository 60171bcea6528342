// paged_mma.cuh -- paged attention of few rows on warp-level tensor-core MMAs (mma.sync m16n8k16, f16 operands, f32
// accumulators).
//
// Codes are exact in f16.  A row of Q is scaled by a
// power of two and split into f16 hi + lo, which lie 8 rows apart in one A operand: a product over 16 rows serves 8 rows of
// queries, and the sum of its two halves is the score.  P is split without a power of its own, so what is
// left out of a weight is 2^-22 of it or 2^-32 of the row's largest.  (With the power that the tcgen05 kernel has, which follows weight
// times value scale, 64 sequences of one token over up to 4096 took 13.6 us in place of 13.2.)  A block of 16 positions has
// its scale of the keys multiplied to the scores, its scale of the values to the block's output, which is a fresh accumulator
// added to f32 registers.  So every product is exact, and no sum stays in the tensor cores (whose adds truncate) for longer.
//
// A warp takes 8 R rows and every WK-th pair of blocks of its CTA's share; each lane copies (cp.async) the 64 bytes of a block that it
// reads itself, so that a ring of its own needs no barrier.  WR row groups x WK shares are the CTA's 4 warps.  The CTAs of a
// cluster share the positions of a unit (sequence, KV head, row tile) and join through distributed shared memory; where one
// cluster per unit would leave SMs idle, several do, and paged_combine_kernel joins their parts.
//
// What bounds it: 64 sequences of one token over up to 4096, 14 / 2 heads, e4m3: 13.3 us for 33 MB.  Of 19 thousand cycles the loop is
// 9 to 10 (6 to 7 TB/s while it runs), 5 pass before its first block is there (length, page, scale, block: four dependent loads),
// 4 in the joins.  Steps of one block: 20.7 us, as a warp's waits come twice as often; e4m3 turned into f16 by shifts and a product
// in place of its conversion instruction 19.2 where that has 15.0.  CTAs: one wave at 4 (3 with 16 rows a warp) on an SM; two waves
// 18.6, half a wave 15.5.
#pragma once

#include "decode_mma.cuh"
#include "paged.cuh"

namespace cvattn {
namespace paged {

using dmma::mma16816;
using dmma::quad_max;
using dmma::quad_sum;
using dtc::pow2f;

constexpr int kMmaWarps = 4;
constexpr int kStages = 3;               // steps in flight per warp
constexpr int kPair = 2;                 // blocks of a step
constexpr int kStageBytes = kPair * 2 * kBlockBytes;
constexpr int kMaxCluster = 8;
constexpr float kLazy = 8.0f;            // a running maximum is raised when a score passes it by 2^8
constexpr float kOffs = 7.0f;            // P is kept 2^7 larger, far from f16's subnormals

struct AttArgs {
    cvattn_paged_attention_params p;
    int G, blocks;                       // query heads per KV head; blocks of a page
    int n_splits;                        // clusters per unit
    uint32_t by_G, by_parts;             // inverse_of(G); of the CTAs that share a unit (tcgen05: the list)
    float scale_log2;
    float *ws_ml, *ws_o;                 // [seq][KV head][split][max_q * G][2], [..][64]
    int* status;
};

// x / n for x below 2^31 / n, without a division (which takes some 25 instructions, on the way to a CTA's first load): with
// inverse = (2^31 + e) / n, e < n, the product is off by x e / (n 2^31) < 1 / n.
__host__ __device__ constexpr uint32_t inverse_of(uint32_t n) { return ((1u << 31) + n - 1) / n; }
__device__ __forceinline__ int divided(int x, uint32_t inverse) { return (int)__umulhi((uint32_t)x << 1, inverse); }
// c / parts of n, c <= parts <= 2^10.
__device__ __forceinline__ int cut_at(int c, int n, int parts, uint32_t by_parts) {
    const uint32_t q = (uint32_t)n / (uint32_t)parts, rest = (uint32_t)n - q * parts;
    return c * (int)q + divided(c * (int)rest, by_parts);
}

__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t peer_addr(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ float4 peer_ld4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float2 peer_ld2(uint32_t addr) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0,%1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
    return v;
}

// Four codes as two pairs of f16.
template <int F> __device__ __forceinline__ void to_f16(uint32_t w, uint32_t& a, uint32_t& b) {
    if constexpr (F == kI8) {
        a = dtc::hsub2_u32(__byte_perm(w, 0x64646464u, 0x4140u), dtc::kF16x2_1152);
        b = dtc::hsub2_u32(__byte_perm(w, 0x64646464u, 0x4342u), dtc::kF16x2_1152);
    } else {
        asm("{\n\t.reg .b16 x, y;\n\tmov.b32 {x, y}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, x;\n\tcvt.rn.f16x2.e4m3x2 %1, y;\n\t}"
            : "=r"(a), "=r"(b) : "r"(w));
    }
}

__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    unsigned long long ra = *reinterpret_cast<unsigned long long*>(&a), rb = *reinterpret_cast<unsigned long long*>(&b), rd;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(rd) : "l"(ra), "l"(rb));
    return *reinterpret_cast<float2*>(&rd);
}
// x = hi + lo in f16 pairs, hi the nearest.
__device__ __forceinline__ void split_near(float2 x, uint32_t& hi, uint32_t& lo) {
    hi = tc::pack_f16x2(x.x, x.y);
    float a, b;
    asm("{\n\t.reg .b16 h, g;\n\tmov.b32 {h, g}, %2;\n\tfma.rn.f32.f16 %0, h, %3, %4;\n\tfma.rn.f32.f16 %1, g, %3, %5;\n\t}"
        : "=f"(a), "=f"(b) : "r"(hi), "h"((uint16_t)0xBC00u), "f"(x.x), "f"(x.y));
    lo = tc::pack_f16x2(a, b);
}
// Power of two that brings a row's largest query value into [128, 256) (from 2^-119 on; smaller ones it makes normal).
__device__ __forceinline__ int query_exp(float amax) { return min(7 - (max((__float_as_int(amax) >> 23) & 0xff, 1) - 127), 126); }
// A product into a fresh accumulator.
__device__ __forceinline__ void mma_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}

// The lengths of one sequence; (0, 0) if they are out of range.
struct AttLens {
    int L, n;
};
__device__ __forceinline__ AttLens att_lens(const AttArgs& a, int s, bool record) {
    AttLens x;
    x.L = a.p.kv_len[s];
    x.n = a.p.n_q ? a.p.n_q[s] : a.p.max_q;
    if (x.L < 0 || x.L > a.p.max_kv_len || x.n < 0 || x.n > a.p.max_q) {
        if (record) record_status(a.status, kStatusBadLength);
        x.L = x.n = 0;
    }
    return x;
}

// Joins parts (max, sum, output) of a row, and writes it or its part of a split.
struct Join {
    float M = -INFINITY, l = 0.0f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    __device__ __forceinline__ void add(float2 ml, float4 v) {  // M known
        if (ml.x == -INFINITY) return;
        const float f = exp2f(ml.x - M);
        l = fmaf(f, ml.y, l);
        o.x = fmaf(f, v.x, o.x); o.y = fmaf(f, v.y, o.y); o.z = fmaf(f, v.z, o.z); o.w = fmaf(f, v.w, o.w);
    }
    __device__ __forceinline__ void write(const AttArgs& a, int s, int kvh, int r, int c) const {
        const bool seen = M != -INFINITY;
        const float inv = seen ? 1.0f / l : 0.0f;
        const int tok = divided(r, a.by_G), h = kvh * a.G + r - tok * a.G;
        *reinterpret_cast<float4*>(a.p.out + (int64_t)s * a.p.out_nb_seq + (int64_t)tok * a.p.out_nb_tok + h * kD + c * 4) =
            make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
        if (a.p.lse && c == 0)
            a.p.lse[((int64_t)s * a.p.max_q + tok) * a.p.n_q_heads + h] = seen ? (M + log2f(l)) * 0.69314718055994531f : -INFINITY;
    }
    __device__ __forceinline__ void part(const AttArgs& a, int s, int kvh, int split, int r, int c) const {
        const int64_t slot = (((int64_t)s * a.p.pool.n_heads + kvh) * a.n_splits + split) * (a.p.max_q * a.G) + r;
        if (M != -INFINITY) *reinterpret_cast<float4*>(a.ws_o + slot * kD + c * 4) = o;
        if (c == 0) *reinterpret_cast<float2*>(a.ws_ml + slot * 2) = make_float2(M, l);
    }
};

template <int R> struct MmaSmem {
    static constexpr int kRows = 8 * R;                          // of a warp
    static constexpr int kRing = kMmaWarps * kStages * kStageBytes;
    static constexpr int kScales = kMmaWarps * kStages * kPair * 8;
    static constexpr int kPad = kD + 4;
    // (at the end, in the ring's place) the warps' rows, then the CTA's
    static constexpr int kOut = kMmaWarps * kRows * kPad * 4, kMl = kMmaWarps * kRows * 8;
    static constexpr int kEnd = 2 * (kOut + kMl);
    static constexpr int kBytes = (kRing > kEnd ? kRing : kEnd) + kScales;
};

template <int F, int R>
__global__ void __launch_bounds__(kMmaWarps * 32, R == 1 ? 4 : 3) paged_mma_kernel(const __grid_constant__ AttArgs a) {
    using S = MmaSmem<R>;
    extern __shared__ __align__(1024) uint8_t smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gid = lane >> 2, tig = lane & 3;
    const int s = blockIdx.z;
    const int kvh = blockIdx.y % a.p.pool.n_heads, r0 = blockIdx.y / a.p.pool.n_heads * (S::kRows * kMmaWarps);
    const int C = cluster_size(), rank = cluster_rank(), split = blockIdx.x / C;
    griddep_wait();
    const AttLens x = att_lens(a, s, tid == 0 && blockIdx.x == 0 && blockIdx.y == 0);
    const int rows = x.n * a.G, all_rows = a.p.max_q * a.G;
    // this warp: rows rw .., blocks first + wk, + WK, .. of the CTA's share
    const int groups = (min(rows - r0, S::kRows * kMmaWarps) + S::kRows - 1) / S::kRows;
    const int WR = groups <= 1 ? 1 : groups <= 2 ? 2 : 4, WK = kMmaWarps / WR;
    const int wr = warp % WR, wk = warp / WR;
    const int rw = r0 + wr * S::kRows;
    // row r of token i sees the positions below L - n + i + 1
    const int before = x.L - x.n + 1;
    const int last_row = min(rows, r0 + S::kRows * kMmaWarps) - 1;
    const int end = last_row >= r0 ? max(0, before + divided(last_row, a.by_G)) : 0;
    const int n_blocks = (end + kBlock - 1) / kBlock, shares = C * a.n_splits, share = split * C + rank;
    const int n_steps = (n_blocks + kPair - 1) / kPair;
    const int s0 = cut_at(share, n_steps, shares, a.by_parts), s1 = cut_at(share + 1, n_steps, shares, a.by_parts);
    const int steps = rw < rows ? max(0, (s1 - s0 - wk + WK - 1) / WK) : 0;

    const int32_t* table = a.p.table + (int64_t)s * a.p.table_nb_seq;
    const int shift = __ffs(a.blocks) - 1;
    // lane i knows of block i & 1 of the warp's step 16 c + i / 2: where it lies, and its scales
    int64_t off = 0, next_off = 0;
    float2 sc = make_float2(-1.0f, 0.0f), next_sc = sc;  // (-1: not seen)
    auto look = [&](int chunk, int64_t& o, float2& f) {
        const int b = kPair * (s0 + wk + (16 * chunk + (lane >> 1)) * WK) + (lane & 1);
        o = 0;
        f = make_float2(-1.0f, 0.0f);
        if (16 * chunk + (lane >> 1) >= steps || b >= n_blocks) return;
        const int entry = b >> shift, page = page_of(table, entry, a.p.pool.n_pages);
        if (page < 0) {
            record_status(a.status, kStatusBadPage);
            return;
        }
        const int in = ((kvh - entry) << shift) + b;
        o = page * a.p.pool.nb_page + (int64_t)in * kBlockBytes;
        f.x = a.p.pool.k_scale[page * a.p.pool.nb_scale + in];
        f.y = a.p.pool.v_scale[page * a.p.pool.nb_scale + in];
    };
    const uint8_t* kp = static_cast<const uint8_t*>(a.p.pool.k) + (4 * (gid >> 1) + (gid & 1)) * kD + 16 * tig;
    const uint8_t* vp = static_cast<const uint8_t*>(a.p.pool.v) + lane * 16;
    const uint8_t* ring = smem + warp * kStages * kStageBytes;
    const uint32_t ring_at = smem_addr(ring) + lane * 16;
    float2* scales = reinterpret_cast<float2*>(smem + S::kBytes - S::kScales) + warp * kStages * kPair;
    int to = 0;  // the slot that is filled next
    auto issue = [&](int k) {
        if (k < steps) {
            if (k && (k & 15) == 0) {
                off = next_off;
                sc = next_sc;
            }
            if ((k & 15) == 4) look((k >> 4) + 1, next_off, next_sc);
#pragma unroll
            for (int e = 0; e < kPair; ++e) {
                const int64_t at = __shfl_sync(0xffffffffu, off, 2 * (k & 15) + e);
                const uint32_t dst = ring_at + to * kStageBytes + e * 2 * kBlockBytes;
                copy16(dst, kp + at);
                copy16(dst + 512, kp + at + 2 * kD);
                copy16(dst + 1024, vp + at);
                copy16(dst + 1536, vp + at + 512);
            }
            if ((lane >> 1) == (k & 15)) scales[to * kPair + (lane & 1)] = sc;
        }
        to = to + 1 == kStages ? 0 : to + 1;
        copies_done();
    };
    look(0, off, sc);
#pragma unroll
    for (int k = 0; k < kStages - 1; ++k) issue(k);

    uint32_t qa[R][4][4];   // A operands of Q by k-step: rows gid the hi, rows gid + 8 the lo parts
    float rs[R];            // score factors
    int lim[R];             // positions that the row sees
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int r = rw + 8 * i + gid, tok = divided(r, a.by_G);
        const float* q = a.p.q + (int64_t)s * a.p.q_nb_seq + (int64_t)tok * a.p.q_nb_tok + (kvh * a.G + r - tok * a.G) * kD + 16 * tig;
        float4 e[4];
        float am = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            e[j] = r < rows ? *reinterpret_cast<const float4*>(q + 4 * j) : make_float4(0.f, 0.f, 0.f, 0.f);
            am = fmaxf(am, fmaxf(fmaxf(fabsf(e[j].x), fabsf(e[j].y)), fmaxf(fabsf(e[j].z), fabsf(e[j].w))));
        }
        const int ex = query_exp(quad_max(am));
        const float f = pow2f(ex);
        rs[i] = pow2f(-ex) * a.scale_log2;
        lim[i] = r < rows ? before + tok : 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            split_near(make_float2(e[j].x * f, e[j].y * f), qa[i][j][0], qa[i][j][1]);
            split_near(make_float2(e[j].z * f, e[j].w * f), qa[i][j][2], qa[i][j][3]);
        }
    }
    const int sure = before + divided(rw, a.by_G);  // positions below it every row of the warp sees
    float2 O[R][8], l[R];
    float base[R], thr[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        base[i] = 0.0f;
        thr[i] = -INFINITY;  // nothing seen: any score raises the reference
        l[i] = make_float2(0.f, 0.f);
#pragma unroll
        for (int j = 0; j < 8; ++j) O[i][j] = make_float2(0.f, 0.f);
    }

    int slot = 0;
#pragma unroll 1
    for (int k = 0; k < steps; ++k) {
        copies_wait<kStages - 2>();
        __syncwarp();  // the scales of this step; and everybody has left the slot before
        issue(k + kStages - 1);
        const uint4* in = reinterpret_cast<const uint4*>(ring + slot * kStageBytes + lane * 16);
        const float4 f4 = *reinterpret_cast<const float4*>(scales + slot * kPair);
        const float ks[kPair] = {f4.x, f4.z}, vs[kPair] = {f4.y, f4.w};
        slot = slot + 1 == kStages ? 0 : slot + 1;
        float2 sco[R][2 * kPair];  // scores by block and tile: positions 4 tig + 2 tile, + 1
#pragma unroll
        for (int e = 0; e < kPair; ++e)
#pragma unroll
            for (int tt = 0; tt < 2; ++tt) {
                const uint4 w = in[128 * e + 32 * tt];
                uint32_t b[8];
                to_f16<F>(w.x, b[0], b[1]);
                to_f16<F>(w.y, b[2], b[3]);
                to_f16<F>(w.z, b[4], b[5]);
                to_f16<F>(w.w, b[6], b[7]);
#pragma unroll
                for (int i = 0; i < R; ++i) {
                    float c[4];
                    mma_first(c, qa[i][0], b[0], b[1]);
                    mma16816(c, qa[i][1], b[2], b[3]);
                    mma16816(c, qa[i][2], b[4], b[5]);
                    mma16816(c, qa[i][3], b[6], b[7]);
                    const float g = rs[i] * ks[e];
                    sco[i][2 * e + tt] = ffma2(add2(make_float2(c[0], c[1]), make_float2(c[2], c[3])), make_float2(g, g), make_float2(-base[i], -base[i]));
                }
            }
        const int j0 = kPair * (s0 + wk + k * WK) * kBlock;
        const bool hidden = ks[0] < 0.0f || ks[1] < 0.0f;
        uint32_t there[kPair] = {0xffffffffu, 0xffffffffu};  // the lane's four positions that exist, as bytes
        if (j0 + kPair * kBlock > sure || hidden) {  // some row may not see some position of the step
#pragma unroll
            for (int e = 0; e < kPair; ++e) {
                const int first = j0 + e * kBlock + 4 * tig, exist = ks[e] < 0.0f ? 0 : end - first;
                there[e] = exist >= 4 ? 0xffffffffu : exist <= 0 ? 0u : (1u << (8 * exist)) - 1u;
#pragma unroll
                for (int i = 0; i < R; ++i) {
                    const int left = ks[e] < 0.0f ? 0 : lim[i] - first;
                    if (left < 1) sco[i][2 * e].x = -INFINITY;
                    if (left < 2) sco[i][2 * e].y = -INFINITY;
                    if (left < 3) sco[i][2 * e + 1].x = -INFINITY;
                    if (left < 4) sco[i][2 * e + 1].y = -INFINITY;
                }
            }
        }
        float mx[R];
        bool up = false;
#pragma unroll
        for (int i = 0; i < R; ++i) {
            mx[i] = fmaxf(sco[i][0].x, sco[i][0].y);
#pragma unroll
            for (int t = 1; t < 2 * kPair; ++t) mx[i] = fmaxf(mx[i], fmaxf(sco[i][t].x, sco[i][t].y));
            up |= mx[i] > thr[i];
        }
        if (__any_sync(0xffffffffu, up)) {
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const float top = quad_max(mx[i]);
                if (top > thr[i]) {
                    const float by = top - kOffs, g = thr[i] == -INFINITY ? 0.0f : fast_exp2(-by);
                    base[i] += by;
                    thr[i] = kLazy + kOffs;
                    l[i].x *= g;
                    l[i].y *= g;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        O[i][j].x *= g;
                        O[i][j].y *= g;
                    }
#pragma unroll
                    for (int t = 0; t < 2 * kPair; ++t) {
                        sco[i][t].x -= by;
                        sco[i][t].y -= by;
                    }
                }
            }
        }
        uint32_t pa[R][kPair][4];
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int t = 0; t < 2 * kPair; ++t) {
                sco[i][t] = make_float2(fast_exp2(sco[i][t].x), fast_exp2(sco[i][t].y));
                split_near(sco[i][t], pa[i][t >> 1][2 * (t & 1)], pa[i][t >> 1][2 * (t & 1) + 1]);
                l[i] = add2(l[i], sco[i][t]);
            }
#pragma unroll
        for (int e = 0; e < kPair; ++e)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint4 w = in[128 * e + 64 + 32 * h];
                if (F == kE4M3 && there[e] != 0xffffffffu) {  // (what lies past the end may be NaN)
                    w.x &= there[e];
                    w.y &= there[e];
                    w.z &= there[e];
                    w.w &= there[e];
                }
                uint32_t b[8];
                to_f16<F>(w.x, b[0], b[1]);
                to_f16<F>(w.y, b[2], b[3]);
                to_f16<F>(w.z, b[4], b[5]);
                to_f16<F>(w.w, b[6], b[7]);
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int i = 0; i < R; ++i) {
                        float c[4];
                        mma_first(c, pa[i][e], b[2 * j], b[2 * j + 1]);
                        O[i][4 * h + j] = ffma2(make_float2(vs[e], vs[e]), add2(make_float2(c[0], c[1]), make_float2(c[2], c[3])), O[i][4 * h + j]);
                    }
            }
    }
    griddep_launch_dependents();

    // the warps' rows, joined over the CTA, then over the cluster
    copies_wait<0>();
    __syncthreads();
    float* wo = reinterpret_cast<float*>(smem);
    float2* wml = reinterpret_cast<float2*>(smem + 2 * S::kOut);
    float *co = wo + S::kOut / 4;
    float2* cml = wml + S::kMl / 8;
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int row = warp * S::kRows + 8 * i + gid;
        const float ls = quad_sum(l[i].x + l[i].y);
        // (a row whose scores are all NaN raises nothing, but was seen)
        if (tig == 0) wml[row] = make_float2(thr[i] == -INFINITY && ls == 0.0f ? -INFINITY : base[i], ls);
#pragma unroll
        for (int j = 0; j < 8; ++j) *reinterpret_cast<float2*>(wo + row * S::kPad + 8 * j + 2 * tig) = O[i][j];
    }
    __syncthreads();
    const int here = min(all_rows - r0, S::kRows * kMmaWarps);
    const bool direct = a.n_splits == 1;
    for (int i = tid; i < here * 16; i += kMmaWarps * 32) {
        const int c = i & 15, rl = i >> 4, r = r0 + rl;
        const int w0 = rl / S::kRows, in = rl % S::kRows;  // share k: warp w0 + k * WR
        Join j;
        if (r < rows) {
            for (int k = 0; k < WK; ++k) j.M = fmaxf(j.M, wml[(w0 + k * WR) * S::kRows + in].x);
            for (int k = 0; k < WK; ++k) {
                const int row = (w0 + k * WR) * S::kRows + in;
                j.add(wml[row], *reinterpret_cast<const float4*>(wo + row * S::kPad + 4 * c));
            }
        }
        if (C == 1) {
            if (direct) j.write(a, s, kvh, r, c);
            else j.part(a, s, kvh, split, r, c);
        } else {
            *reinterpret_cast<float4*>(co + rl * S::kPad + 4 * c) = j.o;
            if (c == 0) cml[rl] = make_float2(j.M, j.l);
        }
    }
    if (C == 1) return;
    cluster_arrive();
    cluster_wait();
    const uint32_t oa = smem_addr(co), ma = smem_addr(cml);
    for (int i = tid * C + rank; i < here * 16; i += kMmaWarps * 32 * C) {
        const int c = i & 15, rl = i >> 4;
        float2 ml[kMaxCluster];
        float4 v[kMaxCluster];
        Join j;
#pragma unroll
        for (int k = 0; k < kMaxCluster; ++k)
            if (k < C) {
                ml[k] = peer_ld2(peer_addr(ma + rl * 8, k));
                v[k] = peer_ld4(peer_addr(oa + (rl * S::kPad + 4 * c) * 4, k));
                j.M = fmaxf(j.M, ml[k].x);
            }
#pragma unroll
        for (int k = 0; k < kMaxCluster; ++k)
            if (k < C) j.add(ml[k], v[k]);
        if (direct) j.write(a, s, kvh, r0 + rl, c);
        else j.part(a, s, kvh, split, r0 + rl, c);
    }
    cluster_arrive();  // nobody leaves while others read its rows
    cluster_wait();
}

}  // namespace paged
}  // namespace cvattn
