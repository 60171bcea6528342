// kv_scores_tc.cuh -- attention scores on the 5th-generation tensor cores (tcgen05),
// for f16 and block-quantized caches, many key tiles and up to 512 rows.
//
// The product is taken transposed, S^T = K Q^T: a TMEM lane, and so a thread, is a
// key, and the sum over the rows is a sum along the thread's columns, with no
// exchange at all.  A key's block scales are then two scalars of its thread, so the
// quants go into the product as the integers they are: S = d0 S0 + d1 S1 (+ mins),
// with Q in f16 hi + lo scaled per row.  A group has two S buffers in TMEM (128 rows
// of an f16 cache, 64 of a quantized one, whose S0 and S1 lie side by side), so the
// next rows' product runs while it sums one up.
//
// The key tiles (128 keys) of all units (sequence, KV head) form one list, cut
// evenly over the CTAs; a run is a CTA's part of one unit and shares its Q.
//   warps 0-3, 4-7  groups: tile n of the CTA is summed up by group n & 1; all of them
//                   prepare Q at the start of a run
//   warps 8-11, 12-15  producers of the groups' tiles, a thread per key: f16 tile and
//                   scales from the raw rows; an f16 cache is copied straight into the
//                   tile
//   warps 16, 17    MMA issuers of the groups
//   warp 18         loader: raw rows of the next tiles, one bulk copy each where they hold
//                   at most two heads and lie packed (else the producers copy the slices)
// What bounds it: 8 sequences of 8192 positions, 64 rows of 14 heads, f16: 40.2 us, 187 TFLOP/s.
// A group sums 128 x 128 in 2800 cycles, in which the exponentials of both groups take 2048 of
// the SM's unit; the sums are 34K of a CTA's 63K active cycles (over all of them the unit is 40 %
// busy).  The rest is the start and Q: no product begins before all rows of a run are prepared.
// 64 sequences of up to 4096, 4 rows, Q8_0: 19.9 us for 20 MB; start and change of runs (10K and
// 2K cycles) are half of it, the rest the tiles' conversion.
#pragma once

#include "kv_scores.cuh"
#include "tree_tc.cuh"

namespace cvattn {
namespace kvscore {

using tree::elect_one;
using tree::kTcTile;
using tree::kTcTileBytes;
using tree::max3;
using tree::tc_cut;
using tree::tc_wait;

constexpr int kTcThreads = 19 * 32;
constexpr int kTcMaxSeq = 1024;
constexpr int kTcMaxRows = 512;      // (token, head) rows of a KV head whose Q fits shared memory
constexpr int kTcRowTiles = kTcMaxRows / 128;
constexpr int kTcRawBuffers = 8;
// Tiles whose scales are kept: tile n is written once S of tile n - 2 is done, which a group may still have to read together
// with that of n - 4; S of n - 2 took the buffer of n - 6, whose scales have been read.
constexpr int kTcScales = 6;

struct TcArgs {
    Args a;
    uint32_t inv_g;                  // ceil(2^16 / G)
    int grid;
    int raw_buffers;                 // 2, and what fits the Q tiles that these rows do not need (up to kTcRawBuffers)
};

struct TcBars {
    uint64_t k_full[4], k_empty[4];  // by stage
    uint64_t raw_full[kTcRawBuffers], raw_empty[kTcRawBuffers];
    uint64_t q_full, q_seen;         // by run: written; both issuers know (so they miss none)
    uint64_t s_full[2][2], s_empty[2][2];  // by group and S buffer
    uint32_t tmem_base;
    int err;
    int any_out;                     // some row of the run is left out
};

template <int KT>
struct TcShape {
    static constexpr bool K_Q = KT != kF16;
    static constexpr int kStages = K_Q ? 2 : 4;
    static constexpr int kSRows = K_Q ? 64 : 128;                         // rows of an S buffer
    static constexpr int kQ = 0;                                          // [row tile][hi, lo] tiles
    static constexpr int kTiles = kTcRowTiles * 2 * kTcTileBytes;
    static constexpr int kRaw = kTiles + kStages * kTcTileBytes;          // two buffers of up to two heads' rows
    static constexpr int kRawOne = K_Q ? 2 * kTcTile * raw_stride(KT) : 0;
    static constexpr int kInfo = kRaw + 2 * kRawOne;                      // float2 per row: factor, -log-sum; then the block sums of Q
    static constexpr int kFar = kInfo + kTcMaxRows * 16;
    static constexpr int kScale = kFar + kTcMaxRows * 4;                  // [tile n % 6][scales, mins][block][key]
    static constexpr int kBars = kScale + (K_Q ? kTcScales * 4 * kTcTile * 4 : 0);
    static constexpr int kPref = kBars + (int)((sizeof(TcBars) + 15) / 16 * 16);
    static constexpr int kBytes = kPref + (kTcMaxSeq + 4) * 4;
    static_assert(kBytes <= 227 * 1024, "one CTA per SM");
};

// A CTA's walk through its part of the list.  Lengths are read again where a run starts (they are few).
struct Run {
    int s, kvh, i, end, t0, T, L, n;
    __device__ __forceinline__ void sequence(const Args& a, int seq) {
        s = seq;
        L = a.kv_len[seq];
        n = a.n_rows ? a.n_rows[seq] : a.max_rows;
        T = (L + kTcTile - 1) / kTcTile;
    }
    __device__ __forceinline__ void start(const Args& a, const int32_t* pref, int entry, int hi) {
        i = end = entry;
        if (entry >= hi) return;
        int lo = 0, up = a.n_seq;  // last s with pref[s] <= entry: its list is not empty
        while (up - lo > 1) {
            const int mid = (lo + up) >> 1;
            if (pref[mid] <= entry) lo = mid;
            else up = mid;
        }
        sequence(a, lo);
        kvh = (entry - pref[lo]) / T;
        t0 = entry - pref[lo] - kvh * T;
        end = min(hi, i + T - t0);
    }
    __device__ __forceinline__ void next(const Args& a, const int32_t* pref, int hi) {
        i = end;
        if (i >= hi) return;
        t0 = 0;
        if (++kvh == a.Hkv) {
            kvh = 0;
            int q = s + 1;
            while (pref[q + 1] == i) ++q;  // sequences without entries
            sequence(a, q);
        }
        end = min(hi, i + T);
    }
};

// Row 0 (every head) of the tile at list entry e of run r.
__device__ __forceinline__ const uint8_t* tile_rows(const Args& a, const Run& r, int e) {
    const uint8_t* b = a.k_seq_ptrs ? reinterpret_cast<const uint8_t*>(a.k_seq_ptrs[r.s]) : a.k + (int64_t)r.s * a.k_nb2;
    return b + (int64_t)(r.t0 + e - r.i) * kTcTile * a.k_nb1;
}
// Whether a tile's rows come by one bulk copy: packed, 16-byte aligned, at most two heads.
__device__ __forceinline__ bool whole_rows(const Args& a, const uint8_t* rows, int slice) {
    return a.Hkv <= 2 && a.k_nb1 == a.Hkv * slice && (reinterpret_cast<uintptr_t>(rows) & 15) == 0;
}
// Raw buffers: two behind the tiles, then the end of the Q tiles, whose last ones no row needs.
template <int KT>
__device__ __forceinline__ uint8_t* raw_at(uint8_t* smem, int b) {
    using Sh = TcShape<KT>;
    return b < 2 ? smem + Sh::kRaw + b * Sh::kRawOne : smem + Sh::kTiles - (b - 1) * Sh::kRawOne;
}

template <int KT>
__global__ void __launch_bounds__(kTcThreads, 1) scores_tc_kernel(const __grid_constant__ TcArgs ta) {
    using Sh = TcShape<KT>;
    constexpr bool K_Q = Sh::K_Q, K_MIN = BlockTraits<KT>::HAS_MIN;
    constexpr int kSt = Sh::kStages, slice = 2 * group_bytes(KT);
    extern __shared__ __align__(1024) uint8_t smem[];
    const Args& a = ta.a;
    TcBars* B = reinterpret_cast<TcBars*>(smem + Sh::kBars);
    int32_t* pref = reinterpret_cast<int32_t*>(smem + Sh::kPref);
    if (smem_addr(smem) & 1023u) {
        if (threadIdx.x == 0) record_status(a.status, kStatusTimeout);
        return;
    }
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int i = 0; i < 4; ++i) {
            mbar_init(&B->k_full[i], 128);
            mbar_init(&B->k_empty[i], 1);
        }
        for (int i = 0; i < kTcRawBuffers; ++i) {
            mbar_init(&B->raw_full[i], 1);
            mbar_init(&B->raw_empty[i], 128);
        }
        for (int g = 0; g < 2; ++g) {
            for (int b = 0; b < 2; ++b) {
                mbar_init(&B->s_full[g][b], 1);
                mbar_init(&B->s_empty[g][b], 128);
            }
        }
        mbar_init(&B->q_full, 256);
        mbar_init(&B->q_seen, 2);
        B->err = 0;
        B->any_out = 0;
        fence_mbar_init();
    }
    if (warp == 0) {
        tc::tmem_alloc(&B->tmem_base, 512);
        tc::tmem_relinquish();
    }
    griddep_wait();
    if (warp == 1) {  // list entries before each sequence
        int carry = 0;
        for (int base = 0; base < a.n_seq; base += 32) {
            const int s = base + lane;
            int x = 0, L, n;
            if (s < a.n_seq && lens_of(a, s, L, n, blockIdx.x == 0)) x = (L + kTcTile - 1) / kTcTile * a.Hkv;
            int incl = x;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += y;
            }
            if (s < a.n_seq) pref[s] = carry + incl - x;
            carry += __shfl_sync(0xffffffffu, incl, 31);
        }
        if (lane == 0) pref[a.n_seq] = carry;
    }
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = B->tmem_base;
    const int total = pref[a.n_seq];
    const int lo = tc_cut(blockIdx.x, total, ta.grid), hi = tc_cut(blockIdx.x + 1, total, ta.grid);
    Run r;
    r.start(a, pref, lo, hi);
    float4* info = reinterpret_cast<float4*>(smem + Sh::kInfo);
    float2* qsum = reinterpret_cast<float2*>(smem + Sh::kInfo + kTcMaxRows * 8);
    int* far = reinterpret_cast<int*>(smem + Sh::kFar);
    float* scale = reinterpret_cast<float*>(smem + Sh::kScale);

    if (warp < 8) {
        // ------------------------------------------------------ group g: thread = key of a tile
        const int g = warp >> 2, quad = warp & 3, key = quad * 32 + lane;
        const uint32_t st = tmem + ((uint32_t)(quad * 32) << 16) + g * 256;
        constexpr int kCols = 16;  // columns at a time
        uint32_t k = 0, n_run = 0;  // S tiles of this group, runs so far
        bool ok = true;
        for (; r.i < hi; r.next(a, pref, hi), ++n_run) {
            const int rows = r.n * a.G, R = max(rows, 1);  // (without rows: one that is left out, so that every tile has its S)
            if (n_run) ok = ok && tc_wait(&B->q_seen, (n_run - 1) & 1, &B->err, 59);
            // every S of the last run has been read: its Q may go
            if (!fp::prod_bar_and(1, 256, ok)) { ok = false; break; }
            if (tid == 0) B->any_out = 0;
            asm volatile("bar.sync 2, 256;" ::: "memory");
            // 4 lanes a row, 16 dims each; rows from R to the next multiple of 32 are zeros
            const int c = lane & 3;
#pragma unroll 2
            for (int q0 = warp * 8 + (lane >> 2); q0 < (R + 31) / 32 * 32; q0 += 64) {
                const int t = (int)(((uint32_t)q0 * ta.inv_g) >> 16), h = r.kvh * a.G + q0 - t * a.G;
                float4 v[4];
                float ls = -INFINITY;
                int at = t;
                if (q0 < rows && a.rows) at = a.rows[(int64_t)r.s * a.max_rows + t];
                const bool there = q0 < rows && at >= 0 && at < a.n_q_rows;
                if (there) ls = a.lse[((int64_t)r.s * a.n_q_rows + at) * a.Hq + h];
                else if (q0 < rows) record_status(a.status, kStatusBadPosition);
                const float4* q = reinterpret_cast<const float4*>(a.q + (int64_t)r.s * a.q_nb_seq + (int64_t)at * a.q_nb_node + h * kD + 16 * c);
#pragma unroll
                for (int u = 0; u < 4; ++u) v[u] = there ? q[u] : make_float4(0.f, 0.f, 0.f, 0.f);
                const bool real = ls != -INFINITY;
                if (q0 < R && !real) B->any_out = 1;
                float am = 0.0f, qs = 0.0f;
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    if (!real) v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
                    am = max3(am, fmaxf(fabsf(v[u].x), fabsf(v[u].y)), fmaxf(fabsf(v[u].z), fabsf(v[u].w)));
                    if constexpr (K_MIN) qs += (v[u].x + v[u].y) + (v[u].z + v[u].w);
                }
                am = quad_max(am);
                if constexpr (K_MIN) qs += __shfl_xor_sync(0xffffffffu, qs, 1);  // over the two lanes of a block
                const int ex = dtc::norm_exp(am);
                const float sc = pow2f(ex);
                uint8_t* qh = smem + Sh::kQ + (q0 >> 7) * 2 * kTcTileBytes;
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    uint4 wh, wl;
                    split2(v[2 * u].x * sc, v[2 * u].y * sc, wh.x, wl.x);
                    split2(v[2 * u].z * sc, v[2 * u].w * sc, wh.y, wl.y);
                    split2(v[2 * u + 1].x * sc, v[2 * u + 1].y * sc, wh.z, wl.z);
                    split2(v[2 * u + 1].z * sc, v[2 * u + 1].w * sc, wh.w, wl.w);
                    const uint32_t o = tc::sw128_offset(q0 & 127, 2 * c + u);
                    *reinterpret_cast<uint4*>(qh + o) = wh;
                    *reinterpret_cast<uint4*>(qh + kTcTileBytes + o) = wl;
                }
                if (c == 0) {
                    reinterpret_cast<float2*>(info)[q0] = make_float2(pow2f(-ex) * a.scale_log2, real ? -ls * 1.4426950408889634f : -INFINITY);
                    far[q0] = real ? r.L - r.n + t + 1 : 0;
                }
                if (K_MIN && (c & 1) == 0) reinterpret_cast<float*>(qsum + q0)[c >> 1] = qs * a.scale_log2;
            }
            fence_proxy_async_smem();
            mbar_arrive(&B->q_full);
            asm volatile("bar.sync 2, 256;" ::: "memory");
            const bool any_out = B->any_out != 0;
            for (int j = r.i + ((r.i ^ lo ^ g) & 1); ok && j < r.end; j += 2) {
                const int n = j - lo, p0 = (r.t0 + j - r.i) * kTcTile, count = min(kTcTile, r.L - p0);
                const int64_t at = (int64_t)r.s * a.nb_seq + (int64_t)r.kvh * a.nb_head + p0 + key;
                const float old = key < count ? a.scores[at] : 0.0f;
                const bool masked = any_out || p0 + kTcTile > r.L - r.n + 1;  // some (row, key) may be unseen
                float d0 = 1.0f, d1 = 1.0f, m0 = 0.0f, m1 = 0.0f, s0 = 0.0f, s1 = 0.0f, s2 = 0.0f, s3 = 0.0f;
                for (int r0 = 0; r0 < R; r0 += Sh::kSRows, ++k) {
                    ok = tc_wait(&B->s_full[g][k & 1], (k >> 1) & 1, &B->err, 51);
                    if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
                    tc::fence_after();
                    if (K_Q && r0 == 0) {
                        const float* sp = scale + n % kTcScales * 4 * kTcTile + key;
                        d0 = sp[0];
                        d1 = sp[kTcTile];
                        if constexpr (K_MIN) {
                            m0 = sp[2 * kTcTile];
                            m1 = sp[3 * kTcTile];
                        }
                    }
                    const uint32_t sb = st + (k & 1) * 128;
                    const int cols = min(Sh::kSRows, R - r0);
                    uint32_t u[kCols], w[kCols];
                    auto load = [&](int c) {
                        tc::tmem_ld16(sb + c, u);
                        if constexpr (K_Q) tc::tmem_ld16(sb + 64 + c, w);
                    };
                    load(0);
                    tc::tmem_ld_wait();
#pragma unroll 1
                    for (int c = 0; c < cols; c += kCols) {
                        const float4* ri = info + (r0 + c) / 2;
                        float p[kCols];
#pragma unroll
                        for (int e = 0; e < kCols; e += 2) {
                            const float4 f = ri[e / 2];
                            float o0 = f.y, o1 = f.w;
                            if constexpr (K_MIN) {
                                const float4 qq = reinterpret_cast<const float4*>(qsum + r0 + c)[e / 2];
                                o0 = fmaf(m0, qq.x, fmaf(m1, qq.y, o0));
                                o1 = fmaf(m0, qq.z, fmaf(m1, qq.w, o1));
                            }
                            float v0 = __uint_as_float(u[e]), v1 = __uint_as_float(u[e + 1]);
                            if constexpr (K_Q) {
                                v0 = fmaf(v0, d0, __uint_as_float(w[e]) * d1);
                                v1 = fmaf(v1, d0, __uint_as_float(w[e + 1]) * d1);
                            }
                            p[e] = fmaf(v0, f.x, o0);
                            p[e + 1] = fmaf(v1, f.z, o1);
                        }
                        load(min(c + kCols, Sh::kSRows - kCols));  // under way during the exponentials
#pragma unroll
                        for (int e = 0; e < kCols; ++e) p[e] = fast_exp2(p[e]);
                        if (masked) {
                            const int* fr = far + r0 + c;
#pragma unroll
                            for (int e = 0; e < kCols; ++e)
                                if (p0 + key >= fr[e]) p[e] = 0.0f;
                        }
#pragma unroll
                        for (int e = 0; e < kCols; e += 4) {
                            s0 += p[e];
                            s1 += p[e + 1];
                            s2 += p[e + 2];
                            s3 += p[e + 3];
                        }
                        tc::tmem_ld_wait();
                    }
                    tc::fence_before();
                    mbar_arrive(&B->s_empty[g][k & 1]);
                }
                if (ok && key < count) a.out[at] = fmaf(a.decay, old, (s0 + s1) + (s2 + s3));
            }
            ok = __all_sync(0xffffffffu, ok);
        }
    } else if (warp < 16) {
        // ------------------------------------------------------ producer of group g's tiles: thread = key
        const int g = (warp - 8) >> 2, key = tid - 256 - g * 128;
        const int nbuf = ta.raw_buffers;
        bool ok = true;
        if constexpr (K_Q) {
            for (int n = g; lo + n < hi; n += 2) {
                while (lo + n >= r.end) r.next(a, pref, hi);
                const int count = min(kTcTile, r.L - (r.t0 + lo + n - r.i) * kTcTile), sg = n & 1, b = n % nbuf;
                const uint8_t* src = tile_rows(a, r, lo + n);
                ok = ok && tc_wait(&B->raw_full[b], (n / nbuf) & 1, &B->err, 52);
                if (!fp::prod_bar_and(4 + g, 128, ok)) break;
                uint8_t* raw = raw_at<KT>(smem, b);
                const bool whole = whole_rows(a, src, slice);
                if (!whole) {
                    src += r.kvh * slice;
                    const int unit = ((reinterpret_cast<uint64_t>(src) | (uint64_t)a.k_nb1) & 3) == 0 ? 4 : 2;
                    const int w = slice / unit, per = 128 / w, k0 = key / w, col = (key - k0 * w) * unit;
#pragma unroll 4
                    for (int kk = k0; k0 < per && kk < count; kk += per) {
                        const uint8_t* from = src + (int64_t)kk * a.k_nb1 + col;
                        uint8_t* to = raw + kk * raw_stride(KT) + col;
                        if (unit == 4) tree::cp_async4(to, from, true);
                        else *reinterpret_cast<uint16_t*>(to) = *reinterpret_cast<const uint16_t*>(from);
                    }
                    tree::cp_async_commit();
                    tree::cp_async_wait<0>();
                    asm volatile("bar.sync %0, 128;" ::"r"(4 + g) : "memory");
                }
                if (n >= 2) ok = tc_wait(&B->k_empty[sg], (n / 2 - 1) & 1, &B->err, 54);
                if (ok) {
                    const uint8_t* row = raw + (whole ? key * a.Hkv * slice + r.kvh * slice : key * raw_stride(KT));
                    uint8_t* tile = smem + Sh::kTiles + sg * kTcTileBytes;
                    uint32_t w0[16], w1[16];
                    float d0, m0, d1, m1;
                    convert_block<KT, 0>(row, w0, d0, m0);
                    convert_block<KT, 1>(row, w1, d1, m1);
                    store_block(tile, key, 0, w0);
                    store_block(tile, key, 1, w1);
                    float* sp = scale + n % kTcScales * 4 * kTcTile + key;
                    const bool there = key < count;
                    sp[0] = there ? d0 : 0.0f;
                    sp[kTcTile] = there ? d1 : 0.0f;
                    if constexpr (K_MIN) {
                        sp[2 * kTcTile] = there ? m0 : 0.0f;
                        sp[3 * kTcTile] = there ? m1 : 0.0f;
                    }
                    fence_proxy_async_smem();
                    mbar_arrive(&B->k_full[sg]);
                    mbar_arrive(&B->raw_empty[b]);
                }
            }
        } else {
            // the group's tiles n, n + 2, ..: the copies of the next one run while this one is used
            Run rf = r;
            auto start = [&](int n) {
                const int e = lo + n, sg = n % kSt;
                if (e < hi) {
                    while (e >= rf.end) rf.next(a, pref, hi);
                    const int count = min(kTcTile, rf.L - (rf.t0 + e - rf.i) * kTcTile);
                    const uint8_t* src = tile_rows(a, rf, e) + rf.kvh * slice;
                    if (n >= kSt) ok = ok && tc_wait(&B->k_empty[sg], (n / kSt - 1) & 1, &B->err, 53);
                    uint8_t* dst = smem + Sh::kTiles + sg * kTcTileBytes;
                    const uint64_t al = reinterpret_cast<uint64_t>(src) | (uint64_t)a.k_nb1;
                    const int unit = (al & 15) == 0 ? 16 : (al & 3) == 0 ? 4 : 2, w = 128 / unit, per = 128 / w;
                    const int k0 = key / w, col = (key - k0 * w) * unit;
#pragma unroll 4
                    for (int kk = k0; ok && kk < kTcTile; kk += per) {
                        const bool there = kk < count;
                        const uint8_t* from = there ? src + (int64_t)kk * a.k_nb1 + col : src;
                        uint8_t* to = dst + kk * 128 + (col ^ ((kk & 7) << 4));
                        if (unit == 16) tree::cp_async16(to, from, there);
                        else if (unit == 4) tree::cp_async4(to, from, there);
                        else *reinterpret_cast<uint16_t*>(to) = there ? *reinterpret_cast<const uint16_t*>(from) : (uint16_t)0;
                    }
                }
                tree::cp_async_commit();
            };
            start(g);
            for (int n = g; lo + n < hi; n += 2) {
                tree::cp_async_wait<0>();
                if (ok) {
                    fence_proxy_async_smem();
                    mbar_arrive(&B->k_full[n % kSt]);
                }
                start(n + 2);  // (may have to wait for its stage)
            }
            tree::cp_async_wait<0>();
        }
    } else if (warp == 18) {
        // ------------------------------------------------------ loader
        if constexpr (K_Q) {
            if (lane == 0) {
                const int nbuf = ta.raw_buffers;
                int b = 0, n = 0;
                uint32_t turn = 0;
                bool ok = true;
                for (; ok && lo + n < hi; ++n) {
                    if (lo + n == r.end) r.next(a, pref, hi);
                    if (turn) ok = tc_wait(&B->raw_empty[b], (turn - 1) & 1, &B->err, 58);
                    if (!ok) break;
                    const uint8_t* src = tile_rows(a, r, lo + n);
                    uint32_t main = 0;
                    if (whole_rows(a, src, slice)) {
                        uint8_t* dst = raw_at<KT>(smem, b);
                        const int bytes = min(kTcTile, r.L - (r.t0 + lo + n - r.i) * kTcTile) * a.Hkv * slice;
                        main = (uint32_t)bytes & ~15u;
                        fence_proxy_async_smem();  // the reads of what was there come first
                        for (int x = (int)main; x < bytes; x += 2) *reinterpret_cast<uint16_t*>(dst + x) = *reinterpret_cast<const uint16_t*>(src + x);
                        mbar_arrive_expect_tx(&B->raw_full[b], main);
                        if (main) bulk_g2s(dst, src, main, &B->raw_full[b]);
                    } else {
                        mbar_arrive(&B->raw_full[b]);
                    }
                    if (++b == nbuf) {
                        b = 0;
                        ++turn;
                    }
                }
                // no copy outlives the CTA: every buffer's last one has landed (bounded, also after an error)
                for (int k = 1; k <= nbuf && k <= n; ++k) {
                    const int last = n - k;
                    for (int x = 0; x < 4096 && !mbar_try_wait_hint(&B->raw_full[last % nbuf], (last / nbuf) & 1, 1000u); ++x) {}
                }
            }
        }
    } else {
        // ------------------------------------------------------ MMA issuer of group g: the warp walks, one lane issues
        const int g = __shfl_sync(0xffffffffu, warp, 0) - 16;
        const uint64_t dq0 = tc::sdesc_sw128(smem_addr(smem + Sh::kQ), 16, 1024);
        const uint64_t dt0 = tc::sdesc_sw128(smem_addr(smem + Sh::kTiles), 16, 1024);
        const uint32_t sp0 = tmem + g * 256;
        uint32_t k = 0, n_run = 0;
        bool ok = true;
        for (; ok && r.i < hi; r.next(a, pref, hi), ++n_run) {
            const int R = max(r.n * a.G, 1);
            ok = tc_wait(&B->q_full, n_run & 1, &B->err, 55);
            ok = __all_sync(0xffffffffu, ok);
            if (lane == 0) mbar_arrive(&B->q_seen);
            for (int j = r.i + ((r.i ^ lo ^ g) & 1); ok && j < r.end; j += 2) {
                const int n = j - lo, sg = n % kSt;
                ok = tc_wait(&B->k_full[sg], (n / kSt) & 1, &B->err, 56);
                ok = __all_sync(0xffffffffu, ok);
                tc::fence_after();
                const uint64_t dk = dt0 + (uint64_t)(sg * (kTcTileBytes >> 4));
                for (int r0 = 0; ok && r0 < R; r0 += Sh::kSRows, ++k) {
                    if (k >= 2) ok = tc_wait(&B->s_empty[g][k & 1], ((k >> 1) - 1) & 1, &B->err, 57);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    tc::fence_after();
                    const uint32_t idesc = tc::idesc_f16_f32(128, (min(Sh::kSRows, R - r0) + 15) / 16 * 16, false);
                    const uint64_t dh = dq0 + (uint64_t)((r0 >> 7) * 2 * (kTcTileBytes >> 4) + (r0 & 127) * 8), dl = dh + (kTcTileBytes >> 4);
                    const uint32_t sp = sp0 + (k & 1) * 128;
                    if (elect_one()) {
                        if constexpr (K_Q) {
#pragma unroll
                            for (int b = 0; b < 2; ++b) {  // the low parts of Q first, while the sums are small
                                tc::mma_ss(sp + 64 * b, dk + 4 * b, dl + 4 * b, idesc, 0u);
                                tc::mma_ss(sp + 64 * b, dk + 4 * b + 2, dl + 4 * b + 2, idesc, 1u);
                                tc::mma_ss(sp + 64 * b, dk + 4 * b, dh + 4 * b, idesc, 1u);
                                tc::mma_ss(sp + 64 * b, dk + 4 * b + 2, dh + 4 * b + 2, idesc, 1u);
                            }
                        } else {
#pragma unroll
                            for (int kk = 0; kk < 4; ++kk) tc::mma_ss(sp, dk + 2 * kk, dl + 2 * kk, idesc, kk > 0 ? 1u : 0u);
#pragma unroll
                            for (int kk = 0; kk < 4; ++kk) tc::mma_ss(sp, dk + 2 * kk, dh + 2 * kk, idesc, 1u);
                        }
                        tc::mma_commit(&B->s_full[g][k & 1]);
                    }
                    __syncwarp();
                }
                if (ok && elect_one()) tc::mma_commit(&B->k_empty[sg]);
                __syncwarp();
            }
            ok = __all_sync(0xffffffffu, ok);
        }
    }
    tc::fence_before();
    __syncthreads();
    if (warp == 0) {
        tc::fence_after();
        tc::tmem_dealloc(tmem, 512);
    }
    if (tid == 0 && B->err) record_status(a.status, kStatusTimeout | (B->err << 8));
}

// Launch for K type KT (kv_scores_tc_inst.cu, one unit per K type).
template <int KT> cudaError_t launch_tc_for_k(cudaStream_t stream, const TcArgs& a);

}  // namespace kvscore
}  // namespace cvattn
