// tree_tc.cuh -- tree attention on the 5th-generation tensor cores (tcgen05), for
// f16 and block-quantized caches and more than 32 rows per KV head.
//
// Work is cut evenly: the key tiles (128 keys) of all units (sequence, KV head,
// tile of 128 rows) form one list, and CTA c of G takes the entries [c N / G,
// (c + 1) N / G).  A run is the part of one unit that a CTA has; a whole unit is
// written out directly, parts go to the workspace and tree_tc_combine_kernel joins
// them.  (Ragged sequences and few long ones fill the SMs alike.)
//   warps 0-3, 4-7  softmax groups: thread = row = TMEM lane; group g takes the
//                   CTA's tiles 2 k + g
//   warps 8-11      producer: raw rows by cp.async, then f16 tiles (128B swizzle);
//                   f16 caches are copied straight into the tiles
//   warp 12         issues S = Q K^T, up to two tiles ahead of the softmax
//   warp 13         issues O = P V            (14, 15 fill up their warpgroup)
// Precision: products of split numbers.  x = hi + lo in f16, S = Qh Kh + Ql Kh
// (+ Qh Kl), O = Ph Vh + Pl Vh (+ Ph Vl); the dropped low x low term is 2^-22 of the
// largest.  Q is scaled per row, K and V per tile, by powers of two so that hi and
// lo keep their bits; P is kept 2^7 large.  A scale d times integer quants splits in
// two half-precision instructions: hi = RN(d q), lo = d q - hi, exact.  An f16 cache
// is its own hi and has no lo.
// The output of a tile is a fresh accumulator, added in f32 to the row's registers:
// adds inside the tensor cores truncate, and over a long cache that would show.
// TMEM: three S buffers of 128 columns, tile n in n % 3, each overwritten 32 keys at
// a time by that chunk's P (16 columns hi, 16 lo): a group never waits for the
// S of its next tile.  Two outputs of 64 columns, one per group, read back while
// the group's next tile is on its way.
#pragma once

#include "flash_pipe.cuh"
#include "tree_mma.cuh"

namespace cvattn {
namespace tree {

constexpr int kTcTile = 128;
constexpr int kTcRows = 128;
constexpr int kTcThreads = 16 * 32;
// Registers of a thread by role: launched with 128; 256 * 168 + 128 * 96 + 128 * 80 <= 512 * 128.
constexpr int kTcRegsSoftmax = 168, kTcRegsProducer = 96, kTcRegsIssuer = 80;
static_assert(256 * kTcRegsSoftmax + 128 * kTcRegsProducer + 128 * kTcRegsIssuer <= 65536, "the block's registers");
constexpr int kTcMaxSeq = 1024;       // prefix table in shared memory
constexpr int kTcExps = 8;            // tiles whose scales may be in flight
constexpr int kTcTileBytes = kTcTile * kD * 2;
constexpr float kTcOffs = 7.0f;

struct TcArgs {
    Args a;
    uint32_t inv_g;                   // ceil(2^16 / G): r * inv_g >> 16 = r / G for r < 2^13 / G
    int grid;                         // CTAs that share the list
    float* ws_o;                      // [2 * grid][128][64]
    float* ws_ml;                     // [2 * grid][128][2]
    int32_t* ws_pref;                 // [n_seq + 1], written by CTA 0 for the combine
};

struct TcBars {
    uint64_t k_full[5], v_full[5], k_empty[5], v_empty[5];  // by stage
    uint64_t q_full;
    uint64_t s_full[3], p_full[3], s_free[3];               // by S buffer
    uint64_t o_full[2];                                     // by group
    uint32_t tmem_base;
    int err;
    uint32_t maxk[2], maxv[2];        // largest |scale| of a tile, by tile parity
    float2 exps[kTcExps];             // 2^-e of K and V of tile i at i % kTcExps
    uint32_t bad[kTcExps][4];         // draft keys whose V is not finite
    int32_t first_run[12];            // Run at the start of the CTA's part
};

template <int KT, int VT>
struct TcShape {
    static constexpr int NK = KT == kF16 ? 1 : 2, NV = VT == kF16 ? 1 : 2;  // pieces of an operand
    static constexpr int kStages = NK + NV == 2 ? 5 : NK + NV == 3 ? 3 : 2;
    static constexpr int kStage = (NK + NV) * kTcTileBytes;
    static constexpr int rawK = NK == 1 ? 0 : kTcTile * raw_stride(KT), rawV = NV == 1 ? 0 : kTcTile * raw_stride(VT);
    static constexpr int kQ = 0;                       // Q hi, Q lo; then the groups' halves at a run's end
    static constexpr int kTiles = 2 * kTcTileBytes;
    static constexpr int kRaw = kTiles + kStages * kStage;
    static constexpr int kMl = kRaw + 2 * (rawK + rawV);
    static constexpr int kBars = kMl + 2 * kTcRows * 8;
    static constexpr int kPref = kBars + (int)((sizeof(TcBars) + 15) / 16 * 16);
    static constexpr int kLen = kPref + (kTcMaxSeq + 4) * 4, kNodes = kLen + kTcMaxSeq * 4;
    static constexpr int kBytes = kNodes + kTcMaxSeq * 2;
    static_assert(kBytes <= 227 * 1024, "one CTA per SM");
};

template <int N> __device__ __forceinline__ void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r != 0;
}
// x - h, h an f16: what rounding x to h left over (exact)
__device__ __forceinline__ float less_f16(float x, uint16_t h) {
    float r;
    asm("fma.rn.f32.f16 %0, %1, %2, %3;" : "=f"(r) : "h"(h), "h"((uint16_t)0xBC00u), "f"(x));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// Bounded wait in little code (there are many): gives up after kWaitBudgetNs, or once another role has given up.
__device__ __forceinline__ bool tc_wait(uint64_t* bar, uint32_t parity, int* err, int* status, int site) {
    uint64_t t0 = 0;
#pragma unroll 1
    for (uint32_t i = 0; !mbar_try_wait_hint(bar, parity, 20000u); ++i) {
        if ((i & 63) != 63) continue;
        const uint64_t now = global_timer_ns();
        if (t0 == 0) t0 = now;
        const bool late = now - t0 > kWaitBudgetNs;
        if (late) {
            record_status(status, kStatusTimeout | (site << 8));
            *reinterpret_cast<volatile int*>(err) = 1;
        }
        if (late || *reinterpret_cast<volatile int*>(err)) return false;
    }
    return true;
}

__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    unsigned long long ra = *reinterpret_cast<unsigned long long*>(&a), rb = *reinterpret_cast<unsigned long long*>(&b), rd;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(rd) : "l"(ra), "l"(rb));
    return *reinterpret_cast<float2*>(&rd);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    unsigned long long ra = *reinterpret_cast<unsigned long long*>(&a), rb = *reinterpret_cast<unsigned long long*>(&b), rd;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(rd) : "l"(ra), "l"(rb));
    return *reinterpret_cast<float2*>(&rd);
}

// Units of sequence s: row tiles times KV heads, row tile major.
__device__ __forceinline__ int units_of(const Args& a, const Lens& x) { return (x.n * a.G + kTcRows - 1) / kTcRows * a.Hkv; }

// A CTA's walk through its part of the list, run by run.  Lengths come from shared memory (SeqTab), so that a new run
// costs no trip to global memory and no division.
struct SeqTab {
    const int32_t *pref, *len;
    const uint16_t* nodes;
};
struct Run {
    int s, kvh, rt;       // unit: sequence, KV head, tile of 128 rows
    int i, end;           // list entries [i, end) of this run
    int t0, T;            // its first tile, and the unit's tiles
    int L, n, cache_tiles, units_left;

    __device__ __forceinline__ void sequence(const Args& a, const SeqTab& tab, int seq) {
        s = seq;
        L = tab.len[seq];
        n = tab.nodes[seq];
        cache_tiles = (L + kTcTile - 1) / kTcTile;
        T = n == 0 ? 0 : cache_tiles + (a.kd ? (n + kTcTile - 1) / kTcTile : 0);
    }
    __device__ __forceinline__ void start(const Args& a, const SeqTab& tab, int entry, int hi) {
        i = end = entry;
        if (entry >= hi) return;
        int lo = 0, up = a.n_seq;  // last s with pref[s] <= entry: its list is not empty
        while (up - lo > 1) {
            const int mid = (lo + up) >> 1;
            if (tab.pref[mid] <= entry) lo = mid;
            else up = mid;
        }
        sequence(a, tab, lo);
        const int u = (entry - tab.pref[lo]) / T;
        t0 = entry - tab.pref[lo] - u * T;
        rt = u / a.Hkv;
        kvh = u - rt * a.Hkv;
        units_left = (tab.pref[lo + 1] - tab.pref[lo]) / T - u - 1;
        end = min(hi, i + T - t0);
    }
    __device__ __forceinline__ void next(const Args& a, const SeqTab& tab, int hi) {
        i = end;
        if (i >= hi) return;
        t0 = 0;
        if (units_left > 0) {
            --units_left;
            if (++kvh == a.Hkv) {
                kvh = 0;
                ++rt;
            }
        } else {
            int q = s + 1;
            while (tab.pref[q + 1] == i) ++q;  // sequences without entries
            sequence(a, tab, q);
            rt = kvh = 0;
            units_left = (n * a.G + kTcRows - 1) / kTcRows * a.Hkv - 1;
        }
        end = min(hi, i + T);
    }
    __device__ __forceinline__ void tile(int entry, bool& draft, int& p0, int& count) const {
        const int t = t0 + (entry - i);
        draft = t >= cache_tiles;
        p0 = (draft ? t - cache_tiles : t) * kTcTile;
        count = min(kTcTile, (draft ? n : L) - p0);
    }
};

__device__ __forceinline__ int tc_cut(int c, int n, int g) { return (int)((long long)c * n / g); }
__device__ __forceinline__ int tc_owner(int i, int n, int g) { return (int)(((long long)(i + 1) * g - 1) / n); }

// hi and lo of 32 values of one key into rows of two tiles; w holds exact integers (convert_group), d and m the block's
// scale and min times the tile's power of two.
template <int T>
__device__ __forceinline__ void split_block(uint8_t* hi_tile, uint8_t* lo_tile, int key, int blk, const uint32_t (&w)[16], float d, float m) {
    uint32_t h[16], l[16];
    if constexpr (!BlockTraits<T>::HAS_MIN) {
        const __half2 d2 = __float2half2_rn(d);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const __half2 q = *reinterpret_cast<const __half2*>(&w[i]);
            const __half2 p = __hmul2_rn(d2, q);
            const __half2 e = __hfma2(d2, q, __hneg2(p));
            h[i] = *reinterpret_cast<const uint32_t*>(&p);
            l[i] = *reinterpret_cast<const uint32_t*>(&e);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float2 q = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            split2(fmaf(q.x, d, m), fmaf(q.y, d, m), h[i], l[i]);
        }
    }
    store_block(hi_tile, key, blk, h);
    store_block(lo_tile, key, blk, l);
}

// Power of two that brings the largest scale (or min) of a tile to [2^6, 2^7): quants times it stay below 2^15.
__device__ __forceinline__ int tile_exp(float mx) {
    if (!(mx > 0.0f)) return 0;
    const int e = 6 - dstream::ilog2f(mx);
    return e > 100 ? 100 : (e < -100 ? -100 : e);
}

template <int KT, int VT>
__global__ void __launch_bounds__(kTcThreads, 1) tree_tc_kernel(const __grid_constant__ TcArgs ta) {
    using Sh = TcShape<KT, VT>;
    constexpr int NK = Sh::NK, NV = Sh::NV, kSt = Sh::kStages;
    constexpr int sliceK = 2 * group_bytes(KT), sliceV = 2 * group_bytes(VT);
    extern __shared__ __align__(1024) uint8_t smem[];
    const Args& a = ta.a;
    TcBars* B = reinterpret_cast<TcBars*>(smem + Sh::kBars);
    int32_t* pref = reinterpret_cast<int32_t*>(smem + Sh::kPref);
    const SeqTab tab{pref, reinterpret_cast<int32_t*>(smem + Sh::kLen), reinterpret_cast<uint16_t*>(smem + Sh::kNodes)};
    if (smem_addr(smem) & 1023u) {
        if (threadIdx.x == 0) record_status(a.status, kStatusTimeout);
        return;
    }
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (tid == 0) {
        for (int i = 0; i < kSt; ++i) {
            mbar_init(&B->k_full[i], 128);
            mbar_init(&B->v_full[i], 128);
            mbar_init(&B->k_empty[i], 1);
            mbar_init(&B->v_empty[i], 1);
        }
        mbar_init(&B->q_full, 256);
        for (int b = 0; b < 3; ++b) {
            mbar_init(&B->s_full[b], 1);
            mbar_init(&B->p_full[b], 128);
            mbar_init(&B->s_free[b], 1);
        }
        for (int g = 0; g < 2; ++g) {
            mbar_init(&B->o_full[g], 1);
            B->maxk[g] = B->maxv[g] = 0u;
        }
        B->err = 0;
        fence_mbar_init();
    }
    if (warp == 0) {
        tc::tmem_alloc(&B->tmem_base, 512);
        tc::tmem_relinquish();
    }
    if (warp == 1) {  // list entries before each sequence
        int carry = 0;
        for (int base = 0; base < a.n_seq; base += 32) {
            const int s = base + lane;
            int n = 0;
            if (s < a.n_seq) {
                const Lens x = lens_of(a, s, blockIdx.x == 0);
                n = x.tiles * units_of(a, x);
                reinterpret_cast<int32_t*>(smem + Sh::kLen)[s] = x.L;
                reinterpret_cast<uint16_t*>(smem + Sh::kNodes)[s] = (uint16_t)x.n;
            }
            int incl = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += y;
            }
            if (s < a.n_seq) {
                pref[s] = carry + incl - n;
                if (blockIdx.x == 0) ta.ws_pref[s] = carry + incl - n;
            }
            carry += __shfl_sync(0xffffffffu, incl, 31);
        }
        if (lane == 0) {
            pref[a.n_seq] = carry;
            if (blockIdx.x == 0) ta.ws_pref[a.n_seq] = carry;
        }
        __syncwarp();
        Run r;
        r.start(a, tab, tc_cut(blockIdx.x, carry, ta.grid), tc_cut(blockIdx.x + 1, carry, ta.grid));
        static_assert(sizeof(Run) <= sizeof(B->first_run), "a run in shared memory");
        if (lane == 0) *reinterpret_cast<Run*>(B->first_run) = r;
    }
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    griddep_launch_dependents();
    const uint32_t tmem = B->tmem_base;
    const int total = pref[a.n_seq];
    const int lo = tc_cut(blockIdx.x, total, ta.grid), hi = tc_cut(blockIdx.x + 1, total, ta.grid);
    Run r = *reinterpret_cast<const Run*>(B->first_run);

    if (warp < 8) {
        // ------------------------------------------------------ softmax group g
        regs_up<kTcRegsSoftmax>();
        const int g = warp >> 2, quad = warp & 3, row = quad * 32 + lane;
        const uint32_t lane_base = (uint32_t)(quad * 32) << 16;
        const uint32_t ot = tmem + lane_base + 384 + g * 64;
        uint8_t* qhi = smem + Sh::kQ;
        uint8_t* qlo = qhi + kTcTileBytes;
        float4* xch = reinterpret_cast<float4*>(smem + Sh::kQ) + row * 16;  // group 1's output row at a run's end
        float2* mls = reinterpret_cast<float2*>(smem + Sh::kMl) + row;
        uint32_t k = 0;  // tiles of this group so far
        bool ok = true;
        for (; r.i < hi; r.next(a, tab, hi)) {
            const int rr = r.rt * kTcRows + row, rows = r.n * a.G;
            const bool real = rr < rows;
            const bool warp_real = r.rt * kTcRows + quad * 32 < rows;  // some row of this warp is
            const int node = (int)(((uint32_t)rr * ta.inv_g) >> 16), h = r.kvh * a.G + rr - node * a.G;
            const int64_t orow = (int64_t)r.s * a.out_nb_seq + (int64_t)node * a.out_nb_node + h * kD;
            // Q: both groups look at the whole row, each writes its half of the dims
            float rs;
            {
                const float4* q = reinterpret_cast<const float4*>(a.q + (int64_t)r.s * a.q_nb_seq + (int64_t)node * a.q_nb_node + h * kD);
                float am = 0.0f;
                if (real) {
#pragma unroll 4
                    for (int c = 0; c < 16; ++c) {
                        const float4 v = q[c];
                        am = max3(am, fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w)));
                    }
                }
                const int ex = dtc::norm_exp(am);
                const float sc = a.scale_log2 < 0.0f ? -pow2f(ex) : pow2f(ex);
                rs = pow2f(-ex) * fabsf(a.scale_log2);
                // nothing reads the last run's Q, or its exchanged rows, any more
                if (r.i != lo) asm volatile("bar.sync 1, 256;" ::: "memory");
#pragma unroll 1
                for (int c = 4 * g; c < 4 * g + 4; ++c) {
                    const float4 u = real ? q[2 * c] : make_float4(0.f, 0.f, 0.f, 0.f), v = real ? q[2 * c + 1] : u;
                    uint4 wh, wl;
                    split2(u.x * sc, u.y * sc, wh.x, wl.x);
                    split2(u.z * sc, u.w * sc, wh.y, wl.y);
                    split2(v.x * sc, v.y * sc, wh.z, wl.z);
                    split2(v.z * sc, v.w * sc, wh.w, wl.w);
                    const uint32_t at = tc::sw128_offset(row, c);
                    *reinterpret_cast<uint4*>(qhi + at) = wh;
                    *reinterpret_cast<uint4*>(qlo + at) = wl;
                }
                fence_proxy_async_smem();
                mbar_arrive(&B->q_full);
            }
            float2 O[32];
#pragma unroll
            for (int d = 0; d < 32; ++d) O[d] = make_float2(0.f, 0.f);
            float base = 0.0f, thr = -INFINITY, l = 0.0f, vs_last = 0.0f;
            bool pending = false;  // a tile's output still to be added, times vs_last
            bool spoiled = false;  // the row sees a drafted value that is not finite
            auto add_output = [&]() {
                uint32_t o0[32], o1[32];
                tc::tmem_ld32(ot, o0);
                tc::tmem_ld32(ot + 32, o1);
                tc::tmem_ld_wait();
                const float2 f = make_float2(vs_last, vs_last);
#pragma unroll
                for (int d = 0; d < 16; ++d) {
                    O[d] = ffma2(make_float2(__uint_as_float(o0[2 * d]), __uint_as_float(o0[2 * d + 1])), f, O[d]);
                    O[16 + d] = ffma2(make_float2(__uint_as_float(o1[2 * d]), __uint_as_float(o1[2 * d + 1])), f, O[16 + d]);
                }
            };
            for (int j = r.i + ((r.i ^ g ^ lo) & 1); j < r.end; j += 2) {  // the CTA's tiles j - lo of parity g
                bool draft;
                int p0, count;
                r.tile(j, draft, p0, count);
                const int n = j - lo, buf = n % 3;
                const uint32_t sp = tmem + lane_base + buf * 128;
                ok = tc_wait(&B->s_full[buf], (n / 3) & 1, &B->err, a.status, 31);
                if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
                tc::fence_after();
                if (warp_real) {
                    uint32_t sv[32];
                    tc::tmem_ld32(sp, sv);
                    const float2 ex = B->exps[(j - lo) % kTcExps];
                    const float rst = fmaxf(rs * ex.x, 1e-37f);  // above 0, so that what is masked stays -infinity
                    const bool masked = draft || count < kTcTile;
                    tc::tmem_ld_wait();
#pragma unroll 1
                    for (int c = 0; c < 4; ++c) {
                        if (masked) {
                            const int left = count - 32 * c;
                            uint32_t bits = left >= 32 ? 0xffffffffu : left <= 0 ? 0u : (1u << left) - 1u;
                            if (draft && bits && real) {
                                const int j0 = p0 + 32 * c;
                                if (a.mask) bits &= a.mask[(int64_t)r.s * a.mask_nb_seq + (int64_t)node * a.mask_words + (j0 >> 5)];
                                else if (node < j0 + 31) bits &= node < j0 ? 0u : (2u << (node - j0)) - 1u;
                            }
#pragma unroll
                            for (int d = 0; d < 32; ++d)
                                if (!((bits >> d) & 1u)) sv[d] = 0xff800000u;
                        }
                        // the largest score of the row's 32 keys (rst > 0, so that of S)
                        float mx;
                        {
                            float m4[4];
#pragma unroll
                            for (int u = 0; u < 4; ++u) {
                                const uint32_t* w = sv + 8 * u;
                                m4[u] = max3(max3(fmaxf(__uint_as_float(w[0]), __uint_as_float(w[1])), __uint_as_float(w[2]), __uint_as_float(w[3])),
                                             max3(__uint_as_float(w[4]), __uint_as_float(w[5]), __uint_as_float(w[6])), __uint_as_float(w[7]));
                            }
                            mx = fmaf(max3(fmaxf(m4[0], m4[1]), m4[2], m4[3]), rst, -base);
                        }
                        if (__any_sync(0xffffffffu, mx > thr)) {
                            float f = 1.0f;
                            if (mx > thr) {
                                const float up = mx - kTcOffs;
                                f = thr == -INFINITY ? 0.0f : fast_exp2(-up);
                                base += up;
                                thr = kLazy + kTcOffs;
                                l *= f;
                                vs_last *= f;
                            }
                            const float2 f2 = make_float2(f, f);
#pragma unroll
                            for (int d = 0; d < 32; ++d) O[d] = mul2(O[d], f2);
                            if (c) tc::tmem_st_wait();
#pragma unroll 1
                            for (int e = 0; e < 2 * c; ++e) {  // this tile's P so far, 16 keys at a time
                                uint32_t ph[8], pl[8];
                                const uint32_t at = sp + 32 * (e >> 1) + 8 * (e & 1);
                                tc::tmem_ld8(at, ph);
                                tc::tmem_ld8(at + 16, pl);
                                tc::tmem_ld_wait();
#pragma unroll
                                for (int d = 0; d < 8; ++d) {
                                    const float2 u = __half22float2(*reinterpret_cast<const __half2*>(&ph[d]));
                                    const float2 w = __half22float2(*reinterpret_cast<const __half2*>(&pl[d]));
                                    split2((u.x + w.x) * f, (u.y + w.y) * f, ph[d], pl[d]);
                                }
                                tc::tmem_st8(at, ph);
                                tc::tmem_st8(at + 16, pl);
                            }
                        }
                        float2 x[16];
                        {
                            const float2 f = make_float2(rst, rst), b = make_float2(-base, -base);
#pragma unroll
                            for (int d = 0; d < 16; ++d)
                                x[d] = ffma2(make_float2(__uint_as_float(sv[2 * d]), __uint_as_float(sv[2 * d + 1])), f, b);
                        }
                        tc::tmem_ld32(sp + 32 * min(c + 1, 3), sv);  // under way during this chunk's arithmetic
                        float2 l0 = make_float2(0.f, 0.f), l1 = l0;
#pragma unroll
                        for (int d = 0; d < 16; d += 2) {
                            x[d].x = fast_exp2(x[d].x);
                            x[d].y = fast_exp2(x[d].y);
                            x[d + 1].x = fast_exp2(x[d + 1].x);
                            x[d + 1].y = fast_exp2(x[d + 1].y);
                            l0 = add2(l0, x[d]);
                            l1 = add2(l1, x[d + 1]);
                        }
                        l0 = add2(l0, l1);
                        l += l0.x + l0.y;
                        if (draft) {
                            // keys whose V is not finite have zeros in the tile; a row that sees one is NaN in the end
                            const uint32_t bad = B->bad[(j - lo) % kTcExps][c];
                            if (bad) {
#pragma unroll
                                for (int d = 0; d < 16; ++d)
                                    spoiled |= ((bad >> (2 * d) & 1u) && x[d].x != 0.0f) || ((bad >> (2 * d + 1) & 1u) && x[d].y != 0.0f);
                            }
                        }
                        uint32_t pv[32];
#pragma unroll
                        for (int d = 0; d < 16; ++d) {
                            pv[d] = tc::pack_f16x2(x[d].x, x[d].y);
                            pv[16 + d] = tc::pack_f16x2(less_f16(x[d].x, (uint16_t)pv[d]), less_f16(x[d].y, (uint16_t)(pv[d] >> 16)));
                        }
                        tc::tmem_st32(sp + 32 * c, pv);
                        tc::tmem_ld_wait();
                    }
                    if (pending) {  // the output of the group's tile before this one (o_full counts every tile of the group)
                        ok = tc_wait(&B->o_full[g], (k - 1) & 1, &B->err, a.status, 32);
                        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
                        tc::fence_after();
                        add_output();
                    }
                    vs_last = ex.y;
                    pending = true;
                    tc::tmem_st_wait();
                }
                ++k;
                tc::fence_before();
                mbar_arrive(&B->p_full[buf]);
            }
            if (ok && pending) {
                ok = tc_wait(&B->o_full[g], (k - 1) & 1, &B->err, a.status, 32);
                ok = __all_sync(0xffffffffu, ok);
                tc::fence_after();
                if (ok) add_output();
            }
            tc::fence_before();
            if (!fp::prod_bar_and(2, 256, ok)) break;  // every MMA of the run is done; all threads leave together
            const float m_mine = thr == -INFINITY && l == 0.0f ? -INFINITY : base;  // (NaN scores raise nothing)
            if (g == 1) {
#pragma unroll
                for (int c = 0; c < 16; ++c) xch[c ^ (row & 7)] = make_float4(O[2 * c].x, O[2 * c].y, O[2 * c + 1].x, O[2 * c + 1].y);
                mls[0] = make_float2(m_mine, l);
                mls[kTcRows] = make_float2(spoiled ? 1.0f : 0.0f, 0.0f);
            }
            asm volatile("bar.sync 3, 256;" ::: "memory");
            if (g == 0 && real) {
                const float2 other = *mls;
                const float M = fmaxf(m_mine, other.x);
                const float f0 = m_mine == -INFINITY ? 0.0f : exp2f(m_mine - M), f1 = other.x == -INFINITY ? 0.0f : exp2f(other.x - M);
                const float sum = (m_mine == -INFINITY ? 0.0f : f0 * l) + (other.x == -INFINITY ? 0.0f : f1 * other.y);
                const bool whole = r.end - r.i == r.T, seen = M != -INFINITY;
                spoiled |= mls[kTcRows].x != 0.0f;
                const float inv = spoiled ? __int_as_float(0x7fc00000) : !whole ? 1.0f : seen ? 1.0f / sum : 0.0f;
                const int64_t slot = (int64_t)(2 * blockIdx.x + (r.i == lo ? 0 : 1)) * kTcRows + row;
                float4* dst = reinterpret_cast<float4*>(whole ? a.out + orow : ta.ws_o + slot * kD);
                const float2 g0 = make_float2(f0 * inv, f0 * inv), g1 = make_float2(f1 * inv, f1 * inv);
#pragma unroll
                for (int c = 0; c < 16; ++c) {
                    const float4 w = xch[c ^ (row & 7)];
                    const float2 u = ffma2(g1, make_float2(w.x, w.y), mul2(g0, O[2 * c])), v = ffma2(g1, make_float2(w.z, w.w), mul2(g0, O[2 * c + 1]));
                    dst[c] = make_float4(u.x, u.y, v.x, v.y);
                }
                if (!whole) *reinterpret_cast<float2*>(ta.ws_ml + slot * 2) = make_float2(M, sum);
                else if (a.lse)
                    a.lse[((int64_t)r.s * a.max_nodes + node) * a.Hq + h] = seen ? (M + log2f(sum)) * 0.69314718055994531f : -INFINITY;
            }
        }
    } else if (warp < 12) {
        // ------------------------------------------------------ producer: thread = key
        regs_down<kTcRegsProducer>();
        const int key = tid - 256;
        // keys [0, count) of a tile into shared memory, zeros up to 128
        auto copy = [&](auto type_tag, bool raw, uint8_t* dst, const uint8_t* src, int64_t nb1, int count) {
            constexpr int T = decltype(type_tag)::value;
            const uint64_t al = reinterpret_cast<uint64_t>(src) | (uint64_t)nb1;
            if (T == kF16 && (al & 15) == 0) {
                // 8 chunks of 16 bytes per key: this thread's chunk of every 16th key, whose swizzle is the same
                const int k0 = key >> 3, col = (key & 7) << 4;
                const uint8_t* from = src + (int64_t)k0 * nb1 + col;
                uint8_t* to = dst + k0 * 128 + (col ^ ((k0 & 7) << 4));
                const int64_t step = 16 * nb1;
                if (count == kTcTile) {
#pragma unroll
                    for (int u = 0; u < 8; ++u) cp_async16(to + u * 2048, from + u * step, true);
                } else {
#pragma unroll 1
                    for (int u = 0; u < 8; ++u) cp_async16(to + u * 2048, k0 + 16 * u < count ? from + u * step : src, k0 + 16 * u < count);
                }
                return;
            }
            const int unit = (al & 3) == 0 ? 4 : 2;
            const int w = 2 * group_bytes(T) / unit, per = unit == 4 ? 128 / (group_bytes(T) / 2) : 128 / group_bytes(T);
            const int k0 = unit == 4 ? key / (group_bytes(T) / 2) : key / group_bytes(T), col = (key - k0 * w) * unit;
            if (k0 >= per) return;
            const uint8_t* from = src + (int64_t)k0 * nb1 + col;
            const int64_t step = (int64_t)per * nb1;
            if (raw && unit == 4) {
                uint8_t* to = dst + k0 * raw_stride(T) + col;
                const int tstep = per * raw_stride(T);
                int kk = k0;
#pragma unroll 4
                for (; kk < count; kk += per, from += step, to += tstep) cp_async4(to, from, true);
#pragma unroll 1
                for (; kk < kTcTile; kk += per, to += tstep) *reinterpret_cast<uint32_t*>(to) = 0u;
                return;
            }
#pragma unroll 1
            for (int kk = k0; kk < kTcTile; kk += per, from += step) {
                const bool there = kk < count;
                uint8_t* to = raw ? dst + kk * raw_stride(T) + col : dst + kk * 128 + (col ^ ((kk & 7) << 4));
                if (unit == 4) cp_async4(to, there ? from : src, there);
                else *reinterpret_cast<uint16_t*>(to) = there ? *reinterpret_cast<const uint16_t*>(from) : (uint16_t)0;
            }
        };
        // the runs of the tile whose copies start and of the tile that is finished
        Run ri = r, rc = r;
        int ii = lo;
        bool ok = true;
        auto issue = [&](int n) {        // copies of the CTA's tile n (list entry ii)
            if (ii < hi) {
                if (ii == ri.end) ri.next(a, tab, hi);
                bool draft;
                int p0, count;
                ri.tile(ii, draft, p0, count);
                const uint8_t* ks = (draft ? a.kd + (int64_t)ri.s * a.kd_nb2 : seq_base(a.k_seq_ptrs, a.k, a.k_nb2, ri.s)) + ri.kvh * sliceK;
                const uint8_t* vs = (draft ? a.vd + (int64_t)ri.s * a.vd_nb2 : seq_base(a.v_seq_ptrs, a.v, a.v_nb2, ri.s)) + ri.kvh * sliceV;
                const int64_t nk = draft ? a.kd_nb1 : a.k_nb1, nv = draft ? a.vd_nb1 : a.v_nb1;
                const int st = n % kSt;
                uint8_t* tiles = smem + Sh::kTiles + st * Sh::kStage;
                uint8_t* raw = smem + Sh::kRaw + (n & 1) * (Sh::rawK + Sh::rawV);
                const uint32_t use = n / kSt;
                if constexpr (NK == 1)
                    if (use > 0) ok = ok && tc_wait(&B->k_empty[st], (use - 1) & 1, &B->err, a.status, 33);
                if (ok) copy(std::integral_constant<int, KT>{}, NK == 2, NK == 2 ? raw : tiles, ks + (int64_t)p0 * nk, nk, count);
                if constexpr (NV == 1)
                    if (use > 0) ok = ok && tc_wait(&B->v_empty[st], (use - 1) & 1, &B->err, a.status, 34);
                if (ok) copy(std::integral_constant<int, VT>{}, NV == 2, NV == 2 ? raw + Sh::rawK : tiles + NK * kTcTileBytes, vs + (int64_t)p0 * nv, nv, count);
                ++ii;
            }
            cp_async_commit();
        };
        constexpr int kAhead = NK + NV == 2 ? kSt - 2 : 1;  // tiles whose copies run ahead of the finished one
#pragma unroll 1
        for (int n = -kAhead; lo + n < hi; ++n) {
            if (n >= 0) {
                cp_async_wait<kAhead - 1>();
                // every thread's copies of the tile have landed, and every thread is done with the tile before (or all leave)
                if (!fp::prod_bar_and(4, 128, ok)) break;
            }
            // raw copies of the next tile first; copies into a stage may have to wait for it, so they come last
            if constexpr (NK + NV == 4) issue(n + kAhead);
            if (n >= 0) {
            if (lo + n == rc.end) rc.next(a, tab, hi);
            bool draft;
            int p0, count;
            rc.tile(lo + n, draft, p0, count);
            const int st = n % kSt;
            const uint32_t use = n / kSt;
            uint8_t* tiles = smem + Sh::kTiles + st * Sh::kStage;
            const uint8_t* rawk = smem + Sh::kRaw + (n & 1) * (Sh::rawK + Sh::rawV);
            const uint8_t* rawv = rawk + Sh::rawK;
            bool bad = false;
            float fk = 1.0f, fv = 1.0f;
            if constexpr (NK + NV > 2) {
                // the tile's largest scales
                uint32_t mk = 0, mv = 0;
                auto scale_max = [&](auto type_tag, const uint8_t* rowp, bool& special) {
                    constexpr int T = decltype(type_tag)::value;
                    uint32_t m = 0;
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        const uint8_t* gb = rowp + b * group_bytes(T);
                        float d = fabsf(h2f(*reinterpret_cast<const uint16_t*>(gb)));
                        if constexpr (BlockTraits<T>::HAS_MIN) {
                            // |d q + m| <= 16 d + |m + 16 d|: in units of 127 quants of a scale
                            const float mm = h2f(*reinterpret_cast<const uint16_t*>(gb + BlockTraits<T>::OFF_M));
                            special |= !isfinite(mm);
                            d = (32.0f * d + fabsf(mm)) * (1.0f / 64.0f);
                        }
                        special |= !isfinite(d);
                        if (isfinite(d)) m = max(m, __float_as_uint(d));
                    }
                    return __reduce_max_sync(0xffffffffu, m);
                };
                bool kbad = false;
                if constexpr (NK == 2) mk = scale_max(std::integral_constant<int, KT>{}, rawk + key * raw_stride(KT), kbad);
                if constexpr (NV == 2) mv = scale_max(std::integral_constant<int, VT>{}, rawv + key * raw_stride(VT), bad);
                if (lane == 0) {
                    if (mk) atomicMax(&B->maxk[n & 1], mk);
                    if (mv) atomicMax(&B->maxv[n & 1], mv);
                }
                asm volatile("bar.sync 5, 128;" ::: "memory");
                const int ek = tile_exp(__uint_as_float(B->maxk[n & 1])), ev = tile_exp(__uint_as_float(B->maxv[n & 1]));
                fk = pow2f(ek);
                fv = pow2f(ev);
                if (key == 0) {
                    B->exps[n % kTcExps] = make_float2(NK == 2 ? pow2f(-ek) : 1.0f, NV == 2 ? pow2f(-ev) : 1.0f);
                    B->maxk[(n + 1) & 1] = B->maxv[(n + 1) & 1] = 0u;
                }
            } else if (key == 0) {
                B->exps[n % kTcExps] = make_float2(1.0f, 1.0f);
            }
            if constexpr (NV == 1) {
                if (draft) {  // this thread's key
                    uint4* p = reinterpret_cast<uint4*>(tiles + NK * kTcTileBytes + key * 128);
                    for (int c = 0; c < 8; ++c) {
                        const uint4 w = p[c];
                        bad |= f16x2_special(w.x) || f16x2_special(w.y) || f16x2_special(w.z) || f16x2_special(w.w);
                    }
                    if (bad)
                        for (int c = 0; c < 8; ++c) p[c] = make_uint4(0u, 0u, 0u, 0u);
                }
            }
            if (draft) {  // (the softmax reads it with S)
                const uint32_t vote = __ballot_sync(0xffffffffu, bad);
                if (lane == 0) B->bad[n % kTcExps][key >> 5] = vote;
            }
            if constexpr (NK == 2) {
                if (use > 0) ok = ok && tc_wait(&B->k_empty[st], (use - 1) & 1, &B->err, a.status, 35);
                if (ok) {
                    uint32_t w0[16], w1[16];
                    float d0, m0, d1, m1;
                    convert_block<KT, 0>(rawk + key * raw_stride(KT), w0, d0, m0);
                    convert_block<KT, 1>(rawk + key * raw_stride(KT), w1, d1, m1);
                    split_block<KT>(tiles, tiles + kTcTileBytes, key, 0, w0, d0 * fk, m0 * fk);
                    split_block<KT>(tiles, tiles + kTcTileBytes, key, 1, w1, d1 * fk, m1 * fk);
                }
            }
            if (ok) {
                fence_proxy_async_smem();
                mbar_arrive(&B->k_full[st]);
            }
            if constexpr (NV == 2) {
                if (use > 0) ok = ok && tc_wait(&B->v_empty[st], (use - 1) & 1, &B->err, a.status, 36);
                if (ok) {
                    const bool drop = draft && bad;
                    uint32_t w0[16], w1[16];
                    float d0, m0, d1, m1;
                    convert_block<VT, 0>(rawv + key * raw_stride(VT), w0, d0, m0);
                    convert_block<VT, 1>(rawv + key * raw_stride(VT), w1, d1, m1);
                    uint8_t* vt = tiles + NK * kTcTileBytes;
                    split_block<VT>(vt, vt + kTcTileBytes, key, 0, w0, drop ? 0.0f : d0 * fv, drop ? 0.0f : m0 * fv);
                    split_block<VT>(vt, vt + kTcTileBytes, key, 1, w1, drop ? 0.0f : d1 * fv, drop ? 0.0f : m1 * fv);
                }
            }
            if (ok) {
                fence_proxy_async_smem();
                mbar_arrive(&B->v_full[st]);
            }
            }
            if constexpr (NK + NV < 4) issue(n + kAhead);
        }
        cp_async_wait<0>();
    } else {
        regs_down<kTcRegsIssuer>();
        // ------------------------------------------------------ MMA issuers: the whole warp walks, one lane issues
        const int which = __shfl_sync(0xffffffffu, warp, 0);
        const uint64_t dt0 = tc::sdesc_sw128(smem_addr(smem + Sh::kTiles), 16, 1024);
        bool ok = true;
        if (which == 12) {
            const uint32_t idesc = tc::idesc_f16_f32(128, kTcTile, false);
            const uint64_t dqh = tc::sdesc_sw128(smem_addr(smem + Sh::kQ), 16, 1024);
            const uint64_t dql = tc::sdesc_sw128(smem_addr(smem + Sh::kQ) + kTcTileBytes, 16, 1024);
            uint32_t n_run = 0;
            int n = 0, st = 0, buf = 0;
            uint32_t use = 0, turn = 0;  // n / kSt, n / 3
            for (; ok && r.i < hi; r.next(a, tab, hi), ++n_run) {
                ok = tc_wait(&B->q_full, n_run & 1, &B->err, a.status, 37);
                for (int j = r.i; ok && j < r.end; ++j, ++n) {
                    ok = tc_wait(&B->k_full[st], use & 1, &B->err, a.status, 38);
                    if (ok && n >= 3) ok = tc_wait(&B->s_free[buf], (turn - 1) & 1, &B->err, a.status, 40);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    tc::fence_after();
                    const uint64_t dk = dt0 + (uint64_t)(st * (Sh::kStage >> 4));
                    const uint32_t sp = tmem + buf * 128;
                    if (elect_one()) {
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk) {  // small terms first, while the sums are small
                            tc::mma_ss(sp, dql + kk * 2, dk + kk * 2, idesc, kk > 0 ? 1u : 0u);
                            if constexpr (NK == 2) tc::mma_ss(sp, dqh + kk * 2, dk + (kTcTileBytes >> 4) + kk * 2, idesc, 1u);
                        }
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk) tc::mma_ss(sp, dqh + kk * 2, dk + kk * 2, idesc, 1u);
                        tc::mma_commit(&B->s_full[buf]);
                        tc::mma_commit(&B->k_empty[st]);
                    }
                    __syncwarp();
                    if (++st == kSt) { st = 0; ++use; }
                    if (++buf == 3) { buf = 0; ++turn; }
                }
                ok = __all_sync(0xffffffffu, ok);
            }
        } else if (which == 13) {
            const uint32_t idesc = tc::idesc_f16_f32(128, 64, true);
            int st = 0, buf = 0;
            uint32_t use = 0, turn = 0;
            for (int n = 0; ok && lo + n < hi; ++n) {
                ok = tc_wait(&B->v_full[st], use & 1, &B->err, a.status, 41);
                if (ok) ok = tc_wait(&B->p_full[buf], turn & 1, &B->err, a.status, 39);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tc::fence_after();
                const uint64_t dv = dt0 + (uint64_t)(st * (Sh::kStage >> 4) + NK * (kTcTileBytes >> 4));
                const uint32_t sp = tmem + buf * 128, ot = tmem + 384 + (n & 1) * 64;
                if (elect_one()) {
#pragma unroll
                    for (int kk = 0; kk < 8; ++kk) {
                        const uint32_t ph = sp + 32 * (kk >> 1) + 8 * (kk & 1);
                        tc::mma_ts(ot, ph + 16, dv + kk * 128, idesc, kk > 0 ? 1u : 0u);
                        if constexpr (NV == 2) tc::mma_ts(ot, ph, dv + (kTcTileBytes >> 4) + kk * 128, idesc, 1u);
                    }
#pragma unroll
                    for (int kk = 0; kk < 8; ++kk) tc::mma_ts(ot, sp + 32 * (kk >> 1) + 8 * (kk & 1), dv + kk * 128, idesc, 1u);
                    tc::mma_commit(&B->o_full[n & 1]);
                    tc::mma_commit(&B->v_empty[st]);
                    tc::mma_commit(&B->s_free[buf]);
                }
                __syncwarp();
                if (++st == kSt) { st = 0; ++use; }
                if (++buf == 3) { buf = 0; ++turn; }
            }
        }
    }

    tc::fence_before();
    __syncthreads();
    if (warp == 0) {
        tc::fence_after();
        tc::tmem_dealloc(tmem, 512);
    }
}

// Join of the parts of units that several CTAs shared, and the rows that no unit
// holds (a sequence without keys, rows past the last node).  16 threads per row
// (4 dims each) follow every kLanes-th part.
template <int kLanes>
__global__ void __launch_bounds__(256) tree_tc_combine_kernel(const __grid_constant__ TcArgs ta) {
    constexpr int kPer = 16 / kLanes;
    __shared__ float4 so[16][16];
    __shared__ float2 sml[16];
    const Args& a = ta.a;
    griddep_wait();
    const int unit = threadIdx.x >> 4, c = threadIdx.x & 15, lane = unit % kLanes;
    const int all_rows = a.max_nodes * a.G;
    const int r = blockIdx.x * kPer + unit / kLanes, kvh = blockIdx.y, s = blockIdx.z;
    const Lens x = lens_of(a, s, false);
    const int node = r / a.G, h = kvh * a.G + r % a.G, rt = r / kTcRows;
    const int n = ta.ws_pref[a.n_seq];
    int b0 = 0, c0 = 0, c1 = -1;
    if (r < x.n * a.G && x.tiles > 0) {
        b0 = ta.ws_pref[s] + (rt * a.Hkv + kvh) * x.tiles;
        c0 = tc_owner(b0, n, ta.grid);
        c1 = tc_owner(b0 + x.tiles - 1, n, ta.grid);
        if (kLanes == 1 && c0 == c1) return;  // written whole
    }
    const bool done = c0 == c1;
    float M = -INFINITY, l = 0.0f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k0 = c0 + lane; k0 <= c1 && !done; k0 += 4 * kLanes) {
        float2 ml[4];
        float4 v[4];
        float top = M;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int cta = k0 + u * kLanes;
            ml[u] = make_float2(-INFINITY, 0.0f);
            if (cta <= c1) {
                const int64_t slot = 2 * cta + (tc_cut(cta, n, ta.grid) >= b0 ? 0 : 1);
                const int64_t at = slot * kTcRows + r % kTcRows;
                if (tc_cut(cta + 1, n, ta.grid) > tc_cut(cta, n, ta.grid)) {
                    ml[u] = *reinterpret_cast<const float2*>(ta.ws_ml + at * 2);
                    v[u] = *reinterpret_cast<const float4*>(ta.ws_o + at * kD + c * 4);
                }
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
        if (lane || done) return;
        M = -INFINITY;
#pragma unroll
        for (int k = 0; k < kLanes; ++k) M = fmaxf(M, sml[unit + k].x);
        l = 0.0f;
        o = make_float4(0.f, 0.f, 0.f, 0.f);
        if (M != -INFINITY) {
#pragma unroll
            for (int k = 0; k < kLanes; ++k) {
                if (sml[unit + k].x == -INFINITY) continue;
                const float f = exp2f(sml[unit + k].x - M);
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

// Launch for K type KT (tree_tc_inst.cu, one unit per K type).
template <int KT> cudaError_t launch_tc_for_k(cudaStream_t stream, const TcArgs& a);

}  // namespace tree
}  // namespace cvattn
