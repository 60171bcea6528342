// tree_tc.cuh -- tree attention on the 5th-generation tensor cores (tcgen05), for
// f16 and block-quantized caches and much work (kTcMinWork, tree_decode.cu).
//
// Work is cut evenly: the key tiles (128 keys) of all units (sequence, KV head,
// tile of 128 rows) form one list, and CTA c of G takes the entries [c N / G,
// (c + 1) N / G).  A run is the part of one unit that a CTA has; a whole unit is
// written out directly, parts go to the workspace and tree_tc_combine_kernel joins
// them.  (Ragged sequences and few long ones fill the SMs alike.)
//   warps 0-3, 4-7  softmax groups: thread = row = TMEM lane; group g takes the
//                   CTA's tiles 2 k + g
//   warps 8-11      producer of the K tiles, 12-15 of the V tiles: cp.async of the raw rows
//                   two tiles ahead, then thread = key: f16 tiles (128B swizzle) from
//                   them; f16 caches are copied straight into the tiles
//   warp 16         issues S = Q K^T, up to two tiles ahead of the softmax
//   warp 17         issues O = P V
//   (warps 18, 19 only complete the last warpgroup)
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
// Drafts that a row does not see may be of any size, and a tile has one power of two: a tile
// of quantized drafts whose largest scales would cost the others bits (kLeastExp) is marked
// by its producers, gets no weight in the products and is added row by row in f32.
// What bounds it: the softmax's instructions.  A tile of 128 rows x 128 keys costs the two
// groups together some 2100 cycles (exponentials alone 1024, products 770).  16 sequences of
// 4096 positions, 64 nodes, 14 / 2 heads, f16: 60.5 us, 252 TFLOP/s (twice that in the tensor
// cores, for hi and lo); 29 tiles a CTA and the start are four fifths of its active cycles.
// Few tiles per CTA are bound by the start (10K cycles: launch, lists, first rows, a cold
// instruction cache) and, for quants, by the producers (a tile's copies and conversion 2700
// cycles): 64 sequences of 128 to 2048, 8 nodes, Q8_0 / Q4_0: 39.4 us (nine tiles and the
// start are 34K of 53K active cycles; the rest is not accounted for); one of 65536, 16 nodes,
// Q8_0: 31.7 us, 565 GB/s.  All with the join's launch, calls in a graph.
#pragma once

#include "flash_pipe.cuh"
#include "tree_mma.cuh"

namespace cvattn {
namespace tree {

constexpr int kTcTile = 128;
constexpr int kTcRows = 128;
constexpr int kTcThreads = 20 * 32;
// Registers of a thread by role: launched with 96; 256 * 160 + 256 * 64 + 128 * 32 <= 640 * 96.
constexpr int kTcRegsSoftmax = 160, kTcRegsProducer = 64, kTcRegsOther = 32;
static_assert(256 * kTcRegsSoftmax + 256 * kTcRegsProducer + 128 * kTcRegsOther <= 640 * 96, "the block's registers");
constexpr int kTcMaxSeq = 1024;       // prefix table in shared memory
constexpr int kTcExps = 8;            // tiles whose scales may be in flight
constexpr int kTcTileBytes = kTcTile * kD * 2;
constexpr float kTcOffs = 7.0f;

struct TcArgs {
    Args a;
    uint32_t inv_g;                   // ceil(2^16 / G): r * inv_g >> 16 = r / G while r (G inv_g - 2^16) < 2^16: G <= 8, so r < 13107
    int grid;                         // CTAs that share the list
    float* ws_o;                      // [2 * grid][128][64]
    float* ws_ml;                     // [2 * grid][128][2]
    int32_t* ws_pref;                 // [n_seq + 1], written by CTA 0 for the combine
};

struct TcBars {
    uint64_t k_full[5], v_full[5], k_empty[5], v_empty[5];  // by stage
    uint64_t rawk_full[3], rawv_full[3];                    // by tile n % 3
    uint64_t q_full;
    uint64_t s_full[3], p_full[3], s_free[3];               // by S buffer
    uint64_t o_full[2];                                     // by group
    uint32_t tmem_base;
    int err;
    uint32_t maxk[3], maxv[3];        // largest |scale| of tile n at n % 3
    float expk[kTcExps], expv[kTcExps];  // 2^-e of K and V of tile n at n % kTcExps
    uint32_t starts[kTcExps];         // whether the tile starts a run
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
    static constexpr int kMl = kRaw + 3 * (rawK + rawV);
    static constexpr int kRs = kMl + 2 * kTcRows * 8;  // score factors of the rows
    static constexpr int kBars = kRs + kTcRows * 4;
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
// Bounded wait in little code (it stands at every step of every role): gives up after kTcTries suspensions of up to 20 us, or
// once another role has given up.  *err keeps the site; the kernel's end records it.
constexpr uint32_t kTcTries = 100000;
__device__ __forceinline__ bool tc_wait(uint64_t* bar, uint32_t parity, int* err, int site) {
#pragma unroll 1
    for (uint32_t i = 0; !mbar_try_wait_hint(bar, parity, 20000u); ++i) {
        if (i >= kTcTries) *reinterpret_cast<volatile int*>(err) = site;
        if (*reinterpret_cast<volatile int*>(err)) return false;
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

// hi and lo of a key's 64 values into its rows of two tiles, times the tile's power of two f; `keep` false: zeros.  Eight
// values at a time in a loop that is not unrolled: five roles run different code on an SM, and what they loop over has to
// stay in its instruction cache together (64 sequences of up to 2048 positions, Q8_0 and Q4_0, 56 rows: 52.9 us unrolled, 43.3 so).
template <int T>
__device__ __forceinline__ void split_row(uint8_t* hi_tile, uint8_t* lo_tile, int key, const uint8_t* row, float f, bool keep) {
    using BT = BlockTraits<T>;
    constexpr bool kFive = BT::OFF_QH >= 0;
    constexpr uint32_t bias = T == kQ8_0 ? dtc::kF16x2_1152 : kFive ? dtc::kF16x2_1040 : dtc::kF16x2_1032;
    uint8_t* to = hi_tile + key * 128;
    const int apart = (int)(lo_tile - hi_tile);
    const uint32_t swz = (key & 7) << 4;
#pragma unroll 1
    for (int b = 0; b < 2; ++b) {
        const uint8_t* g = row + b * group_bytes(T);
        float d = h2f(*reinterpret_cast<const uint16_t*>(g)), m = 0.0f;
        if constexpr (BT::HAS_MIN) m = fmaf(kFive ? 16.0f : 8.0f, d, h2f(*reinterpret_cast<const uint16_t*>(g + BT::OFF_M)));
        d = keep ? d * f : 0.0f;
        m = keep ? m * f : 0.0f;
        const __half2 d2 = __float2half2_rn(d);
        uint32_t qh = 0;
        if constexpr (kFive) qh = *reinterpret_cast<const uint16_t*>(g + BT::OFF_QH) | (uint32_t)*reinterpret_cast<const uint16_t*>(g + BT::OFF_QH + 2) << 16;
        const uint32_t off = b * group_bytes(T) + BT::OFF_QS;  // rows start at multiples of 4
        const uint32_t* words = reinterpret_cast<const uint32_t*>(row + (off & ~3u));
        const uint32_t turn = (off & 2) * 8;
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
            // bytes of the quants of values 8 c .. 8 c + 7
            const uint32_t* w = words + 2 * (T == kQ8_0 ? c : c & 1);
            const uint32_t mid = w[1];
            uint32_t x[2] = {__funnelshift_r(w[0], mid, turn), __funnelshift_r(mid, w[2], turn)}, h[4], l[4];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                if constexpr (T == kQ8_0) {
                    x[u] ^= 0x80808080u;
                } else {
                    x[u] = x[u] >> (4 * (c >> 1)) & 0x0f0f0f0fu;
                    if constexpr (kFive) x[u] |= (((qh >> (8 * c + 4 * u) & 15u) * 0x00204081u) & 0x01010101u) << 4;
                }
#pragma unroll
                for (int v = 0; v < 2; ++v) {  // exact integers in f16
                    const uint32_t n = dtc::hsub2_u32(__byte_perm(x[u], 0x64646464u, v ? 0x4342u : 0x4140u), bias);
                    const __half2 q = *reinterpret_cast<const __half2*>(&n);
                    if constexpr (BT::HAS_MIN) {
                        const float2 y = __half22float2(q);
                        split2(fmaf(y.x, d, m), fmaf(y.y, d, m), h[2 * u + v], l[2 * u + v]);
                    } else {
                        const __half2 p = __hmul2_rn(d2, q), e = __hfma2(d2, q, __hneg2(p));
                        h[2 * u + v] = *reinterpret_cast<const uint32_t*>(&p);
                        l[2 * u + v] = *reinterpret_cast<const uint32_t*>(&e);
                    }
                }
            }
            uint8_t* at = to + ((uint32_t)(64 * b + 16 * c) ^ swz);
            *reinterpret_cast<uint4*>(at) = make_uint4(h[0], h[1], h[2], h[3]);
            *reinterpret_cast<uint4*>(at + apart) = make_uint4(l[0], l[1], l[2], l[3]);
        }
    }
}

// Power of two that brings the largest scale (or min) of a tile to [2^6, 2^7): quants times it stay below 2^15.
__device__ __forceinline__ int tile_exp(float mx) {
    if (!(mx > 0.0f)) return 0;
    const int e = 6 - dstream::ilog2f(mx);
    return e > 100 ? 100 : (e < -100 ? -100 : e);
}

// Rows of list entry e (every head), of K or V.
struct TileRows {
    const uint8_t* at;
    int64_t nb1;
    int count;
    bool draft;
};
__device__ __forceinline__ TileRows tile_rows(const Args& a, const Run& r, int e, bool kV) {
    TileRows x;
    int p0;
    r.tile(e, x.draft, p0, x.count);
    x.nb1 = x.draft ? (kV ? a.vd_nb1 : a.kd_nb1) : (kV ? a.v_nb1 : a.k_nb1);
    const uint8_t* b = x.draft ? (kV ? a.vd + (int64_t)r.s * a.vd_nb2 : a.kd + (int64_t)r.s * a.kd_nb2)
                               : (kV ? seq_base(a.v_seq_ptrs, a.v, a.v_nb2, r.s) : seq_base(a.k_seq_ptrs, a.k, a.k_nb2, r.s));
    x.at = b + (int64_t)p0 * x.nb1;
    return x;
}

// A producer group's 128 threads: the slices of run r's head in the rows of entry e, to rows of raw_stride bytes; every
// thread's copies arrive on `full`.
template <int T>
__device__ __forceinline__ void load_slices(const Args& a, const Run& r, int e, uint8_t* dst, uint64_t* full, int t, bool kV) {
    constexpr int kWords = group_bytes(T) / 2, per = 128 / kWords;  // 4-byte words of a slice, keys per pass
    const TileRows x = tile_rows(a, r, e, kV);
    const uint8_t* src = x.at + r.kvh * 2 * group_bytes(T);
    if (((reinterpret_cast<uint64_t>(src) | (uint64_t)x.nb1) & 3) == 0) {
        const int k0 = t / kWords, col = (t - k0 * kWords) * 4;
        if (k0 < per) {
            const uint8_t* from = src + (int64_t)k0 * x.nb1 + col;
            uint32_t to = smem_addr(dst + k0 * raw_stride(T) + col);
            const int64_t step = (int64_t)per * x.nb1;
#pragma unroll 4
            for (int kk = k0; kk < x.count; kk += per, from += step, to += per * raw_stride(T))
                asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to), "l"(from) : "memory");
        }
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_addr(full)) : "memory");
    } else {
        constexpr int kHalves = 2 * kWords;
#pragma unroll 1
        for (int i = t; i < x.count * kHalves; i += 128) {
            const int kk = i / kHalves, h = i - kk * kHalves;
            *reinterpret_cast<uint16_t*>(dst + kk * raw_stride(T) + 2 * h) = *reinterpret_cast<const uint16_t*>(src + (int64_t)kk * x.nb1 + 2 * h);
        }
        mbar_arrive(full);
    }
}

// Largest |scale| of a row's two blocks (for types with a min a bound of |value| / 64), finite ones only.
template <int T>
__device__ __forceinline__ uint32_t row_max(const uint8_t* row, bool& special) {
    uint32_t m = 0;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
        const uint8_t* gb = row + b * group_bytes(T);
        float d = fabsf(h2f(*reinterpret_cast<const uint16_t*>(gb)));
        if constexpr (BlockTraits<T>::HAS_MIN) {
            const float mm = h2f(*reinterpret_cast<const uint16_t*>(gb + BlockTraits<T>::OFF_M));
            special |= !isfinite(mm);
            d = (32.0f * d + fabsf(mm)) * (1.0f / 64.0f);
        }
        special |= !isfinite(d);
        if (isfinite(d)) m = max(m, __float_as_uint(d));
    }
    return m;
}

// Least exponent e (tile_exp) of a tile of drafts that goes through f16.  With e >= 0 scales, f16 themselves, and hi and lo stay exact
// however small they are; values with a min are rounded to multiples of 2^-25 / 2^e.  Below it the tile's largest row, which a row of
// queries may not see, would cost the other rows bits.
template <int T> constexpr int kLeastExp = BlockTraits<T>::HAS_MIN ? 2 : 0;

// A producer warpgroup: the K (or V) tiles of the CTA, thread = key.
template <int KT, int VT, bool kV>
__device__ __forceinline__ void produce(const TcArgs& ta, uint8_t* smem, TcBars* B, const SeqTab& tab, Run r, int lo, int hi) {
    using Sh = TcShape<KT, VT>;
    constexpr int T = kV ? VT : KT, kSt = Sh::kStages, kBar = kV ? 5 : 4, raw = kV ? Sh::rawV : Sh::rawK;
    const Args& a = ta.a;
    const int key = threadIdx.x - (kV ? 384 : 256), lane = threadIdx.x & 31;
    uint8_t* tiles0 = smem + Sh::kTiles + (kV ? Sh::NK * kTcTileBytes : 0);
    uint64_t* full = kV ? B->v_full : B->k_full;
    uint64_t* empty = kV ? B->v_empty : B->k_empty;
    bool ok = true;
    if constexpr (T != kF16) {
        uint64_t* raw_full = kV ? B->rawv_full : B->rawk_full;
        uint32_t* slots = kV ? B->maxv : B->maxk;
        uint8_t* raw0 = smem + Sh::kRaw + (kV ? 3 * Sh::rawK : 0);
        Run rs = r;  // run of the tile that is fetched, two ahead of the one that is converted
        int st = 0, slot = 0, ahead = 0, first = 1;  // slot, ahead: n % 3, (n + 2) % 3
        uint32_t use = 0, turn = 0;                  // n / kSt, n / 3
#pragma unroll 1
        for (int n = -2; lo + n < hi; ++n) {
            bool draft = false, bad = false, there = false;
            const uint8_t* row = raw0 + slot * raw + key * raw_stride(T);
            if (n >= 0) {
                if (lo + n == r.end) {
                    r.next(a, tab, hi);
                    first = 1;
                }
                int p0, count;
                r.tile(lo + n, draft, p0, count);
                there = key < count;
                ok = ok && tc_wait(&raw_full[slot], turn & 1, &B->err, kV ? 43 : 42);
                const uint32_t m = __reduce_max_sync(0xffffffffu, ok && there ? row_max<T>(row, bad) : 0u);
                if (lane == 0 && m) atomicMax(&slots[slot], m);
                if (!fp::prod_bar_and(kBar, 128, ok)) break;  // (all leave together)
            }
            // every thread is past tile n - 1, whose buffer takes tile n + 2
            if (lo + n + 2 < hi) {
                if (lo + n + 2 == rs.end) rs.next(a, tab, hi);
                load_slices<T>(a, rs, lo + n + 2, raw0 + ahead * raw, &raw_full[ahead], key, kV);
            }
            ahead = ahead == 2 ? 0 : ahead + 1;
            if (n < 0) continue;
            const int e = tile_exp(__uint_as_float(slots[slot]));
            if (++slot == 3) {
                slot = 0;
                ++turn;
            }
            if (key == 0) {
                slots[slot == 2 ? 0 : slot + 1] = 0u;  // of the tile after the next: read by all before this barrier
                (kV ? B->expv : B->expk)[n % kTcExps] = draft && e < kLeastExp<T> ? 0.0f : pow2f(-e);  // (0: kept out of the products)
                if (!kV) B->starts[n % kTcExps] = (uint32_t)first;
            }
            first = 0;
            if (kV && draft) {  // which keys hold values that are not finite (their tile rows are zeros)
                const uint32_t vote = __ballot_sync(0xffffffffu, bad);
                if (lane == 0) B->bad[n % kTcExps][key >> 5] = vote;
            }
            const bool keep = there && !(kV && draft && bad);
            const float f = pow2f(e);
            if (use) ok = ok && tc_wait(&empty[st], (use - 1) & 1, &B->err, kV ? 36 : 35);
            if (ok) {
                uint8_t* tile = tiles0 + st * Sh::kStage;
                split_row<T>(tile, tile + kTcTileBytes, key, row, f, keep);
                fence_proxy_async_smem();
                mbar_arrive(&full[st]);
            }
            if (++st == kSt) {
                st = 0;
                ++use;
            }
        }
        // (after an error tiles are under way that nobody waited for; these copies are in no group)
        asm volatile("cp.async.wait_all;" ::: "memory");
    } else {
        // f16 rows straight into the tiles, kPre of them ahead of the one that is handed on
        constexpr int kPre = kSt - 2, slice = 2 * kD;
        Run rs = r;
        auto start = [&](int n) {
            if (lo + n < hi) {
                if (lo + n == rs.end) rs.next(a, tab, hi);
                const TileRows x = tile_rows(a, rs, lo + n, kV);
                const uint8_t* src = x.at + rs.kvh * slice;
                if (n >= kSt) ok = ok && tc_wait(&empty[n % kSt], (n / kSt - 1) & 1, &B->err, kV ? 34 : 33);
                uint8_t* dst = tiles0 + (n % kSt) * Sh::kStage;
                const uint64_t al = reinterpret_cast<uint64_t>(src) | (uint64_t)x.nb1;
                if (ok && (al & 15) == 0) {
                    // 8 chunks of 16 bytes per key: this thread's chunk of every 16th key, whose swizzle is the same
                    const int k0 = key >> 3, col = (key & 7) << 4;
                    const uint8_t* from = src + (int64_t)k0 * x.nb1 + col;
                    uint8_t* to = dst + k0 * 128 + (col ^ ((k0 & 7) << 4));
                    const int64_t step = 16 * x.nb1;
#pragma unroll
                    for (int u = 0; u < 8; ++u) cp_async16(to + u * 2048, k0 + 16 * u < x.count ? from + u * step : src, k0 + 16 * u < x.count);
                } else if (ok) {
                    const int unit = (al & 3) == 0 ? 4 : 2, w = slice / unit, per = unit;
                    const int k0 = key / w, col = (key - k0 * w) * unit;
#pragma unroll 1
                    for (int kk = k0; kk < kTcTile; kk += per) {
                        const bool there = kk < x.count;
                        const uint8_t* from = there ? src + (int64_t)kk * x.nb1 + col : src;
                        uint8_t* to = dst + kk * 128 + (col ^ ((kk & 7) << 4));
                        if (unit == 4) cp_async4(to, from, there);
                        else *reinterpret_cast<uint16_t*>(to) = there ? *reinterpret_cast<const uint16_t*>(from) : (uint16_t)0;
                    }
                }
            }
            cp_async_commit();
        };
        int first = 1;
#pragma unroll 1
        for (int n = -kPre; lo + n < hi; ++n) {
            if (n >= 0) {
                if (lo + n == r.end) {
                    r.next(a, tab, hi);
                    first = 1;
                }
                bool draft;
                int p0, count;
                r.tile(lo + n, draft, p0, count);
                cp_async_wait<kPre - 1>();
                if (kV && draft) {
                    if (!fp::prod_bar_and(kBar, 128, ok)) break;  // every thread's copies have landed (or all leave)
                    bool bad = false;
                    uint4* p = reinterpret_cast<uint4*>(tiles0 + (n % kSt) * Sh::kStage + key * 128);
#pragma unroll 1
                    for (int c = 0; c < 8; ++c) {
                        const uint4 w = p[c];
                        bad |= f16x2_special(w.x) || f16x2_special(w.y) || f16x2_special(w.z) || f16x2_special(w.w);
                    }
#pragma unroll 1
                    for (int c = 0; bad && c < 8; ++c) p[c] = make_uint4(0u, 0u, 0u, 0u);
                    const uint32_t vote = __ballot_sync(0xffffffffu, bad);
                    if (lane == 0) B->bad[n % kTcExps][key >> 5] = vote;
                }
                if (key == 0) {
                    (kV ? B->expv : B->expk)[n % kTcExps] = 1.0f;
                    if (!kV) B->starts[n % kTcExps] = (uint32_t)first;
                }
                first = 0;
                if (ok) {
                    fence_proxy_async_smem();
                    mbar_arrive(&full[n % kSt]);
                }
            }
            start(n + kPre);  // (may have to wait for its stage, so it comes last)
        }
        cp_async_wait<0>();
    }
}

template <int KT, int VT>
__global__ void __launch_bounds__(kTcThreads, 1) tree_tc_kernel(const __grid_constant__ TcArgs ta) {
    using Sh = TcShape<KT, VT>;
    constexpr int NK = Sh::NK, NV = Sh::NV, kSt = Sh::kStages;
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
        }
        for (int b = 0; b < 3; ++b) {
            mbar_init(&B->rawk_full[b], 128);
            mbar_init(&B->rawv_full[b], 128);
            B->maxk[b] = B->maxv[b] = 0u;
        }
        B->err = 0;
        fence_mbar_init();
    }
    if (warp == 0) {
        tc::tmem_alloc(&B->tmem_base, 512);
        tc::tmem_relinquish();
    }
    if (warp == 1) {  // list entries before each sequence
        griddep_wait();  // (every other thread touches global memory after the __syncthreads below)
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
        float* rsb = reinterpret_cast<float*>(smem + Sh::kRs);
        uint32_t k = 0;  // tiles of this group so far
        bool ok = true;
        for (; r.i < hi; r.next(a, tab, hi)) {
            const int rr = r.rt * kTcRows + row, rows = r.n * a.G;
            const bool real = rr < rows;
            const bool warp_real = r.rt * kTcRows + quad * 32 < rows;  // some row of this warp is
            const int node = (int)(((uint32_t)rr * ta.inv_g) >> 16), h = r.kvh * a.G + rr - node * a.G;
            const int64_t orow = (int64_t)r.s * a.out_nb_seq + (int64_t)node * a.out_nb_node + h * kD;
            // Q: four lanes a row, 16 dims each
            // (nothing reads the last run's Q, or its exchanged rows, any more)
            if (r.i != lo) asm volatile("bar.sync 1, 256;" ::: "memory");
#pragma unroll 1
            for (int q0 = tid >> 2; q0 < kTcRows; q0 += 64) {
                const int qr = r.rt * kTcRows + q0, qn = (int)(((uint32_t)qr * ta.inv_g) >> 16), c = lane & 3;
                const float4* q = reinterpret_cast<const float4*>(a.q + (int64_t)r.s * a.q_nb_seq + (int64_t)qn * a.q_nb_node +
                                                                  (r.kvh * a.G + qr - qn * a.G) * kD + 16 * c);
                float4 v[4];
                float am = 0.0f;
#pragma unroll
                for (int u = 0; u < 4; ++u) v[u] = qr < rows ? q[u] : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int u = 0; u < 4; ++u) am = max3(am, fmaxf(fabsf(v[u].x), fabsf(v[u].y)), fmaxf(fabsf(v[u].z), fabsf(v[u].w)));
                const int ex = dtc::norm_exp(quad_max(am));
                const float sc = a.scale_log2 < 0.0f ? -pow2f(ex) : pow2f(ex);
                if (c == 0) rsb[q0] = pow2f(-ex) * fabsf(a.scale_log2);
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    uint4 wh, wl;
                    split2(v[2 * u].x * sc, v[2 * u].y * sc, wh.x, wl.x);
                    split2(v[2 * u].z * sc, v[2 * u].w * sc, wh.y, wl.y);
                    split2(v[2 * u + 1].x * sc, v[2 * u + 1].y * sc, wh.z, wl.z);
                    split2(v[2 * u + 1].z * sc, v[2 * u + 1].w * sc, wh.w, wl.w);
                    const uint32_t at = tc::sw128_offset(q0, 2 * c + u);
                    *reinterpret_cast<uint4*>(qhi + at) = wh;
                    *reinterpret_cast<uint4*>(qlo + at) = wl;
                }
            }
            fence_proxy_async_smem();
            mbar_arrive(&B->q_full);
            asm volatile("bar.sync 3, 256;" ::: "memory");
            const float rs = rsb[row];
            float2 O[32];
#pragma unroll
            for (int d = 0; d < 32; ++d) O[d] = make_float2(0.f, 0.f);
            float base = 0.0f, thr = -INFINITY, l = 0.0f, vs_last = 1.0f;
            bool pending = false;  // a tile's output still to be added, times vs_last and its V's 2^-e
            int n_last = 0;        // that tile
            bool spoiled = false;  // the row sees a drafted value that is not finite
            // drafts p0 + 32 c .. + 31 of a tile of `count` that the row sees
            auto seen_drafts = [&](int p0, int count, int c) -> uint32_t {
                const int left = count - 32 * c, j0 = p0 + 32 * c;
                const uint32_t bits = left >= 32 ? 0xffffffffu : left <= 0 ? 0u : (1u << left) - 1u;
                if (bits == 0) return 0u;
                if (a.mask) return bits & a.mask[(int64_t)r.s * a.mask_nb_seq + (int64_t)node * a.mask_words + (j0 >> 5)];
                return node >= j0 + 31 ? bits : node < j0 ? 0u : bits & ((2u << (node - j0)) - 1u);
            };
            auto add_output = [&]() {
                uint32_t o0[32], o1[32];
                tc::tmem_ld32(ot, o0);
                tc::tmem_ld32(ot + 32, o1);
                tc::tmem_ld_wait();
                {   // keys whose V is not finite have zeros in the tile; a row that sees one is NaN in the end
                    bool draft;
                    int p0, count;
                    r.tile(lo + n_last, draft, p0, count);
#pragma unroll 1
                    for (int c = 0; draft && c < 4; ++c) {
                        const uint32_t bad = B->bad[n_last % kTcExps][c];
                        if (bad && real) spoiled |= (bad & seen_drafts(p0, count, c)) != 0;
                    }
                }
                const float vs = vs_last * B->expv[n_last % kTcExps];
                const float2 f = make_float2(vs, vs);
#pragma unroll
                for (int d = 0; d < 16; ++d) {
                    O[d] = ffma2(make_float2(__uint_as_float(o0[2 * d]), __uint_as_float(o0[2 * d + 1])), f, O[d]);
                    O[16 + d] = ffma2(make_float2(__uint_as_float(o1[2 * d]), __uint_as_float(o1[2 * d + 1])), f, O[16 + d]);
                }
            };
            // The drafts of a tile that f16 does not hold beside one another (the group's last tile), in f32 and one after another: a
            // lane has two dims of the key and the value, and every lane its row, which adds up only what it sees.  Its weights are
            // in l already where only V kept the tile out (vs_last is not 0).
            auto key_by_key = [&]() {
                bool draft;
                int p0, count;
                r.tile(lo + n_last, draft, p0, count);
                int s = r.s, t = threadIdx.x;
                asm volatile("" : "+r"(s), "+r"(t));  // (addresses are formed here: ahead of the tiles' loop they would cost its registers)
                const int rr = r.rt * kTcRows + (t & 127), node = (int)(((uint32_t)rr * ta.inv_g) >> 16);
                const float2* q = reinterpret_cast<const float2*>(a.q + (int64_t)s * a.q_nb_seq +
                                                                  (real ? (int64_t)node * a.q_nb_node + (r.kvh * a.G + rr - node * a.G) * kD : 0));
                const int blk = r.kvh * 2 + ((t >> 4) & 1), e = 2 * t & 31;
#pragma unroll 1
                for (int c = 0; c < 4; ++c) {
                    const uint32_t bits = real ? seen_drafts(p0, count, c) : 0u;
#pragma unroll 1
                    for (uint32_t any = __reduce_or_sync(0xffffffffu, bits); any; any &= any - 1) {
                        const int b = __ffs(any) - 1;
                        const int64_t at = p0 + 32 * c + b;
                        const uint8_t* kr = a.kd + (int64_t)s * a.kd_nb2 + at * a.kd_nb1 + blk * group_bytes(KT);
                        const uint8_t* vr = a.vd + (int64_t)s * a.vd_nb2 + at * a.vd_nb1 + blk * group_bytes(VT);
                        const float k0 = dequant_elem<KT>(kr, e), k1 = dequant_elem<KT>(kr, e + 1);
                        const float v0 = dequant_elem<VT>(vr, e), v1 = dequant_elem<VT>(vr, e + 1);
                        float x = 0.0f;
#pragma unroll 4
                        for (int d = 0; d < 32; ++d) {
                            const float2 y = q[d];
                            x = fmaf(y.x, __shfl_sync(0xffffffffu, k0, d), x);
                            x = fmaf(y.y, __shfl_sync(0xffffffffu, k1, d), x);
                        }
                        x = (bits >> b) & 1u ? fmaf(x, a.scale_log2, -base) : -INFINITY;
                        if (__any_sync(0xffffffffu, x > thr)) {
                            float f = 1.0f;
                            if (x > thr) {
                                const float up = x - kTcOffs;
                                f = thr == -INFINITY ? 0.0f : fast_exp2(-up);
                                base += up;
                                thr = kLazy + kTcOffs;
                                l *= f;
                                x -= up;
                            }
                            const float2 f2 = make_float2(f, f);
#pragma unroll
                            for (int d = 0; d < 32; ++d) O[d] = mul2(O[d], f2);
                        }
                        const float p = fast_exp2(x);
                        if (vs_last == 0.0f) l += p;
                        const float2 p2 = make_float2(p, p);
#pragma unroll
                        for (int d = 0; d < 32; ++d) {
                            const float2 v = make_float2(__shfl_sync(0xffffffffu, v0, d), __shfl_sync(0xffffffffu, v1, d));
                            if (p != 0.0f) O[d] = ffma2(p2, v, O[d]);
                        }
                    }
                }
            };
            for (int j = r.i + ((r.i ^ g ^ lo) & 1); j < r.end; j += 2) {  // the CTA's tiles j - lo of parity g
                bool draft;
                int p0, count;
                r.tile(j, draft, p0, count);
                const int n = j - lo, buf = n % 3;
                // (Of a buffer's phases a group sees every second one, always of the same parity.  It cannot pass on an older one:
                // S of tile n - 3, the phase before, was committed ahead of S of n - 2, which this group has seen.)
                const uint32_t sp = tmem + lane_base + buf * 128;
                ok = tc_wait(&B->s_full[buf], (n / 3) & 1, &B->err, 31);
                if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
                tc::fence_after();
                if constexpr (NK == 2) {
                    if (B->expk[n % kTcExps] == 0.0f) count = 0;  // none of its keys is seen here
                }
                if (warp_real) {
                    uint32_t sv[32];
                    tc::tmem_ld32(sp, sv);
                    const float rst = fmaxf(rs * B->expk[n % kTcExps], 1e-37f);  // above 0, so that what is masked stays -infinity
                    const bool masked = draft || count < kTcTile;
                    tc::tmem_ld_wait();
#pragma unroll 1
                    for (int c = 0; c < 4; ++c) {
                        if (masked) {
                            const int left = count - 32 * c;
                            const uint32_t bits = draft && real ? seen_drafts(p0, count, c)
                                                  : left >= 32 ? 0xffffffffu : left <= 0 ? 0u : (1u << left) - 1u;
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
                        ok = tc_wait(&B->o_full[g], (k - 1) & 1, &B->err, 32);
                        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
                        tc::fence_after();
                        add_output();
                    }
                    vs_last = NK == 2 && B->expk[n % kTcExps] == 0.0f ? 0.0f : 1.0f;
                    n_last = n;
                    pending = true;
                    tc::tmem_st_wait();
                }
                ++k;
                tc::fence_before();
                mbar_arrive(&B->p_full[buf]);
            }
            if (ok && pending) {
                ok = tc_wait(&B->o_full[g], (k - 1) & 1, &B->err, 32);
                ok = __all_sync(0xffffffffu, ok);
                tc::fence_after();
                if (ok) add_output();
            }
            if constexpr (NK == 2 || NV == 2)
                if (ok && pending && vs_last * B->expv[n_last % kTcExps] == 0.0f) key_by_key();
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
        regs_down<kTcRegsProducer>();
        produce<KT, VT, false>(ta, smem, B, tab, r, lo, hi);
    } else if (warp < 16) {
        regs_down<kTcRegsProducer>();
        produce<KT, VT, true>(ta, smem, B, tab, r, lo, hi);
    } else {
        regs_down<kTcRegsOther>();
        // ------------------------------------------------------ MMA issuers: the whole warp walks, one lane issues
        const int which = __shfl_sync(0xffffffffu, warp, 0);
        const uint64_t dt0 = tc::sdesc_sw128(smem_addr(smem + Sh::kTiles), 16, 1024);
        bool ok = true;
        if (which == 16) {
            const uint32_t idesc = tc::idesc_f16_f32(128, kTcTile, false);
            const uint64_t dqh = tc::sdesc_sw128(smem_addr(smem + Sh::kQ), 16, 1024);
            const uint64_t dql = tc::sdesc_sw128(smem_addr(smem + Sh::kQ) + kTcTileBytes, 16, 1024);
            int st = 0, buf = 0;
            uint32_t use = 0, turn = 0, n_run = 0;  // n / kSt, n / 3
            for (int n = 0; ok && lo + n < hi; ++n) {
                ok = tc_wait(&B->k_full[st], use & 1, &B->err, 38);
                if (ok && B->starts[n % kTcExps]) ok = tc_wait(&B->q_full, n_run++ & 1, &B->err, 37);
                if (ok && n >= 3) ok = tc_wait(&B->s_free[buf], (turn - 1) & 1, &B->err, 40);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tc::fence_after();
                const uint64_t dk = dt0 + (uint64_t)(st * (Sh::kStage >> 4));
                const uint32_t sp = tmem + buf * 128;
                if (elect_one()) {
#pragma unroll 1
                    for (int kk = 0; kk < 4; ++kk) {  // small terms first, while the sums are small
                        tc::mma_ss(sp, dql + kk * 2, dk + kk * 2, idesc, kk > 0 ? 1u : 0u);
                        if constexpr (NK == 2) tc::mma_ss(sp, dqh + kk * 2, dk + (kTcTileBytes >> 4) + kk * 2, idesc, 1u);
                    }
#pragma unroll 1
                    for (int kk = 0; kk < 4; ++kk) tc::mma_ss(sp, dqh + kk * 2, dk + kk * 2, idesc, 1u);
                    tc::mma_commit(&B->s_full[buf]);
                    tc::mma_commit(&B->k_empty[st]);
                }
                __syncwarp();
                if (++st == kSt) { st = 0; ++use; }
                if (++buf == 3) { buf = 0; ++turn; }
            }
        } else if (which == 17) {
            const uint32_t idesc = tc::idesc_f16_f32(128, 64, true);
            int st = 0, buf = 0;
            uint32_t use = 0, turn = 0;
            for (int n = 0; ok && lo + n < hi; ++n) {
                ok = tc_wait(&B->v_full[st], use & 1, &B->err, 41);
                if (ok) ok = tc_wait(&B->p_full[buf], turn & 1, &B->err, 39);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tc::fence_after();
                const uint64_t dv = dt0 + (uint64_t)(st * (Sh::kStage >> 4) + NK * (kTcTileBytes >> 4));
                const uint32_t sp = tmem + buf * 128, ot = tmem + 384 + (n & 1) * 64;
                if (elect_one()) {
#pragma unroll 1
                    for (int kk = 0; kk < 8; ++kk) {
                        const uint32_t ph = sp + 32 * (kk >> 1) + 8 * (kk & 1);
                        tc::mma_ts(ot, ph + 16, dv + kk * 128, idesc, kk > 0 ? 1u : 0u);
                        if constexpr (NV == 2) tc::mma_ts(ot, ph, dv + (kTcTileBytes >> 4) + kk * 128, idesc, 1u);
                    }
#pragma unroll 1
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
    if (tid == 0 && B->err) record_status(a.status, kStatusTimeout | (B->err << 8));
}

// Join of the parts of units that several CTAs shared, and the rows that no unit
// holds (a sequence without keys, rows past the last node).  16 threads per row
// (4 dims each) follow every kLanes-th part.  Bound by its latency, most of which its
// early launch hides: 2 to 3 us of the calls above.
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
