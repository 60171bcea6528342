// paged_tc.cuh -- paged attention of many rows on the 5th-generation tensor cores (tcgen05).
//
// Work is cut evenly: the key tiles (128 positions) of all units (sequence, tile of 128 rows, KV head), each unit up to the
// last position that one of its rows sees, form one list, in which kTcGap empty entries follow each unit's (a change of units
// takes a CTA as long), and CTA c of G takes the entries [c N / G, (c + 1) N / G).  A run is the part of one unit that a CTA has; a
// whole unit is written out directly, parts go to the workspace and paged_tc_combine_kernel joins them.
//   warps 0-3, 4-7  softmax groups: thread = row = TMEM lane; group g takes the CTA's tiles 2 k + g
//   warps 8-11      producers: codes to f16 tiles (128B swizzle), two warps K, two V, which is transposed as its blocks lie; Q of the
//                   next run while the softmax is still at this one
//   warp 12         issues S = Q K^T, up to two tiles ahead of the softmax;  warp 13 issues O = P V
//   warp 14         looks the tiles' pages up, copies their blocks (1 KB each, cp.async.bulk) and scales, up to three tiles ahead
//   (warp 15 only completes the last warpgroup)
// Precision: codes are exact in f16, Q and P' = P w are split in f16 hi + lo, so S = Qh K + Ql K and O = Ph V + Pl V.  A block's
// key scale multiplies its 16 columns of S; its value scale times a power of two of the row is w.  That power follows the largest
// P times value scale that the row has seen, apart from the reference that follows its largest score, so P' keeps 2^-22 of itself
// or 2^-27 of the row's largest such product, and what a row does not see costs it nothing.  Both references move by whole powers of
// two, exactly.  The output of a tile is a fresh accumulator, added in f32 to the row's registers: adds inside the tensor cores
// truncate.
// TMEM: three S buffers of 128 columns, tile n in n % 3, each overwritten 32 positions at a time by that chunk's P' (16 columns
// hi, 16 lo); two outputs of 64 columns, one per group, read back while the group's next tile is on its way.
// What bounds it: a tile takes a CTA about 2800 cycles, as its softmax groups take 5600 for every second one (850 for 32 positions:
// maxima, exponentials, the split into hi and lo; neither fewer instructions for that split nor faster producers changed the sum).  The
// first S is there after 11 thousand cycles (lengths, list, page, block, f16 tile, all run once, with cold instructions),
// the last tile's end takes 6.  16 sequences of 16 rows over 8192, i8: 38.4 us (the bytes alone take 5.4; tensor pipe 24 % of active
// cycles, exponentials' unit 24 %, issue 38 %); 4 of 512 rows over up to 2501, e4m3: 44.2.
#pragma once

#include <cfloat>

#include "flash_pipe.cuh"
#include "paged_mma.cuh"

namespace cvattn {
namespace paged {

constexpr int kTcTile = 128;   // positions
constexpr int kTcRows = 128;
constexpr int kTcThreads = 16 * 32;
// Registers of a thread by role: launched with 128.
constexpr int kTcRegsSoftmax = 200, kTcRegsProducer = 72, kTcRegsOther = 32;
static_assert(256 * kTcRegsSoftmax + 128 * kTcRegsProducer + 128 * kTcRegsOther <= 512 * 128, "the block's registers");
constexpr int kTcMaxSeq = 1024;  // tables in shared memory
constexpr int kTcSt = 3;         // K and V tiles under way
constexpr int kTcRaw = 3;        // tiles of codes under way
constexpr int kTcGap = 4;        // what a change of runs costs, in tiles (us of 16 x 16 over 8192 | 4 x 512 of 2501: 2 43.7 | 52.1,
                                 // 4 41.7 | 47.6, 6 42.5 | 48.5, 8 42.7 | 49.0; none 43.4 | 64)
constexpr int kTcInfos = 8;      // tiles whose scales may be in use
constexpr int kTcTileBytes = kTcTile * kD * 2;
constexpr int kTcBlocks = kTcTile / kBlock;

struct TcAttArgs {
    AttArgs a;
    int grid;          // CTAs that share the list
    float* ws_o;       // [2 * grid][128][64]
    float* ws_ml;      // [2 * grid][128][2]
    int32_t* ws_pref;  // [n_seq + 1], written by CTA 0 for the combine
};

struct __align__(16) TcInfo {   // of a tile
    float4 scales[kTcBlocks / 2];  // by 32 positions: two blocks' of the keys, of the values
    float lg;                      // log2 of the largest of the latter (of 0: -infinity), about
    uint32_t valid;             // blocks that have a page
    uint32_t starts, last;      // whether the tile starts a run; is the CTA's last
    int32_t count;              // positions that exist
};

struct TcAttBars {
    uint64_t k_full[kTcSt], v_full[kTcSt], k_empty[kTcSt], v_empty[kTcSt];  // by stage
    uint64_t raw_full[kTcRaw], raw_empty[kTcRaw];                           // by slot of codes
    uint64_t q_full[2], q_free[2];                                          // by Q buffer: run n in n % 2
    uint64_t s_full[3], p_full[3], s_free[3];                               // by S buffer
    uint64_t o_full[2];                                                     // by group
    uint32_t tmem_base;
    int err;
    TcInfo info[kTcInfos];      // tile n at n % kTcInfos
    int32_t first_run[16];      // TcRun at the start of the CTA's part
    int32_t hi;                 // the part's end
};

struct TcSmem {
    static constexpr int kQ = 0;                            // [run % 2][Q hi, Q lo]; at the run's end its output
    static constexpr int kTiles = 4 * kTcTileBytes;         // [stage][K, V]
    static constexpr int kRaw = kTiles + kTcSt * 2 * kTcTileBytes;  // [slot][K, V][block]
    static constexpr int kRawBytes = 2 * kTcBlocks * kBlockBytes;
    static constexpr int kMl = kRaw + kTcRaw * kRawBytes;
    static constexpr int kRs = kMl + kTcRows * 8;           // [run % 2] score factors of the rows
    static constexpr int kBars = kRs + 2 * kTcRows * 4;
    static constexpr int kPref = kBars + (int)((sizeof(TcAttBars) + 15) / 16 * 16);
    static constexpr int kLen = kPref + (kTcMaxSeq + 4) * 4, kRowsOf = kLen + kTcMaxSeq * 4;
    static constexpr int kBytes = kRowsOf + kTcMaxSeq * 4;
};
static_assert(TcSmem::kBytes <= 227 * 1024, "one CTA per SM");
static_assert(TcSmem::kBars % 16 == 0 && sizeof(TcInfo) % 16 == 0, "pairs of scales are read at once");

template <int N> __device__ __forceinline__ void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r != 0;
}
__device__ __forceinline__ float less_f16(float x, uint16_t h) {  // x - h, exact where h is x's nearest f16
    float r;
    asm("fma.rn.f32.f16 %0, %1, %2, %3;" : "=f"(r) : "h"(h), "h"((uint16_t)0xBC00u), "f"(x));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    unsigned long long ra = *reinterpret_cast<unsigned long long*>(&a), rb = *reinterpret_cast<unsigned long long*>(&b), rd;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(rd) : "l"(ra), "l"(rb));
    return *reinterpret_cast<float2*>(&rd);
}
__device__ __forceinline__ float log2_of(float scale) { return scale > 0.0f ? __log2f(scale) : -INFINITY; }
// 2^e for whole e <= 0 (0 below f32's normal numbers).
__device__ __forceinline__ float shrink_by(float e) { return e < -126.0f ? 0.0f : pow2f((int)e); }

// What a row's weights and outputs are kept relative to.  P is 2^(score - base); a score above thr raises base.  P' is P times value
// scale times wk = 2^ko, and a score plus log2 of its value scale above thr_o lowers ko: to a largest P' of 2^kOutOffs, with room up to
// 2^15, which leaves lo's last bit (2^-24) 2^-27 of it.  (From 2^7 on, as P, P' outgrew its room and was rounded anew in TMEM more often
// than P: 16 sequences of 16 rows over 8192 40.6 us, 38.4 so.)  Both move by whole powers of two, exactly.  (thr, thr_o -infinity: no
// score, no scale above 0 yet)
constexpr float kOutOffs = 3.0f;
struct RowRef {
    float base = 0.0f, thr = -INFINITY, ko = 0.0f, wk = 1.0f, thr_o = -INFINITY;
    // Below it no score passes thr, nor with a value scale of up to 2^lg thr_o.
    __device__ __forceinline__ float quiet(float lg) const { return fminf(thr, thr_o - lg); }
    // (past FLT_MAX only where P is below 2^-113)
    __device__ __forceinline__ float weight(float scale) const { return fminf(scale * wk, FLT_MAX); }
    // Of outputs, to units of P times value.
    __device__ __forceinline__ float unit() const { return pow2f(-(int)ko); }
    // For largest scores m0, m1 of blocks with value scales s0, s1: returns what is to be taken from scores, the outputs' factor in f;
    // l, the sum of P, is brought along.
    __device__ __forceinline__ float raise(float m0, float s0, float m1, float s1, float& l, float& f) {
        float top = fmaxf(m0 + log2_of(s0), m1 + log2_of(s1)), up = 0.0f;
        const float mx = fmaxf(m0, m1);
        if (mx > thr) {
            up = rintf(mx) - kOffs;
            l *= thr == -INFINITY ? 0.0f : shrink_by(-up);
            base += up;
            thr = kLazy + kOffs;
            top -= up;
        }
        const bool had = thr_o != -INFINITY;
        const float k = had ? ko + up : 0.0f;  // what leaves the outputs as they are
        ko = k;
        if (top > thr_o - up) {
            ko = kOutOffs - rintf(top);
            thr_o = 0.0f;
        }
        ko = fminf(fmaxf(ko, -126.0f), 126.0f);
        wk = pow2f((int)ko);
        f = had ? shrink_by(ko - k) : 1.0f;
        if (thr_o != -INFINITY) thr_o = kLazy + kOffs - ko;
        return up;
    }
};

// Bounded wait: gives up after kTcTries suspensions of up to 20 us, or once another role has given up.  *err keeps the site; the
// kernel's end records it.
constexpr uint32_t kTcTries = 100000;
__device__ __forceinline__ bool tc_wait(uint64_t* bar, uint32_t parity, int* err, int site) {
#pragma unroll 1
    for (uint32_t i = 0; !mbar_try_wait_hint(bar, parity, 20000u); ++i) {
        if (i >= kTcTries) *reinterpret_cast<volatile int*>(err) = site;
        if (*reinterpret_cast<volatile int*>(err)) return false;
    }
    return true;
}

// Positions that the last row of row tile rt sees, of a sequence with L positions and n of them as rows.
__device__ __forceinline__ int tc_end(const AttArgs& a, int L, int n, int rt) {  // n > 0
    const int last = min(n * a.G, (rt + 1) * kTcRows) - 1;
    return max(0, L - n + 1 + divided(last, a.by_G));
}
__device__ __forceinline__ int tc_tiles(const AttArgs& a, int L, int n, int rt) { return (tc_end(a, L, n, rt) + kTcTile - 1) / kTcTile; }
// List entries of a unit.
__device__ __forceinline__ int tc_entries(const AttArgs& a, int L, int n, int rt) {
    const int T = tc_tiles(a, L, n, rt);
    return T ? T + kTcGap : 0;
}
// Where CTA c's part of n entries begins; whose part entry i lies in.
__device__ __forceinline__ int tc_cut(const TcAttArgs& ta, int c, int n) { return cut_at(c, n, ta.grid, ta.a.by_parts); }
__device__ __forceinline__ int tc_owner(const TcAttArgs& ta, int i, int n) {
    int c = min((int)((float)i * (float)ta.grid / (float)n), ta.grid - 1);  // off by one at most
    while (tc_cut(ta, c, n) > i) --c;
    while (tc_cut(ta, c + 1, n) <= i) ++c;
    return c;
}

struct TcTab {  // in shared memory, by sequence: list entries before it, positions, rows (tokens)
    const int32_t *pref, *len, *n;
};
// A CTA's walk through its part [lo, hi) of the list, run by run.
struct TcRun {
    int s, kvh, rt;   // unit
    int v;            // its first entry
    int t0, t1, T;    // the CTA's tiles of it (none: the part has ended), the unit's
    int at;           // tiles of the CTA before this run
    int L, n, see;    // positions, tokens, positions that the unit's last row sees

    __device__ __forceinline__ void unit(const AttArgs& a) {
        see = tc_end(a, L, n, rt);
        T = (see + kTcTile - 1) / kTcTile;
    }
    __device__ __forceinline__ void start(const AttArgs& a, const TcTab& tab, int lo, int hi) {
        at = t0 = t1 = 0;
        if (lo >= hi) return;
        int below = 0, up = a.p.n_seq;  // last s with pref[s] <= lo: its list is not empty
        while (up - below > 1) {
            const int mid = (below + up) >> 1;
            if (tab.pref[mid] <= lo) below = mid;
            else up = mid;
        }
        s = below;
        L = tab.len[s];
        n = tab.n[s];
        int e = lo - tab.pref[s];
        rt = 0;
        for (unit(a); T == 0 || e >= (T + kTcGap) * a.p.pool.n_heads; unit(a)) {
            if (T) e -= (T + kTcGap) * a.p.pool.n_heads;
            ++rt;
        }
        kvh = e / (T + kTcGap);
        t0 = e - kvh * (T + kTcGap);
        v = lo - t0;
        t1 = min(T, hi - v);
        if (t0 >= T) {
            t0 = t1;
            next(a, tab, hi);
        }
    }
    __device__ __forceinline__ void next(const AttArgs& a, const TcTab& tab, int hi) {
        at += t1 - t0;
        v += T + kTcGap;
        t0 = t1 = 0;
        if (v >= hi) return;
        if (++kvh == a.p.pool.n_heads) {
            kvh = 0;
            if (++rt * kTcRows >= n * a.G) {
                do ++s;
                while (tab.pref[s + 1] == tab.pref[s]);
                L = tab.len[s];
                n = tab.n[s];
                rt = 0;
            }
            for (unit(a); T == 0; unit(a)) ++rt;  // (row tiles without entries come first)
        }
        t1 = min(T, hi - v);
    }
};

// Codes of 0 where `keep` is 0.
template <int F> __device__ __forceinline__ void keep_bytes(uint4& v, uint32_t keep) {
    const uint32_t zero = F == kI8 ? 0x80808080u & ~keep : 0u;
    v = make_uint4((v.x & keep) | zero, (v.y & keep) | zero, (v.z & keep) | zero, (v.w & keep) | zero);
}

// Warp 14: lane i < 8 looks after block i of each tile.
__device__ __forceinline__ void tc_load(const TcAttArgs& ta, uint8_t* smem, TcAttBars* B, const TcTab& tab, TcRun r, int hi) {
    const AttArgs& a = ta.a;
    const int lane = threadIdx.x & 31, shift = __ffs(a.blocks) - 1;
    // of the tile that is looked up: whether this lane has a block, its page and place; the tile's positions
    bool has = false;
    int page = -1, in = 0, count = 0, first = 1, t = r.t0;
    auto look = [&]() {
        has = false;
        count = 0;
        if (r.t0 == r.t1) return;
        first = t == r.t0;
        if (t == r.t1) {
            r.next(a, tab, hi);
            if (r.t0 == r.t1) return;
            t = r.t0;
            first = 1;
        }
        const int p0 = t * kTcTile, b = p0 / kBlock + lane, at = b >> shift;
        ++t;
        count = min(kTcTile, r.see - p0);
        has = lane < kTcBlocks && lane * kBlock < count;
        if (has) {
            page = __ldg(a.p.table + (int64_t)r.s * a.p.table_nb_seq + at);  // (looked at when the tile's turn has come)
            in = ((r.kvh - at) << shift) + b;
        }
    };
    bool ok = true;
    int slot = 0, n = 0;
    uint32_t use = 0;
    look();
#pragma unroll 1
    for (; count > 0; ++n) {
        if (use) ok = tc_wait(&B->raw_empty[slot], (use - 1) & 1, &B->err, 34);
        if (!__all_sync(0xffffffffu, ok)) break;
        const bool good = has && (uint32_t)page < (uint32_t)a.p.pool.n_pages;
        if (has && !good) record_status(a.status, kStatusBadPage);
        const uint32_t valid = __ballot_sync(0xffffffffu, good);
        const int64_t at = good ? page * a.p.pool.nb_page + (int64_t)in * kBlockBytes : 0, sat = good ? page * a.p.pool.nb_scale + in : 0;
        const float ks = good ? a.p.pool.k_scale[sat] : 0.0f, vs = good ? a.p.pool.v_scale[sat] : 0.0f;
        if (lane == 0) mbar_arrive_expect_tx(&B->raw_full[slot], __popc(valid) * 2 * kBlockBytes);
        __syncwarp();
        uint8_t* raw = smem + TcSmem::kRaw + slot * TcSmem::kRawBytes;
        if (good) {
            bulk_g2s(raw + lane * kBlockBytes, static_cast<const uint8_t*>(a.p.pool.k) + at, kBlockBytes, &B->raw_full[slot]);
            bulk_g2s(raw + (kTcBlocks + lane) * kBlockBytes, static_cast<const uint8_t*>(a.p.pool.v) + at, kBlockBytes, &B->raw_full[slot]);
        }
        const uint32_t last = t == r.t1 && r.v + r.T + kTcGap >= hi;
        TcInfo& info = B->info[n % kTcInfos];
        const float ks1 = __shfl_down_sync(0xffffffffu, ks, 1), vs1 = __shfl_down_sync(0xffffffffu, vs, 1);
        const float most = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(fmaxf(vs, 0.0f))));
        if (lane < kTcBlocks && !(lane & 1)) info.scales[lane >> 1] = make_float4(ks, ks1, vs, vs1);
        if (lane == 0) {
            info.lg = log2_of(most);
            info.valid = valid;
            info.starts = (uint32_t)first;
            info.last = last;
            info.count = count;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&B->raw_full[slot]);  // (the second of its two arrivals: what is said of the tile)
        look();
        if (++slot == kTcRaw) {
            slot = 0;
            ++use;
        }
    }
    // after an error copies are under way that nobody waited for
    if (!ok)
        for (int k = n > kTcRaw ? n - kTcRaw : 0; k < n; ++k)
            for (uint32_t i = 0; i < kTcTries && !mbar_try_wait_hint(&B->raw_full[k % kTcRaw], (k / kTcRaw) & 1, 20000u); ++i) {}
}

// Q of a run, by kThreads threads: four lanes a row, 16 dims each.
template <int kThreads> __device__ __forceinline__ void tc_queries(const AttArgs& a, uint8_t* smem, const TcRun& r, int buf) {
    const int t = threadIdx.x & (kThreads - 1), c = t & 3, rows = r.n * a.G;
    uint8_t* hi = smem + TcSmem::kQ + buf * 2 * kTcTileBytes;
    float* rsb = reinterpret_cast<float*>(smem + TcSmem::kRs) + buf * kTcRows;
#pragma unroll 2
    for (int q0 = t >> 2; q0 < kTcRows; q0 += kThreads / 4) {
        const int qr = r.rt * kTcRows + q0, qt = divided(qr, a.by_G);
        const float4* q = reinterpret_cast<const float4*>(a.p.q + (int64_t)r.s * a.p.q_nb_seq + (int64_t)qt * a.p.q_nb_tok +
                                                          (r.kvh * a.G + qr - qt * a.G) * kD + 16 * c);
        float4 v[4];
        float am = 0.0f;
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = qr < rows ? q[u] : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int u = 0; u < 4; ++u) am = fmaxf(am, fmaxf(fmaxf(fabsf(v[u].x), fabsf(v[u].y)), fmaxf(fabsf(v[u].z), fabsf(v[u].w))));
        const int ex = query_exp(quad_max(am));
        const float f = pow2f(ex);
        if (c == 0) rsb[q0] = pow2f(-ex) * a.scale_log2;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            uint4 wh, wl;
            split_near(make_float2(v[2 * u].x * f, v[2 * u].y * f), wh.x, wl.x);
            split_near(make_float2(v[2 * u].z * f, v[2 * u].w * f), wh.y, wl.y);
            split_near(make_float2(v[2 * u + 1].x * f, v[2 * u + 1].y * f), wh.z, wl.z);
            split_near(make_float2(v[2 * u + 1].z * f, v[2 * u + 1].w * f), wh.w, wl.w);
            const uint32_t at = tc::sw128_offset(q0, 2 * c + u);
            *reinterpret_cast<uint4*>(hi + at) = wh;
            *reinterpret_cast<uint4*>(hi + kTcTileBytes + at) = wl;
        }
    }
    fence_proxy_async_smem();
}

// The producers: Q of each run but the first, then warps 0 and 1 turn a tile's keys into f16 rows, 2 and 3 its values, four blocks each.
template <int F> __device__ __forceinline__ void tc_produce(const TcAttArgs& ta, uint8_t* smem, TcAttBars* B, const TcTab& tab, TcRun r, int hi) {
    const int w = threadIdx.x >> 5 & 1, lane = threadIdx.x & 31;
    const bool keys = !(threadIdx.x & 64);
    // keys: rows 8 apart, which swizzle alike; values: pieces (half of the dims, g, quarters 2 u and 2 u + 1) to rows of dims, 64
    // positions each
    const int k0 = ((2 * (lane & 3)) ^ (lane >> 2)) * 16, k1 = k0 ^ 16;
    const int u = lane & 1, g = lane >> 1 & 7, h = lane >> 4;
    const int to0 = keys ? (w * 64 + (lane >> 2)) * 128 : kTcTileBytes + w * (kTcTileBytes / 2) + (32 * h + g) * 128;
    const int from0 = keys ? 4 * w * 64 + lane : (kTcBlocks + 4 * w) * 64 + h * 32 + 4 * g + 2 * u;
    uint64_t *empty = keys ? B->k_empty : B->v_empty, *full = keys ? B->k_full : B->v_full;
    bool ok = true;
    int st = 0, slot = 0;
    uint32_t use = 0, turn = 0, run = 0;
    bool last = r.t0 == r.t1;
#pragma unroll 1
    for (int n = 0; !last; ++n) {
        ok = tc_wait(&B->raw_full[slot], turn & 1, &B->err, 33);
        if (!__all_sync(0xffffffffu, ok)) break;
        last = B->info[n % kTcInfos].last;
        if (n && B->info[n % kTcInfos].starts) {
            r.next(ta.a, tab, hi);
            if (++run > 1) ok = tc_wait(&B->q_free[run & 1], ((run >> 1) - 1) & 1, &B->err, 42);
            if (!__all_sync(0xffffffffu, ok)) break;
            tc_queries<128>(ta.a, smem, r, run & 1);
            mbar_arrive(&B->q_full[run & 1]);
        }
        if (ok && use) ok = tc_wait(&empty[st], (use - 1) & 1, &B->err, 35);
        if (!__all_sync(0xffffffffu, ok)) break;
        uint8_t* tile = smem + TcSmem::kTiles + st * 2 * kTcTileBytes + to0;
        const uint4* raw = reinterpret_cast<const uint4*>(smem + TcSmem::kRaw + slot * TcSmem::kRawBytes) + from0;
        if (keys) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                uint4 d[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) d[i] = raw[(4 * e + i) * 32];
                if (e) mbar_arrive(&B->raw_empty[slot]);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint4 x, y;
                    to_f16<F>(d[i].x, x.x, x.y);
                    to_f16<F>(d[i].y, x.z, x.w);
                    to_f16<F>(d[i].z, y.x, y.y);
                    to_f16<F>(d[i].w, y.z, y.w);
                    *reinterpret_cast<uint4*>(tile + (4 * e + i) * 8 * 128 + k0) = x;
                    *reinterpret_cast<uint4*>(tile + (4 * e + i) * 8 * 128 + k1) = y;
                }
            }
        } else {
            const uint32_t valid = B->info[n % kTcInfos].valid;
            const int count = B->info[n % kTcInfos].count;
#pragma unroll
            for (int e0 = 0; e0 < 4; e0 += 2) {
                uint4 v[4];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    v[2 * e] = raw[(e0 + e) * 64];
                    v[2 * e + 1] = raw[(e0 + e) * 64 + 1];
                }
                if (e0) mbar_arrive(&B->raw_empty[slot]);
                if (count < kTcTile || valid != 0xffu) {  // (what lies past the end may be NaN)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        // positions 8 u .. + 7 of the block that exist, four bytes at a time
                        const int b = 4 * w + e0 + e, left = valid >> b & 1u ? count - b * kBlock - 8 * u : 0;
                        keep_bytes<F>(v[2 * e], left >= 4 ? 0xffffffffu : left <= 0 ? 0u : (1u << (8 * left)) - 1u);
                        keep_bytes<F>(v[2 * e + 1], left >= 8 ? 0xffffffffu : left <= 4 ? 0u : (1u << (8 * (left - 4))) - 1u);
                    }
                }
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const uint32_t x[4] = {v[2 * e].x, v[2 * e].y, v[2 * e].z, v[2 * e].w};
                    const uint32_t y[4] = {v[2 * e + 1].x, v[2 * e + 1].y, v[2 * e + 1].z, v[2 * e + 1].w};
                    uint8_t* to = tile + (((e0 + e) * 2 + u) ^ g) * 16;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        uint4 o;
                        to_f16<F>(x[j], o.x, o.y);
                        to_f16<F>(y[j], o.z, o.w);
                        *reinterpret_cast<uint4*>(to + j * 8 * 128) = o;
                    }
                }
            }
        }
        fence_proxy_async_smem();
        mbar_arrive(&full[st]);
        if (++st == kTcSt) {
            st = 0;
            ++use;
        }
        if (++slot == kTcRaw) {
            slot = 0;
            ++turn;
        }
    }
}

template <int F>
__global__ void __launch_bounds__(kTcThreads, 1) paged_tc_kernel(const __grid_constant__ TcAttArgs ta) {
    using Sh = TcSmem;
    extern __shared__ __align__(1024) uint8_t smem[];
    const AttArgs& a = ta.a;
    TcAttBars* B = reinterpret_cast<TcAttBars*>(smem + Sh::kBars);
    int32_t* pref = reinterpret_cast<int32_t*>(smem + Sh::kPref);
    int32_t *len = reinterpret_cast<int32_t*>(smem + Sh::kLen), *toks = reinterpret_cast<int32_t*>(smem + Sh::kRowsOf);
    const TcTab tab{pref, len, toks};
    if (smem_addr(smem) & 1023u) {
        if (threadIdx.x == 0) record_status(a.status, kStatusTimeout);
        return;
    }
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int i = 0; i < kTcSt; ++i) {
            mbar_init(&B->k_full[i], 64);
            mbar_init(&B->v_full[i], 64);
            mbar_init(&B->k_empty[i], 1);
            mbar_init(&B->v_empty[i], 1);
        }
        for (int i = 0; i < kTcRaw; ++i) {
            mbar_init(&B->raw_full[i], 2);
            mbar_init(&B->raw_empty[i], 128);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&B->q_full[b], 128);
            mbar_init(&B->q_free[b], 256);
        }
        for (int b = 0; b < 3; ++b) {
            mbar_init(&B->s_full[b], 1);
            mbar_init(&B->p_full[b], 128);
            mbar_init(&B->s_free[b], 1);
        }
        for (int g = 0; g < 2; ++g) mbar_init(&B->o_full[g], 1);
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
        for (int base = 0; base < a.p.n_seq; base += 32) {
            const int s = base + lane;
            int n = 0;
            if (s < a.p.n_seq) {
                const AttLens x = att_lens(a, s, blockIdx.x == 0);
                for (int rt = 0; rt * kTcRows < x.n * a.G; ++rt) n += tc_entries(a, x.L, x.n, rt);
                n *= a.p.pool.n_heads;
                len[s] = x.L;
                toks[s] = x.n;
            }
            int incl = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += y;
            }
            if (s < a.p.n_seq) {
                pref[s] = carry + incl - n;
                if (blockIdx.x == 0) ta.ws_pref[s] = carry + incl - n;
            }
            carry += __shfl_sync(0xffffffffu, incl, 31);
        }
        if (lane == 0) {
            pref[a.p.n_seq] = carry;
            if (blockIdx.x == 0) ta.ws_pref[a.p.n_seq] = carry;
        }
        __syncwarp();
        TcRun r{};
        const int lo = tc_cut(ta, blockIdx.x, carry), hi = tc_cut(ta, blockIdx.x + 1, carry);
        r.start(a, tab, lo, hi);
        if (lane == 0) B->hi = hi;
        static_assert(sizeof(TcRun) <= sizeof(B->first_run), "a run in shared memory");
        if (lane == 0) *reinterpret_cast<TcRun*>(B->first_run) = r;
    }
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    griddep_launch_dependents();
    const uint32_t tmem = B->tmem_base;
    const int hi = B->hi;
    TcRun r = *reinterpret_cast<const TcRun*>(B->first_run);

    if (warp < 8) {
        // ------------------------------------------------------ softmax group g
        regs_up<kTcRegsSoftmax>();
        const int g = warp >> 2, quad = warp & 3, row = quad * 32 + lane;
        const uint32_t lane_base = (uint32_t)(quad * 32) << 16;
        const uint32_t ot = tmem + lane_base + 384 + g * 64;
        float2* mls = reinterpret_cast<float2*>(smem + Sh::kMl) + row;
        const float* rsb = reinterpret_cast<const float*>(smem + Sh::kRs);
        uint32_t k = 0, run = 0;  // tiles of this group, runs so far
        bool ok = true;
        if (r.t0 < r.t1) {
            tc_queries<256>(a, smem, r, 0);
            asm volatile("bar.sync 3, 256;" ::: "memory");
            if (g == 0) mbar_arrive(&B->q_full[0]);
        }
        for (; r.t0 < r.t1; r.next(a, tab, hi), ++run) {
            const int rr = r.rt * kTcRows + row, rows = r.n * a.G, before = r.L - r.n + 1;
            const bool real = rr < rows;
            const bool warp_real = r.rt * kTcRows + quad * 32 < rows;  // some row of this warp is
            const int tok = divided(rr, a.by_G), h = r.kvh * a.G + rr - tok * a.G;
            const int lim = real ? before + tok : 0;                   // positions that the row sees
            const int sure = before + divided(r.rt * kTcRows, a.by_G);          // that all rows of the unit do
            ok = tc_wait(&B->q_full[run & 1], run >> 1 & 1, &B->err, 37);
            ok = __all_sync(0xffffffffu, ok);
            const float rs = rsb[(run & 1) * kTcRows + row];
            float2 O[32];
#pragma unroll
            for (int d = 0; d < 32; ++d) O[d] = make_float2(0.f, 0.f);
            RowRef ref;
            float l = 0.0f, late = 1.0f;
            bool pending = false;  // a tile's output still to be added, times late
            auto add_output = [&]() {
                uint32_t o0[32];
                const float2 f = make_float2(late, late);
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    tc::tmem_ld32(ot + 32 * e, o0);
                    tc::tmem_ld_wait();
#pragma unroll
                    for (int d = 0; d < 16; ++d)
                        O[16 * e + d] = ffma2(make_float2(__uint_as_float(o0[2 * d]), __uint_as_float(o0[2 * d + 1])), f, O[16 * e + d]);
                }
            };
            for (int n = r.at + ((r.at ^ g) & 1); ok && n < r.at + r.t1 - r.t0; n += 2) {  // the CTA's tiles of parity g
                const int p0 = (r.t0 + n - r.at) * kTcTile, buf = n % 3;
                // (Of a buffer's phases a group sees every second one, always of the same parity.  It cannot pass on an older one:
                // S of tile n - 3, the phase before, was committed ahead of S of n - 2, which this group has seen.)
                const uint32_t sp = tmem + lane_base + buf * 128;
                ok = tc_wait(&B->s_full[buf], (n / 3) & 1, &B->err, 31);
                if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
                tc::fence_after();
                const TcInfo& info = B->info[n % kTcInfos];
                if (warp_real) {
                    uint32_t sv[32];
                    tc::tmem_ld32(sp, sv);
                    const uint32_t valid = info.valid;
                    const bool masked = p0 + kTcTile > sure || valid != 0xffu;
                    float quiet = ref.quiet(info.lg);
                    tc::tmem_ld_wait();
#pragma unroll 1
                    for (int c = 0; c < 4; ++c) {
                        const float4 sc = info.scales[c];
                        const float2 ks = make_float2(sc.x, sc.y);
                        float2 w = make_float2(ref.weight(sc.z), ref.weight(sc.w));
                        float2 x[16];
                        {
                            const float f0 = rs * ks.x, f1 = rs * ks.y;
                            const float2 b = make_float2(-ref.base, -ref.base);
#pragma unroll
                            for (int d = 0; d < 16; ++d) {
                                const float f = d < 8 ? f0 : f1;
                                x[d] = ffma2(make_float2(__uint_as_float(sv[2 * d]), __uint_as_float(sv[2 * d + 1])), make_float2(f, f), b);
                            }
                        }
                        tc::tmem_ld32(sp + 32 * min(c + 1, 3), sv);  // under way during this chunk's arithmetic
                        if (masked) {
                            const int left = lim - p0 - 32 * c;
                            uint32_t bits = left >= 32 ? 0xffffffffu : left <= 0 ? 0u : (1u << left) - 1u;
                            if (!(valid >> (2 * c) & 1u)) bits &= 0xffff0000u;
                            if (!(valid >> (2 * c + 1) & 1u)) bits &= 0x0000ffffu;
#pragma unroll
                            for (int d = 0; d < 16; ++d) {
                                if (!(bits >> (2 * d) & 1u)) x[d].x = -INFINITY;
                                if (!(bits >> (2 * d + 1) & 1u)) x[d].y = -INFINITY;
                            }
                        }
                        float m4[4];
#pragma unroll
                        for (int u = 0; u < 4; ++u)
                            m4[u] = max3(max3(max3(x[4 * u].x, x[4 * u].y, x[4 * u + 1].x), x[4 * u + 1].y, x[4 * u + 2].x),
                                         fmaxf(x[4 * u + 2].y, x[4 * u + 3].x), x[4 * u + 3].y);
                        const float m0 = fmaxf(m4[0], m4[1]), m1 = fmaxf(m4[2], m4[3]), mx = fmaxf(m0, m1);
                        if (__any_sync(0xffffffffu, mx > quiet)) {
                            float f;
                            const float up = ref.raise(m0, sc.z, m1, sc.w, l, f);
                            late *= f;
                            quiet = ref.quiet(info.lg);
                            w = make_float2(ref.weight(sc.z), ref.weight(sc.w));
#pragma unroll
                            for (int d = 0; d < 16; ++d) {
                                x[d].x -= up;
                                x[d].y -= up;
                            }
                            const bool shrinks = __any_sync(0xffffffffu, f != 1.0f);
                            if (shrinks) {
                                const float2 f2 = make_float2(f, f);
#pragma unroll
                                for (int d = 0; d < 32; ++d) O[d] = mul2(O[d], f2);
                            }
                            if (shrinks && c) {  // this tile's P' so far, 16 positions at a time
                                tc::tmem_ld_wait();
                                tc::tmem_st_wait();
#pragma unroll 1
                                for (int e = 0; e < 2 * c; ++e) {
                                    uint32_t ph[8], pl[8];
                                    const uint32_t at = sp + 32 * (e >> 1) + 8 * (e & 1);
                                    tc::tmem_ld8(at, ph);
                                    tc::tmem_ld8(at + 16, pl);
                                    tc::tmem_ld_wait();
#pragma unroll
                                    for (int d = 0; d < 8; ++d) {
                                        const float2 u = __half22float2(*reinterpret_cast<const __half2*>(&ph[d]));
                                        const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&pl[d]));
                                        split_near(make_float2((u.x + y.x) * f, (u.y + y.y) * f), ph[d], pl[d]);
                                    }
                                    tc::tmem_st8(at, ph);
                                    tc::tmem_st8(at + 16, pl);
                                }
                            }
                        }
                        float2 l0 = make_float2(0.f, 0.f), l1 = l0;
                        uint32_t pv[32];
#pragma unroll
                        for (int d = 0; d < 16; ++d) {
                            x[d].x = fast_exp2(x[d].x);
                            x[d].y = fast_exp2(x[d].y);
                            if (d & 1) l1 = add2(l1, x[d]);
                            else l0 = add2(l0, x[d]);
                            const float wd = d < 8 ? w.x : w.y;
                            const float2 y = mul2(x[d], make_float2(wd, wd));
                            pv[d] = tc::pack_f16x2(y.x, y.y);
                            pv[16 + d] = tc::pack_f16x2(less_f16(y.x, (uint16_t)pv[d]), less_f16(y.y, (uint16_t)(pv[d] >> 16)));
                        }
                        l0 = add2(l0, l1);
                        l += l0.x + l0.y;
                        tc::tmem_st32(sp + 32 * c, pv);
                        tc::tmem_ld_wait();
                    }
                    if (pending) {  // the output of the group's tile before this one (o_full counts every tile of the group)
                        ok = tc_wait(&B->o_full[g], (k - 1) & 1, &B->err, 32);
                        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
                        tc::fence_after();
                        add_output();
                    }
                    late = 1.0f;
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
            tc::fence_before();
            if (!fp::prod_bar_and(2, 256, ok)) break;  // every MMA of the run is done; all threads leave together
            const float m_mine = ref.thr == -INFINITY && l == 0.0f ? -INFINITY : ref.base;  // (NaN scores raise nothing)
            const float unit = ref.unit();
#pragma unroll
            for (int d = 0; d < 32; ++d) O[d] = mul2(O[d], make_float2(unit, unit));
            // group 1's rows to where Q was, joined there by group 0, written by both
            float4* rows_at = reinterpret_cast<float4*>(smem + Sh::kQ + (run & 1) * 2 * kTcTileBytes);
            float4* mine = rows_at + row * 16;
            if (g == 1) {
#pragma unroll
                for (int c = 0; c < 16; ++c) mine[c ^ (row & 7)] = make_float4(O[2 * c].x, O[2 * c].y, O[2 * c + 1].x, O[2 * c + 1].y);
                *mls = make_float2(m_mine, l);
            }
            asm volatile("bar.sync 3, 256;" ::: "memory");
            const bool whole = r.t1 - r.t0 == r.T;
            const int64_t slot = (int64_t)(2 * blockIdx.x + (r.at == 0 ? 0 : 1)) * kTcRows;
            if (g == 0) {
                const float2 other = *mls;
                const float M = fmaxf(m_mine, other.x);
                const float f0 = m_mine == -INFINITY ? 0.0f : exp2f(m_mine - M), f1 = other.x == -INFINITY ? 0.0f : exp2f(other.x - M);
                const float sum = (m_mine == -INFINITY ? 0.0f : f0 * l) + (other.x == -INFINITY ? 0.0f : f1 * other.y);
                const bool seen = M != -INFINITY;
                const float inv = !whole ? 1.0f : seen ? 1.0f / sum : 0.0f;
                const float2 g0 = make_float2(f0 * inv, f0 * inv), g1 = make_float2(f1 * inv, f1 * inv);
#pragma unroll
                for (int c = 0; c < 16; ++c) {
                    const float4 w = mine[c ^ (row & 7)];
                    const float2 u = ffma2(g1, make_float2(w.x, w.y), mul2(g0, O[2 * c])), v = ffma2(g1, make_float2(w.z, w.w), mul2(g0, O[2 * c + 1]));
                    mine[c ^ (row & 7)] = make_float4(u.x, u.y, v.x, v.y);
                }
                if (real) {
                    if (!whole) *reinterpret_cast<float2*>(ta.ws_ml + (slot + row) * 2) = make_float2(M, sum);
                    else if (a.p.lse)
                        a.p.lse[((int64_t)r.s * a.p.max_q + tok) * a.p.n_q_heads + h] = seen ? (M + log2f(sum)) * 0.69314718055994531f : -INFINITY;
                }
            }
            asm volatile("bar.sync 3, 256;" ::: "memory");
#pragma unroll 4
            for (int rl = tid >> 4; rl < kTcRows; rl += 16) {  // 16 lanes a row
                const int c = tid & 15, qr = r.rt * kTcRows + rl, qt = divided(qr, a.by_G);
                if (qr >= rows) break;
                const float4 v = rows_at[rl * 16 + (c ^ (rl & 7))];
                float* dst = whole ? a.p.out + (int64_t)r.s * a.p.out_nb_seq + (int64_t)qt * a.p.out_nb_tok + (r.kvh * a.G + qr - qt * a.G) * kD
                                   : ta.ws_o + (slot + rl) * kD;
                reinterpret_cast<float4*>(dst)[c] = v;
            }
            mbar_arrive(&B->q_free[run & 1]);
        }
    } else if (warp < 12) {
        regs_down<kTcRegsProducer>();
        tc_produce<F>(ta, smem, B, tab, r, hi);
    } else {
        regs_down<kTcRegsOther>();
        // ------------------------------------------------------ MMA issuers: the whole warp walks, one lane issues
        const int which = __shfl_sync(0xffffffffu, warp, 0);
        const uint64_t dt0 = tc::sdesc_sw128(smem_addr(smem + Sh::kTiles), 16, 1024);
        constexpr uint64_t kStep = 2 * kTcTileBytes >> 4;
        bool ok = true, last = r.t0 == r.t1;
        int st = 0, buf = 0;
        uint32_t use = 0, turn = 0, n_run = 0;  // n / kTcSt, n / 3
        if (which == 12) {
            const uint32_t idesc = tc::idesc_f16_f32(128, kTcTile, false);
            const uint64_t dq0 = tc::sdesc_sw128(smem_addr(smem + Sh::kQ), 16, 1024);
            uint64_t dqh = dq0;
            for (int n = 0; !last; ++n) {
                ok = tc_wait(&B->k_full[st], use & 1, &B->err, 38);
                last = B->info[n % kTcInfos].last;
                if (ok && B->info[n % kTcInfos].starts) {
                    ok = tc_wait(&B->q_full[n_run & 1], n_run >> 1 & 1, &B->err, 43);
                    dqh = dq0 + (n_run++ & 1) * (2 * kTcTileBytes >> 4);
                }
                if (ok && n >= 3) ok = tc_wait(&B->s_free[buf], (turn - 1) & 1, &B->err, 40);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tc::fence_after();
                const uint64_t dk = dt0 + (uint64_t)st * kStep, dql = dqh + (kTcTileBytes >> 4);
                const uint32_t sp = tmem + buf * 128;
                if (elect_one()) {
#pragma unroll 1
                    for (int kk = 0; kk < 4; ++kk) tc::mma_ss(sp, dql + kk * 2, dk + kk * 2, idesc, kk > 0 ? 1u : 0u);  // small terms first
#pragma unroll 1
                    for (int kk = 0; kk < 4; ++kk) tc::mma_ss(sp, dqh + kk * 2, dk + kk * 2, idesc, 1u);
                    tc::mma_commit(&B->s_full[buf]);
                    tc::mma_commit(&B->k_empty[st]);
                }
                __syncwarp();
                if (++st == kTcSt) { st = 0; ++use; }
                if (++buf == 3) { buf = 0; ++turn; }
            }
        } else if (which == 13) {
            const uint32_t idesc = tc::idesc_f16_f32(128, 64, false);
            for (int n = 0; !last; ++n) {
                ok = tc_wait(&B->v_full[st], use & 1, &B->err, 41);
                last = B->info[n % kTcInfos].last;
                if (ok) ok = tc_wait(&B->p_full[buf], turn & 1, &B->err, 39);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tc::fence_after();
                const uint64_t dv = dt0 + (uint64_t)st * kStep + (kTcTileBytes >> 4);
                const uint32_t sp = tmem + buf * 128, ot = tmem + 384 + (n & 1) * 64;
                if (elect_one()) {
#pragma unroll 1
                    for (int kk = 0; kk < 8; ++kk)
                        tc::mma_ts(ot, sp + 32 * (kk >> 1) + 8 * (kk & 1) + 16, dv + (kk >> 2) * (kTcTileBytes >> 5) + (kk & 3) * 2, idesc, kk > 0 ? 1u : 0u);
#pragma unroll 1
                    for (int kk = 0; kk < 8; ++kk)
                        tc::mma_ts(ot, sp + 32 * (kk >> 1) + 8 * (kk & 1), dv + (kk >> 2) * (kTcTileBytes >> 5) + (kk & 3) * 2, idesc, 1u);
                    tc::mma_commit(&B->o_full[n & 1]);
                    tc::mma_commit(&B->v_empty[st]);
                    tc::mma_commit(&B->s_free[buf]);
                }
                __syncwarp();
                if (++st == kTcSt) { st = 0; ++use; }
                if (++buf == 3) { buf = 0; ++turn; }
            }
        } else if (which == 14) {
            tc_load(ta, smem, B, tab, r, hi);
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

// Join of the parts of units that several CTAs shared, and the rows that no unit holds (rows that see nothing, or past the last
// token).  16 threads per row (4 dims each) follow every kLanes-th part.
template <int kLanes>
__global__ void __launch_bounds__(256) paged_tc_combine_kernel(const __grid_constant__ TcAttArgs ta) {
    constexpr int kPer = 16 / kLanes;
    __shared__ float4 so[16][16];
    __shared__ float2 sml[16];
    const AttArgs& a = ta.a;
    griddep_wait();
    const int unit = threadIdx.x >> 4, c = threadIdx.x & 15, lane = unit % kLanes;
    const int all_rows = a.p.max_q * a.G;
    const int r = blockIdx.x * kPer + unit / kLanes, kvh = blockIdx.y, s = blockIdx.z;
    const AttLens x = att_lens(a, s, false);
    const int rt = r / kTcRows, n = ta.ws_pref[a.p.n_seq];
    int b0 = 0, c0 = 0, c1 = -1;
    if (r < x.n * a.G) {
        const int T = tc_tiles(a, x.L, x.n, rt);
        if (T > 0) {
            b0 = ta.ws_pref[s] + kvh * (T + kTcGap);
            int above = 0;  // the unit's 16 threads share the row tiles before it
            for (int i = c; i < rt; i += 16) above += tc_entries(a, x.L, x.n, i);
#pragma unroll
            for (int w = 8; w > 0; w >>= 1) above += __shfl_xor_sync(0xffffu << (threadIdx.x & 16), above, w);
            b0 += above * a.p.pool.n_heads;
            c0 = tc_owner(ta, b0, n);
            c1 = tc_owner(ta, b0 + T - 1, n);
            if (kLanes == 1 && c0 == c1) return;  // written whole
        }
    }
    const bool done = c0 == c1;
    Join j;
    for (int k0 = c0 + lane; k0 <= c1 && !done; k0 += 4 * kLanes) {
        float2 ml[4];
        float4 v[4];
        float top = j.M;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int cta = k0 + u * kLanes;
            ml[u] = make_float2(-INFINITY, 0.0f);
            const int from = tc_cut(ta, cta, n);
            if (cta <= c1 && tc_cut(ta, cta + 1, n) > from) {
                const int64_t at = (int64_t)(2 * cta + (from >= b0 - kTcGap ? 0 : 1)) * kTcRows + r % kTcRows;
                ml[u] = *reinterpret_cast<const float2*>(ta.ws_ml + at * 2);
                v[u] = *reinterpret_cast<const float4*>(ta.ws_o + at * kD + c * 4);
            }
            top = fmaxf(top, ml[u].x);
        }
        if (top == -INFINITY) continue;
        const float f0 = exp2f(j.M - top);
        j.M = top;
        j.l *= f0;
        j.o.x *= f0; j.o.y *= f0; j.o.z *= f0; j.o.w *= f0;
#pragma unroll
        for (int u = 0; u < 4; ++u) j.add(ml[u], v[u]);
    }
    if constexpr (kLanes > 1) {
        so[unit][c] = j.o;
        if (c == 0) sml[unit] = make_float2(j.M, j.l);
        __syncthreads();
        if (lane || done) return;
        j = Join();
#pragma unroll
        for (int k = 0; k < kLanes; ++k) j.M = fmaxf(j.M, sml[unit + k].x);
#pragma unroll
        for (int k = 0; k < kLanes; ++k) j.add(sml[unit + k], so[unit + k][c]);
    }
    if (r < all_rows) j.write(a, s, kvh, r, c);
}

}  // namespace paged
}  // namespace cvattn
