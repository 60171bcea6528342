// tree_mma.cuh -- tree attention on warp-level tensor-core MMAs (mma.sync
// m16n8k16, f16 operands, f32 accumulators) for f16 and block-quantized caches.
//
// The arithmetic is exact where the cache is: quants are integers, exact in f16,
// their block scales (and mins) stay aside in f32; Q is scaled per row by a power
// of two and split into f16 hi + lo; P' = p d_V 2^ev is split the same way.  Every
// product is then exact in the f32 accumulators and what is left out is below
// 2^-22 of the largest term.
//
// A CTA takes one split of one sequence, one KV head and up to 128 rows.  Its 8
// warps are WR row tiles of 16 rows x WK slices of the keys, where WR follows the
// rows that the sequence really has.  Tiles of up to 128 keys arrive by cp.async
// into a ring of raw rows; all threads then turn the tile's quants into f16 tiles
// (once, however many rows there are) and its scales into an f32 table.  An f16
// cache needs neither: its ring slots are the tiles.  A warp walks its 16-key
// steps with ldmatrix: S in registers, lazy running maximum (raised when a score
// passes it by more than 2^8, with the output rescaled), P' as the A operand of
// P.V without leaving the registers.  Adds inside the tensor cores truncate, so
// their chains are kept short: every 8 steps the output moves to f32 sums in
// shared memory.  Warps that share rows merge at the end.
// What bounds it: one sequence of 300 positions, 4 nodes, Q8_0: 10 us with the join, latency
// (two launches, a tile's way through copy, conversion, products and merge).  3 sequences of
// up to 777, 27 nodes, 16 / 16 heads, Q5_1 / Q4_1: 17.7 us for 3.5 MB, the instructions of
// conversion and softmax (1.4 a cycle and SM; DRAM and tensor cores idle).
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
constexpr int kFlush = 8;     // steps between moves of the output to its f32 sums
constexpr int kOutPad = kD + 4;
constexpr int kMaxStages = 4;
constexpr int kHalfSm = 112 * 1024;  // shared memory of a CTA when two share an SM
constexpr float kLazy = 8.0f;
// The least scale d_V 2^ev of a drafted value that goes through f16: what hi + lo leave out of P' is then below 2^-19 of a
// weight of 1.  (ev brings the largest scale of a first tile to [2^4, 2^5), so ordinary drafts lie well above.)
constexpr float kLeastScale = 1.0f / 64.0f;

struct Shape {
    int row_groups;    // CTAs along the rows, 128 rows each
    int stages;        // ring slots
};

// Bytes between the keys of a raw tile: an odd number of words, so that the 32 keys that a warp converts lie in
// different banks; f16 rows are tiles already.
__host__ __device__ constexpr int raw_stride(int t) {
    return t == kF16 ? 2 * kD : ((2 * group_bytes(t) / 4) | 1) * 4;
}

struct Smem {
    int maxv, tab, out, ml, kf, vf, ring, k_bytes, stage, total;
    __host__ __device__ Smem(int kt, int vt, int stages) {
        int o = 0;
        maxv = o; o += 32;
        tab = o;
        const bool km = kt == kQ4_1 || kt == kQ5_1, vm = vt == kQ4_1 || vt == kQ5_1;
        o += ((kt == kF16 ? 0 : 2) + (km ? 2 : 0) + (vt == kF16 ? 0 : 2) + (vm ? 2 : 0)) * kKeys * 4;
        out = o; o += kWarps * 16 * kOutPad * 4;  // f32 sums of the warps' outputs
        ml = o; o += kWarps * 16 * 8;
        o = (o + 127) / 128 * 128;
        kf = o; o += kt == kF16 ? 0 : kKeys * 2 * kD;
        vf = o; o += vt == kF16 ? 0 : kKeys * 2 * kD;
        ring = o;
        k_bytes = (kKeys * raw_stride(kt) + 127) / 128 * 128;
        stage = k_bytes + (kKeys * raw_stride(vt) + 127) / 128 * 128;
        o += stages * stage;
        total = o;
    }
};

__device__ __forceinline__ void cp_async4(void* dst, const void* src, bool real) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_addr(dst)), "l"(src), "r"(real ? 4 : 0) : "memory");
}
__device__ __forceinline__ void cp_async16(void* dst, const void* src, bool real) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_addr(dst)), "l"(src), "r"(real ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
// The same product into a fresh accumulator.
__device__ __forceinline__ void mma16816_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}

// Copies of one tensor's raw tiles: each thread has its own 16-, 4- or 2-byte column of a row and every per-th key.
template <int T>
struct Fetch {
    int unit, key0, col, per;
    __device__ __forceinline__ Fetch(const uint8_t* base, int64_t nb1) {
        const uint64_t x = reinterpret_cast<uint64_t>(base) | (uint64_t)nb1;
        unit = T == kF16 && (x & 15) == 0 ? 16 : (x & 3) == 0 ? 4 : 2;
        const int w = 2 * group_bytes(T) / unit;
        per = kWarps * 32 / w;
        key0 = threadIdx.x / w;
        col = (threadIdx.x - key0 * w) * unit;
        if (key0 >= per) key0 = 1 << 20;
    }
    // Keys [0, count) of the tile at src, and zeros up to the next multiple of 16.
    __device__ __forceinline__ void operator()(uint8_t* dst, const uint8_t* src, int64_t nb1, int count) const {
        const int end = (count + kSub - 1) & ~(kSub - 1);
        const uint8_t* s = src + (int64_t)key0 * nb1 + col;
        const int64_t ds = (int64_t)per * nb1;
        for (int key = key0; key < end; key += per, s += ds) {
            const bool real = key < count;
            const uint8_t* from = real ? s : src;
            int at = col;
            if constexpr (T == kF16) at ^= (key & 7) << 4;
            uint8_t* d = dst + key * raw_stride(T) + at;
            if (unit == 16) cp_async16(d, from, real);
            else if (unit == 4) cp_async4(d, from, real);
            else *reinterpret_cast<uint16_t*>(d) = real ? *reinterpret_cast<const uint16_t*>(from) : (uint16_t)0;
        }
    }
};

// 32 values of one key into its row of an f16 tile (128-byte rows, 16-byte chunks XORed with the key mod 8).
__device__ __forceinline__ void store_block(uint8_t* tile, int key, int blk, const uint32_t (&w)[16]) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
        *reinterpret_cast<uint4*>(tile + key * 128 + (((4 * blk + i) ^ (key & 7)) << 4)) =
            make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
}

// Block BLK of a head's raw slice, which starts at a multiple of 4 bytes (so the quants' alignment is known).
template <int T, int BLK>
__device__ __forceinline__ void convert_block(const uint8_t* slice, uint32_t (&w)[16], float& d, float& m) {
    dtc::convert_group<T>(static_cast<const uint8_t*>(__builtin_assume_aligned(slice, 4)) + BLK * group_bytes(T), w, d, m);
}

__device__ __forceinline__ bool f16x2_special(uint32_t w) {
    return (w & 0x7C00u) == 0x7C00u || (w & 0x7C000000u) == 0x7C000000u;
}

template <int KT, int VT>
__global__ void __launch_bounds__(kWarps * 32, 2) tree_mma_kernel(const __grid_constant__ Args a, const Shape sh) {
    extern __shared__ __align__(128) uint8_t smem[];
    constexpr int sliceK = 2 * group_bytes(KT), sliceV = 2 * group_bytes(VT);  // bytes of the head in a row
    constexpr bool K_Q = KT != kF16, V_Q = VT != kF16;
    constexpr bool K_MIN = BlockTraits<KT>::HAS_MIN, V_MIN = BlockTraits<VT>::HAS_MIN;
    constexpr float kOffs = V_Q ? 0.0f : 7.0f;  // f16 V: P is kept 2^7 larger, far from f16's subnormals
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gid = lane >> 2, tig = lane & 3;
    const int s = blockIdx.z, split = blockIdx.x;
    const int kvh = blockIdx.y % a.Hkv, r0 = blockIdx.y / a.Hkv * (16 * kWarps);
    griddep_wait();
    const Lens x = lens_of(a, s, tid == 0 && blockIdx.x == 0 && blockIdx.y == 0);
    const int rows = x.n * a.G, all_rows = a.max_nodes * a.G;
    const int tile0 = split * a.split_tiles, tile1 = min(x.tiles, tile0 + a.split_tiles);
    const bool direct = a.n_splits == 1;
    if (!direct && (tile0 >= tile1 || r0 >= rows)) return;
    const Smem L(KT, VT, sh.stages);
    const uint8_t* kb = seq_base(a.k_seq_ptrs, a.k, a.k_nb2, s) + kvh * sliceK;
    const uint8_t* vb = seq_base(a.v_seq_ptrs, a.v, a.v_nb2, s) + kvh * sliceV;
    const uint8_t* kdb = a.kd ? a.kd + (int64_t)s * a.kd_nb2 + kvh * sliceK : nullptr;
    const uint8_t* vdb = a.vd ? a.vd + (int64_t)s * a.vd_nb2 + kvh * sliceV : nullptr;
    const Fetch<KT> fetch_k(kb, a.k_nb1);
    const Fetch<VT> fetch_v(vb, a.v_nb1);

    const int n_local = r0 < rows ? max(0, tile1 - tile0) : 0;
    auto issue = [&](int t, int slot) {  // tile tile0 + t into a ring slot
        if (t < n_local) {
            const int tile = tile0 + t;
            const bool draft = tile >= x.cache_tiles;
            const int p0 = (draft ? tile - x.cache_tiles : tile) * a.tile;
            const int count = min(a.tile, (draft ? x.n : x.L) - p0);
            uint8_t* d = smem + L.ring + slot * L.stage;
            if (!draft) {
                fetch_k(d, kb + (int64_t)p0 * a.k_nb1, a.k_nb1, count);
                fetch_v(d + L.k_bytes, vb + (int64_t)p0 * a.v_nb1, a.v_nb1, count);
            } else {
                Fetch<KT>(kdb, a.kd_nb1)(d, kdb + (int64_t)p0 * a.kd_nb1, a.kd_nb1, count);
                Fetch<VT>(vdb, a.vd_nb1)(d + L.k_bytes, vdb + (int64_t)p0 * a.vd_nb1, a.vd_nb1, count);
            }
        }
        cp_async_commit();
    };
    for (int t = 0; t < sh.stages - 1; ++t) issue(t, t);

    // this warp: row tile wr of WR, key steps wk, wk + WK, ..
    const int row_tiles = (min(rows - r0, 16 * kWarps) + 15) / 16;
    const int wr_all = row_tiles <= 1 ? 1 : row_tiles <= 2 ? 2 : row_tiles <= 4 ? 4 : 8, wk_all = kWarps / wr_all;
    const int wr = warp % wr_all, wk = warp / wr_all;
    const int rw = r0 + wr * 16;    // its first row
    const bool idle = rw >= rows;
    uint32_t qa[4][2][4];           // A fragments of Q: [k-step][hi, lo]
    float rs[2], qs0[2], qs1[2];    // score factor, sums of Q over the two blocks (rows gid, gid + 8)
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const int r = rw + half * 8 + gid;
        const float* q = a.q + (int64_t)s * a.q_nb_seq + (int64_t)(r / a.G) * a.q_nb_node + (kvh * a.G + r % a.G) * kD + 2 * tig;
        float2 e[8];  // dims 8 i + 2 tig, + 1
        float am = 0.0f, sum[2] = {0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            e[i] = r < rows ? *reinterpret_cast<const float2*>(q + 8 * i) : make_float2(0.f, 0.f);
            am = fmaxf(am, fmaxf(fabsf(e[i].x), fabsf(e[i].y)));
            sum[i >> 2] += e[i].x + e[i].y;
        }
        const int ex = dtc::norm_exp(quad_max(am));
        const float sc = pow2f(ex);
        rs[half] = pow2f(-ex) * a.scale_log2;
        qs0[half] = K_MIN ? quad_sum(sum[0]) * a.scale_log2 : 0.0f;
        qs1[half] = K_MIN ? quad_sum(sum[1]) * a.scale_log2 : 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) split2(e[i].x * sc, e[i].y * sc, qa[i >> 1][0][2 * (i & 1) + half], qa[i >> 1][1][2 * (i & 1) + half]);
    }
    float O[8][4], base[2], thr[2], l[2], om[2][2], cum[2];
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) O[j][i] = 0.0f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        base[h] = 0.0f;
        thr[h] = -INFINITY;  // nothing seen: any score raises the reference
        l[h] = 0.0f;
        om[h][0] = om[h][1] = 0.0f;
        cum[h] = 0.0f;       // what the sums in shared memory still have to be multiplied by (none there yet)
    }
    int since = 0;           // steps since the output moved there
    float* sum_row = reinterpret_cast<float*>(smem + L.out) + (warp * 16 + gid) * kOutPad + 2 * tig;
    // sums = sums * cum + O, in the fragments' own order: tile j, columns 2 tig, 2 tig + 1 of rows gid and gid + 8
    auto flush = [&]() {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float* p = sum_row + h * 8 * kOutPad;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                float2 v = make_float2(O[j][2 * h], O[j][2 * h + 1]);
                if (cum[h] != 0.0f) {
                    const float2 w = *reinterpret_cast<const float2*>(p + 8 * j);
                    v.x = fmaf(w.x, cum[h], v.x);
                    v.y = fmaf(w.y, cum[h], v.y);
                }
                *reinterpret_cast<float2*>(p + 8 * j) = v;
                O[j][2 * h] = O[j][2 * h + 1] = 0.0f;
            }
            cum[h] = 1.0f;
        }
        since = 0;
    };
    if (tid < 8) reinterpret_cast<uint32_t*>(smem + L.maxv)[tid] = 0u;
    __syncthreads();

    int ev = 0;
    bool ev_set = false;

    // tables of this tile: [K scale, K min, V scale, V min][block][key]
    float* th = reinterpret_cast<float*>(smem + L.tab);
    constexpr int oKm = K_Q ? 2 * kKeys : 0, oV = oKm + (K_MIN ? 2 * kKeys : 0), oVm = oV + (V_Q ? 2 * kKeys : 0);
    uint32_t* maxv = reinterpret_cast<uint32_t*>(smem + L.maxv);
    const uint32_t lrow = lane & 7, lmat = lane >> 3;  // ldmatrix: this lane's row of its matrix

    int slot = 0, free_slot = sh.stages - 1;  // of tile t, and of the tile before it, which every warp has left
    for (int t = 0; t < n_local; ++t) {
        if (sh.stages == 4) cp_async_wait<2>();
        else if (sh.stages == 3) cp_async_wait<1>();
        else cp_async_wait<0>();
        __syncthreads();
        issue(t + sh.stages - 1, free_slot);
        uint8_t* kraw = smem + L.ring + slot * L.stage;
        uint8_t* vraw = kraw + L.k_bytes;
        free_slot = slot;
        slot = slot + 1 == sh.stages ? 0 : slot + 1;
        const int tile = tile0 + t;
        const bool draft = tile >= x.cache_tiles;
        const int p0 = (draft ? tile - x.cache_tiles : tile) * a.tile;
        const int count = min(a.tile, (draft ? x.n : x.L) - p0);
        if constexpr (K_Q || V_Q) {
            const int blk = warp & 1, key = (warp >> 1) * 32 + lane;  // 32 keys of one block per warp
            if ((warp >> 1) * 32 < count) {  // (keys up to a multiple of 16 are there, later ones are not used)
                if constexpr (K_Q) {
                    uint32_t w[16];
                    float d, m;
                    dtc::convert_group<KT>(kraw + key * raw_stride(KT) + blk * group_bytes(KT), w, d, m);
                    store_block(smem + L.kf, key, blk, w);
                    th[blk * kKeys + key] = d;
                    if constexpr (K_MIN) th[oKm + blk * kKeys + key] = m;
                }
                if constexpr (V_Q) {
                    uint32_t w[16];
                    float d, m;
                    dtc::convert_group<VT>(vraw + key * raw_stride(VT) + blk * group_bytes(VT), w, d, m);
                    store_block(smem + L.vf, key, blk, w);
                    th[oV + blk * kKeys + key] = d;
                    if constexpr (V_MIN) th[oVm + blk * kKeys + key] = m;
                    const uint32_t mx = __reduce_max_sync(0xffffffffu, key < count && isfinite(d) ? __float_as_uint(fabsf(d)) : 0u);
                    if (lane == 0 && mx) atomicMax(&maxv[t & 1], mx);
                }
            }
            __syncthreads();
            if (tid == 0) maxv[(t + 1) & 1] = 0u;
        }
        if (idle) continue;
        float vf = 1.0f;  // 2^ev
        if constexpr (V_Q) {
            const float mv = __uint_as_float(maxv[t & 1]);
            if (mv > 0.0f) {
                const int now = ev_set ? dstream::ilog2f(mv) + ev : 0;
                if (!ev_set || now < dmma::kEvMin || now > dmma::kEvMax) {
                    const int evn = dstream::v_exp_target(mv);
                    if (ev_set) {
                        const float f = pow2f(evn - ev);
                        cum[0] *= f;
                        cum[1] *= f;
#pragma unroll
                        for (int j = 0; j < 8; ++j)
#pragma unroll
                            for (int i = 0; i < 4; ++i) O[j][i] *= f;
                    }
                    ev = evn;
                    ev_set = true;
                }
            }
            vf = pow2f(ev);
        }
        const uint32_t kt = smem_addr(K_Q ? smem + L.kf : kraw), vt = smem_addr(V_Q ? smem + L.vf : vraw);
        const int steps = (count + kSub - 1) / kSub;
#pragma unroll 1
        for (int sub = wk; sub < steps; sub += wk_all) {
            float sc[2][4];  // [8-key tile][row gid: 2 keys, row gid + 8: 2 keys]
            {
                float acc[K_Q ? 2 : 1][2][4];
#pragma unroll
                for (int tt = 0; tt < 2; ++tt) {
                    // matrices: dims 8 c .. 8 c + 7 of 8 keys, four chunks c at a time
                    const uint32_t krow = kt + (kSub * sub + 8 * tt + lrow) * 128;
                    constexpr int b1 = K_Q ? 1 : 0;
                    uint32_t r[4];
                    ldsm4(r, krow + ((lmat ^ lrow) << 4));
                    // small terms first, while the sums are small: adds inside the tensor cores truncate
                    mma16816_first(acc[0][tt], qa[0][1], r[0], r[1]);
                    mma16816(acc[0][tt], qa[1][1], r[2], r[3]);
                    if constexpr (K_Q) {
                        mma16816(acc[0][tt], qa[0][0], r[0], r[1]);
                        mma16816(acc[0][tt], qa[1][0], r[2], r[3]);
                        ldsm4(r, krow + (((4 + lmat) ^ lrow) << 4));
                        mma16816_first(acc[b1][tt], qa[2][1], r[0], r[1]);
                        mma16816(acc[b1][tt], qa[3][1], r[2], r[3]);
                        mma16816(acc[b1][tt], qa[2][0], r[0], r[1]);
                        mma16816(acc[b1][tt], qa[3][0], r[2], r[3]);
                    } else {
                        uint32_t u[4];
                        ldsm4(u, krow + (((4 + lmat) ^ lrow) << 4));
                        mma16816(acc[0][tt], qa[2][1], u[0], u[1]);
                        mma16816(acc[0][tt], qa[3][1], u[2], u[3]);
                        mma16816(acc[0][tt], qa[0][0], r[0], r[1]);
                        mma16816(acc[0][tt], qa[1][0], r[2], r[3]);
                        mma16816(acc[0][tt], qa[2][0], u[0], u[1]);
                        mma16816(acc[0][tt], qa[3][0], u[2], u[3]);
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
                        for (int i = 0; i < 4; ++i) {
                            const int h = i >> 1;
                            const float e0 = (i & 1) ? d0.y : d0.x, e1 = (i & 1) ? d1.y : d1.x;
                            const float v = fmaf(acc[0][tt][i], e0, acc[1][tt][i] * e1);
                            float off = -base[h];
                            if constexpr (K_MIN)
                                off = fmaf((i & 1) ? m0.y : m0.x, qs0[h], fmaf((i & 1) ? m1.y : m1.x, qs1[h], off));
                            sc[tt][i] = fmaf(v, rs[h], off);
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i) sc[tt][i] = fmaf(acc[0][tt][i], rs[i >> 1], -base[i >> 1]);
                    }
                }
            }
            const bool masked = draft || count - sub * kSub < kSub;  // some (row, key) of the step may be unseen
            if (masked) {
                const int j0 = p0 + kSub * sub, left = count - kSub * sub;  // keys of this step that exist
                const uint32_t exist = left >= kSub ? 0xffffu : (1u << left) - 1u;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int r = rw + h * 8 + gid;
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
                            if (!((bits >> (8 * tt + 2 * tig + e)) & 1u)) sc[tt][2 * h + e] = -INFINITY;
                }
            }
            float mx[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) mx[h] = fmaxf(fmaxf(sc[0][2 * h], sc[0][2 * h + 1]), fmaxf(sc[1][2 * h], sc[1][2 * h + 1]));
            if (__any_sync(0xffffffffu, mx[0] > thr[0] || mx[1] > thr[1])) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float top = quad_max(mx[h]);
                    if (top > thr[h]) {
                        const float up = top - kOffs;
                        const float f = thr[h] == -INFINITY ? 0.0f : fast_exp2(-up);
                        base[h] += up;
                        thr[h] = kLazy + kOffs;
                        l[h] *= f;
                        cum[h] *= f;
                        om[h][0] *= f;
                        om[h][1] *= f;
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            O[j][2 * h] *= f;
                            O[j][2 * h + 1] *= f;
                        }
#pragma unroll
                        for (int tt = 0; tt < 2; ++tt) {
                            sc[tt][2 * h] -= up;
                            sc[tt][2 * h + 1] -= up;
                        }
                    }
                }
            }
#pragma unroll
            for (int tt = 0; tt < 2; ++tt)
#pragma unroll
                for (int i = 0; i < 4; ++i) sc[tt][i] = fast_exp2(sc[tt][i]);
#pragma unroll
            for (int h = 0; h < 2; ++h) l[h] += (sc[0][2 * h] + sc[0][2 * h + 1]) + (sc[1][2 * h] + sc[1][2 * h + 1]);
            float2 dv[2][2], vm[2][2];  // [block][8-key tile]
            if constexpr (V_Q) {
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int tt = 0; tt < 2; ++tt) {
                        const float* tv = th + b * kKeys + kSub * sub + 8 * tt + 2 * tig;
                        dv[b][tt] = *reinterpret_cast<const float2*>(tv + oV);
                        dv[b][tt].x *= vf;
                        dv[b][tt].y *= vf;
                        vm[b][tt] = make_float2(0.f, 0.f);
                        if constexpr (V_MIN) vm[b][tt] = *reinterpret_cast<const float2*>(tv + oVm);
                    }
            }
            if (draft) {
                // Drafts hold anything where no row may look: a step whose values are not all finite, or lie so far below the
                // largest of the tile (which a row may not see) that P' would leave f16's normal numbers, is added up key by
                // key, and keys that a row does not see are left out instead of being multiplied by zero.
                bool special = false;
                if constexpr (V_Q) {
#pragma unroll
                    for (int b = 0; b < 2; ++b)
#pragma unroll
                        for (int tt = 0; tt < 2; ++tt) {
                            special |= !isfinite(dv[b][tt].x) || !isfinite(dv[b][tt].y);
                            special |= !isfinite(vm[b][tt].x) || !isfinite(vm[b][tt].y);
                            special |= dv[b][tt].x != 0.0f && fabsf(dv[b][tt].x) < kLeastScale;
                            special |= dv[b][tt].y != 0.0f && fabsf(dv[b][tt].y) < kLeastScale;
                        }
                } else {
#pragma unroll 1
                    for (int k = 0; k < 4; ++k) {
                        const uint4 w = *reinterpret_cast<const uint4*>(vraw + (kSub * sub + 4 * k) * 128 + lane * 16);  // 4 keys
                        special |= f16x2_special(w.x) || f16x2_special(w.y) || f16x2_special(w.z) || f16x2_special(w.w);
                    }
                }
                if (__any_sync(0xffffffffu, special)) {
#pragma unroll 1
                    for (int k = 0; k < kSub; ++k) {
                        const int key = kSub * sub + k, src = (lane & ~3) | ((k & 7) >> 1);
                        const float ca = k & 8 ? (k & 1 ? sc[1][1] : sc[1][0]) : (k & 1 ? sc[0][1] : sc[0][0]);
                        const float cb = k & 8 ? (k & 1 ? sc[1][3] : sc[1][2]) : (k & 1 ? sc[0][3] : sc[0][2]);
                        const float pa = __shfl_sync(0xffffffffu, ca, src), pb = __shfl_sync(0xffffffffu, cb, src);
#pragma unroll
                        for (int j = 0; j < 8; ++j)
#pragma unroll
                            for (int c = 0; c < 2; ++c) {
                                const int d = 8 * j + 2 * tig + c;
                                float v;
                                if constexpr (VT == kF16)
                                    v = h2f(*reinterpret_cast<const uint16_t*>(vraw + key * 128 + ((2 * d) ^ ((key & 7) << 4))));
                                else
                                    v = dequant_elem<VT>(vraw + key * raw_stride(VT) + (d >> 5) * group_bytes(VT), d & 31);
                                if (pa != 0.0f) O[j][c] = fmaf(pa * vf, v, O[j][c]);
                                if (pb != 0.0f) O[j][2 + c] = fmaf(pb * vf, v, O[j][2 + c]);
                            }
                    }
                    continue;
                }
            }
            // V: matrices (keys 0-7, chunk c), (8-15, c), (0-7, c + 1), (8-15, c + 1) give two dim tiles
            const uint32_t vrow = vt + (kSub * sub + 8 * (lmat & 1) + lrow) * 128;
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                if constexpr (V_Q) {
                    if constexpr (V_MIN) {
#pragma unroll
                        for (int tt = 0; tt < 2; ++tt)
#pragma unroll
                            for (int h = 0; h < 2; ++h)
                                om[h][b] = fmaf(sc[tt][2 * h], vm[b][tt].x, fmaf(sc[tt][2 * h + 1], vm[b][tt].y, om[h][b]));
                    }
#pragma unroll
                    for (int tt = 0; tt < 2; ++tt)
#pragma unroll
                        for (int h = 0; h < 2; ++h)
                            split2(sc[tt][2 * h] * dv[b][tt].x, sc[tt][2 * h + 1] * dv[b][tt].y, hi[2 * tt + h], lo[2 * tt + h]);
                } else if (b == 0) {
#pragma unroll
                    for (int tt = 0; tt < 2; ++tt)
#pragma unroll
                        for (int h = 0; h < 2; ++h) split2(sc[tt][2 * h], sc[tt][2 * h + 1], hi[2 * tt + h], lo[2 * tt + h]);
                }
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    uint32_t r[4];
                    ldsm4t(r, vrow + (((4 * b + 2 * u + (lmat >> 1)) ^ lrow) << 4));
                    const int j = 4 * b + 2 * u;
                    mma16816(O[j], lo, r[0], r[1]);
                    mma16816(O[j + 1], lo, r[2], r[3]);
                    mma16816(O[j], hi, r[0], r[1]);
                    mma16816(O[j + 1], hi, r[2], r[3]);
                }
            }
            if (++since == kFlush) flush();
        }
    }
    flush();
    griddep_launch_dependents();

    // the warps' rows as (max, sum) and f32 sums, joined over the WK slices
    float2* ml = reinterpret_cast<float2*>(smem + L.ml);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const float ls = quad_sum(l[h]);
        const float uf = V_Q ? pow2f(-ev) : 1.0f;
        float o0 = 0.0f, o1 = 0.0f;
        if constexpr (V_MIN) {
            o0 = quad_sum(om[h][0]);
            o1 = quad_sum(om[h][1]);
        }
        if constexpr (V_Q) {
            float* p = sum_row + h * 8 * kOutPad;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                p[8 * j] = fmaf(p[8 * j], uf, j < 4 ? o0 : o1);
                p[8 * j + 1] = fmaf(p[8 * j + 1], uf, j < 4 ? o0 : o1);
            }
        }
        // (a row whose scores are all NaN raises nothing, but was seen)
        if (tig == 0) ml[warp * 16 + h * 8 + gid] = make_float2(thr[h] == -INFINITY && ls == 0.0f ? -INFINITY : base[h], ls);
    }
    __syncthreads();
    const float* ob = reinterpret_cast<const float*>(smem + L.out);
    const int rows_here = min((direct ? all_rows : rows) - r0, 16 * kWarps);
    for (int i = tid; i < rows_here * 16; i += kWarps * 32) {
        const int c = i & 15, rl = i >> 4, r = r0 + rl;
        const int w0 = rl >> 4, in = rl & 15;  // slice k: warp w0 + k * WR
        const bool real = r < rows;
        float M = -INFINITY;
        for (int k = 0; real && k < wk_all; ++k) M = fmaxf(M, ml[(w0 + k * wr_all) * 16 + in].x);
        float sum = 0.0f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        if (M != -INFINITY)
            for (int k = 0; k < wk_all; ++k) {
                const int row = (w0 + k * wr_all) * 16 + in;
                const float2 e = ml[row];
                if (e.x == -INFINITY) continue;
                const float f = exp2f(e.x - M);
                const float4 v = *reinterpret_cast<const float4*>(ob + row * kOutPad + 4 * c);
                sum = fmaf(f, e.y, sum);
                o.x = fmaf(f, v.x, o.x); o.y = fmaf(f, v.y, o.y); o.z = fmaf(f, v.z, o.z); o.w = fmaf(f, v.w, o.w);
            }
        if (direct) {
            const bool seen = M != -INFINITY;
            const float inv = seen ? 1.0f / sum : 0.0f;
            const int node = r / a.G, h = kvh * a.G + r % a.G;
            *reinterpret_cast<float4*>(a.out + (int64_t)s * a.out_nb_seq + (int64_t)node * a.out_nb_node + h * kD + c * 4) =
                make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
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
template <int KT> cudaError_t launch_mma_for_k(cudaStream_t stream, const Args& a, const Shape& sh);

}  // namespace tree
}  // namespace cvattn
