// paged_append.cu -- rows rounded into the pages of an 8-bit cache, and read back.
#include "launch.cuh"
#include "paged.cuh"

namespace cvattn {
namespace paged {

// A warp takes one block of one head, keys or values: 16 x 64 f32 values, 32 a lane, in the order in which it writes their
// codes.  Every block has one writer, so rows that the block held are read, rounded anew and written in place.
// Bound by latency and instructions: 16 sequences of up to 1500 rows of 2 heads, 13.4 MB of f32 to 3.4 MB, 7.6 us, and read back
// 5.6 (3 TB/s); a warp a row took 16.7 and 12.4.  One token for 64 sequences: 4.2 us, a launch and three dependent loads (length,
// page, the block's old scale).
constexpr int kAppendWarps = 4;

// Value (of 32) e of a lane: position and dim, in the order of the block's bytes (four of them a word).
template <bool V> __device__ __forceinline__ int t_of(int lane, int e) { return V ? (lane & 3) * 4 + (e & 3) : 2 * (e >> 2) + (lane >> 4); }
template <bool V> __device__ __forceinline__ int d_of(int lane, int e) {
    return V ? (e >> 4) * 32 + ((e >> 2) & 3) * 8 + (lane >> 2) : (lane & 15) * 4 + (e & 3);
}
// Byte of word w (of 8) of a lane.
template <bool V> __device__ __forceinline__ int word_at(int lane, int w) {
    return V ? (w >> 2) * 512 + lane * 16 + (w & 3) * 4 : w * 128 + lane * 4;
}

// Four codes of x / scale (inv: 1 / scale in f32), finite values whose quotients the format holds; where one of them is next to a
// border between two codes, `near` is set.
template <int F> __device__ __forceinline__ uint32_t four_codes(const float* x, float inv, bool& near) {
    constexpr float lo = 1.0f - 0x1p-21f, hi = 1.0f + 0x1p-21f;
    uint32_t a[4], b[4];
    if constexpr (F == kI8) {
        constexpr float magic = 12582912.0f + 128.0f;  // 1.5 * 2^23: the sum has the nearest integer, ties to even, in its low bits
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float y = x[i] * inv;
            a[i] = __float_as_uint(fmaf(y, lo, magic));
            b[i] = __float_as_uint(fmaf(y, hi, magic));
        }
        const uint32_t u = __byte_perm(__byte_perm(a[0], a[1], 0x0040), __byte_perm(a[2], a[3], 0x0040), 0x5410);
        const uint32_t v = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
        near |= u != v;
        return u;
    } else {
        uint16_t u[2], v[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float y0 = x[2 * i] * inv, y1 = x[2 * i + 1] * inv;
            asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(u[i]) : "f"(y1 * lo), "f"(y0 * lo));
            asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(v[i]) : "f"(y1 * hi), "f"(y0 * hi));
        }
        const uint32_t p = u[0] | (uint32_t)u[1] << 16, q = v[0] | (uint32_t)v[1] << 16;
        near |= p != q;
        return p;
    }
}

// Any value's code.
template <int F> __device__ __noinline__ uint32_t any_code(float v, float inv, float scale) {
    if (isnan(v) || scale == 0.0f) return F == kI8 ? 128u : 0u;
    return nearest_code<F>(v * inv, v, scale);
}
// A code under a larger scale.
template <int F> __device__ __noinline__ uint32_t code_again(uint32_t old, float was, float shrink, float scale) {
    const float v = code_value<F>(old);
    return nearest_code<F>(v * shrink, (double)v * was, scale);
}

template <int F, bool V>
__device__ __forceinline__ void append_block(const cvattn_paged_append_params& p, const float* src, int page, int in, int t0, int t1, int lane) {
    uint8_t* codes = static_cast<uint8_t*>(V ? p.pool.v : p.pool.k) + page * p.pool.nb_page + (int64_t)in * kBlockBytes;
    float* scale_at = (V ? p.pool.v_scale : p.pool.k_scale) + page * p.pool.nb_scale + in;
    float x[32];
    if constexpr (V) {
#pragma unroll
        for (int e = 0; e < 32; ++e) {
            const int t = t_of<V>(lane, e);
            x[e] = t >= t0 && t < t1 ? src[t * p.nb_row + d_of<V>(lane, e)] : 0.0f;
        }
    } else {
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
            const int t = t_of<V>(lane, e);
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            if (t >= t0 && t < t1) v = *reinterpret_cast<const float4*>(src + t * p.nb_row + d_of<V>(lane, e));
            x[e] = v.x;
            x[e + 1] = v.y;
            x[e + 2] = v.z;
            x[e + 3] = v.w;
        }
    }
    const float was = t0 > 0 ? fmaxf(*scale_at, 0.0f) : 0.0f;  // (NaN: 0)
    uint32_t old[8] = {};
    const bool partial = t0 > 0 || t1 < kBlock;
    if (partial) {
#pragma unroll
        for (int w = 0; w < 8; ++w) old[w] = *reinterpret_cast<const uint32_t*>(codes + word_at<V>(lane, w));
    }
    float amax = 0.0f;
    bool odd = false;  // values that are not finite
#pragma unroll
    for (int e = 0; e < 32; ++e) {
        const float a = fabsf(x[e]);
        odd |= !(a < INFINITY);
        if (a < INFINITY) amax = fmaxf(amax, a);
    }
    amax = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(amax)));
    const float scale = fmaxf(was, scale_of<F>(amax));
    const bool grows = t0 > 0 && scale > was;
    const float inv = scale > 0.0f ? __fdiv_rn(1.0f, scale) : 0.0f;
    const float shrink = grows ? __fdiv_rn(was, scale) : 1.0f;
    __syncwarp();
    if (lane == 0) *scale_at = scale;
    odd |= scale == 0.0f;
#pragma unroll
    for (int w = 0; w < 8; ++w) {
        bool slow = odd;
        uint32_t word = four_codes<F>(x + 4 * w, inv, slow);
        if (slow) {
            word = 0;
#pragma unroll
            for (int c = 0; c < 4; ++c) word |= any_code<F>(x[4 * w + c], inv, scale) << (8 * c);
        }
        if (partial) {
            uint32_t mine = 0;  // bytes of new rows
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int t = t_of<V>(lane, 4 * w + c);
                if (t >= t0 && t < t1) mine |= 0xffu << (8 * c);
                if (t < t0 && grows) {
                    mine |= 0xffu << (8 * c);
                    word = (word & ~(0xffu << (8 * c))) | code_again<F>(old[w] >> (8 * c) & 0xffu, was, shrink, scale) << (8 * c);
                }
            }
            if (mine == 0) continue;
            word = (word & mine) | (old[w] & ~mine);
        }
        *reinterpret_cast<uint32_t*>(codes + word_at<V>(lane, w)) = word;
    }
}

template <int F>
__global__ void __launch_bounds__(kAppendWarps * 32) paged_append_kernel(const __grid_constant__ cvattn_paged_append_params p, int* status) {
    griddep_wait();
    const int lane = threadIdx.x & 31, s = blockIdx.y;
    const int per = 2 * p.pool.n_heads;
    const int unit = blockIdx.x * kAppendWarps + (threadIdx.x >> 5);
    const int L = p.kv_len[s], n = p.n_new ? p.n_new[s] : p.max_new;
    const int64_t room = (int64_t)p.table_width * p.pool.page_size;
    if (L < 0 || n < 0 || n > p.max_new || (int64_t)L + n > room) {
        if (threadIdx.x == 0 && blockIdx.x == 0) record_status(status, kStatusBadLength);
        return;
    }
    const int b = L / kBlock + unit / per;  // block of the sequence
    if (n == 0 || (int64_t)b * kBlock >= (int64_t)L + n) return;
    const int part = unit % per, head = part >> 1;
    const int blocks = p.pool.page_size / kBlock;
    const int page = page_of(p.table + s * p.table_nb_seq, b / blocks, p.pool.n_pages);
    if (page < 0 || (p.refs && p.refs[page] > 1)) {
        if (lane == 0) record_status(status, page < 0 ? kStatusBadPage : kStatusSharedPage);
        return;
    }
    const int in = head * blocks + b % blocks;
    const int t0 = max(0, L - b * kBlock), t1 = min(kBlock, L + n - b * kBlock);  // the new positions
    const int64_t at = s * p.nb_seq + (int64_t)(b * kBlock - L) * p.nb_row + head * kD;
    if (part & 1) append_block<F, true>(p, p.v + at, page, in, t0, t1, lane);
    else append_block<F, false>(p, p.k + at, page, in, t0, t1, lane);
}

// A warp takes one block of one head, keys or values.
template <int F, bool V>
__device__ __forceinline__ void read_block(const cvattn_paged_read_params& p, float* dst, int page, int in, int t0, int t1, int t2, int lane) {
    uint32_t codes[8] = {};
    float scale = 0.0f;
    if (page >= 0) {
        const uint8_t* from = static_cast<const uint8_t*>(V ? p.pool.v : p.pool.k) + page * p.pool.nb_page + (int64_t)in * kBlockBytes;
        scale = ((V ? p.pool.v_scale : p.pool.k_scale) + page * p.pool.nb_scale)[in];
#pragma unroll
        for (int w = 0; w < 8; ++w) codes[w] = *reinterpret_cast<const uint32_t*>(from + word_at<V>(lane, w));
    }
#pragma unroll
    for (int w = 0; w < 8; ++w) {
        float x[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const int t = t_of<V>(lane, 4 * w + c);
            x[c] = page >= 0 && t < t1 ? code_value<F>(codes[w] >> (8 * c) & 0xffu) * scale : 0.0f;
            if (V && t >= t0 && t < t2) dst[t * p.nb_row + d_of<V>(lane, 4 * w + c)] = x[c];
        }
        const int t = t_of<V>(lane, 4 * w);
        if (!V && t >= t0 && t < t2) *reinterpret_cast<float4*>(dst + t * p.nb_row + d_of<V>(lane, 4 * w)) = make_float4(x[0], x[1], x[2], x[3]);
    }
}

template <int F>
__global__ void __launch_bounds__(kAppendWarps * 32) paged_read_kernel(const __grid_constant__ cvattn_paged_read_params p, int* status) {
    griddep_wait();
    const int lane = threadIdx.x & 31, s = blockIdx.y;
    const int per = 2 * p.pool.n_heads;
    const int unit = blockIdx.x * kAppendWarps + (threadIdx.x >> 5);
    int first = p.first ? p.first[s] : 0, n = p.n_rows ? p.n_rows[s] : p.max_rows;
    if (first < 0 || n < 0 || n > p.max_rows || (int64_t)first + n > (int64_t)p.table_width * p.pool.page_size) {
        if (threadIdx.x == 0 && blockIdx.x == 0) record_status(status, kStatusBadLength);
        first = n = 0;
    }
    // rows up to max_rows are written, those from n on as zeros
    const int b = first / kBlock + unit / per;
    const int64_t p0 = (int64_t)b * kBlock, left = (int64_t)first + p.max_rows - p0;
    if (left <= 0) return;
    const int part = unit % per, head = part >> 1, blocks = p.pool.page_size / kBlock;
    const int t0 = (int)max((int64_t)0, first - p0), t1 = (int)min((int64_t)kBlock, max((int64_t)0, first + n - p0)), t2 = (int)min((int64_t)kBlock, left);
    int page = -1;
    if (t1 > t0) {
        page = page_of(p.table + s * p.table_nb_seq, b / blocks, p.pool.n_pages);
        if (page < 0 && lane == 0) record_status(status, kStatusBadPage);
    }
    const int in = head * blocks + b % blocks;
    const int64_t at = s * p.nb_seq + (p0 - first) * p.nb_row + head * kD;
    if (part & 1) read_block<F, true>(p, p.v + at, page, in, t0, t1, t2, lane);
    else read_block<F, false>(p, p.k + at, page, in, t0, t1, t2, lane);
}

}  // namespace paged

cudaError_t launch_paged_append(cudaStream_t stream, const cvattn_paged_append_params& p, int* status) {
    using namespace paged;
    const int64_t blocks = ((int64_t)p.max_new + 2 * kBlock - 2) / kBlock;  // most that max_new rows touch
    const int64_t units = blocks * 2 * p.pool.n_heads;
    const dim3 grid((unsigned)((units + kAppendWarps - 1) / kAppendWarps), (unsigned)p.n_seq);
    auto* fn = p.pool.format == kI8 ? paged_append_kernel<kI8> : paged_append_kernel<kE4M3>;
    return launch_overlapped(fn, grid, kAppendWarps * 32, 0, stream, p, status);
}

cudaError_t launch_paged_read(cudaStream_t stream, const cvattn_paged_read_params& p, int* status) {
    using namespace paged;
    const int64_t blocks = ((int64_t)p.max_rows + 2 * kBlock - 2) / kBlock, units = blocks * 2 * p.pool.n_heads;
    const dim3 grid((unsigned)((units + kAppendWarps - 1) / kAppendWarps), (unsigned)p.n_seq);
    auto* fn = p.pool.format == kI8 ? paged_read_kernel<kI8> : paged_read_kernel<kE4M3>;
    return launch_overlapped(fn, grid, kAppendWarps * 32, 0, stream, p, status);
}

}  // namespace cvattn
