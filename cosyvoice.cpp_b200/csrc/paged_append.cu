// paged_append.cu -- rows rounded into the pages of an 8-bit cache, and read back.
#include "launch.cuh"
#include "paged.cuh"

namespace cvattn {
namespace paged {

// A warp takes one block of one head, keys or values: 16 x 64 f32 values, 32 a lane, in the order in which it writes their
// codes.  Every block has one writer, so rows that the block held are read, rounded anew and written in place.
constexpr int kAppendWarps = 4;

// Value (of 32) e of a lane: position and dim, in the order of the block's bytes (four of them a word).
__device__ __forceinline__ void place_of(bool values, int lane, int e, int& t, int& d) {
    if (values) {  // words (half, lane, tile): 4 positions of one dim
        t = (lane & 3) * 4 + (e & 3);
        d = (e >> 4) * 32 + ((e >> 2) & 3) * 8 + (lane >> 2);
    } else {       // words of two rows at a time: 4 values of one position
        t = 2 * (e >> 2) + (lane >> 4);
        d = (lane & 15) * 4 + (e & 3);
    }
}
// Byte of word w (of 8) of a lane.
__device__ __forceinline__ int word_at(bool values, int lane, int w) {
    return values ? (w >> 2) * 512 + lane * 16 + (w & 3) * 4 : w * 128 + lane * 4;
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
    const int64_t b = (int64_t)L / kBlock + unit / per;  // block of the sequence
    if (n == 0 || b * kBlock >= (int64_t)L + n) return;
    const int part = unit % per, head = part >> 1;
    const bool values = part & 1;
    const int blocks = p.pool.page_size / kBlock;
    const int page = page_of(p.table + s * p.table_nb_seq, (int)(b / blocks), p.pool.n_pages);
    if (page < 0 || (p.refs && p.refs[page] > 1)) {
        if (lane == 0) record_status(status, page < 0 ? kStatusBadPage : kStatusSharedPage);
        return;
    }
    const int in = head * blocks + (int)(b % blocks);
    uint8_t* codes = static_cast<uint8_t*>(values ? p.pool.v : p.pool.k) + page * p.pool.nb_page + (int64_t)in * kBlockBytes;
    float* scale_at = (values ? p.pool.v_scale : p.pool.k_scale) + page * p.pool.nb_scale + in;
    const int t0 = (int)max((int64_t)0, L - b * kBlock), t1 = (int)min((int64_t)kBlock, L + n - b * kBlock);  // the new positions
    const float* src = (values ? p.v : p.k) + s * p.nb_seq + (b * kBlock - L) * p.nb_row + head * kD;

    float x[32];
    float amax = 0.0f;
#pragma unroll
    for (int e = 0; e < 32; ++e) {
        int t, d;
        place_of(values, lane, e, t, d);
        x[e] = t >= t0 && t < t1 ? src[t * p.nb_row + d] : 0.0f;
        const float a = fabsf(x[e]);
        if (a < INFINITY) amax = fmaxf(amax, a);
    }
    amax = warp_max_abs(amax);
    const float was = t0 > 0 ? fmaxf(*scale_at, 0.0f) : 0.0f;  // (NaN: 0)
    const float fresh = scale_of<F>(amax);
    const float scale = fmaxf(was, fresh);
    const bool grows = t0 > 0 && scale > was;
    const float inv = scale > 0.0f ? __fdiv_rn(1.0f, scale) : 0.0f;
    const float shrink = grows ? __fdiv_rn(was, scale) : 1.0f;
    __syncwarp();
    if (lane == 0) *scale_at = scale;
#pragma unroll
    for (int w = 0; w < 8; ++w) {
        uint32_t* at = reinterpret_cast<uint32_t*>(codes + word_at(values, lane, w));
        int first, last, d;
        place_of(values, lane, 4 * w, first, d);
        place_of(values, lane, 4 * w + 3, last, d);
        if (first >= t1 || (last < t0 && !grows)) continue;  // nothing of the word changes
        uint32_t word = first >= t0 && last < t1 ? 0u : *at;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            int t;
            place_of(values, lane, 4 * w + c, t, d);
            const uint32_t old = word >> (8 * c) & 0xffu;
            uint32_t code = old;
            if (t >= t0 && t < t1) {
                const float v = x[4 * w + c];
                if (isnan(v) || scale == 0.0f) code = F == kI8 ? 128u : 0u;
                else code = nearest_code<F>(v * inv, v, scale);
            } else if (t < t0 && grows) {
                const float v = code_value<F>(old);
                code = nearest_code<F>(v * shrink, (double)v * was, scale);
            }
            word = (word & ~(0xffu << (8 * c))) | code << (8 * c);
        }
        *at = word;
    }
}

// A thread takes four neighbouring values of one row, keys or values.
template <int F>
__global__ void __launch_bounds__(256) paged_read_kernel(const __grid_constant__ cvattn_paged_read_params p, int* status) {
    griddep_wait();
    const int s = blockIdx.y, per = 2 * p.pool.n_heads * (kD / 4);
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= (int64_t)p.max_rows * per) return;
    const int row = (int)(i / per), c = (int)(i % per), d = c % (kD / 4) * 4, head = c / (kD / 4) % p.pool.n_heads;
    const bool values = c / (kD / 4) >= p.pool.n_heads;
    const int first = p.first ? p.first[s] : 0, n = p.n_rows ? p.n_rows[s] : p.max_rows;
    float4 out = make_float4(0.f, 0.f, 0.f, 0.f);
    const bool bad = first < 0 || n < 0 || n > p.max_rows || (int64_t)first + n > (int64_t)p.table_width * p.pool.page_size;
    if (bad) {
        if (i == 0) record_status(status, kStatusBadLength);
    } else if (row < n) {
        const int at = first + row, blocks = p.pool.page_size / kBlock;
        const int page = page_of(p.table + s * p.table_nb_seq, at / p.pool.page_size, p.pool.n_pages);
        if (page < 0) {
            record_status(status, kStatusBadPage);
        } else {
            const int in = head * blocks + at % p.pool.page_size / kBlock, t = at % kBlock;
            const uint8_t* codes = static_cast<const uint8_t*>(values ? p.pool.v : p.pool.k) + page * p.pool.nb_page + (int64_t)in * kBlockBytes;
            const float scale = ((values ? p.pool.v_scale : p.pool.k_scale) + page * p.pool.nb_scale)[in];
            float* o = &out.x;
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = code_value<F>(codes[values ? v_place(t, d + e) : t * kD + d + e]) * scale;
        }
    }
    *reinterpret_cast<float4*>((values ? p.v : p.k) + s * p.nb_seq + row * p.nb_row + head * kD + d) = out;
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
    const int64_t items = (int64_t)p.max_rows * 2 * p.pool.n_heads * (kD / 4);
    const dim3 grid((unsigned)((items + 255) / 256), (unsigned)p.n_seq);
    auto* fn = p.pool.format == kI8 ? paged_read_kernel<kI8> : paged_read_kernel<kE4M3>;
    return launch_overlapped(fn, grid, 256, 0, stream, p, status);
}

}  // namespace cvattn
