// pages.cu -- what the tables of a paged cache hold next, and the pages that are copied for it.
#include "launch.cuh"
#include "paged.cuh"

namespace cvattn {
namespace paged {

constexpr int kBookThreads = 1024;
constexpr int kMaxPools = 48;  // pools of one copy launch (kernel arguments)

// Workspace, int32: the next table [n_seq][width], per page its holders, writers and first writer, free pages in order,
// copies (source, target), their count.
struct Books {
    int32_t *next, *refs, *writers, *lowest, *list, *from, *to, *n_copies;
    size_t bytes;
    Books(void* base, int64_t n_seq, int64_t width, int64_t n_pages) {
        int32_t* w = static_cast<int32_t*>(base);
        const int64_t most = n_pages > n_seq ? n_pages : n_seq;
        n_copies = w; w += 4;
        next = w; w += n_seq * width;
        refs = w; w += n_pages;
        writers = w; w += n_pages;
        lowest = w; w += n_pages;
        list = w; w += n_pages;
        from = w; w += most;
        to = w; w += most;
        bytes = (size_t)(w - static_cast<int32_t*>(base)) * 4;
    }
};

// Exclusive sum over the block of one number a thread; every thread gets the total too.
__device__ __forceinline__ int block_scan(int x, int& total) {
    __shared__ int sums[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int y = x;
#pragma unroll
    for (int w = 1; w < 32; w <<= 1) {
        const int z = __shfl_up_sync(0xffffffffu, y, w);
        if (lane >= w) y += z;
    }
    __syncthreads();  // (sums may be in use from the call before)
    if (lane == 31) sums[warp] = y;
    __syncthreads();
    int before = 0, all = 0;
    for (int w = 0; w < (int)(blockDim.x >> 5); ++w) {
        const int v = sums[w];
        if (w < warp) before += v;
        all += v;
    }
    total = all;
    return before + y - x;
}

__global__ void __launch_bounds__(kBookThreads) pages_assign_kernel(const __grid_constant__ cvattn_pages_assign_params p, Books w, int P,
                                                                    int n_pages, int* status) {
    griddep_wait();
    const int tid = threadIdx.x, width = p.table_width;
    for (int i = tid; i < n_pages; i += kBookThreads) {
        w.refs[i] = w.writers[i] = 0;
        w.lowest[i] = INT32_MAX;
    }
    __syncthreads();
    // kept entries
    auto wish = [&](int s, int& src, int& keep, int& need) {
        src = p.src ? p.src[s] : s;
        keep = p.keep[s];
        need = p.need[s];
        const int64_t most = (int64_t)width * P;
        if (src < 0 || src >= p.n_seq || keep < 0 || keep > most || need < 0 || need > most) {
            record_status(status, kStatusBadLength);
            src = s;
            keep = need = 0;
        }
    };
    for (int64_t i = tid; i < (int64_t)p.n_seq * width; i += kBookThreads) {
        const int s = (int)(i / width), j = (int)(i % width);
        int src, keep, need, page = -1;
        wish(s, src, keep, need);
        if (j < (keep + P - 1) / P) {
            page = page_of(p.table + src * p.table_nb_seq, j, n_pages);
            if (page < 0) record_status(status, kStatusBadPage);
            else atomicAdd(&w.refs[page], 1);
        }
        w.next[i] = page;
    }
    __syncthreads();
    // who writes into a shared tail
    auto tail_of = [&](int s, int keep, int need) {
        return need > keep && keep % P ? w.next[(int64_t)s * width + keep / P] : -1;
    };
    for (int s = tid; s < p.n_seq; s += kBookThreads) {
        int src, keep, need;
        wish(s, src, keep, need);
        const int tail = tail_of(s, keep, need);
        if (tail >= 0) {
            atomicAdd(&w.writers[tail], 1);
            atomicMin(&w.lowest[tail], s);
        }
    }
    __syncthreads();
    // free pages in order
    int n_free = 0;
    for (int i0 = 0; i0 < n_pages; i0 += kBookThreads) {
        const int i = i0 + tid;
        const int is = i < n_pages && w.refs[i] == 0;
        int total;
        const int at = n_free + block_scan(is, total);
        if (is) w.list[at] = i;
        n_free += total;
    }
    __syncthreads();
    // sequence by sequence
    int asked = 0, copied = 0;
    for (int s0 = 0; s0 < p.n_seq; s0 += kBookThreads) {
        const int s = s0 + tid;
        int src, keep = 0, need = 0, tail = -1, copies = 0, fresh = 0;
        if (s < p.n_seq) {
            wish(s, src, keep, need);
            tail = tail_of(s, keep, need);
            copies = tail >= 0 && w.refs[tail] > 1 && !(w.writers[tail] == w.refs[tail] && w.lowest[tail] == s);
            fresh = max(0, (need + P - 1) / P - (keep + P - 1) / P) + copies;
        }
        int total;
        const int before = asked + block_scan(fresh, total);
        asked += total;
        const bool granted = before + fresh <= n_free;
        const int which = copied + block_scan(granted ? copies : 0, total);
        copied += total;
        if (s < p.n_seq) {
            p.room[s] = granted ? max(keep, need) : keep;
            if (granted) {
                if (copies) {
                    w.from[which] = tail;
                    w.to[which] = w.list[before];
                }
                for (int k = 0; k < fresh; ++k) w.next[(int64_t)s * width + (keep + P - 1) / P - copies + k] = w.list[before + k];
            }
        }
    }
    if (tid == 0) *w.n_copies = copied;
    __syncthreads();
    for (int64_t i = tid; i < (int64_t)p.n_seq * width; i += kBookThreads) p.table_out[i / width * p.table_nb_seq + i % width] = w.next[i];
    if (p.refs) {
        for (int i = tid; i < n_pages; i += kBookThreads) p.refs[i] = 0;
        __syncthreads();
        for (int64_t i = tid; i < (int64_t)p.n_seq * width; i += kBookThreads)
            if (w.next[i] >= 0) atomicAdd(&p.refs[w.next[i]], 1);
    }
}

__global__ void __launch_bounds__(kBookThreads) pages_compact_kernel(const __grid_constant__ cvattn_pages_compact_params p, Books w,
                                                                     int n_pages, int* status) {
    griddep_wait();
    const int tid = threadIdx.x, width = p.table_width;
    for (int i = tid; i < n_pages; i += kBookThreads) w.refs[i] = 0;
    __syncthreads();
    for (int64_t i = tid; i < (int64_t)p.n_seq * width; i += kBookThreads) {
        const int page = page_of(p.table + i / width * p.table_nb_seq, (int)(i % width), n_pages);
        if (page >= 0) atomicAdd(&w.refs[page], 1);
    }
    __syncthreads();
    int live = 0;
    for (int i0 = 0; i0 < n_pages; i0 += kBookThreads) {
        const int i = i0 + tid;
        int total;
        block_scan(i < n_pages && w.refs[i] > 0, total);
        live += total;
    }
    int moved = 0, free = 0;
    for (int i0 = 0; i0 < n_pages; i0 += kBookThreads) {
        const int i = i0 + tid;
        const bool real = i < n_pages, held = real && w.refs[i] > 0;
        int total;
        int at = moved + block_scan(held && i >= live, total);
        moved += total;
        if (held && i >= live) w.from[at] = i;
        at = free + block_scan(real && !held && i < live, total);
        free += total;
        if (real && !held && i < live) w.to[at] = i;
        if (real) w.list[i] = i;  // where a page goes
    }
    __syncthreads();
    for (int i = tid; i < moved; i += kBookThreads) w.list[w.from[i]] = w.to[i];
    if (tid == 0) {
        *w.n_copies = moved;
        *p.n_live = live;
    }
    __syncthreads();
    for (int64_t i = tid; i < (int64_t)p.n_seq * width; i += kBookThreads) {
        const int page = page_of(p.table + i / width * p.table_nb_seq, (int)(i % width), n_pages);
        p.table_out[i / width * p.table_nb_seq + i % width] = page < 0 ? -1 : w.list[page];
    }
    if (p.refs) {
        for (int i = tid; i < n_pages; i += kBookThreads) p.refs[i] = 0;
        __syncthreads();
        for (int i = tid; i < n_pages; i += kBookThreads)
            if (w.refs[i] > 0) p.refs[w.list[i]] = w.refs[i];
    }
}

// Page from[c] of every pool to page to[c].
struct CopyArgs {
    uint8_t* data[2 * kMaxPools];
    float* scale[2 * kMaxPools];
    int64_t nb_page[kMaxPools], nb_scale[kMaxPools];
    int32_t bytes[kMaxPools], scales[kMaxPools];
    const int32_t *from, *to, *n_copies;
    int n;  // tensors: keys and values of each pool
};

__global__ void __launch_bounds__(256) pages_copy_kernel(const __grid_constant__ CopyArgs a) {
    griddep_wait();
    const int64_t n = (int64_t)*a.n_copies * a.n;
    for (int64_t u = blockIdx.x; u < n; u += gridDim.x) {
        const int c = (int)(u / a.n), t = (int)(u % a.n), pool = t >> 1;
        const int64_t from = a.from[c], to = a.to[c];
        const uint4* src = reinterpret_cast<const uint4*>(a.data[t] + from * a.nb_page[pool]);
        uint4* dst = reinterpret_cast<uint4*>(a.data[t] + to * a.nb_page[pool]);
        for (int i = threadIdx.x; i < a.bytes[pool] / 16; i += 256) dst[i] = src[i];
        for (int i = threadIdx.x; i < a.scales[pool]; i += 256) a.scale[t][to * a.nb_scale[pool] + i] = a.scale[t][from * a.nb_scale[pool] + i];
    }
}

static cudaError_t copy_pages(cudaStream_t stream, const cvattn_page_pool* pools, int n_pools, const Books& w) {
    for (int at = 0; at < n_pools; at += kMaxPools) {
        CopyArgs a{};
        const int n = n_pools - at < kMaxPools ? n_pools - at : kMaxPools;
        for (int i = 0; i < n; ++i) {
            const cvattn_page_pool& q = pools[at + i];
            a.data[2 * i] = static_cast<uint8_t*>(q.k);
            a.data[2 * i + 1] = static_cast<uint8_t*>(q.v);
            a.scale[2 * i] = q.k_scale;
            a.scale[2 * i + 1] = q.v_scale;
            a.nb_page[i] = q.nb_page;
            a.nb_scale[i] = q.nb_scale;
            a.bytes[i] = q.n_heads * q.page_size * kD;
            a.scales[i] = q.n_heads * q.page_size / kBlock;
        }
        a.from = w.from;
        a.to = w.to;
        a.n_copies = w.n_copies;
        a.n = 2 * n;
        const cudaError_t e = launch_overlapped(pages_copy_kernel, 148 * 4, 256, 0, stream, a);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

}  // namespace paged

size_t pages_workspace_bytes(int n_seq, int table_width, int n_pages) { return paged::Books(nullptr, n_seq, table_width, n_pages).bytes; }

cudaError_t launch_pages_assign(cudaStream_t stream, const cvattn_pages_assign_params& p, int page_size, int n_pages, int* status) {
    const paged::Books w(p.workspace, p.n_seq, p.table_width, n_pages);
    const cudaError_t e = launch_overlapped(paged::pages_assign_kernel, 1, paged::kBookThreads, 0, stream, p, w, page_size, n_pages, status);
    return e != cudaSuccess ? e : paged::copy_pages(stream, p.pools, p.n_pools, w);
}

cudaError_t launch_pages_compact(cudaStream_t stream, const cvattn_pages_compact_params& p, int n_pages, int* status) {
    const paged::Books w(p.workspace, p.n_seq, p.table_width, n_pages);
    const cudaError_t e = launch_overlapped(paged::pages_compact_kernel, 1, paged::kBookThreads, 0, stream, p, w, n_pages, status);
    return e != cudaSuccess ? e : paged::copy_pages(stream, p.pools, p.n_pools, w);
}

}  // namespace cvattn
