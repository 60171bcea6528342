// pages.cu -- what the tables of a paged cache hold next, and the pages that are copied for it.
#include "launch.cuh"
#include "paged.cuh"

namespace cvattn {
namespace paged {

constexpr int kBookThreads = 1024;  // (block_scan: 32 warps)
constexpr int kMaxBookCtas = 8;  // of one cluster
constexpr int kMaxPools = 48;    // pools of one copy launch (kernel arguments)

// Workspace, int32: copies' count; the next table [n_seq][width]; per page its holders, writers and first writer, where it goes
// or the free pages in order; per sequence what is asked for it; copies (source, target).
// Where next, refs, writers, lowest and list fit into one CTA's shared memory, they lie there: then the books take one CTA, and
// what takes a cluster barrier and a trip to L2 otherwise takes a block barrier.  An assignment to
// 64 sequences: 16.0 us by a cluster, 13.2 in shared memory, 10.0 since this form's code is a kernel of its own and the wishes are read
// once.  All of it is latency (barriers, each behind a dependent load, and instructions fetched once).  Where the books do not fit, us
// of assignment | compaction with the copies (16 positions, one pool of one head): 500 x 40 entries of 20000 pages 19.5 | 19.0, 60 x 30
// of 60000 22.3 | 22.0, 8192 x 1 of 8000 34.9 | 19.4, 1024 x 256 of 100000 58.5 | 73.8; just below, 256 x 40 of 8000 in shared memory
// 18.0 | 16.0.
struct Books {
    int32_t *n_copies, *next, *refs, *writers, *lowest, *list, *src, *keep, *need, *from, *to;
    size_t bytes;
    Books(void* base, int64_t n_seq, int64_t width, int64_t n_pages) {
        const int64_t most = n_pages > n_seq ? n_pages : n_seq;
        int64_t at = 0;
        const auto take = [&](int64_t n) {
            int32_t* p = base ? static_cast<int32_t*>(base) + at : nullptr;
            at += n;
            return p;
        };
        n_copies = take(4);
        next = take(n_seq * width);
        refs = take(n_pages);
        writers = take(n_pages);
        lowest = take(n_pages);
        list = take(n_pages);
        src = take(n_seq);
        keep = take(n_seq);
        need = take(n_seq);
        from = take(most);
        to = take(most);
        bytes = (size_t)at * 4;
    }
    // Bytes of the arrays that may lie in shared memory, and their places there.
    static __host__ __device__ int64_t local_bytes(int64_t entries, int64_t n_pages, int64_t n_seq) { return 4 * (entries + 4 * n_pages + 3 * n_seq); }
    __device__ __forceinline__ void move_in(int32_t* to, int entries, int n_pages, int n_seq) {
        next = to;
        refs = next + entries;
        writers = refs + n_pages;
        lowest = writers + n_pages;
        list = lowest + n_pages;
        src = list + n_pages;
        keep = src + n_seq;
        need = keep + n_seq;
    }
};
constexpr int kLocalBytes = 200 * 1024;

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// The CTAs of one cluster keep the books together: what one writes to the workspace the others read after a cluster barrier.
// With the books in shared memory there is one CTA (kLocal, apart so that its code is short: run once, it is bound by fetching its
// instructions).
template <bool kLocal> struct Crew {
    int C, rank, at, of;  // CTAs, this one; this thread's place among all of theirs, how many
    __device__ __forceinline__ Crew() {
        uint32_t c = 1, r = 0;
        if (!kLocal) {
            asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(c));
            asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
        }
        C = c;
        rank = r;
        at = rank * kBookThreads + threadIdx.x;
        of = C * kBookThreads;
    }
    __device__ __forceinline__ void sync() const {
        if (kLocal) __syncthreads();
        else cluster_sync();
    }
};

// Exclusive sums over the block of two numbers a thread, and their totals.  (Packed in 64 bits: one pass.)
__device__ __forceinline__ void block_scan(int& a, int& b, int& total_a, int& total_b) {
    __shared__ long long sums[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long x = (long long)a << 32 | b;
    auto scan = [&](long long y) {
#pragma unroll
        for (int w = 1; w < 32; w <<= 1) {
            const long long z = __shfl_up_sync(0xffffffffu, y, w);
            if (lane >= w) y += z;
        }
        return y;
    };
    long long y = scan(x);
    __syncthreads();  // (sums may be in use from the call before)
    if (lane == 31) sums[warp] = y;
    __syncthreads();
    const long long v = scan(sums[lane]), all = __shfl_sync(0xffffffffu, v, 31), before = __shfl_sync(0xffffffffu, v, max(warp, 1) - 1);
    y += (warp ? before : 0) - x;
    a = (int)(y >> 32);
    b = (int)y;
    total_a = (int)(all >> 32);
    total_b = (int)all;
}

// Exclusive sums over the crew's items in order, `per` neighbouring ones a thread: value(i) of item i gives two numbers, take(i,
// before) gets the sums before it.  All threads get the totals.
template <bool kLocal, class V, class F> __device__ __forceinline__ int2 crew_scan(const Crew<kLocal>& crew, int n, V value, F take) {
    __shared__ int2 sums[kMaxBookCtas];
    const int per = (n + crew.of - 1) / crew.of, i0 = min(n, crew.at * per), i1 = min(n, i0 + per);
    int a = 0, b = 0, ta, tb;
#pragma unroll 1
    for (int i = i0; i < i1; ++i) {
        const int2 v = value(i);
        a += v.x;
        b += v.y;
    }
    block_scan(a, b, ta, tb);
    if (!kLocal) {
        crew.sync();  // (sums may be in use from the scan before)
        if ((int)threadIdx.x < crew.C) {
            uint32_t to;
            asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(smem_addr(&sums[crew.rank])), "r"((int)threadIdx.x));
            asm volatile("st.shared::cluster.v2.s32 [%0], {%1, %2};" ::"r"(to), "r"(ta), "r"(tb) : "memory");
        }
        __syncwarp();
        crew.sync();
        ta = tb = 0;
        for (int k = 0; k < crew.C; ++k) {
            if (k < crew.rank) {
                a += sums[k].x;
                b += sums[k].y;
            }
            ta += sums[k].x;
            tb += sums[k].y;
        }
    }
#pragma unroll 1
    for (int i = i0; i < i1; ++i) {
        const int2 v = value(i);
        take(i, make_int2(a, b));
        a += v.x;
        b += v.y;
    }
    return make_int2(ta, tb);
}

template <bool kLocal>
__global__ void __launch_bounds__(kBookThreads) pages_assign_kernel(const __grid_constant__ cvattn_pages_assign_params p, Books w, int P,
                                                                    int n_pages, int* status) {
    extern __shared__ int32_t local_books[];
    const Crew<kLocal> crew;
    griddep_wait();
    const int width = p.table_width;
    if (kLocal) w.move_in(local_books, p.n_seq * width, n_pages, p.n_seq);
#pragma unroll 1
    for (int i = crew.at; i < n_pages; i += crew.of) {
        w.refs[i] = w.writers[i] = 0;
        w.lowest[i] = INT32_MAX;
    }
    if (crew.at == 0) *w.n_copies = 0;
    const int64_t most = (int64_t)width * P;
#pragma unroll 1
    for (int s = crew.at; s < p.n_seq; s += crew.of) {
        int src = p.src ? p.src[s] : s, keep = p.keep[s], need = p.need[s];
        if (src < 0 || src >= p.n_seq || keep < 0 || keep > most || need < 0 || need > most) {
            record_status(status, kStatusBadLength);
            src = s;
            keep = need = 0;
        }
        w.src[s] = src;
        w.keep[s] = keep;
        w.need[s] = need;
    }
    crew.sync();
    // kept entries, and who writes into a partly filled page
#pragma unroll 2
    for (int i = crew.at; i < p.n_seq * width; i += crew.of) {
        const int s = i / width, j = i - s * width, keep = w.keep[s], need = w.need[s];
        int page = -1;
        if (j < (keep + P - 1) / P) {
            page = page_of(p.table + w.src[s] * p.table_nb_seq, j, n_pages);
            if (page < 0) {
                record_status(status, kStatusBadPage);
            } else {
                atomicAdd(&w.refs[page], 1);
                if (need > keep && keep % P && j == keep / P) {
                    atomicAdd(&w.writers[page], 1);
                    atomicMin(&w.lowest[page], s);
                }
            }
        }
        w.next[i] = page;
    }
    crew.sync();
    // free pages in order
    const int n_free = crew_scan(crew, n_pages, [&](int i) { return make_int2(w.refs[i] == 0, 0); },
                                 [&](int i, int2 before) {
                                     if (w.refs[i] == 0) w.list[before.x] = i;
                                 }).x;
    crew.sync();
    // sequence by sequence: the pages that it asks for, and whether it copies its tail
    auto asks = [&](int s, int& keep, int& need, int& tail) {
        keep = w.keep[s];
        need = w.need[s];
        tail = need > keep && keep % P ? w.next[(int64_t)s * width + keep / P] : -1;
        const int copies = tail >= 0 && w.refs[tail] > 1 && !(w.writers[tail] == w.refs[tail] && w.lowest[tail] == s);
        return make_int2(max(0, (need + P - 1) / P - (keep + P - 1) / P) + copies, copies);
    };
    int keep, need, tail;
    // (the sums only grow, so all behind the first without room are without it, and the copies before one with room have room too)
    crew_scan(crew, p.n_seq, [&](int s) { return asks(s, keep, need, tail); },
              [&](int s, int2 before) {
                  const int2 v = asks(s, keep, need, tail);
                  const bool granted = before.x + v.x <= n_free;
                  p.room[s] = granted ? max(keep, need) : keep;
                  if (!granted) return;
                  if (v.y) {
                      w.from[before.y] = tail;
                      w.to[before.y] = w.list[before.x];
                      atomicMax(w.n_copies, before.y + 1);
                  }
                  const int first = (keep + P - 1) / P - v.y;
#pragma unroll 1
                  for (int k = 0; k < v.x; ++k) w.next[(int64_t)s * width + first + k] = w.list[before.x + k];
              });
    crew.sync();
#pragma unroll 1
    for (int i = crew.at; i < p.n_seq * width; i += crew.of) p.table_out[(int64_t)(i / width) * p.table_nb_seq + i % width] = w.next[i];
    if (p.refs) {
        int32_t* refs = kLocal ? w.refs : p.refs;
#pragma unroll 1
        for (int i = crew.at; i < n_pages; i += crew.of) refs[i] = 0;
        crew.sync();
#pragma unroll 1
        for (int i = crew.at; i < p.n_seq * width; i += crew.of)
            if (w.next[i] >= 0) atomicAdd(&refs[w.next[i]], 1);
        if (kLocal) {
            crew.sync();
#pragma unroll 1
            for (int i = crew.at; i < n_pages; i += crew.of) p.refs[i] = refs[i];
        }
    }
}

template <bool kLocal>
__global__ void __launch_bounds__(kBookThreads) pages_compact_kernel(const __grid_constant__ cvattn_pages_compact_params p, Books w,
                                                                     int n_pages, int* status) {
    extern __shared__ int32_t local_books[];
    const Crew<kLocal> crew;
    griddep_wait();
    const int width = p.table_width;
    if (kLocal) w.move_in(local_books, p.n_seq * width, n_pages, p.n_seq);
    for (int i = crew.at; i < n_pages; i += crew.of) w.refs[i] = 0;
    crew.sync();
    for (int i = crew.at; i < p.n_seq * width; i += crew.of) {
        const int page = page_of(p.table + (int64_t)(i / width) * p.table_nb_seq, i % width, n_pages);
        w.next[i] = page;
        if (page >= 0) atomicAdd(&w.refs[page], 1);
    }
    crew.sync();
    const int live = crew_scan(crew, n_pages, [&](int i) { return make_int2(w.refs[i] > 0, 0); }, [](int, int2) {}).x;
    // the k-th held page from `live` on goes to the k-th free one below it
    const int moved = crew_scan(crew, n_pages, [&](int i) { return make_int2(w.refs[i] > 0 && i >= live, w.refs[i] == 0 && i < live); },
                                [&](int i, int2 before) {
                                    if (w.refs[i] > 0 && i >= live) w.from[before.x] = i;
                                    if (w.refs[i] == 0 && i < live) w.to[before.y] = i;
                                    w.list[i] = i;
                                }).x;
    crew.sync();
    for (int i = crew.at; i < moved; i += crew.of) w.list[w.from[i]] = w.to[i];
    if (crew.at == 0) {
        *w.n_copies = moved;
        *p.n_live = live;
    }
    if (p.refs)
        for (int i = crew.at; i < n_pages; i += crew.of) p.refs[i] = 0;
    crew.sync();
    for (int i = crew.at; i < p.n_seq * width; i += crew.of)
        p.table_out[(int64_t)(i / width) * p.table_nb_seq + i % width] = w.next[i] < 0 ? -1 : w.list[w.next[i]];
    if (p.refs)
        for (int i = crew.at; i < n_pages; i += crew.of)
            if (w.refs[i] > 0) p.refs[w.list[i]] = w.refs[i];
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

// A warp takes 2 KB of a page of one tensor at a time, four 16-byte loads a lane before the first store: what a page's copy waits
// for is its loads' latency, and 4736 warps of 2 KB keep 9.7 MB in flight.  Bound by memory: 51 MB read and written in about 13 us
// (7.9 TB/s together: most of what is written is still in L2 at the end).  With one 16-byte load a lane at a time a compaction took 47,
// where it takes 20 now.
constexpr int kCopyThreads = 256, kPiece = 2048;

__global__ void __launch_bounds__(kCopyThreads) pages_copy_kernel(const __grid_constant__ CopyArgs a) {
    griddep_wait();
    const int t = blockIdx.y, pool = t >> 1, lane = threadIdx.x & 31;
    const int pieces = (a.bytes[pool] + kPiece - 1) / kPiece, n = *a.n_copies * pieces;
    for (int u = blockIdx.x * (kCopyThreads / 32) + (threadIdx.x >> 5); u < n; u += gridDim.x * (kCopyThreads / 32)) {
        const int c = u / pieces, at = (u - c * pieces) * kPiece + lane * 16;
        const int64_t from = a.from[c], to = a.to[c];
        const uint8_t* src = a.data[t] + from * a.nb_page[pool] + at;
        uint8_t* dst = a.data[t] + to * a.nb_page[pool] + at;
        uint4 v[kPiece / 512];
#pragma unroll
        for (int i = 0; i < kPiece / 512; ++i)
            if (at + i * 512 < a.bytes[pool]) v[i] = __ldcs(reinterpret_cast<const uint4*>(src + i * 512));
#pragma unroll
        for (int i = 0; i < kPiece / 512; ++i)
            if (at + i * 512 < a.bytes[pool]) *reinterpret_cast<uint4*>(dst + i * 512) = v[i];
        if (u == c * pieces)
            for (int i = lane; i < a.scales[pool]; i += 32) a.scale[t][to * a.nb_scale[pool] + i] = a.scale[t][from * a.nb_scale[pool] + i];
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
        const int ctas = (148 * 8 + a.n - 1) / a.n;
        const cudaError_t e = launch_overlapped(pages_copy_kernel, dim3((unsigned)ctas, (unsigned)a.n), kCopyThreads, 0, stream, a);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

}  // namespace paged

size_t pages_workspace_bytes(int n_seq, int table_width, int n_pages) { return paged::Books(nullptr, n_seq, table_width, n_pages).bytes; }

// CTAs that keep books in the workspace: four entries or pages a thread at least.
static int book_ctas(int64_t entries, int n_pages) {
    const int64_t items = entries > n_pages ? entries : n_pages;
    int c = 1;
    while (c < paged::kMaxBookCtas && items > (int64_t)c * 4 * paged::kBookThreads) c *= 2;
    return c;
}

// One of two kernels: with the books in shared memory where they fit, or by a cluster.
template <class Local, class Crewed, class... A>
static cudaError_t keep_books(Local* local, Crewed* crewed, cudaStream_t stream, int64_t entries, int n_pages, int n_seq, const A&... args) {
    const int64_t bytes = paged::Books::local_bytes(entries, n_pages, n_seq);
    if (bytes <= paged::kLocalBytes) {
        const cudaError_t e = cudaFuncSetAttribute(local, cudaFuncAttributeMaxDynamicSharedMemorySize, paged::kLocalBytes);
        return e != cudaSuccess ? e : launch_overlapped(local, dim3(1), paged::kBookThreads, (size_t)bytes, stream, args...);
    }
    const int c = book_ctas(entries, n_pages);
    return launch_overlapped_clusters(crewed, dim3((unsigned)c), paged::kBookThreads, 0, c, stream, args...);
}

cudaError_t launch_pages_assign(cudaStream_t stream, const cvattn_pages_assign_params& p, int page_size, int n_pages, int* status) {
    const paged::Books w(p.workspace, p.n_seq, p.table_width, n_pages);
    const cudaError_t e = keep_books(paged::pages_assign_kernel<true>, paged::pages_assign_kernel<false>, stream, (int64_t)p.n_seq * p.table_width,
                                     n_pages, p.n_seq, p, w, page_size, n_pages, status);
    return e != cudaSuccess ? e : paged::copy_pages(stream, p.pools, p.n_pools, w);
}

cudaError_t launch_pages_compact(cudaStream_t stream, const cvattn_pages_compact_params& p, int n_pages, int* status) {
    const paged::Books w(p.workspace, p.n_seq, p.table_width, n_pages);
    const cudaError_t e = keep_books(paged::pages_compact_kernel<true>, paged::pages_compact_kernel<false>, stream, (int64_t)p.n_seq * p.table_width,
                                     n_pages, p.n_seq, p, w, n_pages, status);
    return e != cudaSuccess ? e : paged::copy_pages(stream, p.pools, p.n_pools, w);
}

}  // namespace cvattn
