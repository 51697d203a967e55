// kv_pages.hip — who holds which page of a paged KV cache: sequences forked,
// resized (pages taken and given back, a shared last page copied before it is
// written), the pool compacted, and the slots of a batch's new tokens. All of
// it on the device, from tables that lie there, so a decode loop (or a graph
// of one) needs no host in between.
#include <algorithm>

#include "kv.h"
#include "rt_internal.h"

namespace wv {
namespace {

constexpr int kMaxSeqs = 16384;    // of a table: one column of it lies in LDS
constexpr int kPlanThreads = 1024;
constexpr int kCopyBlocks = 4096;  // of a copy, twice what runs at once

typedef int32_t i4 __attribute__((ext_vector_type(4), aligned(4)));

struct Tables {
    int32_t *pages, *len, *refs;
    int n_seqs, max_pages, n_pages, page_shift;
};

// A table's work array.
struct Work {
    int32_t* n;           // [16]: pairs to copy; pages held
    int32_t *src, *dst;   // [pairs]: pages to copy, from (-1: none) and to
    int32_t *tail, *off;  // [n_seqs]: positions of such a page to copy; where a sequence's free pages begin in `a`
    int32_t *a, *b;       // [n_pages]
};
int64_t work_pairs(int n_seqs, int n_pages) { return std::max(n_seqs, n_pages / 2 + 1); }
int64_t work_ints(int n_seqs, int n_pages) {
    return 16 + 2 * work_pairs(n_seqs, n_pages) + 2 * int64_t(n_seqs) + 2 * int64_t(n_pages);
}
Work work_of(int32_t* w, int n_seqs, int n_pages) {
    const int64_t m = work_pairs(n_seqs, n_pages);
    Work k;
    k.n = w, k.src = w + 16, k.dst = k.src + m, k.tail = k.dst + m, k.off = k.tail + n_seqs;
    k.a = k.off + n_seqs, k.b = k.a + n_pages;
    return k;
}

// Counts that atomics of this kernel have written: past the L1, which does not see those.
__device__ __forceinline__ int32_t ld_now(const int32_t* p) {
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void add_to(int32_t* p, int32_t v) {
    __hip_atomic_fetch_add(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// What the block's threads wrote before is there for the ones that read after.
__device__ __forceinline__ void block_fence() {
    __threadfence();
    __syncthreads();
    __threadfence();
}

// Sum of v over the threads before this one, and over all of them. `lds`: 17 values.
template <class T>
__device__ __forceinline__ T scan_before(T v, T* lds, T& all) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    T x = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const T o = __shfl_up(x, d, 64);
        if (lane >= d) x += o;
    }
    if (lane == 63) lds[wave] = x;
    __syncthreads();
    T before = 0;
    all = 0;
#pragma unroll
    for (int w = 0; w < kPlanThreads / 64; ++w) {
        if (w < wave) before += lds[w];
        all += lds[w];
    }
    __syncthreads();
    return before + x - v;
}

// Four counts from `at` on; those past the pool read as held.
__device__ __forceinline__ i4 four_refs(const int32_t* refs, int at, int n) {
    if (at + 4 <= n) return *reinterpret_cast<const i4*>(refs + at);
    i4 x = {1, 1, 1, 1};
    for (int k = 0; k < 4; ++k)
        if (at + k < n) x[k] = refs[at + k];
    return x;
}

__device__ __forceinline__ int pages_of(int len, int shift) { return (len + (1 << shift) - 1) >> shift; }

// The whole of resize but the copies, by one block: its steps depend on each
// other, and a table's entries and the pool's counts are a few 10 KB.
__global__ void __launch_bounds__(kPlanThreads) k_pages_resize(Tables t, Work w, const int32_t* __restrict__ to,
                                                               int32_t* __restrict__ ok) {
    __shared__ int64_t lds[17];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, P = t.page_shift;
    const int width = t.max_pages << P;  // below 2^31
    auto length = [&](int b) { return min(max(t.len[b], 0), width); };
    auto target = [&](int b) { return max(to[b], 0); };

    // those that shrink, a wave each
    for (int b = wave; b < t.n_seqs; b += kPlanThreads / 64) {
        const int have = length(b), want = target(b);
        if (want >= have) continue;
        int32_t* row = t.pages + int64_t(b) * t.max_pages;
        for (int e = pages_of(want, P) + lane; e < pages_of(have, P); e += 64) {
            const int p = row[e];
            if (unsigned(p) < unsigned(t.n_pages)) add_to(t.refs + p, -1);
            row[e] = -1;
        }
    }
    block_fence();
    // The page that a growing sequence's next position lies in, if it has rows already: how many such sequences
    // share it, and the last of them. (A sequence that shrank still has its old length here: it does not grow.)
    auto last_page = [&](int b) {
        const int have = length(b), want = target(b);
        if (want <= have || want > width || !(have & ((1 << P) - 1))) return -1;
        const int p = t.pages[int64_t(b) * t.max_pages + (have >> P)];
        return unsigned(p) < unsigned(t.n_pages) ? p : -1;
    };
    for (int b = tid; b < t.n_seqs; b += kPlanThreads)
        if (const int p = last_page(b); p >= 0) w.a[p] = 0, w.b[p] = -1;
    block_fence();
    for (int b = tid; b < t.n_seqs; b += kPlanThreads)
        if (const int p = last_page(b); p >= 0) {
            add_to(w.a + p, 1);
            __hip_atomic_fetch_max(w.b + p, b, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
    block_fence();
    // pages that each needs, and where in the list of free ones they begin
    int64_t total = 0;
    for (int b0 = 0; b0 < t.n_seqs; b0 += kPlanThreads) {
        const int b = b0 + tid;
        int64_t need = 0;
        int copy = -1;
        bool grows = false;
        if (b < t.n_seqs) {
            const int have = length(b), want = target(b);
            grows = want > have && want <= width;
            if (grows) {
                const int p = last_page(b);
                if (p >= 0) {
                    const int refs = ld_now(t.refs + p);
                    if (refs > 1 && !(ld_now(w.a + p) == refs && ld_now(w.b + p) == b)) copy = p;
                }
                need = pages_of(want, P) - pages_of(have, P) + (copy >= 0);
            }
        }
        int64_t all;
        const int64_t off = total + scan_before(need, lds, all);
        if (b < t.n_seqs) {
            w.src[b] = copy;
            // past the pool's end no sequence is served any more, wherever it would begin
            w.off[b] = grows ? int(min(off, int64_t(t.n_pages) + 1)) : -1;
        }
        total += all;
    }
    block_fence();
    // the lowest free pages, as many as are needed
    const int most = int(min(total, int64_t(t.n_pages)));
    int found = 0;
    for (int base = 0; base < t.n_pages && found < most; base += 4 * kPlanThreads) {
        const int at = base + 4 * tid;
        const i4 r = four_refs(t.refs, at, t.n_pages);
        const int n = (r[0] <= 0) + (r[1] <= 0) + (r[2] <= 0) + (r[3] <= 0);
        int64_t all;
        int64_t i = found + scan_before(int64_t(n), lds, all);
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (r[k] <= 0 && i++ < most) w.a[i - 1] = at + k;
        found += int(all);
    }
    found = min(found, most);
    block_fence();
    // those that grow, a wave each
    for (int b = wave; b < t.n_seqs; b += kPlanThreads / 64) {
        const int have = length(b), want = target(b), off = w.off[b], old = w.src[b];
        bool done = want <= width;
        int from = -1, into = -1;
        if (off >= 0) {
            const int first = pages_of(have, P) - (old >= 0), n = pages_of(want, P) - first;
            done = int64_t(off) + n <= found;
            if (done) {
                int32_t* row = t.pages + int64_t(b) * t.max_pages + first;
                for (int e = lane; e < n; e += 64) {
                    const int p = w.a[off + e];
                    row[e] = p;
                    t.refs[p] = 1;
                }
                if (old >= 0) from = old, into = w.a[off];
            }
        }
        if (lane == 0) {
            if (from >= 0) add_to(t.refs + from, -1);
            w.src[b] = from;
            w.dst[b] = into;
            w.tail[b] = have & ((1 << P) - 1);
            if (done) t.len[b] = want;
            ok[b] = done;
        }
    }
    if (tid == 0) w.n[0] = t.n_seqs;
}

// Copies pages of all layers: pair i from src[i] to dst[i], of its first
// tail[i] positions (NULL: all) the blocks of 32 that they lie in. A block
// takes K or V (with its half of the scales) of one pair, layer and KV head.
struct Copy {
    uint8_t* base;
    size_t layer_bytes, code_bytes;
    int n_layers, n_kv, block_bytes, page_shift, n_pages;
    const int32_t *src, *dst, *tail, *count;
    int pairs;  // at most; count (if not NULL) holds how many there are
};
__device__ __forceinline__ void copy_item(const Copy& c, int64_t item) {
    const int part = int(item & 1);
    item >>= 1;
    const int head = int(item % c.n_kv);
    item /= c.n_kv;
    const int layer = int(item % c.n_layers);
    const int64_t i = item / c.n_layers;
    const int from = c.src[i], into = c.dst[i], pb = c.page_shift - 5;
    if (unsigned(from) >= unsigned(c.n_pages) || unsigned(into) >= unsigned(c.n_pages) || from == into) return;
    const int blocks = c.tail ? (c.tail[i] + 31) >> 5 : 1 << pb;
    uint8_t* codes = c.base + size_t(layer) * c.layer_bytes + part * c.code_bytes;
    const int64_t b0 = (int64_t(from) * c.n_kv + head) << pb, b1 = (int64_t(into) * c.n_kv + head) << pb;
    const uint4* p = reinterpret_cast<const uint4*>(codes + b0 * c.block_bytes);
    uint4* q = reinterpret_cast<uint4*>(codes + b1 * c.block_bytes);
    const int units = blocks * (c.block_bytes / 16);
    for (int u = threadIdx.x; u < units; u += 256) q[u] = p[u];
    // octets of a block's scales: [4][K 8, V 8]
    float* scales = reinterpret_cast<float*>(c.base + size_t(layer) * c.layer_bytes + 2 * c.code_bytes);
    for (int u = threadIdx.x; u < blocks * 32; u += 256) {
        const int at = (u >> 5) * kKvScales + ((u >> 3) & 3) * 16 + 8 * part + (u & 7);
        scales[b1 * kKvScales + at] = scales[b0 * kKvScales + at];
    }
}
__global__ void __launch_bounds__(256) k_pages_copy(Copy c) {
    const int64_t pairs = c.count ? min(*c.count, c.pairs) : c.pairs;
    const int64_t items = pairs * c.n_layers * c.n_kv * 2;
    for (int64_t i = blockIdx.x; i < items; i += gridDim.x) copy_item(c, i);
}

// Rows of the table trade places, `cols` columns of all of them to a block,
// through LDS, so that every row is read before any is written; the last block
// does the same for the lengths. Entries that a sequence does not hold are -1
// and count for nothing.
__global__ void __launch_bounds__(256) k_pages_fork(Tables t, const int32_t* __restrict__ parent, int cols) {
    extern __shared__ int32_t old[];
    const bool lens = blockIdx.x == gridDim.x - 1;
    const int c0 = lens ? 0 : blockIdx.x * cols, n = lens ? 1 : min(cols, t.max_pages - c0);
    int32_t* rows = lens ? t.len : t.pages + c0;
    const int64_t stride = lens ? 1 : t.max_pages;
    for (int i = threadIdx.x; i < t.n_seqs * n; i += 256) old[i] = rows[(i / n) * stride + i % n];
    __syncthreads();
    for (int i = threadIdx.x; i < t.n_seqs * n; i += 256) {
        const int b = i / n, p = parent[b];
        if (p == b || p < -1 || p >= t.n_seqs) continue;
        const int was = old[i], now = p < 0 ? (lens ? 0 : -1) : old[p * n + i % n];
        if (was == now) continue;
        rows[b * stride + i % n] = now;
        if (lens) continue;
        if (unsigned(now) < unsigned(t.n_pages)) add_to(t.refs + now, 1);
        if (unsigned(was) < unsigned(t.n_pages)) add_to(t.refs + was, -1);
    }
}

// Where every page of a compacted pool lies: the i-th held page from U on
// moves to the i-th free one below U. One block; src and dst list the moves,
// b the new place of the pages from U on.
__global__ void __launch_bounds__(kPlanThreads) k_pages_plan(Tables t, Work w, int32_t* __restrict__ used) {
    __shared__ int64_t lds[17];
    const int tid = threadIdx.x;
    int64_t mine = 0, U;
    for (int at = 4 * tid; at < t.n_pages; at += 4 * kPlanThreads) {
        const i4 r = four_refs(t.refs, at, t.n_pages);
        for (int k = 0; k < 4; ++k) mine += at + k < t.n_pages && r[k] > 0;
    }
    scan_before(mine, lds, U);
    int64_t holes = 0, moves = 0;
    for (int base = 0; base < t.n_pages; base += 4 * kPlanThreads) {
        const int at = base + 4 * tid;
        const i4 r = four_refs(t.refs, at, t.n_pages);
        int64_t n = 0;  // free pages below U, held ones from U on: no page is both
        for (int k = 0; k < 4; ++k) {
            const int p = at + k;
            if (p < t.n_pages) n += p < U ? int64_t(r[k] <= 0) << 32 : int64_t(r[k] > 0);
        }
        int64_t all;
        const int64_t before = scan_before(n, lds, all);
        int64_t h = holes + (before >> 32), m = moves + (before & 0xffffffff);
        for (int k = 0; k < 4; ++k) {
            const int p = at + k;
            if (p >= t.n_pages) break;
            if (p < U) {
                if (r[k] <= 0) w.dst[h++] = p;
            } else if (r[k] > 0) {
                w.src[m++] = p;
            }
        }
        holes += all >> 32;
        moves += all & 0xffffffff;
    }
    block_fence();
    for (int64_t i = U + tid; i < t.n_pages; i += kPlanThreads) w.b[i] = int(i);
    block_fence();
    for (int64_t i = tid; i < moves; i += kPlanThreads) {
        const int from = w.src[i], into = w.dst[i];
        w.b[from] = into;
        t.refs[into] = t.refs[from];
        t.refs[from] = 0;
    }
    if (tid == 0) {
        w.n[0] = int(moves);
        w.n[1] = int(U);
        if (used) *used = int(U);
    }
}
// The tables' entries follow.
__global__ void __launch_bounds__(256) k_pages_remap(Tables t, Work w) {
    const int U = w.n[1];
    const int64_t n = int64_t(t.n_seqs) * t.max_pages;
    for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < n; i += int64_t(gridDim.x) * 256) {
        const int p = t.pages[i];
        if (p >= U && p < t.n_pages) t.pages[i] = w.b[p];
    }
}

// Slot and position of every new token of a batch.
__global__ void __launch_bounds__(256) k_kv_slots(const int32_t* __restrict__ cu, const int32_t* __restrict__ kv_len,
                                                  const int32_t* __restrict__ pages, int n_seqs, int n_tokens,
                                                  int max_pages, int page_shift, int n_pages,
                                                  int64_t* __restrict__ slots, int32_t* __restrict__ pos) {
    const int t = blockIdx.x * 256 + threadIdx.x;
    if (t >= n_tokens) return;
    int lo = 0, hi = n_seqs;  // sequences whose rows begin at or before t
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (cu[mid] <= t)
            lo = mid + 1;
        else
            hi = mid;
    }
    const int b = lo - 1;
    int64_t slot = -1;
    int p = 0;
    if (b >= 0 && t < min(cu[b + 1], n_tokens)) {
        const int64_t q = int64_t(max(kv_len[b], 0)) - min(cu[b + 1], n_tokens) + t;
        p = int(q);
        if (q >= 0 && q >> page_shift < max_pages) {
            const int pg = pages[int64_t(b) * max_pages + (q >> page_shift)];
            if (unsigned(pg) < unsigned(n_pages)) slot = (int64_t(pg) << page_shift) + (q & ((1 << page_shift) - 1));
        }
    }
    slots[t] = slot;
    if (pos) pos[t] = p;
}

int launch_copy(const KvCache& c, const int32_t* src, const int32_t* dst, const int32_t* tail, const int32_t* count,
                int pairs, hipStream_t s) {
    Copy k{};
    k.base = c.base, k.layer_bytes = c.layer_bytes, k.code_bytes = c.code_bytes;
    k.n_layers = c.c.n_layers, k.n_kv = c.c.n_kv_heads, k.block_bytes = 32 * c.c.head_dim * kv_code_bytes(c.c.type);
    k.page_shift = c.layer(0).page_shift, k.n_pages = c.c.n_pages;
    k.src = src, k.dst = dst, k.tail = tail, k.count = count, k.pairs = pairs;
    const int64_t pages = std::min<int64_t>(int64_t(pairs) * k.n_layers, kCopyBlocks);  // no overflow below
    hipLaunchKernelGGL(k_pages_copy, dim3(unsigned(std::min<int64_t>(pages * k.n_kv * 2, kCopyBlocks))), dim3(256), 0, s, k);
    return int(hipGetLastError());
}

// The checks that the calls on a table share.
int check_tables(const char* what, uint64_t cache, const wv_kv_tables* t, KvCache& c, Tables& k, Work& w) {
    if (!kv_lookup(cache, c)) return rt_fail(WV_E_HANDLE, "%s: unknown cache %llu", what, (unsigned long long)cache);
    if (!t) return rt_fail(WV_E_ARG, "%s: nil tables", what);
    if (t->n_seqs < 0 || t->max_pages < 0 || t->n_seqs > kMaxSeqs)
        return rt_fail(WV_E_SHAPE, "%s: a table of %d sequences (at most %d) of %d pages", what, t->n_seqs, kMaxSeqs,
                       t->max_pages);
    if (int64_t(t->max_pages) * c.c.page_size >= int64_t(1) << 31)
        return rt_fail(WV_E_SHAPE, "%s: a table of %d pages of %d positions (2^31 and more)", what, t->max_pages,
                       c.c.page_size);
    if (t->n_seqs && ((t->max_pages && !t->d_pages) || !t->d_kv_len || !t->d_refs || !t->d_work))
        return rt_fail(WV_E_ARG, "%s: nil pages/kv_len/refs/work", what);
    k = {t->d_pages, t->d_kv_len, t->d_refs, t->n_seqs, t->max_pages, c.c.n_pages, c.layer(0).page_shift};
    w = work_of(t->d_work, t->n_seqs, c.c.n_pages);
    return WV_OK;
}

}  // namespace
}  // namespace wv

using namespace wv;

extern "C" {

int wv_kv_tables_work(uint64_t cache, int32_t n_seqs, int32_t max_pages, size_t* bytes) {
    KvCache c;
    Tables k;
    Work w;
    const wv_kv_tables t{n_seqs, max_pages, &n_seqs, &n_seqs, &n_seqs, &n_seqs};
    const int rc = check_tables("wv_kv_tables_work", cache, &t, c, k, w);
    if (rc) return rc;
    if (!bytes) return rt_fail(WV_E_ARG, "wv_kv_tables_work: nil bytes");
    *bytes = size_t(work_ints(n_seqs, c.c.n_pages)) * sizeof(int32_t);
    return WV_OK;
}

int wv_kv_fork_dev(uint64_t cache, const wv_kv_tables* tables, const int32_t* d_parent, void* stream) {
    KvCache c;
    Tables k;
    Work w;
    const int rc = check_tables("wv_kv_fork", cache, tables, c, k, w);
    if (rc || !k.n_seqs) return rc;
    if (!d_parent) return rt_fail(WV_E_ARG, "wv_kv_fork: nil parent");
    (void)hipSetDevice(c.device);
    int cols = 64;
    while (cols > 1 && cols * k.n_seqs > 4096) cols /= 2;
    const unsigned blocks = unsigned((int64_t(k.max_pages) + cols - 1) / cols) + 1;
    hipLaunchKernelGGL(k_pages_fork, dim3(blocks), dim3(256), unsigned(cols) * unsigned(k.n_seqs) * 4u,
                       rt_stream(stream, c.device), k, d_parent, cols);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? WV_OK : rt_hip_fail(e, "wv_kv_fork: kernel launch");
}

int wv_kv_resize_dev(uint64_t cache, const wv_kv_tables* tables, const int32_t* d_len, int32_t* d_ok, void* stream) {
    KvCache c;
    Tables k;
    Work w;
    const int rc = check_tables("wv_kv_resize", cache, tables, c, k, w);
    if (rc || !k.n_seqs) return rc;
    if (!d_len || !d_ok) return rt_fail(WV_E_ARG, "wv_kv_resize: nil len/ok");
    (void)hipSetDevice(c.device);
    hipStream_t s = rt_stream(stream, c.device);
    hipLaunchKernelGGL(k_pages_resize, dim3(1), dim3(kPlanThreads), 0, s, k, w, d_len, d_ok);
    const int e = launch_copy(c, w.src, w.dst, w.tail, nullptr, k.n_seqs, s);
    return e == hipSuccess ? WV_OK : rt_hip_fail(hipError_t(e), "wv_kv_resize: kernel launch");
}

int wv_kv_compact_dev(uint64_t cache, const wv_kv_tables* tables, int32_t* d_used, void* stream) {
    KvCache c;
    Tables k;
    Work w;
    const int rc = check_tables("wv_kv_compact", cache, tables, c, k, w);
    if (rc || !k.n_seqs) return rc;
    (void)hipSetDevice(c.device);
    hipStream_t s = rt_stream(stream, c.device);
    hipLaunchKernelGGL(k_pages_plan, dim3(1), dim3(kPlanThreads), 0, s, k, w, d_used);
    const int64_t entries = int64_t(k.n_seqs) * k.max_pages;
    if (entries)
        hipLaunchKernelGGL(k_pages_remap, dim3(unsigned(std::min<int64_t>((entries + 255) / 256, 2048))), dim3(256), 0,
                           s, k, w);
    const int e = launch_copy(c, w.src, w.dst, nullptr, w.n, k.n_pages / 2 + 1, s);
    return e == hipSuccess ? WV_OK : rt_hip_fail(hipError_t(e), "wv_kv_compact: kernel launch");
}

int wv_kv_copy_pages_dev(uint64_t cache, const int32_t* d_src, const int32_t* d_dst, int32_t n, void* stream) {
    KvCache c;
    if (!kv_lookup(cache, c))
        return rt_fail(WV_E_HANDLE, "wv_kv_copy_pages: unknown cache %llu", (unsigned long long)cache);
    if (n < 0) return rt_fail(WV_E_SHAPE, "wv_kv_copy_pages: negative count %d", n);
    if (!n) return WV_OK;
    if (!d_src || !d_dst) return rt_fail(WV_E_ARG, "wv_kv_copy_pages: nil src/dst");
    (void)hipSetDevice(c.device);
    const int e = launch_copy(c, d_src, d_dst, nullptr, nullptr, n, rt_stream(stream, c.device));
    return e == hipSuccess ? WV_OK : rt_hip_fail(hipError_t(e), "wv_kv_copy_pages: kernel launch");
}

int wv_kv_slots_dev(uint64_t cache, const wv_kv_batch* batch, int64_t* d_slots, int32_t* d_pos, void* stream) {
    KvCache c;
    if (!kv_lookup(cache, c)) return rt_fail(WV_E_HANDLE, "wv_kv_slots: unknown cache %llu", (unsigned long long)cache);
    if (!batch) return rt_fail(WV_E_ARG, "wv_kv_slots: nil batch");
    const wv_kv_batch& b = *batch;
    if (b.n_seqs < 0 || b.n_tokens < 0 || b.max_pages < 0 || b.n_tokens > 1 << 28 || b.n_seqs > 1 << 24)
        return rt_fail(WV_E_SHAPE, "wv_kv_slots: %d sequences, %d tokens, %d pages", b.n_seqs, b.n_tokens, b.max_pages);
    if (int64_t(b.max_pages) * c.c.page_size >= int64_t(1) << 31)
        return rt_fail(WV_E_SHAPE, "wv_kv_slots: a table of %d pages of %d positions (2^31 and more)", b.max_pages,
                       c.c.page_size);
    if (!b.n_tokens) return WV_OK;
    if (!d_slots || (b.n_seqs && (!b.d_cu_q || !b.d_kv_len || (b.max_pages && !b.d_pages))))
        return rt_fail(WV_E_ARG, "wv_kv_slots: nil slots/cu_q/kv_len/pages");
    (void)hipSetDevice(c.device);
    hipLaunchKernelGGL(k_kv_slots, dim3(unsigned((b.n_tokens + 255) / 256)), dim3(256), 0, rt_stream(stream, c.device),
                       b.d_cu_q, b.d_kv_len, b.d_pages, b.n_seqs, b.n_tokens, b.max_pages, c.layer(0).page_shift,
                       c.c.n_pages, d_slots, d_pos);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? WV_OK : rt_hip_fail(e, "wv_kv_slots: kernel launch");
}

}  // extern "C"
