// kv_pages.hip — who holds which page of a paged KV cache: sequences forked,
// resized (pages taken and given back, a shared last page copied before it is
// written), the pool compacted, and the slots of a batch's new tokens. All of
// it on the device, from tables that lie there, so a decode loop (or a graph
// of one) needs no host in between.
#include <algorithm>

#include "kv.h"
#include "rt_internal.h"
#include "wave_ops.h"

namespace wv {
namespace {

constexpr int kMaxSeqs = 16384;    // of a table: one column of it lies in LDS
constexpr int kPlanThreads = 1024;
constexpr int kCopyBlocks = 4096;  // of a copy, twice what runs at once (2048: up to 8% slower; 8192 the same)

typedef int32_t i4 __attribute__((ext_vector_type(4)));

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

// A count that other threads of this block may have changed by atomics: past the L1, which does not see those.
__device__ __forceinline__ int32_t ld_now(const int32_t* p) {
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void add_to(int32_t* p, int32_t v) {
    __hip_atomic_fetch_add(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Sum of v over the threads before this one, and over all of them. A wave's sums are held at 2^32 - 1, which no pool
// has pages for. `lds`: 32 values, two turns' worth, so that one barrier does.
__device__ __forceinline__ int64_t scan_before(uint32_t v, uint32_t* lds, int& turn, int64_t& all) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t x = v;
    auto add = [&](int o) { x = __builtin_elementwise_add_sat(x, uint32_t(o)); };
    add(dpp_i<kDppRowShr1>(0, int(x)));
    add(dpp_i<kDppRowShr2>(0, int(x)));
    add(dpp_i<kDppRowShr4, 0xf, 0xe>(0, int(x)));
    add(dpp_i<kDppRowShr8, 0xf, 0xc>(0, int(x)));
    add(dpp_i<kDppRowBcast15, 0xa>(0, int(x)));
    add(dpp_i<kDppRowBcast31, 0xc>(0, int(x)));
    uint32_t* l = lds + 16 * (turn++ & 1);
    if (lane == 63) l[wave] = x;
    __syncthreads();
    int64_t before = int64_t(x) - v;
    all = 0;
#pragma unroll
    for (int w = 0; w < kPlanThreads / 64; ++w) {
        if (w < wave) before += l[w];
        all += l[w];
    }
    return before;
}

// Four counts from `at` on; those past the pool read as held.
__device__ __forceinline__ i4 four_refs(const int32_t* refs, int at, int n) {
    i4 x = {1, 1, 1, 1};
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if (at + k < n) x[k] = ld_now(refs + at + k);
    return x;
}

__device__ __forceinline__ int pages_of(int len, int shift) { return (len + (1 << shift) - 1) >> shift; }

// f(sequence's value, entry) for the entries 0 .. n - 1 of each lane's sequence: a few by the lane itself, the rest
// by the whole wave, one sequence after the other.
constexpr int kOwnEntries = 4;
template <class F>
__device__ __forceinline__ void for_entries(int n, int lane_value, F f) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int e = 0; e < kOwnEntries; ++e)
        if (e < n) f(lane_value, e);
    for (uint64_t m = __ballot(n > kOwnEntries); m; m &= m - 1) {
        const int w = __builtin_ctzll(m);
        const int k = __builtin_amdgcn_readlane(n, w), v = __builtin_amdgcn_readlane(lane_value, w);
        for (int e = kOwnEntries + lane; e < k; e += 64) f(v, e);
    }
}

// The whole of resize but the copies, by one block: its steps depend on each
// other, and a table's entries and the pool's counts are a few 10 KB. No other
// block touches them, so a barrier orders them (its threads' stores and atomics
// are in the L2 by then), and no step needs a fence for the whole device, which
// costs some 3 us each. A thread takes a sequence. 256 sequences of 65 pages in a
// pool of 17000 6.6 us: a chain of steps, each a load's latency.
__global__ void __launch_bounds__(kPlanThreads) k_pages_resize(Tables t, Work w, const int32_t* __restrict__ to,
                                                               int32_t* __restrict__ ok) {
    __shared__ uint32_t lds[32];
    int turn = 0;
    const int tid = threadIdx.x, P = t.page_shift;
    const int width = t.max_pages << P;  // below 2^31
    auto length = [&](int b) { return b < t.n_seqs ? min(max(t.len[b], 0), width) : 0; };
    auto target = [&](int b) { return b < t.n_seqs ? max(to[b], 0) : 0; };
    // The page that a growing sequence's next position lies in, if it has rows already.
    auto last_page = [&](int b, int have, int want) {
        if (want <= have || want > width || !(have & ((1 << P) - 1))) return -1;
        const int p = t.pages[int64_t(b) * t.max_pages + (have >> P)];
        return unsigned(p) < unsigned(t.n_pages) ? p : -1;
    };

    for (int b0 = 0; b0 < t.n_seqs; b0 += kPlanThreads) {
        const int b = b0 + tid, have = length(b), want = target(b);
        // those that shrink give their pages back
        const int keep = pages_of(want, P);
        for_entries(want < have ? pages_of(have, P) - keep : 0, b, [&](int s, int e) {
            // the wave's other lanes know the sequence alone
            int32_t* entry = t.pages + int64_t(s) * t.max_pages + pages_of(target(s), P) + e;
            const int p = *entry;
            if (unsigned(p) < unsigned(t.n_pages)) add_to(t.refs + p, -1);
            *entry = -1;
        });
        if (const int p = last_page(b, have, want); p >= 0) w.a[p] = 0, w.b[p] = -1;
    }
    __syncthreads();
    // how many sequences grow out of a page, and the last of them
    for (int b = tid; b < t.n_seqs; b += kPlanThreads)
        if (const int p = last_page(b, length(b), target(b)); p >= 0) {
            add_to(w.a + p, 1);
            __hip_atomic_fetch_max(w.b + p, b, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
    __syncthreads();
    // pages that each needs, and where in the list of free ones they begin
    int64_t total = 0;
    for (int b0 = 0; b0 < t.n_seqs; b0 += kPlanThreads) {
        const int b = b0 + tid, have = length(b), want = target(b), p = last_page(b, have, want);
        const bool grows = want > have && want <= width;
        int copy = -1;
        if (p >= 0) {
            const int refs = ld_now(t.refs + p), out = ld_now(w.a + p), last = ld_now(w.b + p);
            if (refs > 1 && !(out == refs && last == b)) copy = p;
        }
        int64_t all;
        const int64_t off =
            total + scan_before(grows ? uint32_t(pages_of(want, P) - pages_of(have, P) + (copy >= 0)) : 0u, lds, turn, all);
        if (b < t.n_seqs) {
            w.src[b] = copy;
            w.off[b] = grows ? int(min(off, int64_t(t.n_pages) + 1)) : -1;  // past the pool none is served, wherever
        }
        total += all;
    }
    // the lowest free pages, as many as are needed
    const int most = int(min(total, int64_t(t.n_pages)));
    int found = 0;
    __syncthreads();  // w.a counted
    for (int base = 0; base < t.n_pages && found < most; base += 4 * kPlanThreads) {
        const int at = base + 4 * tid;
        const i4 r = four_refs(t.refs, at, t.n_pages);
        int64_t all;
        int64_t i = found + scan_before((r[0] <= 0) + (r[1] <= 0) + (r[2] <= 0) + (r[3] <= 0), lds, turn, all);
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (r[k] <= 0 && i++ < most) w.a[i - 1] = at + k;
        found += int(all);
    }
    found = min(found, most);
    __syncthreads();
    // those that grow take them
    for (int b0 = 0; b0 < t.n_seqs; b0 += kPlanThreads) {
        const int b = b0 + tid, have = length(b), want = target(b);
        const int off = b < t.n_seqs ? w.off[b] : -1, old = b < t.n_seqs ? w.src[b] : -1;
        const int n = off >= 0 ? pages_of(want, P) - pages_of(have, P) + (old >= 0) : 0;
        const bool serve = off >= 0 && int64_t(off) + n <= found;
        for_entries(serve ? n : 0, b, [&](int s, int e) {
            const int p = w.a[w.off[s] + e];
            t.pages[int64_t(s) * t.max_pages + pages_of(length(s), P) - (w.src[s] >= 0) + e] = p;
            t.refs[p] = 1;
        });
        const int into = serve && old >= 0 ? w.a[off] : -1;
        // every lane's entries are written (the wave's lanes read its sequences' lengths and copies until here)
        __builtin_amdgcn_wave_barrier();
        if (b < t.n_seqs) {
            if (into >= 0) add_to(t.refs + old, -1);
            w.src[b] = into >= 0 ? old : -1;
            w.dst[b] = into;
            w.tail[b] = have & ((1 << P) - 1);
            const bool done = serve || want <= have;
            if (done) t.len[b] = want;
            ok[b] = done;
        }
    }
}

// Copies pages of all layers: pair i from src[i] to dst[i], of its first
// tail[i] positions (NULL: all) what holds them: whole blocks of 32, of the
// last one a unit's first keys (K) and the octets that they lie in (V, scales).
// A block takes K or V (with its half of the scales) of one pair and KV head,
// in one group of layers. Bound by the bytes: 64 whole pages of 64 fp16
// positions, 4 layers of 8 heads of 128, 69 MB, 18.6 us, 512 214 us, 5.2 TB/s read
// and written (a large copy: 5.1); none of 256 3.9 us.
struct Copy {
    uint8_t* base;
    size_t layer_bytes, code_bytes;
    int n_layers, n_kv, block_bytes, page_shift, n_pages;
    int groups;  // of the layers
    const int32_t *src, *dst, *tail, *count;
    int pairs;  // at most; count (if not NULL) holds how many there are
};
__device__ __forceinline__ void copy_item(const Copy& c, int64_t item) {
    const int part = int(item & 1);
    item >>= 1;
    const int head = int(item % c.n_kv);
    item /= c.n_kv;
    const int group = int(item % c.groups);
    const int64_t i = item / c.groups;
    const int from = c.src[i], into = c.dst[i], pb = c.page_shift - 5;
    if (unsigned(from) >= unsigned(c.n_pages) || unsigned(into) >= unsigned(c.n_pages) || from == into) return;
    const int keys = c.tail ? c.tail[i] : 1 << c.page_shift, whole = keys >> 5, rest = keys & 31;
    const int64_t b0 = (int64_t(from) * c.n_kv + head) << pb, b1 = (int64_t(into) * c.n_kv + head) << pb;
    const int bu = c.block_bytes / 16, units = whole * bu;
    for (int layer = group; layer < c.n_layers; layer += c.groups) {
        uint8_t* codes = c.base + size_t(layer) * c.layer_bytes + part * c.code_bytes;
        const uint4* p = reinterpret_cast<const uint4*>(codes + b0 * c.block_bytes);
        uint4* q = reinterpret_cast<uint4*>(codes + b1 * c.block_bytes);
        for (int u = threadIdx.x; u < units; u += 256) q[u] = p[u];
        // octet o = 2a + b of a block holds no key before 16a + 4b
        auto octet_used = [&](int o) { return 16 * (o >> 1) + 4 * (o & 1) < rest; };
        if (rest)
            for (int u = threadIdx.x; u < bu; u += 256)
                if (part ? octet_used(4 * u / bu) : (u & 31) < rest) q[units + u] = p[units + u];
        float* scales = reinterpret_cast<float*>(c.base + size_t(layer) * c.layer_bytes + 2 * c.code_bytes);
        for (int u = threadIdx.x; u < (whole + (rest > 0)) * 32; u += 256) {
            const int o = (u >> 3) & 3, at = (u >> 5) * kKvScales + o * 16 + 8 * part + (u & 7);
            if ((u >> 5) < whole || octet_used(o)) scales[b1 * kKvScales + at] = scales[b0 * kKvScales + at];
        }
    }
}
__global__ void __launch_bounds__(256) k_pages_copy(Copy c) {
    const int64_t pairs = c.count ? min(*c.count, c.pairs) : c.pairs;
    const int64_t items = pairs * c.groups * c.n_kv * 2;
    for (int64_t i = blockIdx.x; i < items; i += gridDim.x) copy_item(c, i);
}

// Rows of the table trade places, 2^shift columns of all of them to a block,
// through LDS, so that every row is read before any is written; the last block
// does the same for the lengths. Entries that a sequence does not hold are -1
// and count for nothing. Bound by the latency of its three loads in a row and
// the counts' atomics: 8 sequences 2.3 us (a launch), 64 of 1024 pages 3.5, 1024
// of 512 8.8 (blocks of 256 threads: 5.2 and 15.8).
__global__ void __launch_bounds__(1024) k_pages_fork(Tables t, const int32_t* __restrict__ parent, int shift) {
    extern __shared__ int32_t old[];
    const bool lens = blockIdx.x == gridDim.x - 1;
    if (lens) shift = 0;
    const int c0 = lens ? 0 : blockIdx.x << shift, n = lens ? 1 : min(1 << shift, t.max_pages - c0);
    int32_t* rows = lens ? t.len : t.pages + c0;
    const int64_t stride = lens ? 1 : t.max_pages;
    const int c = threadIdx.x & ((1 << shift) - 1), step = int(blockDim.x) >> shift;
    for (int b = threadIdx.x >> shift; b < t.n_seqs; b += step) old[(b << shift) + c] = c < n ? rows[b * stride + c] : -1;
    __syncthreads();
    for (int b = threadIdx.x >> shift; b < t.n_seqs; b += step) {
        const int p = parent[b];
        if (p == b || p < -1 || p >= t.n_seqs) continue;
        const int was = old[(b << shift) + c], now = p < 0 ? (lens ? 0 : -1) : old[(p << shift) + c];
        if (was == now || c >= n) continue;
        rows[b * stride + c] = now;
        if (lens) continue;
        if (unsigned(now) < unsigned(t.n_pages)) add_to(t.refs + now, 1);
        if (unsigned(was) < unsigned(t.n_pages)) add_to(t.refs + was, -1);
    }
}

// Where every page of a compacted pool lies: the i-th held page from U on
// moves to the i-th free one below U. One block; src and dst list the moves,
// b the new place of the pages from U on.
__global__ void __launch_bounds__(kPlanThreads) k_pages_plan(Tables t, Work w, int32_t* __restrict__ used) {
    __shared__ uint32_t lds[32];
    int turn = 0;
    const int tid = threadIdx.x;
    uint32_t mine = 0;
    for (int at = 4 * tid; at < t.n_pages; at += 4 * kPlanThreads) {
        const i4 r = four_refs(t.refs, at, t.n_pages);
#pragma unroll
        for (int k = 0; k < 4; ++k) mine += at + k < t.n_pages && r[k] > 0;
    }
    int64_t U, all;
    scan_before(mine, lds, turn, U);
    int64_t holes = 0, moves = 0;
    for (int base = 0; base < t.n_pages; base += 4 * kPlanThreads) {
        const int at = base + 4 * tid;
        const i4 r = four_refs(t.refs, at, t.n_pages);
        uint32_t n = 0;  // free pages below U in the upper half, held ones from U on in the lower: 4096 of them at most
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int p = at + k;
            if (p < t.n_pages) n += p < U ? uint32_t(r[k] <= 0) << 16 : uint32_t(r[k] > 0);
        }
        const int64_t before = scan_before(n, lds, turn, all);
        int64_t h = holes + (before >> 16), m = moves + (before & 0xffff);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int p = at + k;
            if (p >= t.n_pages) continue;
            if (p < U) {
                if (r[k] <= 0) w.dst[h++] = p;
            } else {
                w.b[p] = p;
                if (r[k] > 0) w.src[m++] = p;
            }
        }
        holes += all >> 16;
        moves += all & 0xffff;
    }
    __syncthreads();
    for (int64_t i = tid; i < moves; i += kPlanThreads) {
        const int from = w.src[i], into = w.dst[i];
        w.b[from] = into;
        t.refs[into] = ld_now(t.refs + from);
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

// Slot and position of every new token of a batch. A block has the sequences'
// first rows in LDS (of more than 4096 every 2nd, 4th .. of them) and searches there. ok (may be null): a sequence
// with a 0 was refused its new positions. Its rows would fall on the last ones that it holds, and maybe others too.
constexpr int kSlotSeqs = 4096;
__global__ void __launch_bounds__(256) k_kv_slots(const int32_t* __restrict__ cu, const int32_t* __restrict__ kv_len,
                                                  const int32_t* __restrict__ pages, int n_seqs, int n_tokens,
                                                  int max_pages, int page_shift, int n_pages, int step,
                                                  const int32_t* __restrict__ ok, int64_t* __restrict__ slots,
                                                  int32_t* __restrict__ pos) {
    __shared__ int32_t first[kSlotSeqs];
    const int t = blockIdx.x * 256 + threadIdx.x, n = (n_seqs + (1 << step) - 1) >> step;
    for (int i = threadIdx.x; i < n; i += 256) first[i] = cu[i << step];
    __syncthreads();
    if (t >= n_tokens) return;
    int lo = 0, hi = n;  // how many of them begin at or before t
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (first[mid] <= t)
            lo = mid + 1;
        else
            hi = mid;
    }
    lo = max(lo - 1, 0) << step, hi = min(lo + (1 << step), n_seqs);
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if ((step ? cu[mid] : first[mid]) <= t)
            lo = mid + 1;
        else
            hi = mid;
    }
    const int b = lo - 1;
    int64_t slot = -1;
    int p = 0;
    if (b >= 0) {
        const int end = min(cu[b + 1], n_tokens);
        if (t < end && (!ok || ok[b])) {
            const int64_t q = int64_t(max(kv_len[b], 0)) - end + t;
            p = int(q);
            if (q >= 0 && q >> page_shift < max_pages) {
                const int pg = pages[int64_t(b) * max_pages + (q >> page_shift)];
                if (unsigned(pg) < unsigned(n_pages))
                    slot = (int64_t(pg) << page_shift) + (q & ((1 << page_shift) - 1));
            }
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
    // a layer to a block while there are few pairs, all layers where there are many (one page of 32 layers 4.4 / 28.8 us,
    // 8 18.6 / 51, 64 221 / 220, 200 710 / 696)
    const int64_t items = int64_t(pairs) * k.n_kv * 2;
    k.groups = int(std::max<int64_t>(1, std::min<int64_t>(k.n_layers, kCopyBlocks / items)));
    hipLaunchKernelGGL(k_pages_copy, dim3(unsigned(std::min<int64_t>(items * k.groups, kCopyBlocks))), dim3(256), 0, s, k);
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

// wv_kv_slots_dev, and with ok wv_kv_slots_served_dev.
int slots_of(const char* what, uint64_t cache, const wv_kv_batch* batch, const int32_t* ok, int64_t* d_slots,
             int32_t* d_pos, void* stream) {
    KvCache c;
    if (!kv_lookup(cache, c)) return rt_fail(WV_E_HANDLE, "%s: unknown cache %llu", what, (unsigned long long)cache);
    if (!batch) return rt_fail(WV_E_ARG, "%s: nil batch", what);
    const wv_kv_batch& b = *batch;
    if (b.n_seqs < 0 || b.n_tokens < 0 || b.max_pages < 0 || b.n_tokens > 1 << 28 || b.n_seqs > 1 << 24)
        return rt_fail(WV_E_SHAPE, "%s: %d sequences, %d tokens, %d pages", what, b.n_seqs, b.n_tokens, b.max_pages);
    if (int64_t(b.max_pages) * c.c.page_size >= int64_t(1) << 31)
        return rt_fail(WV_E_SHAPE, "%s: a table of %d pages of %d positions (2^31 and more)", what, b.max_pages,
                       c.c.page_size);
    if (!b.n_tokens) return WV_OK;
    if (!d_slots || (b.n_seqs && (!b.d_cu_q || !b.d_kv_len || (b.max_pages && !b.d_pages))))
        return rt_fail(WV_E_ARG, "%s: nil slots/cu_q/kv_len/pages", what);
    (void)hipSetDevice(c.device);
    int step = 0;
    while ((int64_t(b.n_seqs) + (1 << step) - 1) >> step > kSlotSeqs) ++step;
    hipLaunchKernelGGL(k_kv_slots, dim3(unsigned((b.n_tokens + 255) / 256)), dim3(256), 0, rt_stream(stream, c.device),
                       b.d_cu_q, b.d_kv_len, b.d_pages, b.n_seqs, b.n_tokens, b.max_pages, c.layer(0).page_shift,
                       c.c.n_pages, step, ok, d_slots, d_pos);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? WV_OK : rt_hip_fail(e, what);
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
    // An entry a thread, but four before fewer than 4 columns stay together (of 1 / 2 / 4 / 8 / 16 columns: 64 sequences
    // of 1024 pages 8.6 / 5.9 / 4.4 / 3.9 / 3.5 us, 256 9.0 / 6.1 / 5.0 / 4.8 / 5.8, 1024 of 512 12.3 / 9.1 / 8.8 / 10.1).
    int shift = 5;
    while (shift > 0 && (k.n_seqs << shift) > (shift > 2 ? 1024 : 4096)) --shift;
    const unsigned blocks = unsigned((int64_t(k.max_pages) + (1 << shift) - 1) >> shift) + 1;
    const unsigned threads = unsigned(std::min(1024, ((k.n_seqs << shift) + 63) & ~63));
    hipLaunchKernelGGL(k_pages_fork, dim3(blocks), dim3(threads), unsigned(k.n_seqs) * 4u << shift,
                       rt_stream(stream, c.device), k, d_parent, shift);
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
    return slots_of("wv_kv_slots", cache, batch, nullptr, d_slots, d_pos, stream);
}

int wv_kv_slots_served_dev(uint64_t cache, const wv_kv_batch* batch, const int32_t* d_ok, int64_t* d_slots,
                           int32_t* d_pos, void* stream) {
    if (batch && batch->n_seqs > 0 && batch->n_tokens > 0 && !d_ok)
        return rt_fail(WV_E_ARG, "wv_kv_slots_served: nil ok");
    return slots_of("wv_kv_slots_served", cache, batch, d_ok, d_slots, d_pos, stream);
}

}  // extern "C"
