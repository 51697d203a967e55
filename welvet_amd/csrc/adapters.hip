// adapters.hip — low-rank adapters of many requests beside a shared
// projection: y_t = base_t + s_a B_a (A_a x_t), a the adapter of t's sequence.
//
// Two launches: h = A x in ranges of the columns (so that one token's rows
// still fill the GPU), whose sums meet when B h reads them, in order of the
// ranges. A and B stay 16-bit, x, h and all sums are f32.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <mutex>
#include <new>
#include <unordered_map>
#include <vector>

#include "../../include/welvet_hip.h"
#include "rt_internal.h"
#include "wave_ops.h"

namespace wv {
namespace {

constexpr int kMaxSets = 4;      // of a call
constexpr int kMaxRank = 256;
constexpr int kChunk = 512;      // columns that a wave takes at a time, 8 to a lane
constexpr int kMaxRanges = 32;   // of the columns

struct Set {
    wv_adapters_config c{};
    int device = 0;
    int R = 0, C = 0;         // ranks and columns as stored: multiples of 16 and 64, zeros behind the adapter's own
    uint16_t* a = nullptr;    // [n_adapters][R][C]
    uint16_t* b = nullptr;    // [n_adapters][rows][R]
    int32_t* rank = nullptr;  // [n_adapters], 0: unset
    float* scale = nullptr;   // [n_adapters]
};
std::mutex g_mu;
std::unordered_map<uint64_t, Set> g_sets;
uint64_t g_next = 1;

bool set_lookup(uint64_t h, Set& out) {
    std::lock_guard<std::mutex> lk(g_mu);
    auto it = g_sets.find(h);
    if (it == g_sets.end()) return false;
    out = it->second;
    return true;
}

typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));

// One set of a call as the kernels see it.
struct SetArgs {
    const uint16_t *a, *b;
    const int32_t* rank;
    const float* scale;
    const float* base;
    float* y;
    float* h;  // [ranges][n_tokens][R]
    int64_t ys, bs;
    int rows, R, C, n_adapters;
};
struct Args {
    SetArgs set[kMaxSets];
    const float* x;
    const int32_t *cu, *which;
    int64_t xs;
    int cols, n_seqs, n_tokens, ranges, range;  // range: columns of one, a multiple of kChunk
};

template <int TYPE>
__device__ __forceinline__ float low(uint32_t w) {
    return TYPE == WV_ADAPTER_BF16 ? __uint_as_float(w << 16) : float(__builtin_bit_cast(_Float16, uint16_t(w)));
}
template <int TYPE>
__device__ __forceinline__ float high(uint32_t w) {
    return TYPE == WV_ADAPTER_BF16 ? __uint_as_float(w & 0xffff0000) : float(__builtin_bit_cast(_Float16, uint16_t(w >> 16)));
}

// The sequence of row t, -1 behind the last one: 64 at a time, after a look at sequence t itself, which it is
// wherever every sequence has one token.
__device__ __forceinline__ int sequence_of(const Args& a, int t) {
    if (t < a.n_seqs && a.cu[t] == t && a.cu[t + 1] == t + 1) return t;
    const int lane = threadIdx.x & 63;
    for (int s0 = 0; s0 < a.n_seqs; s0 += 64) {
        const int s = s0 + lane;
        const int end = s < a.n_seqs ? a.cu[s + 1] : INT32_MAX;
        const uint64_t behind = __ballot(end > t);
        if (!behind) continue;
        const int b = s0 + __builtin_ctzll(behind);
        return b < a.n_seqs && a.cu[b] <= t ? b : -1;
    }
    return -1;
}

// A token's h: a wave takes every fourth group of ranks, a lane 8 columns at a time.
template <int TYPE>
__global__ void __launch_bounds__(256) k_adapt_down(Args a) {
    const int t = blockIdx.y, range = blockIdx.x;
    const SetArgs& s = a.set[blockIdx.z];
    const int b = sequence_of(a, t);
    if (b < 0) return;
    const int id = a.which[b];
    if (unsigned(id) >= unsigned(s.n_adapters)) return;
    const int rank = s.rank[id];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint16_t* A = s.a + int64_t(id) * s.R * s.C;
    const float* x = a.x + int64_t(t) * a.xs;
    float* h = s.h + (int64_t(range) * a.n_tokens + t) * s.R;
    const int c0 = range * a.range, c1 = min(c0 + a.range, a.cols);
    for (int r0 = 4 * wave; r0 < rank; r0 += 16) {
        float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int c = c0 + 8 * lane; c < c1; c += kChunk) {
            float v[8];
            if (c + 8 <= a.cols) {
                const f4 lo = *reinterpret_cast<const f4*>(x + c), hi = *reinterpret_cast<const f4*>(x + c + 4);
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = lo[i], v[4 + i] = hi[i];
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = c + i < a.cols ? x[c + i] : 0.0f;
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint4 w = *reinterpret_cast<const uint4*>(A + int64_t(r0 + k) * s.C + c);
                const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    sum[k] = fmaf(low<TYPE>(u[i]), v[2 * i], sum[k]);
                    sum[k] = fmaf(high<TYPE>(u[i]), v[2 * i + 1], sum[k]);
                }
            }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float y = wave_total(sum[k]);
            if (lane == 0 && r0 + k < rank) h[r0 + k] = y;
        }
    }
}

// y of 256 rows of one token.
template <int TYPE>
__global__ void __launch_bounds__(256) k_adapt_up(Args a) {
    __shared__ float h[kMaxRank];
    const int t = blockIdx.y, o = blockIdx.x * 256 + threadIdx.x;
    const SetArgs& s = a.set[blockIdx.z];
    if (blockIdx.x * 256 >= s.rows) return;
    const int b = sequence_of(a, t);
    if (b < 0) return;
    const int id = a.which[b];
    const int rank = unsigned(id) < unsigned(s.n_adapters) ? s.rank[id] : 0;
    for (int r = threadIdx.x; r < s.R && rank; r += 256) {
        float x = 0.0f;
        if (r < rank)
            for (int i = 0; i < a.ranges; ++i) x += s.h[(int64_t(i) * a.n_tokens + t) * s.R + r];
        h[r] = x * s.scale[id];
    }
    __syncthreads();
    if (o >= s.rows) return;
    const float* base = s.base + t * s.bs + o;
    float* y = s.y + t * s.ys + o;
    if (!rank) {
        if (base != y) *y = *base;
        return;
    }
    const uint16_t* B = s.b + (int64_t(id) * s.rows + o) * s.R;
    float sum = 0.0f;
    for (int r = 0; r < rank; r += 8) {
        const uint4 w = *reinterpret_cast<const uint4*>(B + r);
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            sum = fmaf(low<TYPE>(u[i]), h[r + 2 * i], sum);
            sum = fmaf(high<TYPE>(u[i]), h[r + 2 * i + 1], sum);
        }
    }
    *y = *base + sum;
}

// Into how many ranges the columns are cut: about eight blocks a CU, and ranges of whole chunks.
int adapt_ranges(int cols, int n_tokens, int n_sets, int& range) {
    const int chunks = (cols + kChunk - 1) / kChunk;
    const int want = std::max<int>(1, std::min({int(2048 / std::min<int64_t>(int64_t(n_tokens) * n_sets, 2048)), chunks, kMaxRanges}));
    const int each = (chunks + want - 1) / want;
    range = each * kChunk;
    return (chunks + each - 1) / each;
}

template <int TYPE>
int launch_adapters(const Args& a, int n_sets, hipStream_t s) {
    int rows = 0;
    for (int i = 0; i < n_sets; ++i) rows = std::max(rows, a.set[i].rows);
    hipLaunchKernelGGL(k_adapt_down<TYPE>, dim3(unsigned(a.ranges), unsigned(a.n_tokens), unsigned(n_sets)), dim3(256),
                       0, s, a);
    hipLaunchKernelGGL(k_adapt_up<TYPE>, dim3(unsigned((rows + 255) / 256), unsigned(a.n_tokens), unsigned(n_sets)),
                       dim3(256), 0, s, a);
    return int(hipGetLastError());
}

}  // namespace
}  // namespace wv

using namespace wv;

namespace {

// The checks of a call: its sets (all over as many columns, of one type and device) and sizes.
int check_call(const char* what, const wv_adapter_batch* b, const wv_adapter_rows* sets, int32_t n_sets, Set* s) {
    if (!b || !sets) return rt_fail(WV_E_ARG, "%s: nil batch/sets", what);
    if (n_sets < 1 || n_sets > kMaxSets) return rt_fail(WV_E_SHAPE, "%s: %d sets (1 to %d)", what, n_sets, kMaxSets);
    for (int i = 0; i < n_sets; ++i) {
        if (!set_lookup(sets[i].adapters, s[i]))
            return rt_fail(WV_E_HANDLE, "%s: unknown adapters %llu", what, (unsigned long long)sets[i].adapters);
        if (s[i].c.cols != s[0].c.cols || s[i].c.type != s[0].c.type || s[i].device != s[0].device)
            return rt_fail(WV_E_SHAPE, "%s: sets of %d and %d columns, types %d and %d, devices %d and %d", what,
                           s[0].c.cols, s[i].c.cols, s[0].c.type, s[i].c.type, s[0].device, s[i].device);
    }
    if (b->n_seqs < 0 || b->n_tokens < 0 || b->max_q < 0 || b->n_tokens > 65535 || b->n_seqs > 1 << 24)
        return rt_fail(WV_E_SHAPE, "%s: %d sequences, %d tokens (at most 65535), max_q %d", what, b->n_seqs, b->n_tokens,
                       b->max_q);
    return WV_OK;
}

size_t scratch_floats(const Set* s, int n_sets, int n_tokens, int ranges) {
    size_t n = 0;
    for (int i = 0; i < n_sets; ++i) n += size_t(ranges) * size_t(n_tokens) * size_t(s[i].R);
    return n;
}

}  // namespace

extern "C" {

int wv_adapters_create(const wv_adapters_config* cfg, uint64_t* adapters) {
    if (!cfg || !adapters) return rt_fail(WV_E_ARG, "wv_adapters_create: nil argument");
    const wv_adapters_config& c = *cfg;
    if (c.rows <= 0 || c.cols <= 0 || c.n_adapters <= 0)
        return rt_fail(WV_E_SHAPE, "wv_adapters_create: non-positive dimension");
    if (c.rows > 1 << 24 || c.cols > 1 << 24 || c.n_adapters > 1 << 20)
        return rt_fail(WV_E_SHAPE, "wv_adapters_create: %d x %d (at most 2^24), %d adapters (at most 2^20)", c.rows,
                       c.cols, c.n_adapters);
    if (c.max_rank < 1 || c.max_rank > kMaxRank)
        return rt_fail(WV_E_SHAPE, "wv_adapters_create: max_rank %d (1 to %d)", c.max_rank, kMaxRank);
    if (c.type != WV_ADAPTER_F16 && c.type != WV_ADAPTER_BF16)
        return rt_fail(WV_E_FORMAT, "wv_adapters_create: type %d", c.type);
    int rc = rt_ensure_init();
    if (rc) return rc;
    Set s;
    s.c = c;
    s.device = rt_current_device();
    s.R = (c.max_rank + 15) / 16 * 16;
    s.C = (c.cols + 63) / 64 * 64;
    const size_t n = size_t(c.n_adapters), na = n * s.R * s.C * 2, nb = n * c.rows * s.R * 2;
    // one allocation: A, B (both multiples of 16 bytes), ranks, scales
    uint8_t* p = nullptr;
    hipError_t e = hipMalloc(reinterpret_cast<void**>(&p), na + nb + n * 8);
    if (e != hipSuccess) {
        (void)hipGetLastError();
        return rt_hip_fail(e, "wv_adapters_create: weights");
    }
    s.a = reinterpret_cast<uint16_t*>(p);
    s.b = reinterpret_cast<uint16_t*>(p + na);
    s.rank = reinterpret_cast<int32_t*>(p + na + nb);
    s.scale = reinterpret_cast<float*>(s.rank + n);
    hipStream_t st = rt_stream(nullptr, s.device);
    e = hipMemsetAsync(s.rank, 0, n * 8, st);
    if (e == hipSuccess) e = hipStreamSynchronize(st);
    if (e != hipSuccess) {
        (void)hipFree(p);
        return rt_hip_fail(e, "wv_adapters_create: clear");
    }
    try {
        std::lock_guard<std::mutex> lk(g_mu);
        g_sets[g_next] = s;
        *adapters = g_next++;
    } catch (const std::bad_alloc&) {
        (void)hipFree(p);
        return rt_fail(WV_E_OOM, "wv_adapters_create: host memory exhausted");
    }
    return WV_OK;
}

int wv_adapters_set(uint64_t adapters, int32_t index, int32_t rank, float scale, const uint16_t* a,
                    const uint16_t* b) try {
    Set s;
    if (!set_lookup(adapters, s))
        return rt_fail(WV_E_HANDLE, "wv_adapters_set: unknown adapters %llu", (unsigned long long)adapters);
    if (index < 0 || index >= s.c.n_adapters)
        return rt_fail(WV_E_ARG, "wv_adapters_set: adapter %d of %d", index, s.c.n_adapters);
    if (rank < 0 || rank > s.c.max_rank)
        return rt_fail(WV_E_SHAPE, "wv_adapters_set: rank %d of at most %d", rank, s.c.max_rank);
    if (!std::isfinite(scale)) return rt_fail(WV_E_ARG, "wv_adapters_set: scale %g", double(scale));
    if (rank && (!a || !b)) return rt_fail(WV_E_ARG, "wv_adapters_set: nil a/b");
    const size_t R = size_t(s.R), C = size_t(s.C), rows = size_t(s.c.rows), cols = size_t(s.c.cols), r = size_t(rank);
    std::vector<uint16_t> ha(rank ? R * C : 0), hb(rank ? rows * R : 0);
    for (size_t i = 0; i < r; ++i) std::memcpy(&ha[i * C], a + i * cols, cols * 2);
    for (size_t i = 0; i < rows && r; ++i) std::memcpy(&hb[i * R], b + i * r, r * 2);
    (void)hipSetDevice(s.device);
    hipError_t e = hipDeviceSynchronize();  // calls that still read the adapter
    if (e == hipSuccess && r) e = hipMemcpy(s.a + size_t(index) * R * C, ha.data(), ha.size() * 2, hipMemcpyHostToDevice);
    if (e == hipSuccess && r) e = hipMemcpy(s.b + size_t(index) * rows * R, hb.data(), hb.size() * 2, hipMemcpyHostToDevice);
    if (e == hipSuccess) e = hipMemcpy(s.scale + index, &scale, 4, hipMemcpyHostToDevice);
    if (e == hipSuccess) e = hipMemcpy(s.rank + index, &rank, 4, hipMemcpyHostToDevice);
    return e == hipSuccess ? WV_OK : rt_hip_fail(e, "wv_adapters_set");
} catch (const std::bad_alloc&) {
    return rt_fail(WV_E_OOM, "wv_adapters_set: host memory exhausted");
}

int wv_adapters_free(uint64_t adapters) {
    Set s;
    {
        std::lock_guard<std::mutex> lk(g_mu);
        auto it = g_sets.find(adapters);
        if (it == g_sets.end())
            return rt_fail(WV_E_HANDLE, "wv_adapters_free: unknown adapters %llu", (unsigned long long)adapters);
        s = it->second;
        g_sets.erase(it);
    }
    (void)hipSetDevice(s.device);
    const hipError_t e = hipFree(s.a);  // waits for the device's work
    return e == hipSuccess ? WV_OK : rt_hip_fail(e, "wv_adapters_free");
}

int wv_adapters_scratch(const wv_adapter_batch* batch, const wv_adapter_rows* sets, int32_t n_sets, size_t* bytes) {
    Set s[kMaxSets];
    const int rc = check_call("wv_adapters_scratch", batch, sets, n_sets, s);
    if (rc) return rc;
    if (!bytes) return rt_fail(WV_E_ARG, "wv_adapters_scratch: nil bytes");
    int range;
    *bytes = scratch_floats(s, n_sets, batch->n_tokens, adapt_ranges(s[0].c.cols, std::max(batch->n_tokens, 1), n_sets, range)) * 4;
    return WV_OK;
}

int wv_adapters_dev(const wv_adapter_batch* batch, const float* d_x, int64_t x_stride, const wv_adapter_rows* sets,
                    int32_t n_sets, void* d_scratch, size_t scratch_bytes, void* stream) {
    Set s[kMaxSets];
    int rc = check_call("wv_adapters", batch, sets, n_sets, s);
    if (rc) return rc;
    Args a{};
    a.cols = s[0].c.cols, a.n_seqs = batch->n_seqs, a.n_tokens = batch->n_tokens;
    if (!x_stride) x_stride = a.cols;
    if (x_stride < a.cols)
        return rt_fail(WV_E_SHAPE, "wv_adapters: row stride %lld under the row's %d floats", (long long)x_stride, a.cols);
    for (int i = 0; i < n_sets; ++i) {
        const wv_adapter_rows& r = sets[i];
        SetArgs& k = a.set[i];
        const int64_t w = s[i].c.rows;
        k.ys = r.y_stride ? r.y_stride : w;
        k.base = r.d_base ? r.d_base : r.d_y;
        k.bs = r.d_base ? (r.base_stride ? r.base_stride : w) : k.ys;
        k.y = r.d_y;
        if (k.ys < w || k.bs < w)
            return rt_fail(WV_E_SHAPE, "wv_adapters: row strides %lld and %lld under the row's %lld floats",
                           (long long)k.ys, (long long)k.bs, (long long)w);
        if (k.y && k.base == k.y && k.bs != k.ys)  // rows written would be others' base still to be read
            return rt_fail(WV_E_SHAPE, "wv_adapters: base is y, at row strides of %lld and %lld", (long long)k.bs,
                           (long long)k.ys);
        k.a = s[i].a, k.b = s[i].b, k.rank = s[i].rank, k.scale = s[i].scale;
        k.rows = s[i].c.rows, k.R = s[i].R, k.C = s[i].C, k.n_adapters = s[i].c.n_adapters;
    }
    if (!a.n_seqs || !a.n_tokens) return WV_OK;
    if (!d_x || !batch->d_cu_q || !batch->d_adapter) return rt_fail(WV_E_ARG, "wv_adapters: nil x/cu_q/adapter");
    for (int i = 0; i < n_sets; ++i)
        if (!a.set[i].y) return rt_fail(WV_E_ARG, "wv_adapters: nil y");
    a.x = d_x, a.xs = x_stride, a.cu = batch->d_cu_q, a.which = batch->d_adapter;
    a.ranges = adapt_ranges(a.cols, a.n_tokens, n_sets, a.range);
    (void)hipSetDevice(s[0].device);
    hipStream_t st = rt_stream(stream, s[0].device);
    const size_t floats = scratch_floats(s, n_sets, a.n_tokens, a.ranges);
    RtScratch sc;
    float* h = static_cast<float*>(d_scratch);
    if (d_scratch) {
        if (reinterpret_cast<uintptr_t>(d_scratch) & 15) return rt_fail(WV_E_ARG, "wv_adapters: scratch not 16-byte aligned");
        if (scratch_bytes < floats * 4)
            return rt_fail(WV_E_SHAPE, "wv_adapters: %zu bytes of scratch, needs %zu", scratch_bytes, floats * 4);
    } else if (rt_capturing(st)) {  // what a replay writes must not lie in a slot that other calls take
        return rt_fail(WV_E_ARG, "wv_adapters: a captured call needs scratch of its own");
    } else {
        if ((rc = sc.get(floats, st, "wv_adapters: scratch"))) return rc;
        h = sc.f();
    }
    for (int i = 0; i < n_sets; ++i) {
        a.set[i].h = h;
        h += size_t(a.ranges) * size_t(a.n_tokens) * size_t(a.set[i].R);
    }
    const int e = s[0].c.type == WV_ADAPTER_BF16 ? launch_adapters<WV_ADAPTER_BF16>(a, n_sets, st)
                                                 : launch_adapters<WV_ADAPTER_F16>(a, n_sets, st);
    return e == hipSuccess ? WV_OK : rt_hip_fail(hipError_t(e), "wv_adapters: kernel launch");
}

}  // extern "C"
