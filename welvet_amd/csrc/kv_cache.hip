// kv_cache.hip — the paged KV cache: its handles, and the kernels that
// quantise rows as they are written and read them back.
#include <algorithm>
#include <mutex>
#include <new>
#include <unordered_map>

#include "kv.h"
#include "rt_internal.h"

namespace wv {
namespace {

std::mutex g_mu;
std::unordered_map<uint64_t, KvCache> g_caches;
uint64_t g_next = 1;

constexpr float kTiny = 7.888609052210118e-31f;  // 2^-100: rows below it are held as zeros

// A row's scale from its largest magnitude (bad: it holds a NaN or infinity)
// and the factor its values take before rounding. F16: powers of two, so the
// product is exact and amax / scale lies in [2^14, 2^15). Q8: amax / 127 in
// f32; the factor is only near 1 / scale, q8_code() puts the last digit right.
__device__ __forceinline__ float row_scale(float amax, bool bad, int type, float& inv) {
    inv = 0.0f;
    if (bad) return __int_as_float(0x7fc00000);
    if (amax < kTiny) return 0.0f;
    if (type == WV_KV_F16) {
        const int e = int(__float_as_uint(amax) >> 23) - 127;  // amax is normal
        inv = __uint_as_float(uint32_t(14 - e + 127) << 23);
        return __uint_as_float(uint32_t(e - 14 + 127) << 23);
    }
    const float s = amax / 127.0f;
    inv = 1.0f / s;
    return s;
}

// |x| / s rounded half away from zero, exactly: n is within one of it, and
// the remainder d = |x| - n s is a multiple of ulp(s) / 2 below s, so the fma
// returns it without rounding and its comparison with s / 2 is exact.
__device__ __forceinline__ int q8_code(float x, float s, float inv) {
    const float ax = fabsf(x);
    float n = rintf(ax * inv);
    const float d = fmaf(-n, s, ax);
    n += d >= 0.5f * s ? 1.0f : d < -0.5f * s ? -1.0f : 0.0f;
    const int c = min(int(n), 127);
    return x < 0.0f ? -c : c;
}

// The largest magnitude of a row over its HD / 4 lanes (32 or 16), and
// whether any of its values is a NaN or infinity.
template <int HD>
__device__ __forceinline__ float row_amax(const float4 x, bool& bad) {
    float m = fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w)));
    const float lim = 3.402823466e38f;
    int b = !(fabsf(x.x) <= lim && fabsf(x.y) <= lim && fabsf(x.z) <= lim && fabsf(x.w) <= lim);
#pragma unroll
    for (int d = HD / 8; d >= 1; d >>= 1) {
        m = fmaxf(m, __shfl_xor(m, d, 64));
        b |= __shfl_xor(b, d, 64);
    }
    bad = b != 0;
    return m;
}

__device__ __forceinline__ float4 ld4(const float* p, bool aligned) {
    if (aligned) return *reinterpret_cast<const float4*>(p);
    return make_float4(p[0], p[1], p[2], p[3]);
}

// Where a slot lies: its block and the key in it; false outside the pool.
__device__ __forceinline__ bool place(const KvView& c, int64_t slot, int head, int64_t& block, int& kk) {
    const int64_t page = slot >> c.page_shift;
    if (slot < 0 || page >= c.n_pages) return false;
    const int off = int(slot & ((1 << c.page_shift) - 1));
    block = kv_block(c, page, head, off);
    kk = off & 31;
    return true;
}

// One row (token, KV head) per HD / 4 lanes, 4 dims of K and of V each.
template <int HD, int TYPE>
__global__ void __launch_bounds__(256) k_kv_write(KvView c, const float* __restrict__ k, const float* __restrict__ v,
                                                  int64_t ks, int64_t vs, const int64_t* __restrict__ slots, int n,
                                                  bool aligned) {
    constexpr int LR = HD / 4;
    const int64_t row = int64_t(blockIdx.x) * (256 / LR) + threadIdx.x / LR;
    const int d = 4 * (threadIdx.x % LR);
    const int64_t t = row / c.n_kv;
    const int head = int(row % c.n_kv);
    if (t >= n) return;
    int64_t block;
    int kk;
    if (!place(c, slots[t], head, block, kk)) return;
    const float4 xk = ld4(k + t * ks + head * HD + d, aligned);
    const float4 xv = ld4(v + t * vs + head * HD + d, aligned);
    bool bk, bv;
    const float ak = row_amax<HD>(xk, bk), av = row_amax<HD>(xv, bv);
    float ik, iv;
    const float sk = row_scale(ak, bk, TYPE, ik), sv = row_scale(av, bv, TYPE, iv);
    int o, j;
    kv_key_octet(kk, o, j);
    constexpr int E = TYPE == WV_KV_F16 ? 2 : 1;
    uint8_t* kb = c.k + block * (32 * HD * E);
    uint8_t* vb = c.v + block * (32 * HD * E);
    const float fk[4] = {xk.x, xk.y, xk.z, xk.w}, fv[4] = {xv.x, xv.y, xv.z, xv.w};
    if (TYPE == WV_KV_F16) {
        typedef _Float16 h4 __attribute__((ext_vector_type(4)));
        h4 ck;
#pragma unroll
        for (int i = 0; i < 4; ++i) ck[i] = bk ? _Float16(0) : _Float16(fk[i] * ik);
        *reinterpret_cast<h4*>(kb + ((d / 8) * 32 + kk) * 16 + (d % 8) * 2) = ck;
        _Float16* vh = reinterpret_cast<_Float16*>(vb) + (o * HD + d) * 8 + j;
#pragma unroll
        for (int i = 0; i < 4; ++i) vh[8 * i] = bv ? _Float16(0) : _Float16(fv[i] * iv);
    } else {
        uint32_t ck = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) ck |= uint32_t((bk || sk == 0.0f ? 0 : q8_code(fk[i], sk, ik)) + 128) << (8 * i);
        *reinterpret_cast<uint32_t*>(kb + ((d / 16) * 32 + kk) * 16 + d % 16) = ck;
        uint8_t* vq = vb + (o * HD + d) * 8 + j;
#pragma unroll
        for (int i = 0; i < 4; ++i) vq[8 * i] = uint8_t((bv || sv == 0.0f ? 0 : q8_code(fv[i], sv, iv)) + 128);
    }
    if (d == 0) {
        float* sb = c.s + block * kKvScales + o * 16 + j;
        sb[0] = sk;
        sb[8] = sv;
    }
}

template <int HD, int TYPE>
__global__ void __launch_bounds__(256) k_kv_read(KvView c, const int64_t* __restrict__ slots, int n,
                                                 float* __restrict__ k, float* __restrict__ v, int64_t ks, int64_t vs,
                                                 bool aligned) {
    constexpr int LR = HD / 4;
    const int64_t row = int64_t(blockIdx.x) * (256 / LR) + threadIdx.x / LR;
    const int d = 4 * (threadIdx.x % LR);
    const int64_t t = row / c.n_kv;
    const int head = int(row % c.n_kv);
    if (t >= n) return;
    float yk[4] = {0, 0, 0, 0}, yv[4] = {0, 0, 0, 0};
    int64_t block;
    int kk;
    if (place(c, slots[t], head, block, kk)) {
        int o, j;
        kv_key_octet(kk, o, j);
        constexpr int E = TYPE == WV_KV_F16 ? 2 : 1;
        const uint8_t* kb = c.k + block * (32 * HD * E);
        const uint8_t* vb = c.v + block * (32 * HD * E);
        const float* sb = c.s + block * kKvScales + o * 16 + j;
        const float sk = sb[0], sv = sb[8];
        if (TYPE == WV_KV_F16) {
            typedef _Float16 h4 __attribute__((ext_vector_type(4)));
            const h4 ck = *reinterpret_cast<const h4*>(kb + ((d / 8) * 32 + kk) * 16 + (d % 8) * 2);
            const _Float16* vh = reinterpret_cast<const _Float16*>(vb) + (o * HD + d) * 8 + j;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                yk[i] = float(ck[i]) * sk;
                yv[i] = float(vh[8 * i]) * sv;
            }
        } else {
            const uint32_t ck = *reinterpret_cast<const uint32_t*>(kb + ((d / 16) * 32 + kk) * 16 + d % 16);
            const uint8_t* vq = vb + (o * HD + d) * 8 + j;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                yk[i] = float(int((ck >> (8 * i)) & 255) - 128) * sk;
                yv[i] = float(int(vq[8 * i]) - 128) * sv;
            }
        }
    }
    float* ok = k + t * ks + head * HD + d;
    float* ov = v + t * vs + head * HD + d;
    if (aligned) {
        *reinterpret_cast<float4*>(ok) = make_float4(yk[0], yk[1], yk[2], yk[3]);
        *reinterpret_cast<float4*>(ov) = make_float4(yv[0], yv[1], yv[2], yv[3]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) ok[i] = yk[i], ov[i] = yv[i];
    }
}

// Rows that float4 accesses reach: base and stride multiples of 16 bytes.
bool rows_aligned(const void* a, const void* b, int64_t sa, int64_t sb) {
    return !((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) & 15) && sa % 4 == 0 && sb % 4 == 0;
}

}  // namespace

bool kv_lookup(uint64_t h, KvCache& out) {
    std::lock_guard<std::mutex> lk(g_mu);
    auto it = g_caches.find(h);
    if (it == g_caches.end()) return false;
    out = it->second;
    return true;
}

int launch_kv_write(const KvView& c, const float* k, const float* v, int64_t ks, int64_t vs, const int64_t* slots,
                    int n, hipStream_t s) {
    const bool al = rows_aligned(k, v, ks, vs);
    const int per = 256 / (c.hd / 4);
    const dim3 grid(unsigned((int64_t(n) * c.n_kv + per - 1) / per));
    auto go = [&](auto kern) { hipLaunchKernelGGL(kern, grid, dim3(256), 0, s, c, k, v, ks, vs, slots, n, al); };
    if (c.hd == 128)
        c.type == WV_KV_F16 ? go(k_kv_write<128, WV_KV_F16>) : go(k_kv_write<128, WV_KV_Q8>);
    else
        c.type == WV_KV_F16 ? go(k_kv_write<64, WV_KV_F16>) : go(k_kv_write<64, WV_KV_Q8>);
    return int(hipGetLastError());
}

int launch_kv_read(const KvView& c, const int64_t* slots, int n, float* k, float* v, int64_t ks, int64_t vs,
                   hipStream_t s) {
    const bool al = rows_aligned(k, v, ks, vs);
    const int per = 256 / (c.hd / 4);
    const dim3 grid(unsigned((int64_t(n) * c.n_kv + per - 1) / per));
    auto go = [&](auto kern) { hipLaunchKernelGGL(kern, grid, dim3(256), 0, s, c, slots, n, k, v, ks, vs, al); };
    if (c.hd == 128)
        c.type == WV_KV_F16 ? go(k_kv_read<128, WV_KV_F16>) : go(k_kv_read<128, WV_KV_Q8>);
    else
        c.type == WV_KV_F16 ? go(k_kv_read<64, WV_KV_F16>) : go(k_kv_read<64, WV_KV_Q8>);
    return int(hipGetLastError());
}

}  // namespace wv

using namespace wv;

namespace {

// The checks that wv_kv_write_dev and wv_kv_read_dev share; strides of 0 become dense ones.
int check_rows(const char* what, uint64_t cache, int32_t layer, const void* k, const void* v, int64_t& ks, int64_t& vs,
               const void* slots, int32_t n, KvCache& c) {
    if (!kv_lookup(cache, c)) return rt_fail(WV_E_HANDLE, "%s: unknown cache %llu", what, (unsigned long long)cache);
    if (layer < 0 || layer >= c.c.n_layers) return rt_fail(WV_E_ARG, "%s: layer %d of %d", what, layer, c.c.n_layers);
    if (n < 0) return rt_fail(WV_E_SHAPE, "%s: negative row count %d", what, n);
    const int64_t w = int64_t(c.c.n_kv_heads) * c.c.head_dim;
    if (!ks) ks = w;
    if (!vs) vs = w;
    if (ks < w || vs < w)
        return rt_fail(WV_E_SHAPE, "%s: row strides %lld and %lld under the row's %lld floats", what, (long long)ks,
                       (long long)vs, (long long)w);
    if (n && (!k || !v || !slots)) return rt_fail(WV_E_ARG, "%s: nil k/v/slots", what);
    if (int64_t(n) * c.c.n_kv_heads >= int64_t(1) << 31)
        return rt_fail(WV_E_SHAPE, "%s: %d rows of %d heads in one call", what, n, c.c.n_kv_heads);
    return WV_OK;
}

}  // namespace

extern "C" {

int wv_kv_create(const wv_kv_config* cfg, uint64_t* cache) {
    if (!cfg || !cache) return rt_fail(WV_E_ARG, "wv_kv_create: nil argument");
    const wv_kv_config& c = *cfg;
    if (c.n_layers <= 0 || c.n_kv_heads <= 0 || c.n_pages <= 0)
        return rt_fail(WV_E_SHAPE, "wv_kv_create: non-positive dimension");
    if (c.head_dim != 64 && c.head_dim != 128)
        return rt_fail(WV_E_SHAPE, "wv_kv_create: head_dim %d (64 or 128)", c.head_dim);
    if (c.page_size != 32 && c.page_size != 64 && c.page_size != 128 && c.page_size != 256)
        return rt_fail(WV_E_SHAPE, "wv_kv_create: page_size %d (32, 64, 128 or 256)", c.page_size);
    if (c.type != WV_KV_F16 && c.type != WV_KV_Q8) return rt_fail(WV_E_FORMAT, "wv_kv_create: type %d", c.type);
    if (c.n_kv_heads > 4096) return rt_fail(WV_E_SHAPE, "wv_kv_create: %d KV heads (at most 4096)", c.n_kv_heads);
    if (int64_t(c.n_pages) * c.page_size >= int64_t(1) << 31)
        return rt_fail(WV_E_SHAPE, "wv_kv_create: %d pages of %d positions (2^31 and more)", c.n_pages, c.page_size);
    KvCache k;
    k.c = c;
    // at most 2^31 positions x 2^12 heads x 2^8 bytes: no overflow
    const size_t rows = size_t(c.n_pages) * size_t(c.page_size) * size_t(c.n_kv_heads);
    k.code_bytes = rows * size_t(c.head_dim) * size_t(kv_code_bytes(c.type));
    k.layer_bytes = 2 * k.code_bytes + rows * 2 * sizeof(float);
    if (k.layer_bytes > (size_t(1) << 62) / size_t(c.n_layers))
        return rt_fail(WV_E_OOM, "wv_kv_create: %zu bytes for each of %d layers", k.layer_bytes, c.n_layers);
    k.bytes = k.layer_bytes * size_t(c.n_layers);
    int rc = rt_ensure_init();
    if (rc) return rc;
    k.device = rt_current_device();
    hipError_t e = hipMalloc(reinterpret_cast<void**>(&k.base), k.bytes);
    if (e != hipSuccess) {
        (void)hipGetLastError();
        return rt_hip_fail(e, "wv_kv_create: pools");
    }
    // unwritten positions read 0: code 0 (the int8 codes' bias), scale 0
    hipStream_t s = rt_stream(nullptr, k.device);
    for (int l = 0; l < c.n_layers && e == hipSuccess; ++l) {
        uint8_t* p = k.base + size_t(l) * k.layer_bytes;
        e = hipMemsetAsync(p, c.type == WV_KV_Q8 ? 128 : 0, 2 * k.code_bytes, s);
        if (e == hipSuccess) e = hipMemsetAsync(p + 2 * k.code_bytes, 0, k.layer_bytes - 2 * k.code_bytes, s);
    }
    if (e == hipSuccess) e = hipStreamSynchronize(s);
    if (e != hipSuccess) {
        (void)hipFree(k.base);
        return rt_hip_fail(e, "wv_kv_create: clear");
    }
    try {
        std::lock_guard<std::mutex> lk(g_mu);
        g_caches[g_next] = k;
        *cache = g_next++;
    } catch (const std::bad_alloc&) {
        (void)hipFree(k.base);
        return rt_fail(WV_E_OOM, "wv_kv_create: host memory exhausted");
    }
    return WV_OK;
}

int wv_kv_info(uint64_t cache, wv_kv_config* cfg, size_t* device_bytes) {
    KvCache c;
    if (!kv_lookup(cache, c)) return rt_fail(WV_E_HANDLE, "wv_kv_info: unknown cache %llu", (unsigned long long)cache);
    if (cfg) *cfg = c.c;
    if (device_bytes) *device_bytes = c.bytes;
    return WV_OK;
}

int wv_kv_free(uint64_t cache) {
    KvCache c;
    {
        std::lock_guard<std::mutex> lk(g_mu);
        auto it = g_caches.find(cache);
        if (it == g_caches.end())
            return rt_fail(WV_E_HANDLE, "wv_kv_free: unknown cache %llu", (unsigned long long)cache);
        c = it->second;
        g_caches.erase(it);
    }
    (void)hipSetDevice(c.device);
    const hipError_t e = hipFree(c.base);  // waits for the device's work
    return e == hipSuccess ? WV_OK : rt_hip_fail(e, "wv_kv_free");
}

int wv_kv_write_dev(uint64_t cache, int32_t layer, const float* d_k, const float* d_v, int64_t k_stride,
                    int64_t v_stride, const int64_t* d_slots, int32_t n, void* stream) {
    KvCache c;
    const int rc = check_rows("wv_kv_write", cache, layer, d_k, d_v, k_stride, v_stride, d_slots, n, c);
    if (rc || !n) return rc;
    (void)hipSetDevice(c.device);
    const int e = launch_kv_write(c.layer(layer), d_k, d_v, k_stride, v_stride, d_slots, n, rt_stream(stream, c.device));
    return e == hipSuccess ? WV_OK : rt_hip_fail(hipError_t(e), "wv_kv_write: kernel launch");
}

int wv_kv_read_dev(uint64_t cache, int32_t layer, const int64_t* d_slots, int32_t n, float* d_k, float* d_v,
                   int64_t k_stride, int64_t v_stride, void* stream) {
    KvCache c;
    const int rc = check_rows("wv_kv_read", cache, layer, d_k, d_v, k_stride, v_stride, d_slots, n, c);
    if (rc || !n) return rc;
    (void)hipSetDevice(c.device);
    const int e = launch_kv_read(c.layer(layer), d_slots, n, d_k, d_v, k_stride, v_stride, rt_stream(stream, c.device));
    return e == hipSuccess ? WV_OK : rt_hip_fail(hipError_t(e), "wv_kv_read: kernel launch");
}

}  // extern "C"
