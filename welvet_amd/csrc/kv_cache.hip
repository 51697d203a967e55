// kv_cache.hip — the paged KV cache: its handles, and the kernels that
// quantise rows as they are written and read them back.
#include <algorithm>
#include <mutex>
#include <new>
#include <type_traits>
#include <unordered_map>

#include "kv.h"
#include "rt_internal.h"

namespace wv {
namespace {

std::mutex g_mu;
std::unordered_map<uint64_t, KvCache> g_caches;
uint64_t g_next = 1;

constexpr float kTiny = 7.888609052210118e-31f;  // 2^-100: rows below it are held as zeros

constexpr float kMostQ8 = 8454659.0f * 3.1691265005705735e29f;  // 8454659 2^98: the largest with a finite 127-fold
constexpr float kMostF16 = 1.0384593717069655e34f;  // 2^113, a row's largest scale: codes end under 2^15 there

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
    const float s = fminf(amax / 127.0f, kMostQ8);
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

// The largest magnitude of a row over its HD / 4 lanes (32 or 16), as bits:
// those of NaN and infinity are the largest.
template <int HD>
__device__ __forceinline__ float row_amax(const float4 x, bool& bad) {
    constexpr uint32_t A = 0x7fffffff;
    uint32_t m = max(max(__float_as_uint(x.x) & A, __float_as_uint(x.y) & A),
                     max(__float_as_uint(x.z) & A, __float_as_uint(x.w) & A));
#pragma unroll
    for (int d = HD / 8; d >= 1; d >>= 1) m = max(m, uint32_t(__shfl_xor(int(m), d, 64)));
    bad = m >= 0x7f800000;
    return __uint_as_float(m);
}

// Rows lie at any multiple of 4 bytes.
typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));
__device__ __forceinline__ float4 ld4(const float* p) {
    const f4 x = *reinterpret_cast<const f4*>(p);
    return make_float4(x.x, x.y, x.z, x.w);
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

// Stored past the caches: 16384 tokens of 8 heads are read back in 39 us so,
// in 63 with plain stores.
__device__ __forceinline__ void st4(float* p, const float4 y) {
    __builtin_nontemporal_store(f4{y.x, y.y, y.z, y.w}, reinterpret_cast<f4*>(p));
}

// A row's scale, and the codes of this lane's four values of it, the first lowest.
template <int HD, int TYPE>
__device__ __forceinline__ uint64_t row_codes(const float4 x, float& s) {
    bool bad;
    const float amax = row_amax<HD>(x, bad);
    float inv;
    s = row_scale(amax, bad, TYPE, inv);
    const float f[4] = {x.x, x.y, x.z, x.w}, most = s == kMostF16 ? 32752.0f : 32768.0f;
    uint64_t c = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (TYPE == WV_KV_F16)
            c |= uint64_t(__builtin_bit_cast(
                     uint16_t, bad ? _Float16(0) : _Float16(__builtin_amdgcn_fmed3f(f[i] * inv, -most, most)))) << (16 * i);
        else
            c |= uint64_t(uint32_t((bad || s == 0.0f ? 0 : q8_code(f[i], s, inv)) + 128)) << (8 * i);
    }
    return c;
}
template <int TYPE>
__device__ __forceinline__ void put4(uint8_t* p, uint64_t c) {
    if (TYPE == WV_KV_F16)
        *reinterpret_cast<uint64_t*>(p) = c;
    else
        *reinterpret_cast<uint32_t*>(p) = uint32_t(c);
}
// Four codes' values.
template <int TYPE>
__device__ __forceinline__ float4 row_values(uint64_t c, float s) {
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        y[i] = TYPE == WV_KV_F16 ? float(__builtin_bit_cast(_Float16, uint16_t(c >> (16 * i)))) * s
                                 : float(int(c >> (8 * i) & 255) - 128) * s;
    return make_float4(y[0], y[1], y[2], y[3]);
}
template <int TYPE>
__device__ __forceinline__ uint64_t get4(const uint8_t* p) {
    return TYPE == WV_KV_F16 ? *reinterpret_cast<const uint64_t*>(p) : *reinterpret_cast<const uint32_t*>(p);
}

// From this many rows (tokens times KV heads) on a block takes 32 of them.
// Fewer do not fill the GPU, and a tile's steps one after the other take
// longer than a row's. Tiles against row by row, fp16, head dim 128, 8 heads:
// 64 tokens in order 5.6 to 4.1 us written, 4.6 to 4.1 read; 1024 tokens 6.3
// to 10.1 and 5.2 to 7.2; 16384 tokens 39 to 98 and 39 to 75, which is a large
// copy's rate. In no order 1024 tokens 11.3 to 11.4 and 10.4 to 8.8, 16384
// tokens 135 to 139 and 82 to 97.
constexpr int kTileRows = 8192;

// Many rows: 32 tokens of one KV head to a block, their codes through LDS, so
// that K leaves as whole 16-byte units and V as words of four keys, where four
// rows in a row have the four slots of such a word; the rows left go code by
// code. `lead`: the rows with which a word begins, `cov`: those in one.
struct Tile {
    int64_t block[32];
    int kk[32];       // -1: outside the pool
    float sk[32], sv[32];
    uint32_t lead, cov;
};
// By the first wave: places the tile's slots.
__device__ __forceinline__ void tile_place(const KvView& c, Tile& t, const int64_t* slots, int64_t t0, int n, int head) {
    if (threadIdx.x >= 64) return;
    const int r = threadIdx.x & 31;
    const int64_t slot = t0 + r < n ? slots[t0 + r] : -1;
    int64_t block = 0;
    int kk = 0;
    const bool in = place(c, slot, head, block, kk);
    bool lead = in && kk % 4 == 0 && r < 29;
#pragma unroll
    for (int i = 1; i < 4; ++i) lead = uint64_t(__shfl(slot, (r + i) & 31, 64)) == uint64_t(slot) + i && lead;
    const uint32_t m = uint32_t(__ballot(lead));
    if (threadIdx.x < 32) {
        t.block[r] = block;
        t.kk[r] = in ? kk : -1;
        if (r == 0) t.lead = m, t.cov = m | m << 1 | m << 2 | m << 3;
    }
}

// One row (token, KV head) per HD / 4 lanes, 4 dims of K and of V each.
template <int HD, int TYPE>
__global__ void __launch_bounds__(256) k_kv_write(KvView c, const float* __restrict__ k, const float* __restrict__ v,
                                                  int64_t ks, int64_t vs, const int64_t* __restrict__ slots, int n) {
    constexpr int LR = HD / 4;
    const int64_t row = int64_t(blockIdx.x) * (256 / LR) + threadIdx.x / LR;
    const int d = 4 * (threadIdx.x % LR);
    const int64_t t = row / c.n_kv;
    const int head = int(row % c.n_kv);
    if (t >= n) return;
    int64_t block;
    int kk;
    if (!place(c, slots[t], head, block, kk)) return;
    const float4 xk = ld4(k + t * ks + head * HD + d);
    const float4 xv = ld4(v + t * vs + head * HD + d);
    float sk, sv;
    const uint64_t ck = row_codes<HD, TYPE>(xk, sk), cv = row_codes<HD, TYPE>(xv, sv);
    int o, j;
    kv_key_octet(kk, o, j);
    constexpr int E = TYPE == WV_KV_F16 ? 2 : 1;
    put4<TYPE>(c.k + block * (32 * HD * E) + (d * E / 16 * 32 + kk) * 16 + d * E % 16, ck);
    uint8_t* vb = c.v + block * (32 * HD * E) + ((o * HD + d) * 8 + j) * E;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (TYPE == WV_KV_F16)
            *reinterpret_cast<uint16_t*>(vb + 16 * i) = uint16_t(cv >> (16 * i));
        else
            vb[8 * i] = uint8_t(cv >> (8 * i));
    }
    if (d == 0) {
        float* sb = c.s + block * kKvScales + o * 16 + j;
        sb[0] = sk;
        sb[8] = sv;
    }
}

template <int HD, int TYPE>
__global__ void __launch_bounds__(256) k_kv_write_tile(KvView c, const float* __restrict__ k,
                                                       const float* __restrict__ v, int64_t ks, int64_t vs,
                                                       const int64_t* __restrict__ slots, int n) {
    constexpr int E = TYPE == WV_KV_F16 ? 2 : 1, LR = HD / 4, RP = 256 / LR, NP = 32 / RP, RS = HD * E + 16;
    __shared__ Tile tl;
    __shared__ __align__(16) uint8_t lk[32 * RS], lv[32 * RS];
    const int64_t t0 = int64_t(blockIdx.x) / c.n_kv * 32;
    const int head = int(int64_t(blockIdx.x) % c.n_kv);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int d = 4 * (tid % LR), r0 = tid / LR;
    float4 xk[NP], xv[NP];
#pragma unroll
    for (int p = 0; p < NP; ++p) {
        const int64_t t = t0 + p * RP + r0;
        xk[p] = t < n ? ld4(k + t * ks + head * HD + d) : float4{};
        xv[p] = t < n ? ld4(v + t * vs + head * HD + d) : float4{};
    }
    tile_place(c, tl, slots, t0, n, head);
#pragma unroll
    for (int p = 0; p < NP; ++p) {
        const int r = p * RP + r0;
        float sk, sv;
        put4<TYPE>(lk + r * RS + d * E, row_codes<HD, TYPE>(xk[p], sk));
        put4<TYPE>(lv + r * RS + d * E, row_codes<HD, TYPE>(xv[p], sv));
        if (d == 0) tl.sk[r] = sk, tl.sv[r] = sv;
    }
    __syncthreads();
    {
        const int r = tid & 31, kk = tl.kk[r];
        if (kk >= 0) {
            const int64_t block = tl.block[r];
            uint8_t* kb = c.k + block * (32 * HD * E) + kk * 16;
#pragma unroll
            for (int u = tid >> 5; u < HD * E / 16; u += 8)
                *reinterpret_cast<uint4*>(kb + u * 512) = *reinterpret_cast<const uint4*>(lk + r * RS + u * 16);
            if (tid < 64) {
                int o, j;
                kv_key_octet(kk, o, j);
                c.s[block * kKvScales + o * 16 + 8 * (tid >> 5) + j] = tid < 32 ? tl.sk[r] : tl.sv[r];
            }
        }
    }
    const int dv = 2 * lane;  // two dims to a lane
    if (dv >= HD) return;
    const uint32_t lead = __builtin_amdgcn_readfirstlane(tl.lead), cov = __builtin_amdgcn_readfirstlane(tl.cov);
    int turn = 0;
    for (uint32_t m = lead; m; m &= m - 1) {
        if ((turn++ & 3) != wave) continue;
        const int r = __builtin_ctz(m);
        int o, j;
        kv_key_octet(tl.kk[r], o, j);
        uint8_t* vb = c.v + tl.block[r] * (32 * HD * E) + ((o * HD + dv) * 8 + j) * E;
        const uint8_t* x = lv + r * RS + dv * E;
        if (TYPE == WV_KV_F16) {
            uint32_t y[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) y[i] = *reinterpret_cast<const uint32_t*>(x + i * RS);
            *reinterpret_cast<uint2*>(vb) = make_uint2((y[0] & 0xffff) | y[1] << 16, (y[2] & 0xffff) | y[3] << 16);
            *reinterpret_cast<uint2*>(vb + 16) =
                make_uint2(y[0] >> 16 | (y[1] & 0xffff0000), y[2] >> 16 | (y[3] & 0xffff0000));
        } else {
            uint32_t y[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) y[i] = *reinterpret_cast<const uint16_t*>(x + i * RS);
            *reinterpret_cast<uint32_t*>(vb) =
                (y[0] & 255) | (y[1] & 255) << 8 | (y[2] & 255) << 16 | (y[3] & 255) << 24;
            *reinterpret_cast<uint32_t*>(vb + 8) = y[0] >> 8 | (y[1] >> 8) << 8 | (y[2] >> 8) << 16 | (y[3] >> 8) << 24;
        }
    }
    for (uint32_t m = ~cov; m; m &= m - 1) {
        if ((turn++ & 3) != wave) continue;
        const int r = __builtin_ctz(m), kk = tl.kk[r];
        if (kk < 0) continue;
        int o, j;
        kv_key_octet(kk, o, j);
        uint8_t* vb = c.v + tl.block[r] * (32 * HD * E) + ((o * HD + dv) * 8 + j) * E;
        const uint8_t* x = lv + r * RS + dv * E;
        if (TYPE == WV_KV_F16) {
            const uint32_t y = *reinterpret_cast<const uint32_t*>(x);
            *reinterpret_cast<uint16_t*>(vb) = uint16_t(y);
            *reinterpret_cast<uint16_t*>(vb + 16) = uint16_t(y >> 16);
        } else {
            vb[0] = x[0];
            vb[8] = x[1];
        }
    }
}

template <int HD, int TYPE>
__global__ void __launch_bounds__(256) k_kv_read(KvView c, const int64_t* __restrict__ slots, int n,
                                                 float* __restrict__ k, float* __restrict__ v, int64_t ks, int64_t vs) {
    constexpr int LR = HD / 4;
    const int64_t row = int64_t(blockIdx.x) * (256 / LR) + threadIdx.x / LR;
    const int d = 4 * (threadIdx.x % LR);
    const int64_t t = row / c.n_kv;
    const int head = int(row % c.n_kv);
    if (t >= n) return;
    float4 yk{}, yv{};
    int64_t block;
    int kk;
    if (place(c, slots[t], head, block, kk)) {
        int o, j;
        kv_key_octet(kk, o, j);
        constexpr int E = TYPE == WV_KV_F16 ? 2 : 1;
        const float* sb = c.s + block * kKvScales + o * 16 + j;
        const uint8_t* vb = c.v + block * (32 * HD * E) + ((o * HD + d) * 8 + j) * E;
        uint64_t cv = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            cv |= TYPE == WV_KV_F16 ? uint64_t(*reinterpret_cast<const uint16_t*>(vb + 16 * i)) << (16 * i)
                                    : uint64_t(vb[8 * i]) << (8 * i);
        yk = row_values<TYPE>(get4<TYPE>(c.k + block * (32 * HD * E) + (d * E / 16 * 32 + kk) * 16 + d * E % 16), sb[0]);
        yv = row_values<TYPE>(cv, sb[8]);
    }
    st4(k + t * ks + head * HD + d, yk);
    st4(v + t * vs + head * HD + d, yv);
}

// Many rows: the way back, 32 tokens of one KV head to a block.
template <int HD, int TYPE>
__global__ void __launch_bounds__(256) k_kv_read_tile(KvView c, const int64_t* __restrict__ slots, int n,
                                                      float* __restrict__ k, float* __restrict__ v, int64_t ks,
                                                      int64_t vs) {
    constexpr int E = TYPE == WV_KV_F16 ? 2 : 1, LR = HD / 4, RP = 256 / LR, NP = 32 / RP, RS = HD * E + 16;
    __shared__ Tile tl;
    __shared__ __align__(16) uint8_t lk[32 * RS], lv[32 * RS];
    const int64_t t0 = int64_t(blockIdx.x) / c.n_kv * 32;
    const int head = int(int64_t(blockIdx.x) % c.n_kv);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    tile_place(c, tl, slots, t0, n, head);
    __syncthreads();
    {
        const int r = tid & 31, kk = tl.kk[r];
        if (kk >= 0) {
            const int64_t block = tl.block[r];
            const uint8_t* kb = c.k + block * (32 * HD * E) + kk * 16;
#pragma unroll
            for (int u = tid >> 5; u < HD * E / 16; u += 8)
                *reinterpret_cast<uint4*>(lk + r * RS + u * 16) = *reinterpret_cast<const uint4*>(kb + u * 512);
            if (tid < 64) {
                int o, j;
                kv_key_octet(kk, o, j);
                const float x = c.s[block * kKvScales + o * 16 + 8 * (tid >> 5) + j];
                (tid < 32 ? tl.sk : tl.sv)[r] = x;
            }
        }
    }
    const int dv = 2 * lane;  // two dims to a lane
    if (dv < HD) {
        const uint32_t lead = __builtin_amdgcn_readfirstlane(tl.lead), cov = __builtin_amdgcn_readfirstlane(tl.cov);
        int turn = 0;
        for (uint32_t m = lead; m; m &= m - 1) {
            if ((turn++ & 3) != wave) continue;
            const int r = __builtin_ctz(m);
            int o, j;
            kv_key_octet(tl.kk[r], o, j);
            const uint8_t* vb = c.v + tl.block[r] * (32 * HD * E) + ((o * HD + dv) * 8 + j) * E;
            uint8_t* x = lv + r * RS + dv * E;
            if (TYPE == WV_KV_F16) {
                const uint2 a = *reinterpret_cast<const uint2*>(vb), b = *reinterpret_cast<const uint2*>(vb + 16);
                *reinterpret_cast<uint32_t*>(x) = (a.x & 0xffff) | b.x << 16;
                *reinterpret_cast<uint32_t*>(x + RS) = a.x >> 16 | (b.x & 0xffff0000);
                *reinterpret_cast<uint32_t*>(x + 2 * RS) = (a.y & 0xffff) | b.y << 16;
                *reinterpret_cast<uint32_t*>(x + 3 * RS) = a.y >> 16 | (b.y & 0xffff0000);
            } else {
                const uint32_t a = *reinterpret_cast<const uint32_t*>(vb), b = *reinterpret_cast<const uint32_t*>(vb + 8);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    *reinterpret_cast<uint16_t*>(x + i * RS) =
                        uint16_t(((a >> (8 * i)) & 255) | ((b >> (8 * i)) & 255) << 8);
            }
        }
        for (uint32_t m = ~cov; m; m &= m - 1) {
            if ((turn++ & 3) != wave) continue;
            const int r = __builtin_ctz(m), kk = tl.kk[r];
            if (kk < 0) continue;
            int o, j;
            kv_key_octet(kk, o, j);
            const uint8_t* vb = c.v + tl.block[r] * (32 * HD * E) + ((o * HD + dv) * 8 + j) * E;
            uint8_t* x = lv + r * RS + dv * E;
            if (TYPE == WV_KV_F16)
                *reinterpret_cast<uint32_t*>(x) = *reinterpret_cast<const uint16_t*>(vb) |
                                                  uint32_t(*reinterpret_cast<const uint16_t*>(vb + 16)) << 16;
            else
                *reinterpret_cast<uint16_t*>(x) = uint16_t(vb[0] | vb[8] << 8);
        }
    }
    __syncthreads();
    const int d = 4 * (tid % LR), r0 = tid / LR;
#pragma unroll
    for (int p = 0; p < NP; ++p) {
        const int r = p * RP + r0;
        const int64_t t = t0 + r;
        if (t >= n) return;
        float4 yk{}, yv{};
        if (tl.kk[r] >= 0) {
            yk = row_values<TYPE>(get4<TYPE>(lk + r * RS + d * E), tl.sk[r]);
            yv = row_values<TYPE>(get4<TYPE>(lv + r * RS + d * E), tl.sv[r]);
        }
        st4(k + t * ks + head * HD + d, yk);
        st4(v + t * vs + head * HD + d, yv);
    }
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
    const bool tile = int64_t(n) * c.n_kv >= kTileRows;
    const int per = 256 / (c.hd / 4);
    const int64_t blocks = tile ? (int64_t(n) + 31) / 32 * c.n_kv : (int64_t(n) * c.n_kv + per - 1) / per;
    auto go = [&](auto kern) { hipLaunchKernelGGL(kern, dim3(unsigned(blocks)), dim3(256), 0, s, c, k, v, ks, vs, slots, n); };
    auto pick = [&](auto hd, auto type) {
        constexpr int HD = decltype(hd)::value, TYPE = decltype(type)::value;
        tile ? go(k_kv_write_tile<HD, TYPE>) : go(k_kv_write<HD, TYPE>);
    };
    std::integral_constant<int, 128> h128;
    std::integral_constant<int, 64> h64;
    std::integral_constant<int, WV_KV_F16> f16;
    std::integral_constant<int, WV_KV_Q8> q8;
    if (c.hd == 128)
        c.type == WV_KV_F16 ? pick(h128, f16) : pick(h128, q8);
    else
        c.type == WV_KV_F16 ? pick(h64, f16) : pick(h64, q8);
    return int(hipGetLastError());
}

int launch_kv_read(const KvView& c, const int64_t* slots, int n, float* k, float* v, int64_t ks, int64_t vs,
                   hipStream_t s) {
    const bool tile = int64_t(n) * c.n_kv >= kTileRows;
    const int per = 256 / (c.hd / 4);
    const int64_t blocks = tile ? (int64_t(n) + 31) / 32 * c.n_kv : (int64_t(n) * c.n_kv + per - 1) / per;
    auto go = [&](auto kern) { hipLaunchKernelGGL(kern, dim3(unsigned(blocks)), dim3(256), 0, s, c, slots, n, k, v, ks, vs); };
    auto pick = [&](auto hd, auto type) {
        constexpr int HD = decltype(hd)::value, TYPE = decltype(type)::value;
        tile ? go(k_kv_read_tile<HD, TYPE>) : go(k_kv_read<HD, TYPE>);
    };
    std::integral_constant<int, 128> h128;
    std::integral_constant<int, 64> h64;
    std::integral_constant<int, WV_KV_F16> f16;
    std::integral_constant<int, WV_KV_Q8> q8;
    if (c.hd == 128)
        c.type == WV_KV_F16 ? pick(h128, f16) : pick(h128, q8);
    else
        c.type == WV_KV_F16 ? pick(h64, f16) : pick(h64, q8);
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
    if (int64_t(n) * c.c.n_kv_heads > int64_t(1) << 28)
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
