// kv_attention.hip — causal attention of a batch's new tokens over the paged
// KV cache.
//
// With t = scale log2(e) q.K the row's output is sum_j 2^(t_j - m) V_j over
// sum_j 2^(t_j - m), m the running maximum rounded up to a whole number: one
// pass over the keys, the sums so far scaled by 2^(m_old - m_new), exactly,
// when m grows. K and V are codes c with a
// scale s per key, exact in fp16, so with the query row split in two fp16
// terms q = 2^e (qh + ql) (22 bits)
//   t_j = (c_j.qh + c_j.ql) s_j * (2^e scale log2 e)
// on the fp16 matrix cores with f32 sums. For the second product the
// probabilities take the V scales, P_j = 2^14 p_j s_j 2^-E, with E the running
// exponent of the largest scale that the row has met among the keys it attends
// (P_j then fills fp16's range whatever the values' magnitude, and nothing else
// in the block has a part in a row's bits), and are split as ph + pl the same way.
#include <algorithm>
#include <cmath>

#include "kv.h"
#include "rt_internal.h"
#include "wave_ops.h"

namespace wv {
namespace {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr double kLog2e = 1.4426950408889634;
constexpr float kNoMax = -3.0e38f;  // m of a row that has met no key
constexpr float kLeast = 1.4e-45f;  // of a row's factor: times the -inf of a masked key it stays -inf
constexpr int kMaxSplits = 64;
constexpr int kTileRows = 512;      // rows of a sequence from which on the tile kernel is thought of
constexpr int kMaxGridY = 1 << 15;  // tiles of a launch
constexpr int kFewRows = 256;  // query rows of a sequence and KV head up to which the row kernel takes it

// 8 biased int8 codes (two words) as fp16: 0x6400 | b is 1024 + b, less 1152
// the code; one byte permute and half a packed subtraction per code pair.
__device__ __forceinline__ h8 q8_half(uint32_t x, uint32_t y) {
    union {
        uint32_t u[4];
        h2 h[4];
        h8 v;
    } r;
    r.u[0] = __builtin_amdgcn_perm(0x64646464u, x, 0x04010400u);
    r.u[1] = __builtin_amdgcn_perm(0x64646464u, x, 0x04030402u);
    r.u[2] = __builtin_amdgcn_perm(0x64646464u, y, 0x04010400u);
    r.u[3] = __builtin_amdgcn_perm(0x64646464u, y, 0x04030402u);
    const h2 b = {_Float16(1152.0f), _Float16(1152.0f)};
#pragma unroll
    for (int i = 0; i < 4; ++i) r.h[i] -= b;
    return r.v;
}
__device__ __forceinline__ h8 as_half(uint4 x) { return __builtin_bit_cast(h8, x); }
__device__ __forceinline__ h8 as_half(u4 x) { return __builtin_bit_cast(h8, x); }

// hi + lo of 8 floats: hi truncated to fp16, lo the rounded rest (a mixed fma
// each: fp16 in, fp16 out).
__device__ __forceinline__ void split8(const float* x, h8& hi, h8& lo) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const auto h = __builtin_amdgcn_cvt_pkrtz(x[i], x[i + 1]);
        hi[i] = _Float16(h[0]);
        hi[i + 1] = _Float16(h[1]);
        lo[i] = _Float16(fmaf(float(hi[i]), -1.0f, x[i]));
        lo[i + 1] = _Float16(fmaf(float(hi[i + 1]), -1.0f, x[i + 1]));
    }
}

// Maximum / sum over the lanes l, l ^ 16, l ^ 32, l ^ 48.
__device__ __forceinline__ float max_over_quads(float v) {
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_over_quads(float v) {
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Ties a value to this place among the other volatile statements: what makes
// it comes before, what uses it after.
template <class V>
__device__ __forceinline__ void pin(V& v) { asm volatile("" : "+v"(v)); }

// A block's barrier for what lies in LDS: unlike __syncthreads it does not wait
// for loads from memory that are on their way into registers.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// Largest of 32 lanes' bit patterns of floats >= 0 (lanes 32..63 hold the same), in one instruction a step.
__device__ __forceinline__ uint32_t max_of_32(float v) {
    uint32_t x = __float_as_uint(v);
    x = max(x, uint32_t(dpp_i<kDppRowShr1>(0, int(x))));
    x = max(x, uint32_t(dpp_i<kDppRowShr2>(0, int(x))));
    x = max(x, uint32_t(dpp_i<kDppRowShr4>(0, int(x))));
    x = max(x, uint32_t(dpp_i<kDppRowShr8>(0, int(x))));
    x = max(x, uint32_t(dpp_i<kDppRowBcast15>(0, int(x))));
    return uint32_t(__builtin_amdgcn_readlane(int(x), 31));
}

// A tile of query rows: row = token * G + head of the group, in one sequence.
struct Tile {
    int seq = -1, r0 = 0, rows = 0;  // first row of the tile, rows of the sequence
    int q0 = 0, n = 0, kv_len = 0;   // the sequence's first token row, new tokens, keys
};

// Tile `idx` of the batch's tiles of RT rows, over the sequences with at
// least min_rows and at most max_rows rows, in order of the sequences: every
// wave scans 64 sequences at a time. False: past the last tile. The first
// `skip` tiles of a sequence do not count.
template <int RT>
__device__ __forceinline__ bool find_tile(const KvAttn& a, int G, int idx, int min_rows, int max_rows, Tile& t,
                                          int skip = 0) {
    const int lane = threadIdx.x & 63;
    for (int base = 0; base < a.n_seqs; base += 64) {
        const int s = base + lane;
        int c0 = 0, n = 0, tiles = 0;
        if (s < a.n_seqs) {
            c0 = min(max(a.cu[s], 0), a.n_tokens);
            n = min(max(a.cu[s + 1], c0), a.n_tokens) - c0;
            const int rows = n * G;
            if (rows >= min_rows && rows <= max_rows) tiles = max((rows + RT - 1) / RT - skip, 0);
        }
        int incl = tiles;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int o = __shfl_up(incl, d, 64);
            if (lane >= d) incl += o;
        }
        const int total = __builtin_amdgcn_readlane(incl, 63);
        if (idx < total) {
            const int w = __ffsll((unsigned long long)__ballot(incl > idx)) - 1;
            t.seq = base + w;
            t.q0 = __builtin_amdgcn_readlane(c0, w);
            t.n = __builtin_amdgcn_readlane(n, w);
            t.rows = t.n * G;
            t.r0 = (skip + idx - (__builtin_amdgcn_readlane(incl, w) - __builtin_amdgcn_readlane(tiles, w))) * RT;
            t.kv_len = max(a.kv_len[t.seq], 0);
            return true;
        }
        idx -= total;
    }
    return false;
}

// The 32-key blocks [begin, end) that split `sp` of a tile's rows
// r0 .. r0 + RT - 1 walks, and the positions of its first and last row.
struct Range {
    int begin, end, p_first, p_last, limit;
};
template <int RT>
__device__ __forceinline__ Range tile_range(const KvAttn& a, const Tile& t, int G, int sp, int least) {
    Range r;
    r.limit = min(t.kv_len, a.max_pages << a.c.page_shift);
    r.p_first = t.kv_len - t.n + t.r0 / G;
    r.p_last = t.kv_len - t.n + min(t.r0 + RT - 1, t.rows - 1) / G;
    const int lo = a.window > 0 ? max(0, r.p_first - a.window + 1) : 0;
    const int hi = min(r.limit - 1, r.p_last);
    r.begin = lo >> 5;
    r.end = hi >= lo ? (hi >> 5) + 1 : r.begin;
    const int nb = r.end - r.begin;
    const int chunk = max(least, (nb + a.splits - 1) / a.splits);
    r.begin = min(r.begin + sp * chunk, r.end);
    r.end = min(r.begin + chunk, r.end);
    return r;
}

// A query row of magnitude amax: the power of two `inv` that brings it into
// fp16's range ([2^14, 2^15)), and the factor from its scores in units of
// 1 / kScore to t. Sums of codes times queries reach 2^37 and K scales 2^113,
// so scores are held 2^-23 times as large until they meet this factor.
constexpr float kScore = 1.1920929e-7f;  // 2^-23, on the K scales
__device__ __forceinline__ float row_unit(float amax, float scale, float& inv) {
    const int e = min(max(int(__float_as_uint(amax) >> 23) - 127, -113), 127);
    inv = __uint_as_float(uint32_t(14 - e + 127) << 23);
    return float(fmin(fmax(ldexp(double(scale) * kLog2e, e - 14 + 23), double(kLeast)), 3.4028234e38));
}

// Few rows: 16 query rows of one sequence and KV head per block, each of its
// 4 waves over its own 32-key blocks (every fourth of the block's range), in
// registers from the cache to the sums: a lane's 16-byte loads are operands
// of the 16x16x32 products as they lie in the cache. S^T = K Q^T leaves a
// lane (row l & 15, octet l >> 4) with the 8 keys of its octet, which are its
// operand of O^T += V^T P^T. The waves' sums meet in LDS. A single token's row
// is bound by the codes' bytes: 64 sequences of 1 to 8192 int8 keys, 32 heads
// over 8 of 128, 134 us, 5.2 TB/s; one of 131071 fp16 keys 106 us, 5.2 TB/s. A
// short one by a wave's chain from score to second product, 1.1 to 1.5 us a key
// block, and by the join's launch: 2048 int8 keys 8 + 3 us.
// ONCE: no other block reads a sequence's keys, and they are loaded past the
// caches (131071 fp16 keys 106 us, else 112); not where several tiles read them
// (64 tokens of 32 heads over 8000 fp16 keys 56 us so, else 43).
template <int HD, int TYPE, bool ONCE>
__device__ __forceinline__ void attn_rows(const KvAttn& a, int G, const Tile& t, int kvh, int sp) {
    constexpr int E = TYPE == WV_KV_F16 ? 2 : 1;
    constexpr int S = HD / 32;                   // k steps of a score product
    constexpr int NK = S / (TYPE == WV_KV_F16 ? 1 : 2);   // 16-byte K loads of a 16-key tile
    constexpr int T = HD / 16;                   // dim tiles of the output
    constexpr int NV = T / (TYPE == WV_KV_F16 ? 1 : 2);   // 16-byte V loads
    constexpr int BB = 32 * HD * E;              // bytes of a block
    constexpr int LD = HD + 4;
    __shared__ float red[4][16][LD];
    __shared__ float rm[4][16], rl[4][16];

    const Range rg = tile_range<16>(a, t, G, sp, 4);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 15, g = lane >> 4;

    const int row = t.r0 + n;
    const bool live = row < t.rows;
    const int pos = t.kv_len - t.n + (live ? row : t.r0) / G;
    const int first = a.window > 0 ? pos - a.window + 1 : 0;

    // the query row: dims of lane group g in the order of the K codes
    h8 qh[S], ql[S];
    float qs;
    {
        const int tok = (live ? row : t.r0) / G, h = kvh * G + (live ? row : t.r0) % G;
        const float* qp = a.q + int64_t(t.q0 + tok) * a.qs + h * HD;
        float x[S][8], m = 0.0f;
#pragma unroll
        for (int s = 0; s < S; ++s)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int d = TYPE == WV_KV_F16 ? 8 * (4 * s + g) + j : 16 * (4 * (s / 2) + g) + 8 * (s % 2) + j;
                x[s][j] = qp[d];
                m = fmaxf(m, fabsf(x[s][j]));
            }
        float inv;
        qs = row_unit(max_over_quads(m), a.scale, inv);
#pragma unroll
        for (int s = 0; s < S; ++s) {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[s][j] *= inv;
            split8(x[s], qh[s], ql[s]);
        }
    }

    f4 o[T];
#pragma unroll
    for (int i = 0; i < T; ++i) o[i] = f4{0, 0, 0, 0};
    float mx = kNoMax, l = 0.0f;
    int eo = -200;  // E of the lane's row: its outputs are in units of 2^eo

    const int32_t* pages = a.pages + int64_t(t.seq) * a.max_pages;
    const int pb = a.c.page_shift - 5;  // log2 blocks per page
    auto block_at = [&](int kb, bool& ok) {
        const int pg = __builtin_amdgcn_readfirstlane(pages[kb >> pb]);
        ok = unsigned(pg) < unsigned(a.c.n_pages);
        return kv_block(a.c, ok ? pg : 0, kvh, (kb & ((1 << pb) - 1)) << 5);
    };
    // key of A row n in tile x: index x * 4 + (n & 3) of octet n >> 2
    const int key0 = kv_octet_key(n >> 2, n & 3);
    uint4 kr[2][NK], vr[NV];
    float4 sk[2], sv[2];
    auto load_k = [&](int64_t b) {
        const uint4* p = reinterpret_cast<const uint4*>(a.c.k + b * BB) + g * 32 + key0;
        if (ONCE) {
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int i = 0; i < NK; ++i) kr[x][i] = ld_nt16(p + 128 * i + 8 * x);
        } else {
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int i = 0; i < NK; ++i) kr[x][i] = p[128 * i + 8 * x];
        }
    };
    auto load_v = [&](int64_t b) {
        const uint4* p = reinterpret_cast<const uint4*>(a.c.v + b * BB + g * HD * 8 * E) + n;
        if (ONCE) {
#pragma unroll
            for (int i = 0; i < NV; ++i) vr[i] = ld_nt16(p + 16 * i);
        } else {
#pragma unroll
            for (int i = 0; i < NV; ++i) vr[i] = p[16 * i];
        }
    };
    auto load_s = [&](int64_t b) {
        const float4* p = reinterpret_cast<const float4*>(a.c.s + b * kKvScales + g * 16);
        sk[0] = p[0], sk[1] = p[1], sv[0] = p[2], sv[1] = p[3];
    };

    int kb = rg.begin + wave;
    bool ok = false;
    int64_t blk = 0;
    if (kb < rg.end) {
        blk = block_at(kb, ok);
        load_s(blk);
        load_k(blk);
        load_v(blk);
    }
    while (kb < rg.end) {
        const int next = kb + 4;
        bool nok = false;
        int64_t nblk = 0;
        if (next < rg.end) nblk = block_at(next, nok);
        f4 s0 = {0, 0, 0, 0}, s1 = {0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < S; ++s) {
            h8 f0, f1;
            if (TYPE == WV_KV_F16) {
                f0 = as_half(kr[0][s]), f1 = as_half(kr[1][s]);
            } else {
                const uint4 u0 = kr[0][s / 2], u1 = kr[1][s / 2];
                f0 = s % 2 ? q8_half(u0.z, u0.w) : q8_half(u0.x, u0.y);
                f1 = s % 2 ? q8_half(u1.z, u1.w) : q8_half(u1.x, u1.y);
            }
            s0 = __builtin_amdgcn_mfma_f32_16x16x32_f16(f0, ql[s], s0, 0, 0, 0);
            s1 = __builtin_amdgcn_mfma_f32_16x16x32_f16(f1, ql[s], s1, 0, 0, 0);
            s0 = __builtin_amdgcn_mfma_f32_16x16x32_f16(f0, qh[s], s0, 0, 0, 0);
            s1 = __builtin_amdgcn_mfma_f32_16x16x32_f16(f1, qh[s], s1, 0, 0, 0);
        }
        float ks[8] = {sk[0].x, sk[0].y, sk[0].z, sk[0].w, sk[1].x, sk[1].y, sk[1].z, sk[1].w};
        float vs[8] = {sv[0].x, sv[0].y, sv[0].z, sv[0].w, sv[1].x, sv[1].y, sv[1].z, sv[1].w};
#pragma unroll
        for (int j = 0; j < 8; ++j) {  // a NaN V scale makes the score NaN, where the mask can drop it
            ks[j] = vs[j] == vs[j] ? ks[j] * kScore : vs[j];
            vs[j] = fmaxf(vs[j], 0.0f);
        }
        if (next < rg.end) {
            load_s(nblk);
            load_k(nblk);
        }
        if (ok) {
            float p[8], top = 0.0f, m = -INFINITY;
#pragma unroll
            for (int j = 0; j < 8; ++j) p[j] = (j < 4 ? s0[j & 3] : s1[j & 3]) * ks[j];
            // whole: every row of the tile attends every key of the block
            const int k0 = kb << 5;
            const bool whole = k0 + 31 <= rg.p_first && k0 + 31 < rg.limit &&
                               (a.window <= 0 || k0 > rg.p_last - a.window);
            if (!whole) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int key = k0 + kv_octet_key(g, j);
                    if (key > pos || key < first || key >= rg.limit) p[j] = -INFINITY, vs[j] = 0.0f;
                }
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                m = fmaxf(m, p[j]);
                top = fmaxf(top, vs[j]);
            }
            m = max_over_quads(m);
            top = max_over_quads(top);
            const int en = max(eo, int(__float_as_uint(top) >> 23) - 126);  // top < 2^en
            m = fmaxf(mx, ceilf(m * qs));
            float add = 0.0f;
            const float al = __builtin_amdgcn_exp2f(mx - m), f = al * ldexpf(1.0f, max(eo - en, -250));
            eo = en;
            mx = m;
            const float unit = ldexpf(1.0f, -eo), up = 14.0f - m;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float e = __builtin_amdgcn_exp2f(fmaf(p[j], qs, up));
                add += e;
                p[j] = e * (vs[j] * unit);
            }
            l = fmaf(l, al, add);
            h8 ph, pl;
            split8(p, ph, pl);
            if (__ballot(f != 1.0f)) {
#pragma unroll
                for (int i = 0; i < T; ++i) o[i] *= f;
            }
#pragma unroll
            for (int i = 0; i < T; ++i) {
                h8 fv;
                if (TYPE == WV_KV_F16) {
                    fv = as_half(vr[i]);
                } else {
                    const uint4 u = vr[i / 2];
                    fv = i % 2 ? q8_half(u.z, u.w) : q8_half(u.x, u.y);
                }
                o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fv, pl, o[i], 0, 0, 0);
                o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fv, ph, o[i], 0, 0, 0);
            }
        }
        if (next < rg.end) load_v(nblk);
        kb = next;
        ok = nok;
    }

    // the waves' rows y_w = O_w / l_w, each of its own keys' V, weighed by their shares of L = sum_w 2^(m_w - M) l_w:
    // no value on the way is larger than the largest |V|
    l = sum_over_quads(l);
    const float back = ldexpf(1.0f, max(eo, -126)), wl = l != 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
    for (int i = 0; i < T; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int md = 4 * g + k;
            const int d = TYPE == WV_KV_F16 ? 16 * i + md : 32 * (i / 2) + 2 * md + i % 2;
            red[wave][n][d] = o[i][k] * wl * back;
        }
    if (g == 0) {
        rm[wave][n] = mx;
        rl[wave][n] = l;
    }
    __syncthreads();
    const int r = threadIdx.x >> 4, c = threadIdx.x & 15;
    const int orow = t.r0 + r;
    if (orow >= t.rows) return;
    float M = -INFINITY, w[4], L = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (rl[i][r] != 0.0f) M = fmaxf(M, rm[i][r]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        w[i] = rl[i][r] != 0.0f ? __builtin_amdgcn_exp2f(rm[i][r] - M) * rl[i][r] : 0.0f;
        L += w[i];
    }
    const int tok = t.q0 + orow / G, head = kvh * G + orow % G;
    const float inv = L != 0.0f ? 1.0f / L : 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] *= inv;
    float* dst = a.part ? a.part + ((int64_t(tok) * a.n_heads + head) * a.splits + sp) * LD
                        : a.out + int64_t(tok) * a.os + head * HD;
#pragma unroll
    for (int d = c; d < HD; d += 16) {
        float x = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (w[i] != 0.0f) x += w[i] * red[i][r][d];
        dst[d] = x;
    }
    if (a.part && c == 0) {
        dst[HD] = M;
        dst[HD + 1] = L;
    }
}

// With ONCE a sequence's first tile, commonly its only one, is its block's
// without a search: 256 sequences of 100 fp16 keys 33 us against 40.
template <int HD, int TYPE, bool ONCE>
__global__ void __launch_bounds__(256, 2) k_kv_attn_rows(KvAttn a, int G, int max_rows, int tile0) {
    Tile t;
    const int y = tile0 + int(blockIdx.y);
    if (ONCE && y < a.n_seqs) {
        t.seq = y;
        t.q0 = min(max(a.cu[y], 0), a.n_tokens);
        t.n = min(max(a.cu[y + 1], t.q0), a.n_tokens) - t.q0;
        t.rows = t.n * G;
        t.kv_len = max(a.kv_len[y], 0);
        if (!t.n) return;
    } else if (!find_tile<16>(a, G, ONCE ? y - a.n_seqs : y, 1, max_rows, t, ONCE)) {
        return;
    }
    attn_rows<HD, TYPE, ONCE>(a, G, t, blockIdx.x, blockIdx.z);
}

// Many rows: 128 query rows of one sequence and KV head per block, 32 to a
// wave, over blocks of 32 keys that the four waves stage through LDS, as fp16
// codes in operand order (a 16-byte unit per lane, so staging and reading are
// linear and free of bank conflicts). S^T = K Q^T on 32x32x16 products leaves
// a lane with one row (l & 31) and the 8 keys of octets h and 2 + h (h = l >>
// 5), which are its operand of O^T += V^T P^T.
//
// A key block costs a wave 32 products (1024 cycles of the matrix unit) and
// about as long on the vector unit, so one iteration holds three key blocks:
// the products O += V P of the last one and S of the next one run under the
// exponentials of the one between. The codes of the key block after those are
// on their way into registers. With the scales lies the exponent of their
// largest, which is what E takes of a key block that a wave's rows attend whole.
// A row's E is its own: one multiplication a probability, 2.6 % of a long chunk
// against an E for the whole block, which took bits from rows whose mask hides a
// large V. A second copy of the step for such rows costs the others as much.
// 2048 tokens of 32 heads over 16384 int8 keys: 982 to 994 us across cards, up
// to 1050 TFLOP/s of two-term products, where an fp16 library product of 8192^3
// reaches 1155. The matrix unit is busy 48 % of the cycles, the vector unit's
// issue 53 %; without the exponentials it would take 0.95 of that, without the
// products 0.90. A prompt of 2047 tokens: 100 us, for half of which the longest
// tile runs alone on its CU. Dropped, since they gained nothing: two groups of
// four waves half a tile apart, or on halves of the keys; a barrier every second
// step; steps of 64 keys.
template <int HD, int TYPE>
__global__ void __launch_bounds__(256, 2) k_kv_attn_tile(KvAttn a, int G, int min_rows, int tile0) {
    constexpr int E = TYPE == WV_KV_F16 ? 2 : 1;
    constexpr int BB = 32 * HD * E;   // bytes of a block's codes
    constexpr int S = HD / 16;        // k steps of a score product
    constexpr int T = HD / 32;        // dim tiles of the output
    constexpr int UN = 32 * HD / 8;   // 16-byte fp16 units of a staged block
    constexpr int CU = BB / 16;       // 16-byte units of a block's codes
    constexpr int NU = (CU + 255) / 256;  // 16-byte loads of a thread
    constexpr int LD = HD + 4;
    __shared__ u4 lk[2][UN], lv[2][UN];
    __shared__ float ls[4][kKvScales];  // K and V scales by octet
    __shared__ float lt[4];             // exponent of the largest V scale

    const int kvh = blockIdx.x, sp = blockIdx.z;
    // a sequence's later tiles walk more keys and start first; where all blocks
    // run at once, two to a CU, the second half goes up again, so that the two
    // of a CU walk about as many keys as those of any other
    const int half = (gridDim.y + 1) / 2, y = int(blockIdx.y);
    const bool once = gridDim.x * gridDim.y * gridDim.z <= 512;
    const int idx = tile0 + (once && y >= half ? y - half : int(gridDim.y) - 1 - y);
    Tile t;
    if (!find_tile<128>(a, G, idx, min_rows, INT32_MAX, t)) return;
    const Range rg = tile_range<128>(a, t, G, sp, 8);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 31, h = lane >> 5;

    const int wr0 = t.r0 + 32 * wave;  // the wave's first row
    const bool busy = wr0 < t.rows;
    const int row = min(wr0 + n, t.rows - 1);
    const int pos = t.kv_len - t.n + row / G;
    const int first = a.window > 0 ? pos - a.window + 1 : 0;
    const int w_first = t.kv_len - t.n + min(wr0, t.rows - 1) / G;       // positions of the wave's first
    const int w_last = t.kv_len - t.n + min(wr0 + 31, t.rows - 1) / G;   // and last row

    const int32_t* pages = a.pages + int64_t(t.seq) * a.max_pages;
    const int pb = a.c.page_shift - 5;
    // Key block i of the range; one past it is read as the last and masked. Lane l holds the page of the
    // i'th with i % 64 = l: asked for in ascending order, the table is read once in 64.
    const int nb = rg.end - rg.begin;
    int pg64 = 0;
    auto block_at = [&](int i, bool& ok) {
        if ((i & 63) == 0) pg64 = pages[(rg.begin + min(i + lane, nb - 1)) >> pb];
        const int pg = __builtin_amdgcn_readlane(pg64, i & 63);
        ok = i < nb && unsigned(pg) < unsigned(a.c.n_pages);
        return kv_block(a.c, ok ? pg : 0, kvh, ((rg.begin + i) & ((1 << pb) - 1)) << 5);
    };
    const bool loads = CU >= 256 || tid < CU;
    u4 kr[NU], vr[NU];
    float sk = 0.0f, sv = 0.0f;
    int64_t kblk = 0, vblk = 0;  // the blocks of kr and of the V codes to load next
    auto load_k = [&](int64_t blk) {
        if (loads)
#pragma unroll
            for (int i = 0; i < NU; ++i)
                kr[i] = *reinterpret_cast<const u4*>(a.c.k + blk * BB + (i * 256 + tid) * 16);
    };
    auto load_s = [&](int64_t blk) {  // lanes 0..31: in order of octets
        const float* p = a.c.s + blk * kKvScales + (n >> 3) * 16 + (n & 7);
        sk = p[0];
        sv = p[8];
    };
    auto load_v = [&](int64_t blk) {
        if (loads)
#pragma unroll
            for (int i = 0; i < NU; ++i)
                vr[i] = *reinterpret_cast<const u4*>(a.c.v + blk * BB + (i * 256 + tid) * 16);
    };
    auto stage_k = [&](int buf) {
        if (loads)
#pragma unroll
            for (int i = 0; i < NU; ++i) {
                const int u = i * 256 + tid;
                if (TYPE == WV_KV_F16) {
                    lk[buf][u] = kr[i];
                } else {
                    u4* d = &lk[buf][(u >> 5) * 64 + (u & 31)];  // units 2c and 2c + 1 of a key
                    d[0] = __builtin_bit_cast(u4, q8_half(kr[i].x, kr[i].y));
                    d[32] = __builtin_bit_cast(u4, q8_half(kr[i].z, kr[i].w));
                }
            }
    };
    auto stage_s = [&](int kb, bool ok, int ring) {
        const int key = (kb << 5) + kv_octet_key(n >> 3, n & 7);
        const float v = ok && key < rg.limit ? fmaxf(sv, 0.0f) : 0.0f;
        const int et = int(max_of_32(v) >> 23) - 126;  // the largest is below 2^et
        if (lane < 32) {
            float* d = &ls[ring][(n >> 3) * 16 + (n & 7)];
            d[0] = sv == sv ? sk * kScore : sv;  // a NaN V scale makes the score NaN, where the mask can drop it
            d[8] = v;
        }
        if (lane == 0) lt[ring] = float(et);
    };
    auto stage_v = [&](int buf) {
        if (loads)
#pragma unroll
            for (int i = 0; i < NU; ++i) {
                const int u = i * 256 + tid;
                if (TYPE == WV_KV_F16) {
                    lv[buf][u] = vr[i];
                } else {
                    // two dims of an octet, side by side: every other four lanes store the second one
                    // first, so that eight lanes reach all banks
                    const u4 v0 = __builtin_bit_cast(u4, q8_half(vr[i].x, vr[i].y));
                    const u4 v1 = __builtin_bit_cast(u4, q8_half(vr[i].z, vr[i].w));
                    const int f = (tid >> 2) & 1;
                    lv[buf][2 * u + f] = f ? v1 : v0;
                    lv[buf][2 * u + 1 - f] = f ? v0 : v1;
                }
            }
    };

    h8 qh[S], ql[S];
    float qs;
    {
        const float* qp = a.q + int64_t(t.q0 + row / G) * a.qs + (kvh * G + row % G) * HD + 8 * h;
        float x[S][8], m = 0.0f;
#pragma unroll
        for (int s = 0; s < S; ++s)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                x[s][j] = qp[16 * s + j];
                m = fmaxf(m, fabsf(x[s][j]));
            }
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(m), __float_as_uint(m), false, false);
        float inv;
        qs = row_unit(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])), a.scale, inv);
#pragma unroll
        for (int s = 0; s < S; ++s) {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[s][j] *= inv;
            split8(x[s], qh[s], ql[s]);
        }
    }
    f16v o[T];
#pragma unroll
    for (int i = 0; i < T; ++i)
#pragma unroll
        for (int k = 0; k < 16; ++k) o[i][k] = 0.0f;
    float mx = kNoMax, l = 0.0f, er = -113.0f;  // er: E of the lane's row (no scale is smaller)
    u4 ph[2] = {}, pl[2] = {};  // the probabilities that wait for their product, as fp16

    auto qk = [&](int buf, f16v& s) {
#pragma unroll
        for (int k = 0; k < 16; ++k) s[k] = 0.0f;
#pragma unroll
        for (int c = 0; c < S; ++c) {
            const h8 x = as_half(lk[buf][(2 * c + h) * 32 + n]);
            s = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, ql[c], s, 0, 0, 0);
            s = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, qh[c], s, 0, 0, 0);
        }
    };
    auto pv = [&](int buf) {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            h8 fv[T];
#pragma unroll
            for (int i = 0; i < T; ++i) {
                fv[i] = as_half(lv[buf][(2 * q + h) * HD + 32 * i + n]);
                o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fv[i], as_half(pl[q]), o[i], 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < T; ++i) o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fv[i], as_half(ph[q]), o[i], 0, 0, 0);
        }
    };

    bool ok0 = false, ok1 = false, ok2 = false;  // whether the key blocks b, b + 1, b + 2 exist
    f16v sa, sb;
    if (nb) {
        const int64_t first_blk = block_at(0, ok0);
        load_k(first_blk);
        load_v(first_blk);
        vblk = block_at(1, ok1);
        kblk = block_at(2, ok2);
        stage_k(0);
        load_k(vblk);
        if (2 * tid < UN) lv[1][2 * tid] = lv[1][2 * tid + 1] = u4{};  // times P = 0 in the first iteration
        if (wave == 0) {
            load_s(first_blk);
            stage_s(rg.begin, ok0, 0);
            load_s(vblk);
            stage_s(rg.begin + 1, ok1, 1);
            load_s(kblk);
        }
        stage_k(1);
        load_k(kblk);
    }
    __syncthreads();
    // Key block b, its scores in s0: those of b + 1 into s1.
    auto step = [&](int b, f16v& s0, f16v& s1) {
        const int k0 = (rg.begin + b) << 5, cur = b & 1, ring = b & 3;
        const bool live = busy && ok0 && k0 <= w_last && !(a.window > 0 && k0 + 31 <= w_first - a.window);
        const bool whole = live && k0 + 31 <= w_first && k0 + 31 < rg.limit && (a.window <= 0 || k0 > w_last - a.window);
        f4 ks[4];
#pragma unroll
        for (int q = 0; q < 4; ++q)
            ks[q] = *reinterpret_cast<const f4*>(&ls[ring][(2 * (q >> 1) + h) * 16 + 4 * (q & 1)]);
        const float et = lt[ring];
        auto v_at = [&](int f) { return as_half(lv[cur ^ 1][(2 * (f / T) + h) * HD + 32 * (f % T) + n]); };
        auto k_at = [&](int c) { return as_half(lk[cur ^ 1][(2 * c + h) * 32 + n]); };
        h8 f0 = v_at(0), f1 = v_at(1);
#pragma unroll
        for (int i = 0; i < 16; ++i) s0[i] *= ks[i >> 2][i & 3];
        if (!whole) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int key = k0 + 8 * (i >> 2) + 4 * h + (i & 3);
                if (!live || key > pos || key < first || key >= rg.limit) s0[i] = -INFINITY;
            }
        }
        // O += V P of key block b - 1, two dim tiles at a time. Between the products, piece by piece: K of
        // b + 2 and V of b into the buffers that the last barrier freed, the loads after those, the maximum.
        // The pins keep products and pieces in turn.
        float m = -INFINITY, al = 0.0f, up = 0.0f;
        bool ok3 = false;
        auto piece = [&](int i) {
            if (i == 0) stage_k(cur);
            if (i == T / 2) stage_v(cur);
            if (i == T) {
                load_v(vblk);
                vblk = kblk;
                kblk = block_at(b + 3, ok3);
                load_k(kblk);
            }
            if (i == 2 * T - 2) {
#pragma unroll
                for (int e = 0; e < 16; ++e) m = fmaxf(m, s0[e]);
                pin(m);
            }
            if (i == 2 * T - 1) {
                const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(m), __float_as_uint(m), false, false);
                m = fmaxf(mx, ceilf(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])) * qs));
                al = __builtin_amdgcn_exp2f(mx - m);
                up = 14.0f - m;
                mx = m;
                pin(up);
            }
        };
        h8 x[2] = {k_at(0), k_at(1)};
#pragma unroll
        for (int f = 0; f < 2 * T; f += 2) {
            const int q = f / T, i = f % T;
            h8 g0 = f0, g1 = f1;
            pin(g0), pin(g1);
            if (f + 2 < 2 * T) f0 = v_at(f + 2), f1 = v_at(f + 3);
            o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(g0, as_half(pl[q]), o[i], 0, 0, 0);
            o[i + 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(g1, as_half(pl[q]), o[i + 1], 0, 0, 0);
            piece(f);
            pin(g0), pin(g1);
            o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(g0, as_half(ph[q]), o[i], 0, 0, 0);
            o[i + 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(g1, as_half(ph[q]), o[i + 1], 0, 0, 0);
            piece(f + 1);
        }
        float en = er;
        if (whole) {
            en = fmaxf(er, et);
        } else if (live) {
            float top = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const f4 v = *reinterpret_cast<const f4*>(&ls[ring][(2 * (i >> 1) + h) * 16 + 8 + 4 * (i & 1)]);
#pragma unroll
                for (int k = 0; k < 4; ++k) top = fmaxf(top, s0[4 * i + k] != -INFINITY ? v[k] : 0.0f);
            }
            const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
            en = fmaxf(er, float(int(max(r[0], r[1]) >> 23) - 126));
        }
        const float f = al * __builtin_amdgcn_exp2f(er - en), unit = __builtin_amdgcn_exp2f(-en);
        l *= al;
        er = en;
        // The scores of b + 1; between the products the probabilities of b, some keys at a time
#pragma unroll
        for (int e = 0; e < 16; ++e) s1[e] = 0.0f;
        float add[2] = {0.0f, 0.0f};
        f4 vs[2];
        vs[0] = *reinterpret_cast<const f4*>(&ls[ring][h * 16 + 8]);
#pragma unroll
        for (int c = 0; c < S; ++c) {
            h8 y = x[c & 1];
            pin(y);
            if (c + 2 < S) x[c & 1] = k_at(c + 2);
            if (c % (S / 4) == 0 && c < S - S / 4)
                vs[(4 * c / S + 1) & 1] = *reinterpret_cast<const f4*>(
                    &ls[ring][(2 * ((4 * c / S + 1) >> 1) + h) * 16 + 8 + 4 * ((4 * c / S + 1) & 1)]);
            s1 = __builtin_amdgcn_mfma_f32_32x32x16_f16(y, ql[c], s1, 0, 0, 0);
            s1 = __builtin_amdgcn_mfma_f32_32x32x16_f16(y, qh[c], s1, 0, 0, 0);
#pragma unroll
            for (int e = 16 / S * c; e < 16 / S * (c + 1); e += 2) {
                const int q = e / 8, i = e % 8 / 2;
                const float e0 = __builtin_amdgcn_exp2f(fmaf(s0[e], qs, up));
                const float e1 = __builtin_amdgcn_exp2f(fmaf(s0[e + 1], qs, up));
                add[q] += e0;
                add[q] += e1;
                const float p0 = e0 * unit * vs[(e >> 2) & 1][e & 3], p1 = e1 * unit * vs[(e >> 2) & 1][(e + 1) & 3];
                const auto hi = __builtin_amdgcn_cvt_pkrtz(p0, p1);
                const h2 lo = {_Float16(fmaf(float(hi[0]), -1.0f, p0)), _Float16(fmaf(float(hi[1]), -1.0f, p1))};
                uint32_t wh = __builtin_bit_cast(uint32_t, hi), wl = __builtin_bit_cast(uint32_t, lo);
                pin(wh), pin(wl), pin(add[q]);
                ph[q][i] = wh, pl[q][i] = wl;
            }
        }
        l += add[0] + add[1];
        if (wave == 0) {
            stage_s(rg.begin + b + 2, ok2, (b + 2) & 3);
            load_s(kblk);
        }
        ok0 = ok1, ok1 = ok2, ok2 = ok3;
        if (__ballot(f != 1.0f)) {
#pragma unroll
            for (int i = 0; i < T; ++i)
#pragma unroll
                for (int k = 0; k < 16; ++k) o[i][k] *= f;
        }
        lds_barrier();
    };
    if (nb) qk(0, sa);
    // The first step stages into the buffer that qk(0) reads.
    lds_barrier();
    int b = 0;
    for (; b + 1 < nb; b += 2) {
        step(b, sa, sb);
        step(b + 1, sb, sa);
    }
    if (b < nb) step(b++, sa, sb);
    if (nb) pv((nb - 1) & 1);
    if (!busy || wr0 + n >= t.rows) return;
    const auto lr = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
    l = __uint_as_float(lr[0]) + __uint_as_float(lr[1]);
    const int64_t orow = int64_t(t.q0 + row / G);
    const int head = kvh * G + row % G;
    const float back = ldexpf(1.0f, int(er));
    const float inv = l != 0.0f ? 1.0f / l : 0.0f;  // back / l may be subnormal
    float* dst = a.part ? a.part + ((orow * a.n_heads + head) * a.splits + sp) * LD : a.out + orow * a.os + head * HD;
    const bool al = a.part || (!(reinterpret_cast<uintptr_t>(a.out) & 15) && !(a.os & 3));
#pragma unroll
    for (int i = 0; i < T; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            f4 x;
#pragma unroll
            for (int k = 0; k < 4; ++k) x[k] = o[i][4 * q + k] * inv * back;
            float* d = dst + 32 * i + 8 * q + 4 * h;
            if (al) {
                *reinterpret_cast<f4*>(d) = x;
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k) d[k] = x[k];
            }
        }
    if (a.part && h == 0) {
        dst[HD] = mx;
        dst[HD + 1] = l;
    }
}

// The key ranges of one (token, head) row joined: the ranges' maxima and sums
// weigh their rows, each divided by its own sum already, added in the order of
// the ranges by four waves.
// 3 us for one token's 32 rows of 10 ranges: a launch.
template <int HD>
__global__ void __launch_bounds__(256) k_kv_attn_join(KvAttn a) {
    constexpr int LD = HD + 4, W = HD / 64;
    __shared__ float red[4][HD];
    const int tok = blockIdx.x, head = blockIdx.y;
    if (tok < a.cu[0] || tok >= min(a.cu[a.n_seqs], a.n_tokens)) return;
    const float* p = a.part + (int64_t(tok) * a.n_heads + head) * a.splits * LD;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float m = -INFINITY, l = 0.0f;
    if (lane < a.splits) {
        m = p[lane * LD + HD];
        l = p[lane * LD + HD + 1];
    }
    const float M = wave_maximum(l != 0.0f ? m : -INFINITY);
    float w = l != 0.0f ? __builtin_amdgcn_exp2f(m - M) * l : 0.0f;
    const float L = wave_total(w);
    w = L != 0.0f ? w / L : 0.0f;
    float x[W];
#pragma unroll
    for (int i = 0; i < W; ++i) x[i] = 0.0f;
    for (int s0 = wave; s0 < a.splits; s0 += 16) {  // four ranges' rows in flight
        float y[4][W];
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int i = 0; i < W; ++i) y[k][i] = s0 + 4 * k < a.splits ? p[(s0 + 4 * k) * LD + W * lane + i] : 0.0f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float ws = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(w), (s0 + 4 * k) & 63));
#pragma unroll
            for (int i = 0; i < W; ++i)
                if (s0 + 4 * k < a.splits) x[i] += ws * y[k][i];
        }
    }
#pragma unroll
    for (int i = 0; i < W; ++i) red[wave][W * lane + i] = x[i];
    __syncthreads();
    if (threadIdx.x < HD) {
        const int d = threadIdx.x;
        const float y = red[0][d] + red[1][d] + red[2][d] + red[3][d];
        a.out[int64_t(tok) * a.os + head * HD + d] = y;
    }
}

}  // namespace

// How a call is run. The tile kernel reads and converts the keys once for 128
// rows and the row kernel for 16, but a tile steps through its key blocks one
// after the other, 1.4 us each for one block a CU and 2.0 for two, so that few
// tiles, or short ones, leave the GPU waiting. This compares what the two
// take, in us, fitted to calls of 128 to 3500 new tokens over 300 to 50000
// keys. Row against tile kernel as measured, 32 heads over 8, head_dim 128: 512
// new over 512 keys 23 / 32, over 16384 552 / 302; 1024 over 1024 50 / 56, over
// 4096 230 / 172; 1508 over 1508 98 / 84; 1900 over 16384 2460 / 957; 1900 with
// a window of 512 96 / 54; head_dim 64, 1900 over 1900 76 / 91. Of a batch, the
// tile kernel takes the sequences of more than kFewRows rows.
KvPlan kv_attn_plan(const KvView& c, int n_seqs, int n_tokens, int max_pages, int max_q, int n_heads, int window) {
    if (!n_seqs || !n_tokens) return {false, false, 1};
    const int64_t G = n_heads / c.n_kv, rows = n_tokens * G;
    const int64_t most_q = max_q ? std::min(max_q, n_tokens) : (n_tokens + n_seqs - 1) / n_seqs;
    const int64_t width = int64_t(max_pages) << c.page_shift;
    const int64_t seqs = std::min(n_seqs, n_tokens);
    // key blocks that the last tile of `RT` rows walks, and one on average
    const auto last = [&](int64_t RT) {
        return double(window > 0 ? std::min<int64_t>(width, window + RT / G + 31) : width) / 32.0;
    };
    const double causal = window > 0 ? 0.0 : double(std::min(most_q, width)) / 64.0;
    const int64_t keys = window > 0 ? std::min<int64_t>(width, int64_t(window) + most_q) : width;
    const int64_t blocks = std::max<int64_t>((keys + 31) / 32, 1);
    const int64_t t16 = std::max<int64_t>((rows + 15) / 16, seqs) * c.n_kv;
    if (most_q * G >= kTileRows) {
        const int64_t t128 = std::max<int64_t>((rows + 127) / 128, seqs) * c.n_kv;
        const int64_t s128 = std::max<int64_t>(1, std::min<int64_t>({512 / t128, blocks / 32, kMaxSplits}));
        const bool wide = c.hd == 128;
        // what the last tile takes, or all of them at two blocks a CU, and the join's partial rows
        double tile = (wide ? 15.0 : 10.0) + std::max(last(128) / double(s128) * (wide ? 1.6 : 1.25),
                                                      double(t128) * (last(128) - causal) / 256.0 * (wide ? 1.15 : 0.9));
        if (s128 > 1) tile += 5.0 + double(t128 * s128) * 128.0 * double(c.hd + 4) * 8.0 / 5.2e6;
        const double steps = double(t16) * (last(16) - 0.65 * causal);
        double row = 3.0 + double(t16) * (1.8 / 512.0) + steps / (wide ? 1150.0 : 2300.0);
        const double block_bytes = 64.0 * c.hd * kv_code_bytes(c.type);
        if (last(16) * block_bytes > 2e6)  // more than stays in an L2
            row = std::max(row, double(t16) * (last(16) - causal) * block_bytes / 11e6);
        if (tile < row) return {true, false, int(s128)};
    }
    // Row kernel: ranges for two blocks a CU; more cost their join more than they gain (8192 keys, one token:
    // 8 / 16 / 64 ranges 18.7 / 15.1 / 21.6 us). Its waves take four key blocks at a time, in 1.1 to 1.6 us, or
    // what the bytes take of sequences half as long as the longest; ranges add a launch of 4.5 us. One token,
    // 32 heads over 8, without and with ranges: 100 keys 6.3 / 11.1 us, 500 9.3 / 11.0, 1000 13.7 / 12.4, 2048
    // 22.1 / 12.6; 48 tokens of 2048 keys each 41.5 / 43.6.
    const double block_us = 64.0 * c.hd * kv_code_bytes(c.type) * double(seqs * c.n_kv) / 5.2e6;
    const auto walk = [&](int64_t n) {
        return std::max(double(blocks) / (4.0 * double(n)) * (c.hd == 128 ? 1.5 : 1.1), 0.5 * double(blocks) * block_us);
    };
    const int64_t best = int64_t(std::sqrt(1.6 * double(blocks)) + 0.5);
    const int64_t n = std::max<int64_t>(1, std::min<int64_t>({768 / t16, best, blocks / 4, kMaxSplits}));
    return {false, most_q * G <= 16, walk(1) <= walk(n) + 4.5 + 0.15 * double(n) ? 1 : int(n)};
}

size_t kv_attn_part_floats(const KvView& c, int n_tokens, int n_heads, int splits) {
    return splits > 1 ? size_t(n_tokens) * size_t(n_heads) * size_t(splits) * size_t(c.hd + 4) : 0;
}

int launch_kv_attn(const KvAttn& a, hipStream_t s) {
    const int G = a.n_heads / a.c.n_kv;
    const int64_t rows = int64_t(a.n_tokens) * G;
    const bool f16 = a.c.type == WV_KV_F16;
    auto go = [&](auto kern, int64_t tiles, int bound) {
        for (int64_t t0 = 0; t0 < tiles; t0 += kMaxGridY) {
            const dim3 grid{unsigned(a.c.n_kv), unsigned(std::min<int64_t>(tiles - t0, kMaxGridY)), unsigned(a.splits)};
            hipLaunchKernelGGL(kern, grid, dim3(256), 0, s, a, G, bound, int(t0));
        }
    };
    const bool many = a.many, few = !many || a.n_seqs > 1;
    if (few) {
        const int64_t tiles = (rows + 15) / 16 + a.n_seqs;
        const int most = many ? kFewRows : INT32_MAX;
        auto rows_go = [&](auto once, auto again) { a.once ? go(once, tiles, most) : go(again, tiles, most); };
        if (a.c.hd == 128)
            f16 ? rows_go(k_kv_attn_rows<128, WV_KV_F16, true>, k_kv_attn_rows<128, WV_KV_F16, false>)
                : rows_go(k_kv_attn_rows<128, WV_KV_Q8, true>, k_kv_attn_rows<128, WV_KV_Q8, false>);
        else
            f16 ? rows_go(k_kv_attn_rows<64, WV_KV_F16, true>, k_kv_attn_rows<64, WV_KV_F16, false>)
                : rows_go(k_kv_attn_rows<64, WV_KV_Q8, true>, k_kv_attn_rows<64, WV_KV_Q8, false>);
    }
    if (many) {
        const int64_t tiles = (rows + 127) / 128 + a.n_seqs;
        const int least = few ? kFewRows + 1 : 1;
        if (a.c.hd == 128)
            f16 ? go(k_kv_attn_tile<128, WV_KV_F16>, tiles, least)
                : go(k_kv_attn_tile<128, WV_KV_Q8>, tiles, least);
        else
            f16 ? go(k_kv_attn_tile<64, WV_KV_F16>, tiles, least)
                : go(k_kv_attn_tile<64, WV_KV_Q8>, tiles, least);
    }
    if (a.splits > 1) {
        const dim3 jg{unsigned(a.n_tokens), unsigned(a.n_heads)};
        if (a.c.hd == 128)
            hipLaunchKernelGGL(k_kv_attn_join<128>, jg, dim3(256), 0, s, a);
        else
            hipLaunchKernelGGL(k_kv_attn_join<64>, jg, dim3(256), 0, s, a);
    }
    return int(hipGetLastError());
}

}  // namespace wv

using namespace wv;

namespace {

// The checks of a batch's sizes.
int check_batch(const char* what, uint64_t cache, const wv_kv_batch* b, int32_t n_heads, int32_t window, KvCache& c) {
    if (!kv_lookup(cache, c)) return rt_fail(WV_E_HANDLE, "%s: unknown cache %llu", what, (unsigned long long)cache);
    if (!b) return rt_fail(WV_E_ARG, "%s: nil batch", what);
    if (n_heads <= 0 || n_heads % c.c.n_kv_heads || n_heads > 65535)
        return rt_fail(WV_E_SHAPE, "%s: %d heads over %d KV heads", what, n_heads, c.c.n_kv_heads);
    if (b->n_seqs < 0 || b->n_tokens < 0 || b->max_pages < 0 || b->max_q < 0 || window < 0)
        return rt_fail(WV_E_SHAPE, "%s: negative size (seqs %d, tokens %d, pages %d, max_q %d, window %d)", what,
                       b->n_seqs, b->n_tokens, b->max_pages, b->max_q, window);
    if (int64_t(b->max_pages) * c.c.page_size >= int64_t(1) << 31)
        return rt_fail(WV_E_SHAPE, "%s: a table of %d pages of %d positions (2^31 and more)", what, b->max_pages,
                       c.c.page_size);
    if (int64_t(b->n_tokens) * n_heads >= int64_t(1) << 31 || b->n_tokens > 1 << 28 || b->n_seqs > 1 << 24)
        return rt_fail(WV_E_SHAPE, "%s: %d tokens of %d heads, %d sequences in one call", what, b->n_tokens, n_heads,
                       b->n_seqs);
    return WV_OK;
}

}  // namespace

extern "C" {

int wv_kv_attention_scratch(uint64_t cache, const wv_kv_batch* batch, int32_t n_heads, int32_t window,
                            size_t* bytes) {
    KvCache c;
    const int rc = check_batch("wv_kv_attention_scratch", cache, batch, n_heads, window, c);
    if (rc) return rc;
    if (!bytes) return rt_fail(WV_E_ARG, "wv_kv_attention_scratch: nil bytes");
    const KvView v = c.layer(0);
    const int sp =
        kv_attn_plan(v, batch->n_seqs, batch->n_tokens, batch->max_pages, batch->max_q, n_heads, std::min(window, 1 << 30)).splits;
    *bytes = kv_attn_part_floats(v, batch->n_tokens, n_heads, sp) * sizeof(float);
    return WV_OK;
}

int wv_kv_attention_dev(uint64_t cache, int32_t layer, const wv_kv_batch* batch, const float* d_q, int64_t q_stride,
                        int32_t n_heads, float scale, int32_t window, float* d_out, int64_t out_stride,
                        void* d_scratch, size_t scratch_bytes, void* stream) {
    KvCache c;
    int rc = check_batch("wv_kv_attention", cache, batch, n_heads, window, c);
    if (rc) return rc;
    if (layer < 0 || layer >= c.c.n_layers)
        return rt_fail(WV_E_ARG, "wv_kv_attention: layer %d of %d", layer, c.c.n_layers);
    if (!(scale > 0.0f) || !std::isfinite(scale)) return rt_fail(WV_E_ARG, "wv_kv_attention: scale %g", double(scale));
    const int64_t w = int64_t(n_heads) * c.c.head_dim;
    if (!q_stride) q_stride = w;
    if (!out_stride) out_stride = w;
    if (q_stride < w || out_stride < w)
        return rt_fail(WV_E_SHAPE, "wv_kv_attention: row strides %lld and %lld under the row's %lld floats",
                       (long long)q_stride, (long long)out_stride, (long long)w);
    if (d_q && d_q == d_out && q_stride != out_stride)  // rows written would be others' queries still to be read
        return rt_fail(WV_E_SHAPE, "wv_kv_attention: out is q, at row strides of %lld and %lld", (long long)out_stride,
                       (long long)q_stride);
    if (!batch->n_seqs || !batch->n_tokens) return WV_OK;
    if (!d_q || !d_out || !batch->d_cu_q || !batch->d_kv_len || (batch->max_pages && !batch->d_pages))
        return rt_fail(WV_E_ARG, "wv_kv_attention: nil q/out/cu_q/kv_len/pages");
    (void)hipSetDevice(c.device);
    hipStream_t s = rt_stream(stream, c.device);
    KvAttn a{};
    a.c = c.layer(layer);
    a.q = d_q, a.out = d_out, a.qs = q_stride, a.os = out_stride;
    a.cu = batch->d_cu_q, a.kv_len = batch->d_kv_len, a.pages = batch->d_pages;
    a.n_seqs = batch->n_seqs, a.n_tokens = batch->n_tokens, a.max_pages = batch->max_pages;
    a.n_heads = n_heads, a.window = std::min(window, 1 << 30), a.scale = scale;
    const KvPlan plan = kv_attn_plan(a.c, a.n_seqs, a.n_tokens, a.max_pages, batch->max_q, n_heads, a.window);
    a.splits = plan.splits, a.many = plan.many, a.once = plan.once;
    const size_t floats = kv_attn_part_floats(a.c, a.n_tokens, n_heads, a.splits);
    RtScratch sc;
    if (d_scratch) {
        if (reinterpret_cast<uintptr_t>(d_scratch) & 15)
            return rt_fail(WV_E_ARG, "wv_kv_attention: scratch not 16-byte aligned");
        if (scratch_bytes < floats * sizeof(float))
            return rt_fail(WV_E_SHAPE, "wv_kv_attention: %zu bytes of scratch, needs %zu", scratch_bytes,
                           floats * sizeof(float));
        if (floats) a.part = static_cast<float*>(d_scratch);
    } else if (floats && rt_capturing(s)) {
        a.splits = 1;  // what a replay writes must not lie in a slot that other calls take
    } else if (floats) {
        if ((rc = sc.get(floats, s, "wv_kv_attention: scratch"))) return rc;
        a.part = sc.f();
    }
    const int e = launch_kv_attn(a, s);
    return e == hipSuccess ? WV_OK : rt_hip_fail(hipError_t(e), "wv_kv_attention: kernel launch");
}

}  // extern "C"
