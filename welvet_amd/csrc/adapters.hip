// adapters.hip — low-rank adapters of many requests beside a shared
// projection: y_t = base_t + s_a B_a (A_a x_t), a the adapter of t's sequence.
//
// Two launches: h = A x in ranges of the columns (so that one token's rows
// still fill the GPU), whose sums meet when B h reads them, in order of the
// ranges. A and B stay 16-bit, x, h and all sums are f32.
// Of few rows bound by two launches and the weights' latency: one token, two sets
// of rank 16 on 14336 x 4096, 3.3 + 3.8 us; 64 requests of one, three sets of rank
// 32 on 1024 x 4096, 7.2 + 5.9 (50 MB of A and B from the caches). Of many by base
// and y, and by x: 2184 rows of 12 requests, rank 64 on 14336 x 4096, 14.8 + 56.7 us
// (250 MB of base and y at a large copy's 5.1 TB/s: 49), fp16 13.9 + 42.3. Rows by
// adapter: 256 requests, 8 adapters of rank 64, three sets on 1024 x 4096, 15.6 + 8.9;
// of rank 128 on 4096 x 14336 21.0 + 18.3.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <mutex>
#include <new>
#include <type_traits>
#include <unordered_map>
#include <vector>

#include "../../include/welvet_hip.h"
#include "rt_internal.h"
#include "wave_ops.h"

namespace wv {
namespace {

constexpr int kMaxSets = 4;      // of a call
constexpr int kMaxRank = 256;
constexpr int kTile = 32;        // token rows of a block
// Rows of a tile up to which they go without matrix products. 8 sequences over 4096 x 4096, rank 16 / 64: of 4 rows
// 6.9 / 10.7 us, of 6 as tiles 8.8 / 10.1; of 8 rows without 8.6 / 15.6, as tiles 9.1 / 10.3.
constexpr int kFew = 4;
constexpr int kChunk = 512;      // columns that a wave takes at a time of such a row, 8 to a lane
constexpr int kMaxRanges = 32;   // of the columns
// How a call's rows are taken: FEW rows of a sequence at a time, tiles of a sequence, or tiles of an adapter.
constexpr int kTiles = 0, kGrouped = -1;
constexpr int kGroupIds = 256, kGroupSeqs = 1024;  // adapters and sequences of a grouped call, at most

struct Known {
    int32_t rank;
    float scale;
};
struct Set {
    wv_adapters_config c{};
    int device = 0;
    // Ranks, columns and rows as stored: multiples of 16, 64 and 32, zeros behind the adapter's own.
    int R = 0, C = 0, O = 0;
    uint16_t* a = nullptr;    // [n_adapters][R][C]
    uint16_t* b = nullptr;    // [n_adapters][O / 32][R / 8][32 rows][8 ranks]: 64 lanes' operands of a product lie together
    Known* known = nullptr;   // [n_adapters], rank 0: unset
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
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef float g4 __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));

// One set of a call as the kernels see it.
struct SetArgs {
    const uint16_t *a, *b;
    const Known* known;
    const float* base;
    float* y;
    float* h;  // [ranges][n_tokens][R]
    int64_t ys, bs;
    int rows, R, C, O, n_adapters;
    int block0;  // of the blocks over all sets' outputs, its first
};
struct Args {
    SetArgs set[kMaxSets];
    const float* x;
    const int32_t *cu, *which;
    int64_t xs;
    int cols, n_seqs, n_tokens, ranges, range;  // range: columns of one, a multiple of kChunk
    int n_sets, ranks;                           // ranks: R of all sets
    int ids;                                     // adapters of the set that has most
};

template <int TYPE>
__device__ __forceinline__ float low(uint32_t w) {
    return TYPE == WV_ADAPTER_BF16 ? __uint_as_float(w << 16) : float(__builtin_bit_cast(_Float16, uint16_t(w)));
}
template <int TYPE>
__device__ __forceinline__ float high(uint32_t w) {
    return TYPE == WV_ADAPTER_BF16 ? __uint_as_float(w & 0xffff0000) : float(__builtin_bit_cast(_Float16, uint16_t(w >> 16)));
}

// Token rows of one sequence, 32 at most, from t0 on, or of one adapter, as listed.
struct Tile {
    int t0, n, id;  // its adapter
    const int* list = nullptr;
    __device__ __forceinline__ int row(int i) const { return list ? list[i] : t0 + i; }
    __device__ __forceinline__ int from_first(int i) const { return list ? list[i] : i; }
};
// The rows of sequence s.
__device__ __forceinline__ int rows_of(const Args& a, int s, int& first) {
    first = min(max(a.cu[s], 0), a.n_tokens);
    return min(max(a.cu[s + 1], first), a.n_tokens) - first;
}
// Sum over this lane and those before it.
__device__ __forceinline__ int sum_so_far(int x) {
    x += dpp_i<kDppRowShr1>(0, x);
    x += dpp_i<kDppRowShr2>(0, x);
    x += dpp_i<kDppRowShr4, 0xf, 0xe>(0, x);
    x += dpp_i<kDppRowShr8, 0xf, 0xc>(0, x);
    x += dpp_i<kDppRowBcast15, 0xa>(0, x);
    return x + dpp_i<kDppRowBcast31, 0xc>(0, x);
}
// Tile `idx`: the first one of sequence idx, then all further ones in order of the sequences, found 64 sequences at a
// time. False: there is none. FEW: a sequence is one tile, whatever its length.
template <bool FEW>
__device__ __forceinline__ bool find_tile(const Args& a, int idx, Tile& t) {
    if (FEW || idx < a.n_seqs) {
        t.id = a.which[idx];
        t.n = rows_of(a, idx, t.t0);
        if (!FEW) t.n = min(t.n, kTile);
        return t.n > 0;
    }
    idx -= a.n_seqs;
    const int lane = threadIdx.x & 63;
    for (int base = 0; base < a.n_seqs; base += 64) {
        const int s = base + lane;
        int c0 = 0, n = 0;
        if (s < a.n_seqs) n = rows_of(a, s, c0);
        const int tiles = max((n + kTile - 1) / kTile - 1, 0), incl = sum_so_far(tiles);
        const int total = __builtin_amdgcn_readlane(incl, 63);
        if (idx < total) {
            const int w = __builtin_ctzll(__ballot(incl > idx));
            const int skip = kTile * (1 + idx - (__builtin_amdgcn_readlane(incl, w) - __builtin_amdgcn_readlane(tiles, w)));
            t.id = a.which[base + w];
            t.t0 = __builtin_amdgcn_readlane(c0, w) + skip;
            t.n = min(__builtin_amdgcn_readlane(n, w) - skip, kTile);
            return true;
        }
        idx -= total;
    }
    return false;
}

// Tile `idx` of the rows in order of their adapters (those without one last): every block counts the adapters' rows,
// finds its 32 of them and lists them in their order, so that blocks agree. 256 sequences at a time, a thread each.
__device__ __forceinline__ bool find_group(const Args& a, int idx, Tile& t) {
    __shared__ int count[kGroupIds + 1], list[kTile], sums[kGroupSeqs / 64];
    const int tid = threadIdx.x, lane = tid & 63;
    int key = -1, c0 = 0, n = 0;
    auto load = [&](int s) {
        n = 0;
        if (s < a.n_seqs) n = rows_of(a, s, c0), key = int(min(unsigned(a.which[s]), unsigned(a.ids)));
    };
    for (int i = tid; i <= a.ids; i += 256) count[i] = 0;
    __syncthreads();
    for (int base = 0; base < a.n_seqs; base += 256) {
        load(base + tid);
        if (n) atomicAdd(&count[key], n);
    }
    __syncthreads();
    int id = -1, skip = 0;
    for (int base = 0; base <= a.ids && id < 0; base += 64) {
        const int tiles = base + lane <= a.ids ? (count[base + lane] + kTile - 1) / kTile : 0, incl = sum_so_far(tiles);
        const int total = __builtin_amdgcn_readlane(incl, 63);
        if (idx < total) {
            const int w = __builtin_ctzll(__ballot(incl > idx));
            id = base + w;
            skip = kTile * (idx - (__builtin_amdgcn_readlane(incl, w) - __builtin_amdgcn_readlane(tiles, w)));
        }
        idx -= total;
    }
    if (id < 0) return false;
    int before = 0;
    for (int base = 0; base < a.n_seqs; base += 256) {
        if (a.n_seqs > 256) load(base + tid);
        const int rows = key == id ? n : 0, incl = sum_so_far(rows);
        int* l = sums + base / 64;
        if (lane == 63) l[tid >> 6] = incl;
        __syncthreads();
        int first = before + incl - rows - skip;  // its rows' places in the list
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            if (w < tid >> 6) first += l[w];
            before += l[w];
        }
        for (int i = max(-first, 0); i < rows && first + i < kTile; ++i) list[first + i] = c0 + i;
    }
    __syncthreads();
    t.t0 = 0;
    t.n = min(count[id] - skip, kTile);
    t.id = id < a.ids ? id : -1;
    t.list = list;
    return true;
}

// What this wave's lanes wrote to LDS is there for its other lanes.
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// 8 consecutive floats of a row, zeros behind its end.
__device__ __forceinline__ void load8(const float* x, int c, int cols, float* v) {
    if (c + 8 <= cols) {
        const f4 lo = *reinterpret_cast<const f4*>(x + c), hi = *reinterpret_cast<const f4*>(x + c + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = lo[i], v[4 + i] = hi[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = c + i < cols ? x[c + i] : 0.0f;
    }
}
template <int TYPE>
__device__ __forceinline__ void wide8(uint4 w, float* v) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) v[2 * i] = low<TYPE>(u[i]), v[2 * i + 1] = high<TYPE>(u[i]);
}

// Eight f32 values as NT terms of the weights' type, whose products with a weight are exact in f32. bf16: three terms
// hold all 24 bits, but for what lies under 2^-133, bf16's smallest (f32's normal values end at 2^-126). Lifting rows under
// 2^-94 from there was right and cost the others: 2000 rows of rank 128 at three projections 127 us for 119, 256 requests
// 26.0 for 25.1. fp16: two hold 22, of values that a power of two has brought into its range.
template <int TYPE>
struct Terms {
    static constexpr int N = TYPE == WV_ADAPTER_BF16 ? 3 : 2;
    uint4 t[N];
};
template <int TYPE>
__device__ __forceinline__ Terms<TYPE> split8(const float* x) {
    Terms<TYPE> r;
    uint32_t w[Terms<TYPE>::N][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float a = x[2 * i], b = x[2 * i + 1];
        if constexpr (TYPE == WV_ADAPTER_BF16) {
#pragma unroll
            for (int k = 0; k < 3; ++k) {  // truncated, the rest exactly
                w[k][i] = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
                a -= __uint_as_float(__float_as_uint(a) & 0xffff0000u);
                b -= __uint_as_float(__float_as_uint(b) & 0xffff0000u);
            }
        } else {
            const auto hi = __builtin_amdgcn_cvt_pkrtz(a, b);
            const h2 lo = {_Float16(fmaf(float(hi[0]), -1.0f, a)), _Float16(fmaf(float(hi[1]), -1.0f, b))};
            w[0][i] = __builtin_bit_cast(uint32_t, hi);
            w[1][i] = __builtin_bit_cast(uint32_t, lo);
        }
    }
#pragma unroll
    for (int k = 0; k < Terms<TYPE>::N; ++k) r.t[k] = make_uint4(w[k][0], w[k][1], w[k][2], w[k][3]);
    return r;
}
// acc += 32 rows of weights x 32 columns of values, 16 deep: the smallest terms first.
template <int TYPE>
__device__ __forceinline__ f16v product(uint4 w, const Terms<TYPE>& x, f16v acc) {
#pragma unroll
    for (int k = Terms<TYPE>::N - 1; k >= 0; --k) {
        if constexpr (TYPE == WV_ADAPTER_BF16)
            acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8, w), __builtin_bit_cast(b8, x.t[k]), acc, 0, 0, 0);
        else
            acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, w), __builtin_bit_cast(h8, x.t[k]), acc, 0, 0, 0);
    }
    return acc;
}
// Exponent e of a magnitude's bits (it is below 2^(e + 1)), within what a normal power of two in f32 brings to 2^14
// (2^(14 - e)) and back (2^(e - 14): from kLeast on; one less has no bits, and took whole rows with it); of the larger
// of this lane's and lane ^ 32's. What lies under 2^kLeast comes to less than 2^14, and to no less than fp16 holds.
constexpr int kLeast = -112;
__device__ __forceinline__ int exponent(uint32_t bits) { return min(max(int(bits >> 23) - 127, kLeast), 127); }
__device__ __forceinline__ int pair_exponent(float m) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(m), __float_as_uint(m), false, false);
    return exponent(max(r[0], r[1]));
}
__device__ __forceinline__ float power(int e) { return __uint_as_float(uint32_t(e + 127) << 23); }

// a's lower half of lanes plus its upper one, and b's in the upper half; a's rows 0 and 2 plus its 1 and 3, and b's in
// those; a row's total, in its last lane.
__device__ __forceinline__ float fold_halves(float a, float b) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float fold_rows(float a, float b) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float row_total(float x) {
    x += __int_as_float(dpp_i<kDppRowShr1>(0, __float_as_int(x)));
    x += __int_as_float(dpp_i<kDppRowShr2>(0, __float_as_int(x)));
    x += __int_as_float(dpp_i<kDppRowShr4, 0xf, 0xe>(0, __float_as_int(x)));
    return x + __int_as_float(dpp_i<kDppRowShr8, 0xf, 0xc>(0, __float_as_int(x)));
}

// h of NT of the tokens, those from `have` on the last one again: a wave takes every fourth group of four ranks, a lane 8
// columns at a time, and meets the others at a group's end. The first loads do not wait for the adapter's rank (there are
// 16 rows in A at least). Where the range is one chunk, the tokens' columns stay in registers and the next group of A is
// on its way while one is summed (3 to 8% of a call); with more chunks there are blocks enough to wait for.
template <int TYPE, int NT>
__device__ __forceinline__ void down_rows(const Args& a, const SetArgs& s, int t0, int have, int id, int c0, int c1, float* h) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int cl = c0 + 8 * lane;
    const uint16_t* A = s.a + int64_t(id) * s.R * s.C;
    uint4 w[4];
    float v[NT][8], sum[4][NT];
    auto load_x = [&](int c) {
#pragma unroll
        for (int n = 0; n < NT; ++n) load8(a.x + int64_t(t0 + min(n, have - 1)) * a.xs, cl + c, a.cols, v[n]);
    };
    auto load_w = [&](int r0, int c) {
        const int at = min(cl + c, s.C - 8);  // where there is no such column, x is 0
#pragma unroll
        for (int k = 0; k < 4; ++k) w[k] = *reinterpret_cast<const uint4*>(A + int64_t(r0 + k) * s.C + at);
    };
    auto clear = [&] {
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int n = 0; n < NT; ++n) sum[k][n] = 0.0f;
    };
    auto add = [&](const uint4 (&u)[4]) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            float f[8];
            wide8<TYPE>(u[k], f);
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 8; ++i) sum[k][n] = fmaf(f[i], v[n][i], sum[k][n]);
        }
    };
    // the sums over the lanes: the four ranks' in a row of 16 lanes each, then in its last
    auto store = [&](int r0, int rank) {
        const int r = r0 + (lane >> 4);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const float y = row_total(fold_rows(fold_halves(sum[0][n], sum[2][n]), fold_halves(sum[1][n], sum[3][n])));
            if ((lane & 15) == 15 && r < rank && n < have) h[int64_t(n) * s.R + r] = y;
        }
    };
    load_x(0);
    load_w(4 * wave, 0);
    const int rank = s.known[id].rank;
    if (c1 - c0 <= kChunk) {
        for (int r0 = 4 * wave; r0 < rank; r0 += 16) {
            const uint4 u[4] = {w[0], w[1], w[2], w[3]};
            load_w(r0 + 16 < rank ? r0 + 16 : r0, 0);
            clear();
            add(u);
            store(r0, rank);
        }
        return;
    }
    for (int r0 = 4 * wave; r0 < rank; r0 += 16) {
        clear();
        for (int c = 0; c < c1 - c0; c += kChunk) {
            if (c || r0 >= 16) load_x(c), load_w(r0, c);
            add(w);
        }
        store(r0, rank);
    }
}
// h of a short sequence, NT rows at a time.
template <int TYPE, int NT>
__device__ __forceinline__ void down_few(const Args& a, const SetArgs& s, const Tile& t, int id, int c0, int c1, float* h) {
    for (int n = 0; n < t.n; n += NT, h += NT * s.R) down_rows<TYPE, NT>(a, s, t.t0 + n, min(t.n - n, NT), id, c0, c1, h);
}

// h of a tile of tokens for all sets, whose ranks follow one another, 32 NR of them to a block, on products of 32 ranks
// x 32 tokens x 16 columns: a lane holds the same 16 columns of its rank's row and of its token's (lanes from 32 on the
// 16 behind those), straight from memory. The block's waves take every fourth 32 columns and meet in LDS.
template <int TYPE, int NR>
__device__ __forceinline__ void down_tile(const Args& a, const Tile& t, int range, int c0, int c1, float* lds) {
    constexpr int LD = 32 * NR + 4;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 31, hi = lane >> 5;
    const int row_n = t.row(min(n, t.n - 1));
    const float* x = a.x + int64_t(row_n) * a.xs;
    // rank r of all sets: its set, and the rank there
    auto set_of = [&](int& r) {
        int i = 0;
        while (i + 1 < kMaxSets && r >= a.set[i].R) r -= a.set[i++].R;
        return i;
    };
    const int r0 = 32 * NR * blockIdx.z;
    f16v acc[NR];
    const uint16_t* row[NR];
#pragma unroll
    for (int k = 0; k < NR; ++k) {
        int r = min(r0 + 32 * k + n, a.ranks - 1);
        const SetArgs& s = a.set[set_of(r)];
        // of a set that does not know the adapter, anything: nobody reads it
        const int id = unsigned(t.id) < unsigned(s.n_adapters) ? t.id : 0;
        row[k] = s.a + (int64_t(id) * s.R + r) * s.C;
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[k][i] = 0.0f;
    }
    float v[16];
    uint4 w[NR][2];
    auto load_a = [&](int c) {
#pragma unroll
        for (int k = 0; k < NR; ++k) {
            w[k][0] = *reinterpret_cast<const uint4*>(row[k] + c);
            w[k][1] = *reinterpret_cast<const uint4*>(row[k] + c + 8);
        }
    };
    auto load_x = [&](int c) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const f4 y = *reinterpret_cast<const f4*>(x + c + 4 * q);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[4 * q + i] = y[i];
        }
    };
    int e = kLeast;  // fp16: the token's sums so far are in units of 2^(e - 14)
    auto step = [&](auto next) {
        if constexpr (TYPE == WV_ADAPTER_F16) {
            float m = 0.0f;
#pragma unroll
            for (int i = 0; i < 16; ++i) m = fmaxf(m, fabsf(v[i]));
            const int en = max(e, pair_exponent(m));
            if (__ballot(en != e)) {
                const float f = ldexpf(1.0f, max(e - en, -200));
#pragma unroll
                for (int k = 0; k < NR; ++k) acc[k] *= f;
            }
            e = en;
            const float up = power(14 - e);
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] *= up;
        }
        const Terms<TYPE> x0 = split8<TYPE>(v), x1 = split8<TYPE>(v + 8);
        uint4 u[NR][2];
#pragma unroll
        for (int k = 0; k < NR; ++k) u[k][0] = w[k][0], u[k][1] = w[k][1];
        next();
#pragma unroll
        for (int k = 0; k < NR; ++k) acc[k] = product<TYPE>(u[k][0], x0, acc[k]);
#pragma unroll
        for (int k = 0; k < NR; ++k) acc[k] = product<TYPE>(u[k][1], x1, acc[k]);
    };
    // whole steps without a branch (what would be loaded behind the last one is that one again), then what is left
    // of a row, where A, padded with zeros to multiples of 64 columns, goes on
    const int steps = (min(c1, a.cols) - c0) / 32, mine = (steps - wave + 3) / 4;
    const int at = c0 + 32 * wave + 16 * hi;
    if (mine > 0) {
        load_x(at), load_a(at);
        for (int i = 0; i < mine; ++i) {
            const int c = at + 128 * min(i + 1, mine - 1);
            step([&] { load_x(c), load_a(c); });
        }
    }
    if (const int c = c0 + 32 * steps + 16 * hi; c0 + 32 * steps < min(c1, a.cols) && (steps & 3) == wave) {
        load8(x, c, a.cols, v);
        load8(x, c + 8, a.cols, v + 8);
        load_a(c);
        step([] {});
    }
    if constexpr (TYPE == WV_ADAPTER_F16) {
#pragma unroll
        for (int k = 0; k < NR; ++k) acc[k] *= power(e - 14);
    }
    // waves 2 and 3 to 0 and 1, then 1 to 0
#pragma unroll
    for (int step = 2; step >= 1; step /= 2) {
        float* mine = lds + ((wave & (step - 1)) * 32 + n) * LD + 4 * hi;
        __syncthreads();
        if (wave >= step && wave < 2 * step) {
#pragma unroll
            for (int k = 0; k < NR; ++k)
#pragma unroll
                for (int q = 0; q < 4; ++q)
#pragma unroll
                    for (int i = 0; i < 4; ++i) mine[32 * k + 8 * q + i] = acc[k][4 * q + i];
        }
        __syncthreads();
        if (wave < step) {
#pragma unroll
            for (int k = 0; k < NR; ++k)
#pragma unroll
                for (int q = 0; q < 4; ++q)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[k][4 * q + i] += mine[32 * k + 8 * q + i];
        }
    }
    if (wave == 0 && n < t.n) {
#pragma unroll
        for (int k = 0; k < NR; ++k)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                int r = r0 + 32 * k + 8 * q + 4 * hi;
                if (r >= a.ranks) continue;
                const SetArgs& s = a.set[set_of(r)];  // the ranks of a set are a multiple of 16
                *reinterpret_cast<f4*>(s.h + (int64_t(range) * a.n_tokens + row_n) * s.R + r) =
                    f4{acc[k][4 * q], acc[k][4 * q + 1], acc[k][4 * q + 2], acc[k][4 * q + 3]};
            }
    }
}

// FEW (1, kFew; kTiles and kGrouped: not so): the caller says that no sequence has more rows (if one has, they go FEW at a time). Without,
// the rows of a short one go singly: four at a time take registers that tiles want (18.5 us for 2000 rows of rank 64 over
// 4096 columns, else 19.6).
template <int TYPE, int NR, int FEW>
__global__ void __launch_bounds__(256) k_adapt_down(Args a, int tile0) {
    __shared__ float lds[FEW > 0 ? 1 : 2 * 32 * (32 * NR + 4)];
    Tile t;
    if (!(FEW == kGrouped ? find_group(a, tile0 + int(blockIdx.y), t) : find_tile<(FEW > 0)>(a, tile0 + int(blockIdx.y), t))) return;
    const int range = FEW > 0 ? blockIdx.x % a.ranges : blockIdx.x, c0 = range * a.range;
    auto few = [&](const SetArgs& s) {
        if (unsigned(t.id) < unsigned(s.n_adapters))
            down_few<TYPE, (FEW > 0 ? FEW : 1)>(a, s, t, t.id, c0, min(c0 + a.range, a.cols),
                                          s.h + (int64_t(range) * a.n_tokens + t.t0) * s.R);
    };
    if constexpr (FEW > 0) {
        few(a.set[blockIdx.x / a.ranges]);
    } else if (FEW == kTiles && t.n <= kFew) {
        for (int i = blockIdx.z; i < a.n_sets; i += gridDim.z) few(a.set[i]);
    } else if (t.id >= 0) {
        down_tile<TYPE, NR>(a, t, range, c0, min(c0 + a.range, a.set[0].C), lds);
    }
}

// Rows of h into LDS (NR * 32 + 4 floats each), the ranges summed in their order, with the adapter's scale. What lies
// behind the adapter's own ranks is anything until it is masked.
template <int NR>
__device__ __forceinline__ void stage_h(const Args& a, const SetArgs& s, const Tile& t, int n0, int rows, int rank,
                                        float scale, float* h) {
    constexpr int LD = 32 * NR + 4;
    for (int i = threadIdx.x; i < 8 * NR * rows; i += 256) {
        const int n = i / (8 * NR), r = 4 * (i % (8 * NR));
        f4 x = {0.0f, 0.0f, 0.0f, 0.0f};
        if (r < s.R && n0 + n < t.n) {
            const float* p = s.h + (int64_t(t.t0) + n0 + n) * s.R + r;
            const int64_t step = int64_t(a.n_tokens) * s.R;
            int k = 0;
            for (; k + 8 <= a.ranges; k += 8) {
                f4 y[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) y[j] = *reinterpret_cast<const f4*>(p + (k + j) * step);
#pragma unroll
                for (int j = 0; j < 8; ++j) x += y[j];
            }
            for (; k < a.ranges; ++k) x += *reinterpret_cast<const f4*>(p + k * step);
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = r + j < rank ? x[j] * scale : 0.0f;
        }
        *reinterpret_cast<f4*>(h + n * LD + r) = x;
    }
}

// y of the block's outputs for a few tokens, NT at a time: a thread takes an output, and has its row of B on the
// way before it looks at anything else.
template <int TYPE, int NR, int NT>
__device__ __forceinline__ void up_few(const Args& a, const SetArgs& s, const Tile& t, int id, int first, int last,
                                       const float* base, float* y, float* h) {
    constexpr int LD = 32 * NR + 4, NB = NR < 2 ? 4 : 8;  // 16-byte units of B that are loaded ahead
    const uint16_t* B = s.b + (int64_t(id) * s.O + first) * s.R;
    const int rank = s.known[id].rank;
    const float scale = s.known[id].scale;
    for (int n0 = 0; n0 < t.n; n0 += NT) {
        const int rows = min(t.n - n0, NT);
        for (int o = threadIdx.x; o - int(threadIdx.x) < last - first; o += 256) {
            const bool in = o < last - first;
            const uint16_t* row = B + int64_t(in ? o & ~31 : 0) * s.R + 8 * (o & 31);
            uint4 w[NB];
#pragma unroll
            for (int k = 0; k < NB; ++k) w[k] = 8 * k < s.R ? *reinterpret_cast<const uint4*>(row + 256 * k) : uint4{};
            float sum[NT];
#pragma unroll
            for (int n = 0; n < NT; ++n) sum[n] = in && n < rows ? base[(n0 + n) * s.bs + first + o] : 0.0f;
            if (o == int(threadIdx.x)) {
                if (n0) __syncthreads();
                stage_h<NR>(a, s, t, n0, rows, rank, scale, h);
                __syncthreads();
            }
            float add[NT] = {};
            auto unit = [&](uint4 u, int r) {
                float f[8];
                wide8<TYPE>(u, f);
#pragma unroll
                for (int n = 0; n < NT; ++n)
                    if (n < rows)
#pragma unroll
                        for (int i = 0; i < 8; ++i) add[n] = fmaf(f[i], h[n * LD + r + i], add[n]);
            };
#pragma unroll
            for (int k = 0; k < NB; ++k)
                if (8 * k < rank) unit(w[k], 8 * k);
            for (int r = 8 * NB; r < rank; r += 8) unit(*reinterpret_cast<const uint4*>(row + 32 * r), r);
#pragma unroll
            for (int n = 0; n < NT; ++n)
                if (in && n < rows) y[(n0 + n) * s.ys + first + o] = sum[n] + add[n];
        }
    }
}

// What up_tile keeps in LDS: the tile's h as operands, [16 ranks][term][lane] units of 16 bytes, the tokens' scales,
// and rows of 36 floats in which a wave's outputs change lanes (16 lanes' 16-byte accesses reach all banks).
constexpr int kSwap = 36;
template <int TYPE, int NR>
struct UpLds {
    uint4 h[2 * NR][Terms<TYPE>::N][64];
    uint32_t most[32];
    float swap[4][32 * kSwap];
};

// The tile's h: the ranges summed in their order, with the adapter's scale, as operands of the products. What lies
// behind the adapter's own ranks is anything until it is masked.
template <int TYPE, int NR>
__device__ __forceinline__ void stage_operands(const Args& a, const SetArgs& s, const Tile& t, int rank, float scale,
                                               UpLds<TYPE, NR>& l) {
    f4 x[NR];
    const int64_t step = int64_t(a.n_tokens) * s.R;
#pragma unroll
    for (int j = 0; j < NR; ++j) {
        const int i = threadIdx.x + 256 * j, n = i / (8 * NR), r = 4 * (i % (8 * NR));
        x[j] = f4{0.0f, 0.0f, 0.0f, 0.0f};
        if (r < s.R && n < t.n) {
            const float* p = s.h + int64_t(t.row(n)) * s.R + r;
            int k = 0;
            for (; k + 4 <= a.ranges; k += 4) {
                f4 y[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) y[c] = *reinterpret_cast<const f4*>(p + (k + c) * step);
#pragma unroll
                for (int c = 0; c < 4; ++c) x[j] += y[c];
            }
            for (; k < a.ranges; ++k) x[j] += *reinterpret_cast<const f4*>(p + k * step);
#pragma unroll
            for (int c = 0; c < 4; ++c) x[j][c] = r + c < rank ? x[j][c] * scale : 0.0f;
        }
    }
    if constexpr (TYPE == WV_ADAPTER_F16) {  // the token's largest, which its power of two goes by
        if (threadIdx.x < 32) l.most[threadIdx.x] = 0;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < NR; ++j) {
            const int n = (threadIdx.x + 256 * j) / (8 * NR);
            const float m = fmaxf(fmaxf(fabsf(x[j][0]), fabsf(x[j][1])), fmaxf(fabsf(x[j][2]), fabsf(x[j][3])));
            atomicMax(&l.most[n], __float_as_uint(m));
        }
        __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < NR; ++j) {
        const int i = threadIdx.x + 256 * j, n = i / (8 * NR), r = 4 * (i % (8 * NR));
        float v[8] = {x[j][0], x[j][1], x[j][2], x[j][3]};
        if constexpr (TYPE == WV_ADAPTER_F16) {
            const float up = power(14 - exponent(l.most[n]));
#pragma unroll
            for (int c = 0; c < 4; ++c) v[c] *= up;
        }
        const Terms<TYPE> w = split8<TYPE>(v);
#pragma unroll
        for (int k = 0; k < Terms<TYPE>::N; ++k)
            reinterpret_cast<uint2*>(&l.h[r / 16][k][n + 32 * ((r / 8) & 1)])[(r / 4) & 1] = make_uint2(w.t[k].x, w.t[k].y);
    }
    __syncthreads();
}

// y of the block's outputs for a tile, on products of 32 outputs x 32 tokens x 16 ranks. A lane ends with 16 outputs
// of one token; through LDS they become four times 4 side by side, 8 lanes a row, as base and y are read and written,
// past the caches (a prompt's rows are more than they hold). B and base of the next step are on their way meanwhile; a
// second step ahead takes the registers of a fourth block a CU and gained nothing.
template <int TYPE, int NR>
__device__ __forceinline__ void up_tile(const Args& a, const SetArgs& s, const Tile& t, int id, int rank, int first,
                                        int last, const float* base, float* y, UpLds<TYPE, NR>& l) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 31, hi = lane >> 5, m = lane >> 3, o4 = 4 * (lane & 7);
    const uint16_t* B = s.b + int64_t(id) * s.O * s.R + 8 * lane;
    float* swap = l.swap[wave];
    // Nothing in a step branches, so that loads stay on their way: rows behind the tile's last are that one again (to
    // the same place), ranks behind the stored ones the last ones (times h = 0), what would be loaded behind the last
    // whole 32 outputs are those again.
    const int whole = first + ((last - first) & ~31);
    int64_t rb[4], ry[4];
    int rs[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int r = min(8 * q + m, t.n - 1);
        const int64_t at = t.from_first(r);
        rb[q] = at * s.bs + o4, ry[q] = at * s.ys + o4, rs[q] = r * kSwap + o4;
    }
    uint4 w[2 * NR];
    f4 was[4];
    auto load_b = [&](int o0) {
        const uint16_t* row = B + int64_t(min(o0, (last - 1) & ~31)) * s.R;
#pragma unroll
        for (int k = 0; k < 2 * NR; ++k) w[k] = *reinterpret_cast<const uint4*>(row + 32 * min(16 * k, s.R - 16));
    };
    auto load_base = [&](int o0) {
        const float* p = base + max(min(o0, whole - 32), first);
#pragma unroll
        for (int q = 0; q < 4; ++q) was[q] = __builtin_nontemporal_load(reinterpret_cast<const f4*>(p + rb[q]));
    };
    auto outputs = [&](f16v& acc) {
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[i] = 0.0f;
#pragma unroll
        for (int k = 0; k < 2 * NR; ++k) {
            Terms<TYPE> h;
#pragma unroll
            for (int c = 0; c < Terms<TYPE>::N; ++c) h.t[c] = l.h[k][c][lane];
            acc = product<TYPE>(w[k], h, acc);
        }
    };
    float unit = 1.0f;
    auto turn = [&](f16v acc) {  // into swap, in units of 1
        if constexpr (TYPE == WV_ADAPTER_F16) acc *= unit;
#pragma unroll
        for (int q = 0; q < 4; ++q)
            *reinterpret_cast<g4*>(swap + n * kSwap + 8 * q + 4 * hi) = g4{acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]};
        wave_sync();
    };
    int o0 = first + 32 * wave;
    if (whole > first) load_base(o0);
    load_b(o0);
    stage_operands<TYPE, NR>(a, s, t, rank, s.known[id].scale, l);
    if constexpr (TYPE == WV_ADAPTER_F16) unit = power(exponent(l.most[n]) - 14);
    // what was loaded so far is there (h came after it): the steps' waits need not allow for it
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
    for (; o0 < whole; o0 += 128) {
        f16v acc;
        outputs(acc);
        __builtin_amdgcn_sched_barrier(0);
        load_b(o0 + 128);
        __builtin_amdgcn_sched_barrier(0);
        turn(acc);
        f4 sum[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) sum[q] = was[q] + f4(*reinterpret_cast<const g4*>(swap + rs[q]));
        wave_sync();
        load_base(o0 + 128);
#pragma unroll
        for (int q = 0; q < 4; ++q) __builtin_nontemporal_store(sum[q], reinterpret_cast<f4*>(y + o0 + ry[q]));
        __builtin_amdgcn_sched_barrier(0);
    }
    if (o0 >= last || o0 != whole) return;
    f16v acc;  // fewer than 32 outputs are left
    outputs(acc);
    turn(acc);
    for (int i = lane; i < 32 * t.n; i += 64)
        if (const int r = i >> 5, o = o0 + (i & 31); o < last) {
            const int64_t at = t.from_first(r);
            y[at * s.ys + o] = base[at * s.bs + o] + swap[r * kSwap + (i & 31)];
        }
}

// Rows without an adapter: a wave a row, eight of them on their way.
__device__ __forceinline__ void copy_rows(const SetArgs& s, const Tile& t, int first, int last, const float* base, float* y) {
    const int wave = threadIdx.x >> 6;
    for (int o = first + 4 * int(threadIdx.x & 63); o < last; o += 256) {
        if (o + 4 > last) {
            for (int n = wave; n < t.n; n += 4)
                for (int i = o; i < last; ++i) y[t.from_first(n) * s.ys + i] = base[t.from_first(n) * s.bs + i];
            continue;
        }
        f4 x[kTile / 4];
#pragma unroll
        for (int i = 0; i < kTile / 4; ++i)
            if (const int n = wave + 4 * i; n < t.n) x[i] = *reinterpret_cast<const f4*>(base + t.from_first(n) * s.bs + o);
#pragma unroll
        for (int i = 0; i < kTile / 4; ++i)
            if (const int n = wave + 4 * i; n < t.n) *reinterpret_cast<f4*>(y + t.from_first(n) * s.ys + o) = x[i];
    }
}

struct Nothing {};
template <int TYPE, int NR, int FEW>
__global__ void __launch_bounds__(256) k_adapt_up(Args a, int tile0, int turns) {
    __shared__ __align__(16) float h[(FEW > 0 ? FEW : kFew) * (32 * NR + 4)];
    __shared__ std::conditional_t<(FEW > 0), Nothing, UpLds<TYPE, NR>> lds;
    int set = 0;
    while (set + 1 < kMaxSets && int(blockIdx.x) >= a.set[set + 1].block0) ++set;
    const SetArgs& s = a.set[set];
    const int first = (int(blockIdx.x) - s.block0) * 256 * turns;
    Tile t;
    if (!(FEW == kGrouped ? find_group(a, tile0 + int(blockIdx.y), t) : find_tile<(FEW > 0)>(a, tile0 + int(blockIdx.y), t))) return;
    const int id = t.id;
    const int last = min(first + 256 * turns, s.rows);
    const float* base = s.base + t.t0 * s.bs;
    float* y = s.y + t.t0 * s.ys;
    const bool known = unsigned(id) < unsigned(s.n_adapters);
    if constexpr (FEW != kGrouped) {
        if (known && (FEW > 0 || t.n <= kFew)) {
            up_few<TYPE, NR, (FEW > 0 ? FEW : kFew)>(a, s, t, id, first, last, base, y, h);
            return;
        }
    }
    if constexpr (FEW <= 0) {
        if (const int rank = known ? s.known[id].rank : 0; rank) {
            up_tile<TYPE, NR>(a, s, t, id, rank, first, last, base, y, lds);
            return;
        }
    }
    if (base == y) return;
    if constexpr (FEW > 0) {
        for (int n = 0; n < t.n; ++n)
            for (int o = first + int(threadIdx.x); o < last; o += 256) y[n * s.ys + o] = base[n * s.bs + o];
    } else {
        copy_rows(s, t, first, last, base, y);
    }
}

int most_ids(const Set* s, int n_sets) {
    int n = 0;
    for (int i = 0; i < n_sets; ++i) n = std::max(n, s[i].c.n_adapters);
    return n;
}
// How a call's rows are taken. Short sequences' by adapter where that saves more of A's and B's traffic than finding
// them costs, some 4 us a call: the more, the more sequences there are (by sequence / by adapter, 8 adapters, rank 64 on
// 4096 x 4096: 64 sequences 9.7 / 11.9 us, 128 13.1 / 12.7, 256 21.5 / 16.7, 600 45 / 29; rank 16: 256 12.6 / 12.4; rank
// 128 on 4096 x 14336: 64 28 / 26, 256 74 / 36), and not where an adapter has fewer than four (256 sequences: 32 adapters
// 25 / 24, 64 32 / 36, three sets 63 / 50; of 128, two sets of rank 128, as many adapters 106 / 158). How many adapters
// are in use the host does not see: it goes by how many the sets have room for.
int adapt_mode(const Set* s, int n_sets, const wv_adapter_batch& b) {
    const int most = b.max_q ? b.max_q : b.n_tokens, ids = most_ids(s, n_sets);
    if (most > kFew) return kTiles;
    double bytes = 0.0;
    for (int i = 0; i < n_sets; ++i) bytes += 2.0 * s[i].R * (double(s[i].C) + s[i].O);
    const double n = std::min(b.n_seqs, b.n_tokens);
    if (ids <= kGroupIds && b.n_seqs <= kGroupSeqs && b.n_tokens >= 4 * ids && n * n * bytes >= 15e9) return kGrouped;
    return most <= 1 ? 1 : kFew;
}
int64_t adapt_tiles(const wv_adapter_batch& b, int mode, int ids) {  // at most
    if (mode > 0) return b.n_seqs;
    return (mode == kGrouped ? std::min(b.n_seqs, ids + 1) : b.n_seqs) + b.n_tokens / kTile;
}

// Into how many ranges the columns are cut: about eight blocks a CU (two: 11.5 us for 64 rows of three sets of rank 32,
// four or more 11.0), and ranges of whole chunks (of 128 columns, 32 ranges: 8 rows over 4096 columns 9.5 us, else 8.7).
int adapt_ranges(const Set* s, int n_sets, const wv_adapter_batch& b, int& range) {
    const int chunks = (s[0].c.cols + kChunk - 1) / kChunk, mode = adapt_mode(s, n_sets, b);
    const int64_t blocks = mode > 0 ? int64_t(std::min(b.n_seqs, b.n_tokens)) * n_sets : adapt_tiles(b, mode, most_ids(s, n_sets));
    const int want = int(std::max<int64_t>(1, std::min<int64_t>({2048 / std::max<int64_t>(blocks, 1), chunks, kMaxRanges})));
    const int each = (chunks + want - 1) / want;
    range = each * kChunk;
    return (chunks + each - 1) / each;
}

template <int TYPE>
int launch_adapters(Args& a, int mode, int64_t tiles, hipStream_t s) {
    int64_t units = 0, blocks = 0;
    int R = 0;
    for (int i = 0; i < a.n_sets; ++i) units += (a.set[i].rows + 255) / 256, R = std::max(R, a.set[i].R);
    // Outputs of a block: 256, or twice that where there are blocks enough (1 / 2 / 4 turns: 12 sequences of 350 tokens,
    // 14336 outputs of rank 64, 158 / 143 / 148 us; 2 of 100 15.8 / 16.7 / 22.2).
    const int turns = units * tiles >= 1 << 11 ? 2 : 1;
    for (int i = 0; i < kMaxSets; ++i) {
        a.set[i].block0 = i < a.n_sets ? int(blocks) : INT32_MAX;
        if (i < a.n_sets) blocks += (a.set[i].rows + 256 * turns - 1) / (256 * turns);
    }
    auto go = [&](auto kern, int64_t x, int z, auto... more) {
        for (int64_t t0 = 0; t0 < tiles; t0 += 1 << 15) {
            const dim3 grid{unsigned(x), unsigned(std::min<int64_t>(tiles - t0, 1 << 15)), unsigned(z)};
            hipLaunchKernelGGL(kern, grid, dim3(256), 0, s, a, int(t0), more...);
        }
    };
    auto up = [&](auto nr) {
        constexpr int NR = decltype(nr)::value;
        mode == 1          ? go(k_adapt_up<TYPE, NR, 1>, blocks, 1, turns)
        : mode == kFew     ? go(k_adapt_up<TYPE, NR, kFew>, blocks, 1, turns)
        : mode == kGrouped ? go(k_adapt_up<TYPE, NR, kGrouped>, blocks, 1, turns)
                           : go(k_adapt_up<TYPE, NR, kTiles>, blocks, 1, turns);
    };
    std::integral_constant<int, 1> n1;
    std::integral_constant<int, 2> n2;
    std::integral_constant<int, 4> n4;
    std::integral_constant<int, 8> n8;
    if (mode > 0) {
        go(mode == 1 ? k_adapt_down<TYPE, 1, 1> : k_adapt_down<TYPE, 1, kFew>, int64_t(a.ranges) * a.n_sets, 1);
    } else {
        // Ranks of a block, 32 nr: all of them, as the terms of x are split once for them, unless a block a CU takes them
        // in parts (all / in parts: 3 sets of rank 32 over 4096 columns, 8 sequences of 8 tokens, 14.3 / 9.9 us with the
        // launch for B; 2 sets of rank 128, one of 10, 18.4 / 12.6; but 16 of 30 tokens, 384 blocks, 18.7 / 18.8, 64 of 8,
        // 1536 blocks, 23.3 / 25.0).
        auto parts = [&](int nr) { return (a.ranks + 32 * nr - 1) / (32 * nr); };
        auto fits = [&](int nr) { return parts(nr) == 1 || a.ranges * tiles * parts(nr) <= 256; };
        auto down = [&](auto nr) {
            constexpr int NR = decltype(nr)::value;
            go(mode == kGrouped ? k_adapt_down<TYPE, NR, kGrouped> : k_adapt_down<TYPE, NR, kTiles>, a.ranges, parts(NR));
        };
        fits(1) ? down(n1) : fits(2) ? down(n2) : down(n4);  // more than 128 would take all of a SIMD's registers for one wave
    }
    R <= 32 ? up(n1) : R <= 64 ? up(n2) : R <= 128 ? up(n4) : up(n8);
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
    s.O = (c.rows + 31) / 32 * 32;
    const size_t n = size_t(c.n_adapters), na = n * s.R * s.C * 2, nb = n * s.O * s.R * 2;
    // one allocation: A, B (both multiples of 16 bytes), ranks and scales
    uint8_t* p = nullptr;
    hipError_t e = hipMalloc(reinterpret_cast<void**>(&p), na + nb + n * sizeof(Known));
    if (e != hipSuccess) {
        (void)hipGetLastError();
        return rt_hip_fail(e, "wv_adapters_create: weights");
    }
    s.a = reinterpret_cast<uint16_t*>(p);
    s.b = reinterpret_cast<uint16_t*>(p + na);
    s.known = reinterpret_cast<Known*>(p + na + nb);
    hipStream_t st = rt_stream(nullptr, s.device);
    e = hipMemsetAsync(s.known, 0, n * sizeof(Known), st);
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
    const size_t R = size_t(s.R), C = size_t(s.C), O = size_t(s.O), rows = size_t(s.c.rows), cols = size_t(s.c.cols);
    const size_t r = size_t(rank);
    std::vector<uint16_t> ha(rank ? R * C : 0), hb(rank ? O * R : 0);
    for (size_t i = 0; i < r; ++i) std::memcpy(&ha[i * C], a + i * cols, cols * 2);
    for (size_t o = 0; o < rows; ++o)
        for (size_t i = 0; i < r; i += 8)
            std::memcpy(&hb[o / 32 * 32 * R + i / 8 * 256 + o % 32 * 8], b + o * r + i, std::min<size_t>(8, r - i) * 2);
    (void)hipSetDevice(s.device);
    hipError_t e = hipDeviceSynchronize();  // calls that still read the adapter
    if (e == hipSuccess && r) e = hipMemcpy(s.a + size_t(index) * R * C, ha.data(), ha.size() * 2, hipMemcpyHostToDevice);
    if (e == hipSuccess && r) e = hipMemcpy(s.b + size_t(index) * O * R, hb.data(), hb.size() * 2, hipMemcpyHostToDevice);
    const Known k{rank, scale};
    if (e == hipSuccess) e = hipMemcpy(s.known + index, &k, sizeof k, hipMemcpyHostToDevice);
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
    *bytes = scratch_floats(s, n_sets, batch->n_tokens, adapt_ranges(s, n_sets, *batch, range)) * 4;
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
        k.a = s[i].a, k.b = s[i].b, k.known = s[i].known;
        k.rows = s[i].c.rows, k.R = s[i].R, k.C = s[i].C, k.O = s[i].O, k.n_adapters = s[i].c.n_adapters;
    }
    if (!a.n_seqs || !a.n_tokens) return WV_OK;
    if (!d_x || !batch->d_cu_q || !batch->d_adapter) return rt_fail(WV_E_ARG, "wv_adapters: nil x/cu_q/adapter");
    for (int i = 0; i < n_sets; ++i)
        if (!a.set[i].y) return rt_fail(WV_E_ARG, "wv_adapters: nil y");
    for (int i = 0; i < n_sets; ++i) {  // blocks of one set would write what others' read or write
        if (a.set[i].y == d_x) return rt_fail(WV_E_ARG, "wv_adapters: the rows of set %d are x", i);
        for (int j = 0; j < n_sets; ++j)
            if (i != j && (a.set[i].y == a.set[j].y || a.set[i].y == a.set[j].base))
                return rt_fail(WV_E_ARG, "wv_adapters: the rows of set %d are those of set %d", i, j);
    }
    a.n_sets = n_sets;
    for (int i = 0; i < n_sets; ++i) a.ranks += s[i].R;
    a.x = d_x, a.xs = x_stride, a.cu = batch->d_cu_q, a.which = batch->d_adapter;
    a.ids = most_ids(s, n_sets);
    a.ranges = adapt_ranges(s, n_sets, *batch, a.range);
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
    const int mode = adapt_mode(s, n_sets, *batch);
    const int64_t tiles = adapt_tiles(*batch, mode, a.ids);
    const int e = s[0].c.type == WV_ADAPTER_BF16 ? launch_adapters<WV_ADAPTER_BF16>(a, mode, tiles, st)
                                                 : launch_adapters<WV_ADAPTER_F16>(a, mode, tiles, st);
    return e == hipSuccess ? WV_OK : rt_hip_fail(hipError_t(e), "wv_adapters: kernel launch");
}

}  // extern "C"
