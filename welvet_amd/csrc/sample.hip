// sample.hip — the draw of each row's next token from its logits.
//
// w_i = 2^(a_i), a_i = (l_i - max) log2(e) / T, held as integers in units of
// 2^-44 wherever they are summed: the sums are exact, so nothing depends on
// the order in which threads add. Tokens are ordered by falling logit, equal
// ones by index; a cut (l*, i*) keeps the tokens in front of it and itself.
//
// A row needs its logits once from memory: 33 MB of 64 rows of 128000 take
// 6.3 us at a large copy's rate. What binds is the passes over them: the
// maximum; a histogram of the weights (their logarithms in bins, counts for
// top-k); a pass that collects the cut's bin and sums what is kept in front of
// it by segments of 1024 tokens, each some 20 instructions a logit; and the
// steps between them, which one block after the other waits for. Rows of up to
// 32768 logits stay in LDS meanwhile (256 rows of 32000: greedy 8.9 us, top-k
// of 40 15, top-p 29, top-k of 400 and top-p 37, no filter 20), those of up to
// 4096 and 8192 dealt out so that all waves have some (10 of 1530, top-k of 400
// and top-p: 21 to 13 us). Of larger ones, where rows are few, each is cut over
// several blocks, below (64 of 128000: top-p 46 us, by whole rows 92).
// The loops stay small: with the row in registers, unrolled, instruction fetch
// took most of the time (greedy, one row of 32000: 23 us, from LDS 5).
#include <algorithm>
#include <cmath>

#include "rt_internal.h"
#include "sample.h"
#include "wave_ops.h"

namespace wv {
namespace {

typedef unsigned long long u64;

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kBins = 2048;         // of falling a, kPerUnit to a factor of two; the last holds the rest
constexpr float kPerUnit = 64.0f;
constexpr int kList = 512;          // tokens ranked one per thread
constexpr int kFewK = 128;          // top-k up to which the candidates alone are looked at
constexpr int kPass = 4 * kThreads; // tokens of a pass of the block, four to a thread
constexpr int kSegment = 1024;      // tokens that a wave goes through in four passes, in order of index
constexpr int kTurn = 4 * kPass;    // tokens of four passes
constexpr int kMaxVocab = 1 << 19;  // 2^19 weights of at most 2^44 stay below 2^63
constexpr int kSegments = kMaxVocab / kSegment;
constexpr int kResident = 32768;    // logits of a row that stay in LDS
// Where a row lies: in memory, read in every pass; or in LDS, of so many passes
// at most that a turn takes them all, or of up to kResident logits.
enum { kStream, kLong, kTwo, kOne };
constexpr int row_floats(int R) { return R == kLong ? kResident : R == kTwo ? 2 * kPass : R == kOne ? kPass : 4; }

// Order-preserving integer of a float (NaN does not occur).
__device__ __forceinline__ uint32_t order_key(float x) {
    const uint32_t b = __float_as_uint(x == 0.0f ? 0.0f : x);  // -0 and 0 are equal
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
// Tokens as integers whose falling order is the tokens' order.
__device__ __forceinline__ u64 token_key(float l, int i) { return u64(order_key(l)) << 32 | uint32_t(~i); }
__device__ __forceinline__ float key_logit(u64 key) {
    const uint32_t o = uint32_t(key >> 32);
    return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}

// The row's scale: log2(e) / T in two floats, and the difference to the
// maximum from which on weights are 0.
struct Scale {
    float max, hi, lo, least;
};
// log2 weight of logit l, monotone in l; the maximum itself (infinite or not) has 0.
__device__ __forceinline__ float log_weight(const Scale& c, float l) {
    const float t = fmaxf(fminf(l - c.max, 0.0f), c.least);  // inf - inf: min(NaN, 0) = 0
    return fmaf(t, c.hi, t * c.lo);
}
__device__ __forceinline__ float weight(const Scale& c, float l) { return __builtin_amdgcn_exp2f(log_weight(c, l)); }
__device__ __forceinline__ int bin_of(float a) { return int(fminf(-a * kPerUnit, float(kBins - 1))); }
// A weight in units of 2^-44: adding 256 leaves them in a double's last bits.
__device__ __forceinline__ u64 fixed(float w) {
    return u64(__double_as_longlong(256.0 + double(w)) - __double_as_longlong(256.0));
}

template <int Ctrl, int RowMask, int BankMask>
__device__ __forceinline__ u64 dpp_u64(u64 v) {
    const uint32_t lo = uint32_t(dpp_i<Ctrl, RowMask, BankMask>(0, int(uint32_t(v))));
    const uint32_t hi = uint32_t(dpp_i<Ctrl, RowMask, BankMask>(0, int(uint32_t(v >> 32))));
    return u64(hi) << 32 | lo;
}
// Inclusive sums over the lanes.
__device__ __forceinline__ u64 wave_scan(u64 v) {
    v += dpp_u64<kDppRowShr1, 0xf, 0xf>(v);
    v += dpp_u64<kDppRowShr2, 0xf, 0xf>(v);
    v += dpp_u64<kDppRowShr4, 0xf, 0xe>(v);
    v += dpp_u64<kDppRowShr8, 0xf, 0xc>(v);
    v += dpp_u64<kDppRowBcast15, 0xa, 0xf>(v);
    v += dpp_u64<kDppRowBcast31, 0xc, 0xf>(v);
    return v;
}

__device__ __forceinline__ u64 last_lane(u64 v) {
    const uint32_t lo = uint32_t(__builtin_amdgcn_readlane(int(uint32_t(v)), 63));
    return u64(uint32_t(__builtin_amdgcn_readlane(int(uint32_t(v >> 32)), 63))) << 32 | lo;
}

template <int R>
struct Shared {
    float row[row_floats(R)];
    u64 hist[kBins];
    alignas(16) u64 list[kList];
    alignas(16) u64 weights[kList];
    u64 seg[R != kStream ? kResident / kSegment : kSegments];
    u64 part[kWaves];
    u64 key;   // a result of one thread for all
    u64 sum;
    int at, n;
};

// One row, read from memory once where it fits LDS, else in every pass.
// each4(f): f(four logits, index of the first, pass) for this thread's ones;
// in a turn (four passes; for short rows two or one) a wave meets a segment,
// 1024 (512, 256) consecutive tokens in order, 256 a pass. NaN and what lies behind the row are -inf, which no step counts.
template <int R>
struct Row {
    const float* p;
    float* lds;
    int vocab;

    __device__ __forceinline__ float4 fetch(int i) const {
        float4 x = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        if (i + 3 < vocab) {  // one load at any multiple of 4 bytes
            typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));
            const f4 y = *reinterpret_cast<const f4*>(p + i);
            x = make_float4(y.x, y.y, y.z, y.w);
        } else {
            if (i < vocab) x.x = p[i];
            if (i + 1 < vocab) x.y = p[i + 1];
            if (i + 2 < vocab) x.z = p[i + 2];
            if (i + 3 < vocab) x.w = p[i + 3];
        }
        return x;
    }
    __device__ __forceinline__ static float4 clean(float4 x) {
        x.x = fmaxf(x.x, -INFINITY);  // NaN: the other operand
        x.y = fmaxf(x.y, -INFINITY);
        x.z = fmaxf(x.z, -INFINITY);
        x.w = fmaxf(x.w, -INFINITY);
        return x;
    }
    // log2 of a turn's passes; a segment is 256 tokens times them. Short rows spread over all waves.
    static constexpr __device__ int lg() { return R == kOne ? 0 : R == kTwo ? 1 : 2; }
    static constexpr __device__ int segment() { return 256 << lg(); }
    __device__ __forceinline__ int segments() const { return (vocab + segment() - 1) >> (8 + lg()); }
    __device__ __forceinline__ bool ends_segment(int k) const { return (k & ((1 << lg()) - 1)) == (1 << lg()) - 1; }
    // Whole turns.
    __device__ __forceinline__ int passes() const { return (vocab + (kPass << lg()) - 1) / (kPass << lg()) << lg(); }
    // Where the wave's segment of pass k begins.
    __device__ __forceinline__ int begin(int k) const {
        return (k >> lg()) * (kPass << lg()) + __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6)) * segment();
    }
    __device__ __forceinline__ int index(int k) const {
        return begin(k) + (k & ((1 << lg()) - 1)) * 256 + 4 * int(threadIdx.x & 63);
    }
    // Passes k0 .. k1 - 1 from memory, four passes' loads on their way.
    template <class F>
    __device__ __forceinline__ void range(int k0, int k1, F f) const {
        float4 x[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = k0 + k < k1 ? fetch(index(k0 + k)) : float4{};
        for (int k = k0; k < k1; ++k) {
            const float4 y = x[0];
            x[0] = x[1], x[1] = x[2], x[2] = x[3];
            if (k + 4 < k1) x[3] = fetch(index(k + 4));
            f(clean(y), index(k), k);
        }
    }
    template <class F>
    __device__ __forceinline__ void stream(F f) const {
        range(0, passes(), f);
    }
    // The first pass over the row, which fills LDS.
    template <class F>
    __device__ __forceinline__ void first(F f) const {
        if constexpr (R != kStream) {
            float4 x[row_floats(R) / kPass];
#pragma unroll
            for (int k = 0; k < row_floats(R) / kPass; ++k) x[k] = fetch(index(k));
#pragma unroll
            for (int k = 0; k < row_floats(R) / kPass; ++k) {
                x[k] = clean(x[k]);
                *reinterpret_cast<float4*>(lds + index(k)) = x[k];
                f(x[k], index(k), k);
            }
        } else {
            stream(f);
        }
    }
    template <class F>
    __device__ __forceinline__ void each4(F f) const {
        if constexpr (R != kStream) {
            // as far as the wave has segments of the row
            const int n = (vocab - begin(0) + (kPass << lg()) - 1) / (kPass << lg()) << lg();
            for (int k = 0; k < n; ++k) f(*reinterpret_cast<const float4*>(lds + index(k)), index(k), k);
        } else {
            stream(f);
        }
    }
    template <class F>
    __device__ __forceinline__ void each(F f) const {
        each4([&](float4 x, int i, int) {
            f(x.x, i);
            f(x.y, i + 1);
            f(x.z, i + 2);
            f(x.w, i + 3);
        });
    }
    // Four logits from index i (a multiple of 4) on.
    __device__ __forceinline__ float4 at(int i) const {
        if constexpr (R != kStream) return *reinterpret_cast<const float4*>(lds + i);
        return clean(fetch(i));
    }
};

template <int R>
__device__ __forceinline__ void clear_hist(Shared<R>& s) {
#pragma unroll
    for (int i = 0; i < kBins / kThreads; ++i) s.hist[threadIdx.x + i * kThreads] = 0;
    if (threadIdx.x == 0) s.n = 0;
    __syncthreads();
}

// v[0 .. n) (n at most 2 * 1024) added up in order: the index where the sum
// reaches `target` (> 0) into s.at, the sum in front of it into s.sum, and the
// whole sum returned. s.at is -1 where the whole is less.
template <int R>
__device__ __forceinline__ u64 find_in(Shared<R>& s, const u64* v, int n, u64 target) {
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    if (t == 0) s.at = -1;
    const u64 x = 2 * t < n ? v[2 * t] : 0, y = 2 * t + 1 < n ? v[2 * t + 1] : 0;
    const u64 incl = wave_scan(x + y);
    if (lane == 63) s.part[wave] = incl;
    __syncthreads();
    u64 before = 0, whole = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        const u64 p = s.part[w];
        if (w < wave) before += p;
        whole += p;
    }
    before += incl - (x + y);
    if (before < target && before + x + y >= target) {
        const bool first = before + x >= target;
        s.at = 2 * t + !first;
        s.sum = first ? before : before + x;
    }
    __syncthreads();
    return whole;
}

// Where tokens of one logit l share the cut: the `nth` (from 1) of them by index.
template <int R>
__device__ __forceinline__ u64 nth_equal(Shared<R>& s, const Row<R>& row, float l, u64 nth) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int segs = row.segments();
    int c = 0;
    row.each4([&](float4 x, int, int k) {
        c += (x.x == l) + (x.y == l) + (x.z == l) + (x.w == l);
        if (row.ends_segment(k)) {
            const int n = wave_total_i(c), sg = (k >> row.lg()) * kWaves + wave;
            if (lane == 0 && sg < segs) s.seg[sg] = u64(n);
            c = 0;
        }
    });
    __syncthreads();
    find_in(s, s.seg, segs, nth);
    const int sg = s.at;
    const u64 want = nth - s.sum;
    if (wave == 0) {
        u64 before = 0;
        for (int q = 0; q < 1 << row.lg(); ++q) {
            const int i = sg * row.segment() + q * 256 + 4 * lane;
            const float4 x = row.at(i);
            const float v[4] = {x.x, x.y, x.z, x.w};
            u64 n = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) n += v[j] == l;
            const u64 incl = before + wave_scan(n);
            u64 at = incl - n;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (v[j] == l && ++at == want) s.key = token_key(l, i + j);
            before = last_lane(incl);
        }
    }
    __syncthreads();
    return s.key;
}

// Ranks the n tokens of the list, one per thread: how many of them, and how
// much weight, come before this thread's in the tokens' order. LDS reads bind:
// some 20 us for 400 tokens, so that whole rows cut such a top-k by bins instead.
template <int R>
__device__ __forceinline__ void rank_list(const Shared<R>& s, int n, u64 key, int& rank, u64& mass) {
    rank = 0;
    mass = 0;
    const ulonglong2* keys = reinterpret_cast<const ulonglong2*>(s.list);
    const ulonglong2* weights = reinterpret_cast<const ulonglong2*>(s.weights);
#pragma unroll 4
    for (int j = 0; j < n / 2; ++j) {
        const ulonglong2 k = keys[j], w = weights[j];
        rank += (k.x > key) + (k.y > key);
        mass += (k.x > key ? w.x : 0) + (k.y > key ? w.y : 0);
    }
    if (n & 1) {
        const bool b = s.list[n - 1] > key;
        rank += b;
        mass += b ? s.weights[n - 1] : 0;
    }
}

// The cut that keeps, of the tokens down to `floor` (0: all), the first
// `target` (by_mass: the shortest prefix whose weights reach target); floor
// where there are not as many. s.hist holds their counts (weights) by bin.
template <int R>
__device__ __forceinline__ u64 find_cut(Shared<R>& s, const Row<R>& row, const Scale& c, u64 floor, u64 target,
                                     bool by_mass) {
    find_in(s, s.hist, kBins, target);
    const int bin = s.at;
    if (bin < 0) return floor;
    const u64 left = target - s.sum;  // of this bin
    __syncthreads();
    clear_hist(s);
    row.each([&](float l, int i) {
        const float a = log_weight(c, l);
        if (bin_of(a) == bin && l > -INFINITY && token_key(l, i) >= floor) {
            const int at = atomicAdd(&s.n, 1);
            if (at < kList) {
                s.list[at] = token_key(l, i);
                s.weights[at] = fixed(__builtin_amdgcn_exp2f(a));
            }
        }
    });
    __syncthreads();
    const int n = s.n;
    if (n <= kList) {
        if (int(threadIdx.x) < n) {
            const u64 key = s.list[threadIdx.x];
            int rank;
            u64 mass;
            rank_list(s, n, key, rank, mass);
            const bool cut = by_mass ? mass < left && mass + s.weights[threadIdx.x] >= left : u64(rank) + 1 == left;
            if (cut) s.key = key;
        }
        __syncthreads();
        return s.key;
    }
    // many tokens in one bin: their logits' bits from the top, 11, 11 and 10
    u64 rest = left;
    uint32_t prefix = 0, mask = 0;
    for (int shift = 21; shift >= 0; shift = shift > 10 ? 10 : shift > 0 ? 0 : -1) {
        const int bits = shift == 0 ? 10 : 11;
        clear_hist(s);
        row.each([&](float l, int i) {
            const uint32_t k = ~order_key(l);  // falls with the logit
            const float a = log_weight(c, l);
            if (bin_of(a) == bin && l > -INFINITY && token_key(l, i) >= floor && (k & mask) == prefix)
                atomicAdd(&s.hist[(k >> shift) & ((1u << bits) - 1)], by_mass ? fixed(__builtin_amdgcn_exp2f(a)) : u64(1));
        });
        __syncthreads();
        find_in(s, s.hist, kBins, rest);
        rest -= s.sum;
        prefix |= uint32_t(s.at) << shift;
        mask |= ((1u << bits) - 1) << shift;
        __syncthreads();
    }
    const float l = key_logit(u64(~prefix) << 32);
    u64 nth = rest;
    if (by_mass) {
        const u64 w = fixed(weight(c, l));
        nth = (rest + w - 1) / w;
    }
    return nth_equal(s, row, l, nth);
}

__device__ __forceinline__ void put(const SampleArgs& a, int row, int token, float prob) {
    if (a.tokens) a.tokens[row] = token;
    if (a.probs) a.probs[row] = prob;
    if (a.state) {
        a.state[2] = token;
        a.state[1] = token;
        const int k = a.state[3];
        if (k < a.gen_cap) a.gen[k] = token;
        a.state[3] = k + 1;
        if (a.advance) a.state[0] += 1;
    }
}

// A row's settings, cleaned.
struct Settings {
    float temp, top_p, min_p, u;
    int top_k;
    bool greedy, by_k, by_p;
};
__device__ __forceinline__ Settings settings(const SampleArgs& a, int r) {
    Settings x;
    x.temp = a.p.temperature ? a.p.temperature[r] : 1.0f;
    x.top_k = a.p.top_k ? a.p.top_k[r] : 0;
    x.top_p = a.p.top_p ? a.p.top_p[r] : 1.0f;
    const float m = a.p.min_p ? a.p.min_p[r] : 0.0f;
    x.min_p = m > 0.0f ? fminf(m, 1.0f) : 0.0f;
    const float u = a.p.uniform[a.state ? a.state[3] : r];
    x.u = u >= 0.0f ? fminf(u, 0.99999994f) : 0.0f;
    x.greedy = !(x.temp > 0.0f) || x.top_k == 1 || x.top_p <= 0.0f;
    x.by_k = x.top_k > 0 && x.top_k < a.vocab;
    x.by_p = x.top_p < 1.0f;
    return x;
}
__device__ __forceinline__ Scale scale_of(float max, float temp) {
    Scale c;
    c.max = max;
    // an infinite maximum takes all, whatever the temperature
    const double cd = max < INFINITY ? fmin(1.4426950408889634 / double(temp), 1e30) : 1.0;
    c.hi = float(cd);
    c.lo = cd < 1e30 ? float(cd - double(c.hi)) : 0.0f;
    c.least = c.hi > 1e-36f ? -200.0f / c.hi : -3.4028235e38f;
    return c;
}

// Which of the tokens in front of a cut (0: all) are kept, and their weights.
struct Kept {
    Scale c;
    float cl, min_p;
    int ci;
    __device__ __forceinline__ Kept(const Scale& c, u64 cut, float min_p)
        : c(c), cl(cut ? key_logit(cut) : -INFINITY), min_p(min_p), ci(cut ? int(~uint32_t(cut)) : -1) {}
    // in units of 1, a multiple of 2^-44
    __device__ __forceinline__ double operator()(float l, int i) const {
        const float w = weight(c, l);
        const bool k = (l > cl || (l == cl && i <= ci)) && w >= min_p;
        return k ? (256.0 + double(w)) - 256.0 : 0.0;
    }
};

// The wave's sum of doubles that are multiples of 2^-44, in units of it: up to
// 1024, so in integers.
__device__ __forceinline__ u64 segment_sum(double v) { return last_lane(wave_scan(u64(v * 17592186044416.0))); }

// The place of u among s.seg, the kept weights of each segment, and in the
// segment where it lies.
template <int R>
__device__ __forceinline__ void pick(const SampleArgs& a, Shared<R>& s, const Row<R>& row, int r, const Kept& kept,
                                     float u) {
    const int segs = row.segments(), lane = threadIdx.x & 63;
    const u64 total = find_in(s, s.seg, segs, ~u64(0));
    const u64 want = u64(double(u) * double(total));
    find_in(s, s.seg, segs, want + 1);
    if (threadIdx.x < 64) {
        u64 at = s.sum;
        float4 x[4];
#pragma unroll
        for (int q = 0; q < 4; ++q)
            if (q < 1 << row.lg()) x[q] = row.at(s.at * row.segment() + q * 256 + 4 * lane);
        for (int q = 0; q < 1 << row.lg(); ++q) {
            const int i = s.at * row.segment() + q * 256 + 4 * lane;
            const float y[4] = {x[0].x, x[0].y, x[0].z, x[0].w};
            x[0] = x[1], x[1] = x[2], x[2] = x[3];
            u64 v[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = u64(kept(y[j], i + j) * 17592186044416.0);
            const u64 sum = (v[0] + v[1]) + (v[2] + v[3]), incl = at + wave_scan(sum);
            u64 before = incl - sum;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (v[j] && before <= want && want < before + v[j])
                    put(a, r, i + j, float(double(v[j]) / double(total)));
                before += v[j];
            }
            at = last_lane(incl);
        }
    }
}

// The draw among the n tokens of the list, which holds the top_k at least.
template <int R>
__device__ __forceinline__ void pick_from_list(const SampleArgs& a, Shared<R>& s, int r, const Settings& x,
                                               const Scale& c, int n) {
    const int t = threadIdx.x;
    u64 key = 0, w = 0, mass = 0;
    int rank = kList;
    if (t < n) {
        key = s.list[t];
        w = s.weights[t];
        rank_list(s, n, key, rank, mass);
    }
    if (t < n && rank == min(x.top_k, n) - 1) s.sum = mass + w;  // what the top k hold
    __syncthreads();
    bool keep = rank < x.top_k;
    if (x.by_p) keep = keep && mass < max(u64(1), u64(ceil(double(x.top_p) * double(s.sum))));
    keep = keep && weight(c, key_logit(key)) >= x.min_p;
    // by index: the kept tokens in front of this one, and all
    if (!keep) w = 0;
    if (t < n) s.weights[t] = w;
    __syncthreads();
    u64 before = 0, total = 0;
    if (t < n) {
        const ulonglong2* keys = reinterpret_cast<const ulonglong2*>(s.list);
        const ulonglong2* weights = reinterpret_cast<const ulonglong2*>(s.weights);
        const uint32_t mine = uint32_t(key);  // ~index: larger is earlier
#pragma unroll 4
        for (int j = 0; j < n / 2; ++j) {
            const ulonglong2 k = keys[j], v = weights[j];
            total += v.x + v.y;
            before += (uint32_t(k.x) > mine ? v.x : 0) + (uint32_t(k.y) > mine ? v.y : 0);
        }
        if (n & 1) {
            const u64 v = s.weights[n - 1];
            total += v;
            if (uint32_t(s.list[n - 1]) > mine) before += v;
        }
    }
    const u64 want = u64(double(x.u) * double(total));
    if (w && before <= want && want < before + w) put(a, r, int(~uint32_t(key)), float(double(w) / double(total)));
}

// What a cut in `bin` (kBins: none) does with the tokens from key `floor` on:
// those of the bin (`few`: down to its end) go into the list, the weights of
// those in front of it, from min_p on, come back for their segment's sum.
template <bool FLOOR, int R>
struct Visit {
    Shared<R>& s;
    const Scale& c;
    u64 floor;
    float min_p, front, lo, hi;  // bin_of() in terms of y = -log_weight kPerUnit
    __device__ __forceinline__ Visit(Shared<R>& s, const Scale& c, u64 floor, float min_p, int bin, bool few)
        : s(s), c(c), floor(floor), min_p(min_p) {
        front = bin < kBins ? float(bin) : INFINITY;
        lo = few ? -1.0f : front;
        hi = bin < kBins - 1 ? float(bin + 1) : bin < kBins || few ? INFINITY : -1.0f;
    }
    __device__ __forceinline__ double operator()(float l, int i) const {
        const float x = log_weight(c, l), y = -x * kPerUnit;
        const float w = __builtin_amdgcn_exp2f(x);
        const bool in = l > -INFINITY && (!FLOOR || token_key(l, i) >= floor);
        if (in && y >= lo && y < hi) {
            const int at = atomicAdd(&s.n, 1);
            if (at < kList) {
                s.list[at] = token_key(l, i);
                s.weights[at] = fixed(w);
            }
            return 0.0;
        }
        return in && y < front && w >= min_p ? (256.0 + double(w)) - 256.0 : 0.0;
    }
    __device__ __forceinline__ double four(float4 x, int i) const {
        return ((*this)(x.x, i) + (*this)(x.y, i + 1)) + ((*this)(x.z, i + 2) + (*this)(x.w, i + 3));
    }
};
// Adds a pass's weights up and leaves the sum of a segment with its last pass.
// A segment's weights of at most 1 are steps of 2^-44 and so are a thread's sums of 16.
template <int R>
struct SegmentSum {
    const Row<R>& row;
    u64* seg;
    double sum = 0.0;
    __device__ __forceinline__ SegmentSum(const Row<R>& row, u64* seg) : row(row), seg(seg) {}
    __device__ __forceinline__ void operator()(double v, int k) {
        sum += v;
        if (!row.ends_segment(k)) return;
        const u64 all = segment_sum(sum);
        const int sg = (k >> row.lg()) * kWaves + int(threadIdx.x >> 6);
        if ((threadIdx.x & 63) == 0 && sg < row.segments()) seg[sg] = all;
        sum = 0.0;
    }
};
// The cut among the n tokens of the bin's list, where `left` is what it keeps
// of them: into s.key; what it keeps, from min_p on, into their segments.
template <int R>
__device__ __forceinline__ void cut_list(Shared<R>& s, const Row<R>& row, const Scale& c, int n, u64 left, bool by_mass, float min_p) {
    const int t = threadIdx.x;
    u64 key = 0, mass = 0, w = 0;
    int rank = 0;
    if (t < n) {
        key = s.list[t], w = s.weights[t];
        rank_list(s, n, key, rank, mass);
        if (by_mass ? mass < left && mass + w >= left : u64(rank) + 1 == left) s.key = key;
    }
    __syncthreads();
    if (t < n && key >= s.key && weight(c, key_logit(key)) >= min_p)
        atomicAdd(&s.seg[int(~uint32_t(key)) >> (8 + row.lg())], w);
    __syncthreads();
}

// A whole row by one block.
template <int R>
__device__ __forceinline__ void sample_row(const SampleArgs& a, Shared<R>& s, int r) {
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const Row<R> row{a.logits + int64_t(r) * a.stride, s.row, a.vocab};
    const Settings set = settings(a, r);
    float top = -INFINITY;  // this thread's largest
    row.first([&](float4 x, int, int) { top = fmaxf(fmaxf(fmaxf(x.x, x.y), fmaxf(x.z, x.w)), top); });
    const float wm = wave_maximum(top);
    if (lane == 0) s.part[wave] = __float_as_uint(wm);
    if (t == 0) s.key = 0;
    __syncthreads();
    Scale c;
    c.max = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) c.max = fmaxf(c.max, __uint_as_float(uint32_t(s.part[w])));
    if (c.max == -INFINITY) {  // every token masked
        if (t == 0) put(a, r, -1, 0.0f);
        return;
    }
    if (set.greedy) {  // the largest logit's first index
        if (top == c.max) {
            u64 best = 0;
            row.each([&](float l, int i) {
                if (l == c.max) best = max(best, token_key(l, i));
            });
            atomicMax(&s.key, best);
        }
        __syncthreads();
        if (t == 0) put(a, r, int(~uint32_t(s.key)), 1.0f);
        return;
    }
    c = scale_of(c.max, set.temp);
    __syncthreads();

    if (set.by_k && set.top_k <= kFewK) {
        // the top_k threads with the largest maxima hold top_k tokens at least as
        // large as the least of these: it bounds the candidates (to its bin)
        clear_hist(s);
        const int bin = bin_of(log_weight(c, top));
        if (top > -INFINITY) atomicAdd(&s.hist[bin], u64(1));
        __syncthreads();
        find_in(s, s.hist, kBins, u64(set.top_k));
        const int last = s.at < 0 ? kBins : s.at;
        __syncthreads();
        if (t == 0) s.sum = ~u64(0);
        __syncthreads();
        if (last < kBins && bin <= last && top > -INFINITY) atomicMin(&s.sum, u64(order_key(top)));
        __syncthreads();
        const float least = last < kBins ? key_logit(s.sum << 32) : -INFINITY;
        row.each([&](float l, int i) {
            if (l >= least && l > -INFINITY) {
                const int at = atomicAdd(&s.n, 1);
                if (at < kList) {
                    s.list[at] = token_key(l, i);
                    s.weights[at] = fixed(weight(c, l));
                }
            }
        });
        __syncthreads();
        const int n = s.n;
        if (n <= kList) return pick_from_list(a, s, r, set, c, n);
        __syncthreads();
    }

    u64 cut = 0;  // the last token kept, 0: all
    bool ready = false, summed = false;
#pragma unroll 1
    for (int mass = 0; mass < 2; ++mass) {  // top-k by counts, then top-p by weights
        if (!(mass ? set.by_p : set.by_k)) continue;
        auto histogram = [&] {
            clear_hist(s);
            row.each([&](float l, int i) {
                const float x = log_weight(c, l);
                if (l > -INFINITY && token_key(l, i) >= cut)
                    atomicAdd(&s.hist[bin_of(x)], mass ? fixed(__builtin_amdgcn_exp2f(x)) : u64(1));
            });
            __syncthreads();
        };
        if (!ready) histogram();
        u64 target = u64(set.top_k);
        if (mass) {
            const u64 whole = find_in(s, s.hist, kBins, ~u64(0));
            target = max(u64(1), min(whole, u64(ceil(double(set.top_p) * double(whole)))));
        }
        if (mass || !set.by_p) {  // the last cut: the segments' sums in the same pass
            find_in(s, s.hist, kBins, target);
            const int bin = s.at < 0 ? kBins : s.at;
            const u64 left = target - s.sum;
            __syncthreads();
            if (t == 0) s.key = cut;
            SegmentSum<R> sums(row, s.seg);
            if (cut) {
                const Visit<true, R> visit(s, c, cut, set.min_p, bin, false);
                row.each4([&](float4 x, int i, int k) { sums(visit.four(x, i), k); });
            } else {
                const Visit<false, R> visit(s, c, cut, set.min_p, bin, false);
                row.each4([&](float4 x, int i, int k) { sums(visit.four(x, i), k); });
            }
            __syncthreads();
            const int n = s.n;
            if (n <= kList) {
                if (n) cut_list(s, row, c, n, left, mass != 0, set.min_p);
                cut = s.key;
                summed = true;
                break;
            }
            __syncthreads();
        } else {  // top-k in front of top-p: the weights' histogram in the pass that collects the cut's bin
            find_in(s, s.hist, kBins, target);
            const int bin = s.at;
            const u64 left = target - s.sum;
            __syncthreads();
            if (bin >= 0) {
                clear_hist(s);
                row.each([&](float l, int i) {
                    const float x = log_weight(c, l);
                    const int at_bin = bin_of(x);
                    if (at_bin > bin || l == -INFINITY) return;
                    const u64 w = fixed(__builtin_amdgcn_exp2f(x));
                    if (at_bin < bin) {
                        atomicAdd(&s.hist[at_bin], w);
                    } else if (const int at = atomicAdd(&s.n, 1); at < kList) {
                        s.list[at] = token_key(l, i);
                        s.weights[at] = w;
                    }
                });
                __syncthreads();
                const int n = s.n;
                if (n <= kList) {
                    if (t < n) {
                        u64 before;
                        int rank;
                        rank_list(s, n, s.list[t], rank, before);
                        if (u64(rank) < left) atomicAdd(&s.hist[bin], s.weights[t]);
                        if (u64(rank) + 1 == left) s.key = s.list[t];
                    }
                    __syncthreads();
                    cut = s.key;
                    ready = true;
                    if (t == 0) s.n = 0;
                    __syncthreads();
                    continue;
                }
                __syncthreads();
                histogram();
            }
        }
        cut = find_cut(s, row, c, cut, target, mass != 0);
        __syncthreads();
    }
    // the kept weights of each segment, then the place of u among them
    const Kept kept(c, cut, set.min_p);
    if (!summed) {
        SegmentSum<R> sums(row, s.seg);
        row.each4([&](float4 x, int i, int k) {
            sums((kept(x.x, i) + kept(x.y, i + 1)) + (kept(x.z, i + 2) + kept(x.w, i + 3)), k);
        });
    }
    __syncthreads();
    pick(a, s, row, r, kept, set.u);
}

template <int R>
__global__ void __launch_bounds__(kThreads) k_sample(SampleArgs a) {
    extern __shared__ __align__(16) uint8_t raw[];
    sample_row(a, *reinterpret_cast<Shared<R>*>(raw), blockIdx.x);
}

// ---------------------------------------------------------------------------
// Rows of many logits, few of them: a row is cut into slices of whole passes,
// one to a block, in four launches that hand on through memory
//   max    the slices' maxima
//   hist   counts (weights) of the slices' tokens by bin, for the first cut
//   collect  the cut's bin from all slices' histograms; its tokens into the
//            row's list, the weights of the bins in front of it by segment
//   finish one block a row: the list's cut, and the place of u
// Rows that do not fit this (top_p with a larger top_k than the list takes, a
// bin of more tokens than that) are done whole by the last launch. 64 rows of
// 128000 with top-p: 5.7, 12.2, 17.4 and 10.1 us; loading a pass's logits in
// front of the wait for the maximum costs registers, and so a block a CU (25
// for 17.7).
// ---------------------------------------------------------------------------

struct alignas(16) SliceRow {
    u64 key;   // greedy: the largest token
    int n;     // tokens of the list; over kList: more than it holds
    u64 left;  // what the cut keeps of its bin: tokens with top-k, weight with top-p
    float max[64];
    u64 list[kList], weights[kList];
    u64 seg[kSegments];
};
struct Slices {
    SliceRow* rows;
    u64* hist;      // [row][kBins]
    int n, passes;  // slices of a row, passes of a slice
};

__device__ __forceinline__ float row_max(const Slices& p, int r) {
    const int lane = threadIdx.x & 63;
    return wave_maximum(lane < p.n ? p.rows[r].max[lane] : -INFINITY);
}
// The list takes all tokens down to the bin of the top-k cut, and the draw is among them.
__device__ __forceinline__ bool few(const Settings& x) { return x.by_k && (x.top_k <= kFewK || (x.by_p && x.top_k <= kList)); }
__device__ __forceinline__ bool sliced(const Settings& x) { return !(x.by_k && x.by_p && x.top_k > kList); }

__global__ void __launch_bounds__(kThreads) k_slice_max(SampleArgs a, Slices p) {
    __shared__ float part[kWaves];
    const int r = blockIdx.y, sl = blockIdx.x;
    const Row<kStream> row{a.logits + int64_t(r) * a.stride, nullptr, a.vocab};
    float top = -INFINITY;
    row.range(sl * p.passes, min((sl + 1) * p.passes, row.passes()),
              [&](float4 x, int, int) { top = fmaxf(fmaxf(fmaxf(x.x, x.y), fmaxf(x.z, x.w)), top); });
    top = wave_maximum(top);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
    __syncthreads();
    for (int i = sl * kThreads + threadIdx.x; i < kBins; i += p.n * kThreads) p.hist[int64_t(r) * kBins + i] = 0;
    if (threadIdx.x == 0) {
        for (int w = 1; w < kWaves; ++w) top = fmaxf(top, part[w]);
        p.rows[r].max[sl] = top;
        if (sl == 0) p.rows[r].key = 0, p.rows[r].n = 0;
    }
}

__global__ void __launch_bounds__(kThreads) k_slice_hist(SampleArgs a, Slices p) {
    __shared__ u64 hist[kBins];
    const int r = blockIdx.y, sl = blockIdx.x;
    const Row<kStream> row{a.logits + int64_t(r) * a.stride, nullptr, a.vocab};
    const int k0 = sl * p.passes, k1 = min((sl + 1) * p.passes, row.passes());
    const Settings set = settings(a, r);
    const float max = row_max(p, r);
    if (max == -INFINITY || set.greedy || !(set.by_k || set.by_p) || !sliced(set)) return;
    const Scale c = scale_of(max, set.temp);
    for (int i = threadIdx.x; i < kBins; i += kThreads) hist[i] = 0;
    __syncthreads();
    auto add = [&](float l) {
        const float x = log_weight(c, l);
        if (l > -INFINITY) atomicAdd(&hist[bin_of(x)], set.by_k ? u64(1) : fixed(__builtin_amdgcn_exp2f(x)));
    };
    row.range(k0, k1, [&](float4 x, int, int) {
        add(x.x);
        add(x.y);
        add(x.z);
        add(x.w);
    });
    __syncthreads();
    // sums of integers: the same in any order
    for (int i = threadIdx.x; i < kBins; i += kThreads)
        if (hist[i]) atomicAdd(&p.hist[int64_t(r) * kBins + i], hist[i]);
}

__global__ void __launch_bounds__(kThreads) k_slice_collect(SampleArgs a, Slices p) {
    extern __shared__ __align__(16) uint8_t raw[];
    Shared<kStream>& s = *reinterpret_cast<Shared<kStream>*>(raw);
    const int r = blockIdx.y, sl = blockIdx.x, t = threadIdx.x;
    SliceRow& g = p.rows[r];
    const Row<kStream> row{a.logits + int64_t(r) * a.stride, nullptr, a.vocab};
    const int k0 = sl * p.passes, k1 = min((sl + 1) * p.passes, row.passes());
    const Settings set = settings(a, r);
    const float max = row_max(p, r);
    if (max == -INFINITY || !sliced(set)) return;
    if (set.greedy) {
        if (g.max[sl] != max) return;
        u64 best = 0;
        row.range(k0, k1, [&](float4 x, int i, int) {
            const float v[4] = {x.x, x.y, x.z, x.w};
            for (int j = 3; j >= 0; --j)
                if (v[j] == max) best = best > token_key(max, i + j) ? best : token_key(max, i + j);
        });
        if (best) atomicMax(&g.key, best);
        return;
    }
    const Scale c = scale_of(max, set.temp);
    int bin = kBins;
    if (set.by_k || set.by_p) {
        static_assert(kBins == 2 * kThreads, "two bins to a thread");
        reinterpret_cast<ulonglong2*>(s.hist)[t] = reinterpret_cast<const ulonglong2*>(p.hist + int64_t(r) * kBins)[t];
        __syncthreads();
        u64 target = u64(set.top_k);
        if (!set.by_k) {
            const u64 whole = find_in(s, s.hist, kBins, ~u64(0));
            target = u64(ceil(double(set.top_p) * double(whole)));
            target = target > whole ? whole : target < 1 ? 1 : target;
        }
        __syncthreads();
        find_in(s, s.hist, kBins, target);
        if (s.at >= 0) bin = s.at;
        if (sl == 0 && t == 0) g.left = bin < kBins ? target - s.sum : 0;
    }
    if (t == 0) s.n = 0;
    __syncthreads();
    const Visit<false, kStream> visit(s, c, 0, set.min_p, bin, few(set));
    SegmentSum<kStream> sums(row, g.seg);
    row.range(k0, k1, [&](float4 x, int i, int k) { sums(visit.four(x, i), k); });
    __syncthreads();
    const int n = s.n;  // this slice's share of the row's list
    if (!n) return;
    if (t == 0) s.at = atomicAdd(&g.n, n);
    __syncthreads();
    if (t < n && s.at + t < kList) g.list[s.at + t] = s.list[t], g.weights[s.at + t] = s.weights[t];
}

__global__ void __launch_bounds__(kThreads) k_slice_finish(SampleArgs a, Slices p) {
    extern __shared__ __align__(16) uint8_t raw[];
    Shared<kStream>& s = *reinterpret_cast<Shared<kStream>*>(raw);
    const int r = blockIdx.x, t = threadIdx.x;
    static_assert(kSegments <= kThreads, "a segment to a thread");
    const SliceRow& g = p.rows[r];
    const Settings set = settings(a, r);
    const float max = row_max(p, r);
    if (max == -INFINITY) {  // every token masked
        if (t == 0) put(a, r, -1, 0.0f);
        return;
    }
    const int n = g.n;
    if (!sliced(set) || (!set.greedy && n > kList)) return sample_row(a, s, r);
    if (set.greedy) {
        if (t == 0) put(a, r, int(~uint32_t(g.key)), 1.0f);
        return;
    }
    const Scale c = scale_of(max, set.temp);
    if (t < n) s.list[t] = g.list[t], s.weights[t] = g.weights[t];
    const int segs = (a.vocab + kSegment - 1) / kSegment;
    if (t < segs) s.seg[t] = g.seg[t];
    const u64 left = g.left;
    if (t == 0) s.key = 0;
    __syncthreads();
    if (few(set)) return pick_from_list(a, s, r, set, c, n);
    const Row<kStream> row{a.logits + int64_t(r) * a.stride, nullptr, a.vocab};
    if (n) cut_list(s, row, c, n, left, !set.by_k, set.min_p);
    pick(a, s, row, r, Kept(c, s.key, set.min_p), set.u);
}

}  // namespace

// Slices of a row: enough that the rows fill the GPU, of a turn at least; 0:
// rows are done whole, where they fit LDS or are many. By slices and whole, 64
// rows of 128000 logits: top-p 46 and 92 us, top-k of 40 39 and 37; 200 rows:
// 90 and 95, 85 and 42.
int sample_slices(int rows, int vocab) {
    if (vocab <= kResident || rows > 128) return 0;
    const int turns = (vocab + kTurn - 1) / kTurn;
    const int want = std::max(1, std::min({64, turns, 512 / rows}));
    const int each = (turns + want - 1) / want;
    return (turns + each - 1) / each;
}
size_t sample_scratch_floats(int rows, int vocab) {
    const size_t n = size_t(sample_slices(rows, vocab));
    return n ? size_t(rows) * (sizeof(SliceRow) + kBins * sizeof(u64)) / sizeof(float) : 0;
}

int launch_sample(const SampleArgs& a, hipStream_t s, float* scratch) {
    const int n = scratch ? sample_slices(a.rows, a.vocab) : 0;
    if (n) {
        const int turns = (a.vocab + kTurn - 1) / kTurn;
        Slices p{reinterpret_cast<SliceRow*>(scratch), nullptr, n, 4 * ((turns + n - 1) / n)};
        p.hist = reinterpret_cast<u64*>(p.rows + a.rows);
        const dim3 grid{unsigned(n), unsigned(a.rows)};
        hipLaunchKernelGGL(k_slice_max, grid, dim3(kThreads), 0, s, a, p);
        hipLaunchKernelGGL(k_slice_hist, grid, dim3(kThreads), 0, s, a, p);
        hipLaunchKernelGGL(k_slice_collect, grid, dim3(kThreads), unsigned(sizeof(Shared<kStream>)), s, a, p);
        hipLaunchKernelGGL(k_slice_finish, dim3(unsigned(a.rows)), dim3(kThreads), unsigned(sizeof(Shared<kStream>)), s,
                           a, p);
        return int(hipGetLastError());
    }
    auto go = [&](auto kern, size_t lds) {
        hipLaunchKernelGGL(kern, dim3(unsigned(a.rows)), dim3(kThreads), unsigned(lds), s, a);
    };
    if (a.vocab <= row_floats(kOne))
        go(k_sample<kOne>, sizeof(Shared<kOne>));
    else if (a.vocab <= row_floats(kTwo))
        go(k_sample<kTwo>, sizeof(Shared<kTwo>));
    else if (a.vocab <= kResident)
        go(k_sample<kLong>, sizeof(Shared<kLong>));
    else
        go(k_sample<kStream>, sizeof(Shared<kStream>));
    return int(hipGetLastError());
}

}  // namespace wv

using namespace wv;

extern "C" int wv_sample_dev(const float* d_logits, int64_t stride, int32_t rows, int32_t vocab,
                             const wv_sampling* sampling, int32_t* d_tokens, float* d_probs, void* stream) {
    if (!sampling) return rt_fail(WV_E_ARG, "wv_sample: nil sampling");
    if (rows < 0 || rows > 1 << 20 || vocab <= 0 || vocab > kMaxVocab)
        return rt_fail(WV_E_SHAPE, "wv_sample: %d rows (at most 2^20) of %d logits (1 to %d)", rows, vocab, kMaxVocab);
    if (!stride) stride = vocab;
    if (stride < vocab)
        return rt_fail(WV_E_SHAPE, "wv_sample: row stride %lld under %d logits", (long long)stride, vocab);
    if (!rows) return WV_OK;
    if (!d_logits || !d_tokens || !sampling->uniform) return rt_fail(WV_E_ARG, "wv_sample: nil logits/tokens/uniform");
    const int rc = rt_ensure_init();
    if (rc) return rc;
    SampleArgs a{};
    a.logits = d_logits, a.stride = stride, a.rows = rows, a.vocab = vocab;
    a.p = *sampling, a.tokens = d_tokens, a.probs = d_probs;
    // no handle says where the rows lie: on the stream's device, whose scratch the call then takes
    int dev = rt_current_device();
    hipStream_t st = rt_stream(stream, dev);
    if (hipDevice_t of; stream && hipStreamGetDevice(st, &of) == hipSuccess) dev = of;
    (void)hipSetDevice(dev);
    RtScratch sc;  // not under capture: what a replay writes must not lie in a slot that other calls take
    const size_t floats = rt_capturing(st) ? 0 : sample_scratch_floats(rows, vocab);
    if (floats)
        if (const int e = sc.get(floats, st, "wv_sample: scratch")) return e;
    const int e = launch_sample(a, st, floats ? sc.f() : nullptr);
    return e == hipSuccess ? WV_OK : rt_hip_fail(hipError_t(e), "wv_sample: kernel launch");
}
