// sample.hip — the draw of each row's next token from its logits.
//
// w_i = 2^(a_i), a_i = (l_i - max) log2(e) / T, held as integers in units of
// 2^-44 wherever they are summed: the sums are exact, so nothing depends on
// the order in which threads add. Tokens are ordered by falling logit, equal
// ones by index; a cut (l*, i*) keeps the tokens in front of it and itself.
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
constexpr int kList = kThreads;     // tokens ranked one per thread
constexpr int kFewK = 128;          // top-k up to which the candidates alone are looked at
constexpr int kSegment = 256;       // tokens of a wave's pass, in order of index
constexpr int kMaxVocab = 1 << 19;  // 2^19 weights of at most 2^44 stay below 2^63
constexpr int kSegments = kMaxVocab / kSegment;

// Order-preserving integer of a float (NaN does not occur).
__device__ __forceinline__ uint32_t order_key(float x) {
    const uint32_t b = __float_as_uint(x == 0.0f ? 0.0f : x);  // -0 and 0 are equal
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
// Tokens as integers whose falling order is the tokens' order.
__device__ __forceinline__ u64 token_key(float l, int i) { return u64(order_key(l)) << 32 | uint32_t(~i); }

// The row's scale: log2(e) / T in two floats.
struct Scale {
    float max, hi, lo;
};
// log2 weight and weight of logit l. a is monotone in l; the product's and
// the scale's rounding, which a drops, come back to first order in w.
__device__ __forceinline__ float log_weight(const Scale& c, float l) {
    return l == c.max ? 0.0f : (l - c.max) * c.hi;
}
__device__ __forceinline__ float weight(const Scale& c, float l) {
    if (l == c.max) return 1.0f;
    const float t = l - c.max, a = t * c.hi;
    const float e = fmaf(t, c.lo, fmaf(t, c.hi, -a));
    const float w = __builtin_amdgcn_exp2f(a);
    return a > -100.0f ? fminf(fmaf(w, e * 0.6931472f, w), 1.0f) : 0.0f;
}
__device__ __forceinline__ int bin_of(float a) { return int(fminf(-a * kPerUnit, float(kBins - 1))); }
// A weight in units of 2^-44: adding 256 leaves them in a double's last bits.
__device__ __forceinline__ u64 fixed(float w) {
    return u64(__double_as_longlong(256.0 + double(w)) - __double_as_longlong(256.0));
}

__device__ __forceinline__ u64 shfl_up64(u64 v, int d) {
    const uint32_t lo = __shfl_up(uint32_t(v), d, 64), hi = __shfl_up(uint32_t(v >> 32), d, 64);
    return u64(hi) << 32 | lo;
}
__device__ __forceinline__ u64 wave_scan(u64 v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const u64 o = shfl_up64(v, d);
        if (lane >= d) v += o;
    }
    return v;
}
__device__ __forceinline__ u64 wave_sum(u64 v) {
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) {
        const uint32_t lo = __shfl_xor(uint32_t(v), d, 64), hi = __shfl_xor(uint32_t(v >> 32), d, 64);
        v += u64(hi) << 32 | lo;
    }
    return v;
}

struct Shared {
    u64 hist[kBins];
    u64 list[kList];
    u64 weights[kList];
    u64 seg[kSegments];
    u64 part[kWaves];
    u64 key;   // a result of one thread for all
    u64 sum;
    int at, n;
};

// One row: its logits in registers (N > 0: at most N * 1024) or read again in
// every pass. f(l, index) of this thread's logits; 256 consecutive ones to a
// wave's pass. NaN counts as -inf.
template <int N>
struct Row {
    const float* p;
    int vocab;
    bool aligned;
    float r[N > 0 ? N : 1];

    __device__ __forceinline__ float4 at(int i) const {
        float4 x = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        if (aligned && i + 3 < vocab) {
            x = *reinterpret_cast<const float4*>(p + i);
        } else {
            if (i < vocab) x.x = p[i];
            if (i + 1 < vocab) x.y = p[i + 1];
            if (i + 2 < vocab) x.z = p[i + 2];
            if (i + 3 < vocab) x.w = p[i + 3];
        }
        x.x = x.x == x.x ? x.x : -INFINITY;
        x.y = x.y == x.y ? x.y : -INFINITY;
        x.z = x.z == x.z ? x.z : -INFINITY;
        x.w = x.w == x.w ? x.w : -INFINITY;
        return x;
    }
    __device__ __forceinline__ void load() {
        if constexpr (N > 0) {
#pragma unroll
            for (int k = 0; k < N / 4; ++k) {
                const float4 x = at(4 * kThreads * k + 4 * int(threadIdx.x));
                r[4 * k] = x.x, r[4 * k + 1] = x.y, r[4 * k + 2] = x.z, r[4 * k + 3] = x.w;
            }
        }
    }
    // f(four logits, index of the first, pass)
    template <class F>
    __device__ __forceinline__ void each4(F f) const {
        if constexpr (N > 0) {
#pragma unroll
            for (int k = 0; k < N / 4; ++k)
                f(make_float4(r[4 * k], r[4 * k + 1], r[4 * k + 2], r[4 * k + 3]),
                  4 * kThreads * k + 4 * int(threadIdx.x), k);
        } else {
            const int passes = (vocab + 4 * kThreads - 1) / (4 * kThreads);
            for (int k = 0; k < passes; ++k) {
                const int i = 4 * kThreads * k + 4 * int(threadIdx.x);
                f(at(i), i, k);
            }
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
};

__device__ __forceinline__ void clear_hist(Shared& s) {
    s.hist[threadIdx.x] = 0;
    s.hist[threadIdx.x + kThreads] = 0;
    if (threadIdx.x == 0) s.n = 0;
    __syncthreads();
}

// v[0 .. n) (n at most 2 * 1024) added up in order: the index where the sum
// reaches `target` (> 0) into s.at, the sum in front of it into s.sum, and the
// whole sum returned. s.at stays -1 where the whole is less.
__device__ u64 find_in(Shared& s, const u64* v, int n, u64 target) {
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    if (t == 0) s.at = -1;
    const u64 x = 2 * t < n ? v[2 * t] : 0, y = 2 * t + 1 < n ? v[2 * t + 1] : 0;
    const u64 incl = wave_scan(x + y);
    if (lane == 63) s.part[wave] = incl;
    __syncthreads();
    u64 before = 0, whole = 0;
    for (int w = 0; w < kWaves; ++w) {
        if (w < wave) before += s.part[w];
        whole += s.part[w];
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

// The cut's token where tokens of the same logit l share it: the `nth` (from
// 1) of them by index.
template <int N>
__device__ u64 nth_equal(Shared& s, const Row<N>& row, float l, u64 nth) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int segs = (row.vocab + kSegment - 1) / kSegment;
    row.each4([&](float4 x, int i, int k) {
        const int c = (i < row.vocab && x.x == l) + (i + 1 < row.vocab && x.y == l) + (i + 2 < row.vocab && x.z == l) +
                      (i + 3 < row.vocab && x.w == l);
        const u64 n = wave_sum(u64(c));
        const int sg = k * kWaves + wave;
        if (lane == 0 && sg < segs) s.seg[sg] = n;
    });
    __syncthreads();
    find_in(s, s.seg, segs, nth);
    const int sg = s.at;
    const u64 want = nth - s.sum;
    if (wave == 0) {
        const int i = sg * kSegment + 4 * lane;
        const float4 x = row.at(i);
        const float v[4] = {x.x, x.y, x.z, x.w};
        u64 c = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) c += i + j < row.vocab && v[j] == l;
        u64 before = wave_scan(c) - c;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (i + j < row.vocab && v[j] == l && ++before == want) s.key = token_key(l, i + j);
    }
    __syncthreads();
    return s.key;
}

// Ranks the s.n tokens of the list, one per thread: how many of them, and how
// much weight, come before this thread's in the tokens' order.
__device__ __forceinline__ void rank_list(const Shared& s, int n, u64 key, int& rank, u64& mass) {
    rank = 0;
    mass = 0;
    for (int j = 0; j < n; ++j) {
        const bool b = s.list[j] > key;
        rank += b;
        mass += b ? s.weights[j] : 0;
    }
}

__device__ __forceinline__ float key_logit(u64 key) {
    const uint32_t o = uint32_t(key >> 32);
    return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}

// The cut that keeps, of the tokens down to `floor` (0: all), the first
// `target` (MASS: the shortest prefix whose weights reach target). s.hist
// holds their counts (weights) by bin.
template <bool MASS, int N>
__device__ u64 find_cut(Shared& s, const Row<N>& row, const Scale& c, u64 floor, u64 target) {
    find_in(s, s.hist, kBins, target);
    const int bin = s.at;
    const u64 left = target - s.sum;  // of this bin
    __syncthreads();
    clear_hist(s);
    auto in_bin = [&](float l, int i) {
        return i < row.vocab && bin_of(log_weight(c, l)) == bin && token_key(l, i) >= floor;
    };
    row.each([&](float l, int i) {
        if (in_bin(l, i)) {
            const int at = atomicAdd(&s.n, 1);
            if (at < kList) {
                s.list[at] = token_key(l, i);
                if (MASS) s.weights[at] = fixed(weight(c, l));
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
            const bool cut = MASS ? mass < left && mass + s.weights[threadIdx.x] >= left : u64(rank) + 1 == left;
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
            if (in_bin(l, i) && (k & mask) == prefix)
                atomicAdd(&s.hist[(k >> shift) & ((1u << bits) - 1)], MASS ? fixed(weight(c, l)) : u64(1));
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
    if (MASS) {
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

// One row per block.
template <int N>
__global__ void __launch_bounds__(kThreads) k_sample(SampleArgs a, bool aligned) {
    __shared__ Shared s;
    const int r = blockIdx.x, t = threadIdx.x, lane = t & 63, wave = t >> 6;
    Row<N> row;
    row.p = a.logits + int64_t(r) * a.stride;
    row.vocab = a.vocab;
    row.aligned = aligned;
    row.load();

    float top = -INFINITY;  // this thread's largest
    row.each([&](float l, int) { top = fmaxf(top, l); });
    const float wm = wave_maximum(top);
    if (lane == 0) s.part[wave] = __float_as_uint(wm);
    if (t == 0) s.key = 0;
    __syncthreads();
    Scale c;
    c.max = __uint_as_float(uint32_t(s.part[0]));
    for (int w = 1; w < kWaves; ++w) c.max = fmaxf(c.max, __uint_as_float(uint32_t(s.part[w])));
    if (c.max == -INFINITY) {  // every token masked
        if (t == 0) put(a, r, -1, 0.0f);
        return;
    }
    const float temp = a.p.d_temperature ? a.p.d_temperature[r] : 1.0f;
    const int top_k = a.p.d_top_k ? a.p.d_top_k[r] : 0;
    const float top_p = a.p.d_top_p ? a.p.d_top_p[r] : 1.0f;
    float min_p = a.p.d_min_p ? a.p.d_min_p[r] : 0.0f;
    min_p = min_p > 0.0f ? fminf(min_p, 1.0f) : 0.0f;
    if (!(temp > 0.0f) || top_k == 1 || top_p <= 0.0f) {  // the largest logit's first index
        u64 best = 0;
        row.each([&](float l, int i) {
            if (l == c.max && i < a.vocab) best = max(best, token_key(l, i));
        });
        if (best) atomicMax(&s.key, best);
        __syncthreads();
        if (t == 0) put(a, r, int(~uint32_t(s.key)), 1.0f);
        return;
    }
    const double cd = fmin(1.4426950408889634 / double(temp), 1e30);
    c.hi = float(cd);
    c.lo = cd < 1e30 ? float(cd - double(c.hi)) : 0.0f;
    float u = a.p.d_uniform[a.state ? a.state[3] : r];
    u = u >= 0.0f ? fminf(u, 0.99999994f) : 0.0f;
    const bool by_k = top_k > 0 && top_k < a.vocab, by_p = top_p < 1.0f;
    __syncthreads();

    if (by_k && top_k <= kFewK) {
        // the top_k threads with the largest maxima hold top_k tokens at least as
        // large as the least of these: their bins bound the candidates
        clear_hist(s);
        if (top > -INFINITY) atomicAdd(&s.hist[bin_of(log_weight(c, top))], u64(1));
        __syncthreads();
        find_in(s, s.hist, kBins, u64(top_k));
        const int last = s.at < 0 ? kBins - 1 : s.at;
        row.each([&](float l, int i) {
            if (i < a.vocab && bin_of(log_weight(c, l)) <= last) {
                const int at = atomicAdd(&s.n, 1);
                if (at < kList) {
                    s.list[at] = token_key(l, i);
                    s.weights[at] = fixed(weight(c, l));
                }
            }
        });
        __syncthreads();
        const int n = s.n;
        if (n <= kList) {
            u64 key = 0, w = 0, mass = 0;
            int rank = kList;
            if (t < n) {
                key = s.list[t];
                w = s.weights[t];
                rank_list(s, n, key, rank, mass);
            }
            if (t < n && rank == min(top_k, n) - 1) s.sum = mass + w;  // what the top k hold
            __syncthreads();
            bool keep = rank < top_k;
            if (by_p) keep = keep && mass < max(u64(1), u64(ceil(double(top_p) * double(s.sum))));
            keep = keep && weight(c, key_logit(key)) >= min_p;
            // by index: the kept tokens in front of this one, and all
            if (!keep) w = 0;
            __syncthreads();
            if (t < n) s.weights[t] = w;
            __syncthreads();
            u64 before = 0, total = 0;
            if (t < n)
                for (int j = 0; j < n; ++j) {
                    const u64 v = s.weights[j];
                    total += v;
                    if (uint32_t(s.list[j]) > uint32_t(key)) before += v;  // ~index: larger is earlier
                }
            const u64 want = u64(double(u) * double(total));
            if (w && before <= want && want < before + w)
                put(a, r, int(~uint32_t(key)), float(double(w) / double(total)));
            return;
        }
        __syncthreads();
    }

    u64 cut = 0;  // the last token kept, 0: all
    if (by_k) {
        clear_hist(s);
        row.each([&](float l, int i) {
            if (i < a.vocab) atomicAdd(&s.hist[bin_of(log_weight(c, l))], u64(1));
        });
        __syncthreads();
        cut = find_cut<false>(s, row, c, 0, u64(top_k));
        __syncthreads();
    }
    if (by_p) {
        clear_hist(s);
        row.each([&](float l, int i) {
            if (i < a.vocab && token_key(l, i) >= cut) atomicAdd(&s.hist[bin_of(log_weight(c, l))], fixed(weight(c, l)));
        });
        __syncthreads();
        const u64 whole = find_in(s, s.hist, kBins, ~u64(0));
        cut = find_cut<true>(s, row, c, cut, max(u64(1), min(whole, u64(ceil(double(top_p) * double(whole))))));
        __syncthreads();
    }
    // the kept weights of each 256 tokens, then the place of u among them
    auto kept = [&](float l, int i) {
        if (i >= a.vocab || token_key(l, i) < cut) return u64(0);
        const float w = weight(c, l);
        return w >= min_p ? fixed(w) : u64(0);
    };
    const int segs = (a.vocab + kSegment - 1) / kSegment;
    row.each4([&](float4 x, int i, int k) {
        const u64 v = wave_sum(kept(x.x, i) + kept(x.y, i + 1) + kept(x.z, i + 2) + kept(x.w, i + 3));
        const int sg = k * kWaves + wave;
        if (lane == 0 && sg < segs) s.seg[sg] = v;
    });
    __syncthreads();
    const u64 total = find_in(s, s.seg, segs, ~u64(0));
    const u64 want = u64(double(u) * double(total));
    find_in(s, s.seg, segs, want + 1);
    if (wave == 0) {
        const int i = s.at * kSegment + 4 * lane;
        const float4 x = row.at(i);
        const u64 v[4] = {kept(x.x, i), kept(x.y, i + 1), kept(x.z, i + 2), kept(x.w, i + 3)};
        const u64 sum = v[0] + v[1] + v[2] + v[3];
        u64 before = s.sum + wave_scan(sum) - sum;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (v[j] && before <= want && want < before + v[j])
                put(a, r, i + j, float(double(v[j]) / double(total)));
            before += v[j];
        }
    }
}

}  // namespace

int launch_sample(const SampleArgs& a, hipStream_t s) {
    const bool al = !(reinterpret_cast<uintptr_t>(a.logits) & 15) && a.stride % 4 == 0;
    auto go = [&](auto kern) { hipLaunchKernelGGL(kern, dim3(unsigned(a.rows)), dim3(kThreads), 0, s, a, al); };
    if (a.vocab <= 8 * kThreads)
        go(k_sample<8>);
    else if (a.vocab <= 32 * kThreads)
        go(k_sample<32>);
    else
        go(k_sample<0>);
    return int(hipGetLastError());
}

}  // namespace wv

using namespace wv;

extern "C" int wv_sample_dev(const float* d_logits, int64_t stride, int32_t rows, int32_t vocab,
                             const wv_sampling* sampling, int32_t* d_tokens, float* d_probs, void* stream) {
    if (!sampling) return rt_fail(WV_E_ARG, "wv_sample: nil sampling");
    if (rows < 0 || vocab <= 0 || vocab > kMaxVocab)
        return rt_fail(WV_E_SHAPE, "wv_sample: %d rows of %d logits (1 to %d)", rows, vocab, kMaxVocab);
    if (!stride) stride = vocab;
    if (stride < vocab)
        return rt_fail(WV_E_SHAPE, "wv_sample: row stride %lld under %d logits", (long long)stride, vocab);
    if (!rows) return WV_OK;
    if (!d_logits || !d_tokens || !sampling->d_uniform) return rt_fail(WV_E_ARG, "wv_sample: nil logits/tokens/uniform");
    const int rc = rt_ensure_init();
    if (rc) return rc;
    SampleArgs a{};
    a.logits = d_logits, a.stride = stride, a.rows = rows, a.vocab = vocab;
    a.p = *sampling, a.tokens = d_tokens, a.probs = d_probs;
    const int e = launch_sample(a, rt_stream(stream, rt_current_device()));
    return e == hipSuccess ? WV_OK : rt_hip_fail(hipError_t(e), "wv_sample: kernel launch");
}
