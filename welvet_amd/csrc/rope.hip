// rope.hip — rotary positions: pairs of a head's values turned by an angle that
// grows with the row's position.
//
// Pair i of the first rot values of a head, (a, b) at (i, i + rot/2) or at
// (2i, 2i + 1), becomes gain (a cos t - b sin t, a sin t + b cos t) with
// t = pos f_i (layers/mha/rope.go:6-21 is the first layout with f_i =
// theta^(-2i/rot)). The handle keeps f_i / 2 pi in f64: the turns pos f_i /
// 2 pi are taken modulo one there, where a position of 2^31 leaves 2^-22 of a
// turn and one of 2^17 2^-36, and the sine and cosine of what is left in f32.
//
// Bound by the rows' bytes: 8191 rows of 40 heads of 128 in 63.6 us, 5.3 TB/s read
// and written (a large copy: 5.1); a launch, 4.7 us, up to 64 rows. Every value
// turned by a thread of its own, with an angle for each, took 132 us.
#include <algorithm>
#include <cmath>
#include <mutex>
#include <new>
#include <unordered_map>
#include <vector>

#include "../../include/welvet_hip.h"
#include "rt_internal.h"

namespace wv {
namespace {

struct Rope {
    wv_rope_config c{};
    int device = 0;
    double* turns = nullptr;  // [rot_dim / 2]
};
std::mutex g_mu;
std::unordered_map<uint64_t, Rope> g_ropes;
uint64_t g_next = 1;

bool rope_lookup(uint64_t h, Rope& out) {
    std::lock_guard<std::mutex> lk(g_mu);
    auto it = g_ropes.find(h);
    if (it == g_ropes.end()) return false;
    out = it->second;
    return true;
}

struct RopeRows {
    const float* x;
    float* y;
    int64_t xs, ys;
    int heads;
};
struct RopeArgs {
    RopeRows q, k;
    const double* turns;
    const int32_t* pos;
    int n, hd, rot;
    float gain;
};

// Cosine and sine, with the gain, of pair d at position p.
__device__ __forceinline__ void turn_of(const RopeArgs& a, double p, int d, float& c, float& s) {
    const double turn = p * a.turns[d];
    sincospif(2.0f * float(turn - rint(turn)), &s, &c);
    s *= a.gain, c *= a.gain;
}

typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));

// Eight values a thread: four pairs, or values that stay (of pairs side by side, where rot ends within the eight, both).
// A thread keeps its four angles and turns them in every head that is its; kAhead heads' values are on their way before
// the sines are taken. NT: rows of more than the caches hold are written past them.
constexpr int kAhead = 3;
template <bool PAIRS, bool NT>
__global__ void __launch_bounds__(256) k_rope8(RopeArgs a, int units, int heads_a_pass) {
    const int t = blockIdx.x, hp = threadIdx.x / units, u = threadIdx.x - hp * units;
    if (hp >= heads_a_pass) return;
    const int heads = a.q.heads + a.k.heads, half = a.rot / 2, turned = (a.rot + 7) / 8;
    const bool stays = u >= turned;
    const int i0 = stays || PAIRS ? 8 * u : 4 * u, i1 = stays || PAIRS ? i0 + 4 : i0 + half;
    const int step = heads_a_pass * gridDim.y;
    const float* x[kAhead];
    float* y[kAhead];
    f4 lo[kAhead], hi[kAhead];
    auto load = [&](int h0) {
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const int h = min(h0 + k * step, heads - 1);
            const bool q = h < a.q.heads;
            const RopeRows& r = q ? a.q : a.k;
            const int64_t at = int64_t(q ? h : h - a.q.heads) * a.hd;
            x[k] = r.x + t * r.xs + at;
            y[k] = r.y + t * r.ys + at;
            lo[k] = *reinterpret_cast<const f4*>(x[k] + i0);
            hi[k] = *reinterpret_cast<const f4*>(x[k] + i1);
        }
    };
    int h0 = hp + heads_a_pass * blockIdx.y;
    if (h0 >= heads) return;
    load(h0);
    float c[4], s[4];
    if (!stays) {
        const double p = double(a.pos[t]);
#pragma unroll
        for (int i = 0; i < 4; ++i) turn_of(a, p, PAIRS ? min(4 * u + i, half - 1) : 4 * u + i, c[i], s[i]);
    }
    for (; h0 < heads; h0 += kAhead * step, load(h0)) {
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            if (h0 + k * step >= heads || (stays && x[k] == y[k])) continue;
            f4 l = lo[k], m = hi[k];
            if (!stays) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    // values a and b of pair i
                    const float p = PAIRS ? (i < 2 ? lo[k][2 * i] : hi[k][2 * i - 4]) : lo[k][i];
                    const float r = PAIRS ? (i < 2 ? lo[k][2 * i + 1] : hi[k][2 * i - 3]) : hi[k][i];
                    float v = fmaf(p, c[i], -(r * s[i])), w = fmaf(p, s[i], r * c[i]);
                    if (PAIRS && 4 * u + i >= half) v = p, w = r;
                    if (!PAIRS)
                        l[i] = v, m[i] = w;
                    else if (i < 2)
                        l[2 * i] = v, l[2 * i + 1] = w;
                    else
                        m[2 * i - 4] = v, m[2 * i - 3] = w;
                }
            }
            if (NT) {
                __builtin_nontemporal_store(l, reinterpret_cast<f4*>(y[k] + i0));
                __builtin_nontemporal_store(m, reinterpret_cast<f4*>(y[k] + i1));
            } else {
                *reinterpret_cast<f4*>(y[k] + i0) = l;
                *reinterpret_cast<f4*>(y[k] + i1) = m;
            }
        }
    }
}

// Heads that are no multiple of eight values, or not turned by one: a pair, or a value that stays, a thread.
template <bool PAIRS>
__global__ void __launch_bounds__(256) k_rope(RopeArgs a) {
    const int t = blockIdx.x, half = a.rot / 2;
    const int per = half + (a.hd - a.rot);  // a head's pairs, and its values that stay
    const double p = double(a.pos[t]);
    for (int i = blockIdx.y * 256 + threadIdx.x; i < per * (a.q.heads + a.k.heads); i += gridDim.y * 256) {
        int h = i / per;
        const int d = i % per;
        const RopeRows& r = h < a.q.heads ? a.q : a.k;
        if (h >= a.q.heads) h -= a.q.heads;
        const float* x = r.x + t * r.xs + int64_t(h) * a.hd;
        float* y = r.y + t * r.ys + int64_t(h) * a.hd;
        if (d >= half) {
            const int j = d - half + a.rot;
            if (x != y) y[j] = x[j];
            continue;
        }
        float s, c;
        turn_of(a, p, d, c, s);
        const int i0 = PAIRS ? 2 * d : d, i1 = PAIRS ? 2 * d + 1 : d + half;
        const float x0 = x[i0], x1 = x[i1];
        y[i0] = fmaf(x0, c, -(x1 * s));
        y[i1] = fmaf(x0, s, x1 * c);
    }
}

// f_i / 2 pi of every pair.
std::vector<double> rope_turns(const wv_rope_config& c) {
    const double two_pi = 6.283185307179586476925286766559;
    const int half = c.rot_dim / 2;
    std::vector<double> f(static_cast<size_t>(half));
    const double theta = c.scaling == WV_ROPE_BASE ? c.theta * std::pow(c.factor, double(c.rot_dim) / double(c.rot_dim - 2))
                                                   : c.theta;
    double i0 = 0.0, i1 = 0.0;
    if (c.scaling == WV_ROPE_RAMP_DIMS) {
        const auto at = [&](double n) { return c.rot_dim * std::log(c.trained / (two_pi * n)) / (2.0 * std::log(theta)); };
        // as published the range ends at rot - 1, behind the last pair: of long trained lengths that pair is not all scaled
        i0 = std::fmin(std::fmax(std::floor(at(c.high)), 0.0), c.rot_dim - 1.0);
        i1 = std::fmin(std::fmax(std::ceil(at(c.low)), 0.0), c.rot_dim - 1.0);
    }
    for (int i = 0; i < half; ++i) {
        double w = std::pow(theta, -2.0 * i / c.rot_dim);
        if (c.scaling == WV_ROPE_LINEAR) w /= c.factor;
        if (c.scaling == WV_ROPE_RAMP_DIMS || c.scaling == WV_ROPE_RAMP_TURNS) {
            double r = c.scaling == WV_ROPE_RAMP_DIMS ? 1.0 - (i - i0) / std::fmax(i1 - i0, 0.001)
                                                      : (c.trained * w / two_pi - c.low) / (c.high - c.low);
            r = std::fmin(std::fmax(r, 0.0), 1.0);
            w = w * (1.0 - r) / c.factor + w * r;
        }
        f[size_t(i)] = w / two_pi;
    }
    return f;
}

}  // namespace
}  // namespace wv

using namespace wv;

extern "C" {

int wv_rope_create(const wv_rope_config* cfg, uint64_t* rope) try {
    if (!cfg || !rope) return rt_fail(WV_E_ARG, "wv_rope_create: nil argument");
    const wv_rope_config& c = *cfg;
    if (c.head_dim < 2 || c.head_dim > 1024 || c.rot_dim < 2 || c.rot_dim > c.head_dim || c.rot_dim % 2)
        return rt_fail(WV_E_SHAPE, "wv_rope_create: %d of %d values of a head (an even number, heads of 2 to 1024)",
                       c.rot_dim, c.head_dim);
    if (c.layout != WV_ROPE_HALF && c.layout != WV_ROPE_PAIRS)
        return rt_fail(WV_E_ARG, "wv_rope_create: layout %d", c.layout);
    if (c.scaling < WV_ROPE_NONE || c.scaling > WV_ROPE_RAMP_TURNS)
        return rt_fail(WV_E_ARG, "wv_rope_create: scaling %d", c.scaling);
    if (!(c.theta > 1.0) || !std::isfinite(c.theta) || !(float(c.gain) > 0.0f) || !std::isfinite(float(c.gain)))
        return rt_fail(WV_E_ARG, "wv_rope_create: theta %g, gain %g", c.theta, c.gain);
    if (c.scaling != WV_ROPE_NONE && (!(c.factor > 0.0) || !std::isfinite(c.factor)))
        return rt_fail(WV_E_ARG, "wv_rope_create: factor %g", c.factor);
    if (c.scaling == WV_ROPE_BASE && (c.rot_dim < 4 || !(c.theta * std::pow(c.factor, c.rot_dim / (c.rot_dim - 2.0)) > 1.0)))
        return rt_fail(WV_E_ARG, "wv_rope_create: theta %g by factor %g on %d values", c.theta, c.factor, c.rot_dim);
    if (c.scaling >= WV_ROPE_RAMP_DIMS && (c.trained <= 0 || !(c.low > 0.0) || !(c.high > c.low) || !std::isfinite(c.high)))
        return rt_fail(WV_E_ARG, "wv_rope_create: %d trained positions, turns %g to %g", c.trained, c.low, c.high);
    Rope r;
    r.c = c;
    const std::vector<double> turns = rope_turns(c);
    // a factor next to 0 has no frequencies, and a gain that f32 does not hold would make NaN of zeros
    for (const double t : turns)
        if (!std::isfinite(t)) return rt_fail(WV_E_ARG, "wv_rope_create: frequencies past f64 at factor %g", c.factor);
    int rc = rt_ensure_init();
    if (rc) return rc;
    r.device = rt_current_device();
    hipError_t e = hipMalloc(reinterpret_cast<void**>(&r.turns), turns.size() * sizeof(double));
    if (e == hipSuccess) {
        e = hipMemcpy(r.turns, turns.data(), turns.size() * sizeof(double), hipMemcpyHostToDevice);
        if (e != hipSuccess) (void)hipFree(r.turns);
    }
    if (e != hipSuccess) {
        (void)hipGetLastError();
        return rt_hip_fail(e, "wv_rope_create: frequencies");
    }
    try {
        std::lock_guard<std::mutex> lk(g_mu);
        g_ropes[g_next] = r;
        *rope = g_next++;
    } catch (const std::bad_alloc&) {
        (void)hipFree(r.turns);
        throw;
    }
    return WV_OK;
} catch (const std::bad_alloc&) {
    return rt_fail(WV_E_OOM, "wv_rope_create: host memory exhausted");
}

int wv_rope_free(uint64_t rope) {
    Rope r;
    {
        std::lock_guard<std::mutex> lk(g_mu);
        auto it = g_ropes.find(rope);
        if (it == g_ropes.end())
            return rt_fail(WV_E_HANDLE, "wv_rope_free: unknown rope %llu", (unsigned long long)rope);
        r = it->second;
        g_ropes.erase(it);
    }
    (void)hipSetDevice(r.device);
    const hipError_t e = hipFree(r.turns);  // waits for the device's work
    return e == hipSuccess ? WV_OK : rt_hip_fail(e, "wv_rope_free");
}

int wv_rope_dev(uint64_t rope, const int32_t* d_pos, int32_t n, const wv_rope_rows* q, const wv_rope_rows* k,
                void* stream) {
    Rope r;
    if (!rope_lookup(rope, r)) return rt_fail(WV_E_HANDLE, "wv_rope: unknown rope %llu", (unsigned long long)rope);
    if (n < 0 || n > 1 << 23) return rt_fail(WV_E_SHAPE, "wv_rope: %d rows (at most 2^23)", n);  // 2^31 threads a launch
    RopeArgs a{};
    const wv_rope_rows* in[2] = {q, k};
    RopeRows* to[2] = {&a.q, &a.k};
    for (int i = 0; i < 2; ++i) {
        if (!in[i] || !in[i]->n_heads) continue;
        const wv_rope_rows& x = *in[i];
        if (x.n_heads < 0 || x.n_heads > 65535) return rt_fail(WV_E_SHAPE, "wv_rope: %d heads", x.n_heads);
        const int64_t w = int64_t(x.n_heads) * r.c.head_dim;
        RopeRows& y = *to[i];
        y = {x.d_x, x.d_y ? x.d_y : const_cast<float*>(x.d_x), x.x_stride ? x.x_stride : w,
             x.d_y ? (x.y_stride ? x.y_stride : w) : (x.x_stride ? x.x_stride : w), x.n_heads};
        if (y.xs < w || y.ys < w)
            return rt_fail(WV_E_SHAPE, "wv_rope: row strides %lld and %lld under the row's %lld floats", (long long)y.xs,
                           (long long)y.ys, (long long)w);
        if (n && !x.d_x) return rt_fail(WV_E_ARG, "wv_rope: nil rows");
        if (y.x == y.y && y.xs != y.ys)  // rows written would be others still to be read
            return rt_fail(WV_E_SHAPE, "wv_rope: rows turned in place at strides of %lld and %lld", (long long)y.xs,
                           (long long)y.ys);
    }
    if (!n || !(a.q.heads + a.k.heads)) return WV_OK;
    if (!d_pos) return rt_fail(WV_E_ARG, "wv_rope: nil pos");
    if (a.q.heads && a.k.heads && (a.q.y == a.k.y || a.q.y == a.k.x || a.k.y == a.q.x))  // turned once, twice or half
        return rt_fail(WV_E_ARG, "wv_rope: the rows of q are those of k");
    a.turns = r.turns, a.pos = d_pos, a.n = n, a.hd = r.c.head_dim, a.rot = r.c.rot_dim, a.gain = float(r.c.gain);
    (void)hipSetDevice(r.device);
    hipStream_t s = rt_stream(stream, r.device);
    const bool pairs = r.c.layout == WV_ROPE_PAIRS;
    const int heads = a.q.heads + a.k.heads;
    if (a.hd % 8 == 0 && (pairs || a.rot % 8 == 0)) {
        const int units = a.hd / 8, pass = 256 / units, passes = (heads + pass - 1) / pass;
        // One block turns all heads of a row, unless there are few rows (2047 of 40 heads of 128 in one block each 14.0
        // us, in two 15.1, in three 17.1). Past the caches from 16 MB on: 512 rows 4.8 us so, else 5.9; 64 rows 4.7.
        const int split = std::min(passes, std::max(1, 256 / n));
        const bool nt = int64_t(n) * heads * a.hd * 8 > int64_t(16) << 20;
        auto kern = pairs ? (nt ? k_rope8<true, true> : k_rope8<true, false>) : (nt ? k_rope8<false, true> : k_rope8<false, false>);
        hipLaunchKernelGGL(kern, dim3(unsigned(n), unsigned(split)), dim3(256), 0, s, a, units, pass);
    } else {
        hipLaunchKernelGGL(pairs ? k_rope<true> : k_rope<false>, dim3(unsigned(n)), dim3(256), 0, s, a);
    }
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? WV_OK : rt_hip_fail(e, "wv_rope: kernel launch");
}

}  // extern "C"
