// rope.hip — rotary positions: pairs of a head's values turned by an angle that
// grows with the row's position.
//
// Pair i of the first rot values of a head, (a, b) at (i, i + rot/2) or at
// (2i, 2i + 1), becomes gain (a cos t - b sin t, a sin t + b cos t) with
// t = pos f_i (layers/mha/rope.go:6-21 is the first layout with f_i =
// theta^(-2i/rot)). The handle keeps f_i / 2 pi in f64: the turns pos f_i /
// 2 pi are taken modulo one there, where a position of 2^31 leaves 2^-22 of a
// turn and one of 2^17 2^-36, and the sine and cosine of what is left in f32.
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

// A thread keeps the angle of one pair and turns it in every head that is its.
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
        const double turn = p * a.turns[d];
        float s, c;
        sincospif(2.0f * float(turn - rint(turn)), &s, &c);
        s *= a.gain, c *= a.gain;
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
        i0 = std::fmin(std::fmax(std::floor(at(c.high)), 0.0), half - 1.0);
        i1 = std::fmin(std::fmax(std::ceil(at(c.low)), 0.0), half - 1.0);
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
    if (!(c.theta > 1.0) || !std::isfinite(c.theta) || !(c.gain > 0.0) || !std::isfinite(c.gain))
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
    if (n < 0 || n > 1 << 28) return rt_fail(WV_E_SHAPE, "wv_rope: %d rows", n);
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
    a.turns = r.turns, a.pos = d_pos, a.n = n, a.hd = r.c.head_dim, a.rot = r.c.rot_dim, a.gain = float(r.c.gain);
    (void)hipSetDevice(r.device);
    hipStream_t s = rt_stream(stream, r.device);
    hipLaunchKernelGGL(r.c.layout == WV_ROPE_PAIRS ? k_rope<true> : k_rope<false>, dim3(unsigned(n)), dim3(256), 0, s, a);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? WV_OK : rt_hip_fail(e, "wv_rope: kernel launch");
}

}  // extern "C"
