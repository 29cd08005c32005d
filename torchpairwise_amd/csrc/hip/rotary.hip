// Rotary positions: every pair of features of a row turns by position * frequency, so that the inner
// product of two rows depends on the difference of their positions.
//   (u, w) -> scale (u cos t - w sin t, u sin t + w cos t)
// Bound by memory: each row is read and written once (4 x 16 x 8192 x 128 bf16: 55 us, 4.9 TB/s, the rate of
// a copy).  A thread owns one group of kPairs pairs of
// one position and walks over heads, so that its angles (64-bit products, which a position of 10^6
// needs: fp32 holds its angle to 0.06) are formed once for all of them.
#include <math.h>

#include "common.hpp"

namespace tpw {
namespace {

struct RotaryArgs {
    const void *x;
    void *out;
    const int64_t *positions;
    const double *frequencies;
    int64_t xb, xh, xn, ob, oh, on, pb, pn;
    int64_t batch, heads, n, d, pairs, groups, head_parts;
    float scale, sign;
};

// cos and sin of t = position * frequency in turns: the fraction of t / 2 pi in 64 bits, then fp32.
__device__ __forceinline__ void angle(double position, double turns, float scale, float sign, float &c, float &s) {
    double t = position * turns;
    t -= rint(t);
    // what the angle loses in 32 bits turns the sine and cosine a little further
    const float hi = (float)t, lo = (float)(t - (double)hi) * 6.28318530717958648f;
    float ss, cc;
    sincospif(2.0f * hi, &ss, &cc);
    c = __builtin_fmaf(-lo, ss, cc) * scale;
    s = __builtin_fmaf(lo, cc, ss) * scale * sign;
}

// P pairs at a time: P consecutive features of both halves, or 2 P consecutive ones (INTERLEAVED).
template <typename T, int P, bool INTERLEAVED>
__device__ __forceinline__ void turn(const T *x, T *o, int64_t p0, int64_t pairs, const float (&c)[P],
                                     const float (&s)[P]) {
    constexpr int kAlign = 2 * P * sizeof(T) < 16 ? 2 * P * sizeof(T) : 16;
    T u[P], w[P];
    if constexpr (P == 1) {
        const int64_t i = INTERLEAVED ? 2 * p0 : p0, j = INTERLEAVED ? i + 1 : p0 + pairs;
        u[0] = x[i];
        w[0] = x[j];
        const float a = to_f32(u[0]), b = to_f32(w[0]);
        from_f32(o + i, a * c[0] - b * s[0]);
        from_f32(o + j, a * s[0] + b * c[0]);
    } else if constexpr (INTERLEAVED) {
        T v[2 * P], r[2 * P];
        __builtin_memcpy(v, __builtin_assume_aligned(x + 2 * p0, kAlign), sizeof(v));
#pragma unroll
        for (int e = 0; e < P; ++e) {
            const float a = to_f32(v[2 * e]), b = to_f32(v[2 * e + 1]);
            from_f32(&r[2 * e], a * c[e] - b * s[e]);
            from_f32(&r[2 * e + 1], a * s[e] + b * c[e]);
        }
        __builtin_memcpy(__builtin_assume_aligned(o + 2 * p0, kAlign), r, sizeof(r));
    } else {
        T ru[P], rw[P];
        __builtin_memcpy(u, __builtin_assume_aligned(x + p0, P * sizeof(T)), sizeof(u));
        __builtin_memcpy(w, __builtin_assume_aligned(x + p0 + pairs, P * sizeof(T)), sizeof(w));
#pragma unroll
        for (int e = 0; e < P; ++e) {
            const float a = to_f32(u[e]), b = to_f32(w[e]);
            from_f32(&ru[e], a * c[e] - b * s[e]);
            from_f32(&rw[e], a * s[e] + b * c[e]);
        }
        __builtin_memcpy(__builtin_assume_aligned(o + p0, P * sizeof(T)), ru, sizeof(ru));
        __builtin_memcpy(__builtin_assume_aligned(o + p0 + pairs, P * sizeof(T)), rw, sizeof(rw));
    }
}

// Threads: [batch, head part, row, group], groups = pair groups, then groups of 2 P copied features.
template <typename T, int P, bool INTERLEAVED>
__global__ __launch_bounds__(256) void rotary_kernel(const RotaryArgs a) {
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t gi = id % a.groups, r = id / a.groups, i = r % a.n, bp = r / a.n;
    const int64_t b = bp / a.head_parts, part = bp % a.head_parts;
    if (b >= a.batch) return;
    const int64_t h0 = a.heads * part / a.head_parts, h1 = a.heads * (part + 1) / a.head_parts;
    const T *x = reinterpret_cast<const T *>(a.x) + b * a.xb + i * a.xn;
    T *o = reinterpret_cast<T *>(a.out) + b * a.ob + i * a.on;
    const int64_t turned = a.pairs / P;
    if (gi < turned) {
        const double pos = (double)a.positions[b * a.pb + i * a.pn];
        float c[P], s[P];
#pragma unroll
        for (int e = 0; e < P; ++e)
            angle(pos, a.frequencies[gi * P + e] * 0.15915494309189533577, a.scale, a.sign, c[e], s[e]);
        for (int64_t h = h0; h < h1; ++h)
            turn<T, P, INTERLEAVED>(x + h * a.xh, o + h * a.oh, gi * P, a.pairs, c, s);
    } else {
        const int64_t f = 2 * a.pairs + (gi - turned) * 2 * P;
        for (int64_t h = h0; h < h1; ++h) {
            T v[2 * P];
            if constexpr (P == 1) {
                for (int e = 0; e < 2; ++e)
                    if (f + e < a.d) o[h * a.oh + f + e] = x[h * a.xh + f + e];
            } else {
                constexpr int kAlign = 2 * P * sizeof(T) < 16 ? 2 * P * sizeof(T) : 16;
                __builtin_memcpy(v, __builtin_assume_aligned(x + h * a.xh + f, kAlign), sizeof(v));
                __builtin_memcpy(__builtin_assume_aligned(o + h * a.oh + f, kAlign), v, sizeof(v));
            }
        }
    }
}

template <typename T, int P>
int launch(RotaryArgs &a, int interleaved, hipStream_t s) {
    a.groups = a.pairs / P + cdiv(a.d - 2 * a.pairs, 2 * P);
    // heads are shared out until the threads fill the card
    const int64_t one = a.batch * a.n * a.groups;
    int64_t parts = cdiv((int64_t)256 * 2048, one);
    a.head_parts = parts < a.heads ? parts : a.heads;
    const int64_t blocks = cdiv(one * a.head_parts, 256);
    TPW_REQUIRE(blocks < (int64_t(1) << 31), "rotary: too many rows");
    if (interleaved)
        hipLaunchKernelGGL((rotary_kernel<T, P, true>), dim3((unsigned)blocks), dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL((rotary_kernel<T, P, false>), dim3((unsigned)blocks), dim3(256), 0, s, a);
    return check_launch("rotary_kernel");
}

}  // namespace
}  // namespace tpw

using namespace tpw;

extern "C" int tpw_rotary(const void *x, int dtype, int64_t batch, int64_t heads, int64_t n, int64_t d,
                          const int64_t *xs, const int64_t *positions, const int64_t *ps, const double *frequencies,
                          int64_t pairs, int interleaved, int inverse, double scale, void *out, const int64_t *os,
                          void *stream) {
    TPW_REQUIRE(dtype == TPW_F32 || dtype == TPW_BF16, "rotary: float32 or bfloat16 rows");
    TPW_REQUIRE(batch >= 0 && heads >= 0 && n >= 0 && d >= 0 && pairs >= 0 && 2 * pairs <= d, "rotary: invalid sizes");
    TPW_REQUIRE(scale == scale && fabs(scale) <= 3e38, "rotary: scale must be finite");
    if (batch * heads * n * d == 0) return TPW_OK;
    TPW_REQUIRE(x && out && xs && os && (pairs == 0 || (positions && ps && frequencies)), "rotary: null operand");
    RotaryArgs a = {};
    a.x = x;
    a.out = out;
    a.positions = positions;
    a.frequencies = frequencies;
    a.xb = xs[0], a.xh = xs[1], a.xn = xs[2];
    a.ob = os[0], a.oh = os[1], a.on = os[2];
    if (ps) a.pb = ps[0], a.pn = ps[1];
    a.batch = batch, a.heads = heads, a.n = n, a.d = d, a.pairs = pairs;
    a.scale = (float)scale;
    a.sign = inverse ? -1.0f : 1.0f;
    // a group of P pairs is read as two runs of P features, or as one of 2 P: each has to start at a
    // multiple of its size and hold whole groups
    const int64_t size = dtype == TPW_F32 ? 4 : 2;
    const auto fits = [&](int64_t p) {
        const int64_t bytes = (interleaved ? 2 * p : p) * size, align = bytes < 16 ? bytes : 16;
        const auto at = [&](const void *q, int64_t b, int64_t h, int64_t r) {
            return reinterpret_cast<uintptr_t>(q) % align == 0 && b * size % align == 0 && h * size % align == 0 &&
                   r * size % align == 0;
        };
        const int64_t rest = d - 2 * pairs, copy = 2 * p * size < 16 ? 2 * p * size : 16;
        return pairs % p == 0 && at(x, a.xb, a.xh, a.xn) && at(out, a.ob, a.oh, a.on) &&
               (rest == 0 || (rest % (2 * p) == 0 && 2 * pairs * size % copy == 0 &&
                              reinterpret_cast<uintptr_t>(x) % copy == 0 &&
                              reinterpret_cast<uintptr_t>(out) % copy == 0 &&
                              a.xb * size % copy == 0 && a.xh * size % copy == 0 && a.xn * size % copy == 0 &&
                              a.ob * size % copy == 0 && a.oh * size % copy == 0 && a.on * size % copy == 0));
    };
    hipStream_t s = as_stream(stream);
    if (dtype == TPW_F32) {
        if (fits(4)) return launch<float, 4>(a, interleaved, s);
        if (fits(2)) return launch<float, 2>(a, interleaved, s);
        return launch<float, 1>(a, interleaved, s);
    }
    if (fits(8)) return launch<uint16_t, 8>(a, interleaved, s);
    if (fits(4)) return launch<uint16_t, 4>(a, interleaved, s);
    if (fits(2)) return launch<uint16_t, 2>(a, interleaved, s);
    return launch<uint16_t, 1>(a, interleaved, s);
}
