// Sums that log probabilities and entropies come from, shared by the kernels that read logits and the one that computes them.
//
// Of a part of a row of logits x: m its maximum, s = sum exp(x - m), t = sum exp(x - m) (x - m).  Then over the whole row
//     log p(i) = (x_i - m) - log s,      entropy = -sum p log p = log s - t / s      (both terms are >= 0: nothing cancels).
// When the maximum rises by delta the sums are carried over with f = exp(-delta): t <- f (t - s delta), s <- f s.
//
// Differences below -1000 count as -1000, where exp is 0 already: a logit of -inf, or of the type's lowest number, then adds 0 to s and
// to t.  NaN and +inf make s and t NaN, as they do in the formulas.
#pragma once

#include "common.cuh"

namespace pb {

constexpr float kScoreLog2e = 1.4426950408889634f;
constexpr float kFar = -1000.0f;         // exp of it is 0, and times any sum of 32 bits' worth of elements it stays finite

struct Stats {
    float m, s, t;
};

// 2^x by the special-function unit alone: 2 ulp like exp2f, results below 2^-126 are 0 (beside a sum that holds exp(0) = 1).
__device__ __forceinline__ float pow2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Brings `a` and `b` under the larger of their maxima.  A part without a number has m = -inf, and s = t = 0 (or NaN).
__device__ __forceinline__ Stats join(const Stats& a, const Stats& b) {
    const float m = fmaxf(a.m, b.m);
    const float da = a.m == -INFINITY ? 0.0f : fmaxf(a.m - m, kFar), db = b.m == -INFINITY ? 0.0f : fmaxf(b.m - m, kFar);
    const float fa = pow2(da * kScoreLog2e), fb = pow2(db * kScoreLog2e);
    return Stats{m, a.s * fa + b.s * fb, fa * (a.t + a.s * da) + fb * (b.t + b.s * db)};
}

// The lanes' sums as one, the same in all lanes.
__device__ __forceinline__ Stats warp_join(Stats st) {
    const float m = warp_max(st.m);
    const float delta = st.m == -INFINITY ? 0.0f : fmaxf(st.m - m, kFar), f = pow2(delta * kScoreLog2e);
    return Stats{m, warp_sum(st.s * f), warp_sum(f * (st.t + st.s * delta))};
}

// Two float32 at a time (one instruction each on sm_100).
typedef unsigned long long Two;
__device__ __forceinline__ Two two(float a, float b) {
    Two v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
    return v;
}
__device__ __forceinline__ void apart(Two v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ Two add2(Two a, Two b) {
    Two v;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
    return v;
}
__device__ __forceinline__ Two mul2(Two a, Two b) {
    Two v;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
    return v;
}
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) {
    Two v;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
    return v;
}

// Brings the sums under `top` where that is beyond their maximum.
__device__ __forceinline__ void raise(Stats& st, float top) {
    if (top > st.m) {
        if (st.m > -INFINITY) {
            const float delta = fmaxf(st.m - top, kFar), f = pow2(delta * kScoreLog2e);
            st.t = f * (st.t + st.s * delta);
            st.s *= f;
        }
        st.m = top;
    }
}

// Adds N logits (N even) to sums under `base`; BOUNDED: none is so far below it that the difference overflows.  Two pairs of sums of each
// kind are kept apart, so that additions do not wait for one another.
template <bool BOUNDED, int N>
__device__ __forceinline__ void add_under(Stats& st, float base, const float (&x)[N]) {
    const Two lower = two(-base, -base), log2e = two(kScoreLog2e, kScoreLog2e);
    Two s[2] = {0, 0}, t[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < N; i += 2) {
        Two d = add2(two(x[i], x[i + 1]), lower);
        const Two y = mul2(d, log2e);
        float y0, y1;
        apart(y, y0, y1);
        const Two e = two(pow2(y0), pow2(y1));
        if (!BOUNDED) {
            float d0, d1;
            apart(d, d0, d1);
            d = two(fmaxf(d0, kFar), fmaxf(d1, kFar));
        }
        s[i / 2 % 2] = add2(s[i / 2 % 2], e);
        t[i / 2 % 2] = fma2(e, d, t[i / 2 % 2]);
    }
    float s0, s1, t0, t1;
    apart(add2(s[0], s[1]), s0, s1);
    apart(add2(t[0], t[1]), t0, t1);
    st.s += s0 + s1;
    st.t += t0 + t1;
}
template <int N>
__device__ __forceinline__ void add_bounded(Stats& st, float base, const float (&x)[N]) { add_under<true>(st, base, x); }

// Adds N logits.
template <int N>
__device__ __forceinline__ void add_logits(Stats& st, const float (&x)[N]) {
    float top = x[0];
#pragma unroll
    for (int i = 1; i < N; ++i) top = fmaxf(top, x[i]);
    raise(st, top);
    add_under<false>(st, st.m == -INFINITY ? 0.0f : st.m, x);
}

// The sums of one logit.
__device__ __forceinline__ Stats one_logit(float x) {
    const float d = x == -INFINITY ? x : x - x, e = pow2(d);                  // x - x: 0, or NaN for NaN and +inf
    return Stats{x == x ? x : -INFINITY, e, e * fmaxf(d, kFar)};
}

}  // namespace pb
