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
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const Stats other = {__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.s, o), __shfl_xor_sync(0xffffffffu, st.t, o)};
        st = join(st, other);
    }
    return st;
}

// Adds N logits.  Four sums of each kind are kept apart, so that additions do not wait for one another.
template <int N>
__device__ __forceinline__ void add_logits(Stats& st, const float (&x)[N]) {
    float top = x[0];
#pragma unroll
    for (int i = 1; i < N; ++i) top = fmaxf(top, x[i]);
    if (top > st.m) {
        if (st.m > -INFINITY) {
            const float delta = fmaxf(st.m - top, kFar), f = pow2(delta * kScoreLog2e);
            st.t = f * (st.t + st.s * delta);
            st.s *= f;
        }
        st.m = top;
    }
    const float base = st.m == -INFINITY ? 0.0f : st.m;
    constexpr int kApart = N < 4 ? N : 4;
    float s[kApart] = {}, t[kApart] = {};
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float d = x[i] - base, e = pow2(d * kScoreLog2e);
        s[i % kApart] += e;
        t[i % kApart] = fmaf(e, fmaxf(d, kFar), t[i % kApart]);
    }
#pragma unroll
    for (int i = 1; i < kApart; ++i) { s[0] += s[i]; t[0] += t[i]; }
    st.s += s[0];
    st.t += t[0];
}

}  // namespace pb
