// What the kernels of the gated recurrence share: a call's arguments and a token's terms.
#pragma once

#include "common.cuh"
#include "pair.cuh"

namespace mb2 {
namespace rec {

// Two channels at a time: packed fp32 pairs (pair.cuh).
__device__ __forceinline__ float lo(uint64_t v) { return __uint_as_float(lo_of(v)); }
__device__ __forceinline__ float hi(uint64_t v) { return __uint_as_float(hi_of(v)); }
__device__ __forceinline__ uint64_t pack(float a, float b) {
    return pair(__float_as_uint(a), __float_as_uint(b));
}

__device__ __forceinline__ float rcp(float v) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float rsq(float v) {
    float r;
    asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {      // a NaN stays
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// log2 of a at an open gate: -sharpness softplus(decay) / ln 2
__device__ __forceinline__ float log2_decay(float decay, float sharpness) {
    return -sharpness * (fmaxf(decay, 0.0f) + log1pf(expf(-fabsf(decay)))) * kLog2e;
}

// Factors of the packed arithmetic, which takes no immediates.
struct Factors {
    uint64_t neg_log2e, one, neg_one, c[6];
    static constexpr int N = 9;
    static constexpr float kLog = -kLog2e;
    __device__ __forceinline__ static float value(int i) {
        constexpr float v[N] = {kLog, 1.0f, -1.0f, -0.6931471824645996f, -0.24022649228572845f,
                                -0.05550357326865196f, -0.009618237614631653f,
                                -0.0013390850508585572f, -0.00015403512225020677f};
        return v[i];
    }
    __device__ __forceinline__ static Factors set() {
        Factors f;
        uint64_t *to = &f.neg_log2e;
#pragma unroll
        for (int i = 0; i < N; ++i) to[i] = pair(value(i));
        return f;
    }
};

// e^-v
__device__ __forceinline__ uint64_t exp_neg(uint64_t v, const Factors &k) {
    const uint64_t t = mul2(v, k.neg_log2e);
    return pack(ex2(lo(t)), ex2(hi(t)));
}
// 1 + e^-v; its reciprocal is sigmoid(v), exactly 0 at v = -inf
__device__ __forceinline__ uint64_t one_plus_exp(uint64_t v, const Factors &k) {
    return add2(exp_neg(v, k), k.one);
}
__device__ __forceinline__ uint64_t rcp2(uint64_t v) { return pack(rcp(lo(v)), rcp(hi(v))); }
// 1 - sigmoid(v) = e^-v sigmoid(v) from both, to its own few units: sigmoid(v) taken from 1
// would leave its rounding, 2^-24, where v is high.  0 where sigmoid(v) is.
__device__ __forceinline__ uint64_t rest_of(uint64_t exp_neg_v, uint64_t sigmoid) {
    constexpr float kMost = 8.507059173023462e37f;    // 2^126: infinity times 0 is not wanted
    return mul2(pack(fminf(lo(exp_neg_v), kMost), fminf(hi(exp_neg_v), kMost)), sigmoid);
}

// a = 2^u and 1 - a^2 for u <= 0, both to within a few units of their own: near u = 0,
// where layers start, 1 - a^2 from a rounded a would lose what a's last bit is worth
// (2^-24 of 1e-3), and an exponential whose errors lean to one side would add them up
// over the 1 / (1 - a) tokens that a state remembers.
//   n = rint(u), f = u - n (exact), q = 1 - 2^f = f P(f)
//   (P: degree 5, fitted in 64 bits by relative error, 2.1e-8 on |f| <= 1/2),
//   1 - a = 2^n q + (1 - 2^n),  a = 2^n - 2^n q,  1 - a^2 = (1 - a) + (1 - a) a.
// MILD: u >= -1/2, so that n = 0.  On the FMA pipe alone: the MUFU has four other
// operations a token.  u below -126 counts as -126 (a = 1.2e-38); a NaN stays.
struct Decay {
    uint64_t a, y;
};
template <bool MILD> __device__ __forceinline__ Decay decay_of(uint64_t u, const Factors &k) {
    uint64_t f = u, s = 0;
    if constexpr (!MILD) {
        constexpr float kRound = 12582912.0f;         // 1.5 * 2^23: leaves rint(u) in the low bits
        u = pack(max_nan(lo(u), -126.0f), max_nan(hi(u), -126.0f));
        const uint64_t t = add2(u, pair(kRound));
        f = fma2(add2(t, pair(-kRound)), k.neg_one, u);
        constexpr uint32_t kOne = 127u << 23;
        s = pair(lo_of(t) * (1u << 23) + kOne, hi_of(t) * (1u << 23) + kOne);   // 2^n
    }
    uint64_t p = fma2(f, k.c[5], k.c[4]);
    p = fma2(p, f, k.c[3]);
    p = fma2(p, f, k.c[2]);
    p = fma2(p, f, k.c[1]);
    p = fma2(p, f, k.c[0]);
    uint64_t less = mul2(p, f);                       // 1 - a
    Decay d;
    if constexpr (MILD) {
        d.a = fma2(less, k.neg_one, k.one);
    } else {
        d.a = fma2(mul2(s, k.neg_one), less, s);
        less = fma2(s, less, fma2(s, k.neg_one, k.one));
    }
    d.y = fma2(less, d.a, less);
    return d;
}
// whether no channel of the warp can leave MILD's range, whatever its gate (0 < r <= 1)
__device__ __forceinline__ bool mild(uint64_t log2a) {
    return __all_sync(0xffffffffu, lo(log2a) >= -0.5f && hi(log2a) >= -0.5f);
}

constexpr float kTiny = 7.52316384526264e-37f;        // 2^-120
constexpr float kFloor = 7.888609052210118e-31f;      // 2^-100, nothing beside kTiny's root

// sqrt(y) / d for y = 1 - a^2 and d = 1 + e^-v, v the input gate: one rsqrt for the root and
// the sigmoid.  For d up to kFar (v above -43.6), beyond which y d^2 may be infinite and the
// result 0; where d itself is infinite (v below -88.7) 0 is what it should be.  0 at y = 0 (a
// closed decay gate).
constexpr float kFar = 9.223372036854775808e18f;      // 2^63, 0x5f000000
__device__ __forceinline__ uint64_t near_input_factor(uint64_t y, uint64_t d) {
    const uint64_t w = mul2(pack(fmaxf(lo(y), kTiny), fmaxf(hi(y), kTiny)), mul2(d, d));
    return mul2(y, pack(rsq(lo(w)), rsq(hi(w))));
}
// The same for all d: 0 where 1 / d is below the normal numbers (v below -87).  A value's
// bits are near_input_factor's wherever that holds, whatever the value beside it.
__device__ __forceinline__ uint64_t input_factor(uint64_t y, uint64_t d) {
    uint64_t f = near_input_factor(y, d);
    if (lo(d) > kFar || hi(d) > kFar) {
        const uint64_t m = mul2(y, pack(rsq(fmaxf(lo(y), kTiny)), rsq(fmaxf(hi(y), kTiny))));
        const uint64_t far = mul2(m, rcp2(d));
        f = pack(lo(d) > kFar ? lo(far) : lo(f), hi(d) > kFar ? hi(far) : hi(f));
    }
    return f;
}
struct Args {
    const void *x, *ig, *rg;
    const float *decay;
    float sharpness;
    int64_t xs[2], is[2], rs[2];              // batch and token strides
    const float *h0;
    const int32_t *cu;
    int64_t batch, seqlen, width, seqs;
    void *h;
    float *h_last, *saved;
    const void *dh;
    int64_t ds[2];
    const float *dlast;
    void *dx, *dig, *drg;
    float *ddecay, *dh0;
};

}  // namespace rec
}  // namespace mb2
