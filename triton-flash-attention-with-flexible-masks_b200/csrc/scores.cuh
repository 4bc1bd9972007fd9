// What attention_scored does to a score between Q K^T and the softmax, in the log2 domain that the tensor-core kernels work in:
//   y_ij = log2(e) * (cap * tanh(s_ij * sm_scale / cap) - slope_h * |i + gap - j|)
// without a cap y = log2(e) * (s * sm_scale - ...). The gradient through the cap is the factor 1 - tanh^2 = 1 - (y before the bias / A)^2,
// A = cap * log2(e).
//
// tanh: where a warp's scores are all at most `cap` (after the scale), x * (an even polynomial of x), fitted by interpolation of
// tanh(x) / x over x^2 in [0, 1] at Chebyshev's points; relative error 7.3e-7. That is eight packed FMAs for two scores and no
// special-function unit, which the exponentials keep busy. Elsewhere 1 - 2 / (1 + e^2x), whose absolute error of some 2^-23 is relative to a
// tanh of at least 0.76 in one of them. Close to 0 the second form would lose the small scores of a large cap.
#pragma once
#include "common.cuh"

namespace fa {

struct ScoreArgs {
    const float* slopes;  // [H], null: none
    float cap;            // 0: none
    int on;               // any of cap, slopes and the mask's prefix is given
    float k;              // sm_scale / cap
    float k2e;            // 2 log2(e) k
    float a;              // cap log2(e)
    float inv_a;
    float most;           // |s| up to which tanh is the polynomial: 1 / k
};

constexpr float kScoreLog2e = 1.4426950408889634f;

inline ScoreArgs make_score_args(float cap, const float* slopes, bool prefix, float sm_scale) {
    ScoreArgs s{};
    s.slopes = slopes;
    s.cap = cap;
    s.on = cap > 0.f || slopes || prefix;
    if (cap > 0.f) {
        s.k = sm_scale / cap;
        s.k2e = 2.f * kScoreLog2e * s.k;
        s.a = cap * kScoreLog2e;
        s.inv_a = 1.f / s.a;
        s.most = 1.f / s.k;
    }
    return s;
}

// tanh(x) = x (c0 + c1 x^2 + ... + c5 x^10) for |x| <= 1
__device__ constexpr float kTanhPoly[6] = {0.999999395f, -0.333289514f, 0.132807206f, -0.0515859884f, 0.0167208552f, -0.00305822904f};

__device__ __forceinline__ float fast_rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Does any of a warp's scores (N a thread) ask for the second form?
template <int N>
__device__ __forceinline__ bool any_beyond(const float* v, float most) {
    float m0 = 0.f, m1 = 0.f;
#pragma unroll
    for (int x = 0; x < N; x += 4) {
        m0 = max3(m0, fabsf(v[x]), fabsf(v[x + 1]));
        m1 = max3(m1, fabsf(v[x + 2]), fabsf(v[x + 3]));
    }
    return __any_sync(0xffffffffu, fmaxf(m0, m1) > most);
}

// log2(e) cap tanh(s sm_scale / cap) of two scores
__device__ __forceinline__ uint64_t cap_small(uint64_t s2, const ScoreArgs& a) {
    const uint64_t x2 = mul_f2(s2, pack_f2(a.k, a.k)), u2 = mul_f2(x2, x2);
    uint64_t t = pack_f2(kTanhPoly[5], kTanhPoly[5]);
#pragma unroll
    for (int i = 4; i >= 0; --i) t = fma_f2(t, u2, pack_f2(kTanhPoly[i], kTanhPoly[i]));
    return mul_f2(mul_f2(x2, pack_f2(a.a, a.a)), t);
}
__device__ __forceinline__ float cap_any(float s, const ScoreArgs& a) {
    return fmaf(-2.f * a.a, fast_rcp(1.f + fast_exp2(s * a.k2e)), a.a);
}
__device__ __forceinline__ uint64_t cap_pair(uint64_t s2, const ScoreArgs& a, bool beyond) {
    if (!beyond) return cap_small(s2, a);
    float s0, s1;
    unpack_f2(s2, s0, s1);
    return pack_f2(cap_any(s0, a), cap_any(s1, a));
}
// 1 - tanh^2 of two capped scores
__device__ __forceinline__ uint64_t cap_slope(uint64_t y2, const ScoreArgs& a) {
    const uint64_t t2 = mul_f2(y2, pack_f2(a.inv_a, a.inv_a));
    float t0, t1;
    unpack_f2(t2, t0, t1);
    return fma_f2(t2, pack_f2(-t0, -t1), pack_f2(1.f, 1.f));
}

// The bias of the entries of one tile. The distance i + gap - j of an entry that the masks keep has one sign over most tiles (with a causal
// mask and no prefix over all): there the bias is linear in it, elsewhere the distance's size is taken.
struct Bias {
    float s;    // -log2(e) slope, or +: of tiles whose keys all lie ahead; 0: no bias
    bool both;  // both signs occur
    // least and most: distances of the tile's corners. slope: log2(e) times the head's
    __device__ __forceinline__ Bias(float slope, bool never_ahead, int least, int most) {
        both = slope != 0.f && !never_ahead && least < 0 && most > 0;
        s = !never_ahead && !both && least < 0 ? slope : -slope;
    }
    // of distances d + x and d + x + step (x and step known to the compiler); sd = s * d
    __device__ __forceinline__ uint64_t pair(float d, float sd, float x, float step) const {
        if (both) return pack_f2(s * fabsf(d + x), s * fabsf(d + (x + step)));
        return pack_f2(fmaf(s, x, sd), fmaf(s, x + step, sd));
    }
};

// 32 neighbouring scores of one row, in place, to the log2 domain; d: distance of the first one
__device__ __forceinline__ void score_row(float* v, const ScoreArgs& a, const Bias& bias, float c, int dist) {
    const float d = float(dist), sd = bias.s * d;
    if (a.cap > 0.f) {
        if (!any_beyond<32>(v, a.most)) {
#pragma unroll
            for (int x = 0; x < 32; x += 2) unpack_f2(cap_small(pack_f2(v[x], v[x + 1]), a), v[x], v[x + 1]);
        } else {
#pragma unroll
            for (int x = 0; x < 32; ++x) v[x] = cap_any(v[x], a);
        }
    } else {
#pragma unroll
        for (int x = 0; x < 32; x += 2) unpack_f2(mul_f2(pack_f2(v[x], v[x + 1]), pack_f2(c, c)), v[x], v[x + 1]);
    }
    if (bias.s != 0.f) {
#pragma unroll
        for (int x = 0; x < 32; x += 2) unpack_f2(add_f2(pack_f2(v[x], v[x + 1]), bias.pair(d, sd, float(-x), -1.f)), v[x], v[x + 1]);
    }
}

}  // namespace fa
