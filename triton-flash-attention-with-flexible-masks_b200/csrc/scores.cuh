// What attention_scored does to a score between Q K^T and the softmax, in the log2 domain that the tensor-core kernels work in:
//   y_ij = log2(e) * (cap * tanh(s_ij * sm_scale / cap) - slope_h * |i + gap - j|)
// without a cap y = log2(e) * (s * sm_scale - ...). The gradient through the cap is the factor 1 - tanh^2 = 1 - (y before the bias / a)^2,
// a = cap * log2(e).
//
// The capped score is s * (an even polynomial of s) where all of a warp's are at most 0.9 cap: tanh(x) / x over x^2 in [0, 0.81] by interpolation at
// Chebyshev's points, with a and sm_scale / cap multiplied into its coefficients. Its relative error, 2.9e-6, is up to a cap of 64 1.4e-4 of an exponential, a quarter of the rounding of P to
// fp16; for larger caps, whose scores may be hundreds or thousands, it is interpolated up to 0.75 cap (5.8e-7) or 0.6 cap (7.4e-8) instead, for scores beyond that take the other form: forward of
// 16 x 4096 x 128 causal, greatest score 0.85 cap, interpolated up to 0.9 | 0.75 | 0.6 cap 90 | 93 | 136 us. That is six packed FMAs for two
// scores and nothing of the special-function unit, which the exponentials keep busy. Beyond, a score is a - 2 a / (1 + 2^(2 log2(e) x)), whose absolute error
// is some 2^-22 of a: close to 0 that form would lose the small scores of a large cap, so that a warp with a score beyond the polynomial works out both forms and takes each score's own.
//
// What bounds it: what two softmax warps a scheduler get through of a tile's straight code (no unit is full: issue slots 46 %, MUFU 40, tensor pipe 40 with a cap), so that each
// instruction shows: 2 x 16 x 4096 x 128 causal, capped | biased, 80 | 71 million instructions, issue slots 46 | 47 %.
// Forward of 32 / 8 heads x 5801 x 128 causal, unchanged, capped, biased, both: 259, 330, 298, 399 us; kernels of a step of 16 x 8111 x 128 in documents, us,
// forward 112, 164, 130, 178, dK/dV 178, 222, 194, 242, dQ 138, 177, 146, 198.
// Tried and taken back (the same forward, cap 50 | cap 20, which at deviation 4 goes through both forms now and then; now 330 | 463): five terms for 7.1e-7 up to 0.75 cap 325 | 682; six up
// to the cap 352 | 378; a quotient of polynomials of degree 2, up to 2.5 caps, with one reciprocal for two scores 426 | 418; eight terms up to 1.4 cap as a second unrolled
// form 358 | 528 (registers); the cap of the next 16 scores in front of the exponentials of these, as the source goes, 328 | -. The bias as one more product of 16 columns on the tensor cores (slope and position in three 16-bit parts): the biased forward 277 for 298, but 8 ragged
// sequences over a paged cache 222 for 218 and an encoder's step 136 for 134, for a quarter more code.
#pragma once
#include "common.cuh"

namespace fa {

// Instances of the attention kernels
enum : int {
    SCORE_PLAIN = 0,   // attention
    SCORE_BIAS = 1,    // a bias, and perhaps a prefix
    SCORE_CAPPED = 2,  // a cap, and perhaps a prefix
    SCORE_CAPPED_BIAS = SCORE_BIAS | SCORE_CAPPED,
    SCORE_PREFIX = 4,  // a prefix alone: the scores are attention's
    // A window, and perhaps a prefix, with or without the changes above. What it costs is that tiles at both ends
    // of a window, and those of the first keys, take as long as whole ones: 2 x 16 / 4 heads x 4000 x 128, bf16, forward |
    // forward and backward, us, long series of calls under the power cap, causal 138 | 580; window 1024 81 | 337, with 4
    // first keys 87 | 368; window 2048 with 4 first keys 123 | 513.
    SCORE_WINDOW = 8,
};
// Does an instance change the scores?
__host__ __device__ constexpr bool score_changed(int kind) { return (kind & SCORE_CAPPED_BIAS) != 0; }

constexpr int kTanhTerms = 5;

struct ScoreArgs {
    const float* slopes;  // [H], null: none
    float cap;            // 0: none
    int kind;             // SCORE_*
    float poly[kTanhTerms];  // capped score = s (poly[0] + poly[1] s^2 + ...) up to |s| = most
    float most;
    float k2e;            // 2 log2(e) sm_scale / cap
    float k;              // sm_scale / cap
    float a;              // cap log2(e)
    float minus_inv_a2;   // -1 / a^2
};

constexpr float kScoreLog2e = 1.4426950408889634f;

inline ScoreArgs make_score_args(float cap, const float* slopes, bool prefix, float sm_scale, bool window = false) {
    // tanh(x) / x up to x = kUpTo: the widest that is off by less than 1.5e-4 of an exponential at the greatest score
    constexpr double kUpTo[3] = {0.9, 0.75, 0.6};
    constexpr double kTanh[3][kTanhTerms] = {{0.999997105, -0.333153478, 0.131495683, -0.0471230871, 0.010487992},   // 2.9e-6 of the value
                                             {0.999999424, -0.333281921, 0.132584621, -0.0500416086, 0.0129166518},  // 5.8e-7
                                             {0.999999926, -0.33332302, 0.133100644, -0.0520966534, 0.0154687513}};  // 7.4e-8
    // largest x at which the terms from x^(2i) on are below 2e-7 of the sum
    constexpr double kWithout[kTanhTerms] = {0.0, 7.3e-4, 0.0349, 0.125, 0.241};
    const int fit = cap <= 64.f ? 0 : cap <= 320.f ? 1 : 2;
    ScoreArgs s{};
    s.slopes = slopes;
    s.cap = cap;
    s.kind = (cap > 0.f ? SCORE_CAPPED : SCORE_PLAIN) | (slopes ? SCORE_BIAS : SCORE_PLAIN);
    if (window) s.kind |= SCORE_WINDOW;
    if (prefix && s.kind == SCORE_PLAIN) s.kind = SCORE_PREFIX;
    if (cap > 0.f) {
        const double a = double(cap) * 1.4426950408889634, k = double(sm_scale) / cap;
        double power = a * k, most = kUpTo[fit];
        for (int i = 0; i < kTanhTerms; ++i, power *= k * k) {
            const double c = kTanh[fit][i] * power, size = c < 0 ? -c : c;
            // a coefficient that fp32 cannot hold is left out, with the scores that need it
            if (i > 0 && !(size > 1e-37 && size < 1e37)) most = most < kWithout[i] ? most : kWithout[i];
            else s.poly[i] = float(c);
        }
        s.most = float(most / k < 1e38 ? most / k : 1e38);
        s.k = float(k < 1e37 ? k : 1e37);
        s.k2e = float(2.885390081777927 * k < 1e38 ? 2.885390081777927 * k : 1e38);
        s.a = float(a);
        s.minus_inv_a2 = float(-1.0 / (a * a));
    }
    return s;
}

__device__ __forceinline__ float fast_rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Does any of a warp's scores (N a thread) lie beyond the polynomial?
template <int N>
__device__ __forceinline__ bool any_beyond(const float* v, float most) {
    float m[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int x = 0; x < N; x += 8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) m[i] = max3(m[i], fabsf(v[x + 2 * i]), fabsf(v[x + 2 * i + 1]));
    }
    return __any_sync(0xffffffffu, fmaxf(max3(m[0], m[1], m[2]), m[3]) > most);
}

// poly[0] + poly[1] s^2 + ... of two scores
__device__ __forceinline__ uint64_t cap_poly(uint64_t s2, const ScoreArgs& a) {
    const uint64_t u2 = mul_f2(s2, s2);
    uint64_t t = pack_f2(a.poly[kTanhTerms - 1], a.poly[kTanhTerms - 1]);
#pragma unroll
    for (int i = kTanhTerms - 2; i >= 0; --i) t = fma_f2(t, u2, pack_f2(a.poly[i], a.poly[i]));
    return t;
}
// the capped score of one that the polynomial covers: the bits of its place in a pair
__device__ __forceinline__ float cap_one(float s, const ScoreArgs& a) {
    const float u = __fmul_rn(s, s);
    float t = a.poly[kTanhTerms - 1];
#pragma unroll
    for (int i = kTanhTerms - 2; i >= 0; --i) t = fmaf(t, u, a.poly[i]);
    return __fmul_rn(s, t);
}
// two capped scores, whatever their size, with b2 added to them: each by the form that is exact for it (the other one's error goes by the cap), and one that the polynomial
// covers to the bits that it has in a warp without any that it does not. So a score beyond it, perhaps one that a mask hides, is nothing to its neighbours.
__device__ __forceinline__ uint64_t cap_any(uint64_t s2, uint64_t b2, const ScoreArgs& a) {
    float s0, s1, x0, x1, p0, p1;
    unpack_f2(s2, s0, s1);
    unpack_f2(mul_f2(s2, pack_f2(a.k2e, a.k2e)), x0, x1);
    unpack_f2(add_f2(pack_f2(fast_exp2(x0), fast_exp2(x1)), pack_f2(1.f, 1.f)), x0, x1);
    unpack_f2(add_f2(fma_f2(pack_f2(fast_rcp(x0), fast_rcp(x1)), pack_f2(-2.f * a.a, -2.f * a.a), pack_f2(a.a, a.a)), b2), x0, x1);
    unpack_f2(fma_f2(s2, cap_poly(s2, a), b2), p0, p1);
    return pack_f2(fabsf(s0) <= a.most ? p0 : x0, fabsf(s1) <= a.most ? p1 : x1);
}
// 1 - tanh^2 of two capped scores
__device__ __forceinline__ uint64_t cap_slope(uint64_t y2, const ScoreArgs& a) {
    return fma_f2(mul_f2(y2, y2), pack_f2(a.minus_inv_a2, a.minus_inv_a2), pack_f2(1.f, 1.f));
}

// The bias of the entries of one tile. The distance i + gap - j of an entry that the masks keep has one sign over most tiles (with a causal
// mask and no prefix over all): there the bias is linear in it, elsewhere the distance's size is taken.
struct Bias {
    float s;     // -log2(e) slope, or +: of tiles whose keys all lie ahead; 0: no bias
    float line;  // the same where the bias is linear, 0 where both signs occur
    bool both;
    // least and most: distances of the tile's corners. slope: log2(e) times the head's
    __device__ __forceinline__ Bias(float slope, bool never_ahead, int least, int most) {
        both = slope != 0.f && !never_ahead && least < 0 && most > 0;
        s = !never_ahead && !both && least < 0 ? slope : -slope;
        line = both ? 0.f : s;
    }
};

// What a tile's biased scores are computed relative to: the row's running reference point, `run`, but where the bias of the tile's middle, at distance `mid`, is far from it, that bias. (After
// a sequence's first keys, or the beginning of a scattered document, come keys whose biases are thousands away: relative to the old point each step along the row would round at that size.
// bf16, 30000 keys, window 100, slopes up to 0.84: rows off by 3.6 times what P's rounding allows.) The caller moves the scores by the two points' distance when it knows their maximum. What it
// costs where no tile is far: steps of 16 x 8 heads x 577 x 32 without a causal mask 130.0 -> 130.9 us, of 16 heads x 8111 x 128 in documents, capped, 702 -> 708.
constexpr float kFarReference = 256.f;
__device__ __forceinline__ float tile_reference(const Bias& bias, float run, int mid) {
    const float own = bias.line * float(mid);
    return bias.s != 0.f && fabsf(own - run) > kFarReference && fabsf(own) < INFINITY ? own : run;
}

// v[x] = f(v[x], x) for the N values of a thread, kStep at a time, in a loop that moves them all on: for what is rarely done. Unrolled, it would be most of the
// code of the softmax warps, which is fetched again and again.
template <int N, int kStep, class F>
__device__ __forceinline__ void rolled(float* v, F f) {
#pragma unroll 1
    for (int x0 = 0; x0 < N; x0 += kStep) {
        float first[kStep];
#pragma unroll
        for (int x = 0; x < kStep; ++x) first[x] = f(v[x], x0 + x);
#pragma unroll
        for (int x = 0; x + kStep < N; ++x) v[x] = v[x + kStep];
#pragma unroll
        for (int x = 0; x < kStep; ++x) v[N - kStep + x] = first[x];
    }
}
// The same two at a time: f(values, x0, x) for those of x0 + x, x0 a multiple of kStep.
template <int N, int kStep, class F>
__device__ __forceinline__ void rolled_pairs(float* v, F f) {
#pragma unroll 1
    for (int x0 = 0; x0 < N; x0 += kStep) {
        float first[kStep];
#pragma unroll
        for (int x = 0; x < kStep; x += 2) unpack_f2(f(pack_f2(v[x], v[x + 1]), x0, x), first[x], first[x + 1]);
#pragma unroll
        for (int x = 0; x + kStep < N; ++x) v[x] = v[x + kStep];
#pragma unroll
        for (int x = 0; x < kStep; ++x) v[N - kStep + x] = first[x];
    }
}

// N neighbouring scores of one row (a multiple of 32), in place, to the log2 domain, less `ref`; dist: distance of the first one. real: the row is a
// query's (what lies in other rows of the tile must not tell the warp which form of the tanh to take, and so the last bits).
template <int KIND, int N>
__device__ __forceinline__ void score_row(float* v, const ScoreArgs& a, const Bias& bias, float c, int dist, bool real, float ref) {
    constexpr bool kCapped = (KIND & SCORE_CAPPED) != 0, kBias = (KIND & SCORE_BIAS) != 0;
    constexpr int kStep = kBias ? 16 : 32;  // (with a bias 32 do not fit the registers)
    const bool beyond = kCapped && any_beyond<N>(v, real ? a.most : INFINITY);
    if (KIND == SCORE_BIAS && bias.both) {  // (in front of what follows it costs the other tiles less)
        const float d = float(dist), e = bias.s / c;
        rolled<N, kStep>(v, [&](float y, int x) { return fmaf(e, fabsf(d - float(x)), y); });
    }
    auto each = [&](auto score) {  // score(two scores, what is added to them)
#pragma unroll
        for (int q = 0; q < N; q += 32) {
            uint64_t b2 = pack_f2(-ref, -ref);
            if constexpr (kBias) {
                const float d = float(dist - q);
                b2 = pack_f2(fmaf(bias.line, d, -ref), fmaf(bias.line, d - 1.f, -ref));
            }
#pragma unroll
            for (int x = q; x < q + 32; x += 2) {
                unpack_f2(score(pack_f2(v[x], v[x + 1]), b2), v[x], v[x + 1]);
                if (kBias && x + 2 < q + 32) b2 = add_f2(b2, pack_f2(-2.f * bias.line, -2.f * bias.line));
            }
        }
    };
    if constexpr (kCapped) {
        if (N == kBlk && !kBias && !beyond) {
            rolled_pairs<N, kStep>(v, [&](uint64_t s2, int, int) { return fma_f2(s2, cap_poly(s2, a), pack_f2(-ref, -ref)); });  // (a tile with a mask: the others are capped elsewhere)
        } else if (beyond) {
            // 16 at a time: with 32 the registers do not do, with 8 a call of 16 x 4096 x 128 most of whose tiles go this way takes 224 us for 179
            uint64_t b2 = pack_f2(-ref, -ref);
            rolled_pairs<N, 16>(v, [&](uint64_t s2, int x0, int x) {
                if (kBias && x == 0 && x0 % 32 == 0) {  // (as in `each`)
                    const float d = float(dist - x0);
                    b2 = pack_f2(fmaf(bias.line, d, -ref), fmaf(bias.line, d - 1.f, -ref));
                }
                const uint64_t y2 = cap_any(s2, b2, a);
                if constexpr (kBias) b2 = add_f2(b2, pack_f2(-2.f * bias.line, -2.f * bias.line));
                return y2;
            });
        } else {
            each([&](uint64_t s2, uint64_t b2) { return fma_f2(s2, cap_poly(s2, a), b2); });
        }
    } else {
        each([&](uint64_t s2, uint64_t b2) { return fma_f2(s2, pack_f2(c, c), b2); });
    }
    if (KIND == SCORE_CAPPED_BIAS && bias.both) {
        const float d = float(dist);
        rolled<N, kStep>(v, [&](float y, int x) { return fmaf(bias.s, fabsf(d - float(x)), y); });
    }
}

// The same as above without bias and reference: scores to capped scores, for the backward kernels.
template <int N>
__device__ __forceinline__ void cap_scores(float* v, const ScoreArgs& a) {
    // (both in straight code: with the rare one in a loop of 16 at a time dQ of 16 x 4096 x 128 causal, none of whose scores is beyond, takes 127 us for 120)
    if (any_beyond<N>(v, a.most)) {
#pragma unroll
        for (int x = 0; x < N; x += 2) unpack_f2(cap_any(pack_f2(v[x], v[x + 1]), 0, a), v[x], v[x + 1]);
    } else {
#pragma unroll
        for (int x = 0; x < N; x += 2) {
            const uint64_t s2 = pack_f2(v[x], v[x + 1]);
            unpack_f2(mul_f2(s2, cap_poly(s2, a)), v[x], v[x + 1]);
        }
    }
}

}  // namespace fa
