// mg_attention_math.cuh -- arithmetic of the attention and rotary kernels:
// exponentials, pairs of fp32 operations, maxima, the capped score's tanh.
#pragma once

#include "mg_attention_common.cuh"

namespace mg {

constexpr float kLog2e = 1.44269504088896341f;
constexpr float kLn2 = 0.693147180559945309f;

__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp(float x)
{
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The largest of three, and of three magnitudes (NaN where all are, or is skipped).
__device__ __forceinline__ float max3(float a, float b, float c)
{
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float max3_abs(float a, float b, float c)
{
    float r;
    asm("max.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// The largest of N values (of their magnitudes): four chains, two values a step.
template <int N, bool kAbs>
__device__ __forceinline__ float max_of(const float (&s)[N])
{
    float t[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) t[i] = kAbs ? fabsf(s[i]) : s[i];
#pragma unroll
    for (int i = 4; i + 8 <= N; i += 8)
#pragma unroll
        for (int k = 0; k < 4; ++k)
            t[k] = kAbs ? max3_abs(t[k], s[i + 2 * k], s[i + 2 * k + 1]) : max3(t[k], s[i + 2 * k], s[i + 2 * k + 1]);
#pragma unroll
    for (int k = 0; k < 4; ++k)      // N is a multiple of 8: four are left
        t[k] = kAbs ? fmaxf(t[k], fabsf(s[N - 4 + k])) : fmaxf(t[k], s[N - 4 + k]);
    return fmaxf(max3(t[0], t[1], t[2]), t[3]);
}

// Two fp32 operations in one instruction.
__device__ __forceinline__ uint64_t pack2(float a, float b)
{
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpack2(uint64_t r, float& a, float& b)
{
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(r));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c)
{
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b)
{
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b)
{
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint32_t bf16x2(float lo, float hi)
{
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// tanh(x) for |x| <= 1: x times a polynomial in x^2 (least maximum of the
// relative error over [0, 1], fitted by reweighted least squares: 1.4e-7 with
// its fp32 evaluation), two values at a time.
__device__ __forceinline__ uint64_t tanh_small2(uint64_t x)
{
    const uint64_t u = mul2(x, x);
    uint64_t r = pack2(0.001041021547280252f, 0.001041021547280252f);
    r = fma2(r, u, pack2(-0.00620337575674057f, -0.00620337575674057f));
    r = fma2(r, u, pack2(0.02028997614979744f, 0.02028997614979744f));
    r = fma2(r, u, pack2(-0.05345702916383743f, -0.05345702916383743f));
    r = fma2(r, u, pack2(0.13325203955173492f, 0.13325203955173492f));
    r = fma2(r, u, pack2(-0.33332839608192444f, -0.33332839608192444f));
    r = fma2(r, u, pack2(0.9999999403953552f, 0.9999999403953552f));
    return mul2(r, x);
}
// tanh(x) for any x: 1 - 2 / (1 + exp(2x)); its error is absolute, some 2^-23.
__device__ __forceinline__ float tanh_any(float x) { return fmaf(-2.f, rcp(1.f + ex2(x * (2.f * kLog2e))), 1.f); }

__device__ __forceinline__ float tanh_fast(float x)
{
    float small, other;
    unpack2(tanh_small2(pack2(x, x)), small, other);
    return fabsf(x) <= 1.f ? small : tanh_any(x);
}

// tanh(x) for |x| <= 1/2 with four terms (fitted as above: 6e-7), from the
// unscaled score: x = s * pre, tc[k] = pre^(2k + 1) times the coefficient.
struct CapCurve {
    float tc[4];
    float bound;        // |s| up to this: |x| <= 1/2; 0 where a coefficient would leave fp32's range
    float pre;          // |scale| / cap
};

// s[i] <- tanh(s[i] * pre). What bounds this is the fp32 pipe: the four-term form
// is 5 operations a score, where the warp's scores are all below half the cap
// (the usual case); with scores up to the cap it is 9, and beyond it an
// exponential and a reciprocal.
template <int N>
__device__ __forceinline__ void cap_scores(float (&s)[N], const CapCurve& cc)
{
    const float top = max_of<N, true>(s);
    if (!__any_sync(~0u, !(top <= cc.bound))) {
        const uint64_t c0 = pack2(cc.tc[0], cc.tc[0]), c1 = pack2(cc.tc[1], cc.tc[1]), c2 = pack2(cc.tc[2], cc.tc[2]),
                       c3 = pack2(cc.tc[3], cc.tc[3]);
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const uint64_t x = pack2(s[i], s[i + 1]), u = mul2(x, x);
            unpack2(mul2(x, fma2(u, fma2(u, fma2(u, c3, c2), c1), c0)), s[i], s[i + 1]);
        }
    } else if (!__any_sync(~0u, !(top * cc.pre <= 1.f))) {
        const uint64_t a = pack2(cc.pre, cc.pre);
#pragma unroll
        for (int i = 0; i < N; i += 2) unpack2(tanh_small2(mul2(a, pack2(s[i], s[i + 1]))), s[i], s[i + 1]);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) s[i] = tanh_any(s[i] * cc.pre);
    }
}

}  // namespace mg
