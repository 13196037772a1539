// mg_attention_common.cuh -- what the attention kernels share: parameters, the
// rule which keys a query sees, and the score's curve.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math_constants.h>
#include <stdint.h>

namespace mg {

struct AttnParams {
    int B, H, Hkv, Lq, Lk, D;
    int causal;
    float scale, cap;
    int64_t qs[3], ks[3], vs[3], os[3];          // batch, head, row
    int64_t dos[3], dqs[3], dks[3], dvs[3];
    const float* slopes;
    const int32_t* docs;
    const int32_t* prefix;
    const void *q, *k, *v, *dout;
    void *out, *dq, *dk, *dv;
    float* lse;
    float* delta;
    float* fine;                                 // log of each row's sum of exp(s - lse): what lse is short of
};

// A row of keys shared by several blocks of the forward kernels, where there are
// too few queries to fill the GPU: each leaves its part's out, and the maximum and the sum that
// it is taken against, in fp32. (From the parts' lse, their weights would carry its rounding, 2^-24 |lse|.)
struct RowParts {
    int parts;           // 1: the block writes out and lse itself
    float* out;          // [parts][B * H][Lq][D]
    float2* stat;        // [parts][B * H][Lq] (m, l): lse = (m + log2 l) ln 2
};

// A gradient's sum over the streamed rows, shared by several blocks.
struct GradParts {
    int parts;           // 1: the block writes the gradient itself
    float* acc;          // [parts][B * heads][rows][D] of dQ, or of dK
    float* other;        // as acc: of the correction's product (dQ of 16-bit tensors), or of dV
    float* r;            // [parts][B * H][Lq] the rows' sums (dQ): of P * (dP - delta) of 16-bit tensors, of P of fp32
};

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// Position of query i, and its document id: -1 for a query that has none.
__device__ __forceinline__ int query_pos(const AttnParams& p, int i) { return i + p.Lk - p.Lq; }

__device__ __forceinline__ int doc_at(const AttnParams& p, int b, int pos)
{
    return pos >= 0 && pos < p.Lk ? __ldg(p.docs + (int64_t)b * p.Lk + pos) : -1;
}

// Whether the query at position qpos (document qdoc) sees key j (document kdoc).
__device__ __forceinline__ bool sees(const AttnParams& p, int qpos, int qdoc, int j, int kdoc, int prefix)
{
    return (!p.causal || j <= qpos || j < prefix) && (p.docs == nullptr || (qdoc >= 0 && qdoc == kdoc));
}

// The score of one pair from the scaled product t: capped and biased. `bend`
// receives tanh(t / cap) (0 without a cap).
__device__ __forceinline__ float score(float t, float cap, float slope, int dist, float& bend)
{
    bend = 0.f;
    if (cap > 0.f) {
        bend = tanhf(t / cap);
        t = cap * bend;
    }
    return t - slope * (float)(dist < 0 ? -dist : dist);
}

}  // namespace mg
