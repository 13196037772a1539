// mg_attention_simt.cuh -- attention and its gradients in 32-bit arithmetic on
// the CUDA cores, for any head_dim up to 128, any strides and any alignment.
//
// Forward: one block of 256 threads per 32 queries of one head. The block walks
// the keys in tiles of 32 and keeps, per query, the running maximum m, the sum
// l of exp(s - m) and the output accumulator; a tile whose keys raise the
// maximum rescales l and the accumulator by exp(m_old - m_new). Thread (r, c8)
// = (tid / 8, tid % 8) owns query r and the elements c8, c8 + 8, ... of the head,
// so the eight threads of a query share its statistics by shuffles and the
// score of the query against keys c8, c8 + 8, ... is a dot product of two
// shared-memory rows (pitch D + 1: no bank conflicts where D is even; at D = 127 all rows
// begin in one bank). It is the form that takes any call, and it is slow: causal [1, 16 over 4,
// 2048, D], D = 100: 2.6 ms forward, 11.7 ms gradients; D = 127: 8.7 and 45.9 ms; the tensor-core
// kernels at D = 128: 41 and 146 us in bf16, 176 and 1137 us in fp32; 32-bit torch operations 1.3 and 2.8 ms.
// Backward: the same tiles seen from the keys (dK, dV: one block per 32 keys of a
// key-value head, walking the queries of all its query heads in order, so that
// no atomics are needed) and from the queries (dQ).
#pragma once

#include "mg_attention_common.cuh"

namespace mg {

constexpr int kSimtTile = 32;
constexpr int kSimtThreads = 256;
constexpr int kSimtMaxD = 128;

// Loads rows [r0, r0 + 32) of a matrix into shared memory as fp32, zeros beyond
// `rows` and for rows of padding (doc ids at doc[row] < 0).
template <typename T>
__device__ __forceinline__ void simt_load(float* dst, int pitch, const T* src, int64_t stride, int r0, int rows, int D,
                                          const int32_t* doc, int doc_shift)
{
    for (int i = threadIdx.x; i < kSimtTile * D; i += kSimtThreads) {
        const int r = i / D, c = i - r * D, row = r0 + r;
        bool live = row < rows;
        if (live && doc) {
            const int at = row + doc_shift;
            live = at >= 0 && __ldg(doc + at) >= 0;
        }
        dst[r * pitch + c] = live ? to_f32(src[(int64_t)row * stride + c]) : 0.f;
    }
}

__device__ __forceinline__ float simt_dot(const float* a, const float* b, int D)
{
    float s = 0.f;
    for (int d = 0; d < D; ++d) s = fmaf(a[d], b[d], s);
    return s;
}

// First key tile end: keys at or beyond this are seen by no query up to position qmax.
__device__ __forceinline__ int key_end(const AttnParams& p, int qmax, int prefix)
{
    if (!p.causal) return p.Lk;
    const int e = max(qmax + 1, prefix);
    return max(0, min(p.Lk, e));
}

template <typename T>
__global__ void __launch_bounds__(kSimtThreads) attn_simt_forward(const __grid_constant__ AttnParams p)
{
    extern __shared__ float sm[];
    const int pitch = p.D + 1;
    float* Q = sm;
    float* K = Q + kSimtTile * pitch;
    float* V = K + kSimtTile * pitch;
    float* P = V + kSimtTile * pitch;            // [32][33]
    __shared__ int kdoc[kSimtTile];

    const int tiles = (p.Lq + kSimtTile - 1) / kSimtTile, bh = blockIdx.x / tiles;
    const int h = bh % p.H, b = bh / p.H, kv = h / (p.H / p.Hkv);
    const int q0 = (blockIdx.x - bh * tiles) * kSimtTile;
    const int r = threadIdx.x / 8, c8 = threadIdx.x % 8;
    const T* qp = (const T*)p.q + b * p.qs[0] + h * p.qs[1];
    const T* kp = (const T*)p.k + b * p.ks[0] + kv * p.ks[1];
    const T* vp = (const T*)p.v + b * p.vs[0] + kv * p.vs[1];
    const int32_t* docs = p.docs ? p.docs + (int64_t)b * p.Lk : nullptr;
    const int prefix = p.prefix ? __ldg(p.prefix + b) : 0;
    const float slope = p.slopes ? __ldg(p.slopes + h) : 0.f;
    const int qpos = query_pos(p, q0 + r);
    const int qdoc = docs ? doc_at(p, b, qpos) : 0;

    simt_load(Q, pitch, qp, p.qs[2], q0, p.Lq, p.D, docs, p.Lk - p.Lq);
    float acc[kSimtMaxD / 8];
#pragma unroll
    for (int i = 0; i < kSimtMaxD / 8; ++i) acc[i] = 0.f;
    float m = -CUDART_INF_F, l = 0.f;
    const int jend = key_end(p, query_pos(p, min(q0 + kSimtTile, p.Lq) - 1), prefix);
    for (int j0 = 0; j0 < jend; j0 += kSimtTile) {
        __syncthreads();
        simt_load(K, pitch, kp, p.ks[2], j0, p.Lk, p.D, docs, 0);
        simt_load(V, pitch, vp, p.vs[2], j0, p.Lk, p.D, docs, 0);
        if (docs && threadIdx.x < kSimtTile) kdoc[threadIdx.x] = doc_at(p, b, j0 + threadIdx.x);
        __syncthreads();
        float s[4], top = -CUDART_INF_F;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int c = c8 + 8 * i, j = j0 + c;
            float bend;
            s[i] = -CUDART_INF_F;
            if (j < p.Lk && q0 + r < p.Lq && sees(p, qpos, qdoc, j, docs ? kdoc[c] : 0, prefix))
                s[i] = score(p.scale * simt_dot(Q + r * pitch, K + c * pitch, p.D), p.cap, slope, qpos - j, bend);
            top = fmaxf(top, s[i]);
        }
#pragma unroll
        for (int o = 1; o < 8; o *= 2) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
        const float mn = fmaxf(m, top);
        const float base = mn == -CUDART_INF_F ? 0.f : mn;
        const float fix = expf(m - base);      // 0 while nothing has been seen
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float e = expf(s[i] - base);
            P[r * 33 + c8 + 8 * i] = e;
            sum += e;
        }
#pragma unroll
        for (int o = 1; o < 8; o *= 2) sum += __shfl_xor_sync(~0u, sum, o);
        l = l * fix + sum;
        m = mn;
        __syncwarp();
#pragma unroll
        for (int i = 0; i < kSimtMaxD / 8; ++i) {
            const int d = c8 + 8 * i;
            if (d >= p.D) break;
            float a = acc[i] * fix;
            for (int c = 0; c < kSimtTile; ++c) a = fmaf(P[r * 33 + c], V[c * pitch + d], a);
            acc[i] = a;
        }
    }
    if (q0 + r >= p.Lq) return;
    const float inv = l > 0.f ? 1.f / l : l;             // 0: no key; NaN stays
    T* op = (T*)p.out + b * p.os[0] + h * p.os[1] + (int64_t)(q0 + r) * p.os[2];
#pragma unroll
    for (int i = 0; i < kSimtMaxD / 8; ++i) {
        const int d = c8 + 8 * i;
        if (d < p.D) op[d] = from_f32<T>(acc[i] * inv);
    }
    if (c8 == 0) p.lse[((int64_t)b * p.H + h) * p.Lq + q0 + r] = l == 0.f ? -CUDART_INF_F : m + logf(l);
}

// delta[b][h][i] = sum_d dout * out: one warp per row; 0 for a row that saw nothing.
template <typename T>
__global__ void attn_delta_kernel(const __grid_constant__ AttnParams p)
{
    const int64_t row = (int64_t)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32;
    if (row >= (int64_t)p.B * p.H * p.Lq) return;
    const int i = (int)(row % p.Lq);
    const int h = (int)(row / p.Lq % p.H), b = (int)(row / p.Lq / p.H);
    float s = 0.f;
    if (p.lse[row] != -CUDART_INF_F) {
        const T* o = (const T*)p.out + b * p.os[0] + h * p.os[1] + (int64_t)i * p.os[2];
        const T* g = (const T*)p.dout + b * p.dos[0] + h * p.dos[1] + (int64_t)i * p.dos[2];
        for (int d = threadIdx.x % 32; d < p.D; d += 32) s = fmaf(to_f32(o[d]), to_f32(g[d]), s);
    }
#pragma unroll
    for (int o = 16; o; o /= 2) s += __shfl_xor_sync(~0u, s, o);
    if (threadIdx.x % 32 == 0) p.delta[row] = s;
}

// P, P * curve and dS of pair (query, key) from the two products. fine: what lse is short of (dQ's kernel finds it).
__device__ __forceinline__ void simt_grad(const AttnParams& p, bool seen, float qk, float dov, float lse, float fine,
                                          float delta, float slope, int dist, float& P, float& PC, float& dS)
{
    P = PC = dS = 0.f;
    if (!seen) return;
    float bend;
    const float s = score(p.scale * qk, p.cap, slope, dist, bend);
    P = expf((s - lse) - fine);
    PC = P * (1.f - bend * bend);
    dS = P * (dov - delta) * (1.f - bend * bend) * p.scale;
}

// dQ. With 16-bit tensors delta carries the rounding of out, which is as large as dP - delta where the
// values of a row have much in common. The true delta makes the row's sum of P * (dP - delta) zero, so
// what that sum is is delta's error r: dQ loses r times sum P curve k, and delta becomes exact for dK,
// which is computed after it. The row's sum of P, 1 but for the rounding of the fp32 lse, divides dQ, and its
// logarithm goes to dK and dV in the same way. Without the first, gradients of values that differ in their last
// bit alone are off by their own size; it costs 6 % (bf16 [4, 8, 512, 33]: gradients 588 -> 624 us). Two blocks
// an SM: with the 163 registers that it would take, 709 us.
template <typename T>
__global__ void __launch_bounds__(kSimtThreads, 2) attn_simt_backward_dq(const __grid_constant__ AttnParams p)
{
    extern __shared__ float sm[];
    const int pitch = p.D + 1;
    float* Q = sm;
    float* G = Q + kSimtTile * pitch;
    float* K = G + kSimtTile * pitch;
    float* V = K + kSimtTile * pitch;
    float* S = V + kSimtTile * pitch;
    constexpr bool kCorrect = sizeof(T) == 2;
    float2* SC = reinterpret_cast<float2*>(S);   // dS and P * curve side by side, where delta is corrected
    __shared__ int kdoc[kSimtTile];

    const int tiles = (p.Lq + kSimtTile - 1) / kSimtTile, bh = blockIdx.x / tiles;
    const int h = bh % p.H, b = bh / p.H, kv = h / (p.H / p.Hkv);
    const int q0 = (blockIdx.x - bh * tiles) * kSimtTile;
    const int r = threadIdx.x / 8, c8 = threadIdx.x % 8;
    const T* kp = (const T*)p.k + b * p.ks[0] + kv * p.ks[1];
    const T* vp = (const T*)p.v + b * p.vs[0] + kv * p.vs[1];
    const int32_t* docs = p.docs ? p.docs + (int64_t)b * p.Lk : nullptr;
    const int prefix = p.prefix ? __ldg(p.prefix + b) : 0;
    const float slope = p.slopes ? __ldg(p.slopes + h) : 0.f;
    const int qpos = query_pos(p, q0 + r);
    const int qdoc = docs ? doc_at(p, b, qpos) : 0;
    const int64_t row = ((int64_t)b * p.H + h) * p.Lq + q0 + r;
    const bool live = q0 + r < p.Lq;
    const float lse = live ? p.lse[row] : 0.f, delta = live ? p.delta[row] : 0.f;

    simt_load(Q, pitch, (const T*)p.q + b * p.qs[0] + h * p.qs[1], p.qs[2], q0, p.Lq, p.D, docs, p.Lk - p.Lq);
    simt_load(G, pitch, (const T*)p.dout + b * p.dos[0] + h * p.dos[1], p.dos[2], q0, p.Lq, p.D, docs, p.Lk - p.Lq);
    float acc[kSimtMaxD / 8], off[kSimtMaxD / 8], rest = 0.f, total = 0.f;
#pragma unroll
    for (int i = 0; i < kSimtMaxD / 8; ++i) acc[i] = off[i] = 0.f;
    const int jend = key_end(p, query_pos(p, min(q0 + kSimtTile, p.Lq) - 1), prefix);
    for (int j0 = 0; j0 < jend; j0 += kSimtTile) {
        __syncthreads();
        simt_load(K, pitch, kp, p.ks[2], j0, p.Lk, p.D, docs, 0);
        simt_load(V, pitch, vp, p.vs[2], j0, p.Lk, p.D, docs, 0);
        if (docs && threadIdx.x < kSimtTile) kdoc[threadIdx.x] = doc_at(p, b, j0 + threadIdx.x);
        __syncthreads();
        float part = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int c = c8 + 8 * i, j = j0 + c;
            const bool seen = live && j < p.Lk && sees(p, qpos, qdoc, j, docs ? kdoc[c] : 0, prefix);
            float P, PC, dS;
            const float dP = simt_dot(G + r * pitch, V + c * pitch, p.D);
            simt_grad(p, seen, simt_dot(Q + r * pitch, K + c * pitch, p.D), dP, lse, 0.f, delta, slope, qpos - j, P, PC, dS);
            part += P;
            if (kCorrect) {
                SC[r * 33 + c] = make_float2(dS, PC);
                if (seen) rest = fmaf(P, dP - delta, rest);
            } else {
                S[r * 33 + c] = dS;
            }
        }
        total += part;
        __syncwarp();
#pragma unroll
        for (int i = 0; i < kSimtMaxD / 8; ++i) {
            const int d = c8 + 8 * i;
            if (d >= p.D) break;
            float a = acc[i], o = off[i];
            for (int c = 0; c < kSimtTile; ++c) {
                const float2 x = kCorrect ? SC[r * 33 + c] : make_float2(S[r * 33 + c], 0.f);
                a = fmaf(x.x, K[c * pitch + d], a);
                if (kCorrect) o = fmaf(x.y, K[c * pitch + d], o);
            }
            acc[i] = a;
            off[i] = o;
        }
    }
#pragma unroll
    for (int o = 1; o < 8; o *= 2) {
        total += __shfl_xor_sync(~0u, total, o);
        rest += __shfl_xor_sync(~0u, rest, o);
    }
    if (!live) return;
    const float inv = total == 0.f ? 1.f : 1.f / total;
    rest *= inv;
    if (c8 == 0) {
        p.fine[row] = total == 0.f ? 0.f : logf(total);
        if (kCorrect) p.delta[row] = delta + rest;
    }
    T* o = (T*)p.dq + b * p.dqs[0] + h * p.dqs[1] + (int64_t)(q0 + r) * p.dqs[2];
#pragma unroll
    for (int i = 0; i < kSimtMaxD / 8; ++i) {
        const int d = c8 + 8 * i;
        if (d < p.D) o[d] = from_f32<T>((kCorrect ? fmaf(-rest * p.scale, off[i], acc[i]) : acc[i]) * inv);
    }
}

template <typename T>
__global__ void __launch_bounds__(kSimtThreads) attn_simt_backward_dkv(const __grid_constant__ AttnParams p)
{
    extern __shared__ float sm[];
    const int pitch = p.D + 1;
    float* K = sm;
    float* V = K + kSimtTile * pitch;
    float* Q = V + kSimtTile * pitch;
    float* G = Q + kSimtTile * pitch;
    float* PT = G + kSimtTile * pitch;           // [key][query]
    float* ST = PT + kSimtTile * 33;
    __shared__ int qdoc[kSimtTile];

    const int tiles = (p.Lk + kSimtTile - 1) / kSimtTile, bh = blockIdx.x / tiles;
    const int kv = bh % p.Hkv, b = bh / p.Hkv, group = p.H / p.Hkv;
    const int j0 = (blockIdx.x - bh * tiles) * kSimtTile;
    const int r = threadIdx.x / 8, c8 = threadIdx.x % 8, j = j0 + r;
    const int32_t* docs = p.docs ? p.docs + (int64_t)b * p.Lk : nullptr;
    const int prefix = p.prefix ? __ldg(p.prefix + b) : 0;
    const int kdoc = docs ? doc_at(p, b, j) : 0;

    simt_load(K, pitch, (const T*)p.k + b * p.ks[0] + kv * p.ks[1], p.ks[2], j0, p.Lk, p.D, docs, 0);
    simt_load(V, pitch, (const T*)p.v + b * p.vs[0] + kv * p.vs[1], p.vs[2], j0, p.Lk, p.D, docs, 0);
    float dk[kSimtMaxD / 8], dv[kSimtMaxD / 8];
#pragma unroll
    for (int i = 0; i < kSimtMaxD / 8; ++i) dk[i] = dv[i] = 0.f;
    // queries before position j0 see none of these keys, unless a prefix covers one
    const int first = p.causal && j0 >= prefix ? max(0, j0 - (p.Lk - p.Lq)) / kSimtTile * kSimtTile : 0;
    for (int h = kv * group; h < (kv + 1) * group; ++h) {
        const T* qp = (const T*)p.q + b * p.qs[0] + h * p.qs[1];
        const T* gp = (const T*)p.dout + b * p.dos[0] + h * p.dos[1];
        const float slope = p.slopes ? __ldg(p.slopes + h) : 0.f;
        for (int q0 = first; q0 < p.Lq; q0 += kSimtTile) {
            __syncthreads();
            simt_load(Q, pitch, qp, p.qs[2], q0, p.Lq, p.D, docs, p.Lk - p.Lq);
            simt_load(G, pitch, gp, p.dos[2], q0, p.Lq, p.D, docs, p.Lk - p.Lq);
            if (docs && threadIdx.x < kSimtTile) qdoc[threadIdx.x] = doc_at(p, b, query_pos(p, q0 + threadIdx.x));
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int c = c8 + 8 * i, q = q0 + c, qpos = query_pos(p, q);
                const int64_t row = ((int64_t)b * p.H + h) * p.Lq + q;
                const bool seen = q < p.Lq && j < p.Lk && sees(p, qpos, docs ? qdoc[c] : 0, j, kdoc, prefix);
                float P, PC, dS;
                simt_grad(p, seen, simt_dot(Q + c * pitch, K + r * pitch, p.D),
                          simt_dot(G + c * pitch, V + r * pitch, p.D), seen ? p.lse[row] : 0.f,
                          seen ? p.fine[row] : 0.f, seen ? p.delta[row] : 0.f, slope, qpos - j, P, PC, dS);
                PT[r * 33 + c] = P;
                ST[r * 33 + c] = dS;
            }
            __syncwarp();
#pragma unroll
            for (int i = 0; i < kSimtMaxD / 8; ++i) {
                const int d = c8 + 8 * i;
                if (d >= p.D) break;
                float a = dk[i], v = dv[i];
                for (int c = 0; c < kSimtTile; ++c) {
                    a = fmaf(ST[r * 33 + c], Q[c * pitch + d], a);
                    v = fmaf(PT[r * 33 + c], G[c * pitch + d], v);
                }
                dk[i] = a;
                dv[i] = v;
            }
        }
    }
    if (j >= p.Lk) return;
    T* ok = (T*)p.dk + b * p.dks[0] + kv * p.dks[1] + (int64_t)j * p.dks[2];
    T* ov = (T*)p.dv + b * p.dvs[0] + kv * p.dvs[1] + (int64_t)j * p.dvs[2];
#pragma unroll
    for (int i = 0; i < kSimtMaxD / 8; ++i) {
        const int d = c8 + 8 * i;
        if (d < p.D) {
            ok[d] = from_f32<T>(dk[i]);
            ov[d] = from_f32<T>(dv[i]);
        }
    }
}

}  // namespace mg
