// mg_paged.cuh -- attention of one new token per request over a paged cache,
// split over the cache's length and joined.
//
// One block reads `chunk` keys of one key-value head of one request, once, for
// all query heads that share it (in groups of kPagedHeads), and leaves per query
// head the maximum m, the sum l = sum exp(s - m) and the sum of exp(s - m) v. A
// request of one chunk is finished there; otherwise a second kernel joins its
// chunks: M = max m, out = sum exp(m - M) acc / sum exp(m - M) l.
// The bound is the cache's bytes.
#pragma once

#include "mg_attention_common.cuh"

namespace mg {

struct PagedParams {
    int B, H, Hkv, D, page, pages, width;
    float scale, cap;
    int64_t qs[2], os[2], ks[3], vs[3], kns[2], vns[2];
    int64_t table_stride;
    const float* slopes;
    const int32_t* table;
    const int32_t* lengths;      // NULL: every request has `length` keys
    int length;
    const int32_t* docs;         // rows of contiguous keys: the document of each, or NULL
    const void* q;
    void *k, *v;                 // the cache; written only where k_new is given
    const void *k_new, *v_new;
    void* out;
    float* lse;
    int chunk, splits;           // keys a block reads; blocks along the length
    float* part;                 // [B * H][splits][D] accumulators
    float2* stat;                // [B * H][splits] (m, l)
    int* status;
};

constexpr int kPagedThreads = 128;
constexpr int kPagedHeads = 8;

// Number of keys of request b; a length beyond the table is cut off there.
__device__ __forceinline__ int paged_length(const PagedParams& p, int b)
{
    if (p.lengths == nullptr) return p.length;
    const int64_t most = (int64_t)p.width * p.page;
    const int n = __ldg(p.lengths + b);
    return n < 0 ? 0 : n > most ? (int)most : n;
}

__device__ __forceinline__ void paged_report(const PagedParams& p, int code)
{
    if (atomicCAS(p.status, 0, 1 /* MG_ERR_INVALID */) == 0) p.status[1] = code;
}

constexpr int kPagedBadPage = 101, kPagedBadLength = 102;   // detail codes of mg_device_status()

// Cache rows of key j of request b (k and v strides differ): false if its page
// is not one of the pool's.
__device__ __forceinline__ bool paged_row(const PagedParams& p, int b, int j, int& page, int& row)
{
    if (p.table == nullptr) {
        page = b;
        row = j;
        return true;
    }
    const int n = j / p.page;
    page = __ldg(p.table + b * p.table_stride + n);
    row = j - n * p.page;
    return page >= 0 && page < p.pages;
}

// Simple form: a warp per key, lanes over the head's elements.
template <typename T>
__global__ void __launch_bounds__(kPagedThreads) paged_simt_kernel(const __grid_constant__ PagedParams p)
{
    const int split = blockIdx.x % p.splits;
    const int bh = blockIdx.x / p.splits;
    const int groups = p.H / p.Hkv, packs = (groups + kPagedHeads - 1) / kPagedHeads;
    const int pack = bh % packs, kv = bh / packs % p.Hkv, b = bh / packs / p.Hkv;
    const int len = paged_length(p, b);
    if (threadIdx.x == 0 && split == 0 && p.lengths && __ldg(p.lengths + b) != len) paged_report(p, kPagedBadLength);
    const int j0 = split * p.chunk, j1 = min(len, j0 + p.chunk);
    const int h0 = kv * groups + pack * kPagedHeads, nh = min(kPagedHeads, groups - pack * kPagedHeads);
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    constexpr int kWarps = kPagedThreads / 32, kPer = MG_MAX_HEAD_DIM / 32;
    if (j0 >= j1 && split > 0) return;      // a chunk beyond the request's keys is not joined

    float q[kPagedHeads][kPer], acc[kPagedHeads][kPer], m[kPagedHeads], l[kPagedHeads], slope[kPagedHeads];
    const int qdoc = p.docs && len > 0 ? __ldg(p.docs + (int64_t)b * p.length + len - 1) : 0;
#pragma unroll
    for (int g = 0; g < kPagedHeads; ++g) {
        m[g] = -CUDART_INF_F;
        l[g] = 0.f;
        slope[g] = p.slopes && g < nh ? __ldg(p.slopes + h0 + g) : 0.f;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int d = lane + 32 * i;
            acc[g][i] = 0.f;
            q[g][i] = g < nh && d < p.D ? to_f32(((const T*)p.q)[b * p.qs[0] + (h0 + g) * p.qs[1] + d]) : 0.f;
        }
    }
    for (int j = j0 + warp; j < j1; j += kWarps) {
        int page, row;
        const bool have = paged_row(p, b, j, page, row);
        const bool fresh = p.k_new != nullptr && j == len - 1;
        if (!have) {
            if (lane == 0) paged_report(p, kPagedBadPage);
            continue;
        }
        if (p.docs) {
            const int kdoc = __ldg(p.docs + (int64_t)b * p.length + j);
            if (qdoc < 0 || kdoc != qdoc) continue;
        }
        T* kc = (T*)p.k + page * p.ks[0] + row * p.ks[1] + kv * p.ks[2];
        T* vc = (T*)p.v + page * p.vs[0] + row * p.vs[1] + kv * p.vs[2];
        const T* kr = fresh ? (const T*)p.k_new + b * p.kns[0] + kv * p.kns[1] : kc;
        const T* vr = fresh ? (const T*)p.v_new + b * p.vns[0] + kv * p.vns[1] : vc;
        float k[kPer], v[kPer];
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int d = lane + 32 * i;
            const bool in = d < p.D;
            const T tk = in ? kr[d] : from_f32<T>(0.f), tv = in ? vr[d] : from_f32<T>(0.f);
            k[i] = to_f32(tk);
            v[i] = to_f32(tv);
            if (fresh && pack == 0 && in) {
                kc[d] = tk;
                vc[d] = tv;
            }
        }
#pragma unroll
        for (int g = 0; g < kPagedHeads; ++g) {
            if (g >= nh) break;
            float s = 0.f, bend;
#pragma unroll
            for (int i = 0; i < kPer; ++i) s = fmaf(q[g][i], k[i], s);
#pragma unroll
            for (int o = 16; o; o /= 2) s += __shfl_xor_sync(~0u, s, o);
            s = score(p.scale * s, p.cap, slope[g], len - 1 - j, bend);
            const float mn = fmaxf(m[g], s);
            if (mn == -CUDART_INF_F) continue;
            const float fix = expf(m[g] - mn), e = expf(s - mn);
            m[g] = mn;
            l[g] = l[g] * fix + e;
#pragma unroll
            for (int i = 0; i < kPer; ++i) acc[g][i] = fmaf(e, v[i], acc[g][i] * fix);
        }
    }
    // join the block's warps
    __shared__ float sm_m[kWarps][kPagedHeads], sm_l[kWarps][kPagedHeads];
    __shared__ float sm_acc[kWarps][kPagedHeads][MG_MAX_HEAD_DIM];
#pragma unroll
    for (int g = 0; g < kPagedHeads; ++g) {
        if (lane == 0) sm_m[warp][g] = m[g], sm_l[warp][g] = l[g];
#pragma unroll
        for (int i = 0; i < kPer; ++i) sm_acc[warp][g][lane + 32 * i] = acc[g][i];
    }
    __syncthreads();
    for (int g = warp; g < nh; g += kWarps) {
        float M = -CUDART_INF_F;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) M = fmaxf(M, sm_m[w][g]);
        const float base = M == -CUDART_INF_F ? 0.f : M;
        float L = 0.f, f[kWarps];
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            f[w] = expf(sm_m[w][g] - base);
            L += f[w] * sm_l[w][g];
        }
        const int64_t row = (int64_t)b * p.H + h0 + g;
        const float inv = L > 0.f ? 1.f / L : 0.f;
        for (int d = lane; d < p.D; d += 32) {
            float a = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) a = fmaf(f[w], sm_acc[w][g][d], a);
            if (p.splits == 1) ((T*)p.out)[b * p.os[0] + (h0 + g) * p.os[1] + d] = from_f32<T>(a * inv);
            else p.part[(row * p.splits + split) * p.D + d] = a;
        }
        if (lane == 0) {
            if (p.splits == 1) p.lse[row] = L > 0.f ? M + logf(L) : -CUDART_INF_F;
            else p.stat[row * p.splits + split] = make_float2(M, L);
        }
    }
}

// Joins the chunks of one query head: one warp per head.
template <typename T>
__global__ void __launch_bounds__(kPagedThreads) paged_join_kernel(const __grid_constant__ PagedParams p)
{
    const int64_t row = (int64_t)blockIdx.x * (kPagedThreads / 32) + threadIdx.x / 32;
    if (row >= (int64_t)p.B * p.H) return;
    const int lane = threadIdx.x % 32;
    const int b = (int)(row / p.H), h = (int)(row % p.H);
    const int n = max(1, (paged_length(p, b) + p.chunk - 1) / p.chunk);
    const float2* st = p.stat + row * p.splits;
    float M = -CUDART_INF_F;
    for (int s = lane; s < n; s += 32) M = fmaxf(M, st[s].x);
#pragma unroll
    for (int o = 16; o; o /= 2) M = fmaxf(M, __shfl_xor_sync(~0u, M, o));
    const float base = M == -CUDART_INF_F ? 0.f : M;
    float L = 0.f;
    for (int s = lane; s < n; s += 32) L += expf(st[s].x - base) * st[s].y;
#pragma unroll
    for (int o = 16; o; o /= 2) L += __shfl_xor_sync(~0u, L, o);
    const float inv = L > 0.f ? 1.f / L : 0.f;
    T* out = (T*)p.out + b * p.os[0] + h * p.os[1];
    for (int d = lane; d < p.D; d += 32) {
        float a = 0.f;
        for (int s = 0; s < n; ++s) a = fmaf(expf(st[s].x - base), p.part[(row * p.splits + s) * p.D + d], a);
        out[d] = from_f32<T>(a * inv);
    }
    if (lane == 0) p.lse[row] = L > 0.f ? M + logf(L) : -CUDART_INF_F;
}

}  // namespace mg
