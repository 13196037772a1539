// mg_paged.cuh -- attention of one new token per request over a paged cache,
// split over the cache's length and joined.
//
// Two forms. paged_kernel streams the cache through shared memory (rows on
// 16-byte boundaries); paged_simt_kernel takes any strides.
//
// One block reads a chunk of the keys of one key-value head of one request for the
// query heads that share it, in packs of kPagedHeads (fp32, and the simple form) or 16
// (bf16): heads beyond a pack read the cache again. It leaves per query head the
// maximum m, the sum l = sum exp(s - m) and the sum of exp(s - m) v; in the streaming form
// scores and m are in powers of two. A call of one chunk a request is finished there;
// otherwise the chunks are joined, inside a cluster where a call is small and
// by a second kernel else: M = max m, out = sum exp(m - M) acc / sum exp(m - M) l.
// The bound is the cache's bytes.
#pragma once

#include "mg_attention_math.cuh"
#include "mg_ptx.cuh"

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
    int page_shift;              // log2(page), or -1
    int splits, least;           // blocks along the length of a request; fewest keys of one
    CapCurve curve;              // of the cap, with a cap
    float* part;                 // [B * H][splits][D] accumulators
    float2* stat;                // [B * H][splits] (m, l)
    int powers;                  // m, and the scores, in powers of two (streaming form); else natural
    int* status;
};

constexpr int kPagedThreads = 128;
constexpr int kPagedHeads = 8;

// Number of keys of request b; a length beyond the table is cut off there: what lies
// beyond, the token to append among it, is neither read nor written.
__device__ __forceinline__ int paged_length(const PagedParams& p, int b)
{
    if (p.lengths == nullptr) return p.length;
    const int64_t most = (int64_t)p.width * p.page;
    const int n = __ldg(p.lengths + b);
    return n < 0 ? 0 : n > most ? (int)most : n;
}

// Place of the token that request b of `len` keys appends, or -1: none, or one that its table has no room for.
__device__ __forceinline__ int paged_append(const PagedParams& p, int b, int len)
{
    return p.k_new != nullptr && len > 0 && __ldg(p.lengths + b) == len ? len - 1 : -1;
}

// Keys that a block of a request of `len` keys reads: its share, but no less than
// `least`, in whole rounds of the block's four tiles. By the request's own length:
// the block table may be much wider.
__device__ __forceinline__ int paged_chunk(const PagedParams& p, int len)
{
    const int share = (len + p.splits - 1) / p.splits;
    return (max(share, p.least) + 63) / 64 * 64;
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
    const int n = p.page_shift >= 0 ? j >> p.page_shift : j / p.page;
    page = __ldg(p.table + b * p.table_stride + n);
    row = j - n * p.page;
    return page >= 0 && page < p.pages;
}

__device__ __forceinline__ float4 lds4(uint32_t addr)
{
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
    return v;
}

__device__ __forceinline__ float paged_lse(const PagedParams& p, float M, float L)
{
    return L == 0.f ? -CUDART_INF_F : (p.powers ? M * kLn2 : M) + logf(L);
}

// What one warp does with a finished chunk of one query head: the result where
// the call has one chunk a request, else its part of the join. M: as p.powers says.
template <typename T, typename F>
__device__ __forceinline__ void paged_store(const PagedParams& p, int b, int h, int split, float M, float L, int lane,
                                            F&& acc)
{
    const int64_t row = (int64_t)b * p.H + h;
    const float inv = L > 0.f ? 1.f / L : L;           // 0: no key; NaN stays
    for (int d = lane; d < p.D; d += 32) {
        const float a = acc(d);
        if (p.splits == 1) ((T*)p.out)[b * p.os[0] + h * p.os[1] + d] = from_f32<T>(a * inv);
        else p.part[(row * p.splits + split) * p.D + d] = a;
    }
    if (lane == 0) {
        if (p.splits == 1) p.lse[row] = paged_lse(p, M, L);
        else p.stat[row * p.splits + split] = make_float2(M, L);
    }
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
    const int chunk = paged_chunk(p, len);
    const int j0 = min(len, split * chunk), j1 = min(len, j0 + chunk);
    const int h0 = kv * groups + pack * kPagedHeads, nh = min(kPagedHeads, groups - pack * kPagedHeads);
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    constexpr int kWarps = kPagedThreads / 32, kPer = MG_MAX_HEAD_DIM / 32;
    if (j0 >= j1 && split > 0) return;      // a chunk beyond the request's keys is not joined
    const int append = paged_append(p, b, len);

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
        const bool fresh = j == append;
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
            if (mn == -CUDART_INF_F && s == mn) continue;      // NaN is counted, and stays in l
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
        paged_store<T>(p, b, h0 + g, split, M, L, lane, [&](int d) {
            float a = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) a = fmaf(f[w], sm_acc[w][g][d], a);
            return a;
        });
    }
}

// ---------------------------------------------------------------- streaming form
// Each warp walks tiles of 16 keys of its block's chunk (every fourth tile) and
// keeps kPagedStages of them in flight into shared memory by 16-byte
// asynchronous copies, so that the loads of the next tiles run under the
// arithmetic of this one and no warp waits for another: a block of 4 warps has
// up to 4 * 2 * 16 * D elements of keys and values on the way. A row's 16-byte
// pieces are permuted by its number (piece ^ (row & 7)), so that reading one
// piece of 8 rows meets 8 different groups of banks. What a page table entry or
// a document hides is filled with zeros instead of being loaded, and masked.
//
// bf16: the query heads of the key-value head are the 16 rows of m16n8k16
// products (S = Q K^T, O += P V; P in the layout that S leaves it in): with
// one to sixteen heads to a key-value head the loads bound the kernel, not the
// arithmetic, so the warp-level instruction is enough here. fp32: a lane has one key (half of the head
// each in two lanes) for the scores and D / 32 elements of the output.
constexpr int kPagedStages = 2;          // 3 leave a block less an SM: 102 -> 120 us, 115 -> 141 us (ragged, long)
constexpr int kPagedTile = 16;
constexpr int kPagedWarps = kPagedThreads / 32;

template <typename T>
__host__ __device__ constexpr int paged_pack() { return sizeof(T) == 2 ? 16 : kPagedHeads; }    // query heads of a block

template <typename T, int DP>
constexpr size_t paged_smem()
{
    const size_t ring = (size_t)kPagedWarps * kPagedStages * 2 * kPagedTile * DP * sizeof(T);
    const size_t join = (size_t)(kPagedWarps + 1) * paged_pack<T>() * DP * sizeof(float) + paged_pack<T>() * sizeof(float2);
    return ring > join ? ring : join;
}

// Words of another block's shared memory (shared::cluster addresses).
__device__ __forceinline__ float remote1(uint32_t addr)
{
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float2 remote2(uint32_t addr)
{
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
    return v;
}

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool live)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// What a warp keeps of its keys: bf16.
template <typename T, int DP>
struct PagedAcc {
    uint32_t q[DP / 16][4];      // A operand: rows g and g + 8, elements 2t, 2t + 1 (+ 8) of each 16
    float o[DP / 8][4];
    float m[2], l[2], slope[2];  // heads g and g + 8; l of this lane's keys alone
    __device__ __forceinline__ void init(const PagedParams& p, int b, int h0, int nh, int lane, const float*)
    {
        const int g = lane / 4, t = lane % 4;
        const T* q0 = (const T*)p.q + b * p.qs[0] + (h0 + g) * p.qs[1];
        const T* q1 = q0 + 8 * p.qs[1];
        const auto two = [&](const T* x, bool head, int d) {
            __nv_bfloat162 v;
            v.x = head && d < p.D ? x[d] : __float2bfloat16(0.f);
            v.y = head && d + 1 < p.D ? x[d + 1] : __float2bfloat16(0.f);
            return *reinterpret_cast<uint32_t*>(&v);
        };
#pragma unroll
        for (int k = 0; k < DP / 16; ++k) {
            q[k][0] = two(q0, g < nh, 16 * k + 2 * t);
            q[k][1] = two(q1, g + 8 < nh, 16 * k + 2 * t);
            q[k][2] = two(q0, g < nh, 16 * k + 2 * t + 8);
            q[k][3] = two(q1, g + 8 < nh, 16 * k + 2 * t + 8);
        }
#pragma unroll
        for (int i = 0; i < DP / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            m[i] = -CUDART_INF_F;
            l[i] = 0.f;
            slope[i] = p.slopes && g + 8 * i < nh ? __ldg(p.slopes + h0 + g + 8 * i) * kLog2e : 0.f;
        }
    }
    // Tile of 16 keys at sk, sv; key i is seen where bit i of `seen` is set and stands `back - i` before the query.
    __device__ __forceinline__ void tile(const PagedParams& p, uint32_t sk, uint32_t sv, uint32_t seen, int back, int nh,
                                         int lane)
    {
        const int t = lane % 4;
        float s[2][4] = {};
#pragma unroll
        for (int k = 0; k < DP / 16; ++k) {
            // matrices: keys 0-7 of both halves of the 16 elements, then keys 8-15
            const int row = (lane & 7) + (lane >> 4) * 8, piece = 2 * k + ((lane >> 3) & 1);
            uint32_t b[4];
            ldmatrix4(b, sk + row * (DP * 2) + ((piece ^ (row & 7)) << 4));
            mma16816(s[0], q[k], b[0], b[1]);
            mma16816(s[1], q[k], b[2], b[3]);
        }
        float mul = p.scale * kLog2e;
        if (p.cap > 0.f) {
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = p.scale < 0.f ? -s[i / 4][i % 4] : s[i / 4][i % 4];
            cap_scores(x, p.curve);
#pragma unroll
            for (int i = 0; i < 8; ++i) s[i / 4][i % 4] = x[i];
            mul = p.cap * kLog2e;
        }
        uint32_t a[4];
        if (p.slopes != nullptr) weights<true, false>(s, mul, seen, back, t, a);
        else if (seen != 0xFFFFu) weights<false, false>(s, mul, seen, back, t, a);
        else weights<false, true>(s, mul, seen, back, t, a);
#pragma unroll
        for (int k = 0; k < DP / 16; ++k) {
            // matrices: keys 0-7 and 8-15 of 8 elements, then of the next 8
            const int row = lane & 15, piece = 2 * k + (lane >> 4);
            uint32_t b[4];
            ldmatrix4_trans(b, sv + row * (DP * 2) + ((piece ^ (row & 7)) << 4));
            mma16816(o[2 * k], a, b[0], b[1]);
            mma16816(o[2 * k + 1], a, b[2], b[3]);
        }
    }
    // Weights of a tile's scores (their powers of two are s * mul - slope * distance) as the A operand of the second
    // product; m, l and o follow a new maximum. kAll: every key is seen, the usual tile.
    template <bool kBias, bool kAll>
    __device__ __forceinline__ void weights(const float (&s)[2][4], float mul, uint32_t seen, int back, int t, uint32_t (&a)[4])
    {
        float top[2] = {-CUDART_INF_F, -CUDART_INF_F};
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int key = 8 * n + 2 * t + (i & 1);
                const float x = kBias ? fmaf(s[n][i], mul, -slope[i >> 1] * (float)(back - key)) : s[n][i] * mul;
                top[i >> 1] = fmaxf(top[i >> 1], kAll || (seen >> key & 1) ? x : -CUDART_INF_F);
            }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            top[i] = fmaxf(top[i], __shfl_xor_sync(~0u, top[i], 1));
            top[i] = fmaxf(top[i], __shfl_xor_sync(~0u, top[i], 2));
        }
        // the maximum in use follows once it is 2^8 behind (or there was none)
        const bool up0 = m[0] == -CUDART_INF_F ? top[0] > m[0] : top[0] - m[0] > 8.f;
        const bool up1 = m[1] == -CUDART_INF_F ? top[1] > m[1] : top[1] - m[1] > 8.f;
        if (__any_sync(~0u, up0 || up1)) {
            const float n0 = up0 ? top[0] : m[0], n1 = up1 ? top[1] : m[1];
            const float f0 = up0 ? ex2(m[0] - n0) : 1.f, f1 = up1 ? ex2(m[1] - n1) : 1.f;
            m[0] = n0, m[1] = n1;
            l[0] *= f0, l[1] *= f1;
#pragma unroll
            for (int i = 0; i < DP / 8; ++i) o[i][0] *= f0, o[i][1] *= f0, o[i][2] *= f1, o[i][3] *= f1;
        }
        const float b[2] = {m[0] == -CUDART_INF_F ? 0.f : -m[0], m[1] == -CUDART_INF_F ? 0.f : -m[1]};
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            // score and maximum in one rounding: the scores' own, 2^-24 of their size, would stay in the weights
            float e[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int key = 8 * n + 2 * t + (i & 1);
                const float x = fmaf(s[n][i], mul, kBias ? fmaf(-slope[i >> 1], (float)(back - key), b[i >> 1]) : b[i >> 1]);
                e[i] = ex2(kAll || (seen >> key & 1) ? x : -CUDART_INF_F);
            }
            const float e0 = e[0], e1 = e[1], e2 = e[2], e3 = e[3];
            l[0] += e0 + e1;
            l[1] += e2 + e3;
            const __nv_bfloat162 x = __floats2bfloat162_rn(e0, e1), y = __floats2bfloat162_rn(e2, e3);
            a[2 * n] = *reinterpret_cast<const uint32_t*>(&x);
            a[2 * n + 1] = *reinterpret_cast<const uint32_t*>(&y);
        }
    }
    __device__ __forceinline__ void finish(float* sm_m, float* sm_l, float* sm_o, int nh, int lane)
    {
        const int g = lane / 4, t = lane % 4;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            l[i] += __shfl_xor_sync(~0u, l[i], 1);
            l[i] += __shfl_xor_sync(~0u, l[i], 2);
            if (t == 0) sm_m[g + 8 * i] = m[i], sm_l[g + 8 * i] = l[i];
        }
#pragma unroll
        for (int i = 0; i < DP / 8; ++i) {
            float2* lo = reinterpret_cast<float2*>(sm_o + g * DP + 8 * i + 2 * t);
            float2* hi = reinterpret_cast<float2*>(sm_o + (g + 8) * DP + 8 * i + 2 * t);
            *lo = make_float2(o[i][0], o[i][1]);
            *hi = make_float2(o[i][2], o[i][3]);
        }
    }
};

// fp32. For the scores a lane has one key and half of the head; for the output it
// has half of the keys (its half warp's eight) and every sixteenth piece of the head.
template <int DP>
struct PagedAcc<float, DP> {
    static constexpr int kPer = DP / 64;     // pieces of four elements a lane
    const float* q;              // [heads][DP] in shared memory
    float4 o[kPagedHeads][kPer];
    float m[kPagedHeads], l[kPagedHeads], slope[kPagedHeads];
    __device__ __forceinline__ void init(const PagedParams& p, int, int h0, int nh, int, const float* sq)
    {
        q = sq;
#pragma unroll
        for (int g = 0; g < kPagedHeads; ++g) {
            m[g] = -CUDART_INF_F;
            l[g] = 0.f;
            slope[g] = p.slopes && g < nh ? __ldg(p.slopes + h0 + g) * kLog2e : 0.f;
#pragma unroll
            for (int i = 0; i < kPer; ++i) o[g][i] = make_float4(0.f, 0.f, 0.f, 0.f);
        }
    }
    __device__ __forceinline__ void tile(const PagedParams& p, uint32_t sk, uint32_t sv, uint32_t seen, int back, int nh,
                                         int lane)
    {
        const int key = lane & 15, half = lane >> 4;
        float s[kPagedHeads];
#pragma unroll
        for (int g = 0; g < kPagedHeads; ++g) s[g] = 0.f;
#pragma unroll
        for (int i = 0; i < DP / 8; ++i) {
            const int piece = half * (DP / 8) + i;
            const float4 k4 = lds4(sk + key * (DP * 4) + ((piece ^ (key & 7)) << 4));
#pragma unroll
            for (int g = 0; g < kPagedHeads; ++g) {
                if (g >= nh) break;
                const float4 q4 = *reinterpret_cast<const float4*>(q + g * DP + 4 * piece);
                s[g] = fmaf(q4.x, k4.x, fmaf(q4.y, k4.y, fmaf(q4.z, k4.z, fmaf(q4.w, k4.w, s[g]))));
            }
        }
        const float mul = (p.cap > 0.f ? p.cap : p.scale) * kLog2e, far = (float)(back - key);
        const bool in = (seen >> key) & 1;
#pragma unroll
        for (int g = 0; g < kPagedHeads; ++g) {
            if (g >= nh) break;
            float x = s[g] + __shfl_xor_sync(~0u, s[g], 16);
            if (p.cap > 0.f) x = tanhf(x * p.scale / p.cap);
            float top = in ? fmaf(x, mul, -slope[g] * far) : -CUDART_INF_F;
#pragma unroll
            for (int w = 8; w; w /= 2) top = fmaxf(top, __shfl_xor_sync(~0u, top, w));
            if (m[g] == -CUDART_INF_F ? top > m[g] : top - m[g] > 8.f) {     // the same for the whole warp
                const float f = ex2(m[g] - top);
                m[g] = top;
                l[g] *= f;
#pragma unroll
                for (int i = 0; i < kPer; ++i) o[g][i].x *= f, o[g][i].y *= f, o[g][i].z *= f, o[g][i].w *= f;
            }
            // score and maximum in one rounding
            s[g] = ex2(in ? fmaf(x, mul, fmaf(-slope[g], far, m[g] == -CUDART_INF_F ? 0.f : -m[g])) : -CUDART_INF_F);
            l[g] += half ? 0.f : s[g];
        }
#pragma unroll
        for (int r = 0; r < kPagedTile / 2; ++r) {
            const int row = r + 8 * half;
            float4 v[kPer];
#pragma unroll
            for (int i = 0; i < kPer; ++i) v[i] = lds4(sv + row * (DP * 4) + (((lane & 15) + 16 * i) ^ (row & 7)) * 16);
#pragma unroll
            for (int g = 0; g < kPagedHeads; ++g) {
                if (g >= nh) break;
                const float e = __shfl_sync(~0u, s[g], row);
#pragma unroll
                for (int i = 0; i < kPer; ++i) {
                    o[g][i].x = fmaf(e, v[i].x, o[g][i].x), o[g][i].y = fmaf(e, v[i].y, o[g][i].y);
                    o[g][i].z = fmaf(e, v[i].z, o[g][i].z), o[g][i].w = fmaf(e, v[i].w, o[g][i].w);
                }
            }
        }
    }
    __device__ __forceinline__ void finish(float* sm_m, float* sm_l, float* sm_o, int nh, int lane)
    {
#pragma unroll
        for (int g = 0; g < kPagedHeads; ++g) {
            if (g >= nh) break;
            for (int w = 8; w; w /= 2) l[g] += __shfl_xor_sync(~0u, l[g], w);
            if (lane == 0) sm_m[g] = m[g], sm_l[g] = l[g];
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                float4 x = o[g][i];
                x.x += __shfl_xor_sync(~0u, x.x, 16), x.y += __shfl_xor_sync(~0u, x.y, 16);
                x.z += __shfl_xor_sync(~0u, x.z, 16), x.w += __shfl_xor_sync(~0u, x.w, 16);
                if (lane < 16) *reinterpret_cast<float4*>(sm_o + g * DP + 4 * (lane + 16 * i)) = x;
            }
        }
    }
};

// kCluster: the chunks of a head are the blocks of one cluster, which join them
// over distributed shared memory: one launch and no scratch, for calls whose blocks
// are on the GPU all at once anyway (a block without keys has to stay to the end).
template <typename T, int DP, bool kCluster>
__global__ void __launch_bounds__(kPagedThreads) paged_kernel(const __grid_constant__ PagedParams p)
{
    constexpr int kPack = paged_pack<T>(), kPieces = DP * (int)sizeof(T) / 16;
    constexpr uint32_t kTileBytes = kPagedTile * DP * sizeof(T);
    extern __shared__ __align__(128) uint8_t paged_dyn[];
    __shared__ float sm_m[kPagedWarps][16], sm_l[kPagedWarps][16];
    __shared__ __align__(16) float sq[sizeof(T) == 4 ? kPagedHeads * DP : 4];
    __shared__ uint32_t sm_seen[kPagedWarps][kPagedStages];
    __shared__ ulonglong2 sm_rows[kPagedWarps][kPagedTile];

    const int split = blockIdx.x % p.splits, bh = blockIdx.x / p.splits;
    const int groups = p.H / p.Hkv, packs = (groups + kPack - 1) / kPack;
    const int pack = bh % packs, kv = bh / packs % p.Hkv, b = bh / packs / p.Hkv;
    const int len = paged_length(p, b);
    if (threadIdx.x == 0 && split == 0 && p.lengths && __ldg(p.lengths + b) != len) paged_report(p, kPagedBadLength);
    const int chunk = paged_chunk(p, len);
    const int j0 = min(len, split * chunk), j1 = min(len, j0 + chunk);
    if (!kCluster && j0 >= j1 && split > 0) return;      // a chunk beyond the request's keys is not joined
    const int h0 = kv * groups + pack * kPack, nh = min(kPack, groups - pack * kPack);
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(paged_dyn) + warp * kPagedStages * 2 * kTileBytes;
    const int qdoc = p.docs && len > 0 ? __ldg(p.docs + (int64_t)b * p.length + len - 1) : 0;
    const int append = paged_append(p, b, len);

    // Tile n of this warp: keys j0 + (4 n + warp) * 16 and on. Lanes 0-15 find the
    // rows of a key each and leave them to the others in shared memory.
    const auto issue = [&](int n) {
        const int j = j0 + (n * kPagedWarps + warp) * kPagedTile + lane;
        bool live = lane < kPagedTile && j < j1;
        T *kc = nullptr, *vc = nullptr;
        if (live) {
            int page, row;
            if (!paged_row(p, b, j, page, row)) {
                paged_report(p, kPagedBadPage);
                live = false;
            } else if (p.docs && (qdoc < 0 || __ldg(p.docs + (int64_t)b * p.length + j) != qdoc)) {
                live = false;
            } else {
                kc = (T*)p.k + page * p.ks[0] + row * p.ks[1] + kv * p.ks[2];
                vc = (T*)p.v + page * p.vs[0] + row * p.vs[1] + kv * p.vs[2];
            }
        }
        ulonglong2* rows = sm_rows[warp];
        __syncwarp();
        if (lane < kPagedTile) rows[lane] = make_ulonglong2((unsigned long long)kc, (unsigned long long)vc);
        const uint32_t seen = __ballot_sync(~0u, live);
        if (lane == 0) sm_seen[warp][n % kPagedStages] = seen;
        // the token's own key and value go to the cache, and are read from where they came
        const int last = append - (j0 + (n * kPagedWarps + warp) * kPagedTile);
        if (last >= 0 && last < kPagedTile && (seen >> last & 1)) {
            __syncwarp();
            const ulonglong2 at = rows[last];
            const bool is_v = lane >= 16;
            const T* src = is_v ? (const T*)p.v_new + b * p.vns[0] + kv * p.vns[1]
                                : (const T*)p.k_new + b * p.kns[0] + kv * p.kns[1];
            T* out = (T*)(is_v ? at.y : at.x);
            __syncwarp();
            if (pack == 0)
                for (int e = (lane & 15) * (16 / (int)sizeof(T)); e < p.D; e += 16 * (16 / (int)sizeof(T)))
                    *reinterpret_cast<uint4*>(out + e) = *reinterpret_cast<const uint4*>(src + e);
            if (lane == last) rows[lane] = make_ulonglong2((unsigned long long)((const T*)p.k_new + b * p.kns[0] + kv * p.kns[1]),
                                                           (unsigned long long)((const T*)p.v_new + b * p.vns[0] + kv * p.vns[1]));
        }
        __syncwarp();
        const uint32_t dst = ring + (n % kPagedStages) * 2 * kTileBytes;
        constexpr int kStep = 32 / kPieces;              // rows a warp copies at a time
        const int c = lane % kPieces, e = c * (16 / (int)sizeof(T));
#pragma unroll
        for (int i = 0; i < kPagedTile / kStep; ++i) {
            const int r = lane / kPieces + i * kStep;
            const ulonglong2 at = rows[r];
            const bool in = at.x != 0 && e < p.D;
            const uint32_t to = dst + r * (DP * (int)sizeof(T)) + ((c ^ (r & 7)) << 4);
            copy16(to, (const T*)(in ? at.x : (unsigned long long)p.k) + (in ? e : 0), in);
            copy16(to + kTileBytes, (const T*)(in ? at.y : (unsigned long long)p.v) + (in ? e : 0), in);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    const int tiles = max(0, (j1 - j0 + kPagedTile - 1) / kPagedTile);
    const int mine = tiles > warp ? (tiles - warp + kPagedWarps - 1) / kPagedWarps : 0;
#pragma unroll
    for (int n = 0; n < kPagedStages - 1; ++n) {
        if (n < mine) issue(n);
        else asm volatile("cp.async.commit_group;" ::: "memory");
    }
    if (sizeof(T) == 4) {
        for (int i = threadIdx.x; i < nh * DP; i += kPagedThreads) {
            const int g = i / DP, d = i % DP;
            sq[i] = d < p.D ? to_f32(((const T*)p.q)[b * p.qs[0] + (h0 + g) * p.qs[1] + d]) : 0.f;
        }
        __syncthreads();
    }
    PagedAcc<T, DP> acc;
    acc.init(p, b, h0, nh, lane, sq);
    for (int n = 0; n < mine; ++n) {
        __syncwarp();
        if (n + kPagedStages - 1 < mine) issue(n + kPagedStages - 1);
        else asm volatile("cp.async.commit_group;" ::: "memory");
        asm volatile("cp.async.wait_group %0;" ::"n"(kPagedStages - 1) : "memory");
        __syncwarp();
        const uint32_t at = ring + (n % kPagedStages) * 2 * kTileBytes;
        acc.tile(p, at, at + kTileBytes, sm_seen[warp][n % kPagedStages],
                 len - 1 - (j0 + (n * kPagedWarps + warp) * kPagedTile), nh, lane);
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    __syncthreads();                        // the rings become the join's buffer
    float* so = reinterpret_cast<float*>(paged_dyn);
    float* block_o = so + kPagedWarps * kPack * DP;        // the block's own result, read by the cluster
    float2* block_ml = reinterpret_cast<float2*>(block_o + kPack * DP);
    acc.finish(sm_m[warp], sm_l[warp], so + warp * kPack * DP, nh, lane);
    __syncthreads();
    for (int g = warp; g < nh; g += kPagedWarps) {
        float M = -CUDART_INF_F, L = 0.f, f[kPagedWarps];
#pragma unroll
        for (int w = 0; w < kPagedWarps; ++w) M = fmaxf(M, sm_m[w][g]);
        const float base = M == -CUDART_INF_F ? 0.f : M;
#pragma unroll
        for (int w = 0; w < kPagedWarps; ++w) {
            f[w] = ex2(sm_m[w][g] - base);
            L = fmaf(f[w], sm_l[w][g], L);
        }
        const auto joined = [&](int d) {
            float a = 0.f;
#pragma unroll
            for (int w = 0; w < kPagedWarps; ++w) a = fmaf(f[w], so[(w * kPack + g) * DP + d], a);
            return a;
        };
        if constexpr (kCluster) {
            for (int d = lane; d < p.D; d += 32) block_o[g * DP + d] = joined(d);
            if (lane == 0) block_ml[g] = make_float2(M, L);
        } else {
            paged_store<T>(p, b, h0 + g, split, M, L, lane, joined);
        }
    }
    if constexpr (kCluster) {
        // head g of the pack is finished by block g % splits
        cluster_sync_all();
        for (int g = split + warp * p.splits; g < nh; g += kPagedWarps * p.splits) {
            float2 x = make_float2(-CUDART_INF_F, 0.f);
            if (lane < p.splits) x = remote2(cluster_map(smem_u32(&block_ml[g]), lane));
            float M = x.x;
#pragma unroll
            for (int o = 16; o; o /= 2) M = fmaxf(M, __shfl_xor_sync(~0u, M, o));
            const float f = ex2(x.x - (M == -CUDART_INF_F ? 0.f : M));
            float L = f * x.y;
#pragma unroll
            for (int o = 16; o; o /= 2) L += __shfl_xor_sync(~0u, L, o);
            const float inv = L > 0.f ? 1.f / L : L;       // 0: no key; NaN stays
            T* out = (T*)p.out + b * p.os[0] + (h0 + g) * p.os[1];
            for (int d0 = 0; d0 < p.D; d0 += 32) {
                const int d = d0 + lane;
                float a = 0.f;
                for (int s = 0; s < p.splits; ++s) {
                    const float w = __shfl_sync(~0u, f, s);
                    if (d < p.D) a = fmaf(w, remote1(cluster_map(smem_u32(&block_o[g * DP + d]), s)), a);
                }
                if (d < p.D) out[d] = from_f32<T>(a * inv);
            }
            if (lane == 0) p.lse[(int64_t)b * p.H + h0 + g] = paged_lse(p, M, L);
        }
        cluster_sync_all();                  // nobody leaves while its results are read
    }
}

// Joins the chunks of one query head: a block per head, D / 4 lanes to a chunk's
// accumulators. Launched while the chunks are still being read (programmatic
// dependent launch): it waits for them before it touches their results.
constexpr int kJoinThreads = 512;            // at most

template <typename T>
__global__ void __launch_bounds__(kJoinThreads) paged_join_kernel(const __grid_constant__ PagedParams p)
{
    __shared__ float weight[kJoinThreads], red[2][kJoinThreads / 32];
    __shared__ float4 acc[kJoinThreads];
    const int threads = blockDim.x;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int64_t row = blockIdx.x;
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const int b = (int)(row / p.H), h = (int)(row % p.H);
    const int len = paged_length(p, b), chunk = paged_chunk(p, len), n = max(1, (len + chunk - 1) / chunk);
    const float2* st = p.stat + row * p.splits;
    float M = -CUDART_INF_F;
    for (int s = threadIdx.x; s < n; s += threads) M = fmaxf(M, st[s].x);
#pragma unroll
    for (int o = 16; o; o /= 2) M = fmaxf(M, __shfl_xor_sync(~0u, M, o));
    if (lane == 0) red[0][warp] = M;
    __syncthreads();
    for (int w = 0; w < threads / 32; ++w) M = fmaxf(M, red[0][w]);
    const float base = M == -CUDART_INF_F ? 0.f : M;
    // rows of accumulators are read as pieces of four elements where they allow it
    const int width = p.D % 4 ? 1 : 4, lanes = (p.D + width - 1) / width, sets = max(1, threads / lanes);
    const int set = threadIdx.x / lanes, piece = threadIdx.x % lanes;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    float L = 0.f;
    for (int s0 = 0; s0 < n; s0 += threads) {
        __syncthreads();
        const int s = s0 + threadIdx.x;
        float w = 0.f;
        if (s < n) {
            const float2 x = st[s];
            w = p.powers ? ex2(x.x - base) : expf(x.x - base);
            L = fmaf(w, x.y, L);
        }
        weight[threadIdx.x] = w;
        __syncthreads();
        if (set < sets)
#pragma unroll 4
            for (int i = set; i < min(threads, n - s0); i += sets) {
                const float* src = p.part + (row * p.splits + s0 + i) * p.D + piece * width;
                const float f = weight[i];
                if (width == 4) {
                    const float4 v = *reinterpret_cast<const float4*>(src);
                    a.x = fmaf(f, v.x, a.x), a.y = fmaf(f, v.y, a.y), a.z = fmaf(f, v.z, a.z), a.w = fmaf(f, v.w, a.w);
                } else {
                    a.x = fmaf(f, *src, a.x);
                }
            }
    }
#pragma unroll
    for (int o = 16; o; o /= 2) L += __shfl_xor_sync(~0u, L, o);
    if (lane == 0) red[1][warp] = L;
    acc[threadIdx.x] = a;
    __syncthreads();
    L = 0.f;
    for (int w = 0; w < threads / 32; ++w) L += red[1][w];
    const float inv = L > 0.f ? 1.f / L : L;           // 0: no key; NaN stays
    if (set == 0) {
        for (int i = 1; i < sets; ++i) {
            const float4 v = acc[i * lanes + piece];
            a.x += v.x, a.y += v.y, a.z += v.z, a.w += v.w;
        }
        T* out = (T*)p.out + b * p.os[0] + h * p.os[1] + piece * width;
        out[0] = from_f32<T>(a.x * inv);
        if (width == 4) out[1] = from_f32<T>(a.y * inv), out[2] = from_f32<T>(a.z * inv), out[3] = from_f32<T>(a.w * inv);
    }
    if (threadIdx.x == 0) p.lse[row] = paged_lse(p, M, L);
}

}  // namespace mg
