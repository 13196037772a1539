// mg_attention_tc.cuh -- attention of 16-bit tensors on the 5th-generation
// tensor cores.
//
// Forward: one block per 128 queries of one head; two blocks share an SM. Per
// tile of 128 keys
//     S = Q K^T        (tcgen05, Q and K in shared memory, S in tensor memory)
//     P = exp2(S - m)  (eight warps; warps w and w + 4 have the same 32 queries, a
//                       thread a query, and half of the keys each: no shuffles)
//     O += P V         (tcgen05, P from tensor memory, written over S)
// with the running maximum m of each query in a register. O stays in tensor
// memory; it is rescaled only when a row's maximum has grown by more than 2^8
// since it was last used (P is then at most 2^8, exact in bf16's range, and the
// division by the row sum at the end takes the factor out).
//
// Why this shape: a tile's exponentials take as long as both of its products at
// head_dim 128 (16 a clock and SM: 1024 clocks), so the tensor core has to work on one
// tile while the exponentials of another are taken. Two blocks an SM with one tile
// each do that without any hand-off between them; each needs half of the tensor memory
// (128 columns S, 64 or 128 columns O) and one buffer for K and for V, refilled by TMA as
// soon as its product is done. bf16 [1, 16 over 4, 8192, 128], causal, capped: 384 to 387 us,
// 711 to 716 TFLOP/s. Of a tile pair's 4500 clocks the fp32 pipe is busy 35 %, the exponential
// unit 38 %, the integer pipe 20 % and the tensor pipe 38 %: no unit is full. What bounds it is
// that inside a block scores, exponentials and output follow one another, and only the SM's
// second block fills the gaps.
#pragma once

#include "mg_attention_math.cuh"
#include "mg_tc16.cuh"

namespace mg {

// ---------------------------------------------------------------- documents
// Per 128 positions of a row: the smallest and the largest document id, ids
// below 0 (padding) counted as -1. One warp each.
__global__ void attn_doc_tiles_kernel(const int32_t* __restrict__ docs, int2* __restrict__ tiles, int B, int Lk)
{
    const int per = (Lk + 127) / 128;
    const int64_t t = (int64_t)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32;
    if (t >= (int64_t)B * per) return;
    const int b = (int)(t / per), j0 = (int)(t % per) * 128, lane = threadIdx.x % 32;
    int lo = INT_MAX, hi = -1;
    for (int j = j0 + lane; j < min(Lk, j0 + 128); j += 32) {
        const int d = max(-1, __ldg(docs + (int64_t)b * Lk + j));
        lo = min(lo, d);
        hi = max(hi, d);
    }
    lo = __reduce_min_sync(~0u, lo);
    hi = __reduce_max_sync(~0u, hi);
    if (lane == 0) tiles[t] = make_int2(lo, hi);
}

// The one document that positions [pos, pos + n) have in common by the tiles of
// 128, or -1 (some padding, several documents, positions outside the row).
__device__ __forceinline__ int common_doc(const int2* tiles, int pos, int n, int Lk)
{
    if (pos < 0 || pos + n > Lk) return -1;
    const int2 a = __ldg(tiles + (pos >> 7)), b = __ldg(tiles + ((pos + n - 1) >> 7));
    return a.x == a.y && b.x == b.y && a.x == b.x ? a.x : -1;
}

// Whether a document of positions [pos, pos + n) can be one of `want`'s range.
__device__ __forceinline__ bool docs_meet(const int2* tiles, int pos, int n, int Lk, int2 want)
{
    const int p0 = max(pos, 0), p1 = min(pos + n, Lk);
    for (int t = p0 >> 7; t * 128 < p1; ++t) {
        const int2 r = __ldg(tiles + t);
        if (r.y >= 0 && want.y >= 0 && max(r.x, 0) <= want.y && r.y >= max(want.x, 0)) return true;
    }
    return false;
}

// The span of the documents of positions [pos, pos + n), by the tiles of 128: {0, -1} if there is none.
__device__ __forceinline__ int2 docs_of(const int2* tiles, int pos, int n, int Lk)
{
    int2 m = make_int2(INT_MAX, -1);
    const int p1 = min(pos + n, Lk);
    for (int t = max(pos, 0) >> 7; t * 128 < p1; ++t) {
        const int2 r = __ldg(tiles + t);
        if (r.y >= 0) m = make_int2(min(m.x, max(r.x, 0)), max(m.y, r.y));
    }
    return m;
}

// Narrows tiles [t0, t1) of `step` positions (the first at position pos0) to the
// span of those whose documents meet `want`. Whole warp, the same in every warp.
__device__ __forceinline__ void narrow_to_docs(const int2* tiles, int Lk, int pos0, int step, int2 want, int& t0, int& t1)
{
    const int lane = threadIdx.x % 32;
    int lo = INT_MAX, hi = 0;
    for (int t = t0 + lane; t < t1; t += 32)
        if (docs_meet(tiles, pos0 + t * step, step, Lk, want)) {
            lo = min(lo, t);
            hi = t + 1;
        }
    lo = __reduce_min_sync(~0u, lo);
    t1 = __reduce_max_sync(~0u, hi);
    t0 = min(lo, t1);
}

// ---------------------------------------------------------------- masks
// Masks are words, bit i for column i of 32: tests of single bits of a word cost
// one instruction to several columns, comparisons of positions and documents two to
// three to each (the masked tiles were bound by them).
__device__ __forceinline__ uint32_t bits_below(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u; }

// got[w] bit i: whether theirs[w] of lane i is this thread's document `mine` (below 0:
// none is). One round for each document among the warp's own. Whole warp.
template <int W>
__device__ __forceinline__ void same_document(int mine, const int (&theirs)[W], uint32_t (&got)[W])
{
#pragma unroll
    for (int w = 0; w < W; ++w) got[w] = 0;
    uint32_t todo = __ballot_sync(~0u, mine >= 0);
    while (todo) {
        const int v = __shfl_sync(~0u, mine, __ffs(todo) - 1);
        todo &= ~__ballot_sync(~0u, mine == v);
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const uint32_t m = __ballot_sync(~0u, theirs[w] == v);
            if (mine == v) got[w] = m;
        }
    }
}

// ---------------------------------------------------------------- parameters
struct TcAttnParams {
    CUtensorMap q, k, v;         // {D, rows, heads, batch}, boxes of 64 x 128 rows
    AttnParams a;
    const int2* doc_tiles;       // [B][ceil(Lk / 128)], with documents
    int head_step[3], batch_step[3];   // of q, k, v: 0 where the dim is broadcast (stride 0)
    uint32_t idesc_s;            // of S = Q K^T: A negated where the scale is negative
    float scale;                 // |scale|
    CapCurve curve;
    RowParts rows;
    int* status;
};

struct TcState {
    uint64_t q_full, k_full, v_full, s_full, s_free, p_full[2], o_full, pair[4], drain;
    uint32_t tmem;
    int failed;
    int loads[2];                // tiles of K and of V that were asked for
    float top[2][2][128];        // [tile parity][half][query] maximum of half a row; at the end its sum
};

__device__ __forceinline__ void tc_report(int* status, int where)
{
    if (atomicCAS(status, 0, 5 /* MG_ERR_TIMEOUT */) == 0) status[1] = where;
}

// One 128-row tile, DP columns: DP / 64 boxes.
template <int DP>
__device__ __forceinline__ void tc_load_tile(const CUtensorMap* map, uint32_t bar, uint32_t dst, int rows, int row,
                                             int head, int batch)
{
    mbar_arrive_expect_tx(bar, (uint32_t)rows * DP * 2u);
#pragma unroll
    for (int c = 0; c < DP; c += 64)
        tma_load(map, bar, dst + (uint32_t)(c / 64) * rows * 128u, 4, c, row, head, batch, 0);
}

// Zeroes the rows of padding (documents below 0, or no position at all) of a
// tile that has landed: a product with weight 0 then adds 0 whatever they held. Whole warp.
template <int DP>
__device__ __forceinline__ void tc_clear_padding(uint32_t tile, int rows, const int32_t* docs, int pos0, int Lk, int lane)
{
    for (int r = lane; r < rows; r += 32) {
        const int pos = pos0 + r;
        if (pos >= 0 && pos < Lk && __ldg(docs + pos) >= 0) continue;
#pragma unroll
        for (int c = 0; c < DP / 64; ++c)
#pragma unroll
            for (int x = 0; x < 8; ++x)
                asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(tile + (uint32_t)c * rows * 128u +
                                                                             (uint32_t)r * 128u + x * 16u),
                             "r"(0)
                             : "memory");
    }
    fence_proxy_async_smem();
    __syncwarp();
}

// The block's share of tiles [t0, t1): part of `parts`.
__device__ __forceinline__ void share_of_row(int part, int parts, int& t0, int& t1)
{
    const int each = (max(0, t1 - t0) + parts - 1) / parts;
    t0 += part * each;
    t1 = min(t1, t0 + each);
}

// Joins the parts of each row: with w_s = 2^(m_s - max m) l_s, out = sum w_s out_s / sum w_s.
// One warp to a row, four elements to a lane.
template <typename T>
__global__ void __launch_bounds__(256) attn_join_kernel(const __grid_constant__ AttnParams p, RowParts rows)
{
    const int64_t all = (int64_t)p.B * p.H * p.Lq, at = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) / 32;
    if (at >= all) return;
    const int lane = threadIdx.x % 32;
    float top = -CUDART_INF_F;
    for (int s = 0; s < rows.parts; ++s) top = fmaxf(top, __ldg(rows.stat + s * all + at).x);
    const float base = top == -CUDART_INF_F ? 0.f : top;
    float sum = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    const bool in = lane * 4 < p.D;
    for (int s = 0; s < rows.parts; ++s) {
        const float2 st = __ldg(rows.stat + s * all + at);
        const float w = ex2(st.x - base) * st.y;
        sum += w;
        if (!in || w == 0.f) continue;
        const float4 x = __ldg(reinterpret_cast<const float4*>(rows.out + (s * all + at) * p.D) + lane);
        o.x = fmaf(w, x.x, o.x), o.y = fmaf(w, x.y, o.y), o.z = fmaf(w, x.z, o.z), o.w = fmaf(w, x.w, o.w);
    }
    const float inv = sum > 0.f ? 1.f / sum : sum;      // 0: no key; NaN stays
    const int64_t bh = at / p.Lq;
    const int row = (int)(at - bh * p.Lq), h = (int)(bh % p.H), b = (int)(bh / p.H);
    T* out = (T*)p.out + b * p.os[0] + h * p.os[1] + row * p.os[2] + lane * 4;
    if (in) {
        out[0] = from_f32<T>(o.x * inv), out[1] = from_f32<T>(o.y * inv);
        out[2] = from_f32<T>(o.z * inv), out[3] = from_f32<T>(o.w * inv);
    }
    if (lane == 0) p.lse[at] = sum == 0.f ? -CUDART_INF_F : (base + log2f(sum)) * kLn2;
}

constexpr int kTcFwdThreads = 320;       // eight warps of exponentials, loads, products

template <int DP>
constexpr size_t tc_forward_smem() { return 3 * 128 * DP * 2 + 1024; }

template <int DP, bool kCap, bool kBias>
__global__ void __launch_bounds__(kTcFwdThreads, 2) attn_tc_forward(const __grid_constant__ TcAttnParams tp)
{
    extern __shared__ uint8_t dyn[];
    __shared__ TcState st;
    const AttnParams& p = tp.a;
    const uint32_t base = (smem_u32(dyn) + 1023u) & ~1023u;
    const uint32_t sQ = base, sK = base + 128 * DP * 2, sV = sK + 128 * DP * 2;
    const int warp = __shfl_sync(~0u, threadIdx.x / 32, 0), lane = threadIdx.x % 32;   // uniform: so are the roles

    // blocks with the most keys first
    const int heads = p.B * p.H, qtiles = (p.Lq + 127) / 128;
    const int part = blockIdx.x % tp.rows.parts, block = blockIdx.x / tp.rows.parts;
    const int qt = qtiles - 1 - block / heads, bh = block % heads;
    const int h = bh % p.H, b = bh / p.H, kv = h / (p.H / p.Hkv);
    const int q0 = qt * 128, shift = p.Lk - p.Lq;
    const int32_t* docs = p.docs ? p.docs + (int64_t)b * p.Lk : nullptr;
    const int prefix = p.prefix ? __ldg(p.prefix + b) : 0;
    const int qlast = min(q0 + 127, p.Lq - 1) + shift;

    if (threadIdx.x == 0) {
        mbar_init(smem_u32(&st.q_full), 1);
        mbar_init(smem_u32(&st.k_full), 1);
        mbar_init(smem_u32(&st.v_full), 1);
        mbar_init(smem_u32(&st.s_full), 1);
        mbar_init(smem_u32(&st.s_free), 8);
        mbar_init(smem_u32(&st.p_full[0]), 8);
        mbar_init(smem_u32(&st.p_full[1]), 4);
        mbar_init(smem_u32(&st.o_full), 1);
        for (int i = 0; i < 4; ++i) mbar_init(smem_u32(&st.pair[i]), 2);
        mbar_init(smem_u32(&st.drain), 1);
        mbar_fence_init();
        st.failed = 0;
        st.loads[0] = st.loads[1] = 0;
    }
    if (warp == 9) {
        tmem_alloc(smem_u32(&st.tmem), 256);
        tmem_relinquish();
    }
    // Tiles [t0, t1) hold every key that a query of this block sees.
    const int kend = !p.causal ? p.Lk : max(0, min(p.Lk, max(qlast + 1, prefix)));
    int t0 = 0, t1 = (kend + 127) / 128;
    const int2* dt = docs ? tp.doc_tiles + (int64_t)b * ((p.Lk + 127) / 128) : nullptr;
    if (docs) narrow_to_docs(dt, p.Lk, 0, 128, docs_of(dt, q0 + shift, 128, p.Lk), t0, t1);
    share_of_row(part, tp.rows.parts, t0, t1);
    const int n = max(0, t1 - t0);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    // Scores in columns 0-127. With heads of up to 64 there is room for P beside
    // them, and the next scores are computed while this tile's exponentials are
    // taken; with longer heads P lies over the scores.
    constexpr bool kBeside = DP == 64;
    const uint32_t tS = st.tmem, tP = tS + (kBeside ? 128 : 0), tO = tS + (kBeside ? 192 : 128);
    volatile int* failed = &st.failed;

    if (warp == 8) {
        // ------------------------------------------------ loads
        if (lane == 0 && n > 0) {
            const int hk = kv * tp.head_step[1], bk = b * tp.batch_step[1];
            const int hv = kv * tp.head_step[2], bv = b * tp.batch_step[2];
            tc_load_tile<DP>(&tp.q, smem_u32(&st.q_full), sQ, 128, q0, h * tp.head_step[0], b * tp.batch_step[0]);
            for (int j = 0; j < n; ++j) {
                if (j > 0 && !tc_wait(smem_u32(&st.s_full), (j - 1) & 1, failed)) break;
                tc_load_tile<DP>(&tp.k, smem_u32(&st.k_full), sK, 128, (t0 + j) * 128, hk, bk);
                st.loads[0] = j + 1;
                if (j > 0 && !tc_wait(smem_u32(&st.o_full), (j - 1) & 1, failed)) break;
                tc_load_tile<DP>(&tp.v, smem_u32(&st.v_full), sV, 128, (t0 + j) * 128, hv, bv);
                st.loads[1] = j + 1;
            }
        }
    } else if (warp == 9) {
        // ------------------------------------------------ products
        constexpr uint32_t idesc_o = idesc_bf16(128, DP, false, true);
        bool ok = n == 0 || __all_sync(~0u, tc_wait(smem_u32(&st.q_full), 0, failed));
        const auto scores_of = [&](int j) {       // S = Q K(j)^T
            ok = ok && tc_wait(smem_u32(&st.k_full), j & 1, failed) &&
                 (!kBeside || j == 0 || tc_wait(smem_u32(&st.s_free), (j - 1) & 1, failed));
            ok = __all_sync(~0u, ok);
            if (!ok) return;
            tc_fence_after();
#pragma unroll
            for (int k = 0; k < DP / 16; ++k)
                tc_mma_f16(tS, desc_k_major(sQ, 128, k), desc_k_major(sK, 128, k), tp.idesc_s, k > 0);
            tc_commit_warp(smem_u32(&st.s_full));
        };
        const auto output_of = [&](int j) {       // O += P V(j), half of the keys at a time
            ok = __all_sync(~0u, ok && tc_wait(smem_u32(&st.v_full), j & 1, failed));
            if (!ok) return;
            if (docs && __ldg(&dt[t0 + j]).x < 0) tc_clear_padding<DP>(sV, 128, docs, (t0 + j) * 128, p.Lk, lane);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                ok = __all_sync(~0u, ok && tc_wait(smem_u32(&st.p_full[half]), j & 1, failed));
                if (!ok) return;
                tc_fence_after();
#pragma unroll
                for (int k = 4 * half; k < 4 * half + 4; ++k)
                    tc_mma_f16_ta(tO, tP + 8 * k, desc_mn_major(sV, 128, k), idesc_o, j > 0 || k > 0);
                if (half) tc_commit_warp(smem_u32(&st.o_full));
            }
        };
        for (int j = 0; j <= n && n > 0 && ok; ++j) {
            if (kBeside && j < n) scores_of(j);
            if (ok && j > 0) output_of(j - 1);
            if (!kBeside && ok && j < n) scores_of(j);
        }
        if (!ok) {
            __syncwarp();
            tc_commit_warp(smem_u32(&st.drain));
            if (lane == 0) {
                tc_report(tp.status, 201);
                tc_drain(smem_u32(&st.drain), 0);
            }
            __syncwarp();
        }
    } else {
        // ------------------------------------------------ softmax
        // Warps w and w + 4 have the same 32 queries, each half of the keys.
        const int half = warp / 4, r = threadIdx.x % 128, row = q0 + r, qpos = row + shift;
        const uint32_t lanes = (uint32_t)(warp % 4) << 21;      // this warp's 32 lanes of tensor memory
        const uint32_t pair = smem_u32(&st.pair[warp % 4]);     // where the two warps meet
        const int qdoc = docs ? doc_at(p, b, qpos) : 0;
        const int common = docs ? (q0 + 128 <= p.Lq ? common_doc(dt, q0 + shift, 128, p.Lk) : -1) : 0;
        // keys before `upto` are seen as far as causal and prefix go
        const int upto = qdoc < 0 ? 0 : !p.causal ? p.Lk : min(p.Lk, max(qpos + 1, prefix));
        // scores are kept in units whose multiple by `mul` is the power of two
        const float mul = kCap ? p.cap * kLog2e : tp.scale * kLog2e;
        const float slope = kBias ? __ldg(p.slopes + h) / (kCap ? p.cap : tp.scale) : 0.f;
        float m = -CUDART_INF_F;     // maximum in use; the power of two is m * mul
        uint64_t sum[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[i] = pack2(0.f, 0.f);
        bool ok = true;
        // documents of a tile's keys (this lane's two) and their span, a tile ahead
        int kdoc[2] = {-1, -1};
        int2 span = make_int2(0, 0);
        const auto look_up = [&](int j) {
            const int k0 = (t0 + j) * 128 + 64 * half;
            span = __ldg(dt + t0 + j);
            kdoc[0] = doc_at(p, b, k0 + lane);
            kdoc[1] = doc_at(p, b, k0 + 32 + lane);
        };
        if (docs && n > 0) look_up(0);
        for (int j = 0; j < n; ++j) {
            const int k0 = (t0 + j) * 128 + 64 * half;
            // whether any of the half tile's pairs is masked (same for all threads of the half)
            bool full = k0 + 64 <= p.Lk && (!p.causal || k0 + 63 <= q0 + shift || k0 + 64 <= prefix);
            if (docs) full = full && common >= 0 && span.x == span.y && span.x == common;
            uint32_t seen[2] = {~0u, ~0u};
            if (!full) {
                if (docs) same_document(qdoc, kdoc, seen);
                seen[0] &= bits_below(upto - k0);
                seen[1] &= bits_below(upto - k0 - 32);
            }
            if (docs && j + 1 < n) look_up(j + 1);
            ok = __all_sync(~0u, tc_wait(smem_u32(&st.s_full), j & 1, failed));
            if (!ok) break;
            tc_fence_after();
            float s[64];
            tmem_ld_x64(tS + lanes + 64 * half, s);
            if (kBeside) {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&st.s_free));
            }
            if (kCap) cap_scores(s, tp.curve);
            if (kBias) {
                const float far = (float)(qpos - k0);
#pragma unroll
                for (int c = 0; c < 64; ++c) s[c] = fmaf(-slope, fabsf(far - (float)c), s[c]);
            }
            if (!full) {
#pragma unroll
                for (int c = 0; c < 64; ++c) s[c] = seen[c / 32] >> (c % 32) & 1 ? s[c] : -CUDART_INF_F;
            }
            // the row's maximum; past this barrier both halves have their scores in registers
            const float mine = max_of<64, false>(s);
            st.top[j & 1][half][r] = mine;
            __syncwarp();
            if (lane == 0) mbar_arrive(pair);
            ok = __all_sync(~0u, (j == 0 || tc_wait(smem_u32(&st.o_full), (j - 1) & 1, failed)) &&
                                     tc_wait(pair, j & 1, failed));
            if (!ok) break;
            const float top = fmaxf(mine, st.top[j & 1][half ^ 1][r]);
            // rescale O and the sum where the maximum has outgrown the one in use
            const bool grown = m == -CUDART_INF_F ? top > m : (top - m) * mul > 8.f;
            if (__any_sync(~0u, grown)) {
                const float mn = grown ? top : m;
                if (j > 0) {
                    tc_fence_after();
                    // by the rounded powers of two that P is taken against
                    const float f = m == -CUDART_INF_F ? 0.f : ex2(__fmul_rn(m, mul) - __fmul_rn(mn, mul));
#pragma unroll 1
                    for (int c = half * (DP / 2); c < (half + 1) * (DP / 2); c += 16) {
                        float o[16];
                        uint32_t w[16];
                        tmem_ld_x16(tO + lanes + c, o);
#pragma unroll
                        for (int i = 0; i < 16; ++i) w[i] = __float_as_uint(o[i] * f);
                        tmem_st_x16(tO + lanes + c, w);
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) sum[i] = mul2(sum[i], pack2(f, f));
                    tmem_wait_st();
                }
                m = mn;
            }
            if (half) {              // O may be added to as far as this half goes
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&st.p_full[0]));
            }
            const float base2 = m == -CUDART_INF_F ? 0.f : __fmul_rn(m, mul);
            const uint64_t mul_2 = pack2(mul, mul), base_2 = pack2(-base2, -base2);
#pragma unroll
            for (int c = 0; c < 64; c += 32) {
                uint32_t w[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    float x, y;
                    unpack2(fma2(pack2(s[c + 2 * i], s[c + 2 * i + 1]), mul_2, base_2), x, y);
                    x = ex2(x);
                    y = ex2(y);
                    sum[i % 4] = add2(sum[i % 4], pack2(x, y));
                    w[i] = bf16x2(x, y);
                }
                tmem_st_x16(tP + lanes + 32 * half + c / 2, w);
            }
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&st.p_full[half]));
        }
        float l, lb;
        unpack2(add2(add2(sum[0], sum[1]), add2(sum[2], sum[3])), l, lb);
        st.top[n & 1][half][r] = l + lb;
        __syncwarp();
        if (lane == 0) mbar_arrive(pair);
        ok = ok && (n == 0 || tc_wait(smem_u32(&st.o_full), (n - 1) & 1, failed)) && tc_wait(pair, n & 1, failed);
        ok = __all_sync(~0u, ok);
        if (ok) {
            tc_fence_after();
            l = st.top[n & 1][0][r] + st.top[n & 1][1][r];
            if ((l == 0.f && m != -CUDART_INF_F) || l == CUDART_INF_F) l = CUDART_NAN_F;   // scores too large to resolve
            const float inv = l > 0.f ? 1.f / l : l;       // 0: no key; NaN stays
            const bool store = row < p.Lq;
            __nv_bfloat16* out = (__nv_bfloat16*)p.out + b * p.os[0] + h * p.os[1] + (int64_t)row * p.os[2];
            const int c1 = min(p.D, (half + 1) * (DP / 2));
#pragma unroll 1
            for (int c = half * (DP / 2); c < c1; c += 32) {
                float o[32];
                if (n > 0) {
                    tmem_ld_x32(tO + lanes + c, o);
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = 0.f;
                }
                if (!store) continue;
                if (tp.rows.parts > 1) {
                    float* to = tp.rows.out + (((int64_t)part * p.B * p.H + bh) * p.Lq + row) * p.D + c;
#pragma unroll
                    for (int i = 0; i < 32; i += 4)
                        if (c + i + 4 <= c1)
                            *reinterpret_cast<float4*>(to + i) =
                                make_float4(o[i] * inv, o[i + 1] * inv, o[i + 2] * inv, o[i + 3] * inv);
                    continue;
                }
#pragma unroll
                for (int i = 0; i < 32; i += 8)
                    if (c + i + 8 <= c1)
                        *reinterpret_cast<uint4*>(out + c + i) =
                            make_uint4(bf16x2(o[i] * inv, o[i + 1] * inv), bf16x2(o[i + 2] * inv, o[i + 3] * inv),
                                       bf16x2(o[i + 4] * inv, o[i + 5] * inv), bf16x2(o[i + 6] * inv, o[i + 7] * inv));
            }
            if (store && half == 0) {
                const float m2 = m == -CUDART_INF_F ? 0.f : __fmul_rn(m, mul);
                const int64_t at = (int64_t)bh * p.Lq + row;
                if (tp.rows.parts == 1) p.lse[at] = l == 0.f ? -CUDART_INF_F : (m2 + log2f(l)) * kLn2;
                else tp.rows.stat[(int64_t)part * p.B * p.H * p.Lq + at] = make_float2(l == 0.f ? -CUDART_INF_F : m2, l);
            }
        }
        if (!ok && lane == 0) tc_report(tp.status, 202);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (st.failed && threadIdx.x == 0 && n > 0) {     // copies that nobody waited for
        tc_drain(smem_u32(&st.q_full), 0);
        if (st.loads[0]) tc_drain(smem_u32(&st.k_full), (st.loads[0] - 1) & 1);
        if (st.loads[1]) tc_drain(smem_u32(&st.v_full), (st.loads[1] - 1) & 1);
    }
    if (warp == 9) tmem_dealloc(st.tmem, 256);
}

}  // namespace mg
