// mg_attention_tc32.cuh -- attention of fp32 tensors on the 5th-generation tensor
// cores at fp32 accuracy.
//
// Each fp32 operand x is the sum of three bf16 numbers, x = x0 + x1 + x2, each the
// rounding of what the ones before it leave (8 bits each: all 24 of x), and a
// product is the six of their products that reach 2^-24 of it: x0 y2 + x2 y0 +
// x1 y1 + x0 y1 + x1 y0 + x0 y0, issued smallest first into one fp32 accumulator, so
// that its truncating additions lose no more than those of x0 y0 alone. Six
// products of 16-bit operands cost as much as the three of 3xTF32, take 6 bytes
// of shared memory an element instead of 8, and keep fp32's range. An
// accumulator in tensor memory holds one tile; the sum over the tiles is kept
// in registers (with one accumulator over a long row the truncations add up).
//
// Forward: one block per NQ tiles of 128 queries of one head, one warpgroup to
// each (thread i: query i), one warpgroup that loads fp32 tiles of 64 keys and
// values, splits them and writes the pieces to shared memory, one warp that
// issues the products. A tile's keys and values are split once for the NQ query tiles,
// and the tensor core works on one of them while the other's exponentials are
// taken.
#pragma once

#include "mg_attention_tc.cuh"

namespace mg {

// Two numbers into their three pieces.
__device__ __forceinline__ void split3(float a, float b, uint32_t (&w)[3])
{
    w[0] = bf16x2(a, b);
    a -= __uint_as_float(w[0] << 16);
    b -= __uint_as_float(w[0] & 0xFFFF0000u);
    w[1] = bf16x2(a, b);
    a -= __uint_as_float(w[1] << 16);
    b -= __uint_as_float(w[1] & 0xFFFF0000u);
    w[2] = bf16x2(a, b);
}

// The six products of pieces, smallest first.
__device__ constexpr int kPieceA[6] = {0, 2, 1, 0, 1, 0};
__device__ constexpr int kPieceB[6] = {2, 0, 1, 1, 0, 0};

// An item: 8 elements of a row. Loads them (zeros for rows that are not there or
// are padding) ...
__device__ __forceinline__ void tc32_fetch(float4 (&x)[2], const float* src, bool live)
{
    x[0] = x[1] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (live) {
        x[0] = __ldg(reinterpret_cast<const float4*>(src));
        x[1] = __ldg(reinterpret_cast<const float4*>(src) + 1);
    }
}
// ... and writes their pieces into a tile of `rows` rows (128-byte swizzle; piece i `piece` bytes on).
__device__ __forceinline__ void tc32_put(uint32_t tile, int rows, uint32_t piece, int r, int c, const float4 (&x)[2])
{
    uint32_t w[4][3];
    split3(x[0].x, x[0].y, w[0]);
    split3(x[0].z, x[0].w, w[1]);
    split3(x[1].x, x[1].y, w[2]);
    split3(x[1].z, x[1].w, w[3]);
    const uint32_t at = tile + (uint32_t)(c >> 3) * rows * 128u + r * 128u + (((c & 7) ^ (r & 7)) << 4);
#pragma unroll
    for (int i = 0; i < 3; ++i)
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at + i * piece), "r"(w[0][i]), "r"(w[1][i]),
                     "r"(w[2][i]), "r"(w[3][i])
                     : "memory");
}

// As cap_scores, at fp32 accuracy for every size of score.
template <int N>
__device__ __forceinline__ void cap_scores32(float (&s)[N], float pre, float cap2)
{
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = cap2 * tanh_fast(s[i] * pre);
}

struct Tc32Params {
    AttnParams a;
    const int2* doc_tiles;
    uint32_t idesc_s;            // of S: A negated where the scale is negative
    float scale;                 // |scale|
    int* status;
};

template <int NQ>
struct Tc32State {
    uint64_t q_full[NQ], kv_full[2], kv_empty[2], s_full[NQ], p_full[NQ], o_full[NQ], drain;
    uint32_t tmem;
    int failed;
    int range[NQ][2];
    int qdoc[NQ][2];
    int qpad[NQ];
    alignas(16) int kdoc[NQ * 4][64];
};

template <int DP>
constexpr int tc32_nq() { return DP == 64 ? 2 : 1; }
template <int DP>
constexpr int tc32_stages() { return DP == 64 ? 2 : 1; }
// One warpgroup to each query tile, three warps that load, one that issues: 8 or
// 12 warps, so that a thread may have 255 or 168 registers.
constexpr int kTc32LoadWarps = 3;
template <int DP>
constexpr int tc32_threads() { return tc32_nq<DP>() * 128 + kTc32LoadWarps * 32 + 32; }
template <int DP>
constexpr size_t tc32_forward_smem()
{
    return (size_t)(tc32_nq<DP>() * 128 + tc32_stages<DP>() * 2 * 64) * DP * 6 + 1024;
}

template <int DP, bool kCap, bool kBias>
__global__ void __launch_bounds__(DP == 64 ? 384 : 256, 1) attn_tc32_forward(const __grid_constant__ Tc32Params tp)
{
    constexpr int NQ = DP == 64 ? 2 : 1, kStages = DP == 64 ? 2 : 1;
    constexpr uint32_t kPieceQ = 128 * DP * 2, kPieceK = 64 * DP * 2;
    extern __shared__ uint8_t dyn[];
    __shared__ Tc32State<NQ> st;
    const AttnParams& p = tp.a;
    const uint32_t base = (smem_u32(dyn) + 1023u) & ~1023u;
    const uint32_t sQ = base, sKV = base + NQ * 3 * kPieceQ;
    const int warp = __shfl_sync(~0u, threadIdx.x / 32, 0), lane = threadIdx.x % 32;   // uniform: so are the roles
    constexpr int kLoadWarp = NQ * 4, kMmaWarp = NQ * 4 + kTc32LoadWarps;

    const int heads = p.B * p.H, blocks = (p.Lq + NQ * 128 - 1) / (NQ * 128);
    const int qb = blocks - 1 - blockIdx.x / heads, bh = blockIdx.x % heads;
    const int h = bh % p.H, b = bh / p.H, kv = h / (p.H / p.Hkv);
    const int q0 = qb * NQ * 128, shift = p.Lk - p.Lq;
    const int32_t* docs = p.docs ? p.docs + (int64_t)b * p.Lk : nullptr;
    const int2* dt = p.docs ? tp.doc_tiles + (int64_t)b * ((p.Lk + 127) / 128) : nullptr;
    const int prefix = p.prefix ? __ldg(p.prefix + b) : 0;

    if (threadIdx.x == 0) {
        for (int t = 0; t < NQ; ++t) {
            mbar_init(smem_u32(&st.q_full[t]), 4);
            mbar_init(smem_u32(&st.s_full[t]), 1);
            mbar_init(smem_u32(&st.p_full[t]), 4);
            mbar_init(smem_u32(&st.o_full[t]), 1);
            st.range[t][0] = INT_MAX;
            st.range[t][1] = 0;
            st.qdoc[t][0] = INT_MAX;
            st.qdoc[t][1] = -1;
            st.qpad[t] = 0;
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(smem_u32(&st.kv_full[s]), kTc32LoadWarps);
            mbar_init(smem_u32(&st.kv_empty[s]), 1);
        }
        mbar_init(smem_u32(&st.drain), 1);
        mbar_fence_init();
        st.failed = 0;
    }
    if (warp == kMmaWarp) {
        tmem_alloc(smem_u32(&st.tmem), 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    // Tiles of 64 keys [a, e) that query tile t sees something of.
    int a[NQ], e[NQ];
    for (int t = 0; t < NQ; ++t) {
        const int first = q0 + t * 128, last = min(first + 127, p.Lq - 1) + shift;
        a[t] = 0;
        e[t] = first >= p.Lq ? 0 : ((!p.causal ? p.Lk : max(0, min(p.Lk, max(last + 1, prefix)))) + 63) / 64;
    }
    if (docs) {
        for (int i = threadIdx.x; i < NQ * 128; i += blockDim.x) {
            if (q0 + i >= p.Lq) continue;
            const int d = doc_at(p, b, q0 + i + shift), t = i / 128;
            if (d >= 0) {
                atomicMin(&st.qdoc[t][0], d);
                atomicMax(&st.qdoc[t][1], d);
            } else {
                st.qpad[t] = 1;
            }
        }
        __syncthreads();
        for (int t = 0; t < NQ; ++t)
            for (int i = threadIdx.x; i < e[t]; i += blockDim.x) {
                const int2 r = __ldg(dt + i / 2);
                if (r.x <= st.qdoc[t][1] && r.y >= st.qdoc[t][0]) {
                    atomicMin(&st.range[t][0], i);
                    atomicMax(&st.range[t][1], i + 1);
                }
            }
        __syncthreads();
        for (int t = 0; t < NQ; ++t) {
            a[t] = min(st.range[t][0], st.range[t][1]);
            e[t] = st.range[t][1];
        }
    }
    int lo = INT_MAX, hi = 0;
    for (int t = 0; t < NQ; ++t)
        if (a[t] < e[t]) lo = min(lo, a[t]), hi = max(hi, e[t]);
    lo = min(lo, hi);
    const int n = hi - lo;
    volatile int* failed = &st.failed;
    const auto sK = [&](int j) { return sKV + (uint32_t)(j % kStages) * 6 * kPieceK; };
    const auto sV = [&](int j) { return sK(j) + 3 * kPieceK; };

    if (warp >= kLoadWarp && warp < kMmaWarp) {
        // ------------------------------------------------ loads and splits of keys and values
        constexpr int kLoaders = kTc32LoadWarps * 32, kItems = (64 * (DP / 8) + kLoaders - 1) / kLoaders;
        const int tid = threadIdx.x - kLoadWarp * 32;
        const float* kp = (const float*)p.k + b * p.ks[0] + kv * p.ks[1];
        const float* vp = (const float*)p.v + b * p.vs[0] + kv * p.vs[1];
        const auto fetch = [&](const float* src, int64_t stride, int j, float4 (&x)[kItems][2]) {
#pragma unroll
            for (int i = 0; i < kItems; ++i) {
                const int item = i * kLoaders + tid, r = item / (DP / 8), c = item % (DP / 8), row = (lo + j) * 64 + r;
                const bool live = r < 64 && row < p.Lk && c * 8 < p.D && (!docs || __ldg(docs + row) >= 0);
                tc32_fetch(x[i], src + (int64_t)row * stride + c * 8, live);
            }
        };
        const auto put = [&](uint32_t tile, const float4 (&x)[kItems][2]) {
#pragma unroll
            for (int i = 0; i < kItems; ++i) {
                const int item = i * kLoaders + tid, r = item / (DP / 8), c = item % (DP / 8);
                if (r < 64) tc32_put(tile, 64, kPieceK, r, c, x[i]);
            }
        };
        bool ok = true;
        for (int j = 0; j < n && ok; ++j) {
            float4 x[kItems][2], y[kStages > 1 ? kItems : 1][2];
            fetch(kp, p.ks[2], j, x);
            if constexpr (kStages > 1) fetch(vp, p.vs[2], j, y);
            if (j >= kStages)
                ok = __all_sync(~0u, tc_wait(smem_u32(&st.kv_empty[j % kStages]), (j / kStages - 1) & 1, failed));
            if (!ok) break;
            put(sK(j), x);
            if constexpr (kStages > 1) {
                put(sV(j), y);
            } else {
                fetch(vp, p.vs[2], j, x);
                put(sV(j), x);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&st.kv_full[j % kStages]));
        }
    } else if (warp == kMmaWarp) {
        // ------------------------------------------------ products
        constexpr uint32_t idesc_o = idesc_bf16(128, DP, false, true);
        bool ok = true;
        // S = Q K(j)^T of query tile t
        const auto scores_of = [&](int t, int j) {
            const int first = a[t] - lo;
            if (j < first || j >= e[t] - lo) return;
            ok = ok && tc_wait(smem_u32(&st.kv_full[j % kStages]), (j / kStages) & 1, failed) &&
                 (j > first || tc_wait(smem_u32(&st.q_full[t]), 0, failed)) &&
                 (j == first || tc_wait(smem_u32(&st.p_full[t]), (j - 1 - first) & 1, failed));
            ok = __all_sync(~0u, ok);
            if (!ok) return;
            tc_fence_after();
            {
                const uint32_t q = sQ + t * 3 * kPieceQ;
#pragma unroll
                for (int x = 0; x < 6; ++x)
#pragma unroll
                    for (int k = 0; k < DP / 16; ++k)
                        tc_mma_f16(st.tmem + t * 256, desc_k_major(q + kPieceA[x] * kPieceQ, 128, k),
                                   desc_k_major(sK(j) + kPieceB[x] * kPieceK, 64, k), tp.idesc_s, x + k > 0);
                tc_commit_warp(smem_u32(&st.s_full[t]));
            }
            __syncwarp();
        };
        // this tile's part of O: P V(j)
        const auto output_of = [&](int t, int j) {
            const int first = a[t] - lo;
            if (j < first || j >= e[t] - lo) return;
            ok = __all_sync(~0u, ok && tc_wait(smem_u32(&st.p_full[t]), (j - first) & 1, failed));
            if (!ok) return;
            tc_fence_after();
            {
                const uint32_t tP = st.tmem + t * 256 + 64;
#pragma unroll
                for (int x = 0; x < 6; ++x)
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        tc_mma_f16_ta(tP + 96, tP + kPieceA[x] * 32 + 8 * k,
                                      desc_mn_major(sV(j) + kPieceB[x] * kPieceK, 64, k), idesc_o, x + k > 0);
                tc_commit_warp(smem_u32(&st.o_full[t]));
            }
            __syncwarp();
        };
        for (int j = 0; j <= n && n > 0 && ok; ++j) {
            // with two stages the next scores go before the last output, with one they have to wait for it
            for (int t = 0; t < NQ && ok; ++t) {
                if (kStages > 1 && j < n) scores_of(t, j);
                if (ok && j > 0) output_of(t, j - 1);
            }
            if (ok && j > 0) tc_commit_warp(smem_u32(&st.kv_empty[(j - 1) % kStages]));
            __syncwarp();
            if (kStages == 1 && ok && j < n) scores_of(0, j);
        }
        if (!ok) {
            __syncwarp();
            tc_commit_warp(smem_u32(&st.drain));
            if (lane == 0) {
                tc_report(tp.status, 221);
                tc_drain(smem_u32(&st.drain), 0);
            }
            __syncwarp();
        }
    } else {
        // ------------------------------------------------ softmax of query tile t
        const int t = warp / 4, tid = threadIdx.x % 128, row = q0 + t * 128 + tid, qpos = row + shift;
        const int qfirst = q0 + t * 128;
        const uint32_t lanes = (uint32_t)(warp % 4) << 21;
        const uint32_t tS = st.tmem + t * 256 + lanes, tP = tS + 64, tO = tS + 160;
        const int first = a[t], steps = e[t] - a[t];
        bool ok = true;
        if (steps > 0) {
            const float* qp = (const float*)p.q + b * p.qs[0] + h * p.qs[1];
#pragma unroll 4
            for (int i = 0; i < 128 * (DP / 8) / 128; ++i) {
                const int r = (i * 128 + tid) / (DP / 8), c = (i * 128 + tid) % (DP / 8), at = qfirst + r;
                float4 x[2];
                tc32_fetch(x, qp + (int64_t)at * p.qs[2] + c * 8,
                           at < p.Lq && c * 8 < p.D && (!docs || doc_at(p, b, at + shift) >= 0));
                tc32_put(sQ + t * 3 * kPieceQ, 128, kPieceQ, r, c, x);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&st.q_full[t]));
        }
        const int qdoc = docs ? doc_at(p, b, qpos) : 0;
        const bool one_doc = !docs || (st.qdoc[t][0] == st.qdoc[t][1] && !st.qpad[t] && qfirst + 127 < p.Lq);
        const int upto = qdoc < 0 ? 0 : !p.causal ? p.Lk : min(p.Lk, max(qpos + 1, prefix));
        const float mul = kCap ? 1.f : tp.scale * kLog2e;
        const float slope = kBias ? __ldg(p.slopes + h) * (kCap ? kLog2e : 1.f / tp.scale) : 0.f;
        const float pre = kCap ? tp.scale / p.cap : 0.f, cap2 = p.cap * kLog2e;
        float m = -CUDART_INF_F, l = 0.f, o[DP];
#pragma unroll
        for (int i = 0; i < DP; ++i) o[i] = 0.f;
        for (int i = 0; i < steps; ++i) {
            const int k0 = (first + i) * 64;
            bool full = k0 + 64 <= p.Lk && (!p.causal || k0 + 63 <= qfirst + shift || k0 + 64 <= prefix);
            if (docs) {
                full = full && one_doc && common_doc(dt, k0, 64, p.Lk) == st.qdoc[t][0];
                if (!full) {
                    __syncwarp();
                    st.kdoc[warp][lane] = doc_at(p, b, k0 + lane);
                    st.kdoc[warp][lane + 32] = doc_at(p, b, k0 + 32 + lane);
                    __syncwarp();
                }
            }
            const float far = (float)(qpos - k0);
            const int lim = upto - k0;
            // columns [c0, c0 + 32) of the scores, masked; capped and biased unless `raw`
            const auto scores = [&](int c0, float (&s)[32], bool raw) {
                tmem_ld_x32(tS + c0, s);
                if (kCap && !raw) cap_scores32(s, pre, cap2);
                if (kBias) {
#pragma unroll
                    for (int c = 0; c < 32; ++c) s[c] = fmaf(-slope, fabsf(far - (float)(c0 + c)), s[c]);
                }
                if (!full) {
#pragma unroll
                    for (int c = 0; c < 32; ++c) {
                        bool seen = c0 + c < lim;
                        if (docs) seen = seen && st.kdoc[warp][c0 + c] == qdoc;
                        s[c] = seen ? s[c] : -CUDART_INF_F;
                    }
                }
            };
            ok = __all_sync(~0u, tc_wait(smem_u32(&st.s_full[t]), i & 1, failed));
            if (!ok) break;
            tc_fence_after();
            // the maximum first (a cap alone keeps the order: it is applied to the maximum only)
            constexpr bool kLate = kCap && !kBias;
            float top = -CUDART_INF_F;
#pragma unroll
            for (int c0 = 0; c0 < 64; c0 += 32) {
                float s[32];
                scores(c0, s, kLate);
#pragma unroll
                for (int c = 0; c < 32; ++c) top = fmaxf(top, s[c]);
            }
            if (kLate && top != -CUDART_INF_F) top = cap2 * tanh_fast(top * pre);
            const float mn = fmaxf(m, top);
            const float f = m == -CUDART_INF_F ? 0.f : ex2((m - mn) * mul);
            m = mn;
            l *= f;
            if (i > 0) {             // the tile before's part of the output
                ok = __all_sync(~0u, tc_wait(smem_u32(&st.o_full[t]), (i - 1) & 1, failed));
                if (!ok) break;
                tc_fence_after();
#pragma unroll
                for (int c0 = 0; c0 < DP; c0 += 32) {
                    float x[32];
                    tmem_ld_x32(tO + c0, x);
#pragma unroll
                    for (int c = 0; c < 32; ++c) o[c0 + c] = (o[c0 + c] + x[c]) * f;
                }
            }
            const float base2 = m == -CUDART_INF_F ? 0.f : m * mul;
            float sum = 0.f;
#pragma unroll
            for (int c0 = 0; c0 < 64; c0 += 32) {
                float s[32];
                scores(c0, s, false);
                uint32_t w[3][16];
#pragma unroll
                for (int c = 0; c < 32; c += 2) {
                    const float x = ex2(fmaf(s[c], mul, -base2)), y = ex2(fmaf(s[c + 1], mul, -base2));
                    sum += x + y;
                    uint32_t pc[3];
                    split3(x, y, pc);
#pragma unroll
                    for (int k = 0; k < 3; ++k) w[k][c / 2] = pc[k];
                }
#pragma unroll
                for (int k = 0; k < 3; ++k) tmem_st_x16(tP + 32 * k + c0 / 2, w[k]);
            }
            l += sum;
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&st.p_full[t]));
        }
        if (ok && steps > 0) ok = __all_sync(~0u, tc_wait(smem_u32(&st.o_full[t]), (steps - 1) & 1, failed));
        if (ok) {
            tc_fence_after();
            const float inv = l > 0.f ? 1.f / l : l;
            float* out = (float*)p.out + b * p.os[0] + h * p.os[1] + (int64_t)row * p.os[2];
#pragma unroll
            for (int c0 = 0; c0 < DP; c0 += 32) {
                float x[32];
                if (steps > 0) {
                    tmem_ld_x32(tO + c0, x);
                } else {
#pragma unroll
                    for (int c = 0; c < 32; ++c) x[c] = 0.f;
                }
                if (row >= p.Lq) continue;
#pragma unroll
                for (int c = 0; c < 32; c += 4)
                    if (c0 + c < p.D)
                        *reinterpret_cast<float4*>(out + c0 + c) =
                            make_float4((o[c0 + c] + x[c]) * inv, (o[c0 + c + 1] + x[c + 1]) * inv,
                                        (o[c0 + c + 2] + x[c + 2]) * inv, (o[c0 + c + 3] + x[c + 3]) * inv);
            }
            if (row < p.Lq)
                p.lse[((int64_t)b * p.H + h) * p.Lq + row] =
                    l == 0.f ? -CUDART_INF_F : ((m == -CUDART_INF_F ? 0.f : m * mul) + log2f(l)) * kLn2;
        }
        if (!ok && lane == 0) tc_report(tp.status, 222);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == kMmaWarp) tmem_dealloc(st.tmem, 512);
}

}  // namespace mg
