// mg_attention_tc32.cuh -- attention of fp32 tensors on the 5th-generation tensor
// cores at fp32 accuracy.
//
// Each fp32 operand x is the sum of three bf16 numbers, x = x0 + x1 + x2: its 24 bits
// cut into three times 8 (exactly), and a product is the six largest of their nine
// products: x0 y2 + x2 y0 + x1 y1 + x0 y1 + x1 y0 + x0 y0, issued smallest first
// into one fp32 accumulator, so that its truncating additions lose no more than
// those of x0 y0 alone. (The pieces are cut, not rounded, and carry x's sign: what is
// dropped, x1 y2 + x2 y1 + x2 y2, is some 2^-23 of the product, below 2^-21, and
// always taken from its size.) Six products of 16-bit operands cost as
// much as the three of 3xTF32, take 6 bytes of shared memory an element instead
// of 8, and keep fp32's range. An accumulator in tensor memory holds one tile;
// the sum over the tiles is kept in registers (with one accumulator over a long
// row the truncations add up).
//
// Forward: one block per 128 queries of one head: four warps of exponentials
// (thread i: query i), three that load fp32 tiles of 64 keys and values, split
// them and write the pieces to shared memory, one that issues the products. With
// heads of up to 64 two blocks share an SM (96 KB of shared memory and 256 columns
// each), so that one's products run under the other's exponentials. What bounds it is the
// latency of the exponentials' and splits' instructions, not the tensor core.
// Exponentials are taken against the maximum of the tiles before, in one pass
// over the scores; a tile that exceeds it by more than 2^40 is done again.
#pragma once

#include "mg_attention_tc.cuh"

namespace mg {

// Two numbers into their three pieces, the first in the lower half of each word.
__device__ __forceinline__ void split3(float a, float b, uint32_t (&w)[3])
{
    const uint64_t minus = pack2(-1.f, -1.f);
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        const uint32_t x = __float_as_uint(a), y = __float_as_uint(b);
        w[i] = __byte_perm(x, y, 0x7632);
        if (i == 2) break;
        unpack2(fma2(pack2(__uint_as_float(x & 0xFFFF0000u), __uint_as_float(y & 0xFFFF0000u)), minus, pack2(a, b)), a, b);
    }
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
__device__ __forceinline__ void cap_scores32(float (&s)[N], float pre)
{
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = tanh_fast(s[i] * pre);
}

struct Tc32Params {
    AttnParams a;
    const int2* doc_tiles;
    uint32_t idesc_s;            // of S: A negated where the scale is negative
    float scale;                 // |scale|
    RowParts rows;
    int* status;
};

struct Tc32State {
    uint64_t q_full, k_full, v_full, s_full, p_full, o_full, drain;
    uint32_t tmem;
    int failed;
};

// Four warps of exponentials, three that load, one that issues.
constexpr int kTc32LoadWarps = 3;
constexpr int kTc32Threads = (4 + kTc32LoadWarps + 1) * 32;
template <int DP>
constexpr size_t tc32_forward_smem() { return (size_t)(128 + 2 * 64) * DP * 6 + 1024; }

template <int DP, bool kCap, bool kBias>
__global__ void __launch_bounds__(kTc32Threads, DP == 64 ? 2 : 1) attn_tc32_forward(const __grid_constant__ Tc32Params tp)
{
    constexpr uint32_t kPieceQ = 128 * DP * 2, kPieceK = 64 * DP * 2, kColumns = DP == 64 ? 256 : 512;
    extern __shared__ uint8_t dyn[];
    __shared__ Tc32State st;
    const AttnParams& p = tp.a;
    const uint32_t base = (smem_u32(dyn) + 1023u) & ~1023u;
    const uint32_t sQ = base, sK = base + 3 * kPieceQ, sV = sK + 3 * kPieceK;
    const int warp = __shfl_sync(~0u, threadIdx.x / 32, 0), lane = threadIdx.x % 32;   // uniform: so are the roles
    constexpr int kLoadWarp = 4, kMmaWarp = 4 + kTc32LoadWarps;

    const int heads = p.B * p.H, qtiles = (p.Lq + 127) / 128;
    const int part = blockIdx.x % tp.rows.parts, block = blockIdx.x / tp.rows.parts;
    const int qt = qtiles - 1 - block / heads, bh = block % heads;
    const int h = bh % p.H, b = bh / p.H, kv = h / (p.H / p.Hkv);
    const int q0 = qt * 128, shift = p.Lk - p.Lq;
    const int32_t* docs = p.docs ? p.docs + (int64_t)b * p.Lk : nullptr;
    const int2* dt = p.docs ? tp.doc_tiles + (int64_t)b * ((p.Lk + 127) / 128) : nullptr;
    const int prefix = p.prefix ? __ldg(p.prefix + b) : 0;
    const int qlast = min(q0 + 127, p.Lq - 1) + shift;

    if (threadIdx.x == 0) {
        mbar_init(smem_u32(&st.q_full), 4);
        mbar_init(smem_u32(&st.k_full), kTc32LoadWarps);
        mbar_init(smem_u32(&st.v_full), kTc32LoadWarps);
        mbar_init(smem_u32(&st.s_full), 1);
        mbar_init(smem_u32(&st.p_full), 4);
        mbar_init(smem_u32(&st.o_full), 1);
        mbar_init(smem_u32(&st.drain), 1);
        mbar_fence_init();
        st.failed = 0;
    }
    if (warp == kMmaWarp) {
        tmem_alloc(smem_u32(&st.tmem), kColumns);
        tmem_relinquish();
    }
    // Tiles of 64 keys [t0, t1) that a query of this block sees something of.
    int t0 = 0, t1 = ((!p.causal ? p.Lk : max(0, min(p.Lk, max(qlast + 1, prefix)))) + 63) / 64;
    if (docs) narrow_to_docs(dt, p.Lk, 0, 64, docs_of(dt, q0 + shift, 128, p.Lk), t0, t1);
    share_of_row(part, tp.rows.parts, t0, t1);
    const int n = max(0, t1 - t0);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    volatile int* failed = &st.failed;

    if (warp >= kLoadWarp && warp < kMmaWarp) {
        // ------------------------------------------------ loads and splits of keys and values
        // item i of a thread: 8 elements of row r0 + i * kRows, always the same columns
        constexpr int kRows = kTc32LoadWarps * 32 / (DP / 8), kItems = (64 + kRows - 1) / kRows;
        const int tid = threadIdx.x - kLoadWarp * 32, r0 = tid / (DP / 8), c = tid % (DP / 8);
        const bool in = c * 8 < p.D;
        const float* kp = (const float*)p.k + b * p.ks[0] + kv * p.ks[1] + c * 8;
        const float* vp = (const float*)p.v + b * p.vs[0] + kv * p.vs[1] + c * 8;
        const auto fetch = [&](const float* src, int64_t stride, int j, float4 (&x)[kItems][2]) {
            const int row0 = (t0 + j) * 64 + r0;
            const float* at = src + row0 * stride;
#pragma unroll
            for (int i = 0; i < kItems; ++i) {
                const int row = row0 + i * kRows;
                const bool live = in && r0 + i * kRows < 64 && row < p.Lk && (!docs || __ldg(docs + row) >= 0);
                tc32_fetch(x[i], at + i * kRows * stride, live);
            }
        };
        const auto put = [&](uint32_t tile, uint32_t full, const float4 (&x)[kItems][2]) {
#pragma unroll
            for (int i = 0; i < kItems; ++i)
                if (r0 + i * kRows < 64) tc32_put(tile, 64, kPieceK, r0 + i * kRows, c, x[i]);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(full);
        };
        bool ok = true;
        for (int j = 0; j < n; ++j) {
            float4 x[kItems][2];
            fetch(kp, p.ks[2], j, x);
            if (j > 0) ok = __all_sync(~0u, tc_wait(smem_u32(&st.s_full), (j - 1) & 1, failed));
            if (!ok) break;
            put(sK, smem_u32(&st.k_full), x);
            fetch(vp, p.vs[2], j, x);
            if (j > 0) ok = __all_sync(~0u, tc_wait(smem_u32(&st.o_full), (j - 1) & 1, failed));
            if (!ok) break;
            put(sV, smem_u32(&st.v_full), x);
        }
    } else if (warp == kMmaWarp) {
        // ------------------------------------------------ products
        constexpr uint32_t idesc_o = idesc_bf16(128, DP, false, true);
        const uint32_t tS = st.tmem, tP = tS + 64, tO = tS + 160;
        bool ok = n == 0 || __all_sync(~0u, tc_wait(smem_u32(&st.q_full), 0, failed));
        for (int j = 0; j <= n && n > 0 && ok; ++j) {
            if (j > 0) {      // the tile before's part of O: P V
                ok = __all_sync(~0u, tc_wait(smem_u32(&st.v_full), (j - 1) & 1, failed) &&
                                         tc_wait(smem_u32(&st.p_full), (j - 1) & 1, failed));
                if (!ok) break;
                tc_fence_after();
#pragma unroll
                for (int x = 0; x < 6; ++x)
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        tc_mma_f16_ta(tO, tP + kPieceA[x] * 32 + 8 * k, desc_mn_major(sV + kPieceB[x] * kPieceK, 64, k),
                                      idesc_o, x + k > 0);
                tc_commit_warp(smem_u32(&st.o_full));
            }
            if (j < n) {      // S = Q K^T
                ok = __all_sync(~0u, tc_wait(smem_u32(&st.k_full), j & 1, failed));
                if (!ok) break;
                tc_fence_after();
#pragma unroll
                for (int x = 0; x < 6; ++x)
#pragma unroll
                    for (int k = 0; k < DP / 16; ++k)
                        tc_mma_f16(tS, desc_k_major(sQ + kPieceA[x] * kPieceQ, 128, k),
                                   desc_k_major(sK + kPieceB[x] * kPieceK, 64, k), tp.idesc_s, x + k > 0);
                tc_commit_warp(smem_u32(&st.s_full));
            }
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
        // ------------------------------------------------ softmax
        const int tid = threadIdx.x, row = q0 + tid, qpos = row + shift;
        const uint32_t lanes = (uint32_t)warp << 21;
        const uint32_t tS = st.tmem + lanes, tP = tS + 64, tO = tS + 160;
        bool ok = true;
        if (n > 0) {
            const float* qp = (const float*)p.q + b * p.qs[0] + h * p.qs[1];
#pragma unroll
            for (int i0 = 0; i0 < DP / 8; i0 += 8) {
                float4 x[8][2];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int r = ((i0 + i) * 128 + tid) / (DP / 8), c = ((i0 + i) * 128 + tid) % (DP / 8), at = q0 + r;
                    tc32_fetch(x[i], qp + (int64_t)at * p.qs[2] + c * 8,
                               at < p.Lq && c * 8 < p.D && (!docs || doc_at(p, b, at + shift) >= 0));
                }
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    tc32_put(sQ, 128, kPieceQ, ((i0 + i) * 128 + tid) / (DP / 8), ((i0 + i) * 128 + tid) % (DP / 8), x[i]);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&st.q_full));
        }
        const int qdoc = docs ? doc_at(p, b, qpos) : 0;
        const int common = docs ? (q0 + 128 <= p.Lq ? common_doc(dt, q0 + shift, 128, p.Lk) : -1) : 0;
        const int upto = qdoc < 0 ? 0 : !p.causal ? p.Lk : min(p.Lk, max(qpos + 1, prefix));
        // powers of two: a score's is s * mul - slope * distance
        const float mul = kCap ? p.cap * kLog2e : tp.scale * kLog2e, pre = kCap ? tp.scale / p.cap : 0.f;
        const float slope = kBias ? __ldg(p.slopes + h) * kLog2e : 0.f;
        // m: the maximum in use; f: what the output so far is to be multiplied by after the next tile's part is added
        float m = -CUDART_INF_F, l = 0.f, f = 1.f, o[DP];
#pragma unroll
        for (int i = 0; i < DP; ++i) o[i] = 0.f;
        for (int i = 0; i < n; ++i) {
            const int k0 = (t0 + i) * 64;
            bool full = k0 + 64 <= p.Lk && (!p.causal || k0 + 63 <= q0 + shift || k0 + 64 <= prefix);
            if (docs) full = full && common >= 0 && common_doc(dt, k0, 64, p.Lk) == common;
            uint32_t seen[2] = {~0u, ~0u};
            if (!full) {
                if (docs) {
                    const int kdoc[2] = {doc_at(p, b, k0 + lane), doc_at(p, b, k0 + 32 + lane)};
                    same_document(qdoc, kdoc, seen);
                }
                seen[0] &= bits_below(upto - k0);
                seen[1] &= bits_below(upto - k0 - 32);
            }
            const float far = (float)(qpos - k0);
            // columns [c0, c0 + 16): the powers of two less `base`, -inf where masked
            const auto powers = [&](int c0, float base, float (&s)[16]) {
                tmem_ld_x16(tS + c0, s);
                if (kCap) cap_scores32(s, pre);
#pragma unroll
                for (int c = 0; c < 16; c += 2) {
                    float b0 = -base, b1 = -base;
                    if (kBias) {
                        b0 = fmaf(-slope, fabsf(far - (float)(c0 + c)), b0);
                        b1 = fmaf(-slope, fabsf(far - (float)(c0 + c + 1)), b1);
                    }
                    unpack2(fma2(pack2(s[c], s[c + 1]), pack2(mul, mul), pack2(b0, b1)), s[c], s[c + 1]);
                }
                if (full) return;
#pragma unroll
                for (int c = 0; c < 16; ++c) s[c] = seen[c0 / 32] >> (c0 % 32 + c) & 1 ? s[c] : -CUDART_INF_F;
            };
            ok = __all_sync(~0u, tc_wait(smem_u32(&st.s_full), i & 1, failed));
            if (!ok) break;
            tc_fence_after();
            if (i > 0) {             // the tile before's part of the output (complete: it was issued before the scores)
                ok = __all_sync(~0u, tc_wait(smem_u32(&st.o_full), (i - 1) & 1, failed));
                if (!ok) break;
                tc_fence_after();
#pragma unroll
                for (int c0 = 0; c0 < DP; c0 += 32) {
                    float x[32];
                    tmem_ld_x32(tO + c0, x);
#pragma unroll
                    for (int c = 0; c < 32; c += 2)
                        unpack2(mul2(add2(pack2(o[c0 + c], o[c0 + c + 1]), pack2(x[c], x[c + 1])), pack2(f, f)), o[c0 + c],
                                o[c0 + c + 1]);
                }
                f = 1.f;
            }
            float top;               // the tile's maximum, above the one in use
            uint64_t sum;
            if (__any_sync(~0u, m == -CUDART_INF_F)) {       // no maximum to go by yet
                top = -CUDART_INF_F;
#pragma unroll
                for (int c0 = 0; c0 < 64; c0 += 16) {
                    float s[16];
                    powers(c0, 0.f, s);
                    top = fmaxf(top, max_of<16, false>(s));
                }
                m = m == -CUDART_INF_F ? top : m;
            }
            // A pass more suffices for a row far above its maximum in use. With powers beyond 2^29 what
            // rounding leaves of the maximum may itself be above it, whatever is added: hence the limit.
            for (int pass = 0;; ++pass) {
                const float base = m == -CUDART_INF_F ? 0.f : m;
                uint64_t part[2] = {pack2(0.f, 0.f), pack2(0.f, 0.f)};
                top = -CUDART_INF_F;
#pragma unroll
                for (int c0 = 0; c0 < 64; c0 += 16) {
                    float s[16];
                    powers(c0, base, s);
                    top = fmaxf(top, max_of<16, false>(s));
                    uint32_t w[3][8];
#pragma unroll
                    for (int c = 0; c < 16; c += 2) {
                        const float x = ex2(s[c]), y = ex2(s[c + 1]);
                        part[c / 2 % 2] = add2(part[c / 2 % 2], pack2(x, y));
                        uint32_t pc[3];
                        split3(x, y, pc);
#pragma unroll
                        for (int k = 0; k < 3; ++k) w[k][c / 2] = pc[k];
                    }
#pragma unroll
                    for (int k = 0; k < 3; ++k) tmem_st_x8(tP + 32 * k + c0 / 2, w[k]);
                }
                sum = add2(part[0], part[1]);
                // far above the maximum in use: again with its own
                const bool high = top > 40.f;
                if (pass == 2 || !__any_sync(~0u, high)) break;
                if (high) {
                    m = base + top;
                    const float g = ex2(base - m);       // not -top: m is rounded
                    l *= g;
#pragma unroll
                    for (int c = 0; c < DP; ++c) o[c] *= g;
                }
            }
            {
                float x, y;
                unpack2(sum, x, y);
                l += x + y;
            }
            if (top > 8.f) {
                const float up = m + top;
                f = ex2(m - up);
                l *= f;
                m = up;
            }
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&st.p_full));
        }
        if (ok && n > 0) ok = __all_sync(~0u, tc_wait(smem_u32(&st.o_full), (n - 1) & 1, failed));
        if (ok) {
            tc_fence_after();
            if ((l == 0.f && m != -CUDART_INF_F) || l == CUDART_INF_F) l = CUDART_NAN_F;   // scores too large to resolve
            const float g = f * (l > 0.f ? 1.f / l : l);   // 0: no key; NaN stays
            float* out = tp.rows.parts > 1 ? tp.rows.out + (((int64_t)part * p.B * p.H + bh) * p.Lq + row) * p.D
                                           : (float*)p.out + b * p.os[0] + h * p.os[1] + (int64_t)row * p.os[2];
#pragma unroll
            for (int c0 = 0; c0 < DP; c0 += 32) {
                float x[32];
                if (n > 0) {
                    tmem_ld_x32(tO + c0, x);
                } else {
#pragma unroll
                    for (int c = 0; c < 32; ++c) x[c] = 0.f;
                }
                if (row >= p.Lq) continue;
#pragma unroll
                for (int c = 0; c < 32; c += 4)
                    if (c0 + c < p.D) {
                        *reinterpret_cast<float4*>(out + c0 + c) =
                            make_float4((o[c0 + c] + x[c]) * g, (o[c0 + c + 1] + x[c + 1]) * g,
                                        (o[c0 + c + 2] + x[c + 2]) * g, (o[c0 + c + 3] + x[c + 3]) * g);
                    }
            }
            if (row < p.Lq) {
                const float m2 = m == -CUDART_INF_F ? 0.f : m;
                const int64_t at = (int64_t)bh * p.Lq + row;
                if (tp.rows.parts == 1) p.lse[at] = l == 0.f ? -CUDART_INF_F : (m2 + log2f(l)) * kLn2;
                else tp.rows.stat[(int64_t)part * p.B * p.H * p.Lq + at] = make_float2(l == 0.f ? -CUDART_INF_F : m2, l);
            }
        }
        if (!ok && lane == 0) tc_report(tp.status, 222);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == kMmaWarp) tmem_dealloc(st.tmem, kColumns);
}

}  // namespace mg
