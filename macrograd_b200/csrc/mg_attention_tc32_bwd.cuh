// mg_attention_tc32_bwd.cuh -- gradients of attention of fp32 tensors on the
// 5th-generation tensor cores at fp32 accuracy.
//
// The two forms of mg_attention_tc_bwd.cuh (queries resident: dQ; keys resident:
// dK, dV), with every product made of the six of mg_attention_tc32.cuh. Two
// warpgroups share a tile of kN streamed rows: warpgroup g has half of the columns of S and
// dP, writes the pieces of its part of P and dS to tensor memory, and adds its
// share of each tile's accumulators up in registers. The tensor core runs S and dP of
// the next tile while the exponentials of this one are taken.
//
// P = exp2(S - lse) carries the rounding of the fp32 lse, 2^-24 |lse|, and that of lse log2(e)
// (gradients off by 1e-6 to 2.7e-6 with |lse| of 25 to 50). Both are the same for a whole row: the
// form with the queries resident, which runs first, adds up each row's P, divides dQ by the sum, and
// leaves its logarithm for the other form to take off the exponents.
//
// Heads of up to 64: the pieces of 128 resident rows and of two stages of kN = 64
// streamed rows of two tensors fill the shared memory (96 + 96 KB).
// Heads of up to 128: X0's pieces lie in tensor memory (3 x 64 columns, the A operand
// of S), kN = 32, and one accumulator of 128 columns is all that is left, so dK and
// dV take a launch each (8 products in all instead of 7).
#pragma once

#include "mg_attention_tc32.cuh"
#include "mg_attention_tc_bwd.cuh"

namespace mg {

struct Tc32BwdParams {
    AttnParams a;
    const int2* doc_tiles;
    const float* lse2;           // as TcBwdParams
    const float* delta;
    float* fine;                 // [B * H][Lp] log2 of the row's sum of exp2(S - lse2), from the form with the queries resident
    int Lp;
    uint32_t idesc_s;
    float scale;                 // |scale|
    int* status;
    GradParts parts;
};

// What a launch accumulates: dS Y0 (dQ or dK), P Y1 (dV), or both.
enum : int { kTakeBoth = 0, kTakeDs = 1, kTakeP = 2 };

struct Tc32BwdState {
    uint64_t x_full, y_full[2], y_empty[2], s_full, s_free, p_full, acc_full, sum_full, drain;
    uint32_t tmem;
    int failed;
    alignas(16) float lse2[2][64];       // negated
    alignas(16) float delta[2][64];      // negated
    alignas(16) float fine[2][64];       // negated
};

constexpr int kTc32BwdThreads = 384;     // two warpgroups, three warps that load, one that issues
constexpr size_t kTc32BwdSmem = (size_t)(2 * 128 + 2 * 2 * 64) * 64 * 6 + 1024;
static_assert(kTc32BwdSmem == (size_t)(128 + 2 * 2 * 32) * 128 * 6 + 1024, "both head sizes take the same");
// With a KB of the system's own: beyond 196 KB the SM gives shared memory 228, and L1 half of what it had (dQ 84 -> 90 us).
static_assert(kTc32BwdSmem + sizeof(Tc32BwdState) + 1024 <= 196 * 1024, "the L1's share");

template <int DP, bool kKeys, int kTake, bool kCap, bool kBias>
__global__ void __launch_bounds__(kTc32BwdThreads, 1) attn_tc32_backward(const __grid_constant__ Tc32BwdParams tp)
{
    constexpr bool kXt = DP == 128;                  // X0 in tensor memory
    constexpr int kN = kXt ? 32 : 64;                // streamed rows of a tile
    constexpr int kCols = kN / 2;                    // of them, a thread's
    static_assert(kTake != kTakeBoth || (kKeys && !kXt), "two accumulators: keys resident, heads of up to 64");
    static_assert(kTake != kTakeP || kKeys, "dV needs the keys resident");
    constexpr uint32_t kPieceX = 128 * DP * 2, kPieceY = kN * DP * 2;
    extern __shared__ uint8_t dyn[];
    __shared__ Tc32BwdState st;
    const AttnParams& p = tp.a;
    const uint32_t base = (smem_u32(dyn) + 1023u) & ~1023u;
    const uint32_t sX0 = base, sX1 = base + (kXt ? 0 : 3 * kPieceX), sY = sX1 + 3 * kPieceX;
    const int warp = __shfl_sync(~0u, threadIdx.x / 32, 0), lane = threadIdx.x % 32;   // uniform: so are the roles

    const int nhead = kKeys ? p.Hkv : p.H, xrows = kKeys ? p.Lk : p.Lq, yrows = kKeys ? p.Lq : p.Lk;
    const int xtiles = (xrows + 127) / 128, part = blockIdx.x % tp.parts.parts, block = blockIdx.x / tp.parts.parts;
    const int bh = block % (p.B * nhead), rank = block / (p.B * nhead);
    const int x0 = (kKeys ? rank : xtiles - 1 - rank) * 128;
    const int xh = bh % nhead, b = bh / nhead, group = p.H / p.Hkv;
    const int shift = p.Lk - p.Lq;
    const int32_t* docs = p.docs ? p.docs + (int64_t)b * p.Lk : nullptr;
    const int2* dt = p.docs ? tp.doc_tiles + (int64_t)b * ((p.Lk + 127) / 128) : nullptr;
    const int prefix = p.prefix ? __ldg(p.prefix + b) : 0;
    const int xpos = kKeys ? x0 : x0 + shift;

    if (threadIdx.x == 0) {
        mbar_init(smem_u32(&st.x_full), 8);
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&st.y_full[i]), kTc32LoadWarps);
            mbar_init(smem_u32(&st.y_empty[i]), 1);
        }
        mbar_init(smem_u32(&st.s_full), 1);
        mbar_init(smem_u32(&st.s_free), 8);
        mbar_init(smem_u32(&st.p_full), 8);
        mbar_init(smem_u32(&st.acc_full), 1);
        mbar_init(smem_u32(&st.sum_full), 8);
        mbar_init(smem_u32(&st.drain), 1);
        mbar_fence_init();
        st.failed = 0;
    }
    if (warp == 11) {
        tmem_alloc(smem_u32(&st.tmem), 512);
        tmem_relinquish();
    }
    int t0, t1;
    stream_range<kKeys>(p, docs, dt, prefix, x0, xpos, shift, t0, t1);
    t0 *= 64 / kN, t1 *= 64 / kN;
    int i0, n;                                       // the block's share of the steps
    const int tiles = max(0, t1 - t0);
    share_of_steps(part, tp.parts.parts, kKeys ? tiles * group : tiles, i0, n);
    if (!kKeys) t0 += i0;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    // columns: X0's pieces, S, dP, the pieces of P and of dS, the accumulators
    const uint32_t tX = st.tmem, tS = tX + (kXt ? 192 : 0), tdP = tS + kN, tP = tdP + kN;
    const uint32_t tdS = tP + (kXt ? 0 : 96), tA = st.tmem + (kXt ? 384 : 320), tB = tA + (kXt ? 0 : 64);
    volatile int* failed = &st.failed;
    const auto sY0 = [&](int i) { return sY + (uint32_t)(i & 1) * 6 * kPieceY; };

    if (warp >= 8 && warp < 11) {
        // ------------------------------------------------ loads and splits of the streamed rows
        // item k of a thread: 8 elements of row r0 + k * kRows of both tensors, always the same columns
        constexpr int kRows = kTc32LoadWarps * 32 / (DP / 8), kItems = (kN + kRows - 1) / kRows;
        const int tid = threadIdx.x - 256, r0 = tid / (DP / 8), c = tid % (DP / 8);
        const bool in = c * 8 < p.D;
        const int64_t* s0 = kKeys ? p.qs : p.ks;
        const int64_t* s1 = kKeys ? p.dos : p.vs;
        const float* src0 = (const float*)(kKeys ? p.q : p.k) + b * s0[0] + c * 8;
        const float* src1 = (const float*)(kKeys ? p.dout : p.v) + b * s1[0] + c * 8;
        const int64_t step0 = s0[2], step1 = s1[2];
        bool ok = true;
        for (int i = 0; i < n && ok; ++i) {
            const int yh = kKeys ? xh * group + (i0 + i) / tiles : xh / group;
            const int y0 = (t0 + (kKeys ? (i0 + i) % tiles : i)) * kN;
            const float* a0 = src0 + yh * s0[1] + (y0 + r0) * step0;
            const float* a1 = src1 + yh * s1[1] + (y0 + r0) * step1;
            float4 x[kItems][2], y[kItems][2];
#pragma unroll
            for (int k = 0; k < kItems; ++k) {
                const int row = y0 + r0 + k * kRows;
                const bool live = in && r0 + k * kRows < kN && row < yrows &&
                                  (!docs || doc_at(p, b, row + (kKeys ? shift : 0)) >= 0);
                tc32_fetch(x[k], a0 + k * kRows * step0, live);
                tc32_fetch(y[k], a1 + k * kRows * step1, live);
            }
            float lse2 = 0.f, delta = 0.f, fine = 0.f;
            if (kKeys && tid < kN) {
                const int64_t at = ((int64_t)b * p.H + yh) * tp.Lp + y0 + tid;
                lse2 = tp.lse2[at];
                delta = tp.delta[at];
                if (y0 + tid < p.Lq) fine = tp.fine[at];
            }
            if (i >= 2) ok = __all_sync(~0u, tc_wait(smem_u32(&st.y_empty[i & 1]), (i / 2 - 1) & 1, failed));
            if (!ok) break;
#pragma unroll
            for (int k = 0; k < kItems; ++k) {
                if (r0 + k * kRows >= kN) continue;
                tc32_put(sY0(i), kN, kPieceY, r0 + k * kRows, c, x[k]);
                tc32_put(sY0(i) + 3 * kPieceY, kN, kPieceY, r0 + k * kRows, c, y[k]);
            }
            if (kKeys && tid < kN) {
                st.lse2[i & 1][tid] = -lse2;
                st.delta[i & 1][tid] = -delta;
                st.fine[i & 1][tid] = -fine;
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&st.y_full[i & 1]));
        }
    } else if (warp == 11) {
        // ------------------------------------------------ products
        constexpr uint32_t idesc_dp = idesc_bf16(128, kN, false, false), idesc_acc = idesc_bf16(128, DP, false, true);
        bool ok = true;
        for (int i = 0; i <= n && n > 0 && ok; ++i) {
            if (i < n) {
                ok = tc_wait(smem_u32(&st.y_full[i & 1]), (i >> 1) & 1, failed) &&
                     (i > 0 ? tc_wait(smem_u32(&st.s_free), (i - 1) & 1, failed)
                            : tc_wait(smem_u32(&st.x_full), 0, failed));
                ok = __all_sync(~0u, ok);
                if (!ok) break;
                tc_fence_after();
#pragma unroll
                for (int x = 0; x < 6; ++x)
#pragma unroll
                    for (int k = 0; k < DP / 16; ++k) {
                        const uint64_t y = desc_k_major(sY0(i) + kPieceB[x] * kPieceY, kN, k);
                        if constexpr (kXt) tc_mma_f16_ta(tS, tX + kPieceA[x] * 64 + 8 * k, y, tp.idesc_s, x + k > 0);
                        else tc_mma_f16(tS, desc_k_major(sX0 + kPieceA[x] * kPieceX, 128, k), y, tp.idesc_s, x + k > 0);
                    }
                if constexpr (kTake != kTakeP) {
#pragma unroll
                    for (int x = 0; x < 6; ++x)
#pragma unroll
                        for (int k = 0; k < DP / 16; ++k)
                            tc_mma_f16(tdP, desc_k_major(sX1 + kPieceA[x] * kPieceX, 128, k),
                                       desc_k_major(sY0(i) + (3 + kPieceB[x]) * kPieceY, kN, k), idesc_dp, x + k > 0);
                }
                tc_commit_warp(smem_u32(&st.s_full));
            }
            if (i > 0) {
                const int j = i - 1;
                ok = __all_sync(~0u, tc_wait(smem_u32(&st.p_full), j & 1, failed));
                if (!ok) break;
                tc_fence_after();
                if constexpr (kTake != kTakeDs) {
#pragma unroll
                    for (int x = 0; x < 6; ++x)
#pragma unroll
                        for (int k = 0; k < kN / 16; ++k)
                            tc_mma_f16_ta(tB, tP + kPieceA[x] * kCols + 8 * k,
                                          desc_mn_major(sY0(j) + (3 + kPieceB[x]) * kPieceY, kN, k), idesc_acc,
                                          x + k > 0);
                }
                if constexpr (kTake != kTakeP) {
#pragma unroll
                    for (int x = 0; x < 6; ++x)
#pragma unroll
                        for (int k = 0; k < kN / 16; ++k)
                            tc_mma_f16_ta(tA, tdS + kPieceA[x] * kCols + 8 * k,
                                          desc_mn_major(sY0(j) + kPieceB[x] * kPieceY, kN, k), idesc_acc, x + k > 0);
                }
                tc_commit_warp(smem_u32(&st.acc_full));
                tc_commit_warp(smem_u32(&st.y_empty[j & 1]));
            }
        }
        if (!ok) {
            __syncwarp();
            tc_commit_warp(smem_u32(&st.drain));
            if (lane == 0) {
                tc_report(tp.status, 231);
                tc_drain(smem_u32(&st.drain), 0);
            }
            __syncwarp();
        }
    } else {
        // ------------------------------------------------ P and dS
        const int wg = warp / 4, r = threadIdx.x % 128, col = kCols * wg;    // resident row, first column
        const uint32_t lanes = (uint32_t)(warp % 4) << 21;
        const int pos = xpos + r;
        bool ok = true;
        if (n > 0) {
            const int64_t* s = kKeys ? (wg ? p.vs : p.ks) : (wg ? p.dos : p.qs);
            const float* src = (const float*)(kKeys ? (wg ? p.v : p.k) : (wg ? p.dout : p.q)) + b * s[0] + xh * s[1];
            if (kXt && wg == 0) {
                // this thread's row of X0 into its lane of tensor memory, two elements to a column
                const int row = x0 + r;
                const bool live = row < xrows && (!docs || doc_at(p, b, row + (kKeys ? 0 : shift)) >= 0);
#pragma unroll 1
                for (int c = 0; c < DP; c += 32) {
                    uint32_t w[3][16];
#pragma unroll
                    for (int e = 0; e < 32; e += 8) {
                        float4 x[2];
                        tc32_fetch(x, src + row * s[2] + c + e, live && c + e < p.D);
                        uint32_t pc[4][3];
                        split3(x[0].x, x[0].y, pc[0]);
                        split3(x[0].z, x[0].w, pc[1]);
                        split3(x[1].x, x[1].y, pc[2]);
                        split3(x[1].z, x[1].w, pc[3]);
#pragma unroll
                        for (int k = 0; k < 4; ++k)
#pragma unroll
                            for (int z = 0; z < 3; ++z) w[z][e / 2 + k] = pc[k][z];
                    }
#pragma unroll
                    for (int z = 0; z < 3; ++z) tmem_st_x16(tX + lanes + 64 * z + c / 2, w[z]);
                }
                tmem_wait_st();
                tc_fence_before();
            } else if (!kXt || kTake != kTakeP) {
#pragma unroll 1
                for (int first = 0; first < DP / 8; first += 8) {
                    float4 x[8][2];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int item = (first + i) * 128 + r, row = x0 + item / (DP / 8), e = item % (DP / 8);
                        tc32_fetch(x[i], src + row * s[2] + e * 8,
                                   row < xrows && e * 8 < p.D && (!docs || doc_at(p, b, row + (kKeys ? 0 : shift)) >= 0));
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int item = (first + i) * 128 + r;
                        tc32_put(wg ? sX1 : sX0, 128, kPieceX, item / (DP / 8), item % (DP / 8), x[i]);
                    }
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&st.x_full));
        }
        const int rdoc = docs ? (x0 + r < xrows ? doc_at(p, b, pos) : -1) : 0;
        const int common = docs ? (x0 + 128 <= xrows ? common_doc(dt, xpos, 128, p.Lk) : -1) : 0;
        const float mul = kCap ? p.cap * kLog2e : tp.scale * kLog2e, pre = kCap ? tp.scale / p.cap : 0.f;
        float lse2 = 0.f, delta = 0.f;
        if (!kKeys) {
            const int64_t at = ((int64_t)b * p.H + xh) * tp.Lp + x0 + r;
            lse2 = -tp.lse2[at];
            delta = -tp.delta[at];
        }
        // this thread's part of its row's accumulators: dK (warpgroup 0) or dV (1), or half of the only one
        constexpr int kAcc = kTake == kTakeBoth ? DP : DP / 2;
        const int ocol = kTake == kTakeBoth ? 0 : kAcc * wg;
        const bool is_dv = kTake == kTakeP || (kTake == kTakeBoth && wg == 1);
        const uint32_t tAcc = (is_dv ? tB : tA) + ocol + lanes;
        float o[kAcc];
#pragma unroll
        for (int i = 0; i < kAcc; ++i) o[i] = 0.f;
        uint64_t psum = pack2(0.f, 0.f);                // this thread's part of its row's sum of P
        const auto add_up = [&]() {
#pragma unroll
            for (int c = 0; c < kAcc; c += 32) {
                float x[32];
                tmem_ld_x32(tAcc + c, x);
#pragma unroll
                for (int k = 0; k < 32; k += 2)
                    unpack2(add2(pack2(o[c + k], o[c + k + 1]), pack2(x[k], x[k + 1])), o[c + k], o[c + k + 1]);
            }
        };
        // this lane's document of a tile's streamed rows, a tile ahead
        const auto y_of = [&](int i) { return (t0 + (kKeys ? (i0 + i) % tiles : i)) * kN; };
        int ydoc[1] = {docs && n > 0 ? doc_at(p, b, y_of(0) + (kKeys ? shift : 0) + col + lane) : -1};
        for (int i = 0; i < n; ++i) {
            const int h = kKeys ? xh * group + (i0 + i) / tiles : xh;
            const int y0 = y_of(i), ypos = y0 + (kKeys ? shift : 0);
            const float slope = kBias ? __ldg(p.slopes + h) * kLog2e : 0.f;
            bool full;
            uint32_t seen[1] = {~0u};
            if (kKeys) full = !p.causal || ypos >= xpos + 127 || xpos + 128 <= prefix;
            else full = ypos + kN <= p.Lk && (!p.causal || ypos + kN - 1 <= xpos || ypos + kN <= prefix);
            if (docs) full = full && common >= 0 && (!kKeys || y0 + kN <= p.Lq) && common_doc(dt, ypos, kN, p.Lk) == common;
            if (!full) {
                if (docs) same_document(rdoc, ydoc, seen);
                if (!kKeys) seen[0] &= bits_below((!p.causal ? p.Lk : min(p.Lk, max(pos + 1, prefix))) - ypos - col);
                else if (p.causal && pos >= prefix) seen[0] &= ~bits_below(pos - ypos - col);
            }
            if (docs && i + 1 < n) ydoc[0] = doc_at(p, b, y_of(i + 1) + (kKeys ? shift : 0) + col + lane);
            ok = __all_sync(~0u, tc_wait(smem_u32(&st.s_full), i & 1, failed) &&
                                     (!kKeys || tc_wait(smem_u32(&st.y_full[i & 1]), (i >> 1) & 1, failed)));
            if (!ok) break;
            tc_fence_after();
            float v[kCols], g[kCols];
#pragma unroll
            for (int c0 = 0; c0 < kCols; c0 += 16) {
                tmem_ld_x16(tS + lanes + col + c0, *reinterpret_cast<float(*)[16]>(v + c0));
                if (kTake != kTakeP) tmem_ld_x16(tdP + lanes + col + c0, *reinterpret_cast<float(*)[16]>(g + c0));
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&st.s_free));
            if (i > 0) {
                ok = __all_sync(~0u, tc_wait(smem_u32(&st.acc_full), (i - 1) & 1, failed));
                if (!ok) break;
                tc_fence_after();
                add_up();
            }
            if (kCap) cap_scores32(v, pre);
            const float far = (float)(pos - ypos - col);
            const uint64_t mul_2 = pack2(mul, mul);
            uint64_t tsum = pack2(0.f, 0.f);            // of this tile: long rows add up tiles, not pairs
#pragma unroll
            for (int c0 = 0; c0 < kCols; c0 += 16) {
                float e[16];
#pragma unroll
                for (int c = 0; c < 16; c += 4) {
                    float nl[4] = {lse2, lse2, lse2, lse2};
                    if (kKeys) {
                        const float4 x = *reinterpret_cast<const float4*>(&st.lse2[i & 1][col + c0 + c]);
                        nl[0] = x.x, nl[1] = x.y, nl[2] = x.z, nl[3] = x.w;
                    }
                    if (kBias) {
#pragma unroll
                        for (int k = 0; k < 4; ++k) nl[k] = fmaf(-slope, fabsf(far - (float)(c0 + c + k)), nl[k]);
                    }
#pragma unroll
                    for (int k = 0; k < 4; k += 2) {
                        uint64_t x = fma2(pack2(v[c0 + c + k], v[c0 + c + k + 1]), mul_2, pack2(nl[k], nl[k + 1]));
                        if (kKeys) x = add2(x, *reinterpret_cast<const uint64_t*>(&st.fine[i & 1][col + c0 + c + k]));
                        unpack2(x, e[c + k], e[c + k + 1]);
                        e[c + k] = ex2(e[c + k]);
                        e[c + k + 1] = ex2(e[c + k + 1]);
                    }
                }
                if (!full) {
                    // a pair that is not seen: P = 0, and its dP does not count
#pragma unroll
                    for (int c = 0; c < 16; ++c) e[c] = seen[0] >> (c0 + c) & 1 ? e[c] : 0.f;
                }
                if (!kKeys) {
#pragma unroll
                    for (int c = 0; c < 16; c += 2) tsum = add2(tsum, pack2(e[c], e[c + 1]));
                }
                if (kTake != kTakeDs) {
                    uint32_t w[3][8];
#pragma unroll
                    for (int c = 0; c < 16; c += 2) {
                        uint32_t pc[3];
                        split3(e[c], e[c + 1], pc);
#pragma unroll
                        for (int k = 0; k < 3; ++k) w[k][c / 2] = pc[k];
                    }
#pragma unroll
                    for (int k = 0; k < 3; ++k) tmem_st_x8(tP + lanes + kCols * k + (col + c0) / 2, w[k]);
                }
                if constexpr (kTake != kTakeP) {
                    // dS = P * curve * (dP - delta)
                    uint32_t w[3][8];
#pragma unroll
                    for (int c = 0; c < 16; c += 4) {
                        float nd[4] = {delta, delta, delta, delta};
                        if (kKeys) {
                            const float4 x = *reinterpret_cast<const float4*>(&st.delta[i & 1][col + c0 + c]);
                            nd[0] = x.x, nd[1] = x.y, nd[2] = x.z, nd[3] = x.w;
                        }
#pragma unroll
                        for (int k = 0; k < 4; k += 2) {
                            const int at = c0 + c + k;
                            uint64_t q = pack2(e[c + k], e[c + k + 1]);
                            if (kCap) {
                                const uint64_t t = pack2(v[at], v[at + 1]);
                                q = mul2(q, fma2(mul2(t, pack2(-1.f, -1.f)), t, pack2(1.f, 1.f)));
                            }
                            float x, y;
                            unpack2(mul2(q, add2(pack2(g[at], g[at + 1]), pack2(nd[k], nd[k + 1]))), x, y);
                            if (!full) {
                                x = e[c + k] == 0.f ? 0.f : x;
                                y = e[c + k + 1] == 0.f ? 0.f : y;
                            }
                            uint32_t pc[3];
                            split3(x, y, pc);
#pragma unroll
                            for (int z = 0; z < 3; ++z) w[z][(c + k) / 2] = pc[z];
                        }
                    }
#pragma unroll
                    for (int k = 0; k < 3; ++k) tmem_st_x8(tdS + lanes + kCols * k + (col + c0) / 2, w[k]);
                }
            }
            if (!kKeys) psum = add2(psum, tsum);
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&st.p_full));
        }
        if (ok && n > 0) {
            ok = __all_sync(~0u, tc_wait(smem_u32(&st.acc_full), (n - 1) & 1, failed));
            if (ok) {
                tc_fence_after();
                add_up();
            }
        }
        float total = 0.f;                              // of the row's P, in this block's share of the keys
        if (!kKeys) {
            float odd;
            unpack2(psum, total, odd);
            // in the place of the streamed rows, which nobody reads any more
            float* sums = reinterpret_cast<float*>(dyn + (sY - smem_u32(dyn)));
            sums[128 * wg + r] = total + odd;
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&st.sum_full));
            ok = __all_sync(~0u, ok && tc_wait(smem_u32(&st.sum_full), 0, failed));
            total = sums[r] + sums[128 + r];
        }
        if (ok && x0 + r < xrows) {
            if (!kKeys && wg == 0) {
                if (tp.parts.parts == 1) tp.fine[((int64_t)b * p.H + xh) * tp.Lp + x0 + r] = total == 0.f ? 0.f : log2f(total);
                else tp.parts.r[((int64_t)part * p.B * p.H + bh) * p.Lq + x0 + r] = total;
            }
            const int64_t* os = kKeys ? (is_dv ? p.dvs : p.dks) : p.dqs;
            float* out = tp.parts.parts == 1
                             ? (float*)(kKeys ? (is_dv ? p.dv : p.dk) : p.dq) + b * os[0] + xh * os[1] + (int64_t)(x0 + r) * os[2]
                             : (is_dv ? tp.parts.other : tp.parts.acc) +
                                   ((((int64_t)blockIdx.x % tp.parts.parts) * p.B + b) * nhead + xh) * xrows * p.D + (int64_t)(x0 + r) * p.D;
            out += ocol;
            const float f = is_dv ? 1.f : !kKeys && tp.parts.parts == 1 && total != 0.f ? p.scale / total : p.scale;
            const int cols = p.D - ocol;
#pragma unroll
            for (int c = 0; c < kAcc; c += 4)
                if (c < cols)
                    *reinterpret_cast<float4*>(out + c) = make_float4(o[c] * f, o[c + 1] * f, o[c + 2] * f, o[c + 3] * f);
        }
        if (!ok && lane == 0) tc_report(tp.status, 232);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 11) tmem_dealloc(st.tmem, 512);
}

}  // namespace mg
