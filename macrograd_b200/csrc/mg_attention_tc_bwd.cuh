// mg_attention_tc_bwd.cuh -- gradients of attention of 16-bit tensors on the
// 5th-generation tensor cores.
//
// One kernel in two forms. A block keeps 128 rows of two tensors X0, X1 in shared
// memory and streams tiles of 64 rows of two others, Y0, Y1:
//     S = X0 Y0^T,  dP = X1 Y1^T            (tensor memory, fp32)
//     P = exp2(S - lse),  dS = P * (dP - delta) * curve
//     acc += dS Y0   (and acc' += P Y1)     (P, dS from tensor memory, bf16)
// With the queries resident (X = q, dout; Y = k, v) acc is dQ. With the keys
// resident (X = k, v; Y = q, dout) S and dP are transposed, acc is dK and acc' is
// dV, summed over the query heads that share the key-value head. So no gradient
// is added to by two blocks: no atomics, and the same bits every time, for 8
// products instead of the 5 of a single kernel that would add dQ up atomically.
// Where there are fewer blocks than SMs, several share the streamed tiles of the same
// resident rows; each leaves its part in scratch, and attn_grad_join_kernel adds them up.
//
// delta = rowsum(dout * out) carries the 16-bit rounding of out, which dS = P * (dP -
// delta) magnifies where a row's weight lies on few keys (errors of dQ and dK of 0.4 %
// where the rounding of the result itself is 0.17 %) and where its values have much in
// common (errors as large as dQ and dK). The true delta makes the row's sum of
// P * (dP - delta) zero, so what that sum is in fp32 is delta's error r: the form with
// the queries resident, which runs first, adds it to delta for the other one, and
// corrects its own dQ by r times acc' = sum P * curve * k (the eighth product).
// P and dS go back to tensor memory over S and dP, as the A operand of the
// second pair of products: they never pass through shared memory.
//
// Two sets of eight warps take the tiles in turn, each with S and dP columns of its
// own, so that the tensor core works for one while the other takes exponentials. In a
// set two warps share 32 rows, 32 of the tile's columns each: the work is bound by
// the latency of its instructions, which four warps a scheduler hide better than two (with
// two, a tile took 3800 clocks of its set's time). P lies over S and dS over dP, which are all the columns there are at head_dim 128 (2 x (64 +
// 64) + 128 + 128 = 512, hence one block an SM), so a set's next S is issued
// as soon as its P has been multiplied (the queries resident: as soon as S is in
// registers), under the dS of the same tile, and its next dP after its dS: it
// finds both when it comes to them. Issued together, after dS, they cost each
// set another 2700 clocks a tile.
#pragma once

#include "mg_attention_tc.cuh"

namespace mg {

constexpr int kTcBwdThreads = 576;       // two sets of eight warps, loads, products
constexpr int kTcBwdLoadWarp = 16, kTcBwdMmaWarp = 17;
constexpr int kTcBwdStages = 4;

struct TcBwdParams {
    CUtensorMap x0, x1, y0, y1;          // boxes of 64 x 128 rows (x), 64 x 64 rows (y)
    AttnParams a;
    const int2* doc_tiles;
    const float* lse2;                   // [B * H][Lp] lse * log2(e); +inf where no key is seen
    float* delta;                        // [B * H][Lp]; made exact by the form with the queries resident
    int Lp;                              // q_len rounded up to 128
    int head_step[4], batch_step[4];     // of q, k, v, dout
    uint32_t idesc_s;
    float scale;                         // |scale|
    CapCurve curve;
    int* status;
    GradParts parts;
};

// lse2 and delta of each row, padded with rows whose P is 0. 16 lanes to a row of
// up to 128 elements, 8 each, and four rows at once: bound by the reads of out and dout.
__device__ __forceinline__ void load8(const __nv_bfloat16* x, float (&v)[8])
{
    const uint4 w = *reinterpret_cast<const uint4*>(x);
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&w);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float2 f = __bfloat1622float2(h[k]);
        v[2 * k] = f.x, v[2 * k + 1] = f.y;
    }
}
__device__ __forceinline__ void load8(const float* x, float (&v)[8])
{
    const float4 a = *reinterpret_cast<const float4*>(x), b = *reinterpret_cast<const float4*>(x + 4);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}

constexpr int kStatsRows = 4;            // of a group of 16 lanes; divides Lp

template <typename T>
__global__ void __launch_bounds__(256) attn_tc_stats_kernel(const __grid_constant__ AttnParams p, int Lp,
                                                            float* __restrict__ lse2, float* __restrict__ delta)
{
    const uint32_t group = blockIdx.x * (blockDim.x / 16) + threadIdx.x / 16, per = (uint32_t)Lp / kStatsRows;
    if (group >= (uint32_t)p.B * p.H * per) return;     // an even number of groups: whole warps
    const int part = threadIdx.x % 16;
    // heads first: their rows lie side by side where heads were split from [batch, length, heads * D]
    const uint32_t at_h = group / (uint32_t)p.H, h = group - at_h * (uint32_t)p.H, b = at_h / per, bh = b * (uint32_t)p.H + h;
    const int i0 = (int)(at_h - b * per) * kStatsRows;
    const T* out = (const T*)p.out + b * p.os[0] + h * p.os[1] + part * 8;
    const T* dout = (const T*)p.dout + b * p.dos[0] + h * p.dos[1] + part * 8;
    float o[kStatsRows][8], g[kStatsRows][8], lse[kStatsRows];
#pragma unroll
    for (int k = 0; k < kStatsRows; ++k) {
        const int i = i0 + k;
        lse[k] = i < p.Lq ? __ldg(p.lse + (int64_t)bh * p.Lq + i) : -CUDART_INF_F;
        if (i < p.Lq && part * 8 < p.D) {
            load8(out + i * p.os[2], o[k]);
            load8(dout + i * p.dos[2], g[k]);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) o[k][e] = g[k][e] = 0.f;
        }
    }
    float sum[kStatsRows];
#pragma unroll
    for (int k = 0; k < kStatsRows; ++k) {
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) s = fmaf(o[k][e], g[k][e], s);
#pragma unroll
        for (int w = 8; w; w /= 2) s += __shfl_xor_sync(~0u, s, w);
        // a row that sees nothing: P = 0 whatever its dout holds
        sum[k] = lse[k] == -CUDART_INF_F ? 0.f : s;
        lse[k] = lse[k] == -CUDART_INF_F ? CUDART_INF_F : lse[k] * kLog2e;
    }
    if (part == 0) {
        const int64_t at = (int64_t)bh * Lp + i0;
        *reinterpret_cast<float4*>(lse2 + at) = make_float4(lse[0], lse[1], lse[2], lse[3]);
        *reinterpret_cast<float4*>(delta + at) = make_float4(sum[0], sum[1], sum[2], sum[3]);
    }
}

struct TcBwdState {
    uint64_t x_full, y_full[kTcBwdStages], y_empty[kTcBwdStages];
    uint64_t s_full[2], dp_full[2], p_full[2], ds_full[2], acc_full, sum_full, drain;
    float sums[4][128];                  // a quarter of the warps each: the rows' sums of P * (dP - delta)
    uint32_t tmem;
    int failed;
    int loads;                           // stages that were asked for
    alignas(16) float lse2[kTcBwdStages][64];
    alignas(16) float delta[kTcBwdStages][64];
};

__device__ __forceinline__ void bulk_load(uint32_t bar, uint32_t dst, const void* src, uint32_t bytes)
{
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
                 "l"(src), "r"(bytes), "r"(bar)
                 : "memory");
}

// Tiles [t0, t1) of 64 streamed rows that meet the 128 resident rows from x0 (at
// position xpos) in some pair. Whole warps.
template <bool kKeys>
__device__ __forceinline__ void stream_range(const AttnParams& p, const int32_t* docs, const int2* dt, int prefix,
                                             int x0, int xpos, int shift, int& t0, int& t1)
{
    t0 = 0;
    if (kKeys) {
        if (p.causal && x0 >= prefix) t0 = min(max(0, x0 - shift), p.Lq) / 64;
        t1 = (p.Lq + 63) / 64;
    } else {
        const int last = min(x0 + 127, p.Lq - 1) + shift;
        t1 = ((!p.causal ? p.Lk : max(0, min(p.Lk, max(last + 1, prefix)))) + 63) / 64;
    }
    if (docs) narrow_to_docs(dt, p.Lk, kKeys ? shift : 0, 64, docs_of(dt, xpos, 128, p.Lk), t0, t1);
}

// Steps [i0, i0 + n) of `all`: part of `parts`.
__device__ __forceinline__ void share_of_steps(int part, int parts, int all, int& i0, int& n)
{
    const int each = (all + parts - 1) / parts;
    i0 = min(all, part * each);
    n = min(all, i0 + each) - i0;
}

// Adds up the parts of a gradient in their order (blockIdx.y: acc, other). One warp to a row,
// four elements to a lane. kJoinCorrect: dQ of 16-bit tensors, less the rows' sums r times the
// other product, and delta made exact. kJoinWeights: dQ of fp32 tensors, divided by the rows'
// sums of P, whose logarithm is kept.
enum : int { kJoinPlain = 0, kJoinCorrect = 1, kJoinWeights = 2 };
struct GradJoin {
    GradParts parts;
    int heads, L, D, Lp;
    int64_t rows;                        // B * heads * L
    void* out[2];
    int64_t os[2][3];
    float* delta;
    float* fine;                         // log2 of the sums of P
};

template <typename T, int kForm>
__global__ void __launch_bounds__(256) attn_grad_join_kernel(const __grid_constant__ GradJoin j)
{
    const int64_t row = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) / 32;
    if (row >= j.rows) return;
    const int d = threadIdx.x % 32 * 4;
    const bool in = d < j.D;
    const auto sum_of = [&](const float* src) {
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
        if (in)
            for (int s = 0; s < j.parts.parts; ++s) {
                const float4 x = __ldg(reinterpret_cast<const float4*>(src + (s * j.rows + row) * j.D + d));
                a.x += x.x, a.y += x.y, a.z += x.z, a.w += x.w;
            }
        return a;
    };
    const int64_t bh = row / j.L;
    const int i = (int)(row - bh * j.L), h = (int)(bh % j.heads), b = (int)(bh / j.heads);
    float4 a = sum_of(blockIdx.y ? j.parts.other : j.parts.acc);
    float r = 0.f;
    if (kForm != kJoinPlain)
        for (int s = 0; s < j.parts.parts; ++s) r += __ldg(j.parts.r + s * j.rows + row);
    if (kForm == kJoinWeights) {
        const float inv = r == 0.f ? 1.f : 1.f / r;
        a.x *= inv, a.y *= inv, a.z *= inv, a.w *= inv;
        if (d == 0) j.fine[bh * j.Lp + i] = r == 0.f ? 0.f : log2f(r);
    }
    if (kForm == kJoinCorrect) {
        const float4 w = sum_of(j.parts.other);
        a.x = fmaf(-r, w.x, a.x), a.y = fmaf(-r, w.y, a.y), a.z = fmaf(-r, w.z, a.z), a.w = fmaf(-r, w.w, a.w);
        if (d == 0) j.delta[bh * j.Lp + i] += r;
    }
    if (!in) return;
    const int64_t* os = j.os[blockIdx.y];
    T* out = (T*)j.out[blockIdx.y] + b * os[0] + h * os[1] + i * os[2] + d;
    out[0] = from_f32<T>(a.x), out[1] = from_f32<T>(a.y), out[2] = from_f32<T>(a.z), out[3] = from_f32<T>(a.w);
}

template <int DP>
constexpr size_t tc_backward_smem() { return (2 * 128 + kTcBwdStages * 2 * 64) * DP * 2 + 1024; }

template <int DP, bool kKeys, bool kCap, bool kBias>
__global__ void __launch_bounds__(kTcBwdThreads, 1) attn_tc_backward(const __grid_constant__ TcBwdParams tp)
{
    extern __shared__ uint8_t dyn[];
    __shared__ TcBwdState st;
    const AttnParams& p = tp.a;
    constexpr uint32_t kX = 128 * DP * 2, kY = 64 * DP * 2;
    const uint32_t base = (smem_u32(dyn) + 1023u) & ~1023u;
    const uint32_t sX0 = base, sX1 = base + kX, sY = base + 2 * kX;
    const int warp = __shfl_sync(~0u, threadIdx.x / 32, 0), lane = threadIdx.x % 32;   // uniform: so are the roles

    // blocks with the most tiles first: the first keys, the last queries
    const int nhead = kKeys ? p.Hkv : p.H, xrows = kKeys ? p.Lk : p.Lq;
    const int xtiles = (xrows + 127) / 128, part = blockIdx.x % tp.parts.parts, block = blockIdx.x / tp.parts.parts;
    const int bh = block % (p.B * nhead), rank = block / (p.B * nhead);
    const int x0 = (kKeys ? rank : xtiles - 1 - rank) * 128;
    const int xh = bh % nhead, b = bh / nhead, group = p.H / p.Hkv;
    const int shift = p.Lk - p.Lq;
    const int32_t* docs = p.docs ? p.docs + (int64_t)b * p.Lk : nullptr;
    const int2* dt = p.docs ? tp.doc_tiles + (int64_t)b * ((p.Lk + 127) / 128) : nullptr;
    const int prefix = p.prefix ? __ldg(p.prefix + b) : 0;
    const int xpos = kKeys ? x0 : x0 + shift;            // position of the first resident row

    if (threadIdx.x == 0) {
        mbar_init(smem_u32(&st.x_full), 1);
        for (int i = 0; i < kTcBwdStages; ++i) {
            mbar_init(smem_u32(&st.y_full[i]), 1);
            mbar_init(smem_u32(&st.y_empty[i]), 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&st.s_full[i]), 1);
            mbar_init(smem_u32(&st.dp_full[i]), 1);
            mbar_init(smem_u32(&st.p_full[i]), 8);
            mbar_init(smem_u32(&st.ds_full[i]), 8);
        }
        mbar_init(smem_u32(&st.acc_full), 1);
        mbar_init(smem_u32(&st.sum_full), 16);
        mbar_init(smem_u32(&st.drain), 1);
        mbar_fence_init();
        st.failed = 0;
        st.loads = 0;
    }
    if (warp == kTcBwdMmaWarp) {
        tmem_alloc(smem_u32(&st.tmem), 512);
        tmem_relinquish();
    }
    int t0, t1;
    stream_range<kKeys>(p, docs, dt, prefix, x0, xpos, shift, t0, t1);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    int i0, n;                                           // the block's share of the steps
    const int tiles = max(0, t1 - t0);
    share_of_steps(part, tp.parts.parts, kKeys ? tiles * group : tiles, i0, n);
    if (!kKeys) t0 += i0;
    const uint32_t tA = st.tmem + 256, tB = tA + DP;     // accumulators: dS Y0, P Y1 (the queries resident: P curve Y0)
    volatile int* failed = &st.failed;
    // columns of step i's S and dP; the 16-bit P and dS of columns [32 h, 32 h + 32) lie in the first 16 of these
    const auto tS = [&](int i) { return st.tmem + 128 * (i & 1); };
    const auto sY0 = [&](int i) { return sY + (uint32_t)(i % kTcBwdStages) * 2 * kY; };

    if (warp == kTcBwdLoadWarp) {
        // ------------------------------------------------ loads
        if (lane == 0 && n > 0) {
            constexpr int X0 = kKeys ? 1 : 0, X1 = kKeys ? 2 : 3, Y0 = kKeys ? 0 : 1, Y1 = kKeys ? 3 : 2;
            const uint32_t xb = smem_u32(&st.x_full);
            mbar_arrive_expect_tx(xb, 2 * kX);
            for (int c = 0; c < DP; c += 64) {
                tma_load(&tp.x0, xb, sX0 + c / 64 * 128 * 128, 4, c, x0, xh * tp.head_step[X0], b * tp.batch_step[X0], 0);
                tma_load(&tp.x1, xb, sX1 + c / 64 * 128 * 128, 4, c, x0, xh * tp.head_step[X1], b * tp.batch_step[X1], 0);
            }
            for (int i = 0; i < n; ++i) {
                const int s = i % kTcBwdStages;
                if (i >= kTcBwdStages && !tc_wait(smem_u32(&st.y_empty[s]), (i / kTcBwdStages - 1) & 1, failed)) break;
                const int yh = kKeys ? xh * group + (i0 + i) / tiles : xh / group;
                const int y0 = (t0 + (kKeys ? (i0 + i) % tiles : i)) * 64;
                const uint32_t yb = smem_u32(&st.y_full[s]);
                mbar_arrive_expect_tx(yb, 2 * kY + (kKeys ? 512u : 0u));
                for (int c = 0; c < DP; c += 64) {
                    tma_load(&tp.y0, yb, sY0(i) + c / 64 * 64 * 128, 4, c, y0, yh * tp.head_step[Y0],
                             b * tp.batch_step[Y0], 0);
                    tma_load(&tp.y1, yb, sY0(i) + kY + c / 64 * 64 * 128, 4, c, y0, yh * tp.head_step[Y1],
                             b * tp.batch_step[Y1], 0);
                }
                if (kKeys) {
                    const int64_t at = ((int64_t)b * p.H + yh) * tp.Lp + y0;
                    bulk_load(yb, smem_u32(st.lse2[s]), tp.lse2 + at, 256);
                    bulk_load(yb, smem_u32(st.delta[s]), tp.delta + at, 256);
                }
                st.loads = i + 1;
            }
        }
    } else if (warp == kTcBwdMmaWarp) {
        // ------------------------------------------------ products
        constexpr uint32_t idesc_dp = idesc_bf16(128, 64, false, false), idesc_acc = idesc_bf16(128, DP, false, true);
        bool ok = n == 0 || __all_sync(~0u, tc_wait(smem_u32(&st.x_full), 0, failed));
        const auto scores_of = [&](int i) {       // S, from the tile's first use on
            const int s = i % kTcBwdStages;
            ok = __all_sync(~0u, ok && tc_wait(smem_u32(&st.y_full[s]), (i / kTcBwdStages) & 1, failed));
            if (!ok) return;
            if (docs) {
                const int y0 = (t0 + (kKeys ? (i0 + i) % tiles : i)) * 64, pos = y0 + (kKeys ? shift : 0);
                bool pad = pos < 0 || pos + 64 > p.Lk;
                if (!pad) pad = __ldg(dt + (pos >> 7)).x < 0 || __ldg(dt + ((pos + 63) >> 7)).x < 0;
                if (pad) {
                    tc_clear_padding<DP>(sY0(i), 64, docs, pos, p.Lk, lane);
                    tc_clear_padding<DP>(sY0(i) + kY, 64, docs, pos, p.Lk, lane);
                }
            }
            tc_fence_after();
#pragma unroll
            for (int k = 0; k < DP / 16; ++k)
                tc_mma_f16(tS(i), desc_k_major(sX0, 128, k), desc_k_major(sY0(i), 64, k), tp.idesc_s, k > 0);
            tc_commit_warp(smem_u32(&st.s_full[i & 1]));
        };
        const auto dp_of = [&](int i) {           // dP
            if (!ok) return;
#pragma unroll
            for (int k = 0; k < DP / 16; ++k)
                tc_mma_f16(tS(i) + 64, desc_k_major(sX1, 128, k), desc_k_major(sY0(i) + kY, 64, k), idesc_dp, k > 0);
            tc_commit_warp(smem_u32(&st.dp_full[i & 1]));
        };
        for (int i = 0; i < min(n, 2); ++i) {
            scores_of(i);
            dp_of(i);
        }
        for (int i = 0; i < n && ok; ++i) {
            ok = __all_sync(~0u, tc_wait(smem_u32(&st.p_full[i & 1]), (i >> 1) & 1, failed));
            if (!ok) break;
            tc_fence_after();
#pragma unroll
            for (int k = 0; k < 4; ++k)
                tc_mma_f16_ta(tB, tS(i) + 8 * k + 16 * (k / 2), desc_mn_major(sY0(i) + (kKeys ? kY : 0), 64, k), idesc_acc,
                              i > 0 || k > 0);
            if (i + 2 < n) scores_of(i + 2);
            ok = __all_sync(~0u, ok && tc_wait(smem_u32(&st.ds_full[i & 1]), (i >> 1) & 1, failed));
            if (!ok) break;
            tc_fence_after();
#pragma unroll
            for (int k = 0; k < 4; ++k)
                tc_mma_f16_ta(tA, tS(i) + 64 + 8 * k + 16 * (k / 2), desc_mn_major(sY0(i), 64, k), idesc_acc, i > 0 || k > 0);
            tc_commit_warp(smem_u32(&st.y_empty[i % kTcBwdStages]));
            if (i + 1 == n) tc_commit_warp(smem_u32(&st.acc_full));
            if (i + 2 < n) dp_of(i + 2);
        }
        if (!ok) {
            __syncwarp();
            tc_commit_warp(smem_u32(&st.drain));
            if (lane == 0) {
                tc_report(tp.status, 211);
                tc_drain(smem_u32(&st.drain), 0);
            }
            __syncwarp();
        }
    } else {
        // ------------------------------------------------ P and dS
        const int set = warp / 8, col = 32 * (warp / 4 % 2), r = threadIdx.x % 128;   // resident row, first column
        const uint32_t lanes = (uint32_t)(warp % 4) << 21;
        const int pos = xpos + r;
        const int rdoc = docs ? (x0 + r < xrows ? doc_at(p, b, pos) : -1) : 0;
        const int common = docs ? (x0 + 128 <= xrows ? common_doc(dt, xpos, 128, p.Lk) : -1) : 0;
        const float mul = kCap ? p.cap * kLog2e : tp.scale * kLog2e;
        float lse2 = 0.f, delta = 0.f;
        if (!kKeys) {
            const int64_t at = ((int64_t)b * p.H + xh) * tp.Lp + x0 + r;
            lse2 = tp.lse2[at];
            delta = tp.delta[at];
        }
        uint64_t rsum2 = pack2(0.f, 0.f);   // this thread's part of its row's sum of P * (dP - delta)
        bool ok = true;
        // this lane's document of a tile's streamed rows, a tile of the set ahead
        const auto y_of = [&](int i) { return (t0 + (kKeys ? (i0 + i) % tiles : i)) * 64; };
        int ydoc[1] = {docs && set < n ? doc_at(p, b, y_of(set) + (kKeys ? shift : 0) + col + lane) : -1};
        for (int i = set; i < n; i += 2) {
            const int h = kKeys ? xh * group + (i0 + i) / tiles : xh;
            const int y0 = y_of(i), ypos = y0 + (kKeys ? shift : 0);
            const int s = i % kTcBwdStages;
            const float slope = kBias ? __ldg(p.slopes + h) * kLog2e : 0.f;
            bool full;
            uint32_t seen[1] = {~0u};
            if (kKeys) full = !p.causal || ypos >= xpos + 127 || xpos + 128 <= prefix;
            else full = ypos + 64 <= p.Lk && (!p.causal || ypos + 63 <= xpos || ypos + 64 <= prefix);
            if (docs) full = full && common >= 0 && (!kKeys || y0 + 64 <= p.Lq) && common_doc(dt, ypos, 64, p.Lk) == common;
            if (!full) {
                if (docs) same_document(rdoc, ydoc, seen);
                if (!kKeys) seen[0] &= bits_below((!p.causal ? p.Lk : min(p.Lk, max(pos + 1, prefix))) - ypos - col);
                else if (p.causal && pos >= prefix) seen[0] &= ~bits_below(pos - ypos - col);
            }
            if (docs && i + 2 < n) ydoc[0] = doc_at(p, b, y_of(i + 2) + (kKeys ? shift : 0) + col + lane);
            ok = __all_sync(~0u, tc_wait(smem_u32(&st.s_full[set]), (i >> 1) & 1, failed) &&
                                     (!kKeys || tc_wait(smem_u32(&st.y_full[s]), (i / kTcBwdStages) & 1, failed)));
            if (!ok) break;
            tc_fence_after();
            float v[32];
            tmem_ld_x32(tS(i) + lanes + col, v);
            if (kCap) cap_scores(v, tp.curve);      // tanh of the score over the cap
            uint32_t w[16];
            const float far = (float)(pos - ypos - col);
            const uint64_t mul_2 = pack2(mul, mul);
#pragma unroll
            for (int c = 0; c < 32; c += 4) {
                float nl[4] = {-lse2, -lse2, -lse2, -lse2};
                if (kKeys) {
                    const float4 x = *reinterpret_cast<const float4*>(&st.lse2[s][col + c]);
                    nl[0] = -x.x, nl[1] = -x.y, nl[2] = -x.z, nl[3] = -x.w;
                }
                if (kBias) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) nl[k] = fmaf(-slope, fabsf(far - (float)(c + k)), nl[k]);
                }
                float e[4];
#pragma unroll
                for (int k = 0; k < 4; k += 2) {
                    unpack2(fma2(pack2(v[c + k], v[c + k + 1]), mul_2, pack2(nl[k], nl[k + 1])), e[k], e[k + 1]);
                    e[k] = ex2(e[k]);
                    e[k + 1] = ex2(e[k + 1]);
                }
                if (!full) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const bool in = seen[0] >> (c + k) & 1;
                        e[k] = in ? e[k] : 0.f;
                        if (kCap) v[c + k] = in ? v[c + k] : 0.f;
                    }
                }
                if (kKeys || !kCap) {
                    w[c / 2] = bf16x2(e[0], e[1]);
                    w[c / 2 + 1] = bf16x2(e[2], e[3]);
                }
#pragma unroll
                for (int k = 0; k < 4; k += 2) {
                    uint64_t q = pack2(e[k], e[k + 1]);
                    if (kCap) {
                        const uint64_t t = pack2(v[c + k], v[c + k + 1]);
                        q = mul2(q, fma2(mul2(t, pack2(-1.f, -1.f)), t, pack2(1.f, 1.f)));
                    }
                    unpack2(q, v[c + k], v[c + k + 1]);
                    // what the curve takes off P, for the row's sum
                    if (!kKeys && kCap) w[(c + k) / 2] = bf16x2(e[k] - v[c + k], e[k + 1] - v[c + k + 1]);
                }
            }
            if (!kKeys && kCap) {
                // the correction's product takes P * curve
                uint32_t pc[16];
#pragma unroll
                for (int c = 0; c < 32; c += 2) pc[c / 2] = bf16x2(v[c], v[c + 1]);
                tmem_st_x16(tS(i) + lanes + col, pc);
            } else {
                tmem_st_x16(tS(i) + lanes + col, w);
            }
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&st.p_full[set]));
            ok = __all_sync(~0u, tc_wait(smem_u32(&st.dp_full[set]), (i >> 1) & 1, failed));
            if (!ok) break;
            tc_fence_after();
#pragma unroll
            for (int c0 = 0; c0 < 32; c0 += 16) {
                float g[16];
                uint32_t ds[8];
                tmem_ld_x16(tS(i) + 64 + lanes + col + c0, g);
#pragma unroll
                for (int c = 0; c < 16; c += 4) {
                    float nd[4] = {-delta, -delta, -delta, -delta};
                    if (kKeys) {
                        const float4 x = *reinterpret_cast<const float4*>(&st.delta[s][col + c0 + c]);
                        nd[0] = -x.x, nd[1] = -x.y, nd[2] = -x.z, nd[3] = -x.w;
                    }
                    float e[4];
#pragma unroll
                    for (int k = 0; k < 4; k += 2) {
                        const int at = c0 + c + k;
                        const uint64_t d = add2(pack2(g[c + k], g[c + k + 1]), pack2(nd[k], nd[k + 1]));
                        uint64_t x = mul2(pack2(v[at], v[at + 1]), d);
                        unpack2(x, e[k], e[k + 1]);
                        if (!full) {
                            e[k] = v[at] == 0.f ? 0.f : e[k];
                            e[k + 1] = v[at + 1] == 0.f ? 0.f : e[k + 1];
                            x = pack2(e[k], e[k + 1]);
                        }
                        if (!kKeys && kCap) {
                            // P * (dP - delta): what the curve takes off is added again
                            const uint64_t off = pack2(__uint_as_float(w[at / 2] << 16), __uint_as_float(w[at / 2] & 0xFFFF0000u));
                            if (full) {
                                x = fma2(off, d, x);
                            } else {
                                float a, c2, o0, o1;
                                unpack2(mul2(off, d), a, c2);
                                unpack2(off, o0, o1);
                                x = add2(x, pack2(o0 == 0.f ? 0.f : a, o1 == 0.f ? 0.f : c2));
                            }
                        }
                        if (!kKeys) rsum2 = add2(rsum2, x);
                    }
                    ds[c / 2] = bf16x2(e[0], e[1]);
                    ds[c / 2 + 1] = bf16x2(e[2], e[3]);
                }
                tmem_st_x8(tS(i) + 64 + lanes + col + c0 / 2, ds);
            }
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&st.ds_full[set]));
        }
        float rsum = 0.f;
        if (!kKeys) {
            float odd;
            unpack2(rsum2, rsum, odd);
            st.sums[warp / 4][r] = rsum + odd;
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&st.sum_full));
            ok = ok && tc_wait(smem_u32(&st.sum_full), 0, failed);
        }
        if (n > 0) ok = ok && tc_wait(smem_u32(&st.acc_full), 0, failed);
        ok = __all_sync(~0u, ok);
        if (ok) {
            tc_fence_after();
            if (!kKeys) {
                rsum = (st.sums[0][r] + st.sums[1][r]) + (st.sums[2][r] + st.sums[3][r]);
                if (warp < 4 && x0 + r < xrows) {
                    if (tp.parts.parts == 1) tp.delta[(int64_t)bh * tp.Lp + x0 + r] = delta + rsum;
                    else tp.parts.r[((int64_t)part * p.B * p.H + bh) * p.Lq + x0 + r] = rsum;
                }
            }
            // with the keys: half of dK or of dV to each four warps; with the queries: a quarter of dQ
            const int quarter = warp / 4;
            const bool is_dv = kKeys && quarter >= 2;
            const int64_t* os = kKeys ? (is_dv ? p.dvs : p.dks) : p.dqs;
            __nv_bfloat16* out = (__nv_bfloat16*)(kKeys ? (is_dv ? p.dv : p.dk) : p.dq) + b * os[0] + xh * os[1] +
                                 (int64_t)(x0 + r) * os[2];
            const float f = is_dv ? 1.f : p.scale;
            const int c0 = kKeys ? quarter % 2 * (DP / 2) : quarter * (DP / 4), c1 = min(p.D, c0 + DP / (kKeys ? 2 : 4));
            if (tp.parts.parts > 1) {
                const int64_t at = (((int64_t)part * p.B * nhead + bh) * xrows + x0 + r) * p.D;
#pragma unroll 1
                for (int which = 0; which < (kKeys ? 1 : 2); ++which) {
                    const bool second = kKeys ? is_dv : which == 1;
                    float* to = (second ? tp.parts.other : tp.parts.acc) + at;
#pragma unroll 1
                    for (int c = c0; c < c1; c += 16) {
                        float o[16];
                        if (n > 0) tmem_ld_x16((second ? tB : tA) + lanes + c, o);
                        if (x0 + r >= xrows) continue;
#pragma unroll
                        for (int k = 0; k < 16; k += 4)
                            if (c + k < c1)
                                *reinterpret_cast<float4*>(to + c + k) =
                                    n > 0 ? make_float4(o[k] * f, o[k + 1] * f, o[k + 2] * f, o[k + 3] * f)
                                          : make_float4(0.f, 0.f, 0.f, 0.f);
                    }
                }
            }
#pragma unroll 1
            for (int c = c0; c < c1 && tp.parts.parts == 1; c += 16) {
                float o[16];
                if (n > 0) {
                    tmem_ld_x16((is_dv ? tB : tA) + lanes + c, o);
                    if (!kKeys) {
                        float w[16];
                        tmem_ld_x16(tB + lanes + c, w);
#pragma unroll
                        for (int k = 0; k < 16; ++k) o[k] = fmaf(-rsum, w[k], o[k]);
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < 16; ++k) o[k] = 0.f;
                }
                if (x0 + r >= xrows) continue;
#pragma unroll
                for (int k = 0; k < 16; k += 8)
                    if (c + k + 8 <= c1)
                        *reinterpret_cast<uint4*>(out + c + k) =
                            make_uint4(bf16x2(o[k] * f, o[k + 1] * f), bf16x2(o[k + 2] * f, o[k + 3] * f),
                                       bf16x2(o[k + 4] * f, o[k + 5] * f), bf16x2(o[k + 6] * f, o[k + 7] * f));
            }
        }
        if (!ok && lane == 0) tc_report(tp.status, 212);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (st.failed && threadIdx.x == 0 && n > 0) {        // copies that nobody waited for
        tc_drain(smem_u32(&st.x_full), 0);
        for (int i = max(0, st.loads - kTcBwdStages); i < st.loads; ++i)
            tc_drain(smem_u32(&st.y_full[i % kTcBwdStages]), (i / kTcBwdStages) & 1);
    }
    if (warp == kTcBwdMmaWarp) tmem_dealloc(st.tmem, 512);
}

}  // namespace mg
