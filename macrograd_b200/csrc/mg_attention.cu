// mg_attention.cu -- host side and C ABI of the attention operators: checks of
// arguments, choice of kernel, scratch, launches.
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstring>

#include "mg_attention.h"
#include "mg_host.h"
#include "mg_attention_simt.cuh"
#include "mg_attention_tc.cuh"
#include "mg_attention_tc_bwd.cuh"
#include "mg_attention_tc32.cuh"
#include "mg_attention_tc32_bwd.cuh"
#include "mg_paged.cuh"
#include "mg_rotary.cuh"

using mg::host::Device;
using mg::host::fail;
using mg::host::Range;
using mg::host::Scratch;

namespace {

int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

size_t elem_size(int dtype) { return dtype == MG_F32 ? 4 : 2; }

mg_status launched(const char* what)
{
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return fail(MG_ERR_CUDA, "%s: launch failed: %s", what, cudaGetErrorString(e));
    mg::host::count_launch();
    return MG_OK;
}

// Opts kernel K in to `smem` bytes of dynamic shared memory, once on each device.
template <auto K>
mg_status allow_smem(const Device& dev, size_t smem)
{
    static std::atomic<uint64_t> done{0};     // a bit a device; the library serves 64
    const uint64_t bit = 1ull << dev.ordinal;
    if (done.load(std::memory_order_acquire) & bit) return MG_OK;
    MG_HOST_TRY(cudaFuncSetAttribute(K, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    done.fetch_or(bit, std::memory_order_release);
    return MG_OK;
}

#define MG_TRY(call)                     \
    do {                                 \
        const mg_status s_ = (call);     \
        if (s_ != MG_OK) return s_;      \
    } while (0)

// ---------------------------------------------------------------- attention
mg_status check_attention(const mg_attention_desc* d, const char* who)
{
    if (!d) return fail(MG_ERR_INVALID, "%s: descriptor is NULL", who);
    if (d->dtype != MG_F32 && d->dtype != MG_BF16)
        return fail(MG_ERR_INVALID, "%s: dtype %d is neither MG_F32 nor MG_BF16", who, d->dtype);
    if (d->batch < 0 || d->heads < 1 || d->kv_heads < 1 || d->q_len < 0 || d->k_len < 0)
        return fail(MG_ERR_INVALID, "%s: batch %d, heads %d, kv_heads %d, q_len %d, k_len %d out of range", who,
                    d->batch, d->heads, d->kv_heads, d->q_len, d->k_len);
    if (d->heads % d->kv_heads)
        return fail(MG_ERR_INVALID, "%s: heads %d is not a multiple of kv_heads %d", who, d->heads, d->kv_heads);
    if (d->head_dim < 1 || d->head_dim > MG_MAX_HEAD_DIM)
        return fail(MG_ERR_UNSUPPORTED, "%s: head_dim %d is outside 1..%d", who, d->head_dim, MG_MAX_HEAD_DIM);
    if (!std::isfinite(d->scale)) return fail(MG_ERR_INVALID, "%s: scale is not finite", who);
    if (!(d->cap >= 0.f) || !std::isfinite(d->cap))
        return fail(MG_ERR_INVALID, "%s: cap must be 0 (none) or a positive number", who);
    if (d->prefix && !d->causal) return fail(MG_ERR_INVALID, "%s: a prefix needs causal", who);
    if ((int64_t)d->q_len + d->k_len >= (1ll << 30)) return fail(MG_ERR_UNSUPPORTED, "%s: rows are too long", who);
    const int64_t rows = (int64_t)d->batch * d->heads * std::max(ceil_div(d->q_len, 32), ceil_div(d->k_len, 32));
    if (rows >= (1ll << 31) - 1) return fail(MG_ERR_UNSUPPORTED, "%s: batch * heads * rows is too large", who);
    return MG_OK;
}

mg::AttnParams attention_params(const mg_attention_desc* d)
{
    mg::AttnParams p = {};
    p.B = d->batch, p.H = d->heads, p.Hkv = d->kv_heads, p.Lq = d->q_len, p.Lk = d->k_len, p.D = d->head_dim;
    p.causal = d->causal != 0;
    p.scale = d->scale, p.cap = d->cap;
    // a dim of one element may carry any stride
    for (int i = 0; i < 3; ++i) {
        p.qs[i] = d->q_stride[i], p.ks[i] = d->k_stride[i], p.vs[i] = d->v_stride[i], p.os[i] = d->out_stride[i];
        p.dos[i] = d->dout_stride[i], p.dqs[i] = d->dq_stride[i];
        p.dks[i] = d->dk_stride[i], p.dvs[i] = d->dv_stride[i];
        const int qn = i == 0 ? d->batch : i == 1 ? d->heads : d->q_len;
        const int kn = i == 0 ? d->batch : i == 1 ? d->kv_heads : d->k_len;
        if (qn == 1) p.qs[i] = p.os[i] = p.dos[i] = p.dqs[i] = 0;
        if (kn == 1) p.ks[i] = p.vs[i] = p.dks[i] = p.dvs[i] = 0;
    }
    p.slopes = d->slopes, p.docs = d->documents, p.prefix = d->prefix;
    return p;
}

template <typename K>
mg_status simt_launch(K kernel, int blocks, int rows_in_smem, int tiles33, const mg::AttnParams& p, cudaStream_t st,
                      const char* what)
{
    const size_t smem = sizeof(float) * ((size_t)rows_in_smem * mg::kSimtTile * (p.D + 1) +
                                         (size_t)tiles33 * mg::kSimtTile * 33);
    MG_HOST_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    kernel<<<blocks, mg::kSimtThreads, smem, st>>>(p);
    return launched(what);
}

template <typename T>
mg_status forward_simt(const mg::AttnParams& p, cudaStream_t st)
{
    return simt_launch(mg::attn_simt_forward<T>, p.B * p.H * ceil_div(p.Lq, mg::kSimtTile), 3, 1, p, st,
                       "mg_attention");
}

template <typename T>
mg_status backward_simt(const mg::AttnParams& p, cudaStream_t st)
{
    const char* who = "mg_attention_backward";
    if (p.Lq > 0) {
        mg::attn_delta_kernel<T><<<ceil_div((int64_t)p.B * p.H * p.Lq, 8), 256, 0, st>>>(p);
        MG_TRY(launched(who));
        MG_TRY(simt_launch(mg::attn_simt_backward_dq<T>, p.B * p.H * ceil_div(p.Lq, mg::kSimtTile), 4, 1, p, st, who));
    }
    if (p.Lk > 0)
        MG_TRY(simt_launch(mg::attn_simt_backward_dkv<T>, p.B * p.Hkv * ceil_div(p.Lk, mg::kSimtTile), 4, 2, p, st,
                           who));
    return MG_OK;
}

// Whether rows at `ptr` with these strides start on multiples of `vec` elements.
bool aligned(const void* ptr, const int64_t* strides, int n, size_t elem, int vec)
{
    if (reinterpret_cast<uintptr_t>(ptr) % (elem * vec)) return false;
    for (int i = 0; i < n; ++i)
        if (strides[i] % vec) return false;
    return true;
}

// ---------------------------------------------------------------- tensor cores
// The tensor-core kernels read and store rows of whole 16-byte vectors, 16-bit
// tensors through TMA; a scale of 0 would turn their masked scores (-inf) into
// NaN. Everything else runs on the CUDA cores.
bool tc_serves(const mg_attention_desc* d, const mg::AttnParams& p, std::initializer_list<const void*> rows_q,
               std::initializer_list<const void*> rows_k)
{
    if (d->head_dim % 8 || d->scale == 0.f || !std::isfinite(1.f / d->scale)) return false;
    const int vec = d->dtype == MG_BF16 ? 8 : 4;
    for (const void* x : rows_q)
        if (reinterpret_cast<uintptr_t>(x) % 16) return false;
    for (const void* x : rows_k)
        if (reinterpret_cast<uintptr_t>(x) % 16) return false;
    for (int i = 0; i < 3; ++i)
        for (int64_t s : {p.qs[i], p.ks[i], p.vs[i], p.os[i], p.dos[i], p.dqs[i], p.dks[i], p.dvs[i]})
            if (s % vec || s < 0 || s >= (1ll << 38)) return false;
    if (d->dtype == MG_F32) return true;
    const bool rows_repeat = (p.Lq > 1 && (p.qs[2] == 0 || (p.dout && p.dos[2] == 0))) ||
                             (p.Lk > 1 && (p.ks[2] == 0 || p.vs[2] == 0));
    return !rows_repeat;
}

// Map of [batch][heads][rows][D] for boxes of `box_rows` rows of 64 elements.
mg_status tc_map(CUtensorMap* map, int* head_step, int* batch_step, const void* base, const int64_t* stride, int D,
                 int rows, int heads, int batch, int box_rows)
{
    *head_step = stride[1] != 0;
    *batch_step = stride[0] != 0;
    const uint64_t dims[4] = {(uint64_t)D, (uint64_t)rows, *head_step ? (uint64_t)heads : 1,
                              *batch_step ? (uint64_t)batch : 1};
    const uint64_t any = (uint64_t)(D + 7) / 8 * 16;      // of a dim of one element
    uint64_t st[3];
    for (int i = 0; i < 3; ++i) st[i] = stride[2 - i] ? (uint64_t)stride[2 - i] * 2 : any;
    const uint32_t box[4] = {64, (uint32_t)box_rows, 1, 1};
    return mg::host::encode_bf16(map, base, 4, dims, st, box);
}

// The terms of the capped score's curve for products of magnitude |scale| (see mg::CapCurve).
mg::CapCurve cap_curve(float scale, float cap)
{
    mg::CapCurve cc = {};
    if (!(cap > 0.f)) return cc;
    const double pre = (double)scale / cap, c[4] = {0.999999463558197, -0.33326318860054016, 0.13190296292304993,
                                                    -0.04440222308039665};
    cc.pre = (float)pre;
    cc.bound = pre > 1e-5 && pre < 1e4 ? (float)(0.5 / pre) : 0.f;
    double power = pre;
    for (int i = 0; i < 4; ++i, power *= pre * pre) cc.tc[i] = (float)(c[i] * power);
    return cc;
}

mg_status tc_params(mg::TcAttnParams* t, const mg::AttnParams& p, const Device& dev, Scratch& ws, cudaStream_t st,
                    const char* who)
{
    t->a = p;
    t->scale = std::fabs(p.scale);
    t->idesc_s = mg::idesc_bf16(128, 128, false, false, p.scale < 0.f);
    t->status = dev.status;
    t->curve = cap_curve(t->scale, p.cap);
    if (p.docs) {
        const int64_t tiles = (int64_t)p.B * ceil_div(p.Lk, 128);
        int2* dt = static_cast<int2*>(ws.get(std::max<int64_t>(1, tiles) * sizeof(int2)));
        if (!dt) return fail(MG_ERR_ALLOC, "%s: no scratch for the documents' tiles", who);
        t->doc_tiles = dt;
        if (tiles) {
            mg::attn_doc_tiles_kernel<<<ceil_div(tiles, 4), 128, 0, st>>>(p.docs, dt, p.B, p.Lk);
            MG_TRY(launched(who));
        }
    }
    return MG_OK;
}

template <int DP, bool kCap, bool kBias>
mg_status launch_tc_forward(const mg::TcAttnParams& t, const Device& dev, cudaStream_t st)
{
    constexpr auto kernel = mg::attn_tc_forward<DP, kCap, kBias>;
    constexpr size_t smem = mg::tc_forward_smem<DP>();
    MG_TRY(allow_smem<kernel>(dev, smem));
    kernel<<<ceil_div(t.a.Lq, 128) * t.a.B * t.a.H, mg::kTcFwdThreads, smem, st>>>(t);
    return launched("mg_attention");
}

template <int DP>
mg_status launch_tc_forward(const mg::TcAttnParams& t, const Device& dev, cudaStream_t st)
{
    const bool cap = t.a.cap > 0.f, bias = t.a.slopes != nullptr;
    return cap ? (bias ? launch_tc_forward<DP, true, true>(t, dev, st) : launch_tc_forward<DP, true, false>(t, dev, st))
               : (bias ? launch_tc_forward<DP, false, true>(t, dev, st) : launch_tc_forward<DP, false, false>(t, dev, st));
}

mg_status forward_tc(const mg::AttnParams& p, const Device& dev, void* stream)
{
    mg::TcAttnParams t = {};
    Scratch ws(dev, stream);
    cudaStream_t st = (cudaStream_t)stream;
    MG_TRY(tc_params(&t, p, dev, ws, st, "mg_attention"));
    MG_TRY(tc_map(&t.q, &t.head_step[0], &t.batch_step[0], p.q, p.qs, p.D, p.Lq, p.H, p.B, 128));
    MG_TRY(tc_map(&t.k, &t.head_step[1], &t.batch_step[1], p.k, p.ks, p.D, p.Lk, p.Hkv, p.B, 128));
    MG_TRY(tc_map(&t.v, &t.head_step[2], &t.batch_step[2], p.v, p.vs, p.D, p.Lk, p.Hkv, p.B, 128));
    return p.D <= 64 ? launch_tc_forward<64>(t, dev, st) : launch_tc_forward<128>(t, dev, st);
}

template <int DP, bool kKeys, bool kCap, bool kBias>
mg_status launch_tc_backward(const mg::TcBwdParams& t, const Device& dev, cudaStream_t st)
{
    constexpr auto kernel = mg::attn_tc_backward<DP, kKeys, kCap, kBias>;
    constexpr size_t smem = mg::tc_backward_smem<DP>();
    MG_TRY(allow_smem<kernel>(dev, smem));
    const int blocks = kKeys ? ceil_div(t.a.Lk, 128) * t.a.B * t.a.Hkv : ceil_div(t.a.Lq, 128) * t.a.B * t.a.H;
    kernel<<<blocks, mg::kTcBwdThreads, smem, st>>>(t);
    return launched("mg_attention_backward");
}

template <int DP, bool kKeys>
mg_status launch_tc_backward(const mg::TcBwdParams& t, const Device& dev, cudaStream_t st)
{
    const bool cap = t.a.cap > 0.f, bias = t.a.slopes != nullptr;
    return cap ? (bias ? launch_tc_backward<DP, kKeys, true, true>(t, dev, st)
                       : launch_tc_backward<DP, kKeys, true, false>(t, dev, st))
               : (bias ? launch_tc_backward<DP, kKeys, false, true>(t, dev, st)
                       : launch_tc_backward<DP, kKeys, false, false>(t, dev, st));
}

mg_status backward_tc(const mg::AttnParams& p, const Device& dev, void* stream)
{
    const char* who = "mg_attention_backward";
    mg::TcAttnParams f = {};
    mg::TcBwdParams t = {};
    Scratch ws(dev, stream);
    cudaStream_t st = (cudaStream_t)stream;
    MG_TRY(tc_params(&f, p, dev, ws, st, who));
    t.a = p, t.doc_tiles = f.doc_tiles, t.scale = f.scale, t.curve = f.curve, t.status = f.status;
    t.idesc_s = mg::idesc_bf16(128, 64, false, false, p.scale < 0.f);
    t.Lp = ceil_div(p.Lq, 128) * 128;
    const int64_t rows = (int64_t)p.B * p.H * t.Lp;
    float* stats = static_cast<float*>(ws.get(2 * rows * sizeof(float)));
    if (!stats) return fail(MG_ERR_ALLOC, "%s: no scratch for the row sums", who);
    t.lse2 = stats, t.delta = stats + rows;
    mg::attn_tc_stats_kernel<__nv_bfloat16><<<ceil_div(rows, 16), 256, 0, st>>>(p, t.Lp, stats, stats + rows);
    MG_TRY(launched(who));
    int* hs = t.head_step;
    int* bs = t.batch_step;
    // the queries resident: dQ, and delta made exact
    MG_TRY(tc_map(&t.x0, &hs[0], &bs[0], p.q, p.qs, p.D, p.Lq, p.H, p.B, 128));
    MG_TRY(tc_map(&t.x1, &hs[3], &bs[3], p.dout, p.dos, p.D, p.Lq, p.H, p.B, 128));
    MG_TRY(tc_map(&t.y0, &hs[1], &bs[1], p.k, p.ks, p.D, p.Lk, p.Hkv, p.B, 64));
    MG_TRY(tc_map(&t.y1, &hs[2], &bs[2], p.v, p.vs, p.D, p.Lk, p.Hkv, p.B, 64));
    MG_TRY((p.D <= 64 ? launch_tc_backward<64, false>(t, dev, st) : launch_tc_backward<128, false>(t, dev, st)));
    // the keys resident: dK, dV
    MG_TRY(tc_map(&t.x0, &hs[1], &bs[1], p.k, p.ks, p.D, p.Lk, p.Hkv, p.B, 128));
    MG_TRY(tc_map(&t.x1, &hs[2], &bs[2], p.v, p.vs, p.D, p.Lk, p.Hkv, p.B, 128));
    MG_TRY(tc_map(&t.y0, &hs[0], &bs[0], p.q, p.qs, p.D, p.Lq, p.H, p.B, 64));
    MG_TRY(tc_map(&t.y1, &hs[3], &bs[3], p.dout, p.dos, p.D, p.Lq, p.H, p.B, 64));
    return p.D <= 64 ? launch_tc_backward<64, true>(t, dev, st) : launch_tc_backward<128, true>(t, dev, st);
}

template <int DP, bool kCap, bool kBias>
mg_status launch_tc32_forward(const mg::Tc32Params& t, const Device& dev, cudaStream_t st)
{
    constexpr auto kernel = mg::attn_tc32_forward<DP, kCap, kBias>;
    constexpr size_t smem = mg::tc32_forward_smem<DP>();
    MG_TRY(allow_smem<kernel>(dev, smem));
    kernel<<<ceil_div(t.a.Lq, 128) * t.a.B * t.a.H, mg::kTc32Threads, smem, st>>>(t);
    return launched("mg_attention");
}

template <int DP>
mg_status launch_tc32_forward(const mg::Tc32Params& t, const Device& dev, cudaStream_t st)
{
    const bool cap = t.a.cap > 0.f, bias = t.a.slopes != nullptr;
    return cap ? (bias ? launch_tc32_forward<DP, true, true>(t, dev, st) : launch_tc32_forward<DP, true, false>(t, dev, st))
               : (bias ? launch_tc32_forward<DP, false, true>(t, dev, st) : launch_tc32_forward<DP, false, false>(t, dev, st));
}

mg_status forward_tc32(const mg::AttnParams& p, const Device& dev, void* stream)
{
    mg::TcAttnParams f = {};
    Scratch ws(dev, stream);
    cudaStream_t st = (cudaStream_t)stream;
    MG_TRY(tc_params(&f, p, dev, ws, st, "mg_attention"));
    mg::Tc32Params t = {p, f.doc_tiles, mg::idesc_bf16(128, 64, false, false, p.scale < 0.f), f.scale, f.status};
    return p.D <= 64 ? launch_tc32_forward<64>(t, dev, st) : launch_tc32_forward<128>(t, dev, st);
}

template <int DP, bool kKeys, int kTake, bool kCap, bool kBias>
mg_status launch_tc32_backward(const mg::Tc32BwdParams& t, const Device& dev, cudaStream_t st)
{
    constexpr auto kernel = mg::attn_tc32_backward<DP, kKeys, kTake, kCap, kBias>;
    MG_TRY(allow_smem<kernel>(dev, mg::kTc32BwdSmem));
    const int blocks = kKeys ? ceil_div(t.a.Lk, 128) * t.a.B * t.a.Hkv : ceil_div(t.a.Lq, 128) * t.a.B * t.a.H;
    kernel<<<blocks, mg::kTc32BwdThreads, mg::kTc32BwdSmem, st>>>(t);
    return launched("mg_attention_backward");
}

template <int DP, bool kKeys, int kTake>
mg_status launch_tc32_backward(const mg::Tc32BwdParams& t, const Device& dev, cudaStream_t st)
{
    const bool cap = t.a.cap > 0.f, bias = t.a.slopes != nullptr;
    return cap ? (bias ? launch_tc32_backward<DP, kKeys, kTake, true, true>(t, dev, st)
                       : launch_tc32_backward<DP, kKeys, kTake, true, false>(t, dev, st))
               : (bias ? launch_tc32_backward<DP, kKeys, kTake, false, true>(t, dev, st)
                       : launch_tc32_backward<DP, kKeys, kTake, false, false>(t, dev, st));
}

mg_status backward_tc32(const mg::AttnParams& p, const Device& dev, void* stream)
{
    const char* who = "mg_attention_backward";
    mg::TcAttnParams f = {};
    Scratch ws(dev, stream);
    cudaStream_t st = (cudaStream_t)stream;
    MG_TRY(tc_params(&f, p, dev, ws, st, who));
    const int Lp = ceil_div(p.Lq, 128) * 128;
    const int64_t rows = (int64_t)p.B * p.H * Lp;
    float* stats = static_cast<float*>(ws.get(2 * rows * sizeof(float)));
    if (!stats) return fail(MG_ERR_ALLOC, "%s: no scratch for the row sums", who);
    mg::attn_tc_stats_kernel<float><<<ceil_div(rows, 16), 256, 0, st>>>(p, Lp, stats, stats + rows);
    MG_TRY(launched(who));
    mg::Tc32BwdParams t = {p, f.doc_tiles, stats, stats + rows, Lp, 0, f.scale, f.status};
    t.idesc_s = mg::idesc_bf16(128, p.D <= 64 ? 64 : 32, false, false, p.scale < 0.f);
    if (p.D <= 64) {
        MG_TRY((launch_tc32_backward<64, true, mg::kTakeBoth>(t, dev, st)));
        return launch_tc32_backward<64, false, mg::kTakeDs>(t, dev, st);
    }
    MG_TRY((launch_tc32_backward<128, true, mg::kTakeDs>(t, dev, st)));
    MG_TRY((launch_tc32_backward<128, true, mg::kTakeP>(t, dev, st)));
    return launch_tc32_backward<128, false, mg::kTakeDs>(t, dev, st);
}

// ---------------------------------------------------------------- paged
template <typename T, int DP>
mg_status launch_paged_kernel(const mg::PagedParams& p, const Device& dev, int blocks, bool cluster, cudaStream_t st)
{
    constexpr size_t smem = mg::paged_smem<T, DP>();
    if (!cluster) {
        MG_TRY((allow_smem<mg::paged_kernel<T, DP, false>>(dev, smem)));
        mg::paged_kernel<T, DP, false><<<blocks, mg::kPagedThreads, smem, st>>>(p);
        return MG_OK;
    }
    MG_TRY((allow_smem<mg::paged_kernel<T, DP, true>>(dev, smem)));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3(mg::kPagedThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute size = {};
    size.id = cudaLaunchAttributeClusterDimension;
    size.val.clusterDim.x = (unsigned)p.splits;
    size.val.clusterDim.y = size.val.clusterDim.z = 1;
    cfg.attrs = &size;
    cfg.numAttrs = 1;
    MG_HOST_TRY(cudaLaunchKernelEx(&cfg, mg::paged_kernel<T, DP, true>, p));
    return MG_OK;
}

// Splits: enough blocks to fill the GPU several times over, so that requests of
// uneven lengths even out, but no chunk shorter than 128 keys.
template <typename T>
mg_status launch_paged(mg::PagedParams& p, int longest, const Device& dev, Scratch& ws, cudaStream_t st,
                       const char* who)
{
    const int vec = 16 / (int)sizeof(T);
    bool stream = p.D % vec == 0 && aligned(p.k, p.ks, 3, sizeof(T), vec) && aligned(p.v, p.vs, 3, sizeof(T), vec);
    if (p.k_new) stream = stream && aligned(p.k_new, p.kns, 2, sizeof(T), vec) &&
                          aligned(p.v_new, p.vns, 2, sizeof(T), vec);
    const int group = p.H / p.Hkv, packs = ceil_div(group, stream ? mg::paged_pack<T>() : mg::kPagedHeads);
    const int64_t heads = (int64_t)p.B * p.Hkv * packs;
    const int64_t want = std::max<int64_t>(1, (int64_t)dev.sm_count * 24 / heads);
    const int most = std::max(1, ceil_div(longest, 128));
    int splits = (int)std::min<int64_t>(want, most);
    p.chunk = std::max(1, ceil_div(longest, splits));
    p.splits = splits = std::max(1, ceil_div(longest, p.chunk));
    if (heads * splits >= (1ll << 31) - 1) return fail(MG_ERR_UNSUPPORTED, "%s: batch is too large", who);
    p.curve = cap_curve(std::fabs(p.scale), p.cap);
    p.page_shift = -1;
    if (p.page > 0 && (p.page & (p.page - 1)) == 0)
        for (p.page_shift = 0; (1 << p.page_shift) < p.page;) ++p.page_shift;
    if ((int64_t)p.B * p.H >= (1ll << 31) - 1) return fail(MG_ERR_UNSUPPORTED, "%s: batch is too large", who);
    // few blocks, and no more chunks than a cluster may have: joined there
    const bool cluster = stream && splits > 1 && splits <= 8 && heads * splits <= dev.sm_count;
    if (splits > 1 && !cluster) {
        const size_t rows = (size_t)p.B * p.H * splits;
        const size_t part = (rows * p.D * sizeof(float) + 15) / 16 * 16;
        uint8_t* mem = static_cast<uint8_t*>(ws.get(part + rows * sizeof(float2)));
        p.part = reinterpret_cast<float*>(mem);
        p.stat = reinterpret_cast<float2*>(mem + part);
        if (!mem) return fail(MG_ERR_ALLOC, "%s: no scratch for %zu chunks", who, rows);
    }
    const int blocks = (int)(heads * splits);
    if (!stream) mg::paged_simt_kernel<T><<<blocks, mg::kPagedThreads, 0, st>>>(p);
    else MG_TRY((p.D <= 64 ? launch_paged_kernel<T, 64>(p, dev, blocks, cluster, st)
                           : launch_paged_kernel<T, 128>(p, dev, blocks, cluster, st)));
    MG_TRY(launched(who));
    if (splits > 1 && !cluster) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)(p.B * p.H));
        cfg.blockDim = dim3(mg::kJoinThreads);
        cfg.stream = st;
        cudaLaunchAttribute early = {};
        early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
        early.val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = &early;
        cfg.numAttrs = 1;
        MG_HOST_TRY(cudaLaunchKernelEx(&cfg, mg::paged_join_kernel<T>, p));
        MG_TRY(launched(who));
    }
    return MG_OK;
}

// ---------------------------------------------------------------- rotary
template <typename T, int VEC>
mg_status launch_rotary(mg::RotaryParams& p, const Device& dev, cudaStream_t st)
{
    p.units = p.pairs / VEC;
    p.tail_units = (p.D - 2 * p.pairs) / VEC;
    // Tokens of a block: enough that each thread has a pair's sines to compute and
    // a few items to turn, but blocks for the whole GPU where there are few tokens.
    const int64_t tokens = (int64_t)p.B * p.L, items = (int64_t)(p.H + p.Hkv) * (p.units + p.tail_units);
    int64_t per_block = std::max<int64_t>(1, std::min<int64_t>(std::min(mg::kRotaryTokens, mg::kRotaryThreads / std::max(1, p.pairs)),
                                                               tokens / (4 * dev.sm_count)));
    while (per_block > 1 && per_block * items > 8 * mg::kRotaryThreads) --per_block;
    p.tokens = (int)per_block;
    const int64_t blocks = (tokens + per_block - 1) / per_block;
    if (tokens + per_block >= (1ll << 31)) return fail(MG_ERR_UNSUPPORTED, "mg_rotary: too many tokens for one call");
    const size_t smem = (size_t)2 * per_block * p.pairs * sizeof(float);
    mg::rotary_kernel<T, VEC><<<(unsigned)blocks, mg::kRotaryThreads, smem, st>>>(p);
    return launched("mg_rotary");
}

}  // namespace

extern "C" {

mg_status mg_attention(const mg_attention_desc* d, void* out, float* lse, const void* q, const void* k,
                       const void* v, void* stream)
{
    Range range("mg_attention");
    MG_TRY(check_attention(d, "mg_attention"));
    if (d->batch == 0 || d->q_len == 0) return MG_OK;
    if (!out || !lse || !q || (d->k_len > 0 && (!k || !v)))
        return fail(MG_ERR_INVALID, "mg_attention: a tensor is NULL");
    Device dev;
    MG_TRY(mg::host::device(&dev));
    mg::AttnParams p = attention_params(d);
    p.out = out, p.lse = lse, p.q = q, p.k = k, p.v = v;
    cudaStream_t st = (cudaStream_t)stream;
    if (d->q_len == 1) {
        // One query: its row of keys is split over the GPU, as a paged cache of
        // one page per batch would be. Its position is the last key's, so that
        // causal and prefix masks hide nothing.
        mg::PagedParams g = {};
        g.B = p.B, g.H = p.H, g.Hkv = p.Hkv, g.D = p.D;
        g.scale = p.scale, g.cap = p.cap, g.slopes = p.slopes;
        g.length = p.Lk, g.docs = p.docs;
        g.qs[0] = p.qs[0], g.qs[1] = p.qs[1], g.os[0] = p.os[0], g.os[1] = p.os[1];
        g.ks[0] = p.ks[0], g.ks[1] = p.ks[2], g.ks[2] = p.ks[1];
        g.vs[0] = p.vs[0], g.vs[1] = p.vs[2], g.vs[2] = p.vs[1];
        g.q = q, g.k = const_cast<void*>(k), g.v = const_cast<void*>(v), g.out = out, g.lse = lse;
        g.status = dev.status;
        Scratch ws(dev, stream);
        return d->dtype == MG_F32 ? launch_paged<float>(g, p.Lk, dev, ws, st, "mg_attention")
                                  : launch_paged<__nv_bfloat16>(g, p.Lk, dev, ws, st, "mg_attention");
    }
    if (p.Lk > 0 && tc_serves(d, p, {q, out}, {k, v}))
        return d->dtype == MG_F32 ? forward_tc32(p, dev, stream) : forward_tc(p, dev, stream);
    return d->dtype == MG_F32 ? forward_simt<float>(p, st) : forward_simt<__nv_bfloat16>(p, st);
}

mg_status mg_attention_backward(const mg_attention_desc* d, void* dq, void* dk, void* dv, const void* dout,
                                const void* q, const void* k, const void* v, const void* out, const float* lse,
                                void* stream)
{
    Range range("mg_attention_backward");
    MG_TRY(check_attention(d, "mg_attention_backward"));
    if (d->batch == 0 || (d->q_len == 0 && d->k_len == 0)) return MG_OK;
    if ((d->q_len > 0 && (!dq || !dout || !q || !out || !lse)) || (d->k_len > 0 && (!dk || !dv || !k || !v)))
        return fail(MG_ERR_INVALID, "mg_attention_backward: a tensor is NULL");
    Device dev;
    MG_TRY(mg::host::device(&dev));
    mg::AttnParams p = attention_params(d);
    p.q = q, p.k = k, p.v = v, p.out = const_cast<void*>(out), p.dout = dout, p.lse = const_cast<float*>(lse);
    p.dq = dq, p.dk = dk, p.dv = dv;
    if (d->q_len > 0 && d->k_len > 0 && tc_serves(d, p, {q, out, dout, dq}, {k, v, dk, dv}))
        return d->dtype == MG_BF16 ? backward_tc(p, dev, stream) : backward_tc32(p, dev, stream);
    Scratch ws(dev, stream);
    if (d->q_len > 0) {
        p.delta = static_cast<float*>(ws.get(sizeof(float) * d->batch * d->heads * (size_t)d->q_len));
        if (!p.delta) return fail(MG_ERR_ALLOC, "mg_attention_backward: no scratch for the row sums");
    }
    cudaStream_t st = (cudaStream_t)stream;
    return d->dtype == MG_F32 ? backward_simt<float>(p, st) : backward_simt<__nv_bfloat16>(p, st);
}

mg_status mg_rotary(const mg_rotary_desc* d, void* out_q, void* out_k, const void* q, const void* k, void* stream)
{
    Range range("mg_rotary");
    if (!d) return fail(MG_ERR_INVALID, "mg_rotary: descriptor is NULL");
    if (d->dtype != MG_F32 && d->dtype != MG_BF16)
        return fail(MG_ERR_INVALID, "mg_rotary: dtype %d is neither MG_F32 nor MG_BF16", d->dtype);
    if (d->batch < 0 || d->heads < 0 || d->kv_heads < 0 || d->len < 0 || d->head_dim < 1)
        return fail(MG_ERR_INVALID, "mg_rotary: batch %d, heads %d, kv_heads %d, len %d, head_dim %d out of range",
                    d->batch, d->heads, d->kv_heads, d->len, d->head_dim);
    if (d->pairs < 0 || d->pairs > d->head_dim / 2)
        return fail(MG_ERR_INVALID, "mg_rotary: %d pairs do not fit a head of %d", d->pairs, d->head_dim);
    if (d->pairs > mg::kRotaryMaxPairs)
        return fail(MG_ERR_UNSUPPORTED, "mg_rotary: %d pairs, %d at most", d->pairs, mg::kRotaryMaxPairs);
    if (!std::isfinite(d->magnitude)) return fail(MG_ERR_INVALID, "mg_rotary: magnitude is not finite");
    const int kvh = k ? d->kv_heads : 0;
    if (d->batch == 0 || d->len == 0 || d->heads + kvh == 0) return MG_OK;
    if ((d->heads > 0 && (!q || !out_q)) || (kvh > 0 && !out_k))
        return fail(MG_ERR_INVALID, "mg_rotary: a tensor is NULL");
    if (d->pairs > 0 && (!d->positions || !d->frequencies))
        return fail(MG_ERR_INVALID, "mg_rotary: positions and frequencies are needed");
    Device dev;
    MG_TRY(mg::host::device(&dev));
    mg::RotaryParams p = {};
    p.B = d->batch, p.H = d->heads, p.Hkv = kvh, p.L = d->len, p.D = d->head_dim, p.pairs = d->pairs;
    p.interleaved = d->interleaved != 0, p.inverse = d->inverse != 0, p.magnitude = d->magnitude;
    // a dim of one element may carry any stride
    for (int i = 0; i < 3; ++i) {
        p.qs[i] = d->q_stride[i], p.ks[i] = d->k_stride[i];
        p.oqs[i] = d->out_q_stride[i], p.oks[i] = d->out_k_stride[i];
        const int n = i == 0 ? d->batch : d->len;   // a dim of one element may carry any stride
        if (i == 1 ? d->heads == 1 : n == 1) p.qs[i] = p.oqs[i] = 0;
        if (i == 1 ? kvh == 1 : n == 1) p.ks[i] = p.oks[i] = 0;
    }
    p.pos_stride = d->position_stride, p.positions = d->positions, p.frequencies = d->frequencies;
    p.q = q, p.k = k, p.oq = out_q, p.ok = out_k;
    // The widest vector that every row, the pairs and the rest of the head allow.
    const size_t e = elem_size(d->dtype);
    int vec = (int)(16 / e);
    while (vec > 1) {
        bool ok = p.pairs % vec == 0 && (p.D - 2 * p.pairs) % vec == 0;
        if (p.H) ok = ok && aligned(q, p.qs, 3, e, vec) && aligned(out_q, p.oqs, 3, e, vec);
        if (kvh) ok = ok && aligned(k, p.ks, 3, e, vec) && aligned(out_k, p.oks, 3, e, vec);
        if (ok) break;
        vec /= 2;
    }
    cudaStream_t st = (cudaStream_t)stream;
    using bf16 = __nv_bfloat16;
    if (d->dtype == MG_F32)
        return vec == 4 ? launch_rotary<float, 4>(p, dev, st)
             : vec == 2 ? launch_rotary<float, 2>(p, dev, st) : launch_rotary<float, 1>(p, dev, st);
    return vec == 8 ? launch_rotary<bf16, 8>(p, dev, st) : vec == 4 ? launch_rotary<bf16, 4>(p, dev, st)
         : vec == 2 ? launch_rotary<bf16, 2>(p, dev, st) : launch_rotary<bf16, 1>(p, dev, st);
}

mg_status mg_paged_attention(const mg_paged_desc* d, void* out, float* lse, const void* q, void* k_pages,
                             void* v_pages, const void* k_new, const void* v_new, void* stream)
{
    Range range("mg_paged_attention");
    const char* who = "mg_paged_attention";
    if (!d) return fail(MG_ERR_INVALID, "%s: descriptor is NULL", who);
    if (d->dtype != MG_F32 && d->dtype != MG_BF16)
        return fail(MG_ERR_INVALID, "%s: dtype %d is neither MG_F32 nor MG_BF16", who, d->dtype);
    if (d->batch < 0 || d->heads < 1 || d->kv_heads < 1 || d->page_size < 1 || d->pages < 0 || d->table_width < 0)
        return fail(MG_ERR_INVALID,
                    "%s: batch %d, heads %d, kv_heads %d, page_size %d, pages %d, table_width %d out of range", who,
                    d->batch, d->heads, d->kv_heads, d->page_size, d->pages, d->table_width);
    if (d->heads % d->kv_heads)
        return fail(MG_ERR_INVALID, "%s: heads %d is not a multiple of kv_heads %d", who, d->heads, d->kv_heads);
    if (d->head_dim < 1 || d->head_dim > MG_MAX_HEAD_DIM)
        return fail(MG_ERR_UNSUPPORTED, "%s: head_dim %d is outside 1..%d", who, d->head_dim, MG_MAX_HEAD_DIM);
    if (!std::isfinite(d->scale)) return fail(MG_ERR_INVALID, "%s: scale is not finite", who);
    if (!(d->cap >= 0.f) || !std::isfinite(d->cap))
        return fail(MG_ERR_INVALID, "%s: cap must be 0 (none) or a positive number", who);
    if ((k_new == nullptr) != (v_new == nullptr))
        return fail(MG_ERR_INVALID, "%s: k_new and v_new come together", who);
    if (d->batch == 0) return MG_OK;
    const int64_t longest = (int64_t)d->table_width * d->page_size;
    if (longest >= (1ll << 30)) return fail(MG_ERR_UNSUPPORTED, "%s: the block table is too wide", who);
    if (!out || !lse || !q || !d->lengths || (longest > 0 && (!k_pages || !v_pages || !d->block_table)))
        return fail(MG_ERR_INVALID, "%s: a tensor is NULL", who);
    Device dev;
    MG_TRY(mg::host::device(&dev));
    mg::PagedParams p = {};
    p.B = d->batch, p.H = d->heads, p.Hkv = d->kv_heads, p.D = d->head_dim;
    p.page = d->page_size, p.pages = d->pages, p.width = d->table_width;
    p.scale = d->scale, p.cap = d->cap;
    for (int i = 0; i < 3; ++i) p.ks[i] = d->k_stride[i], p.vs[i] = d->v_stride[i];
    for (int i = 0; i < 2; ++i) {
        p.qs[i] = d->q_stride[i], p.os[i] = d->out_stride[i];
        p.kns[i] = d->k_new_stride[i], p.vns[i] = d->v_new_stride[i];
    }
    p.table_stride = d->table_stride, p.slopes = d->slopes, p.table = d->block_table, p.lengths = d->lengths;
    p.q = q, p.k = k_pages, p.v = v_pages, p.k_new = k_new, p.v_new = v_new, p.out = out, p.lse = lse;
    p.status = dev.status;
    Scratch ws(dev, stream);
    cudaStream_t st = (cudaStream_t)stream;
    return d->dtype == MG_F32 ? launch_paged<float>(p, (int)longest, dev, ws, st, who)
                              : launch_paged<__nv_bfloat16>(p, (int)longest, dev, ws, st, who);
}

}  // extern "C"
