// mg_attention.cu -- host side and C ABI of attention over whole rows and its
// gradients: checks of arguments, choice of kernel, scratch, launches.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <initializer_list>

#include "mg_attention_host.h"
#include "mg_attention_simt.cuh"
#include "mg_attention_tc.cuh"
#include "mg_attention_tc_bwd.cuh"
#include "mg_attention_tc32.cuh"
#include "mg_attention_tc32_bwd.cuh"

using namespace mg::host;

namespace {

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
    MG_TRY(check_scores(d->scale, d->cap, who));
    if (d->prefix && !d->causal) return fail(MG_ERR_INVALID, "%s: a prefix needs causal", who);
    if ((int64_t)d->q_len + d->k_len >= (1ll << 30)) return fail(MG_ERR_UNSUPPORTED, "%s: rows are too long", who);
    const int64_t rows = (int64_t)d->batch * d->heads * std::max(ceil_div(d->q_len, 32), ceil_div(d->k_len, 32));
    if (rows >= (1ll << 31) - 1) return fail(MG_ERR_UNSUPPORTED, "%s: batch * heads * rows is too large", who);
    return MG_OK;
}

// Blocks store their results while others still read the inputs.
mg_status check_places(const mg_attention_desc* d, const void* out, const float* lse, const void* q, const void* k,
                       const void* v, const char* who)
{
    const auto arg = [&](const char* name, const void* at, const int64_t* s, int heads, int rows) {
        return heads_arg(name, at, d->dtype, s, d->batch, heads, rows, d->head_dim);
    };
    const Arg o = arg("out", out, d->out_stride, d->heads, d->q_len), l = lse_arg(lse, (int64_t)d->batch * d->heads * d->q_len);
    const Arg in[3] = {arg("q", q, d->q_stride, d->heads, d->q_len), arg("k", k, d->k_stride, d->kv_heads, d->k_len),
                       arg("v", v, d->v_stride, d->kv_heads, d->k_len)};
    for (int i = 0; i < 3; ++i) {
        MG_TRY(apart(o, in[i], who, i == 0));       // a block of queries is read before its results take its place
        MG_TRY(apart(l, in[i], who));
    }
    return apart(l, o, who);
}

// dQ is written before dK and dV are computed.
mg_status check_gradient_places(const mg_attention_desc* d, const void* dq, const void* dk, const void* dv,
                                const void* dout, const void* q, const void* k, const void* v, const void* out,
                                const float* lse, const char* who)
{
    const auto arg = [&](const char* name, const void* at, const int64_t* s, bool key) {
        return heads_arg(name, at, d->dtype, s, d->batch, key ? d->kv_heads : d->heads, key ? d->k_len : d->q_len,
                         d->head_dim);
    };
    const Arg grad[3] = {arg("dq", dq, d->dq_stride, false), arg("dk", dk, d->dk_stride, true),
                         arg("dv", dv, d->dv_stride, true)};
    const Arg in[6] = {arg("q", q, d->q_stride, false),       arg("k", k, d->k_stride, true),
                       arg("v", v, d->v_stride, true),        arg("dout", dout, d->dout_stride, false),
                       arg("out", out, d->out_stride, false), lse_arg(lse, (int64_t)d->batch * d->heads * d->q_len)};
    for (int i = 0; i < 3; ++i) {
        for (const Arg& x : in) MG_TRY(apart(grad[i], x, who));
        for (int j = i + 1; j < 3; ++j) MG_TRY(apart(grad[i], grad[j], who));
    }
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

// The shared memory that kernel K may take is the kernel's, not the call's: it is set once, to
// what the longest heads take, so that calls of several host threads do not lower it for one another.
template <auto K>
mg_status simt_launch(int blocks, int rows_in_smem, int tiles33, const mg::AttnParams& p, const Device& dev,
                      cudaStream_t st, const char* what)
{
    const auto smem = [&](int D) {
        return sizeof(float) * ((size_t)rows_in_smem * mg::kSimtTile * (D + 1) + (size_t)tiles33 * mg::kSimtTile * 33);
    };
    MG_TRY(allow_smem<K>(dev, smem(mg::kSimtMaxD)));
    K<<<blocks, mg::kSimtThreads, smem(p.D), st>>>(p);
    return launched(what);
}

template <typename T>
mg_status forward_simt(const mg::AttnParams& p, const Device& dev, cudaStream_t st)
{
    return simt_launch<mg::attn_simt_forward<T>>(p.B * p.H * ceil_div(p.Lq, mg::kSimtTile), 3, 1, p, dev, st,
                                                 "mg_attention");
}

template <typename T>
mg_status backward_simt(const mg::AttnParams& p, const Device& dev, cudaStream_t st)
{
    const char* who = "mg_attention_backward";
    if (p.Lq > 0) {
        mg::attn_delta_kernel<T><<<ceil_div((int64_t)p.B * p.H * p.Lq, 8), 256, 0, st>>>(p);
        MG_TRY(launched(who));
        MG_TRY(simt_launch<mg::attn_simt_backward_dq<T>>(p.B * p.H * ceil_div(p.Lq, mg::kSimtTile), 4,
                                                         sizeof(T) == 2 ? 2 : 1, p, dev, st, who));
    }
    if (p.Lk > 0)
        MG_TRY(simt_launch<mg::attn_simt_backward_dkv<T>>(p.B * p.Hkv * ceil_div(p.Lk, mg::kSimtTile), 4, 2, p, dev,
                                                          st, who));
    return MG_OK;
}

// ---------------------------------------------------------------- tensor cores
// The tensor-core kernels read and store rows of whole 16-byte vectors, 16-bit
// tensors through TMA; a scale of 0 would turn their masked scores (-inf) into
// NaN. Everything else runs on the CUDA cores.
bool tc_serves(const mg_attention_desc* d, const mg::AttnParams& p, std::initializer_list<const void*> rows_q,
               std::initializer_list<const void*> rows_k)
{
    if (d->head_dim % 8 || std::fabs(d->scale) < 1e-30f || !tame(d->scale, d->cap)) return false;
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

// Parts of a row of keys: where the blocks (of 128 queries of a head) would leave
// places on the GPU empty, each row is shared by as many as fill them, of no less than 512
// keys each (the join costs a few microseconds). Scratch for more than one.
mg_status share_rows(mg::RowParts* r, const mg::AttnParams& p, int places, Scratch& ws)
{
    const int64_t blocks = (int64_t)ceil_div(p.Lq, 128) * p.B * p.H;
    r->parts = (int)std::max<int64_t>(1, std::min<int64_t>(places / blocks, ceil_div(p.Lk, 512)));
    if (r->parts == 1) return MG_OK;
    const int64_t rows = (int64_t)r->parts * p.B * p.H * p.Lq;
    r->out = static_cast<float*>(ws.get(rows * (p.D + 2) * sizeof(float)));      // p.D is a multiple of 8
    if (!r->out) return fail(MG_ERR_ALLOC, "mg_attention: no scratch for %d parts of each row", r->parts);
    r->stat = reinterpret_cast<float2*>(r->out + rows * p.D);
    return MG_OK;
}

template <typename T>
mg_status join_rows(const mg::RowParts& r, const mg::AttnParams& p, cudaStream_t st)
{
    if (r.parts == 1) return MG_OK;
    mg::attn_join_kernel<T><<<ceil_div((int64_t)p.B * p.H * p.Lq, 8), 256, 0, st>>>(p, r);
    return launched("mg_attention");
}

template <int DP, bool kCap, bool kBias>
mg_status launch_tc_forward(const mg::TcAttnParams& t, const Device& dev, cudaStream_t st)
{
    constexpr auto kernel = mg::attn_tc_forward<DP, kCap, kBias>;
    constexpr size_t smem = mg::tc_forward_smem<DP>();
    MG_TRY(allow_smem<kernel>(dev, smem));
    kernel<<<ceil_div(t.a.Lq, 128) * t.a.B * t.a.H * t.rows.parts, mg::kTcFwdThreads, smem, st>>>(t);
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
    MG_TRY(share_rows(&t.rows, p, 2 * dev.sm_count, ws));
    MG_TRY((p.D <= 64 ? launch_tc_forward<64>(t, dev, st) : launch_tc_forward<128>(t, dev, st)));
    return join_rows<__nv_bfloat16>(t.rows, p, st);
}

// Parts of a gradient's sum: where blocks (of 128 rows of a head, `steps` streamed tiles of
// `tile` rows each) would leave SMs empty, as many as fill them, joined in their order. No
// less than 256 rows to a part, 128 in fp32, whose rows take longer: measured with 256 / 128,
// fp32 4 heads of 64, 500 rows 54 / 42 us, bf16 16 heads over 1 of 128, 300 rows 55 / 58 us. Whole sums
// took 99 and 105 us; bf16 8 heads over 2 of 128, 2048 rows 178 -> 99 us, fp32 1024 rows 940 -> 213 us. (The
// share's arithmetic costs the fp32 kernel 2 % where every SM has its block: 219 -> 223 us.)
mg_status share_gradient(mg::GradParts* g, int64_t blocks, int64_t steps, int tile, int least, int64_t rows, int D,
                         bool second, bool sums, const Device& dev, Scratch& ws)
{
    *g = {};
    g->parts = (int)std::max<int64_t>(1, std::min<int64_t>(dev.sm_count / blocks, ceil_div(steps * tile, least)));
    if (g->parts == 1) return MG_OK;
    const int64_t each = g->parts * rows * D, accs = each * (second ? 2 : 1), all = accs + (sums ? g->parts * rows : 0);
    g->acc = static_cast<float*>(ws.get(all * sizeof(float)));
    if (!g->acc) return fail(MG_ERR_ALLOC, "mg_attention_backward: no scratch for %d parts of each sum", g->parts);
    if (second) g->other = g->acc + each;
    if (sums) g->r = g->acc + accs;
    return MG_OK;
}

// dQ's, and dK's and dV's.
mg_status share_dq(mg::GradParts* g, const mg::AttnParams& p, int tile, int least, bool correct, const Device& dev,
                   Scratch& ws)
{
    return share_gradient(g, (int64_t)ceil_div(p.Lq, 128) * p.B * p.H, ceil_div(p.Lk, tile), tile, least,
                          (int64_t)p.B * p.H * p.Lq, p.D, correct, true, dev, ws);
}
mg_status share_dkv(mg::GradParts* g, const mg::AttnParams& p, int tile, int least, const Device& dev, Scratch& ws)
{
    return share_gradient(g, (int64_t)ceil_div(p.Lk, 128) * p.B * p.Hkv, (int64_t)(p.H / p.Hkv) * ceil_div(p.Lq, tile),
                          tile, least, (int64_t)p.B * p.Hkv * p.Lk, p.D, true, false, dev, ws);
}

template <typename T, int kForm>
mg_status join_dq(const mg::GradParts& g, const mg::AttnParams& p, float* delta, float* fine, int Lp, cudaStream_t st)
{
    if (g.parts == 1) return MG_OK;
    mg::GradJoin j = {g, p.H, p.Lq, p.D, Lp, (int64_t)p.B * p.H * p.Lq, {p.dq, nullptr}, {}, delta, fine};
    std::copy(p.dqs, p.dqs + 3, j.os[0]);
    mg::attn_grad_join_kernel<T, kForm><<<ceil_div(j.rows, 8), 256, 0, st>>>(j);
    return launched("mg_attention_backward");
}
template <typename T>
mg_status join_dkv(const mg::GradParts& g, const mg::AttnParams& p, cudaStream_t st)
{
    if (g.parts == 1) return MG_OK;
    mg::GradJoin j = {g, p.Hkv, p.Lk, p.D, 0, (int64_t)p.B * p.Hkv * p.Lk, {p.dk, p.dv}, {}, nullptr, nullptr};
    std::copy(p.dks, p.dks + 3, j.os[0]);
    std::copy(p.dvs, p.dvs + 3, j.os[1]);
    mg::attn_grad_join_kernel<T, mg::kJoinPlain><<<dim3(ceil_div(j.rows, 8), 2), 256, 0, st>>>(j);
    return launched("mg_attention_backward");
}

template <int DP, bool kKeys, bool kCap, bool kBias>
mg_status launch_tc_backward(const mg::TcBwdParams& t, const Device& dev, cudaStream_t st)
{
    constexpr auto kernel = mg::attn_tc_backward<DP, kKeys, kCap, kBias>;
    constexpr size_t smem = mg::tc_backward_smem<DP>();
    MG_TRY(allow_smem<kernel>(dev, smem));
    const int blocks = kKeys ? ceil_div(t.a.Lk, 128) * t.a.B * t.a.Hkv : ceil_div(t.a.Lq, 128) * t.a.B * t.a.H;
    kernel<<<blocks * t.parts.parts, mg::kTcBwdThreads, smem, st>>>(t);
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
    mg::attn_tc_stats_kernel<__nv_bfloat16><<<ceil_div(rows, 16 * mg::kStatsRows), 256, 0, st>>>(p, t.Lp, stats, stats + rows);
    MG_TRY(launched(who));
    int* hs = t.head_step;
    int* bs = t.batch_step;
    // the queries resident: dQ, and delta made exact
    MG_TRY(tc_map(&t.x0, &hs[0], &bs[0], p.q, p.qs, p.D, p.Lq, p.H, p.B, 128));
    MG_TRY(tc_map(&t.x1, &hs[3], &bs[3], p.dout, p.dos, p.D, p.Lq, p.H, p.B, 128));
    MG_TRY(tc_map(&t.y0, &hs[1], &bs[1], p.k, p.ks, p.D, p.Lk, p.Hkv, p.B, 64));
    MG_TRY(tc_map(&t.y1, &hs[2], &bs[2], p.v, p.vs, p.D, p.Lk, p.Hkv, p.B, 64));
    MG_TRY(share_dq(&t.parts, p, 64, 256, true, dev, ws));
    MG_TRY((p.D <= 64 ? launch_tc_backward<64, false>(t, dev, st) : launch_tc_backward<128, false>(t, dev, st)));
    MG_TRY((join_dq<__nv_bfloat16, mg::kJoinCorrect>(t.parts, p, t.delta, nullptr, t.Lp, st)));
    // the keys resident: dK, dV
    MG_TRY(tc_map(&t.x0, &hs[1], &bs[1], p.k, p.ks, p.D, p.Lk, p.Hkv, p.B, 128));
    MG_TRY(tc_map(&t.x1, &hs[2], &bs[2], p.v, p.vs, p.D, p.Lk, p.Hkv, p.B, 128));
    MG_TRY(tc_map(&t.y0, &hs[0], &bs[0], p.q, p.qs, p.D, p.Lq, p.H, p.B, 64));
    MG_TRY(tc_map(&t.y1, &hs[3], &bs[3], p.dout, p.dos, p.D, p.Lq, p.H, p.B, 64));
    MG_TRY(share_dkv(&t.parts, p, 64, 256, dev, ws));
    MG_TRY((p.D <= 64 ? launch_tc_backward<64, true>(t, dev, st) : launch_tc_backward<128, true>(t, dev, st)));
    return join_dkv<__nv_bfloat16>(t.parts, p, st);
}

template <int DP, bool kCap, bool kBias>
mg_status launch_tc32_forward(const mg::Tc32Params& t, const Device& dev, cudaStream_t st)
{
    constexpr auto kernel = mg::attn_tc32_forward<DP, kCap, kBias>;
    constexpr size_t smem = mg::tc32_forward_smem<DP>();
    MG_TRY(allow_smem<kernel>(dev, smem));
    kernel<<<ceil_div(t.a.Lq, 128) * t.a.B * t.a.H * t.rows.parts, mg::kTc32Threads, smem, st>>>(t);
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
    mg::Tc32Params t = {p, f.doc_tiles, mg::idesc_bf16(128, 64, false, false, p.scale < 0.f), f.scale, {}, f.status};
    MG_TRY(share_rows(&t.rows, p, (p.D <= 64 ? 2 : 1) * dev.sm_count, ws));
    MG_TRY((p.D <= 64 ? launch_tc32_forward<64>(t, dev, st) : launch_tc32_forward<128>(t, dev, st)));
    return join_rows<float>(t.rows, p, st);
}

template <int DP, bool kKeys, int kTake, bool kCap, bool kBias>
mg_status launch_tc32_backward(const mg::Tc32BwdParams& t, const Device& dev, cudaStream_t st)
{
    constexpr auto kernel = mg::attn_tc32_backward<DP, kKeys, kTake, kCap, kBias>;
    MG_TRY(allow_smem<kernel>(dev, mg::kTc32BwdSmem));
    const int blocks = kKeys ? ceil_div(t.a.Lk, 128) * t.a.B * t.a.Hkv : ceil_div(t.a.Lq, 128) * t.a.B * t.a.H;
    kernel<<<blocks * t.parts.parts, mg::kTc32BwdThreads, mg::kTc32BwdSmem, st>>>(t);
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
    float* stats = static_cast<float*>(ws.get(3 * rows * sizeof(float)));
    if (!stats) return fail(MG_ERR_ALLOC, "%s: no scratch for the row sums", who);
    mg::attn_tc_stats_kernel<float><<<ceil_div(rows, 16 * mg::kStatsRows), 256, 0, st>>>(p, Lp, stats, stats + rows);
    MG_TRY(launched(who));
    mg::Tc32BwdParams t = {p, f.doc_tiles, stats, stats + rows, stats + 2 * rows, Lp, 0, f.scale, f.status};
    t.idesc_s = mg::idesc_bf16(128, p.D <= 64 ? 64 : 32, false, false, p.scale < 0.f);
    const int tile = p.D <= 64 ? 64 : 32;
    // dQ, and what the rows' lse are short of
    MG_TRY(share_dq(&t.parts, p, tile, 128, false, dev, ws));
    MG_TRY((p.D <= 64 ? launch_tc32_backward<64, false, mg::kTakeDs>(t, dev, st)
                      : launch_tc32_backward<128, false, mg::kTakeDs>(t, dev, st)));
    MG_TRY((join_dq<float, mg::kJoinWeights>(t.parts, p, nullptr, t.fine, Lp, st)));
    MG_TRY(share_dkv(&t.parts, p, tile, 128, dev, ws));
    if (p.D <= 64) {
        MG_TRY((launch_tc32_backward<64, true, mg::kTakeBoth>(t, dev, st)));
    } else {
        MG_TRY((launch_tc32_backward<128, true, mg::kTakeDs>(t, dev, st)));
        MG_TRY((launch_tc32_backward<128, true, mg::kTakeP>(t, dev, st)));
    }
    return join_dkv<float>(t.parts, p, st);
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
    MG_TRY(check_places(d, out, lse, q, k, v, "mg_attention"));
    Device dev;
    MG_TRY(mg::host::device(&dev));
    mg::AttnParams p = attention_params(d);
    p.out = out, p.lse = lse, p.q = q, p.k = k, p.v = v;
    cudaStream_t st = (cudaStream_t)stream;
    if (d->q_len == 1) {
        // One query: its row of keys is split over the GPU, as a paged cache of one page
        // per batch would be. Its position is the last key's, so that causal and prefix
        // masks hide nothing.
        return mg::host::single_query(p, d->dtype, dev, stream);
    }
    if (p.Lk > 0 && tc_serves(d, p, {q, out}, {k, v}))
        return d->dtype == MG_F32 ? forward_tc32(p, dev, stream) : forward_tc(p, dev, stream);
    return d->dtype == MG_F32 ? forward_simt<float>(p, dev, st) : forward_simt<__nv_bfloat16>(p, dev, st);
}

mg_status mg_attention_backward(const mg_attention_desc* d, void* dq, void* dk, void* dv, const void* dout,
                                const void* q, const void* k, const void* v, const void* out, const float* lse,
                                void* stream)
{
    Range range("mg_attention_backward");
    MG_TRY(check_attention(d, "mg_attention_backward"));
    // the row statistics are numbered in 32 bits, four rows of a head (padded to 128) at a time
    if ((int64_t)d->batch * d->heads * ceil_div(d->q_len, 128) >= (1ll << 27))
        return fail(MG_ERR_UNSUPPORTED, "mg_attention_backward: batch * heads * rows is too large");
    if (d->batch == 0 || (d->q_len == 0 && d->k_len == 0)) return MG_OK;
    if ((d->q_len > 0 && (!dq || !dout || !q || !out || !lse)) || (d->k_len > 0 && (!dk || !dv || !k || !v)))
        return fail(MG_ERR_INVALID, "mg_attention_backward: a tensor is NULL");
    MG_TRY(check_gradient_places(d, dq, dk, dv, dout, q, k, v, out, lse, "mg_attention_backward"));
    Device dev;
    MG_TRY(mg::host::device(&dev));
    mg::AttnParams p = attention_params(d);
    p.q = q, p.k = k, p.v = v, p.out = const_cast<void*>(out), p.dout = dout, p.lse = const_cast<float*>(lse);
    p.dq = dq, p.dk = dk, p.dv = dv;
    if (d->q_len > 0 && d->k_len > 0 && tc_serves(d, p, {q, out, dout, dq}, {k, v, dk, dv}))
        return d->dtype == MG_BF16 ? backward_tc(p, dev, stream) : backward_tc32(p, dev, stream);
    Scratch ws(dev, stream);
    if (d->q_len > 0) {
        const size_t rows = (size_t)d->batch * d->heads * d->q_len;
        p.delta = static_cast<float*>(ws.get(2 * rows * sizeof(float)));
        if (!p.delta) return fail(MG_ERR_ALLOC, "mg_attention_backward: no scratch for the row sums");
        p.fine = p.delta + rows;
    }
    cudaStream_t st = (cudaStream_t)stream;
    return d->dtype == MG_F32 ? backward_simt<float>(p, dev, st) : backward_simt<__nv_bfloat16>(p, dev, st);
}

}  // extern "C"
