// mg_paged.cu -- host side and C ABI of rotary positions and of paged attention.
#include <cuda_runtime.h>

#include <algorithm>

#include "mg_attention_host.h"
#include "mg_paged.cuh"
#include "mg_rotary.cuh"

using namespace mg::host;

namespace {

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

// Splits: 16 blocks an SM, so that requests of uneven lengths even out, but no chunk
// shorter than 128 keys, or 512 where there are heads enough for the GPU (a block's
// start costs what 100 keys do: 113 -> 111 us for the 32 requests). Measured with 8 / 16 / 24 / 48: 32 requests of 1..8192 keys
// 120 / 102 / 105 / 120 us, two of 100 000 108 / 115 / 120 / 139 us.
template <typename T>
mg_status launch_paged(mg::PagedParams& p, int longest, const Device& dev, Scratch& ws, cudaStream_t st,
                       const char* who)
{
    const int vec = 16 / (int)sizeof(T);
    bool stream = tame(p.scale, p.cap) && p.D % vec == 0 && aligned(p.k, p.ks, 3, sizeof(T), vec) && aligned(p.v, p.vs, 3, sizeof(T), vec);
    if (p.k_new) stream = stream && aligned(p.k_new, p.kns, 2, sizeof(T), vec) &&
                          aligned(p.v_new, p.vns, 2, sizeof(T), vec);
    p.powers = stream;
    const int group = p.H / p.Hkv, packs = ceil_div(group, stream ? mg::paged_pack<T>() : mg::kPagedHeads);
    const int64_t heads = (int64_t)p.B * p.Hkv * packs;
    const int64_t want = std::max<int64_t>(1, (int64_t)dev.sm_count * 16 / heads);
    const int most = std::max(1, ceil_div(longest, 128));
    const int splits = p.splits = (int)std::min<int64_t>(want, most);
    p.least = heads >= dev.sm_count ? 512 : 128;
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
        cfg.blockDim = dim3(splits > 64 ? mg::kJoinThreads : mg::kJoinThreads / 4);
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

// A thread reads its own elements before it writes them, and none of another's.
mg_status check_rotary_places(const mg_rotary_desc* d, int kv_heads, const void* out_q, const void* out_k, const void* q,
                              const void* k)
{
    const char* who = "mg_rotary";
    const auto arg = [&](const char* name, const void* at, const int64_t* s, int heads) {
        return heads_arg(name, at, d->dtype, s, d->batch, heads, d->len, d->head_dim);
    };
    const Arg oq = arg("out_q", out_q, d->out_q_stride, d->heads), ok = arg("out_k", out_k, d->out_k_stride, kv_heads);
    const Arg iq = arg("q", q, d->q_stride, d->heads), ik = arg("k", k, d->k_stride, kv_heads);
    MG_TRY(apart(oq, iq, who, true));
    MG_TRY(apart(ok, ik, who, true));
    MG_TRY(apart(oq, ik, who));
    MG_TRY(apart(ok, iq, who));
    return apart(oq, ok, who);
}

mg_status check_paged_places(const mg_paged_desc* d, const void* out, const float* lse, const void* q,
                             const void* k_pages, const void* v_pages, const void* k_new, const void* v_new,
                             const char* who)
{
    const auto pool = [&](const char* name, const void* at, const int64_t* s) {
        return heads_arg(name, at, d->dtype, s, d->pages, d->page_size, d->kv_heads, d->head_dim);
    };
    const auto rows = [&](const char* name, const void* at, const int64_t* s, int heads) {
        return rows_arg(name, at, d->dtype, s, at ? d->batch : 0, heads, d->head_dim);
    };
    const Arg o = rows("out", out, d->out_stride, d->heads), l = lse_arg(lse, (int64_t)d->batch * d->heads);
    const Arg in[5] = {rows("q", q, d->q_stride, d->heads), pool("k_pages", k_pages, d->k_stride),
                       pool("v_pages", v_pages, d->v_stride), rows("k_new", k_new, d->k_new_stride, d->kv_heads),
                       rows("v_new", v_new, d->v_new_stride, d->kv_heads)};
    for (int i = 0; i < 5; ++i) {
        MG_TRY(apart(o, in[i], who, i == 0));
        MG_TRY(apart(l, in[i], who));
    }
    MG_TRY(apart(l, o, who));
    return k_new ? apart(in[1], in[2], who) : MG_OK;
}

}  // namespace

namespace mg {
namespace host {

mg_status single_query(const AttnParams& p, int dtype, const Device& dev, void* stream)
{
    PagedParams g = {};
    g.B = p.B, g.H = p.H, g.Hkv = p.Hkv, g.D = p.D;
    g.scale = p.scale, g.cap = p.cap, g.slopes = p.slopes;
    g.length = p.Lk, g.docs = p.docs;
    g.qs[0] = p.qs[0], g.qs[1] = p.qs[1], g.os[0] = p.os[0], g.os[1] = p.os[1];
    g.ks[0] = p.ks[0], g.ks[1] = p.ks[2], g.ks[2] = p.ks[1];
    g.vs[0] = p.vs[0], g.vs[1] = p.vs[2], g.vs[2] = p.vs[1];
    g.q = p.q, g.k = const_cast<void*>(p.k), g.v = const_cast<void*>(p.v), g.out = p.out, g.lse = p.lse;
    g.status = dev.status;
    Scratch ws(dev, stream);
    return dtype == MG_F32 ? launch_paged<float>(g, p.Lk, dev, ws, (cudaStream_t)stream, "mg_attention")
                              : launch_paged<__nv_bfloat16>(g, p.Lk, dev, ws, (cudaStream_t)stream, "mg_attention");
}

}  // namespace host
}  // namespace mg

extern "C" {

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
    MG_TRY(check_rotary_places(d, kvh, out_q, out_k, q, k));
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
    MG_TRY(check_scores(d->scale, d->cap, who));
    if ((k_new == nullptr) != (v_new == nullptr))
        return fail(MG_ERR_INVALID, "%s: k_new and v_new come together", who);
    if (d->batch == 0) return MG_OK;
    const int64_t longest = (int64_t)d->table_width * d->page_size;
    if (longest >= (1ll << 30)) return fail(MG_ERR_UNSUPPORTED, "%s: the block table is too wide", who);
    if (!out || !lse || !q || !d->lengths || (longest > 0 && (!k_pages || !v_pages || !d->block_table)))
        return fail(MG_ERR_INVALID, "%s: a tensor is NULL", who);
    MG_TRY(check_paged_places(d, out, lse, q, k_pages, v_pages, k_new, v_new, who));
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
