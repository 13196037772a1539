// mg_attention_host.h -- what the host sides of the attention operators share.
#pragma once

#include <atomic>
#include <cmath>

#include "mg_attention.h"
#include "mg_attention_math.cuh"
#include "mg_host.h"
#include "mg_overlap.h"

#define MG_TRY(call)                     \
    do {                                 \
        const mg_status s_ = (call);     \
        if (s_ != MG_OK) return s_;      \
    } while (0)

namespace mg {
namespace host {

inline int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

inline size_t elem_size(int dtype) { return dtype == MG_F32 ? 4 : 2; }

inline mg_status launched(const char* what)
{
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return fail(MG_ERR_CUDA, "%s: launch failed: %s", what, cudaGetErrorString(e));
    count_launch();
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

// Sizes of scale and cap that every kernel's products and powers of two stay in range for.
constexpr float kMostScale = 1e30f, kLeastCap = 1e-30f;

inline mg_status check_scores(float scale, float cap, const char* who)
{
    if (!(std::fabs(scale) <= kMostScale)) return fail(MG_ERR_INVALID, "%s: scale must be a number within +-1e30", who);
    if (cap != 0.f && !(cap >= kLeastCap && cap <= kMostScale))
        return fail(MG_ERR_INVALID, "%s: cap must be 0 (none) or within 1e-30..1e30", who);
    return MG_OK;
}

// Whether scale / cap is in range for the kernels that multiply by it (the others
// divide their scaled product by the cap).
inline bool tame(float scale, float cap)
{
    const double pre = std::fabs((double)scale / cap);
    return cap == 0.f || (pre > 1e-30 && pre < 1e30);
}

// Whether rows at `ptr` with these strides start on multiples of `vec` elements.
inline bool aligned(const void* ptr, const int64_t* strides, int n, size_t elem, int vec)
{
    if (reinterpret_cast<uintptr_t>(ptr) % (elem * vec)) return false;
    for (int i = 0; i < n; ++i)
        if (strides[i] % vec) return false;
    return true;
}

// A tensor by its argument's name, for the checks of where outputs lie.
struct Arg {
    const char* name;
    View view;
    Span span;
};

inline Arg heads_arg(const char* name, const void* at, int dtype, const int64_t* stride, int64_t n0, int64_t n1, int64_t n2,
                     int head_dim)
{
    const View v = {at, (int)elem_size(dtype), {n0, n1, n2, head_dim}, {stride[0], stride[1], stride[2], 1}};
    return {name, v, span_of(v)};
}
inline Arg rows_arg(const char* name, const void* at, int dtype, const int64_t* stride, int64_t n0, int64_t n1, int head_dim)
{
    const View v = {at, (int)elem_size(dtype), {n0, n1, 1, head_dim}, {stride[0], stride[1], 0, 1}};
    return {name, v, span_of(v)};
}
inline Arg lse_arg(const void* at, int64_t n)
{
    const View v = {at, 4, {n, 1, 1, 1}, {1, 0, 0, 0}};
    return {"lse", v, span_of(v)};
}

// Refuses an output that shares memory with `other`; `itself`: it may be the same elements in the same places.
inline mg_status apart(const Arg& out, const Arg& other, const char* who, bool itself = false)
{
    if (out.span.lo >= other.span.hi || other.span.lo >= out.span.hi) return MG_OK;
    if (!views_meet(out.view, other.view) || (itself && same_view(out.view, other.view))) return MG_OK;
    return fail(MG_ERR_INVALID, "%s: %s overlaps %s", who, out.name, other.name);
}

// The terms of the capped score's curve for products of magnitude |scale| (see CapCurve).
inline CapCurve cap_curve(float scale, float cap)
{
    CapCurve cc = {};
    if (!(cap > 0.f)) return cc;
    const double pre = (double)scale / cap, c[4] = {0.999999463558197, -0.33326318860054016, 0.13190296292304993,
                                                    -0.04440222308039665};
    cc.pre = (float)pre;
    cc.bound = pre > 1e-5 && pre < 1e4 ? (float)(0.5 / pre) : 0.f;
    double power = pre;
    for (int i = 0; i < 4; ++i, power *= pre * pre) cc.tc[i] = (float)(c[i] * power);
    return cc;
}

// Attention of one query per row (mg_paged.cu).
mg_status single_query(const AttnParams& p, int dtype, const Device& dev, void* stream);

}  // namespace host
}  // namespace mg
