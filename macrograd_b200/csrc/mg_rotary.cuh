// mg_rotary.cuh -- rotary positions: each pair (a, b) of a head turned by
// position * frequency.
//
// The angle of a far position (10^6 and more radians) has no correct digits in
// fp32, so it is kept in turns as a 64-bit fixed-point fraction: frequency / 2 pi
// as an unsigned 0.64 number, times the position modulo 2^64 -- the integer
// product drops whole turns exactly. Its upper 32 bits, read as a signed number,
// are the angle in (-1/2, 1/2] turns, and sincospi needs no further reduction.
// Frequencies below one turn a position are exact to 2^-53 of themselves, so the
// angle at position 2^31 is off by less than 2^-22 turns from the double's own.
//
// Bound by memory: every element is read once and written once. A thread turns
// VEC pairs (two 16-byte vectors of a 16-bit head, VEC = 8) and uses their sines
// for `heads_per_thread` heads of the same token.
#pragma once

#include "mg_attention_common.cuh"

namespace mg {

struct RotaryParams {
    int B, H, Hkv, L, D, pairs;
    int interleaved, inverse;
    float magnitude;
    int64_t qs[3], ks[3], oqs[3], oks[3];
    int64_t pos_stride;
    const int32_t* positions;
    const double* frequencies;
    const void *q, *k;
    void *oq, *ok;
    int heads_per_thread;       // heads one thread turns
    int groups;                 // ceil((H + Hkv) / heads_per_thread)
    int units, tail_units;      // vector units of the turning part and of the rest
    int64_t total;              // B * L * groups * (units + tail_units)
};

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) RotVec {
    T x[VEC];
};

template <typename T, int VEC>
__global__ void __launch_bounds__(128) rotary_kernel(const __grid_constant__ RotaryParams p)
{
    using V = RotVec<T, VEC>;
    const int64_t t = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (t >= p.total) return;
    const int per = p.units + p.tail_units;
    const int u = (int)(t % per);
    const int64_t rest = t / per;
    const int group = (int)(rest % p.groups);
    const int64_t token = rest / p.groups;
    const int l = (int)(token % p.L), b = (int)(token / p.L);

    float cs[VEC], sn[VEC];
    int64_t at0, at1;           // element offsets of the thread's two vectors
    const bool turns = u < p.units;
    if (turns) {
        const int64_t pos = __ldg(p.positions + b * p.pos_stride + l);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            // turns a position as a signed 0.64 fixed-point number (whole turns dropped)
            double f = __ldg(p.frequencies + u * VEC + i) * 0.15915494309189533577;   // 1 / (2 pi)
            f -= rint(f);
            const int64_t fixed = f >= 0.5 ? INT64_MIN : (int64_t)(f * 18446744073709551616.0);
            const uint64_t angle = (uint64_t)fixed * (uint64_t)pos;
            // the nearest 32-bit fraction: half turns of (-1, 1]
            const int32_t top = (int32_t)(uint32_t)((angle + 0x80000000ull) >> 32);
            sincospif((float)top * 4.656612873077393e-10f, &sn[i], &cs[i]);   // 2^-31
            if (p.inverse) sn[i] = -sn[i];
            sn[i] *= p.magnitude;
            cs[i] *= p.magnitude;
        }
        at0 = p.interleaved ? (int64_t)u * 2 * VEC : (int64_t)u * VEC;
        at1 = p.interleaved ? at0 + VEC : at0 + p.pairs;
    } else {
        at0 = 2 * (int64_t)p.pairs + (int64_t)(u - p.units) * VEC;
        at1 = at0;
    }
    const int h1 = min(p.H + p.Hkv, (group + 1) * p.heads_per_thread);
#pragma unroll 4
    for (int hh = group * p.heads_per_thread; hh < h1; ++hh) {
        const bool isq = hh < p.H;
        const int h = isq ? hh : hh - p.H;
        const T* src;
        T* dst;
        if (isq) {
            src = (const T*)p.q + b * p.qs[0] + h * p.qs[1] + l * p.qs[2];
            dst = (T*)p.oq + b * p.oqs[0] + h * p.oqs[1] + l * p.oqs[2];
        } else {
            src = (const T*)p.k + b * p.ks[0] + h * p.ks[1] + l * p.ks[2];
            dst = (T*)p.ok + b * p.oks[0] + h * p.oks[1] + l * p.oks[2];
        }
        V x = *reinterpret_cast<const V*>(src + at0);
        if (!turns) {
            *reinterpret_cast<V*>(dst + at0) = x;
            continue;
        }
        V y = *reinterpret_cast<const V*>(src + at1);
        if (p.interleaved) {
            // vectors (x, y) hold VEC pairs of neighbours
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                T* lo = 2 * i < VEC ? &x.x[(2 * i) % VEC] : &y.x[(2 * i) % VEC];
                T* hi = 2 * i + 1 < VEC ? &x.x[(2 * i + 1) % VEC] : &y.x[(2 * i + 1) % VEC];
                const float a = to_f32(*lo), c = to_f32(*hi);
                *lo = from_f32<T>(a * cs[i] - c * sn[i]);
                *hi = from_f32<T>(a * sn[i] + c * cs[i]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float a = to_f32(x.x[i]), c = to_f32(y.x[i]);
                x.x[i] = from_f32<T>(a * cs[i] - c * sn[i]);
                y.x[i] = from_f32<T>(a * sn[i] + c * cs[i]);
            }
        }
        *reinterpret_cast<V*>(dst + at0) = x;
        *reinterpret_cast<V*>(dst + at1) = y;
    }
}

}  // namespace mg
