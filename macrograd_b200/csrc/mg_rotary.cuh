// mg_rotary.cuh -- rotary positions: each pair (a, b) of a head turned by
// position * frequency.
//
// The angle of a far position (10^6 and more radians) has no correct digits in
// fp32, so it is kept in turns as a 64-bit fixed-point fraction: frequency / 2 pi
// as an unsigned 0.64 number, times the position modulo 2^64 -- the integer
// product drops whole turns exactly. Its upper 32 bits, read as a signed number,
// are the angle in [-1/2, 1/2) turns, and sincospi needs no further reduction.
// Frequencies below one turn a position are exact to 2^-53 of themselves, so the
// angle at position 2^31 is off by less than 2^-22 turns from the double's own.
//
// Bound by memory: every element is read once and written once. A block takes a few
// tokens: its threads first compute the tokens' sines and cosines, one pair each, into
// shared memory, and then turn all of the tokens' heads, VEC pairs at a time (two
// 16-byte vectors of a 16-bit head, VEC = 8), two items a thread on the way at once.
// With the sines in registers, for several heads of a thread, a gradient call of [2,
// 8192, 40, 128] took 87 us (16 lanes of state for each of 8 pairs left too few
// threads), here 67 us (76 % of the measured copy rate).
#pragma once

#include "mg_attention_math.cuh"

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
    int tokens;                 // tokens of a block
    int units, tail_units;      // vector units of a head's turning part and of its rest
};

constexpr int kRotaryThreads = 256;
constexpr int kRotaryTokens = 32;        // of a block at most
constexpr int kRotaryMaxPairs = 4096;     // a token's sines and cosines: 32 KB

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC < 16 ? sizeof(T) * VEC : 16) RotVec {
    T x[VEC];
};

// The pairs (x[i], y[i]).
template <typename T, int VEC>
__device__ __forceinline__ void turn_halves(RotVec<T, VEC>& x, RotVec<T, VEC>& y, const float* cs, const float* sn)
{
    if constexpr (VEC % 2 == 0) {
#pragma unroll
        for (int i = 0; i < VEC; i += 2) {
            const uint64_t a = pack2(to_f32(x.x[i]), to_f32(x.x[i + 1])), c = pack2(to_f32(y.x[i]), to_f32(y.x[i + 1]));
            const uint64_t co = pack2(cs[i], cs[i + 1]), si = pack2(sn[i], sn[i + 1]), ns = pack2(-sn[i], -sn[i + 1]);
            float r0, r1;
            unpack2(fma2(a, co, mul2(c, ns)), r0, r1);
            x.x[i] = from_f32<T>(r0), x.x[i + 1] = from_f32<T>(r1);
            unpack2(fma2(a, si, mul2(c, co)), r0, r1);
            y.x[i] = from_f32<T>(r0), y.x[i + 1] = from_f32<T>(r1);
        }
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const float a = to_f32(x.x[i]), c = to_f32(y.x[i]);
            x.x[i] = from_f32<T>(a * cs[i] - c * sn[i]);
            y.x[i] = from_f32<T>(a * sn[i] + c * cs[i]);
        }
    }
}
// Neighbours: x and y hold VEC pairs one after another.
template <typename T, int VEC>
__device__ __forceinline__ void turn_neighbours(RotVec<T, VEC>& x, RotVec<T, VEC>& y, const float* cs, const float* sn)
{
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        T* lo = 2 * i < VEC ? &x.x[(2 * i) % VEC] : &y.x[(2 * i) % VEC];
        T* hi = 2 * i + 1 < VEC ? &x.x[(2 * i + 1) % VEC] : &y.x[(2 * i + 1) % VEC];
        const float a = to_f32(*lo), c = to_f32(*hi);
        *lo = from_f32<T>(a * cs[i] - c * sn[i]);
        *hi = from_f32<T>(a * sn[i] + c * cs[i]);
    }
}

template <typename T, int VEC>
__global__ void __launch_bounds__(kRotaryThreads, 4) rotary_kernel(const __grid_constant__ RotaryParams p)
{
    using V = RotVec<T, VEC>;
    struct Rows {
        const T *q, *k;
        T *oq, *ok;
    };
    __shared__ Rows row[kRotaryTokens];
    extern __shared__ __align__(16) float rotary_sm[];
    float* cs = rotary_sm;                        // [tokens][pairs]
    float* sn = rotary_sm + p.tokens * p.pairs;
    const uint32_t token0 = blockIdx.x * (uint32_t)p.tokens, all = (uint32_t)p.B * (uint32_t)p.L;
    const int count = (int)min((uint32_t)p.tokens, all - token0);
    const int b0 = (int)(token0 / (uint32_t)p.L), l0 = (int)(token0 - (uint32_t)b0 * (uint32_t)p.L);
    // batch and place of the block's token t
    const auto where = [&](int t, int& b, int& l) {
        b = b0, l = l0 + t;
        while (l >= p.L) l -= p.L, ++b;
    };

    for (int t = threadIdx.x; t < count; t += kRotaryThreads) {
        int b, l;
        where(t, b, l);
        row[t] = {(const T*)p.q + b * p.qs[0] + l * p.qs[2], (const T*)p.k + b * p.ks[0] + l * p.ks[2],
                  (T*)p.oq + b * p.oqs[0] + l * p.oqs[2], (T*)p.ok + b * p.oks[0] + l * p.oks[2]};
    }
    for (int i = threadIdx.x; i < count * p.pairs; i += kRotaryThreads) {
        const int t = i / p.pairs, pair = i - t * p.pairs;
        int b, l;
        where(t, b, l);
        const int64_t pos = __ldg(p.positions + b * p.pos_stride + l);
        // turns a position as a signed 0.64 fixed-point number (whole turns dropped)
        double f = __ldg(p.frequencies + pair) * 0.15915494309189533577;   // 1 / (2 pi)
        f -= rint(f);
        const int64_t fixed = f >= 0.5 ? INT64_MIN : (int64_t)(f * 18446744073709551616.0);
        const uint64_t angle = (uint64_t)fixed * (uint64_t)pos;
        // the nearest 32-bit fraction: half turns of [-1, 1)
        const int32_t top = (int32_t)(uint32_t)((angle + 0x80000000ull) >> 32);
        float s, c;
        sincospif((float)top * 4.656612873077393e-10f, &s, &c);   // 2^-31
        cs[i] = c * p.magnitude;
        sn[i] = (p.inverse ? -s : s) * p.magnitude;
    }
    __syncthreads();

    // A thread keeps its place in the head (unit u) and walks the rows (token, head)
    // of the block; with more units than threads it takes several places in turn.
    const int heads = p.H + p.Hkv, per = p.units + p.tail_units;
    const int lanes = min(per, kRotaryThreads), rows = kRotaryThreads / lanes;
    const int mine = threadIdx.x / lanes;
    if (mine >= rows) return;
    for (int u = threadIdx.x % lanes; u < per; u += lanes) {
        const bool turns = u < p.units;
        const int at0 = !turns ? 2 * p.pairs + (u - p.units) * VEC : p.interleaved ? u * 2 * VEC : u * VEC;
        const int at1 = p.interleaved ? at0 + VEC : at0 + p.pairs;
        int t = 0, hh = mine;
        const auto step = [&]() {
            while (hh >= heads) hh -= heads, ++t;
        };
        step();
        while (t < count) {
            // two items at a time, their loads before their stores (a thread touches its
            // own elements alone, so that the output may be the input)
            V a[2], c[2];
            T* dst[2];
            int ts[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                ts[i] = t;
                if (t < count) {
                    const bool q = hh < p.H;
                    const T* src = q ? row[t].q + hh * p.qs[1] : row[t].k + (hh - p.H) * p.ks[1];
                    dst[i] = q ? row[t].oq + hh * p.oqs[1] : row[t].ok + (hh - p.H) * p.oks[1];
                    a[i] = *reinterpret_cast<const V*>(src + at0);
                    if (turns) c[i] = *reinterpret_cast<const V*>(src + at1);
                }
                hh += rows;
                step();
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (ts[i] >= count) break;
                if (turns) {
                    const RotVec<float, VEC> co = *reinterpret_cast<const RotVec<float, VEC>*>(cs + ts[i] * p.pairs + u * VEC);
                    const RotVec<float, VEC> si = *reinterpret_cast<const RotVec<float, VEC>*>(sn + ts[i] * p.pairs + u * VEC);
                    if (p.interleaved) turn_neighbours<T, VEC>(a[i], c[i], co.x, si.x);
                    else turn_halves<T, VEC>(a[i], c[i], co.x, si.x);
                    *reinterpret_cast<V*>(dst[i] + at1) = c[i];
                }
                *reinterpret_cast<V*>(dst[i] + at0) = a[i];
            }
        }
    }
}

}  // namespace mg
