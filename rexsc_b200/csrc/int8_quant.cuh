// Quantisation of values to 8 bits.
//
// A row with the largest magnitude a is held as  s = a / 127 (fp32)  and  q = rne(127 x / a), decided by the exact quotient.
// t = x * fl(127 / a) in fp32 is off by 2^-23 of it at the most.
//   * 16-bit x and a: the quotient is a border k + 1/2 or further than 2^-19 of its value from every border (with integers X, A
//     below 2^11 it is 127 X / (A 2^e), and 254 X - (2 k + 1) A 2^e is a whole number).  So t rounded to 21 bits, which borders
//     have, is a border where the quotient is one, and else on its side: rounding that to a whole number, ties to even, is q.
//   * fp32 values: a t further than 2^-16 from a border decides.  For the others, one in thirty thousand, the sign of the
//     remainder 127 x - border * a does, which fp32 gives exactly (quant_exact).
// A row of zeros has s = 0 and q = 0.  A row that holds an infinity or a NaN has s = NaN and q = 0: its products are NaN and
// nobody else's are.
#pragma once

#include <type_traits>

#include "int8.cuh"

namespace rexsc {

namespace {

constexpr float kMagic = 12582912.f; // 1.5 * 2^23: adding it rounds |t| < 2^22 to the nearest whole number, ties to even

// rne(127 x / a), |x| <= a, a > 0 finite.  Both are scaled by a power of two (exactly: a subnormal x is scaled up, and x is
// no smaller than a / 254 where the border decides).  r is the nearest whole number or, next to a border b = r +- 1/2, one of
// its two neighbours.  hi + lo = 127 x exactly; next to a border hi - b a is a multiple of 2^-24 of a's binade of less than
// 2^10 of them, so exact too, and adding lo to it cannot change the sign of the sum; elsewhere the sign is clear.
__device__ __noinline__ int quant_exact(float x, float a)
{
    const float f = a < 0x1p-60f ? 0x1p80f : a > 0x1p60f ? 0x1p-64f : 1.f;
    const float xs = x * f, as = a * f, inv = __fdiv_rn(127.f, as);
    const float r = __fsub_rn(__fmaf_rn(xs, inv, kMagic), kMagic);
    const float up = copysignf(1.f, __fmaf_rn(xs, inv, -r)), border = r + 0.5f * up;
    const float hi = __fmul_rn(127.f, xs), lo = __fmaf_rn(127.f, xs, -hi);
    const float over = __fadd_rn(__fmaf_rn(-border, as, hi), lo) * up; // > 0: beyond the border
    const int q = (int)r;
    return over > 0.f || (over == 0.f && (q & 1)) ? q + (int)up : q;
}

// four whole numbers' low bytes in one word
__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d)
{
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// x * inv to the nearest whole number in the low byte; far: how far off that is at the most
__device__ __forceinline__ uint32_t quant_near(float x, float inv, float &far)
{
    const float r = __fmaf_rn(x, inv, kMagic);
    far = fmaxf(far, fabsf(__fmaf_rn(x, inv, __fsub_rn(kMagic, r))));
    return __float_as_uint(r);
}
constexpr float kFar = 0.5f - 1.526e-5f; // further off than this: too near to a border

// q of eight values of a row whose largest magnitude is a > 0 (finite); inv = 127 / a, or 0 where that overflows.
// kShort: the values and a have 11 significant bits at the most.
template <bool kShort>
__device__ __forceinline__ uint2 quant8(const float (&x)[8], float a, float inv)
{
    uint32_t q[8];
    float far = 0.f;
    if constexpr (kShort) {
#pragma unroll
        for (int i = 0; i < 8; i++)
            q[i] = __float_as_uint(__fadd_rn(__uint_as_float((__float_as_uint(__fmul_rn(x[i], inv)) + 4u) & ~7u), kMagic));
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) q[i] = quant_near(x[i], inv, far);
    }
    if (far > kFar || inv == 0.f) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            float off = 0.f;
            quant_near(x[i], inv, off);
            if (off > kFar || inv == 0.f) q[i] = (uint32_t)quant_exact(x[i], a);
        }
    }
    return make_uint2(pack4(q[0], q[1], q[2], q[3]), pack4(q[4], q[5], q[6], q[7]));
}

__device__ __forceinline__ float inverse_of(float a) { return a < 7.9e-31f ? 0.f : __fdiv_rn(127.f, a); }

// eight neighbouring values as they lie in memory
template <typename T> struct Raw;
template <> struct Raw<float> {
    float v[8];
};
template <typename T> struct Raw {
    uint32_t w[4];
};
__device__ __forceinline__ void load_raw(const float *p, Raw<float> &r)
{
    const float4 a = *reinterpret_cast<const float4 *>(p), b = *reinterpret_cast<const float4 *>(p + 4);
    r.v[0] = a.x, r.v[1] = a.y, r.v[2] = a.z, r.v[3] = a.w, r.v[4] = b.x, r.v[5] = b.y, r.v[6] = b.z, r.v[7] = b.w;
}
template <typename T> __device__ __forceinline__ void load_raw(const T *p, Raw<T> &r)
{
    const uint4 u = *reinterpret_cast<const uint4 *>(p);
    r.w[0] = u.x, r.w[1] = u.y, r.w[2] = u.z, r.w[3] = u.w;
}
// from column c on, zeros behind the last column; vec: rows begin on 16 bytes
__device__ __forceinline__ void load_raw(const float *row, long long c, long long cols, bool vec, Raw<float> &r)
{
    if (vec && c + 8 <= cols) {
        load_raw(row + c, r);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) r.v[i] = c + i < cols ? row[c + i] : 0.f;
    }
}
template <typename T>
__device__ __forceinline__ void load_raw(const T *row, long long c, long long cols, bool vec, Raw<T> &r)
{
    if (vec && c + 8 <= cols) {
        load_raw(row + c, r);
    } else {
        const uint16_t *p = reinterpret_cast<const uint16_t *>(row);
#pragma unroll
        for (int i = 0; i < 4; i++)
            r.w[i] = (c + 2 * i < cols ? (uint32_t)p[c + 2 * i] : 0u) | (c + 2 * i + 1 < cols ? (uint32_t)p[c + 2 * i + 1] << 16 : 0u);
    }
}
__device__ __forceinline__ void clear_raw(Raw<float> &r)
{
#pragma unroll
    for (int i = 0; i < 8; i++) r.v[i] = 0.f;
}
template <typename T> __device__ __forceinline__ void clear_raw(Raw<T> &r) { r.w[0] = r.w[1] = r.w[2] = r.w[3] = 0u; }
__device__ __forceinline__ void widen(const Raw<float> &r, float (&v)[8])
{
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = r.v[i];
}
__device__ __forceinline__ void widen(const Raw<__half> &r, float (&v)[8])
{
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&r.w[i]));
        v[2 * i] = f.x, v[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ void widen(const Raw<__nv_bfloat16> &r, float (&v)[8])
{
#pragma unroll
    for (int i = 0; i < 4; i++) v[2 * i] = __uint_as_float(r.w[i] << 16), v[2 * i + 1] = __uint_as_float(r.w[i] & 0xffff0000u);
}
// Largest magnitude of what has been seen, as bits (of an fp32, or of two 16-bit values side by side): ordered like the
// values, infinities above them, NaNs above those.
__device__ __forceinline__ void most_of(const Raw<float> &r, uint32_t &most)
{
#pragma unroll
    for (int i = 0; i < 8; i++) most = max(most, __float_as_uint(r.v[i]) & 0x7fffffffu);
}
template <typename T> __device__ __forceinline__ void most_of(const Raw<T> &r, uint32_t &most)
{
#pragma unroll
    for (int i = 0; i < 4; i++) most = __vmaxu2(most, r.w[i] & 0x7fff7fffu);
}
template <typename T> __device__ __forceinline__ uint32_t most_as_f32(uint32_t most)
{
    if constexpr (sizeof(T) == 4) return most;
    most = max(most & 0xffffu, most >> 16);
    if constexpr (std::is_same<T, __half>::value) return __float_as_uint(__half2float(__ushort_as_half((unsigned short)most)));
    return most << 16;
}

} // namespace

} // namespace rexsc
