// AdamW over many tensors at once, moments in 32 or in 8 bits.
//
//   g' = g / grad_scale         m' = b1 m + (1 - b1) g'        v' = b2 v + (1 - b2) g'^2
//   p' = p (1 - lr wd) - lr / (1 - b1^t) * m' / (sqrt(v') / sqrt(1 - b2^t) + eps)
//
// in fp32; t is the number of steps including this one and lives on the device, so a step can be captured into a graph and a
// step that a GradScaler's found_inf cancels leaves everything, t included, as it was.
//
// The moments of all tensors of a group lie in flat buffers in which every tensor begins on a block of 256 elements; a warp
// updates a block, eight neighbouring elements per lane.  The list of tensors travels as a kernel argument: no table in
// device memory that a captured graph or another stream could share, and one launch for up to 640 tensors.
//
// 8 bits: a block holds m as sm * e4m3 and r = sqrt(v) as sr * e4m3, sm = max|m'| / 448, sr = max r' / 448 (r and not v: its
// range is half as many octaves, 17.8 of which e4m3 covers).  Values are cut to e4m3 and rounded up where the cut-off
// fraction plus a threshold u reaches a step; u = frac(place * a + t * b) is equidistributed over the steps of one place and
// over the places of one step.  Rounding to nearest would freeze v: it decays by 0.1 % a step, r by 0.05 %, where half a step
// of e4m3 is 3 to 6 %.  With u the mean over the steps is right, without random numbers whose state a checkpoint would have
// to carry.  r' > 0 is never stored as 0: a later step would divide by eps alone.  A block whose largest value is below
// 2^-100 is stored as zeros.  A gradient that is no finite number makes its element's moments so, and in 8 bits its block's.
//
// What bounds it.  32-bit moments: memory, 28 bytes an element with fp32 weights and gradients (134M bf16 gradients on fp32
// weights in 530 us, 6.58 TB/s).  8-bit moments: arithmetic; 16 bytes an element, or 10 with bf16 weights and gradients, would
// take 206 us for 134M of those, and 54 instructions an element take 300.
#include <cuda_fp8.h>
#include <math.h>
#include <type_traits>

#include "int8.cuh"

namespace rexsc {

namespace {

constexpr int kBlock = 256;      // elements of a block (of a scale)
// With 8-bit moments the arithmetic needs 96 registers a thread: five CTAs of 128 threads fit an SM (two of 256: 4 % slower).
// With 32-bit ones three CTAs an SM that stay (6.65 TB/s on 134M fp32 weights) are better than more of them in turns (6.4).
template <bool kBits8> constexpr int kThreadsOf = kBits8 ? 128 : 256;
template <bool kBits8> constexpr int kCtasOf = kBits8 ? 5 : 3;
constexpr int kSmallList = 64, kLargeList = 640;

struct AdamTensor {
    void *p;
    const void *g;
    long long n;
    unsigned first;  // its first block
    int vec;         // p and g can be read eight elements at a time
};

struct AdamArgs {
    float *m, *v;                    // 32-bit moments, or null
    uint8_t *m8, *r8;                // 8-bit moments
    float *ms, *rs;
    long long *step;                 // [0] steps so far, [1] blocks of this launch that are done
    const float *lr_ptr, *grad_scale, *found_inf;
    float lr, b1, c1, b2, c2, eps, wd;
    double log_b1, log_b2;
    int g_dtype, tensors, advance;   // advance: the last launch of the step counts it
    unsigned first, last;            // blocks of this launch
};

template <int kList>
struct AdamLaunch {
    AdamArgs a;
    AdamTensor t[kList];
};

__device__ __forceinline__ void load8v(const float *p, float (&v)[8])
{
    asm volatile("ld.global.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]) : "l"(p));
}
// Eight neighbouring elements as they lie in memory (16-bit types: in the first four words)
struct Raw8 {
    uint32_t w[8];
};
__device__ __forceinline__ void load_raw(const void *p, int dtype, Raw8 &r)
{
    if (dtype == REXSC_F32) {
        asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(r.w[0]), "=r"(r.w[1]), "=r"(r.w[2]), "=r"(r.w[3]), "=r"(r.w[4]), "=r"(r.w[5]), "=r"(r.w[6]), "=r"(r.w[7])
                     : "l"(p));
    } else {
        const uint4 u = *static_cast<const uint4 *>(p);
        r.w[0] = u.x, r.w[1] = u.y, r.w[2] = u.z, r.w[3] = u.w;
    }
}
// one at a time, `left` of them; the others are 0
__device__ __forceinline__ void load_some(const void *p, int dtype, int left, Raw8 &r)
{
    if (dtype == REXSC_F32) {
        const uint32_t *q = static_cast<const uint32_t *>(p);
#pragma unroll
        for (int i = 0; i < 8; i++) r.w[i] = i < left ? q[i] : 0u;
    } else {
        const uint16_t *q = static_cast<const uint16_t *>(p);
#pragma unroll
        for (int i = 0; i < 4; i++)
            r.w[i] = (2 * i < left ? (uint32_t)q[2 * i] : 0u) | (2 * i + 1 < left ? (uint32_t)q[2 * i + 1] << 16 : 0u);
    }
}
__device__ __forceinline__ void widen(const Raw8 &r, int dtype, float (&v)[8])
{
    if (dtype == REXSC_F32) {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = __uint_as_float(r.w[i]);
    } else if (dtype == REXSC_F16) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&r.w[i]));
            v[2 * i] = f.x, v[2 * i + 1] = f.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) v[2 * i] = __uint_as_float(r.w[i] << 16), v[2 * i + 1] = __uint_as_float(r.w[i] & 0xffff0000u);
    }
}
template <typename T> constexpr int kDtypeOf = sizeof(T) == 4 ? REXSC_F32 : std::is_same<T, __half>::value ? REXSC_F16 : REXSC_BF16;
__device__ __forceinline__ void store8v(float *p, const float (&v)[8])
{
    asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(v[0]), "f"(v[1]), "f"(v[2]),
                 "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]) : "memory");
}
__device__ __forceinline__ void store8v(__half *p, const float (&v)[8])
{
    __half2 h[4];
#pragma unroll
    for (int i = 0; i < 4; i++) h[i] = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
    *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<const uint4 *>(h);
}
__device__ __forceinline__ void store8v(__nv_bfloat16 *p, const float (&v)[8])
{
    __nv_bfloat162 h[4];
#pragma unroll
    for (int i = 0; i < 4; i++) h[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
    *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<const uint4 *>(h);
}
template <typename T> __device__ __forceinline__ T narrow(float v);
template <> __device__ __forceinline__ float narrow<float>(float v) { return v; }
template <> __device__ __forceinline__ __half narrow<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// two fp32 in a register pair; every operation rounds each of them as the scalar one does
typedef unsigned long long Pair;
__device__ __forceinline__ Pair pair(float lo, float hi)
{
    Pair r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ Pair both(float v) { return pair(v, v); }
__device__ __forceinline__ void apart(Pair p, float &lo, float &hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(p)); }
__device__ __forceinline__ Pair mul2(Pair a, Pair b)
{
    Pair d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
// (by halves: from a product and an addition of pairs the compiler makes one operation with one rounding, .rn or not)
__device__ __forceinline__ Pair add2(Pair a, Pair b)
{
    float a0, a1, b0, b1;
    apart(a, a0, a1);
    apart(b, b0, b1);
    return pair(__fadd_rn(a0, b0), __fadd_rn(a1, b1));
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c)
{
    Pair d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}

// eight e4m3 codes (4 exponent bits with bias 7, 3 of mantissa, steps of 2^-9 below 2^-6), times a scale
__device__ __forceinline__ void from_e4m3(uint2 codes, float scale, Pair (&v)[4])
{
    const Pair s = both(scale);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t two = i < 2 ? codes.x : codes.y;
        const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(i & 1 ? two >> 16 : two & 0xffff), __NV_E4M3);
        const float2 f = __half22float2(__half2(h));
        v[i] = mul2(pair(f.x, f.y), s);
    }
}
// The magnitude of y, at most 448, to e4m3, rounded up by the threshold u / 2^20.  From 2^-6 on the fraction is the low 20 bits
// of y's mantissa; below, steps are 2^-9 and the fraction that of |y| * 2^9 plus the threshold, a sum in fp32 whose whole part
// an addition of 2^23 that rounds down leaves in the low bits.  (Only the low byte counts: y's sign does not reach it.)
__device__ __forceinline__ uint32_t to_e4m3_normal(float y, uint32_t u) { return (__float_as_uint(y) + u - ((127u - 7u) << 23)) >> 20; }
__device__ __forceinline__ uint32_t to_e4m3_small(float y, uint32_t u)
{
    const float part = __fadd_rn(__uint_as_float(0x3f800000u | u << 3), -1.f);
    return __float_as_uint(__fadd_rd(__fmaf_rn(fabsf(y), 512.f, part), 8388608.f));
}
// byte `at` of four words
__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d, uint32_t at)
{
    const uint32_t sel = at | (at + 4) << 4;
    return __byte_perm(__byte_perm(a, b, sel), __byte_perm(c, d, sel), 0x5410);
}
// Eight values y in units of a block's scale as e4m3, without their signs; over: the largest of the block is above 448 (by a
// rounding); least: what is not 0 is not stored as 0.  Blocks whose values all lie above 2^-6 (1 / 28672 of the largest) skip
// the small steps.
__device__ __forceinline__ uint2 store_e4m3(float (&y)[8], bool over, const uint32_t (&u)[8], bool least)
{
    float low = 448.f;
#pragma unroll
    for (int i = 0; i < 8; i++) low = fminf(low, fabsf(y[i]));
    if (over) { // (the same for the block)
#pragma unroll
        for (int i = 0; i < 8; i++) y[i] = fminf(fmaxf(y[i], -448.f), 448.f);
    }
    uint32_t c[8];
#pragma unroll
    for (int i = 0; i < 8; i++) c[i] = to_e4m3_normal(y[i], u[i]);
    if (low < 0x1p-6f) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            if (fabsf(y[i]) < 0x1p-6f) c[i] = to_e4m3_small(y[i], u[i]) & 0xff;
            if (least && fabsf(y[i]) > 0.f) c[i] = max(c[i], 1u);
        }
    }
    return make_uint2(pack4(c[0], c[1], c[2], c[3], 0) & 0x7f7f7f7fu, pack4(c[4], c[5], c[6], c[7], 0) & 0x7f7f7f7fu);
}
__device__ __forceinline__ float max_nan(float a, float b)
{
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// Of -v, v > 0, the root's negative: rsqrt's estimate y of 1 / sqrt(v), g = v y, and Newton's step g + (v - g^2) y / 2, whose
// error before its rounding is below 2^-42 of the root: correctly rounded but where a root lies that near to the middle of
// two numbers, and then one of them (none of 10^9 random values differed from sqrt.rn, which takes twice the instructions).
// For v in [2^-100, 2^126] only.
__device__ __forceinline__ Pair minus_root(Pair minus_v, float v0, float v1)
{
    float y0, y1;
    asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y0) : "f"(v0));
    asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y1) : "f"(v1));
    const Pair y = pair(y0, y1), q = mul2(minus_v, y);
    return fma2(fma2(q, q, minus_v), mul2(y, both(0.5f)), q);
}
__device__ __forceinline__ float reciprocal(float x)
{
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// kSame: gradients have the weights' type (known here: a tenth of the time with 8-bit moments)
template <typename P, bool kBits8, bool kSame, int kList>
__global__ void __launch_bounds__(kThreadsOf<kBits8>, kCtasOf<kBits8>)
adamw_kernel(const __grid_constant__ AdamLaunch<kList> l)
{
    const AdamArgs &a = l.a;
    wait_previous_launch(); // (the next one does not begin before this one's end: it may read weights before it waits)
    if (a.found_inf && *a.found_inf != 0.f) return;
    const int lane = threadIdx.x & 31;
    const long long t = a.step[0] + 1;
    const float lr = a.lr_ptr ? *a.lr_ptr : a.lr;
    const float unscale = a.grad_scale ? __fdiv_rn(1.f, *a.grad_scale) : 1.f;
    const float keep = 1.f - lr * a.wd;
    const float size = lr / -expm1f((float)((double)t * a.log_b1));
    const float root = rsqrtf(-expm1f((float)((double)t * a.log_b2)));
    constexpr int kWarps = kThreadsOf<kBits8> / 32;
    const unsigned warps = gridDim.x * kWarps;

    // A block's inputs.  With 8-bit moments those of the next one are under way during the computation for this one, which
    // is long enough that the warps an SM holds would not cover the memory's latency.
    struct Block {
        P *p_at;  // this lane's elements of the weights
        int left; // how many of its eight exist; -1: a block of no tensor of the list
        int vec;
        Raw8 p, g;
        uint2 cm, cr;
        float sm, sr;
    };
    // the tensor that blocks are taken from: its blocks, and its pointers as if it began at block 0 (the flat buffers' place
    // is then its offset too; most blocks need nothing else)
    int at = -1;
    unsigned first = 0, end = 0, whole = 0; // whole: blocks up to here lie wholly in the tensor
    P *p_base = nullptr;
    const char *g_base = nullptr;
    const int g_dtype = kSame ? kDtypeOf<P> : a.g_dtype, g_size = g_dtype == REXSC_F32 ? 4 : 2;
    auto load = [&](unsigned b, Block &x) {
        if (b >= end) {
            // the last tensor that begins at b or before; blocks only rise, so the search goes on from where it was
            int lo = at < 0 ? 0 : at, hi = a.tensors;
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (l.t[mid].first <= b) lo = mid; else hi = mid;
            }
            if (lo != at) {
                at = lo;
                const AdamTensor &t = l.t[lo];
                first = t.first;
                end = first + (unsigned)((t.n + kBlock - 1) / kBlock);
                whole = t.vec ? first + (unsigned)(t.n / kBlock) : first;
                p_base = static_cast<P *>(t.p) - (size_t)first * kBlock;
                g_base = static_cast<const char *>(t.g) - (size_t)first * kBlock * g_size;
            }
            if (b >= end) {
                x.left = -1;
                return;
            }
        }
        const size_t pos = (size_t)b * kBlock + lane * 8;
        x.p_at = p_base + pos;
        const char *g_at = g_base + pos * g_size;
        if (b < whole) {
            x.left = 8, x.vec = 1;
            load_raw(x.p_at, kDtypeOf<P>, x.p);
            load_raw(g_at, g_dtype, x.g);
        } else {
            const AdamTensor &t = l.t[at];
            const long long left = t.n - ((long long)(b - first) * kBlock + lane * 8);
            x.left = left < 0 ? 0 : left < 8 ? (int)left : 8, x.vec = t.vec;
            load_some(x.p_at, kDtypeOf<P>, x.left, x.p);
            load_some(g_at, g_dtype, x.left, x.g);
        }
        if constexpr (kBits8) {
            x.cm = *reinterpret_cast<const uint2 *>(a.m8 + pos), x.cr = *reinterpret_cast<const uint2 *>(a.r8 + pos);
            x.sm = a.ms[b], x.sr = a.rs[b];
        }
    };
    auto update = [&](unsigned b, const Block &x) {
        if (x.left < 0) return;
        const size_t pos = (size_t)b * kBlock + lane * 8; // in the flat buffers
        float p[8], g[8];
        widen(x.p, kDtypeOf<P>, p);
        widen(x.g, g_dtype, g);
        auto store_p = [&]() {
            if (x.vec && x.left == 8) {
                store8v(x.p_at, p);
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++)
                    if (i < x.left) x.p_at[i] = narrow<P>(p[i]);
            }
        };
        // (each operation on the moments is rounded by itself: what is stored in 8 bits is then the same wherever it is
        //  computed.  The divisor of the weights' change is 0, or not below the smaller of eps, which is a normal number or 0,
        //  and 2^-74: its approximate reciprocal takes subnormal numbers for 0.)
        if constexpr (!kBits8) {
            float m[8], v[8];
            load8v(a.m + pos, m);
            load8v(a.v + pos, v);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                g[i] = __fmul_rn(g[i], unscale);
                m[i] = __fadd_rn(__fmul_rn(a.b1, m[i]), __fmul_rn(a.c1, g[i]));
                v[i] = __fadd_rn(__fmul_rn(a.b2, v[i]), __fmul_rn(a.c2, __fmul_rn(g[i], g[i])));
                p[i] = fmaf(-size * m[i], reciprocal(fmaf(__fsqrt_rn(v[i]), root, a.eps)), p[i] * keep);
            }
            store_p();
            store8v(a.m + pos, m);
            store8v(a.v + pos, v);
        } else {
            // two at a time; v and its root with the other sign, which saves the root's step two operations
            Pair m2[4], r2[4];
            from_e4m3(x.cm, x.sm, m2);
            from_e4m3(x.cr, x.sr, r2);
            uint32_t odd = 0; // how far beyond the range of minus_root
            float v[8];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const Pair gp = mul2(pair(g[2 * i], g[2 * i + 1]), both(unscale));
                m2[i] = add2(mul2(both(a.b1), m2[i]), mul2(both(a.c1), gp));
                r2[i] = add2(mul2(both(-a.b2), mul2(r2[i], r2[i])), mul2(both(-a.c2), mul2(gp, gp)));
                float v0, v1;
                apart(r2[i], v0, v1);
                v[2 * i] = -v0, v[2 * i + 1] = -v1;
                odd = max(odd, max(__float_as_uint(-v0) - 0x0d800000u, __float_as_uint(-v1) - 0x0d800000u)); // 2^-100
                r2[i] = minus_root(r2[i], -v0, -v1);
            }
            if (odd > 0x7e800000u - 0x0d800000u) { // 2^126; zeros and NaN come out above it too
#pragma unroll
                for (int i = 0; i < 4; i++) r2[i] = pair(-__fsqrt_rn(v[2 * i]), -__fsqrt_rn(v[2 * i + 1]));
            }
            float most_m = 0.f;
            uint32_t bits_r = 0; // (negative numbers, as bits: the largest magnitude is the largest, a NaN larger still)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                float d0, d1, m0, m1, r0, r1;
                apart(fma2(r2[i], both(-root), both(a.eps)), d0, d1);
                const Pair pn = fma2(mul2(m2[i], both(-size)), pair(reciprocal(d0), reciprocal(d1)),
                                     mul2(pair(p[2 * i], p[2 * i + 1]), both(keep)));
                apart(pn, p[2 * i], p[2 * i + 1]);
                apart(m2[i], m0, m1);
                apart(r2[i], r0, r1);
                most_m = max_nan(max_nan(most_m, fabsf(m0)), fabsf(m1));
                bits_r = max(bits_r, max(__float_as_uint(r0), __float_as_uint(r1)));
            }
            store_p();
            most_m = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(most_m)));
            const float most_r = __uint_as_float(__reduce_max_sync(0xffffffffu, bits_r) & 0x7fffffffu);
            // the block's four quotients, one to a lane
            const float most = lane & 1 ? most_r : most_m;
            float quotient = __fdiv_rn(lane & 2 ? most : 448.f, lane & 2 ? 448.f : most);
            if (most < 0x1p-100f) quotient = 0.f;
            const float per_m = __shfl_sync(0xffffffffu, quotient, 0), per_r = __shfl_sync(0xffffffffu, quotient, 1);
            if (lane == 2) a.ms[b] = quotient;
            if (lane == 3) a.rs[b] = quotient;
            const uint32_t u0 = (uint32_t)pos * 0xC13FA9A9u + (uint32_t)t * 0x9E3779B9u;
            uint32_t u[8];
            float y[8];
#pragma unroll
            for (int i = 0; i < 8; i++) u[i] = (u0 + i * 0xC13FA9A9u) >> 12;
#pragma unroll
            for (int i = 0; i < 4; i++) apart(mul2(m2[i], both(per_m)), y[2 * i], y[2 * i + 1]);
            auto sign = [&](int i) { return __float_as_uint(y[i]); };
            const uint32_t signs0 = pack4(sign(0), sign(1), sign(2), sign(3), 3) & 0x80808080u;
            const uint32_t signs1 = pack4(sign(4), sign(5), sign(6), sign(7), 3) & 0x80808080u;
            const uint2 wm = store_e4m3(y, !(__fmul_rn(most_m, per_m) <= 448.f), u, false);
            *reinterpret_cast<uint2 *>(a.m8 + pos) = make_uint2(wm.x | signs0, wm.y | signs1);
#pragma unroll
            for (int i = 0; i < 8; i++) u[i] = 0xfffffu - u[i];
#pragma unroll
            for (int i = 0; i < 4; i++) apart(mul2(r2[i], both(-per_r)), y[2 * i], y[2 * i + 1]);
            *reinterpret_cast<uint2 *>(a.r8 + pos) = store_e4m3(y, !(__fmul_rn(most_r, per_r) <= 448.f), u, true);
        }
    };
    unsigned b = a.first + blockIdx.x * kWarps + (threadIdx.x >> 5);
    Block now, next;
    if (kBits8 && b < a.last) load(b, now);
    for (; b < a.last; b += warps) {
        if (!kBits8) load(b, now);
        else if (b + warps < a.last) load(b + warps, next);
        const Block x = now;
        now = next;
        update(b, x);
    }
    // the last block of the launch to get here counts the step: all others have read the count
    if (a.advance) {
        __syncthreads();
        if (threadIdx.x == 0) {
            __threadfence();
            unsigned *done = reinterpret_cast<unsigned *>(a.step + 1);
            if (atomicAdd(done, 1u) == gridDim.x - 1) {
                *done = 0;
                a.step[0] = t;
            }
        }
    }
}

template <typename P, bool kBits8>
int launch_list(const AdamArgs &a, const rexsc_adamw_tensor *list, cudaStream_t st)
{
    auto fill = [&](AdamTensor *t) {
        const uintptr_t p_align = sizeof(P) == 4 ? 31 : 15, g_align = a.g_dtype == REXSC_F32 ? 31 : 15;
        for (int i = 0; i < a.tensors; i++)
            t[i] = AdamTensor{list[i].d_param, list[i].d_grad, list[i].numel, (unsigned)list[i].first_block,
                              !(reinterpret_cast<uintptr_t>(list[i].d_param) & p_align) &&
                                  !(reinterpret_cast<uintptr_t>(list[i].d_grad) & g_align)};
    };
    constexpr int kThreads = kThreadsOf<kBits8>, kWarps = kThreads / 32;
    const long long blocks = ((long long)a.last - a.first + kWarps - 1) / kWarps;
    const unsigned most = 148 * kCtasOf<kBits8>, grid = (unsigned)(blocks < most ? blocks : most);
    const bool same = a.g_dtype == kDtypeOf<P>;
    if (a.tensors <= kSmallList) {
        AdamLaunch<kSmallList> l;
        l.a = a;
        fill(l.t);
        return launch_under("adamw_kernel", same ? adamw_kernel<P, kBits8, true, kSmallList> : adamw_kernel<P, kBits8, false, kSmallList>,
                            grid, kThreads, 0, st, l);
    } else {
        AdamLaunch<kLargeList> l;
        l.a = a;
        fill(l.t);
        return launch_under("adamw_kernel", same ? adamw_kernel<P, kBits8, true, kLargeList> : adamw_kernel<P, kBits8, false, kLargeList>,
                            grid, kThreads, 0, st, l);
    }
}

} // namespace

} // namespace rexsc

using namespace rexsc;

extern "C" int rexsc_adamw_step(const rexsc_adamw_desc *desc, const rexsc_adamw_tensor *tensors, int32_t count, void *stream)
{
    if (!desc || count < 0 || (count > 0 && !tensors) || !desc->d_step) return REXSC_E_BAD_ARG;
    const rexsc_adamw_desc &d = *desc;
    const bool bits8 = d.state_bits == 8;
    if ((d.state_bits != 8 && d.state_bits != 32) || d.param_dtype < REXSC_F32 || d.param_dtype > REXSC_BF16 ||
        d.grad_dtype < REXSC_F32 || d.grad_dtype > REXSC_BF16 || !(d.beta1 >= 0. && d.beta1 < 1.) ||
        !(d.beta2 >= 0. && d.beta2 < 1.) || !(d.eps == 0. || (d.eps >= 0x1p-126 && d.eps < 0x1p126)) || !(d.weight_decay >= 0.) || (!d.d_lr && !(d.lr >= 0.)) ||
        !d.d_exp_avg || !d.d_exp_avg_sq || (bits8 && (!d.d_exp_avg_scale || !d.d_exp_avg_sq_scale)) ||
        ((reinterpret_cast<uintptr_t>(d.d_exp_avg) | reinterpret_cast<uintptr_t>(d.d_exp_avg_sq)) & 31) ||
        (reinterpret_cast<uintptr_t>(d.d_step) & 7))
        return REXSC_E_BAD_ARG;
    long long next = 0;
    for (int i = 0; i < count; i++) {
        const rexsc_adamw_tensor &t = tensors[i];
        if (!t.d_param || !t.d_grad || t.numel < 1 || t.first_block < next) return REXSC_E_BAD_ARG;
        next = t.first_block + (t.numel + kBlock - 1) / kBlock;
        if (next > 0x7fffffffll) return REXSC_E_TOO_LONG;
    }
    AdamArgs a = {};
    if (bits8) {
        a.m8 = static_cast<uint8_t *>(d.d_exp_avg), a.r8 = static_cast<uint8_t *>(d.d_exp_avg_sq);
        a.ms = d.d_exp_avg_scale, a.rs = d.d_exp_avg_sq_scale;
    } else {
        a.m = static_cast<float *>(d.d_exp_avg), a.v = static_cast<float *>(d.d_exp_avg_sq);
    }
    a.step = reinterpret_cast<long long *>(d.d_step);
    a.lr_ptr = d.d_lr, a.grad_scale = d.d_grad_scale, a.found_inf = d.d_found_inf;
    a.lr = (float)d.lr, a.b1 = (float)d.beta1, a.c1 = (float)(1. - d.beta1), a.b2 = (float)d.beta2, a.c2 = (float)(1. - d.beta2);
    a.eps = (float)d.eps, a.wd = (float)d.weight_decay;
    a.log_b1 = log(d.beta1), a.log_b2 = log(d.beta2);
    a.g_dtype = d.grad_dtype;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    for (int i = 0; i < count; i += kLargeList) {
        a.tensors = count - i < kLargeList ? count - i : kLargeList;
        const rexsc_adamw_tensor &last = tensors[i + a.tensors - 1];
        a.first = (unsigned)tensors[i].first_block;
        a.last = (unsigned)(last.first_block + (last.numel + kBlock - 1) / kBlock);
        a.advance = d.advance && i + a.tensors == count;
        int rc;
        if (d.param_dtype == REXSC_F32)
            rc = bits8 ? launch_list<float, true>(a, tensors + i, st) : launch_list<float, false>(a, tensors + i, st);
        else if (d.param_dtype == REXSC_F16)
            rc = bits8 ? launch_list<__half, true>(a, tensors + i, st) : launch_list<__half, false>(a, tensors + i, st);
        else
            rc = bits8 ? launch_list<__nv_bfloat16, true>(a, tensors + i, st) : launch_list<__nv_bfloat16, false>(a, tensors + i, st);
        if (rc != REXSC_OK) return rc;
    }
    return REXSC_OK;
}
