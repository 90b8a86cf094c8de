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
// What bounds it: memory.  Per element 28 bytes (fp32 weights and gradients, 32-bit moments), 16 with 8-bit moments.
#include <math.h>

#include "common.cuh"

namespace rexsc {

namespace {

constexpr int kBlock = 256;      // elements of a block (of a scale)
constexpr int kThreads = 256;
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
__device__ __forceinline__ void load8v(const __half *p, float (&v)[8])
{
    const uint4 u = *reinterpret_cast<const uint4 *>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
        v[2 * i] = f.x, v[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ void load8v(const __nv_bfloat16 *p, float (&v)[8])
{
    const uint4 u = *reinterpret_cast<const uint4 *>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; i++) v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
}
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

// elements [e, e + 8) of a tensor of n; zeros behind its end
template <typename T>
__device__ __forceinline__ void load_elems(const T *p, long long e, long long n, int vec, float (&v)[8])
{
    if (vec && e + 8 <= n) {
        load8v(p + e, v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = e + i < n ? load_as_float(p + e + i, 0) : 0.f;
    }
}

// e4m3 <-> fp32 by the bits: 4 exponent bits (bias 7), 3 of mantissa, steps of 2^-9 below 2^-6
__device__ __forceinline__ float from_e4m3(uint32_t code) // (sign in bit 7; the two NaN codes come out as NaN)
{
    const uint32_t mag = code & 0x7f;
    const float v = mag >= 8 ? __uint_as_float((mag << 20) + ((127 - 7) << 23)) : (float)mag * 0x1p-9f;
    const float w = mag == 0x7f ? __uint_as_float(0x7fc00000u) : v;
    return code & 0x80 ? -w : w;
}
// y in [0, 448 (1 + 2^-22)], u < 2^20
__device__ __forceinline__ uint32_t to_e4m3(float y, uint32_t u)
{
    const uint32_t normal = ((__float_as_uint(y) + u) >> 20) - ((127 - 7) << 3);
    const uint32_t small = (uint32_t)__float2int_rd(__fadd_rn(__fmul_rn(y, 512.f), __fmul_rn((float)u, 0x1p-20f)));
    return min(y < 0x1p-6f ? small : normal, 126u);
}

template <typename P, bool kBits8, int kList>
__global__ void __launch_bounds__(kThreads)
adamw_kernel(const __grid_constant__ AdamLaunch<kList> l)
{
    const AdamArgs &a = l.a;
    if (a.found_inf && *a.found_inf != 0.f) return;
    const int lane = threadIdx.x & 31;
    const long long t = a.step[0] + 1;
    const float lr = a.lr_ptr ? *a.lr_ptr : a.lr;
    const float unscale = a.grad_scale ? __fdiv_rn(1.f, *a.grad_scale) : 1.f;
    const float keep = 1.f - lr * a.wd;
    const float size = lr / -expm1f((float)((double)t * a.log_b1));
    const float root = rsqrtf(-expm1f((float)((double)t * a.log_b2)));
    const unsigned warps = gridDim.x * (kThreads / 32);
    int at = 0;
    for (unsigned b = a.first + blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); b < a.last; b += warps) {
        // the last tensor that begins at b or before; blocks only rise, so the search goes on from where it was
        if (at + 1 < a.tensors && l.t[at + 1].first <= b) {
            int lo = at + 1, hi = a.tensors;
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (l.t[mid].first <= b) lo = mid; else hi = mid;
            }
            at = lo;
        }
        const AdamTensor &x = l.t[at];
        if ((long long)(b - x.first) * kBlock >= x.n) continue; // a block of no tensor of the list
        const long long e = (long long)(b - x.first) * kBlock + lane * 8; // in the tensor
        const size_t pos = (size_t)b * kBlock + lane * 8;                 // in the flat buffers
        P *px = static_cast<P *>(x.p);
        float p[8], g[8], m[8], v[8];
        load_elems(px, e, x.n, x.vec, p);
        if (a.g_dtype == REXSC_F32) load_elems(static_cast<const float *>(x.g), e, x.n, x.vec, g);
        else if (a.g_dtype == REXSC_F16) load_elems(static_cast<const __half *>(x.g), e, x.n, x.vec, g);
        else load_elems(static_cast<const __nv_bfloat16 *>(x.g), e, x.n, x.vec, g);
        if constexpr (kBits8) {
            const uint2 cm = *reinterpret_cast<const uint2 *>(a.m8 + pos), cr = *reinterpret_cast<const uint2 *>(a.r8 + pos);
            const float sm = a.ms[b], sr = a.rs[b];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                m[i] = __fmul_rn(from_e4m3((i < 4 ? cm.x : cm.y) >> (8 * (i & 3)) & 0xff), sm);
                const float r = __fmul_rn(from_e4m3((i < 4 ? cr.x : cr.y) >> (8 * (i & 3)) & 0xff), sr);
                v[i] = __fmul_rn(r, r);
            }
        } else {
            load8v(a.m + pos, m);
            load8v(a.v + pos, v);
        }
        float r[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            // (each operation rounded by itself: what is stored in 8 bits is then the same wherever it is computed)
            g[i] = __fmul_rn(g[i], unscale);
            m[i] = __fadd_rn(__fmul_rn(a.b1, m[i]), __fmul_rn(a.c1, g[i]));
            v[i] = __fadd_rn(__fmul_rn(a.b2, v[i]), __fmul_rn(a.c2, __fmul_rn(g[i], g[i])));
            r[i] = __fsqrt_rn(v[i]);
            p[i] = p[i] * keep - __fdividef(size * m[i], fmaf(r[i], root, a.eps));
        }
        if (x.vec && e + 8 <= x.n) {
            store8v(px + e, p);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (e + i < x.n) px[e + i] = narrow<P>(p[i]);
        }
        if constexpr (kBits8) {
            uint32_t am = 0, ar = 0; // bits: a NaN is larger than everything
#pragma unroll
            for (int i = 0; i < 8; i++) am = max(am, __float_as_uint(m[i]) & 0x7fffffffu), ar = max(ar, __float_as_uint(r[i]) & 0x7fffffffu);
            const float most_m = __uint_as_float(__reduce_max_sync(0xffffffffu, am)), most_r = __uint_as_float(__reduce_max_sync(0xffffffffu, ar));
            const float per_m = most_m < 0x1p-100f ? 0.f : __fdiv_rn(448.f, most_m), per_r = most_r < 0x1p-100f ? 0.f : __fdiv_rn(448.f, most_r);
            if (lane == 0) {
                a.ms[b] = most_m < 0x1p-100f ? 0.f : __fdiv_rn(most_m, 448.f);
                a.rs[b] = most_r < 0x1p-100f ? 0.f : __fdiv_rn(most_r, 448.f);
            }
            uint32_t wm[2] = {0, 0}, wr[2] = {0, 0};
            const uint32_t u0 = (uint32_t)pos * 0xC13FA9A9u + (uint32_t)t * 0x9E3779B9u;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const uint32_t u = u0 + i * 0xC13FA9A9u;
                const uint32_t code_m = to_e4m3(__fmul_rn(fabsf(m[i]), per_m), u >> 12) | (__float_as_uint(m[i]) >> 31) << 7;
                const float y = __fmul_rn(r[i], per_r);
                const uint32_t code_r = max(to_e4m3(y, ~u >> 12), y > 0.f ? 1u : 0u);
                wm[i >> 2] |= code_m << (8 * (i & 3));
                wr[i >> 2] |= code_r << (8 * (i & 3));
            }
            *reinterpret_cast<uint2 *>(a.m8 + pos) = make_uint2(wm[0], wm[1]);
            *reinterpret_cast<uint2 *>(a.r8 + pos) = make_uint2(wr[0], wr[1]);
        } else {
            store8v(a.m + pos, m);
            store8v(a.v + pos, v);
        }
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
    const long long blocks = ((long long)a.last - a.first + kThreads / 32 - 1) / (kThreads / 32);
    const unsigned grid = (unsigned)(blocks < 148 * 8 ? blocks : 148 * 8);
    if (a.tensors <= kSmallList) {
        AdamLaunch<kSmallList> l;
        l.a = a;
        fill(l.t);
        adamw_kernel<P, kBits8, kSmallList><<<grid, kThreads, 0, st>>>(l);
    } else {
        AdamLaunch<kLargeList> l;
        l.a = a;
        fill(l.t);
        adamw_kernel<P, kBits8, kLargeList><<<grid, kThreads, 0, st>>>(l);
    }
    REXSC_LAUNCH_CHECK("adamw_kernel");
    return REXSC_OK;
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
        !(d.beta2 >= 0. && d.beta2 < 1.) || !(d.eps >= 0.) || !(d.weight_decay >= 0.) || (!d.d_lr && !(d.lr >= 0.)) ||
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
