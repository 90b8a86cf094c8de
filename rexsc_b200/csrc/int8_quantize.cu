// Quantisation of matrices to 8 bits: rows (tokens of activations, output channels of weights), and rows and columns of a
// gradient in one go.
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

constexpr int kQThreads = 256;

// kWarps warps (1, 2, 4 or 8) have a row; four chunks of eight values per lane stay in registers between the pass for the
// largest magnitude and the one that quantises, columns beyond those are read twice.  Fewer values per lane would leave the
// row's own work (its division, addresses and the exchange between its warps) as long as the values'.
constexpr int kChunks = 4;
template <typename T, int kWarps>
__global__ void __launch_bounds__(kQThreads, sizeof(T) == 4 ? 3 : 4)
quantize_rows_kernel(const T *__restrict__ x, long long rows, long long cols, long long stride, int vec, long long rows_out,
                     long long tcols, int8_t *__restrict__ data, float *__restrict__ scale)
{
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    __shared__ uint32_t part[2][8];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int team = warp / kWarps, sub = threadIdx.x - team * 32 * kWarps; // row of the block, place among its threads
    constexpr int kRowsPerBlock = 8 / kWarps, kSpan = 32 * kWarps * 8;
    const long long padded = tcols * kI8Tile;
    int turn = 0;
    for (long long r = (long long)blockIdx.x * kRowsPerBlock + team; r < rows_out;
         r += (long long)gridDim.x * kRowsPerBlock, turn ^= 1) {
        int8_t *const to = data + i8_offset(r, sub * 8, tcols); // the row's 16 KiB tiles lie one behind the other
        auto place = [&](int j) { return reinterpret_cast<uint2 *>(to + (size_t)j * (kSpan / kI8Tile) * kI8TileBytes); };
        const int turns = (int)((padded - sub * 8 + kSpan - 1) / kSpan); // chunks of this thread
        if (r >= rows) { // (the same for all threads of a row)
            for (int j = 0; j < turns; j++) *place(j) = make_uint2(0u, 0u);
            continue;
        }
        const T *row = x + r * stride;
        Raw<T> v[kChunks];
        uint32_t most = 0;
#pragma unroll
        for (int j = 0; j < kChunks; j++) {
            const long long c = (long long)j * kSpan + sub * 8;
            if (c < cols) load_raw(row, c, cols, vec, v[j]);
            else clear_raw(v[j]);
        }
#pragma unroll
        for (int j = 0; j < kChunks; j++) most_of(v[j], most);
        for (long long c = (long long)kChunks * kSpan + sub * 8; c < cols; c += kSpan) {
            Raw<T> w;
            load_raw(row, c, cols, vec, w);
            most_of(w, most);
        }
        most = __reduce_max_sync(0xffffffffu, most_as_f32<T>(most));
        if (kWarps > 1) {
            if (lane == 0) part[turn][warp] = most;
            // (the row's own warps; the other half of `part` may still be read by a slower one)
            asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "r"(32 * kWarps) : "memory");
            most = __reduce_max_sync(0xffffffffu, part[turn][team * kWarps + lane % kWarps]);
        }
        const bool fine = most < 0x7f800000u;
        const float a = __uint_as_float(most);
        if (sub == 0) scale[r] = fine ? __fdiv_rn(a, 127.f) : __uint_as_float(0x7fc00000u);
        const bool zero = !fine || most == 0;
        const float inv = zero ? 0.f : inverse_of(a);
        auto store = [&](const Raw<T> &raw, int j) {
            float f[8];
            widen(raw, f);
            *place(j) = zero ? make_uint2(0u, 0u) : quant8<sizeof(T) == 2>(f, a, inv);
        };
#pragma unroll
        for (int j = 0; j < kChunks; j++)
            if (j < turns) store(v[j], j);
        for (int j = kChunks; j < turns; j++) {
            Raw<T> w;
            load_raw(row, (long long)j * kSpan + sub * 8, cols, vec, w);
            store(w, j);
        }
    }
}

template <typename T>
int quantize_rows(const T *x, long long rows, long long cols, long long stride, int8_t *data, float *scale, bool pad_rows,
                  cudaStream_t st)
{
    const long long tcols = i8_tiles(cols), rows_out = pad_rows ? i8_tiles(rows) * kI8Tile : rows;
    const int vec = ((reinterpret_cast<uintptr_t>(x) | (uintptr_t)(stride * (long long)sizeof(T))) & 15) == 0;
    auto launch = [&](auto kernel, int rows_per_block) {
        const long long blocks = (rows_out + rows_per_block - 1) / rows_per_block, most = 148 * (sizeof(T) == 4 ? 3 : 4);
        kernel<<<(unsigned)(blocks < most ? blocks : most), kQThreads, 0, st>>>(x, rows, cols, stride, vec, rows_out, tcols, data, scale);
    };
    // as many warps as leave every lane at most kChunks chunks, where eight can
    if (cols <= 32 * 8 * kChunks) launch(quantize_rows_kernel<T, 1>, 8);
    else if (cols <= 64 * 8 * kChunks) launch(quantize_rows_kernel<T, 2>, 4);
    else if (cols <= 128 * 8 * kChunks) launch(quantize_rows_kernel<T, 4>, 2);
    else launch(quantize_rows_kernel<T, 8>, 1);
    REXSC_LAUNCH_CHECK("quantize_rows_kernel");
    return REXSC_OK;
}

// plain row-major int8 <-> tiled
__global__ void __launch_bounds__(256)
pack_kernel(const int8_t *__restrict__ q, long long rows, long long cols, long long stride, long long tcols, long long chunks,
            int8_t *__restrict__ data)
{
    const long long per_row = tcols * (kI8Tile / 8);
    for (long long e = blockIdx.x * 256ll + threadIdx.x; e < chunks; e += gridDim.x * 256ll) {
        const long long r = e / per_row, c = (e - r * per_row) * 8;
        uint32_t w[2] = {0u, 0u};
        if (r < rows)
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (c + i < cols) w[i >> 2] |= (uint32_t)(uint8_t)q[r * stride + c + i] << (8 * (i & 3));
        *reinterpret_cast<uint2 *>(data + i8_offset(r, c, tcols)) = make_uint2(w[0], w[1]);
    }
}
__global__ void __launch_bounds__(256)
unpack_kernel(const int8_t *__restrict__ data, long long rows, long long cols, long long tcols, int8_t *__restrict__ q)
{
    const long long per_row = (cols + 7) / 8;
    for (long long e = blockIdx.x * 256ll + threadIdx.x; e < rows * per_row; e += gridDim.x * 256ll) {
        const long long r = e / per_row, c = (e - r * per_row) * 8;
        const uint2 w = *reinterpret_cast<const uint2 *>(data + i8_offset(r, c, tcols));
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (c + i < cols) q[r * cols + c + i] = (int8_t)((i < 4 ? w.x : w.y) >> (8 * (i & 3)));
    }
}

unsigned blocks_for(long long items)
{
    const long long b = (items + 255) / 256;
    return (unsigned)(b < 1 ? 1 : b < 148 * 16 ? b : 148 * 16);
}

// ---- gradients of an output: rows and columns -----------------------------------------------------------------
// g[m, n] = fl32(dy[m, n] col_scale[n]) is quantised by rows, h[m, n] = fl32(dy[m, n] row_scale[m]) by columns: each folds
// in the scales of the operand whose rows its contraction runs over.  Two passes over dy: the first leaves the largest
// magnitudes (an atomic maximum of bits: the order does not matter) and per block of rows the column sums for the bias, the
// second quantises.  Up to about 100 MB of dy the second pass finds it in L2.
constexpr int kGCols = 256;  // columns of a block: a warp has a row of it, eight columns a lane

// max that lets a NaN through
__device__ __forceinline__ float max_nan(float a, float b)
{
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

template <typename T>
__global__ void __launch_bounds__(256, 4)
grad_amax_kernel(const T *__restrict__ dy, long long m, long long n, long long stride, int vec, unsigned col_blocks, int rows,
                 const float *__restrict__ row_scale, const float *__restrict__ col_scale, uint32_t *__restrict__ row_most,
                 uint32_t *__restrict__ col_most, float *__restrict__ sums)
{
    __shared__ float cmax[8][kGCols], csum[8][kGCols];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const unsigned row_block = blockIdx.x / col_blocks, col_block = blockIdx.x - row_block * col_blocks;
    const long long c = (long long)col_block * kGCols + lane * 8, r0 = (long long)row_block * rows;
    const long long r1 = r0 + rows < m ? r0 + rows : m;
    float cs[8], cm[8], s[8];
#pragma unroll
    for (int i = 0; i < 8; i++) cs[i] = col_scale && c + i < n ? col_scale[c + i] : 0.f, cm[i] = 0.f, s[i] = 0.f;
    // (columns behind the last one: their values are 0 and so is their scale; what a NaN row scale makes of them is not kept)
    auto take = [&](const Raw<T> &raw, long long r) {
        float v[8];
        widen(raw, v);
        const float rs = row_scale ? row_scale[r] : 0.f;
        float rm = 0.f;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            rm = max_nan(rm, fabsf(__fmul_rn(v[i], cs[i])));
            cm[i] = max_nan(cm[i], fabsf(__fmul_rn(v[i], rs)));
            s[i] += v[i];
        }
        if (row_most) {
            const uint32_t all = __reduce_max_sync(0xffffffffu, __float_as_uint(rm));
            if (lane == 0) atomicMax(row_most + r, all);
        }
    };
    constexpr int kAhead = 4; // rows of a warp that are loaded together
    for (long long r = r0 + warp; r < r1; r += 8 * kAhead) {
        Raw<T> raw[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; j++)
            if (r + 8 * j < r1) load_raw(dy + (r + 8 * j) * stride, c, n, vec, raw[j]);
#pragma unroll
        for (int j = 0; j < kAhead; j++)
            if (r + 8 * j < r1) take(raw[j], r + 8 * j);
    }
#pragma unroll
    for (int i = 0; i < 8; i++) cmax[warp][i * 32 + lane] = cm[i], csum[warp][i * 32 + lane] = s[i];
    __syncthreads();
    const long long col = (long long)col_block * kGCols + threadIdx.x;
    const int at = (threadIdx.x & 7) * 32 + (threadIdx.x >> 3);
    if (col >= n) return;
    float most = 0.f, sum = 0.f;
#pragma unroll
    for (int w = 0; w < 8; w++) most = max_nan(most, cmax[w][at]), sum += csum[w][at];
    if (col_most) atomicMax(col_most + col, __float_as_uint(most));
    if (sums) sums[(long long)row_block * n + col] = sum;
}

// A block quantises a tile of 128 rows x 256 columns both ways; the blocks of the first tile row also finish the bias's
// gradient and the columns' scales, those of the first tile column the rows' scales.  A row (column) that is not finite gets
// the scale NaN; what its integers are does not matter then.
template <typename T, typename B>
__global__ void __launch_bounds__(256, 4)
grad_quantize_kernel(const T *__restrict__ dy, long long m, long long n, long long stride, int vec, unsigned col_blocks,
                     const float *__restrict__ row_scale, const float *__restrict__ col_scale,
                     const uint32_t *__restrict__ row_most, const uint32_t *__restrict__ col_most,
                     const float *__restrict__ sums, int sum_blocks, long long tcols, int8_t *__restrict__ qg,
                     float *__restrict__ sg, int8_t *__restrict__ qh, float *__restrict__ sh, B *__restrict__ db)
{
    __shared__ float row_a[kI8Tile], row_inv[kI8Tile], row_s[kI8Tile];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const unsigned row_block = blockIdx.x / col_blocks, col_block = blockIdx.x - row_block * col_blocks;
    const long long c = (long long)col_block * kGCols + lane * 8, r0 = (long long)row_block * kI8Tile;
    const float nan = __uint_as_float(0x7fc00000u);
    if (row_block == 0) {
        const long long col = (long long)col_block * kGCols + threadIdx.x;
        if (col < n) {
            if (db) {
                float s = 0.f;
                for (int b = 0; b < sum_blocks; b++) s += sums[(long long)b * n + col];
                db[col] = (B)s;
            }
            if (sh) {
                const uint32_t most = col_most[col];
                sh[col] = most < 0x7f800000u ? __fdiv_rn(__uint_as_float(most), 127.f) : nan;
            }
        }
    }
    if (threadIdx.x < kI8Tile) {
        const long long r = r0 + threadIdx.x;
        const uint32_t most = qg && r < m ? row_most[r] : 0u;
        const bool live = most != 0 && most < 0x7f800000u;
        row_a[threadIdx.x] = live ? __uint_as_float(most) : 0.f;
        row_inv[threadIdx.x] = live ? inverse_of(__uint_as_float(most)) : 0.f;
        row_s[threadIdx.x] = qh && r < m ? row_scale[r] : 0.f;
        if (sg && col_block == 0 && r < m) sg[r] = most < 0x7f800000u ? __fdiv_rn(__uint_as_float(most), 127.f) : nan;
    }
    __syncthreads();
    if (c >= tcols * kI8Tile) return;
    float cs[8], ci[8];
    bool tiny = false; // a column of this lane whose 127 / a overflows: every value takes the exact way
#pragma unroll
    for (int i = 0; i < 8; i++) {
        cs[i] = qg && c + i < n ? col_scale[c + i] : 0.f;
        const uint32_t most = qh && c + i < n ? col_most[c + i] : 0u;
        const bool live = most != 0 && most < 0x7f800000u;
        ci[i] = live ? inverse_of(__uint_as_float(most)) : 0.f;
        tiny |= live && ci[i] == 0.f;
    }
    // of row 0's chunk, without the swizzle (r0 and the block's first column begin a tile)
    const size_t base = ((size_t)row_block * tcols + (size_t)(c >> 7)) * kI8TileBytes + (size_t)(lane & 1) * 8;
    auto take = [&](const Raw<T> &raw, int row) { // row of the tile
        float v[8], x[8];
        widen(raw, v);
        const size_t at = base + row * 128 + (((lane >> 1 & 7) ^ (row & 7)) << 4);
        if (qg) {
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = __fmul_rn(v[i], cs[i]);
            const float a = row_a[row];
            *reinterpret_cast<uint2 *>(qg + at) = a > 0.f ? quant8<false>(x, a, row_inv[row]) : make_uint2(0u, 0u);
        }
        if (qh) {
            const float rs = row_s[row];
            uint32_t q[8];
            float far = 0.f;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                x[i] = __fmul_rn(v[i], rs);
                q[i] = quant_near(x[i], ci[i], far);
            }
            if (far > kFar || tiny) {
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    float off = 0.f;
                    quant_near(x[i], ci[i], off);
                    if (off > kFar || ci[i] == 0.f) {
                        const float a = c + i < n ? __uint_as_float(col_most[c + i]) : 0.f;
                        q[i] = a > 0.f ? (uint32_t)quant_exact(x[i], a) : 0u;
                    }
                }
            }
            *reinterpret_cast<uint2 *>(qh + at) = make_uint2(pack4(q[0], q[1], q[2], q[3]), pack4(q[4], q[5], q[6], q[7]));
        }
    };
    constexpr int kAhead = 2;
#pragma unroll 1
    for (int j = 0; j < kI8Tile / 8; j += kAhead) {
        Raw<T> raw[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; i++) {
            const long long r = r0 + (j + i) * 8 + warp;
            if (r < m) load_raw(dy + r * stride, c, n, vec, raw[i]);
            else clear_raw(raw[i]);
        }
#pragma unroll
        for (int i = 0; i < kAhead; i++) take(raw[i], (j + i) * 8 + warp);
    }
}

} // namespace

int launch_i8_quantize_rows(const void *d_x, int dtype, long long rows, long long cols, long long stride, int8_t *d_data,
                            float *d_scale, bool pad_rows, cudaStream_t st)
{
    switch (dtype) {
    case REXSC_F32: return quantize_rows(static_cast<const float *>(d_x), rows, cols, stride, d_data, d_scale, pad_rows, st);
    case REXSC_F16: return quantize_rows(static_cast<const __half *>(d_x), rows, cols, stride, d_data, d_scale, pad_rows, st);
    default: return quantize_rows(static_cast<const __nv_bfloat16 *>(d_x), rows, cols, stride, d_data, d_scale, pad_rows, st);
    }
}

namespace {

bool known_dtype(int d) { return d == REXSC_F32 || d == REXSC_F16 || d == REXSC_BF16; }

// Rows of a block of the first pass: long enough that its end (atomics, sums) is a small part, as long as every SM gets two
// blocks.  It follows from the sizes alone: the bias's sum has one order.
int grad_rows(long long m, long long n)
{
    const long long cols = (n + kGCols - 1) / kGCols;
    int rows = 256;
    while (rows > 32 && (m + rows - 1) / rows * cols < 2 * 148) rows /= 2;
    return rows;
}

// scratch of the backward pass
struct GradBuffers {
    uint32_t *row_most, *col_most;
    float *sg, *sh, *sums;
    int8_t *qg, *qh;
    size_t clear, total;
};

GradBuffers grad_buffers(uint8_t *ws, long long m, long long n, bool want_dx, bool want_dw, bool want_db)
{
    GradBuffers b;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at = align_up(at + bytes, 256);
        return ws + here;
    };
    b.row_most = reinterpret_cast<uint32_t *>(take(want_dx ? m * 4 : 0));
    b.col_most = reinterpret_cast<uint32_t *>(take(want_dw ? n * 4 : 0));
    b.clear = at;
    b.sg = reinterpret_cast<float *>(take(want_dx ? m * 4 : 0));
    b.sh = reinterpret_cast<float *>(take(want_dw ? n * 4 : 0));
    b.sums = reinterpret_cast<float *>(take(want_db ? ((m + grad_rows(m, n) - 1) / grad_rows(m, n)) * n * 4 : 0));
    b.qg = reinterpret_cast<int8_t *>(take(want_dx ? i8_bytes(m, n) : 0));
    b.qh = reinterpret_cast<int8_t *>(take(want_dw ? i8_bytes(m, n) : 0));
    b.total = at;
    return b;
}

template <typename T>
int grad_quantize(const T *dy, long long m, long long n, long long stride, const float *row_scale, const float *col_scale,
                  const GradBuffers &b, bool want_dx, bool want_dw, void *db, int db_dtype, cudaStream_t st)
{
    const int vec = ((reinterpret_cast<uintptr_t>(dy) | (uintptr_t)(stride * (long long)sizeof(T))) & 15) == 0;
    const int rows = grad_rows(m, n);
    const long long sum_blocks = (m + rows - 1) / rows, tcols = i8_tiles(n);
    const unsigned gx = (unsigned)((n + kGCols - 1) / kGCols);
    if (b.clear) REXSC_CUDA_CHECK(cudaMemsetAsync(b.row_most, 0, b.clear, st));
    grad_amax_kernel<T><<<(unsigned)(gx * sum_blocks), 256, 0, st>>>(
        dy, m, n, stride, vec, gx, rows, want_dw ? row_scale : nullptr, want_dx ? col_scale : nullptr,
        want_dx ? b.row_most : nullptr, want_dw ? b.col_most : nullptr, db ? b.sums : nullptr);
    REXSC_LAUNCH_CHECK("grad_amax_kernel");
    const unsigned grid = (unsigned)(gx * i8_tiles(m));
#define REXSC_I8_GRAD(B)                                                                                               \
    grad_quantize_kernel<T, B><<<grid, 256, 0, st>>>(                                                                 \
        dy, m, n, stride, vec, gx, row_scale, col_scale, b.row_most, b.col_most, b.sums, (int)sum_blocks, tcols,          \
        want_dx ? b.qg : nullptr, want_dx ? b.sg : nullptr, want_dw ? b.qh : nullptr, want_dw ? b.sh : nullptr,       \
        static_cast<B *>(db))
    if (db_dtype == REXSC_F16) REXSC_I8_GRAD(__half);
    else if (db_dtype == REXSC_BF16) REXSC_I8_GRAD(__nv_bfloat16);
    else REXSC_I8_GRAD(float);
#undef REXSC_I8_GRAD
    REXSC_LAUNCH_CHECK("grad_quantize_kernel");
    return REXSC_OK;
}

// operand whose contraction runs along the matrix's columns / rows
I8Operand along_columns(const int8_t *data, long long rows, long long cols)
{
    return I8Operand{data, i8_tiles(cols), 1, i8_tiles(rows), 0};
}
I8Operand along_rows(const int8_t *data, long long rows, long long cols)
{
    (void)rows;
    return I8Operand{data, 1, i8_tiles(cols), i8_tiles(cols), 1};
}

bool known_kernel(int k) { return k >= REXSC_INT8_AUTO && k <= REXSC_INT8_PAIR; }
bool good_extent(long long v) { return v >= 1 && v <= (1ll << 30); }

} // namespace

} // namespace rexsc

using namespace rexsc;

extern "C" size_t rexsc_int8_data_size(int64_t rows, int64_t cols)
{
    if (!good_extent(rows) || !good_extent(cols)) return 0;
    return i8_bytes(rows, cols);
}

extern "C" int rexsc_int8_quantize(const void *d_x, int32_t dtype, int64_t rows, int64_t cols, int64_t row_stride,
                                   int8_t *d_data, float *d_scale, void *stream)
{
    if (!d_x || !d_data || !d_scale || !known_dtype(dtype) || !good_extent(rows) || !good_extent(cols) || row_stride < 0 ||
        (reinterpret_cast<uintptr_t>(d_data) & 255))
        return REXSC_E_BAD_ARG;
    return launch_i8_quantize_rows(d_x, dtype, rows, cols, row_stride, d_data, d_scale, true, static_cast<cudaStream_t>(stream));
}

extern "C" int rexsc_int8_pack(const int8_t *d_q, int64_t rows, int64_t cols, int64_t row_stride, int8_t *d_data, void *stream)
{
    if (!d_q || !d_data || !good_extent(rows) || !good_extent(cols) || row_stride < 0 ||
        (reinterpret_cast<uintptr_t>(d_data) & 255))
        return REXSC_E_BAD_ARG;
    const long long tcols = i8_tiles(cols), chunks = i8_tiles(rows) * kI8Tile * tcols * (kI8Tile / 8);
    pack_kernel<<<blocks_for(chunks), 256, 0, static_cast<cudaStream_t>(stream)>>>(d_q, rows, cols, row_stride, tcols, chunks, d_data);
    REXSC_LAUNCH_CHECK("pack_kernel");
    return REXSC_OK;
}

extern "C" int rexsc_int8_unpack(const int8_t *d_data, int64_t rows, int64_t cols, int8_t *d_q, void *stream)
{
    if (!d_q || !d_data || !good_extent(rows) || !good_extent(cols) || (reinterpret_cast<uintptr_t>(d_data) & 255))
        return REXSC_E_BAD_ARG;
    unpack_kernel<<<blocks_for(rows * ((cols + 7) / 8)), 256, 0, static_cast<cudaStream_t>(stream)>>>(d_data, rows, cols, i8_tiles(cols), d_q);
    REXSC_LAUNCH_CHECK("unpack_kernel");
    return REXSC_OK;
}

extern "C" int rexsc_int8_matmul(const int8_t *d_a, const float *d_a_scale, const int8_t *d_b, const float *d_b_scale,
                                 const void *d_bias, int32_t bias_dtype, int64_t m, int64_t n, int64_t k, void *d_out,
                                 int32_t out_dtype, int32_t kernel, void *stream)
{
    if (!d_a || !d_a_scale || !d_b || !d_b_scale || !d_out || !good_extent(m) || !good_extent(n) || !good_extent(k) ||
        !known_dtype(out_dtype) || !known_kernel(kernel) || (d_bias && !known_dtype(bias_dtype)) ||
        ((reinterpret_cast<uintptr_t>(d_a) | reinterpret_cast<uintptr_t>(d_b)) & 255))
        return REXSC_E_BAD_ARG;
    if (k > kI8MaxDot) return REXSC_E_TOO_LONG;
    I8Product p{along_columns(d_a, m, k), along_columns(d_b, n, k), m, n, k, d_a_scale, d_b_scale, d_bias, bias_dtype,
                d_out, out_dtype, n};
    return launch_i8_product(p, kernel, false, static_cast<cudaStream_t>(stream));
}

extern "C" size_t rexsc_int8_linear_workspace_size(int64_t m, int64_t k)
{
    if (!good_extent(m) || !good_extent(k) || k > kI8MaxDot) return 0;
    return align_up((size_t)m * 4, 256) + i8_bytes(m, k);
}

extern "C" int rexsc_int8_linear_fwd(const void *d_x, int32_t dtype, int64_t m, int64_t k, int64_t row_stride,
                                     const int8_t *d_w, const float *d_w_scale, int64_t n, const void *d_bias,
                                     int32_t bias_dtype, void *d_out, int32_t out_dtype, int32_t kernel,
                                     void *d_workspace, size_t workspace_bytes, void *stream)
{
    if (!d_x || !d_w || !d_w_scale || !d_out || !good_extent(m) || !good_extent(n) || !good_extent(k) || row_stride < 0 ||
        !known_dtype(dtype) || !known_dtype(out_dtype) || !known_kernel(kernel) || (d_bias && !known_dtype(bias_dtype)) ||
        (reinterpret_cast<uintptr_t>(d_w) & 255))
        return REXSC_E_BAD_ARG;
    if (k > kI8MaxDot) return REXSC_E_TOO_LONG;
    if (!d_workspace || workspace_bytes < rexsc_int8_linear_workspace_size(m, k) || (reinterpret_cast<uintptr_t>(d_workspace) & 255))
        return REXSC_E_WORKSPACE;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    float *sx = static_cast<float *>(d_workspace);
    int8_t *qx = reinterpret_cast<int8_t *>(static_cast<uint8_t *>(d_workspace) + align_up((size_t)m * 4, 256));
    // (rows that pad the last tile stay as they are: they only reach outputs that are not stored)
    int rc = launch_i8_quantize_rows(d_x, dtype, m, k, row_stride, qx, sx, false, st);
    if (rc != REXSC_OK) return rc;
    I8Product p{along_columns(qx, m, k), along_columns(d_w, n, k), m, n, k, sx, d_w_scale, d_bias, bias_dtype, d_out, out_dtype, n};
    return launch_i8_product(p, kernel, true, st);
}

extern "C" size_t rexsc_int8_linear_bwd_workspace_size(int64_t m, int64_t n, int32_t want_dx, int32_t want_dw, int32_t want_db)
{
    if (!good_extent(m) || !good_extent(n)) return 0;
    return grad_buffers(nullptr, m, n, want_dx != 0, want_dw != 0, want_db != 0).total + 256;
}

extern "C" int rexsc_int8_linear_bwd(const void *d_dy, int32_t dtype, int64_t m, int64_t n, int64_t k, int64_t row_stride,
                                     const int8_t *d_x, const float *d_x_scale, const int8_t *d_w, const float *d_w_scale,
                                     void *d_dx, int32_t dx_dtype, void *d_dw, int32_t dw_dtype, void *d_db, int32_t db_dtype,
                                     int32_t kernel, void *d_workspace, size_t workspace_bytes, void *stream)
{
    if (!d_dy || !good_extent(m) || !good_extent(n) || !good_extent(k) || row_stride < 0 || !known_dtype(dtype) ||
        !known_kernel(kernel) || (!d_dx && !d_dw && !d_db) || (d_dx && (!d_w || !d_w_scale || !known_dtype(dx_dtype))) ||
        (d_dw && (!d_x || !d_x_scale || !known_dtype(dw_dtype))) || (d_db && !known_dtype(db_dtype)) ||
        ((reinterpret_cast<uintptr_t>(d_x) | reinterpret_cast<uintptr_t>(d_w)) & 255))
        return REXSC_E_BAD_ARG;
    if ((d_dx && n > kI8MaxDot) || (d_dw && m > kI8MaxDot)) return REXSC_E_TOO_LONG;
    if (!d_workspace || workspace_bytes < rexsc_int8_linear_bwd_workspace_size(m, n, d_dx != nullptr, d_dw != nullptr, d_db != nullptr) ||
        (reinterpret_cast<uintptr_t>(d_workspace) & 255))
        return REXSC_E_WORKSPACE;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const GradBuffers b = grad_buffers(static_cast<uint8_t *>(d_workspace), m, n, d_dx != nullptr, d_dw != nullptr, d_db != nullptr);
    int rc;
    if (dtype == REXSC_F32)
        rc = grad_quantize(static_cast<const float *>(d_dy), m, n, row_stride, d_x_scale, d_w_scale, b, d_dx != nullptr, d_dw != nullptr, d_db, db_dtype, st);
    else if (dtype == REXSC_F16)
        rc = grad_quantize(static_cast<const __half *>(d_dy), m, n, row_stride, d_x_scale, d_w_scale, b, d_dx != nullptr, d_dw != nullptr, d_db, db_dtype, st);
    else
        rc = grad_quantize(static_cast<const __nv_bfloat16 *>(d_dy), m, n, row_stride, d_x_scale, d_w_scale, b, d_dx != nullptr, d_dw != nullptr, d_db, db_dtype, st);
    if (rc != REXSC_OK) return rc;
    if (d_dx) {
        I8Product p{along_columns(b.qg, m, n), along_rows(d_w, n, k), m, k, n, b.sg, nullptr, nullptr, 0, d_dx, dx_dtype, k};
        rc = launch_i8_product(p, kernel, false, st);
        if (rc != REXSC_OK) return rc;
    }
    if (d_dw) {
        I8Product p{along_rows(b.qh, m, n), along_rows(d_x, m, k), n, k, m, b.sh, nullptr, nullptr, 0, d_dw, dw_dtype, k};
        rc = launch_i8_product(p, kernel, false, st);
    }
    return rc;
}
