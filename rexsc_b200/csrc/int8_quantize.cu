// Quantisation of matrices to 8 bits: rows (tokens of activations, output channels of weights), and rows and columns of a
// gradient in one go.
//
// A row with the largest magnitude a is held as  s = a / 127 (fp32)  and  q = rne(127 x / a).  q is that of the exact
// quotient: x * (127 / a) in fp32 is off by less than 2^-15 at 127, so a value further than 2^-14 from the border between
// two whole numbers is decided by it, and the few others (one in ten thousand) are divided in fp64, where products are
// exact and a quotient that is not on the border cannot be rounded onto it (it is at least 2^-40 away from it).
// A row of zeros has s = 0 and q = 0.  A row that holds an infinity or a NaN has s = NaN and q = 0: its products are NaN and
// nobody else's are.
#include "int8.cuh"

namespace rexsc {

namespace {

constexpr float kMagic = 12582912.f; // 1.5 * 2^23: adding it rounds |t| < 2^22 to the nearest whole number, ties to even

__device__ __noinline__ int quant_exact(float x, float a)
{
    return __double2int_rn((double)x * 127.0 / (double)a);
}

// four whole numbers' low bytes in one word
__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d)
{
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// q of eight values of a row whose largest magnitude is a > 0 (finite); inv = 127 / a, or 0 where that overflows
__device__ __forceinline__ uint2 quant8(const float (&x)[8], float a, float inv)
{
    uint32_t q[8];
    float far = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float t = __fmul_rn(x[i], inv), r = __fadd_rn(t, kMagic);
        q[i] = __float_as_uint(r);
        far = fmaxf(far, fabsf(__fsub_rn(t, __fsub_rn(r, kMagic))));
    }
    if (far > 0.5f - 6.104e-5f || inv == 0.f) {
#pragma unroll
        for (int i = 0; i < 8; i++) q[i] = (uint32_t)quant_exact(x[i], a);
    }
    return make_uint2(pack4(q[0], q[1], q[2], q[3]), pack4(q[4], q[5], q[6], q[7]));
}

__device__ __forceinline__ float inverse_of(float a) { return a < 7.9e-31f ? 0.f : __fdiv_rn(127.f, a); }

__device__ __forceinline__ void load8(const float *p, float (&v)[8])
{
    const float4 a = *reinterpret_cast<const float4 *>(p), b = *reinterpret_cast<const float4 *>(p + 4);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
__device__ __forceinline__ void load8(const __half *p, float (&v)[8])
{
    const uint4 u = *reinterpret_cast<const uint4 *>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
        v[2 * i] = f.x, v[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ void load8(const __nv_bfloat16 *p, float (&v)[8])
{
    const uint4 u = *reinterpret_cast<const uint4 *>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; i++) v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
}
// eight values from column c on, zeros behind the last column; vec: rows begin on 16 bytes
template <typename T>
__device__ __forceinline__ void load8_edge(const T *row, long long c, long long cols, bool vec, float (&v)[8])
{
    if (vec && c + 8 <= cols) {
        load8(row + c, v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = c + i < cols ? load_as_float(row + c + i, 0) : 0.f;
    }
}

// largest magnitude as the bits of an fp32: ordered like the values, infinities above them, NaNs above those
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

constexpr int kQThreads = 256;

// kWarps warps (1 or 8) per row, kChunks chunks of eight values per lane held in registers between the pass for the largest
// magnitude and the one that quantises; columns beyond those are read twice.
template <typename T, int kWarps, int kChunks>
__global__ void __launch_bounds__(kQThreads)
quantize_rows_kernel(const T *__restrict__ x, long long rows, long long cols, long long stride, int vec, long long rows_out,
                     long long tcols, int8_t *__restrict__ data, float *__restrict__ scale)
{
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    __shared__ uint32_t part[2][8];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int sub = kWarps == 1 ? lane : (int)threadIdx.x; // place of the thread among those of its row
    constexpr int kRowsPerBlock = 8 / kWarps, kSpan = 32 * kWarps * 8;
    const long long padded = tcols * kI8Tile;
    int turn = 0;
    for (long long r = (long long)blockIdx.x * kRowsPerBlock + (kWarps == 1 ? warp : 0); r < rows_out;
         r += (long long)gridDim.x * kRowsPerBlock, turn ^= 1) {
        if (r >= rows) { // (the same for all threads of a row)
            for (long long c = sub * 8; c < padded; c += kSpan)
                *reinterpret_cast<uint2 *>(data + i8_offset(r, c, tcols)) = make_uint2(0u, 0u);
            continue;
        }
        const T *row = x + r * stride;
        float v[kChunks][8];
        uint32_t most = 0;
#pragma unroll
        for (int j = 0; j < kChunks; j++) {
            const long long c = (long long)j * kSpan + sub * 8;
            if (c < cols) {
                load8_edge(row, c, cols, vec, v[j]);
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++) v[j][i] = 0.f;
            }
        }
#pragma unroll
        for (int j = 0; j < kChunks; j++)
#pragma unroll
            for (int i = 0; i < 8; i++) most = max(most, abs_bits(v[j][i]));
        for (long long c = (long long)kChunks * kSpan + sub * 8; c < cols; c += kSpan) {
            float w[8];
            load8_edge(row, c, cols, vec, w);
#pragma unroll
            for (int i = 0; i < 8; i++) most = max(most, abs_bits(w[i]));
        }
        most = __reduce_max_sync(0xffffffffu, most);
        if (kWarps > 1) {
            if (lane == 0) part[turn][warp] = most;
            __syncthreads(); // (the other half of `part` may still be read by a slower warp)
#pragma unroll
            for (int i = 0; i < 8; i++) most = max(most, part[turn][i]);
        }
        const bool fine = most < 0x7f800000u;
        const float a = __uint_as_float(most);
        if (sub == 0) scale[r] = fine ? __fdiv_rn(a, 127.f) : __uint_as_float(0x7fc00000u);
        const bool zero = !fine || most == 0;
        const float inv = zero ? 0.f : inverse_of(a);
#pragma unroll
        for (int j = 0; j < kChunks; j++) {
            const long long c = (long long)j * kSpan + sub * 8;
            if (c < padded)
                *reinterpret_cast<uint2 *>(data + i8_offset(r, c, tcols)) = zero ? make_uint2(0u, 0u) : quant8(v[j], a, inv);
        }
        for (long long c = (long long)kChunks * kSpan + sub * 8; c < padded; c += kSpan) {
            float w[8];
            load8_edge(row, c, cols, vec, w);
            *reinterpret_cast<uint2 *>(data + i8_offset(r, c, tcols)) = zero ? make_uint2(0u, 0u) : quant8(w, a, inv);
        }
    }
}

template <typename T>
int quantize_rows(const T *x, long long rows, long long cols, long long stride, int8_t *data, float *scale, bool pad_rows,
                  cudaStream_t st)
{
    const long long tcols = i8_tiles(cols), rows_out = pad_rows ? i8_tiles(rows) * kI8Tile : rows;
    const int vec = ((reinterpret_cast<uintptr_t>(x) | (uintptr_t)(stride * (long long)sizeof(T))) & 15) == 0;
    const long long most = 148 * 8;
    if (cols <= 1024) {
        const long long blocks = (rows_out + 7) / 8;
        quantize_rows_kernel<T, 1, 4><<<(unsigned)(blocks < most ? blocks : most), kQThreads, 0, st>>>(
            x, rows, cols, stride, vec, rows_out, tcols, data, scale);
    } else {
        const unsigned blocks = (unsigned)(rows_out < most ? rows_out : most);
        if (cols <= 4096)
            quantize_rows_kernel<T, 8, 2><<<blocks, kQThreads, 0, st>>>(x, rows, cols, stride, vec, rows_out, tcols, data, scale);
        else
            quantize_rows_kernel<T, 8, 4><<<blocks, kQThreads, 0, st>>>(x, rows, cols, stride, vec, rows_out, tcols, data, scale);
    }
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
constexpr int kGRows = 64;   // rows of a block of the first pass
constexpr int kGCols = 256;  // columns of a block

template <typename T>
__global__ void __launch_bounds__(256)
grad_amax_kernel(const T *__restrict__ dy, long long m, long long n, long long stride, int vec, unsigned col_blocks,
                 const float *__restrict__ row_scale, const float *__restrict__ col_scale, uint32_t *__restrict__ row_most,
                 uint32_t *__restrict__ col_most, float *__restrict__ sums)
{
    __shared__ uint32_t cmax[8][kGCols];
    __shared__ float csum[8][kGCols];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const unsigned row_block = blockIdx.x / col_blocks, col_block = blockIdx.x - row_block * col_blocks;
    const long long c = (long long)col_block * kGCols + lane * 8, r0 = (long long)row_block * kGRows;
    float cs[8];
    uint32_t cm[8] = {};
    float s[8] = {};
#pragma unroll
    for (int i = 0; i < 8; i++) cs[i] = col_scale && c + i < n ? col_scale[c + i] : 0.f;
#pragma unroll 4
    for (int j = 0; j < kGRows / 8; j++) {
        const long long r = r0 + j * 8 + warp;
        if (r >= m) break;
        float v[8];
        load8_edge(dy + r * stride, c, n, vec, v);
        const float rs = row_scale ? row_scale[r] : 0.f;
        uint32_t rm = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            // (0 behind the last column whatever the scales are: its value is 0 and its column scale too; a NaN row scale
            //  there would only touch columns that are not kept)
            rm = max(rm, abs_bits(__fmul_rn(v[i], cs[i])));
            cm[i] = max(cm[i], abs_bits(__fmul_rn(v[i], rs)));
            s[i] += v[i];
        }
        if (row_most) {
            rm = __reduce_max_sync(0xffffffffu, rm);
            if (lane == 0) atomicMax(row_most + r, rm);
        }
    }
#pragma unroll
    for (int i = 0; i < 8; i++) cmax[warp][lane * 8 + i] = cm[i], csum[warp][lane * 8 + i] = s[i];
    __syncthreads();
    const long long col = (long long)col_block * kGCols + threadIdx.x;
    if (col >= n) return;
    uint32_t most = 0;
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < 8; w++) most = max(most, cmax[w][threadIdx.x]), sum += csum[w][threadIdx.x];
    if (col_most) atomicMax(col_most + col, most);
    if (sums) sums[(long long)row_block * n + col] = sum;
}

// A block quantises a tile of 128 rows x 256 columns both ways; the blocks of the first tile row also finish the bias's
// gradient and the columns' scales, those of the first tile column the rows' scales.
template <typename T, typename B>
__global__ void __launch_bounds__(256)
grad_quantize_kernel(const T *__restrict__ dy, long long m, long long n, long long stride, int vec, unsigned col_blocks,
                     const float *__restrict__ row_scale, const float *__restrict__ col_scale,
                     const uint32_t *__restrict__ row_most, const uint32_t *__restrict__ col_most,
                     const float *__restrict__ sums, int sum_blocks, long long tcols, int8_t *__restrict__ qg,
                     float *__restrict__ sg, int8_t *__restrict__ qh, float *__restrict__ sh, B *__restrict__ db)
{
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
    if (sg && col_block == 0 && threadIdx.x < kI8Tile && r0 + threadIdx.x < m) {
        const uint32_t most = row_most[r0 + threadIdx.x];
        sg[r0 + threadIdx.x] = most < 0x7f800000u ? __fdiv_rn(__uint_as_float(most), 127.f) : nan;
    }
    if (c >= tcols * kI8Tile) return;
    float cs[8], ca[8], ci[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        cs[i] = qg && c + i < n ? col_scale[c + i] : 0.f;
        const uint32_t most = qh && c + i < n ? col_most[c + i] : 0u;
        const bool live = most != 0 && most < 0x7f800000u;
        ca[i] = live ? __uint_as_float(most) : 0.f;
        ci[i] = live ? inverse_of(ca[i]) : 0.f;
    }
#pragma unroll 4
    for (int j = 0; j < kI8Tile / 8; j++) {
        const long long r = r0 + j * 8 + warp;
        float v[8];
        if (r < m) {
            load8_edge(dy + r * stride, c, n, vec, v);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = 0.f;
        }
        const size_t at = i8_offset(r, c, tcols);
        if (qg) {
            const uint32_t most = r < m ? row_most[r] : 0u;
            uint2 q = make_uint2(0u, 0u);
            if (most != 0 && most < 0x7f800000u) {
                float g[8];
#pragma unroll
                for (int i = 0; i < 8; i++) g[i] = __fmul_rn(v[i], cs[i]);
                q = quant8(g, __uint_as_float(most), inverse_of(__uint_as_float(most)));
            }
            *reinterpret_cast<uint2 *>(qg + at) = q;
        }
        if (qh) {
            const float rs = r < m ? row_scale[r] : 0.f;
            uint32_t q[8];
            float h[8], far = 0.f;
            bool tiny = false;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                h[i] = ca[i] != 0.f ? __fmul_rn(v[i], rs) : 0.f;
                const float t = __fmul_rn(h[i], ci[i]), w = __fadd_rn(t, kMagic);
                q[i] = __float_as_uint(w);
                far = fmaxf(far, fabsf(__fsub_rn(t, __fsub_rn(w, kMagic))));
                tiny |= ci[i] == 0.f && ca[i] != 0.f;
            }
            if (far > 0.5f - 6.104e-5f || tiny) {
#pragma unroll
                for (int i = 0; i < 8; i++) q[i] = ca[i] != 0.f ? (uint32_t)quant_exact(h[i], ca[i]) : 0u;
            }
            *reinterpret_cast<uint2 *>(qh + at) = make_uint2(pack4(q[0], q[1], q[2], q[3]), pack4(q[4], q[5], q[6], q[7]));
        }
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
    b.sums = reinterpret_cast<float *>(take(want_db ? ((m + kGRows - 1) / kGRows) * n * 4 : 0));
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
    const long long sum_blocks = (m + kGRows - 1) / kGRows, tcols = i8_tiles(n);
    const unsigned gx = (unsigned)((n + kGCols - 1) / kGCols);
    if (b.clear) REXSC_CUDA_CHECK(cudaMemsetAsync(b.row_most, 0, b.clear, st));
    grad_amax_kernel<T><<<(unsigned)(gx * sum_blocks), 256, 0, st>>>(
        dy, m, n, stride, vec, gx, want_dw ? row_scale : nullptr, want_dx ? col_scale : nullptr,
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
