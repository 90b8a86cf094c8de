// Quantisation of matrices to 8 bits (int8_quant.cuh has the rule): rows (tokens of activations, output channels of weights),
// and rows and columns of a gradient in one go.
#include "int8_quant.cuh"

namespace rexsc {

namespace {

constexpr int kQThreads = 256;

// kWarps warps (1, 2, 4 or 8) have a row; four chunks of eight values per lane stay in registers between the pass for the
// largest magnitude and the one that quantises, columns beyond those are read twice.  Fewer values per lane would leave the
// row's own work (its division, addresses and the exchange between its warps) as long as the values'.  Bound by memory latency
// at the 32 warps an SM that 64 registers leave: bf16 8192 x 8192 in 40 us (5.0 TB/s), 8192 x 4096 in 22 us; the arithmetic on
// pairs of values saves a tenth of the instructions and no time.
constexpr int kChunks = 4;
template <typename T, int kWarps>
__global__ void __launch_bounds__(kQThreads, sizeof(T) == 4 ? 3 : 4)
quantize_rows_kernel(const T *__restrict__ x, long long rows, long long cols, long long stride, int vec, long long rows_out,
                     long long tcols, int8_t *__restrict__ data, float *__restrict__ scale)
{
    wait_previous_launch();
    allow_next_launch();
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
        return launch_under("quantize_rows_kernel", kernel, (unsigned)(blocks < most ? blocks : most), kQThreads, 0, st, x, rows,
                            cols, stride, vec, rows_out, tcols, data, scale);
    };
    // as many warps as leave every lane at most kChunks chunks, where eight can
    if (cols <= 32 * 8 * kChunks) return launch(quantize_rows_kernel<T, 1>, 8);
    if (cols <= 64 * 8 * kChunks) return launch(quantize_rows_kernel<T, 2>, 4);
    if (cols <= 128 * 8 * kChunks) return launch(quantize_rows_kernel<T, 4>, 2);
    return launch(quantize_rows_kernel<T, 8>, 1);
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
// in the scales of the operand whose rows its contraction runs over.  Two passes over dy: in the first every block leaves the
// largest magnitudes of its rows and columns and their sums, for the bias; the second joins those (no atomics and nothing to
// clear) and quantises.  The bias's sum is in fp32 along the rows of a warp (32 of them up to 32768 tokens, 512 at the most)
// and in 64 bits across warps and blocks, so that its error does not grow with the tokens.  Up to about 100 MB of dy the second pass finds it in L2.  8192 x 4096 bf16: 22 and 39 us (67 MB read,
// 67 MB read and 67 MB written), bound by latency with half the warps an SM could hold: 64 registers a thread; at 48 or 80 the
// second pass takes 53 and 47 us.  Arithmetic on pairs of values saves instructions here too, and no time.
constexpr int kGCols = 256;  // columns of a tile of the first pass: a warp has a row of it, eight columns a lane

// max that lets a NaN through
__device__ __forceinline__ float max_nan(float a, float b)
{
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// rows x (tiles * 256) columns a block; row_most [column block][m], col_most and sums [row block][n]
template <typename T>
__global__ void __launch_bounds__(256, 4)
grad_amax_kernel(const T *__restrict__ dy, long long m, long long n, long long stride, int vec, unsigned col_blocks, int tiles,
                 int rows, const float *__restrict__ row_scale, const float *__restrict__ col_scale,
                 uint32_t *__restrict__ row_most, uint32_t *__restrict__ col_most, float *__restrict__ sums)
{
    wait_previous_launch();
    allow_next_launch();
    __shared__ float cmax[8][kGCols], csum[8][kGCols];
    extern __shared__ uint32_t rmax[]; // [rows]; a row is always the same warp's
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const unsigned row_block = blockIdx.x / col_blocks, col_block = blockIdx.x - row_block * col_blocks;
    const long long r0 = (long long)row_block * rows, r1 = r0 + rows < m ? r0 + rows : m;
    for (int tile = 0; tile < tiles; tile++) {
        const long long c0 = ((long long)col_block * tiles + tile) * kGCols, c = c0 + lane * 8;
        if (c0 >= n) break;
        float cs[8], cm[8], s[8];
#pragma unroll
        for (int i = 0; i < 8; i++) cs[i] = col_scale && c + i < n ? col_scale[c + i] : 0.f, cm[i] = 0.f, s[i] = 0.f;
        // (columns behind the last one: their values are 0 and so is their scale; what a NaN row scale makes of them is not
        //  kept)
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
                uint32_t all = __reduce_max_sync(0xffffffffu, __float_as_uint(rm));
                if (lane == 0) rmax[r - r0] = tile ? max(all, rmax[r - r0]) : all;
            }
        };
        constexpr int kAhead = 4; // rows of a warp that are loaded together
        long long r = r0 + warp;
        if (vec && c0 + kGCols <= n) { // (no edge: addresses and bounds are a third of the instructions otherwise)
            const T *at = dy + r * stride + c;
            const long long pace = 8 * stride;
            for (; r + 8 * (kAhead - 1) < r1; r += 8 * kAhead, at += kAhead * pace) {
                Raw<T> raw[kAhead];
#pragma unroll
                for (int j = 0; j < kAhead; j++) load_raw(at + j * pace, raw[j]);
#pragma unroll
                for (int j = 0; j < kAhead; j++) take(raw[j], r + 8 * j);
            }
        }
        for (; r < r1; r += 8) {
            Raw<T> raw;
            load_raw(dy + r * stride, c, n, vec, raw);
            take(raw, r);
        }
        if (tile) __syncthreads(); // the tile before has been read
#pragma unroll
        for (int i = 0; i < 8; i++) cmax[warp][i * 32 + lane] = cm[i], csum[warp][i * 32 + lane] = s[i];
        __syncthreads();
        const long long col = c0 + threadIdx.x;
        const int at = (threadIdx.x & 7) * 32 + (threadIdx.x >> 3);
        if (col < n) {
            float most = 0.f;
            double sum = 0.; // (in fp32 every warp of every block could lose a half step)
#pragma unroll
            for (int w = 0; w < 8; w++) most = max_nan(most, cmax[w][at]), sum += csum[w][at];
            if (col_most) col_most[(long long)row_block * n + col] = __float_as_uint(most);
            if (sums) sums[(long long)row_block * n + col] = (float)sum;
        }
    }
    if (row_most) // (behind the last tile's barrier)
        for (int i = threadIdx.x; r0 + i < r1; i += 256) row_most[(long long)col_block * m + r0 + i] = rmax[i];
}

// A block quantises a tile of 128 rows x 256 columns both ways; the blocks of the first tile row also finish the bias's
// gradient and the columns' scales, those of the first tile column the rows' scales.  A row (column) that is not finite gets
// the scale NaN; what its integers are does not matter then.
template <typename T, typename B>
__global__ void __launch_bounds__(256, 4)
grad_quantize_kernel(const T *__restrict__ dy, long long m, long long n, long long stride, int vec, unsigned col_blocks,
                     const float *__restrict__ row_scale, const float *__restrict__ col_scale,
                     const uint32_t *__restrict__ row_most, int row_parts, const uint32_t *__restrict__ col_most,
                     const float *__restrict__ sums, int col_parts, long long tcols, int8_t *__restrict__ qg,
                     float *__restrict__ sg, int8_t *__restrict__ qh, float *__restrict__ sh, B *__restrict__ db)
{
    wait_previous_launch();
    allow_next_launch();
    __shared__ float row_a[kI8Tile], row_inv[kI8Tile], row_s[kI8Tile];
    __shared__ __align__(16) float col_a[kGCols], col_inv[kGCols], col_s[kGCols];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const unsigned row_block = blockIdx.x / col_blocks, col_block = blockIdx.x - row_block * col_blocks;
    const long long c = (long long)col_block * kGCols + lane * 8, r0 = (long long)row_block * kI8Tile;
    const float nan = __uint_as_float(0x7fc00000u);
    const long long col = (long long)col_block * kGCols + threadIdx.x;
    if (qh) {
        uint32_t most = 0;
        if (col < n)
#pragma unroll 8
            for (int b = 0; b < col_parts; b++) most = max(most, col_most[(long long)b * n + col]);
        const bool live = most != 0 && most < 0x7f800000u;
        col_a[threadIdx.x] = live ? __uint_as_float(most) : 0.f;
        col_inv[threadIdx.x] = live ? inverse_of(__uint_as_float(most)) : 0.f;
        if (row_block == 0 && col < n) sh[col] = most < 0x7f800000u ? __fdiv_rn(__uint_as_float(most), 127.f) : nan;
    }
    col_s[threadIdx.x] = qg && col < n ? col_scale[col] : 0.f;
    if (db && row_block == 0 && col < n) {
        double s = 0.;
#pragma unroll 8
        for (int b = 0; b < col_parts; b++) s += sums[(long long)b * n + col];
        db[col] = (B)s;
    }
    if (threadIdx.x < kI8Tile) {
        const long long r = r0 + threadIdx.x;
        uint32_t most = 0;
        if (qg && r < m)
#pragma unroll 8
            for (int b = 0; b < row_parts; b++) most = max(most, row_most[(long long)b * m + r]);
        const bool live = most != 0 && most < 0x7f800000u;
        row_a[threadIdx.x] = live ? __uint_as_float(most) : 0.f;
        row_inv[threadIdx.x] = live ? inverse_of(__uint_as_float(most)) : 0.f;
        row_s[threadIdx.x] = qh && r < m ? row_scale[r] : 0.f;
        if (qg && col_block == 0 && r < m) sg[r] = most < 0x7f800000u ? __fdiv_rn(__uint_as_float(most), 127.f) : nan;
    }
    __syncthreads();
    if (c >= tcols * kI8Tile) return;
    bool tiny = false; // a column of this lane whose 127 / a overflows: every value takes the exact way
#pragma unroll
    for (int i = 0; i < 8; i++) tiny |= qh && col_inv[lane * 8 + i] == 0.f && col_a[lane * 8 + i] > 0.f;
    // (the columns' scales stay in shared memory: in registers they leave no room for the loads ahead)
    auto eight = [&](const float *from, float (&v)[8]) {
        const float4 p = *reinterpret_cast<const float4 *>(from + lane * 8), q = *reinterpret_cast<const float4 *>(from + lane * 8 + 4);
        v[0] = p.x, v[1] = p.y, v[2] = p.z, v[3] = p.w, v[4] = q.x, v[5] = q.y, v[6] = q.z, v[7] = q.w;
    };
    // of row 0's chunk, without the swizzle (r0 and the block's first column begin a tile)
    const size_t base = ((size_t)row_block * tcols + (size_t)(c >> 7)) * kI8TileBytes + (size_t)(lane & 1) * 8;
    auto take = [&](const Raw<T> &raw, int row) { // row of the tile
        float v[8], x[8];
        widen(raw, v);
        const size_t at = base + row * 128 + (((lane >> 1 & 7) ^ (row & 7)) << 4);
        if (qg) {
            float cs[8];
            eight(col_s, cs);
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = __fmul_rn(v[i], cs[i]);
            const float a = row_a[row];
            *reinterpret_cast<uint2 *>(qg + at) = a > 0.f ? quant8<false>(x, a, row_inv[row]) : make_uint2(0u, 0u);
        }
        if (qh) {
            const float rs = row_s[row];
            uint32_t q[8];
            float far = 0.f, ci[8];
            eight(col_inv, ci);
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
                        const float a = col_a[lane * 8 + i];
                        q[i] = a > 0.f ? (uint32_t)quant_exact(x[i], a) : 0u;
                    }
                }
            }
            *reinterpret_cast<uint2 *>(qh + at) = make_uint2(pack4(q[0], q[1], q[2], q[3]), pack4(q[4], q[5], q[6], q[7]));
        }
    };
    const T *at = dy + (r0 + warp) * stride + c;
    const long long pace = 8 * stride;
    if (vec && r0 + kI8Tile <= m && (long long)(col_block + 1) * kGCols <= n) {
        constexpr int kAhead = 4;
#pragma unroll 1
        for (int row = warp; row < kI8Tile; row += 8 * kAhead, at += kAhead * pace) {
            Raw<T> raw[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; i++) load_raw(at + i * pace, raw[i]);
#pragma unroll
            for (int i = 0; i < kAhead; i++) take(raw[i], row + 8 * i);
        }
    } else {
#pragma unroll 1
        for (int row = warp; row < kI8Tile; row += 8) {
            Raw<T> raw;
            if (r0 + row < m) load_raw(dy + (r0 + row) * stride, c, n, vec, raw);
            else clear_raw(raw);
            take(raw, row);
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

// Blocks of the first pass.  They follow from the sizes alone: the bias's sum has one order.  Rows: long enough that a block's
// end is a small part, as long as every SM gets two blocks, and in 128 parts at the most (up to half a million rows); columns
// in 16 parts at the most (the second pass joins them in every block).  8192 x 4096 bf16, both passes: blocks of 64 rows
// 76 us, 128 rows 68, 256 rows 62, 448 rows 68.
struct GradBlocks {
    int rows, tiles, row_blocks, col_blocks;
    GradBlocks(long long m, long long n)
    {
        const long long cols = (n + kGCols - 1) / kGCols;
        tiles = (int)((cols + 15) / 16);
        col_blocks = (int)((cols + tiles - 1) / tiles);
        rows = 256;
        while (rows > 32 && (m + rows - 1) / rows * col_blocks < 2 * 148) rows /= 2;
        const long long least = ((m + 127) / 128 + 7) / 8 * 8;
        if (rows < least) rows = (int)(least < 4096 ? least : 4096); // (kept in shared memory)
        row_blocks = (int)((m + rows - 1) / rows);
    }
};

// scratch of the backward pass
struct GradBuffers {
    uint32_t *row_most, *col_most;
    float *sg, *sh, *sums;
    int8_t *qg, *qh;
    size_t total;
};

GradBuffers grad_buffers(uint8_t *ws, long long m, long long n, bool want_dx, bool want_dw, bool want_db)
{
    const GradBlocks g(m, n);
    GradBuffers b;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at = align_up(at + bytes, 256);
        return ws + here;
    };
    b.row_most = reinterpret_cast<uint32_t *>(take(want_dx ? (size_t)g.col_blocks * m * 4 : 0));
    b.col_most = reinterpret_cast<uint32_t *>(take(want_dw ? (size_t)g.row_blocks * n * 4 : 0));
    b.sums = reinterpret_cast<float *>(take(want_db ? (size_t)g.row_blocks * n * 4 : 0));
    b.sg = reinterpret_cast<float *>(take(want_dx ? (size_t)m * 4 : 0));
    b.sh = reinterpret_cast<float *>(take(want_dw ? (size_t)n * 4 : 0));
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
    const GradBlocks g(m, n);
    const long long tcols = i8_tiles(n), col_blocks = (n + kGCols - 1) / kGCols, blocks = col_blocks * i8_tiles(m);
    const size_t smem = (size_t)g.rows * 4;
    if (blocks > 0x7fffffffll) return REXSC_E_UNSUPPORTED;
    const int rc = launch_under("grad_amax_kernel", grad_amax_kernel<T>, (unsigned)(g.col_blocks * g.row_blocks), 256, smem, st,
                                dy, m, n, stride, vec, (unsigned)g.col_blocks, g.tiles, g.rows, want_dw ? row_scale : nullptr,
                                want_dx ? col_scale : nullptr, want_dx ? b.row_most : nullptr, want_dw ? b.col_most : nullptr,
                                db ? b.sums : nullptr);
    if (rc != REXSC_OK) return rc;
    auto second = [&](auto *to) {
        return launch_under("grad_quantize_kernel", grad_quantize_kernel<T, std::remove_pointer_t<decltype(to)>>, (unsigned)blocks,
                            256, 0, st, dy, m, n, stride, vec, (unsigned)col_blocks, row_scale, col_scale, b.row_most,
                            g.col_blocks, b.col_most, b.sums, g.row_blocks, tcols, want_dx ? b.qg : nullptr, b.sg,
                            want_dw ? b.qh : nullptr, b.sh, to);
    };
    if (db_dtype == REXSC_F16) return second(static_cast<__half *>(db));
    if (db_dtype == REXSC_BF16) return second(static_cast<__nv_bfloat16 *>(db));
    return second(static_cast<float *>(db));
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

extern "C" size_t rexsc_int8_linear_workspace_size(int64_t m, int64_t n, int64_t k, int32_t kernel)
{
    if (!good_extent(m) || !good_extent(n) || !good_extent(k) || k > kI8MaxDot || !known_kernel(kernel) || i8_tokens_fit(m, n, k, kernel))
        return 0;
    return align_up((size_t)m * 4, 256) + i8_bytes(m, k);
}

extern "C" int rexsc_int8_linear_fwd(const void *d_x, int32_t dtype, int64_t m, int64_t k, int64_t row_stride,
                                     const int8_t *d_w, const float *d_w_scale, int64_t n, const void *d_bias,
                                     int32_t bias_dtype, void *d_out, int32_t out_dtype, int32_t kernel, void *d_workspace,
                                     size_t workspace_bytes, void *stream)
{
    if (!d_x || !d_w || !d_w_scale || !d_out || !good_extent(m) || !good_extent(n) || !good_extent(k) || row_stride < 0 ||
        !known_dtype(dtype) || !known_dtype(out_dtype) || !known_kernel(kernel) || (d_bias && !known_dtype(bias_dtype)) ||
        (reinterpret_cast<uintptr_t>(d_w) & 255))
        return REXSC_E_BAD_ARG;
    if (k > kI8MaxDot) return REXSC_E_TOO_LONG;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    I8Product p{{}, along_columns(d_w, n, k), m, n, k, nullptr, d_w_scale, d_bias, bias_dtype, d_out, out_dtype, n};
    if (i8_tokens_fit(m, n, k, kernel)) return launch_i8_tokens(d_x, dtype, row_stride, p, st);
    if (!d_workspace || workspace_bytes < rexsc_int8_linear_workspace_size(m, n, k, kernel) || (reinterpret_cast<uintptr_t>(d_workspace) & 255))
        return REXSC_E_WORKSPACE;
    float *sx = static_cast<float *>(d_workspace);
    int8_t *qx = reinterpret_cast<int8_t *>(static_cast<uint8_t *>(d_workspace) + align_up((size_t)m * 4, 256));
    // (rows that pad the last tile stay as they are: they only reach outputs that are not stored)
    const int rc = launch_i8_quantize_rows(d_x, dtype, m, k, row_stride, qx, sx, false, st);
    if (rc != REXSC_OK) return rc;
    p.a = along_columns(qx, m, k);
    p.row_scale = sx;
    return launch_i8_product(p, kernel, true, st);
}

extern "C" int rexsc_int8_linear_train_fwd(const void *d_x, int32_t dtype, int64_t m, int64_t k, int64_t x_stride,
                                           const void *d_w, int32_t w_dtype, int64_t n, int64_t w_stride, const void *d_bias,
                                           int32_t bias_dtype, int8_t *d_xq, float *d_x_scale, int8_t *d_wq, float *d_w_scale,
                                           void *d_out, int32_t out_dtype, int32_t kernel, void *stream)
{
    if (!d_x || !d_xq || !d_x_scale || !d_wq || !d_w_scale || !d_out || !good_extent(m) || !good_extent(n) || !good_extent(k) ||
        x_stride < 0 || w_stride < 0 || !known_dtype(dtype) || (d_w && !known_dtype(w_dtype)) || !known_dtype(out_dtype) ||
        !known_kernel(kernel) || (d_bias && !known_dtype(bias_dtype)) ||
        ((reinterpret_cast<uintptr_t>(d_xq) | reinterpret_cast<uintptr_t>(d_wq)) & 255))
        return REXSC_E_BAD_ARG;
    if (k > kI8MaxDot) return REXSC_E_TOO_LONG;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    // (the weights first: the product reads them before it waits for the launch in front of it)
    int rc = d_w ? launch_i8_quantize_rows(d_w, w_dtype, n, k, w_stride, d_wq, d_w_scale, true, st) : REXSC_OK;
    if (rc == REXSC_OK) rc = launch_i8_quantize_rows(d_x, dtype, m, k, x_stride, d_xq, d_x_scale, true, st);
    if (rc != REXSC_OK) return rc;
    I8Product p{along_columns(d_xq, m, k), along_columns(d_wq, n, k), m, n, k, d_x_scale, d_w_scale, d_bias, bias_dtype, d_out, out_dtype, n};
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
    const I8Product px{along_columns(b.qg, m, n), along_rows(d_w, n, k), m, k, n, b.sg, nullptr, nullptr, 0, d_dx, dx_dtype, k};
    const I8Product pw{along_rows(b.qh, m, n), along_rows(d_x, m, k), n, k, m, b.sh, nullptr, nullptr, 0, d_dw, dw_dtype, k};
    if (d_dx && d_dw) return launch_i8_products(px, pw, kernel, true, st);
    if (d_dx) return launch_i8_product(px, kernel, true, st);
    return d_dw ? launch_i8_product(pw, kernel, true, st) : REXSC_OK;
}
