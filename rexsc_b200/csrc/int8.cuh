// 8-bit matrices of the linear layers: their layout, and the quantisation of one value.
//
// Layout ("tiled"): an R x C matrix of int8 is cut into tiles of 128 rows x 128 columns, tile (i, j) at
// (i * ceil(C / 128) + j) * 16 KiB.  Inside a tile, row r's 128 bytes lie at r * 128 and its 16-byte chunks are permuted,
// chunk c at c ^ (r & 7): the 128-byte swizzle of the tensor core's shared-memory operands.  A tile is therefore one
// contiguous copy, and the same image serves as an operand whose contraction runs along the columns (K-major: y = x w^T)
// and as one whose contraction runs along the rows (MN-major: the gradients), without a transposed copy.
// Columns that pad the last tile are zero; rows that pad it are zero where the matrix is a handle of the caller's.
#pragma once

#include "common.cuh"

namespace rexsc {

constexpr int kI8Tile = 128;                    // rows and columns of a tile
constexpr int kI8TileBytes = kI8Tile * kI8Tile; // 16 KiB
constexpr long long kI8MaxDot = REXSC_INT8_MAX_DOT; // sums of so many products of -128 .. 127 do not overflow int32
static_assert(kI8MaxDot * 128 * 128 < (1ll << 31), "int32 sums");

static inline long long i8_tiles(long long n) { return (n + kI8Tile - 1) / kI8Tile; }
static inline size_t i8_bytes(long long rows, long long cols) { return (size_t)i8_tiles(rows) * i8_tiles(cols) * kI8TileBytes; }
static inline size_t dtype_bytes(int dtype) { return dtype == REXSC_F32 ? 4 : 2; }

// byte offset of column c (a multiple of 8 for 8-byte accesses) of row r; tcols = tiles per tile row
__device__ __forceinline__ size_t i8_offset(long long r, long long c, long long tcols)
{
    return ((size_t)(r >> 7) * tcols + (size_t)(c >> 7)) * kI8TileBytes + (size_t)(r & 127) * 128 +
           (size_t)(((((int)c >> 4) & 7) ^ ((int)r & 7)) << 4) + (size_t)(c & 15);
}

// ---- launches that begin under the end of the one before them on their stream ----------------------------------
// What keeps them in order:
//   * a kernel waits for the launch before it (wait_previous_launch) before it touches global memory; only products read
//     weights that were quantised earlier sooner;
//   * it lets the next one begin (allow_next_launch) after that wait, and after it has taken its TMEM: when a kernel begins,
//     all but the launch right before it has finished, the one that wrote those weights too, and a kernel that holds TMEM
//     while it waits keeps none from the one it waits for.
// One token through 4096 x 4096, call after call: 8.4 us, 10.2 without.
__device__ __forceinline__ void wait_previous_launch() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void allow_next_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <typename... P, typename... A>
int launch_under(const char *what, void (*kernel)(P...), unsigned blocks, unsigned threads, size_t smem, cudaStream_t st, A... args)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(blocks);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
    note_kernel_launch();
    if (e != cudaSuccess) {
        cudaGetLastError();
        set_cuda_error(e, what);
        return REXSC_E_CUDA;
    }
    return REXSC_OK;
}

// ---- host launchers ------------------------------------------------------------------------------------------
int launch_i8_quantize_rows(const void *d_x, int dtype, long long rows, long long cols, long long stride, int8_t *d_data,
                            float *d_scale, bool pad_rows, cudaStream_t st);

// out[i, j] = (sum_k a[i, k] b[j, k]) * row_scale[i] * col_scale[j] + bias[j]
struct I8Operand {
    const int8_t *data;
    long long step_mn, step_k; // tiles from one 128-row block of the operand to the next, and from one 128-step of the
                               // contraction to the next
    long long mn_tiles;        // 128-row blocks that exist
    int mn_major;              // 0: a tile's rows are the operand's rows; 1: a tile's rows are the contraction
};
struct I8Product {
    I8Operand a, b;
    long long m, n, k;      // rows and columns of the output, length of the contraction
    const float *row_scale; // [m]
    const float *col_scale; // [n] or null
    const void *bias;       // [n] or null
    int bias_dtype;
    void *out;
    int out_dtype;
    long long out_stride;   // elements between rows of the output
};
// kernel: REXSC_INT8_*.  after_quantize: the launch may begin while the previous one on the stream (which writes operand a) still runs
int launch_i8_product(const I8Product &p, int kernel, bool after_quantize, cudaStream_t st);
// two products that do not depend on one another, in one launch where both are small
int launch_i8_products(const I8Product &p, const I8Product &q, int kernel, bool after_quantize, cudaStream_t st);
// a few tokens that the product's kernel quantises by itself: x takes the place of p.a and p.row_scale
bool i8_tokens_fit(long long m, long long n, long long k, int kernel);
int launch_i8_tokens(const void *x, int dtype, long long stride, const I8Product &p, cudaStream_t st);

} // namespace rexsc
