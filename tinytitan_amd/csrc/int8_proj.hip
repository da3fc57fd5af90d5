// Products of 8-bit integers: y[t][r] = fp16(token_scale[t] * weight_scale[r] * sum_k weight[r][k] * level[t][k]), the sum exact in
// 32-bit integers, over tokens quantised one by one:
//   token_scale = max |x| / 127,  level = round(x / token_scale)     (ties to even; both divisions as fp32 rounds them)
// A token of zeros has scale and levels zero.  A token with an infinite or NaN element has a NaN for a scale and zero levels: its
// outputs are NaN, other tokens' are their own.
#include "internal.h"
#include "wave_ops.h"

namespace tt {

namespace {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef int i4 __attribute__((ext_vector_type(4)));
typedef int i16v __attribute__((ext_vector_type(16)));
typedef unsigned u4 __attribute__((ext_vector_type(4)));
typedef unsigned u2 __attribute__((ext_vector_type(2)));

// The largest magnitude of eight halves, as bits: magnitudes are ordered as their bits are, and what is not finite is 0x7c00 or more.
__device__ __forceinline__ unsigned largest_bits(unsigned so_far, const u4 &x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) so_far = max(so_far, max(x[i] & 0x7fffu, (x[i] >> 16) & 0x7fffu));
    return so_far;
}
__device__ __forceinline__ float half_of_bits(unsigned bits) { return (float)__builtin_bit_cast(_Float16, (unsigned short)bits); }
__device__ __forceinline__ float token_scale(unsigned largest) { return largest >= 0x7c00u ? __builtin_nanf("") : half_of_bits(largest) / 127.0f; }
// Eight halves as levels; `scale` 0 or NaN: zeros.
__device__ __forceinline__ u2 levels_of(const u4 &x, float scale) {
    u2 out = {0u, 0u};
    const bool some = scale > 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float v = half_of_bits((x[i >> 1] >> (16 * (i & 1))) & 0xffffu);
        const int level = some ? (int)__builtin_rintf(v / scale) : 0;
        out[i >> 2] |= ((unsigned)level & 0xffu) << (8 * (i & 3));
    }
    return out;
}

// A workgroup per token.
__global__ __launch_bounds__(256) void quantise_rows_kernel(const _Float16 *x, long long x_stride, int columns, int8_t *levels, long long levels_stride,
                                                            float *scales) {
    __shared__ unsigned found[4];
    const long long token = blockIdx.x;
    const u4 *const row = reinterpret_cast<const u4 *>(x + token * x_stride);
    const int pieces = columns / 8;
    unsigned largest = 0;
    for (int i = threadIdx.x; i < pieces; i += 256) largest = largest_bits(largest, row[i]);
#pragma unroll
    for (int step = 32; step > 0; step /= 2) largest = max(largest, (unsigned)__shfl_xor((int)largest, step));
    if ((threadIdx.x & 63) == 0) found[threadIdx.x >> 6] = largest;
    __syncthreads();
    const float scale = token_scale(max(max(found[0], found[1]), max(found[2], found[3])));
    u2 *const to = reinterpret_cast<u2 *>(levels + token * levels_stride);
    for (int i = threadIdx.x; i < pieces; i += 256) to[i] = levels_of(row[i], scale);
    if (threadIdx.x == 0) scales[token] = scale;
}

struct ProductArgs {
    const int8_t *weights;
    const float *weight_scales;
    const int8_t *levels;
    const float *scales;
    _Float16 *y;
    long long levels_stride, y_stride;
    int rows, columns, tokens;
};

// A wavefront per 32 x 32 outputs, operands from memory as they are needed.
__global__ __launch_bounds__(256) void int8_tiles_kernel(const ProductArgs a) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, li = lane & 31, g = lane >> 5;
    const int row0 = (blockIdx.x * 4 + wave) * 32, token0 = blockIdx.y * 32;
    if (row0 >= a.rows) return;
    const int row = min(row0 + li, a.rows - 1), token = min(token0 + li, a.tokens - 1);
    const int8_t *const w = a.weights + (long long)row * a.columns;
    const int8_t *const x = a.levels + token * a.levels_stride;
    i16v acc = (i16v)0;
    for (int k = 16 * g; k < (a.columns + 31) / 32 * 32; k += 32) {
        i4 wf = (i4)0, xf = (i4)0;
        if (k < a.columns) {
            wf = *reinterpret_cast<const i4 *>(w + k);
            xf = *reinterpret_cast<const i4 *>(x + k);
        }
        acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(wf, xf, acc, 0, 0, 0);
    }
    if (token0 + li >= a.tokens) return;
    const float scale = a.scales[token];
    _Float16 *const to = a.y + token * a.y_stride;
#pragma unroll
    for (int v = 0; v < 16; ++v) {
        const int r = row0 + 8 * (v >> 2) + 4 * g + (v & 3);
        if (r < a.rows) to[r] = (_Float16)((float)acc[v] * a.weight_scales[r] * scale);
    }
}

bool aligned(const void *p, size_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

// (the sums of products of two levels, at most 2^14 each, stay below 2^31)
bool columns_served(int columns) { return columns % 16 == 0 && columns < 131072; }

int check_quantise(const tt_half *x, size_t x_stride, int token_count, int columns, const int8_t *levels, size_t levels_stride, const float *scales) {
    if (!x || !levels || !scales || token_count <= 0 || columns <= 0) return TT_HIP_ERR_INVALID_ARGUMENT;
    if (!columns_served(columns) || x_stride < (size_t)columns || x_stride % 8 != 0 || levels_stride < (size_t)columns || levels_stride % 16 != 0 ||
        !aligned(x, 16) || !aligned(levels, 16))
        return TT_HIP_ERR_SHAPE;
    return TT_HIP_OK;
}
int check_product(const int8_t *weights, const float *weight_scales, const tt_half *y, int rows, int columns, int token_count, size_t y_stride) {
    if (!weights || !weight_scales || !y || rows <= 0 || columns <= 0 || token_count <= 0) return TT_HIP_ERR_INVALID_ARGUMENT;
    if (!columns_served(columns) || !aligned(weights, 16) || y_stride < (size_t)rows) return TT_HIP_ERR_SHAPE;
    return TT_HIP_OK;
}

int launch_quantise(tt_hip_ctx *ctx, const tt_half *x, size_t x_stride, int token_count, int columns, int8_t *levels, size_t levels_stride, float *scales) {
    launch_profiled(ctx, quantise_rows_kernel, dim3((unsigned)token_count), dim3(256), 0u, reinterpret_cast<const _Float16 *>(x), (long long)x_stride,
                    columns, levels, (long long)levels_stride, scales);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? TT_HIP_OK : hip_fail(ctx, e, "quantise_rows_kernel launch");
}

int launch_product(tt_hip_ctx *ctx, const ProductArgs &a) {
    launch_profiled(ctx, int8_tiles_kernel, dim3((unsigned)((a.rows + 127) / 128), (unsigned)((a.tokens + 31) / 32)), dim3(256), 0u, a);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? TT_HIP_OK : hip_fail(ctx, e, "int8_tiles_kernel launch");
}

// The context's store for tokens that a call quantises itself: their levels, then their scales.
int ensure_levels(tt_hip_ctx *ctx, size_t bytes) {
    if (bytes <= ctx->levels_bytes) return TT_HIP_OK;
    if (ctx->capturing) return TT_HIP_ERR_BUSY;
    hipError_t e = hipStreamSynchronize(ctx->stream);
    if (e != hipSuccess) return hip_fail(ctx, e, "hipStreamSynchronize");
    if (ctx->levels) (void)hipFree(ctx->levels);
    ctx->levels = nullptr;
    ctx->levels_bytes = 0;
    ++ctx->generation;
    const size_t want = bytes + bytes / 4;
    e = hipMalloc(reinterpret_cast<void **>(&ctx->levels), want);
    if (e != hipSuccess) return hip_fail(ctx, e, "hipMalloc(token levels)");
    ctx->levels_bytes = want;
    return TT_HIP_OK;
}

}  // namespace

}  // namespace tt

using namespace tt;

extern "C" {

int tt_hip_int8_quantise_rows(tt_hip_ctx *ctx, const tt_half *x, size_t x_stride, int token_count, int columns, int8_t *levels,
                              size_t levels_stride, float *scales) {
    if (!ctx) return TT_HIP_ERR_INVALID_ARGUMENT;
    const int st = check_quantise(x, x_stride, token_count, columns, levels, levels_stride, scales);
    if (st != TT_HIP_OK) return st;
    BusyGuard guard(ctx);
    if (!guard.ok) return TT_HIP_ERR_BUSY;
    if (hipSetDevice(ctx->device) != hipSuccess) return TT_HIP_ERR_HIP;
    return launch_quantise(ctx, x, x_stride, token_count, columns, levels, levels_stride, scales);
}

int tt_hip_int8_projection_levels(tt_hip_ctx *ctx, const int8_t *weights, const float *weight_scales, const int8_t *levels, size_t levels_stride,
                                  const float *scales, tt_half *y, int rows, int columns, int token_count, size_t y_stride) {
    if (!ctx) return TT_HIP_ERR_INVALID_ARGUMENT;
    const int st = check_product(weights, weight_scales, y, rows, columns, token_count, y_stride);
    if (st != TT_HIP_OK) return st;
    if (!levels || !scales) return TT_HIP_ERR_INVALID_ARGUMENT;
    if (!aligned(levels, 16) || levels_stride < (size_t)columns || levels_stride % 16 != 0) return TT_HIP_ERR_SHAPE;
    BusyGuard guard(ctx);
    if (!guard.ok) return TT_HIP_ERR_BUSY;
    if (hipSetDevice(ctx->device) != hipSuccess) return TT_HIP_ERR_HIP;
    return launch_product(ctx, ProductArgs{weights, weight_scales, levels, scales, reinterpret_cast<_Float16 *>(y), (long long)levels_stride,
                                           (long long)y_stride, rows, columns, token_count});
}

int tt_hip_int8_projection(tt_hip_ctx *ctx, const int8_t *weights, const float *weight_scales, const tt_half *x, size_t x_stride, tt_half *y, int rows,
                           int columns, int token_count, size_t y_stride) {
    if (!ctx) return TT_HIP_ERR_INVALID_ARGUMENT;
    const int st = check_product(weights, weight_scales, y, rows, columns, token_count, y_stride);
    if (st != TT_HIP_OK) return st;
    if (!x) return TT_HIP_ERR_INVALID_ARGUMENT;
    if (x_stride < (size_t)columns || x_stride % 8 != 0 || !aligned(x, 16)) return TT_HIP_ERR_SHAPE;
    BusyGuard guard(ctx);
    if (!guard.ok) return TT_HIP_ERR_BUSY;
    if (hipSetDevice(ctx->device) != hipSuccess) return TT_HIP_ERR_HIP;
    const size_t level_bytes = ((size_t)token_count * columns + 255) & ~(size_t)255;
    int done = ensure_levels(ctx, level_bytes + (size_t)token_count * sizeof(float));
    if (done != TT_HIP_OK) return done;
    float *const scales = reinterpret_cast<float *>(ctx->levels + level_bytes);
    done = launch_quantise(ctx, x, x_stride, token_count, columns, ctx->levels, (size_t)columns, scales);
    if (done != TT_HIP_OK) return done;
    return launch_product(ctx, ProductArgs{weights, weight_scales, ctx->levels, scales, reinterpret_cast<_Float16 *>(y), columns, (long long)y_stride, rows,
                                           columns, token_count});
}

}  // extern "C"
