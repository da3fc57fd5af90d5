// Differential attention: a head's weights are the difference of two softmax maps over the cache.
//
//   a   = softmax(scale K1 q1) V - lambda softmax(scale K2 q2) V       q1, q2: the halves of the head's query row, K1, K2 those of
//   out = gate * out_scale * weight * a / rms(a)                        the KV head's key rows; lambda per head, or per token and head
//
// The passes over K and V are those of plain attention with two rows a head: the split-K kernel's kKeepMaps, whose tiles take the maps of
// the heads that share a KV head together, so that the cache is read once for both.  A launch of one split has both maps' sums in its LDS and
// writes the finished rows (32/8 heads of 128 behind 300 keys 8.5 -> 5.6 us, 24 rows behind 3,000 over 8 bits 33.7 -> 28.2).  Here are the launches and
// the pass behind those of several splits, which adds up their partial results of both maps (as attn_join.hip does: the rows' o and l about a common
// maximum), subtracts, and applies norm and gate in fp32 with one rounding.  A row that sees no key gives zeros.
//
// Memory bounds a long decode: 205 MB behind 100,001 keys of 16/2 heads of 256 take 40 us, the pass alone 32 (6.4 TB/s).  The join reads 2 KiB
// a (token, head) and split, by one CU an item, since the norm needs the whole row: 112 splits, 7 us.
//
// Roundings, beside the last one of a row: the matrix instructions' operands are fp16, as in every kernel here.  A weight of either map is rounded to it for
// the second product (its sum is that of the rounded weights over fp16 pages).  Over quantised pages so is a K operand, level * scale + bias, and in
// the split-K kernel a weight once more behind its product with a group's V scale, once for the group's 64 dims where a widened V operand would be
// rounded in each; in front of the chunk kernel every value of K and V is, whose pages are dequantised to fp16.  Against 64 bits 2.5 - 3e-4 over fp16
// pages (2-norm; the final rounding alone is 2.0e-4) and 4.6 - 7e-4 over 8 and 4 bits: a difference of maps keeps the errors of both and little of
// their sums.
#include <algorithm>

#include "splitk_kernel.h"

namespace tt {

namespace {

typedef float f2 __attribute__((ext_vector_type(2)));

// A (token, head) item is D / 4 threads of four dims each, and G of those that share its splits, for both maps or (BY_MAP) for each; a workgroup is
// ITEMS of them.  With many splits it waits for memory, and then for one item's sums behind each other: BY_MAP, a thread has most of what it asks for
// on its way at once (8 x 14 splits; of heads of 256, whose 1,024 threads have 128 registers each, 8 x 8) and adds up half as many.  us a decode step, 16 groups
// for both maps / 8 for each: 16/2 heads of 256 behind 20,000 keys 18.1 / 17.3, behind 100,000 40.5 / 39.6, 3 rows behind 9,000 14.4 / 13.6, 32/8 of 128 behind
// 40,000 30.3 / 29.6, 16/4 of 64 behind 60,000 15.2 / 14.4.
template <int D, int G, bool BY_MAP>
__global__ __launch_bounds__((BY_MAP ? 2 : 1) * G * D / 4 > 256 ? (BY_MAP ? 2 : 1) * G * D / 4 : 256) void attn_maps_join_kernel(const MapsJoinArgs a) {
    constexpr int LANES = D / 4, PER_ITEM = (BY_MAP ? 2 : 1) * G * LANES, THREADS = PER_ITEM > 256 ? PER_ITEM : 256, ITEMS = THREADS / PER_ITEM;
    constexpr int BATCH = BY_MAP ? (D == 256 ? 8 : 14) : 4, MAPS = BY_MAP ? 1 : 2;
    __shared__ f4 sums[G > 1 ? 2 : 1][G][G > 1 ? ITEMS * LANES : 1];
    __shared__ f2 stats[G > 1 ? 2 : 1][G][ITEMS];
    const int lane = threadIdx.x % LANES, in_group = threadIdx.x / LANES, item = in_group % ITEMS, g = in_group / ITEMS % G;
    const int first_map = BY_MAP ? in_group / (ITEMS * G) : 0;  // this thread's, of MAPS
    const int d = lane * 4, seq = blockIdx.y;
    const unsigned at_item = blockIdx.x * ITEMS + item, heads = a.heads;  // (rows x heads fit 31 bits)
    const bool real = at_item < (unsigned)a.rows * heads;
    const int row = real ? (int)(at_item / heads) : 0, head = real ? (int)(at_item - row * heads) : 0;
    const JoinSeq sq = a.seq[seq];
    // (asked for here, in front of the partial results)
    const float lambda = a.maps.lambda[seq * a.lambda_seq_stride + row * a.maps.lambda_stride + head];
    h4 gate = (h4)(_Float16)0.0f;
    if (a.gate) {
        gate = *(const __attribute__((address_space(1))) h4_unaligned *)(global_halves)(a.gate + seq * a.g_seq_stride + row * a.g_tok_stride + (long long)head * D + d);
    }
    const f4 weight = map_weight4(a.maps, d);
    // The tile's splits, as the pass counted them.
    const PassParts &p = a.parts;
    const int tok_tile = (unsigned)row / (unsigned)p.tt, t0 = tok_tile * p.tt, tile_end = max(0, min(sq.total, sq.start + min(t0 + p.tt, a.rows)));
    const int first_lim = min(sq.total, sq.start + t0 + 1);
    const int k0 = a.window > 0 && first_lim > a.window ? (first_lim - a.window) & ~31 : 0;
    const int n = (int)((unsigned)(max(tile_end - k0, 1) + p.split_len - 1) / (unsigned)p.split_len);
    const size_t stride = (size_t)p.n_tiles * p.nt;
    f4 acc[MAPS];
    float m[MAPS], l[MAPS];
#pragma unroll
    for (int map = 0; map < MAPS; ++map) {
        acc[map] = (f4)0.0f;
        m[map] = kNegBig;
        l[map] = 0.0f;
    }
    // The maps' rows in split 0: next to each other, but where a tile ends between them.
    const int kvh = (unsigned)(2 * head) / (unsigned)a.group2, in_kvh = 2 * head - kvh * a.group2;
    const int hsub = (unsigned)in_kvh / (unsigned)p.gh, in_tile = in_kvh - hsub * p.gh;
    const size_t first_row = (size_t)((kvh * p.hsubs + hsub) * p.tok_tiles + tok_tile) * p.nt + (row - t0) * p.gh + in_tile + (size_t)sq.first_split * stride;
    const size_t second_row = in_tile + 1 < p.gh ? first_row + 1 : first_row + (size_t)p.tok_tiles * p.nt - in_tile;
    const size_t at[2] = {first_map ? second_row : first_row, second_row};
    for (int first = g; first < n; first += G * BATCH) {
        f4 o[MAPS][BATCH];
        f2 ml[MAPS][BATCH];
        // (a split that is not there is not asked for: read as the last one again, they were most of what a workgroup fetched)
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
#pragma unroll
            for (int map = 0; map < MAPS; ++map) {
                ml[map][i] = f2{kNegBig, 0.0f};
                o[map][i] = (f4)0.0f;
            }
            if (first + i * G < n) {
                const size_t s = (size_t)(first + i * G) * stride;
#pragma unroll
                for (int map = 0; map < MAPS; ++map) {
                    ml[map][i] = *reinterpret_cast<const f2 *>(p.ml + (at[map] + s) * 2);
                    o[map][i] = *reinterpret_cast<const f4 *>(p.o + (at[map] + s) * D + d);
                }
            }
        }
#pragma unroll
        for (int map = 0; map < MAPS; ++map) {
            float top = m[map];
#pragma unroll
            for (int i = 0; i < BATCH; ++i) top = fmaxf(top, ml[map][i][0]);
            const float keep = fast_exp2(m[map] - top);
            l[map] *= keep;
            acc[map] *= keep;
            m[map] = top;
#pragma unroll
            for (int i = 0; i < BATCH; ++i) {
                const float f = fast_exp2(ml[map][i][0] - top);
                l[map] += f * ml[map][i][1];
                acc[map] += f * o[map][i];
            }
        }
    }
    if constexpr (G > 1) {
#pragma unroll
        for (int map = 0; map < MAPS; ++map) {
            sums[first_map + map][g][item * LANES + lane] = acc[map];
            if (lane == 0) stats[first_map + map][g][item] = f2{m[map], l[map]};
        }
        __syncthreads();
        if (!BY_MAP && g != 0) return;
        if (g == 0) {
#pragma unroll
            for (int map = 0; map < MAPS; ++map) {
                float top = kNegBig;
#pragma unroll
                for (int i = 0; i < G; ++i) top = fmaxf(top, stats[first_map + map][i][item][0]);
                acc[map] = (f4)0.0f;
                l[map] = 0.0f;
#pragma unroll
                for (int i = 0; i < G; ++i) {
                    const float f = fast_exp2(stats[first_map + map][i][item][0] - top);
                    l[map] += f * stats[first_map + map][i][item][1];
                    acc[map] += f * sums[first_map + map][i][item * LANES + lane];
                }
            }
        }
    }
    f4 a1 = acc[0] * (l[0] > 0.0f ? 1.0f / l[0] : 0.0f), a2 = acc[MAPS - 1] * (l[MAPS - 1] > 0.0f ? 1.0f / l[MAPS - 1] : 0.0f);
    if constexpr (BY_MAP) {
        if (g == 0 && first_map) sums[1][0][item * LANES + lane] = a2;  // (which this thread alone has read)
        __syncthreads();
        if (g != 0 || first_map) return;
        a2 = sums[1][0][item * LANES + lane];
    }
    f4 out;
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = map_difference(a1[i], a2[i], lambda);
    const float scale = map_row_scale<LANES>(a.maps, out);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        out[i] *= scale * weight[i];
        if (a.gate) out[i] *= sigmoid((float)gate[i]);
    }
    if (!real) return;
    _Float16 *const to = a.out + seq * a.o_seq_stride + row * a.o_tok_stride + (long long)head * D + d;
    const h4 r = {(_Float16)out[0], (_Float16)out[1], (_Float16)out[2], (_Float16)out[3]};
    if (a.aligned) {
        *reinterpret_cast<h4 *>(to) = r;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) to[i] = r[i];
    }
}

// A wavefront per head: lambda = exp(q1 . k1) - exp(q2 . k2) + init.
__global__ __launch_bounds__(64) void diff_lambda_kernel(const float *q1, const float *k1, const float *q2, const float *k2, long long stride, int dims,
                                                         float init, float *lambda) {
    const long long at = blockIdx.x * stride;
    float first = 0.0f, second = 0.0f;
    for (int i = threadIdx.x; i < dims; i += 64) {
        first += q1[at + i] * k1[at + i];
        second += q2[at + i] * k2[at + i];
    }
#pragma unroll
    for (int step = 32; step > 0; step /= 2) {
        first += __shfl_xor(first, step);
        second += __shfl_xor(second, step);
    }
    if (threadIdx.x == 0) lambda[blockIdx.x] = expf(first) - expf(second) + init;
}

template <int D, int G, bool BY_MAP>
void launch_join_of(tt_hip_ctx *ctx, int n_seq, const MapsJoinArgs &args) {
    constexpr int PER_ITEM = (BY_MAP ? 2 : 1) * G * D / 4, THREADS = PER_ITEM > 256 ? PER_ITEM : 256, ITEMS = THREADS / PER_ITEM;
    const long long items = (long long)args.rows * args.heads;
    hipLaunchKernelGGL((attn_maps_join_kernel<D, G, BY_MAP>), dim3((unsigned)((items + ITEMS - 1) / ITEMS), (unsigned)n_seq), dim3(THREADS), 0, ctx->stream, args);
}
template <int D>
void launch_join_by_splits(tt_hip_ctx *ctx, int n_seq, const MapsJoinArgs &args, int most_splits) {
    if (most_splits <= 4) launch_join_of<D, 1, false>(ctx, n_seq, args);
    else if (most_splits <= 16 || (long long)args.rows * args.heads * n_seq >= 4 * ctx->n_cus) launch_join_of<D, 4, false>(ctx, n_seq, args);
    else launch_join_of<D, 8, true>(ctx, n_seq, args);
}

template <int D, int NT, int BITS, int STREAM>
int launch_pass(tt_hip_ctx *ctx, const LaunchPlan &plan, int n_seq, const SplitKMaps &args) {
    auto kernel = attn_splitk_kernel<D, NT, 4, BITS, kKeepMaps, STREAM>;
    dim3 grid((unsigned)plan.n_splits_max, (unsigned)plan.n_tiles, (unsigned)n_seq);
    if (plan.packed_splits > 0) grid = dim3((unsigned)plan.packed_splits, (unsigned)plan.n_tiles);
    if (plan.xcd_grid) grid = dim3((unsigned)(((long long)plan.n_splits_max * plan.n_tiles + 7) / 8 * 8), 1u, (unsigned)n_seq);
    launch_profiled(ctx, kernel, grid, dim3(256), (unsigned)plan.lds_bytes, args);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? TT_HIP_OK : hip_fail(ctx, e, "attn_splitk_kernel launch");
}

}  // namespace

int configure_maps_kernels(tt_hip_ctx *ctx) {
    hipError_t e = hipSuccess;
#define TT_CFG(DD, NN, BB, SS) \
    if (e == hipSuccess) e = hipFuncSetAttribute(reinterpret_cast<const void *>(attn_splitk_kernel<DD, NN, 4, BB, kKeepMaps, SS>), \
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds_bytes_for(DD, NN, 4));
#define TT_CFG_BITS(DD, NN) \
    TT_CFG(DD, NN, 16, 0) TT_CFG(DD, NN, 16, 1) TT_CFG(DD, NN, 8, 0) TT_CFG(DD, NN, 8, 1) TT_CFG(DD, NN, 4, 0) TT_CFG(DD, NN, 4, 1)
    TT_CFG_BITS(256, 16) TT_CFG_BITS(256, 32) TT_CFG_BITS(128, 16) TT_CFG_BITS(128, 32) TT_CFG_BITS(64, 16) TT_CFG_BITS(64, 32)
#undef TT_CFG_BITS
#undef TT_CFG
    return e == hipSuccess ? TT_HIP_OK : hip_fail(ctx, e, "hipFuncSetAttribute(split-K max dynamic LDS)");
}

int launch_splitk_maps(tt_hip_ctx *ctx, const LaunchPlan &plan, int head_dim, int n_seq, const SplitKMaps &args, int kv_bits) {
#define TT_CASE(DD, NN)                                                                                        \
    if (head_dim == DD && plan.nt == NN) {                                                                     \
        if (kv_bits == 16) return plan.stream ? launch_pass<DD, NN, 16, 1>(ctx, plan, n_seq, args) : launch_pass<DD, NN, 16, 0>(ctx, plan, n_seq, args); \
        if (kv_bits == 8) return plan.stream ? launch_pass<DD, NN, 8, 1>(ctx, plan, n_seq, args) : launch_pass<DD, NN, 8, 0>(ctx, plan, n_seq, args);    \
        if (kv_bits == 4) return plan.stream ? launch_pass<DD, NN, 4, 1>(ctx, plan, n_seq, args) : launch_pass<DD, NN, 4, 0>(ctx, plan, n_seq, args);    \
    }
    TT_CASE(256, 16)
    TT_CASE(256, 32)
    TT_CASE(128, 16)
    TT_CASE(128, 32)
    TT_CASE(64, 16)
    TT_CASE(64, 32)
#undef TT_CASE
    return TT_HIP_ERR_SHAPE;
}

int launch_maps_join(tt_hip_ctx *ctx, int head_dim, int n_seq, const MapsJoinArgs &args, int most_splits) {
    if (n_seq > kMaxSeqPerLaunch || (long long)args.rows * args.heads > 0x7fffffffll) return TT_HIP_ERR_SHAPE;
    switch (head_dim) {
        case 256: launch_join_by_splits<256>(ctx, n_seq, args, most_splits); break;
        case 128: launch_join_by_splits<128>(ctx, n_seq, args, most_splits); break;
        case 64: launch_join_by_splits<64>(ctx, n_seq, args, most_splits); break;
        default: return TT_HIP_ERR_SHAPE;
    }
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? TT_HIP_OK : hip_fail(ctx, e, "attn_maps_join_kernel launch");
}

}  // namespace tt

using namespace tt;

extern "C" int tt_hip_diff_lambda(tt_hip_ctx *ctx, const float *q1, const float *k1, const float *q2, const float *k2, size_t vector_stride, int n_heads,
                                  int dims, float lambda_init, float *lambda) {
    if (!ctx || !q1 || !k1 || !q2 || !k2 || !lambda || n_heads <= 0 || dims <= 0) return TT_HIP_ERR_INVALID_ARGUMENT;
    if (vector_stride != 0 && vector_stride < (size_t)dims) return TT_HIP_ERR_SHAPE;
    BusyGuard guard(ctx);
    if (!guard.ok) return TT_HIP_ERR_BUSY;
    if (hipSetDevice(ctx->device) != hipSuccess) return TT_HIP_ERR_HIP;
    hipLaunchKernelGGL(diff_lambda_kernel, dim3((unsigned)n_heads), dim3(64), 0, ctx->stream, q1, k1, q2, k2, (long long)vector_stride, dims, lambda_init,
                       lambda);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? TT_HIP_OK : hip_fail(ctx, e, "diff_lambda_kernel launch");
}
