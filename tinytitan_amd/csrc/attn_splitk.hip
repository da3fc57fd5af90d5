// Split-K flash attention (splitk_kernel.h): its launches, and the pass that combines the splits' partial results.
#include <algorithm>
#include <type_traits>

#include "splitk_kernel.h"

namespace tt {

// ---------------------------------------------------------------------------
// Pass 2: cross-split log-sum-exp combine, gate and fp16 store.
// grid = (row within tile * D/64 + dim chunk, tile, sequence), 256 threads.
// Every wave first finds the row's global max over all splits (a few scalars
// per lane), which makes the per-split terms independent: a thread owns 4
// output dims (lane % 16) of the workgroup's 64-dim chunk and the splits
// 4 * wave + lane / 16, + 16, ..., all loads in flight at once; the 16 split
// groups add up through two shuffles and LDS.  All-empty input yields zeros
// (sources/TinyTitanCore/Metal/Attention/attention.metal:418-427).
// ---------------------------------------------------------------------------
// What such a pass takes is its chain of trips to memory, and it is two: the arguments, then the gate, the
// maxima and the partial rows together -- with the gate converted where it was loaded, its arguments read in a trip of
// their own and the second 64 maxima behind the first they were five.  A decode step's launch 0.2 us less (two layers of 7
// sequences of 300 .. 9,000 keys over 4 bits 40.8 -> 40.0 us, four of one of 20,010 over 8 bits 78.2 -> 77.4), the rows kernel
// behind a chunk of 128 rows over key ranges 2.2 (two layers behind 32,640 keys 240.5 -> 236.1).
typedef float f2 __attribute__((ext_vector_type(2)));
typedef const __attribute__((address_space(1))) f2 *global_pairs;  // part_ml: a partial row's (max, sum)
typedef const __attribute__((address_space(1))) char *global_bytes;

// What attn_combine_kernel reads in the place of a split that is not there: a partial row of zeros.  (Any other row's values would do but for
// infinite ones, which a factor of zero makes NaN of; a select behind the load is instructions on every value, a branch around it a wait of its own.)
static __device__ __align__(256) float no_split[256];
__device__ __forceinline__ global_bytes no_row() {
    global_bytes at = (global_bytes)no_split;
    asm("" : "+s"(at));  // (an address like the others, not zeros the compiler knows of and branches to)
    return at;
}

__device__ __forceinline__ int splits_of(const TileInfo &ti, int split_len) {
    return (int)((unsigned)(max(ti.tile_end - ti.k0, 1) + split_len - 1) / (unsigned)split_len);  // (an empty range has one, of zeros)
}

template <int D, int NT, bool SINKS>
__global__ __launch_bounds__(256) void attn_combine_kernel([[maybe_unused]] const SplitKArgs args) {  // (load_args reads them)
    constexpr int DCH = D / 64;
    __shared__ float sm[4][68];
    const int n = blockIdx.x / DCH, dchunk = blockIdx.x - n * DCH;
    const int tile = blockIdx.y, seq = blockIdx.z;
    SplitKHot a;
    SplitKSeq sq;
    SplitKOut out;
    load_args(a, sq, out, seq);
    const TileInfo ti = tile_info<SINKS>(a, sq, tile);
    if (n >= ti.tile_rows * a.gh) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int n_splits = splits_of(ti, a.split_len);
    // partial rows of split s: ((first_split + s) * n_tiles + tile) * NT + n
    const size_t tstride = (size_t)a.n_tiles * NT;
    const size_t first_row = (size_t)sq.first_split * tstride + (size_t)tile * NT + n;
    const int d = dchunk * 64 + (lane & 15) * 4;
    const global_pairs ml = (global_pairs)a.part_ml + first_row;
    const global_bytes rows = (global_bytes)a.part_o + (first_row * D + d) * sizeof(float);
    const global_bytes zeros = no_row() + d * sizeof(float);
    auto partial_row = [&](int s) {
        return *(const __attribute__((address_space(1))) f4 *)(s < n_splits ? rows + s * tstride * (D * sizeof(float)) : zeros);
    };
    // the gate of the dim that a thread of the first wavefront stores at the end, first of all requests
    const int tl = (n * a.gh_inv) >> 16;
    const int hh = ti.kvh * a.group + ti.hsub * a.gh + (n - tl * a.gh);
    const long long out_dim = (long long)hh * D + dchunk * 64 + lane;
    const bool gated = wave == 0 && out.gate;
    _Float16 gate = (_Float16)0.0f;
    if (gated) gate = ((global_halves)out.gate)[seq * out.g_seq_stride + (ti.t0 + tl) * out.g_tok_stride + out_dim];
    const int s0 = wave * 4 + (lane >> 4);
    f4 acc = (f4)0.0f;
    float l = 0.0f, factor = 1.0f;
    // This thread's first BATCH splits are requested BEFORE the global max is known: their
    // addresses do not depend on it, so the max's loads and these share one trip to memory.
    auto sum_splits = [&](auto batch) {
        constexpr int BATCH = decltype(batch)::value, MAXIMA = (BATCH * 16 + 63) / 64;
        f4 po[BATCH];
        f2 pml[BATCH];
        float maxima[MAXIMA];
#pragma unroll
        for (int i = 0; i < MAXIMA; ++i) maxima[i] = ml[min(lane + 64 * i, n_splits - 1) * tstride][0];
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            const int s = s0 + 16 * i;
            pml[i] = ml[(s < n_splits ? s : 0) * tstride];
            po[i] = partial_row(s);
        }
        __builtin_amdgcn_sched_barrier(0);  // (the maximum's wait is not to come in front of the rest of the requests)
        if (gated) {
            factor = sigmoid((float)gate);
            asm volatile("" : "+v"(factor));  // (here, while the rows are on their way, and not behind their sums)
        }
        float mg = maxima[0];
#pragma unroll
        for (int i = 1; i < MAXIMA; ++i) mg = fmaxf(mg, maxima[i]);
        for (int s = lane + 64 * MAXIMA; s < n_splits; s += 64) mg = fmaxf(mg, ml[s * tstride][0]);
        mg = wave_max_f32(mg, lane);
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            const float f = s0 + 16 * i < n_splits ? fast_exp2(pml[i][0] - mg) : 0.0f;
            l += f * pml[i][1];
            acc += f * po[i];
        }
#pragma unroll 4
        for (int s = s0 + 16 * BATCH; s < n_splits; s += 16) {
            const f2 p = ml[s * tstride];
            const float f = fast_exp2(p[0] - mg);
            l += f * p[1];
            acc += f * partial_row(s);
        }
    };
    // (few splits: requests for the places of more would each pass through the CU's vector memory path; 34 splits in places for 64,
    // four layers of 4 rows behind 8,190 keys over 8 bits, 83.8 us, in places for 128 84.3)
    if (n_splits <= 32) sum_splits(std::integral_constant<int, 2>{});
    else if (n_splits <= 64) sum_splits(std::integral_constant<int, 4>{});
    else sum_splits(std::integral_constant<int, 8>{});
    // (lanes l, l ^ 16, l ^ 32, l ^ 48, added in that order: v_permlane16_swap / v_permlane32_swap, no trip through LDS)
    l = sum_across_quarters(l);
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = sum_across_quarters(acc[i]);
    if (lane < 16) *reinterpret_cast<f4 *>(&sm[wave][lane * 4]) = acc;
    if (lane == 0) sm[wave][64] = l;
    __syncthreads();
    if (wave == 0) {
        float o = 0.0f, lsum = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            lsum += sm[w][64];
            o += sm[w][lane];
        }
        o *= lsum > 0.0f ? 1.0f / lsum : 0.0f;
        if (gated) o *= factor;
        typedef __attribute__((address_space(1))) _Float16 *global_out;
        ((global_out)out.out)[seq * out.o_seq_stride + (ti.t0 + tl) * out.o_tok_stride + out_dim] = (_Float16)o;
    }
}

// Pass 2 for launches of many tiles with few splits each (a chunk through the split-K tiles, or through the chunk
// kernel over key ranges): one workgroup per four rows of a tile instead of one per (row, 64 dims) -- the many tiny
// workgroups of attn_combine_kernel cost more to dispatch than these take to run.  A thread owns one (row, 4 dims)
// item and all of its splits, up to kCombineRowsSplits at a time: their loads are requested together, so a thread makes
// one trip to memory per turn, not one per split (the host sends more than two turns' worth to the other kernel).
// grid = (NT / 4, tile, sequence), 256 threads.
constexpr int kCombineRowsSplits = 16;

template <int D, int NT, bool SINKS>
__global__ __launch_bounds__(256) void attn_combine_rows_kernel([[maybe_unused]] const SplitKArgs args) {  // (load_args reads them)
    constexpr int D4 = D / 4, ROWS = 4;
    static_assert(ROWS * D4 <= 256, "an item a thread");
    const int tile = blockIdx.y, seq = blockIdx.z;
    SplitKHot a;
    SplitKSeq sq;
    SplitKOut out;
    load_args(a, sq, out, seq);
    const TileInfo ti = tile_info<SINKS>(a, sq, tile);
    const int n = blockIdx.x * ROWS + (int)threadIdx.x / D4, d = ((int)threadIdx.x % D4) * 4;
    if ((int)threadIdx.x >= ROWS * D4 || n >= ti.tile_rows * a.gh) return;
    const int n_splits = splits_of(ti, a.split_len);
    const size_t tstride = (size_t)a.n_tiles * NT;
    const size_t first_row = (size_t)sq.first_split * tstride + (size_t)tile * NT + blockIdx.x * ROWS;
    const unsigned row_at = threadIdx.x * 16u, ml_at = threadIdx.x / D4 * 8u;  // this thread's in a split's four rows and pairs
    const int tl = (n * a.gh_inv) >> 16;
    const int hh = ti.kvh * a.group + ti.hsub * a.gh + (n - tl * a.gh);
    const bool aligned = (a.flags & kHotAligned) != 0;
    const h4 gate4 = load_gate4(out, seq, ti.t0 + tl, hh, d, D);
    float mg = kNegBig, l = 0.0f;
    f4 acc = (f4)0.0f;
    auto turn = [&](auto splits, int first) {
        constexpr int SPLITS = decltype(splits)::value;
        // Places past the row's last split read as zeros: the descriptors end behind it.  (Any other row's values times a factor of zero
        // would do but for infinite ones, which become NaN; the host keeps 16 places of a launch within 4 GiB.)
        const size_t base = first_row + first * tstride;
        const unsigned there = min(n_splits - first, SPLITS) * (unsigned)tstride;
        const __amdgpu_buffer_rsrc_t rows = make_rsrc(a.part_o + base * D, there * (unsigned)(D * sizeof(float)));
        const __amdgpu_buffer_rsrc_t pairs = make_rsrc(a.part_ml + base * 2, there * (unsigned)(2 * sizeof(float)));
        unsigned row_next = row_at, ml_next = ml_at, stride = (unsigned)tstride;
        f2 pml[SPLITS];
        f4 po[SPLITS];
        // Requests in this order: six pairs and rows in turn, the other pairs, the other rows.  (16 ranges of 128 rows of 16/2 heads of 256, 33 MB: 7.4 us,
        // all in turn 7.9, all rows in front 8.2, all pairs 7.85.)
        constexpr int IN_TURN = SPLITS < 6 ? SPLITS : 6;
        auto ask_row = [&](int i) {
            po[i] = __builtin_bit_cast(f4, __builtin_amdgcn_raw_buffer_load_b128(rows, row_next, 0, 0));
            row_next += stride * (unsigned)(D * sizeof(float));
        };
#pragma unroll
        for (int i = 0; i < SPLITS; ++i) {
            pml[i] = __builtin_bit_cast(f2, __builtin_amdgcn_raw_buffer_load_b64(pairs, ml_next, 0, 0));
            asm volatile("" : "+s"(stride));  // (a place's offset is worked out here, not in front of all of them in a register of its own)
            ml_next += stride * (unsigned)sizeof(f2);
            if (i < IN_TURN) ask_row(i);
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int i = IN_TURN; i < SPLITS; ++i) {
            asm volatile("" : "+s"(stride));
            ask_row(i);
            __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_sched_barrier(0);  // (left alone, a request goes out when a row before it has come: fewer registers)
        float m_new = mg;
#pragma unroll
        for (int i = 0; i < SPLITS; ++i) m_new = fmaxf(m_new, first + i < n_splits ? pml[i][0] : kNegBig);
        const float keep = fast_exp2(mg - m_new);  // (first turn: what is kept is zero anyway)
        l *= keep;
        acc *= keep;
        mg = m_new;
#pragma unroll
        for (int i = 0; i < SPLITS; ++i) {
            const float f = first + i < n_splits ? fast_exp2(pml[i][0] - mg) : 0.0f;
            l += f * pml[i][1];
            acc += f * po[i];
        }
    };
    // (one turn up to kCombineRowsSplits splits, of four places where there are no more)
    if (n_splits <= 4) turn(std::integral_constant<int, 4>{}, 0);
    else
        for (int first = 0; first < n_splits; first += kCombineRowsSplits) turn(std::integral_constant<int, kCombineRowsSplits>{}, first);
    store_out4_gated(out, seq, ti.t0 + tl, hh, d, D, acc, l > 0.0f ? 1.0f / l : 0.0f, aligned, gate4);
}

// ---------------------------------------------------------------------------
// Host side: planning and launch.
// ---------------------------------------------------------------------------

// Behind the merge regions: the lists of touched blocks of a per-query selection, one per wave.
int plan_launch(const tt_hip_ctx *ctx, int kind, int n_seq, int n_q_heads, int n_kv_heads, int head_dim, int rows,
                long long total_keys, int min_keys, int max_keys, LaunchPlan *plan, int kv_bits, bool small_tiles_ok) {
    const int st = plan_splitk(ctx->n_cus, ctx->split_override, kind, n_seq, n_q_heads, n_kv_heads, head_dim, rows, total_keys, min_keys, max_keys,
                               plan, kv_bits, small_tiles_ok);
    if (st == TT_HIP_OK) plan->lds_bytes = lds_bytes_for(head_dim, plan->nt, plan->waves);
    return st;
}

template <int D, int NT, bool SINKS>
static int launch_combine_one(tt_hip_ctx *ctx, const LaunchPlan &plan, int n_seq, const SplitKArgs &args) {
    // Many tiles with few splits each: from 64 of its workgroups on (8 sequences' decode rows, 4 sequences' verify
    // rows; a verify pass of 8 x 4 rows at 65k keys 174.5 -> 170.1 us a step, 8 sequences x 8 rows at 4k keys 36.9 ->
    // 30.0 us; with 32 workgroups -- 4 sequences' decode rows -- the other kernel is ahead, 13.1 against 14.3 us).
    // (a turn's places are offsets of 32 bits)
    const bool near = (unsigned long long)plan.n_tiles * NT * D * sizeof(float) * kCombineRowsSplits <= 0xffffffffull;
    if (near && plan.n_splits_max <= 2 * kCombineRowsSplits && (long long)plan.n_tiles * n_seq * (NT / 4) >= 64) {
        dim3 cgrid((unsigned)(NT / 4), (unsigned)plan.n_tiles, (unsigned)n_seq);
        hipLaunchKernelGGL((attn_combine_rows_kernel<D, NT, SINKS>), cgrid, dim3(256), 0, ctx->stream, args);
    } else {
        // (a workgroup per row that a tile can have and 64 dims of it: tiles of 16 with 8 rows in use launch no idle half)
        const int tile_rows = args.hot.rows < plan.tt ? args.hot.rows : plan.tt;
        dim3 cgrid((unsigned)(tile_rows * plan.gh * (D / 64)), (unsigned)plan.n_tiles, (unsigned)n_seq);
        hipLaunchKernelGGL((attn_combine_kernel<D, NT, SINKS>), cgrid, dim3(256), 0, ctx->stream, args);
    }
    hipError_t e = hipGetLastError();
    return e == hipSuccess ? TT_HIP_OK : hip_fail(ctx, e, "attn_combine_kernel launch");
}

template <int D, int NT, int WAVES, int BITS, int KEEP = 0, int STREAM = 0>
static int launch_one(tt_hip_ctx *ctx, const LaunchPlan &plan, int n_seq, const SplitKArgs &args) {
    auto kernel = attn_splitk_kernel<D, NT, WAVES, BITS, KEEP, STREAM>;  // its LDS limit was raised when the context was created
    dim3 grid((unsigned)plan.n_splits_max, (unsigned)plan.n_tiles, (unsigned)n_seq);
    if (plan.packed_splits > 0) grid = dim3((unsigned)plan.packed_splits, (unsigned)plan.n_tiles);
    if (plan.xcd_grid) grid = dim3((unsigned)(((long long)plan.n_splits_max * plan.n_tiles + 7) / 8 * 8), 1u, (unsigned)n_seq);
    launch_profiled(ctx, kernel, grid, dim3(WAVES * 64), (unsigned)(plan.lds_bytes + keep_list_bytes(KEEP, WAVES)), args);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return hip_fail(ctx, e, "attn_splitk_kernel launch");
    if (plan.n_splits_max > 1 && !plan.partials_only && !ctx->pass_only) return launch_combine_one<D, NT, KEEP == kKeepSinks>(ctx, plan, n_seq, args);
    return TT_HIP_OK;
}


// Every instantiation's dynamic LDS limit (a compile-time constant of the kernel), set once per device when a
// context is created on it: no launch has to configure anything, so none is refused inside a graph capture
// and nothing is remembered outside the context.
template <int D, int NT, int BITS, int KEEP>
static hipError_t configure_one() {
    hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(attn_splitk_kernel<D, NT, 4, BITS, KEEP, 0>),
                                       hipFuncAttributeMaxDynamicSharedMemorySize,
                                       (int)std::max(lds_bytes_for(D, NT, 4) + keep_list_bytes(KEEP, 4), KEEP == kKeepRows ? front_lds_bytes(D) : 0));
    if constexpr (D == 256 && NT == 32 && BITS == 16 && KEEP == 0) {
        if (e == hipSuccess)
            e = hipFuncSetAttribute(reinterpret_cast<const void *>(attn_splitk_kernel<D, NT, 4, BITS, KEEP, 2>),
                                    hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds_bytes_for(D, NT, 4));
    }
    if constexpr (KEEP < 2 || KEEP == kKeepSinks) {  // (a chunk's per-query selections come with many token tiles: never streamed)
        if (e == hipSuccess)
            e = hipFuncSetAttribute(reinterpret_cast<const void *>(attn_splitk_kernel<D, NT, 4, BITS, KEEP, 1>),
                                    hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds_bytes_for(D, NT, 4));
    }
    return e;
}
template <int D, int NT>
static hipError_t configure_tile() {
    hipError_t e = hipSuccess;
#define TT_CFG(BB, KK) \
    if (e == hipSuccess) e = configure_one<D, NT, BB, KK>();
    TT_CFG(16, 0) TT_CFG(8, 0) TT_CFG(4, 0)
    TT_CFG(16, 1) TT_CFG(8, 1) TT_CFG(4, 1)
    TT_CFG(16, 2) TT_CFG(8, 2) TT_CFG(4, 2)
    if constexpr (D != 256) { TT_CFG(16, 3) }  // (heads of 256: by key always)
    TT_CFG(8, 3) TT_CFG(4, 3)
    if constexpr (NT == 32) { TT_CFG(16, 4) }
    if constexpr (lists_fetch_by_key(D, 16)) { TT_CFG(16, 5) }
    TT_CFG(16, kKeepSinks) TT_CFG(8, kKeepSinks) TT_CFG(4, kKeepSinks)
    TT_CFG(16, kKeepPieces) TT_CFG(8, kKeepPieces) TT_CFG(4, kKeepPieces)
    TT_CFG(16, kKeepRows) TT_CFG(8, kKeepRows) TT_CFG(4, kKeepRows)
#undef TT_CFG
    return e;
}
int configure_splitk_kernels(tt_hip_ctx *ctx) {
    hipError_t e = configure_tile<256, 16>();
    if (e == hipSuccess) e = configure_tile<256, 32>();
    if (e == hipSuccess) e = configure_tile<128, 16>();
    if (e == hipSuccess) e = configure_tile<128, 32>();
    if (e == hipSuccess) e = configure_tile<64, 16>();
    if (e == hipSuccess) e = configure_tile<64, 32>();
    return e == hipSuccess ? TT_HIP_OK : hip_fail(ctx, e, "hipFuncSetAttribute(split-K max dynamic LDS)");
}

// The combine pass on its own: for partials written by another kernel in this kernel's layout.
int launch_combine(tt_hip_ctx *ctx, const LaunchPlan &plan, int head_dim, int n_seq, const SplitKArgs &args) {
    if (plan.n_tiles > 65535 || n_seq > 65535) return TT_HIP_ERR_SHAPE;
    const bool sinks = (args.hot.flags & kHotSinks) != 0;
#define TT_CASE(DD, NN)              \
    if (head_dim == DD && plan.nt == NN) \
        return sinks ? launch_combine_one<DD, NN, true>(ctx, plan, n_seq, args) : launch_combine_one<DD, NN, false>(ctx, plan, n_seq, args);
    TT_CASE(256, 16)
    TT_CASE(256, 32)
    TT_CASE(128, 16)
    TT_CASE(128, 32)
    TT_CASE(64, 16)
    TT_CASE(64, 32)
#undef TT_CASE
    return TT_HIP_ERR_SHAPE;
}

int launch_splitk_pair(tt_hip_ctx *ctx, int head_dim, int nt, int kv_bits, bool packed_rows, unsigned groups, const SplitKPair &args) {
    auto launch = [&](auto kernel) {
        const size_t lds = std::max(lds_bytes_for(head_dim, nt, 4), packed_rows ? front_lds_bytes(head_dim) : 0);
        launch_profiled(ctx, kernel, dim3(groups), dim3(256), (unsigned)lds, args);
        const hipError_t e = hipGetLastError();
        return e == hipSuccess ? (int)TT_HIP_OK : hip_fail(ctx, e, "attn_splitk_kernel launch");
    };
#define TT_CASE(DD, NN)                                                                  \
    if (head_dim == DD && nt == NN && packed_rows) {                                     \
        if (kv_bits == 16) return launch(attn_splitk_kernel<DD, NN, 4, 16, kKeepRows>);  \
        if (kv_bits == 8) return launch(attn_splitk_kernel<DD, NN, 4, 8, kKeepRows>);    \
        if (kv_bits == 4) return launch(attn_splitk_kernel<DD, NN, 4, 4, kKeepRows>);    \
    }                                                                                    \
    if (head_dim == DD && nt == NN) {                                                    \
        if (kv_bits == 16) return launch(attn_splitk_kernel<DD, NN, 4, 16, kKeepPieces>); \
        if (kv_bits == 8) return launch(attn_splitk_kernel<DD, NN, 4, 8, kKeepPieces>);   \
        if (kv_bits == 4) return launch(attn_splitk_kernel<DD, NN, 4, 4, kKeepPieces>);   \
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

int launch_splitk(tt_hip_ctx *ctx, const LaunchPlan &plan, int head_dim, int n_seq, const SplitKArgs &args, int kv_bits) {
    if (n_seq > kMaxSeqPerLaunch || plan.waves != 4) return TT_HIP_ERR_INVALID_ARGUMENT;
    if (plan.n_tiles > 65535 || n_seq > 65535) return TT_HIP_ERR_SHAPE;
#define TT_CASE(DD, NN)                                                                              \
    if (head_dim == DD && plan.nt == NN) {                                                           \
        if constexpr (NN == 32) {                                                                    \
            if (args.plan_blocks && args.plan_groups) return launch_one<DD, NN, 4, 16, 4>(ctx, plan, n_seq, args); \
        }                                                                                            \
        if constexpr (lists_fetch_by_key(DD, 16)) {                                                  \
            if (args.plan_blocks && args.plan_by_key) return launch_one<DD, NN, 4, 16, 5>(ctx, plan, n_seq, args); \
        }                                                                                            \
        if (args.plan_blocks) {                                                                      \
            if constexpr (DD != 256) {                                                               \
                if (kv_bits == 16) return launch_one<DD, NN, 4, 16, 3>(ctx, plan, n_seq, args);      \
            }                                                                                        \
            if (kv_bits == 8) return launch_one<DD, NN, 4, 8, 3>(ctx, plan, n_seq, args);            \
            if (kv_bits == 4) return launch_one<DD, NN, 4, 4, 3>(ctx, plan, n_seq, args);            \
        }                                                                                            \
        if (args.keep && args.keep_row_stride > 0) {                                                 \
            if (kv_bits == 16) return launch_one<DD, NN, 4, 16, 2>(ctx, plan, n_seq, args);          \
            if (kv_bits == 8) return launch_one<DD, NN, 4, 8, 2>(ctx, plan, n_seq, args);            \
            if (kv_bits == 4) return launch_one<DD, NN, 4, 4, 2>(ctx, plan, n_seq, args);            \
        }                                                                                            \
        if (args.keep && plan.stream) {                                                              \
            if (kv_bits == 16) return launch_one<DD, NN, 4, 16, 1, 1>(ctx, plan, n_seq, args);       \
            if (kv_bits == 8) return launch_one<DD, NN, 4, 8, 1, 1>(ctx, plan, n_seq, args);         \
            if (kv_bits == 4) return launch_one<DD, NN, 4, 4, 1, 1>(ctx, plan, n_seq, args);         \
        }                                                                                            \
        if (args.keep) {                                                                             \
            if (kv_bits == 16) return launch_one<DD, NN, 4, 16, 1>(ctx, plan, n_seq, args);          \
            if (kv_bits == 8) return launch_one<DD, NN, 4, 8, 1>(ctx, plan, n_seq, args);            \
            if (kv_bits == 4) return launch_one<DD, NN, 4, 4, 1>(ctx, plan, n_seq, args);            \
        }                                                                                            \
        if ((args.hot.flags & kHotSinks) && plan.stream) {                                           \
            if (kv_bits == 16) return launch_one<DD, NN, 4, 16, kKeepSinks, 1>(ctx, plan, n_seq, args); \
            if (kv_bits == 8) return launch_one<DD, NN, 4, 8, kKeepSinks, 1>(ctx, plan, n_seq, args); \
            if (kv_bits == 4) return launch_one<DD, NN, 4, 4, kKeepSinks, 1>(ctx, plan, n_seq, args); \
        }                                                                                            \
        if (args.hot.flags & kHotSinks) {                                                            \
            if (kv_bits == 16) return launch_one<DD, NN, 4, 16, kKeepSinks>(ctx, plan, n_seq, args); \
            if (kv_bits == 8) return launch_one<DD, NN, 4, 8, kKeepSinks>(ctx, plan, n_seq, args);   \
            if (kv_bits == 4) return launch_one<DD, NN, 4, 4, kKeepSinks>(ctx, plan, n_seq, args);   \
        }                                                                                            \
        if (plan.stream) {                                                                           \
            if constexpr (DD == 256 && NN == 32) {                                                   \
                if (kv_bits == 16 && plan.paired) return launch_one<DD, NN, 4, 16, 0, 2>(ctx, plan, n_seq, args); \
            }                                                                                        \
            if (kv_bits == 16) return launch_one<DD, NN, 4, 16, 0, 1>(ctx, plan, n_seq, args);       \
            if (kv_bits == 8) return launch_one<DD, NN, 4, 8, 0, 1>(ctx, plan, n_seq, args);         \
            if (kv_bits == 4) return launch_one<DD, NN, 4, 4, 0, 1>(ctx, plan, n_seq, args);         \
        }                                                                                            \
        if (kv_bits == 16) return launch_one<DD, NN, 4, 16>(ctx, plan, n_seq, args);                 \
        if (kv_bits == 8) return launch_one<DD, NN, 4, 8>(ctx, plan, n_seq, args);                   \
        if (kv_bits == 4) return launch_one<DD, NN, 4, 4>(ctx, plan, n_seq, args);                   \
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

}  // namespace tt
