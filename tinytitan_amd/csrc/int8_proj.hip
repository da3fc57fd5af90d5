// Products of 8-bit integers: y[t][r] = fp16(token_scale[t] * weight_scale[r] * sum_k weight[r][k] * level[t][k]), the sum exact in
// 32-bit integers, over tokens quantised one by one:
//   token_scale = max |x| / 127,  level = round(x / token_scale)     (ties to even; both divisions as fp32 rounds them)
// A token of zeros has scale and levels zero.  A token with an infinite or NaN element has a NaN for a scale and zero levels: its
// outputs are NaN, other tokens' are their own.
#include <algorithm>
#include <type_traits>

#include "int8_plan.h"
#include "internal.h"
#include "lds_copy.h"
#include "wave_ops.h"

namespace tt {

namespace {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef float f4 __attribute__((ext_vector_type(4)));
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
// Eight halves as levels, round(x / scale); `scale` 0 or NaN: zeros.  The division by its reciprocal, rounded to nearest, with one correction
// of the quotient's remainder, which gives the division's own bits (Markstein's theorem; nothing here overflows or is subnormal).
struct Divisor {
    float scale, inverse;
    __device__ __forceinline__ explicit Divisor(float s) : scale(s > 0.0f ? s : 1.0f), inverse(s > 0.0f ? 1.0f / s : 0.0f) {}
};
__device__ __forceinline__ u2 levels_of(const u4 &x, const Divisor &by) {
    u2 out = {0u, 0u};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float v = half_of_bits((x[i >> 1] >> (16 * (i & 1))) & 0xffffu);
        const float q = v * by.inverse;
        const int level = (int)__builtin_rintf(__builtin_fmaf(__builtin_fmaf(-q, by.scale, v), by.inverse, q));
        out[i >> 2] |= ((unsigned)level & 0xffu) << (8 * (i & 3));
    }
    return out;
}
__device__ __forceinline__ unsigned largest_of_wave(unsigned x) {
#pragma unroll
    for (int step = 32; step > 0; step /= 2) x = max(x, (unsigned)__shfl_xor((int)x, step));
    return x;
}

// A workgroup per token, whose pieces of eight stay in registers between the search for the largest and the division: up to HELD a thread,
// 2,048 HELD columns; what lies behind those is read twice.
template <int HELD>
__global__ __launch_bounds__(256) void quantise_rows_kernel(const _Float16 *x, long long x_stride, int columns, int8_t *levels, long long levels_stride,
                                                            float *scales) {
    __shared__ unsigned found[4];
    const long long token = blockIdx.x;
    const u4 *const row = reinterpret_cast<const u4 *>(x + token * x_stride);
    const int pieces = columns / 8;
    u4 held[HELD];
    unsigned largest = 0;
#pragma unroll
    for (int i = 0; i < HELD; ++i) held[i] = row[min(i * 256 + (int)threadIdx.x, pieces - 1)];
    for (int i = HELD * 256 + threadIdx.x; i < pieces; i += 256) largest = largest_bits(largest, row[i]);
#pragma unroll
    for (int i = 0; i < HELD; ++i) largest = largest_bits(largest, held[i]);
    largest = largest_of_wave(largest);
    if ((threadIdx.x & 63) == 0) found[threadIdx.x >> 6] = largest;
    __syncthreads();
    const float scale = token_scale(max(max(found[0], found[1]), max(found[2], found[3])));
    const Divisor by(scale);
    u2 *const to = reinterpret_cast<u2 *>(levels + token * levels_stride);
#pragma unroll
    for (int i = 0; i < HELD; ++i)
        if (i * 256 + (int)threadIdx.x < pieces) to[i * 256 + threadIdx.x] = levels_of(held[i], by);
    for (int i = HELD * 256 + threadIdx.x; i < pieces; i += 256) to[i] = levels_of(row[i], by);
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

// ---- few tokens ----------------------------------------------------------------------------------------------------------------
//
// What the weights' bytes take to read: each is read once.  A workgroup is 16 RT channels and up to 16 NT tokens; of K, in stages of
// 128 columns, every wavefront takes its own and keeps a ring of DEPTH of them in LDS, its own too, so that no wavefront waits for another
// before the end, when their sums, exact in any order, meet.  Rows come by whole lines, eight of them a copy straight into LDS, in the order that
// the many tokens' kernel has them in: a load of v_mfma_i32_16x16x64_i8's operands from memory takes sixteen rows in pieces of 16 bytes that
// the vector memory path handles one by one, a quarter of its rate (one token, 9,216 x 2,048: 11.8 us so).
// Tokens' rows go the same way, or, FUSED, are quantised into LDS by the workgroup itself beside its first weights' way (up to four
// tokens, a wavefront each or more, whose halves and levels lie in LDS behind the rings).
constexpr int kStageBytes = 128;
constexpr int kFusedTokens = 4;
// Tokens that a workgroup shares its wavefronts out to: a power of two.
__host__ __device__ constexpr int fused_tokens(int tokens) { return tokens <= 1 ? 1 : tokens <= 2 ? 2 : 4; }

template <int RT, int NT, int WAVES, int DEPTH, bool FUSED>
__global__ __launch_bounds__(WAVES * 64) void int8_ring_kernel(const ProductArgs a, const _Float16 *halves, long long halves_stride) {
    constexpr int ROWS = 16 * RT + (FUSED ? 0 : 16 * NT), COPIES = ROWS / 8, STAGE = ROWS * kStageBytes;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), li = lane & 15, g = lane >> 4;
    const int row0 = blockIdx.x * 16 * RT;
    const int stages = (a.columns + kStageBytes - 1) / kStageBytes, mine = (stages - wave + WAVES - 1) / WAVES;  // stages wave, wave + WAVES, ...
    // Copies: eight rows' lines each, piece c of row r at place c ^ (r % 8); rows past the end are the last one again, pieces past a row's
    // end its last stage's first one.
    const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) void *)smem;
    const int in_copy = lane >> 3, piece = 16 * ((lane & 7) ^ in_copy);
    unsigned from[COPIES];
#pragma unroll
    for (int c = 0; c < COPIES; ++c) {
        const int r = 8 * c + in_copy;
        from[c] = c < 2 * RT ? (unsigned)min(r, a.rows - 1 - row0) * (unsigned)a.columns + (unsigned)piece
                             : (unsigned)min(r - 16 * RT, a.tokens - 1) * (unsigned)a.levels_stride + (unsigned)piece;
    }
    const int8_t *const w = a.weights + (long long)row0 * a.columns;
    char *const ring = smem + wave * (DEPTH * STAGE);
    __shared__ float token_scales[kFusedTokens];
    auto copy_stage = [&](int i) {  // the wavefront's i-th
        const int s = wave + i * WAVES;
        const unsigned back = s * kStageBytes + piece < a.columns ? 0u : (unsigned)piece;
        const unsigned to = lds0 + (unsigned)(wave * DEPTH + i % DEPTH) * STAGE;
#pragma unroll
        for (int c = 0; c < COPIES; ++c) copy16_global_to_lds((c < 2 * RT ? w : a.levels) + (size_t)s * kStageBytes, from[c] - back, to + c * 1024u);
    };
    // FUSED: behind the rings the tokens' levels, `pitch` bytes from one to the next, and behind those the wavefronts' shares of the tokens
    // as they come.  A token is `share` wavefronts', whose pieces go straight to LDS in front of the first weights: asked for behind them, or
    // waited for as the compiler would, they were there when those were (one token, 2,048 x 4,096: 6.8 us).
    const int pitch = a.columns + 16;
    char *const levels = smem + WAVES * DEPTH * STAGE;
    if constexpr (FUSED) {
        __shared__ unsigned found[WAVES];
        const int share = WAVES / fused_tokens(a.tokens), token = wave / share, part = wave - token * share, pieces = a.columns / 8;
        const int held = (pieces + 64 * share - 1) / (64 * share);  // a lane's pieces
        const unsigned raw = (unsigned)(WAVES * DEPTH * STAGE + a.tokens * pitch + wave * held * 1024);
        const _Float16 *const row = halves + min(token, a.tokens - 1) * halves_stride;
        for (int i = 0; i < held; ++i)
            copy16_global_to_lds(row, (unsigned)min((i * share + part) * 64 + lane, pieces - 1) * 16u, lds0 + raw + (unsigned)i * 1024u);
        const int ahead = min(DEPTH - 1, mine);
        for (int i = 0; i < ahead; ++i) copy_stage(i);
        if (ahead == DEPTH - 1) TT_WAIT_VMCNT((DEPTH - 1) * COPIES);
        else TT_WAIT_VMCNT(0);
        asm volatile("" ::: "memory");
        const u4 *const mine_raw = reinterpret_cast<const u4 *>(smem + raw) + lane;
        unsigned largest = 0;
        for (int i = 0; i < held; ++i) largest = largest_bits(largest, mine_raw[i * 64]);
        largest = largest_of_wave(largest);
        if (lane == 0) found[wave] = largest;
        __syncthreads();
        if (token < a.tokens) {
            for (int i = 0; i < share; ++i) largest = max(largest, found[token * share + i]);
            const float scale = token_scale(largest);
            const Divisor by(scale);
            for (int i = 0; i < held; ++i) {
                const int at = (i * share + part) * 64 + lane;
                if (at < pieces) *reinterpret_cast<u2 *>(levels + token * pitch + at * 8) = levels_of(mine_raw[i * 64], by);
            }
            if (part == 0 && lane == 0) token_scales[token] = scale;
        }
        __syncthreads();
    } else {
        for (int i = 0; i < min(DEPTH - 1, mine); ++i) copy_stage(i);
    }
    const char *const my_levels = levels + min(li, a.tokens - 1) * pitch;

    i4 acc[RT][NT];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[r][n] = (i4)0;
    const int line = li * kStageBytes;
    for (int i = 0; i < mine; ++i) {
        // (the place of the stage before this one, whose products are done, takes the copies of the one DEPTH - 1 ahead)
        if (i + DEPTH - 1 < mine) {
            copy_stage(i + DEPTH - 1);
            TT_WAIT_VMCNT((DEPTH - 1) * COPIES);
        } else {
            TT_WAIT_VMCNT(0);
        }
        asm volatile("" ::: "memory");
        const char *const stage = ring + (i % DEPTH) * STAGE;
        const int k0 = (wave + i * WAVES) * kStageBytes + 16 * g;
#pragma unroll
        for (int step = 0; step < 2; ++step) {
            const int at = ((4 * step + g) ^ (li & 7)) * 16, k = k0 + 64 * step;
            const bool real = k < a.columns;  // (past the end: whatever lies there times levels of zero)
            i4 wf[RT], xf[NT];
#pragma unroll
            for (int r = 0; r < RT; ++r) wf[r] = *reinterpret_cast<const i4 *>(stage + 16 * r * kStageBytes + line + at);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                if constexpr (FUSED) xf[n] = *reinterpret_cast<const i4 *>(my_levels + (real ? k : 0));
                else xf[n] = *reinterpret_cast<const i4 *>(stage + 16 * (RT + n) * kStageBytes + line + at);
                xf[n] = real ? xf[n] : (i4)0;
            }
#pragma unroll
            for (int r = 0; r < RT; ++r)
#pragma unroll
                for (int n = 0; n < NT; ++n) acc[r][n] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[r], xf[n], acc[r][n], 0, 0, 0);
        }
    }
    __syncthreads();  // (the rings' place is the sums')
    // [row tile][token tile][wavefront][lane][4 channels]
    i4 *const sums = reinterpret_cast<i4 *>(smem);
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int n = 0; n < NT; ++n) sums[((r * NT + n) * WAVES + wave) * 64 + lane] = acc[r][n];
    __syncthreads();
    for (int at = threadIdx.x; at < RT * NT * 64; at += WAVES * 64) {
        const int tile = at >> 6, r = tile / NT, n = tile - r * NT, l = at & 63;
        i4 sum = (i4)0;
#pragma unroll
        for (int v = 0; v < WAVES; ++v) sum += sums[(tile * WAVES + v) * 64 + l];
        const int token = 16 * n + (l & 15), row = row0 + 16 * r + 4 * (l >> 4);
        if (token >= a.tokens) continue;
        const float scale = FUSED ? token_scales[token] : a.scales[token];
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (row + e < a.rows) a.y[token * a.y_stride + row + e] = (_Float16)((float)sum[e] * a.weight_scales[row + e] * scale);
    }
}

constexpr size_t kMostLds = 160 * 1024 - 512;  // (less than the chip's, for what the kernels hold besides)
template <int RT, int NT, int WAVES, int DEPTH, bool FUSED>
size_t ring_lds_bytes(int tokens, int columns) {
    const size_t rings = (size_t)WAVES * DEPTH * (16 * RT + (FUSED ? 0 : 16 * NT)) * kStageBytes;
    const size_t per_pass = 64 * 8 * (size_t)(WAVES / fused_tokens(tokens)), raw = (columns + per_pass - 1) / per_pass * WAVES * 1024;
    return std::max<size_t>((size_t)RT * NT * WAVES * 1024, rings + (FUSED ? (size_t)tokens * (columns + 16) + raw : 0));
}
template <int RT, int NT, int WAVES, int DEPTH, bool FUSED>
hipError_t configure_ring() {
    return hipFuncSetAttribute(reinterpret_cast<const void *>(int8_ring_kernel<RT, NT, WAVES, DEPTH, FUSED>), hipFuncAttributeMaxDynamicSharedMemorySize,
                               (int)(FUSED ? kMostLds : ring_lds_bytes<RT, NT, WAVES, DEPTH, false>(1, 16)));
}
template <int RT, int NT, int WAVES, int DEPTH, bool FUSED>
void launch_ring(tt_hip_ctx *ctx, const ProductArgs &a, const _Float16 *halves = nullptr, long long halves_stride = 0) {
    static_assert(WAVES >= kFusedTokens && (DEPTH - 1) * (2 * RT + (FUSED ? 0 : 2 * NT)) <= 63, "a wavefront a token at least; what vmcnt counts to");
    launch_profiled(ctx, int8_ring_kernel<RT, NT, WAVES, DEPTH, FUSED>, dim3((unsigned)((a.rows + 16 * RT - 1) / (16 * RT))), dim3(WAVES * 64),
                    (unsigned)ring_lds_bytes<RT, NT, WAVES, DEPTH, FUSED>(a.tokens, a.columns), a, halves, halves_stride);
}

// ---- many tokens ---------------------------------------------------------------------------------------------------------------
//
// A workgroup's TM channels x TN tokens, four wavefronts of TM / 2 x TN / 2 each, v_mfma_i32_32x32x32_i8.  K goes by stages of 128: a
// row's 128 bytes are one line, copied into LDS as they are but for the order of their 16-byte pieces, piece c of row r at place
// c ^ (r % 8), so that the 32 rows of an operand read lie in all banks.  The copies go straight to LDS; BUFFERS stages of them.
//
// One barrier a stage, in front of the matrix products of its last step: every wavefront then holds the stage's last operands in registers, so
// that the stage's place may be filled again, and the next stage has landed, so that its first operands are read beside those
// products -- the matrix pipe never waits for a stage to begin.
template <int TM, int TN, int BUFFERS>
__global__ __launch_bounds__(256, 1) void int8_gemm_kernel(const ProductArgs a, int m_tiles, int n_tiles, int per_xcd) {
    constexpr int MT = TM / 64, NT = TN / 64;      // 32 x 32 tiles of a wavefront
    constexpr int COPIES = (TM + TN) / 32;         // of 1 KiB (eight rows) that a wavefront issues a stage
    constexpr int BUFFER = (TM + TN) * kStageBytes;
    constexpr int STEPS = kStageBytes / 32;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), li = lane & 31, g = lane >> 5;

    // Workgroup b runs on XCD b % 8: every XCD takes a run of the tiles, in groups of eight tiles of channels that go through the
    // tokens together, so that what its workgroups read side by side is in its L2 for several of them.
    const int at = (int)(blockIdx.x & 7) * per_xcd + (int)(blockIdx.x >> 3);
    if (at >= m_tiles * n_tiles) return;
    const int group = at / (8 * n_tiles), in_group = at - group * 8 * n_tiles, group_m = min(m_tiles - group * 8, 8);
    const int n_tile = in_group / group_m, m_tile = group * 8 + in_group - n_tile * group_m;
    const int row0 = m_tile * TM, token0 = n_tile * TN;

    // This wavefront's copies: those of channels first, then those of tokens; rows past the end are the last one again.
    const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) void *)smem;
    const int in_copy = lane >> 3, piece = 16 * ((lane & 7) ^ in_copy);
    unsigned from[COPIES];
#pragma unroll
    for (int c = 0; c < COPIES; ++c) {
        const int r = (c * 4 + wave) * 8 + in_copy;
        from[c] = c * 32 < TM ? (unsigned)min(r, a.rows - 1 - row0) * (unsigned)a.columns + (unsigned)piece
                              : (unsigned)min(r - TM, a.tokens - 1 - token0) * (unsigned)a.levels_stride + (unsigned)piece;
    }
    const int8_t *w = a.weights + (long long)row0 * a.columns, *x = a.levels + (long long)token0 * a.levels_stride;
    const int stages = (a.columns + kStageBytes - 1) / kStageBytes;
    // Copies of stage s (its place: buffer s % BUFFERS).  Of a row's last stage the pieces behind its end are its first piece again.
    auto copy = [&](int c, int s, unsigned to) {
        const unsigned back = s * kStageBytes + piece < a.columns ? 0u : (unsigned)piece;
        copy16_global_to_lds((c * 32 < TM ? w : x) + (size_t)s * kStageBytes, from[c] - back, to + (unsigned)(c * 4 + wave) * 1024u);
    };

    i4 wf[2][MT], xf[2][NT];
    i16v acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = (i16v)0;
    // Operands of a step: 16 bytes of a row each, its piece 2 step + g.
    const int w_at = ((wave >> 1) * (TM / 2) + li) * kStageBytes, x_at = (TM + (wave & 1) * (TN / 2) + li) * kStageBytes;
    int in_row[STEPS];
#pragma unroll
    for (int step = 0; step < STEPS; ++step) in_row[step] = ((2 * step + g) ^ (li & 7)) * 16;
    auto read = [&](int into, int buffer, int step, int i) {  // the i-th of them
        if (i < MT) wf[into][i < MT ? i : 0] = *reinterpret_cast<const i4 *>(smem + (buffer * BUFFER + w_at + in_row[step]) + 32 * i * kStageBytes);
        else xf[into][i < MT ? 0 : i - MT] = *reinterpret_cast<const i4 *>(smem + (buffer * BUFFER + x_at + in_row[step]) + 32 * (i - MT) * kStageBytes);
    };
    // Stage s, out of `buffer`: a copy or an operand of the next step behind every product, in that order.  What is copied past the last stage is
    // that again, into a place that nobody reads, so that one count of copies on their way holds for every stage.
    auto run_stage = [&](auto last_one, int s, int buffer) {
        constexpr bool LAST = decltype(last_one)::value;
        const int next = buffer + 1 == BUFFERS ? 0 : buffer + 1, ahead = buffer == 0 ? BUFFERS - 1 : buffer - 1;
        const int copied = min(s + BUFFERS - 1, stages - 1);
        const unsigned to = lds0 + (unsigned)ahead * BUFFER;
#pragma unroll
        for (int step = 0; step < STEPS; ++step) {
            constexpr int PRODUCTS = MT * NT, SPREAD = (STEPS - 1) * PRODUCTS;
            if (step + 1 == STEPS && !LAST) {
                TT_WAIT_VMCNT((BUFFERS - 2) * COPIES);  // (the next stage's have landed)
                __syncthreads();
            }
            if constexpr (LAST) {  // the columns behind the row's end: levels of zero, whatever the weights' place holds
                const int k = s * kStageBytes + 32 * step + 16 * g;
#pragma unroll
                for (int j = 0; j < NT; ++j) xf[step & 1][j] = k < a.columns ? xf[step & 1][j] : (i4)0;
            }
#pragma unroll
            for (int u = 0; u < PRODUCTS; ++u) {
                const int i = u / NT, j = u % NT;
                acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(wf[step & 1][i], xf[step & 1][j], acc[i][j], 0, 0, 0);
#pragma unroll
                for (int r = 0; r < MT + NT; ++r) {
                    if (r * PRODUCTS / (MT + NT) / (PRODUCTS >= 8 ? 2 : 1) != u) continue;
                    if (step + 1 < STEPS) read((step + 1) & 1, buffer, step + 1, r);
                    else if (!LAST) read(0, next, 0, r);
                }
                if (!LAST && step + 1 < STEPS) {
#pragma unroll
                    for (int c = 0; c < COPIES; ++c)
                        if (c * SPREAD / COPIES == step * PRODUCTS + u) copy(c, copied, to);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    };

    static_assert(BUFFERS >= 2 && STEPS % 2 == 0);
#pragma unroll
    for (int s = 0; s < BUFFERS - 1; ++s)
#pragma unroll
        for (int c = 0; c < COPIES; ++c) copy(c, min(s, stages - 1), lds0 + (unsigned)s * BUFFER);
    TT_WAIT_VMCNT((BUFFERS - 2) * COPIES);
    __syncthreads();
#pragma unroll
    for (int r = 0; r < MT + NT; ++r) read(0, 0, 0, r);
    int buffer = 0;
#pragma nounroll
    for (int s = 0; s + 1 < stages; ++s) {
        run_stage(std::false_type{}, s, buffer);
        buffer = buffer + 1 == BUFFERS ? 0 : buffer + 1;
    }
    run_stage(std::true_type{}, stages - 1, buffer);
    TT_WAIT_VMCNT(0);
    __syncthreads();

    // The rows go out through LDS, 32 tokens x TM / 2 channels at a time, a place of its own for every wavefront: a store is 16 bytes a lane of
    // consecutive channels.
    constexpr int PITCH = TM / 2 * 2 + 16, LANES = TM / 2 / 8, ROWS = 64 / LANES;  // bytes; lanes of a token, tokens of a store
    float *const channel_scales = reinterpret_cast<float *>(smem + 4 * 32 * PITCH);
    if (threadIdx.x < TM) channel_scales[threadIdx.x] = a.weight_scales[min(row0 + (int)threadIdx.x, a.rows - 1)];
    __syncthreads();
    char *const stage = smem + wave * 32 * PITCH;
    const int wave_row0 = row0 + (wave >> 1) * (TM / 2), wave_token0 = token0 + (wave & 1) * (TN / 2);
    const bool whole = (a.y_stride % 8 == 0) && (reinterpret_cast<size_t>(a.y) & 15) == 0;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const int token = wave_token0 + 32 * j + li;
        const float scale = a.scales[min(token, a.tokens - 1)];
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int v = 0; v < 16; v += 4) {
                const int r = 32 * i + 8 * (v >> 2) + 4 * g;
                const f4 channel = *reinterpret_cast<const f4 *>(channel_scales + (wave >> 1) * (TM / 2) + r);
                h4 out;
#pragma unroll
                for (int e = 0; e < 4; ++e) out[e] = (_Float16)((float)acc[i][j][v + e] * channel[e] * scale);
                *reinterpret_cast<h4 *>(stage + li * PITCH + r * 2) = out;
            }
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int t = 0; t < 32; t += ROWS) {
            const int row = t + lane / LANES, first = (lane % LANES) * 8, to_token = wave_token0 + 32 * j + row, r = wave_row0 + first;
            const h8 out = *reinterpret_cast<const h8 *>(stage + row * PITCH + first * 2);
            if (to_token < a.tokens) {
                _Float16 *const to = a.y + to_token * a.y_stride + r;
                if (whole && r + 8 <= a.rows) {
                    *reinterpret_cast<h8 *>(to) = out;
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (r + e < a.rows) to[e] = out[e];
                }
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
}

template <int TM, int TN, int BUFFERS>
constexpr size_t gemm_lds_bytes() {
    return std::max<size_t>((size_t)BUFFERS * (TM + TN) * kStageBytes, (size_t)4 * 32 * (TM + 16) + TM * sizeof(float));
}
template <int TM, int TN, int BUFFERS>
hipError_t configure_gemm() {
    return hipFuncSetAttribute(reinterpret_cast<const void *>(int8_gemm_kernel<TM, TN, BUFFERS>), hipFuncAttributeMaxDynamicSharedMemorySize,
                               (int)gemm_lds_bytes<TM, TN, BUFFERS>());
}
template <int TM, int TN, int BUFFERS>
void launch_gemm(tt_hip_ctx *ctx, const ProductArgs &a) {
    const int m_tiles = (a.rows + TM - 1) / TM, n_tiles = (a.tokens + TN - 1) / TN;
    const int per_xcd = (int)(((long long)m_tiles * n_tiles + 7) / 8);
    launch_profiled(ctx, int8_gemm_kernel<TM, TN, BUFFERS>, dim3((unsigned)per_xcd * 8u), dim3(256), (unsigned)gemm_lds_bytes<TM, TN, BUFFERS>(), a, m_tiles,
                    n_tiles, per_xcd);
}

// The smallest tiles: the four wavefronts take a stage's four steps of 32 columns, one each, of the WHOLE tile, and add up their sums (exact in
// integers, in any order) at the end.  A stage's operands then leave LDS once, not for two wavefronts each, and there is a barrier for four times the
// products.  Every wavefront owns OWN tiles of 32 x 32 behind each other in channels, whose sums of the other three it adds to its own.  Two workgroups fit
// a CU with four buffers.  us, tiles of 64 x 64 with TM / 2 x TN / 2 a wavefront / these: 512 tokens 2,048 x 4,096 11.6 / 9.8, 333 2,048 x 2,048 7.4 / 6.5,
// 100 2,048 x 2,048 6.9 / 6.1, 300 300 x 8,192 18.2 / 15.1, 70 6,144 x 5,120 13.6 / 12.3.  Of 128 x 64 they are even (777 tokens, 2,311 x 4,096 19.4 / 18.8, 200
// 5,120 x 5,120 16.6 / 18.3 the other way): there the copies' way from the L2s bounds both, 12 TB/s.
template <int TM, int TN, int BUFFERS>
struct StepsShape {
    static constexpr int MT = TM / 32, NT = TN / 32, OWN = MT * NT / 4, BUFFER = (TM + TN) * kStageBytes;
    static constexpr int PITCH = OWN * 32 * 2 + 16, STAGING = 4 * 32 * PITCH;
    static constexpr size_t LDS = std::max<size_t>({(size_t)BUFFERS * BUFFER, (size_t)12 * OWN * 4096, (size_t)STAGING + TM * sizeof(float)});
    static_assert(OWN >= 1 && NT <= 4 && 4 % NT == 0 && MT % OWN == 0);
};
template <int TM, int TN, int BUFFERS>
__global__ __launch_bounds__(256, 1) void int8_steps_kernel(const ProductArgs a, int m_tiles, int n_tiles, int per_xcd) {
    typedef StepsShape<TM, TN, BUFFERS> C;
    constexpr int MT = C::MT, NT = C::NT, OWN = C::OWN, BUFFER = C::BUFFER;
    constexpr int COPIES = (TM + TN) / 32;  // of 1 KiB (eight rows) that a wavefront issues a stage
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), li = lane & 31, g = lane >> 5;

    // (workgroups, copies and the order of a line's pieces as above)
    const int at = (int)(blockIdx.x & 7) * per_xcd + (int)(blockIdx.x >> 3);
    if (at >= m_tiles * n_tiles) return;
    const int group = at / (8 * n_tiles), in_group = at - group * 8 * n_tiles, group_m = min(m_tiles - group * 8, 8);
    const int n_tile = in_group / group_m, m_tile = group * 8 + in_group - n_tile * group_m;
    const int row0 = m_tile * TM, token0 = n_tile * TN;
    const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) void *)smem;
    const int in_copy = lane >> 3, piece = 16 * ((lane & 7) ^ in_copy);
    unsigned from[COPIES];
#pragma unroll
    for (int c = 0; c < COPIES; ++c) {
        const int r = (c * 4 + wave) * 8 + in_copy;
        from[c] = c * 32 < TM ? (unsigned)min(r, a.rows - 1 - row0) * (unsigned)a.columns + (unsigned)piece
                              : (unsigned)min(r - TM, a.tokens - 1 - token0) * (unsigned)a.levels_stride + (unsigned)piece;
    }
    const int8_t *w = a.weights + (long long)row0 * a.columns, *x = a.levels + (long long)token0 * a.levels_stride;
    const int stages = (a.columns + kStageBytes - 1) / kStageBytes;
    auto copy = [&](int c, int s, int buffer) {
        const unsigned back = s * kStageBytes + piece < a.columns ? 0u : (unsigned)piece;
        copy16_global_to_lds((c * 32 < TM ? w : x) + (size_t)s * kStageBytes, from[c] - back, lds0 + (unsigned)buffer * BUFFER + (unsigned)(c * 4 + wave) * 1024u);
    };
    i16v acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = (i16v)0;
    // A stage's operands of this wavefront: 16 bytes of a row each, its piece 2 wave + g.
    const int in_line = li * kStageBytes + ((2 * wave + g) ^ (li & 7)) * 16;
    struct Operands {
        i4 w[MT], x[NT];
    };
    auto read = [&](Operands &into, int buffer, int r) {
        const char *const line = smem + buffer * BUFFER + in_line;
        if (r < MT) into.w[r < MT ? r : 0] = *reinterpret_cast<const i4 *>(line + 32 * r * kStageBytes);
        else into.x[r < MT ? 0 : r - MT] = *reinterpret_cast<const i4 *>(line + (TM + 32 * (r - MT)) * kStageBytes);
    };
    // Stage s: behind the barrier the next stage has landed and every wavefront holds this one's operands, so that its place is filled again.  (Past
    // the last stage: that again, into a place that nobody reads.)
    auto run_stage = [&](auto last_one, int s, int buffer, Operands &now, Operands &next) __attribute__((always_inline)) {
        constexpr bool LAST = decltype(last_one)::value;
        constexpr int PRODUCTS = MT * NT, WORK = MT + NT + COPIES;
        if constexpr (LAST) {  // the columns behind the row's end: levels of zero, whatever the weights' place holds
            const int k = s * kStageBytes + 32 * wave + 16 * g;
#pragma unroll
            for (int j = 0; j < NT; ++j) now.x[j] = k < a.columns ? now.x[j] : (i4)0;
        } else {
            TT_WAIT_VMCNT((BUFFERS - 2) * COPIES);
            __syncthreads();
        }
        const int behind = buffer + 1 == BUFFERS ? 0 : buffer + 1, copied = min(s + BUFFERS, stages - 1);
#pragma unroll
        for (int u = 0; u < PRODUCTS; ++u) {
            const int i = u / NT, j = u % NT;
            acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(now.w[i], now.x[j], acc[i][j], 0, 0, 0);
            if constexpr (!LAST) {
#pragma unroll
                for (int r = 0; r < WORK; ++r) {
                    if (r * PRODUCTS / WORK != u) continue;
                    if (r < MT + NT) read(next, behind, r);
                    else copy(r - MT - NT, copied, buffer);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    static_assert(BUFFERS >= 3);
#pragma unroll
    for (int s = 0; s < BUFFERS; ++s)
#pragma unroll
        for (int c = 0; c < COPIES; ++c) copy(c, min(s, stages - 1), s);
    TT_WAIT_VMCNT((BUFFERS - 1) * COPIES);
    __syncthreads();
    Operands even, odd;
#pragma unroll
    for (int r = 0; r < MT + NT; ++r) read(even, 0, r);
    int buffer = 0, s = 0;
    auto step_on = [&] { buffer = buffer + 1 == BUFFERS ? 0 : buffer + 1; };
#pragma nounroll
    for (; s + 2 < stages; s += 2) {
        run_stage(std::false_type{}, s, buffer, even, odd);
        step_on();
        run_stage(std::false_type{}, s + 1, buffer, odd, even);
        step_on();
    }
    if (s + 1 < stages) {
        run_stage(std::false_type{}, s, buffer, even, odd);
        run_stage(std::true_type{}, s + 1, buffer, odd, even);
    } else {
        run_stage(std::true_type{}, s, buffer, even, odd);
    }
    TT_WAIT_VMCNT(0);
    __syncthreads();

    // The sums to their owners: owner o's tiles are (i0 .. i0 + OWN, j), i0 = o / NT * OWN, j = o % NT.
    i16v mine[OWN];
#pragma unroll
    for (int o = 0; o < 4; ++o) {
        const int i0 = o / NT * OWN, j = o % NT;
        if (wave == o) {
#pragma unroll
            for (int t = 0; t < OWN; ++t) mine[t] = acc[i0 + t][j];
        } else {
            i4 *const to = reinterpret_cast<i4 *>(smem + (3 * o + (wave < o ? wave : wave - 1)) * OWN * 4096) + lane;
#pragma unroll
            for (int t = 0; t < OWN; ++t)
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    const i16v &x = acc[i0 + t][j];
                    to[(t * 4 + v) * 64] = i4{x[4 * v], x[4 * v + 1], x[4 * v + 2], x[4 * v + 3]};
                }
        }
    }
    __syncthreads();
#pragma unroll
    for (int other = 0; other < 3; ++other) {
        const i4 *const of = reinterpret_cast<const i4 *>(smem + (3 * wave + other) * OWN * 4096) + lane;
#pragma unroll
        for (int t = 0; t < OWN; ++t)
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                const i4 x = of[(t * 4 + v) * 64];
#pragma unroll
                for (int e = 0; e < 4; ++e) mine[t][4 * v + e] += x[e];
            }
    }
    __syncthreads();

    // The rows out through LDS, as above.
    constexpr int PITCH = C::PITCH, LANES = OWN * 32 / 8, ROWS = 64 / LANES;
    float *const channel_scales = reinterpret_cast<float *>(smem + C::STAGING);
    if (threadIdx.x < TM) channel_scales[threadIdx.x] = a.weight_scales[min(row0 + (int)threadIdx.x, a.rows - 1)];
    __syncthreads();
    char *const stage = smem + wave * 32 * PITCH;
    const int wave_row = wave / NT * OWN * 32, wave_token0 = token0 + 32 * (wave % NT);
    const bool whole = (a.y_stride % 8 == 0) && (reinterpret_cast<size_t>(a.y) & 15) == 0;
    const float scale = a.scales[min(wave_token0 + li, a.tokens - 1)];
#pragma unroll
    for (int t = 0; t < OWN; ++t)
#pragma unroll
        for (int v = 0; v < 16; v += 4) {
            const int r = 32 * t + 8 * (v >> 2) + 4 * g;
            const f4 channel = *reinterpret_cast<const f4 *>(channel_scales + wave_row + r);
            h4 out;
#pragma unroll
            for (int e = 0; e < 4; ++e) out[e] = (_Float16)((float)mine[t][v + e] * channel[e] * scale);
            *reinterpret_cast<h4 *>(stage + li * PITCH + r * 2) = out;
        }
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int t = 0; t < 32; t += ROWS) {
        const int row = t + lane / LANES, first = (lane % LANES) * 8, to_token = wave_token0 + row, r = row0 + wave_row + first;
        const h8 out = *reinterpret_cast<const h8 *>(stage + row * PITCH + first * 2);
        if (to_token < a.tokens) {
            _Float16 *const to = a.y + to_token * a.y_stride + r;
            if (whole && r + 8 <= a.rows) {
                *reinterpret_cast<h8 *>(to) = out;
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (r + e < a.rows) to[e] = out[e];
            }
        }
    }
}
template <int TM, int TN, int BUFFERS>
hipError_t configure_steps() {
    return hipFuncSetAttribute(reinterpret_cast<const void *>(int8_steps_kernel<TM, TN, BUFFERS>), hipFuncAttributeMaxDynamicSharedMemorySize,
                               (int)StepsShape<TM, TN, BUFFERS>::LDS);
}
template <int TM, int TN, int BUFFERS>
void launch_steps(tt_hip_ctx *ctx, const ProductArgs &a) {
    static_assert(BUFFERS * ((TM + TN) / 32) <= 63 && StepsShape<TM, TN, BUFFERS>::LDS <= 160 * 1024, "what vmcnt counts to; LDS");
    const int m_tiles = (a.rows + TM - 1) / TM, n_tiles = (a.tokens + TN - 1) / TN;
    const int per_xcd = (int)(((long long)m_tiles * n_tiles + 7) / 8);
    launch_profiled(ctx, int8_steps_kernel<TM, TN, BUFFERS>, dim3((unsigned)per_xcd * 8u), dim3(256), (unsigned)StepsShape<TM, TN, BUFFERS>::LDS, a, m_tiles,
                    n_tiles, per_xcd);
}

bool aligned(const void *p, size_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

// Tokens that a call quantises: a workgroup of 256 threads each, of which a launch has fewer than 2^32.
bool tokens_served(int tokens) { return tokens < 1 << 24; }
// (the sums of products of two levels, at most 2^14 each, stay below 2^31)
bool columns_served(int columns) { return columns % 16 == 0 && columns < 131072; }

int check_quantise(const tt_half *x, size_t x_stride, int token_count, int columns, const int8_t *levels, size_t levels_stride, const float *scales) {
    if (!x || !levels || !scales || token_count <= 0 || columns <= 0) return TT_HIP_ERR_INVALID_ARGUMENT;
    if (!columns_served(columns) || !tokens_served(token_count) || x_stride < (size_t)columns || x_stride % 8 != 0 || levels_stride < (size_t)columns || levels_stride % 16 != 0 ||
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
    auto launch = [&](auto kernel) {
        launch_profiled(ctx, kernel, dim3((unsigned)token_count), dim3(256), 0u, reinterpret_cast<const _Float16 *>(x), (long long)x_stride, columns, levels,
                        (long long)levels_stride, scales);
    };
    if (columns <= 2048) launch(quantise_rows_kernel<1>);
    else if (columns <= 4096) launch(quantise_rows_kernel<2>);
    else launch(quantise_rows_kernel<4>);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? TT_HIP_OK : hip_fail(ctx, e, "quantise_rows_kernel launch");
}

// Tiles of the many tokens' kernel: what they are estimated to take, rounds of workgroups times their stages, us as measured with every CU
// at work (4,096 tokens, 9,216 x 5,120; 777, 2,311 x 4,096; 1,024 and 128, 4,096 x 4,096).
struct GemmTile {
    int tm, tn;
    double stage_us, fixed_us;
};
constexpr GemmTile kGemmTiles[] = {{256, 256, 1.75, 10.0}, {128, 256, 0.95, 5.0}, {128, 128, 0.62, 3.0}, {128, 64, 0.5, 2.0}, {64, 128, 0.46, 2.0}, {64, 64, 0.25, 3.0}};
int gemm_tile(const tt_hip_ctx *ctx, const ProductArgs &a) {
    int best = 0;
    double best_us = 0.0;
    for (int i = 0; i < (int)(sizeof(kGemmTiles) / sizeof(kGemmTiles[0])); ++i) {
        const GemmTile &t = kGemmTiles[i];
        const long long groups = (long long)((a.rows + t.tm - 1) / t.tm) * ((a.tokens + t.tn - 1) / t.tn);
        const double us = t.fixed_us + (double)((groups + ctx->n_cus - 1) / ctx->n_cus) * ((a.columns + kStageBytes - 1) / kStageBytes) * t.stage_us;
        if (i == 0 || us < best_us) {
            best = i;
            best_us = us;
        }
    }
    return best;
}
void launch_by_rule(tt_hip_ctx *ctx, const ProductArgs &a) {
    const int tiles = int8_ring_tiles(ctx->n_cus, a.rows), token_tiles = (a.tokens + 15) / 16;
    if (token_tiles <= 4 && !(tiles == 4 && token_tiles == 4)) {
        switch (tiles * 10 + token_tiles) {
            case 11: return launch_ring<1, 1, 8, 2, false>(ctx, a);
            case 12: return launch_ring<1, 2, 8, 3, false>(ctx, a);
            case 13: return launch_ring<1, 3, 4, 4, false>(ctx, a);
            case 14: return launch_ring<1, 4, 4, 4, false>(ctx, a);
            case 21: return launch_ring<2, 1, 8, 2, false>(ctx, a);
            case 22: return launch_ring<2, 2, 8, 2, false>(ctx, a);
            case 23: return launch_ring<2, 3, 8, 2, false>(ctx, a);
            case 24: return launch_ring<2, 4, 4, 3, false>(ctx, a);
            case 41: return launch_ring<4, 1, 4, 3, false>(ctx, a);
            case 42: return launch_ring<4, 2, 4, 3, false>(ctx, a);
            default: return launch_ring<4, 3, 4, 2, false>(ctx, a);
        }
    }
    switch (gemm_tile(ctx, a)) {
        case 0: return launch_gemm<256, 256, 2>(ctx, a);
        case 1: return launch_gemm<128, 256, 3>(ctx, a);
        case 2: return launch_gemm<128, 128, 4>(ctx, a);
        case 3: return launch_gemm<128, 64, 3>(ctx, a);
        case 4: return launch_gemm<64, 128, 6>(ctx, a);
        default: return launch_steps<64, 64, 4>(ctx, a);
    }
}

int launched(tt_hip_ctx *ctx) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? TT_HIP_OK : hip_fail(ctx, e, "8-bit product launch");
}
int launch_product(tt_hip_ctx *ctx, const ProductArgs &a) {
    launch_by_rule(ctx, a);
    return launched(ctx);
}
// The product whose workgroups quantise the tokens themselves: up to four, where the levels and the rings fit LDS.  `served` says whether.  A launch
// less, of 3 us, for what every workgroup spends on them (us on the device, with it / by two launches: one token, 2,048 x 4,096 5.9 /
// 9.2, four 7.4 / 9.5, 9,216 x 2,048 7.6 / 11.3, four 7.9 / 11.1, 5,120 x 6,144 8.6 / 13.1).
int launch_fused(tt_hip_ctx *ctx, const ProductArgs &a, const _Float16 *halves, long long halves_stride, bool *served) {
    const int tiles = int8_ring_tiles(ctx->n_cus, a.rows);
    const size_t lds = tiles == 4   ? ring_lds_bytes<4, 1, 4, 3, true>(a.tokens, a.columns)
                       : tiles == 2 ? ring_lds_bytes<2, 1, 8, 3, true>(a.tokens, a.columns)
                                    : ring_lds_bytes<1, 1, 8, 4, true>(a.tokens, a.columns);
    *served = a.tokens <= kFusedTokens && lds <= kMostLds;
    if (!*served) return TT_HIP_OK;
    if (tiles == 4) launch_ring<4, 1, 4, 3, true>(ctx, a, halves, halves_stride);
    else if (tiles == 2) launch_ring<2, 1, 8, 3, true>(ctx, a, halves, halves_stride);
    else launch_ring<1, 1, 8, 4, true>(ctx, a, halves, halves_stride);
    return launched(ctx);
}

// The context's store for tokens that a call quantises itself: their levels, then their scales.
int ensure_levels(tt_hip_ctx *ctx, size_t bytes) {
    if (bytes <= ctx->levels_bytes) return TT_HIP_OK;
    if (ctx->capturing) return TT_HIP_ERR_BUSY;
    hipError_t e = hipStreamSynchronize(ctx->stream);
    if (e != hipSuccess) return hip_fail(ctx, e, "hipStreamSynchronize");
    if (ctx->levels) ++ctx->generation;  // (a store that there was not yet is in no graph)
    if (ctx->levels) (void)hipFree(ctx->levels);
    ctx->levels = nullptr;
    ctx->levels_bytes = 0;
    const size_t want = bytes + bytes / 4;
    e = hipMalloc(reinterpret_cast<void **>(&ctx->levels), want);
    if (e != hipSuccess) return hip_fail(ctx, e, "hipMalloc(token levels)");
    ctx->levels_bytes = want;
    return TT_HIP_OK;
}

}  // namespace

int configure_int8_kernels(tt_hip_ctx *ctx) {
    hipError_t e = hipSuccess;
#define TT_CFG(...) \
    if (e == hipSuccess) e = __VA_ARGS__();
    TT_CFG(configure_gemm<256, 256, 2>) TT_CFG(configure_gemm<128, 256, 3>) TT_CFG(configure_gemm<128, 128, 4>) TT_CFG(configure_gemm<128, 64, 3>)
    TT_CFG(configure_gemm<64, 128, 6>) TT_CFG(configure_steps<64, 64, 4>)
    TT_CFG(configure_ring<1, 1, 8, 2, false>) TT_CFG(configure_ring<1, 2, 8, 3, false>) TT_CFG(configure_ring<1, 3, 4, 4, false>)
    TT_CFG(configure_ring<1, 4, 4, 4, false>) TT_CFG(configure_ring<2, 1, 8, 2, false>) TT_CFG(configure_ring<2, 2, 8, 2, false>)
    TT_CFG(configure_ring<2, 3, 8, 2, false>) TT_CFG(configure_ring<2, 4, 4, 3, false>) TT_CFG(configure_ring<4, 1, 4, 3, false>)
    TT_CFG(configure_ring<4, 2, 4, 3, false>) TT_CFG(configure_ring<4, 3, 4, 2, false>)
    TT_CFG(configure_ring<1, 1, 8, 4, true>) TT_CFG(configure_ring<2, 1, 8, 3, true>) TT_CFG(configure_ring<4, 1, 4, 3, true>)
#undef TT_CFG
    return e == hipSuccess ? TT_HIP_OK : hip_fail(ctx, e, "hipFuncSetAttribute(8-bit product max dynamic LDS)");
}

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
    if (!aligned(levels, 16) || levels_stride < (size_t)columns || levels_stride % 16 != 0 || levels_stride >= (1u << 24)) return TT_HIP_ERR_SHAPE;
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
    if (!tokens_served(token_count) || x_stride < (size_t)columns || x_stride % 8 != 0 || !aligned(x, 16)) return TT_HIP_ERR_SHAPE;
    BusyGuard guard(ctx);
    if (!guard.ok) return TT_HIP_ERR_BUSY;
    if (hipSetDevice(ctx->device) != hipSuccess) return TT_HIP_ERR_HIP;
    bool served = false;
    const int fused = launch_fused(ctx, ProductArgs{weights, weight_scales, nullptr, nullptr, reinterpret_cast<_Float16 *>(y), 0, (long long)y_stride, rows,
                                                    columns, token_count}, reinterpret_cast<const _Float16 *>(x), (long long)x_stride, &served);
    if (served || fused != TT_HIP_OK) return fused;
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
