// Rows whose keys lie in two pieces: the last pass over the partial results that one pass over each piece has left.
//
// A row's result over keys A and B with softmax statistics (m, l) and unnormalised sums o of each, m the maximum of either:
//   o = (2^(m_A - m) o_A + 2^(m_B - m) o_B) / (2^(m_A - m) l_A + 2^(m_B - m) l_B)
// and the same over any number of splits of either piece, so the splits of both are added up in one go; then the gate, in fp32, and one
// rounding.  A row that sees nothing gives zeros.
//
// What it takes is its trips to memory, one for the arguments and as few as may be for the partial rows: a workgroup is one (token, head) and
// DIMS dims of it, its threads own four dims of every G-th split, G = 1024 / DIMS, and ask for BATCH of those at once.  Rows of many splits
// go by 64 dims (sixteen splits side by side, up to 128 in one trip), rows of few in one workgroup, of which there are then fewer, and so do
// as many rows as fill the chip, whose splits are then read in longer runs (64 tokens of 16 heads of 256, 33 MB of partial
// results, by 64 dims / by 128 / whole 10.8 / 8.9 / 8.4 us; 18 of 24, 6.0 / 5.7 / 5.9; 20 of 32 heads of 128, 4.9 / 4.3 / 4.3).
#include <algorithm>

#include "internal.h"
#include "wave_ops.h"

namespace tt {

namespace {

typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f2 __attribute__((ext_vector_type(2)));
constexpr float kNegBig = -1.0e30f;

// Row n of tile `tile` in split 0 of a pass, for token `tok` of a sequence and q head `head`.
__device__ __forceinline__ size_t part_row(const PassParts &p, int group, int tok, int head) {
    const int kvh = head / group, in_group = head - kvh * group;
    if (p.gh == 0) {
        const int row = tok * group + in_group;
        return (size_t)(kvh * p.tok_tiles + row / p.nt) * p.nt + row % p.nt;
    }
    const int hsub = in_group / p.gh, tok_tile = tok / p.tt;
    const int tile = (kvh * p.hsubs + hsub) * p.tok_tiles + tok_tile;
    return (size_t)tile * p.nt + (tok - tok_tile * p.tt) * p.gh + (in_group - hsub * p.gh);
}

template <int D, int DIMS, int BATCH>
__global__ __launch_bounds__(256) void attn_join_kernel(const JoinArgs a) {
    constexpr int LANES = DIMS / 4, G = 256 / LANES, PARTS = D / DIMS;
    __shared__ f4 sums[G][LANES];
    __shared__ f2 stats[G];
    const int head = blockIdx.x / PARTS, row = blockIdx.y, seq = blockIdx.z;
    const int lane = threadIdx.x % LANES, g = threadIdx.x / LANES, d = (blockIdx.x - head * PARTS) * DIMS + lane * 4;
    const JoinSeq sq = a.seq[seq];
    _Float16 gate[4] = {};
    if (a.gate && g == 0) {
        const _Float16 *at = a.gate + seq * a.g_seq_stride + row * a.g_tok_stride + (long long)head * D + d;
#pragma unroll
        for (int i = 0; i < 4; ++i) gate[i] = at[i];
    }
    // The splits of both pieces in one count: where split s lies is `base + s * stride` of its piece.
    const size_t front_stride = (size_t)a.front.n_tiles * a.front.nt, own_stride = (size_t)a.own.n_tiles * a.own.nt;
    const size_t front_row = part_row(a.front, a.group, seq * a.rows + row, head);
    const size_t own_row = part_row(a.own, a.group, row, head) + (size_t)sq.first_split * own_stride;
    const int tile_end = min(sq.total, sq.start + min((row / a.own.tt + 1) * a.own.tt, a.rows));
    const int n = a.front_splits + max((max(tile_end, 0) + a.own.split_len - 1) / a.own.split_len, 1);
    float m = kNegBig, l = 0.0f;
    f4 acc = (f4)0.0f;
    for (int first = g; first < n; first += G * BATCH) {
        f4 o[BATCH];
        f2 ml[BATCH];
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            const int s = min(first + i * G, n - 1);
            const bool front = s < a.front_splits;
            const size_t at = front ? front_row + s * front_stride : own_row + (s - a.front_splits) * own_stride;
            ml[i] = *reinterpret_cast<const f2 *>((front ? a.front.ml : a.own.ml) + at * 2);
            o[i] = *reinterpret_cast<const f4 *>((front ? a.front.o : a.own.o) + at * D + d);
        }
        float top = m;
#pragma unroll
        for (int i = 0; i < BATCH; ++i) top = fmaxf(top, ml[i][0]);
        const float keep = __builtin_amdgcn_exp2f(m - top);
        l *= keep;
        acc *= keep;
        m = top;
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            if (first + i * G >= n) break;  // (not a factor of zero, which an infinite value makes NaN of)
            const float f = __builtin_amdgcn_exp2f(ml[i][0] - m);
            l += f * ml[i][1];
            acc += f * o[i];
        }
    }
    sums[g][lane] = acc;
    if (lane == 0) stats[g] = f2{m, l};
    __syncthreads();
    if (g != 0) return;
#pragma unroll
    for (int i = 1; i < G; ++i) m = fmaxf(m, stats[i][0]);
    f4 out = (f4)0.0f;
    float total = 0.0f;
#pragma unroll
    for (int i = 0; i < G; ++i) {
        const float f = __builtin_amdgcn_exp2f(stats[i][0] - m);
        total += f * stats[i][1];
        out += f * sums[i][lane];
    }
    out *= total > 0.0f ? 1.0f / total : 0.0f;
    if (a.gate) {
#pragma unroll
        for (int i = 0; i < 4; ++i) out[i] *= sigmoid((float)gate[i]);
    }
    _Float16 *const at = a.out + seq * a.o_seq_stride + row * a.o_tok_stride + (long long)head * D + d;
    const h4 r = {(_Float16)out[0], (_Float16)out[1], (_Float16)out[2], (_Float16)out[3]};
    if (a.aligned) {
        *reinterpret_cast<h4 *>(at) = r;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) at[i] = r[i];
    }
}

template <int D>
void launch_join_of(tt_hip_ctx *ctx, int n_seq, const JoinArgs &args) {
    int most = 0;  // splits of a row
    for (int i = 0; i < n_seq; ++i) most = std::max(most, args.seq[i].total);
    most = args.front_splits + std::max((most + args.own.split_len - 1) / args.own.split_len, 1);
    auto launch = [&](auto kernel, int parts) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)(args.heads * parts), (unsigned)args.rows, (unsigned)n_seq), dim3(256), 0, ctx->stream, args);
    };
    if (most <= 4 * 1024 / D || (long long)args.heads * args.rows * n_seq >= 2 * ctx->n_cus) launch(attn_join_kernel<D, D, 4>, 1);
    else if (most <= 64) launch(attn_join_kernel<D, 64, 4>, D / 64);
    else launch(attn_join_kernel<D, 64, 8>, D / 64);
}

}  // namespace

int launch_join(tt_hip_ctx *ctx, int head_dim, int n_seq, const JoinArgs &args) {
    if (n_seq > kMaxSeqPerLaunch || args.rows > 65535) return TT_HIP_ERR_SHAPE;
    switch (head_dim) {
        case 256: launch_join_of<256>(ctx, n_seq, args); break;
        case 128: launch_join_of<128>(ctx, n_seq, args); break;
        case 64: launch_join_of<64>(ctx, n_seq, args); break;
        default: return TT_HIP_ERR_SHAPE;
    }
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? TT_HIP_OK : hip_fail(ctx, e, "attn_join_kernel launch");
}

}  // namespace tt
