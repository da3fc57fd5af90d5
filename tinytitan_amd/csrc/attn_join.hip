// Rows whose keys lie in two pieces: the last pass over the partial results that one pass over each piece has left.
//
// A row's result over keys A and B with softmax statistics (m, l) and unnormalised sums o of each, m the maximum of either:
//   o = (2^(m_A - m) o_A + 2^(m_B - m) o_B) / (2^(m_A - m) l_A + 2^(m_B - m) l_B)
// and the same over any number of splits of either piece, so the splits of both are added up in one go; then the gate, in fp32, and one
// rounding.  A row that sees nothing gives zeros.
//
// What it takes is a trip to memory for the arguments and one for the partial rows: a workgroup is one (token, head), its threads own
// four dims of every G-th split each, and ask for kBatch of those at once.
#include "internal.h"
#include "wave_ops.h"

namespace tt {

namespace {

typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f2 __attribute__((ext_vector_type(2)));
constexpr float kNegBig = -1.0e30f;
constexpr int kBatch = 4;

// Row n of tile `tile` in split 0 of a pass, for token `tok` of a sequence and q head `head`.
__device__ __forceinline__ size_t part_row(const PassParts &p, int group, int tok, int head) {
    const int kvh = head / group, in_group = head - kvh * group;
    const int hsub = in_group / p.gh, tok_tile = tok / p.tt;
    const int tile = (kvh * p.hsubs + hsub) * p.tok_tiles + tok_tile;
    return (size_t)tile * p.nt + (tok - tok_tile * p.tt) * p.gh + (in_group - hsub * p.gh);
}

template <int D>
__global__ __launch_bounds__(256) void attn_join_kernel(const JoinArgs a) {
    constexpr int D4 = D / 4, G = 256 / D4;
    __shared__ f4 sums[G][D4];
    __shared__ f2 stats[G];
    const int head = blockIdx.x, row = blockIdx.y, seq = blockIdx.z;
    const int d = (threadIdx.x % D4) * 4, g = threadIdx.x / D4;
    const JoinSeq sq = a.seq[seq];
    const _Float16 *gate_at = a.gate + seq * a.g_seq_stride + row * a.g_tok_stride + (long long)head * D + d;
    _Float16 gate[4] = {};
    if (a.gate && g == 0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) gate[i] = gate_at[i];
    }
    const size_t front_row = part_row(a.front, a.group, seq * a.rows + row, head);
    const size_t own_row = part_row(a.own, a.group, row, head) + (size_t)sq.first_split * a.own.n_tiles * a.own.nt;
    const int tile_end = min(sq.total, sq.start + min((row / a.own.tt + 1) * a.own.tt, a.rows));
    const int n = a.front_splits + max((max(tile_end, 0) + a.own.split_len - 1) / a.own.split_len, 1);
    float m = kNegBig, l = 0.0f;
    f4 acc = (f4)0.0f;
    for (int first = g; first < n; first += G * kBatch) {
        f4 o[kBatch];
        f2 ml[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int s = min(first + i * G, n - 1);
            const bool front = s < a.front_splits;
            const PassParts &p = front ? a.front : a.own;
            const size_t at = (front ? front_row : own_row) + (size_t)(front ? s : s - a.front_splits) * p.n_tiles * p.nt;
            ml[i] = *reinterpret_cast<const f2 *>(p.ml + at * 2);
            o[i] = *reinterpret_cast<const f4 *>(p.o + at * D + d);
        }
        float top = m;
#pragma unroll
        for (int i = 0; i < kBatch; ++i) top = fmaxf(top, ml[i][0]);
        const float keep = __builtin_amdgcn_exp2f(m - top);
        l *= keep;
        acc *= keep;
        m = top;
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            if (first + i * G >= n) break;  // (not a factor of zero, which an infinite value makes NaN of)
            const float f = __builtin_amdgcn_exp2f(ml[i][0] - m);
            l += f * ml[i][1];
            acc += f * o[i];
        }
    }
    sums[g][threadIdx.x % D4] = acc;
    if (threadIdx.x % D4 == 0) stats[g] = f2{m, l};
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
        out += f * sums[i][threadIdx.x];
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

}  // namespace

int launch_join(tt_hip_ctx *ctx, int head_dim, int n_seq, const JoinArgs &args) {
    if (n_seq > kMaxSeqPerLaunch || args.rows > 65535) return TT_HIP_ERR_SHAPE;
    const dim3 grid((unsigned)args.heads, (unsigned)args.rows, (unsigned)n_seq);
    switch (head_dim) {
        case 256: hipLaunchKernelGGL(attn_join_kernel<256>, grid, dim3(256), 0, ctx->stream, args); break;
        case 128: hipLaunchKernelGGL(attn_join_kernel<128>, grid, dim3(256), 0, ctx->stream, args); break;
        case 64: hipLaunchKernelGGL(attn_join_kernel<64>, grid, dim3(256), 0, ctx->stream, args); break;
        default: return TT_HIP_ERR_SHAPE;
    }
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? TT_HIP_OK : hip_fail(ctx, e, "attn_join_kernel launch");
}

}  // namespace tt
