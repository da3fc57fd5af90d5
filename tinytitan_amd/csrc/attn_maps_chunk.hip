// Differential attention of a causal chunk on gfx950 MFMA (attn_maps.hip tells the operator).
//
// Transposed as the other attention kernels are, a lane owns a query row:
//   S^T[key][row] = K_m . Q_m^T      A = K fragment, of map m's half of the dims,  B = Q^T fragment, both in registers
//   O^T[d][row]  += V^T . P^T        A = V^T fragment out of LDS,                  B = P^T as it left S^T's registers
// with v_mfma_f32_32x32x16_f16.  A workgroup takes 128 rows, four tiles of 32 (heads that share a KV head, of one or more tiles of tokens).  Heads of 256
// and 64: four wavefronts, 2 p + m with map m of tiles 2 p and 2 p + 1; heads of 128: eight, 2 p + m with map m of tile p.  The maps of a tile
// meet at the end.
//
// What shapes it: LDS hands out 64 bytes a cycle and CU, half of what a matrix product wants whose operand comes from there each time.  So with two tiles an
// operand of V is used twice, and K, whose blocks lie in memory as the operands are, comes straight into registers, a block ahead.
// Of heads of 256 a block of keys is 48 products a wavefront, 1,536 cycles, beside 80 KiB of LDS traffic a CU, 1,280, and 48 KiB through the
// vector memory path, 768.  One wavefront a SIMD has all 512 registers (256 of them sums over V), so nothing but its own order hides one kind of work
// behind another: the softmax of block i is cut into pieces of a few instructions each, one between any two of the products of block i's
// scores and block i - 1's values.  Heads of 128 leave room for two wavefronts a SIMD with a tile each, which hide each other's waits (one wavefront with
// two tiles issued 68 % of its cycles, with the matrix pipe busy for 41, and waited 19; the two issue 92 % of their SIMD's, the matrix pipe 48) at nearly twice
// the LDS traffic, 72 KiB a block with the copies, 1,152 cycles, in place of 40, beside 768 of products.  Heads of 64 are bound by their instructions: a
// product has twice the exponentials, conversions and maxima of one of 128, the two wavefronts of a SIMD issue 112 cycles in 100 (of different kinds
// side by side), and the matrix pipe is busy for 38.
//
// Measured, us a call: 4,096 rows behind 4,500 keys 586 - 605 with 16/2 heads of 256 (1.09 - 1.12 PFLOP/s, of 1.22 that a library product reaches),
// 704 with 32/8 of 128 (0.94; two tiles a wavefront 716), 240 - 249 with 16/4 of 64 (0.66 - 0.69); 777 rows behind 9,000 of 32/8 heads of 128 230 - 235
// (two tiles 252).  Tried and not kept, heads of 256 / of 128 with two tiles: the copies of V in front of all reads of K +16 / +23 %, each in
// front of one +2 / +1; a barrier every second step, eight blocks of V, +2 / +1; the sums of the weights by dot products of pairs
// +4 / +6; two workgroups a CU for heads of 128, in 256 registers, +23.  Those sums as one more tile of values, of ones, which takes an eleventh of the vector
// instructions away and makes two products of them: heads of 128 +2 on a full chip and even below, of 64 even.
#include <algorithm>

#include "lds_copy.h"
#include "splitk_kernel.h"

namespace tt {

namespace {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
constexpr float kChunkRescale = 8.0f;
constexpr int kVRing = 4;  // blocks of V in LDS: the one in hand, the next two, and the one that every wavefront is done with

struct MapsChunkArgs {
    const _Float16 *k_slot, *v_slot;  // page of KV head 0 of the slot
    const _Float16 *q, *gate;
    _Float16 *out;
    long long page_elems, q_stride, g_stride, o_stride;
    MapHeads maps;
    int n_kv_heads, group, hs, sets;  // hs: heads of a workgroup (4, 2 or 1), of which a KV head has `sets`
    int tok_tiles;                    // of 128 / hs tokens
    int xs, per_kvh;                  // XCDs of a KV head (0: dealt out as they come), workgroups of one
    int start, q_len, kv_valid, window, ring_blocks;
    float scale_log2e;
    int n_splits, split_blocks;  // n_splits > 1: ranges of this many blocks, partial results
    float *part_o, *part_ml;     // [split][(row of maps) * tok_tiles + tile][token of the tile]
    int aligned;
};

template <int D>
struct ChunkShape {
    static constexpr int RT = D == 128 ? 1 : 2, WAVES = 8 / RT;  // row tiles of a wavefront, wavefronts
    static constexpr int KS = D / 32, MT = D / 32, VF = 2 * MT, CPW = VF / WAVES;  // score steps of a map, tiles of dims, V fragments of a block, copies a wavefront
    static constexpr int V_BYTES = 64 * D, RING_BYTES = kVRing * V_BYTES;
    static constexpr int X_BYTES = 128 * D;               // a tile's sums on their way to the other map's wavefront
    static constexpr int STAGE_PITCH = 64 + 16, STAGE_BYTES = 32 * STAGE_PITCH;
    static constexpr int STAGE_OFF = std::max(RING_BYTES, 4 * X_BYTES);
    static constexpr int LDS = STAGE_OFF + 4 * STAGE_BYTES;
};

// The products of the scores, in vector registers: the compiler gives every matrix instruction of a kernel with 512 registers accumulation registers,
// and those are the sums over V alone.  What the compiler does about an instruction's wait states it does not do for these:
//   a product reads the sum of the one before it as it comes (the same registers), and the first takes a zero for it, not one that was just written;
//   a vector instruction that reads a sum wants 19 cycles of four clocks behind the last of its products.  Every product of this size holds the
//   matrix pipe for eight of those cycles, so that two more products issued in between are room enough.
//   a product wants two cycles of four clocks behind a vector instruction that writes one of its operands; K's come from memory, the queries' are not
//   written in the loop (an operand parked in an accumulation register and fetched right here gave wrong scores).
// tests/test_wait_states_maps.py looks for each in the compiler's listing.
__device__ __forceinline__ void first_score(f16v &s, h8 k, h8 q) { asm volatile("v_mfma_f32_32x32x16_f16 %0, %1, %2, 0" : "=&v"(s) : "v"(k), "v"(q)); }
__device__ __forceinline__ void next_score(f16v &s, h8 k, h8 q) { asm volatile("v_mfma_f32_32x32x16_f16 %0, %1, %2, %0" : "+v"(s) : "v"(k), "v"(q)); }
// ... where no two products follow.
__device__ __forceinline__ void settle(f16v &s) { asm volatile("s_nop 15\n\ts_nop 7" : "+v"(s)); }

__device__ __forceinline__ float max3(float x, float y, float z) {  // (written as a maximum of maxima, each operand is first made canonical)
    float most;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(most) : "v"(x), "v"(y), "v"(z));
    return most;
}
// A sum over V stays in accumulation registers, wherever control flow comes from: told so behind everything that writes it, or the compiler moves
// the sums to vector registers and back around every block.
__device__ __forceinline__ void keep_sum(f16v &o) { asm volatile("" : "+a"(o)); }
// ... where it is read in a branch of the first or the second map's wavefronts, in words of its own: else the two are made one that selects
// every register.
template <bool SECOND>
__device__ __forceinline__ void keep_sum_of(const f16v &o) {
    if constexpr (SECOND) asm volatile("; the second map" ::"a"(o));
    else asm volatile("; the first map" ::"a"(o));
}

template <typename F, int... I>
__device__ __forceinline__ void unrolled_over(std::integer_sequence<int, I...>, F f) {
    (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void unrolled(F f) {
    unrolled_over(std::make_integer_sequence<int, N>{}, f);
}
// `pieces` pieces of work over the slots [from, slots): the first one of slot `slot`.
constexpr int piece_of_slot(int slot, int from, int slots, int pieces) {
    return slot <= from ? 0 : ((slot - from) * pieces + slots - from - 1) / (slots - from);
}

template <int D>
__global__ __launch_bounds__(64 * ChunkShape<D>::WAVES, D == 256 ? 1 : 2) void attn_maps_chunk_kernel(const MapsChunkArgs a) {
    typedef ChunkShape<D> C;
    constexpr int RT = C::RT, KS = C::KS, MT = C::MT, VF = C::VF, CPW = C::CPW, BLOCK = 64 * D;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), li = lane & 31, g = lane >> 5;
    const int map = wave & 1, pair = wave >> 1;

    // Workgroup -> (KV head, range, tile of tokens, set of heads); the longest tiles first, a KV head's on its own XCDs.
    int kvh, r;
    if (a.xs > 0) {
        const int x = blockIdx.x & 7;
        kvh = x / a.xs;
        r = (int)(blockIdx.x >> 3) * a.xs + (x - kvh * a.xs);
    } else {
        kvh = blockIdx.x / a.per_kvh;
        r = blockIdx.x - kvh * a.per_kvh;
    }
    if (r >= a.per_kvh) return;
    const int per_split = a.tok_tiles * a.sets, split = r / per_split, in_split = r - split * per_split;
    const int tile = a.tok_tiles - 1 - in_split / a.sets, set = in_split % a.sets;
    const int span = 128 / a.hs, t0 = tile * span;  // tokens of the workgroup

    // The blocks it walks: from the one of the first key that its first row sees to the one of its last row's last key.
    const int end = min(a.kv_valid, a.start + min(a.q_len, t0 + span));
    const int first_key = a.window > 0 && a.start + t0 + 1 > a.window ? a.start + t0 + 1 - a.window : 0;
    const int jb = (first_key >> 5) + split * a.split_blocks, nb_all = ((end + 31) >> 5) - jb;
    const int nb = a.n_splits > 1 ? min(nb_all, a.split_blocks) : nb_all;
    if (nb <= 0) return;

    // This wavefront's rows: RT tiles, from RT pair on.
    int head[RT], tok[RT], lim[RT], lo[RT];
    bool valid[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int u = RT * pair + rt;
        head[rt] = kvh * a.group + set * a.hs + u % a.hs;
        tok[rt] = t0 + 32 * (u / a.hs) + li;
        valid[rt] = tok[rt] < a.q_len;
        // (a row that is not there sees everything: no block is masked for it, and nobody looks at it)
        lim[rt] = valid[rt] ? min(a.kv_valid, a.start + tok[rt] + 1) : 0x7fffffff;
        lo[rt] = valid[rt] && a.window > 0 && a.start + tok[rt] + 1 > a.window ? a.start + tok[rt] + 1 - a.window : 0;
    }
    // Blocks from first_masked on, and with a window those up to last_below, hide keys from some row of the wavefront.
    const int wave_t0 = t0 + 32 * (RT * pair / a.hs), wave_t1 = t0 + 32 * ((RT * pair + RT - 1) / a.hs) + 31;
    const int first_masked = min(a.start + wave_t0 + 1, a.kv_valid) >> 5;
    const int last_below = a.window > 0 && a.start + wave_t1 + 1 > a.window ? (a.start + wave_t1 - a.window) >> 5 : -1;

    const __amdgpu_buffer_rsrc_t rk = make_rsrc(a.k_slot + (size_t)kvh * a.page_elems, (unsigned)(a.page_elems * 2));
    const _Float16 *const v_page = a.v_slot + (size_t)kvh * a.page_elems;
    // Where a block of the walk lies in the page, in bytes, from block to block; past the last one that again.
    struct Place {
        unsigned at, wrap;
        int left;
        __device__ __forceinline__ void next() {
            const unsigned on = at + (unsigned)BLOCK;
            at = left > 0 ? (on == wrap ? 0u : on) : at;
            --left;
        }
    };
    Place k_at{(unsigned)(a.ring_blocks ? jb % a.ring_blocks : jb) * (unsigned)BLOCK, a.ring_blocks ? (unsigned)a.ring_blocks * (unsigned)BLOCK : 0xffffffffu, nb - 1};
    Place v_at = k_at;
    const unsigned k_lane = (unsigned)(map * (BLOCK / 2) + lane * 16);
    const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) void *)smem;
    unsigned v_from[CPW];
#pragma unroll
    for (int c = 0; c < CPW; ++c) {
        const int f = wave * CPW + c;
        v_from[c] = 2u * (unsigned)(v_piece(D, li, g) + v_piece(D, 32 * (f >> 1), 2 * (f & 1)));
    }
    auto copy_v = [&](int i, int c) {  // of block i, which lies at v_at
        copy16_global_to_lds(reinterpret_cast<const char *>(v_page) + v_at.at, v_from[c], lds0 + (unsigned)((i % kVRing) * C::V_BYTES + (wave * CPW + c) * 1024));
    };

    h8 q[RT][KS], kf[KS];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const global_halves row = (global_halves)(a.q + (long long)(valid[rt] ? tok[rt] : 0) * a.q_stride + (long long)head[rt] * D + map * (D / 2) + 8 * g);
#pragma unroll
        for (int t = 0; t < KS; ++t) q[rt][t] = load_h8(row + 16 * t);
    }
#pragma unroll
    for (int t = 0; t < KS; ++t) kf[t] = buf_load_h8<0>(rk, k_lane, k_at.at + t * 1024);
    k_at.next();
#pragma unroll
    for (int i = 0; i < kVRing - 1; ++i) {
#pragma unroll
        for (int c = 0; c < CPW; ++c) copy_v(i, c);
        v_at.next();
    }
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int t = 0; t < KS; ++t) q[rt][t] = valid[rt] ? q[rt][t] : (h8)(_Float16)0;

    f16v o[RT][MT], s[RT];
    float m[RT], l[RT], l_odd[RT], mx[RT], alpha[RT];
    h8 p[RT][2];  // weights of the block whose values are next
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            o[rt][mt] = (f16v)0.0f;
            keep_sum(o[rt][mt]);
        }
        m[rt] = kNegBig;
        l[rt] = l_odd[rt] = 0.0f;
    }
    // The softmax of a tile's block in PIECES pieces: two of the maximum, two of the reference, and of each of the lane's eight pairs of keys two, so
    // that no piece reads an exponential of its own.
    constexpr int PIECES = 2 + 2 + 2 * 8;
    auto soften = [&](auto rt_c, auto piece_c, h8 (&p_next)[RT][2]) __attribute__((always_inline)) {
        constexpr int rt = decltype(rt_c)::value, piece = decltype(piece_c)::value;
        if constexpr (piece < 2) {
            constexpr int v = 8 * piece;
            float x = max3(s[rt][v], s[rt][v + 1], s[rt][v + 2]);
            x = max3(x, s[rt][v + 3], s[rt][v + 4]);
            x = max3(x, s[rt][v + 5], s[rt][v + 6]);
            mx[rt] = piece == 0 ? max3(x, s[rt][v + 7], s[rt][v + 7]) : max3(x, s[rt][v + 7], mx[rt]);
        } else if constexpr (piece == 2) {
            mx[rt] = max_across_halves(mx[rt]) * a.scale_log2e;
        } else if constexpr (piece == 3) {
            const bool move = mx[rt] > m[rt] + kChunkRescale;  // (a row's first visible block always moves)
            const float moved = move ? mx[rt] : m[rt];
            alpha[rt] = fast_exp2(m[rt] - moved);  // (1 where it stays)
            l[rt] *= alpha[rt];
            l_odd[rt] *= alpha[rt];
            m[rt] = moved;
        } else {
            constexpr int v = (piece - 4) / 2 * 2;
            if constexpr (piece % 2 == 0) {
                s[rt][v] = fast_exp2(__builtin_fmaf(s[rt][v], a.scale_log2e, -m[rt]));
                s[rt][v + 1] = fast_exp2(__builtin_fmaf(s[rt][v + 1], a.scale_log2e, -m[rt]));
            } else {
                // (the sum over the rounded weights, those that the products with V see)
                const h2 w = {(_Float16)s[rt][v], (_Float16)s[rt][v + 1]};
                asm("v_fma_mix_f32 %0, %1, 1.0, %0 op_sel_hi:[1,0,0]" : "+v"(l[rt]) : "v"(w));
                asm("v_fma_mix_f32 %0, %1, 1.0, %0 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "+v"(l_odd[rt]) : "v"(w));
                p_next[rt][v >> 3][v & 7] = w[0];
                p_next[rt][v >> 3][(v & 7) + 1] = w[1];
            }
        }
    };
    auto hide = [&](int rt, int block) __attribute__((always_inline)) {
        int base = (block << 5) + 4 * g;
        asm volatile("" : "+v"(base));  // (or the keys' numbers are made in front of the branch, in every step)
#pragma unroll
        for (int v = 0; v < 16; ++v) {
            const int key = base + 8 * (v >> 2) + (v & 3);
            if (key >= lim[rt] || key < lo[rt]) s[rt][v] = -INFINITY;
        }
    };
    // Keys of block i that some row of the workgroup sees, bit by bit.
    auto seen_of = [&](int i) { return keys_between(first_key - ((jb + i) << 5), end - ((jb + i) << 5)); };
    // Values of keys that no row sees, whatever the cache holds there, as zeros: a weight of zero would make NaN of an infinite one.  Every wavefront
    // those of its own copies, which have landed; they are in the walk's first block and in the sequence's last one.
    auto drop_unseen_of = [&](int i) __attribute__((always_inline)) {
        const unsigned seen = seen_of(i);
        if (seen == ~0u) return;
#pragma unroll
        for (int c = 0; c < CPW; ++c) {
            h8 *const at = reinterpret_cast<h8 *>(smem + (i % kVRing) * C::V_BYTES + (wave * CPW + c) * 1024 + lane * 16);
            unsigned mask[4];
            seen_words(mask, 2 * ((wave * CPW + c) & 1) + g, seen);
            *at = only_seen(*at, mask);
        }
    };
    auto read_v = [&](int i, int f) { return *reinterpret_cast<const h8 *>(smem + (i % kVRing) * C::V_BYTES + f * 1024 + lane * 16); };
    // Step i: the scores of block i, and between their products and those of block i - 1's values the softmax of block i.
    unsigned ring = 0;  // where block i - 1's values lie in LDS
    auto step = [&](int i, const h8 (&p_now)[RT][2], h8 (&p_next)[RT][2]) __attribute__((always_inline)) {
        constexpr int CHAIN = (RT - 1) * KS, SLOTS = CHAIN + 2 * RT * MT, FROM = 2;  // (a tile's scores are read behind the third product after their last)
        // V of block i - 1 has landed (K and V of the two steps since may be on their way; block 0's: see in front of the loop), and every wavefront
        // is done with the block whose place the copies of this step take.
        TT_WAIT_VMCNT(2 * (KS + CPW));
        __syncthreads();
        const unsigned next_k = k_at.at;
        const bool hidden = jb + i >= first_masked || jb + i <= last_below;
        const char *const v_block = smem + ring + lane * 16, *const v_next = reinterpret_cast<const char *>(v_page) + v_at.at;
        ring = (ring + C::V_BYTES) & (C::RING_BYTES - 1);
        const unsigned v_to = lds0 + ((ring + 2 * C::V_BYTES) & (C::RING_BYTES - 1)) + (unsigned)(wave * CPW) * 1024u;  // block i + 2's place
        h8 vf[2][2];  // two tiles of dims
        auto read_v = [&](int mt) __attribute__((always_inline)) {
#pragma unroll
            for (int t = 0; t < 2; ++t) vf[mt & 1][t] = *reinterpret_cast<const h8 *>(v_block + (2 * mt + t) * 1024);
        };
#pragma unroll
        for (int t = 0; t < KS; ++t) {
            if (t == 0) first_score(s[0], kf[0], q[0][0]);
            else next_score(s[0], kf[t], q[0][t]);
            if (t < 2) read_v(t);
            if constexpr (RT == 1) kf[t] = buf_load_h8<0>(rk, k_lane + (t & 3) * 1024, next_k + (t >> 2) * 4096);
            __builtin_amdgcn_sched_barrier(0);
        }
        if (hidden) {
            settle(s[0]);
            hide(0, jb + i);
        }
        unrolled<SLOTS>([&](auto slot_c) __attribute__((always_inline)) {
            constexpr int slot = decltype(slot_c)::value;
            if constexpr (slot < CHAIN) {
                if constexpr (slot == 0) first_score(s[RT - 1], kf[0], q[RT - 1][0]);
                else next_score(s[RT - 1], kf[slot], q[RT - 1][slot]);
                kf[slot] = buf_load_h8<0>(rk, k_lane + (slot & 3) * 1024, next_k + (slot >> 2) * 4096);
            } else {
                // (two products in a row to a sum: 32 cycles each, 36 where the sum is another every time)
                constexpr int u = slot - CHAIN, mt = u / (2 * RT), rt = (u >> 1) % RT, t = u & 1;
                if constexpr (RT == 2 && u == 0) {
                    if (hidden) {
                        settle(s[RT - 1]);
                        hide(RT - 1, jb + i);
                    }
                }
                o[rt][mt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[mt & 1][t], p_now[rt][t], o[rt][mt], 0, 0, 0);
                keep_sum(o[rt][mt]);
                if constexpr (rt == RT - 1 && t == 1 && mt + 2 < MT) read_v(mt + 2);
                constexpr int EVERY = 2 * RT * MT / CPW;
                if constexpr (u % EVERY == 2) copy16_global_to_lds(v_next, v_from[u / EVERY], v_to + (u / EVERY) * 1024u);
            }
            constexpr int first = piece_of_slot(slot, FROM, SLOTS, RT * PIECES), behind = piece_of_slot(slot + 1, FROM, SLOTS, RT * PIECES);
            if constexpr (RT == 2 && first < behind && first <= PIECES && behind > PIECES) static_assert(slot >= KS + 2, "the other tile's scores");
            unrolled<behind - first>([&](auto at) __attribute__((always_inline)) {
                constexpr int piece = first + decltype(at)::value;
                if constexpr (piece % PIECES == 0) asm volatile("" : "+v"(s[piece / PIECES]));  // (not read before here)
                soften(std::integral_constant<int, piece / PIECES>{}, std::integral_constant<int, piece % PIECES>{}, p_next);
            });
            __builtin_amdgcn_sched_barrier(0);
        });
        k_at.next();
        v_at.next();
    };
    auto copy_weights = [&](const h8 (&from)[RT][2], h8 (&to)[RT][2]) __attribute__((always_inline)) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int t = 0; t < 2; ++t) to[rt][t] = from[rt][t];
    };

    // Block 0's scores and softmax.
#pragma unroll
    for (int t = 0; t < KS; ++t) {
        if (t == 0) {
            first_score(s[0], kf[0], q[0][0]);
            if constexpr (RT == 2) first_score(s[1], kf[0], q[1][0]);
        } else {
            next_score(s[0], kf[t], q[0][t]);
            if constexpr (RT == 2) next_score(s[1], kf[t], q[1][t]);
        }
        kf[t] = buf_load_h8<0>(rk, k_lane, k_at.at + t * 1024);
    }
    k_at.next();
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) settle(s[rt]);
    if (jb >= first_masked || jb <= last_below) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) hide(rt, jb);
    }
    unrolled<RT * PIECES>([&](auto piece) __attribute__((always_inline)) {
        soften(std::integral_constant<int, decltype(piece)::value / PIECES>{}, std::integral_constant<int, decltype(piece)::value % PIECES>{}, p);
    });
    // Block 0's values have landed: behind their copies there are only two blocks' and one block's K, not the two that the first step's wait lets be
    // on their way.  (The compiler's own waits for K, which count the copies without knowing them, say so too, in another place in every build.)
    TT_WAIT_VMCNT(KS + 2 * CPW);
    const int last = nb - 1;
    if (last > 0 && seen_of(0) != ~0u) {
        TT_WAIT_VMCNT(0);
        asm volatile("" ::: "memory");
        drop_unseen_of(0);
    }
    // A run of steps is a loop of its own, left where a row's reference moves: with the rare scaling of the sums inside it the compiler moved them
    // about in every step.
    for (int i = 1; i <= last;) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) keep_sum(o[rt][mt]);
        bool scale_sums;
#pragma nounroll
        do {  // (two steps a turn, with the weights' registers in turn, were 5 % slower at heads of 128 and do not fit at heads of 256)
            h8 p_next[RT][2];
            step(i, p, p_next);
            ++i;
            scale_sums = __any(alpha[0] != 1.0f || alpha[RT - 1] != 1.0f);
            copy_weights(p_next, p);
        } while (!scale_sums && i <= last);
        if (scale_sums) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    // (one at a time, and each kept where it is: no registers are left to have several on their way)
                    keep_sum(o[rt][mt]);
                    o[rt][mt] *= alpha[rt];
                    keep_sum(o[rt][mt]);
                    __builtin_amdgcn_sched_barrier(0);
                }
        }
    }
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) keep_sum(o[rt][mt]);
    // The last block's values.
    TT_WAIT_VMCNT(0);
    asm volatile("" ::: "memory");
    drop_unseen_of(last);
    __syncthreads();
#pragma unroll
    for (int f = 0; f < VF; ++f) {
        const h8 x = read_v(last, f);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            o[rt][f >> 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, p[rt][f & 1], o[rt][f >> 1], 0, 0, 0);
            keep_sum(o[rt][f >> 1]);
        }
    }
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) l[rt] = sum_across_halves(l[rt] + l_odd[rt]);

    // Lane (li, g), register v of tile mt holds dim 32 mt + 8 (v / 4) + 4 g + v % 4 of row li.
    if (a.n_splits > 1) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            if (!valid[rt]) continue;
            const size_t row = (((size_t)split * (2 * a.group * a.n_kv_heads) + 2 * head[rt] + map) * a.tok_tiles + tile) * span + (tok[rt] - t0);
            float *const po = a.part_o + row * D + 4 * g;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int vq = 0; vq < 4; ++vq) {
                    const f4 x = {o[rt][mt][4 * vq], o[rt][mt][4 * vq + 1], o[rt][mt][4 * vq + 2], o[rt][mt][4 * vq + 3]};
                    *reinterpret_cast<f4 *>(po + 32 * mt + 8 * vq) = x;
                }
            if (g == 0) {
                a.part_ml[row * 2] = m[rt];
                a.part_ml[row * 2 + 1] = l[rt];
            }
        }
        return;
    }

    // The maps of a tile meet: of two tiles wavefront (pair, map) takes the pair's tile `map` and hands its sums of the other one over, as they are; of one
    // tile the second map's wavefront hands them to the first's.  What follows
    // is done once a workgroup, straight on, so that its time goes by its length: the sums are chosen by branches, no select of each register,
    // and the tile's difference lies in LDS, so that norm, gate and stores are a short loop over tiles of 32 dims.
    __syncthreads();  // (the ring's place is the sums')
    f4 *const to_partner = reinterpret_cast<f4 *>(smem + (RT == 2 ? wave : pair) * C::X_BYTES) + lane;
    f4 *const from_partner = reinterpret_cast<f4 *>(smem + (RT == 2 ? wave ^ 1 : pair) * C::X_BYTES) + lane;
    float *const sums = reinterpret_cast<float *>(smem + C::STAGE_OFF);
    const bool second_tile = RT == 2 && map;
    const float my_l = second_tile ? l[RT - 1] : l[0];
    const int my_tok = second_tile ? tok[RT - 1] : tok[0], my_head = second_tile ? head[RT - 1] : head[0];
    const bool my_valid = second_tile ? valid[RT - 1] : valid[0];
    const float lambda = a.maps.lambda[(long long)(my_valid ? my_tok : 0) * a.maps.lambda_stride + my_head];
    auto hand_over = [&](const f16v (&x)[MT], auto second) __attribute__((always_inline)) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            keep_sum_of<decltype(second)::value>(x[mt]);
#pragma unroll
            for (int vq = 0; vq < 4; ++vq) to_partner[(mt * 4 + vq) * 64] = f4{x[mt][4 * vq], x[mt][4 * vq + 1], x[mt][4 * vq + 2], x[mt][4 * vq + 3]};
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    if constexpr (RT == 2) {
        if (map) hand_over(o[0], std::true_type{});
        else hand_over(o[1], std::false_type{});
    } else if (map) {
        hand_over(o[0], std::true_type{});
    }
    sums[wave * 64 + lane] = map ? l[0] : l[RT - 1];
    __syncthreads();
    const float their_l = sums[(wave ^ 1) * 64 + lane];
    const float my_inv = my_l > 0.0f ? 1.0f / my_l : 0.0f, their_inv = their_l > 0.0f ? 1.0f / their_l : 0.0f;
    float squares = 0.0f;
    auto subtract = [&](const f16v (&x)[MT], auto second) __attribute__((always_inline)) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            keep_sum_of<decltype(second)::value>(x[mt]);
#pragma unroll
            for (int vq = 0; vq < 4; ++vq) {
                const f4 theirs = from_partner[(mt * 4 + vq) * 64];
                f4 d;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float mine = x[mt][4 * vq + e] * my_inv, other = theirs[e] * their_inv;
                    d[e] = decltype(second)::value ? map_difference(other, mine, lambda) : map_difference(mine, other, lambda);
                    squares += d[e] * d[e];
                }
                from_partner[(mt * 4 + vq) * 64] = d;  // (what this lane alone reads)
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    if constexpr (RT == 2) {
        if (map) subtract(o[1], std::true_type{});
        else subtract(o[0], std::false_type{});
    } else if (!map) {
        subtract(o[0], std::false_type{});
    }
    float scale = a.maps.out_scale;
    if (a.maps.norm) {
        squares = sum_across_halves(squares);
        scale *= squares == 0.0f ? 0.0f : 1.0f / sqrtf(squares * (1.0f / D) + a.maps.eps);
    }
    __syncthreads();  // (the sums of the weights have been read: their place is the rows')
    if (RT == 1 && map) return;
    // Norm weight and gate, and the rows out through LDS, 32 dims at a time: a store writes 64 bytes of 16 rows.
    char *const stage = smem + C::STAGE_OFF + (RT == 2 ? wave : pair) * C::STAGE_BYTES;
    const int out_row = lane >> 2, out_piece = lane & 3, tile_tok = my_tok - li;
    const global_halves gate_row = (global_halves)(a.gate + (long long)(my_valid ? my_tok : 0) * a.g_stride + (long long)my_head * D + 4 * g);
    h4 gate[4];
    uint16_t weight[16];
    auto load = [&](int mt) __attribute__((always_inline)) {
#pragma unroll
        for (int vq = 0; vq < 4; ++vq) {
            if (a.gate) gate[vq] = *(const __attribute__((address_space(1))) h4_unaligned *)(gate_row + 32 * mt + 8 * vq);
            if (a.maps.norm) {
#pragma unroll
                for (int e = 0; e < 4; ++e) weight[4 * vq + e] = a.maps.norm[32 * mt + 8 * vq + 4 * g + e];
            }
        }
    };
    load(0);
#pragma nounroll
    for (int mt = 0; mt < MT; ++mt) {
        f4 y[4];
#pragma unroll
        for (int vq = 0; vq < 4; ++vq) {
            y[vq] = from_partner[(mt * 4 + vq) * 64] * scale;
            if (a.maps.norm) {
#pragma unroll
                for (int e = 0; e < 4; ++e) y[vq][e] *= __builtin_bit_cast(float, (unsigned)weight[4 * vq + e] << 16);
            }
            if (a.gate) {
#pragma unroll
                for (int e = 0; e < 4; ++e) y[vq][e] *= sigmoid((float)gate[vq][e]);
            }
            const h4 x = {(_Float16)y[vq][0], (_Float16)y[vq][1], (_Float16)y[vq][2], (_Float16)y[vq][3]};
            *reinterpret_cast<h4 *>(stage + li * C::STAGE_PITCH + (8 * vq + 4 * g) * 2) = x;
        }
        if (mt + 1 < MT) load(mt + 1);
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int row = 16 * half + out_row, t = tile_tok + row;
            const h8 x = *reinterpret_cast<const h8 *>(stage + row * C::STAGE_PITCH + out_piece * 16);
            if (t < a.q_len) {
                _Float16 *const to = a.out + (long long)t * a.o_stride + (long long)my_head * D + 32 * mt + out_piece * 8;
                if (a.aligned) {
                    *reinterpret_cast<h8 *>(to) = x;
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) to[e] = x[e];
                }
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
}

template <int D>
hipError_t configure_chunk() {
    return hipFuncSetAttribute(reinterpret_cast<const void *>(attn_maps_chunk_kernel<D>), hipFuncAttributeMaxDynamicSharedMemorySize, ChunkShape<D>::LDS);
}

}  // namespace

int configure_maps_chunk_kernels(tt_hip_ctx *ctx) {
    hipError_t e = configure_chunk<256>();
    if (e == hipSuccess) e = configure_chunk<128>();
    if (e == hipSuccess) e = configure_chunk<64>();
    return e == hipSuccess ? TT_HIP_OK : hip_fail(ctx, e, "hipFuncSetAttribute(two-map chunk max dynamic LDS)");
}

int launch_maps_chunk(tt_hip_ctx *ctx, int head_dim, int n_kv_heads, const MapsChunk &c) {
    MapsChunkArgs a{};
    a.k_slot = c.pages.k;
    a.v_slot = c.pages.v;
    a.page_elems = c.pages.page_elems;
    a.ring_blocks = c.pages.ring_blocks;
    a.q = c.q;
    a.gate = c.gate;
    a.out = c.out;
    a.q_stride = c.q_stride;
    a.g_stride = c.g_stride;
    a.o_stride = c.o_stride;
    a.maps = c.maps;
    a.n_kv_heads = n_kv_heads;
    a.group = c.n_q_heads / n_kv_heads;
    a.hs = maps_chunk_heads(a.group);
    a.sets = a.group / a.hs;
    const int span = 128 / a.hs;
    a.tok_tiles = (c.q_len + span - 1) / span;
    a.start = c.start;
    a.q_len = c.q_len;
    a.kv_valid = c.kv_valid;
    a.window = c.window;
    a.scale_log2e = c.scale * 1.4426950408889634f;
    a.n_splits = c.n_splits;
    a.split_blocks = c.split_blocks;
    a.part_o = c.part_o;
    a.part_ml = c.part_ml;
    a.aligned = c.aligned;
    a.per_kvh = a.sets * a.tok_tiles * a.n_splits;
    a.xs = n_kv_heads <= 8 && 8 % n_kv_heads == 0 ? 8 / n_kv_heads : 0;
    const unsigned grid = a.xs > 0 ? 8u * (unsigned)((a.per_kvh + a.xs - 1) / a.xs) : (unsigned)(a.per_kvh * n_kv_heads);
    switch (head_dim) {
        case 256: launch_profiled(ctx, attn_maps_chunk_kernel<256>, dim3(grid), dim3(64 * ChunkShape<256>::WAVES), (unsigned)ChunkShape<256>::LDS, a); break;
        case 128: launch_profiled(ctx, attn_maps_chunk_kernel<128>, dim3(grid), dim3(64 * ChunkShape<128>::WAVES), (unsigned)ChunkShape<128>::LDS, a); break;
        case 64: launch_profiled(ctx, attn_maps_chunk_kernel<64>, dim3(grid), dim3(64 * ChunkShape<64>::WAVES), (unsigned)ChunkShape<64>::LDS, a); break;
        default: return TT_HIP_ERR_SHAPE;
    }
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? TT_HIP_OK : hip_fail(ctx, e, "attn_maps_chunk_kernel launch");
}

}  // namespace tt
