// The gradient of attention.  With p = exp(s - lse), s = scale q k^T, and the gradient d of the result,
//
//   delta[m] = sum_o d[m, o] out[m, o],   ds[m, n] = p[m, n] (sum_o d[m, o] v[n, o] - delta[m]),
//   grad_q = scale ds k,   grad_k = scale ds^T q,   grad_v = p^T d.
//
// Two kernels, each of which computes s and ds again from its operands: one owns rows and walks the keys (grad_q), one owns
// keys and walks the rows of all heads, and all entries, that share them (grad_k, grad_v).  Seven products instead of the five
// of one kernel, but every sum is made by one workgroup in a fixed order: no atomics, and no 32-bit gradient of the queries
// in memory.
//
// As in the forward kernel, a product's result registers are the next product's operand: the rows' kernel computes s^T[n, row]
// and multiplies K^T ds^T, the keys' kernel computes s[row, n] and multiplies d^T p and q^T ds.  p and ds are rounded to the
// operands' type for that.  In fp16, p is 2^15 times itself there, so that many keys of small weights keep their bits; ds, which is as it stands above, without the
// scale, has to lie between 6e-8 and 65504 in magnitude: gradients of the result want a loss scale that brings them there.
#pragma once

#include "attention.hpp"

namespace kmc {

template <typename T, int DP>
struct AttGradShape {
    static constexpr int ROW_BYTES = DP * static_cast<int>(sizeof(T));
    static constexpr int KEYS = ROW_BYTES <= 256 ? 64 : 32;         // per tile of the rows' kernel
    static constexpr int WAVES_PER_SIMD = ROW_BYTES <= 256 ? 2 : 1;
    static constexpr int WAVES_PER_SIMD_K = ROW_BYTES <= 128 ? 2 : 1;
    static constexpr int ROWS = 32;                                 // per tile of the keys' kernel
    static constexpr int PAIR = 2 * ROWS * AttLds<T, DP>::STRIDE;   // bytes of a tile of queries and one of gradients
    static constexpr int DEEP = PAIR <= 16384 ? 6 : PAIR <= 32768 ? 4 : 2;      // buffers for them that fit LDS (twice, where two workgroups share a CU)
};

// p of a score from the row's statistics.
__device__ __forceinline__ float att_weight(float s, float scale_log2, float lse2) { return __builtin_amdgcn_exp2f(__builtin_fmaf(s, scale_log2, -lse2)); }

// An lse of this size or more (4096 to base 2) is not exact enough for p = exp(s - lse): fp32 rounds it, and its product with log2(e), to 2^-12 or worse each, which
// p is then off by as a factor; at 2^30 that factor is any power of two up to 2^64.  The queries' kernel walks the keys of such rows once more in front, for the
// largest score, the sum of the exponentials relative to it and delta; p is then exp2((s - largest) scale_log2 - log2(sum)), as in the forward kernel.
constexpr float ATT_LARGEST_LSE = ATT_LARGEST_BASE * ATT_LN_2;

// Powers of two in the keys' kernel, where p is an operand: p times 2^LIFT, which is at most 2^15 in fp16; the sums of grad_v and the factor of ds take it out.
template <typename T> constexpr float ATT_GRAD_LIFT = std::is_same<T, _Float16>::value ? 15.0f : 0.0f;
template <typename T> constexpr float ATT_GRAD_LOWER = std::is_same<T, _Float16>::value ? 0x1p-15f : 1.0f;

// lse to base 2 for the exponentials; a row without keys gets +inf, which makes all its weights 0.
__device__ __forceinline__ float att_lse2(float lse) { return lse == -__builtin_inff() ? __builtin_inff() : lse * ATT_LOG2_E; }

// Two products of 32 rows of two tiles in LDS with operands of the wave's own, by turns: s (scores) and ds (gradients of the result times values).
// Between the matrix instructions, with VECTOR, the vector work of the scores before: `quad(q)` makes the weights of registers
// 4 q .. 4 q + 3.
template <typename T, int DP, bool ORDERED, bool VECTOR, bool BOTH = true, typename Quad>
__device__ __forceinline__ void att_two_scores(att_f32x16 &s, att_f32x16 &ds, const att_lds_byte *s_tile, const att_vec8<T> (&s_own)[DP / 16],
                                               const att_lds_byte *ds_tile, const att_vec8<T> (&ds_own)[DP / 16], int lane, Quad quad)
{
    typedef AttGroups<T, DP> G;
    constexpr int AT_ONCE = DP * sizeof(T) > 512 ? 1 : 2, ALL = G::STEPS / AT_ONCE;
    att_vec8<T> f[2][2 * AT_ONCE];
    auto read = [&](att_vec8<T> (&to)[2 * AT_ONCE], int i) {
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j) {
            to[2 * j] = att_read_row<T, DP>(s_tile, 0, 16 * (AT_ONCE * i + j), lane);
            if (BOTH) to[2 * j + 1] = att_read_row<T, DP>(ds_tile, 0, 16 * (AT_ONCE * i + j), lane);
        }
    };
    read(f[0], 0);
    s = ds = att_f32x16{0};
    att_region<ORDERED>();
#pragma unroll
    for (int i = 0; i < ALL; ++i) {
        if (i + 1 < ALL) read(f[(i + 1) & 1], i + 1);
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j) {
            s = att_mma(f[i & 1][2 * j], s_own[AT_ONCE * i + j], s);
            if (BOTH) ds = att_mma(f[i & 1][2 * j + 1], ds_own[AT_ONCE * i + j], ds);
        }
        if (VECTOR)
#pragma unroll
            for (int q = 4 * i / ALL; q < 4 * (i + 1) / ALL; ++q) quad(q);
        att_order<ORDERED, 2 * AT_ONCE * G::READS_ROW, 2 * AT_ONCE * G::MMAS, VECTOR ? (sizeof(T) == 4 ? 1 : 48 / (2 * G::STEPS) + 1) : 0>();
        att_region<ORDERED>();
    }
}

// A workgroup per (batch entry, head of keys, range of keys, 128 rows); a wave per 32 rows, whose queries and gradients it keeps in registers.
// Three products, two of which share what is read of a tile: 1.47 ms at 4 x 4096 x 4096, 32 heads on 8 x 128 bf16, the matrix cores busy 59 % of the time.
template <typename T, int DP, bool ALIGNED, bool ORDERED = ATT_ORDERED<T, DP, ALIGNED>>
__global__ __launch_bounds__(256, (AttGradShape<T, DP>::WAVES_PER_SIMD)) void attention_grad_queries(const AttentionGradArgs args)
{
    typedef AttGradShape<T, DP> Shape;
    constexpr int KT = Shape::KEYS;
    constexpr int TILE = KT * AttLds<T, DP>::STRIDE;
    __shared__ __attribute__((aligned(1024))) att_lds_byte lds[4 * TILE];       // keys and values, two tiles of each
    __shared__ float shifts[128];               // with `large`, of the rows: not in a register that the loop holds
    __shared__ int large_rows[4];               // of the waves
    const int lane = threadIdx.x & 63, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int block = static_cast<int>(blockIdx.x) + args.first_block;
    int id = (block & 7) * (args.q_grid >> 3) + (block >> 3);
    if (id >= args.q_workgroups) return;
    const int row_tile = id % args.q_row_tiles;
    id /= args.q_row_tiles;
    const int split = id % args.q_splits;
    id /= args.q_splits;
    const int entry = id % args.l, g = id / args.l;             // one head of all entries, whose lengths differ, on an XCD

    const int rows = args.m * args.r;
    const int first_row = row_tile * 128 + 32 * wave, row = first_row + lane % 32;
    const bool works = first_row < rows;
    const int token = (row < rows ? row : 0) / args.r, head = g * args.r + (row < rows ? row : 0) % args.r;
    const i64 at = (static_cast<i64>(entry) * args.m + token) * (static_cast<i64>(args.g) * args.r) + head;
    const T *q = static_cast<const T *>(args.q) + entry * args.q_ls + token * args.q_ms + head * args.q_hs;
    const T *d = static_cast<const T *>(args.grad_out) + entry * args.grad_out_ls + token * args.grad_out_ms + head * args.grad_out_hs;
    const T *out = static_cast<const T *>(args.out) + entry * args.out_ls + token * args.out_ms + head * args.out_hs;

    const float lse = args.lse[at];
    att_vec8<T> query[DP / 16], grad[DP / 16];
    float delta = 0.0f;
#pragma unroll
    for (int step = 0; step < DP / 16; ++step) {
        query[step] = att_load8<T, ALIGNED>(q, 16 * step + 8 * half, args.k);
        if (args.query_factor != 1.0f)
#pragma unroll
            for (int j = 0; j < 8; ++j) query[step][j] = static_cast<T>(static_cast<float>(query[step][j]) * args.query_factor);
        grad[step] = att_load8<T, ALIGNED>(d, 16 * step + 8 * half, args.o);
        const att_vec8<T> result = att_load8<T, ALIGNED>(out, 16 * step + 8 * half, args.o);
#pragma unroll
        for (int j = 0; j < 8; ++j) delta = __builtin_fmaf(static_cast<float>(grad[step][j]), static_cast<float>(result[j]), delta);
    }
    delta = att_sum_of_halves(delta);
    float lse2 = att_lse2(lse), shift = 0.0f;
    bool large = false;                         // one of the workgroup's 128 rows has a large lse
    if (args.row_shift) {
        const bool mine = __any(!(fabsf(lse) < ATT_LARGEST_LSE) && lse != -__builtin_inff());
        if (lane == 0) large_rows[wave] = mine;
        __syncthreads();
        large = __builtin_amdgcn_readfirstlane(large_rows[0] | large_rows[1] | large_rows[2] | large_rows[3]) != 0;
    }

    const AttentionKeys &keys = args.keys;
    const int length = att_length(keys, entry);
    int begin, end;
    att_range(length, KT, split, args.q_splits, &begin, &end);
    const bool one_tile = length <= KT;
    const i64 rows_total = static_cast<i64>(args.l) * args.m * args.g * args.r;
    const T *k = static_cast<const T *>(keys.k) + entry * keys.k_ls + g * keys.k_gs;
    const T *v = static_cast<const T *>(keys.v) + entry * keys.v_ls + g * keys.v_gs;
    AttTile<T, DP, KT, 256, ALIGNED> next_k, next_v;
    if ((one_tile || large) && begin < end) {
        // Few keys: delta from the rounded result would be off by as much as ds is large, so it is summed from the weights themselves,
        // which are normalised again while they are at hand (a single key's weight is exactly 1, its ds exactly 0).
        float top = -__builtin_inff(), total = 0.0f, inner = 0.0f;
#pragma unroll 1
        for (int n = 0; n < length; n += KT) {
            const att_u64 kept = att_kept_keys(keys, entry, n, length, lane);
            if (n > 0) __syncthreads();                 // the tile before has been read
            next_k.begin(k + n * keys.k_ns, keys.k_ns, length - n, args.k, lds, threadIdx.x, kept);
            next_v.begin(v + n * keys.v_ns, keys.v_ns, length - n, args.o, lds + TILE, threadIdx.x, kept);
            next_k.finish(lds, threadIdx.x);
            next_v.finish(lds + TILE, threadIdx.x);
            __syncthreads();
#pragma unroll 1
            for (int b = 0; b < KT / 32 && 32 * b < length - n; ++b) {
                att_f32x16 s = {0}, ds = {0};
#pragma unroll
                for (int step = 0; step < DP / 16; ++step) {
                    s = att_mma(att_read_row<T, DP>(lds, 32 * b, 16 * step, lane), query[step], s);
                    ds = att_mma(att_read_row<T, DP>(lds + TILE, 32 * b, 16 * step, lane), grad[step], ds);
                }
                const unsigned mine = static_cast<unsigned>(kept >> (32 * b)) >> (4 * half);
                float from = 0.0f, base = lse2;
                if (large) {                            // weights relative to the largest score so far
                    float block_top = -__builtin_inff();
#pragma unroll
                    for (int i = 0; i < 16; ++i) block_top = fmaxf(block_top, mine >> att_row(i, 0) & 1 ? s[i] : -__builtin_inff());
                    block_top = att_max_of_halves(block_top);
                    if (block_top > top) {
                        const float shrink = __builtin_amdgcn_exp2f((top - block_top) * args.scale_log2);
                        total *= shrink;
                        inner *= shrink;
                        top = block_top;
                    }
                    from = top == -__builtin_inff() ? 0.0f : top;
                    base = 0.0f;
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const bool counts = mine >> att_row(i, 0) & 1;
                    const float p = !counts ? 0.0f : length == 1 ? 1.0f : att_weight(s[i] - from, args.scale_log2, base);
                    total += p;
                    inner = counts ? __builtin_fmaf(p, ds[i], inner) : inner;
                }
            }
        }
        total = att_sum_of_halves(total);
        inner = att_sum_of_halves(inner);
        if (total == 0.0f) {
            lse2 = __builtin_inff();
        } else {
            delta = inner / total;
            shift = large ? top : 0.0f;
            lse2 = (large ? 0.0f : lse2) + (length > 1 ? __builtin_amdgcn_logf(total) : 0.0f);
        }
    }
    if (lse2 == __builtin_inff()) delta = 0.0f;         // (no key: the gradient is 0 whatever that of the result is)
    if (block == 0 && threadIdx.x == 0) {               // for rows that do not exist: weights of 0
        args.stats[2 * rows_total] = __builtin_inff();
        args.stats[2 * rows_total + 1] = 0.0f;
    }
    if (split == 0 && row < rows && half == 0) {
        float *stats = args.stats + (static_cast<i64>(entry) * args.g * args.r + head) * args.m + token;
        stats[0] = lse2 - ATT_GRAD_LIFT<T>;
        stats[rows_total] = delta * ATT_GRAD_LOWER<T>;
        if (args.row_shift) args.row_shift[stats - args.stats] = shift;
    }
    if (args.row_flags && split == 0 && threadIdx.x == 0) args.row_flags[(static_cast<i64>(entry) * args.g + g) * args.q_row_tiles + row_tile] = large;
    att_f32x16 acc[DP / 32];
#pragma unroll
    for (int o = 0; o < DP / 32; ++o) acc[o] = att_f32x16{0};
    if ((DP > 128 || large) && half == 0) shifts[32 * wave + lane] = shift;
    int odd = 0;
    att_wait_for_loads();
    const i64 k_stride = keys.k_ns, v_stride = keys.v_ns;
    const int k_width = args.k, v_width = args.o;
    const bool masked = keys.mask != nullptr;
    const float scale_log2 = args.scale_log2;
    auto ask = [&](i64 n, att_lds_byte *to, att_u64 kept) {
        const int some = end - static_cast<int>(n);
        if (masked) {
            next_k.begin(k + n * k_stride, k_stride, some, k_width, to, threadIdx.x, kept);
            next_v.begin(v + n * v_stride, v_stride, some, v_width, to + TILE, threadIdx.x, kept);
        } else {
            next_k.begin(k + n * k_stride, k_stride, some, k_width, to, threadIdx.x);
            next_v.begin(v + n * v_stride, v_stride, some, v_width, to + TILE, threadIdx.x);
        }
    };
    auto ask_kept = [&](i64 n) { return masked && n < end ? att_ask_kept(keys, entry, static_cast<int>(n), end, lane) : 0; };
    att_u64 kept = masked ? __ballot(ask_kept(begin) != 0) : att_low_bits(end - begin), then_kept;
    int next_kept = ask_kept(static_cast<i64>(begin) + KT);
    if (begin < end) {
        __syncthreads();
        ask(begin, lds, kept);
    }
    for (int n = begin; n < end; n += KT, odd ^= 1, kept = then_kept) {
        then_kept = masked ? __ballot(next_kept != 0) : att_low_bits(end - n - KT);
        next_kept = ask_kept(static_cast<i64>(n) + 2 * KT);
        att_lds_byte *key_tile = lds + 2 * odd * TILE, *value_tile = key_tile + TILE;
        next_k.finish(key_tile, threadIdx.x);
        next_v.finish(value_tile, threadIdx.x);
        __syncthreads();
        if (n + KT < end) ask(n + KT, lds + 2 * (odd ^ 1) * TILE, then_kept);
        if (!works) continue;
        // (overlapping the blocks, as the keys' kernel does with its tiles, takes more registers than two waves per SIMD have: 1.77 instead of 1.53 ms at
        // 4 x 4096 x 4096 x 32 heads of 128)
#pragma unroll
        for (int b = 0; b < KT / 32; ++b) {
            if (b > 0 && 32 * b >= end - n) break;
            constexpr int BLOCK = 32 * AttLds<T, DP>::STRIDE;
            att_f32x16 s, ds;
            typedef AttGroups<T, DP> G;
            att_vec8<T> x[2], f[2][G::COLUMNS];
            const att_lds_byte *block = key_tile + b * BLOCK;
            att_two_scores<T, DP, ORDERED, false>(s, ds, block, query, value_tile + b * BLOCK, grad, lane, [](int) {});
            att_read_columns<T, DP>(f[0], block, 0, 0, lane);
            const unsigned here = static_cast<unsigned>(kept >> (32 * b));
            if constexpr (DP > 128) {
                // (a branch in front of the weights costs these kernels more than 16 subtractions: 526 us instead of 590 in fp32 of 256 features, 2 x 1000 x 1500 x 8 heads)
                s -= shifts[32 * wave + lane % 32];
#pragma unroll
                for (int i = 0; i < 16; ++i) ds[i] = att_weight(s[i], scale_log2, lse2) * (ds[i] - delta);
                if (here != ~0u) {
                    att_rare();
                    const unsigned rows = __builtin_amdgcn_readfirstlane(here);
#pragma unroll
                    for (int i = 0; i < 16; ++i) ds[i] = att_has_row(rows, i) ? ds[i] : 0.0f;
                }
            } else {
                if (large || here != ~0u) {
                    att_rare();
                    const unsigned rows = __builtin_amdgcn_readfirstlane(here);
                    if (large) s -= shifts[32 * wave + lane % 32];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        s[i] = att_has_row(rows, i) ? s[i] : -__builtin_inff();
                        ds[i] = att_has_row(rows, i) ? ds[i] : 0.0f;
                    }
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) ds[i] = att_weight(s[i], scale_log2, lse2) * (ds[i] - delta);
            }
            x[0] = att_operand<T>(ds, 0);
            x[1] = att_operand<T>(ds, 1);
#pragma unroll
            for (int i = 0; i < 2 * G::COLUMN_GROUPS; ++i) {
                const int step = i / G::COLUMN_GROUPS, group = i % G::COLUMN_GROUPS;
                if (i + 1 < 2 * G::COLUMN_GROUPS)
                    att_read_columns<T, DP>(f[(i + 1) & 1], block, 16 * ((i + 1) / G::COLUMN_GROUPS), (i + 1) % G::COLUMN_GROUPS, lane);
#pragma unroll
                for (int o = 0; o < G::COLUMNS; ++o) acc[G::COLUMNS * group + o] = att_mma(f[i & 1][o], x[step], acc[G::COLUMNS * group + o]);
                if (G::COLUMN_GROUPS > 1) {
                    att_order<ORDERED, G::COLUMNS * G::READS_T, G::COLUMNS * G::MMAS, 0>();
                    att_region<ORDERED>();
                }
            }
        }
    }
    if (row >= rows) return;
    if (args.q_splits > 1) {
        float *to = args.partial_q + (split * rows_total + at) * args.partial_k_width;
#pragma unroll
        for (int o = 0; o < DP / 32; ++o)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (32 * o + att_row(i, half) < args.k) to[32 * o + att_row(i, half)] = acc[o][i];
        return;
    }
    T *to = static_cast<T *>(args.grad_q) + at * args.k;
    att_store_columns<T, DP, ALIGNED>(to, acc, args.scale, args.k, half);
}

// A workgroup per (entry of the keys, head of keys, part of the rows, 128 keys); a wave per 32 keys, whose keys and values it keeps in registers.
//
// Turn i: the scores of tile i + 1 (32 rows) on the matrix cores while the vector units make the weights and gradients of tile i from its scores, then
// the two products of tile i.  Behind the buffers of these two tiles stand as many as fit for those on their way: the workgroups of a head walk its rows in step,
// so every tile comes from far, and one turn is shorter than that takes (4 x 4096 x 4096, 32 heads on 8 x 128 bf16: 4.2 ms with one tile on its way, 2.6
// with four; one wave per SIMD, whose 64 KB of keys, values and their gradients fill its registers).  What bounds it with 128 features is that one wave's work follows
// its own: the matrix cores are busy 39 % of the time, LDS, of which every wave reads each tile twice by rows and twice by columns, 24 %, vector instructions 29 %.
// Waves with 64 keys would halve the reads, and have no registers for it (3.4 ms, with spills whose reloads wait for the tiles on their way); a barrier after two
// tiles instead of one changes nothing.  With 64 features, 8 x 1000 x 1500 keys at most x 16 heads, 115 us: the matrix cores are busy 23 % of the time, vector instructions 28 %.
//
// In fp32, 32 keys and values of more than 128 features and their gradients are 512 registers by themselves.  There a launch makes one of the two gradients, and
// the scores are computed twice (2 x 1000 x 1500 x 8 heads of 256: 800 us for both, 1180 in one launch with its spills).
enum AttKeysPart { ATT_BOTH, ATT_GRAD_KEYS, ATT_GRAD_VALUES };

template <typename T, int DP, bool ALIGNED, AttKeysPart PART, bool ORDERED = ATT_ORDERED<T, DP, ALIGNED>>
__global__ __launch_bounds__(256, (AttGradShape<T, DP>::WAVES_PER_SIMD_K)) void attention_grad_keys(const AttentionGradArgs args)
{
    typedef AttGradShape<T, DP> Shape;
    typedef AttGroups<T, DP> G;
    constexpr int RT = Shape::ROWS, TILE = RT * AttLds<T, DP>::STRIDE;
    typedef AttTile<T, DP, RT, 256, ALIGNED> Tile;
    constexpr bool OF_KEYS = PART != ATT_GRAD_VALUES, OF_VALUES = PART != ATT_GRAD_KEYS;
    constexpr int BUFFERS = Tile::DIRECT || Shape::DEEP == 2 ? Shape::DEEP : 3;
    constexpr bool OVERLAP = DP <= 128;                                 // (wider rows leave no registers for the scores of two tiles)
    constexpr int AHEAD = BUFFERS - (OVERLAP ? 2 : 1);                  // tiles on their way behind those in use
    static_assert(AHEAD > 0, "a tile on its way");
    static_assert(!OVERLAP || PART == ATT_BOTH, "a part walks one tile at a time");
    constexpr int LOADS = 2 * Tile::PER_THREAD + 1;                     // of a wave for a tile
    __shared__ __attribute__((aligned(1024))) att_lds_byte lds[2 * BUFFERS * TILE];     // queries and gradients of the result
    __shared__ __attribute__((aligned(256))) float all_stats[BUFFERS][2 * RT];           // lse to base 2 and delta of a tile's rows
    const unsigned stats_lds = att_lds_address(all_stats);
    const int lane = threadIdx.x & 63, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int block = static_cast<int>(blockIdx.x) + args.first_block;
    int id = (block & 7) * (args.k_grid >> 3) + (block >> 3);
    if (id >= args.k_workgroups) return;
    const int key_tile = id % args.key_tiles;
    id /= args.key_tiles;
    const int split = id % args.k_splits;
    id /= args.k_splits;
    const int key_entry = id % args.key_entries, g = id / args.key_entries;

    const AttentionKeys &keys = args.keys;
    const int first_key = key_tile * 128, n = first_key + 32 * wave + lane % 32;
    const bool exists = n < keys.n;
    const T *k = static_cast<const T *>(keys.k) + key_entry * keys.k_ls + (exists ? n : 0) * keys.k_ns + g * keys.k_gs;
    const T *v = static_cast<const T *>(keys.v) + key_entry * keys.v_ls + (exists ? n : 0) * keys.v_ns + g * keys.v_gs;
    att_vec8<T> key[DP / 16], value[DP / 16];
#pragma unroll
    for (int step = 0; step < DP / 16; ++step) {
        key[step] = att_load8<T, ALIGNED>(k, 16 * step + 8 * half, args.k);
        if (args.query_factor != 1.0f)
#pragma unroll
            for (int j = 0; j < 8; ++j) key[step][j] = static_cast<T>(static_cast<float>(key[step][j]) * args.query_factor);
        if (OF_KEYS) value[step] = att_load8<T, ALIGNED>(v, 16 * step + 8 * half, args.o);
    }
    // the rows: entries that share the keys, their heads, 32 queries at a time; this workgroup's part of them
    const int tiles_m = (args.m + RT - 1) / RT;
    const i64 per_entry = static_cast<i64>(args.r) * tiles_m;
    const int entries = args.key_entries == args.l ? 1 : args.l;
    const i64 per_split = (per_entry * entries + args.k_splits - 1) / args.k_splits;
    const float scale_log2 = args.scale_log2;
    const i64 part_first = split * per_split, part_last = part_first + per_split;
    const i64 rows_total = static_cast<i64>(args.l) * args.m * args.g * args.r;
    bool ever_kept = false;
    // not 0 if a row of an entry and this head of keys has a shift
    auto ask_large = [&](int e) {
        int some = 0;
        if (args.row_flags && e < entries)
            for (int i = lane; i < args.q_row_tiles; i += 64) some |= args.row_flags[(static_cast<i64>(key_entry + e) * args.g + g) * args.q_row_tiles + i];
        return some;
    };
    const int first_entry = static_cast<int>(part_first / per_entry);
    int some_large = ask_large(first_entry);
    att_wait_for_loads();
    att_f32x16 acc_k[DP / 32], acc_v[DP / 32];
#pragma unroll
    for (int o = 0; o < DP / 32; ++o) acc_k[o] = acc_v[o] = att_f32x16{0};

    for (int e = first_entry; e < entries && e * per_entry < part_last; some_large = ask_large(++e)) {
        const int entry = key_entry + e;
        const int first = static_cast<int>(part_first > e * per_entry ? part_first - e * per_entry : 0);
        const int count = static_cast<int>((part_last < (e + 1) * per_entry ? part_last - e * per_entry : per_entry) - first);
        const bool large = __any(some_large != 0);
        const int length = att_length(keys, entry);
        const att_u64 kept_keys[2] = {att_kept_keys(keys, entry, first_key, length, lane), att_kept_keys(keys, entry, first_key + 64, length, lane)};
        if (!(kept_keys[0] | kept_keys[1])) continue;
        // A key that does not take part has a column of the products of its own, whatever it holds: its gradient is set to zero at the end, unless another entry
        // that shares it adds to it.
        const bool kept = static_cast<unsigned>(kept_keys[wave >> 1] >> (32 * (wave & 1))) >> (lane & 31) & 1;
        const bool clear = entries > 1 && !__all(kept);
        ever_kept |= kept;

        // What moves from tile to tile: addresses in scalar registers that grow by one of two steps.
        Tile next_q, next_d;
        constexpr int SIZE = static_cast<int>(sizeof(T));
        const int m = args.m, q_width = args.k, d_width = args.o;
        int m0 = first % tiles_m * RT, to = 0, left = count;                    // of the next tile to load
        const int head = g * args.r + first / tiles_m, last_m0 = (tiles_m - 1) * RT;
        att_u64 q_at = att_uniform(static_cast<const T *>(args.q) + entry * args.q_ls + m0 * args.q_ms + head * args.q_hs);
        att_u64 d_at = att_uniform(static_cast<const T *>(args.grad_out) + entry * args.grad_out_ls + m0 * args.grad_out_ms + head * args.grad_out_hs);
        const i64 q_next = RT * args.q_ms * SIZE, q_wrap = (args.q_hs - last_m0 * args.q_ms) * SIZE;
        const i64 d_next = RT * args.grad_out_ms * SIZE, d_wrap = (args.grad_out_hs - last_m0 * args.grad_out_ms) * SIZE;
        const int q_step = static_cast<int>(args.q_ms) * SIZE, d_step = static_cast<int>(args.grad_out_ms) * SIZE;
        const float *stats_at = args.stats + (static_cast<i64>(entry) * args.g * args.r + head) * m + m0 + (lane < RT ? 0 : rows_total) + lane % RT;
        const float *const stats_behind = args.stats + 2 * rows_total + (lane < RT ? 0 : 1);
        auto begin = [&]() {
            const bool last = m0 == last_m0;
            const int some = left <= 0 ? 0 : last ? m - last_m0 : RT;           // (behind the last tile: nothing is read)
            att_lds_byte *q_tile = lds + 2 * to * TILE;
            if constexpr (Tile::DIRECT) {
                next_q.begin_at(att_descriptor<T>(q_at, q_step, some, q_width), q_step, q_width, q_tile, threadIdx.x);
                next_d.begin_at(att_descriptor<T>(d_at, d_step, some, d_width), d_step, d_width, q_tile + TILE, threadIdx.x);
            } else {
                next_q.begin(reinterpret_cast<const T *>(q_at), args.q_ms, some, q_width, q_tile, threadIdx.x);
                next_d.begin(reinterpret_cast<const T *>(d_at), args.grad_out_ms, some, d_width, q_tile + TILE, threadIdx.x);
            }
            // (all waves load the same: they count the same loads; rows that do not exist get the pair behind all others)
            att_load_words(lane % RT < some ? stats_at : stats_behind, stats_lds + 8 * RT * to);
            --left;
            m0 = last ? 0 : m0 + RT;
            q_at += last ? q_wrap : q_next;
            d_at += last ? d_wrap : d_next;
            stats_at += last ? m - last_m0 : RT;
            if (Tile::DIRECT) to = to + 1 == BUFFERS ? 0 : to + 1;
        };
        // The tile asked for longest ago has arrived; AHEAD - 1 others may be on their way.
        auto finish = [&]() {
            if constexpr (Tile::DIRECT) {
                att_wait_for_loads<(AHEAD - 1) * LOADS>();
            } else {
                att_wait_for_loads();
                att_lds_byte *q_tile = lds + 2 * to * TILE;
                next_q.finish(q_tile, threadIdx.x);
                next_d.finish(q_tile + TILE, threadIdx.x);
                to = to + 1 == BUFFERS ? 0 : to + 1;
            }
        };
        int now = 0;                    // the buffer of the current tile
        auto then = [&]() { return now + 1 == BUFFERS ? 0 : now + 1; };
        att_f32x16 s_a, ds_a, s_b, ds_b;
        att_vec8<T> p[2], x[2];
        float weight[16];
        // of the tile whose weights are made next
        int shift_m0 = m0;
        const float *shift_at = args.row_shift + (static_cast<i64>(entry) * args.g * args.r + head) * m + m0;
        auto shift_scores = [&](att_f32x16 &s) {
            if (!large) return;
            att_rare();
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] -= shift_m0 + att_row(i, half) < m ? shift_at[att_row(i, half)] : 0.0f;
            const bool last = shift_m0 == last_m0;
            shift_at += last ? m - last_m0 : RT;
            shift_m0 = last ? 0 : shift_m0 + RT;
        };
        auto make_weights = [&](const att_f32x16 &s, int q) {
            const att_f32x4 lse2 = *reinterpret_cast<const att_f32x4 *>(all_stats[now] + 8 * q + 4 * half);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                weight[4 * q + j] = att_weight(s[4 * q + j], scale_log2, lse2[j]);
                p[q / 2][4 * (q % 2) + j] = static_cast<T>(weight[4 * q + j]);
            }
        };
        auto make_gradients = [&](const att_f32x16 &ds, int q) {
            const att_f32x4 delta = *reinterpret_cast<const att_f32x4 *>(all_stats[now] + RT + 8 * q + 4 * half);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                x[q / 2][4 * (q % 2) + j] = static_cast<T>(weight[4 * q + j] * __builtin_fmaf(ds[4 * q + j], ATT_GRAD_LOWER<T>, -delta[j]));
        };
        auto products = [&](att_f32x16 &ds) {
            const att_lds_byte *q_tile = lds + 2 * now * TILE, *d_tile = q_tile + TILE;
            if (clear) {
                unsigned keep = kept ? ~0u : 0u;
                asm volatile("" : "+v"(keep));              // (nothing of this is made in front of the branch)
                typedef unsigned words __attribute__((ext_vector_type(sizeof(att_vec8<T>) / 4)));
#pragma unroll
                for (int step = 0; step < 2; ++step) p[step] = __builtin_bit_cast(att_vec8<T>, __builtin_bit_cast(words, p[step]) & keep);
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float w = weight[i], d = ds[i];               // (of an element of a vector, the builtin takes the first)
                    weight[i] = __builtin_bit_cast(float, __builtin_bit_cast(unsigned, w) & keep);
                    ds[i] = __builtin_bit_cast(float, __builtin_bit_cast(unsigned, d) & keep);
                }
            }
            // four steps of 16 rows: two of the gradients, two of the queries
            constexpr int FIRST = OF_VALUES ? 0 : 2 * G::COLUMN_GROUPS, ALL = OF_KEYS ? 4 * G::COLUMN_GROUPS : 2 * G::COLUMN_GROUPS;
            if (!OF_VALUES)
#pragma unroll
                for (int q = 0; q < 4; ++q) make_gradients(ds, q);
            att_vec8<T> f[2][G::COLUMNS];
            auto read = [&](att_vec8<T> (&to)[G::COLUMNS], int i) {
                const int step = i / G::COLUMN_GROUPS;
                att_read_columns<T, DP>(to, step < 2 ? d_tile : q_tile, 16 * (step % 2), i % G::COLUMN_GROUPS, lane);
            };
            read(f[0], FIRST);
            att_region<ORDERED>();
#pragma unroll
            for (int i = FIRST; i < ALL; ++i) {
                const int step = i / G::COLUMN_GROUPS, group = i % G::COLUMN_GROUPS;
                if (i + 1 < ALL) read(f[(i + 1) & 1], i + 1);
#pragma unroll
                for (int o = 0; o < G::COLUMNS; ++o) {
                    att_f32x16 &to = step < 2 ? acc_v[G::COLUMNS * group + o] : acc_k[G::COLUMNS * group + o];
                    to = att_mma(f[i & 1][o], step < 2 ? p[step] : x[step - 2], to);
                }
                if (OF_KEYS && step < 2 && group == 0) {
                    make_gradients(ds, 2 * step);
                    make_gradients(ds, 2 * step + 1);
                    att_order<ORDERED, G::COLUMNS * G::READS_T, G::COLUMNS * G::MMAS, (G::MMAS > 1 ? 2 : 24 / G::COLUMNS)>();
                } else {
                    att_order<ORDERED, G::COLUMNS * G::READS_T, G::COLUMNS * G::MMAS, 0>();
                }
                att_region<ORDERED>();
            }
        };
        auto next_tile = [&]() {
            finish();
            __syncthreads();
            now = then();
        };
        auto turn = [&](att_f32x16 &s, att_f32x16 &ds, att_f32x16 &next_s, att_f32x16 &next_ds) {
            shift_scores(s);
            begin();
            const att_lds_byte *q_tile = lds + 2 * then() * TILE;
            att_two_scores<T, DP, ORDERED, true>(next_s, next_ds, q_tile, key, q_tile + TILE, value, lane, [&](int q) { make_weights(s, q); });
            products(ds);
            next_tile();
        };

        __syncthreads();                // an entry before this one is done with the buffers
#pragma unroll 1
        for (int i = 0; i < BUFFERS - 1; ++i) {
            begin();
            if (!Tile::DIRECT) finish();
        }
        att_wait_for_loads();
        __syncthreads();
        if constexpr (OVERLAP) {
            att_two_scores<T, DP, ORDERED, false>(s_a, ds_a, lds, key, lds + TILE, value, lane, [](int) {});
            int i = 1;
            for (; i + 1 < count; i += 2) {
                turn(s_a, ds_a, s_b, ds_b);
                turn(s_b, ds_b, s_a, ds_a);
            }
            if (i < count) {
                turn(s_a, ds_a, s_b, ds_b);
                s_a = s_b;
                ds_a = ds_b;
            }
            shift_scores(s_a);
#pragma unroll
            for (int q = 0; q < 4; ++q) make_weights(s_a, q);
            products(ds_a);
        } else {
#pragma unroll 1
            for (int i = 0; i < count; ++i) {
                begin();
                const att_lds_byte *q_tile = lds + 2 * now * TILE;
                att_two_scores<T, DP, ORDERED, false, OF_KEYS>(s_a, ds_a, q_tile, key, q_tile + TILE, value, lane, [](int) {});
                shift_scores(s_a);
#pragma unroll
                for (int q = 0; q < 4; ++q) make_weights(s_a, q);
                products(ds_a);
                next_tile();
            }
        }
        att_wait_for_loads();
    }
    if (!exists) return;
    if (!ever_kept)
#pragma unroll
        for (int o = 0; o < DP / 32; ++o) acc_k[o] = acc_v[o] = att_f32x16{0};
    const i64 at = (static_cast<i64>(key_entry) * keys.n + n) * args.g + g;
    if (args.k_splits > 1) {
        const i64 slot = split * (static_cast<i64>(args.key_entries) * keys.n * args.g) + at;
        float *to_k = args.partial_k + slot * args.partial_k_width, *to_v = args.partial_v + slot * args.partial_o_width;
#pragma unroll
        for (int o = 0; o < DP / 32; ++o)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int column = 32 * o + att_row(i, half);
                if (OF_KEYS && column < args.k) to_k[column] = acc_k[o][i];
                if (OF_VALUES && column < args.o) to_v[column] = acc_v[o][i];
            }
        return;
    }
    if (OF_KEYS) att_store_columns<T, DP, ALIGNED>(static_cast<T *>(args.grad_k) + at * args.k, acc_k, args.scale, args.k, half);
    if (OF_VALUES) att_store_columns<T, DP, ALIGNED>(static_cast<T *>(args.grad_v) + at * args.o, acc_v, ATT_GRAD_LOWER<T>, args.o, half);
}

// The parts of a cut gradient, added in their order.
template <typename T>
__global__ __launch_bounds__(256) void attention_sum(const AttentionSumArgs args)
{
    const i64 step = static_cast<i64>(gridDim.x) * 256;
    for (i64 i = static_cast<i64>(blockIdx.x) * 256 + threadIdx.x; i < args.first[3]; i += step) {
        const int which = i >= args.first[2] ? 2 : i >= args.first[1] ? 1 : 0;
        const AttentionSum &sum = args.part[which];
        const i64 at = i - args.first[which];
        const float *from = sum.partial + at / sum.width * sum.partial_width + at % sum.width;
        const i64 stride = sum.rows * sum.partial_width;
        float total = 0.0f;
#pragma unroll 8
        for (int part = 0; part < sum.splits; ++part) total += from[part * stride];
        static_cast<T *>(sum.out)[at] = static_cast<T>(total * sum.factor);
    }
}

}  // namespace kmc
