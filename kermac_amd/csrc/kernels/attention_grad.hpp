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
// operands' type for that (ds in fp16 keeps numbers down to 6e-8: gradients far below 1e-4 want the usual loss scaling).
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
    static constexpr int BOTH = ATT_STRIDE<T, DP> + ATT_STRIDE_T<T, DP>;        // a row as it is, and one to be read transposed
};

// ds of a 32 x 32 result from scores, d v^T, and the row's statistics: p comes back in `s`.
__device__ __forceinline__ float att_weight(float s, float scale_log2, float lse2) { return __builtin_amdgcn_exp2f(__builtin_fmaf(s, scale_log2, -lse2)); }

// lse to base 2 for the exponentials; a row without keys gets +inf, which makes all its weights 0.
__device__ __forceinline__ float att_lse2(float lse) { return lse == -__builtin_inff() ? __builtin_inff() : lse * ATT_LOG2_E; }

template <typename T, int DP, bool ALIGNED>
__global__ __launch_bounds__(256, (AttGradShape<T, DP>::WAVES_PER_SIMD)) void attention_grad_queries(const AttentionGradArgs args)
{
    typedef AttGradShape<T, DP> Shape;
    constexpr int KT = Shape::KEYS;
    __shared__ __attribute__((aligned(16))) T lds[KT * (Shape::BOTH + ATT_STRIDE<T, DP>)];
    T *key_tile = lds, *value_tile = key_tile + KT * ATT_STRIDE<T, DP>, *key_tile_t = value_tile + KT * ATT_STRIDE<T, DP>;
    const int lane = threadIdx.x & 63, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int id = (blockIdx.x & 7) * (args.q_grid >> 3) + (blockIdx.x >> 3);
    if (id >= args.q_workgroups) return;
    const int row_tile = id % args.q_row_tiles;
    id /= args.q_row_tiles;
    const int split = id % args.q_splits;
    id /= args.q_splits;
    const int g = id % args.g, entry = id / args.g;

    const int rows = args.m * args.r;
    const int first_row = row_tile * 128 + 32 * wave, row = first_row + lane % 32;
    const bool works = first_row < rows;
    const int token = (row < rows ? row : 0) / args.r, head = g * args.r + (row < rows ? row : 0) % args.r;
    const i64 at = (static_cast<i64>(entry) * args.m + token) * (static_cast<i64>(args.g) * args.r) + head;
    const T *q = static_cast<const T *>(args.q) + entry * args.q_ls + token * args.q_ms + head * args.q_hs;
    const T *d = static_cast<const T *>(args.grad_out) + entry * args.grad_out_ls + token * args.grad_out_ms + head * args.grad_out_hs;
    const T *out = static_cast<const T *>(args.out) + entry * args.out_ls + token * args.out_ms + head * args.out_hs;

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
    delta += att_other_half(delta);
    float lse2 = att_lse2(args.lse[at]);

    att_f32x16 acc[DP / 32];
#pragma unroll
    for (int o = 0; o < DP / 32; ++o) acc[o] = att_f32x16{0};

    const AttentionKeys &keys = args.keys;
    const int length = att_length(keys, entry);
    int begin, end;
    att_range(length, KT, split, args.q_splits, &begin, &end);
    const bool one_tile = length <= KT;
    const i64 rows_total = static_cast<i64>(args.l) * args.m * args.g * args.r;
    const T *k = static_cast<const T *>(keys.k) + entry * keys.k_ls + g * keys.k_gs;
    const T *v = static_cast<const T *>(keys.v) + entry * keys.v_ls + g * keys.v_gs;
    AttTile<T, DP, KT, 256, ALIGNED> next_k, next_v;
    if (one_tile && begin < end) {
        // Few keys: delta from the rounded result would be off by as much as ds is large, so it is summed from the weights themselves,
        // which are normalised again while they are at hand (a single key's weight is exactly 1, its ds exactly 0).
        const att_u64 kept = att_kept_keys(keys, entry, begin, end, lane);
        next_k.load(k, keys.k_ns, end, args.k, threadIdx.x);
        next_v.load(v, keys.v_ns, end, args.o, threadIdx.x);
        if (keys.mask) {
            next_k.clear(threadIdx.x, kept);
            next_v.clear(threadIdx.x, kept);
        }
        next_k.template store<ATT_STRIDE<T, DP>>(key_tile, threadIdx.x);
        next_v.template store<ATT_STRIDE<T, DP>>(value_tile, threadIdx.x);
        __syncthreads();
        float total = 0.0f, inner = 0.0f;
#pragma unroll 1
        for (int b = 0; b < KT / 32; ++b) {
            att_f32x16 s = {0}, ds = {0};
#pragma unroll
            for (int step = 0; step < DP / 16; ++step) {
                s = att_mma(att_read_row<T, DP>(key_tile, ATT_STRIDE<T, DP>, 32 * b + lane % 32, 16 * step + 8 * half), query[step], s);
                ds = att_mma(att_read_row<T, DP>(value_tile, ATT_STRIDE<T, DP>, 32 * b + lane % 32, 16 * step + 8 * half), grad[step], ds);
            }
            const unsigned mine = static_cast<unsigned>(kept >> (32 * b)) >> (4 * half);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const bool counts = mine >> att_row(i, 0) & 1;
                const float p = !counts ? 0.0f : length == 1 ? 1.0f : att_weight(s[i], args.scale_log2, lse2);
                total += p;
                inner = __builtin_fmaf(p, ds[i], inner);
            }
        }
        total += att_other_half(total);
        inner += att_other_half(inner);
        if (total > 0.0f) {
            delta = inner / total;
            if (length > 1) lse2 += __builtin_amdgcn_logf(total);
        }
    }
    if (split == 0 && row < rows && half == 0) {
        args.stats[at] = lse2;
        args.stats[rows_total + at] = delta;
    }
    if (begin < end) {
        next_k.load(k + begin * keys.k_ns, keys.k_ns, end - begin, args.k, threadIdx.x);
        next_v.load(v + begin * keys.v_ns, keys.v_ns, end - begin, args.o, threadIdx.x);
    }
    for (int n = begin; n < end; n += KT) {
        const att_u64 kept = att_kept_keys(keys, entry, n, end, lane);
        __syncthreads();
        if (keys.mask) {
            next_k.clear(threadIdx.x, kept);
            next_v.clear(threadIdx.x, kept);
        }
        next_k.template store<ATT_STRIDE<T, DP>>(key_tile, threadIdx.x);
        next_k.template store<ATT_STRIDE_T<T, DP>>(key_tile_t, threadIdx.x);
        next_v.template store<ATT_STRIDE<T, DP>>(value_tile, threadIdx.x);
        __syncthreads();
        if (n + KT < end) {
            const i64 next = n + KT;
            next_k.load(k + next * keys.k_ns, keys.k_ns, end - static_cast<int>(next), args.k, threadIdx.x);
            next_v.load(v + next * keys.v_ns, keys.v_ns, end - static_cast<int>(next), args.o, threadIdx.x);
        }
        if (!works) continue;
#pragma unroll
        for (int b = 0; b < KT / 32; ++b) {
            att_f32x16 s = {0}, ds = {0};
#pragma unroll
            for (int step = 0; step < DP / 16; ++step)
                s = att_mma(att_read_row<T, DP>(key_tile, ATT_STRIDE<T, DP>, 32 * b + lane % 32, 16 * step + 8 * half), query[step], s);
#pragma unroll
            for (int step = 0; step < DP / 16; ++step)
                ds = att_mma(att_read_row<T, DP>(value_tile, ATT_STRIDE<T, DP>, 32 * b + lane % 32, 16 * step + 8 * half), grad[step], ds);
            const unsigned here = static_cast<unsigned>(kept >> (32 * b));
#pragma unroll
            for (int i = 0; i < 16; ++i) ds[i] = att_weight(s[i], args.scale_log2, lse2) * (ds[i] - delta);
            if (here != ~0u) {
                att_rare();
                const unsigned mine = here >> (4 * half);
#pragma unroll
                for (int i = 0; i < 16; ++i) ds[i] = mine >> att_row(i, 0) & 1 ? ds[i] : 0.0f;
            }
#pragma unroll
            for (int step = 0; step < 2; ++step) {
                const att_vec8<T> x = att_operand<T>(ds, step);
#pragma unroll
                for (int o = 0; o < DP / 32; ++o)
                    acc[o] = att_mma(att_read_transposed(key_tile_t, ATT_STRIDE_T<T, DP>, 32 * b + 16 * step, 32 * o, lane), x, acc[o]);
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

// A workgroup per (entry of the keys, head of keys, part of the rows, 128 keys); a wave per 32 keys.
template <typename T, int DP, bool ALIGNED>
__global__ __launch_bounds__(256, (AttGradShape<T, DP>::WAVES_PER_SIMD_K)) void attention_grad_keys(const AttentionGradArgs args)
{
    typedef AttGradShape<T, DP> Shape;
    constexpr int RT = Shape::ROWS;
    __shared__ __attribute__((aligned(16))) T lds[2 * RT * Shape::BOTH];
    __shared__ __attribute__((aligned(16))) float stats[2 * RT];
    T *q_tile = lds, *d_tile = q_tile + RT * ATT_STRIDE<T, DP>;
    T *q_tile_t = d_tile + RT * ATT_STRIDE<T, DP>, *d_tile_t = q_tile_t + RT * ATT_STRIDE_T<T, DP>;
    const int lane = threadIdx.x & 63, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int id = (blockIdx.x & 7) * (args.k_grid >> 3) + (blockIdx.x >> 3);
    if (id >= args.k_workgroups) return;
    const int key_tile = id % args.key_tiles;
    id /= args.key_tiles;
    const int split = id % args.k_splits;
    id /= args.k_splits;
    const int g = id % args.g, key_entry = id / args.g;

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
        value[step] = att_load8<T, ALIGNED>(v, 16 * step + 8 * half, args.o);
    }
    att_f32x16 acc_k[DP / 32], acc_v[DP / 32];
#pragma unroll
    for (int o = 0; o < DP / 32; ++o) acc_k[o] = acc_v[o] = att_f32x16{0};

    // the rows: entries that share the keys, their heads, 32 queries at a time; this part of them
    const int tiles_m = (args.m + RT - 1) / RT;
    const i64 per_entry = static_cast<i64>(args.r) * tiles_m;
    const i64 items = per_entry * (args.key_entries == args.l ? 1 : args.l);
    const i64 per_split = (items + args.k_splits - 1) / args.k_splits;
    i64 item = split * per_split;
    const i64 last = item + per_split < items ? item + per_split : items;
    int entry = key_entry + static_cast<int>(item / per_entry);
    int head = static_cast<int>(item % per_entry / tiles_m), m0 = static_cast<int>(item % tiles_m) * RT;

    bool kept = false, all_kept = false;            // this lane's key takes part in the current entry; all of this wave's do
    bool fresh = true;
    // Goes on to the next tile whose entry meets one of the workgroup's keys; the same decisions in all waves.
    auto find = [&]() {
        while (item < last) {
            if (fresh) {
                const int length = att_length(keys, entry);
                const att_u64 low = att_kept_keys(keys, entry, first_key, length, lane), high = att_kept_keys(keys, entry, first_key + 64, length, lane);
                if (low | high) break;
                item += per_entry - (static_cast<i64>(head) * tiles_m + m0 / RT);
                ++entry;
                head = m0 = 0;
            } else {
                break;
            }
        }
    };
    auto keys_of_entry = [&](int of) {
        kept = exists && n < att_length(keys, of) && (!keys.mask || keys.mask[of * keys.mask_ls + n * keys.mask_ns] != 0);
        all_kept = __all(kept);
    };
    const i64 rows_total = static_cast<i64>(args.l) * args.m * args.g * args.r;
    AttTile<T, DP, RT, 256, ALIGNED> next_q, next_d;
    float next_stat = 0.0f;
    auto load = [&]() {
        const int some = args.m - m0;
        const int h = g * args.r + head;
        next_q.load(static_cast<const T *>(args.q) + entry * args.q_ls + m0 * args.q_ms + h * args.q_hs, args.q_ms, some, args.k, threadIdx.x);
        next_d.load(static_cast<const T *>(args.grad_out) + entry * args.grad_out_ls + m0 * args.grad_out_ms + h * args.grad_out_hs, args.grad_out_ms,
                    some, args.o, threadIdx.x);
        const int i = threadIdx.x % RT;
        const i64 at = (static_cast<i64>(entry) * args.m + m0 + i) * (static_cast<i64>(args.g) * args.r) + h;
        if (threadIdx.x < RT) next_stat = i < some ? args.stats[at] : __builtin_inff();
        else if (threadIdx.x < 2 * RT) next_stat = i < some ? args.stats[rows_total + at] : 0.0f;
    };
    find();
    int kept_entry = -1;
    if (item < last) load();
    while (item < last) {
        if (entry != kept_entry) {
            keys_of_entry(entry);
            kept_entry = entry;
        }
        __syncthreads();
        next_q.template store<ATT_STRIDE<T, DP>>(q_tile, threadIdx.x);
        next_q.template store<ATT_STRIDE_T<T, DP>>(q_tile_t, threadIdx.x);
        next_d.template store<ATT_STRIDE<T, DP>>(d_tile, threadIdx.x);
        next_d.template store<ATT_STRIDE_T<T, DP>>(d_tile_t, threadIdx.x);
        if (threadIdx.x < 2 * RT) stats[threadIdx.x] = next_stat;
        __syncthreads();
        ++item;
        fresh = false;
        m0 += RT;
        if (m0 >= args.m) {
            m0 = 0;
            if (++head == args.r) {
                head = 0;
                ++entry;
                fresh = true;
            }
        }
        find();
        if (item < last) load();

        att_f32x16 s = {0}, ds = {0};
#pragma unroll
        for (int step = 0; step < DP / 16; ++step)
            s = att_mma(att_read_row<T, DP>(q_tile, ATT_STRIDE<T, DP>, lane % 32, 16 * step + 8 * half), key[step], s);
#pragma unroll
        for (int step = 0; step < DP / 16; ++step)
            ds = att_mma(att_read_row<T, DP>(d_tile, ATT_STRIDE<T, DP>, lane % 32, 16 * step + 8 * half), value[step], ds);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const att_f32x4 lse2 = *reinterpret_cast<const att_f32x4 *>(stats + 8 * q + 4 * half);
            const att_f32x4 delta = *reinterpret_cast<const att_f32x4 *>(stats + RT + 8 * q + 4 * half);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                s[4 * q + j] = att_weight(s[4 * q + j], args.scale_log2, lse2[j]);
                ds[4 * q + j] = s[4 * q + j] * (ds[4 * q + j] - delta[j]);
            }
        }
        if (!all_kept) {
            att_rare();
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[i] = kept ? s[i] : 0.0f;
                ds[i] = kept ? ds[i] : 0.0f;
            }
        }
#pragma unroll
        for (int step = 0; step < 2; ++step) {
            const att_vec8<T> p = att_operand<T>(s, step);
#pragma unroll
            for (int o = 0; o < DP / 32; ++o) acc_v[o] = att_mma(att_read_transposed(d_tile_t, ATT_STRIDE_T<T, DP>, 16 * step, 32 * o, lane), p, acc_v[o]);
        }
#pragma unroll
        for (int step = 0; step < 2; ++step) {
            const att_vec8<T> x = att_operand<T>(ds, step);
#pragma unroll
            for (int o = 0; o < DP / 32; ++o) acc_k[o] = att_mma(att_read_transposed(q_tile_t, ATT_STRIDE_T<T, DP>, 16 * step, 32 * o, lane), x, acc_k[o]);
        }
    }
    if (!exists) return;
    const i64 at = (static_cast<i64>(key_entry) * keys.n + n) * args.g + g;
    if (args.k_splits > 1) {
        const i64 slot = split * (static_cast<i64>(args.key_entries) * keys.n * args.g) + at;
        float *to_k = args.partial_k + slot * args.partial_k_width, *to_v = args.partial_v + slot * args.partial_o_width;
#pragma unroll
        for (int o = 0; o < DP / 32; ++o)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int column = 32 * o + att_row(i, half);
                if (column < args.k) to_k[column] = acc_k[o][i];
                if (column < args.o) to_v[column] = acc_v[o][i];
            }
        return;
    }
    att_store_columns<T, DP, ALIGNED>(static_cast<T *>(args.grad_k) + at * args.k, acc_k, args.scale, args.k, half);
    att_store_columns<T, DP, ALIGNED>(static_cast<T *>(args.grad_v) + at * args.o, acc_v, 1.0f, args.o, half);
}

// The parts of a cut gradient, added in their order.
template <typename T>
__global__ __launch_bounds__(256) void attention_sum(const AttentionSumArgs args)
{
    const i64 count = args.rows * args.width, step = static_cast<i64>(gridDim.x) * 256;
    for (i64 i = static_cast<i64>(blockIdx.x) * 256 + threadIdx.x; i < count; i += step) {
        const float *from = args.partial + i / args.width * args.partial_width + i % args.width;
        float sum = 0.0f;
        for (int part = 0; part < args.splits; ++part) sum += from[part * args.rows * args.partial_width];
        static_cast<T *>(args.out)[i] = static_cast<T>(sum * args.factor);
    }
}

}  // namespace kmc
