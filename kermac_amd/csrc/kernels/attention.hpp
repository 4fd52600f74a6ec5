// Attention: a kernel matrix exp(scale <q, k>) whose rows are divided by their sums, times values.
//
//   s[m, n] = scale sum_k q[m, k] k[n, k],   lse[m] = log sum_n exp s[m, n],   out[m, o] = sum_n exp(s[m, n] - lse[m]) v[n, o]
//
// over the keys n that take part.  One pass over keys and values: a running maximum and a running sum per query, the
// output rescaled when the maximum has grown (both in fp32; exponentials to base 2 with log2(e) folded into the scale).
//
// Queries of the heads that share a head of keys are the rows of one problem: row r is query r / R of head r % R
// (R heads per head of keys), so keys and values are read once for all of them.  Queries of all batch entries
// against one common set of keys are one problem in the same way.
//
// The products run on the 32 x 32 matrix instruction with the scores transposed, s^T[n, row] = K Q^T: a lane then owns one
// row of the softmax (two lanes, for alternating groups of four keys), its statistics are one register each, and the
// registers that hold s^T are, in the order in which they stand, the operand of out^T[o, row] = V^T P^T if the
// contraction takes the keys of a step as 4 h + {0..3}, 8 + 4 h + {0..3} for half wave h.  V^T comes from row-major tiles in
// LDS by the transposing read (16-bit types) or by 32-bit reads (fp32).  P is rounded to the type of the values, half a step per
// weight, which leaves about as large an error in the result as its own rounding does (bf16, 8 x 4096 x 8192: 2.3e-3 in all, 1.7e-3 where weights stay in 32 bits); fp32 keeps every bit.
#pragma once

#include <hip/hip_runtime.h>

#include <type_traits>

#include "attention_args.hpp"

namespace kmc {

typedef float att_f32x16 __attribute__((ext_vector_type(16)));
typedef float att_f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned att_u32x4 __attribute__((ext_vector_type(4)));
typedef short att_s16x4 __attribute__((ext_vector_type(4)));
typedef unsigned long long att_u64;

template <typename T> struct AttVector { typedef T type __attribute__((ext_vector_type(8))); };
template <typename T> using att_vec8 = typename AttVector<T>::type;

constexpr float ATT_LOG2_E = 1.4426950408889634f;
constexpr float ATT_LN_2 = 0.6931471805599453f;

// c += a b over 16 k: lane l holds row (of a) or column (of b) l % 32 and 8 of the k, those of half wave l / 32.
__device__ __forceinline__ att_f32x16 att_mma(att_vec8<__bf16> a, att_vec8<__bf16> b, att_f32x16 c)
{
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ att_f32x16 att_mma(att_vec8<_Float16> a, att_vec8<_Float16> b, att_f32x16 c)
{
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ att_f32x16 att_mma(att_vec8<float> a, att_vec8<float> b, att_f32x16 c)
{
#pragma unroll
    for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
    return c;
}

// Register i of a 32 x 32 result holds row att_row(i, half wave) of column lane % 32.
__device__ __forceinline__ constexpr int att_row(int i, int half) { return 8 * (i / 4) + 4 * half + i % 4; }

// Whether bit att_row(i, half) of `rows`, the same in all lanes, is set: a mask in scalar registers, so that a selection is one vector instruction.
__device__ __forceinline__ bool att_has_row(unsigned rows, int i)
{
    const int low = static_cast<int>(rows << (31 - att_row(i, 0))) >> 31, high = static_cast<int>(rows << (31 - att_row(i, 1))) >> 31;
    return __builtin_amdgcn_inverse_ballot_w64(static_cast<att_u64>(static_cast<unsigned>(high)) << 32 | static_cast<unsigned>(low));
}

// The sum and the maximum of a value over the two lanes of a column.
__device__ __forceinline__ float att_sum_of_halves(float x)
{
    const auto both = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x), false, false);
    return __builtin_bit_cast(float, static_cast<unsigned>(both[0])) + __builtin_bit_cast(float, static_cast<unsigned>(both[1]));
}
__device__ __forceinline__ float att_max_of_halves(float x)
{
    const auto both = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x), false, false);
    return fmaxf(__builtin_bit_cast(float, static_cast<unsigned>(both[0])), __builtin_bit_cast(float, static_cast<unsigned>(both[1])));
}

// A tile of rows of DP elements in LDS, read both ways: 16 bytes of a row per lane, 16 rows at a time, and transposed, which touches 4 rows x 64 bytes per
// half wave.  Row r holds its 16-byte piece c in place c ^ swizzle(r) / 16: sixteen consecutive rows then have a given piece in different banks, and four
// rows a given four pieces (no bank conflict is counted).  Rows take a power of two of bytes: those of 96 elements the place of 128.
template <typename T, int DP>
struct AttLds {
    static constexpr int PIECE = 16 / static_cast<int>(sizeof(T));      // elements of 16 bytes
    static constexpr int STRIDE = (DP == 96 ? 128 : DP) * static_cast<int>(sizeof(T));
    // The bits that the swizzle of row r turns in a byte offset; linear in the bits of r.  Two rows of 128 bytes share a line of banks.
    static __device__ __forceinline__ constexpr int swizzle(int r)
    {
        return STRIDE == 128 ? ((r >> 1 & 1) << 2 | (r >> 2 & 3)) << 4 : ((r & 3) << 2 | (r >> 2 & 3)) << 4;
    }
    static __device__ __forceinline__ constexpr int offset(int row, int piece) { return row * STRIDE + (16 * piece ^ swizzle(row)); }
};

typedef unsigned char att_lds_byte;

// Eight elements of row `row` + lane % 32 from element k + 8 (lane / 32) on; row and k multiples of 32 and 16.
template <typename T, int DP>
__device__ __forceinline__ att_vec8<T> att_read_row(const att_lds_byte *tile, int row, int k, int lane)
{
    typedef AttLds<T, DP> Lds;
    const int size = static_cast<int>(sizeof(T));
    const int mine = (lane & 31) * Lds::STRIDE + (8 * size * (lane >> 5) ^ Lds::swizzle(lane & 31));
    const int here = mine ^ k * size;
    const att_lds_byte *p = tile + row * Lds::STRIDE;
    att_vec8<T> x;
    if constexpr (sizeof(T) == 2) {
        x = *reinterpret_cast<const att_vec8<T> *>(p + here);
    } else {
        const att_f32x4 low = *reinterpret_cast<const att_f32x4 *>(p + here);
        const att_f32x4 high = *reinterpret_cast<const att_f32x4 *>(p + (here ^ 16));
#pragma unroll
        for (int j = 0; j < 4; ++j) { x[j] = low[j]; x[4 + j] = high[j]; }
    }
    return x;
}

// Lane l gets column `column` + l % 32 of the 16 rows from `row` on, in the order 4 h + {0..3}, 8 + 4 h + {0..3}; row and column multiples of 16 and 32.
template <typename T, int DP>
__device__ __forceinline__ att_vec8<T> att_read_transposed(const att_lds_byte *tile, int row, int column, int lane)
{
    typedef AttLds<T, DP> Lds;
    const int half = lane >> 5;
    att_vec8<T> x;
    if constexpr (sizeof(T) == 2) {
        const int r = 4 * half + (lane & 15) / 4;
        const int mine = r * Lds::STRIDE + (((32 * (lane >> 4 & 1) + 8 * (lane & 3)) ^ Lds::swizzle(r)));
        const att_lds_byte *p = tile + row * Lds::STRIDE + (mine ^ 2 * column);
        typedef __attribute__((address_space(3))) att_s16x4 lds_s16x4;
        union { att_s16x4 part[2]; att_vec8<T> whole; } u;
        u.part[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(p));
        const int behind = mine ^ 2 * column ^ Lds::swizzle(8);       // the same place of row r + 8
        u.part[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(tile + (row + 8) * Lds::STRIDE + behind));
        x = u.whole;
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int r = 4 * half + j;
            const int mine = r * Lds::STRIDE + (4 * (lane & 31) ^ Lds::swizzle(r));
            const int here = mine ^ 4 * column;
            x[j] = *reinterpret_cast<const float *>(tile + row * Lds::STRIDE + here);
            x[4 + j] = *reinterpret_cast<const float *>(tile + (row + 8) * Lds::STRIDE + (here ^ Lds::swizzle(8)));
        }
    }
    return x;
}

// Eight fp32 values of a result, registers 8 step .. 8 step + 7, rounded to the operand type.
template <typename T>
__device__ __forceinline__ att_vec8<T> att_operand(const att_f32x16 &x, int step)
{
    att_vec8<T> y;
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = static_cast<T>(x[8 * step + j]);
    return y;
}

// 16 bytes of a row of `width` elements from element `at` on; what lies behind the row reads as zero.
template <typename T, bool ALIGNED>
__device__ __forceinline__ att_u32x4 att_load16(const T *row, int at, int width)
{
    constexpr int COUNT = 16 / sizeof(T);
    att_u32x4 x = {0, 0, 0, 0};
    if constexpr (ALIGNED) {
        if (at < width) x = *reinterpret_cast<const att_u32x4 *>(row + at);       // width is a multiple of COUNT
    } else {
        union { T value[COUNT]; att_u32x4 whole; } u;
#pragma unroll
        for (int j = 0; j < COUNT; ++j) u.value[j] = at + j < width ? row[at + j] : static_cast<T>(0.0f);
        x = u.whole;
    }
    return x;
}

// Eight elements of a row, for an operand that is kept in registers.
template <typename T, bool ALIGNED>
__device__ __forceinline__ att_vec8<T> att_load8(const T *row, int at, int width)
{
    union { att_u32x4 part[sizeof(T) / 2]; att_vec8<T> whole; } u;
#pragma unroll
    for (unsigned j = 0; j < sizeof(T) / 2; ++j) u.part[j] = att_load16<T, ALIGNED>(row, at + j * (16 / static_cast<int>(sizeof(T))), width);
    return u.whole;
}

constexpr int ATT_BUFFER_FORMAT = 0x00020000;        // 32-bit data, as raw buffers of this architecture want it

// Keeps the compiler from merging a rare case into the common path as selections.
__device__ __forceinline__ void att_rare() { asm volatile(""); }

typedef int att_s32x4 __attribute__((ext_vector_type(4)));

// The rows of a tile in memory: rows 0 .. rows - 1 of base, `width` elements each, `stride` apart; what lies outside reads as zero without a branch
// per load.
template <typename T>
__device__ __forceinline__ att_s32x4 att_descriptor(att_u64 address, int step, int rows, int width)
{
    const int bytes = rows > 0 ? (rows - 1) * step + width * static_cast<int>(sizeof(T)) : 0;
    return att_s32x4{__builtin_amdgcn_readfirstlane(static_cast<int>(address)), __builtin_amdgcn_readfirstlane(static_cast<int>(address >> 32) & 0xffff),
                     __builtin_amdgcn_readfirstlane(bytes), ATT_BUFFER_FORMAT};
}

// An address that is the same in all lanes, in scalar registers.
template <typename T>
__device__ __forceinline__ att_u64 att_uniform(const T *p)
{
    const att_u64 address = reinterpret_cast<att_u64>(p);
    const unsigned low = __builtin_amdgcn_readfirstlane(static_cast<int>(address)), high = __builtin_amdgcn_readfirstlane(static_cast<int>(address >> 32));
    return static_cast<att_u64>(high) << 32 | low;
}

template <typename T>
__device__ __forceinline__ unsigned att_lds_address(const T *p)
{
    return static_cast<unsigned>(reinterpret_cast<size_t>((const __attribute__((address_space(3))) T *)p));
}

// 4 bytes per lane from memory straight into LDS: lane l's to the address `to` + 4 l.
__device__ __forceinline__ void att_load_words(const float *from, unsigned to)
{
    typedef const __attribute__((address_space(1))) float *global_float;
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off"
                 : : "v"((global_float)from), "s"(__builtin_amdgcn_readfirstlane(to)) : "memory", "m0");
}

// At most IN_FLIGHT loads are outstanding, and the compiler knows: it would otherwise wait, in front of the first use of a register that was loaded
// before a loop, for everything that is outstanding in every turn of the loop, the tiles on their way to LDS included (a third of the run time).
template <int IN_FLIGHT = 0>
__device__ __forceinline__ void att_wait_for_loads()
{
    static_assert(IN_FLIGHT < 64, "the counter has six bits");
    asm volatile("" : : : "memory");
    __builtin_amdgcn_s_waitcnt(0x0f70 | (IN_FLIGHT & 15) | (IN_FLIGHT >> 4) << 14);         // vmcnt, the other counters as they are
    asm volatile("" : : : "memory");
}

// No read of LDS is outstanding: what is asked for next may overwrite what was read, and a read whose register is not used yet may not have been made.
// (A barrier waits for that by itself.)
__device__ __forceinline__ void att_wait_for_reads()
{
    asm volatile("" : : : "memory");
    __builtin_amdgcn_s_waitcnt(0xc07f);         // lgkmcnt 0, the other counters as they are
    asm volatile("" : : : "memory");
}

// A tile of ROWS rows of DP elements on its way from memory to LDS.  begin() asks for it, finish() has it written.  DIRECT: from memory straight into LDS, 1 KB per
// wave and instruction, each lane fetching the piece that belongs where its 16 bytes end up; no register waits for it.  Otherwise (unaligned rows,
// tiles of one wave, whose next tile waits in registers while LDS holds the current one, unless a row of 1 KB asks too many) through registers.
template <typename T, int DP, int ROWS, int THREADS, bool ALIGNED>
struct AttTile {
    typedef AttLds<T, DP> Lds;
    static constexpr bool DIRECT = ALIGNED && (THREADS > 64 || Lds::STRIDE == 1024);
    static constexpr int SLOTS = Lds::STRIDE / 16;                      // threads of a row
    static constexpr int ROW_STEP = THREADS / SLOTS;
    static constexpr int PER_THREAD = ROWS / ROW_STEP;                  // loads of a thread
    static_assert(THREADS % SLOTS == 0 && ROWS % ROW_STEP == 0 && PER_THREAD > 0, "whole rows per step");
    static_assert(ROW_STEP <= 32, "has_row shifts 32 bits");
    att_u32x4 held[DIRECT ? 1 : PER_THREAD];

    static __device__ __forceinline__ bool has_row(att_u64 kept, int row, int j) { return static_cast<unsigned>(kept >> (j * ROW_STEP)) >> row & 1; }

    // DIRECT, from a tile's descriptor.  A load may read a scalar register that a vector instruction wrote only 5 wait states behind it, which the hardware does not wait for
    // and the compiler does not see to in front of assembly.  Five here cost up to 2 % (16 questions behind a prefix 198 -> 203 us), and scalar instructions or six other states
    // stand in between wherever the compiler puts a descriptor together: a test reads that from the built library.
    __device__ __forceinline__ void begin_at(att_s32x4 from, int step, int width, att_lds_byte *tile, int thread, att_u64 kept = ~0ull)
    {
        constexpr int SIZE = static_cast<int>(sizeof(T));
        const int row = thread / SLOTS;
        const unsigned to = att_lds_address(tile) + __builtin_amdgcn_readfirstlane(thread / 64) * (64 / SLOTS * Lds::STRIDE);
#pragma unroll
        for (int j = 0; j < PER_THREAD; ++j) {
            const int r = row + j * ROW_STEP, at = (16 * (thread % SLOTS) ^ Lds::swizzle(row) ^ Lds::swizzle(j * ROW_STEP)) / SIZE;
            const unsigned offset = at < width && has_row(kept, row, j) ? static_cast<unsigned>(r * step + at * SIZE) : 0x80000000u;
            const unsigned lds = __builtin_amdgcn_readfirstlane(to + j * ROW_STEP * Lds::STRIDE);
            asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" : : "v"(offset), "s"(from), "s"(lds) : "memory", "m0");
        }
    }

    // Rows whose bit in `kept` is not set become zeros: nothing is read of them.
    __device__ __forceinline__ void begin(const T *base, i64 stride, int rows, int width, att_lds_byte *tile, int thread, att_u64 kept = ~0ull)
    {
        constexpr int SIZE = static_cast<int>(sizeof(T));
        const int row = thread / SLOTS, step = static_cast<int>(stride) * SIZE;
        if constexpr (DIRECT) {
            begin_at(att_descriptor<T>(reinterpret_cast<att_u64>(base), step, rows < ROWS ? rows : ROWS, width), step, width, tile, thread, kept);
        } else if constexpr (ALIGNED) {
            const int some = rows < ROWS ? rows : ROWS, bytes = some > 0 ? (some - 1) * step + width * SIZE : 0;
            const __amdgpu_buffer_rsrc_t from = __builtin_amdgcn_make_buffer_rsrc(const_cast<T *>(base), 0, bytes, ATT_BUFFER_FORMAT);
            const int at = thread % SLOTS * Lds::PIECE;
            unsigned offset = at < width ? static_cast<unsigned>(row * step + at * SIZE) : 0x80000000u;
#pragma unroll
            for (int j = 0; j < PER_THREAD; ++j) {
                held[j] = __builtin_amdgcn_raw_buffer_load_b128(from, has_row(kept, row, j) ? offset : 0x80000000u, 0, 0);
                offset += ROW_STEP * step;
            }
        } else {
            const T *p = base + row * stride;
#pragma unroll
            for (int j = 0; j < PER_THREAD; ++j) {
                held[j] = att_u32x4{0, 0, 0, 0};
                if (row + j * ROW_STEP < rows && has_row(kept, row, j)) held[j] = att_load16<T, false>(p, thread % SLOTS * Lds::PIECE, width);
                p += ROW_STEP * stride;
            }
        }
    }

    // Followed by a barrier.  IN_FLIGHT: loads that were asked for later and may still be on their way.
    template <int IN_FLIGHT = 0>
    __device__ __forceinline__ void finish(att_lds_byte *tile, int thread) const
    {
        if constexpr (DIRECT) {
            att_wait_for_loads<IN_FLIGHT>();
        } else {
            const int row = thread / SLOTS, piece = thread % SLOTS;
#pragma unroll
            for (int j = 0; j < PER_THREAD; ++j) *reinterpret_cast<att_u32x4 *>(tile + Lds::offset(row + j * ROW_STEP, piece)) = held[j];
        }
    }
};

// The low `count` bits, count clamped to 0 .. 64.
__device__ __forceinline__ att_u64 att_low_bits(int count)
{
    return count >= 64 ? ~0ull : count <= 0 ? 0ull : (1ull << count) - 1;
}

// Not 0 if key n0 + lane exists and takes part.  Asked for a tile ahead: a wait for it in front of every tile takes as long as the tile's products do.
__device__ __forceinline__ int att_ask_kept(const AttentionKeys &keys, int entry, int n0, int end, int lane)
{
    const int n = n0 + lane;
    int kept = n < end;
    if (kept && keys.mask) kept = keys.mask[entry * keys.mask_ls + n * keys.mask_ns];
    return kept;
}

// One bit per key n0 .. n0 + 63: the key exists and takes part.  The same in all waves of a workgroup.
__device__ __forceinline__ att_u64 att_kept_keys(const AttentionKeys &keys, int entry, int n0, int end, int lane)
{
    return __ballot(att_ask_kept(keys, entry, n0, end, lane) != 0);
}

__device__ __forceinline__ int att_length(const AttentionKeys &keys, int entry)
{
    if (!keys.lengths) return keys.n;
    const int length = keys.lengths[entry];
    return length < 0 ? 0 : length < keys.n ? length : keys.n;
}

// Writes of a wave to LDS are seen by its other lanes: LDS serves a wave in order, the compiler has to keep that order.
__device__ __forceinline__ void att_wave_sync()
{
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// What a wave carries along the keys for its 32 rows.  The weight of a score s (a product, not scaled yet) is exp2((s - shift) scale_log2 - base): 2^LIFT for the
// score that the row's weights are relative to, one of the largest so far.
template <int DP>
struct AttState {
    att_f32x16 out[DP / 32];
    float shift, base, sum;      // shift is -inf before the first key; sum of this lane's weights
    bool shifted;                // a row of the wave has a shift
};

// Weights in fp16 are 2^7 times what they are in the other types.  With ATT_HEADROOM they reach 2^15 of the type's 2^16, and at the other end a weight keeps bits down to
// 2^-31 of the largest: behind one key that stands out by 18 (to base e), the others' weights of 2^-26 would be 0, whatever their number.  Sum and output keep
// the factor, which the division takes out.
template <typename T> constexpr float ATT_LIFT = std::is_same<T, _Float16>::value ? 7.0f : 0.0f;

// What weights relative to the score `top` take.  In 16 bits, base = top scale_log2 rounded to fp32 and no shift, one instruction less per weight: the weight of `top` is
// then 2^LIFT times exp2 of that rounding's error, at most 2^-12 up to a base of 2^12, which the rounding to the operands' type takes away.  Where the base is larger (that error
// grows to any size: at 2^30 a weight would be 2^32, or 0 in every type) and in fp32, top is subtracted first, and its weight is exactly 2^LIFT.
constexpr float ATT_LARGEST_BASE = 4096.0f;

template <typename T>
__device__ __forceinline__ void att_relative_to(float top, float scale_log2, float *shift, float *base)
{
    const float product = top * scale_log2;
    const bool shifted = sizeof(T) == 4 || !(fabsf(product) < ATT_LARGEST_BASE);
    *shift = shifted ? top : 0.0f;
    *base = shifted ? -ATT_LIFT<T> : __builtin_fmaf(top, scale_log2, -ATT_LIFT<T>);
}

// The log of a row's sum of exponentials from that relative to the shift, to base 2.  -inf stands for a row without keys and for no other.
__device__ __forceinline__ float att_natural_lse(float shift, float lse2, float scale_log2)
{
    if (lse2 == -__builtin_inff()) return lse2;
    const float lse = __builtin_fmaf(lse2, ATT_LN_2, shift * (scale_log2 * ATT_LN_2));
    return lse == -__builtin_inff() ? -__FLT_MAX__ : lse;
}

// Outputs and sums are rescaled only when a score passes the one they are relative to by 2^8: weights stay below 2^(8 + LIFT), inside every type,
// and after the first tiles the 64 or more multiplications per tile are not made.
constexpr float ATT_HEADROOM = 8.0f;

// Fragments are read from LDS a group ahead of the matrix instructions that use them.  The compiler, left alone, reads each one in front of its
// use and waits for it; these fix the order within a region: READS reads, then the matrix instructions, each followed by VALU vector instructions.
// Only in kernels that have registers for all their values: around spilled ones a fixed order makes more of them (355 registers instead of 291 in the gradient of the
// queries in fp32 of 256 features; unaligned rows of 128 features in 16 bits, gradients of 2 x 1000 x 2000 x 8 heads: 354 us instead of 325).  The build refuses an
// ORDERED kernel that spills.
template <typename T, int DP, bool ALIGNED> constexpr bool ATT_ORDERED = ALIGNED && DP <= 128;

template <bool ORDERED, int READS, int MMAS, int VALU>
__device__ __forceinline__ void att_order()
{
    if constexpr (ORDERED) {
        __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
#pragma unroll
        for (int i = 0; i < MMAS; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            if (VALU > 0) __builtin_amdgcn_sched_group_barrier(0x002, VALU, 0);
        }
    }
}
template <bool ORDERED>
__device__ __forceinline__ void att_region()
{
    if constexpr (ORDERED) __builtin_amdgcn_sched_barrier(0);
}

template <typename T, int DP>
struct AttGroups {
    static constexpr int STEPS = DP / 16;                               // of a contraction over features
    static constexpr int GROUP = STEPS % 4 == 0 ? 4 : 3;                // fragments of a group
    static constexpr int GROUPS = STEPS / GROUP;
    static constexpr int MMAS = sizeof(T) == 4 ? 8 : 1;                 // matrix instructions per fragment
    static constexpr int READS_ROW = sizeof(T) == 4 ? 2 : 1;
    static constexpr int READS_T = sizeof(T) == 4 ? 8 : 2;
    static constexpr int COLUMNS = DP / 32 <= 4 ? DP / 32 : sizeof(T) == 4 ? 2 : 4;     // fragments of a group of transposed ones
    static constexpr int COLUMN_GROUPS = DP / 32 / COLUMNS;             // for all columns of 16 rows
};

template <typename T, int DP, int GROUP>
__device__ __forceinline__ void att_read_group(att_vec8<T> (&f)[GROUP], const att_lds_byte *tile, int row, int group, int lane)
{
#pragma unroll
    for (int i = 0; i < GROUP; ++i) f[i] = att_read_row<T, DP>(tile, row, 16 * (GROUP * group + i), lane);
}

// Group `group` of the columns of 16 rows, transposed.
template <typename T, int DP, int COLUMNS>
__device__ __forceinline__ void att_read_columns(att_vec8<T> (&f)[COLUMNS], const att_lds_byte *tile, int row, int group, int lane)
{
#pragma unroll
    for (int o = 0; o < COLUMNS; ++o) f[o] = att_read_transposed<T, DP>(tile, row, 32 * (COLUMNS * group + o), lane);
}

// s^T of a tile of KT keys in LDS and the 32 rows whose queries are in `query`, and the largest of each lane's scores.  One block of 32 keys after the
// other; the maximum over a block is taken beside the matrix instructions of the next.
template <typename T, int DP, int KT, bool ORDERED>
__device__ __forceinline__ float att_scores(att_f32x16 (&s)[KT / 32], const att_vec8<T> (&query)[DP / 16], const att_lds_byte *keys, int lane)
{
    typedef AttGroups<T, DP> G;
    constexpr int ALL = KT / 32 * G::GROUPS, EACH = 16 / G::GROUPS;
    att_vec8<T> f[2][G::GROUP];
    att_read_group<T, DP>(f[0], keys, 0, 0, lane);
#pragma unroll
    for (int b = 0; b < KT / 32; ++b) s[b] = att_f32x16{0};
    float top = -__builtin_inff();
    att_region<ORDERED>();
#pragma unroll
    for (int i = 0; i < ALL; ++i) {
        const int b = i / G::GROUPS, group = i % G::GROUPS;
        if (i + 1 < ALL) att_read_group<T, DP>(f[(i + 1) & 1], keys, 32 * ((i + 1) / G::GROUPS), (i + 1) % G::GROUPS, lane);
#pragma unroll
        for (int j = 0; j < G::GROUP; ++j) s[b] = att_mma(f[i & 1][j], query[G::GROUP * group + j], s[b]);
        if (b > 0)
#pragma unroll
            for (int j = EACH * group; j < (group + 1 == G::GROUPS ? 16 : EACH * (group + 1)); ++j) top = fmaxf(top, s[b - 1][j]);
        att_order<ORDERED, G::GROUP * G::READS_ROW, G::GROUP * G::MMAS, 0>();
        att_region<ORDERED>();
    }
#pragma unroll
    for (int j = 0; j < 16; ++j) top = fmaxf(top, s[KT / 32 - 1][j]);
    return top;
}

// Masks a tile's scores (`kept` has a bit per key, the same in all lanes; with `causal`, this lane's row meets the first `limit` of them only) and, where
// the weight of one would pass 2^(8 + LIFT), makes the weights relative to the largest, whose own is then 2^LIFT in the operands' type (a row of one key gets its value
// without a rounding).  What was made before is rescaled: output and sum, and `weights` that wait for their product and are rounded once more.  Shifts are
// subtracted from the scores.
template <typename T, int DP, int KT>
__device__ __forceinline__ void att_rebase(AttState<DP> &state, att_vec8<T> (&weights)[KT / 16], att_f32x16 (&s)[KT / 32], float top, float scale_log2, att_u64 kept,
                                           bool causal, int limit, int lane)
{
    const att_u64 all = KT == 64 ? ~0ull : (1ull << KT) - 1;
    if ((kept & all) != all) {
        att_rare();
        top = -__builtin_inff();
#pragma unroll
        for (int b = 0; b < KT / 32; ++b) {
            const unsigned rows = __builtin_amdgcn_readfirstlane(static_cast<unsigned>(kept >> (32 * b)));
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[b][i] = att_has_row(rows, i) ? s[b][i] : -__builtin_inff();
                top = fmaxf(top, s[b][i]);
            }
        }
    }
    if (causal && !__all(limit >= KT)) {
        att_rare();
        top = -__builtin_inff();
#pragma unroll
        for (int b = 0; b < KT / 32; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[b][i] = 32 * b + att_row(i, 0) < limit - 4 * (lane >> 5) ? s[b][i] : -__builtin_inff();
                top = fmaxf(top, s[b][i]);
            }
    }
    top = att_max_of_halves(top);
    const float above = __builtin_fmaf(top - state.shift, scale_log2, -state.base);     // the largest weight, to base 2; not a number without keys
    if (__any(above > ATT_HEADROOM + ATT_LIFT<T>)) {
        att_rare();
        float shift, base, shrink = 1.0f;
        att_relative_to<T>(top, scale_log2, &shift, &base);
        if (above > ATT_LIFT<T>) {
            shrink = __builtin_amdgcn_exp2f(__builtin_fmaf(state.shift - shift, scale_log2, state.base - base));
            state.shift = shift;
            state.base = base;
        }
        state.shifted = __any(state.shift != 0.0f && state.shift != -__builtin_inff());
        state.sum *= shrink;
#pragma unroll
        for (int o = 0; o < DP / 32; ++o) state.out[o] *= shrink;
#pragma unroll
        for (int step = 0; step < KT / 16; ++step)
#pragma unroll
            for (int j = 0; j < 8; ++j) weights[step][j] = static_cast<T>(static_cast<float>(weights[step][j]) * shrink);
    }
    if (sizeof(T) == 4 || state.shifted) {
        if (sizeof(T) != 4) att_rare();
        const float shift = state.shift == -__builtin_inff() ? 0.0f : state.shift;
#pragma unroll
        for (int b = 0; b < KT / 32; ++b) s[b] -= shift;
    }
}

// The weights of 16 keys, in the operands' type.
template <typename T, int DP, int KT>
__device__ __forceinline__ att_vec8<T> att_weights(AttState<DP> &state, const att_f32x16 (&s)[KT / 32], int step, float scale_log2, float base)
{
    float p[8], sum = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        p[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[step / 2][8 * (step % 2) + j], scale_log2, -base));
        sum += p[j];
    }
    state.sum += sum;
    att_vec8<T> weights;
#pragma unroll
    for (int j = 0; j < 8; ++j) weights[j] = static_cast<T>(p[j]);
    return weights;
}

// out^T += V^T p^T over the KT keys of a tile; with NEXT, the weights give way to those of the scores s.  `first`: the first group of V's columns.
template <typename T, int DP, int KT, bool NEXT, bool ORDERED>
__device__ __forceinline__ void att_add_values(AttState<DP> &state, att_vec8<T> (&weights)[KT / 16], const att_lds_byte *values,
                                               const att_vec8<T> (&first)[AttGroups<T, DP>::COLUMNS], const att_f32x16 (&s)[KT / 32], float scale_log2, float base,
                                               int lane)
{
    typedef AttGroups<T, DP> G;
    constexpr int ALL = KT / 16 * G::COLUMN_GROUPS;
    att_vec8<T> f[2][G::COLUMNS];
#pragma unroll
    for (int o = 0; o < G::COLUMNS; ++o) f[0][o] = first[o];
#pragma unroll
    for (int i = 0; i < ALL; ++i) {
        const int step = i / G::COLUMN_GROUPS, group = i % G::COLUMN_GROUPS;
        if (i + 1 < ALL) att_read_columns<T, DP>(f[(i + 1) & 1], values, 16 * ((i + 1) / G::COLUMN_GROUPS), (i + 1) % G::COLUMN_GROUPS, lane);
#pragma unroll
        for (int o = 0; o < G::COLUMNS; ++o) {
            att_f32x16 &out = state.out[G::COLUMNS * group + o];
            out = att_mma(f[i & 1][o], weights[step], out);
        }
        const bool last = group + 1 == G::COLUMN_GROUPS;
        if (NEXT && last) weights[step] = att_weights<T, DP, KT>(state, s, step, scale_log2, base);
        att_order<ORDERED, G::COLUMNS * G::READS_T, G::COLUMNS * G::MMAS, NEXT ? (G::MMAS > 1 ? 1 : DP <= 64 ? 14 : 7) : 0>();
        att_region<ORDERED>();
    }
}

// Keys [begin, end) of a segment for split `split` of `splits`, in whole tiles.
__device__ __forceinline__ void att_range(int length, int tile, int split, int splits, int *begin, int *end)
{
    const int tiles = (length + tile - 1) / tile;
    const i64 per_split = static_cast<i64>((tiles + splits - 1) / splits) * tile;
    const i64 first = split * per_split;
    *begin = first < length ? static_cast<int>(first) : length;
    *end = length - *begin < per_split ? length : static_cast<int>(*begin + per_split);
}

// Where row `row` of a problem's entry lives.
struct AttRow { int entry, query, head; };
__device__ __forceinline__ AttRow att_find_row(const AttentionArgs &args, int first_entry, int g, int row)
{
    const int token = row / args.r;
    AttRow at;
    at.head = g * args.r + row % args.r;
    at.entry = first_entry + token / args.m;
    at.query = token % args.m;
    return at;
}

// What a workgroup holds in LDS.
template <typename T, int DP>
struct AttForwardShape {
    static constexpr int WAVES = 4;
    static constexpr int ROW_BYTES = AttLds<T, DP>::STRIDE;
    // Waves that share the keys: a ring of two tiles of keys and one of two tiles of values.
    static constexpr int SHARED_KEYS = ROW_BYTES <= 512 ? 64 : 32;
    static constexpr int SHARED_BYTES = 4 * SHARED_KEYS * ROW_BYTES;
    // Waves with keys of their own.
    static constexpr int OWN_KEYS = 32;
    // Rows of 1 KB: two tiles for every wave do not fit LDS, and half of the waves would leave half of the matrix cores idle, which in fp32 take longer than
    // the memory.  Keys and values take turns in one tile then (1 token x 20000 keys x 8 heads of 256 fp32: 125 us, with two waves of two tiles 10 % more).
    static constexpr bool OWN_TURNS = ROW_BYTES > 512;
    static constexpr int OWN_BYTES = (OWN_TURNS ? 1 : 2) * WAVES * OWN_KEYS * ROW_BYTES;
    static constexpr int JOIN_BYTES = (WAVES - 1) * (DP * 32 + 64) * 4 + 256 * WAVES;
    static constexpr int BYTES_1 = SHARED_BYTES > OWN_BYTES ? SHARED_BYTES : OWN_BYTES;
    static constexpr int BYTES = BYTES_1 > JOIN_BYTES ? BYTES_1 : JOIN_BYTES;
    static constexpr int WAVES_PER_SIMD = ROW_BYTES <= 256 ? 2 : 1;
};

// A lane's column of results [DP, 32] as the row of `width` elements that it is in memory, times a factor.
template <typename T, int DP, bool ALIGNED>
__device__ __forceinline__ void att_store_columns(T *to, const att_f32x16 (&x)[DP / 32], float factor, int width, int half)
{
#pragma unroll
    for (int o = 0; o < DP / 32; ++o)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int column = 32 * o + 8 * q + 4 * half;
            typedef T four __attribute__((ext_vector_type(4)));
            four y;
#pragma unroll
            for (int j = 0; j < 4; ++j) y[j] = static_cast<T>(x[o][4 * q + j] * factor);
            if (ALIGNED) {
                if (column < width) *reinterpret_cast<four *>(to + column) = y;
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (column + j < width) to[column + j] = y[j];
            }
        }
}

// Writes a wave's 32 rows: the result itself, or for attention_join a partial result, its shift and its lse beside the shift (to base 2).
template <typename T, int DP, bool ALIGNED>
__device__ __forceinline__ void att_forward_write(const AttentionArgs &args, const AttentionJob &job, const AttState<DP> &state, float sum, int entry, int g,
                                                  int row, int split, int lane)
{
    if (row >= job.rows) return;
    const int half = lane >> 5;
    const AttRow at = att_find_row(args, entry, g, row);
    const i64 id = (static_cast<i64>(at.entry) * args.m + at.query) * (static_cast<i64>(args.g) * args.r) + at.head;
    const float inverse = sum > 0.0f ? 1.0f / sum : sum == 0.0f ? 0.0f : sum;      // a row without keys gets zeros, not a number stays
    const float lse2 = sum == 0.0f ? -__builtin_inff() : state.base + __builtin_amdgcn_logf(sum);
    if (job.partial) {
        const i64 slot = static_cast<i64>(job.slot + split) * args.rows_total + id;
        if (half == 0) {
            // (-inf says that the part has no keys; one whose scores are all not a number has no shift either, and stays one)
            args.partial_shift[slot] = sum == 0.0f ? -__builtin_inff() : state.shift == -__builtin_inff() ? 0.0f : state.shift;
            args.partial_lse[slot] = lse2;
        }
        if (sum == 0.0f) return;                                                    // nobody reads it
        float *to = args.partial_out + slot * args.partial_width;
#pragma unroll
        for (int o = 0; o < DP / 32; ++o)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int column = 32 * o + 8 * q + 4 * half;
                if (column < args.partial_width) {
                    const att_f32x4 x = {state.out[o][4 * q] * inverse, state.out[o][4 * q + 1] * inverse, state.out[o][4 * q + 2] * inverse,
                                         state.out[o][4 * q + 3] * inverse};
                    *reinterpret_cast<att_f32x4 *>(to + column) = x;
                }
            }
        return;
    }
    if (args.lse && half == 0) args.lse[id] = att_natural_lse(state.shift, lse2, args.scale_log2);
    att_store_columns<T, DP, ALIGNED>(static_cast<T *>(args.out) + at.entry * args.out_ls + at.query * args.out_ms + at.head * args.out_hs, state.out, inverse,
                                      args.o, half);
}

template <typename T, int DP, bool ALIGNED>
__device__ __forceinline__ void att_load_queries(const AttentionArgs &args, const AttentionJob &job, int entry, int g, int row, int lane, att_vec8<T> (&query)[DP / 16])
{
    const int half = lane >> 5;
    const AttRow at = att_find_row(args, entry, g, row < job.rows ? row : 0);
    const T *from = static_cast<const T *>(args.q) + at.entry * args.q_ls + at.query * args.q_ms + at.head * args.q_hs;
#pragma unroll
    for (int step = 0; step < DP / 16; ++step) {
        query[step] = att_load8<T, ALIGNED>(from, 16 * step + 8 * half, args.k);
        if (args.query_factor != 1.0f)                                              // -1 or 0: exact
#pragma unroll
            for (int j = 0; j < 8; ++j) query[step][j] = static_cast<T>(static_cast<float>(query[step][j]) * args.query_factor);
    }
}

// A workgroup per (batch entry, head of keys, range of keys, tile of rows).
//
// More than 32 rows: WAVES waves of 32 rows each share the tiles of keys and values.  With 128 features in 16 bits the matrix cores are busy 52 % of the time, under
// the power limit, vector instructions and reads of LDS take the rest of a wave's turn.
// 8 entries x 4096 queries x 8192 keys x 32 heads on 8 x 128 bf16: 4.1 ms, 1.1 PFLOP/s (a large
// bf16 matrix product of the library's reaches 1.24).  Measured and left out: 64 rows per wave (half the reads from LDS, one wave per SIMD: 7.0 ms), 8
// waves that share a tile (the same time), tiles of 32 keys in deeper rings (4.8 ms).  fp32: 72 useful TFLOP/s of 154 at
// 2 x 1000 x 2900 x 8 heads of 64, of which 80 % of the keys take part; the matrix cores are busy 64 % of the time.
//
// At most 32 rows (single tokens): reading keys and values is all the work, so every wave walks tiles of its own without waiting for the others,
// and the waves' results are joined at the end.  32 entries x 1 query x up to 4000 keys x 16 heads of 64 bf16: 90 us, 4.4 TB/s (a large copy
// reaches 4.8); 4 x 32768 keys x 16 heads of 128: 192 us, 5.6 TB/s.
template <typename T, int DP, bool ALIGNED, bool ORDERED = ATT_ORDERED<T, DP, ALIGNED>>
__global__ __launch_bounds__(256, (AttForwardShape<T, DP>::WAVES_PER_SIMD)) void attention_forward(const AttentionArgs args)
{
    typedef AttForwardShape<T, DP> Shape;
    constexpr int WAVES = Shape::WAVES, THREADS = 64 * WAVES;
    __shared__ __attribute__((aligned(1024))) att_lds_byte lds[Shape::BYTES];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

    // The prefix's workgroups come first: they are bound by the matrix cores and are about as many as fit the chip at most, so those of the sequences'
    // own keys, bound by memory, run beside and behind them (128 sequences behind 65536 tokens, before other steps: 233 us, with the two kinds alternating 276; now 210).
    // XCD x gets a contiguous part of a job's list, in which the tiles of rows of one set of keys stand together: they share its L2.
    int id = static_cast<int>(blockIdx.x) + args.first_block;
    const bool second = id >= args.job[0].grid;
    const AttentionJob &job = args.job[second];
    if (second) id -= args.job[0].grid;
    id = (id & 7) * (job.grid >> 3) + (id >> 3);
    if (id >= job.workgroups) return;
    const int row_tile = id % job.row_tiles;
    id /= job.row_tiles;
    int g, split, entry;
    if (job.own_keys) {             // the heads of the same tokens, which stand side by side in memory, at the same time
        g = id % args.g;
        id /= args.g;
        split = id % job.splits;
        id /= job.splits;
        entry = id;
    } else {                        // one head of all entries, whose lengths differ, on an XCD
        split = id % job.splits;
        id /= job.splits;
        entry = id % job.entries;
        g = id / job.entries;
    }

    AttState<DP> state;
    att_vec8<T> query[DP / 16];
#pragma unroll
    for (int o = 0; o < DP / 32; ++o) state.out[o] = att_f32x16{0};
    state.shift = -__builtin_inff();
    state.base = state.sum = 0.0f;
    state.shifted = false;

    if (!job.own_keys) {
        constexpr int KT = Shape::SHARED_KEYS, TILE = KT * Shape::ROW_BYTES, ROWS = 32 * WAVES;
        const int first_row = row_tile * ROWS + 32 * wave, row = first_row + lane % 32;
        const bool works = first_row < job.rows;
        att_load_queries<T, DP, ALIGNED>(args, job, entry, g, row, lane, query);
        att_wait_for_loads();
        for (int segment = job.first_segment; segment < job.last_segment; ++segment) {
            const AttentionKeys &keys = args.keys[segment];
            const i64 k_stride = keys.k_ns, v_stride = keys.v_ns;
            const bool masked = keys.mask != nullptr, causal = keys.causal;
            const int length = att_length(keys, entry);
            int begin, end;
            att_range(length, KT, split, job.splits, &begin, &end);
            // query i of a sequence's last m tokens sees the tokens up to its own
            const int limit = keys.causal ? length - args.m + 1 + row / args.r : 0x7fffffff;
            if (keys.causal) {
                const int last_row = (row_tile + 1) * ROWS < job.rows ? (row_tile + 1) * ROWS - 1 : job.rows - 1;
                const int last_limit = length - args.m + 1 + last_row / args.r;
                end = end < last_limit ? end : last_limit;
            }
            const T *k = static_cast<const T *>(keys.k) + entry * keys.k_ls + g * keys.k_gs;
            const T *v = static_cast<const T *>(keys.v) + entry * keys.v_ls + g * keys.v_gs;
            if (begin >= end) continue;
            // Iteration i: scores of tile i, then the values of tile i - 1 times their weights while the exponentials of tile i are made: the matrix
            // cores and the vector units work at the same time.  It asks for the keys of tile i + 1 and the values of tile i.
            typedef AttTile<T, DP, KT, THREADS, ALIGNED> Tile;
            att_lds_byte *key_ring = lds, *value_ring = lds + 2 * TILE;
            Tile next_k, next_v;
            att_f32x16 s[KT / 32];
            att_vec8<T> weights[KT / 16], first[AttGroups<T, DP>::COLUMNS];
            float top, base;
#pragma unroll
            for (int step = 0; step < KT / 16; ++step) weights[step] = att_vec8<T>{0};
            const float scale_log2 = args.scale_log2;
            const int k_width = args.k, v_width = args.o;
            int now = 0;                                // which of two tiles
            auto ask_keys = [&](int n, int slot) { next_k.begin(k + n * k_stride, k_stride, end - n, k_width, key_ring + slot * TILE, threadIdx.x); };
            auto ask = [&](int n, att_u64 kept) {
                if (n + KT < end) ask_keys(n + KT, now ^ 1);
                if (masked) {
                    next_v.begin(v + n * v_stride, v_stride, end - n, v_width, value_ring + now * TILE, threadIdx.x, kept);
                } else {
                    next_v.begin(v + n * v_stride, v_stride, end - n, v_width, value_ring + now * TILE, threadIdx.x);
                }
            };
            auto got = [&](int n) {                     // the keys of the next tile and the values of this one have arrived
                if (n + KT < end) next_k.finish(key_ring + (now ^ 1) * TILE, threadIdx.x);
                next_v.finish(value_ring + now * TILE, threadIdx.x);
                __syncthreads();
                now ^= 1;
            };
            __syncthreads();                            // a segment before this one is done with the buffers
            ask_keys(begin, 0);
            next_k.finish(key_ring, threadIdx.x);
            __syncthreads();
            auto rebase = [&](int n, att_u64 kept) {
                att_rebase<T, DP, KT>(state, weights, s, top, scale_log2, kept, causal, limit - n, lane);
                base = state.base;
            };
            int next_kept = 0;
            auto kept_keys = [&](int n) {
                if (!masked) return att_low_bits(end - n);
                const att_u64 kept = __ballot(next_kept != 0);
                next_kept = n + KT < end ? att_ask_kept(keys, entry, n + KT, end, lane) : 0;
                return kept;
            };
            if (masked) next_kept = att_ask_kept(keys, entry, begin, end, lane);
            att_u64 kept = kept_keys(begin);
            ask(begin, kept);
            if (works) {
                top = att_scores<T, DP, KT, ORDERED>(s, query, key_ring, lane);
                rebase(begin, kept);
#pragma unroll
                for (int step = 0; step < KT / 16; ++step) weights[step] = att_weights<T, DP, KT>(state, s, step, scale_log2, base);
            }
            got(begin);
            for (int n = begin + KT; n < end; n += KT) {
                kept = kept_keys(n);
                ask(n, kept);
                if (works) {
                    const att_lds_byte *values = value_ring + (now ^ 1) * TILE;
                    top = att_scores<T, DP, KT, ORDERED>(s, query, key_ring + now * TILE, lane);
                    att_read_columns<T, DP>(first, values, 0, 0, lane);
                    rebase(n, kept);
                    att_add_values<T, DP, KT, true, ORDERED>(state, weights, values, first, s, scale_log2, base, lane);
                }
                got(n);
            }
            if (works) {
                const att_lds_byte *values = value_ring + (now ^ 1) * TILE;
                att_read_columns<T, DP>(first, values, 0, 0, lane);
                att_add_values<T, DP, KT, false, ORDERED>(state, weights, values, first, s, 0.0f, base, lane);
            }
        }
        if (!works) return;
        att_forward_write<T, DP, ALIGNED>(args, job, state, att_sum_of_halves(state.sum), entry, g, row, split, lane);
    } else {
        constexpr int KT = Shape::OWN_KEYS;
        constexpr bool TURNS = Shape::OWN_TURNS;
        att_lds_byte *key_tile = lds + (TURNS ? 1 : 2) * wave * KT * Shape::ROW_BYTES, *value_tile = TURNS ? key_tile : key_tile + KT * Shape::ROW_BYTES;
        const int row = lane % 32;                                      // at most 32 rows: one tile
        att_load_queries<T, DP, ALIGNED>(args, job, entry, g, row, lane, query);
        for (int segment = job.first_segment; segment < job.last_segment; ++segment) {
            const AttentionKeys &keys = args.keys[segment];
            const int length = att_length(keys, entry);
            int begin, end;
            att_range(length, KT, split, job.splits, &begin, &end);
            const int limit = keys.causal ? length - args.m + 1 + row / args.r : 0x7fffffff;
            const T *k = static_cast<const T *>(keys.k) + entry * keys.k_ls + g * keys.k_gs;
            const T *v = static_cast<const T *>(keys.v) + entry * keys.v_ls + g * keys.v_gs;
            typedef AttTile<T, DP, KT, 64, ALIGNED> Tile;
            static_assert(TURNS || !Tile::DIRECT, "the next tile waits in registers");
            Tile next_k, next_v;
            auto ask_keys = [&](i64 n) { next_k.begin(k + n * keys.k_ns, keys.k_ns, end - static_cast<int>(n), args.k, key_tile, lane); };
            auto ask_values = [&](i64 n, att_u64 kept) {
                if (keys.mask) {
                    next_v.begin(v + n * keys.v_ns, keys.v_ns, end - static_cast<int>(n), args.o, value_tile, lane, kept);
                } else {
                    next_v.begin(v + n * keys.v_ns, keys.v_ns, end - static_cast<int>(n), args.o, value_tile, lane);
                }
            };
            i64 n = begin + wave * KT;
            auto ask_kept = [&](i64 n) { return n < end ? att_ask_kept(keys, entry, static_cast<int>(n), end, lane) : 0; };
            att_u64 kept = __ballot(ask_kept(n) != 0);
            int next_kept = ask_kept(n + KT * WAVES);
            if (!TURNS && n < end) {
                ask_keys(n);
                ask_values(n, kept);
            }
            for (; n < end; n += KT * WAVES) {
                const i64 at = n + KT * WAVES;
                const att_u64 then_kept = __ballot(next_kept != 0);
                next_kept = ask_kept(at + KT * WAVES);
                att_f32x16 s[KT / 32];
                att_vec8<T> weights[KT / 16] = {}, first[AttGroups<T, DP>::COLUMNS];
                float top;
                if (TURNS) {
                    att_wait_for_reads();                   // those of the values before
                    ask_keys(n);
                }
                next_k.finish(key_tile, lane);
                if (TURNS) {
                    att_wave_sync();
                    top = att_scores<T, DP, KT, ORDERED>(s, query, key_tile, lane);
                    att_wave_sync();
                    att_wait_for_reads();
                    ask_values(n, kept);
                }
                next_v.finish(value_tile, lane);
                att_wave_sync();
                if (!TURNS) {
                    if (at < end) {
                        ask_keys(at);
                        ask_values(at, then_kept);
                    }
                    top = att_scores<T, DP, KT, ORDERED>(s, query, key_tile, lane);
                }
                att_rebase<T, DP, KT>(state, weights, s, top, args.scale_log2, kept, keys.causal, limit - static_cast<int>(n), lane);
                const float base = state.base;
#pragma unroll
                for (int step = 0; step < KT / 16; ++step) weights[step] = att_weights<T, DP, KT>(state, s, step, args.scale_log2, base);
                att_read_columns<T, DP>(first, value_tile, 0, 0, lane);
                att_add_values<T, DP, KT, false, ORDERED>(state, weights, value_tile, first, s, 0.0f, base, lane);
                att_wave_sync();
                kept = then_kept;
            }
        }
        // join the waves: sums and outputs relative to the largest score that one of them has, added in the order of the waves
        float sum = att_sum_of_halves(state.sum);
        float *shifts = reinterpret_cast<float *>(lds), *bases = shifts + 32 * WAVES;      // [WAVES][32] each, then (WAVES - 1) waves' sums and outputs
        float *others = bases + 32 * WAVES;
        __syncthreads();
        if (lane < 32) {
            shifts[wave * 32 + lane] = state.shift;
            bases[wave * 32 + lane] = state.base;
        }
        __syncthreads();
        float shift = shifts[lane % 32], base = bases[lane % 32];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) {
            const float other_shift = shifts[w * 32 + lane % 32], other_base = bases[w * 32 + lane % 32];
            // a shift above 0 is larger than every base without one, and a shift below 0 smaller
            const bool larger = other_shift > shift || (other_shift == shift && other_base > base);
            shift = larger ? other_shift : shift;
            base = larger ? other_base : base;
        }
        __syncthreads();
        const float shrink = state.shift == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(__builtin_fmaf(state.shift - shift, args.scale_log2, state.base - base));
        state.shift = shift;
        state.base = base;
        sum *= shrink;
#pragma unroll
        for (int o = 0; o < DP / 32; ++o) state.out[o] *= shrink;
        if (wave > 0) {
            float *mine = others + (wave - 1) * (DP * 32 + 64);
#pragma unroll
            for (int o = 0; o < DP / 32; ++o)
#pragma unroll
                for (int i = 0; i < 16; ++i) mine[(16 * o + i) * 64 + lane] = state.out[o][i];
            mine[DP * 32 + lane] = sum;
        }
        __syncthreads();
        if (wave > 0) return;
#pragma unroll 1
        for (int w = 0; w < WAVES - 1; ++w) {
            const float *from = others + w * (DP * 32 + 64);
#pragma unroll
            for (int o = 0; o < DP / 32; ++o)
#pragma unroll
                for (int i = 0; i < 16; ++i) state.out[o][i] += from[(16 * o + i) * 64 + lane];
            sum += from[DP * 32 + lane];
        }
        att_forward_write<T, DP, ALIGNED>(args, job, state, sum, entry, g, row, split, lane);
    }
}

// The partial results of one row, weighted by exp(lse of the part - lse of all).  A wave per row, the parts in their order.  The weights come
// first, a lane per part, so that the loads of the results, eight parts at a time, do not wait for them one by one.  They are relative to the part with the
// largest shift, and the largest lse among those (without keys both are -inf).
template <typename T>
__global__ __launch_bounds__(256) void attention_join(const AttentionArgs args)
{
    const int lane = threadIdx.x & 63;
    static_assert(ATT_MAX_SLOTS == 128, "two parts per lane");
    for (i64 id = static_cast<i64>(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); id < args.rows_total; id += static_cast<i64>(gridDim.x) * 4) {
        float shifts[2], lses[2], weight[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const bool part = 64 * j + lane < args.slots;
            shifts[j] = part ? args.partial_shift[(64 * j + lane) * args.rows_total + id] : -__builtin_inff();
            lses[j] = part ? args.partial_lse[(64 * j + lane) * args.rows_total + id] : -__builtin_inff();
        }
        float shift = fmaxf(shifts[0], shifts[1]);
#pragma unroll
        for (int step = 32; step > 0; step >>= 1) shift = fmaxf(shift, __shfl_xor(shift, step));
        float base = fmaxf(shifts[0] == shift ? lses[0] : -__builtin_inff(), shifts[1] == shift ? lses[1] : -__builtin_inff());
#pragma unroll
        for (int step = 32; step > 0; step >>= 1) base = fmaxf(base, __shfl_xor(base, step));
#pragma unroll
        for (int j = 0; j < 2; ++j)
            weight[j] = shifts[j] == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(__builtin_fmaf(shifts[j] - shift, args.scale_log2, lses[j] - base));
        float sum = weight[0] + weight[1];
#pragma unroll
        for (int step = 32; step > 0; step >>= 1) sum += __shfl_xor(sum, step);
        float out[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        constexpr int AT_ONCE = 8;
        for (int part = 0; part < args.slots; part += AT_ONCE) {
            float x[AT_ONCE][4];
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u) {
                const i64 slot = (part + u < args.slots ? part + u : 0) * args.rows_total + id;
#pragma unroll
                for (int j = 0; j < 4; ++j) x[u][j] = 64 * j + lane < args.o ? args.partial_out[slot * args.partial_width + 64 * j + lane] : 0.0f;
            }
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u) {
                const float w = part + u < args.slots ? __shfl(weight[part >= 64], (part + u) & 63) : 0.0f;
#pragma unroll
                for (int j = 0; j < 4; ++j) out[j] += w != 0.0f ? w * x[u][j] : 0.0f;         // a part without keys wrote nothing
            }
        }
        const float inverse = sum > 0.0f ? 1.0f / sum : sum == 0.0f ? 0.0f : sum;
        const i64 token = id / (static_cast<i64>(args.g) * args.r);
        const int head = static_cast<int>(id % (static_cast<i64>(args.g) * args.r));
        if (args.lse && lane == 0) args.lse[id] = att_natural_lse(shift, sum == 0.0f ? -__builtin_inff() : base + __builtin_amdgcn_logf(sum), args.scale_log2);
        T *to = static_cast<T *>(args.out) + token / args.m * args.out_ls + token % args.m * args.out_ms + head * args.out_hs;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (64 * j + lane < args.o) to[64 * j + lane] = static_cast<T>(out[j] * inverse);
    }
}

}  // namespace kmc
