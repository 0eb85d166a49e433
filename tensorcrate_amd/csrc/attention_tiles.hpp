// What the attention kernels of one element type S share: matrix products over
// 16-byte operand words, tiles of rows in LDS that are read by rows and by
// columns, and the words of a head's row.
#pragma once

#include "heads.hpp"

namespace tc {
namespace attention {

constexpr uint32_t kNone = 0xffffffffu;
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

#if defined(TC_ATTENTION_TYPE)

namespace {

using S = TC_ATTENTION_TYPE;

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr bool kWide = sizeof(S) == 4;
constexpr int E = kWordElements<S>;        // elements of a 16-byte word
constexpr bool kHalf = Elem<S>::dtype == TC_F16;
// Elements of the summed axis that one operand word of both halves of a wave
// covers: a word's elements in each half.
constexpr int kDeep = 2 * E;

// acc += a . b over kDeep elements: lane l has row (or column) l % 32 of a (or
// b), and of the summed axis what its half l / 32 holds, the same in both.
__device__ __forceinline__ f32x16 product(uint4 a, uint4 b, f32x16 acc) {
    if constexpr (kWide) {
        acc = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.x), __uint_as_float(b.x), acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.y), __uint_as_float(b.y), acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.z), __uint_as_float(b.z), acc, 0, 0, 0);
        return __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.w), __uint_as_float(b.w), acc, 0, 0, 0);
    } else if constexpr (kHalf) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), acc,
                                                      0, 0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b),
                                                       acc, 0, 0, 0);
    }
}

// Register i of a 32 x 32 result is its row `row_of(i, half)`, column l % 32.
__device__ __forceinline__ int row_of(int i, int half) { return 8 * (i / 4) + 4 * half + i % 4; }

// Registers n E .. n E + E of a result as operand word n, summed over the rows.
__device__ __forceinline__ uint4 operand(const f32x16& v, int n) {
    Words<S, E> out;
    float part[E];
#pragma unroll
    for (int e = 0; e < E; e++) part[e] = v[n * E + e];
    out.put(part);
    return out.w[0];
}

// ---- tiles in LDS -------------------------------------------------------------------

// ROWS rows of SIZE elements (a multiple of 32, zeros behind a head's own) in
// 16-byte words.  Within groups of kGroup words a row's words are permuted by
// an exclusive or with `mixed(row)`, so that neither 16 rows' words of one
// column nor 4 rows' of a transposing read meet in a bank (64 banks, 256
// bytes).  `mixed` only moves bits, so that the place of (row, word) is one
// number of the lane, exclusive-ored and added to what is the same in all
// lanes: the reads below take that number (`Lanes`), and few registers hold
// all addresses.
struct Lanes {
    uint32_t row;     // of `by_row`
    uint32_t column;  // of `by_column`
};

template <int SIZE, int ROWS>
struct Tile {
    static constexpr int kWords = SIZE / E;  // of a row: 4, 8, 12, 16, 24 or 32
    static constexpr int kGroup = kWords % 16 == 0 ? 16 : kWords % 8 == 0 ? 8 : 4;
    static constexpr int kBytes = ROWS * kWords * 16;
    char* at;

    __device__ __forceinline__ static constexpr int mixed(int row) {
        return kGroup == 16  ? (row & 3) << 2 | (row >> 2 & 3)
               : kGroup == 8 ? (row >> 1 & 1) << 2 | (row >> 2 & 3)
                             : row >> 2 & 3;
    }
    __device__ __forceinline__ static int permuted(int row, int word) { return word ^ mixed(row); }
    __device__ __forceinline__ static uint32_t place(int row, int word) {
        return (row * kWords + permuted(row, word)) * 16;
    }
    // The place (row, word) away from a lane's, whose row and word have none of
    // the bits of these.
    __device__ __forceinline__ char* from(uint32_t lanes, int row, int word) const {
        return at + (lanes ^ static_cast<uint32_t>((mixed(row) ^ word % kGroup) * 16)) +
               (row * kWords + word / kGroup * kGroup) * 16;
    }
    __device__ __forceinline__ static Lanes lanes_of(int lane) {
        Lanes out;
        out.row = place(lane % 32, lane / 32);
        if constexpr (kWide) {
            out.column = place(4 * (lane / 32), lane % 32 / 4) + lane % 4 * 4;
        } else {
            // Lane j of 16 addresses 4 columns of row j / 4 and receives the 4
            // rows of column j.
            out.column = place(4 * (lane / 32) + lane % 16 / 4, 2 * (lane / 16 % 2) + lane % 4 / 2) + lane % 2 * 8;
        }
        return out;
    }
    __device__ __forceinline__ char* word(int row, int word) const { return at + place(row, word); }
    // Operand word n of row `rows` + l % 32, `rows` a multiple of 32.
    __device__ __forceinline__ uint4 by_row(const Lanes& lanes, int rows, int n) const {
        return *reinterpret_cast<const uint4*>(from(lanes.row, rows, 2 * n));
    }
    // Operand word of column `columns` + l % 32, summed over the kDeep rows from
    // `rows` on in the order of `row_of`; multiples of 32 and kDeep.
    __device__ __forceinline__ uint4 by_column(const Lanes& lanes, int rows, int columns) const {
        if constexpr (kWide) {
            uint32_t v[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                v[j] = *reinterpret_cast<const uint32_t*>(from(lanes.column, rows + j, columns / E));
            }
            return make_uint4(v[0], v[1], v[2], v[3]);
        } else {
            const u32x2 a = __builtin_bit_cast(u32x2, transposed(from(lanes.column, rows, columns / E)));
            const u32x2 b = __builtin_bit_cast(u32x2, transposed(from(lanes.column, rows + 8, columns / E)));
            return make_uint4(a.x, a.y, b.x, b.y);
        }
    }
    __device__ __forceinline__ static s16x4 transposed(const char* lds) {
        return __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) s16x4*)(const_cast<char*>(lds)));
    }
    // Four consecutive elements of a row from a column that is a multiple of 4.
    __device__ __forceinline__ void four(int row, int column, float (&out)[4]) const {
        const S* from = reinterpret_cast<const S*>(word(row, column / E)) + column % E;
#pragma unroll
        for (int j = 0; j < 4; j++) out[j] = Elem<S>::widen(from[j]);
    }
};

// Word `word` of a head's row, zeros past its size.
__device__ __forceinline__ uint4 head_word(const S* row, int word, uint32_t size) {
    const uint32_t first = word * E;
    if (first + E <= size) return load_any_word<false>(row + first);
    Words<S, E> out;
    float v[E];
#pragma unroll
    for (int e = 0; e < E; e++) v[e] = first + e < size ? Elem<S>::widen(row[first + e]) : 0.0f;
    out.put(v);
    return out.w[0];
}

// The bits that infinities and NaNs have set, of each element in 32 bits.
constexpr uint32_t kSpecial = kWide ? 0x7f800000u : kHalf ? 0x7c007c00u : 0x7f807f80u;

// Whether one of the elements in these 32 bits is an infinity or a NaN; and
// the same with zeros in their place.
__device__ __forceinline__ bool special_bits(uint32_t bits) {
    if constexpr (kWide) return (bits & kSpecial) == kSpecial;
    return (bits & kSpecial & 0xffffu) == (kSpecial & 0xffffu) || (bits & kSpecial >> 16 << 16) == kSpecial >> 16 << 16;
}
__device__ __forceinline__ uint32_t finite_bits(uint32_t bits) {
    if constexpr (kWide) return special_bits(bits) ? 0u : bits;
    if ((bits & kSpecial & 0xffffu) == (kSpecial & 0xffffu)) bits &= 0xffff0000u;
    if ((bits & kSpecial >> 16 << 16) == kSpecial >> 16 << 16) bits &= 0xffffu;
    return bits;
}

__device__ __forceinline__ float power2(float v) { return __builtin_amdgcn_exp2f(v); }

}  // namespace

#endif  // TC_ATTENTION_TYPE

}  // namespace attention
}  // namespace tc
