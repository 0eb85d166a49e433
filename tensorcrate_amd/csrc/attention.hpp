// Causal attention over packed sequences, forward and backward: the kernels,
// for one element type S (attention_*.hip builds them).
//
// With c = scale, over the keys j that query i sees (those of its own sequence
// up to itself; query heads share key heads in groups):
//   s_ij = c q_i . k_j,  l_i = log sum_j exp s_ij,  p_ij = exp(s_ij - l_i)
//   o_i = sum_j p_ij v_j
// and from do, with the s_ij and p_ij computed again,
//   D_i = do_i . o_i,  ds_ij = p_ij (do_i . v_j - D_i)
//   dq_i = c sum_j ds_ij k_j,  dk_j = c sum_i ds_ij q_i,  dv_j = sum_i p_ij do_i
// Forward, the sum over j runs once over tiles of keys with a running maximum;
// backward, one kernel sums over keys (dq) and one over queries (dk, dv), so
// that each result is written by one wave in one order, at the price of
// computing s and do . v twice: 7 products where 5 would do with atomics,
// whose order would change the bits.
//
// All of it is bound by the matrix cores and by the vector unit's exponentials
// beside them.  A wave holds 32 queries (32 keys for dk, dv) as the columns of
// 32 x 32 products whose other operand comes from a tile in LDS that the
// block's four waves share: s transposed is k . q^T, so a lane has 16 keys of
// one query, sums over keys are sums in its registers (and one exchange with
// the lane that has the other 16), and those registers, rounded, are already
// the operand of the next product, o^T = v^T . p^T, if the sum over keys runs
// in the order in which lanes hold them.  That product reads v's tile by
// columns: with gfx950's transposing LDS read for 16-bit types, element by
// element for f32.  p and ds are rounded to the operands' type for it, once;
// sums, maxima and all else are f32.  The least normal f16 is 2^-14, which p
// of a long sequence and ds fall below: in f16 p is rounded times 2^14 (or 2^6
// forward, where it may reach 2^8), and ds, which is at most twice the largest
// |do| times the largest |v|, times the power of two that brings that below
// 2^15.
//
// Sequences lie one behind another, and tiles of tokens do not stop at their
// ends: a tile that some row of a wave sees only in part is masked element by
// element.  A masked weight is 0, and 0 times an infinity or a NaN would be a
// NaN, so a tile that is masked and holds such a value takes a slow path: the
// product with zeros in their place, then theirs alone where the weight is not
// 0.
#pragma once

#include <type_traits>

#include "rows.hpp"

namespace tc {
namespace attention {

constexpr int kThreads = 256;
constexpr uint32_t kOwned = 128;  // queries (or keys) of a block, 32 a wave
constexpr uint32_t kNone = 0xffffffffu;
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

struct Steps {
    uint64_t token, head;
};

struct Shape {
    uint32_t heads, group;  // query heads, and of them to a key head
    uint32_t size;
    uint32_t tokens;
    uint32_t sequences;  // 0: all tokens are one
    const uint32_t* offsets;
    float scale;
    Steps q, k, v, out;
};

// The launches of one element type.
struct Launches {
    int (*forward)(const Shape&, const void* q, const void* k, const void* v, void* out, float* normalizers);
    int (*backward)(const Shape&, const void* d_out, const void* q, const void* k, const void* v, const void* out,
                    const float* normalizers, void* dq, void* dk, void* dv);
};
const Launches& f32_launches();
const Launches& f16_launches();
const Launches& bf16_launches();

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
constexpr uint32_t kSwept = kWide ? 32 : 64;  // rows of a tile in LDS
constexpr bool kHalf = Elem<S>::dtype == TC_F16;
// Powers of two that weights are rounded times, forward and backward.
constexpr float kForwardPower = kHalf ? 6.0f : 0.0f, kBackPower = kHalf ? 14.0f : 0.0f;
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
// 16-byte words.  A row's words are permuted within groups by its number, so
// that neither 16 rows' words of one column nor 4 rows' of a transposing read
// meet in a bank (64 banks, 256 bytes).
template <int SIZE, int ROWS>
struct Tile {
    static constexpr int kWords = SIZE / E;  // of a row: 4, 8, 12, 16, 24 or 32
    static constexpr int kBytes = ROWS * kWords * 16;
    char* at;

    __device__ __forceinline__ static int permuted(int row, int word) {
        if constexpr (kWords % 16 == 0) return word ^ ((row & 3) << 2 | (row >> 2 & 3));
        if constexpr (kWords % 8 == 0) return word ^ ((row >> 1 & 1) << 2 | (row >> 2 & 3));
        return word ^ (row >> 2 & 3);
    }
    __device__ __forceinline__ char* word(int row, int word) const {
        return at + (row * kWords + permuted(row, word)) * 16;
    }
    // Operand word n of row `row`, which is this lane's own row.
    __device__ __forceinline__ uint4 by_row(int row, int n, int half) const {
        return *reinterpret_cast<const uint4*>(word(row, 2 * n + half));
    }
    // Operand word of column `columns` + l % 32, summed over the kDeep rows from
    // `rows` on in the order of `row_of`.
    __device__ __forceinline__ uint4 by_column(int rows, int columns, int lane) const {
        if constexpr (kWide) {
            float v[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int column = columns + lane % 32;
                v[j] = reinterpret_cast<const float*>(word(rows + 4 * (lane / 32) + j, column / E))[column % E];
            }
            return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]),
                              __float_as_uint(v[3]));
        } else {
            // Lane j of 16 addresses 4 columns of row j / 4 and receives the 4
            // rows of column j.
            const int row = rows + 4 * (lane / 32) + lane % 16 / 4;
            const int column = columns + 16 * (lane / 16 % 2) + 4 * (lane % 4);
            const s16x4 low = transposed(word(row, column / E) + column % E * 2);
            const s16x4 high = transposed(word(row + 8, column / E) + column % E * 2);
            const u32x2 a = __builtin_bit_cast(u32x2, low), b = __builtin_bit_cast(u32x2, high);
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

// A tile on its way from memory: each thread's words of it in registers.
template <int SIZE, int ROWS>
struct Flight {
    static constexpr int kWords = SIZE / E;
    static constexpr int kEach = ROWS * kWords / kThreads;
    static_assert(ROWS * kWords % kThreads == 0, "every thread has as many words");
    uint4 words[kEach];

    // Rows first .. first + ROWS of a head, zeros from token `limit` on.
    __device__ __forceinline__ void load(const S* head, uint64_t step, uint32_t first, uint32_t limit, uint32_t size) {
#pragma unroll
        for (int k = 0; k < kEach; k++) {
            const int i = threadIdx.x + k * kThreads;
            const uint32_t token = first + i / kWords;
            words[k] = token < limit ? head_word(head + token * step, i % kWords, size) : make_uint4(0, 0, 0, 0);
        }
    }
    __device__ __forceinline__ void store(const Tile<SIZE, ROWS>& tile) const {
#pragma unroll
        for (int k = 0; k < kEach; k++) {
            const int i = threadIdx.x + k * kThreads;
            *reinterpret_cast<uint4*>(tile.word(i / kWords, i % kWords)) = words[k];
        }
    }
    // Whether any of this thread's elements is an infinity or a NaN.
    __device__ __forceinline__ bool special() const {
        bool any = false;
#pragma unroll
        for (int k = 0; k < kEach; k++) {
            any |= special_bits(words[k].x) || special_bits(words[k].y) || special_bits(words[k].z) ||
                   special_bits(words[k].w);
        }
        return any;
    }
};

// ---- sequences ------------------------------------------------------------------------

struct Span {
    uint32_t first, end;  // of the token's sequence; kNone, 0 if it is in none
};

// Whatever the offsets hold, a span lies within the tokens.
__device__ __forceinline__ Span span_of(const Shape& shape, uint32_t token) {
    if (token >= shape.tokens) return {kNone, 0};
    if (shape.sequences == 0) return {0, shape.tokens};
    uint32_t low = 0, high = shape.sequences;
    while (high - low > 1) {
        const uint32_t middle = (low + high) / 2;
        if (shape.offsets[middle] <= token) low = middle;
        else high = middle;
    }
    const uint32_t first = shape.offsets[low], end = shape.offsets[low + 1];
    if (token < first || token >= end) return {kNone, 0};
    return {first, end < shape.tokens ? end : shape.tokens};
}

// The token behind the last sequence.
__device__ __forceinline__ uint32_t limit_of(const Shape& shape) {
    if (shape.sequences == 0) return shape.tokens;
    const uint32_t end = shape.offsets[shape.sequences];
    return end < shape.tokens ? end : shape.tokens;
}

__device__ __forceinline__ uint32_t wave_least(uint32_t v) {
    for (int offset = 32; offset > 0; offset >>= 1) {
        const uint32_t other = __shfl_xor(v, offset);
        v = other < v ? other : v;
    }
    return __builtin_amdgcn_readfirstlane(v);
}
__device__ __forceinline__ uint32_t wave_most(uint32_t v) { return ~wave_least(~v); }

// The least of the waves' first values and the most of their second ones.
__device__ __forceinline__ void over_waves(const uint32_t (&values)[2][kThreads / 64], uint32_t* least, uint32_t* most) {
    *least = values[0][0], *most = values[1][0];
    for (int w = 1; w < kThreads / 64; w++) {
        *least = values[0][w] < *least ? values[0][w] : *least;
        *most = values[1][w] > *most ? values[1][w] : *most;
    }
}

// `v` of this lane and of the one that has the same column in the other half.
__device__ __forceinline__ float halves_most(float v) {
    const uint32_t bits = __float_as_uint(v);
    const auto both = __builtin_amdgcn_permlane32_swap(bits, bits, false, false);
    return fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1]));
}
__device__ __forceinline__ float halves_sum(float v) {
    const uint32_t bits = __float_as_uint(v);
    const auto both = __builtin_amdgcn_permlane32_swap(bits, bits, false, false);
    return __uint_as_float(both[0]) + __uint_as_float(both[1]);
}

__device__ __forceinline__ float power2(float v) { return __builtin_amdgcn_exp2f(v); }

// ---- sums over a tile's rows ------------------------------------------------------------

// acc (SIZE x 32 columns) += the transpose of 32 rows of the tile times the
// 32 x 32 weights; with FINITE, of the tile's finite elements.
template <int SIZE, int ROWS, bool FINITE>
__device__ __forceinline__ void weighted(f32x16 (&acc)[SIZE / 32], const Tile<SIZE, ROWS>& tile, int rows,
                                         const f32x16& weights, int lane) {
#pragma unroll
    for (int n = 0; n < 32 / kDeep; n++) {
        const uint4 weight = operand(weights, n);
#pragma unroll
        for (int t = 0; t < SIZE / 32; t++) {
            uint4 column = tile.by_column(rows + n * kDeep, t * 32, lane);
            if constexpr (FINITE) {
                column = make_uint4(finite_bits(column.x), finite_bits(column.y), finite_bits(column.z),
                                    finite_bits(column.w));
            }
            acc[t] = product(column, weight, acc[t]);
        }
    }
}

// The products of the tile's other elements with weights that are not 0, 8
// rows at a time through `scratch` (8 x 32 floats of the wave's own).
template <int SIZE, int ROWS>
__device__ __forceinline__ void weighted_specials(f32x16 (&acc)[SIZE / 32], const Tile<SIZE, ROWS>& tile, int rows,
                                                  const f32x16& weights, int lane, float* scratch) {
    const int half = lane / 32;
#pragma unroll
    for (int g = 0; g < 4; g++) {
        // In order within the wave, but not to be reordered by the compiler.
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int j = 0; j < 4; j++) scratch[(4 * half + j) * 32 + lane % 32] = weights[4 * g + j];
        __builtin_amdgcn_wave_barrier();
#pragma unroll 1
        for (int r = 0; r < 8; r++) {
            const float weight = scratch[r * 32 + lane % 32];
#pragma unroll
            for (int t = 0; t < SIZE / 32; t++) {
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    float v[4];
                    tile.four(rows + 8 * g + r, t * 32 + 8 * q + 4 * half, v);
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        if (weight != 0.0f && !(fabsf(v[j]) < INFINITY)) acc[t][4 * q + j] += weight * v[j];
                    }
                }
            }
        }
    }
}

// Both, where a tile is masked and `special`, or the plain product.
template <int SIZE, int ROWS>
__device__ __forceinline__ void add_weighted(bool special, f32x16 (&acc)[SIZE / 32], const Tile<SIZE, ROWS>& tile,
                                             int rows, const f32x16& weights, int lane, float* scratch) {
    if (__builtin_expect(special, false)) {
        weighted<SIZE, ROWS, true>(acc, tile, rows, weights, lane);
        weighted_specials<SIZE, ROWS>(acc, tile, rows, weights, lane, scratch);
    } else {
        weighted<SIZE, ROWS, false>(acc, tile, rows, weights, lane);
    }
}

// A lane's column of acc, scaled, to a row of `size` elements of type T.
template <typename T, int SIZE>
__device__ __forceinline__ void store_column(T* row, const f32x16 (&acc)[SIZE / 32], float scale, uint32_t size,
                                             int half) {
#pragma unroll
    for (int t = 0; t < SIZE / 32; t++) {
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const uint32_t first = t * 32 + 8 * q + 4 * half;
            T v[4];
#pragma unroll
            for (int j = 0; j < 4; j++) v[j] = Elem<T>::narrow(acc[t][4 * q + j] * scale);
            if (first + 4 <= size) {
                typedef uint32_t piece __attribute__((ext_vector_type(sizeof(T)), aligned(sizeof(T))));
                piece bits;
                __builtin_memcpy(&bits, v, sizeof(bits));
                *reinterpret_cast<piece*>(row + first) = bits;
            } else {
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    if (first + j < size) row[first + j] = v[j];
                }
            }
        }
    }
}

// ---- forward ---------------------------------------------------------------------------

template <int SIZE>
__global__ void __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(2)))
    forward_kernel(const Shape shape, const S* __restrict__ q, const S* __restrict__ k, const S* __restrict__ v,
                   S* __restrict__ out, float* __restrict__ normalizers) {
    using KeyTile = Tile<SIZE, kSwept>;
    __shared__ __attribute__((aligned(16))) char lds[4 * KeyTile::kBytes];
    __shared__ float scratch[kThreads / 64][8 * 32];
    __shared__ uint32_t seen[2][kThreads / 64];
    constexpr int kOperands = SIZE / kDeep;

    const int lane = threadIdx.x % 64, half = lane / 32, wave = threadIdx.x / 64;
    // The latest tokens, which see the most keys, first.
    const uint32_t tiles = (shape.tokens + kOwned - 1) / kOwned;
    const uint32_t head = blockIdx.x % shape.heads;
    const uint32_t first = (tiles - 1 - blockIdx.x / shape.heads) * kOwned;
    const uint32_t wave_first = first + wave * 32;
    const uint32_t token = wave_first + lane % 32;
    const Span span = span_of(shape, token);
    const uint32_t limit = limit_of(shape);
    // Keys that some, and that all, of the wave's queries may see.
    const uint32_t some = wave_least(span.first), all = wave_most(span.first);
    if (lane == 0) seen[0][wave] = some, seen[1][wave] = all;

    const S* query = q + (token < shape.tokens ? token : 0) * shape.q.token + head * shape.q.head;
    uint4 queries[kOperands];
#pragma unroll
    for (int n = 0; n < kOperands; n++) queries[n] = head_word(query, 2 * n + half, shape.size);
    __syncthreads();
    uint32_t begin, block_all;
    over_waves(seen, &begin, &block_all);

    const S* keys = k + head / shape.group * shape.k.head;
    const S* values = v + head / shape.group * shape.v.head;
    const float c = shape.scale * kLog2e;
    f32x16 acc[SIZE / 32] = {};
    float most = -INFINITY, total = 0.0f;  // of this half's keys

    const uint32_t end = first + kOwned < limit ? first + kOwned : limit;
    if (begin < end) {
        Flight<SIZE, kSwept> key_words, value_words;
        uint32_t at = begin / kSwept * kSwept;
        key_words.load(keys, shape.k.token, at, limit, shape.size);
        value_words.load(values, shape.v.token, at, limit, shape.size);
        // Masked for some query of the block (and the same for all its waves):
        // before a sequence's first key or past the first query.
        const auto masked = [&](uint32_t tile) { return tile < block_all || tile + kSwept - 1 > first; };
        int turn = 0;
        key_words.store(KeyTile{lds});
        value_words.store(KeyTile{lds + 2 * KeyTile::kBytes});
        bool special = __syncthreads_or(value_words.special());
        for (; at < end; at += kSwept, turn ^= 1) {
            const KeyTile key_tile{lds + turn * KeyTile::kBytes};
            const KeyTile value_tile{lds + (2 + turn) * KeyTile::kBytes};
            const uint32_t next = at + kSwept;
            if (next < end) {
                key_words.load(keys, shape.k.token, next, limit, shape.size);
                value_words.load(values, shape.v.token, next, limit, shape.size);
            }
            if (at < wave_first + 32 && at + kSwept > some) {
                f32x16 scores[kSwept / 32];
#pragma unroll
                for (int b = 0; b < static_cast<int>(kSwept) / 32; b++) {
                    f32x16 s = {};
#pragma unroll
                    for (int n = 0; n < kOperands; n++) {
                        s = product(key_tile.by_row(b * 32 + lane % 32, n, half), queries[n], s);
                    }
                    scores[b] = s;
                }
                const bool whole = at >= all && at + kSwept - 1 <= wave_first;
                if (!whole) {
#pragma unroll
                    for (int b = 0; b < static_cast<int>(kSwept) / 32; b++) {
#pragma unroll
                        for (int i = 0; i < 16; i++) {
                            const uint32_t key = at + b * 32 + row_of(i, half);
                            if (key < span.first || key > token) scores[b][i] = -INFINITY;
                        }
                    }
                }
                float high = -INFINITY;
#pragma unroll
                for (int b = 0; b < static_cast<int>(kSwept) / 32; b++) {
#pragma unroll
                    for (int i = 0; i < 16; i++) high = fmaxf(high, scores[b][i]);
                }
                high = halves_most(high) * c;
                // The maximum only moves when it grows past 2^8: the weights
                // stay that small, and the sums are rarely rescaled.
                const bool grows = high > most + 8.0f;
                if (__ballot(grows) != 0) {
                    const float factor = grows ? power2(most - high) : 1.0f;
                    if (grows) most = high;
                    total *= factor;
#pragma unroll
                    for (int t = 0; t < SIZE / 32; t++) acc[t] *= factor;
                }
                const float origin = (most == -INFINITY ? 0.0f : most) - kForwardPower;
#pragma unroll
                for (int b = 0; b < static_cast<int>(kSwept) / 32; b++) {
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        scores[b][i] = power2(fmaf(scores[b][i], c, -origin));
                        total += scores[b][i];
                    }
                }
#pragma unroll
                for (int b = 0; b < static_cast<int>(kSwept) / 32; b++) {
                    add_weighted<SIZE, kSwept>(!whole && special, acc, value_tile, b * 32, scores[b], lane, scratch[wave]);
                }
            }
            if (next < end) {
                key_words.store(KeyTile{lds + (turn ^ 1) * KeyTile::kBytes});
                value_words.store(KeyTile{lds + (2 + (turn ^ 1)) * KeyTile::kBytes});
                if (masked(next)) {
                    special = __syncthreads_or(value_words.special());
                } else {
                    special = false;
                    __syncthreads();
                }
            }
        }
    }
    total = halves_sum(total);
    if (token >= shape.tokens) return;
    store_column<S, SIZE>(out + token * shape.out.token + head * shape.out.head, acc, total == 0.0f ? 0.0f : 1.0f / total,
                          shape.size, half);
    if (normalizers != nullptr && half == 0) {
        normalizers[uint64_t{head} * shape.tokens + token] =
            total == 0.0f ? -INFINITY : (most + log2f(total) - kForwardPower) * kLn2;
    }
}

// ---- backward ----------------------------------------------------------------------------

// sums[head][token] = do . o, 16 lanes a row of a head; and in f16 the bits of
// the largest finite |do|^2 and |v|^2 of any row into `largest`.
__global__ void __launch_bounds__(kThreads)
    dots_kernel(const Shape shape, const S* __restrict__ d_out, const S* __restrict__ out, const S* __restrict__ v,
                float* __restrict__ sums, uint32_t* __restrict__ largest) {
    const uint64_t first = uint64_t{blockIdx.x} * (kThreads / 16) + threadIdx.x / 16;
    const uint64_t apart = uint64_t{gridDim.x} * (kThreads / 16);
    const auto dot = [&](const S* a, const S* b) {
        float sum = 0.0f;
        for (uint32_t word = threadIdx.x % 16; word * E < shape.size; word += 16) {
            const Words<S, E> x{{head_word(a, word, shape.size)}}, y{{head_word(b, word, shape.size)}};
#pragma unroll
            for (int e = 0; e < E; e++) sum = fmaf(x.at(e), y.at(e), sum);
        }
        return row16<Added>(sum);
    };
    float most[2] = {};
    const auto note = [&](int which, float square) {
        if (square < INFINITY) most[which] = fmaxf(most[which], square);
    };
    for (uint64_t row = first; row < uint64_t{shape.tokens} * shape.heads; row += apart) {
        const uint32_t token = static_cast<uint32_t>(row / shape.heads), head = static_cast<uint32_t>(row % shape.heads);
        const uint64_t at = token * shape.out.token + head * shape.out.head;
        const float sum = dot(d_out + at, out + at);
        if (threadIdx.x % 16 == 0) sums[uint64_t{head} * shape.tokens + token] = sum;
        if constexpr (kHalf) note(0, dot(d_out + at, d_out + at));
    }
    if constexpr (kHalf) {
        const uint32_t heads = shape.heads / shape.group;
        for (uint64_t row = first; row < uint64_t{shape.tokens} * heads; row += apart) {
            const S* value = v + row / heads * shape.v.token + row % heads * shape.v.head;
            note(1, dot(value, value));
        }
        __shared__ float shared[2][kMostWaves];
        for (int which = 0; which < 2; which++) {
            const float all = block_join<Largest>(most[which], shared[which]);
            if (threadIdx.x == 0) atomicMax(largest + which, __float_as_uint(all));
        }
    }
}

// The power of two that ds is rounded times.
__device__ __forceinline__ float ds_factor(const uint32_t* largest) {
    if constexpr (!kHalf) return 1.0f;
    const float bound = sqrtf(__uint_as_float(largest[0])) * sqrtf(__uint_as_float(largest[1]));
    return bound == 0.0f ? 1.0f : ldexpf(1.0f, 13 - ilogbf(bound));
}

// dq: as forward, with the weights from the normalizers.
template <int SIZE>
__global__ void __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(2)))
    queries_kernel(const Shape shape, const S* __restrict__ d_out, const S* __restrict__ q, const S* __restrict__ k,
                   const S* __restrict__ v, const float* __restrict__ normalizers, const float* __restrict__ dots,
                   const uint32_t* __restrict__ largest, S* __restrict__ dq) {
    using KeyTile = Tile<SIZE, kSwept>;
    __shared__ __attribute__((aligned(16))) char lds[4 * KeyTile::kBytes];
    __shared__ float scratch[kThreads / 64][8 * 32];
    __shared__ uint32_t seen[2][kThreads / 64];
    constexpr int kOperands = SIZE / kDeep;

    const int lane = threadIdx.x % 64, half = lane / 32, wave = threadIdx.x / 64;
    const uint32_t tiles = (shape.tokens + kOwned - 1) / kOwned;
    const uint32_t head = blockIdx.x % shape.heads;
    const uint32_t first = (tiles - 1 - blockIdx.x / shape.heads) * kOwned;
    const uint32_t wave_first = first + wave * 32;
    const uint32_t token = wave_first + lane % 32;
    const Span span = span_of(shape, token);
    const uint32_t limit = limit_of(shape);
    const uint32_t some = wave_least(span.first), all = wave_most(span.first);
    if (lane == 0) seen[0][wave] = some, seen[1][wave] = all;

    const uint32_t inside = token < shape.tokens ? token : 0;
    const S* query = q + inside * shape.q.token + head * shape.q.head;
    const S* d_row = d_out + inside * shape.out.token + head * shape.out.head;
    uint4 queries[kOperands], d_rows[kOperands];
#pragma unroll
    for (int n = 0; n < kOperands; n++) {
        queries[n] = head_word(query, 2 * n + half, shape.size);
        d_rows[n] = head_word(d_row, 2 * n + half, shape.size);
    }
    const float normalizer = normalizers[uint64_t{head} * shape.tokens + inside] * kLog2e;
    const float factor = ds_factor(largest);
    const float dot = dots[uint64_t{head} * shape.tokens + inside] * factor;
    __syncthreads();
    uint32_t begin, block_all;
    over_waves(seen, &begin, &block_all);

    const S* keys = k + head / shape.group * shape.k.head;
    const S* values = v + head / shape.group * shape.v.head;
    const float c = shape.scale * kLog2e;
    f32x16 acc[SIZE / 32] = {};

    const uint32_t end = first + kOwned < limit ? first + kOwned : limit;
    if (begin < end) {
        Flight<SIZE, kSwept> key_words, value_words;
        uint32_t at = begin / kSwept * kSwept;
        key_words.load(keys, shape.k.token, at, limit, shape.size);
        value_words.load(values, shape.v.token, at, limit, shape.size);
        const auto masked = [&](uint32_t tile) { return tile < block_all || tile + kSwept - 1 > first; };
        int turn = 0;
        key_words.store(KeyTile{lds});
        value_words.store(KeyTile{lds + 2 * KeyTile::kBytes});
        bool special = __syncthreads_or(key_words.special());
        for (; at < end; at += kSwept, turn ^= 1) {
            const KeyTile key_tile{lds + turn * KeyTile::kBytes};
            const KeyTile value_tile{lds + (2 + turn) * KeyTile::kBytes};
            const uint32_t next = at + kSwept;
            if (next < end) {
                key_words.load(keys, shape.k.token, next, limit, shape.size);
                value_words.load(values, shape.v.token, next, limit, shape.size);
            }
            if (at < wave_first + 32 && at + kSwept > some) {
                const bool whole = at >= all && at + kSwept - 1 <= wave_first;
#pragma unroll
                for (int b = 0; b < static_cast<int>(kSwept) / 32; b++) {
                    f32x16 s = {}, d = {};
#pragma unroll
                    for (int n = 0; n < kOperands; n++) {
                        s = product(key_tile.by_row(b * 32 + lane % 32, n, half), queries[n], s);
                        d = product(value_tile.by_row(b * 32 + lane % 32, n, half), d_rows[n], d);
                    }
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        s[i] = power2(fmaf(s[i], c, -normalizer)) * fmaf(d[i], factor, -dot);
                    }
                    if (!whole) {
#pragma unroll
                        for (int i = 0; i < 16; i++) {
                            const uint32_t key = at + b * 32 + row_of(i, half);
                            if (key < span.first || key > token) s[i] = 0.0f;
                        }
                    }
                    add_weighted<SIZE, kSwept>(!whole && special, acc, key_tile, b * 32, s, lane, scratch[wave]);
                }
            }
            if (next < end) {
                key_words.store(KeyTile{lds + (turn ^ 1) * KeyTile::kBytes});
                value_words.store(KeyTile{lds + (2 + (turn ^ 1)) * KeyTile::kBytes});
                if (masked(next)) {
                    special = __syncthreads_or(key_words.special());
                } else {
                    special = false;
                    __syncthreads();
                }
            }
        }
    }
    if (token >= shape.tokens) return;
    store_column<S, SIZE>(dq + token * shape.q.token + head * shape.q.head, acc, shape.scale / factor, shape.size, half);
}

// dk and dv of 128 keys from the queries of one of `splits` shares of the
// heads that the key head serves.  With several shares they are left in f32
// as `parts`[key head][share][dk, dv][token][size], to be added in their order.
template <int SIZE>
__global__ void __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(1)))
    keys_kernel(const Shape shape, uint32_t splits, const S* __restrict__ d_out, const S* __restrict__ q,
                const S* __restrict__ k, const S* __restrict__ v, const float* __restrict__ normalizers,
                const float* __restrict__ dots, const uint32_t* __restrict__ largest, S* __restrict__ dk, S* __restrict__ dv,
                float* __restrict__ parts) {
    using QueryTile = Tile<SIZE, kSwept>;
    __shared__ __attribute__((aligned(16))) char lds[4 * QueryTile::kBytes];
    __shared__ __attribute__((aligned(16))) float row_values[2][2][kSwept];
    __shared__ float scratch[kThreads / 64][8 * 32];
    __shared__ uint32_t seen[2][kThreads / 64];
    constexpr int kOperands = SIZE / kDeep;

    const int lane = threadIdx.x % 64, half = lane / 32, wave = threadIdx.x / 64;
    // The first tokens, which are seen by the most queries, first.
    const uint32_t key_heads = shape.heads / shape.group;
    const uint32_t columns = key_heads * splits;
    const uint32_t key_head = blockIdx.x % columns / splits, share = blockIdx.x % splits;
    const uint32_t share_heads = shape.group / splits;
    const uint32_t first_head = key_head * shape.group + share * share_heads;
    const uint32_t first = blockIdx.x / columns * kOwned;
    const uint32_t wave_first = first + wave * 32;
    const uint32_t token = wave_first + lane % 32;
    const Span span = span_of(shape, token);
    const uint32_t limit = limit_of(shape);
    // Queries before which all, and some, of the wave's keys are seen.
    const uint32_t all = wave_least(span.end), some = wave_most(span.end);
    if (lane == 0) seen[0][wave] = all, seen[1][wave] = some;

    const uint32_t inside = token < shape.tokens ? token : 0;
    const S* key = k + inside * shape.k.token + key_head * shape.k.head;
    const S* value = v + inside * shape.v.token + key_head * shape.v.head;
    uint4 keys[kOperands], values[kOperands];
#pragma unroll
    for (int n = 0; n < kOperands; n++) {
        keys[n] = head_word(key, 2 * n + half, shape.size);
        values[n] = head_word(value, 2 * n + half, shape.size);
    }
    __syncthreads();
    uint32_t block_all, end;
    over_waves(seen, &block_all, &end);

    const float c = shape.scale * kLog2e;
    // p is rounded times 2^kBackPower, ds times `factor`.
    const float factor = ds_factor(largest), ds_scale = factor * power2(-kBackPower);
    f32x16 acc_k[SIZE / 32] = {}, acc_v[SIZE / 32] = {};
    if (first < end) {
        Flight<SIZE, kSwept> query_words, d_words;
        float row_value = 0.0f;  // of one row: threads below kSwept the normalizer, the next ones the dot
        const uint32_t per_head = (end - first + kSwept - 1) / kSwept;
        const uint32_t turns = per_head * share_heads;
        const auto load = [&](uint32_t n) {
            const uint32_t head = first_head + n / per_head, at = first + n % per_head * kSwept;
            query_words.load(q + head * shape.q.head, shape.q.token, at, limit, shape.size);
            d_words.load(d_out + head * shape.out.head, shape.out.token, at, limit, shape.size);
            if (threadIdx.x < 2 * kSwept) {
                const uint32_t row = at + threadIdx.x % kSwept;
                const float* from = threadIdx.x < kSwept ? normalizers : dots;
                row_value = row < limit ? from[uint64_t{head} * shape.tokens + row] : 0.0f;
                row_value = threadIdx.x < kSwept ? fmaf(row_value, kLog2e, -kBackPower) : row_value * ds_scale;
            }
        };
        const auto store = [&](int turn) {
            query_words.store(QueryTile{lds + turn * QueryTile::kBytes});
            d_words.store(QueryTile{lds + (2 + turn) * QueryTile::kBytes});
            if (threadIdx.x < 2 * kSwept) row_values[turn][threadIdx.x / kSwept][threadIdx.x % kSwept] = row_value;
        };
        // Masked for some key of the block: before its last key, or past a
        // sequence's end.
        const auto masked = [&](uint32_t at) { return at < first + kOwned - 1 || at + kSwept > block_all; };
        load(0);
        store(0);
        bool special = __syncthreads_or(query_words.special() || d_words.special());
        for (uint32_t n = 0; n < turns; n++) {
            const int turn = n % 2;
            const uint32_t at = first + n % per_head * kSwept;
            const QueryTile query_tile{lds + turn * QueryTile::kBytes};
            const QueryTile d_tile{lds + (2 + turn) * QueryTile::kBytes};
            if (n + 1 < turns) load(n + 1);
            if (at + kSwept > wave_first && at < some) {
                const bool whole = at >= wave_first + 31 && at + kSwept <= all;
#pragma unroll
                for (int b = 0; b < static_cast<int>(kSwept) / 32; b++) {
                    f32x16 s = {}, d = {};
#pragma unroll
                    for (int n = 0; n < kOperands; n++) {
                        s = product(query_tile.by_row(b * 32 + lane % 32, n, half), keys[n], s);
                        d = product(d_tile.by_row(b * 32 + lane % 32, n, half), values[n], d);
                    }
#pragma unroll
                    for (int g = 0; g < 4; g++) {
                        const int row = b * 32 + 8 * g + 4 * half;
                        const float4 normalizer = *reinterpret_cast<const float4*>(&row_values[turn][0][row]);
                        const float4 dot = *reinterpret_cast<const float4*>(&row_values[turn][1][row]);
                        const float l[4] = {normalizer.x, normalizer.y, normalizer.z, normalizer.w};
                        const float o[4] = {dot.x, dot.y, dot.z, dot.w};
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            s[4 * g + j] = power2(fmaf(s[4 * g + j], c, -l[j]));
                            d[4 * g + j] = s[4 * g + j] * fmaf(d[4 * g + j], ds_scale, -o[j]);
                        }
                    }
                    if (!whole) {
#pragma unroll
                        for (int i = 0; i < 16; i++) {
                            const uint32_t query = at + b * 32 + row_of(i, half);
                            if (query < token || query >= span.end) s[i] = 0.0f, d[i] = 0.0f;
                        }
                    }
                    add_weighted<SIZE, kSwept>(!whole && special, acc_v, d_tile, b * 32, s, lane, scratch[wave]);
                    add_weighted<SIZE, kSwept>(!whole && special, acc_k, query_tile, b * 32, d, lane, scratch[wave]);
                }
            }
            if (n + 1 < turns) {
                store(turn ^ 1);
                if (masked(first + (n + 1) % per_head * kSwept)) {
                    special = __syncthreads_or(query_words.special() || d_words.special());
                } else {
                    special = false;
                    __syncthreads();
                }
            }
        }
    }
    if (token >= shape.tokens) return;
    const float scale_k = shape.scale / factor, scale_v = power2(-kBackPower);
    if (splits == 1) {
        store_column<S, SIZE>(dk + token * shape.k.token + key_head * shape.k.head, acc_k, scale_k, shape.size, half);
        store_column<S, SIZE>(dv + token * shape.v.token + key_head * shape.v.head, acc_v, scale_v, shape.size, half);
    } else {
        const uint64_t plane = uint64_t{shape.tokens} * shape.size;
        float* to = parts + (uint64_t{key_head} * splits + share) * 2 * plane + uint64_t{token} * shape.size;
        store_column<float, SIZE>(to, acc_k, scale_k, shape.size, half);
        store_column<float, SIZE>(to + plane, acc_v, scale_v, shape.size, half);
    }
}

// The shares of dk and dv added: a thread an element of both.
__global__ void __launch_bounds__(kThreads)
    shares_kernel(const Shape shape, uint32_t splits, const float* __restrict__ parts, S* __restrict__ dk,
                  S* __restrict__ dv) {
    const uint64_t plane = uint64_t{shape.tokens} * shape.size;
    const uint32_t key_heads = shape.heads / shape.group;
    const uint64_t stride = uint64_t{gridDim.x} * kThreads;
    for (uint64_t i = uint64_t{blockIdx.x} * kThreads + threadIdx.x; i < plane * key_heads; i += stride) {
        const uint64_t key_head = i / plane, at = i % plane;
        const uint64_t token = at / shape.size, column = at % shape.size;
        const float* from = parts + key_head * splits * 2 * plane + at;
        float sum_k = from[0], sum_v = from[plane];
        for (uint32_t n = 1; n < splits; n++) {
            sum_k += from[n * 2 * plane];
            sum_v += from[n * 2 * plane + plane];
        }
        dk[token * shape.k.token + key_head * shape.k.head + column] = Elem<S>::narrow(sum_k);
        dv[token * shape.v.token + key_head * shape.v.head + column] = Elem<S>::narrow(sum_v);
    }
}

// ---- launches ------------------------------------------------------------------------------

// `call` with the head size rounded up to 32.
template <typename Call>
int by_size(uint32_t size, Call&& call) {
    if (size <= 32) return call(std::integral_constant<int, 32>());
    if (size <= 64) return call(std::integral_constant<int, 64>());
    if (size <= 96) return call(std::integral_constant<int, 96>());
    return call(std::integral_constant<int, 128>());
}

int forward(const Shape& shape, const void* q, const void* k, const void* v, void* out, float* normalizers) {
    TC_STREAM(s);
    const uint32_t tiles = (shape.tokens + kOwned - 1) / kOwned;
    return by_size(shape.size, [&](auto size) {
        forward_kernel<decltype(size)::value><<<tiles * shape.heads, kThreads, 0, s>>>(
            shape, static_cast<const S*>(q), static_cast<const S*>(k), static_cast<const S*>(v), static_cast<S*>(out),
            normalizers);
        return check_launch("attention");
    });
}

int backward(const Shape& shape, const void* d_out, const void* q, const void* k, const void* v, const void* out,
             const float* normalizers, void* dq, void* dk, void* dv) {
    TC_STREAM(s);
    const char* what = "attention, backward";
    const uint32_t tiles = (shape.tokens + kOwned - 1) / kOwned;
    const uint32_t key_heads = shape.heads / shape.group;
    // Shares of a key head's queries where the key heads alone would leave the
    // compute units idle: the most that divide its heads, up to four blocks
    // for every compute unit.
    uint32_t splits = 1;
    for (uint32_t n = 2; n <= shape.group; n++) {
        if (shape.group % n == 0 && uint64_t{tiles} * key_heads * splits < static_cast<uint64_t>(compute_units()) * 4) {
            splits = n;
        }
    }
    const uint64_t rows = uint64_t{shape.tokens} * shape.heads;
    Scratch dots((rows + 2) * sizeof(float));
    Scratch parts(splits > 1 ? uint64_t{key_heads} * splits * 2 * shape.tokens * shape.size * sizeof(float) : 0);
    if (dots.status != TC_OK) return dots.status;
    if (parts.status != TC_OK) return parts.status;
    float* sums = static_cast<float*>(dots.ptr) + 2;
    uint32_t* largest = static_cast<uint32_t*>(dots.ptr);
    int status = TC_OK;
    if constexpr (kHalf) {
        const uint32_t none = 0;
        status = tc_fill(largest, 2, sizeof(none), &none);
        if (status != TC_OK) return status;
    }
    dots_kernel<<<grid_for(rows, kThreads / 16, 8), kThreads, 0, s>>>(
        shape, static_cast<const S*>(d_out), static_cast<const S*>(out), static_cast<const S*>(v), sums,
        largest);
    status = check_launch(what);
    if (status != TC_OK) return status;
    status = by_size(shape.size, [&](auto size) {
        keys_kernel<decltype(size)::value><<<tiles * key_heads * splits, kThreads, 0, s>>>(
            shape, splits, static_cast<const S*>(d_out), static_cast<const S*>(q), static_cast<const S*>(k),
            static_cast<const S*>(v), normalizers, sums, largest, static_cast<S*>(dk), static_cast<S*>(dv),
            static_cast<float*>(parts.ptr));
        const int launched = check_launch(what);
        if (launched != TC_OK) return launched;
        queries_kernel<decltype(size)::value><<<tiles * shape.heads, kThreads, 0, s>>>(
            shape, static_cast<const S*>(d_out), static_cast<const S*>(q), static_cast<const S*>(k),
            static_cast<const S*>(v), normalizers, sums, largest, static_cast<S*>(dq));
        return check_launch(what);
    });
    if (status != TC_OK || splits == 1) return status;
    const uint64_t elements = uint64_t{shape.tokens} * shape.size * key_heads;
    shares_kernel<<<grid_for(elements, kThreads), kThreads, 0, s>>>(shape, splits, static_cast<float*>(parts.ptr),
                                                                    static_cast<S*>(dk), static_cast<S*>(dv));
    return check_launch(what);
}

}  // namespace

#endif  // TC_ATTENTION_TYPE

}  // namespace attention
}  // namespace tc
