// Attention of new tokens over a cache of keys and values: the kernels, for
// one element type S (cache_attention_*.hip builds them).
//
// With c = scale, over the keys j that query i sees:
//   s_ij = c q_i . k_j,  l_i = log sum_j exp s_ij,  o_i = sum_j exp(s_ij - l_i) v_j.
// A sum over any part J of the keys is held as (m, t, a): the maximum m of its
// scores, t = sum exp(s - m), a = sum exp(s - m) v.  Two parts join into one
// with the larger maximum and both sums scaled down to it, in any grouping, so
// the keys of a sequence may be split over waves and blocks.
//   Bound by memory: a new token's keys and values are read once and used for
// the few query heads that share a key head.  So the keys of all sequences and
// key heads are one line of units, cut evenly over as many blocks as the chip
// holds, whatever the lengths are (`Line`); a block's waves take tiles of their
// unit each and join at the end of a sequence's part, and parts of a sequence
// that lie in several blocks are joined by a second kernel.
//   A prefix that all sequences share is a line of its own, of as many blocks
// of query rows as all tokens' heads fill: its keys are read once for each of
// those and not for each sequence.
//
// A wave holds 16 query rows (token and head of a key head's group; RB times
// as many where there are more) as the columns of 16 x 16 products.  s
// transposed is k . q^T, so that a lane has 4 keys of a row in each product's
// result, and those registers are the operand of o^T = v^T . p^T.  Keys and
// values go through registers to the wave's own tile in LDS, since rows on
// pages have no step between them and 8-bit entries are widened on the way:
// whole numbers up to 127 are exact in every type, and their scales go into
// the scores and the weights.  The next tile's rows are in flight meanwhile.
#pragma once

#include "attention_tiles.hpp"
#include "cache.hpp"

namespace tc {
namespace cache {

constexpr int kAttendThreads = 256;
constexpr int kAttendWaves = kAttendThreads / 64;

// One launch's operands.
struct Attention {
    Pool pool;
    Batch batch;
    uint32_t query_heads, group;
    DivMod group_of;  // divides by group
    float scale;
    const void* query;
    Steps query_steps;
    void* out;
    Steps out_steps;
    float* normalizers;
};

// Where an item (a key head's block of query rows of a sequence) has its
// results: whole in the rows' own place, or in the blocks first to last, the
// first one's in `slot`, the others' in their first slot.
struct Plan {
    uint32_t first, last, slot, whole;
};

// Partial results.  A block has two slots, for parts at its two ends.
struct Parts {
    float* slots;         // [2 blocks][rows][size]
    float2* slot_stats;   // [2 blocks][rows] (maximum, in powers of two; sum)
    float* rows;          // [token][query head][size], of whole items
    float2* row_stats;
    Plan* plans;
};

// The launches of one element type; `blocks` of the first kernel.
struct AttentionLaunches {
    // Items' parts over the sequences' own keys, or with `prefix` over the
    // prefix; `final`: whole items are results.
    int (*attend)(const Attention&, const Parts&, bool quant, bool prefix, bool final, int row_blocks, uint32_t blocks);
    int (*join)(const Attention&, const Parts& own, const Parts& prefix, bool quant, int own_row_blocks,
                int prefix_row_blocks, uint32_t blocks);
};
const AttentionLaunches& attend_f32();
const AttentionLaunches& attend_f16();
const AttentionLaunches& attend_bf16();

// The keys that a query row sees of `count` ones, the last of whose tokens has
// `left` - 1 tokens of its sequence behind it and `length` of them in all
// (with those of a prefix before them).
__host__ __device__ inline uint32_t seen_of(uint64_t length, uint32_t left, uint64_t before, uint64_t count) {
    const uint64_t upto = before + length + 1;  // past the query's own place, plus `left`
    const uint64_t seen = upto > left ? upto - left : 0;
    return static_cast<uint32_t>(seen < count ? seen : count);
}

// Index of a sequence's first item among the plans: no two sequences' overlap,
// without a sum over the ones before.
__device__ __forceinline__ uint64_t first_item(const Attention& a, uint32_t rows, uint32_t sequence, uint32_t token) {
    return (uint64_t{token} * a.group / rows + sequence) * a.pool.heads;
}

#if defined(TC_ATTENTION_TYPE)

namespace {

using attention::E;
using attention::f16x8;
using attention::bf16x8;
using attention::head_word;
using attention::kHalf;
using attention::kWide;
using attention::power2;
using attention::S;
using attention::s16x4;
using attention::u32x2;

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kKeys = kWide ? 16 : 32;  // rows of a wave's tile
constexpr uint32_t kUnit = kKeys * kAttendWaves;
constexpr int kBlocks16 = kKeys / 16;
// Elements of the summed axis that one operand word of all quarters covers.
constexpr int kDeep16 = 4 * E;

// acc += a . b over kDeep16 elements: lane l has row (or column) l % 16 of a
// (or b), and of the summed axis what its quarter l / 16 holds, the same in
// both.  Of the result lane l has rows 4 (l / 16) to 4 (l / 16) + 4 of column
// l % 16.
template <typename T>
__device__ __forceinline__ f32x4 product16(uint4 a, uint4 b, f32x4 acc) {
    if constexpr (sizeof(T) == 4) {
        acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.x), __uint_as_float(b.x), acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.y), __uint_as_float(b.y), acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.z), __uint_as_float(b.z), acc, 0, 0, 0);
        return __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.w), __uint_as_float(b.w), acc, 0, 0, 0);
    } else if constexpr (Elem<T>::dtype == TC_F16) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), acc,
                                                      0, 0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b),
                                                       acc, 0, 0, 0);
    }
}

// `v` joined over the four lanes that have the same column.
template <typename Op>
__device__ __forceinline__ float quarters(float v) {
    const uint32_t bits = __float_as_uint(v);
    const auto rows = __builtin_amdgcn_permlane16_swap(bits, bits, false, false);
    v = Op::join(__uint_as_float(rows[0]), __uint_as_float(rows[1]));
    const uint32_t half = __float_as_uint(v);
    const auto halves = __builtin_amdgcn_permlane32_swap(half, half, false, false);
    return Op::join(__uint_as_float(halves[0]), __uint_as_float(halves[1]));
}

// A tile of kKeys rows, read 16 rows at a time.
template <int SIZE>
struct KeyTile : attention::Tile<SIZE, kKeys> {
    using Base = attention::Tile<SIZE, kKeys>;
    // A lane's places for `by_row` and `by_column`.
    __device__ __forceinline__ static uint32_t row_place(int lane) { return Base::place(lane % 16, lane / 16); }
    __device__ __forceinline__ static uint32_t column_place(int lane) {
        if constexpr (kWide) return Base::place(4 * (lane / 16), lane % 16 / 4) + lane % 4 * 4;
        // Lane j of 16 addresses 4 columns of row j / 4 and receives the 4 rows
        // of column j.
        else return Base::place(4 * (lane / 16) + lane % 16 / 4, lane % 4 / 2) + lane % 2 * 8;
    }
    // Operand word n of row 16 b + l % 16.
    __device__ __forceinline__ uint4 by_row(uint32_t place, int b, int n) const {
        return *reinterpret_cast<const uint4*>(this->from(place, 16 * b, 4 * n));
    }
    // Operand word of column 16 t + l % 16, summed over the rows in the order
    // of products' results.
    __device__ __forceinline__ uint4 by_column(uint32_t place, int t) const {
        if constexpr (kWide) {
            uint32_t v[4];
#pragma unroll
            for (int j = 0; j < 4; j++) v[j] = *reinterpret_cast<const uint32_t*>(this->from(place, j, 4 * t));
            return make_uint4(v[0], v[1], v[2], v[3]);
        } else {
            const u32x2 a = __builtin_bit_cast(u32x2, Base::transposed(this->from(place, 0, 2 * t)));
            const u32x2 b = __builtin_bit_cast(u32x2, Base::transposed(this->from(place, 16, 2 * t)));
            return make_uint4(a.x, a.y, b.x, b.y);
        }
    }
};

// 16 whole numbers of 8 bits as elements of T.
template <typename T>
__device__ __forceinline__ void widened(uint4 bytes, Words<T, 16>& out) {
    const uint32_t four[4] = {bytes.x, bytes.y, bytes.z, bytes.w};
    float v[16];
#pragma unroll
    for (int e = 0; e < 16; e++) v[e] = static_cast<float>(static_cast<int8_t>(four[e / 4] >> (8 * (e % 4))));
    out.put(v);
}

// Which values a sweep takes: the finite ones as they are, or as ones the
// negative or the positive infinities, the NaNs, or all three where their
// weight is 0 (which makes a NaN as well); all others as zeros.
enum { kFinite = 0, kMinus = 1, kPlus = 2, kNaN = 3, kZero = 4 };
__device__ __forceinline__ uint32_t picked(uint32_t bits, int pick) {
    if (pick == kFinite) return attention::finite_bits(bits);
    constexpr uint32_t infinity = kWide ? 0x7f800000u : kHalf ? 0x7c00u : 0x7f80u;
    constexpr uint32_t sign = kWide ? 0x80000000u : 0x8000u, one = kWide ? 0x3f800000u : kHalf ? 0x3c00u : 0x3f80u;
    const auto taken = [&](uint32_t v) {
        const bool is = pick == kMinus  ? v == (infinity | sign)
                        : pick == kPlus ? v == infinity
                        : pick == kNaN  ? (v & ~sign) > infinity
                                        : (v & ~sign) >= infinity;
        return is ? one : 0u;
    };
    if constexpr (kWide) return taken(bits);
    return taken(bits & 0xffffu) | taken(bits >> 16) << 16;
}

// Order within a wave's own LDS is the program's; the compiler is told here.
__device__ __forceinline__ void wave_order() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// A sequence of the line (or the prefix): its tokens here and its keys.
struct Sequence {
    uint32_t first, tokens;
    uint32_t keys;  // that its pages hold
    uint64_t length;
    const uint32_t* pages;
    uint32_t page_count;
};
template <bool PREFIX>
__device__ __forceinline__ Sequence sequence_at(const Attention& a, uint32_t sequence) {
    if constexpr (PREFIX) {
        const uint32_t count = static_cast<uint32_t>((uint64_t{a.batch.prefix} + a.pool.page_size - 1) / a.pool.page_size);
        return {0, a.batch.tokens, a.batch.prefix, a.batch.prefix, a.batch.prefix_pages, count};
    } else {
        const Span span = span_of(a.batch, sequence);
        const uint32_t length = a.batch.lengths[sequence], most = a.batch.most_pages * a.pool.page_size;
        return {span.first,
                span.end > span.first ? span.end - span.first : 0,
                length < most ? length : most,
                length,
                a.batch.pages + uint64_t{sequence} * a.batch.most_pages,
                a.batch.most_pages};
    }
}

// The units of all items one behind another: sequences, of each the key heads,
// of each the blocks of ROWS query rows, of each the units of kUnit keys.
template <int ROWS>
struct Line {
    __device__ __forceinline__ static uint32_t units(const Sequence& s) { return (s.keys + kUnit - 1) / kUnit; }
    __device__ __forceinline__ static uint32_t blocks(const Attention& a, const Sequence& s) {
        return static_cast<uint32_t>((uint64_t{s.tokens} * a.group + ROWS - 1) / ROWS);
    }
    __device__ __forceinline__ static uint64_t count(const Attention& a, const Sequence& s) {
        return uint64_t{units(s)} * blocks(a, s) * a.pool.heads;
    }
};

template <int SIZE, int RB, bool QUANT, bool PREFIX>
__global__ void __launch_bounds__(kAttendThreads) __attribute__((amdgpu_waves_per_eu(2)))
    attend_kernel(const Attention a, const Parts parts, bool final) {
    constexpr int ROWS = 16 * RB;
    using LineOf = Line<ROWS>;
    using TileOf = KeyTile<SIZE>;
    // Weights and values are multiplied in S, but 8-bit entries with bf16
    // weights where S is f16, whose range scales may leave.
    using V = std::conditional_t<QUANT && kHalf, bf16_t, S>;
    constexpr bool kTwoParts = sizeof(V) == 2 && Elem<V>::dtype == TC_BF16;
    constexpr float kPower = sizeof(V) == 2 && Elem<V>::dtype == TC_F16 ? 6.0f : 0.0f;
    constexpr int kOperands = SIZE / kDeep16;
    constexpr int kEntry = QUANT ? 1 : static_cast<int>(sizeof(S));
    constexpr int kRowWords = SIZE * kEntry / 16;
    constexpr int kEach = (kKeys * kRowWords + 63) / 64;
    constexpr int kStride = SIZE + 4;  // of a row where waves join

    __shared__ __attribute__((aligned(1024))) char tiles[kAttendWaves][2 * TileOf::kBytes];
    __shared__ float scales[QUANT ? kAttendWaves : 1][64];
    __shared__ float2 stats[kAttendWaves][ROWS];
    __shared__ uint64_t sums[kAttendWaves], found[2];
    static_assert(sizeof(tiles) >= kAttendWaves * 16 * kStride * sizeof(float), "waves join in the tiles' place");

    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, quarter = lane / 16;

    // ---- this block's units ----------------------------------------------------
    const uint32_t sequences = PREFIX ? 1 : a.batch.sequences;
    uint64_t total_units = 0;
    if constexpr (PREFIX) {
        total_units = LineOf::count(a, sequence_at<true>(a, 0));
    } else {
        uint64_t mine = 0;
        for (uint32_t n = threadIdx.x; n < sequences; n += kAttendThreads) mine += LineOf::count(a, sequence_at<false>(a, n));
        for (int offset = 32; offset > 0; offset >>= 1) mine += __shfl_xor(static_cast<unsigned long long>(mine), offset);
        if (lane == 0) sums[wave] = mine;
        __syncthreads();
        for (int w = 0; w < kAttendWaves; w++) total_units += sums[w];
        __syncthreads();
    }
    // No block has nothing, so that every block between two parts of an item
    // has a part of it.
    const uint64_t blocks = total_units < gridDim.x ? total_units : gridDim.x;
    if (blockIdx.x >= blocks) return;
    const uint64_t begin = blockIdx.x * total_units / blocks, end = (blockIdx.x + 1) * total_units / blocks;

    uint32_t sequence = 0;
    uint64_t before = 0;  // units of the sequences before
    if constexpr (!PREFIX) {
        for (uint32_t from = 0; from < sequences; from += kAttendThreads) {
            const uint32_t n = from + threadIdx.x;
            const uint64_t count = n < sequences ? LineOf::count(a, sequence_at<false>(a, n)) : 0;
            uint64_t upto = count;
            for (int offset = 1; offset < 64; offset *= 2) {
                const uint64_t other = __shfl_up(static_cast<unsigned long long>(upto), offset);
                if (lane >= offset) upto += other;
            }
            if (lane == 63) sums[wave] = upto;
            __syncthreads();
            uint64_t all = 0;
            for (int w = 0; w < kAttendWaves; w++) {
                if (w < wave) upto += sums[w];
                all += sums[w];
            }
            const uint64_t start = before + upto - count;
            if (begin >= start && begin - start < count) found[0] = n, found[1] = start;
            __syncthreads();
            if (begin - before < all) break;  // the same for the whole block
            before += all;
        }
        sequence = static_cast<uint32_t>(found[0]);
        before = found[1];
        sequence = __builtin_amdgcn_readfirstlane(sequence);
    }

    const TileOf key_tile{tiles[wave]};
    const TileOf value_tile{tiles[wave] + TileOf::kBytes};
    const uint32_t row_place = TileOf::row_place(lane), column_place = TileOf::column_place(lane);
    const float c = a.scale * attention::kLog2e;

    for (uint64_t unit = begin; unit < end;) {
        const Sequence s = sequence_at<PREFIX>(a, sequence);
        const uint32_t units = LineOf::units(s), row_blocks = LineOf::blocks(a, s);
        const uint64_t count = uint64_t{units} * row_blocks * a.pool.heads;
        if (unit - before >= count) {
            before += count;
            sequence++;
            continue;
        }
        const uint32_t item = static_cast<uint32_t>((unit - before) / units);
        const uint32_t unit_0 = static_cast<uint32_t>((unit - before) % units);
        const uint32_t unit_1 = end - unit < units - unit_0 ? unit_0 + static_cast<uint32_t>(end - unit) : units;
        const uint32_t key_head = item / row_blocks, row_block = item % row_blocks;
        const bool whole = unit_0 == 0 && unit_1 == units;
        // (An item's first part is the block's first if both begin together.)
        const uint32_t slot = 2 * blockIdx.x + (unit > begin);
        if (unit_0 == 0 && threadIdx.x == 0) {
            const uint64_t last_unit = unit + units - 1;
            const uint64_t last = ((last_unit + 1) * blocks - 1) / total_units;
            const uint64_t at = (PREFIX ? 0 : first_item(a, ROWS, sequence, s.first)) + item;
            parts.plans[at] = {blockIdx.x, static_cast<uint32_t>(last), slot, whole};
        }

        // ---- the item's query rows -------------------------------------------------
        const uint32_t rows = s.tokens * a.group - row_block * ROWS < ROWS ? s.tokens * a.group - row_block * ROWS : ROWS;
        uint4 queries[RB][kOperands];
        uint32_t seen[RB];
        uint32_t least = s.keys, most_seen = 0;
#pragma unroll
        for (int r = 0; r < RB; r++) {
            const uint32_t row = r * 16 + lane % 16, number = row_block * ROWS + row;
            const bool real = row < rows;
            const uint32_t place = a.group_of.div(real ? number : 0);
            const uint32_t token = s.first + place;
            const uint32_t head = key_head * a.group + (real ? number : 0) - place * a.group;
            if constexpr (PREFIX) {
                Span span;
                const uint32_t own = sequence_of(a.batch, token, &span);
                seen[r] = own == kNowhere ? s.keys : seen_of(a.batch.lengths[own], span.end - token, s.keys, s.keys);
            } else {
                seen[r] = seen_of(s.length, s.tokens - place, 0, s.keys);
            }
            if (!real) seen[r] = s.keys;
            if (real) {
                least = seen[r] < least ? seen[r] : least;
                most_seen = seen[r] > most_seen ? seen[r] : most_seen;
            }
            const S* from = static_cast<const S*>(a.query) + token * a.query_steps.token + head * a.query_steps.head;
#pragma unroll
            for (int n = 0; n < kOperands; n++) {
                queries[r][n] = real ? head_word(from, 4 * n + quarter, a.pool.size) : make_uint4(0, 0, 0, 0);
            }
        }
        for (int offset = 8; offset > 0; offset >>= 1) {
            const uint32_t other = __shfl_xor(least, offset), more = __shfl_xor(most_seen, offset);
            least = other < least ? other : least;
            most_seen = more > most_seen ? more : most_seen;
        }
        least = __builtin_amdgcn_readfirstlane(least);
        most_seen = __builtin_amdgcn_readfirstlane(most_seen);

        // ---- a sweep over the part's tiles -----------------------------------------
        f32x4 acc[RB][SIZE / 16];
        float most[RB], total[RB];

        const uint32_t key_end = uint64_t{unit_1} * kUnit < most_seen ? unit_1 * kUnit : most_seen;
        uint32_t tile = 0;
        uint4 key_words[kEach], value_words[kEach];
        float entry_scale = 0.0f;
        // The page of key l % 32 of the tile at `at`, and its row there.
        const auto page_at = [&](uint32_t at) {
            const uint32_t key = at + lane % 32;
            const uint32_t n = a.pool.pages_of.div(key);
            return lane % 32 < kKeys && key < key_end && n < s.page_count ? s.pages[n] : kNowhere;
        };
        const auto row_at = [&](uint32_t at, uint32_t page) {
            const uint32_t key = at + lane % 32;
            const uint32_t slot_in = key - a.pool.pages_of.div(key) * a.pool.page_size;
            return page < a.pool.page_count ? (page * a.pool.heads + key_head) * a.pool.page_size + slot_in : kNowhere;
        };
        const auto fetch = [&](uint32_t row) {
            const uint32_t row_bytes = a.pool.row * kEntry;
#pragma unroll
            for (int k = 0; k < kEach; k++) {
                const int i = k * 64 + lane;
                const uint32_t from = __shfl(row, i / kRowWords < kKeys ? i / kRowWords : 0);
                const uint32_t byte = i % kRowWords * 16;
                key_words[k] = value_words[k] = make_uint4(0, 0, 0, 0);
                if (i < kKeys * kRowWords && from != kNowhere && byte < row_bytes) {
                    const uint64_t place = uint64_t{from} * row_bytes + byte;
                    key_words[k] = load_word<false>(static_cast<const char*>(a.pool.keys) + place);
                    value_words[k] = load_word<false>(static_cast<const char*>(a.pool.values) + place);
                }
            }
            if constexpr (QUANT) {
                entry_scale = row == kNowhere ? 0.0f : (lane < 32 ? a.pool.key_scales : a.pool.value_scales)[row];
            }
        };
        const auto land = [&]() {
#pragma unroll
            for (int k = 0; k < kEach; k++) {
                const int i = k * 64 + lane;
                if (kKeys * kRowWords % 64 != 0 && i >= kKeys * kRowWords) continue;
                const int row = i / kRowWords, word = i % kRowWords;
                if constexpr (QUANT) {
                    Words<S, 16> keys;
                    Words<V, 16> values;
                    widened(key_words[k], keys);
                    widened(value_words[k], values);
#pragma unroll
                    for (int w = 0; w < 16 / E; w++) {
                        *reinterpret_cast<uint4*>(key_tile.word(row, word * (16 / E) + w)) = keys.w[w];
                        *reinterpret_cast<uint4*>(value_tile.word(row, word * (16 / E) + w)) = values.w[w];
                    }
                } else {
                    *reinterpret_cast<uint4*>(key_tile.word(row, word)) = key_words[k];
                    *reinterpret_cast<uint4*>(value_tile.word(row, word)) = value_words[k];
                }
            }
            if constexpr (QUANT) scales[wave][lane] = entry_scale;
        };
        uint32_t next_page = kNowhere;
        [[maybe_unused]] int pick = kFinite;
        const auto turn = [&](auto is_masked, auto is_slow) {
            constexpr bool MASKED = decltype(is_masked)::value, SLOW = decltype(is_slow)::value;
            wave_order();
            land();
            wave_order();
            const uint32_t next = tile + kUnit;
            if (next < key_end) {
                fetch(row_at(next, next_page));
                next_page = page_at(next + kUnit);
            }
            // Scores, and their maximum over the tile.
            f32x4 scores[RB][kBlocks16];
#pragma unroll
            for (int b = 0; b < kBlocks16; b++) {
#pragma unroll
                for (int r = 0; r < RB; r++) scores[r][b] = f32x4{};
#pragma unroll
                for (int n = 0; n < kOperands; n++) {
                    const uint4 keys = key_tile.by_row(row_place, b, n);
#pragma unroll
                    for (int r = 0; r < RB; r++) scores[r][b] = product16<S>(keys, queries[r][n], scores[r][b]);
                }
                if constexpr (QUANT) {
                    const f32x4 scale = *reinterpret_cast<const f32x4*>(&scales[wave][16 * b + 4 * quarter]);
#pragma unroll
                    for (int r = 0; r < RB; r++) {
#pragma unroll
                        for (int i = 0; i < 4; i++) scores[r][b][i] *= scale[i];
                    }
                }
            }
#pragma unroll
            for (int r = 0; r < RB; r++) {
                if constexpr (MASKED) {
#pragma unroll
                    for (int b = 0; b < kBlocks16; b++) {
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            if (tile + 16 * b + 4 * quarter + i >= seen[r]) scores[r][b][i] = -INFINITY;
                        }
                    }
                }
                float high = -INFINITY;
#pragma unroll
                for (int b = 0; b < kBlocks16; b++) {
#pragma unroll
                    for (int i = 0; i < 4; i++) high = fmaxf(high, scores[r][b][i]);
                }
                high = quarters<Largest>(high) * c;
                // The maximum only moves when it grows past 2^8: the weights
                // stay that small, and the sums are rarely rescaled.
                const bool grows = high > most[r] + 8.0f;
                if (__ballot(grows) != 0) {
                    const float factor = grows ? power2(most[r] - high) : 1.0f;
                    if (grows) most[r] = high;
                    total[r] *= factor;
#pragma unroll
                    for (int t = 0; t < SIZE / 16; t++) acc[r][t] *= factor;
                }
                const float origin = (most[r] == -INFINITY ? 0.0f : most[r]) - kPower;
#pragma unroll
                for (int b = 0; b < kBlocks16; b++) {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        scores[r][b][i] = power2(fmaf(scores[r][b][i], c, -origin));
                        total[r] += scores[r][b][i];
                    }
                    if constexpr (QUANT) {
                        const f32x4 scale = *reinterpret_cast<const f32x4*>(&scales[wave][32 + 16 * b + 4 * quarter]);
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const bool out_of = MASKED && tile + 16 * b + 4 * quarter + i >= seen[r];
                            scores[r][b][i] = out_of ? 0.0f : scores[r][b][i] * scale[i];
                        }
                    }
                }
            }
            // The weights as operands: their rounding to V, and where that
            // keeps 8 bits, the rounding of what it leaves.
            uint4 high_part[RB], low_part[RB];
#pragma unroll
            for (int r = 0; r < RB; r++) {
                float v[E];
#pragma unroll
                for (int e = 0; e < E; e++) {
                    v[e] = scores[r][e / 4][e % 4];
                    if (SLOW && pick != kFinite) {
                        const bool sees = tile + 16 * (e / 4) + 4 * quarter + e % 4 < seen[r];
                        v[e] = (pick == kNaN ? sees : pick == kZero ? sees && v[e] == 0.0f : v[e] != 0.0f) ? 1.0f : 0.0f;
                    }
                }
                Words<V, E> high, low;
                high.put(v);
                high_part[r] = high.w[0];
                if constexpr (kTwoParts) {
#pragma unroll
                    for (int e = 0; e < E; e++) v[e] -= high.at(e);
                    low.put(v);
                    low_part[r] = low.w[0];
                }
            }
#pragma unroll
            for (int t = 0; t < SIZE / 16; t++) {
                uint4 values = value_tile.by_column(column_place, t);
                if constexpr (SLOW) {
                    values = make_uint4(picked(values.x, pick), picked(values.y, pick), picked(values.z, pick),
                                        picked(values.w, pick));
                }
#pragma unroll
                for (int r = 0; r < RB; r++) {
                    acc[r][t] = product16<V>(values, high_part[r], acc[r][t]);
                    if constexpr (kTwoParts) acc[r][t] = product16<V>(values, low_part[r], acc[r][t]);
                }
            }
            tile = next;
        };
        const auto sweep = [&](auto is_slow) {
#pragma unroll
            for (int r = 0; r < RB; r++) {
                most[r] = -INFINITY, total[r] = 0.0f;
#pragma unroll
                for (int t = 0; t < SIZE / 16; t++) acc[r][t] = f32x4{};
            }
            tile = unit_0 * kUnit + wave * kKeys;
            if (tile >= key_end) return;
            fetch(row_at(tile, page_at(tile)));
            next_page = page_at(tile + kUnit);
            // (Rows past `key_end` are masked too.)
            const uint32_t plain_end = least < key_end ? least : key_end;
            if constexpr (!decltype(is_slow)::value) {
                while (tile < plain_end && plain_end - tile >= kKeys) turn(std::false_type(), is_slow);
            }
            while (tile < key_end) turn(std::true_type(), is_slow);
        };
        sweep(std::false_type());
        if constexpr (!QUANT) {
            // A value that is an infinity or a NaN has spoiled every row, its
            // weight being 0 in those that do not see it, or 0 in the second of
            // two parts.  So once more for each kind of them, counting those
            // that are seen, and at last without them.
            bool spoiled = false;
#pragma unroll
            for (int r = 0; r < RB; r++) {
#pragma unroll
                for (int t = 0; t < SIZE / 16; t++) {
#pragma unroll
                    for (int i = 0; i < 4; i++) spoiled |= !(fabsf(acc[r][t][i]) < INFINITY);
                }
            }
            if (__builtin_expect(__ballot(spoiled) != 0, false)) {
                uint32_t up[RB] = {}, down[RB] = {};  // a bit an element, both for a NaN
#pragma unroll 1
                for (pick = kZero; pick >= kFinite; pick--) {
                    sweep(std::true_type());
                    if (pick == kFinite) break;
#pragma unroll
                    for (int r = 0; r < RB; r++) {
                        uint32_t bits = 0;
#pragma unroll
                        for (int t = 0; t < SIZE / 16; t++) {
#pragma unroll
                            for (int i = 0; i < 4; i++) bits |= acc[r][t][i] > 0.0f ? 1u << (4 * t + i) : 0u;
                        }
                        if (pick != kMinus) up[r] |= bits;
                        if (pick != kPlus) down[r] |= bits;
                    }
                }
#pragma unroll
                for (int r = 0; r < RB; r++) {
#pragma unroll
                    for (int t = 0; t < SIZE / 16; t++) {
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            if (up[r] >> (4 * t + i) & 1) acc[r][t][i] += INFINITY;
                            if (down[r] >> (4 * t + i) & 1) acc[r][t][i] -= INFINITY;
                        }
                    }
                }
            }
        }

        // ---- the waves' sums joined, and stored --------------------------------------
#pragma unroll
        for (int r = 0; r < RB; r++) {
            total[r] = quarters<Added>(total[r]);
            if (lane < 16) stats[wave][r * 16 + lane] = make_float2(most[r], total[r]);
        }
        __syncthreads();
        float* const shared = reinterpret_cast<float*>(&tiles[0][0]);
#pragma unroll
        for (int r = 0; r < RB; r++) {
            const auto over_waves = [&](uint32_t row, float* top, float* all) {
                *top = -INFINITY, *all = 0.0f;
                for (int w = 0; w < kAttendWaves; w++) *top = fmaxf(*top, stats[w][row].x);
                const float origin = *top == -INFINITY ? 0.0f : *top;
                for (int w = 0; w < kAttendWaves; w++) *all += power2(stats[w][row].x - origin) * stats[w][row].y;
            };
            float top, all;
            over_waves(r * 16 + lane % 16, &top, &all);
            const float factor = power2(most[r] - (top == -INFINITY ? 0.0f : top));
#pragma unroll
            for (int t = 0; t < SIZE / 16; t++) {
                *reinterpret_cast<f32x4*>(shared + (wave * 16 + lane % 16) * kStride + 16 * t + 4 * quarter) =
                    acc[r][t] * factor;
            }
            __syncthreads();
            for (uint32_t i = threadIdx.x; i < 16 * SIZE / 4; i += kAttendThreads) {
                const uint32_t row = i / (SIZE / 4), column = i % (SIZE / 4) * 4;
                if (r * 16 + row >= rows) continue;
                f32x4 v = *reinterpret_cast<const f32x4*>(shared + row * kStride + column);
                for (int w = 1; w < kAttendWaves; w++) {
                    v += *reinterpret_cast<const f32x4*>(shared + (w * 16 + row) * kStride + column);
                }
                over_waves(r * 16 + row, &top, &all);
                const uint32_t number = row_block * ROWS + r * 16 + row;
                const uint32_t place = a.group_of.div(number);
                const uint32_t token = s.first + place, head = key_head * a.group + number - place * a.group;
                if (whole && final) {
                    // (A sum of 0 over keys that are seen is of scores of
                    // -infinity alone: 0 / 0.)
                    const bool sees = seen_of(s.length, s.tokens - place, 0, s.keys) > 0;
                    S* const to = static_cast<S*>(a.out) + token * a.out_steps.token + head * a.out_steps.head;
                    const float scale = sees ? 1.0f / all : 0.0f;
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        if (column + j < a.pool.size) to[column + j] = Elem<S>::narrow(sees ? v[j] * scale : 0.0f);
                    }
                    if (column == 0 && a.normalizers != nullptr) {
                        a.normalizers[uint64_t{head} * a.batch.tokens + token] =
                            all == 0.0f ? -INFINITY : (top + log2f(all) - kPower) * attention::kLn2;
                    }
                } else {
                    const uint64_t at = whole ? uint64_t{token} * a.query_heads + head
                                              : uint64_t{slot} * ROWS + r * 16 + row;
                    float* const to = (whole ? parts.rows : parts.slots) + at * SIZE + column;
                    *reinterpret_cast<f32x4*>(to) = v;
                    if (column == 0) (whole ? parts.row_stats : parts.slot_stats)[at] = make_float2(top, all);
                }
            }
            __syncthreads();
        }
        unit += unit_1 - unit_0;
    }
}

// Each row's parts joined, a block a row: the row's own sequence's and the
// prefix's, in the order of their blocks, 8 of them at a time.
template <int SIZE>
__global__ void __launch_bounds__(kAttendThreads)
    join_kernel(const Attention a, const Parts own, const Parts prefix, uint32_t own_rows, uint32_t prefix_rows,
                uint32_t blocks, bool half_power) {
    constexpr int kGroups = kAttendThreads / 32;
    __shared__ f32x4 sums[kGroups][32];
    __shared__ float totals[kGroups];
    for (uint64_t row = blockIdx.x; row < uint64_t{a.batch.tokens} * a.query_heads; row += gridDim.x) {
        const uint32_t token = static_cast<uint32_t>(row / a.query_heads);
        const uint32_t head = static_cast<uint32_t>(row % a.query_heads);
        const uint32_t key_head = head / a.group, within = head % a.group;
        Span span{0, 0};
        const uint32_t sequence = wave_sequence_of(a.batch, token, &span);

        // A line's parts of the row: n of them, the first at `first` of its
        // slots, or the one of a whole item.
        struct Found {
            uint32_t n = 0, first_block = 0, first_slot = 0, line = 0;
            uint64_t within = 0;
            bool whole = false;
        } mine, shared;
        bool sees = false;
        if (sequence != kNowhere) {
            const Sequence s = sequence_at<false>(a, sequence);
            const uint32_t place = token - s.first, left = s.tokens - place;
            const auto find = [&](const Parts& parts, uint32_t rows, uint64_t first, uint64_t number,
                                  uint32_t row_blocks) {
                Found f;
                const uint32_t block = static_cast<uint32_t>(number / rows);
                const Plan plan = parts.plans[first + uint64_t{key_head} * row_blocks + block];
                f.whole = plan.whole != 0;
                f.n = f.whole ? 1 : plan.first <= plan.last && plan.last < blocks ? plan.last - plan.first + 1 : 0;
                f.first_block = plan.first, f.first_slot = plan.slot;
                f.line = rows;
                f.within = number % rows;
                return f;
            };
            if (s.keys > 0) {
                const uint32_t row_blocks = static_cast<uint32_t>((uint64_t{s.tokens} * a.group + own_rows - 1) / own_rows);
                mine = find(own, own_rows, first_item(a, own_rows, sequence, s.first),
                            uint64_t{place} * a.group + within, row_blocks);
                sees = seen_of(s.length, left, 0, s.keys) > 0;
            }
            if (a.batch.prefix > 0) {
                const uint32_t row_blocks =
                    static_cast<uint32_t>((uint64_t{a.batch.tokens} * a.group + prefix_rows - 1) / prefix_rows);
                shared = find(prefix, prefix_rows, 0, uint64_t{token} * a.group + within, row_blocks);
                sees = sees || seen_of(s.length, left, a.batch.prefix, a.batch.prefix) > 0;
            }
        }
        const uint32_t count = mine.n + shared.n;
        // A whole item without a prefix is a result already.
        if (count == 1 && mine.n == 1 && mine.whole && a.batch.prefix == 0) continue;

        const auto place_of = [&](uint32_t n, const float** values, const float2** stats) {
            const bool is_mine = n < mine.n;
            const Found& f = is_mine ? mine : shared;
            const Parts& parts = is_mine ? own : prefix;
            n = is_mine ? n : n - mine.n;
            const uint64_t at = f.whole ? row : (n == 0 ? f.first_slot : uint64_t{2} * (f.first_block + n)) * f.line + f.within;
            *values = (f.whole ? parts.rows : parts.slots) + at * SIZE;
            *stats = (f.whole ? parts.row_stats : parts.slot_stats) + at;
        };
        const float* values;
        const float2* stats;
        float top = -INFINITY;
        for (uint32_t n = threadIdx.x % 64; n < count; n += 64) {
            place_of(n, &values, &stats);
            top = fmaxf(top, stats->x);
        }
        top = wave64<Largest>(top);
        const float origin = top == -INFINITY ? 0.0f : top;
        const uint32_t group = threadIdx.x / 32, column = threadIdx.x % 32 * 4;
        f32x4 sum = {};
        float total = 0.0f;
        for (uint32_t n = group; n < count; n += kGroups) {
            place_of(n, &values, &stats);
            const float factor = power2(stats->x - origin);
            total += factor * stats->y;
            if (column < SIZE) sum += factor * *reinterpret_cast<const f32x4*>(values + column);
        }
        sums[group][threadIdx.x % 32] = sum;
        if (threadIdx.x % 32 == 0) totals[group] = total;
        __syncthreads();
        if (threadIdx.x < 32) {
            for (int g = 1; g < kGroups; g++) {
                sum += sums[g][threadIdx.x];
                total += totals[g];
            }
            S* const to = static_cast<S*>(a.out) + token * a.out_steps.token + head * a.out_steps.head;
            const float scale = sees ? 1.0f / total : 0.0f;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if (column + j < a.pool.size) to[column + j] = Elem<S>::narrow(sees ? sum[j] * scale : 0.0f);
            }
            if (threadIdx.x == 0 && a.normalizers != nullptr) {
                a.normalizers[uint64_t{head} * a.batch.tokens + token] =
                    total == 0.0f ? -INFINITY : (top + log2f(total) - (half_power ? 6.0f : 0.0f)) * attention::kLn2;
            }
        }
        __syncthreads();
    }
}

#define TC_CACHE_SIZE(size, ...)                        \
    if (size <= 32) {                                   \
        constexpr int SIZE = 32; __VA_ARGS__;           \
    } else if (size <= 64) {                            \
        constexpr int SIZE = 64; __VA_ARGS__;           \
    } else if (size <= 96) {                            \
        constexpr int SIZE = 96; __VA_ARGS__;           \
    } else {                                            \
        constexpr int SIZE = 128; __VA_ARGS__;          \
    }

template <int SIZE, int RB, bool QUANT>
void attend_rows(const Attention& a, const Parts& parts, bool prefix, bool final, uint32_t blocks, hipStream_t s) {
    if (prefix) {
        attend_kernel<SIZE, RB, QUANT, true><<<blocks, kAttendThreads, 0, s>>>(a, parts, false);
    } else {
        attend_kernel<SIZE, RB, QUANT, false><<<blocks, kAttendThreads, 0, s>>>(a, parts, final);
    }
}

int attend(const Attention& a, const Parts& parts, bool quant, bool prefix, bool final, int row_blocks,
           uint32_t blocks) {
    TC_STREAM(s);
    TC_CACHE_SIZE(a.pool.size, {
        if (quant) {
            if (row_blocks == 1) attend_rows<SIZE, 1, true>(a, parts, prefix, final, blocks, s);
            else attend_rows<SIZE, 2, true>(a, parts, prefix, final, blocks, s);
        } else {
            if (row_blocks == 1) attend_rows<SIZE, 1, false>(a, parts, prefix, final, blocks, s);
            else attend_rows<SIZE, 2, false>(a, parts, prefix, final, blocks, s);
        }
    })
    return check_launch("cache attention");
}

int join(const Attention& a, const Parts& own, const Parts& prefix, bool quant, int own_row_blocks,
         int prefix_row_blocks, uint32_t blocks) {
    TC_STREAM(s);
    const uint64_t rows = uint64_t{a.batch.tokens} * a.query_heads;
    const uint32_t grid = rows < (1u << 20) ? static_cast<uint32_t>(rows) : 1u << 20;
    TC_CACHE_SIZE(a.pool.size, {
        join_kernel<SIZE><<<grid, kAttendThreads, 0, s>>>(a, own, prefix, 16 * own_row_blocks, 16 * prefix_row_blocks,
                                                          blocks, kHalf && !quant);
    })
    return check_launch("cache attention");
}

}  // namespace

#endif  // TC_ATTENTION_TYPE

}  // namespace cache
}  // namespace tc
