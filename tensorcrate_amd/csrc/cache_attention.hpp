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
// the few query heads that share a key head.  So the tiles of all sequences and
// key heads are one line, cut evenly over as many waves as the chip holds,
// whatever the lengths are (`Line`); parts of a sequence that lie in several
// waves are joined by a second kernel.  (Every block of a sequence's query rows
// counts as all of its keys: of a prompt's first rows, which see few, most tiles
// are passed over, so that for prompts the cut is not even.)
//   A prefix that all sequences share is a line of its own, of as many blocks
// of query rows as all tokens' heads fill: its keys are read once for each of
// those and not for each sequence.
//
// A wave holds 16 query rows (token and head of a key head's group) as the
// columns of 16 x 16 products.  s transposed is k . q^T, so that a lane has 4
// keys of a row in each product's result, and those registers are the operand of
// o^T = v^T . p^T.  Keys and values go through registers to a tile in LDS, since
// rows on pages have no step between them and 8-bit entries are widened on the
// way; the next tiles' rows are in flight meanwhile.  Where at most 16 rows share
// keys, each of a block's four waves has its own tiles, every fourth one, and the
// waves join at a part's end; where more do, the waves have 16 rows each and
// share every tile (SHARED), so that keys are read and widened once for 64 rows.
//
// For the products with the values the weights are taken in two parts where
// those have 16 bits, 16 bits of each and the rounding of what that leaves: bf16
// keeps 16 bits so, f16 21; f32 keeps all.  (In f16 one part alone, 2^-11 of each
// weight, took 155 instead of 170 us for 512 new of 8704 tokens, and as long
// where memory bounds; results in f16 were off by up to 1.4 times as much.)
// 8-bit entries, whole numbers to 127 that every type holds, are widened to the
// queries' type for the scores, which take the keys' scales afterwards.  The
// values' scales go into the weights, so that under 16-bit queries weights and
// values are multiplied as bf16 (`Weighed`).
//
// Measured: 64 sequences to 8192 tokens, 32 heads on 8 of 128, bf16: 220 us (5.7
// TB/s in the first kernel); 4 to 100000 in 8 bits 113 us; 24 to 3000 with 5 new
// tokens of 12 heads of 80, f16, 47; one of 1000 13, of which 4 are the join; 80
// to 500 behind 8000 shared tokens in 8 bits 77 (own keys 31, prefix 40, join);
// 512 new of 8704 tokens 163 us (435 TFLOP/s), a prompt of 2048 155.
// With waves that each stored parts of their own, instead of joining in LDS, the
// last case's own keys took 10 us less, and the longer ones more.
#pragma once

#include "attention_tiles.hpp"
#include "cache.hpp"

namespace tc {
namespace cache {

constexpr int kAttendThreads = 256;
constexpr int kAttendWaves = kAttendThreads / 64;
// The first kernel's two forms: blocks of 16 query rows, whose waves take a tile
// each and join at the end of a part, or of 64 rows, 16 a wave, that share each
// tile (SHARED).
constexpr uint32_t rows_of_form(bool shared) { return shared ? 64 : 16; }
// Blocks of a compute unit at a time.  (Registers just allow them: over plain
// entries of 65 elements and more a lane keeps 2 to 16 values in memory.)
constexpr uint32_t blocks_of_form(bool shared) { return shared ? 3 : 2; }

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

// Where a query row's parts over a line are: in the row's own place if it is
// kWhole, or with the blocks first to last (none if last is less), the first
// one's at `place` of the slots, the others' in their first slot.  kSees: the
// row sees keys of the line; kOutside: it is of no sequence.
enum { kWhole = 1, kSees = 2, kOutside = 4 };
struct Found {
    uint32_t first, last, place, marks;
};

// Partial results.  A block has two slots, for parts at its two ends.
struct Parts {
    float* slots;        // [2 blocks][rows][size]
    float2* slot_stats;  // [2 blocks][rows] (maximum, in powers of two; sum)
    float* rows;         // [token][query head][size], of whole items
    float2* row_stats;
    Found* found;   // [token][query head]
    uint32_t* cut;  // whether any token comes before its sequence's first
};

// The launches of one element type.
struct AttentionLaunches {
    // Items' parts over the sequences' own keys, or with `prefix` over the
    // prefix; `final`: whole items are results.
    int (*attend)(const Attention&, const Parts&, bool quant, bool prefix, bool final, bool shared);
    int (*join)(const Attention&, const Parts& own, const Parts& prefix, bool quant, bool own_shared,
                bool prefix_shared);
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

constexpr int kKeys = kWide ? 16 : 32;  // rows of a tile: what a product of weights with values sums over
constexpr int kBlocks16 = kKeys / 16;

// A value that is the same in the whole wave, kept as one.
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ uint64_t uniform(uint64_t v) {
    return uniform(static_cast<uint32_t>(v)) | uint64_t{uniform(static_cast<uint32_t>(v >> 32))} << 32;
}
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
    // Operand word of column 16 t + l % 16, summed over the rows in the order of
    // products' results.
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
    if constexpr (Elem<T>::dtype == TC_F16) {
        // Behind the upper byte of 1024 in f16, whose step is 1: 1024 + 128 + q.
        typedef _Float16 pair __attribute__((ext_vector_type(2)));
        uint32_t* const to = reinterpret_cast<uint32_t*>(out.w);
#pragma unroll
        for (int n = 0; n < 4; n++) {
            const uint32_t shifted = four[n] ^ 0x80808080u;
            const pair low = __builtin_bit_cast(pair, __builtin_amdgcn_perm(0x64646464u, shifted, 0x04010400u));
            const pair high = __builtin_bit_cast(pair, __builtin_amdgcn_perm(0x64646464u, shifted, 0x04030402u));
            const pair origin = {static_cast<_Float16>(1152.0f), static_cast<_Float16>(1152.0f)};
            to[2 * n] = __builtin_bit_cast(uint32_t, low - origin);
            to[2 * n + 1] = __builtin_bit_cast(uint32_t, high - origin);
        }
    } else {
        float v[16];
#pragma unroll
        for (int e = 0; e < 16; e++) v[e] = static_cast<float>(static_cast<int8_t>(four[e / 4] >> (8 * (e % 4))));
        out.put(v);
    }
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

// body(0), body(1), ... body(N - 1), each a constant.
template <int N, typename F>
__device__ __forceinline__ void each(F&& body) {
    if constexpr (N > 0) {
        each<N - 1>(body);
        body(std::integral_constant<int, N - 1>());
    }
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

// The tiles of all items one behind another: sequences, of each the key heads,
// of each the blocks of ROWS query rows, of each the tiles of kKeys keys.
template <int ROWS>
struct Line {
    __device__ __forceinline__ static uint32_t tiles(const Sequence& s) { return (s.keys + kKeys - 1) / kKeys; }
    __device__ __forceinline__ static uint32_t blocks(const Attention& a, const Sequence& s) {
        return static_cast<uint32_t>((uint64_t{s.tokens} * a.group + ROWS - 1) / ROWS);
    }
    __device__ __forceinline__ static uint64_t count(const Attention& a, const Sequence& s) {
        return uint64_t{tiles(s)} * blocks(a, s) * a.pool.heads;
    }
};

// Four elements from `first` on to a row of `size`.
__device__ __forceinline__ void store_four(S* row, uint32_t first, uint32_t size, f32x4 v) {
    typedef uint32_t piece __attribute__((ext_vector_type(sizeof(S)), aligned(sizeof(S))));
    S out[4];
#pragma unroll
    for (int j = 0; j < 4; j++) out[j] = Elem<S>::narrow(v[j]);
    if (first + 4 <= size) {
        piece bits;
        __builtin_memcpy(&bits, out, sizeof(bits));
        *reinterpret_cast<piece*>(row + first) = bits;
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (first + j < size) row[first + j] = out[j];
        }
    }
}

// The type that weights and values are multiplied in.  With 8-bit entries the
// values' scales go into the weights, which then have a range that f16 lacks:
// a value whose scale is 2^30 times the others' and its weight next to nothing
// took the others' weights below f16's smallest number.  bf16 has f32's range,
// and 8-bit numbers are exact in it.
template <bool QUANT>
using Weighed = std::conditional_t<QUANT && kHalf, bf16_t, S>;

// Power of two that weights are rounded times in f16, whose least normal is
// 2^-14: the largest, which may reach 2^8, stay below 2^15.
constexpr float power_of(bool quant) { return kHalf && !quant ? 6.0f : 0.0f; }

template <int SIZE, bool SHARED, bool QUANT, bool PREFIX>
__global__ void __launch_bounds__(kAttendThreads) __attribute__((amdgpu_waves_per_eu(blocks_of_form(SHARED))))
    attend_kernel(const Attention a, const Parts parts, bool final) {
    constexpr int ROWS = rows_of_form(SHARED);
    constexpr int kMovers = SHARED ? kAttendThreads : 64;  // threads that move a tile
    using LineOf = Line<ROWS>;
    using TileOf = KeyTile<SIZE>;
    // The type that weights and values are multiplied in.
    using V = Weighed<QUANT>;
    constexpr bool kTwoParts = sizeof(V) == 2;
    constexpr float kPower = power_of(QUANT);
    constexpr int kOperands = SIZE / kDeep16;
    constexpr int kEntry = QUANT ? 1 : static_cast<int>(sizeof(S));
    constexpr int kRowWords = SIZE * kEntry / 16;
    constexpr int kEach = (kKeys * kRowWords + kMovers - 1) / kMovers;
    // Words of a tile's row.  Of the two (or four) that a word of 8-bit entries
    // becomes, each goes to its own part of the row: neighbouring lanes then
    // write neighbouring words.
    constexpr int kSpread = QUANT ? 16 / E : 1;
    const auto element_of = [](int column) {  // that is at this column of a tile, for runs of E
        const int word = column / E;
        return (word % kRowWords * kSpread + word / kRowWords) * E + column % E;
    };
    constexpr int kStages = SHARED ? 2 : kAttendWaves;
    constexpr uint32_t kStep = kKeys * (SHARED ? 1 : kAttendWaves);  // from one tile of a wave to the next
    constexpr int kStride = SIZE + 4;  // of a row where waves join
    // Tiles in flight, of 8 kEach registers each.
    constexpr int kMostAhead = SHARED ? 2 : 4;
    constexpr int kAhead = 8 / kEach < 1 ? 1 : 8 / kEach > kMostAhead ? kMostAhead : 8 / kEach;

    __shared__ __attribute__((aligned(1024))) char tiles[kStages][2 * TileOf::kBytes];
    __shared__ __attribute__((aligned(16))) float scales[QUANT ? kStages : 1][64];
    __shared__ uint64_t sums[kAttendWaves], found[2];
    __shared__ float2 stats[SHARED ? 1 : kAttendWaves][16];
    static_assert(SHARED || sizeof(tiles) >= kAttendWaves * 16 * kStride * sizeof(float), "waves join in the tiles' place");

    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, quarter = lane / 16;

    // ---- this block's tiles -----------------------------------------------------
    const uint32_t sequences = PREFIX ? 1 : a.batch.sequences;
    uint64_t total_tiles = 0;
    [[maybe_unused]] uint64_t count_here = 0, upto_here = 0;  // of this thread's sequence, and with those before
    if constexpr (PREFIX) {
        total_tiles = LineOf::count(a, sequence_at<true>(a, 0));
    } else {
        // (With up to kAttendThreads sequences each thread keeps its one's.)
        uint64_t mine = 0;
        bool cut = false;
        for (uint32_t n = threadIdx.x; n < sequences; n += kAttendThreads) {
            const Sequence s = sequence_at<false>(a, n);
            count_here = LineOf::count(a, s);
            cut = cut || s.length < s.tokens;
            mine += count_here;
        }
        if (sequences == 0 || a.batch.offsets != nullptr) {
            const uint64_t all = uint64_t{a.batch.tokens} * a.query_heads;
            const auto upto = [&](uint32_t n) {
                const uint32_t token = sequences == 0 ? a.batch.tokens : a.batch.offsets[n];
                return uint64_t{token < a.batch.tokens ? token : a.batch.tokens} * a.query_heads;
            };
            const uint64_t step = uint64_t{gridDim.x} * kAttendThreads, mine_first = uint64_t{blockIdx.x} * kAttendThreads + threadIdx.x;
            for (uint64_t i = mine_first; i < upto(0); i += step) parts.found[i] = {1, 0, 0, kOutside};
            for (uint64_t i = upto(sequences) + mine_first; i < all; i += step) parts.found[i] = {1, 0, 0, kOutside};
        }
        upto_here = mine;
        for (int offset = 1; offset < 64; offset *= 2) {
            const uint64_t other = __shfl_up(static_cast<unsigned long long>(upto_here), offset);
            if (lane >= offset) upto_here += other;
        }
        if (lane == 63) sums[wave] = upto_here;
        cut = __syncthreads_or(cut);
        if (cut || a.batch.most_pages == 0) {
            // The rows of sequences without keys are no block's item: they are
            // marked by the block whose turn the sequence is.
            for (uint32_t n = blockIdx.x; n < sequences; n += gridDim.x) {
                const Sequence s = sequence_at<false>(a, n);
                if (s.keys != 0) continue;
                const uint64_t from = uint64_t{s.first} * a.query_heads, count = uint64_t{s.tokens} * a.query_heads;
                for (uint64_t i = threadIdx.x; i < count; i += kAttendThreads) parts.found[from + i] = {1, 0, 0, 0};
            }
        }
        for (int w = 0; w < kAttendWaves; w++) {
            if (w < wave) upto_here += sums[w];
            total_tiles += sums[w];
        }
        total_tiles = uniform(total_tiles);
        if (blockIdx.x == 0 && threadIdx.x == 0) *parts.cut = cut;
    }
    // No block has nothing, so that every one between two parts of an item has
    // a part of it.
    const uint64_t blocks = total_tiles < gridDim.x ? total_tiles : gridDim.x;
    if (blockIdx.x >= blocks) return;
    const uint64_t begin = blockIdx.x * total_tiles / blocks, end = (blockIdx.x + uint64_t{1}) * total_tiles / blocks;

    uint32_t sequence = 0;
    uint64_t before = 0;  // tiles of the sequences before
    if constexpr (!PREFIX) {
        const auto find = [&](uint32_t n, uint64_t start, uint64_t count) {
            if (begin >= start && begin - start < count) found[0] = n, found[1] = start;
        };
        if (sequences <= kAttendThreads) find(threadIdx.x, upto_here - count_here, count_here);
        __syncthreads();
        for (uint32_t from = 0; sequences > kAttendThreads && from < sequences; from += kAttendThreads) {
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
            find(n, before + upto - count, count);
            __syncthreads();
            if (begin - before < all) break;  // the same for the whole block
            before += all;
        }
        sequence = uniform(static_cast<uint32_t>(found[0]));
        before = uniform(found[1]);
    }
    [[maybe_unused]] bool cut = false;
    if constexpr (PREFIX) cut = uniform(*parts.cut) != 0;

    const uint32_t row_place = TileOf::row_place(lane), column_place = TileOf::column_place(lane);
    int stage = SHARED ? 0 : wave;

    for (uint64_t at = begin; at < end;) {
        Sequence s = sequence_at<PREFIX>(a, sequence);
        if constexpr (!PREFIX) {
            s.first = uniform(s.first), s.tokens = uniform(s.tokens), s.keys = uniform(s.keys), s.length = uniform(s.length);
        }
        const uint32_t tile_count = LineOf::tiles(s), row_blocks = LineOf::blocks(a, s);
        const uint64_t count = uint64_t{tile_count} * row_blocks * a.pool.heads;
        if (at - before >= count) {
            before += count;
            sequence++;
            continue;
        }
        const uint32_t item = static_cast<uint32_t>((at - before) / tile_count);
        const uint32_t tile_0 = static_cast<uint32_t>((at - before) % tile_count);
        const uint32_t tile_1 = end - at < tile_count - tile_0 ? tile_0 + static_cast<uint32_t>(end - at) : tile_count;
        const uint32_t key_head = item / row_blocks, row_block = item % row_blocks;
        const bool whole = tile_0 == 0 && tile_1 == tile_count;
        // (An item's first part is the block's first if both begin together.)
        const uint32_t slot = 2 * blockIdx.x + (at > begin);

        // ---- this lane's query row ---------------------------------------------------
        const uint32_t first_row = row_block * ROWS, left_rows = s.tokens * a.group - first_row;
        const uint32_t rows = left_rows < ROWS ? left_rows : ROWS;
        const uint32_t row = (SHARED ? wave * 16 : 0) + lane % 16;
        const bool real = row < rows;
        const uint32_t place = a.group_of.div(real ? first_row + row : 0);
        const uint32_t token = s.first + place;
        const uint32_t head = key_head * a.group + (real ? first_row + row : 0) - place * a.group;
        uint32_t seen = s.keys;
        if (real) {
            if constexpr (PREFIX) {
                Span span;
                const uint32_t own = cut ? sequence_of(a.batch, token, &span) : kNowhere;
                if (own != kNowhere) seen = seen_of(a.batch.lengths[own], span.end - token, s.keys, s.keys);
            } else {
                seen = seen_of(s.length, s.tokens - place, 0, s.keys);
            }
            if (tile_0 == 0 && quarter == 0 && (SHARED || wave == 0)) {
                const uint64_t last = ((at + tile_count) * blocks - 1) / total_tiles;
                parts.found[uint64_t{token} * a.query_heads + head] = {
                    blockIdx.x, static_cast<uint32_t>(last), slot * ROWS + row,
                    static_cast<uint32_t>((whole ? kWhole : 0) | (seen > 0 ? kSees : 0))};
            }
        }
        // Keys that every, and that any, row of the block sees.
        uint32_t least, most_seen = s.keys;
        if constexpr (PREFIX) {
            const bool all_see = seen == s.keys;
            least = (SHARED ? __syncthreads_and(all_see) : __ballot(!all_see) == 0) ? s.keys : 0;
        } else {
            least = seen_of(s.length, s.tokens - a.group_of.div(first_row), 0, s.keys);
            most_seen = seen_of(s.length, s.tokens - a.group_of.div(first_row + rows - 1), 0, s.keys);
        }
        least = uniform(least), most_seen = uniform(most_seen);
        const uint32_t key_end = uint64_t{tile_1} * kKeys < most_seen ? tile_1 * kKeys : most_seen;

        // ---- tiles on their way --------------------------------------------------------
        uint4 key_words[kAhead][kEach], value_words[kAhead][kEach];
        float entry_scale[kAhead];  // of keys in the lower half of a wave, of values in the upper
        // The page of key l % 32 of the tile at `first`, and its row there.
        const auto page_at = [&](uint32_t first) {
            const uint32_t key = first + lane % 32;
            const uint32_t n = a.pool.pages_of.div(key);
            return lane % 32 < kKeys && key < key_end && n < s.page_count ? s.pages[n] : kNowhere;
        };
        const auto row_at = [&](uint32_t first, uint32_t page) {
            const uint32_t key = first + lane % 32;
            const uint32_t within = key - a.pool.pages_of.div(key) * a.pool.page_size;
            return page < a.pool.page_count ? (page * a.pool.heads + key_head) * a.pool.page_size + within : kNowhere;
        };
        const uint32_t row_bytes = a.pool.row * kEntry;
        const uint32_t mover = SHARED ? threadIdx.x : lane;
        const auto fetch = [&](auto set, uint32_t from_row) {
            constexpr int d = decltype(set)::value;
            // Where pages hold whole runs of 16 tokens and the tile is full, a
            // run's first row tells the others': one address of the wave's, and
            // one number of the lane's.
            const bool runs = a.pool.page_size % 16 == 0 && row_bytes == kRowWords * 16 &&
                              __ballot(from_row == kNowhere && lane % 32 < kKeys) == 0;
            if (runs) {
                uint64_t run[kBlocks16];
#pragma unroll
                for (int n = 0; n < kBlocks16; n++) {
                    run[n] = uint64_t{static_cast<uint32_t>(__builtin_amdgcn_readlane(from_row, 16 * n))} * row_bytes;
                }
#pragma unroll
                for (int k = 0; k < kEach; k++) {
                    const int i = k * kMovers + mover;
                    if (kKeys * kRowWords % kMovers != 0 && i >= kKeys * kRowWords) continue;
                    const uint64_t from = run[kBlocks16 > 1 && i / kRowWords >= 16 ? 1 : 0] + i % (16 * kRowWords) * 16;
                    key_words[d][k] = load_word<false>(static_cast<const char*>(a.pool.keys) + from);
                    value_words[d][k] = load_word<false>(static_cast<const char*>(a.pool.values) + from);
                }
            } else {
                // (The lane's numbers are found here: kept through the loop they
                // would take registers of the path above.)
                uint32_t here = mover;
                asm volatile("" : "+v"(here));
#pragma unroll
                for (int k = 0; k < kEach; k++) {
                    const int i = k * kMovers + here;
                    const uint32_t from = __shfl(from_row, i / kRowWords < kKeys ? i / kRowWords : 0);
                    const uint32_t byte = i % kRowWords * 16;
                    key_words[d][k] = value_words[d][k] = make_uint4(0, 0, 0, 0);
                    if (i < kKeys * kRowWords && from != kNowhere && byte < row_bytes) {
                        const uint64_t at_byte = uint64_t{from} * row_bytes + byte;
                        key_words[d][k] = load_word<false>(static_cast<const char*>(a.pool.keys) + at_byte);
                        value_words[d][k] = load_word<false>(static_cast<const char*>(a.pool.values) + at_byte);
                    }
                }
            }
            if constexpr (QUANT) {
                entry_scale[d] =
                    from_row == kNowhere ? 0.0f : (lane < 32 ? a.pool.key_scales : a.pool.value_scales)[from_row];
            }
        };
        uint32_t tile = 0;
        uint32_t pages[kAhead], next_page[2];  // of the first tiles, and of the next ones to fetch
        const auto find_pages = [&]() {
            tile = (tile_0 + (SHARED ? 0 : wave)) * kKeys;
            each<kAhead>([&](auto n) { pages[n.value] = page_at(tile + n.value * kStep); });
            next_page[0] = page_at(tile + kAhead * kStep);
            next_page[1] = page_at(tile + (kAhead + 1) * kStep);
        };
        const auto fetch_first = [&]() {
            each<kAhead>([&](auto n) { fetch(n, row_at(tile + n.value * kStep, pages[n.value])); });
        };
        find_pages();

        // ---- queries -------------------------------------------------------------------
        uint4 queries[kOperands];
        const S* from = static_cast<const S*>(a.query) + token * a.query_steps.token + head * a.query_steps.head;
#pragma unroll
        for (int n = 0; n < kOperands; n++) {
            const int word = element_of((4 * n + quarter) * E) / E;
            queries[n] = real ? head_word(from, word, a.pool.size) : make_uint4(0, 0, 0, 0);
        }
        fetch_first();
        const float factor = a.scale * attention::kLog2e;  // of the scores, in powers of two

        // ---- a sweep over the part's tiles -----------------------------------------
        f32x4 acc[SIZE / 16];
        float most, total;
        // Where the lane's first word of a tile lands, of which the others' places
        // follow if a row's words and the rows a step has are powers of two.
        constexpr int kStepRows = kMovers / kRowWords;
        constexpr bool kRegular = (kRowWords & (kRowWords - 1)) == 0 && kMovers % kRowWords == 0 &&
                                  kKeys * kRowWords % kMovers == 0;
        const uint32_t mover_place = TileOf::Base::place(mover / kRowWords, mover % kRowWords);
        const auto land = [&](auto set, const TileOf& key_tile, const TileOf& value_tile) {
            constexpr int d = decltype(set)::value;
            const auto place_in = [&](const TileOf& to, int k, int w) {
                if constexpr (kRegular) return to.from(mover_place, k * kStepRows, w * kRowWords);
                const int i = k * kMovers + mover;
                return to.word(i / kRowWords, i % kRowWords + w * kRowWords);
            };
#pragma unroll
            for (int k = 0; k < kEach; k++) {
                if (kKeys * kRowWords % kMovers != 0 && k * kMovers + mover >= kKeys * kRowWords) continue;
                if constexpr (QUANT) {
                    Words<S, 16> keys;
                    Words<V, 16> values;
                    widened(key_words[d][k], keys);
                    widened(value_words[d][k], values);
#pragma unroll
                    for (int w = 0; w < kSpread; w++) {
                        *reinterpret_cast<uint4*>(place_in(key_tile, k, w)) = keys.w[w];
                        *reinterpret_cast<uint4*>(place_in(value_tile, k, w)) = values.w[w];
                    }
                } else {
                    *reinterpret_cast<uint4*>(place_in(key_tile, k, 0)) = key_words[d][k];
                    *reinterpret_cast<uint4*>(place_in(value_tile, k, 0)) = value_words[d][k];
                }
            }
            if constexpr (QUANT) {
                if (!SHARED || wave == 0) scales[stage][lane] = entry_scale[d];
            }
        };
        [[maybe_unused]] int pick = kFinite;
        // The tile that is in `set`; its next one's page is the `parity`-th.
        const auto turn = [&](auto set, auto parity, auto is_slow) {
            constexpr bool SLOW = decltype(is_slow)::value;
            constexpr int p = decltype(parity)::value;
            // (Keys past `key_end` are seen by no row, or by none that is real.)
            const bool masked = tile + kKeys > least || tile + kKeys > key_end;
            const TileOf key_tile{tiles[stage]};
            const TileOf value_tile{tiles[stage] + TileOf::kBytes};
            // A stage that a block shares was read before the last barrier; a
            // wave's own is in the order of the program.
            if constexpr (!SHARED) wave_order();
            land(set, key_tile, value_tile);
            if constexpr (SHARED) __syncthreads();
            else wave_order();
            const uint32_t next = tile + kAhead * kStep;
            if (next < key_end) {
                fetch(set, row_at(next, next_page[p]));
                next_page[p] = page_at(next + 2 * kStep);
            }
            // Scores, and their maximum over the tile.
            f32x4 scores[kBlocks16];
#pragma unroll
            for (int b = 0; b < kBlocks16; b++) {
                scores[b] = f32x4{};
#pragma unroll
                for (int n = 0; n < kOperands; n++) {
                    scores[b] = product16<S>(key_tile.by_row(row_place, b, n), queries[n], scores[b]);
                }
                if constexpr (QUANT) scores[b] *= *reinterpret_cast<const f32x4*>(&scales[stage][16 * b + 4 * quarter]);
            }
            const auto sees = [&](int b, int i) { return tile + 16 * b + 4 * quarter + i < seen; };
            if (masked) {
#pragma unroll
                for (int b = 0; b < kBlocks16; b++) {
#pragma unroll
                    for (int i = 0; i < 4; i++) scores[b][i] = sees(b, i) ? scores[b][i] : -INFINITY;
                }
            }
            float high = -INFINITY;
#pragma unroll
            for (int b = 0; b < kBlocks16; b++) {
#pragma unroll
                for (int i = 0; i < 4; i++) high = fmaxf(high, scores[b][i]);
            }
            high = quarters<Largest>(high) * factor;
            // The maximum only moves when it grows past 2^8: the weights stay
            // that small, and the sums are rarely rescaled.
            const bool grows = high > most + 8.0f;
            if (__ballot(grows) != 0) {
                const float kept = grows ? power2(most - high) : 1.0f;
                if (grows) most = high;
                total *= kept;
#pragma unroll
                for (int t = 0; t < SIZE / 16; t++) acc[t] *= kept;
            }
            const float origin = (most == -INFINITY ? 0.0f : most) - kPower;
#pragma unroll
            for (int b = 0; b < kBlocks16; b++) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    scores[b][i] = power2(fmaf(scores[b][i], factor, -origin));
                    total += scores[b][i];
                }
                if constexpr (QUANT) {
                    scores[b] *= *reinterpret_cast<const f32x4*>(&scales[stage][32 + 16 * b + 4 * quarter]);
                    if (masked) {
                        // (A scale may be a NaN.)
#pragma unroll
                        for (int i = 0; i < 4; i++) scores[b][i] = sees(b, i) ? scores[b][i] : 0.0f;
                    }
                }
            }
            // The weights as operands, and their products with the values.
            float v[E];
#pragma unroll
            for (int e = 0; e < E; e++) {
                v[e] = scores[e / 4][e % 4];
                if (SLOW && pick != kFinite) {
                    const bool one = pick == kNaN    ? sees(e / 4, e % 4)
                                     : pick == kZero ? sees(e / 4, e % 4) && v[e] == 0.0f
                                                     : v[e] != 0.0f;
                    v[e] = one ? 1.0f : 0.0f;
                }
            }
            Words<V, E> high_part, low_part;
            if constexpr (Elem<V>::dtype == TC_F16) {
                // Cut off, two by one instruction: the second part takes what is
                // left (512 new of 8704 tokens 170 us so, 181 rounded).
                uint32_t* const to = reinterpret_cast<uint32_t*>(high_part.w);
#pragma unroll
                for (int e = 0; e < E; e += 2) {
                    to[e / 2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(v[e], v[e + 1]));
                }
            } else {
                high_part.put(v);
            }
            if constexpr (kTwoParts) {
#pragma unroll
                for (int e = 0; e < E; e++) v[e] -= high_part.at(e);
                low_part.put(v);
            }
#pragma unroll
            for (int t = 0; t < SIZE / 16; t++) {
                uint4 values = value_tile.by_column(column_place, t);
                if constexpr (SLOW) {
                    values = make_uint4(picked(values.x, pick), picked(values.y, pick), picked(values.z, pick),
                                        picked(values.w, pick));
                }
                acc[t] = product16<V>(values, high_part.w[0], acc[t]);
                if constexpr (kTwoParts) acc[t] = product16<V>(values, low_part.w[0], acc[t]);
            }
            tile += kStep;
            if constexpr (SHARED) stage ^= 1;
        };
        // Over the tiles, of which the first are on their way.
        const auto sweep = [&](auto is_slow) {
            if constexpr (!decltype(is_slow)::value) most = -INFINITY;
            total = 0.0f;
#pragma unroll
            for (int t = 0; t < SIZE / 16; t++) acc[t] = f32x4{};
            while (tile < key_end) {
                each<(kAhead > 2 ? kAhead : 2)>([&](auto n) {
                    if (n.value == 0 || tile < key_end) {
                        turn(std::integral_constant<int, n.value % kAhead>(), std::integral_constant<int, n.value % 2>(),
                             is_slow);
                    }
                });
            }
        };
        sweep(std::false_type());
        if constexpr (!QUANT) {
            // A value that is an infinity or a NaN has spoiled every row, its
            // weight being 0 in those that do not see it, or 0 in the second of
            // two parts.  So once more for each kind of them, counting those
            // that are seen, and at last without them; against the maximum that
            // the first sweep ended with, so that what it counts is not scaled
            // down by scores that come later.
            bool spoiled = false;
#pragma unroll
            for (int t = 0; t < SIZE / 16; t++) {
#pragma unroll
                for (int i = 0; i < 4; i++) spoiled |= !(fabsf(acc[t][i]) < INFINITY);
            }
            const bool any = SHARED ? __syncthreads_or(spoiled) != 0 : __ballot(spoiled) != 0;
            if (__builtin_expect(any, false)) {
                uint32_t up = 0, down = 0;  // a bit an element, both for a NaN
#pragma unroll 1
                for (pick = kZero; pick >= kFinite; pick--) {
                    find_pages();
                    fetch_first();
                    sweep(std::true_type());
                    if (pick == kFinite) break;
                    uint32_t bits = 0;
#pragma unroll
                    for (int t = 0; t < SIZE / 16; t++) {
#pragma unroll
                        for (int i = 0; i < 4; i++) bits |= acc[t][i] > 0.0f ? 1u << (4 * t + i) : 0u;
                    }
                    if (pick != kMinus) up |= bits;
                    if (pick != kPlus) down |= bits;
                }
#pragma unroll
                for (int t = 0; t < SIZE / 16; t++) {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        if (up >> (4 * t + i) & 1) acc[t][i] += INFINITY;
                        if (down >> (4 * t + i) & 1) acc[t][i] -= INFINITY;
                    }
                }
            }
        }

        // ---- the part's sums stored ----------------------------------------------------
        const auto store = [&](uint32_t of_token, uint32_t of_head, uint32_t slot_row, bool any, uint32_t column, f32x4 v,
                               float top, float all) {
            if (whole && final) {
                // (A sum of 0 over keys that are seen is of scores of -infinity
                // alone: 0 / 0.)
                S* const to = static_cast<S*>(a.out) + of_token * a.out_steps.token + of_head * a.out_steps.head;
                store_four(to, column, a.pool.size, any ? v * (1.0f / all) : f32x4{});
                if (column == 0 && a.normalizers != nullptr) {
                    a.normalizers[uint64_t{of_head} * a.batch.tokens + of_token] =
                        all == 0.0f ? -INFINITY : (top + log2f(all) - kPower) * attention::kLn2;
                }
            } else {
                const uint64_t to = whole ? uint64_t{of_token} * a.query_heads + of_head : uint64_t{slot} * ROWS + slot_row;
                *reinterpret_cast<f32x4*>((whole ? parts.rows : parts.slots) + to * SIZE + column) = v;
                if (column == 0) (whole ? parts.row_stats : parts.slot_stats)[to] = make_float2(top, all);
            }
        };
        const float all = quarters<Added>(total);
        if constexpr (SHARED) {
            if (real) {
#pragma unroll
                for (int t = 0; t < SIZE / 16; t++) {
                    store(token, head, row, seen > 0, element_of(16 * t + 4 * quarter), acc[t], most, all);
                }
            }
        } else {
            // The waves' sums joined, each against the largest maximum.
            if (lane < 16) stats[wave][lane] = make_float2(most, all);
            __syncthreads();
            const auto joined = [&](uint32_t of_row, float* top, float* sum) {
                *top = -INFINITY, *sum = 0.0f;
                for (int w = 0; w < kAttendWaves; w++) *top = fmaxf(*top, stats[w][of_row].x);
                const float origin = *top == -INFINITY ? 0.0f : *top;
                for (int w = 0; w < kAttendWaves; w++) *sum += power2(stats[w][of_row].x - origin) * stats[w][of_row].y;
            };
            float top, sum;
            joined(lane % 16, &top, &sum);
            const float kept = power2(most - (top == -INFINITY ? 0.0f : top));
            float* const joint = reinterpret_cast<float*>(&tiles[0][0]);
#pragma unroll
            for (int t = 0; t < SIZE / 16; t++) {
                *reinterpret_cast<f32x4*>(joint + (wave * 16 + lane % 16) * kStride + element_of(16 * t + 4 * quarter)) =
                    acc[t] * kept;
            }
            __syncthreads();
            for (uint32_t i = threadIdx.x; i < 16 * SIZE / 4; i += kAttendThreads) {
                const uint32_t of_row = i / (SIZE / 4), column = i % (SIZE / 4) * 4;
                if (of_row >= rows) continue;
                f32x4 v = *reinterpret_cast<const f32x4*>(joint + of_row * kStride + column);
                for (int w = 1; w < kAttendWaves; w++) {
                    v += *reinterpret_cast<const f32x4*>(joint + (w * 16 + of_row) * kStride + column);
                }
                joined(of_row, &top, &sum);
                const uint32_t of_place = a.group_of.div(first_row + of_row);
                const bool any = PREFIX || seen_of(s.length, s.tokens - of_place, 0, s.keys) > 0;
                store(s.first + of_place, key_head * a.group + first_row + of_row - of_place * a.group, of_row, any, column,
                      v, top, sum);
            }
            __syncthreads();
        }
        at += tile_1 - tile_0;
    }
}

// Each row's parts joined, by WAVES waves: the row's own sequence's and the
// prefix's, in the order of their blocks, two a wave at a time.
template <int SIZE, int WAVES>
__global__ void __launch_bounds__(kAttendThreads)
    join_kernel(const Attention a, const Parts own, const Parts prefix, uint32_t own_rows, uint32_t prefix_rows,
                uint32_t own_blocks, uint32_t prefix_blocks, float power) {
    constexpr int kRows = kAttendWaves / WAVES;  // of a block
    __shared__ f32x4 sums[WAVES > 1 ? WAVES : 1][32];
    __shared__ float2 stats_of[WAVES > 1 ? WAVES : 1];
    const int wave = threadIdx.x / 64 % WAVES;
    const uint64_t apart = uint64_t{gridDim.x} * kRows, all_rows = uint64_t{a.batch.tokens} * a.query_heads;
    for (uint64_t at = uint64_t{blockIdx.x} * kRows + threadIdx.x / 64 / WAVES; at < all_rows; at += apart) {
        const uint32_t row = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(at));
        const uint32_t token = row / a.query_heads, head = row % a.query_heads;
        const Found mine = own.found[row];
        const Found shared = a.batch.prefix > 0 ? prefix.found[row] : Found{1, 0, 0, 0};
        // (Offsets that do not rise leave rows that no item has: what is found
        // for them is none of the slots, or any.)
        const auto count_of = [](const Found& f, uint32_t blocks, uint32_t line) {
            return f.marks & kWhole                                                               ? 1
                   : f.first <= f.last && f.last < blocks && f.place < 2 * uint64_t{blocks} * line ? f.last - f.first + 1
                                                                                                   : 0;
        };
        const bool outside = (mine.marks & kOutside) != 0;
        const uint32_t mine_count = outside ? 0 : count_of(mine, own_blocks, own_rows);
        const uint32_t count = outside ? 0 : mine_count + count_of(shared, prefix_blocks, prefix_rows);
        const bool sees = !outside && ((mine.marks | shared.marks) & kSees) != 0;
        // A whole item without a prefix is a result already.
        if (mine_count == 1 && (mine.marks & kWhole) && a.batch.prefix == 0) continue;

        const uint32_t half = threadIdx.x % 64 / 32, column = threadIdx.x % 32 * 4;
        float top = -INFINITY, total = 0.0f;
        f32x4 sum = {};
        // Four parts in flight: their loads, then their sums.
        constexpr int kParts = 4;
        for (uint32_t first = 2 * wave + half; first < count; first += kParts * 2 * WAVES) {
            float2 stats[kParts];
            f32x4 values[kParts];
#pragma unroll
            for (int k = 0; k < kParts; k++) {
                const uint32_t i = first + k * 2 * WAVES;
                stats[k] = make_float2(-INFINITY, 0.0f);
                values[k] = f32x4{};
                if (i >= count) continue;
                const bool is_mine = i < mine_count;
                const Found& f = is_mine ? mine : shared;
                const Parts& parts = is_mine ? own : prefix;
                const uint32_t n = is_mine ? i : i - mine_count, line = is_mine ? own_rows : prefix_rows;
                // (`line` is a power of two.)
                const bool whole = (f.marks & kWhole) != 0;
                const uint32_t place = whole ? row : n == 0 ? f.place : 2 * (f.first + n) * line + (f.place & (line - 1));
                stats[k] = (whole ? parts.row_stats : parts.slot_stats)[place];
                if (column < SIZE) {
                    values[k] =
                        *reinterpret_cast<const f32x4*>((whole ? parts.rows : parts.slots) + uint64_t{place} * SIZE + column);
                }
            }
#pragma unroll
            for (int k = 0; k < kParts; k++) {
                const float higher = fmaxf(top, stats[k].x), origin = higher == -INFINITY ? 0.0f : higher;
                const float kept = power2(top - origin), added = power2(stats[k].x - origin);
                total = fmaf(total, kept, stats[k].y * added);
                sum = sum * kept + values[k] * added;
                top = higher;
            }
        }
        float higher = fmaxf(top, __shfl_xor(top, 32));
        const float kept = power2(top - (higher == -INFINITY ? 0.0f : higher));
        total *= kept;
        total += __shfl_xor(total, 32);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            sum[j] *= kept;
            sum[j] += __shfl_xor(sum[j], 32);
        }
        if constexpr (WAVES > 1) {
            if (half == 0) sums[wave][threadIdx.x % 32] = sum;
            if (threadIdx.x % 64 == 0) stats_of[wave] = make_float2(higher, total);
            __syncthreads();
            higher = -INFINITY, total = 0.0f, sum = f32x4{};
            for (int w = 0; w < WAVES; w++) higher = fmaxf(higher, stats_of[w].x);
            for (int w = 0; w < WAVES; w++) {
                const float factor = power2(stats_of[w].x - (higher == -INFINITY ? 0.0f : higher));
                total += stats_of[w].y * factor;
                sum += sums[w][threadIdx.x % 32] * factor;
            }
            __syncthreads();
        }
        if (half == 0 && wave == 0) {
            S* const to = static_cast<S*>(a.out) + token * a.out_steps.token + head * a.out_steps.head;
            const float scale = 1.0f / total;
            store_four(to, column, a.pool.size, sees ? sum * scale : f32x4{});
            if (threadIdx.x % 32 == 0 && a.normalizers != nullptr) {
                a.normalizers[uint64_t{head} * a.batch.tokens + token] =
                    total == 0.0f ? -INFINITY : (higher + log2f(total) - power) * attention::kLn2;
            }
        }
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

template <int SIZE, bool QUANT>
void attend_size(const Attention& a, const Parts& parts, bool prefix, bool final, bool shared, hipStream_t s) {
    const uint32_t blocks = static_cast<uint32_t>(compute_units()) * blocks_of_form(shared);
    const auto kernel = shared ? prefix ? attend_kernel<SIZE, true, QUANT, true> : attend_kernel<SIZE, true, QUANT, false>
                        : prefix ? attend_kernel<SIZE, false, QUANT, true>
                                 : attend_kernel<SIZE, false, QUANT, false>;
    kernel<<<blocks, kAttendThreads, 0, s>>>(a, parts, final);
}

int attend(const Attention& a, const Parts& parts, bool quant, bool prefix, bool final, bool shared) {
    TC_STREAM(s);
    TC_CACHE_SIZE(a.pool.size, {
        if (quant) {
            attend_size<SIZE, true>(a, parts, prefix, final, shared, s);
        } else {
            attend_size<SIZE, false>(a, parts, prefix, final, shared, s);
        }
    })
    return check_launch("cache attention");
}

int join(const Attention& a, const Parts& own, const Parts& prefix, bool quant, bool own_shared, bool prefix_shared) {
    TC_STREAM(s);
    const uint32_t units = static_cast<uint32_t>(compute_units());
    const uint64_t rows = uint64_t{a.batch.tokens} * a.query_heads;
    // A block a row where rows are few and their parts, therefore, many.  (One
    // sequence of 1000 tokens 13.1 us, with a wave a row 17.1, four of 100000 113
    // and 118; the other way 64 sequences of 32 heads 226 instead of 220.)
    const bool few = rows <= uint64_t{units} * 4;
    const uint64_t turns = few ? rows : (rows + kAttendWaves - 1) / kAttendWaves;
    const uint32_t grid = turns < (1u << 20) ? static_cast<uint32_t>(turns) : 1u << 20;
    const float power = power_of(quant);
    TC_CACHE_SIZE(a.pool.size, {
        const auto kernel = few ? join_kernel<SIZE, kAttendWaves> : join_kernel<SIZE, 1>;
        kernel<<<grid, kAttendThreads, 0, s>>>(a, own, prefix, rows_of_form(own_shared), rows_of_form(prefix_shared),
                                               units * blocks_of_form(own_shared),
                                               units * blocks_of_form(prefix_shared), power);
    })
    return check_launch("cache attention");
}

}  // namespace

#endif  // TC_ATTENTION_TYPE

}  // namespace cache
}  // namespace tc
