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
// forward, where it may reach 2^8), and ds, which is at most 2 |do| |v|, times
// the power of two that brings the largest of that in its own sum below 2^15.
//
// Measured (a large bf16 product reaches 1372 TFLOP/s): 8192 tokens, 16 heads
// of 128 on 4 key heads, bf16, 1252 us in all, of which forward 306 (900
// TFLOP/s, the matrix cores busy 54% of the time), dq 395 (1040, 60%), dk and dv
// 616 (890, 47%; both with the two products that the other computes too); 16384
// tokens, 8 heads of 64 on one, forward 323 us (850); 7001 f16 tokens of 19
// sequences, 12 heads of 80, forward and backward 154 us, in which the matrix
// cores are busy 19 to 23% of the time and waves wait for 42 to 46% of theirs:
// a tile's loads are issued one tile before all of them are waited for.  What
// carried it: loads straight to LDS (forward 397 -> 330 us), one number a lane
// for all LDS addresses and a path without masks (330 -> 305), 256 keys a block
// for dk and dv (816 -> 675 then), blocks by sequence (7001 tokens, 237 -> 154).
//   Rows that are no whole 16-byte words go through registers to LDS, several
// times slower: those 8192 tokens with heads of 127 4280 us, the 16384 with
// heads of 63 1464.  f32, 4096 tokens, 8 heads on 2: of 64 1251 us forward and
// backward (48 TFLOP/s of the 143 of a large product), of 128 2555; the
// gradients' kernels of f32 heads past 64 keep up to 22 registers a tile in
// memory.
//
// Sequences lie one behind another.  A tile that some row of a wave sees only
// in part is masked element by element.  A masked weight is 0, and 0 times an
// infinity or a NaN would be a NaN, so a tile that is masked and holds such a
// value takes a slow path: the product with zeros in their place, then theirs
// alone where the weight is not 0.
#pragma once

#include <type_traits>
#include <utility>

#include "attention_tiles.hpp"

namespace tc {
namespace attention {

constexpr int kThreads = 256;
constexpr uint32_t kOwned = 128;  // queries (or keys) of a block, 32 a wave
constexpr int kBufferFlags = 0x00020000;       // raw 32-bit data
constexpr uint32_t kOutside = 0x80000000u;    // an offset past any buffer resource here
constexpr int kWaitForAll = 0x7 << 4;          // vmcnt(0), lgkmcnt(0)

struct Shape {
    uint32_t heads, group;  // query heads, and of them to a key head
    uint32_t size;
    uint32_t tokens;
    uint32_t sequences;  // 0: all tokens are one
    uint32_t by_sequence;  // blocks end where sequences do (`Owned`)
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

constexpr uint32_t kSwept = kWide ? 32 : 64;  // rows of a tile in LDS
// Powers of two that weights are rounded times, forward and backward.
constexpr float kForwardPower = kHalf ? 6.0f : 0.0f, kBackPower = kHalf ? 14.0f : 0.0f;

// How tiles get from memory to LDS.  DIRECT, for rows of whole 16-byte words:
// loads that write LDS themselves, each lane fetching the word that belongs
// where it writes, zeros past the rows and a head's size because those lie
// past the buffer resource.  Otherwise through registers, word by word.
template <int SIZE, int ROWS, bool DIRECT, int THREADS = kThreads>
struct Stager {
    static constexpr int kWords = SIZE / E;
    static constexpr int kEach = ROWS * kWords / THREADS;
    static_assert(ROWS * kWords % THREADS == 0, "every thread has as many words");
    using LdsTile = Tile<SIZE, ROWS>;

    uint64_t step;
    uint32_t size;
    uint32_t offsets[DIRECT ? kEach : 1];
    uint4 words[DIRECT ? 1 : kEach];

    __device__ __forceinline__ Stager(uint64_t token_step, uint32_t head_size) : step(token_step), size(head_size) {
        if constexpr (DIRECT) {
#pragma unroll
            for (int k = 0; k < kEach; k++) {
                const int i = threadIdx.x + k * THREADS;
                const int row = i / kWords, word = LdsTile::permuted(row, i % kWords);
                offsets[k] = word * E < static_cast<int>(size)
                                 ? (row * static_cast<uint32_t>(step) + word * E) * sizeof(S)
                                 : kOutside;
            }
        }
    }
    // Rows first .. first + ROWS of a head towards `tile`, zeros from token
    // `limit` on; all arguments the same for the whole wave.
    __device__ __forceinline__ void fetch(const LdsTile& tile, const S* head, uint32_t first, uint32_t limit) {
        if constexpr (DIRECT) {
            const uint32_t rows = first >= limit ? 0 : limit - first < ROWS ? limit - first : ROWS;
            const uint32_t bytes = rows == 0 ? 0 : ((rows - 1) * static_cast<uint32_t>(step) + size) * sizeof(S);
            const int wave = threadIdx.x / 64;
#if defined(__HIP_DEVICE_COMPILE__)  // the host's pass drops kernels over these builtins
            const auto resource =
                __builtin_amdgcn_make_buffer_rsrc(const_cast<S*>(head + first * step), 0, bytes, kBufferFlags);
#pragma unroll
            for (int k = 0; k < kEach; k++) {
                char* to = tile.at + 1024 * (wave + k * (THREADS / 64));
                __builtin_amdgcn_raw_ptr_buffer_load_lds(resource, (__attribute__((address_space(3))) void*)to, 16,
                                                         offsets[k], 0, 0, 0);
            }
#else
            (void)bytes, (void)wave;
#endif
        } else {
#pragma unroll
            for (int k = 0; k < kEach; k++) {
                const int i = threadIdx.x + k * THREADS;
                const uint32_t token = first + i / kWords;
                words[k] = token < limit ? head_word(head + token * step, i % kWords, size) : make_uint4(0, 0, 0, 0);
            }
        }
    }
    // The last rows fetched are in LDS, for this thread, when this returns.
    __device__ __forceinline__ void land(const LdsTile& tile) const {
        if constexpr (DIRECT) {
            __builtin_amdgcn_s_waitcnt(kWaitForAll);
        } else {
#pragma unroll
            for (int k = 0; k < kEach; k++) {
                const int i = threadIdx.x + k * THREADS;
                *reinterpret_cast<uint4*>(tile.word(i / kWords, i % kWords)) = words[k];
            }
        }
    }
};

// Whether any of this thread's share of a tile is an infinity or a NaN.
template <int THREADS, int SIZE, int ROWS>
__device__ __forceinline__ bool specials_in(const Tile<SIZE, ROWS>& tile) {
    bool any = false;
#pragma unroll
    for (int k = 0; k < ROWS * Tile<SIZE, ROWS>::kWords / THREADS; k++) {
        const uint4 w = reinterpret_cast<const uint4*>(tile.at)[threadIdx.x + k * THREADS];
        any |= special_bits(w.x) || special_bits(w.y) || special_bits(w.z) || special_bits(w.w);
    }
    return any;
}

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
        const uint32_t middle = low + (high - low) / 2;  // their sum may pass 32 bits
        if (shape.offsets[middle] <= token) low = middle;
        else high = middle;
    }
    const uint32_t first = shape.offsets[low], end = shape.offsets[low + 1];
    if (token < first || token >= end) return {kNone, 0};
    return {first, end < shape.tokens ? end : shape.tokens};
}

// The tokens that a block owns: from `first` on, `end` not among them.
//   By sequence, a block's tokens are of one sequence (or of none: those before
// the first and past the last offset are taken like one), and what it sweeps
// ends with it; otherwise tiles are every kOwned tokens, cheaper to find, and
// each lane has its own token's span.
struct Owned {
    uint32_t first, end;
    Span span;  // by sequence: of all its tokens
};

// Tile `tile` of `owned` tokens; kNone as `first` past the last one.  Its
// sequence is the one whose tiles, counted over the sequences before it, have
// it: a scan of THREADS sequences at a time.  `backwards` takes a sequence's
// last tile first.
template <int THREADS>
__device__ __forceinline__ Owned owned_by(const Shape& shape, uint32_t owned, uint32_t tile, bool backwards) {
    if (!shape.by_sequence) {
        const uint32_t tiles = (shape.tokens + owned - 1) / owned;
        const uint32_t first = (backwards ? tiles - 1 - tile : tile) * owned;
        return {first, shape.tokens, {0, shape.tokens}};
    }
    __shared__ uint32_t sums[THREADS / 64];
    __shared__ Owned found;
    if (threadIdx.x == 0) found = {kNone, 0, {kNone, 0}};
    uint32_t passed = 0;
    for (uint32_t from = 0; from < shape.sequences + 2; from += THREADS) {
        const uint32_t n = from + threadIdx.x;  // 0 and sequences + 1: of no sequence
        uint32_t first = 0, end = 0;
        if (n < shape.sequences + 2) {
            first = n == 0 ? 0 : shape.offsets[n - 1];
            end = n == shape.sequences + 1 ? shape.tokens : shape.offsets[n];
            end = end < shape.tokens ? end : shape.tokens;
        }
        const uint32_t count = first < end ? (end - first + owned - 1) / owned : 0;
        uint32_t upto = count;
        for (int offset = 1; offset < 64; offset *= 2) {
            const uint32_t other = __shfl_up(upto, offset);
            if (static_cast<int>(threadIdx.x % 64) >= offset) upto += other;
        }
        if (threadIdx.x % 64 == 63) sums[threadIdx.x / 64] = upto;
        __syncthreads();
        uint32_t all = 0;
        for (int w = 0; w < THREADS / 64; w++) {
            if (w < static_cast<int>(threadIdx.x / 64)) upto += sums[w];
            all += sums[w];
        }
        const uint32_t within = tile - (passed + upto - count);  // wraps where the tile is before these
        if (tile >= passed + upto - count && within < count) {
            const bool none = n == 0 || n == shape.sequences + 1;
            found = {first + (backwards ? count - 1 - within : within) * owned, end,
                     none ? Span{kNone, 0} : Span{first, end}};
        }
        passed += all;
        __syncthreads();
    }
    const auto uniform = [](uint32_t v) { return static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(v)); };
    return {uniform(found.first), uniform(found.end), {uniform(found.span.first), uniform(found.span.end)}};
}

// The token behind the last sequence.
__device__ __forceinline__ uint32_t limit_of(const Shape& shape) {
    if (shape.sequences == 0) return shape.tokens;
    const uint32_t end = __builtin_amdgcn_readfirstlane(shape.offsets[shape.sequences]);
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
template <int WAVES>
__device__ __forceinline__ void over_waves(const uint32_t (&values)[2][WAVES], uint32_t* least, uint32_t* most) {
    *least = values[0][0], *most = values[1][0];
    for (int w = 1; w < WAVES; w++) {
        *least = values[0][w] < *least ? values[0][w] : *least;
        *most = values[1][w] > *most ? values[1][w] : *most;
    }
    *least = __builtin_amdgcn_readfirstlane(*least);
    *most = __builtin_amdgcn_readfirstlane(*most);
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

// ---- sums over a tile's rows ------------------------------------------------------------

// acc (SIZE x 32 columns) += the transpose of 32 rows of the tile times the
// 32 x 32 weights; with FINITE, of the tile's finite elements.
template <int SIZE, int ROWS, bool FINITE>
__device__ __forceinline__ void weighted(f32x16 (&acc)[SIZE / 32], const Tile<SIZE, ROWS>& tile, int rows,
                                         const f32x16& weights, const Lanes& lanes) {
#pragma unroll
    for (int n = 0; n < 32 / kDeep; n++) {
        const uint4 weight = operand(weights, n);
#pragma unroll
        for (int t = 0; t < SIZE / 32; t++) {
            uint4 column = tile.by_column(lanes, rows + n * kDeep, t * 32);
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
                    // One read at a time: registers here would be missing in
                    // the loop that this is the exception of.
                    __builtin_amdgcn_sched_barrier(0);
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

// Both, where a tile is MASKED and `special`, or the plain product.
template <int SIZE, int ROWS, bool MASKED>
__device__ __forceinline__ void add_weighted(bool special, f32x16 (&acc)[SIZE / 32], const Tile<SIZE, ROWS>& tile,
                                             int rows, const f32x16& weights, const Lanes& lanes, int lane,
                                             float* scratch) {
    if (MASKED && __builtin_expect(special, false)) {
        weighted<SIZE, ROWS, true>(acc, tile, rows, weights, lanes);
        weighted_specials<SIZE, ROWS>(acc, tile, rows, weights, lane, scratch);
    } else {
        weighted<SIZE, ROWS, false>(acc, tile, rows, weights, lanes);
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

template <int SIZE, bool DIRECT>
__global__ void __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(2)))
    forward_kernel(const Shape shape, const S* __restrict__ q, const S* __restrict__ k, const S* __restrict__ v,
                   S* __restrict__ out, float* __restrict__ normalizers) {
    using KeyTile = Tile<SIZE, kSwept>;
    // A stage an array, so that reads of one do not wait for loads to the other.
    __shared__ __attribute__((aligned(1024))) char stage_0[2 * KeyTile::kBytes], stage_1[2 * KeyTile::kBytes];
    __shared__ float scratch[kThreads / 64][8 * 32];
    __shared__ uint32_t seen[2][kThreads / 64], marks[2];
    constexpr int kOperands = SIZE / kDeep;

    const int lane = threadIdx.x % 64, half = lane / 32, wave = threadIdx.x / 64;
    const Lanes lanes = KeyTile::lanes_of(lane);
    // The latest tokens, which see the most keys, first.
    const uint32_t head = blockIdx.x % shape.heads;
    const Owned mine = owned_by<kThreads>(shape, kOwned, blockIdx.x / shape.heads, true);
    const uint32_t first = mine.first;
    if (first == kNone) return;
    const uint32_t wave_first = first + wave * 32;
    const uint32_t token = wave_first + lane % 32;
    // (Lanes past the block's tokens work as if they had one, for nothing.)
    const Span span = shape.by_sequence ? mine.span : span_of(shape, token);
    const uint32_t limit = shape.by_sequence ? mine.end : limit_of(shape);
    // Keys that some, and that all, of the wave's queries may see.
    const uint32_t some = wave_least(span.first), all = wave_most(span.first);
    if (lane == 0) seen[0][wave] = some, seen[1][wave] = all;
    if (threadIdx.x < 2) marks[threadIdx.x] = 0;

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
    // One sweep over the keys.  Without SLOW it ends, true, at the first masked
    // tile with a special value: what handles those is kept out of the sweep's
    // registers.
    const auto sweep = [&](auto is_slow) {
        constexpr bool SLOW = decltype(is_slow)::value;
        most = -INFINITY, total = 0.0f;
#pragma unroll
        for (int t = 0; t < SIZE / 32; t++) acc[t] = f32x16{};
        // Masked for some query of the block (and the same for all its waves):
        // before a sequence's first key or past the first query.
        const auto masked = [&](uint32_t tile) { return tile < block_all || tile + kSwept - 1 > first; };
        Stager<SIZE, kSwept, DIRECT> key_stager(shape.k.token, shape.size), value_stager(shape.v.token, shape.size);
        uint32_t at = shape.by_sequence ? begin : begin / kSwept * kSwept;
        bool special = false;
        const auto fetch = [&](char* stage, uint32_t tile) {
            key_stager.fetch(KeyTile{stage}, keys, tile, limit);
            value_stager.fetch(KeyTile{stage + KeyTile::kBytes}, values, tile, limit);
        };
        const auto land = [&](char* stage, uint32_t tile) {
            key_stager.land(KeyTile{stage});
            value_stager.land(KeyTile{stage + KeyTile::kBytes});
            // What this thread fetched it may look at before the others have
            // theirs; a stage's mark names the tile, so that none is cleared.
            uint32_t& mark = marks[stage == stage_1];
            if (masked(tile) && specials_in<kThreads>(KeyTile{stage + KeyTile::kBytes})) mark = tile + 1;
            __syncthreads();
            special = masked(tile) && __builtin_amdgcn_readfirstlane(mark) == tile + 1;
        };
        // The tile at `at` in stage `here`, while the next one is on its way.
        const auto turn = [&](char* here, char* there) {
            const KeyTile key_tile{here}, value_tile{here + KeyTile::kBytes};
            const uint32_t next = at + kSwept;
            if (next < end) fetch(there, next);
            const auto tile = [&](auto is_whole) {
                constexpr bool WHOLE = decltype(is_whole)::value;
                f32x16 scores[kSwept / 32];
#pragma unroll
                for (int b = 0; b < static_cast<int>(kSwept) / 32; b++) {
                    f32x16 s = {};
#pragma unroll
                    for (int n = 0; n < kOperands; n++) {
                        s = product(key_tile.by_row(lanes, b * 32, n), queries[n], s);
                    }
                    scores[b] = s;
                }
                if constexpr (!WHOLE) {
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
                    add_weighted<SIZE, kSwept, SLOW && !WHOLE>(special, acc, value_tile, b * 32, scores[b], lanes, lane, scratch[wave]);
                }
            };
            if (at >= all && at + kSwept - 1 <= wave_first) {
                tile(std::true_type());
            } else if (at < wave_first + 32 && at + kSwept > some) {
                tile(std::false_type());
            }
            if (next < end) land(there, next);
            at = next;
        };
        fetch(stage_0, at);
        land(stage_0, at);
        while (at < end) {
            if (!SLOW && special) return true;
            turn(stage_0, stage_1);
            if (!SLOW && special) return true;
            if (at < end) turn(stage_1, stage_0);
        }
        return false;
    };
    if (begin < end && sweep(std::false_type())) {
        __syncthreads();
        sweep(std::true_type());
    }
    total = halves_sum(total);
    if (token >= mine.end) return;
    // (A total of 0 within a sequence is of scores of -infinity alone: 0 / 0.)
    store_column<S, SIZE>(out + token * shape.out.token + head * shape.out.head, acc,
                          span.first == kNone ? 0.0f : 1.0f / total, shape.size, half);
    if (normalizers != nullptr && half == 0) {
        normalizers[uint64_t{head} * shape.tokens + token] =
            total == 0.0f ? -INFINITY : (most + log2f(total) - kForwardPower) * kLn2;
    }
}

// ---- backward ----------------------------------------------------------------------------

// sums[head][token] = do . o, 16 lanes a row of a head; and in f16 behind them
// |do|^2, as much room for the largest of it from each token on
// (`queries_kernel`), and |v|^2, [key head][token]; 0 where a square is no
// finite number.
// Bound by memory; 7001 f16 tokens of 12 heads of 80, 40 MB, 10.2 us (12.6 with
// do read for each of its two sums and places divided in 64 bits).
__global__ void __launch_bounds__(kThreads)
    dots_kernel(const Shape shape, const S* __restrict__ d_out, const S* __restrict__ out, const S* __restrict__ v,
                float* __restrict__ sums) {
    const uint64_t first = uint64_t{blockIdx.x} * (kThreads / 16) + threadIdx.x / 16;
    const uint64_t apart = uint64_t{gridDim.x} * (kThreads / 16);
    const uint64_t rows = uint64_t{shape.tokens} * shape.heads;
    const bool writes = threadIdx.x % 16 == 0;
    const auto finite = [](float square) { return square < INFINITY ? square : 0.0f; };
    // A row's place: 64 bits only divide where rows are that many.
    const auto place = [&](uint64_t row, uint32_t heads, Steps steps, uint32_t* token, uint32_t* head) {
        if (row >> 32 == 0) {
            *token = static_cast<uint32_t>(row) / heads, *head = static_cast<uint32_t>(row) % heads;
        } else {
            *token = static_cast<uint32_t>(row / heads), *head = static_cast<uint32_t>(row % heads);
        }
        return *token * steps.token + *head * steps.head;
    };
    uint32_t token, head;
    for (uint64_t row = first; row < rows; row += apart) {
        const uint64_t at = place(row, shape.heads, shape.out, &token, &head);
        float sum = 0.0f, square = 0.0f;
        for (uint32_t word = threadIdx.x % 16; word * E < shape.size; word += 16) {
            const Words<S, E> x{{head_word(d_out + at, word, shape.size)}}, y{{head_word(out + at, word, shape.size)}};
#pragma unroll
            for (int e = 0; e < E; e++) {
                sum = fmaf(x.at(e), y.at(e), sum);
                if constexpr (kHalf) square = fmaf(x.at(e), x.at(e), square);
            }
        }
        sum = row16<Added>(sum);
        const uint64_t to = uint64_t{head} * shape.tokens + token;
        if (writes) sums[to] = sum;
        if constexpr (kHalf) {
            square = row16<Added>(square);
            if (writes) sums[rows + to] = finite(square);
        }
    }
    if constexpr (kHalf) {
        const uint32_t heads = shape.heads / shape.group;
        for (uint64_t row = first; row < uint64_t{shape.tokens} * heads; row += apart) {
            const S* value = v + place(row, heads, shape.v, &token, &head);
            float square = 0.0f;
            for (uint32_t word = threadIdx.x % 16; word * E < shape.size; word += 16) {
                const Words<S, E> x{{head_word(value, word, shape.size)}};
#pragma unroll
                for (int e = 0; e < E; e++) square = fmaf(x.at(e), x.at(e), square);
            }
            square = row16<Added>(square);
            if (writes) sums[3 * rows + uint64_t{head} * shape.tokens + token] = finite(square);
        }
    }
}

// The largest of `values`, by token: among the tokens of a sequence up to each
// lane's own, or with BEHIND from it on.  The block has the 32 tokens of each
// wave from `first` on, and one sequence at most reaches past them there.
template <bool BEHIND>
__device__ __forceinline__ float most_of_sum(const Shape& shape, const float* __restrict__ values, uint32_t first,
                                             uint32_t token, const Span& span, float (*scratch)[8 * 32]) {
    const uint32_t wave = threadIdx.x / 64, column = threadIdx.x % 32;
    __shared__ uint32_t edge;
    if (threadIdx.x == (BEHIND ? kThreads - 1 : 0)) edge = BEHIND ? span.end : span.first;
    __syncthreads();
    const uint32_t from = BEHIND ? first + kOwned : edge, to = BEHIND ? edge : first;
    float past = 0.0f;
    if (from < to) {
#pragma unroll 8
        for (uint32_t i = from + threadIdx.x; i < to; i += kThreads) past = fmaxf(past, values[i]);
    }
    past = wave64<Largest>(past);
    float most = token < shape.tokens ? values[token] : 0.0f;
    for (uint32_t offset = 1; offset < 32; offset *= 2) {
        const float other = BEHIND ? __shfl_down(most, offset, 32) : __shfl_up(most, offset, 32);
        const bool seen = BEHIND ? column + offset < 32 && token + offset < span.end
                                 : column >= offset && token - offset >= span.first;
        if (seen) most = fmaxf(most, other);
    }
    float(&held)[8 * 32] = scratch[wave];
    if (threadIdx.x % 64 < 32) held[column] = most;
    if (threadIdx.x % 64 == 0) held[32] = past;
    __syncthreads();
    for (uint32_t w = 0; w < kThreads / 64; w++) {
        past = fmaxf(past, scratch[w][32]);
        if (BEHIND ? w > wave && first + w * 32 < span.end : w < wave && first + w * 32 + 31 >= span.first) {
            most = fmaxf(most, scratch[w][BEHIND ? 0 : 31]);
        }
    }
    __syncthreads();  // `scratch` is free
    return (BEHIND ? span.end > first + kOwned : span.first < first) ? fmaxf(most, past) : most;
}

// The power of two that ds of a sum are rounded times in f16, from the largest
// |do|^2 and |v|^2 among them: those of rows that are no part of the sum would
// take its bits.  7001 tokens, 12 heads of 80: 154 us, as with one power for all
// sums from a kernel of its own; 165 where the power followed each tile's ds
// (and 1773 against 1348 for 8192 tokens, 16 heads of 128, out of registers).
__device__ __forceinline__ float ds_factor(float d_square, float v_square) {
    const float bound = sqrtf(d_square) * sqrtf(v_square);
    return bound == 0.0f ? 1.0f : ldexpf(1.0f, 13 - ilogbf(bound));
}

// dq: as forward, with the weights from the normalizers.
template <int SIZE, bool DIRECT>
__global__ void __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(2)))
    queries_kernel(const Shape shape, const S* __restrict__ d_out, const S* __restrict__ q, const S* __restrict__ k,
                   const S* __restrict__ v, const float* __restrict__ normalizers, float* __restrict__ dots,
                   S* __restrict__ dq) {
    using KeyTile = Tile<SIZE, kSwept>;
    // A stage an array, so that reads of one do not wait for loads to the other.
    __shared__ __attribute__((aligned(1024))) char stage_0[2 * KeyTile::kBytes], stage_1[2 * KeyTile::kBytes];
    __shared__ float scratch[kThreads / 64][8 * 32];
    __shared__ uint32_t seen[2][kThreads / 64], marks[2];
    constexpr int kOperands = SIZE / kDeep;

    const int lane = threadIdx.x % 64, half = lane / 32, wave = threadIdx.x / 64;
    const Lanes lanes = KeyTile::lanes_of(lane);
    const uint32_t head = blockIdx.x % shape.heads;
    const Owned mine = owned_by<kThreads>(shape, kOwned, blockIdx.x / shape.heads, true);
    const uint32_t first = mine.first;
    if (first == kNone) return;
    const uint32_t wave_first = first + wave * 32;
    const uint32_t token = wave_first + lane % 32;
    // (Lanes past the block's tokens work as if they had one, for nothing.)
    const Span span = shape.by_sequence ? mine.span : span_of(shape, token);
    const uint32_t limit = shape.by_sequence ? mine.end : limit_of(shape);
    const uint32_t some = wave_least(span.first), all = wave_most(span.first);
    if (lane == 0) seen[0][wave] = some, seen[1][wave] = all;
    if (threadIdx.x < 2) marks[threadIdx.x] = 0;

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
    float dot = dots[uint64_t{head} * shape.tokens + inside];
    __syncthreads();
    uint32_t begin, block_all;
    over_waves(seen, &begin, &block_all);
    float factor = 1.0f;
    if constexpr (kHalf) {
        const uint64_t rows = uint64_t{shape.tokens} * shape.heads;
        const float* d_squares = dots + rows + uint64_t{head} * shape.tokens;
        const float* v_squares = dots + 3 * rows + uint64_t{head / shape.group} * shape.tokens;
        factor = ds_factor(d_squares[inside], most_of_sum<false>(shape, v_squares, first, token, span, scratch));
        dot *= factor;
        // For the kernel of dk and dv, which runs next.
        const float later = most_of_sum<true>(shape, d_squares, first, token, span, scratch);
        if (half == 0 && token < mine.end) dots[2 * rows + uint64_t{head} * shape.tokens + token] = later;
    }

    const S* keys = k + head / shape.group * shape.k.head;
    const S* values = v + head / shape.group * shape.v.head;
    const float c = shape.scale * kLog2e;
    f32x16 acc[SIZE / 32] = {};

    const uint32_t end = first + kOwned < limit ? first + kOwned : limit;
    // The first tokens of a sequence see few keys.  There o is as large as the
    // v_j, and what it lost when it was rounded to 16 bits weighs as much in
    // ds as ds's own rounding and more (2 tokens: dq off by 0.37%, where all
    // other roundings come to 0.23%; it falls with the root of the number of
    // keys).  So D of a sequence's first kOwned tokens is summed from the p_ij
    // and do_i . v_j, and left for the kernel of dk and dv, which runs next.
    if constexpr (!kWide) {
        const bool early = span.first != kNone && token >= span.first && token - span.first < kOwned;
        const uint32_t wave_early = wave_least(early ? span.first : kNone);
        __syncthreads();
        if (lane == 0) seen[0][wave] = wave_early;
        __syncthreads();
        uint32_t early_begin, unused;
        over_waves(seen, &early_begin, &unused);
        if (early_begin < end) {
            Stager<SIZE, kSwept, DIRECT> key_stager(shape.k.token, shape.size), value_stager(shape.v.token, shape.size);
            const KeyTile key_tile{stage_0}, value_tile{stage_0 + KeyTile::kBytes};
            float sum = 0.0f;
            for (uint32_t at = early_begin; at < end; at += kSwept) {
                key_stager.fetch(key_tile, keys, at, limit);
                value_stager.fetch(value_tile, values, at, limit);
                key_stager.land(key_tile);
                value_stager.land(value_tile);
                __syncthreads();
#pragma unroll 1
                for (int b = 0; b < static_cast<int>(kSwept) / 32; b++) {
                    f32x16 s = {}, d = {};
#pragma unroll
                    for (int n = 0; n < kOperands; n++) {
                        s = product(key_tile.by_row(lanes, b * 32, n), queries[n], s);
                        d = product(value_tile.by_row(lanes, b * 32, n), d_rows[n], d);
                    }
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        const uint32_t key = at + b * 32 + row_of(i, half);
                        const float weighted_dot = power2(fmaf(s[i], c, -normalizer)) * d[i];
                        if (key >= span.first && key <= token) sum += weighted_dot;
                    }
                }
                __syncthreads();
            }
            sum = halves_sum(sum);
            if (early) dot = sum * factor;
            if (early && half == 0 && token < mine.end) dots[uint64_t{head} * shape.tokens + token] = sum;
        }
    }
    // One sweep over the keys.  Without SLOW it ends, true, at the first masked
    // tile with a special value: what handles those is kept out of the sweep's
    // registers.
    const auto sweep = [&](auto is_slow) {
        constexpr bool SLOW = decltype(is_slow)::value;
#pragma unroll
        for (int t = 0; t < SIZE / 32; t++) acc[t] = f32x16{};
        // Masked for some query of the block (and the same for all its waves):
        // before a sequence's first key or past the first query.
        const auto masked = [&](uint32_t tile) { return tile < block_all || tile + kSwept - 1 > first; };
        Stager<SIZE, kSwept, DIRECT> key_stager(shape.k.token, shape.size), value_stager(shape.v.token, shape.size);
        uint32_t at = shape.by_sequence ? begin : begin / kSwept * kSwept;
        bool special = false;
        const auto fetch = [&](char* stage, uint32_t tile) {
            key_stager.fetch(KeyTile{stage}, keys, tile, limit);
            value_stager.fetch(KeyTile{stage + KeyTile::kBytes}, values, tile, limit);
        };
        const auto land = [&](char* stage, uint32_t tile) {
            key_stager.land(KeyTile{stage});
            value_stager.land(KeyTile{stage + KeyTile::kBytes});
            // What this thread fetched it may look at before the others have
            // theirs; a stage's mark names the tile, so that none is cleared.
            uint32_t& mark = marks[stage == stage_1];
            if (masked(tile) && specials_in<kThreads>(KeyTile{stage})) mark = tile + 1;
            __syncthreads();
            special = masked(tile) && __builtin_amdgcn_readfirstlane(mark) == tile + 1;
        };
        // The tile at `at` in stage `here`, while the next one is on its way.
        const auto turn = [&](char* here, char* there) {
            const KeyTile key_tile{here}, value_tile{here + KeyTile::kBytes};
            const uint32_t next = at + kSwept;
            if (next < end) fetch(there, next);
            const auto keys_of_32 = [&](int b, auto is_whole) {
                constexpr bool WHOLE = decltype(is_whole)::value;
                f32x16 s = {}, d = {};
#pragma unroll
                for (int n = 0; n < kOperands; n++) {
                    s = product(key_tile.by_row(lanes, b * 32, n), queries[n], s);
                    d = product(value_tile.by_row(lanes, b * 32, n), d_rows[n], d);
                }
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    s[i] = power2(fmaf(s[i], c, -normalizer)) * fmaf(d[i], factor, -dot);
                    if constexpr (!WHOLE) {
                        const uint32_t key = at + b * 32 + row_of(i, half);
                        if (key < span.first || key > token) s[i] = 0.0f;
                    }
                }
                add_weighted<SIZE, kSwept, SLOW && !WHOLE>(special, acc, key_tile, b * 32, s, lanes, lane, scratch[wave]);
            };
            if (at >= all && at + kSwept - 1 <= wave_first) {
#pragma unroll
                for (int b = 0; b < static_cast<int>(kSwept) / 32; b++) keys_of_32(b, std::true_type());
            } else if (at < wave_first + 32 && at + kSwept > some) {
#pragma unroll 1
                for (int b = 0; b < static_cast<int>(kSwept) / 32; b++) keys_of_32(b, std::false_type());
            }
            if (next < end) land(there, next);
            at = next;
        };
        fetch(stage_0, at);
        land(stage_0, at);
        while (at < end) {
            if (!SLOW && special) return true;
            turn(stage_0, stage_1);
            if (!SLOW && special) return true;
            if (at < end) turn(stage_1, stage_0);
        }
        return false;
    };
    if (begin < end && sweep(std::false_type())) {
        __syncthreads();
        sweep(std::true_type());
    }
    if (token >= mine.end) return;
    store_column<S, SIZE>(dq + token * shape.q.token + head * shape.q.head, acc, shape.scale / factor, shape.size, half);
}

// dk and dv of 128 keys from the queries of one of `splits` shares of the
// heads that the key head serves.  With several shares they are left in f32
// as `parts`[key head][share][dk, dv][token][size], to be added in their order.
// Threads of a block: a wave of 32 keys each, all that a compute unit holds
// where LDS leaves room for one block.  In the largest 16-bit heads it holds the
// values, so that registers let two waves share a matrix core: 8192 bf16 tokens,
// 16 heads of 128, 816 us with the values in registers and one wave, 776 with
// blocks of 128 keys and tiles of 32 queries, 675 so, all three timed as it was
// chosen (616 now).
constexpr int key_threads(int size) { return !kWide && size > 96 ? 512 : kThreads; }

template <int SIZE, bool DIRECT>
__global__ void __launch_bounds__(key_threads(SIZE)) __attribute__((amdgpu_waves_per_eu(kWide && SIZE > 96 ? 1 : 2)))
    keys_kernel(const Shape shape, uint32_t splits, const S* __restrict__ d_out, const S* __restrict__ q,
                const S* __restrict__ k, const S* __restrict__ v, const float* __restrict__ normalizers,
                const float* __restrict__ dots, S* __restrict__ dk, S* __restrict__ dv, float* __restrict__ parts) {
    constexpr bool kValuesInLds = SIZE > 96;
    constexpr int kWaves = key_threads(SIZE) / 64;
    constexpr uint32_t kKeys = 32 * kWaves;
    using QueryTile = Tile<SIZE, kSwept>;
    using ValueTile = Tile<SIZE, kKeys>;
    __shared__ __attribute__((aligned(1024))) char value_lds[kValuesInLds ? ValueTile::kBytes : 16];
    __shared__ __attribute__((aligned(1024))) char stage_0[2 * QueryTile::kBytes], stage_1[2 * QueryTile::kBytes];
    __shared__ __attribute__((aligned(16))) float values_0[2][kSwept], values_1[2][kSwept];
    __shared__ float scratch[kWaves][8 * 32];
    __shared__ uint32_t seen[2][kWaves], marks[2];
    constexpr int kOperands = SIZE / kDeep;

    const int lane = threadIdx.x % 64, half = lane / 32, wave = threadIdx.x / 64;
    const Lanes lanes = QueryTile::lanes_of(lane);
    // The first tokens, which are seen by the most queries, first.
    const uint32_t key_heads = shape.heads / shape.group;
    const uint32_t columns = key_heads * splits;
    const uint32_t key_head = blockIdx.x % columns / splits, share = blockIdx.x % splits;
    const uint32_t share_heads = shape.group / splits;
    const uint32_t first_head = key_head * shape.group + share * share_heads;
    const Owned mine = owned_by<key_threads(SIZE)>(shape, kKeys, blockIdx.x / columns, false);
    const uint32_t first = mine.first;
    if (first == kNone) return;
    const uint32_t wave_first = first + wave * 32;
    const uint32_t token = wave_first + lane % 32;
    // (Lanes past the block's tokens work as if they had one, for nothing.)
    const Span span = shape.by_sequence ? mine.span : span_of(shape, token);
    const uint32_t limit = shape.by_sequence ? mine.end : limit_of(shape);
    // Queries before which all, and some, of the wave's keys are seen.
    const uint32_t all = wave_least(span.end), some = wave_most(span.end);
    if (lane == 0) seen[0][wave] = all, seen[1][wave] = some;
    if (threadIdx.x < 2) marks[threadIdx.x] = 0;

    const uint32_t inside = token < shape.tokens ? token : 0;
    const S* key = k + inside * shape.k.token + key_head * shape.k.head;
    const S* value = v + inside * shape.v.token + key_head * shape.v.head;
    const ValueTile own_values{value_lds + wave * 32 * ValueTile::kWords * 16};  // each wave its own 32 rows
    uint4 keys[kOperands], values[kValuesInLds ? 1 : kOperands];
#pragma unroll
    for (int n = 0; n < kOperands; n++) {
        keys[n] = head_word(key, 2 * n + half, shape.size);
        const uint4 word = head_word(value, 2 * n + half, shape.size);
        if constexpr (kValuesInLds) {
            *reinterpret_cast<uint4*>(own_values.word(lane % 32, 2 * n + half)) = word;
        } else {
            values[n] = word;
        }
    }
    __syncthreads();
    uint32_t block_all, end;
    over_waves(seen, &block_all, &end);

    const float c = shape.scale * kLog2e;
    // p is rounded times 2^kBackPower, ds times `factor`.
    float factor = 1.0f;
    if constexpr (kHalf) {
        const uint64_t rows = uint64_t{shape.tokens} * shape.heads;
        float d_square = 0.0f;
        for (uint32_t h = first_head; h < first_head + share_heads; h++) {
            d_square = fmaxf(d_square, dots[2 * rows + uint64_t{h} * shape.tokens + inside]);
        }
        factor = ds_factor(d_square, dots[3 * rows + uint64_t{key_head} * shape.tokens + inside]);
    }
    const float ds_scale = factor * power2(-kBackPower);
    f32x16 acc_k[SIZE / 32] = {}, acc_v[SIZE / 32] = {};
    // One sweep over the queries, as over the keys in the kernels above.
    const auto sweep = [&](auto is_slow) {
        constexpr bool SLOW = decltype(is_slow)::value;
#pragma unroll
        for (int t = 0; t < SIZE / 32; t++) acc_k[t] = f32x16{}, acc_v[t] = f32x16{};
        Stager<SIZE, kSwept, DIRECT, key_threads(SIZE)> query_stager(shape.q.token, shape.size), d_stager(shape.out.token, shape.size);
        float row_value = 0.0f;  // of one row: threads below kSwept the normalizer, the next ones the dot
        const uint32_t per_head = (end - first + kSwept - 1) / kSwept;
        const uint32_t turns = per_head * share_heads;
        bool special = false;
        // Masked for some key of the block: before its last key, or past a
        // sequence's end.
        const auto masked = [&](uint32_t at) { return at < first + kKeys - 1 || at + kSwept > block_all; };
        const auto tile_of = [&](uint32_t n) { return first + n % per_head * kSwept; };
        const auto fetch = [&](char* stage, uint32_t n) {
            const uint32_t head = first_head + n / per_head, at = tile_of(n);
            query_stager.fetch(QueryTile{stage}, q + head * shape.q.head, at, limit);
            d_stager.fetch(QueryTile{stage + QueryTile::kBytes}, d_out + head * shape.out.head, at, limit);
            if (threadIdx.x < 2 * kSwept) {
                const uint32_t row = at + threadIdx.x % kSwept;
                const float* from = threadIdx.x < kSwept ? normalizers : dots;
                row_value = row < limit ? from[uint64_t{head} * shape.tokens + row] : 0.0f;
            }
        };
        const auto land = [&](char* stage, float (&values_here)[2][kSwept], uint32_t n) {
            query_stager.land(QueryTile{stage});
            d_stager.land(QueryTile{stage + QueryTile::kBytes});
            if (threadIdx.x < 2 * kSwept) {
                if (threadIdx.x < kSwept) row_value = fmaf(row_value, kLog2e, -kBackPower);
                values_here[threadIdx.x / kSwept][threadIdx.x % kSwept] = row_value;
            }
            uint32_t& mark = marks[stage == stage_1];
            if (masked(tile_of(n)) && (specials_in<key_threads(SIZE)>(QueryTile{stage}) ||
                                       specials_in<key_threads(SIZE)>(QueryTile{stage + QueryTile::kBytes}))) {
                mark = n + 1;
            }
            __syncthreads();
            special = masked(tile_of(n)) && __builtin_amdgcn_readfirstlane(mark) == n + 1;
        };
        uint32_t n = 0;
        const auto turn = [&](char* here, const float (&row_values)[2][kSwept], char* there,
                              float (&values_there)[2][kSwept]) {
            const uint32_t at = tile_of(n);
            const QueryTile query_tile{here}, d_tile{here + QueryTile::kBytes};
            if (n + 1 < turns) fetch(there, n + 1);
            const auto rows_of_32 = [&](int b, auto is_whole) {
                constexpr bool WHOLE = decltype(is_whole)::value;
                f32x16 s = {}, d = {};
#pragma unroll
                for (int o = 0; o < kOperands; o++) {
                    s = product(query_tile.by_row(lanes, b * 32, o), keys[o], s);
                    if constexpr (kValuesInLds) {
                        d = product(d_tile.by_row(lanes, b * 32, o), own_values.by_row(lanes, 0, o), d);
                    } else {
                        d = product(d_tile.by_row(lanes, b * 32, o), values[o], d);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int g = 0; g < 4; g++) {
                    const int row = b * 32 + 8 * g + 4 * half;
                    const float4 normalizer = *reinterpret_cast<const float4*>(&row_values[0][row]);
                    const float4 dot = *reinterpret_cast<const float4*>(&row_values[1][row]);
                    const float l[4] = {normalizer.x, normalizer.y, normalizer.z, normalizer.w};
                    const float o[4] = {dot.x, dot.y, dot.z, dot.w};
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const int i = 4 * g + j;
                        s[i] = power2(fmaf(s[i], c, -l[j]));
                        d[i] = s[i] * (d[i] - o[j]);
                        if constexpr (kHalf) d[i] *= ds_scale;
                        if constexpr (!WHOLE) {
                            const uint32_t query = at + b * 32 + row_of(i, half);
                            if (query < token || query >= span.end) s[i] = 0.0f, d[i] = 0.0f;
                        }
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
                add_weighted<SIZE, kSwept, SLOW && !WHOLE>(special, acc_v, d_tile, b * 32, s, lanes, lane, scratch[wave]);
                __builtin_amdgcn_sched_barrier(0);
                add_weighted<SIZE, kSwept, SLOW && !WHOLE>(special, acc_k, query_tile, b * 32, d, lanes, lane, scratch[wave]);
            };
            // 32 rows at a time, whole or masked: the scores and do . v of 64
            // would take 32 registers more.
            if (at >= wave_first + 31 && at + kSwept <= all) {
#pragma unroll 1
                for (int b = 0; b < static_cast<int>(kSwept) / 32; b++) rows_of_32(b, std::true_type());
            } else if (at + kSwept > wave_first && at < some) {
#pragma unroll 1
                for (int b = 0; b < static_cast<int>(kSwept) / 32; b++) rows_of_32(b, std::false_type());
            }
            if (n + 1 < turns) land(there, values_there, n + 1);
            n++;
        };
        fetch(stage_0, 0);
        land(stage_0, values_0, 0);
        while (n < turns) {
            if (!SLOW && special) return true;
            turn(stage_0, values_0, stage_1, values_1);
            if (!SLOW && special) return true;
            if (n < turns) turn(stage_1, values_1, stage_0, values_0);
        }
        return false;
    };
    if (first < end && sweep(std::false_type())) {
        __syncthreads();
        sweep(std::true_type());
    }
    if (token >= mine.end) return;
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

// Whether tiles of these rows may be loaded straight to LDS: whole aligned
// words, and a tile within 31 bits of its first byte.
bool direct(uint32_t size, std::initializer_list<std::pair<const void*, Steps>> operands) {
    bool all = size % E == 0;
    for (const auto& operand : operands) {
        all = all && aligned16(operand.first) && operand.second.token % E == 0 && operand.second.head % E == 0 &&
              operand.second.token < (uint64_t{1} << 31) / (kSwept * sizeof(S));
    }
    return all;
}

// The body with SIZE, the head size rounded up to 32, and DIRECT.
#define TC_ATTENTION_SIZE(size, ...)                    \
    if (size <= 32) {                                   \
        constexpr int SIZE = 32; __VA_ARGS__;           \
    } else if (size <= 64) {                            \
        constexpr int SIZE = 64; __VA_ARGS__;           \
    } else if (size <= 96) {                            \
        constexpr int SIZE = 96; __VA_ARGS__;           \
    } else {                                            \
        constexpr int SIZE = 128; __VA_ARGS__;          \
    }
#define TC_ATTENTION_FORM(size, is_direct, ...)                                      \
    if (is_direct) {                                                                 \
        constexpr bool DIRECT = true; TC_ATTENTION_SIZE(size, __VA_ARGS__)           \
    } else {                                                                         \
        constexpr bool DIRECT = false; TC_ATTENTION_SIZE(size, __VA_ARGS__)          \
    }

// At most as many tiles of `owned` tokens as `owned_by` finds.
uint32_t tiles_of(const Shape& shape, uint32_t owned) {
    const uint32_t tiles = (shape.tokens + owned - 1) / owned;
    return shape.by_sequence ? tiles + shape.sequences + 2 : tiles;
}

int forward(const Shape& shape, const void* q, const void* k, const void* v, void* out, float* normalizers) {
    TC_STREAM(s);
    const uint32_t tiles = tiles_of(shape, kOwned);
    const bool straight = direct(shape.size, {{k, shape.k}, {v, shape.v}});
    TC_ATTENTION_FORM(shape.size, straight,
                      forward_kernel<SIZE, DIRECT><<<tiles * shape.heads, kThreads, 0, s>>>(
                          shape, static_cast<const S*>(q), static_cast<const S*>(k), static_cast<const S*>(v),
                          static_cast<S*>(out), normalizers))
    return check_launch("attention");
}

int backward(const Shape& shape, const void* d_out, const void* q, const void* k, const void* v, const void* out,
             const float* normalizers, void* dq, void* dk, void* dv) {
    TC_STREAM(s);
    const char* what = "attention, backward";
    const uint32_t tiles = tiles_of(shape, kOwned);
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
    Scratch dots((kHalf ? 3 * rows + uint64_t{shape.tokens} * key_heads : rows) * sizeof(float));
    Scratch parts(splits > 1 ? uint64_t{key_heads} * splits * 2 * shape.tokens * shape.size * sizeof(float) : 0);
    if (dots.status != TC_OK) return dots.status;
    if (parts.status != TC_OK) return parts.status;
    float* sums = static_cast<float*>(dots.ptr);
    const S* d = static_cast<const S*>(d_out);
    const S* queries = static_cast<const S*>(q);
    const S* keys = static_cast<const S*>(k);
    const S* values = static_cast<const S*>(v);
    dots_kernel<<<grid_for(rows, kThreads / 16, 8), kThreads, 0, s>>>(shape, d, static_cast<const S*>(out), values,
                                                                      sums);
    int status = check_launch(what);
    if (status != TC_OK) return status;
    const bool keys_straight = direct(shape.size, {{k, shape.k}, {v, shape.v}});
    TC_ATTENTION_FORM(shape.size, keys_straight,
                      queries_kernel<SIZE, DIRECT><<<tiles * shape.heads, kThreads, 0, s>>>(
                          shape, d, queries, keys, values, normalizers, sums, static_cast<S*>(dq)))
    status = check_launch(what);
    if (status != TC_OK) return status;
    const bool rows_straight = direct(shape.size, {{q, shape.q}, {d_out, shape.out}});
    TC_ATTENTION_FORM(shape.size, rows_straight,
                      const uint32_t key_tiles = tiles_of(shape, key_threads(SIZE) / 2);
                      keys_kernel<SIZE, DIRECT><<<key_tiles * key_heads * splits, key_threads(SIZE), 0, s>>>(
                          shape, splits, d, queries, keys, values, normalizers, sums, static_cast<S*>(dk),
                          static_cast<S*>(dv), static_cast<float*>(parts.ptr)))
    status = check_launch(what);
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
