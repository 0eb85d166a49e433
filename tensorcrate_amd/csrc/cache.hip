// A cache of keys and values in pages: the checks of its calls, and the rows of
// new tokens written into it and read back.
//
// In 8 bits a row x is kept as whole numbers q with a scale of its own:
//   s = max|x| / 127,  q = round(x / s),  read as q s,
// in 32 bits, each operation rounded as IEEE says, so that any other program
// that computes it gets the same numbers.  (At 8 bits a row, whole numbers
// with a scale are off by at most max|x| / 254 each; the 8-bit floats with
// three bits of fraction by up to |x| / 16.)
//
// Bound by memory, or for a few tokens by the chain of reads that finds a
// row's place (offsets, length, page).  A block takes a few tokens' rows, so
// that this chain is walked once for many of them: 16 lanes hold a row, 8
// elements each, and the largest magnitude is taken in registers.  A key's row
// and a value's go together, two such pairs in flight.
//   Measured: 25000 tokens of 8 heads of 128, f16 kept in 8 bits, written in 41
// us and read in 28 (82 us together with one row at a time); 64 tokens in bf16
// 4.3 and 3.4, which is a launch and the chain.

#include "cache.hpp"

namespace tc {
namespace cache {

int check_pool(const std::string& what, const tc_cache* given, Pool* pool) {
    if (given == nullptr) return fail(TC_INVALID, what + ": no cache");
    const tc_cache& c = *given;
    if (dtype_size(c.dtype) == 0 || c.dtype == TC_F64) {
        return fail(TC_UNSUPPORTED, what + ": no kernel for " + dtype_name(c.dtype));
    }
    if (c.format != TC_CACHE_PLAIN && c.format != TC_CACHE_INT8) {
        return fail(TC_INVALID, what + ": a cache of format " + std::to_string(c.format));
    }
    if (c.key_heads == 0 || c.head_size == 0) return fail(TC_INVALID, what + ": heads of no elements");
    if (c.head_size > 128) {
        return fail(TC_UNSUPPORTED, what + ": heads of " + std::to_string(c.head_size) + " elements, more than 128");
    }
    if (c.key_heads > (1u << 24)) {  // twice as many rows of a block's tokens are counted in 32 bits
        return fail(TC_UNSUPPORTED, what + ": " + std::to_string(c.key_heads) + " key heads");
    }
    if (c.page_size == 0) return fail(TC_INVALID, what + ": pages of no tokens");
    uint64_t rows = 0;
    if (__builtin_mul_overflow(uint64_t{c.page_count} * c.key_heads, uint64_t{c.page_size}, &rows) ||
        rows >= (uint64_t{1} << 32)) {
        return fail(TC_UNSUPPORTED, what + ": " + std::to_string(c.page_count) + " pages of " +
                                        std::to_string(c.page_size) + " tokens of " + std::to_string(c.key_heads) +
                                        " heads");
    }
    const uint32_t word = c.format == TC_CACHE_INT8 ? 16 : 16 / static_cast<uint32_t>(dtype_size(c.dtype));
    *pool = Pool{c.key_heads,
                 c.head_size,
                 (c.head_size + word - 1) / word * word,
                 c.page_size,
                 c.page_count,
                 DivMod(c.page_size),
                 c.keys,
                 c.values,
                 c.key_scales,
                 c.value_scales};
    return TC_OK;
}

int check_batch(const std::string& what, const tc_cache_batch* given, const Pool& pool, Batch* batch) {
    if (given == nullptr) return fail(TC_INVALID, what + ": no batch");
    const tc_cache_batch& b = *given;
    if (b.tokens > 0x7fffff00u || b.sequences > 0xffffffu) {
        return fail(TC_UNSUPPORTED, what + ": " + std::to_string(b.tokens) + " tokens of " +
                                        std::to_string(b.sequences) + " sequences");
    }
    if (b.offsets == nullptr && b.tokens != b.sequences) {
        return fail(TC_INVALID, what + ": " + std::to_string(b.tokens) + " tokens of " + std::to_string(b.sequences) +
                                    " sequences without offsets");
    }
    // Keys are counted in 32 bits with room for some tiles behind them.
    if (uint64_t{b.most_pages} * pool.page_size > 0xfffff000u || b.prefix_length > 0xfffff000u) {
        return fail(TC_UNSUPPORTED, what + ": sequences of " + std::to_string(b.most_pages) + " pages of " +
                                        std::to_string(pool.page_size) + " tokens behind a prefix of " +
                                        std::to_string(b.prefix_length));
    }
    if (b.tokens > 0 && b.sequences > 0 && (b.lengths == nullptr || (b.most_pages > 0 && b.pages == nullptr))) {
        return null_operand(what.c_str());
    }
    if (b.tokens > 0 && b.prefix_length > 0 && b.prefix_pages == nullptr) return null_operand(what.c_str());
    *batch = Batch{static_cast<uint32_t>(b.tokens), b.sequences, b.most_pages, b.prefix_length, b.offsets, b.lengths,
                   b.pages, b.prefix_pages};
    return TC_OK;
}

namespace {

constexpr int kThreads = 256;
constexpr int kGroups = kThreads / 16;  // rows that a block holds at a time
constexpr int kAtOnce = 2;  // pairs of rows whose loads a lane has in flight

// Where the call's rows lie outside the cache.
template <typename P>
struct Rows {
    P key, value;
    Steps key_steps, value_steps;
};

struct LargestBits {
    __device__ static float join(float a, float b) {
        const uint32_t x = __float_as_uint(a), y = __float_as_uint(b);
        return __uint_as_float(x > y ? x : y);
    }
};

// Elements 8 lane .. 8 lane + 8 of a row of `size`, as `tail_of` leaves them.
// Words that reach past the row are taken from its last elements on instead, in
// all lanes alike: a branch that zeroes registers, or takes elements one by one,
// waits for all loads before it (3 sequences to 9000 tokens of 3 f32 heads of 75,
// written and read: 41.9 us so, 39.1 this way).
template <typename S>
__device__ __forceinline__ void load_eight(const S* row, uint32_t lane, uint32_t size, Words<S, 8>& out) {
    constexpr uint32_t E = kWordElements<S>;
    if (size >= E) {
#pragma unroll
        for (int w = 0; w < Words<S, 8>::kCount; w++) {
            const uint32_t at = 8 * lane + w * E;
            out.w[w] = load_any_word<false>(row + (at + E <= size ? at : size - E));
        }
    } else {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = 8 * lane + e < size ? Elem<S>::widen(row[8 * lane + e]) : 0.0f;
        out.put(v);
    }
}
// What `load_eight` has brought, with zeros behind the row.
template <typename S>
__device__ __forceinline__ void tail_of(uint32_t lane, uint32_t size, Words<S, 8>& words) {
    constexpr uint32_t E = kWordElements<S>;
    if (size < E || size == 128) return;
#pragma unroll
    for (int w = 0; w < Words<S, 8>::kCount; w++) {
        // Elements that the word begins too early.
        const uint32_t at = 8 * lane + w * E, early = at + E <= size ? 0 : at + E - size;
        uint4 v = words.w[w];
        const uint32_t whole = early * sizeof(S) / 4;  // 32-bit parts
        if constexpr (sizeof(S) == 2) {
            const uint32_t half = early % 2 * 16;
            v = make_uint4(__builtin_amdgcn_alignbit(v.y, v.x, half), __builtin_amdgcn_alignbit(v.z, v.y, half),
                           __builtin_amdgcn_alignbit(v.w, v.z, half), v.w >> half);
        }
        if (whole & 1) v = make_uint4(v.y, v.z, v.w, 0);
        if (whole & 2) v = make_uint4(v.z, v.w, 0, 0);
        words.w[w] = whole >= 4 ? make_uint4(0, 0, 0, 0) : v;
    }
}
template <typename S>
__device__ __forceinline__ void store_eight(S* row, uint32_t lane, uint32_t size, const Words<S, 8>& words) {
    if (8 * lane + 8 <= size) {
        words.template store<false>(row + 8 * lane);
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) {
            if (8 * lane + e < size) row[8 * lane + e] = Elem<S>::narrow(words.at(e));
        }
    }
}

// The row of a token's first head in the pool, kNowhere if the token has no
// place; `sequence` has it, `end` is past the sequence's last token here.
__device__ __forceinline__ uint32_t row_of_token(const Pool& pool, const Batch& batch, uint32_t sequence, uint32_t token,
                                                 uint32_t end) {
    if (sequence == kNowhere) return kNowhere;
    // The sequence's tokens here are its last.
    const uint32_t length = batch.lengths[sequence], left = end - token;
    if (length < left) return kNowhere;
    return row_of(pool, batch.pages + uint64_t{sequence} * batch.most_pages, batch.most_pages, 0, length - left);
}

constexpr uint32_t kMostTokens = 8;  // of a block at a time

// A block's tokens at a time, and the row in the pool of each one's first head:
// of a single token found by each wave, of several by a thread each, which goes
// on from the first token's sequence (each step a read that the next one waits
// for, so that few of them count more than many lanes).
struct Tokens {
    uint64_t first;
    uint32_t here;

    __device__ __forceinline__ void find(const Pool& pool, const Batch& batch, uint32_t per_block, uint32_t* found,
                                         uint32_t* only) const {
        Span span{0, 0};
        uint32_t token = static_cast<uint32_t>(first);
        if (per_block == 1) {
            const uint32_t sequence = wave_sequence_of(batch, token, &span);
            *only = row_of_token(pool, batch, sequence, token, span.end);
            return;
        }
        __syncthreads();
        if (threadIdx.x < 64) {
            uint32_t sequence = wave_sequence_of(batch, token, &span);
            if (threadIdx.x < here) {
                token += threadIdx.x;
                if (sequence != kNowhere && token >= span.end && sequence + 1 < batch.sequences) {
                    sequence++;
                    span = span_of(batch, sequence);
                }
                if (sequence == kNowhere || token < span.first || token >= span.end) {
                    sequence = sequence_of(batch, token, &span);
                }
                found[threadIdx.x] = row_of_token(pool, batch, sequence, token, span.end);
            }
        }
        __syncthreads();
    }
};

// The largest magnitude's bits of 8 elements, in 32 bits: past those of the
// largest finite number where one is an infinity or a NaN.
template <typename S>
__device__ __forceinline__ float largest_of(const Words<S, 8>& words) {
    const uint32_t* const w = reinterpret_cast<const uint32_t*>(words.w);
    if constexpr (sizeof(S) == 2) {
        typedef uint16_t pair __attribute__((ext_vector_type(2)));
        pair most = __builtin_bit_cast(pair, w[0] & 0x7fff7fffu);
#pragma unroll
        for (int n = 1; n < 4; n++) most = __builtin_elementwise_max(most, __builtin_bit_cast(pair, w[n] & 0x7fff7fffu));
        const uint16_t bits = most.x > most.y ? most.x : most.y;
        return Elem<S>::widen(__builtin_bit_cast(S, bits));
    } else {
        float most = 0.0f;
#pragma unroll
        for (int n = 0; n < 8; n++) most = LargestBits::join(most, __uint_as_float(w[n] & 0x7fffffffu));
        return most;
    }
}

// round(v / scale) as 8 whole numbers of 8 bits.  The quotients' nearest whole
// numbers are those of the products with an approximate reciprocal, which are
// off by less than 127 * 2^-22, unless one lies next to the middle of two: then,
// and where the reciprocal is no number, the quotients themselves are rounded.
// Adding 1.5 * 2^23 rounds to a whole number, ties to even, and leaves it in the
// sum's last bits.  (Quotients alone took 56 us for 16001 tokens of 16 rows of
// 128 f16 elements.)
__device__ __forceinline__ uint2 quantised(const float (&v)[8], float scale) {
    constexpr float kWhole = 12582912.0f;
    const float reciprocal = __builtin_amdgcn_rcpf(scale);
    uint32_t bits[8];
    float off = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const float t = v[e] * reciprocal, sum = t + kWhole;
        bits[e] = __float_as_uint(sum);
        off = fmaxf(off, fabsf(t - (sum - kWhole)));
    }
    // (With a scale of 2^-120 or more the reciprocal is a normal number.)
    if (!(scale >= 0x1p-120f) || off > 0.49995f) {
        const bool some = scale > 0.0f;  // neither 0 nor a NaN
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float q = some ? fminf(fmaxf(rintf(v[e] / scale), -127.0f), 127.0f) : 0.0f;
            bits[e] = static_cast<uint32_t>(static_cast<int>(q));
        }
    }
    // The last bytes of four, in order.
    const auto four = [&](int n) {
        return __builtin_amdgcn_perm(bits[n + 1], bits[n], 0x0c0c0400u) |
               __builtin_amdgcn_perm(bits[n + 3], bits[n + 2], 0x04000c0cu);
    };
    return make_uint2(four(0), four(4));
}

// Both rows of a token's head at a time, that of its key and that of its value:
// their place in the pool is the same.
template <typename S, bool QUANT>
__global__ void __launch_bounds__(kThreads)
    write_kernel(const Pool pool, const Batch batch, const Rows<const S*> rows, uint32_t per_block) {
    __shared__ uint32_t found[kMostTokens];
    const uint32_t lane = threadIdx.x % 16, group = threadIdx.x / 16;
    const Steps steps[2] = {rows.key_steps, rows.value_steps};
    for (uint64_t first = uint64_t{blockIdx.x} * per_block; first < batch.tokens; first += uint64_t{gridDim.x} * per_block) {
        const Tokens tokens{first, static_cast<uint32_t>(batch.tokens - first < per_block ? batch.tokens - first : per_block)};
        uint32_t only = kNowhere;
        RowWalk<2, kGroups> from(pool.heads, steps, group, first), to = from;
        Words<S, 8> keys[kAtOnce], values[kAtOnce];
        const auto load = [&]() {
#pragma unroll
            for (int k = 0; k < kAtOnce; k++, from.move()) {
                if (from.token >= tokens.here) continue;
                load_eight(rows.key + from.at[0], lane, pool.size, keys[k]);
                load_eight(rows.value + from.at[1], lane, pool.size, values[k]);
            }
        };
        const auto put = [&](const Words<S, 8>& words, void* entries, float* scales, uint32_t row) {
            if constexpr (QUANT) {
                const float most = row16<LargestBits>(largest_of(words));
                const bool finite = __float_as_uint(most) < 0x7f800000u;
                const float scale = finite ? most / 127.0f : __uint_as_float(0x7fc00000u);
                float v[8];
                words.get(v);
                const uint2 packed = quantised(v, scale);
                if (8 * lane < pool.row) {
                    *reinterpret_cast<uint2*>(static_cast<char*>(entries) + uint64_t{row} * pool.row + 8 * lane) = packed;
                }
                if (lane == 0) scales[row] = scale;
            } else {
                S* const at_row = static_cast<S*>(entries) + uint64_t{row} * pool.row + 8 * lane;
#pragma unroll
                for (int w = 0; w < Words<S, 8>::kCount; w++) {
                    if (8 * lane + w * kWordElements<S> < pool.row) {
                        store_word<false>(at_row + w * kWordElements<S>, words.w[w]);
                    }
                }
            }
        };
        // (The places are found while the first rows are on their way.)
        load();
        tokens.find(pool, batch, per_block, found, &only);
        while (to.token < tokens.here) {
#pragma unroll
            for (int k = 0; k < kAtOnce; k++, to.move()) {
                if (to.token >= tokens.here) continue;
                const uint32_t at = per_block == 1 ? only : found[to.token];
                if (at == kNowhere) continue;
                const uint32_t row = at + to.head * pool.page_size;
                tail_of(lane, pool.size, keys[k]);
                tail_of(lane, pool.size, values[k]);
                put(keys[k], pool.keys, pool.key_scales, row);
                put(values[k], pool.values, pool.value_scales, row);
            }
            if (to.token < tokens.here) load();
        }
    }
}

template <typename S, bool QUANT>
__global__ void __launch_bounds__(kThreads)
    read_kernel(const Pool pool, const Batch batch, const Rows<S*> rows, uint32_t per_block) {
    __shared__ uint32_t found[kMostTokens];
    const uint32_t lane = threadIdx.x % 16, group = threadIdx.x / 16;
    const Steps steps[2] = {rows.key_steps, rows.value_steps};
    struct Entries {
        Words<S, 8> words;
        uint2 packed;
        float scale;
    };
    const auto get = [&](const void* entries, const float* scales, uint32_t row, bool some, Entries& out) {
        out.packed = make_uint2(0, 0), out.scale = 0.0f;
#pragma unroll
        for (int w = 0; w < Words<S, 8>::kCount; w++) out.words.w[w] = make_uint4(0, 0, 0, 0);
        if (!some) return;
        if constexpr (QUANT) {
            if (8 * lane < pool.row) {
                out.packed = *reinterpret_cast<const uint2*>(static_cast<const char*>(entries) + uint64_t{row} * pool.row +
                                                             8 * lane);
            }
            out.scale = scales[row];
        } else {
            const S* const at_row = static_cast<const S*>(entries) + uint64_t{row} * pool.row + 8 * lane;
#pragma unroll
            for (int w = 0; w < Words<S, 8>::kCount; w++) {
                if (8 * lane + w * kWordElements<S> < pool.row) {
                    out.words.w[w] = load_word<false>(at_row + w * kWordElements<S>);
                }
            }
        }
    };
    const auto put = [&](Entries& in, S* row) {
        if constexpr (QUANT) {
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const uint32_t four = e < 4 ? in.packed.x : in.packed.y;
                v[e] = static_cast<float>(static_cast<int8_t>(four >> (8 * (e % 4)))) * in.scale;
            }
            in.words.put(v);
        }
        store_eight(row, lane, pool.size, in.words);
    };
    for (uint64_t first = uint64_t{blockIdx.x} * per_block; first < batch.tokens; first += uint64_t{gridDim.x} * per_block) {
        const Tokens tokens{first, static_cast<uint32_t>(batch.tokens - first < per_block ? batch.tokens - first : per_block)};
        uint32_t only = kNowhere;
        tokens.find(pool, batch, per_block, found, &only);
        RowWalk<2, kGroups> from(pool.heads, steps, group, first), to = from;
        while (to.token < tokens.here) {
            Entries keys[kAtOnce], values[kAtOnce];
#pragma unroll
            for (int k = 0; k < kAtOnce; k++, from.move()) {
                const uint32_t at = from.token >= tokens.here ? kNowhere : per_block == 1 ? only : found[from.token];
                const uint32_t row = at + from.head * pool.page_size;
                get(pool.keys, pool.key_scales, row, at != kNowhere, keys[k]);
                get(pool.values, pool.value_scales, row, at != kNowhere, values[k]);
            }
#pragma unroll
            for (int k = 0; k < kAtOnce; k++, to.move()) {
                if (to.token >= tokens.here) continue;
                put(keys[k], rows.key + to.at[0]);
                put(values[k], rows.value + to.at[1]);
            }
        }
    }
}

// The tokens of a block at a time: one where tokens are few, several where
// blocks of them fill the chip.  (25000 tokens written and read in 69 us, one at a
// time in 114; 64 tokens in 8, eight at a time in 15.)
uint32_t per_block_of(const Batch& batch) {
    return batch.tokens >= static_cast<uint32_t>(compute_units()) * 2 * kMostTokens ? kMostTokens : 1;
}

// What both calls check; `*nothing` if there is nothing to do.
int check(const char* what, const tc_cache* cache, const tc_cache_batch* given, const void* key, Steps key_steps,
          const void* value, Steps value_steps, Pool* pool, Batch* batch, bool* nothing) {
    int status = check_pool(what, cache, pool);
    if (status == TC_OK) status = check_batch(what, given, *pool, batch);
    if (status == TC_OK) status = check_heads(what, "keys", key_steps, pool->heads, batch->tokens, pool->size);
    if (status == TC_OK) status = check_heads(what, "values", value_steps, pool->heads, batch->tokens, pool->size);
    if (status != TC_OK) return status;
    *nothing = batch->tokens == 0;
    if (!*nothing && any_null({key, value})) return null_operand(what);
    return TC_OK;
}

}  // namespace

// The pool's own pointers, of a call that reads or writes it.
int check_storage(const std::string& what, const tc_cache& cache, const Pool& pool) {
    if (pool.page_count == 0) return TC_OK;
    if (any_null({cache.keys, cache.values}) ||
        (cache.format == TC_CACHE_INT8 && any_null({cache.key_scales, cache.value_scales}))) {
        return null_operand(what.c_str());
    }
    if (!aligned16(cache.keys) || !aligned16(cache.values)) {
        return fail(TC_INVALID, what + ": keys or values that are not 16-byte aligned");
    }
    return TC_OK;
}

}  // namespace cache
}  // namespace tc

using namespace tc;

extern "C" {

int tc_cache_bytes(const tc_cache* cache, uint64_t* entries, uint64_t* scales) {
    cache::Pool pool;
    const int status = cache::check_pool("cache", cache, &pool);
    if (status != TC_OK) return status;
    if (entries == nullptr || scales == nullptr) return null_operand("cache");
    const bool quant = cache->format == TC_CACHE_INT8;
    const uint64_t rows = uint64_t{pool.page_count} * pool.heads * pool.page_size;
    *entries = rows * pool.row * (quant ? 1 : dtype_size(cache->dtype));
    *scales = quant ? rows * sizeof(float) : 0;
    return TC_OK;
}

int tc_cache_write(const tc_cache* cache, const tc_cache_batch* batch, const void* key, uint64_t key_token_step,
                   uint64_t key_head_step, const void* value, uint64_t value_token_step, uint64_t value_head_step) {
    const char* what = "cache write";
    const Steps key_steps{key_token_step, key_head_step}, value_steps{value_token_step, value_head_step};
    cache::Pool pool;
    cache::Batch checked;
    bool nothing = false;
    int status = cache::check(what, cache, batch, key, key_steps, value, value_steps, &pool, &checked, &nothing);
    if (status == TC_OK) status = cache::check_storage(what, *cache, pool);
    if (status != TC_OK || nothing) return status;
    TC_STREAM(s);
    const uint32_t per_block = cache::per_block_of(checked);
    const uint32_t blocks = grid_for(checked.tokens, per_block, 32);
    TC_DISPATCH_FLOAT(cache->dtype, what, S, {
        const cache::Rows<const S*> rows{static_cast<const S*>(key), static_cast<const S*>(value), key_steps,
                                         value_steps};
        if (cache->format == TC_CACHE_INT8) {
            cache::write_kernel<S, true><<<blocks, cache::kThreads, 0, s>>>(pool, checked, rows, per_block);
        } else {
            cache::write_kernel<S, false><<<blocks, cache::kThreads, 0, s>>>(pool, checked, rows, per_block);
        }
    })
    return check_launch(what);
}

int tc_cache_read(const tc_cache* cache, const tc_cache_batch* batch, void* key, uint64_t key_token_step,
                  uint64_t key_head_step, void* value, uint64_t value_token_step, uint64_t value_head_step) {
    const char* what = "cache read";
    const Steps key_steps{key_token_step, key_head_step}, value_steps{value_token_step, value_head_step};
    cache::Pool pool;
    cache::Batch checked;
    bool nothing = false;
    int status = cache::check(what, cache, batch, key, key_steps, value, value_steps, &pool, &checked, &nothing);
    if (status == TC_OK) status = cache::check_storage(what, *cache, pool);
    if (status != TC_OK || nothing) return status;
    TC_STREAM(s);
    const uint32_t per_block = cache::per_block_of(checked);
    const uint32_t blocks = grid_for(checked.tokens, per_block, 32);
    TC_DISPATCH_FLOAT(cache->dtype, what, S, {
        const cache::Rows<S*> rows{static_cast<S*>(key), static_cast<S*>(value), key_steps, value_steps};
        if (cache->format == TC_CACHE_INT8) {
            cache::read_kernel<S, true><<<blocks, cache::kThreads, 0, s>>>(pool, checked, rows, per_block);
        } else {
            cache::read_kernel<S, false><<<blocks, cache::kThreads, 0, s>>>(pool, checked, rows, per_block);
        }
    })
    return check_launch(what);
}

}  // extern "C"
