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
// row's place (offsets, length, page).  A wave takes a token's rows, so that
// this chain is walked once for several of them: 16 lanes hold a row, 8
// elements each, and the largest magnitude is taken in registers.

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
constexpr int kAtOnce = 4;  // rows whose loads a lane has in flight

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

// Elements 8 lane .. 8 lane + 8 of a row of `size`, zeros behind it.
template <typename S>
__device__ __forceinline__ void load_eight(const S* row, uint32_t lane, uint32_t size, Words<S, 8>& out) {
    if (8 * lane + 8 <= size) {
        out.template load<false>(row + 8 * lane);
    } else {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = 8 * lane + e < size ? Elem<S>::widen(row[8 * lane + e]) : 0.0f;
        out.put(v);
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

// A wave's token and its share of the token's rows, keys before values.
struct Share {
    uint32_t token, part;
};
__device__ __forceinline__ Share share_of(uint64_t unit, uint32_t parts) {
    return {static_cast<uint32_t>(unit / parts), static_cast<uint32_t>(unit % parts)};
}

// The place of the token's position in its sequence: the sequence and the
// position, or kNowhere.
struct Place {
    uint32_t sequence, at;
};
__device__ __forceinline__ Place place_of(const Batch& batch, uint32_t token) {
    Span span;
    const uint32_t sequence = wave_sequence_of(batch, token, &span);
    if (sequence == kNowhere) return {kNowhere, 0};
    // The sequence's tokens here are its last.
    const uint32_t length = batch.lengths[sequence], left = span.end - token;
    return length < left ? Place{kNowhere, 0} : Place{sequence, length - left};
}

template <typename S, bool QUANT>
__global__ void __launch_bounds__(kThreads)
    write_kernel(const Pool pool, const Batch batch, const Rows<const S*> rows, uint32_t parts) {
    const uint32_t lane = threadIdx.x % 16, turn = threadIdx.x % 64 / 16;
    const uint64_t units = uint64_t{batch.tokens} * parts, waves = uint64_t{gridDim.x} * (kThreads / 64);
    for (uint64_t unit = uint64_t{blockIdx.x} * (kThreads / 64) + threadIdx.x / 64; unit < units; unit += waves) {
        const Share share = share_of(unit, parts);
        const Place place = place_of(batch, share.token);
        if (place.sequence == kNowhere) continue;
        const uint32_t first = row_of(pool, batch.pages + uint64_t{place.sequence} * batch.most_pages,
                                      batch.most_pages, 0, place.at);
        if (first == kNowhere) continue;
        for (uint32_t base = share.part * 4; base < 2 * pool.heads; base += parts * 4 * kAtOnce) {
            Words<S, 8> words[kAtOnce];
#pragma unroll
            for (int k = 0; k < kAtOnce; k++) {
                const uint32_t n = base + k * parts * 4 + turn;
                if (n >= 2 * pool.heads) continue;
                const bool key = n < pool.heads;
                const uint32_t head = key ? n : n - pool.heads;
                const Steps steps = key ? rows.key_steps : rows.value_steps;
                load_eight((key ? rows.key : rows.value) + share.token * steps.token + head * steps.head, lane,
                           pool.size, words[k]);
            }
#pragma unroll
            for (int k = 0; k < kAtOnce; k++) {
                const uint32_t n = base + k * parts * 4 + turn;
                if (n >= 2 * pool.heads) continue;
                const bool key = n < pool.heads;
                const uint32_t row = first + (key ? n : n - pool.heads) * pool.page_size;
                void* const entries = key ? pool.keys : pool.values;
                if constexpr (QUANT) {
                    float v[8], most = 0.0f;
                    words[k].get(v);
#pragma unroll
                    for (int e = 0; e < 8; e++) most = LargestBits::join(most, fabsf(v[e]));
                    most = row16<LargestBits>(most);
                    // Bits past the largest finite number's: an infinity or a NaN.
                    const bool finite = __float_as_uint(most) < 0x7f800000u;
                    const float scale = finite ? most / 127.0f : __uint_as_float(0x7fc00000u);
                    uint32_t packed[2] = {0, 0};
                    if (finite && scale > 0.0f) {
#pragma unroll
                        for (int e = 0; e < 8; e++) {
                            const float q = fminf(fmaxf(rintf(v[e] / scale), -127.0f), 127.0f);
                            packed[e / 4] |= (static_cast<uint32_t>(static_cast<int>(q)) & 0xffu) << (8 * (e % 4));
                        }
                    }
                    if (8 * lane < pool.row) {
                        *reinterpret_cast<uint2*>(static_cast<char*>(entries) + uint64_t{row} * pool.row + 8 * lane) =
                            make_uint2(packed[0], packed[1]);
                    }
                    if (lane == 0) (key ? pool.key_scales : pool.value_scales)[row] = scale;
                } else {
                    S* const to = static_cast<S*>(entries) + uint64_t{row} * pool.row + 8 * lane;
#pragma unroll
                    for (int w = 0; w < Words<S, 8>::kCount; w++) {
                        if (8 * lane + w * kWordElements<S> < pool.row) {
                            store_word<false>(to + w * kWordElements<S>, words[k].w[w]);
                        }
                    }
                }
            }
        }
    }
}

template <typename S, bool QUANT>
__global__ void __launch_bounds__(kThreads)
    read_kernel(const Pool pool, const Batch batch, const Rows<S*> rows, uint32_t parts) {
    const uint32_t lane = threadIdx.x % 16, turn = threadIdx.x % 64 / 16;
    const uint64_t units = uint64_t{batch.tokens} * parts, waves = uint64_t{gridDim.x} * (kThreads / 64);
    for (uint64_t unit = uint64_t{blockIdx.x} * (kThreads / 64) + threadIdx.x / 64; unit < units; unit += waves) {
        const Share share = share_of(unit, parts);
        const Place place = place_of(batch, share.token);
        const uint32_t first = place.sequence == kNowhere
                                   ? kNowhere
                                   : row_of(pool, batch.pages + uint64_t{place.sequence} * batch.most_pages,
                                            batch.most_pages, 0, place.at);
        for (uint32_t base = share.part * 4; base < 2 * pool.heads; base += parts * 4 * kAtOnce) {
            Words<S, 8> words[kAtOnce];
            uint2 packed[kAtOnce];
            float scales[kAtOnce];
#pragma unroll
            for (int k = 0; k < kAtOnce; k++) {
                const uint32_t n = base + k * parts * 4 + turn;
                packed[k] = make_uint2(0, 0), scales[k] = 0.0f;
#pragma unroll
                for (int w = 0; w < Words<S, 8>::kCount; w++) words[k].w[w] = make_uint4(0, 0, 0, 0);
                if (n >= 2 * pool.heads || first == kNowhere) continue;
                const bool key = n < pool.heads;
                const uint32_t row = first + (key ? n : n - pool.heads) * pool.page_size;
                const void* const entries = key ? pool.keys : pool.values;
                if constexpr (QUANT) {
                    if (8 * lane < pool.row) {
                        packed[k] = *reinterpret_cast<const uint2*>(static_cast<const char*>(entries) +
                                                                    uint64_t{row} * pool.row + 8 * lane);
                    }
                    scales[k] = (key ? pool.key_scales : pool.value_scales)[row];
                } else {
                    const S* const from = static_cast<const S*>(entries) + uint64_t{row} * pool.row + 8 * lane;
#pragma unroll
                    for (int w = 0; w < Words<S, 8>::kCount; w++) {
                        if (8 * lane + w * kWordElements<S> < pool.row) {
                            words[k].w[w] = load_word<false>(from + w * kWordElements<S>);
                        }
                    }
                }
            }
#pragma unroll
            for (int k = 0; k < kAtOnce; k++) {
                const uint32_t n = base + k * parts * 4 + turn;
                if (n >= 2 * pool.heads) continue;
                if constexpr (QUANT) {
                    float v[8];
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const uint32_t four = e < 4 ? packed[k].x : packed[k].y;
                        v[e] = static_cast<float>(static_cast<int8_t>(four >> (8 * (e % 4)))) * scales[k];
                    }
                    words[k].put(v);
                }
                const bool key = n < pool.heads;
                const uint32_t head = key ? n : n - pool.heads;
                const Steps steps = key ? rows.key_steps : rows.value_steps;
                store_eight((key ? rows.key : rows.value) + share.token * steps.token + head * steps.head, lane,
                            pool.size, words[k]);
            }
        }
    }
}

// The waves that share a token's rows: all that can where tokens are few, one
// where they fill the chip.
uint32_t parts_of(const Pool& pool, const Batch& batch) {
    const uint32_t most = (2 * pool.heads + 3) / 4;
    return batch.tokens >= static_cast<uint32_t>(compute_units()) * 8 ? 1 : most;
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
    const uint32_t parts = cache::parts_of(pool, checked);
    const uint32_t blocks = grid_for(uint64_t{checked.tokens} * parts, cache::kThreads / 64, 32);
    TC_DISPATCH_FLOAT(cache->dtype, what, S, {
        const cache::Rows<const S*> rows{static_cast<const S*>(key), static_cast<const S*>(value), key_steps,
                                         value_steps};
        if (cache->format == TC_CACHE_INT8) {
            cache::write_kernel<S, true><<<blocks, cache::kThreads, 0, s>>>(pool, checked, rows, parts);
        } else {
            cache::write_kernel<S, false><<<blocks, cache::kThreads, 0, s>>>(pool, checked, rows, parts);
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
    const uint32_t parts = cache::parts_of(pool, checked);
    const uint32_t blocks = grid_for(uint64_t{checked.tokens} * parts, cache::kThreads / 64, 32);
    TC_DISPATCH_FLOAT(cache->dtype, what, S, {
        const cache::Rows<S*> rows{static_cast<S*>(key), static_cast<S*>(value), key_steps, value_steps};
        if (cache->format == TC_CACHE_INT8) {
            cache::read_kernel<S, true><<<blocks, cache::kThreads, 0, s>>>(pool, checked, rows, parts);
        } else {
            cache::read_kernel<S, false><<<blocks, cache::kThreads, 0, s>>>(pool, checked, rows, parts);
        }
    })
    return check_launch(what);
}

}  // extern "C"
