// What the kernels over a cache of keys and values share: the pool of pages,
// the sequences of a call, and where a token's rows lie.
#pragma once

#include "heads.hpp"

namespace tc {
namespace cache {

constexpr uint32_t kNowhere = 0xffffffffu;  // as a row or a sequence: none

struct Pool {
    uint32_t heads, size;
    uint32_t row;  // elements from one row to the next
    uint32_t page_size, page_count;
    DivMod pages_of;  // divides by page_size
    void* keys;
    void* values;
    float* key_scales;
    float* value_scales;
};

struct Batch {
    uint32_t tokens, sequences, most_pages;
    uint32_t prefix;
    const uint32_t* offsets;
    const uint32_t* lengths;
    const uint32_t* pages;
    const uint32_t* prefix_pages;
};

// The row in the pool of token `at` of a sequence that has `count` pages.
__device__ __forceinline__ uint32_t row_of(const Pool& pool, const uint32_t* pages, uint32_t count, uint32_t head,
                                           uint32_t at) {
    const uint32_t n = pool.pages_of.div(at);
    if (n >= count) return kNowhere;
    const uint32_t page = pages[n];
    return page < pool.page_count ? (page * pool.heads + head) * pool.page_size + (at - n * pool.page_size) : kNowhere;
}

// The tokens of a sequence in a call, within the call's whatever the offsets
// hold.
struct Span {
    uint32_t first, end;
};
__device__ __forceinline__ Span span_of(const Batch& batch, uint32_t sequence) {
    if (batch.offsets == nullptr) return {sequence, sequence + 1};
    const uint32_t first = batch.offsets[sequence], end = batch.offsets[sequence + 1];
    return {first < batch.tokens ? first : batch.tokens, end < batch.tokens ? end : batch.tokens};
}

// The sequence that has `token`, kNowhere if none has; `span` its tokens.  Of
// sequences that begin at the same token the last one may have any.
__device__ __forceinline__ uint32_t sequence_of(const Batch& batch, uint32_t token, Span* span) {
    if (batch.sequences == 0) return kNowhere;
    uint32_t low = 0;
    if (batch.offsets == nullptr) {
        low = token;
    } else {
        uint32_t high = batch.sequences;
        while (high - low > 1) {
            const uint32_t middle = low + (high - low) / 2;
            if (batch.offsets[middle] <= token) low = middle;
            else high = middle;
        }
    }
    *span = span_of(batch, low);
    return token >= span->first && token < span->end ? low : kNowhere;
}

// The same for a token that is the same in the whole wave, which asks 64
// places at a time.
__device__ __forceinline__ uint32_t wave_sequence_of(const Batch& batch, uint32_t token, Span* span) {
    if (batch.sequences == 0) return kNowhere;
    uint32_t low = 0;
    if (batch.offsets == nullptr) {
        low = token;
    } else {
        const uint32_t lane = threadIdx.x % 64;
        uint32_t count = batch.sequences;
        while (count > 1) {
            const uint32_t step = (count + 63) / 64;
            const uint64_t at = uint64_t{lane} * step;
            const bool before = at < count && batch.offsets[low + static_cast<uint32_t>(at)] <= token;
            const uint64_t passed = __ballot(before);
            if (passed == 0) break;
            const uint32_t last = static_cast<uint32_t>(__popcll(passed)) - 1;
            low += last * step;
            count = count - last * step < step ? count - last * step : step;
        }
        low = __builtin_amdgcn_readfirstlane(low);
    }
    *span = span_of(batch, low);
    return token >= span->first && token < span->end ? low : kNowhere;
}

// Checks of a call's arguments (cache.hip).
int check_pool(const std::string& what, const tc_cache* given, Pool* pool);
int check_batch(const std::string& what, const tc_cache_batch* given, const Pool& pool, Batch* batch);
int check_storage(const std::string& what, const tc_cache& cache, const Pool& pool);

}  // namespace cache
}  // namespace tc
