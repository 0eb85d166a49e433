// The entry point of attention over a cache: its checks, its workspace and the
// launches of each type (cache_attention.hpp).
#include "cache_attention.hpp"

namespace tc {
namespace cache {
namespace {

// Whether blocks share tiles, where `rows` query rows share keys.  (320 rows over
// a prefix of 8000 tokens in 8 bits: 40 us so, 59 with 16 rows a block.  4 or 5
// rows the other way: 4 sequences to 100000 tokens 176 us instead of 113, heads
// of 80 in f16 65 instead of 47.)  For own keys it is the mean of a call's
// sequences that tells: a prompt among many single tokens goes by these.
bool shares(uint64_t rows) { return rows > 16; }

// The storage of one line's parts.
struct Storage {
    Scratch slots, slot_stats, rows, row_stats, found, cut;

    Storage(uint64_t slot_rows, uint64_t whole_rows, uint64_t all_rows, uint64_t size)
        : slots(slot_rows * size * sizeof(float)),
          slot_stats(slot_rows * sizeof(float2)),
          rows(whole_rows * size * sizeof(float)),
          row_stats(whole_rows * sizeof(float2)),
          found(all_rows * sizeof(Found)),
          cut(sizeof(uint32_t)) {}
    int status() const {
        for (int s : {slots.status, slot_stats.status, rows.status, row_stats.status, found.status, cut.status}) {
            if (s != TC_OK) return s;
        }
        return TC_OK;
    }
    Parts parts() const {
        return {static_cast<float*>(slots.ptr), static_cast<float2*>(slot_stats.ptr), static_cast<float*>(rows.ptr),
                static_cast<float2*>(row_stats.ptr), static_cast<Found*>(found.ptr), static_cast<uint32_t*>(cut.ptr)};
    }
};

int run(const AttentionLaunches& launches, const Attention& a, bool quant) {
    const uint64_t units = static_cast<uint64_t>(compute_units());
    const uint64_t size = (a.pool.size + 31) / 32 * 32, tokens = a.batch.tokens, rows = tokens * a.query_heads;
    const bool prefix = a.batch.prefix > 0;
    const uint64_t sequences = a.batch.sequences;
    const bool own_shared = shares(tokens * a.group / (sequences > 0 ? sequences : 1));
    const bool prefix_shared = shares(tokens * a.group);
    const auto slot_rows = [&](bool form) { return 2 * units * blocks_of_form(form) * rows_of_form(form); };
    const Storage own(slot_rows(own_shared), prefix ? rows : 0, rows, size);
    const Storage shared(prefix ? slot_rows(prefix_shared) : 0, prefix ? rows : 0, prefix ? rows : 0, size);
    if (own.status() != TC_OK) return own.status();
    if (shared.status() != TC_OK) return shared.status();
    // (The first launch tells the second whether any token does not see the
    // whole prefix.)
    Parts prefix_parts = shared.parts();
    prefix_parts.cut = own.parts().cut;
    int status = launches.attend(a, own.parts(), quant, false, !prefix, own_shared);
    if (status == TC_OK && prefix) status = launches.attend(a, prefix_parts, quant, true, false, prefix_shared);
    if (status != TC_OK) return status;
    return launches.join(a, own.parts(), shared.parts(), quant, own_shared, prefix_shared);
}

}  // namespace
}  // namespace cache
}  // namespace tc

using namespace tc;

extern "C" {

int tc_cache_attention(const tc_cache* cache, const tc_cache_batch* batch, uint32_t query_heads, float scale,
                       const void* query, uint64_t query_token_step, uint64_t query_head_step, void* out,
                       uint64_t out_token_step, uint64_t out_head_step, float* normalizers) {
    const char* what = "cache attention";
    cache::Attention a{};
    int status = cache::check_pool(what, cache, &a.pool);
    if (status == TC_OK) status = cache::check_batch(what, batch, a.pool, &a.batch);
    if (status != TC_OK) return status;
    if (query_heads == 0 || query_heads % a.pool.heads != 0) {
        return fail(TC_INVALID, std::string(what) + ": " + std::to_string(query_heads) +
                                    " query heads do not share " + std::to_string(a.pool.heads) + " key heads evenly");
    }
    if (!(scale > 0.0f && scale < INFINITY)) {
        return fail(TC_INVALID, std::string(what) + ": a scale of " + std::to_string(scale));
    }
    // Query rows are counted in 32 bits.
    if (uint64_t{a.batch.tokens} * query_heads > 0x7fffff00u) {
        return fail(TC_UNSUPPORTED, std::string(what) + ": " + std::to_string(a.batch.tokens) + " tokens of " +
                                        std::to_string(query_heads) + " heads");
    }
    a.query_heads = query_heads;
    a.group = query_heads / a.pool.heads;
    a.group_of = DivMod(a.group);
    a.scale = scale;
    a.query = query, a.query_steps = {query_token_step, query_head_step};
    a.out = out, a.out_steps = {out_token_step, out_head_step};
    a.normalizers = normalizers;
    status = check_heads(what, "queries", a.query_steps, query_heads, a.batch.tokens, a.pool.size);
    if (status == TC_OK) status = check_heads(what, "results", a.out_steps, query_heads, a.batch.tokens, a.pool.size);
    if (status == TC_OK) status = cache::check_storage(what, *cache, a.pool);
    if (status != TC_OK || a.batch.tokens == 0) return status;
    if (any_null({query, out})) return null_operand(what);
    const bool quant = cache->format == TC_CACHE_INT8;
    switch (cache->dtype) {
        case TC_F32: return cache::run(cache::attend_f32(), a, quant);
        case TC_F16: return cache::run(cache::attend_f16(), a, quant);
        default: return cache::run(cache::attend_bf16(), a, quant);
    }
}

}  // extern "C"
