// The entry point of attention over a cache: its checks, its workspace and the
// launches of each type (cache_attention.hpp).
#include "cache_attention.hpp"

namespace tc {
namespace cache {
namespace {

// The form for `rows` query rows that share keys.
int form_of(uint64_t rows) { return rows <= 16 ? kRows16 : rows <= 32 ? kRows32 : kRows128; }

// The storage of one line's parts.
struct Storage {
    Scratch slots, slot_stats, rows, row_stats, plans, cut;

    Storage(uint64_t slot_rows, uint64_t whole_rows, uint64_t items, uint64_t size)
        : slots(slot_rows * size * sizeof(float)),
          slot_stats(slot_rows * sizeof(float2)),
          rows(whole_rows * size * sizeof(float)),
          row_stats(whole_rows * sizeof(float2)),
          plans(items * sizeof(Plan)),
          cut(sizeof(uint32_t)) {}
    int status() const {
        for (int s : {slots.status, slot_stats.status, rows.status, row_stats.status, plans.status, cut.status}) {
            if (s != TC_OK) return s;
        }
        return TC_OK;
    }
    Parts parts() const {
        return {static_cast<float*>(slots.ptr), static_cast<float2*>(slot_stats.ptr), static_cast<float*>(rows.ptr),
                static_cast<float2*>(row_stats.ptr), static_cast<Plan*>(plans.ptr), static_cast<uint32_t*>(cut.ptr)};
    }
};

int run(const AttentionLaunches& launches, const Attention& a, bool quant) {
    const uint32_t blocks = static_cast<uint32_t>(compute_units()) * 2;
    const uint64_t size = (a.pool.size + 31) / 32 * 32, tokens = a.batch.tokens, rows = tokens * a.query_heads;
    const bool prefix = a.batch.prefix > 0;
    const uint64_t sequences = a.batch.sequences;
    const int own_form = form_of(tokens * a.group / (sequences > 0 ? sequences : 1));
    const int prefix_form = form_of(tokens * a.group);
    const uint64_t own_rows = rows_of_form(own_form), prefix_rows = rows_of_form(prefix_form);
    const Storage own(2 * uint64_t{workers_of(own_form, blocks)} * own_rows, prefix ? rows : 0,
                      (tokens * a.group / own_rows + sequences) * a.pool.heads, size);
    const Storage shared(prefix ? 2 * uint64_t{workers_of(prefix_form, blocks)} * prefix_rows : 0, prefix ? rows : 0,
                         prefix ? (tokens * a.group / prefix_rows + 1) * a.pool.heads : 0, size);
    if (own.status() != TC_OK) return own.status();
    if (shared.status() != TC_OK) return shared.status();
    // (The first launch tells the second whether any token does not see the
    // whole prefix.)
    Parts prefix_parts = shared.parts();
    prefix_parts.cut = own.parts().cut;
    int status = launches.attend(a, own.parts(), quant, false, !prefix, own_form, blocks);
    if (status == TC_OK && prefix) status = launches.attend(a, prefix_parts, quant, true, false, prefix_form, blocks);
    if (status != TC_OK) return status;
    return launches.join(a, own.parts(), shared.parts(), quant, own_form, prefix_form, blocks);
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
