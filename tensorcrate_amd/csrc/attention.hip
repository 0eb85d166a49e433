// The entry points of attention: their checks, and the launches of each type
// (attention.hpp).
#include "attention.hpp"

namespace tc {
namespace {

using attention::Shape;

// Whether blocks end where sequences do.  Then no block sweeps the keys of two
// sequences for the few rows that it has of each, but every sequence's last
// block is filled only in part: worth it where sequences are of 128 tokens on
// average, or where all the blocks run at once anyway.  Forward and backward,
// f16, 12 heads of 80, tiles across sequences and by sequence: 8192 tokens of
// 32 sequences 218 and 180 us, of 64 172 and 160, of 128 155 and 172, of 256
// 144 and 230; 200 tokens of 3 sequences 57 and 46.
bool by_sequence(const tc_attention_shape& a) {
    const uint64_t tiles = a.tokens / attention::kOwned;
    return a.sequences > 0 && (tiles >= a.sequences || (tiles + a.sequences + 2) * a.query_heads <=
                                                           static_cast<uint64_t>(compute_units()) * 2);
}

int check(const std::string& what, const tc_attention_shape* given, Shape* shape, const attention::Launches** launches) {
    if (given == nullptr) return fail(TC_INVALID, what + ": no shape");
    const tc_attention_shape& a = *given;
    switch (a.dtype) {
        case TC_F32: *launches = &attention::f32_launches(); break;
        case TC_F16: *launches = &attention::f16_launches(); break;
        case TC_BF16: *launches = &attention::bf16_launches(); break;
        default: return fail(TC_UNSUPPORTED, what + ": no kernel for " + dtype_name(a.dtype));
    }
    if (a.query_heads == 0 || a.key_heads == 0 || a.query_heads % a.key_heads != 0) {
        return fail(TC_INVALID, what + ": " + std::to_string(a.query_heads) + " query heads do not share " +
                                    std::to_string(a.key_heads) + " key heads evenly");
    }
    if (a.head_size == 0) return fail(TC_INVALID, what + ": heads of no elements");
    if (a.head_size > 128) {
        return fail(TC_UNSUPPORTED, what + ": heads of " + std::to_string(a.head_size) + " elements, more than 128");
    }
    if (!(a.scale > 0.0f && a.scale < INFINITY)) {
        return fail(TC_INVALID, what + ": a scale of " + std::to_string(a.scale));
    }
    // Tokens are counted in 32 bits with room for a tile behind them, and a
    // dispatch holds fewer than 2^32 work-items, 256 for every 128 tokens.
    const bool apart = by_sequence(a);
    const uint64_t tiles = a.tokens / attention::kOwned + 1 + (apart ? uint64_t{a.sequences} + 2 : 0);
    if (a.tokens > 0x7fffff00u || tiles > 0xffffffu / a.query_heads) {
        return fail(TC_UNSUPPORTED, what + ": " + std::to_string(a.tokens) + " tokens of " +
                                        std::to_string(a.query_heads) + " heads");
    }
    const struct {
        const char* name;
        Steps steps;
        uint32_t heads;
    } operands[] = {{"queries", {a.query_token_step, a.query_head_step}, a.query_heads},
                    {"keys", {a.key_token_step, a.key_head_step}, a.key_heads},
                    {"values", {a.value_token_step, a.value_head_step}, a.key_heads},
                    {"results", {a.out_token_step, a.out_head_step}, a.query_heads}};
    for (const auto& o : operands) {
        const int status = check_heads(what, o.name, o.steps, o.heads, a.tokens, a.head_size);
        if (status != TC_OK) return status;
    }
    if (a.sequences > 0 && a.tokens > 0 && a.offsets == nullptr) return null_operand(what.c_str());
    *shape = Shape{a.query_heads,
                   a.query_heads / a.key_heads,
                   a.head_size,
                   static_cast<uint32_t>(a.tokens),
                   a.sequences,
                   apart,
                   a.offsets,
                   a.scale,
                   {a.query_token_step, a.query_head_step},
                   {a.key_token_step, a.key_head_step},
                   {a.value_token_step, a.value_head_step},
                   {a.out_token_step, a.out_head_step}};
    return TC_OK;
}

}  // namespace
}  // namespace tc

using namespace tc;

extern "C" {

int tc_attention(const tc_attention_shape* shape, const void* query, const void* key, const void* value, void* out,
                 float* normalizers) {
    Shape checked;
    const attention::Launches* launches = nullptr;
    const int status = check("attention", shape, &checked, &launches);
    if (status != TC_OK || checked.tokens == 0) return status;
    if (any_null({query, key, value, out})) return null_operand("attention");
    return launches->forward(checked, query, key, value, out, normalizers);
}

int tc_attention_backward(const tc_attention_shape* shape, const void* d_out, const void* query, const void* key,
                          const void* value, const void* out, const float* normalizers, void* d_query, void* d_key,
                          void* d_value) {
    Shape checked;
    const attention::Launches* launches = nullptr;
    const int status = check("attention, backward", shape, &checked, &launches);
    if (status != TC_OK || checked.tokens == 0) return status;
    if (any_null({d_out, query, key, value, out, normalizers, d_query, d_key, d_value})) {
        return null_operand("attention, backward");
    }
    return launches->backward(checked, d_out, query, key, value, out, normalizers, d_query, d_key, d_value);
}

}  // extern "C"
