// What the operators over heads share: where the rows of a tensor [token][head]
// lie, and the check that they do not overlap.
#pragma once

#include "rows.hpp"

namespace tc {

struct Steps {
    uint64_t token, head;
};

// TC_OK if rows of `size` elements of `tokens` tokens and `heads` heads, these
// steps apart, do not overlap and lie within the address space.
inline int check_heads(const std::string& what, const char* name, Steps steps, uint32_t heads, uint64_t tokens,
                       uint32_t size) {
    if (heads == 0) return TC_OK;
    // Whichever of the two axes steps further has to step past the other.
    const bool by_token = steps.token >= steps.head;
    const uint64_t inner = by_token ? steps.head : steps.token, outer = by_token ? steps.token : steps.head;
    const uint64_t inner_count = by_token ? heads : tokens, outer_count = by_token ? tokens : heads;
    uint64_t within = 0, whole = 0;
    const bool fits = !__builtin_mul_overflow(inner, inner_count - (inner_count > 0), &within) &&
                      !__builtin_add_overflow(within, uint64_t{size}, &within) &&
                      !__builtin_mul_overflow(outer, outer_count, &whole) && whole < (uint64_t{1} << 60) &&
                      within < (uint64_t{1} << 60);
    if (!fits) return fail(TC_INVALID, what + ": the " + name + " reach past the address space");
    if ((inner_count > 1 && inner < size) || (outer_count > 1 && outer < within)) {
        return fail(TC_INVALID, what + ": the " + name + " of heads of " + std::to_string(size) +
                                    " elements, tokens " + std::to_string(steps.token) + " and heads " +
                                    std::to_string(steps.head) + " apart, overlap");
    }
    return TC_OK;
}

}  // namespace tc
