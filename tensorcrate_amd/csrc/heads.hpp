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

// The rows of a tensor [token][head] that one of a block's GROUPS groups of lanes
// takes, every GROUPS-th from token `first` on: token (from there) and head, and
// the row's place in each of some layouts, moved on by sums that are the same
// for the block.
template <int LAYOUTS, int GROUPS>
struct RowWalk {
    uint32_t heads, tokens_on, heads_on;
    uint64_t on[LAYOUTS], wrap[LAYOUTS];
    uint32_t token, head;
    uint64_t at[LAYOUTS];

    __device__ __forceinline__ RowWalk(uint32_t count, const Steps (&steps)[LAYOUTS], uint32_t group, uint64_t first)
        : heads(count), tokens_on(GROUPS / count), heads_on(GROUPS % count), token(group / count), head(group % count) {
#pragma unroll
        for (int n = 0; n < LAYOUTS; n++) {
            on[n] = tokens_on * steps[n].token + heads_on * steps[n].head;
            wrap[n] = steps[n].token - heads * steps[n].head;
            at[n] = (first + token) * steps[n].token + head * steps[n].head;
        }
    }
    __device__ __forceinline__ void move() {
        token += tokens_on, head += heads_on;
        const bool over = head >= heads;
        token += over;
        head -= over ? heads : 0;
#pragma unroll
        for (int n = 0; n < LAYOUTS; n++) at[n] += on[n] + (over ? wrap[n] : 0);
    }
};

}  // namespace tc
