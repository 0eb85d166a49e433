// The norm of each head of queries and keys and the rotation of its elements
// by position, in one pass, and the gradients.
//
// Of a head x of n elements with weight w, at position t of frequencies f:
//   r = 1 / sqrt(mean(x^2) + epsilon),  y = x r w  (or y = x without a norm),
// and for each pair (y_a, y_b) of the rotated elements, with angle t f_i:
//   z_a = y_a cos - y_b sin,  z_b = y_b cos + y_a sin.
// Backward from dz: dy is dz turned back by the same angles, and with u = x r
// and g = dy w
//   dx = r (g - u mean(g u)),  dw = sum over tokens and heads of dy u.
// Both are bound by memory: x (backward dz and x) is read once and one result
// written.  16 lanes hold a head, 4 pairs each, so that the norm is a sum in
// registers and no pair is split.  r is computed again backward: it takes no
// read that is not made anyway.
//
// Cosines and sines are one per token and pair, for all heads of the token: a
// block computes those of a few tokens into LDS and then walks their heads.
// An angle is a product in 64 bits, reduced to a part of a turn there, so that
// far positions lose nothing; the functions of that part are taken in 32.
//
// Measured: 16384 tokens of 40 heads of 128 in bf16 forward 62 us (5.4 TB/s), of 36
// backward with both weights 91 us (5.0), of which the weights' second launch is
// some 5; 16 tokens 4.9 us, a launch's time.  With one row of a lane's on its way
// those were 115, 145 and 6.8 us.

#include <type_traits>

#include "heads.hpp"

namespace tc {
namespace {

constexpr int kThreads = 256;
constexpr int kGroups = kThreads / 16;  // rows that a block holds at a time
constexpr uint32_t kMostPairs = 64;     // of a head
constexpr uint32_t kForwardPerUnit = 6, kBackPerUnit = 4;  // blocks of a compute unit
constexpr uint32_t kMostTokens = 4;     // whose cosines and sines a block holds

template <typename S, typename W>
struct Rotary {
    uint32_t heads[2];  // of queries and keys
    uint32_t size, half;  // elements of a head, and rotated pairs
    bool normalize;
    float epsilon;
    uint64_t tokens;
    uint32_t chunk;  // tokens of a block's turn
    const uint32_t* positions;
    const float* frequencies;
    // Forward x and z; backward dz, x and dx.
    const S* from[2];
    Steps from_steps[2];
    const S* x[2];
    Steps x_steps[2];
    S* to[2];
    Steps to_steps[2];
    const W* weight[2];
};

// The elements of a head that lane j of 16 holds: the 4 pairs from 4 j on, as
// 8 slots.  A rotated pair p is (p, p + half) or, as neighbours, (2p, 2p + 1);
// behind the rotated elements pairs are neighbours, and nothing turns them.
// Where a lane's elements are whole runs of 4 (or 8) it moves them as words,
// at any alignment; the others one by one.
template <bool HALVES>
struct Lane {
    uint32_t pair, size, half;
    uint32_t first, second;  // columns of slots 0 and 4, of whole runs
    // Whole runs, and whether the lane has elements at all: one that has none
    // reads the head's first ones, since a branch that zeroes its registers
    // would wait for the other lanes' loads, and adds nothing to any sum.
    bool whole, has;

    __device__ __forceinline__ Lane(uint32_t lane, uint32_t n, uint32_t turned)
        : pair(4 * lane), size(n), half(turned) {
        const bool halves = HALVES && pair + 4 <= half;
        first = halves ? pair : 2 * pair;
        second = halves ? pair + half : 2 * pair + 4;
        whole = halves || ((!HALVES || pair >= half) && 2 * pair + 8 <= size);
        has = pair < half || 2 * pair < size;
        if (!has && size >= 8) whole = true, first = 0, second = 4;
    }
    __device__ __forceinline__ static constexpr int a(int i) { return HALVES ? i : 2 * i; }
    __device__ __forceinline__ static constexpr int b(int i) { return HALVES ? i + 4 : 2 * i + 1; }
    // Column of a slot, `size` or more if it has none.
    __device__ __forceinline__ uint32_t column(int slot) const {
        if (!has) return size;
        if (whole) return slot < 4 ? first + slot : second + slot - 4;
        return scattered(pair, slot);
    }
    __device__ __forceinline__ uint32_t scattered(uint32_t from, int slot) const {
        const uint32_t p = from + (HALVES ? slot % 4 : slot / 2);
        const uint32_t other = HALVES ? slot / 4 : slot % 2;
        return HALVES && p < half ? p + other * half : 2 * p + other;
    }
    // `pair`, so that columns are found where they are used: kept through the
    // loop over rows they would take registers of all lanes.
    __device__ __forceinline__ uint32_t here() const {
        uint32_t from = pair;
        asm volatile("" : "+v"(from));
        return from;
    }
    template <bool NT, typename S>
    __device__ __forceinline__ void load(const S* row, Words<S, 8>& out) const {
        typedef uint32_t piece __attribute__((ext_vector_type(sizeof(S)), aligned(sizeof(S))));
        if (whole) {
            const piece* const from[2] = {reinterpret_cast<const piece*>(row + first),
                                          reinterpret_cast<const piece*>(row + second)};
            const piece low = NT ? __builtin_nontemporal_load(from[0]) : *from[0];
            const piece high = NT ? __builtin_nontemporal_load(from[1]) : *from[1];
            __builtin_memcpy(out.w, &low, sizeof(low));
            __builtin_memcpy(reinterpret_cast<char*>(out.w) + sizeof(low), &high, sizeof(high));
        } else {
            const uint32_t from = here();
            float v[8];
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const uint32_t c = scattered(from, k);
                v[k] = c < size ? Elem<S>::widen(row[c]) : 0.0f;
            }
            out.put(v);
        }
    }
    template <bool NT, typename S>
    __device__ __forceinline__ void store(S* row, const float (&v)[8]) const {
        typedef uint32_t piece __attribute__((ext_vector_type(sizeof(S)), aligned(sizeof(S))));
        if (!has) return;
        if (whole) {
            Words<S, 8> words;
            words.put(v);
            piece low, high;
            __builtin_memcpy(&low, words.w, sizeof(low));
            __builtin_memcpy(&high, reinterpret_cast<const char*>(words.w) + sizeof(low), sizeof(high));
            if constexpr (NT) {
                __builtin_nontemporal_store(low, reinterpret_cast<piece*>(row + first));
                __builtin_nontemporal_store(high, reinterpret_cast<piece*>(row + second));
            } else {
                *reinterpret_cast<piece*>(row + first) = low;
                *reinterpret_cast<piece*>(row + second) = high;
            }
        } else {
            const uint32_t from = here();
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const uint32_t c = scattered(from, k);
                if (c < size) row[c] = Elem<S>::narrow(v[k]);
            }
        }
    }
    // The pairs' turns, back with SIGN -1.
    template <int SIGN>
    __device__ __forceinline__ void turn(float (&v)[8], const float2* turns) const {
        if (pair >= half) return;
        const bool all = pair + 4 <= half;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 t = turns[pair + i];
            const float x = v[a(i)], y = v[b(i)], s = SIGN < 0 ? -t.y : t.y;
            const bool turned = all || pair + i < half;
            v[a(i)] = turned ? fmaf(x, t.x, -(y * s)) : x;
            v[b(i)] = turned ? fmaf(y, t.x, x * s) : y;
        }
    }
};

// 1 / sqrt(v), by the instruction, which takes no subnormal number.
__device__ __forceinline__ float reciprocal_root(float v) {
    const bool small = v < 0x1p-100f;
    const float root = __builtin_amdgcn_rsqf(small ? v * 0x1p64f : v);
    return small ? root * 0x1p32f : root;
}

// `sums` (BACK; null if no weight's gradient is wanted): of each block, for
// queries and then keys, 8 slots of 16 lanes.
template <typename S, typename W, bool HALVES, bool BACK, bool NT>
__global__ void __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(BACK ? kBackPerUnit : kForwardPerUnit))) rotary_kernel(const Rotary<S, W> r, float* __restrict__ sums) {
    __shared__ __attribute__((aligned(16))) float2 turns[2][kMostTokens][kMostPairs];
    const uint32_t lane = threadIdx.x % 16, group = threadIdx.x / 16;
    const Lane<HALVES> at(lane, r.size, r.half);
    const float part = 1.0f / static_cast<float>(r.size);

    // Each lane's weights, the same for the block's groups.
    __shared__ __attribute__((aligned(16))) float weights[2][16][8];
    if (threadIdx.x < 2 * 16 * 8) {
        const uint32_t n = threadIdx.x / 128, k = threadIdx.x % 8, of = threadIdx.x / 8 % 16;
        const uint32_t c = Lane<HALVES>(of, r.size, r.half).column(k);
        const W* const from = n == 0 ? r.weight[0] : r.weight[1];
        weights[n][of][k] = from != nullptr && c < r.size ? Elem<W>::widen(from[c]) : 1.0f;
    }
    float along[BACK ? 2 : 1][8] = {};

    const auto tokens_at = [&](uint64_t first) {
        return r.tokens <= first ? 0 : r.tokens - first < r.chunk ? static_cast<uint32_t>(r.tokens - first) : r.chunk;
    };
    const auto find_turns = [&](int stage, uint64_t first) {
        for (uint32_t i = threadIdx.x; i < tokens_at(first) * r.half; i += kThreads) {
            const uint32_t token = i / r.half, pair = i % r.half;
            const uint32_t position =
                r.positions != nullptr ? r.positions[first + token] : static_cast<uint32_t>(first + token);
            // In turns: 1 / (2 pi) to 64 bits.
            const double angle = static_cast<double>(position) * static_cast<double>(r.frequencies[pair]) *
                                 0.15915494309189533577;
            float2 turn;
            sincospif(2.0f * static_cast<float>(angle - rint(angle)), &turn.y, &turn.x);
            turns[stage][token][pair] = turn;
        }
    };
    // A row's words on their way: of x forward, of dz and x backward.
    struct Fetched {
        Words<S, 8> row, x;
    };
    constexpr int LAYOUTS = BACK ? 3 : 2;
    const auto walk_of = [&](auto which, uint64_t first) {
        constexpr int n = decltype(which)::value;
        const Steps steps[3] = {r.from_steps[n], r.to_steps[n], r.x_steps[n]};
        return RowWalk<LAYOUTS, kGroups>(r.heads[n], reinterpret_cast<const Steps(&)[LAYOUTS]>(steps), group, first);
    };
    const auto fetch = [&](auto which, const RowWalk<LAYOUTS, kGroups>& walk, Fetched& out) {
        constexpr int n = decltype(which)::value;
        at.template load<NT>(r.from[n] + walk.at[0], out.row);
        if constexpr (BACK) {
            if (r.normalize) at.template load<NT>(r.x[n] + walk.at[2], out.x);
        }
    };
    // The rows of queries or keys of `here` tokens, the first of them in `next`
    // and each one's successor in flight.
    const auto rows_of = [&](auto which, int stage, RowWalk<LAYOUTS, kGroups>& walk, uint32_t here, Fetched& next) {
        constexpr int n = decltype(which)::value;
        while (walk.token < here) {
            const uint32_t token = walk.token;
            S* const to = r.to[n] + walk.at[1];
            float v[8], x[8];
            next.row.get(v);
            if constexpr (BACK) next.x.get(x);
            walk.move();
            if (walk.token < here) fetch(which, walk, next);
            float scale = 1.0f;
            if (r.normalize) {
                float squares = 0.0f;
#pragma unroll
                for (int k = 0; k < 8; k++) squares = fmaf(BACK ? x[k] : v[k], BACK ? x[k] : v[k], squares);
                scale = reciprocal_root(fmaf(row16<Added>(at.has ? squares : 0.0f), part, r.epsilon));
            }
            if constexpr (!BACK) {
                if (r.normalize) {
#pragma unroll
                    for (int k = 0; k < 8; k++) v[k] = v[k] * scale * weights[n][lane][k];
                }
                at.template turn<1>(v, turns[stage][token]);
            } else {
                at.template turn<-1>(v, turns[stage][token]);
                if (r.normalize) {
                    float dot = 0.0f;
#pragma unroll
                    for (int k = 0; k < 8; k++) {
                        x[k] *= scale;
                        along[n][k] = fmaf(v[k], x[k], along[n][k]);
                        v[k] *= weights[n][lane][k];
                        dot = fmaf(v[k], x[k], dot);
                    }
                    dot = row16<Added>(at.has ? dot : 0.0f) * part;
#pragma unroll
                    for (int k = 0; k < 8; k++) v[k] = scale * fmaf(-x[k], dot, v[k]);
                }
            }
            at.template store<NT>(to, v);
        }
    };

    const uint64_t apart = uint64_t{gridDim.x} * r.chunk;
    uint64_t first = uint64_t{blockIdx.x} * r.chunk;
    const std::integral_constant<int, 0> queries;
    const std::integral_constant<int, 1> keys;
    Fetched next_query, next_key;
    // The first query row of a turn is on its way before the last turn's keys
    // are done, the first key row before the turn's queries are.
    const auto begin = [&](auto which, uint64_t from, Fetched& out) {
        constexpr int n = decltype(which)::value;
        if (r.heads[n] == 0) return;
        const RowWalk<LAYOUTS, kGroups> walk = walk_of(which, from);
        if (walk.token < tokens_at(from)) fetch(which, walk, out);
    };
    begin(queries, first, next_query);
    find_turns(0, first);
    int stage = 0;
    for (; first < r.tokens; first += apart, stage ^= 1) {
        // (The stage that is written was read before the last barrier.)
        __syncthreads();
        const uint32_t here = tokens_at(first);
        begin(keys, first, next_key);
        find_turns(stage ^ 1, first + apart);
        if (r.heads[0] > 0) {
            RowWalk<LAYOUTS, kGroups> walk = walk_of(queries, first);
            rows_of(queries, stage, walk, here, next_query);
        }
        begin(queries, first + apart, next_query);
        if (r.heads[1] > 0) {
            RowWalk<LAYOUTS, kGroups> walk = walk_of(keys, first);
            rows_of(keys, stage, walk, here, next_key);
        }
    }
    if constexpr (BACK) {
        if (sums == nullptr) return;
        // The wave's four rows, in registers, then the waves in order.
        __shared__ float shared[kThreads / 64][2][8][16];
#pragma unroll
        for (int n = 0; n < 2; n++) {
#pragma unroll
            for (int k = 0; k < 8; k++) {
                float v = along[n][k];
                v += __shfl_xor(v, 16);
                v += __shfl_xor(v, 32);
                if (threadIdx.x % 64 < 16) shared[threadIdx.x / 64][n][k][lane] = v;
            }
        }
        __syncthreads();
        const float* all = &shared[0][0][0][0];
        float v = all[threadIdx.x];
        for (int w = 1; w < kThreads / 64; w++) v += all[w * 256 + threadIdx.x];
        sums[uint64_t{blockIdx.x} * 256 + threadIdx.x] = v;
    }
}

// Both weights' gradients: the blocks' sums of one slot by a wave, each lane
// every 64th block's, the lanes in a fixed order.
template <typename W, bool HALVES>
__global__ void __launch_bounds__(kThreads)
    rotary_weights_kernel(const float* __restrict__ sums, uint32_t blocks, uint32_t size, uint32_t half,
                          W* d_query_weight, W* d_key_weight) {
    const uint32_t place = blockIdx.x * (kThreads / 64) + threadIdx.x / 64;  // of 256
    const uint32_t n = place / 128, slot = place / 16 % 8, lane = place % 16;
    float sum = 0.0f;
#pragma unroll 8
    for (uint32_t b = threadIdx.x % 64; b < blocks; b += 64) sum += sums[uint64_t{b} * 256 + place];
    sum = wave64<Added>(sum);
    const uint32_t column = Lane<HALVES>(lane, size, half).column(slot);
    W* to = n == 0 ? d_query_weight : d_key_weight;
    if (threadIdx.x % 64 == 0 && to != nullptr && column < size) to[column] = Elem<W>::narrow(sum);
}

template <typename S, typename W, bool BACK>
int rotary(const tc_rotary_shape& a, Rotary<S, W> r, W* d_query_weight, W* d_key_weight, const char* what) {
    TC_STREAM(s);
    r.heads[0] = a.query_heads, r.heads[1] = a.key_heads;
    r.size = a.head_size, r.half = a.rotary_size / 2;
    r.normalize = a.normalize != 0;
    r.epsilon = a.epsilon;
    r.tokens = a.tokens;
    r.positions = a.positions, r.frequencies = a.frequencies;
    // As many blocks as run at once, walking the tokens together: several at a
    // time where there are many (gradients of 7001 tokens of 24 heads of 80 29 us,
    // one at a time 36; 16384 of 36 heads 91 and 94, forward of 40 heads 62 and 60),
    // else one (16 tokens 4.9 us, four at a time 8.5).
    const uint32_t per_unit = BACK ? kBackPerUnit : kForwardPerUnit;
    const uint64_t units = static_cast<uint64_t>(compute_units());
    r.chunk = a.tokens >= units * per_unit * 2 ? kMostTokens : 1;
    const bool weights = BACK && (d_query_weight != nullptr || d_key_weight != nullptr);
    const bool rows = a.tokens > 0 && a.query_heads + uint64_t{a.key_heads} > 0;
    const uint32_t blocks = rows ? grid_for(a.tokens, r.chunk, per_unit) : 0;
    Scratch scratch(weights ? uint64_t{blocks} * 256 * sizeof(float) : 0);
    if (scratch.status != TC_OK) return scratch.status;
    float* sums = weights ? static_cast<float*>(scratch.ptr) : nullptr;
    const bool halves = a.pairs == TC_ROTARY_HALVES;
    int status = TC_OK;
    if (rows) {
        const uint64_t moved = (BACK ? 3 : 2) * sizeof(S) * a.tokens * r.size * (uint64_t{r.heads[0]} + r.heads[1]);
        const bool streams = moved >= kStreamBytes;
        if (halves && streams) rotary_kernel<S, W, true, BACK, true><<<blocks, kThreads, 0, s>>>(r, sums);
        if (halves && !streams) rotary_kernel<S, W, true, BACK, false><<<blocks, kThreads, 0, s>>>(r, sums);
        if (!halves && streams) rotary_kernel<S, W, false, BACK, true><<<blocks, kThreads, 0, s>>>(r, sums);
        if (!halves && !streams) rotary_kernel<S, W, false, BACK, false><<<blocks, kThreads, 0, s>>>(r, sums);
        status = check_launch(what);
    }
    if (status != TC_OK || !weights) return status;
    if (halves) {
        rotary_weights_kernel<W, true><<<256 / (kThreads / 64), kThreads, 0, s>>>(sums, blocks, r.size, r.half,
                                                                                  d_query_weight, d_key_weight);
    } else {
        rotary_weights_kernel<W, false><<<256 / (kThreads / 64), kThreads, 0, s>>>(sums, blocks, r.size, r.half,
                                                                                   d_query_weight, d_key_weight);
    }
    return check_launch(what);
}

int check_rotary(const std::string& what, const tc_rotary_shape* given, bool weights) {
    if (given == nullptr) return fail(TC_INVALID, what + ": no shape");
    const tc_rotary_shape& a = *given;
    if (dtype_size(a.dtype) == 0 || a.dtype == TC_F64) {
        return fail(TC_UNSUPPORTED, what + ": no kernel for " + dtype_name(a.dtype));
    }
    if (a.weight_dtype != a.dtype && a.weight_dtype != TC_F32) {
        return fail(TC_UNSUPPORTED, what + ": no kernel for " + dtype_name(a.dtype) + " heads with a " +
                                        dtype_name(a.weight_dtype) + " weight");
    }
    if (a.head_size == 0) return fail(TC_INVALID, what + ": heads of no elements");
    if (a.head_size > 2 * kMostPairs) {
        return fail(TC_UNSUPPORTED, what + ": heads of " + std::to_string(a.head_size) + " elements, more than 128");
    }
    if (a.rotary_size % 2 != 0 || a.rotary_size > a.head_size) {
        return fail(TC_INVALID, what + ": " + std::to_string(a.rotary_size) + " rotated of " +
                                    std::to_string(a.head_size) + " elements");
    }
    if (a.pairs != TC_ROTARY_HALVES && a.pairs != TC_ROTARY_NEIGHBOURS) {
        return fail(TC_INVALID, what + ": pairs of kind " + std::to_string(a.pairs));
    }
    if (a.normalize != 0 && !(a.epsilon >= 0.0f && a.epsilon < INFINITY)) {
        return fail(TC_INVALID, what + ": an epsilon of " + std::to_string(a.epsilon));
    }
    if (a.normalize == 0 && weights) return fail(TC_INVALID, what + ": a weight without a norm");
    // A block's rows, and tokens as positions, are counted in 32 bits.
    if (a.tokens > UINT32_MAX || a.query_heads > (1u << 24) || a.key_heads > (1u << 24)) {
        return fail(TC_UNSUPPORTED, what + ": " + std::to_string(a.tokens) + " tokens of " +
                                        std::to_string(a.query_heads) + " and " + std::to_string(a.key_heads) +
                                        " heads");
    }
    const struct {
        const char* name;
        Steps steps;
        uint32_t heads;
    } operands[] = {{"queries", {a.query_token_step, a.query_head_step}, a.query_heads},
                    {"keys", {a.key_token_step, a.key_head_step}, a.key_heads},
                    {"rotated queries", {a.query_out_token_step, a.query_out_head_step}, a.query_heads},
                    {"rotated keys", {a.key_out_token_step, a.key_out_head_step}, a.key_heads}};
    for (const auto& o : operands) {
        const int status = check_heads(what, o.name, o.steps, o.heads, a.tokens, a.head_size);
        if (status != TC_OK) return status;
    }
    if (a.tokens > 0 && a.rotary_size > 0 && a.frequencies == nullptr) return null_operand(what.c_str());
    return TC_OK;
}

}  // namespace
}  // namespace tc

using namespace tc;

// `f(S rows' type, W weight's type)` for the shape's two type codes.
#define TC_ROTARY_TYPES(shape, what, ...)                                  \
    TC_DISPATCH_FLOAT(shape.dtype, what, S, {                              \
        if (shape.weight_dtype == TC_F32) {                                \
            using W = float; __VA_ARGS__;                                  \
        } else {                                                           \
            using W = S; __VA_ARGS__;                                      \
        }                                                                  \
    })

extern "C" {

int tc_rotary_norm(const tc_rotary_shape* shape, const void* query, const void* key, const void* query_weight,
                   const void* key_weight, void* query_out, void* key_out) {
    const char* what = "rotary norm";
    const int status = check_rotary(what, shape, query_weight != nullptr || key_weight != nullptr);
    if (status != TC_OK) return status;
    const tc_rotary_shape& a = *shape;
    if (a.tokens == 0) return TC_OK;
    if (a.query_heads > 0 && any_null({query, query_out})) return null_operand(what);
    if (a.key_heads > 0 && any_null({key, key_out})) return null_operand(what);
    TC_ROTARY_TYPES(a, what, {
        Rotary<S, W> r{};
        r.from[0] = static_cast<const S*>(query), r.from[1] = static_cast<const S*>(key);
        r.from_steps[0] = {a.query_token_step, a.query_head_step};
        r.from_steps[1] = {a.key_token_step, a.key_head_step};
        r.to[0] = static_cast<S*>(query_out), r.to[1] = static_cast<S*>(key_out);
        r.to_steps[0] = {a.query_out_token_step, a.query_out_head_step};
        r.to_steps[1] = {a.key_out_token_step, a.key_out_head_step};
        r.weight[0] = static_cast<const W*>(query_weight), r.weight[1] = static_cast<const W*>(key_weight);
        return rotary<S, W, false>(a, r, nullptr, nullptr, what);
    })
    return TC_OK;
}

int tc_rotary_norm_backward(const tc_rotary_shape* shape, const void* d_query_out, const void* d_key_out,
                            const void* query, const void* key, const void* query_weight, const void* key_weight,
                            void* d_query, void* d_key, void* d_query_weight, void* d_key_weight) {
    const char* what = "rotary norm, backward";
    const int status = check_rotary(
        what, shape,
        query_weight != nullptr || key_weight != nullptr || d_query_weight != nullptr || d_key_weight != nullptr);
    if (status != TC_OK) return status;
    const tc_rotary_shape& a = *shape;
    if (a.tokens == 0 && d_query_weight == nullptr && d_key_weight == nullptr) return TC_OK;
    if (a.tokens > 0 && a.query_heads > 0 &&
        (any_null({d_query_out, d_query}) || (a.normalize != 0 && query == nullptr))) {
        return null_operand(what);
    }
    if (a.tokens > 0 && a.key_heads > 0 && (any_null({d_key_out, d_key}) || (a.normalize != 0 && key == nullptr))) {
        return null_operand(what);
    }
    TC_ROTARY_TYPES(a, what, {
        Rotary<S, W> r{};
        r.from[0] = static_cast<const S*>(d_query_out), r.from[1] = static_cast<const S*>(d_key_out);
        r.from_steps[0] = {a.query_out_token_step, a.query_out_head_step};
        r.from_steps[1] = {a.key_out_token_step, a.key_out_head_step};
        r.x[0] = static_cast<const S*>(query), r.x[1] = static_cast<const S*>(key);
        r.to[0] = static_cast<S*>(d_query), r.to[1] = static_cast<S*>(d_key);
        r.x_steps[0] = r.to_steps[0] = {a.query_token_step, a.query_head_step};
        r.x_steps[1] = r.to_steps[1] = {a.key_token_step, a.key_head_step};
        r.weight[0] = static_cast<const W*>(query_weight), r.weight[1] = static_cast<const W*>(key_weight);
        return rotary<S, W, true>(a, r, static_cast<W*>(d_query_weight), static_cast<W*>(d_key_weight), what);
    })
    return TC_OK;
}

}  // extern "C"
