// Log probabilities of tokens, their entropy and the most probable ones, and
// the gradient of the logits.
//
// Of a row of logits x, with m the largest,
//   s = sum exp(x - m),  t = sum (x - m) exp(x - m),
//   l = m + log s                 the normalizer, log sum exp x
//   log p(j) = (x_j - m) - log s
//   H = log s - t / s             the entropy, -sum p log p
// all from one read of the row: a lane keeps m, s and t of what it has read
// and rescales s and t when m grows (t' = (t + s (m - m')) exp(m - m')), and
// the lanes', waves' and blocks' states are joined the same way, in a fixed
// order.
//
// The gradient, from g of log p(token) and h of H:
//   d_j = g (j == token) - p_j (g + h (log p_j + H)),  p_j = exp(x_j - l)
//
// Both are bound by memory, the forward pass at one read of the logits, the
// backward pass at one read and one write; forward the exponentials come to
// nearly as much.  Measured (a large copy moves 6.5 TB/s): 4096 bf16 rows of
// 100000, 819 MB, 151 us, with the top 8 192 to 197 and the top 64 270 (f16 159,
// 206 and 274); the gradient of 4096 bf16 rows of 50001, odd rows, 142 us,
// 5.8 TB/s; 16 f32 rows of 50001 with the top 20, split over 25 blocks each and
// joined, 12.7 us.  Rows are read in words that are 16-byte aligned wherever the
// row starts, its first and last elements one by one.  A block takes a row; few
// rows are split over several blocks each, and a second kernel joins them.
//
// The most probable tokens are kept by a 64-bit key, the logit's bits in
// order above the token's complement, so that equal logits go to the lowest
// token and no two keys are equal.  A block collects in LDS the keys that may
// be among its best: of the first batch those at or above a logit that enough
// lanes reach, then those above the last of the best so far, from which it
// selects after batches 1, 2, 4, 8 and every eighth, so that few keys pass
// and no batch waits for another.  Where they do not fit (logits that rise
// along the row, or thousands of equal ones) or are too few (fewer tokens
// possible than wanted), the block reads its part again, batch by batch: of a
// batch that would not fit, only keys at least as high as the k-th highest of
// the lanes' highest are taken, and those are in k lanes.

#include <type_traits>

#include "rows.hpp"

namespace tc {
namespace {

constexpr int kThreads = 256;
constexpr int kBatch = 4;  // words a lane reads at a time
constexpr uint32_t kMostTop = 64;
constexpr uint64_t kMostParts = 64;  // of a row
constexpr int kRoom = 3072;  // keys collected at most
// Collected keys beyond which a block selects: kRoom less a batch's most,
// kMostTop lanes of kBatch words of 8.
constexpr int kFull = kRoom - static_cast<int>(kMostTop) * kBatch * 8;
constexpr float kLog2e = 1.44269504088896340736f;

// ---- a row's state ----------------------------------------------------------------

struct State {
    float most = -INFINITY;  // m
    float sum = 0.0f;        // s
    float mean = 0.0f;       // t
};

__device__ __forceinline__ float power(float v) { return __builtin_amdgcn_exp2f(v * kLog2e); }

// Differences of logits below which a power is 0 in 32 bits, by far: larger
// ones are taken for this one where they are multiplied by such a power, which
// is 0 times infinity where the difference or its product with a sum overflows
// (logits masked with the type's lowest number, or with -infinity).
constexpr float kVanished = -1000.0f;

// The state with another m, not less than its own.
// A state of nothing but -infinity holds zeros (or the NaN of a NaN logit),
// which stay.
__device__ __forceinline__ void move(State& s, float to) {
    const float shift = s.most == -INFINITY ? 0.0f : fmaxf(s.most - to, kVanished);
    const float factor = power(shift);
    s.mean = fmaf(s.sum, shift, s.mean) * factor;
    s.sum *= factor;
    s.most = to;
}

// Joined over the block, in every lane; `shared` holds three floats a wave.
__device__ __forceinline__ State joined(State s, float (*shared)[kThreads / 64]) {
    move(s, wave64<Largest>(s.most));
    s.sum = wave64<Added>(s.sum);
    s.mean = wave64<Added>(s.mean);
    const int wave = threadIdx.x / 64;
    if (threadIdx.x % 64 == 0) shared[0][wave] = s.most, shared[1][wave] = s.sum, shared[2][wave] = s.mean;
    __syncthreads();
    State all{shared[0][0], shared[1][0], shared[2][0]};
    float most = all.most;
    for (int w = 1; w < kThreads / 64; w++) most = fmaxf(most, shared[0][w]);
    move(all, most);
    for (int w = 1; w < kThreads / 64; w++) {
        State other{shared[0][w], shared[1][w], shared[2][w]};
        move(other, most);
        all.sum += other.sum;
        all.mean += other.mean;
    }
    return all;
}

// ---- the order of logits ------------------------------------------------------------

// Whole numbers in the order of the floats, -0 as 0, a NaN below all.
__device__ __forceinline__ uint32_t ordered(float v) {
    const uint32_t bits = __float_as_uint(v + 0.0f);
    if (v != v) return 0;
    return bits >> 31 ? ~bits : bits | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t order) {
    return __uint_as_float(order >> 31 ? order & 0x7fffffffu : ~order);
}
__device__ __forceinline__ uint64_t key_of(float v, uint32_t token) {
    return static_cast<uint64_t>(ordered(v)) << 32 | ~token;
}
__device__ __forceinline__ float logit_of(uint64_t key) { return unordered(static_cast<uint32_t>(key >> 32)); }
__device__ __forceinline__ uint32_t token_of(uint64_t key) { return ~static_cast<uint32_t>(key); }

// The order of -infinity: of every logit that is no number above it.
constexpr uint32_t kLowest = 0x007fffff;

// The highest order of 16 bits, zeros below them, that `lanes` lanes of the
// wave reach (0: fewer have any logit), bit by bit.
__device__ __forceinline__ uint32_t reached_by(int lanes, uint32_t order) {
    uint32_t reached = 0;
    for (int bit = 31; bit >= 16; bit--) {
        const uint32_t next = reached | 1u << bit;
        if (__popcll(__ballot(order >= next)) >= lanes) reached = next;
    }
    return reached;
}

// The keys that a block has collected.
struct Keys {
    uint64_t keys[kRoom];
    uint64_t best[kMostTop];
    uint64_t highest[kThreads];  // of each lane's batch
    uint64_t lowest;             // of the batch's keys that are taken
    uint32_t reached[kThreads / 64];
    int count;
};

// How many of the keys are above `key`.  Eight are read at a time: one by one
// the reads' latency, not their number, is what a rank would take.
__device__ __forceinline__ int rank_among(const uint64_t* keys, int count, uint64_t key) {
    int rank = 0, j = 0;
    for (; j + 8 <= count; j += 8) {
        uint64_t other[8];
#pragma unroll
        for (int q = 0; q < 8; q++) other[q] = keys[j + q];
#pragma unroll
        for (int q = 0; q < 8; q++) rank += other[q] > key;
    }
    for (; j < count; j++) rank += keys[j] > key;
    return rank;
}

// The `top` highest of the collected keys, in order, are what is left of them.
__device__ void select(Keys& k, int count, int top) {
    for (int i = threadIdx.x; i < count; i += kThreads) {
        const uint64_t key = k.keys[i];
        const int rank = rank_among(k.keys, count, key);
        if (rank < top) k.best[rank] = key;
    }
    __syncthreads();
    const int left = count < top ? count : top;
    for (int i = threadIdx.x; i < left; i += kThreads) k.keys[i] = k.best[i];
    if (threadIdx.x == 0) k.count = left;
    __syncthreads();
}

// The `top` best keys of words first .. end of a row (or all, if fewer), in
// order, whatever the logits: every batch waits for the one before.
template <typename S, bool NT>
__device__ void collect_again(const Row<S>& row, uint64_t first, uint64_t end, int top, Keys& k) {
    constexpr int E = Row<S>::E;
    uint32_t least = 0;   // a logit's order has to be above it to be among the best
    bool enough = false;  // ... once there are `top` of them: later tokens lose ties
    int count = 0;
    if (threadIdx.x == 0) k.count = 0;
    __syncthreads();
    for (uint64_t from = first; from < end; from += kBatch * kThreads) {
        // `body(key)` of each element of the lane's batch that may be taken.
        const auto each = [&](auto&& body) {
            for (int u = 0; u < kBatch; u++) {
                const uint64_t word = from + u * kThreads + threadIdx.x;
                if (word >= end) break;
                const int64_t column = row.column(word);
                Words<S, E> words;
                row.template load<false>(word, words);
#pragma unroll
                for (int e = 0; e < E; e++) {
                    const float v = words.at(e);
                    if (row.has(column + e) && !(enough && ordered(v) <= least)) {
                        body(key_of(v, static_cast<uint32_t>(column + e)));
                    }
                }
            }
        };
        const auto put = [&](uint64_t key) {
            const int to = atomicAdd(&k.count, 1);
            if (to < kRoom) k.keys[to] = key;
        };
        const int before = count;
        if (enough) {
            each(put);
            __syncthreads();
            count = k.count;
            __syncthreads();
        }
        if (!enough || count > kRoom) {
            // Too many, or nothing yet to hold them against.
            uint64_t own = 0;
            each([&](uint64_t key) { own = key > own ? key : own; });
            k.highest[threadIdx.x] = own;
            if (threadIdx.x == 0) k.count = before, k.lowest = 0;
            __syncthreads();
            const int rank = rank_among(k.highest, kThreads, own);
            if (own != 0 && rank == top - 1) k.lowest = own;  // one lane at most: keys differ
            __syncthreads();
            const uint64_t lowest = k.lowest;
            each([&](uint64_t key) {
                if (key >= lowest) put(key);
            });
            __syncthreads();
            count = k.count;
            __syncthreads();
        }
        if (count > kFull || !enough) {
            select(k, count, top);
            count = count < top ? count : top;
            enough = count == top;
            if (enough) least = static_cast<uint32_t>(k.keys[top - 1] >> 32);
        }
    }
    select(k, count, top);
}

struct Results {
    const uint32_t* tokens;
    float* log_probabilities;
    float* normalizers;
    float* entropies;
    uint32_t top;
    float* top_log_probabilities;
    uint32_t* top_tokens;

    // Of the rows from `first` on.
    Results from(uint64_t first) const {
        const auto at = [&](auto* p, uint64_t each) { return p != nullptr ? p + first * each : nullptr; };
        return {at(tokens, 1), at(log_probabilities, 1), at(normalizers, 1), at(entropies, 1), top,
                at(top_log_probabilities, top), at(top_tokens, top)};
    }
};

// log p of a logit from the row's state.
__device__ __forceinline__ float log_probability(const State& s, float logit) {
    if (s.most == -INFINITY && s.sum == 0.0f) return -INFINITY;  // nothing is possible
    return (logit - s.most) - logf(s.sum);
}

// The logit of the row's token, `*some` false where it has none; read before the row
// is, so that the results do not wait for it.
template <typename S>
__device__ __forceinline__ float given_logit(const S* row, uint64_t cols, uint64_t at, const Results& out, bool* some) {
    const uint32_t token = out.tokens != nullptr ? out.tokens[at] : ~0u;
    *some = token < cols;
    return *some ? Elem<S>::widen(row[token]) : 0.0f;
}

// One lane writes the row's results.
__device__ void finish(const State& s, float logit, bool some, uint64_t at, const Results& out) {
    const bool none = s.most == -INFINITY && s.sum == 0.0f;
    if (out.normalizers != nullptr) out.normalizers[at] = none ? -INFINITY : s.most + logf(s.sum);
    if (out.entropies != nullptr) out.entropies[at] = none ? 0.0f : logf(s.sum) - s.mean / s.sum;
    if (out.log_probabilities != nullptr) out.log_probabilities[at] = some ? log_probability(s, logit) : 0.0f;
}

// A block takes part blockIdx % parts, of `part_words` words, of row
// blockIdx / parts.  With one part the results are written here.
template <typename S, bool TOP, bool NT>
__global__ void __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(TOP ? 5 : 6)))
    tokens_kernel(const S* logits, uint64_t step, uint64_t cols, uint32_t parts, uint64_t part_words,
                  Results out, State* left, uint64_t* left_keys) {
    constexpr int E = kWordElements<S>;
    __shared__ float shared[3][kThreads / 64];
    __shared__ std::conditional_t<TOP, Keys, char> keys;
    (void)keys;
    const uint64_t at = blockIdx.x / parts;
    const uint32_t part = blockIdx.x % parts;
    const Row<S> row(logits + at * step, cols);
    const uint64_t first = part * part_words;
    const uint64_t words = row.words();
    const uint64_t end = first + part_words < words ? first + part_words : words;
    const int top = TOP ? static_cast<int>(out.top) : 0;

    bool some;
    const float logit = given_logit(row.row, cols, at, out, &some);
    State state;
    float least = -INFINITY;  // a logit has to be above it to be collected
    bool fits = true;         // what was collected
    if constexpr (TOP) {
        if (threadIdx.x == 0) keys.count = 0;
    }

    Words<S, E> next[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; u++) {
        const uint64_t word = first + u * kThreads + threadIdx.x;
        if (word < end) row.template load<NT>(word, next[u]);
    }
    uint32_t batch = 0;
    for (uint64_t from = first; from < end; from += kBatch * kThreads) {
        float value[kBatch][E];
        float highest[kBatch], most = -INFINITY;
#pragma unroll
        for (int u = 0; u < kBatch; u++) {
            const uint64_t word = from + u * kThreads + threadIdx.x;
            if (word < end) {
                next[u].get(value[u]);
            } else {
#pragma unroll
                for (int e = 0; e < E; e++) value[u][e] = -INFINITY;
            }
            highest[u] = -INFINITY;
#pragma unroll
            for (int e = 0; e < E; e++) highest[u] = fmaxf(highest[u], value[u][e]);
            most = fmaxf(most, highest[u]);
            const uint64_t later = word + kBatch * kThreads;
            if (later < end) row.template load<NT>(later, next[u]);
        }
        if (most > state.most) move(state, most);
        const float origin = state.most == -INFINITY ? 0.0f : state.most;
#pragma unroll
        for (int u = 0; u < kBatch; u++) {
#pragma unroll
            for (int e = 0; e < E; e++) {
                const float d = value[u][e] - origin;
                const float p = power(d);
                state.sum += p;
                state.mean = fmaf(fmaxf(d, kVanished), p, state.mean);
            }
        }
        if constexpr (TOP) {
            if (batch++ == 0) {
                // The least of the waves' logits that a wave's share of the
                // top is at or above: `top` lanes' highest are.
                const uint32_t reached = reached_by((top + kThreads / 64 - 1) / (kThreads / 64), ordered(most));
                if (threadIdx.x % 64 == 0) keys.reached[threadIdx.x / 64] = reached;
                __syncthreads();
                uint32_t all = keys.reached[0];
                for (int w = 1; w < kThreads / 64; w++) all = keys.reached[w] < all ? keys.reached[w] : all;
                if (all > kLowest) least = unordered(all - 1);
            }
            if (fits && most > least) {
#pragma unroll
                for (int u = 0; u < kBatch; u++) {
                    if (!(highest[u] > least)) continue;
                    int to = 0;
#pragma unroll
                    for (int e = 0; e < E; e++) to += value[u][e] > least;
                    to = atomicAdd(&keys.count, to);
                    const uint32_t column = static_cast<uint32_t>(row.column(from + u * kThreads + threadIdx.x));
#pragma unroll
                    for (int e = 0; e < E; e++) {
                        if (!(value[u][e] > least)) continue;
                        if (to < kRoom) keys.keys[to] = key_of(value[u][e], column + e);
                        to++;
                    }
                }
            }
            if ((batch & (batch - 1)) == 0 || batch % 8 == 0) {
                __syncthreads();
                const int count = keys.count;
                __syncthreads();
                fits = count <= kRoom;
                if (fits && count >= top) {
                    select(keys, count, top);
                    least = logit_of(keys.keys[top - 1]);
                }
            }
        }
    }
    state = joined(state, shared);
    if constexpr (TOP) {
        __syncthreads();
        int count = keys.count;
        __syncthreads();
        if (count < top || count > kRoom) {
            collect_again<S, NT>(row, first, end, top, keys);
            count = keys.count;
        } else {
            select(keys, count, top);
            count = top;
        }
        for (int i = threadIdx.x; i < top; i += kThreads) {
            if (parts == 1) {
                out.top_log_probabilities[at * top + i] = log_probability(state, logit_of(keys.keys[i]));
                out.top_tokens[at * top + i] = token_of(keys.keys[i]);
            } else {
                left_keys[static_cast<uint64_t>(blockIdx.x) * top + i] = i < count ? keys.keys[i] : 0;
            }
        }
    }
    if (threadIdx.x != 0) return;
    if (parts == 1) {
        finish(state, logit, some, at, out);
    } else {
        left[blockIdx.x] = state;
    }
}

// A row's parts joined: a block a row.  Each part's keys are in order, so if
// the j-th of n parts is at or above a bound, j n keys are: with j n at least
// `top`, no key below it is among the row's, and few are above it.
template <typename S>
__global__ void __launch_bounds__(kThreads)
    join_tokens_kernel(const S* logits, uint64_t step, uint64_t cols, uint32_t parts, Results out, const State* left,
                       const uint64_t* left_keys) {
    __shared__ float shared[3][kThreads / 64];
    __shared__ uint64_t keys[kMostParts * kMostTop];
    __shared__ int survivors;
    const uint64_t at = blockIdx.x;
    const uint32_t top = out.top;
    // Everything that is read is on its way before anything is worked on.
    bool some;
    const float logit = given_logit(logits + at * step, cols, at, out, &some);
    State state;
    if (threadIdx.x < parts) state = left[at * parts + threadIdx.x];
    uint64_t mine[kMostParts * kMostTop / kThreads];
    const uint32_t depth = (top + parts - 1) / parts, part = threadIdx.x % 64;
    const uint64_t jth = top > 0 && part < parts ? left_keys[(at * parts + part) * top + depth - 1] : 0;
#pragma unroll
    for (int k = 0; k < static_cast<int>(kMostParts * kMostTop) / kThreads; k++) {
        const uint32_t i = threadIdx.x + k * kThreads;
        mine[k] = i < parts * top ? left_keys[at * parts * top + i] : 0;
    }
    if (threadIdx.x == 0) survivors = 0;
    state = joined(state, shared);
    if (threadIdx.x == 0) finish(state, logit, some, at, out);
    if (top == 0) return;
    const uint32_t reached =
        reached_by(static_cast<int>((top + depth - 1) / depth), static_cast<uint32_t>(jth >> 32));
    const uint64_t lowest = reached > 0 ? static_cast<uint64_t>(reached) << 32 : 1;  // 0 is no key
#pragma unroll
    for (const uint64_t key : mine) {
        if (key >= lowest) keys[atomicAdd(&survivors, 1)] = key;
    }
    __syncthreads();
    const int count = survivors;
    for (int i = threadIdx.x; i < count; i += kThreads) {
        const uint64_t key = keys[i];
        const uint32_t rank = static_cast<uint32_t>(rank_among(keys, count, key));
        if (rank >= top) continue;
        out.top_log_probabilities[at * top + rank] = log_probability(state, logit_of(key));
        out.top_tokens[at * top + rank] = token_of(key);
    }
}

// ---- the gradient ----------------------------------------------------------------------

struct Gradients {
    const uint32_t* tokens;
    const float* normalizers;
    const float* entropies;
    const float* d_log_probabilities;
    const float* d_entropies;

    // Of the rows from `first` on.
    Gradients from(uint64_t first) const {
        const auto at = [&](auto* p) { return p != nullptr ? p + first : nullptr; };
        return {at(tokens), at(normalizers), at(entropies), at(d_log_probabilities), at(d_entropies)};
    }
};

// A block takes kBatch words a lane of a row.  Every element is read and
// written by the same lane, so the gradient may take the logits' place.
template <typename S, bool ENTROPY, bool NT>
__global__ void __launch_bounds__(kThreads)
    tokens_back_kernel(const S* logits, uint64_t step, uint64_t cols, uint32_t parts, Gradients in, S* d_logits,
                       uint64_t d_step) {
    constexpr int E = kWordElements<S>;
    const uint64_t at = blockIdx.x / parts;
    const uint64_t first = static_cast<uint64_t>(blockIdx.x % parts) * kBatch * kThreads + threadIdx.x;
    const Row<S> row(logits + at * step, cols);
    S* to = d_logits + at * d_step;
    const uint64_t words = row.words();

    const float normalizer = in.normalizers[at];
    const uint32_t token = in.d_log_probabilities != nullptr ? in.tokens[at] : ~0u;
    const float g = token < cols ? in.d_log_probabilities[at] : 0.0f;
    const float h = ENTROPY ? in.d_entropies[at] : 0.0f;
    // -p (g + h (log p + H)) = p (base + slope log p)
    const float base = ENTROPY ? -(g + h * in.entropies[at]) : -g, slope = -h;
    // A row that nothing asks of, or that has nothing possible, has no gradient.
    const bool none = (g == 0.0f && h == 0.0f) || normalizer == -INFINITY;

    Words<S, E> in_words[kBatch];
    if (!none) {
#pragma unroll
        for (int u = 0; u < kBatch; u++) {
            if (first + u * kThreads < words) row.template load<NT>(first + u * kThreads, in_words[u]);
        }
    }
#pragma unroll
    for (int u = 0; u < kBatch; u++) {
        const uint64_t word = first + u * kThreads;
        if (word >= words) break;
        const int64_t column = row.column(word);
        float v[E];
        if (none) {
#pragma unroll
            for (int e = 0; e < E; e++) v[e] = 0.0f;
        } else {
            in_words[u].get(v);
#pragma unroll
            for (int e = 0; e < E; e++) {
                const float log_p = v[e] - normalizer;
                const float p = power(log_p);
                v[e] = ENTROPY ? p * fmaf(slope, fmaxf(log_p, kVanished), base) : p * base;
            }
            const int64_t place = static_cast<int64_t>(token) - column;
            if (g != 0.0f && place >= 0 && place < E) {
#pragma unroll
                for (int e = 0; e < E; e++) v[e] += e == place ? g : 0.0f;
            }
        }
        row.template store<NT>(word, to, v);
    }
}

// ---- launches ------------------------------------------------------------------------------

// A dispatch holds fewer than 2^32 work-items: rows beyond that many blocks
// take another launch.
constexpr uint64_t kMostBlocks = 0xffffffffu / kThreads;

// `call(first row, rows)` over all rows in turn, `parts` blocks a row.
template <typename Call>
int in_launches(uint64_t rows, uint64_t parts, Call&& call) {
    const uint64_t most = kMostBlocks / parts;
    for (uint64_t first = 0; first < rows; first += most) {
        const int status = call(first, rows - first < most ? rows - first : most);
        if (status != TC_OK) return status;
    }
    return TC_OK;
}

template <typename S>
int tokens(const S* logits, uint64_t step, uint64_t rows, uint64_t cols, const Results& out) {
    TC_STREAM(s);
    const uint64_t words = (cols + 2 * kWordElements<S> - 2) / kWordElements<S>;  // at most, wherever a row starts
    // As many parts as give every compute unit four blocks, of two words a
    // lane at least.
    const uint64_t wanted = (static_cast<uint64_t>(compute_units()) * 4 + rows - 1) / rows;
    const uint64_t most = (words + 2 * kThreads - 1) / (2 * kThreads);
    uint64_t parts = wanted < most ? wanted : most;
    if (parts > kMostParts) parts = kMostParts;
    const uint64_t part_words = ((words + parts - 1) / parts + kThreads - 1) / kThreads * kThreads;
    parts = (words + part_words - 1) / part_words;
    Scratch left(parts > 1 ? rows * parts * sizeof(State) : 0);
    Scratch left_keys(parts > 1 ? rows * parts * out.top * sizeof(uint64_t) : 0);
    if (left.status != TC_OK) return left.status;
    if (left_keys.status != TC_OK) return left_keys.status;
    State* states = static_cast<State*>(left.ptr);
    uint64_t* keys = static_cast<uint64_t*>(left_keys.ptr);
    const bool streams = sizeof(S) * rows * cols >= kStreamBytes;
    return in_launches(rows, parts, [&](uint64_t first, uint64_t count) {
        const Results here = out.from(first);
        const S* from = logits + first * step;
        const auto launch = [&](auto kernel) {
            kernel<<<static_cast<uint32_t>(count * parts), kThreads, 0, s>>>(
                from, step, cols, static_cast<uint32_t>(parts), part_words, here, states, keys);
        };
        if (out.top > 0) {
            if (streams) launch(tokens_kernel<S, true, true>);
            else launch(tokens_kernel<S, true, false>);
        } else {
            if (streams) launch(tokens_kernel<S, false, true>);
            else launch(tokens_kernel<S, false, false>);
        }
        const int status = check_launch("log probabilities");
        if (status != TC_OK || parts == 1) return status;
        join_tokens_kernel<S><<<static_cast<uint32_t>(count), kThreads, 0, s>>>(
            from, step, cols, static_cast<uint32_t>(parts), here, states, keys);
        return check_launch("log probabilities");
    });
}

template <typename S>
int tokens_back(const S* logits, uint64_t step, uint64_t rows, uint64_t cols, const Gradients& in, S* d_logits,
                uint64_t d_step) {
    TC_STREAM(s);
    const uint64_t words = (cols + 2 * kWordElements<S> - 2) / kWordElements<S>;
    const uint64_t parts = (words + kBatch * kThreads - 1) / (kBatch * kThreads);
    const bool streams = 2 * sizeof(S) * rows * cols >= kStreamBytes;
    return in_launches(rows, parts, [&](uint64_t first, uint64_t count) {
        const Gradients here = in.from(first);
        const auto launch = [&](auto kernel) {
            kernel<<<static_cast<uint32_t>(count * parts), kThreads, 0, s>>>(
                logits + first * step, step, cols, static_cast<uint32_t>(parts), here, d_logits + first * d_step,
                d_step);
        };
        if (in.d_entropies != nullptr) {
            if (streams) launch(tokens_back_kernel<S, true, true>);
            else launch(tokens_back_kernel<S, true, false>);
        } else {
            if (streams) launch(tokens_back_kernel<S, false, true>);
            else launch(tokens_back_kernel<S, false, false>);
        }
        return check_launch("log probabilities, backward");
    });
}

int check_tokens(const std::string& what, uint32_t dtype, uint64_t rows, uint64_t cols,
                 std::initializer_list<uint64_t> steps) {
    if (dtype_size(dtype) == 0 || dtype == TC_F64) return fail(TC_UNSUPPORTED, what + ": no kernel for " + dtype_name(dtype));
    if (cols >= 0xffffffffu) {
        return fail(TC_UNSUPPORTED, what + ": a token of 32 bits does not reach " + std::to_string(cols) + " logits");
    }
    for (uint64_t step : steps) {
        if (rows > 1 && step < cols) {
            return fail(TC_INVALID, what + ": rows of " + std::to_string(cols) + " elements " + std::to_string(step) +
                                        " apart overlap");
        }
        if (rows > 0 && step > UINT64_MAX / 8 / rows) {
            return fail(TC_INVALID, what + ": " + std::to_string(rows) + " rows " + std::to_string(step) +
                                        " apart reach past the address space");
        }
    }
    return TC_OK;
}

}  // namespace
}  // namespace tc

using namespace tc;

extern "C" {

int tc_log_probabilities(uint32_t dtype, const void* logits, uint64_t step, uint64_t rows, uint64_t cols,
                         const uint32_t* tokens, float* log_probabilities, float* normalizers, float* entropies,
                         uint32_t top, float* top_log_probabilities, uint32_t* top_tokens) {
    const char* what = "log probabilities";
    const int status = check_tokens(what, dtype, rows, cols, {step});
    if (status != TC_OK) return status;
    if (top > kMostTop) {
        return fail(TC_UNSUPPORTED, std::string(what) + ": the top " + std::to_string(top) + " of at most " +
                                        std::to_string(kMostTop));
    }
    if (top > cols) {
        return fail(TC_INVALID, std::string(what) + ": the top " + std::to_string(top) + " of " + std::to_string(cols) +
                                    " logits");
    }
    if (rows == 0) return TC_OK;
    if (cols == 0) return fail(TC_INVALID, std::string(what) + ": rows of no logits");
    if (logits == nullptr || (tokens == nullptr) != (log_probabilities == nullptr) ||
        (top > 0 && any_null({top_log_probabilities, top_tokens}))) {
        return null_operand(what);
    }
    const Results out{tokens, log_probabilities, normalizers, entropies, top, top_log_probabilities, top_tokens};
    TC_DISPATCH_FLOAT(dtype, what, S, return ::tc::tokens<S>(static_cast<const S*>(logits), step, rows, cols, out))
    return TC_OK;
}

int tc_log_probabilities_backward(uint32_t dtype, const void* logits, uint64_t step, uint64_t rows, uint64_t cols,
                                  const uint32_t* tokens, const float* normalizers, const float* entropies,
                                  const float* d_log_probabilities, const float* d_entropies, void* d_logits,
                                  uint64_t d_step) {
    const char* what = "log probabilities, backward";
    const int status = check_tokens(what, dtype, rows, cols, {step, d_step});
    if (status != TC_OK) return status;
    if (rows == 0) return TC_OK;
    if (cols == 0) return fail(TC_INVALID, std::string(what) + ": rows of no logits");
    if (any_null({logits, normalizers, d_logits}) || (d_log_probabilities != nullptr && tokens == nullptr) ||
        (d_entropies != nullptr && entropies == nullptr)) {
        return null_operand(what);
    }
    const Gradients in{tokens, normalizers, entropies, d_log_probabilities, d_entropies};
    TC_DISPATCH_FLOAT(dtype, what, S, return tokens_back<S>(static_cast<const S*>(logits), step, rows, cols, in,
                                                           static_cast<S*>(d_logits), d_step))
    return TC_OK;
}

}  // extern "C"
