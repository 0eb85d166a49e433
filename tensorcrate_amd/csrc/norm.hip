// Layer norm of rows and its gradients.
//
// Forward, of a row x of n elements, with weight w and bias b:
//   m = mean(x),  s = 1 / sqrt(mean((x - m)^2) + epsilon),  y = (x - m) s w + b
// Backward, with u = (x - m) s and g = dy w:
//   dx = s (g - mean(g) - u mean(g u)),  dw = sum over rows dy u,
//   db = sum over rows dy
// Both are bound by memory: the forward pass reads x once and writes y once,
// the backward pass reads dy and x once and writes dx once.  So a row is held
// in registers from its one read on, by 16 lanes, a wave or a block, and the
// variance is the second sum over those registers (exact about the mean, where
// a sum of squares would cancel).  A group of lanes walks rows a grid apart
// with the next row's words already in flight, and keeps its columns' weights.
//
// Measured (a large copy moves 6.5 TB/s): 16384 bf16 rows of 4096 forward
// 47 us, 5.7 TB/s, and backward 89, 4.5 TB/s; 10007 f16 rows of 2050, views that
// start at any element, with an f32 weight, backward 40 us, 3.1 TB/s: 33.5 at
// 2048 columns (3.7), 4 more for the fifth word of a lane that two columns more
// take, 3 for the odd starts.  4 to 5 of each are the launch that adds dw and
// db.  With an f16 weight those rows take 55 us, since that form keeps some 25
// of a lane's words in memory.  8192 f32 rows of 4096 backward 79 us, 5.1 TB/s;
// 64 of 1024 forward the 4 us of a launch.
// One word a lane instead of two and grids that fill the chip without walking
// rows took 68 and 52 us forward; one row a block backward 47.
//
// dw and db are sums over all rows: a lane sums its columns over the rows of
// its walk in registers, each block writes those sums once, and a second
// kernel adds the blocks' in block order, so the result does not depend on
// timing.  Everything is summed in f32 and rounded to its type once.

#include "rows.hpp"

namespace tc {
namespace {

constexpr uint32_t kMostLanes = 1024;  // of a block
constexpr uint32_t kBackThreads = 512;  // at most, backward, whose sums over rows fill the registers
// Elements of a row that one lane of a block holds at most.
constexpr int kForwardHeld = 16, kBackHeld = 32;

// The columns that one lane of a row holds: VECTORS words a row's lanes apart.
// The layout leaves no word but a lane's last one ragged or past the row's
// end, so that only the last is checked.
template <int E, int VECTORS>
struct Held {
    uint64_t first;   // column of the lane's first word
    uint64_t apart;   // columns between its words
    Run<E> last;

    __device__ __forceinline__ Held(uint32_t lane, uint32_t lanes, uint64_t cols)
        : first(uint64_t{lane} * E),
          apart(uint64_t{lanes} * E),
          last(lane + uint64_t{lanes} * (VECTORS - 1), cols) {}
    __device__ __forceinline__ bool live(int v) const { return v < VECTORS - 1 || last.live(); }
    __device__ __forceinline__ bool partial(int v) const { return v == VECTORS - 1 && last.partial(); }
    __device__ __forceinline__ bool own(int v, int e) const { return v < VECTORS - 1 || last.own(e); }
    __device__ __forceinline__ uint64_t column(int v) const {
        return v < VECTORS - 1 ? first + v * apart : last.start;
    }

    template <bool NT, typename T>
    __device__ __forceinline__ void load(const T* row, Words<T, E> (&words)[VECTORS]) const {
#pragma unroll
        for (int v = 0; v < VECTORS - 1; v++) words[v].template load<NT>(row + first + v * apart);
        if (last.live()) last.template load<NT>(row, words[VECTORS - 1]);
    }
    template <bool NT, typename T>
    __device__ __forceinline__ void store(T* row, int v, const float (&value)[E]) const {
        if (v < VECTORS - 1) {
            Words<T, E> words;
            words.put(value);
            words.template store<NT>(row + first + v * apart);
        } else {
            last.template store<NT>(row, value);
        }
    }
};

// LANES lanes a row: 16 or 64, several rows a block, or 0 for the block.
template <typename S, typename W, int LANES, int VECTORS, bool NT>
__global__ void __launch_bounds__(LANES ? 256 : kMostLanes)
    norm_kernel(const S* x, uint64_t x_step, uint64_t rows, uint64_t cols, const W* weight, const W* bias,
                float epsilon, S* y, uint64_t y_step, float* means, float* scales) {
    constexpr int E = kWordElements<S>;
    __shared__ float shared[2][kMostWaves];
    const uint32_t lanes = LANES ? LANES : blockDim.x;
    const uint32_t lane = threadIdx.x % lanes;
    const uint64_t groups = static_cast<uint64_t>(gridDim.x) * (blockDim.x / lanes);
    uint64_t row = static_cast<uint64_t>(blockIdx.x) * (blockDim.x / lanes) + threadIdx.x / lanes;
    if (row >= rows) return;  // the whole group

    const Held<E, VECTORS> held(lane, lanes, cols);
    Words<W, E> w[VECTORS], b[VECTORS];
    if (weight != nullptr) held.template load<false>(weight, w);
    if (bias != nullptr) held.template load<false>(bias, b);

    const float count = static_cast<float>(cols);
    Words<S, E> next[VECTORS];
    held.template load<NT>(x + row * x_step, next);
    for (; row < rows; row += groups) {
        float value[VECTORS][E];
        float sum = 0.0f;
#pragma unroll
        for (int v = 0; v < VECTORS; v++) {
            if (!held.live(v)) continue;
            next[v].get(value[v]);
            float part = 0.0f;
#pragma unroll
            for (int e = 0; e < E; e++) part += value[v][e];
            if (held.partial(v)) {
                part = 0.0f;
#pragma unroll
                for (int e = 0; e < E; e++) part += held.own(v, e) ? value[v][e] : 0.0f;
            }
            sum += part;
        }
        if (row + groups < rows) held.template load<NT>(x + (row + groups) * x_step, next);
        const float mean = row_join<LANES, Added>(sum, shared[0]) / count;
        float squares = 0.0f;
#pragma unroll
        for (int v = 0; v < VECTORS; v++) {
            if (!held.live(v)) continue;
            float part = 0.0f;
#pragma unroll
            for (int e = 0; e < E; e++) {
                value[v][e] -= mean;
                part = fmaf(value[v][e], value[v][e], part);
            }
            if (held.partial(v)) {
                part = 0.0f;
#pragma unroll
                for (int e = 0; e < E; e++) part += held.own(v, e) ? value[v][e] * value[v][e] : 0.0f;
            }
            squares += part;
        }
        const float scale = 1.0f / sqrtf(row_join<LANES, Added>(squares, shared[1]) / count + epsilon);
#pragma unroll
        for (int v = 0; v < VECTORS; v++) {
            if (!held.live(v)) continue;
#pragma unroll
            for (int e = 0; e < E; e++) {
                value[v][e] *= scale;
                if (weight != nullptr) value[v][e] *= w[v].at(e);
                if (bias != nullptr) value[v][e] += b[v].at(e);
            }
            held.template store<NT>(y + row * y_step, v, value[v]);
        }
        if (lane == 0) {
            if (means != nullptr) means[row] = mean;
            if (scales != nullptr) scales[row] = scale;
        }
    }
}

// Rows longer than a block's registers: a block a row, which it reads three
// times (from the caches, mostly).  Elements are read and written one by one
// at a row's ragged end, so that y may be x.  2000 bf16 rows of 40000: 225 us,
// 1.4 TB/s, and 418 backward, 1.1 TB/s.
template <typename S, typename W>
__global__ void __launch_bounds__(kMostLanes)
    norm_long_kernel(const S* x, uint64_t x_step, uint64_t rows, uint64_t cols, const W* weight, const W* bias,
                     float epsilon, S* y, uint64_t y_step, float* means, float* scales) {
    constexpr int E = kWordElements<S>;
    __shared__ float shared[2][kMostWaves];
    const uint64_t whole = cols / E * E;
    const float count = static_cast<float>(cols);
    for (uint64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const S* from = x + row * x_step;
        S* to = y + row * y_step;
        const auto each = [&](auto&& body) {
            for (uint64_t at = static_cast<uint64_t>(threadIdx.x) * E; at < whole; at += uint64_t{blockDim.x} * E) {
                Words<S, E> words;
                words.template load<false>(from + at);
                float v[E];
                words.get(v);
                body(at, v, E);
            }
            if (threadIdx.x < cols - whole) {
                float v[E] = {Elem<S>::widen(from[whole + threadIdx.x])};
                body(whole + threadIdx.x, v, 1);
            }
        };
        float sum = 0.0f;
        each([&](uint64_t, float (&v)[E], int n) {
#pragma unroll
            for (int e = 0; e < E; e++) sum += e < n ? v[e] : 0.0f;
        });
        const float mean = block_join<Added>(sum, shared[0]) / count;
        float squares = 0.0f;
        each([&](uint64_t, float (&v)[E], int n) {
#pragma unroll
            for (int e = 0; e < E; e++) squares += e < n ? (v[e] - mean) * (v[e] - mean) : 0.0f;
        });
        const float scale = 1.0f / sqrtf(block_join<Added>(squares, shared[1]) / count + epsilon);
        each([&](uint64_t at, float (&v)[E], int n) {
#pragma unroll
            for (int e = 0; e < E; e++) {
                if (e >= n) continue;
                v[e] = (v[e] - mean) * scale;
                if (weight != nullptr) v[e] *= Elem<W>::widen(weight[at + e]);
                if (bias != nullptr) v[e] += Elem<W>::widen(bias[at + e]);
            }
            if (n == E) {
                Words<S, E> words;
                words.put(v);
                words.template store<false>(to + at);
            } else {
                to[at] = Elem<S>::narrow(v[0]);
            }
        });
        if (threadIdx.x == 0) {
            if (means != nullptr) means[row] = mean;
            if (scales != nullptr) scales[row] = scale;
        }
    }
}

// The gradients.  `partial` (null if neither dw nor db is wanted) holds, for
// each block, cols sums of dy u and then cols sums of dy.
template <typename S, typename W, int LANES, int VECTORS, bool NT>
__global__ void __launch_bounds__(kBackThreads)
    norm_back_kernel(const S* dy, uint64_t dy_step, const S* x, uint64_t x_step,
                     uint64_t rows, uint64_t cols, const W* weight, const float* __restrict__ means,
                     const float* __restrict__ scales, S* dx, uint64_t dx_step, float* __restrict__ partial) {
    constexpr int E = kWordElements<S>;
    __shared__ float shared[2][2][kMostWaves];
    const uint32_t lanes = LANES ? LANES : blockDim.x;
    const uint32_t lane = threadIdx.x % lanes;
    const uint64_t groups = static_cast<uint64_t>(gridDim.x) * (blockDim.x / lanes);
    uint64_t row = static_cast<uint64_t>(blockIdx.x) * (blockDim.x / lanes) + threadIdx.x / lanes;

    const Held<E, VECTORS> held(lane, lanes, cols);
    // The weight's columns: in registers, or for a wave's longer rows in LDS,
    // the same for every wave.
    constexpr bool SHARED_WEIGHT = LANES == 64 && VECTORS > 2;
    __shared__ uint4 weights[SHARED_WEIGHT ? VECTORS * Words<W, E>::kCount * 64 : 1];
    Words<W, E> w[SHARED_WEIGHT ? 1 : VECTORS];
    if constexpr (SHARED_WEIGHT) {
        if (weight != nullptr && threadIdx.x < 64) {
            Words<W, E> all[VECTORS];
            held.template load<false>(weight, all);
#pragma unroll
            for (int v = 0; v < VECTORS; v++) {
#pragma unroll
                for (int k = 0; k < Words<W, E>::kCount; k++) {
                    weights[(v * Words<W, E>::kCount + k) * 64 + lane] = all[v].w[k];
                }
            }
        }
        __syncthreads();
    } else {
        if (weight != nullptr) held.template load<false>(weight, w);
    }
    const auto weight_words = [&](int v) {
        if constexpr (SHARED_WEIGHT) {
            Words<W, E> out;
#pragma unroll
            for (int k = 0; k < Words<W, E>::kCount; k++) {
                out.w[k] = weights[(v * Words<W, E>::kCount + k) * 64 + lane];
            }
            return out;
        } else {
            return w[v];
        }
    };
    float dw[VECTORS][E] = {}, db[VECTORS][E] = {};

    Words<S, E> next_x[VECTORS], next_dy[VECTORS];
    float next_mean = 0.0f, next_scale = 0.0f;
    const auto fetch = [&](uint64_t at) {
        held.template load<NT>(x + at * x_step, next_x);
        held.template load<NT>(dy + at * dy_step, next_dy);
        next_mean = means[at];
        next_scale = scales[at];
    };
    // The next row's words are in flight while this one's are worked on.
    constexpr bool KEPT = VECTORS * E > (LANES ? 32 : 16);
    if (row < rows) fetch(row);
    int turn = 0;
    for (; row < rows; row += groups) {
        const float mean = next_mean, scale = next_scale;
        // u and g of a word, from dy, x and the weight as they are stored.
        // Where a lane holds many words it keeps those for the second pass
        // rather than the 32-bit values, which would not fit its registers.
        float u[KEPT ? 1 : VECTORS][E], g[KEPT ? 1 : VECTORS][E];
        Words<S, E> now_x[KEPT ? VECTORS : 1], now_dy[KEPT ? VECTORS : 1];
        float sum = 0.0f, along = 0.0f;
#pragma unroll
        for (int v = 0; v < VECTORS; v++) {
            if (!held.live(v)) continue;
            float(&uv)[E] = u[KEPT ? 0 : v];
            float(&gv)[E] = g[KEPT ? 0 : v];
            if constexpr (KEPT) now_x[v] = next_x[v], now_dy[v] = next_dy[v];
            next_x[v].get(uv);
            next_dy[v].get(gv);
            Words<W, E> here;
            if (weight != nullptr) here = weight_words(v);
            if (held.partial(v)) {
                // A neighbour's elements and those past a short row add
                // nothing to the sums.
                float one = 0.0f, two = 0.0f;
#pragma unroll
                for (int e = 0; e < E; e++) {
                    uv[e] = (uv[e] - mean) * scale;
                    if (held.own(v, e)) {
                        dw[v][e] = fmaf(gv[e], uv[e], dw[v][e]);
                        db[v][e] += gv[e];
                    }
                    if (weight != nullptr) gv[e] *= here.at(e);
                    if (held.own(v, e)) {
                        one += gv[e];
                        two = fmaf(gv[e], uv[e], two);
                    }
                }
                sum += one;
                along += two;
            } else {
#pragma unroll
                for (int e = 0; e < E; e++) {
                    uv[e] = (uv[e] - mean) * scale;
                    dw[v][e] = fmaf(gv[e], uv[e], dw[v][e]);
                    db[v][e] += gv[e];
                    if (weight != nullptr) gv[e] *= here.at(e);
                    sum += gv[e];
                    along = fmaf(gv[e], uv[e], along);
                }
            }
        }
        if (row + groups < rows) fetch(row + groups);
        if (dx == nullptr) continue;
        if constexpr (LANES == 0) {
            // Both sums past one barrier, in buffers that alternate.
            sum = wave64<Added>(sum);
            along = wave64<Added>(along);
            const int waves = blockDim.x / 64;
            if (waves > 1) {
                float(&at)[2][kMostWaves] = shared[turn];
                turn ^= 1;
                if (threadIdx.x % 64 == 0) {
                    at[0][threadIdx.x / 64] = sum;
                    at[1][threadIdx.x / 64] = along;
                }
                __syncthreads();
                sum = at[0][0];
                along = at[1][0];
                for (int k = 1; k < waves; k++) {
                    sum += at[0][k];
                    along += at[1][k];
                }
            }
        } else {
            sum = row_join<LANES, Added>(sum, nullptr);
            along = row_join<LANES, Added>(along, nullptr);
        }
        const float mean_g = sum / static_cast<float>(cols), mean_gu = along / static_cast<float>(cols);
#pragma unroll
        for (int v = 0; v < VECTORS; v++) {
            if (!held.live(v)) continue;
            float(&uv)[E] = u[KEPT ? 0 : v];
            float(&gv)[E] = g[KEPT ? 0 : v];
            if constexpr (KEPT) {
                now_x[v].get(uv);
                now_dy[v].get(gv);
                Words<W, E> here;
                if (weight != nullptr) here = weight_words(v);
#pragma unroll
                for (int e = 0; e < E; e++) {
                    uv[e] = (uv[e] - mean) * scale;
                    if (weight != nullptr) gv[e] *= here.at(e);
                }
            }
#pragma unroll
            for (int e = 0; e < E; e++) gv[e] = scale * (gv[e] - mean_g - uv[e] * mean_gu);
            held.template store<NT>(dx + row * dx_step, v, gv);
        }
    }
    if (partial == nullptr) return;

    // The block's groups hold the same columns: halves added to halves.
    if constexpr (LANES != 0) {
        constexpr int HALF = kBackThreads / 2;
        __shared__ float other[HALF * VECTORS * E];
        for (int most = HALF; most >= LANES; most /= 2) {
            for (int which = 0; which < 2; which++) {
                __syncthreads();
                if (threadIdx.x >= most && threadIdx.x < 2 * most) {
#pragma unroll
                    for (int v = 0; v < VECTORS; v++) {
#pragma unroll
                        for (int e = 0; e < E; e++) {
                            other[(v * E + e) * HALF + threadIdx.x - most] = which ? db[v][e] : dw[v][e];
                        }
                    }
                }
                __syncthreads();
                if (threadIdx.x < most) {
#pragma unroll
                    for (int v = 0; v < VECTORS; v++) {
#pragma unroll
                        for (int e = 0; e < E; e++) {
                            const float more = other[(v * E + e) * HALF + threadIdx.x];
                            if (which) {
                                db[v][e] += more;
                            } else {
                                dw[v][e] += more;
                            }
                        }
                    }
                }
            }
        }
        if (threadIdx.x >= LANES) return;
    }
    float* sums = partial + static_cast<uint64_t>(blockIdx.x) * 2 * cols;
#pragma unroll
    for (int v = 0; v < VECTORS; v++) {
        if (!held.live(v)) continue;
#pragma unroll
        for (int e = 0; e < E; e++) {
            if (!held.own(v, e)) continue;
            sums[held.column(v) + e] = dw[v][e];
            sums[cols + held.column(v) + e] = db[v][e];
        }
    }
}

// Rows longer than a block's registers: dx, a block a row read twice.
template <typename S, typename W>
__global__ void __launch_bounds__(kMostLanes)
    norm_back_long_kernel(const S* dy, uint64_t dy_step, const S* x, uint64_t x_step, uint64_t rows,
                          uint64_t cols, const W* weight, const float* __restrict__ means,
                          const float* __restrict__ scales, S* dx, uint64_t dx_step) {
    __shared__ float shared[2][kMostWaves];
    const float count = static_cast<float>(cols);
    for (uint64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const float mean = means[row], scale = scales[row];
        float sum = 0.0f, along = 0.0f;
        for (uint64_t c = threadIdx.x; c < cols; c += blockDim.x) {
            const float g = Elem<S>::widen(dy[row * dy_step + c]) * (weight != nullptr ? Elem<W>::widen(weight[c]) : 1.0f);
            sum += g;
            along += g * ((Elem<S>::widen(x[row * x_step + c]) - mean) * scale);
        }
        sum = block_join<Added>(sum, shared[0]) / count;
        along = block_join<Added>(along, shared[1]) / count;
        for (uint64_t c = threadIdx.x; c < cols; c += blockDim.x) {
            const float g = Elem<S>::widen(dy[row * dy_step + c]) * (weight != nullptr ? Elem<W>::widen(weight[c]) : 1.0f);
            const float u = (Elem<S>::widen(x[row * x_step + c]) - mean) * scale;
            dx[row * dx_step + c] = Elem<S>::narrow(scale * (g - sum - u * along));
        }
        __syncthreads();  // the next row writes `shared` again
    }
}

// ... and their dw and db: a lane a column, blockIdx.y a share of the rows.
template <typename S>
__global__ void __launch_bounds__(256)
    norm_back_columns_kernel(const S* __restrict__ dy, uint64_t dy_step, const S* __restrict__ x, uint64_t x_step,
                             uint64_t rows, uint64_t cols, const float* __restrict__ means,
                             const float* __restrict__ scales, float* __restrict__ partial) {
    const uint64_t c = static_cast<uint64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (c >= cols) return;
    float dw = 0.0f, db = 0.0f;
    for (uint64_t row = blockIdx.y; row < rows; row += gridDim.y) {
        const float g = Elem<S>::widen(dy[row * dy_step + c]);
        dw = fmaf(g, (Elem<S>::widen(x[row * x_step + c]) - means[row]) * scales[row], dw);
        db += g;
    }
    float* sums = partial + static_cast<uint64_t>(blockIdx.y) * 2 * cols;
    sums[c] = dw;
    sums[cols + c] = db;
}

// out[c] = the sum over `parts` of partial[part][c] in a fixed order, for the
// 2 x cols columns: 16 columns a block, of which each of 64 lanes takes every
// 64th part; a wave's four sums are added in registers, then the waves'.
template <typename W>
__global__ void __launch_bounds__(1024)
    add_parts_kernel(const float* __restrict__ partial, uint32_t parts, uint64_t cols, W* dweight, W* dbias) {
    __shared__ float shared[16][16];
    const uint32_t column = threadIdx.x % 16, turn = threadIdx.x / 16;
    const uint64_t c = static_cast<uint64_t>(blockIdx.x) * 16 + column;
    float sum = 0.0f;
    if (c < 2 * cols) {
#pragma unroll 8
        for (uint32_t p = turn; p < parts; p += 64) sum += partial[static_cast<uint64_t>(p) * 2 * cols + c];
    }
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
    if (threadIdx.x % 64 < 16) shared[threadIdx.x / 64][column] = sum;
    __syncthreads();
    if (turn != 0 || c >= 2 * cols) return;
#pragma unroll
    for (int k = 1; k < 16; k++) sum += shared[k][column];
    W* out = c < cols ? dweight : dbias;
    if (out != nullptr) out[c < cols ? c : c - cols] = Elem<W>::narrow(sum);
}

// How the lanes are laid over rows of `cols` elements, `run` of them a
// 16-byte word.
struct Layout {
    int lanes = 0;         // 16, 64, or 0 for a block of `threads`
    int vectors = 0;       // words a lane; 0 for rows too long for registers
    uint32_t threads = 0;  // of a block
};

// Rows of up to 64 x `wave` words take a wave, several rows to a block of
// `block` threads; longer ones a block of at most `most` threads, two words a
// lane at least and `held` elements at most.  With `wave` 5, past 256 words, as
// waves and as blocks: 10007 f16 rows of 2050 forward 17.2 and 22.6 us, of 2560
// (320 words) 21.8 and 24.5, 16384 f32 rows of 1025 26.6 and 34.9; backward with
// an f32 weight 40.5 and 48.7, 42.3 and 49.0, 45.7 and 52.1, but with an f16 one,
// whose waves keep words in memory, 55 and 50, 69 and 49.
Layout layout_of(uint64_t cols, int run, uint32_t block, int wave, uint32_t most, int held) {
    const uint64_t words = (cols + run - 1) / run;
    Layout out;
    out.threads = block;
    if (words <= 16) {
        out.lanes = 16, out.vectors = 1;
        return out;
    }
    if (words <= 64 * static_cast<uint64_t>(wave)) {
        out.lanes = 64, out.vectors = static_cast<int>((words + 63) / 64);
        return out;
    }
    for (const int vectors : {2, 4, 6, 7, 8}) {
        const uint64_t threads = ((words + vectors - 1) / vectors + 63) / 64 * 64;
        // Only a lane's last word may lie past the row's end (`Held`).
        if (vectors * run > held || threads > most || (vectors - 1) * threads >= words) continue;
        out.vectors = vectors;
        out.threads = static_cast<uint32_t>(threads);
        return out;
    }
    out.vectors = 0, out.threads = kMostLanes;
    return out;
}

// As many blocks as `threads_per_cu` on every compute unit allow, or fewer
// that have all the rows.
uint32_t blocks_of(const Layout& layout, uint64_t rows, uint32_t threads_per_cu) {
    const uint64_t per_block = layout.lanes ? layout.threads / layout.lanes : 1;
    const uint64_t wanted = (rows + per_block - 1) / per_block;
    uint64_t most = uint64_t{static_cast<uint32_t>(compute_units())} *
                    (threads_per_cu > layout.threads ? threads_per_cu / layout.threads : 1);
    // A dispatch holds fewer than 2^32 work-items.
    if (most > 0xffffffffu / layout.threads) most = 0xffffffffu / layout.threads;
    return static_cast<uint32_t>(wanted < most ? wanted : most);
}

// The body with LANES and VECTORS of the layout of at most HELD elements a
// lane.
#define TC_NORM_FORM(layout, S, HELD, ...)                               \
    if (layout.lanes == 16) {                                            \
        constexpr int LANES = 16, VECTORS = 1; __VA_ARGS__;              \
    } else if (layout.lanes == 64 && layout.vectors == 1) {              \
        constexpr int LANES = 64, VECTORS = 1; __VA_ARGS__;              \
    } else if (layout.lanes == 64 && layout.vectors == 2) {              \
        constexpr int LANES = 64, VECTORS = 2; __VA_ARGS__;              \
    } else if (layout.lanes == 64 && layout.vectors == 3) {              \
        constexpr int LANES = 64, VECTORS = 3; __VA_ARGS__;              \
    } else if (layout.lanes == 64 && layout.vectors == 4) {              \
        constexpr int LANES = 64, VECTORS = 4; __VA_ARGS__;              \
    } else if (layout.lanes == 64) {                                     \
        constexpr int LANES = 64, VECTORS = 5; __VA_ARGS__;              \
    } else if (layout.vectors == 2) {                                    \
        constexpr int LANES = 0, VECTORS = 2; __VA_ARGS__;               \
    } else if constexpr (kWordElements<S> * 4 <= HELD) {                 \
        if (layout.vectors == 4) {                                       \
            constexpr int LANES = 0, VECTORS = 4; __VA_ARGS__;           \
        } else if constexpr (kWordElements<S> * 8 <= HELD) {             \
            if (layout.vectors == 6) {                                   \
                constexpr int LANES = 0, VECTORS = 6; __VA_ARGS__;       \
            } else if (layout.vectors == 7) {                            \
                constexpr int LANES = 0, VECTORS = 7; __VA_ARGS__;       \
            } else {                                                     \
                constexpr int LANES = 0, VECTORS = 8; __VA_ARGS__;       \
            }                                                            \
        }                                                                \
    }

template <typename S, typename W>
int norm(const S* x, uint64_t x_step, uint64_t rows, uint64_t cols, const W* weight, const W* bias, float epsilon,
         S* y, uint64_t y_step, float* means, float* scales) {
    TC_STREAM(s);
    const Layout layout = layout_of(cols, kWordElements<S>, 256, 5, kMostLanes, kForwardHeld);
    if (layout.vectors == 0) {
        norm_long_kernel<S, W><<<grid_for(rows, 1, 2), kMostLanes, 0, s>>>(x, x_step, rows, cols, weight, bias,
                                                                          epsilon, y, y_step, means, scales);
        return check_launch("layer norm");
    }
    // Groups that need no barrier take a row each; blocks walk the rows, a
    // compute unit's wavefronts half filled.
    const uint32_t blocks = blocks_of(layout, rows, layout.lanes ? 1u << 30 : 1024);
    const bool streams = 2 * sizeof(S) * rows * cols >= kStreamBytes;
    TC_NORM_FORM(layout, S, kForwardHeld, {
        if (streams) {
            norm_kernel<S, W, LANES, VECTORS, true><<<blocks, layout.threads, 0, s>>>(
                x, x_step, rows, cols, weight, bias, epsilon, y, y_step, means, scales);
        } else {
            norm_kernel<S, W, LANES, VECTORS, false><<<blocks, layout.threads, 0, s>>>(
                x, x_step, rows, cols, weight, bias, epsilon, y, y_step, means, scales);
        }
    })
    return check_launch("layer norm");
}

template <typename S, typename W>
int norm_back(const S* dy, uint64_t dy_step, const S* x, uint64_t x_step, uint64_t rows, uint64_t cols,
              const W* weight, const float* means, const float* scales, S* dx, uint64_t dx_step, W* dweight,
              W* dbias) {
    TC_STREAM(s);
    const bool columns = dweight != nullptr || dbias != nullptr;
    const Layout layout = layout_of(cols, kWordElements<S>, kBackThreads, 5, kBackThreads, kBackHeld);
    // Every block writes 8 bytes a column at its end, so the fewer the better:
    // half the wavefronts that a compute unit holds, but all of them where a
    // lane holds so little that loads in flight are few.  Measured over 10007
    // f16 rows of 2050: 512 threads 41 us, 1024 48; over 8192 f32 rows of 4096
    // (8 elements a lane): 93 and 79.
    const uint32_t per_cu = layout.lanes == 0 && layout.vectors * kWordElements<S> <= 8 ? 1024 : 512;
    const uint32_t row_blocks = layout.vectors == 0 ? grid_for(rows, 64, 1) : blocks_of(layout, rows, per_cu);
    const uint32_t parts = rows == 0 ? 0 : row_blocks;
    Scratch partial(columns ? uint64_t{parts} * 2 * cols * sizeof(float) : 0);
    if (partial.status != TC_OK) return partial.status;
    float* sums = columns ? static_cast<float*>(partial.ptr) : nullptr;
    int status = TC_OK;
    if (rows > 0 && layout.vectors == 0) {
        if (columns) {
            const dim3 grid(static_cast<uint32_t>((cols + 255) / 256), parts);
            norm_back_columns_kernel<S><<<grid, 256, 0, s>>>(dy, dy_step, x, x_step, rows, cols, means, scales, sums);
            status = check_launch("layer norm, backward");
        }
        if (status == TC_OK && dx != nullptr) {
            norm_back_long_kernel<S, W><<<grid_for(rows, 1, 2), kMostLanes, 0, s>>>(
                dy, dy_step, x, x_step, rows, cols, weight, means, scales, dx, dx_step);
            status = check_launch("layer norm, backward");
        }
    } else if (rows > 0) {
        const bool streams = 3 * sizeof(S) * rows * cols >= kStreamBytes;
        TC_NORM_FORM(layout, S, kBackHeld, {
            if (streams) {
                norm_back_kernel<S, W, LANES, VECTORS, true><<<row_blocks, layout.threads, 0, s>>>(
                    dy, dy_step, x, x_step, rows, cols, weight, means, scales, dx, dx_step, sums);
            } else {
                norm_back_kernel<S, W, LANES, VECTORS, false><<<row_blocks, layout.threads, 0, s>>>(
                    dy, dy_step, x, x_step, rows, cols, weight, means, scales, dx, dx_step, sums);
            }
        })
        status = check_launch("layer norm, backward");
    }
    if (status != TC_OK || !columns) return status;
    add_parts_kernel<W><<<static_cast<uint32_t>((2 * cols + 15) / 16), 1024, 0, s>>>(sums, parts, cols, dweight, dbias);
    return check_launch("layer norm, backward");
}

// The checks both passes share.
int check_norm(const char* what, uint32_t dtype, uint32_t weight_dtype, uint64_t rows, uint64_t cols,
               std::initializer_list<uint64_t> steps) {
    if (dtype_size(dtype) == 0 || dtype == TC_F64) {
        return fail(TC_UNSUPPORTED, std::string(what) + ": no kernel for " + dtype_name(dtype));
    }
    if (weight_dtype != dtype && weight_dtype != TC_F32) {
        return fail(TC_UNSUPPORTED, std::string(what) + ": no kernel for " + dtype_name(dtype) + " rows with a " +
                                        dtype_name(weight_dtype) + " weight");
    }
    for (uint64_t step : steps) {
        if (rows > 1 && step < cols) {
            return fail(TC_INVALID, std::string(what) + ": rows of " + std::to_string(cols) + " elements " +
                                        std::to_string(step) + " apart overlap");
        }
        if (rows > 0 && step > UINT64_MAX / 8 / rows) {
            return fail(TC_INVALID, std::string(what) + ": " + std::to_string(rows) + " rows " +
                                        std::to_string(step) + " apart reach past the address space");
        }
    }
    if (cols != 0 && rows > UINT64_MAX / 8 / cols) {
        return fail(TC_INVALID, std::string(what) + ": shape [" + std::to_string(rows) + ", " + std::to_string(cols) +
                                    "] has more elements than fit in a usize");
    }
    if (cols > (uint64_t{1} << 24)) {  // 128 work-items a column are to stay below 2^32
        return fail(TC_UNSUPPORTED, std::string(what) + ": rows of " + std::to_string(cols) + " elements");
    }
    return TC_OK;
}

}  // namespace
}  // namespace tc

using namespace tc;

// `f(S rows' type, W weight's type)` for the two type codes.
#define TC_NORM_TYPES(dtype, weight_dtype, what, ...)                    \
    TC_DISPATCH_FLOAT(dtype, what, S, {                                  \
        if (weight_dtype == TC_F32) {                                    \
            using W = float; __VA_ARGS__;                                \
        } else {                                                         \
            using W = S; __VA_ARGS__;                                    \
        }                                                                \
    })

extern "C" {

int tc_layer_norm(uint32_t dtype, uint32_t weight_dtype, const void* x, uint64_t x_step, uint64_t rows, uint64_t cols,
                  const void* weight, const void* bias, float epsilon, void* y, uint64_t y_step, float* means,
                  float* scales) {
    const int status = check_norm("layer norm", dtype, weight_dtype, rows, cols, {x_step, y_step});
    if (status != TC_OK) return status;
    if (rows == 0) return TC_OK;
    if (cols == 0) return fail(TC_INVALID, "layer norm: rows of no elements");
    if (any_null({x, y})) return null_operand("layer norm");
    TC_NORM_TYPES(dtype, weight_dtype, "layer norm",
                  return norm<S, W>(static_cast<const S*>(x), x_step, rows, cols, static_cast<const W*>(weight),
                                    static_cast<const W*>(bias), epsilon, static_cast<S*>(y), y_step, means, scales))
    return TC_OK;
}

int tc_layer_norm_backward(uint32_t dtype, uint32_t weight_dtype, const void* dy, uint64_t dy_step, const void* x,
                           uint64_t x_step, uint64_t rows, uint64_t cols, const void* weight, const float* means,
                           const float* scales, void* dx, uint64_t dx_step, void* dweight, void* dbias) {
    const char* what = "layer norm, backward";
    const int status = check_norm(what, dtype, weight_dtype, rows, cols, {dy_step, x_step, dx != nullptr ? dx_step : cols});
    if (status != TC_OK) return status;
    if (cols == 0) return rows == 0 ? TC_OK : fail(TC_INVALID, std::string(what) + ": rows of no elements");
    if (rows > 0 && any_null({dy, x, means, scales})) return null_operand(what);
    if (dx == nullptr && dweight == nullptr && dbias == nullptr) return TC_OK;
    if (rows == 0 && dweight == nullptr && dbias == nullptr) return TC_OK;
    TC_NORM_TYPES(dtype, weight_dtype, what,
                  return norm_back<S, W>(static_cast<const S*>(dy), dy_step, static_cast<const S*>(x), x_step, rows,
                                         cols, static_cast<const W*>(weight), means, scales, static_cast<S*>(dx),
                                         dx_step, static_cast<W*>(dweight), static_cast<W*>(dbias)))
    return TC_OK;
}

}  // extern "C"
