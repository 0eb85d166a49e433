// What the kernels over rows share: sums across a row's lanes in registers,
// and a row's elements as 16-byte words at any alignment and any length.
#pragma once

#include "common.hpp"

namespace tc {

// A scratch block freed when it leaves scope (stream order keeps it alive
// until the queued work has read it).
struct Scratch {
    void* ptr = nullptr;
    int status = TC_OK;
    explicit Scratch(uint64_t bytes) { status = tc_alloc(bytes, &ptr); }
    ~Scratch() {
        if (ptr != nullptr) tc_free(ptr);
    }
    Scratch(const Scratch&) = delete;
    Scratch& operator=(const Scratch&) = delete;
};

// ---- across lanes ---------------------------------------------------------------

template <int CONTROL>
__device__ __forceinline__ float moved(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CONTROL, 0xf, 0xf, true));
}

struct Added {
    __device__ static float join(float a, float b) { return a + b; }
};
struct Largest {
    __device__ static float join(float a, float b) { return fmaxf(a, b); }
};

// `v` joined over each 16 lanes, in every one of them: within the quads, then
// the mirrored halves and rows, all in registers.
template <typename Op>
__device__ __forceinline__ float row16(float v) {
    v = Op::join(v, moved<0xb1>(v));   // lane ^ 1
    v = Op::join(v, moved<0x4e>(v));   // lane ^ 2
    v = Op::join(v, moved<0x141>(v));  // 7 - lane of each 8
    return Op::join(v, moved<0x140>(v));  // 15 - lane
}

// Over the whole wave, in every lane; the same bits in all of them, since
// each step joins the same two values on both sides.
template <typename Op>
__device__ __forceinline__ float wave64(float v) {
    v = row16<Op>(v);
    const uint32_t bits = __float_as_uint(v);
    const auto rows = __builtin_amdgcn_permlane16_swap(bits, bits, false, false);
    v = Op::join(__uint_as_float(rows[0]), __uint_as_float(rows[1]));
    const uint32_t half = __float_as_uint(v);
    const auto halves = __builtin_amdgcn_permlane32_swap(half, half, false, false);
    return Op::join(__uint_as_float(halves[0]), __uint_as_float(halves[1]));
}

constexpr int kMostWaves = 16;  // of a block of 1024

// Over the block, in every lane, in wave order.  One barrier: `shared`
// (kMostWaves floats) is free for the block's next use of it once another
// barrier has passed, so a loop alternates between two or more of them.
template <typename Op>
__device__ __forceinline__ float block_join(float v, float* shared) {
    v = wave64<Op>(v);
    const int waves = blockDim.x / 64;
    if (waves == 1) return v;
    if (threadIdx.x % 64 == 0) shared[threadIdx.x / 64] = v;
    __syncthreads();
    float all = shared[0];
    for (int w = 1; w < waves; w++) all = Op::join(all, shared[w]);
    return all;
}

// Over the LANES lanes (16 or 64) that hold a row, or with LANES 0 the block.
template <int LANES, typename Op>
__device__ __forceinline__ float row_join(float v, float* shared) {
    if constexpr (LANES == 16) return row16<Op>(v);
    if constexpr (LANES == 64) return wave64<Op>(v);
    return block_join<Op>(v, shared);
}

// ---- a row's words ----------------------------------------------------------------

// Elements of type T as E floats' worth of words, kept as they were read.
template <typename T, int E>
struct Words {
    static constexpr int kCount = E * static_cast<int>(sizeof(T)) / 16;
    uint4 w[kCount];

    __device__ __forceinline__ float at(int e) const {
        const int per = 16 / static_cast<int>(sizeof(T));
        const uint4& q = w[e / per];
        if constexpr (sizeof(T) == 4) {
            const uint32_t v = e % 4 == 0 ? q.x : e % 4 == 1 ? q.y : e % 4 == 2 ? q.z : q.w;
            return __uint_as_float(v);
        } else {
            const int pair = e % per / 2;
            const uint32_t v = pair == 0 ? q.x : pair == 1 ? q.y : pair == 2 ? q.z : q.w;
            const uint16_t half = static_cast<uint16_t>(e % 2 ? v >> 16 : v);
            return Elem<T>::widen(__builtin_bit_cast(T, half));
        }
    }
    __device__ __forceinline__ void get(float (&out)[E]) const {
#pragma unroll
        for (int e = 0; e < E; e++) out[e] = at(e);
    }
    __device__ __forceinline__ void put(const float (&v)[E]) {
        uint32_t* to = reinterpret_cast<uint32_t*>(w);
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int e = 0; e < E; e++) to[e] = __float_as_uint(v[e]);
        } else {
            typedef float pair_f32 __attribute__((ext_vector_type(2)));
            typedef __bf16 pair_bf16 __attribute__((ext_vector_type(2)));
#pragma unroll
            for (int e = 0; e < E; e += 2) {
                if constexpr (Elem<T>::dtype == TC_BF16) {
                    // Both in one conversion, to nearest even as f32_to_bf16_bits.
                    to[e / 2] = __builtin_bit_cast(
                        uint32_t, __builtin_convertvector(pair_f32{v[e], v[e + 1]}, pair_bf16));
                } else {
                    to[e / 2] =
                        __builtin_bit_cast(uint16_t, Elem<T>::narrow(v[e])) |
                        (static_cast<uint32_t>(__builtin_bit_cast(uint16_t, Elem<T>::narrow(v[e + 1]))) << 16);
                }
            }
        }
    }
    template <bool NT>
    __device__ __forceinline__ void load(const T* from) {
#pragma unroll
        for (int k = 0; k < kCount; k++) w[k] = load_any_word<NT>(from + k * (16 / sizeof(T)));
    }
    template <bool NT>
    __device__ __forceinline__ void store(T* to) const {
#pragma unroll
        for (int k = 0; k < kCount; k++) store_any_word<NT>(to + k * (16 / sizeof(T)), w[k]);
    }
};

// Which elements of a row of `cols` its run `index` of E elements covers.
// The last run of a row that is no whole number of them starts E before the
// row's end, over elements that the run before it covers too: it reads and
// writes whole words, and only counts from `from` on.  A row shorter than E
// is one run of `to` elements, read one by one.
template <int E>
struct Run {
    uint64_t start = 0;
    int from = 0, to = 0;  // elements of the run that are its own

    Run() = default;
    __device__ __forceinline__ Run(uint64_t index, uint64_t cols) {
        const uint64_t first = index * E;
        if (first >= cols) return;
        if (cols < E) {
            to = static_cast<int>(cols);
            return;
        }
        start = first + E <= cols ? first : cols - E;
        from = static_cast<int>(first - start);
        to = E;
    }
    __device__ __forceinline__ bool live() const { return to > 0; }
    __device__ __forceinline__ bool partial() const { return from > 0 || to < E; }
    __device__ __forceinline__ bool own(int e) const { return e >= from && e < to; }

    template <bool NT, typename T>
    __device__ __forceinline__ void load(const T* row, Words<T, E>& words) const {
        if (to == E) {
            words.template load<NT>(row + start);
        } else {
            float v[E];
#pragma unroll
            for (int e = 0; e < E; e++) v[e] = e < to ? Elem<T>::widen(row[e]) : 0.0f;
            words.put(v);
        }
    }
    template <bool NT, typename T>
    __device__ __forceinline__ void store(T* row, const float (&v)[E]) const {
        if (to == E) {
            Words<T, E> words;
            words.put(v);
            words.template store<NT>(row + start);
        } else {
#pragma unroll
            for (int e = 0; e < E; e++) {
                if (e < to) row[e] = Elem<T>::narrow(v[e]);
            }
        }
    }
};

// Elements of a 16-byte word.
template <typename T>
constexpr int kWordElements = 16 / static_cast<int>(sizeof(T));

// A row in the words of memory, 16-byte aligned wherever it starts: the first
// may begin before the row and the last end behind it, and of those only the
// row's elements are read (`around` in place of the others) and written.
template <typename S>
struct Row {
    static constexpr int E = kWordElements<S>;
    const S* row;
    uint64_t cols;
    int lead;  // elements of the first word that are not the row's

    __device__ __forceinline__ Row(const S* at, uint64_t n)
        : row(at), cols(n), lead(static_cast<int>(reinterpret_cast<uintptr_t>(at) / sizeof(S) % E)) {}
    __device__ __forceinline__ uint64_t words() const { return (cols + lead + E - 1) / E; }
    // Column of the word's first element (of word 0, possibly before the row).
    __device__ __forceinline__ int64_t column(uint64_t word) const {
        return static_cast<int64_t>(word * E) - lead;
    }
    __device__ __forceinline__ bool whole(int64_t column) const {
        return column >= 0 && column + E <= static_cast<int64_t>(cols);
    }
    __device__ __forceinline__ bool has(int64_t column) const {
        return column >= 0 && column < static_cast<int64_t>(cols);
    }
    template <bool NT>
    __device__ __forceinline__ void load(uint64_t word, Words<S, E>& out, float around = -INFINITY) const {
        const int64_t at = column(word);
        if (whole(at)) {
            out.template load<NT>(row + at);
        } else {
            float v[E];
#pragma unroll
            for (int e = 0; e < E; e++) v[e] = has(at + e) ? Elem<S>::widen(row[at + e]) : around;
            out.put(v);
        }
    }
    // The word's results, to the same columns of another row.
    template <bool NT>
    __device__ __forceinline__ void store(uint64_t word, S* to, const float (&v)[E]) const {
        const int64_t at = column(word);
        if (whole(at)) {
            Words<S, E> out;
            out.put(v);
            out.template store<NT>(to + at);
        } else {
#pragma unroll
            for (int e = 0; e < E; e++) {
                if (has(at + e)) to[at + e] = Elem<S>::narrow(v[e]);
            }
        }
    }
};

}  // namespace tc
