// The norm over all of a model's gradients, and the gradients scaled down to a
// largest norm:
//   n = sqrt(sum over tensors and elements of g^2),  out = g f,
//   f = limit / n where n is above the limit and finite in 32 bits, else 1.
// Bound by memory: g is read for the norm, and again (n is not known before
// all of it is) to be written.  The second pass goes through the tensors
// backwards, so that it finds in the 256 MiB Infinity Cache what the first
// one read last, and streams past the cache what it writes (25 M f32, 201 MB
// read and written once each: 61 us with plain stores, 53 so).
//
// Measured: those gradients now 51 us, 19 for the norm (5.2 TB/s) and 31 to
// scale (6.4); 300 tensors of 300 M elements, 1.83 GB moved, 339 us, 5.4 TB/s
// (336 where the norm read words of memory whose lanes hold other elements for
// every alignment).  Eight words a lane at a time instead of four took 403.
//
// The tensors' pointers and lengths travel in the kernels' arguments, up to
// kTable of them a launch, so that no table is uploaded; blocks take chunks
// of kChunk words of any of them.  Squares are summed in 64 bits, where those
// of no two finite 32-bit numbers overflow or vanish; a block writes one sum,
// and the sums are added in block order.

#include <math.h>

#include <new>

#include "rows.hpp"

namespace tc {
namespace {

constexpr int kThreads = 256;
constexpr int kInFlight = 4;  // words a lane reads at a time
constexpr uint64_t kChunk = uint64_t{kThreads} * kInFlight;  // words of a block's turn
constexpr int kTable = 140;        // tensors of a launch: 4 KiB of arguments less 164 bytes
constexpr uint32_t kDirect = 4096;  // sums that every scaling block adds by itself

struct Entry {
    const void* from;
    void* to;
    uint64_t length : 48;
    uint64_t dtype : 16;
};

struct Table {
    Entry entries[kTable];
    uint32_t first[kTable + 1];  // chunk, in the order of the entries
    uint32_t count;

    // The entry that has `chunk`.
    __device__ __forceinline__ uint32_t of(uint32_t chunk) const {
        uint32_t low = 0, high = count;
        while (high - low > 1) {
            const uint32_t middle = (low + high) / 2;
            if (first[middle] <= chunk) low = middle;
            else high = middle;
        }
        return low;
    }
};

// The sum of `v` over the block, in every lane, in lane and wave order.
__device__ __forceinline__ double block_sum(double v, double* shared) {
    for (int offset = 32; offset > 0; offset >>= 1) v += __shfl_xor(v, offset);
    if (threadIdx.x % 64 == 0) shared[threadIdx.x / 64] = v;
    __syncthreads();
    double all = shared[0];
    for (int w = 1; w < kThreads / 64; w++) all += shared[w];
    return all;
}

template <typename S>
__device__ __forceinline__ double squares(const Entry& entry, uint64_t first) {
    constexpr int E = kWordElements<S>;
    // Words from the tensor's start on, wherever it is, so that its address
    // has no part in which squares are added first.
    const S* from = static_cast<const S*>(entry.from);
    const uint64_t length = entry.length, words = (length + E - 1) / E;
    Words<S, E> in[kInFlight];
#pragma unroll
    for (int u = 0; u < kInFlight; u++) {
        const uint64_t word = first + u * kThreads + threadIdx.x, at = word * E;
        if (at + E <= length) {
            in[u].template load<false>(from + at);
        } else if (word < words) {
            float v[E];
#pragma unroll
            for (int e = 0; e < E; e++) v[e] = at + e < length ? Elem<S>::widen(from[at + e]) : 0.0f;
            in[u].put(v);
        }
    }
    double sum = 0.0;
#pragma unroll
    for (int u = 0; u < kInFlight; u++) {
        if (first + u * kThreads + threadIdx.x >= words) break;
#pragma unroll
        for (int e = 0; e < E; e++) {
            const double v = static_cast<double>(in[u].at(e));
            sum = fma(v, v, sum);
        }
    }
    return sum;
}

__global__ void __launch_bounds__(kThreads) squares_kernel(const Table table, uint32_t chunks, double* sums) {
    __shared__ double shared[kThreads / 64];
    double sum = 0.0;
    for (uint32_t chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x) {
        const uint32_t at = table.of(chunk);
        const Entry& entry = table.entries[at];
        const uint64_t first = (chunk - table.first[at]) * kChunk;
        if (entry.dtype == TC_F32) sum += squares<float>(entry, first);
        else if (entry.dtype == TC_F16) sum += squares<_Float16>(entry, first);
        else sum += squares<bf16_t>(entry, first);
    }
    sum = block_sum(sum, shared);
    if (threadIdx.x == 0) sums[blockIdx.x] = sum;
}

// The sum of all blocks' sums, in every lane of the block.
__device__ __forceinline__ double total_of(const double* sums, uint32_t count, double* shared) {
    double sum = 0.0;
#pragma unroll 4
    for (uint32_t k = threadIdx.x; k < count; k += kThreads) sum += sums[k];
    return block_sum(sum, shared);
}

// Many sums to one, or the norm alone.
__global__ void __launch_bounds__(kThreads) total_kernel(const double* sums, uint32_t count, double* total, float* norm) {
    __shared__ double shared[kThreads / 64];
    const double sum = total_of(sums, count, shared);
    if (threadIdx.x != 0) return;
    if (total != nullptr) *total = sum;
    if (norm != nullptr) *norm = static_cast<float>(sqrt(sum));
}

template <typename S>
__device__ __forceinline__ void scale(const Entry& entry, uint64_t first, float factor) {
    constexpr int E = kWordElements<S>;
    const Row<S> row(static_cast<const S*>(entry.from), entry.length);
    const uint64_t words = row.words();
    S* to = static_cast<S*>(entry.to);
    Words<S, E> in[kInFlight];
#pragma unroll
    for (int u = 0; u < kInFlight; u++) {
        const uint64_t word = first + u * kThreads + threadIdx.x;
        if (word < words) row.template load<true>(word, in[u], 0.0f);
    }
#pragma unroll
    for (int u = 0; u < kInFlight; u++) {
        const uint64_t word = first + u * kThreads + threadIdx.x;
        if (word >= words) break;
        float v[E];
        in[u].get(v);
#pragma unroll
        for (int e = 0; e < E; e++) v[e] *= factor;
        row.template store<true>(word, to, v);
    }
}

__global__ void __launch_bounds__(kThreads)
    scale_kernel(const Table table, uint32_t chunks, const double* sums, uint32_t count, float limit, float* norm) {
    __shared__ double shared[kThreads / 64];
    const double all = sqrt(total_of(sums, count, shared));
    if (norm != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *norm = static_cast<float>(all);
    const bool clips = all > limit && static_cast<float>(all) < INFINITY;
    const float factor = clips ? static_cast<float>(limit / all) : 1.0f;
    for (uint32_t turn = blockIdx.x; turn < chunks; turn += gridDim.x) {
        const uint32_t chunk = chunks - 1 - turn;
        const uint32_t at = table.of(chunk);
        const Entry& entry = table.entries[at];
        if (!clips && entry.from == entry.to) continue;
        const uint64_t first = (chunk - table.first[at]) * kChunk;
        if (entry.dtype == TC_F32) scale<float>(entry, first, factor);
        else if (entry.dtype == TC_F16) scale<_Float16>(entry, first, factor);
        else scale<bf16_t>(entry, first, factor);
    }
}

// The tensors in tables of at most kTable entries and 2^31 chunks.
struct Launch {
    Table table;
    uint32_t chunks;
    uint32_t blocks;
};

std::vector<Launch> launches_of(uint32_t count, const uint32_t* dtypes, const void* const* tensors, const uint64_t* lens,
                                void* const* outputs) {
    std::vector<Launch> out;
    const uint32_t most = static_cast<uint32_t>(compute_units()) * 8;
    for (uint32_t k = 0; k < count; k++) {
        if (lens[k] == 0) continue;
        // At most, wherever the tensor starts.
        const uint64_t words = lens[k] / (16 / dtype_size(dtypes[k])) + 2;
        const uint32_t chunks = static_cast<uint32_t>((words + kChunk - 1) / kChunk);
        if (out.empty() || out.back().table.count == kTable || out.back().chunks > 0x7fffffffu - chunks) {
            out.emplace_back();
        }
        Launch& here = out.back();
        Table& table = here.table;
        table.entries[table.count] = Entry{tensors[k], outputs != nullptr ? outputs[k] : nullptr, lens[k], static_cast<uint16_t>(dtypes[k])};
        table.first[table.count++] = here.chunks;
        here.chunks += chunks;
        table.first[table.count] = here.chunks;
        here.blocks = here.chunks < most ? here.chunks : most;
    }
    return out;
}

int check_tensors(const char* what, uint32_t count, const uint32_t* dtypes, const void* const* tensors,
                  const uint64_t* lens, void* const* outputs, const float* norm) {
    if (norm == nullptr || (count > 0 && (dtypes == nullptr || tensors == nullptr || lens == nullptr))) {
        return null_operand(what);
    }
    for (uint32_t k = 0; k < count; k++) {
        if (dtype_size(dtypes[k]) == 0 || dtypes[k] == TC_F64) {
            return fail(TC_UNSUPPORTED, std::string(what) + ": no kernel for " + dtype_name(dtypes[k]));
        }
        if (lens[k] > (uint64_t{1} << 40)) {  // 2^28 chunks at most, past any memory
            return fail(TC_INVALID, std::string(what) + ": a tensor of " + std::to_string(lens[k]) + " elements");
        }
    }
    if (null_slot(tensors, lens, count) || (outputs != nullptr && null_slot(outputs, lens, count))) {
        return null_operand(what);
    }
    return TC_OK;
}

int clip(const char* what, uint32_t count, const uint32_t* dtypes, const void* const* tensors, const uint64_t* lens,
         float limit, void* const* outputs, float* norm) {
    TC_STREAM(s);
    const std::vector<Launch> launches = launches_of(count, dtypes, tensors, lens, outputs);
    uint64_t blocks = 0;
    for (const Launch& launch : launches) blocks += launch.blocks;
    if (blocks > 0x7fffffffu) return fail(TC_UNSUPPORTED, std::string(what) + ": too many tensors");
    Scratch scratch((blocks + 1) * sizeof(double));
    if (scratch.status != TC_OK) return scratch.status;
    double* sums = static_cast<double*>(scratch.ptr) + 1;
    uint64_t at = 0;
    for (const Launch& launch : launches) {
        squares_kernel<<<launch.blocks, kThreads, 0, s>>>(launch.table, launch.chunks, sums + at);
        const int status = check_launch(what);
        if (status != TC_OK) return status;
        at += launch.blocks;
    }
    uint32_t parts = static_cast<uint32_t>(blocks);
    if (outputs == nullptr || launches.empty() || parts > kDirect) {
        total_kernel<<<1, kThreads, 0, s>>>(sums, parts, sums - 1, norm);
        const int status = check_launch(what);
        if (status != TC_OK || outputs == nullptr) return status;
        norm = nullptr;
        sums--, parts = 1;
    }
    for (size_t k = launches.size(); k-- > 0;) {
        scale_kernel<<<launches[k].blocks, kThreads, 0, s>>>(launches[k].table, launches[k].chunks, sums, parts, limit,
                                                             norm);
        const int status = check_launch(what);
        if (status != TC_OK) return status;
        norm = nullptr;
    }
    return TC_OK;
}

}  // namespace
}  // namespace tc

using namespace tc;

extern "C" {

int tc_global_norm(uint32_t count, const uint32_t* dtypes, const void* const* tensors, const uint64_t* lens,
                   float* norm) {
    const int status = check_tensors("global norm", count, dtypes, tensors, lens, nullptr, norm);
    if (status != TC_OK) return status;
    try {
        return clip("global norm", count, dtypes, tensors, lens, 0.0f, nullptr, norm);
    } catch (const std::bad_alloc&) {
        return fail(TC_OUT_OF_MEMORY, "global norm: no memory for the tensors' list");
    }
}

int tc_clip_global_norm(uint32_t count, const uint32_t* dtypes, const void* const* tensors, const uint64_t* lens,
                        float limit, void* const* outputs, float* norm) {
    const char* what = "clip by global norm";
    if (!(limit >= 0.0f)) return fail(TC_INVALID, std::string(what) + ": a largest norm of " + std::to_string(limit));
    if (count > 0 && outputs == nullptr) return null_operand(what);
    const int status = check_tensors(what, count, dtypes, tensors, lens, outputs, norm);
    if (status != TC_OK) return status;
    try {
        return clip(what, count, dtypes, tensors, lens, limit, outputs, norm);
    } catch (const std::bad_alloc&) {
        return fail(TC_OUT_OF_MEMORY, std::string(what) + ": no memory for the tensors' list");
    }
}

}  // extern "C"
