// evict.hip -- the lightest blocks leave their rows: eviction from a paged cache by accumulated attention weight.
//
// A row of n = ceil(len / 16) blocks over its budget keeps the first sink_blocks, the last recent_blocks and, of the rest, the
// heaviest by mass (without masses: the latest), ties to the lowest index. What stays moves down in order, table and masses alike;
// the reference counts of the others fall by one. No key or value moves.
//
// One workgroup a row. The border between what stays and what goes is the k-th largest mass, found digit by digit
// (11 bits a pass, from the top) over the masses as ordered 32-bit integers; blocks at the border itself are dealt out by index.
// Traffic is 16 bytes a block; a row's chain of loads, passes and barriers is what it costs, so rows of up to 16384 blocks
// are read once into registers, a thread every 1024th block, and what stays is numbered by the waves' ballots of all of them at once
// (64 rows of 262 blocks 5.7 us; counting every block's rank among the others instead, from LDS, 8.8). Longer rows are bound by one CU's
// scattered writes and atomics (32 rows of 2-8k blocks 25 us, 12 of them with the reference counts; with registers for 16k blocks 29.5), and
// rows whose masses are all equal by the one counter that they meet in (16 us more there).
#include <algorithm>
#include <string>

#include "pa_internal.h"

namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;

// Masses as integers of the same order: NaN above all, -0 as 0.
__device__ __forceinline__ uint32_t ordered(float x) {
    if (x != x) return 0xffffffffu;
    const uint32_t u = __float_as_uint(x + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Exclusive prefix of `flag` over the workgroup's threads on top of `base`, which moves on by the workgroup's count.
__device__ __forceinline__ int place(bool flag, int* s_count, int& base) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint64_t votes = __ballot(flag);
    if (lane == 0) s_count[wave] = __popcll(votes);
    __syncthreads();
    int at = base + __popcll(votes & ((1ull << lane) - 1)), sum = 0;
#pragma unroll
    for (int w = 0; w < kWaves; w++) {
        at += w < wave ? s_count[w] : 0;
        sum += s_count[w];
    }
    base += sum;
    __syncthreads();
    return at;
}

// Rows of at most 1024 K blocks.
template <int K>
__global__ __launch_bounds__(kThreads) void evict_short_kernel(int32_t* __restrict__ tables, int32_t* __restrict__ lens,
                                                               float* __restrict__ mass, int32_t width, int32_t sink,
                                                               int32_t recent, int32_t budget, int32_t num_blocks,
                                                               int32_t* __restrict__ refcounts, int32_t* __restrict__ evicted) {
    __shared__ int s_hist[2048], s_count[K * kWaves], s_sum[kWaves];
    __shared__ int s_digit, s_rest;
    const int r = blockIdx.x;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int32_t* const row = tables + static_cast<int64_t>(r) * width;
    float* const weight = mass ? mass + static_cast<int64_t>(r) * width : nullptr;
    int id[K];
    float w[K];
#pragma unroll
    for (int i = 0; i < K; i++) {  // beside the length's load, whether the row is cut or not
        const int b = i * kThreads + static_cast<int>(threadIdx.x);
        id[i] = b < width ? row[b] : -1;
        w[i] = weight && b < width ? weight[b] : 0.0f;
    }
    const int len = lens[r];
    const int n = static_cast<int>(min((static_cast<int64_t>(len) + 15) / 16, static_cast<int64_t>(width)));
    if (len <= 0 || n <= budget) {
        if (evicted && threadIdx.x == 0) evicted[r] = 0;
        return;
    }
    const int lo = sink, hi = n - recent;  // what may go
    int rest = budget - sink - recent;     // of these, how many stay
    bool may[K];
#pragma unroll
    for (int i = 0; i < K; i++) {
        const int b = i * kThreads + static_cast<int>(threadIdx.x);
        may[i] = b >= lo && b < hi;
    }
    // Numbers the set flags in the order of the blocks: at[i] for block i * kThreads + thread. (Its barriers also stand between the reads
    // above and the writes below.)
    const auto number = [&](const bool (&flag)[K], int (&at)[K]) {
        uint64_t votes[K];
#pragma unroll
        for (int i = 0; i < K; i++) {
            votes[i] = __ballot(flag[i]);
            if (lane == 0) s_count[i * kWaves + wave] = __popcll(votes[i]);
        }
        __syncthreads();
        if (wave == 0) {  // lane l: K / 4 of the counts in turn
            constexpr int PER = (K * kWaves + 63) / 64;
            int c[PER], sum = 0;
#pragma unroll
            for (int j = 0; j < PER; j++) {
                c[j] = PER * lane + j < K * kWaves ? s_count[PER * lane + j] : 0;
                sum += c[j];
            }
            int before = pa::wave_prefix(sum) - sum;
#pragma unroll
            for (int j = 0; j < PER; j++) {
                if (PER * lane + j < K * kWaves) s_count[PER * lane + j] = before;
                before += c[j];
            }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < K; i++) at[i] = s_count[i * kWaves + wave] + __popcll(votes[i] & ((1ull << lane) - 1));
        __syncthreads();  // s_count is free again
    };
    bool stays[K];
    int to[K];
    if (weight && rest > 0) {
        uint32_t border = 0;  // above it stays, at it the first `rest` do
#pragma unroll
        for (int pass = 0; pass < 3; pass++) {
            const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
            for (int i = threadIdx.x; i < 2048; i += kThreads) s_hist[i] = 0;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < K; i++) {
                const uint32_t k = ordered(w[i]);
                if (may[i] && (pass == 0 || (k ^ border) >> (shift + bits) == 0)) atomicAdd(&s_hist[k >> shift & ((1u << bits) - 1)], 1);
            }
            __syncthreads();
            // thread t: digits 2 t, 2 t + 1; what lies above each
            const int c0 = s_hist[2 * threadIdx.x], c1 = s_hist[2 * threadIdx.x + 1];
            const int upto = pa::wave_prefix(c0 + c1);
            if (lane == 63) s_sum[wave] = upto;
            __syncthreads();
            int above = -upto;
#pragma unroll
            for (int v = 0; v < kWaves; v++) above += v >= wave ? s_sum[v] : 0;
            if (above < rest && above + c1 >= rest) {
                s_digit = 2 * threadIdx.x + 1;
                s_rest = rest - above;
            }
            above += c1;
            if (above < rest && above + c0 >= rest) {
                s_digit = 2 * threadIdx.x;
                s_rest = rest - above;
            }
            __syncthreads();
            border |= static_cast<uint32_t>(s_digit) << shift;
            rest = s_rest;
        }
        bool tie[K];
#pragma unroll
        for (int i = 0; i < K; i++) tie[i] = may[i] && ordered(w[i]) == border;
        number(tie, to);
#pragma unroll
        for (int i = 0; i < K; i++) stays[i] = !may[i] || ordered(w[i]) > border || (tie[i] && to[i] < rest);
    } else {
#pragma unroll
        for (int i = 0; i < K; i++) stays[i] = !may[i] || i * kThreads + static_cast<int>(threadIdx.x) >= hi - (weight ? 0 : rest);
    }
#pragma unroll
    for (int i = 0; i < K; i++) stays[i] &= i * kThreads + static_cast<int>(threadIdx.x) < width;
    number(stays, to);
    const int gone = n - budget;
#pragma unroll
    for (int i = 0; i < K; i++) {
        const int b = i * kThreads + static_cast<int>(threadIdx.x);
        if (stays[i]) {
            row[to[i]] = id[i];
            if (weight) weight[to[i]] = w[i];
        } else if (b < width && id[i] >= 0 && id[i] < num_blocks) {
            atomicSub(&refcounts[id[i]], 1);
        }
        if (b < width && b >= width - gone) {  // behind the last that stays
            row[b] = -1;
            if (weight) weight[b] = 0.0f;
        }
    }
    if (threadIdx.x == 0) {
        lens[r] = len - 16 * gone;
        if (evicted) evicted[r] = gone;
    }
}

// Rows of any width, in chunks of 1024 blocks.
__global__ __launch_bounds__(kThreads) void evict_kernel(int32_t* __restrict__ tables, int32_t* __restrict__ lens,
                                                         float* __restrict__ mass, int32_t width, int32_t sink,
                                                         int32_t recent, int32_t budget, int32_t num_blocks,
                                                         int32_t* __restrict__ refcounts, int32_t* __restrict__ evicted) {
    __shared__ int s_hist[256], s_count[kWaves];
    __shared__ int s_digit, s_rest;
    const int r = blockIdx.x;
    const int len = lens[r];
    const int n = static_cast<int>(min((static_cast<int64_t>(len) + 15) / 16, static_cast<int64_t>(width)));
    if (len <= 0 || n <= budget) {
        if (evicted && threadIdx.x == 0) evicted[r] = 0;
        return;
    }
    int32_t* const row = tables + static_cast<int64_t>(r) * width;
    float* const weight = mass ? mass + static_cast<int64_t>(r) * width : nullptr;
    const int lo = sink, hi = n - recent;  // what may go
    int rest = budget - sink - recent;     // of these, how many stay
    uint32_t border = 0xffffffffu;         // above it stays, at it the first `rest` do
    bool all_below = rest == 0;
    if (weight && rest > 0) {
        border = 0;
        for (int shift = 24; shift >= 0; shift -= 8) {
            for (int i = threadIdx.x; i < 256; i += kThreads) s_hist[i] = 0;
            __syncthreads();
            for (int b = lo + threadIdx.x; b < hi; b += kThreads) {
                const uint32_t k = ordered(weight[b]);
                if (shift == 24 || (k ^ border) >> (shift + 8) == 0) atomicAdd(&s_hist[k >> shift & 255u], 1);
            }
            __syncthreads();
            if (threadIdx.x < 64) {  // lane l: digits 4 l .. 4 l + 3; the counts above each
                const int l = threadIdx.x;
                int c[4], sum = 0;
#pragma unroll
                for (int i = 0; i < 4; i++) sum += c[i] = s_hist[4 * l + i];
                const int upto = pa::wave_prefix(sum);
                int above = __builtin_amdgcn_readlane(upto, 63) - upto;
#pragma unroll
                for (int i = 3; i >= 0; i--) {
                    if (above < rest && above + c[i] >= rest) {
                        s_digit = 4 * l + i;
                        s_rest = rest - above;
                    }
                    above += c[i];
                }
            }
            __syncthreads();
            border |= static_cast<uint32_t>(s_digit) << shift;
            rest = s_rest;
        }
    }
    int kept = 0, ties = 0;
    const int latest = hi - rest;  // without masses
    for (int b0 = 0; b0 < width; b0 += kThreads) {
        const int b = b0 + static_cast<int>(threadIdx.x);
        const int id = b < width ? row[b] : -1;
        const float w = weight && b < width ? weight[b] : 0.0f;
        const bool may = b >= lo && b < hi;
        bool stays = b < width && !may;
        if (weight) {
            const uint32_t k = ordered(w);
            const bool tie = may && !all_below && k == border;
            const int at = place(tie, s_count, ties);
            stays |= may && !all_below && (k > border || (tie && at < rest));
        } else {
            stays |= may && b >= latest;
        }
        const int to = place(stays, s_count, kept);  // (its barriers stand between the reads above and the writes below)
        if (stays) {
            row[to] = id;
            if (weight) weight[to] = w;
        } else if (b < width && id >= 0 && id < num_blocks) {
            atomicSub(&refcounts[id], 1);
        }
    }
    __syncthreads();
    for (int b = kept + static_cast<int>(threadIdx.x); b < width; b += kThreads) {
        row[b] = -1;
        if (weight) weight[b] = 0.0f;
    }
    if (threadIdx.x == 0) {
        lens[r] = len - 16 * (n - budget);
        if (evicted) evicted[r] = n - budget;
    }
}

}  // namespace

extern "C" pa_status pa_evict_blocks(pa_stream* stream, const pa_config* cfg, int32_t* block_tables, int32_t* lens,
                                     float* block_mass, int32_t num_rows, int32_t max_blocks_per_seq, int32_t sink_blocks,
                                     int32_t recent_blocks, int32_t budget, int32_t* refcounts, int32_t* evicted) {
    const char* const f = "pa_evict_blocks";
    pa_status st = pa::check_config(cfg, f);
    if (st != PA_SUCCESS) return st;
    if (num_rows < 0 || max_blocks_per_seq < 0)
        return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": negative size");
    if (sink_blocks < 0 || recent_blocks < 1 || static_cast<int64_t>(sink_blocks) + recent_blocks > budget)
        return pa::set_error(PA_ERROR_INVALID_ARGUMENT,
                             std::string(f) + ": sink_blocks >= 0, recent_blocks >= 1 and sink_blocks + recent_blocks <= budget");
    if (num_rows == 0 || max_blocks_per_seq == 0) return pa::clear_error();
    if (!block_tables || !lens || !refcounts)
        return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": null pointer");
    if (max_blocks_per_seq > INT32_MAX / pa::kBlockSize)
        return pa::set_error(PA_ERROR_UNSUPPORTED, std::string(f) + ": max_blocks_per_seq * 16 must fit 32 bits");
    if (!pa::fits_grid(num_rows, kThreads)) return pa::set_error(PA_ERROR_UNSUPPORTED, std::string(f) + ": too many rows for one call");
    pa::StreamDevice dev(stream);
    const auto go = [&](auto kernel) {
        kernel<<<num_rows, kThreads, 0, pa::native(stream)>>>(block_tables, lens, block_mass, max_blocks_per_seq, sink_blocks,
                                                              recent_blocks, budget, cfg->num_blocks, refcounts, evicted);
    };
    // The fewest registers that a row fits (64 rows of 262 blocks in those for 1024 / 4096 / 8192 / 16384: 5.7 / 7.1 / 9.0 / 13.3 us, by the
    // kernel of any width 6.3; 32 rows of 8000: 23.8 in those for 8192, 28.0 and 36.9; of 16000: 45, 75).
    if (max_blocks_per_seq <= kThreads) go(evict_short_kernel<1>);
    else if (max_blocks_per_seq <= 4 * kThreads) go(evict_short_kernel<4>);
    else if (max_blocks_per_seq <= 8 * kThreads) go(evict_short_kernel<8>);
    else if (max_blocks_per_seq <= 16 * kThreads) go(evict_short_kernel<16>);
    else go(evict_kernel);
    PA_HIP_CHECK(hipGetLastError());
    return pa::clear_error();
}
