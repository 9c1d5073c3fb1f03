// block_select.hip -- the blocks a query token attends to: a score for every block of its context
// from the block's key bounds (key_bounds.hip), and the best of them in ascending order.
//
// For query token r, KV head h with the group's query heads g, block b of its sequence:
//   up_d = sum_g max(q_gd, 0),  down_d = sum_g min(q_gd, 0)
//   score(b) = k_scale_b * sum_d (up_d * hi_bd + down_d * lo_bd)      (k_scale: int8 caches)
// which is at least sum_g max_t q_g . k_t over the block's keys. Kept: the first `sink` blocks, the
// last `recent`, and of the rest the best scores up to `budget` in all, equal scores by the lowest
// index. The outcome is a set of indices, so sums are held in 64 bits: two orders of a 32-bit sum would
// choose differently wherever two scores near the border are closer than its rounding.
//
// Two launches. The scores read 2 D elements per (block, KV head), which bounds them by traffic (a
// sixteenth of the K and V bytes): one wave per 64 blocks of a KV head, 16-byte loads. The choice is
// one workgroup per (query token, KV head): see block_choose_kernel.
#include <algorithm>
#include <string>

#include "pa_internal.h"

namespace {

constexpr int kScoreWaves = 4;
constexpr int kScoreBlocks = 64;      // blocks per wave: a lane per block id
constexpr int kMaxBlocks = 1 << 17;   // blocks of one context: the choice's bit masks in LDS

struct SelectArgs {
    const void* q;
    const void* bounds;
    const float* k_scale;
    const int32_t* tables;
    const int32_t* query_seqs;  // null: query r belongs to sequence r
    const int32_t* context_lens;
    double* scores;             // [num_queries][Hkv][max_blocks]
    int32_t* selected;          // [num_queries][Hkv][budget]
    int32_t num_seqs, width, num_queries, max_blocks, max_len;
    int32_t hkv, group, num_blocks;
    int32_t sink, recent, budget;
    int32_t q_bf16;
};

// Blocks of query r's context, 0 if its sequence is out of range.
__device__ __forceinline__ int context_blocks(const SelectArgs& a, int r, int& seq) {
    seq = a.query_seqs ? a.query_seqs[r] : r;
    if (seq < 0 || seq >= a.num_seqs) return 0;
    const int len = min(min(a.context_lens[r], a.max_len), static_cast<int>(min(static_cast<int64_t>(a.width) * 16,
                                                                                static_cast<int64_t>(INT32_MAX))));
    return len <= 0 ? 0 : (len - 1) / 16 + 1;
}

// 64 bits in two DPP moves or lane exchanges.
__device__ __forceinline__ double shfl_xor_f64(double v, int o) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __shfl_xor(static_cast<uint32_t>(u), o, 64), hi = __shfl_xor(static_cast<uint32_t>(u >> 32), o, 64);
    return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}

template <int KV>
__device__ __forceinline__ float elem(const uint4& w, int e) {
    const uint32_t x[4] = {w.x, w.y, w.z, w.w};
    if constexpr (KV == PA_DTYPE_FP32) return __uint_as_float(x[e]);
    else if constexpr (KV == PA_DTYPE_BF16) return e & 1 ? pa::bf16_hi(x[e >> 1]) : pa::bf16_lo(x[e >> 1]);
    else return pa::i8_at(x[e >> 2], e & 3);
}

// Wave u: KV head u % Hkv, blocks 64 c .. of query r's context, c = u / Hkv % chunks, r = u / Hkv / chunks.
// The bounds of one (block, KV head) are 2 D elements in a row; LB lanes take 16 bytes each of them
// (W times), 64 / LB blocks an instruction.
template <int D, int KV>
__global__ __launch_bounds__(64 * kScoreWaves) void block_score_kernel(const SelectArgs a, int32_t chunks) {
    constexpr int ELT = KV == PA_DTYPE_FP32 ? 4 : KV == PA_DTYPE_BF16 ? 2 : 1;
    constexpr int E = 16 / ELT;
    constexpr int WORDS = 2 * D / E;              // 16-byte words per (block, KV head)
    constexpr int LB = WORDS < 64 ? WORDS : 64;   // lanes per block
    constexpr int W = WORDS / LB;                 // words per lane
    constexpr int NBI = 64 / LB;                  // blocks per load instruction
    constexpr int UN = 8;                         // load instructions in flight
    static_assert(LB % UN == 0, "a chunk is a whole number of batches");
    const int lane = threadIdx.x & 63;
    const int64_t u = static_cast<int64_t>(blockIdx.x) * kScoreWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int h = static_cast<int>(u % a.hkv);
    const int64_t rc = u / a.hkv;
    const int c = static_cast<int>(rc % chunks), r = static_cast<int>(rc / chunks);
    if (r >= a.num_queries) return;
    int seq;
    const int nblk = context_blocks(a, r, seq);
    const int first = c * kScoreBlocks, last = min(first + kScoreBlocks, nblk - a.recent);
    if (nblk <= a.budget || first >= last) return;  // nothing to choose, or no block of the chunk takes part
    int id = -1;
    if (first + lane < last) id = a.tables[static_cast<int64_t>(seq) * a.width + first + lane];
    if (id >= a.num_blocks) id = -1;
    // weights of this lane's elements
    const int at = lane % LB;
    double wt[W][E];
#pragma unroll
    for (int w = 0; w < W; w++) {
        const int i0 = (w * LB + at) * E;
        const bool up = i0 >= D;
        const int d0 = up ? i0 - D : i0;
#pragma unroll
        for (int e = 0; e < E; e++) wt[w][e] = 0.0;
        for (int g = 0; g < a.group; g++) {
            const int64_t qa = (static_cast<int64_t>(r) * a.hkv * a.group + h * a.group + g) * D + d0;
#pragma unroll
            for (int e = 0; e < E; e++) {
                const float x = a.q_bf16 ? pa::bf16_to_f32(static_cast<const uint16_t*>(a.q)[qa + e])
                                         : static_cast<const float*>(a.q)[qa + e];
                wt[w][e] += static_cast<double>(up ? __builtin_elementwise_maximum(x, 0.0f) : __builtin_elementwise_minimum(x, 0.0f));
            }
        }
    }
    double* out = a.scores + (static_cast<int64_t>(r) * a.hkv + h) * a.max_blocks;
    const char* base = static_cast<const char*>(a.bounds);
    for (int i0 = 0; i0 < LB && first + i0 * NBI < last; i0 += UN) {
        uint4 v[UN][W];
        int ids[UN];
#pragma unroll
        for (int k = 0; k < UN; k++) {
            ids[k] = __shfl(id, (i0 + k) * NBI + lane / LB, 64);
#pragma unroll
            for (int w = 0; w < W; w++) {
                v[k][w] = make_uint4(0, 0, 0, 0);
                if (ids[k] >= 0)
                    v[k][w] = reinterpret_cast<const uint4*>(base + (static_cast<int64_t>(ids[k]) * a.hkv + h) * 2 * D * ELT)[w * LB + at];
            }
        }
#pragma unroll
        for (int k = 0; k < UN; k++) {
            double s = 0.0;
#pragma unroll
            for (int w = 0; w < W; w++)
#pragma unroll
                for (int e = 0; e < E; e++) s = __builtin_fma(static_cast<double>(elem<KV>(v[k][w], e)), wt[w][e], s);
#pragma unroll
            for (int o = 1; o < LB; o <<= 1) s += shfl_xor_f64(s, o);
            if constexpr (KV == PA_DTYPE_INT8)
                s *= ids[k] >= 0 ? static_cast<double>(a.k_scale[static_cast<int64_t>(ids[k]) * a.hkv + h]) : 0.0;
            const int b = first + (i0 + k) * NBI + lane / LB;
            if (at == 0 && b < last) out[b] = s;
        }
    }
}

// Scores as 64-bit keys in the same order: NaN above everything (such a block is kept, and the
// attention over it shows the NaN), the two zeros equal.
__device__ __forceinline__ uint64_t key_of(double s) {
    if (s != s) return ~0ull;
    const uint64_t b = __builtin_bit_cast(uint64_t, s + 0.0);
    return b >> 63 ? ~b : b | 1ull << 63;
}

// Counts over the workgroup; every thread gets the sum. s_cnt: one int per wave.
template <int T>
__device__ __forceinline__ int block_count(int mine, int* s_cnt) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) mine += __shfl_xor(mine, o, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s_cnt[threadIdx.x >> 6] = mine;
    __syncthreads();
    int sum = 0;
#pragma unroll
    for (int w = 0; w < T / 64; w++) sum += s_cnt[w];
    return sum;
}

// Exclusive prefix of the set bits of `words` 64-bit words, into pre; by the first wave.
__device__ __forceinline__ void word_prefix(const uint64_t* mask, int* pre, int words) {
    if (threadIdx.x >= 64) return;
    const int lane = threadIdx.x;
    int run = 0;
    for (int w0 = 0; w0 < words; w0 += 64) {
        const int n = w0 + lane < words ? __popcll(mask[w0 + lane]) : 0;
        int incl = n;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int v = __shfl_up(incl, o, 64);
            if (lane >= o) incl += v;
        }
        if (w0 + lane < words) pre[w0 + lane] = run + incl - n;
        run += __shfl(incl, 63, 64);
    }
}

// One workgroup per (query token, KV head). Of the m candidates (the blocks between the sink and the
// recent ones) the `need` best: K, the need-th largest key, is built bit by bit from the top (a count of the
// keys >= a trial value a bit); keys above K are kept, and of those equal to K the first ones.
// Lanes hold consecutive candidates, so a ballot is a 64-bit mask of them, and the places of the
// kept ones in the ascending list are prefix counts of the masks' bits.
template <int T>
__global__ __launch_bounds__(T) void block_choose_kernel(const SelectArgs a) {
    extern __shared__ uint64_t s_mask[];  // [words] masks, then [words] int prefixes
    __shared__ int s_cnt[T / 64];
    const int tid = threadIdx.x, lane = tid & 63;
    const int64_t row = blockIdx.x;
    const int r = static_cast<int>(row / a.hkv);
    int seq;
    const int nblk = context_blocks(a, r, seq);
    int32_t* out = a.selected + row * a.budget;
    if (nblk <= a.budget) {
        for (int i = tid; i < a.budget; i += T) out[i] = i < nblk ? i : -1;
        return;
    }
    const int s0 = a.sink, r0 = nblk - a.recent;
    const int m = r0 - s0, need = a.budget - a.sink - a.recent;  // 0 <= need < m
    const double* scores = a.scores + row * a.max_blocks + s0;
    const int words = (m + 63) / 64;
    int* pre = reinterpret_cast<int*>(s_mask + words);
    const int steps = (m + T - 1) / T;
    uint64_t K = 0;
    if (need > 0) {
        for (int bit = 63; bit >= 0; bit--) {
            const uint64_t trial = K | 1ull << bit;
            int mine = 0;
            for (int j = 0; j < steps; j++) {
                const int i = tid + T * j;
                if (i < m) mine += key_of(scores[i]) >= trial;
            }
            if (block_count<T>(mine, s_cnt) >= need) K = trial;
        }
    }
    int above = 0;
    for (int j = 0; j < steps; j++) {
        const int i = tid + T * j;
        if (i < m) above += key_of(scores[i]) > K;
    }
    above = need > 0 ? block_count<T>(above, s_cnt) : 0;
    // the equal ones in order
    for (int j = 0; j < steps; j++) {
        const int i = tid + T * j;
        const uint64_t eq = __ballot(i < m && key_of(scores[min(i, m - 1)]) == K);
        if (lane == 0 && i < m) s_mask[i >> 6] = eq;
    }
    __syncthreads();
    word_prefix(s_mask, pre, words);
    __syncthreads();
    for (int j = 0; j < steps; j++) {
        const int i = tid + T * j;
        bool keep = false;
        if (i < m && need > 0) {
            const uint64_t k = key_of(scores[i]);
            const int rank = pre[i >> 6] + __popcll(s_mask[i >> 6] & ((1ull << lane) - 1));
            keep = k > K || (k == K && above + rank < need);
        }
        const uint64_t kept = __ballot(keep);
        if (lane == 0 && i < m) s_mask[i >> 6] = kept;  // this wave alone reads and writes its words
    }
    __syncthreads();
    word_prefix(s_mask, pre, words);
    __syncthreads();
    for (int j = 0; j < steps; j++) {
        const int i = tid + T * j;
        if (i >= m) break;
        const uint64_t kept = s_mask[i >> 6];
        if (kept >> lane & 1) out[s0 + pre[i >> 6] + __popcll(kept & ((1ull << lane) - 1))] = s0 + i;
    }
    for (int i = tid; i < a.sink + a.recent; i += T)
        out[i < a.sink ? i : a.budget - a.recent + (i - a.sink)] = i < a.sink ? i : r0 + (i - a.sink);
}

template <int D>
void launch_score(const SelectArgs& a, int kv, uint32_t grid, int32_t chunks, hipStream_t s) {
    if (kv == PA_DTYPE_FP32) block_score_kernel<D, PA_DTYPE_FP32><<<grid, 64 * kScoreWaves, 0, s>>>(a, chunks);
    else if (kv == PA_DTYPE_BF16) block_score_kernel<D, PA_DTYPE_BF16><<<grid, 64 * kScoreWaves, 0, s>>>(a, chunks);
    else if constexpr (D >= 64) block_score_kernel<D, PA_DTYPE_INT8><<<grid, 64 * kScoreWaves, 0, s>>>(a, chunks);
}

pa_status check_sizes(const std::string& f, const pa_config* cfg, int32_t num_queries, int32_t max_context_len) {
    if (num_queries < 0 || max_context_len < 0)
        return pa::set_error(PA_ERROR_INVALID_ARGUMENT, f + ": negative size");
    if (max_context_len > kMaxBlocks * pa::kBlockSize)
        return pa::set_error(PA_ERROR_UNSUPPORTED, f + ": max_context_len must be <= " +
                                                       std::to_string(kMaxBlocks * pa::kBlockSize));
    if (static_cast<int64_t>(num_queries) * cfg->num_kv_heads > 1 << 24)
        return pa::set_error(PA_ERROR_UNSUPPORTED, f + ": too many query tokens for one call");
    return PA_SUCCESS;
}

size_t score_bytes(const pa_config* cfg, int32_t num_queries, int32_t max_context_len) {
    return static_cast<size_t>(num_queries) * cfg->num_kv_heads * ((static_cast<size_t>(max_context_len) + 15) / 16) * 8;
}

}  // namespace

extern "C" {

pa_status pa_select_workspace_size(const pa_config* cfg, int32_t num_queries, int32_t max_context_len, size_t* bytes) {
    const std::string f = "pa_select_workspace_size";
    pa_status st = pa::check_config(cfg, f.c_str());
    if (st != PA_SUCCESS) return st;
    if (!bytes) return pa::set_error(PA_ERROR_INVALID_ARGUMENT, f + ": bytes is null");
    st = check_sizes(f, cfg, num_queries, max_context_len);
    if (st != PA_SUCCESS) return st;
    *bytes = score_bytes(cfg, num_queries, max_context_len);
    return pa::clear_error();
}

pa_status pa_select_blocks(pa_stream* stream, const pa_config* cfg, const void* q, const void* key_bounds,
                           const float* k_scale, const int32_t* block_tables, int32_t num_seqs,
                           int32_t max_blocks_per_seq, const int32_t* query_seqs, const int32_t* context_lens,
                           int32_t num_queries, int32_t max_context_len, int32_t sink_blocks, int32_t recent_blocks,
                           int32_t budget, int32_t* selected, void* workspace, size_t workspace_bytes) {
    const std::string f = "pa_select_blocks";
    pa_status st = pa::check_config(cfg, f.c_str());
    if (st != PA_SUCCESS) return st;
    if (num_seqs < 0 || max_blocks_per_seq < 0) return pa::set_error(PA_ERROR_INVALID_ARGUMENT, f + ": negative size");
    st = check_sizes(f, cfg, num_queries, max_context_len);
    if (st != PA_SUCCESS) return st;
    if (sink_blocks < 0 || recent_blocks < 1)
        return pa::set_error(PA_ERROR_INVALID_ARGUMENT, f + ": sink_blocks must be >= 0 and recent_blocks >= 1");
    if (budget < 1 || static_cast<int64_t>(sink_blocks) + recent_blocks > budget)
        return pa::set_error(PA_ERROR_INVALID_ARGUMENT, f + ": budget must hold the sink and recent blocks");
    if (static_cast<int64_t>(num_queries) * cfg->num_kv_heads * budget > INT32_MAX)
        return pa::set_error(PA_ERROR_UNSUPPORTED, f + ": too many query tokens for one call");
    if (num_queries == 0) return pa::clear_error();
    if (!q || !key_bounds || !block_tables || !context_lens || !selected)
        return pa::set_error(PA_ERROR_INVALID_ARGUMENT, f + ": null pointer");
    if (!query_seqs && num_queries != num_seqs)
        return pa::set_error(PA_ERROR_INVALID_ARGUMENT, f + ": num_queries must be num_seqs when query_seqs is null");
    if (cfg->kv_dtype == PA_DTYPE_INT8 && !k_scale)
        return pa::set_error(PA_ERROR_INVALID_ARGUMENT, f + ": int8 cache needs k_scale");
    if (!pa::aligned16(key_bounds))
        return pa::set_error(PA_ERROR_INVALID_ARGUMENT, f + ": key_bounds must be 16-byte aligned");
    const size_t need = score_bytes(cfg, num_queries, max_context_len);
    if (need > workspace_bytes || (need > 0 && !workspace))
        return pa::set_error(PA_ERROR_WORKSPACE_TOO_SMALL, f + ": workspace needs " + std::to_string(need) + " bytes");
    if (reinterpret_cast<uintptr_t>(workspace) & 7)
        return pa::set_error(PA_ERROR_INVALID_ARGUMENT, f + ": workspace must be 8-byte aligned");
    SelectArgs a{};
    a.q = q;
    a.bounds = key_bounds;
    a.k_scale = k_scale;
    a.tables = block_tables;
    a.query_seqs = query_seqs;
    a.context_lens = context_lens;
    a.scores = static_cast<double*>(workspace);
    a.selected = selected;
    a.num_seqs = num_seqs;
    a.width = max_blocks_per_seq;
    a.num_queries = num_queries;
    a.max_blocks = (max_context_len + 15) / 16;
    a.max_len = max_context_len;
    a.hkv = cfg->num_kv_heads;
    a.group = cfg->num_q_heads / cfg->num_kv_heads;
    a.num_blocks = cfg->num_blocks;
    a.sink = sink_blocks;
    a.recent = recent_blocks;
    a.budget = budget;
    a.q_bf16 = cfg->q_dtype == PA_DTYPE_BF16;
    pa::StreamDevice dev(stream);
    hipStream_t s = pa::native(stream);
    const int32_t most = std::min(a.max_blocks, max_blocks_per_seq);  // blocks of the longest context
    if (most > budget) {
        const int32_t chunks = (most + kScoreBlocks - 1) / kScoreBlocks;
        const int64_t waves = static_cast<int64_t>(num_queries) * chunks * cfg->num_kv_heads;
        const int64_t grid = (waves + kScoreWaves - 1) / kScoreWaves;
        if (grid > INT32_MAX) return pa::set_error(PA_ERROR_UNSUPPORTED, f + ": too many blocks for one call");
        switch (cfg->head_dim) {
            case 32: launch_score<32>(a, cfg->kv_dtype, static_cast<uint32_t>(grid), chunks, s); break;
            case 64: launch_score<64>(a, cfg->kv_dtype, static_cast<uint32_t>(grid), chunks, s); break;
            case 128: launch_score<128>(a, cfg->kv_dtype, static_cast<uint32_t>(grid), chunks, s); break;
            default: launch_score<256>(a, cfg->kv_dtype, static_cast<uint32_t>(grid), chunks, s); break;
        }
        PA_HIP_CHECK(hipGetLastError());
    }
    const size_t words = (static_cast<size_t>(most) + 63) / 64;
    block_choose_kernel<1024><<<num_queries * cfg->num_kv_heads, 1024, words * 12 + 8, s>>>(a);
    PA_HIP_CHECK(hipGetLastError());
    return pa::clear_error();
}

}  // extern "C"
