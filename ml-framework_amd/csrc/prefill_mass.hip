// prefill_mass.hip -- the weight that the last query tokens of a chunk give each block of their context.
//
// For sequence s and block b, over the last `last` queries i of its chunk, all query heads h and the visible tokens t of the block (as in
// window_prefill.h):   mass[s][b] += sum_i sum_h sum_t exp(scale q_ih . k_t - lse_ih)
// with the softmax's logarithm lse that the attention of the chunk left, so that keys are read once, and values not at all.
//
// A wave takes two blocks of a sequence and adds up all their columns (query, head) of all KV heads by itself, 32 columns a product
// (K . Q^T as in window_prefill.h), so the sum has one order whatever the timing.
#include <algorithm>
#include <string>

#include "window_prefill.h"

namespace {

struct MassArgs {
    const void* q;
    const float* lse;
    const int32_t* q_start_loc;
    const int32_t* prefix_lens;
    const void* k_cache;
    const float* k_scale;
    const int32_t* block_tables;
    float* mass;
    int32_t num_kv_heads, group, max_blocks_per_seq, num_blocks, max_context_len, last, sink, window;
    float scale;
};

template <int D, int KV, bool QF32>
__global__ __launch_bounds__(256) void prefill_mass_kernel(const MassArgs a) {
    constexpr bool I8 = KV == PA_DTYPE_INT8;
    constexpr int NP = KV == PA_DTYPE_FP32 ? 3 : 1, NQ = QF32 ? 3 : 1, NS = D / 16;
    const int lane = threadIdx.x & 63, n = lane & 31, hf = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int seq = blockIdx.y, Hkv = a.num_kv_heads, G = a.group, Hq = Hkv * G;
    const int q0 = a.q_start_loc[seq], Lc = a.q_start_loc[seq + 1] - q0;
    const int m = min(a.last, Lc);
    if (m <= 0) return;
    const int P = max(a.prefix_lens[seq], 0);
    const int T = static_cast<int>(min(min(static_cast<int64_t>(P) + Lc, static_cast<int64_t>(a.max_blocks_per_seq) * 16),
                                       static_cast<int64_t>(a.max_context_len)));
    const pa::WindowSpan span(P, Lc - m, Lc - 1, T, a.sink, a.window);
    const int e0 = 2 * (static_cast<int>(blockIdx.x) * 4 + wave);
    if (e0 >= span.entries()) return;
    const int32_t* table = a.block_tables + static_cast<int64_t>(seq) * a.max_blocks_per_seq;
    const int lb[2] = {span.block(e0), e0 + 1 < span.entries() ? span.block(e0 + 1) : -1};
    int id[2];
#pragma unroll
    for (int u = 0; u < 2; u++) {
        id[u] = lb[u] >= 0 ? table[lb[u]] : -1;
        if (id[u] >= a.num_blocks) id[u] = -1;
    }
    const int tok[2] = {16 * lb[0], lb[1] >= 0 ? 16 * lb[1] : INT32_MAX - 64};
    const bool all = span.all_see_block(tok[0]) && span.all_see_block(tok[1]);
    const int64_t columns = static_cast<int64_t>(m) * G;
    const int mine = n >> 4;  // the block of the lane's row of K
    const int krow = pa::key_of_row(n);
    float sum[2] = {0.0f, 0.0f};
    for (int kvh = 0; kvh < Hkv; kvh++) {
        uint4 kop[NP][NS];
        const int64_t tile = (static_cast<int64_t>(max(mine ? id[1] : id[0], 0)) * Hkv + kvh) * 16 * D;
        const bool real = (mine ? id[1] : id[0]) >= 0;
#pragma unroll
        for (int s = 0; s < NS; s++) {
            uint4 x[NP];
#pragma unroll
            for (int p = 0; p < NP; p++) x[p] = make_uint4(0, 0, 0, 0);
            if (real) pa::load_planes<KV, NP>(a.k_cache, tile + krow * D + 16 * s + 8 * hf, x);
#pragma unroll
            for (int p = 0; p < NP; p++) kop[p][s] = x[p];
        }
        float ks[2] = {1.0f, 1.0f};
        if constexpr (I8)
#pragma unroll
            for (int u = 0; u < 2; u++) ks[u] = id[u] >= 0 ? a.k_scale[static_cast<int64_t>(id[u]) * Hkv + kvh] : 0.0f;
        for (int64_t c0 = 0; c0 < columns; c0 += 32) {
            const int64_t c = min(c0 + n, columns - 1);
            const int i = static_cast<int>(c / G);
            const int qi = Lc - m + i;
            const int64_t row = (static_cast<int64_t>(q0) + qi) * Hq + kvh * G + (c - static_cast<int64_t>(i) * G);
            const float lse = a.lse[row] * 1.4426950408889634f;
            pa::f32x16_t s;
#pragma unroll
            for (int e = 0; e < 16; e++) s[e] = 0.0f;
#pragma unroll
            for (int sl = 0; sl < NS; sl++) {
                uint4 qx[NQ];
                pa::load_planes<QF32 ? PA_DTYPE_FP32 : PA_DTYPE_BF16, NQ>(a.q, row * D + 16 * sl + 8 * hf, qx);
#pragma unroll
                for (int p = 0; p < NP; p++)
#pragma unroll
                    for (int q = 0; q < NQ; q++)
                        if (p + q <= 2) s = pa::mfma32(kop[p][sl], qx[q], s);
            }
            const int hi = min(T, P + qi + 1), lo = a.window > 0 ? max(0, P + qi + 1 - a.window) : 0;
            const bool counts = c0 + n < columns;
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const float f = a.scale * 1.4426950408889634f * ks[u];
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const int t = tok[u] + 8 * hf + j;
                    const float w = __builtin_amdgcn_exp2f(s[8 * u + j] * f - lse);
                    const bool seen = counts && (all || (t < hi && (t >= lo || t < span.sink)));
                    sum[u] += seen ? w : 0.0f;
                }
            }
        }
    }
#pragma unroll
    for (int u = 0; u < 2; u++) {
        const float w = pa::wave_sum(sum[u]);
        if (lane == 0 && lb[u] >= 0) a.mass[static_cast<int64_t>(seq) * a.max_blocks_per_seq + lb[u]] += w;
    }
}

template <int D>
void launch(const MassArgs& a, int kv, bool q_f32, dim3 grid, hipStream_t s) {
    const auto by_q = [&](auto k) {
        constexpr int KV = decltype(k)::value;
        if (q_f32) prefill_mass_kernel<D, KV, true><<<grid, 256, 0, s>>>(a);
        else prefill_mass_kernel<D, KV, false><<<grid, 256, 0, s>>>(a);
    };
    if (kv == PA_DTYPE_FP32) by_q(std::integral_constant<int, PA_DTYPE_FP32>());
    else if (kv == PA_DTYPE_BF16) by_q(std::integral_constant<int, PA_DTYPE_BF16>());
    else if constexpr (D >= 64) by_q(std::integral_constant<int, PA_DTYPE_INT8>());
}

}  // namespace

extern "C" pa_status pa_prefill_mass(pa_stream* stream, const pa_config* cfg, const void* q, const float* lse,
                                     const int32_t* q_start_loc, const int32_t* prefix_lens, const void* k_cache,
                                     const float* k_scale, const int32_t* block_tables, int32_t num_seqs,
                                     int32_t max_blocks_per_seq, int32_t max_context_len, int32_t last_queries,
                                     int32_t sink_tokens, int32_t window, float* block_mass) {
    const char* const f = "pa_prefill_mass";
    pa_status st = pa::check_config(cfg, f);
    if (st != PA_SUCCESS) return st;
    if (num_seqs < 0 || max_blocks_per_seq < 0 || max_context_len < 0 || last_queries < 0)
        return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": negative size");
    if (sink_tokens < 0 || window < 0)
        return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": sink_tokens and window must not be negative");
    if (max_blocks_per_seq > INT32_MAX / pa::kBlockSize)
        return pa::set_error(PA_ERROR_UNSUPPORTED, std::string(f) + ": max_blocks_per_seq * 16 must fit 32 bits");
    if (num_seqs > 65535) return pa::set_error(PA_ERROR_UNSUPPORTED, std::string(f) + ": num_seqs must be <= 65535");
    if (num_seqs == 0 || last_queries == 0 || max_context_len == 0 || max_blocks_per_seq == 0) return pa::clear_error();
    if (!q || !lse || !q_start_loc || !prefix_lens || !k_cache || !block_tables || !block_mass)
        return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": null pointer");
    if (cfg->kv_dtype == PA_DTYPE_INT8 && !k_scale)
        return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": int8 cache needs k_scale");
    if (!pa::aligned16(k_cache) || !pa::aligned16(q))
        return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": q and k_cache must be 16-byte aligned");
    int64_t blocks = std::min<int64_t>((static_cast<int64_t>(max_context_len) + 15) / 16, max_blocks_per_seq);
    if (window > 0)
        blocks = std::min(blocks, (static_cast<int64_t>(std::min(sink_tokens, max_context_len)) + 15) / 16 +
                                      (static_cast<int64_t>(window) + last_queries + 14) / 16 + 1);
    const MassArgs a{q,          lse,       q_start_loc,       prefix_lens,          k_cache,         k_scale,
                     block_tables, block_mass, cfg->num_kv_heads, cfg->num_q_heads / cfg->num_kv_heads, max_blocks_per_seq,
                     cfg->num_blocks, max_context_len, last_queries, sink_tokens, window, pa::resolve_scale(cfg)};
    pa::StreamDevice dev(stream);
    hipStream_t s = pa::native(stream);
    const dim3 grid(static_cast<uint32_t>((blocks + 7) / 8), num_seqs);
    const bool q_f32 = cfg->q_dtype == PA_DTYPE_FP32;
    switch (cfg->head_dim) {
        case 32: launch<32>(a, cfg->kv_dtype, q_f32, grid, s); break;
        case 64: launch<64>(a, cfg->kv_dtype, q_f32, grid, s); break;
        case 128: launch<128>(a, cfg->kv_dtype, q_f32, grid, s); break;
        default: launch<256>(a, cfg->kv_dtype, q_f32, grid, s); break;
    }
    PA_HIP_CHECK(hipGetLastError());
    return pa::clear_error();
}
