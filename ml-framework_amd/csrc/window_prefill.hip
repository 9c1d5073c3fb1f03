// window_prefill.hip -- entry points of the chunks' attention over a window and sinks (window_prefill.h).
#include <algorithm>
#include <string>

#include "window_prefill.h"

namespace {

constexpr int64_t kSplitGroups = 512;  // workgroups of a call whose keys are cut, at most

struct Plan {
    bool share;
    int32_t cols, per, splits;
};
// Waves share a set of columns, each with its own blocks, where a (sequence, KV head) has few or workgroups of 128 columns would leave CUs
// half empty. Measured at (32, 8, 128) bf16, window 1024, shared / own: 32 sequences of 16 tokens 35 / 52 us, 20: 52 / 57, 32: 60 / 61, 64:
// 113 / 84; 512 tokens of one sequence 29 / 45 (128 workgroups of own columns), of two 55 / 59, of four 105 / 83.
// The keys are cut over workgroups up to one a CU, of 16 pairs of blocks at least, and up to two where that leaves 32: 4 sequences of 4 tokens
// on 8192: 36 us in 8 parts of 32 pairs, 41 in 4 and in 16; on 2048: 18 us in 4 parts of 16, 21 in 2, 19 in 8; one chunk of 256 on 8192, 256
// workgroups: 87 us in 2 parts, 105 whole.
Plan plan_of(const pa_config* cfg, int32_t num_seqs, int32_t max_chunk_len, int64_t blocks) {
    Plan p{};
    const int64_t columns = static_cast<int64_t>(max_chunk_len) * (cfg->num_q_heads / cfg->num_kv_heads);
    const int64_t groups = static_cast<int64_t>(num_seqs) * cfg->num_kv_heads;
    p.share = pa::window_shares(cfg->head_dim, cfg->kv_dtype) && (columns <= 96 || groups * ((columns + 127) / 128) <= 256);
    p.cols = p.share ? 32 : 128;
    p.per = static_cast<int32_t>((columns + p.cols - 1) / p.cols);
    const int64_t pairs = (blocks + 1) / 2, wgs = groups * p.per;
    p.splits = 1;
    const int64_t least = p.share ? 16 : 4;  // (four waves of a set of columns take the pairs in turn)
    if (wgs > 0) p.splits = static_cast<int32_t>(std::max({int64_t{1}, std::min(256 / wgs, pairs / least), std::min(kSplitGroups / wgs, pairs / (2 * least))}));
    return p;
}

// The most blocks that a workgroup's columns see.
int64_t most_blocks(int32_t max_chunk_len, int32_t max_len, int32_t sink, int32_t window) {
    const int64_t all = (static_cast<int64_t>(max_len) + 15) / 16;
    if (window == 0) return all;
    return std::min(all, (std::min<int64_t>(sink, max_len) + 15) / 16 +
                             (static_cast<int64_t>(window) + std::min(max_chunk_len, 128) + 14) / 16 + 1);
}

pa_status check_shape(const char* f, const pa_config* cfg, int32_t num_seqs, int32_t max_chunk_len, int32_t max_context_len,
                      int32_t sink, int32_t window) {
    pa_status st = pa::check_config(cfg, f);
    if (st != PA_SUCCESS) return st;
    if (num_seqs < 0 || max_chunk_len < 0 || max_context_len < 0)
        return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": negative size");
    if (sink < 0 || window < 0)
        return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": sink_tokens and window must not be negative");
    if (static_cast<int64_t>(num_seqs) * cfg->num_kv_heads > 65535)
        return pa::set_error(PA_ERROR_UNSUPPORTED, std::string(f) + ": num_seqs * num_kv_heads must be <= 65535");
    if (static_cast<int64_t>(max_chunk_len) * (cfg->num_q_heads / cfg->num_kv_heads) > INT32_MAX)
        return pa::set_error(PA_ERROR_UNSUPPORTED, std::string(f) + ": max_chunk_len times the heads of a group must fit 32 bits");
    return PA_SUCCESS;
}

}  // namespace

extern "C" {

pa_status pa_window_prefill_workspace_size(const pa_config* cfg, int32_t num_seqs, int32_t max_chunk_len,
                                           int32_t max_context_len, int32_t sink_tokens, int32_t window, size_t* bytes) {
    const char* const f = "pa_window_prefill_workspace_size";
    pa_status st = check_shape(f, cfg, num_seqs, max_chunk_len, max_context_len, sink_tokens, window);
    if (st != PA_SUCCESS) return st;
    if (!bytes) return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": bytes is null");
    // what no call of at most these sizes exceeds (a smaller one may be cut where a larger one is not)
    const int64_t cols = pa::window_shares(cfg->head_dim, cfg->kv_dtype) ? 32 : 128;
    *bytes = num_seqs == 0 || max_chunk_len == 0 || max_context_len == 0
                 ? 0
                 : static_cast<size_t>(kSplitGroups * cols) * (cfg->head_dim + 2) * sizeof(float);
    return pa::clear_error();
}

pa_status pa_window_prefill(pa_stream* stream, const pa_config* cfg, float* out, const void* q,
                            const int32_t* q_start_loc, const int32_t* prefix_lens, const void* k_cache,
                            const void* v_cache, const float* k_scale, const float* v_scale,
                            const int32_t* block_tables, int32_t num_seqs, int32_t max_blocks_per_seq,
                            int32_t max_chunk_len, int32_t max_context_len, int32_t sink_tokens, int32_t window,
                            float* lse, void* workspace, size_t workspace_bytes) {
    const char* const f = "pa_window_prefill";
    pa_status st = check_shape(f, cfg, num_seqs, max_chunk_len, max_context_len, sink_tokens, window);
    if (st != PA_SUCCESS) return st;
    if (max_blocks_per_seq < 0) return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": negative size");
    if (max_blocks_per_seq > INT32_MAX / pa::kBlockSize)
        return pa::set_error(PA_ERROR_UNSUPPORTED, std::string(f) + ": max_blocks_per_seq * 16 must fit 32 bits");
    if (num_seqs == 0 || max_chunk_len == 0) return pa::clear_error();
    if (!out || !q || !q_start_loc || !prefix_lens || !k_cache || !v_cache || !block_tables)
        return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": null pointer");
    if (cfg->kv_dtype == PA_DTYPE_INT8 && (!k_scale || !v_scale))
        return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": int8 cache needs k_scale and v_scale");
    if (!pa::aligned16(k_cache) || !pa::aligned16(v_cache) || !pa::aligned16(q) || !pa::aligned16(out))
        return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": out, q and cache pointers must be 16-byte aligned");
    const Plan p = plan_of(cfg, num_seqs, max_chunk_len, most_blocks(max_chunk_len, max_context_len, sink_tokens, window));
    const int64_t groups = static_cast<int64_t>(num_seqs) * cfg->num_kv_heads;
    const int64_t slots = p.splits > 1 ? groups * p.per * p.splits * p.cols : 0;
    const size_t need = static_cast<size_t>(slots) * (cfg->head_dim + 2) * sizeof(float);
    if (need > workspace_bytes || (need > 0 && !workspace))
        return pa::set_error(PA_ERROR_WORKSPACE_TOO_SMALL, std::string(f) + ": workspace needs " + std::to_string(need) + " bytes");
    if (need > 0 && !pa::aligned16(workspace))
        return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": workspace must be 16-byte aligned");
    const int64_t nwg = pa::placed_grid(groups, p.per);
    if (!pa::fits_grid(nwg * p.splits, 256)) return pa::set_error(PA_ERROR_UNSUPPORTED, std::string(f) + ": too many query tokens for one call");
    pa::WindowPrefillArgs a{};
    a.out = out;
    a.lse = lse;
    a.q = q;
    a.k_cache = k_cache;
    a.v_cache = v_cache;
    a.k_scale = k_scale;
    a.v_scale = v_scale;
    a.q_start_loc = q_start_loc;
    a.prefix_lens = prefix_lens;
    a.block_tables = block_tables;
    a.ws_o = static_cast<float*>(workspace);
    a.ws_ml = reinterpret_cast<float2*>(a.ws_o + slots * cfg->head_dim);
    a.num_kv_heads = cfg->num_kv_heads;
    a.group = cfg->num_q_heads / cfg->num_kv_heads;
    a.max_blocks_per_seq = max_blocks_per_seq;
    a.num_blocks = cfg->num_blocks;
    a.max_context_len = max_context_len;
    a.max_chunk_len = max_chunk_len;
    a.sink = sink_tokens;
    a.window = window;
    a.scale = pa::resolve_scale(cfg);
    a.per = p.per;
    a.num_groups = static_cast<int32_t>(groups);
    a.splits = p.splits;
    pa::StreamDevice dev(stream);
    hipStream_t s = pa::native(stream);
    const bool q_f32 = cfg->q_dtype == PA_DTYPE_FP32;
    const uint32_t n = static_cast<uint32_t>(nwg);
    switch (cfg->head_dim) {
        case 32: pa::launch_window_prefill<32>(a, cfg->kv_dtype, q_f32, p.share, n, s); break;
        case 64: pa::launch_window_prefill<64>(a, cfg->kv_dtype, q_f32, p.share, n, s); break;
        case 128: pa::launch_window_prefill<128>(a, cfg->kv_dtype, q_f32, p.share, n, s); break;
        default: pa::launch_window_prefill<256>(a, cfg->kv_dtype, q_f32, p.share, n, s); break;
    }
    PA_HIP_CHECK(hipGetLastError());
    return pa::clear_error();
}

}  // extern "C"
