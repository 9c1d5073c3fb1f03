// window_decode.hip -- entry points of the attention over a window and sinks for single tokens (window_decode.h).
#include <algorithm>
#include <string>

#include "window_decode.h"

namespace {

// The most blocks that a context of up to max_len tokens shows of itself.
int64_t most_blocks(int32_t max_len, int32_t sink, int32_t window) {
    const int64_t all = (static_cast<int64_t>(max_len) + 15) / 16;
    if (window == 0) return all;
    return std::min(all, (std::min<int64_t>(sink, max_len) + 15) / 16 + (static_cast<int64_t>(window) + 14) / 16 + 1);
}

// A call's launches take at most kWindowSeqs sequences each, one after another over the same workspace.
struct Plan {
    int32_t seqs, groups;
    int64_t slots, entries;  // entries: with every row filled up to whole ranges
    bool merge;
};

Plan plan_of(const pa_config* cfg, int32_t num_seqs, int64_t blocks) {
    const int32_t G = cfg->num_q_heads / cfg->num_kv_heads;
    Plan p{};
    p.seqs = std::min(num_seqs, pa::kWindowSeqs);
    const int64_t full = pa::window_decode_groups(cfg->head_dim, cfg->kv_dtype), rows = static_cast<int64_t>(p.seqs) * cfg->num_kv_heads;
    const int64_t ranges = rows * ((blocks + pa::kWindowLeast - 1) / pa::kWindowLeast);
    p.groups = static_cast<int32_t>(std::max<int64_t>(1, std::min(full, ranges)));
    p.merge = p.groups > 1;
    p.slots = 2 * std::min(full, ranges) * G;
    p.entries = ranges * pa::kWindowLeast;
    return p;
}

struct Layout {
    size_t m, l, starts, parts, total, bytes;
};
Layout layout_of(const pa_config* cfg, const Plan& p, bool mass) {
    Layout w{};
    const size_t G = cfg->num_q_heads / cfg->num_kv_heads;
    w.m = p.slots * cfg->head_dim * sizeof(float);
    w.l = w.m + p.slots * sizeof(float);
    w.starts = w.l + p.slots * sizeof(float);
    w.parts = (w.starts + (static_cast<size_t>(p.seqs) + 2) * sizeof(int32_t) + 7) & ~size_t{7};
    w.total = w.parts + (mass ? p.entries * G * sizeof(float2) : 0);
    w.bytes = w.total + (mass ? static_cast<size_t>(p.seqs) * cfg->num_q_heads * sizeof(float2) : 0);
    return w;
}

pa_status check_shape(const char* f, const pa_config* cfg, int32_t num_seqs, int32_t max_context_len, int32_t sink,
                      int32_t window) {
    pa_status st = pa::check_config(cfg, f);
    if (st != PA_SUCCESS) return st;
    const int32_t g = cfg->num_q_heads / cfg->num_kv_heads;
    if (g > 16 || (g & (g - 1)) != 0)
        return pa::set_error(PA_ERROR_UNSUPPORTED, std::string(f) + ": num_q_heads / num_kv_heads must be 1, 2, 4, 8 or 16");
    if (num_seqs < 0 || max_context_len < 0) return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": negative size");
    if (sink < 0 || window < 0)
        return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": sink_tokens and window must not be negative");
    if (std::min<int64_t>(num_seqs, pa::kWindowSeqs) * cfg->num_kv_heads * std::max<int64_t>(1, most_blocks(max_context_len, sink, window)) > INT32_MAX)
        return pa::set_error(PA_ERROR_UNSUPPORTED, std::string(f) + ": too many blocks for one call");
    return PA_SUCCESS;
}

}  // namespace

extern "C" {

pa_status pa_window_decode_workspace_size(const pa_config* cfg, int32_t num_seqs, int32_t max_context_len,
                                          int32_t sink_tokens, int32_t window, int32_t with_mass, size_t* bytes) {
    const char* const f = "pa_window_decode_workspace_size";
    pa_status st = check_shape(f, cfg, num_seqs, max_context_len, sink_tokens, window);
    if (st != PA_SUCCESS) return st;
    if (!bytes) return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": bytes is null");
    *bytes = layout_of(cfg, plan_of(cfg, num_seqs, most_blocks(max_context_len, sink_tokens, window)), with_mass != 0).bytes;
    return pa::clear_error();
}

pa_status pa_window_decode(pa_stream* stream, const pa_config* cfg, float* out, const void* q, const void* k_cache,
                           const void* v_cache, const float* k_scale, const float* v_scale,
                           const int32_t* block_tables, const int32_t* context_lens, int32_t num_seqs,
                           int32_t max_blocks_per_seq, int32_t max_context_len, int32_t sink_tokens, int32_t window,
                           float* block_mass, void* workspace, size_t workspace_bytes) {
    const char* const f = "pa_window_decode";
    pa_status st = check_shape(f, cfg, num_seqs, max_context_len, sink_tokens, window);
    if (st != PA_SUCCESS) return st;
    if (max_blocks_per_seq < 0) return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": negative size");
    if (max_blocks_per_seq > INT32_MAX / pa::kBlockSize)
        return pa::set_error(PA_ERROR_UNSUPPORTED, std::string(f) + ": max_blocks_per_seq * 16 must fit 32 bits");
    if (num_seqs == 0) return pa::clear_error();
    if (!out || !q || !k_cache || !v_cache || !block_tables || !context_lens)
        return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": null pointer");
    if (cfg->kv_dtype == PA_DTYPE_INT8 && (!k_scale || !v_scale))
        return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": int8 cache needs k_scale and v_scale");
    if (!pa::aligned16(k_cache) || !pa::aligned16(v_cache) || !pa::aligned16(q))
        return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": q and cache pointers must be 16-byte aligned");
    const int64_t blocks = most_blocks(max_context_len, sink_tokens, window);
    const Plan p = plan_of(cfg, num_seqs, blocks);
    const Layout w = layout_of(cfg, p, block_mass != nullptr);
    if (w.bytes > workspace_bytes || !workspace)
        return pa::set_error(PA_ERROR_WORKSPACE_TOO_SMALL, std::string(f) + ": workspace needs " + std::to_string(w.bytes) + " bytes");
    if (reinterpret_cast<uintptr_t>(workspace) & 7)
        return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": workspace must be 8-byte aligned");
    const int32_t G = cfg->num_q_heads / cfg->num_kv_heads;
    // the parts of cut rows are joined by a wave per (row, query head), four to a workgroup, masses added by a thread a block
    if (!pa::fits_grid((static_cast<int64_t>(p.seqs) * cfg->num_q_heads + 3) / 4 + p.seqs * ((blocks + 255) / 256), 256))
        return pa::set_error(PA_ERROR_UNSUPPORTED, std::string(f) + ": too many heads for one call");
    char* const ws = static_cast<char*>(workspace);
    pa::WindowArgs a{};
    a.d.k_cache = k_cache;
    a.d.v_cache = v_cache;
    a.d.k_scale = k_scale;
    a.d.v_scale = v_scale;
    a.d.ws_o = reinterpret_cast<float*>(ws);
    a.d.ws_m = reinterpret_cast<float*>(ws + w.m);
    a.d.ws_l = reinterpret_cast<float*>(ws + w.l);
    a.d.num_kv_heads = cfg->num_kv_heads;
    a.d.group = G;
    a.d.max_blocks_per_seq = max_blocks_per_seq;
    a.d.num_blocks = cfg->num_blocks;
    a.d.max_context_len = max_context_len;
    a.d.scale = pa::resolve_scale(cfg);
    a.starts = reinterpret_cast<int32_t*>(ws + w.starts);
    a.parts = block_mass ? reinterpret_cast<float2*>(ws + w.parts) : nullptr;
    a.total = reinterpret_cast<float2*>(ws + w.total);
    a.sink = sink_tokens;
    a.window = window;
    a.mass_chunks = block_mass ? static_cast<int32_t>((blocks + 255) / 256) : 0;
    a.groups = p.groups;
    pa::StreamDevice dev(stream);
    hipStream_t s = pa::native(stream);
    const bool q_f32 = cfg->q_dtype == PA_DTYPE_FP32;
    for (int32_t s0 = 0; s0 < num_seqs; s0 += pa::kWindowSeqs) {
        a.num_seqs = std::min(pa::kWindowSeqs, num_seqs - s0);
        const int64_t q0 = static_cast<int64_t>(s0) * cfg->num_q_heads * cfg->head_dim;
        a.d.out = out + q0;
        a.d.q = static_cast<const char*>(q) + q0 * (q_f32 ? 4 : 2);
        a.d.block_tables = block_tables + static_cast<int64_t>(s0) * max_blocks_per_seq;
        a.d.context_lens = context_lens + s0;
        a.mass = block_mass ? block_mass + static_cast<int64_t>(s0) * max_blocks_per_seq : nullptr;
        a.merge_groups = p.merge ? static_cast<int32_t>((static_cast<int64_t>(a.num_seqs) * cfg->num_q_heads + 3) / 4) : 0;
        switch (cfg->head_dim) {
            case 32: pa::launch_window_decode<32>(a, cfg->kv_dtype, q_f32, s); break;
            case 64: pa::launch_window_decode<64>(a, cfg->kv_dtype, q_f32, s); break;
            case 128: pa::launch_window_decode<128>(a, cfg->kv_dtype, q_f32, s); break;
            default: pa::launch_window_decode<256>(a, cfg->kv_dtype, q_f32, s); break;
        }
        PA_HIP_CHECK(hipGetLastError());
    }
    return pa::clear_error();
}

}  // extern "C"
