// sparse_decode.hip -- entry points of the attention over selected blocks (sparse_decode.h).
#include <algorithm>
#include <string>

#include "sparse_decode.h"

namespace {

// List entries per workgroup: equal ranges for the workgroups of a full chip, of two entries a wave at least, or of one
// where that cuts no row into more than kParts parts and every range still has a CU: 8 rows of 64 blocks (bf16, fp32,
// D 128) 11.5 and 16.4 us with two, 10.8 and 14.1 with one; 8 rows of 400 (bf16, D 64) 12.6 in 25 parts a row, 15.8 in 50.
// Whole rows where they give no workgroup more than kWaste entries, or a third, over an equal range: a cut row costs
// another start, another exchange of states and the merge. (bf16, D 128, equal ranges against whole rows: 136 rows of 40
// blocks 18.8 and 13.4 us, 384 of 40 32.3 and 27.8; at 32 entries more, 384 of 64, 40.4 and 39.4, at 34, 296 of 40, 24.8
// and 27.7, at 62, 8 of 64, 11.2 and 14.4.) The limit is in entries, 8 KB each in these; where an entry is 2 KB (int8, D 64) or
// 32 KB (fp32, D 256) whole rows may be worth more or less than it says: not measured.
constexpr int32_t kParts = 8;
constexpr int32_t kWaste = 32;
int32_t sparse_range(const pa_config* cfg, int64_t rows, int32_t budget) {
    const int32_t waves = pa::sparse_waves(cfg->head_dim), groups = pa::sparse_groups(cfg->head_dim, cfg->kv_dtype);
    int64_t r = (rows * budget + groups - 1) / groups;
    const int64_t whole = (rows + groups - 1) / groups * budget;
    if (whole - r <= kWaste) return static_cast<int32_t>(whole);
    r = std::max(r, budget <= kParts * waves ? std::max<int64_t>(waves, (rows * budget + pa::kSparseCUs - 1) / pa::kSparseCUs) : 2 * waves);
    if (r > budget * 3ll / 4 && r <= budget) return budget;
    return static_cast<int32_t>((r + waves - 1) / waves * waves);
}

// Slots of partial states: two per range, none if no row is cut.
size_t slot_count(const pa_config* cfg, int32_t num_queries, int32_t budget) {
    const int64_t rows = static_cast<int64_t>(num_queries) * cfg->num_kv_heads;
    if (rows == 0 || budget == 0) return 0;
    const int32_t range = sparse_range(cfg, rows, budget);
    return range % budget == 0 ? 0 : 2 * static_cast<size_t>((rows * budget + range - 1) / range) * (cfg->num_q_heads / cfg->num_kv_heads);
}

// What no call of that many query tokens and entries, or of fewer, exceeds (fewer rows may be cut where more are not).
size_t most_slots(const pa_config* cfg, int32_t num_queries, int32_t budget) {
    const int64_t all = static_cast<int64_t>(num_queries) * cfg->num_kv_heads * budget;
    const int64_t least = pa::sparse_waves(cfg->head_dim);
    const int64_t ranges = std::min<int64_t>(pa::sparse_groups(cfg->head_dim, cfg->kv_dtype), (all + least - 1) / least);
    return 2 * static_cast<size_t>(ranges) * (cfg->num_q_heads / cfg->num_kv_heads);
}

pa_status check_shape(const char* f, const pa_config* cfg, int32_t num_queries, int32_t budget) {
    pa_status st = pa::check_config(cfg, f);
    if (st != PA_SUCCESS) return st;
    const int32_t g = cfg->num_q_heads / cfg->num_kv_heads;
    if (g > 16 || (g & (g - 1)) != 0)
        return pa::set_error(PA_ERROR_UNSUPPORTED, std::string(f) + ": num_q_heads / num_kv_heads must be 1, 2, 4, 8 or 16");
    if (num_queries < 0 || budget < 0) return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": negative size");
    if (static_cast<int64_t>(num_queries) * cfg->num_kv_heads * std::max(budget, 1) > INT32_MAX)
        return pa::set_error(PA_ERROR_UNSUPPORTED, std::string(f) + ": too many query tokens for one call");
    return PA_SUCCESS;
}

}  // namespace

extern "C" {

pa_status pa_sparse_workspace_size(const pa_config* cfg, int32_t num_queries, int32_t budget, size_t* bytes) {
    const char* const f = "pa_sparse_workspace_size";
    pa_status st = check_shape(f, cfg, num_queries, budget);
    if (st != PA_SUCCESS) return st;
    if (!bytes) return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": bytes is null");
    *bytes = most_slots(cfg, num_queries, budget) * (cfg->head_dim + 2) * sizeof(float);
    return pa::clear_error();
}

pa_status pa_sparse_decode(pa_stream* stream, const pa_config* cfg, float* out, const void* q, const void* k_cache,
                           const void* v_cache, const float* k_scale, const float* v_scale,
                           const int32_t* block_tables, int32_t num_seqs, int32_t max_blocks_per_seq,
                           const int32_t* query_seqs, const int32_t* context_lens, int32_t num_queries,
                           int32_t max_context_len, const int32_t* selected, int32_t budget, void* workspace,
                           size_t workspace_bytes) {
    const char* const f = "pa_sparse_decode";
    pa_status st = check_shape(f, cfg, num_queries, budget);
    if (st != PA_SUCCESS) return st;
    if (num_seqs < 0 || max_blocks_per_seq < 0 || max_context_len < 0)
        return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": negative size");
    if (max_blocks_per_seq > INT32_MAX / pa::kBlockSize)
        return pa::set_error(PA_ERROR_UNSUPPORTED, std::string(f) + ": max_blocks_per_seq * 16 must fit 32 bits");
    if (num_queries == 0) return pa::clear_error();
    if (budget == 0) return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": budget must be >= 1");
    if (!out || !q || !k_cache || !v_cache || !block_tables || !context_lens || !selected)
        return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": null pointer");
    if (!query_seqs && num_queries != num_seqs)
        return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": num_queries must be num_seqs when query_seqs is null");
    if (cfg->kv_dtype == PA_DTYPE_INT8 && (!k_scale || !v_scale))
        return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": int8 cache needs k_scale and v_scale");
    if (!pa::aligned16(k_cache) || !pa::aligned16(v_cache) || !pa::aligned16(q))
        return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": q and cache pointers must be 16-byte aligned");
    const size_t partials = slot_count(cfg, num_queries, budget);
    const size_t need = partials * (cfg->head_dim + 2) * sizeof(float);
    if (need > workspace_bytes || (need > 0 && !workspace))
        return pa::set_error(PA_ERROR_WORKSPACE_TOO_SMALL, std::string(f) + ": workspace needs " + std::to_string(need) + " bytes");
    // the parts of cut rows are joined by a wave per (row, query head), four to a workgroup
    if (partials > 0 && !pa::fits_grid((static_cast<int64_t>(num_queries) * cfg->num_q_heads + 3) / 4, 256))
        return pa::set_error(PA_ERROR_UNSUPPORTED, std::string(f) + ": too many query tokens for one call");
    if (reinterpret_cast<uintptr_t>(workspace) & 3)
        return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": workspace must be 4-byte aligned");
    pa::SparseArgs a{};
    a.d.out = out;
    a.d.q = q;
    a.d.k_cache = k_cache;
    a.d.v_cache = v_cache;
    a.d.k_scale = k_scale;
    a.d.v_scale = v_scale;
    a.d.block_tables = block_tables;
    a.d.context_lens = context_lens;
    a.d.ws_o = static_cast<float*>(workspace);
    a.d.ws_m = a.d.ws_o + partials * cfg->head_dim;
    a.d.ws_l = a.d.ws_m + partials;
    a.d.num_kv_heads = cfg->num_kv_heads;
    a.d.group = cfg->num_q_heads / cfg->num_kv_heads;
    a.d.max_blocks_per_seq = max_blocks_per_seq;
    a.d.num_blocks = cfg->num_blocks;
    a.d.max_context_len = max_context_len;
    a.d.scale = pa::resolve_scale(cfg);
    a.query_seqs = query_seqs;
    a.selected = selected;
    a.num_seqs = num_seqs;
    a.budget = budget;
    a.rows = num_queries * cfg->num_kv_heads;
    a.range = sparse_range(cfg, a.rows, budget);
    pa::StreamDevice dev(stream);
    hipStream_t s = pa::native(stream);
    const bool q_f32 = cfg->q_dtype == PA_DTYPE_FP32;
    switch (cfg->head_dim) {
        case 32: pa::launch_sparse_decode<32>(a, cfg->kv_dtype, q_f32, s); break;
        case 64: pa::launch_sparse_decode<64>(a, cfg->kv_dtype, q_f32, s); break;
        case 128: pa::launch_sparse_decode<128>(a, cfg->kv_dtype, q_f32, s); break;
        default: pa::launch_sparse_decode<256>(a, cfg->kv_dtype, q_f32, s); break;
    }
    PA_HIP_CHECK(hipGetLastError());
    return pa::clear_error();
}

}  // extern "C"
