// prefill_mass.hip -- the weight that the last query tokens of a chunk give each block of their context.
//
// For sequence s and block b, over the last `last` queries i of its chunk, all query heads h and the visible tokens t of the block (as in
// window_prefill.h):   mass[s][b] += sum_i sum_h sum_t exp(scale q_ih . k_t - lse_ih)
// with the softmax's logarithm lse that the attention of the chunk left, so that keys are read once, and values not at all.
//
// A wave holds the keys of two blocks of one KV head as matrix operands and meets 32 columns (query, head) after the other
// (K . Q^T as in window_prefill.h), which four waves with blocks of their own read from LDS: there a column's operands are formed once,
// the next ones on their way from memory meanwhile. A workgroup has two (four) such sets of waves, which share out its (KV head, 32 columns)
// in order; a wave adds up a block's weights over its heads and columns in registers, and the sets' sums are added at the end, so that
// no timing enters. Few blocks: sets of one wave, six to eight of them, which share out the same two blocks' (KV head, 32 columns). Keys are read once however many queries there are.
// What bounds it: 9 prompts of 2-8k tokens, 32 queries, bf16: 42 us, 17 of them the keys' bytes; 31 us for a workgroup alone on its
// CU, 40 for two, and no more than that are there: each step is operands, eight products that wait for one another, exponentials and a
// barrier in turn (1.4 us). Waves that hold 128 columns in registers instead and load them for themselves, 16 bytes of a row a lane,
// 65 us; two waves to a set 44 us, and twice the time for fp32 queries; columns loaded two steps ahead 46 us (registers).
// fp32 queries (three products): one of 30000 tokens, 64 queries, int8: 68 us, 37 of them at the rate of a large matrix product; LDS
// gives their operands no faster than the products take them. Two sets instead of four 78 us.
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

// Eight keys' values as they stand in the cache.
template <int KV> struct RawKeys { uint4 x; };
template <> struct RawKeys<PA_DTYPE_FP32> { pa::f32x4_t x, y; };
template <> struct RawKeys<PA_DTYPE_INT8> { uint2 x; };

template <int KV>
__device__ __forceinline__ void load_raw(RawKeys<KV>& r, const char* at) {
    if constexpr (KV == PA_DTYPE_FP32) {
        r.x = reinterpret_cast<const pa::f32x4_t*>(at)[0];
        r.y = reinterpret_cast<const pa::f32x4_t*>(at)[1];
    } else if constexpr (KV == PA_DTYPE_BF16) {
        r.x = *reinterpret_cast<const uint4*>(at);
    } else {
        r.x = *reinterpret_cast<const uint2*>(at);
    }
}
template <int KV, int NP, bool NEAR>
__device__ __forceinline__ void raw_planes(const RawKeys<KV>& r, uint4 (&plane)[NP]) {
    if constexpr (KV == PA_DTYPE_FP32) {
        const float v[8] = {r.x[0], r.x[1], r.x[2], r.x[3], r.y[0], r.y[1], r.y[2], r.y[3]};
        if constexpr (NEAR) pa::bf16_planes_near<true>(v, plane);  // (fp32 keys under fp32 queries)
        else pa::bf16_planes(v, plane);
    } else if constexpr (KV == PA_DTYPE_BF16) {
        plane[0] = r.x;
    } else {
        const uint32_t x = r.x.x ^ 0x80808080u, y = r.x.y ^ 0x80808080u;
        plane[0] = make_uint4(pa::bf16_pair_of(x, 0), pa::bf16_pair_of(x, 2), pa::bf16_pair_of(y, 0), pa::bf16_pair_of(y, 2));
    }
}

// Waves of a set, which share the columns' operands. few: one.
__host__ __device__ constexpr int mass_waves(bool few) { return few ? 1 : 4; }

// Whether two workgroups fit a CU: 128 registers a lane.
__host__ __device__ constexpr bool mass_two(int d, int kv, bool q_f32) { return !q_f32 && kv != PA_DTYPE_FP32 && d <= 128; }
// Sets of a workgroup: four where registers allow four waves a SIMD, but LDS (three parts of each column) only one workgroup a CU.
// few: what LDS holds, at most eight.
__host__ __device__ constexpr int mass_sets(int d, int kv, bool q_f32, bool few) {
    const int fit = 150 * 1024 / ((q_f32 ? 3 : 1) * d * 64);
    return few ? fit < 8 ? fit : 8 : q_f32 && kv != PA_DTYPE_FP32 && d <= 128 ? 4 : 2;
}
__host__ __device__ constexpr int mass_threads(int d, int kv, bool q_f32, bool few) { return 64 * mass_waves(few) * mass_sets(d, kv, q_f32, few); }
// Whether there is such a form: where LDS holds more sets than workgroups of many blocks have, and registers the keys' three parts.
__host__ __device__ constexpr bool mass_has_few(int d, int kv, bool q_f32) { return d <= 128 || (kv != PA_DTYPE_FP32 && !q_f32); }

// A barrier for what stands in LDS: loads from memory stay under way.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

template <int D, int KV, bool QF32, bool FEW>
__global__ __launch_bounds__(mass_threads(D, KV, QF32, FEW), !FEW && (mass_two(D, KV, QF32) || mass_sets(D, KV, QF32, FEW) == 4) ? 4 : 2) void prefill_mass_kernel(const MassArgs a) {
    constexpr bool I8 = KV == PA_DTYPE_INT8;
    constexpr int NP = KV == PA_DTYPE_FP32 ? 3 : 1, NQ = QF32 ? 3 : 1, NS = D / 16;
    constexpr int ELT = KV == PA_DTYPE_FP32 ? 4 : I8 ? 1 : 2, QKV = QF32 ? PA_DTYPE_FP32 : PA_DTYPE_BF16;
    constexpr int SW = mass_waves(FEW), SETS = mass_sets(D, KV, QF32, FEW);
    constexpr int SET = NS * 64;                                     // 16-byte pieces of 32 columns' operands, of one part
    constexpr int NB = 2 * SETS * NQ * SET * 16 <= (!FEW && mass_two(D, KV, QF32) ? 64 : 128) * 1024 ? 2 : 1;  // buffers of a set
    constexpr bool EARLY = !FEW && !mass_two(D, KV, QF32) && SETS == 2 && (NP == 1 || D < 256);                       // the next head's keys loaded early: registers for it
    constexpr int PER = (SET + 64 * SW - 1) / (64 * SW);  // pieces a thread brings
    __shared__ uint4 s_q[SETS][NB][NQ][SET];
    __shared__ float s_lse[SETS][NB][32];
    __shared__ int s_at[SETS][NB][32];  // the columns' positions
    __shared__ float s_sum[SETS][SW][2];
    const int lane = threadIdx.x & 63, n = lane & 31, hf = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int set = wave / SW, tid = threadIdx.x % (64 * SW);
    const int seq = blockIdx.y, Hkv = a.num_kv_heads, G = a.group, Hq = Hkv * G;
    const int q0 = a.q_start_loc[seq], Lc = a.q_start_loc[seq + 1] - q0;
    const int m = min(a.last, Lc);
    if (m <= 0) return;
    const int P = max(a.prefix_lens[seq], 0);
    const int T = static_cast<int>(min(min(static_cast<int64_t>(P) + Lc, static_cast<int64_t>(a.max_blocks_per_seq) * 16),
                                       static_cast<int64_t>(a.max_context_len)));
    const pa::WindowSpan span(P, Lc - m, Lc - 1, T, a.sink, a.window);
    const int entries = span.entries();
    if (2 * SW * static_cast<int>(blockIdx.x) >= entries) return;
    const int32_t* table = a.block_tables + static_cast<int64_t>(seq) * a.max_blocks_per_seq;

    // this wave's blocks, the same ones in all sets; a wave past the last has none, but brings operands
    const int e0 = 2 * (SW * static_cast<int>(blockIdx.x) + wave % SW);
    int lb[2], id[2];
#pragma unroll
    for (int u = 0; u < 2; u++) {
        lb[u] = e0 + u < entries ? span.block(e0 + u) : -1;
        id[u] = lb[u] >= 0 ? table[lb[u]] : -1;
        if (id[u] >= a.num_blocks) id[u] = -1;
    }
    const bool live = lb[0] >= 0;
    const int tok[2] = {live ? 16 * lb[0] : INT32_MAX - 64, lb[1] >= 0 ? 16 * lb[1] : INT32_MAX - 64};
    const int krow = pa::key_of_row(n);                                      // the lane's row of K: key krow of
    const int my_id = __builtin_amdgcn_readfirstlane(id[0]) >= 0 && (n < 16 || id[1] < 0) ? id[0] : id[1];  // its block, or the other where there is none
    const bool there[2] = {id[0] >= 0, id[1] >= 0};                          // (else the scores are set to 0)
    const bool plain = there[0] && there[1] && span.all_see_block(tok[0]) && span.all_see_block(tok[1]);

    const int columns = m * G, chunks = (columns + 31) / 32;
    // (KV head, chunk) by (KV head, chunk) in a row, cut evenly over the sets
    const int all = Hkv * chunks, first = set * all / SETS, steps = (set + 1) * all / SETS - first;
    const int most = (all + SETS - 1) / SETS;  // of any set: the barriers are the workgroup's
    // bf16 keys are their own operands: the next head's are loaded straight into the registers that the last chunk's products have left
    constexpr bool DIRECT = KV == PA_DTYPE_BF16;
    RawKeys<KV> raw[DIRECT ? 1 : NS] = {};
    uint4 kop[NP][NS] = {};
    auto load_keys = [&](int kvh) {
        if (my_id < 0) return;
        const char* const at = static_cast<const char*>(a.k_cache) +
                               ((static_cast<int64_t>(my_id) * Hkv + kvh) * 16 * D + krow * D + 8 * hf) * ELT;
#pragma unroll
        for (int sl = 0; sl < NS; sl++)
            if constexpr (DIRECT) kop[0][sl] = *reinterpret_cast<const uint4*>(at + 16 * sl * ELT);
            else load_raw<KV>(raw[sl], at + 16 * sl * ELT);
    };
    // Columns 32 chunk .. of KV head kvh: D / 8 threads bring a column, 16 (32) bytes of bf16 (fp32) each, so that a wave reads whole lines.
    // A lane reads piece 2 slab + half of column n: the pieces of a column lie at column ^ piece, so that the 16 threads that write them
    // at once meet 16 different 16-byte positions of a 256-byte line.
    constexpr int PC = D / 8, STEP = 64 * SW / PC;  // pieces of a column, columns at a time
    struct Bring {
        RawKeys<QKV> x[PER];
        float lse;
        int at;
    };
    const int piece = tid % PC;
    // of the columns that are loaded next: how many steps', which; query and head of the chunk's first column
    int left = steps, load_kvh = first / chunks, load_chunk = first % chunks, load_i = 32 * load_chunk / G, load_g = 32 * load_chunk % G;
    const int add_i = 32 / G, add_g = 32 % G;
    const float per_g = 1.0f / static_cast<float>(G);
    auto load_columns = [&](Bring& to) {
        if (left-- <= 0) return;
        const int kvh = load_kvh, chunk = load_chunk, i0 = load_i, g0 = load_g;
        const bool wrap = chunk == chunks - 1;
        load_chunk = wrap ? 0 : chunk + 1;
        load_kvh = wrap ? kvh + 1 : kvh;
        load_g = wrap ? 0 : g0 + add_g >= G ? g0 + add_g - G : g0 + add_g;
        load_i = wrap ? 0 : i0 + add_i + (g0 + add_g >= G);
        // (the quotient of a number below G + 32 by G, exact: its half above a whole number outweighs what the product is off by)
        const auto row_of = [&](int col, int& i) {
            const int x = g0 + min(col, columns - 1 - 32 * chunk), by = static_cast<int>((static_cast<float>(x) + 0.5f) * per_g);
            i = i0 + by;
            return (static_cast<int64_t>(q0) + Lc - m + i) * Hq + kvh * G + (x - by * G);
        };
        int i;
#pragma unroll
        for (int j = 0; j < PER; j++) {
            if (STEP > 32 && tid >= 32 * PC) break;
            load_raw<QKV>(to.x[j], static_cast<const char*>(a.q) + (row_of(tid / PC + STEP * j, i) * D + 8 * piece) * (QF32 ? 4 : 2));
        }
        if (tid < 32) {
            const int64_t row = row_of(tid, i);
            to.lse = 32 * chunk + tid < columns ? a.lse[row] * 1.4426950408889634f : INFINITY;  // no such column: no weight
            to.at = P + Lc - m + i;
        }
    };
    auto store_columns = [&](const Bring& from, int b) {
#pragma unroll
        for (int j = 0; j < PER; j++) {
            if (STEP > 32 && tid >= 32 * PC) break;
            uint4 op[NQ];
            raw_planes<QKV, NQ, false>(from.x[j], op);
#pragma unroll
            for (int q = 0; q < NQ; q++) s_q[set][b][q][32 * piece + ((tid / PC + STEP * j) ^ (piece & 15))] = op[q];
        }
        if (tid < 32) {
            s_lse[set][b][tid] = from.lse;
            s_at[set][b][tid] = from.at;
        }
    };
    const float c2 = a.scale * 1.4426950408889634f;
    float sum[2] = {0.0f, 0.0f}, f[2] = {c2, c2};
    Bring bring;  // the next step's columns, on their way while one is computed
    int kvh = load_kvh, chunk = load_chunk;  // of step k
    if (steps > 0) {
        if (EARLY || DIRECT) load_keys(kvh);
        load_columns(bring);
        store_columns(bring, 0);
    }
    for (int k = 0; k < most; k++) {
        const int b = NB == 2 ? k & 1 : 0;
        lds_barrier();  // step k's operands stand in LDS
        load_columns(bring);
        if (k < steps && live) {
            if (k == 0 || chunk == 0) {
                if constexpr (!DIRECT) {
                    if (!EARLY) load_keys(kvh);
#pragma unroll
                    for (int sl = 0; sl < NS; sl++) {
                        uint4 x[NP];
                        raw_planes<KV, NP, NQ == 3>(raw[sl], x);
#pragma unroll
                        for (int p = 0; p < NP; p++) kop[p][sl] = x[p];
                    }
                }
                if constexpr (I8)
#pragma unroll
                    for (int u = 0; u < 2; u++) f[u] = there[u] ? c2 * a.k_scale[static_cast<int64_t>(id[u]) * Hkv + kvh] : c2;
                if (!DIRECT && EARLY && (kvh + 1) * chunks < first + steps) load_keys(kvh + 1);
            }
            pa::f32x16_t product;
#pragma unroll
            for (int e = 0; e < 16; e++) product[e] = 0.0f;
#pragma unroll
            for (int sl = 0; sl < NS; sl++)
#pragma unroll
                for (int q = 0; q < NQ; q++) {
                    const uint4 qop = s_q[set][b][q][32 * (2 * sl + hf) + (n ^ ((2 * sl + hf) & 15))];
#pragma unroll
                    for (int p = 0; p < NP; p++)
                        if (p + q <= 2) product = pa::mfma32(kop[p][sl], qop, product);
                }
            const float lse = s_lse[set][b][n];
            const int at = s_at[set][b][n];
            // (single values from here on: hipcc has mixed up the elements of a product that was changed in place under a branch)
            float x[16];
#pragma unroll
            for (int e = 0; e < 16; e++) x[e] = e == 15 ? pa::settled(product[e]) : product[e];
            if (DIRECT && chunk == chunks - 1 && k + 1 < steps) load_keys(kvh + 1);
            if (plain) {
#pragma unroll
                for (int u = 0; u < 2; u++)
#pragma unroll
                    for (int j = 0; j < 8; j++) sum[u] += __builtin_amdgcn_exp2f(__builtin_fmaf(x[8 * u + j], f[u], -lse));
            } else {
                const int hi = min(T, at + 1), lo = a.window > 0 ? max(0, at + 1 - a.window) : 0;
#pragma unroll
                for (int u = 0; u < 2; u++)
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const int t = tok[u] + 8 * hf + j;
                        const float y = __builtin_fmaf(there[u] ? x[8 * u + j] : 0.0f, f[u], -lse);
                        // (an unseen token's weight is 0 whatever its score, the block's scale and the logarithm are)
                        sum[u] += t < hi && (t >= lo || t < span.sink) ? __builtin_amdgcn_exp2f(y) : 0.0f;
                    }
            }
        }
        if (NB == 1) lds_barrier();
        if (k + 1 < steps) store_columns(bring, NB == 2 ? b ^ 1 : 0);
        chunk = chunk == chunks - 1 ? 0 : chunk + 1;
        kvh = chunk == 0 ? kvh + 1 : kvh;
    }
#pragma unroll
    for (int u = 0; u < 2; u++) {
        const float w = pa::wave_sum(sum[u]);
        if (lane == 0) s_sum[set][wave % SW][u] = w;
    }
    __syncthreads();
    if (set == 0 && lane < 2 && (lane ? lb[1] : lb[0]) >= 0) {
        float w = s_sum[0][wave][lane];
#pragma unroll
        for (int i = 1; i < SETS; i++) w += s_sum[i][wave][lane];
        a.mass[static_cast<int64_t>(seq) * a.max_blocks_per_seq + (lane ? lb[1] : lb[0])] += w;
    }
}

template <int D>
void launch(const MassArgs& a, int kv, bool q_f32, bool few, dim3 grid, hipStream_t s) {
    const auto by_few = [&](auto k, auto q) {
        constexpr int KV = decltype(k)::value;
        constexpr bool Q = decltype(q)::value;
        if constexpr (mass_has_few(D, KV, Q)) {
            if (few) {
                prefill_mass_kernel<D, KV, Q, true><<<grid, mass_threads(D, KV, Q, true), 0, s>>>(a);
                return;
            }
        }
        prefill_mass_kernel<D, KV, Q, false><<<grid, mass_threads(D, KV, Q, false), 0, s>>>(a);
    };
    const auto by_q = [&](auto k) {
        if (q_f32) by_few(k, std::true_type());
        else by_few(k, std::false_type());
    };
    if (kv == PA_DTYPE_FP32) by_q(std::integral_constant<int, PA_DTYPE_FP32>());
    else if (kv == PA_DTYPE_BF16) by_q(std::integral_constant<int, PA_DTYPE_BF16>());
    else if constexpr (D >= 64) by_q(std::integral_constant<int, PA_DTYPE_INT8>());
}

// Workgroups of eight blocks up to which workgroups of two (so at most one a CU) share the work: every step's operands are then formed four times
// as often, but a set has an eighth of the steps instead of half (fp32 queries: a sixth, a quarter). Measured at (32, 8, 128) bf16, eight / two: one
// prompt of 500 tokens, 46 queries 35 / 16 us, of 8000 (63 workgroups of eight) 36 / 17, of 16000 38 / 33, of 30000 42 / 64; 16 of 500, 16 queries
// 19 / 10; fp32 queries 46 / 32, 47 / 36, 51 / 70, 55 / 133; 23 / 18.
constexpr int64_t kFewGroups = 64;

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
    if (static_cast<int64_t>(last_queries) * cfg->num_q_heads > INT32_MAX / 2)
        return pa::set_error(PA_ERROR_UNSUPPORTED, std::string(f) + ": last_queries * num_q_heads must fit 30 bits");
    if (cfg->num_q_heads / cfg->num_kv_heads > 1 << 20)
        return pa::set_error(PA_ERROR_UNSUPPORTED, std::string(f) + ": num_q_heads / num_kv_heads must be <= 2^20");
    if (num_seqs == 0 || last_queries == 0 || max_context_len == 0 || max_blocks_per_seq == 0) return pa::clear_error();
    int64_t blocks = std::min<int64_t>((static_cast<int64_t>(max_context_len) + 15) / 16, max_blocks_per_seq);
    if (window > 0)
        blocks = std::min(blocks, (static_cast<int64_t>(std::min(sink_tokens, max_context_len)) + 15) / 16 +
                                      (static_cast<int64_t>(window) + last_queries + 14) / 16 + 1);
    const bool q_f32 = cfg->q_dtype == PA_DTYPE_FP32;
    const bool few = mass_has_few(cfg->head_dim, cfg->kv_dtype, q_f32) && num_seqs * ((blocks + 7) / 8) <= kFewGroups;
    const int64_t a_group = 2 * mass_waves(few), groups = (blocks + a_group - 1) / a_group;
    if (!pa::fits_grid(groups, mass_threads(cfg->head_dim, cfg->kv_dtype, q_f32, few)))
        return pa::set_error(PA_ERROR_UNSUPPORTED, std::string(f) + ": too many blocks for one call");
    if (!q || !lse || !q_start_loc || !prefix_lens || !k_cache || !block_tables || !block_mass)
        return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": null pointer");
    if (cfg->kv_dtype == PA_DTYPE_INT8 && !k_scale)
        return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": int8 cache needs k_scale");
    if (!pa::aligned16(k_cache) || !pa::aligned16(q))
        return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": q and k_cache must be 16-byte aligned");
    const MassArgs a{q,          lse,       q_start_loc,       prefix_lens,          k_cache,         k_scale,
                     block_tables, block_mass, cfg->num_kv_heads, cfg->num_q_heads / cfg->num_kv_heads, max_blocks_per_seq,
                     cfg->num_blocks, max_context_len, last_queries, sink_tokens, window, pa::resolve_scale(cfg)};
    pa::StreamDevice dev(stream);
    hipStream_t s = pa::native(stream);
    const dim3 grid(static_cast<uint32_t>(groups), num_seqs);
    switch (cfg->head_dim) {
        case 32: launch<32>(a, cfg->kv_dtype, q_f32, few, grid, s); break;
        case 64: launch<64>(a, cfg->kv_dtype, q_f32, few, grid, s); break;
        case 128: launch<128>(a, cfg->kv_dtype, q_f32, few, grid, s); break;
        default: launch<256>(a, cfg->kv_dtype, q_f32, few, grid, s); break;
    }
    PA_HIP_CHECK(hipGetLastError());
    return pa::clear_error();
}
