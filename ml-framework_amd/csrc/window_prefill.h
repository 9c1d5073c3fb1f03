// window_prefill.h -- attention of chunks of query tokens, each over a sliding window and a few first tokens that stay visible.
//
// For sequence s, the query at position p = prefix + i of its chunk, KV head h and query head g of its group, over the tokens t
// with t <= p and (t > p - window or t < sink) (window 0: all t <= p):
//   s_t = scale * q_g . k_t,  out = sum_t exp(s_t - max s) v_t / sum_t exp(s_t - max s),  lse = ln sum_t exp(s_t)
//
// The (query, query head) pairs of one (sequence, KV head), query by query, are the columns of the matrix products: a wave
// takes 32 of them, whatever the ratio of heads is, and a workgroup streams the blocks that any of its columns
// sees through LDS, two at a time. Per pair of blocks, on v_mfma_f32_32x32x16_bf16:
//   S^T[32 keys][32 columns] = K . Q^T, whose rows are permuted so that a lane ends up with 8 consecutive tokens of each block for
//     its column;
//   O^T[D][32 columns] += V^T . P^T, whose P operand is what the lane then holds and whose accumulators belong to the lane's
//     own column: maxima, sums and the rescale need one exchange with the other half of the wave.
// Results are as exact as fp32 sums of exact products: bf16 keys and values and int8 codes are one bf16 operand, fp32 ones the sum of
// three (8 bits each), and so are fp32 queries; products of parts below 2^-24 are left out. P is two bf16 parts rounded to
// nearest (off by 2^-18 at most, 0.7e-6 in the mean square), three for fp32 caches.
#pragma once

#include <cfloat>

#include "decode_common.h"

namespace pa {

typedef float f32x16_t __attribute__((ext_vector_type(16)));

struct WindowPrefillArgs {
    float* out;
    float* lse;  // or null
    const void* q;
    const void* k_cache;
    const void* v_cache;
    const float* k_scale;
    const float* v_scale;
    const int32_t* q_start_loc;
    const int32_t* prefix_lens;
    const int32_t* block_tables;
    float* ws_o;    // parts of cut columns: [part][columns of a workgroup][D]
    float2* ws_ml;  // their (maximum, sum)
    int32_t num_kv_heads, group, max_blocks_per_seq, num_blocks, max_context_len, max_chunk_len;
    int32_t sink, window;
    float scale;
    int32_t per;         // workgroups (of different columns) per (sequence, KV head)
    int32_t num_groups;  // num_seqs * num_kv_heads
    int32_t splits;      // parts that a workgroup's keys are cut into
};

// Parts 0, 1, 2 of an fp32 value: its top 8 bits, the next 8, the rest; each exact in bf16.
__device__ __forceinline__ void bf16_split3(float x, float (&part)[3]) {
    part[0] = __uint_as_float(__float_as_uint(x) & 0xffff0000u);
    const float r = x - part[0];
    part[1] = __uint_as_float(__float_as_uint(r) & 0xffff0000u);
    part[2] = r - part[1];
}
// Eight values as NP bf16 operands: one (values that are exact in bf16) or three.
template <int NP>
__device__ __forceinline__ void bf16_planes(const float (&x)[8], uint4 (&plane)[NP]) {
    uint32_t w[NP][4];
#pragma unroll
    for (int e = 0; e < 4; e++) {
        if constexpr (NP == 1) {
            w[0][e] = pack_bf16_trunc(x[2 * e], x[2 * e + 1]);
        } else {
            float a[3], b[3];
            bf16_split3(x[2 * e], a);
            bf16_split3(x[2 * e + 1], b);
#pragma unroll
            for (int p = 0; p < NP; p++) w[p][e] = pack_bf16_trunc(a[p], b[p]);
        }
    }
#pragma unroll
    for (int p = 0; p < NP; p++) plane[p] = make_uint4(w[p][0], w[p][1], w[p][2], w[p][3]);
}
// Elements i .. i + 7 of a cache or of the queries as NP bf16 operands (i a multiple of 8, the array 16-byte aligned).
template <int KV, int NP>
__device__ __forceinline__ void load_planes(const void* base, int64_t i, uint4 (&plane)[NP]) {
    if constexpr (KV == PA_DTYPE_BF16) {
        static_assert(NP == 1, "bf16 is its own operand");
        plane[0] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + i);
    } else if constexpr (KV == PA_DTYPE_FP32) {
        const f32x4_t a = *reinterpret_cast<const f32x4_t*>(static_cast<const float*>(base) + i);
        const f32x4_t b = *reinterpret_cast<const f32x4_t*>(static_cast<const float*>(base) + i + 4);
        const float x[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
        bf16_planes<NP>(x, plane);
    } else {
        const uint2 w = *reinterpret_cast<const uint2*>(static_cast<const int8_t*>(base) + i);
        plane[0] = make_uint4(pack_i8pair(w.x, 0), pack_i8pair(w.x, 2), pack_i8pair(w.y, 0), pack_i8pair(w.y, 2));
    }
}
__device__ __forceinline__ f32x16_t mfma32(const uint4& a, const uint4& b, const f32x16_t& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}
// A value made where it stands. hipcc (ROCm 7.2) counts too few waits where a branch, taken, lies between a matrix instruction and the
// first read of its result: a product's last registers then lacked its last terms now and then (seen at 7 wait states of
// 11). What reads a product first is therefore kept in the product's own block by this.
__device__ __forceinline__ float settled(float x) {
    asm volatile("" : "+v"(x));
    return x;
}
// The other half of the wave's value joined with this lane's.
__device__ __forceinline__ float halves_max(float x) {
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float halves_sum(float x) {
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}
// The row of a 32-row operand is key (row % 16 permuted) of block row / 16: lane half hf then holds keys 8 hf .. 8 hf + 7 of
// block u in registers 8 u .. 8 u + 7 of the product.
__device__ __forceinline__ int key_of_row(int m) { return 8 * ((m >> 2) & 1) + 4 * ((m >> 3) & 1) + (m & 3); }

// What the columns of a chunk's queries [i0, i1] see of a context of T tokens: tokens [0, sink) and [lo, hi), every column
// those of [lo_all, hi_all) too. Blocks [0, first), then [low, end).
struct WindowSpan {
    int lo, hi, lo_all, hi_all, sink, first, low, end;
    __device__ __forceinline__ WindowSpan(int P, int i0, int i1, int T, int sinks, int window) {
        hi = min(T, P + i1 + 1);
        hi_all = min(T, P + i0 + 1);
        lo = window > 0 ? max(0, P + i0 + 1 - window) : 0;
        lo_all = window > 0 ? max(0, P + i1 + 1 - window) : 0;
        sink = min(sinks, T);
        low = lo / 16;
        end = max(low, (hi + 15) / 16);
        first = min((min(sink, hi) + 15) / 16, low);
    }
    __device__ __forceinline__ int entries() const { return first + end - low; }
    __device__ __forceinline__ int block(int e) const { return e < first ? e : e - first + low; }
    __device__ __forceinline__ bool some_see(int t) const { return t < hi && (t >= lo || t < sink); }
    __device__ __forceinline__ bool all_see(int t) const { return t < hi_all && (t >= lo_all || t < sink); }
    __device__ __forceinline__ bool all_see_block(int t) const { return t + 16 <= hi_all && (t >= lo_all || t + 16 <= sink); }
    __device__ __forceinline__ bool none_see_block(int t) const { return t >= hi || (t + 16 <= lo && t >= sink); }
};

// LDS: operands of 8 values (16 bytes). K row r (of 16), operand column c (of D / 8) at kpos; V dim d, tokens 8 h .. at vpos. The
// 16 lanes that gfx950 serves in one clock (quads {0, 3, 5, 6} and {1, 2, 4, 7} of a half-wave) then read 16 different
// 16-byte positions of a 256-byte line: their rows are 16 different keys, their dims 8 of either half of 32.
template <int D>
struct WindowTile {
    static constexpr int RC = D / 8, CHUNKS = 16 * RC;  // operands per K row, per tile
    __device__ static constexpr int kpos(int r, int c) {
        return RC >= 16 ? r * RC + (c ^ r) : r * RC + (c ^ ((r / (16 / RC)) & (RC - 1)));
    }
    __device__ static constexpr int vpos(int d, int h) { return 2 * d + (h ^ ((d >> 4) & 1)); }
};

// Waves that share a set of 32 columns where columns are few (each takes its own pair of blocks): as many as LDS has room for.
__host__ __device__ constexpr int window_key_waves(int d, int kv) { return kv != PA_DTYPE_FP32 || d <= 64 ? 4 : d == 128 ? 2 : 1; }

template <int D, int KV, bool QF32, int KS>
__global__ __launch_bounds__(256, D > 128 ? 1 : 2) void window_prefill_kernel(const WindowPrefillArgs a) {
    constexpr bool F32 = KV == PA_DTYPE_FP32, I8 = KV == PA_DTYPE_INT8;
    constexpr int NP = F32 ? 3 : 1, NQ = QF32 ? 3 : 1, PP = F32 ? 3 : 2;  // operands of a cache value, a query's, a probability's
    constexpr int NS = D / 16, ND = D / 32, SETS = 4 / KS, COLS = 32 * SETS;
    using TL = WindowTile<D>;
    constexpr int TILE = 16 * D, CH = TL::CHUNKS;
    __shared__ uint4 s_k[KS][2][NP][CH], s_v[KS][2][NP][CH];
    __shared__ float s_ks[2 * KS], s_vs[2 * KS];
    __shared__ float2 s_ml[4][32];
    __shared__ int s_bad[4];
    const int lane = threadIdx.x & 63, n = lane & 31, hf = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int set = wave / KS, ks = wave % KS;
    const int split = blockIdx.y;
    int gi, wk;
    if (!place_workgroup(a.num_groups, a.per, gi, wk)) return;
    const int Hkv = a.num_kv_heads, G = a.group, Hq = Hkv * G;
    const int seq = gi / Hkv, kvh = gi - seq * Hkv;
    const int q0 = a.q_start_loc[seq];
    const int Lc = min(a.q_start_loc[seq + 1] - q0, a.max_chunk_len);
    wk = a.per - 1 - wk;  // without a window the last columns have the most keys
    const int64_t columns = static_cast<int64_t>(Lc) * G, c_wg = static_cast<int64_t>(wk) * COLS;
    if (c_wg >= columns) return;
    const int P = max(a.prefix_lens[seq], 0);
    const int T = static_cast<int>(min(min(static_cast<int64_t>(P) + Lc, static_cast<int64_t>(a.max_blocks_per_seq) * 16),
                                       static_cast<int64_t>(a.max_context_len)));
    const WindowSpan span(P, static_cast<int>(c_wg / G), static_cast<int>((min(columns, c_wg + COLS) - 1) / G), T, a.sink, a.window);
    const int32_t* table = a.block_tables + static_cast<int64_t>(seq) * a.max_blocks_per_seq;
    // this workgroup's part of the list, in pairs of blocks
    const int pairs = (span.entries() + 1) / 2, share = (pairs + a.splits - 1) / a.splits;
    const int pair0 = min(split * share, pairs), pair1 = min(pair0 + share, pairs);

    // this wave's columns; those past the last are computed as the last and not stored
    const int64_t c_set = min(c_wg + 32 * set, columns - 1), c_end = min(columns, c_wg + 32 * set + 32);
    const bool live = c_wg + 32 * set < columns;
    const WindowSpan mine(P, static_cast<int>(c_set / G), static_cast<int>((max(c_end, c_set + 1) - 1) / G), T, a.sink, a.window);
    const int64_t col = min(c_wg + 32 * set + n, columns - 1);
    const int qi = static_cast<int>(col / G), head = kvh * G + static_cast<int>(col - static_cast<int64_t>(qi) * G);
    const int hi = min(T, P + qi + 1), lo = a.window > 0 ? max(0, P + qi + 1 - a.window) : 0;
    const int64_t qrow = (static_cast<int64_t>(q0) + qi) * Hq + head;

    uint4 qv[NQ][NS];
#pragma unroll
    for (int s = 0; s < NS; s++) {
        uint4 x[NQ];
        load_planes<QF32 ? PA_DTYPE_FP32 : PA_DTYPE_BF16, NQ>(a.q, qrow * D + 16 * s + 8 * hf, x);
#pragma unroll
        for (int p = 0; p < NQ; p++) qv[p][s] = x[p];
    }
    const float c2 = a.scale * 1.4426950408889634f;
    float m_run = -INFINITY, l_run = 0.0f;
    f32x16_t acc[ND];
#pragma unroll
    for (int t = 0; t < ND; t++)
#pragma unroll
        for (int i = 0; i < 16; i++) acc[t][i] = 0.0f;

    for (int pr = pair0; pr < pair1; pr += KS) {
        __syncthreads();
        for (int x = threadIdx.x; x < KS * 2 * 2 * CH; x += 256) {
            const int b = x / (2 * CH), y = x % (2 * CH), ch = y % CH;
            const bool is_v = y >= CH;
            const int e = 2 * pr + b;
            const int lb = span.block(min(e, max(span.entries() - 1, 0)));
            int id = e < span.entries() && e < 2 * pair1 ? table[lb] : -1;
            if (id >= a.num_blocks) id = -1;
            uint4 plane[NP];
#pragma unroll
            for (int p = 0; p < NP; p++) plane[p] = make_uint4(0, 0, 0, 0);
            if (id >= 0)
                load_planes<KV, NP>(is_v ? a.v_cache : a.k_cache, (static_cast<int64_t>(id) * Hkv + kvh) * TILE + 8 * ch, plane);
            if (!is_v) {
#pragma unroll
                for (int p = 0; p < NP; p++) s_k[b >> 1][b & 1][p][TL::kpos(ch / TL::RC, ch % TL::RC)] = plane[p];
            } else {
                const int t = 16 * lb + 8 * (ch & 1);
                uint32_t keep[4];  // values that no column sees are zeros: what unused slots hold does not matter
#pragma unroll
                for (int j = 0; j < 4; j++)
                    keep[j] = (span.some_see(t + 2 * j) ? 0xffffu : 0u) | (span.some_see(t + 2 * j + 1) ? 0xffff0000u : 0u);
#pragma unroll
                for (int p = 0; p < NP; p++)
                    s_v[b >> 1][b & 1][p][TL::vpos(ch >> 1, ch & 1)] =
                        make_uint4(plane[p].x & keep[0], plane[p].y & keep[1], plane[p].z & keep[2], plane[p].w & keep[3]);
            }
            if constexpr (I8) {
                if (y == 0) {
                    s_ks[b] = id >= 0 ? a.k_scale[static_cast<int64_t>(id) * Hkv + kvh] : 0.0f;
                    s_vs[b] = id >= 0 ? a.v_scale[static_cast<int64_t>(id) * Hkv + kvh] : 0.0f;
                }
            }
        }
        __syncthreads();
        const int e0 = 2 * (pr + ks);
        if (!live || pr + ks >= pair1) continue;
        const int tok0 = 16 * span.block(e0);
        const int tok1 = e0 + 1 < span.entries() ? 16 * span.block(e0 + 1) : INT32_MAX - 64;  // no such block: past every end
        if (mine.none_see_block(tok0) && mine.none_see_block(tok1)) continue;
        f32x16_t s;
#pragma unroll
        for (int i = 0; i < 16; i++) s[i] = 0.0f;
        const int krow = key_of_row(n);
#pragma unroll
        for (int sl = 0; sl < NS; sl++) {
            uint4 kop[NP];
#pragma unroll
            for (int p = 0; p < NP; p++) kop[p] = s_k[ks][n >> 4][p][TL::kpos(krow, 2 * sl + hf)];
#pragma unroll
            for (int p = 0; p < NP; p++)
#pragma unroll
                for (int q = 0; q < NQ; q++)
                    if (p + q <= 2) s = mfma32(kop[p], qv[q][sl], s);
        }
        // lane: tokens tok_u + 8 hf + j of its column in s[8 u + j]
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const float f = I8 ? c2 * s_ks[2 * ks + u] : c2;
#pragma unroll
            for (int j = 0; j < 8; j++) s[8 * u + j] = settled(s[8 * u + j] * f);
            const int tok = u ? tok1 : tok0;
            if (!mine.all_see_block(tok)) {
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const int t = tok + 8 * hf + j;
                    s[8 * u + j] = t < hi && (t >= lo || t < span.sink) ? s[8 * u + j] : -INFINITY;
                }
            }
        }
        float bm = s[0];
#pragma unroll
        for (int i = 1; i < 16; i++) bm = fmaxf(bm, s[i]);
        bm = halves_max(bm);
        const bool grow = bm > m_run + 8.0f || (m_run == -INFINITY && bm > -INFINITY);
        if (__any(grow)) {
            const float m_new = grow ? bm : m_run;
            const float alpha = grow ? __builtin_amdgcn_exp2f(m_run - m_new) : 1.0f;
            l_run *= alpha;
            m_run = m_new;
#pragma unroll
            for (int t = 0; t < ND; t++)
#pragma unroll
                for (int i = 0; i < 16; i++) acc[t][i] *= alpha;
        }
        const float m0 = m_run == -INFINITY ? 0.0f : m_run;
#pragma unroll
        for (int i = 0; i < 16; i++) {
            s[i] = __builtin_amdgcn_exp2f(s[i] - m0);
            l_run += s[i];
        }
#pragma unroll
        for (int u = 0; u < 2; u++) {
            uint4 pop[PP];
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                x[j] = s[8 * u + j];
                if constexpr (I8) x[j] = x[j] == 0.0f ? 0.0f : x[j] * s_vs[2 * ks + u];  // (whatever the scale of an unseen block is)
            }
            if constexpr (F32) {
                bf16_planes<PP>(x, pop);
            } else {
                uint32_t w[2][4];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    w[0][e] = pack_bf16_rne(x[2 * e], x[2 * e + 1]);
                    w[1][e] = pack_bf16_rne(x[2 * e] - bf16_lo(w[0][e]), x[2 * e + 1] - bf16_hi(w[0][e]));
                }
#pragma unroll
                for (int p = 0; p < 2; p++) pop[p] = make_uint4(w[p][0], w[p][1], w[p][2], w[p][3]);
            }
#pragma unroll
            for (int t = 0; t < ND; t++) {
                uint4 vop[NP];
#pragma unroll
                for (int p = 0; p < NP; p++) vop[p] = s_v[ks][u][p][TL::vpos(32 * t + n, hf)];
#pragma unroll
                for (int p = 0; p < NP; p++)
#pragma unroll
                    for (int q = 0; q < PP; q++)
                        if (p + q <= 2) acc[t] = mfma32(vop[p], pop[q], acc[t]);
            }
        }
    }

    // ---- the outcome ----
    const bool stored = live && c_wg + 32 * set + n < columns;
    const bool sees = hi > lo || min(span.sink, hi) > 0;  // the column has a token at all
    const int64_t slot = (static_cast<int64_t>(gi) * a.per + wk) * a.splits + split;
    auto finish = [&](int64_t row, int c, int dim, f32x4_t o, float M, float L, bool any) {
        if (a.splits > 1) {
            *reinterpret_cast<f32x4_t*>(a.ws_o + (slot * COLS + c) * D + dim) = o;
            if (dim == 0) a.ws_ml[slot * COLS + c] = make_float2(M, L);
        } else {
            *reinterpret_cast<f32x4_t*>(a.out + row * D + dim) = any ? o * (1.0f / L) : f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
            if (a.lse && dim == 0) a.lse[row] = any ? (M + __builtin_amdgcn_logf(L)) * 0.6931471805599453f : -INFINITY;
        }
    };
    // A value that is not finite at a token that some of the wave's columns see and others do not would reach
    // the others as 0 times it. Where the outcome is not finite the values of such tokens are looked at, and if that is the cause
    // the columns are computed again one by one (each over its own tokens only).
    bool done = false;
    if constexpr (!I8) {
        bool odd = !(fabsf(l_run) < INFINITY);
#pragma unroll
        for (int t = 0; t < ND; t++)
#pragma unroll
            for (int i = 0; i < 16; i++) odd |= !(fabsf(acc[t][i]) < INFINITY);
        bool redo = live && __any(odd);
        if constexpr (KS > 1) {
            if (lane == 0) s_bad[wave] = redo;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < KS; w++) redo |= s_bad[set * KS + w] != 0;
        }
        if (redo) {
            bool hit = false;
            for (int e = 2 * pair0; e < min(2 * pair1, span.entries()); e++) {
                const int tok = 16 * span.block(e);
                const int id = table[tok / 16];
                if (id < 0 || id >= a.num_blocks || mine.all_see_block(tok)) continue;
                for (int i = lane; i < TILE; i += 64) {
                    const int t = tok + (i & 15);
                    const int64_t at = (static_cast<int64_t>(id) * Hkv + kvh) * TILE + i;
                    const float v = F32 ? static_cast<const float*>(a.v_cache)[at] : bf16_to_f32(static_cast<const uint16_t*>(a.v_cache)[at]);
                    hit |= span.some_see(t) && !mine.all_see(t) && !(fabsf(v) < INFINITY);
                }
            }
            if (__any(hit)) {
                constexpr int DPL = (D + 63) / 64;
                if (KS == 1 || ks == 0) {
                    for (int c = 0; c < 32 && c_wg + 32 * set + c < columns; c++) {
                        const int64_t cc = c_wg + 32 * set + c;
                        const int i = static_cast<int>(cc / G), h = kvh * G + static_cast<int>(cc - static_cast<int64_t>(i) * G);
                        const int chi = min(T, P + i + 1), clo = a.window > 0 ? max(0, P + i + 1 - a.window) : 0;
                        const int64_t row = (static_cast<int64_t>(q0) + i) * Hq + h;
                        float qx[DPL], o[DPL], M = -INFINITY, L = 0.0f;
#pragma unroll
                        for (int k = 0; k < DPL; k++) {
                            const int64_t at = row * D + min(lane + 64 * k, D - 1);
                            qx[k] = QF32 ? static_cast<const float*>(a.q)[at] : bf16_to_f32(static_cast<const uint16_t*>(a.q)[at]);
                            if (lane + 64 * k >= D) qx[k] = 0.0f;
                            o[k] = 0.0f;
                        }
                        for (int e = 2 * pair0; e < min(2 * pair1, span.entries()); e++) {
                            const int tok = 16 * span.block(e);
                            int id = table[tok / 16];
                            if (id >= a.num_blocks) id = -1;
                            const int64_t tile = (static_cast<int64_t>(max(id, 0)) * Hkv + kvh) * TILE;
                            for (int j = 0; j < 16; j++) {
                                if (!(tok + j < chi && (tok + j >= clo || tok + j < span.sink))) continue;
                                float x = 0.0f, v[DPL];
#pragma unroll
                                for (int k = 0; k < DPL; k++) {
                                    const int d = min(lane + 64 * k, D - 1);
                                    const int64_t ka = tile + j * D + d, va = tile + d * 16 + j;
                                    const float kx = F32 ? static_cast<const float*>(a.k_cache)[ka] : bf16_to_f32(static_cast<const uint16_t*>(a.k_cache)[ka]);
                                    v[k] = F32 ? static_cast<const float*>(a.v_cache)[va] : bf16_to_f32(static_cast<const uint16_t*>(a.v_cache)[va]);
                                    if (id < 0) v[k] = 0.0f;
                                    if (lane + 64 * k < D && id >= 0) x = __builtin_fmaf(qx[k], kx, x);
                                }
                                x = wave_sum(x) * c2;
                                const float m_new = fmaxf(M, x);
                                const float f = m_new == M ? 1.0f : __builtin_amdgcn_exp2f(M - m_new);
                                const float p = __builtin_amdgcn_exp2f(x - (m_new == -INFINITY ? 0.0f : m_new));
                                L = L * f + p;
#pragma unroll
                                for (int k = 0; k < DPL; k++) o[k] = o[k] * f + p * v[k];
                                M = m_new;
                            }
                        }
                        const bool any = chi > clo || min(span.sink, chi) > 0;
#pragma unroll
                        for (int k = 0; k < DPL; k++) {
                            if (lane + 64 * k >= D) continue;
                            if (a.splits > 1) a.ws_o[(slot * COLS + 32 * set + c) * D + lane + 64 * k] = o[k];
                            else a.out[row * D + lane + 64 * k] = any ? o[k] * (1.0f / L) : 0.0f;
                        }
                        if (lane == 0) {
                            if (a.splits > 1) a.ws_ml[slot * COLS + 32 * set + c] = make_float2(M, L);
                            else if (a.lse) a.lse[row] = any ? (M + __builtin_amdgcn_logf(L)) * 0.6931471805599453f : -INFINITY;
                        }
                    }
                }
                done = true;  // (the set's waves agree: it follows from the same values)
            }
        }
    }
    const float l_tot = halves_sum(l_run);
    if constexpr (KS == 1) {
        if (!stored || done) return;
#pragma unroll
        for (int t = 0; t < ND; t++)
#pragma unroll
            for (int b = 0; b < 4; b++)
                finish(qrow, 32 * set + n, 32 * t + 8 * b + 4 * hf, f32x4_t{acc[t][4 * b], acc[t][4 * b + 1], acc[t][4 * b + 2], acc[t][4 * b + 3]},
                       m_run, l_tot, sees);
    } else {
        // every wave leaves its state; piece (t, b) of the dims is added up and stored by wave (4 t + b) % KS of the set
        f32x4_t* const s_o = reinterpret_cast<f32x4_t*>(&s_k[0][0][0][0]);
        static_assert(sizeof(s_k) >= 2 * 32 * D * sizeof(float), "half of the waves' states fit the keys' tiles");
        f32x4_t* const s_o2 = reinterpret_cast<f32x4_t*>(&s_v[0][0][0][0]);
        __syncthreads();
        const auto place = [&](int w, int i) -> f32x4_t* { return (w < 2 ? s_o : s_o2) + ((w & 1) * 4 * ND + i) * 64 + lane; };
        if (hf == 0) s_ml[wave][n] = make_float2(m_run, l_tot);
#pragma unroll
        for (int t = 0; t < ND; t++)
#pragma unroll
            for (int b = 0; b < 4; b++)
                *place(wave, 4 * t + b) = f32x4_t{acc[t][4 * b], acc[t][4 * b + 1], acc[t][4 * b + 2], acc[t][4 * b + 3]};
        __syncthreads();
        if (!stored || done) return;
        float M = -INFINITY, L = 0.0f, f[KS];
#pragma unroll
        for (int w = 0; w < KS; w++) M = fmaxf(M, s_ml[set * KS + w][n].x);
#pragma unroll
        for (int w = 0; w < KS; w++) {
            const float2 x = s_ml[set * KS + w][n];
            f[w] = x.x == M ? 1.0f : __builtin_amdgcn_exp2f(x.x - M);
            L += x.y * f[w];
        }
#pragma unroll
        for (int i = 0; i < 4 * ND; i++) {
            if (i % KS != ks) continue;
            f32x4_t o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int w = 0; w < KS; w++) o += *place(set * KS + w, i) * f[w];
            finish(qrow, 32 * set + n, 32 * (i / 4) + 8 * (i % 4) + 4 * hf, o, M, L, sees);
        }
    }
}

// The parts of columns whose keys were cut: a wave a column, lanes over dims.
template <int D>
__global__ __launch_bounds__(256) void window_prefill_merge_kernel(const WindowPrefillArgs a, int cols) {
    constexpr int DPL = (D + 63) / 64;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int gi = blockIdx.y;
    const int Hkv = a.num_kv_heads, G = a.group;
    const int seq = gi / Hkv, kvh = gi - seq * Hkv;
    const int q0 = a.q_start_loc[seq];
    const int Lc = min(a.q_start_loc[seq + 1] - q0, a.max_chunk_len);
    const int64_t col = static_cast<int64_t>(blockIdx.x) * 4 + wave;
    if (col >= static_cast<int64_t>(Lc) * G) return;
    const int qi = static_cast<int>(col / G), g = static_cast<int>(col - static_cast<int64_t>(qi) * G);
    const int P = max(a.prefix_lens[seq], 0);
    const int T = static_cast<int>(min(min(static_cast<int64_t>(P) + Lc, static_cast<int64_t>(a.max_blocks_per_seq) * 16),
                                       static_cast<int64_t>(a.max_context_len)));
    const int hi = min(T, P + qi + 1), lo = a.window > 0 ? max(0, P + qi + 1 - a.window) : 0;
    const bool sees = hi > lo || min(min(a.sink, T), hi) > 0;
    const int64_t base = (static_cast<int64_t>(gi) * a.per + col / cols) * a.splits;
    const auto part = [&](int sp) { return (base + sp) * cols + col % cols; };
    float M = -INFINITY, L = 0.0f, o[DPL];
    for (int sp = 0; sp < a.splits; sp++) M = fmaxf(M, a.ws_ml[part(sp)].x);
#pragma unroll
    for (int k = 0; k < DPL; k++) o[k] = 0.0f;
    for (int sp = 0; sp < a.splits; sp++) {
        const float2 x = a.ws_ml[part(sp)];
        const float f = x.x == M ? 1.0f : __builtin_amdgcn_exp2f(x.x - M);
        L += x.y * f;
#pragma unroll
        for (int k = 0; k < DPL; k++) o[k] += a.ws_o[part(sp) * D + min(lane + 64 * k, D - 1)] * f;
    }
    const int64_t row = (static_cast<int64_t>(q0) + qi) * Hkv * G + kvh * G + g;
#pragma unroll
    for (int k = 0; k < DPL; k++)
        if (lane + 64 * k < D) a.out[row * D + lane + 64 * k] = sees ? o[k] * (1.0f / L) : 0.0f;
    if (a.lse && lane == 0) a.lse[row] = sees ? (M + __builtin_amdgcn_logf(L)) * 0.6931471805599453f : -INFINITY;
}

// ks: waves that share a set of columns, 1 or window_key_waves.
template <int D>
void launch_window_prefill(const WindowPrefillArgs& a, int kv_dtype, bool q_f32, int ks, uint32_t nwg, hipStream_t s) {
    const auto go = [&](auto kv, auto qf, auto k) {
        constexpr int KV = decltype(kv)::value, KS = decltype(k)::value;
        window_prefill_kernel<D, KV, decltype(qf)::value, KS><<<dim3(nwg, a.splits), 256, 0, s>>>(a);
    };
    const auto by_ks = [&](auto kv, auto qf) {
        constexpr int KW = window_key_waves(D, decltype(kv)::value);
        if (KW > 1 && ks > 1) go(kv, qf, std::integral_constant<int, KW>());
        else go(kv, qf, std::integral_constant<int, 1>());
    };
    const auto by_q = [&](auto kv) {
        if (q_f32) by_ks(kv, std::true_type());
        else by_ks(kv, std::false_type());
    };
    if (kv_dtype == PA_DTYPE_FP32) by_q(std::integral_constant<int, PA_DTYPE_FP32>());
    else if (kv_dtype == PA_DTYPE_BF16) by_q(std::integral_constant<int, PA_DTYPE_BF16>());
    else if constexpr (D >= 64) by_q(std::integral_constant<int, PA_DTYPE_INT8>());
    if (a.splits > 1) {
        const int64_t columns = static_cast<int64_t>(a.max_chunk_len) * a.group;
        window_prefill_merge_kernel<D><<<dim3(static_cast<uint32_t>((columns + 3) / 4), a.num_groups), 256, 0, s>>>(a, 128 / ks);
    }
}
#ifndef PA_WINDOW_INSTANTIATE
extern template void launch_window_prefill<32>(const WindowPrefillArgs&, int, bool, int, uint32_t, hipStream_t);
extern template void launch_window_prefill<64>(const WindowPrefillArgs&, int, bool, int, uint32_t, hipStream_t);
extern template void launch_window_prefill<128>(const WindowPrefillArgs&, int, bool, int, uint32_t, hipStream_t);
extern template void launch_window_prefill<256>(const WindowPrefillArgs&, int, bool, int, uint32_t, hipStream_t);
#endif

}  // namespace pa
