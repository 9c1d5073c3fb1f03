// window_prefill.h -- attention of chunks of query tokens, each over a sliding window and a few first tokens that stay visible.
//
// For sequence s, the query at position p = prefix + i of its chunk, KV head h and query head g of its group, over the tokens t
// with t <= p and (t > p - window or t < sink) (window 0: all t <= p):
//   s_t = scale * q_g . k_t,  out = sum_t exp(s_t - max s) v_t / sum_t exp(s_t - max s),  lse = ln sum_t exp(s_t)
//
// The (query, query head) pairs of one (sequence, KV head), query by query, are the columns of the matrix products: a wave
// takes 32 of them, whatever the ratio of heads is, and streams the blocks that any of them sees through LDS, two at a time.
// Per pair of blocks, on v_mfma_f32_32x32x16_bf16:
//   S^T[32 keys][32 columns] = K . Q^T, whose rows are permuted so that a lane ends up with 8 consecutive tokens of each block for
//     its column;
//   O^T[D][32 columns] += V^T . P^T, whose P operand is what the lane then holds and whose accumulators belong to the lane's
//     own column: maxima, sums and the rescale need one exchange with the other half of the wave.
// Tiles go from memory straight into LDS (16-byte loads with the LDS bit, in inline asm with explicit waits) in the cache's type. Where
// columns are many, the four waves of a workgroup take 32 each and share a ring of pairs, two of them in flight; where they are
// few, the waves share the columns and every one streams pairs of its own through a slot of its own, without a barrier: the next
// pair's keys go out when this pair's have been read, its values likewise, and the waves' states meet at the end.
// Results are as exact as fp32 sums of exact products: bf16 keys and values and int8 codes are one bf16 operand, fp32 values
// (queries, probabilities, caches) the sum of three (8 bits each); where both operands are such, at most 2^-22 of a product is left out
// (bf16_planes_near). (With probabilities of two rounded parts results are 2.5e-6 from 64 bits, so 0.4e-6.)
// What bounds it: few columns, memory (32 sequences, 3-5 tokens each over a window of 1024, (32, 8, 128) bf16: 32 us, 27 traced, 5.2 TB/s); many, the
// matrix products and what is issued beside them in two waves a SIMD (8 x 512 tokens over that window 136 to 144 us, 2 x 4096 267 to 290 from card to
// card: 0.85 to 0.9 and 0.9 to 1.0 PFLOP/s counting the four products of exact probabilities, where a large matrix product reaches 1.26). On one card:
// probabilities in two fp16 parts, values converted in LDS by the waves, 163 and 317 us against 143 and 282 (registers); the next pair's scores
// beside this pair's probabilities 147 and 290. fp32 caches: 270 us for 16 x 42 tokens on 4982, (16, 4, 128).
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
// Eight values as three bf16 operands that sum to them.
__device__ __forceinline__ void bf16_planes(const float (&x)[8], uint4 (&plane)[3]) {
    uint32_t w[3][4];
#pragma unroll
    for (int e = 0; e < 4; e++) {
        float a[3], b[3];
        bf16_split3(x[2 * e], a);
        bf16_split3(x[2 * e + 1], b);
#pragma unroll
        for (int p = 0; p < 3; p++) w[p][e] = pack_bf16_trunc(a[p], b[p]);
    }
#pragma unroll
    for (int p = 0; p < 3; p++) plane[p] = make_uint4(w[p][0], w[p][1], w[p][2], w[p][3]);
}
// Two values rounded to the nearest in one conversion. (The empty asm keeps the conversions where they are written: prompts' masses of
// (32, 8, 128) 122 us for 166. The instruction itself in inline asm would read what v_exp_f32 has only just formed: hipcc sees to no wait there.)
typedef float f32x2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t pack_bf16_near(float lo, float hi) {
    uint32_t w = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t{lo, hi}), bf16x2_t));
    asm("" : "+v"(w));
    return w;
}
// As bf16_planes, the first and second operand rounded to the nearest instead of cut off, for one factor of products that have both
// in parts, where those of parts 1 x 2, 2 x 1 and 2 x 2 are left out. Of parts that are all cut off this is up to 2^-21 of a product (2 * 2^-7 *
// 2^-15), and always missing. Rounded parts are at most 2^-8 (the second) and 2^-17 (the third) of the value and of either sign, so it is
// less than 2^-22 (2^-8 * 2^-15 + 2^-17 * 2^-7), of either sign. The other factor stays cut off: the one that is split more often.
// LARGE: values that rounding would make infinite too.
template <bool LARGE>
__device__ __forceinline__ void bf16_planes_near(const float (&x)[8], uint4 (&plane)[3]) {
    const float most = __uint_as_float(0x7f7f0000u);  // the largest of bf16
    uint32_t w[3][4];
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const float a = x[2 * e], b = x[2 * e + 1];
        w[0][e] = LARGE ? pack_bf16_near(fminf(fmaxf(a, -most), most), fminf(fmaxf(b, -most), most)) : pack_bf16_near(a, b);
        const float ra = a - bf16_lo(w[0][e]), rb = b - bf16_hi(w[0][e]);
        w[1][e] = pack_bf16_near(ra, rb);
        w[2][e] = pack_bf16_trunc(ra - bf16_lo(w[1][e]), rb - bf16_hi(w[1][e]));
    }
#pragma unroll
    for (int p = 0; p < 3; p++) plane[p] = make_uint4(w[p][0], w[p][1], w[p][2], w[p][3]);
}
// Elements i .. i + 7 of the queries as NP bf16 operands (i a multiple of 8, the array 16-byte aligned). NEAR: of products with fp32 keys.
template <int NP, bool NEAR>
__device__ __forceinline__ void load_planes(const void* q, int64_t i, uint4 (&plane)[NP]) {
    if constexpr (NP == 1) {
        plane[0] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(q) + i);
    } else {
        const f32x4_t a = *reinterpret_cast<const f32x4_t*>(static_cast<const float*>(q) + i);
        const f32x4_t b = *reinterpret_cast<const f32x4_t*>(static_cast<const float*>(q) + i + 4);
        const float x[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
        if constexpr (NEAR) bf16_planes_near<true>(x, plane);
        else bf16_planes(x, plane);
    }
}
// Which of two bf16 are not finite: bit 15, bit 31.
__device__ __forceinline__ uint32_t bf16_odd(uint32_t w) { return ((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u; }
// A mask of those that are.
__device__ __forceinline__ uint32_t bf16_finite(uint32_t w) { return ~((bf16_odd(w) >> 15) * 0xffffu); }
__device__ __forceinline__ f32x16_t mfma32(const uint4& a, const uint4& b, const f32x16_t& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
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
    __device__ __forceinline__ bool all_see_block(int t) const { return t + 16 <= hi_all && (t >= lo_all || t + 16 <= sink); }
    __device__ __forceinline__ bool hides_some(int t) const { return !(t + 16 <= hi && (t >= lo || t + 16 <= sink)); }
    __device__ __forceinline__ bool none_see_block(int t) const { return t >= hi || (t + 16 <= lo && t >= sink); }
};

// A block's tiles in LDS, in 16-byte pieces: K row r (of 16), piece c (of RC) at kpos; V dim d, piece x (of ELT) at vpos. The 16 lanes
// that gfx950 serves in one clock (quads {0, 3, 5, 6} and {1, 2, 4, 7} of a half-wave) read one piece column of 16 different keys, or one
// piece of 16 dims; with these XORs they meet 16 different 16-byte positions of a 256-byte line (int8: 8 bytes of each).
template <int D, int ELT>
struct WindowTile {
    static constexpr int RC = D * ELT / 16, CH = 16 * RC;  // pieces per K row, per tile
    static constexpr int SEG = CH / 64;                     // loads of a wave per tile
    __device__ static constexpr int kswz(int r) { return RC >= 16 ? r : r * RC / 16 & (RC - 1); }
    __device__ static constexpr int vswz(int d) { return ELT == 2 ? (d >> 4) & 1 : ELT == 4 ? (d >> 2) & 3 : 0; }
    __device__ static constexpr int kpos(int r, int c) { return r * RC + (c ^ kswz(r)); }
    __device__ static constexpr int vpos(int d, int x) { return d * ELT + (x ^ vswz(d)); }
    // the memory piece that stands at position p (the XORs are their own inverse)
    __device__ static constexpr int ksrc(int p) { return p / RC * RC + (p % RC ^ kswz(p / RC)); }
    __device__ static constexpr int vsrc(int p) { return p / ELT * ELT + (p % ELT ^ vswz(p / ELT)); }
};

// Whether the waves of a workgroup may share 32 columns (the slots of four waves fit LDS).
__host__ __device__ constexpr bool window_shares(int d, int kv) { return kv != PA_DTYPE_FP32 || d <= 128; }
// Workgroups a CU holds: by LDS and registers.
__host__ __device__ constexpr int window_groups(int d, int kv) { return d <= 128 && kv != PA_DTYPE_FP32 ? 2 : 1; }

// What a column is: query token and head, the tokens it sees.
struct WindowColumn {
    int64_t row;  // of q, out and lse
    int hi, lo;
    __device__ __forceinline__ WindowColumn(const WindowPrefillArgs& a, int64_t c, int q0, int kvh, int P, int T) {
        const int i = static_cast<int>(c / a.group);
        row = (static_cast<int64_t>(q0) + i) * a.num_kv_heads * a.group + kvh * a.group + (c - static_cast<int64_t>(i) * a.group);
        hi = min(T, P + i + 1);
        lo = a.window > 0 ? max(0, P + i + 1 - a.window) : 0;
    }
    __device__ __forceinline__ bool sees(int t, int sink) const { return t < hi && (t >= lo || t < sink); }
    __device__ __forceinline__ bool any(int sink) const { return hi > lo || min(sink, hi) > 0; }
};

// SHARE: the waves share 32 columns and take pairs of blocks in turn; else each has 32 columns of its own and all take every pair.
template <int D, int KV, bool QF32, bool SHARE>
__global__ __launch_bounds__(256, window_groups(D, KV)) void window_prefill_kernel(const WindowPrefillArgs a) {
    constexpr bool F32 = KV == PA_DTYPE_FP32, I8 = KV == PA_DTYPE_INT8;
    constexpr int NP = F32 ? 3 : 1, NQ = QF32 ? 3 : 1, PP = 3;  // bf16 operands of a cache value, a query's, a probability's
    constexpr int ELT = F32 ? 4 : I8 ? 1 : 2;
    constexpr int NS = D / 16, ND = D / 32, COLS = SHARE ? 32 : 128;
    using TL = WindowTile<D, ELT>;
    constexpr int TILE = 16 * D, CH = TL::CH, SEG = TL::SEG, SLOT = 4 * CH;  // a slot: K, V of one block, K, V of the other
    constexpr int RING = F32 && D > 128 ? 2 : 3;                              // slots of the shared ring
    constexpr int AHEAD = SHARE ? 1 : RING - 1;                               // pairs in flight
    constexpr int STATE = 32 * D * 4 / 16;                                    // a wave's O in LDS
    constexpr int PIECES = SHARE ? 4 * (SLOT > STATE ? SLOT : STATE) : RING * SLOT;
    __shared__ uint4 s_tile[PIECES];
    __shared__ float2 s_ml[4][32];
    const int lane = threadIdx.x & 63, n = lane & 31, hf = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    __builtin_assume(wave >= 0 && wave < 4);
    const int split = blockIdx.y;
    int gi, wk;
    if (!place_workgroup(a.num_groups, a.per, gi, wk)) return;
    const int Hkv = a.num_kv_heads, G = a.group;
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
    const int entries = span.entries();
    const int pairs = (entries + 1) / 2, share = (pairs + a.splits - 1) / a.splits;
    const int pair0 = min(split * share, pairs), pair1 = min(pair0 + share, pairs);
    const int count = SHARE ? max(0, (pair1 - pair0 - wave + 3) / 4) : pair1 - pair0;  // this wave's pairs
    auto pair_of = [&](int j) { return SHARE ? pair0 + wave + 4 * j : pair0 + j; };

    // this wave's columns; those past the last are computed as the last and not stored
    const int64_t c_wave = c_wg + (SHARE ? 0 : 32 * wave);
    const bool live = c_wave < columns;
    const WindowSpan mine(P, static_cast<int>(min(c_wave, columns - 1) / G), static_cast<int>((min(columns, c_wave + 32) - 1) / G), T, a.sink, a.window);
    const WindowColumn col(a, min(c_wave + n, columns - 1), q0, kvh, P, T);

    uint4 qv[NQ][NS];
#pragma unroll
    for (int s = 0; s < NS; s++) {
        uint4 x[NQ];
        load_planes<NQ, F32>(a.q, col.row * D + 16 * s + 8 * hf, x);
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

    // ---- the stream ----
    // Ids (and int8 scales) of 32 pairs of this wave's at a time: lane l has block l % 2 of pair l / 2. The loads of the tiles are counted
    // by hand, so nothing else may be under way: the wave waits for a refill at once.
    int ids = -1;
    float ks_lane = 0.0f, vs_lane = 0.0f;
    auto refill = [&](int j) {
        const int pr = pair_of(j + (lane >> 1)), e = 2 * pr + (lane & 1);
        ids = -1;
        if (j + (lane >> 1) < count && e < entries) ids = table[span.block(e)];
        if (ids >= a.num_blocks) ids = -1;
        if constexpr (I8) {
            ks_lane = ids >= 0 ? a.k_scale[static_cast<int64_t>(ids) * Hkv + kvh] : 0.0f;
            vs_lane = ids >= 0 ? a.v_scale[static_cast<int64_t>(ids) * Hkv + kvh] : 0.0f;
        }
        __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
        asm volatile("" : "+v"(ids), "+v"(ks_lane), "+v"(vs_lane)::"memory");
    };
    uint32_t koff[SEG], voff[SEG];  // this lane's place in the tile of each load
#pragma unroll
    for (int j = 0; j < SEG; j++) {
        koff[j] = 16 * TL::ksrc(64 * j + lane);
        voff[j] = 16 * TL::vsrc(64 * j + lane);
    }
    const uint32_t base = lds_address(s_tile);
    const char* const kc = static_cast<const char*>(a.k_cache);
    const char* const vc = static_cast<const char*>(a.v_cache);
    // One tile into LDS; no such block reads as zeros through a zero-sized descriptor, so that every pair is as many loads.
    auto fetch = [&](const char* cache, const uint32_t (&off)[SEG], int id, uint32_t to) {
        const int64_t at = (static_cast<int64_t>(id >= 0 ? id : 0) * Hkv + kvh) * TILE * ELT;
        u32x4_t rsrc = buffer_rsrc_words(cache + at, id >= 0 ? TILE * ELT : 0);
#pragma unroll
        for (int i = 0; i < 4; i++) rsrc[i] = __builtin_amdgcn_readfirstlane(rsrc[i]);  // (uniform, but not seen to be everywhere)
#pragma unroll
        for (int j = 0; j < SEG; j++) lds_load16(rsrc, off[j], to + 1024 * j);
    };
    // SHARE: both blocks' K (or V) tiles into this wave's slot.
    auto fetch_own = [&](bool v, int j) {
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const int id = __builtin_amdgcn_readlane(ids, 2 * (j & 31) + u);
            fetch(v ? vc : kc, v ? voff : koff, id, base + 16 * (wave * SLOT + (2 * u + v) * CH));
        }
    };
    // Ring: wave w brings tile w % 2 (K, V) of block w / 2 of pair j.
    auto fetch_shared = [&](int j, int slot) {
        const int id = __builtin_amdgcn_readlane(ids, 2 * (j & 31) + (wave >> 1));
        const uint32_t to = base + 16 * (slot * SLOT + wave * CH);
        if (wave & 1) fetch(vc, voff, id, to);
        else fetch(kc, koff, id, to);
    };
    float sc[AHEAD + 1][4];  // int8: K and V scales of the pairs under way, [0]: of this one
    auto take_scales = [&](int at, int j) {
        if constexpr (I8) {
#pragma unroll
            for (int u = 0; u < 2; u++) {
                sc[at][u] = readlane_f(ks_lane, 2 * (j & 31) + u);
                sc[at][2 + u] = readlane_f(vs_lane, 2 * (j & 31) + u);
            }
        }
    };
    // The bf16 operands of 8 values that stand in `part` (fp32: and the piece behind it), masked by token where `keep` says so.
    auto operand = [&](const uint4* tile, int p0, int p1, uint4 (&op)[NP]) {
        if constexpr (I8) {
            const uint2 w = *reinterpret_cast<const uint2*>(reinterpret_cast<const char*>(tile + p0) + 8 * hf);
            const uint32_t x = w.x ^ 0x80808080u, y = w.y ^ 0x80808080u;
            op[0] = make_uint4(bf16_pair_of(x, 0), bf16_pair_of(x, 2), bf16_pair_of(y, 0), bf16_pair_of(y, 2));
        } else if constexpr (F32) {
            const f32x4_t x = __builtin_bit_cast(f32x4_t, tile[p0]), y = __builtin_bit_cast(f32x4_t, tile[p1]);
            const float v[8] = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
            bf16_planes(v, op);
        } else {
            op[0] = tile[p0];
        }
    };

    bool any_odd = false;  // values that are not finite have been met at tokens that some of the wave's columns see and others may not
    const int krow = key_of_row(n);
    auto compute = [&](const uint4* slot, int j, auto after_keys, auto before_values) {
        const int e0 = 2 * pair_of(j);
        const int tok[2] = {16 * span.block(e0), e0 + 1 < entries ? 16 * span.block(e0 + 1) : INT32_MAX - 64};  // no such block: past every end
        f32x16_t product;
#pragma unroll
        for (int i = 0; i < 16; i++) product[i] = 0.0f;
        const uint4* const kt = slot + (n >> 4) * 2 * CH;
#pragma unroll
        for (int sl = 0; sl < NS; sl++) {
            uint4 kop[NP];
            if constexpr (I8) operand(kt, TL::kpos(krow, sl), 0, kop);
            else if constexpr (F32) operand(kt, TL::kpos(krow, 4 * sl + 2 * hf), TL::kpos(krow, 4 * sl + 2 * hf + 1), kop);
            else operand(kt, TL::kpos(krow, 2 * sl + hf), 0, kop);
#pragma unroll
            for (int p = 0; p < NP; p++)
#pragma unroll
                for (int q = 0; q < NQ; q++)
                    if (p + q <= 2) product = mfma32(kop[p], qv[q][sl], product);
        }
        // (single values from here on: hipcc has mixed up the elements of a product that was changed in place under a branch)
        float s[16];
#pragma unroll
        for (int i = 0; i < 16; i++) s[i] = i == 15 ? settled(product[i]) : product[i];
        after_keys();
        // lane: tokens tok[u] + 8 hf + i of its column in s[8 u + i]
        float f[2] = {c2, c2};
        if constexpr (I8) {
#pragma unroll
            for (int u = 0; u < 2; u++) {
                f[u] = c2 * sc[0][u];
#pragma unroll
                for (int i = 0; i < 8; i++) s[8 * u + i] *= f[u];
                f[u] = 1.0f;
            }
        }
#pragma unroll
        for (int u = 0; u < 2; u++) {
            if (mine.all_see_block(tok[u])) continue;
#pragma unroll
            for (int i = 0; i < 8; i++) s[8 * u + i] = col.sees(tok[u] + 8 * hf + i, span.sink) ? s[8 * u + i] : -INFINITY;
        }
        float bm = s[0];
#pragma unroll
        for (int i = 1; i < 16; i++) bm = fmaxf(bm, s[i]);
        bm = halves_max(bm) * f[0];
        const bool grow = bm > m_run + 8.0f || (m_run == -INFINITY && bm > -INFINITY);
        if (__any(grow)) {
            const float m_new = grow ? bm : m_run;
            const float alpha = grow ? __builtin_amdgcn_exp2f(m_run - m_new) : 1.0f;
            l_run *= alpha;
            m_run = m_new;
#pragma unroll
            for (int t = 0; t < ND; t++) acc[t] *= alpha;
        }
        const float m0 = m_run == -INFINITY ? 0.0f : m_run;
#pragma unroll
        for (int i = 0; i < 16; i++) {
            s[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], f[0], -m0));
            l_run += s[i];
        }
        before_values();
#pragma unroll
        for (int u = 0; u < 2; u++) {
            uint4 pop[PP];
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                x[i] = s[8 * u + i];
                if constexpr (I8) x[i] = x[i] == 0.0f ? 0.0f : x[i] * sc[0][2 + u];  // (whatever the scale of an unseen block is)
            }
            if constexpr (F32) bf16_planes_near<false>(x, pop);
            else bf16_planes(x, pop);
            uint4 vop[ND][NP];
            const uint4* const vt = slot + (2 * u + 1) * CH;
#pragma unroll
            for (int t = 0; t < ND; t++) {
                const int d = 32 * t + n;
                if constexpr (I8) operand(vt, TL::vpos(d, 0), 0, vop[t]);
                else if constexpr (F32) operand(vt, TL::vpos(d, 2 * hf), TL::vpos(d, 2 * hf + 1), vop[t]);
                else operand(vt, TL::vpos(d, hf), 0, vop[t]);
            }
            if (!I8 && !mine.all_see_block(tok[u])) {
                if (mine.hides_some(tok[u])) {  // values that no column sees are zeros: what unused slots hold does not matter
                    uint32_t keep[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int t = tok[u] + 8 * hf + 2 * i;
                        keep[i] = (mine.some_see(t) ? 0xffffu : 0u) | (mine.some_see(t + 1) ? 0xffff0000u : 0u);
                    }
#pragma unroll
                    for (int t = 0; t < ND; t++)
#pragma unroll
                        for (int p = 0; p < NP; p++)
                            vop[t][p] = make_uint4(vop[t][p].x & keep[0], vop[t][p].y & keep[1], vop[t][p].z & keep[2], vop[t][p].w & keep[3]);
                }
                uint32_t odd = 0;
#pragma unroll
                for (int t = 0; t < ND; t++) odd |= bf16_odd(vop[t][0].x) | bf16_odd(vop[t][0].y) | bf16_odd(vop[t][0].z) | bf16_odd(vop[t][0].w);
                if (__any(odd != 0)) {  // they would reach columns that do not see them as 0 times them: zeros for now
                    any_odd = true;
#pragma unroll
                    for (int t = 0; t < ND; t++) {
                        const uint4 x = vop[t][0];
#pragma unroll
                        for (int p = 0; p < NP; p++) {
                            vop[t][p].x &= bf16_finite(x.x);
                            vop[t][p].y &= bf16_finite(x.y);
                            vop[t][p].z &= bf16_finite(x.z);
                            vop[t][p].w &= bf16_finite(x.w);
                        }
                    }
                }
            }
#pragma unroll
            for (int q = 0; q < PP; q++)
#pragma unroll
                for (int t = 0; t < ND; t++)
#pragma unroll
                    for (int p = 0; p < NP; p++)
                        if (p + q <= 2) acc[t] = mfma32(vop[t][p], pop[q], acc[t]);
        }
    };
    auto none_see = [&](int j) {
        const int e0 = 2 * pair_of(j);
        return mine.none_see_block(16 * span.block(e0)) && (e0 + 1 >= entries || mine.none_see_block(16 * span.block(e0 + 1)));
    };

    if constexpr (SHARE) {
        if (count > 0) {
            refill(0);
            fetch_own(false, 0);
            fetch_own(true, 0);
            take_scales(0, 0);
        }
        const uint4* const slot = s_tile + wave * SLOT;
        for (int j = 0; j < count; j++) {
            // (the next pair's loads go out from the ids of its own stretch; past the last they read nothing)
            const auto after_keys = [&]() {
                if (((j + 1) & 31) == 0) refill(j + 1);
                take_scales(AHEAD, j + 1);
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // this pair's keys have been read
                fetch_own(false, j + 1);
            };
            const auto before_values = [&]() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * SEG) : "memory"); };
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * SEG) : "memory");  // the keys have come, the values may be under way
            compute(slot, j, after_keys, before_values);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            fetch_own(true, j + 1);
#pragma unroll
            for (int i = 0; i < 4; i++) sc[0][i] = sc[AHEAD][i];
        }
    } else {
        refill(0);
#pragma unroll
        for (int j = 0; j < AHEAD; j++) {
            fetch_shared(j, j);
            take_scales(j, j);
        }
        int at = 0, to = AHEAD;  // slots of this pair and of the one that goes out
        for (int j = 0; j < count; j++) {
            // this wave's part of the pair has come, and with the barrier the others'; the slot to be filled has been read
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(SEG * (AHEAD - 1)) : "memory");
            if (((j + AHEAD) & 31) == 0) refill(j + AHEAD);
            fetch_shared(j + AHEAD, to);
            take_scales(AHEAD, j + AHEAD);
            if (live && !none_see(j)) compute(s_tile + at * SLOT, j, []() {}, []() {});
#pragma unroll
            for (int k = 0; k < AHEAD; k++)
#pragma unroll
                for (int i = 0; i < 4; i++) sc[k][i] = sc[k + 1][i];
            at = at == RING - 1 ? 0 : at + 1;
            to = to == RING - 1 ? 0 : to + 1;
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no write into LDS may outlive the stream

    // ---- the outcome ----
    const bool stored = live && c_wave + n < columns;
    const bool sees = col.any(span.sink);
    const int64_t slot0 = ((static_cast<int64_t>(gi) * a.per + wk) * a.splits + split) * COLS + (SHARE ? 0 : 32 * wave);
    auto finish = [&](int dim, f32x4_t o, float M, float L) {
        if (a.splits > 1) {
            *reinterpret_cast<f32x4_t*>(a.ws_o + (slot0 + n) * D + dim) = o;
            if (dim == 0) a.ws_ml[slot0 + n] = make_float2(M, L);
        } else {
            *reinterpret_cast<f32x4_t*>(a.out + col.row * D + dim) = sees ? o * (1.0f / L) : f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
            if (a.lse && dim == 0) a.lse[col.row] = sees ? (M + __builtin_amdgcn_logf(L)) * 0.6931471805599453f : -INFINITY;
        }
    };
    // The zeros that stood in for such values become NaN in the columns that see their tokens: how many of them a column sees in a channel is a
    // matrix product too, of the values' operand with 1 for each of them and the probabilities' with 1 for each token that is seen. (2 prompts
    // of 4096 whose values are all NaN: 1.1 times the time of finite ones; their columns one by one, a key at a time, 280 times. Looking at the
    // values of such blocks takes 5 % where they are most of what is read, windows of 64 at head size 64, else nothing that shows.)
    if constexpr (!I8) {
        if (any_odd) {
            for (int j = 0; j < 2 * count; j++) {
                const int e = 2 * pair_of(j >> 1) + (j & 1);
                if (e >= entries) continue;
                const int tok = 16 * span.block(e), id = table[tok / 16];
                if (id < 0 || id >= a.num_blocks || mine.all_see_block(tok)) continue;
                uint32_t sees[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int t = tok + 8 * hf + 2 * i;
                    sees[i] = (col.sees(t, span.sink) ? 0x3f80u : 0u) | (col.sees(t + 1, span.sink) ? 0x3f800000u : 0u);
                }
                const char* const tile = vc + (static_cast<int64_t>(id) * Hkv + kvh) * TILE * ELT;
#pragma unroll
                for (int t = 0; t < ND; t++) {
                    uint32_t odd[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const char* const at = tile + ((32 * t + n) * 16 + 8 * hf + 2 * i) * ELT;
                        odd[i] = F32 ? bf16_odd(pack_bf16_trunc(reinterpret_cast<const float*>(at)[0], reinterpret_cast<const float*>(at)[1]))
                                     : bf16_odd(*reinterpret_cast<const uint32_t*>(at));
                        odd[i] = (odd[i] >> 15) * 0x3f80u;
                    }
                    f32x16_t sum;
#pragma unroll
                    for (int i = 0; i < 16; i++) sum[i] = 0.0f;
                    sum = mfma32(make_uint4(odd[0], odd[1], odd[2], odd[3]), make_uint4(sees[0], sees[1], sees[2], sees[3]), sum);
                    sum = sum * 3e38f * 3e38f;  // 0 or infinite
                    acc[t] += sum - sum;
                }
            }
        }
    }
    const float l_tot = halves_sum(l_run);
    if constexpr (!SHARE) {
        if (!stored) return;
#pragma unroll
        for (int t = 0; t < ND; t++)
#pragma unroll
            for (int b = 0; b < 4; b++)
                finish(32 * t + 8 * b + 4 * hf, f32x4_t{acc[t][4 * b], acc[t][4 * b + 1], acc[t][4 * b + 2], acc[t][4 * b + 3]}, m_run, l_tot);
    } else {
        // every wave leaves its state; piece (t, b) of the dims is added up and stored by wave (4 t + b) % 4
        __syncthreads();
        const auto place = [&](int w, int i) -> uint4& { return s_tile[w * STATE + i * 64 + lane]; };
        if (hf == 0) s_ml[wave][n] = make_float2(m_run, l_tot);
#pragma unroll
        for (int t = 0; t < ND; t++)
#pragma unroll
            for (int b = 0; b < 4; b++)
                place(wave, 4 * t + b) = __builtin_bit_cast(uint4, f32x4_t{acc[t][4 * b], acc[t][4 * b + 1], acc[t][4 * b + 2], acc[t][4 * b + 3]});
        __syncthreads();
        if (!stored) return;
        float M = -INFINITY, L = 0.0f, f[4];
#pragma unroll
        for (int w = 0; w < 4; w++) M = fmaxf(M, s_ml[w][n].x);
#pragma unroll
        for (int w = 0; w < 4; w++) {
            const float2 x = s_ml[w][n];
            f[w] = x.x == M ? 1.0f : __builtin_amdgcn_exp2f(x.x - M);
            L += x.y * f[w];
        }
#pragma unroll
        for (int i = 0; i < 4 * ND; i++) {
            if (i % 4 != wave) continue;
            f32x4_t o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int w = 0; w < 4; w++) o += __builtin_bit_cast(f32x4_t, place(w, i)) * f[w];
            finish(32 * (i / 4) + 8 * (i % 4) + 4 * hf, o, M, L);
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

// share: the waves of a workgroup share 32 columns.
template <int D>
void launch_window_prefill(const WindowPrefillArgs& a, int kv_dtype, bool q_f32, bool share, uint32_t nwg, hipStream_t s) {
    const auto by_share = [&](auto kv, auto qf) {
        constexpr int KV = decltype(kv)::value;
        const dim3 grid(nwg, a.splits);
        if constexpr (window_shares(D, KV)) {
            if (share) {
                window_prefill_kernel<D, KV, decltype(qf)::value, true><<<grid, 256, 0, s>>>(a);
                return;
            }
        }
        window_prefill_kernel<D, KV, decltype(qf)::value, false><<<grid, 256, 0, s>>>(a);
    };
    const auto by_q = [&](auto kv) {
        if (q_f32) by_share(kv, std::true_type());
        else by_share(kv, std::false_type());
    };
    if (kv_dtype == PA_DTYPE_FP32) by_q(std::integral_constant<int, PA_DTYPE_FP32>());
    else if (kv_dtype == PA_DTYPE_BF16) by_q(std::integral_constant<int, PA_DTYPE_BF16>());
    else if constexpr (D >= 64) by_q(std::integral_constant<int, PA_DTYPE_INT8>());
    if (a.splits > 1) {
        const int64_t columns = static_cast<int64_t>(a.max_chunk_len) * a.group;
        window_prefill_merge_kernel<D><<<dim3(static_cast<uint32_t>((columns + 3) / 4), a.num_groups), 256, 0, s>>>(a, share ? 32 : 128);
    }
}
#ifndef PA_WINDOW_INSTANTIATE
extern template void launch_window_prefill<32>(const WindowPrefillArgs&, int, bool, bool, uint32_t, hipStream_t);
extern template void launch_window_prefill<64>(const WindowPrefillArgs&, int, bool, bool, uint32_t, hipStream_t);
extern template void launch_window_prefill<128>(const WindowPrefillArgs&, int, bool, bool, uint32_t, hipStream_t);
extern template void launch_window_prefill<256>(const WindowPrefillArgs&, int, bool, bool, uint32_t, hipStream_t);
#endif

}  // namespace pa
