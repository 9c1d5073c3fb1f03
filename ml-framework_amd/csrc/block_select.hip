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
// sixteenth of the K and V bytes): a wave per 32 blocks of a KV head (int8: 128), 16-byte loads. The choice is
// one workgroup per (query token, KV head): see block_choose_kernel. (Both in one launch, a workgroup a row, is slower at
// every size tried: one row of 313 blocks 10.7 us where this takes 9.1, 512 rows 26.6 and 21.4.)
#include <algorithm>
#include <string>

#include "pa_internal.h"

namespace {

constexpr int kScoreWaves = 4;
constexpr int kScoreBlocks = 64;      // blocks per wave at most: a lane per block id
constexpr int64_t kScoreWorkers = 4096;  // waves that fill the chip
constexpr int kQueryTile = 4;         // queries scored together where sequences have several
constexpr int kMaxBlocks = 1 << 17;   // blocks of one context: the choice's bit masks in LDS

struct SelectArgs {
    const void* q;
    const void* bounds;
    const float* k_scale;
    const int32_t* tables;
    const int32_t* query_seqs;  // null: query r belongs to sequence r
    const int32_t* context_lens;
    double* scores;             // [num_queries][Hkv][max_blocks]
    uint4* digits;              // int8: [num_queries][Hkv][kDigits][2 D] bytes
    double* units;              // int8: [num_queries][Hkv]
    int32_t* selected;          // [num_queries][Hkv][budget]
    int32_t num_seqs, width, num_queries, max_blocks, max_len;
    int32_t hkv, group, num_blocks;
    int32_t sink, recent, budget;
    int32_t q_bf16;
};

// Blocks of a context of `len` tokens.
__device__ __forceinline__ int blocks_of(const SelectArgs& a, int len) {
    len = min(min(len, a.max_len), static_cast<int>(min(static_cast<int64_t>(a.width) * 16, static_cast<int64_t>(INT32_MAX))));
    return len <= 0 ? 0 : (len - 1) / 16 + 1;
}
// Blocks of query r's context, 0 if its sequence is out of range.
__device__ __forceinline__ int context_blocks(const SelectArgs& a, int r) {
    const int seq = a.query_seqs ? a.query_seqs[r] : r;
    return seq < 0 || seq >= a.num_seqs ? 0 : blocks_of(a, a.context_lens[r]);
}

// Element e of a 16-byte word of bounds (exact).
template <int KV>
__device__ __forceinline__ float elem(const uint4& w, int e) {
    const uint32_t x[4] = {w.x, w.y, w.z, w.w};
    if constexpr (KV == PA_DTYPE_FP32) return __uint_as_float(x[e]);
    else return e & 1 ? pa::bf16_hi(x[e >> 1]) : pa::bf16_lo(x[e >> 1]);
}

typedef int i32x4 __attribute__((ext_vector_type(4)));
// Bounds are read once: non-temporal loads (32 sequences of 8k to 32k tokens, 8 heads of 128 channels, bf16: 35.3 us
// a selection, 39.9 with ordinary ones; as the int8 kernel below has it).
__device__ __forceinline__ uint4 load_once(const uint4* p) {
    return __builtin_bit_cast(uint4, __builtin_nontemporal_load(reinterpret_cast<const i32x4*>(p)));
}

struct Words {
    uint32_t lo, hi;
};
__device__ __forceinline__ Words words(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    return {static_cast<uint32_t>(u), static_cast<uint32_t>(u >> 32)};
}
__device__ __forceinline__ double from_words(uint32_t lo, uint32_t hi) {
    return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}
template <int CTRL, int BANKS = 0xF>
__device__ __forceinline__ uint32_t dpp(uint32_t old, uint32_t src) {
    return __builtin_amdgcn_update_dpp(old, src, CTRL, 0xF, BANKS, false);
}
// a summed over lane pairs 32 (16, 8) apart in the lower lanes of each pair, b in the upper ones: one exchange
// for two sums.
__device__ __forceinline__ double pair32(double a, double b) {
    const Words x = words(a), y = words(b);
    const auto lo = __builtin_amdgcn_permlane32_swap(x.lo, y.lo, false, false);
    const auto hi = __builtin_amdgcn_permlane32_swap(x.hi, y.hi, false, false);
    return from_words(lo[0], hi[0]) + from_words(lo[1], hi[1]);
}
__device__ __forceinline__ double pair16(double a, double b) {
    const Words x = words(a), y = words(b);
    const auto lo = __builtin_amdgcn_permlane16_swap(x.lo, y.lo, false, false);
    const auto hi = __builtin_amdgcn_permlane16_swap(x.hi, y.hi, false, false);
    return from_words(lo[0], hi[0]) + from_words(lo[1], hi[1]);
}
__device__ __forceinline__ double pair8(double a, double b) {
    const Words x = words(a), y = words(b);  // row_ror:8 into lanes 8 .. 15 of a row, and into lanes 0 .. 7
    return from_words(dpp<0x128, 0xC>(x.lo, y.lo), dpp<0x128, 0xC>(x.hi, y.hi)) +
           from_words(dpp<0x128, 0x3>(y.lo, x.lo), dpp<0x128, 0x3>(y.hi, x.hi));
}
// v summed over each group of 8 lanes.
__device__ __forceinline__ double sum8(double v) {
    Words x = words(v);
    v += from_words(dpp<0xB1>(x.lo, x.lo), dpp<0xB1>(x.hi, x.hi));
    x = words(v);
    v += from_words(dpp<0x4E>(x.lo, x.lo), dpp<0x4E>(x.hi, x.hi));
    x = words(v);
    return v + from_words(dpp<0x141>(x.lo, x.lo), dpp<0x141>(x.hi, x.hi));
}

// v summed with the value 16 or 8 lanes away.
template <int O>
__device__ __forceinline__ double sum_across(double v) {
    return O == 16 ? pair16(v, v) : pair8(v, v);
}

// Queries scored together: r[t], and the end of its scored blocks in the chunk that starts at `first`.
template <int QT>
struct QueryGroup {
    int r[QT], end[QT];
    int count, last;
    __device__ __forceinline__ void add(const SelectArgs& a, int query, int nblk, int first, int per) {
        // nothing to choose, or no block of the chunk takes part: the end is not past the start
        const int e = nblk > a.budget ? min(first + per, nblk - a.recent) : 0;
#pragma unroll
        for (int t = 0; t < QT; t++)
            if (t == count) {
                r[t] = query;
                end[t] = e;
            }
        count++;
        last = max(last, e);
    }
    __device__ __forceinline__ void clear() {
        count = last = 0;
#pragma unroll
        for (int t = 0; t < QT; t++) r[t] = end[t] = 0;
    }
};

// f(group, sequence, id) for the queries of unit `unit`: the query itself, or (QT > 1) all those of sequence
// `unit`, QT at a time. id: the sequence's table entry at block `at` of its context, read without waiting for the
// context's length (any value past it). Everything else is the same in all lanes of the wave.
template <int QT, typename F>
__device__ __forceinline__ void for_query_groups(const SelectArgs& a, int unit, int first, int per, int at, F&& f) {
    QueryGroup<QT> g;
    g.clear();
    if constexpr (QT == 1) {
        const int seq = a.query_seqs ? a.query_seqs[unit] : unit;
        const bool some = seq >= 0 && seq < a.num_seqs;
        const int id = some ? a.tables[static_cast<int64_t>(seq) * a.width + min(at, a.width - 1)] : -1;
        g.add(a, unit, some ? blocks_of(a, a.context_lens[unit]) : 0, first, per);
        if (g.last > first) f(g, seq, id);
    } else {
        const int lane = threadIdx.x & 63;
        const int id = a.tables[static_cast<int64_t>(unit) * a.width + min(at, a.width - 1)];
        uint64_t of = 0;  // queries of the sequence among the 64 before j0 that are still to do
        int j0 = 0, len = 0;
        for (;;) {
            while (g.count < QT) {
                if (of) {
                    const int k = __builtin_ctzll(of);
                    of &= of - 1;
                    g.add(a, j0 - 64 + k, blocks_of(a, __builtin_amdgcn_readlane(len, k)), first, per);
                } else if (j0 < a.num_queries) {
                    const int j = min(j0 + lane, a.num_queries - 1);
                    len = a.context_lens[j];
                    of = __ballot(j0 + lane < a.num_queries && a.query_seqs[j] == unit);
                    j0 += 64;
                } else {
                    break;
                }
            }
            if (g.last > first) f(g, unit, id);  // (in one place: the code of a kernel this short is fetched once)
            if (g.count < QT) break;
            g.clear();
        }
    }
}

// What a query's value weighs a channel's maximum (up) or minimum with; NaN stays NaN.
__device__ __forceinline__ double weight_of(float q, bool up) {
    return static_cast<double>(up ? __builtin_elementwise_maximum(q, 0.0f) : __builtin_elementwise_minimum(q, 0.0f));
}
// The weights of N channels (an even number) from `i` on (elements of q) over the query heads of the group, D apart; four heads'
// loads are issued together.
template <int N, int D>
__device__ __forceinline__ void group_weights(const SelectArgs& a, int64_t i, bool up, double (&w)[N]) {
#pragma unroll
    for (int e = 0; e < N; e++) w[e] = 0.0;
    for (int j0 = 0; j0 < a.group; j0 += 4) {
        float f[4][N];
        if (a.q_bf16) {
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const uint16_t* q = static_cast<const uint16_t*>(a.q) + i + min(j0 + k, a.group - 1) * D;
#pragma unroll
                for (int e = 0; e < N; e += 2) {
                    const uint32_t x = reinterpret_cast<const uint32_t*>(q)[e / 2];
                    f[k][e] = pa::bf16_lo(x);
                    f[k][e + 1] = pa::bf16_hi(x);
                }
            }
        } else {
#pragma unroll
            for (int k = 0; k < 4; k++)
#pragma unroll
                for (int e = 0; e < N; e++) f[k][e] = (static_cast<const float*>(a.q) + i + min(j0 + k, a.group - 1) * D)[e];
        }
#pragma unroll
        for (int k = 0; k < 4; k++)
#pragma unroll
            for (int e = 0; e < N; e++) w[e] += j0 + k < a.group ? weight_of(f[k][e], up) : 0.0;
    }
}

// ---- fp32 and bf16 bounds ----
// Load instructions issued together.
__host__ __device__ constexpr int score_batch(int queries) { return queries == 1 ? 8 : 4; }
// Waves per SIMD that the registers are held to.
__host__ __device__ constexpr int score_waves(int d, int kv, int queries) {
    return queries > 1 || (kv == PA_DTYPE_FP32 && d == 256) ? 2 : 4;
}

// One wave: KV head u % Hkv, blocks c * per .. of the context of unit u / Hkv / chunks (a query, or with QT > 1 a
// sequence, whose queries are scored QT at a time from one read of its bounds), c = u / Hkv % chunks.
// The bounds of a (block, KV head) are 2 D elements in a row; LB lanes take 16 bytes each of them
// (W times), 64 / LB blocks an instruction, UN instructions together and the next ones on their way
// meanwhile. The lanes' sums meet by transposing exchanges, which halve their number a step: 8 sums over 32
// lanes cost 12 additions instead of 40.
template <int D, int KV, int QT>
__global__ __launch_bounds__(64 * kScoreWaves, score_waves(D, KV, QT)) void block_score_kernel(const SelectArgs a, int32_t units,
                                                                                              int32_t chunks, int32_t per) {
    constexpr int ELT = KV == PA_DTYPE_FP32 ? 4 : 2;
    constexpr int E = 16 / ELT;
    constexpr int WORDS = 2 * D / E;              // 16-byte words per (block, KV head)
    constexpr int LB = WORDS < 64 ? WORDS : 64;   // lanes per block
    constexpr int W = WORDS / LB;                 // words per lane
    constexpr int NBI = 64 / LB;                  // blocks per load instruction
    constexpr int UN = score_batch(QT);
    // sums left after the exchanges over 32, 16 and 8 lanes
    constexpr int M32 = LB >= 64 ? UN / 2 : UN;
    constexpr int M16 = LB >= 32 && M32 > 1 ? M32 / 2 : M32;
    constexpr int KEPT = LB >= 16 && M16 > 1 ? M16 / 2 : M16;
    const int lane = threadIdx.x & 63, at = lane % LB;
    const uint32_t u = blockIdx.x * kScoreWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t rc = u / static_cast<uint32_t>(a.hkv);
    const int h = static_cast<int>(u - rc * a.hkv);
    const uint32_t unit = rc / static_cast<uint32_t>(chunks);
    const int first = static_cast<int>(rc - unit * chunks) * per;
    if (unit >= static_cast<uint32_t>(units)) return;
    // The block a lane's kept sum k belongs to within a batch: instruction `mine` + k, block lane / LB of it.
    const int mine = (M32 < UN && lane & 32 ? M32 : 0) + (M16 < M32 && lane & 16 ? M16 : 0) + (KEPT < M16 && lane & 8 ? KEPT : 0);
    // no sum is written twice: lanes that hold copies are left out
    const bool writes = !(LB >= 32 && M16 == M32 && lane & 16) && !(LB >= 16 && KEPT == M16 && lane & 8);
    const char* base = static_cast<const char*>(a.bounds);

    for_query_groups<QT>(a, static_cast<int>(unit), first, per, first + lane, [&](const QueryGroup<QT>& g, int seq, int id) {
        const int n = g.last - first;
        double wt[QT][W][E];
#pragma unroll
        for (int t = 0; t < QT; t++)
#pragma unroll
            for (int w = 0; w < W; w++) {
                const int i0 = (w * LB + at) * E;
                const bool up = i0 >= D;
                group_weights<E, D>(a, (static_cast<int64_t>(g.r[t]) * a.hkv + h) * a.group * D + (up ? i0 - D : i0), up, wt[t][w]);
            }
        // Blocks out of the pool, and those past the chunk, load block 0 and their score is dropped: loads without a
        // branch let the compiler wait for the oldest batch alone (with one it waited for all in flight).
        if (lane >= n || id >= a.num_blocks) id = -1;
        uint4 v[2][UN][W];
        auto load = [&](int i0, uint4 (&x)[UN][W]) {
            const uint4* at_block[UN];
#pragma unroll
            for (int k = 0; k < UN; k++) {
                const int b = max(0, __shfl(id, min((i0 + k) * NBI + lane / LB, 63), 64));
                at_block[k] = reinterpret_cast<const uint4*>(base + (static_cast<int64_t>(b) * a.hkv + h) * 2 * D * ELT) + at;
            }
#pragma unroll
            for (int k = 0; k < UN; k++)
#pragma unroll
                for (int w = 0; w < W; w++) x[k][w] = load_once(at_block[k] + w * LB);
        };
        load(0, v[0]);
        load(UN, v[1]);
#pragma unroll 1
        for (int i0 = 0; i0 * NBI < n; i0 += 2 * UN) {
#pragma unroll
            for (int half = 0; half < 2; half++) {
                const int i = i0 + half * UN;  // (past the chunk in the last round: nothing is kept of it)
#pragma unroll
                for (int t = 0; t < QT; t++) {
                    if (t >= g.count) break;
                    double s[UN];
#pragma unroll
                    for (int k = 0; k < UN; k++) {
                        s[k] = 0.0;
#pragma unroll
                        for (int w = 0; w < W; w++)
#pragma unroll
                            for (int e = 0; e < E; e++)
                                s[k] = __builtin_fma(static_cast<double>(elem<KV>(v[half][k][w], e)), wt[t][w][e], s[k]);
                    }
                    // exchanges over 32, 16 and 8 lanes, where the block spans them
                    if constexpr (LB >= 64) {
#pragma unroll
                        for (int k = 0; k < M32; k++) s[k] = pair32(s[k], s[k + M32]);
                    }
                    if constexpr (LB >= 32) {
#pragma unroll
                        for (int k = 0; k < M16; k++) s[k] = M16 < M32 ? pair16(s[k], s[(k + M16) % UN]) : sum_across<16>(s[k]);
                    }
                    if constexpr (LB >= 16) {
#pragma unroll
                        for (int k = 0; k < KEPT; k++) s[k] = KEPT < M16 ? pair8(s[k], s[(k + KEPT) % UN]) : sum_across<8>(s[k]);
                    }
                    double keep = 0.0;
#pragma unroll
                    for (int k = 0; k < KEPT; k++) {
                        s[k] = sum8(s[k]);
                        keep = (lane & 7) == k ? s[k] : keep;
                    }
                    const int j = (i + mine + (lane & 7)) * NBI + lane / LB;
                    const int b = first + j;
                    if (__shfl(id, j & 63, 64) < 0) keep = 0.0;
                    if ((lane & 7) < KEPT && writes && b < g.end[t])
                        a.scores[(static_cast<int64_t>(g.r[t]) * a.hkv + h) * a.max_blocks + b] = keep;
                }
                load(i + 2 * UN, v[half]);
            }
        }
    });
}

// ---- int8 bounds ----
// The codes go to the int8 matrix instruction as they are, 16 blocks a tile, against the weights as 47-bit
// integers in units of 2^(e - 45), 2^e <= the largest weight < 2^(e + 1), in six signed base-256 digits: one
// column a digit, eight columns a query, two queries a tile. The instruction sums the products over all 2 D
// channels in 32 bits exactly; a block's score is its six column sums by their places, times the unit and
// k_scale. The sums go through LDS to a lane per (query, block). Over 108 MB of bounds, three queries a sequence:
// 114 us with byte dot products in the vector unit, 44 with the columns summed across lanes in fp64, 32 with
// the sums through LDS, 29 with the codes through LDS as well: whole rows a load instead of half lines, which also lets
// the loads be non-temporal (67 us without that); 30 with the digit sums joined in 64 bits.
constexpr int kDigits = 6;
constexpr int kInt8Waves = 4;
constexpr int kInt8Ahead = 2;  // tiles on their way (4: 32.3 us)
constexpr int kInt8Blocks = 128;  // blocks per wave (29.2 us; 64: 31.6; 256 56.8 a selection where 128 took 48.0)

// The digits of a (query, KV head), made once: one wave each. (Made by every wave of the scores, they took 27 of
// its 46 us.)
template <int D>
__global__ __launch_bounds__(64) void int8_weights_kernel(const SelectArgs a) {
    constexpr int N = 2 * D / 64;  // weights per lane
    const int64_t u = blockIdx.x;
    const int lane = threadIdx.x, i0 = N * lane;
    const bool up = i0 >= D;
    double x[N];
    group_weights<N, D>(a, u * a.group * D + (up ? i0 - D : i0), up, x);
    // The largest weight's exponent, in 64 bits: a finite query's sums over its heads may pass fp32's largest value.
    constexpr float kNone = -4096.0f, kBad = 4096.0f;  // no weight but zeros; one that is not finite
    double top = 0.0;
    bool finite = true;
#pragma unroll
    for (int e = 0; e < N; e++) {
        finite &= fabs(x[e]) < static_cast<double>(INFINITY);
        top = fmax(top, fabs(x[e]));
    }
    const float most = pa::wave_max_dpp(!finite ? kBad : top > 0.0 ? static_cast<float>(__builtin_amdgcn_frexp_exp(top) - 1) : kNone);
    const bool bad = most == kBad;
    const int ex = bad || most == kNone ? 0 : static_cast<int>(most);
    if (lane == 0) a.units[u] = bad ? static_cast<double>(__builtin_nanf("")) : __builtin_amdgcn_ldexp(1.0, ex - 45);
    // |z| <= 2^46; with 128 added in every place the digits are plain bytes, 128 too large each
    uint64_t y[N];
#pragma unroll
    for (int e = 0; e < N; e++) {
        const int64_t z = bad ? 0 : static_cast<int64_t>(__builtin_rint(__builtin_amdgcn_ldexp(x[e], 45 - ex)));
        y[e] = static_cast<uint64_t>(z + 0x808080808080ll) ^ 0x808080808080ull;
    }
#pragma unroll
    for (int j = 0; j < kDigits; j++) {
        uint8_t* to = reinterpret_cast<uint8_t*>(a.digits) + (u * kDigits + j) * 2 * D + i0;
        if constexpr (N == 2) {
            *reinterpret_cast<uint16_t*>(to) = static_cast<uint16_t>((y[0] >> (8 * j) & 255) | (y[1] >> (8 * j) & 255) << 8);
        } else {
#pragma unroll
            for (int e = 0; e < N; e += 4)
                *reinterpret_cast<uint32_t*>(to + e) = static_cast<uint32_t>(
                    (y[e] >> (8 * j) & 255) | (y[e + 1] >> (8 * j) & 255) << 8 | (y[e + 2] >> (8 * j) & 255) << 16 |
                    (y[e + 3] >> (8 * j) & 255) << 24);
        }
    }
}

// One wave: KV head u % Hkv, blocks c * per .. of the context of unit u / Hkv / chunks, c = u / Hkv % chunks, 64 ids at a
// time, two tiles on their way while a third is scored. (The waves of a workgroup take neighbouring heads of the
// same blocks, whose bounds lie side by side.)
template <int D, int QT>
__global__ __launch_bounds__(64 * kInt8Waves, D == 256 ? 2 : QT > 1 ? 3 : 4) void block_score_int8_kernel(const SelectArgs a, int32_t units,
                                                                                            int32_t chunks, int32_t per) {
    constexpr int SL = 2 * D / 64;            // matrix slabs of 64 channels
    constexpr int SETS = (QT + 1) / 2;
    constexpr int TILES = kScoreBlocks / 16;
    constexpr int PPR = 2 * D / 16, RPI = 64 / PPR;  // 16-byte pieces of a block's bounds; blocks per load
    __shared__ uint4 s_tile[kInt8Waves][16][PPR];    // of each wave: a tile, piece p of block b at p ^ b (no bank twice)
    __shared__ i32x4 s_sum[kInt8Waves][SETS * 16][4];  // of each wave: [column][block] sums of a tile
    const int lane = threadIdx.x & 63, q4 = lane >> 4, n = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t u = blockIdx.x * kInt8Waves + wave;
    const uint32_t rc = u / static_cast<uint32_t>(a.hkv), unit = rc / static_cast<uint32_t>(chunks);
    const int h = static_cast<int>(u - rc * a.hkv);
    const int start = static_cast<int>(rc - unit * chunks) * per;
    if (unit >= static_cast<uint32_t>(units)) return;
    const char* base = static_cast<const char*>(a.bounds);
    for_query_groups<QT>(a, static_cast<int>(unit), start, per, start + lane, [&](const QueryGroup<QT>& g, int seq, int id) {
        int first = start;
        if (first + lane >= g.last || id >= a.num_blocks) id = -1;
        // column n: digit n % 8 of query n / 8 of the pair
        i32x4 wt[SETS][SL];
#pragma unroll
        for (int p = 0; p < SETS; p++) {
            const int j = n & 7;
            const bool used = 2 * p + (n >> 3) < g.count && j < kDigits;
            const int r = QT > 1 && n >= 8 ? g.r[(2 * p + 1) % QT] : g.r[2 * p];  // of a query that is not there: query 0
            const int64_t of = static_cast<int64_t>(r) * a.hkv + h;
            const uint4* digit = a.digits + (of * kDigits + min(j, kDigits - 1)) * (2 * D / 16) + q4;
#pragma unroll
            for (int s = 0; s < SL; s++) {
                const i32x4 x = __builtin_bit_cast(i32x4, digit[4 * s]);
                wt[p][s] = used ? x : i32x4{0, 0, 0, 0};
            }
        }
        // this lane's part of a tile's outcome: query q4 of the group, block n
        int r_of = 0, end_of = 0;
#pragma unroll
        for (int t = 0; t < QT; t++)
            if (t == q4) {
                r_of = g.r[t];
                end_of = g.end[t];
            }
        const int64_t row_of = static_cast<int64_t>(r_of) * a.hkv + h;
        const double unit_of = a.units[row_of];
        double* out = a.scores + row_of * a.max_blocks;
        uint4 v[kInt8Ahead][SL];
        float ks[kInt8Ahead];
        auto load = [&](int gi, uint4 (&x)[SL], float& sc) {  // tile gi: blocks side by side, a row of lanes each
            // (a block out of the pool or past the chunk: block 0, times a scale of zero)
#pragma unroll
            for (int i = 0; i < SL; i++) {
                const int b = max(0, __shfl(id, (16 * gi + RPI * i + lane / PPR) & 63, 64));
                x[i] = load_once(reinterpret_cast<const uint4*>(base + (static_cast<int64_t>(b) * a.hkv + h) * 2 * D) + lane % PPR);
            }
            const int o = __shfl(id, (16 * gi + n) & 63, 64);
            const float k = a.k_scale[static_cast<int64_t>(max(0, o)) * a.hkv + h];
            sc = o >= 0 ? k : 0.0f;
        };
#pragma unroll
        for (int k = 0; k < kInt8Ahead; k++) load(k, v[k], ks[k]);
        while (first < g.last) {
            // the ids of the next 64 blocks
            const int after = first + kScoreBlocks;
            int next = -1;
            if (after + lane < g.last) next = a.tables[static_cast<int64_t>(seq) * a.width + after + lane];
#pragma unroll 1
            for (int g0 = 0; g0 < TILES; g0 += kInt8Ahead) {
#pragma unroll
                for (int k = 0; k < kInt8Ahead; k++) {
                    const int gi = g0 + k;
#pragma unroll
                    for (int i = 0; i < SL; i++) {
                        const int row = RPI * i + lane / PPR;
                        s_tile[wave][row][(lane % PPR) ^ (row % PPR)] = v[k][i];
                    }
                    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                    __builtin_amdgcn_wave_barrier();
                    i32x4 x[SL];  // the matrix operand: lane (q4, n) codes 64 s + 16 q4 .. of block n
#pragma unroll
                    for (int s = 0; s < SL; s++) x[s] = __builtin_bit_cast(i32x4, s_tile[wave][n][(4 * s + q4) ^ (n % PPR)]);
#pragma unroll
                    for (int p = 0; p < SETS; p++) {
                        i32x4 acc = {0, 0, 0, 0};
#pragma unroll
                        for (int s = 0; s < SL; s++)
                            acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(x[s], wt[p][s], acc, 0, 0, 0);
                        s_sum[wave][16 * p + n][q4] = acc;  // blocks 4 q4 .. + 3 of column n
                    }
                    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                    __builtin_amdgcn_wave_barrier();
                    // A column sum is at most 2^23 (512 places, codes and digits down to -128) and a pair of digits 2^31 + 2^23,
                    // more than 32 bits hold: joined in 64, exactly.
                    const int32_t* sums = reinterpret_cast<const int32_t*>(s_sum[wave][8 * (q4 < QT ? q4 : 0)]) + n;
                    double y = 0.0;
#pragma unroll
                    for (int j = kDigits - 2; j >= 0; j -= 2)
                        y = __builtin_fma(y, 65536.0, __builtin_fma(static_cast<double>(sums[16 * (j + 1)]), 256.0, static_cast<double>(sums[16 * j])));
                    const int b = first + 16 * gi + n;
                    if (q4 < QT && b < end_of) out[b] = y * unit_of * static_cast<double>(ks[k]);
                    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                    __builtin_amdgcn_wave_barrier();
                    if (gi == TILES - kInt8Ahead) id = next < a.num_blocks ? next : -1;  // the next ones' tiles follow
                    load((gi + kInt8Ahead) % TILES, v[k], ks[k]);
                }
            }
            first = after;
        }
    });
}

// Scores as 64-bit keys in the same order: NaN above everything (such a block is kept, and the
// attention over it shows the NaN), the two zeros equal. No key is 0.
__device__ __forceinline__ uint64_t key_of(double s) {
    if (s != s) return ~0ull;
    const uint64_t b = __builtin_bit_cast(uint64_t, s + 0.0);
    return b >> 63 ? ~b : b | 1ull << 63;
}

// Exclusive prefix of the set bits of `words` 64-bit words, into pre; by the first wave.
__device__ __forceinline__ void word_prefix(const uint64_t* mask, int* pre, int words) {
    if (threadIdx.x >= 64) return;
    const int lane = threadIdx.x;
    int run = 0;
    for (int w0 = 0; w0 < words; w0 += 64) {
        const int n = w0 + lane < words ? __popcll(mask[w0 + lane]) : 0;
        const int incl = pa::wave_prefix(n);
        if (w0 + lane < words) pre[w0 + lane] = run + incl - n;
        run += __builtin_amdgcn_readlane(incl, 63);
    }
}

constexpr int kBins = 1024;
constexpr int kBorder = 512;  // scores of the border bin that are ranked one against another
constexpr int kHeld = 12288;  // candidates of a row that fit LDS beside the rest

// One workgroup per (query token, KV head): of the m candidates (the blocks between the sink and the
// recent ones) the `need` best. A histogram over the scores' range (in fp32, whose roundings keep the
// order: not strictly, but a bin never holds a score above one of a higher bin) finds the bin in which the
// border lies; the few scores in it are ranked one against another by their 64 bits and their index. Where
// the range is not finite or the bin too full (equal scores), K, the need-th largest key, is built bit by bit
// instead, and the first of the keys equal to K fill up. HELD: the scores are kept in LDS in fp32 for the bins (the
// 64 bits of the few that need them are read again); else they are read again for every pass.
// Lanes hold consecutive candidates, so a ballot is a 64-bit mask of them, and the places of the
// kept ones in the ascending list are prefix counts of the masks' bits.
template <int T, bool HELD>
__global__ __launch_bounds__(T) void block_choose_kernel(const SelectArgs a) {
    static_assert(kBorder <= T, "a thread per score of the border bin");
    extern __shared__ uint64_t s_mask[];  // [words] masks, [words] int prefixes, HELD: [m] scores in fp32
    __shared__ int s_cnt[T / 64];
    __shared__ float s_lo[T / 64], s_hi[T / 64];
    __shared__ int s_hist[kBins];
    __shared__ uint64_t s_key[kBorder];
    __shared__ int s_idx[kBorder];
    __shared__ int s_bin, s_above, s_len;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int row = blockIdx.x;
    const int nblk = context_blocks(a, row / a.hkv);
    int32_t* out = a.selected + static_cast<int64_t>(row) * a.budget;
    if (nblk <= a.budget) {
        for (int i = tid; i < a.budget; i += T) out[i] = i < nblk ? i : -1;
        return;
    }
    const int s0 = a.sink, r0 = nblk - a.recent;
    const int m = r0 - s0, need = a.budget - a.sink - a.recent;  // 0 <= need < m
    const double* scores = a.scores + static_cast<int64_t>(row) * a.max_blocks + s0;
    const int words = (m + 63) / 64, padded = words * 64;
    int* pre = reinterpret_cast<int*>(s_mask + words);
    float* s_score = reinterpret_cast<float*>(pre + words);
    auto rounded = [&](double x) { return x != x ? INFINITY : static_cast<float>(x); };
    auto score = [&](int i) { return HELD ? s_score[i] : rounded(scores[i]); };
    // sum of `mine` over the workgroup
    auto count = [&](int mine) {
        for (int o = 1; o < 64; o <<= 1) mine += __shfl_xor(mine, o, 64);
        __syncthreads();
        if (lane == 0) s_cnt[wave] = mine;
        __syncthreads();
        int sum = 0;
        for (int w = 0; w < T / 64; w++) sum += s_cnt[w];
        return sum;
    };

    float lo = INFINITY, hi = -INFINITY;
#pragma unroll 8
    for (int i = tid; i < m; i += T) {
        const float f = rounded(scores[i]);
        if constexpr (HELD) s_score[i] = f;
        lo = fminf(lo, f);
        hi = fmaxf(hi, f);
    }
    lo = -pa::wave_max_dpp(-lo);
    hi = pa::wave_max_dpp(hi);
    if (lane == 0) {
        s_lo[wave] = lo;
        s_hi[wave] = hi;
    }
    for (int b = tid; b < kBins; b += T) s_hist[b] = 0;
    if (tid == 0) s_len = 0;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < T / 64; w++) {
        lo = fminf(lo, s_lo[w]);
        hi = fmaxf(hi, s_hi[w]);
    }
    const float per = static_cast<float>(kBins) / (hi - lo);
    bool whole = need == 0 || !(per > 0.0f && per < INFINITY && hi < INFINITY && lo > -INFINITY);
    auto bin_of = [&](float f) { return min(kBins - 1, static_cast<int>((f - lo) * per)); };
    if (!whole) {
#pragma unroll 4
        for (int i = tid; i < m; i += T) atomicAdd(&s_hist[bin_of(score(i))], 1);
        __syncthreads();
        // bins from the top: thread t takes PB of them; the one the border lies in is unique
        constexpr int PB = kBins / T > 0 ? kBins / T : 1;
        int n[PB], sum = 0;
#pragma unroll
        for (int k = 0; k < PB; k++) {
            const int b = kBins - 1 - (tid * PB + k);
            n[k] = b >= 0 ? s_hist[b] : 0;
            sum += n[k];
        }
        const int incl = pa::wave_prefix(sum);
        if (lane == 63) s_cnt[wave] = incl;
        __syncthreads();
        int above = incl - sum;
#pragma unroll
        for (int w = 0; w < T / 64; w++) {
            const int c = s_cnt[w];
            above += w < wave ? c : 0;
        }
#pragma unroll
        for (int k = 0; k < PB; k++) {
            if (above < need && need <= above + n[k]) {
                s_bin = kBins - 1 - (tid * PB + k);
                s_above = above;
            }
            above += n[k];
        }
        __syncthreads();
        const int border = s_bin;
        for (int i = tid; i < padded; i += T) {
            const int b = i < m ? bin_of(score(i)) : -1;
            const uint64_t kept = __ballot(b > border);
            if (lane == 0) s_mask[i >> 6] = kept;
            if (b == border) {
                const int p = atomicAdd(&s_len, 1);
                if (p < kBorder) s_idx[p] = i;
            }
        }
        __syncthreads();
        const int len = s_len;
        whole = len > kBorder;
        if (!whole) {  // (kBorder <= T: a thread per score of the border bin)
            const int more = need - s_above;
            const uint64_t k = tid < len ? key_of(scores[s_idx[tid]]) : 0;
            if (tid < len) s_key[tid] = k;
            __syncthreads();
            if (tid < len) {
                const int i = s_idx[tid];
                int rank = 0;
#pragma unroll 4
                for (int l = 0; l < len; l++) rank += s_key[l] > k || (s_key[l] == k && s_idx[l] < i);
                if (rank < more) atomicOr(reinterpret_cast<unsigned long long*>(&s_mask[i >> 6]), 1ull << (i & 63));
            }
        }
    }
    if (whole) {
        uint64_t K = 0;
        if (need > 0) {
#pragma unroll 1
            for (int bit = 63; bit >= 0; bit--) {
                const uint64_t trial = K | 1ull << bit;
                int mine = 0;
#pragma unroll 1
                for (int i = tid; i < m; i += T) mine += key_of(scores[i]) >= trial;
                if (count(mine) >= need) K = trial;
            }
        }
        int above = 0;
#pragma unroll 1
        for (int i = tid; i < m; i += T) above += key_of(scores[i]) > K;
        above = count(above);
#pragma unroll 1
        for (int i = tid; i < padded; i += T) {
            const uint64_t eq = __ballot(i < m && key_of(scores[min(i, m - 1)]) == K);
            if (lane == 0) s_mask[i >> 6] = eq;
        }
        __syncthreads();
        word_prefix(s_mask, pre, words);
        __syncthreads();
#pragma unroll 1
        for (int i = tid; i < padded; i += T) {
            bool keep = false;
            if (i < m && need > 0) {
                const uint64_t k = key_of(scores[i]);
                const int rank = pre[i >> 6] + __popcll(s_mask[i >> 6] & ((1ull << lane) - 1));
                keep = k > K || (k == K && above + rank < need);
            }
            const uint64_t kept = __ballot(keep);
            if (lane == 0) s_mask[i >> 6] = kept;  // this wave alone reads and writes its words
        }
    }
    __syncthreads();
    word_prefix(s_mask, pre, words);
    __syncthreads();
#pragma unroll 4
    for (int i = tid; i < m; i += T) {
        const uint64_t kept = s_mask[i >> 6];
        if (kept >> lane & 1) out[s0 + pre[i >> 6] + __popcll(kept & ((1ull << lane) - 1))] = s0 + i;
    }
    for (int i = tid; i < a.sink + a.recent; i += T)
        out[i < a.sink ? i : a.budget - a.recent + (i - a.sink)] = i < a.sink ? i : r0 + (i - a.sink);
}

// Launches the scores; nothing, and false, for more workgroups than a grid holds.
template <int D>
bool launch_score(const SelectArgs& a, int kv, int32_t most, hipStream_t s) {
    // Units are sequences where they have several queries each on average, else queries.
    const bool grouped = a.query_seqs && a.num_queries > a.num_seqs;
    const int32_t units = grouped ? a.num_seqs : a.num_queries;
    if (units == 0) return true;  // queries of no sequence: nothing is scored
    if (kv == PA_DTYPE_INT8) {
        if constexpr (D >= 64) {
            const int32_t per = kInt8Blocks;
            const int32_t chunks = (most + per - 1) / per;
            const int64_t waves = static_cast<int64_t>(units) * chunks * a.hkv;
            const int64_t grid = (waves + kInt8Waves - 1) / kInt8Waves;
            if (!pa::fits_grid(grid, 64 * kInt8Waves)) return false;
            const auto go = [&](auto kernel) { kernel<<<static_cast<uint32_t>(grid), 64 * kInt8Waves, 0, s>>>(a, units, chunks, per); };
            int8_weights_kernel<D><<<a.num_queries * a.hkv, 64, 0, s>>>(a);
            if (grouped) go(block_score_int8_kernel<D, kQueryTile>);
            else go(block_score_int8_kernel<D, 1>);
        }
        return true;
    }
    // Blocks per wave: 32 (64 time the same where the chip is full, 16 leave too little to stream: 49 us a selection of
    // 32 long contexts where 32 took 42), a batch at least, halved while the waves are too few for the chip.
    const int32_t lanes = std::min(64, 2 * D * (kv == PA_DTYPE_FP32 ? 4 : 2) / 16);
    const int32_t batch = 64 / lanes * score_batch(grouped ? kQueryTile : 1);
    int32_t per = std::max(batch, 32);
    while (per > batch && static_cast<int64_t>(units) * a.hkv * ((most + per - 1) / per) < kScoreWorkers) per /= 2;
    const int32_t chunks = (most + per - 1) / per;
    const int64_t waves = static_cast<int64_t>(units) * chunks * a.hkv;
    const int64_t grid = (waves + kScoreWaves - 1) / kScoreWaves;
    if (!pa::fits_grid(grid, 64 * kScoreWaves)) return false;
    const auto go = [&](auto kernel) { kernel<<<static_cast<uint32_t>(grid), 64 * kScoreWaves, 0, s>>>(a, units, chunks, per); };
    if (kv == PA_DTYPE_FP32) {
        if (grouped) go(block_score_kernel<D, PA_DTYPE_FP32, kQueryTile>);
        else go(block_score_kernel<D, PA_DTYPE_FP32, 1>);
    } else {
        if (grouped) go(block_score_kernel<D, PA_DTYPE_BF16, kQueryTile>);
        else go(block_score_kernel<D, PA_DTYPE_BF16, 1>);
    }
    return true;
}

template <int T, bool HELD>
void launch_choose(const SelectArgs& a, int32_t most, hipStream_t s) {
    const size_t words = (static_cast<size_t>(most) + 63) / 64;
    block_choose_kernel<T, HELD><<<a.num_queries * a.hkv, T, words * (12 + (HELD ? 256 : 0)) + 8, s>>>(a);
}

pa_status check_sizes(const char* f, const pa_config* cfg, int32_t num_queries, int32_t max_context_len) {
    if (num_queries < 0 || max_context_len < 0)
        return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": negative size");
    if (max_context_len > kMaxBlocks * pa::kBlockSize)
        return pa::set_error(PA_ERROR_UNSUPPORTED, std::string(f) + ": max_context_len must be <= " +
                                                       std::to_string(kMaxBlocks * pa::kBlockSize));
    if (static_cast<int64_t>(num_queries) * cfg->num_kv_heads > 1 << 24)
        return pa::set_error(PA_ERROR_UNSUPPORTED, std::string(f) + ": too many query tokens for one call");
    return PA_SUCCESS;
}

// Workspace: int8 digits and units, then the scores.
size_t digit_bytes(const pa_config* cfg, int32_t num_queries) {
    return cfg->kv_dtype == PA_DTYPE_INT8 ? static_cast<size_t>(num_queries) * cfg->num_kv_heads * kDigits * 2 * cfg->head_dim : 0;
}
size_t unit_bytes(const pa_config* cfg, int32_t num_queries) {
    return cfg->kv_dtype == PA_DTYPE_INT8 ? static_cast<size_t>(num_queries) * cfg->num_kv_heads * 8 : 0;
}
size_t workspace_of(const pa_config* cfg, int32_t num_queries, int32_t max_context_len) {
    return digit_bytes(cfg, num_queries) + unit_bytes(cfg, num_queries) +
           static_cast<size_t>(num_queries) * cfg->num_kv_heads * ((static_cast<size_t>(max_context_len) + 15) / 16) * 8;
}

}  // namespace

extern "C" {

pa_status pa_select_workspace_size(const pa_config* cfg, int32_t num_queries, int32_t max_context_len, size_t* bytes) {
    const char* const f = "pa_select_workspace_size";
    pa_status st = pa::check_config(cfg, f);
    if (st != PA_SUCCESS) return st;
    if (!bytes) return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": bytes is null");
    st = check_sizes(f, cfg, num_queries, max_context_len);
    if (st != PA_SUCCESS) return st;
    *bytes = workspace_of(cfg, num_queries, max_context_len);
    return pa::clear_error();
}

pa_status pa_select_blocks(pa_stream* stream, const pa_config* cfg, const void* q, const void* key_bounds,
                           const float* k_scale, const int32_t* block_tables, int32_t num_seqs,
                           int32_t max_blocks_per_seq, const int32_t* query_seqs, const int32_t* context_lens,
                           int32_t num_queries, int32_t max_context_len, int32_t sink_blocks, int32_t recent_blocks,
                           int32_t budget, int32_t* selected, void* workspace, size_t workspace_bytes) {
    const char* const f = "pa_select_blocks";
    pa_status st = pa::check_config(cfg, f);
    if (st != PA_SUCCESS) return st;
    if (num_seqs < 0 || max_blocks_per_seq < 0) return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": negative size");
    st = check_sizes(f, cfg, num_queries, max_context_len);
    if (st != PA_SUCCESS) return st;
    if (sink_blocks < 0 || recent_blocks < 1)
        return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": sink_blocks must be >= 0 and recent_blocks >= 1");
    if (budget < 1 || static_cast<int64_t>(sink_blocks) + recent_blocks > budget)
        return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": budget must hold the sink and recent blocks");
    if (static_cast<int64_t>(num_queries) * cfg->num_kv_heads * budget > INT32_MAX)
        return pa::set_error(PA_ERROR_UNSUPPORTED, std::string(f) + ": too many query tokens for one call");
    if (num_queries == 0) return pa::clear_error();
    if (cfg->num_blocks == 0) return pa::set_error(PA_ERROR_INVALID_CONFIG, std::string(f) + ": num_blocks must be > 0");
    if (!q || !key_bounds || !block_tables || !context_lens || !selected)
        return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": null pointer");
    if (!query_seqs && num_queries != num_seqs)
        return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": num_queries must be num_seqs when query_seqs is null");
    if (cfg->kv_dtype == PA_DTYPE_INT8 && !k_scale)
        return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": int8 cache needs k_scale");
    if (!pa::aligned16(key_bounds) || !pa::aligned16(q))
        return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": q and key_bounds must be 16-byte aligned");
    const size_t need = workspace_of(cfg, num_queries, max_context_len);
    if (need > workspace_bytes || (need > 0 && !workspace))
        return pa::set_error(PA_ERROR_WORKSPACE_TOO_SMALL, std::string(f) + ": workspace needs " + std::to_string(need) + " bytes");
    if (!pa::aligned16(workspace))
        return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": workspace must be 16-byte aligned");
    SelectArgs a{};
    a.q = q;
    a.bounds = key_bounds;
    a.k_scale = k_scale;
    a.tables = block_tables;
    a.query_seqs = query_seqs;
    a.context_lens = context_lens;
    a.digits = static_cast<uint4*>(workspace);
    a.units = reinterpret_cast<double*>(static_cast<char*>(workspace) + digit_bytes(cfg, num_queries));
    a.scores = a.units + unit_bytes(cfg, num_queries) / 8;
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
    // Threads a row of the choice: 512 of 1024 blocks 5.1 us, 256 5.7; 1024 of 2048 blocks 7.0 us, 512 8.0.
    const int32_t threads = most <= 1024 ? 512 : 1024;
    if (!pa::fits_grid(static_cast<int64_t>(num_queries) * a.hkv, threads))
        return pa::set_error(PA_ERROR_UNSUPPORTED, std::string(f) + ": too many query tokens for one call");
    if (most > budget) {
        bool fits = true;
        switch (cfg->head_dim) {
            case 32: fits = launch_score<32>(a, cfg->kv_dtype, most, s); break;
            case 64: fits = launch_score<64>(a, cfg->kv_dtype, most, s); break;
            case 128: fits = launch_score<128>(a, cfg->kv_dtype, most, s); break;
            default: fits = launch_score<256>(a, cfg->kv_dtype, most, s); break;
        }
        if (!fits) return pa::set_error(PA_ERROR_UNSUPPORTED, std::string(f) + ": too many blocks for one call");
        PA_HIP_CHECK(hipGetLastError());
    }
    if (threads == 512) launch_choose<512, true>(a, most, s);
    else if (most <= kHeld) launch_choose<1024, true>(a, most, s);
    else launch_choose<1024, false>(a, most, s);
    PA_HIP_CHECK(hipGetLastError());
    return pa::clear_error();
}

}  // extern "C"
