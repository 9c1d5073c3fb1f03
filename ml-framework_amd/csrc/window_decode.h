// window_decode.h -- attention of single query tokens over a sliding window and a few first tokens that stay visible.
//
// For sequence r of T cached tokens, KV head h and query head g of its group, over the tokens t with t < sink or
// T - window <= t < T (window 0: all of them):
//   s_t = scale * q_g . k_t,  out_g = sum_t exp(s_t - max s) v_t / sum_t exp(s_t - max s)
// and, where masses are kept, mass[r][t / 16] += sum_h sum_g exp(s_t - max s) / sum_t' exp(s_t' - max s). T is cut at the table's width and
// max_context_len first: the query stands at the end of what is read.
//
// A row is a (sequence, KV head); its list is the blocks that hold a visible token: those of the sinks, then those of
// the window. The lists are laid end to end and cut into equal ranges, one for each workgroup of a chip full of them, as
// in sparse_decode.h, whose arithmetic this kernel shares: exact products (an fp32 value as three bf16 parts in
// the matrix columns that a group of G heads leaves idle), sums in fp32, two register buffers a wave, the waves' states
// met in LDS at a segment's end. Here the lists follow from the lengths, so nothing but the table is read for them, and the
// ranges go by what the rows really hold: every workgroup adds up the lengths itself (at most kWindowSeqs a launch). Where the chip
// is not full, every row is filled up to whole ranges in what is laid end to end.
// What bounds it: memory where rows are many (64 sequences, window 1024 and 4 sinks, (32, 8, 128) bf16: 50 us, the decode itself 43 at 4.5 TB/s; 48
// over 4096 tokens, int8: 91 us, 4.5 TB/s in runs of 2 KiB; 32 of 2-8k tokens with masses: 113 us, of which the decode 92 at 6.3 TB/s and what
// follows 9), else round trips: 7 us and the launch behind (one sequence 10.8 us). Eight waves a workgroup with whole-list ranges, values from
// LDS that the compiler did not see to be uniform, and a launch each for cut rows and masses took 10 to 15 % more.
#pragma once

#include "sparse_decode.h"

namespace pa {

constexpr int kWindowSeqs = 2047;  // sequences of one launch: their lists' starts stand in LDS

struct WindowArgs {
    DecodeArgs d;          // caches, q, out, tables, lengths, shape; ws_o / ws_m / ws_l: [2 * workgroups][G]
    int32_t* starts;       // [num_seqs + 1] entries (of one KV head) before each sequence, then the range
    float2* parts;         // masses: (maximum, sum) of every list entry's tokens, [Hkv * starts + ..][G]; else null
    float2* total;         // masses: (maximum, sum) of every row that was not cut, [num_seqs][Hq]
    float* mass;           // [num_seqs][max_blocks_per_seq]
    int32_t num_seqs, sink, window;
    int32_t groups;        // workgroups
    int32_t merge_groups;  // of the launch behind: workgroups that join cut rows, and (masses) per sequence
    int32_t mass_chunks;
};

// The list of a context of T tokens: blocks [0, first), then [low, end).
struct WindowList {
    int first, low, end;
    __device__ __forceinline__ int entries() const { return first + end - low; }
    __device__ __forceinline__ int block(int e) const { return e < first ? e : e - first + low; }
};
__device__ __forceinline__ int window_begin(int T, int window) { return window > 0 ? max(0, T - window) : 0; }
__device__ __forceinline__ WindowList window_list(int T, int sink, int window) {
    const int low = window_begin(T, window) / 16;
    return {min((min(sink, T) + 15) / 16, low), low, (T + 15) / 16};
}

// Waves of a workgroup, list entries of a range at least, workgroups of a full chip.
__host__ __device__ constexpr int window_waves(int) { return 4; }
constexpr int kWindowLeast = 8;  // (one sequence, 8 KV heads, (32, 8, 128) bf16: 4 / 8 / 16 entries 11.4 / 11.3 / 12.1 us at 1040 tokens, 17.2 / 14.0 / 13.2 at 4096)
__host__ __device__ constexpr int window_decode_groups(int head_dim, int kv) {
    return sparse_groups(head_dim, kv) * sparse_waves(head_dim) / window_waves(head_dim);
}

// How the lists are dealt out: sequence r's entries (of one KV head) from s_starts[r], its length in s_lens[r]; what a workgroup
// takes. One workgroup, W waves. The rule, for lists of `all` entries in all:
//   whole rows where all are of one length and that gives no CU more than 24 entries, or a third, over an equal share: a cut row costs
//   another start, another exchange of states and the merge ((32, 8, 128) bf16, whole / cut: one sequence of 16 blocks 9.6 / 10.2 us, of 32
//   12.1 / 10.4, of 40 13.7 / 10.8; 16 of 32 blocks 13.9 / 14.8; 60 of 64 blocks 45.1 / 49.7; 40 of 64, a CU's share 128 for 80, 39.1 / 36.8);
//   the least range where there are workgroups for every row's last range to be a part of one (the chip is not full): no workgroup
//   starts twice (one sequence of 1028 tokens, 8 KV heads: 11.7 us, with ranges across rows 13.5);
//   equal ranges.
template <int W>
__device__ __forceinline__ uint32_t window_starts(const WindowArgs& a, int32_t* s_starts, int32_t* s_lens) {
    constexpr int PER = (kWindowSeqs + 64 * W) / (64 * W);
    __shared__ int s_sum[W], s_ranges[W], s_most[W];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int per = (a.num_seqs + 64 * W) / (64 * W);  // sequences a thread: 1 .. PER
    const auto ranges_of = [&](int entries) { return (entries + kWindowLeast - 1) / kWindowLeast; };
    int raw[PER], sum = 0, most = 0, ranges = 0;
#pragma unroll
    for (int i = 0; i < PER; i++) {
        if (i >= per) break;
        const int r = threadIdx.x * per + i;
        raw[i] = r < a.num_seqs ? a.d.context_lens[r] : 0;
    }
#pragma unroll
    for (int i = 0; i < PER; i++) {
        if (i >= per) break;
        const int len = max(0, clamp_len(a.d, raw[i]));
        s_lens[threadIdx.x * per + i] = len;
        raw[i] = window_list(len, a.sink, a.window).entries();
        sum += raw[i];
        most = max(most, raw[i]);
        ranges += ranges_of(raw[i]);
    }
    const int upto = wave_prefix(sum), ranges_upto = wave_prefix(ranges);
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) most = max(most, __shfl_xor(most, o, 64));
    if (lane == 63) {
        s_sum[wave] = upto;
        s_ranges[wave] = ranges_upto;
        s_most[wave] = most;
    }
    __syncthreads();
    int at = upto - sum, ranges_at = ranges_upto - ranges, total = 0, ranges_total = 0;
#pragma unroll
    for (int w = 0; w < W; w++) {
        at += w < wave ? s_sum[w] : 0;
        ranges_at += w < wave ? s_ranges[w] : 0;
        total += s_sum[w];
        ranges_total += s_ranges[w];
        most = max(most, s_most[w]);
    }
    total = __builtin_amdgcn_readfirstlane(total);
    ranges_total = __builtin_amdgcn_readfirstlane(ranges_total);
    most = __builtin_amdgcn_readfirstlane(most);
    const uint32_t Hkv = a.d.num_kv_heads, rows = a.num_seqs * Hkv, all = total * Hkv;
    uint32_t range = max((all + a.groups - 1) / a.groups, static_cast<uint32_t>(kWindowLeast));
    range = (range + W - 1) / W * W;
    bool fill = ranges_total * Hkv <= static_cast<uint32_t>(a.groups);
    if (most > 0 && most * rows == all) {
        const uint32_t even = (all + kSparseCUs - 1) / kSparseCUs, whole = (rows + kSparseCUs - 1) / kSparseCUs * most;  // a CU's
        if (whole <= even + 24 || 3 * whole < 4 * even) {
            range = (rows + a.groups - 1) / a.groups * most;
            fill = false;
        }
    }
    if (fill) {
        range = kWindowLeast;
        at = ranges_at * kWindowLeast;
    }
#pragma unroll
    for (int i = 0; i < PER; i++) {
        if (i >= per) break;
        const int r = threadIdx.x * per + i;
        if (r <= a.num_seqs) s_starts[r] = at;
        at += fill ? ranges_of(raw[i]) * kWindowLeast : raw[i];
    }
    __syncthreads();
    return range;
}

// PASSES: matrix passes of a split operand, 16 / G parts a pass (G <= 4: 1, 8: 2, 16: 3).
template <int D, int KV, bool QF32, int PASSES>
__global__ __launch_bounds__(64 * window_waves(D), window_decode_groups(D, KV) / kSparseCUs * window_waves(D) / 4) void window_decode_kernel(const WindowArgs a) {
    constexpr bool F32 = KV == PA_DTYPE_FP32, I8 = KV == PA_DTYPE_INT8;
    constexpr int NT = D / 16;
    constexpr int W = window_waves(D);
    constexpr int NB = kSparseBuffers;
    constexpr int CH = D < 64 ? D : 64;  // dims per exchange round
    __shared__ float s_m[W][16], s_l[W][16];
    __shared__ float s_o[W][16][CH];
    __shared__ int32_t s_starts[kWindowSeqs + 1], s_lens[kWindowSeqs + 64 * W];
    const int lane = threadIdx.x & 63, q4 = lane >> 4, n = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int Hkv = a.d.num_kv_heads, G = a.d.group;
    const uint32_t range = window_starts<W>(a, s_starts, s_lens);
    const uint32_t all = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(s_starts[a.num_seqs])) * Hkv;
    if (blockIdx.x == 0) {
        for (int r = threadIdx.x; r <= a.num_seqs; r += 64 * W) a.starts[r] = s_starts[r];
        if (threadIdx.x == 0) a.starts[a.num_seqs + 1] = static_cast<int32_t>(range);
    }
    // sequences without a visible token: zeros
    for (int r = blockIdx.x; r < a.num_seqs; r += a.groups)
        if (s_starts[r] == s_starts[r + 1])
            for (int i = threadIdx.x; i < Hkv * G * D; i += 64 * W) a.d.out[static_cast<int64_t>(r) * Hkv * G * D + i] = 0.0f;
    uint32_t at_entry = blockIdx.x * range;
    const uint32_t stop = min(all, at_entry + range);
    if (blockIdx.x >= (all + range - 1) / range) return;
    int r = 0;  // the sequence of the first entry: the last one that starts at or before it
    // (what LDS gives is the same in every lane, and has to be seen to be: descriptors and branches follow from it)
    const auto start_of = [&](int i) { return static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(s_starts[i])); };
    for (int hi = a.num_seqs; r + 1 < hi;) {
        const int mid = (r + hi) >> 1;
        if (start_of(mid) * Hkv <= at_entry) r = mid;
        else hi = mid;
    }
    for (; at_entry < stop;) {
    while (start_of(r + 1) * Hkv <= at_entry) r++;
    const uint32_t base = start_of(r) * Hkv;
    const uint32_t pitch = start_of(r + 1) - start_of(r);  // of a row: its entries, filled up where ranges do not cross rows
    const int kvh = static_cast<int>((at_entry - base) / pitch);
    const uint32_t entry0 = base + kvh * pitch;  // of the row
    const int beg = static_cast<int>(at_entry - entry0);
    at_entry += min(pitch - beg, stop - at_entry);
    const int row = r * Hkv + kvh;
    const int T = __builtin_amdgcn_readfirstlane(s_lens[r]);
    const int lo = window_begin(T, a.window), sink = min(a.sink, T);
    const WindowList list = window_list(T, a.sink, a.window);
    const int held = list.entries(), end = min(held, static_cast<int>(at_entry - entry0));
    const int32_t* table = a.d.block_tables + static_cast<int64_t>(r) * a.d.max_blocks_per_seq;
    // Lane l holds the wave's l-th block of a stretch of 64 W entries: its place in the sequence, its physical block. No
    // load is under a condition, which would make the compiler wait at its end: past the segment the last entry is read again.
    int lb = list.block(min(beg + wave + W * lane, end - 1));
    int id = table[lb];
    bool listed = beg + wave + W * lane < end;

    const float scale = a.d.scale * kLog2e;
    const SparseQuery<D, KV, QF32, PASSES> query(a.d, static_cast<int64_t>(r) * Hkv * G + kvh * G, scale, q4, n);
    SparseState<D, KV, PASSES> state;
    bool any = false;

    for (int e0 = beg + wave; e0 < end;) {
        if (!listed || id >= a.d.num_blocks) id = -1;
        float ks = 0.0f, vs = 0.0f;
        if constexpr (I8) {
            if (id >= 0) {
                ks = a.d.k_scale[static_cast<int64_t>(id) * Hkv + kvh];
                vs = a.d.v_scale[static_cast<int64_t>(id) * Hkv + kvh];
            }
        }
        const int count = min(64, (end - e0 + W - 1) / W);  // the wave's blocks of this stretch, in lanes 0 ..
        any = true;
        int upto = 0;
        SparseBuf<D, KV> buf[NB];
        int at[NB];
        auto load = [&](SparseBuf<D, KV>& b, int& j) {
            j = upto < count ? upto++ : -1;
            sparse_load<D, KV>(a.d, b, j >= 0 ? __builtin_amdgcn_readlane(id, j) : -1, kvh);
        };
        auto compute = [&](SparseBuf<D, KV>& b, int j) {
            float sc[4];
            query.scores(b, ks, j, G, scale, sc);
            const int tok = __builtin_amdgcn_readlane(lb, j) * 16;  // the block's first token
            const int t0 = tok + (KV == PA_DTYPE_BF16 ? 4 * tok_group<KV>(q4) : 4 * q4);
            sparse_v_arrange<D, KV>(b);
            if ((tok < lo && tok + 16 > sink) || tok + 16 > T) {  // not every token of the block is seen
                bool seen[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    seen[i] = t0 + i < T && (t0 + i >= lo || t0 + i < sink);
                    sc[i] = seen[i] ? sc[i] : -INFINITY;
                }
                // their values too: a zero times what an unseen slot may hold (Inf, NaN) is not zero
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    if constexpr (F32) {
#pragma unroll
                        for (int i = 0; i < 4; i++) b.v[t][i] = seen[i] ? b.v[t][i] : 0.0f;
                    } else if constexpr (!I8) {
                        b.v[t].x &= (seen[0] ? 0xffffu : 0u) | (seen[1] ? 0xffff0000u : 0u);
                        b.v[t].y &= (seen[2] ? 0xffffu : 0u) | (seen[3] ? 0xffff0000u : 0u);
                    }
                }
            }
            const float m0 = state.follow(sc, q4);
            float p[4], psum = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                p[i] = __builtin_amdgcn_exp2f(sc[i] - m0);
                psum += p[i];
            }
            state.l_run += psum;
            if (a.parts) {
                const float sum = rows_sum(psum);
                if (lane < G)  // (no score above -inf: a maximum that makes nothing of the sum, which is 0 or NaN)
                    a.parts[(static_cast<int64_t>(entry0) + e0 + W * j) * G + lane] = make_float2(state.m_run == -INFINITY ? -FLT_MAX : state.m_run, sum);
            }
            if constexpr (I8) {
                const float vf = readlane_f(vs, j);
                // (an unseen token's zero stays one whatever the block's scale is)
#pragma unroll
                for (int i = 0; i < 4; i++) p[i] = p[i] == 0.0f ? 0.0f : p[i] * vf;
            }
            state.add(p, b, G, n);
        };
#pragma unroll
        for (int i = 0; i < NB - 1; i++) load(buf[i], at[i]);
        bool more = true;
        while (more) {
#pragma unroll
            for (int i = 0; i < NB; i++) {
                load(buf[(i + NB - 1) % NB], at[(i + NB - 1) % NB]);
                if (at[i] < 0) {
                    more = false;
                    break;
                }
                compute(buf[i], at[i]);
            }
        }
        e0 += 64 * W;
        if (e0 < end) {
            lb = list.block(min(e0 + W * lane, end - 1));
            id = table[lb];
            listed = e0 + W * lane < end;
        }
    }

    // ---- the waves' states meet ----
    // A wave that saw blocks but no score above -inf is told from one that saw none by the lowest finite maximum:
    // where no score of the row is, its sum is 0 and the outcome 0 / 0. A NaN score leaves the sum NaN.
    if (any && state.m_run == -INFINITY) state.m_run = -FLT_MAX;
    const float l_tot = rows_sum(state.l_run);
    if (q4 == 0) {
        s_m[wave][n] = state.m_run;
        s_l[wave][n] = l_tot;
    }
    constexpr int TT = CH / 16;                                             // tiles per round
    constexpr int NPART = F32 ? 1 : PASSES == 1 ? 3 : PASSES == 2 ? 2 : 1;  // rows of O that hold a head's parts
#pragma unroll
    for (int c = 0; c < D / CH; c++) {
        if (c > 0) __syncthreads();
#pragma unroll
        for (int tt = 0; tt < TT; tt++)
#pragma unroll
            for (int i = 0; i < 4; i++) s_o[wave][4 * q4 + i][16 * tt + n] = state.acc[c * TT + tt][i];
        __syncthreads();
        for (int idx = threadIdx.x; idx < G * CH; idx += 64 * W) {
            const int g = idx / CH, d = idx % CH;
            // every read of LDS goes out before any is used
            float m[W], l[W], x[W][NPART];
#pragma unroll
            for (int w = 0; w < W; w++) {
                m[w] = s_m[w][g];
                l[w] = s_l[w][g];
#pragma unroll
                for (int k = 0; k < NPART; k++) x[w][k] = s_o[w][g + G * k][d];
            }
            float M = m[0];
#pragma unroll
            for (int w = 1; w < W; w++) M = fmaxf(M, m[w]);
            float L = 0.0f, o = 0.0f;
#pragma unroll
            for (int w = 0; w < W; w++) {
                const float f = m[w] == M ? 1.0f : __builtin_amdgcn_exp2f(m[w] - M);
                float y = x[w][0];
#pragma unroll
                for (int k = 1; k < NPART; k++) y += x[w][k];
                L += l[w] * f;
                o += y * f;
            }
            const int dim = c * CH + d;
            if (end - beg == held) {
                a.d.out[(static_cast<int64_t>(row) * G + g) * D + dim] = o / L;
                if (a.parts && dim == 0) a.total[static_cast<int64_t>(row) * G + g] = make_float2(M, L);
            } else {
                const int64_t pi = (2 * static_cast<int64_t>(blockIdx.x) + (beg == 0)) * G + g;
                a.d.ws_o[pi * D + dim] = o;
                if (dim == 0) {
                    a.d.ws_m[pi] = M;
                    a.d.ws_l[pi] = L;
                }
            }
        }
    }
    if (at_entry < stop) __syncthreads();  // the states have been read
    }
}

// What a row's parts are: list entries [e0, e0 + held), parts in the ranges first .. last. The first part lies in slot 1 of its range, the
// others in slot 0 of theirs.
__device__ __forceinline__ int64_t window_part(uint32_t w, uint32_t first, int G, int g) {
    return (2 * static_cast<int64_t>(w) + (w == first)) * G + g;
}

// The masses of sequence r's list entries from 256 chunk: entry e gets the weights of its block, the sum over query heads h of
// parts.sum * exp2(parts.max - M_h) / L_h in the order of the heads, so that no timing enters. A thread an entry; the heads' M and
// 1 / L stand in LDS. 8 bytes a query head and block are read, against 32 D of the keys and values that the decode reads for it.
__device__ __forceinline__ void window_masses(const WindowArgs& a, int r, int chunk) {
    constexpr int kHeads = 128;  // in LDS at a time
    constexpr int kAhead = 8;    // loads that go out together
    __shared__ float2 s_total[kHeads];
    const int G = a.d.group, Hkv = a.d.num_kv_heads, Hq = Hkv * G;
    const uint32_t before = a.starts[r], pitch = a.starts[r + 1] - before, range = a.starts[a.num_seqs + 1];
    const WindowList list = window_list(max(0, clamp_len(a.d, a.d.context_lens[r])), a.sink, a.window);
    const uint32_t held = list.entries(), e = 256u * chunk + threadIdx.x;
    if (256u * chunk >= held) return;
    float sum = 0.0f;
    for (int h0 = 0; h0 < Hq; h0 += kHeads) {
        if (h0 > 0) __syncthreads();
        const int own = h0 + static_cast<int>(threadIdx.x);
        if (threadIdx.x < kHeads && own < Hq) {
            const int kvh = own / G, g = own - kvh * G;
            const uint32_t e0 = before * Hkv + kvh * pitch, first = e0 / range, last = (e0 + held - 1) / range;
            float M, L;
            if (first == last) {
                const float2 t = a.total[static_cast<int64_t>(r) * Hq + own];
                M = t.x;
                L = t.y;
            } else {
                M = -INFINITY;
                L = 0.0f;
                for (uint32_t w0 = first; w0 <= last; w0 += kAhead) {
                    float m[kAhead], l[kAhead];
#pragma unroll
                    for (int j = 0; j < kAhead; j++) {
                        const int64_t pi = window_part(min(w0 + j, last), first, G, g);
                        m[j] = a.d.ws_m[pi];
                        l[j] = w0 + j <= last ? a.d.ws_l[pi] : 0.0f;
                    }
                    float top = M;
#pragma unroll
                    for (int j = 0; j < kAhead; j++) top = fmaxf(top, m[j]);
                    L *= M == top ? 1.0f : __builtin_amdgcn_exp2f(M - top);
#pragma unroll
                    for (int j = 0; j < kAhead; j++) L += l[j] * (m[j] == top ? 1.0f : __builtin_amdgcn_exp2f(m[j] - top));
                    M = top;
                }
            }
            s_total[threadIdx.x] = make_float2(M, 1.0f / L);
        }
        __syncthreads();
        if (e >= held) continue;
        const int end = min(Hq, h0 + kHeads);
        for (int h = h0; h < end; h += kAhead) {
            float2 p[kAhead];
#pragma unroll
            for (int j = 0; j < kAhead; j++) {
                const int own = min(h + j, end - 1), kvh = own / G;
                p[j] = a.parts[(static_cast<int64_t>(before) * Hkv + static_cast<int64_t>(kvh) * pitch + e) * G + (own - kvh * G)];
            }
#pragma unroll
            for (int j = 0; j < kAhead; j++) {
                const float2 t = s_total[min(h + j, end - 1) - h0];
                if (h + j < end) sum += p[j].y * __builtin_amdgcn_exp2f(p[j].x - t.x) * t.y;
            }
        }
    }
    if (e >= held) return;
    a.mass[static_cast<int64_t>(r) * a.d.max_blocks_per_seq + list.block(e)] += sum;
}

// What follows the decode, in one launch: the parts of rows that were cut, a wave per (row, query head), lanes over dims, in the first
// a.merge_groups workgroups; then the masses.
template <int D>
__global__ __launch_bounds__(256) void window_finish_kernel(const WindowArgs a) {
    if (static_cast<int>(blockIdx.x) >= a.merge_groups) {
        const int i = static_cast<int>(blockIdx.x) - a.merge_groups;
        window_masses(a, i / a.mass_chunks, i % a.mass_chunks);
        return;
    }
    constexpr int DPL = (D + 63) / 64;
    const int lane = threadIdx.x & 63, G = a.d.group, Hkv = a.d.num_kv_heads;
    const int64_t u = static_cast<int64_t>(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (u >= static_cast<int64_t>(a.num_seqs) * Hkv * G) return;
    const uint32_t row = static_cast<uint32_t>(u / G), range = a.starts[a.num_seqs + 1];
    const int g = static_cast<int>(u - static_cast<int64_t>(row) * G);
    const int r = static_cast<int>(row) / Hkv, kvh = static_cast<int>(row) - r * Hkv;
    const uint32_t before = a.starts[r], pitch = a.starts[r + 1] - before;
    if (pitch == 0) return;
    const uint32_t e0 = before * Hkv + kvh * pitch, first = e0 / range, last = (e0 + pitch - 1) / range;
    if (first == last) return;  // written whole
    const auto part = [&](uint32_t w) { return window_part(w, first, G, g); };
    // Lanes hold the maxima and sums of 64 parts, the outputs are loaded kAhead parts at a time, the first ones
    // beside the maxima.
    constexpr int kAhead = 8;
    float x[kAhead][DPL];
    auto load = [&](uint32_t w0) {
#pragma unroll
        for (int j = 0; j < kAhead; j++) {
            const int64_t pi = part(min(w0 + j, last));
#pragma unroll
            for (int k = 0; k < DPL; k++) x[j][k] = a.d.ws_o[pi * D + min(lane + 64 * k, D - 1)];
        }
    };
    load(first);
    float M = -INFINITY;
    for (uint32_t w0 = first; w0 <= last; w0 += 64) M = fmaxf(M, a.d.ws_m[part(min(w0 + lane, last))]);
    M = wave_max_dpp(M);
    float L = 0.0f, o[DPL];
#pragma unroll
    for (int k = 0; k < DPL; k++) o[k] = 0.0f;
    for (uint32_t w0 = first; w0 <= last; w0 += 64) {
        const int64_t pi = part(min(w0 + lane, last));
        const float m = a.d.ws_m[pi], l = a.d.ws_l[pi];
        const float f = w0 + lane > last ? 0.0f : m == M ? 1.0f : __builtin_amdgcn_exp2f(m - M);
        L += w0 + lane > last ? 0.0f : l * f;
        for (uint32_t w = w0; w <= min(last, w0 + 63); w += kAhead) {
            if (w > first) load(w);
#pragma unroll
            for (int j = 0; j < kAhead; j++) {
                if (w + j > last) break;
                const float fj = readlane_f(f, static_cast<int>(w + j - w0));
#pragma unroll
                for (int k = 0; k < DPL; k++) o[k] += x[j][k] * fj;
            }
        }
    }
    L = wave_sum(L);
#pragma unroll
    for (int k = 0; k < DPL; k++)
        if (lane + 64 * k < D) a.d.out[u * D + lane + 64 * k] = o[k] / L;
}

template <int D>
void launch_window_decode(const WindowArgs& a, int kv_dtype, bool q_f32, hipStream_t s) {
    const int G = a.d.group;
    const auto go = [&](auto kernel) { kernel<<<a.groups, 64 * window_waves(D), 0, s>>>(a); };
    const auto by_q = [&](auto kv, auto passes) {
        constexpr int KV = decltype(kv)::value, P = decltype(passes)::value;
        if (q_f32) go(window_decode_kernel<D, KV, true, P>);
        else go(window_decode_kernel<D, KV, false, P>);
    };
    const auto by_group = [&](auto kv) {
        if (G <= 4) by_q(kv, std::integral_constant<int, 1>());
        else if (G == 8) by_q(kv, std::integral_constant<int, 2>());
        else by_q(kv, std::integral_constant<int, 3>());
    };
    if (kv_dtype == PA_DTYPE_FP32) by_q(std::integral_constant<int, PA_DTYPE_FP32>(), std::integral_constant<int, 1>());
    else if (kv_dtype == PA_DTYPE_BF16) by_group(std::integral_constant<int, PA_DTYPE_BF16>());
    else if constexpr (D >= 64) by_group(std::integral_constant<int, PA_DTYPE_INT8>());
    const uint32_t behind = a.merge_groups + static_cast<uint32_t>(a.num_seqs) * a.mass_chunks;
    if (behind > 0) window_finish_kernel<D><<<behind, 256, 0, s>>>(a);
}
#ifndef PA_WINDOW_INSTANTIATE
extern template void launch_window_decode<32>(const WindowArgs&, int, bool, hipStream_t);
extern template void launch_window_decode<64>(const WindowArgs&, int, bool, hipStream_t);
extern template void launch_window_decode<128>(const WindowArgs&, int, bool, hipStream_t);
extern template void launch_window_decode<256>(const WindowArgs&, int, bool, hipStream_t);
#endif

}  // namespace pa
