// sparse_decode.h -- attention of single query tokens over the blocks selected for each KV head.
//
// For query token r, KV head h, query head g of its group, over the tokens t of the listed blocks:
//   s_t = scale * q_g . k_t,  out_g = sum_t exp(s_t - max s) v_t / sum_t exp(s_t - max s)
//
// The lists differ by KV head, so a row is a (query token, KV head). The rows' lists are laid end to end and
// cut into ranges of equal length, one for each workgroup of a chip full of them, so that every CU streams the
// same number of blocks whatever the number of rows, as long as the lists are full: entries are counted as `budget` has
// them, the -1 behind a short list too. The part of a row in a range is a segment; a workgroup works
// its segments off one after another. Its waves take a segment's blocks in turn (wave w: entries w, w +
// waves, ..); a wave streams its blocks through rotating register buffers, one pass with the running maximum
// and sum, and no wave waits for another until the segment ends. There the waves' states meet in LDS; a
// segment that is a whole row is finished at once, the parts of the others (at most two a range) by a merge launch.
// Measured: 256 rows of 128 bf16 blocks (D 128, 269 MB) 47 us, 5.7 TB/s; in two workgroups a row, with
// a merge, 55 us. 384 rows of 255 int8 blocks (404 MB) 82 us, 4.9 TB/s; in three rounds of half rows 95 us.
//
// K and V are read once and G = Hq / Hkv query heads share them (2 G flops a byte at bf16): traffic
// bounds it. The matrix instructions are 16 columns wide and G is 1 to 16, so the columns that a
// group leaves idle carry precision instead: an fp32 value is exactly the sum of three bf16 parts (8
// bits each, cut off one after the other), and part p of head g sits in column g + G p. An fp32
// query's three partial scores are summed across columns; P's three parts make three rows of O, which
// are summed when the row ends. Every product is then exact and every sum in fp32, at the
// instruction count of a single bf16 product for G <= 4 (two passes for G = 8, three for 16). fp32 caches
// run on fp32 matrix instructions. int8 keys go to the byte matrix instruction as they are, against Q as a
// 31-bit integer in units of 2^(e - 30), 2^e > max |q|, in four signed digits, one in each group of columns: these products are
// exact too, but of a Q rounded by up to 2^-30 of its largest value, which is what fp32 sums would keep beside that one,
// and less where its codes are zero (a fifth digit would take a second pass at G = 4); P V runs
// in bf16 as above, its codes converted by placing them in the fraction of 2^23 (an instruction of a quarter of the
// conversion's time). The int8 case is bound by its traffic all the same: with the P V product left out
// altogether it took 86 us of 87. What it lacks against bf16 is the run length, 2 KiB instead of 4 a tile.
#pragma once

#include <cfloat>

#include "decode_mfma.h"

namespace pa {

struct SparseArgs {
    DecodeArgs d;  // caches, q, out, tables, lengths, shape; ws_o / ws_m / ws_l: [slots][G]
    const int32_t* query_seqs;  // null: query r belongs to sequence r
    const int32_t* selected;    // [num_queries][Hkv][budget]
    int32_t num_seqs, budget;
    int32_t rows, range;        // rows; list entries per workgroup (rows * budget fits 32 bits)
};

// Workgroups of a full chip: one per CU; two for blocks of few bytes, whose kernels fit 128 registers (D 64, 512 rows:
// int8 of 128 blocks 38 us with one, 31 with two; bf16 of 64 blocks 24.9 and 23.5; fp32, at 147 registers, stays with
// one, and int8 with D 128 spills if it is made to fit: 103 us where one took 82).
constexpr int kSparseCUs = 256;
__host__ __device__ constexpr int sparse_groups(int head_dim, int kv) {
    return head_dim <= 64 && head_dim * (kv == PA_DTYPE_FP32 ? 4 : kv == PA_DTYPE_BF16 ? 2 : 1) <= 128 ? 2 * kSparseCUs : kSparseCUs;
}
// Waves of a workgroup. For D 256 one per SIMD, since two would have no registers for a second buffer (512 rows: 64
// fp32 blocks 311 us with two and one buffer, 217 with one and two buffers; 128 int8 blocks 155 and 112). fp32 at D 256 still
// spills 32 registers and bf16 at D 64 with fp32 queries and 16 heads a group 3; the former's 217 us are 4.9 TB/s all the same.
__host__ __device__ constexpr int sparse_waves(int head_dim) { return head_dim >= 256 ? 4 : 8; }
constexpr float kLog2e = 1.4426950408889634f;
// Rescaling is deferred until the maximum grows by this (log2 units): P stays below 2^11.
constexpr float kSparseRescale = 11.0f;

// x += the value a rotation by O lanes within each row of 16.
template <int O>
__device__ __forceinline__ float add_ror(float x) {
    return x + __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x120 + O, 0xF, 0xF, false));
}

// Parts 0, 1, 2 of an fp32 value: its top 8 bits, the next 8, the rest; each exact in bf16.
__device__ __forceinline__ float bf16_part(float x, int part) {
    const float hi = __uint_as_float(__float_as_uint(x) & 0xffff0000u);
    const float r = x - hi;
    const float mid = __uint_as_float(__float_as_uint(r) & 0xffff0000u);
    return part == 0 ? hi : part == 1 ? mid : r - mid;
}

// K and V registers of one block, by cache type.
template <int D, int KV>
struct SparseBuf {
    typename MfmaRaw<KV>::K k[D / 32];
    typename MfmaRaw<KV>::V v[D / 16];
};
template <int D>
struct SparseBuf<D, PA_DTYPE_FP32> {
    f32x4_t k[D / 16];  // lane (q4, n): row n, dims 16 u + 4 q4 ..
    f32x4_t v[D / 16];  // dim 16 t + n, tokens 4 q4 ..
};

// Loads of block bid of KV head kv; bid < 0 reads nothing and gives zeros.
template <int D, int KV>
__device__ __forceinline__ void sparse_load(const DecodeArgs& a, SparseBuf<D, KV>& b, int bid, int kv) {
    if constexpr (KV != PA_DTYPE_FP32) {
        load_block<D, KV>(a, b.k, b.v, bid, kv);
    } else {
        constexpr int TILE = 16 * D * 4;
        const int lane = threadIdx.x & 63, q4 = lane >> 4, n = lane & 15;
        const int64_t tile = bid >= 0 ? (static_cast<int64_t>(bid) * a.num_kv_heads + kv) * TILE : 0;
        const int bytes = bid >= 0 ? TILE : 0;
        const __amdgpu_buffer_rsrc_t rk = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<char*>(static_cast<const char*>(a.k_cache) + tile), 0, bytes, kBufferFlags);
        const __amdgpu_buffer_rsrc_t rv = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<char*>(static_cast<const char*>(a.v_cache) + tile), 0, bytes, kBufferFlags);
#pragma unroll
        for (int u = 0; u < D / 16; u++) b.k[u] = buffer_load<f32x4_t>(rk, n * D * 4 + 64 * u + 16 * q4);
#pragma unroll
        for (int t = 0; t < D / 16; t++) b.v[t] = buffer_load<f32x4_t>(rv, (16 * t + n) * 64 + 16 * q4);
    }
}

// The PV operand of four tokens of one dim.
__device__ __forceinline__ s16x4_t sparse_v_operand(const uint2& r) { return v_operand(r); }
__device__ __forceinline__ s16x4_t sparse_v_operand(uint32_t r) {
    const uint32_t w = r ^ 0x80808080u;
    return __builtin_bit_cast(s16x4_t, make_uint2(bf16_pair_of(w, 0), bf16_pair_of(w, 2)));
}

// Register buffers of a wave: the one consumed and those in flight. (Three cost more registers and time nothing
// less: bf16 47.7 us of two, 47.9 of three; int8 86.6, 88.5, 91.7 of four, 96.6 of six; one: 107.)
constexpr int kSparseBuffers = 2;

// The Q operand of a row, whose head 0 starts at q0: column n holds head n % G (part n / G of it where Q is split).
template <int D, int KV, bool QF32, int PASSES>
struct SparseQuery {
    static constexpr bool F32 = KV == PA_DTYPE_FP32, I8 = KV == PA_DTYPE_INT8;
    static constexpr int NSLAB = D / 32;
    static constexpr int NI8 = I8 ? D / 64 : 1;  // QK slabs of 64 dims
    static constexpr int QP = I8 ? (PASSES == 3 ? 4 : PASSES) : QF32 && !F32 ? PASSES : 1;  // passes of Q
    bf16x8_t qb[F32 || I8 ? 1 : QP][F32 || I8 ? 1 : NSLAB];
    float qf[F32 ? D / 4 : 1];
    i32x4_t qd[I8 ? QP : 1][NI8];   // int8: digits of dims (D / 4) q4 + 16 t ..
    float place[I8 ? QP : 1];       // what a unit of this column's sums is worth
    __device__ __forceinline__ SparseQuery(const DecodeArgs& a, int64_t q0, float scale, int q4, int n) {
        const int G = a.group;
        q0 = (q0 + n % G) * D;
        if constexpr (F32) {
#pragma unroll
            for (int u = 0; u < D / 16; u++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int64_t i = q0 + 16 * u + 4 * q4 + j;
                    qf[4 * u + j] = QF32 ? static_cast<const float*>(a.q)[i]
                                         : bf16_to_f32(static_cast<const uint16_t*>(a.q)[i]);
                }
        } else if constexpr (I8) {
            float x[D / 4];
            float top = 0.0f;
#pragma unroll
            for (int e = 0; e < D / 4; e++) {
                const int64_t i = q0 + (D / 4) * q4 + e;
                x[e] = QF32 ? static_cast<const float*>(a.q)[i] : bf16_to_f32(static_cast<const uint16_t*>(a.q)[i]);
                const float f = fabsf(x[e]);
                top = fmaxf(top, f < INFINITY ? f : INFINITY);  // NaN too
            }
            top = rows_max(top);
            const bool bad = !(top < INFINITY);
            // |q| < 2^ex; below 2^-96 (nothing that fp32 sums would keep) all of it counts as zero
            const int ex = max(bad ? 0 : __builtin_amdgcn_frexp_expf(top), -95);
            int32_t z[D / 4];
#pragma unroll
            for (int e = 0; e < D / 4; e++)  // |z| <= 2^30, biased so that its lower three bytes are digits + 128
                z[e] = (bad ? 0 : static_cast<int32_t>(__builtin_rintf(__builtin_amdgcn_ldexpf(x[e], 30 - ex)))) + 0x808080;
#pragma unroll
            for (int p = 0; p < QP; p++) {
                const int j = QP == 1 ? n / G : p * (16 / G) + n / G;  // this column's digit
                const int shift = 8 * min(j, 3);
                const uint32_t flip = j < 3 ? 0x80808080u : 0u, keep = j < 4 ? 0xffffffffu : 0u;
                place[p] = bad ? __builtin_nanf("") : j < 4 ? __builtin_amdgcn_ldexpf(scale, ex - 30 + 8 * j) : 0.0f;
#pragma unroll
                for (int t = 0; t < NI8; t++) {
                    uint32_t w[4];
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        w[k] = 0;
#pragma unroll
                        for (int b = 0; b < 4; b++)
                            w[k] |= (static_cast<uint32_t>(z[16 * t + 4 * k + b]) >> shift & 255u) << (8 * b);
                        w[k] = (w[k] ^ flip) & keep;
                    }
                    qd[p][t] = __builtin_bit_cast(i32x4_t, make_uint4(w[0], w[1], w[2], w[3]));
                }
            }
        } else {
#pragma unroll
            for (int s = 0; s < NSLAB; s++) {
                const int64_t i = q0 + k_dim0<D, KV>(s, q4);
                if constexpr (!QF32) {
                    qb[0][s] = __builtin_bit_cast(bf16x8_t, *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.q) + i));
                } else {
                    const f32x4_t* src = reinterpret_cast<const f32x4_t*>(static_cast<const float*>(a.q) + i);
                    const f32x4_t x0 = src[0], x1 = src[1];
#pragma unroll
                    for (int p = 0; p < QP; p++) {
                        const int part_n = PASSES == 1 ? n / G : p * (16 / G) + n / G;
                        uint32_t w[4];
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const float lo = bf16_part(e < 2 ? x0[2 * e] : x1[2 * e - 4], part_n);
                            const float hi = bf16_part(e < 2 ? x0[2 * e + 1] : x1[2 * e - 3], part_n);
                            w[e] = part_n < 3 ? pack_bf16_trunc(lo, hi) : 0;
                        }
                        qb[p][s] = __builtin_bit_cast(bf16x8_t, make_uint4(w[0], w[1], w[2], w[3]));
                    }
                }
            }
        }
    }
    // The scores of a block's tokens (this lane: its four, for its column's head) in log2 units.
    __device__ __forceinline__ void scores(const SparseBuf<D, KV>& b, float ks, int j, int G, float scale, float (&sc)[4]) const {
        f32x4_t s = {0.0f, 0.0f, 0.0f, 0.0f};
        if constexpr (F32) {
#pragma unroll
            for (int u = 0; u < D / 16; u++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    s = __builtin_amdgcn_mfma_f32_16x16x4f32(b.k[u][i], qf[4 * u + i], s, 0, 0, 0);
        } else if constexpr (I8) {
            const float k_scale = readlane_f(ks, j);
            i32x4_t c[QP];
#pragma unroll
            for (int p = 0; p < QP; p++) {
                c[p] = i32x4_t{0, 0, 0, 0};
#pragma unroll
                for (int t = 0; t < NI8; t++)
                    c[p] = __builtin_amdgcn_mfma_i32_16x16x64_i8(
                        __builtin_bit_cast(i32x4_t, make_uint4(b.k[2 * t].x, b.k[2 * t].y, b.k[2 * t + 1].x, b.k[2 * t + 1].y)),
                        qd[p][t], c[p], 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
#pragma unroll
                for (int p = 0; p < QP; p++) s[i] = __builtin_fmaf(static_cast<float>(c[p][i]), place[p], s[i]);
                s[i] *= k_scale;
            }
        } else {
#pragma unroll
            for (int sl = 0; sl < NSLAB; sl++) {
                const bf16x8_t kop = k_operand(b.k[sl]);
#pragma unroll
                for (int p = 0; p < QP; p++) s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kop, qb[p][sl], s, 0, 0, 0);
            }
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            float x = s[i];
            if constexpr ((QF32 && !F32) || I8) {  // the partial scores of a head's parts
                if (G <= 8) x = add_ror<8>(x);
                if (G <= 4) x = add_ror<4>(x);
                if (G <= 2) x = add_ror<2>(x);
                if (G <= 1) x = add_ror<1>(x);
            }
            sc[i] = I8 ? x : x * scale;
        }
    }
};

// Values as P V takes them.
template <int D, int KV>
__device__ __forceinline__ void sparse_v_arrange(SparseBuf<D, KV>& b) {
    if constexpr (KV == PA_DTYPE_INT8) {
#pragma unroll
        for (int u = 0; u < D / 64; u++) int8_v_transpose(b.v[4 * u], b.v[4 * u + 1], b.v[4 * u + 2], b.v[4 * u + 3]);
    } else if constexpr (KV == PA_DTYPE_BF16) {
#pragma unroll
        for (int u = 0; u < D / 32; u++) bf16_v_exchange(b.v[2 * u], b.v[2 * u + 1]);
    }
}

// A wave's running maxima, sums and outputs. (The waves' exchange at a segment's end stands in each kernel: shared as well, the int8
// decodes took 1 to 2 % more.)
template <int D, int KV, int PASSES>
struct SparseState {
    static constexpr bool F32 = KV == PA_DTYPE_FP32;
    static constexpr int NT = D / 16;
    static constexpr int PP = F32 ? 1 : PASSES;  // passes of P
    float m_run = -INFINITY, l_run = 0.0f;
    f32x4_t acc[NT];
    __device__ __forceinline__ SparseState() {
#pragma unroll
        for (int t = 0; t < NT; t++) acc[t] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    }
    // The maximum follows a block's scores; what is subtracted from them.
    __device__ __forceinline__ float follow(const float (&sc)[4], int q4) {
        const float bm = rows_max(fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3])));
        const bool grow = bm > m_run + kSparseRescale || (m_run == -INFINITY && bm > -INFINITY);
        if (__any(grow)) {
            const float m_new = grow ? bm : m_run;
            const float alpha = grow ? __builtin_amdgcn_exp2f(m_run - m_new) : 1.0f;
            l_run *= alpha;
            m_run = m_new;
            float ar[4];
#pragma unroll
            for (int i = 0; i < 4; i++) ar[i] = __shfl(alpha, 4 * q4 + i, 64);
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) acc[t][i] *= ar[i];
        }
        return m_run == -INFINITY ? 0.0f : m_run;  // no score above -inf yet: P is zero
    }
    // O += P V
    __device__ __forceinline__ void add(const float (&p)[4], const SparseBuf<D, KV>& b, int G, int n) {
        if constexpr (F32) {
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    acc[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(p[i], b.v[t][i], acc[t], 0, 0, 0);
            if constexpr (D == 256) settle<2>();  // (read 9 wait states of 10 later otherwise)
        } else {
            s16x4_t pb[PP];
#pragma unroll
            for (int q = 0; q < PP; q++) {
                const int part_n = PASSES == 1 ? n / G : q * (16 / G) + n / G;
                float x[4];
#pragma unroll
                for (int i = 0; i < 4; i++) x[i] = part_n < 3 ? bf16_part(p[i], part_n) : 0.0f;
                pb[q] = __builtin_bit_cast(s16x4_t, make_uint2(pack_bf16_trunc(x[0], x[1]), pack_bf16_trunc(x[2], x[3])));
            }
#pragma unroll
            for (int t = 0; t < NT; t++) {
                const s16x4_t vop = sparse_v_operand(b.v[t]);
#pragma unroll
                for (int q = 0; q < PP; q++) acc[t] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(pb[q], vop, acc[t], 0, 0, 0);
            }
        }
    }
};

// PASSES: matrix passes of a split operand, 16 / G parts a pass (G <= 4: 1, 8: 2, 16: 3).
template <int D, int KV, bool QF32, int PASSES>
__global__ __launch_bounds__(64 * sparse_waves(D), sparse_groups(D, KV) / kSparseCUs * sparse_waves(D) / 4) void sparse_decode_kernel(const SparseArgs a) {
    constexpr bool F32 = KV == PA_DTYPE_FP32;
    constexpr int NT = D / 16;
    constexpr int W = sparse_waves(D);
    constexpr int NB = kSparseBuffers;
    constexpr int CH = D < 64 ? D : 64;  // dims per exchange round
    __shared__ float s_m[W][16], s_l[W][16];
    __shared__ float s_o[W][16][CH];
    const int lane = threadIdx.x & 63, q4 = lane >> 4, n = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int Hkv = a.d.num_kv_heads, G = a.d.group;
    const uint32_t budget = a.budget, all = static_cast<uint32_t>(a.rows) * budget;
    uint32_t at_entry = blockIdx.x * static_cast<uint32_t>(a.range);
    const uint32_t stop = min(all, at_entry + a.range);
    for (; at_entry < stop;) {
    const int row = static_cast<int>(at_entry / budget);
    const int beg = static_cast<int>(at_entry - row * budget);
    const int end = static_cast<int>(min(budget, beg + (stop - at_entry)));
    at_entry += end - beg;
    const int r = row / Hkv, kvh = row - r * Hkv;
    // Lane l holds the wave's l-th block of a stretch of 64 W entries: its place in the sequence, its physical block. The
    // first stretch's places come together with the sequence's number and length, its blocks while Q is split. No load is
    // under a condition, which would make the compiler wait at its end: past the segment the last entry is read again,
    // and where there is no table or place in it, the list.
    const int32_t* list = a.selected + static_cast<int64_t>(row) * a.budget;
    int lb = list[min(beg + wave + W * lane, end - 1)];
    const int raw_len = a.d.context_lens[r], named = (a.query_seqs ? a.query_seqs : a.d.context_lens)[r];
    const int seq = a.query_seqs ? named : r;
    const int T = seq >= 0 && seq < a.num_seqs ? clamp_len(a.d, raw_len) : 0;
    const int nblk = T <= 0 ? 0 : (T + 15) / 16;
    const int32_t* table = T > 0 ? a.d.block_tables + static_cast<int64_t>(seq) * a.d.max_blocks_per_seq : list;
    int id;
    bool listed;
    auto find = [&](int e0) {
        listed = (e0 + W * lane < end) & (lb >= 0) & (lb < nblk);
        id = table[listed ? lb : 0];
    };
    find(beg + wave);

    const float scale = a.d.scale * kLog2e;
    const SparseQuery<D, KV, QF32, PASSES> query(a.d, static_cast<int64_t>(r) * Hkv * G + kvh * G, scale, q4, n);
    SparseState<D, KV, PASSES> state;
    bool any = false;

    for (int e0 = beg + wave; e0 < end;) {
        if (!listed || id >= a.d.num_blocks) id = -1;
        float ks = 0.0f, vs = 0.0f;
        if constexpr (KV == PA_DTYPE_INT8) {
            if (id >= 0) {
                ks = a.d.k_scale[static_cast<int64_t>(id) * Hkv + kvh];
                vs = a.d.v_scale[static_cast<int64_t>(id) * Hkv + kvh];
            }
        }
        uint64_t todo = __ballot(listed);
        any |= todo != 0;
        auto next = [&]() {
            if (!todo) return -1;
            const int j = __builtin_ctzll(todo);
            todo &= todo - 1;
            return j;
        };
        SparseBuf<D, KV> buf[NB];
        int at[NB];
        auto load = [&](SparseBuf<D, KV>& b, int& j) {
            j = next();
            sparse_load<D, KV>(a.d, b, j >= 0 ? __builtin_amdgcn_readlane(id, j) : -1, kvh);
        };
        auto compute = [&](SparseBuf<D, KV>& b, int j) {
            float sc[4];
            query.scores(b, ks, j, G, scale, sc);
            const int lbj = __builtin_amdgcn_readlane(lb, j);
            const int t0 = KV == PA_DTYPE_BF16 ? 4 * tok_group<KV>(q4) : 4 * q4;
            sparse_v_arrange<D, KV>(b);
            if (static_cast<int64_t>(lbj) * 16 + 16 > T) {  // the context ends inside the block
                const int lim = T - lbj * 16 - t0;          // of this lane's four tokens
#pragma unroll
                for (int i = 0; i < 4; i++) sc[i] = i < lim ? sc[i] : -INFINITY;
                // their values too: a zero times what an unused slot may hold (Inf, NaN) is not zero
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    if constexpr (KV == PA_DTYPE_FP32) {
#pragma unroll
                        for (int i = 0; i < 4; i++) b.v[t][i] = i < lim ? b.v[t][i] : 0.0f;
                    } else if constexpr (KV == PA_DTYPE_BF16) {
                        b.v[t].x = lim >= 2 ? b.v[t].x : lim == 1 ? b.v[t].x & 0xffffu : 0u;
                        b.v[t].y = lim >= 4 ? b.v[t].y : lim == 3 ? b.v[t].y & 0xffffu : 0u;
                    }
                }
            }
            const float m0 = state.follow(sc, q4);
            float p[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                p[i] = __builtin_amdgcn_exp2f(sc[i] - m0);
                state.l_run += p[i];
            }
            if constexpr (KV == PA_DTYPE_INT8) {
                const float vf = readlane_f(vs, j);
#pragma unroll
                for (int i = 0; i < 4; i++) p[i] *= vf;
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
            lb = list[min(e0 + W * lane, end - 1)];
            find(e0);
        }
    }

    // ---- the waves' states meet ----
    // A wave that saw tokens but no score above -inf is told from one that saw none by the lowest finite maximum:
    // where no score of the row is, its sum is 0 and the outcome 0 / 0. A NaN score leaves the sum NaN. (The exchange
    // with a branch per wave and its reads one by one took 8000 of 17000 cycles at 8 rows of 64 blocks: 12.1 us for
    // 10.8 with the merge.)
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
            if (end - beg == a.budget) {
                a.d.out[(static_cast<int64_t>(row) * G + g) * D + dim] = M == -INFINITY ? 0.0f : o / L;  // no token: zeros
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

// The parts of a row that was cut: one wave per (row, query head), lanes over dims. The first part lies in slot 1
// of its range, the others in slot 0 of theirs.
template <int D>
__global__ __launch_bounds__(256) void sparse_merge_kernel(const SparseArgs a) {
    constexpr int DPL = (D + 63) / 64;
    const int lane = threadIdx.x & 63, G = a.d.group;
    const int64_t u = static_cast<int64_t>(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (u >= static_cast<int64_t>(a.rows) * G) return;
    const uint32_t row = static_cast<uint32_t>(u) / G, range = a.range;
    const int g = static_cast<int>(u - static_cast<int64_t>(row) * G);
    const uint32_t first = row * a.budget / range, last = (row * a.budget + a.budget - 1) / range;
    if (first == last) return;  // written whole
    const auto part = [&](uint32_t w) { return (2 * static_cast<int64_t>(w) + (w == first)) * G + g; };
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
        if (lane + 64 * k < D) a.d.out[u * D + lane + 64 * k] = M == -INFINITY ? 0.0f : o[k] / L;
}

template <int D>
void launch_sparse_decode(const SparseArgs& a, int kv_dtype, bool q_f32, hipStream_t s) {
    const uint32_t all = static_cast<uint32_t>(a.rows) * a.budget, grid = (all + a.range - 1) / a.range;
    const int G = a.d.group;
    const auto go = [&](auto kernel) { kernel<<<grid, 64 * sparse_waves(D), 0, s>>>(a); };
    const auto by_q = [&](auto kv, auto passes) {
        constexpr int KV = decltype(kv)::value, P = decltype(passes)::value;
        if (q_f32) go(sparse_decode_kernel<D, KV, true, P>);
        else go(sparse_decode_kernel<D, KV, false, P>);
    };
    const auto by_group = [&](auto kv) {
        if (G <= 4) by_q(kv, std::integral_constant<int, 1>());
        else if (G == 8) by_q(kv, std::integral_constant<int, 2>());
        else by_q(kv, std::integral_constant<int, 3>());
    };
    if (kv_dtype == PA_DTYPE_FP32) by_q(std::integral_constant<int, PA_DTYPE_FP32>(), std::integral_constant<int, 1>());
    else if (kv_dtype == PA_DTYPE_BF16) by_group(std::integral_constant<int, PA_DTYPE_BF16>());
    else if constexpr (D >= 64) by_group(std::integral_constant<int, PA_DTYPE_INT8>());
    if (a.range % a.budget != 0) {
        const int64_t waves = static_cast<int64_t>(a.rows) * G;
        sparse_merge_kernel<D><<<static_cast<uint32_t>((waves + 3) / 4), 256, 0, s>>>(a);
    }
}
#ifndef PA_SPARSE_INSTANTIATE
extern template void launch_sparse_decode<32>(const SparseArgs&, int, bool, hipStream_t);
extern template void launch_sparse_decode<64>(const SparseArgs&, int, bool, hipStream_t);
extern template void launch_sparse_decode<128>(const SparseArgs&, int, bool, hipStream_t);
extern template void launch_sparse_decode<256>(const SparseArgs&, int, bool, hipStream_t);
#endif

}  // namespace pa
