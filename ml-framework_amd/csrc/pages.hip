// pages.hip -- the books of a paged cache kept on the device: which row of the block tables holds
// which physical blocks, how many rows hold each (refcounts), forking and freeing of rows, blocks for new
// tokens with copy on write, compaction of the pool, and the copies these ask for.
//
// The reference keeps these books on the host: refcounts in BlockShareManager (src/MLFramework/
// Inference/PagedAttention/Sharing/BlockShareManager.cs:34-105), the free list in
// KVCacheBlockManager (KVCacheBlockManager.cs:70-174). A row holds the entries of its whole width that
// lie in [0, num_blocks); every other entry is empty. A block is free when its refcount is 0.
//
// All of it is whole numbers. Refcounts change by integer atomics, whose sums do not depend on their
// order; places in a list come from prefix counts in row order, never from an atomic counter, so the
// same books give the same result every time.
#include <algorithm>
#include <string>

#include "pa_internal.h"

namespace {

constexpr int kForkThreads = 256;
constexpr int kBookThreads = 1024;
constexpr int kCopyThreads = 256;

// ---- fork --------------------------------------------------------------------------------------
// Workgroups 0 .. num_out - 1 write an out row each; the num_in behind them settle the refcounts of an in
// row: its blocks are held by as many rows as the out rows that name it, instead of by one.
__global__ __launch_bounds__(kForkThreads) void pages_fork_kernel(const int32_t* __restrict__ tables_in,
                                                                 const int32_t* __restrict__ lens_in, int32_t num_in,
                                                                 const int32_t* __restrict__ src, int32_t* __restrict__ tables_out,
                                                                 int32_t* __restrict__ lens_out, int32_t num_out,
                                                                 int32_t width, int32_t* __restrict__ refs, int32_t num_blocks) {
    const int tid = threadIdx.x;
    if (static_cast<int>(blockIdx.x) < num_out) {
        const int i = blockIdx.x;
        const int from = src[i];
        const bool some = from >= 0 && from < num_in;
        const int32_t* in = tables_in + static_cast<int64_t>(some ? from : 0) * width;
        int32_t* out = tables_out + static_cast<int64_t>(i) * width;
        for (int j = tid; j < width; j += kForkThreads) out[j] = some ? in[j] : -1;
        if (tid == 0) lens_out[i] = some ? lens_in[from] : 0;
        return;
    }
    const int i = blockIdx.x - num_out;
    int uses = 0;
    for (int j = tid; j < num_out; j += kForkThreads) uses += src[j] == i;
    __shared__ int s_uses[kForkThreads / 64];
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) uses += __shfl_xor(uses, o, 64);
    if ((tid & 63) == 0) s_uses[tid >> 6] = uses;
    __syncthreads();
    uses = 0;
#pragma unroll
    for (int w = 0; w < kForkThreads / 64; w++) uses += s_uses[w];
    if (uses == 1) return;
    const int32_t* in = tables_in + static_cast<int64_t>(i) * width;
    for (int j = tid; j < width; j += kForkThreads) {
        const int id = in[j];
        if (id >= 0 && id < num_blocks) atomicAdd(refs + id, uses - 1);
    }
}

// ---- helpers of the one-workgroup kernels --------------------------------------------------------
constexpr int kBookWaves = kBookThreads / 64;
// The sum of `mine` (the same in every lane of a wave) over the waves before this one, and over all.
__device__ __forceinline__ int waves_before(int mine, int* s_wave, int& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    __syncthreads();  // the previous call's sums have been read
    if (lane == 0) s_wave[wave] = mine;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kBookWaves; w++) {
        const int v = s_wave[w];
        before += w < wave ? v : 0;
        total += v;
    }
    return before;
}
// Set bits of a ballot in the lanes below this one.
__device__ __forceinline__ int lanes_before(uint64_t mask) {
    return __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(mask >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(mask), 0));
}
// Exclusive prefix of a truth value over the workgroup, and the total.
__device__ __forceinline__ int block_prefix(bool mine, int* s_wave, int& total) {
    const uint64_t mask = __ballot(mine);
    return waves_before(__popcll(mask), s_wave, total) + lanes_before(mask);
}
__device__ __forceinline__ int load_now(const int32_t* p) {
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void store_now(int32_t* p, int v) {
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// The workgroup's global writes before it are seen by its reads behind it.
__device__ __forceinline__ void block_sync_global() {
    __threadfence();
    __syncthreads();
}

// ---- reserve -----------------------------------------------------------------------------------
struct ReserveArgs {
    int32_t* tables;
    const int32_t* lens;
    const int32_t* num_new;
    int32_t* refs;
    int32_t* pairs;   // [rows][2]
    int32_t* status;  // [2]
    int32_t* count;   // [num_blocks] scratch: demands of a shared block in this call
    int32_t* last;    // [num_blocks] scratch: the last of them
    int32_t* fresh;   // [demands] scratch: the blocks given out, in order
    int32_t* want;    // [demands] scratch: the demand of each place
    int32_t rows, width, num_blocks, reach;
};

// Demand e = row * reach + j: the j-th block that the row's new tokens go to. Its table entry, or
// null when the row has no such block.
__device__ __forceinline__ int32_t* demand_entry(const ReserveArgs& a, int64_t e, int& row, int& lb) {
    row = static_cast<int>(e / a.reach);
    const int j = static_cast<int>(e - static_cast<int64_t>(row) * a.reach);
    const int len = a.lens[row], n = a.num_new[row];
    if (len < 0 || n <= 0) return nullptr;
    lb = len / 16 + j;
    if (static_cast<int64_t>(lb) * 16 >= static_cast<int64_t>(len) + n || lb >= a.width) return nullptr;
    return a.tables + static_cast<int64_t>(row) * a.width + lb;
}

// In row order, a block a demand: an empty entry takes the lowest free block; an entry that other rows
// hold too takes one in its place (copy on write), except for the last of the rows that hold it when all
// of them ask in this call: it keeps the block, as it would if the rows were worked off one by one.
//
// Up to kBookThreads demands, a thread each: three dependent loads (lengths; table entry; refcount) behind the
// refcounts of the pool's first blocks, and everything else in registers and LDS. What bounds it is the chain of those
// round trips and of the barriers. (The scan's eight loads are compiled to a branch and a wait each, since they
// are under a condition, so they are round trips of this chain too.)
static_assert(2 * kBookThreads == 1 << 11, "the hash has 11 bits");
constexpr int kScan = 8;  // 64-block words of a wave per scan of the pool: 8192 blocks a round
__global__ __launch_bounds__(kBookThreads) void pages_reserve_small_kernel(const ReserveArgs a) {
    __shared__ int s_wave[kBookWaves], s_fresh[kBookThreads];
    // shared blocks that are asked for, by a hash of the id: how many ask, and the last that does
    __shared__ int s_id[2 * kBookThreads], s_count[2 * kBookThreads], s_last[2 * kBookThreads];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    // free[k]: the blocks base + 64 k + lane of this wave's part of the round that are free
    uint64_t free[kScan];
    int refs[kScan];
    auto read = [&](int64_t base) {
#pragma unroll
        for (int k = 0; k < kScan; k++) {
            const int64_t b = base + 64 * (kScan * wave + k) + lane;
            refs[k] = b < a.num_blocks ? a.refs[b] : 1;
        }
    };
    read(0);
    const bool asks = tid < a.rows * a.reach;
    int row = 0, lb = 0;
    int32_t* entry = asks ? demand_entry(a, tid, row, lb) : nullptr;
    int id = entry ? *entry : -1;
    if (id >= a.num_blocks) id = -1;
    const int held = entry && id >= 0 ? a.refs[id] : 0;
    const bool shared = held > 1;
    bool takes = entry && id < 0;
    if (__syncthreads_or(shared)) {
        for (int i = tid; i < 2 * kBookThreads; i += kBookThreads) {
            s_id[i] = -1;
            s_count[i] = 0;
            s_last[i] = -1;
        }
        __syncthreads();
        uint32_t slot = (static_cast<uint32_t>(id) * 2654435761u) >> 21;
        if (shared) {
            for (;;) {  // at most half of the places are ever taken
                const int there = atomicCAS(&s_id[slot], -1, id);
                if (there == -1 || there == id) break;
                slot = (slot + 1) % (2 * kBookThreads);
            }
            atomicAdd(&s_count[slot], 1);
            atomicMax(&s_last[slot], tid);
        }
        __syncthreads();
        if (shared) takes = !(s_count[slot] == held && s_last[slot] == tid);
    }
    int need;
    const int at = block_prefix(takes, s_wave, need);
    int found = 0;
    for (int64_t base = 0; found < need && base < a.num_blocks; base += 64 * kScan * kBookWaves) {
        if (base > 0) read(base);
        int mine = 0, total;
#pragma unroll
        for (int k = 0; k < kScan; k++) {
            free[k] = __ballot(refs[k] <= 0);
            mine += __popcll(free[k]);
        }
        int rank = found + waves_before(mine, s_wave, total);
#pragma unroll
        for (int k = 0; k < kScan; k++) {
            const int r = rank + lanes_before(free[k]);
            if ((free[k] >> lane & 1) && r < need) s_fresh[r] = static_cast<int>(base) + 64 * (kScan * wave + k) + lane;
            rank += __popcll(free[k]);
        }
        found += total;
    }
    if (tid == 0) {
        a.status[0] = found >= need ? need : 0;
        a.status[1] = found >= need ? 0 : need - found;
    }
    __syncthreads();
    int from = -1, to = -1;
    if (takes && found >= need) {
        const int b = s_fresh[at];
        if (id >= 0) {
            atomicSub(a.refs + id, 1);
            if (static_cast<int64_t>(lb) * 16 < a.lens[row]) {  // it holds tokens of the row
                from = id;
                to = b;
            }
        }
        *entry = b;
        a.refs[b] = 1;
    }
    // only a row's first demand can be for a block that holds tokens
    if (asks && tid % a.reach == 0) {
        a.pairs[2 * (tid / a.reach)] = from;
        a.pairs[2 * (tid / a.reach) + 1] = to;
    }
}

// Any number of demands: the same through lists in the workspace.
__global__ __launch_bounds__(kBookThreads) void pages_reserve_kernel(const ReserveArgs a) {
    __shared__ int s_wave[kBookThreads / 64];
    const int tid = threadIdx.x;
    const int64_t demands = static_cast<int64_t>(a.rows) * a.reach;
    for (int64_t i = tid; i < 2 * static_cast<int64_t>(a.rows); i += kBookThreads) a.pairs[i] = -1;
    for (int64_t e = tid; e < demands; e += kBookThreads) {
        int row, lb;
        const int32_t* p = demand_entry(a, e, row, lb);
        const int id = p ? *p : -1;
        if (id >= 0 && id < a.num_blocks && a.refs[id] > 1) {
            store_now(a.count + id, 0);
            store_now(a.last + id, -1);
        }
    }
    block_sync_global();
    for (int64_t e = tid; e < demands; e += kBookThreads) {
        int row, lb;
        const int32_t* p = demand_entry(a, e, row, lb);
        const int id = p ? *p : -1;
        if (id >= 0 && id < a.num_blocks && a.refs[id] > 1) {
            atomicAdd(a.count + id, 1);
            atomicMax(a.last + id, static_cast<int>(e));
        }
    }
    block_sync_global();
    int need = 0;
    for (int64_t e0 = 0; e0 < demands; e0 += kBookThreads) {
        const int64_t e = e0 + tid;
        bool takes = false;
        if (e < demands) {
            int row, lb;
            const int32_t* p = demand_entry(a, e, row, lb);
            if (p) {
                const int id = *p;
                if (id < 0 || id >= a.num_blocks) {
                    takes = true;
                } else if (a.refs[id] > 1) {
                    takes = !(load_now(a.count + id) == a.refs[id] && load_now(a.last + id) == static_cast<int>(e));
                }
            }
        }
        int total;
        const int at = need + block_prefix(takes, s_wave, total);
        if (takes) store_now(a.want + at, static_cast<int>(e));
        need += total;
    }
    // the lowest free blocks
    int found = 0;
    for (int64_t b0 = 0; b0 < a.num_blocks && found < need; b0 += kBookThreads) {
        const int64_t b = b0 + tid;
        const bool is_free = b < a.num_blocks && a.refs[b] <= 0;
        int total;
        const int at = found + block_prefix(is_free, s_wave, total);
        if (is_free && at < need) store_now(a.fresh + at, static_cast<int>(b));
        found += total;
    }
    if (tid == 0) {
        a.status[0] = found >= need ? need : 0;
        a.status[1] = found >= need ? 0 : need - found;
    }
    if (found < need) return;
    block_sync_global();
    for (int i = tid; i < need; i += kBookThreads) {
        const int e = load_now(a.want + i), b = load_now(a.fresh + i);
        int row, lb;
        int32_t* p = demand_entry(a, e, row, lb);
        const int old = *p;
        if (old >= 0 && old < a.num_blocks) {
            atomicSub(a.refs + old, 1);
            if (static_cast<int64_t>(lb) * 16 < a.lens[row]) {  // it holds tokens of the row
                a.pairs[2 * static_cast<int64_t>(row)] = old;
                a.pairs[2 * static_cast<int64_t>(row) + 1] = b;
            }
        }
        *p = b;
        a.refs[b] = 1;
    }
}

// ---- compaction --------------------------------------------------------------------------------
struct CompactArgs {
    int32_t* tables;
    int32_t* refs;
    int32_t* pairs;   // [max_moves][2]
    int32_t* status;  // [2]
    int32_t* rank;    // [num_blocks] scratch: the place of a moved block in the list
    int32_t* counts;  // [2] scratch: moves, the lowest moved block
    int32_t num_blocks, max_moves;
    int64_t entries;  // table entries
};

// The i-th highest live block goes to the i-th lowest free one while that is lower, at most max_moves.
// With L live blocks in all, those are the live blocks at or above L and the free ones below it.
// A word is a ballot over 64 blocks; with the words and the live blocks before each of them in LDS a block's place
// among the live ones is a count of bits. Pools of up to 262144 blocks are read once.
constexpr int kWords = 4096;
__global__ __launch_bounds__(kBookThreads) void pages_compact_kernel(const CompactArgs a) {
    __shared__ uint64_t s_word[kWords];  // live blocks
    __shared__ int s_before[kWords];     // live blocks of the round before each word
    __shared__ int s_wave[kBookWaves];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    constexpr int kRound = 64 * kWords;
    const auto words_of = [&](int base) { return static_cast<int>(min(static_cast<int64_t>(kWords), (static_cast<int64_t>(a.num_blocks) - base + 63) / 64)); };
    // the words of the blocks from `base` on; returns their live blocks
    const auto scan = [&](int base) {
        const int words = words_of(base);
        __syncthreads();  // the words of the round before have been read
        constexpr int UN = 8;  // words a step; each load, being under a condition, is waited for before the next
        for (int k0 = wave; k0 < words; k0 += UN * kBookWaves) {
            int refs[UN];
#pragma unroll
            for (int j = 0; j < UN; j++) {
                const int64_t b = static_cast<int64_t>(base) + 64 * (k0 + j * kBookWaves) + lane;
                refs[j] = b < a.num_blocks ? a.refs[b] : 0;
            }
#pragma unroll
            for (int j = 0; j < UN; j++) {
                const uint64_t w = __ballot(refs[j] > 0);
                if (lane == 0 && k0 + j * kBookWaves < words) s_word[k0 + j * kBookWaves] = w;
            }
        }
        __syncthreads();
        constexpr int PT = kWords / kBookThreads;
        int n[PT], mine = 0, total;
#pragma unroll
        for (int k = 0; k < PT; k++) {
            n[k] = tid * PT + k < words ? __popcll(s_word[tid * PT + k]) : 0;
            mine += n[k];
        }
        const int incl = pa::wave_prefix(mine);
        int at = waves_before(__builtin_amdgcn_readlane(incl, 63), s_wave, total) + incl - mine;
#pragma unroll
        for (int k = 0; k < PT; k++) {
            if (tid * PT + k < words) s_before[tid * PT + k] = at;
            at += n[k];
        }
        __syncthreads();
        return total;
    };
    int live = 0;
    for (int64_t base = 0; base < a.num_blocks; base += kRound) live += scan(static_cast<int>(base));
    int low = 0;  // live blocks below `live`
    const bool once = a.num_blocks <= kRound;
    for (int64_t base = 0, before = 0; base < live; base += kRound) {
        const int total = once ? live : scan(static_cast<int>(base));
        const int64_t at = live - base;
        if (at >= 64ll * words_of(static_cast<int>(base))) {
            low = static_cast<int>(before) + total;
        } else {
            low = static_cast<int>(before) + s_before[at / 64] + __popcll(s_word[at / 64] & ((1ull << (at % 64)) - 1));
        }
        before += total;
    }
    const int full = live - low, n = min(full, a.max_moves);
    int before = 0;  // live blocks of earlier rounds
    for (int64_t base = 0; base < a.num_blocks; base += kRound) {
        const int total = once ? live : scan(static_cast<int>(base));
        const int words = words_of(static_cast<int>(base));
        for (int k = wave; k < words; k += kBookWaves) {
            const uint64_t word = s_word[k];
            const int64_t b64 = base + 64 * k + lane;
            const int lb = before + s_before[k] + lanes_before(word);  // live blocks below b
            if (b64 >= a.num_blocks) continue;
            const int b = static_cast<int>(b64), i = live - 1 - lb;  // i: a live block's place from the top
            if (!(word >> lane & 1)) {
                if (b < live && b - lb < n) a.pairs[2 * static_cast<int64_t>(b - lb) + 1] = b;
            } else if (i < n) {  // (at or above `live`)
                a.pairs[2 * static_cast<int64_t>(i)] = b;
                a.rank[b] = i;
                if (i == n - 1) a.counts[1] = b;
            } else if (i == n && n < full) {
                a.status[1] = b + 1;  // the highest that stays, where the moves are cut short
            }
        }
        before += total;
    }
    if (tid == 0) {
        a.status[0] = a.counts[0] = n;
        if (n == full) a.status[1] = live;
    }
}

// Refcounts move along, table entries of moved blocks take the new names, and the list's tail is cleared.
__global__ __launch_bounds__(256) void pages_rename_kernel(const CompactArgs a) {
    const int n = a.counts[0], lowest = n > 0 ? a.counts[1] : a.num_blocks;
    const int64_t first = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x, step = static_cast<int64_t>(gridDim.x) * 256;
    for (int64_t i = first; i < a.max_moves; i += step) {
        if (i < n) {
            const int s = a.pairs[2 * i], d = a.pairs[2 * i + 1];
            a.refs[d] = a.refs[s];
            a.refs[s] = 0;
        } else {
            a.pairs[2 * i] = -1;
            a.pairs[2 * i + 1] = -1;
        }
    }
    for (int64_t i = first; i < a.entries; i += step) {
        const int id = a.tables[i];
        if (id < lowest || id >= a.num_blocks) continue;
        const int k = a.rank[id];  // written for every moved block; anything for an id that was not live
        if (k >= 0 && k < n && a.pairs[2 * static_cast<int64_t>(k)] == id) a.tables[i] = a.pairs[2 * static_cast<int64_t>(k) + 1];
    }
}

// ---- copies ------------------------------------------------------------------------------------
struct CopyArgs {
    char* k;
    char* v;
    char* bounds;    // null: none
    float* stat[4];  // k_scale, v_scale, k_absmax, v_absmax (int8)
    const int32_t* pairs;
    const int32_t* num_pairs;  // null: max_pairs
    int64_t part;              // bytes of K (of V) per block
    int64_t bound;             // bytes of the key bounds per block
    int32_t max_pairs, pieces, num_blocks, hkv;
};
constexpr int kPieceWords = 2;  // 16-byte words a lane
constexpr int kPieceBytes = kCopyThreads * 16 * kPieceWords;
constexpr int kCopyGroups = 8192;  // (2048: 82.6 us where this takes 81.6, 2.3k pages of 64 KB)

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// Piece u % pieces of pair u / pieces: K in pieces, V likewise, then the key bounds, then the statistics.
__global__ __launch_bounds__(kCopyThreads) void copy_pages_kernel(const CopyArgs c) {
    const int n = c.num_pairs ? max(0, min(*c.num_pairs, c.max_pairs)) : c.max_pairs;
    const int64_t units = static_cast<int64_t>(n) * c.pieces;
    const int kp = static_cast<int>((c.part + kPieceBytes - 1) / kPieceBytes);
    const int bp = static_cast<int>((c.bound + kPieceBytes - 1) / kPieceBytes);
    const int tid = threadIdx.x;
    for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
        const int64_t i = u / c.pieces;
        int piece = static_cast<int>(u - i * c.pieces);
        const int32_t src = c.pairs[2 * i], dst = c.pairs[2 * i + 1];
        if (src < 0 || src >= c.num_blocks || dst < 0 || dst >= c.num_blocks || src == dst) continue;
        char* base = c.k;
        int64_t len = c.part;
        if (piece >= kp) {
            piece -= kp;
            base = c.v;
            if (piece >= kp) {
                piece -= kp;
                base = c.bounds;
                len = c.bound;
                if (piece >= bp) {  // the statistics
                    for (int k = tid; k < 4 * c.hkv; k += kCopyThreads) {
                        float* s = c.stat[k / c.hkv];
                        const int h = k % c.hkv;
                        s[static_cast<int64_t>(dst) * c.hkv + h] = s[static_cast<int64_t>(src) * c.hkv + h];
                    }
                    continue;
                }
            }
        }
        const int64_t off = static_cast<int64_t>(piece) * kPieceBytes + tid * 16;
        const u32x4* from = reinterpret_cast<const u32x4*>(base + src * len + off);
        u32x4* to = reinterpret_cast<u32x4*>(base + dst * len + off);
        u32x4 x[kPieceWords];
#pragma unroll
        for (int k = 0; k < kPieceWords; k++)
            if (off + k * kCopyThreads * 16 < len) x[k] = __builtin_nontemporal_load(from + k * kCopyThreads);
#pragma unroll
        for (int k = 0; k < kPieceWords; k++)
            if (off + k * kCopyThreads * 16 < len) __builtin_nontemporal_store(x[k], to + k * kCopyThreads);
    }
}

// Scratch of reserve (four lists) and compact (a list and two counts), ints.
int64_t scratch_ints(const pa_config* cfg, int32_t num_rows, int32_t width) {
    const int64_t nb = cfg->num_blocks, demands = static_cast<int64_t>(num_rows) * width;
    return std::max(2 * nb + 2 * demands, nb + 2);
}

bool overlap(const void* a, int64_t na, const void* b, int64_t nb) {
    const char *x = static_cast<const char*>(a), *y = static_cast<const char*>(b);
    return x < y + nb && y < x + na;
}

}  // namespace

extern "C" {

pa_status pa_pages_workspace_size(const pa_config* cfg, int32_t num_rows, int32_t max_blocks_per_seq, size_t* bytes) {
    const char* const f = "pa_pages_workspace_size";
    pa_status st = pa::check_config(cfg, f);
    if (st != PA_SUCCESS) return st;
    if (!bytes) return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": bytes is null");
    if (num_rows < 0 || max_blocks_per_seq < 0) return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": negative size");
    *bytes = static_cast<size_t>(scratch_ints(cfg, num_rows, max_blocks_per_seq)) * 4;
    return pa::clear_error();
}

pa_status pa_pages_fork(pa_stream* stream, const pa_config* cfg, const int32_t* tables_in, const int32_t* lens_in,
                        int32_t num_in, const int32_t* src, int32_t* tables_out, int32_t* lens_out, int32_t num_out,
                        int32_t max_blocks_per_seq, int32_t* refcounts) {
    const char* const f = "pa_pages_fork";
    pa_status st = pa::check_config(cfg, f);
    if (st != PA_SUCCESS) return st;
    if (num_in < 0 || num_out < 0 || max_blocks_per_seq < 0)
        return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": negative size");
    if (static_cast<int64_t>(num_in) + num_out == 0) return pa::clear_error();
    if (!pa::fits_grid(static_cast<int64_t>(num_in) + num_out, kForkThreads))
        return pa::set_error(PA_ERROR_UNSUPPORTED, std::string(f) + ": too many rows for one call");
    if (!refcounts || (num_in > 0 && (!tables_in || !lens_in)) || (num_out > 0 && (!src || !tables_out || !lens_out)))
        return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": null pointer");
    const int64_t row = static_cast<int64_t>(max_blocks_per_seq) * 4;
    if (num_in > 0 && num_out > 0 &&
        (overlap(tables_in, num_in * row, tables_out, num_out * row) || overlap(lens_in, num_in * 4ll, lens_out, num_out * 4ll) ||
         overlap(src, num_out * 4ll, lens_out, num_out * 4ll) || overlap(src, num_out * 4ll, tables_out, num_out * row)))
        return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": the out rows must not overlap the inputs");
    pa::StreamDevice dev(stream);
    pages_fork_kernel<<<num_out + num_in, kForkThreads, 0, pa::native(stream)>>>(
        tables_in, lens_in, num_in, src, tables_out, lens_out, num_out, max_blocks_per_seq, refcounts, cfg->num_blocks);
    PA_HIP_CHECK(hipGetLastError());
    return pa::clear_error();
}

pa_status pa_pages_reserve(pa_stream* stream, const pa_config* cfg, int32_t* tables, const int32_t* lens,
                           const int32_t* num_new, int32_t num_rows, int32_t max_blocks_per_seq,
                           int32_t max_new_per_row, int32_t* refcounts, int32_t* copy_pairs, int32_t* status,
                           void* workspace, size_t workspace_bytes) {
    const char* const f = "pa_pages_reserve";
    pa_status st = pa::check_config(cfg, f);
    if (st != PA_SUCCESS) return st;
    if (num_rows < 0 || max_blocks_per_seq < 0 || max_new_per_row < 0)
        return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": negative size");
    if (!status) return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": status is null");
    if (num_rows > 0 && (!tables || !lens || !num_new || !refcounts || !copy_pairs))
        return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": null pointer");
    // Blocks that one row's new tokens can touch.
    const int64_t reach = std::min<int64_t>(max_new_per_row == 0 ? 0 : (static_cast<int64_t>(max_new_per_row) + 14) / 16 + 1,
                                            max_blocks_per_seq);
    if (reach * num_rows > INT32_MAX) return pa::set_error(PA_ERROR_UNSUPPORTED, std::string(f) + ": too many rows for one call");
    const size_t need = static_cast<size_t>(scratch_ints(cfg, num_rows, max_blocks_per_seq)) * 4;
    if (need > workspace_bytes || (need > 0 && !workspace))
        return pa::set_error(PA_ERROR_WORKSPACE_TOO_SMALL, std::string(f) + ": workspace needs " + std::to_string(need) + " bytes");
    if (reinterpret_cast<uintptr_t>(workspace) & 3)
        return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": workspace must be 4-byte aligned");
    ReserveArgs a{};
    a.tables = tables;
    a.lens = lens;
    a.num_new = num_new;
    a.refs = refcounts;
    a.pairs = copy_pairs;
    a.status = status;
    a.count = static_cast<int32_t*>(workspace);
    a.last = a.count + cfg->num_blocks;
    a.fresh = a.last + cfg->num_blocks;
    a.want = a.fresh + static_cast<int64_t>(num_rows) * max_blocks_per_seq;
    a.rows = num_rows;
    a.width = max_blocks_per_seq;
    a.num_blocks = cfg->num_blocks;
    a.reach = static_cast<int32_t>(reach);
    pa::StreamDevice dev(stream);
    // (no rows: refcounts may be null, and only the other kernel reads them for a demand alone)
    if (num_rows > 0 && reach >= 1 && reach * num_rows <= kBookThreads)
        pages_reserve_small_kernel<<<1, kBookThreads, 0, pa::native(stream)>>>(a);
    else
        pages_reserve_kernel<<<1, kBookThreads, 0, pa::native(stream)>>>(a);
    PA_HIP_CHECK(hipGetLastError());
    return pa::clear_error();
}

pa_status pa_pages_compact(pa_stream* stream, const pa_config* cfg, int32_t* tables, int32_t num_rows,
                           int32_t max_blocks_per_seq, int32_t* refcounts, int32_t max_moves, int32_t* pairs,
                           int32_t* status, void* workspace, size_t workspace_bytes) {
    const char* const f = "pa_pages_compact";
    pa_status st = pa::check_config(cfg, f);
    if (st != PA_SUCCESS) return st;
    if (num_rows < 0 || max_blocks_per_seq < 0 || max_moves < 0)
        return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": negative size");
    if (!status || (cfg->num_blocks > 0 && !refcounts) || (max_moves > 0 && !pairs) ||
        (num_rows > 0 && max_blocks_per_seq > 0 && !tables))
        return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": null pointer");
    const size_t need = static_cast<size_t>(scratch_ints(cfg, num_rows, max_blocks_per_seq)) * 4;
    if (need > workspace_bytes || !workspace)
        return pa::set_error(PA_ERROR_WORKSPACE_TOO_SMALL, std::string(f) + ": workspace needs " + std::to_string(need) + " bytes");
    if (reinterpret_cast<uintptr_t>(workspace) & 3)
        return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": workspace must be 4-byte aligned");
    CompactArgs a{};
    a.tables = tables;
    a.refs = refcounts;
    a.pairs = pairs;
    a.status = status;
    a.rank = static_cast<int32_t*>(workspace);
    a.counts = a.rank + cfg->num_blocks;
    a.num_blocks = cfg->num_blocks;
    a.max_moves = max_moves;
    a.entries = static_cast<int64_t>(num_rows) * max_blocks_per_seq;
    pa::StreamDevice dev(stream);
    hipStream_t s = pa::native(stream);
    pages_compact_kernel<<<1, kBookThreads, 0, s>>>(a);
    PA_HIP_CHECK(hipGetLastError());
    const int64_t work = std::max<int64_t>(a.entries, max_moves);
    if (work > 0) {
        pages_rename_kernel<<<static_cast<uint32_t>(std::min<int64_t>((work + 255) / 256, 1024)), 256, 0, s>>>(a);
        PA_HIP_CHECK(hipGetLastError());
    }
    return pa::clear_error();
}

pa_status pa_copy_pages(pa_stream* stream, const pa_config* cfg, void* k_cache, void* v_cache, float* k_scale,
                        float* v_scale, float* k_absmax, float* v_absmax, void* key_bounds, const int32_t* pairs,
                        int32_t max_pairs, const int32_t* num_pairs) {
    const char* const f = "pa_copy_pages";
    pa_status st = pa::check_config(cfg, f);
    if (st != PA_SUCCESS) return st;
    if (max_pairs < 0) return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": max_pairs < 0");
    if (!k_cache || !v_cache) return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": null cache pointer");
    if (!pa::aligned16(k_cache) || !pa::aligned16(v_cache) || !pa::aligned16(key_bounds))
        return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": cache and key_bounds pointers must be 16-byte aligned");
    const bool int8 = cfg->kv_dtype == PA_DTYPE_INT8;
    if (int8 && (!k_scale || !v_scale || !k_absmax || !v_absmax))
        return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": int8 cache needs scales and absmax");
    if (max_pairs == 0) return pa::clear_error();
    if (!pairs) return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": pairs is null");
    CopyArgs c{};
    c.k = static_cast<char*>(k_cache);
    c.v = static_cast<char*>(v_cache);
    c.bounds = static_cast<char*>(key_bounds);
    c.stat[0] = k_scale;
    c.stat[1] = v_scale;
    c.stat[2] = k_absmax;
    c.stat[3] = v_absmax;
    c.pairs = pairs;
    c.num_pairs = num_pairs;
    const int64_t head = static_cast<int64_t>(cfg->num_kv_heads) * cfg->head_dim * pa::kv_bytes(cfg);
    c.part = head * pa::kBlockSize;
    c.bound = key_bounds ? head * 2 : 0;
    c.max_pairs = max_pairs;
    c.pieces = static_cast<int32_t>(2 * ((c.part + kPieceBytes - 1) / kPieceBytes) +
                                    (c.bound + kPieceBytes - 1) / kPieceBytes) + (int8 ? 1 : 0);
    c.num_blocks = cfg->num_blocks;
    c.hkv = cfg->num_kv_heads;
    pa::StreamDevice dev(stream);
    const int64_t units = static_cast<int64_t>(max_pairs) * c.pieces;
    copy_pages_kernel<<<static_cast<uint32_t>(std::min<int64_t>(units, kCopyGroups)), kCopyThreads, 0, pa::native(stream)>>>(c);
    PA_HIP_CHECK(hipGetLastError());
    return pa::clear_error();
}

}  // extern "C"
