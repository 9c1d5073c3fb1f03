// key_bounds.hip -- channel-wise bounds of a block's keys, the summary that block selection scores.
//
// For block b, KV head h and channel d:
//   bounds[b][h][0][d] = min over the block's tokens t of K[b][h][t][d],  bounds[b][h][1][d] = max,
// in the cache's own type (int8: codes), so nothing is rounded and the bounds of a block are the
// same whatever order its tokens came in. A NaN key makes its channel's bounds NaN.
//
// Traffic is all there is to it: 16 D elements read and 2 D written per (block, KV head). A wave
// takes one tile: 16-byte loads, 64 / (D elt / 16) token rows an instruction, every load of the tile issued
// before the first is used; the rows held by different lane groups meet in log2 steps of shuffles.
#include <algorithm>
#include <string>

#include "pa_internal.h"

namespace {

constexpr int kWaves = 4;

// IEEE minimum / maximum that keep NaN (v_minimum3 / v_maximum3 on gfx950).
__device__ __forceinline__ float min_nan(float a, float b) { return __builtin_elementwise_minimum(a, b); }
__device__ __forceinline__ float max_nan(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// Element e of a 16-byte word as fp32 (exact for every type).
template <int KV>
__device__ __forceinline__ float elem(const uint4& w, int e) {
    const uint32_t x[4] = {w.x, w.y, w.z, w.w};
    if constexpr (KV == PA_DTYPE_FP32) return __uint_as_float(x[e]);
    else if constexpr (KV == PA_DTYPE_BF16) return e & 1 ? pa::bf16_hi(x[e >> 1]) : pa::bf16_lo(x[e >> 1]);
    else return pa::i8_at(x[e >> 2], e & 3);
}

// The inverse of elem() for values that came from it.
template <int KV, int N>
__device__ __forceinline__ uint4 pack(const float (&v)[N]) {
    uint32_t x[4] = {0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < N; e++) {
        if constexpr (KV == PA_DTYPE_FP32) x[e] = __float_as_uint(v[e]);
        else if constexpr (KV == PA_DTYPE_BF16) x[e >> 1] |= (__float_as_uint(v[e]) >> 16) << (16 * (e & 1));
        else x[e >> 2] |= (static_cast<uint32_t>(static_cast<int>(v[e])) & 255u) << (8 * (e & 3));
    }
    return make_uint4(x[0], x[1], x[2], x[3]);
}

// Wave u: KV head u % Hkv of the (u / Hkv)-th block from the first that sequence `seq` writes to.
template <int D, int KV>
__global__ __launch_bounds__(64 * kWaves) void key_bounds_kernel(const void* __restrict__ k_cache,
                                                                const int32_t* __restrict__ tables, int32_t width,
                                                                const int32_t* __restrict__ start_pos,
                                                                const int32_t* __restrict__ num_new, int32_t reach,
                                                                int32_t hkv, int32_t num_blocks,
                                                                void* __restrict__ bounds) {
    constexpr int ELT = KV == PA_DTYPE_FP32 ? 4 : KV == PA_DTYPE_BF16 ? 2 : 1;
    constexpr int E = 16 / ELT;     // elements per word
    constexpr int LPR = D / E;      // lanes per token row
    constexpr int RPI = 64 / LPR;   // token rows per load instruction
    constexpr int NI = 16 / RPI;    // load instructions per tile
    static_assert(LPR <= 64 && RPI <= 16, "tile shape");
    const int seq = blockIdx.y;
    const int lane = threadIdx.x & 63;
    const int u = blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int j = u / hkv, h = u - j * hkv;
    const int start = start_pos[seq], n = num_new[seq];
    if (j >= reach || start < 0 || n <= 0) return;
    const int64_t end = static_cast<int64_t>(start) + n;
    const int lb = start / 16 + j;
    if (static_cast<int64_t>(lb) * 16 >= end || lb >= width) return;
    const int id = tables[static_cast<int64_t>(seq) * width + lb];
    if (id < 0 || id >= num_blocks) return;
    const int held = static_cast<int>(min(static_cast<int64_t>(16), end - static_cast<int64_t>(lb) * 16));
    const int64_t tile = (static_cast<int64_t>(id) * hkv + h) * 16 * D * ELT;
    const int col = lane % LPR, row = lane / LPR;
    const uint4* src = reinterpret_cast<const uint4*>(static_cast<const char*>(k_cache) + tile);
    uint4 w[NI];
#pragma unroll
    for (int i = 0; i < NI; i++) {
        const int t = min(i * RPI + row, held - 1);  // rows past the block's tokens repeat its last one
        w[i] = src[t * LPR + col];
    }
    float lo[E], hi[E];
#pragma unroll
    for (int e = 0; e < E; e++) lo[e] = hi[e] = elem<KV>(w[0], e);
#pragma unroll
    for (int i = 1; i < NI; i++)
#pragma unroll
        for (int e = 0; e < E; e++) {
            const float x = elem<KV>(w[i], e);
            lo[e] = min_nan(lo[e], x);
            hi[e] = max_nan(hi[e], x);
        }
#pragma unroll
    for (int o = LPR; o < 64; o <<= 1)
#pragma unroll
        for (int e = 0; e < E; e++) {
            lo[e] = min_nan(lo[e], __shfl_xor(lo[e], o, 64));
            hi[e] = max_nan(hi[e], __shfl_xor(hi[e], o, 64));
        }
    uint4* dst = reinterpret_cast<uint4*>(static_cast<char*>(bounds) +
                                          (static_cast<int64_t>(id) * hkv + h) * 2 * D * ELT);
    if constexpr (RPI >= 2) {  // row group 0 writes the minima, group 1 the maxima behind them
        if (row < 2) dst[row * LPR + col] = row == 0 ? pack<KV>(lo) : pack<KV>(hi);
    } else {
        dst[col] = pack<KV>(lo);
        dst[LPR + col] = pack<KV>(hi);
    }
}

template <int D>
void launch(int kv, dim3 grid, hipStream_t s, const void* k, const int32_t* tables, int32_t width, const int32_t* start,
            const int32_t* num_new, int32_t reach, int32_t hkv, int32_t nb, void* bounds) {
    if (kv == PA_DTYPE_FP32)
        key_bounds_kernel<D, PA_DTYPE_FP32><<<grid, 64 * kWaves, 0, s>>>(k, tables, width, start, num_new, reach, hkv, nb, bounds);
    else if (kv == PA_DTYPE_BF16)
        key_bounds_kernel<D, PA_DTYPE_BF16><<<grid, 64 * kWaves, 0, s>>>(k, tables, width, start, num_new, reach, hkv, nb, bounds);
    else if constexpr (D >= 64)
        key_bounds_kernel<D, PA_DTYPE_INT8><<<grid, 64 * kWaves, 0, s>>>(k, tables, width, start, num_new, reach, hkv, nb, bounds);
}

}  // namespace

extern "C" {

pa_status pa_key_bounds_bytes(const pa_config* cfg, size_t* bytes) {
    pa_status st = pa::check_config(cfg, "pa_key_bounds_bytes");
    if (st != PA_SUCCESS) return st;
    if (!bytes) return pa::set_error(PA_ERROR_INVALID_ARGUMENT, "pa_key_bounds_bytes: bytes is null");
    *bytes = static_cast<size_t>(cfg->num_blocks) * cfg->num_kv_heads * 2 * cfg->head_dim * pa::kv_bytes(cfg);
    return pa::clear_error();
}

pa_status pa_key_bounds_update(pa_stream* stream, const pa_config* cfg, const void* k_cache, const int32_t* block_tables,
                               int32_t max_blocks_per_seq, const int32_t* start_pos, const int32_t* num_new,
                               int32_t num_seqs, int32_t max_new_per_seq, void* key_bounds) {
    const char* const f = "pa_key_bounds_update";
    pa_status st = pa::check_config(cfg, f);
    if (st != PA_SUCCESS) return st;
    if (num_seqs < 0 || max_new_per_seq < 0 || max_blocks_per_seq < 0)
        return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": negative size");
    if (num_seqs == 0 || max_new_per_seq == 0 || max_blocks_per_seq == 0) return pa::clear_error();
    if (num_seqs > 65535) return pa::set_error(PA_ERROR_UNSUPPORTED, std::string(f) + ": num_seqs must be <= 65535");
    if (!k_cache || !block_tables || !start_pos || !num_new || !key_bounds)
        return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": null pointer");
    if (!pa::aligned16(k_cache) || !pa::aligned16(key_bounds))
        return pa::set_error(PA_ERROR_INVALID_ARGUMENT, std::string(f) + ": k_cache and key_bounds must be 16-byte aligned");
    // A sequence's new tokens touch at most this many blocks (the first may start inside one).
    const int64_t reach = std::min<int64_t>((static_cast<int64_t>(max_new_per_seq) + 14) / 16 + 1, max_blocks_per_seq);
    const int64_t groups = (reach * cfg->num_kv_heads + kWaves - 1) / kWaves;
    if (!pa::fits_grid(groups, 64 * kWaves)) return pa::set_error(PA_ERROR_UNSUPPORTED, std::string(f) + ": too many blocks for one call");
    pa::StreamDevice dev(stream);
    const dim3 grid(static_cast<uint32_t>(groups), num_seqs);
    hipStream_t s = pa::native(stream);
    const auto go = [&](auto launcher) {
        launcher(cfg->kv_dtype, grid, s, k_cache, block_tables, max_blocks_per_seq, start_pos, num_new,
                 static_cast<int32_t>(reach), cfg->num_kv_heads, cfg->num_blocks, key_bounds);
    };
    switch (cfg->head_dim) {
        case 32: go(launch<32>); break;
        case 64: go(launch<64>); break;
        case 128: go(launch<128>); break;
        default: go(launch<256>); break;
    }
    PA_HIP_CHECK(hipGetLastError());
    return pa::clear_error();
}

}  // extern "C"
