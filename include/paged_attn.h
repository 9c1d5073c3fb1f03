/*
 * paged_attn.h -- C-ABI of libpa_hip.so, the MI355X (gfx950) paged-attention backend.
 *
 * The reference framework (werwedc/ml-framework, C#/.NET) reaches native code only through
 * P/Invoke declarations with CallingConvention.Cdecl into libraries it does not ship:
 *   - the CUDA runtime surface of its HAL   src/MLFramework/HAL/CUDA/CudaApi.cs:9-269
 *   - its custom-kernel library             src/MLFramework/HAL/CUDA/CudaKernels.cs:10-141
 *   - the paged-attention operator stub     src/MLFramework/Inference/PagedAttention/Kernels/
 *                                           CudaPagedAttentionKernel.cs:11-49 (throws)
 * Every entry point below replaces one of those declarations (cited per function) or fills the
 * operator stub. All functions are extern "C", take plain pointers and sizes, return a pa_status
 * (0 = success) and never throw. Launch functions validate their arguments on the host and return
 * an error without launching anything when a check fails. Device pointers are owned by the
 * caller; the library never frees memory it did not allocate through pa_alloc.
 *
 * Threading: launch functions are asynchronous on the given stream and return after enqueue. The
 * library keeps no mutable global state except a thread-local last-error string and the per-device
 * scratch array of pa_paged_decode_noalloc, so one pa_device may be driven from several host
 * threads, each with its own stream (pa_paged_decode_noalloc calls excepted: they share the scratch).
 */
#ifndef PAGED_ATTN_H
#define PAGED_ATTN_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define PA_API_VERSION_MAJOR 1
#define PA_API_VERSION_MINOR 1

/* Status codes. Mirrors the integer-error-to-exception mapping of the reference HAL
 * (src/MLFramework/HAL/CUDA/CudaError.cs, CudaException.CheckError used at CudaDevice.cs:15-21). */
typedef enum pa_status {
    PA_SUCCESS = 0,
    PA_ERROR_INVALID_ARGUMENT = 1,   /* null pointer, negative count, out-of-range value      */
    PA_ERROR_INVALID_CONFIG = 2,     /* pa_config inconsistent (heads, head_dim, block size)  */
    PA_ERROR_OUT_OF_MEMORY = 3,      /* device allocation failed                              */
    PA_ERROR_HIP = 4,                /* a HIP runtime call failed; see pa_get_last_error      */
    PA_ERROR_UNSUPPORTED = 5,        /* dtype / head_dim / GQA ratio not compiled             */
    PA_ERROR_WORKSPACE_TOO_SMALL = 6,/* caller workspace smaller than pa_*_workspace_size     */
    PA_ERROR_NO_DEVICE = 7           /* no HIP device with that ordinal                       */
} pa_status;

/* Element types. Values follow the order of MLFramework.Core.DataType only where they coincide
 * (src/MLFramework/Core/DataType.cs:6-21); the ABI fixes its own numbering. */
typedef enum pa_dtype {
    PA_DTYPE_FP32 = 0,
    PA_DTYPE_BF16 = 1,   /* stored as the upper 16 bits of fp32 (truncating conversion,
                            src/MLFramework/Amp/BFloat16.cs:99-117)                              */
    PA_DTYPE_INT8 = 2    /* symmetric int8 with an fp32 scale per (block, KV head)            */
} pa_dtype;

/* Attention phase, numbered as MlFramework.Inference.PagedAttention.Phases.AttentionPhase
 * (Phases/AttentionPhase.cs:6-17): Prefill = 0, Decode = 1. */
typedef enum pa_phase { PA_PHASE_PREFILL = 0, PA_PHASE_DECODE = 1 } pa_phase;

/* pa_config.flags */
#define PA_FLAG_NONE 0u
/* Chunked prefill: apply the reference's mask rule literally (mask only when phase == Decode and
 * the number of cached keys exceeds the number of queries, StandardPagedAttentionKernel.cs:57),
 * i.e. no mask when the prefix is empty or the phase is Prefill. Default: always causal. */
#define PA_FLAG_REFERENCE_LITERAL_MASK 1u
/* Chunked prefill: no mask at all -- the reference's Prefill phase, used by the dense
 * IPagedAttentionKernel interface when called with AttentionPhase.Prefill. */
#define PA_FLAG_NO_MASK 2u

/* Shape/dtype record passed by pointer to every launch function.
 * KV cache layout (per layer, K and V in separate buffers of kv_dtype), one tile per
 * (block, KV head) as in the reference's intended per-block tensor [layers, heads, blockSize,
 * headDim] (src/MLFramework/Inference/PagedAttention/Layers/PagedAttentionLayer.cs:315):
 *   K: [num_blocks][num_kv_heads][block_size][head_dim]   (token rows, row-major)
 *   V: [num_blocks][num_kv_heads][head_dim][block_size]   (dim rows: the tile is transposed so
 *      that P.V reads the 16 tokens of one dimension as one contiguous run)
 * int8 scales and running absolute maxima: fp32 [num_blocks][num_kv_heads], K and V separately. */
typedef struct pa_config {
    int32_t block_size;     /* tokens per physical block; 16 in every shipped configuration    */
    int32_t num_q_heads;    /* Hq                                                               */
    int32_t num_kv_heads;   /* Hkv; Hq % Hkv == 0, query head h reads KV head h / (Hq / Hkv)    */
    int32_t head_dim;       /* D: 64, 128 or 256; 32 for fp32 / bf16 caches (decode, append)  */
    int32_t kv_dtype;       /* pa_dtype of the cache                                            */
    int32_t q_dtype;        /* pa_dtype of Q and of the new K/V handed to pa_kv_append (FP32/BF16) */
    int32_t num_blocks;     /* physical blocks in the pool; ids outside [0, num_blocks) are
                               never dereferenced (decode/prefill read their tokens as zeros,
                               append skips their slots)                                        */
    float   scale;          /* softmax scale; <= 0 selects 1/sqrtf(head_dim)
                               (StandardPagedAttentionKernel.cs:18,28)                          */
    int32_t partition_size; /* decode split-K granularity in tokens; 0 = library default: the
                               batch's blocks are cut into one equal range per resident
                               workgroup (bf16/int8) or 256-token partitions (fp32). Otherwise a
                               multiple of 64 in [64, 4096] (bf16/int8) or 256/512 (fp32).      */
    uint32_t flags;         /* PA_FLAG_*                                                        */
    int32_t num_splits;     /* bf16/int8 decode: 0 = split by partition_size (above); P in
                               [1, 256] = every sequence's context is cut into P partitions of
                               whole blocks (ceil(blocks / P) each, fewer when the sequence has
                               fewer blocks), each streamed by its own worker per KV head and
                               merged with a log-sum-exp reduction -- the per-sequence split-K of
                               DecodeOrchestrator-style long-context decode. Requires
                               partition_size == 0; must be 0 for fp32 caches; the shared-prefix
                               decode ignores it.                                               */
} pa_config;

typedef struct pa_device pa_device;
typedef struct pa_stream pa_stream;
typedef struct pa_event pa_event;
typedef struct pa_graph pa_graph;

typedef struct pa_device_props {
    char name[256];
    char arch[64];             /* e.g. "gfx950:sramecc+:xnack-" */
    size_t total_memory;
    int32_t compute_units;
    int32_t ordinal;
} pa_device_props;

typedef enum pa_memcpy_kind {
    PA_MEMCPY_HOST_TO_HOST = 0,
    PA_MEMCPY_HOST_TO_DEVICE = 1,
    PA_MEMCPY_DEVICE_TO_HOST = 2,
    PA_MEMCPY_DEVICE_TO_DEVICE = 3,
    PA_MEMCPY_DEFAULT = 4
} pa_memcpy_kind;

/* ---- library / errors --------------------------------------------------------------------- */
pa_status pa_get_version(int32_t* major, int32_t* minor);
const char* pa_status_string(pa_status status);
/* Copies the calling thread's last error message (NUL-terminated, truncated to buf_len). */
pa_status pa_get_last_error(char* buf, size_t buf_len);

/* ---- device (replaces CudaApi.CudaGetDeviceCount/CudaSetDevice/CudaGetDeviceProperties/
 *      CudaDeviceSynchronize, CudaApi.cs:18-37;
 *      backs IDevice, src/MLFramework/HAL/IDevice.cs:6-42) ------------------------------------ */
pa_status pa_device_count(int32_t* count);
pa_status pa_device_open(int32_t ordinal, pa_device** out_device);
pa_status pa_device_close(pa_device* device);
pa_status pa_device_get_props(const pa_device* device, pa_device_props* props);
pa_status pa_device_synchronize(pa_device* device);

/* ---- memory (replaces CudaApi.CudaMalloc/CudaFree/CudaMemcpy/CudaMemset, CudaApi.cs:46-75;
 *      backs IMemoryAllocator/IMemoryBuffer, HAL/IMemoryAllocator.cs:6-43) ------------------- */
pa_status pa_alloc(pa_device* device, size_t bytes, void** dptr);
pa_status pa_free(pa_device* device, void* dptr);
/* Asynchronous on `stream` when it is non-null, otherwise synchronous. */
pa_status pa_memcpy(void* dst, const void* src, size_t bytes, int32_t kind, pa_stream* stream);
/* Refuses (PA_ERROR_INVALID_ARGUMENT) a stream that is capturing a graph: no memset is recorded. */
pa_status pa_memset(void* dst, int32_t value, size_t bytes, pa_stream* stream);

/* ---- streams and events (replace CudaApi.CudaStreamCreate/Destroy/Synchronize and
 *      CudaEventCreate/Destroy/Record/Query and CudaStreamWaitEvent, CudaApi.cs:81-128;
 *      back IStream/IEvent, HAL/IStream.cs:6-32, HAL/IEvent.cs:6-22) ---------------------- */
pa_status pa_stream_create(pa_device* device, pa_stream** out_stream);
/* Wraps an existing hipStream_t without taking ownership (interop with other HIP users). */
pa_status pa_stream_wrap(pa_device* device, void* hip_stream, pa_stream** out_stream);
pa_status pa_stream_native(const pa_stream* stream, void** hip_stream);
pa_status pa_stream_destroy(pa_stream* stream);
pa_status pa_stream_synchronize(pa_stream* stream);
pa_status pa_stream_wait_event(pa_stream* stream, pa_event* event);
pa_status pa_event_create(pa_device* device, pa_event** out_event);
pa_status pa_event_destroy(pa_event* event);
pa_status pa_event_record(pa_event* event, pa_stream* stream);
pa_status pa_event_query(pa_event* event, int32_t* completed);
pa_status pa_event_synchronize(pa_event* event);
pa_status pa_event_elapsed_ms(pa_event* start, pa_event* end, float* ms);

/* ---- graphs (replace the CUDA HAL's graph capture and replay: CUDAGraphCapture.BeginCapture /
 *      EndCapture, HAL/CUDA/Graphs/CUDAGraphCapture.cs:24-61, and CUDAGraph's instantiate /
 *      Execute / Validate / Dispose, HAL/CUDA/Graphs/CUDAGraph.cs:33-160) --------------------- */
/* Starts capturing the work enqueued on `stream` (thread-local capture mode, as the reference's
 * CaptureModeThreadLocal): launches made through this library on `stream` are recorded, not run,
 * until pa_graph_capture_end. `stream` must be a pa_stream (the null stream cannot capture). */
pa_status pa_graph_capture_begin(pa_stream* stream);
/* Ends the capture on `stream` and instantiates the graph; *out_graph replays the recorded work
 * with the same arguments (the same device buffers, whose contents the caller updates between
 * replays). On failure the capture is ended and no graph is returned. */
pa_status pa_graph_capture_end(pa_stream* stream, pa_graph** out_graph);
/* Replays the graph on `stream` (asynchronous). */
pa_status pa_graph_launch(pa_graph* graph, pa_stream* stream);
/* Number of nodes (kernel launches and copies) the graph holds. */
pa_status pa_graph_node_count(const pa_graph* graph, size_t* count);
pa_status pa_graph_destroy(pa_graph* graph);

/* ---- paged-attention operators (fill CudaPagedAttentionKernel.ComputePagedAttention,
 *      CudaPagedAttentionKernel.cs:24-36, behind IPagedAttentionKernel,
 *      Kernels/IPagedAttentionKernel.cs:11-34) ------------------------------------------------ */

/* Slot mapping for new tokens (device arrays). For sequence s, new token j (0 <= j < num_new[s])
 * sits at logical position p = start_pos[s] + j and gets
 *     slot_mapping[token_offset[s] + j] = block_tables[s][p / B] * B + p % B,
 * or -1 when that table entry is negative or p / B >= max_blocks_per_seq. This is the intended
 * BlockTable mapping (block k of a sequence holds tokens [k*B, (k+1)*B),
 * tests/MLFramework.Tests/Inference/PagedAttention/BlockTableTests.cs:115-134) combined with the
 * append position of PagedAttentionLayer.UpdateKVCache (Layers/PagedAttentionLayer.cs:256-272). */
pa_status pa_build_slot_mapping(pa_stream* stream, const pa_config* cfg,
                                const int32_t* block_tables, int32_t max_blocks_per_seq,
                                const int32_t* start_pos, const int32_t* num_new,
                                const int32_t* token_offset, int32_t num_seqs,
                                int32_t max_new_per_seq, int64_t* slot_mapping);

/* KV append / scatter (fills PagedAttentionLayer.UpdateKVCache/CopyTensorToBlock,
 * Layers/PagedAttentionLayer.cs:244-327, which is a no-op in the reference).
 * k_new, v_new: [n_tok][num_kv_heads][head_dim] of cfg->q_dtype (FP32 or BF16).
 * slot_mapping: [n_tok] int64, -1 = skip. Slots must be < num_blocks * block_size (others are
 *   skipped) and distinct: two new tokens of one call at one slot race.
 * FP32/BF16 caches store the converted value (fp32 -> bf16 truncates).
 * INT8 caches keep, per (block, KV head), an fp32 running absmax and scale = absmax / 127.
 *   Per call, the new tokens of one block raise absmax to max(absmax, max|x_new|); when it grows,
 *   every other slot of that block is requantised from q * old_scale with the new scale, then
 *   the new tokens are quantised with it. Quantisation is QuantizeSymmetric
 *   (src/MLFramework/Quantization/Operations/QuantizationOperations.cs:188-200).
 *   A block's new tokens may sit anywhere in the call's token list (split by other blocks'
 *   tokens or invalid slots); its segments (maximal runs of them) are applied in call order.
 *   The int8 append scans the slot list once per touched block (to find whether another token of
 *   the call lands in it), so its cost grows as blocks x n_tok: prompts above about 16k tokens are
 *   best appended in calls of at most that many tokens.
 *   k_scale/v_scale/k_absmax/v_absmax are required for INT8 and ignored otherwise. */
pa_status pa_kv_append(pa_stream* stream, const pa_config* cfg,
                       const void* k_new, const void* v_new,
                       const int64_t* slot_mapping, int32_t n_tok,
                       void* k_cache, void* v_cache,
                       float* k_scale, float* v_scale, float* k_absmax, float* v_absmax);

/* Bytes of device workspace pa_paged_decode / pa_paged_decode_append need for up to num_seqs
 * sequences of up to max_context_len tokens. bf16/int8 caches always need one (split partial
 * results and per-sequence offsets); fp32 caches only when a sequence spans several partitions
 * (else 0). The contents need no initialisation, and calls that share a workspace must not run
 * concurrently. */
pa_status pa_decode_workspace_size(const pa_config* cfg, int32_t num_seqs,
                                   int32_t max_context_len, size_t* bytes);

/* Ragged paged decode: one query token per sequence attends to its first context_lens[s] cached
 * tokens (the new token already appended), as DecodeOrchestrator.BatchDecode does with one
 * kernel call per sequence (Phases/DecodeOrchestrator.cs:64-109).
 *   out: [num_seqs][num_q_heads][head_dim] fp32
 *   q:   [num_seqs][num_q_heads][head_dim] of cfg->q_dtype
 *   block_tables: [num_seqs][max_blocks_per_seq] int32, context_lens: [num_seqs] int32
 *   max_context_len: host-side upper bound of context_lens (sizes the grid); tokens beyond it,
 *   or beyond max_blocks_per_seq * block_size, are not read. Tokens whose table entry lies
 *   outside [0, num_blocks) read as zero keys and values (never dereferenced).
 * Long sequences are split across workgroups (cfg->partition_size) and merged with a log-sum-exp
 * reduction through `workspace`. A sequence with context_len <= 0 produces zeros. */
pa_status pa_paged_decode(pa_stream* stream, const pa_config* cfg, float* out, const void* q,
                          const void* k_cache, const void* v_cache,
                          const float* k_scale, const float* v_scale,
                          const int32_t* block_tables, const int32_t* context_lens,
                          int32_t num_seqs, int32_t max_blocks_per_seq, int32_t max_context_len,
                          void* workspace, size_t workspace_bytes);

/* Fused decode layer-step: appends the token at position context_lens[s] - 1 of every sequence
 * (k_new/v_new [num_seqs][num_kv_heads][head_dim] of cfg->q_dtype) into the cache, then runs
 * pa_paged_decode. Cache bytes, int8 scales and absmax after the call are exactly those of
 * pa_kv_append with slot_mapping[s] = block_tables[s][(T-1)/16] * 16 + (T-1) % 16 followed by
 * pa_paged_decode; for bf16 caches both happen in one kernel (the rows stream their first T - 1
 * cached tokens and the new token joins each row's softmax from k_new / v_new, truncated to bf16 as
 * the cache stores it; it is written into the cache when every row has been read), for int8 caches the
 * quantising append is a launch of its own ahead of the decode, and for fp32 caches a plain
 * copy kernel.
 * Sequences that share the block a token is appended to (rows of one table): every slot may be
 * appended to once per call, and the cache ends up holding every token. Where the context of one
 * sequence covers another's new slot, int8 and fp32 caches give it the new token; bf16 caches give it
 * what the slot held before the call. (A call of more than 2047 sequences, 65535 for fp32 caches, is
 * worked off as several calls of that many at most, in order.)
 * No reference counterpart: the reference appends (PagedAttentionLayer.UpdateKVCache,
 * Layers/PagedAttentionLayer.cs:244-296) and decodes (DecodeOrchestrator.ComputeDecodeAttention,
 * Phases/DecodeOrchestrator.cs:64-80) in two steps; this is those two steps in one call.
 * Sequences with context_len <= 0 append nothing and produce zeros. */
pa_status pa_paged_decode_append(pa_stream* stream, const pa_config* cfg, float* out, const void* q,
                                 const void* k_new, const void* v_new, void* k_cache, void* v_cache,
                                 float* k_scale, float* v_scale, float* k_absmax, float* v_absmax,
                                 const int32_t* block_tables, const int32_t* context_lens,
                                 int32_t num_seqs, int32_t max_blocks_per_seq, int32_t max_context_len,
                                 void* workspace, size_t workspace_bytes);

/* Bytes of device scratch the library holds per device for pa_paged_decode_noalloc. */
#define PA_NOALLOC_SCRATCH_BYTES (32u << 20)

/* pa_paged_decode for callers that cannot allocate (code under HIP graph capture, tight serving
 * loops, harnesses that forbid allocation): the same arguments without a workspace; the split-K
 * partials go to a device array of PA_NOALLOC_SCRATCH_BYTES that the library holds on each device
 * (resolved at pa_device_open, or at this call's first use on a device) until the process ends.
 * The call allocates nothing. It returns PA_ERROR_WORKSPACE_TOO_SMALL, launching nothing, when
 * pa_decode_workspace_size for the same shape exceeds PA_NOALLOC_SCRATCH_BYTES. Every call on a
 * device shares that device's array: calls that overlap on one device (two streams, two threads)
 * race. No counterpart in the reference: it serves the callers that cannot allocate. */
pa_status pa_paged_decode_noalloc(pa_stream* stream, const pa_config* cfg, float* out, const void* q,
                                  const void* k_cache, const void* v_cache,
                                  const float* k_scale, const float* v_scale,
                                  const int32_t* block_tables, const int32_t* context_lens,
                                  int32_t num_seqs, int32_t max_blocks_per_seq, int32_t max_context_len);

/* ---- Shared-prefix decode ----
 * Sequences forked from one parent share the parent's first physical blocks (copy-on-write:
 * the same block ids lead their tables; BlockShareManager.ShareBlock,
 * Inference/PagedAttention/Sharing/BlockShareManager.cs:34-54, keeps the refcounts). The result
 * is that of pa_paged_decode; the shared blocks are read once per group of up to 16 / G
 * sequences (G = num_q_heads / num_kv_heads) instead of once per sequence. No reference
 * counterpart: the reference decodes every sequence over its whole table. */

/* Bytes of the device plan for num_seqs sequences. */
pa_status pa_prefix_plan_bytes(int32_t num_seqs, size_t* bytes);

/* Builds the plan into `plan` (device memory, plan_bytes >= pa_prefix_plan_bytes) from the host
 * array shared_with_prev[num_seqs]: shared_with_prev[s] = number of leading block-table entries
 * sequence s has in common with sequence s - 1 (entry 0 is ignored; 0 = no link). Linked runs
 * are cut into groups of at most 16 / G sequences sharing the run's minimum link; *num_groups
 * receives the group count to pass to pa_paged_decode_prefix. The plan depends only on the
 * grouping, not on the context lengths, so it is rebuilt only when sequences fork or leave.
 * Synchronises `stream` (host-to-device copy); refused while the stream captures a graph. */
pa_status pa_prefix_plan_build(pa_stream* stream, const pa_config* cfg, int32_t num_seqs,
                               const int32_t* shared_with_prev, void* plan, size_t plan_bytes,
                               int32_t* num_groups);

/* The same plan written to host memory (plan_host, plan_bytes >= pa_prefix_plan_bytes), for a
 * caller that uploads it itself: int32 records {first sequence, members, shared blocks} for each
 * of the *num_groups groups, then {group or -1, shared blocks or 0} for each sequence. No GPU
 * call. */
pa_status pa_prefix_plan_fill(const pa_config* cfg, int32_t num_seqs, const int32_t* shared_with_prev,
                              int32_t* plan_host, size_t plan_bytes, int32_t* num_groups);

/* Workspace of pa_paged_decode_prefix for up to num_seqs sequences of up to max_context_len. */
pa_status pa_prefix_workspace_size(const pa_config* cfg, int32_t num_seqs, int32_t max_context_len,
                                   size_t* bytes);

/* pa_paged_decode over the same arguments plus a plan from pa_prefix_plan_build (same num_seqs
 * and head ratio). Contract: within a group the shared block ids are identical in every table
 * and every member's context_len covers the shared blocks (>= 16 * shared); a plan that breaks
 * it gives wrong attention but never reads outside the arguments. BF16 or INT8 caches;
 * num_seqs + num_groups <= 2047; cfg->partition_size is not used (equal ranges per worker). */
pa_status pa_paged_decode_prefix(pa_stream* stream, const pa_config* cfg, float* out, const void* q,
                                 const void* k_cache, const void* v_cache,
                                 const float* k_scale, const float* v_scale,
                                 const int32_t* block_tables, const int32_t* context_lens,
                                 int32_t num_seqs, int32_t max_blocks_per_seq, int32_t max_context_len,
                                 const void* plan, int32_t num_groups,
                                 void* workspace, size_t workspace_bytes);

/* Chunked prefill: prefill sequence s has chunk_len[s] = q_start_loc[s+1] - q_start_loc[s] new
 * query tokens at absolute positions prefix_lens[s] + i; the chunk's K/V must already be appended,
 * so keys are positions [0, prefix_lens[s] + chunk_len[s]) read through block_tables[s].
 * Query i attends to keys 0 .. prefix_lens[s] + i (bottom-right aligned causal mask,
 * StandardPagedAttentionKernel.cs:219-255); see PA_FLAG_REFERENCE_LITERAL_MASK.
 *   out: [total_q][num_q_heads][head_dim] fp32, q: [total_q][num_q_heads][head_dim] of
 *   cfg->q_dtype (BF16 or FP32); caches of any kv_dtype. BF16 and INT8 caches take head_dim 64,
 *   128 or 256 and compute on bf16 / fp16 MFMA operands; FP32 caches (head_dim 32 .. 256) compute
 *   in fp32 throughout (fp32 MFMA operands and accumulation), which is what the dense
 *   ComputePagedAttention of IPagedAttentionKernel (Kernels/IPagedAttentionKernel.cs:13-28) needs
 *   for more than one query: one launch over the prompt instead of one decode row per query.
 *   max_chunk_len: host-side upper bound of the chunk lengths.
 * Range: every finite cache value is accepted. The P.V product runs on fp16 operands; int8
 * caches fold log2 of each block's V scale into the softmax exponent, so P times the scale stays
 * within fp16 for any scale; query tiles that read a V magnitude above 65504 (fp16's largest)
 * from a bf16 cache are detected and computed again in fp32 (a slower path, taken only for such
 * inputs). Queries and keys that are not finite give outputs that are not, at the usual speed. */
pa_status pa_chunked_prefill(pa_stream* stream, const pa_config* cfg, float* out, const void* q,
                             const int32_t* q_start_loc, const int32_t* prefix_lens,
                             const void* k_cache, const void* v_cache,
                             const float* k_scale, const float* v_scale,
                             const int32_t* block_tables, int32_t num_seqs,
                             int32_t max_blocks_per_seq, int32_t max_chunk_len);

/* ---- whole-block moves: copy-on-write and swap (the copy the reference leaves to a comment at
 *      beam divergence, BeamSearchBlockSharing.OnBeamDivergence, Sharing/BeamSearchBlockSharing.cs:
 *      69-79, over the refcounts of BlockShareManager.cs:34-105; and the block data moves of
 *      IPagedAttentionCache.GetBlockData / StoreBlockData, ContinuousBatching/KVCache/
 *      IPagedAttentionCache.cs:40-47, CacheBlockData.cs:7-12, which has no implementation) ----
 * Cache pointers (and the packed buffer) must be 16-byte aligned. int8 caches carry their
 * per-(block, KV head) k_scale, v_scale, k_absmax, v_absmax with the codes. */

/* Bytes of one packed block record: K of all KV heads (num_kv_heads * 16 * head_dim elements),
 * then V (same), then for int8 k_scale[Hkv], v_scale[Hkv], k_absmax[Hkv], v_absmax[Hkv] (fp32).
 * A multiple of 16. */
pa_status pa_block_bytes(const pa_config* cfg, size_t* bytes);
/* Copy-on-write: block_pairs [num_pairs][2] int32 (device) = (src, dst); every KV head's K and V
 * tiles (and int8 statistics) of block src are copied into block dst. Pairs with an id outside
 * [0, num_blocks) or src == dst are skipped. Within one call no block may be written twice, nor
 * be both a source and a destination. */
pa_status pa_copy_blocks(pa_stream* stream, const pa_config* cfg, void* k_cache, void* v_cache,
                         float* k_scale, float* v_scale, float* k_absmax, float* v_absmax,
                         const int32_t* block_pairs, int32_t num_pairs);
/* Swap-out: record i of `packed` ([n] records of pa_block_bytes, device memory; pa_memcpy moves
 * the records to and from host memory) receives block block_ids[i] (device int32), bit for bit.
 * Ids outside [0, num_blocks) are skipped (their records are not written). */
pa_status pa_gather_blocks(pa_stream* stream, const pa_config* cfg, const void* k_cache, const void* v_cache,
                           const float* k_scale, const float* v_scale, const float* k_absmax,
                           const float* v_absmax, const int32_t* block_ids, int32_t n, void* packed);
/* Swap-in: block block_ids[i] receives record i of `packed`, bit for bit (ids outside
 * [0, num_blocks) skipped; no block twice in one call). */
pa_status pa_scatter_blocks(pa_stream* stream, const pa_config* cfg, void* k_cache, void* v_cache,
                            float* k_scale, float* v_scale, float* k_absmax, float* v_absmax,
                            const int32_t* block_ids, int32_t n, const void* packed);
/* GetBlockData: tokens [0, tokens) (tokens <= 16) of block `block` as fp32, k_out / v_out
 * [tokens][num_kv_heads][head_dim] (device memory); bf16 widens exactly, int8 is code * scale.
 * k_scale/v_scale are needed for int8 only. */
pa_status pa_read_block_f32(pa_stream* stream, const pa_config* cfg, const void* k_cache, const void* v_cache,
                            const float* k_scale, const float* v_scale, int32_t block, int32_t tokens,
                            float* k_out, float* v_out);
/* StoreBlockData: tokens [0, tokens) of block `block` from fp32 k_in / v_in
 * [tokens][num_kv_heads][head_dim]; the cache bytes and int8 statistics afterwards are those of
 * pa_kv_append with fp32 input at slots block * 16 + t (row 0 is written, so an int8 block
 * starts afresh with scale = absmax of the new rows / 127). */
pa_status pa_write_block_f32(pa_stream* stream, const pa_config* cfg, void* k_cache, void* v_cache,
                             float* k_scale, float* v_scale, float* k_absmax, float* v_absmax,
                             int32_t block, int32_t tokens, const float* k_in, const float* v_in);

/* ---- attention over selected blocks, for long contexts ----
 * A decode step that reads a bounded number of blocks however long the context is: every block has
 * bounds of its keys, a query scores all blocks of its context from their bounds (a sixteenth of the
 * K and V bytes), and attends to the best of them. No reference counterpart: the reference decodes over
 * the whole context (DecodeOrchestrator.ComputeDecodeAttention, Phases/DecodeOrchestrator.cs:64-80).
 *
 * Query tokens: query r is one token with its own context length context_lens[r], of the sequence
 * query_seqs[r] (a row of the block tables, num_seqs of them); several queries may be of one sequence (drafted
 * tokens that are verified together). query_seqs null: query r belongs to sequence r, and num_queries
 * must be num_seqs. A query whose query_seqs entry is out of range has an empty context. Contexts are
 * read up to max_context_len and max_blocks_per_seq * 16 tokens. None of these calls allocates or
 * synchronises; all may be captured into a graph. Calls that share a workspace must not overlap. A call that needs a
 * launch of 2^32 threads or more is refused (PA_ERROR_UNSUPPORTED) before anything is launched. */

/* Bytes of the key bounds of the pool: [num_blocks][num_kv_heads][2][head_dim] elements of kv_dtype
 * (index 0: minimum, 1: maximum of each channel over the block's keys; int8 caches: of the codes, to
 * be read with the block's k_scale). */
pa_status pa_key_bounds_bytes(const pa_config* cfg, size_t* bytes);
/* Brings the bounds up to date after tokens were written into the cache (pa_kv_append and the calls
 * that append): for sequence s, every block that holds one of its tokens start_pos[s] ..
 * start_pos[s] + num_new[s] - 1 gets the bounds of the keys that it holds up to the last of them, read from
 * the cache. max_new_per_seq: host-side upper bound of num_new; it bounds the blocks that are looked at, the first
 * (max_new_per_seq + 14) / 16 + 1 (none for 0) that the new tokens lie in, and tokens in further ones are not.
 * Sequences with start_pos < 0 or num_new <= 0, table entries outside [0, num_blocks) and positions beyond
 * max_blocks_per_seq * 16 are skipped. A NaN key makes its channel's bounds NaN. Two sequences of one call
 * that name the same block must hold the same tokens in it. num_seqs at most 65535; k_cache and key_bounds
 * 16-byte aligned. */
pa_status pa_key_bounds_update(pa_stream* stream, const pa_config* cfg, const void* k_cache,
                               const int32_t* block_tables, int32_t max_blocks_per_seq,
                               const int32_t* start_pos, const int32_t* num_new, int32_t num_seqs,
                               int32_t max_new_per_seq, void* key_bounds);

/* Bytes of workspace of pa_select_blocks (8 per query, KV head and block, and for int8 caches 12 head_dim + 8
 * per query and KV head; 16-byte aligned). */
pa_status pa_select_workspace_size(const pa_config* cfg, int32_t num_queries, int32_t max_context_len, size_t* bytes);
/* The blocks each query attends to, for each KV head:
 *   selected: [num_queries][num_kv_heads][budget] int32, logical block indices in ascending order, -1
 *   behind the last. A context of at most `budget` blocks is selected whole. Otherwise the first
 *   sink_blocks and the last recent_blocks are, and the rest of the budget goes to the blocks with the
 *   largest scores
 *     sum_d (sum_g max(q_gd, 0)) hi_bd + (sum_g min(q_gd, 0)) lo_bd       (g: the heads of the group)
 *   (times k_scale for int8 caches), an upper bound of sum_g max_t q_g . k_t; equal scores go to the
 *   lowest index, a score that is NaN comes first (int8 caches: any score of a query that is not finite
 *   is). Scores are summed in 64 bits; for int8 caches from the sums over the group's heads rounded, each by at
 *   most 2^-46 of the largest of them, so scores closer than this makes may come in either order. Blocks whose
 *   table entry lies outside [0, num_blocks) score 0. The bounds of the sink and recent blocks do not matter
 *   (they need not be up to date while they are among the recent ones).
 *   q: [num_queries][num_q_heads][head_dim] of q_dtype; recent_blocks >= 1 (the block of the newest
 *   token), sink_blocks + recent_blocks <= budget, max_context_len <= 2097152; q and key_bounds 16-byte
 *   aligned. */
pa_status pa_select_blocks(pa_stream* stream, const pa_config* cfg, const void* q, const void* key_bounds,
                           const float* k_scale, const int32_t* block_tables, int32_t num_seqs,
                           int32_t max_blocks_per_seq, const int32_t* query_seqs, const int32_t* context_lens,
                           int32_t num_queries, int32_t max_context_len, int32_t sink_blocks,
                           int32_t recent_blocks, int32_t budget, int32_t* selected, void* workspace,
                           size_t workspace_bytes);

/* Bytes of workspace that pa_sparse_decode needs for up to num_queries query tokens and lists of up to budget
 * entries (partial results of rows that are split; at most a few MB; 4-byte aligned). A call whose own rows are not
 * split needs none. */
pa_status pa_sparse_workspace_size(const pa_config* cfg, int32_t num_queries, int32_t budget, size_t* bytes);
/* pa_paged_decode over the listed blocks only: query r's heads of KV head h attend to the tokens
 * (those before context_lens[r]) of the logical blocks selected[r][h][0 .. budget).
 *   out: [num_queries][num_q_heads][head_dim] fp32
 * Lists come from pa_select_blocks or from the caller: entries that are negative or at or past the end
 * of the context are skipped wherever they stand, in any order; a block listed twice counts twice.
 * Blocks whose table entry lies outside [0, num_blocks) read as zero keys and values. A query without
 * a listed token gives zeros. What unused slots of a block hold (NaN, Inf) does not matter. Queries
 * that are not finite, NaN keys, and keys that make a score +Inf give outputs that are not finite, and so do values that are
 * not, in their channel. A score of -Inf counts nothing beside finite ones (fp32 queries of bf16 caches, whose products
 * are formed in parts: it may be NaN); a query with no other gives NaN. Sums are in fp32; products are exact, for int8 caches
 * with queries that were rounded by at most 2^-30 of the largest value of their head (or 2^-126, where that is more) and
 * probabilities whose product with v_scale was rounded to fp32. num_q_heads / num_kv_heads: 1, 2, 4, 8 or
 * 16. q and caches 16-byte aligned. */
pa_status pa_sparse_decode(pa_stream* stream, const pa_config* cfg, float* out, const void* q,
                           const void* k_cache, const void* v_cache, const float* k_scale,
                           const float* v_scale, const int32_t* block_tables, int32_t num_seqs,
                           int32_t max_blocks_per_seq, const int32_t* query_seqs, const int32_t* context_lens,
                           int32_t num_queries, int32_t max_context_len, const int32_t* selected,
                           int32_t budget, void* workspace, size_t workspace_bytes);

/* ---- the books of the pool on the device ----
 * Which blocks a sequence holds and how many hold a block, changed by kernels in stream order, so that a
 * step that forks, frees or extends sequences may be captured into a graph; whether its reservation succeeded
 * is for the step itself or the host to ask before anything is appended (pa_pages_reserve)
 * (the reference keeps these books on the host: BlockShareManager.cs:34-105, KVCacheBlockManager.cs:
 * 70-174). The caller owns the arrays:
 *   refcounts    [num_blocks] int32: rows (and other owners, such as a prefix cache) that hold the block;
 *                0: free
 *   block tables [rows][max_blocks_per_seq] int32: a row holds its entries in [0, num_blocks); every other
 *                entry must be negative (-1), those behind its last block too
 * Results depend on the books alone, never on timing. Calls on one set of books must not overlap. */

/* New rows from old ones: out row i is a copy of in row src[i] (table and length), or empty (length 0,
 * every entry -1) when src[i] is outside [0, num_in). Every in row gives up its blocks and every out
 * row takes hold of its own, so this forks (a row named twice), frees (a row not named) and reorders
 * sequences or beams in one call. refcounts change in place; the out arrays must not overlap the in
 * arrays. Blocks whose count falls to 0 are free. num_in + num_out below 2^24. */
pa_status pa_pages_fork(pa_stream* stream, const pa_config* cfg, const int32_t* tables_in, const int32_t* lens_in,
                        int32_t num_in, const int32_t* src, int32_t* tables_out, int32_t* lens_out,
                        int32_t num_out, int32_t max_blocks_per_seq, int32_t* refcounts);

/* Bytes of workspace of pa_pages_reserve and pa_pages_compact (4-byte aligned). */
pa_status pa_pages_workspace_size(const pa_config* cfg, int32_t num_rows, int32_t max_blocks_per_seq, size_t* bytes);

/* Makes room for num_new[i] more tokens of row i at positions lens[i] .. (lens itself is the caller's to
 * advance): every block of theirs that the row does not hold is taken from the free ones, and every one
 * that others hold too is replaced by a free one (copy on write). Rows are worked off in order, the
 * lowest free block first; when every holder of a shared block asks for it in this call, the last of them
 * keeps it. copy_pairs [num_rows][2]: (old, new) where the replaced block holds tokens of the row, else
 * (-1, -1); copy them with pa_copy_pages (or pa_copy_blocks) before the new tokens are written.
 * status [2] (device): the blocks taken, and 0; or, when there are too few free blocks, 0 and how many are
 * missing, with nothing else changed. max_new_per_row: host-side upper bound of num_new; of
 * the blocks that a row's new tokens lie in the first (max_new_per_row + 14) / 16 + 1 are looked at (none for 0).
 * Positions beyond max_blocks_per_seq * 16 get no block; rows with num_new <= 0 or a negative length ask for none.
 * Then append (pa_build_slot_mapping, pa_kv_append), bring the key bounds up to date and advance lens; but not when blocks are missing (status[1] != 0): the tables are then as they were, so a row's tokens
 * would go into blocks that others still hold, or nowhere. Nothing behind this call looks at status by itself. Either the
 * host reads it before the append is enqueued, or knows that there is room before the call (it takes at most
 * num_rows times the blocks that max_new_per_row tokens can touch), or the step makes the append harmless on the device: start
 * positions of INT32_MIN for pa_build_slot_mapping and pa_key_bounds_update where status[1] != 0 (their slots are
 * -1, which every append by slots skips; no bounds are touched; pa_paged_decode_append goes by the context length: 0), and
 * lens advanced by nothing. */
pa_status pa_pages_reserve(pa_stream* stream, const pa_config* cfg, int32_t* tables, const int32_t* lens,
                           const int32_t* num_new, int32_t num_rows, int32_t max_blocks_per_seq,
                           int32_t max_new_per_row, int32_t* refcounts, int32_t* copy_pairs, int32_t* status,
                           void* workspace, size_t workspace_bytes);

/* Moves the highest live blocks into the lowest free ones while that lowers them, at most max_moves:
 * pairs [max_moves][2] gets (from, to), (-1, -1) behind the last; refcounts move along and the tables'
 * entries are renamed (other owners rename theirs by the pairs). status [2] (device): the moves, and the
 * number of blocks from 0 on that contain every live one afterwards (the pool above it may be given
 * back). Copy the data of every layer with pa_copy_pages(pairs, max_moves, status) before the blocks are
 * read or reserved. */
pa_status pa_pages_compact(pa_stream* stream, const pa_config* cfg, int32_t* tables, int32_t num_rows,
                           int32_t max_blocks_per_seq, int32_t* refcounts, int32_t max_moves, int32_t* pairs,
                           int32_t* status, void* workspace, size_t workspace_bytes);

/* pa_copy_blocks for pairs whose number is on the device, with the key bounds: the first
 * min(*num_pairs, max_pairs) pairs (num_pairs null: max_pairs) are copied, K, V, int8 statistics and, unless
 * null, key_bounds. Pairs with an id outside [0, num_blocks) or src == dst are skipped. Within one call no
 * block may be written twice, nor be both a source and a destination. */
pa_status pa_copy_pages(pa_stream* stream, const pa_config* cfg, void* k_cache, void* v_cache,
                        float* k_scale, float* v_scale, float* k_absmax, float* v_absmax, void* key_bounds,
                        const int32_t* pairs, int32_t max_pairs, const int32_t* num_pairs);

/* ---- caches of bounded size: a sliding window, first tokens that stay visible, eviction by weight ----
 * A model with a sliding window sees the last `window` tokens and the first sink_tokens of a sequence; its blocks
 * between these may go. A model without one can be served from a bounded cache all the same: what weight attention gives each
 * block is added up, and the blocks that got the least leave their rows. No reference counterpart: the reference attends
 * to the whole context (DecodeOrchestrator.ComputeDecodeAttention, Phases/DecodeOrchestrator.cs:64-80) and frees a
 * sequence's blocks only with the sequence (KVCacheBlockManager.cs:70-174).
 *
 * Visible tokens: the query at position p sees the tokens t <= p with t > p - window or t < sink_tokens (window 0: every t <= p).
 * Positions are places in the row's table: when blocks between the sinks and the window have left it, the same
 * sink_tokens and window still name the same tokens. (Where the model rotates keys by their position, the caller rotates them
 * before the append, by the position in the text, and they keep it.)
 * Masses: block_mass [rows][max_blocks_per_seq] fp32, one value for each entry of the block tables, the caller's to set to 0 when a
 * row begins; a forked row's masses are copied with its table by the caller.
 * Contexts are read up to max_context_len and max_blocks_per_seq * 16 tokens; blocks whose table entry lies outside
 * [0, num_blocks) read as zero keys and values. What tokens hold that a query does not see (unused slots of a block, expired
 * tokens; NaN, Inf) does not matter to it. Queries that are not finite, NaN keys, and keys that make a score +Inf give outputs (and
 * masses) that are not finite, and so do values that are not, in their channel. A score of -Inf counts nothing beside
 * finite ones (fp32 queries of bf16 caches and fp32 caches, whose products are formed in parts: it may be NaN); a query with no other
 * gives NaN. int8 caches: scales must be finite. Values are added up before the sum is divided by the softmax's, so beyond 2^116 /
 * (tokens seen) they may overflow. None of these calls allocates or synchronises; all may be captured
 * into a graph. Calls that share a workspace or masses must not overlap. */

/* Bytes of workspace of pa_window_decode for up to num_seqs sequences of up to max_context_len tokens (8-byte aligned); with_mass
 * non-zero: for calls that keep masses. */
pa_status pa_window_decode_workspace_size(const pa_config* cfg, int32_t num_seqs, int32_t max_context_len,
                                          int32_t sink_tokens, int32_t window, int32_t with_mass, size_t* bytes);
/* pa_paged_decode over the visible tokens: one query token per sequence, at the last position of its context (already
 * appended). A context longer than max_context_len or max_blocks_per_seq * 16 counts as one of that length, its window too, as in
 * pa_paged_decode (a chunk's queries keep their positions, see pa_window_prefill). Only blocks that hold a visible token
 * are read, their table entries too.
 *   out: [num_seqs][num_q_heads][head_dim] fp32, q: [num_seqs][num_q_heads][head_dim] of q_dtype
 * block_mass null, or [num_seqs][max_blocks_per_seq]: every visible block's entry grows by the softmax weights of its
 * visible tokens, summed over the query heads in a fixed order (num_q_heads in all for each sequence).
 * A sequence with context_lens[s] <= 0 gives zeros. Any kv_dtype and head_dim; num_q_heads / num_kv_heads: 1, 2, 4, 8 or
 * 16. Sums are in fp32; products are exact, for int8 caches as pa_sparse_decode forms them. q and caches 16-byte
 * aligned. (A call of more than 2047 sequences is worked off as several of that many at most, in order.) */
pa_status pa_window_decode(pa_stream* stream, const pa_config* cfg, float* out, const void* q, const void* k_cache,
                           const void* v_cache, const float* k_scale, const float* v_scale,
                           const int32_t* block_tables, const int32_t* context_lens, int32_t num_seqs,
                           int32_t max_blocks_per_seq, int32_t max_context_len, int32_t sink_tokens, int32_t window,
                           float* block_mass, void* workspace, size_t workspace_bytes);

/* Bytes of workspace of pa_window_prefill for up to num_seqs chunks of up to max_chunk_len tokens in contexts of up to
 * max_context_len (16-byte aligned). A call whose keys are not cut needs none. */
pa_status pa_window_prefill_workspace_size(const pa_config* cfg, int32_t num_seqs, int32_t max_chunk_len,
                                           int32_t max_context_len, int32_t sink_tokens, int32_t window, size_t* bytes);
/* pa_chunked_prefill over the visible tokens: chunk s has q_start_loc[s + 1] - q_start_loc[s] query tokens at positions
 * prefix_lens[s] + i, its keys and values already appended; from single tokens and a few drafted ones to whole prompts.
 *   out: [total_q][num_q_heads][head_dim] fp32, q: [total_q][num_q_heads][head_dim] of q_dtype
 *   lse: null, or [total_q][num_q_heads] fp32: ln of the sum of exp(scale q.k) over the visible tokens
 *   max_chunk_len, max_context_len: host-side upper bounds of the chunks and of prefix + chunk; query tokens beyond
 *   the former are not computed.
 * A query that sees no token (its window lies past the table or max_context_len) gives zeros, and -Inf in lse. Any
 * kv_dtype, head_dim and ratio of heads; num_seqs * num_kv_heads at most 65535. Sums are in fp32. Products are exact,
 * but for at most 2^-22 of each, of either sign, where both operands are fp32 (queries, probabilities, caches). out, q
 * and caches 16-byte aligned. cfg->flags (masks) are not read. */
pa_status pa_window_prefill(pa_stream* stream, const pa_config* cfg, float* out, const void* q,
                            const int32_t* q_start_loc, const int32_t* prefix_lens, const void* k_cache,
                            const void* v_cache, const float* k_scale, const float* v_scale,
                            const int32_t* block_tables, int32_t num_seqs, int32_t max_blocks_per_seq,
                            int32_t max_chunk_len, int32_t max_context_len, int32_t sink_tokens, int32_t window,
                            float* lse, void* workspace, size_t workspace_bytes);

/* The masses of a prompt, before its first eviction: over the last `last_queries` tokens of every chunk (all of a shorter one)
 * and their heads,
 *   block_mass[s][b] += sum of exp(scale q.k - lse) over the visible tokens of block b, in a fixed order.
 * q, q_start_loc, prefix_lens, max_context_len, sink_tokens and window are those of the pa_window_prefill call that left lse,
 * and no chunk may be longer than that call's max_chunk_len (the lse of tokens beyond it was never written, and weights by
 * it would stay in the masses). Rows of q and lse other than the last queries' are not read. Keys alone are read,
 * products are that call's. num_seqs at most 65535, num_q_heads / num_kv_heads at most 2^20, last_queries * num_q_heads
 * below 2^30, and where there is no window max_context_len up to 5 * 10^8 (some types take more); q and k_cache 16-byte
 * aligned. */
pa_status pa_prefill_mass(pa_stream* stream, const pa_config* cfg, const void* q, const float* lse,
                          const int32_t* q_start_loc, const int32_t* prefix_lens, const void* k_cache,
                          const float* k_scale, const int32_t* block_tables, int32_t num_seqs,
                          int32_t max_blocks_per_seq, int32_t max_context_len, int32_t last_queries,
                          int32_t sink_tokens, int32_t window, float* block_mass);

/* Rows over their budget give up blocks. A row of n = ceil(lens[i] / 16) > budget blocks keeps the first sink_blocks, the last
 * recent_blocks and, of the others, the budget - sink_blocks - recent_blocks of the largest mass (equal masses:
 * the lowest index; NaN counts as the largest); block_mass null: the last ones. What stays moves down in order, masses along;
 * entries behind the row's blocks (reserved ahead) move with them, -1 (and mass 0) follows. lens[i] falls by 16 for each
 * block that left, and its count in refcounts (the page books, see pa_pages_fork) by one
 * for every row that gave it up; at 0 it is free. Entries outside [0, num_blocks) leave like others, without a count.
 *   evicted: null, or [num_rows] int32: the blocks that each row gave up (0: the row is as it was)
 * recent_blocks >= 1 (the newest token's block may be unfinished), sink_blocks + recent_blocks <= budget. The results depend on
 * the arrays alone. No key or value moves: int8 scales and key bounds stay with their blocks. */
pa_status pa_evict_blocks(pa_stream* stream, const pa_config* cfg, int32_t* block_tables, int32_t* lens,
                          float* block_mass, int32_t num_rows, int32_t max_blocks_per_seq, int32_t sink_blocks,
                          int32_t recent_blocks, int32_t budget, int32_t* refcounts, int32_t* evicted);

/* ---- the projections either side of attention (PagedAttentionLayer.ComputeAttention's
 *      _queryProj/_keyProj/_valueProj.Forward + UpdateKVCache and _outputProj.Forward,
 *      Layers/PagedAttentionLayer.cs:112-142; Linear.Forward y = x W^T without bias,
 *      Modules/Linear.cs:81-110). bf16 weights and activations (cfg->q_dtype must be BF16), fp32
 *      accumulation. Batches of at most 64 tokens (decode) run on a weight-streaming MFMA kernel
 *      with the k range split over workgroups (partials added in a fixed order, so results are
 *      deterministic); larger batches, operands not 16-byte aligned, a reduced dimension (hidden
 *      for Q/K/V, Hq * head_dim for O) not a multiple of 64, and output column counts not a
 *      multiple of 16 run on rocBLAS. The first rocBLAS call on a device creates
 *      its handle, so make one call of that shape before capturing these into a graph. ---- */

/* Bytes of workspace pa_qkv_project_append needs for n_tok tokens: for n_tok <= 64, the split
 * partials [splits][n_tok][(num_q_heads + 2 num_kv_heads) head_dim] fp32 (splits <= 8); above,
 * the fp32 GEMM output [n_tok][(num_q_heads + 2 num_kv_heads) head_dim]. Either way the GEMM
 * output y sits at the start of the workspace after the call. */
pa_status pa_qkv_workspace_size(const pa_config* cfg, int32_t n_tok, size_t* bytes);
/* x [n_tok][hidden] bf16; w_qkv [(Hq + 2 Hkv) * head_dim][hidden] bf16, the rows of Wq, then Wk,
 * then Wv. y = x w_qkv^T (fp32); q_out [n_tok][Hq][head_dim] (bf16) = y's Q columns truncated; the
 * K and V columns are appended into the cache at slot_mapping exactly as pa_kv_append does with
 * fp32 input (the int8 statistics included). */
pa_status pa_qkv_project_append(pa_stream* stream, const pa_config* cfg, const void* x, const void* w_qkv,
                                int32_t hidden, int32_t n_tok, const int64_t* slot_mapping, void* q_out,
                                void* k_cache, void* v_cache, float* k_scale, float* v_scale,
                                float* k_absmax, float* v_absmax, void* workspace, size_t workspace_bytes);
/* Bytes of workspace pa_o_project needs for n_tok tokens and `hidden` output columns: for
 * n_tok <= 64 the larger of the split partials [splits - 1][n_tok][hidden] fp32 and a bf16 copy
 * of the attention output; above, the bf16 copy. */
pa_status pa_o_workspace_size(const pa_config* cfg, int32_t hidden, int32_t n_tok, size_t* bytes);
/* attn [n_tok][Hq][head_dim] fp32 (the decode / prefill output), truncated to bf16;
 * w_o [hidden][Hq * head_dim] bf16; y [n_tok][hidden] fp32 = attn_bf16 w_o^T. */
pa_status pa_o_project(pa_stream* stream, const pa_config* cfg, const float* attn, const void* w_o,
                       int32_t hidden, int32_t n_tok, float* y, void* workspace, size_t workspace_bytes);

#ifdef __cplusplus
}
#endif

#endif /* PAGED_ATTN_H */
