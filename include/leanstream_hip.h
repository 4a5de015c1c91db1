/* C ABI of the MI355X streaming sparse INT4 MLP library (libleanstream_hip.so).
 *
 * Plain pointers and sizes only. Every entry point names the LeanStream interface it
 * replaces; a binding written against those interfaces maps one-to-one:
 *
 *   ls_hip_create / _create_table / _destroy    <- ls_triton_create / _create_table / _destroy
 *                                                  (include/leanstream/triton_cuda.h:50-52)
 *   ls_hip_bind                                 <- ls_triton_bind (triton_cuda.h:54-55); HIP kernels are
 *                                                  compiled in, so bind takes buffers + geometry
 *   ls_hip_enqueue                              <- ls_triton_enqueue (triton_cuda.h:56) merged with
 *                                                  ComputeBackend::enqueue (include/leanstream/runtime.h:12-13)
 *   ls_hip_complete                             <- ComputeBackend::complete (runtime.h:14)
 *   ls_hip_compute_backend                      <- TritonBackend::view (backends/triton/enqueue.cpp:46)
 *   ls_hip_select / ls_quantize_io_load         <- KernelSelector::select / quantize_io_load
 *                                                  (include/leanstream/kernel_selector.h:26,33)
 *   ls_hip_host_alloc / _free / _release_u32 /
 *   ls_hip_acquire_all                          <- tm_alloc / tm_free / tm_release / tm_acquire_all
 *                                                  (backends/triton/mapped.cpp:9-30)
 *   ls_queue_*                                  <- ExecutionQueue (include/leanstream/execution_queue.h:19-34)
 *   ls_rank_groups                              <- top-k ranking of ls_predict (predictor/predictor_cpu.cpp:192-201)
 *   ls_stream_create / _destroy / _run / _queue <- the end-to-end decode loop over Runtime / LayerStep
 *                                                  (examples/end_to_end/main.cu:58-72) with the I/O
 *                                                  transport replaced: HostStagingIO (pinned host store ->
 *                                                  hipMemcpyAsync) instead of the O_DIRECT engine behind
 *                                                  WeightManager (src/io/stream_io.h:45-65)
 *
 * Return values: 0 on success, a positive errno (EINVAL, ENOTSUP, ...) for rejected
 * arguments, or a positive hipError_t for a failed launch.
 */
#ifndef LEANSTREAM_HIP_H
#define LEANSTREAM_HIP_H
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Five 32-bit words, identical to leanstream::runtime::ExecDesc. */
typedef struct ls_exec_desc {
    uint32_t logical_group, physical_group, source_slot, dest_slot, source_kind;
} ls_exec_desc;

/* Identical to leanstream::runtime::DeviceExecQueue. */
typedef struct ls_device_queue {
    ls_exec_desc* descriptors;
    uint32_t* ready_indices;
    void* control; /* 128-byte QueueControl in host-coherent memory */
    uint32_t capacity;
} ls_device_queue;

/* Identical to leanstream::runtime::HipLayerBuffers. */
typedef struct ls_hip_layer_buffers {
    uint32_t width, group_size, batch, slot_capacity;
    uint32_t cache_groups, staging_groups, physical_groups, queue_capacity;
    const void* cache;
    const void* staging;
    const void* scales;
    void* hidden;
    void* partial;            /* reserved, unused (the reduction accumulates in backend-owned fixed point) */
    void* y32;
    uint32_t* executions;
    uint64_t* first_compute;
    uint32_t* claim_log;      /* optional: 4 words per range taken, queue_capacity ranges */
    uint64_t* stamps;         /* optional: [12 * compute units][32] (leanstream/hip_backend.h) */
} ls_hip_layer_buffers;

/* Consumer modes (leanstream::runtime::ConsumerMode). */
enum { LS_MODE_BATCH_COMPAT = 0, LS_MODE_PROGRESSIVE = 1, LS_MODE_AUTO = 2 };
/* Device status bits returned by ls_hip_status. */
enum { LS_STATUS_TIMEOUT = 1, LS_STATUS_QUEUE_ERROR = 2, LS_STATUS_BAD_DESCRIPTOR = 4, LS_STATUS_RANGE = 8,
       LS_STATUS_QUEUE_UNCONSUMED = 16 /* dense (batch 5..32) launch whose layer published queue entries */ };

/* ---- backend ---- */
void* ls_hip_create(void);
void* ls_hip_create_table(const uint8_t* entries, uint32_t layers, uint32_t buckets);
void ls_hip_destroy(void* backend);
int ls_hip_bind(void* backend, const ls_hip_layer_buffers* buffers);
int ls_hip_enqueue(void* backend, uint32_t layer, uint32_t bucket, uint32_t epoch, const void* input, void* output,
                   void* stream, const ls_exec_desc* core, uint32_t core_count, const ls_device_queue* queue,
                   uint32_t mode);
int ls_hip_complete(void* backend, uint32_t layer);
/* Writes a leanstream::runtime::ComputeBackend (context + 5 function pointers). */
int ls_hip_compute_backend(void* backend, void* out_compute_backend, uint64_t out_bytes);
uint32_t ls_hip_status(void* backend);
void ls_hip_clear_status(void* backend);
void ls_hip_set_spin_limit(void* backend, uint64_t ticks_100mhz);
/* TritonBackend::arm_context / arm_final_prediction / b_done (include/leanstream/triton_cuda.h:30-33):
 * every later enqueue calls arm(context) and records b_done (a hipEvent_t, may be NULL) at the
 * consumer -> reduction boundary -- between the split sequence's stage B and reduction launches,
 * after a fused or dense launch. A nonzero arm code is returned by the enqueue, whose launch is
 * nevertheless whole (the reduction runs, the completion word comes). NULL arm and b_done
 * remove the hook. EINVAL for a NULL backend. */
int ls_hip_set_stage_hook(void* backend, int (*arm)(void*), void* context, void* b_done);
/* Identical to leanstream::runtime::HipEpilogue (include/leanstream/hip_backend.h): the layer
 * epilogue run after every later enqueue on the same stream -- hidden = fp16(residual + y)
 * (the Triton reduction's PUBLISH path, backends/triton/reduction.py:17-28), optionally
 * RMSNorm(hidden) * norm_weight (examples/ministral/native/predictor_shared_input.cu:16-41),
 * then hidden_flag / norm_flag receive the enqueue's epoch (system-scope release) and
 * bell += 1. A fused launch (the default entry point, batch 1..4) runs it in its own last
 * workgroup once every worker is out, and its completion word follows the epilogue; the split
 * entry point and the dense path (batch 5..32) launch it after the layer, where the
 * completion word does not cover it. A failed layer -- its launch raised a status bit (sticky
 * until ls_hip_clear_status) or its queue's error word is set -- gets neither flag nor the
 * bell, and its rows are not the layer's output. Readers of hidden wait on the flags. NULL removes
 * it. EINVAL for an unbound backend or an inconsistent block. */
typedef struct ls_hip_epilogue {
    const void* residual;
    void* hidden;
    uint32_t* hidden_flag;
    const void* norm_weight;
    void* norm_output;
    uint32_t* norm_flag;
    uint32_t* bell;
    float norm_eps;
} ls_hip_epilogue;
int ls_hip_set_epilogue(void* backend, const ls_hip_epilogue* epilogue);
/* ---- layer chains ----
 * Identical to leanstream::runtime::HipChainLayer. A sequence of layers computed by one persistent
 * launch (batch 1, 64-neuron groups, width 1024 or 4096). Layer i's hidden state
 * fp16(residual_i + y_i) -- the epilogue's publication (backends/triton/reduction.py:17-22) -- is
 * handed over inside the grid: it is layer i + 1's residual, and its input as it is or, with
 * norm_weight, as RMSNorm(hidden) * norm_weight (examples/ministral/native/predictor_shared_input.cu:
 * 16-41), so later layers' weights stream while earlier layers finish. No LeanStream C++
 * counterpart: LeanStream submits future layers ahead and gates each on an input-ready epoch
 * (docs/architecture.md:9, backends/triton/core.py:20-28). The first layer's input (and optional
 * residual) is read as the stream finds it; every later layer's input and residual must be NULL,
 * and the first layer's norm_weight NULL. Layer i gets sequence ls_hip_last_seq() - count + 1 + i;
 * the completion word (ls_hip_done_seq) takes each layer's sequence once every wave is out of it,
 * and then hidden_flag receives the epoch (system release) and bell += 1, unless a status bit is
 * set. ls_hip_complete covers the whole chain. Returns EINVAL for an invalid block, ENOTSUP for a
 * geometry without chain kernels, EBUSY while more than 1024 layers are in flight. */
typedef struct ls_hip_chain_layer {
    const ls_exec_desc* core;
    const void* cache;
    const void* staging;
    const void* scales;
    const void* input;
    const void* residual;
    const void* norm_weight;
    void* output;
    float* output32;
    void* hidden;
    uint32_t* hidden_flag;
    uint32_t* bell;
    uint32_t core_count, cache_groups, staging_groups, physical_groups, epoch;
    float norm_eps;
} ls_hip_chain_layer;
int ls_hip_enqueue_chain(void* backend, const ls_hip_chain_layer* layers, uint32_t count, void* stream);
/* Diagnostics: per-layer phase stamps of chains of at most `layers` layers,
 * [layers][(ls_hip_chain_workers() + 1) * 4][32] u64 (100 MHz clock); NULL removes them. */
int ls_hip_set_chain_stamps(void* backend, uint64_t* stamps, uint32_t layers);
uint32_t ls_hip_chain_workers(void* backend);
uint32_t ls_hip_last_seq(void* backend);
uint32_t ls_hip_done_seq(void* backend);
/* Down-projection items (256-column tiles) per unit: d / 256. */
uint32_t ls_hip_slices(void* backend);
/* Overrides the selected candidate's persistent worker count (0 = the candidate's own
 * value). No reference counterpart: a tuning knob of the persistent launch. */
void ls_hip_set_workers(void* backend, uint32_t workers);
uint32_t ls_hip_select(void* backend, uint32_t layer, uint32_t bucket);
int ls_hip_last_candidate(void* backend);
uint32_t ls_hip_max_workers(void* backend);
uint32_t ls_quantize_io_load(uint32_t remaining, uint32_t total, uint32_t buckets);

/* ---- allocation-free resident layer ----
 * No counterpart in LeanStream. For callers that cannot allocate device memory (code under
 * HIP graph capture, tight serving loops, harnesses that forbid hipMalloc): one layer whose
 * groups are all resident (the core descriptors; no ready queue), computed as ls_hip_enqueue
 * computes it (fused persistent kernel, same bits) with its synchronisation words,
 * accumulators and h rows in a per-GPU device array of the library (about 1.9 MB, held until
 * the process ends) instead of the buffers ls_hip_bind allocates. Calls no hipMalloc/hipFree.
 * Stream-ordered: output (fp16 [batch][width]), output32 (optional fp32) and status (optional
 * device-visible word, cleared by the call, LS_STATUS_* bits) are valid once the stream
 * reaches the end of the call. Calls that overlap on one GPU race on the shared array.
 * Limits: width <= 8192 (a multiple of 256 with kernels built for it), batch 1..4 (ENOTSUP
 * above), core_count <= 1024 and core_count * group_size <= 32768 (ENOSPC beyond). */
int ls_hip_core_layer_noalloc(uint32_t width, uint32_t group_size, uint32_t batch, const void* cache,
                              uint32_t cache_groups, const void* scales, uint32_t scale_groups, const ls_exec_desc* core,
                              uint32_t core_count, const void* input, void* output, float* output32, uint32_t* status,
                              void* stream);

/* ---- coherent host memory (fine-grained, GPU-visible at system scope) ---- */
void* ls_hip_host_alloc(uint64_t bytes);
void ls_hip_host_free(void* ptr);
void ls_hip_release_u32(void* base, int64_t index, uint32_t value);
int ls_hip_acquire_all(const void* base, int32_t count, uint32_t value, int32_t timeout_ms);

/* ---- ready-queue producer (serialized; see ExecutionQueue) ---- */
void* ls_queue_create(const ls_device_queue* view);
void ls_queue_destroy(void* queue);
void ls_queue_reset(void* queue, uint32_t epoch);
void ls_queue_prepare(void* queue, uint32_t total);
void ls_queue_append_unpublished(void* queue, uint32_t index);
void ls_queue_activate(void* queue);
void ls_queue_seal(void* queue, uint32_t total);
void ls_queue_publish_all(void* queue);
void ls_queue_publish(void* queue, uint32_t index);
void ls_queue_fail(void* queue, uint32_t error);
/* Background publisher: publishes order[i] at time offset_ns[i] after start (busy
 * wait on the host clock). If fail_after < count, publishes fail_after entries and
 * then fails the queue with fail_code. Returns a handle for ls_publisher_join. */
void* ls_publisher_start(void* queue, const uint32_t* order, const uint64_t* offset_ns, uint32_t count,
                         uint32_t fail_after, uint32_t fail_code);
int ls_publisher_join(void* publisher);

/* ---- group selection ---- */
/* Top-k logical ids by (score descending, id ascending); -1 on non-finite scores. */
int ls_rank_groups(const float* scores, uint32_t count, uint32_t k, int32_t* out);

/* ---- streaming decode over host-staged layers ---- */
/* Copy engines: SDMA engines driven directly (no HIP stream), or hipMemcpyAsync streams. */
enum { LS_COPY_SDMA = 0, LS_COPY_HIP = 1 };
/* Identical to leanstream::runtime::GroupLayout (file_offset = offset in the host store). */
typedef struct ls_group_layout {
    uint32_t logical_group, physical_group;
    uint64_t file_offset;
    uint32_t bytes, reserved;
} ls_group_layout;

typedef struct ls_stream_setup {
    void* backend;            /* ls_hip_create handle, bound with staging = `staging` */
    const void* host_store;   /* pinned host memory holding every layer's packed groups */
    uint64_t host_bytes;
    void* staging;            /* device arena: logical group g at g * staging_stride */
    uint64_t staging_bytes;
    uint64_t group_bytes, staging_stride;
    uint32_t group_count;     /* logical groups per layer */
    uint32_t layers;          /* Runtime layer contexts */
    uint32_t qd;              /* copies in flight, 1..32 */
    uint32_t copy_engine;     /* LS_COPY_SDMA or LS_COPY_HIP */
    uint32_t copy_queues;     /* SDMA engines (1..16) or hipMemcpyAsync streams (1..2), round robin */
    uint32_t copy_chunk;      /* SDMA: bytes per copy piece (0 = one copy per group) */
    uint32_t mode;            /* LS_MODE_* */
    int32_t device;
} ls_stream_setup;

typedef struct ls_stream_layer {
    const ls_group_layout* layout; /* [group_count] */
    const int32_t* rank;           /* update_prediction priority order */
    uint32_t rank_count;
    const int32_t* final_ids;      /* finalize order */
    uint32_t final_count;
    const uint64_t* arrival_ns;    /* optional [group_count]: earliest copy start after begin */
    const void* input;             /* device fp16 x */
    void* output;                  /* device fp16 y */
} ls_stream_layer;

/* NULL on invalid setup or allocation failure. */
void* ls_stream_create(const ls_stream_setup* setup);
void ls_stream_destroy(void* decoder);
/* The decoder's ready queue (descriptors, publication order, control words). */
int ls_stream_queue(void* decoder, ls_device_queue* out);
/* Runs `count` layers in order on `stream` (Runtime layer id = (first_layer + i) % layers).
 * times: optional [count][7] ns after the call's start: begin, after begin_layer, after
 * update_prediction, after enqueue_compute, after finalize, completion observed (left 0
 * when the launch's completion was not observed), after commit. stamps: optional [count][group_count][3] ns after each layer's begin: admission,
 * copy submission, copy completion. Stops at the first failing layer and returns its code
 * (ETIMEDOUT when the kernel does not complete within timeout_ms). */
int ls_stream_run(void* decoder, const ls_stream_layer* layers, uint32_t count, uint32_t first_layer, void* stream,
                  uint64_t* times, uint64_t* stamps, int32_t timeout_ms);
/* Failure injection of the transport (the role of LeanStream's STREAM_TESTING read hook,
 * src/io/stream_io.h): from now on every copy of logical group `group` into the staging
 * arena is refused with `error` (a positive errno) at submission, as a failed read would
 * be; error 0 clears it. The layer then fails with that code through the queue's error
 * word, as a real transport error does. */
int ls_stream_inject_copy_error(void* decoder, uint32_t group, int32_t error);

/* ---- the operators around the MLP of a decode step ----
 * LeanStream leaves them to the application (its Ministral example decodes with kernels of its own:
 * examples/ministral/python/attention_decode_kernels.py:5-97 for rotary positions and grouped-query
 * attention, native/predictor_shared_input.cu:16-41 for the norm). Each call is one block of arguments,
 * checked on the host and put on `stream`; it allocates nothing, never synchronizes and can be captured
 * into a graph. Blocks are plain data and can be reused. Strides are in elements, the last dimension of
 * every tensor is contiguous, and lengths that only the device knows (q_start, context) are read there.
 * A block's optional `status` word (device-visible) gets LS_STATUS_RANGE for a sequence whose lengths do
 * not fit its bounds and LS_STATUS_BAD_DESCRIPTOR for a visible key without a valid page; it is never
 * cleared by a call. Return values: 0, EINVAL for an inconsistent block, ENOTSUP for a shape without
 * kernels, ENOSPC for too small a workspace, or a hipError_t. */
enum { LS_TYPE_F16 = 0, LS_TYPE_BF16 = 1, LS_TYPE_F32 = 2 };

/* Attention of new tokens over a paged cache. Token i of sequence s (its n = q_start[s + 1] - q_start[s]
 * tokens follow one another in q) stands at position p = context[s] - n + i and sees the keys j <= p, with
 * a window only those with j > p - window or j < sinks:
 *   out = sum_j softmax_j(scale q . k_j) v_j, 0 for a token that sees no key;
 *   lse = log sum_j exp(scale q . k_j), -inf for such a token (optional, fp32 [tokens][q_heads]).
 * Query head h reads KV head h / (q_heads / kv_heads). Key j of sequence s is slot j % page_size of page
 * page_table[s * table_stride + j / page_size]; entries of pages that no token sees are not read as pages
 * (any value). Slots that a token does not see do not change its result, whatever they hold. A sequence
 * whose context is out of bounds counts as one with no keys, one whose q_start is out of bounds as one with
 * no tokens, whose rows of out stay as they are (both: status RANGE); a key in a page outside [0, pages)
 * counts as a key and value of zeros (status BAD_DESCRIPTOR).
 * scale > 0; head_dim 64, 128 or 256; page_size a power of two; F16 or BF16 throughout; q, out, the pages and the
 * workspace 16-byte aligned, the others 4-byte, strides multiples of 8. The workspace (ls_hip_attention_workspace
 * bytes, zeroed once by the caller, then left alone) may be shared by calls that follow one another on one stream. */
typedef struct ls_hip_attention {
    const void* q;                /* [tokens][q_heads][head_dim] */
    void* out;                    /* [tokens][q_heads][head_dim] */
    float* lse;
    const void* k_pages;          /* [pages][kv_heads][page_size][head_dim], in any order of strides */
    const void* v_pages;
    const int32_t* page_table;    /* [sequences][table_width] */
    const int32_t* q_start;       /* [sequences + 1] */
    const int32_t* context;       /* [sequences], new tokens included */
    void* workspace;
    uint32_t* status;
    uint64_t workspace_bytes;
    int64_t q_token_stride, q_head_stride, out_token_stride, out_head_stride;
    int64_t k_page_stride, k_head_stride, k_slot_stride, v_page_stride, v_head_stride, v_slot_stride;
    int64_t table_stride;
    uint32_t tokens, sequences, q_heads, kv_heads, head_dim, pages, page_size, table_width;
    uint32_t max_new, max_context; /* bounds of a sequence's n and context */
    uint32_t window, sinks;        /* window 0: none */
    uint32_t dtype;
    float scale;
} ls_hip_attention;
uint64_t ls_hip_attention_workspace(const ls_hip_attention* attention);
int ls_hip_attention_enqueue(const ls_hip_attention* attention, void* stream);

/* New tokens into a paged cache: q_out = rotated q; each token's rotated k and its v into the slot of its
 * position (positions, q_start, context, page_table as above). Rotary pairs (i, i + rot / 2), or
 * (2i, 2i + 1) when interleaved: a' = a cos - b sin, b' = b cos + a sin with row p of the fp32 tables,
 * rounded once; dimensions from rot on are copied. rot 0 copies everything (cos and sin NULL). A token at a
 * negative position, or from `positions` on with rot > 0, or without a valid page is left out (its q_out
 * row too) and raises the status. q and q_out may be one tensor. head_dim even; F16 or BF16. */
typedef struct ls_hip_append {
    const void* q;                /* [tokens][q_heads][head_dim], or NULL with q_heads 0 */
    const void* k;                /* [tokens][kv_heads][head_dim] */
    const void* v;
    const float* cos;             /* [positions][rot / 2] */
    const float* sin;
    void* q_out;
    void* k_pages;
    void* v_pages;
    const int32_t* page_table;
    const int32_t* q_start;
    const int32_t* context;
    uint32_t* status;
    int64_t q_token_stride, q_head_stride, k_token_stride, k_head_stride, v_token_stride, v_head_stride;
    int64_t q_out_token_stride, q_out_head_stride;
    int64_t k_page_stride, k_head_page_stride, k_slot_stride, v_page_stride, v_head_page_stride, v_slot_stride;
    int64_t table_stride;
    uint32_t tokens, sequences, q_heads, kv_heads, head_dim, rot, positions, pages, page_size, table_width;
    uint32_t interleaved, dtype;
} ls_hip_append;
int ls_hip_append_enqueue(const ls_hip_append* append, void* stream);

/* Between two blocks, row by row, in fp32 and rounded once per output:
 *   z = post_weight ? block / rms(block) * (weight_offset + post_weight) : block
 *   h = residual_scale * residual + gate * z          (gate absent: 1)
 *   hidden = h; normed = h / rms(h) * (weight_offset + pre_weight)
 * with rms(x) = sqrt(mean(x^2) + eps). gate_stride 0: one gate row for all. hidden or normed may be NULL
 * (not both; normed needs pre_weight); hidden may be residual, and either may be block. width <= 16384,
 * F16, BF16 or F32 throughout, any alignment of an element. */
typedef struct ls_hip_block_norm {
    const void* block;
    const void* residual;
    const void* gate;
    const void* post_weight;
    const void* pre_weight;
    void* hidden;
    void* normed;
    int64_t block_stride, residual_stride, gate_stride, hidden_stride, normed_stride;
    uint32_t rows, width, dtype;
    float residual_scale, weight_offset, eps;
} ls_hip_block_norm;
int ls_hip_block_norm_enqueue(const ls_hip_block_norm* norm, void* stream);

/* One token a row from given random numbers. With top the row's largest logit and e_i = exp((l_i - top) / T)
 * the tokens are ranked by (logit descending, id ascending); of them keep the first top_k (top_k <= 0: all), of
 * these those whose better-ranked ones weigh less than top_p of all of these, of these those with e_i >= min_p;
 * the best one always stays. The token is the lowest kept id whose weight with the kept ids below it exceeds
 * uniform * (kept weight). Exponentials are fp32. With top_k, and with min_p alone, they are weighed in whole steps of
 * 2^-32 (less than half a step: never drawn), top_p and uniform in steps of 2^-24. Without a filter, and with top_p but
 * no top_k, the row's weight is a sum of fp32 exponentials, 8 or 16 at a time in fp32 and from there in 64-bit floats,
 * in an order that the numbers of rows and logits fix; the share at which top_p cuts and that at which the token is drawn
 * are then within 2^-20 of the definition's. Equal calls give equal results; a row whose top_p or uniform lies that near
 * to the edge between two tokens may get the one or the other in a call of another number of rows.
 * temperature <= 0 (or NaN): the best token. NaN logits count as -inf; a row without a logit above -inf gives token -1
 * and logprob -inf. logprob (optional): the logarithm of e_token over the kept weight.
 * temperature, top_k, top_p, min_p: per row, or NULL for 1, all, 1, 0. vocab <= 2^20.
 * The workspace (ls_hip_sample_workspace bytes, any contents) may be shared by calls of this kind that follow
 * one another on one stream, not with attention's. */
typedef struct ls_hip_sample {
    const void* logits;           /* [rows][vocab], F16, BF16 or F32 */
    const float* uniform;         /* [rows] in [0, 1) */
    const float* temperature;
    const int32_t* top_k;
    const float* top_p;
    const float* min_p;
    int32_t* tokens;
    float* logprob;
    void* workspace;
    uint64_t workspace_bytes;
    int64_t row_stride;
    uint32_t rows, vocab, dtype;
} ls_hip_sample;
uint64_t ls_hip_sample_workspace(const ls_hip_sample* sample);
int ls_hip_sample_enqueue(const ls_hip_sample* sample, void* stream);

/* ---- synthetic workload generation on the device (counter-based splitmix64) ---- */
int ls_synth_bytes(void* dst, uint64_t bytes, uint64_t seed, void* stream);
int ls_synth_uniform_f16(void* dst, uint64_t count, uint64_t seed, double lo, double hi, void* stream);
int ls_synth_normal_f16(void* dst, uint64_t count, uint64_t seed, void* stream);
int ls_synth_normal_bf16(void* dst, uint64_t count, uint64_t seed, void* stream);
/* No reference counterpart; a benchmark utility: holds `stream` (one wave) until the host sets
 * the host-coherent word *flag nonzero, or limit_ticks of the 100 MHz device clock pass. Work
 * queued behind it starts back to back once it is released, without the host's submission
 * latency in between. EINVAL for a NULL flag or a zero limit. */
int ls_hold_stream(void* stream, const uint32_t* flag, uint64_t limit_ticks);

#ifdef __cplusplus
}
#endif
#endif
