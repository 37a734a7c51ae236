/*
 * hayai_cuda.h -- C ABI of the B200 (sm_100a) quantized-FFN backend.
 *
 * This is the drop-in boundary for Hayai's FFN hot path.  Every entry point is
 * extern "C", takes plain pointers and sizes, returns an int status (HC_OK = 0)
 * and never throws or aborts across the ABI; the message of the last failure on
 * the calling thread is available from hc_last_error().
 *
 * Each declaration cites the reference interface it replaces (paths relative to
 * the aitups/hayai repository root).  The reference backend is
 * hayai-opencl's OpenClEngine (crates/hayai-opencl/src/compute.rs,
 * async_gemv.rs), dispatched from hayai-core's EngineOrchestrator
 * (crates/hayai-core/src/orchestrator.rs).
 *
 * Conventions
 *  - ggml_type uses GGUF's GgmlType ids (crates/hayai-model/src/gguf_types.rs:6-40):
 *    F32=0, F16=1, Q4_0=2, Q4_1=3, Q5_0=6, Q5_1=7, Q8_0=8, Q8_1=9, Q2_K=10, Q3_K=11, Q4_K=12,
 *    Q5_K=13, Q6_K=14, Q8_K=15, IQ2_XXS=16, IQ2_XS=17, IQ3_XXS=18, IQ4_NL=20, IQ3_S=21, IQ2_S=22,
 *    IQ4_XS=23, BF16=30 (the formats of gemv_row_bytes, compute.rs:877-907).
 *    Q4_K, Q6_K and Q8_0 run on the tensor-core kernels (tile-major upload); the others on
 *    CUDA-core kernels over the raw GGUF rows.  Any other id is HC_ERR_UNSUPPORTED.
 *  - A weight matrix is GGUF-layout: nrows = m rows of ncols = n columns, each row
 *    n/QK consecutive blocks (crates/hayai-model/src/quant.rs:28-37); y[m] = W x[n].
 *  - "host" pointers are ordinary CPU memory, borrowed for the call only (or until
 *    hc_pending_wait for the async call).  "_dev" entry points take device pointers
 *    of the engine's GPU, enqueue on the engine's stream and return without waiting.
 *  - An engine is externally synchronised (the reference keeps its orchestrator
 *    behind a Mutex, orchestrator.rs:65-68); engines on different GPUs are independent.
 */
#ifndef HAYAI_CUDA_H
#define HAYAI_CUDA_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- status codes ---------------------------------------------------------- */
#define HC_OK 0
#define HC_ERR_INVALID 1     /* bad shape / size / argument (compute.rs:912-951 validation) */
#define HC_ERR_UNSUPPORTED 2 /* no kernel for this ggml type (orchestrator.rs:403-409 hard fail) */
#define HC_ERR_CUDA 3        /* CUDA runtime error */
#define HC_ERR_RANGE 4       /* an activation is outside the f16 range used by the tensor-core split */
#define HC_ERR_NCCL 5        /* collective failed */
#define HC_ERR_TIMEOUT 6     /* a bounded device wait expired */

typedef struct hc_engine hc_engine;   /* one GPU + stream: OpenClEngine (crates/hayai-opencl/src/context.rs:23) */
typedef struct hc_weights hc_weights; /* a resident weight matrix (one-time upload) */
typedef struct hc_pending hc_pending; /* in-flight GEMV: PendingGemv (crates/hayai-opencl/src/async_gemv.rs:15-57) */

/* Message of the last failure on this thread ("" if none).  Replaces
 * OpenClError::ClError(String) (crates/hayai-opencl/src/context.rs:14). */
const char* hc_last_error(void);

/* Number of CUDA devices.  Replaces discover_opencl_devices (crates/hayai-opencl/src/device.rs). */
int hc_device_count(int* out);

/* Create / destroy an engine on `device`.  Replaces OpenClEngine::init_device
 * (crates/hayai-opencl/src/context.rs:106). */
int hc_engine_init(int device, hc_engine** out);
int hc_engine_free(hc_engine* eng);

/* Enqueue on the caller's CUDA stream (cudaStream_t as void*; NULL = the legacy default
 * stream), or go back to the engine's own non-blocking stream. */
int hc_engine_set_stream(hc_engine* eng, void* stream);
int hc_engine_use_own_stream(hc_engine* eng);
int hc_engine_get_stream(hc_engine* eng, void** stream);

/* Wait for all work on the engine stream and report any device-side error. */
int hc_sync(hc_engine* eng);

/* Packed bytes per row for n columns; HC_ERR_INVALID if n is not a multiple of the
 * block.  Replaces gemv_row_bytes (crates/hayai-opencl/src/compute.rs:877-907). */
int hc_gemv_row_bytes(int ggml_type, size_t n, size_t* out);

/* ---- resident weights --------------------------------------------------------
 * One-time upload of an m x n GGUF-layout matrix into HBM, rewritten into the GPU
 * layout of its format.  Replaces the device mirror / resident preload
 * (allocate_resident_for_pool, crates/hayai-opencl/src/hetero_scratch.rs:243) and
 * the ping-pong streaming it fed.  Validation as validate_gemv_weights
 * (compute.rs:912-933). */
int hc_weights_upload(hc_engine* eng, int ggml_type, size_t m, size_t n, const void* host_bytes, size_t len,
                      hc_weights** out);
/* Same, from GGUF-layout bytes already on the engine's GPU (GgmlWeightBind::Device,
 * compute.rs:21-27). */
int hc_weights_from_device(hc_engine* eng, int ggml_type, size_t m, size_t n, const void* dev_bytes, size_t len,
                           hc_weights** out);
int hc_weights_free(hc_weights* w);
/* ggml_type, m, n and resident bytes of a weights object. */
int hc_weights_info(const hc_weights* w, int* ggml_type, size_t* m, size_t* n, size_t* bytes);

/* ---- GEMV ---------------------------------------------------------------------- */
/* y[m] = W x[n] with host weights, host input/output; blocking.  Replaces
 * OpenClEngine::ggml_gemv_dispatch (compute.rs:281-385) and the per-type wrappers
 * ggml_gemv_q4_k / q6_k / q8_0 (compute.rs:153-276). */
int hc_ggml_gemv_dispatch(hc_engine* eng, int ggml_type, size_t m, size_t n, const uint8_t* weights,
                          size_t weights_len, const float* input, float* output);

/* Resident weights, host input/output; blocking.  Replaces ggml_gemv_dispatch_bound
 * (compute.rs:388-461) and EngineOrchestrator::execute_quant_gemv (orchestrator.rs:222-234). */
int hc_ggml_gemv_bound(hc_engine* eng, const hc_weights* w, const float* input, float* output);

/* `batch` input rows [batch][n] -> outputs [batch][m]; blocking.  Replaces
 * ggml_gemv_batched_q4_k (compute.rs:179-257) and execute_quant_gemv_batched
 * (orchestrator.rs:240-269) for every type. */
int hc_ggml_gemv_batched(hc_engine* eng, const hc_weights* w, const float* inputs, float* outputs, size_t batch);

/* Asynchronous GEMV: ggml_gemv_async / ggml_gemv_async_from_device
 * (async_gemv.rs:90-130).  hc_pending_wait copies the m outputs into `output`
 * (PendingGemv::wait, async_gemv.rs:27); hc_pending_free waits first, as
 * PendingGemv::drop does (async_gemv.rs:48-57). */
int hc_ggml_gemv_async(hc_engine* eng, const hc_weights* w, const float* input, hc_pending** out);
int hc_pending_wait(hc_pending* p, float* output, size_t m);
int hc_pending_free(hc_pending* p);

/* Device pointers: y[v][ldy] = resid[v][ldr] (if non-NULL) + W x[v][ldx] for v < nvec,
 * enqueued on the engine stream.  x must be 16-byte aligned with ldx % 4 == 0. */
int hc_gemv_dev(hc_engine* eng, const hc_weights* w, const float* x, size_t ldx, float* y, size_t ldy,
                const float* resid, size_t ldr, size_t nvec);

/* hc_gemv_dev for Q4_K, Q6_K and Q8_0 weights that allocates nothing.  No counterpart in
 * the reference: it exists for callers that cannot let a library call cudaMalloc -- hosts
 * whose device memory belongs to their own pool allocator, and decode loops that cannot
 * absorb the device synchronisation a cudaMalloc/cudaFree may cause.  The scratch the
 * stream-K split needs comes from a static device array of the library (4 MiB of partial
 * sums + 16384 tile counters per GPU, held until exit); a matrix that needs more is
 * rejected with HC_ERR_INVALID (every Llama-3 8B/70B FFN matrix and a 128256 x 4096 output
 * projection fit; M above 262144 never does).  Every call looks the array's address up
 * on the current device (cudaGetSymbolAddress, which allocates nothing); on the first call
 * on a device that lookup also loads the library's device code there, so make that first
 * call before any stream capture.  All calls on a device share the array, so calls that overlap
 * on the GPU race: serialise them.  Other formats return HC_ERR_UNSUPPORTED. */
int hc_gemv_dev_noalloc(hc_engine* eng, const hc_weights* w, const float* x, size_t ldx, float* y, size_t ldy,
                        const float* resid, size_t ldr, size_t nvec);

/* Toy 16-entry LUT-Q4 matmul (two nibbles per byte, low nibble first); blocking.
 * Replaces OpenClEngine::lut_matmul_q4 (compute.rs:45-128) and
 * EngineOrchestrator::execute_lut_matmul (orchestrator.rs:198-218). */
int hc_lut_matmul_q4(hc_engine* eng, size_t m, size_t n, const uint8_t* weights_q4, const float* lut16,
                     const float* input, float* output);
int hc_lut_matmul_q4_dev(hc_engine* eng, size_t m, size_t n, const uint8_t* weights_q4, const float* lut16,
                         const float* input, float* output);

/* ---- SwiGLU FFN block -------------------------------------------------------------
 * y = W_down (silu(W_gate x) * (W_up x)), the block of run_ffn_block
 * (crates/hayai-core/src/stream_infer.rs:574-606) with the host SiLU*up combine
 * (:3836-3840) fused on the device.  gate/up are d_ff x k_in, down is n_out x d_ff.
 * Host version: blocking, no residual. */
int hc_ffn_swiglu(hc_engine* eng, const hc_weights* gate, const hc_weights* up, const hc_weights* down,
                  const float* x, float* y, size_t nvec);
/* Device version: y[v] = resid[v] (optional) + FFN(x[v]); h_ws is a device scratch of
 * nvec * d_ff floats (NULL = engine workspace).  x/y rows are k_in / n_out floats. */
int hc_ffn_swiglu_dev(hc_engine* eng, const hc_weights* gate, const hc_weights* up, const hc_weights* down,
                      const float* x, float* y, const float* resid, float* h_ws, size_t nvec);

/* The fused first half of the block alone: h[v] = silu(W_gate xn[v]) * (W_up xn[v]), one
 * kernel reading both matrices (ffn_begin_gate_up_scratch + the SiLU*up combine,
 * stream_infer.rs:3752-3840).  xn = rms_norm(x, norm_w, eps) over the first norm_len
 * entries of each row (crates/hayai-cpu/src/attention.rs:142-147) when norm_w (device,
 * norm_len floats) is non-NULL, else x.  h is [nvec][d_ff]. */
int hc_ffn_gateup_dev(hc_engine* eng, const hc_weights* gate, const hc_weights* up, const float* x, float* h,
                      size_t nvec, const float* norm_w, size_t norm_len, float eps);

/* Stack of n_layers FFN sublayers with pre-norm and residual, as in a decode step
 * (stream_infer.rs:2166-2170 rms_norm(x, ffn_norm) then :3752-3864):
 *     x <- x + FFN_l(rms_norm(x, norm_w[l], eps))        for l = 0..n_layers-1
 * norm_w is an array of n_layers device pointers (n_out floats each), or NULL for no
 * normalization.  x is [nvec][k_in] with k_in >= n_out (rows zero-padded for K-quant
 * block alignment; norm and residual cover the first n_out entries).  _dev works in place
 * on device memory (captured once into a CUDA graph and replayed); the host version
 * copies x in and the result out. */
int hc_ffn_stack_dev(hc_engine* eng, const hc_weights* const* gate, const hc_weights* const* up,
                     const hc_weights* const* down, const float* const* norm_w, float eps, size_t n_layers,
                     float* x, size_t nvec);
int hc_ffn_stack(hc_engine* eng, const hc_weights* const* gate, const hc_weights* const* up,
                 const hc_weights* const* down, const float* const* norm_w, float eps, size_t n_layers,
                 const float* x_in, float* x_out, size_t nvec);

/* ---- tensor / expert parallelism (one process per GPU) -----------------------------
 * No reference counterpart: the reference has no multi-GPU FFN.  A group of `world` ranks
 * (<= 8, one GPU each) shares exchange regions: hc_peer_open allocates this rank's region
 * (bytes >= 12 MiB; zeroed) and writes its CUDA IPC handle (hc_peer_handle_bytes bytes) to
 * handle_out; the caller gathers every rank's handle over its own process group, in rank
 * order, and passes them to hc_peer_connect; then all ranks must pass a host barrier before
 * the first parallel call.  Kernels store partial results into the peers' regions over
 * NVLink and signal each other with system-scope atomics (waits bounded by one second:
 * HC_ERR_TIMEOUT).  Parallel calls are collective: every rank makes the same calls in the
 * same order.  hc_peer_close (after a host barrier) unmaps and frees. */
int hc_peer_handle_bytes(size_t* out);
int hc_peer_open(hc_engine* eng, int rank, int world, size_t bytes, void* handle_out);
int hc_peer_connect(hc_engine* eng, const void* handles);
int hc_peer_close(hc_engine* eng);
/* This rank's exchange region (device address and size) for diagnostics: its layout holds
 * the exchange counters and epochs.  No reference counterpart. */
int hc_peer_region(hc_engine* eng, void** region, size_t* bytes);

/* Tensor-parallel FFN stack, the config-5 sharding of Llama-3-70B: rank p holds gate/up rows
 * and down columns [p*F/P, (p+1)*F/P) of every layer (F = d_ff, column shards whole
 * super-blocks).  x [nvec][d_model] is replicated; each layer's down output is all-reduced
 * over the ranks' exchange regions (stream_infer.rs:2166's residual add after the down GEMV,
 * with the sum over shards) and added in rank order, so x ends identical on every rank.
 * nvec = 1: inside the persistent stack kernel.  nvec > 1: per-layer kernels plus one
 * all-reduce kernel per layer, as one CUDA graph; the region must then hold
 * 8 MiB + 4 KiB + 8 * P * nvec * d_model bytes (hc_peer_open's `bytes`). */
int hc_ffn_stack_tp_dev(hc_engine* eng, const hc_weights* const* gate, const hc_weights* const* up,
                        const hc_weights* const* down, const float* const* norm_w, float eps, size_t n_layers,
                        float* x, size_t nvec);
int hc_ffn_stack_tp(hc_engine* eng, const hc_weights* const* gate, const hc_weights* const* up,
                    const hc_weights* const* down, const float* const* norm_w, float eps, size_t n_layers,
                    const float* x_in, float* x_out, size_t nvec);

/* ---- MoE ---------------------------------------------------------------------------
 * Routing of route_experts (crates/hayai-core/src/moe_infer.rs:868-935, with
 * top_k_indices :852-862 and MoeMeta exec_plan.rs:244-272), on the device, for
 * n_tok score rows [n_tok][n_expert].  ids are bit-exact with the reference for
 * identical scores; weights follow the reference's softmax/sigmoid in f32. */
int hc_route_experts_dev(hc_engine* eng, const float* scores, const float* bias, size_t n_tok, size_t n_expert,
                         size_t top_k, size_t n_group, size_t topk_group, int gating, int norm_topk_prob,
                         float routed_scaling_factor, int32_t* ids, float* weights);

/* Router GEMV with the reference's summation order (gemv_f32, quant.rs:358-369:
 * sequential sum += w*x, no FMA), so scores are bit-identical to the CPU path. */
int hc_router_scores_dev(hc_engine* eng, const float* router_w, size_t n_expert, size_t d_model, const float* x,
                         size_t n_tok, float* scores);

/* Expert-routed SwiGLU FFN for n_tok tokens (forward_moe's router -> top-k ->
 * per-expert FFN -> weighted sum, moe_infer.rs:221-264, :342-376, :449-455):
 * y[t] = sum_i w_i * FFN_{e_i}(x[t]) (no residual).  Experts are given as arrays of
 * n_expert weight handles.  ids_out/w_out (device, [n_tok][top_k], may be NULL)
 * receive the routing. */
int hc_moe_ffn_dev(hc_engine* eng, const float* router_w, size_t n_expert, size_t top_k, int norm_topk_prob,
                   float routed_scaling_factor, const hc_weights* const* gate, const hc_weights* const* up,
                   const hc_weights* const* down, const float* x, size_t n_tok, float* y, int32_t* ids_out,
                   float* w_out);

/* Expert-parallel MoE FFN (the Qwen3-30B-A3B sharding): this rank holds experts
 * [expert_lo, expert_lo + n_local) (gate/up/down arrays of n_local handles); router_w
 * covers all n_expert experts and x [n_tok][d_model] is replicated, so every rank routes
 * identically.  Each rank computes the (token, slot) pairs routed to its experts and stores
 * their down rows into every rank's exchange region over NVLink (the all-to-all of routed
 * outputs, fused into the expert GEMV's epilogue); after a cross-GPU signal every rank adds
 * the rows in top-k order (moe_infer.rs:449-455), so y is identical on all ranks and does
 * not depend on the rank count.  Needs a connected peer group; collective. */
int hc_moe_ffn_ep_dev(hc_engine* eng, const float* router_w, size_t n_expert, size_t top_k, int norm_topk_prob,
                      float routed_scaling_factor, const hc_weights* const* gate, const hc_weights* const* up,
                      const hc_weights* const* down, size_t expert_lo, size_t n_local, const float* x, size_t n_tok,
                      float* y, int32_t* ids_out, float* w_out);

/* A stack of MoE layers for n_tok tokens, x <- x + MoE_l(x) for l = 0..n_layers-1 (the
 * residual add of the callers of forward_moe, moe_infer.rs:222-223), in place on device
 * memory, captured once into a CUDA graph and replayed.  router_w: n_layers device pointers
 * ([n_expert][d_model] each); gate/up/down: n_layers x n_expert handles, layer-major.  The
 * _ep variant holds experts [expert_lo, expert_lo + n_local) of every layer (n_layers x
 * n_local handles) and exchanges the routed rows as hc_moe_ffn_ep_dev does; collective. */
int hc_moe_stack_dev(hc_engine* eng, size_t n_layers, const float* const* router_w, size_t n_expert, size_t top_k,
                     int norm_topk_prob, float routed_scaling_factor, const hc_weights* const* gate,
                     const hc_weights* const* up, const hc_weights* const* down, float* x, size_t n_tok);
int hc_moe_stack_ep_dev(hc_engine* eng, size_t n_layers, const float* const* router_w, size_t n_expert,
                        size_t top_k, int norm_topk_prob, float routed_scaling_factor, const hc_weights* const* gate,
                        const hc_weights* const* up, const hc_weights* const* down, size_t expert_lo, size_t n_local,
                        float* x, size_t n_tok);

/* ---- paged key/value cache and attention over it ------------------------------------
 * Counterpart of the reference's KV cache and decode attention (crates/hayai-cpu/src/
 * kv_cache.rs, attention.rs; device form crates/hayai-opencl/src/attn.rs), over pages that
 * sequences of a batch share out of one pool.  All pointers are device memory of the engine's
 * GPU; the calls enqueue on the engine's stream.
 *
 * hc_kv_cache: one layer's pool.  k and v hold n_pages x n_heads x page_size rows of head_dim
 * (64 or 128) elements: F16, BF16, or 8-bit codes (type 24, GGUF's I8) with one f32 scale per row,
 * value = code * scale.  Row (page, head, r) starts at page * page_stride + head * head_stride +
 * r * row_stride elements; strides are whole multiples of 64 bytes.  Scale (page, head, r) is at
 * page * scale_page_stride + head * page_size + r.
 *
 * hc_kv_batch: n_seq sequences.  Sequence s has kv_len[s] tokens, at positions 0.. of the pages
 * page_table[s * table_stride + position / page_size]; its last q_start[s+1] - q_start[s] tokens
 * are the step's new ones, rows [q_start[s], q_start[s+1]) of the packed row arrays of n_tok rows
 * (q_start ascends; rows that no sequence has are left alone, as are tokens before position 0).
 * max_new is the host's bound on any sequence's new tokens (0: n_tok); a sequence with more is
 * still computed, at lower speed.  Page numbers, lengths or offsets out of range touch no
 * memory out of the pool: they are cut to it, and hc_sync reports HC_ERR_INVALID. */
#define HC_KV_MAX_SEQ 2048
typedef struct hc_kv_cache {
    int type, n_pages, n_heads, page_size, head_dim;
    void *k, *v;
    float *k_scale, *v_scale; /* 8-bit codes only */
    size_t page_stride, head_stride, row_stride, scale_page_stride;
} hc_kv_cache;
typedef struct hc_kv_batch {
    int n_seq, n_tok, max_new, max_pages;
    const int32_t* page_table;
    size_t table_stride;
    const int32_t *q_start, *kv_len;
} hc_kv_batch;

/* Store the new tokens' rows k, v [n_tok][n_heads * head_dim] (leading dimensions ldk, ldv; dtype
 * F32, F16 or BF16) in the cache.  8-bit: scale = max|x| * f32(1/127) and code = x / scale to
 * nearest even, both in f32; a row that is not finite reads back as NaN. */
int hc_kv_append_dev(hc_engine* eng, const hc_kv_cache* cache, const hc_kv_batch* batch, int dtype, const void* k,
                     size_t ldk, const void* v, size_t ldv);

/* Gather the same rows back out of the cache, as the values they stand for (with kv_len[s] new
 * tokens for a sequence: all of it). */
int hc_kv_read_dev(hc_engine* eng, const hc_kv_cache* cache, const hc_kv_batch* batch, int dtype, void* k, size_t ldk,
                   void* v, size_t ldv);

/* out_i = sum_j softmax_j(scale q_i . k_j) v_j for the new tokens' n_heads query heads (q, out
 * [n_tok][n_heads * head_dim], leading dimensions ldq, ldo, of one dtype), n_heads a multiple of
 * the cache's (query head h reads kv head h / (n_heads / cache heads)).  causal: a token sees the
 * positions up to its own, of which window > 0 leaves the last `window` and the first `sink`; else
 * all kv_len.  lse (NULL or [n_tok][n_heads]) receives log sum_j exp(scale q_i . k_j).  A token
 * that sees nothing gets out 0 and lse -inf.  out must not overlap q.  Partial results lie in the
 * engine, about 40 MB for the calls on each stream and as much for those captured on it, made by the
 * first such call (also inside a capture) and kept: calls on two streams, and a graph beside direct
 * calls, may be in flight together, but of the graphs captured on one stream only one at a time. */
int hc_attn_paged_dev(hc_engine* eng, const hc_kv_cache* cache, const hc_kv_batch* batch, int dtype, size_t n_heads,
                      const void* q, size_t ldq, void* out, size_t ldo, float* lse, float scale, int causal, int window,
                      int sink);

/* Sequences of a batch that share their first tokens (an instruction, a document): group g is the batch's
 * sequences [seq_start[g], seq_start[g+1]) (seq_start ascends; sequences in no group share nothing), whose
 * first length[g] positions hold the same keys and values, as hc_kv_fork_dev leaves them.  They are read by the
 * pages of the group's first sequence that has new tokens; those without may have gone.  Of a length past the tokens
 * that every such sequence had before its new ones, that much is shared.  max_new is the host's bound on any group's
 * new tokens (0: n_tok); a group with more is still computed, at lower speed.  least: how many tokens of reading the
 * call's sharing has to save, over all groups, to be made (0: by a rule of the library's, on the prefixes' lengths, the
 * sequences' rows and the types, which leaves it where it would be slower). */
typedef struct hc_kv_shared {
    int n_groups, max_new;
    int64_t least;
    const int32_t *seq_start, *length; /* n_groups + 1, n_groups; device */
} hc_kv_shared;

/* hc_attn_paged_dev (causal, without a window) for groups of sequences with shared tokens, which are read once
 * for the group and seen by all its rows together.  Its notes hold here too.  Where sharing is made, results are
 * other roundings of the same sums: f32 rows keep their terms; 16-bit rows' weights are rounded to the products' type
 * part by part (bf16; or f16, in which weights below 2^-21 of a part's largest have fewer bits), single tokens' too,
 * whose weights hc_attn_paged_dev rounds at a size of their own for every few positions.  Between the call's kernels
 * partial results lie in the engine, in a workspace of up to 4.5 * n_tok * n_heads * (head_dim + 2) floats and 21 MB (for
 * many single tokens, and f32 rows, up to 3.5), which grows with the calls in powers of two, past 256 MB in quarters of
 * them.  It is made before the device knows whether sharing is worth it; where there is no room for it, nothing is shared. */
int hc_attn_shared_dev(hc_engine* eng, const hc_kv_cache* cache, const hc_kv_batch* batch, const hc_kv_shared* shared,
                       int dtype, size_t n_heads, const void* q, size_t ldq, void* out, size_t ldo, float* lse, float scale);

/* ---- rotary positions -----------------------------------------------------------------
 * Counterpart of the reference's RoPE (crates/hayai-cpu/src/attention.rs).  The first rot_dim values of a head
 * are rot_dim / 2 pairs, (i, i + rot_dim / 2) in the half layout, (2 i, 2 i + 1) in pairs; at position p pair i,
 * (a, b), becomes amplitude * (a c - b s, a s + b c) with c = cos(p t_i), s = sin(p t_i).  The rest of a head
 * stays.  The frequencies are kept as fractions of a turn, 2^64 to the turn, so that every position of 32
 * bits, negative ones as well, has its angle to 2^-32 of a turn. */
#define HC_ROPE_HALF 0
#define HC_ROPE_PAIRS 1
#define HC_ROPE_MAX 128
typedef struct hc_rope {
    int layout, head_dim, rot_dim; /* both even, head_dim at most 2 * HC_ROPE_MAX */
    float amplitude;
    uint64_t turns[HC_ROPE_MAX]; /* t_i / 2 pi of a turn */
} hc_rope;

/* Fill in *out (host memory only): t_i = base^(-2 i / rot_dim) / factors[i] (NULL: ones; rot_dim / 2 of them, as a
 * GGUF file's rope_freqs), rot_dim 0 for the whole head.  Longer contexts: original = 0 divides every t_i by `factor`
 * (linear scaling); original > 0, the context that the model was trained with, divides by bands: with the r =
 * original * t_i / 2 pi turns that it made there and g = (r - low) / (high - low) held to [0, 1], t_i becomes
 * t_i * ((1 - g) / factor + g).  (With amplitude 0.1 ln factor + 1 that is YaRN, Peng et al. 2023.) */
int hc_rope_init(hc_rope* out, int layout, int head_dim, int rot_dim, double base, double factor, double original,
                 double low, double high, const float* factors, float amplitude);

/* Turn the rows x [n_tok][n_heads * head_dim] (leading dimension ldx; dtype F32, F16 or BF16) by positions [n_tok]
 * into out, which is x itself or does not overlap it. */
int hc_rope_dev(hc_engine* eng, const hc_rope* rope, int dtype, size_t n_tok, size_t n_heads, const int32_t* positions,
                const void* x, size_t ldx, void* out, size_t ldo);

/* hc_kv_append_dev for keys that are turned by their positions in the cache on the way, and the n_heads query heads
 * with them, in one launch: q [n_tok][n_heads * head_dim] into q_out (q itself, or overlapping none of the rows).
 * rot_dim is a multiple of 16, in pairs of 8.  8-bit codes are of the turned values, unrounded. */
int hc_kv_append_rope_dev(hc_engine* eng, const hc_kv_cache* cache, const hc_kv_batch* batch, const hc_rope* rope, int dtype,
                          size_t n_heads, const void* q, size_t ldq, void* q_out, size_t ldqo, const void* k, size_t ldk,
                          const void* v, size_t ldv);

/* ---- the cache's bookkeeping ------------------------------------------------------------
 * Page tables, lengths and holders of the pool's pages, on the device.  Slot s holds kv_len[s] tokens in the pages
 * page_table[s * table_stride + 0 ..]; refs[p] is the number of table entries in use that name page p, 0 for a free
 * page.  Every layer's cache has the same shape and follows the same tables.  A slot's last page, where it is partly
 * filled, belongs to the slot alone, so that appending never writes what another slot reads; whole pages may be
 * shared.  An array of slots, kv_len and the page table serve as a hc_kv_batch's with n_seq = n_slots.
 * Calls on one hc_kv_pages are made on one stream, or in an order that the caller sees to; they keep their plan in
 * `scratch`.  Left out, and reported by hc_sync as HC_ERR_INVALID, are items whose slots or lengths (those that the slots
 * have, as well) are out of range, or the number of the partly filled page that they keep; a slot's second time in a
 * call; forks into slots that hold tokens; and items for which no free page is left, with all later ones that take
 * pages.  Whole pages' numbers that are out of range are reported and otherwise left as they are: a child gets its
 * parent's, and they are neither counted nor given back. */
typedef struct hc_kv_pages {
    int n_slots, max_pages, n_layers;
    int32_t* page_table; /* [n_slots][table_stride] */
    size_t table_stride;
    int32_t *kv_len, *refs;    /* [n_slots], [n_pages] */
    int32_t* scratch;          /* hc_kv_pages_scratch(n_pages) ints */
    const hc_kv_cache* layers; /* host array, at most 256; pages of at most 2^26 tokens */
} hc_kv_pages;
int hc_kv_pages_scratch(int n_pages, size_t* out);

/* Slot children[i] becomes a copy of slot parents[i] (device arrays; n at most HC_KV_MAX_SEQ): it shares the whole
 * pages and gets the rest copied to a page of its own, the lowest free one, in the order of i.  Parents are taken as
 * they were before the call. */
int hc_kv_fork_dev(hc_engine* eng, const hc_kv_pages* pages, int n, const int32_t* parents, const int32_t* children);

/* Slot slots[i] gets the length lens[i]: pages are taken (the lowest that were free before the call, in the order
 * of i and of the table) or given back; a length of 0 lets the slot go.  Where the last page kept is partly filled then,
 * and other table entries named it before the call, the slot gets a copy of it, whatever the call's other items do.
 * Pages that the call gives back are free for the next one. */
int hc_kv_resize_dev(hc_engine* eng, const hc_kv_pages* pages, int n, const int32_t* slots, const int32_t* lens);

/* The pages in use move to the lowest numbers: of u of them, those numbered u and more go, in ascending order, to the
 * free ones below.  The tables follow, and moved (NULL or [n_pages]) receives every page's new number. */
int hc_kv_compact_dev(hc_engine* eng, const hc_kv_pages* pages, int32_t* moved);

/* ---- synthetic data ----------------------------------------------------------------
 * Seeded N(mean, std^2) floats on the device (splitmix64 at a position + Box-Muller in
 * double; the same stream as the test oracle's generator up to last-bit differences of
 * the device's double log/sin/cos). */
int hc_synth_normal_dev(hc_engine* eng, uint64_t seed, size_t n, float mean, float stdv, float* out);
/* Quantize n device floats into GGUF blocks on the device.  Q4_K restates the reference
 * quantizer bit-exactly (quantize_q4_k, crates/hayai-model/src/q4k.rs:85-160); Q6_K and
 * Q8_0 use this library's own quantizers (the reference has none). */
int hc_quantize_dev(hc_engine* eng, int ggml_type, const float* x, size_t n, uint8_t* out);

#ifdef __cplusplus
}
#endif

#endif /* HAYAI_CUDA_H */
