/*
 * qwen_hip.h -- C ABI of the MI355X (gfx950) Qwen3-MoE decode engine.
 *
 * This is the drop-in boundary for the reference's compute backend.  The
 * reference binds its backends through a Rust trait (src/backend.rs:14-23):
 *
 *     pub trait Backend {
 *         fn matvec(&mut self, model: &Gguf, name: &str, expert: Option<usize>,
 *                   x: &[f32]) -> Result<Vec<f32>>;
 *         fn stats(&self) -> &Stats;
 *     }
 *
 * and drives the token loop through `Model::forward` (src/model.rs:209-302).
 * Each entry point below names the reference interface it replaces.
 *
 * Conventions (all entry points):
 *   - return 0 on success, nonzero on failure; qh_last_error() then returns a
 *     message owned by the context (the anyhow message of the reference);
 *   - plain host pointers and sizes; caller-owned host buffers; the context
 *     owns every device allocation;
 *   - one context per host thread, calls block until host-visible outputs are
 *     ready (`&mut self` + blocking poll in the reference);
 *   - no silent CPU fallback: without a usable gfx950 device qh_create fails.
 */
#ifndef QWEN_HIP_H
#define QWEN_HIP_H
#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct qh_ctx qh_ctx;

/* == backend::Stats (src/backend.rs:7-13). */
typedef struct {
    uint64_t matvecs;        /* matvecs performed (a fused token step counts the
                                reference's 3 + 1 + 1 + 3*top per layer + 1)   */
    uint64_t uploaded_bytes; /* host->device bytes (weights at load, inputs)  */
    uint64_t cache_hits;     /* always 0: all weights stay resident in HBM    */
    double matvec_ms;        /* wall time spent in matvec / forward calls     */
} qh_stats_t;

/* == model::Config (src/model.rs:5-19). */
typedef struct {
    uint64_t hidden, layers, heads, kvheads, head_dim, experts, top, intermediate,
        vocab, max_context;
    float eps, theta;
} qh_config_t;

/* Creates a context on HIP device `device` (one HIP stream per context).
 * Replaces `Vulkan::new` (src/backend.rs:95-161) / `Compute::backend`
 * (src/main.rs:42-60).  Fails if the device is not gfx950. */
int qh_create(int device, qh_ctx **out);
void qh_destroy(qh_ctx *ctx);
/* Message of the last failure on this context (or, when ctx is NULL, of
 * qh_create and of this thread's calls without a context). */
const char *qh_last_error(const qh_ctx *ctx);

/* Parses and validates a GGUF image held in host memory and uploads every
 * tensor to HBM once (no LRU cache, no buffer splitting).  Replaces
 * `Gguf::open` (src/gguf.rs:102-195) + `Model::new` (src/model.rs:173-201)
 * with the same checks and error behaviour; `context` is the `--ctx` limit.
 * A new load invalidates the previous model (src/backend.rs:357-361). */
int qh_load_model(qh_ctx *ctx, const void *gguf_image, size_t len, size_t context);
/* Same, reading the file at `path`. */
int qh_load_model_file(qh_ctx *ctx, const char *path, size_t context);
int qh_model_config(const qh_ctx *ctx, qh_config_t *out);
/* Number of models loaded into this context so far (no counterpart in the
 * reference, where each Model owns its weights): a caller that keeps a
 * handle to "the loaded model" compares it with the value seen at load time
 * to detect that a later load replaced it. */
int qh_model_generation(const qh_ctx *ctx, uint64_t *out);
/* == Gguf::tensor (src/gguf.rs:196-200): GGML kind, rank and dims of a
 * loaded tensor (dims[0] = columns); "missing tensor {name}" otherwise. */
int qh_tensor_info(const qh_ctx *ctx, const char *name, uint32_t *kind, size_t *rank,
                   uint64_t dims[3]);
/* Sum of tensor payload bytes (src/main.rs:128 packed_weight_bytes). */
int qh_packed_weight_bytes(const qh_ctx *ctx, uint64_t *out);

/* == the `inspect` command (src/main.rs:119-131): Gguf::open + Config::from_gguf
 * + validate_tensors + the context check ("invalid context") + Config::kv_bytes
 * (src/model.rs:150-156, "KV size overflow"), on the file at `path`, with no
 * device work and no context object.  On failure qh_last_error(NULL) holds
 * the message. */
typedef struct {
    qh_config_t config;
    uint64_t tensor_count;
    uint64_t packed_weight_bytes;
    uint64_t kv_f32_bytes_at_context;
} qh_inspect_t;
int qh_inspect(const char *path, size_t context, qh_inspect_t *out);

/* == `Vulkan::devices` (src/backend.rs:162-172) for HIP: number of devices and
 * a one-line description "name (arch, CUs, GiB)" of device `device`.  On
 * failure qh_last_error(NULL) holds the message. */
int qh_device_count(int *out);
int qh_device_name(int device, char *buf, size_t cap);

/* == Backend::matvec (src/backend.rs:14-23, resolution as `matrix`
 * src/backend.rs:57-75): y[rows] = W x for tensor `name`, expert slab
 * `expert` (-1 = None).  Errors: missing tensor, rank mismatch, expert out
 * of bounds, cols != len(x). */
int qh_matvec(qh_ctx *ctx, const char *name, int64_t expert, const float *x, size_t cols,
              float *y, size_t rows);
/* == Backend::stats (src/backend.rs:22). */
int qh_stats(const qh_ctx *ctx, qh_stats_t *out);

/* == Vulkan::packed_matvec test surface (src/backend.rs:173-182): packed
 * GGUF rows given directly.  kind is the GGML type id (0 F32, 1 F16, 2 Q4_0,
 * 8 Q8_0, 12 Q4_K, 13 Q5_K, 14 Q6_K). */
int qh_packed_matvec(qh_ctx *ctx, const void *data, size_t len, uint32_t kind, size_t rows,
                     size_t cols, const float *x, float *y);

/* The per-expert down projections of one MoE layer (the loop of
 * src/model.rs:274-284) as one streaming launch: y[b] = W_b x[b] for b < nvec
 * (1-8), data = the nvec matrices of rows x cols packed GGUF rows back to
 * back, x = nvec x cols floats, y = nvec x rows floats.  Block-quantised
 * formats only (kinds 2, 8, 12, 13, 14), rows of up to 8,192 columns and at
 * most 12,288 x floats in all; other shapes are refused with an error. */
int qh_packed_matvec_batch(qh_ctx *ctx, const void *data, size_t len, uint32_t kind, size_t rows,
                           size_t cols, size_t nvec, const float *x, float *y);

/* == quant::decode (src/quant.rs:81-84) on the device, for `rows` packed
 * rows: out[rows*cols].  Bit-exact with the reference decoder. */
int qh_dequant(qh_ctx *ctx, const void *data, size_t len, uint32_t kind, size_t rows, size_t cols,
               float *out);

/* == ops::route (src/ops.rs:45-56): top `top` expert ids (descending, total
 * order, lower index on ties) and softmax over the chosen logits. */
int qh_route(qh_ctx *ctx, const float *logits, size_t n, size_t top, uint32_t *ids, float *w);

/* == Sampler::sample with temperature 0 (src/sampling.rs:26-35). */
int qh_argmax(qh_ctx *ctx, const float *logits, size_t n, uint32_t *out);

/* == ops::attention (src/ops.rs:57-98); k/v time-major [t][kvheads][d],
 * klen = t*kvheads*d floats. */
int qh_attention(qh_ctx *ctx, const float *q, const float *k, const float *v, size_t klen,
                 size_t heads, size_t kvheads, size_t d, float *out);
/* qh_attention on device buffers that allocates nothing (no counterpart in
 * the reference; for callers that cannot allocate: code under HIP graph
 * capture, tight serving loops, harnesses that forbid hipMalloc).  q, k, v
 * and out are device pointers in qh_attention's layouts; the kernel's chunk
 * partials and counters live in fixed 1 MiB device areas of the library
 * (eight per GPU).  Both entry points cap the key chunks per KV head at what
 * an area holds (a chunk then takes several key tiles), so any history
 * length runs; a shape one chunk of whose partials alone exceeds it
 * (heads x (head_dim + 2) floats > 1 MiB) is refused with an error.  stream NULL:
 * the context's stream, and the call returns when out is written; otherwise
 * the work is enqueued on that HIP stream and the call returns at once.
 * Calls may overlap, from any streams and host threads (a context's own calls
 * come from one thread), and a captured call's graph may be replayed on any
 * stream beside them.  A call takes an area that no call under way on another
 * stream uses; where there is none, and under graph capture, the attention
 * runs without scratch, with the same bits for head_dim 64 or 128, at most
 * eight query heads per KV head and q, k and v aligned to 16 bytes, else with
 * its sums in another order.  It is slower then for long histories (3,581
 * keys, 32 / 4 heads of 128: 70 us, 11 with an area).  A stream is destroyed
 * only when its calls have ended. */
int qh_attention_noalloc(qh_ctx *ctx, const float *q, const float *k, const float *v, size_t klen,
                         size_t heads, size_t kvheads, size_t d, float *out, void *stream);

/* == Model::forward (src/model.rs:209-216): one causal token step on the
 * device (embedding, every layer, KV append, final norm, vocab projection,
 * finite check).  logits (room for logits_cap floats; the model's vocab are
 * written) and argmax may be NULL; logits_cap below the vocabulary is an
 * error.  On error the KV cache and position are reset, as the reference
 * rolls back. */
int qh_forward(qh_ctx *ctx, uint32_t token, float *logits, size_t logits_cap, uint32_t *argmax);
/* Sequential prefill of `n_prompt` tokens followed by `n_new` greedy tokens,
 * all chained on the device with no per-token host round trip (the
 * src/main.rs:250-282 loop with temperature 0).  out_tokens receives the
 * n_new generated ids; logits_last (room for logits_cap floats, nullable)
 * the logits that produced the last generated token.  A call that fails
 * writes neither. */
int qh_generate(qh_ctx *ctx, const uint32_t *prompt, size_t n_prompt, size_t n_new,
                uint32_t *out_tokens, float *logits_last, size_t logits_cap);
/* == Sampler (src/sampling.rs:3-65) with its rand 0.8.8 StdRng stream
 * (ChaCha12 seeded by seed_from_u64), host-side state: qh_sampler_create
 * replaces Sampler::new (src/sampling.rs:10-25) with its check ("invalid
 * sampling parameters", message in qh_last_error(NULL)); top_k 0 = no
 * truncation.  qh_sampler_draw returns the stream's next rng.gen::<f32>(). */
typedef struct qh_sampler qh_sampler;
int qh_sampler_create(uint64_t seed, float temperature, size_t top_k, float top_p, qh_sampler **out);
void qh_sampler_destroy(qh_sampler *sampler);
int qh_sampler_draw(qh_sampler *sampler, float *out);
/* The padding-vocab mask of src/main.rs:262-266: ids with valid[id] == 0 read
 * as f32::MIN in qh_sample (vocab bytes; NULL clears it). */
int qh_set_valid_tokens(qh_ctx *ctx, const uint8_t *valid, size_t n);
/* == Sampler::sample (src/sampling.rs:26-63) on the logits of the last token
 * step, on the device: greedy at temperature 0, else top-k, temperature,
 * top-p and one draw from the stream (consumed only on success), over any
 * number of candidates (up to 4096 sorted in one workgroup's LDS, more in
 * HBM).  Errors: "invalid logits"; more than 1,048,576 logits. */
int qh_sample(qh_ctx *ctx, qh_sampler *sampler, uint32_t *out);
/* The same on n caller logits with an optional mask (valid may be NULL). */
int qh_sample_logits(qh_ctx *ctx, qh_sampler *sampler, const float *logits, const uint8_t *valid,
                     size_t n, uint32_t *out);
/* == Model::reset (src/model.rs:202-208). */
int qh_reset(qh_ctx *ctx);
/* == Model::position (src/model.rs:170). */
int qh_position(const qh_ctx *ctx, size_t *out);

/* Batched prefill of `n` prompt tokens from the current position: replaces
 * the sequential prompt loop of src/main.rs:250-256 (one Model::forward per
 * prompt token, src/model.rs:209-302) with layer-at-a-time fp16 matrix-core
 * GEMMs and a causal flash-attention pass, in chunks of up to 2048 tokens.
 * Fills the KV cache for those positions, writes the greedy id after the
 * last prompt token to the device token ring (so qh_forward / qh_generate
 * continue from it), advances the position by n.  logits (room for
 * logits_cap floats) and argmax (nullable) receive the last prompt token's
 * output.  Numerics: fp16
 * operands with fp32 accumulation (logits within about 1e-2 relative of the
 * FP32 path).  Models the batched path does not cover (head_dim != 128, more
 * than 8 query heads per KV head, more than 128 experts, widths that are not
 * whole 256-column super-blocks (a query width of whole pairs of them),
 * projections that are not block-quantised)
 * run the prompt through the exact token step instead, one per token on the
 * device (the same bits as n qh_forward calls).  Errors as that loop of
 * forwards: the first prompt token at the context limit fails with "context
 * limit N reached", a token outside the vocabulary with "token outside
 * vocabulary" (src/model.rs:219-223), and every failure leaves a clean cache
 * at position 0 (src/model.rs:209-216) and logits and argmax as they were. */
int qh_prefill(qh_ctx *ctx, const uint32_t *prompt, size_t n, float *logits, size_t logits_cap,
               uint32_t *argmax);
/* Prefill implementation (no counterpart in the reference, whose prompt loop
 * is one forward per token): *out = 1 when qh_prefill runs the loaded model's
 * prompts through the batched GEMM path, 0 when through the exact token step. */
int qh_prefill_batched(const qh_ctx *ctx, int *out);
/* Diagnostics (no reference counterpart): how many prompts the batched
 * prefill has run again through the exact token step in this context because
 * its fp16 operands could not hold them (an activation above 65504 in
 * magnitude after an RMSNorm, in q, k or v, or out of the SwiGLU) or its
 * router or output logits were not finite.  The rerun's results are the exact
 * step's (the same bits as n qh_forward calls). */
int qh_prefill_reruns(const qh_ctx *ctx, uint64_t *out);
/* Memory control (no counterpart in the reference, which holds one copy of
 * the weights): frees the batched prefill's device memory, the tile-layout
 * copy of every layer's projection matrices (as many bytes again as their
 * row layout) and the chunk buffers.  The KV cache, the position and the
 * token step's weights stay; the next batched prefill builds both again.
 * For callers that prefill once and then decode with the memory given back. */
int qh_prefill_release(qh_ctx *ctx);
/* Device bytes the batched prefill holds now (tile copies + chunk buffers);
 * 0 before the first batched prefill and after qh_prefill_release. */
int qh_prefill_bytes(const qh_ctx *ctx, uint64_t *out);

/* One decoder layer (the loop body src/model.rs:227-287) applied to x[hidden]
 * in place at position `pos`, with this layer's KV history replaced by
 * kprev/vprev (time-major, `pos` positions).  ids/w (nullable) receive the
 * routed experts.  Resets the model position to 0 afterwards. */
int qh_layer_forward(qh_ctx *ctx, size_t layer, float *x, size_t pos, const float *kprev,
                     const float *vprev, uint32_t *ids, float *w);

/* Token-step implementation (no counterpart in the reference, whose step is
 * host-driven): *out = 1 when qh_forward / qh_generate / qh_layer_forward run
 * the persistent single-launch step (one workgroup per CU, phases handed over
 * through memory), 0 when they run the per-phase kernels.  The persistent
 * step covers Qwen3-MoE shapes with block-quantised projections (one format
 * for q, k, o, gate and up, v and down in it or Q6_K); other models always
 * use the per-phase kernels. */
int qh_persistent(const qh_ctx *ctx, int *out);
/* Selects the implementation for the loaded model (enable = 0: per-phase
 * kernels).  Enabling fails when the model is not covered. */
int qh_set_persistent(qh_ctx *ctx, int enable);

/* Diagnostics of the token steps (no counterpart in the reference, whose
 * KV cache and routing are private to Model): qh_route_log copies the
 * routed experts recorded for positions [pos0, pos0 + n), ids[n][layers][top]
 * in rank order, as the last step that processed each position (qh_forward,
 * qh_generate, qh_prefill, either step implementation) chose them;
 * qh_read_kv copies layer `layer`'s K and V for those positions in the
 * reference's time-major layout [t][kvheads][head_dim] (src/ops.rs:84,93);
 * qh_route_gap_log copies, for the same steps, how close each routing
 * decision was: gaps[n][layers] = (top-th - (top+1)-th largest router logit)
 * / max |router logit| (+inf when every expert is routed), a decision with a
 * gap near 0 being one that rounding may turn either way. */
int qh_route_log(qh_ctx *ctx, size_t pos0, size_t n, uint32_t *ids);
int qh_route_gap_log(qh_ctx *ctx, size_t pos0, size_t n, float *gaps);
int qh_read_kv(qh_ctx *ctx, size_t layer, size_t pos0, size_t n, float *k, float *v);

/* Fault injection for tests of the failure paths (no counterpart in the
 * reference): QH_FAULT_ABORT raises the persistent step's abort flag, so the
 * next step's waits give up at once (every kernel still exits normally) and
 * the step fails with "device synchronisation timed out" and a reset. */
#define QH_FAULT_ABORT 1u
int qh_fault_inject(qh_ctx *ctx, uint32_t kind);

/* Persistent-step timing (no counterpart in the reference): `steps` decode
 * steps continuing from the current position, queued back to back, with HIP
 * events on the context's stream around each step's one k_decode launch;
 * ms_decode receives its mean milliseconds per token.  ms_embed receives the time between the
 * step's first event and that launch (the embedding row is computed inside
 * k_decode, so it is an empty interval).  Fails unless the persistent step is
 * selected. */
int qh_profile_decode(qh_ctx *ctx, size_t steps, double *ms_embed, double *ms_decode);

/* Benchmark surface: `warmup` untimed then `steps` timed greedy decode steps
 * continuing from the current position, timed with HIP events on the
 * context's stream.  ms_total receives the timed milliseconds. */
int qh_bench_decode(qh_ctx *ctx, size_t warmup, size_t steps, double *ms_total);

/* Per-kernel-class timing of `steps` decode steps launched one kernel at a
 * time with HIP events between kernels on the context's stream (continuing
 * from the current position).  ms_by_class[QH_NUM_KERNEL_CLASSES] receives
 * the mean GPU milliseconds per token of each class, in this order:
 * qkv (norm + q/k/v projections), attention (Q/K norm, RoPE, KV append,
 * attention), oproj (output projection, residual, router partials), gateup
 * (router top-k, gate/up projections, SwiGLU), down (down projections,
 * combine, residual), vocab (final norm, vocab projection), finish
 * (argmax, next token). */
#define QH_NUM_KERNEL_CLASSES 7
int qh_profile_step(qh_ctx *ctx, size_t steps, double *ms_by_class, size_t nclass);

/* Timing of one benchmarked matvec shape. */
typedef struct qh_matvec_timing {
    double mean_ms;   /* back-to-back launches rotating over the copies: elapsed / iters */
    double median_ms; /* median over iters launches, each between its own pair of events */
    double empty_ms;  /* back-to-back launches of an empty kernel: the launch floor */
} qh_matvec_timing_t;

/* Benchmark surface for matvecs with device-resident inputs (no reference
 * counterpart).  data holds nvec (1-8) matrices of rows x cols packed GGUF
 * rows back to back, x their nvec input vectors (nvec x cols floats): nvec = 1
 * is Backend::matvec's launch, nvec > 1 the streaming kernel's batched form
 * (one launch for the routed experts' down projections of a MoE layer).
 * `copies` copies of the matrices are uploaded so that successive launches
 * stream distinct HBM rather than the 256 MB MALL; `iters` launches rotate
 * over them.  Fails if an output is not finite. */
int qh_bench_matvec(qh_ctx *ctx, const void *data, size_t len, uint32_t kind, size_t rows,
                    size_t cols, size_t nvec, const float *x, size_t copies, size_t iters,
                    qh_matvec_timing_t *out);

/* Read-only stream ceiling (no reference counterpart): `bytes` of device
 * memory, `copies` copies rotated over, each 16-byte word loaded once per
 * launch by a plain streaming kernel; mean and median launch times as for
 * qh_bench_matvec (empty_ms is 0).  The matvec bandwidths are read against it. */
int qh_bench_read(qh_ctx *ctx, size_t bytes, size_t copies, size_t iters, qh_matvec_timing_t *out);

/* ---- operators on device tensors --------------------------------------- *
 * For a program that serves several sequences from device memory of its own
 * (no counterpart in the reference, which holds one sequence): a key-value
 * cache in pages (append, attention of new tokens, eviction; pages given out and
 * taken back; drafted tokens attended and accepted) and the log probabilities of
 * tokens.  They allocate nothing and keep nothing;
 * what they read and write is device memory of the context's device.
 *
 *   - element kinds: 0 F32, 1 F16, 30 BF16 (GGML's ids), and in a cache 8 Q8_0;
 *   - strides count elements; the last dimension is contiguous; a tensor is
 *     aligned to its elements (kernels for tensors and strides aligned to 16
 *     bytes are faster);
 *   - stream NULL: the context's stream, and the call returns when its outputs
 *     are written (its inputs must be there); QH_NULL_STREAM: the device's null
 *     stream; else that HIP stream.  With a stream the call returns at once,
 *     and may be captured into a graph.  A workspace belongs to one call at a
 *     time: calls that may overlap, and graphs that may be replayed beside
 *     each other, need one each;
 *   - arguments on the host are checked, with an error; what lies in device
 *     memory (lengths, page ids, targets) is checked by the kernels, which read
 *     and write nothing out of range: each call says what it does instead.  What
 *     a call reads must not change before it ends, nor be one of its outputs
 *     where it does not say so, and an output's elements share no memory;
 *   - the calling thread's current HIP device is left as it was. */
#define QH_NULL_STREAM ((void *)(intptr_t)-1)
#define QH_BF16 30u

/* A cache: element j of KV head g of slot s of page p is element p *
 * page_stride + s * token_stride + g * head_stride + j of k and of v.  Q8_0
 * (kind 8): k and v hold int8 codes, and k_scale and v_scale the f16 scale of
 * each 32 of them at that offset / 32; dim and the strides are multiples of 32.
 * dim is at most 256. */
typedef struct {
    void *k, *v;
    void *k_scale, *v_scale; /* kind 8 only */
    uint32_t kind, page, kvheads, dim;
    uint64_t pages;
    size_t page_stride, token_stride, head_stride;
} qh_pages_t;

/* Sequences: key t of sequence b is in slot t % page of page table[b *
 * table_stride + t / page], t < length[b].  most: no length is above it (and
 * table_pages pages hold that many); a sequence whose length is negative or
 * above it counts as out of range.  A length of 0 is a row of padding. */
typedef struct {
    const int32_t *table;
    const int32_t *length;
    size_t table_stride, table_pages;
    uint32_t batch, most;
} qh_sequences_t;

/* [rows][heads][dim] of F32, F16 or BF16. */
typedef struct {
    void *data;
    uint32_t kind;
    size_t row_stride, head_stride;
} qh_heads_t;

/* Q/K norm and RoPE on the way into the cache, and the queries that go with
 * the keys.  q NULL data: no queries.  q_norm / k_norm: RMSNorm weights [dim]
 * (NULL: none).  rope: (cos, sin) pairs [rope_rows][dim / 2], NeoX pairing
 * (NULL: none; dim even); position: the row of each token (NULL: its place in
 * its sequence).  A position outside the table makes the token's q and k NaN. */
typedef struct {
    qh_heads_t q, q_out;
    uint32_t heads;
    const float *q_norm, *k_norm;
    float eps;
    const float *rope;
    size_t rope_rows;
    const int32_t *position;
} qh_append_t;

/* Appends n tokens' k and v ([n][kvheads][dim]).  The lengths count them:
 * sequence b's tokens are first[b] .. first[b + 1] - 1 of k and v (first:
 * batch + 1 ascending numbers; NULL: one token each, n = batch), the last of
 * them at length[b] - 1.  Values are rounded once to the cache's kind (Q8_0:
 * scale max |x| / 127 of each 32, rounded to f16, and the code nearest to x / that
 * scale, which can be one off from GGML's own quantiser; a block with a value that
 * is not finite, or past 127 x 65504, becomes NaN).  Tokens without a place (in
 * front of first[0] or behind first[batch], a length of 0 or out of range) leave
 * every output as it was, those of a page id outside the cache leave the cache as it
 * was.  Two sequences must not append to the same slot.  more: nullable. */
int qh_paged_append(qh_ctx *ctx, const qh_pages_t *cache, const qh_sequences_t *seqs, const int32_t *first, size_t n,
                    const qh_heads_t *k, const qh_heads_t *v, const qh_append_t *more, void *stream);

/* Softmax weights of a cache's keys, summed over each KV head's query heads:
 * in ([batch][kvheads][most], NULL: zeros) plus this call's to out, for every
 * key of a sequence; out behind a sequence's keys is left as it was.  in and
 * out may be the same. */
typedef struct {
    const float *in;
    float *out;
    size_t in_row, in_head, out_row, out_head; /* strides of sequences and KV heads */
} qh_key_weights_t;

/* Attention of one token per sequence over its cached keys (qh_attention's
 * formula with a scale of the caller's): q and out [batch][heads][dim], heads a
 * multiple of kvheads, query head h reading KV head h / (heads / kvheads).
 * Sums in 32 bits, out rounded once to its kind; values whose sum over a
 * sequence's keys is past 32 bits' range (from 2^128 / keys on) may come out not
 * finite.  With an out of F16 or BF16 and queries of the cache's own 16-bit kind, or
 * 16-bit ones over Q8_0, a key's softmax weight enters the products with 17 bits
 * (BF16) or 23 (F16, Q8_0); with an F32 out everything is in 32 bits and takes half
 * as long again.  A sequence without keys, or whose scores are all -inf, gives
 * zeros; one with a length or a page id out of range NaN.  weights nullable; the
 * weights of a sequence whose length is out of range are left as they were, those
 * of one with such a page become NaN.  A Q8_0 cache's values (code times scale) past
 * f16's range, 65504, come out not finite with F16 or BF16 queries and outputs; with
 * F32 ones they are read in 32 bits.  q and out may be the same. */
int qh_paged_attention(qh_ctx *ctx, const qh_pages_t *cache, const qh_sequences_t *seqs, const qh_heads_t *q,
                       uint32_t heads, float scale, const qh_heads_t *out, const qh_key_weights_t *weights,
                       void *workspace, size_t workspace_bytes, void *stream);
/* Bytes of workspace that a call of these shapes needs (0: none; its pointer
 * may then be NULL, else it is aligned to 16 bytes).  With weights it holds every
 * score, batch x heads x most x 4 bytes whatever the lengths are (1 GiB for 64
 * sequences of up to 131,072 keys and 32 heads); without, at most some 34 MB. */
int qh_paged_attention_bytes(qh_ctx *ctx, const qh_pages_t *cache, const qh_sequences_t *seqs, uint32_t heads,
                             int with_weights, size_t *out);

/* Brings every sequence to at most keep keys (fewer than 2^30 - 63 to move): of a
 * longer one every KV head keeps its first `first` keys, its last `recent` and the
 * heaviest of those
 * between by weights ([batch][kvheads][most], strides weight_row and
 * weight_head; total order as f32::total_cmp, the lower index on ties).  Kept
 * keys move in ascending order to the slots 0.. of the pages to[b * to_stride +
 * i] (to_pages of them a row; those that kept keys need are all different), which
 * no sequence of the call may read.  Outputs: kept[batch][kvheads][keep] their
 * indexes (-1 behind them), kept_weights [batch][kvheads][keep] their weights (0
 * behind them), new_length[batch]; none may lie where the call reads (lengths,
 * page tables, weights, from their first element to their last) or another
 * output lies.  A sequence with a length or a page id out of range keeps nothing
 * (length 0). */
int qh_paged_evict(qh_ctx *ctx, const qh_pages_t *cache, const qh_sequences_t *seqs, const float *weights,
                   size_t weight_row, size_t weight_head, size_t keep, size_t first, size_t recent, const int32_t *to,
                   size_t to_stride, size_t to_pages, int32_t *kept, float *kept_weights, int32_t *new_length,
                   void *stream);

/* Attention of several new tokens per sequence, packed: sequence b's are rows
 * first[b] .. first[b + 1] - 1 of q and out ([n][heads][dim]), and their keys are
 * the last of its length[b] keys (appended before).  Token i of m new ones sees the
 * keys up to its own, length - m + i: a whole prompt, the next piece of one, or a
 * single token.  Formula, element kinds and what is out of range as in
 * qh_paged_attention, but: a row gives NaN where one of the keys that it sees is in a
 * page out of range; the rows of a sequence whose length is out of range or below its
 * new tokens give NaN; rows of no sequence (in front of first[0], behind first[batch],
 * or of a sequence whose bounds do not ascend within 0 .. n) are left as they were.
 * Keys and values that a row does not see take no part in it, whatever they hold.
 * Sums and maxima in 32 bits, out rounded once to its kind.  With queries and out of
 * 16 bits over a cache of the queries' kind a key's softmax weight enters the products
 * with 17 bits (BF16) or 23 (F16, in steps no finer than 2^-35 of a row's largest weight, so
 * that one below 2^-36 of it may count nothing).  BF16 queries and out over Q8_0 (heads up
 * to 128 wide, a multiple of 8, rows aligned to 8 bytes) are taken in F16 products:
 * weights (in steps no finer than 2^-31 of the largest) and values (code times scale) are
 * rounded once to F16, so a value past 65504 comes out not finite, and an
 * element of a query is rounded below 2^-31 of the largest finite one of its row and
 * lost below 2^-39.  All other mixes and an F32 out are in 32 bits.  Rows that the bounds
 * give to two sequences hold what either makes of them, values of both mixed.  q and
 * out may be the same.  A call whose tokens times heads pass 2^31, or with the keys
 * 2^62, is refused. */
int qh_paged_prompts(qh_ctx *ctx, const qh_pages_t *cache, const qh_sequences_t *seqs, const int32_t *first, size_t n,
                     const qh_heads_t *q, uint32_t heads, float scale, const qh_heads_t *out, void *workspace,
                     size_t workspace_bytes, void *stream);
/* The same for drafted tokens: a sequence's new tokens are the nodes of a tree, at
 * most 64 (more give NaN), and node i sees every key in front of them and the key of
 * node j where bit j of ancestors[i] ([n]) is set (its own bit, too, is the caller's;
 * bits at or past the number of nodes are ignored).  A row that sees no key gives
 * zeros; one page out of range gives NaN in all of its sequence's rows. */
int qh_paged_tree(qh_ctx *ctx, const qh_pages_t *cache, const qh_sequences_t *seqs, const int32_t *first, size_t n,
                  const uint64_t *ancestors, const qh_heads_t *q, uint32_t heads, float scale, const qh_heads_t *out,
                  void *workspace, size_t workspace_bytes, void *stream);
/* Bytes of workspace that either call needs for these shapes, at most some 68 MB (0:
 * none; its pointer may then be NULL, else it is aligned to 16 bytes).  Calls that may
 * run at once have one each. */
int qh_paged_prompts_bytes(qh_ctx *ctx, const qh_pages_t *cache, const qh_sequences_t *seqs, size_t n, uint32_t heads,
                           size_t *out);

/* Pages of `page` slots each: the ids free[0 .. count[0]) are in no table, the last
 * of them is the next to go.  Both lie in device memory and are the caller's; free
 * has room for `pages` ids.  The plans of a pool run one after another. */
typedef struct {
    int32_t *free, *count;
    uint64_t pages;
    uint32_t page;
} qh_pool_t;

/* What a plan gives out; first and length are needed.  The others are [n], a row for
 * each new token, packed as first says, and may be NULL; -1 (ancestors: 0) behind the
 * last token. */
typedef struct {
    int32_t *length;     /* [batch] new lengths; may be the lengths read */
    int32_t *first;      /* [batch + 1] new tokens in front of each sequence's, and in all */
    int64_t *slot;       /* page id * page + slot within it */
    int32_t *position;   /* the token's place; with parents its depth behind the context */
    int32_t *sequence;
    uint64_t *ancestors; /* with parents: the token's own bit and its ancestors' */
} qh_plan_t;

/* Grows sequences by grow[b] tokens (shrinks them where it is negative): table rows
 * ([batch][table_pages], table_stride apart) of which held[b] entries are in use get
 * pages from the pool, or give those back that the new length does not need, all in
 * place.  Pages that are given back may go to a sequence that grows in the same call.
 * A sequence that grows keeps the pages that it holds beyond its new length; one whose
 * grow is 0 or less gives back all that its new length does not need.
 * Growth is served in the sequences' order, and from the first on that asks for more
 * pages than are left, or brings the new tokens past n, no sequence grows: it keeps
 * its length and gets no tokens (first tells).  So does one whose length, held pages or
 * new length are out of range (of 0 .. table_pages * page).  Pages go out from the
 * stack's end, in order of sequence and place, and come back in the opposite order,
 * so that what is claimed and given back leaves the stack as it was.
 * parents (nullable, [n], packed as the tokens are): each sequence's new tokens are a
 * tree, parents[i] the number (within its sequence) of i's parent, -1 for a root; what
 * is no earlier node counts as -1, and nodes from the 64th on get no ancestors and
 * their place as position. */
int qh_paged_plan(qh_ctx *ctx, const qh_pool_t *pool, int32_t *table, size_t table_stride, size_t table_pages,
                  int32_t *held, const int32_t *length, const int32_t *grow, uint32_t batch, size_t n,
                  const int32_t *parents, const qh_plan_t *out, void *stream);

/* Accepts drafted tokens: sequence b's new tokens (the last keys of its length[b], as
 * in qh_paged_tree) are a tree with its root in front (node 0, a token that is
 * certain), parents and tokens ([n]) as drafted, chosen[i] the model's choice after
 * node i.  From the root on the walk goes to the first later node whose parent is the
 * node reached and whose token is the one chosen there.  The nodes reached are
 * accepted: their keys and values move, in all `layers` caches (of one shape, kind and
 * strides, with the same tables), to the slots behind the context, in order.
 * Outputs: new_length[batch] = length - nodes + accepted; accepted[batch] (root
 * included); path[n]: the accepted nodes' numbers from the sequence's first row on, -1
 * in its other rows and in those in front of first[0] and behind first[batch] (a
 * batch of 0 writes nothing); next[batch] = chosen at the last of them.  A sequence without
 * nodes, with more than 64, or whose length, bounds or pages (those of its nodes) are
 * out of range: length as it was, 0 accepted, next -1, nothing moves (and
 * the rows of one whose bounds do not ascend within 0 .. n are left as they were; rows
 * that the bounds give to two, or that lie in a sequence and in front of first[0] or
 * behind first[batch], hold what either has there).  No
 * output may lie where the call reads, no cache is given twice, and the pages that hold
 * a sequence's nodes are in no other sequence. */
int qh_paged_accept(qh_ctx *ctx, const qh_pages_t *caches, size_t layers, const qh_sequences_t *seqs,
                    const int32_t *first, size_t n, const int32_t *parents, const int32_t *tokens,
                    const int32_t *chosen, int32_t *new_length, int32_t *accepted, int32_t *path, int32_t *next,
                    void *stream);

/* Rows of logits ([rows][vocab], row_stride) of F32, F16 or BF16: logp[rows] =
 * log softmax at target[rows] (both nullable), entropy[rows] (nullable), and the
 * top (0-128, at most vocab) ids of each row in descending total order, the
 * lower id on ties, with their log probabilities (top_ids, top_logp
 * [rows][top]).  valid: nullable [vocab] mask, ids with 0 read as f32::MIN (as
 * in qh_sample_logits).  Sums in 32 bits.  A row that holds NaN or +inf gives
 * NaN, one of -inf alone log probabilities of -inf and an entropy of 0, a target
 * outside the vocabulary NaN.  At most 2^24 logits a row. */
int qh_logprobs(qh_ctx *ctx, const void *logits, uint32_t kind, size_t rows, size_t vocab, size_t row_stride,
                const int32_t *target, const uint8_t *valid, size_t top, float *logp, float *entropy, int32_t *top_ids,
                float *top_logp, void *workspace, size_t workspace_bytes, void *stream);
int qh_logprobs_bytes(qh_ctx *ctx, size_t rows, size_t vocab, size_t top, size_t *out);
/* The same for the logits of the last token step (with qh_set_valid_tokens'
 * mask), read where they are: target nullable, outputs on the host (top_ids and
 * top_logp hold top values). */
int qh_last_logprobs(qh_ctx *ctx, const uint32_t *target, size_t top, float *logp, float *entropy, uint32_t *top_ids,
                     float *top_logp);

#ifdef __cplusplus
}
#endif
#endif
