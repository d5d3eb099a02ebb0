/* z2h.h — C ABI of libzonos2_hip.so, the MI355X (gfx950) ragged continuous-batching decode step of
 * the ZONOS2 MoE backbone.
 *
 * Every entry point is extern "C", takes plain pointers and sizes, and returns an int status
 * (Z2H_OK == 0). The per-context message of the last failure is available from z2h_last_error().
 * No C++ exception crosses this boundary. A context is not reentrant: one thread drives it, as in
 * the reference (src/server.cpp:905-911, docs/INTERNALS.md:200).
 *
 * Weights live in a reference-counted z2h_model (the reference's zonos2_model, loaded once); each
 * z2h_ctx (the reference's zonos2_batch_ctx: KV cache, scratch, step graphs) holds one reference, so
 * several batch contexts can share one model. z2h_create is the one-call form: model and context.
 *
 * Reference interfaces replaced (file:line in Zyphra/zonos2.cpp):
 *   z2h_model_create      zonos2_model_load hparams    src/zonos2.cpp:15-97, src/zonos2.h:124
 *   z2h_model_upload_tensor zonos2_model_load tensors  src/zonos2.cpp:100-119, name map 137-183
 *   z2h_model_finalize    zonos2_model_load field map  src/zonos2.cpp:126-185
 *   z2h_model_release     zonos2_model_free            src/zonos2.h:125, src/zonos2.cpp:188-195
 *   z2h_create_batch      zonos2_batch_init            src/zonos2-graph.cpp:639-690 (KV alloc, S rounding)
 *   z2h_create            zonos2_model_load + zonos2_batch_init in one call
 *   z2h_upload_tensor     as z2h_model_upload_tensor on the context's model
 *   z2h_finalize          as z2h_model_finalize, then the context's scratch
 *   z2h_step              zonos2_batch_step            src/zonos2-graph.cpp:762-837 (+ slot_logits 839-841)
 *   z2h_prefill           zonos2_batch_slot_prefill    src/zonos2-graph.cpp:703-760
 *   z2h_speaker_embed     the speaker column of build_graph, src/zonos2-graph.cpp:262-297
 *   z2h_moe_forward       build_moe                    src/zonos2-graph.cpp:191-239 (one MoE layer)
 *   z2h_set_expert_mask   zonos2_set_expert_mask       src/zonos2.cpp:203-239, src/zonos2.h:136
 *   z2h_destroy           zonos2_batch_free            src/zonos2-graph.cpp:692-701 (+ drops the model reference)
 * Without a reference counterpart: the mixed pass, the operators on device tensors around a paged cache (z2h_rope_rows,
 * z2h_paged_append, z2h_paged_plan, z2h_paged_attn, z2h_verify, z2h_prompt_attn, z2h_moe_rows, z2h_pages_fork, z2h_pages_compact)
 * with the paged pass over them (z2h_step_paged), capture, graph and profiling switches.
 */
#ifndef Z2H_H
#define Z2H_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum {
    Z2H_OK = 0,
    Z2H_EINVAL = 1,     /* bad argument (shape, range, missing tensor) */
    Z2H_ENOMEM = 2,     /* device or host allocation failed */
    Z2H_EDEVICE = 3,    /* HIP runtime error */
    Z2H_ESTATE = 4,     /* call not valid in the context's current state */
    Z2H_ENOTSUP = 5     /* unsupported tensor type / layout */
};

/* GGUF tensor type ids accepted by z2h_upload_tensor */
enum { Z2H_F32 = 0, Z2H_F16 = 1, Z2H_Q8_0 = 8, Z2H_Q4_K = 12, Z2H_Q6_K = 14 };

/* Mirrors zonos2_hparams (src/zonos2.h:14-50); router_dim = router_down.ne1 (src/zonos2.cpp:241-246). */
typedef struct z2h_hparams {
    int32_t n_layer, n_embd, head_dim, n_head, n_head_kv, n_ff, n_expert, n_ctx_train;
    float   rope_freq_base, rms_eps, qk_norm_eps, logit_softcap;
    int32_t n_codebooks, codebook_size, audio_vocab, eoa_id, audio_pad_id, text_vocab;
    int32_t spk_dim, spk_lda_dim;
    int32_t router_dim;
    const int32_t * expert_used;   /* [n_layer]: 0 = dense FFN, else MoE top-k */
} z2h_hparams;

typedef struct z2h_model z2h_model;
typedef struct z2h_ctx z2h_ctx;

/* Weights only, on HIP device `device`; refcount 1. Upload every tensor, then finalize. */
int z2h_model_create(const z2h_hparams * hp, int device, z2h_model ** out);
/* Tensor hand-over as for z2h_upload_tensor below. */
int z2h_model_upload_tensor(z2h_model * m, const char * name, int type, const int64_t ne[4],
                            const void * data, size_t nbytes);
/* Checks that every tensor the forward pass needs is present; no uploads afterwards. */
int z2h_model_finalize(z2h_model * m);
/* Expert mask / router-logit bias (see z2h_set_expert_mask / z2h_set_logit_bias) on the model: every
 * context sharing it sees the change at its next step. No step may be in flight on any of them. */
int z2h_model_set_expert_mask(z2h_model * m, int layer, const uint8_t * keep);
int z2h_model_set_logit_bias(z2h_model * m, int layer, const float * bias);
/* Depth prune (zonos2_model::layer_skip, src/zonos2.h:116-121; src/zonos2-graph.cpp:334-341):
 * skip[L] != 0 bypasses block L in every following step and prefill (attention, KV append and FFN are
 * not run; the residual passes through unchanged; the router state threads past it). skip has
 * n_layer entries; NULL clears. */
int z2h_model_set_layer_skip(z2h_model * m, const uint8_t * skip);
const char * z2h_model_last_error(const z2h_model * m);
/* Drops one reference; the weights are freed with the last one (contexts hold one each). */
void z2h_model_release(z2h_model * m);

/* A batch context over a model (takes a reference; the model may be finalized before or after, through
 * z2h_finalize). n_slots decode slots of slot_cap_frames rows each (rounded up to a multiple of 256,
 * as the reference does); the KV cache is zero-filled. */
int z2h_create_batch(z2h_model * m, int n_slots, int slot_cap_frames, z2h_ctx ** out);
/* The same with room for max_rows rows per pass (z2h_step_mixed, z2h_moe_forward; at least n_slots
 * and Z2H_PREFILL_CHUNK_MAX); the step scratch grows with it (about 0.2 MB per row at d_model 2048,
 * plus attention partials for max_rows x slot_cap / 32 chunks). No reference counterpart. */
int z2h_create_batch_rows(z2h_model * m, int n_slots, int slot_cap_frames, int max_rows, z2h_ctx ** out);

/* A new model on HIP device `device` and a batch context over it (which then holds the model's only
 * reference) in one call. */
int z2h_create(const z2h_hparams * hp, int n_slots, int slot_cap_frames, int device, z2h_ctx ** out);

/* Hand over one GGUF tensor: name as in the reference GGUF, ggml ne order (ne0 fastest, unused = 1),
 * host bytes in GGUF block layout. The bytes are copied (repacked for the device) before return. */
int z2h_upload_tensor(z2h_ctx * ctx, const char * name, int type, const int64_t ne[4],
                      const void * data, size_t nbytes);

/* After all uploads: finalizes the context's model (if not yet) and allocates the step scratch. */
int z2h_finalize(z2h_ctx * ctx);

/* Slot rows per slot after rounding (the reference's slot_cap). */
int z2h_slot_cap(const z2h_ctx * ctx);

/* Write / read KV rows [row0, row0+n_rows) of `slot` in layer `layer`. Host layout
 * [n_rows][n_head_kv][head_dim] of f16 bits; either pointer may be NULL. */
int z2h_kv_write(z2h_ctx * ctx, int layer, int slot, int row0, int n_rows, const uint16_t * k, const uint16_t * v);
int z2h_kv_read(z2h_ctx * ctx, int layer, int slot, int row0, int n_rows, uint16_t * k, uint16_t * v);

/* One batched decode step over n_active columns. slot_idx[i] selects the KV band, n_past[i] is the
 * row the new K/V are written at (the row count already in the cache), ids is [n_active][n_codebooks+1]
 * (audio codes then the text id), or NULL when emb ([n_active][n_embd] fp32, injected in place of the
 * summed embedding before emb_norm) is given. out_logits receives [n_active][n_codebooks][audio_vocab]
 * post-softcap logits, or stays on the device only (out_logits NULL) for z2h_sample. Unlike the
 * reference, idle slots are simply not listed (no padded columns). */
int z2h_step(z2h_ctx * ctx, int n_active, const int32_t * slot_idx, const int32_t * n_past,
             const int32_t * ids, const float * emb, float * out_logits);

/* Same step with device-resident inputs/outputs, enqueued on `stream` (a hipStream_t, NULL = the
 * context's stream) without synchronizing. d_slot_idx/d_n_past: [n_active] int32; d_ids or d_emb as
 * above; d_logits [n_active][n_codebooks*audio_vocab]. h_n_past must hold the same n_past values on
 * the host (grid sizing for the ragged attention). */
int z2h_step_device(z2h_ctx * ctx, int n_active, const int32_t * d_slot_idx, const int32_t * d_n_past,
                    const int32_t * h_n_past, const int32_t * d_ids, const float * d_emb,
                    float * d_logits, void * stream);

/* Prefill n0 prompt rows into `slot` (rows [0, n0)), causal within the prompt as in the reference's
 * per-slot prefill: the rows attend each other's fp32 K/V (src/zonos2-graph.cpp:155-169) while their
 * f16 rows are written to the slot's cache for the decode steps; ids [n0][n_codebooks+1]. spk
 * (optional, [spk_dim]) replaces row spk_pos's embedding by spk_proj(spk_lda(spk)) (+ delta [n_embd]
 * if non-NULL). last_logits receives the final row's [n_codebooks][audio_vocab] logits. */
int z2h_prefill(z2h_ctx * ctx, int slot, const int32_t * ids, int n0, const float * spk, int spk_pos,
                const float * delta, float * last_logits);

/* The speaker rows of n speaker vectors (spk [n][spk_dim]; n <= Z2H_SPEAKER_MAX): spk_proj(spk_lda(spk)
 * + b_lda) + b_proj (+ delta [n][n_embd] if non-NULL), into out [n][n_embd] (host memory) - the
 * column the reference writes over a prompt row before emb_norm (src/zonos2-graph.cpp:262-297), for
 * callers that place speaker rows in a mixed pass themselves (emb_map / emb of z2h_step_mixed);
 * z2h_prefill computes its speaker row the same way. Synchronizes the context's stream. */
#define Z2H_SPEAKER_MAX 64
int z2h_speaker_embed(z2h_ctx * ctx, int n, const float * spk, const float * delta, float * out);

/* One pass over n_rows rows from any slots, decode columns and prefill-chunk rows mixed (the
 * reference has no mixed pass; it is its zonos2_batch_step and zonos2_batch_slot_prefill graphs in
 * one, src/zonos2-graph.cpp:703-837). Row t writes slot_idx[t]'s cache row n_past[t] and attends to
 * that slot's rows [0, n_past[t]], including rows of this pass: every row's K/V is appended before
 * the attention. No two rows may share (slot, n_past). ids [n_rows][n_codebooks+1]; emb_map (NULL, or
 * [n_rows]: -1 = the row sums its ids, e >= 0 = the row takes emb[e], e.g. a speaker prefix row) with
 * emb [n_emb][n_embd]. out_logits [n_out][n_codebooks][audio_vocab] receives the logits of rows
 * out_rows[0 .. n_out) (the output head runs on those rows only). n_rows and n_out are limited by
 * the context's row capacity (z2h_create_batch_rows). */
int z2h_step_mixed(z2h_ctx * ctx, int n_rows, const int32_t * slot_idx, const int32_t * n_past, const int32_t * ids,
                   const int32_t * emb_map, const float * emb, int n_emb, int n_out, const int32_t * out_rows, float * out_logits);

/* Rows per prefill chunk (1 .. the context's row capacity, max(n_slots, Z2H_PREFILL_CHUNK_MAX, max_rows);
 * default the capacity, so a prompt that fits is one pass and streams each layer's weights once).
 * A chunk's rows go through each layer together (the projections and expert matmuls see them as one
 * batch; every row appends its K/V before the chunk's attention), so a prompt of n0 rows takes
 * ceil(n0 / rows) passes instead of n0 single-row steps. Any chunk size gives the same results. No
 * reference counterpart: the reference builds one graph over the whole prompt. */
#define Z2H_PREFILL_CHUNK_MAX 256
int z2h_set_prefill_chunk(z2h_ctx * ctx, int rows);

/* One MoE layer (build_moe) on n_tokens host rows x [n_tokens][n_embd] (the layer's ffn_in); state_in
 * ([n_tokens][router_dim], may be NULL) is the previous MoE layer's router state. out [n_tokens][n_embd]. */
int z2h_moe_forward(z2h_ctx * ctx, int layer, int n_tokens, const float * x, const float * state_in, float * out);
/* Device-pointer variant, enqueued on `stream` without synchronizing. */
int z2h_moe_forward_device(z2h_ctx * ctx, int layer, int n_tokens, const float * d_x, const float * d_state_in,
                           float * d_out, void * stream);

/* One MoE layer (as z2h_moe_forward_device) on a model alone, allocating nothing: no context, and no
 * hipMalloc / hipFree or other allocating call. No counterpart in the reference: it is for callers
 * that cannot allocate device memory (code under HIP graph capture, tight serving loops, harnesses
 * that forbid it). Every intermediate buffer (activation encodings, routing, route lists, SwiGLU
 * rows, per-route outputs, the router state unless d_state_out is given) is carved from a static
 * device array of 16 MiB per GPU, held until the process ends; a call whose buffers would not fit
 * (n_tokens x top-k routes at the model's widths) is refused with Z2H_EINVAL before any launch, as
 * is n_tokens * top-k > 1024. Calls on one GPU share that array: calls that overlap on one GPU (two
 * streams, two threads) race and must be serialized by the caller. Enqueued on `stream` (NULL: the
 * null stream) without synchronizing. d_x [n_tokens][n_embd] (the layer's ffn_in), d_state_in
 * ([n_tokens][router_dim] or NULL), d_state_out (NULL, or [n_tokens][router_dim] receiving this
 * layer's router state), d_out [n_tokens][n_embd]. Results are bit-identical to z2h_moe_forward_device.
 * The caller's current HIP device is the same on return. Errors: z2h_model_last_error. */
int z2h_model_moe_forward_noalloc(z2h_model * m, int layer, int n_tokens, const float * d_x, const float * d_state_in,
                                  float * d_state_out, float * d_out, void * stream);

/* Runtime expert mask for one MoE layer: keep[e] != 0 keeps expert e routable (logits and selection
 * scores of the others get -inf); keep == NULL clears the layer's mask. */
int z2h_set_expert_mask(z2h_ctx * ctx, int layer, const uint8_t * keep);

/* Depth prune on the context's model (see z2h_model_set_layer_skip). */
int z2h_set_layer_skip(z2h_ctx * ctx, const uint8_t * skip);

/* Additive pre-softmax router-logit bias for one MoE layer ([n_expert] fp32, NULL clears). Not a
 * reference input: a benchmark hook to impose a skewed expert popularity. */
int z2h_set_logit_bias(z2h_ctx * ctx, int layer, const float * bias);

/* Frame sampling on the device, for callers that keep the logits in HBM. It follows the reference's
 * per-codebook sampler (src/zonos2-sampler.cpp:16-77, called per slot by zonos2_slot_sample,
 * src/zonos2-graph.cpp:843-870) with the random generator left on the host: column i, codebook cb
 * applies the repetition penalty over hist, temperature, top-k (logit descending), softmax (float
 * exp terms over a double sum), top-p, min-p and draws at u * kept mass along the candidates, with
 * equal logits and probabilities in the orders that the reference's std::partial_sort / std::sort
 * (GCC 11 libstdc++) give them. u[i][cb] is the canonical double in [0, 1) that the host sampler's
 * std::uniform_real_distribution would take from its mt19937 (std::generate_canonical<double, 53>);
 * it is not used where the kept mass is 0 (for finite logits: min_p > 1), where the host sampler
 * takes no draw.
 * The exp terms are exp(x) computed in double and rounded to float, so a draw can differ from the
 * host sampler's (glibc expf) only where the two roundings differ by an ulp and u falls between the
 * two cumulative sums.
 *   d_logits  [n_active][n_codebooks][audio_vocab] on the device, NULL = the last z2h_step's logits
 *   sp        [n_active] settings (greedy takes the first maximum of the raw logits)
 *   hist      [n_active][n_codebooks][hist_cap] recent codes, oldest first (NULL: no penalty);
 *             hist_len [n_active][n_codebooks] entries used; hist_cap <= Z2H_SAMPLE_HIST_MAX
 *   u         [n_active][n_codebooks];  codes out [n_active][n_codebooks] (host memory)
 * Synchronizes the context's stream. */
#define Z2H_SAMPLE_HIST_MAX 256
typedef struct z2h_sampling {
    float   temperature;
    int32_t top_k;            /* 0 or >= audio_vocab: every id is a candidate */
    float   top_p;            /* 0 disables */
    float   min_p;            /* 0 disables */
    float   rep_penalty;
    int32_t rep_codebooks;    /* codebooks cb < rep_codebooks get the penalty */
    int32_t greedy;
    int32_t reserved;
} z2h_sampling;
int z2h_sample(z2h_ctx * ctx, int n_active, const float * d_logits, const z2h_sampling * sp, const int32_t * hist,
               const int32_t * hist_len, int hist_cap, const double * u, int32_t * codes);

/* Device-resident step tables (no reference counterpart; the reference repacks ids, positions and its
 * mask on the host every step, src/zonos2-graph.cpp:773-813). z2h_sample_feed is z2h_sample on the
 * last step's logits (which must come from z2h_step, z2h_step_resident or the graph path of
 * z2h_step_device with ids) that also writes each column's next input frame (its codes + the text pad
 * id text_vocab) and n_past + 1 into the context's step tables; z2h_step_resident(ctx, n) then runs
 * the next step of the same n columns from those tables without any host upload, leaving the logits
 * on the device (enqueued, not synchronized). Any other step, prefill or sample clears the tables. */
int z2h_sample_feed(z2h_ctx * ctx, int n_active, const z2h_sampling * sp, const int32_t * hist, const int32_t * hist_len,
                    int hist_cap, const double * u, int32_t * codes);
int z2h_step_resident(z2h_ctx * ctx, int n_active);

/* ---------------------------------------------------------------------------------------------------------
 * Operators on device tensors around a paged key / value cache (no reference counterpart: the reference keeps one
 * contiguous band per slot, src/zonos2-graph.cpp:639-690, and its decode step, like z2h_step, reads a prompt that
 * requests share once per request). For callers that keep their own buffers; z2h_step_paged, at the end of the section,
 * runs the model's layers over them. The operators take a context for its device and its error string only: no tensor,
 * no weights and no z2h_finalize are needed, nothing is allocated, nothing synchronizes, and every call may be captured
 * into a HIP graph. All tensors are on the context's device. Work is enqueued on `stream` (a hipStream_t, NULL = the null stream); the
 * caller's current device is the same on return. Strides are in elements. No rows (no sequences to verify): nothing is done, and
 * their tensors may be NULL.
 *
 * Tables of lengths, positions and pages are read on the device and are not checked on the host: an entry out of range
 * never leads outside the buffers described to the call (each function says what it does then). */
enum { Z2H_BF16 = 30 };

/* Rotary positions. Of each head's first n_dims dims, pair i of n_dims / 2 is (2i, 2i + 1), or with `halves`
 * (i, i + n_dims / 2); at position p it turns by p theta'_i and is scaled by mscale. The dims behind n_dims stay as they are.
 *   theta_i = base^(-2i / n_dims),  theta'_i = theta_i (g_i + (1 - g_i) / factor)
 * orig_ctx = 0: g_i = 0 (every pair slowed by `factor`; 1 = plain). orig_ctx > 0, for contexts `factor` times as long
 * as the orig_ctx positions of training: with r_i = orig_ctx theta_i / (2 pi) turns within these,
 * g_i = clamp((r_i - low_turns) / (high_turns - low_turns), 0, 1): fast pairs keep their speed, slow ones are stretched.
 * Angles are formed in 64 bits, so far positions keep their phase. */
typedef struct z2h_rope {
    float   base;
    int32_t n_dims;           /* even, 0 .. head_dim */
    int32_t halves;
    float   factor;
    float   low_turns, high_turns;
    int32_t orig_ctx;
    float   mscale;
} z2h_rope;

/* A paged cache of one layer: k and v are [n_pages][n_head_kv][page_rows][head_dim] of Z2H_F16 or Z2H_BF16, page_stride
 * apart (at least n_head_kv * page_rows * head_dim; a multiple of 8; k and v 16-byte aligned). page_rows is a power of two
 * from 16 to 4096, head_dim 32, 64 or 128. Row r of sequence s is row r % page_rows of page
 * table[s * table_len + r / page_rows]; `table` is [n_seq][table_len] on the device. Sequences may name the same pages. */
typedef struct z2h_pages {
    void *  k, * v;
    int64_t page_stride;
    int32_t type, n_pages, page_rows, n_head_kv, head_dim;
    int32_t n_seq, table_len;
    const int32_t * table;
} z2h_pages;

/* Rotate n_rows rows of n_head heads at positions d_pos [n_rows]: out = rope(x), both [n_rows][n_head][head_dim] of `type`
 * (Z2H_F32, Z2H_F16 or Z2H_BF16), rows x_stride / out_stride apart. head_dim is even, at most 128. d_out may be d_x
 * (with the same stride). Products and sums in fp32, rounded once. */
int z2h_rope_rows(z2h_ctx * ctx, const z2h_rope * rope, int n_rows, int n_head, int head_dim, int type, const void * d_x,
                  int64_t x_stride, void * d_out, int64_t out_stride, const int32_t * d_pos, void * stream);

/* Append n_rows rows to a paged cache: row t's keys, rotated at d_pos[t], and its values become row d_pos[t] of sequence
 * d_seq[t]; its n_head query heads, rotated likewise, go to d_q_out. d_k, d_v [n_rows][n_head_kv][head_dim] and d_q,
 * d_q_out [n_rows][n_head][head_dim] are of `type` (Z2H_F32, Z2H_F16 or Z2H_BF16), rows *_stride apart, so that they may
 * be columns of one fused projection; d_q NULL: keys and values only. d_q_out may be d_q. Rounded once to the cache's type.
 * No two rows may share (sequence, position). A row with d_seq[t] outside [0, n_seq) is padding: nothing of it is
 * read or written. A row whose position lies outside the table, or whose page is outside [0, n_pages), leaves the cache
 * as it was; its queries are rotated. */
int z2h_paged_append(z2h_ctx * ctx, const z2h_pages * pages, const z2h_rope * rope, int n_rows, const int32_t * d_seq,
                     const int32_t * d_pos, int type, const void * d_k, int64_t k_stride, const void * d_v, int64_t v_stride,
                     int n_head, const void * d_q, int64_t q_stride, void * d_q_out, int64_t q_out_stride, void * stream);

/* Attention of a batch of sequences over a paged cache, where groups of sequences may share a prefix (a voice prompt)
 * that is read and multiplied once for the whole group.
 *
 * z2h_paged_plan lays out the work from the lengths, which it reads on the device, into the workspace; z2h_paged_attn
 * may then be called any number of times (every layer of a step) with the same shapes and workspace. Sequence s has
 * query rows [d_row_start[s], d_row_start[s + 1]) of the batch (d_row_start [n_seq + 1] ascending from 0 to n_rows; no
 * rows: the sequence sits this call out) and d_kv_len[s] cache rows, its query rows' own among them: row j of m sees
 * rows [0, d_kv_len[s] - m + j]. A row that sees nothing gives zeros. Group g is sequences [d_group_start[g],
 * d_group_start[g + 1]) (d_group_start [n_group + 1] ascending), whose first d_prefix_len[g] cache rows hold the same
 * values: they are read through the group's first sequence, and only as many as it has. Sequences outside every group
 * share nothing; n_group may be 0. A page entry outside [0, n_pages) reads as page 0; lengths are clamped to the
 * table. Row or group tables that are not ascending make no plan: z2h_paged_attn then leaves d_out as it was.
 *
 * z2h_paged_attn: d_out = softmax(scale q k^T) v for d_q [n_rows][n_head][head_dim], rows q_stride / out_stride apart,
 * n_head a multiple of n_head_kv, at most 64 query heads per key head; query head h reads key head h / (n_head /
 * n_head_kv). `type` is Z2H_F32 or Z2H_F16 over Z2H_F16 pages, or Z2H_BF16 over Z2H_BF16 pages. d_out may be d_q (with
 * the same stride). Softmax and sums in fp32; the weights meet the
 * values to 2^-16 of them (bf16) or 2^-22. Results do not depend on timing (no atomics). Cache rows that a row does not see
 * do not reach it, whatever they hold. A value that is not finite reaches every row that sees it; a key whose score is minus
 * infinity has no weight, and one whose score is infinity or no number leaves the row without a number. (Rows that see such a
 * cache row take longer: about 1.5 ms over 16384 keys.)
 *
 * The workspace (z2h_paged_ws_bytes; 0 = the shapes are refused, see z2h_last_error; 256-byte aligned) holds the plan
 * and the partial results of one call at a time: calls and graphs that may overlap need one each. z2h_paged_attn with
 * another shape than the plan's leaves d_out as it was. */
int64_t z2h_paged_ws_bytes(z2h_ctx * ctx, const z2h_pages * pages, int n_head, int n_rows, int n_group);
int z2h_paged_plan(z2h_ctx * ctx, const z2h_pages * pages, int n_head, int n_rows, const int32_t * d_row_start,
                   const int32_t * d_kv_len, int n_group, const int32_t * d_group_start, const int32_t * d_prefix_len,
                   void * d_ws, int64_t ws_bytes, void * stream);
int z2h_paged_attn(z2h_ctx * ctx, const z2h_pages * pages, int n_head, int n_rows, int n_group, float scale, int type,
                   const void * d_q, int64_t q_stride, void * d_out, int64_t out_stride, void * d_ws, int64_t ws_bytes,
                   void * stream);

/* Verification of drafted frames against the target's probabilities, with the random numbers given (the device
 * counterpart of z2h_sample for speculative decoding). Sequence s has d_n_draft[s] drafted frames (clamped to 0 ..
 * n_draft_max; NULL: n_draft_max each) of n_codebooks codes, d_draft [n_seq][n_draft_max][n_codebooks]. d_target
 * [n_seq][n_draft_max + 1] [n_codebooks][vocab] is what the target model says at each drafted frame and behind the
 * last: probabilities, or with d_temperature [n_seq] logits, p = softmax(logits / temperature) (0 or less: all mass on
 * the first largest logit). d_draft_probs [n_seq][n_draft_max][n_codebooks][vocab] are the probabilities q that the
 * drafts were drawn from; NULL: the drafts were not drawn (q = 1 at the drafted code). The codes are judged in order,
 * frame by frame and codebook by codebook: code x is kept iff u q(x) < p(x), u = d_u_accept
 * [n_seq][n_draft_max][n_codebooks]. Behind the first code that is not kept, in frame k codebook c, the sequence ends:
 * d_n_accept[s] = k whole frames are kept, and d_codes[s] ([n_seq][n_codebooks]) is the frame that follows them: the
 * kept codes of frame k before c, at c a draw from max(p - q, 0) (from p where that has no mass), behind c draws from
 * p of frame k. With every code kept it is a draw from p of the frame behind the last draft. A draw takes the first
 * code whose cumulative mass exceeds u (total mass), u = d_u_draw [n_seq][n_codebooks], and if rounding leaves none,
 * the last with mass. So the frames are distributed as the target's own, codebook by codebook. Probabilities, sums and
 * comparisons in 64 bits. Random numbers are doubles in [0, 1). A drafted code outside [0, vocab) is not kept.
 * Probabilities that are no numbers or have no mass give some code in range. vocab is at most 2^20. The workspace
 * (z2h_verify_ws_bytes; 0: the sizes are refused; 256-byte aligned) holds one call at a time. */
int64_t z2h_verify_ws_bytes(int n_seq, int n_draft_max, int n_codebooks, int vocab);
int z2h_verify(z2h_ctx * ctx, int n_seq, int n_draft_max, int n_codebooks, int vocab, const int32_t * d_draft,
               const int32_t * d_n_draft, const float * d_target, const float * d_temperature, const float * d_draft_probs,
               const double * d_u_accept, const double * d_u_draw, int32_t * d_n_accept, int32_t * d_codes, void * d_ws,
               int64_t ws_bytes, void * stream);

/* Attention of whole prompts that lie packed one behind the other: sequence s is rows [d_row_start[s], d_row_start[s + 1]) of
 * d_q [n_rows][n_head][head_dim] and of d_k, d_v [n_rows][n_head_kv][head_dim] (d_row_start [n_seq + 1] ascending on the device), and row r of it
 * attends to its sequence's rows up to r itself: d_out = softmax(scale q k^T) v, [n_rows][n_head][head_dim]. The rows' keys and values are
 * read as they lie, columns of one fused projection say (rows *_stride apart), before or after z2h_paged_append puts them into pages. All
 * four are of `type` (Z2H_F32, Z2H_F16 or Z2H_BF16); head_dim is 32, 64 or 128, n_head a multiple of n_head_kv, at most 64 query heads
 * per key head; query head h reads key head h / (n_head / n_head_kv). d_out may be d_q (with the same stride). A sequence may have no
 * rows; rows of no sequence are left as they were. Entries of d_row_start are clamped to 0 .. n_rows; rows between entries that descend
 * get some value or none.
 * Softmax and sums in fp32; F32 rows are multiplied in fp32, 16-bit rows' weights meet the values to 2^-16 of them (bf16) or 2^-22. Results do
 * not depend on timing (no atomics). Rows that a row does not see do not reach it, whatever they hold. A value that is not finite reaches
 * every row that sees it; a key whose score is minus infinity has no weight, and one whose score is infinity or no number leaves the row
 * without a number; a row none of whose keys has a weight gives zeros. Scores are formed in fp32; one beyond its range may count as infinite. (Rows that
 * see such a value take longer, since they are formed a second time, key by key: 200 times as long where all of 8191 rows do.) */
int z2h_prompt_attn(z2h_ctx * ctx, int n_seq, const int32_t * d_row_start, int n_rows, int n_head, int n_head_kv, int head_dim,
                    float scale, int type, const void * d_q, int64_t q_stride, const void * d_k, int64_t k_stride, const void * d_v,
                    int64_t v_stride, void * d_out, int64_t out_stride, void * stream);

/* The experts of one mixture-of-experts layer: gate and up [n_expert][n_ff][n_embd], down [n_expert][n_embd][n_ff], of Z2H_F16 or
 * Z2H_BF16, 16-byte aligned; n_embd and n_ff are multiples of 8 (8 .. 65536), n_expert 1 .. 1024. */
typedef struct z2h_experts {
    const void * gate, * up, * down;
    int32_t type, n_expert, n_ff, n_embd;
} z2h_experts;

/* A mixture-of-experts layer for a few rows (a step's, a request's drafts; 1 .. Z2H_MOE_ROWS_MAX), in two or three launches:
 *   p = softmax(d_logits of the row), the top_k experts by p + d_bias (NULL: by the logits; equal ones: the lower index first), w = p of these,
 *   divided by their sum if `renorm` is not 0;   out = sum_j w_j down_e(j) (silu(gate_e(j) x) * (up_e(j) x)).
 * p, p + d_bias and w are formed in 64 bits (a logit more than 745 below the row's largest makes a p of 0), w is rounded to fp32; with
 * `renorm` w is right however small the chosen experts' p are.
 * d_logits [n_rows][n_expert] are fp32, d_bias [n_expert]. d_x and d_out are [n_rows][n_embd] of `type`, rows *_stride apart: Z2H_F32 or
 * Z2H_F16 with F16 experts, Z2H_BF16 with BF16 ones; d_out may be d_x. d_sel and d_weights [n_rows][top_k] (either may be NULL) receive the
 * experts and their w, the first the one with the largest p + bias. An expert whose logit is minus infinity is never taken: -1 and 0
 * stand in the places that remain, and a row without any expert gives zeros. A row with a logit or a sum p + bias that is no number, or
 * with an infinite logit, has no number as its result, and -1 and no number in d_sel and d_weights. top_k is 1 .. min(n_expert, 16).
 * Sums in fp32; fp32 rows meet the weights as two f16 numbers, off by 2^-22 of the largest of 256 neighbours at most, and so do the products
 * silu(..) * .. (three bf16 numbers with bf16 experts, 2^-24 of each). A row that holds a value that is not finite has results that are not
 * finite, and no other row's change. Results do not depend on timing.
 * The workspace (z2h_moe_rows_ws_bytes; 0: the sizes are refused; 256-byte aligned) holds one call at a time: calls and graphs that may
 * overlap need one each. */
#define Z2H_MOE_ROWS_MAX 128
int64_t z2h_moe_rows_ws_bytes(const z2h_experts * experts, int n_rows, int top_k);
int z2h_moe_rows(z2h_ctx * ctx, const z2h_experts * experts, int n_rows, int top_k, int renorm, const float * d_logits,
                 const float * d_bias, int type, const void * d_x, int64_t x_stride, void * d_out, int64_t out_stride, int32_t * d_sel,
                 float * d_weights, void * d_ws, int64_t ws_bytes, void * stream);

/* The pages of a paged cache as sequences come, share, grow and go, without a word from the host: the calls below change the page table
 * (`pages->table`, written here) and d_refs [n_pages], which says for every page how many table entries name it (0: free), and copy
 * what has to be copied in all n_layer layers. `pages` describes layer 0; layer L's k and v lie L * layer_stride elements behind (as in
 * z2h_step_paged). A sequence holds the pages that its table row names before the first entry outside [0, n_pages); entries behind
 * that one are not looked at, and -1 is written where a sequence has no page. n_pages is at most 2^22. To begin: every entry -1, every
 * count 0. The workspace (z2h_pages_ws_bytes, n the fork's items; 0: the sizes are refused; 256-byte aligned) holds one call at a time;
 * calls on the same cache follow each other on one stream.
 *
 * z2h_pages_fork: item i makes sequence d_dst[i] the holder of the first d_rows[i] rows of sequence d_src[i], with room for d_room[i] rows.
 * What the destination held is given up. Whole pages of the rows are shared; the rows in the last, partly filled page are copied into a
 * page of its own, so that both sequences may go on; pages for the rest of the room are new (nothing is written to them). With
 * d_src[i] == d_dst[i] the sequence keeps its own rows: it is cut off (0 rows and no room: ended), given room, or both, and its
 * partly filled page is copied only if another sequence names that page too. Rows are clamped to 0 .. what the source holds, the room to rows ..
 * the table's. New pages are the free ones, those that the call's destinations gave up among them, lowest first, in the order of
 * the items and of their entries. d_held[i] (NULL: not told) is the number of rows that the destination now has pages for: the room, or where
 * no page was left, less: the pages up to there. An item whose source or destination is outside [0, n_seq), whose destination an
 * item before it has too, or whose source is not its destination but an item's changes nothing: -1. n is at most 4096.
 *
 * z2h_pages_compact: the pages in use become pages 0 .. n_used - 1: those from n_used on move, in ascending order, to the free ones before, in
 * ascending order. The new table goes to d_table_out [n_seq][table_len] and the new counts to d_refs_out [n_pages] (either may be the old
 * one itself), n_used to d_n_used (NULL: not told). A moved page's old place keeps what it holds. An entry that names a page with a
 * count of 0 becomes -1 or stays. */
int64_t z2h_pages_ws_bytes(z2h_ctx * ctx, const z2h_pages * pages, int n);
int z2h_pages_fork(z2h_ctx * ctx, const z2h_pages * pages, int n_layer, int64_t layer_stride, int32_t * d_refs, int n, const int32_t * d_src,
                   const int32_t * d_dst, const int32_t * d_rows, const int32_t * d_room, int32_t * d_held, void * d_ws, int64_t ws_bytes,
                   void * stream);
int z2h_pages_compact(z2h_ctx * ctx, const z2h_pages * pages, int n_layer, int64_t layer_stride, int32_t * d_refs, int32_t * d_table_out,
                      int32_t * d_refs_out, int32_t * d_n_used, void * d_ws, int64_t ws_bytes, void * stream);

/* The pass of z2h_step_mixed over a paged cache in place of the context's bands: the model's layers with
 * z2h_paged_append, z2h_paged_plan and z2h_paged_attn in them. A prompt that sequences share is stored once and read
 * once per pass, and a sequence may bring any number of rows: a chunk of its prompt, one frame, or a frame and the
 * drafts behind it, whose logits z2h_verify then judges.
 *
 * `pages` describes layer 0 (Z2H_F16, the model's n_head_kv and head_dim; n_seq and table_len as the caller likes);
 * layer L's k and v lie L * layer_stride elements behind (a multiple of 8, at least n_pages * page_stride), the page
 * table is the same for all layers and stays as it is during the call. row_start [n_seq + 1], kv_len [n_seq],
 * group_start [n_group + 1] and prefix_len [n_group] are on the host and mean what they do in z2h_paged_plan, with
 * row_start[n_seq] = n_rows: sequence s's m rows become its cache rows kv_len[s] - m .. kv_len[s] - 1, row j of them
 * attends to rows [0, kv_len[s] - m + j], of this pass or earlier ones. Only a group's first sequence may bring rows
 * of the group's prefix. No two sequences' rows may lie in the same cache row.
 *
 * ids, emb_map, emb, n_emb, n_out and out_rows are those of z2h_step_mixed. The logits of the n_out rows go to
 * d_logits (device, [n_out][n_codebooks][audio_vocab]; NULL: the context's own buffer) and, if out_logits is not NULL,
 * to the host. d_ws is a workspace of z2h_step_paged_ws_bytes (0: refused, see z2h_last_error; 256-byte aligned). The
 * call works on the context's stream and returns when it is done; work of other streams on the cache has to be done
 * before. Not while a debug capture is on; a profiling window leaves out the paged operators' launches. */
int64_t z2h_step_paged_ws_bytes(z2h_ctx * ctx, const z2h_pages * pages, int n_rows, int n_group);
int z2h_step_paged(z2h_ctx * ctx, const z2h_pages * pages, int64_t layer_stride, int n_rows, const int32_t * row_start,
                   const int32_t * kv_len, int n_group, const int32_t * group_start, const int32_t * prefix_len,
                   const int32_t * ids, const int32_t * emb_map, const float * emb, int n_emb, int n_out,
                   const int32_t * out_rows, float * out_logits, float * d_logits, void * d_ws, int64_t ws_bytes);

/* Debug capture of per-layer intermediates of the following steps (off by default). */
enum {
    Z2H_CAP_RES_IN = 0, Z2H_CAP_ATTN_IN, Z2H_CAP_Q, Z2H_CAP_K, Z2H_CAP_V, Z2H_CAP_GATE, Z2H_CAP_ATTN_O,
    Z2H_CAP_ATTN_OUT, Z2H_CAP_FFN_IN, Z2H_CAP_ROUTER_STATE, Z2H_CAP_ROUTER_LOGITS, Z2H_CAP_PROBS,
    Z2H_CAP_SEL, Z2H_CAP_WEIGHTS, Z2H_CAP_FFN_OUT, Z2H_CAP_OUT_NORM, Z2H_CAP_COUNTS, Z2H_CAP_OFFSETS,
    Z2H_CAP_PERM, Z2H_CAP_EXPERT_OUT, Z2H_CAP_COUNT_
};
int z2h_set_capture(z2h_ctx * ctx, int enable);
/* Copy capture `what` of `layer` (ignored for OUT_NORM) from the last step / moe_forward into host.
 * Sizes: see z2h_capture_bytes. SEL and WEIGHTS hold the layer's [n_tokens][top_k of that layer]
 * rows at the start of a buffer sized for the model's largest top-k. */
int64_t z2h_capture_bytes(z2h_ctx * ctx, int what, int n_tokens);
int z2h_read_capture(z2h_ctx * ctx, int layer, int what, void * host, size_t nbytes);

/* Replay each step from a HIP graph captured once per (batch width, id/embedding input) pair
 * (default on; the counterpart of the reference's CUDA-graph replay of its decode-graph ladder,
 * CMakeLists.txt:34, src/zonos2-graph.cpp:670-680). Steps with capture or profiling run eagerly. */
int z2h_set_graphs(z2h_ctx * ctx, int enable);

/* Per-kernel-family timing with HIP events recorded around every launch on the context's stream
 * (the reference's only equivalent is the ZONOS2_PROFILE_STEP phase split, src/zonos2-graph.cpp:768,
 * 815-829). Between begin and end every launch is bracketed by an event pair; end synchronizes and
 * writes the summed milliseconds and launch counts per family. Up to 16384 launches per window. */
enum {
    Z2H_KF_RESNORM = 0, Z2H_KF_GEMV_QKV, Z2H_KF_QKV_POST, Z2H_KF_ATTN, Z2H_KF_ATTN_COMBINE, Z2H_KF_GEMV_WO,
    Z2H_KF_ROUTER_DOWN, Z2H_KF_ROUTER_TAIL, Z2H_KF_GEMV_GATEUP, Z2H_KF_GEMV_DOWN, Z2H_KF_GEMV_DENSE,
    Z2H_KF_GEMV_HEAD, Z2H_KF_SWIGLU, Z2H_KF_COUNT_
};
int z2h_profile_begin(z2h_ctx * ctx);
int z2h_profile_end(z2h_ctx * ctx, double * ms, int32_t * launches);

/* Device memory held by weights (the shared model), KV cache and scratch (bytes). */
int64_t z2h_device_bytes(const z2h_ctx * ctx, int what /* 0 weights, 1 kv, 2 scratch */);

/* Message of the context's last failure. */
const char * z2h_last_error(const z2h_ctx * ctx);
void z2h_destroy(z2h_ctx * ctx);

#ifdef __cplusplus
}
#endif
#endif /* Z2H_H */
