/*
 * omg_hip.h -- C ABI of the MI355X decision-path engine.
 *
 * This is the drop-in boundary for the reference's omg-wgpu engine surface
 * (bokuweb/grande, crates/omg-wgpu): load a checkpoint, run
 * forward(state, branches) as one block-causal pass, read out rows at the
 * wanted positions, and keep / serialise / restore the state's f16 K/V.
 * Each entry point names the reference item it replaces (path:line in the
 * reference checkout).
 *
 * Conventions
 *   - Opaque handles; plain pointers and sizes; no exceptions cross.
 *   - Status: 0 = ok, negative = error class (OMG_E_*); omg_last_error()
 *     returns the calling thread's last message (the reference's anyhow
 *     strings, engine.rs:1503-1581).  Functions returning a handle return
 *     NULL on failure.
 *   - One engine is not thread-safe; callers serialise (the reference's
 *     server gives the engine one thread, omg-server/src/lib.rs:57-99).
 *   - Token ids are uint32 in the checkpoint's vocabulary.
 */
#ifndef OMG_HIP_H
#define OMG_HIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define OMG_OK 0
#define OMG_E_INVALID (-1)  /* bad argument or request */
#define OMG_E_CAPACITY (-2) /* capacity / max_rows / 4095-branch limits */
#define OMG_E_DEVICE (-3)   /* HIP runtime failure */
#define OMG_E_STATE (-4)    /* state bytes rejected */
#define OMG_E_IO (-5)       /* file system */
#define OMG_E_MISSING (-6)  /* tensors missing at finish */

/* model.rs:337-371 Dtype (codes = Dtype::code) */
#define OMG_DTYPE_F16 0
#define OMG_DTYPE_Q8 1
#define OMG_DTYPE_Q4 2

/* omg-core backend.rs:14-20 Want.  OMG_WANT_LABELS and OMG_WANT_LABELS_LSE
 * have no counterpart in the reference, whose Readout::distribution
 * (readout.rs:124-146) reads the full logits row on the host to pick the
 * label columns and take log_sum_exp (math.rs:13-17) for candidate_mass:
 *   LABELS      k floats per row: the logits of the given label ids;
 *   LABELS_LSE  k + 1 floats per row: the same k logits, then the
 *               log-sum-exp of the row over the whole vocabulary (f32), so
 *               candidate_mass = exp(lse(labels) - row[k]) needs no
 *               vocabulary-wide readback. */
#define OMG_WANT_LOGITS 0
#define OMG_WANT_HIDDEN 1
#define OMG_WANT_LABELS 2
#define OMG_WANT_LABELS_LSE 3

/* omg-core backend.rs:92-104 PrefixSource (0 = none yet) */
#define OMG_SRC_NONE 0
#define OMG_SRC_RESIDENT 1
#define OMG_SRC_RAM 2
#define OMG_SRC_DISK 3
#define OMG_SRC_DECODED 4

typedef struct omg_engine omg_engine;
typedef struct omg_builder omg_builder;

/* omg-core backend.rs:22-30 BranchTokens: tokens + ascending wanted indices. */
typedef struct {
    const uint32_t *tokens;
    size_t ntokens;
    const uint32_t *want;
    size_t nwant;
} omg_branch;

/* omg-core backend.rs:38-45 / engine.rs:26-38 Group. */
typedef struct {
    const uint32_t *prefix;
    size_t prefix_len;
    const omg_branch *branches;
    size_t nbranches;
} omg_group;

/* The Backend facts callers read: n_embd / n_vocab / bos (backend.rs:124-128)
 * and the shape the engine was built for (model.rs:27-63). */
typedef struct {
    uint32_t vocab, d, layers, heads, kv_heads, head_dim, bos;
    uint64_t capacity, max_rows;
} omg_config_t;

/* Thread-local message of the last failure on this thread. */
const char *omg_last_error(void);

/* ---- loading (engine.rs:763-1335, backend.rs:28-71) ---- */

/* EngineBuilder::new(Config::from_json(config.json)) (engine.rs:845-869). */
omg_builder *omg_builder_new(const char *config_json);
/* EngineBuilder::push (engine.rs:888-933): one catalogued tensor, encoded as
 * model.rs QTensor (payload + f16 block scales for Q8/Q4). */
int omg_builder_push(omg_builder *b, const char *name, int dtype, const int64_t *shape, size_t ndim,
                     const void *data, size_t nbytes, const void *scales, size_t nscale_bytes);
/* A host checkpoint (model.rs:540-546 Weights): the seeded random weights
 * of tests/reference.rs:106-139 for a config (linears in `linear_dtype`,
 * the embedding in `embed_dtype`), or an exported directory
 * (model.rs:742-795).  Tensors are in the reference's QTensor encoding;
 * omg_weights_get hands out borrowed pointers valid until omg_weights_free. */
typedef struct omg_weights omg_weights;
omg_weights *omg_synth(const char *config_json, uint64_t seed, int linear_dtype, int embed_dtype);
omg_weights *omg_load_dir(const char *dir);
size_t omg_weights_count(const omg_weights *w);
int omg_weights_get(const omg_weights *w, size_t i, const char **name, int *dtype, int64_t *shape,
                    size_t *ndim, const uint8_t **data, size_t *nbytes, const uint8_t **scales,
                    size_t *nscale_bytes);
void omg_weights_free(omg_weights *w);
/* A llama.cpp GGUF file (v2/v3, gemma3) read directly: the metadata and
 * tensor mapping of tools/export_wgpu_gguf.py:112-296 (q / k / v fused per
 * layer, Q8_0 / Q4_0 blocks split into codes and scales, f32 / bf16 to
 * f16).  The reference reaches a GGUF through that export step; this reads
 * the file itself. */
omg_weights *omg_load_gguf(const char *path);
/* Engine::new's loop over the catalogue (engine.rs:1341-1351). */
int omg_builder_push_weights(omg_builder *b, const omg_weights *w);
/* EngineBuilder::missing (engine.rs:875-885): newline-separated names into
 * buf; returns how many are missing. */
size_t omg_builder_missing(omg_builder *b, char *buf, size_t len);
/* EngineBuilder::finish (engine.rs:952-1334).  Consumes the builder even on
 * failure. */
omg_engine *omg_builder_finish(omg_builder *b, size_t capacity, size_t max_rows);
void omg_builder_free(omg_builder *b);
/* WgpuBackend::load for an exported directory: config.json + manifest.json
 * + *.bin (backend.rs:28-71, model.rs:742-795). */
omg_engine *omg_open_dir(const char *dir, size_t capacity, size_t max_rows);
/* An engine straight from a GGUF file (omg_load_gguf's tensors). */
omg_engine *omg_open_gguf(const char *path, size_t capacity, size_t max_rows);
void omg_close(omg_engine *e);
int omg_config(const omg_engine *e, omg_config_t *out);
/* Engine::warmup (engine.rs:1356-1366). */
int omg_warmup(omg_engine *e);

/* ---- the pass (engine.rs:1386-1940) ---- */

/* Engine::evaluate_groups / Backend::evaluate_many (engine.rs:1404-1444,
 * backend.rs:142-152).  Rows are written densely into `out` in (group,
 * branch, want) order; width n_embd (HIDDEN), n_vocab (LOGITS), nlabels
 * (LABELS, with label_ids) or nlabels + 1 (LABELS_LSE).  prefix_sources (may be NULL) gets one
 * OMG_SRC_* per group. */
int omg_evaluate_groups(omg_engine *e, const omg_group *groups, size_t ngroups, int want,
                        const uint32_t *label_ids, size_t nlabels, float *out, size_t out_floats,
                        int *prefix_sources);
/* Readout::Pointer's head (omg-core readout.rs:17-29, PointerHead): two
 * affine maps d -> dp, weights row-major [dp][d] and biases [dp], f32; the
 * engine keeps a device copy.  w_q = NULL clears it. */
int omg_set_pointer_head(omg_engine *e, size_t d, size_t dp, const float *w_q, const float *b_q,
                         const float *w_k, const float *b_k);
/* The roles of wanted rows for omg_evaluate_pointer (readout.rs Mark). */
#define OMG_ROLE_NONE 0   /* Mark::Last: not scored */
#define OMG_ROLE_OPT 1    /* Mark::OptEnd: an option's `</opt>` row */
#define OMG_ROLE_DECIDE 2 /* Mark::Decide: the `<decide>` row */
/* Readout::distribution's pointer branch (readout.rs:149-173) on the
 * device: omg_evaluate_groups with Want::Hidden whose rows are scored by the
 * pointer head (readout.rs:37-44) instead of read back.  roles: one per
 * wanted row in (group, branch, want) order, each branch with exactly one
 * OMG_ROLE_DECIDE row ("no decide row" otherwise).  out: each branch's
 * option logits (its OMG_ROLE_OPT rows in want order), branch after branch
 * in (group, branch) order; *written (may be NULL) = their count. */
int omg_evaluate_pointer(omg_engine *e, const omg_group *groups, size_t ngroups, const uint8_t *roles,
                         size_t nroles, float *out, size_t out_floats, size_t *written, int *prefix_sources);
/* Engine::evaluate (engine.rs:1386-1396): one group. */
int omg_evaluate(omg_engine *e, const uint32_t *prefix, size_t prefix_len, const omg_branch *branches,
                 size_t nbranches, int want, const uint32_t *label_ids, size_t nlabels, float *out,
                 size_t out_floats);
/* Engine::prefix_source (engine.rs:2158-2161): OMG_SRC_* of the last pass. */
int omg_prefix_source(const omg_engine *e);
/* Engine::is_resident (engine.rs:2152-2156). */
int omg_is_resident(const omg_engine *e, const uint32_t *prefix, size_t n);
/* Engine::evict_resident (engine.rs:2163-2166). */
void omg_evict_resident(omg_engine *e);

/* ---- state (engine.rs:499-641, 1942-2150) ---- */

/* Engine::set_state_cache (engine.rs:1945-1954): RAM LRU of `bytes`, files
 * in `dir` (NULL or "" = none), states tagged with `model_id`. */
int omg_set_state_cache(omg_engine *e, size_t bytes, const char *dir, const char *model_id);
/* Engine::save_state + SavedState::to_bytes (engine.rs:1977-1979, 517-534):
 * the GRWS1 bytes of the prefix at cache rows 0..n; free with
 * omg_free_bytes. */
int omg_save_state(omg_engine *e, const uint32_t *prefix, size_t n, const char *model_id, uint8_t **bytes,
                   size_t *len);
/* SavedState::from_bytes + Engine::restore_state (engine.rs:536-579,
 * 2051-2092): the prefix is resident afterwards. */
int omg_restore_state(omg_engine *e, const uint8_t *bytes, size_t len, const char *model_id);
void omg_free_bytes(uint8_t *p);

/* ---- host-side pieces (no GPU needed) ---- */

/* QTensor::quantize_q8 / quantize_q4 (model.rs:408-466); dtype Q8 or Q4. */
int omg_quantize(int dtype, const float *values, size_t n, uint8_t *data, uint8_t *scales);
/* The packing of Engine::run (engine.rs:1512-1571) with `first` laid out
 * first and its prefix resident when `resident`: ids, meta (4 int32 per
 * token: position, sequence id, first key row, own row + 1) and wanted
 * (4 int64 per row: group, branch, slot, workspace row).  Sizes in/out.
 * align <= 1 gives the reference's layout; align > 1 the engine's own,
 * where every group after the first starts on a multiple of `align` cache
 * rows (padding rows: token 0, sequence id -1), unless that needs more
 * than `rows` rows. */
int omg_pack(const omg_group *groups, size_t ngroups, size_t first, int resident, size_t align, size_t rows,
             uint32_t *ids, int32_t *meta, int64_t *wanted, size_t *n_ids, size_t *n_wanted);
/* state_key (engine.rs:625-641): FNV-1a 64 of model id, 0, prefix. */
uint64_t omg_state_key(const char *model_id, const uint32_t *prefix, size_t n);
/* SavedState::from_bytes (engine.rs:536-579) without an engine: 0 and the
 * prefix length / layer count, or OMG_E_STATE with the reason. */
int omg_state_check(const uint8_t *bytes, size_t len, const char *model_id, size_t *prefix_len,
                    size_t *nlayers);

/* ---- measurement (no counterpart in the reference; bench.py and the
 * kernel tests use them) ---- */

/* Pack + upload one request whose first group's prefix is resident (or not)
 * and keep it for omg_pass_launch, which replays the pass's device work
 * (forward + readout at the wanted rows) on the engine's stream with no host
 * transfer.  omg_sync waits for it.  Any evaluate (omg_evaluate_groups,
 * omg_evaluate_pointer) or omg_restore_state in between uploads over the
 * prepared pass's inputs and cancels it: omg_pass_launch, omg_pass_graph
 * and omg_pass_read then fail with "no prepared pass" until the next
 * omg_pass_prepare. */
int omg_pass_prepare(omg_engine *e, const omg_group *groups, size_t ngroups, int want,
                     const uint32_t *label_ids, size_t nlabels, int first_resident);
int omg_pass_launch(omg_engine *e);
/* No counterpart in the reference (it records one command buffer per
 * request, engine.rs:1761-1861): capture the prepared pass's kernel
 * launches into a HIP graph (on != 0), which omg_pass_launch then replays
 * as one submission; on = 0, the next omg_pass_prepare or any evaluate
 * drops it. */
int omg_pass_graph(omg_engine *e, int on);
/* The prepared pass's rows after its launches (waits for them), in wanted
 * order (group, branch, slot), width as omg_evaluate_groups gives them. */
int omg_pass_read(omg_engine *e, float *out, size_t out_floats, size_t *written);
int omg_sync(omg_engine *e);
/* HIP-event time per kernel of every launch while on; the report is lines
 * "name launches total_ms". */
int omg_profile(omg_engine *e, int on);
size_t omg_profile_report(omg_engine *e, char *buf, size_t len);
/* No counterpart in the reference, whose pass runs every layer for every
 * row (engine.rs:1674-1751).  By default, from the last layer that writes
 * K/V (the model's last layer, or with Gemma 4's K/V-sharing layers the
 * last layer before them) past its attention, the pass runs for the rows a
 * request reads out only: that layer's attention for the query tiles that
 * hold them, then o, norms, gate/up, down and the per-layer block on the
 * gathered rows, and every later layer on those rows alone (its keys and
 * values are an earlier layer's cache, so no other row reaches them).
 * Every K/V cache is still written for every row.  on != 0 runs every
 * layer for every row as the reference does.  The rows a pass returns are
 * the same bits either way.  From the next pass on. */
int omg_set_full_last_layer(omg_engine *e, int on);

/* Kernel-level entry points on device pointers (the reference's matmul.rs
 * kernel tests): a weight uploaded in the device layout, then
 * Y[m][N] = f16(X)[m][K] . W^T (f32) or act = gelu(X.Wg^T) * (X.Wu^T)
 * (f16).  stream NULL = the null stream. */
typedef struct omg_weight omg_weight;
omg_weight *omg_weight_upload(int dtype, int64_t rows, int64_t cols, const void *data, const void *scales);
void omg_weight_free(omg_weight *w);
int omg_dev_gemm(const omg_weight *w, const void *x_f16, int64_t ldx, int64_t m, float *y, int64_t ldy,
                 void *stream);
int omg_dev_gemm_geglu(const omg_weight *wg, const omg_weight *wu, const void *x_f16, int64_t ldx, int64_t m,
                       void *act_f16, int64_t ldact, void *stream);
/* The label readout on device pointers (logits.wgsl's product, then what
 * readout.rs:124-146 takes from the row): rows f32 [nrows][d] times the
 * embedding `embed` [vocab][d] in f32, softcap applied when > 0, then per
 * row the logits of the device-resident label ids and the log-sum-exp of
 * the full vocabulary row: out f32 [nrows][nlabels + 1].  `rows` must be
 * 16-byte aligned.  Label ids must be below vocab; the device-resident ids
 * are not checked before the launch, and an id past the vocabulary gives
 * NaN in its column.  The split rows, the partials and (above 512 labels)
 * the full logits live in scratch device memory: up to 64 MiB kept with the
 * weight from call to call, whatever their streams; a call that finds it in
 * use on another stream, is being captured or needs more allocates and frees
 * its own in stream order. */
int omg_dev_label_readout(const omg_weight *embed, const float *rows, int64_t nrows, const uint32_t *labels,
                          int64_t nlabels, float softcap, float *out, void *stream);
/* No counterpart in the reference.  omg_dev_label_readout for callers that
 * cannot allocate (code under HIP graph capture, tight serving loops):
 * same arguments and results, nothing allocated; its scratch is a fixed
 * 17 MiB device array per GPU, of which 4,194,304 floats must hold
 * nrows * vocab (rounded up to even) + 2 * nrows * ceil(vocab / 64) floats,
 * else OMG_E_CAPACITY.
 * Calls that overlap on one GPU share that array and race. */
int omg_dev_label_readout_noalloc(const omg_weight *embed, const float *rows, int64_t nrows, const uint32_t *labels,
                                  int64_t nlabels, float softcap, float *out, void *stream);
/* The embedding gather + first norm kernel (embed.wgsl + rmsnorm.wgsl):
 * x[t][d] = deq(E[ids[t]]) * scale (f32), hn[t][d] = f16(rmsnorm(x) * w)
 * with w (f32, d entries) already offset.  Device pointers. */
int omg_dev_embed_norm(const omg_weight *embed, const uint32_t *ids, int64_t t, float scale, const float *w,
                       float eps, float *x, void *hn_f16, void *stream);

/* Kernel-level entry points of the encoder path, on device pointers:
 * the gated GEMM with the exact (erf) GELU (matmul_gated.wgsl GELU_ERF = 1);
 * Y = f16(max(X.W^T + bias, 0)) (matmul.wgsl then bias_act.wgsl mode 1);
 * the fused [q | k | v] projection scattered per 64-wide head as f16 with
 * bias, RoPE from `rope` ([pos][32] (cos, sin) pairs; NULL = none, then
 * `meta` may be NULL) and the q scale (rope_bi.wgsl): q16 / k16
 * [heads][tpad][64], vt [heads][tpad/32][64][32] with key k of a tile at
 * column 8*((k%16)/4) + 4*(k/16) + k%4; and the bidirectional attention
 * over those arrays (attention_bi.wgsl): out [t][heads*64] f16. */
int omg_dev_gemm_geglu_erf(const omg_weight *wg, const omg_weight *wu, const void *x_f16, int64_t ldx, int64_t m,
                           void *act_f16, int64_t ldact, void *stream);
int omg_dev_gemm_bias_relu(const omg_weight *w, const void *x_f16, int64_t ldx, int64_t m, const void *bias_f16,
                           void *y_f16, int64_t ldy, void *stream);
int omg_dev_qkv_heads(const omg_weight *w, const void *x_f16, int64_t ldx, int64_t m, const void *bias_f16,
                      const float *rope, const int32_t *meta, float qscale, int64_t tpad, void *q16, void *k16,
                      void *vt, void *stream);
int omg_dev_attention_bi(const void *q16, const void *k16, const void *vt, const int32_t *meta, int heads, int64_t t,
                         int64_t tpad, int window, void *out_f16, void *stream);

/* ---- carrying answers on token by token (no counterpart in the reference,
 * whose answers are read at given positions) ----
 * A paged K/V cache, the append that fills it and the attention that reads
 * it, on device pointers, asynchronous on `stream` (NULL = the null stream)
 * of the current device, which holds the buffers.  Nothing is allocated and
 * nothing is kept between calls: every call can be captured into a HIP
 * graph.  Element types of matrices and caches: */
#define OMG_ELEM_F16 0
#define OMG_ELEM_BF16 1
#define OMG_ELEM_F32 2 /* sources and logits only, not caches */

/* A pool of pages of K/V rows: row r (0 <= r < page) of KV head g on page p
 * at element p * page_stride + (g * page + r) * head_dim of `k` and of `v`.
 * head_dim 64, 128, 256 or 512; page 16, 32, 64, 128 or 256 rows;
 * page_stride 0 = kv_heads * page * head_dim, else at least that and a
 * multiple of 8; k and v 16-byte aligned. */
typedef struct {
    int dtype; /* OMG_ELEM_F16 or OMG_ELEM_BF16 */
    int kv_heads, head_dim, page;
    int64_t npages, page_stride;
    void *k, *v;
} omg_paged_kv;

/* A batch of sequences with t new tokens in all, as int32 device arrays:
 * sequence s has the token rows [start[s], start[s + 1]) (start NULL: row s,
 * then t = nseq) and, these included, lens[s] rows of its own in the cache;
 * row i is row i % page of page table[s * table_ld + i / page], for
 * i / page < max_pages (max_pages * page and prefix_len below 2^30, nseq up
 * to 2^20, t up to 2^24).  Its new tokens are the last of its rows.  All
 * sequences follow a shared prefix of prefix_len rows on the pages
 * prefix_table[i / page] (prefix_len 0: none): row i of a sequence has the
 * position prefix_len + i.
 *
 * The device arrays are not checked before the launch.  What they name
 * outside their arrays is left out: keys on a page outside [0, npages) or
 * past max_pages are seen by no query and written by no append, and token
 * rows that no sequence has (rows behind the last sequence's) leave their
 * outputs as they were.  start must not descend.  Two sequences may share
 * pages; a cache row that two tokens of one append name is left with the
 * elements of either. */
typedef struct {
    int64_t nseq, t;
    const int32_t *lens, *table;
    int64_t table_ld, max_pages;
    const int32_t *start;        /* [nseq + 1] or NULL */
    const int32_t *prefix_table; /* [ceil(prefix_len / page)] */
    int64_t prefix_len;
} omg_paged_batch;

/* What an append takes its rows from: for token row i, head h and column c
 * element i * ld + h * head_dim + c of q (heads of them; NULL: no queries)
 * and i * ldkv + h * head_dim + c of k and v (kv_heads of them; both NULL:
 * no keys and values, a layer that reads another's cache).  Pointers 16-byte
 * aligned, ld and ldkv whole 16 bytes. */
#define OMG_ROPE_HALF 0        /* pairs (i, i + rope_dims / 2), i < rope_dims / 2 */
#define OMG_ROPE_INTERLEAVED 1 /* pairs (2 i, 2 i + 1) */
#define OMG_ROPE_HEAD_HALF 2   /* pairs (i, i + head_dim / 2), i < rope_dims / 2 */
typedef struct {
    int dtype, heads; /* OMG_ELEM_F32, or the cache's type */
    const void *q, *k, *v;
    int64_t ld, ldkv;
    const float *rope; /* [rope_rows][rope_dims / 2] (cos, sin) pairs; NULL: no rotation */
    int64_t rope_rows;
    int rope_dims, rope_layout;  /* rope_dims a multiple of 16, at most head_dim */
    const int32_t *positions;    /* [t] rows of the table; NULL: the tokens' positions */
    const float *q_norm, *k_norm; /* [head_dim] RMS norm weights (any offset included); NULL: no norm */
    int v_norm;                  /* != 0: v rows normed, without weights */
    float eps, q_scale;
} omg_kv_source;

/* Per token: q heads normed, rotated, times q_scale into q_out (row stride
 * ldq elements, a multiple of 8; the cache's type); k heads normed and
 * rotated and v heads (normed) into the token's cache row.  f32 arithmetic,
 * one rounding.  Positions outside the table count as its first or last
 * row.  q_out may be the source's own q rows where type and stride are the
 * same. */
int omg_dev_kv_append(const omg_paged_kv *kv, const omg_paged_batch *b, const omg_kv_source *src, void *q_out,
                      int64_t ldq, void *stream);

/* Attention of the batch's token rows (`heads` query heads, heads a multiple
 * of kv_heads, t * heads below 2^26; row i, head h at q + i * ldq + h * head_dim) over the cache:
 * a token sees the whole shared prefix and its sequence's own rows up to its
 * own, of these (window > 0) the ones less than `window` positions back.
 *   out = softmax(scale * q . k) v, lse = log(sum exp(scale * q . k))
 * out (row stride ldo) has the cache's type, lse [t][heads] f32 (may be
 * NULL); a token that sees no key gets zeros and -infinity.  The prefix's
 * keys and values are read once for a tile of query rows, whatever
 * sequences these belong to.  What stands in cache rows that a token does
 * not see, infinities and NaN among it, does not reach the token.  (Where a
 * value is infinite or NaN, or a sum of bf16 values passes f32's largest, the
 * rows that meet it take all their keys again one by one: right, and some
 * hundred times slower.)  A window saves the keys outside it; the work is
 * shared out as without one.
 * scale positive; q and out 16-byte aligned and apart, ldq and ldo multiples
 * of 8.  f32 sums; the softmax's probabilities are rounded to the cache's type
 * for their product with the values, not in their sum: equal values come out
 * within half a step.  A mean of finite values is finite.
 *
 * workspace: omg_dev_attention_shared_workspace bytes (a function of the
 * shapes alone: nseq, t, max_pages, prefix_len, heads and the cache's;
 * negative: an OMG_E_* status), 16-byte aligned, this call's own until it
 * has run. */
int64_t omg_dev_attention_shared_workspace(const omg_paged_kv *kv, const omg_paged_batch *b, int heads);
int omg_dev_attention_shared(const omg_paged_kv *kv, const omg_paged_batch *b, int heads, const void *q, int64_t ldq,
                             void *out, int64_t ldo, float *lse, float scale, int window, void *workspace,
                             size_t workspace_bytes, void *stream);

/* The same for drafted tokens: of its sequence's new rows a token sees not
 * those up to its own but those whose bits are set in its mask, bit j % 32 of
 * word mask[i * mask_ld + j / 32] for token row i and the j-th new token of
 * its sequence (the token itself has a bit like any other; new tokens past
 * the words are not seen).  For a tree the bits are the token's ancestors and
 * itself.  Its sequence's rows before the new ones and the prefix it sees
 * whole or, with a window > 0, as far as they lie less than `window`
 * positions before positions[i] (device int32 [t], the rows that an append
 * takes from its table; may be NULL without a window); the window leaves the
 * new rows to the masks.  mask_ld 1 to 2^20. */
int64_t omg_dev_attention_tree_workspace(const omg_paged_kv *kv, const omg_paged_batch *b, int heads);
int omg_dev_attention_tree(const omg_paged_kv *kv, const omg_paged_batch *b, int heads, const void *q, int64_t ldq,
                           void *out, int64_t ldo, float *lse, float scale, const uint32_t *mask, int64_t mask_ld,
                           int window, const int32_t *positions, void *workspace, size_t workspace_bytes,
                           void *stream);

/* Attention over few blocks, a block being a page of the cache.  means
 * [npages][kv_heads][head_dim] (f32, 16-byte aligned) are the mean keys of the
 * pages; omg_dev_block_means sets those of the pages that the batch's new rows
 * are on, over the rows up to lens[s] (64-bit sums, one rounding), and leaves
 * the others: one call behind each append keeps them, the prefix's by the call
 * that made it as a sequence of its own.  So does one behind rows that move: of
 * a draft closed up by omg_dev_kv_keep the draft's batch with the lengths that
 * are left, of an eviction one whose new rows are all that stay.
 *
 * A token's blocks are numbered through the prefix's pages, then its sequence's
 * own ones; score = sum over a KV head's query heads of q . mean (64-bit sums,
 * rounded to f32).  For each token and KV head the block of the token's own
 * row and, of those before it, the blocks - 1 of the highest score are chosen
 * (ties: the first ones; NaN lowest; all, where there are no more), and
 *   out, lse = omg_dev_attention_shared's over their rows
 * up to the token's own.  chosen [t][kv_heads][blocks] (int32, may be NULL)
 * gets the numbers, ascending, -1 behind the last.  A page outside the pool has
 * the score 0 and no rows.  There is no window.  blocks 1 to 4096; alignments,
 * strides, sizes, scale, numbers and workspace as there. */
int omg_dev_block_means(const omg_paged_kv *kv, const omg_paged_batch *b, float *means, void *stream);
int64_t omg_dev_attention_blocks_workspace(const omg_paged_kv *kv, const omg_paged_batch *b, int heads, int64_t blocks);
int omg_dev_attention_blocks(const omg_paged_kv *kv, const omg_paged_batch *b, int heads, const void *q, int64_t ldq,
                             void *out, int64_t ldo, float *lse, float scale, const float *means, int64_t blocks,
                             int32_t *chosen, void *workspace, size_t workspace_bytes, void *stream);

/* The attention weight that the batch's tokens give each own row of their
 * sequences, added to what it has gathered before:
 *   weights[(s * kv_heads + h) * ldw + i] += sum exp(scale * q . k_i - lse)
 * over the tokens of sequence s that see its row i (as omg_dev_attention_shared
 * lets them, window included) and the query heads of KV head h; lse [t][heads]
 * is what that call gave (its prefix keys in it; minus infinity: a token that
 * sees nothing).  f32 sums in an order that the shapes fix.  A row's weight
 * hears from its own key alone, infinite and NaN ones too (a key whose scores
 * hold these may take its tokens again one by one: right, and slower); rows from
 * lens[s] on and on pages outside the pool keep theirs.  ldw at least max_pages * page.
 * Sizes, scale and workspace as there; ldq at most 2^24.  The launch is made for
 * sequences with about alike numbers of tokens: a prompt's call of its own is many
 * times faster than one with single tokens' sequences. */
int64_t omg_dev_attention_weights_workspace(const omg_paged_kv *kv, const omg_paged_batch *b, int heads);
int omg_dev_attention_weights(const omg_paged_kv *kv, const omg_paged_batch *b, int heads, const void *q, int64_t ldq,
                              const float *lse, float scale, int window, float *weights, int64_t ldw, void *workspace,
                              size_t workspace_bytes, void *stream);

/* Rows that stay: row first[s] + j of sequence s (first NULL: row j) becomes
 * what its row rows[j] was, K and V, for j < count; `rows` (int32, device) holds
 * a list per sequence, rows_ld apart, for all its KV heads, or per_head != 0 a
 * list per sequence and KV head, list s * kv_heads + h.  So an accepted path of
 * drafted tokens closes up (first: the rows before the draft), or what an
 * eviction leaves moves down.
 *   to_table NULL: in place.  No row stands before its new place (rows[j] >=
 * first[s] + j, as in every list that ascends; one that does is left out).
 * Pages with rows that move belong to one sequence.
 *   to_table [nseq][to_ld]: the pages of the new rows, none of which any
 * sequence's list is read from; rows in any order, also twice.
 * Entries below zero or past the table, and rows on pages outside the pool,
 * move nothing.  Of the batch nseq, the table and its sizes count; its lengths
 * stay as they are.  count at most max_pages * page. */
int omg_dev_kv_keep(const omg_paged_kv *kv, const omg_paged_batch *b, const int32_t *rows, int64_t rows_ld,
                    int64_t count, const int32_t *first, int per_head, const int32_t *to_table, int64_t to_ld,
                    void *stream);

/* Eviction by weight: of the n = lens[s] own rows (as far as the table reaches)
 * of each sequence and KV head
 * `keep` stay (all, where n is no more), the `recent` last ones and of the
 * others those of the largest weights[(s * kv_heads + h) * ldw + i] (ties: the
 * first rows; NaN lowest), in their order.  rows [nseq][kv_heads][keep]
 * (int32) gets their numbers, -1 behind the last; kept (lists kept_ld apart;
 * NULL: the weights themselves) their weights and zeros for the other rows, up
 * to n or kept_ld; K and V move as omg_dev_kv_keep moves them, in place or to
 * the pages of to_table (then all that stays moves, also of short sequences).
 * The caller's lengths become min(n, keep), its new tokens' positions go on
 * from where they were (omg_kv_source.positions), and a window, which counts
 * rows, no longer counts positions.  keep at most max_pages * page, ldw at least that. */
int omg_dev_kv_evict(const omg_paged_kv *kv, const omg_paged_batch *b, int64_t keep, int64_t recent, float *weights,
                     int64_t ldw, int32_t *rows, float *kept, int64_t kept_ld, const int32_t *to_table, int64_t to_ld,
                     void *stream);

/* The next token of each row of logits (row r, token i at logits[r * ld + i];
 * dtype OMG_ELEM_F32, F16 or BF16; any ld from vocab up), drawn with the
 * given random number u[r] in [0, 1).  With z the row, M its maximum and
 * w_i = exp((z_i - M) / temperature):
 *   1. top_k: the k largest z stay (ties: the lowest indexes first);
 *   2. top_p: of these, largest first, a token stays while the mass before
 *      it is under top_p times the mass of all of step 1 (the first always);
 *   3. min_p: of these, tokens with w_i >= min_p stay (the largest always);
 *   4. the token is the first kept one, in index order, whose running mass
 *      exceeds u times the mass of all kept tokens.
 * logprob (may be NULL) is log(w_token / mass of the kept).  Each parameter
 * is a device array of a value per row, or NULL (off): temperature (NULL:
 * 1; <= 0 or NaN: the first largest z, logprob 0), top_k (<= 0: off), top_p
 * (>= 1 or NaN: off), min_p (<= 0 or NaN: off).  u outside [0, 1) counts as
 * the nearest inside, NaN as 0.
 * Masked tokens are -infinity or NaN and are never drawn; a row with nothing
 * else gives token -1 and logprob -infinity.  Masses are sums of w rounded
 * to 2^-42 (the whole mass of a row of more than 32,768 tokens: sums of w in
 * 64 bits), so a token under 2^-43 of the largest is not drawn, and the same
 * call gives the same tokens.
 * vocab up to 2^20, rows to 2^21.  workspace: omg_dev_sample_workspace bytes (negative: an
 * OMG_E_* status; 0 for rows of up to 32,768 tokens), 16-byte aligned, this
 * call's own until it has run. */
int64_t omg_dev_sample_workspace(int64_t rows, int64_t vocab);
typedef struct {
    int dtype;
    int64_t rows, vocab, ld;
    const void *logits;
    const float *u;
    const float *temperature;
    const int32_t *top_k;
    const float *top_p, *min_p;
    int32_t *tokens;
    float *logprob;
} omg_sample_args;
int omg_dev_sample(const omg_sample_args *a, void *workspace, size_t workspace_bytes, void *stream);

/* ---- the bidirectional encoder path (crates/omg-wgpu/src/laya.rs) ----
 * An mmBERT / ModernBERT encoder with Laya's decision head: every question
 * is one sequence; a request's sequences run as one packed pass isolated by
 * the attention mask; the scorer and the act head read the [CLS] and [MASK]
 * rows on the device. */
typedef struct omg_laya omg_laya;
typedef struct omg_laya_builder omg_laya_builder;

/* laya.rs:468-476 Sequence: token ids, the token index of each option's
 * [MASK] (option order), question type (0 choice, 1 score, 2 noul). */
typedef struct {
    const uint32_t *ids;
    size_t nids;
    const uint32_t *markers;
    size_t nmarkers;
    int qtype;
} omg_laya_seq;

typedef struct {
    uint32_t vocab, d, layers, heads, ff, head_layers, act_out, max_len;
    uint32_t cls, sep, mask, pad;
    uint64_t capacity, max_rows;
} omg_laya_config_t;

/* LayaBuilder::new(config_from_export(config.json)) (laya.rs:312-323,
 * 623-645): the encoder config.json with the agent config under
 * "laya_agent" and the special token ids under "laya_tokens"
 * ({"cls_token": id, ...}; the reference resolves surface forms with its
 * tokenizer, which stays on the caller's side). */
omg_laya_builder *omg_laya_builder_new(const char *config_json);
/* LayaBuilder::push (laya.rs:662-709). */
int omg_laya_builder_push(omg_laya_builder *b, const char *name, int dtype, const int64_t *shape, size_t ndim,
                          const void *data, size_t nbytes, const void *scales, size_t nscale_bytes);
/* LayaEngine::new's loop over the catalogue (laya.rs:1115-1124). */
int omg_laya_builder_push_weights(omg_laya_builder *b, const omg_weights *w);
/* LayaBuilder::missing (laya.rs:651-660). */
size_t omg_laya_builder_missing(omg_laya_builder *b, char *buf, size_t len);
/* LayaBuilder::finish (laya.rs:711-1083); consumes the builder. */
omg_laya *omg_laya_builder_finish(omg_laya_builder *b, size_t capacity, size_t max_rows);
void omg_laya_builder_free(omg_laya_builder *b);
/* Seeded weights for a config (LayaConfig::tensors order, laya.rs:252-305)
 * from the xorshift of tests/reference.rs:17-38: linears U(-1, 1) /
 * sqrt(fan-in), embedding U(-1, 1), type embedding x 0.15, norm weights
 * 1 + U/2, biases U/50; the reference ships no generator for this model. */
omg_weights *omg_laya_synth(const char *config_json, uint64_t seed, int linear_dtype, int embed_dtype);
/* LayaBackend::load for an exported directory (laya/backend.rs:61-91,
 * tools/export_laya.py): config.json (encoder config + laya_agent +
 * laya_tokens), manifest.json, *.bin; the engine is warmed up
 * (laya.rs:1126-1135).  special_ids (cls, sep, mask, pad), when not NULL,
 * replace laya_tokens: the reference resolves their surface forms with
 * the checkpoint's tokenizer, which stays with the caller. */
omg_laya *omg_laya_open_dir(const char *dir, const uint32_t *special_ids, size_t capacity, size_t max_rows);
/* The same directory's tensors as a host checkpoint. */
omg_weights *omg_laya_load_dir(const char *dir, const uint32_t *special_ids);
void omg_laya_close(omg_laya *e);
int omg_laya_config(const omg_laya *e, omg_laya_config_t *out);
/* LayaEngine::warmup (laya.rs:1126-1135). */
int omg_laya_warmup(omg_laya *e);
/* LayaEngine::hidden (laya.rs:1138-1432): per sequence the [CLS] row then
 * each marker's row, d floats each, dense in sequence order. */
int omg_laya_hidden(omg_laya *e, const omg_laya_seq *seqs, size_t n, float *out, size_t out_floats);
/* LayaEngine::evaluate (laya.rs:1435-1485): the scorer's raw logit per
 * marker, dense in sequence order, and the act probability per sequence
 * (NaN without an act head). */
int omg_laya_evaluate(omg_laya *e, const omg_laya_seq *seqs, size_t n, float *logits, size_t nlogits, float *act,
                      size_t nact);
/* LayaConfig::temperature_for (laya.rs:234-248). */
int omg_laya_temperature(const omg_laya *e, int qtype, size_t k, float *out);
/* Measurement, as omg_pass_prepare / omg_pass_launch / omg_sync / omg_profile:
 * a launch is the device work of one omg_laya_evaluate, the forward pass, the
 * scorer and the act head. */
int omg_laya_prepare(omg_laya *e, const omg_laya_seq *seqs, size_t n);
int omg_laya_launch(omg_laya *e);
int omg_laya_sync(omg_laya *e);
int omg_laya_profile(omg_laya *e, int on);
size_t omg_laya_profile_report(omg_laya *e, char *buf, size_t len);
/* No counterpart in the reference, whose head layers run every row
 * (laya.rs:1346-1392).  By default the last decision-head layer runs past
 * its attention for the read-out rows only (o projection, LayerNorm, l1,
 * l2 on the gathered [CLS] and marker rows); on != 0 runs it for every row.
 * The rows are the same bits either way.  From the next pass on. */
int omg_laya_set_full_last_layer(omg_laya *e, int on);

#ifdef __cplusplus
}
#endif
#endif
