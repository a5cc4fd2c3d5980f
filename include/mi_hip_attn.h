/*
 * mi_hip_attn.h -- C ABI of the MI355X (gfx950) batched GQA attention
 * backend for the mini-infer engine.
 *
 * What it replaces: the three CPU graph ops
 *   MI_OP_ATTN_QK   src/ops_cpu.cpp:356-380  (scores  S[i,j,h] = K[:,h/n_rep,i].Q[:,h,j])
 *   MI_OP_SOFTMAX   src/ops_cpu.cpp:304-346  (causal, scaled, per (j,h) row)
 *   MI_OP_ATTN_KQV  src/ops_cpu.cpp:386-410  (O[o,h,j] = sum_t V[o,h/n_rep,t].P[t,j,h])
 * plus the KV cache that feeds them (src/model_qwen2.cpp:557-596, the K/V
 * append CPY nodes of src/model_qwen2.cpp:156-159) and the per-node dispatch
 * point of the executor (src/ops_cpu.cpp:481-530, src/threadpool.cpp:171-180).
 *
 * Conventions
 *   - Every function returns an int status (MI_HIP_OK == 0). It never throws
 *     and never aborts on bad arguments; the message of the last failure on
 *     the calling thread is returned by mi_hip_last_error().
 *   - Layouts are the engine's: Q and O are [head_dim, n_head, n_tokens], the
 *     K and V caches are [head_dim, n_head_kv, n_ctx] per layer, ne[0]
 *     innermost, strides in bytes. Q head h reads KV head h / n_rep: GQA is an
 *     index mapping, no K/V row is ever copied per head.
 *   - Pointers named "device" must be device (HBM) addresses; "host" pointers
 *     are ordinary host memory.
 *   - `stream` is a hipStream_t passed as void*; NULL means the null stream.
 *     Calls enqueue work and return; the caller synchronises the stream.
 */
#ifndef MI_HIP_ATTN_H
#define MI_HIP_ATTN_H

#include <stddef.h>
#include <stdint.h>

#include "mi_tensor.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- status codes ------------------------------------------------------ */
#define MI_HIP_OK 0
#define MI_HIP_E_INVALID 1     /* an argument is out of range or inconsistent */
#define MI_HIP_E_NODEVICE 2    /* no usable gfx950 device */
#define MI_HIP_E_RUNTIME 3     /* a HIP runtime call failed */
#define MI_HIP_E_NOMEM 4       /* device allocation refused (or over the limit) */
#define MI_HIP_E_UNSUPPORTED 5 /* valid request outside what the kernels cover */
#define MI_HIP_E_STATE 6       /* called before mi_hip_init / on a dead object */
#define MI_HIP_E_LOST 7        /* a decode launch lost a record (its group's output is NaN) */

/* ---- library lifetime -------------------------------------------------- */

/* Selects `device` for this library and checks it is gfx950.
 * Counterpart of the engine's one-time setup in mi_kv_cache_init
 * (src/model_qwen2.cpp:557-596); idempotent for the same device. */
int mi_hip_init(int device);

/* Releases library-owned device memory (the default workspace). KV caches
 * and workspaces must have been destroyed by the caller first. */
int mi_hip_shutdown(void);

/* Thread-local text of the last failure ("" if none). */
const char* mi_hip_last_error(void);

/* Writes sizeof(mi_tensor), offsetof(type, ne, nb, op, op_params, src, data,
 * view_src, view_offs, n_children, flags, name, extra) and sizeof(mi_cgraph)
 * into out[0..14] (n >= 15) so a caller can verify it shares the layout of
 * src/tensor.h:122-160 and src/graph.h:19-47. */
int mi_hip_abi_layout(size_t* out, int n);

/* ---- device allocation accounting -------------------------------------- */

/* The engine forbids steady-state allocation (tests/test_zero_alloc.cpp).
 * Every device allocation this library makes goes through one counter. */
typedef struct mi_hip_alloc_stats {
  uint64_t n_malloc;
  uint64_t n_free;
  uint64_t bytes_live;
  uint64_t bytes_peak;
} mi_hip_alloc_stats;

int mi_hip_get_alloc_stats(mi_hip_alloc_stats* out);

/* Caps the library's live device bytes (0 = no cap). An allocation that
 * would exceed the cap fails with MI_HIP_E_NOMEM before calling HIP. */
int mi_hip_set_alloc_limit(uint64_t bytes);

/* ---- decode workspace ---------------------------------------------------- */

/* The split-KV decode kernel's scratch: one partial-result record per
 * workgroup, per-group counters (dynamic sub-tile claims, merge election,
 * arrivals) and status words; and the parts that mi_hip_attn_tree and
 * mi_hip_logits_adjust join. Launches that share a workspace must be
 * ordered (one stream, or synchronised); launches on different workspaces may
 * run concurrently. Every KV cache owns one (mi_hip_kv_workspace); callers
 * that attend over explicit tensors create their own, or fall back to the
 * library's default workspace (created by mi_hip_init, shared by every call
 * that names none). No counterpart in the reference: its CPU kernels need no
 * scratch beyond the graph allocator's arena (src/gallocr.cpp). */
typedef struct mi_hip_workspace mi_hip_workspace;

typedef struct mi_hip_workspace_desc {
  int32_t n_head_kv;  /* KV heads of the problems it serves */
  int32_t n_head;     /* Q heads (multiple of n_head_kv) */
  int32_t head_dim;   /* 64 or 128 */
} mi_hip_workspace_desc;

/* One device allocation covering any decode launch of up to 32 items of this
 * head shape (mi_hip_attn_decode_batch's limit per launch) and, with 17 MB (head_dim
 * 64) or 34 MB of parts, any call of mi_hip_attn_tree, mi_hip_attn_paged and
 * mi_hip_logits_adjust, and those of mi_hip_verify_draft whose scratch (the size is
 * given there) the parts hold. Where the allocation limit or the device has no room
 * for the parts, a workspace (a cache's own and the default one too) is made without
 * them: mi_hip_attn_tree and mi_hip_attn_paged then keep each sequence's keys in one
 * piece, which is slow over long caches, and mi_hip_logits_adjust's ids and
 * mi_hip_verify_draft are refused with it (MI_HIP_E_UNSUPPORTED). */
int mi_hip_workspace_create(const mi_hip_workspace_desc* desc, mi_hip_workspace** out);
int mi_hip_workspace_destroy(mi_hip_workspace* ws);

typedef struct mi_hip_workspace_status {
  uint32_t early_fallbacks; /* early merges whose bounded wait ran out (results still exact) */
  uint32_t lost_groups;     /* groups whose output was set to NaN (never expected) */
} mi_hip_workspace_status;

/* Synchronises `stream`, reports the status words accumulated since the last
 * call and clears them. Returns MI_HIP_E_LOST if any group was lost (its
 * counters are then reset too), MI_HIP_OK otherwise. */
int mi_hip_workspace_check(mi_hip_workspace* ws, void* stream, mi_hip_workspace_status* out);

/* Rounds of polls an early merger makes before it falls back to the
 * last-arriver merge (default 4096). Tuning and tests; 0 makes every early
 * merge fall back. */
int mi_hip_workspace_set_poll_limit(mi_hip_workspace* ws, int32_t rounds);

/* Decode planner knobs (initialised from MI_HIP_DECODE_KPG, _EARLY, _SOLO and
 * _CLAIM at mi_hip_init): kpg > 0 forces that many workgroups per group (0:
 * planned); early = 0 disables the early merge, 1 uses it when every
 * workgroup of a launch fits on the device at once, 2 always; solo: groups
 * that one workgroup's ring covers in at most `solo` rounds get one
 * workgroup; claim: split groups whose waves each stream at least `claim`
 * ring rounds take sub-tiles from device counters (0: never). A negative
 * value keeps the current setting. Tuning and tests; no counterpart in the
 * reference. */
int mi_hip_decode_tuning(int32_t kpg, int32_t early, int32_t solo, int32_t claim);

/* Deterministic fused attention (on = 1, the default): every wave of the
 * decode and prefill kernels takes a fixed share of its workgroup's work, so
 * each output is the same bits on every run with the same inputs and launch
 * shape (the merges across waves and workgroups run in a fixed order). Off
 * (0): each wave takes the next piece of work from a counter, so a wave that
 * memory serves sooner takes more -- about 1% faster on the 24-layer
 * n_kv 4096 decode, with results that differ from run to run in the last
 * bits. Process-wide; takes effect for launches issued afterwards. No
 * counterpart in the reference (its CPU kernels are deterministic by
 * construction: src/ops_cpu.cpp:38-53). */
int mi_hip_set_deterministic(int32_t on);

/* Matrix cores of the prefill kernel's QK and PV products.
 *   MI_HIP_PREFILL_AUTO (the default): MI_HIP_PREFILL_F32 with an F32 cache,
 *     the split form below with an F16 cache (whose f16 products are exact
 *     in the cache operand); within the 1e-4 bar at any score magnitude
 *     either way.
 *   MI_HIP_PREFILL_F32: v_mfma_f32_32x32x2f32 (float products, as the
 *     reference's ops; an F16 cache widened to float), within the 1e-4 bar
 *     at any score magnitude.
 *   MI_HIP_PREFILL_SPLIT_BF16: with an F32 cache every float operand is split
 *     into a pair of bf16 (hi = round(x), lo = round(x - hi),
 *     |x - hi - lo| <= 2^-17 |x|) and each product is lo.hi + hi.lo + hi.hi
 *     on v_mfma_f32_32x32x16_bf16 with float accumulation: ~2^-16 relative
 *     error per product, three bf16 products at 16x the FP32 matrix rate,
 *     within the 1e-4 bar only while scale * |q| * |k| stays small (N(0,1)
 *     inputs with q and k scaled by up to 2). With an F16 cache the cache
 *     operand is used as it is and Q and the probabilities are split into
 *     f16 pairs (~2^-22 relative; a wave whose |q| exceeds 2^14 scales its
 *     queries by a power of two first): two v_mfma_f32_32x32x16_f16 per
 *     product step, within the bar at any score magnitude.
 * Process-wide. No counterpart in the reference. */
#define MI_HIP_PREFILL_F32 0
#define MI_HIP_PREFILL_SPLIT_BF16 1
#define MI_HIP_PREFILL_AUTO 2
int mi_hip_set_prefill_mode(int32_t mode);

/* Products of the decode kernel (one query row per head).
 *   MI_HIP_DECODE_MATRIX: QK and PV on the matrix cores (16x16 MFMAs; head
 *     columns padded to 16). F32 cache operands are split into bf16 pairs as
 *     in MI_HIP_PREFILL_SPLIT_BF16 (lo.hi + hi.lo + hi.hi); an F16 cache is
 *     used as it is, with Q and the probabilities split into f16 pairs (a
 *     head whose |q| exceeds 2^14 is scaled by a power of two first). ~1e-5
 *     relative per product.
 *   MI_HIP_DECODE_VALU: float multiply-adds on the vector units (exact
 *     float products).
 *   MI_HIP_DECODE_STREAM: float multiply-adds on the vector units in the
 *     streaming kernel (K/V straight into registers, each group's parts
 *     merged by the last to arrive), for head_dim 64 or 128 and groups that
 *     span several workgroups; other launches take MI_HIP_DECODE_VALU.
 *   MI_HIP_DECODE_AUTO (the default): the vector units (MI_HIP_DECODE_VALU)
 *     for an F32 cache; for an F16 cache the matrix cores, except for short
 *     launches whose heads can be split between workgroups so that each
 *     wave streams at most about 2 sub-tiles of 16 positions (the split is a
 *     vector-unit form, faster there).
 * The split bf16 pairs of the matrix form carry ~2^-16 relative error per
 * product into the scores, so with an F32 cache it stays within the 1e-4 bar
 * only while scale * |q| * |k| stays small (N(0,1) inputs with q and k
 * scaled by up to 2); the other forms are within it at any magnitude.
 * Process-wide. No counterpart in the reference. */
#define MI_HIP_DECODE_VALU 0
#define MI_HIP_DECODE_MATRIX 1
#define MI_HIP_DECODE_AUTO 2
#define MI_HIP_DECODE_STREAM 3
int mi_hip_set_decode_mode(int32_t mode);

/* ---- device-resident KV cache ------------------------------------------ */

typedef struct mi_hip_kv mi_hip_kv;

/* Cache elements of 8 bits (a cache type only: no tensor of the engine has it).
 * A group of values shares a scale d, the smallest f16 number with
 * 127 d >= max |x|; each value is kept as the int8 nearest to x / d (ties to
 * even) and stands for that many times d, so it is at most d / 2 off. A K row
 * has a group for each 32 dims, a V row is one group. 1.06 and 1.02 to 1.03
 * bytes per value. A group with an infinity or a NaN, or with max |x| above
 * 8319008, reads back as NaN. Everything that takes a cache handle takes one of
 * this type, except mi_hip_attn_fwd_reference_order and
 * mi_hip_attn_decode_batch_noalloc (MI_HIP_E_UNSUPPORTED). mi_hip_kv_view gives
 * the int8 values, mi_hip_kv_scales the scales. No counterpart in the
 * reference. */
#define MI_HIP_TYPE_Q8 100

typedef struct mi_hip_kv_desc {
  int32_t n_layer;
  int32_t n_ctx;
  int32_t n_head_kv;
  int32_t head_dim;  /* 64 or 128 */
  int32_t n_head;    /* Q heads (multiple of n_head_kv); sizes staging */
  int32_t type;      /* MI_TYPE_F32, MI_TYPE_F16 or MI_HIP_TYPE_Q8 cache elements */
} mi_hip_kv_desc;

/* One device allocation holding every layer's K and V as
 * [head_dim, n_head_kv, n_ctx] (position-major, the layout of
 * src/model_qwen2.cpp:564-577), plus the host-node staging buffer (sized for
 * n_ctx) and the cache's own decode workspace (covering a decode launch of up
 * to 32 items of this head shape, and the parts of mi_hip_attn_tree: 17 MB at
 * head_dim 64, 34 MB at 128). Nothing is allocated afterwards.
 * Replaces mi_kv_cache_init's host KV context (src/model_qwen2.cpp:564-577). */
int mi_hip_kv_create(const mi_hip_kv_desc* desc, mi_hip_kv** out);
int mi_hip_kv_destroy(mi_hip_kv* kv);

/* A cache whose n_ctx rows are pages of `page_size` rows (a power of two of at
 * least 16 that divides n_ctx), dealt out to sequences by block tables: row r of a
 * layer is row r % page_size of page r / page_size, and a sequence's position t
 * lies in row table[t / page_size] * page_size + t % page_size. mi_hip_paged_append
 * fills it and mi_hip_attn_paged reads it; mi_hip_kv_write (device sources),
 * mi_hip_kv_read, mi_hip_kv_view and mi_hip_kv_scales take a row where they say
 * position. What reads a cache as one sequence refuses it (MI_HIP_E_UNSUPPORTED):
 * the other attention entry points, mi_hip_rope_append, mi_hip_norm_rope_append,
 * mi_hip_kv_keep and mi_hip_kv_bind. No staging for host nodes; its workspace is
 * for the paged calls (parts of 39 MB at head_dim 64, 77 MB at 128). No counterpart
 * in the reference. */
int mi_hip_kv_create_paged(const mi_hip_kv_desc* desc, int32_t page_size, mi_hip_kv** out);

/* The cache's own decode workspace (owned by the cache; do not destroy). */
int mi_hip_kv_workspace(mi_hip_kv* kv, mi_hip_workspace** out);

/* Device view of one layer's cache: which = 0 for K, 1 for V. Fills the
 * device address and the engine-style ne[4]/nb[4]. */
int mi_hip_kv_view(mi_hip_kv* kv, int layer, int which, void** data, int64_t ne[4],
                   size_t nb[4]);

/* Writes n_tokens F32 rows src[head_dim, n_head_kv, n_tokens] (byte strides
 * src_nb[0..2]) into positions [pos0, pos0 + n_tokens) of layer `layer`'s
 * K (which = 0) or V (which = 1); F16 caches round to nearest even, 8-bit
 * caches quantise each row.
 * src_on_device = 0 for a host source, 1 for a device source.
 * This is the CPY-into-kv_write_view node (src/model_qwen2.cpp:99-103,
 * 156-159; src/ops_cpu.cpp:446-460). Host sources are synchronous. */
int mi_hip_kv_write(mi_hip_kv* kv, int layer, int which, int pos0, int n_tokens,
                    const float* src, const size_t src_nb[3], int src_on_device,
                    void* stream);

/* Device view of the scales of one layer of an 8-bit cache: f16
 * [head_dim / 32, n_head_kv, n_ctx] of K (which = 0), [1, n_head_kv, n_ctx] of
 * V (which = 1). */
int mi_hip_kv_scales(mi_hip_kv* kv, int layer, int which, void** data, int64_t ne[4],
                     size_t nb[4]);

/* Reads positions [pos0, pos0 + n_tokens) of layer `layer`'s K (which = 0) or
 * V (which = 1) into device rows dst[head_dim, n_head_kv, n_tokens] (byte
 * strides dst_nb[0..2]) of type MI_TYPE_F32 or MI_TYPE_F16 (rounded to nearest
 * even). The values are what the attention reads: exact for an F32 dst. No
 * counterpart in the reference. */
int mi_hip_kv_read(mi_hip_kv* kv, int layer, int which, int pos0, int n_tokens, void* dst,
                   int dst_type, const size_t dst_nb[3], void* stream);

/* Keeps the accepted rows of a tree of drafted tokens: row n_past + idx[i]
 * becomes row n_past + i, i < n_idx, of K and V of every layer. idx (host) is
 * strictly increasing, at most 256 rows and at most 32767 behind n_past; rows
 * from n_past + n_idx on keep what they hold. No counterpart in the
 * reference. */
int mi_hip_kv_keep(mi_hip_kv* kv, int n_past, const int32_t* idx, int n_idx, void* stream);

/* Associates the engine's host KV tensor (the persistent leaf whose
 * view_src-flattened views the CPY nodes write through, and which the
 * ATTN_QK/ATTN_KQV nodes read as src[1]) with a layer of `kv`, for
 * mi_hip_compute_forward. Keyed by the tensor's address, never by its
 * `extra` field (the engine's allocator rewrites `extra` every step,
 * src/gallocr.cpp:120-121). */
int mi_hip_kv_bind(mi_hip_kv* kv, int layer, int which, const mi_tensor* host_kv);

/* ---- fused attention ---------------------------------------------------- */

typedef struct mi_hip_attn_args {
  /* K/V source: either a cache + layer (kv != NULL) ... */
  mi_hip_kv* kv;
  int32_t layer;
  /* ... or explicit device tensors [head_dim, n_head_kv, >= n_past+n_tokens]. */
  const void* k;
  const void* v;
  size_t k_nb[3];
  size_t v_nb[3];
  int32_t kv_type;   /* MI_TYPE_F32 / MI_TYPE_F16 (explicit tensors only) */
  int32_t head_dim;  /* explicit tensors only */
  int32_t n_head_kv; /* explicit tensors only */
  /* Queries: device [head_dim, n_head, n_tokens], byte strides q_nb. */
  const float* q;
  size_t q_nb[3];
  /* Output: device [head_dim, n_head, n_tokens], byte strides out_nb. */
  float* out;
  size_t out_nb[3];
  int32_t n_head;
  int32_t n_rep;    /* n_head / n_head_kv (op_params[1] of ATTN_QK) */
  int32_t n_past;   /* keys [0, n_past + j] visible to query j */
  int32_t n_tokens; /* 1 = decode kernel, > 1 = prefill kernel */
  float scale;      /* op_params[1] of SOFTMAX, 1/sqrt(head_dim) in the engine */
  void* stream;
  /* Decode scratch: this workspace if non-NULL, else kv's own, else the
   * library default (read from the first item of a batch). */
  mi_hip_workspace* ws;
} mi_hip_attn_args;

/* The whole ATTN_QK -> causal SOFTMAX -> ATTN_KQV triple in one pass that
 * never materialises scores or probabilities: the split-KV decode kernel when
 * n_tokens == 1, the MFMA prefill kernel otherwise. Equivalent to running
 * mi_compute_attn_qk, mi_compute_softmax and mi_compute_attn_kqv
 * (src/ops_cpu.cpp:304-410) on the nodes built by src/model_qwen2.cpp:169-172,
 * within floating-point tolerance. */
int mi_hip_attn_fwd(const mi_hip_attn_args* args);

/* The same triple in the reference's own operation order, so that the output
 * equals mi_compute_attn_qk -> mi_compute_softmax -> mi_compute_attn_kqv
 * (src/ops_cpu.cpp:304-410) on the nodes of src/model_qwen2.cpp:169-172 BIT
 * FOR BIT, not within tolerance: each score's dot product d ascending with
 * every product and sum rounded, the maximum, the host C library's expf, the
 * sum of the exponentials key by key, the correctly rounded 1 / sum, and each
 * output element's sum over the keys in order. The device engine's
 * MI_HIP_QWEN2_ATTN_REFERENCE_ORDER mode runs it. F32 cache only, head_dim 64
 * or 128, n_past + n_tokens <= 32768 (MI_HIP_E_UNSUPPORTED otherwise). The
 * ordered sums make a row's cost linear in its key count on one lane: a
 * parity path, slower than mi_hip_attn_fwd. */
int mi_hip_attn_fwd_reference_order(const mi_hip_attn_args* args);

/* n_items independent single-token decode problems of one shape (same
 * head_dim, n_head, n_rep, K/V element type; n_past may differ) in ONE
 * launch, e.g. many sequences' caches, or a stack of layers in a benchmark.
 * No counterpart in the reference (it runs one node per layer).
 * Decode launches take a fresh stamp on their workspace from the host at
 * every call, so a call on a stream under graph capture is refused with
 * MI_HIP_E_UNSUPPORTED (a replayed launch would reuse its stamp); the same
 * holds for every decode entry point. */
int mi_hip_attn_decode_batch(const mi_hip_attn_args* items, int n_items, void* stream);

/* mi_hip_attn_decode_batch for callers that cannot allocate device memory
 * (tight serving loops, harnesses that forbid hipMalloc). No counterpart in
 * the reference. Like every decode entry point it is refused on a stream
 * under graph capture. It ignores the items' ws and
 * their caches' workspaces and uses a fixed 4 MB scratch array that each GPU
 * holds from library load until the process ends (at most 128 groups, i.e.
 * items x n_head_kv x head chunks, and records for ~460-900 workgroups); a
 * larger launch fails with MI_HIP_E_UNSUPPORTED. It calls no hipMalloc or
 * hipFree. Every call on one GPU shares that GPU's scratch: calls that
 * overlap on the device (different streams, unsynchronised) race and must
 * not be issued; calls ordered on one stream are safe. */
int mi_hip_attn_decode_batch_noalloc(const mi_hip_attn_args* items, int n_items, void* stream);

/* ---- attention of a tree of drafted tokens ------------------------------ */

/* Which of its own keys each query of an item sees: bit i % 64 of word i / 64
 * of row j is set if query j sees key n_past + i, i < n_tokens (bits past that
 * are not read). Device memory, rows nb bytes apart, 8-byte aligned. bits NULL:
 * query j sees keys n_past + 0 .. n_past + j (a chain). Every query sees the
 * n_past keys before. */
typedef struct mi_hip_tree_mask {
  const uint64_t* bits;
  size_t nb;
} mi_hip_tree_mask;

/* Attention of n_tokens queries per item whose own K/V rows are the cache rows
 * n_past .. n_past + n_tokens - 1 (a tree of drafted tokens appended in one
 * step, a chunk of a prompt, or one token): out_j = softmax over the keys that
 * query j sees of scale q_j.k_t, times v_t. F32, F16 and 8-bit caches; items
 * share the head shape, element type and scale, n_past and n_tokens may differ.
 * masks: one per item, or NULL (every item a chain). A query that sees no key
 * gives zeros, and so does one whose every score is below float's range. What
 * lies in rows that a query does not see never shows in its output, infinities
 * and NaN included; an infinite value in a row that it sees may give NaN for
 * infinity, and so may a score above float's range. Products: an F16 or 8-bit
 * cache's values are taken as they are, queries and probabilities as two f16
 * numbers each (22 bits); an F32 cache's and its queries are float products up to
 * 32 query rows per KV head (n_tokens * n_rep of the largest of up to 32 items
 * launched together), and two f16 numbers on both sides above that (a value at most
 * 2^-22 of itself, 2^-39 of its row's largest, or 2^-124 in V, off). All sums are
 * in float.
 * Scratch for joining the parts of long caches: ws of the first item, else its
 * cache's workspace, else the library default; calls that share one must be
 * ordered. Nothing is kept in it between calls, so unlike the other decode entry
 * points this one may be captured into a graph (pointers, n_past and n_tokens
 * as at the capture; the masks are read at each replay). The same bits on every
 * run. mi_hip_attn_fwd and mi_hip_attn_decode_batch on an 8-bit cache run this.
 * No counterpart in the reference. */
int mi_hip_attn_tree(const mi_hip_attn_args* items, const mi_hip_tree_mask* masks, int n_items,
                     void* stream);

/* ---- many requests over a paged cache -------------------------------------- */

/* A step's block tables, row and position of each token, from the requests'
 * lengths, without a word from the host. All pointers are device memory, 4-byte
 * aligned. Sequence i has n_cached[i] positions in the cache that stay, adds
 * n_new[i] tokens, and holds the first held[i] entries of its row of table; it
 * needs ceil((n_cached + n_new) / page_size) pages (0 for one that has ended).
 * Free pages lie in ring, a queue of n_pages entries: ring_at = {head, tail}, 0 <=
 * head < n_pages, those of head .. tail - 1 modulo n_pages are free. Pages that are
 * missing come from the head, in the order of the sequences, pages held beyond the
 * need go to the tail. A sequence is refused, and keeps its pages, if it takes
 * pages and what it and those before it take is more than are free, if its need is
 * more than max_pages, or if its tokens do not end within max_tokens. Written:
 *   held_out, ring_at_out (may be held and ring_at), ring, and table, whose entries
 *     behind a sequence's pages stay as they are;
 *   n_kv[i]: n_cached + n_new, 0 if refused;
 *   q_off[0 .. n_seq]: where each sequence's tokens begin, q_off[n_seq] their number;
 *   slots[t], pos[t], seq[t]: token t's cache row (-1 if its sequence is refused or
 *     its page is none), position and sequence; -1, 0 and -1 from q_off[n_seq] to
 *     max_tokens (a batch that is padded). pos and seq may be NULL;
 *   n_refused: how many sequences are refused, or NULL.
 * A refused sequence's tokens keep their places in the batch, without rows: what
 * mi_hip_verify_draft says of them does not count, its cached length stays as it is.
 * Each page is free or held by one sequence, and once: the call does not count a
 * page's users, and one that is held twice would be given back twice. Pages that
 * sequences share stay out of it (table may begin behind them).
 * Negative lengths count as 0. At most 2^30 sequences (MI_HIP_E_UNSUPPORTED). No
 * other memory of the call may overlap what it writes (with held or ring_at in place
 * one workgroup does the whole call, else large batches have several: 1024 requests
 * with 38000 tokens take 40 us in place, else 7). Calls on one pool must be ordered.
 * May be captured into a graph. No counterpart in the reference. */
typedef struct mi_hip_page_tables_args {
  int32_t n_seq;
  int32_t page_size;  /* a power of two of at least 16 */
  int32_t n_pages;
  int32_t max_pages;  /* entries of a row of table */
  int32_t max_tokens; /* entries of slots, pos and seq */
  const int32_t* n_cached;
  const int32_t* n_new;
  const int32_t* held;
  int32_t* held_out;
  int32_t* table;
  size_t table_nb;    /* bytes between rows */
  int32_t* ring;
  const int32_t* ring_at;
  int32_t* ring_at_out;
  int32_t* n_kv;
  int32_t* q_off;
  int32_t* slots;
  int32_t* pos;
  int32_t* seq;
  int32_t* n_refused;
  void* stream;
} mi_hip_page_tables_args;

int mi_hip_page_tables(const mi_hip_page_tables_args* args);

/* mi_hip_norm_rope_append into rows of a paged cache, with positions of one or
 * several axes (time, height, width): pair j of a token's dims is turned by the
 * float product pos[axis[j]][token] * frequency j. K and V go to the cache row
 * slots[token]; those of a token whose slot is outside [0, n_ctx) are not stored
 * (its Q is written). No two tokens may have the same slot. May be captured into a
 * graph. No counterpart in the reference. */
typedef struct mi_hip_paged_append_args {
  mi_hip_kv* kv;        /* of mi_hip_kv_create_paged */
  int32_t layer;
  int32_t n_tokens;
  const int32_t* slots; /* device, n_tokens cache rows */
  int32_t n_dims;       /* rotated dims (even, <= head_dim) */
  float freq_base;      /* frequencies freq_base^(-2p / n_dims), unless freq is given */
  const float* freq;    /* host, n_dims / 2 frequencies, or NULL */
  const int32_t* pos;   /* device, n_tokens positions of each axis */
  size_t pos_nb;        /* bytes between axes */
  int32_t n_axes;       /* 1 to 4 */
  const int32_t* axis;  /* host, n_dims / 2 axes, or NULL: all of axis 0 */
  float eps;
  const float* q_norm;  /* device, head_dim weights, or NULL: no norm */
  const float* k_norm;
  int32_t n_head;       /* Q heads */
  const float* q;       /* may be NULL (no Q) */
  size_t q_nb[3];
  float* q_out;         /* may be q, with the same strides */
  size_t q_out_nb[3];
  const float* k;
  size_t k_nb[3];
  const float* v;
  size_t v_nb[3];
  void* stream;
} mi_hip_paged_append_args;

int mi_hip_paged_append(const mi_hip_paged_append_args* args);

/* Attention of each sequence's new tokens over its pages. Sequence i's queries are
 * the rows q_off[i] .. q_off[i + 1] - 1 of q, its last positions: query j of them
 * stands at n_kv[i] - (their number) + j and sees the positions up to its own. The
 * lengths are read on the device, so a step needs no word from the host, and a
 * captured call takes those of each replay. A query that sees no key gives zeros;
 * rows of out outside every sequence stay as they are. What lies behind a query's
 * position never shows in its output, infinities and NaN included. A position whose
 * table entry is not in [0, n_ctx / page_size) has a row of NaN. Lengths count as
 * clamped: q_off to [0, n_tokens], n_kv to [0, max_pages * page_size]; of a sequence
 * with more than max_new queries the rest are left as they were. q_off ascends: the
 * sequences' rows do not overlap, and the limit on tiles below counts them once. A
 * max_new that is known chooses the kernel: without it single tokens take the one
 * that has room for chunks (32 over 2000 keys, 14/2 heads of 64, F16: 19 us, with
 * max_new 1 15). Products, sums and values that are not finite as in
 * mi_hip_attn_tree, with the choice of kernel per sequence: few query rows (n_rep
 * times its queries) are up to 16, or up to 32 where max_new allows no sequence
 * more, others the rows beyond. The same bits on every run with the same lengths. At
 * most 2^20 sequences, 2^26 query rows (tokens times heads), 2^30 positions of a
 * sequence, and 2^31 tiles of 32 positions in all (MI_HIP_E_UNSUPPORTED). Scratch
 * for joining the parts of long sequences: ws, else the cache's own; calls that
 * share one must be ordered. May be captured into a graph. No counterpart in the
 * reference. */
typedef struct mi_hip_attn_paged_args {
  mi_hip_kv* kv;          /* of mi_hip_kv_create_paged */
  int32_t layer;
  int32_t n_seq;
  int32_t n_tokens;       /* rows of q and out */
  int32_t max_new;        /* most queries of a sequence (0: n_tokens) */
  const int32_t* q_off;   /* device, n_seq + 1 */
  const int32_t* n_kv;    /* device, n_seq: positions, the queries' own included */
  const int32_t* table;   /* device, n_seq rows of max_pages page numbers */
  size_t table_nb;        /* bytes between rows */
  int32_t max_pages;
  int32_t n_head;
  const float* q;         /* device [head_dim, n_head, n_tokens] */
  size_t q_nb[3];
  float* out;
  size_t out_nb[3];
  float scale;
  mi_hip_workspace* ws;
  void* stream;
} mi_hip_attn_paged_args;

int mi_hip_attn_paged(const mi_hip_attn_paged_args* args);

/* Verification of drafted tokens against the target's probabilities, so that the
 * tokens that come out are distributed as if the target had drawn each. A sequence's
 * nodes are the rows off[i] .. off[i + 1] - 1 (at most 1024; those behind are not
 * looked at): node 0 is its last certain token, node c a drafted token[c] after node
 * parent[c] < c (NULL: c - 1), and row c of logits is the target's after node c,
 * p_c = softmax(logits / temperature), in 64 bits; temperature 0 has p_c one at the
 * lowest of the largest logits. From node 0 on, the children of the node v that was
 * accepted last are looked at in order; child c is accepted
 *   draft NULL (tokens taken as certain): if u_c Z < p_v(token_c), Z = 1 less the
 *     p_v of the children of v that were turned down (a token turned down before: never);
 *   draft given (token_c was drawn from the probabilities in row c of draft; chains
 *     only, parent NULL): if u_c draft_c(token_c) < p_v(token_c).
 * When no child is left, the next token is drawn by u of node 0: the lowest t for
 * which the sum of w up to t is above u times the sum of w, w = p_v without the
 * tokens turned down, or max(p_v - draft_c, 0) for the turned down c. Written, for
 * sequence i with row strides path_nb and tokens_nb:
 *   n_path[i]: the accepted nodes, node 0 among them (1 .. max_path; where there are
 *     max_path, the children of the last are not looked at), 0 for one without nodes;
 *   path: their numbers in the sequence, as mi_hip_kv_keep takes them, then -1;
 *   tokens: the accepted drafted tokens and the token drawn, n_path in all, then -1.
 * The token drawn is -1 if its row has a NaN or a +infinity, or nothing but -infinity
 * (then no child is accepted either), and where every w is 0; child tokens outside
 * [0, n_vocab) are turned down. u is clamped to [0, 1), a NaN to 0; a temperature of
 * +infinity has all finite logits alike, a negative one or NaN counts as 0. At most
 * 2^30 sequences (MI_HIP_E_UNSUPPORTED). Scratch: the parts of ws, else of the
 * library default (34 MB); of them a call takes, with c = n_vocab / 2048 rounded up,
 * at most 16 c n_rows + (8 c + 40) min(n_seq, 1024) bytes, and is refused where they
 * hold less than it takes (MI_HIP_E_UNSUPPORTED). Calls that share one must be
 * ordered. May be captured into a graph. No counterpart in the reference. */
typedef struct mi_hip_verify_args {
  const float* logits;      /* device, n_rows rows of n_vocab */
  size_t nb;                /* bytes between rows */
  int32_t n_vocab;
  int32_t n_rows;
  int32_t n_seq;
  const int32_t* off;       /* device, n_seq + 1 */
  const int32_t* token;     /* device, n_rows */
  const int32_t* parent;    /* device, n_rows, or NULL */
  const float* draft;       /* device, n_rows rows of n_vocab (those of node 0 are not read), or NULL */
  size_t draft_nb;
  const float* temperature; /* device, n_seq, or NULL: 1 */
  const float* u;           /* device, n_rows numbers in [0, 1) */
  int32_t max_path;         /* entries of a row of path and of tokens */
  int32_t* n_path;          /* device, n_seq */
  int32_t* path;
  size_t path_nb;
  int32_t* tokens;
  size_t tokens_nb;
  mi_hip_workspace* ws;
  void* stream;
} mi_hip_verify_args;

int mi_hip_verify_draft(const mi_hip_verify_args* args);

/* ---- node-level operators on device tensors ----------------------------- */
/*
 * Same signature idea as the engine's kernels (src/ops_cpu.h:3-12): the node
 * `dst` carries op, op_params and src[], and every tensor's `data` is a DEVICE
 * address. Strides are honoured as in mi_f32_ptr (src/ops_cpu.cpp:38-41).
 */

/* MI_OP_ATTN_QK (src/ops_cpu.cpp:356-380; builder src/graph.cpp:241-253). */
int mi_hip_op_attn_qk(mi_tensor* dst, void* stream);
/* MI_OP_SOFTMAX (src/ops_cpu.cpp:304-346; builder src/graph.cpp:156-163). */
int mi_hip_op_softmax(mi_tensor* dst, void* stream);
/* MI_OP_ATTN_KQV (src/ops_cpu.cpp:386-410; builder src/graph.cpp:263-273). */
int mi_hip_op_attn_kqv(mi_tensor* dst, void* stream);
/* The fused triple given its last node: dst is the ATTN_KQV node,
 * dst->src[0] the SOFTMAX node, dst->src[0]->src[0] the ATTN_QK node. */
int mi_hip_op_attn_fused(mi_tensor* dst, void* stream);

/* MI_OP_ROPE (src/ops_cpu.cpp:270-302; builder src/graph.cpp:146-154,
 * op_params n_past, n_dims, freq_base): rotary embedding of dst->src[0]
 * [head_dim, n_heads, n_tokens] into dst (may be the same memory), NEOX
 * halves (element p pairs with p + n_dims/2), token i at position n_past + i.
 * The frequencies base^(-2p/n_dims) are the host's powf values, as in the
 * engine; the angle's cosine and sine are computed on the device. n_dims must
 * be even, at most head_dim and at most 256. */
int mi_hip_op_rope(mi_tensor* dst, void* stream);

/* ---- the step after attention: Q8_0 matrix-vector products -------------- */

/* MI_OP_QUANTIZE_Q8_0 (src/ops_cpu.cpp:462-479, row quantizer
 * src/quant.cpp:188-210; builder src/graph.cpp:117-128): dst (type
 * MI_TYPE_Q8_0_ACT, blocks of a float scale and 32 int8) from an F32 src of
 * the same ne[], each row contiguous (nb[0] = 4), ne[0] a multiple of 32.
 * Bit-exact: amax/127 scale, round half to even, clamp to [-127, 127]. */
int mi_hip_op_quantize_q8_0(mi_tensor* dst, void* stream);

/* MI_OP_MUL_MAT with Q8_0 weights (src/ops_cpu.cpp:226-236; builder
 * src/graph.cpp:130-144): dst [n, m] F32 = src[0] (MI_TYPE_Q8_0 [k, n], GGUF
 * blocks, row i at nb[1] * i) times src[1] (MI_TYPE_Q8_0_ACT [k, m], column j
 * at nb[1] * j), e.g. the attention output projection. Bit-exact with the
 * reference's default dot product (src/quant_avx2.cpp:174-185). F32 and F16
 * weights are not handled here (MI_HIP_E_UNSUPPORTED). */
int mi_hip_op_mul_mat(mi_tensor* dst, void* stream);

/* ---- the step before attention: RoPE and the KV append, fused ---------- */

/* One layer's qh_rot = rope(qh); kh_rot = rope(kh); cpy(kh_rot -> cache K
 * rows [n_past, n_past + n_tokens)); cpy(vh -> cache V rows) of
 * src/model_qwen2.cpp:153-159, in one launch on device tensors, so Q, K and
 * V never pass through host memory. Shapes [head_dim, heads, n_tokens] with
 * byte strides nb[0..2] (q/q_out: n_head heads, k/v: the cache's n_head_kv).
 * q may be NULL (no Q); q_out may equal q. F16 caches round K and V to
 * nearest even, like mi_hip_kv_write. */
typedef struct mi_hip_rope_args {
  mi_hip_kv* kv;
  int32_t layer;
  int32_t n_past;
  int32_t n_tokens;
  int32_t n_dims;   /* rotated dims (even, <= head_dim), op_params[1] of ROPE */
  float freq_base;  /* op_params[2] of ROPE */
  int32_t n_head;   /* Q heads */
  const float* q;
  size_t q_nb[3];
  float* q_out;
  size_t q_out_nb[3];
  const float* k;
  size_t k_nb[3];
  const float* v;
  size_t v_nb[3];
  void* stream;
} mi_hip_rope_args;

int mi_hip_rope_append(const mi_hip_rope_args* args);

/* mi_hip_rope_append for models that norm queries and keys per head, and for
 * tokens at positions of their own. Per row x of Q and K (one head of one
 * token): y = x / sqrt(mean(x^2) + eps) * w where the norm's weights are given,
 * then the rotation of MI_OP_ROPE at the token's position (the angle is one
 * float product, position * frequency); Q into q_out (which may equal q, with
 * the same strides), K and V into the cache rows n_past + token. Without
 * weights, pos and freq the results of mi_hip_rope_append. Any cache type. May
 * be captured into a graph. No counterpart in the reference. */
typedef struct mi_hip_norm_rope_args {
  mi_hip_kv* kv;
  int32_t layer;
  int32_t n_past;       /* first cache row written */
  int32_t n_tokens;
  int32_t n_dims;       /* rotated dims (even, <= head_dim) */
  float freq_base;      /* frequencies freq_base^(-2p / n_dims), unless freq is given */
  const float* freq;    /* host, n_dims / 2 frequencies, or NULL */
  const int32_t* pos;   /* device, n_tokens positions, or NULL: n_past + token */
  float eps;
  const float* q_norm;  /* device, head_dim weights, or NULL: no norm */
  const float* k_norm;
  int32_t n_head;       /* Q heads */
  const float* q;       /* may be NULL (no Q) */
  size_t q_nb[3];
  float* q_out;
  size_t q_out_nb[3];
  const float* k;
  size_t k_nb[3];
  const float* v;
  size_t v_nb[3];
  void* stream;
} mi_hip_norm_rope_args;

int mi_hip_norm_rope_append(const mi_hip_norm_rope_args* args);

/* ---- from logits to greedy ids ------------------------------------------- */

/* Penalties, biases and a grammar's mask on rows of logits (one per sequence,
 * or per drafted token), and the greedy id of each row. For token t that stands
 * c times in the row's history, each step rounded to float:
 *   c > 0:  y = x > 0 ? x / repeat : x * repeat;  y -= c * frequency + presence
 *   y += the sum of t's biases, in the list's order
 *   y = -inf where the mask's bit t is clear
 * ids: the lowest t with the largest y (mi_qwen2_sample_greedy's rule,
 * src/model_qwen2.cpp:690-700), -1 if every y is -inf or NaN. All pointers are
 * device memory; offsets have n_rows + 1 entries, row r's list is
 * [off[r], off[r + 1]). Ids outside [0, n_vocab) in the lists are passed over.
 * Calls for ids that share a workspace must be ordered. May be captured into a
 * graph. No counterpart in the reference. */
typedef struct mi_hip_logits_args {
  const float* logits;
  size_t nb;                /* bytes between rows */
  float* out;               /* may be logits */
  size_t out_nb;
  int32_t n_vocab;
  int32_t n_rows;
  const float* penalties;   /* repeat, frequency, presence of each row, or NULL (with no history) */
  const int32_t* hist;      /* token ids, or NULL */
  const int32_t* hist_off;
  const int32_t* bias_id;   /* token ids, or NULL */
  const float* bias;
  const int32_t* bias_off;
  const uint32_t* mask;     /* bit t % 32 of word t / 32: token t is allowed; or NULL */
  size_t mask_nb;           /* bytes between rows; 0: one row for all */
  int32_t* ids;             /* greedy ids, or NULL */
  mi_hip_workspace* ws;     /* scratch for ids, or NULL: the library default */
  void* stream;
} mi_hip_logits_args;

int mi_hip_logits_adjust(const mi_hip_logits_args* args);

/* ---- executor hook for host-resident graphs ------------------------------ */

/* Plans one step's graph (call after the allocator assigned data, before
 * execution): marks every ATTN_QK -> SOFTMAX -> ATTN_KQV chain whose scores
 * and probabilities have no other reader as fused. Allocation-free. */
int mi_hip_graph_prepare(const mi_cgraph* graph);

/* Drop-in for the dispatch in mi_compute_forward (src/ops_cpu.cpp:481-530),
 * same (dst, ith, nth) contract as every engine kernel (src/ops_cpu.h:3-12)
 * and the executor's per-node barrier (src/threadpool.cpp:171-180).
 * Returns 1 if the node belongs to this backend (the caller then skips its CPU
 * kernel), 0 if it does not, -1 on error (see mi_hip_last_error). Only ith == 0
 * does work: it enqueues the node on the KV cache's stream and waits for it,
 * so the node's host output is complete before the caller's barrier. Nodes
 * handled: CPY into a bound KV tensor; ATTN_QK and SOFTMAX of a planned fused
 * chain (no-ops); ATTN_KQV of a planned fused chain (the fused launch). */
int mi_hip_compute_forward(mi_tensor* dst, int ith, int nth);

/* Host-resident attention nodes (opt-in, default off): with on = 1,
 * mi_hip_compute_forward also takes ATTN_QK, SOFTMAX and ATTN_KQV nodes that
 * are not part of a fused chain on a bound KV cache -- e.g. a model whose
 * head_dim the fused kernels do not cover (they take 64 and 128), so its
 * cache stays on the host -- and runs each on the node kernels (bit-exact
 * with src/ops_cpu.cpp:304-410): its sources are copied to a staging buffer
 * (grown, and therefore allocated, to the largest node seen), the node runs,
 * its output is copied back before the call returns. A correctness path for
 * such models, not a throughput one. Process-wide. No counterpart in the
 * reference. */
int mi_hip_set_host_nodes(int32_t on);

/* ---- read-bandwidth ceiling ---------------------------------------------- */

/* The device counterpart of tools/bench_memread.cpp (the engine's read-only
 * bandwidth ceiling: a load-and-accumulate pass, one reduced sum per worker,
 * no writes to the source): n_sums workgroups each sum one contiguous slice
 * of src[0, bytes) (float data) and write sums[w]; sum(sums) is the sum of
 * the buffer up to float rounding. src is device memory, 16-byte aligned,
 * bytes a multiple of 16; sums is device memory of n_sums floats, 1 <= n_sums
 * <= 65536. Timed by the caller on `stream`: bytes / kernel time is the
 * measured ceiling that the decode kernels are compared with. */
int mi_hip_memread(const void* src, size_t bytes, float* sums, int32_t n_sums, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* MI_HIP_ATTN_H */
