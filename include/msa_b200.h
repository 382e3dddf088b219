/*
 * msa_b200.h -- C ABI of libmsa_b200.so, the sm_100a implementation of the
 * MiniMax-Sparse-Attention hot path (paged / sparse FMHA forward, page top-k
 * selection, split-KV LSE merge).
 *
 * Every entry point replaces one native export of the upstream msa_for_sail
 * package (paths below are relative to the upstream project root).  All
 * functions take plain pointers and sizes, enqueue work on the given CUDA
 * stream, never synchronise, and return 0 or a negative MSA_ERR_* code.
 * Unless stated otherwise they allocate nothing: every buffer is owned by the
 * caller (upstream: "every tensor is allocated by Python", api.py:1374-1389).
 */
#ifndef MSA_B200_H_
#define MSA_B200_H_

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define MSA_OK               0
#define MSA_ERR_BAD_ARG     -1   /* NULL / inconsistent argument                    */
#define MSA_ERR_UNSUPPORTED -2   /* combination the library does not implement     */
#define MSA_ERR_LAUNCH      -3   /* cudaGetLastError() after the launch was not OK */
#define MSA_ERR_TOO_LARGE   -4   /* size beyond a documented maximum               */

/* element types */
#define MSA_DT_BF16 0
#define MSA_DT_E4M3 1
#define MSA_DT_F32  2
#define MSA_DT_KV4  3   /* caches only: e2m1 codes with an e4m3 scale for each 16 elements.  The tile of one (page, KV head) is
                           9216 contiguous bytes: 128 rows of 64 bytes (element 2i in the low half of byte i), then
                           128 rows of 8 scales.  Strides of such a cache are in bytes, multiples of 16 */

/* msa_fmha_fwd mode bits (upstream SparseAttnMode, csrc/include/fmha_fusion.hpp:42-54) */
#define MSA_FLAG_OUT_O      1   /* compute P.V and write O                      */
#define MSA_FLAG_OUT_SCORE  2   /* write per-128-key-tile row max of raw q.k    */
#define MSA_FLAG_SPARSE     4   /* iterate kv_block_indexes instead of all keys */

/* device status word values (written only when MsaFmhaParams.status != NULL) */
#define MSA_STATUS_OK        0
#define MSA_STATUS_TIMEOUT   1   /* a bounded wait inside a kernel gave up       */
#define MSA_STATUS_BOUNDS    2   /* bounds-checked build only (-DMSA_BOUNDS_CHECK): an index read from a
                                    caller's table (work item, page table, token -> batch map) was out of
                                    range; it was clamped into range before use                            */

typedef void* msa_stream_t;      /* a cudaStream_t */

/* One unit of dense work: BLOCK_M packed rows of one (batch item, head group)
 * against KV tiles [kv_tile_begin, kv_tile_end) of 128 keys.  Replaces the
 * upstream 64-bit packed work item + kv_tile_begin/end/split arrays
 * (csrc/include/fmha_tile_scheduler.hpp:49-55, api.py:841-845). */
typedef struct MsaWorkItem {
  int32_t batch;          /* batch item                                            */
  int32_t head0;          /* first query head covered by this item                 */
  int32_t row0;           /* first packed row (row = token_in_seq * pack + head_in_pack) */
  int32_t kv_tile_begin;  /* first 128-key tile                                    */
  int32_t kv_tile_end;    /* one past the last tile                                */
  int32_t split;          /* split index for the partial workspace (0 if unsplit)  */
  int32_t num_rows;       /* packed rows of this item (<= block_m)                  */
  int32_t kv_tile_skip;   /* tiles that no row of a windowed item sees: tile t of the item is tile t of the keys for
                             t < ceil(sink_tokens / 128), tile t + kv_tile_skip from there on (0 without a window) */
} MsaWorkItem;

/* Arguments of the FMHA forward.  Field-for-field successor of the upstream
 * FMHACutlassSailParams (csrc/fmha_sail_params.h:10-77) minus the PPU-only
 * members.  Strides are in elements. */
typedef struct MsaFmhaParams {
  const void*    q;                /* [total_q, Hq, 128] bf16 | e4m3                         */
  const void*    k;                /* ragged [sum_kv, Hkv, 128] or paged 4-D, bf16 | e4m3   */
  const void*    v;                /* same layout as k (may be NULL without MSA_FLAG_OUT_O)  */
  void*          out;              /* [total_q, Hq, 128] bf16 or NULL                        */
  float*         lse;              /* [total_q, Hq] natural-log LSE or NULL                  */
  void*          max_score;        /* [Hq, max_k_tiles, total_q] f32 | bf16 or NULL          */
  float*         partial_o;        /* split workspace [S, total_q, Hq, 128] f32 or NULL      */
  float*         partial_lse;      /* split workspace [S, total_q, Hq] f32 or NULL           */
  const int32_t* qo_start;         /* [B+1] first token of each batch item                   */
  const int32_t* kv_start;         /* [B+1] first key of each item (ragged only)             */
  const int32_t* kv_len;           /* [B]                                                    */
  const int32_t* qo_offset;        /* [B] row i sees key j iff i + qo_offset >= j            */
  const int32_t* kv_page_indptr;   /* [B+1] (paged)                                          */
  const int32_t* kv_indices;       /* flat physical page table (paged)                       */
  const int32_t* kv_block_indexes; /* [total_q, Hkv, kv_block_num] logical pages (sparse)    */
  const int32_t* token_batch;      /* [total_q] batch item of each token (sparse)            */
  const MsaWorkItem* work;         /* [num_work] (dense)                                     */
  const float*   k_scale_head;     /* optional [Hkv] de-quantisation scale of K             */
  const float*   v_scale_head;     /* optional [Hkv] de-quantisation scale of V             */
  int32_t*       status;           /* optional device status word                            */
  const int32_t* page_batch;       /* optional [num_logical_pages] batch item owning each entry of kv_indices */
  void*          sparse_ws;        /* optional workspace of msa_sparse_workspace_bytes() bytes: enables the
                                      page-major (KV-outer) sparse prefill path                             */
  int64_t        sparse_ws_bytes;
  int64_t q_stride_tok, q_stride_head;
  int64_t k_stride_page, k_stride_head, k_stride_tok;   /* ragged: page stride unused       */
  int64_t v_stride_page, v_stride_head, v_stride_tok;
  int64_t out_stride_tok, out_stride_head;
  int64_t kbi_stride_tok, kbi_stride_head;
  int64_t kv_extent;       /* outermost extent of k / v: total keys (ragged) or pages in the pool */
  int32_t total_q, num_qo_heads, num_kv_heads, batch;
  int32_t num_work;        /* dense: work items; sparse: ignored                             */
  int32_t block_m;         /* 16, 64, 128 packed rows per item; 256 selects the tcgen05 kernel */
  int32_t pack;            /* query heads folded into the row dimension (1 or Hq/Hkv)        */
  int32_t page_size;       /* 0 = ragged K/V                                                 */
  int32_t kv_block_num;    /* sparse: entries per (token, kv head)                           */
  int32_t num_splits;      /* size of the S dimension of the partial workspace (1 = unsplit) */
  int32_t max_k_tiles;     /* second dimension of max_score                                  */
  int32_t num_logical_pages; /* length of kv_indices (sparse page-major path)                        */
  int32_t decode_rows;     /* > 0: every item has at most this many packed rows (<= 128) and may run on the
                              tcgen05 decode kernel; 0: do not use it.  Rows past it are left out     */
  int32_t q_dtype, kv_dtype, max_score_dtype;
  int32_t flags;           /* MSA_FLAG_*                                                     */
  float   sm_scale;        /* q_scale * k_scale * softmax scale                              */
  float   out_scale;       /* v_scale * o_scale                                              */
  int32_t window;          /* > 0: row i, at place t = i + qo_offset, sees key j <= t iff j > t - window or j < sink_tokens.
                              Dense work lists made with the same two numbers, MSA_FLAG_OUT_O only; 0: every key up to t */
  int32_t sink_tokens;
  int32_t num_sms;         /* with a window: SMs that CTAs which share an item are spread over; 0 = all 148                */
  int32_t num_page_entries; /* length of kv_indices: places past its end read as its last entry; 0 = not given,
                              every place that the lengths reach is read (kv_dtype = MSA_DT_KV4: num_logical_pages) */
} MsaFmhaParams;

/* FMHA forward: dense ragged / dense paged / sparse, optional split-KV partials.
 * Replaces the per-variant export `run` (csrc/fmha_sail_variant_run.cu.jinja:17-43,261
 * -> run_fmha_fwd, csrc/include/fmha_cutlass_sm80.cuh:185-486).  With
 * partial_o != NULL the kernel writes normalised partial O and LSE per split
 * and the caller runs msa_lse_merge afterwards. */
int msa_fmha_fwd(const MsaFmhaParams* params, msa_stream_t stream);

/* Bytes of MsaFmhaParams.sparse_ws needed by the page-major sparse prefill path (reverse
 * index page -> tokens, per-slot partial O in bf16 and LSE).  No upstream counterpart: there
 * sparse attention always runs token by token (csrc/include/prepare_plan_metadata.cuh:90-112). */
int64_t msa_sparse_workspace_bytes(int64_t total_q, int32_t num_qo_heads, int32_t num_kv_heads,
                                   int32_t kv_block_num, int64_t num_logical_pages);

/* Split-KV merge: out[t,h,:] = sum_s w_s * partial_o[s,t,h,:] / sum_s w_s with
 * w_s = exp(partial_lse[s,t,h] - max_s); a -inf LSE gives weight 0 and its
 * partial is ignored.  splits_per_row ([total_q] or NULL = num_splits for all)
 * bounds s per token.  Replaces `reduction` (csrc/fmha_sm80_reduction.cu:42-104,
 * csrc/include/sm80_fmha_reduction.hpp:74-216). */
int msa_lse_merge(const void* partial_o, int32_t partial_dtype /* MSA_DT_F32 | MSA_DT_BF16 */,
                  const float* partial_lse,
                  const int32_t* splits_per_row, void* out, float* lse_out,
                  int32_t num_splits, int32_t total_q, int32_t num_heads,
                  int64_t out_stride_tok, int64_t out_stride_head,
                  float out_scale, msa_stream_t stream);

/* The same merge with two more degrees of freedom, for partials that do not sit in the dense
 * [S, total_q, H, ...] arrangement and for callers that want the result unrounded:
 *  - o_split_stride / lse_split_stride: elements between split s and split s + 1 of partial_o /
 *    partial_lse (<= 0: the dense default total_q*H*128 / total_q*H).  Lets one buffer hold
 *    several ranks' packed (O, LSE) blocks as an all-gather delivers them;
 *  - out_dtype: MSA_DT_BF16 or MSA_DT_F32 (the fp32 result of a local merge is what a rank
 *    contributes to a cross-GPU merge).
 * No upstream counterpart beyond `reduction` itself (upstream is single-device). */
int msa_lse_merge_ex(const void* partial_o, int32_t partial_dtype, const float* partial_lse,
                     const int32_t* splits_per_row, void* out, int32_t out_dtype, float* lse_out,
                     int32_t num_splits, int32_t total_q, int32_t num_heads,
                     int64_t o_split_stride, int64_t lse_split_stride,
                     int64_t out_stride_tok, int64_t out_stride_head,
                     float out_scale, msa_stream_t stream);

/* The merge of dense fp32 partials [S, total_q, H, 128] with a warp for each row, or a CTA where there are many splits of few
 * rows: 0.2 to 0.7 of the time of msa_lse_merge.  Sums are taken in another (fixed) order. */
int msa_lse_merge_many(const float* partial_o, const float* partial_lse, const int32_t* splits_per_row, void* out,
                       int32_t out_dtype, float* lse_out, int32_t num_splits, int32_t total_q, int32_t num_heads,
                       int64_t out_stride_tok, int64_t out_stride_head, float out_scale, msa_stream_t stream);

/* Page top-k: per (head, token) row of scores[H, K, T] pick the `topk` best
 * pages of [0, num_valid_pages) by (score desc, index asc), emit them
 * ascending into out[T, H, topk] (int32), pad with -1.  Pages [0, force_begin)
 * and [nvp - force_end, nvp) rank as FLT_MAX.  topk in {4, 8, 16, 32}.
 * Replaces `sparse_topk_select` (csrc/sparse_topk_select.cu:19-88,
 * csrc/include/sparse_topk_select.cuh:1410-1459).  Needs no workspace. */
int msa_topk_select(const void* scores, int32_t score_dtype, int32_t* out,
                    int32_t num_heads, int32_t max_k_tiles, int32_t total_q,
                    int32_t topk, int32_t num_valid_pages,
                    int32_t force_begin, int32_t force_end, msa_stream_t stream);

/* Host-side planner for the dense path: enumerates (batch, head group, row
 * tile) items, cuts long KV ranges into splits, orders items longest first.
 * Host arrays in, host arrays out (the caller uploads `work`).  Replaces
 * `prepare_plan_metadata` + `plan` (csrc/prepare_plan_metadata.cu:19-37,
 * csrc/fmha_sm80_plan.cu:20-37; behaviour spec: tests/integration/
 * test_plan_correctness.py:58-190 -- every tile exactly once, split ranges
 * contiguous from 0).  Returns the number of items written, or a negative
 * error (MSA_ERR_TOO_LARGE if `capacity` is too small). */
typedef struct MsaPlanArgs {
  const int32_t* qo_len;      /* [B] host */
  const int32_t* kv_len;      /* [B] host */
  const int32_t* qo_offset;   /* [B] host */
  int32_t batch;
  int32_t num_qo_heads, num_kv_heads;
  int32_t block_m;            /* 16 / 64 / 128 / 256 */
  int32_t pack;               /* 1 or Hq/Hkv   */
  int32_t num_splits;         /* >=1 fixed; <=0 adaptive with -num_splits as the ceiling */
  int32_t num_sms;            /* device SM count (adaptive mode target)  */
  int32_t ctas_per_sm;        /* items an SM runs side by side; 0 = 1; < 0: all items cut alike, for two waves of the
                               * SMs, and uncut where there are as many (adaptive mode) */
  int32_t window;             /* as in MsaFmhaParams: a row tile then has the tiles that its rows see, see kv_tile_skip */
  int32_t sink_tokens;
  int32_t cluster;            /* with a window, adaptive mode: CTAs that may share an uncut item at run time (16: at most 16 packed rows
                               * over ragged keys or pages of a multiple of 32 keys; 2: at most 128 over pages of 128 keys, `pack`
                               * dividing 128; else 0); items stay uncut where that is as good */
} MsaPlanArgs;
int msa_plan_dense(const MsaPlanArgs* args, MsaWorkItem* work, int32_t capacity,
                   int32_t* splits_per_row /* [total_q] host */,
                   int32_t* max_splits_out);

/* Planning on the device, for callers that capture plan + run into one CUDA graph and only
 * update the length tensors between replays (upstream: `graph_safe=True`, the
 * prepare_plan_metadata + plan kernels, api.py:916-941, 1040-1048, 1196-1203).
 * Everything that sizes a launch is fixed when the graph is built: batch, the number of
 * row tiles per batch item (`row_tiles` >= ceil(max qo_len * pack / block_m)), the split count.
 * One kernel launch on `stream`; reads no device memory on the host, allocates nothing.
 * Fills, for i in [0, batch):  qo_start / kv_start (exclusive prefix sums, [batch + 1]; qo_start never above max_total_q, where
 * that is not 0: tokens of lengths that sum to more are in no sequence and in no work item, if qo_start is given),
 * kv_len_out, qo_offset_out (causal: kv_len - qo_len where qo_offset_in is NULL or
 * negative; non-causal: `noncausal_offset`), kv_page_indptr ([batch + 1], pages of
 * `page_size` keys, NULL for ragged K/V), token_batch ([max_total_q], NULL when unused),
 * splits_per_row ([max_total_q]: num_splits for real tokens, 0 for the padding past the last
 * one, so that a merge over max_total_q rows writes zeros there) and the work list: exactly
 * batch * row_tiles * (num_qo_heads / pack) * num_splits items, item
 * (((b * row_tiles + r) * groups) + g) * S + s = row tile (row_tiles - 1 - r) of batch item b
 * (later rows first: under a causal mask they see more keys), head group g, the s-th of S
 * equal chunks of the key tiles those rows can see.  A row tile past the item's rows, or a
 * chunk past its tiles, is an item with num_rows = 0 / an empty tile range.  NULL outputs
 * are skipped. */
typedef struct MsaPlanDeviceArgs {
  const int32_t* qo_len;       /* [B] device */
  const int32_t* kv_len;       /* [B] device */
  const int32_t* qo_offset_in; /* [B] device or NULL */
  int32_t* qo_start;
  int32_t* kv_start;
  int32_t* kv_len_out;
  int32_t* qo_offset_out;
  int32_t* kv_page_indptr;
  int32_t* token_batch;
  int32_t* splits_per_row;
  MsaWorkItem* work;
  int32_t batch;
  int32_t num_qo_heads, num_kv_heads;
  int32_t block_m, pack, num_splits;
  int32_t page_size;           /* <= 0: ragged */
  int32_t causal;
  int32_t noncausal_offset;
  int32_t max_total_q;
  int32_t row_tiles;           /* >= 1 */
  int32_t window;              /* as in MsaPlanArgs */
  int32_t sink_tokens;
} MsaPlanDeviceArgs;
int msa_plan_device(const MsaPlanDeviceArgs* args, msa_stream_t stream);

/* Split-KV forward + merge with the partial-result scratch held inside the library.
 * No counterpart in the upstream project (there the caller always owns the split
 * workspace, api.py:141-167).  It exists for embedders that may not allocate device
 * memory at call time -- an engine whose memory pool owns the whole device after
 * start-up, a sandboxed plugin host that passes tensors but no allocator.  Same
 * arguments and the same argument checks as msa_fmha_fwd (dense or sparse, MSA_FLAG_OUT_O
 * only, block_m 16/64/128) with partial_o / partial_lse left NULL and num_splits = the S of
 * the work list; the result goes to params->out (and params->lse).  `splits_per_row`
 * ([total_q] device int32, or NULL) has the meaning it has in msa_lse_merge: how many of
 * the S slots of a token the merge looks at; NULL = all S.  Either way a slot that no work
 * item of this call wrote counts as empty: the call first marks every slot as empty (LSE
 * -inf), so a short or empty work list gives zeros / -inf LSE, never a value left behind by
 * an earlier call.  The call performs no cudaMalloc / cudaFree and calls no allocating
 * routine.
 *  - Limit: num_splits * total_q * num_qo_heads <= MSA_STATIC_SCRATCH_MAX_ROWS,
 *    otherwise MSA_ERR_TOO_LARGE.  The array (about 8.5 MB) is resident on every GPU
 *    that loads the library, until the process exits.
 *  - The first call on a device resolves the array's device address; make that first
 *    call before any stream capture on that device.
 *  - All calls on a device share the one array: two calls whose kernels overlap on the
 *    GPU (different streams) race on it.  Serialise them on one stream. */
#define MSA_STATIC_SCRATCH_MAX_ROWS 16384
int msa_fmha_fwd_split_static(const MsaFmhaParams* params, const int32_t* splits_per_row,
                              msa_stream_t stream);

/* msa_fmha_fwd with split partials (partial_o, partial_lse and num_splits set) and the merge of them, msa_lse_merge_many, into out and lse: one
 * call.  out_dtype: MSA_DT_BF16 or MSA_DT_F32, strides of out in elements of it; its rows begin at multiples of 16 bytes, as in an unsplit call.
 * What the merge would refuse is refused before anything is launched. */
int msa_fmha_fwd_merged(const MsaFmhaParams* params, const int32_t* splits_per_row, int32_t out_dtype, msa_stream_t stream);

/* msa_fmha_fwd with kv_dtype = MSA_DT_KV4: q bf16 or e4m3, paged k and v with page_size 128, MSA_FLAG_OUT_O only (with or
 * without MSA_FLAG_SPARSE), block_m 16 / 64 / 128; up to 128 packed rows per work item.  Longer queries and scores: unpack
 * the pages with msa_kv4_read and run on the copy.  num_logical_pages is the length of kv_indices; entries past it and pages
 * outside [0, kv_extent) are clamped.  17 to 128 rows of dense items run on the tensor-core kernel, whose waits report to
 * `status`.  msa_fmha_fwd_split_static does not take it. */

/* Per-head RMS norm of q and k, rotary positions, and the write of k and v into a paged cache, in one pass over a step's
 * tokens.  Any of q, k, v may be NULL (k needs k_out or k_cache; v needs v_cache).  q, k, v and the outputs are bf16 unless a
 * dtype says otherwise, head_dim 128, strides in elements (a KV4 cache: bytes); in-place (q_out == q) is allowed.
 *  - norm != 0: x / sqrt(mean(x^2) + eps) * weight; weights [128] (stride 0) or one row per head, f32 or bf16, NULL = 1.
 *  - rotary elements (a multiple of 32, 0 = none) are rotated in pairs (i, i + rotary / 2), or (2i, 2i + 1) if interleaved,
 *    by positions[axis[n]][token] * turns[n] for pair n; turns[n] = the frequency in turns per position, as a
 *    64-bit fraction (modulo 1).
 *  - cache: row of token t at slot_map[t] = page * page_size + offset; a negative slot, or one past num_pages, writes
 *    nothing.  Slots of one call are distinct.  Keys are computed in 64 bits and rounded to 32 and to bf16, then divided by
 *    k_scale * k_scale_head[head] and rounded to the cache's type (bf16 caches: as they are); values likewise.
 *  - e4m3 queries: rounded to bf16, divided by q_scale and rounded to e4m3.
 * No upstream counterpart (upstream starts at the attention call). */
typedef struct MsaNormRopeArgs {
  const void* q; const void* k; const void* v;
  const void* q_weight; const void* k_weight;
  const void* positions;           /* int32 or int64, [axes][tokens] */
  const int64_t* turns;            /* [rotary / 2] device */
  const int32_t* axis;             /* [rotary / 2] device */
  void* q_out; void* k_out; void* k_cache; void* v_cache;
  const int32_t* slot_map;         /* [tokens] device */
  const float* k_scale_head; const float* v_scale_head;   /* [num_kv_heads] or NULL */
  int32_t* status;
  int64_t pos_stride_axis;
  int64_t q_stride_tok, q_stride_head, k_stride_tok, k_stride_head, v_stride_tok, v_stride_head;
  int64_t q_out_stride_tok, q_out_stride_head, k_out_stride_tok, k_out_stride_head;
  int64_t q_weight_stride, k_weight_stride;
  int64_t k_cache_stride_page, k_cache_stride_head, k_cache_stride_tok;
  int64_t v_cache_stride_page, v_cache_stride_head, v_cache_stride_tok;
  int32_t tokens, num_qo_heads, num_kv_heads, rotary, interleaved, norm;
  int32_t weight_dtype, q_out_dtype, cache_dtype, pos_int64, page_size, num_pages;
  float eps, q_scale, k_scale, v_scale;
} MsaNormRopeArgs;
int msa_norm_rope(const MsaNormRopeArgs* args, msa_stream_t stream);

/* Rows of a KV4 cache as bf16 (exact).  whole_pages == 0: out[i][head] = row slot_map[i] (zeros for a negative slot or one past
 * num_pages); != 0: out[i][head][128][128] = page slot_map[i] (the nearest one for a number outside [0, num_pages)), for the first
 * *num_used entries or all; what is behind them is left as it was. */
typedef struct MsaKv4ReadArgs {
  const void* cache;
  void* out;
  const int32_t* slot_map;         /* [rows] device: slots, or pages */
  int32_t* status;
  const int32_t* num_used;         /* whole_pages: [1] device, entries that count (the last one of kv_page_indptr), or NULL: all */
  int64_t stride_page, stride_head;
  int32_t rows, num_kv_heads, num_pages, whole_pages;
} MsaKv4ReadArgs;
int msa_kv4_read(const MsaKv4ReadArgs* args, msa_stream_t stream);

/* The page table, slots and positions of a step from its requests' lengths, all on the device:
 *  - kv_indices [max_total_pages] / kv_page_indptr [batch + 1]: the flat table that the attention call reads; entries
 *    behind the last page are -1;
 *  - slot_map / positions [max_total_q]: of every new token (the last qo_len keys of its request); -1 / 0 behind the last.
 * With num_held, free_pages, num_free (all or none): pages that a request needs beyond the num_held[b] entries of its
 * block_table row come from the top of the stack free_pages[0, num_free) in the order of the requests, and are written into
 * the row; num_held_out / num_free_out (may be num_held / num_free) receive the new counts.  num_missing: pages and tokens
 * that found no place (an empty stack, a row of the table or an output that is too short).  Such a page is 0 in
 * kv_indices (attention over it stays in bounds but means nothing), -1 in block_table, and its tokens have slot -1.
 * kv_page_indptr counts the pages that a kv_indices of max_total_pages has no place for as well: give the attention call
 * num_page_entries = max_total_pages, and they read as its last entry. */
typedef struct MsaPageTablesArgs {
  const int32_t* qo_len;           /* [B] device: new tokens */
  const int32_t* kv_len;           /* [B] device: keys with them */
  int32_t* block_table;            /* [B][table_width] device, table_stride apart */
  const int32_t* num_held;         /* [B] device or NULL */
  const int32_t* free_pages;       /* [free_capacity] device or NULL */
  const int32_t* num_free;         /* [1] device or NULL */
  int32_t* kv_indices;
  int32_t* kv_page_indptr;
  int32_t* slot_map;
  int32_t* positions;
  int32_t* num_held_out;           /* [B] or NULL */
  int32_t* num_free_out;           /* [1] or NULL */
  int32_t* num_missing;            /* [1] or NULL */
  int32_t* workspace;              /* msa_page_tables_workspace_bytes(batch) bytes */
  int64_t table_stride;
  int32_t batch, table_width, page_size, max_total_q, max_total_pages, free_capacity;
} MsaPageTablesArgs;
int64_t msa_page_tables_workspace_bytes(int32_t batch);
int msa_page_tables(const MsaPageTablesArgs* args, msa_stream_t stream);

/* Pages of a cache: copies, rows of a block table that share pages, pages given back, pages in use moved together.
 *
 * A block table [batch][table_width], table_stride apart, has the page of each page_size tokens of a request; num_held[b] entries of
 * row b are set, -1 among them for pages given back from the middle.  free_pages[0, *num_free) is the stack of free pages that
 * msa_page_tables takes from.  shares[p] (NULL: each page is in one row) is the number of rows that hold page p beyond the first.
 * Everything is on the device, and updated in place; results do not depend on the order of threads.  No upstream counterpart. */

/* One tensor that holds something of every page: a page is `parts` pieces of part_bytes, stride_part bytes apart, from
 * base + page * stride_page (bytes) on.  Any alignment; multiples of 16 bytes are fastest. */
typedef struct MsaPageCache {
  void* base;
  int64_t stride_page, stride_part;
  int32_t parts, part_bytes;
  int32_t token_bytes;             /* bytes of one token in a piece, tokens in order; -1: each piece is a token; 0: neither, such
                                      pages are copied whole where others are copied up to a token */
  int32_t reserved;
} MsaPageCache;

/* Page src[i] to page dst[i] in every cache, for i in [0, count); a number outside [0, num_pages) copies nothing.  A page
 * of dst is in dst once and not in src. */
typedef struct MsaPagesCopyArgs {
  const MsaPageCache* caches;      /* [num_caches] HOST */
  const int32_t* src;              /* [count] device */
  const int32_t* dst;
  int32_t* status;
  int32_t num_caches, count, num_pages, page_size;
} MsaPagesCopyArgs;
int msa_pages_copy(const MsaPagesCopyArgs* args, msa_stream_t stream);

/* Row children[i] becomes a fork of row parents[i]: it shares the full pages of the first kv_len tokens (shares + 1 each), and gets a copy of
 * the used part of the last page in a page from the stack, in the order of i.  kv_len and num_held of the child are set.
 * An entry with a negative number does nothing.  Entries whose row is not in the table, is its own parent, holds pages already or was
 * named as a child before are not made, and counted in num_missing; so is a child for whose last page the stack has none: it ends with its last
 * full page.  Rows are read as they were before the call. */
typedef struct MsaPagesForkArgs {
  const MsaPageCache* caches;      /* [num_caches] HOST */
  int32_t* block_table;
  int32_t* num_held;               /* [batch] */
  int32_t* kv_len;                 /* [batch] */
  const int32_t* parents;          /* [count] device */
  const int32_t* children;
  const int32_t* free_pages;
  int32_t* num_free;               /* [1] */
  int32_t* shares;                 /* [num_pages] */
  int32_t* num_missing;            /* [1] or NULL */
  int32_t* workspace;              /* msa_pages_fork_workspace_bytes(batch, count) bytes */
  int64_t table_stride;
  int32_t num_caches, count, num_pages, page_size, batch, table_width, free_capacity;
} MsaPagesForkArgs;
int64_t msa_pages_fork_workspace_bytes(int32_t batch, int32_t count);
int msa_pages_fork(const MsaPagesForkArgs* args, msa_stream_t stream);

/* Row b keeps the pages of its first kv_len[b] tokens; with a window (as in MsaFmhaParams) also only those that a query at place
 * kv_len[b] or later sees.  The other entries become -1, their pages lose a share, and those that nobody shares go onto the stack in the order of
 * the entries (row, then column; of several entries with one page the first).  num_held becomes the pages of the length.
 * Numbers outside [0, num_pages) are dropped.
 *
 * A row whose length was cut back into a page that other rows hold would write its next token there.  With caches such a row then takes a page from
 * the stack, in the order of the rows, that gets a copy of its tokens, and gives up its share (the last row, if all that hold the page are such
 * rows, keeps it).  num_shared: rows that are left with such a page, since the stack had none or there are no caches. */
typedef struct MsaPagesFreeArgs {
  const MsaPageCache* caches;      /* [num_caches] HOST; needs shares */
  int32_t* block_table;
  int32_t* num_held;               /* [batch] */
  const int32_t* kv_len;           /* [batch] */
  int32_t* free_pages;             /* [free_capacity] */
  int32_t* num_free;               /* [1] */
  int32_t* shares;                 /* [num_pages] or NULL */
  int32_t* num_freed;              /* [1] or NULL: pages that went onto the stack */
  int32_t* num_shared;             /* [1] or NULL; needs shares */
  int32_t* workspace;              /* msa_pages_free_workspace_bytes(batch, table_width) bytes */
  int64_t table_stride;
  int32_t num_caches, batch, table_width, page_size, free_capacity, num_pages, window, sink_tokens;
} MsaPagesFreeArgs;
int64_t msa_pages_free_workspace_bytes(int32_t batch, int32_t table_width);
int msa_pages_free(const MsaPagesFreeArgs* args, msa_stream_t stream);

/* The pages that rows hold move to the lowest of the places that they and the free pages have: of those in use that lie higher, the lowest goes to
 * the lowest free place, and so on.  Table, shares and caches follow; the stack has the free pages afterwards, the lowest on
 * top.  Pages in no row and not on the stack stay where they are.  src / dst: the moves, -1 behind them. */
typedef struct MsaPagesCompactArgs {
  const MsaPageCache* caches;      /* [num_caches] HOST */
  int32_t* block_table;
  const int32_t* num_held;         /* [batch] */
  int32_t* free_pages;             /* [free_capacity] */
  int32_t* num_free;               /* [1] */
  int32_t* shares;                 /* [num_pages] or NULL */
  int32_t* src;                    /* [num_pages] */
  int32_t* dst;
  int32_t* num_moved;              /* [1] */
  int32_t* workspace;              /* msa_pages_compact_workspace_bytes(num_pages) bytes */
  int64_t table_stride;
  int32_t num_caches, num_pages, page_size, batch, table_width, free_capacity;
} MsaPagesCompactArgs;
int64_t msa_pages_compact_workspace_bytes(int32_t num_pages);
int msa_pages_compact(const MsaPagesCompactArgs* args, msa_stream_t stream);

/* Human-readable text of an MSA_ERR_* code. */
const char* msa_status_string(int code);

/* Library build info: returns the SM architecture the kernels were built for (100). */
int msa_build_arch(void);

/* sizeof() of the ABI structs as the library was compiled: 0 = MsaFmhaParams,
 * 1 = MsaWorkItem, 2 = MsaPlanArgs, 3 = MsaPlanDeviceArgs, 4 = MsaNormRopeArgs, 5 = MsaKv4ReadArgs,
 * 6 = MsaPageTablesArgs, 7 = MsaPageCache, 8 = MsaPagesCopyArgs, 9 = MsaPagesForkArgs, 10 = MsaPagesFreeArgs,
 * 11 = MsaPagesCompactArgs.  Lets a foreign-language binding verify its
 * own struct declaration at load time. */
int msa_sizeof(int which);

#ifdef __cplusplus
}
#endif
#endif /* MSA_B200_H_ */
