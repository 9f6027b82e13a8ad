/*
 * orthocache_paged.h -- the operators around a paged key-value cache, part of
 * liborthocache_hip.so's C ABI (see orthocache_hip.h for the conventions:
 * device pointers, element strides, an int status, work on the stream given,
 * no synchronisation, no allocation).
 *
 * The reference has no counterpart of any of them: it takes filled caches
 * and fixed block tables.
 *
 * A paged cache is (num_blocks, num_kv_heads, block_size, head_dim), K and V
 * alike; token t of sequence b lives in block block_tables[b][t / block_size],
 * slot t % block_size, as in orthocache_hip.h.  Entries past a sequence's own
 * blocks are -1 (any value outside [0, num_blocks) is never followed: it sets
 * *error_flag, if given, where a token needs it).
 */
#ifndef ORTHOCACHE_PAGED_H
#define ORTHOCACHE_PAGED_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/*
 * oc_apply_rotary -- rotary positions.  Pair i (0 <= i < rotary_dim / 2) of a
 * row x is (x[i], x[i + rotary_dim / 2]), or with interleaved (x[2i],
 * x[2i + 1]).  At position n its angle is a = n * inv_freq[i], formed and
 * reduced in float64, and
 *   y = scale * (x0 cos a - x1 sin a, x1 cos a + x0 sin a)
 * in float32, rounded once; with backward the transposed rotation (a -> -a),
 * which takes the gradient of y to that of x.  Columns from rotary_dim on are
 * copied.  Two tensors (queries and keys) share one launch; x[1] may be NULL.
 * y may be x (in place).
 */
typedef struct oc_rotary_params {
  const void* x[2];               /* (batch, heads[i], tokens, head_dim), head_dim contiguous */
  void* y[2];
  int64_t x_stride_b[2], x_stride_h[2], x_stride_s[2];  /* elements */
  int64_t y_stride_b[2], y_stride_h[2], y_stride_s[2];
  int32_t heads[2];
  int32_t dtype;                  /* OC_F32 / OC_F16 / OC_BF16 */
  int32_t batch, tokens, head_dim, rotary_dim;
  int32_t interleaved, backward;
  int32_t positions_64;           /* positions are int64 (else int32) */
  const void* positions;          /* (batch, tokens), tokens contiguous */
  int64_t positions_stride_b;     /* 0: shared by the batch */
  const double* inv_freq;         /* (rotary_dim / 2) radians per position */
  float scale;
} oc_rotary_params;

int oc_apply_rotary(const oc_rotary_params* p, void* stream);

/*
 * oc_append_paged -- the new tokens of every sequence go into its pages:
 * row i of sequence b's rows cu_seqlens[b] .. cu_seqlens[b + 1) (row b alone
 * without cu_seqlens) is its token n = context_lens[b] + i - cu_seqlens[b].
 * Its keys, turned as by oc_apply_rotary (inv_freq NULL: not turned) at
 * position positions[i] (NULL: n), and its values are written to that token's
 * slot; its queries, turned alike, to q_out.  fp8-e4m3fn caches take
 * round(clamp(x / scale, -448, 448)), a NaN staying NaN.  Sequences with
 * context_lens[b] < 0 and rows outside every sequence write nothing to the
 * cache and zeros to q_out.  A token whose block id is outside [0,
 * num_blocks), or past the table's columns, writes nothing to the cache and
 * sets *error_flag, if given.  cu_seqlens must not decrease.
 */
typedef struct oc_append_params {
  const void* q;                  /* (tokens, num_q_heads, head_dim) or NULL */
  const void* k;                  /* (tokens, num_kv_heads, head_dim) */
  const void* v;
  void* q_out;                    /* (tokens, num_q_heads, head_dim) */
  int64_t q_stride_s, q_stride_h, k_stride_s, k_stride_h, v_stride_s, v_stride_h;
  int64_t q_out_stride_s, q_out_stride_h;
  void* k_cache;
  void* v_cache;
  int64_t k_cache_stride_b, k_cache_stride_h, k_cache_stride_s;  /* block, head, slot */
  int64_t v_cache_stride_b, v_cache_stride_h, v_cache_stride_s;
  int32_t dtype;                  /* of q, k, v: OC_F32 / OC_F16 / OC_BF16 */
  int32_t cache_dtype;            /* OC_F32 .. OC_FP8_E4M3FN */
  int32_t tokens, num_seqs, num_q_heads, num_kv_heads, head_dim, rotary_dim;
  int32_t block_size;             /* a power of two */
  int32_t max_blocks;             /* columns of the table */
  int64_t num_blocks;
  const int32_t* block_tables;
  int64_t bt_stride;
  const int32_t* context_lens;    /* (num_seqs) tokens cached before the call */
  const int32_t* cu_seqlens;      /* (num_seqs + 1) or NULL (tokens == num_seqs) */
  const void* positions;          /* (tokens) or NULL */
  int32_t positions_64, interleaved;
  const double* inv_freq;         /* (rotary_dim / 2) or NULL */
  float scale, k_scale, v_scale;
  int32_t* error_flag;
} oc_append_params;

int oc_append_paged(const oc_append_params* p, void* stream);

/*
 * What oc_attend_paged and oc_attend_prompt do to the scores.  For the query
 * at place i and the key at place j:
 *   z = scale * q.k;  softcap > 0: z = softcap * tanh(z / softcap)
 *   slopes: z -= slopes[head] * |i - j|
 * and j is seen by i when
 *   (j <= i and (window <= 0 or i - j < window)) or j < prefix_lens[b]
 * (and more, said at the entry points).  A query that sees nothing gets
 * zeros; what is not seen has no effect, NaN and infinities among it.
 */
typedef struct oc_score_mods {
  float scale, softcap;
  const float* slopes;            /* (num_q_heads) or NULL */
  const int32_t* prefix_lens;     /* (batch) or NULL */
  const uint8_t* evict;           /* (batch, num_kv_heads, evict_cols): 1 = the 64-token tile is evicted, or NULL */
  int64_t evict_stride_b, evict_stride_h;
  int32_t evict_cols;             /* tiles past them are not evicted */
  int32_t window;
} oc_score_mods;

/*
 * oc_attend_paged -- attention of one new token per sequence, which is the
 * last cached one: place i = context_lens[b] - 1 over places j <= i.  Complete
 * 64-token tiles may be evicted; a partial last tile is attended.  K =
 * k_scale * cache, V = v_scale * cache.  float32 accumulation, out in dtype.
 * context_lens are clamped to 0 .. max_blocks * block_size.
 */
typedef struct oc_attend_paged_params {
  const void* q;                  /* (num_seqs, num_q_heads, head_dim) */
  int64_t q_stride_b, q_stride_h;
  const void* k;
  const void* v;
  int64_t k_stride_b, k_stride_h, k_stride_s;  /* block, head, slot */
  int64_t v_stride_b, v_stride_h, v_stride_s;
  const int32_t* block_tables;
  int64_t bt_stride, num_blocks;
  const int32_t* context_lens;    /* (num_seqs) */
  int32_t max_blocks, block_size;
  int32_t dtype;                  /* of q and out: OC_F32 / OC_F16 / OC_BF16 */
  int32_t cache_dtype;            /* dtype or OC_FP8_E4M3FN */
  int32_t num_seqs, num_q_heads, num_kv_heads, head_dim;  /* head_dim a multiple of 8 up to 512 */
  float k_scale, v_scale;
  oc_score_mods mods;
  int32_t num_splits;             /* parts of a sequence's tiles (1024 at most); 0: chosen from the sizes */
  int32_t portable;               /* 1: the portable kernel whatever the shape */
  void* out;                      /* (num_seqs, num_q_heads, head_dim) */
  int64_t out_stride_b, out_stride_h;
  int32_t* error_flag;
  void* workspace;                /* oc_attend_paged_workspace_size(p) bytes, any content */
  size_t workspace_bytes;
} oc_attend_paged_params;

size_t oc_attend_paged_workspace_size(const oc_attend_paged_params* p);
int oc_attend_paged(const oc_attend_paged_params* p, void* stream);

/*
 * oc_attend_prompt -- attention of q_len queries over kv_len keys, query s at
 * place i = s + kv_len - q_len.  With documents, i sees j only when
 * documents[b][i] == documents[b][j] and neither is negative.  Complete
 * 64-token tiles may be evicted.  dtype F32 / F16 / BF16, head_dim 64 or
 * 128, kv_len up to 2^24, float32 accumulation; 16-bit probabilities are
 * rounded once to the type before P V.
 */
typedef struct oc_attend_prompt_params {
  const void* q;                  /* (batch, num_q_heads, q_len, head_dim) */
  int64_t q_stride_b, q_stride_h, q_stride_s;
  const void* k;                  /* (batch, num_kv_heads, kv_len, head_dim) */
  int64_t k_stride_b, k_stride_h, k_stride_s;
  const void* v;
  int64_t v_stride_b, v_stride_h, v_stride_s;
  void* out;                      /* (batch, num_q_heads, q_len, head_dim) */
  int64_t out_stride_b, out_stride_h, out_stride_s;
  int32_t dtype;
  int32_t batch, num_q_heads, num_kv_heads, q_len, kv_len, head_dim;
  const int32_t* documents;       /* (batch, kv_len) or NULL */
  int64_t documents_stride_b;
  oc_score_mods mods;
  void* workspace;                /* oc_attend_prompt_workspace_size(p) bytes, 16-byte aligned, any content */
  size_t workspace_bytes;
} oc_attend_prompt_params;

/* bytes of workspace oc_attend_prompt needs, from p's sizes, types, window and whether it has documents and prefix_lens
   (0 for many calls without documents) */
size_t oc_attend_prompt_workspace_size(const oc_attend_prompt_params* p);
int oc_attend_prompt(const oc_attend_prompt_params* p, void* stream);

/* bits of a page operator's status */
#define OC_PAGES_NO_ROOM 1     /* fewer free blocks than the call needs */
#define OC_PAGES_BAD_PARENT 2  /* a parent outside [-1, num_seqs) */
#define OC_PAGES_TOO_LONG 4    /* a sequence needs more blocks than the table has columns */
#define OC_PAGES_BAD_BLOCK 8   /* a table entry that is needed is outside [0, num_blocks) */

/*
 * oc_fork_pages -- child i of the new tables continues sequence parents[i],
 * with room for new_tokens[i] more (-1: an empty sequence without room).  A parent with no child
 * ends.  Full blocks are shared; a last block that is not full has one owner:
 * the parent's first child where ref_counts says that no one else holds it,
 * and the others get a copy (of the slots that hold tokens, in every layer, K
 * and V) in a fresh block.  Fresh blocks are those with ref_counts 0 before
 * the call, lowest first, in the order of the children.  A row of the result
 * holds ceil((len + new_tokens) / block_size) blocks, then -1; entries of the
 * old tables past a sequence's tokens are given back.  ref_counts counts a
 * block's holders: the result has one less for each old row that held it and
 * one more for each new row.  Outputs must not overlap the inputs.
 * *status gets 0, or bits OC_PAGES_*: then no block is written, the new
 * tables are empty (-1, lengths 0) and the new counts the old ones.  Only an
 * entry outside [0, num_blocks) before a sequence's last one lets the call go
 * on: it becomes -1 in the children, and OC_PAGES_BAD_BLOCK is set.  At most
 * 2^20 table columns and 2^30 blocks.
 */
typedef struct oc_fork_params {
  void* k_cache;                  /* (layers, num_blocks, num_kv_heads, block_size, head_dim), rows contiguous */
  void* v_cache;
  int64_t k_stride_l, k_stride_b, k_stride_h, k_stride_s;
  int64_t v_stride_l, v_stride_b, v_stride_h, v_stride_s;
  int32_t cache_dtype, layers, num_kv_heads, head_dim;
  int32_t block_size;
  int32_t num_seqs, num_children; /* up to 4096 each */
  int32_t max_blocks, out_max_blocks;
  int64_t num_blocks;
  const int32_t* block_tables;
  int64_t bt_stride;
  const int32_t* context_lens;
  const int32_t* ref_counts;      /* (num_blocks) */
  const int32_t* parents;         /* (num_children) or NULL: child i continues sequence i (num_children == num_seqs) */
  const int32_t* new_tokens;      /* (num_children) or NULL: 0 */
  int32_t* out_block_tables;
  int64_t out_bt_stride;
  int32_t* out_context_lens;
  int32_t* out_ref_counts;
  int32_t* status;
  void* workspace;                /* oc_fork_pages_workspace_size(p) bytes, any content */
  size_t workspace_bytes;
} oc_fork_params;

size_t oc_fork_pages_workspace_size(const oc_fork_params* p);
int oc_fork_pages(const oc_fork_params* p, void* stream);

/*
 * oc_evict_pages -- the complete 64-token tiles that every kv head evicts leave
 * their sequences: out_block_tables has the blocks of the others in order,
 * then -1; lengths shrink by 64 tokens a tile; the blocks lose a holder.
 * tile_map[b][t] is the old tile of new tile t (-1 past the last).  Entries
 * past a sequence's tokens are given back.  block_size divides 64.  Outputs
 * must not overlap the inputs.  *status as oc_fork_pages, OC_PAGES_BAD_BLOCK
 * alone: an entry outside [0, num_blocks) among the kept ones becomes -1, and
 * none is counted.
 */
typedef struct oc_evict_params {
  int32_t num_seqs, num_kv_heads, block_size, max_blocks;
  int64_t num_blocks;
  const int32_t* block_tables;
  int64_t bt_stride;
  const int32_t* context_lens;
  const int32_t* ref_counts;
  const uint8_t* evict;           /* (num_seqs, num_kv_heads, evict_cols) */
  int64_t evict_stride_b, evict_stride_h;
  int32_t evict_cols;
  int32_t tile_map_cols;          /* ceil(max_blocks * block_size / 64) */
  int32_t* out_block_tables;
  int64_t out_bt_stride;
  int32_t* out_context_lens;
  int32_t* out_ref_counts;
  int32_t* tile_map;              /* (num_seqs, tile_map_cols) */
  int32_t* status;
} oc_evict_params;

int oc_evict_pages(const oc_evict_params* p, void* stream);

/* sizeof of the parameter blocks as compiled, for binding checks: rotary,
 * append, attend_paged, attend_prompt, fork, evict */
void oc_paged_params_bytes(size_t sizes[6]);

#ifdef __cplusplus
}
#endif

#endif /* ORTHOCACHE_PAGED_H */
