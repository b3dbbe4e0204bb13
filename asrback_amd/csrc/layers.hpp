// Entry points of the package's own model layers (asrback_amd/*.py): the
// element-wise work around the attention calls of asrattn.h.  Not part of
// the C ABI that replaces the reference's attention ops; the same
// conventions hold (device pointers, element strides, a stream, no
// allocation, no synchronization, asrattn_last_error for messages).
#pragma once

#include <stddef.h>
#include <stdint.h>

#include "asrattn.h"

extern "C" {

// The rows a prompt pass prepares for its attention: per-head RMSNorm and
// rotary embedding of the queries and keys, the values' RMSNorm without
// weights (v_norm), and the writes of keys and values to the cache.
//
//   q' = rot(norm(q, q_norm), cos, sin)     -> q_out
//   k' = rot(norm(k, k_norm), cos, sin)     -> k_out and the cache
//   v' = norm(v, 1) (v_norm != 0; else v)   -> v_out (if given) and the cache
//
// with asrattn_decode_append's norm and rot, rounded in the element type as
// the reference's ops round.  Token t of sequence b (batch x tokens of them)
// is row b * tokens + t of the outputs, which are contiguous.  Its cache slot
// is (rows[b * tokens + t], positions[b * tokens + t]), or (rows[b], t) with
// positions NULL; negative indices count from the end, and slots outside the
// cache are not written.  With a block table (int32, bt_stride entries per
// cache row) the slot lies in page block_table[row][position / page_size]
// of the pool, or in the sink page num_pages where that is outside [0,
// num_pages).  k NULL: queries only.
typedef struct asrlayer_prompt_params {
  const void *q, *k, *v;
  void *q_out, *k_out, *v_out;
  void *k_cache, *v_cache;
  int64_t q_batch_stride, q_token_stride, q_head_stride;
  int64_t k_batch_stride, k_token_stride, k_head_stride;
  int64_t v_batch_stride, v_token_stride, v_head_stride;
  // Cache: row (paged: page), position and head strides, and its extent.
  int64_t kc_row_stride, kc_pos_stride, kc_head_stride;
  int64_t vc_row_stride, vc_pos_stride, vc_head_stride;
  int64_t cache_rows, cache_length;
  const int64_t *rows, *positions;
  const int32_t* block_table;
  int64_t bt_stride;
  int32_t page_size, num_pages;
  const void *q_norm, *k_norm;  // (head_dim,)
  const void *cos, *sin;        // (batch, tokens, head_dim) by the strides below
  int64_t rope_batch_stride, rope_token_stride;
  float q_eps, k_eps, v_eps;
  int32_t v_norm;
  int32_t batch, tokens, heads_q, heads_kv, head_dim, dtype;
} asrlayer_prompt_params;

int asrlayer_prompt_rows(const asrlayer_prompt_params* params, void* stream);

// Linear layers over the few rows of a decoder step:
//
//   out[i] = act(norm(x) w[i]^T + b[i])             (i < 3, n[i] > 0)
//   out[i] = residual + (norm(x) w[i]^T + b[i])     (residual given)
//
// with norm the layer norm over the k inputs (ln_weight NULL: none), sums in
// float32 and each result rounded in the element type where the separate
// torch ops round: after the norm, after the product and bias, after the
// activation, after the residual sum.  x: (rows, k), rows x_row_stride
// apart; w[i]: (n[i], k), contiguous; b[i]: (n[i]) or NULL; out[i]: (rows,
// n[i]), contiguous; residual: (rows, n[0]), with one matrix.  act 0: none,
// 1: gelu (exact).  rows 1 .. 16; k a multiple of 16 bytes and at most 1024
// times that.
typedef struct asrlayer_linear_params {
  const void* x;
  int64_t x_row_stride;
  const void *ln_weight, *ln_bias;
  const void* w[3];
  const void* b[3];
  void* out[3];
  const void* residual;
  int64_t r_row_stride;
  float ln_eps;
  int32_t n[3];
  int32_t rows, k, act, dtype;
} asrlayer_linear_params;

int asrlayer_rows_linear(const asrlayer_linear_params* params, void* stream);

// A decoder step's input: out[r] = token_weight[tokens[r * token_stride]] +
// position_weight[positions[r]], tables (vocab, width) and (length, width), all
// contiguous; rows whose token or position lies outside are NaN.  width a
// multiple of 16 bytes.
typedef struct asrlayer_embed_params {
  const void *token_weight, *position_weight;
  const int64_t *tokens, *positions;
  void* out;
  int64_t token_stride, vocab, length;
  int32_t rows, width, dtype;
} asrlayer_embed_params;

int asrlayer_embed_rows(const asrlayer_embed_params* params, void* stream);

// A linear layer over bf16 rows (batch x rows of k inputs, n outputs each):
//
//   out[b, t, :] = x[b, t, :] w^T + bias        (accumulate 0; bias or NULL)
//   out[b, t, :] = out[b, t, :] + x[b, t, :] w^T    (accumulate 1, no bias)
//
// with float32 sums, rounded once.  w (n, k) contiguous; rows x_row_stride
// and out_row_stride apart.  used (int32[batch], device, or NULL): rows t >=
// used[b] are neither read nor written.  k a multiple of 64, n of 8.
typedef struct asrlayer_gemm_params {
  const void *x, *w, *bias;
  void* out;
  const int32_t* used;
  int64_t x_batch_stride, x_row_stride, out_batch_stride, out_row_stride;
  int32_t batch, rows, n, k, accumulate;
} asrlayer_gemm_params;

int asrlayer_gemm(const asrlayer_gemm_params* params, void* stream);

// Attention of drafted tokens over a cache and the drafted tokens before them:
// per sequence b, token t, query head h of kv head h / (heads_q / heads_kv),
//
//   s_j  = scale q[b, t, h] . k[b, j]          j < n_b
//   s'_i = scale q[b, t, h] . k_draft[b, i]    bit i of masks[b, t] set
//   out[b, t, h] = softmax over both, times v and v_draft
//
// n_b = lengths[b] (int32, or int64 with lengths64) clamped to [0, max_len_k].
// A token with mask 0 is none: its rows are zeros.  Mask bits at tokens and
// past them count for nothing.  tokens at most 64; q, out (batch, tokens,
// heads_q, head_dim); k_draft, v_draft (batch, tokens, heads_kv, head_dim);
// k, v (batch, max_len_k, heads_kv, head_dim), or with a block table pools as
// asrattn_decode_paged takes them (keys of entries outside the pool are
// skipped).  head_dim 64, 128 or 256.  The workspace holds the partials of
// split keys (asrlayer_tree_workspace_size, 256-byte aligned); its contents
// before the call do not matter, and calls that share it run in stream order.
typedef struct asrlayer_tree_params {
  const void *q, *k, *v, *k_draft, *v_draft;
  void* out;
  int64_t q_batch_stride, q_token_stride, q_head_stride;
  int64_t k_batch_stride, k_token_stride, k_head_stride;
  int64_t v_batch_stride, v_token_stride, v_head_stride;
  int64_t kd_batch_stride, kd_token_stride, kd_head_stride;
  int64_t vd_batch_stride, vd_token_stride, vd_head_stride;
  int64_t o_batch_stride, o_token_stride, o_head_stride;
  const int64_t* masks;  // (batch, tokens): rows masks_batch_stride apart
  int64_t masks_batch_stride;
  const void* lengths;
  const int32_t* block_table;
  int64_t bt_stride, k_page_stride, v_page_stride;
  int32_t page_size, num_pages;
  int32_t lengths64, batch, tokens, heads_q, heads_kv, head_dim, max_len_k, dtype;
  float scale;
} asrlayer_tree_params;

int asrlayer_tree(const asrlayer_tree_params* params, void* workspace, size_t workspace_bytes, void* stream);

// Workspace bytes of these sizes (tensors and strides may be unset): 0 when the
// call runs unsplit, (size_t)-1 for sizes it does not take; otherwise enough for
// any smaller batch and fewer tokens as well.
size_t asrlayer_tree_workspace_size(const asrlayer_tree_params* params);

// Ancestor masks of drafted trees: masks[b, t] has bit t and the bits of t's
// ancestors.  parents (batch, tokens), rows parents_batch_stride apart: a
// token before t, or -1 (as is any value from t on) for none; below -1 the
// token is padding and its mask 0.  depths[b, t] counts t's ancestors (0 for
// padding).  tokens at most 64; masks and depths contiguous.
int asrlayer_tree_masks(const int64_t* parents, int64_t parents_batch_stride, int64_t batch, int32_t tokens,
                        int64_t* masks, int64_t* depths, void* stream);

// The walk of a greedy choice down drafted trees, from token 0: the next token
// is the first one after it whose parent it is and that equals its choice.
//
//   path[b, i]    the i-th token of the walk, -1 past its end
//   emitted[b, i] choices[b, path[b, i]], -1 past its end
//   count[b]      its length: 0 where limit[b] <= 0 or token 0 is padding
//                 (parent below -1), else at least 1 and at most limit[b]
//
// tokens, choices, path, emitted (batch, width) contiguous; parents rows
// parents_batch_stride apart; limit (batch) or NULL; width at most 64.
int asrlayer_accept(const int64_t* tokens, const int64_t* parents, int64_t parents_batch_stride,
                    const int64_t* choices, const int64_t* limit, int64_t batch, int32_t width, int64_t* path,
                    int64_t* emitted, int64_t* count, void* stream);

// Accepted tokens' keys and values from the draft buffers into the cache, for
// every layer l, sequence b and i < count[b]:
//
//   k[l, b, lengths[b] + i] = k_draft[l, b, path[b, i]]     and v likewise
//
// k, v (layers, batch, max_len_k, heads_kv, head_dim), or with a block table
// pools (layers, num_pages, page_size, heads_kv, head_dim); drafts (layers,
// batch, tokens, heads_kv, head_dim).  Positions outside [0, max_len_k) or on
// no page, and path entries outside [0, tokens), are not written.
typedef struct asrlayer_commit_params {
  const void *k_draft, *v_draft;
  void *k, *v;
  int64_t kd_layer_stride, kd_batch_stride, kd_token_stride, kd_head_stride;
  int64_t vd_layer_stride, vd_batch_stride, vd_token_stride, vd_head_stride;
  // Batch strides are page strides with a block table.
  int64_t k_layer_stride, k_batch_stride, k_token_stride, k_head_stride;
  int64_t v_layer_stride, v_batch_stride, v_token_stride, v_head_stride;
  const int64_t *path, *count;  // (batch, tokens) and (batch), contiguous
  const void* lengths;
  const int32_t* block_table;
  int64_t bt_stride;
  int32_t page_size, num_pages;
  int32_t lengths64, layers, batch, tokens, heads_kv, head_dim, max_len_k, dtype;
} asrlayer_commit_params;

int asrlayer_commit(const asrlayer_commit_params* params, void* stream);

// Rows through a matrix of 4-bit weights with group scales:
//
//   out[r, n] = sum_k x[r, k] scale[n, k / group] (q[n, k] - zero[n, k / group]) (+ bias[n])
//
// q and zero in 0 .. 15 (zeros NULL: 8), sums in float32, rounded once.  x
// rows x_row_stride apart; out rows out_row_stride apart; scales and bias in
// x's type; group 32, 64 or 128, k a multiple of it.  The matrix lies in blocks
// of 16 outputs by 128 inputs, padded to whole blocks (scales of padding 0):
//
//   packed (n / 16, k / 128, 64, 4) dwords: dword s of lane 16 g + i holds
//     output i's inputs 32 s + 8 g + j, j = 0 2 4 6 1 3 5 7 from the low nibble up
//   scales (n / 16, k / 128, 4, 128 / group, 4): of outputs 4 g .. 4 g + 3, g the
//     third index, over the block's groups
//   zeros  the same, four to two bytes, from the low nibble up
typedef struct asrlayer_linear4_params {
  const void* x;
  int64_t x_row_stride;
  const void *packed, *scales, *zeros, *bias;
  void* out;
  int64_t out_row_stride;
  int64_t rows;
  int32_t n, k, group, dtype;
} asrlayer_linear4_params;

int asrlayer_linear4(const asrlayer_linear4_params* params, void* stream);

}  // extern "C"
