// Launchers of the attention kernels; the C ABI (api.hip) validates the
// parameters before calling them.
#pragma once

#include <hip/hip_runtime.h>

#include "asrattn.h"
#include "fsmn.hpp"
#include "layers.hpp"

namespace asrattn {

// Decoder step over `splits` workgroups per (sequence, kv head); for
// splits > 1 the workspace holds the partial outputs
// float[batch][heads_q][splits][head_dim], (max, sum) pairs
// float[batch][heads_q][splits][2] and an arrival word per (sequence, kv
// head); the split that arrives last folds the partials.
// append: the fused prologue of asrattn_decode_append, or null; paged: the
// page table of asrattn_decode_paged, or null.
hipError_t launch_decode(const asrattn_decode_params& p, const asrattn_append_params* append,
                         const asrattn_paged_kv* paged, int splits, float* ws_o, float* ws_ml,
                         unsigned long long* ws_arrive, hipStream_t stream);
// The most keys a row can use (its window or the cache), waves per workgroup
// (page_size 0: not paged) and key rows one wave load covers.
int decode_span(const asrattn_decode_params& p);
int decode_waves(const asrattn_decode_params& p, int splits, int page_size);
int decode_keys_per_wave(int dtype, int head_dim);
bool decode_supported(int dtype, int head_dim, int group);

// Multi-row forward on matrix cores with K/V streamed into an LDS ring by
// DMA (bf16, head_dim 64 or 128, K/V spans addressable with 32-bit offsets).
// fsmn (or null): the FSMN memory computed in the same launch (kernel size
// at most kFsmnFusedKernel).
hipError_t launch_fwd_ring(const asrattn_fwd_params& p, const FsmnArgs* fsmn, hipStream_t stream);
bool fwd_ring_supported(const asrattn_fwd_params& p);

// Greedy choice per row of fp32 logits: argmax (first index on ties) and its
// log-probability; suppress (uint8 per vocabulary entry) may be null.
// Splits per row of the two-launch choice (1: one workgroup per row).
int choose_splits(int64_t rows, int64_t vocab);
// Workspace bytes of the split form (0 when one workgroup per row is used).
size_t choose_workspace_bytes(int64_t rows, int64_t vocab);
// workspace: at least choose_workspace_bytes, or null for one workgroup per row.
hipError_t launch_choose(const float* logits, int64_t rows, int64_t vocab, int64_t row_stride, const uint8_t* suppress,
                         int64_t* token, float* logprob, void* workspace, hipStream_t stream);

// Multi-row forward in fp32 on the matrix cores (head_dim 64, 128, 256 or
// 512, K/V spans addressable with 32-bit offsets).
hipError_t launch_fwd_f32mm(const asrattn_fwd_params& p, hipStream_t stream);
bool fwd_f32mm_supported(const asrattn_fwd_params& p);
// Its head_dim 64 (fwd_f32row.hip), and whether that kernel is the faster one.
bool fwd_f32row_takes(const asrattn_fwd_params& p);
hipError_t launch_fwd_f32row(const asrattn_fwd_params& p, hipStream_t stream);

// Multi-row forward on the vector ALUs (fp32 or bf16): the fallback for
// layouts the matrix-core kernels do not address, and the reference-precision
// check of those kernels.
hipError_t launch_fwd_valu(const asrattn_fwd_params& p, hipStream_t stream);
bool fwd_valu_supported(int dtype, int head_dim);

// Blocked local attention with relative position scores (asrattn_local),
// and the LDS it stages per workgroup.
hipError_t launch_local(const asrattn_local_params& p, hipStream_t stream);
size_t local_lds_bytes(const asrattn_local_params& p);

// SAN-M's FSMN memory on its own (fp32 or bf16, head_dim 64 or 128, kernel
// size at most kFsmnMaxKernel) for the padded layout of p (values p.v, frame
// counts p.seqused_k).
hipError_t launch_fsmn(const asrattn_fwd_params& p, const FsmnArgs& f, hipStream_t stream);

// A prompt pass's rows (asrlayer_prompt_rows; head_dim 64, 128, 256 or 512).
hipError_t launch_prompt_rows(const asrlayer_prompt_params& p, hipStream_t stream);

// A decoder step's linear layers over few rows (asrlayer_rows_linear).
hipError_t launch_rows_linear(const asrlayer_linear_params& p, hipStream_t stream);

// Token and position embeddings of a decoder step (asrlayer_embed_rows).
hipError_t launch_embed_rows(const asrlayer_embed_params& p, hipStream_t stream);

// Attention of drafted trees (asrlayer_tree) over `splits` workgroups per
// (sequence, kv head, block of query rows); for splits > 1 the workspace holds
// the partials and an arrival word per such unit, and the split that arrives
// last folds them.
struct TreePlan {
  int row_tiles;   // 16-row tiles a workgroup holds
  int row_blocks;  // workgroups over a kv head's query rows
  int splits;
  int waves;        // of a workgroup
  bool fold_apart;  // fold the partials in a launch of its own
};
TreePlan tree_plan(const asrlayer_tree_params& p);
hipError_t launch_tree(const asrlayer_tree_params& p, const TreePlan& plan, float* ws_o, float* ws_ml,
                       unsigned long long* ws_arrive, hipStream_t stream);

// Drafted trees' masks, walk and commit (asrlayer_tree_masks, asrlayer_accept,
// asrlayer_commit).
hipError_t launch_tree_masks(const int64_t* parents, int64_t parents_batch_stride, int64_t batch, int tokens,
                             int64_t* masks, int64_t* depths, hipStream_t stream);
hipError_t launch_accept(const int64_t* tokens, const int64_t* parents, int64_t parents_batch_stride,
                         const int64_t* choices, const int64_t* limit, int64_t batch, int width, int64_t* path,
                         int64_t* emitted, int64_t* count, hipStream_t stream);
hipError_t launch_commit(const asrlayer_commit_params& p, hipStream_t stream);

// Rows through a matrix of 4-bit weights (asrlayer_linear4).
hipError_t launch_linear4(const asrlayer_linear4_params& p, hipStream_t stream);

// A tag for a split launch's arrival words that no other launch of the process
// has (decode.hip).
unsigned long long launch_tag();

// A linear layer over bf16 rows (asrlayer_gemm).
hipError_t launch_gemm(const asrlayer_gemm_params& p, hipStream_t stream);

}  // namespace asrattn
