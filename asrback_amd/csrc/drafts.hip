// What surrounds the attention of drafted trees (tree.hip): the trees' ancestor
// masks, the greedy choice's walk down them, and the accepted tokens' way into
// the cache.  All three are bound by their launch (a kernel that does nothing
// takes 1.8 us): a tree has at most 64 tokens, one to a lane.
#include "kernels.hpp"
#include "row_ops.hpp"

namespace asrattn {
namespace {

// A wave per tree.  Parents come before their children, so in step t lane t's
// mask is final once lane t - 1's is: a scan over the lanes, each step one lane
// read.
__global__ __launch_bounds__(64) void tree_masks_kernel(const int64_t* parents, int64_t parents_batch_stride, int tokens,
                                                        int64_t* masks, int64_t* depths) {
  const int64_t b = blockIdx.x;
  const int lane = threadIdx.x;
  const int64_t parent = parents[b * parents_batch_stride + min(lane, tokens - 1)];
  const int up = parent >= 0 && parent < lane ? (int)parent : -1;
  uint64_t mask = lane < tokens && parent >= -1 ? 1ull << lane : 0ull;
  for (int t = 1; t < tokens; ++t) {
    const int from = __builtin_amdgcn_readlane(up, t);
    if (from < 0) continue;  // uniform
    const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)mask, from);
    const uint32_t hi = __builtin_amdgcn_readlane((uint32_t)(mask >> 32), from);
    if (lane == t) mask |= (uint64_t)hi << 32 | lo;
  }
  if (lane < tokens) {
    masks[b * tokens + lane] = (int64_t)mask;
    depths[b * tokens + lane] = max((int)__popcll(mask) - 1, 0);
  }
}

// A wave per tree: lane j holds token j.  Each step is one comparison on all
// lanes, a ballot and two lane reads of the token found; it ends because tokens
// rise.
__global__ __launch_bounds__(64) void accept_kernel(const int64_t* tokens, const int64_t* parents,
                                                    int64_t parents_batch_stride, const int64_t* choices,
                                                    const int64_t* limit, int width, int64_t* path, int64_t* emitted,
                                                    int64_t* count) {
  const int64_t b = blockIdx.x;
  const int lane = threadIdx.x;
  const int at = min(lane, width - 1);
  const int64_t token = tokens[b * width + at], parent = parents[b * parents_batch_stride + at];
  const int64_t choice = choices[b * width + at];
  const int64_t most = limit != nullptr ? load_uniform(limit + b) : width;
  int now = 0, steps = 0;
  int64_t mine = -1, said = -1;
  bool going = most > 0 && __builtin_amdgcn_readfirstlane((int)(parent >= -1)) != 0;
  while (going) {
    const uint64_t chosen = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(choice >> 32), now) << 32 |
                            (uint32_t)__builtin_amdgcn_readlane((int)choice, now);
    if (lane == steps) {
      mine = now;
      said = (int64_t)chosen;
    }
    ++steps;
    const uint64_t next = __ballot(lane < width && lane > now && parent == now && token == (int64_t)chosen);
    going = next != 0 && steps < most;
    if (going) now = __ffsll((unsigned long long)next) - 1;
  }
  if (lane < width) {
    path[b * width + lane] = mine;
    emitted[b * width + lane] = said;
  }
  if (lane == 0) count[b] = steps;
}

// A workgroup per (accepted step, sequence, layer) copies a position's keys and
// values, 16 bytes a thread; the others end at once.
__global__ __launch_bounds__(256) void commit_kernel(const asrlayer_commit_params p, int es) {
  const int step = blockIdx.x, b = blockIdx.y, layer = blockIdx.z;
  // Loaded together: each would be a round trip of its own.
  const int64_t count = load_uniform(p.count + b), from = load_uniform(p.path + (int64_t)b * p.tokens + step);
  const int64_t n = p.lengths64 ? load_uniform(static_cast<const int64_t*>(p.lengths) + b)
                                : (int64_t)load_uniform(static_cast<const int32_t*>(p.lengths) + b);
  if (step >= count || from < 0 || from >= p.tokens || n < 0 || n >= p.max_len_k - step) return;
  const int to = (int)n + step;
  int row = b, slot = to;
  if (p.block_table != nullptr) {
    const int page = to / p.page_size;
    row = load_uniform(p.block_table + (int64_t)b * p.bt_stride + page);
    slot = to - page * p.page_size;
    if (row < 0 || row >= p.num_pages) return;
  }
  const char* ks = static_cast<const char*>(p.k_draft) +
                   (layer * p.kd_layer_stride + b * p.kd_batch_stride + from * p.kd_token_stride) * es;
  const char* vs = static_cast<const char*>(p.v_draft) +
                   (layer * p.vd_layer_stride + b * p.vd_batch_stride + from * p.vd_token_stride) * es;
  char* kt = static_cast<char*>(p.k) + (layer * p.k_layer_stride + row * p.k_batch_stride + slot * p.k_token_stride) * es;
  char* vt = static_cast<char*>(p.v) + (layer * p.v_layer_stride + row * p.v_batch_stride + slot * p.v_token_stride) * es;
  const int vecs = p.head_dim * es / 16;
  for (int i = threadIdx.x; i < p.heads_kv * vecs; i += 256) {
    const int64_t h = i / vecs, at = i % vecs * 16;
    const uint4 x = *reinterpret_cast<const uint4*>(ks + h * p.kd_head_stride * es + at);
    const uint4 y = *reinterpret_cast<const uint4*>(vs + h * p.vd_head_stride * es + at);
    *reinterpret_cast<uint4*>(kt + h * p.k_head_stride * es + at) = x;
    *reinterpret_cast<uint4*>(vt + h * p.v_head_stride * es + at) = y;
  }
}

}  // namespace

hipError_t launch_tree_masks(const int64_t* parents, int64_t parents_batch_stride, int64_t batch, int tokens,
                             int64_t* masks, int64_t* depths, hipStream_t stream) {
  hipLaunchKernelGGL(tree_masks_kernel, dim3((unsigned)batch), dim3(64), 0, stream, parents, parents_batch_stride, tokens,
                     masks, depths);
  return hipGetLastError();
}

hipError_t launch_accept(const int64_t* tokens, const int64_t* parents, int64_t parents_batch_stride,
                         const int64_t* choices, const int64_t* limit, int64_t batch, int width, int64_t* path,
                         int64_t* emitted, int64_t* count, hipStream_t stream) {
  hipLaunchKernelGGL(accept_kernel, dim3((unsigned)batch), dim3(64), 0, stream, tokens, parents, parents_batch_stride,
                     choices, limit, width, path, emitted, count);
  return hipGetLastError();
}

hipError_t launch_commit(const asrlayer_commit_params& p, hipStream_t stream) {
  hipLaunchKernelGGL(commit_kernel, dim3(p.tokens, p.batch, p.layers), dim3(256), 0, stream, p,
                     p.dtype == ASRATTN_BF16 ? 2 : 4);
  return hipGetLastError();
}

}  // namespace asrattn
