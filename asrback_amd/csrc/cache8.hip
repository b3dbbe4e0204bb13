// The 8-bit cache's writes and reading back (asrlayer_write8, asrlayer_read8).
//
// Both are bound by memory: a write reads each new row (one head of one token)
// once and writes half (float32: a quarter) of it and its scale; reading back is the
// reverse.  A write's workgroup takes one token, whose slot it looks up once; a row
// is held by LPK lanes of 16 bytes, neighbouring lane groups take neighbouring
// rows, so a wave reads whole cache lines, and the row's largest magnitude is a
// maximum over its lanes.  The norms and the rotation of a decoder's queries and
// keys happen on the same registers first, as in prompt_rows.hip.
#include "kernels.hpp"
#include "layers.hpp"
#include "round8.hpp"
#include "row_ops.hpp"

namespace asrattn {
namespace {

constexpr int kThreads = 256;

// The pool entry and the position in it of position pos of sequence b; entry < 0:
// none.
struct Slot {
  int64_t entry, pos;
};
__device__ __forceinline__ Slot slot_of(const asrlayer_cache8& c, int64_t b, int64_t pos) {
  if (b < 0 || b >= c.batch || pos < 0 || pos >= c.max_len) return {-1, 0};
  if (c.block_table == nullptr) return {b, pos};
  const int32_t page = c.block_table[b * c.bt_stride + pos / c.page_size];
  if (page < 0 || page >= c.num_pages) return {-1, 0};
  return {page, pos % c.page_size};
}

template <typename T, int HD>
__global__ __launch_bounds__(kThreads) void write8_kernel(const asrlayer_write8_params p) {
  constexpr int EPL = Elem<T>::kPerVec, LPK = HD / EPL, NG = kThreads / LPK;
  const asrlayer_cache8& c = p.cache;
  const int sub = threadIdx.x % LPK, group = threadIdx.x / LPK;
  const int64_t tok = blockIdx.x;
  const int rows = p.heads_q + 2 * c.heads_kv;  // queries, keys, values
  const bool norm = p.q_norm != nullptr, rot = p.cos != nullptr;

  const Slot slot = slot_of(c, p.rows != nullptr ? p.rows[tok] : tok, p.positions[tok]);
  uint4 cs{}, sn{};
  if (rot) {
    cs = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.cos) + tok * p.rope_stride + sub * EPL);
    sn = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.sin) + tok * p.rope_stride + sub * EPL);
  }
  // Rows past the last repeat it (and are not stored): every lane takes part in the
  // row sums.
  for (int r0 = 0; r0 < rows; r0 += NG) {
    const int r = min(r0 + group, rows - 1);
    const bool is_q = r < p.heads_q, is_v = r >= p.heads_q + c.heads_kv;
    const int h = is_q ? r : r - p.heads_q - (is_v ? c.heads_kv : 0);
    const T* src = static_cast<const T*>(is_q ? p.q : is_v ? p.v : p.k);
    src += tok * (is_q ? p.q_token_stride : is_v ? p.v_token_stride : p.k_token_stride) +
           h * (is_q ? p.q_head_stride : is_v ? p.v_head_stride : p.k_head_stride) + sub * EPL;
    uint4 raw = *reinterpret_cast<const uint4*>(src);
    if (norm || rot) {
      uint4 w{};
      if (norm) w = *reinterpret_cast<const uint4*>(static_cast<const T*>(is_q ? p.q_norm : p.k_norm) + sub * EPL);
      raw = prologue_row<T, HD, LPK>(raw, norm, norm && !is_v, true, w, rot, rot && !is_v, cs, sn,
                                     is_q ? p.q_eps : p.k_eps, sub);
    }
    float x[EPL];
    unpack<T>(raw, x);
    uint32_t largest = 0;
#pragma unroll
    for (int e = 0; e < EPL; ++e) largest = max(largest, magnitude(x[e]));
    const Scale8 s = scale8(group_umax<LPK>(largest));
    if (r0 + group >= rows) continue;
    T* whole = static_cast<T*>(is_q ? p.q_out : is_v ? nullptr : p.k_out);
    if (whole != nullptr)
      *reinterpret_cast<uint4*>(whole + (tok * (is_q ? p.heads_q : c.heads_kv) + h) * HD + sub * EPL) = raw;
    if (is_q || slot.entry < 0) continue;
    int8_t* at = static_cast<int8_t*>(is_v ? c.v : c.k);
    at += slot.entry * (is_v ? c.v_batch_stride : c.k_batch_stride) + slot.pos * (is_v ? c.v_token_stride : c.k_token_stride) +
          h * (is_v ? c.v_head_stride : c.k_head_stride) + sub * EPL;
    if constexpr (EPL == 8)
      *reinterpret_cast<uint2*>(at) = make_uint2(round8x4(x, s), round8x4(x + 4, s));
    else
      *reinterpret_cast<uint32_t*>(at) = round8x4(x, s);
    if (sub == 0) {
      float* scale = static_cast<float*>(is_v ? c.v_scales : c.k_scales);
      scale[slot.entry * (is_v ? c.vs_batch_stride : c.ks_batch_stride) + h * (is_v ? c.vs_head_stride : c.ks_head_stride) +
            slot.pos] = s.scale;
    }
  }
}

// A lane takes 16 bytes of one row; a workgroup kThreads of them in the outputs'
// order.
template <typename T>
__global__ __launch_bounds__(kThreads) void read8_kernel(const asrlayer_read8_params p, int pieces, int head_shift) {
  const asrlayer_cache8& c = p.cache;
  const int64_t b = blockIdx.y;
  const int64_t item = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  const int per = 1 << head_shift;  // pieces of a row
  const int64_t pos = item / pieces;
  if (pos >= c.max_len) return;
  const int within = (int)(item - pos * pieces), h = within >> head_shift, piece = within & (per - 1);
  int64_t n = c.max_len;
  if (p.lengths != nullptr)
    n = p.lengths64 ? static_cast<const int64_t*>(p.lengths)[b] : static_cast<const int32_t*>(p.lengths)[b];
  Slot slot{-1, 0};
  if (pos < n) slot = slot_of(c, b, pos);
  const bool values = blockIdx.z != 0;
  float x[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) x[e] = 0.f;
  if (slot.entry >= 0) {
    const int8_t* at = static_cast<const int8_t*>(values ? c.v : c.k) +
                       slot.entry * (values ? c.v_batch_stride : c.k_batch_stride) +
                       slot.pos * (values ? c.v_token_stride : c.k_token_stride) +
                       h * (values ? c.v_head_stride : c.k_head_stride) + piece * 16;
    const uint4 raw = *reinterpret_cast<const uint4*>(at);
    const float scale = static_cast<const float*>(values ? c.v_scales : c.k_scales)
        [slot.entry * (values ? c.vs_batch_stride : c.ks_batch_stride) +
         h * (values ? c.vs_head_stride : c.ks_head_stride) + slot.pos];
    const uint32_t words[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] = (float)(int8_t)(words[e / 4] >> (8 * (e % 4))) * scale;
  }
  T* out = static_cast<T*>(values ? p.v_out : p.k_out) + (b * c.max_len * pieces + item) * 16;
  constexpr int EPL = Elem<T>::kPerVec;
#pragma unroll
  for (int v = 0; v < 16 / EPL; ++v) *reinterpret_cast<uint4*>(out + v * EPL) = pack<T>(x + v * EPL);
}

template <typename T>
hipError_t launch_write(const asrlayer_write8_params& p, hipStream_t stream) {
  const dim3 grid((unsigned)p.tokens), block(kThreads);
  switch (p.cache.head_dim) {
    case 64: hipLaunchKernelGGL((write8_kernel<T, 64>), grid, block, 0, stream, p); break;
    case 128: hipLaunchKernelGGL((write8_kernel<T, 128>), grid, block, 0, stream, p); break;
    default: hipLaunchKernelGGL((write8_kernel<T, 256>), grid, block, 0, stream, p); break;
  }
  return hipGetLastError();
}

}  // namespace

hipError_t launch_write8(const asrlayer_write8_params& p, hipStream_t stream) {
  return p.dtype == ASRATTN_BF16 ? launch_write<bf16_raw>(p, stream) : launch_write<float>(p, stream);
}

hipError_t launch_read8(const asrlayer_read8_params& p, hipStream_t stream) {
  const int head_shift = p.cache.head_dim == 64 ? 2 : p.cache.head_dim == 128 ? 3 : 4;
  const int pieces = p.cache.heads_kv << head_shift;
  const int64_t blocks = ((int64_t)p.cache.max_len * pieces + kThreads - 1) / kThreads;
  const dim3 grid((unsigned)blocks, (unsigned)p.cache.batch, 2), block(kThreads);
  if (p.dtype == ASRATTN_BF16)
    hipLaunchKernelGGL((read8_kernel<bf16_raw>), grid, block, 0, stream, p, pieces, head_shift);
  else
    hipLaunchKernelGGL((read8_kernel<float>), grid, block, 0, stream, p, pieces, head_shift);
  return hipGetLastError();
}

}  // namespace asrattn
