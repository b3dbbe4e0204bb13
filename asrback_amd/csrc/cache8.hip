// The 8-bit cache's writes and reading back (asrlayer_write8, asrlayer_read8).
//
// Both are bound by memory: a write reads each new row (one head of one token)
// once and writes half (float32: a quarter) of it and its scale; reading back is the
// reverse.  A row is held by LPK lanes of 16 bytes, and its largest magnitude is a
// maximum over its lanes.  The norms and the rotation of a decoder's queries and
// keys happen on the same registers first, as in prompt_rows.hip.
//
// Many rows come by tokens: a workgroup takes neighbouring tokens' queries, keys or
// values of four heads, so that its scales lie next to each other in memory, a token's
// slot and tables are looked up for four rows, and what tells queries, keys and values
// apart is uniform, which leaves per row little but the loads, the rounding and the
// stores.  Two prompts of 20 000 tokens, 8 heads of 128, bf16: 49.5 us (5.0 TB/s; a workgroup
// per token, its rows one by one: 79), with 16 heads of queries and the norms 126 (157).
// 8 of 430 into pages: 9.2 us, with queries 15.1, of which the chain of position, page
// and stores is a good part.  A step's few rows spread over the card, 3.3 us.  Reading back
// two of 20 000 of 32768: 69 us (5.1 TB/s); 8 of 430 of 1024: 9.8 us.
#include "kernels.hpp"
#include "layers.hpp"
#include "quantize8.hpp"
#include "row_ops.hpp"

namespace asrattn {
namespace {

constexpr int kThreads = 256;

// The pool entry and the position in it of position pos of sequence b; entry < 0:
// none.
struct Slot {
  int64_t entry;
  uint32_t pos;
};
__device__ __forceinline__ Slot slot_of(const asrlayer_cache8& c, int page_shift, int64_t b, int64_t pos) {
  if (b < 0 || b >= c.batch || pos < 0 || pos >= c.max_len) return {-1, 0};
  const uint32_t at = (uint32_t)pos;  // below 2^30
  if (c.block_table == nullptr) return {b, at};
  const int32_t page = c.block_table[b * c.bt_stride + (at >> page_shift)];
  if (page < 0 || page >= c.num_pages) return {-1, 0};
  return {page, at & ((1u << page_shift) - 1)};
}

// `rows` of a token: queries, keys, values.  U == 0: a lane group takes one of all
// tokens' rows; otherwise U heads of one of the three of its token.
template <typename T, int HD, int U>
__global__ __launch_bounds__(kThreads) void write8_kernel(const asrlayer_write8_params p, int page_shift, uint32_t rows) {
  constexpr int EPL = Elem<T>::kPerVec, LPK = HD / EPL, NG = kThreads / LPK, N = U > 0 ? U : 1;
  const asrlayer_cache8& c = p.cache;
  const int sub = threadIdx.x % LPK;
  const uint32_t at = blockIdx.x * NG + threadIdx.x / LPK;
  uint32_t tok = at;
  bool is_q, is_v;
  int h0, heads = 1;  // of this lane group
  if constexpr (U > 0) {
    int block = blockIdx.y;
    const int q_blocks = (p.heads_q + U - 1) / U, kv_blocks = (c.heads_kv + U - 1) / U;
    is_q = block < q_blocks;
    is_v = block >= q_blocks + kv_blocks;
    h0 = (block - (is_q ? 0 : is_v ? q_blocks + kv_blocks : q_blocks)) * U;
    heads = min(U, (is_q ? p.heads_q : c.heads_kv) - h0);
  } else {
    tok = at / rows;
    const int r = (int)(at - tok * rows);
    is_q = r < p.heads_q;
    is_v = r >= p.heads_q + c.heads_kv;
    h0 = is_q ? r : r - p.heads_q - (is_v ? c.heads_kv : 0);
  }
  // Tokens past the last repeat it (and are not stored): every lane takes part in the
  // row sums.
  const bool there = tok < p.tokens;
  tok = there ? tok : (uint32_t)p.tokens - 1;
  const bool norm = p.q_norm != nullptr && !is_v, rot = p.cos != nullptr && !is_v;

  uint4 raw[N], cs{}, sn{}, w{};
  const int64_t head_step = is_q ? p.q_head_stride : is_v ? p.v_head_stride : p.k_head_stride;
  const T* src = static_cast<const T*>(is_q ? p.q : is_v ? p.v : p.k) + h0 * head_step +
                 tok * (is_q ? p.q_token_stride : is_v ? p.v_token_stride : p.k_token_stride) + sub * EPL;
#pragma unroll
  for (int u = 0; u < N; ++u)
    if (u < heads) raw[u] = *reinterpret_cast<const uint4*>(src + u * head_step);
  if (rot) {
    cs = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.cos) + tok * p.rope_stride + sub * EPL);
    sn = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.sin) + tok * p.rope_stride + sub * EPL);
  }
  if (norm) w = *reinterpret_cast<const uint4*>(static_cast<const T*>(is_q ? p.q_norm : p.k_norm) + sub * EPL);
  const Slot slot = is_q ? Slot{-1, 0} : slot_of(c, page_shift, p.rows != nullptr ? p.rows[tok] : tok, p.positions[tok]);
  const bool held = there && slot.entry >= 0;
  const int64_t entry = held ? slot.entry : 0;
  const uint32_t pos = held ? slot.pos : 0;
  const int64_t to_step = is_v ? c.v_head_stride : c.k_head_stride, scale_step = is_v ? c.vs_head_stride : c.ks_head_stride;
  int8_t* const to = static_cast<int8_t*>(is_v ? c.v : c.k) + entry * (is_v ? c.v_batch_stride : c.k_batch_stride) +
                     pos * (is_v ? c.v_token_stride : c.k_token_stride) + h0 * to_step + sub * EPL;
  float* const scale = static_cast<float*>(is_v ? c.v_scales : c.k_scales) +
                       entry * (is_v ? c.vs_batch_stride : c.ks_batch_stride) + pos + h0 * scale_step;
  T* const whole = static_cast<T*>(is_q ? p.q_out : is_v ? nullptr : p.k_out);
  T* const out = whole + ((int64_t)tok * (is_q ? p.heads_q : c.heads_kv) + h0) * HD + sub * EPL;
#pragma unroll
  for (int u = 0; u < N; ++u) {
    if (u >= heads) break;
    // (of all lanes at once: U == 0 has keys beside values)
    const bool any_norm = U > 0 ? norm : p.q_norm != nullptr, any_rot = U > 0 ? rot : p.cos != nullptr;
    if (any_norm || any_rot)
      raw[u] = prologue_row<T, HD, LPK>(raw[u], any_norm, norm, true, w, any_rot, rot, cs, sn, is_q ? p.q_eps : p.k_eps, sub);
    if (whole != nullptr && there) *reinterpret_cast<uint4*>(out + u * HD) = raw[u];
    if (U > 0 && is_q) continue;
    float x[EPL];
    unpack<T>(raw[u], x);
    uint32_t largest = 0;
#pragma unroll
    for (int e = 0; e < EPL; ++e) largest = max(largest, magnitude(x[e]));
    const Scale8 s = scale8(group_umax<LPK>(largest));
    if (!held) continue;
    uint32_t bytes[EPL / 4];
    bytes_of<T>(x, s, bytes);
    if constexpr (EPL == 8)
      *reinterpret_cast<uint2*>(to + u * to_step) = make_uint2(bytes[0], bytes[EPL / 4 - 1]);
    else
      *reinterpret_cast<uint32_t*>(to + u * to_step) = bytes[0];
    if (sub == 0) scale[u * scale_step] = s.scale;
  }
}

// Pieces of 16 bytes in the outputs' order, a lane's kReads of them kThreads apart (8 rows
// of 1024, 430 held: 9.8 us with two, 10.7 with four; with one 9.4, but 42.6 for 40.5 where
// most are empty).
constexpr int kReads = 2;
template <typename T>
__global__ __launch_bounds__(kThreads) void read8_kernel(const asrlayer_read8_params p, int page_shift, uint32_t pieces,
                                                         int head_shift) {
  constexpr int EPL = Elem<T>::kPerVec, U = kReads;
  const asrlayer_cache8& c = p.cache;
  const int64_t b = blockIdx.y;
  const uint32_t first = blockIdx.x * (kThreads * U) + threadIdx.x, items = c.max_len * pieces;  // below 2^31
  int64_t n = c.max_len;
  if (p.lengths != nullptr)
    n = p.lengths64 ? load_uniform(static_cast<const int64_t*>(p.lengths) + b)
                    : load_uniform(static_cast<const int32_t*>(p.lengths) + b);
  const bool values = blockIdx.z != 0;
  const int8_t* data = static_cast<const int8_t*>(values ? c.v : c.k);
  const float* scales = static_cast<const float*>(values ? c.v_scales : c.k_scales);
  uint32_t raw[U][EPL / 4];
  float scale[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t item = min(first + u * kThreads, items - 1), pos = item / pieces, within = item - pos * pieces;
    const int h = (int)(within >> head_shift), piece = (int)(within & ((1u << head_shift) - 1));
    Slot slot{-1, 0};
    if (pos < n) slot = slot_of(c, page_shift, b, pos);
    scale[u] = 0.f;
#pragma unroll
    for (int w = 0; w < EPL / 4; ++w) raw[u][w] = 0;
    if (slot.entry >= 0) {
      const int8_t* at = data + slot.entry * (values ? c.v_batch_stride : c.k_batch_stride) +
                         slot.pos * (values ? c.v_token_stride : c.k_token_stride) +
                         h * (values ? c.v_head_stride : c.k_head_stride) + piece * EPL;
      scale[u] = scales[slot.entry * (values ? c.vs_batch_stride : c.ks_batch_stride) +
                        h * (values ? c.vs_head_stride : c.ks_head_stride) + slot.pos];
      if constexpr (EPL == 8) {
        const uint2 two = *reinterpret_cast<const uint2*>(at);
        raw[u][0] = two.x;
        raw[u][EPL / 4 - 1] = two.y;
      } else {
        raw[u][0] = *reinterpret_cast<const uint32_t*>(at);
      }
    }
  }
  T* out = static_cast<T*>(values ? p.v_out : p.k_out) + b * items * EPL;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t item = first + u * kThreads;
    if (item >= items) continue;
    float x[EPL];
#pragma unroll
    for (int e = 0; e < EPL; ++e) x[e] = (float)(int8_t)(raw[u][e / 4] >> (8 * (e % 4))) * scale[u];
    *reinterpret_cast<uint4*>(out + (int64_t)item * EPL) = pack<T>(x);
  }
}

template <typename T, int HD>
hipError_t launch_write_head(const asrlayer_write8_params& p, int page_shift, hipStream_t stream) {
  constexpr int NG = kThreads * Elem<T>::kPerVec / HD;
  const uint32_t rows = p.heads_q + 2 * p.cache.heads_kv, items = (uint32_t)p.tokens * rows;
  // By tokens once the rows are more than the card's 2048 workgroups hold at once (5 x
  // 1500 tokens, 6 heads of 64, float32: 11.3 us, row by row 13.0).
  constexpr int U = 4;
  const uint32_t blocks = (p.heads_q + U - 1) / U + 2 * ((p.cache.heads_kv + U - 1) / U);
  if (items > 2048 * NG)
    hipLaunchKernelGGL((write8_kernel<T, HD, U>), dim3(((uint32_t)p.tokens + NG - 1) / NG, blocks), dim3(kThreads), 0, stream,
                       p, page_shift, rows);
  else
    hipLaunchKernelGGL((write8_kernel<T, HD, 0>), dim3((items + NG - 1) / NG), dim3(kThreads), 0, stream, p, page_shift, rows);
  return hipGetLastError();
}

template <typename T>
hipError_t launch_write(const asrlayer_write8_params& p, int page_shift, hipStream_t stream) {
  switch (p.cache.head_dim) {
    case 64: return launch_write_head<T, 64>(p, page_shift, stream);
    case 128: return launch_write_head<T, 128>(p, page_shift, stream);
    default: return launch_write_head<T, 256>(p, page_shift, stream);
  }
}

template <typename T>
hipError_t launch_read(const asrlayer_read8_params& p, int page_shift, hipStream_t stream) {
  int head_shift = 0;
  while ((Elem<T>::kPerVec << head_shift) < p.cache.head_dim) ++head_shift;
  const uint32_t pieces = (uint32_t)p.cache.heads_kv << head_shift, per = kThreads * kReads;
  const dim3 grid((unsigned)(((uint64_t)p.cache.max_len * pieces + per - 1) / per), (unsigned)p.cache.batch, 2);
  hipLaunchKernelGGL((read8_kernel<T>), grid, dim3(kThreads), 0, stream, p, page_shift, pieces, head_shift);
  return hipGetLastError();
}

int page_shift_of(const asrlayer_cache8& c) {
  int shift = 0;
  while (c.block_table != nullptr && (1LL << shift) < c.page_size) ++shift;
  return shift;
}

}  // namespace

hipError_t launch_write8(const asrlayer_write8_params& p, hipStream_t stream) {
  const int shift = page_shift_of(p.cache);
  return p.dtype == ASRATTN_BF16 ? launch_write<bf16_raw>(p, shift, stream) : launch_write<float>(p, shift, stream);
}

hipError_t launch_read8(const asrlayer_read8_params& p, hipStream_t stream) {
  const int shift = page_shift_of(p.cache);
  return p.dtype == ASRATTN_BF16 ? launch_read<bf16_raw>(p, shift, stream) : launch_read<float>(p, shift, stream);
}

}  // namespace asrattn
