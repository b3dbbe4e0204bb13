// A decoder step's attention over a cache of 8-bit keys and values
// (asrlayer_decode8), with the step's write and what comes before it (asrlayer_append8).
//
// One query per sequence: g query heads share a kv head's n keys, each of which is
// read once, 2 (head_dim + 4) bytes with its value and scales, for 4 g head_dim
// operations.  Bound by reading the cache, once the 8-bit values become operands
// cheaply enough:
//
//   * A whole number up to 255 is exact in bf16, so scores and outputs are bf16
//     matrix products of the stored numbers, and the scales enter beside them: a key's
//     multiplies its scores, a value's its weights.  bf16 queries enter as they are and
//     float32 ones as three bf16 that sum to them; every product is exact.  The weights
//     times the values' scales enter as two bf16 (three in float32): 2^-17 (2^-24) of
//     each is lost.
//   * Converting two numbers takes three vector instructions, most of the arithmetic of a
//     few heads.  With bf16 queries 0x80 is added to the bytes instead, one instruction for
//     four, and a permutation puts u = x + 128 into the low byte of each half: as bf16
//     that is u 2^-133, exactly, subnormal up to 127 (the matrix units take those as they
//     are).  Powers of two in the queries and in the values' scales make up for it, and
//     128 times the queries' (the weights') sum is taken off at the end, itself a product
//     with the bytes of zeros.  In float32 terms that are up to 255 / 127 times larger than
//     the answer's cancel, so float32 queries are converted for.
//   * Scores come out transposed, S^T = K Q^T: a lane holds four keys' scores of one
//     head for each 16 keys, so a head's softmax state is a scalar per lane and the
//     weights are already the operand of O^T = V^T P^T.
//   * A wave takes tiles of 32 keys.  A lane of V^T's operand needs eight keys of one
//     dimension: it loads the same piece of eight values' rows, and the conversion
//     picks its byte, so nothing changes lanes.  A lane of K's operand holds 16
//     consecutive dimensions of one key, two products' worth; the keys are loaded whole,
//     neighbouring lanes in one, and change lanes through the wave's own LDS.
//   * The next tile loads while this one is computed; the 64 scales of a tile are one
//     load, spread over the lanes through LDS as well.
//
// Waves merge in LDS at the end; splits of the keys leave partials in the workspace,
// and the split that arrives last folds them (decode_kernels.hpp describes the arrival
// words).  Maxima, sums and outputs are float32 until the one rounding at the end.
//
// Measured with 16 heads over 8 of 128, bf16, every call on another cache: 64 sequences
// of 400 to 560 keys, pages of 64, 17.2 us (65 MB at 3.8 TB/s; where it took 18.0, with
// conversions, an unshuffled load of the keys and a merge of one head at a time 20.5); two
// of about 52 000, 45.9 us (223 MB at 4.9 TB/s; 47.8 and 64.9); one of 480, 7.9 us, a chain
// of round trips: length, keys, LDS, partials, arrival, fold.  Heads of 64 have half as many
// bytes a tile for the same exchange through LDS: 16 sequences of 1500 keys, 12 heads, take
// 17.2 us (39 MB at 2.3 TB/s), 16.1 with keys loaded straight into the operand and bytes
// converted.
#include <cmath>

#include "common.hpp"
#include "kernels.hpp"
#include "quantize8.hpp"
#include "row_ops.hpp"

namespace asrattn {
namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2_t __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4_t __attribute__((ext_vector_type(4)));

constexpr int kKeys = 32;  // of a tile, in two halves
// Cache policy of data read once (common.hpp, buffer_load16_stream).
constexpr int kNontemporal = 2;

struct Decode8Args {
  asrlayer_decode8_params p;
  asrlayer_append8_params n;  // of the variant that appends (its step is p)
  int page_shift, head_tiles;
  int share;       // workgroups of a block of heads, that share all sequences' keys (0: one each)
  int splits;      // of every sequence (0: by their lengths)
  int tile_heads;  // query heads of a block, at most 16
  float c;         // scale * log2(e): c_part 2^c_power
  float c_part;
  int c_power;
  float* ws_o;     // [block][workgroup][tile_heads][head_dim]
  float* ws_ml;    // [block][workgroup][tile_heads][2]
  unsigned long long* ws_arrive;  // [block][sequence]
  unsigned long long tag;
};

template <typename T, int HD>
struct Decode8Shape {
  static constexpr int kQP = sizeof(T) == 2 ? 1 : 3;  // bf16 parts of a query
  static constexpr int kWP = sizeof(T) == 2 ? 2 : 3;  // of a weight
  static constexpr int kKP = HD / 64;                 // a lane's 16-byte pieces of a key
  static constexpr int kVB = HD / 16;                 // bytes of a lane's piece of a value: 16-row tiles of O^T
  static constexpr int kVD = kVB / 4;                 // dwords of it
  static constexpr bool kBiased = sizeof(T) == 2;     // products of biased bytes, where the scales allow it
  static constexpr float kUnit = kBiased ? 0x1p13f : 1.f;  // of the sums of weights and values
  static constexpr int kMerged = 8;                   // heads merged at a time
  static constexpr int kLPR = HD / 16;                // 16-byte pieces of a key
  static constexpr int kPerSimd = HD == 64 ? 4 : 2;   // waves that the registers leave room for on a SIMD
};

// Where piece c of key r of a tile lies in LDS, so that the 16 keys a product's operand
// takes a piece of lie in 16 different groups of banks.
template <int LPR>
__device__ __forceinline__ int lds_piece(int r, int c) {
  return r * LPR + (LPR == 4 ? c ^ ((r >> 2) & 3) : LPR == 8 ? c ^ ((r >> 1) & 7) : c ^ (r & 15));
}

__device__ __forceinline__ f32x4_t mfma_bf16(const uint4& a, const uint4& b, const f32x4_t& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0,
                                                 0, 0);
}

// Byte e of a dword as a float.
__device__ __forceinline__ float byte_of(uint32_t x, int e) { return (float)(int8_t)(x >> (8 * e)); }

// Two floats of at most 8 significant bits as bf16: their high halves.
__device__ __forceinline__ uint32_t high_halves(float a, float b) {
  return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
}

// Four 8-bit numbers as bf16.
__device__ __forceinline__ uint2 widen(uint32_t x) {
  return make_uint2(high_halves(byte_of(x, 0), byte_of(x, 1)), high_halves(byte_of(x, 2), byte_of(x, 3)));
}

// The same without a conversion, for what has 0x80 added to every byte: a bf16 of the
// bits u in 0 .. 255 is u 2^-133, of which numbers below 128 are subnormal and the others
// follow on.  byte_pair takes byte e of two dwords.
constexpr uint32_t kBias = 0x80808080u;
__device__ __forceinline__ uint2 widen_biased(uint32_t x) {
  return make_uint2(__builtin_amdgcn_perm(x, x, 0x0c010c00u), __builtin_amdgcn_perm(x, x, 0x0c030c02u));
}
__device__ __forceinline__ uint32_t byte_pair(uint32_t a, uint32_t b, int e) {
  return __builtin_amdgcn_perm(b, a, 0x0c040c00u + (uint32_t)e * 0x00010001u);
}

// The leading bf16 of two floats, and what is left of them.
__device__ __forceinline__ uint32_t take_part(float& a, float& b) {
  const uint32_t r = high_halves(a, b);
  a -= __uint_as_float(__float_as_uint(a) & 0xffff0000u);
  b -= __uint_as_float(__float_as_uint(b) & 0xffff0000u);
  return r;
}

__device__ __forceinline__ float row_max(float x) {
  float a, b;
  lane_pair<16>(x, a, b);
  x = fmaxf(a, b);
  lane_pair<32>(x, a, b);
  return fmaxf(a, b);
}
__device__ __forceinline__ float row_sum(float x) {
  float a, b;
  lane_pair<16>(x, a, b);
  x = a + b;
  lane_pair<32>(x, a, b);
  return a + b;
}

__device__ __forceinline__ uint64_t uniform64(uint64_t x) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32 |
         (uint32_t)__builtin_amdgcn_readfirstlane((int)x);
}

// Dimensions d .. d + 3 of a query head: the weighted sum of values over the sum of
// the weights.
template <typename T>
__device__ __forceinline__ void store_head(const Decode8Args& a, int b, int head, int d, const float* x, float sum) {
  T* op = static_cast<T*>(a.p.out) + (int64_t)b * a.p.o_batch_stride + (int64_t)head * a.p.o_head_stride + d;
#pragma unroll
  for (int e = 0; e < 4; ++e) Elem<T>::store1(op + e, sum == 0.f ? 0.f : x[e] * Decode8Shape<T, 64>::kUnit / sum);
}

// Sum (in lane 0) and running sums over the first lanes of a wave.
__device__ __forceinline__ int lanes_sum(int x, int lanes) {
  for (int d = 1; d < lanes; d *= 2) x += __shfl_xor(x, d, 64);
  return __builtin_amdgcn_readfirstlane(x);
}
__device__ __forceinline__ int lanes_prefix(int x, int lanes) {
  for (int d = 1; d < lanes; d *= 2) {
    const int y = __shfl_up(x, d, 64);
    x += (int)(threadIdx.x & 63) >= d ? y : 0;
  }
  return x;
}

// APPEND: the queries get their norm and rotation here, and the sequence's new key and
// value are rounded, written, and attended to beside the tiles: the softmax of the last
// split's last wave, which has the fewest, begins with them.  One of 480 keys (16 heads
// over 8 of 128) 9.3 us, in two launches 11.2; 64 of them 18.4 and 19.5; one of 16 000
// 19.2 and 21.1.
template <typename T, int HD, int W, bool PAGED, bool APPEND>
__global__ __launch_bounds__(64 * W, (Decode8Shape<T, HD>::kPerSimd)) void decode8_kernel(const Decode8Args a) {
  using S = Decode8Shape<T, HD>;
  constexpr int kQP = S::kQP, kWP = S::kWP, kKP = S::kKP, kVB = S::kVB, kVD = S::kVD;
  const asrlayer_decode8_params& p = a.p;
  const asrlayer_cache8& c = p.cache;
  const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int hkv = blockIdx.y / a.head_tiles, ht = blockIdx.y % a.head_tiles;
  const int group = p.heads_q / c.heads_kv;
  const int head0 = hkv * group + ht * 16, held = min(16, group - ht * 16);

  // The workgroup's sequence, its keys, and its split of them.
  auto keys_of = [&](int64_t have) { return have < 0 ? 0 : have < c.max_len ? (int)have : c.max_len; };
  auto first_of = [&](int n) { return p.window > 0 && n > p.window ? n - p.window : 0; };
  // Keys of sequence j, the new one among them, where `load` reads a number.
  auto have_of = [&](int j, auto load) {
    if constexpr (APPEND) {
      const int64_t pos = load(a.n.positions + j);
      return pos < c.max_len ? keys_of(pos + 1) : c.max_len;
    }
    if (p.lengths == nullptr) return c.max_len;
    return keys_of(p.lengths64 ? load(static_cast<const int64_t*>(p.lengths) + j)
                               : (int64_t)load(static_cast<const int32_t*>(p.lengths) + j));
  };
  auto uniformly = [](auto* p) { return load_uniform(p); };
  int b = blockIdx.z, n, split = 0, splits = 1;
  if (a.share == 0) {
    n = have_of(b, uniformly);
  } else if (a.splits > 0) {
    b = blockIdx.x / a.splits;
    split = blockIdx.x - b * a.splits;
    splits = a.splits;
    n = have_of(b, uniformly);
  } else {
    // Sequences get workgroups by their tiles: every `per` of them one, where per is whole
    // turns of the waves, and about the fewest for which the workgroups do not run out (they
    // are at least twice as many as the sequences, and cannot with twice the fewest).  A
    // lane counts two sequences' (the splits are at most 128 sequences').
    int held_keys[2], count[2], tiles = 0;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int j = 2 * lane + s;
      const int have = j < c.batch ? have_of(j, [](auto* p) { return *p; }) : 0;
      held_keys[s] = have;
      count[s] = have / kKeys + (have % kKeys != 0) - first_of(have) / kKeys;
      tiles += count[s];
    }
    const int lanes = (c.batch + 1) / 2;
    const uint32_t total = lanes_sum(tiles, lanes);
    uint32_t per = max((total + a.share - 1) / a.share, 1u);
    const uint32_t more = max(per / (16 * W), 1u) * W;
    per = (per + W - 1) / W * W;
    for (;; per += more) {
      int taken = 0;
#pragma unroll
      for (int s = 0; s < 2; ++s)
        taken += 2 * lane + s < c.batch ? max(1, (int)(((uint32_t)count[s] + per - 1) / per)) : 0;
      if (lanes_sum(taken, lanes) <= a.share) break;
    }
#pragma unroll
    for (int s = 0; s < 2; ++s)
      count[s] = 2 * lane + s < c.batch ? max(1, (int)(((uint32_t)count[s] + per - 1) / per)) : 0;
    const int x = blockIdx.x, from = lanes_prefix(count[0] + count[1], lanes) - count[0] - count[1];
    const bool second = x >= from + count[0];
    const unsigned long long hit = __ballot(x >= from && x < from + count[0] + count[1]);
    if (hit == 0) return;  // one of those to spare
    const int at = __ffsll(hit) - 1;
    b = 2 * at + (__builtin_amdgcn_readlane(second, at) ? 1 : 0);
    split = x - __builtin_amdgcn_readlane(second ? from + count[0] : from, at);
    splits = __builtin_amdgcn_readlane(second ? count[1] : count[0], at);
    n = __builtin_amdgcn_readlane(second ? held_keys[1] : held_keys[0], at);
  }
  n = __builtin_amdgcn_readfirstlane(n);
  const bool split_keys = splits > 1;
  unsigned long long* const arrive = a.ws_arrive + (int64_t)blockIdx.y * c.batch + b;
  unsigned long long arrive_old = 0;
  if (split_keys && threadIdx.x == 0)
    arrive_old = __hip_atomic_load(arrive, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);

  // The tiles' keys; after them, the waves' sums of kMerged heads.
  constexpr int kKeyPieces = kKeys * S::kLPR, kMerged = S::kMerged, kSumPieces = W * kMerged * (HD + 4) / 4;
  __shared__ uint4 sm_pool[W * kKeyPieces > kSumPieces ? W * kKeyPieces : kSumPieces];
  uint4* const sm_k = sm_pool + wave * kKeyPieces;
  float(*const sm_o)[kMerged][HD + 4] = reinterpret_cast<float(*)[kMerged][HD + 4]>(sm_pool);
  __shared__ uint4 sm_q[2 * kKP * kQP * 64];
  __shared__ float sm_m[W][16], sm_l[W][16];
  __shared__ __attribute__((aligned(16))) float sm_scale[W][64];
  __shared__ uint32_t sm_largest[W];
  __shared__ int sm_last;

  constexpr int EPL = Elem<T>::kPerVec, LPK = HD / EPL, kGroups = 64 * W / LPK;
  constexpr int kRowTurns = APPEND ? (16 + 2 + kGroups - 1) / kGroups : 1;
  const int sub = threadIdx.x % LPK;
  __shared__ uint4 sm_new[APPEND ? 2 * HD / 16 : 1];  // the new key's and value's bytes
  __shared__ float sm_new_scale[2];
  uint4 row[kRowTurns], weights[kRowTurns], cs{}, sn{};
  int new_page = 0, new_pos = -1;  // where the new key goes (-1: nowhere)
  if constexpr (APPEND) {
    // Rows of LPK lanes: the queries', and the new key and value of the last split.
    cs = reinterpret_cast<const uint4*>(static_cast<const T*>(a.n.cos) + b * a.n.rope_stride)[sub];
    sn = reinterpret_cast<const uint4*>(static_cast<const T*>(a.n.sin) + b * a.n.rope_stride)[sub];
#pragma unroll
    for (int turn = 0; turn < kRowTurns; ++turn) {
      const int r = min(turn * kGroups + (int)threadIdx.x / LPK, split == splits - 1 ? held + 1 : held - 1);
      const T* from = r < held ? static_cast<const T*>(p.q) + (int64_t)b * p.q_batch_stride + (int64_t)(head0 + r) * p.q_head_stride
                      : r == held ? static_cast<const T*>(a.n.k) + (int64_t)b * a.n.k_batch_stride + hkv * a.n.k_head_stride
                                  : static_cast<const T*>(a.n.v) + (int64_t)b * a.n.v_batch_stride + hkv * a.n.v_head_stride;
      row[turn] = reinterpret_cast<const uint4*>(from)[sub];
      weights[turn] = static_cast<const uint4*>(r < held ? a.n.q_norm : a.n.k_norm)[sub];
    }
    const int64_t pos = load_uniform(a.n.positions + b);
    if (pos >= 0 && pos < c.max_len) {
      new_pos = (int)pos;
      if constexpr (PAGED) {
        new_page = load_uniform(c.block_table + (int64_t)b * c.bt_stride + (new_pos >> a.page_shift));
        if (new_page < 0 || new_page >= c.num_pages) new_pos = -1;
      }
    }
  }

  // The queries' pieces, 8 dimensions each: lane's piece u of its head (heads past the
  // last repeat it) goes to (u, part, lane) of LDS.
  constexpr int kQTurns = (2 * kKP + W - 1) / W, kQVecs = sizeof(T) / 2;
  uint4 raw_q[kQTurns][kQVecs];
  auto read_queries = [&](const T* at, int64_t head_step) {
#pragma unroll
    for (int turn = 0; turn < kQTurns; ++turn) {
      const int u = min(turn * W + wave, 2 * kKP - 1);
      const T* from = at + min(i, held - 1) * head_step + 64 * (u / 2) + 16 * g + 8 * (u % 2);
#pragma unroll
      for (int x = 0; x < kQVecs; ++x) raw_q[turn][x] = reinterpret_cast<const uint4*>(from)[x];
    }
  };
  if constexpr (!APPEND)
    read_queries(static_cast<const T*>(p.q) + (int64_t)b * p.q_batch_stride + (int64_t)head0 * p.q_head_stride,
                 p.q_head_stride);

  // The positions: from a multiple of a tile on, up to the new key.
  const int first = first_of(n);
  if (APPEND && new_pos >= 0) n = new_pos;
  const int tile0 = first / kKeys, tiles = n / kKeys + (n % kKeys != 0) - tile0;
  const int per = (tiles + splits - 1) / splits;
  const int t0 = tile0 + min(tiles, split * per), t1 = min(tile0 + tiles, t0 + per);

  // Where a half tile's 16 positions lie: the pool entry (-1: nowhere), the first of
  // them in it, and how many are there.
  struct Half {
    int64_t entry;
    int64_t at;
    int keys;
  };
  const int32_t* const table = PAGED ? c.block_table + (int64_t)b * c.bt_stride : nullptr;
  auto page_of = [&](int t, int h) -> int {
    if constexpr (!PAGED) return 0;
    const int pos = t * kKeys + 16 * h;
    const int page = load_uniform(table + (t < t1 && pos < n ? pos >> a.page_shift : 0));
    return page < c.num_pages ? page : -1;
  };
  auto half_of = [&](int t, int h, int page) -> Half {
    const int pos = t * kKeys + 16 * h;
    Half x;
    x.keys = t < t1 ? min(max(n - pos, 0), 16) : 0;
    x.entry = b;
    x.at = pos;
    if constexpr (PAGED) {
      x.keys = page >= 0 ? x.keys : 0;
      x.entry = max(page, 0);
      x.at = pos & ((1 << a.page_shift) - 1);
    }
    return x;
  };
  auto rsrc_of = [&](const Half& x, bool values) {
    const int64_t step = values ? c.v_token_stride : c.k_token_stride;
    const uint64_t at = (uint64_t)(values ? c.v : c.k) + x.entry * (values ? c.v_batch_stride : c.k_batch_stride) +
                        hkv * (values ? c.v_head_stride : c.k_head_stride) + x.at * step;
    const uint32_t bytes = x.keys > 0 ? (uint32_t)(x.keys - 1) * (uint32_t)step + HD : 0u;
    return buffer_rsrc(reinterpret_cast<const void*>(uniform64(at)), __builtin_amdgcn_readfirstlane(bytes));
  };

  uint4 k[2][kKP];
  uint32_t v[2][4][kVD];
  float scale;      // lanes 0 .. 31: the keys', 32 .. 63: the values'
  int keys[2];      // of the tile held
  // Positions behind a half tile's are past its resource, and read as zeros (or, closer
  // together than a head is wide, as some other of its bytes: their scores and weights
  // are set by their index, and a stored number is never infinite).
  const uint32_t kstep = (uint32_t)c.k_token_stride, vstep = (uint32_t)c.v_token_stride;
  const uint32_t koff = lane / S::kLPR * kstep + lane % S::kLPR * 16, voff = 4 * g * vstep + i * kVB;
  // (The halves' pages are scalars by themselves: an array of them that the lambdas pass on
  // would be put into LDS, at an address that depends on the launch's packet in host memory.)
  auto load_keys = [&](int t, int page0, int page1) {
    const Half x0 = half_of(t, 0, page0), x1 = half_of(t, 1, page1);
    keys[0] = x0.keys;
    keys[1] = x1.keys;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const __amdgpu_buffer_rsrc_t rsrc = rsrc_of(h == 0 ? x0 : x1, false);
#pragma unroll
      for (int u = 0; u < kKP; ++u) k[h][u] = buffer_load16_stream(rsrc, koff + u * (64 / S::kLPR) * kstep);
    }
    // The tile's scales.
    const bool second = (lane & 16) != 0, values = lane >= 32;
    const int64_t entry = second ? x1.entry : x0.entry, at = second ? x1.at : x0.at;
    const bool there = i < (second ? x1.keys : x0.keys);
    const float* ptr = static_cast<const float*>(values ? c.v_scales : c.k_scales);
    const int64_t off = entry * (values ? c.vs_batch_stride : c.ks_batch_stride) +
                        hkv * (values ? c.vs_head_stride : c.ks_head_stride) + at + i;
    scale = ptr[there ? off : 0];
  };
  auto load_values = [&](int t, int page0, int page1) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const __amdgpu_buffer_rsrc_t rsrc = rsrc_of(half_of(t, h, h == 0 ? page0 : page1), true);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const uint32_t off = voff + r * vstep;
        if constexpr (kVD == 4) {
          const u32x4_t w = __builtin_amdgcn_raw_buffer_load_b128(rsrc, off, 0, kNontemporal);
#pragma unroll
          for (int d = 0; d < 4; ++d) v[h][r][d % kVD] = w[d];
        } else if constexpr (kVD == 2) {
          const u32x2_t w = __builtin_amdgcn_raw_buffer_load_b64(rsrc, off, 0, kNontemporal);
          v[h][r][0] = w[0];
          v[h][r][kVD - 1] = w[1];
        } else {
          v[h][r][0] = __builtin_amdgcn_raw_buffer_load_b32(rsrc, off, 0, kNontemporal);
        }
      }
    }
  };

  f32x4_t o[kVB];
  float m = kNegInf, l = 0.f;  // l: the lane's own keys only
#pragma unroll
  for (int e = 0; e < kVB; ++e) o[e] = f32x4_t{0.f, 0.f, 0.f, 0.f};

  int t = t0 + wave;
  int next0 = 0, next1 = 0;  // the next tile's pages
  if (t < t1) {
    const int page0 = page_of(t, 0), page1 = page_of(t, 1);
    next0 = page_of(t + W, 0);
    next1 = page_of(t + W, 1);
    load_keys(t, page0, page1);
    load_values(t, page0, page1);
  }
  // (LDS-only barriers: the keys and values stay in flight.)
  auto lds_barrier = [] {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
  };
  if constexpr (APPEND) {
    uint4* const rows = sm_pool;
    uint32_t largest_q = 0;
#pragma unroll
    for (int turn = 0; turn < kRowTurns; ++turn) {
      const int r = turn * kGroups + (int)threadIdx.x / LPK;
      const bool is_v = r == held + 1;
      const uint4 out = prologue_row<T, HD, LPK>(row[turn], true, !is_v, true, weights[turn], true, !is_v, cs, sn,
                                                 r < held ? a.n.q_eps : a.n.k_eps, sub);
      float x[EPL];
      unpack<T>(out, x);
      uint32_t largest = 0;
#pragma unroll
      for (int e = 0; e < EPL; ++e) largest = max(largest, magnitude(x[e]));
      const Scale8 s = scale8(group_umax<LPK>(largest));
      if (r < held) {
        rows[r * LPK + sub] = out;
        largest_q = max(largest_q, largest);
      } else if (split == splits - 1 && r <= held + 1) {
        uint32_t bytes[EPL / 4];
        bytes_of<T>(x, s, bytes);
        __builtin_memcpy(reinterpret_cast<char*>(sm_new) + (is_v ? HD : 0) + sub * EPL, bytes, EPL);
        if (sub == 0) sm_new_scale[is_v] = s.scale;
        if (ht == 0 && new_pos >= 0) {
          const int64_t entry = PAGED ? new_page : b;
          const int64_t at = PAGED ? new_pos & ((1 << a.page_shift) - 1) : new_pos;
          int8_t* to = static_cast<int8_t*>(is_v ? c.v : c.k) + entry * (is_v ? c.v_batch_stride : c.k_batch_stride) +
                       at * (is_v ? c.v_token_stride : c.k_token_stride) + hkv * (is_v ? c.v_head_stride : c.k_head_stride);
          if constexpr (EPL == 8)
            reinterpret_cast<uint2*>(to)[sub] = make_uint2(bytes[0], bytes[EPL / 4 - 1]);
          else
            reinterpret_cast<uint32_t*>(to)[sub] = bytes[0];
          if (sub == 0)
            static_cast<float*>(is_v ? c.v_scales : c.k_scales)
                [entry * (is_v ? c.vs_batch_stride : c.ks_batch_stride) + hkv * (is_v ? c.vs_head_stride : c.ks_head_stride) +
                 at] = s.scale;
        }
      }
    }
    if constexpr (S::kBiased) {
      largest_q = group_umax<64>(largest_q);
      if (lane == 0) sm_largest[wave] = largest_q;
    }
    lds_barrier();
    read_queries(reinterpret_cast<const T*>(rows), HD);
  }
  // bf16 queries are multiplied by 2^up below, and the keys' scales take that off again:
  // where bytes are biased they are multiplied by biased_unit, c 2^(133 - up), and where
  // they are converted key_unit puts c 2^-up to them, which alone may be less than float32
  // holds.
  float biased_unit = 0.f;
  int up = 0;
  auto key_unit = [&](float key_scale) {
    return S::kBiased ? __builtin_ldexpf(key_scale * a.c_part, a.c_power - up) : key_scale * a.c;
  };
  f32x4_t bias{0.f, 0.f, 0.f, 0.f};
  if constexpr (S::kBiased) {
    // The queries times a power of two that puts their largest near 2^100, so that
    // products with u 2^-133 are ordinary numbers.
    uint32_t largest = 0;
    if constexpr (!APPEND) {
#pragma unroll
      for (int turn = 0; turn < kQTurns; ++turn) {
        float x[8];
        unpack<bf16_raw>(raw_q[turn][0], x);
#pragma unroll
        for (int e = 0; e < 8; ++e) largest = max(largest, magnitude(x[e]));
      }
      largest = group_umax<64>(largest);
      if (lane == 0) sm_largest[wave] = largest;
      lds_barrier();
    }
#pragma unroll
    for (int u = 0; u < W; ++u) largest = max(largest, sm_largest[u]);
    up = 100 - ((int)(__builtin_amdgcn_readfirstlane(largest) >> 23) - 127);
    auto scalar = [](float x) { return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(x))); };
    biased_unit = scalar(__builtin_ldexpf(a.c, 133 - up));
#pragma unroll
    for (int turn = 0; turn < kQTurns; ++turn) {
      float x[8];
      unpack<bf16_raw>(raw_q[turn][0], x);
#pragma unroll
      for (int d = 0; d < 8; ++d) x[d] = __builtin_ldexpf(x[d], up);
      if (turn * W + wave < 2 * kKP) sm_q[(turn * W + wave) * 64 + lane] = pack<bf16_raw>(x);
    }
    lds_barrier();
    // The products with keys of zeros, each 128 too high.
    constexpr uint32_t kZeros = 0x00800080u;
#pragma unroll
    for (int u = 0; u < 2 * kKP; ++u) bias = mfma_bf16(make_uint4(kZeros, kZeros, kZeros, kZeros), sm_q[u * 64 + lane], bias);
    bias = -bias;
  } else {
#pragma unroll
    for (int turn = 0; turn < kQTurns; ++turn) {
      float x[8];
      unpack<float>(raw_q[turn][0], x);
      unpack<float>(raw_q[turn][kQVecs - 1], x + 4);
      if (turn * W + wave < 2 * kKP) {
#pragma unroll
        for (int part = 0; part < kQP; ++part)
          sm_q[((turn * W + wave) * kQP + part) * 64 + lane] =
              make_uint4(take_part(x[0], x[1]), take_part(x[2], x[3]), take_part(x[4], x[5]), take_part(x[6], x[7]));
      }
    }
    lds_barrier();
  }
  f32x4_t weighed{0.f, 0.f, 0.f, 0.f};  // products of the weights with biased zeros
  // Scores of 16 keys of the wave's LDS.
  auto scores_of = [&](int h, auto widened, f32x4_t sum) {
#pragma unroll
    for (int u = 0; u < kKP; ++u) {
      const uint4 raw = sm_k[lds_piece<S::kLPR>(16 * h + i, 4 * u + g)];
      const uint2 w0 = widened(raw.x), w1 = widened(raw.y), w2 = widened(raw.z), w3 = widened(raw.w);
      const uint4 lo = make_uint4(w0.x, w0.y, w1.x, w1.y), hi = make_uint4(w2.x, w2.y, w3.x, w3.y);
#pragma unroll
      for (int part = kQP - 1; part >= 0; --part) {
        sum = mfma_bf16(lo, sm_q[(2 * u * kQP + part) * 64 + lane], sum);
        sum = mfma_bf16(hi, sm_q[((2 * u + 1) * kQP + part) * 64 + lane], sum);
      }
    }
    return sum;
  };
  if (APPEND && new_pos >= 0 && split == splits - 1 && wave == W - 1) {
    // The new key as the first of 16 (the others are whatever lies there, and not looked at).
    if (lane < S::kLPR) sm_k[lds_piece<S::kLPR>(0, lane)] = sm_new[lane];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
    __builtin_amdgcn_wave_barrier();
    const f32x4_t s = scores_of(0, [](uint32_t x) { return widen(x); }, f32x4_t{0.f, 0.f, 0.f, 0.f});
    m = __shfl(s[0] * key_unit(sm_new_scale[0]), i, 64);
    l = g == 0 ? 1.f : 0.f;
    const float vs = sm_new_scale[1] * (1.f / S::kUnit);
    const uint32_t* value = reinterpret_cast<const uint32_t*>(sm_new + HD / 16) + g * kVB;
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int e = 0; e < kVB; ++e) o[e][r] = byte_of(value[(r * kVB + e) / 4], e % 4) * vs;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
    __builtin_amdgcn_wave_barrier();
  }
  {
    while (t < t1) {
      // The keys and the scales change lanes through the wave's own LDS.
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int u = 0; u < kKP; ++u)
          sm_k[lds_piece<S::kLPR>(16 * h + u * (64 / S::kLPR) + lane / S::kLPR, lane % S::kLPR)] = k[h][u];
      if (!(i < ((lane & 16) != 0 ? keys[1] : keys[0]) && t * kKeys + (lane & 31) >= first)) scale = 0.f;
      // Scales that the powers of two would put out of range (a value's above 128, a key's
      // above some 2^95 over the largest query): the tile's bytes are converted.
      const float biased = scale * (lane < 32 ? biased_unit : 0x1p120f);
      const bool convert = !S::kBiased || __any(!(fabsf(biased) <= 0x1p127f));
      sm_scale[wave][lane] = convert ? (lane < 32 ? key_unit(scale) : scale * (S::kBiased ? 0x1p-13f : 1.f)) : biased;
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
      __builtin_amdgcn_wave_barrier();
      f32x4_t s[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (S::kBiased && __builtin_expect(!convert, 1))
          s[h] = scores_of(h, [](uint32_t x) { return widen_biased(x ^ kBias); }, bias);
        else
          s[h] = scores_of(h, [](uint32_t x) { return widen(x); }, f32x4_t{0.f, 0.f, 0.f, 0.f});
      }
      const int pos = t * kKeys + 4 * g;
      float x[2][4], vs[2][4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float4 ks = *reinterpret_cast<const float4*>(&sm_scale[wave][16 * h + 4 * g]);
        const float4 w = *reinterpret_cast<const float4*>(&sm_scale[wave][32 + 16 * h + 4 * g]);
        vs[h][0] = w.x, vs[h][1] = w.y, vs[h][2] = w.z, vs[h][3] = w.w;
        x[h][0] = s[h][0] * ks.x, x[h][1] = s[h][1] * ks.y;
        x[h][2] = s[h][2] * ks.z, x[h][3] = s[h][3] * ks.w;
      }
      if (keys[0] + keys[1] < kKeys || t * kKeys < first) {
        asm volatile("");  // a branch: most tiles are whole
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (4 * g + r >= keys[h] || pos + 16 * h + r < first) x[h][r] = kNegInf;
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
      __builtin_amdgcn_wave_barrier();
      load_keys(t + W, next0, next1);

      float top = kNegInf;
#pragma unroll
      for (int h = 0; h < 2; ++h) top = fmaxf(top, fmaxf(fmaxf(x[h][0], x[h][1]), fmaxf(x[h][2], x[h][3])));
      const float mn = fmaxf(m, row_max(top));
      const float mu = mn == kNegInf ? 0.f : mn;
      if (!__all(mn == m)) {
        const float alpha = fast_exp2(m - mu);
        l *= alpha;
        weighed *= alpha;
#pragma unroll
        for (int e = 0; e < kVB; ++e) o[e] *= alpha;
      }
      m = mn;
      uint4 w[kWP];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float e = fast_exp2(x[h][r] - mu);
          l += e;
          x[h][r] = e * vs[h][r];
        }
#pragma unroll
      for (int part = 0; part < kWP; ++part) {
        auto take = [&](float& a, float& b) { return part == kWP - 1 ? pack_bf16x2(a, b) : take_part(a, b); };
        w[part] = make_uint4(take(x[0][0], x[0][1]), take(x[0][2], x[0][3]), take(x[1][0], x[1][1]), take(x[1][2], x[1][3]));
      }
      // O^T += V^T P^T
      if (S::kBiased && __builtin_expect(!convert, 1)) {
        constexpr uint32_t kZeros = 0x00800080u;
#pragma unroll
        for (int part = kWP - 1; part >= 0; --part)
          weighed = mfma_bf16(make_uint4(kZeros, kZeros, kZeros, kZeros), w[part], weighed);
#pragma unroll
        for (int d = 0; d < kVD; ++d) {
          uint32_t y[2][4];
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int r = 0; r < 4; ++r) y[h][r] = v[h][r][d] ^ kBias;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint4 rows = make_uint4(byte_pair(y[0][0], y[0][1], e), byte_pair(y[0][2], y[0][3], e),
                                          byte_pair(y[1][0], y[1][1], e), byte_pair(y[1][2], y[1][3], e));
#pragma unroll
            for (int part = kWP - 1; part >= 0; --part) o[4 * d + e] = mfma_bf16(rows, w[part], o[4 * d + e]);
          }
        }
      } else {
#pragma unroll
        for (int d = 0; d < kVD; ++d)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint4 rows = make_uint4(high_halves(byte_of(v[0][0][d], e), byte_of(v[0][1][d], e)),
                                          high_halves(byte_of(v[0][2][d], e), byte_of(v[0][3][d], e)),
                                          high_halves(byte_of(v[1][0][d], e), byte_of(v[1][1][d], e)),
                                          high_halves(byte_of(v[1][2][d], e), byte_of(v[1][3][d], e)));
#pragma unroll
            for (int part = kWP - 1; part >= 0; --part) o[4 * d + e] = mfma_bf16(rows, w[part], o[4 * d + e]);
          }
      }
      load_values(t + W, next0, next1);
      t += W;
      next0 = page_of(t + W, 0);
      next1 = page_of(t + W, 1);
    }
  }
  // Tag the unit's arrival word.
  if (split_keys && threadIdx.x == 0 && (arrive_old >> 16) != a.tag)
    __hip_atomic_compare_exchange_strong(arrive, &arrive_old, a.tag << 16, __ATOMIC_RELAXED, __ATOMIC_RELAXED,
                                         __HIP_MEMORY_SCOPE_AGENT);

  // Merge the waves, kMerged heads at a time: accumulator r of tile e is dimension (4 g +
  // r) kVB + e.
  if constexpr (S::kBiased) {
#pragma unroll
    for (int e = 0; e < kVB; ++e) o[e] -= weighed;
  }
  const float sum_keys = row_sum(l);
  if (g == 0) {
    sm_m[wave][i] = m;
    sm_l[wave][i] = sum_keys;
  }
  const int64_t split_row = ((int64_t)blockIdx.y * a.share + blockIdx.x) * a.tile_heads;
  const int64_t unit_rows = split_row - (int64_t)split * a.tile_heads;
  for (int h0 = 0; h0 < held; h0 += kMerged) {
    __syncthreads();
    if (i >= h0 && i < h0 + kMerged) {
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int e = 0; e < kVB; e += 4)
          *reinterpret_cast<float4*>(&sm_o[wave][i - h0][(4 * g + r) * kVB + e]) =
              make_float4(o[e][r], o[e + 1][r], o[e + 2][r], o[e + 3][r]);
    }
    __syncthreads();
    for (int it = threadIdx.x; it < min(held - h0, kMerged) * (HD / 4); it += 64 * W) {
      const int row = it / (HD / 4), d = it % (HD / 4) * 4, head = h0 + row;
      float mx = kNegInf;
#pragma unroll
      for (int u = 0; u < W; ++u) mx = fmaxf(mx, sm_m[u][head]);
      const float mu = mx == kNegInf ? 0.f : mx;
      float sum = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int u = 0; u < W; ++u) {
        const float wt = fast_exp2(sm_m[u][head] - mu);
        const float4 y = *reinterpret_cast<const float4*>(&sm_o[u][row][d]);
        sum = fmaf(sm_l[u][head], wt, sum);
        x[0] = fmaf(y.x, wt, x[0]);
        x[1] = fmaf(y.y, wt, x[1]);
        x[2] = fmaf(y.z, wt, x[2]);
        x[3] = fmaf(y.w, wt, x[3]);
      }
      if (split_keys) {
        const int64_t to = split_row + head;
        float* po = a.ws_o + to * HD + d;
        store_shared2(po, x[0], x[1]);
        store_shared2(po + 2, x[2], x[3]);
        if (d == 0) store_shared2(a.ws_ml + to * 2, mx, sum);
      } else {
        store_head<T>(a, b, head0 + head, d, x, sum);
      }
    }
  }
  if (!split_keys) return;

  // Arrive once every wave's partial stores are in memory.
  __builtin_amdgcn_s_waitcnt(kWaitVmem);
  __syncthreads();
  if (threadIdx.x == 0) {
    const unsigned long long before = __hip_atomic_fetch_add(arrive, 1ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    sm_last = (int)(before & 0xffffull) == splits - 1;
    if (sm_last) __hip_atomic_store(arrive, 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!sm_last) return;  // uniform over the workgroup

  // Groups of threads share the splits, eight a round trip, and join in LDS.
  const int items = held * (HD / 4), parts = max(1, min(64 * W / items, (splits + 7) / 8));
  float* const joined = reinterpret_cast<float*>(sm_pool);
  for (int at = threadIdx.x; at < parts * items; at += 64 * W) {
    const int part = at / items, it = at - part * items, row = it / (HD / 4), d = it % (HD / 4) * 4;
    float mx = kNegInf, sum = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
    constexpr int kBatch = 8;
    for (int s0 = part; s0 < splits; s0 += kBatch * parts) {
      float pm[kBatch], pl[kBatch], px[kBatch][4];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int64_t from = unit_rows + (int64_t)min(s0 + u * parts, splits - 1) * a.tile_heads + row;
        load_shared2(a.ws_ml + from * 2, pm[u], pl[u]);
        load_shared2(a.ws_o + from * HD + d, px[u][0], px[u][1]);
        load_shared2(a.ws_o + from * HD + d + 2, px[u][2], px[u][3]);
      }
      float mn = mx;
#pragma unroll
      for (int u = 0; u < kBatch; ++u) mn = fmaxf(mn, pm[u]);  // (the surplus repeats the last split)
      const float mu = mn == kNegInf ? 0.f : mn;
      const float w0 = fast_exp2(mx - mu);
      mx = mn;
      sum *= w0;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] *= w0;
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        if (s0 + u * parts >= splits) continue;
        const float wt = fast_exp2(pm[u] - mu);
        sum = fmaf(pl[u], wt, sum);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = fmaf(px[u][e], wt, x[e]);
      }
    }
    if (parts == 1) {
      store_head<T>(a, b, head0 + row, d, x, sum);
    } else {
      float* to = joined + at * 6;
      to[0] = mx, to[1] = sum;
#pragma unroll
      for (int e = 0; e < 4; ++e) to[2 + e] = x[e];
    }
  }
  if (parts == 1) return;
  __syncthreads();
  for (int it = threadIdx.x; it < items; it += 64 * W) {
    float mx = kNegInf, sum = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
    for (int part = 0; part < parts; ++part) mx = fmaxf(mx, joined[(part * items + it) * 6]);
    const float mu = mx == kNegInf ? 0.f : mx;
    for (int part = 0; part < parts; ++part) {
      const float* from = joined + (part * items + it) * 6;
      const float wt = fast_exp2(from[0] - mu);
      sum = fmaf(from[1], wt, sum);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = fmaf(from[2 + e], wt, x[e]);
    }
    store_head<T>(a, b, head0 + it / (HD / 4), it % (HD / 4) * 4, x, sum);
  }
}

template <typename T, int HD, int W, bool APPEND>
hipError_t launch_waves(const Decode8Args& a, hipStream_t stream) {
  const bool split = a.share > 0;
  const dim3 grid(split ? a.share : 1, a.p.cache.heads_kv * a.head_tiles, split ? 1 : a.p.cache.batch), block(64 * W);
  if (a.p.cache.block_table != nullptr)
    hipLaunchKernelGGL((decode8_kernel<T, HD, W, true, APPEND>), grid, block, 0, stream, a);
  else
    hipLaunchKernelGGL((decode8_kernel<T, HD, W, false, APPEND>), grid, block, 0, stream, a);
  return hipGetLastError();
}

template <typename T, int HD, bool APPEND>
hipError_t launch_head(const Decode8Args& a, const Decode8Plan& plan, hipStream_t stream) {
  return plan.waves == 8 ? launch_waves<T, HD, 8, APPEND>(a, stream) : launch_waves<T, HD, 4, APPEND>(a, stream);
}

template <typename T, bool APPEND>
hipError_t launch_typed(const Decode8Args& a, const Decode8Plan& plan, hipStream_t stream) {
  switch (a.p.cache.head_dim) {
    case 64: return launch_head<T, 64, APPEND>(a, plan, stream);
    case 128: return launch_head<T, 128, APPEND>(a, plan, stream);
    default: return launch_head<T, 256, APPEND>(a, plan, stream);
  }
}

template <bool APPEND>
hipError_t launch_step(const Decode8Args& a, const Decode8Plan& plan, hipStream_t stream) {
  return a.p.dtype == ASRATTN_BF16 ? launch_typed<bf16_raw, APPEND>(a, plan, stream)
                                   : launch_typed<float, APPEND>(a, plan, stream);
}

}  // namespace

// A unit is a sequence's block of query heads.  256 units or more fill the card with
// workgroups of four waves, several to a compute unit (64 sequences of 8 kv heads 18.0 us,
// with eight waves 23.6); fewer leave it to the eight waves of one (one of 4000 keys in
// splits 11.0, with four 14.0).  Up to 128, keys are split over about 256 workgroups,
// at least a turn of the waves each.  Long keys of several sequences are split by
// lengths, which the device knows alone: two of 40 001 and 65 511 keys of room for 65 536
// 47.8 us, in equal splits 56.0; where lengths are alike (8 of 8000 to 8192, 2 kv
// heads) finding the split costs 1.3 of 15.6 us, and below 4096 keys more than it gives.
Decode8Plan decode8_plan(const asrlayer_decode8_params& p) {
  const asrlayer_cache8& c = p.cache;
  Decode8Plan plan;
  const int group = p.heads_q / c.heads_kv;
  plan.head_tiles = (group + 15) / 16;
  const int span = p.window > 0 && p.window < c.max_len ? p.window : c.max_len;
  const long long blocks = (long long)c.heads_kv * plan.head_tiles, units = blocks * c.batch;
  plan.share = plan.splits = 0;
  plan.waves = units > 256 ? 4 : 8;
  if (units >= 1 && units <= 128 && units * span < (1LL << 35)) {
    if (c.batch > 1 && span >= 4096) {
      plan.waves = 4;
      plan.share = (int)(256 / blocks);
    } else {
      const int by_units = (int)(256 / units), by_keys = span / (plan.waves * kKeys);
      plan.splits = by_units < by_keys ? by_units : by_keys;
      plan.splits = plan.splits <= 1 ? 0 : plan.splits;
      plan.share = plan.splits * c.batch;
    }
  }
  return plan;
}

hipError_t launch_decode8(const asrlayer_decode8_params& p, const asrlayer_append8_params* append, const Decode8Plan& plan,
                          float* ws_o, float* ws_ml, unsigned long long* ws_arrive, hipStream_t stream) {
  Decode8Args a{};
  a.p = p;
  if (append != nullptr) a.n = *append;
  a.page_shift = 0;
  while (p.cache.block_table != nullptr && (1 << a.page_shift) < p.cache.page_size) ++a.page_shift;
  a.head_tiles = plan.head_tiles;
  a.share = plan.share;
  a.splits = plan.splits;
  const int group = p.heads_q / p.cache.heads_kv;
  a.tile_heads = group < 16 ? group : 16;
  a.c = p.scale * kLog2e;
  a.c_part = std::frexp(p.scale, &a.c_power) * kLog2e;
  a.ws_o = ws_o;
  a.ws_ml = ws_ml;
  a.ws_arrive = ws_arrive;
  a.tag = plan.share > 0 ? launch_tag() : 0;
  return append != nullptr ? launch_step<true>(a, plan, stream) : launch_step<false>(a, plan, stream);
}

}  // namespace asrattn
