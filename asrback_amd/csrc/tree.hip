// Attention of a tree of drafted tokens over a key/value cache
// (asrlayer_tree).
//
// T drafted tokens of G query heads a kv head make M = T G query rows over the
// same keys: the cache's n, which every row sees, and the T drafted ones, of
// which a row sees its token's ancestors (a bit mask).  A key and its value are
// read once for 4 M head_dim operations, M flops a byte in bf16, so up to a few
// hundred rows the step is bound by reading the cache, and the rows ride along on
// the matrix cores:
//
//   * A workgroup takes 16 or 32 rows of one (sequence, kv head) and a range of its
//     keys; its waves take tiles of 16 or 32 keys in turn, each wave with all the
//     rows and a softmax state of its own.  A wave loads its next tile's keys while
//     it weighs the values and its next values while it scores the keys; there are
//     no barriers between the first and the last tile.
//   * Loads go over whole positions (consecutive lanes, consecutive bytes: a load
//     whose neighbouring lanes lie in different positions takes four times as long in
//     the vector cache, and bound the kernel).  The product of keys and queries needs
//     16 different keys in neighbouring lanes, so the keys change lanes through the
//     wave's own LDS; the values' product wants 16 dimensions there and takes them
//     from the registers.
//   * Scores come out transposed, S^T = K Q^T: a lane then holds four keys'
//     scores of one query row for each 16 keys, so the softmax state of a row
//     is a scalar per lane, its reduction two lane swaps, and the weights are
//     already the operand of O^T = V^T P^T, whose accumulators again lie one
//     row to a lane.  The order of the keys inside a product is free as long as
//     both operands agree, which is what lets the scores' layout be the
//     operand's.
//   * V^T needs, per lane, four (f32: one) keys of one dimension.  In float32 the
//     loads give that.  In bf16 a lane loads a row of eight dimensions of each of
//     eight keys and pairs them up with byte permutes (one for two elements).
//
// Waves merge in LDS at the end; splits of the keys leave partials in the
// workspace, and the split that arrives last folds them, as in the decoder step's
// kernel (decode_kernels.hpp: the arrival words' protocol is described there).
//
// Weights are rounded to bf16 for the product with bf16 values (half a step, at
// most 2^-8 of each), sums, maxima and outputs are float32 until the one rounding at
// the end; float32 inputs stay float32 throughout.
#include <type_traits>

#include "common.hpp"
#include "kernels.hpp"
#include "row_ops.hpp"

namespace asrattn {
namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef short short4_t __attribute__((ext_vector_type(4)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef unsigned short u16x2_t __attribute__((ext_vector_type(2)));
typedef short i16x2_t __attribute__((ext_vector_type(2)));
typedef unsigned int u32x2_t __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4_t __attribute__((ext_vector_type(4)));

// Cache policy of device scope (sc1).
constexpr int kDeviceScope = 16;

struct TreeArgs {
  asrlayer_tree_params p;
  int page_shift, rows, row_blocks, splits;
  bool out_vectors;  // out's rows take vectors of four elements
  bool fold_apart;   // the fold is a launch of its own
  float c;  // scale * log2(e)
  float group_inv;  // 1 / query heads per kv head
  float* ws_o;   // [unit][split][16 row_tiles][head_dim]
  float* ws_ml;  // [unit][split][16 row_tiles][2]
  unsigned long long* ws_arrive;  // [unit]
  unsigned long long tag;
};

template <typename T, int HD>
struct TreeShape {
  static constexpr int kES = (int)sizeof(T);
  // 16-key parts of a tile: two make up the bf16 product's depth, where they fit
  // the registers.
  static constexpr int kSub = kES == 2 && HD <= 128 ? 2 : 1;
  // The most waves of a workgroup (of a kilobyte a position, four: 512 registers
  // each).
  static constexpr int kWaves = HD * kES > 512 ? 4 : 8;
  // Waves the registers leave room for on a SIMD, said to the compiler: for one of
  // four waves it would take twice the registers, and half the workgroups fit.
  static constexpr int kWavesPerSimd = HD * kES > 512 ? 1 : 2;
  static constexpr int kKeys = 16 * kSub;           // keys of a tile
  static constexpr int kKV = HD * kES / 64;         // a lane's 16-byte pieces of a key part
  static constexpr int kLPR = HD * kES / 16;        // 16-byte pieces of a position
  static constexpr int kVB = HD * kES >= 256 ? 16 : 8;  // bytes of a lane's piece of a value
  static constexpr int kVD = kVB / 4;               // dwords of it
  static constexpr int kEV = kVB / kES;             // elements of it
  static constexpr int kNC = HD / (16 * kEV);       // pieces of a value per lane
  static constexpr int kTiles = HD / 16;            // 16-row tiles of O^T
  static constexpr int kDC = HD < 128 ? HD : 128;   // dimensions merged at a time
};

__device__ __forceinline__ f32x4_t mfma_bf16(const uint4& a, const uint4& b, const f32x4_t& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0,
                                                 0, 0);
}
// The same over four keys a lane.
__device__ __forceinline__ f32x4_t mfma_bf16(const uint2& a, const uint2& b, const f32x4_t& c) {
  return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(short4_t, a), __builtin_bit_cast(short4_t, b), c, 0,
                                                   0, 0);
}
__device__ __forceinline__ f32x4_t mfma_f32(uint32_t a, uint32_t b, const f32x4_t& c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a), __uint_as_float(b), c, 0, 0, 0);
}

// acc += (16 keys x 64 bytes) (16 rows x 64 bytes)^T
template <typename T>
__device__ __forceinline__ f32x4_t score_piece(const uint4& k, const uint4& q, f32x4_t acc) {
  if constexpr (sizeof(T) == 2) return mfma_bf16(k, q, acc);
  acc = mfma_f32(k.x, q.x, acc);
  acc = mfma_f32(k.y, q.y, acc);
  acc = mfma_f32(k.z, q.z, acc);
  return mfma_f32(k.w, q.w, acc);
}

template <int B>
__device__ __forceinline__ void load_piece(__amdgpu_buffer_rsrc_t rsrc, uint32_t off, uint32_t* out) {
  if constexpr (B == 16) {
    const u32x4_t v = __builtin_amdgcn_raw_buffer_load_b128(rsrc, off, 0, 0);
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = v[i];
  } else {
    const u32x2_t v = __builtin_amdgcn_raw_buffer_load_b64(rsrc, off, 0, 0);
    out[0] = v[0];
    out[1] = v[1];
  }
}

// Sum or maximum over the four lanes that hold one query row (16 apart).
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

// Ones over the infinities and NaN of a dword of T: one more in the exponent carries
// into the sign.
template <typename T>
__device__ __forceinline__ uint32_t not_finite(uint32_t x) {
  if constexpr (sizeof(T) == 4) return (uint32_t)((int32_t)((x & 0x7fffffffu) + 0x00800000u) >> 31);
  const u16x2_t t = __builtin_bit_cast(u16x2_t, x & 0x7fff7fffu) + (unsigned short)0x80;
  return __builtin_bit_cast(uint32_t, __builtin_bit_cast(i16x2_t, t) >> (short)15);
}

// Offset of a load that is to return zeros.
constexpr uint32_t kNowhere = 0x7ff00000u;

// The token of query row m and the row's head within its kv head's.  A row's token
// is below 64 and m + 0.5 at least 0.5 / group away from a multiple of group, which the
// float32 product, off by 2^-22 of itself, resolves up to 4096 heads.
struct Row {
  int token, head;
};
__device__ __forceinline__ Row row_of(const TreeArgs& a, int group, int m) {
  const int t = (int)(((float)m + 0.5f) * a.group_inv);
  return {t, m - t * group};
}

// 16 bytes of a partial that another workgroup of the launch reads: written through
// to memory and read from there (device scope), as the L2 caches of different XCDs
// are not coherent.
__device__ __forceinline__ void store_shared4(__amdgpu_buffer_rsrc_t rsrc, uint32_t off, const float* x) {
  const u32x4_t v = {__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3])};
  __builtin_amdgcn_raw_buffer_store_b128(v, rsrc, off, 0, kDeviceScope);
}
__device__ __forceinline__ void load_shared4(__amdgpu_buffer_rsrc_t rsrc, uint32_t off, float* x) {
  const u32x4_t v = __builtin_amdgcn_raw_buffer_load_b128(rsrc, off, 0, kDeviceScope);
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = __uint_as_float(v[e]);
}

// Dimensions d .. d + 3 of a query row: the weighted sum of values over the sum of
// the weights.
template <typename T>
__device__ __forceinline__ void store_row(const TreeArgs& a, int b, int hkv, int mrow, int d, const float* x, float sum) {
  const asrlayer_tree_params& p = a.p;
  const int group = p.heads_q / p.heads_kv;
  const Row r = row_of(a, group, mrow);
  T* op = static_cast<T*>(p.out) + (int64_t)b * p.o_batch_stride + (int64_t)r.token * p.o_token_stride +
          (int64_t)(hkv * group + r.head) * p.o_head_stride + d;
  float y[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = sum == 0.f ? 0.f : x[e] / sum;
  if (a.out_vectors) {
    if constexpr (sizeof(T) == 2)
      *reinterpret_cast<uint2*>(op) = make_uint2(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]));
    else
      *reinterpret_cast<float4*>(op) = make_float4(y[0], y[1], y[2], y[3]);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) Elem<T>::store1(op + e, y[e]);
  }
}

// Folds the partials of splits first, first + by, ... of a row, dimensions d .. d +
// 3, eight a round trip; split 0's row is row `row` of the unit's first, the others
// follow `apart` rows apart.  Returns the sum of the weights, mx their maximum's exponent.  HERE: the
// partials come from workgroups of the same launch.
template <bool HERE>
__device__ __forceinline__ float fold_splits(const TreeArgs& a, int64_t first_row, int row, int apart, int head_dim, int d,
                                             int first, int by, float& mx, float* x) {
  constexpr int kBatch = 8;
  const int64_t row0 = first_row + row;
  const __amdgpu_buffer_rsrc_t rsrc = buffer_rsrc(a.ws_o + first_row * head_dim, HERE ? a.splits * apart * head_dim * 4 : 0);
  float sum = 0.f;
  mx = kNegInf;
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = 0.f;
  for (int s0 = first; s0 < a.splits; s0 += kBatch * by) {
    float pm[kBatch], pl[kBatch], px[kBatch][4];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int64_t at = row0 + (int64_t)min(s0 + u * by, a.splits - 1) * apart;
      const float* po = a.ws_o + at * head_dim + d;
      if constexpr (HERE) {
        load_shared2(a.ws_ml + at * 2, pm[u], pl[u]);
        load_shared4(rsrc, (uint32_t)(at - first_row) * (head_dim * 4) + d * 4, px[u]);
      } else {
        const float2 ml = *reinterpret_cast<const float2*>(a.ws_ml + at * 2);
        const float4 v = *reinterpret_cast<const float4*>(po);
        pm[u] = ml.x, pl[u] = ml.y;
        px[u][0] = v.x, px[u][1] = v.y, px[u][2] = v.z, px[u][3] = v.w;
      }
    }
    float mn = mx;
#pragma unroll
    for (int u = 0; u < kBatch; ++u) mn = s0 + u * by < a.splits ? fmaxf(mn, pm[u]) : mn;
    const float mu = mn == kNegInf ? 0.f : mn;
    const float w0 = fast_exp2(mx - mu);
    mx = mn;
    sum *= w0;
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] *= w0;
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      if (s0 + u * by >= a.splits) continue;  // the surplus repeats the last split
      const float wt = fast_exp2(pm[u] - mu);
      sum = fmaf(pl[u], wt, sum);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = fmaf(px[u][e], wt, x[e]);
    }
  }
  return sum;
}

// Where piece c of row r lies in a block of rows in LDS, so that the 16 rows a
// matrix operand takes a piece of lie in 16 different groups of banks.
template <int LPR>
__device__ __forceinline__ int lds_piece(int r, int c) {
  return r * LPR + (LPR == 8 ? c ^ ((r >> 1) & 7) : c ^ (r & 15));
}

// A workgroup: RT x 16 query rows, its W waves the shares of the keys.
template <typename T, int HD, int RT, int W, bool PAGED>
__global__ __launch_bounds__(64 * W, (TreeShape<T, HD>::kWavesPerSimd)) void tree_kernel(const TreeArgs a) {
  using S = TreeShape<T, HD>;
  constexpr int kSub = S::kSub, kKeys = S::kKeys, kKV = S::kKV, kVD = S::kVD, kEV = S::kEV, kNC = S::kNC;
  constexpr int kES = S::kES, kDC = S::kDC;
  constexpr int kRows = RT * 16;
  // Queries that would not fit beside the keys, values and sums stay in LDS.
  constexpr bool kQLds = kKV * RT > 8;
  constexpr int kLPR = S::kLPR;
  const asrlayer_tree_params& p = a.p;

  int split = blockIdx.x, hkv = blockIdx.y, b = blockIdx.z, rb = 0;
  if (a.row_blocks > 1) {
    // Workgroups go round the 8 XCDs: those of one range of keys, which differ in
    // their rows, follow each other on one XCD and share its L2.
    const int id = blockIdx.x, turn = id / (8 * a.row_blocks);
    const int range = turn * 8 + id % 8, pair = range / a.splits;
    rb = id / 8 % a.row_blocks;
    split = range % a.splits;
    b = pair / p.heads_kv;
    hkv = pair % p.heads_kv;
    if (b >= p.batch) return;
  }
  const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int group = p.heads_q / p.heads_kv;
  const int64_t unit = ((int64_t)b * p.heads_kv + hkv) * a.row_blocks + rb;
  const bool split_keys = a.splits > 1, fold_here = split_keys && !a.fold_apart;
  unsigned long long* const arrive = a.ws_arrive + unit;
  unsigned long long arrive_old = 0;
  if (fold_here && threadIdx.x == 0)
    arrive_old = __hip_atomic_load(arrive, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);

  // LDS: the keys of each wave and the workgroup's queries; after them, the waves'
  // sums of 16 rows.
  constexpr int kKeyPieces = kKeys * kLPR, kQueryPieces = kRows * kLPR, kSumPieces = W * 16 * (kDC + 4) / 4;
  constexpr int kPieces = W * kKeyPieces + kQueryPieces;
  __shared__ uint4 sm_pool[kPieces > kSumPieces ? kPieces : kSumPieces];
  __shared__ float sm_m[W][RT * 16], sm_l[W][RT * 16];
  __shared__ int sm_last;
  uint4* const sm_k = sm_pool + wave * kKeyPieces;
  uint4* const sm_q = sm_pool + W * kKeyPieces;
  float(*const sm_o)[16][kDC + 4] = reinterpret_cast<float(*)[16][kDC + 4]>(sm_pool);

  // The workgroup's query rows (rows past the last repeat it).  Vectors of the
  // compiler's own: an array of structs it moves to LDS, addressed by sizes that it
  // reads from the launch's packet in host memory (6 us).
  constexpr int kTurns = (kQueryPieces + 64 * W - 1) / (64 * W);
  u32x4_t staged[kTurns];
#pragma unroll
  for (int u = 0; u < kTurns; ++u) {
    const int at = min((int)threadIdx.x + u * 64 * W, kQueryPieces - 1);
    const Row r = row_of(a, group, min(rb * kRows + at / kLPR, a.rows - 1));
    staged[u] = reinterpret_cast<const u32x4_t*>(
        static_cast<const T*>(p.q) + (int64_t)b * p.q_batch_stride + (int64_t)r.token * p.q_token_stride +
        (int64_t)(hkv * group + r.head) * p.q_head_stride)[at % kLPR];
  }
  uint64_t mask[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const Row r = row_of(a, group, min(rb * kRows + rt * 16 + i, a.rows - 1));
    mask[rt] = (uint64_t)p.masks[(int64_t)b * p.masks_batch_stride + r.token];
  }

  // Where tile t's keys and values lie: their first positions' addresses, the
  // positions' distance in bytes, and how many the tile holds (0, as past the
  // split's last tile: nothing is read).  All of it uniform, and a few scalar
  // instructions a tile.
  const uint64_t kbase = (uint64_t)p.k + ((PAGED ? 0 : b * p.k_batch_stride) + hkv * p.k_head_stride) * kES;
  const uint64_t vbase = (uint64_t)p.v + ((PAGED ? 0 : b * p.v_batch_stride) + hkv * p.v_head_stride) * kES;
  const uint64_t kdbase = (uint64_t)p.k_draft + (b * p.kd_batch_stride + hkv * p.kd_head_stride) * kES;
  const uint64_t vdbase = (uint64_t)p.v_draft + (b * p.vd_batch_stride + hkv * p.vd_head_stride) * kES;
  const uint32_t kstep = (uint32_t)p.k_token_stride * kES, vstep = (uint32_t)p.v_token_stride * kES;
  const uint32_t kdstep = (uint32_t)p.kd_token_stride * kES, vdstep = (uint32_t)p.vd_token_stride * kES;
  const int32_t* const pages = PAGED ? p.block_table + (int64_t)b * p.bt_stride : nullptr;
  int n = p.max_len_k;
  if (p.lengths != nullptr) {
    const int64_t held = p.lengths64 ? load_uniform(static_cast<const int64_t*>(p.lengths) + b)
                                     : (int64_t)load_uniform(static_cast<const int32_t*>(p.lengths) + b);
    n = held < 0 ? 0 : held < n ? (int)held : n;
  }
  n = __builtin_amdgcn_readfirstlane(n);
  const int cache_tiles = n / kKeys + (n % kKeys != 0);
  const int tiles = cache_tiles + (p.tokens + kKeys - 1) / kKeys;
  const int per = (tiles + a.splits - 1) / a.splits;
  const int t0 = min(tiles, split * per), t1 = min(tiles, t0 + per);

  // Paged: pool pages of a tile's parts (-1: none), read a tile ahead.
  struct Pages {
    int part[kSub];
  };
  auto pages_of = [&](int t) -> Pages {
    Pages e;
#pragma unroll
    for (int s = 0; s < kSub; ++s) {
      e.part[s] = -1;
      if constexpr (PAGED) {
        const int pi = (t * kKeys + s * 16) >> a.page_shift;
        const int entry = load_uniform(pages + (t < cache_tiles && pi < p.bt_stride ? pi : 0));
        e.part[s] = entry < p.num_pages ? entry : -1;
      }
    }
    return e;
  };
  struct Part {
    __amdgpu_buffer_rsrc_t rsrc;
    uint32_t step;
    int keys;
  };
  auto part_of = [&](int t, int s, bool values, const Pages& e) -> Part {
    const bool drafted = t >= cache_tiles;
    const int j = (drafted ? t - cache_tiles : t) * kKeys + s * 16;
    const uint32_t step = drafted ? (values ? vdstep : kdstep) : (values ? vstep : kstep);
    int keys = t < t1 ? min(max((drafted ? p.tokens : n) - j, 0), 16) : 0;
    uint64_t at = (drafted ? (values ? vdbase : kdbase) : (values ? vbase : kbase));
    uint32_t first = j;  // position in the memory at `at`
    if constexpr (PAGED) {
      const int page = drafted ? 0 : kSub == 1 || s == 0 ? e.part[0] : e.part[kSub - 1];
      first &= drafted ? 0xffffffffu : (1u << a.page_shift) - 1;
      keys = page >= 0 ? keys : 0;
      at += (uint64_t)max(page, 0) * (uint64_t)((values ? p.v_page_stride : p.k_page_stride) * kES);
    }
    at += (uint64_t)first * step;
    const uint64_t uniform_at = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(at >> 32)) << 32 |
                                (uint32_t)__builtin_amdgcn_readfirstlane((int)at);
    const uint32_t bytes = keys > 0 ? (uint32_t)(keys - 1) * step + HD * kES : 0u;
    return {buffer_rsrc(reinterpret_cast<const void*>(uniform_at), __builtin_amdgcn_readfirstlane(bytes)), step, keys};
  };

  // What a wave loads of a tile: keys with whole positions in the lanes of one load,
  // values as the product takes them.
  uint4 k[kSub][kKV];
  uint32_t v[kSub][4][kNC][kVD];
  int keys[kSub];
  auto load_keys = [&](int t, const Pages& e) {
#pragma unroll
    for (int s = 0; s < kSub; ++s) {
      const Part x = part_of(t, s, false, e);
      keys[s] = x.keys;
#pragma unroll
      for (int u = 0; u < kKV; ++u) {
        const int j = u * (64 / kLPR) + lane / kLPR;
        const uint32_t off = j < x.keys ? (uint32_t)j * x.step + lane % kLPR * 16 : kNowhere;
        k[s][u] = buffer_load16(x.rsrc, off);
      }
    }
  };
  auto load_values = [&](int t, const Pages& e) {
#pragma unroll
    for (int s = 0; s < kSub; ++s) {
      const Part x = part_of(t, s, true, e);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int j = 4 * g + r;
        const uint32_t off = j < x.keys ? (uint32_t)j * x.step + i * S::kVB : kNowhere;
#pragma unroll
        for (int c = 0; c < kNC; ++c) load_piece<S::kVB>(x.rsrc, off + c * 16 * S::kVB, v[s][r][c]);
      }
    }
  };
  int t = t0 + wave;
  Pages next_pages;
  {
    const Pages first = pages_of(t);
    next_pages = pages_of(t + W);
    load_keys(t, first);
    load_values(t, first);
  }
  // Tag the unit's arrival word, whose load was issued first of all; the answer
  // is not waited for.
  if (fold_here && threadIdx.x == 0 && (arrive_old >> 16) != a.tag)
    __hip_atomic_compare_exchange_strong(arrive, &arrive_old, a.tag << 16, __ATOMIC_RELAXED, __ATOMIC_RELAXED,
                                         __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
  for (int u = 0; u < kTurns; ++u) {
    const int at = min((int)threadIdx.x + u * 64 * W, kQueryPieces - 1);
    sm_q[lds_piece<kLPR>(at / kLPR, at % kLPR)] = __builtin_bit_cast(uint4, staged[u]);
  }
  // An LDS-only barrier: the keys and values stay in flight across it.
  auto lds_barrier = [] {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
  };
  lds_barrier();
  // The lane's piece c of its row of a row tile, and of its key of a part.
  auto query = [&](int rt, int c) { return sm_q[lds_piece<kLPR>(rt * 16 + i, c * 4 + g)]; };
  uint4 q[kQLds ? 1 : RT][kKV];
  if constexpr (!kQLds) {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int c = 0; c < kKV; ++c) q[rt][c] = query(rt, c);
  }

  f32x4_t o[RT][S::kTiles];
  float m[RT], l[RT];  // l: the lane's own keys only
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    m[rt] = kNegInf;
    l[rt] = 0.f;
#pragma unroll
    for (int e = 0; e < S::kTiles; ++e) o[rt][e] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  unsigned infinite = 0;  // drafted tiles of which values were left out

  // One tile, the next one loading meanwhile: without a branch around the loads
  // the compiler waits for no more of them than it needs.
  auto consume = [&](auto in_draft) {
    constexpr bool drafted = decltype(in_draft)::value;
    // The keys change lanes through the wave's own LDS.
#pragma unroll
    for (int h = 0; h < kSub; ++h)
#pragma unroll
      for (int u = 0; u < kKV; ++u)
        sm_k[lds_piece<kLPR>(h * 16 + u * (64 / kLPR) + lane / kLPR, lane % kLPR)] = k[h][u];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
    __builtin_amdgcn_wave_barrier();
    f32x4_t s[RT][kSub];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int h = 0; h < kSub; ++h) s[rt][h] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < kKV; ++c) {
      uint4 kc[kSub];
#pragma unroll
      for (int h = 0; h < kSub; ++h) kc[h] = sm_k[lds_piece<kLPR>(h * 16 + i, c * 4 + g)];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const uint4 qc = kQLds ? query(rt, c) : q[kQLds ? 0 : rt][c];
#pragma unroll
        for (int h = 0; h < kSub; ++h) s[rt][h] = score_piece<T>(kc[h], qc, s[rt][h]);
      }
    }

    // Keys that a row does not see: past a part's keys, or no ancestor's.
    bool whole = !drafted;
#pragma unroll
    for (int h = 0; h < kSub; ++h) whole = whole && keys[h] == 16;
    if (!whole) {
      const int shift = drafted ? (t - cache_tiles) * kKeys : 0;
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int h = 0; h < kSub; ++h) {
          const uint32_t seen = drafted ? (uint32_t)(mask[rt] >> (shift + h * 16 + 4 * g)) : 0xfu;
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (4 * g + r >= keys[h] || !((seen >> r) & 1u)) s[rt][h][r] = kNegInf;
        }
    }
    load_keys(t + W, next_pages);

    uint32_t w[RT][kSub * 4 * kES / 4];  // the weights as the product's operand
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float top = fmaxf(fmaxf(s[rt][0][0], s[rt][0][1]), fmaxf(s[rt][0][2], s[rt][0][3]));
      if constexpr (kSub == 2) {
        top = fmaxf(top, fmaxf(s[rt][kSub - 1][0], s[rt][kSub - 1][1]));
        top = fmaxf(top, fmaxf(s[rt][kSub - 1][2], s[rt][kSub - 1][3]));
      }
      const float mn = fmaxf(m[rt], row_max(top) * a.c);
      const float mu = mn == kNegInf ? 0.f : mn;
      if (!__all(mn == m[rt])) {
        const float alpha = fast_exp2(m[rt] - mu);
        l[rt] *= alpha;
#pragma unroll
        for (int e = 0; e < S::kTiles; ++e) o[rt][e] *= alpha;
      }
      m[rt] = mn;
      float x[kSub][4];
#pragma unroll
      for (int h = 0; h < kSub; ++h)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          x[h][r] = fast_exp2(fmaf(s[rt][h][r], a.c, -mu));
          l[rt] += x[h][r];
        }
#pragma unroll
      for (int h = 0; h < kSub; ++h) {
        if constexpr (kES == 2) {
          w[rt][h * 2] = pack_bf16x2(x[h][0], x[h][1]);
          w[rt][h * 2 + 1] = pack_bf16x2(x[h][2], x[h][3]);
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r) w[rt][r] = __float_as_uint(x[h][r]);
        }
      }
    }

    // O^T += V^T P^T
    uint32_t bad = 0;
#pragma unroll
    for (int c = 0; c < kNC; ++c) {
      uint32_t x[kSub][4][kVD];  // the lane's piece of its four keys' values
#pragma unroll
      for (int h = 0; h < kSub; ++h)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const uint32_t* at = v[h][r][c];
#pragma unroll
          for (int d = 0; d < kVD; ++d) {
            x[h][r][d] = at[d];
            // A drafted value that some rows must not see may be infinite or NaN, and a
            // weight of zero times it is not zero: such elements leave the product,
            // and the rows that do see them take them as they are, below.
            if constexpr (drafted) {
              const uint32_t left_out = not_finite<T>(at[d]);
              x[h][r][d] = at[d] & ~left_out;
              bad |= left_out;
            }
          }
        }
      if constexpr (kES == 2) {
#pragma unroll
        for (int d = 0; d < kVD; ++d) {
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const uint32_t sel = half ? 0x07060302u : 0x05040100u;
            const uint2 first = make_uint2(__builtin_amdgcn_perm(x[0][1][d], x[0][0][d], sel),
                                           __builtin_amdgcn_perm(x[0][3][d], x[0][2][d], sel));
            const int at = c * kEV + 2 * d + half;
            if constexpr (kSub == 2) {
              const uint4 both = make_uint4(first.x, first.y, __builtin_amdgcn_perm(x[1][1][d], x[1][0][d], sel),
                                            __builtin_amdgcn_perm(x[1][3][d], x[1][2][d], sel));
#pragma unroll
              for (int rt = 0; rt < RT; ++rt)
                o[rt][at] = mfma_bf16(both, make_uint4(w[rt][0], w[rt][1], w[rt][2], w[rt][3]), o[rt][at]);
            } else {
#pragma unroll
              for (int rt = 0; rt < RT; ++rt) o[rt][at] = mfma_bf16(first, make_uint2(w[rt][0], w[rt][1]), o[rt][at]);
            }
          }
        }
      } else {
#pragma unroll
        for (int d = 0; d < kVD; ++d)
#pragma unroll
          for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int r = 0; r < 4; ++r) o[rt][c * kEV + d] = mfma_f32(x[0][r][d], w[rt][r], o[rt][c * kEV + d]);
      }
    }
    if constexpr (drafted) {
      if (__any(bad != 0)) infinite |= 1u << (t - cache_tiles);
    }
    load_values(t + W, next_pages);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
    __builtin_amdgcn_wave_barrier();
    t += W;
    next_pages = pages_of(t + W);
  };
  const int t_cache = min(t1, cache_tiles);
  while (t < t_cache) consume(std::false_type{});
  while (t < t1) consume(std::true_type{});

  // Infinite and NaN drafted values, for the rows that see them.
  if (infinite != 0) {
    for (int j = 0; j < p.tokens; ++j) {
      if (!((infinite >> (j / kKeys)) & 1u)) continue;
      const T* row = static_cast<const T*>(p.v_draft) + (int64_t)b * p.vd_batch_stride + (int64_t)hkv * p.vd_head_stride +
                     (int64_t)j * p.vd_token_stride;
#pragma unroll
      for (int c = 0; c < kNC; ++c)
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int e = 0; e < kEV; ++e) {
            const float x = Elem<T>::load1(row + (c * 16 + g * 4 + r) * kEV + e);
            const float y = (__float_as_uint(x) & 0x7f800000u) == 0x7f800000u ? x : 0.f;
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) o[rt][c * kEV + e][r] += (mask[rt] >> j) & 1u ? y : 0.f;
          }
    }
  }

  // Merge the waves that share the keys, 16 rows and kDC dimensions at a time.
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const float sum = row_sum(l[rt]);
    if (g == 0) {
      sm_m[wave][rt * 16 + i] = mask[rt] != 0 ? m[rt] : kNegInf;
      sm_l[wave][rt * 16 + i] = mask[rt] != 0 ? sum : 0.f;
    }
  }
  auto store_out = [&](int mrow, int d, const float* x, float sum) { store_row<T>(a, b, hkv, mrow, d, x, sum); };
  constexpr int kVecs = kDC / 4;
  const int held = min(kRows, a.rows - rb * kRows);
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
    for (int dc = 0; dc < HD / kDC; ++dc) {
      __syncthreads();
      constexpr int kParts = kDC / (16 * kEV);
#pragma unroll
      for (int c = 0; c < kParts; ++c)
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int e = 0; e < kEV; e += 4) {
            float4 x;
            const int at = (dc * kParts + c) * kEV + e;
            x.x = o[rt][at][r], x.y = o[rt][at + 1][r], x.z = o[rt][at + 2][r], x.w = o[rt][at + 3][r];
            if (mask[rt] == 0) x = make_float4(0.f, 0.f, 0.f, 0.f);
            *reinterpret_cast<float4*>(&sm_o[wave][i][(c * 16 + g * 4 + r) * kEV + e]) = x;
          }
      __syncthreads();
      const int items = min(max(held - rt * 16, 0), 16) * kVecs;
      for (int it = threadIdx.x; it < items; it += 64 * W) {
        const int row = it / kVecs, d = it % kVecs * 4;
        float mx = kNegInf;
#pragma unroll
        for (int u = 0; u < W; ++u) mx = fmaxf(mx, sm_m[u][rt * 16 + row]);
        const float mu = mx == kNegInf ? 0.f : mx;
        float sum = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int u = 0; u < W; ++u) {
          const float wt = fast_exp2(sm_m[u][rt * 16 + row] - mu);
          sum = fmaf(sm_l[u][rt * 16 + row], wt, sum);
          const float4 y = *reinterpret_cast<const float4*>(&sm_o[u][row][d]);
          x[0] = fmaf(y.x, wt, x[0]);
          x[1] = fmaf(y.y, wt, x[1]);
          x[2] = fmaf(y.z, wt, x[2]);
          x[3] = fmaf(y.w, wt, x[3]);
        }
        if (split_keys) {
          const int64_t at = (unit * a.splits + split) * kRows + rt * 16 + row;
          float* po = a.ws_o + at * HD + dc * kDC + d;
          float* pm = a.ws_ml + at * 2;
          if (fold_here) {
            store_shared4(buffer_rsrc(a.ws_o + unit * a.splits * kRows * HD, a.splits * kRows * HD * 4),
                          (uint32_t)(split * kRows + rt * 16 + row) * (HD * 4) + (dc * kDC + d) * 4, x);
            if (dc == 0 && d == 0) store_shared2(pm, mx, sum);
          } else {
            *reinterpret_cast<float4*>(po) = make_float4(x[0], x[1], x[2], x[3]);
            if (dc == 0 && d == 0) *reinterpret_cast<float2*>(pm) = make_float2(mx, sum);
          }
        } else {
          store_out(rb * kRows + rt * 16 + row, dc * kDC + d, x, sum);
        }
      }
    }
  }
  if (!fold_here) return;

  // Arrive once every wave's partial stores are in memory.
  __builtin_amdgcn_s_waitcnt(kWaitVmem);
  __syncthreads();
  if (threadIdx.x == 0) {
    const unsigned long long before =
        __hip_atomic_fetch_add(arrive, 1ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    sm_last = (int)(before & 0xffffull) == a.splits - 1;
    if (sm_last) __hip_atomic_store(arrive, 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!sm_last) return;  // uniform over the workgroup

  for (int it = threadIdx.x; it < held * (HD / 4); it += 64 * W) {
    const int row = it / (HD / 4), d = it % (HD / 4) * 4;
    float mx, x[4];
    const float sum = fold_splits<true>(a, unit * a.splits * kRows, row, kRows, HD, d, 0, 1, mx, x);
    store_out(rb * kRows + row, d, x, sum);
  }
}

// The fold as a launch of its own: a workgroup per row and 128 dimensions, eight
// groups of 32 threads that share the splits and four dimensions a thread, so that
// all partials of up to 64 splits are under way at once.
template <typename T>
__global__ __launch_bounds__(256) void tree_fold_kernel(const TreeArgs a, int block_rows) {
  const asrlayer_tree_params& p = a.p;
  const int64_t unit = blockIdx.y;
  const int rb = (int)(unit % a.row_blocks), row = blockIdx.x;
  if (rb * block_rows + row >= a.rows) return;
  const int col = threadIdx.x & 31, part = threadIdx.x >> 5;
  const int d = blockIdx.z * 128 + col * 4;
  const bool in = d < p.head_dim;
  __shared__ float sm_m[8], sm_l[8];
  __shared__ __attribute__((aligned(16))) float sm_x[8][128];
  float mx, x[4];
  const float sum = fold_splits<false>(a, unit * a.splits * block_rows, row, block_rows, p.head_dim, in ? d : 0, part, 8,
                                       mx, x);
  if (col == 0) {
    sm_m[part] = mx;
    sm_l[part] = sum;
  }
  *reinterpret_cast<float4*>(&sm_x[part][col * 4]) = make_float4(x[0], x[1], x[2], x[3]);
  __syncthreads();
  if (part != 0 || !in) return;
  float top = kNegInf;
#pragma unroll
  for (int u = 0; u < 8; ++u) top = fmaxf(top, sm_m[u]);
  const float mu = top == kNegInf ? 0.f : top;
  float total = 0.f, y[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int u = 0; u < 8; ++u) {
    const float wt = fast_exp2(sm_m[u] - mu);
    total = fmaf(sm_l[u], wt, total);
    const float4 v = *reinterpret_cast<const float4*>(&sm_x[u][col * 4]);
    y[0] = fmaf(v.x, wt, y[0]);
    y[1] = fmaf(v.y, wt, y[1]);
    y[2] = fmaf(v.z, wt, y[2]);
    y[3] = fmaf(v.w, wt, y[3]);
  }
  const int64_t pair = unit / a.row_blocks;
  store_row<T>(a, (int)(pair / p.heads_kv), (int)(pair % p.heads_kv), rb * block_rows + row, d, y, total);
}

template <typename T, int HD, int RT, int W>
hipError_t launch_waves(const TreeArgs& a, hipStream_t stream) {
  const dim3 block(64 * W);
  dim3 grid(a.splits, a.p.heads_kv, a.p.batch);
  if (a.row_blocks > 1) grid = dim3((a.splits * a.p.heads_kv * a.p.batch + 7) / 8 * 8 * a.row_blocks);
  if (a.p.block_table != nullptr)
    hipLaunchKernelGGL((tree_kernel<T, HD, RT, W, true>), grid, block, 0, stream, a);
  else
    hipLaunchKernelGGL((tree_kernel<T, HD, RT, W, false>), grid, block, 0, stream, a);
  return hipGetLastError();
}

template <typename T, int HD>
hipError_t launch_head(const TreeArgs& a, const TreePlan& plan, hipStream_t stream) {
  if constexpr (HD * sizeof(T) <= 512) {
    if (plan.row_tiles == 1 && plan.waves == 8) return launch_waves<T, HD, 1, 8>(a, stream);
  }
  if constexpr (HD * sizeof(T) <= 256) {
    if (plan.row_tiles == 2)
      return plan.waves == 8 ? launch_waves<T, HD, 2, 8>(a, stream) : launch_waves<T, HD, 2, 4>(a, stream);
  }
  return launch_waves<T, HD, 1, 4>(a, stream);
}

template <typename T>
hipError_t launch_typed(const TreeArgs& a, const TreePlan& plan, hipStream_t stream) {
  switch (a.p.head_dim) {
    case 64: return launch_head<T, 64>(a, plan, stream);
    case 128: return launch_head<T, 128>(a, plan, stream);
    case 256: return launch_head<T, 256>(a, plan, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace

TreePlan tree_plan(const asrlayer_tree_params& p) {
  const long long rows = (long long)p.tokens * (p.heads_q / p.heads_kv);
  const int tiles = (int)((rows + 15) / 16);
  const int bytes = p.head_dim * (p.dtype == ASRATTN_BF16 ? 2 : 4);
  const long long pairs = (long long)p.batch * p.heads_kv;
  TreePlan plan;
  // Two row tiles to a workgroup halve the reads of the cache, one makes for more
  // and lighter workgroups: two once their workgroups and splits of 1024 keys fill
  // the GPU (96 rows, 8 heads x 4 sequences over 4000 keys: 34.9 us with two, 44.6
  // with one; 32 rows, 8 x 8 over 480: 13.7 and 11.5).  The sums of two fit beside
  // the keys and values of 256 bytes a position.
  const long long units2 = pairs * ((tiles + 1) / 2);
  plan.row_tiles = tiles >= 2 && bytes <= 256 && units2 * p.max_len_k >= 256 * 1024 ? 2 : 1;
  plan.row_blocks = (tiles + plan.row_tiles - 1) / plan.row_tiles;
  const long long units = pairs * plan.row_blocks;
  // More workgroups than CUs: of four waves, of which two or three fit a CU, so that
  // one's beginning and end hide behind the others (16 rows, 512 workgroups over 480
  // keys: 27.7 us, 33.2 of eight; 128 rows, 1536 over 900: 76.9 and 100.7; 248 rows of
  // 64 dimensions, 1056 over 54: 15.0 and 29.4; 64 workgroups over 480: 14.4 and 11.5).
  // Two waves gain where keys are few (11.4 there) and lose elsewhere (86.1 at 900
  // keys, 108.4 for 86.2 at 3500).
  plan.waves = bytes > 512 || units > 256 ? 4 : 8;
  // The splits of workgroups of so many waves: up to a workgroup a CU, of half a turn's
  // keys at least, where they save two and a half turns: partials, arrival and fold
  // cost about as much (two splits of 480 keys 12.9 us, unsplit 11.5; 1216 keys of 512
  // bytes: four 14.6, unsplit 19.4).
  const int by_units = (int)(256 / (units < 1 ? 1 : units));
  auto splits = [&](int waves) {
    const int turn = waves * (bytes > 256 || p.dtype == ASRATTN_F32 ? 16 : 32);  // keys a workgroup takes at once
    // A turn takes about 1.2 us and a split costs the fold 0.13: the sum of both is least
    // at about the root of eight times the turns (6 rows over 3000 float32 keys of
    // 64: 14.4 us with 42 splits, 10.4 with 14, 14.9 with 4; 2 rows over 4000: 13.5
    // with 32, 10.8 with 11; 16000: 21.8 with 32, 21.1 with 22).
    int most = 1;
    while (most < 64 && (long long)(most + 1) * (most + 1) * turn <= 8LL * p.max_len_k) ++most;
    // The workgroups of a range of keys share an XCD of 32 CUs: no more ranges than
    // whole ones fit (168 rows in 6 blocks, 6 pairs over 10000 keys: 43.8 us with 7
    // splits, 36 workgroups on two XCDs, 29.1 with 6).
    if (plan.row_blocks > 1) {
      const long long whole = 32 / plan.row_blocks * 8 / (pairs < 1 ? 1 : pairs);
      most = most < whole ? most : (int)whole;
    }
    const int by_keys = p.max_len_k / (turn / 2);
    most = most < by_units ? most : by_units;
    most = most < by_keys ? most : by_keys;
    return most > 1 && (long long)p.max_len_k * (most - 1) * 2 >= 5LL * turn * most ? most : 1;
  };
  plan.splits = splits(plan.waves);
  // Rows few enough that their fold costs little are split further, over workgroups
  // of four waves with half the turn, where CUs are left (8 kv heads of 128 in bf16
  // over 1800 keys, eight and four waves: 2 rows 9.5 and 8.9 us, 4 rows 9.6 and 9.3, 8
  // rows 10.0 and 9.8, 12 rows 10.4 and 11.7; over 4000 keys 8 rows 11.5 and 11.5, 12
  // rows 11.8 and 13.4; 2 rows over 16000, all CUs either way, 21.1 and 21.5.  6 heads
  // of 64 in float32 over 440 keys gain up to 16 rows: 8.7 and 8.3).
  if (plan.splits > 1 && plan.waves == 8 && rows <= 4) {
    const int more = splits(4);
    if (more > plan.splits && more < by_units) {
      plan.waves = 4;
      plan.splits = more;
    }
  }
  // One workgroup folds 128 KB of partials in about the time of a launch (65511
  // keys, 262 KB: 67.3 us with a launch, 69.0 without; 64 KB: 16.4 and 15.0).
  const long long held = rows < plan.row_tiles * 16 ? rows : plan.row_tiles * 16;
  plan.fold_apart = plan.splits * held * p.head_dim * 4 > 131072;
  return plan;
}

hipError_t launch_tree(const asrlayer_tree_params& p, const TreePlan& plan, float* ws_o, float* ws_ml,
                       unsigned long long* ws_arrive, hipStream_t stream) {
  TreeArgs a;
  a.p = p;
  a.page_shift = 0;
  while (p.block_table != nullptr && (1 << a.page_shift) < p.page_size) ++a.page_shift;
  a.rows = p.tokens * (p.heads_q / p.heads_kv);
  a.group_inv = 1.f / (float)(p.heads_q / p.heads_kv);
  a.row_blocks = plan.row_blocks;
  a.splits = plan.splits;
  const int64_t per = 4;
  a.out_vectors = reinterpret_cast<uintptr_t>(p.out) % (per * (p.dtype == ASRATTN_BF16 ? 2 : 4)) == 0 &&
                  p.o_batch_stride % per == 0 && p.o_token_stride % per == 0 && p.o_head_stride % per == 0;
  a.c = p.scale * kLog2e;
  a.ws_o = ws_o;
  a.ws_ml = ws_ml;
  a.ws_arrive = ws_arrive;
  a.tag = plan.splits > 1 ? launch_tag() : 0;
  a.fold_apart = plan.splits > 1 && plan.fold_apart;
  hipError_t err = p.dtype == ASRATTN_BF16 ? launch_typed<bf16_raw>(a, plan, stream)
                                           : launch_typed<float>(a, plan, stream);
  if (err != hipSuccess || !a.fold_apart) return err;
  const int block_rows = plan.row_tiles * 16;
  const int most = block_rows < a.rows ? block_rows : a.rows;
  const dim3 grid(most, p.batch * p.heads_kv * plan.row_blocks, (p.head_dim + 127) / 128);
  if (p.dtype == ASRATTN_BF16)
    hipLaunchKernelGGL((tree_fold_kernel<bf16_raw>), grid, dim3(256), 0, stream, a, block_rows);
  else
    hipLaunchKernelGGL((tree_fold_kernel<float>), grid, dim3(256), 0, stream, a, block_rows);
  return hipGetLastError();
}

}  // namespace asrattn
