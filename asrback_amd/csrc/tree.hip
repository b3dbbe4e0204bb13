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
//   * A workgroup takes up to 64 rows of one (sequence, kv head) and a range of
//     its keys; its waves take tiles of keys in turn, each wave with all rows
//     and a softmax state of its own.  Keys and values go from memory to the
//     registers of the one wave that uses them: no LDS, no barriers, and each
//     wave loads its next tile's keys while it weighs the values, its next
//     values while it scores the keys.
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
// Weights are rounded to bf16 for the product with bf16 values (half a step,
// 2^-9 of each), sums, maxima and outputs are float32 until the one rounding at
// the end; float32 inputs stay float32 throughout.
#include "common.hpp"
#include "kernels.hpp"
#include "row_ops.hpp"

namespace asrattn {
namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2_t __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4_t __attribute__((ext_vector_type(4)));

struct TreeArgs {
  asrlayer_tree_params p;
  int page_shift, rows, row_blocks, splits;
  float c;  // scale * log2(e)
  float* ws_o;   // [unit][split][16 row_tiles][head_dim]
  float* ws_ml;  // [unit][split][16 row_tiles][2]
  unsigned long long* ws_arrive;  // [unit]
  unsigned long long tag;
};

template <typename T, int HD>
struct TreeShape {
  static constexpr int kES = (int)sizeof(T);
  static constexpr int kSub = kES == 2 ? 2 : 1;     // 16-key parts of a tile
  static constexpr int kKeys = 16 * kSub;           // keys of a tile
  static constexpr int kKV = HD * kES / 64;         // a lane's 16-byte pieces of a key part
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

// A dword of T with its infinities and NaN replaced by zeros.
template <typename T>
__device__ __forceinline__ uint32_t finite_part(uint32_t x) {
  if constexpr (sizeof(T) == 4) return (x & 0x7f800000u) == 0x7f800000u ? 0u : x;
  const uint32_t lo = (x & 0x7f80u) == 0x7f80u ? 0u : x & 0xffffu;
  return (x & 0x7f800000u) == 0x7f800000u ? lo : (x & 0xffff0000u) | lo;
}

// Offset of a load that is to return zeros.
constexpr uint32_t kNowhere = 0x7ff00000u;

// RT: 16-row tiles of the workgroup; W: its waves.
template <typename T, int HD, int RT, int W, bool PAGED>
__global__ __launch_bounds__(64 * W) void tree_kernel(const TreeArgs a) {
  using S = TreeShape<T, HD>;
  constexpr int kSub = S::kSub, kKeys = S::kKeys, kKV = S::kKV, kVD = S::kVD, kEV = S::kEV, kNC = S::kNC;
  constexpr int kES = S::kES, kDC = S::kDC;
  const asrlayer_tree_params& p = a.p;

  const int split = blockIdx.x;
  const int hkv = blockIdx.y / a.row_blocks, rb = blockIdx.y % a.row_blocks;
  const int b = blockIdx.z;
  const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int group = p.heads_q / p.heads_kv;
  const int64_t unit = ((int64_t)b * p.heads_kv + hkv) * a.row_blocks + rb;
  const bool split_keys = a.splits > 1;
  unsigned long long* const arrive = a.ws_arrive + unit;
  unsigned long long arrive_old = 0;
  if (split_keys && threadIdx.x == 0)
    arrive_old = __hip_atomic_load(arrive, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);

  // The lane's query rows (rows past the last repeat it), 16 bytes of each 64.
  uint4 q[RT][kKV];
  uint64_t mask[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int m = min((rb * RT + rt) * 16 + i, a.rows - 1);
    const int t = m / group, h = hkv * group + m % group;
    const char* qp = static_cast<const char*>(p.q) +
                     ((int64_t)b * p.q_batch_stride + (int64_t)t * p.q_token_stride + (int64_t)h * p.q_head_stride) * kES;
#pragma unroll
    for (int c = 0; c < kKV; ++c) q[rt][c] = *reinterpret_cast<const uint4*>(qp + c * 64 + g * 16);
    mask[rt] = (uint64_t)p.masks[(int64_t)b * p.masks_batch_stride + t];
  }

  int64_t n64 = p.max_len_k;
  if (p.lengths != nullptr)
    n64 = p.lengths64 ? load_uniform(static_cast<const int64_t*>(p.lengths) + b)
                      : (int64_t)load_uniform(static_cast<const int32_t*>(p.lengths) + b);
  const int n = (int)min(max(n64, (int64_t)0), (int64_t)p.max_len_k);
  const int cache_tiles = n / kKeys + (n % kKeys != 0);
  const int tiles = cache_tiles + (p.tokens + kKeys - 1) / kKeys;
  const int per = (tiles + a.splits - 1) / a.splits;
  const int t0 = min(tiles, split * per), t1 = min(tiles, t0 + per);

  const char* const kbase = static_cast<const char*>(p.k) +
                            ((PAGED ? 0 : (int64_t)b * p.k_batch_stride) + (int64_t)hkv * p.k_head_stride) * kES;
  const char* const vbase = static_cast<const char*>(p.v) +
                            ((PAGED ? 0 : (int64_t)b * p.v_batch_stride) + (int64_t)hkv * p.v_head_stride) * kES;
  const char* const kdbase = static_cast<const char*>(p.k_draft) +
                             ((int64_t)b * p.kd_batch_stride + (int64_t)hkv * p.kd_head_stride) * kES;
  const char* const vdbase = static_cast<const char*>(p.v_draft) +
                             ((int64_t)b * p.vd_batch_stride + (int64_t)hkv * p.vd_head_stride) * kES;

  // Part `s` of tile t: its first key's address and its keys (0: none, and
  // nothing is read).  With PAGED a part lies in one page.
  struct Part {
    const char* base;
    int64_t stride;
    int keys;
  };
  auto part_of = [&](int t, int s, bool values) -> Part {
    if (t >= cache_tiles) {
      const int j = (t - cache_tiles) * kKeys + s * 16;
      const int64_t stride = (values ? p.vd_token_stride : p.kd_token_stride) * kES;
      return {(values ? vdbase : kdbase) + j * stride, stride, min(max(p.tokens - j, 0), 16)};
    }
    const int j = t * kKeys + s * 16;
    const int64_t stride = (values ? p.v_token_stride : p.k_token_stride) * kES;
    int keys = min(max(n - j, 0), 16);
    const char* base = values ? vbase : kbase;
    if constexpr (PAGED) {
      int page = -1;
      const int pi = j >> a.page_shift;
      if (keys > 0 && pi < p.bt_stride) {
        const int e = load_uniform(p.block_table + (int64_t)b * p.bt_stride + pi);
        page = e >= 0 && e < p.num_pages ? e : -1;
      }
      if (page < 0) return {base, stride, 0};
      return {base + (page * (values ? p.v_page_stride : p.k_page_stride)) * kES + (j - (pi << a.page_shift)) * stride,
              stride, keys};
    }
    return {base + j * stride, stride, keys};
  };
  auto resource = [&](const Part& x) {
    return buffer_rsrc(x.base, x.keys > 0 ? (uint32_t)((x.keys - 1) * x.stride) + HD * kES : 0u);
  };

  uint4 k[kSub][kKV];
  uint32_t v[kSub][4][kNC][kVD];
  int keys[kSub], next_keys[kSub];
  auto load_keys = [&](int t, int* held) {
#pragma unroll
    for (int s = 0; s < kSub; ++s) {
      const Part x = part_of(t, s, false);
      const __amdgpu_buffer_rsrc_t rs = resource(x);
      held[s] = x.keys;
      const uint32_t off = i < x.keys ? (uint32_t)i * (uint32_t)x.stride + g * 16 : kNowhere;
#pragma unroll
      for (int c = 0; c < kKV; ++c) k[s][c] = buffer_load16(rs, off + c * 64);
    }
  };
  auto load_values = [&](int t) {
#pragma unroll
    for (int s = 0; s < kSub; ++s) {
      const Part x = part_of(t, s, true);
      const __amdgpu_buffer_rsrc_t rs = resource(x);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int j = 4 * g + r;
        const uint32_t off = j < x.keys ? (uint32_t)j * (uint32_t)x.stride + i * S::kVB : kNowhere;
#pragma unroll
        for (int c = 0; c < kNC; ++c) load_piece<S::kVB>(rs, off + c * 16 * S::kVB, v[s][r][c]);
      }
    }
  };

  int t = t0 + wave;
  if (t < t1) {
    load_keys(t, keys);
    load_values(t);
  }
  // Tag the unit's arrival word, whose load was issued first of all; the answer
  // is not waited for.
  if (split_keys && threadIdx.x == 0 && (arrive_old >> 16) != a.tag)
    __hip_atomic_compare_exchange_strong(arrive, &arrive_old, a.tag << 16, __ATOMIC_RELAXED, __ATOMIC_RELAXED,
                                         __HIP_MEMORY_SCOPE_AGENT);

  f32x4_t o[RT][S::kTiles];
  float m[RT], l[RT];  // l: the lane's own keys only
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    m[rt] = kNegInf;
    l[rt] = 0.f;
#pragma unroll
    for (int e = 0; e < S::kTiles; ++e) o[rt][e] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }

  while (t < t1) {
    const int next = t + W;
    const bool drafted = t >= cache_tiles;
    const int draft0 = (t - cache_tiles) * kKeys;
    f32x4_t s[RT][kSub];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int h = 0; h < kSub; ++h) {
        s[rt][h] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < kKV; ++c) s[rt][h] = score_piece<T>(k[h][c], q[rt][c], s[rt][h]);
      }
    if (next < t1) load_keys(next, next_keys);

    // Keys that a row does not see: past a part's keys, or no ancestor's.
    bool whole = !drafted;
#pragma unroll
    for (int h = 0; h < kSub; ++h) whole = whole && keys[h] == 16;
    if (!whole) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int h = 0; h < kSub; ++h) {
          const uint32_t tree = (uint32_t)(mask[rt] >> (drafted ? draft0 + h * 16 + 4 * g : 0));
          const uint32_t seen = drafted ? tree : 0xfu;
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (4 * g + r >= keys[h] || !((seen >> r) & 1u)) s[rt][h][r] = kNegInf;
        }
    }

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

    // A drafted value that some rows must not see may be infinite or NaN, and
    // a weight of zero times it is not zero: such elements leave the product, and
    // the rows that do see them take them as they are.
    if (drafted) {
      bool bad = false;
#pragma unroll
      for (int h = 0; h < kSub; ++h)
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int c = 0; c < kNC; ++c)
#pragma unroll
            for (int d = 0; d < kVD; ++d) {
              const uint32_t x = finite_part<T>(v[h][r][c][d]);
              bad = bad || x != v[h][r][c][d];
              v[h][r][c][d] = x;
            }
      if (__any(bad)) {
        const int held = min(p.tokens - draft0, kKeys);
        for (int j = 0; j < held; ++j) {
          const T* row = reinterpret_cast<const T*>(vdbase) + (int64_t)(draft0 + j) * p.vd_token_stride;
#pragma unroll
          for (int c = 0; c < kNC; ++c)
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
              for (int e = 0; e < kEV; ++e) {
                const float x = Elem<T>::load1(row + (c * 16 + g * 4 + r) * kEV + e);
                const float y = (__float_as_uint(x) & 0x7f800000u) == 0x7f800000u ? x : 0.f;
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
                  o[rt][c * kEV + e][r] += (mask[rt] >> (draft0 + j)) & 1u ? y : 0.f;
              }
        }
      }
    }

    // O^T += V^T P^T
#pragma unroll
    for (int c = 0; c < kNC; ++c) {
      if constexpr (kES == 2) {
#pragma unroll
        for (int d = 0; d < kVD; ++d) {
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const uint32_t sel = half ? 0x07060302u : 0x05040100u;
            uint4 vt;
            vt.x = __builtin_amdgcn_perm(v[0][1][c][d], v[0][0][c][d], sel);
            vt.y = __builtin_amdgcn_perm(v[0][3][c][d], v[0][2][c][d], sel);
            vt.z = __builtin_amdgcn_perm(v[kSub - 1][1][c][d], v[kSub - 1][0][c][d], sel);
            vt.w = __builtin_amdgcn_perm(v[kSub - 1][3][c][d], v[kSub - 1][2][c][d], sel);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
              o[rt][c * kEV + 2 * d + half] =
                  mfma_bf16(vt, make_uint4(w[rt][0], w[rt][1], w[rt][kSub * 2 - 2], w[rt][kSub * 2 - 1]),
                            o[rt][c * kEV + 2 * d + half]);
          }
        }
      } else {
#pragma unroll
        for (int d = 0; d < kVD; ++d)
#pragma unroll
          for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int r = 0; r < 4; ++r) o[rt][c * kEV + d] = mfma_f32(v[0][r][c][d], w[rt][r], o[rt][c * kEV + d]);
      }
    }
    if (next < t1) load_values(next);
#pragma unroll
    for (int h = 0; h < kSub; ++h) keys[h] = next_keys[h];
    t = next;
  }

  // Merge the waves, 16 rows and kDC dimensions at a time.
  __shared__ float sm_m[W][RT * 16], sm_l[W][RT * 16];
  __shared__ __attribute__((aligned(16))) float sm_o[W][16][kDC + 4];
  __shared__ int sm_last;
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const float sum = row_sum(l[rt]);
    if (g == 0) {
      sm_m[wave][rt * 16 + i] = mask[rt] != 0 ? m[rt] : kNegInf;
      sm_l[wave][rt * 16 + i] = mask[rt] != 0 ? sum : 0.f;
    }
  }
  constexpr int kVecs = kDC / 4;
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
    for (int dc = 0; dc < HD / kDC; ++dc) {
      __syncthreads();
      constexpr int kPieces = kDC / (16 * kEV);
#pragma unroll
      for (int c = 0; c < kPieces; ++c)
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int e = 0; e < kEV; e += 4) {
            float4 x;
            const int at = (dc * kPieces + c) * kEV + e;
            x.x = o[rt][at][r], x.y = o[rt][at + 1][r], x.z = o[rt][at + 2][r], x.w = o[rt][at + 3][r];
            if (mask[rt] == 0) x = make_float4(0.f, 0.f, 0.f, 0.f);
            *reinterpret_cast<float4*>(&sm_o[wave][i][(c * 16 + g * 4 + r) * kEV + e]) = x;
          }
      __syncthreads();
      for (int it = threadIdx.x; it < 16 * kVecs; it += 64 * W) {
        const int row = it / kVecs, d = it % kVecs * 4;
        const int mrow = (rb * RT + rt) * 16 + row;
        if (mrow >= a.rows) continue;
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
          const int64_t at = (unit * a.splits + split) * (RT * 16) + rt * 16 + row;
          float* po = a.ws_o + at * HD + dc * kDC + d;
          store_shared2(po, x[0], x[1]);
          store_shared2(po + 2, x[2], x[3]);
          if (dc == 0 && d == 0) store_shared2(a.ws_ml + at * 2, mx, sum);
        } else {
          const int tok = mrow / group, h = hkv * group + mrow % group;
          T* op = static_cast<T*>(p.out) + (int64_t)b * p.o_batch_stride + (int64_t)tok * p.o_token_stride +
                  (int64_t)h * p.o_head_stride + dc * kDC + d;
#pragma unroll
          for (int e = 0; e < 4; ++e) Elem<T>::store1(op + e, sum == 0.f ? 0.f : x[e] / sum);
        }
      }
    }
  }
  if (!split_keys) return;

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

  // Fold the splits' partials, four dimensions a thread, four splits a round trip.
  const int held = min(RT * 16, a.rows - rb * RT * 16);
  constexpr int kBatch = 4;
  for (int it = threadIdx.x; it < held * (HD / 4); it += 64 * W) {
    const int row = it / (HD / 4), d = it % (HD / 4) * 4;
    float mx = kNegInf, sum = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < a.splits; s0 += kBatch) {
      float pm[kBatch], pl[kBatch], px[kBatch][4];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int64_t at = (unit * a.splits + min(s0 + u, a.splits - 1)) * (RT * 16) + row;
        load_shared2(a.ws_ml + at * 2, pm[u], pl[u]);
        load_shared2(a.ws_o + at * HD + d, px[u][0], px[u][1]);
        load_shared2(a.ws_o + at * HD + d + 2, px[u][2], px[u][3]);
      }
      float mn = mx;
#pragma unroll
      for (int u = 0; u < kBatch; ++u) mn = fmaxf(mn, pm[u]);
      const float mu = mn == kNegInf ? 0.f : mn;
      const float w0 = fast_exp2(mx - mu);
      mx = mn;
      sum *= w0;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] *= w0;
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        if (s0 + u >= a.splits) continue;  // uniform; the surplus repeats the last split
        const float wt = fast_exp2(pm[u] - mu);
        sum = fmaf(pl[u], wt, sum);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = fmaf(px[u][e], wt, x[e]);
      }
    }
    const int mrow = rb * RT * 16 + row;
    const int tok = mrow / group, h = hkv * group + mrow % group;
    T* op = static_cast<T*>(p.out) + (int64_t)b * p.o_batch_stride + (int64_t)tok * p.o_token_stride +
            (int64_t)h * p.o_head_stride + d;
#pragma unroll
    for (int e = 0; e < 4; ++e) Elem<T>::store1(op + e, sum == 0.f ? 0.f : x[e] / sum);
  }
}

template <typename T, int HD, int RT>
hipError_t launch_rows(const TreeArgs& a, hipStream_t stream) {
  constexpr int W = 4;
  const dim3 grid(a.splits, a.p.heads_kv * a.row_blocks, a.p.batch);
  if (a.p.block_table != nullptr)
    hipLaunchKernelGGL((tree_kernel<T, HD, RT, W, true>), grid, dim3(64 * W), 0, stream, a);
  else
    hipLaunchKernelGGL((tree_kernel<T, HD, RT, W, false>), grid, dim3(64 * W), 0, stream, a);
  return hipGetLastError();
}

template <typename T, int HD>
hipError_t launch_head(const TreeArgs& a, int row_tiles, hipStream_t stream) {
  if (row_tiles == 1) return launch_rows<T, HD, 1>(a, stream);
  if (row_tiles == 2) return launch_rows<T, HD, 2>(a, stream);
  if constexpr (HD <= 128) {
    if (row_tiles == 4) return launch_rows<T, HD, 4>(a, stream);
  }
  return hipErrorInvalidValue;
}

template <typename T>
hipError_t launch_typed(const TreeArgs& a, int row_tiles, hipStream_t stream) {
  switch (a.p.head_dim) {
    case 64: return launch_head<T, 64>(a, row_tiles, stream);
    case 128: return launch_head<T, 128>(a, row_tiles, stream);
    case 256: return launch_head<T, 256>(a, row_tiles, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace

int tree_most_row_tiles(int head_dim) { return head_dim >= 256 ? 2 : 4; }

TreePlan tree_plan(const asrlayer_tree_params& p) {
  const long long rows = (long long)p.tokens * (p.heads_q / p.heads_kv);
  const int tiles = (int)((rows + 15) / 16), most = tree_most_row_tiles(p.head_dim);
  TreePlan plan;
  plan.row_tiles = tiles <= 1 ? 1 : tiles == 2 || most == 2 ? 2 : 4;
  plan.row_blocks = (tiles + plan.row_tiles - 1) / plan.row_tiles;
  // Units of work; split keys cost a partial of 4 x rows x head_dim bytes
  // written and read a split, so a split holds at least 8 keys a row.
  const long long units = (long long)p.batch * p.heads_kv * plan.row_blocks;
  const int least = plan.row_tiles * 128;
  const int by_keys = p.max_len_k / least < 1 ? 1 : p.max_len_k / least > 64 ? 64 : p.max_len_k / least;
  const int by_units = units >= 256 ? 1 : (int)(256 / (units < 1 ? 1 : units));
  plan.splits = by_keys < by_units ? by_keys : by_units;
  return plan;
}

hipError_t launch_tree(const asrlayer_tree_params& p, const TreePlan& plan, float* ws_o, float* ws_ml,
                       unsigned long long* ws_arrive, hipStream_t stream) {
  TreeArgs a;
  a.p = p;
  a.page_shift = 0;
  while (p.block_table != nullptr && (1 << a.page_shift) < p.page_size) ++a.page_shift;
  a.rows = p.tokens * (p.heads_q / p.heads_kv);
  a.row_blocks = plan.row_blocks;
  a.splits = plan.splits;
  a.c = p.scale * kLog2e;
  a.ws_o = ws_o;
  a.ws_ml = ws_ml;
  a.ws_arrive = ws_arrive;
  a.tag = plan.splits > 1 ? launch_tag() : 0;
  return p.dtype == ASRATTN_BF16 ? launch_typed<bf16_raw>(a, plan.row_tiles, stream)
                                 : launch_typed<float>(a, plan.row_tiles, stream);
}

}  // namespace asrattn
