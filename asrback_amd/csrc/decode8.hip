// A decoder step's attention over a cache of 8-bit keys and values
// (asrlayer_decode8).
//
// One query per sequence: g query heads share a kv head's n keys, each of which is
// read once, 2 (head_dim + 4) bytes with its value and scales, for 4 g head_dim
// operations.  Bound by reading the cache, once the 8-bit values become operands
// cheaply enough:
//
//   * A whole number up to 127 is exact in bf16, so scores and outputs are bf16
//     matrix products of the stored numbers, and the scales enter beside them: a key's
//     multiplies its scores, a value's its weights.  The conversion, three vector
//     instructions for two numbers, is most of the arithmetic, and is shared by up to 16 query
//     heads.  bf16 queries enter as they are and float32 ones as three bf16 that sum to
//     them; every product is exact.  The weights times the values' scales enter as two
//     bf16 (three in float32): 2^-17 (2^-24) of each is lost.
//   * Scores come out transposed, S^T = K Q^T: a lane holds four keys' scores of one
//     head for each 16 keys, so a head's softmax state is a scalar per lane and the
//     weights are already the operand of O^T = V^T P^T.
//   * A wave takes tiles of 32 keys.  A lane of V^T's operand needs eight keys of one
//     dimension: it loads the same piece of eight values' rows, and a conversion
//     picks its byte, so nothing changes lanes.  A lane of K's operand holds 16
//     consecutive dimensions of one key, two products' worth.
//   * The next tile loads while this one is computed; the 64 scales of a tile are one
//     load, spread over the lanes through the wave's own LDS.
//
// Waves merge in LDS at the end; splits of the keys leave partials in the workspace,
// and the split that arrives last folds them (decode_kernels.hpp describes the arrival
// words).  Maxima, sums and outputs are float32 until the one rounding at the end.
#include "common.hpp"
#include "kernels.hpp"
#include "row_ops.hpp"

namespace asrattn {
namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2_t __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4_t __attribute__((ext_vector_type(4)));

// Cache policy of device scope (sc1).
constexpr int kDeviceScope = 16;
// Offset of a load that is to return zeros.
constexpr uint32_t kNowhere = 0x7ff00000u;
constexpr int kKeys = 32;  // of a tile

struct Decode8Args {
  asrlayer_decode8_params p;
  int page_shift, head_tiles, splits;
  int tile_heads;  // query heads of a tile, at most 16
  float c;         // scale * log2(e)
  float* ws_o;     // [unit][split][tile_heads][head_dim]
  float* ws_ml;    // [unit][split][tile_heads][2]
  unsigned long long* ws_arrive;  // [unit]
  unsigned long long tag;
};

template <typename T, int HD>
struct Decode8Shape {
  static constexpr int kQP = sizeof(T) == 2 ? 1 : 3;  // bf16 parts of a query
  static constexpr int kWP = sizeof(T) == 2 ? 2 : 3;  // of a weight
  static constexpr int kKP = HD / 64;                 // a lane's 16-byte pieces of a key
  static constexpr int kVB = HD / 16;                 // bytes of a lane's piece of a value: 16-row tiles of O^T
  static constexpr int kVD = kVB / 4;                 // dwords of it
  static constexpr int kDC = 64;                      // dimensions merged at a time
};

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
  for (int e = 0; e < 4; ++e) Elem<T>::store1(op + e, sum == 0.f ? 0.f : x[e] / sum);
}

template <typename T, int HD, int W, bool PAGED>
__global__ __launch_bounds__(64 * W) void decode8_kernel(const Decode8Args a) {
  using S = Decode8Shape<T, HD>;
  constexpr int kQP = S::kQP, kWP = S::kWP, kKP = S::kKP, kVB = S::kVB, kVD = S::kVD, kDC = S::kDC;
  const asrlayer_decode8_params& p = a.p;
  const asrlayer_cache8& c = p.cache;
  const int split = blockIdx.x, b = blockIdx.z;
  const int hkv = blockIdx.y / a.head_tiles, ht = blockIdx.y % a.head_tiles;
  const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int group = p.heads_q / c.heads_kv;
  const int head0 = hkv * group + ht * 16, held = min(16, group - ht * 16);
  const int64_t unit = ((int64_t)b * c.heads_kv + hkv) * a.head_tiles + ht;
  const bool split_keys = a.splits > 1;
  unsigned long long* const arrive = a.ws_arrive + unit;
  unsigned long long arrive_old = 0;
  if (split_keys && threadIdx.x == 0)
    arrive_old = __hip_atomic_load(arrive, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);

  __shared__ __attribute__((aligned(16))) float sm_o[W][16][kDC + 4];
  __shared__ float sm_m[W][16], sm_l[W][16];
  __shared__ __attribute__((aligned(16))) float sm_scale[W][64];
  __shared__ int sm_last;

  // The positions: from a multiple of a tile on.
  int n = c.max_len;
  if (p.lengths != nullptr) {
    const int64_t have = p.lengths64 ? load_uniform(static_cast<const int64_t*>(p.lengths) + b)
                                     : (int64_t)load_uniform(static_cast<const int32_t*>(p.lengths) + b);
    n = have < 0 ? 0 : have < n ? (int)have : n;
  }
  n = __builtin_amdgcn_readfirstlane(n);
  const int first = p.window > 0 && n > p.window ? n - p.window : 0;
  const int tile0 = first / kKeys, tiles = n / kKeys + (n % kKeys != 0) - tile0;
  const int per = (tiles + a.splits - 1) / a.splits;
  const int t0 = tile0 + min(tiles, split * per), t1 = min(tile0 + tiles, t0 + per);

  // The lane's pieces of its head (heads past the last repeat it).
  uint4 q[kQP][2 * kKP];
  {
    const T* qp = static_cast<const T*>(p.q) + (int64_t)b * p.q_batch_stride +
                  (int64_t)(head0 + min(i, held - 1)) * p.q_head_stride;
#pragma unroll
    for (int u = 0; u < 2 * kKP; ++u) {
      const T* at = qp + 64 * (u / 2) + 16 * g + 8 * (u % 2);
      if constexpr (sizeof(T) == 2) {
        q[0][u] = *reinterpret_cast<const uint4*>(at);
      } else {
        float x[8];
        Elem<float>::load16(at, x);
        Elem<float>::load16(at + 4, x + 4);
#pragma unroll
        for (int part = 0; part < kQP; ++part)
          q[part][u] = make_uint4(take_part(x[0], x[1]), take_part(x[2], x[3]), take_part(x[4], x[5]),
                                  take_part(x[6], x[7]));
      }
    }
  }

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
  const uint32_t kstep = (uint32_t)c.k_token_stride, vstep = (uint32_t)c.v_token_stride;
  struct Pages {
    int half[2];
  };
  auto pages_of = [&](int t) -> Pages { return {{page_of(t, 0), page_of(t, 1)}}; };
  auto load_keys = [&](int t, const Pages& e) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const Half x = half_of(t, h, e.half[h]);
      keys[h] = x.keys;
      const __amdgpu_buffer_rsrc_t rsrc = rsrc_of(x, false);
      const uint32_t off = i < x.keys ? (uint32_t)i * kstep + 16 * g : kNowhere;
#pragma unroll
      for (int u = 0; u < kKP; ++u) k[h][u] = buffer_load16(rsrc, off + 64 * u);
    }
    // The tile's scales.
    const int idx = lane & 15;
    const Half x0 = half_of(t, 0, e.half[0]), x1 = half_of(t, 1, e.half[1]);
    const bool second = (lane & 16) != 0, values = lane >= 32;
    const int64_t entry = second ? x1.entry : x0.entry, at = second ? x1.at : x0.at;
    const bool held_key = idx < (second ? x1.keys : x0.keys) && t * kKeys + (lane & 31) >= first;
    const float* ptr = static_cast<const float*>(values ? c.v_scales : c.k_scales);
    const int64_t off = entry * (values ? c.vs_batch_stride : c.ks_batch_stride) +
                        hkv * (values ? c.vs_head_stride : c.ks_head_stride) + at + idx;
    scale = ptr[held_key ? off : 0];
    scale = held_key ? scale : 0.f;
  };
  auto load_values = [&](int t, const Pages& e) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const Half x = half_of(t, h, e.half[h]);
      const __amdgpu_buffer_rsrc_t rsrc = rsrc_of(x, true);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int j = 4 * g + r;
        const uint32_t off = j < x.keys ? (uint32_t)j * vstep + i * kVB : kNowhere;
        if constexpr (kVD == 4) {
          const u32x4_t w = __builtin_amdgcn_raw_buffer_load_b128(rsrc, off, 0, 0);
#pragma unroll
          for (int d = 0; d < 4; ++d) v[h][r][d % kVD] = w[d];
        } else if constexpr (kVD == 2) {
          const u32x2_t w = __builtin_amdgcn_raw_buffer_load_b64(rsrc, off, 0, 0);
          v[h][r][0] = w[0];
          v[h][r][kVD - 1] = w[1];
        } else {
          v[h][r][0] = __builtin_amdgcn_raw_buffer_load_b32(rsrc, off, 0, 0);
        }
      }
    }
  };

  f32x4_t o[kVB];
  float m = kNegInf, l = 0.f;  // l: the lane's own keys only
#pragma unroll
  for (int e = 0; e < kVB; ++e) o[e] = f32x4_t{0.f, 0.f, 0.f, 0.f};

  int t = t0 + wave;
  if (t < t1) {
    Pages next;
    {
      const Pages now = pages_of(t);
      next = pages_of(t + W);
      load_keys(t, now);
      load_values(t, now);
    }
    while (t < t1) {
      sm_scale[wave][lane] = scale;
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
      __builtin_amdgcn_wave_barrier();
      f32x4_t s[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        s[h] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int u = 0; u < kKP; ++u) {
          const uint4 raw = k[h][u];
          const uint2 w0 = widen(raw.x), w1 = widen(raw.y), w2 = widen(raw.z), w3 = widen(raw.w);
          const uint4 lo = make_uint4(w0.x, w0.y, w1.x, w1.y), hi = make_uint4(w2.x, w2.y, w3.x, w3.y);
#pragma unroll
          for (int part = kQP - 1; part >= 0; --part) {
            s[h] = mfma_bf16(lo, q[part][2 * u], s[h]);
            s[h] = mfma_bf16(hi, q[part][2 * u + 1], s[h]);
          }
        }
      }
      const int pos = t * kKeys + 4 * g;
      float x[2][4], vs[2][4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float4 ks = *reinterpret_cast<const float4*>(&sm_scale[wave][16 * h + 4 * g]);
        const float4 w = *reinterpret_cast<const float4*>(&sm_scale[wave][32 + 16 * h + 4 * g]);
        vs[h][0] = w.x, vs[h][1] = w.y, vs[h][2] = w.z, vs[h][3] = w.w;
        x[h][0] = s[h][0] * (ks.x * a.c), x[h][1] = s[h][1] * (ks.y * a.c);
        x[h][2] = s[h][2] * (ks.z * a.c), x[h][3] = s[h][3] * (ks.w * a.c);
      }
      if (keys[0] < 16 || keys[1] < 16 || t * kKeys < first) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (4 * g + r >= keys[h] || pos + 16 * h + r < first) x[h][r] = kNegInf;
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
      __builtin_amdgcn_wave_barrier();
      load_keys(t + W, next);

      float top = kNegInf;
#pragma unroll
      for (int h = 0; h < 2; ++h) top = fmaxf(top, fmaxf(fmaxf(x[h][0], x[h][1]), fmaxf(x[h][2], x[h][3])));
      const float mn = fmaxf(m, row_max(top));
      const float mu = mn == kNegInf ? 0.f : mn;
      if (!__all(mn == m)) {
        const float alpha = fast_exp2(m - mu);
        l *= alpha;
#pragma unroll
        for (int e = 0; e < kVB; ++e) o[e] *= alpha;
      }
      m = mn;
      uint32_t w[kWP][4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float y[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float e = fast_exp2(x[h][r] - mu);
          l += e;
          y[r] = e * vs[h][r];
        }
#pragma unroll
        for (int part = 0; part < kWP; ++part) {
          w[part][2 * h] = part == kWP - 1 ? pack_bf16x2(y[0], y[1]) : take_part(y[0], y[1]);
          w[part][2 * h + 1] = part == kWP - 1 ? pack_bf16x2(y[2], y[3]) : take_part(y[2], y[3]);
        }
      }
      // O^T += V^T P^T
#pragma unroll
      for (int d = 0; d < kVD; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint4 rows;
          rows.x = high_halves(byte_of(v[0][0][d], e), byte_of(v[0][1][d], e));
          rows.y = high_halves(byte_of(v[0][2][d], e), byte_of(v[0][3][d], e));
          rows.z = high_halves(byte_of(v[1][0][d], e), byte_of(v[1][1][d], e));
          rows.w = high_halves(byte_of(v[1][2][d], e), byte_of(v[1][3][d], e));
#pragma unroll
          for (int part = kWP - 1; part >= 0; --part)
            o[4 * d + e] = mfma_bf16(rows, make_uint4(w[part][0], w[part][1], w[part][2], w[part][3]), o[4 * d + e]);
        }
      load_values(t + W, next);
      t += W;
      next = pages_of(t + W);
    }
  }
  // Tag the unit's arrival word.
  if (split_keys && threadIdx.x == 0 && (arrive_old >> 16) != a.tag)
    __hip_atomic_compare_exchange_strong(arrive, &arrive_old, a.tag << 16, __ATOMIC_RELAXED, __ATOMIC_RELAXED,
                                         __HIP_MEMORY_SCOPE_AGENT);

  // Merge the waves, kDC dimensions at a time: accumulator r of tile e is dimension
  // (4 g + r) kVB + e.
  const float sum_keys = row_sum(l);
  if (g == 0) {
    sm_m[wave][i] = m;
    sm_l[wave][i] = sum_keys;
  }
  const int64_t unit_rows = unit * a.splits * a.tile_heads;
  const int64_t split_row = unit_rows + (int64_t)split * a.tile_heads;
  for (int dc = 0; dc < HD; dc += kDC) {
    __syncthreads();
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int d = (4 * g + r) * kVB - dc;
      if (d >= 0 && d < kDC && i < held) {
#pragma unroll
        for (int e = 0; e < kVB; e += 4)
          *reinterpret_cast<float4*>(&sm_o[wave][i][d + e]) = make_float4(o[e][r], o[e + 1][r], o[e + 2][r], o[e + 3][r]);
      }
    }
    __syncthreads();
    for (int it = threadIdx.x; it < held * (kDC / 4); it += 64 * W) {
      const int row = it / (kDC / 4), d = it % (kDC / 4) * 4;
      float mx = kNegInf;
#pragma unroll
      for (int u = 0; u < W; ++u) mx = fmaxf(mx, sm_m[u][row]);
      const float mu = mx == kNegInf ? 0.f : mx;
      float sum = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int u = 0; u < W; ++u) {
        const float wt = fast_exp2(sm_m[u][row] - mu);
        sum = fmaf(sm_l[u][row], wt, sum);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = fmaf(sm_o[u][row][d + e], wt, x[e]);
      }
      if (split_keys) {
        float* po = a.ws_o + (split_row + row) * HD + dc + d;
        store_shared2(po, x[0], x[1]);
        store_shared2(po + 2, x[2], x[3]);
        if (dc + d == 0) store_shared2(a.ws_ml + (split_row + row) * 2, mx, sum);
      } else {
        store_head<T>(a, b, head0 + row, dc + d, x, sum);
      }
    }
  }
  if (!split_keys) return;

  // Arrive once every wave's partial stores are in memory.
  __builtin_amdgcn_s_waitcnt(kWaitVmem);
  __syncthreads();
  if (threadIdx.x == 0) {
    const unsigned long long before = __hip_atomic_fetch_add(arrive, 1ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    sm_last = (int)(before & 0xffffull) == a.splits - 1;
    if (sm_last) __hip_atomic_store(arrive, 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!sm_last) return;  // uniform over the workgroup

  for (int it = threadIdx.x; it < held * (HD / 4); it += 64 * W) {
    const int row = it / (HD / 4), d = it % (HD / 4) * 4;
    float mx = kNegInf, sum = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
    constexpr int kBatch = 8;  // splits a round trip
    for (int s0 = 0; s0 < a.splits; s0 += kBatch) {
      float pm[kBatch], pl[kBatch], px[kBatch][4];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int64_t at = unit_rows + (int64_t)min(s0 + u, a.splits - 1) * a.tile_heads + row;
        load_shared2(a.ws_ml + at * 2, pm[u], pl[u]);
        load_shared2(a.ws_o + at * HD + d, px[u][0], px[u][1]);
        load_shared2(a.ws_o + at * HD + d + 2, px[u][2], px[u][3]);
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
        if (s0 + u >= a.splits) continue;
        const float wt = fast_exp2(pm[u] - mu);
        sum = fmaf(pl[u], wt, sum);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = fmaf(px[u][e], wt, x[e]);
      }
    }
    store_head<T>(a, b, head0 + row, d, x, sum);
  }
}

template <typename T, int HD, int W>
hipError_t launch_waves(const Decode8Args& a, hipStream_t stream) {
  const dim3 grid(a.splits, a.p.cache.heads_kv * a.head_tiles, a.p.cache.batch), block(64 * W);
  if (a.p.cache.block_table != nullptr)
    hipLaunchKernelGGL((decode8_kernel<T, HD, W, true>), grid, block, 0, stream, a);
  else
    hipLaunchKernelGGL((decode8_kernel<T, HD, W, false>), grid, block, 0, stream, a);
  return hipGetLastError();
}

template <typename T>
hipError_t launch_typed(const Decode8Args& a, int waves, hipStream_t stream) {
  switch (a.p.cache.head_dim) {
    case 64: return waves == 8 ? launch_waves<T, 64, 8>(a, stream) : launch_waves<T, 64, 4>(a, stream);
    case 128: return waves == 8 ? launch_waves<T, 128, 8>(a, stream) : launch_waves<T, 128, 4>(a, stream);
    default: return waves == 8 ? launch_waves<T, 256, 8>(a, stream) : launch_waves<T, 256, 4>(a, stream);
  }
}

}  // namespace

Decode8Plan decode8_plan(const asrlayer_decode8_params& p) {
  const asrlayer_cache8& c = p.cache;
  Decode8Plan plan;
  const int group = p.heads_q / c.heads_kv;
  plan.head_tiles = (group + 15) / 16;
  const long long units = (long long)c.batch * c.heads_kv * plan.head_tiles;
  const int span = p.window > 0 && p.window < c.max_len ? p.window : c.max_len;
  plan.waves = units > 256 ? 4 : 8;
  // At most a workgroup a CU, of a tile a wave at least.
  const int by_units = (int)(256 / (units < 1 ? 1 : units));
  const int by_keys = span / (plan.waves * kKeys);
  plan.splits = by_units < by_keys ? by_units : by_keys;
  plan.splits = plan.splits < 1 ? 1 : plan.splits > 64 ? 64 : plan.splits;
  return plan;
}

hipError_t launch_decode8(const asrlayer_decode8_params& p, const Decode8Plan& plan, float* ws_o, float* ws_ml,
                          unsigned long long* ws_arrive, hipStream_t stream) {
  Decode8Args a;
  a.p = p;
  a.page_shift = 0;
  while (p.cache.block_table != nullptr && (1 << a.page_shift) < p.cache.page_size) ++a.page_shift;
  a.head_tiles = plan.head_tiles;
  a.splits = plan.splits;
  const int group = p.heads_q / p.cache.heads_kv;
  a.tile_heads = group < 16 ? group : 16;
  a.c = p.scale * kLog2e;
  a.ws_o = ws_o;
  a.ws_ml = ws_ml;
  a.ws_arrive = ws_arrive;
  a.tag = plan.splits > 1 ? launch_tag() : 0;
  return p.dtype == ASRATTN_BF16 ? launch_typed<bf16_raw>(a, plan.waves, stream)
                                 : launch_typed<float>(a, plan.waves, stream);
}

}  // namespace asrattn
