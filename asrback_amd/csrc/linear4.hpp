// Rows through a matrix of 4-bit weights with group scales (asrlayer_linear4),
// instantiated per element type in linear4_bf16.hip and linear4_f32.hip.
//
// Up to some hundred rows the product is bound by reading the weights, half a
// byte each, and at small matrices by the launch; the work per weight has to stay
// below the time of its bytes.  So:
//
//   * The matrix lies in blocks of 16 outputs x 128 inputs, 1 KB in the order in
//     which a wave's lanes take it: a load is one 16-byte access per lane over
//     whole cache lines, and the four dwords are four matrix instructions' operand.
//   * bf16: a nibble becomes bf16 by an AND and an OR: 0x3b00 | q is 2^-16 (128 + q)
//     exactly, two elements an instruction (7 for 8 weights).  The 128 and the
//     zero point leave through the accumulator, which starts at
//     -(128 + zero) sum(x) of the group: sum x (128 + q) - (128 + zero) sum x.
//     The sums' float32 rounding is 2^-24 of values up to 143 |x|: with inputs around
//     zero some 30 times the result's own, 2^-19; with a mean the offset's part grows
//     faster than the result, whose weights are around zero (of one deviation, the
//     root mean square over one group of 128: 2^-17).  Both are far below the 2^-8 of
//     the bf16 result.
//     float32: x is split into three bf16 whose sum it is, exactly, and nibbles
//     become bf16 one by one without an offset (only the zero point leaves through
//     the accumulator): every product is exact, and three bf16 matrix instructions take
//     the place of eight float32 ones of twice the time each (16 x 1024 x 40000: 12.0 us
//     for 20.0).
//   * A group's sum comes before its scale, and up to 2^15.2 (float32: 2^12) times the
//     largest |x| passes through the accumulator: 128 inputs, values up to 143 (15) of
//     weights and of the zero point.  So that no sum overflows that the scale brings
//     back into range, sums are kept times 2^-16 (2^-12) until the end.  In bf16 that
//     is in the operand and costs nothing.  float32 x is multiplied by it on its way
//     (16 x 1024 x 40000: 12.0 us for 11.7), and what bf16 cannot hold of it is lost:
//     2^-121 of an x, so that those below 2^-97 go in with fewer bits.
//   * Outputs lie in the rows of the product and x's rows in its columns, so a
//     lane holds four outputs of one x row: a group's scales are one small load
//     for four outputs, the group's sum of x one value per lane.
//   * A workgroup's waves split the inputs, each keeping its part of x in
//     registers, and go through the workgroup's blocks of outputs with it; the
//     next block's weights load while this one's are multiplied (two blocks ahead
//     cost registers and gave 36.1 us for 34.3 at 4 x 2048 x 151936; loads past
//     the caches 33.8, but 8.0 for 7.4 at 64 x 2048 x 4096 and 13.0 for 12.2 at 64
//     x 2048 x 12288).  The waves' sums meet in LDS once a block (two buffers, one
//     barrier that leaves the loads in flight).
//   * The groups' sums of x are products with ones, on the matrix cores that idle
//     meanwhile (64 x 6144 x 2048: 9.8 us for 12.2 with additions; the zero points'
//     products there as well, as one of depth one, gave 10.1).
//   * Every wave of every turn issues the same loads and stores, absent ones with an
//     empty range: the waits count them, and a branch would set them for its shorter
//     path.  That took 41.9 us to 34.3 there.
//   * x is loaded by whole rows (neighbouring lanes in one row; a load whose lanes lie
//     in 16 rows takes four times as long in the vector cache) and changes lanes
//     through the wave's own LDS.
//
// Measured (bf16, group 128): 4 x 2048 x 151936 in 34.5 us, 4.7 TB/s of the 6.0 that
// a reading kernel reaches; 16 x 2048 x 12288 in 6.3 us and 1 x 2048 x 2048 in 3.8,
// where launching (1.8 us) and one round trip each for x and the first weights are
// most; 64 x 6144 x 2048 in 9.8 us, six turns of x through LDS after each other.
#pragma once

#include "common.hpp"
#include "kernels.hpp"
#include "row_ops.hpp"

namespace asrattn {
namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

template <typename T>
struct L4 {
  static constexpr int kXV = sizeof(T) == 2 ? 1 : 2;  // 16-byte vectors of 8 inputs
  static constexpr int kXP = sizeof(T) == 2 ? 1 : 3;  // bf16 parts of an input
  static constexpr float kOffset = sizeof(T) == 2 ? 128.f : 0.f;  // what a weight operand adds to q
  static constexpr float kUnit = sizeof(T) == 2 ? 0x1p-16f : 0x1p-12f;  // what sums are kept times
};

// 8 float32 inputs, times kUnit, as the product's operands: the sum of three bf16, each the
// leading 8 bits of what is left (24 bits: nothing is lost).
__device__ __forceinline__ void l4_parts(const float* in, uint4* x) {
  uint32_t part[3][8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    part[0][j] = __float_as_uint(in[j]);
    const float left = in[j] - __uint_as_float(part[0][j] & 0xffff0000u);
    part[1][j] = __float_as_uint(left);
    part[2][j] = __float_as_uint(left - __uint_as_float(part[1][j] & 0xffff0000u));
  }
#pragma unroll
  for (int c = 0; c < 3; ++c) {
    constexpr uint32_t kHigh = 0x07060302u;  // the high halves of two dwords
    x[c] = make_uint4(__builtin_amdgcn_perm(part[c][1], part[c][0], kHigh),
                      __builtin_amdgcn_perm(part[c][3], part[c][2], kHigh),
                      __builtin_amdgcn_perm(part[c][5], part[c][4], kHigh),
                      __builtin_amdgcn_perm(part[c][7], part[c][6], kHigh));
  }
}

// acc += (16 outputs x 32 inputs) (16 rows x 32 inputs)^T from a dword of
// weights and 8 inputs a lane.
template <typename T, int RT>
__device__ __forceinline__ void l4_step(uint32_t w, const uint4 (*x)[L4<T>::kXP], f32x4_t* acc) {
  uint4 a;
  if constexpr (sizeof(T) == 2) {
    constexpr uint32_t kWeight = 0x3b003b00u;  // 2^-16 (128 + q) in the low bits' place
    a.x = (w & 0x000f000fu) | kWeight;
    a.y = ((w >> 4) & 0x000f000fu) | kWeight;
    a.z = ((w >> 8) & 0x000f000fu) | kWeight;
    a.w = ((w >> 12) & 0x000f000fu) | kWeight;
  } else {
    const uint32_t lo = w & 0x0f0f0f0fu, hi = (w >> 4) & 0x0f0f0f0fu;
    // Nibbles 0 1 2 3 hold inputs 0 2 4 6, nibbles 4 5 6 7 inputs 1 3 5 7.
    const float q[8] = {(float)(lo & 0xffu),         (float)((lo >> 16) & 0xffu), (float)(hi & 0xffu),
                        (float)((hi >> 16) & 0xffu), (float)((lo >> 8) & 0xffu),  (float)(lo >> 24),
                        (float)((hi >> 8) & 0xffu),  (float)(hi >> 24)};
    constexpr uint32_t kHigh = 0x07060302u;  // small integers: bf16 is the high half
    a.x = __builtin_amdgcn_perm(__float_as_uint(q[1]), __float_as_uint(q[0]), kHigh);
    a.y = __builtin_amdgcn_perm(__float_as_uint(q[3]), __float_as_uint(q[2]), kHigh);
    a.z = __builtin_amdgcn_perm(__float_as_uint(q[5]), __float_as_uint(q[4]), kHigh);
    a.w = __builtin_amdgcn_perm(__float_as_uint(q[7]), __float_as_uint(q[6]), kHigh);
  }
#pragma unroll
  for (int c = L4<T>::kXP - 1; c >= 0; --c)
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
      acc[rt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                        __builtin_bit_cast(bf16x8_t, x[rt][c]), acc[rt], 0, 0, 0);
}

// Where 16-byte piece c of row r lies in a block of LPR-piece rows in LDS, so that a
// piece of 16 rows lies in 16 different groups of banks.
template <int LPR>
__device__ __forceinline__ int l4_piece(int r, int c) {
  return r * LPR + (c ^ (r & 15));
}

// The weights a wave multiplies at a time: NB blocks, their scales and zero points.
template <typename T, int NB, int MB, int GROUP>
struct L4Weights {
  static constexpr int kGroups = 128 / GROUP;
  static constexpr int kSV = kGroups * 4 * (int)sizeof(T) / 8;  // scales of a block, in 8 bytes
  uint4 w[MB][NB];
  uint2 s[MB][NB][kSV];
  uint32_t z[MB][NB][(kGroups + 1) / 2];
  float bias[MB];  // of output i
};

// Workgroups whose registers fit a CU.
template <typename T, int W, int RT, int NB, int MB, int GROUP, bool CHUNKED>
constexpr int l4_per_cu() {
  return sizeof(T) == 2 && W == 8 && (GROUP >= 64 || RT == 1) && NB <= 2 && MB == 1 && !(CHUNKED && RT == 2) ? 2 : 1;
}

// RT: 16-row tiles of x; NB: blocks of 128 inputs a wave holds at a time, MB: blocks of
// outputs it multiplies them with; GROUP: inputs of a scale; CHUNKED: more inputs than the waves hold, x following the
// weights chunk by chunk.
template <typename T, int W, int RT, int NB, int MB, int GROUP, bool CHUNKED>
__global__ __launch_bounds__(64 * W, (W / 4 * l4_per_cu<T, W, RT, NB, MB, GROUP, CHUNKED>())) void linear4_kernel(
    const asrlayer_linear4_params p, int blocks_n, int blocks_k) {
  using W4 = L4Weights<T, NB, MB, GROUP>;
  constexpr int kXV = L4<T>::kXV, kGroups = 128 / GROUP, kSteps = GROUP / 32, kSV = W4::kSV;
  constexpr float kOffset = L4<T>::kOffset;
  constexpr int kLPR = 128 * (int)sizeof(T) / 16;  // 16-byte pieces of a row in a block
  const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int waves = blockDim.x >> 6;
  const int64_t row0 = (int64_t)blockIdx.y * (RT * 16);
  const int chunk = waves * NB;  // blocks of inputs the workgroup holds at a time
  const uint4* const packed = static_cast<const uint4*>(p.packed);
  const char* const scales = static_cast<const char*>(p.scales);
  const char* const zeros = static_cast<const char*>(p.zeros);

  __shared__ __attribute__((aligned(16))) float sm[2][W][RT][16][20];
  __shared__ uint4 sm_x[W][16 * kLPR];

  // Absent zero points and bias are loads of nothing, that give 0, and not branches:
  // each path's loads have to be the same for the waits to be exact.
  const uint32_t unset = zeros == nullptr ? 0x88888888u : 0u;
  auto load_w = [&](int cn, int first, W4& a) {
#pragma unroll
    for (int m = 0; m < MB; ++m) {
      const int row = min(cn * MB + m, blocks_n - 1);
      const auto br = buffer_rsrc(static_cast<const T*>(p.bias) + row * 16,
                                  p.bias == nullptr ? 0 : min(16, p.n - row * 16) * (int)sizeof(T));
      if constexpr (sizeof(T) == 2)
        a.bias[m] = __uint_as_float((uint32_t)__builtin_amdgcn_raw_buffer_load_b16(br, i * 2, 0, 0) << 16);
      else
        a.bias[m] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(br, i * 4, 0, 0));
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        const int kb = min(first + nb * waves + wave, blocks_k - 1);  // past the last: x is zero there
        const int64_t block = (int64_t)row * blocks_k + kb;
        a.w[m][nb] = packed[block * 64 + lane];
        const uint2* sp = reinterpret_cast<const uint2*>(scales + (block * 4 + g) * (kSV * 8));
#pragma unroll
        for (int q = 0; q < kSV; ++q) a.s[m][nb][q] = sp[q];
        const auto zr = buffer_rsrc(zeros + block * (kGroups * 8), zeros == nullptr ? 0 : kGroups * 8);
        if constexpr (kGroups == 1) {
          a.z[m][nb][0] = __builtin_amdgcn_raw_buffer_load_b16(zr, g * 2, 0, 0) ^ unset;
        } else if constexpr (kGroups == 2) {
          a.z[m][nb][0] = __builtin_amdgcn_raw_buffer_load_b32(zr, g * 4, 0, 0) ^ unset;
        } else {
          const auto v = __builtin_amdgcn_raw_buffer_load_b64(zr, g * 8, 0, 0);
          a.z[m][nb][0] = v[0] ^ unset, a.z[m][nb][1] = v[1] ^ unset;
        }
      }
    }
  };

  uint4 x[NB][4][RT][L4<T>::kXP];
  float sums[NB][kGroups][RT];  // of x over each group, times kUnit
  // This wave's blocks of inputs from `first` on: x by rows, then as the product takes
  // it, and its sums.
  constexpr int kRows = 64 / kLPR, kTurns = 16 / kRows;  // rows a load, loads a block
  uint4 raw[NB][RT][kTurns];
  auto load_x = [&](int first) {
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const int k = (first + nb * waves + wave) * 128 + lane % kLPR * (16 / (int)sizeof(T));
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int u = 0; u < kTurns; ++u) {
          const int64_t row = min(row0 + rt * 16 + u * kRows + lane / kLPR, p.rows - 1);
          raw[nb][rt][u] = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.x) + row * p.x_row_stride +
                                                           min(k, p.k - 16 / (int)sizeof(T)));
          if (k >= p.k) raw[nb][rt][u] = make_uint4(0u, 0u, 0u, 0u);
        }
    }
  };
  auto settle_x = [&] {
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
        for (int u = 0; u < kTurns; ++u) sm_x[wave][l4_piece<kLPR>(u * kRows + lane / kLPR, lane % kLPR)] = raw[nb][rt][u];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int q = 0; q < kGroups; ++q) {
          float sum = 0.f;
          f32x4_t sums4 = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int s = q * kSteps; s < (q + 1) * kSteps; ++s) {
            uint4 in[kXV];
#pragma unroll
            for (int v = 0; v < kXV; ++v) in[v] = sm_x[wave][l4_piece<kLPR>(i, (s * 4 + g) * kXV + v)];
            if constexpr (sizeof(T) == 2) {
              x[nb][s][rt][0] = in[0];
              // A product with kUnit: every output's row holds the sums.
              const uint4 unit = make_uint4(0x37803780u, 0x37803780u, 0x37803780u, 0x37803780u);
              sums4 = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, unit),
                                                              __builtin_bit_cast(bf16x8_t, in[0]), sums4, 0, 0, 0);
            } else {
              float f[8];
#pragma unroll
              for (int v = 0; v < kXV; ++v) unpack<T>(in[v], f + v * 8 / kXV);
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                f[e] *= L4<T>::kUnit;
                sum += f[e];
              }
              l4_parts(f, x[nb][s][rt]);
            }
          }
          if constexpr (sizeof(T) == 2) {
            sums[nb][q][rt] = sums4[0];
          } else {
            float a, b;
            lane_pair<16>(sum, a, b);
            sum = a + b;
            lane_pair<32>(sum, a, b);
            sums[nb][q][rt] = a + b;
          }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
        __builtin_amdgcn_wave_barrier();
      }
  };

  // The turn (a block of outputs, a chunk of inputs) after one.
  auto after = [&](int& cn, int& first) {
    if (CHUNKED) first += chunk;
    if (!CHUNKED || first >= blocks_k) {
      first = 0;
      cn += gridDim.x;
    }
  };

  W4 a, b;  // this turn's weights and the next's
  int cn = blockIdx.x, first = 0, cn_next = cn, first_next = 0;
  load_w(cn, 0, a);
  load_x(0);
  if (!CHUNKED) settle_x();
  int buffer = 0;
  f32x4_t total[MB][RT];
#pragma unroll
  for (int m = 0; m < MB; ++m)
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) total[m][rt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  while (cn * MB < blocks_n) {
    if (CHUNKED) {
      settle_x();
      load_x(first + chunk < blocks_k ? first + chunk : 0);
    }
    after(cn_next, first_next);
    load_w(cn_next, first_next, b);  // past the last block: the last again
#pragma unroll
    for (int m = 0; m < MB; ++m)
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
      const uint32_t words[4] = {a.w[m][nb].x, a.w[m][nb].y, a.w[m][nb].z, a.w[m][nb].w};
#pragma unroll
      for (int q = 0; q < kGroups; ++q) {
        const uint32_t zr = a.z[m][nb][q / 2] >> (q % 2 * 16);
        float sc[4];
        if constexpr (sizeof(T) == 2) {
          sc[0] = bf16_lo(a.s[m][nb][q].x), sc[1] = bf16_hi(a.s[m][nb][q].x);
          sc[2] = bf16_lo(a.s[m][nb][q].y), sc[3] = bf16_hi(a.s[m][nb][q].y);
        } else {
          sc[0] = __uint_as_float(a.s[m][nb][2 * q].x), sc[1] = __uint_as_float(a.s[m][nb][2 * q].y);
          sc[2] = __uint_as_float(a.s[m][nb][2 * q + 1].x), sc[3] = __uint_as_float(a.s[m][nb][2 * q + 1].y);
        }
        f32x4_t acc[RT];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float zero = kOffset + (float)((zr >> (4 * r)) & 0xfu);
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) acc[rt][r] = -zero * sums[nb][q][rt];
        }
#pragma unroll
        for (int s = 0; s < kSteps; ++s) l4_step<T, RT>(words[q * kSteps + s], x[nb][q * kSteps + s], acc);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int r = 0; r < 4; ++r) total[m][rt][r] = fmaf(acc[rt][r], sc[r], total[m][rt][r]);
      }
    }
    float bias[MB];
#pragma unroll
    for (int m = 0; m < MB; ++m) bias[m] = a.bias[m];
    a = b;
    const int turn = cn;
    after(cn, first);
    if (CHUNKED && cn == turn) continue;  // more inputs of this block; uniform
#pragma unroll
    for (int m = 0; m < MB; ++m) {
      const int block = turn * MB + m;
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        *reinterpret_cast<float4*>(&sm[buffer][wave][rt][i][g * 4]) =
            make_float4(total[m][rt][0], total[m][rt][1], total[m][rt][2], total[m][rt][3]);
        total[m][rt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
      }
      // An LDS-only barrier: the weights stay in flight across it.
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
      __builtin_amdgcn_s_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
      // A wave finishes 2 RT rows, 16 lanes a row.  Every wave issues the same stores
      // (nothing leaves past a row's range): were they in a branch, the wait for the
      // next weights would be set for the path without them and cover later loads too.
      constexpr int kFinish = RT * 16 / W;
      auto finish = [&](int row_w) {
        const int mine = row_w + min(g, kFinish - 1);
        float y = 0.f;
        for (int u = 0; u < waves; ++u) y += sm[buffer][u][mine >> 4][mine & 15][i];
        y = fmaf(y, 1.f / L4<T>::kUnit, bias[m]);
#pragma unroll
        for (int r = 0; r < kFinish; ++r) {
          const int64_t row = row0 + row_w + r;
          const auto rsrc = buffer_rsrc(static_cast<T*>(p.out) + row * p.out_row_stride + block * 16,
                                        row < p.rows ? max(min(16, p.n - block * 16), 0) * (int)sizeof(T) : 0);
          const uint32_t off = g == r ? i * sizeof(T) : 0xffff0000u;
          if constexpr (sizeof(T) == 2)
            __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(unsigned short, (__bf16)y), rsrc, off, 0, 0);
          else
            __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(y), rsrc, off, 0, 0);
        }
      };
      finish(wave * kFinish);
      for (int row_w = (waves + wave) * kFinish; row_w < 16 * RT; row_w += waves * kFinish) finish(row_w);
      buffer ^= 1;
    }
  }
}

template <typename T, int W, int RT, int NB, int MB, bool CHUNKED>
hipError_t launch_l4_group(const asrlayer_linear4_params& p, hipStream_t stream) {
  const int blocks_n = (p.n + 15) / 16, blocks_k = (p.k + 127) / 128;
  const int64_t row_blocks = (p.rows + RT * 16 - 1) / (RT * 16);
  // One workgroup a CU, or two where they fit and the blocks are many: a second one
  // loads x again, so at fewer blocks it costs (16 rows of 2048 to 12288 outputs, 768
  // blocks: 6.9 us with 512 workgroups, 6.6 with 256; 16384: 7.3 and 7.3; 24576: 8.7 and
  // 9.0; 4 rows to 151936: 34.7 and 43.6; two row tiles, 64 rows to 12288: 12.5 and
  // 12.2, 33 rows of 1024 to 16384: 9.4 and 10.2).  Where the blocks are more than the
  // workgroups across, workgroups of the same outputs, one a block of rows, lie a multiple of
  // 8 apart, on one XCD, whose L2 then reads the weights once (80 rows to 151936: 122.1
  // us for 124.1).
  const bool two = (p.group == 32 ? l4_per_cu<T, W, RT, NB, MB, 32, CHUNKED>()
                                  : l4_per_cu<T, W, RT, NB, MB, 128, CHUNKED>()) > 1 && blocks_n * row_blocks >= (RT == 1 ? 1536 : 2048);
  int64_t across = (two ? 512 : 256) / row_blocks;
  if (across > 8) across -= across % 8;
  if (across < 1) across = 1;
  const int turns_n = (blocks_n + MB - 1) / MB;
  const dim3 grid(turns_n < across ? turns_n : across, row_blocks), block(64 * (blocks_k < W ? blocks_k : W));
  if constexpr ((W == 8 || RT == 1) && MB < 4) {
    if (p.group == 32) {
      hipLaunchKernelGGL((linear4_kernel<T, W, RT, NB, MB, 32, CHUNKED>), grid, block, 0, stream, p, blocks_n, blocks_k);
      return hipGetLastError();
    }
  }
  if (p.group == 64)
    hipLaunchKernelGGL((linear4_kernel<T, W, RT, NB, MB, 64, CHUNKED>), grid, block, 0, stream, p, blocks_n, blocks_k);
  else
    hipLaunchKernelGGL((linear4_kernel<T, W, RT, NB, MB, 128, CHUNKED>), grid, block, 0, stream, p, blocks_n, blocks_k);
  return hipGetLastError();
}

// x in chunks: where the GPU has more than one block of outputs a workgroup, two
// or four at a time share a chunk (16 x 5120 x 13824: 24.1 us with one, 18.2 with two,
// 16.0 with four; 64 x 8192 x 4096, 512 blocks: 24.4, 17.3 and 22.3; 256 blocks: 12.2,
// 14.6 and 20.0).  Four take more registers than float32 or groups of 32 leave.
template <typename T, int RT>
hipError_t launch_l4_chunked(const asrlayer_linear4_params& p, hipStream_t stream) {
  const int64_t blocks = (int64_t)((p.n + 15) / 16) * ((p.rows + RT * 16 - 1) / (RT * 16));
  if (blocks <= 256) return launch_l4_group<T, 8, RT, 1, 1, true>(p, stream);
  if constexpr (sizeof(T) == 2) {
    if (blocks > 512 && p.group > 32) return launch_l4_group<T, 8, RT, 1, 4, true>(p, stream);
  }
  return launch_l4_group<T, 8, RT, 1, 2, true>(p, stream);
}

// Two row tiles where 256 workgroups are left: half the reads of the weights (64 x
// 2048 x 12288: 11.1 us for 12.8; 64 x 1024 x 4096: 4.8 for 5.3); with fewer, one
// (24 x 5120 x 1280: 6.2 us for 8.2).  All of x in registers where it fits, so that
// x is read once a workgroup; else in chunks, again for each turn over the outputs:
// 64 x 4096 x 12288 in 17.0 us with 16 waves holding x, 23.1 in chunks; 16 x 4096 x
// 12288 with four blocks a wave in 9.3 us, 10.9 in chunks; 4 x 2560 x 151936 with three
// 54.5, with four, of which some are none, 60.7.  Up to 512 blocks of outputs chunks,
// which two share, are as good (16 x 4096 x 6144: 7.6 us, 7.8 holding x).  Chunks take 16
// waves at 256 blocks or fewer if that halves their number: 8 x 6144 x 2048 (6 chunks
// or 3) in 6.5 us for 7.0; at 24 x 5120 x 1280 (5 or 3) 6.8 for 6.2.  Groups of 32 need
// more registers than 16 waves leave: 32 x 4096 x 6144 in 11.7 us, 19.0 with 16 waves.  So
// does float32, whose x is three times as large: 8 waves, and two row tiles only where
// each wave holds one block of inputs.
template <typename T>
hipError_t launch_l4(const asrlayer_linear4_params& p, hipStream_t stream) {
  const int blocks_n = (p.n + 15) / 16, blocks_k = (p.k + 127) / 128;
  const bool several = sizeof(T) == 2 && blocks_k > 16 && blocks_k <= 32 && blocks_n > 512;  // blocks a wave
  if (p.rows > 16 && (int64_t)blocks_n * ((p.rows + 31) / 32) >= 256 && !(several && p.group == 32) &&
      (sizeof(T) == 2 || blocks_k <= 8)) {
    if (blocks_k <= 8) return launch_l4_group<T, 8, 2, 1, 1, false>(p, stream);
    if constexpr (sizeof(T) == 2) {
      if (blocks_k <= 16) return launch_l4_group<T, 8, 2, 2, 1, false>(p, stream);
      if (blocks_k <= 32 && p.group > 32) return launch_l4_group<T, 16, 2, 2, 1, false>(p, stream);
      return launch_l4_chunked<T, 2>(p, stream);
    }
  }
  if (blocks_k <= 8) return launch_l4_group<T, 8, 1, 1, 1, false>(p, stream);
  if (blocks_k <= 16) return launch_l4_group<T, 8, 1, 2, 1, false>(p, stream);
  if constexpr (sizeof(T) == 2) {
    if (several)
      return blocks_k <= 24 ? launch_l4_group<T, 8, 1, 3, 1, false>(p, stream) : launch_l4_group<T, 8, 1, 4, 1, false>(p, stream);
    if (blocks_n * ((p.rows + 15) / 16) <= 256 && (blocks_k + 15) / 16 * 2 <= (blocks_k + 7) / 8)
      return launch_l4_group<T, 16, 1, 1, 1, true>(p, stream);
  }
  return launch_l4_chunked<T, 1>(p, stream);
}

}  // namespace
}  // namespace asrattn
