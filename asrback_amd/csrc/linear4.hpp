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
//   * bf16: a nibble becomes bf16 by an AND and an OR: 0x4300 | q is 128 + q
//     exactly, two elements an instruction (7 for 8 weights).  The 128 and the
//     zero point leave through the accumulator, which starts at
//     -(128 + zero) sum(x) of the group: sum x (128 + q) - (128 + zero) sum x.
//     The sums' float32 rounding is 2^-24 of values up to 143 |x|, some 30 times
//     the result's own: 2^-19, far below the 2^-8 of the bf16 result.
//     float32: nibbles become floats one by one, and only the zero point leaves
//     that way (the matrix instruction, 8 times slower than bf16's, bounds it).
//   * Outputs lie in the rows of the product and x's rows in its columns, so a
//     lane holds four outputs of one x row: a group's scales are one small load
//     for four outputs, the group's sum of x one value per lane.
//   * A workgroup's waves split the inputs, each keeping its part of x in
//     registers, and go through the workgroup's blocks of outputs with it; the
//     next block's weights load while this one's are multiplied.  The waves' sums
//     meet in LDS once a block (two buffers, one barrier).
#pragma once

#include "common.hpp"
#include "kernels.hpp"
#include "row_ops.hpp"

namespace asrattn {
namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

constexpr int kL4Waves = 8;  // at most, of a workgroup

template <typename T>
struct L4 {
  static constexpr int kXV = sizeof(T) == 2 ? 1 : 2;  // 16-byte vectors of 8 inputs
  static constexpr float kOffset = sizeof(T) == 2 ? 128.f : 0.f;  // what a weight operand adds to q
};

// acc += (16 outputs x 32 inputs) (16 rows x 32 inputs)^T from a dword of
// weights and 8 inputs a lane.
template <typename T, int RT>
__device__ __forceinline__ void l4_step(uint32_t w, const uint4 (*x)[L4<T>::kXV], f32x4_t* acc) {
  if constexpr (sizeof(T) == 2) {
    uint4 a;
    a.x = (w & 0x000f000fu) | 0x43004300u;
    a.y = ((w >> 4) & 0x000f000fu) | 0x43004300u;
    a.z = ((w >> 8) & 0x000f000fu) | 0x43004300u;
    a.w = ((w >> 12) & 0x000f000fu) | 0x43004300u;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
      acc[rt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                        __builtin_bit_cast(bf16x8_t, x[rt][0]), acc[rt], 0, 0, 0);
  } else {
    const uint32_t lo = w & 0x0f0f0f0fu, hi = (w >> 4) & 0x0f0f0f0fu;
    // Nibbles 0 1 2 3 hold inputs 0 2 4 6, nibbles 4 5 6 7 inputs 1 3 5 7.
    const float q[8] = {(float)(lo & 0xffu),         (float)((lo >> 16) & 0xffu), (float)(hi & 0xffu),
                        (float)((hi >> 16) & 0xffu), (float)((lo >> 8) & 0xffu),  (float)(lo >> 24),
                        (float)((hi >> 8) & 0xffu),  (float)(hi >> 24)};
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const uint4 v = x[rt][j / 4];
        const uint32_t xj = j % 4 == 0 ? v.x : j % 4 == 1 ? v.y : j % 4 == 2 ? v.z : v.w;
        acc[rt] = __builtin_amdgcn_mfma_f32_16x16x4f32(q[j], __uint_as_float(xj), acc[rt], 0, 0, 0);
      }
  }
}

// RT: 16-row tiles of x; NB: blocks of 128 inputs a wave keeps; GROUP: inputs of
// a scale.  Waves: kL4Waves or fewer.
template <typename T, int RT, int NB, int GROUP>
__global__ __launch_bounds__(64 * kL4Waves) void linear4_kernel(const asrlayer_linear4_params p, int blocks_n, int blocks_k) {
  constexpr int kXV = L4<T>::kXV, kGroups = 128 / GROUP, kSteps = GROUP / 32;
  constexpr float kOffset = L4<T>::kOffset;
  const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int waves = blockDim.x >> 6;
  const int64_t row0 = (int64_t)blockIdx.y * (RT * 16);
  const int chunk = waves * NB;  // blocks of inputs the workgroup holds at a time
  const uint4* const packed = static_cast<const uint4*>(p.packed);
  const T* const scales = static_cast<const T*>(p.scales);
  const uint16_t* const zeros = static_cast<const uint16_t*>(p.zeros);

  __shared__ __attribute__((aligned(16))) float sm[2][kL4Waves][RT][16][20];

  uint4 x[NB][4][RT][kXV];
  float sums[NB][kGroups][RT];  // of x over each group
  // This wave's blocks of inputs from first on, and x in them.
  auto load_x = [&](int first) {
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const int kb = first + nb * waves + wave;
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const int k = kb * 128 + s * 32 + g * 8;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          const int64_t row = min(row0 + rt * 16 + i, p.rows - 1);
          const T* at = static_cast<const T*>(p.x) + row * p.x_row_stride + min(k, p.k - 8);
#pragma unroll
          for (int v = 0; v < kXV; ++v) {
            x[nb][s][rt][v] = *reinterpret_cast<const uint4*>(at + v * (8 / kXV));
            if (k >= p.k) x[nb][s][rt][v] = make_uint4(0u, 0u, 0u, 0u);
          }
        }
      }
    }
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int q = 0; q < kGroups; ++q)
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          float sum = 0.f;
#pragma unroll
          for (int s = 0; s < kSteps; ++s)
#pragma unroll
            for (int v = 0; v < kXV; ++v) {
              float f[8 / kXV];
              unpack<T>(x[nb][q * kSteps + s][rt][v], f);
#pragma unroll
              for (int e = 0; e < 8 / kXV; ++e) sum += f[e];
            }
          float a, b;
          lane_pair<16>(sum, a, b);
          sum = a + b;
          lane_pair<32>(sum, a, b);
          sums[nb][q][rt] = a + b;
        }
  };

  uint4 w[NB], wn[NB];
  T sc[NB][kGroups][4], scn[NB][kGroups][4];
  uint32_t zr[NB][kGroups], zrn[NB][kGroups];
  auto load_w = [&](int cn, int first, uint4* wv, T (*s)[kGroups][4], uint32_t (*z)[kGroups]) {
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const int kb = min(first + nb * waves + wave, blocks_k - 1);  // past the last: x is zero there
      const int64_t block = (int64_t)cn * blocks_k + kb;
      wv[nb] = packed[block * 64 + lane];
#pragma unroll
      for (int q = 0; q < kGroups; ++q) {
        const int64_t at = block * kGroups + q;
        if constexpr (sizeof(T) == 2) {
          const uint2 v = *reinterpret_cast<const uint2*>(scales + at * 16 + g * 4);
          s[nb][q][0] = (T)v.x, s[nb][q][1] = (T)(v.x >> 16), s[nb][q][2] = (T)v.y, s[nb][q][3] = (T)(v.y >> 16);
        } else {
          const float4 v = *reinterpret_cast<const float4*>(scales + at * 16 + g * 4);
          s[nb][q][0] = v.x, s[nb][q][1] = v.y, s[nb][q][2] = v.z, s[nb][q][3] = v.w;
        }
        z[nb][q] = zeros != nullptr ? (uint32_t)zeros[at * 4 + g] : 0x8888u;
      }
    }
  };

  if (blocks_k <= chunk) load_x(0);
  int buffer = 0;
  int cn = blockIdx.x;
  load_w(min(cn, blocks_n - 1), 0, w, sc, zr);
  for (; cn < blocks_n; cn += gridDim.x) {
    f32x4_t total[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) total[rt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    for (int first = 0; first < blocks_k; first += chunk) {
      if (blocks_k > chunk) load_x(first);
      // The next weights this wave multiplies (the last again at the end).
      const bool last = first + chunk >= blocks_k;
      load_w(last ? min(cn + (int)gridDim.x, blocks_n - 1) : cn, last ? 0 : first + chunk, wn, scn, zrn);
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        const uint32_t words[4] = {w[nb].x, w[nb].y, w[nb].z, w[nb].w};
#pragma unroll
        for (int q = 0; q < kGroups; ++q) {
          f32x4_t acc[RT];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float zero = kOffset + (float)((zr[nb][q] >> (4 * r)) & 0xfu);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) acc[rt][r] = -zero * sums[nb][q][rt];
          }
#pragma unroll
          for (int s = 0; s < kSteps; ++s) l4_step<T, RT>(words[q * kSteps + s], x[nb][q * kSteps + s], acc);
#pragma unroll
          for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int r = 0; r < 4; ++r) total[rt][r] = fmaf(acc[rt][r], Elem<T>::load1(&sc[nb][q][r]), total[rt][r]);
        }
      }
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        w[nb] = wn[nb];
#pragma unroll
        for (int q = 0; q < kGroups; ++q) {
          zr[nb][q] = zrn[nb][q];
#pragma unroll
          for (int r = 0; r < 4; ++r) sc[nb][q][r] = scn[nb][q][r];
        }
      }
    }
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
      *reinterpret_cast<float4*>(&sm[buffer][wave][rt][i][g * 4]) =
          make_float4(total[rt][0], total[rt][1], total[rt][2], total[rt][3]);
    __syncthreads();
    // Four outputs of a row a thread.
    for (int t = threadIdx.x; t < RT * 64; t += blockDim.x) {
      const int rt = t >> 6, r = (t >> 2) & 15, c = (t & 3) * 4;
      const int64_t row = row0 + rt * 16 + r;
      if (row >= p.rows) continue;
      float y[4] = {0.f, 0.f, 0.f, 0.f};
      for (int u = 0; u < waves; ++u) {
        const float4 v = *reinterpret_cast<const float4*>(&sm[buffer][u][rt][r][c]);
        y[0] += v.x, y[1] += v.y, y[2] += v.z, y[3] += v.w;
      }
      T* out = static_cast<T*>(p.out) + row * p.out_row_stride;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int n = cn * 16 + c + e;
        if (n >= p.n) continue;
        if (p.bias != nullptr) y[e] += Elem<T>::load1(static_cast<const T*>(p.bias) + n);
        Elem<T>::store1(out + n, y[e]);
      }
    }
    buffer ^= 1;
  }
}

template <typename T, int RT, int NB>
hipError_t launch_l4_group(const asrlayer_linear4_params& p, int waves, hipStream_t stream) {
  const int blocks_n = (p.n + 15) / 16, blocks_k = (p.k + 127) / 128;
  const int row_blocks = (int)((p.rows + RT * 16 - 1) / (RT * 16));
  const int most = 512 / row_blocks < 1 ? 1 : 512 / row_blocks;
  const dim3 grid(blocks_n < most ? blocks_n : most, row_blocks), block(64 * waves);
  if (p.group == 32)
    hipLaunchKernelGGL((linear4_kernel<T, RT, NB, 32>), grid, block, 0, stream, p, blocks_n, blocks_k);
  else if (p.group == 64)
    hipLaunchKernelGGL((linear4_kernel<T, RT, NB, 64>), grid, block, 0, stream, p, blocks_n, blocks_k);
  else
    hipLaunchKernelGGL((linear4_kernel<T, RT, NB, 128>), grid, block, 0, stream, p, blocks_n, blocks_k);
  return hipGetLastError();
}

template <typename T>
hipError_t launch_l4(const asrlayer_linear4_params& p, hipStream_t stream) {
  const int blocks_k = (p.k + 127) / 128;
  const int waves = blocks_k < kL4Waves ? blocks_k : kL4Waves;
  const int per_wave = (blocks_k + waves - 1) / waves;
  if (p.rows <= 16) {
    if (per_wave <= 1) return launch_l4_group<T, 1, 1>(p, waves, stream);
    if (per_wave <= 2) return launch_l4_group<T, 1, 2>(p, waves, stream);
    return launch_l4_group<T, 1, 4>(p, waves, stream);
  }
  if (p.rows <= 32) {
    if (per_wave <= 1) return launch_l4_group<T, 2, 1>(p, waves, stream);
    return launch_l4_group<T, 2, 2>(p, waves, stream);
  }
  return launch_l4_group<T, 4, 1>(p, waves, stream);
}

}  // namespace
}  // namespace asrattn
