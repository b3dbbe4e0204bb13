// Rows through a matrix of 8-bit weights with a scale per output
// (asrlayer_linear8): the rows are rounded to 8 bits first, then multiplied as whole
// numbers on v_mfma_i32_16x16x64_i8, and the scales, the bias and the gate's
// activation happen on the sums.
//
// Both operands lie in blocks of 16 (rows, outputs) x 64 inputs, 1 KB in the order in
// which a wave's lanes take them.  The outputs are the product's rows, so a lane
// holds four consecutive outputs of one row.
#include "kernels.hpp"
#include "layers.hpp"
#include "ring_common.hpp"
#include "round8.hpp"
#include "row_ops.hpp"

namespace asrattn {
namespace {

using ring::dma16;
using ring::wait_vmcnt;
using ring::xcd_remap;

typedef int i32x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) const i32x4_t* lds_i32x4_ptr;

// An LDS read by byte address, so that its constant part folds into the instruction.
__device__ __forceinline__ i32x4_t lds_read(uint32_t addr) { return *(lds_i32x4_ptr)(size_t)addr; }

constexpr int kThreads = 256;

// 16 inputs of a row from `at` on, zeros past k.
template <typename T>
__device__ __forceinline__ void load_inputs(const T* row, int at, int k, bool vectors, float* x) {
  constexpr int EPL = Elem<T>::kPerVec;
  if (vectors && at + 16 <= k) {
#pragma unroll
    for (int v = 0; v < 16 / EPL; ++v) Elem<T>::load16(row + at + v * EPL, x + v * EPL);
  } else {
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] = at + e < k ? Elem<T>::load1(row + at + e) : 0.f;
  }
}

// A wave rounds a row: its largest magnitude, then 16 inputs a lane at a time.
template <typename T>
__global__ __launch_bounds__(kThreads) void round_rows_kernel(const asrlayer_linear8_params p, uint4* packed, float* scales,
                                                              bool vectors) {
  const int64_t row = (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (row >= p.rows) return;
  const T* x = static_cast<const T*>(p.x) + row * p.x_row_stride;
  const int pieces = (p.k + 15) / 16, blocks = (p.k + 63) / 64;
  uint32_t largest = 0;
  for (int piece = lane; piece < pieces; piece += 64) {
    float v[16];
    load_inputs(x, piece * 16, p.k, vectors, v);
#pragma unroll
    for (int e = 0; e < 16; ++e) largest = max(largest, magnitude(v[e]));
  }
  const Scale8 s = scale8(group_umax<64>(largest));
  if (lane == 0) scales[row] = s.scale;
  uint4* out = packed + (row / 16) * blocks * 64 + row % 16;
  for (int piece = lane; piece < pieces; piece += 64) {
    float v[16];
    load_inputs(x, piece * 16, p.k, vectors, v);
    out[piece * 16] = make_uint4(round8x4(v, s), round8x4(v + 4, s), round8x4(v + 8, s), round8x4(v + 12, s));
  }
}

// The product's sum as a float times both scales, so that nothing on the way
// overflows or loses bits that the result has.
__device__ __forceinline__ float scaled(int sum, float row, float output) {
  const float y = (float)sum;
  return row >= 1.f ? y * output * row : y * row * output;
}

__device__ __forceinline__ float silu(float x) { return x / (1.f + fast_exp2(-kLog2e * x)); }

template <typename T, bool GATED>
__global__ __launch_bounds__(kThreads) void linear8_kernel(const asrlayer_linear8_params p, const uint4* packed,
                                                           const float* row_scales) {
  const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  const int outputs = GATED ? p.n / 2 : p.n;
  const int n0 = (blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6)) * 16;
  if (n0 >= outputs) return;
  const int blocks = (p.k + 63) / 64;
  const int64_t tile = blockIdx.y;
  const uint4* x = packed + tile * blocks * 64 + lane;
  const uint4* w[2];
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int n = min(n0 + i, outputs - 1) + half * outputs * GATED;
    w[half] = static_cast<const uint4*>(p.packed) + (int64_t)(n / 16) * blocks * 64 + g * 16 + n % 16;
  }
  i32x4_t acc[2] = {};
  for (int kb = 0; kb < blocks; ++kb) {
    const i32x4_t xv = __builtin_bit_cast(i32x4_t, x[kb * 64]);
#pragma unroll
    for (int half = 0; half <= GATED; ++half)
      acc[half] = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4_t, w[half][kb * 64]), xv, acc[half], 0, 0, 0);
  }
  const int64_t row = tile * 16 + i;
  if (row >= p.rows) return;
  const float rs = row_scales[row];
  T* out = static_cast<T*>(p.out) + row * p.out_row_stride;
  const T* ws = static_cast<const T*>(p.scales);
  const T* bias = static_cast<const T*>(p.bias);
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int n = n0 + 4 * g + r;
    if (n >= outputs) break;
    float y[2];
#pragma unroll
    for (int half = 0; half <= GATED; ++half) {
      const int at = n + half * outputs;
      y[half] = scaled(acc[half][r], rs, Elem<T>::load1(ws + at));
      if (bias != nullptr) y[half] += Elem<T>::load1(bias + at);
    }
    Elem<T>::store1(out + n, GATED ? silu(y[0]) * y[1] : y[0]);
  }
}

// Stores N consecutive outputs of a row from n on, of which those below `outputs`
// exist.
template <typename T, int N>
__device__ __forceinline__ void store_outputs(T* row, int n, int outputs, bool vectors, const float* y) {
  constexpr int EPL = Elem<T>::kPerVec;
  if (vectors && n + N <= outputs) {
#pragma unroll
    for (int v = 0; v < N / EPL; ++v) *reinterpret_cast<uint4*>(row + n + v * EPL) = pack<T>(y + v * EPL);
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (n + e < outputs) Elem<T>::store1(row + n + e, y[e]);
  }
}

// 256 rows x 256 outputs (gated: 128 gates and their projections): eight waves of
// 128 rows x 64 outputs.  Blocks of both operands, 64 inputs deep, move by DMA into a
// ring of four stages in LDS, 1 KB an instruction, three stages ahead, and one barrier
// a stage separates "landed for every wave" from "free".
//
// The outputs' order inside a wave's 64 is chosen for the stores: product j's row 4 q
// + r is output 16 q + 4 j + r (gated: 8 q + 4 j + r of 32), so a lane ends with 16
// consecutive outputs of a row (8).  Its operand then takes rows of several blocks,
// which lie 64 bytes more than their size apart, so that the 16 rows a read touches at
// a time lie in different banks.
constexpr int kLargeTile = 256, kStages = 4, kPitch = 1024 + 64;
constexpr int kStageBytes = 2 * (kLargeTile / 16) * kPitch;

template <typename T, bool GATED>
__global__ __launch_bounds__(512, 2) void linear8_large_kernel(const asrlayer_linear8_params p, const uint4* packed,
                                                               const float* row_scales, int row_tiles, int col_tiles,
                                                               bool vectors) {
  __shared__ __attribute__((aligned(16))) unsigned char lds[kStages * kStageBytes];
  const int outputs = GATED ? p.n / 2 : p.n;
  const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int wm = wave & 1, wn = wave >> 1;
  const int blocks = (p.k + 63) / 64;

  // Eight tiles of rows share a tile of outputs in turn, so that an XCD's workgroups
  // read few of both.
  const int item = xcd_remap((int)blockIdx.x, (int)gridDim.x);
  constexpr int kGroup = 8;
  const int band = item / (kGroup * col_tiles), first = band * kGroup, within = item - first * col_tiles;
  const int tall = min(kGroup, row_tiles - first);
  const int tile = first + within % tall;
  const int n0 = within / tall * (GATED ? kLargeTile / 2 : kLargeTile);
  const int64_t row0 = (int64_t)tile * kLargeTile;

  // A wave's DMAs of a stage: two blocks of rows, two of outputs.
  const int64_t row_blocks = (p.rows + 15) / 16 - row0 / 16;
  const __amdgpu_buffer_rsrc_t xrs =
      buffer_rsrc(packed + row0 / 16 * blocks * 64, (uint32_t)min((int64_t)16, row_blocks) * (uint32_t)blocks * 1024);
  const int w_first = n0 / 16, w_second = (outputs + n0) / 16;  // blocks (gated: of the projections)
  const int w_blocks = (p.n + 15) / 16;
  const char* const w = static_cast<const char*>(p.packed);
  const __amdgpu_buffer_rsrc_t wrs = buffer_rsrc(w + (int64_t)w_first * blocks * 1024,
                                                 (uint32_t)min(17, w_blocks - w_first) * (uint32_t)blocks * 1024);
  const __amdgpu_buffer_rsrc_t urs = buffer_rsrc(w + (int64_t)w_second * blocks * 1024,
                                                 (uint32_t)min(17, w_blocks - w_second) * (uint32_t)blocks * 1024);
  uint32_t xoff[2], woff[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    xoff[u] = (uint32_t)(2 * wave + u) * (uint32_t)blocks * 1024 + lane * 16;
    // Rows of the matrix, 16 from a multiple of 16 on but for projections behind an odd
    // number of gates.
    const int block = 2 * wave + u;
    int r = block * 16 + i;
    if (GATED && block >= 8) r = r - 128 + (outputs + n0) % 16;
    woff[u] = (uint32_t)(r / 16) * (uint32_t)blocks * 1024 + g * 256 + r % 16 * 16;
  }
  const uint32_t lds_base = (uint32_t)(uintptr_t)lds;
  constexpr uint32_t kW = kLargeTile / 16 * kPitch;  // the outputs' blocks of a stage
  auto issue = [&](int t) {
    const uint32_t base = lds_base + (uint32_t)(t % kStages) * kStageBytes + 2 * wave * kPitch;
    const uint32_t at = (uint32_t)t * 1024;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      dma16(xrs, base + u * kPitch, xoff[u] + at);
      if (GATED && wave >= 4)
        dma16(urs, base + kW + u * kPitch, woff[u] + at);
      else
        dma16(wrs, base + kW + u * kPitch, woff[u] + at);
    }
  };

  // Operand addresses in stage 0.
  const uint32_t xaddr = (lds_base + 8 * wm * kPitch + lane * 16) & 0x3ffffu;
  const int q = i >> 2;
  uint32_t waddr[2];
  if constexpr (GATED) {
    const uint32_t at = kW + (2 * wn + (q >> 1)) * kPitch + g * 256 + (8 * (q & 1) + (i & 3)) * 16;
    waddr[0] = (lds_base + at) & 0x3ffffu;
    waddr[1] = (lds_base + at + 8 * kPitch) & 0x3ffffu;
  } else {
    const uint32_t at = kW + (4 * wn + q) * kPitch + g * 256 + (i & 3) * 16;
    waddr[0] = (lds_base + at) & 0x3ffffu;
    waddr[1] = waddr[0] + 128;
  }
  i32x4_t acc[8][4];
#pragma unroll
  for (int a = 0; a < 8; ++a)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[a][j] = i32x4_t{0, 0, 0, 0};

#pragma unroll
  for (int t = 0; t < kStages - 1; ++t) issue(t);
  for (int t = 0; t < blocks; ++t) {
    // Stage t has landed for every wave, and every wave is done with stage t - 1, whose
    // place the next DMA takes.
    wait_vmcnt<4 * (kStages - 2)>();
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
    issue(t + kStages - 1);
    const uint32_t so = (uint32_t)(t % kStages) * kStageBytes;
    i32x4_t wv[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) wv[j] = lds_read(waddr[j >> 1] + so + (j & 1) * 64);
#pragma unroll
    for (int a = 0; a < 8; ++a) {
      const i32x4_t xv = lds_read(xaddr + so + a * kPitch);
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[a][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wv[j], xv, acc[a][j], 0, 0, 0);
    }
  }
  wait_vmcnt<0>();  // the surplus DMAs, before the workgroup's LDS is another's

  constexpr int N = GATED ? 8 : 16;
  const int n = n0 + (GATED ? 32 : 64) * wn + N * g;
  if (n >= outputs) return;
  const T* ws = static_cast<const T*>(p.scales);
  const T* bias = static_cast<const T*>(p.bias);
  float scale[16], add[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const int at = GATED ? (e < 8 ? min(n + e, outputs - 1) : outputs + min(n + e - 8, outputs - 1)) : min(n + e, outputs - 1);
    scale[e] = Elem<T>::load1(ws + at);
    add[e] = bias != nullptr ? Elem<T>::load1(bias + at) : 0.f;
  }
#pragma unroll
  for (int a = 0; a < 8; ++a) {
    const int64_t row = row0 + 128 * wm + 16 * a + i;
    if (row >= p.rows) continue;
    const float rs = row_scales[row];
    float y[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      y[e] = scaled(acc[a][e / 4][e % 4], rs, scale[e]);
      if (bias != nullptr) y[e] += add[e];
    }
    if constexpr (GATED) {
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = silu(y[e]) * y[e + 8];
    }
    store_outputs<T, N>(static_cast<T*>(p.out) + row * p.out_row_stride, n, outputs, vectors, y);
  }
}

template <typename T>
hipError_t launch_typed(const asrlayer_linear8_params& p, void* workspace, hipStream_t stream) {
  const Linear8Workspace ws = linear8_workspace(p.rows, p.k);
  uint4* packed = static_cast<uint4*>(workspace);
  float* scales = reinterpret_cast<float*>(static_cast<char*>(workspace) + ws.scales);
  const bool vectors = reinterpret_cast<uintptr_t>(p.x) % 16 == 0 && p.x_row_stride % Elem<T>::kPerVec == 0;
  hipLaunchKernelGGL((round_rows_kernel<T>), dim3((unsigned)((p.rows + 3) / 4)), dim3(kThreads), 0, stream, p, packed,
                     scales, vectors);
  hipError_t err = hipGetLastError();
  if (err != hipSuccess) return err;
  const int outputs = p.gated ? p.n / 2 : p.n;
  if (p.rows > 64) {
    const int row_tiles = (int)((p.rows + kLargeTile - 1) / kLargeTile);
    const int wide = p.gated ? kLargeTile / 2 : kLargeTile, col_tiles = (outputs + wide - 1) / wide;
    const bool whole = reinterpret_cast<uintptr_t>(p.out) % 16 == 0 && p.out_row_stride % Elem<T>::kPerVec == 0;
    const dim3 grid((unsigned)((long long)row_tiles * col_tiles));
    if (p.gated)
      hipLaunchKernelGGL((linear8_large_kernel<T, true>), grid, dim3(512), 0, stream, p, packed, scales, row_tiles,
                         col_tiles, whole);
    else
      hipLaunchKernelGGL((linear8_large_kernel<T, false>), grid, dim3(512), 0, stream, p, packed, scales, row_tiles,
                         col_tiles, whole);
    return hipGetLastError();
  }
  const dim3 grid((outputs + 63) / 64, (unsigned)((p.rows + 15) / 16));
  if (p.gated)
    hipLaunchKernelGGL((linear8_kernel<T, true>), grid, dim3(kThreads), 0, stream, p, packed, scales);
  else
    hipLaunchKernelGGL((linear8_kernel<T, false>), grid, dim3(kThreads), 0, stream, p, packed, scales);
  return hipGetLastError();
}

}  // namespace

Linear8Workspace linear8_workspace(int64_t rows, int k) {
  const size_t tiles = (size_t)(rows + 15) / 16;
  Linear8Workspace w;
  w.scales = tiles * ((size_t)(k + 63) / 64) * 1024;
  w.total = w.scales + (tiles * 16 * sizeof(float) + 255) / 256 * 256;
  return w;
}

hipError_t launch_linear8(const asrlayer_linear8_params& p, void* workspace, hipStream_t stream) {
  return p.dtype == ASRATTN_BF16 ? launch_typed<bf16_raw>(p, workspace, stream) : launch_typed<float>(p, workspace, stream);
}

}  // namespace asrattn
