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
#include "round8.hpp"
#include "row_ops.hpp"

namespace asrattn {
namespace {

typedef int i32x4_t __attribute__((ext_vector_type(4)));

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
