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

// ring::dma16 in a kernel that uses M0 for nothing else.
__device__ __forceinline__ void dma16_m0(__amdgpu_buffer_rsrc_t rsrc, uint32_t lds_base, uint32_t voff) {
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 0\n\t"
      "buffer_load_dwordx4 %1, %2, 0 offen lds"
      :
      : "s"(lds_base), "v"(voff), "s"(rsrc)
      : "memory", "m0");
}

// acc += (16 outputs x 64 inputs) (16 rows x 64 inputs)^T.  As inline assembly, so that
// the sums stay in the accumulation registers, all 256 of a wave's (left to itself, the
// compiler copies some of them to the others and back, hundreds a stage).  The compiler
// does not know of the products' time: settle() goes between them and a use of their sums.
__device__ __forceinline__ void multiply(const i32x4_t& w, const i32x4_t& x, i32x4_t& acc) {
  asm volatile("v_mfma_i32_16x16x64_i8 %0, %1, %2, %0" : "+a"(acc) : "v"(w), "v"(x));
}
// One of the sums, from the accumulation registers when it is asked for (again the
// compiler would read all of them ahead).
__device__ __forceinline__ int sum_of(const i32x4_t& acc, int r) {
  int x;
  const int held = acc[r];
  asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(x) : "a"(held));
  return x;
}
__device__ __forceinline__ void settle() { asm volatile("s_nop 15\n\ts_nop 15" ::: "memory"); }

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

// The product's sum, below 2^31, as a float times both scales, so that nothing on the
// way overflows or loses bits that the result has: a row's scale from kFar on goes last.
constexpr float kFar = 0x1p90f;
__device__ __forceinline__ float scaled(int sum, float row, float output) {
  const float y = (float)sum;
  return row >= kFar ? y * output * row : y * row * output;
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

// N consecutive elements.
template <typename T, int N>
__device__ __forceinline__ void load_whole(const T* p, float* x) {
  constexpr int EPL = Elem<T>::kPerVec;
#pragma unroll
  for (int v = 0; v < N / EPL; ++v) Elem<T>::load16(p + v * EPL, x + v * EPL);
}
template <typename T, int N>
__device__ __forceinline__ void store_whole(T* p, const float* x) {
  constexpr int EPL = Elem<T>::kPerVec;
#pragma unroll
  for (int v = 0; v < N / EPL; ++v) *reinterpret_cast<uint4*>(p + v * EPL) = pack<T>(x + v * EPL);
}

// Tiles of 256 rows x 256 outputs (gated: 128 gates and their projections), a workgroup
// a CU that takes one after another: four waves of 128 x 128, the largest that leave
// room for their operands, since what bounds the product is LDS: a wave reads 16 KB of
// it for 64 products.  Blocks of both operands, 64 inputs deep, move by DMA into a ring
// of four stages, 1 KB an instruction, and one barrier a stage separates "landed for
// every wave" from "free".  A stage's operands are read while the one before is
// multiplied, and the next tile's first stages load through the end of this one.
//
// The outputs' order inside a wave's 64 is chosen for the stores: product j's row 4 q
// + r is output 16 q + 4 j + r (gated: 8 q + 4 j + r of 32), so a lane ends with 16
// consecutive outputs of a row (8).  Its operand then takes rows of several blocks,
// which lie 64 bytes more than their size apart, so that the 16 rows a read touches at
// a time lie in different banks.
constexpr int kLargeTile = 256, kStages = 4, kPitch = 1024 + 64;
constexpr int kStageBytes = 2 * (kLargeTile / 16) * kPitch;
// Offset of a DMA that is to write zeros.
constexpr uint32_t kNowhere = 0x7ff00000u;

template <typename T, bool GATED>
__global__ __launch_bounds__(256, 1) void linear8_large_kernel(const asrlayer_linear8_params p, const uint4* packed,
                                                               const float* row_scales, int row_tiles, int col_tiles,
                                                               bool whole) {
  __shared__ __attribute__((aligned(16))) unsigned char lds[kStages * kStageBytes];
  const int outputs = GATED ? p.n / 2 : p.n;
  const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int wm = wave & 1, wn = wave >> 1;
  const int blocks = (p.k + 63) / 64, steps = (blocks + 1) & ~1;  // of a tile: pairs
  const int tiles = row_tiles * col_tiles;

  struct Tile {
    int64_t row0;
    int n0;
  };
  // Eight tiles of rows share a tile of outputs in turn, so that an XCD's workgroups
  // read few of both.
  auto tile_of = [&](int turn) -> Tile {
    // The workgroups of a turn, in the order of the XCDs.
    const int count = min((int)gridDim.x, tiles - turn * (int)gridDim.x);
    const int item = turn * (int)gridDim.x + ((int)blockIdx.x < count ? xcd_remap((int)blockIdx.x, count) : 0);
    constexpr int kGroup = 8;
    const int band = item / (kGroup * col_tiles), first = band * kGroup, within = item - first * col_tiles;
    const int tall = min(kGroup, row_tiles - first);
    return {(int64_t)(first + within % tall) * kLargeTile, within / tall * (GATED ? kLargeTile / 2 : kLargeTile)};
  };
  const int turns = tiles / (int)gridDim.x + ((int)blockIdx.x < tiles % (int)gridDim.x ? 1 : 0);

  // A wave's DMAs of a stage: four blocks of rows, four of outputs.
  uint32_t xoff[4], woff[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int block = 4 * wave + u;
    xoff[u] = (uint32_t)block * (uint32_t)blocks * 1024 + lane * 16;
    // Rows of the matrix, 16 from a multiple of 16 on but for projections behind an odd
    // number of gates.
    int r = block * 16 + i;
    if (GATED && block >= 8) r = r - 128 + outputs % 16;
    woff[u] = (uint32_t)(r / 16) * (uint32_t)blocks * 1024 + g * 256 + r % 16 * 16;
  }
  const int w_blocks = (p.n + 15) / 16;
  const uint32_t block_bytes = (uint32_t)blocks * 1024;
  __amdgpu_buffer_rsrc_t xrs, wrs;
  auto aim = [&](int turn) {
    const Tile tile = tile_of(turn);
    const int64_t row_block = tile.row0 / 16;
    const int left = (int)min((int64_t)16, (p.rows + 15) / 16 - row_block);
    xrs = buffer_rsrc(packed + row_block * blocks * 64, (uint32_t)left * block_bytes);
    const int first = (GATED && wave >= 2 ? outputs + tile.n0 : tile.n0) / 16;
    wrs = buffer_rsrc(static_cast<const char*>(p.packed) + (int64_t)first * block_bytes,
                      (uint32_t)min(17, w_blocks - first) * block_bytes);
  };
  const uint32_t lds_base = (uint32_t)(uintptr_t)lds;
  constexpr uint32_t kW = kLargeTile / 16 * kPitch;  // the outputs' blocks of a stage
  int issue_turn = 0, issue_step = 0;
  uint32_t issue_stage = 0, issue_at = 0;
  auto issue = [&](int u) {
    const uint32_t base = lds_base + issue_stage + (4 * wave + u % 4) * kPitch;
    if (u < 4)
      dma16_m0(xrs, base, xoff[u] + issue_at);
    else
      dma16_m0(wrs, base + kW, woff[u - 4] + issue_at);
  };
  auto issue_next = [&] {
    issue_stage = issue_stage == (kStages - 1) * kStageBytes ? 0 : issue_stage + kStageBytes;
    issue_at += 1024;
    if (++issue_step == steps) {
      issue_step = 0;
      issue_at = 0;
      if (++issue_turn < turns) aim(issue_turn);
    }
    if (issue_step >= blocks || issue_turn >= turns) issue_at = kNowhere;
  };

  // Operand addresses in stage 0.
  const uint32_t xaddr = (lds_base + 8 * wm * kPitch + lane * 16) & 0x3ffffu;
  const int q = i >> 2;
  uint32_t waddr[2];
  if constexpr (GATED) {
    const uint32_t at = kW + (4 * wn + (q >> 1)) * kPitch + g * 256 + (8 * (q & 1) + (i & 3)) * 16;
    waddr[0] = (lds_base + at) & 0x3ffffu;
    waddr[1] = (lds_base + at + 8 * kPitch) & 0x3ffffu;
  } else {
    const uint32_t at = kW + (8 * wn + q) * kPitch + g * 256 + (i & 3) * 16;
    waddr[0] = (lds_base + at) & 0x3ffffu;
    waddr[1] = (lds_base + at + 4 * kPitch) & 0x3ffffu;
  }
  // Product j of a wave's 128 outputs: two times 64 (gated: two times 32 gates, two
  // times 32 projections).
  auto read_w = [&](int j, uint32_t so) {
    if constexpr (GATED)
      return lds_read(waddr[(j >> 1) & 1] + so + (j >> 2) * 2 * kPitch + (j & 1) * 64);
    else
      return lds_read(waddr[j >> 2] + so + (j & 3) * 64);
  };
  i32x4_t acc[8][8], xv[8], w0[8], w1[8];
  // A stage is multiplied, whose operands are held but for the last rows', and the next
  // one's read.  A wave has 16 cycles for each product, the time of a few instructions of
  // others: those go between the products one by one (behind each eight of them a
  // stage took half as long again).
  uint32_t so = 0;
  auto half = [&](const i32x4_t* now, i32x4_t* next) {
    const uint32_t held = so;
    so = so == (kStages - 1) * kStageBytes ? 0 : so + kStageBytes;
#pragma unroll
    for (int a = 0; a < 8; ++a)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        multiply(now[j], xv[a], acc[a][j]);
        if (a == 0 && j == 1) xv[7] = lds_read(xaddr + held + 7 * kPitch);
        if (a == 0 && j == 7) {
          // The next stage has landed for every wave, and every wave has the operands of
          // the one before this, whose place the DMAs take.
          wait_vmcnt<8>();
          asm volatile("" ::: "memory");
          __builtin_amdgcn_s_barrier();
          asm volatile("" ::: "memory");
        }
        if (a > 0 && j == 1) xv[a - 1] = lds_read(xaddr + so + (a - 1) * kPitch);
        if (a > 0 && a < 5 && (j == 3 || j == 5)) next[2 * a - 2 + j / 5] = read_w(2 * a - 2 + j / 5, so);
        if (a > 0 && j == 6) issue(a - 1);
        if (a == 7 && j == 7) issue(7);
      }
    issue_next();
  };

  const T* ws = static_cast<const T*>(p.scales);
  const T* bias = static_cast<const T*>(p.bias);
  aim(0);
  for (int s = 0; s < kStages - 1; ++s) {
#pragma unroll
    for (int u = 0; u < 8; ++u) issue(u);
    issue_next();
  }
  wait_vmcnt<16>();
  __syncthreads();
#pragma unroll
  for (int a = 0; a < 8; ++a) {
    if (a < 7) xv[a] = lds_read(xaddr + a * kPitch);
    w0[a] = read_w(a, 0);
  }
  for (int turn = 0; turn < turns; ++turn) {
#pragma unroll
    for (int a = 0; a < 8; ++a)
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[a][j] = i32x4_t{0, 0, 0, 0};
    settle();
    for (int t = 0; t < steps; t += 2) {
      half(w0, w1);
      half(w1, w0);
    }
    settle();

    // (What follows is computed anew a tile: kept over the products, it would cost the
    // registers that the operands need.)
    int at_lane = lane;
    asm volatile("" : "+v"(at_lane));
    const int ri = at_lane & 15, rg = at_lane >> 4;
    const Tile tile = tile_of(turn);
    constexpr int N = GATED ? 8 : 16;
    const int64_t row_at = tile.row0 + 128 * wm + ri;
    const int n_at = tile.n0 + (GATED ? 64 : 128) * wn + N * rg;
    float rs[8], far = 0.f;
#pragma unroll
    for (int a = 0; a < 8; ++a) {
      rs[a] = row_scales[min(row_at + 16 * a, p.rows - 1)];
      far = fmaxf(far, rs[a]);
    }
    if (whole && !__any(far >= kFar)) {
      // As short as it can be, since it runs once a tile, at the pace its instructions
      // come from memory.
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int n = n_at + (GATED ? 32 : 64) * c;
        if (n >= outputs) break;
        float scale[16], add[16];
#pragma unroll
        for (int e = 0; e < 16; e += N) load_whole<T, N>(ws + (e != 0 ? outputs : 0) + n, scale + e);
        if (bias != nullptr) {
#pragma unroll
          for (int e = 0; e < 16; e += N) load_whole<T, N>(bias + (e != 0 ? outputs : 0) + n, add + e);
        }
        T* out = static_cast<T*>(p.out) + row_at * p.out_row_stride + n;
#pragma unroll
        for (int a = 0; a < 8; ++a) {
          float y[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) y[e] = (float)sum_of(acc[a][4 * c + e / 4], e % 4) * rs[a] * scale[e];
          if (bias != nullptr) {
#pragma unroll
            for (int e = 0; e < 16; ++e) y[e] += add[e];
          }
          if constexpr (GATED) {
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = silu(y[e]) * y[e + 8];
          }
          if (row_at + 16 * a < p.rows) store_whole<T, N>(out, y);
          out += 16 * p.out_row_stride;
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      continue;
    }
    // Outputs that end inside a lane's, or rows that vectors do not write: 16 rows and 64
    // outputs at a time, in a loop.
#pragma unroll 1
    for (int ca = 0; ca < 16; ++ca) {
      const int n = n_at + (GATED ? 32 : 64) * (ca / 8);
      const int64_t row = row_at + 16 * (ca % 8);
      int sums[16];
      switch (ca) {
#define ASR_SUMS(at)                                                                                            \
  case at:                                                                                                      \
    for (int e = 0; e < 16; ++e) sums[e] = sum_of(acc[at % 8][4 * (at / 8) + e / 4], e % 4);                    \
    break;
        ASR_SUMS(0) ASR_SUMS(1) ASR_SUMS(2) ASR_SUMS(3) ASR_SUMS(4) ASR_SUMS(5) ASR_SUMS(6) ASR_SUMS(7)
        ASR_SUMS(8) ASR_SUMS(9) ASR_SUMS(10) ASR_SUMS(11) ASR_SUMS(12) ASR_SUMS(13) ASR_SUMS(14)
        default:
        ASR_SUMS(15)
#undef ASR_SUMS
      }
      const float one = row_scales[min(row, p.rows - 1)];
      float y[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int at = GATED && e >= 8 ? outputs + min(n + e - 8, outputs - 1) : min(n + e, outputs - 1);
        y[e] = scaled(sums[e], one, Elem<T>::load1(ws + at));
        if (bias != nullptr) y[e] += Elem<T>::load1(bias + at);
      }
      if constexpr (GATED) {
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = silu(y[e]) * y[e + 8];
      }
      T* out = static_cast<T*>(p.out) + row * p.out_row_stride + n;
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (row < p.rows && n + e < outputs) Elem<T>::store1(out + e, y[e]);
    }
  }
  wait_vmcnt<0>();  // the surplus DMAs, before the workgroup's LDS is another's
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
    // Whether a lane's outputs are vectors, of the scales and the bias as well.
    const bool whole = (reinterpret_cast<uintptr_t>(p.out) | reinterpret_cast<uintptr_t>(p.scales) |
                        reinterpret_cast<uintptr_t>(p.bias)) % 16 == 0 &&
                       p.out_row_stride % Elem<T>::kPerVec == 0 && outputs % (p.gated ? 8 : 16) == 0;
    const long long tiles = (long long)row_tiles * col_tiles;
    const dim3 grid((unsigned)(tiles < 256 ? tiles : 256));
    if (p.gated)
      hipLaunchKernelGGL((linear8_large_kernel<T, true>), grid, dim3(256), 0, stream, p, packed, scales, row_tiles,
                         col_tiles, whole);
    else
      hipLaunchKernelGGL((linear8_large_kernel<T, false>), grid, dim3(256), 0, stream, p, packed, scales, row_tiles,
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
