// Rows through a matrix of 8-bit weights with a scale per output
// (asrlayer_linear8): the rows are rounded to 8 bits first, then multiplied as whole
// numbers on v_mfma_i32_16x16x64_i8, and the scales, the bias and the gate's
// activation happen on the sums.
//
// Both operands lie in blocks of 16 (rows, outputs) x 64 inputs, 1 KB in the order in
// which a wave's lanes take them: a load is 16 bytes a lane over whole cache lines, and
// a DMA to LDS needs no order of its own.  The outputs are the product's rows, so a lane
// holds four consecutive outputs of one row.
//
// Three ways, by the rows: few rows by workgroups of 16 outputs that read the weights to
// registers, more by tiles through LDS, of which several sizes (launch_typed says which
// and why).  One row of 2048 to 2048 outputs takes 4.5 us, of which the launch and
// two round trips to memory are most; 4099 rows of 2048 to 2 x 6144, gated, 109 to 113 us
// from card to card: 206 G operations at 1.83 to 1.89 P/s.  There the matrix cores are busy
// for 60% of the time, at a clock that their power holds near 1.7 GHz (a single workgroup
// runs at 2.3).
#include "kernels.hpp"
#include "layers.hpp"
#include "ring_common.hpp"
#include "quantize8.hpp"
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

// N consecutive elements at any address of them: global memory takes vectors there
// (2791 rows of 320 inputs to 21497 bf16 outputs 73 us, stored one by one 219; to 21504 45).
template <typename T, int N>
__device__ __forceinline__ void load_whole(const T* p, float* x) {
  constexpr int EPL = Elem<T>::kPerVec;
#pragma unroll
  for (int v = 0; v < N / EPL; ++v) {
    uint4 raw;
    __builtin_memcpy(&raw, p + v * EPL, 16);
    unpack<T>(raw, x + v * EPL);
  }
}
template <typename T, int N>
__device__ __forceinline__ void store_whole(T* p, const float* x) {
  constexpr int EPL = Elem<T>::kPerVec;
#pragma unroll
  for (int v = 0; v < N / EPL; ++v) {
    const uint4 raw = pack<T>(x + v * EPL);
    __builtin_memcpy(p + v * EPL, &raw, 16);
  }
}

// 16 inputs of a row from `at` on, zeros past k, as vectors.
template <typename T>
__device__ __forceinline__ void load_inputs(const T* row, int at, int k, uint4* raw) {
  constexpr int EPL = Elem<T>::kPerVec, kWords = 4 * (16 / EPL);
  if (__builtin_expect(at + 16 <= k, 1)) {
#pragma unroll
    for (int v = 0; v < 16 / EPL; ++v) __builtin_memcpy(raw + v, row + at + v * EPL, 16);
  } else {
    uint32_t words[kWords] = {};
#pragma unroll 1
    for (int e = 0; e < 16 && at + e < k; ++e) {
      uint32_t bits = 0;
      __builtin_memcpy(&bits, row + at + e, sizeof(T));
      if constexpr (EPL == 8) bits <<= e % 2 * 16;
#pragma unroll
      for (int i = 0; i < kWords; ++i) words[i] |= i == e * kWords / 16 ? bits : 0;
    }
#pragma unroll
    for (int v = 0; v < 16 / EPL; ++v) raw[v] = make_uint4(words[4 * v], words[4 * v + 1], words[4 * v + 2], words[4 * v + 3]);
  }
}

// 16 inputs rounded.
template <typename T>
__device__ __forceinline__ uint4 round_inputs(const uint4* raw, const Scale8& s) {
  constexpr int EPL = Elem<T>::kPerVec;
  float x[16];
  uint32_t w[4];
#pragma unroll
  for (int v = 0; v < 16 / EPL; ++v) unpack<T>(raw[v], x + v * EPL);
  bytes_of<T>(x, s, w);
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// ring::dma16 in a kernel where nothing else uses M0 (no LDS instruction of gfx950 does,
// and the compiler has no use of its own there).
__device__ __forceinline__ void dma16_m0(__amdgpu_buffer_rsrc_t rsrc, uint32_t lds_base, uint32_t voff) {
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 0\n\t"
      "buffer_load_dwordx4 %1, %2, 0 offen lds"
      :
      : "s"(lds_base), "v"(voff), "s"(rsrc)
      : "memory");
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

// LANES lanes (a wave or the workgroup) round a row, NP pieces of 16 inputs each, which
// they hold from the one reading for the largest magnitude; longer rows are read again.
// Bound by a round trip to memory, and by the bytes from some thousand rows on.  Eight
// rows share a line of the packed blocks, so an XCD takes neighbouring ones (12000 rows of
// 5120 with a product to 16 outputs 56 us; dealt out one by one, each XCD writes parts of
// every line: 81).
template <typename T, int LANES, int NP>
__global__ __launch_bounds__(kThreads) void round_rows_kernel(const asrlayer_linear8_params p, uint4* packed, float* scales) {
  const int lane = threadIdx.x % LANES;
  const int64_t row = (int64_t)xcd_remap((int)blockIdx.x, (int)gridDim.x) * (kThreads / LANES) + threadIdx.x / LANES;
  if (LANES < kThreads && row >= p.rows) return;  // (uniform over a wave)
  const T* x = static_cast<const T*>(p.x) + row * p.x_row_stride;
  const int pieces = (p.k + 15) / 16, blocks = (p.k + 63) / 64;
  constexpr int EPL = Elem<T>::kPerVec, kVecs = 16 / EPL;
  uint4 v[NP][kVecs];
  uint32_t largest = 0;
  auto take = [&](const uint4* raw) {
#pragma unroll
    for (int i = 0; i < kVecs; ++i) largest = max(largest, largest_of(raw[i], T{}));
  };
#pragma unroll
  for (int u = 0; u < NP; ++u) load_inputs(x, (lane + u * LANES) * 16, p.k, v[u]);
#pragma unroll
  for (int u = 0; u < NP; ++u) take(v[u]);
  for (int piece = lane + NP * LANES; piece < pieces; piece += LANES) {
    uint4 more[kVecs];
    load_inputs(x, piece * 16, p.k, more);
    take(more);
  }
  largest = group_umax<64>(largest);
  if constexpr (LANES == kThreads) {
    __shared__ uint32_t sm[kThreads / 64];
    if (threadIdx.x % 64 == 0) sm[threadIdx.x / 64] = largest;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) largest = max(largest, sm[w]);
  }
  const Scale8 s = scale8(largest);
  if (lane == 0) scales[row] = s.scale;
  uint4* out = packed + (row / 16) * blocks * 64 + row % 16;
  auto store = [&](int piece, const uint4* raw) {
    if (piece < pieces) out[piece * 16] = round_inputs<T>(raw, s);
  };
#pragma unroll
  for (int u = 0; u < NP; ++u) store(lane + u * LANES, v[u]);
  for (int piece = lane + NP * LANES; piece < pieces; piece += LANES) {
    uint4 more[kVecs];
    load_inputs(x, piece * 16, p.k, more);
    store(piece, more);
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

// Few rows: a workgroup takes 16 outputs (gated: and their projections) of 16 RT rows,
// its eight waves every eighth 64 inputs, whose sums meet in LDS at the end.  Bound
// by reading the weights, which go straight to registers, kAhead blocks while the ones
// before are multiplied.  FUSED: up to 16 rows whose values fit LDS are rounded there by
// every workgroup, while its first weights load, in place of a launch before it.
constexpr int kFewWaves = 8;
constexpr int kFusedValues = 16384;  // rounded by every workgroup
constexpr int kFusedBytes = kFusedValues + 16 * 64;  // rows of whole blocks

template <typename T, bool GATED, int RT, bool FUSED>
__global__ __launch_bounds__(64 * kFewWaves, 4) void linear8_few_kernel(const asrlayer_linear8_params p, const uint4* packed,
                                                                        const float* row_scales) {
  constexpr int W = kFewWaves, NW = GATED ? 2 : 1, kAhead = FUSED || RT == 1 ? 4 : 2;
  constexpr int kSums = W * NW * RT * 1024;
  __shared__ __attribute__((aligned(16))) unsigned char lds[FUSED && kFusedBytes > kSums ? kFusedBytes : kSums];
  __shared__ uint32_t sm_largest[16];
  __shared__ float sm_scale[16];
  const int outputs = GATED ? p.n / 2 : p.n;
  const int64_t row0 = (int64_t)blockIdx.y * (16 * RT);
  const int rows = (int)min(p.rows - row0, (int64_t)(16 * RT));
  const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int n0 = blockIdx.x * 16;
  const int blocks = (p.k + 63) / 64;

  // The matrix's blocks that hold the workgroup's outputs (projections behind an odd
  // number of gates lie in two), and the lane's row of them.
  __amdgpu_buffer_rsrc_t wrs[NW];
  uint32_t woff[NW];
#pragma unroll
  for (int h = 0; h < NW; ++h) {
    const int r = h * outputs + min(n0 + i, outputs - 1), first = (h * outputs + n0) / 16;
    const int held = min(2, (p.n + 15) / 16 - first);
    wrs[h] = buffer_rsrc(static_cast<const char*>(p.packed) + (int64_t)first * blocks * 1024, (uint32_t)(held * blocks) * 1024);
    woff[h] = (uint32_t)((r / 16 - first) * blocks) * 1024 + g * 256 + r % 16 * 16;
  }
  const int64_t last = (p.rows - 1) / 16;  // tile of rows (past it: repeated, not stored)
  struct Ahead {
    uint4 w[kAhead][NW];
    uint4 x[FUSED ? 1 : kAhead][FUSED ? 1 : RT];
  };
  auto load = [&](int kb, Ahead& v) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int at = kb + u * W;
      const uint32_t off = at < blocks ? (uint32_t)at * 1024 : 0x7ff00000u;  // past the last: zeros
#pragma unroll
      for (int h = 0; h < NW; ++h) v.w[u][h] = buffer_load16(wrs[h], woff[h] + off);
      if constexpr (!FUSED) {
#pragma unroll
        for (int t = 0; t < RT; ++t)
          v.x[u][t] = packed[(min(row0 / 16 + t, last) * blocks + min(at, blocks - 1)) * 64 + lane];
      }
    }
  };
  Ahead now;
  load(wave, now);

  const float* scales = row_scales + row0;
  if constexpr (FUSED) {
    // Pieces of 16 inputs, the rows' largest magnitudes first.
    const int pieces = blocks * 4, all = rows * pieces;
    if (threadIdx.x < 16) sm_largest[threadIdx.x] = 0;
    __syncthreads();
    const T* x = static_cast<const T*>(p.x);
    for (int at = threadIdx.x; at < all; at += 64 * W) {
      const int row = at / pieces, piece = at - row * pieces;
      uint4 v[16 / Elem<T>::kPerVec];
      load_inputs(x + row * p.x_row_stride, piece * 16, p.k, v);
      uint32_t largest = 0;
#pragma unroll
      for (int e = 0; e < 16 / Elem<T>::kPerVec; ++e) largest = max(largest, largest_of(v[e], T{}));
      // (A row's pieces are a multiple of four.)
      const bool wide = pieces % 16 == 0;
      largest = wide ? group_umax<16>(largest) : group_umax<4>(largest);
      if (lane % (wide ? 16 : 4) == 0) atomicMax(&sm_largest[row], largest);
    }
    __syncthreads();
    if (threadIdx.x < 16) sm_scale[threadIdx.x] = scale8(sm_largest[threadIdx.x]).scale;
    for (int at = threadIdx.x; at < all; at += 64 * W) {
      const int row = at / pieces, piece = at - row * pieces;
      uint4 v[16 / Elem<T>::kPerVec];
      load_inputs(x + row * p.x_row_stride, piece * 16, p.k, v);
      *reinterpret_cast<uint4*>(lds + (piece * rows + row) * 16) = round_inputs<T>(v, scale8(sm_largest[row]));
    }
    __syncthreads();
    scales = sm_scale;
  }
  i32x4_t acc[NW][RT] = {};
  for (int kb = wave; kb < blocks; kb += kAhead * W) {
    Ahead next;
    load(kb + kAhead * W, next);
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        uint4 x;
        if constexpr (FUSED)
          x = *reinterpret_cast<const uint4*>(lds + ((min(kb + u * W, blocks - 1) * 4 + g) * rows + min(i, rows - 1)) * 16);
        else
          x = now.x[u][t];
#pragma unroll
        for (int h = 0; h < NW; ++h)
          acc[h][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4_t, now.w[u][h]),
                                                            __builtin_bit_cast(i32x4_t, x), acc[h][t], 0, 0, 0);
      }
    now = next;
  }
  if constexpr (FUSED) __syncthreads();  // the rows are used up
  i32x4_t* const sums = reinterpret_cast<i32x4_t*>(lds);
#pragma unroll
  for (int h = 0; h < NW; ++h)
#pragma unroll
    for (int t = 0; t < RT; ++t) sums[((wave * NW + h) * RT + t) * 64 + i * 4 + g] = acc[h][t];
  __syncthreads();
  // Four outputs of a row a thread.
  const T* ws = static_cast<const T*>(p.scales);
  const T* bias = static_cast<const T*>(p.bias);
  for (int at = threadIdx.x; at < rows * 4; at += 64 * W) {
    const int row = at / 4, n = n0 + at % 4 * 4;
    i32x4_t sum[NW] = {};
#pragma unroll
    for (int w = 0; w < W; ++w)
#pragma unroll
      for (int h = 0; h < NW; ++h) sum[h] += sums[(w * NW + h) * RT * 64 + at];
    const float rs = scales[row];
    T* out = static_cast<T*>(p.out) + (row0 + row) * p.out_row_stride;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      if (n + r >= outputs) break;
      float y[NW];
#pragma unroll
      for (int h = 0; h < NW; ++h) {
        const int m = n + r + h * outputs;
        y[h] = scaled(sum[h][r], rs, Elem<T>::load1(ws + m));
        if (bias != nullptr) y[h] += Elem<T>::load1(bias + m);
      }
      Elem<T>::store1(out + n + r, GATED ? silu(y[0]) * y[NW - 1] : y[0]);
    }
  }
}

// Tiles of 32 NA rows x 32 NJ outputs (gated: half of them gates, half projections), as
// many workgroups as a CU holds, each of which takes one tile after another: four waves
// of 16 NA x 16 NJ.  Blocks of both operands, 64 inputs deep, move by DMA into a ring
// of S stages in LDS, 1 KB an instruction, and one barrier a stage separates "landed for
// every wave" from "free".  A stage's operands are read while the one before is
// multiplied, and the next tile's first stages load through the end of this one.
//
// The outputs' order inside a wave's 64 is chosen for the stores: product j's row 4 q
// + r is output 16 q + 4 j + r (gated: 8 q + 4 j + r of 32), so a lane ends with 16
// consecutive outputs of a row (8).  Its operand then takes rows of several blocks,
// which lie 64 bytes more than their size apart, so that the 16 rows a read touches at
// a time lie in different banks.
constexpr int kPitch = 1024 + 64;
// Offset of a DMA that is to write zeros.
constexpr uint32_t kNowhere = 0x7ff00000u;

template <int NA, int NJ, int S>
struct LargeShape {
  static constexpr int kRows = 32 * NA, kOutputs = 32 * NJ;
  static constexpr int kStageBytes = 2 * (NA + NJ) * kPitch;
  static constexpr int kDmas = (NA + NJ) / 2;  // of a wave and stage
  static constexpr int kPerCu = 163840 / (S * kStageBytes) < 2 ? 1 : 2;
};

template <typename T, bool GATED, int NA, int NJ, int S>
__global__ __launch_bounds__(256, (LargeShape<NA, NJ, S>::kPerCu)) void linear8_large_kernel(
    const asrlayer_linear8_params p, const uint4* packed, const float* row_scales, int row_tiles, int col_tiles) {
  using Shape = LargeShape<NA, NJ, S>;
  constexpr int kStageBytes = Shape::kStageBytes, kRows = Shape::kRows, kOutputs = Shape::kOutputs, kDmas = Shape::kDmas;
  __shared__ __attribute__((aligned(16))) unsigned char lds[S * kStageBytes];
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
    return {(int64_t)(first + within % tall) * kRows, within / tall * (GATED ? kOutputs / 2 : kOutputs)};
  };
  const int turns = tiles / (int)gridDim.x + ((int)blockIdx.x < tiles % (int)gridDim.x ? 1 : 0);

  // A wave's DMAs of a stage: NA / 2 blocks of rows, NJ / 2 of outputs.
  uint32_t xoff[NA / 2], woff[NJ / 2];
#pragma unroll
  for (int u = 0; u < NA / 2; ++u) xoff[u] = (uint32_t)(NA / 2 * wave + u) * (uint32_t)blocks * 1024 + lane * 16;
#pragma unroll
  for (int u = 0; u < NJ / 2; ++u) {
    // Rows of the matrix, 16 from a multiple of 16 on but for projections behind an odd
    // number of gates.
    const int block = NJ / 2 * wave + u;
    int r = block * 16 + i;
    if (GATED && block >= NJ) r = r - 16 * NJ + outputs % 16;
    woff[u] = (uint32_t)(r / 16) * (uint32_t)blocks * 1024 + g * 256 + r % 16 * 16;
  }
  const int w_blocks = (p.n + 15) / 16;
  const uint32_t block_bytes = (uint32_t)blocks * 1024;
  __amdgpu_buffer_rsrc_t xrs, wrs;
  auto aim = [&](int turn) {
    const Tile tile = tile_of(turn);
    const int64_t row_block = tile.row0 / 16;
    const int left = (int)min((int64_t)(2 * NA), (p.rows + 15) / 16 - row_block);
    xrs = buffer_rsrc(packed + row_block * blocks * 64, (uint32_t)left * block_bytes);
    const int first = (GATED && wave >= 2 ? outputs + tile.n0 : tile.n0) / 16;
    wrs = buffer_rsrc(static_cast<const char*>(p.packed) + (int64_t)first * block_bytes,
                      (uint32_t)min(2 * NJ + 1, w_blocks - first) * block_bytes);
  };
  const uint32_t lds_base = (uint32_t)(uintptr_t)lds;
  constexpr uint32_t kW = 2 * NA * kPitch;  // the outputs' blocks of a stage
  int issue_turn = 0, issue_step = 0;
  uint32_t issue_stage = 0, issue_at = 0;
  auto issue = [&](int u) {
    if (u < NA / 2)
      dma16_m0(xrs, lds_base + issue_stage + (NA / 2 * wave + u) * kPitch, xoff[u % (NA / 2)] + issue_at);
    else
      dma16_m0(wrs, lds_base + issue_stage + kW + (NJ / 2 * wave + u - NA / 2) * kPitch,
               woff[(u - NA / 2) % (NJ / 2)] + issue_at);
  };
  auto issue_next = [&] {
    issue_stage = issue_stage == (S - 1) * kStageBytes ? 0 : issue_stage + kStageBytes;
    issue_at += 1024;
    if (++issue_step == steps) {
      issue_step = 0;
      issue_at = 0;
      if (++issue_turn < turns) aim(issue_turn);
    }
    if (issue_step >= blocks || issue_turn >= turns) issue_at = kNowhere;
  };

  // Operand addresses in stage 0.
  const uint32_t xaddr = (lds_base + NA * wm * kPitch + lane * 16) & 0x3ffffu;
  const int q = i >> 2;
  const uint32_t waddr =
      (lds_base + kW + g * 256 + (i & 3) * 16 +
       (GATED ? (NJ / 2 * wn + (q >> 1)) * kPitch + (q & 1) * 128 : (NJ * wn + q) * kPitch)) & 0x3ffffu;
  // Product j: of 64 outputs, four of them (gated: of 32 gates two, and two of the
  // projections).
  auto read_w = [&](int j, uint32_t so) {
    if constexpr (GATED)
      return lds_read(waddr + so + (j >> 2) * 2 * kPitch + ((j >> 1) & 1) * NJ * kPitch + (j & 1) * 64);
    else
      return lds_read(waddr + so + (j >> 2) * 4 * kPitch + (j & 3) * 64);
  };
  i32x4_t acc[NA][NJ], xv[NA], w0[NJ], w1[NJ];
  // A stage is multiplied, whose operands are held but for the last rows', and the next
  // one's read.  A wave has 16 cycles for each product, the time of a few instructions of
  // others: those go between the products one by one (behind each eight of them a
  // stage took half as long again).
  uint32_t so = 0;
  auto half = [&](const i32x4_t* now, i32x4_t* next) {
    const uint32_t held = so;
    so = so == (S - 1) * kStageBytes ? 0 : so + kStageBytes;
#pragma unroll
    for (int a = 0; a < NA; ++a)
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        multiply(now[j], xv[a], acc[a][j]);
        const int m = a * NJ + j;
        if (m == 1) xv[NA - 1] = lds_read(xaddr + held + (NA - 1) * kPitch);
        if (m == NJ - 1) {
          // The next stage has landed for every wave, and every wave has the operands of
          // the one before this, whose place the DMAs take.
          wait_vmcnt<kDmas * (S - 3)>();
          asm volatile("" ::: "memory");
          __builtin_amdgcn_s_barrier();
          asm volatile("" ::: "memory");
        }
        if (a > 0 && j == 1) xv[a - 1] = lds_read(xaddr + so + (a - 1) * kPitch);
        constexpr int kReads = (NA - 1) * NJ - 3 < 4 * NJ ? (NA - 1) * NJ - 3 : 4 * NJ, kIssues = (NA - 1) * NJ - 3;
#pragma unroll
        for (int u = 0; u < NJ; ++u)
          if (m == NJ + 2 + u * kReads / NJ) next[u] = read_w(u, so);
#pragma unroll
        for (int u = 0; u < kDmas; ++u)
          if (m == NJ + 3 + u * kIssues / kDmas) issue(u);
      }
    issue_next();
  };

  const T* ws = static_cast<const T*>(p.scales);
  const T* bias = static_cast<const T*>(p.bias);
  aim(0);
  for (int s = 0; s < S - 1; ++s) {
#pragma unroll
    for (int u = 0; u < kDmas; ++u) issue(u);
    issue_next();
  }
  wait_vmcnt<kDmas * (S - 2)>();
  __syncthreads();
  for (int turn = 0; turn < turns; ++turn) {
    // (Again, behind the end of a tile, which needs the registers.)
#pragma unroll
    for (int a = 0; a < NA - 1; ++a) xv[a] = lds_read(xaddr + so + a * kPitch);
#pragma unroll
    for (int j = 0; j < NJ; ++j) w0[j] = read_w(j, so);
#pragma unroll
    for (int a = 0; a < NA; ++a)
#pragma unroll
      for (int j = 0; j < NJ; ++j) acc[a][j] = i32x4_t{0, 0, 0, 0};
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
    const int64_t row_at = tile.row0 + 16 * NA * wm + ri;
    const int n_at = tile.n0 + (GATED ? 8 : 16) * NJ * wn + N * rg;
    float rs[NA], far = 0.f;
#pragma unroll
    for (int a = 0; a < NA; ++a) {
      rs[a] = row_scales[min(row_at + 16 * a, p.rows - 1)];
      far = fmaxf(far, rs[a]);
    }
    const bool near = !__any(far >= kFar);
    if (near) {
      // As short as it can be, since it runs once a tile, at the pace its instructions
      // come from memory.
#pragma unroll
      for (int c = 0; c < NJ / 4; ++c) {
        const int n = n_at + (GATED ? 32 : 64) * c;
        if (n + N > outputs) break;
        float scale[16], add[16];
#pragma unroll
        for (int e = 0; e < 16; e += N) load_whole<T, N>(ws + (e != 0 ? outputs : 0) + n, scale + e);
        if (bias != nullptr) {
#pragma unroll
          for (int e = 0; e < 16; e += N) load_whole<T, N>(bias + (e != 0 ? outputs : 0) + n, add + e);
        }
        T* out = static_cast<T*>(p.out) + row_at * p.out_row_stride + n;
#pragma unroll
        for (int a = 0; a < NA; ++a) {
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
      if (outputs % N == 0 || tile.n0 + (GATED ? kOutputs / 2 : kOutputs) <= outputs) continue;
    }
    // Lanes inside whose outputs they end, or rows of far scales: 16 rows and 64 outputs at a
    // time, in a loop.
#pragma unroll 1
    for (int ca = 0; ca < NA * NJ / 4; ++ca) {
      const int n = n_at + (GATED ? 32 : 64) * (ca / NA);
      const int64_t row = row_at + 16 * (ca % NA);
      const bool left = row < p.rows && n < outputs && !(near && n + N <= outputs);
      if (!__any(left)) continue;
      int sums[16];
      switch (ca) {
#define ASR_SUMS(at)                                                                                            \
  case at:                                                                                                      \
    for (int e = 0; e < 16; ++e) sums[e] = sum_of(acc[at % NA][at / NA * 4 % NJ + e / 4], e % 4);               \
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
        if (left && n + e < outputs) Elem<T>::store1(out + e, y[e]);
    }
  }
  wait_vmcnt<0>();  // the surplus DMAs, before the workgroup's LDS is another's
}

template <typename T, int NA, int NJ, int S>
hipError_t launch_large(const asrlayer_linear8_params& p, const uint4* packed, const float* scales, hipStream_t stream) {
  using Shape = LargeShape<NA, NJ, S>;
  const int outputs = p.gated ? p.n / 2 : p.n, wide = p.gated ? Shape::kOutputs / 2 : Shape::kOutputs;
  const int row_tiles = (int)((p.rows + Shape::kRows - 1) / Shape::kRows), col_tiles = (outputs + wide - 1) / wide;
  const long long tiles = (long long)row_tiles * col_tiles, most = 256 * Shape::kPerCu;
  const dim3 grid((unsigned)(tiles < most ? tiles : most));
  if (p.gated)
    hipLaunchKernelGGL((linear8_large_kernel<T, true, NA, NJ, S>), grid, dim3(256), 0, stream, p, packed, scales, row_tiles,
                       col_tiles);
  else
    hipLaunchKernelGGL((linear8_large_kernel<T, false, NA, NJ, S>), grid, dim3(256), 0, stream, p, packed, scales, row_tiles,
                       col_tiles);
  return hipGetLastError();
}

template <typename T, int LANES, int NP>
hipError_t launch_round(const asrlayer_linear8_params& p, uint4* packed, float* scales, hipStream_t stream) {
  constexpr int kRows = kThreads / LANES;
  hipLaunchKernelGGL((round_rows_kernel<T, LANES, NP>), dim3((unsigned)((p.rows + kRows - 1) / kRows)), dim3(kThreads), 0,
                     stream, p, packed, scales);
  return hipGetLastError();
}

template <typename T>
hipError_t launch_rounding(const asrlayer_linear8_params& p, uint4* packed, float* scales, hipStream_t stream) {
  const int pieces = (p.k + 15) / 16;
  if (pieces <= 64) return launch_round<T, 64, 1>(p, packed, scales, stream);
  if (pieces <= 128) return launch_round<T, 64, 2>(p, packed, scales, stream);
  if (pieces <= 256) return launch_round<T, kThreads, 1>(p, packed, scales, stream);
  if (pieces <= 512) return launch_round<T, kThreads, 2>(p, packed, scales, stream);
  return launch_round<T, kThreads, 4>(p, packed, scales, stream);
}

template <typename T, int RT, bool FUSED>
hipError_t launch_few(const asrlayer_linear8_params& p, const uint4* packed, const float* scales,
                      hipStream_t stream) {
  const int outputs = p.gated ? p.n / 2 : p.n;
  const dim3 grid((outputs + 15) / 16, (unsigned)((p.rows + 16 * RT - 1) / (16 * RT))), block(64 * kFewWaves);
  if (p.gated)
    hipLaunchKernelGGL((linear8_few_kernel<T, true, RT, FUSED>), grid, block, 0, stream, p, packed, scales);
  else
    hipLaunchKernelGGL((linear8_few_kernel<T, false, RT, FUSED>), grid, block, 0, stream, p, packed, scales);
  return hipGetLastError();
}

template <typename T>
hipError_t launch_typed(const asrlayer_linear8_params& p, void* workspace, hipStream_t stream) {
  const Linear8Workspace ws = linear8_workspace(p.rows, p.n, p.k, p.gated != 0);
  uint4* packed = static_cast<uint4*>(workspace);
  float* scales = reinterpret_cast<float*>(static_cast<char*>(workspace) + ws.scales);
  const int outputs = p.gated ? p.n / 2 : p.n;
  if (ws.total == 0) return launch_few<T, 1, true>(p, nullptr, nullptr, stream);
  const hipError_t err = launch_rounding<T>(p, packed, scales, stream);
  if (err != hipSuccess) return err;
  if (p.rows <= 16) return launch_few<T, 1, false>(p, packed, scales, stream);
  if (p.rows <= 32) return launch_few<T, 2, false>(p, packed, scales, stream);
  const auto tiles = [&](int rows, int wide) { return (p.rows + rows - 1) / rows * (((long long)outputs + wide - 1) / wide); };
  // Workgroups of 16 outputs and all inputs read the rows anew each: two a CU (128 rows
  // of 2048 to 4096 outputs, 512 of them: 10.6 us, 12.5 in tiles of 64 x 128; 256 to
  // 2048, 512: 10.8 and 12.8; 200 to 4096, 1024: 15.0 and 12.7).
  if (tiles(64, 16) <= 512) return launch_few<T, 4, false>(p, packed, scales, stream);
  // Tiles of 64 x 128 while each has a CU, and a ring of eight stages, to itself (512
  // rows of 6144 to 2048: 25.9 us, 31.4 in tiles of 128 x 128; 512 of 2048 to 4096 14.2 and
  // 16.0; 576, two rounds: 20.7 and 16.2).
  const int wide = p.gated ? 64 : 128;
  if (tiles(64, wide) <= 256) return launch_large<T, 2, 4, 8>(p, packed, scales, stream);
  // Tiles of 128 x 256 against ones of 128 x 128: the same work in 92% of the time.  The card
  // holds 512 workgroups of either, two a CU, and 256 more take a CU each, so a kernel's
  // time goes up with every 256 workgroups: with an even number of steps of the smaller
  // tiles the larger ones have half as many and win, with an odd one they do half a step
  // for nothing, which they have made up for after five of their own.  2048 inputs to 4096
  // outputs, us in the larger and in the smaller tiles:
  //   3035 rows (384 of the larger)   39.5 and 37.3     3163 (400)    40.1 and 43.0
  //   5083 (640)                      58.8 and 54.9     5211 (656)    59.6 and 62.0
  //   7003 (880)                      73.2 and 72.5     7259 (912)    74.6 and 81.0
  //   9051 (1136)                     89.5 and 90.3     9307 (1168)   89.5 and 99.9
  //  10971 (1376)                    109.7 and 111.8   12379 (1552)  122.2 and 127.3
  // of 6144 inputs, gated: 640 of them 148.3 and 134.7, 656 149.3 and 154.4; 880 188.8 and
  // 185.2, 912 191.1 and 208.6; 1376 286.2 and 287.0.  Up to 256 of the larger, a CU to
  // themselves, have too few waves (1755 rows, 224: 30.6 and 27.0).
  const long long big = tiles(128, 2 * wide);
  if (big > 5 * 256 || (big > 256 && (big - 1) % 256 >= 128)) return launch_large<T, 4, 8, 3>(p, packed, scales, stream);
  return launch_large<T, 4, 4, 4>(p, packed, scales, stream);
}

}  // namespace

Linear8Workspace linear8_workspace(int64_t rows, int n, int k, bool gated) {
  // Few values are rounded by every workgroup, while a CU holds all of its workgroups at
  // once: 4 x 2048 to 2 x 6144 outputs (gated) 9.7 us, with a launch before it 10.8; 8 x
  // 2048 to 2048 5.9 and 6.7, to 8192 8.8 and 8.6; 1 x 2048 to 8192 6.9 and 8.2, to 151936
  // 64.2 and 59.8.
  if (rows <= 16 && rows * k <= kFusedValues && (gated ? n / 2 : n) <= 512 * 16) return {0, 0};
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
