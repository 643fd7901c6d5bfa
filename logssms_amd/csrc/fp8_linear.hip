// Matrix product of block-scaled 8-bit operands (fp8.hpp):
//   out[m, n] = sum_b xs[m, b] ws[n / 128, b] sum_{k in block b} x[m, k] w[n, k]
// with x [M, K] and w [N, K] in e4m3, b the blocks of 128 along K.
//
// The scales differ from block to block, so a block's products are summed on
// the matrix cores from zero and added to the fp32 accumulators by one fma per
// value; a matrix instruction takes a whole block (16x16x128) or half of one
// (32x32x64, two chained).  The weights are the left operand, so a lane holds
// consecutive output columns of one token: one xs per lane and wide stores.
//
// Numerics: a block's products are exact, but the 8-bit matrix instructions
// align each group of eight consecutive products to the group's largest and
// drop what falls 2^-13 below it, then add the groups in fp32 (measured with
// single products: one of 2^-13 times its group's largest is kept, one of 2^-14
// dropped).  Against the 2^-8 and 2^-11 of the output's rounding this is 2^-13
// of the largest product of each eight.
#include "fp8.hpp"

namespace gdn {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) void lds_void;
typedef const __attribute__((address_space(4))) float const_float;  // read-only data: scalar loads

struct Linear {
  const uint8_t* x;
  const uint8_t* w;
  const float* xs;
  const float* ws;
  void* out;
  int x_stride, w_stride, out_stride, xs_row;    // of rows, elements
  int64_t xs_block, ws_row, ws_block;            // of the scales, elements
  int M, N, K;
  int tiles_m, tiles_n;
  int wide_out;  // rows of out start at multiples of 16 bytes
};

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc_of(const void* from, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(from), 0, bytes, 0x00020000);
}
// Direct-to-LDS loads of 16 or 4 bytes a lane: lane l lands at lds + 16 l (4 l), zeros where off is past bytes.
__device__ __forceinline__ void dma16(const void* src, uint32_t bytes, uint32_t off, void* lds) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc_of(src, bytes), (lds_void*)lds, 16, off, 0, 0, 0);
}
__device__ __forceinline__ void dma4(const void* src, uint32_t bytes, uint32_t off, void* lds) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc_of(src, bytes), (lds_void*)lds, 4, off, 0, 0, 0);
}
// v, computed where it is used: not kept in a register across the loop around it.
__device__ __forceinline__ int here(int v) {
  asm volatile("" : "+v"(v));
  return v;
}
__device__ __forceinline__ int here_s(int v) {  // the same for a value that all lanes share
  asm volatile("" : "+s"(v));
  return v;
}
__device__ __forceinline__ i32x8 join(i32x4 a, i32x4 b) {
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

// Up to 8 columns of an output row at any even address.
__device__ __forceinline__ void store_any(uint16_t* to, i32x4 v, int columns) {
  if (columns >= 8) {
    __builtin_memcpy(to, &v, 16);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < columns) to[e] = static_cast<uint16_t>(static_cast<uint32_t>(v[e / 2]) >> (16 * (e & 1)));
  }
}
// The first `left` of 16 bytes, zeros behind them.
__device__ __forceinline__ i32x4 mask_tail(i32x4 v, int left) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int bytes = left - 4 * i;
    if (bytes < 4) v[i] = bytes <= 0 ? 0 : v[i] & static_cast<int>((1u << (8 * bytes)) - 1);
  }
  return v;
}

template <int N>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// LDS traffic between the lanes of one wave: in order in hardware, so only the compiler has to be told.
__device__ __forceinline__ void wave_fence() { asm volatile("" ::: "memory"); }
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// ------------------------------------------------------------------ few rows
// Few tokens, or few tiles: what bounds the call is how fast its bytes come in,
// not the matrix cores.  A block owns 16 NT columns of the output for 16 MT
// tokens.  Its W waves split K block by block, each with S stages of LDS of its
// own, so that no barrier stands between their loads, and join their sums
// through LDS in the order of the waves.  (Loaded straight into the registers
// of the matrix instructions, 16 lanes would touch 16 rows at a time: 512 x
// 2048 x 4096 took 36 us.)  Blocks with the same index modulo 8 share an XCD
// and its L2: each XCD takes a contiguous eighth of the tiles, those of the same
// columns side by side (whole columns to an XCD left seven of them idle where N
// is small: 16384 x 48 x 8192 in 152 us, 34 so).
template <int MT, int NT, int W, int S>
struct Few {
  static constexpr int kStage = (NT + MT) * 16 * kFp8Block + 256;  // operands, then the tokens' scales
  static constexpr int kStages = W * S * kStage, kSums = W * MT * NT * 1024;
  static constexpr int kLds = kStages > kSums ? kStages : kSums;
  static constexpr int kLoads = 2 * (NT + MT) + 1;  // per step
  static_assert(kLds <= 160 * 1024 && (S - 1) * kLoads < 64 && MT <= 4, "fits");
};

template <class OUT, int MT, int NT, int W, int S>
__global__ __launch_bounds__(64 * W, 2) void few_rows_kernel(Linear p) {
  using F = Few<MT, NT, W, S>;
  __shared__ __align__(16) uint8_t lds[F::kLds];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t tiles = static_cast<int64_t>(p.tiles_m) * p.tiles_n;
  const int xcd = blockIdx.x & 7, t = static_cast<int>(tiles * xcd / 8) + (blockIdx.x >> 3);
  if (t >= static_cast<int>(tiles * (xcd + 1) / 8)) return;  // whole block
  const int n0 = t / p.tiles_m * 16 * NT, m0 = t % p.tiles_m * 16 * MT;
  const int blocks = (p.K + kFp8Block - 1) / kFp8Block, padded = (p.K + 15) & ~15;
  const int rows_n = min(16 * NT, p.N - n0), rows_m = min(16 * MT, p.M - m0);
  uint8_t* mine = lds + wave * S * F::kStage;
  const uint8_t* w = p.w + static_cast<int64_t>(n0) * p.w_stride;
  const uint8_t* x = p.x + static_cast<int64_t>(m0) * p.x_stride;
  const float* xs = p.xs + static_cast<int64_t>(m0) * p.xs_row;
  const float* ws = p.ws + n0 / kFp8Block * p.ws_row;
  const int ws_next = (n0 / kFp8Block + 1) * kFp8Block - n0;  // columns before the next row of weight scales
  const bool ws_more = n0 / kFp8Block < (p.N - 1) / kFp8Block;

  // A load brings 8 rows, chunk c of row r to c ^ (r / 2 % 8) (the tile kernel says why).
  const int chunk = (lane & 7) ^ (lane >> 4);
  uint32_t w_at[2 * NT], x_at[2 * MT];
#pragma unroll
  for (int j = 0; j < 2 * NT; ++j)
    w_at[j] = static_cast<uint32_t>((8 * j + (lane >> 3)) * p.w_stride) + 16 * (chunk ^ (4 * (j & 1)));
#pragma unroll
  for (int j = 0; j < 2 * MT; ++j)
    x_at[j] = static_cast<uint32_t>((8 * j + (lane >> 3)) * p.x_stride) + 16 * (chunk ^ (4 * (j & 1)));
  const uint32_t xs_at = lane < 16 * MT ? static_cast<uint32_t>(lane * p.xs_row * 4) : 0xffffff00u;
  // past the last block: counted, but nothing in range
  auto load = [&](int b, int stage) __attribute__((always_inline)) {
    const int width = b < blocks ? min(kFp8Block, padded - b * kFp8Block) : 0;
    const uint32_t w_bytes = width ? static_cast<uint32_t>((rows_n - 1) * p.w_stride + width) : 0u;
    const uint32_t x_bytes = width ? static_cast<uint32_t>((rows_m - 1) * p.x_stride + width) : 0u;
    uint8_t* to = mine + stage * F::kStage;
    const bool past[2] = {16 * chunk >= width, 16 * (chunk ^ 4) >= width};
#pragma unroll
    for (int j = 0; j < 2 * NT; ++j)
      dma16(w + b * kFp8Block, w_bytes, past[j & 1] ? 0xffffff00u : w_at[j], to + j * 1024);
#pragma unroll
    for (int j = 0; j < 2 * MT; ++j)
      dma16(x + b * kFp8Block, x_bytes, past[j & 1] ? 0xffffff00u : x_at[j], to + (2 * NT + j) * 1024);
    dma4(xs + b * p.xs_block, width ? static_cast<uint32_t>(((rows_m - 1) * p.xs_row + 1) * 4) : 0u, xs_at,
         to + (NT + MT) * 2048);
  };

  const int r = lane & 15, g = lane >> 4;
  f32x4 acc[NT][MT];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < S - 1; ++i) load(wave + i * W, i);
  int stage = 0;
  for (int b = wave; b < blocks; b += W) {
    load(b + (S - 1) * W, stage == 0 ? S - 1 : stage - 1);
    const float scale[2] = {*(const_float*)(ws + b * p.ws_block),
                            *(const_float*)(ws + (ws_more ? p.ws_row : 0) + b * p.ws_block)};
    wait_loads<(S - 1) * F::kLoads>();
    const uint8_t* from = mine + stage * F::kStage;
    const bool tail = (p.K & 15) && b + 1 == blocks;
    auto frag = [&](int row) __attribute__((always_inline)) {  // lanes (r, g): row r, bytes 32 g .. + 31
      const uint8_t* of = from + (row + r) * kFp8Block;
      i32x4 lo = *reinterpret_cast<const i32x4*>(of + 16 * ((2 * g) ^ (r >> 1)));
      i32x4 hi = *reinterpret_cast<const i32x4*>(of + 16 * ((2 * g + 1) ^ (r >> 1)));
      if (tail) {  // bytes past K inside the last 16
        const int left = p.K - b * kFp8Block - 32 * g;
        lo = mask_tail(lo, left), hi = mask_tail(hi, left - 16);
      }
      return join(lo, hi);
    };
    i32x8 bx[MT];
    float sx[MT];
#pragma unroll
    for (int j = 0; j < MT; ++j) {
      bx[j] = frag(16 * (NT + j));
      sx[j] = *reinterpret_cast<const float*>(from + (NT + MT) * 2048 + 4 * (16 * j + r));
    }
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const i32x8 a = frag(16 * i);
      const float sw = 16 * i < ws_next ? scale[0] : scale[1];
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
        const f32x4 d = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, bx[j], zero, 0, 0, 0, 0, 0, 0);
        const float s = sx[j] * sw;
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][j][e] = fmaf(d[e], s, acc[i][j][e]);
      }
    }
    // the fragments are in registers before a load may overwrite their place
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    stage = stage + 1 == S ? 0 : stage + 1;
  }
  wait_loads<0>();  // those past the last block too
  lds_barrier();    // the stages are free
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j)
      *reinterpret_cast<f32x4*>(lds + ((wave * NT + i) * MT + j) * 1024 + 16 * lane) = acc[i][j];
  lds_barrier();
  // lane (r, g) of a 16 x 16 piece holds columns 4 g .. + 3 of token r
  for (int t = wave; t < NT * MT; t += W) {
    f32x4 sum = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < W; ++i) sum += *reinterpret_cast<const f32x4*>(lds + (i * NT * MT + t) * 1024 + 16 * lane);
    const int m = m0 + 16 * (t % MT) + r, n = n0 + 16 * (t / MT) + 4 * g;
    if (m >= p.M) continue;
    OUT* out = static_cast<OUT*>(p.out) + static_cast<int64_t>(m) * p.out_stride + n;
    if (p.wide_out && n + 4 <= p.N) {
      *reinterpret_cast<uint2*>(out) = make_uint2(out_pack2<OUT>(sum[0], sum[1]), out_pack2<OUT>(sum[2], sum[3]));
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n + e < p.N) out[e] = from_f32<OUT>(sum[e]);
    }
  }
}

// ------------------------------------------------------------------ tiles
// A block of WN x WM waves owns a tile of BN = 32 FN WN columns and BM = 32 FM
// WM tokens at a time.  Both operands of a block of K go straight to LDS, ahead
// of the products, rows of 128 bytes with the 16-byte chunk c of row r at
// c ^ (r / 2 % 8): a fragment read takes the same chunk of 16 consecutive rows
// at a time, two rows of which fill the 64 banks, so this spreads them over all
// of the banks (c ^ (r % 8) cost 4 conflict cycles on each 4).  The direct loads
// land in lane order, so the lanes' source chunks are permuted instead.
//
// What bounds it: 16384 x 12288 x 2048 takes 395 us (2.1 PFLOP/s), 8192^3 460
// (2.4): the matrix cores are busy for 53 and 62 % of the cycles, and the load
// lowers the clock to 1.8 and 1.7 GHz.  The matrix instructions with the scaling
// between them, out of registers, reach 4.8 PFLOP/s.  Of the first
// product's 406 us at the time, the output took 46, the scaling 50 and the second
// barrier 15 (each left out, by turns); loads that touch the lines of later steps
// first made it slower.  The compiled step waits where it need not: for all
// eighteen LDS reads before its first matrix instruction; for the stores of the
// last tile in the first plain step; and for every load in the steps that reload
// one of the three registers that the 256 x 256 tile spills.  Where a CU has one
// tile (256 x 12288 x 2048: 13.5 us, 16 steps) a step takes 0.49 us, 0.24 of them
// matrix instructions.  The four-stage step waits in its middle for all nine reads
// of the next step's operands, because the scalar load of the weight scale is in
// flight among them, and scalar loads can only be waited for together.
template <int WN, int WM, int FN, int FM, int S>
struct Tile {
  static constexpr int kWaves = WN * WM, kThreads = 64 * kWaves;
  static constexpr int BN = 32 * FN * WN, BM = 32 * FM * WM, kRows = BN + BM;
  // 8 rows a load, as many loads for each wave
  static constexpr int JN = BN / 8 / kWaves, JM = BM / 8 / kWaves;
  static_assert(JN * 8 * kWaves == BN && JM * 8 * kWaves == BM, "whole loads for each wave");
  // bytes of a step's operands and scales: 32 tokens' scales for a wave, in 256 bytes of its own
  static constexpr int kW = BN * kFp8Block, kX = BM * kFp8Block, kS = 256 * kWaves;
  static constexpr int kLds = S * (kW + kX + kS);
  static constexpr int kPerCu = 160 * 1024 / kLds, kPerSimd = kPerCu * kWaves / 4;  // blocks, waves
  static constexpr int kStores = 2 * FN * FM;
  // tokens (of 64 columns) of a wave that go out at a time, in place of a step's weights
  static constexpr int kPass = kW / kWaves >= 4096 ? 32 : 16, kOut = kPass * 128;
  // loads that are newer than those that have to be there when a step begins
  static constexpr int kAhead = S == 2 ? JM + 1 : (S - 3) * (JN + JM + 1);
  static_assert(kOut * kWaves <= kW && kLds <= 160 * 1024 && kAhead + kStores < 64, "fits");
  static_assert(BM <= 32 * kWaves, "the scales' loads cover the tokens");
  static_assert(kFp8Block % (32 * FN) == 0 && FN % 2 == 0, "one row of weight scales per wave");
};

template <class OUT, int WN, int WM, int FN, int FM, int S>
__global__ __launch_bounds__(64 * WN * WM, (Tile<WN, WM, FN, FM, S>::kPerSimd)) void tile_kernel(Linear p) {
  using T = Tile<WN, WM, FN, FM, S>;
  __shared__ __align__(16) uint8_t lds[T::kLds];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wn = wave % WN, wm = wave / WN;
  const int padded = (p.K + 15) & ~15;
  // of the 8 rows that a load covers, lane l brings chunk l % 8 of row l / 8, in odd groups of 8 rows the one 4 across
  const int chunk = (lane & 7) ^ (lane >> 4);

  // blocks with the same index modulo 8 share an XCD and its L2: each XCD takes
  // a contiguous range of the tiles, whose order runs over 8 token tiles first
  const int tiles = p.tiles_m * p.tiles_n;
  const int xcd = blockIdx.x & 7, per_xcd = gridDim.x >> 3;
  const int first = static_cast<int>(static_cast<int64_t>(tiles) * xcd / 8) + (blockIdx.x >> 3);
  const int last = static_cast<int>(static_cast<int64_t>(tiles) * (xcd + 1) / 8);
  if (first >= last) return;  // whole block
  auto corner = [&](int t, int& m0, int& n0) __attribute__((always_inline)) {
    const int across = here_s(p.tiles_n), down = here_s(p.tiles_m);
    const int group = t / (8 * across), in = t - group * 8 * across;
    const int height = min(8, down - 8 * group);
    m0 = (8 * group + in % height) * T::BM;
    n0 = in / height * T::BN;
  };
  // A place in the walk over the tiles and, inside a tile, over the blocks of K:
  // what the next loads need, kept in scalars that a step only adds to.
  struct Walk {
    int t, left;               // tile; columns of K from here on
    const uint8_t *w, *x;      // the tile's first rows, at the block of K
    uint32_t w_span, x_span;   // bytes from the first of them to the last
    const float *ws, *xs;      // the wave's scale of the block; the first token's
    uint32_t xs_span;
  };
  auto enter = [&](int t) __attribute__((always_inline)) {
    int m0, n0;
    corner(t, m0, n0);
    const int below = here_s(p.M) - m0, beside = here_s(p.N) - n0;
    const int rows_n = beside < T::BN ? beside : T::BN, rows_m = below < T::BM ? below : T::BM;
    return Walk{t, padded, p.w + static_cast<int64_t>(n0) * p.w_stride, p.x + static_cast<int64_t>(m0) * p.x_stride,
                static_cast<uint32_t>((rows_n - 1) * p.w_stride), static_cast<uint32_t>((rows_m - 1) * p.x_stride),
                p.ws + min((n0 + wn * FN * 32) / kFp8Block, (here_s(p.N) - 1) / kFp8Block) * p.ws_row,
                p.xs + static_cast<int64_t>(m0) * p.xs_row, static_cast<uint32_t>(((rows_m - 1) * p.xs_row + 1) * 4)};
  };
  auto step = [&](Walk& c) __attribute__((always_inline)) {
    c.left -= kFp8Block;
    c.w += kFp8Block, c.x += kFp8Block;
    c.ws += p.ws_block, c.xs += p.xs_block;
  };
  // past the end of K: to the next tile; after the last one (t >= last) the loads
  // are still issued, with nothing in range, so that every step counts the same
  auto turn = [&](Walk& c) __attribute__((always_inline)) {
    if (c.left > 0) return;
    const int t = c.t + per_xcd;
    if (t < last) c = enter(t); else c = Walk{t, 0, c.w, c.x, 0, 0, c.ws, c.xs, 0};
  };
  // The lanes' offsets of each load: 8 rows, a chunk of each per lane.
  uint32_t w_at[T::JN], x_at[T::JM];
#pragma unroll
  for (int j = 0; j < T::JN; ++j)
    w_at[j] = static_cast<uint32_t>(((wave * T::JN + j) * 8 + (lane >> 3)) * p.w_stride) +
              16 * (chunk ^ (4 * ((wave * T::JN + j) & 1)));
#pragma unroll
  for (int j = 0; j < T::JM; ++j)
    x_at[j] = static_cast<uint32_t>(((wave * T::JM + j) * 8 + (lane >> 3)) * p.x_stride) +
              16 * (chunk ^ (4 * ((wave * T::JM + j) & 1)));
  // each wave brings 32 of the tokens' scales (no branch: a branch here lets the compiler move the scaling behind
  // it, for which there are no registers)
  const uint32_t xs_at = lane < 32 ? static_cast<uint32_t>((wave * 32 + lane) * p.xs_row * 4) : 0xffffff00u;
  // whole: the step has 128 columns of K
  auto load_rows = [&](const uint8_t* src, uint32_t span, int left, bool whole, uint32_t at, int group, uint8_t* dst)
                       __attribute__((always_inline)) {
    const int width = whole ? kFp8Block : min(kFp8Block, left);
    const bool past = !whole && 16 * (chunk ^ (4 * (group & 1))) >= width;
    dma16(src, span + width, past ? 0xffffff00u : at, dst + group * 1024);
  };
  auto w_of = [&](int stage) __attribute__((always_inline)) { return lds + stage * T::kW; };
  auto x_of = [&](int stage) __attribute__((always_inline)) { return lds + S * T::kW + stage * T::kX; };
  auto scales_of = [&](int stage) __attribute__((always_inline)) { return lds + S * (T::kW + T::kX) + stage * T::kS; };
  auto load_w = [&](const Walk& c, bool whole, int j, int stage) __attribute__((always_inline)) {
    load_rows(c.w, c.w_span, c.left, whole, w_at[j], wave * T::JN + j, w_of(stage));
  };
  // the last one brings the tokens' scales
  auto load_x = [&](const Walk& c, bool whole, int j, int stage) __attribute__((always_inline)) {
    if (j < T::JM)
      load_rows(c.x, c.x_span, c.left, whole, x_at[j], wave * T::JM + j, x_of(stage));
    else
      dma4(c.xs, c.xs_span, xs_at, scales_of(stage) + wave * 256);
  };

  const int r = lane & 31, g = lane >> 5;
  f32x16 acc[FN][FM];
#pragma unroll
  for (int i = 0; i < FN; ++i)
#pragma unroll
    for (int j = 0; j < FM; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;

  // Loads run S - 1 steps ahead.  Where there are four stages or more, the next
  // step's operands have landed by the time a step begins: their first fragments
  // are read behind the step's last products, whose scaling is left to the next
  // step, so that the matrix cores do not wait at the barrier between them.  Of
  // the two stages that the largest tile has room for, the tokens' is free again
  // after a wave's first products, when their fragments are all in registers: a
  // second barrier there lets the tokens' loads run nearly two steps ahead.
  constexpr bool kDeep = S > 2;
  int stage = 0;
  bool stored = false;
  Walk now = enter(first), ahead = now, ahead_x = now;  // ahead_x: the tokens' own place where S is 2
  auto next = [&](Walk& c) __attribute__((always_inline)) {
    step(c);
    turn(c);
  };
#pragma unroll
  for (int i = 0; i < S - 1; ++i) {
#pragma unroll
    for (int j = 0; j < T::JN; ++j) load_w(ahead, false, j, i);
#pragma unroll
    for (int j = 0; j <= T::JM; ++j) load_x(ahead, false, j, i);
    next(ahead);
    next(ahead_x);
  }
  if (S == 2) {
#pragma unroll
    for (int j = 0; j <= T::JM; ++j) load_x(ahead_x, false, j, 1);
    next(ahead_x);
  }
  float sw = *(const_float*)now.ws;
  i32x8 bx[FM][2], a[2][2], bx_next[FM][2], a_next[2];  // _next: the next step's first ones
  f32x16 d[2];
  float s[FM], sx[FM], s_last = 0.f;  // s_last: of the product whose scaling is left
  auto frag = [&](const uint8_t* base, int row, int half) __attribute__((always_inline)) {
    // lanes (r, g): row r, bytes 64 half + 32 g .. + 31
    const uint8_t* of = base + (row + r) * kFp8Block;
    const int c = 4 * half + 2 * g;
    return join(*reinterpret_cast<const i32x4*>(of + 16 * (c ^ (r >> 1 & 7))),
                *reinterpret_cast<const i32x4*>(of + 16 * ((c + 1) ^ (r >> 1 & 7))));
  };
  auto read_x = [&](int stage, int j, i32x8 (&to)[FM][2]) __attribute__((always_inline)) {
    const int row = (wm * FM + j) * 32;
    to[j][0] = frag(x_of(stage), row, 0);
    to[j][1] = frag(x_of(stage), row, 1);
    sx[j] = *reinterpret_cast<const float*>(scales_of(stage) + row * 8 + r * 4);
  };
  auto read_w = [&](int stage, int i, i32x8 (&to)[2]) __attribute__((always_inline)) {
    to[0] = frag(w_of(stage), (wn * FN + i) * 32, 0);
    to[1] = frag(w_of(stage), (wn * FN + i) * 32, 1);
  };
  auto patch = [&](int stage) __attribute__((always_inline)) {  // bytes past K inside the last 16 of each row
    const int K = here_s(p.K), left = K & 15, in = (K & (kFp8Block - 1)) >> 4;
    for (int row = here(threadIdx.x); row < T::kRows; row += T::kThreads) {
      uint8_t* of = row < T::BN ? w_of(stage) + row * kFp8Block : x_of(stage) + (row - T::BN) * kFp8Block;
      i32x4* v = reinterpret_cast<i32x4*>(of + 16 * (in ^ (row >> 1 & 7)));
      *v = mask_tail(*v, left);
    }
    lds_barrier();
  };
  auto promote = [&](const f32x16& d, float s, int i, int j, int half) __attribute__((always_inline)) {
#pragma unroll
    for (int e = half; e < half + 8; ++e) acc[i][j][e] = fmaf(d[e], s, acc[i][j][e]);
  };
  constexpr int kLast = FN * FM - 1;
  if (kDeep) {
    wait_loads<T::kAhead + T::JN + T::JM + 1>();
    lds_barrier();
    if (padded <= kFp8Block && (p.K & 15)) patch(0);
#pragma unroll
    for (int j = 0; j < FM; ++j) read_x(0, j, bx);
    read_w(0, 0, a[0]);
#pragma unroll
    for (int e = 0; e < 16; ++e) d[kLast & 1][e] = 0.f;
  }
  // One step.  Plain: not a tile's last one nor the one before, and no place turns to another tile behind it.
  auto one_step = [&](auto plainc) __attribute__((always_inline)) {
    constexpr bool kPlain = decltype(plainc)::value;
    // all but the newer loads have landed; a step that is not plain leaves the last tile's stores, which are newer
    // still, in flight too (a plain one, the next step where K has more than a few blocks, waits for most of them)
    if (!kPlain && stored) wait_loads<T::kAhead + T::kStores>(); else wait_loads<T::kAhead>();
    stored = false;
    const bool ends = !kPlain && now.left <= kFp8Block;
    const int into = stage == 0 ? S - 1 : stage - 1;  // the stage that the last step has left
    const int after = stage + 1 == S ? 0 : stage + 1;
    if (kDeep) {
      asm volatile("s_barrier" ::: "memory");  // each wave's reads of the last stage were waited for by its products
      if (!kPlain && (ends ? padded : now.left - kFp8Block) <= kFp8Block && (p.K & 15)) patch(after);
    } else {
      lds_barrier();
      if (!kPlain && ends && (p.K & 15)) patch(stage);
#pragma unroll
      for (int j = 0; j < FM; ++j) read_x(stage, j, bx);
      read_w(stage, 0, a[0]);
    }
    // The loads go between the products: issued all at once they fill the queue, and every wave waits behind it.
    auto load_between = [&](int product) __attribute__((always_inline)) {
      if (S == 2) {  // weights beside the first column fragment, tokens behind the second barrier
        constexpr int kLater = (FN - 1) * FM;
        if (product < FM) {
          for (int k = product * T::JN / FM; k < (product + 1) * T::JN / FM; ++k) load_w(ahead, kPlain, k, into);
        } else {
          for (int k = (product - FM) * (T::JM + 1) / kLater; k < (product - FM + 1) * (T::JM + 1) / kLater; ++k)
            load_x(ahead_x, kPlain, k, stage);
        }
      } else {
        constexpr int kAll = T::JN + T::JM + 1;
        for (int k = product * kAll / (FN * FM); k < (product + 1) * kAll / (FN * FM); ++k) {
          if (k < T::JN) load_w(ahead, kPlain, k, into); else load_x(ahead, kPlain, k - T::JN, into);
        }
      }
    };
#pragma unroll
    for (int i = 0; i < FN; ++i) {
      if (!kDeep && i == 1) lds_barrier();  // every wave holds its tokens' fragments
      if (i + 1 < FN) read_w(stage, i + 1, a[(i + 1) & 1]);
#pragma unroll
      for (int j = 0; j < FM; ++j) {
        const int at = i * FM + j;
        const int from = at > 0 ? at - 1 : kLast;  // the product to scale and add while this one runs
        f32x16 zero = {};
        d[at & 1] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a[i & 1][0], bx[j][0], zero, 0, 0, 0, 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
        if (at == 0) {  // the scales are needed from here on; the next block's weight scale starts on its way
#pragma unroll
          for (int k = 0; k < FM; ++k) s[k] = sx[k] * sw;
          sw = *(const_float*)(now.ws + (ends ? 0 : p.ws_block));
        }
        load_between(at);
        if (at > 0 || kDeep) promote(d[from & 1], at > 0 ? s[from % FM] : s_last, from / FM, from % FM, 0);
        __builtin_amdgcn_sched_barrier(0);
        d[at & 1] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a[i & 1][1], bx[j][1], d[at & 1], 0, 0, 0, 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
        if (kDeep && at == 0) {
          read_w(after, 0, a_next);
#pragma unroll
          for (int k = 0; k < FM; ++k) read_x(after, k, bx_next);
        }
        if (at > 0 || kDeep) promote(d[from & 1], at > 0 ? s[from % FM] : s_last, from / FM, from % FM, 8);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    s_last = s[FM - 1];
    if (kDeep) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        a[0][h] = a_next[h];
#pragma unroll
        for (int k = 0; k < FM; ++k) bx[k][h] = bx_next[k][h];
      }
    }
    if (!kDeep || (!kPlain && ends)) {
      promote(d[kLast & 1], s_last, FN - 1, FM - 1, 0);
      promote(d[kLast & 1], s_last, FN - 1, FM - 1, 8);
    }
    if (!kPlain && ends) {
      // Registers 4 q .. 4 q + 3 hold columns 8 q + 4 g .. + 3 of token r.  The
      // halves of the wave trade theirs, so that a lane has 8 consecutive columns;
      // then kPass tokens of 64 columns at a time go through LDS and out as rows of
      // 128 bytes (as they lie, in pieces of 32 bytes, the stores took 76 us of
      // 16384 x 12288 x 2048; these take 46).  They are not kept in the L2, which
      // the end of the kernel would write back (512 x 12288 x 2048: 19.4 us, 20.4
      // through it).
      int m0, n0;
      corner(now.t, m0, n0);
      const int below = here_s(p.M) - m0, beside = here_s(p.N) - n0, stride = here_s(p.out_stride);
      const int rows = below < T::BM ? below : T::BM;
      const bool wide = here_s(p.wide_out) && (beside % 8 == 0 || beside >= T::BN);
      const int l = here(lane), r = l & 31, g = l >> 5;
      lds_barrier();  // nobody reads this step's weights any more, and no load goes there before the next barrier
      uint8_t* mine = w_of(stage) + wave * T::kOut;
      OUT* tile = static_cast<OUT*>(p.out) + static_cast<int64_t>(m0) * stride + n0;
      const auto rsrc = rsrc_of(tile, (static_cast<uint32_t>(rows - 1) * stride + (beside < T::BN ? beside : T::BN)) * 2u);
#pragma unroll
      for (int i = 0; i < FN; i += 2)
#pragma unroll
        for (int j = 0; j < FM; ++j) {
          i32x4 v[4];
#pragma unroll
          for (int q = 0; q < 8; q += 2) {
            const f32x16& from = acc[i + q / 4][j];
            uint32_t lo[2], hi[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int x = 4 * (q % 4) + 2 * e;
              lo[e] = out_pack2<OUT>(from[x], from[x + 1]);
              hi[e] = out_pack2<OUT>(from[x + 4], from[x + 5]);
              const auto swapped = __builtin_amdgcn_permlane32_swap(lo[e], hi[e], false, false);
              lo[e] = swapped[0], hi[e] = swapped[1];
            }
            v[q / 2] = i32x4{static_cast<int>(lo[0]), static_cast<int>(lo[1]), static_cast<int>(hi[0]),
                             static_cast<int>(hi[1])};  // columns 8 (q + g) .. + 7
          }
#pragma unroll
          for (int pass = 0; pass < 32 / T::kPass; ++pass) {
            if (T::kPass == 32 || r / T::kPass == pass) {
#pragma unroll
              for (int q = 0; q < 8; q += 2)
                *reinterpret_cast<i32x4*>(mine + r % T::kPass * 128 + 16 * ((q + g) ^ (r >> 1 & 7))) = v[q / 2];
            }
            wave_fence();
#pragma unroll
            for (int k = 0; k < T::kPass / 8; ++k) {  // lane l: 8 columns of row 8 k + l / 8
              const int row = 8 * k + (l >> 3), c = l & 7;
              const i32x4 out = *reinterpret_cast<const i32x4*>(mine + row * 128 + 16 * (c ^ (row >> 1 & 7)));
              const int m = (wm * FM + j) * 32 + T::kPass * pass + row, n = (wn * FN + i) * 32 + 8 * c;
              if (wide) {  // always kStores stores: rows and columns that are not there fall out of range
                const bool there = m < rows && n < beside;
                __builtin_amdgcn_raw_buffer_store_b128(
                    out, rsrc, there ? (static_cast<uint32_t>(m) * stride + n) * 2u : 0xffffff00u, 0, 2);
              } else if (m < rows) {
                store_any(reinterpret_cast<uint16_t*>(tile) + static_cast<int64_t>(m) * stride + n, out, beside - n);
              }
            }
            wave_fence();
          }
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[i][j][e] = acc[i + 1][j][e] = 0.f;
        }
      stored = wide;
      if (kDeep) {  // nothing is left to scale: the next tile's first step adds 0 * 0 (an old scale may be infinite)
#pragma unroll
        for (int e = 0; e < 16; ++e) d[kLast & 1][e] = 0.f;
        s_last = 0.f;
      }
    }
    step(now);
    step(ahead);
    step(ahead_x);
    stage = after;
    if (!kPlain) {
      turn(now);
      turn(ahead);
      turn(ahead_x);
      if (ends && now.t < last) sw = *(const_float*)now.ws;
    }
  };
  do {
    const int plain = (min(now.left - kFp8Block, min(ahead.left, S == 2 ? ahead_x.left : ahead.left)) - 1) / kFp8Block;
    for (int i = 0; i < plain; ++i) one_step(std::true_type{});
    one_step(std::false_type{});
  } while (now.t < last);
  wait_loads<0>();  // no load may land in LDS that is somebody else's by then
}

template <class OUT>
int launch_linear(Linear p, hipStream_t s) {
#define GDN_INT(v) std::integral_constant<int, v>{}
  auto few = [&](auto MTc, auto NTc, auto Wc, auto Sc) -> int {
    constexpr int MT = decltype(MTc)::value, NT = decltype(NTc)::value, W = decltype(Wc)::value, S = decltype(Sc)::value;
    p.tiles_m = (p.M + 16 * MT - 1) / (16 * MT);
    p.tiles_n = (p.N + 16 * NT - 1) / (16 * NT);
    const int64_t grid = (static_cast<int64_t>(p.tiles_m) * p.tiles_n + 7) / 8 * 8;
    GDN_REQUIRE(grid <= 0xffffffffll / (64 * W), "gdn_fp8_linear: too many tiles");
    hipLaunchKernelGGL((few_rows_kernel<OUT, MT, NT, W, S>), dim3(static_cast<unsigned>(grid)), dim3(64 * W), 0, s, p);
    return GDN_LAUNCH_CHECK("gdn_fp8_linear launch");
  };
  auto go = [&](auto WNc, auto WMc, auto FNc, auto FMc, auto Sc) -> int {
    constexpr int WN = decltype(WNc)::value, WM = decltype(WMc)::value, FN = decltype(FNc)::value,
                  FM = decltype(FMc)::value, S = decltype(Sc)::value;
    using T = Tile<WN, WM, FN, FM, S>;
    p.tiles_m = (p.M + T::BM - 1) / T::BM;
    p.tiles_n = (p.N + T::BN - 1) / T::BN;
    const int64_t tiles = static_cast<int64_t>(p.tiles_m) * p.tiles_n;
    GDN_REQUIRE(tiles <= 0x7fffffff / 8, "gdn_fp8_linear: too many tiles");
    const int grid = static_cast<int>(tiles < 256 * T::kPerCu ? (tiles + 7) / 8 * 8 : 256 * T::kPerCu);
    hipLaunchKernelGGL((tile_kernel<OUT, WN, WM, FN, FM, S>), dim3(grid), dim3(T::kThreads), 0, s, p);
    return GDN_LAUNCH_CHECK("gdn_fp8_linear launch");
  };
  // Of the tiles, the smallest of which one round covers the output: at most one
  // for each of the 256 CUs.  Smaller ones repeat a round's start and end, larger
  // ones leave CUs idle.  us by tokens x columns of the tile, the chosen first:
  //   1 x 12288 x 2048       16 x 64: 7.2    32 x 64: 7.3     16 x 32: 8.6
  //   32 x 2048 x 4096       16 x 16: 5.3    16 x 32: 5.6     32 x 32: 6.3
  //   128 x 2048 x 4096      32 x 32: 6.8    32 x 64: 8.0     64 x 64: 10.4
  //   384 x 2048 x 4096      48 x 64: 9.7    64 x 64: 10.9    32 x 64: 14.4
  //   512 x 2048 x 4096      64 x 64: 11.1   32 x 64: 15.1    64 x 128: 16.9
  //   539 x 2048 x 4096      64 x 80: 12.2   64 x 64: 18.2    64 x 128: 16.9
  //   64 x 18000 x 2048      64 x 128: 11.5  64 x 80: 12.0
  //   64 x 12288 x 2048      64 x 64: 9.2    64 x 128: 10.7   32 x 64: 11.0
  //   128 x 12288 x 2048     64 x 128: 11.0  64 x 64: 14.4
  //   1024 x 2048 x 4096     64 x 128: 17.7  128 x 128: 20.7
  //   256 x 12288 x 2048     128 x 128: 13.5 two a CU: 15.0   64 x 128: 18.8
  const auto tiles = [&](int m, int n) {
    return static_cast<int64_t>((p.M + m - 1) / m) * ((p.N + n - 1) / n);
  };
  constexpr int kCus = 256;
  if (tiles(16, 16) <= kCus) return few(GDN_INT(1), GDN_INT(1), GDN_INT(8), GDN_INT(2));
  if (tiles(16, 32) <= kCus) return few(GDN_INT(1), GDN_INT(2), GDN_INT(8), GDN_INT(2));
  if (p.M <= 16) return few(GDN_INT(1), GDN_INT(4), GDN_INT(8), GDN_INT(1));  // however many: the weights stream past
  if (tiles(32, 32) <= kCus) return few(GDN_INT(2), GDN_INT(2), GDN_INT(8), GDN_INT(2));
  if (p.M <= 32 || tiles(32, 64) <= kCus) return few(GDN_INT(2), GDN_INT(4), GDN_INT(8), GDN_INT(1));
  if (tiles(48, 64) <= kCus) return few(GDN_INT(3), GDN_INT(4), GDN_INT(8), GDN_INT(1));
  if (tiles(64, 64) <= kCus) return few(GDN_INT(4), GDN_INT(4), GDN_INT(8), GDN_INT(1));
  if (p.M > 64 && tiles(64, 80) <= kCus) return few(GDN_INT(4), GDN_INT(5), GDN_INT(8), GDN_INT(1));
  if (p.M <= 64 || tiles(64, 128) <= kCus) return go(GDN_INT(2), GDN_INT(2), GDN_INT(2), GDN_INT(1), GDN_INT(4));
  if (tiles(128, 128) <= kCus) return go(GDN_INT(2), GDN_INT(4), GDN_INT(2), GDN_INT(1), GDN_INT(4));
  // Several rounds: tiles of 256 x 256, or of 128 x 128 two to a CU.  A round of
  // the first costs 3, a round of 512 of the second 2, half a one 1 (us a step
  // of K, a tile's start and end among them: 1.75, 1.05, 0.7).  1536 x 12288 x
  // 2048: large tiles 58 us, small ones 46; 4096 x 12288 x 2048: large ones 103,
  // small ones 114.
  const int64_t large = 3 * ((tiles(256, 256) + kCus - 1) / kCus), small = tiles(128, 128), rest = small % (2 * kCus);
  if (large < 2 * (small / (2 * kCus)) + (rest > kCus ? 2 : rest > 0))
    return go(GDN_INT(2), GDN_INT(4), GDN_INT(4), GDN_INT(2), GDN_INT(2));
  return go(GDN_INT(2), GDN_INT(2), GDN_INT(2), GDN_INT(2), GDN_INT(2));
#undef GDN_INT
}

}  // namespace
}  // namespace gdn

extern "C" int gdn_fp8_linear(const void* x, int64_t x_row_stride, const float* x_scales, int64_t xs_row_stride,
                              int64_t xs_block_stride, const void* weight, int64_t weight_row_stride,
                              const float* weight_scales, int64_t ws_row_stride, int64_t ws_block_stride, int64_t M,
                              int64_t N, int64_t K, void* out, int out_dtype, int64_t out_row_stride, void* stream) {
  using namespace gdn;
  GDN_REQUIRE(M >= 0 && N > 0 && K > 0, "gdn_fp8_linear: bad shape (%lld x %lld x %lld)", static_cast<long long>(M),
              static_cast<long long>(N), static_cast<long long>(K));
  GDN_REQUIRE(out_dtype == GDN_BF16 || out_dtype == GDN_F16, "gdn_fp8_linear: the output is bf16 or f16");
  if (M == 0) return GDN_OK;
  GDN_REQUIRE(x && x_scales && weight && weight_scales && out, "gdn_fp8_linear: null input");
  // the stride of a single row means nothing: any that keeps the rows behind it out of range
  if (M == 1) x_row_stride = kFp8Block, xs_row_stride = 0, out_row_stride = 0;
  if (N == 1) weight_row_stride = kFp8Block;
  const auto rows_ok = [](const void* ptr, int64_t rows, int64_t stride, int64_t cols) {
    return aligned16(ptr) && (rows == 1 || (stride % 16 == 0 && stride >= cols));
  };
  GDN_REQUIRE(rows_ok(x, M, x_row_stride, K) && rows_ok(weight, N, weight_row_stride, K),
              "gdn_fp8_linear: the rows of x and weight must start at multiples of 16 bytes and not overlap");
  GDN_REQUIRE((M == 1 || out_row_stride >= N) && (reinterpret_cast<uintptr_t>(out) & 1) == 0,
              "gdn_fp8_linear: bad output rows");
  GDN_REQUIRE(((reinterpret_cast<uintptr_t>(x_scales) | reinterpret_cast<uintptr_t>(weight_scales)) & 3) == 0,
              "gdn_fp8_linear: misaligned scales");
  GDN_REQUIRE(xs_row_stride >= 0 && xs_block_stride >= 0 && ws_row_stride >= 0 && ws_block_stride >= 0,
              "gdn_fp8_linear: negative scale strides");
  // offsets inside a tile of up to 256 rows are 32-bit
  constexpr int64_t kMostStride = int64_t{1} << 23, kMost = 0x7ffff000;  // rounded up to a tile: still an int
  if (M > kMost || N > kMost || K > kMost || x_row_stride > kMostStride ||
      weight_row_stride > kMostStride || out_row_stride > kMostStride / 2 || xs_row_stride > kMostStride / 4) {
    set_error("gdn_fp8_linear: sizes from 2^31 - 4095 on, and strides between rows beyond 2^23 bytes of x and weight, "
              "2^22 elements of out and 2^21 of x's scales, are not covered");
    return GDN_ERR_UNSUPPORTED;
  }
  Linear p{static_cast<const uint8_t*>(x), static_cast<const uint8_t*>(weight), x_scales, weight_scales, out,
           static_cast<int>(x_row_stride), static_cast<int>(weight_row_stride), static_cast<int>(out_row_stride),
           static_cast<int>(xs_row_stride), xs_block_stride, ws_row_stride, ws_block_stride, static_cast<int>(M),
           static_cast<int>(N), static_cast<int>(K), 0, 0, 0};
  p.wide_out = aligned16(out) && (M == 1 || out_row_stride % 8 == 0);
  hipStream_t s = static_cast<hipStream_t>(stream);
  return out_dtype == GDN_BF16 ? launch_linear<bf16>(p, s) : launch_linear<f16>(p, s);
}
