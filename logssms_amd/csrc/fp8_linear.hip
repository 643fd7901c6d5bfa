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
  int64_t x_stride, w_stride, out_stride;       // of rows, elements
  int64_t xs_row, xs_block, ws_row, ws_block;   // of the scales, elements
  int M, N, K;
  int tiles_m, tiles_n;
  int wide_out;  // rows of out start at multiples of 16 bytes
};

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc_of(const void* from, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(from), 0, bytes, 0x00020000);
}
// Direct-to-LDS loads of 16 or 4 bytes per active lane: lane l lands at lds + 16 l (4 l), zeros where off is past bytes.
__device__ __forceinline__ void dma16(const void* src, uint32_t bytes, uint32_t off, void* lds) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc_of(src, bytes), (lds_void*)lds, 16, off, 0, 0, 0);
}
__device__ __forceinline__ void dma4(const void* src, uint32_t bytes, uint32_t off, void* lds) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc_of(src, bytes), (lds_void*)lds, 4, off, 0, 0, 0);
}
__device__ __forceinline__ i32x8 join(i32x4 a, i32x4 b) { return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7); }

// 16 bytes of a row from column k on, zeros from K on (K tails of the last
// block alone; the row is readable up to the next multiple of 16).
__device__ __forceinline__ i32x4 mask_tail(i32x4 v, int left) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int bytes = left - 4 * i;
    if (bytes < 4) v[i] = bytes <= 0 ? 0 : v[i] & static_cast<int>((1u << (8 * bytes)) - 1);
  }
  return v;
}
__device__ __forceinline__ i32x4 load_tail(const uint8_t* row, int k, int K) {
  const int left = K - k;
  if (left <= 0) return i32x4{0, 0, 0, 0};
  return mask_tail(*reinterpret_cast<const i32x4*>(row + k), left);
}

// ------------------------------------------------------------------ few rows
// Few tokens: the weights' bytes bound the call.  A block owns 16 columns of
// the output for 16 MT tokens; its waves split K block by block, load both
// operands straight into registers and join their sums through LDS in the
// order of the waves.
constexpr int kFewWaves = 8;

template <class OUT, int MT>
__global__ __launch_bounds__(64 * kFewWaves) void few_rows_kernel(Linear p) {
  __shared__ float part[kFewWaves][MT][64][4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 16 * MT;
  const uint8_t* w = p.w + static_cast<int64_t>(min(n0 + r, p.N - 1)) * p.w_stride;
  const uint8_t* x[MT];
  const float* xs[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const int64_t m = min(m0 + 16 * t + r, p.M - 1);
    x[t] = p.x + m * p.x_stride;
    xs[t] = p.xs + m * p.xs_row;
  }
  const float* ws = p.ws + (n0 / kFp8Block) * p.ws_row;
  const int blocks = (p.K + kFp8Block - 1) / kFp8Block;
  f32x4 acc[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int b = wave; b < blocks; b += kFewWaves) {
    const int k = b * kFp8Block + 16 * g;
    const bool whole = (b + 1) * kFp8Block <= p.K;
    auto frag = [&](const uint8_t* row) {
      if (whole)
        return join(*reinterpret_cast<const i32x4*>(row + k), *reinterpret_cast<const i32x4*>(row + k + 64));
      return join(load_tail(row, k, p.K), load_tail(row, k + 64, p.K));
    };
    const i32x8 a = frag(w);
    const float sw = ws[b * p.ws_block];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      const i32x8 bx = frag(x[t]);
      const float s = xs[t][b * p.xs_block] * sw;
      const f32x4 d = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, bx, f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[t][j] = fmaf(d[j], s, acc[t][j]);
    }
  }
#pragma unroll
  for (int t = 0; t < MT; ++t) *reinterpret_cast<f32x4*>(part[wave][t][lane]) = acc[t];
  __syncthreads();
  // wave t joins token tile t: lane (r, g) holds columns n0 + 4 g .. + 3 of token m0 + 16 t + r
  for (int t = wave; t < MT; t += kFewWaves) {
    f32x4 sum = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < kFewWaves; ++i) sum += *reinterpret_cast<const f32x4*>(part[i][t][lane]);
    const int m = m0 + 16 * t + r, n = n0 + 4 * g;
    if (m >= p.M) continue;
    OUT* out = static_cast<OUT*>(p.out) + m * p.out_stride + n;
    if (p.wide_out && n + 4 <= p.N) {
      *reinterpret_cast<uint2*>(out) = make_uint2(out_pack2<OUT>(sum[0], sum[1]), out_pack2<OUT>(sum[2], sum[3]));
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (n + j < p.N) out[j] = from_f32<OUT>(sum[j]);
    }
  }
}

// ------------------------------------------------------------------ tiles
// A block of WN x WM waves owns a tile of BN = 32 FN WN columns and BM = 32 FM
// WM tokens at a time.  Both operands of a block of K go straight to LDS, one
// step ahead of the products, rows of 128 bytes with the 16-byte chunk c of
// row r at c ^ (r / 2 % 8): a fragment read takes the same chunk of 16
// consecutive rows at a time, two rows of which fill the 64 banks, so this
// spreads them over all of the banks (c ^ (r % 8) cost 4 conflict cycles on
// each 4).  The direct loads land in lane order, so the lanes' source chunks
// are permuted instead.
template <int WN, int WM, int FN, int FM>
struct Tile {
  static constexpr int kWaves = WN * WM, kThreads = 64 * kWaves;
  static constexpr int BN = 32 * FN * WN, BM = 32 * FM * WM, kRows = BN + BM;
  static constexpr int kStage = kRows * kFp8Block + 4 * BM;  // operands, then the tokens' scales
  static constexpr int JN = BN / 8 / kWaves, JM = BM / 8 / kWaves;
  static_assert(JN * 8 * kWaves == BN && JM * 8 * kWaves == BM, "whole loads per wave");
  static_assert(kFp8Block % (32 * FN) == 0, "one row of weight scales per wave");
};

template <class OUT, int WN, int WM, int FN, int FM>
__global__ __launch_bounds__(64 * WN * WM) void tile_kernel(Linear p) {
  using T = Tile<WN, WM, FN, FM>;
  __shared__ __align__(16) uint8_t lds[2 * T::kStage];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wn = wave % WN, wm = wave / WN;
  const int blocks = (p.K + kFp8Block - 1) / kFp8Block;
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
  // What a step's loads need of tile t: its corner, and where the loads of the
  // next block of K start.
  struct Cursor {
    int t, b, m0, n0;
    const uint8_t *x, *w;
    const float* xs;
  };
  auto enter = [&](int t) {
    const int group = t / (8 * p.tiles_n), in = t - group * 8 * p.tiles_n;
    const int height = min(8, p.tiles_m - 8 * group);
    Cursor c;
    c.t = t, c.b = 0;
    c.m0 = (8 * group + in % height) * T::BM;
    c.n0 = in / height * T::BN;
    c.x = p.x + c.m0 * p.x_stride;
    c.w = p.w + c.n0 * p.w_stride;
    c.xs = p.xs + c.m0 * p.xs_row;
    return c;
  };
  auto advance = [&](Cursor& c) {
    if (c.b + 1 == blocks) {
      if (c.t + per_xcd >= last) return false;
      c = enter(c.t + per_xcd);
    } else {
      c.b += 1, c.x += kFp8Block, c.w += kFp8Block, c.xs += p.xs_block;
    }
    return true;
  };

  // The loads of one step, issued piece by piece: piece i < JN + JM brings 8
  // rows per wave, the last piece the tokens' scales.
  struct Loads {
    const void *x, *w, *xs;
    uint32_t x_bytes, w_bytes, xs_bytes;
    int width;
    uint8_t* base;
  };
  auto loads_of = [&](const Cursor& c, bool any, uint8_t* base) {  // any == false: nothing is in range
    const int width = min(kFp8Block, padded - c.b * kFp8Block);
    const int rows_n = min(T::BN, p.N - c.n0), rows_m = min(T::BM, p.M - c.m0);
    auto bytes = [&](int64_t n) { return any ? static_cast<uint32_t>(n) : 0u; };
    return Loads{c.x, c.w, c.xs, bytes((rows_m - 1) * p.x_stride + width), bytes((rows_n - 1) * p.w_stride + width),
                 bytes(((rows_m - 1) * p.xs_row + 1) * 4), width, base};
  };
  const uint32_t w_row = static_cast<uint32_t>((lane >> 3) * p.w_stride);
  const uint32_t x_row = static_cast<uint32_t>((lane >> 3) * p.x_stride);
  const uint32_t xs_at = static_cast<uint32_t>((wave * 64 + lane) * p.xs_row * 4);
  auto issue = [&](const Loads& l, int piece) {
    auto rows = [&](const void* src, uint32_t bytes, uint32_t row, int64_t stride, int group, uint8_t* dst) {
      const int from = 16 * (chunk ^ (4 * (group & 1)));
      const uint32_t off = row + from + static_cast<uint32_t>(group * 8 * stride);
      dma16(src, bytes, from >= l.width ? 0xffffff00u : off, dst + group * 1024);
    };
    if (piece < T::JN) {
      rows(l.w, l.w_bytes, w_row, p.w_stride, wave * T::JN + piece, l.base);
    } else if (piece < T::JN + T::JM) {
      rows(l.x, l.x_bytes, x_row, p.x_stride, wave * T::JM + piece - T::JN, l.base + T::BN * kFp8Block);
    } else if (wave * 64 < T::BM && (T::BM % 64 == 0 || wave * 64 + lane < T::BM)) {
      dma4(l.xs, l.xs_bytes, xs_at, l.base + T::kRows * kFp8Block + wave * 256);
    }
  };

  const int r = lane & 31, g = lane >> 5;
  f32x16 acc[FN][FM];
#pragma unroll
  for (int i = 0; i < FN; ++i)
#pragma unroll
    for (int j = 0; j < FM; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;

  int stage = 0;
  Cursor ahead = enter(first);
  {
    const Loads l = loads_of(ahead, true, lds);
#pragma unroll
    for (int i = 0; i <= T::JN + T::JM; ++i) issue(l, i);
  }
  while (true) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();  // the stage is filled, and nobody reads the other one any more
    const int b = ahead.b, m0 = ahead.m0, n0 = ahead.n0;
    const bool ends = b + 1 == blocks, more = advance(ahead);
    const Loads next = loads_of(ahead, more, lds + (stage ^ 1) * T::kStage);
    issue(next, T::JN + T::JM);
    uint8_t* base = lds + stage * T::kStage;
    if (ends && (p.K & 15)) {  // bytes past K inside the last 16 of each row
      const int left = p.K & 15, at = (p.K & (kFp8Block - 1)) >> 4;
      for (int row = threadIdx.x; row < T::kRows; row += T::kThreads) {
        i32x4* v = reinterpret_cast<i32x4*>(base + row * kFp8Block + 16 * (at ^ (row >> 1 & 7)));
        *v = mask_tail(*v, left);
      }
      __syncthreads();
    }
    auto frag = [&](int row, int half) {  // lanes (r, g): row r, bytes 64 half + 32 g .. + 31
      const uint8_t* at = base + (row + r) * kFp8Block;
      const int c = 4 * half + 2 * g;
      return join(*reinterpret_cast<const i32x4*>(at + 16 * (c ^ (r >> 1 & 7))),
                  *reinterpret_cast<const i32x4*>(at + 16 * ((c + 1) ^ (r >> 1 & 7))));
    };
    const float sw = ((const_float*)p.ws)[min((n0 + wn * FN * 32) / kFp8Block, (p.N - 1) / kFp8Block) * p.ws_row +
                                          b * p.ws_block];
    i32x8 bx[FM][2];
    float s[FM];
#pragma unroll
    for (int j = 0; j < FM; ++j) {
      const int row = (wm * FM + j) * 32;
      bx[j][0] = frag(T::BN + row, 0);
      bx[j][1] = frag(T::BN + row, 1);
      s[j] = reinterpret_cast<const float*>(base + T::kRows * kFp8Block)[row + r] * sw;
    }
    // One fragment and one product ahead: the next columns' fragments are read
    // and the next product runs while the last one's is scaled and added.
    auto promote = [&](const f32x16& d, int i, int j, int half) {
#pragma unroll
      for (int e = half; e < half + 8; ++e) acc[i][j][e] = fmaf(d[e], s[j], acc[i][j][e]);
    };
    i32x8 a[2][2];
    f32x16 d[2];
    a[0][0] = frag(wn * FN * 32, 0);
    a[0][1] = frag(wn * FN * 32, 1);
#pragma unroll
    for (int i = 0; i < FN; ++i) {
      if (i + 1 < FN) {
        a[(i + 1) & 1][0] = frag((wn * FN + i + 1) * 32, 0);
        a[(i + 1) & 1][1] = frag((wn * FN + i + 1) * 32, 1);
      }
      // the next step's loads between the products: issued at once they fill the queue and every wave waits behind it
#pragma unroll
      for (int piece = i * (T::JN + T::JM) / FN; piece < (i + 1) * (T::JN + T::JM) / FN; ++piece) issue(next, piece);
#pragma unroll
      for (int j = 0; j < FM; ++j) {
        const int at = i * FM + j;
        f32x16 zero = {};
        d[at & 1] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a[i & 1][0], bx[j][0], zero, 0, 0, 0, 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
        if (at > 0) promote(d[(at - 1) & 1], (at - 1) / FM, (at - 1) % FM, 0);
        __builtin_amdgcn_sched_barrier(0);
        d[at & 1] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a[i & 1][1], bx[j][1], d[at & 1], 0, 0, 0, 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
        if (at > 0) promote(d[(at - 1) & 1], (at - 1) / FM, (at - 1) % FM, 8);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    promote(d[(FN * FM - 1) & 1], FN - 1, FM - 1, 0);
    promote(d[(FN * FM - 1) & 1], FN - 1, FM - 1, 8);
    if (ends) {
      // registers 4 q .. 4 q + 3 hold columns 8 q + 4 g .. + 3 of token r; the halves of
      // the wave trade theirs, so that a lane stores 8 consecutive columns
#pragma unroll
      for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FM; ++j) {
          const int m = m0 + (wm * FM + j) * 32 + r;
          const int n = n0 + (wn * FN + i) * 32;
          OUT* out = static_cast<OUT*>(p.out) + m * p.out_stride + n;
#pragma unroll
          for (int q = 0; q < 4; q += 2) {
            uint32_t lo[2], hi[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              lo[e] = out_pack2<OUT>(acc[i][j][4 * q + 2 * e], acc[i][j][4 * q + 2 * e + 1]);
              hi[e] = out_pack2<OUT>(acc[i][j][4 * q + 4 + 2 * e], acc[i][j][4 * q + 5 + 2 * e]);
              const auto swapped = __builtin_amdgcn_permlane32_swap(lo[e], hi[e], false, false);
              lo[e] = swapped[0], hi[e] = swapped[1];
            }
            const uint4 v = make_uint4(lo[0], lo[1], hi[0], hi[1]);
            const int c = 8 * (q + g);
            if (m < p.M) {
              if (p.wide_out && n + c + 8 <= p.N) {
                *reinterpret_cast<uint4*>(out + c) = v;
              } else {
                const uint32_t words[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int e = 0; e < 8; ++e)
                  if (n + c + e < p.N)
                    reinterpret_cast<uint16_t*>(out)[c + e] = static_cast<uint16_t>(words[e / 2] >> (16 * (e & 1)));
              }
            }
          }
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
        }
    }
    if (!more) break;
    stage ^= 1;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no load may land in LDS that is somebody else's by then
}

template <class OUT>
int launch_linear(Linear p, hipStream_t s) {
  if (p.M <= 64) {
    const dim3 threads(64 * kFewWaves);
    auto go = [&](auto MTc) {
      constexpr int MT = decltype(MTc)::value;
      hipLaunchKernelGGL((few_rows_kernel<OUT, MT>), dim3((p.N + 15) / 16, (p.M + 16 * MT - 1) / (16 * MT)), threads, 0,
                         s, p);
    };
    if (p.M <= 16) go(std::integral_constant<int, 1>{});
    else if (p.M <= 32) go(std::integral_constant<int, 2>{});
    else go(std::integral_constant<int, 4>{});
    return GDN_LAUNCH_CHECK("gdn_fp8_linear launch");
  }
  auto go = [&](auto WNc, auto WMc, auto FNc, auto FMc) -> int {
    constexpr int WN = decltype(WNc)::value, WM = decltype(WMc)::value, FN = decltype(FNc)::value,
                  FM = decltype(FMc)::value;
    using T = Tile<WN, WM, FN, FM>;
    p.tiles_m = (p.M + T::BM - 1) / T::BM;
    p.tiles_n = (p.N + T::BN - 1) / T::BN;
    const int64_t tiles = static_cast<int64_t>(p.tiles_m) * p.tiles_n;
    GDN_REQUIRE(tiles <= 0x7fffffff / 8, "gdn_fp8_linear: too many tiles");
    constexpr int kPerCu = (160 * 1024) / (2 * T::kStage);
    const int grid = static_cast<int>(tiles < 256 * kPerCu ? (tiles + 7) / 8 * 8 : 256 * kPerCu);
    hipLaunchKernelGGL((tile_kernel<OUT, WN, WM, FN, FM>), dim3(grid), dim3(T::kThreads), 0, s, p);
    return GDN_LAUNCH_CHECK("gdn_fp8_linear launch");
  };
#define GDN_INT(v) std::integral_constant<int, v>{}
  const int64_t big = static_cast<int64_t>((p.M + 255) / 256) * ((p.N + 255) / 256);
  if (big >= 256) return go(GDN_INT(2), GDN_INT(4), GDN_INT(4), GDN_INT(2));
  return go(GDN_INT(2), GDN_INT(2), GDN_INT(2), GDN_INT(2));
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
  // the stride of a single row means nothing
  const int64_t padded = (K + 15) & ~int64_t{15};
  if (M == 1) x_row_stride = padded, xs_row_stride = 0, out_row_stride = N;
  if (N == 1) weight_row_stride = padded;
  const auto rows_ok = [](const void* ptr, int64_t rows, int64_t stride, int64_t cols) {
    return aligned16(ptr) && (rows == 1 || (stride % 16 == 0 && stride >= cols));
  };
  GDN_REQUIRE(rows_ok(x, M, x_row_stride, K) && rows_ok(weight, N, weight_row_stride, K),
              "gdn_fp8_linear: the rows of x and weight must start at multiples of 16 bytes and not overlap");
  GDN_REQUIRE(out_row_stride >= N && (reinterpret_cast<uintptr_t>(out) & 1) == 0, "gdn_fp8_linear: bad output rows");
  GDN_REQUIRE(xs_row_stride >= 0 && xs_block_stride >= 0 && ws_row_stride >= 0 && ws_block_stride >= 0,
              "gdn_fp8_linear: negative scale strides");
  // offsets inside a tile of up to 256 rows are 32-bit
  constexpr int64_t kMostStride = int64_t{1} << 23;
  if (M > 0x7fffff00 || N > 0x7fffff00 || K > 0x7fffff00 || x_row_stride > kMostStride ||
      weight_row_stride > kMostStride || xs_row_stride > kMostStride / 4) {
    set_error("gdn_fp8_linear: sizes or row strides beyond 2^23 are not covered");
    return GDN_ERR_UNSUPPORTED;
  }
  Linear p{static_cast<const uint8_t*>(x), static_cast<const uint8_t*>(weight), x_scales, weight_scales, out,
           x_row_stride, weight_row_stride, out_row_stride, xs_row_stride, xs_block_stride, ws_row_stride,
           ws_block_stride, static_cast<int>(M), static_cast<int>(N), static_cast<int>(K), 0, 0, 0};
  p.wide_out = aligned16(out) && (M == 1 || out_row_stride % 8 == 0);
  hipStream_t s = static_cast<hipStream_t>(stream);
  return out_dtype == GDN_BF16 ? launch_linear<bf16>(p, s) : launch_linear<f16>(p, s);
}
