// Root-mean-square norm of hidden states with the residual's addition, and the
// quantisation of rows to block-scaled 8 bits (fp8.hpp), by itself or as the
// output of the norm or of the gated norm:
//   h = x + residual,  y = h * rsqrt(mean(h^2) + eps) * (weight + offset),
//   out = y, residual_out = h, values / scales = quantised y.
// All of it is computed in fp32 from the io-typed inputs; h and y are rounded
// once each, where they are stored (the norm and the quantisation take the
// unrounded sums).
//
// Bound: HBM.  Per row of the add + quantise form 2 + 2 bytes per element are
// read and 1 + 2 written.  A row is held in registers between its reduction
// and its outputs, so every element is read once.
#include "fp8.hpp"

namespace gdn {
namespace {

constexpr int kThreads = 256;

struct NormRows {
  const void* x;
  const void* residual;  // NULL: none
  const void* weight;
  void* out;             // NULL: not wanted
  void* residual_out;
  Fp8Rows q;             // q.values NULL: not wanted
  int64_t rows, cols;
  int64_t x_stride, residual_stride, out_stride, residual_out_stride;
  int weight_dtype;
  float weight_offset, eps;
};

template <class T, bool VEC>
__device__ __forceinline__ void load_weight(const NormRows& p, int64_t c, float (&w)[8]) {
  if (VEC && p.weight_dtype != GDN_F32) {
    load8<T, VEC>(static_cast<const T*>(p.weight), c, p.cols, w);
  } else if (VEC) {
    load8<float, VEC>(static_cast<const float*>(p.weight), c, p.cols, w);
  } else {
    load8_any(p.weight, p.weight_dtype, c, p.cols, w);
  }
}

// x (+ residual) of row r, columns c .. c + 7.
template <class T, bool VEC>
__device__ __forceinline__ void load_sum(const NormRows& p, int64_t r, int64_t c, float (&h)[8]) {
  load8<T, VEC>(static_cast<const T*>(p.x) + r * p.x_stride, c, p.cols, h);
  if (p.residual) {
    float b[8];
    load8<T, VEC>(static_cast<const T*>(p.residual) + r * p.residual_stride, c, p.cols, b);
#pragma unroll
    for (int e = 0; e < 8; ++e) h[e] += b[e];
  }
}

template <class T, bool VEC>
__device__ __forceinline__ void store_row(const NormRows& p, int64_t r, int64_t vec, const float (&h)[8], float rn) {
  const int64_t c = 8 * vec;
  float y[8];
  load_weight<T, VEC>(p, c, y);
#pragma unroll
  for (int e = 0; e < 8; ++e) y[e] = (h[e] * rn) * (y[e] + p.weight_offset);
  if (p.residual_out) store8<T, VEC>(static_cast<T*>(p.residual_out) + r * p.residual_out_stride, c, p.cols, h);
  if (p.out) store8<T, VEC>(static_cast<T*>(p.out) + r * p.out_stride, c, p.cols, y);
  if (p.q.values) {
    // past the row's end h is 0 but weight + offset may not be finite there: the zeros are set, not computed
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = c + e < p.cols ? y[e] : 0.f;
    store_fp8(p.q, r, vec, p.cols, y);
  }
}

// L lanes of one wave per row, a vector of 8 elements per lane.
template <class T, bool VEC, int L>
__global__ __launch_bounds__(kThreads) void norm_wave_kernel(NormRows p) {
  const int lane = threadIdx.x % L;
  const int64_t r = static_cast<int64_t>(blockIdx.x) * (kThreads / L) + threadIdx.x / L;
  if (r >= p.rows) return;  // whole lane groups
  float h[8];
  float ss = 0.f;
  load_sum<T, VEC>(p, r, 8 * lane, h);
#pragma unroll
  for (int e = 0; e < 8; ++e) ss = fmaf(h[e], h[e], ss);
  const float rn = rsqrtf(head_sum<L>(ss) / static_cast<float>(p.cols) + p.eps);
  store_row<T, VEC>(p, r, lane, h, rn);
}

// One block of B threads per row; N vectors per thread are held, wider rows
// (N == 0) are read a second time for their outputs.
template <class T, bool VEC, int B, int N>
__global__ __launch_bounds__(B) void norm_block_kernel(NormRows p) {
  __shared__ float part[B / 64];
  const int t = threadIdx.x;
  const int64_t r = blockIdx.x;
  const int64_t vecs = (p.cols + kFp8Block - 1) / kFp8Block * (kFp8Block / 8);
  constexpr int kHeld = N > 0 ? N : 1;
  float h[kHeld][8];
  float ss = 0.f;
  if constexpr (N > 0) {
#pragma unroll
    for (int v = 0; v < N; ++v) load_sum<T, VEC>(p, r, 8 * (v * B + t), h[v]);
#pragma unroll
    for (int v = 0; v < N; ++v)
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = fmaf(h[v][e], h[v][e], ss);
  } else {
    for (int64_t v = t; v < vecs; v += B) {
      load_sum<T, VEC>(p, r, 8 * v, h[0]);
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = fmaf(h[0][e], h[0][e], ss);
    }
  }
  ss = head_sum<64>(ss);
  if (t % 64 == 0) part[t / 64] = ss;
  __syncthreads();
  ss = 0.f;
#pragma unroll
  for (int i = 0; i < B / 64; ++i) ss += part[i];
  const float rn = rsqrtf(ss / static_cast<float>(p.cols) + p.eps);
  if constexpr (N > 0) {
#pragma unroll
    for (int v = 0; v < N; ++v) store_row<T, VEC>(p, r, v * B + t, h[v], rn);
  } else {
    // residual_out may be the residual or x itself: an element is read and written by the same thread
    for (int64_t v = t; v < vecs; v += B) {  // whole 16-lane groups
      load_sum<T, VEC>(p, r, 8 * v, h[0]);
      store_row<T, VEC>(p, r, v, h[0], rn);
    }
  }
}

// Quantisation alone: 16 lanes per block of 128, a thread block the same 128
// columns of 16 rows, whose scales lie side by side (16 blocks of one row, each
// scale a line of its own: 4096 rows of 8192 took 22.5 us, 20.7 so).
template <class T, bool VEC>
__global__ __launch_bounds__(kThreads) void quantize_kernel(const T* x, int64_t x_stride, int64_t rows, int64_t cols,
                                                            uint32_t blocks_per_row, Fp8Rows q) {
  const unsigned group = blockIdx.x / blocks_per_row;
  const int64_t r = static_cast<int64_t>(group) * (kThreads / 16) + threadIdx.x / 16;
  if (r >= rows) return;  // whole lane groups
  const int64_t vec = static_cast<int64_t>(blockIdx.x - group * blocks_per_row) * 16 + threadIdx.x % 16;
  float y[8];
  load8<T, VEC>(x + r * x_stride, 8 * vec, cols, y);
  store_fp8(q, r, vec, cols, y);
}

struct GatedRows {
  const void* x;
  const void* gate;
  const void* weight;
  Fp8Rows q;
  int64_t tokens, heads, dim;
  int64_t x_token_stride, x_head_stride;
  int64_t gate_token_stride, gate_head_stride;
  int weight_dtype;
  float eps;
};

// Heads of 8 G channels, G a power of two: G lanes hold a head, 16 a block of
// 128 of the flattened row, and both are aligned groups of one wave.  A thread
// block takes the same columns of 16 rows (8, 4 of wider heads), as the
// quantisation does.  16384 tokens of 32 heads of 128: 74 us, 4.6 TB/s (72
// without the codes' own division; then 84 with an IEEE division in the gate and a
// block along the row: vector instructions).
template <class T, int G>
__global__ __launch_bounds__(kThreads) void gated_vec_kernel(GatedRows p, uint32_t spans_per_row) {
  constexpr int kSpan = G > 16 ? G : 16;  // lanes that must stay together
  const unsigned group = blockIdx.x / spans_per_row;
  const int64_t r = static_cast<int64_t>(group) * (kThreads / kSpan) + threadIdx.x / kSpan;
  if (r >= p.tokens) return;  // whole spans
  const int64_t vec = static_cast<int64_t>(blockIdx.x - group * spans_per_row) * kSpan + threadIdx.x % kSpan;
  const int64_t head = vec / G, c = 8 * (vec % G);
  const bool live = head < p.heads;
  float x[8] = {}, z[8] = {}, w[8] = {};
  if (live) {
    load8<T, true>(static_cast<const T*>(p.x) + r * p.x_token_stride + head * p.x_head_stride, c, p.dim, x);
    load8<T, true>(static_cast<const T*>(p.gate) + r * p.gate_token_stride + head * p.gate_head_stride, c, p.dim, z);
    load8<float, true>(static_cast<const float*>(p.weight), c, p.dim, w);
  }
  float ss = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) ss = fmaf(x[e], x[e], ss);
  const float rn = rsqrtf(head_sum<G>(ss) / static_cast<float>(p.dim) + p.eps);
  float y[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) y[e] = live ? (x[e] * rn) * w[e] * fast_silu(z[e]) : 0.f;
  store_fp8(p.q, r, vec, p.heads * p.dim, y);
}

// Any head width, dtype of the weight and alignment: a block of B threads per
// token, the heads' norms first (L lanes a head), then the row in vectors of 8,
// most of which lie within a head.  The second reading of x comes from the
// caches.  16384 tokens of 5 heads of 96: 13 us (36 element by element).
template <class T, int B, int L>
__global__ __launch_bounds__(B) void gated_any_kernel(GatedRows p) {
  extern __shared__ float rn[];  // [heads]
  const int64_t r = blockIdx.x;
  const T* x = static_cast<const T*>(p.x) + r * p.x_token_stride;
  const T* gate = static_cast<const T*>(p.gate) + r * p.gate_token_stride;
  const uint32_t heads = static_cast<uint32_t>(p.heads), dim = static_cast<uint32_t>(p.dim), cols = heads * dim;
  for (uint32_t head = threadIdx.x / L; head < heads; head += B / L) {  // whole groups of L lanes
    float ss = 0.f;
    for (uint32_t c = 8 * (threadIdx.x % L); c < dim; c += 8 * L) {
      float v[8];
      load8<T, false>(x + head * p.x_head_stride, c, dim, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = fmaf(v[e], v[e], ss);
    }
    ss = head_sum<L>(ss);
    if (threadIdx.x % L == 0) rn[head] = rsqrtf(ss / static_cast<float>(p.dim) + p.eps);
  }
  __syncthreads();
  const uint32_t vecs = (cols + kFp8Block - 1) / kFp8Block * (kFp8Block / 8);
  for (uint32_t vec = threadIdx.x; vec < vecs; vec += B) {  // whole 16-lane groups
    uint32_t head = 8 * vec / dim, c = 8 * vec - head * dim;
    float y[8];
    if (head < heads && c + 8 <= dim) {
      float z[8], w[8];
      load8<T, false>(x + head * p.x_head_stride, c, dim, y);
      load8<T, false>(gate + head * p.gate_head_stride, c, dim, z);
      load8_any(p.weight, p.weight_dtype, c, dim, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = (y[e] * rn[head]) * w[e] * fast_silu(z[e]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        y[e] = 0.f;
        if (head < heads) {
          y[e] = (to_f32(x[head * p.x_head_stride + c]) * rn[head]) * load_any(p.weight, c, p.weight_dtype) *
                 fast_silu(to_f32(gate[head * p.gate_head_stride + c]));
          if (++c == dim) c = 0, ++head;
        }
      }
    }
    store_fp8(p.q, r, vec, cols, y);
  }
}

// ---------------------------------------------------------------- launches
// A launch holds fewer than 2^32 threads.
bool grid_fits(int64_t blocks, int64_t threads) { return blocks <= 0xffffffffll / threads; }

// Lanes that take a row of the norm: one vector of 8 elements each, as far as
// they go (37 rows of 4096 in 3.7 us, 5.3 with four vectors a lane; 100000 of
// 256 in 18 us, 23 with a wave a row).
int row_lanes(int64_t cols) {
  const int64_t vecs = (cols + 7) / 8;
  for (int lanes : {16, 32, 64, 128, 256, 384, 512, 768})
    if (vecs <= lanes) return lanes;
  return 1024;
}

bool known_dtype(int d) { return d == GDN_F32 || d == GDN_BF16 || d == GDN_F16; }

template <class T, bool VEC>
int launch_norm(const NormRows& p, hipStream_t s) {
  auto wave = [&](auto Lc) {
    constexpr int L = decltype(Lc)::value;
    const int64_t blocks = (p.rows + kThreads / L - 1) / (kThreads / L);
    hipLaunchKernelGGL((norm_wave_kernel<T, VEC, L>), dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0, s, p);
  };
  auto block = [&](auto Bc, auto Nc) {
    constexpr int B = decltype(Bc)::value, N = decltype(Nc)::value;
    hipLaunchKernelGGL((norm_block_kernel<T, VEC, B, N>), dim3(static_cast<unsigned>(p.rows)), dim3(B), 0, s, p);
  };
#define GDN_INT(v) std::integral_constant<int, v>{}
  switch (row_lanes(p.cols)) {
    case 16: wave(GDN_INT(16)); break;
    case 32: wave(GDN_INT(32)); break;
    case 64: wave(GDN_INT(64)); break;
    case 128: block(GDN_INT(128), GDN_INT(1)); break;
    case 256: block(GDN_INT(256), GDN_INT(1)); break;
    case 384: block(GDN_INT(384), GDN_INT(1)); break;
    case 512: block(GDN_INT(512), GDN_INT(1)); break;
    case 768: block(GDN_INT(768), GDN_INT(1)); break;
    default:
      if (p.cols <= 8 * 1024) block(GDN_INT(1024), GDN_INT(1));
      else if (p.cols <= 16 * 1024) block(GDN_INT(1024), GDN_INT(2));
      else block(GDN_INT(1024), GDN_INT(0));
  }
  return GDN_LAUNCH_CHECK("gdn_rms_norm launch");
}

template <class T>
int launch_quantize(const T* x, int64_t x_stride, int64_t rows, int64_t cols, const Fp8Rows& q, hipStream_t s) {
  const int64_t per_row = (cols + kFp8Block - 1) / kFp8Block;
  const unsigned blocks = static_cast<unsigned>((rows + kThreads / 16 - 1) / (kThreads / 16) * per_row);
  const bool vec = cols % 8 == 0 && rows_vec(x, x_stride, rows);
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(kThreads), 0, s, x, x_stride, rows, cols,
                       static_cast<uint32_t>(per_row), q);
  };
  if (vec) go(quantize_kernel<T, true>); else go(quantize_kernel<T, false>);
  return GDN_LAUNCH_CHECK("gdn_quantize_fp8 launch");
}

template <class T>
int launch_gated(const GatedRows& p, hipStream_t s) {
  const int64_t cols = p.heads * p.dim;
  const int64_t lanes = p.dim / 8;
  const bool vec = !std::is_same_v<T, float> && p.dim % 8 == 0 && lanes <= 64 && (lanes & (lanes - 1)) == 0 &&
                   p.weight_dtype == GDN_F32 && aligned16(p.weight) && aligned16(p.x) && aligned16(p.gate) &&
                   (p.tokens == 1 || (p.x_token_stride % 8 == 0 && p.gate_token_stride % 8 == 0)) &&
                   (p.heads == 1 || (p.x_head_stride % 8 == 0 && p.gate_head_stride % 8 == 0));
  const uint32_t per_row = static_cast<uint32_t>((cols + kFp8Block - 1) / kFp8Block);
  if constexpr (!std::is_same_v<T, float>) {
    if (vec) {
      auto go = [&](auto Gc) {
        constexpr int G = decltype(Gc)::value;
        constexpr int kSpan = G > 16 ? G : 16;
        const uint32_t spans = (per_row * 16 + kSpan - 1) / kSpan;
        const unsigned blocks = static_cast<unsigned>((p.tokens + kThreads / kSpan - 1) / (kThreads / kSpan) * spans);
        hipLaunchKernelGGL((gated_vec_kernel<T, G>), dim3(blocks), dim3(kThreads), 0, s, p, spans);
      };
      switch (lanes) {
        case 1: go(GDN_INT(1)); break;
        case 2: go(GDN_INT(2)); break;
        case 4: go(GDN_INT(4)); break;
        case 8: go(GDN_INT(8)); break;
        case 16: go(GDN_INT(16)); break;
        case 32: go(GDN_INT(32)); break;
        default: go(GDN_INT(64)); break;
      }
      return GDN_LAUNCH_CHECK("gdn_rms_norm_gated_fp8 launch");
    }
  }
  // rows of up to 128 vectors take one wave, heads of up to 16 vectors 16 lanes
  GDN_REQUIRE(grid_fits(p.tokens, kThreads), "gdn_rms_norm_gated_fp8: too many tokens");
  auto any = [&](auto Bc, auto Lc) {
    constexpr int B = decltype(Bc)::value, L = decltype(Lc)::value;
    hipLaunchKernelGGL((gated_any_kernel<T, B, L>), dim3(static_cast<unsigned>(p.tokens)), dim3(B),
                       static_cast<size_t>(p.heads) * sizeof(float), s, p);
  };
  if (cols <= 1024) {
    if (p.dim <= 128) any(GDN_INT(64), GDN_INT(16)); else any(GDN_INT(64), GDN_INT(64));
  } else {
    if (p.dim <= 128) any(GDN_INT(256), GDN_INT(16)); else any(GDN_INT(256), GDN_INT(64));
  }
  return GDN_LAUNCH_CHECK("gdn_rms_norm_gated_fp8 launch");
}
#undef GDN_INT

// The checks that every destination of quantised rows shares.
int check_fp8_rows(const char* name, const Fp8Rows& q, int64_t rows, int64_t cols) {
  GDN_REQUIRE(q.values && q.scales, "%s: null values or scales", name);
  GDN_REQUIRE(aligned16(q.values) && (rows == 1 || (q.row_stride % 16 == 0 && q.row_stride >= cols)),
              "%s: the values' rows must start at multiples of 16 bytes and not overlap", name);
  GDN_REQUIRE((reinterpret_cast<uintptr_t>(q.scales) & 3) == 0, "%s: misaligned scales", name);
  return GDN_OK;
}

}  // namespace
}  // namespace gdn

extern "C" int gdn_rms_norm(const void* x, int dtype, int64_t rows, int64_t cols, int64_t x_row_stride,
                            const void* residual, int64_t residual_row_stride, const void* weight, int weight_dtype,
                            float weight_offset, float eps, void* residual_out, int64_t residual_out_row_stride,
                            void* out, int64_t out_row_stride, void* values, int64_t values_row_stride, float* scales,
                            int64_t scale_row_stride, int64_t scale_block_stride, void* stream) {
  using namespace gdn;
  GDN_REQUIRE(rows >= 0 && cols > 0, "gdn_rms_norm: bad shape (rows %lld, cols %lld)", static_cast<long long>(rows),
              static_cast<long long>(cols));
  GDN_REQUIRE(known_dtype(dtype) && known_dtype(weight_dtype), "gdn_rms_norm: unknown dtype");
  GDN_REQUIRE(cols <= 0x7fffffff && rows <= 0xffffffffll - kThreads && grid_fits(rows + kThreads / 16, row_lanes(cols)),
              "gdn_rms_norm: too many rows or columns");
  if (rows == 0) return GDN_OK;
  GDN_REQUIRE(x && weight, "gdn_rms_norm: null input");
  GDN_REQUIRE(out || values, "gdn_rms_norm: no output asked for");
  GDN_REQUIRE(!residual_out || residual, "gdn_rms_norm: residual_out without a residual");
  GDN_REQUIRE(!values == !scales, "gdn_rms_norm: values and scales come together");
  NormRows p{x, residual, weight, out, residual_out,
             {static_cast<uint8_t*>(values), values_row_stride, scales, scale_row_stride, scale_block_stride},
             rows, cols, x_row_stride, residual_row_stride, out_row_stride, residual_out_row_stride,
             weight_dtype, weight_offset, eps};
  if (values) {
    const int rc = check_fp8_rows("gdn_rms_norm", p.q, rows, cols);
    if (rc != GDN_OK) return rc;
  }
  const bool vec = cols % 8 == 0 && rows_vec(x, x_row_stride, rows) &&
                   (!residual || rows_vec(residual, residual_row_stride, rows)) && aligned16(weight) &&
                   (weight_dtype == GDN_F32 || weight_dtype == dtype) &&
                   (!out || rows_vec(out, out_row_stride, rows)) &&
                   (!residual_out || rows_vec(residual_out, residual_out_row_stride, rows));
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case GDN_BF16: return vec ? launch_norm<bf16, true>(p, s) : launch_norm<bf16, false>(p, s);
    case GDN_F16: return vec ? launch_norm<f16, true>(p, s) : launch_norm<f16, false>(p, s);
    default: return vec ? launch_norm<float, true>(p, s) : launch_norm<float, false>(p, s);
  }
}

extern "C" int gdn_quantize_fp8(const void* x, int dtype, int64_t rows, int64_t cols, int64_t x_row_stride,
                                void* values, int64_t values_row_stride, float* scales, int64_t scale_row_stride,
                                int64_t scale_block_stride, void* stream) {
  using namespace gdn;
  GDN_REQUIRE(rows >= 0 && cols > 0, "gdn_quantize_fp8: bad shape (rows %lld, cols %lld)",
              static_cast<long long>(rows), static_cast<long long>(cols));
  GDN_REQUIRE(known_dtype(dtype), "gdn_quantize_fp8: unknown dtype");
  GDN_REQUIRE(cols <= 0x7fffffff && rows <= 0x7fffffff &&
                  grid_fits((rows + 15) * ((cols + kFp8Block - 1) / kFp8Block), 16),
              "gdn_quantize_fp8: too many rows");
  if (rows == 0) return GDN_OK;
  GDN_REQUIRE(x, "gdn_quantize_fp8: null input");
  const Fp8Rows q{static_cast<uint8_t*>(values), values_row_stride, scales, scale_row_stride, scale_block_stride};
  const int rc = check_fp8_rows("gdn_quantize_fp8", q, rows, cols);
  if (rc != GDN_OK) return rc;
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case GDN_BF16: return launch_quantize(static_cast<const bf16*>(x), x_row_stride, rows, cols, q, s);
    case GDN_F16: return launch_quantize(static_cast<const f16*>(x), x_row_stride, rows, cols, q, s);
    default: return launch_quantize(static_cast<const float*>(x), x_row_stride, rows, cols, q, s);
  }
}

extern "C" int gdn_rms_norm_gated_fp8(const void* x, int dtype, int64_t tokens, int64_t heads, int64_t dim,
                                      int64_t x_token_stride, int64_t x_head_stride, const void* gate,
                                      int64_t gate_token_stride, int64_t gate_head_stride, const void* weight,
                                      int weight_dtype, float eps, void* values, int64_t values_row_stride,
                                      float* scales, int64_t scale_row_stride, int64_t scale_block_stride,
                                      void* stream) {
  using namespace gdn;
  GDN_REQUIRE(tokens >= 0 && heads > 0 && dim > 0 && heads <= 0x7fffffff && dim <= 0x7fffffff / heads,
              "gdn_rms_norm_gated_fp8: bad shape (tokens %lld, heads %lld, dim %lld)", static_cast<long long>(tokens),
              static_cast<long long>(heads), static_cast<long long>(dim));
  GDN_REQUIRE(known_dtype(dtype) && known_dtype(weight_dtype), "gdn_rms_norm_gated_fp8: unknown dtype");
  GDN_REQUIRE(tokens <= 0x7fffffff && grid_fits((tokens + 15) * ((heads * dim + kFp8Block + 511) / kFp8Block), 16),
              "gdn_rms_norm_gated_fp8: too many tokens");
  if (heads > 16384) {  // the norms of a token's heads are kept in 64 KiB of LDS
    set_error("gdn_rms_norm_gated_fp8: more than 16384 heads");
    return GDN_ERR_UNSUPPORTED;
  }
  if (tokens == 0) return GDN_OK;
  GDN_REQUIRE(x && gate && weight, "gdn_rms_norm_gated_fp8: null input");
  const GatedRows p{x, gate, weight,
                    {static_cast<uint8_t*>(values), values_row_stride, scales, scale_row_stride, scale_block_stride},
                    tokens, heads, dim, x_token_stride, x_head_stride, gate_token_stride, gate_head_stride,
                    weight_dtype, eps};
  const int rc = check_fp8_rows("gdn_rms_norm_gated_fp8", p.q, tokens, heads * dim);
  if (rc != GDN_OK) return rc;
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case GDN_BF16: return launch_gated<bf16>(p, s);
    case GDN_F16: return launch_gated<f16>(p, s);
    default: return launch_gated<float>(p, s);
  }
}
