// Block-scaled 8-bit values (OCP e4m3) shared by the row kernels that write
// them and the product that reads them: a block of 128 consecutive values of a
// row carries one fp32 scale s = max|y| / 448, and q = e4m3(y / s).
#pragma once

#include "common.hpp"

namespace gdn {

constexpr int kFp8Block = 128;
constexpr float kFp8Top = 448.0f;               // the largest e4m3 value
constexpr float kFp8LeastScale = 0x1p-126f;     // a block of zeros; its reciprocal is finite

// Largest magnitude over the aligned 16 lanes that hold one block, as the bits
// of |y|: ordered as integers NaN > infinity > every finite value, so a block
// with a NaN gets a NaN scale and never one of its finite values'.
__device__ __forceinline__ uint32_t block_amax(uint32_t m) {
  auto dpp = [](uint32_t x, auto ctrl) __attribute__((always_inline)) {
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), decltype(ctrl)::value, 0xf, 0xf,
                                                             false));
  };
  m = max(m, dpp(m, std::integral_constant<int, 0xB1>{}));   // quad_perm [1,0,3,2]
  m = max(m, dpp(m, std::integral_constant<int, 0x4E>{}));   // quad_perm [2,3,0,1]
  m = max(m, dpp(m, std::integral_constant<int, 0x141>{}));  // row_half_mirror
  m = max(m, dpp(m, std::integral_constant<int, 0x128>{}));  // row_ror:8
  return m;
}
__device__ __forceinline__ uint32_t abs_bits(float y) { return __float_as_uint(y) & 0x7fffffffu; }

// The scale of a block from its amax bits.  An infinity gives an infinite
// scale (q = NaN for it and 0 for its neighbours, all of which read back as
// NaN); fmaxf would turn a NaN into the least scale, hence the comparison.
__device__ __forceinline__ float block_scale(uint32_t amax_bits) {
  const float s = __uint_as_float(amax_bits) / kFp8Top;
  return s < kFp8LeastScale ? kFp8LeastScale : s;
}

// Eight values over s as e4m3: y / s rounded to fp32, then to the nearest code,
// even ones on ties.  y times 1 / s alone is off by an ulp or two, which is
// enough to take a tie to the wrong side (of 4 M bf16 values 4034 codes were the
// neighbours of y / s's).  So 1 / s gets a Newton step, and y / s one from its
// residual: in fp32 arithmetic on the CPU, for every significand of s, every
// start within an ulp and every y around a code's border, the code is the
// division's, but for the significand of ones.  That one, scales whose residuals
// could be subnormal, and those that are not finite take the division itself.
// (It costs the gated norm of 16384 x 32 x 128 2 to 5 %, 72 to 74 us and 75 to 79
// with other strides of the gate; the other row kernels, further from the vector
// units' rate, up to 2 %.)
__device__ __forceinline__ uint2 pack8_fp8(const float (&y)[8], float s) {
  float q[8];
  if (s >= 0x1p-80f && s < 0x1p+120f && (~__float_as_uint(s) & 0x7fffffu)) {
    float r = __builtin_amdgcn_rcpf(s);
    r = fmaf(fmaf(-s, r, 1.f), r, r);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float about = y[e] * r;
      q[e] = fmaf(-fmaf(about, s, -y[e]), r, about);  // signs so that -0 stays -0
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) q[e] = y[e] / s;
  }
  int lo = 0, hi = 0;
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], lo, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], lo, true);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(q[4], q[5], hi, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(q[6], q[7], hi, true);
  return make_uint2(static_cast<uint32_t>(lo), static_cast<uint32_t>(hi));
}

// Destination of quantised rows: values [rows, cols] at a row stride that is a
// multiple of 16 bytes (the bytes from cols up to the next multiple of 16 are
// written as zeros), scales [rows, ceil(cols / 128)] at any strides.
struct Fp8Rows {
  uint8_t* values;
  int64_t row_stride;
  float* scales;
  int64_t scale_row_stride, scale_block_stride;
};

// Quantise the 8 values y of row r, columns 8 vec .. 8 vec + 7 (zeros from
// cols on), held by lane vec % 16 of the aligned 16-lane group of its block.
__device__ __forceinline__ void store_fp8(const Fp8Rows& q, int64_t r, int64_t vec, int64_t cols,
                                          const float (&y)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) m = max(m, abs_bits(y[e]));
  m = block_amax(m);
  const float s = block_scale(m);
  const int64_t padded = (cols + 15) & ~int64_t{15};
  if (8 * vec < padded)
    *reinterpret_cast<uint2*>(q.values + r * q.row_stride + 8 * vec) = pack8_fp8(y, s);
  if ((vec & 15) == 0 && 8 * vec < cols)
    q.scales[r * q.scale_row_stride + (vec >> 4) * q.scale_block_stride] = s;
}

// Eight elements of a row from column c on as floats; zeros from cols on.
// VEC: cols is a multiple of 8 and the address of 16 bytes.  Without it whole
// vectors still move in pieces of 16 bytes, at whatever address they have (rows
// of 4801: 3.6 to 4.4 TB/s, 1.1 to 2.2 element by element); a row's last ones do not.
template <class T, bool VEC>
__device__ __forceinline__ void load8(const T* row, int64_t c, int64_t cols, float (&x)[8]) {
  if (c + 8 <= cols) {
    const T* at = row + c;
    if constexpr (VEC) at = static_cast<const T*>(__builtin_assume_aligned(at, 16));
    if constexpr (std::is_same_v<T, float>) {
      __builtin_memcpy(x, at, 32);
    } else {
      uint4 v;
      __builtin_memcpy(&v, at, 16);
      unpack8<T>(v, x);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = !VEC && c + e < cols ? to_f32(row[c + e]) : 0.f;
  }
}
template <class T, bool VEC>
__device__ __forceinline__ void store8(T* row, int64_t c, int64_t cols, const float (&y)[8]) {
  if (c + 8 <= cols) {
    T* at = row + c;
    if constexpr (VEC) at = static_cast<T*>(__builtin_assume_aligned(at, 16));
    if constexpr (std::is_same_v<T, float>) {
      __builtin_memcpy(at, y, 32);
    } else {
      const uint4 v = pack8_io<T>(y);
      __builtin_memcpy(at, &v, 16);
    }
  } else if constexpr (!VEC) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c + e < cols) row[c + e] = from_f32<T>(y[e]);
  }
}
// The same from a row of any dtype, at any address.
__device__ __forceinline__ void load8_any(const void* row, int dtype, int64_t c, int64_t cols, float (&x)[8]) {
  switch (dtype) {
    case GDN_BF16: return load8<bf16, false>(static_cast<const bf16*>(row), c, cols, x);
    case GDN_F16: return load8<f16, false>(static_cast<const f16*>(row), c, cols, x);
    default: return load8<float, false>(static_cast<const float*>(row), c, cols, x);
  }
}

// Whether load8 / store8 may take their 16-byte form on rows at this stride.
inline bool rows_vec(const void* p, int64_t row_stride, int64_t rows) {
  return aligned16(p) && (rows == 1 || row_stride % 8 == 0);
}

}  // namespace gdn
