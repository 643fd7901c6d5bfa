// Rotary positions, and the append of keys and values to a paged cache with the
// rotation on the way.
//
// Pair i of a head's first R channels, (x[i], x[i + R/2]) in the half layout or
// (x[2i], x[2i + 1]) interleaved, is turned by the angle 2 pi turns[i] position
// and multiplied by `scale`; the channels behind them pass through.  Angles are
// products in 64 bits of which only the fraction of a revolution is kept: off by at
// most |position turns| 2^-53 revolutions, less than fp32 holds up to positions of some
// 2^30, and there is no table to outgrow.
//
// Bound by memory: 16 bytes a lane, each value read and written once.  A block takes a
// few tokens and some or all of their heads: its cosines and sines are computed once
// into LDS, each thread keeps those of its pairs and walks over the heads, the
// loads of four of them in flight.  16384 tokens, 16/2 heads of 256, a quarter of them
// turned: 72 us, 4.2 TB/s (copies reach 4.9); appended 76 us, 4.4 TB/s; a token 5.5 us, a
// launch and a call from Python.
#include <algorithm>

#include "common.hpp"

namespace gdn {
namespace {

constexpr int kThreads = 256;
constexpr int kAngles = 2048;  // cosines and sines of a block in LDS

// Rows of one operand: [tokens, heads, dim], unit channel stride.
struct Rows {
  const void* src;
  void* dst;
  int64_t src_token, src_head, dst_token, dst_head;  // elements
  int64_t dst_page;                                  // of a cache: dst_token inside a page
};

struct Turn {
  Rows rows[3];  // q, k, v
  int first[4];  // heads before each of them
  const void* positions;
  const double* turns;
  const void* slots;  // NULL: every dst is [tokens, heads, dim]
  int positions_is64, slots_is64;
  int tokens, per_block, heads_a_block, dim, rotated, interleaved;
  Div32 page;
  int64_t capacity;  // slots of the cache
  float scale;
  int copy_rest;  // bit s: operand s has channels behind the rotated ones to copy
};

template <class T> struct Vec16 {
  static constexpr int n = 16 / sizeof(T);
  static __device__ __forceinline__ void get(uint4 raw, float (&x)[n]) { unpack8<T>(raw, x); }
  static __device__ __forceinline__ uint4 put(const float (&x)[n]) { return pack8_io<T>(x); }
};
template <> struct Vec16<float> {
  static constexpr int n = 4;
  static __device__ __forceinline__ void get(uint4 raw, float (&x)[4]) {
    x[0] = __uint_as_float(raw.x), x[1] = __uint_as_float(raw.y);
    x[2] = __uint_as_float(raw.z), x[3] = __uint_as_float(raw.w);
  }
  static __device__ __forceinline__ uint4 put(const float (&x)[4]) {
    return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
  }
};

// The pair (a, b) turned; `cs` holds scale cos and scale sin.
__device__ __forceinline__ void turn_pair(float2 cs, float& a, float& b) {
  const float x = a;
  a = x * cs.x - b * cs.y;
  b = b * cs.x + x * cs.y;
}

// WIDE: rows in pieces of 16 bytes; a unit of work is a pair of pieces (half
// layout), a piece of pairs (interleaved), or a piece behind the rotated ones.
// Otherwise (rows at odd addresses, odd dims) a unit is one pair, or one value: 16384
// tokens of 16 heads of 256 46 us and, one value further on, 151, bound by instructions for
// two bytes a lane.  Heads whose rotated part and rest are whole pieces, as most models'
// are, do not come here.
template <class T, bool WIDE>
__global__ __launch_bounds__(kThreads) void rotary_kernel(Turn p) {
  constexpr int V = WIDE ? Vec16<T>::n : 1, kHeads = 4;
  __shared__ float2 angle[kAngles];
  __shared__ int64_t place[kThreads][2];  // page and offset inside it of a token's slot; page -1: none
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * p.per_block;
  const int count = static_cast<int>(min<int64_t>(p.per_block, p.tokens - t0));
  const int half = p.rotated / 2;
  for (int i = threadIdx.x; i < count * half; i += kThreads) {
    const int t = i / half, pair = i - t * half;
    const double position = static_cast<double>(load_index64(p.positions, t0 + t, p.positions_is64));
    double turns = position * p.turns[pair];
    turns -= rint(turns);
    float s, c;
    sincospif(2.0f * static_cast<float>(turns), &s, &c);
    angle[i] = make_float2(c * p.scale, s * p.scale);
  }
  if (p.slots)
    for (int t = threadIdx.x; t < count; t += kThreads) {
      const int64_t slot = load_index64(p.slots, t0 + t, p.slots_is64);
      const bool in = slot >= 0 && slot < p.capacity;
      place[t][0] = in ? static_cast<int64_t>(p.page.div(static_cast<uint32_t>(slot))) : int64_t{-1};
      place[t][1] = in ? static_cast<int64_t>(p.page.mod(static_cast<uint32_t>(slot))) : int64_t{0};
    }
  __syncthreads();

  const int turned = WIDE && p.interleaved ? p.rotated / V : half / V;  // units of the rotated part
  const int units = turned + (p.dim - p.rotated) / V;
  const int t = units < kThreads ? threadIdx.x / units : 0;
  if (t >= count) return;
  const int64_t token = t0 + t;
  const bool stored = !p.slots || place[t][0] >= 0;
  const int first = blockIdx.y * p.heads_a_block, last = min(p.first[3], first + p.heads_a_block);
  for (int unit = threadIdx.x - t * units; unit < units; unit += units < kThreads ? units : kThreads) {
    const bool pairs = unit < turned;
    // the unit's pieces: `at`, and `half` behind it in the half layout
    const int at = !pairs ? p.rotated + (unit - turned) * V : p.interleaved && !WIDE ? 2 * unit : unit * V;
    const bool two = pairs && (!p.interleaved || !WIDE);
    const int step = p.interleaved ? 1 : half;
    float2 turn[V];
    if (pairs) {
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (!WIDE || !p.interleaved || e < V / 2) turn[e] = angle[t * half + (WIDE && p.interleaved ? at / 2 + e : unit * V + e)];
    }
    for (int base = first; base < last; base += kHeads) {
      using Piece = std::conditional_t<WIDE, uint4, T>;
      Piece a[kHeads], b[kHeads];
      T* to[kHeads];
      bool rotate[kHeads];
#pragma unroll
      for (int j = 0; j < kHeads; ++j) {
        const int head = min(base + j, last - 1);  // the same in all threads
        const int which = head < p.first[1] ? 0 : head < p.first[2] ? 1 : 2;
        const Rows& r = p.rows[which];
        const int64_t of = head - p.first[which];
        const T* from = static_cast<const T*>(r.src) + token * r.src_token + of * r.src_head + at;
        T* dst = static_cast<T*>(r.dst) + of * r.dst_head + at;
        const bool cached = p.slots && which > 0;
        dst += cached ? place[t][0] * r.dst_page + place[t][1] * r.dst_token : token * r.dst_token;
        rotate[j] = pairs && which < 2;
        const bool wanted = base + j < last && (!cached || stored) && (rotate[j] || (p.copy_rest >> which & 1));
        to[j] = wanted ? dst : nullptr;
        if (wanted) {
          a[j] = *reinterpret_cast<const Piece*>(from);
          if (two) b[j] = *reinterpret_cast<const Piece*>(from + step);
        }
      }
#pragma unroll
      for (int j = 0; j < kHeads; ++j) {
        if (!to[j]) continue;
        if (rotate[j]) {
          if constexpr (WIDE) {
            float x[V], y[V];
            Vec16<T>::get(a[j], x);
            if (p.interleaved) {
#pragma unroll
              for (int e = 0; e < V; e += 2) turn_pair(turn[e / 2], x[e], x[e + 1]);
            } else {
              Vec16<T>::get(b[j], y);
#pragma unroll
              for (int e = 0; e < V; ++e) turn_pair(turn[e], x[e], y[e]);
              b[j] = Vec16<T>::put(y);
            }
            a[j] = Vec16<T>::put(x);
          } else {
            float x = to_f32(a[j]), y = to_f32(b[j]);
            turn_pair(turn[0], x, y);
            a[j] = from_f32<T>(x), b[j] = from_f32<T>(y);
          }
        }
        *reinterpret_cast<Piece*>(to[j]) = a[j];
        if (two) *reinterpret_cast<Piece*>(to[j] + step) = b[j];
      }
    }
  }
}

int launch_turn(Turn& p, int dtype, hipStream_t stream) {
  const int size = dtype == GDN_F32 ? 4 : 2, vec = 16 / size;
  const int streams = p.first[3] > p.first[2] ? 3 : 2;
  bool wide = p.dim % vec == 0 && p.rotated % (p.interleaved ? vec : 2 * vec) == 0;
  for (int s = 0; s < streams; ++s) {
    const Rows& r = p.rows[s];
    if (p.first[s + 1] == p.first[s]) continue;
    wide = wide && aligned16(r.src) && aligned16(r.dst) &&
           ((r.src_token | r.src_head | r.dst_token | r.dst_head | r.dst_page) & (vec - 1)) == 0;
    if (s == 2 || (r.src != r.dst && p.dim > p.rotated)) p.copy_rest |= 1 << s;
  }
  // a block's tokens: as many as it has threads for the units of; its heads: the four
  // that are in flight at once, more where blocks enough remain (777 tokens of 40
  // heads, all 128 channels turned: 9.6 us with one head a block, whose cosines and
  // sines are then computed 40 times, 7.1 with four)
  const int v = wide ? vec : 1, turned = wide && p.interleaved ? p.rotated / v : p.rotated / 2 / v;
  const int units = turned + (p.dim - p.rotated) / v;
  p.per_block = std::max(1, kThreads / units);
  const int64_t blocks = (static_cast<int64_t>(p.tokens) + p.per_block - 1) / p.per_block;
  const int64_t heads = p.first[3], share = (heads * blocks + 4095) / 4096 * 4;
  p.heads_a_block = static_cast<int>(std::min<int64_t>(heads, share));
  const dim3 grid(static_cast<uint32_t>(blocks), static_cast<uint32_t>((heads + p.heads_a_block - 1) / p.heads_a_block));
  if (grid.y > 65535 || blocks >= (int64_t{1} << 24)) {  // 2^32 threads of a launch
    set_error("too many heads or tokens");
    return GDN_ERR_UNSUPPORTED;
  }
  auto go = [&](auto kernel) { kernel<<<grid, kThreads, 0, stream>>>(p); };
  switch (dtype) {
    case GDN_F32: wide ? go(rotary_kernel<float, true>) : go(rotary_kernel<float, false>); break;
    case GDN_BF16: wide ? go(rotary_kernel<bf16, true>) : go(rotary_kernel<bf16, false>); break;
    default: wide ? go(rotary_kernel<f16, true>) : go(rotary_kernel<f16, false>); break;
  }
  return GDN_LAUNCH_CHECK("rotary");
}

// Sizes shared by both entry points; GDN_OK, or the error.
int set_turn(Turn& p, int dtype, int64_t tokens, int64_t heads, int64_t dim, const void* positions, int positions_dtype,
             const double* turns, int64_t rotated, int interleaved, float scale) {
  GDN_REQUIRE(dtype == GDN_F32 || dtype == GDN_BF16 || dtype == GDN_F16, "dtype must be f32, bf16 or f16");
  GDN_REQUIRE(tokens >= 0 && tokens < (int64_t{1} << 31) && heads >= 0 && dim > 0, "bad shape");
  GDN_REQUIRE(rotated >= 0 && rotated % 2 == 0 && rotated <= dim, "the rotated channels must be an even part of the head");
  GDN_REQUIRE(tokens == 0 || rotated == 0 || (positions && turns), "null positions or frequencies");
  GDN_REQUIRE(positions_dtype == GDN_I32 || positions_dtype == GDN_I64, "positions must be int32 or int64");
  if (heads * dim >= (int64_t{1} << 24) || dim > 2 * kAngles) {
    set_error("heads x dim up to 2^24, dim up to %d", 2 * kAngles);
    return GDN_ERR_UNSUPPORTED;
  }
  p.positions = positions;
  p.positions_is64 = positions_dtype == GDN_I64;
  p.turns = turns;
  p.tokens = static_cast<int>(tokens);
  p.dim = static_cast<int>(dim);
  p.rotated = static_cast<int>(rotated);
  p.interleaved = interleaved != 0;
  p.scale = scale;
  return GDN_OK;
}

}  // namespace
}  // namespace gdn

using namespace gdn;

extern "C" int gdn_apply_rotary(const void* q, int64_t q_token_stride, int64_t q_head_stride, int64_t q_heads,
                                const void* k, int64_t k_token_stride, int64_t k_head_stride, int64_t k_heads, int dtype,
                                int64_t tokens, int64_t dim, const void* positions, int positions_dtype,
                                const double* turns, int64_t rotated, int interleaved, float scale, void* q_out,
                                int64_t q_out_token_stride, int64_t q_out_head_stride, void* k_out,
                                int64_t k_out_token_stride, int64_t k_out_head_stride, void* stream) {
  Turn p{};
  GDN_REQUIRE(q_heads >= 0 && k_heads >= 0, "bad shape");
  if (const int rc = set_turn(p, dtype, tokens, q_heads + k_heads, dim, positions, positions_dtype, turns, rotated,
                              interleaved, scale))
    return rc;
  if (tokens == 0 || q_heads + k_heads == 0) return GDN_OK;
  GDN_REQUIRE((q_heads == 0 || (q && q_out)) && (k_heads == 0 || (k && k_out)), "null rows");
  p.rows[0] = {q, q_out, q_token_stride, q_head_stride, q_out_token_stride, q_out_head_stride, 0};
  p.rows[1] = {k, k_out, k_token_stride, k_head_stride, k_out_token_stride, k_out_head_stride, 0};
  p.first[1] = static_cast<int>(q_heads);
  p.first[2] = p.first[3] = static_cast<int>(q_heads + k_heads);
  return launch_turn(p, dtype, static_cast<hipStream_t>(stream));
}

extern "C" int gdn_append_paged_kv(const void* k, int64_t k_token_stride, int64_t k_head_stride, const void* v,
                                   int64_t v_token_stride, int64_t v_head_stride, int64_t kv_heads, int dtype,
                                   int64_t tokens, int64_t dim, const void* slots, int slots_dtype, void* k_cache,
                                   int64_t k_page_stride, int64_t k_cache_token_stride, int64_t k_cache_head_stride,
                                   void* v_cache, int64_t v_page_stride, int64_t v_cache_token_stride,
                                   int64_t v_cache_head_stride, int64_t pages, int64_t page_size, const void* positions,
                                   int positions_dtype, const double* turns, int64_t rotated, int interleaved,
                                   float scale, const void* q, int64_t q_token_stride, int64_t q_head_stride,
                                   int64_t q_heads, void* q_out, int64_t q_out_token_stride, int64_t q_out_head_stride,
                                   void* stream) {
  Turn p{};
  GDN_REQUIRE(q_heads >= 0 && kv_heads > 0, "bad shape");
  if (const int rc = set_turn(p, dtype, tokens, q_heads + 2 * kv_heads, dim, positions, positions_dtype, turns, rotated,
                              interleaved, scale))
    return rc;
  GDN_REQUIRE(pages >= 0 && page_size > 0, "bad cache shape");
  GDN_REQUIRE(slots_dtype == GDN_I32 || slots_dtype == GDN_I64, "slots must be int32 or int64");
  if (page_size >= (int64_t{1} << 31) || pages * page_size >= (int64_t{1} << 31)) {
    set_error("a cache of up to 2^31 tokens");
    return GDN_ERR_UNSUPPORTED;
  }
  if (tokens == 0) return GDN_OK;
  GDN_REQUIRE(k && v && slots && (pages == 0 || (k_cache && v_cache)) && (q_heads == 0 || (q && q_out)), "null operand");
  p.rows[0] = {q, q_out, q_token_stride, q_head_stride, q_out_token_stride, q_out_head_stride, 0};
  p.rows[1] = {k, k_cache, k_token_stride, k_head_stride, k_cache_token_stride, k_cache_head_stride, k_page_stride};
  p.rows[2] = {v, v_cache, v_token_stride, v_head_stride, v_cache_token_stride, v_cache_head_stride, v_page_stride};
  p.first[1] = static_cast<int>(q_heads);
  p.first[2] = static_cast<int>(q_heads + kv_heads);
  p.first[3] = static_cast<int>(q_heads + 2 * kv_heads);
  p.slots = slots;
  p.slots_is64 = slots_dtype == GDN_I64;
  p.page = make_div32(page_size);
  p.capacity = pages * page_size;
  return launch_turn(p, dtype, static_cast<hipStream_t>(stream));
}
