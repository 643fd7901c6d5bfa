// Attention over a paged cache for a batch whose requests share prefixes.
//
//   o[t, h] = sum_p softmax_p(scale q[t, h] . k[p]) v[p],  p visible to t
//
// over the positions p of the request that token t belongs to.  The positions
// that a group of requests shares are attended once for the group: all of its
// queries are the rows of one product with the shared keys.  The positions behind
// them are attended request by request.  Each piece of that work leaves, per row,
// the running maximum m and sum l of its scores and the unnormalised sum of the
// values; a last kernel joins the pieces of a row.
//
// A row is one (token, query head): the rows of a key head are the `per` query
// heads that read it, token after token.  Work is cut into items: (segment, key
// head, range of keys, tile of rows), where a segment is a group's shared
// positions or a request's own.  Every block counts the items from the lengths on
// the device (schedule), so that a captured call follows them at each replay.
//
// All products are transposed: S^T = K Q^T and O^T = V^T P^T on 32x32x16 matrix
// instructions.  A lane then holds scores, maximum, sum and output of one row (and
// another lane the other half of its keys), so that a row's statistics take one
// exchange between two lanes, and the accumulators of S^T are the right operand
// of the second product as they stand, with the keys of each 16 in the order
// 0-3, 8-11 | 4-7, 12-15, in which V is read as well.  The weights are rounded to the
// io type for it, since the matrix instructions take no wider ones (their sum is not):
// half a step of each at most, as much again as the rounding of the result (bf16: 2.3e-3
// off 64 bits in all, 1.7e-3 if only the result is rounded).  Maxima, sums and outputs
// stay in fp32, the pieces too.
//
// Many rows are bound by the matrix cores and what feeds them, few rows by memory.
// Measured on an MI355X (reads of long rows 6.2 TB/s, bf16 products of 8192^3 1370
// TFLOP/s): a prompt of 8192 tokens 890-1010 TFLOP/s (dims 256, 128; 64: 650-680), 1024
// requests behind 16384 shared positions 780-860, 64 and 256 requests of 4096 and 1024
// positions with nothing shared 4.9-5.8 TB/s.
#include <algorithm>

#include "common.hpp"

namespace gdn {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) void lds_void;

// Rows of a segment up to which its waves split the keys instead of the rows: a
// matrix instruction's.  (With 16, so that 24 and 32 rows are many, 32/8 heads of 128: 64
// requests of 6 drafts behind 2048 positions 115 us for 113, two of 8 behind 32768 56
// for 59, 512 of 8 behind 256 169 for 153, 64 of 8 behind shared prompts 119 for 112.)
constexpr int kFew = 32;
constexpr int kThreads = 256;  // of every kernel here
constexpr int kCus = 256;
// What an item of many rows costs beside its steps, in steps, what a piece to be joined
// costs more, and what it costs that there are any.  (A prompt of 1024 tokens, 16/2 heads
// of 256, is not split so: 47 us; 58 where it was, at a price of pieces that was half of
// theirs.  One of 2048 77 us, 112 with half of all of them.)
constexpr float kItem = 10.f, kPiece = 16.f, kJoin = 12.f;
// Steps of the longest segment, 2^27 positions in steps of 32: no range is longer, so that its
// end in positions fits an int however much work there is.
constexpr float kLongest = 4194304.f;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kLater = 8.0f;  // a maximum may lag by 2^8 before the sums are rescaled

struct Cache {
  const void* at;
  int64_t page, token, head;  // strides, elements
};

struct Attend {
  const void* q;
  int64_t q_token, q_head;
  Cache k, v;
  const void* table;  // [requests, width] pages
  int64_t table_row;
  const void *lens, *shared, *groups, *cu;  // shared NULL: nothing shared; groups NULL: one; cu NULL: a token each
  int table_is64, lens_is64, shared_is64, groups_is64, cu_is64;
  int tokens, requests, num_groups, heads, kv_heads, per;
  Div32 by_per, by_heads;
  int pages, capacity;  // of the cache; positions of a row of the table
  Div32 page;
  float factor;  // scale log2 e
  void* out;
  int64_t out_token, out_head;
  float* lse;  // [tokens, heads] or NULL
  // workspace: per kind (0: few rows, 1: many) the items' sums [items, rows, dim], statistics (m, l) [items, rows];
  // the first item and the number of key ranges of each segment
  float* sums[2];
  float2* stats[2];
  int items_max[2];
  int few_rows;         // rows kept of an item of few: no segment has more
  float per_target[2];  // key heads over the number of items wanted
  struct Place* places;  // of each segment, for the joining kernel
};
// Where the items of a segment lie, and what it is.
struct alignas(16) Place {
  int item, ranges;  // first item; ranges of keys
  int token, tokens, lo, hi;
  int group;  // of a request (-1: none)
};

// ------------------------------------------------------------------ segments
struct Segment {
  int token, tokens;  // first query token, their number
  int lo, hi;         // positions
  int request;        // whose row of the table is read
  int length;         // of the request, as given (a group's: unused)
  int group;          // of the request, or -1
};

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ int clampi(int64_t v, int lo, int hi) {
  return static_cast<int>(v < lo ? lo : v > hi ? hi : v);
}
// A length as it is given, which may be behind the end of the table or below zero.
__device__ __forceinline__ int length_of(const Attend& p, int request) {
  return clampi(load_index64(p.lens, request, p.lens_is64), INT32_MIN / 2, INT32_MAX);
}
__device__ __forceinline__ int token_of(const Attend& p, int request) {
  return p.cu ? clampi(load_index(p.cu, request, p.cu_is64), 0, p.tokens) : request;
}
__device__ __forceinline__ int group_start(const Attend& p, int g) {
  return p.groups ? clampi(load_index(p.groups, g, p.groups_is64), 0, p.requests) : g == 0 ? 0 : p.requests;
}
__device__ __forceinline__ int shared_of(const Attend& p, int g) {
  return clampi(load_index(p.shared, g, p.shared_is64), 0, p.capacity);
}
// The group of a request: the last that starts at or before it, or -1 where its end does not reach it.
__device__ __forceinline__ int group_of(const Attend& p, int request) {
  if (!p.shared) return -1;
  int lo = 0, hi = p.num_groups - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (group_start(p, mid) <= request) lo = mid; else hi = mid - 1;
  }
  return group_start(p, lo) <= request && request < group_start(p, lo + 1) ? lo : -1;
}
__device__ __forceinline__ int segments_of(const Attend& p) { return p.requests + (p.shared ? p.num_groups : 0); }

// Its loads do not wait for each other, but for those behind a search among groups and
// a group's first and last token.
__device__ __forceinline__ Segment segment(const Attend& p, int s) {
  Segment seg;
  const int shared = p.shared ? p.num_groups : 0;
  const bool own = s >= shared;
  const int request = own ? s - shared : 0, g = !own ? s : p.num_groups > 1 ? group_of(p, request) : 0;
  const int length = length_of(p, request);
  int r0 = 0, r1 = p.requests, common = 0;
  if (shared > 0 && g >= 0) {
    r0 = group_start(p, g), r1 = group_start(p, g + 1);
    common = shared_of(p, g);
  }
  const bool in = shared > 0 && g >= 0 && r0 <= request && request < r1;
  const int first = own ? request : r0, last = own ? request + 1 : max(r0, r1);
  seg.token = token_of(p, first);
  seg.tokens = max(0, token_of(p, last) - seg.token);
  seg.lo = own && in ? common : 0;
  seg.hi = own ? clampi(length, 0, p.capacity) : common;
  seg.request = own ? request : min(r0, p.requests - 1);
  seg.length = own ? length : 0;
  seg.group = own && in ? g : -1;
  return seg;
}

// The request of a token: the last that starts at or before it, found by a whole wave.
__device__ __forceinline__ int request_of(const Attend& p, int token, int lane) {
  int first = 0, count = p.requests;
  while (count > 1) {
    const int each = (count + 63) / 64, at = first + lane * each;
    const bool before = lane * each < count && load_index(p.cu, at, p.cu_is64) <= token;
    const int found = max(1, __popcll(__ballot(before)));
    first += (found - 1) * each;
    count = min(each, count - (found - 1) * each);
  }
  return first;
}
// Cut of a segment: tiles of `rows` rows and units of `unit` positions from a multiple of 16 on.
struct Cut {
  int tiles, units;
  int least;  // units of the tile that sees the fewest: its tokens come first
};
template <bool MANY, int ROWS, int UNIT>
__device__ __forceinline__ Cut cut_of(const Attend& p, const Segment& seg, bool own) {
  const int rows = seg.tokens * p.per, from = seg.lo & ~15;
  if (rows == 0 || (rows > kFew) != MANY || seg.hi <= seg.lo) return {0, 0, 0};
  const int units = (seg.hi - from + UNIT - 1) / UNIT;
  const int seen = clampi(static_cast<int64_t>(seg.length) - seg.tokens - from, 0, seg.hi) / UNIT + 1;
  return {(rows + ROWS - 1) / ROWS, units, own && seen < units ? seen : units};
}

// ------------------------------------------------------------------ schedule
constexpr int kCandidates = 32;
struct alignas(16) Plan {
  int base[kThreads];  // items before each thread's segments
  Segment segments[kThreads];  // each thread's first one: all, of up to kThreads
  float units[kThreads / 64], few[kThreads / 64];
  int count[kThreads / 64];
  int range[2];        // units of a range of shared keys, of a request's own
  int alike;           // one segment of many rows: its items lie in the order of their lengths
};
// What the choice of the ranges looks at: segments (their tiles in all heads, units, least
// units; 1: own, 2: nothing is to be joined if it is not split); of each candidate the
// items, those that are not empty, those of them to be joined, the shared ones, the
// longest of the shared and of the own.
struct Choice {
  int segments, items[kCandidates], filled[kCandidates], pieces[kCandidates], shared[kCandidates];
  int longest[2][kCandidates];
  int cuts[kThreads][4];
};
// One LDS array holds it all in a kernel with direct loads: beside a second one, the
// compiler waits for every load in flight in front of each read.
static_assert(sizeof(Plan) % 8 == 0, "what lies behind it is aligned");

// n / d for d > 0 where the quotient is at most 2^22 (there are up to 2^27 positions, 2^22
// steps): shorter than the exact division, and what a launch runs once it has to fetch
// first.
__device__ __forceinline__ int short_div(int n, int d) {
  int q = static_cast<int>(static_cast<float>(n) * __builtin_amdgcn_rcpf(static_cast<float>(d)));
  const int r = n - q * d;
  q += r >= d ? 1 : r < 0 ? -1 : 0;
  return q;
}
__device__ __forceinline__ int ranges_of(int units, int range) { return short_div(units + range - 1, range); }

// The ranges of keys for items of many rows: of 32 candidates the one under which the
// last block should end first.  Shared items come first and are alike, a block takes
// one of each round; a request's own ones fill what these leave, but for half of their
// longest.  An item costs its steps, kItem, and kPiece if its sums are joined; one that
// sees nothing is priced at nothing, though it starts, and its piece is stored and joined
// like the others.  (Six
// prompts behind 8192 shared positions, 16/2 heads of 256: 272 us in ranges of the
// length that all the work gives a block.  Equal parts of one line of all the work,
// whatever tiles they cut, balance better still, but then no two blocks read the same
// keys at a time, the L2 no longer serves them, and it took a third longer than equal
// ranges.)
__device__ __forceinline__ int2 candidate(float units_a_block, int i) {
  // none is split; otherwise 2, 1.71, 1.5, 1.33, 1.2 .. 0.25 times what a block gets; own ones alike or in eighths
  const int which = i & 15;
  const float shares = which < 6 ? 0.5f + (which - 1) / 12.f : 0.91f + (which - 6) * (which - 6) * 0.038f;
  const int range = which == 0 ? 1 << 30 : static_cast<int>(fminf(units_a_block / shares, kLongest)) + 1;
  return make_int2(range, i < 16 ? range : (range >> 3) + 1);
}
struct Outcome {
  int items, filled, pieces, shared, longest, longest_own;
  // one more segment, `tiles` in all heads, under a range
  __device__ __forceinline__ void add(int tiles, int units, int least, int kind, int2 limit) {
    const bool own = kind & 1, alone = kind & 2;
    const int range = own ? limit.y : limit.x;
    const int ranges = ranges_of(units, min(units, range)), length = ranges_of(units, ranges);
    // on average a tile sees half of the units between the fewest and all, and half of its last range
    const float mean = static_cast<float>(units + least) / static_cast<float>(2 * length) + (least < units ? 0.5f : 0.f);
    items += tiles * ranges;
    const int here = max(tiles, min(tiles * ranges, static_cast<int>(static_cast<float>(tiles) * mean + 0.5f)));
    filled += here;
    pieces += alone && ranges == 1 ? 0 : here;
    shared += own ? 0 : here;
    longest = max(longest, own ? 0 : length), longest_own = max(longest_own, own ? length : 0);
  }
  __device__ __forceinline__ void put(Choice& to, int i) const {
    atomicAdd(&to.items[i], items);
    atomicAdd(&to.filled[i], filled);
    atomicAdd(&to.pieces[i], pieces);
    atomicAdd(&to.shared[i], shared);
    atomicMax(&to.longest[0][i], longest);
    atomicMax(&to.longest[1][i], longest_own);
  }
};
__device__ __forceinline__ int2 choose(const Attend& p, const Choice& choice, float units, int lane, int blocks) {
  int best = lane & (kCandidates - 1);
  const float each = 1.f / static_cast<float>(blocks), own = static_cast<float>(choice.longest[1][best]);
  float time = units + static_cast<float>(choice.filled[best]) * each * kItem + (own > 0.f ? 0.5f * (own + kItem) : 0.f);
  time = fmaxf(time, own + kItem);
  time = fmaxf(time, ceilf(static_cast<float>(choice.shared[best]) * each) * (static_cast<float>(choice.longest[0][best]) + kItem));
  if (choice.pieces[best] > 0) time += kJoin + static_cast<float>(choice.pieces[best]) * each * kPiece;
  if (choice.items[best] > p.items_max[1] && (best & 15) > 0) time = INFINITY;
#pragma unroll
  for (int off = 1; off < kCandidates; off <<= 1) {
    const float other = __shfl_xor(time, off, 64);
    const int which = __shfl_xor(best, off, 64);
    if (other < time || (other == time && which < best)) time = other, best = which;
  }
  return candidate(units, best);
}

// Counts the items of the launch: thread i answers for the segments i, i + kThreads, ...,
// and the items lie thread by thread.  A range of keys of few rows is as long as all of
// their work gives to each of three waves a CU.  Block 0 notes for the joining kernel
// where each segment's items lie.
template <bool MANY, int ROWS, int UNIT>
__device__ __forceinline__ int schedule(const Attend& p, Plan& plan, Choice* choice, int block, int blocks) {
  const int n = segments_of(p), lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float units = 0.f, few = 0.f;  // the same in all blocks; its rounding is in the bound of the items
  int items = 0, before = 0, total = 0;
  int2 range = make_int2(1, 1);  // shared, own
  Segment first{}, second{};  // of this thread
  if (MANY) {
    static_assert(sizeof(Choice) / 4 - 4 * kThreads <= kThreads, "a word a thread");
    if (threadIdx.x < sizeof(Choice) / 4 - 4 * kThreads) reinterpret_cast<int*>(choice)[threadIdx.x] = 0;
    __syncthreads();
  }
  // units, items, places: one loop, so that the code of segment() is there once
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
#pragma unroll 1
    for (int s = threadIdx.x; s < n; s += kThreads) {
      const int which = s / kThreads;
      Segment seg = which == 0 ? first : second;
      if (pass == 0 || which > 1) seg = segment(p, s);
      const Cut c = cut_of<MANY, ROWS, UNIT>(p, seg, s >= segments_of(p) - p.requests);
      const int limit = s >= n - p.requests ? range.y : range.x;
      const int ranges = ranges_of(c.units, MANY ? min(limit, max(1, c.units)) : limit);
      if (pass == 0) {
        if (which == 0) first = seg;
        if (which == 1) second = seg;
        units += static_cast<float>(c.tiles) * static_cast<float>(c.units + c.least) * 0.5f;
        if (MANY && c.tiles == 0) few += static_cast<float>(cut_of<false, kFew, UNIT>(p, seg, false).units);
        if (MANY && c.tiles > 0) {
          const int to = atomicAdd(&choice->segments, 1);
          if (to < kThreads) {
            choice->cuts[to][0] = c.tiles * p.kv_heads, choice->cuts[to][1] = c.units, choice->cuts[to][2] = c.least;
            choice->cuts[to][3] = s < n - p.requests ? 0 : seg.lo == 0 ? 3 : 1;
          }
        }
      } else if (pass == 1) {
        items += c.tiles * p.kv_heads * ranges;
      } else {
        if ((seg.tokens * p.per > kFew) == MANY || p.items_max[0] == 0)  // the kind's, or all in a launch of one kind
          p.places[s] = {before, ranges, seg.token, seg.tokens, seg.lo, seg.hi, seg.group};
        before += c.tiles * p.kv_heads * ranges;
      }
    }
    if (pass == 0) {
      plan.segments[threadIdx.x] = first;
      units = head_sum<64>(units);
      if (MANY) few = head_sum<64>(few);
      if (lane == 0) plan.units[wave] = units, plan.few[wave] = few;
      __syncthreads();
      units = (plan.units[0] + plan.units[1] + plan.units[2] + plan.units[3]) * p.per_target[MANY];
      if (units == 0.f && block > 0) return 0;  // nothing of this kind; block 0 notes the places
      if constexpr (MANY) {
        // Where a CU has two blocks and its few rows take longer to read than its many to
        // multiply, half as many ranges leave fewer pieces and are done as soon (64 x 8 drafts
        // behind shared prompts 118 -> 112 us; 256 requests behind 16384 shared positions
        // with few of their own would take 110 instead of 103.  64 channels, 32/8 heads, 64 x 8
        // drafts behind 16384: 171 us for 189 with as many of their own each, 143 for 125
        // with a sixteenth).
        few = (plan.few[0] + plan.few[1] + plan.few[2] + plan.few[3]) * p.per_target[1];
        if (blocks > kCus && p.items_max[0] > 0 && few > 0.66f * units) units *= 2.f, blocks /= 2;
        // of more segments than that, every one is split alike
        if (choice->segments <= kThreads) {
          const int i = threadIdx.x & (kCandidates - 1);
          Outcome outcome{0, 0, 0, 0, 0, 0};
          for (int e = threadIdx.x / kCandidates; e < choice->segments; e += kThreads / kCandidates)
            outcome.add(choice->cuts[e][0], choice->cuts[e][1], choice->cuts[e][2], choice->cuts[e][3],
                        candidate(units, i));
          if (outcome.items > 0) outcome.put(*choice, i);
          __syncthreads();
          range = choose(p, *choice, units, lane, blocks);
        } else {
          range = candidate(units, 1);
        }
      } else {
        range.x = range.y = static_cast<int>(fminf(units, kLongest)) + 1;
      }
    } else if (pass == 1) {
      int sum = items;
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) {
        const int below = __shfl_up(sum, off, 64);
        if (lane >= off) sum += below;
      }
      if (lane == 63) plan.count[wave] = sum;
      __syncthreads();
      before = sum - items;
#pragma unroll
      for (int w = 0; w < kThreads / 64; ++w) {
        if (w < wave) before += plan.count[w];
        total += plan.count[w];
      }
      plan.base[threadIdx.x] = before;
      if (threadIdx.x == 0) {
        plan.range[0] = range.x, plan.range[1] = range.y;
        if (MANY) plan.alike = choice->segments <= 1;
      }
      if (block > 0) break;
    }
  }
  __syncthreads();
  return min(total, p.items_max[MANY]);
}

struct Item {
  Segment seg;
  int head, tile;  // key head, tile of rows
  int from, to;    // positions, from a multiple of 16
  int ranges;      // of the segment
  bool own;        // of a request, not of a group
};

// The item that is `at` among those of a thread's segments.  Items of many rows lie with the
// last tiles, which see the most, first; of each tile the ranges of keys, of each
// range the heads.
template <bool MANY, int ROWS, int UNIT>
__device__ __forceinline__ Item item_at(const Attend& p, const Plan& plan, int thread, int at) {
  const int n = segments_of(p);
  for (int s = thread;; s += kThreads) {
    const Segment seg = s == thread ? plan.segments[thread] : segment(p, s);
    const bool own = s >= n - p.requests;
    const Cut c = cut_of<MANY, ROWS, UNIT>(p, seg, own);
    const int limit = plan.range[own];
    const int ranges = ranges_of(c.units, MANY ? min(limit, max(1, c.units)) : limit), items = c.tiles * p.kv_heads * ranges;
    if (at < items || s + kThreads >= n) {
      Item it;
      it.seg = seg, it.ranges = ranges, it.own = own;
      const int each = max(1, ranges), length = MANY ? ranges_of(c.units, each) : limit;
      int range;
      if (MANY) {
        const int rest = short_div(at, p.kv_heads), back = short_div(rest, each);
        it.head = at - rest * p.kv_heads, range = rest - back * each, it.tile = max(0, c.tiles - 1 - back);
      } else {
        it.head = short_div(at, each), range = at - it.head * each, it.tile = 0;
      }
      it.from = (seg.lo & ~15) + range * length * UNIT;
      it.to = min(seg.hi, it.from + length * UNIT);
      return it;
    }
    at -= items;
  }
}
// Called by whole waves: what it finds is the same in all lanes, and kept in scalar registers.
template <bool MANY, int ROWS, int UNIT>
__device__ Item item_of(const Attend& p, const Plan& plan, int item) {
  static_assert(kThreads == 256, "four bases a lane");
  const int lane = threadIdx.x & 63;
  int thread = -1;  // the last whose base is at most `item`
#pragma unroll
  for (int i = 0; i < 4; ++i) thread += __popcll(__ballot(plan.base[4 * lane + i] <= item));
  thread = uniform(thread);
  const Item it = item_at<MANY, ROWS, UNIT>(p, plan, thread, item - uniform(plan.base[thread]));
  return {{uniform(it.seg.token), uniform(it.seg.tokens), uniform(it.seg.lo), uniform(it.seg.hi),
           uniform(it.seg.request), uniform(it.seg.length), uniform(it.seg.group)},
          uniform(it.head), uniform(it.tile), uniform(it.from), uniform(it.to), uniform(it.ranges), it.own};
}
// Steps of an item of many rows: nothing behind the last position that a row of its tile sees.
template <int ROWS, int UNIT> __device__ __forceinline__ int steps_of(const Attend& p, const Item& it) {
  int to = it.to;
  if (it.own) {
    const int last_token = min(it.seg.tokens - 1, static_cast<int>(p.by_per.div(it.tile * ROWS + ROWS - 1)));
    to = clampi(static_cast<int64_t>(it.seg.length) - (it.seg.tokens - 1 - last_token), 0, to);
  }
  return to > it.from ? (to - it.from + UNIT - 1) / UNIT : 0;
}

// Up to 64 segments of few rows: every wave counts the same items for itself, a segment a
// lane, without barriers and LDS (one request of 4096 positions, 16/2 heads of 256: 17.0
// us, 18.0 by the general way; 40 of 700, 8/8 heads of 64: 18.2 and 19.8).
struct Lane {
  Segment seg;
  int base, ranges, range;  // items before it, its ranges, units of a range of all
};
template <int ROWS, int UNIT>
__device__ __forceinline__ int count_few(const Attend& p, Lane& mine, bool notes, int lane) {
  const int n = segments_of(p);
  Cut c{0, 0, 0};
  if (lane < n) {
    mine.seg = segment(p, lane);
    c = cut_of<false, ROWS, UNIT>(p, mine.seg, lane >= n - p.requests);
  }
  const float here = static_cast<float>(c.tiles) * static_cast<float>(c.units + c.least) * 0.5f;
  const float units = head_sum<64>(here) * p.per_target[0];
  mine.range = static_cast<int>(fminf(units, kLongest)) + 1;
  mine.ranges = ranges_of(c.units, mine.range);
  const int items = c.tiles * p.kv_heads * mine.ranges;
  int sum = items;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int below = __shfl_up(sum, off, 64);
    if (lane >= off) sum += below;
  }
  mine.base = sum - items;
  if (notes && lane < n && mine.seg.tokens * p.per <= kFew)
    p.places[lane] = {mine.base, mine.ranges, mine.seg.token, mine.seg.tokens, mine.seg.lo, mine.seg.hi, mine.seg.group};
  return min(__builtin_amdgcn_readlane(sum, 63), p.items_max[0]);
}
template <int UNIT> __device__ __forceinline__ Item item_of_few(const Attend& p, const Lane& mine, int item) {
  const int s = __popcll(__ballot(mine.base <= item)) - 1;  // the last whose base is at most `item`
  auto of = [&](int v) __attribute__((always_inline)) { return __builtin_amdgcn_readlane(v, s); };
  Item it;
  it.seg = {of(mine.seg.token),   of(mine.seg.tokens), of(mine.seg.lo),   of(mine.seg.hi),
            of(mine.seg.request), of(mine.seg.length), of(mine.seg.group)};
  it.ranges = of(mine.ranges);
  it.own = s >= segments_of(p) - p.requests;
  it.tile = 0;
  const int across = item - of(mine.base), range = uniform(mine.range);
  it.head = uniform(short_div(across, max(1, it.ranges)));
  it.from = (it.seg.lo & ~15) + (across - it.head * max(1, it.ranges)) * range * UNIT;
  it.to = min(it.seg.hi, it.from + range * UNIT);
  return it;
}

// ------------------------------------------------------------------ matrix instructions and loads
template <class T> struct Op;
template <> struct Op<bf16> {
  using frag = bf16x8;
  static constexpr uint32_t kExponent = 0x7f80;
  static __device__ __forceinline__ f32x16 mma(frag a, frag b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};
template <> struct Op<f16> {
  using frag = f16x8;
  static constexpr uint32_t kExponent = 0x7c00;
  static __device__ __forceinline__ f32x16 mma(frag a, frag b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};

// Where 16 positions from `at` on (a multiple of 16) lie: page (-1: none) and place inside it.
struct Spot {
  int page, in;
};
__device__ __forceinline__ Spot find(const Attend& p, int request, int at, int end) {
  if (at >= end) return {-1, 0};
  const uint32_t index = p.page.div(at);
  const int64_t entry = static_cast<int64_t>(request) * p.table_row + index;
  const int64_t id = load_index64(p.table, entry, p.table_is64);
  return {id < 0 || id >= p.pages ? -1 : static_cast<int>(id), at - static_cast<int>(index * p.page.d)};
}
// The same of 64 times 16 positions, one in each lane, in bytes of a cache, looked up
// together so that the steps' loads wait for no table.
struct Spots {
  int low, high;  // high kNone: nowhere
  static constexpr int kNone = INT32_MIN;
  __device__ __forceinline__ void set(Spot spot, int64_t page, int64_t token) {
    const int64_t bytes = spot.page * page + spot.in * token;
    low = static_cast<int>(bytes), high = spot.page < 0 ? kNone : static_cast<int>(bytes >> 32);
  }
};

template <int N> __device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
__device__ __forceinline__ void reads_done() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// Rows of a head in LDS: [positions][dim], pieces of 16 bytes.  Those of K lie
// at piece ^ (row % 16), those of V at piece ^ 4 (row % 4) (rows of 128 bytes, two
// of which fill the 64 banks: half as many), so that the lanes of one read touch
// different banks: K is read by 16 rows at the same piece, V by 4 rows at 4.
template <int D> struct Tile {
  static constexpr int kPieces = D / 8, kRow = 2 * D;
  static constexpr int kPerLoad = 1024 / kRow;  // rows that a wave's load of 16 bytes a lane brings
  static __device__ __forceinline__ int swizzle_k(int row) { return D == 64 ? (row >> 1) & 7 : row & 15; }
  static __device__ __forceinline__ int swizzle_v(int row) { return D == 64 ? 4 * (row >> 1 & 1) : 4 * (row & 3); }
};

// A direct-to-LDS load of 16 bytes a lane: lane l lands at lds + 16 l, zeros where off is past bytes.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc_of(const void* from, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(from), 0, bytes, 0x00020000);
}
__device__ __forceinline__ void dma16(const void* src, uint32_t bytes, uint32_t off, void* lds) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc_of(src, bytes), (lds_void*)lds, 16, off, 0, 0, 0);
}
// Direct loads of one head's keys or values to LDS, 16 positions at a time: lane l of
// the i-th load of 16 bytes a lane lands 16 l behind lds + 1024 i.
template <int D>
struct Feed {
  static constexpr int kLoads = 16 / Tile<D>::kPerLoad;
  const char* head;      // the head's first channel in the first page
  int64_t page, token;   // strides, bytes
  uint32_t from[kLoads];  // the lane's piece of each load, bytes behind the first position's
  const char* at;        // what aim() has found: the first position, the bytes that may be read
  uint32_t bytes;
  int valid;

  __device__ __forceinline__ void start(const Cache& c, int of, bool values, int lane) {
    using L = Tile<D>;
    head = static_cast<const char*>(c.at) + 2 * of * c.head;
    page = 2 * c.page, token = 2 * c.token;
    const int row = lane / L::kPieces, piece = lane % L::kPieces;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int r = i * L::kPerLoad + row;
      from[i] = r * static_cast<uint32_t>(token) + 16 * (piece ^ (values ? L::swizzle_v(r) : L::swizzle_k(r)));
    }
  }
  // The 16 positions in lane `which` of `spots`, of which `there` (or more than 16) may
  // be read: zeros behind them, and for a page outside of the cache.
  // In two halves, to stand between matrix instructions.
  __device__ __forceinline__ void aim_at(const Spots& spots, int which, int there) {
    const int low = __builtin_amdgcn_readlane(spots.low, which), high = __builtin_amdgcn_readlane(spots.high, which);
    at = head + (static_cast<int64_t>(high) << 32 | static_cast<uint32_t>(low));
    valid = high == Spots::kNone ? 0 : there;
  }
  __device__ __forceinline__ void aim_bytes() {
    bytes = valid > 0 ? ((valid < 16 ? valid : 16) - 1) * static_cast<uint32_t>(token) + Tile<D>::kRow : 0;
  }
  __device__ __forceinline__ void aim(const Spots& spots, int which, int there) {
    aim_at(spots, which, there);
    aim_bytes();
  }
  __device__ __forceinline__ void load(int i, char* lds) const {
    dma16(at, bytes, from[i], lds + 1024 * i);
  }
  __device__ __forceinline__ void load_all(char* lds) const {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) load(i, lds);
  }
};

// Fragments of a tile of keys or values `off` bytes into LDS (a multiple of 1024, and
// this lane's share of it): what differs from one fragment to the next is some bits
// of the offset, and a constant.
//
// Left operand of S^T, channels 16 step .. + 15 of 32 keys from `row` on: lane l holds
// row l % 32, channels 8 (l / 32) .. + 7 of these.
template <int D> __device__ __forceinline__ int lane_k(int lane) {
  return (lane & 31) * Tile<D>::kRow + 16 * ((lane >> 5) ^ Tile<D>::swizzle_k(lane & 31));
}
template <class T, int D>
__device__ __forceinline__ typename Op<T>::frag k_frag(const char* lds, int off, int row, int step) {
  return *reinterpret_cast<const typename Op<T>::frag*>(lds + (off ^ 32 * (step & 7)) + 256 * (step >> 3) +
                                                        row * Tile<D>::kRow);
}
// Left operand of O^T, channels 32 tile .. + 31 of 16 keys from `row` on: lane l holds
// channel l % 32 of these, keys 4 (l / 32) .. + 3 and 8 behind these.  The 16 lanes of a
// read bring 4 rows of 16 channels, lane i of them row i / 4, and receive channel i each.
template <int D> __device__ __forceinline__ int lane_v(int lane) {
  const int row = 4 * (lane >> 5) + ((lane & 15) >> 2), piece = 2 * (lane >> 4 & 1) + ((lane & 3) >> 1);
  return row * Tile<D>::kRow + 16 * (piece ^ Tile<D>::swizzle_v(row)) + 8 * (lane & 1);
}
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
// `restrict` tells the compiler that what is read here is none of the direct loads in
// flight; it would wait for all of them.  (Other reads it tells apart by their types.)
__device__ __forceinline__ s16x4 read_across(lds_s16x4* __restrict__ at) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16(at);
}
template <class T, int D>
__device__ __forceinline__ typename Op<T>::frag v_frag(const char* lds, int off, int row, int tile) {
  const char* at = lds + (off ^ 64 * (tile & 3)) + 256 * (tile >> 2) + row * Tile<D>::kRow;
  const s16x4 a = read_across((lds_s16x4*)(at)), b = read_across((lds_s16x4*)(at + 8 * Tile<D>::kRow));
  return __builtin_bit_cast(typename Op<T>::frag, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}

// v, computed where it stands: not moved down to where it is used.
template <class V> __device__ __forceinline__ V here(V v) {
  asm volatile("" : "+v"(v));
  return v;
}
// Instructions stay on their side of it.
__device__ __forceinline__ void in_order() { __builtin_amdgcn_sched_barrier(0); }

// The lane, found anew.
__device__ __forceinline__ int lane_again() {
  return here(static_cast<int>(__builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u))));
}
// The value of the lane 32 before or behind this one.
__device__ __forceinline__ uint32_t other_half(uint32_t v) {
  const auto halves = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return halves[0] == v ? halves[1] : halves[0];
}
// How many lanes of the wave hold less.
__device__ __forceinline__ int place_among(int v) {
  int n = 0;
#pragma unroll 8
  for (int k = 0; k < 64; ++k) n += __builtin_amdgcn_readlane(v, k) < v ? 1 : 0;
  return n;
}
// The least of a wave's lanes.
__device__ __forceinline__ uint32_t min_of_wave(uint32_t v) {
  auto step = [](uint32_t x, auto ctrl) __attribute__((always_inline)) {
    return min(x, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(-1, static_cast<int>(x), decltype(ctrl)::value, 0xf, 0xf, false)));
  };
  v = step(v, std::integral_constant<int, 0xB1>{});   // quad_perm [1,0,3,2]
  v = step(v, std::integral_constant<int, 0x4E>{});   // quad_perm [2,3,0,1]
  v = step(v, std::integral_constant<int, 0x141>{});  // row_half_mirror
  v = step(v, std::integral_constant<int, 0x128>{});  // row_ror:8
  const uint32_t a = __builtin_amdgcn_readlane(v, 0), b = __builtin_amdgcn_readlane(v, 16);
  const uint32_t c = __builtin_amdgcn_readlane(v, 32), d = __builtin_amdgcn_readlane(v, 48);
  return min(min(a, b), min(c, d));
}
// Of this lane's value and that of the lane 32 before or behind it.
__device__ __forceinline__ float max_of_halves(float v) {
  const auto halves = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(halves[0]), __uint_as_float(halves[1]));
}
__device__ __forceinline__ float sum_of_halves(float v) {
  const auto halves = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(halves[0]) + __uint_as_float(halves[1]);
}

// A weight of zero does not silence a value that is not finite.  Where rows of an
// item do not see all of a tile's positions, such values are taken out of it, and
// for each channel the first position of a positive and of a negative one is kept
// (of both for a NaN): they go to the rows that see it when the item is done.
template <int D> struct NotFinite {
  int found, pad[3];
  int first[2][D];
  __device__ __forceinline__ void clear(int thread, int threads) {
    if (thread == 0) found = 0;
    for (int i = thread; i < 2 * D; i += threads) first[i / D][i % D] = INT32_MAX;
  }
  __device__ __forceinline__ float added(int channel, int limit) const {
    return (first[0][channel] < limit ? INFINITY : 0.f) - (first[1][channel] < limit ? INFINITY : 0.f);
  }
};

// Of the 16 positions from `at` on whose values this wave has brought to LDS.
template <class T, int D>
__device__ __forceinline__ void take_out(char* v, int at, int lo, NotFinite<D>& bad, int lane) {
  using L = Tile<D>;
  constexpr uint32_t kBits = Op<T>::kExponent, kMask = kBits * 0x10001u, kStep = (0x8000u - kBits) * 0x10001u;
  uint32_t found = 0;  // the top bit of a half: its exponent had no room for one more
#pragma unroll
  for (int i = 0; i < 16 / L::kPerLoad; ++i) {
    const u32x4 raw = *reinterpret_cast<const u32x4*>(v + i * 1024 + lane * 16);
    found |= ((raw[0] & kMask) + kStep) | ((raw[1] & kMask) + kStep) | ((raw[2] & kMask) + kStep) | ((raw[3] & kMask) + kStep);
  }
  if (!__any((found & 0x80008000u) != 0)) return;
#pragma unroll 1
  for (int i = 0; i < 16 / L::kPerLoad; ++i) {
    const int row = i * L::kPerLoad + lane / L::kPieces, piece = (lane % L::kPieces) ^ L::swizzle_v(row);
    uint16_t* values = reinterpret_cast<uint16_t*>(v + i * 1024 + lane * 16);
#pragma unroll 1
    for (int e = 0; e < 8; ++e) {
      const uint32_t bits = values[e];
      if ((bits & kBits) != kBits) continue;
      values[e] = 0;
      if (at + row < lo) continue;
      const bool nan = (bits & 0x7fff) != kBits, negative = bits >> 15;
      if (nan || !negative) atomicMin(&bad.first[0][8 * piece + e], at + row);
      if (nan || negative) atomicMin(&bad.first[1][8 * piece + e], at + row);
      bad.found = 1;
    }
  }
}

// Whether an item holds all that its rows see, as the only range of its segment (a tile that
// ends in the first of several is joined all the same): nothing has to be joined.
__device__ __forceinline__ bool whole(const Item& it) { return it.own && it.ranges == 1 && it.seg.lo == 0; }

// Four channels of a finished row.
template <class T>
__device__ __forceinline__ void put4(const Attend& p, int token, int head, int channel, const float (&y)[4]) {
  T* to = static_cast<T*>(p.out) + token * p.out_token + head * p.out_head + channel;
  *reinterpret_cast<uint2*>(to) = make_uint2(out_pack2<T>(y[0], y[1]), out_pack2<T>(y[2], y[3]));
}
// The factor of a piece with maximum m and sum l under the joint maximum; 0 where the
// piece saw nothing (a NaN stays one).
__device__ __forceinline__ float weight_of(float m, float l, float top) { return l == 0.f ? 0.f : fast_exp2(m - top); }
// One over a row's sum of weights.  There are none where it sees nothing: zeros; and where
// all that it sees scores -infinity: NaN, as the softmax of it.
__device__ __forceinline__ float inverse_of(float l, bool sees) { return l != 0.f ? 1.0f / l : sees ? NAN : 0.f; }
__device__ __forceinline__ float lse_of(float m, float l) { return l > 0.f || l != l ? (m + log2f(l)) * kLn2 : -INFINITY; }

// One wave's rows: 32 of them, a lane and its partner 32 lanes on share one.
template <class T, int D>
struct Rows {
  using Frag = typename Op<T>::frag;
  static constexpr int kAhead = 4;  // fragments that are read before their matrix instructions
  Frag q[D / 16];
  f32x16 o[D / 32];
  float m, l;    // maximum of the scaled scores (base 2), and this lane's part of the sum
  int limit;     // positions before it are visible to the row
  int least;     // of the wave's rows

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[i][e] = 0.f;
    m = -INFINITY, l = 0.f;
  }

  // Row `row` of the segment: its queries.
  __device__ __forceinline__ void fetch(const Attend& p, const Item& it, int row, int lane) {
    const bool there = row < it.seg.tokens * p.per;
    const int in = there ? p.by_per.div(row) : 0, token = it.seg.token + in;
    const int head = it.head * p.per + (there ? row - in * p.per : 0);
    const T* from = static_cast<const T*>(p.q) + token * p.q_token + head * p.q_head + 8 * (lane >> 5);
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      const uint4 raw = there ? *reinterpret_cast<const uint4*>(from + 16 * i) : make_uint4(0, 0, 0, 0);
      q[i] = __builtin_bit_cast(Frag, raw);
    }
  }
  // The positions visible to it.
  __device__ __forceinline__ void see(const Attend& p, const Item& it, int row, int lane) {
    const bool there = row < it.seg.tokens * p.per;
    const int in = there ? p.by_per.div(row) : 0, token = it.seg.token + in;
    int length = it.seg.length, behind = it.seg.tokens - 1 - in;  // tokens of the request behind this one
    if (!it.own) {  // uniform
      int r = token, next = token + 1;
      if (p.cu) {
        // the requests of the wave's tokens lie behind that of its first one: their ends in the lanes, searched there
        const int first = request_of(p, uniform(token), lane);
        const int end = token_of(p, min(first + 1 + lane, p.requests));
        int at = 0;
#pragma unroll
        for (int half = 32; half > 0; half >>= 1)
          if (__shfl(end, at + half - 1, 64) <= token) at += half;
        r = first + at, next = __shfl(end, at, 64);
        if (__any(next <= token)) {  // more requests than lanes (most of them empty)
          r = static_cast<int>(find_sequence(p.cu, p.cu_is64, p.requests, token));
          next = token_of(p, r + 1);
        }
      }
      r = min(r, p.requests - 1);
      length = length_of(p, r);
      behind = next - 1 - token;
    }
    const int seen = clampi(static_cast<int64_t>(length) - behind, 0, it.seg.hi);
    limit = there ? seen : 0;
    int a = there ? limit : INT32_MAX;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) a = min(a, __shfl_xor(a, off, 64));
    least = uniform(a);
  }

  // The i-th fragment of 32 TILES positions.
  template <int TILES>
  static __device__ __forceinline__ Frag key(const char* lds, int off, int i) {
    return k_frag<T, D>(lds, off, i / (D / 16) * 32, i % (D / 16));
  }
  template <int TILES>
  static __device__ __forceinline__ Frag value(const char* lds, int off, int i) {
    return v_frag<T, D>(lds, off, 16 * (i % (2 * TILES)), i / (2 * TILES));
  }
  // Scores of 32 TILES positions; the first kAhead fragments are in f.  beside(i) goes
  // behind the i-th matrix instruction.
  template <int TILES, class Beside>
  __device__ __forceinline__ void scores(const char* lds, int off, Frag (&f)[kAhead], f32x16 (&s)[TILES],
                                         Beside beside) const {
    constexpr int kMmas = D / 16 * TILES;
#pragma unroll
    for (int t = 0; t < TILES; ++t)
#pragma unroll
      for (int e = 0; e < 16; ++e) s[t][e] = 0.f;
    in_order();
#pragma unroll
    for (int i = 0; i < kMmas; ++i) {
      s[i / (D / 16)] = Op<T>::mma(f[i % kAhead], q[i % (D / 16)], s[i / (D / 16)]);
      if (i + kAhead < kMmas) f[i % kAhead] = key<TILES>(lds, off, i + kAhead);
      beside(i);
      in_order();
    }
  }
  // Whether some row of the wave does not see all of the 32 TILES positions from `at` on (uniform).
  template <int TILES>
  __device__ __forceinline__ bool partly(const Segment& seg, int at) const {
    return at < seg.lo || at + 32 * TILES > least;
  }
  template <int TILES>
  __device__ __forceinline__ void mask(const Segment& seg, int at, int lane, f32x16 (&s)[TILES]) const {
    if (!partly<TILES>(seg, at)) return;
#pragma unroll
    for (int t = 0; t < TILES; ++t)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int pos = at + 32 * t + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3);
        if (pos < seg.lo || pos >= limit) s[t][e] = -INFINITY;
      }
  }
  // The row's largest score (base 2) from the largest of the lane's own.
  __device__ __forceinline__ float of_row(const Attend& p, float top) const {
    return max_of_halves(top) * p.factor;
  }
  // The maximum raised to `top`, where that is more than 2^8 above it: fp32 sums have room for less.
  __device__ __forceinline__ void raise(float top) {
    const bool grown = top > m + kLater;
    if (!__any(grown)) return;
    const float alpha = grown ? fast_exp2(m - top) : 1.0f;
    m = grown ? top : m;
    l *= alpha;
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[i][e] *= alpha;
  }
  // Elements first .. last - 1 of the scores to weights, in the io type as the right operand.
  template <int TILES>
  __device__ __forceinline__ void weights(const Attend& p, int first, int last, float less, f32x16 (&s)[TILES],
                                          uint4 (&w)[2 * TILES]) {
#pragma unroll
    for (int i = first; i < last; ++i) {
      float& x = reinterpret_cast<float*>(&s[i / 16])[i % 16];
      x = fast_exp2(fmaf(x, p.factor, -less));
      if (i & 1) {
        const uint32_t pair = out_pack2<T>(reinterpret_cast<float*>(&s[i / 16])[i % 16 - 1], x);
        reinterpret_cast<uint32_t*>(&w[i / 8])[i % 8 / 2] = here(pair);
      }
    }
  }
  // Their sum, unrounded.
  template <int TILES> __device__ __forceinline__ void add(int first, int last, const f32x16 (&s)[TILES]) {
#pragma unroll
    for (int i = first; i < last; ++i) l += s[i / 16][i % 16];
  }
  __device__ __forceinline__ float subtracted() const { return m == -INFINITY ? 0.f : m; }
  // O^T += V^T P^T of 32 TILES positions, as above.
  template <int TILES, class Beside>
  __device__ __forceinline__ void values(const char* lds, int off, Frag (&f)[kAhead], const uint4 (&w)[2 * TILES],
                                         Beside beside) {
    constexpr int kMmas = D / 32 * 2 * TILES;
    in_order();
#pragma unroll
    for (int i = 0; i < kMmas; ++i) {
      f32x16& sum = o[i / (2 * TILES)];
      sum = Op<T>::mma(f[i % kAhead], __builtin_bit_cast(Frag, w[i % (2 * TILES)]), sum);
      if (i + kAhead < kMmas) f[i % kAhead] = value<TILES>(lds, off, i + kAhead);
      beside(i);
      in_order();
    }
  }
  __device__ __forceinline__ void add_not_finite(const NotFinite<D>& bad, int lane) {
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[d][e] += bad.added(32 * d + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3), limit);
  }
  // Row `row` of the segment out: finished, or as a piece to be joined, row `to` of its kind's sums.
  __device__ __forceinline__ void put(const Attend& p, const Item& it, int row, int kind, int64_t to, int lane) {
    const float sum = sum_of_halves(l);
    if (row >= it.seg.tokens * p.per) return;
    if (whole(it)) {
      const int in = p.by_per.div(row), token = it.seg.token + in, head = it.head * p.per + row - in * p.per;
      const float inverse = inverse_of(sum, limit > 0);
#pragma unroll
      for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          const float y[4] = {o[d][e] * inverse, o[d][e + 1] * inverse, o[d][e + 2] * inverse, o[d][e + 3] * inverse};
          put4<T>(p, token, head, 32 * d + 2 * e + 4 * (lane >> 5), y);
        }
      if (p.lse && lane < 32) p.lse[static_cast<int64_t>(token) * p.heads + head] = lse_of(m, sum);
    } else {
      float* sums = p.sums[kind] + to * D + 4 * (lane >> 5);
#pragma unroll
      for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int e = 0; e < 16; e += 4)
          *reinterpret_cast<float4*>(sums + 32 * d + 2 * e) = make_float4(o[d][e], o[d][e + 1], o[d][e + 2], o[d][e + 3]);
      if (lane < 32) p.stats[kind][to] = make_float2(m, sum);
    }
  }
};

// ------------------------------------------------------------------ many rows
// Four waves of 32 rows each.  Step j computes the scores of tile j + 1 while it turns
// those of tile j into weights, then adds the values of tile j while it finds the
// next maximum and issues the loads of the keys of tile j + 4 and the values of tile
// j + 2; so keys lie in a ring of four tiles, values in one of three, and a load has
// a step and a half to arrive.  The first fragments of each product are read during
// the last matrix instructions of the one before it.
//
// Of 256 channels a step takes 1.1 us on all CUs at once (955 to 985 TFLOP/s), some 20 us
// of a call are outside of the steps.  The matrix cores are busy for 43 % of a step's
// cycles, vector instructions for 28 % (128 channels: 43 and 52; 64: 29 and 62), LDS reads
// for 22 %: one hardly goes on beside the other.  How long a cycle is, power decides: on
// keys and values of zeros the same call takes as many of them, at 2.27 GHz for 2.03 (128
// channels 2.22 for 1.99), and long runs of steps reach 1247 TFLOP/s (1303 for 942).
// Without its loads to LDS it ran at 1206, with half of its LDS reads at 1033, without
// exponentials at 1010.  (64 rows a wave, its sums in the upper 256
// registers, halve the loads and the reads: 1053 in long runs of steps, but tiles twice as
// high mean twice the pieces to store and to join: 256 requests behind 32768 shared
// positions 193-203 us against 197-201, prompts of 1024 to 4096 tokens 90, 144 and 326
// against 62, 85 and 176.)  Of 64 channels, where a product has too few instructions to
// hide one step's weights and a barrier, a step is 64 keys: eight prompts of 512 tokens
// 117 us, in steps of 32 126.
template <int D> struct Many {
  static constexpr int kRows = 128, kTiles = D == 64 ? 2 : 1, kKeys = 32 * kTiles;
  static constexpr int kTile = kKeys * 2 * D, kKeyRing = 4, kValueRing = 3, kLds = (kKeyRing + kValueRing) * kTile;
  static constexpr int kLoads = 2 * kTile / 1024 / 4;  // of a wave and step
  static constexpr int kShared = kLds + static_cast<int>(sizeof(NotFinite<D>) + sizeof(Plan)) + 16;
  static constexpr int kBlocks = D == 256 ? 1 : 2;  // of a CU
  static_assert(kBlocks * kShared <= 160 * 1024, "fits");
};

// Block `block` of `blocks` of them.
template <class T, int D>
__device__ __forceinline__ void many_rows(const Attend& p, char* lds, int block, int blocks) {
  using M = Many<D>;
  using R = Rows<T, D>;
  constexpr int kTiles = M::kTiles, kScores = 16 * kTiles, kMmas = D / 16 * kTiles, kAhead = R::kAhead;
  NotFinite<D>& bad = *reinterpret_cast<NotFinite<D>*>(lds + M::kLds);
  Plan& plan = *reinterpret_cast<Plan*>(lds + M::kLds + sizeof(bad));
  int* least = reinterpret_cast<int*>(lds + M::kLds + sizeof(bad) + sizeof(Plan));  // of each wave's rows
  static_assert(sizeof(Choice) <= M::kLds, "in the place of the rings, before they are used");
  const int wave = uniform(threadIdx.x >> 6);
  const int total = schedule<true, M::kRows, M::kKeys>(p, plan, reinterpret_cast<Choice*>(lds), block, blocks);
  // Blocks with the same index modulo 8 share an XCD and its L2.  It takes every eighth item
  // (of one head, then, and often of one range of keys).  Of one segment they lie in the
  // order of their lengths, and the blocks take them to and fro; of several each goes to the
  // block that is free first: 64 at a time their steps are looked up, a lane each, put in
  // order and given out.  (Three prompts of 700 tokens behind 4096 shared positions, 16/2
  // heads of 256, 247 us, 407 where each XCD took a run of items and its blocks took them
  // to and fro; six ragged ones behind 8192 194 to 198, 205; one prompt of 3000 tokens 108,
  // 148.  Given out one after the other throughout, four prompts of 1000 tokens, 32/8
  // heads of 128, took 101 us instead of 88, to and fro 82.)
  constexpr bool kTwo = M::kBlocks == 2;
  constexpr uint32_t kNoBlock = (1u << 25) - 1;
  const int across = blocks >> 3, mine = block >> 3, xcd = block & 7, locals = (total + 7 - xcd) >> 3;
  const bool alike = locals <= across || uniform(plan.alike);
  uint32_t load = lane_again() < across ? 0 : kNoBlock;  // of a block: steps
  uint64_t todo = 0;
  bool back = false;
  for (int base = alike ? -across : -64;;) {
    while (todo == 0 && (base += alike ? across : 64) < locals) {
      if (alike) {
        const int at = back ? across - 1 - mine : mine;
        if (base + at < locals) todo = uint64_t{1} << at;
        back = !back;
        continue;
      }
      const int id = lane_again(), count = min(64, locals - base);
      int key = 63 - id;
      if (id < count) {
        const int item = 8 * (base + id) + xcd;
        int thread = 0;  // the last whose base is at most the item
#pragma unroll
        for (int half = kThreads / 2; half > 0; half >>= 1)
          if (plan.base[thread + half] <= item) thread += half;
        const Item it = item_at<true, M::kRows, M::kKeys>(p, plan, thread, item - plan.base[thread]);
        key |= (steps_of<M::kRows, M::kKeys>(p, it) + static_cast<int>(kItem)) << 6;
      }
      // the longest first, places behind the last item at the end
      key = __builtin_amdgcn_ds_permute(4 * (63 - place_among(key)), key);
      int k = 0;
      if (base == 0) {  // the first round: one each; of a CU's two, a short one to the long one
        k = across;
        const int at = kTwo && id >= 32 ? 95 - id : id;
        const int given = __shfl(key, at, 64);
        if (id < k) load += given >> 6;
        todo = uint64_t{1} << (63 - (__builtin_amdgcn_readlane(given, mine) & 63));
      }
      while (k < count) {
        if (k % across == 0 && count - k >= across) {
          // one each, the longest to the one with the least, if that evens them out
          const int place = place_among(static_cast<int>(load << 6 | id));
          const int given = __shfl(key, id < across ? k + place : 0, 64);
          const uint32_t then = min(load + (given >> 6), kNoBlock - 1);
          const float most = static_cast<float>(~min_of_wave(id < across ? ~then : ~0u));
          const float all = head_sum<64>(id < across ? static_cast<float>(then) : 0.f);
          if (most * static_cast<float>(across) <= 1.03f * all) {
            if (id < across) load = then;
            todo |= uint64_t{1} << (63 - (__builtin_amdgcn_readlane(given, mine) & 63));
            k += across;
            continue;
          }
        }
        // two blocks of a CU go on at half the rate each until one is done
        const uint32_t other = kTwo ? other_half(load) : load;
        const int who = min_of_wave((load <= other ? 2 * load : load + other) << 6 | id) & 63;
        const int next = __builtin_amdgcn_readlane(key, k);
        if (id == who) load = min(load + (next >> 6), kNoBlock - 1);
        if (who == mine) todo |= uint64_t{1} << (63 - (next & 63));
        ++k;
      }
    }
    if (todo == 0) break;
    const int item = 8 * (base + __builtin_ctzll(todo)) + xcd;
    todo &= todo - 1;
    const int lane = lane_again();  // what follows from it is not kept in registers from item to item
    const Item it = item_of<true, M::kRows, M::kKeys>(p, plan, item);
    R rows;
    const int row = it.tile * M::kRows + 32 * wave + (lane & 31);
    rows.fetch(p, it, row, lane);
    const int end = it.seg.hi, steps = uniform(steps_of<M::kRows, M::kKeys>(p, it));
    // A wave brings 16 positions of a step: of the keys or of the values, or (steps of 64) of both.  A
    // feed's loads of steps past the end are issued as well, with nothing in range, so that every step counts alike.
    constexpr bool kBoth = kTiles == 2;
    const bool of_values = !kBoth && wave >= 2;
    const int sub = kBoth ? wave : wave & 1;
    Feed<D> feed[kBoth ? 2 : 1];
    Spots spots[kBoth ? 2 : 1];
    feed[0].start(of_values ? p.v : p.k, it.head, of_values, lane);
    if constexpr (kBoth) feed[1].start(p.v, it.head, true, lane);
    auto spot = [&](int which, int tile) __attribute__((always_inline)) {
      if ((tile & 63) == 0)
        spots[which].set(find(p, it.seg.request, it.from + (tile + lane) * M::kKeys + 16 * sub, end), feed[which].page,
                         feed[which].token);
    };
    auto there = [&](int tile) __attribute__((always_inline)) {
      return tile < steps ? end - (it.from + tile * M::kKeys + 16 * sub) : 0;
    };
    auto aim = [&](int which, int tile) __attribute__((always_inline)) {
      spot(which, tile);
      feed[which].aim(spots[which], tile & 63, there(tile));
    };
    char* const share = lds + sub * 32 * D;
    auto key_at = [](int tile) __attribute__((always_inline)) { return tile % M::kKeyRing * M::kTile; };
    auto value_at = [](int slot) __attribute__((always_inline)) { return (M::kKeyRing + slot) * M::kTile; };
    lds_barrier();  // the last item's rings are free
#pragma unroll
    for (int tile = 0; tile < M::kKeyRing; ++tile) {  // keys of tiles 0 to 3, beside the last two values of 0 and 1
      if (!of_values) {
        aim(0, tile);
        feed[0].load_all(share + key_at(tile));
      }
      if (tile >= 2 && (kBoth || of_values)) {
        aim(kBoth ? 1 : 0, tile - 2);
        feed[kBoth ? 1 : 0].load_all(share + value_at(tile - 2));
      }
    }
    bad.clear(threadIdx.x, kThreads);
    rows.clear();
    rows.see(p, it, row, lane);
    if (lane == 0) least[wave] = rows.least;
    wait_loads<2 * M::kLoads>();
    lds_barrier();  // the keys of tiles 0 and 1 are there
    const int all_see = uniform(min(min(least[0], least[1]), min(least[2], least[3])));
    using Scores = f32x16[kTiles];
    Scores s[2];
    uint4 w[2 * kTiles];
    typename R::Frag keys[kAhead], values[kAhead];
    const int of_k = lane_k<D>(lane), of_v = lane_v<D>(lane);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) keys[i] = R::template key<kTiles>(lds, of_k, i);
    rows.template scores<kTiles>(lds, of_k, keys, s[0], [](int) __attribute__((always_inline)) {});
#pragma unroll
    for (int i = 0; i < kAhead; ++i) keys[i] = R::template key<kTiles>(lds, key_at(1) + of_k, i);
    rows.template mask<kTiles>(it.seg, it.from, lane, s[0]);
    float top = -INFINITY;
    auto larger = [&](const Scores& of, int i) __attribute__((always_inline)) { top = fmaxf(top, of[i / 16][i % 16]); };
#pragma unroll
    for (int i = 0; i < kScores; ++i) larger(s[0], i);
    // a tile behind the last is all zeros, and its scores may not raise anything
    if (steps > 0) rows.raise(rows.of_row(p, top));
    int slot = 0;  // of the step's values
    auto advance = [&](int step, Scores& now, Scores& next) __attribute__((always_inline)) {
      wait_loads<M::kLoads>();  // the keys of step + 2 and the values of step
      const int at = it.from + step * M::kKeys;
      if ((kBoth || of_values) && (at < it.seg.lo || at + M::kKeys > all_see))
        take_out<T, D>(share + value_at(slot), at + 16 * sub, it.seg.lo, bad, lane);
      lds_barrier();
      const float less = rows.subtracted();
      const int v_at = value_at(slot) + of_v;
      rows.template scores<kTiles>(lds, key_at(step + 1) + of_k, keys, next, [&](int i) __attribute__((always_inline)) {
        rows.template weights<kTiles>(p, i * kScores / kMmas, (i + 1) * kScores / kMmas, less, now, w);
        if (i >= kMmas - kAhead) values[i - (kMmas - kAhead)] = R::template value<kTiles>(lds, v_at, i - (kMmas - kAhead));
      });
      rows.template mask<kTiles>(it.seg, at + M::kKeys, lane, next);
      // the loads of a later tile, in the shares that the tiles before these have left
      const int later = slot == 0 ? 2 : slot - 1;
      char* to0 = share + (of_values ? value_at(later) : key_at(step));
      char* to1 = share + value_at(later);
      const int ahead = of_values ? step + 2 : step + 4;
      spot(0, ahead);
      if constexpr (kBoth) spot(1, step + 2);
      const int k_next = key_at(step + 2) + of_k;
      top = -INFINITY;
      rows.template values<kTiles>(lds, v_at, values, w, [&](int i) __attribute__((always_inline)) {
        // behind the first quarter: the scores' last matrix instruction is done by then
        constexpr int kFrom = kMmas / 4, kEach = (kScores + kMmas - kFrom - 1) / (kMmas - kFrom);
        constexpr int kIssue = M::kLoads, kHalf = kBoth ? kIssue / 2 : kIssue;
        if (i == 0) feed[0].aim_at(spots[0], ahead & 63, there(ahead));
        if (i == 1) feed[0].aim_bytes();
        if (kBoth && i == 2) feed[kBoth].aim_at(spots[kBoth], (step + 2) & 63, there(step + 2));
        if (kBoth && i == 3) feed[kBoth].aim_bytes();
        if (i >= 2 && i < 2 + kHalf) feed[0].load(i - 2, to0);
        if (kBoth && i >= 4 && i < 4 + kHalf) feed[kBoth].load(i - 4, to1);
        rows.template add<kTiles>(i * kScores / kMmas, (i + 1) * kScores / kMmas, now);
#pragma unroll
        for (int e = 0; e < kEach; ++e)
          if (i >= kFrom && (i - kFrom) * kEach + e < kScores) larger(next, (i - kFrom) * kEach + e);
        if (i >= kMmas - kAhead) keys[i - (kMmas - kAhead)] = R::template key<kTiles>(lds, k_next, i - (kMmas - kAhead));
      });
      if (step + 1 < steps) rows.raise(rows.of_row(p, top));
      slot = slot == 2 ? 0 : slot + 1;
    };
    for (int step = 0; step < steps; step += 2) {
      advance(step, s[0], s[1]);
      if (step + 1 == steps) break;
      advance(step + 1, s[1], s[0]);
    }
    wait_loads<0>();  // those past the end too, before the rings are used again
    if (uniform(bad.found)) rows.add_not_finite(bad, lane);
    rows.put(p, it, row, 1, static_cast<int64_t>(item) * M::kRows + 32 * wave + (lane & 31), lane);
  }
}

// ------------------------------------------------------------------ few rows
// A segment of at most 32 rows: what bounds it is how fast its keys come in, for which
// three waves a CU are about enough.  Each wave takes items of its own, in LDS of its own for 32 positions' keys and values;
// the next keys are loaded when these have become scores, the next values when
// these have been summed.  There is no barrier among the waves.  One request of 4096
// positions, 16/2 heads of 256, is bound by what follows one another: 2 us to count the
// items, 3 to the first loads, 3 for a step and its piece, 2 to the joining kernel's
// launch and 6 in it.
template <int D> struct Few {
  static constexpr int kHalf = 32 * 2 * D, kWave = 2 * kHalf, kLoads = kHalf / 1024;
  static constexpr int kLds = 4 * (kWave + static_cast<int>(sizeof(NotFinite<D>))) + static_cast<int>(sizeof(Plan));
  static constexpr int kBlocks = D == 256 ? 1 : D == 128 ? 2 : 3;  // of a CU
  static_assert(kBlocks * kLds <= 160 * 1024, "fits");
};

template <class T, int D>
__device__ __forceinline__ void few_rows(const Attend& p, char* lds, int block, int blocks) {
  using F = Few<D>;
  using R = Rows<T, D>;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  char* const keys = lds + wave * F::kWave;
  char* const values = keys + F::kHalf;
  NotFinite<D>& bad = reinterpret_cast<NotFinite<D>*>(lds + 4 * F::kWave)[wave];
  Plan& plan = *reinterpret_cast<Plan*>(lds + 4 * (F::kWave + sizeof(bad)));
  const bool small = segments_of(p) <= 64;  // the same in all blocks
  Lane mine{};
  const int total = small ? count_few<kFew, 32>(p, mine, block == 0 && wave == 0, lane)
                          : schedule<false, kFew, 32>(p, plan, nullptr, block, blocks);
  const int of_k = lane_k<D>(lane), of_v = lane_v<D>(lane);
  // neighbours in the order of items share keys or a table, or lie side by side: in one
  // block (64 requests of 4096 positions, 32/8 heads of 128: 188 us, 215 with a block's
  // waves far apart); few items on as many CUs as there are (eight requests of 1000, 16/2
  // heads of 256: 16.3 us, 18.3 with four to a block)
  const int each = min(4, (total + kCus - 1) / kCus);
  for (int item = wave < each ? block * each + wave : total; item < total; item += blocks * each) {
    const Item it = small ? item_of_few<32>(p, mine, item) : item_of<false, kFew, 32>(p, plan, item);
    const int end = it.seg.hi, steps = (it.to - it.from + 31) / 32;
    R rows;
    rows.fetch(p, it, lane & 31, lane);
    Spot spot = find(p, it.seg.request, it.from + 16 * lane, end);
    Feed<D> k_feed, v_feed;
    k_feed.start(p.k, it.head, false, lane);
    v_feed.start(p.v, it.head, true, lane);
    Spots k_spots, v_spots;
    // 32 steps to a lookup; a step's keys are loaded before its values
    auto load_k = [&](int step) __attribute__((always_inline)) {
      if ((step & 31) == 0) {
        if (step > 0) spot = find(p, it.seg.request, it.from + 32 * step + 16 * lane, end);
        k_spots.set(spot, k_feed.page, k_feed.token);
        v_spots.set(spot, v_feed.page, v_feed.token);
      }
      const int there = step < steps ? end - (it.from + 32 * step) : 0, which = 2 * (step & 31);
      k_feed.aim(k_spots, which, there);
      k_feed.load_all(keys);
      k_feed.aim(k_spots, which + 1, there - 16);
      k_feed.load_all(keys + 32 * D);
    };
    auto load_v = [&](int step) __attribute__((always_inline)) {
      const int there = step < steps ? end - (it.from + 32 * step) : 0, which = 2 * (step & 31);
      v_feed.aim(v_spots, which, there);
      v_feed.load_all(values);
      v_feed.aim(v_spots, which + 1, there - 16);
      v_feed.load_all(values + 32 * D);
    };
    load_k(0);
    load_v(0);
    rows.clear();
    rows.see(p, it, lane & 31, lane);
    bool searched = false;
    for (int step = 0; step < steps; ++step) {
      f32x16 s[1];
      uint4 w[2];
      typename R::Frag f[R::kAhead];
      const int at = it.from + 32 * step;
      wait_loads<F::kLoads>();  // the keys; the values may be on their way
#pragma unroll
      for (int i = 0; i < R::kAhead; ++i) f[i] = R::template key<1>(keys, of_k, i);
      rows.template scores<1>(keys, of_k, f, s, [](int) __attribute__((always_inline)) {});
      reads_done();
      load_k(step + 1);
      rows.template mask<1>(it.seg, at, lane, s);
      float top = s[0][0];
#pragma unroll
      for (int e = 1; e < 16; ++e) top = fmaxf(top, s[0][e]);
      rows.raise(rows.of_row(p, top));
      rows.template weights<1>(p, 0, 16, rows.subtracted(), s, w);
      rows.template add<1>(0, 16, s);
      wait_loads<F::kLoads>();
      if (rows.template partly<1>(it.seg, at)) {
        if (!searched) bad.clear(lane, 64);
        searched = true;
        take_out<T, D>(values, at, it.seg.lo, bad, lane);
        take_out<T, D>(values + 32 * D, at + 16, it.seg.lo, bad, lane);
      }
#pragma unroll
      for (int i = 0; i < R::kAhead; ++i) f[i] = R::template value<1>(values, of_v, i);
      rows.template values<1>(values, of_v, f, w, [](int) __attribute__((always_inline)) {});
      reads_done();
      load_v(step + 1);
    }
    if (searched && uniform(bad.found)) rows.add_not_finite(bad, lane);
    rows.put(p, it, lane & 31, 0, static_cast<int64_t>(item) * p.few_rows + (lane & 31), lane);
    wait_loads<0>();  // those past the end too
  }
}

// ------------------------------------------------------------------ kernels
template <class T, int D>
__global__ __launch_bounds__(kThreads, Few<D>::kBlocks) void few_rows_kernel(Attend p) {
  __shared__ __align__(1024) char lds[Few<D>::kLds];
  few_rows<T, D>(p, lds, blockIdx.x, gridDim.x);
}
template <class T, int D>
__global__ __launch_bounds__(kThreads, Many<D>::kBlocks) void many_rows_kernel(Attend p) {
  __shared__ __align__(1024) char lds[Many<D>::kShared];
  many_rows<T, D>(p, lds, blockIdx.x, gridDim.x);
}
// Both in one launch, kCus blocks of one and kCus of the other by turns: the first is
// bound by the matrix cores, the second by memory, and where a CU has room for two
// blocks it runs one of each (64 requests of 8 drafts behind four shared prompts,
// 32/8 heads of 128: 116 us, 141 in two launches, one after the other).
template <class T, int D>
__global__ __launch_bounds__(kThreads, Many<D>::kBlocks) void both_kernel(Attend p) {
  constexpr int kShared = Many<D>::kShared > Few<D>::kLds ? Many<D>::kShared : Few<D>::kLds;
  __shared__ __align__(1024) char lds[kShared];
  const int block = (blockIdx.x / (2 * kCus)) * kCus + blockIdx.x % kCus;
  if (blockIdx.x / kCus % 2 == 0)
    many_rows<T, D>(p, lds, block, kCus * Many<D>::kBlocks);
  else
    few_rows<T, D>(p, lds, block, kCus * Many<D>::kBlocks);
}

// ------------------------------------------------------------------ join
// WAVES waves a row: the pieces of the row's shared and own segments by turns, 64 of
// a wave's at a time: a lane looks up one piece, then all lanes add the pieces.  What
// bounds it is the pieces' bytes, or for few rows one load after another: four waves a
// row up to 1024 rows (64 rows of one request of 4096 positions 20.1 us for the call,
// with one wave 23.9; 256 rows 33.0 and 34.7), one from there on (2048 rows 193.9 us with
// four, 192.1 with one).
template <class T, int D, int WAVES>
__global__ __launch_bounds__(kThreads) void join_kernel(Attend p) {
  constexpr int kRowsABlock = kThreads / (64 * WAVES), kLane = D / 64, kBatch = WAVES > 1 ? 16 : 8;  // channels a lane
  typedef float Channels __attribute__((ext_vector_type(kLane)));
  __shared__ float sums[4][D];
  __shared__ float2 stats[4];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const uint32_t at = blockIdx.x * kRowsABlock + (WAVES == 1 ? wave : 0);
  if (at >= static_cast<uint32_t>(p.tokens) * p.heads) return;  // whole waves, and no barrier behind it then
  const int token = p.by_heads.div(at), head = at - token * p.heads;
  const int request = p.cu ? request_of(p, token, lane) : token, shared = p.shared ? p.num_groups : 0;
  const Place own = p.places[shared + request];
  // tokens behind the last request (or before the first) are nobody's: left as they were
  if (token < token_of(p, request) || token >= token_of(p, request + 1)) return;
  const int kv_head = p.by_per.div(head);
  // pieces of the shared segment, then of the own one
  int many[2], first[2], apart[2], count[2], row[2];
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    count[which] = 0;
    if (!which && own.group < 0) continue;
    const Place place = which ? own : p.places[own.group];
    const int in = (token - place.token) * p.per + head - kv_head * p.per, rows = place.tokens * p.per;
    if (in < 0 || in >= rows || place.hi <= place.lo) continue;
    if (which && place.ranges == 1 && place.lo == 0) return;  // the item wrote the row itself
    many[which] = rows > kFew;
    const int tile_rows = many[which] ? Many<D>::kRows : kFew;
    apart[which] = many[which] ? p.kv_heads : 1;
    const int tile = in / tile_rows, back = (rows + tile_rows - 1) / tile_rows - 1 - tile;
    first[which] = place.item + (many[which] ? back * place.ranges * p.kv_heads + kv_head : kv_head * place.ranges);
    row[which] = in % tile_rows;
    count[which] = place.ranges;
  }
  const int pieces = count[0] + count[1];
  float m = -INFINITY, l = 0.f, y[kLane];
#pragma unroll
  for (int e = 0; e < kLane; ++e) y[e] = 0.f;
  for (int base = 0; base < pieces; base += 64 * WAVES) {
    const int piece = base + lane * WAVES + (WAVES == 1 ? 0 : wave);
    float2 st = make_float2(-INFINITY, 0.f);
    uint64_t from = 0;
    if (piece < pieces) {
      const int which = piece >= count[0], kind = which ? many[1] : many[0];
      const int item = which ? first[1] + (piece - count[0]) * apart[1] : first[0] + piece * apart[0];
      const int64_t to = static_cast<int64_t>(clampi(item, 0, p.items_max[kind] - 1)) * (kind ? Many<D>::kRows : p.few_rows) +
                         (which ? row[1] : row[0]);
      st = p.stats[kind][to];
      from = reinterpret_cast<uint64_t>(p.sums[kind] + to * D);
    }
    float top = st.x;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, 64));
    top = fmaxf(top, m);
    const float old = weight_of(m, l, top), mine = weight_of(st.x, st.y, top);
    float sum = st.y * mine;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off, 64);
    l = l * old + sum;
    m = top;
#pragma unroll
    for (int e = 0; e < kLane; ++e) y[e] *= old;
    const int here = (min(pieces - base, 64 * WAVES) + WAVES - 1 - (WAVES == 1 ? 0 : wave)) / WAVES;
    for (int i = 0; i < here; i += kBatch) {
      Channels part[kBatch];
      float weight[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {  // past the last: that one again, unused
        const int k = min(i + j, here - 1);
        const uint32_t low = __builtin_amdgcn_readlane(static_cast<int>(from), k),
                       high = __builtin_amdgcn_readlane(static_cast<int>(from >> 32), k);
        part[j] = reinterpret_cast<const Channels*>(static_cast<uint64_t>(high) << 32 | low)[lane];
        weight[j] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(mine), k));
      }
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        if (i + j < here) {
#pragma unroll
          for (int e = 0; e < kLane; ++e) y[e] = fmaf(part[j][e], weight[j], y[e]);
        }
    }
  }
  if constexpr (WAVES > 1) {
#pragma unroll
    for (int e = 0; e < kLane; ++e) sums[wave][lane * kLane + e] = y[e];
    if (lane == 0) stats[wave] = make_float2(m, l);
    __syncthreads();
    if (wave > 0) return;
    m = -INFINITY, l = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) m = fmaxf(m, stats[w].x);
#pragma unroll
    for (int e = 0; e < kLane; ++e) y[e] = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const float b = weight_of(stats[w].x, stats[w].y, m);
      l += stats[w].y * b;
#pragma unroll
      for (int e = 0; e < kLane; ++e) y[e] += sums[w][lane * kLane + e] * b;
    }
  }
  bool sees = false;
  if (l == 0.f) sees = own.hi > 0 && length_of(p, request) > own.tokens - 1 - (token - own.token);
  const float inverse = inverse_of(l, sees);
  T* to = static_cast<T*>(p.out) + token * p.out_token + head * p.out_head + lane * kLane;
#pragma unroll
  for (int e = 0; e < kLane; ++e) to[e] = from_f32<T>(y[e] * inverse);
  if (p.lse && lane == 0) p.lse[at] = lse_of(m, l);
}

// ------------------------------------------------------------------ host
inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline int64_t aligned(int64_t n) { return (n + 255) / 256 * 256; }

struct Sizes {
  bool few, many;  // whether segments of that kind can be there
  int64_t items[2], target[2], waves, few_rows;
  int64_t sums[2], stats[2], places, bytes;  // offsets
};

// Bounds from what the host knows.  Each item of few rows is one of `target` (a range
// of keys is at least all units over it, but for the rounding of that sum) or the
// last range of a tile; those of many rows may be cut into four times as many.
Sizes sizes_of(int64_t tokens, int64_t requests, int64_t groups, int64_t heads, int64_t kv_heads, int64_t dim,
               bool varlen) {
  Sizes z{};
  const int64_t per = heads / kv_heads, rows = tokens * per, sets = groups > 0 ? 2 : 1;
  z.few = per <= kFew;
  z.many = rows > kFew && (varlen || per > kFew || groups > 0);
  // Of few rows, fewer than run at once: more bring the keys no faster and leave more pieces
  // (64 requests of 4096 positions, 32/8 heads of 128: 188 us, 190 with 4 a CU, 203 with 8;
  // 64 x 8 drafts behind shared prompts 112, 117, 114; on average over 54 batches 2 % less
  // than with 4, 6 % less than with all that run)
  z.target[0] = 3 * kCus;
  z.target[1] = kCus * (dim == 256 ? 1 : 2);  // blocks
  z.waves = 4 * kCus * (dim == 256 ? 1 : dim == 128 || z.many ? 2 : 3);  // of few rows, that run at once
  z.few_rows = varlen || groups > 0 ? kFew : std::min<int64_t>(per, kFew);
  const int64_t few_tiles = std::min(requests, tokens) + std::min(groups, tokens), many_tiles = sets * (rows / 128 + std::min(requests + groups, rows / kFew + 1));
  z.items[0] = z.few ? z.target[0] + z.target[0] / 64 + few_tiles * kv_heads : 0;
  z.items[1] = z.many ? 4 * z.target[1] + many_tiles * kv_heads : 0;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t from = at;
    at += aligned(bytes);
    return from;
  };
  for (int kind = 0; kind < 2; ++kind) {
    const int64_t n = z.items[kind] * (kind ? 128 : z.few_rows);
    z.sums[kind] = take(n * dim * 4);
    z.stats[kind] = take(n * 8);
  }
  z.places = take((requests + groups) * static_cast<int64_t>(sizeof(Place)));
  z.bytes = at;
  return z;
}

template <class T, int D>
int launch_attend(const Attend& p, const Sizes& z, hipStream_t stream) {
  const uint32_t many = kCus * Many<D>::kBlocks;
  if (z.many && z.few)
    both_kernel<T, D><<<2 * many, kThreads, 0, stream>>>(p);
  else if (z.many)
    many_rows_kernel<T, D><<<many, kThreads, 0, stream>>>(p);
  else
    few_rows_kernel<T, D><<<static_cast<uint32_t>(std::max(ceil_div(std::min(z.items[0], z.waves), 4),
                                                           std::min<int64_t>(z.items[0], kCus))),
                            kThreads, 0, stream>>>(p);
  const int64_t rows = static_cast<int64_t>(p.tokens) * p.heads;
  if (rows <= 4 * kCus)
    join_kernel<T, D, 4><<<static_cast<uint32_t>(rows), kThreads, 0, stream>>>(p);
  else
    join_kernel<T, D, 1><<<static_cast<uint32_t>(ceil_div(rows, 4)), kThreads, 0, stream>>>(p);
  return GDN_LAUNCH_CHECK("paged attention");
}

}  // namespace
}  // namespace gdn

using namespace gdn;

extern "C" int64_t gdn_paged_attention_workspace_bytes(int64_t tokens, int64_t requests, int64_t groups, int64_t heads,
                                                       int64_t kv_heads, int64_t dim, int varlen) {
  if (tokens <= 0 || requests <= 0 || groups < 0 || kv_heads <= 0 || heads < kv_heads || dim <= 0) return 0;
  return sizes_of(tokens, requests, groups, heads, kv_heads, dim, varlen != 0).bytes;
}

extern "C" int gdn_paged_attention(const void* q, int64_t q_token_stride, int64_t q_head_stride, int dtype,
                                   int64_t tokens, int64_t heads, int64_t dim, const void* k_cache,
                                   int64_t k_page_stride, int64_t k_token_stride, int64_t k_head_stride,
                                   const void* v_cache, int64_t v_page_stride, int64_t v_token_stride,
                                   int64_t v_head_stride, int64_t kv_heads, int64_t pages, int64_t page_size,
                                   const void* page_table, int table_dtype, int64_t table_row_stride,
                                   int64_t table_width, const void* seq_lens, int lens_dtype, int64_t requests,
                                   const void* shared_lens, int shared_dtype, const void* group_offsets,
                                   int offsets_dtype, int64_t groups, const void* cu_seqlens, int cu_dtype, float scale,
                                   void* out, int64_t out_token_stride, int64_t out_head_stride, float* lse,
                                   void* workspace, int64_t workspace_bytes, void* stream) {
  GDN_REQUIRE(dtype == GDN_BF16 || dtype == GDN_F16, "dtype must be bf16 or f16");
  GDN_REQUIRE(tokens >= 0 && requests >= 0 && heads > 0 && kv_heads > 0 && heads % kv_heads == 0 && pages >= 0 &&
                  table_width >= 0 && groups >= 0,
              "bad shape");
  GDN_REQUIRE(page_size > 0 && page_size % 16 == 0, "pages of a multiple of 16 tokens");
  GDN_REQUIRE(scale > 0.f && scale <= 3.4e38f, "scale must be positive and finite");
  GDN_REQUIRE(cu_seqlens || tokens == requests, "one token for each request without cu_seqlens");
  GDN_REQUIRE(groups == 0 || shared_lens, "groups without shared lengths");
  GDN_REQUIRE(groups <= 1 || group_offsets, "several groups need their offsets");
  if (dim != 64 && dim != 128 && dim != 256) {
    set_error("head dims 64, 128 and 256");
    return GDN_ERR_UNSUPPORTED;
  }
  // the joining kernel's blocks of 256 threads for four rows each: fewer than 2^32 threads
  if (tokens * heads > (int64_t{1} << 26) - 4 || requests + groups >= (int64_t{1} << 24) ||
      table_width * page_size > (int64_t{1} << 27) || pages >= (int64_t{1} << 31) || kv_heads > (1 << 16)) {
    set_error("up to 2^26 - 4 rows, fewer than 2^24 requests, 2^27 positions, 2^31 pages and 2^16 key heads");
    return GDN_ERR_UNSUPPORTED;
  }
  if (tokens == 0 || requests == 0) return GDN_OK;
  GDN_REQUIRE(q && out && (pages == 0 || (k_cache && v_cache)) && seq_lens && (table_width == 0 || page_table),
              "null operand");
  const int codes[] = {table_dtype, lens_dtype, shared_dtype, offsets_dtype, cu_dtype};
  for (int code : codes) GDN_REQUIRE(code == GDN_I32 || code == GDN_I64, "indices must be int32 or int64");
  const int64_t strides[] = {q_token_stride, q_head_stride, k_page_stride, k_token_stride,
                             k_head_stride,  v_page_stride, v_token_stride, v_head_stride};
  for (int64_t n : strides) GDN_REQUIRE(n % 8 == 0, "rows must start at multiples of 16 bytes");
  GDN_REQUIRE(aligned16(q) && aligned16(k_cache) && aligned16(v_cache), "rows must start at multiples of 16 bytes");
  GDN_REQUIRE(out_token_stride % 4 == 0 && out_head_stride % 4 == 0 && reinterpret_cast<uintptr_t>(out) % 8 == 0,
              "rows of out must start at multiples of 8 bytes");
  // 16 positions are addressed by 32-bit byte offsets
  GDN_REQUIRE(k_token_stride >= 0 && v_token_stride >= 0 && k_token_stride < (1 << 24) && v_token_stride < (1 << 24),
              "tokens of a page up to 2^24 elements apart");
  const Sizes z = sizes_of(tokens, requests, groups, heads, kv_heads, dim, cu_seqlens != nullptr);
  GDN_REQUIRE(workspace && workspace_bytes >= z.bytes && reinterpret_cast<uintptr_t>(workspace) % 16 == 0,
              "a workspace of %lld bytes is needed", static_cast<long long>(z.bytes));

  Attend p{};
  p.q = q, p.q_token = q_token_stride, p.q_head = q_head_stride;
  p.k = {k_cache, k_page_stride, k_token_stride, k_head_stride};
  p.v = {v_cache, v_page_stride, v_token_stride, v_head_stride};
  p.table = page_table, p.table_row = table_row_stride, p.table_is64 = table_dtype == GDN_I64;
  p.lens = seq_lens, p.lens_is64 = lens_dtype == GDN_I64;
  if (groups > 0) p.shared = shared_lens, p.shared_is64 = shared_dtype == GDN_I64;
  p.groups = group_offsets, p.groups_is64 = offsets_dtype == GDN_I64;
  p.cu = cu_seqlens, p.cu_is64 = cu_dtype == GDN_I64;
  p.tokens = static_cast<int>(tokens), p.requests = static_cast<int>(requests), p.num_groups = static_cast<int>(groups);
  p.heads = static_cast<int>(heads), p.kv_heads = static_cast<int>(kv_heads), p.per = static_cast<int>(heads / kv_heads);
  p.by_per = make_div32(p.per), p.by_heads = make_div32(heads);
  p.pages = static_cast<int>(pages), p.capacity = static_cast<int>(table_width * page_size);
  p.page = make_div32(page_size);
  p.factor = scale * kLog2e;
  p.out = out, p.out_token = out_token_stride, p.out_head = out_head_stride;
  p.lse = lse;
  char* ws = static_cast<char*>(workspace);
  for (int kind = 0; kind < 2; ++kind) {
    p.sums[kind] = reinterpret_cast<float*>(ws + z.sums[kind]);
    p.stats[kind] = reinterpret_cast<float2*>(ws + z.stats[kind]);
    p.items_max[kind] = static_cast<int>(z.items[kind]);
    p.per_target[kind] = static_cast<float>(static_cast<double>(kv_heads) / static_cast<double>(z.target[kind]));
  }
  p.places = reinterpret_cast<Place*>(ws + z.places);
  p.few_rows = static_cast<int>(z.few_rows);
  auto go = [&](auto type) {
    using T = decltype(type);
    const hipStream_t on = static_cast<hipStream_t>(stream);
    return dim == 64 ? launch_attend<T, 64>(p, z, on) : dim == 128 ? launch_attend<T, 128>(p, z, on)
                                                                   : launch_attend<T, 256>(p, z, on);
  };
  return dtype == GDN_BF16 ? go(bf16{}) : go(f16{});
}
