// Attention of a few query rows a request over the pages of the 4-bit key / value cache.
//
// The cache is read once: 18 bytes for 32 values, so HBM bounds it: at its rate the SMs could issue about 25 instructions of a
// warp to each token of a head, and take 19.  What keeps them that few: the cache is the A operand of mma.sync.m16n8k16 (16 tokens, or 16 dims, a side), the query
// rows of a group of heads the other (8 of them, none of a tile wasted on a group of 8), so tokens and not heads fill the
// tiles; quants become f16 by one lop3 a pair, as a power of two + q, and what that is above q - 8 leaves the scores through the
// tensor cores too (one tf32 product a tile), the values by an addition, since sums over tokens would not survive it; a key's scale
// multiplies its sum of 32 products in f32, a value's scale joins the softmax weight; weights turn from accumulators into operands
// by movmatrix.
//
// All steps of 32 tokens of all (request, key / value head, 8 rows) stand in one line, which the units share evenly, whatever the
// requests' lengths.  A unit is a team of 1 to 12 warps, each with a ring of tiles of its own that asynchronous copies fill; the team
// takes every tile in turn and joins its warps' results in shared memory.  What a unit has of a (request, head) that others
// share goes to scratch, and the last to arrive joins the parts in the units' order, so results do not depend on timing.
//
// The tensor cores cut every sum that they add to off, about 2^-22 of it on average: a warp's results move to shared memory every kFold
// steps, by f32 additions that round to nearest.  With one sum all the way, equal values over 131,072 tokens came out 4e-4 too small, over
// 2^20 0.8 %.
//
// 64 requests of 1000 to 8000 tokens, 64 heads on 8 of 128: 139 us with steps of 16 tokens, 131 with 32 (one maximum, one exchange
// for both), 116 with asynchronous copies in place of bulk ones (no barrier to wait at), 94 since a team takes whole pairs where
// that costs no more, 90 with joins in the order of the fragments, 86.5 with a kernel for each type, 89 (3.75 TB/s) since results move to
// shared memory, far scores are rounded and rows have powers of two of their own.  What bounds it is issue:
// about 300 instructions to 16 tokens of a head, two of the four that an SM could issue a cycle.  One document of 100,001 tokens and 16
// rows reads as two tiles of rows, each unpacked for itself: 69 us; both in one warp (registers) 78 for 68 then.  12 warps with 168 registers do better than 16 with
// 128 (105 us).  Small calls are a chain: the line from the lengths, the first tiles from memory, the joins.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

#include "kernels.h"
#include "kv_tile.cuh"
#include "paged.h"
#include "tc_common.cuh"

namespace emelb {
namespace {

using kv::Tile;
typedef long long i64;
constexpr unsigned kAll = 0xffffffffu;
constexpr float kLowest = -3.0e38f;   // running maximum before the first token: finite, below every score
constexpr float kSlack = 3.0f;        // a score may pass the running maximum by this (log2) before sums are rescaled
constexpr float kFarScore = 0x1p20f;  // from here on an f32 score's own rounding may be more than that
constexpr int kJoinSteps = 5;         // what joining the parts of units costs, in steps of a warp: with 0, 16 requests
                                      // of 120 to 600 tokens take 24 us for 11, with 20 as long
constexpr int kMostParts = 6;         // parts of a (head, row tile) up to which a team may be smaller: with 3 the 64 requests above
                                      // take 92 us for 89, with 12 as long
constexpr int kEach = 4;              // requests a lane in the search that a warp makes alone
constexpr int kStep = 32;             // tokens a warp takes at a time: two tiles
constexpr int kFold = 64;             // steps of a warp between two moves of its results: 128 products, 2^-16 of them

struct AttendArgs {
  const uint8_t* data;
  const void* q;
  void* out;
  const int32_t *table, *lengths, *query_begin;
  int64_t table_stride, qs, qh, os, oh;
  int requests, table_width, kv_heads, group, queries, max_queries, pages, page_tokens, page_shift, q_vec, out_pairs;
  float scale_log2;
  float *acc, *stats;
  int* arrived;
  int most_units;
  int* bad;
};

// what results are of: how far a softmax weight times a value's scale is rounded goes by it
enum Kind { kBf16, kF16, kF32 };

template <int D, Kind kind>
struct Shape {
  static constexpr int kWarps = kind == kF32 ? 8 : 12;   // one CTA an SM: 255 registers a thread, or 168
  static constexpr int kRows = 8;
  static constexpr int kStages = D == 128 ? 2 : D == 32 ? 4 : 3;
  static constexpr int kStage = 2 * Tile<D>::kBytes;
  static constexpr int kRing = kStages * kStage;
  static constexpr int kSmem = kWarps * kRing + kWarps * kRows * D * 4 + kWarps * 32 * 16;
};

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
// rows {a0, a1} (k and k + 4 alike) times columns {b0, b1}, as tf32
__device__ __forceinline__ void mma_tf32(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%4,%5}, {%6,%7}, {%8,%8,%8,%8};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ uint32_t tf32_of(float x) {
  uint32_t r;
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(x));
  return r;
}
// (a & kMask) | base in one instruction: the base in a register
template <uint32_t kMask>
__device__ __forceinline__ uint32_t field(uint32_t a, uint32_t base) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(a), "n"(kMask), "r"(base));
  return r;
}
// all as 64 + q
__device__ __forceinline__ void spread_even(uint32_t w, uint32_t b64, uint32_t (&p)[4]) {
  p[0] = field<0x00f000f0u>(w << 4, b64);
  p[1] = field<0x00f000f0u>(w, b64);
  p[2] = field<0x00f000f0u>(w >> 4, b64);
  p[3] = field<0x00f000f0u>(w >> 8, b64);
}
// The four nibbles of either half of a word as f16 pairs: 1024 + q, 64 + q and, of the word moved down by 6, 256 + q and 16 + q.  What
// they are above q - 8:
__host__ __device__ constexpr float above_of(int p) { return p == 0 ? 1032.0f : p == 1 ? 72.0f : p == 2 ? 264.0f : 24.0f; }
struct Bases {
  uint32_t b1024, b64, b256, b16;
};
__device__ __forceinline__ void spread(uint32_t w, const Bases& b, uint32_t (&p)[4]) {
  const uint32_t w6 = w >> 6;
  p[0] = field<0x000f000fu>(w, b.b1024);
  p[1] = field<0x00f000f0u>(w, b.b64);
  p[2] = field<0x003c003cu>(w6, b.b256);
  p[3] = field<0x03c003c0u>(w6, b.b16);
}
__device__ __forceinline__ uint32_t turn8x8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t half2_of(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float low_of(uint32_t v) { return __low2float(tc::bits_h2(v)); }
__device__ __forceinline__ float high_of(uint32_t v) { return __high2float(tc::bits_h2(v)); }

template <int N>
__device__ __forceinline__ void lds(uint32_t (&v)[N], uint32_t at) {
  static_assert(N == 1 || N == 2 || N == 4, "words");
  if constexpr (N == 4)
    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(at));
  else if constexpr (N == 2)
    asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(v[0]), "=r"(v[1]) : "r"(at));
  else
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v[0]) : "r"(at));
}
__device__ __forceinline__ float lds_half(uint32_t at) {
  uint16_t v;
  asm volatile("ld.shared.b16 %0, [%1];" : "=h"(v) : "r"(at));
  return __half2float(__ushort_as_half(v));
}

template <Kind kind>
__device__ __forceinline__ float load_query(const AttendArgs& a, int64_t at) {
  if (kind == kF32) return static_cast<const float*>(a.q)[at];
  if (kind == kF16) return __half2float(static_cast<const __half*>(a.q)[at]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(a.q)[at]);
}
// two neighbouring dims
template <Kind kind>
__device__ __forceinline__ void store_pair(const AttendArgs& a, int64_t at, float x, float y) {
  if (kind == kF32) {
    float* p = static_cast<float*>(a.out) + at;
    p[0] = x;
    p[1] = y;
    return;
  }
  uint32_t two;
  if (kind == kF16) {
    two = half2_of(x, y);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    two = *reinterpret_cast<const uint32_t*>(&h);
  }
  uint16_t* p = static_cast<uint16_t*>(a.out) + at;
  if (a.out_pairs) {
    *reinterpret_cast<uint32_t*>(p) = two;
  } else {
    p[0] = (uint16_t)two;
    p[1] = (uint16_t)(two >> 16);
  }
}

__device__ __forceinline__ void cp_async16_fill(uint32_t to, const uint8_t* from, uint32_t size) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(size) : "memory");
}
// Two tiles behind one another in shared memory, 16 bytes a lane and row of 512; the row where they meet comes from both, the last
// may be short.
template <int kBytes, int kAt>
__device__ __forceinline__ void copy_stage(uint32_t to, const uint8_t* from0, uint32_t size0, const uint8_t* from1, uint32_t size1, int lane) {
  if constexpr (kAt < 2 * kBytes) {
    constexpr bool kFirst = kAt + 512 <= kBytes, kSecond = kAt >= kBytes;
    const bool first = kFirst || (!kSecond && lane * 16 < kBytes - kAt);
    const uint8_t* from = first ? from0 : from1;
    const uint32_t size = first ? size0 : size1;
    if constexpr (kFirst)
      asm volatile("cp.async.cg.shared.global [%0 + %3], [%1 + %4], 16, %2;" ::"r"(to), "l"(from0), "r"(size0), "n"(kAt), "n"(kAt) : "memory");
    else if constexpr (kSecond && kAt + 512 <= 2 * kBytes)
      asm volatile("cp.async.cg.shared.global [%0 + %3], [%1 + %4], 16, %2;" ::"r"(to), "l"(from1), "r"(size1), "n"(kAt), "n"(kAt - kBytes) : "memory");
    else if (kAt + lane * 16 < 2 * kBytes)
      cp_async16_fill(to + kAt, from + (first ? kAt : kAt - kBytes), size);
    copy_stage<kBytes, kAt + 512>(to, from0, size0, from1, size1, lane);
  }
}

// Places on the line are ints where the request's sizes leave it shorter than 2^30 steps (with 64 bits everywhere one document of
// 100,001 tokens took 71.3 us for 67.1, calls of few tokens 0.6 to 1 us more).  Sums over the requests that are more than the most are
// taken for values out of range.  2^40 steps are a quarter of an hour; a unit's share of them still counts in 31 bits, since there are
// 148 units at least, with 2^26 steps a pair.
template <class Line>
constexpr i64 kMostSteps = sizeof(Line) == 4 ? 0x3fffffff : (i64)1 << 40;
constexpr int kMostPairs = 1 << 30;
constexpr int kMostTokens = 0x7fffffc0;   // of a request: places up to the end of its last step are ints
// a / b, mostly of small numbers; a >= 0
__device__ __forceinline__ int quot(int a, int b) { return a / b; }
__device__ __forceinline__ i64 quot(i64 a, int b) { return (uint64_t)a >> 32 ? a / b : (i64)((uint32_t)a / (uint32_t)b); }

// one request's part of the line
struct Request {
  int rows;     // query rows
  int first;    // the first of them
  int length;   // tokens
  int steps;    // of one (head, row tile); at least one, so that rows that see nothing are written too
  int sides;    // (head, row tile) pairs
};
template <int ROWS>
__device__ __forceinline__ Request request_at(const AttendArgs& a, int b, bool* wrong) {
  Request r;
  r.first = a.query_begin ? a.query_begin[b] : b;
  r.rows = a.query_begin ? a.query_begin[b + 1] - r.first : 1;
  r.length = a.lengths[b];
  const bool ok = r.rows >= 0 && r.rows <= a.max_queries && r.first >= 0 && r.first <= a.queries - r.rows && r.length >= 0 &&
                  r.length <= kMostTokens && r.length <= (i64)a.table_width * a.page_tokens;
  if (!ok) {
    *wrong = true;
    r.rows = 0;
    r.length = 0;
  }
  r.steps = max(1, (r.length + kStep - 1) / kStep);
  r.sides = a.kv_heads * ((r.rows * a.group + ROWS - 1) / ROWS);
  return r;
}

__device__ __forceinline__ void team_barrier(int team, int threads) {
  if (threads == 32) __syncwarp();
  else asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "r"(threads) : "memory");
}

// kF32: the queries and the weights go in as two f16 operands each.  kF16: a weight's low part goes into its product with the scale,
// so that there is one rounding to f16 and not two (one document of 100,001 tokens: 3 us of 70, its error against exact results 1.3
// and not 1.6 times what the results' own rounding makes)
template <int D, Kind kind, class Line>
__global__ void __launch_bounds__(32 * Shape<D, kind>::kWarps, 1) kv_attend_kernel(const __grid_constant__ AttendArgs a) {
  pdl_trigger();
  pdl_wait();
  using T = Tile<D>;
  using S = Shape<D, kind>;
  constexpr int kWarps = S::kWarps, kThreads = 32 * kWarps;
  constexpr bool kExact = kind == kF32, kFine = kind == kF16;
  constexpr int J = T::kGroups, kRows = S::kRows, kStages = S::kStages, kParts = kExact ? 2 : 1;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ i64 sums[3][kWarps];
  constexpr bool kFar = sizeof(Line) == 8;
  struct Sum {
    Line steps;
    int pairs;
  };
  struct Start {
    Line begin, from, to;   // where the request begins, the team's steps
    int b;
  };
  auto line_of = [](const Request& r) { return (Line)r.sides * r.steps; };
  __shared__ Sum scan[kWarps];
  __shared__ Start starts[kWarps];
  __shared__ __align__(16) float join_m[kWarps][kRows], join_l[kWarps][kRows];
  __shared__ int last_in[kWarps];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  uint8_t* ring = smem + warp * S::kRing;
  const uint32_t ring_at = tc::smem_u32(ring) + lane * 16;
  float4* joint = reinterpret_cast<float4*>(smem + kWarps * S::kRing);
  constexpr int kCells = kRows * D / 4;
  float4* folded = joint + kWarps * kCells;   // maximum and sum of a lane's two rows in what has moved
  bool wrong = false;

  // ---- the line: its length, and where each team of this CTA starts
  const int grid = gridDim.x;
  int team_warps, units, share, more;
  bool split;
  // From the sums over the requests (all: steps; sides: (head, row tile) pairs; most: steps of the longest): if a team each can
  // take the pairs whole in about the time that even shares and joining the units' parts (worth about kJoinSteps steps) take,
  // they do; else teams are as small as kMostParts parts a pair allow, since a team waits for its slowest warp at every pair.
  auto plan = [&](Line all, int sides, int most) {
    const int warps = grid * kWarps;
    split = true;
    for (team_warps = kWarps; team_warps >= 1; --team_warps)
      if (kWarps % team_warps == 0 && (i64)sides * team_warps <= warps && (most + team_warps - 1) / team_warps <= quot(all, warps) + kJoinSteps) {
        split = false;
        break;
      }
    if (!split) {
      units = sides;
      return;
    }
    team_warps = 1;
    while (team_warps < kWarps && (kWarps % team_warps != 0 || (i64)sides * team_warps * kMostParts < warps)) ++team_warps;
    units = (int)min((Line)min(warps / team_warps, a.most_units), quot(all + team_warps - 1, team_warps));
    share = (int)quot(all, units);
    more = (int)(all - (Line)share * units);   // the first `more` units take one step more
  };
  auto start_of = [&](int u) { return (Line)u * share + min(u, more); };
  auto unit_of = [&](Line x) {
    const Line edge = (Line)more * (share + 1);
    return x < edge ? (int)quot(x, share + 1) : more + (int)quot(x - edge, share);
  };
  int team, member, unit, b_start;
  Line b_begin, lo, hi;
  if (a.requests <= 32 * kEach) {
    // every warp for itself, a few requests a lane
    Request each[kEach];
    i64 steps = 0;
    int pairs = 0, most = 0;
    const int per = (a.requests + 31) >> 5;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      each[i] = Request{};
      if (i < per && lane * per + i < a.requests) each[i] = request_at<kRows>(a, lane * per + i, &wrong);
    }
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      steps += (i64)each[i].sides * each[i].steps;
      pairs += each[i].sides;
      if (kFar) pairs = min(pairs, kMostPairs);
      if (each[i].sides) most = max(most, each[i].steps);
    }
    const int my_pairs = pairs;
    const i64 my_steps = steps;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const i64 s = __shfl_up_sync(kAll, steps, o);
      const int p = __shfl_up_sync(kAll, pairs, o);
      if (lane >= o) {
        steps += s;
        pairs = kFar ? (int)min((unsigned)pairs + (unsigned)p, (unsigned)kMostPairs) : pairs + p;
      }
    }
    most = __reduce_max_sync(kAll, most);
    const i64 all = __shfl_sync(kAll, steps, 31);
    const int sides = __shfl_sync(kAll, pairs, 31);
    const bool much = all > kMostSteps<Line> || (kFar && sides >= kMostPairs);
    if (wrong || much) *a.bad = 1;
    if (all == 0 || much) return;
    plan((Line)all, sides, most);
    team = warp / team_warps;
    unit = team * grid + blockIdx.x;
    if (unit >= units) return;
    const Line from = split ? start_of(unit) : unit;
    const int owner = __ffs(__ballot_sync(kAll, (split ? (Line)steps : pairs) > from)) - 1;
    // in the owner's few
    Line at = (Line)(steps - my_steps);
    int first_pair = pairs - my_pairs, long_pair = 0, i = 0;
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      const Line n = line_of(each[k]);
      if (i == k) {
        if (split ? at + n <= from : first_pair + each[k].sides <= from) {
          at += n;
          first_pair += each[k].sides;
          ++i;
        } else {
          long_pair = each[k].steps;
        }
      }
    }
    b_start = __shfl_sync(kAll, lane * per + i, owner);
    b_begin = __shfl_sync(kAll, at, owner);
    first_pair = __shfl_sync(kAll, first_pair, owner);
    long_pair = __shfl_sync(kAll, long_pair, owner);
    lo = split ? from : b_begin + (Line)(unit - first_pair) * long_pair;
    hi = split ? start_of(unit + 1) : lo + long_pair;
  } else {
    i64 all = 0, sides = 0;
    int most = 0;
    for (int b = tid; b < a.requests; b += kThreads) {
      const Request r = request_at<kRows>(a, b, &wrong);
      all += (i64)r.sides * r.steps;
      sides += r.sides;
      if (r.sides) most = max(most, r.steps);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      all += __shfl_xor_sync(kAll, all, o);
      sides += __shfl_xor_sync(kAll, sides, o);
    }
    most = __reduce_max_sync(kAll, most);
    if (lane == 0) {
      sums[0][warp] = all;
      sums[1][warp] = sides;
      sums[2][warp] = most;
    }
    __syncthreads();
    all = sides = 0;
    most = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      all += sums[0][w];
      sides += sums[1][w];
      most = max(most, (int)sums[2][w]);
    }
    const bool much = all > kMostSteps<Line> || sides >= kMostPairs;
    if (wrong || much) *a.bad = 1;
    if (all == 0 || much) return;
    plan((Line)all, (int)sides, most);
    const int teams = kWarps / team_warps;
    Line carry_s = 0;
    int carry_p = 0;
    for (int b0 = 0; b0 < a.requests; b0 += kThreads) {
      const int b = b0 + tid;
      bool skip = false;
      Request r{};
      if (b < a.requests) r = request_at<kRows>(a, b, &skip);
      const Line v = line_of(r);
      Line steps = v;
      int pairs = r.sides;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const Line s = __shfl_up_sync(kAll, steps, o);
        const int p = __shfl_up_sync(kAll, pairs, o);
        if (lane >= o) {
          steps += s;
          pairs += p;
        }
      }
      if (b0) __syncthreads();
      if (lane == 31) scan[warp] = Sum{steps, pairs};
      __syncthreads();
      Line before_s = carry_s;
      int before_p = carry_p;
      for (int w = 0; w < kWarps; ++w) {
        const Sum c = scan[w];
        if (w < warp) {
          before_s += c.steps;
          before_p += c.pairs;
        }
        carry_s += c.steps;
        carry_p += c.pairs;
      }
      steps += before_s;
      pairs += before_p;
      for (int k = 0; k < teams; ++k) {
        const int u = k * grid + blockIdx.x;
        if (u >= units) break;
        const Line x = split ? start_of(u) : u;
        if (split ? x >= steps - v && x < steps : x >= pairs - r.sides && x < pairs) {
          const Line from = split ? x : steps - v + (x - (pairs - r.sides)) * r.steps;
          starts[k] = Start{steps - v, from, split ? start_of(u + 1) : from + r.steps, b};
        }
      }
    }
    __syncthreads();
    team = warp / team_warps;
    unit = team * grid + blockIdx.x;
    if (unit >= units) return;
    const Start& s = starts[team];
    b_start = s.b;
    b_begin = s.begin;
    lo = s.from;
    hi = s.to;
  }
  member = warp % team_warps;
  const int team_threads = 32 * team_warps, span = (int)(hi - lo);   // places in the share count from lo
  const int mine_steps = (span - member + team_warps - 1) / team_warps;   // this warp's: lo + member + k * team_warps

  // ---- copies: lane l of a batch of 32 finds the l-th step of the warp from there, one batch ahead, so that nobody waits for
  // the table
  const int page_tiles = a.page_tokens >> 4;
  int walk_b = b_start;
  Line walk_at = b_begin;                     // a request at or before the batch's first step, where it begins
  uint32_t ahead[2] = {0, 0}, now[2] = {0, 0};   // tiles of this lane's step, counted through the cache, twice and 1; 0: none
  auto find_batch = [&](int k0) {
    const Line x = lo + member + (k0 + lane) * team_warps;
    const bool mine_too = k0 + lane < mine_steps;
    ahead[0] = ahead[1] = 0;
    if (mine_too) {
      bool skip = false;
      int b = walk_b;
      Line begin = walk_at;
      Request r = request_at<kRows>(a, b, &skip);
      while (x >= begin + line_of(r)) {
        begin += line_of(r);
        ++b;
        r = request_at<kRows>(a, b, &skip);
      }
      const int side = (int)quot(x - begin, r.steps), step = (int)(x - begin - (Line)side * r.steps), head = side / (r.sides / a.kv_heads);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int tile = 2 * step + h;
        if (tile * 16 < r.length) {
          const int page = a.table[b * a.table_stride + (tile * 16 >> a.page_shift)];
          if (page < 0 || page >= a.pages) *a.bad = 1;
          else ahead[h] = ((uint32_t)(page * a.kv_heads + head) * page_tiles + (tile & (page_tiles - 1))) << 1 | 1;
        }
      }
      walk_b = b;
      walk_at = begin;
    }
    // the next batch starts from the last lane that found one
    const unsigned found = __ballot_sync(kAll, mine_too);
    const int from = found ? 31 - __clz(found) : 0;
    walk_b = __shfl_sync(kAll, walk_b, from);
    walk_at = __shfl_sync(kAll, walk_at, from);
  };
  // 16 bytes a lane; a tile that is not there is filled with zeros
  const uint8_t* from_lane = a.data + lane * 16;
  auto issue = [&](int k, int s) {
    if (k < mine_steps) {
      if ((k & 31) == 0) {
        now[0] = ahead[0];
        now[1] = ahead[1];
      }
      const uint32_t t0 = __shfl_sync(kAll, now[0], k & 31), t1 = __shfl_sync(kAll, now[1], k & 31);
      const uint32_t to = ring_at + s * S::kStage;
      copy_stage<T::kBytes, 0>(to, from_lane + (uint64_t)(t0 >> 1) * T::kBytes, (t0 & 1) << 4, from_lane + (uint64_t)(t1 >> 1) * T::kBytes, (t1 & 1) << 4, lane);
      // the next batch's places, while there is time
      if ((k & 31) == kStages && k + 32 - kStages < mine_steps) find_batch(k + 32 - kStages);
    }
    cp_async_commit();
  };
  int taken = 0, stage = 0;             // steps done, the stage of the next
  // lanes past the last group, or past the values' scales, look at another's (times 0, or once more)
  const int lane_v = lane % (8 * J), own_scale = (g * J + t % J) * 2;
  const Bases bases{tc::in_register(0x64006400u), tc::in_register(0x54005400u), tc::in_register(0x5c005c00u), tc::in_register(0x4c004c00u)};
  constexpr uint32_t above[4] = {0xe408e408u, 0xd480d480u, 0xdc20dc20u, 0xce00ce00u};   // -1032, -72, -264, -24

  // ---- (request, head, row tile) after (request, head, row tile)
  int b = b_start;
  Line begin = b_begin;
  bool skip = false;
  Request r = request_at<kRows>(a, b, &skip);
  int x = 0;
  while (x < span) {
    while (lo + x >= begin + line_of(r)) {
      begin += line_of(r);
      ++b;
      r = request_at<kRows>(a, b, &skip);
    }
    const int side = (int)quot(lo + x - begin, r.steps), step0 = (int)(lo + x - begin - (Line)side * r.steps);
    const int row_tiles = r.sides / a.kv_heads, head = side / row_tiles, row0 = (side - head * row_tiles) * kRows;
    const int all_rows = r.rows * a.group;
    const int piece_end = min(span, x - step0 + r.steps);

    // queries: this lane's row g of each tile of 8, dims 8t .. 8t+7 of each group
    uint32_t qf[kParts][J][4];
    uint32_t off[2];                                          // of group t and row g, as two tf32
    int see[2];
    float m[2], cap[2], l[2], o[D / 16][4];
    const int row = row0 + g;
    const bool live = row < all_rows;
    const int i = live ? row / a.group : 0;
    const int64_t from = (int64_t)(r.first + i) * a.qs + (int64_t)(head * a.group + (live ? row - i * a.group : 0)) * a.qh;
    off[0] = off[1] = 0;
    uint4 raw[J];
    if (!kExact && a.q_vec) {
#pragma unroll
      for (int j = 0; j < J; ++j) raw[j] = live ? *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.q) + from + 32 * j + 8 * t) : make_uint4(0, 0, 0, 0);
    }
    if (x == 0) {   // the first tiles, while the first queries are on their way
      find_batch(0);
      for (int k = 0; k < kStages; ++k) issue(k, k);
    }
    float all_v[J][8];
#pragma unroll
    for (int j = 0; j < J; ++j) {
      float (&v)[8] = all_v[j];
      if (!kExact && a.q_vec) {
        const uint32_t w[4] = {raw[j].x, raw[j].y, raw[j].z, raw[j].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[2 * e] = kFine ? low_of(w[e]) : __uint_as_float(w[e] << 16);
          v[2 * e + 1] = kFine ? high_of(w[e]) : __uint_as_float(w[e] & 0xffff0000u);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = live ? load_query<kind>(a, from + 32 * j + 8 * t + e) : 0.0f;
      }
    }
    // f16 reaches less far than bf16 and f32: a row goes in times the power of two (at most 2^126) that takes its largest value to
    // 2^13 .. 2^14, and its scores come out times the inverse.  Values 2^27 below it are still normal f16 numbers.
    float largest = 0.0f;
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) largest = fmaxf(largest, fabsf(all_v[j][e]) < INFINITY ? fabsf(all_v[j][e]) : 0.0f);
    largest = fmaxf(largest, __shfl_xor_sync(kAll, largest, 1));
    largest = fmaxf(largest, __shfl_xor_sync(kAll, largest, 2));
    const uint32_t expo = __float_as_uint(largest) >> 23;
    const int power = expo ? min(126, 140 - (int)expo) : 0;       // of row g
    const float raise = __uint_as_float((uint32_t)(127 + power) << 23);
    float unit_score[2];                                          // of rows 2t and 2t + 1
#pragma unroll
    for (int h = 0; h < 2; ++h)
      unit_score[h] = fminf(fmaxf(a.scale_log2 * __uint_as_float((uint32_t)(127 - __shfl_sync(kAll, power, 8 * t + 4 * h)) << 23), 1.2e-38f), 3.0e38f);
#pragma unroll
    for (int j = 0; j < J; ++j) {
      float (&v)[8] = all_v[j];
      float sum = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] *= raise;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t hi2 = half2_of(v[2 * e], v[2 * e + 1]);
        qf[0][j][e] = hi2;
        float two = low_of(hi2) + high_of(hi2);
        if constexpr (kExact) {
          const uint32_t lo2 = half2_of(v[2 * e] - low_of(hi2), v[2 * e + 1] - high_of(hi2));
          qf[1][j][e] = lo2;
          two += low_of(lo2) + high_of(lo2);
        }
        sum = fmaf(kExact ? -72.0f : -above_of(e), two, sum);
      }
      sum += __shfl_xor_sync(kAll, sum, 1);
      sum += __shfl_xor_sync(kAll, sum, 2);
      if (t == j) {
        off[0] = tf32_of(sum);
        off[1] = tf32_of(sum - __uint_as_float(off[0]));
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int rr = min(row0 + 2 * t + h, all_rows - 1);
      see[h] = r.length - r.rows + rr / a.group + 1;
      m[h] = cap[h] = kLowest;
      l[h] = 0.0f;
    }
#pragma unroll
    for (int i16 = 0; i16 < D / 16; ++i16)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i16][e] = 0.0f;
    const int all_see = r.length - r.rows + row0 / a.group + 1;   // the first row's
    // A weight times a value's scale is rounded to f16, whose range is small: weights are taken times 2^-scale_exp as part of what scores
    // are taken against, -neg_m, so that products with the largest scale so far reach 2^15 and f16's grid ends 2^35 below that scale:
    // scale_exp is its exponent less 11, -11 at least, where weights themselves reach 2^14, and 4 at most.  cap: the score that moves the
    // running maximum m; scale_cap: the scale that moves scale_exp, 2^(scale_exp + 12).  Neither happens often.
    // A score is rounded to f32 before -neg_m is taken away, as m was when that was made: of far scores the rounding alone, which a fused
    // multiply-add would leave in, may be so much that weights overflow.  For them cap is the largest, without slack, and -neg_m
    // is rounded up, since it must not fall behind m by more than scale_exp.
    constexpr auto cap_of = [](int exp) { return (uint32_t)(exp + 27) * 0x04000400u; };   // of 4: infinity
    uint32_t scale_cap = cap_of(-11);
    float neg_m[2] = {-kLowest, -kLowest};
    const int piece_stop = max(taken, (piece_end - member + team_warps - 1) / team_warps);
    bool moved = false;

    for (;;) {
      for (const int stop = min(piece_stop, taken + kFold); taken < stop; ++taken) {
        const int pos = member + taken * team_warps;
        cp_async_wait<kStages - 1>();
        __syncwarp();
        const int token0 = (step0 + pos - x) * kStep;
        const uint32_t tiles = tc::smem_u32(ring) + stage * S::kStage;
        const uint32_t at_k = tiles + lane * T::kVecK * 4, at_v = tiles + lane * T::kVecV * 4, at_scale = tiles + g * J * 2, at_own = tiles + own_scale,
                       at_word = tiles + lane_v * 4, at_dv = tiles + t * J * 8;
        const bool whole = token0 + kStep <= all_see;

        // scores: rows are tokens token0 + 16 u + g and + 8, columns the query rows
        float score[2][4];
        uint32_t word[2];                   // this lane's share of the values' scales
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int tile = u * T::kBytes;
          uint32_t one[1];
          lds(one, at_word + tile + T::kScaleV);
          word[u] = one[0] & 0x7fff7fffu;
          uint32_t kw[2][J];
          float dk[2][J];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int jv = 0; jv < J / T::kVecK; ++jv) {
              uint32_t w[T::kVecK];
              lds(w, at_k + tile + (h * (J / T::kVecK) + jv) * 32 * T::kVecK * 4);
#pragma unroll
              for (int e = 0; e < T::kVecK; ++e) kw[h][jv * T::kVecK + e] = w[e];
            }
            const uint32_t sc = at_scale + tile + T::key_scale(8 * h, 0);
            if constexpr (J % 2 == 0) {
              uint32_t w[J / 2];
              lds(w, sc);
#pragma unroll
              for (int e = 0; e < J / 2; ++e) {
                dk[h][2 * e] = low_of(w[e]);
                dk[h][2 * e + 1] = high_of(w[e]);
              }
            } else {
#pragma unroll
              for (int j = 0; j < J; ++j) dk[h][j] = lds_half(sc + 2 * j);
            }
          }
          // the scales times what the operands are above q - 8, of all groups at once (k is the groups, twice), then group by group
          const float d0 = lds_half(at_own + tile + T::key_scale(0, 0)), d1 = lds_half(at_own + tile + T::key_scale(8, 0));
          mma_tf32(score[u], __float_as_uint(d0), __float_as_uint(d1), off[0], off[1]);
#pragma unroll
          for (int j = 0; j < J; ++j) {
            uint32_t p0[4], p1[4];
            if constexpr (kExact) {   // 22 bits of a score's sum of 32 are left below 64 + q, 18 below 1024 + q
              spread_even(kw[0][j], bases.b64, p0);
              spread_even(kw[1][j], bases.b64, p1);
            } else {
              spread(kw[0][j], bases, p0);
              spread(kw[1][j], bases, p1);
            }
            const uint32_t a0[4] = {p0[0], p1[0], p0[1], p1[1]}, a1[4] = {p0[2], p1[2], p0[3], p1[3]};
            float c[4];
            mma_first(c, a0, qf[0][j][0], qf[0][j][1]);
            mma(c, a1, qf[0][j][2], qf[0][j][3]);
            if constexpr (kExact) {
              mma(c, a0, qf[kParts - 1][j][0], qf[kParts - 1][j][1]);
              mma(c, a1, qf[kParts - 1][j][2], qf[kParts - 1][j][3]);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) score[u][e] = fmaf(dk[e >> 1][j], c[e], score[u][e]);
          }
        }
        if (!whole) {
          // behind the request's tokens a page holds anything: no weight, and no say in the exponent
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int t0 = token0 + 16 * u;
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (t0 + g + (e >> 1) * 8 >= see[e & 1]) score[u][e] = -INFINITY;
            const int tok = t0 + lane_v / (2 * J) * 2 + (lane_v & 1) * 8;
            if (tok >= r.length) word[u] = 0;
            else if (tok + 1 >= r.length) word[u] &= 0xffffu;
          }
        }
        // a half of `word` that reaches scale_cap keeps the bit above it
        bool moves = ((((word[0] | 0x80008000u) - scale_cap) | ((word[1] | 0x80008000u) - scale_cap)) & 0x80008000u) != 0;
#pragma unroll
        for (int h = 0; h < 2; ++h)
          moves |= fmaxf(fmaxf(score[0][h], score[0][h + 2]), fmaxf(score[1][h], score[1][h + 2])) > cap[h];
        if (__any_sync(kAll, moves)) {
          int big = (int)max(max(word[0] & 0xffffu, word[0] >> 16), max(word[1] & 0xffffu, word[1] >> 16)) >> 10;
          big = min(4, __reduce_max_sync(kAll, big) - 15 - 11);
          const int e_new = max((int)(scale_cap >> 26) - 27, big);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float top = fmaxf(fmaxf(score[0][h], score[0][h + 2]), fmaxf(score[1][h], score[1][h + 2]));
            top = fmaxf(top, __shfl_xor_sync(kAll, top, 4));
            top = fmaxf(top, __shfl_xor_sync(kAll, top, 8));
            top = fmaxf(top, __shfl_xor_sync(kAll, top, 16));
            m[h] = fmaxf(__fmul_rn(top, unit_score[h]), m[h]);
            cap[h] = fabsf(m[h]) < kFarScore ? (m[h] + kSlack) / unit_score[h] : fmaxf(cap[h], top);
            const float now = -__fadd_ru(m[h], (float)e_new), f = exp2_fast(now - neg_m[h]);
            neg_m[h] = now;
            l[h] *= f;
#pragma unroll
            for (int i16 = 0; i16 < D / 16; ++i16) {
              o[i16][h] *= f;
              o[i16][h + 2] *= f;
            }
          }
          scale_cap = cap_of(e_new);
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
          for (int e = 0; e < 4; e += 2) {
            const float2 x = tc::unpack2(tc::mul2(tc::pack2(score[u][e], score[u][e + 1]), tc::pack2(unit_score[0], unit_score[1])));
            score[u][e] = exp2_fast(__fadd_rn(x.x, neg_m[0]));
            score[u][e + 1] = exp2_fast(__fadd_rn(x.y, neg_m[1]));
          }
          l[0] += score[u][0] + score[u][2];
          l[1] += score[u][1] + score[u][3];
        }
        constexpr int kVV = T::kVecV;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int tile = u * T::kBytes, t0 = token0 + 16 * u;
          // scales of this lane's four tokens, and the weights as operands
          uint32_t dv[J][2], pf[2], low[2];
          if constexpr (J % 2 == 0) {
#pragma unroll
            for (int j = 0; j < J; j += 2) {
              uint32_t w[4];
              lds(w, at_dv + tile + T::kScaleV + j * 8);
              dv[j][0] = w[0]; dv[j][1] = w[1]; dv[j + 1][0] = w[2]; dv[j + 1][1] = w[3];
            }
          } else {
#pragma unroll
            for (int j = 0; j < J; ++j) lds(dv[j], at_dv + tile + T::kScaleV + j * 8);
          }
          if (!whole) {
#pragma unroll
            for (int j = 0; j < J; ++j)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const int tok = t0 + 2 * t + 8 * h;
                if (tok >= r.length) dv[j][h] = 0;
                else if (tok + 1 >= r.length) dv[j][h] &= 0xffffu;
              }
          }
          if constexpr (!kExact) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t two = half2_of(score[u][2 * h], score[u][2 * h + 1]);
              pf[h] = turn8x8(two);
              if constexpr (kFine) low[h] = turn8x8(half2_of(score[u][2 * h] - low_of(two), score[u][2 * h + 1] - high_of(two)));
            }
          }
          uint32_t vw[kVV];
#pragma unroll
          for (int j = 0; j < J; ++j) {
            uint32_t bf[kParts][2];
            if constexpr (!kExact) {
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const __half2 d = tc::bits_h2(dv[j][h]);
                const __half2 p = kFine ? __hfma2(tc::bits_h2(pf[h]), d, __hmul2(tc::bits_h2(low[h]), d)) : __hmul2(tc::bits_h2(pf[h]), d);
                bf[0][h] = tc::h2_bits(p);
              }
            } else {
              // in f32, tokens g and g + 8 a lane, then as two f16
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                float d = lds_half(tiles + tile + T::kScaleV + ((g >> 1) * J + j) * 8 + (g & 1) * 2 + 4 * h);
                if (t0 + g + 8 * h >= r.length) d = 0.0f;
                const float p0 = score[u][2 * h] * d, p1 = score[u][2 * h + 1] * d;
                const uint32_t hi2 = half2_of(p0, p1);
                bf[0][h] = turn8x8(hi2);
                bf[kParts - 1][h] = turn8x8(half2_of(p0 - low_of(hi2), p1 - high_of(hi2)));
              }
            }
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const int i16 = 2 * j + half;
              if (i16 % kVV == 0) lds(vw, at_v + tile + T::kV + i16 / kVV * 32 * kVV * 4);
              uint32_t av[4];
              spread(vw[i16 % kVV], bases, av);
              // centred before the product, exactly: a sum over the tokens would not survive the difference
#pragma unroll
              for (int e = 0; e < 4; ++e) av[e] = tc::h2_bits(__hadd2(tc::bits_h2(av[e]), tc::bits_h2(above[e])));
#pragma unroll
              for (int part = 0; part < kParts; ++part) mma(o[i16], av, bf[part][0], bf[part][1]);
            }
          }
        }
        __syncwarp();
        issue(taken + kStages, stage);
        stage = stage + 1 == kStages ? 0 : stage + 1;
      }
      if (taken == piece_stop) break;
      // to where the team's results meet in the end, which is free until then
      const float4 old = folded[tid];
      const float m0 = -neg_m[0], m1 = -neg_m[1];
      const float f0 = moved ? exp2_fast(old.x - m0) : 0.0f, f1 = moved ? exp2_fast(old.z - m1) : 0.0f;
      folded[tid] = make_float4(m0, moved ? fmaf(old.y, f0, l[0]) : l[0], m1, moved ? fmaf(old.w, f1, l[1]) : l[1]);
      l[0] = l[1] = 0.0f;
#pragma unroll
      for (int i16 = 0; i16 < D / 16; ++i16) {
        float4& cell = joint[warp * kCells + i16 * 32 + lane];
        float4 now = make_float4(o[i16][0], o[i16][1], o[i16][2], o[i16][3]);
        if (moved) {
          const float4 was = cell;
          now = make_float4(fmaf(was.x, f0, now.x), fmaf(was.y, f1, now.y), fmaf(was.z, f0, now.z), fmaf(was.w, f1, now.w));
        }
        cell = now;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i16][e] = 0.0f;
      }
      moved = true;
    }

    // ---- the piece's results.  A cell is what a lane holds of 16 dims: rows 2t and 2t + 1, dims 16 i + 2g and the next.  Cells stay in
    // this order all the way: through shared memory, through scratch, until the last sum is made
    m[0] = -neg_m[0];
    m[1] = -neg_m[1];
    if (moved) {
      const float4 old = folded[tid];
      const float f0 = exp2_fast(old.x - m[0]), f1 = exp2_fast(old.z - m[1]);
      l[0] = fmaf(old.y, f0, l[0]);
      l[1] = fmaf(old.w, f1, l[1]);
#pragma unroll
      for (int i16 = 0; i16 < D / 16; ++i16) {
        const float4 was = joint[warp * kCells + i16 * 32 + lane];
        o[i16][0] = fmaf(was.x, f0, o[i16][0]);
        o[i16][1] = fmaf(was.y, f1, o[i16][1]);
        o[i16][2] = fmaf(was.z, f0, o[i16][2]);
        o[i16][3] = fmaf(was.w, f1, o[i16][3]);
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int s = 4; s < 32; s <<= 1) l[h] += __shfl_xor_sync(kAll, l[h], s);
    const int w0 = team * team_warps, ttid = tid - w0 * 32;
    if (team_warps > 1) {
      if (g == 0) *reinterpret_cast<float2*>(&join_m[warp][2 * t]) = make_float2(m[0], m[1]);
      team_barrier(team, team_threads);
      float f[2];
      float2 top = make_float2(kLowest, kLowest);
#pragma unroll 4
      for (int w = 0; w < team_warps; ++w) {
        const float2 o_m = *reinterpret_cast<const float2*>(&join_m[w0 + w][2 * t]);
        top.x = fmaxf(top.x, o_m.x);
        top.y = fmaxf(top.y, o_m.y);
      }
      f[0] = exp2_fast(m[0] - top.x);
      f[1] = exp2_fast(m[1] - top.y);
      m[0] = top.x;
      m[1] = top.y;
      if (g == 0) *reinterpret_cast<float2*>(&join_l[warp][2 * t]) = make_float2(l[0] * f[0], l[1] * f[1]);
#pragma unroll
      for (int i16 = 0; i16 < D / 16; ++i16)
        joint[warp * kCells + i16 * 32 + lane] =
            make_float4(o[i16][0] * f[0], o[i16][1] * f[1], o[i16][2] * f[0], o[i16][3] * f[1]);
      team_barrier(team, team_threads);
      l[0] = l[1] = 0.0f;
#pragma unroll 4
      for (int w = 0; w < team_warps; ++w) {
        const float2 o_l = *reinterpret_cast<const float2*>(&join_l[w0 + w][2 * t]);
        l[0] += o_l.x;
        l[1] += o_l.y;
      }
    }
    auto cell_of = [&](int c, int i16) {
      if (team_warps == 1) return make_float4(o[i16][0], o[i16][1], o[i16][2], o[i16][3]);
      float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
      for (int w = 0; w < team_warps; ++w) {
        const float4 u = joint[(w0 + w) * kCells + c];
        v.x += u.x;
        v.y += u.y;
        v.z += u.z;
        v.w += u.w;
      }
      return v;
    };
    // rows 2t and 2t + 1 where they are any
    int64_t to[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int rr = row0 + 2 * t + h, i = see[h] - 1 - (r.length - r.rows);
      to[h] = rr < all_rows ? (int64_t)(r.first + i) * a.os + (int64_t)(head * a.group + rr - i * a.group) * a.oh + 2 * g : -1;
    }
    auto put = [&](int i16, const float4& v, float inv0, float inv1) {
      if (to[0] >= 0) store_pair<kind>(a, to[0] + i16 * 16, v.x * inv0, v.z * inv0);
      if (to[1] >= 0) store_pair<kind>(a, to[1] + i16 * 16, v.y * inv1, v.w * inv1);
    };
    auto inverse = [](float sum) { return sum == 0.0f ? 0.0f : 1.0f / sum; };
    const bool all_of_it = step0 == 0 && piece_end == x + r.steps;
    const Line seg = lo + x - step0;
    const int u0 = all_of_it ? unit : unit_of(seg), u1 = all_of_it ? unit : unit_of(seg + r.steps - 1);
    auto part_of = [&](int u) { return 2 * (i64)u + (u == u0 ? 1 : 0); };
    float4* acc = reinterpret_cast<float4*>(a.acc);
    float4* stats = reinterpret_cast<float4*>(a.stats);
#pragma unroll
    for (int k = 0, turn = 0; k < kCells / 32; ++k) {
      const bool others = turn != member;
      turn = turn + 1 == team_warps ? 0 : turn + 1;
      if (others) continue;
      const int c = k * 32 + lane;
      const float4 v = cell_of(c, k);
      if (all_of_it) put(k, v, inverse(l[0]), inverse(l[1]));
      else __stcg(acc + part_of(unit) * kCells + c, v);
    }
    if (!all_of_it) {
      if (member == 0 && g == 0) __stcg(stats + part_of(unit) * (kRows / 2) + t, make_float4(m[0], l[0], m[1], l[1]));
      // the last unit of the (request, head) to arrive joins all parts, in their order
      team_barrier(team, team_threads);
      if (ttid == 0) {
        __threadfence();
        const int last = atomicAdd(a.arrived + u0, 1) == u1 - u0;
        if (last) a.arrived[u0] = 0;
        __threadfence();
        last_in[team] = last;
      }
      team_barrier(team, team_threads);
      if (last_in[team]) {
        // this warp's cells, so many at once and of so many parts that about 16 loads are on their way
        auto join = [&](auto cells, auto parts) {
          constexpr int kAtOnce = decltype(cells)::value, kUnroll = decltype(parts)::value;
          float2 top = make_float2(kLowest, kLowest), sum = make_float2(0.0f, 0.0f);
          float4 v[kAtOnce];
#pragma unroll
          for (int q = 0; q < kAtOnce; ++q) v[q] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll kUnroll
          for (int u = u0; u <= u1; ++u) {
            const float4 ml = __ldcg(stats + part_of(u) * (kRows / 2) + t);
            float4 p[kAtOnce];
#pragma unroll
            for (int q = 0; q < kAtOnce; ++q)
              if (member + q * team_warps < D / 16) p[q] = __ldcg(acc + part_of(u) * kCells + (member + q * team_warps) * 32 + lane);
            const float2 next = make_float2(fmaxf(top.x, ml.x), fmaxf(top.y, ml.z));
            const float k0 = exp2_fast(top.x - next.x), k1 = exp2_fast(top.y - next.y), f0 = exp2_fast(ml.x - next.x), f1 = exp2_fast(ml.z - next.y);
            sum.x = sum.x * k0 + ml.y * f0;
            sum.y = sum.y * k1 + ml.w * f1;
            top = next;
#pragma unroll
            for (int q = 0; q < kAtOnce; ++q)
              if (member + q * team_warps < D / 16) {
                v[q].x = fmaf(v[q].x, k0, p[q].x * f0);
                v[q].y = fmaf(v[q].y, k1, p[q].y * f1);
                v[q].z = fmaf(v[q].z, k0, p[q].z * f0);
                v[q].w = fmaf(v[q].w, k1, p[q].w * f1);
              }
          }
          sum = make_float2(inverse(sum.x), inverse(sum.y));
#pragma unroll
          for (int q = 0; q < kAtOnce; ++q)
            if (member + q * team_warps < D / 16) put(member + q * team_warps, v[q], sum.x, sum.y);
        };
        if (team_warps * 2 < D / 16) join(std::integral_constant<int, D / 16>{}, std::integral_constant<int, 2>{});
        else if (member < D / 16) join(std::integral_constant<int, 2>{}, std::integral_constant<int, 8>{});
      }
    }
    x = piece_end;
    if (x < span) team_barrier(team, team_threads);   // before the next piece's results
  }
}

template <int D, Kind kind, class Line>
cudaError_t launch_line(const AttendArgs& a, int sm_count, bool pdl, cudaStream_t st) {
  using S = Shape<D, kind>;
  const int smem = S::kSmem;
  cudaError_t e = cudaFuncSetAttribute(kv_attend_kernel<D, kind, Line>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  return launch_kernel(kv_attend_kernel<D, kind, Line>, dim3(sm_count), dim3(32 * S::kWarps), smem, st, pdl, a);
}
template <int D, Kind kind>
cudaError_t launch_one(const AttendArgs& a, int sm_count, bool pdl, cudaStream_t st) {
  // the most that requests in order may come to: row tiles as each may have them, or as all of the rows do, and whole rows of the table
  constexpr int kRows = Shape<D, kind>::kRows;
  const i64 each = ((i64)a.max_queries * a.group + kRows - 1) / kRows;
  const i64 tiles = std::min<i64>(a.requests * each, (i64)a.queries * a.group / kRows + a.requests);
  const i64 steps = (std::min<i64>((i64)a.table_width * a.page_tokens, kMostTokens) + kStep - 1) / kStep;
  const bool far = tiles * a.kv_heads > kMostSteps<int> / steps;
  return far ? launch_line<D, kind, i64>(a, sm_count, pdl, st) : launch_line<D, kind, int>(a, sm_count, pdl, st);
}
template <int D>
cudaError_t launch_dim(AttendArgs& a, int type, const KvAttendScratch& s, int sm_count, bool pdl, cudaStream_t st) {
  constexpr uint64_t rows = 8;
  uint64_t units = s.acc_floats / (2 * rows * D);
  units = units < s.stats_floats / (4 * rows) ? units : s.stats_floats / (4 * rows);
  units = units < s.arrived_ints ? units : s.arrived_ints;
  a.most_units = (int)units;
  if (type == EMELB_F32) return launch_one<D, kF32>(a, sm_count, pdl, st);
  return type == EMELB_F16 ? launch_one<D, kF16>(a, sm_count, pdl, st) : launch_one<D, kBf16>(a, sm_count, pdl, st);
}

}  // namespace

cudaError_t launch_kv_attend(const emelb_kv_attend_request& r, const KvAttendScratch& s, int sm_count, int* bad, bool pdl, cudaStream_t st) {
  AttendArgs a{};
  a.data = static_cast<const uint8_t*>(r.cache.data);
  a.q = r.q;
  a.out = r.out;
  a.table = r.table;
  a.lengths = r.lengths;
  a.query_begin = r.query_begin;
  a.table_stride = r.table_stride;
  a.qs = r.q_token_stride;
  a.qh = r.q_head_stride;
  a.os = r.out_token_stride;
  a.oh = r.out_head_stride;
  a.requests = r.requests;
  a.table_width = r.table_width;
  a.kv_heads = r.cache.kv_heads;
  a.group = r.heads / r.cache.kv_heads;
  a.queries = r.queries;
  a.max_queries = r.query_begin ? r.max_queries : 1;
  a.pages = r.cache.pages;
  a.page_tokens = r.cache.page_tokens;
  while ((1 << a.page_shift) < a.page_tokens) ++a.page_shift;
  const int64_t size = r.type == EMELB_F32 ? 4 : 2;
  a.q_vec = reinterpret_cast<uintptr_t>(r.q) % 16 == 0 && a.qs * size % 16 == 0 && a.qh * size % 16 == 0;
  a.out_pairs = reinterpret_cast<uintptr_t>(r.out) % 4 == 0 && a.os % 2 == 0 && a.oh % 2 == 0;
  a.scale_log2 = r.scale * 1.44269504088896340736f;
  a.acc = s.acc;
  a.stats = s.stats;
  a.arrived = s.arrived;
  a.bad = bad;
  switch (r.cache.head_dim) {
    case 32: return launch_dim<32>(a, r.type, s, sm_count, pdl, st);
    case 64: return launch_dim<64>(a, r.type, s, sm_count, pdl, st);
    case 96: return launch_dim<96>(a, r.type, s, sm_count, pdl, st);
    default: return launch_dim<128>(a, r.type, s, sm_count, pdl, st);
  }
}

}  // namespace emelb
