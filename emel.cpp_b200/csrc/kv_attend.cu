// Attention of a few query rows a request over the pages of the 4-bit key / value cache.
//
// The cache is read once: 18 bytes for 32 values, so HBM bounds it, with about 25 instructions of a warp to each token of a head
// at that rate.  What keeps it under them: the cache is the A operand of mma.sync.m16n8k16 (16 tokens, or 16 dims, a side), the query
// rows of a group of heads the other (8 of them, none of a tile wasted on a group of 8), so tokens and not heads fill the
// tiles; quants become f16 by one lop3 a pair (64 + q; the scores' accumulators start at -72 times the queries' sums, values
// are centred by one addition, since a sum over tokens would not survive the difference); a key's scale multiplies its sum of
// 32 products in f32, a value's scale joins the softmax weight; weights turn from accumulators into operands by movmatrix.
//
// All tiles of 16 tokens of all (request, key / value head, 8 rows) stand in one line, which the units share evenly, whatever the
// requests' lengths.  A unit is a team of 1 to 8 warps, each with a ring of tiles of its own that bulk copies fill; the team
// takes every tile in turn and joins its warps' results in shared memory.  What a unit has of a (request, head) that others
// share goes to scratch, and the last to arrive joins the parts in the units' order, so results do not depend on timing.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "kv_tile.cuh"
#include "paged.h"
#include "tc_common.cuh"

namespace emelb {
namespace {

using kv::Tile;
typedef long long i64;
constexpr unsigned kAll = 0xffffffffu;
constexpr int kWarps = 8, kThreads = 32 * kWarps;
constexpr float kLowest = -3.0e38f;   // running maximum before the first token: finite, below every score
constexpr float kSlack = 3.0f;        // a score may pass the running maximum by this (log2) before sums are rescaled
constexpr int kMinShare = 2;          // tiles a warp, below which fewer units share the work

struct AttendArgs {
  const uint8_t* data;
  const void* q;
  void* out;
  const int32_t *table, *lengths, *query_begin;
  int64_t table_stride, qs, qh, os, oh, page_bytes;
  int requests, table_width, kv_heads, group, queries, max_queries, pages, page_tokens, page_shift, type, q_vec;
  float scale_log2;
  float *acc, *stats;
  int* arrived;
  int most_units;
  int *bad, *status;
};

template <int D, int NT>
struct Shape {
  static constexpr int kRows = 8 * NT;
  static constexpr int kStages = D == 128 ? 4 : D == 96 ? 5 : D == 64 ? 8 : 12;
  static constexpr int kRing = kStages * Tile<D>::kBytes;
  static constexpr int kJoinLd = D + 2;
  static constexpr int kSmem = kWarps * kRing + kWarps * kRows * kJoinLd * 4;
};

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
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
__device__ __forceinline__ void lds(uint32_t (&v)[N], const uint8_t* p) {
  if constexpr (N == 4) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
  } else if constexpr (N == 2) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    v[0] = u.x; v[1] = u.y;
  } else {
    v[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}

__device__ __forceinline__ float load_query(const AttendArgs& a, int64_t at) {
  if (a.type == EMELB_F32) return static_cast<const float*>(a.q)[at];
  if (a.type == EMELB_F16) return __half2float(static_cast<const __half*>(a.q)[at]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(a.q)[at]);
}
__device__ __forceinline__ void store_out(const AttendArgs& a, int64_t at, float v) {
  if (a.type == EMELB_F32) static_cast<float*>(a.out)[at] = v;
  else if (a.type == EMELB_F16) static_cast<__half*>(a.out)[at] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(v);
}

// one request's part of the line
struct Request {
  int rows;     // query rows
  int first;    // the first of them
  int length;   // tokens
  int tiles;    // of one (head, row tile); at least one, so that rows that see nothing are written too
  int sides;    // (head, row tile) pairs
};
template <int ROWS>
__device__ __forceinline__ Request request_at(const AttendArgs& a, int b, bool* wrong) {
  Request r;
  r.first = a.query_begin ? a.query_begin[b] : b;
  r.rows = a.query_begin ? a.query_begin[b + 1] - r.first : 1;
  r.length = a.lengths[b];
  const bool ok = r.rows >= 0 && r.rows <= a.max_queries && r.first >= 0 && r.first <= a.queries - r.rows && r.length >= 0 &&
                  r.length <= (i64)a.table_width * a.page_tokens;
  if (!ok) {
    *wrong = true;
    r.rows = 0;
    r.length = 0;
  }
  r.tiles = max(1, (r.length + 15) >> 4);
  r.sides = a.kv_heads * ((r.rows * a.group + ROWS - 1) / ROWS);
  return r;
}

__device__ __forceinline__ void team_barrier(int team, int threads) {
  if (threads == 32) __syncwarp();
  else asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "r"(threads) : "memory");
}

// kExact: f32 queries and results; the queries and the weights then go in as two f16 operands each
template <int D, int NT, bool kExact>
__global__ void __launch_bounds__(kThreads, NT == 1 && !kExact ? 2 : 1) kv_attend_kernel(const __grid_constant__ AttendArgs a) {
  using T = Tile<D>;
  using S = Shape<D, NT>;
  constexpr int J = T::kGroups, kRows = S::kRows, kStages = S::kStages, kParts = kExact ? 2 : 1;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t bars[kWarps][kStages];
  __shared__ int stage_ok[kWarps][kStages];
  __shared__ i64 sums[2][kWarps];
  __shared__ int start_b[kWarps];
  __shared__ i64 start_at[kWarps];
  __shared__ float join_m[kWarps][kRows], join_l[kWarps][kRows];
  __shared__ int last_in[kWarps];
  __shared__ volatile int gave_up;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  uint8_t* ring = smem + warp * S::kRing;
  float* joint = reinterpret_cast<float*>(smem + kWarps * S::kRing);
  bool wrong = false;

  if (tid < kWarps * kStages) tc::mbar_init(tc::smem_u32(&bars[tid / kStages][tid % kStages]), 1);
  if (tid == 0) gave_up = 0;

  // ---- the line: its length, and where each team of this CTA starts
  i64 mine = 0, sides = 0;
  for (int b = tid; b < a.requests; b += kThreads) {
    const Request r = request_at<kRows>(a, b, &wrong);
    mine += (i64)r.sides * r.tiles;
    sides += r.sides;
  }
  i64 line = mine;
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    line += __shfl_xor_sync(kAll, line, o);
    sides += __shfl_xor_sync(kAll, sides, o);
  }
  if (lane == 0) {
    sums[0][warp] = line;
    sums[1][warp] = sides;
  }
  __syncthreads();
  line = sides = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    line += sums[0][w];
    sides += sums[1][w];
  }
  if (wrong) *a.bad = 1;
  if (line == 0) return;
  // teams as small as their share still covers about one (request, head): joining warps costs less than joining units, and
  // joining nothing least
  const int grid = gridDim.x;
  int team_warps = 1;
  while (team_warps < kWarps && sides * team_warps < (i64)grid * kWarps) team_warps *= 2;
  const int teams = kWarps / team_warps;
  i64 units = min((i64)grid * teams, (line + kMinShare * team_warps - 1) / (kMinShare * team_warps));
  units = min(units, (i64)a.most_units);
  auto start_of = [&](i64 u) { return u * line / units; };
  auto unit_of = [&](i64 x) {
    i64 u = x * units / line;
    while (start_of(u + 1) <= x) ++u;
    return u;
  };
  {
    i64 carry = 0;
    for (int b0 = 0; b0 < a.requests; b0 += kThreads) {
      const int b = b0 + tid;
      bool skip = false;
      i64 v = 0;
      if (b < a.requests) {
        const Request r = request_at<kRows>(a, b, &skip);
        v = (i64)r.sides * r.tiles;
      }
      i64 upto = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const i64 u = __shfl_up_sync(kAll, upto, o);
        if (lane >= o) upto += u;
      }
      __syncthreads();
      if (lane == 31) sums[0][warp] = upto;
      __syncthreads();
      i64 before = carry;
      for (int w = 0; w < kWarps; ++w) {
        if (w < warp) before += sums[0][w];
        carry += sums[0][w];
      }
      upto += before;
      for (int k = 0; k < teams; ++k) {
        const i64 u = (i64)k * grid + blockIdx.x;
        if (u < units) {
          const i64 x = start_of(u);
          if (x >= upto - v && x < upto) {
            start_b[k] = b;
            start_at[k] = x - (upto - v);
          }
        }
      }
    }
  }
  __syncthreads();
  const int team = warp / team_warps, member = warp % team_warps, team_threads = 32 * team_warps;
  const i64 unit = (i64)team * grid + blockIdx.x;
  if (unit >= units) return;
  const i64 lo = start_of(unit), hi = start_of(unit + 1);
  const int mine_tiles = (int)((hi - lo - member + team_warps - 1) / team_warps);   // this warp's: lo + member + k * team_warps

  // ---- copies: lane l of a batch of 32 finds the l-th tile of the warp from there
  int walk_b = start_b[team];
  i64 walk_at = lo - start_at[team];    // where that request begins in the line
  i64 tile_addr = 0;                    // of this lane's tile of the batch; 0: nothing to copy
  auto find_batch = [&](int k0) {
    const i64 x = lo + member + (i64)(k0 + lane) * team_warps;
    tile_addr = 0;
    if (k0 + lane < mine_tiles) {
      bool skip = false;
      int b = walk_b;
      i64 begin = walk_at;
      Request r = request_at<kRows>(a, b, &skip);
      while (x >= begin + (i64)r.sides * r.tiles) {
        begin += (i64)r.sides * r.tiles;
        ++b;
        r = request_at<kRows>(a, b, &skip);
      }
      const i64 at = x - begin;
      const int side = (int)(at / r.tiles), tile = (int)(at - (i64)side * r.tiles), head = side / (r.sides / a.kv_heads);
      if (tile * 16 < r.length) {
        const int page = a.table[b * a.table_stride + (tile * 16 >> a.page_shift)];
        if (page < 0 || page >= a.pages) *a.bad = 1;
        else
          tile_addr = reinterpret_cast<i64>(a.data + page * a.page_bytes +
                                            (int64_t)(head * (a.page_tokens >> 4) + (tile & ((a.page_tokens >> 4) - 1))) * T::kBytes);
      }
      walk_b = b;
      walk_at = begin;
    }
    // the next batch starts from the last lane that found one
    const unsigned found = __ballot_sync(kAll, k0 + lane < mine_tiles);
    const int from = found ? 31 - __clz(found) : 0;
    walk_b = __shfl_sync(kAll, walk_b, from);
    walk_at = __shfl_sync(kAll, walk_at, from);
  };
  auto issue = [&](int k) {
    if ((k & 31) == 0) find_batch(k);
    const i64 addr = __shfl_sync(kAll, tile_addr, k & 31);
    if (lane == 0) {
      const int s = k % kStages;
      const uint32_t bar = tc::smem_u32(&bars[warp][s]);
      stage_ok[warp][s] = addr != 0;
      if (addr) {
        tc::mbar_arrive_expect_tx(bar, T::kBytes);
        tc::bulk_g2s(ring + s * T::kBytes, reinterpret_cast<const void*>(addr), T::kBytes, bar);
      } else {
        tc::mbar_arrive(bar);
      }
    }
  };
  int issued = 0, taken = 0;
  bool alive = true;
  int stuck = 0;                        // the copy whose wait ran out
  for (; issued < kStages && issued < mine_tiles; ++issued) issue(issued);

  // ---- (request, head, row tile) after (request, head, row tile)
  int b = start_b[team];
  i64 begin = lo - start_at[team];
  bool skip = false;
  Request r = request_at<kRows>(a, b, &skip);
  i64 x = lo;
  while (x < hi) {
    while (x >= begin + (i64)r.sides * r.tiles) {
      begin += (i64)r.sides * r.tiles;
      ++b;
      r = request_at<kRows>(a, b, &skip);
    }
    const i64 at = x - begin;
    const int side = (int)(at / r.tiles), tile0 = (int)(at - (i64)side * r.tiles);
    const int row_tiles = r.sides / a.kv_heads, head = side / row_tiles, row0 = (side - head * row_tiles) * kRows;
    const int all_rows = r.rows * a.group;
    const i64 piece_end = min(hi, x - tile0 + r.tiles);

    // queries: this lane's row g of each tile of 8, dims 8t .. 8t+7 of each group
    uint32_t qf[kParts][NT][J][4];
    float offset[NT][J][2];
    int see[NT][2];
    float m[NT][2], l[NT][2], o[NT][D / 16][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int row = row0 + nt * 8 + g;
      const bool live = row < all_rows;
      const int i = live ? row / a.group : 0;
      const int64_t from = (int64_t)(r.first + i) * a.qs + (int64_t)(head * a.group + (live ? row - i * a.group : 0)) * a.qh;
#pragma unroll
      for (int j = 0; j < J; ++j) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = 0.0f;
        if (live) {
          const int64_t at8 = from + 32 * j + 8 * t;
          if (a.q_vec && !kExact) {
            const uint4 u = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.q) + at8);
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if (a.type == EMELB_F16) {
                v[2 * e] = low_of(w[e]);
                v[2 * e + 1] = high_of(w[e]);
              } else {
                v[2 * e] = __uint_as_float(w[e] << 16);
                v[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
              }
            }
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = load_query(a, at8 + e);
          }
        }
        float sum = 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t hi2 = half2_of(v[2 * e], v[2 * e + 1]);
          qf[0][nt][j][e] = hi2;
          sum += low_of(hi2) + high_of(hi2);
          if constexpr (kExact) {
            const uint32_t lo2 = half2_of(v[2 * e] - low_of(hi2), v[2 * e + 1] - high_of(hi2));
            qf[1][nt][j][e] = lo2;
            sum += low_of(lo2) + high_of(lo2);
          }
        }
        sum += __shfl_xor_sync(kAll, sum, 1);
        sum += __shfl_xor_sync(kAll, sum, 2);
        offset[nt][j][0] = -72.0f * __shfl_sync(kAll, sum, 8 * t);
        offset[nt][j][1] = -72.0f * __shfl_sync(kAll, sum, 8 * t + 4);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int rr = row0 + nt * 8 + 2 * t + h;
        see[nt][h] = r.length - r.rows + min(rr, all_rows - 1) / a.group + 1;
        m[nt][h] = kLowest;
        l[nt][h] = 0.0f;
      }
#pragma unroll
      for (int i16 = 0; i16 < D / 16; ++i16)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[nt][i16][e] = 0.0f;
    }
    const int all_see = r.length - r.rows + row0 / a.group + 1;   // the first row's
    int scale_exp = -11;                                          // see below

    for (; taken < mine_tiles; ++taken) {
      const i64 pos = lo + member + (i64)taken * team_warps;
      if (pos >= piece_end) break;
      const int s = taken % kStages;
      if (alive && !tc::mbar_wait(tc::smem_u32(&bars[warp][s]), (taken / kStages) & 1, &gave_up)) {
        alive = false;
        stuck = taken;
        *a.status = 1;
      }
      if (__any_sync(kAll, !alive)) {
        if (alive) stuck = taken;
        alive = false;
        continue;
      }
      const int token0 = (tile0 + (int)(pos - x)) * 16;
      const uint8_t* tile = ring + s * T::kBytes;
      const bool here = stage_ok[warp][s];
      const bool whole = here && token0 + 16 <= all_see;

      // scores: rows are tokens token0 + g and + 8, columns the query rows
      float score[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) score[nt][e] = 0.0f;
      uint32_t kw[2][J];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int jv = 0; jv < J / T::kVecK; ++jv) {
          uint32_t w[T::kVecK];
          lds(w, tile + ((h * (J / T::kVecK) + jv) * 32 + lane) * T::kVecK * 4);
#pragma unroll
          for (int e = 0; e < T::kVecK; ++e) kw[h][jv * T::kVecK + e] = w[e];
        }
      const uint32_t nibbles = tc::in_register(0x00f000f0u), base64 = tc::in_register(0x54005400u);
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const uint32_t w0 = kw[0][j], w1 = kw[1][j];
        const uint32_t a0[4] = {tc::mask_or(w0 << 4, nibbles, base64), tc::mask_or(w1 << 4, nibbles, base64),
                                tc::mask_or(w0, nibbles, base64), tc::mask_or(w1, nibbles, base64)};
        const uint32_t a1[4] = {tc::mask_or(w0 >> 4, nibbles, base64), tc::mask_or(w1 >> 4, nibbles, base64),
                                tc::mask_or(w0 >> 8, nibbles, base64), tc::mask_or(w1 >> 8, nibbles, base64)};
        const float d0 = __half2float(*reinterpret_cast<const __half*>(tile + T::key_scale(0, j) + g * J * 2));
        const float d1 = __half2float(*reinterpret_cast<const __half*>(tile + T::key_scale(8, j) + g * J * 2));
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float c[4] = {offset[nt][j][0], offset[nt][j][1], offset[nt][j][0], offset[nt][j][1]};
#pragma unroll
          for (int part = 0; part < kParts; ++part) {
            mma(c, a0, qf[part][nt][j][0], qf[part][nt][j][1]);
            mma(c, a1, qf[part][nt][j][2], qf[part][nt][j][3]);
          }
          score[nt][0] = fmaf(d0, c[0], score[nt][0]);
          score[nt][1] = fmaf(d0, c[1], score[nt][1]);
          score[nt][2] = fmaf(d1, c[2], score[nt][2]);
          score[nt][3] = fmaf(d1, c[3], score[nt][3]);
        }
      }
      // values' scales of this lane's four tokens
      uint32_t dv[J][2];
#pragma unroll
      for (int j = 0; j < J; ++j) lds(dv[j], tile + T::kScaleV + (t * J + j) * 8);
      if (!whole) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (!here || token0 + g + (e >> 1) * 8 >= see[nt][e & 1]) score[nt][e] = -INFINITY;
        // behind the request's tokens a page holds anything: no weight, and a scale that keeps the product one
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int tok = token0 + 2 * t + 8 * h;
            if (!here || tok >= r.length) dv[j][h] = 0;
            else if (tok + 1 >= r.length) dv[j][h] &= 0xffffu;
          }
      }
      // A weight times a value's scale is rounded to f16, whose range is small: weights are taken times 2^-scale_exp, the
      // running exponent of the largest scale, as part of the running maximum.  Neither changes often.
      uint32_t big = 0;
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) big = tc::h2_bits(__hmax2(tc::bits_h2(big), __habs2(tc::bits_h2(dv[j][h]))));
      const int big_exp = min(4, max((int)((big >> 10) & 31), (int)(big >> 26)) - 15);
      bool moves = big_exp > scale_exp;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          moves |= fmaxf(score[nt][h], score[nt][h + 2]) * a.scale_log2 > m[nt][h] + kSlack;
      if (__any_sync(kAll, moves)) {
        const int e_new = max(scale_exp, __reduce_max_sync(kAll, big_exp));
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float top = fmaxf(score[nt][h], score[nt][h + 2]) * a.scale_log2;
            top = fmaxf(top, __shfl_xor_sync(kAll, top, 4));
            top = fmaxf(top, __shfl_xor_sync(kAll, top, 8));
            top = fmaxf(top, __shfl_xor_sync(kAll, top, 16));
            top = fmaxf(top, m[nt][h]);
            const float f = exp2_fast((m[nt][h] - top) + (float)(scale_exp - e_new));
            m[nt][h] = top;
            l[nt][h] *= f;
#pragma unroll
            for (int i16 = 0; i16 < D / 16; ++i16) {
              o[nt][i16][h] *= f;
              o[nt][i16][h + 2] *= f;
            }
          }
        scale_exp = e_new;
      }
      float weight[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float m0 = m[nt][0] + (float)scale_exp, m1 = m[nt][1] + (float)scale_exp;
        weight[nt][0] = exp2_fast(fmaf(score[nt][0], a.scale_log2, -m0));
        weight[nt][1] = exp2_fast(fmaf(score[nt][1], a.scale_log2, -m1));
        weight[nt][2] = exp2_fast(fmaf(score[nt][2], a.scale_log2, -m0));
        weight[nt][3] = exp2_fast(fmaf(score[nt][3], a.scale_log2, -m1));
        l[nt][0] += weight[nt][0] + weight[nt][2];
        l[nt][1] += weight[nt][1] + weight[nt][3];
      }
      uint32_t pf[NT][2];
      if constexpr (!kExact) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          pf[nt][0] = turn8x8(half2_of(weight[nt][0], weight[nt][1]));
          pf[nt][1] = turn8x8(half2_of(weight[nt][2], weight[nt][3]));
        }
      }
      const uint32_t low4 = tc::in_register(0x000f000fu), base1024 = tc::in_register(0x64006400u);
      const __half2 c72 = __float2half2_rn(-72.0f), c1032 = __float2half2_rn(-1032.0f);
      constexpr int kVV = T::kVecV;
      uint32_t vw[kVV];
#pragma unroll
      for (int j = 0; j < J; ++j) {
        uint32_t bf[kParts][NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          if constexpr (!kExact) {
            bf[0][nt][0] = tc::h2_bits(__hmul2(tc::bits_h2(pf[nt][0]), tc::bits_h2(dv[j][0])));
            bf[0][nt][1] = tc::h2_bits(__hmul2(tc::bits_h2(pf[nt][1]), tc::bits_h2(dv[j][1])));
          } else {
            // in f32, tokens g and g + 8 a lane, then as two f16
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float d = __half2float(*reinterpret_cast<const __half*>(tile + T::kScaleV + ((g >> 1) * J + j) * 8 + (g & 1) * 2 + 4 * h));
              if (!here || token0 + g + 8 * h >= r.length) d = 0.0f;
              const float p0 = weight[nt][2 * h] * d, p1 = weight[nt][2 * h + 1] * d;
              const uint32_t hi2 = half2_of(p0, p1);
              bf[0][nt][h] = turn8x8(hi2);
              bf[kParts - 1][nt][h] = turn8x8(half2_of(p0 - low_of(hi2), p1 - high_of(hi2)));
            }
          }
        }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int i16 = 2 * j + half;
          if (i16 % kVV == 0) lds(vw, tile + T::kV + (i16 / kVV * 32 + lane) * kVV * 4);
          const uint32_t w = vw[i16 % kVV], w8 = w >> 8;
          const uint32_t av[4] = {tc::h2_bits(__hadd2(tc::bits_h2(tc::mask_or(w, low4, base1024)), c1032)),
                                  tc::h2_bits(__hadd2(tc::bits_h2(tc::mask_or(w, nibbles, base64)), c72)),
                                  tc::h2_bits(__hadd2(tc::bits_h2(tc::mask_or(w8, low4, base1024)), c1032)),
                                  tc::h2_bits(__hadd2(tc::bits_h2(tc::mask_or(w8, nibbles, base64)), c72))};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int part = 0; part < kParts; ++part) mma(o[nt][i16], av, bf[part][nt][0], bf[part][nt][1]);
        }
      }
      __syncwarp();
      if (issued < mine_tiles) issue(issued++);
    }

    // ---- the team's warps together
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        m[nt][h] += (float)scale_exp;
#pragma unroll
        for (int s = 4; s < 32; s <<= 1) l[nt][h] += __shfl_xor_sync(kAll, l[nt][h], s);
        if (g == 0) {
          join_m[warp][nt * 8 + 2 * t + h] = m[nt][h];
          join_l[warp][nt * 8 + 2 * t + h] = l[nt][h];
        }
      }
    team_barrier(team, team_threads);
    const int w0 = team * team_warps;
    float* mine_o = joint + warp * kRows * S::kJoinLd;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int row = nt * 8 + 2 * t + h;
        float top = kLowest;
        for (int w = 0; w < team_warps; ++w) top = fmaxf(top, join_m[w0 + w][row]);
        const float f = exp2_fast(m[nt][h] - top);
#pragma unroll
        for (int i16 = 0; i16 < D / 16; ++i16)
          *reinterpret_cast<float2*>(mine_o + row * S::kJoinLd + i16 * 16 + 2 * g) =
              make_float2(o[nt][i16][h] * f, o[nt][i16][h + 2] * f);
      }
    team_barrier(team, team_threads);

    const int ttid = tid - w0 * 32;
    const bool all_of_it = tile0 == 0 && piece_end == x + r.tiles;
    const i64 seg = x - tile0;
    const i64 u0 = all_of_it ? unit : unit_of(seg), u1 = all_of_it ? unit : unit_of(seg + r.tiles - 1);
    const i64 slot = 2 * unit + (unit == u0 ? 1 : 0);
    for (int e = ttid; e < kRows * D / 2; e += team_threads) {
      const int row = e / (D / 2), d = e % (D / 2) * 2;
      float top = kLowest, sum = 0.0f;
      for (int w = 0; w < team_warps; ++w) top = fmaxf(top, join_m[w0 + w][row]);
      float2 v = make_float2(0.0f, 0.0f);
      for (int w = 0; w < team_warps; ++w) {
        const float2 p = *reinterpret_cast<const float2*>(joint + (w0 + w) * kRows * S::kJoinLd + row * S::kJoinLd + d);
        v.x += p.x;
        v.y += p.y;
        sum += join_l[w0 + w][row] * exp2_fast(join_m[w0 + w][row] - top);
      }
      if (all_of_it) {
        const int rr = row0 + row;
        if (rr < all_rows) {
          const int i = rr / a.group;
          const int64_t to = (int64_t)(r.first + i) * a.os + (int64_t)(head * a.group + rr - i * a.group) * a.oh + d;
          const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
          store_out(a, to, v.x * inv);
          store_out(a, to + 1, v.y * inv);
        }
      } else {
        *reinterpret_cast<float2*>(a.acc + (slot * kRows + row) * D + d) = v;
        if (d == 0) *reinterpret_cast<float2*>(a.stats + (slot * kRows + row) * 2) = make_float2(top, sum);
      }
    }
    if (!all_of_it) {
      // the last unit of the (request, head) to arrive joins all parts, in order
      __threadfence();
      team_barrier(team, team_threads);
      if (ttid == 0) {
        const int before = atomicAdd(a.arrived + u0, 1);
        last_in[team] = before == (int)(u1 - u0);
        if (last_in[team]) a.arrived[u0] = 0;
      }
      team_barrier(team, team_threads);
      if (last_in[team]) {
        __threadfence();
        for (int e = ttid; e < kRows * D / 2; e += team_threads) {
          const int row = e / (D / 2), d = e % (D / 2) * 2, rr = row0 + row;
          if (rr >= all_rows) continue;
          float top = kLowest, sum = 0.0f;
          float2 v = make_float2(0.0f, 0.0f);
          for (i64 u = u0; u <= u1; ++u) {
            const i64 at2 = (2 * u + (u == u0 ? 1 : 0)) * kRows + row;
            const float2 ml = __ldcg(reinterpret_cast<const float2*>(a.stats + at2 * 2));
            const float2 p = __ldcg(reinterpret_cast<const float2*>(a.acc + at2 * D + d));
            const float t2 = fmaxf(top, ml.x), keep = exp2_fast(top - t2), f = exp2_fast(ml.x - t2);
            v.x = v.x * keep + p.x * f;
            v.y = v.y * keep + p.y * f;
            sum = sum * keep + ml.y * f;
            top = t2;
          }
          const int i = rr / a.group;
          const int64_t to = (int64_t)(r.first + i) * a.os + (int64_t)(head * a.group + rr - i * a.group) * a.oh + d;
          const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
          store_out(a, to, v.x * inv);
          store_out(a, to + 1, v.y * inv);
        }
      }
    }
    team_barrier(team, team_threads);
    x = piece_end;
  }
  // a wait that ran out leaves copies in flight: they end before the warp does
  if (!alive) {
    volatile int own = 0;
    for (; stuck < issued; ++stuck) {
      own = 0;
      tc::mbar_wait(tc::smem_u32(&bars[warp][stuck % kStages]), (stuck / kStages) & 1, &own);
    }
  }
}

template <int D, int NT, bool kExact>
cudaError_t launch_one(const AttendArgs& a, int sm_count, cudaStream_t st) {
  const int smem = Shape<D, NT>::kSmem;
  cudaError_t e = cudaFuncSetAttribute(kv_attend_kernel<D, NT, kExact>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  kv_attend_kernel<D, NT, kExact><<<sm_count * (NT == 1 && !kExact ? 2 : 1), kThreads, smem, st>>>(a);
  return cudaGetLastError();
}
template <int D>
cudaError_t launch_dim(AttendArgs& a, const KvAttendScratch& s, int sm_count, cudaStream_t st) {
  const int nt = (int64_t)a.max_queries * a.group > 8 ? 2 : 1;
  const uint64_t rows = 8 * nt;
  uint64_t units = s.acc_floats / (2 * rows * D);
  units = units < s.stats_floats / (4 * rows) ? units : s.stats_floats / (4 * rows);
  units = units < s.arrived_ints ? units : s.arrived_ints;
  a.most_units = (int)units;
  if (a.type == EMELB_F32) return nt == 1 ? launch_one<D, 1, true>(a, sm_count, st) : launch_one<D, 2, true>(a, sm_count, st);
  return nt == 1 ? launch_one<D, 1, false>(a, sm_count, st) : launch_one<D, 2, false>(a, sm_count, st);
}

}  // namespace

cudaError_t launch_kv_attend(const emelb_kv_attend_request& r, const KvAttendScratch& s, int sm_count, int* bad, int* status, cudaStream_t st) {
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
  a.page_bytes = (int64_t)emelb_kv_page_bytes(r.cache.head_dim, r.cache.kv_heads, r.cache.page_tokens);
  a.requests = r.requests;
  a.table_width = r.table_width;
  a.kv_heads = r.cache.kv_heads;
  a.group = r.heads / r.cache.kv_heads;
  a.queries = r.queries;
  a.max_queries = r.query_begin ? r.max_queries : 1;
  a.pages = r.cache.pages;
  a.page_tokens = r.cache.page_tokens;
  while ((1 << a.page_shift) < a.page_tokens) ++a.page_shift;
  a.type = r.type;
  const int64_t size = r.type == EMELB_F32 ? 4 : 2;
  a.q_vec = reinterpret_cast<uintptr_t>(r.q) % 16 == 0 && a.qs * size % 16 == 0 && a.qh * size % 16 == 0;
  a.scale_log2 = r.scale * 1.44269504088896340736f;
  a.acc = s.acc;
  a.stats = s.stats;
  a.arrived = s.arrived;
  a.bad = bad;
  a.status = status;
  switch (r.cache.head_dim) {
    case 32: return launch_dim<32>(a, s, sm_count, st);
    case 64: return launch_dim<64>(a, s, sm_count, st);
    case 96: return launch_dim<96>(a, s, sm_count, st);
    default: return launch_dim<128>(a, s, sm_count, st);
  }
}

}  // namespace emelb
