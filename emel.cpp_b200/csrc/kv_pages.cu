// Pages of the 4-bit key / value cache: the plan of a step, rows into their slots, rows back out.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "kernels.h"
#include "kv_tile.cuh"
#include "paged.h"

namespace emelb {
namespace {

using kv::kTile;
using kv::Tile;
typedef long long i64;

// ------------------------------------------------------------------ plan
// Three running sums over the requests (tokens, pages lacking, pages given back) decide everything else: new page j is
// entry top - 1 - j of the stack that the ended requests' pages lie on, and row i's request is found by bisection.  Every CTA
// takes the sums for itself, since that is cheaper than handing them over, and then its share of the pages, of the rows, which
// look a new page up where it comes from and not in the table, or of what is left, so that no CTA waits for another.  What is read
// and what is written do not meet, but for `lengths` and free_left where they are `cached` and free_count: with more than one CTA
// those wait in scratch for a second launch.
//
// 1000 requests, 121,984 rows: 10.3 us one behind the other, 12.4 with pages, rows and the requests' numbers in the same CTAs, 21 by a
// cluster of 8 CTAs with a barrier between pages and rows.  Its 1.6 MB take 0.3 us of bandwidth: what is left is a chain, in cycles
// first reads 2,200, sums 3,500, a row's bisection, page and stores 5,400, and the launch.
constexpr int kPlanMost = EMELB_KV_MAX_REQUESTS;
constexpr unsigned kAll = 0xffffffffu;

// inclusive sums over the block; `carry` comes in and goes out as the sums of all blocks of requests so far
template <int N>
__device__ __forceinline__ void block_sums(i64 (&v)[N], i64 (&carry)[N], i64 (*warp_sums)[32]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1)
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const i64 u = __shfl_up_sync(kAll, v[k], o);
      if (lane >= o) v[k] += u;
    }
  if (lane == 31)
#pragma unroll
    for (int k = 0; k < N; ++k) warp_sums[k][warp] = v[k];
  __syncthreads();
  i64 w[N];
#pragma unroll
  for (int k = 0; k < N; ++k) w[k] = lane < warps ? warp_sums[k][lane] : 0;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1)
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const i64 u = __shfl_up_sync(kAll, w[k], o);
      if (lane >= o) w[k] += u;
    }
#pragma unroll
  for (int k = 0; k < N; ++k) {
    v[k] += carry[k] + (warp ? __shfl_sync(kAll, w[k], max(warp - 1, 0)) : 0);
    carry[k] += __shfl_sync(kAll, w[k], 31);
  }
  __syncthreads();
}

// first request whose running sum is above x
__device__ __forceinline__ int owner_of(const int* upto, int n, int x) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (upto[mid] > x) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

__device__ __forceinline__ int clip(i64 v) { return (int)(v < 0 ? 0 : v > 0x7fffffff ? 0x7fffffff : v); }

struct PlanArgs {
  emelb_kv_plan_request r;
  int *lengths, *free_left;   // the request's own, or scratch
  int page_shift;
  int* bad;
};

__global__ void __launch_bounds__(512) kv_plan_kernel(const __grid_constant__ PlanArgs a) {
  pdl_trigger();
  pdl_wait();
  extern __shared__ int plan_smem[];
  __shared__ i64 warp_sums[3][32];
  __shared__ int most_taken;
  const emelb_kv_plan_request& r = a.r;
  const int n = r.requests, P = r.page_tokens, shift = a.page_shift, tid = threadIdx.x, T = blockDim.x;
  // one CTA for all, or some for the rows, as many for the pages and one for the requests' numbers
  const int ranks = max(((int)gridDim.x - 1) / 2, 1), rank = blockIdx.x % ranks;
  const bool alone = gridDim.x == 1, has_rows = blockIdx.x < ranks, has_pages = alone || (blockIdx.x >= ranks && blockIdx.x < 2 * ranks);
  int* tok = plan_smem;         // running sums, each request's own included
  int* need = tok + n;
  int* back = need + n;
  int* had = back + n;          // tokens cached; complemented where the request gets nothing
  const i64 room = (i64)r.table_width * P;
  bool wrong = false;
  if (tid == 0) most_taken = 0;

  i64 all[3] = {0, 0, 0};   // tokens, pages lacking, pages given back
  const int free_count = *r.free_count;
  // a thread has `per` neighbouring requests: their sums from its first on, then what stands before that
  const int per = (n + T - 1) / T, b_first = min(n, tid * per), b_last = min(n, b_first + per);
  i64 mine[3] = {0, 0, 0};
#pragma unroll 4
  for (int b = b_first; b < b_last; ++b) {
    i64 cached = r.cached[b];
    const i64 fresh = r.fresh[b];
    const bool ok = cached >= 0 && fresh >= -1 && cached + (fresh > 0 ? fresh : 0) <= room, ended = fresh < 0;
    wrong |= !ok;
    cached = cached < 0 ? 0 : cached > room ? room : cached;
    const int have = (int)((cached + P - 1) >> shift);
    mine[0] += ended ? 0 : fresh;
    mine[1] += ok && !ended ? ((cached + fresh + P - 1) >> shift) - have : 0;
    mine[2] += ok && ended ? have : 0;
    tok[b] = clip(mine[0]);
    need[b] = clip(mine[1]);
    back[b] = clip(mine[2]);
    had[b] = ok ? (int)cached : ~(int)cached;
  }
  i64 upto[3] = {mine[0], mine[1], mine[2]};
  block_sums(upto, all, warp_sums);
  for (int b = b_first; b < b_last; ++b) {
    const i64 rows_upto = upto[0] - mine[0] + tok[b];
    tok[b] = clip(rows_upto);
    need[b] = clip(upto[1] - mine[1] + need[b]);
    back[b] = clip(upto[2] - mine[2] + back[b]);
    if (rows_upto > r.token_capacity && had[b] >= 0 && r.fresh[b] >= 0) {   // no rows for them, nor for any behind
      had[b] = ~had[b];
      wrong = true;
    }
  }
  const i64 tok_sum = all[0], need_sum = all[1], back_sum = all[2];
  __syncthreads();
  i64 count = free_count;
  if (count < 0 || count > r.pages) {
    wrong = true;
    count = count < 0 ? 0 : r.pages;
  }
  const i64 top = count + back_sum;
  int taken = 0;
  for (int b = tid; b < n; b += T) {
    const int lacks = need[b] - (b ? need[b - 1] : 0);
    if (had[b] >= 0 && lacks > 0) {
      if (need[b] <= top) taken = need[b];
      else had[b] = ~had[b];
    }
  }
  taken = __reduce_max_sync(kAll, taken);
  if ((tid & 31) == 0 && taken) atomicMax(&most_taken, taken);
  __syncthreads();
  taken = most_taken;

  // new page j: from the top of the stack, or of what the ended requests lay on it
  auto new_page = [&](int j) {
    const i64 at = top - 1 - j;
    if (at < count) return r.free_pages[at];
    const int x = (int)(at - count), e = owner_of(back, n, x);
    return r.table[e * r.table_stride + (x - (e ? back[e - 1] : 0))];
  };
  // shares by warps in turn, so that every CTA has some of the rows that cost most
  const int step = ranks * T, me = ((tid >> 5) * ranks + rank) * 32 + (tid & 31);
  for (int j = has_pages ? me : taken; j < taken; j += step) {
    const int b = owner_of(need, n, j), page = new_page(j);
    if (page < 0 || page >= r.pages) wrong = true;
    r.table[b * r.table_stride + ((had[b] + P - 1) >> shift) + (j - (b ? need[b - 1] : 0))] = page;
  }
  // what the ended requests gave back and nobody took
  for (i64 x = has_pages ? me : top; x < top - taken - count; x += step) {
    const int e = owner_of(back, n, (int)x);
    const int page = r.table[e * r.table_stride + (x - (e ? back[e - 1] : 0))];
    if (count + x < r.pages) r.free_pages[count + x] = page;
    if (count + x >= r.pages || page < 0 || page >= r.pages) wrong = true;
  }
  // slots and positions: four neighbouring rows a thread, of which the first is searched for
  const int total = clip(tok_sum < r.token_capacity ? tok_sum : r.token_capacity);
  const bool wide = reinterpret_cast<uintptr_t>(r.slots) % 16 == 0 && reinterpret_cast<uintptr_t>(r.positions) % 16 == 0;
  for (int i0 = has_rows ? 4 * me : 0x7fffffff; i0 < r.token_capacity; i0 = i0 > 0x7fffffff - 4 * step ? 0x7fffffff : i0 + 4 * step) {
    i64 slot[4];
    int p[4], page[4], b = i0 < total ? owner_of(tok, n, i0) : 0;
    constexpr i64 kNew = (i64)1 << 62;
    i64 entry[4];                     // in the table, or the number of a new page
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      entry[e] = -1;
      p[e] = 0;
      if (i0 + e < total) {
        while (tok[b] <= i0 + e) ++b;
        const int h = had[b];
        p[e] = (h < 0 ? ~h : h) + i0 + e - (b ? tok[b - 1] : 0);
        const int col = p[e] >> shift, have = (h + P - 1) >> shift;
        if (h >= 0) entry[e] = col < have ? b * r.table_stride + col : kNew | ((b ? need[b - 1] : 0) + col - have);
      }
    }
    // a page once for its rows: mostly one or two of them, which the warp's lanes look up together
    for (unsigned left = 15; left;) {
      const i64 at = left & 1 ? entry[0] : left & 2 ? entry[1] : left & 4 ? entry[2] : entry[3];
      const int found = at < 0 ? 0 : at < kNew ? r.table[at] : new_page((int)(at & ~kNew));
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (entry[e] == at) {
          page[e] = found;
          left &= ~(1u << e);
        }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const bool sound = page[e] >= 0 && page[e] < r.pages;
      if (!sound) wrong = true;
      slot[e] = entry[e] >= 0 && sound ? ((i64)page[e] << shift) + (p[e] & (P - 1)) : -1;
    }
    if (wide && i0 + 3 < r.token_capacity) {
      *reinterpret_cast<longlong2*>(r.slots + i0) = make_longlong2(slot[0], slot[1]);
      *reinterpret_cast<longlong2*>(r.slots + i0 + 2) = make_longlong2(slot[2], slot[3]);
      *reinterpret_cast<int4*>(r.positions + i0) = make_int4(p[0], p[1], p[2], p[3]);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (i0 + e < r.token_capacity) {
          r.slots[i0 + e] = slot[e];
          r.positions[i0 + e] = p[e];
        }
    }
  }
  // each request's numbers; the barriers of the sums stand between reads and writes of one CTA
  if (blockIdx.x == gridDim.x - 1) {
    auto length_of = [&](int b) {
      const int h = had[b];
      return r.fresh[b] < 0 ? 0 : h >= 0 ? h + (tok[b] - (b ? tok[b - 1] : 0)) : ~h;
    };
    i64 key_sum[1] = {0}, keys[1] = {0};
#pragma unroll 4
    for (int b = b_first; b < b_last; ++b) keys[0] += length_of(b);
    i64 at = -keys[0];
    block_sums(keys, key_sum, warp_sums);
    at += keys[0];
    for (int b = b_first; b < b_last; ++b) {
      const int len = length_of(b);
      at += len;
      a.lengths[b] = len;
      r.query_begin[b + 1] = tok[b] < r.token_capacity ? tok[b] : r.token_capacity;
      r.key_begin[b + 1] = clip(at);
      if (at > 0x7fffffff) wrong = true;
    }
    if (tid == 0) {
      r.query_begin[0] = 0;
      r.key_begin[0] = 0;
      *a.free_left = clip(top - taken);
      *r.shortage = clip(need_sum > top ? need_sum - top : 0);
    }
  }
  if (wrong) *a.bad = 1;
}

__global__ void __launch_bounds__(256) kv_plan_in_place_kernel(const int* lengths, const int* free_left, int n, int* to_lengths, int* to_free_left) {
  pdl_trigger();
  pdl_wait();
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i < n) to_lengths[i] = lengths[i];
  if (i == 0) *to_free_left = *free_left;
}

// ------------------------------------------------------------------ elements
template <class E>
struct Elem;
template <>
struct Elem<float> {
  static __device__ __forceinline__ float in(float x) { return x; }
  static __device__ __forceinline__ float out(float x) { return x; }
};
template <>
struct Elem<__half> {
  static __device__ __forceinline__ float in(__half x) { return __half2float(x); }
  static __device__ __forceinline__ __half out(float x) { return __float2half_rn(x); }
};
template <>
struct Elem<__nv_bfloat16> {
  static __device__ __forceinline__ float in(__nv_bfloat16 x) { return __bfloat162float(x); }
  static __device__ __forceinline__ __nv_bfloat16 out(float x) { return __float2bfloat16_rn(x); }
};

// 8 values of a row, by 16-byte loads where the rows allow them
template <class E>
struct Eight {
  __align__(16) E e[8];
  template <bool kVec>
  __device__ __forceinline__ void load(const E* p) {
    if constexpr (kVec) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(e) / 16; ++i) reinterpret_cast<uint4*>(e)[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = p[i];
    }
  }
  template <bool kVec>
  __device__ __forceinline__ void store(E* p) const {
    if constexpr (kVec) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(e) / 16; ++i) reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(e)[i];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) p[i] = e[i];
    }
  }
};

// ------------------------------------------------------------------ store
// A CTA takes 16 packed rows of a head, or of several in turn where there are CTAs enough.  Four lanes share a group of 32 values, 8
// each, which is a word of keys; the scale comes from the group's largest value by two shuffles.  Values go by bytes, each with its
// own address: they wait in shared memory until a warp can store one pair of dims of 16 rows at a time, which are neighbours where
// the rows fill a tile.
// 32,760 rows of 8 heads of 128 f16: 43 us (4.0 TB/s), 47 with a CTA for each head and rows of either alignment in one kernel, 50
// with the largest value looked for one by one; with its reader 154 when quotients were divisions, 97 by reciprocals.  Issue bounds
// it, 130 instructions to 8 values of a warp; memory alone would take 26.
struct StoreArgs {
  uint8_t* data;
  const void *k, *v;
  const int64_t* slots;
  int64_t ks, kh, vs, vh, limit, page_bytes;
  int tokens, heads, per, page_shift;   // per: heads of a CTA
  int* bad;
};

// the larger, the smaller of either half's values; NaN if one is
template <class E>
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
  uint32_t r;
  if (std::is_same<E, __half>::value) asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <class E>
__device__ __forceinline__ uint32_t min2(uint32_t a, uint32_t b) {
  uint32_t r;
  if (std::is_same<E, __half>::value) asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

constexpr float kMagic = 12582912.0f;   // 1.5 * 2^23: a sum with it has the rounded addend in its low bits

// The scale of the group and the quants of this lane's 8 values, in the low bits of `bits`.
//
// q = floor(x / d + 8.5) within 0 .. 15 is the rounded x / d + 8, ties upwards.  With x and d of 11 bits or fewer a quotient that is
// no tie is at least 2^-12 from one: x * (1 / d) + 8 + 2^-16, off by 2^-19, rounds to the right side of it.  Clamping is left to
// the multiply-add's saturation, of the sum over 15.25.  f32 values may be closer: the borders (c - 8.5) d and (c - 7.5) d, exact in
// f32, are looked at.
template <class E>
__device__ __forceinline__ void quantize8(const Eight<E>& in, __half& scale, uint32_t (&bits)[8]) {
  float x[8], top = 0.0f, low = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = Elem<E>::in(in.e[i]);
  bool nan = false, look = true;
  if constexpr (sizeof(E) == 2) {
    // two values an instruction; in the end the largest stands beside the least, negated, and a NaN in either's place
    const uint32_t* w = reinterpret_cast<const uint32_t*>(in.e);
    const uint32_t hi = max2<E>(max2<E>(w[0], w[1]), max2<E>(w[2], w[3])), lo = min2<E>(min2<E>(w[0], w[1]), min2<E>(w[2], w[3])) ^ 0x80008000u;
    uint32_t both = max2<E>(__byte_perm(hi, lo, 0x5410), __byte_perm(hi, lo, 0x7632));
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) both = max2<E>(both, __shfl_xor_sync(kAll, both, o));
    Eight<E> ends;
    *reinterpret_cast<uint32_t*>(ends.e) = both;
    const float most = Elem<E>::in(ends.e[0]), least = -Elem<E>::in(ends.e[1]);
    top = fmaxf(most, 0.0f);
    low = fminf(least, 0.0f);
    look = __any_sync(kAll, most != most || least != least || (top == -low && top > 0.0f));
  }
  if (look) {
    top = low = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      top = fmaxf(top, x[i]);
      low = fminf(low, x[i]);
      nan |= x[i] != x[i];
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      top = fmaxf(top, __shfl_xor_sync(kAll, top, o));
      low = fminf(low, __shfl_xor_sync(kAll, low, o));
    }
  }
  float m = top > -low ? top : low;
  if (look && __any_sync(kAll, top == -low && top > 0.0f)) {
    // both signs at the largest magnitude: the first of them
    int at = 32;
#pragma unroll
    for (int i = 7; i >= 0; --i)
      if (fabsf(x[i]) == top) at = i * 2 + (x[i] < 0.0f);
    if (at < 32) at += 16 * (threadIdx.x & 3);
    else at = 64;
    at = min(at, __shfl_xor_sync(kAll, at, 1));
    at = min(at, __shfl_xor_sync(kAll, at, 2));
    if (top == -low) m = at & 1 ? low : top;
  }
  scale = __float2half_rn(fminf(fmaxf(m * -0.125f, -65504.0f), 65504.0f));
  const float d = __half2float(scale);
  const float r = sizeof(E) == 4 ? __frcp_rn(d) : __fdividef(1.0f, d), inv = d != 0.0f ? r : 0.0f;
  const float a = inv * (1.0f / 15.25f), b = (8.0f + 0x1p-16f) * (1.0f / 15.25f);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float c = fmaf(__saturatef(fmaf(x[i], a, b)), 15.25f, kMagic);
    bits[i] = __float_as_uint(c);
    if constexpr (sizeof(E) == 4) {
      const float q = c - kMagic, xs = d < 0.0f ? -x[i] : x[i], ds = fabsf(d);
      if (xs < (q - 8.5f) * ds && q > 0.0f) bits[i] -= 1;
      else if (xs >= (q - 7.5f) * ds && q < 15.0f && d != 0.0f) bits[i] += 1;
    }
    if (sizeof(E) == 4 && d == 0.0f) bits[i] = __float_as_uint(kMagic + 8.0f);   // 16 bits: 0 * x + b has rounded to it
  }
  if (look && __any_sync(kAll, nan)) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (x[i] != x[i]) bits[i] = __float_as_uint(kMagic + 8.0f);
  }
}

template <int D, class E, bool kVec>
__global__ void __launch_bounds__(128, 8) kv_store_kernel(const StoreArgs a) {
  pdl_trigger();
  pdl_wait();
  using T = Tile<D>;
  constexpr int kOcts = D / 8, kTurns = (kTile * kOcts + 127) / 128;   // 8-value pieces of a row, turns of a thread
  __shared__ int64_t base[kTile];               // the row's tile of the first head in the cache; -1: skipped
  __shared__ int place[kTile];
  __shared__ __align__(16) uint8_t bytes[kTile][D / 2 + 4];   // values, a pair of dims a byte
  const int tid = threadIdx.x, groups = (a.heads + a.per - 1) / a.per, row0 = blockIdx.x / groups * kTile;
  const int head0 = blockIdx.x % groups * a.per, head1 = min(head0 + a.per, a.heads), head_bytes = T::kBytes << (a.page_shift - 4);
  if (tid < kTile) {
    int64_t p = -1;
    int tau = 0;
    if (row0 + tid < a.tokens) {
      const int64_t s = a.slots[row0 + tid];
      if (s >= a.limit) *a.bad = 1;
      else if (s >= 0) {
        const int in_page = (int)(s & ((1 << a.page_shift) - 1));
        p = (s >> a.page_shift) * a.page_bytes + (int64_t)head0 * head_bytes + (in_page >> 4) * T::kBytes;
        tau = in_page & 15;
      }
    }
    base[tid] = p;
    place[tid] = tau;
  }
  // the loads do not wait for the slots: rows that are skipped are rows all the same
  Eight<E> x[kTurns], y[kTurns];
  auto load = [&](int head) {
#pragma unroll
    for (int k = 0; k < kTurns; ++k) {
      const int w = tid + 128 * k, row = w / kOcts, o = w % kOcts;
      if (row < kTile && row0 + row < a.tokens) {
        x[k].template load<kVec>(static_cast<const E*>(a.k) + (int64_t)(row0 + row) * a.ks + head * a.kh + 8 * o);
        y[k].template load<kVec>(static_cast<const E*>(a.v) + (int64_t)(row0 + row) * a.vs + head * a.vh + 8 * o);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[k].e[i] = y[k].e[i] = Elem<E>::out(0.0f);
      }
    }
  };
  load(head0);
  __syncthreads();
  const int byte_row = tid & 15, byte_g = tid >> 4;   // in the second half: a row and a row pair g of every 16 dims
  const bool byte_live = base[byte_row] >= 0;
  uint8_t* byte_to = a.data + base[byte_row] + T::value_byte(place[byte_row], 2 * byte_g);
  for (int head = head0; head < head1; ++head) {
    const int64_t at = (int64_t)(head - head0) * head_bytes;
#pragma unroll
    for (int k = 0; k < kTurns; ++k) {
      const int w = tid + 128 * k, row = w / kOcts, o = w % kOcts, j = o >> 2, t = o & 3;
      if (row >= kTile) break;   // whole warps
      const bool live = base[row] >= 0;
      uint8_t* p = a.data + base[row] + at;
      __half dk, dv;
      uint32_t q[8];
      quantize8(x[k], dk, q);
      // only the low bits of a sum with the magic number's bits are kept, where those are 0
      const uint32_t even = ((q[6] * 16 + q[4]) * 16 + q[2]) * 16 + q[0], odd = ((q[7] * 16 + q[5]) * 16 + q[3]) * 16 + q[1];
      if (live) {
        const int tau = place[row];
        *reinterpret_cast<uint32_t*>(p + T::key_word(tau, j, t)) = __byte_perm(even, odd, 0x5410);
        if (t == 0) *reinterpret_cast<__half*>(p + T::key_scale(tau, j)) = dk;
      }
      quantize8(y[k], dv, q);
      const uint32_t b01 = __byte_perm(q[1] * 16 + q[0], q[3] * 16 + q[2], 0x0040), b23 = __byte_perm(q[5] * 16 + q[4], q[7] * 16 + q[6], 0x0040);
      *reinterpret_cast<uint32_t*>(&bytes[row][4 * o]) = __byte_perm(b01, b23, 0x5410);
      if (live && t == 0) *reinterpret_cast<__half*>(p + T::value_scale(place[row], j)) = dv;
    }
    if (head + 1 < head1) load(head + 1);
    __syncthreads();
    if (byte_live) {
#pragma unroll
      for (int i = 0; i < D / 16; ++i) byte_to[at + T::value_byte(0, 16 * i) - T::value_byte(0, 0)] = bytes[byte_row][8 * i + byte_g];
    }
    if (head + 1 < head1) __syncthreads();
  }
}

// ------------------------------------------------------------------ load
struct LoadArgs {
  const uint8_t* data;
  void *k, *v;
  const int32_t *table, *first, *lengths, *row_begin;
  int64_t table_stride, ks, kh, vs, vh, page_bytes;
  int requests, heads, per, table_width, rows, pages, page_shift;   // per: heads of a CTA
  int* bad;
};

// Two quants, in bits 0 and 16 of `two`, as values.  (q - 8) * d has 15 bits at most: f32 holds it, and f16's product rounds it once.
template <class E>
__device__ __forceinline__ void dequantize2(uint32_t two, __half2 d, float df, E* out) {
  two = (two & 0x000f000fu) | 0x64006400u;   // 1024 + q
  const __half2 q = __hsub2(*reinterpret_cast<const __half2*>(&two), __float2half2_rn(1032.0f));
  if constexpr (std::is_same<E, __half>::value) {
    *reinterpret_cast<__half2*>(out) = __hmul2(q, d);
  } else if constexpr (std::is_same<E, __nv_bfloat16>::value) {
    *reinterpret_cast<__nv_bfloat162*>(out) = __floats2bfloat162_rn(__low2float(q) * df, __high2float(q) * df);
  } else {
    out[0] = __low2float(q) * df;
    out[1] = __high2float(q) * df;
  }
}

// heads of a CTA at most: 1, 2 and 8 of them took 40, 36 and 35 us in the example below, and 50, 45 and 47 in the one above
constexpr int kLoadHeads = 4, kStoreHeads = 4;

// A CTA takes a tile of a request and head, or of up to kLoadHeads: its 18 * D bytes by 16-byte loads, then rows of 8 values a
// thread.  Request b's tiles stand in slots row_begin[b] / 16 + b * spare and further (two spare ones where its first position may
// lie inside a tile, else one), so a slot finds its request by bisection, without a sum over the requests in front; heads are
// neighbours, whose rows are.
// 32,760 rows of 8 heads of 128 f16: 31 us (5.5 TB/s); 44 when a CTA took 16 packed rows, each with a place of its own in the pages,
// 37 with a tile and a head.  Memory bounds it, and the three reads in a row before a CTA's first byte.
template <int D, class E, bool kVec>
__global__ void __launch_bounds__(128, 10) kv_load_kernel(const LoadArgs a) {
  pdl_trigger();
  pdl_wait();
  using T = Tile<D>;
  __shared__ __align__(16) uint8_t tiles[kLoadHeads][T::kBytes];
  const int tid = threadIdx.x, lane = tid & 31, groups = (a.heads + a.per - 1) / a.per, slot = blockIdx.x / groups, spare = a.first ? 2 : 1;
  const int head0 = blockIdx.x % groups * a.per, heads = min(a.per, a.heads - head0);
  if (head0 == 0 && tid == 127 && slot < a.requests &&   // there are more slots than requests
      (a.row_begin[slot] < 0 || a.row_begin[slot + 1] < a.row_begin[slot] || a.lengths[slot] < 0 || (a.first && a.first[slot] < 0)))
    *a.bad = 1;
  int lo = 0, hi = a.requests;          // the last request whose slots begin at or before this one
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32, b = lo + lane * step;
    const unsigned before = __ballot_sync(kAll, b < hi && (a.row_begin[b] >> 4) + b * spare <= slot);
    const int last = before ? 31 - __clz(before) : 0;
    hi = min(hi, lo + (last + 1) * step);
    lo += last * step;
  }
  const int b = lo, begin = a.row_begin[b], end = min(a.row_begin[b + 1], a.rows);
  const int64_t length = a.lengths[b], first = a.first ? a.first[b] : 0;
  if (begin < 0 || end <= begin) return;
  if (first < 0) return;
  // positions first .. until - 1 go to rows begin and further
  const int64_t until = min(first + (end - begin), length), at = ((first >> 4) + slot - ((begin >> 4) + b * spare)) * kTile;
  const int from = (int)max(first - at, (int64_t)0), to = (int)min(until - at, (int64_t)kTile);
  if (at < 0 || from >= to) return;
  const int64_t col = at >> a.page_shift;
  const int page = col < a.table_width ? a.table[b * a.table_stride + col] : -1;
  if (page < 0 || page >= a.pages) {
    if (tid == 0) *a.bad = 1;
    return;
  }
  const int shift = a.page_shift - 4;
  const uint8_t* p = a.data + page * a.page_bytes + (int64_t)((head0 << shift) + (int)(at >> 4 & ((1 << shift) - 1))) * T::kBytes;
  for (int h = 0; h < heads; ++h, p += T::kBytes << shift)
#pragma unroll
    for (int i = 0; i < T::kBytes / 16; i += 128)
      if (i + tid < T::kBytes / 16) reinterpret_cast<uint4*>(tiles[h])[i + tid] = reinterpret_cast<const uint4*>(p)[i + tid];
  __syncthreads();
  constexpr int kOcts = D / 8;
  const int64_t row0 = begin + (at - first);
#pragma unroll
  for (int k = 0; k < kTile * kOcts; k += 128) {
    const int w = tid + k, tau = w / kOcts, o = w % kOcts, j = o >> 2, t = o & 3;
    if (tau < from || tau >= to) continue;
    E* to_k = static_cast<E*>(a.k) + (row0 + tau) * a.ks + head0 * a.kh + 8 * o;
    E* to_v = static_cast<E*>(a.v) + (row0 + tau) * a.vs + head0 * a.vh + 8 * o;
    const uint8_t* tile = tiles[0];
    for (int h = 0; h < heads; ++h, tile += T::kBytes, to_k += a.kh, to_v += a.vh) {
      Eight<E> x;
      const uint32_t word = *reinterpret_cast<const uint32_t*>(tile + T::key_word(tau, j, t));
      const __half dk = *reinterpret_cast<const __half*>(tile + T::key_scale(tau, j)), dv = *reinterpret_cast<const __half*>(tile + T::value_scale(tau, j));
      const __half2 dk2 = __half2half2(dk), dv2 = __half2half2(dv);
      const float dkf = __half2float(dk), dvf = __half2float(dv);
#pragma unroll
      for (int e = 0; e < 4; ++e) dequantize2(word >> (4 * e), dk2, dkf, x.e + 2 * e);
      x.template store<kVec>(to_k);
#pragma unroll
      for (int e = 0; e < 4; ++e) dequantize2(tile[T::value_byte(tau, 8 * o + 2 * e)] * 0x1001u, dv2, dvf, x.e + 2 * e);
      x.template store<kVec>(to_v);
    }
  }
}

// heads of a CTA: as many as leave 16 CTAs to an SM
int heads_each(int64_t tiles, int heads, int sm_count, int most) {
  const int64_t spare = tiles * heads / ((int64_t)sm_count * 16);
  return (int)std::max<int64_t>(1, std::min<int64_t>({spare, (int64_t)most, (int64_t)heads}));
}

int log2_of(int v) {
  int s = 0;
  while ((1 << s) < v) ++s;
  return s;
}
bool rows_aligned(const void* p, int64_t token, int64_t head, size_t size) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && token * (int64_t)size % 16 == 0 && head * (int64_t)size % 16 == 0;
}
size_t size_of(int type) { return type == EMELB_F32 ? 4 : 2; }

template <class E, bool kVec>
cudaError_t store_typed(int D, unsigned grid, const StoreArgs& a, bool pdl, cudaStream_t st) {
  switch (D) {
    case 32: return launch_kernel(kv_store_kernel<32, E, kVec>, dim3(grid), dim3(128), 0, st, pdl, a);
    case 64: return launch_kernel(kv_store_kernel<64, E, kVec>, dim3(grid), dim3(128), 0, st, pdl, a);
    case 96: return launch_kernel(kv_store_kernel<96, E, kVec>, dim3(grid), dim3(128), 0, st, pdl, a);
    default: return launch_kernel(kv_store_kernel<128, E, kVec>, dim3(grid), dim3(128), 0, st, pdl, a);
  }
}
template <class E>
cudaError_t store_typed(bool vec, int D, unsigned grid, const StoreArgs& a, bool pdl, cudaStream_t st) {
  return vec ? store_typed<E, true>(D, grid, a, pdl, st) : store_typed<E, false>(D, grid, a, pdl, st);
}
template <class E, bool kVec>
cudaError_t load_typed(int D, unsigned grid, const LoadArgs& a, bool pdl, cudaStream_t st) {
  switch (D) {
    case 32: return launch_kernel(kv_load_kernel<32, E, kVec>, dim3(grid), dim3(128), 0, st, pdl, a);
    case 64: return launch_kernel(kv_load_kernel<64, E, kVec>, dim3(grid), dim3(128), 0, st, pdl, a);
    case 96: return launch_kernel(kv_load_kernel<96, E, kVec>, dim3(grid), dim3(128), 0, st, pdl, a);
    default: return launch_kernel(kv_load_kernel<128, E, kVec>, dim3(grid), dim3(128), 0, st, pdl, a);
  }
}
template <class E>
cudaError_t load_typed(bool vec, int D, unsigned grid, const LoadArgs& a, bool pdl, cudaStream_t st) {
  return vec ? load_typed<E, true>(D, grid, a, pdl, st) : load_typed<E, false>(D, grid, a, pdl, st);
}

}  // namespace

cudaError_t launch_kv_plan(const emelb_kv_plan_request& r, int* scratch, int sm_count, int* launches, int* bad, bool pdl, cudaStream_t st) {
  cudaError_t e = cudaFuncSetAttribute(kv_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 16 * kPlanMost);
  if (e != cudaSuccess) return e;
  // a CTA's sums cost what 2000 rows do: few rows and requests are one CTA's.  2048 rows at most of 300 / 1000 / 2000 requests by
  // one CTA 7.1 / 8.3 / 11.2 us, by three 8.4 / 8.4 / 10.5; in place, which three do by two launches, 7.3 / 8.6 / 11.5 and 8.6 / 10.5 / 11.3
  const int threads = r.requests <= 256 && r.token_capacity <= 2048 ? 256 : 512;
  const int teams = std::min(sm_count, (r.token_capacity - 1) / 2048 + 1);
  const bool in_place = r.lengths == r.cached || r.free_left == r.free_count;
  const int ctas = teams == 1 && r.requests <= 1024 ? 1 : 2 * teams + 1;
  const bool aside = ctas > 1 && in_place;
  const PlanArgs a{r, aside ? scratch + 1 : r.lengths, aside ? scratch : r.free_left, log2_of(r.page_tokens), bad};
  // one behind the other: one CTA 5.6 us for 7.2 when it may start early, 60 of them 15.3 for 12.4
  e = launch_kernel(kv_plan_kernel, dim3(ctas), dim3(threads), 16 * r.requests, st, pdl && ctas == 1, a);
  if (e != cudaSuccess) return e;
  *launches = 1;
  if (!aside) return e;
  e = launch_kernel(kv_plan_in_place_kernel, dim3((r.requests + 255) / 256), dim3(256), 0, st, pdl, scratch + 1, scratch, r.requests, r.lengths, r.free_left);
  if (e == cudaSuccess) *launches = 2;
  return e;
}

cudaError_t launch_kv_store(const emelb_kv_store_request& r, int sm_count, int* bad, bool pdl, cudaStream_t st) {
  const size_t size = size_of(r.type);
  StoreArgs a{};
  a.data = static_cast<uint8_t*>(r.cache.data);
  a.k = r.k;
  a.v = r.v;
  a.slots = r.slots;
  a.ks = r.k_token_stride;
  a.kh = r.k_head_stride;
  a.vs = r.v_token_stride;
  a.vh = r.v_head_stride;
  a.limit = (int64_t)r.cache.pages * r.cache.page_tokens;
  a.page_bytes = (int64_t)emelb_kv_page_bytes(r.cache.head_dim, r.cache.kv_heads, r.cache.page_tokens);
  a.tokens = r.tokens;
  a.heads = r.cache.kv_heads;
  a.page_shift = log2_of(r.cache.page_tokens);
  const bool vec = rows_aligned(r.k, a.ks, a.kh, size) && rows_aligned(r.v, a.vs, a.vh, size);
  a.bad = bad;
  const int tiles = (r.tokens + kTile - 1) / kTile;
  a.per = heads_each(tiles, a.heads, sm_count, kStoreHeads);
  const unsigned grid = (unsigned)tiles * ((a.heads + a.per - 1) / a.per);   // heads are neighbours, as their rows
  if (r.type == EMELB_F32) return store_typed<float>(vec, r.cache.head_dim, grid, a, pdl, st);
  if (r.type == EMELB_F16) return store_typed<__half>(vec, r.cache.head_dim, grid, a, pdl, st);
  return store_typed<__nv_bfloat16>(vec, r.cache.head_dim, grid, a, pdl, st);
}

cudaError_t launch_kv_load(const emelb_kv_load_request& r, int sm_count, int* bad, bool pdl, cudaStream_t st) {
  const size_t size = size_of(r.type);
  LoadArgs a{};
  a.data = static_cast<const uint8_t*>(r.cache.data);
  a.k = r.k;
  a.v = r.v;
  a.table = r.table;
  a.first = r.first;
  a.lengths = r.lengths;
  a.row_begin = r.row_begin;
  a.table_stride = r.table_stride;
  a.ks = r.k_token_stride;
  a.kh = r.k_head_stride;
  a.vs = r.v_token_stride;
  a.vh = r.v_head_stride;
  a.page_bytes = (int64_t)emelb_kv_page_bytes(r.cache.head_dim, r.cache.kv_heads, r.cache.page_tokens);
  a.requests = r.requests;
  a.heads = r.cache.kv_heads;
  a.table_width = r.table_width;
  a.rows = r.rows;
  a.pages = r.cache.pages;
  a.page_shift = log2_of(r.cache.page_tokens);
  const bool vec = rows_aligned(r.k, a.ks, a.kh, size) && rows_aligned(r.v, a.vs, a.vh, size);
  a.bad = bad;
  const int tiles = r.rows / kTile + r.requests * (r.first ? 2 : 1);
  a.per = heads_each(r.rows / kTile, a.heads, sm_count, kLoadHeads);
  const unsigned grid = (unsigned)tiles * ((a.heads + a.per - 1) / a.per);
  if (r.type == EMELB_F32) return load_typed<float>(vec, r.cache.head_dim, grid, a, pdl, st);
  if (r.type == EMELB_F16) return load_typed<__half>(vec, r.cache.head_dim, grid, a, pdl, st);
  return load_typed<__nv_bfloat16>(vec, r.cache.head_dim, grid, a, pdl, st);
}

}  // namespace emelb
