// Pages of the 4-bit key / value cache: the plan of a step, rows into their slots, rows back out.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "kv_tile.cuh"
#include "paged.h"

namespace emelb {
namespace {

using kv::kGroup;
using kv::kTile;
using kv::Tile;
typedef long long i64;

// ------------------------------------------------------------------ plan
// Three running sums over the requests (tokens, pages lacking, pages given back) decide everything else: new page j is
// entry top - 1 - j of the stack that the ended requests' pages lie on, and row i's request is found by bisection.  One cluster
// makes the step: every CTA takes the sums for itself, since that is cheaper than handing them over, then the cluster shares
// the pages and, behind a barrier (which also separates the last read of an array from the first write of one that may be
// the same), the rows.
constexpr int kPlanMost = EMELB_KV_MAX_REQUESTS;
constexpr unsigned kAll = 0xffffffffu;

__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// inclusive sum over the block; `carry` comes in and goes out as the sum of all blocks of requests so far
__device__ __forceinline__ i64 block_sum(i64 v, i64& carry, i64* warp_sums) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const i64 u = __shfl_up_sync(kAll, v, o);
    if (lane >= o) v += u;
  }
  if (lane == 31) warp_sums[warp] = v;
  __syncthreads();
  i64 w = lane < warps ? warp_sums[lane] : 0;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const i64 u = __shfl_up_sync(kAll, w, o);
    if (lane >= o) w += u;
  }
  const i64 before = warp ? __shfl_sync(kAll, w, warp - 1) : 0;
  const i64 all = __shfl_sync(kAll, w, 31);
  __syncthreads();
  const i64 out = carry + before + v;
  carry += all;
  return out;
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
  int page_shift;
  int* bad;
};

__global__ void __launch_bounds__(1024) kv_plan_kernel(const __grid_constant__ PlanArgs a) {
  extern __shared__ int plan_smem[];
  __shared__ i64 warp_sums[32];
  __shared__ i64 most_taken;
  const emelb_kv_plan_request& r = a.r;
  const int n = r.requests, P = r.page_tokens, shift = a.page_shift, tid = threadIdx.x, T = blockDim.x;
  const unsigned ranks = gridDim.x, rank = blockIdx.x;   // the grid is one cluster
  int* tok = plan_smem;         // running sums, each request's own included
  int* need = tok + n;
  int* back = need + n;
  int* had = back + n;          // tokens cached; complemented where the request gets nothing
  const i64 room = (i64)r.table_width * P;
  bool wrong = false;
  if (tid == 0) most_taken = 0;

  i64 tok_sum = 0, need_sum = 0, back_sum = 0;
  i64 count = *r.free_count;
  if (count < 0 || count > r.pages) {
    wrong = true;
    count = count < 0 ? 0 : r.pages;
  }
  for (int b0 = 0; b0 < n; b0 += T) {
    const int b = b0 + tid;
    i64 cached = 0, fresh = 0;
    bool ok = b < n;
    if (b < n) {
      cached = r.cached[b];
      fresh = r.fresh[b];
      ok = cached >= 0 && fresh >= -1 && cached + (fresh > 0 ? fresh : 0) <= room;
      wrong |= !ok;
      cached = cached < 0 ? 0 : cached > room ? room : cached;
    }
    const bool ended = fresh < 0;
    const i64 upto = block_sum(ended ? 0 : fresh, tok_sum, warp_sums);
    if (b < n && !ended && upto > r.token_capacity) {
      ok = false;
      wrong = true;
    }
    const int have = (int)((cached + P - 1) >> shift);
    const i64 lacks = ok && !ended ? ((cached + fresh + P - 1) >> shift) - have : 0;
    const i64 n_upto = block_sum(lacks, need_sum, warp_sums);
    const i64 r_upto = block_sum(ok && ended ? have : 0, back_sum, warp_sums);
    if (b < n) {
      tok[b] = clip(upto);
      need[b] = clip(n_upto);
      back[b] = clip(r_upto);
      had[b] = ok ? (int)cached : ~(int)cached;
    }
  }
  __syncthreads();
  const i64 top = count + back_sum;
  i64 taken = 0;
  for (int b = tid; b < n; b += T) {
    const int lacks = need[b] - (b ? need[b - 1] : 0);
    if (had[b] >= 0 && lacks > 0) {
      if (need[b] <= top) taken = need[b];
      else had[b] = ~had[b];
    }
  }
  if (taken) atomicMax(&most_taken, taken);
  __syncthreads();
  taken = most_taken;

  // new pages into the tables
  const int step = (int)ranks * T, me = (int)rank * T + tid;
  for (int j = me; j < taken; j += step) {
    const int b = owner_of(need, n, j);
    const i64 at = top - 1 - j;
    int page;
    if (at < count) {
      page = r.free_pages[at];
    } else {
      const int x = (int)(at - count), e = owner_of(back, n, x);
      page = r.table[e * r.table_stride + (x - (e ? back[e - 1] : 0))];
    }
    if (page < 0 || page >= r.pages) wrong = true;
    r.table[b * r.table_stride + ((had[b] + P - 1) >> shift) + (j - (b ? need[b - 1] : 0))] = page;
  }
  // what the ended requests gave back and nobody took
  for (i64 x = me; x < top - taken - count; x += step) {
    const int e = owner_of(back, n, (int)x);
    if (count + x < r.pages) r.free_pages[count + x] = r.table[e * r.table_stride + (x - (e ? back[e - 1] : 0))];
    else wrong = true;
  }
  if (ranks > 1) cluster_barrier();
  else __syncthreads();

  // slots and positions
  const int total = clip(tok_sum < r.token_capacity ? tok_sum : r.token_capacity);
  for (int i = me; i < r.token_capacity; i += step) {
    i64 slot = -1;
    int p = 0;
    if (i < total) {
      const int b = owner_of(tok, n, i), at = i - (b ? tok[b - 1] : 0);
      const int h = had[b];
      p = (h < 0 ? ~h : h) + at;
      if (h >= 0) {
        const int page = r.table[b * r.table_stride + (p >> shift)];
        if (page >= 0 && page < r.pages) slot = ((i64)page << shift) + (p & (P - 1));
        else wrong = true;
      }
    }
    r.slots[i] = slot;
    r.positions[i] = p;
  }
  // each request's share, by the first CTA (fresh may not be read from an array that was written: it never is one)
  if (rank == 0) {
    i64 key_sum = 0;
    for (int b0 = 0; b0 < n; b0 += T) {
      const int b = b0 + tid;
      i64 len = 0;
      if (b < n) {
        const int h = had[b];
        const bool ended = r.fresh[b] < 0;
        len = ended ? 0 : h >= 0 ? (i64)h + (tok[b] - (b ? tok[b - 1] : 0)) : (i64)~h;
      }
      const i64 upto = block_sum(len, key_sum, warp_sums);
      if (b < n) {
        r.lengths[b] = (int)len;
        r.query_begin[b + 1] = tok[b] < r.token_capacity ? tok[b] : r.token_capacity;
        r.key_begin[b + 1] = clip(upto);
        if (upto > 0x7fffffff) wrong = true;
      }
    }
    if (tid == 0) {
      r.query_begin[0] = 0;
      r.key_begin[0] = 0;
      *r.free_left = clip(top - taken);
      *r.shortage = clip(need_sum > top ? need_sum - top : 0);
    }
  }
  if (wrong) *a.bad = 1;
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
  __device__ __forceinline__ void load(const E* p, bool vec) {
    if (vec) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(e) / 16; ++i) reinterpret_cast<uint4*>(e)[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = p[i];
    }
  }
  __device__ __forceinline__ void store(E* p, bool vec) const {
    if (vec) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(e) / 16; ++i) reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(e)[i];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) p[i] = e[i];
    }
  }
};

// ------------------------------------------------------------------ store
// A CTA takes 16 packed rows of one head.  Four lanes share a group of 32 values, 8 each, which is a word of keys; the scale
// comes from the group's largest value by two shuffles.  Values go by bytes, each with its own address: they wait in shared memory
// until a warp can store one pair of dims of 16 rows at a time, which are neighbours where the rows fill a tile.
struct StoreArgs {
  uint8_t* data;
  const void *k, *v;
  const int64_t* slots;
  int64_t ks, kh, vs, vh, limit, page_bytes;
  int tokens, page_shift, vec;
  int* bad;
};

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
  bool nan = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[i] = Elem<E>::in(in.e[i]);
    top = fmaxf(top, x[i]);
    low = fminf(low, x[i]);
    nan |= x[i] != x[i];
  }
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    top = fmaxf(top, __shfl_xor_sync(kAll, top, o));
    low = fminf(low, __shfl_xor_sync(kAll, low, o));
  }
  float m = top > -low ? top : low;
  if (__any_sync(kAll, top == -low && top > 0.0f)) {
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
  float inv = 0.0f;
  if (d != 0.0f) inv = sizeof(E) == 4 ? __frcp_rn(d) : __fdividef(1.0f, d);
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
    if (d == 0.0f) bits[i] = __float_as_uint(kMagic + 8.0f);
  }
  if (__any_sync(kAll, nan)) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (x[i] != x[i]) bits[i] = __float_as_uint(kMagic + 8.0f);
  }
}

template <int D, class E>
__global__ void __launch_bounds__(128) kv_store_kernel(const StoreArgs a) {
  using T = Tile<D>;
  constexpr int kOcts = D / 8, kTurns = (kTile * kOcts + 127) / 128;   // 8-value pieces of a row, turns of a thread
  __shared__ uint8_t* base[kTile];              // the row's tile of this head; null: skipped
  __shared__ int place[kTile];
  __shared__ __align__(16) uint8_t bytes[kTile][D / 2 + 4];   // values, a pair of dims a byte
  const int tid = threadIdx.x, head = blockIdx.y, row0 = blockIdx.x * kTile;
  if (tid < kTile) {
    uint8_t* p = nullptr;
    int tau = 0;
    if (row0 + tid < a.tokens) {
      const int64_t s = a.slots[row0 + tid];
      if (s >= a.limit) *a.bad = 1;
      else if (s >= 0) {
        const int in_page = (int)(s & ((1 << a.page_shift) - 1));
        const int tiles = 1 << (a.page_shift - 4);
        p = a.data + (s >> a.page_shift) * a.page_bytes + (int64_t)(head * tiles + (in_page >> 4)) * T::kBytes;
        tau = in_page & 15;
      }
    }
    base[tid] = p;
    place[tid] = tau;
  }
  // the loads do not wait for the slots: rows that are skipped are rows all the same
  Eight<E> x[kTurns], y[kTurns];
#pragma unroll
  for (int k = 0; k < kTurns; ++k) {
    const int w = tid + 128 * k, row = w / kOcts, o = w % kOcts;
    if (row < kTile && row0 + row < a.tokens) {
      x[k].load(static_cast<const E*>(a.k) + (int64_t)(row0 + row) * a.ks + head * a.kh + 8 * o, a.vec);
      y[k].load(static_cast<const E*>(a.v) + (int64_t)(row0 + row) * a.vs + head * a.vh + 8 * o, a.vec);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[k].e[i] = y[k].e[i] = Elem<E>::out(0.0f);
    }
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kTurns; ++k) {
    const int w = tid + 128 * k, row = w / kOcts, o = w % kOcts, j = o >> 2, t = o & 3;
    if (row >= kTile) break;   // whole warps
    uint8_t* p = base[row];
    __half dk, dv;
    uint32_t q[8];
    quantize8(x[k], dk, q);
    // only the low bits of a sum with the magic number's bits are kept, where those are 0
    const uint32_t even = ((q[6] * 16 + q[4]) * 16 + q[2]) * 16 + q[0], odd = ((q[7] * 16 + q[5]) * 16 + q[3]) * 16 + q[1];
    if (p) {
      const int tau = place[row];
      *reinterpret_cast<uint32_t*>(p + T::key_word(tau, j, t)) = __byte_perm(even, odd, 0x5410);
      if (t == 0) *reinterpret_cast<__half*>(p + T::key_scale(tau, j)) = dk;
    }
    quantize8(y[k], dv, q);
    const uint32_t b01 = __byte_perm(q[1] * 16 + q[0], q[3] * 16 + q[2], 0x0040), b23 = __byte_perm(q[5] * 16 + q[4], q[7] * 16 + q[6], 0x0040);
    *reinterpret_cast<uint32_t*>(&bytes[row][4 * o]) = __byte_perm(b01, b23, 0x5410);
    if (p && t == 0) *reinterpret_cast<__half*>(p + T::value_scale(place[row], j)) = dv;
  }
  __syncthreads();
  // thread: a row and a row pair g of every 16 dims
  const int row = tid & 15, g = tid >> 4;
  uint8_t* p = base[row];
  if (p) {
    p += T::value_byte(place[row], 2 * g);
#pragma unroll
    for (int i = 0; i < D / 16; ++i) p[T::value_byte(0, 16 * i) - T::value_byte(0, 0)] = bytes[row][8 * i + g];
  }
}

// ------------------------------------------------------------------ load
struct LoadArgs {
  const uint8_t* data;
  void *k, *v;
  const int32_t *table, *first, *lengths, *row_begin;
  int64_t table_stride, ks, kh, vs, vh, page_bytes;
  int requests, table_width, rows, pages, page_shift, vec;
  int* bad;
};

// 8 quants as values: nibble i of `word` (low 16 bits) times d, nibble i + 4 the next (kPairs), or nibbles in order
template <bool kPairs, class E>
__device__ __forceinline__ void dequantize8(uint32_t word, __half scale, Eight<E>& out) {
  const float d = __half2float(scale);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t two = (word >> (4 * i) & 0x000f000fu) | 0x64006400u;   // 1024 + nibbles i and i + 4
    const __half2 q = __hsub2(*reinterpret_cast<const __half2*>(&two), __float2half2_rn(1032.0f));
    out.e[kPairs ? 2 * i : i] = Elem<E>::out(__low2float(q) * d);
    out.e[kPairs ? 2 * i + 1 : i + 4] = Elem<E>::out(__high2float(q) * d);
  }
}

constexpr int kWindow = 127;   // requests behind the first row's whose beginnings are looked at together

template <int D, class E>
__global__ void __launch_bounds__(128) kv_load_kernel(const LoadArgs a) {
  using T = Tile<D>;
  __shared__ const uint8_t* base[kTile];
  __shared__ int place[kTile];
  __shared__ int begins[kWindow + 1];
  __shared__ __align__(16) uint8_t bytes[kTile][D / 2 + 4];
  const int tid = threadIdx.x, head = blockIdx.y, row0 = blockIdx.x * kTile;
  // the request of the first row: how many begin at or before it
  int before = 0;
  for (int b0 = 0; b0 < a.requests; b0 += 128) before += __syncthreads_count(b0 + tid < a.requests && a.row_begin[b0 + tid] <= row0);
  const int b0 = max(before - 1, 0);
  begins[tid] = a.row_begin[min(b0 + tid, a.requests)];
  __syncthreads();
  if (tid < kTile) {
    const uint8_t* p = nullptr;
    int tau = 0;
    const int row = row0 + tid;
    int b = b0;
    while (b < a.requests && (b + 1 - b0 <= kWindow ? begins[b + 1 - b0] : a.row_begin[b + 1]) <= row) ++b;
    if (row < a.rows && b < a.requests && row >= begins[0]) {
      const int begin = b - b0 <= kWindow ? begins[b - b0] : a.row_begin[b];
      const int64_t from = a.first ? a.first[b] : 0, pos = from + row - begin;
      if (from < 0 || pos < from) *a.bad = 1;
      else if (pos < a.lengths[b]) {
        const int64_t col = pos >> a.page_shift;
        const int page = col < a.table_width ? a.table[b * a.table_stride + col] : -1;
        if (page < 0 || page >= a.pages) *a.bad = 1;
        else {
          const int in_page = (int)(pos & ((1 << a.page_shift) - 1)), tiles = 1 << (a.page_shift - 4);
          p = a.data + page * a.page_bytes + (int64_t)(head * tiles + (in_page >> 4)) * T::kBytes;
          tau = in_page & 15;
        }
      }
    }
    base[tid] = p;
    place[tid] = tau;
  }
  __syncthreads();
  {
    const int row = tid & 15, g = tid >> 4;
    const uint8_t* p = base[row];
    if (p) {
      p += T::value_byte(place[row], 2 * g);
      uint8_t v[D / 16];
#pragma unroll
      for (int i = 0; i < D / 16; ++i) v[i] = p[T::value_byte(0, 16 * i) - T::value_byte(0, 0)];
#pragma unroll
      for (int i = 0; i < D / 16; ++i) bytes[row][8 * i + g] = v[i];
    }
  }
  constexpr int kOcts = D / 8;
  for (int w = tid; w < kTile * kOcts; w += 128) {
    const int row = w / kOcts, o = w % kOcts, j = o >> 2, t = o & 3;
    const uint8_t* p = base[row];
    if (!p) continue;
    Eight<E> x;
    dequantize8<true>(*reinterpret_cast<const uint32_t*>(p + T::key_word(place[row], j, t)), *reinterpret_cast<const __half*>(p + T::key_scale(place[row], j)), x);
    x.store(static_cast<E*>(a.k) + (int64_t)(row0 + row) * a.ks + head * a.kh + 8 * o, a.vec);
  }
  __syncthreads();
  for (int w = tid; w < kTile * kOcts; w += 128) {
    const int row = w / kOcts, o = w % kOcts, j = o >> 2;
    const uint8_t* p = base[row];
    if (!p) continue;
    Eight<E> y;
    dequantize8<false>(*reinterpret_cast<const uint32_t*>(&bytes[row][4 * o]), *reinterpret_cast<const __half*>(p + T::value_scale(place[row], j)), y);
    y.store(static_cast<E*>(a.v) + (int64_t)(row0 + row) * a.vs + head * a.vh + 8 * o, a.vec);
  }
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

template <class E>
cudaError_t store_typed(int D, dim3 grid, const StoreArgs& a, cudaStream_t st) {
  switch (D) {
    case 32: kv_store_kernel<32, E><<<grid, 128, 0, st>>>(a); break;
    case 64: kv_store_kernel<64, E><<<grid, 128, 0, st>>>(a); break;
    case 96: kv_store_kernel<96, E><<<grid, 128, 0, st>>>(a); break;
    default: kv_store_kernel<128, E><<<grid, 128, 0, st>>>(a); break;
  }
  return cudaGetLastError();
}
template <class E>
cudaError_t load_typed(int D, dim3 grid, const LoadArgs& a, cudaStream_t st) {
  switch (D) {
    case 32: kv_load_kernel<32, E><<<grid, 128, 0, st>>>(a); break;
    case 64: kv_load_kernel<64, E><<<grid, 128, 0, st>>>(a); break;
    case 96: kv_load_kernel<96, E><<<grid, 128, 0, st>>>(a); break;
    default: kv_load_kernel<128, E><<<grid, 128, 0, st>>>(a); break;
  }
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_kv_plan(const emelb_kv_plan_request& r, int* bad, cudaStream_t st) {
  PlanArgs a{r, log2_of(r.page_tokens), bad};
  const bool small = r.requests <= 256 && r.token_capacity <= 1024;
  const int smem = 16 * r.requests;
  cudaError_t e = cudaFuncSetAttribute(kv_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 16 * kPlanMost);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(small ? 1 : 8);
  cfg.blockDim = dim3(small ? 256 : 1024);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cfg.gridDim.x;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = small ? 0 : 1;
  return cudaLaunchKernelEx(&cfg, kv_plan_kernel, a);
}

cudaError_t launch_kv_store(const emelb_kv_store_request& r, int* bad, cudaStream_t st) {
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
  a.page_shift = log2_of(r.cache.page_tokens);
  a.vec = rows_aligned(r.k, a.ks, a.kh, size) && rows_aligned(r.v, a.vs, a.vh, size);
  a.bad = bad;
  const dim3 grid((r.tokens + kTile - 1) / kTile, r.cache.kv_heads);
  if (r.type == EMELB_F32) return store_typed<float>(r.cache.head_dim, grid, a, st);
  if (r.type == EMELB_F16) return store_typed<__half>(r.cache.head_dim, grid, a, st);
  return store_typed<__nv_bfloat16>(r.cache.head_dim, grid, a, st);
}

cudaError_t launch_kv_load(const emelb_kv_load_request& r, int* bad, cudaStream_t st) {
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
  a.table_width = r.table_width;
  a.rows = r.rows;
  a.pages = r.cache.pages;
  a.page_shift = log2_of(r.cache.page_tokens);
  a.vec = rows_aligned(r.k, a.ks, a.kh, size) && rows_aligned(r.v, a.vs, a.vh, size);
  a.bad = bad;
  const dim3 grid((r.rows + kTile - 1) / kTile, r.cache.kv_heads);
  if (r.type == EMELB_F32) return load_typed<float>(r.cache.head_dim, grid, a, st);
  if (r.type == EMELB_F16) return load_typed<__half>(r.cache.head_dim, grid, a, st);
  return load_typed<__nv_bfloat16>(r.cache.head_dim, grid, a, st);
}

}  // namespace emelb
