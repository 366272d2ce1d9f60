// Attention of packed prompts of different lengths, on the Blackwell tensor cores.
//
// Per request and key / value head, the query rows of the head's group stand behind one another, token after token, so that a
// short prompt fills tiles of rows too.  A pair of tiles of 128 rows walks the keys in tiles of 128:
//   S = Q K^T       tcgen05.mma, operands in shared memory, by TMA; S {128 rows, 128 keys} in TMEM, a row a lane
//   P = exp2(S - m) a thread a row: 128 scores out of TMEM, running maximum and sum, P as 16-bit values back over S
//   O += P V        tcgen05.mma, P as the A operand out of TMEM, V by TMA as it lies in memory (its dims are contiguous: MN-major)
// While the warps of one tile take the exponentials, the tensor cores work for the other.  The running maximum a row's weights are
// taken against follows the true one only when that has passed it by 2^8: only then does O, in TMEM, have to be rescaled.  Weights
// are rounded to the operands' 16 bits, as the tensor cores take them; the sum is of the f32 ones.
//
// The tensor cores cut every sum they add to O off, about 2^-22 of it on average: with O in TMEM all the way one row over 2^20 equal
// keys came out 0.8 % too small, over 2^25 25 %.  So every kFold tiles of keys O moves to scratch, where f32 additions round to nearest,
// and starts anew, as does the sum; weights are summed by tiles before a tile's sum joins the row's.  Up to 8192 keys nothing moves.
//
// A CTA stays and takes pairs of tiles from a common counter (their walks differ by far): a warp finds the next one and asks for its
// queries as soon as the last scores against the ones before are done, another asks for keys and values ahead across pairs, another
// looks at values that not every row may see.  Nothing but the rows' own warps waits while they store results.
//
// Two matrix products of 128 x 128 x head_dim and 128 x 128 exponentials a tile: at head_dim 128 both take the same time (4096
// products, 16 exponentials a cycle and SM: 2048 cycles for two row tiles and 128 keys), at 64 the exponentials bound it.  What a
// row tile waits for, between its last weight and its next score, is the other's time; together they take about 2,900 cycles, and
// a pair of tiles about 5,000 besides (first scores, last mix, results).
//
// us, two prompts of 4100 and 8190 tokens / 13 of 17 to 600, 32 heads of 128: 756 with weights handed over at once and an arrival a
// thread; 659 / 95 by halves and with registers split; 578 / 61 with queries by asynchronous copies; 544 / 52 since CTAs stay.
// Repeated for seconds, at 990 W and 1.58 GHz, the long ones took 640 then; 655 (1,050 TFLOP/s) / 53 since sums keep their digits and far
// scores are looked for.  One prompt of 8192 and heads of 64: 393 (699 TFLOP/s; its exponentials alone take 252).
//
// Measured and left out: an issuer of products for each row tile 613 / - (they fall into step and wait for the same pipes); scores
// of 64 keys in two buffers a row tile, so that none waits for a mix, 588 (products with 64 columns take longer); weights against a
// stale maximum, looked at afterwards, 604; an eighth, a quarter of the exponentials by polynomials on the multiply-adds, no gain,
// +8; at head_dim 64, where TMEM has room, weights beside the scores so that the next scores need not wait for the mix, 421 for 394,
// and turns at the exponentials for the two warps of a scheduler, 394 (558 for 538 at 128).
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "kernels.h"
#include "paged.h"
#include "tc_common.cuh"

namespace emelb {
namespace {

constexpr unsigned kAll = 0xffffffffu;
constexpr int kTileRows = 128, kTileKeys = 128, kTiles = 2;   // tiles of a CTA
constexpr int kLoadWarp = 8, kMmaWarp = 9, kCheckWarp = 10, kPlanWarp = 11, kThreads = 384;   // behind the softmax warps
// registers a thread behind the start, of the 168 that 384 threads launch with: 8 warps x 208 + 4 x 88 = 12 x 168
constexpr int kSoftmaxRegs = 208, kOtherRegs = 88;
static_assert(8 * kSoftmaxRegs + 4 * kOtherRegs <= 12 * 168, "registers");
constexpr float kLowest = -3.0e38f;
constexpr float kSlack = 8.0f;
// f16 weights are taken times 2^7, so that with the slack they reach 2^15 and keep 11 bits down to 2^-21 of the largest; bf16 has range
template <bool kBf16>
constexpr float kRaise = kBf16 ? 0.0f : 7.0f;
constexpr float kFarScore = 0x1p20f;  // from here on an f32 score's own rounding may be more than that
constexpr int kFold = 64;             // key tiles between two moves of O out of TMEM: 512 products, 2^-14 of O
constexpr int kTmemCols = 512;

struct __align__(64) Map {
  unsigned char bytes[128];
};

struct PackedArgs {
  const void* v;
  void* out;
  const int32_t *query_begin, *key_begin;
  int64_t vs, vh, os, oh;
  int requests, kv_heads, group, group_inv, tile_tokens, head_dim, queries, keys, max_queries, causal;
  float scale_log2;
  int64_t items;
  int* next;           // the next item, CTAs that are done: zero between launches
  int *bad, *status;
  float* fold;         // of a CTA: kTiles x {dims of O, the maximum that they were taken against, the sum, far scores' base} x kTileRows
};
constexpr int kFoldDims = 128;
constexpr int kFoldRows = kFoldDims + 3;
static_assert((uint64_t)kTiles * kFoldRows * kTileRows == kPackedFoldFloats, "scratch of a CTA");

template <int DP>
struct Smem {
  static constexpr int kHalf = kTileKeys * 128;          // 64 dims of 128 rows
  static constexpr int kTile = DP / 64 * kHalf;
  static constexpr int kStages = DP == 128 ? 4 : 8;      // of K and V tiles in turn
  static constexpr int kQ = kTiles * kTile;
  static constexpr int kTurn = 32 * 128;                 // where a softmax warp's results turn into rows
  static constexpr int kBytes = kQ + kStages * kTile + 8 * kTurn + 1024;
};

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ uint4 load_shared(uint32_t saddr) {
  uint4 w;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w) : "r"(saddr) : "memory");
  return w;
}
template <bool kBf16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  uint32_t r;
  if (kBf16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const void* map, int x, int y, int z, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst), "l"(map),
               "r"(x), "r"(y), "r"(z), "r"(bar)
               : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* v) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
               "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
               "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
                 "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]),
                 "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]),
                 "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
               : "r"(taddr));
}
// values that were loaded are used behind this
template <int N>
__device__ __forceinline__ void wait_ld(uint32_t (&v)[N]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+r"(v[i]));
}

// Operands in shared memory go by the low words of their descriptors, the address / 16 and, of values, the step to the next 64 dims;
// the high words are alike: 8 rows of 128 bytes an atom, 128-byte swizzle
constexpr uint32_t kDescHigh = (1024 >> 4) | 1u << 14 | 2u << 29;
__device__ __forceinline__ uint32_t row_desc(uint32_t saddr) { return saddr >> 4 | 1u << 16; }
// V {keys, dims} as the B operand: 16 keys further 2048 bytes, the next 64 dims kTileKeys * 128
__device__ __forceinline__ uint32_t value_desc(uint32_t saddr) { return saddr >> 4 | (uint32_t)(kTileKeys * 128 >> 4) << 16; }
// d (+)= a * b, both operands in shared memory
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
      "mov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %5};\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}" ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "r"(kDescHigh)
      : "memory");
}
// the same with A in TMEM
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\t"
      "mov.b64 db, {%2, %5};\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}" ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "r"(kDescHigh)
      : "memory");
}

// With many requests, pairs of row tiles of request b stand in slots first_slot(b) .. first_slot(b + 1) - 1, of which it may leave one empty: tokens
// before it / (two tiles') + b is known from query_begin alone, without a sum over the requests in front.
__device__ __forceinline__ int first_slot(const PackedArgs& a, int b) {
  return (int)((uint32_t)(a.query_begin[b] - a.query_begin[0]) / (uint32_t)(kTiles * a.tile_tokens)) + b;
}

// two row tiles of a request and key / value head
struct Item {
  int valid;                 // 0: no more
  int token, tokens;         // the first query row and how many
  int head;
  int first_key, keys;       // of the request
  int see;                   // keys that the first token sees, were there no end to them (or keys, if no row is hidden anything)
  int n0, n1;                // key tiles that either row tile walks
  int odd;                   // values that are not finite, of keys that only some of the rows see are not in the products
};

// 16 bits as a float; whether they are an infinity or NaN; z + 0 * w for both halves of w
template <bool kBf16>
__device__ __forceinline__ float as_float(uint32_t half) {
  return kBf16 ? __uint_as_float(half << 16) : __half2float(__ushort_as_half((unsigned short)half));
}
template <bool kBf16>
__device__ __forceinline__ bool odd_half(uint32_t half) {
  constexpr uint32_t kExp = kBf16 ? 0x7f80u : 0x7c00u;
  return (half & kExp) == kExp;
}
template <bool kBf16>
__device__ __forceinline__ uint32_t fma_zero(uint32_t z, uint32_t w) {
  uint32_t r;
  if (kBf16) asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(w), "r"(0), "r"(z));
  else asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(w), "r"(0), "r"(z));
  return r;
}

// A row's O, its maximum and its sum so far to scratch, on top of what is there but for the first time; and back into TMEM, where
// results are taken from.  Calls: as code of the loop they cost the 13 prompts 54.6 us, as calls 52.5, which take 51.9 without them
__device__ __forceinline__ float* fold_row(float* fold, int t, int row) {
  return fold + ((uint64_t)blockIdx.x * kTiles + t) * (kFoldRows * kTileRows) + row;
}
template <int DP>
__device__ __noinline__ void fold_away(float* fold, int t, int row, uint32_t o_col, bool first, float m, float2 sums) {
  fold = fold_row(fold, t, row);
  float *at_m = fold + kFoldDims * kTileRows, *at_sum = at_m + kTileRows;
  const float f = first ? 0.0f : exp2_fast(*at_m - m);
  *at_sum = sums.x + sums.y + (first ? 0.0f : *at_sum * f);
  *at_m = m;
#pragma unroll 1
  for (int c = 0; c < DP; c += 32) {
    uint32_t o[32];
    tmem_ld32(o_col + c, o);
    wait_ld(o);
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      float* to = fold + (c + i) * kTileRows;
      *to = first ? __uint_as_float(o[i]) : fmaf(*to, f, __uint_as_float(o[i]));
    }
  }
}
template <int DP>
__device__ __noinline__ float fold_back(float* fold, int t, int row, uint32_t o_col, float m, float sum) {
  fold = fold_row(fold, t, row);
  const float f = exp2_fast(fold[kFoldDims * kTileRows] - m);
#pragma unroll 1
  for (int c = 0; c < DP; c += 32) {
    uint32_t o[32];
    tmem_ld32(o_col + c, o);
    wait_ld(o);
#pragma unroll
    for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(fmaf(fold[(c + i) * kTileRows], f, __uint_as_float(o[i])));
    tc::tmem_st32(o_col + c, o);
  }
  tc::tmem_wait_st();
  return fmaf(fold[(kFoldDims + 1) * kTileRows], f, sum);
}

// Far scores.  The loop takes a weight as 2^(score * scale - m) by one multiply-add, while m is a rounded product: of scores beyond
// 2^27 the rounding alone may be so much that weights overflow.  So scores from kFarScore on are rounded as m is, and put back as
// differences from a base, the largest of the row so far, over the scale; m, returned, and the maximum in scratch count from the base
// as well.  `first`: m and scores still count from 0.
__device__ __noinline__ float rebase(float* fold, int t, int row, uint32_t s_col, int seen, float scale, bool first, float m) {
  fold = fold_row(fold, t, row);
  float *fold_m = fold + kFoldDims * kTileRows, *at_base = fold + (kFoldDims + 2) * kTileRows;
  float top = -INFINITY;
#pragma unroll 1
  for (int c = 0; c < kTileKeys; c += 32) {
    uint32_t s[32];
    tmem_ld32(s_col + c, s);
    wait_ld(s);
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (c + i < seen) top = max_nan(top, __fmul_rn(__uint_as_float(s[i]), scale));
  }
  const float was = first ? m : *at_base;              // kLowest: nothing seen yet
  if (first && m != kLowest) m = 0.0f;
  const float base = max_nan(was, top), by = base - was, inv = 1.0f / scale;
  *at_base = base;
  *fold_m -= first ? base : by;                        // of nothing moved yet: whatever stands there
#pragma unroll 1
  for (int c = 0; c < kTileKeys; c += 32) {
    uint32_t s[32];
    tmem_ld32(s_col + c, s);
    wait_ld(s);
#pragma unroll
    for (int i = 0; i < 32; ++i) s[i] = __float_as_uint((__fmul_rn(__uint_as_float(s[i]), scale) - base) * inv);
    tc::tmem_st32(s_col + c, s);
  }
  tc::tmem_wait_st();
  return max_nan(m - by, kLowest);
}

template <int DP, bool kBf16>
__global__ void __launch_bounds__(kThreads, 1)
    attend_packed_kernel(const __grid_constant__ PackedArgs a, const __grid_constant__ Map q_map, const __grid_constant__ Map k_map,
                         const __grid_constant__ Map v_map) {
  using S = Smem<DP>;
  constexpr int kStages = S::kStages;
  extern __shared__ uint8_t raw[];
  __shared__ uint64_t bars[3 * kStages + 4 * kTiles + 7];
  __shared__ Item items[2];
  __shared__ uint32_t tmem_slot;
  __shared__ int order[32];
  __shared__ volatile int gave_up;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t smem = (tc::smem_u32(raw) + 1023u) & ~1023u;
  const uint32_t bar0 = tc::smem_u32(bars), bar1 = bar0 + 24 * kStages, bar2 = bar1 + 32 * kTiles;
  auto full = [&](int s) { return bar0 + 8 * s; };
  auto empty = [&](int s) { return bar0 + 8 * (kStages + s); };
  auto landed = [&](int s) { return bar0 + 8 * (2 * kStages + s); };   // values that the check warp hands on as full
  auto s_ready = [&](int t) { return bar1 + 8 * t; };
  auto o_ready = [&](int t) { return bar1 + 8 * (kTiles + t); };
  auto p_ready = [&](int t, int half) { return bar1 + 8 * ((2 + half) * kTiles + t); };   // 64 keys each
  auto item_full = [&](int n) { return bar2 + 8 * (n & 1); };
  auto item_empty = [&](int n) { return bar2 + 8 * (2 + (n & 1)); };
  const uint32_t q_ready = bar2 + 32, q_empty = bar2 + 40, drain_bar = bar2 + 48;

  if (tid == 0) {
    for (int s = 0; s < kStages; ++s) {
      tc::mbar_init(full(s), 1);
      tc::mbar_init(empty(s), 1);
      tc::mbar_init(landed(s), 1);
    }
    for (int t = 0; t < kTiles; ++t) {
      tc::mbar_init(s_ready(t), 1);
      tc::mbar_init(p_ready(t, 0), kTileRows / 32);
      tc::mbar_init(p_ready(t, 1), kTileRows / 32);
      tc::mbar_init(o_ready(t), 1);
      tc::mbar_init(item_full(t), 1);
      tc::mbar_init(item_empty(t), 11);   // all warps but the one that fills it
    }
    tc::mbar_init(q_ready, 1);
    tc::mbar_init(q_empty, 1);
    tc::mbar_init(drain_bar, 1);
    gave_up = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  // no kernel holds TMEM while it waits for one that may still ask for some: allocation behind the wait, the next one's start behind it
  if (warp == kMmaWarp) {
    pdl_wait();
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc::smem_u32(&tmem_slot)), "r"(kTmemCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  // row / group by a product: exact, since row < 128 and group <= 128
  auto token_of = [&](int row) { return (int)((uint32_t)row * a.group_inv >> 16); };
  auto sees = [&](const Item& it, int token) { return max(0, min(it.keys, a.causal ? it.see + token : it.see)); };
  auto sound = [&](int b) {
    const int q0 = a.query_begin[b], nq = a.query_begin[b + 1] - q0, k0 = a.key_begin[b], nk = a.key_begin[b + 1] - k0, first = a.query_begin[0];
    return first >= 0 && q0 >= first && nq >= 0 && nq <= a.max_queries && q0 <= a.queries - nq && k0 >= 0 && nk >= 0 && k0 <= a.keys - nk;
  };
  const int most = kTiles * a.tile_tokens;
  auto pairs_of = [&](int nq) { return (int)(((uint32_t)nq + most - 1) / (uint32_t)most); };
  // pair `local` of a request, from its end on: long walks first
  auto make_item = [&](int head, int q0, int nq, int k0, int nk, int local) {
    Item it{};
    const int from = (pairs_of(nq) - 1 - local) * most;
    it.valid = 1;
    it.token = q0 + from;
    it.tokens = min(nq - from, most);
    it.head = head;
    it.first_key = k0;
    it.keys = nk;
    it.see = a.causal ? nk - nq + from + 1 : nk;
    it.n0 = (sees(it, min(it.tokens, a.tile_tokens) - 1) + kTileKeys - 1) / kTileKeys;
    it.n1 = it.tokens > a.tile_tokens ? (sees(it, it.tokens - 1) + kTileKeys - 1) / kTileKeys : 0;
    return it;
  };
  // 2 to 32 requests: the plan warp has one a lane, those with the most keys first, so that the last items are short ones; `upto`
  // are the running sums of their pairs in that order, `who` the lane of the place.
  const bool few = a.requests > 1 && a.requests <= 32;
  int q0 = 0, nq = 0, k0 = 0, nk = 0, who = lane, pairs = 0, upto = 0, items_all = (int)a.items;
  auto rank_requests = [&] {
    if (lane < a.requests && sound(lane)) {
      q0 = a.query_begin[lane];
      nq = a.query_begin[lane + 1] - q0;
      k0 = a.key_begin[lane];
      nk = a.key_begin[lane + 1] - k0;
    }
    pairs = pairs_of(nq);
    int rank = 0;
#pragma unroll 8
    for (int b = 0; b < a.requests; ++b) {   // lanes behind the last stand behind it
      const int keys = __shfl_sync(kAll, nk, b);
      rank += keys > nk || (keys == nk && b < lane);
    }
    order[lane < a.requests ? rank : lane] = lane;
    __syncwarp();
    who = order[lane];
    pairs = __shfl_sync(kAll, pairs, who);
    upto = pairs;
    for (int o = 1; o < a.requests; o <<= 1) {
      const int u = __shfl_up_sync(kAll, upto, o);
      if (lane >= o) upto += u;
    }
    items_all = (int)min((int64_t)__shfl_sync(kAll, upto, a.requests - 1) * a.kv_heads, a.items);
  };
  // the w-th item, by a warp; nothing valid where the slot is empty or the request's numbers are out of range
  auto item_of = [&](int w) {
    const int head = w % a.kv_heads, slot = w / a.kv_heads;
    if (few) {
      const unsigned behind = __ballot_sync(kAll, upto > slot);
      if (!behind) return Item{};
      const int place = __ffs(behind) - 1, from = __shfl_sync(kAll, who, place), local = slot - __shfl_sync(kAll, upto - pairs, place);
      return make_item(head, __shfl_sync(kAll, q0, from), __shfl_sync(kAll, nq, from), __shfl_sync(kAll, k0, from), __shfl_sync(kAll, nk, from), local);
    }
    int lo = 0, hi = a.requests;          // first_slot(lo) <= slot, first_slot(hi) > slot (or hi = requests)
    while (hi - lo > 1) {
      const int step = (hi - lo + 31) / 32, b = lo + lane * step;
      const unsigned before = __ballot_sync(kAll, b < hi && first_slot(a, b) <= slot);
      const int last = before ? 31 - __clz(before) : 0;
      hi = min(hi, lo + (last + 1) * step);
      lo = lo + last * step;
    }
    const int begin = a.query_begin[lo], n = a.query_begin[lo + 1] - begin, first = a.key_begin[lo], keys = a.key_begin[lo + 1] - first, local = slot - first_slot(a, lo);
    return sound(lo) && local >= 0 && local < pairs_of(n) ? make_item(head, begin, n, first, keys, local) : Item{};
  };
  Item it{};
  if (warp == kPlanWarp) {
    if (lane < 3) asm volatile("prefetch.tensormap [%0];" ::"l"(lane == 0 ? &q_map : lane == 1 ? &k_map : &v_map) : "memory");
    pdl_wait();
    if (few) rank_requests();
    it = item_of(blockIdx.x);
  }
  // rows of a tile that no token fills (128 is no multiple of the group): zero for good
  for (int i = a.tile_tokens * a.group * 8 + tid; i < kTileRows * 8; i += kThreads)
    for (int h = 0; h < kTiles * DP / 64; ++h) asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(smem + h * S::kHalf + i * 16), "r"(0) : "memory");
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  pdl_wait();
  pdl_trigger();
  const uint32_t tmem = tmem_slot;
  int loaded = 0, asked = 0;                       // loader: tiles asked for; plan: items whose queries were
  uint32_t on_landed = 0, landed_parity = 0;       // bits of stages: the last tile goes by `landed`; which phase comes next

  // the CTA's n-th item; `one`: a thread alone takes it for its warp
  auto take = [&](int n, Item& it, bool one) {
    bool ok = tc::mbar_wait(item_full(n), n >> 1 & 1, &gave_up);
    if (!one) ok = __all_sync(kAll, ok);
    if (!ok) return false;
    it = items[n & 1];
    if (!one) __syncwarp();
    if (one || lane == 0) tc::mbar_arrive(item_empty(n));
    return it.valid != 0;
  };
  // V tiles that are looked at before the products.  Behind the last key stand other rows, of which P = 0 would make NaN where they
  // hold one: zeroed.  So would a value that is not finite, of a key that only some of the rows see: the product goes without it,
  // and the rows that do see it add it in the end.
  auto ragged = [&](const Item& it, int j) { return it.keys - j * kTileKeys < kTileKeys; };
  auto parted = [&](const Item& it, int j) { return a.causal && (j + 1) * kTileKeys > sees(it, 0); };

  if (warp == kPlanWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    // items while the others work on the one before: the first by the CTA's number, then from the common counter
    bool alive = true;
    for (int n = 0, w = blockIdx.x;;) {
      const bool more = alive && w < items_all;
      if (w != (int)blockIdx.x) it = more ? item_of(w) : Item{};
      if (it.valid || !more) {
        if (n >= 2) alive = __all_sync(kAll, tc::mbar_wait(item_empty(n), (n >> 1) - 1 & 1, &gave_up)) && alive;
        if (alive && lane == 0) {
          items[n & 1] = it;
          tc::mbar_arrive(item_full(n));
        }
      }
      if (!more || !alive) break;
      if (it.valid) {
        // its queries, once the scores of the item before are done with theirs
        if (n > 0) alive = __all_sync(kAll, tc::mbar_wait(q_empty, n - 1 & 1, &gave_up));
        if (alive && lane == 0) {
          const int tiles = it.tokens > a.tile_tokens ? 2 : 1;
          tc::mbar_arrive_expect_tx(q_ready, tiles * (DP / 64) * a.tile_tokens * a.group * 128);
          for (int t = 0; t < tiles; ++t)
            for (int h = 0; h < DP / 64; ++h)
              tma_load_3d(smem + t * S::kTile + h * S::kHalf, &q_map, 64 * h, it.head * a.group, it.token + t * a.tile_tokens, q_ready);
        }
        asked += alive;
        ++n;
      }
      if (lane == 0) w = atomicAdd(a.next, 1) + gridDim.x;
      w = __shfl_sync(kAll, w, 0);
    }
    if (lane == 0 && atomicAdd(a.next + 1, 1) == (int)gridDim.x - 1) {
      a.next[0] = 0;
      a.next[1] = 0;
    }
  } else if (warp == kCheckWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    for (int b = blockIdx.x * 32 + lane; b < a.requests; b += gridDim.x * 32)
      if (!sound(b)) *a.bad = 1;
    bool alive = true;
    Item it;
    for (int n = 0, first = 0; alive && take(n, it, false); ++n) {
      const int tiles = max(it.n0, it.n1);
      for (int j = 0; alive && j < tiles; ++j) {
        const bool some = ragged(it, j), part = parted(it, j);
        if (!some && !part) continue;
        const int s = (first + 2 * j + 1) % kStages;
        alive = __all_sync(kAll, tc::mbar_wait(landed(s), landed_parity >> s & 1, &gave_up));
        landed_parity ^= 1u << s;
        if (!alive) break;
        const uint32_t tile = smem + S::kQ + s * S::kTile;
        if (some) {
          for (int i = (it.keys - j * kTileKeys) * 8 + lane; i < kTileKeys * 8; i += 32)
            for (int h = 0; h < DP / 64; ++h)
              asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(tile + h * S::kHalf + i * 16), "r"(0) : "memory");
          __syncwarp();
        }
        if (part) {
          const int from = max(0, sees(it, 0) - j * kTileKeys) * 8, to = min(it.keys - j * kTileKeys, kTileKeys) * 8;
          uint32_t zero = 0;   // sums of 0 * x
          for (int h = 0; h < DP / 64; ++h)
#pragma unroll 8
            for (int i = from + lane; i < to; i += 32) {
              const uint4 w = load_shared(tile + h * S::kHalf + i * 16);
              zero = fma_zero<kBf16>(fma_zero<kBf16>(fma_zero<kBf16>(fma_zero<kBf16>(zero, w.x), w.y), w.z), w.w);
            }
          if (__any_sync(kAll, zero & 0x7fff7fffu)) {
            for (int h = 0; h < DP / 64; ++h)
              for (int i = 4 * from + lane; i < 4 * to; i += 32) {
                const uint32_t at = tile + h * S::kHalf + i * 4;
                uint32_t w;
                asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w) : "r"(at));
                if (odd_half<kBf16>(w & 0xffffu)) w &= 0xffff0000u;
                if (odd_half<kBf16>(w >> 16)) w &= 0xffffu;
                asm volatile("st.shared.b32 [%0], %1;" ::"r"(at), "r"(w) : "memory");
              }
            if (lane == 0) *const_cast<volatile int*>(&items[n & 1].odd) = 1;
            __threadfence_block();
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(full(s));
      }
      first = (first + 2 * tiles) % kStages;
    }
  } else if (warp == kLoadWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    // K tile, V tile, K tile, ... of the walks
    bool alive = true;
    Item it;
    for (int n = 0; alive && take(n, it, false); ++n) {
      const int count = 2 * max(it.n0, it.n1);
      for (int e = 0; e < count; ++e, ++loaded) {
        const int s = loaded % kStages, j = e >> 1;
        if (loaded >= kStages) alive = __all_sync(kAll, tc::mbar_wait(empty(s), (loaded / kStages - 1) & 1, &gave_up));
        if (!alive) break;
        const bool values = e & 1, check = values && (ragged(it, j) || parted(it, j));
        if (check) {
          landed_parity ^= 1u << s;
          on_landed |= 1u << s;
        } else {
          on_landed &= ~(1u << s);
        }
        if (lane == 0) {
          const uint32_t dst = smem + S::kQ + s * S::kTile, bar = check ? landed(s) : full(s);
          tc::mbar_arrive_expect_tx(bar, S::kTile);
          for (int h = 0; h < DP / 64; ++h) tma_load_3d(dst + h * S::kHalf, values ? &v_map : &k_map, 64 * h, it.head, it.first_key + j * kTileKeys, bar);
        }
      }
    }
  } else if (warp == kMmaWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (tc::elect_one()) {
      constexpr uint32_t type = kBf16 ? 1u : 0u;
      constexpr uint32_t common = 1u << 4 | type << 7 | type << 10 | (uint32_t)(kTileRows >> 4) << 24;
      constexpr uint32_t idesc_s = common | (uint32_t)(kTileKeys >> 3) << 17;
      constexpr uint32_t idesc_o = common | 1u << 16 | (uint32_t)(DP >> 3) << 17;
      // the stages that keys and values are in now, and the parity of their use; of a row tile's weights
      int k_stage = 0, v_stage = 1;
      uint32_t k_parity = 0, v_parity = 0, p_parity[kTiles] = {0, 0};
      auto next = [&](int& stage, uint32_t& parity) {
        stage += 2;
        if (stage >= kStages) {
          stage -= kStages;
          parity ^= 1;
        }
      };
      auto scores = [&](int t) {
        const uint32_t keys = row_desc(smem + S::kQ + k_stage * S::kTile), queries = row_desc(smem + t * S::kTile);
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk) {
          const uint32_t off = (kk / 4 * S::kHalf + kk % 4 * 32) >> 4;
          mma_ss(tmem + t * 128, queries + off, keys + off, idesc_s, kk > 0);
        }
        tc::mma_commit(s_ready(t));
      };
      // One issuer for both row tiles, in turns: the products of one run while the other's exponentials are taken
      bool alive = true;
      Item it;
      for (int n = 0; alive && take(n, it, true); ++n) {
        const int key_tiles = max(it.n0, it.n1);
        alive = tc::mbar_wait(q_ready, n & 1, &gave_up) && (key_tiles == 0 || tc::mbar_wait(full(k_stage), k_parity, &gave_up));
        if (!alive) break;
        tc::fence_after();
        // an item's first scores go where the last weights of the item before stood, behind the mix that reads those
        if (it.n0 > 0) scores(0);
        if (it.n1 > 0) scores(1);
        if (key_tiles <= 1) tc::mma_commit(q_empty);
        for (int j = 0; alive && j < key_tiles; ++j) {
          tc::mma_commit(empty(k_stage));
          next(k_stage, k_parity);
          alive = tc::mbar_wait(full(v_stage), v_parity, &gave_up);
          const uint32_t values = value_desc(smem + S::kQ + v_stage * S::kTile);
#pragma unroll
          for (int t = 0; t < kTiles; ++t) {
            const int n_mine = t ? it.n1 : it.n0;
            if (j < n_mine) {
#pragma unroll
              for (int half = 0; half < 2; ++half) {
                alive = alive && tc::mbar_wait(p_ready(t, half), p_parity[t], &gave_up);
                if (!alive) break;
                tc::fence_after();
#pragma unroll
                for (int kk = 4 * half; kk < 4 * half + 4; ++kk)
                  mma_ts(tmem + 256 + t * 128, tmem + t * 128 + kk * 8, values + (kk * 2048 >> 4), idesc_o, kk > 0 ? 1 : j % kFold != 0);
              }
              p_parity[t] ^= 1;
              if (alive && j + 1 == n_mine) tc::mma_commit(o_ready(t));
            }
            if (t == 0 && j + 1 < key_tiles) alive = alive && tc::mbar_wait(full(k_stage), k_parity, &gave_up);
            if (!alive) break;
            if (j + 1 < n_mine) scores(t);
          }
          if (alive && j + 2 == key_tiles) tc::mma_commit(q_empty);   // the last scores have been issued
          if (alive) tc::mma_commit(empty(v_stage));
          next(v_stage, v_parity);
        }
      }
      if (!alive) {
        // let what was issued end
        volatile int own = 0;
        tc::mma_commit(drain_bar);
        tc::mbar_wait(drain_bar, 0, &own);
      }
    }
    __syncwarp();
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    const int t = warp >> 2, row = tid & 127, token = t * a.tile_tokens + min(token_of(row), a.tile_tokens - 1);   // of the item
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_col = tmem + t * 128 + lanes, o_col = tmem + 256 + t * 128 + lanes;
    const uint32_t turn = smem + S::kQ + kStages * S::kTile + warp * S::kTurn;
    const tc::f2 scale2 = tc::pack2(a.scale_log2, a.scale_log2);
    uint32_t s_parity = 0, o_parity = 0;
    bool alive = true;
    // the item stays in shared memory until it is done: this warp's registers hold scores
    for (int n = 0;; ++n) {
      alive = __all_sync(kAll, tc::mbar_wait(item_full(n), n >> 1 & 1, &gave_up));
      const Item& it = items[n & 1];
      if (!alive || !it.valid) break;
      const int n_mine = t ? it.n1 : it.n0;
      const int see = sees(it, min(token, it.tokens - 1)), see_all = sees(it, t * a.tile_tokens);   // of the row, of every row
      float m = kLowest;
      int far = 0;   // 1: scores count from a base, 2: from this tile on, which is taken once more
      tc::f2 sum2 = tc::pack2(0.0f, 0.0f);
      for (int j = 0; j < n_mine; ++j) {
        alive = __all_sync(kAll, tc::mbar_wait(s_ready(t), s_parity, &gave_up));
        if (!alive) break;
        s_parity ^= 1;
        tc::fence_after();
        if (j > 0 && j % kFold == 0 && far < 2) {   // the mix so far is done, as below
          fold_away<DP>(a.fold, t, row, o_col, j == kFold, m, tc::unpack2(sum2));
          sum2 = tc::pack2(0.0f, 0.0f);
        }
        if (far) {
          m = rebase(a.fold, t, row, s_col, see - j * kTileKeys, a.scale_log2, far == 2, m);
          far = 1;
        }
        uint32_t s[128];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(s_col + 32 * c, s + 32 * c);
        wait_ld(s);
        if ((j + 1) * kTileKeys > see_all) {
          const int in_tile = see - j * kTileKeys;
#pragma unroll
          for (int i = 0; i < 128; ++i)
            if (i >= in_tile) s[i] = __float_as_uint(-INFINITY);
        }
        float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < 128; i += 8)
#pragma unroll
          for (int e = 0; e < 4; ++e) top[e] = max_nan(top[e], max_nan(__uint_as_float(s[i + 2 * e]), __uint_as_float(s[i + 2 * e + 1])));
        // a NaN stays the maximum: the row's weights are all NaN then
        const float now = max_nan(max_nan(top[0], top[1]), max_nan(top[2], top[3])) * a.scale_log2;
        if (__any_sync(kAll, !(now <= m + kSlack))) {
          const float next = max_nan(m, now), f = exp2_fast(m - next);
          if (!far && __any_sync(kAll, fabsf(next) >= kFarScore && next != kLowest)) {
            far = 2;
            s_parity ^= 1;
            --j;
            continue;
          }
          m = next;
          sum2 = tc::mul2(sum2, tc::pack2(f, f));
          // the mix so far: its last product was issued before these scores, so it is done
          if (j % kFold != 0) {
#pragma unroll 1
            for (int c = 0; c < DP; c += 32) {
              uint32_t o[32];
              tmem_ld32(o_col + c, o);
              wait_ld(o);
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
              tc::tmem_st32(o_col + c, o);
            }
          }
        }
        const tc::f2 minus_m = tc::pack2(kRaise<kBf16> - m, kRaise<kBf16> - m);
        tc::f2 tile2 = tc::pack2(0.0f, 0.0f);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint32_t p[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const float2 x = tc::unpack2(tc::fma2(tc::pack2u(s[64 * half + 2 * i], s[64 * half + 2 * i + 1]), scale2, minus_m));
            const float e0 = exp2_fast(x.x), e1 = exp2_fast(x.y);
            tile2 = tc::add2(tile2, tc::pack2(e0, e1));
            p[i] = pack16<kBf16>(e0, e1);
          }
          tc::tmem_st32(s_col + 32 * half, p);
          tc::tmem_wait_st();
          tc::fence_before();
          __syncwarp();
          if (lane == 0) tc::mbar_arrive(p_ready(t, half));
        }
        sum2 = tc::add2(sum2, tile2);
      }
      if (alive && n_mine > 0) {
        alive = __all_sync(kAll, tc::mbar_wait(o_ready(t), o_parity, &gave_up));
        o_parity ^= 1;
      }
      if (!alive) break;
      tc::fence_after();
      const float2 two = tc::unpack2(sum2);
      float sum = two.x + two.y;
      if (n_mine > kFold) sum = fold_back<DP>(a.fold, t, row, o_col, m, sum);
      const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
      // 64 dims at a time through shared memory, so that a warp stores 128 bytes of a row at once; addresses are made here, not kept
      // in registers from item to item
      int l = lane;
      asm volatile("" : "+r"(l));
      const int tokens = it.tokens;
      uint16_t* out = static_cast<uint16_t*>(a.out) + it.token * a.os + (int64_t)it.head * a.group * a.oh;
#pragma unroll 1
      for (int half = 0; half < DP / 64; ++half) {
        if (t * a.tile_tokens >= tokens) break;
        uint32_t o[64];
        tmem_ld32(o_col + 64 * half, o);   // of rows that saw nothing (inv = 0): whatever stands there
        tmem_ld32(o_col + 64 * half + 32, o + 32);
        wait_ld(o);
        if (*const_cast<const volatile int*>(&it.odd)) {
#pragma unroll 1
          for (int key = sees(it, 0); key < see; ++key)
#pragma unroll
            for (int c = 0; c < 8; ++c) {
              if (64 * half + 8 * c >= a.head_dim) break;
              const uint4 w = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.v) + (int64_t)(it.first_key + key) * a.vs +
                                                              (int64_t)it.head * a.vh + 64 * half + 8 * c);
              const uint32_t word[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const uint32_t x = word[e / 2] >> 16 * (e & 1) & 0xffffu;
                if (odd_half<kBf16>(x)) o[8 * c + e] = __float_as_uint(__uint_as_float(o[8 * c + e]) + as_float<kBf16>(x));
              }
            }
        }
        if (__any_sync(kAll, inv == 0.0f)) {
#pragma unroll
          for (int i = 0; i < 64; ++i) o[i] = inv == 0.0f ? 0u : o[i];
        }
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          uint32_t w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) w[e] = pack16<kBf16>(__uint_as_float(o[8 * c + 2 * e]) * inv, __uint_as_float(o[8 * c + 2 * e + 1]) * inv);
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(turn + l * 128 + (c ^ (l & 7)) * 16), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3])
                       : "memory");
        }
        __syncwarp();
        const int c = l & 7;
        uint4 w[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) w[k] = load_shared(turn + (4 * k + (l >> 3)) * 128 + (c ^ ((4 * k + (l >> 3)) & 7)) * 16);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int to_row = (row & ~31) + 4 * k + (l >> 3), in_tile = token_of(to_row), to = t * a.tile_tokens + in_tile, h = to_row - in_tile * a.group;
          if (in_tile < a.tile_tokens && to < tokens && 64 * half + 8 * c < a.head_dim)
            *reinterpret_cast<uint4*>(out + (int64_t)to * a.os + (int64_t)h * a.oh + 64 * half + 8 * c) = w[k];
        }
        __syncwarp();
      }
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(item_empty(n));
    }
  }
  // a wait that ran out: copies in flight end before the CTA does
  __syncwarp();
  if (gave_up) {
    if (tid == 0) *a.status = 1;
    if (warp == kLoadWarp) {
      volatile int own = 0;
      for (int e = max(0, loaded - kStages); e < loaded; ++e) {
        const int s = e % kStages;
        own = 0;
        if (on_landed >> s & 1) tc::mbar_wait(landed(s), ~landed_parity >> s & 1, &own);
        else tc::mbar_wait(full(s), e / kStages & 1, &own);
      }
    }
    if (warp == kPlanWarp && asked > 0) {
      volatile int own = 0;
      tc::mbar_wait(q_ready, asked - 1 & 1, &own);
    }
  }
  tc::fence_before();
  __syncthreads();
  if (warp == kMmaWarp) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
}

// rows {tokens, heads, head_dim} for boxes 64 dims wide
bool encode_rows(Map* map, const void* base, bool bf16, int head_dim, int heads, int tokens, int64_t token_stride, int64_t head_stride, int box_heads,
                 int box_tokens) {
  static_assert(sizeof(CUtensorMap) == sizeof(Map), "tensor map size");
  static const PFN_cuTensorMapEncodeTiled_v12000 encode = [] {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &found) != cudaSuccess) {
      cudaGetLastError();
      fn = nullptr;
    }
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
  }();
  if (!encode) return false;
  // a stride that no second row or head uses may be anything in the request
  if (heads == 1) head_stride = head_dim;
  if (tokens <= 1) token_stride = (int64_t)head_dim * heads;
  const cuuint64_t dims[3] = {(cuuint64_t)head_dim, (cuuint64_t)heads, (cuuint64_t)(tokens > 0 ? tokens : 1)};
  const cuuint64_t strides[2] = {(cuuint64_t)head_stride * 2, (cuuint64_t)token_stride * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)box_heads, (cuuint32_t)box_tokens}, steps[3] = {1, 1, 1};
  return encode(reinterpret_cast<CUtensorMap*>(map), bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(base),
                dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int DP, bool kBf16>
cudaError_t launch_one(const PackedArgs& a, const Map& q, const Map& k, const Map& v, int sm_count, bool pdl, cudaStream_t st) {
  const int smem = Smem<DP>::kBytes;
  cudaError_t e = cudaFuncSetAttribute(attend_packed_kernel<DP, kBf16>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  return launch_kernel(attend_packed_kernel<DP, kBf16>, dim3((unsigned)std::min<int64_t>(a.items, sm_count)), dim3(kThreads), smem, st, pdl, a, q, k, v);
}

}  // namespace

cudaError_t launch_attend_packed(const emelb_attend_packed_request& r, int* next, float* fold, int sm_count, int* bad, int* status, bool pdl, cudaStream_t st) {
  PackedArgs a{};
  a.out = r.out;
  a.query_begin = r.query_begin;
  a.key_begin = r.key_begin;
  a.v = r.v;
  a.vs = r.v_token_stride;
  a.vh = r.v_head_stride;
  a.os = r.out_token_stride;
  a.oh = r.out_head_stride;
  a.requests = r.requests;
  a.kv_heads = r.kv_heads;
  a.group = r.heads / r.kv_heads;
  a.group_inv = (65536 + a.group - 1) / a.group;
  a.tile_tokens = kTileRows / a.group;
  a.head_dim = r.head_dim;
  a.queries = r.queries;
  a.keys = r.keys;
  a.max_queries = r.max_queries;
  a.causal = r.causal != 0;
  a.scale_log2 = r.scale * 1.44269504088896340736f;
  a.items = ((int64_t)a.queries / (kTiles * a.tile_tokens) + a.requests) * a.kv_heads;
  if (a.items > 0x3fffffff) return cudaErrorInvalidValue;
  a.next = next;
  a.bad = bad;
  a.status = status;
  a.fold = fold;
  const bool bf16 = r.type == EMELB_BF16;
  Map q, k, v;
  if (!encode_rows(&q, r.q, bf16, r.head_dim, r.heads, r.queries, r.q_token_stride, r.q_head_stride, a.group, a.tile_tokens) ||
      !encode_rows(&k, r.k, bf16, r.head_dim, r.kv_heads, r.keys, r.k_token_stride, r.k_head_stride, 1, kTileKeys) ||
      !encode_rows(&v, r.v, bf16, r.head_dim, r.kv_heads, r.keys, r.v_token_stride, r.v_head_stride, 1, kTileKeys))
    return cudaErrorInvalidValue;
  if (r.head_dim <= 64) return bf16 ? launch_one<64, true>(a, q, k, v, sm_count, pdl, st) : launch_one<64, false>(a, q, k, v, sm_count, pdl, st);
  return bf16 ? launch_one<128, true>(a, q, k, v, sm_count, pdl, st) : launch_one<128, false>(a, q, k, v, sm_count, pdl, st);
}

}  // namespace emelb
