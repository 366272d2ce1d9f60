// Attention of packed prompts of different lengths, on the Blackwell tensor cores.
//
// Per request and key / value head, the query rows of the head's group stand behind one another, token after token, so that a
// short prompt fills tiles of rows too.  A CTA takes 256 of them as two tiles of 128 and walks the keys in tiles of 128:
//   S = Q K^T       tcgen05.mma, operands in shared memory, K by TMA; S {128 rows, 128 keys} in TMEM, a row a lane
//   P = exp2(S - m) a thread a row: 128 scores out of TMEM, running maximum and sum, P as 16-bit values back over S
//   O += P V        tcgen05.mma, P as the A operand out of TMEM, V by TMA as it lies in memory (its dims are contiguous: MN-major)
// While the warps of one tile take the exponentials, the tensor cores work for the other.  The running maximum a row's weights are
// taken against follows the true one only when that has passed it by 2^8: only then does O, in TMEM, have to be rescaled.
//
// Two matrix products of 128 x 128 x head_dim and 128 x 128 exponentials a tile: at head_dim 128 both take the same time (4096
// products, 16 exponentials a cycle and SM: 2048 cycles for two row tiles and 128 keys), at 64 the exponentials bound it.  What a
// row tile waits for, between its last weight and its next score, is the other's time; together they take about 2,900 cycles.
//
// us, two prompts of 4100 and 8190 tokens, 32 heads of 128: 756 with weights handed over at once and an arrival a thread, 659 by
// halves and with registers split, 578 (1,189 TFLOP/s) since queries come by asynchronous copies.  Measured and left out: an issuer of
// products for each row tile 613 (they fall into step and wait for the same pipes); scores of 64 keys in two buffers a row tile, so
// that none waits for a mix, 588 (products with 64 columns take longer); weights against a stale maximum, looked at afterwards, 604;
// an eighth, a quarter of the exponentials by polynomials on the multiply-adds 578, 586.
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "paged.h"
#include "tc_common.cuh"

namespace emelb {
namespace {

constexpr unsigned kAll = 0xffffffffu;
constexpr int kTileRows = 128, kTileKeys = 128, kTiles = 2;   // tiles of a CTA
constexpr int kLoadWarp = 8, kMmaWarp = 9, kThreads = 384;
// registers a thread behind the start, of the 168 that 384 threads launch with: 8 warps x 208 + 4 x 88 = 12 x 168
constexpr int kSoftmaxRegs = 208, kOtherRegs = 88;
static_assert(8 * kSoftmaxRegs + 4 * kOtherRegs <= 12 * 168, "registers");
constexpr float kLowest = -3.0e38f;
constexpr float kSlack = 8.0f;
constexpr int kTmemCols = 512;

struct __align__(64) Map {
  unsigned char bytes[128];
};

struct PackedArgs {
  const void* q;
  void* out;
  const int32_t *query_begin, *key_begin;
  int64_t qs, qh, os, oh;
  int requests, kv_heads, group, group_inv, head_dim, queries, keys, max_queries, causal;
  float scale_log2;
  int *bad, *status;
};

template <int DP>
struct Smem {
  static constexpr int kHalf = kTileKeys * 128;          // 64 dims of 128 rows
  static constexpr int kTile = DP / 64 * kHalf;
  static constexpr int kStages = DP == 128 ? 5 : 10;     // of K and V tiles in turn
  static constexpr int kQ = kTiles * kTile;
  static constexpr int kBytes = kQ + kStages * kTile + 1024;
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

// Row tiles of request b stand in slots first_slot(b) .. first_slot(b + 1) - 1, of which it may leave one empty: rows before it / 256
// + b is known from query_begin alone, without a sum over the requests in front.
__device__ __forceinline__ int64_t first_slot(const PackedArgs& a, int b) {
  return (int64_t)(a.query_begin[b] - a.query_begin[0]) * a.group / (kTiles * kTileRows) + b;
}

template <int DP, bool kBf16>
__global__ void __launch_bounds__(kThreads, 1)
    attend_packed_kernel(const __grid_constant__ PackedArgs a, const __grid_constant__ Map k_map, const __grid_constant__ Map v_map) {
  using S = Smem<DP>;
  constexpr int kStages = S::kStages;
  extern __shared__ uint8_t raw[];
  __shared__ uint64_t bars[2 * kStages + 5 * kTiles + 2];
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int gave_up;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t smem = (tc::smem_u32(raw) + 1023u) & ~1023u;
  const uint32_t bar0 = tc::smem_u32(bars);
  auto full = [&](int s) { return bar0 + 8 * s; };
  auto empty = [&](int s) { return bar0 + 8 * (kStages + s); };
  auto q_ready = [&](int t) { return bar0 + 8 * (2 * kStages + t); };
  auto s_ready = [&](int t) { return bar0 + 8 * (2 * kStages + kTiles + t); };
  auto o_ready = [&](int t) { return bar0 + 8 * (2 * kStages + 2 * kTiles + t); };
  auto p_ready = [&](int t, int half) { return bar0 + 8 * (2 * kStages + (3 + half) * kTiles + t); };   // 64 keys each
  const uint32_t raw_bar = bar0 + 8 * (2 * kStages + 5 * kTiles), drain_bar = raw_bar + 8;

  // ---- which rows
  const int head = blockIdx.x % a.kv_heads;
  const int64_t slot = blockIdx.x / a.kv_heads;
  int lo = 0, hi = a.requests;          // first_slot(lo) <= slot, first_slot(hi) > slot (or hi = requests)
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32, b = lo + lane * step;
    const unsigned before = __ballot_sync(kAll, b < hi && first_slot(a, b) <= slot);
    const int last = before ? 31 - __clz(before) : 0;
    hi = min(hi, lo + (last + 1) * step);
    lo = lo + last * step;
  }
  const int b = lo;
  const int q0 = a.query_begin[b], nq = a.query_begin[b + 1] - q0, k0 = a.key_begin[b], nk = a.key_begin[b + 1] - k0;
  if (a.query_begin[0] < 0 || q0 < 0 || nq < 0 || nq > a.max_queries || q0 > a.queries - nq || k0 < 0 || nk < 0 || k0 > a.keys - nk) {
    if (tid == 0) *a.bad = 1;
    return;
  }
  const int64_t rows = (int64_t)nq * a.group;
  const int64_t tiles = (rows + kTiles * kTileRows - 1) / (kTiles * kTileRows), local = slot - first_slot(a, b);
  if (local < 0 || local >= tiles) return;
  // rows of this CTA, counted from its first, which is head `part0` of token tok0; long walks first
  const int64_t row0 = (tiles - 1 - local) * (kTiles * kTileRows);
  const int n_rows = (int)min(rows - row0, (int64_t)(kTiles * kTileRows)), tok0 = (int)(row0 / a.group), part0 = (int)(row0 - (int64_t)tok0 * a.group);
  // (part0 + row) / group by a product: exact, since (part0 + row) * group < 2^16
  auto token_of = [&](int row) { return (int)((uint32_t)(part0 + row) * a.group_inv >> 16); };
  // keys that a row sees; row tiles of this CTA walk turns(t) key tiles
  auto sees = [&](int row) { return a.causal ? max(0, min(nk, nk - nq + tok0 + token_of(row) + 1)) : nk; };
  auto turns = [&](int t) {
    const int r = t * kTileRows;
    return r >= n_rows ? 0 : (sees(min(n_rows, r + kTileRows) - 1) + kTileKeys - 1) / kTileKeys;
  };
  const int n0 = turns(0), n1 = turns(1), key_tiles = max(n0, n1);

  if (tid == 0) {
    for (int s = 0; s < kStages; ++s) {
      tc::mbar_init(full(s), 1);
      tc::mbar_init(empty(s), 1);
    }
    for (int t = 0; t < kTiles; ++t) {
      tc::mbar_init(q_ready(t), kTileRows / 32);
      tc::mbar_init(s_ready(t), 1);
      tc::mbar_init(p_ready(t, 0), kTileRows / 32);
      tc::mbar_init(p_ready(t, 1), kTileRows / 32);
      tc::mbar_init(o_ready(t), 1);
    }
    tc::mbar_init(raw_bar, 1);
    tc::mbar_init(drain_bar, 1);
    gave_up = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc::smem_u32(&tmem_slot)), "r"(kTmemCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = tmem_slot;
  int loaded = 0;          // loader: tiles asked for

  if (warp == kLoadWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    // K tile, V tile, K tile, ... of the walk
    bool alive = true;
    for (; alive && loaded < 2 * key_tiles; ++loaded) {
      const int s = loaded % kStages, j = loaded >> 1;
      if (loaded >= kStages) alive = tc::mbar_wait(empty(s), (loaded / kStages - 1) & 1, &gave_up);
      if (!__all_sync(kAll, alive)) break;
      const bool values = loaded & 1;
      const int left = nk - j * kTileKeys;
      // behind the last key stand other rows, of which P = 0 would make NaN where they hold one: zeroed before anyone reads them
      const bool ragged = values && left < kTileKeys;
      const uint32_t dst = smem + S::kQ + s * S::kTile, bar = ragged ? raw_bar : full(s);
      if (lane == 0) {
        tc::mbar_arrive_expect_tx(bar, S::kTile);
        for (int h = 0; h < DP / 64; ++h) tma_load_3d(dst + h * S::kHalf, values ? &v_map : &k_map, 64 * h, head, k0 + j * kTileKeys, bar);
      }
      if (ragged) {
        __syncwarp();
        alive = tc::mbar_wait(raw_bar, 0, &gave_up);
        for (int i = left * 8 + lane; i < kTileKeys * 8; i += 32)
          for (int h = 0; h < DP / 64; ++h)
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(dst + h * S::kHalf + i * 16), "r"(0) : "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(full(s));
      }
    }
  } else if (warp == kMmaWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (tc::elect_one()) {
      constexpr uint32_t type = kBf16 ? 1u : 0u;
      constexpr uint32_t common = 1u << 4 | type << 7 | type << 10 | (uint32_t)(kTileRows >> 4) << 24;
      constexpr uint32_t idesc_s = common | (uint32_t)(kTileKeys >> 3) << 17;
      constexpr uint32_t idesc_o = common | 1u << 16 | (uint32_t)(DP >> 3) << 17;
      // the stages that keys and values are in now, and the parity of their use
      int k_stage = 0, v_stage = 1;
      uint32_t k_parity = 0, v_parity = 0;
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
      // One issuer for both row tiles, in turns: the products of one run while the other's exponentials are taken.  (An issuer each
      // let the tiles fall into step and wait for the same pipes: 613 us instead of 578 for 4100 and 8190 tokens.)
      bool alive = key_tiles == 0 || tc::mbar_wait(full(0), 0, &gave_up);
#pragma unroll
      for (int t = 0; t < kTiles; ++t)
        if (alive && (t ? n1 : n0) > 0) {
          alive = tc::mbar_wait(q_ready(t), 0, &gave_up);
          if (alive) scores(t);
        }
      for (int j = 0; alive && j < key_tiles; ++j) {
        tc::mma_commit(empty(k_stage));
        next(k_stage, k_parity);
        alive = tc::mbar_wait(full(v_stage), v_parity, &gave_up);
        const uint32_t values = value_desc(smem + S::kQ + v_stage * S::kTile);
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
          const int n_mine = t ? n1 : n0;
          if (j < n_mine) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              alive = alive && tc::mbar_wait(p_ready(t, half), j & 1, &gave_up);
              if (!alive) break;
              tc::fence_after();
#pragma unroll
              for (int kk = 4 * half; kk < 4 * half + 4; ++kk)
                mma_ts(tmem + 256 + t * 128, tmem + t * 128 + kk * 8, values + (kk * 2048 >> 4), idesc_o, kk > 0 ? 1 : j > 0);
            }
            if (alive && j + 1 == n_mine) tc::mma_commit(o_ready(t));
          }
          if (t == 0 && j + 1 < key_tiles) alive = alive && tc::mbar_wait(full(k_stage), k_parity, &gave_up);
          if (!alive) break;
          if (j + 1 < n_mine) scores(t);
        }
        if (alive) tc::mma_commit(empty(v_stage));
        next(v_stage, v_parity);
      }
      if (!alive) {
        // let what was issued end
        volatile int own = 0;
        tc::mma_commit(drain_bar);
        tc::mbar_wait(drain_bar, 0, &own);
      }
    }
    __syncwarp();
  } else if (warp > kMmaWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    const int t = warp >> 2, r = tid & 127, n_mine = t ? n1 : n0;
    const int row = t * kTileRows + r;
    const bool live = row < n_rows;
    if (n_mine > 0) {
      // queries: 16-byte pieces of rows into the swizzled K-major layout, zeros behind the last row and the last dim; a thread has
      // the same piece of every eighth (or sixteenth) row, all of them on their way at once
      constexpr int kPieces = DP / 8, kRowStep = kTileRows / kPieces;
      const int c = r % kPieces;
      const uint16_t* from = static_cast<const uint16_t*>(a.q) + (int64_t)(q0 + tok0) * a.qs + (int64_t)head * a.group * a.qh + c * 8;
#pragma unroll
      for (int k = 0; k < kPieces; ++k) {
        const int rr = r / kPieces + kRowStep * k, in_cta = t * kTileRows + rr, tok = token_of(in_cta), h = part0 + in_cta - tok * a.group;
        const bool there = in_cta < n_rows && c * 8 < a.head_dim;
        const uint32_t dst = smem + t * S::kTile + c / 8 * S::kHalf + rr * 128 + ((c % 8) ^ (rr & 7)) * 16;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(there ? from + tok * a.qs + h * a.qh : static_cast<const uint16_t*>(a.q)),
                     "r"(there ? 16 : 0)
                     : "memory");
      }
      cp_async_commit();
      cp_async_wait<0>();
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(q_ready(t));
    }
    const int see = sees(live ? row : n_rows - 1), see_all = n_mine > 0 ? sees(t * kTileRows) : 0;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_col = tmem + t * 128 + lanes, o_col = tmem + 256 + t * 128 + lanes;
    const tc::f2 scale2 = tc::pack2(a.scale_log2, a.scale_log2);
    float m = kLowest;
    tc::f2 sum2 = tc::pack2(0.0f, 0.0f);
    bool alive = true;
    for (int j = 0; j < n_mine; ++j) {
      alive = tc::mbar_wait(s_ready(t), j & 1, &gave_up);
      if (!__all_sync(kAll, alive)) {
        alive = false;
        break;
      }
      tc::fence_after();
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
        m = next;
        sum2 = tc::mul2(sum2, tc::pack2(f, f));
        // the mix so far: its last product was issued before these scores, so it is done
        if (j > 0) {
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
      const tc::f2 minus_m = tc::pack2(-m, -m);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t p[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const float2 x = tc::unpack2(tc::fma2(tc::pack2u(s[64 * half + 2 * i], s[64 * half + 2 * i + 1]), scale2, minus_m));
          const float e0 = exp2_fast(x.x), e1 = exp2_fast(x.y);
          sum2 = tc::add2(sum2, tc::pack2(e0, e1));
          p[i] = pack16<kBf16>(e0, e1);
        }
        tc::tmem_st32(s_col + 32 * half, p);
        tc::tmem_wait_st();
        tc::fence_before();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(p_ready(t, half));
      }
    }
    if (alive && n_mine > 0) alive = tc::mbar_wait(o_ready(t), 0, &gave_up);
    alive = __all_sync(kAll, alive);
    if (alive) {
      tc::fence_after();
      const float2 two = tc::unpack2(sum2);
      const float sum = two.x + two.y, inv = sum == 0.0f ? 0.0f : 1.0f / sum;
      const int tok = token_of(live ? row : 0), h = part0 + (live ? row : 0) - tok * a.group;
      uint16_t* out = static_cast<uint16_t*>(a.out) + (int64_t)(q0 + tok0 + tok) * a.os + (int64_t)(head * a.group + h) * a.oh;
      uint32_t o[DP];
      if (n_mine > 0) {
#pragma unroll
        for (int c = 0; c < DP; c += 32) tmem_ld32(o_col + c, o + c);
        wait_ld(o);
      }
#pragma unroll
      for (int c = 0; c < DP; c += 8) {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          w[e] = inv == 0.0f ? 0u : pack16<kBf16>(__uint_as_float(o[c + 2 * e]) * inv, __uint_as_float(o[c + 2 * e + 1]) * inv);
        if (live && c < a.head_dim) *reinterpret_cast<uint4*>(out + c) = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  }
  // a wait that ran out: copies in flight end before the CTA does
  __syncwarp();
  if (gave_up) {
    if (tid == 0) *a.status = 1;
    if (warp == kLoadWarp) {
      volatile int own = 0;
      for (int e = max(0, loaded - kStages); e < loaded; ++e) {
        own = 0;
        tc::mbar_wait(full(e % kStages), e / kStages & 1, &own);
      }
    }
  }
  tc::fence_before();
  __syncthreads();
  if (warp == kMmaWarp) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
}

// rows {keys, kv_heads, head_dim} for boxes of 128 keys of one head, 64 dims wide
bool encode_rows(Map* map, const void* base, bool bf16, int head_dim, int heads, int keys, int64_t token_stride, int64_t head_stride) {
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
  if (keys <= 1) token_stride = (int64_t)head_dim * heads;
  const cuuint64_t dims[3] = {(cuuint64_t)head_dim, (cuuint64_t)heads, (cuuint64_t)(keys > 0 ? keys : 1)};
  const cuuint64_t strides[2] = {(cuuint64_t)head_stride * 2, (cuuint64_t)token_stride * 2};
  const cuuint32_t box[3] = {64, 1, kTileKeys}, steps[3] = {1, 1, 1};
  return encode(reinterpret_cast<CUtensorMap*>(map), bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(base),
                dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int DP, bool kBf16>
cudaError_t launch_one(const PackedArgs& a, const Map& k, const Map& v, cudaStream_t st) {
  const int smem = Smem<DP>::kBytes;
  cudaError_t e = cudaFuncSetAttribute(attend_packed_kernel<DP, kBf16>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  const int64_t slots = (int64_t)a.queries * a.group / (kTiles * kTileRows) + a.requests;
  if (slots * a.kv_heads > 0x7fffffff) return cudaErrorInvalidValue;
  attend_packed_kernel<DP, kBf16><<<(unsigned)(slots * a.kv_heads), kThreads, smem, st>>>(a, k, v);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_attend_packed(const emelb_attend_packed_request& r, int sm_count, int* bad, int* status, cudaStream_t st) {
  PackedArgs a{};
  a.q = r.q;
  a.out = r.out;
  a.query_begin = r.query_begin;
  a.key_begin = r.key_begin;
  a.qs = r.q_token_stride;
  a.qh = r.q_head_stride;
  a.os = r.out_token_stride;
  a.oh = r.out_head_stride;
  a.requests = r.requests;
  a.kv_heads = r.kv_heads;
  a.group = r.heads / r.kv_heads;
  a.group_inv = (65536 + a.group - 1) / a.group;
  a.head_dim = r.head_dim;
  a.queries = r.queries;
  a.keys = r.keys;
  a.max_queries = r.max_queries;
  a.causal = r.causal != 0;
  a.scale_log2 = r.scale * 1.44269504088896340736f;
  a.bad = bad;
  a.status = status;
  const bool bf16 = r.type == EMELB_BF16;
  Map k, v;
  if (!encode_rows(&k, r.k, bf16, r.head_dim, r.kv_heads, r.keys, r.k_token_stride, r.k_head_stride) ||
      !encode_rows(&v, r.v, bf16, r.head_dim, r.kv_heads, r.keys, r.v_token_stride, r.v_head_stride))
    return cudaErrorInvalidValue;
  if (r.head_dim <= 64) return bf16 ? launch_one<64, true>(a, k, v, st) : launch_one<64, false>(a, k, v, st);
  return bf16 ? launch_one<128, true>(a, k, v, st) : launch_one<128, false>(a, k, v, st);
}

}  // namespace emelb
