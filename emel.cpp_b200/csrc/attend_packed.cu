// Attention of packed prompts of different lengths.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "paged.h"

namespace emelb {
namespace {

constexpr unsigned kAll = 0xffffffffu;

struct PackedArgs {
  emelb_attend_packed_request r;
  int group;
  float scale_log2;
  int* bad;
};

template <class E>
__device__ __forceinline__ float value_of(E x);
template <>
__device__ __forceinline__ float value_of<__half>(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float value_of<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <class E>
__device__ __forceinline__ E elem_of(float x);
template <>
__device__ __forceinline__ __half elem_of<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 elem_of<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// a warp to a (query row, head): 32 keys a turn, a key a lane, then the dims of the mix across the lanes
template <class E>
__global__ void __launch_bounds__(128) attend_packed_rows_kernel(const __grid_constant__ PackedArgs a) {
  const emelb_attend_packed_request& r = a.r;
  __shared__ float query[4][128];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, head = blockIdx.y, row = blockIdx.x * 4 + warp, D = r.head_dim;
  if (row >= r.queries || row < r.query_begin[0] || row >= r.query_begin[r.requests]) return;
  int lo = 0, hi = r.requests - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (r.query_begin[mid] <= row) lo = mid;
    else hi = mid - 1;
  }
  const int q0 = r.query_begin[lo], q1 = r.query_begin[lo + 1], k0 = r.key_begin[lo], k1 = r.key_begin[lo + 1];
  if (q0 < 0 || q1 > r.queries || row >= q1 || q1 - q0 > r.max_queries || k0 < 0 || k1 < k0 || k1 > r.keys) {
    *a.bad = 1;
    return;
  }
  const int sees = r.causal ? min(k1 - k0, k1 - k0 - (q1 - q0) + (row - q0) + 1) : k1 - k0;
  const E* q = static_cast<const E*>(r.q) + row * r.q_token_stride + head * r.q_head_stride;
  const E* k = static_cast<const E*>(r.k) + k0 * r.k_token_stride + head / a.group * r.k_head_stride;
  const E* v = static_cast<const E*>(r.v) + k0 * r.v_token_stride + head / a.group * r.v_head_stride;
  for (int d = lane; d < D; d += 32) query[warp][d] = value_of<E>(q[d]);
  __syncwarp();
  float m = -INFINITY, l = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int j0 = 0; j0 < sees; j0 += 32) {
    const int j = j0 + lane;
    float s = -INFINITY;
    if (j < sees) {
      float dot = 0.0f;
      for (int d = 0; d < D; ++d) dot = fmaf(query[warp][d], value_of<E>(k[j * r.k_token_stride + d]), dot);
      s = dot * a.scale_log2;
    }
    float top = s;
#pragma unroll
    for (int w = 16; w; w >>= 1) top = fmaxf(top, __shfl_xor_sync(kAll, top, w));
    top = fmaxf(top, m);
    const float base = top == -INFINITY ? 0.0f : top, keep = exp2f(m - base), p = exp2f(s - base);
    l = l * keep + warp_sum(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] *= keep;
    for (int jj = 0; jj < min(32, sees - j0); ++jj) {
      const float pj = __shfl_sync(kAll, p, jj);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (lane + 32 * i < D) o[i] = fmaf(pj, value_of<E>(v[(j0 + jj) * r.v_token_stride + lane + 32 * i]), o[i]);
    }
    m = top;
  }
  E* out = static_cast<E*>(r.out) + row * r.out_token_stride + head * r.out_head_stride;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (lane + 32 * i < D) out[lane + 32 * i] = elem_of<E>(o[i] * inv);
}

}  // namespace

cudaError_t launch_attend_packed(const emelb_attend_packed_request& r, int sm_count, int* bad, int* status, cudaStream_t st) {
  PackedArgs a{r, r.heads / r.kv_heads, r.scale * 1.44269504088896340736f, bad};
  const dim3 grid((r.queries + 3) / 4, r.heads);
  if (r.type == EMELB_F16) attend_packed_rows_kernel<__half><<<grid, 128, 0, st>>>(a);
  else attend_packed_rows_kernel<__nv_bfloat16><<<grid, 128, 0, st>>>(a);
  return cudaGetLastError();
}

}  // namespace emelb
