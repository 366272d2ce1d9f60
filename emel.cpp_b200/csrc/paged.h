// Launch interface of the paged operators (internal; include/emelb_paged.h is the public one).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/emelb_paged.h"

namespace emelb {

// `bad`: raised to 1 by a kernel that met a length, page or slot out of range and left it alone
// `scratch`: requests + 1 ints
cudaError_t launch_kv_plan(const emelb_kv_plan_request& r, int* scratch, int sm_count, int* launches, int* bad, bool pdl, cudaStream_t st);
cudaError_t launch_kv_store(const emelb_kv_store_request& r, int sm_count, int* bad, bool pdl, cudaStream_t st);
cudaError_t launch_kv_load(const emelb_kv_load_request& r, int sm_count, int* bad, bool pdl, cudaStream_t st);

// scratch of emelb_kv_attend: two partial results a unit, its arrival counter (zero between launches)
struct KvAttendScratch {
  float* acc;
  uint64_t acc_floats;
  float* stats;
  uint64_t stats_floats;
  int* arrived;
  uint64_t arrived_ints;
};
cudaError_t launch_kv_attend(const emelb_kv_attend_request& r, const KvAttendScratch& s, int sm_count, int* bad, bool pdl, cudaStream_t st);

// `next`: two ints, zero between launches; `fold`: kPackedFoldFloats for each SM; `status`: raised to 1 when a bounded wait ran out
constexpr uint64_t kPackedFoldFloats = 2 * 131 * 128;
cudaError_t launch_attend_packed(const emelb_attend_packed_request& r, int* next, float* fold, int sm_count, int* bad, int* status, bool pdl, cudaStream_t st);

}  // namespace emelb
