// Device helpers of the differential attention kernels.
#pragma once
#include "sc_common.cuh"
#include "sc_diffattn.h"
#include "sc_plan.cuh"

namespace sc {

constexpr float kLog2e = 1.4426950408889634f;

struct LamRef {
  const void* p;
  int count, dtype;
  float value;
  __device__ __forceinline__ float get(int head) const {
    if (!p) return value;
    const int i = count == 1 ? 0 : head;
    if (dtype == SC_F32) return static_cast<const float*>(p)[i];
    if (dtype == SC_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
    return __half2float(static_cast<const __half*>(p)[i]);
  }
};

// Keys that query i (of its sequence) sees: the first `limit` of them.
__device__ __forceinline__ int key_limit(const SeqRec& r, int i, int causal) {
  const int lk = r.k1 - r.k0;
  if (!causal) return lk;
  return max(0, min(lk, i + 1 + lk - (r.q1 - r.q0)));
}

}  // namespace sc
