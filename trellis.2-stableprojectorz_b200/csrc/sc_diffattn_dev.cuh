// Device helpers of the differential attention kernels.
#pragma once
#include <cuda.h>
#include "sc_attn_dev.cuh"
#include "sc_common.cuh"
#include "sc_diffattn.h"
#include "sc_plan.cuh"

namespace sc {

bool make_map_nd(CUtensorMap* m, bool bf16, const void* base, int rank, const uint64_t* dims, const uint64_t* strides,
                 const uint32_t* box);  // sc_conv_tc.cu

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

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const void* tmap, int32_t c0, int32_t c1, int32_t c2,
                                            int32_t c3, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(tmap)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar)
      : "memory");
}

// Descriptor of an MN-major operand in the 128-byte swizzle: 64-element atoms
// along M / N `lbo` bytes apart, groups of 8 K rows 1024 bytes apart.
__device__ __forceinline__ uint64_t smem_desc_mn(uint32_t addr, uint32_t lbo) {
  return (smem_desc(addr, 1024, 2) & ~(0x3FFFull << 16)) | (static_cast<uint64_t>((lbo >> 4) & 0x3FFFu) << 16);
}

}  // namespace sc
