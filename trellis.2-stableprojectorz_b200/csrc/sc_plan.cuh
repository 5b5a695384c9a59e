// Sequence tables of the varlen operators (group norm, differential attention).
//
// A call's sequences are given by host offsets.  The kernels find their work
// from a small table, one record per sequence with work, sorted by first
// item; an item is a unit of work of that sequence (a chunk of rows, a query
// tile, ...), and a CTA finds its sequence by bisection.  Up to kPlanInline
// records travel in the kernel's parameters; longer tables are written to
// device memory by kernels that carry them in their parameters too, so a call
// never copies from pageable host memory and can be captured into a graph.
#pragma once
#include <cstdint>
#include <vector>
#include <cuda_runtime.h>
#include "sc_internal.h"

namespace sc {

struct SeqRec {
  int32_t q0, q1;    // rows (queries) of the sequence
  int32_t k0, k1;    // its key rows (attention)
  int32_t item0;     // first item
  int32_t aux;       // operator-specific
  int32_t part0;     // first row of its partial results (attention)
};

constexpr int kPlanInline = 96;  // 2688 bytes of a kernel's 4 KB of parameters

struct SeqPlan {
  int32_t n = 0;                 // records
  const SeqRec* ext = nullptr;   // device table when n > kPlanInline
  SeqRec in[kPlanInline];
  __device__ __forceinline__ const SeqRec& at(int i) const { return ext ? ext[i] : in[i]; }
  // The record whose items contain `item` (0 <= item < total).
  __device__ __forceinline__ int find(int item) const {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (at(mid).item0 <= item) lo = mid; else hi = mid - 1;
    }
    return lo;
  }
};

// Fills `plan` from host records (no record may have zero items).  *dev
// receives the device table, if one was needed; the caller frees it behind its
// last kernel, also after an error.
sc_status make_plan(Handle* h, const std::vector<SeqRec>& recs, SeqPlan* plan, void** dev);  // sc_plan.cu

}  // namespace sc
