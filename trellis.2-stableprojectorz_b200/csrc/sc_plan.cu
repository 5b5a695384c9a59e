// Device tables of the varlen operators' sequences (sc_plan.cuh).
#include "sc_plan.cuh"

#include <algorithm>

namespace sc {
namespace {

struct PlanChunk {
  int32_t n;
  SeqRec rec[kPlanInline];
};

__global__ void k_plan_write(const __grid_constant__ PlanChunk c, SeqRec* dst) {
  for (int i = threadIdx.x; i < c.n; i += blockDim.x) dst[i] = c.rec[i];
}

}  // namespace

sc_status make_plan(Handle* h, const std::vector<SeqRec>& recs, SeqPlan* plan, void** dev) {
  *dev = nullptr;
  plan->n = static_cast<int32_t>(recs.size());
  plan->ext = nullptr;
  if (recs.size() <= static_cast<size_t>(kPlanInline)) {
    std::copy(recs.begin(), recs.end(), plan->in);
    return SC_OK;
  }
  const cudaError_t e = dev_alloc(h, dev, recs.size() * sizeof(SeqRec));
  if (e != cudaSuccess) {
    *dev = nullptr;
    return cuda_error(h, e, "sequence table");
  }
  SeqRec* d = static_cast<SeqRec*>(*dev);
  for (size_t at = 0; at < recs.size(); at += kPlanInline) {
    PlanChunk c;
    c.n = static_cast<int32_t>(std::min<size_t>(kPlanInline, recs.size() - at));
    std::copy(recs.begin() + at, recs.begin() + at + c.n, c.rec);
    ++h->launches;
    k_plan_write<<<1, kPlanInline, 0, h->stream>>>(c, d + at);
  }
  const cudaError_t le = cudaGetLastError();
  if (le != cudaSuccess) return cuda_error(h, le, "sequence table");
  plan->ext = d;
  return SC_OK;
}

}  // namespace sc
