// Varlen differential attention, forward.
//
// For every sequence, head h and query row i
//   out[i, h] = O_1 - lam_h O_2,  O_m = softmax_j(scale Q_m[i] . K_m[j]) V[j],
// Q_m = q[:, 2h + m], K_m = k[:, 2g + m], V = v[:, g], g = h / (heads / kv_heads).
// Sums and softmax statistics are f32.
#include "sc_diffattn_dev.cuh"

#include <algorithm>
#include <vector>

namespace sc {
namespace {

struct DaFwd {
  const void *q, *k, *v;
  int64_t qs, ks, vs;
  LamRef lam;
  void* out;
  float* lse;
  float* maps;
  int64_t nq;
  int heads, rep, causal;
  float scale_log2;
};

// One warp per (query row, head): 32 keys at a time, one per lane for the
// scores, then four value dims per lane.
template <typename T>
__global__ void __launch_bounds__(128) k_da_fwd_rows(const DaFwd p, const __grid_constant__ SeqPlan plan, int items) {
  const int item = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31, h = blockIdx.y;
  if (item >= items) return;
  const SeqRec& r = plan.at(plan.find(item));
  const int i = item - r.item0, limit = key_limit(r, i, p.causal), g = h / p.rep;
  const int64_t row = r.q0 + i;
  const T* q = static_cast<const T*>(p.q) + row * p.qs + 2 * h * kDaD;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, o[2][4] = {};
  for (int j0 = 0; j0 < limit; j0 += 32) {
    const bool in = j0 + lane < limit;
    const T* k = static_cast<const T*>(p.k) + (r.k0 + static_cast<int64_t>(min(j0 + lane, limit - 1))) * p.ks +
                 2 * g * kDaD;
    float w[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      float d = 0.f;
      for (int e = 0; e < kDaD; ++e) d = fmaf(Cvt<T>::to_f(q[s * kDaD + e]), Cvt<T>::to_f(k[s * kDaD + e]), d);
      d = in ? d * p.scale_log2 : -INFINITY;
      float mx = d;
#pragma unroll
      for (int x = 16; x > 0; x >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
      const float mn = fmaxf(m[s], mx), a = mn == -INFINITY ? 1.f : exp2f(m[s] - mn);
      w[s] = in ? exp2f(d - mn) : 0.f;
      float sum = w[s];
#pragma unroll
      for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
      l[s] = fmaf(l[s], a, sum);
      m[s] = mn;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[s][e] *= a;
    }
    for (int t = 0; t < min(32, limit - j0); ++t) {
      const float w0 = __shfl_sync(0xffffffffu, w[0], t), w1 = __shfl_sync(0xffffffffu, w[1], t);
      const T* v = static_cast<const T*>(p.v) + (r.k0 + static_cast<int64_t>(j0 + t)) * p.vs + g * kDaDv + lane * 4;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float f = Cvt<T>::to_f(v[e]);
        o[0][e] = fmaf(w0, f, o[0][e]);
        o[1][e] = fmaf(w1, f, o[1][e]);
      }
    }
  }
  const float lam = p.lam.get(h), i0 = l[0] > 0.f ? 1.f / l[0] : 0.f, i1 = l[1] > 0.f ? 1.f / l[1] : 0.f;
  const int64_t at = (row * p.heads + h) * kDaDv + lane * 4;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float b = o[1][e] * i1;
    static_cast<T*>(p.out)[at + e] = Cvt<T>::from_f(limit ? fmaf(-lam, b, o[0][e] * i0) : 0.f);
    if (p.maps) {
      p.maps[2 * (at - lane * 4) + lane * 4 + e] = limit ? o[0][e] * i0 : 0.f;
      p.maps[2 * (at - lane * 4) + kDaDv + lane * 4 + e] = limit ? b : 0.f;
    }
  }
  if (p.lse && lane < 2)
    p.lse[(static_cast<int64_t>(lane) * p.heads + h) * p.nq + row] = limit ? m[lane] + log2f(l[lane]) : INFINITY;
}

template <typename T>
sc_status run_forward(Handle* h, const DaArgs& a) {
  std::vector<SeqRec> recs;
  int32_t items = 0;
  for (int b = 0; b < a.batch; ++b) {
    if (a.cu_q[b + 1] == a.cu_q[b]) continue;
    recs.push_back(SeqRec{a.cu_q[b], a.cu_q[b + 1], a.cu_kv[b], a.cu_kv[b + 1], items, b});
    items += a.cu_q[b + 1] - a.cu_q[b];
  }
  SeqPlan plan;
  void* table = nullptr;
  const sc_status st = make_plan(h, recs, &plan, &table);
  if (st != SC_OK) return st;
  DaFwd p{a.q, a.k, a.v, a.qs, a.ks, a.vs, LamRef{a.lam, a.lam_count, a.lam_dtype, a.lam_value}, a.out, a.lse, a.maps,
          a.cu_q[a.batch], a.heads, a.heads / a.kv_heads, a.causal, a.scale * kLog2e};
  ++h->launches;
  k_da_fwd_rows<T><<<dim3((items + 3) / 4, a.heads), 128, 0, h->stream>>>(p, plan, items);
  const cudaError_t e = cudaGetLastError();
  dev_free(h, table);
  return e == cudaSuccess ? SC_OK : cuda_error(h, e, "differential attention launch");
}

}  // namespace

sc_status diff_attention(Handle* h, const DaArgs& a) {
  return a.dtype == SC_BF16 ? run_forward<__nv_bfloat16>(h, a) : run_forward<__half>(h, a);
}

}  // namespace sc
