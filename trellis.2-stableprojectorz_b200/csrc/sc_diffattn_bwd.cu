// Varlen differential attention, backward.
//
// With P_m the softmax maps, recomputed from the forward's log-sum-exps, and
// dP = dO V^T, delta_m = rowsum(dO o O_m):
//   dS_1 = P_1 o (dP - delta_1),  dS_2 = -lam P_2 o (dP - delta_2),
//   dV = (P_1 - lam P_2)^T dO,  dQ_m = scale dS_m K_m,  dK_m = scale dS_m^T Q_m,
//   dlam_h = -sum_rows delta_2,
// dK and dV summed over the heads that share a key / value head.  O_1 and O_2
// are kept by the forward in f32.  Every sum has one fixed order.
#include "sc_diffattn_dev.cuh"

#include <algorithm>
#include <vector>

namespace sc {
namespace {

struct DaBwd {
  const void *q, *k, *v;
  int64_t qs, ks, vs;
  LamRef lam;
  const float* maps;   // [nq][heads][2][128]
  const void* dout;
  const float* lse;    // [2][heads][nq]
  float* delta;        // [2][heads][nq]
  void *dq, *dk, *dv, *dlam;
  int64_t nq;
  int heads, kv_heads, rep, causal;
  float scale, scale_log2;
};

__device__ __forceinline__ float warp_add(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// delta_1, delta_2 of every (row, head), one warp each.
template <typename T>
__global__ void __launch_bounds__(256) k_da_delta(const DaBwd p) {
  const int64_t at = blockIdx.x * 8ll + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (at >= p.nq * p.heads) return;
  const int64_t row = at / p.heads;
  const int h = static_cast<int>(at % p.heads);
  const float4 o1 = reinterpret_cast<const float4*>(p.maps + at * 2 * kDaDv)[lane];
  const float4 o2 = reinterpret_cast<const float4*>(p.maps + at * 2 * kDaDv + kDaDv)[lane];
  const uint2 raw = reinterpret_cast<const uint2*>(static_cast<const T*>(p.dout) + at * kDaDv)[lane];
  const T* g = reinterpret_cast<const T*>(&raw);
  const float g0 = Cvt<T>::to_f(g[0]), g1 = Cvt<T>::to_f(g[1]), g2 = Cvt<T>::to_f(g[2]), g3 = Cvt<T>::to_f(g[3]);
  float d1 = fmaf(g0, o1.x, g1 * o1.y) + fmaf(g2, o1.z, g3 * o1.w);
  float d2 = fmaf(g0, o2.x, g1 * o2.y) + fmaf(g2, o2.z, g3 * o2.w);
  d1 = warp_add(d1);
  d2 = warp_add(d2);
  if (lane == 0) {
    p.delta[h * p.nq + row] = d1;
    p.delta[(p.heads + h) * p.nq + row] = d2;
  }
}

// dlam: one CTA per entry of lam sums -delta_2 over its heads' rows.
__global__ void __launch_bounds__(1024) k_da_dlam(const DaBwd p) {
  __shared__ float s[32];
  const int64_t n = p.lam.count == 1 ? p.nq * p.heads : p.nq;
  const float* d = p.delta + p.heads * p.nq + blockIdx.x * p.nq;
  float a = 0.f;
  for (int64_t i = threadIdx.x; i < n; i += 1024) a += d[i];
  a = warp_add(a);
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = a;
  __syncthreads();
  if (threadIdx.x < 32) {
    a = -warp_add(s[threadIdx.x]);
    if (threadIdx.x == 0) {
      if (p.lam.dtype == SC_F32) static_cast<float*>(p.dlam)[blockIdx.x] = a;
      else if (p.lam.dtype == SC_BF16) static_cast<__nv_bfloat16*>(p.dlam)[blockIdx.x] = __float2bfloat16_rn(a);
      else static_cast<__half*>(p.dlam)[blockIdx.x] = __float2half_rn(a);
    }
  }
}

// p_1, p_2, ds_1, ds_2 of one (query, key) pair, each product over one lane's dims.
template <typename T>
__device__ __forceinline__ void pair(const DaBwd& p, const T* q, const T* k, const T* v, const T* g, int h,
                                     int64_t row, float lam, float (&pm)[2], float (&ds)[2]) {
  float dp = 0.f;
  for (int e = 0; e < kDaDv; ++e) dp = fmaf(Cvt<T>::to_f(g[e]), Cvt<T>::to_f(v[e]), dp);
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    float d = 0.f;
    for (int e = 0; e < kDaD; ++e) d = fmaf(Cvt<T>::to_f(q[s * kDaD + e]), Cvt<T>::to_f(k[s * kDaD + e]), d);
    const int64_t at = (static_cast<int64_t>(s) * p.heads + h) * p.nq + row;
    pm[s] = exp2f(fmaf(d, p.scale_log2, -p.lse[at]));
    ds[s] = (s ? -lam : 1.f) * pm[s] * (dp - p.delta[at]);
  }
}

template <typename T>
__global__ void __launch_bounds__(128) k_da_dq_rows(const DaBwd p, const __grid_constant__ SeqPlan plan, int items) {
  const int item = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31, h = blockIdx.y;
  if (item >= items) return;
  const SeqRec& r = plan.at(plan.find(item));
  const int i = item - r.item0, limit = key_limit(r, i, p.causal), g = h / p.rep;
  const int64_t row = r.q0 + i;
  const T* q = static_cast<const T*>(p.q) + row * p.qs + 2 * h * kDaD;
  const T* go = static_cast<const T*>(p.dout) + (row * p.heads + h) * kDaDv;
  const float lam = p.lam.get(h);
  float acc[2][2] = {};
  for (int j0 = 0; j0 < limit; j0 += 32) {
    const int64_t j = r.k0 + static_cast<int64_t>(min(j0 + lane, limit - 1));
    float pm[2], ds[2];
    pair<T>(p, q, static_cast<const T*>(p.k) + j * p.ks + 2 * g * kDaD, static_cast<const T*>(p.v) + j * p.vs + g * kDaDv,
            go, h, row, lam, pm, ds);
    for (int t = 0; t < min(32, limit - j0); ++t) {
      const T* k = static_cast<const T*>(p.k) + (r.k0 + static_cast<int64_t>(j0 + t)) * p.ks + 2 * g * kDaD + 2 * lane;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const float d = __shfl_sync(0xffffffffu, ds[s], t);
#pragma unroll
        for (int e = 0; e < 2; ++e) acc[s][e] = fmaf(d, Cvt<T>::to_f(k[s * kDaD + e]), acc[s][e]);
      }
    }
  }
  T* dq = static_cast<T*>(p.dq) + (row * 2 * p.heads + 2 * h) * kDaD + 2 * lane;
#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int e = 0; e < 2; ++e) dq[s * kDaD + e] = Cvt<T>::from_f(acc[s][e] * p.scale);
}

template <typename T>
__global__ void __launch_bounds__(128) k_da_dkv_rows(const DaBwd p, const __grid_constant__ SeqPlan plan, int items) {
  const int item = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31, g = blockIdx.y;
  if (item >= items) return;
  const SeqRec& r = plan.at(plan.find(item));
  const int j = item - r.item0, lq = r.q1 - r.q0;
  const int64_t row = r.k0 + j;
  const T* k = static_cast<const T*>(p.k) + row * p.ks + 2 * g * kDaD;
  const T* v = static_cast<const T*>(p.v) + row * p.vs + g * kDaDv;
  const int first = p.causal ? min(lq, max(0, j - (r.k1 - r.k0) + lq)) : 0;  // first query that sees key j
  float ak[2][2] = {}, av[4] = {};
  for (int h = g * p.rep; h < (g + 1) * p.rep; ++h) {
    const float lam = p.lam.get(h);
    for (int i0 = first; i0 < lq; i0 += 32) {
      const int64_t i = r.q0 + static_cast<int64_t>(min(i0 + lane, lq - 1));
      float pm[2], ds[2];
      pair<T>(p, static_cast<const T*>(p.q) + i * p.qs + 2 * h * kDaD, k, v,
              static_cast<const T*>(p.dout) + (i * p.heads + h) * kDaDv, h, i, lam, pm, ds);
      const float pd = fmaf(-lam, pm[1], pm[0]);
      for (int t = 0; t < min(32, lq - i0); ++t) {
        const int64_t it = r.q0 + static_cast<int64_t>(i0 + t);
        const T* q = static_cast<const T*>(p.q) + it * p.qs + 2 * h * kDaD + 2 * lane;
        const T* go = static_cast<const T*>(p.dout) + (it * p.heads + h) * kDaDv + 4 * lane;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const float d = __shfl_sync(0xffffffffu, ds[s], t);
#pragma unroll
          for (int e = 0; e < 2; ++e) ak[s][e] = fmaf(d, Cvt<T>::to_f(q[s * kDaD + e]), ak[s][e]);
        }
        const float d = __shfl_sync(0xffffffffu, pd, t);
#pragma unroll
        for (int e = 0; e < 4; ++e) av[e] = fmaf(d, Cvt<T>::to_f(go[e]), av[e]);
      }
    }
  }
  if (p.dk) {
    T* dk = static_cast<T*>(p.dk) + (row * 2 * p.kv_heads + 2 * g) * kDaD + 2 * lane;
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int e = 0; e < 2; ++e) dk[s * kDaD + e] = Cvt<T>::from_f(ak[s][e] * p.scale);
  }
  if (p.dv) {
    T* dv = static_cast<T*>(p.dv) + (row * p.kv_heads + g) * kDaDv + 4 * lane;
#pragma unroll
    for (int e = 0; e < 4; ++e) dv[e] = Cvt<T>::from_f(av[e]);
  }
}

// Records of the sequences with rows on the chosen side, one item per row.
int32_t row_items(const DaArgs& a, bool keys, std::vector<SeqRec>* recs) {
  int32_t items = 0;
  const int32_t* cu = keys ? a.cu_kv : a.cu_q;
  for (int b = 0; b < a.batch; ++b) {
    if (cu[b + 1] == cu[b]) continue;
    recs->push_back(SeqRec{a.cu_q[b], a.cu_q[b + 1], a.cu_kv[b], a.cu_kv[b + 1], items, b});
    items += cu[b + 1] - cu[b];
  }
  return items;
}

template <typename T>
sc_status run_backward(Handle* h, const DaArgs& a) {
  const int64_t nq = a.cu_q[a.batch];
  DaBwd p{a.q, a.k, a.v, a.qs, a.ks, a.vs, LamRef{a.lam, a.lam_count, a.lam_dtype, a.lam_value}, a.maps, a.dout, a.lse,
          nullptr, a.dq, a.dk, a.dv, a.dlam, nq, a.heads, a.kv_heads, a.heads / a.kv_heads, a.causal, a.scale,
          a.scale * kLog2e};
  void* tables[2] = {nullptr, nullptr};
  cudaError_t e = dev_alloc(h, reinterpret_cast<void**>(&p.delta), sizeof(float) * 2 * a.heads * nq);
  if (e != cudaSuccess) return cuda_error(h, e, "differential attention workspace");
  sc_status st = SC_OK;
  if (nq > 0) {
    ++h->launches;
    k_da_delta<T><<<static_cast<unsigned>((nq * a.heads + 7) / 8), 256, 0, h->stream>>>(p);
  }
  if (a.dlam) {
    ++h->launches;
    k_da_dlam<<<a.lam_count, 1024, 0, h->stream>>>(p);
  }
  for (int keys = 0; keys < 2 && st == SC_OK; ++keys) {
    if (keys ? !a.dk && !a.dv : !a.dq) continue;
    std::vector<SeqRec> recs;
    SeqPlan plan;
    const int32_t items = row_items(a, keys != 0, &recs);
    if (items == 0) continue;
    st = make_plan(h, recs, &plan, &tables[keys]);
    if (st != SC_OK) break;
    ++h->launches;
    const dim3 grid((items + 3) / 4, keys ? a.kv_heads : a.heads);
    if (keys) k_da_dkv_rows<T><<<grid, 128, 0, h->stream>>>(p, plan, items);
    else k_da_dq_rows<T><<<grid, 128, 0, h->stream>>>(p, plan, items);
  }
  e = cudaGetLastError();
  dev_free(h, p.delta);
  dev_free(h, tables[0]);
  dev_free(h, tables[1]);
  if (st != SC_OK) return st;
  return e == cudaSuccess ? SC_OK : cuda_error(h, e, "differential attention backward launch");
}

}  // namespace

sc_status diff_attention_backward(Handle* h, const DaArgs& a) {
  return a.dtype == SC_BF16 ? run_backward<__nv_bfloat16>(h, a) : run_backward<__half>(h, a);
}

}  // namespace sc
