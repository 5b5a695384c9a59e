// Group norm over sparse sequences, channels last, with an optional SiLU.
//
// x [N, C] holds the rows of sequences one after the other; group g of a
// sequence is its rows times the C/G channels [g C/G, (g+1) C/G), with
//   mean, var over the group;  rstd = 1 / sqrt(var + eps);
//   z = (x - mean) rstd w_c + b_c;  y = z or z * sigmoid(z).
// Backward, with dz = dy or dy * sigma(z) (1 + z (1 - sigma(z))), per
// (sequence, channel) sums A = sum dz and B = sum dz xhat, n values a group:
//   dw = sum_seq B, db = sum_seq A,
//   dx = rstd (w dz - (sum_c w A) / n - xhat (sum_c w B) / n).
//
// Rows are cut into chunks, one CTA each.  The first kernel reduces a chunk
// to one (mean, M2) per group (backward: the sums); the second combines its
// sequence's chunks in a fixed order and writes its rows, last chunks first,
// so that it finds the most recently read rows in L2.  Every statistic is
// f32: per thread and channel a running mean and M2 (no difference of large
// sums), merged by counts.  The order of every sum is fixed by the sizes, so
// results repeat bit for bit.
#include "sc_common.cuh"
#include "sc_internal.h"
#include "sc_plan.cuh"

#include <algorithm>
#include <type_traits>
#include <vector>

namespace sc {
namespace {

constexpr int kGnThreads = 512;
constexpr int kGnWarps = kGnThreads / 32;

// V consecutive values of T as one aligned load.
template <int BYTES> struct Word;
template <> struct Word<16> { using type = uint4; };
template <> struct Word<8> { using type = uint2; };
template <> struct Word<4> { using type = uint32_t; };
template <> struct Word<2> { using type = uint16_t; };

template <typename T, int V>
struct Pack {
  using W = typename Word<V * static_cast<int>(sizeof(T))>::type;
  union { W w; T t[V]; };
  __device__ __forceinline__ Pack() {}
  __device__ __forceinline__ void load(const T* p) { w = *reinterpret_cast<const W*>(p); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<W*>(p) = w; }
};

struct GnParams {
  const void* x;
  int64_t xs;          // elements between rows of x
  const void* w;       // [C] or null (1)
  const void* b;       // [C] or null (0)
  int wdtype;
  void* y;             // forward: [N, C]
  const void* dy;      // backward: [N, C]
  void* dx;            // [N, C] or null
  void* dw;            // [C] or null
  void* db;            // [C] or null
  float* stats;        // [sequences][G][2] mean, rstd (forward: or null)
  float2* part;        // [G][items] forward (mean, M2); backward (sum w A, sum w B)
  float* chan;         // backward: [items][2][C] A, B of each chunk
  int c, groups, cg;   // cg = C / G
  int chunk;           // rows per item
  int items;
  float eps;
  int silu;
};

__device__ __forceinline__ float load_w(const void* p, int wdtype, int c, float none) {
  if (!p) return none;
  if (wdtype == SC_F32) return static_cast<const float*>(p)[c];
  if (wdtype == SC_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[c]);
  return __half2float(static_cast<const __half*>(p)[c]);
}
__device__ __forceinline__ void store_w(void* p, int wdtype, int c, float v) {
  if (wdtype == SC_F32) static_cast<float*>(p)[c] = v;
  else if (wdtype == SC_BF16) static_cast<__nv_bfloat16*>(p)[c] = __float2bfloat16_rn(v);
  else static_cast<__half*>(p)[c] = __float2half_rn(v);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// 1 / (1 + e^-z); e^-z overflowing gives 0
__device__ __forceinline__ float sigmoid_f(float z) { return __fdividef(1.f, 1.f + __expf(-z)); }

// The thread's place: column vector tx of TX (then tx + TX, ...; only when a
// row has more vectors than the block threads), row lane ty of TY.
struct Place {
  int tx, ty, TX, TY;
  bool live;
  __device__ __forceinline__ explicit Place(int nvec) {
    TX = min(nvec, kGnThreads);
    TY = kGnThreads / TX;
    tx = threadIdx.x % TX;
    ty = threadIdx.x / TX;
    live = ty < TY;
  }
};

struct Chunk {
  int64_t row0;
  int rows, seq, first_item, seq_items;
  int64_t seq_rows;
  __device__ __forceinline__ Chunk(const SeqPlan& plan, int item, int chunk) {
    const SeqRec& r = plan.at(plan.find(item));
    first_item = r.item0;
    seq = r.aux;
    seq_rows = r.q1 - r.q0;
    seq_items = static_cast<int>((seq_rows + chunk - 1) / chunk);
    row0 = r.q0 + static_cast<int64_t>(item - r.item0) * chunk;
    rows = static_cast<int>(min(static_cast<int64_t>(chunk), r.q1 - row0));
  }
};

template <typename T, int V>
__global__ void __launch_bounds__(kGnThreads)
    k_gn_stats(const GnParams p, const __grid_constant__ SeqPlan plan) {
  extern __shared__ float sm[];  // [TY][C] means, then [TY][C] M2
  const int nvec = p.c / V;
  const Place at(nvec);
  const Chunk ch(plan, blockIdx.x, p.chunk);
  float* s_mean = sm;
  float* s_m2 = sm + at.TY * p.c;
  const T* x = static_cast<const T*>(p.x);
  if (at.live) {
    for (int cv = at.tx; cv < nvec; cv += at.TX) {
      float mean[V], m2[V];
#pragma unroll
      for (int e = 0; e < V; ++e) mean[e] = m2[e] = 0.f;
      const T* px = x + ch.row0 * p.xs + cv * V;
      float n = 0.f;
      auto add = [&](const Pack<T, V>& v) {
        n += 1.f;
        const float inv = __fdividef(1.f, n);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float f = Cvt<T>::to_f(v.t[e]), d = f - mean[e];
          mean[e] = fmaf(d, inv, mean[e]);
          m2[e] = fmaf(d, f - mean[e], m2[e]);
        }
      };
      constexpr int U = 4;
      int r = at.ty;
      for (; r + (U - 1) * at.TY < ch.rows; r += U * at.TY) {
        Pack<T, V> v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u].load(px + static_cast<int64_t>(r + u * at.TY) * p.xs);
#pragma unroll
        for (int u = 0; u < U; ++u) add(v[u]);
      }
      for (; r < ch.rows; r += at.TY) {
        Pack<T, V> v;
        v.load(px + static_cast<int64_t>(r) * p.xs);
        add(v);
      }
#pragma unroll
      for (int e = 0; e < V; ++e) {
        s_mean[at.ty * p.c + cv * V + e] = mean[e];
        s_m2[at.ty * p.c + cv * V + e] = m2[e];
      }
    }
  }
  __syncthreads();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int g = warp; g < p.groups; g += kGnWarps) {
    const int total = min(at.TY, ch.rows) * p.cg;  // row lanes past the rows hold nothing
    float s = 0.f;
    for (int i = lane; i < total; i += 32) {
      const int ty = i / p.cg, c = g * p.cg + i % p.cg;
      s = fmaf(static_cast<float>((ch.rows - ty + at.TY - 1) / at.TY), s_mean[ty * p.c + c], s);
    }
    const float mean = warp_sum(s) / (static_cast<float>(ch.rows) * p.cg);
    float q = 0.f;
    for (int i = lane; i < total; i += 32) {
      const int ty = i / p.cg, c = g * p.cg + i % p.cg;
      const float d = s_mean[ty * p.c + c] - mean;
      q += fmaf(static_cast<float>((ch.rows - ty + at.TY - 1) / at.TY) * d, d, s_m2[ty * p.c + c]);
    }
    q = warp_sum(q);
    if (lane == 0) p.part[static_cast<int64_t>(g) * p.items + blockIdx.x] = make_float2(mean, q);
  }
}

// Mean and rstd of the chunk's sequence from its chunks' (mean, M2), into
// s_mean / s_rstd [G]; every CTA of a sequence computes the same values.
__device__ __forceinline__ void gn_combine(const GnParams& p, const Chunk& ch, float* s_mean, float* s_rstd) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const float n = static_cast<float>(ch.seq_rows) * p.cg;
  for (int g = warp; g < p.groups; g += kGnWarps) {
    const float2* part = p.part + static_cast<int64_t>(g) * p.items + ch.first_item;
    float s = 0.f;
    for (int i = lane; i < ch.seq_items; i += 32) {
      const float ni = static_cast<float>(min(static_cast<int64_t>(p.chunk),
                                              ch.seq_rows - static_cast<int64_t>(i) * p.chunk)) * p.cg;
      s = fmaf(ni, part[i].x, s);
    }
    const float mean = warp_sum(s) / n;
    float q = 0.f;
    for (int i = lane; i < ch.seq_items; i += 32) {
      const float ni = static_cast<float>(min(static_cast<int64_t>(p.chunk),
                                              ch.seq_rows - static_cast<int64_t>(i) * p.chunk)) * p.cg;
      const float2 v = part[i];
      q += fmaf(ni * (v.x - mean), v.x - mean, v.y);
    }
    const float rstd = rsqrtf(warp_sum(q) / n + p.eps);
    if (lane == 0) {
      s_mean[g] = mean;
      s_rstd[g] = rstd;
    }
  }
  __syncthreads();
}

template <typename T, int V>
__global__ void __launch_bounds__(kGnThreads)
    k_gn_apply(const GnParams p, const __grid_constant__ SeqPlan plan) {
  extern __shared__ float sm[];
  float* s_mean = sm;
  float* s_rstd = sm + p.groups;
  const int item = p.items - 1 - blockIdx.x;
  const Chunk ch(plan, item, p.chunk);
  gn_combine(p, ch, s_mean, s_rstd);
  if (p.stats && item == ch.first_item)
    for (int g = threadIdx.x; g < p.groups; g += kGnThreads) {
      float* st = p.stats + (static_cast<int64_t>(ch.seq) * p.groups + g) * 2;
      st[0] = s_mean[g];
      st[1] = s_rstd[g];
    }
  const int nvec = p.c / V;
  const Place at(nvec);
  if (!at.live) return;
  const T* x = static_cast<const T*>(p.x);
  T* y = static_cast<T*>(p.y);
  for (int cv = at.tx; cv < nvec; cv += at.TX) {
    float mean[V], a[V], b[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const int c = cv * V + e, g = c / p.cg;
      mean[e] = s_mean[g];
      a[e] = s_rstd[g] * load_w(p.w, p.wdtype, c, 1.f);
      b[e] = load_w(p.b, p.wdtype, c, 0.f);
    }
    const T* px = x + ch.row0 * p.xs + cv * V;
    T* py = y + ch.row0 * p.c + cv * V;
    auto put = [&](Pack<T, V>& v, int r) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        float z = fmaf(Cvt<T>::to_f(v.t[e]) - mean[e], a[e], b[e]);
        if (p.silu) z *= sigmoid_f(z);
        v.t[e] = Cvt<T>::from_f(z);
      }
      v.store(py + static_cast<int64_t>(r) * p.c);
    };
    constexpr int U = 4;
    int r = at.ty;
    for (; r + (U - 1) * at.TY < ch.rows; r += U * at.TY) {
      Pack<T, V> v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) v[u].load(px + static_cast<int64_t>(r + u * at.TY) * p.xs);
#pragma unroll
      for (int u = 0; u < U; ++u) put(v[u], r + u * at.TY);
    }
    for (; r < ch.rows; r += at.TY) {
      Pack<T, V> v;
      v.load(px + static_cast<int64_t>(r) * p.xs);
      put(v, r);
    }
  }
}

// dz of one value: x -> xhat, and the gradient through the activation.
__device__ __forceinline__ float gn_dz(float x, float dy, float mean, float rstd, float w, float b, int silu,
                                       float& xhat) {
  xhat = (x - mean) * rstd;
  if (!silu) return dy;
  const float z = fmaf(xhat, w, b), s = sigmoid_f(z);
  return dy * s * fmaf(z, 1.f - s, 1.f);
}

template <typename T, int V>
__global__ void __launch_bounds__(kGnThreads)
    k_gn_bwd_sums(const GnParams p, const __grid_constant__ SeqPlan plan) {
  extern __shared__ float sm[];  // [TY][C] A, then [TY][C] B
  const int nvec = p.c / V;
  const Place at(nvec);
  const Chunk ch(plan, blockIdx.x, p.chunk);
  float* s_a = sm;
  float* s_b = sm + at.TY * p.c;
  const T* x = static_cast<const T*>(p.x);
  const T* dy = static_cast<const T*>(p.dy);
  const float* stats = p.stats + static_cast<int64_t>(ch.seq) * p.groups * 2;
  if (at.live) {
    for (int cv = at.tx; cv < nvec; cv += at.TX) {
      float mean[V], rstd[V], w[V], b[V], sa[V], sb[V];
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const int c = cv * V + e, g = c / p.cg;
        mean[e] = stats[2 * g];
        rstd[e] = stats[2 * g + 1];
        w[e] = load_w(p.w, p.wdtype, c, 1.f);
        b[e] = load_w(p.b, p.wdtype, c, 0.f);
        sa[e] = sb[e] = 0.f;
      }
      const T* px = x + ch.row0 * p.xs + cv * V;
      const T* pd = dy + ch.row0 * p.c + cv * V;
      auto add = [&](const Pack<T, V>& v, const Pack<T, V>& d) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          float xhat;
          const float dz = gn_dz(Cvt<T>::to_f(v.t[e]), Cvt<T>::to_f(d.t[e]), mean[e], rstd[e], w[e], b[e], p.silu,
                                 xhat);
          sa[e] += dz;
          sb[e] = fmaf(dz, xhat, sb[e]);
        }
      };
      constexpr int U = 2;
      int r = at.ty;
      for (; r + (U - 1) * at.TY < ch.rows; r += U * at.TY) {
        Pack<T, V> v[U], d[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          v[u].load(px + static_cast<int64_t>(r + u * at.TY) * p.xs);
          d[u].load(pd + static_cast<int64_t>(r + u * at.TY) * p.c);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) add(v[u], d[u]);
      }
      for (; r < ch.rows; r += at.TY) {
        Pack<T, V> v, d;
        v.load(px + static_cast<int64_t>(r) * p.xs);
        d.load(pd + static_cast<int64_t>(r) * p.c);
        add(v, d);
      }
#pragma unroll
      for (int e = 0; e < V; ++e) {
        s_a[at.ty * p.c + cv * V + e] = sa[e];
        s_b[at.ty * p.c + cv * V + e] = sb[e];
      }
    }
  }
  __syncthreads();
  for (int c = threadIdx.x; c < p.c; c += kGnThreads) {
    float a = 0.f, b = 0.f;
    for (int ty = 0; ty < at.TY; ++ty) {
      a += s_a[ty * p.c + c];
      b += s_b[ty * p.c + c];
    }
    s_a[c] = a;  // only this thread reads column c
    s_b[c] = b;
    float* out = p.chan + static_cast<int64_t>(blockIdx.x) * 2 * p.c;
    out[c] = a;
    out[p.c + c] = b;
  }
  __syncthreads();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int g = warp; g < p.groups; g += kGnWarps) {
    float a = 0.f, b = 0.f;
    for (int i = lane; i < p.cg; i += 32) {
      const int c = g * p.cg + i;
      const float w = load_w(p.w, p.wdtype, c, 1.f);
      a = fmaf(w, s_a[c], a);
      b = fmaf(w, s_b[c], b);
    }
    a = warp_sum(a);
    b = warp_sum(b);
    if (lane == 0) p.part[static_cast<int64_t>(g) * p.items + blockIdx.x] = make_float2(a, b);
  }
}

constexpr int kGnChanBlock = 32;  // channels per dw / db CTA

// CTAs [0, items) write dx; the CTAs behind them sum dw and db over the items.
template <typename T, int V>
__global__ void __launch_bounds__(kGnThreads)
    k_gn_bwd_apply(const GnParams p, const __grid_constant__ SeqPlan plan, int dx_items) {
  extern __shared__ float sm[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (static_cast<int>(blockIdx.x) >= dx_items) {
    const int c = (blockIdx.x - dx_items) * kGnChanBlock + lane;
    float a = 0.f, b = 0.f;
    if (c < p.c)
      for (int i = warp; i < p.items; i += kGnWarps) {
        const float* in = p.chan + static_cast<int64_t>(i) * 2 * p.c;
        a += in[c];
        b += in[p.c + c];
      }
    sm[warp * 32 + lane] = a;
    sm[(kGnWarps + warp) * 32 + lane] = b;
    __syncthreads();
    if (warp == 0 && c < p.c) {
      a = b = 0.f;
      for (int k = 0; k < kGnWarps; ++k) {
        a += sm[k * 32 + lane];
        b += sm[(kGnWarps + k) * 32 + lane];
      }
      if (p.dw) store_w(p.dw, p.wdtype, c, b);
      if (p.db) store_w(p.db, p.wdtype, c, a);
    }
    return;
  }
  float* s_m1 = sm;
  float* s_m2 = sm + p.groups;
  const int item = dx_items - 1 - blockIdx.x;
  const Chunk ch(plan, item, p.chunk);
  const float inv_n = 1.f / (static_cast<float>(ch.seq_rows) * p.cg);
  for (int g = warp; g < p.groups; g += kGnWarps) {
    const float2* part = p.part + static_cast<int64_t>(g) * p.items + ch.first_item;
    float a = 0.f, b = 0.f;
    for (int i = lane; i < ch.seq_items; i += 32) {
      const float2 v = part[i];
      a += v.x;
      b += v.y;
    }
    a = warp_sum(a);
    b = warp_sum(b);
    if (lane == 0) {
      s_m1[g] = a * inv_n;
      s_m2[g] = b * inv_n;
    }
  }
  __syncthreads();
  const int nvec = p.c / V;
  const Place at(nvec);
  if (!at.live) return;
  const T* x = static_cast<const T*>(p.x);
  const T* dy = static_cast<const T*>(p.dy);
  T* dx = static_cast<T*>(p.dx);
  const float* stats = p.stats + static_cast<int64_t>(ch.seq) * p.groups * 2;
  for (int cv = at.tx; cv < nvec; cv += at.TX) {
    float mean[V], rstd[V], w[V], b[V], m1[V], m2[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const int c = cv * V + e, g = c / p.cg;
      mean[e] = stats[2 * g];
      rstd[e] = stats[2 * g + 1];
      w[e] = load_w(p.w, p.wdtype, c, 1.f);
      b[e] = load_w(p.b, p.wdtype, c, 0.f);
      m1[e] = s_m1[g];
      m2[e] = s_m2[g];
    }
    const T* px = x + ch.row0 * p.xs + cv * V;
    const T* pd = dy + ch.row0 * p.c + cv * V;
    T* po = dx + ch.row0 * p.c + cv * V;
    auto put = [&](const Pack<T, V>& v, const Pack<T, V>& d, int r) {
      Pack<T, V> o;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        float xhat;
        const float dz = gn_dz(Cvt<T>::to_f(v.t[e]), Cvt<T>::to_f(d.t[e]), mean[e], rstd[e], w[e], b[e], p.silu,
                               xhat);
        o.t[e] = Cvt<T>::from_f(rstd[e] * (fmaf(w[e], dz, -m1[e]) - xhat * m2[e]));
      }
      o.store(po + static_cast<int64_t>(r) * p.c);
    };
    constexpr int U = 2;
    int r = at.ty;
    for (; r + (U - 1) * at.TY < ch.rows; r += U * at.TY) {
      Pack<T, V> v[U], d[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        v[u].load(px + static_cast<int64_t>(r + u * at.TY) * p.xs);
        d[u].load(pd + static_cast<int64_t>(r + u * at.TY) * p.c);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) put(v[u], d[u], r + u * at.TY);
    }
    for (; r < ch.rows; r += at.TY) {
      Pack<T, V> v, d;
      v.load(px + static_cast<int64_t>(r) * p.xs);
      d.load(pd + static_cast<int64_t>(r) * p.c);
      put(v, d, r);
    }
  }
}

// Rows per chunk: about two CTAs' worth of chunks per SM, and at least four
// rows per row lane.
int gn_chunk(const Handle* h, int64_t rows, int nvec) {
  const int ty = kGnThreads / std::min(nvec, kGnThreads);
  const int64_t want = (rows + 2ll * h->num_sms - 1) / (2ll * h->num_sms);
  return static_cast<int>(std::max<int64_t>(want, 4ll * ty));
}

struct GnCall {
  SeqPlan plan;
  void* table = nullptr;
  int items = 0;
};

sc_status gn_plan(Handle* h, const int32_t* cu, int batch, int chunk, GnCall* call) {
  std::vector<SeqRec> recs;
  int64_t items = 0;
  for (int s = 0; s < batch; ++s) {
    const int64_t len = static_cast<int64_t>(cu[s + 1]) - cu[s];
    if (len == 0) continue;
    recs.push_back(SeqRec{cu[s], cu[s + 1], 0, 0, static_cast<int32_t>(items), s});
    items += (len + chunk - 1) / chunk;
  }
  call->items = static_cast<int>(items);
  return make_plan(h, recs, &call->plan, &call->table);
}

// Widest vector of T that divides the rows and their addresses.
template <typename T>
int gn_vec(int c, int64_t xs, const void* const* ptrs, int n) {
  for (int v = 16 / static_cast<int>(sizeof(T)); v > 1; v >>= 1) {
    bool ok = c % v == 0 && xs % v == 0;
    for (int i = 0; i < n; ++i) ok = ok && reinterpret_cast<uintptr_t>(ptrs[i]) % (v * sizeof(T)) == 0;
    if (ok) return v;
  }
  return 1;
}

size_t gn_sum_smem(int c, int nvec) {
  const int ty = kGnThreads / std::min(nvec, kGnThreads);
  return sizeof(float) * 2 * static_cast<size_t>(ty) * c;  // at most 32 KB: TY * C <= 512 * 8 or C <= 4096
}

template <typename T, int V>
sc_status gn_forward_v(Handle* h, GnParams p, const int32_t* cu, int batch) {
  p.chunk = gn_chunk(h, cu[batch], p.c / V);
  GnCall call;
  sc_status st = gn_plan(h, cu, batch, p.chunk, &call);
  if (st != SC_OK) return st;
  p.items = call.items;
  cudaError_t e = dev_alloc(h, reinterpret_cast<void**>(&p.part), sizeof(float2) * p.groups * p.items);
  if (e != cudaSuccess) {
    dev_free(h, call.table);
    return cuda_error(h, e, "group norm workspace");
  }
  h->launches += 2;
  k_gn_stats<T, V><<<p.items, kGnThreads, gn_sum_smem(p.c, p.c / V), h->stream>>>(p, call.plan);
  k_gn_apply<T, V><<<p.items, kGnThreads, sizeof(float) * 2 * p.groups, h->stream>>>(p, call.plan);
  e = cudaGetLastError();
  dev_free(h, p.part);
  dev_free(h, call.table);
  return e == cudaSuccess ? SC_OK : cuda_error(h, e, "group norm launch");
}

template <typename T, int V>
sc_status gn_backward_v(Handle* h, GnParams p, const int32_t* cu, int batch) {
  p.chunk = gn_chunk(h, cu[batch], p.c / V);
  GnCall call;
  sc_status st = gn_plan(h, cu, batch, p.chunk, &call);
  if (st != SC_OK) return st;
  p.items = call.items;
  const size_t part = (sizeof(float2) * p.groups * p.items + 255) / 256 * 256;
  char* ws = nullptr;
  cudaError_t e = dev_alloc(h, reinterpret_cast<void**>(&ws), part + sizeof(float) * 2 * p.c * p.items);
  if (e != cudaSuccess) {
    dev_free(h, call.table);
    return cuda_error(h, e, "group norm workspace");
  }
  p.part = reinterpret_cast<float2*>(ws);
  p.chan = reinterpret_cast<float*>(ws + part);
  const int dx_items = p.dx ? p.items : 0;
  const int chan_ctas = p.dw || p.db ? (p.c + kGnChanBlock - 1) / kGnChanBlock : 0;
  h->launches += 2;
  k_gn_bwd_sums<T, V><<<p.items, kGnThreads, gn_sum_smem(p.c, p.c / V), h->stream>>>(p, call.plan);
  const size_t smem = sizeof(float) * 2 * std::max(p.groups, kGnThreads);
  k_gn_bwd_apply<T, V><<<dx_items + chan_ctas, kGnThreads, smem, h->stream>>>(p, call.plan, dx_items);
  e = cudaGetLastError();
  dev_free(h, ws);
  dev_free(h, call.table);
  return e == cudaSuccess ? SC_OK : cuda_error(h, e, "group norm backward launch");
}

template <typename T>
sc_status gn_dispatch(Handle* h, const GnParams& p, const int32_t* cu, int batch, bool backward) {
  const void* ptrs[4] = {p.x, backward ? p.dy : p.y, backward ? p.dx : p.y, nullptr};
  const int v = gn_vec<T>(p.c, p.xs, ptrs, 3);
  switch (v) {
    case 8:
      if constexpr (sizeof(T) == 2) return backward ? gn_backward_v<T, 8>(h, p, cu, batch) : gn_forward_v<T, 8>(h, p, cu, batch);
      [[fallthrough]];
    case 4: return backward ? gn_backward_v<T, 4>(h, p, cu, batch) : gn_forward_v<T, 4>(h, p, cu, batch);
    case 2: return backward ? gn_backward_v<T, 2>(h, p, cu, batch) : gn_forward_v<T, 2>(h, p, cu, batch);
    default: return backward ? gn_backward_v<T, 1>(h, p, cu, batch) : gn_forward_v<T, 1>(h, p, cu, batch);
  }
}

}  // namespace

sc_status group_norm(Handle* h, const void* x, int64_t x_stride, const void* weight, const void* bias, void* y,
                     float* stats, const int32_t* cu, int batch, int c, int groups, float eps, int silu,
                     sc_dtype dtype, sc_dtype wdtype) {
  GnParams p{};
  p.x = x; p.xs = x_stride; p.w = weight; p.b = bias; p.wdtype = wdtype; p.y = y; p.stats = stats;
  p.c = c; p.groups = groups; p.cg = c / groups; p.eps = eps; p.silu = silu;
  if (dtype == SC_F32) return gn_dispatch<float>(h, p, cu, batch, false);
  if (dtype == SC_BF16) return gn_dispatch<__nv_bfloat16>(h, p, cu, batch, false);
  return gn_dispatch<__half>(h, p, cu, batch, false);
}

sc_status group_norm_backward(Handle* h, const void* x, int64_t x_stride, const void* dy, const void* weight,
                              const void* bias, const float* stats, void* dx, void* dweight, void* dbias,
                              const int32_t* cu, int batch, int c, int groups, int silu, sc_dtype dtype,
                              sc_dtype wdtype) {
  GnParams p{};
  p.x = x; p.xs = x_stride; p.dy = dy; p.w = weight; p.b = bias; p.wdtype = wdtype;
  p.stats = const_cast<float*>(stats); p.dx = dx; p.dw = dweight; p.db = dbias;
  p.c = c; p.groups = groups; p.cg = c / groups; p.silu = silu;
  if (dtype == SC_F32) return gn_dispatch<float>(h, p, cu, batch, true);
  if (dtype == SC_BF16) return gn_dispatch<__nv_bfloat16>(h, p, cu, batch, true);
  return gn_dispatch<__half>(h, p, cu, batch, true);
}

}  // namespace sc
