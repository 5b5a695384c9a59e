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
// Bound: HBM (x read and y written; backward x and dy read, dx written), as long
// as the second pass over x finds part of it in L2.
//
// Rows are cut into chunks, one CTA each, two CTAs per SM.  The first kernel
// reduces a chunk to one (mean, M2) per group (backward: the sums); the second
// combines its sequence's chunks in a fixed order and writes its rows, last
// chunks first, so that it finds the most recently read rows in L2; it is
// launched early (programmatic dependent launch) and waits for the first.
// Short sequences take one kernel: a cluster of up to eight CTAs per sequence
// that exchanges the chunks' (mean, M2) through distributed shared memory.
// Every statistic is f32: per thread and channel a running mean and M2 (no
// difference of large sums), merged by counts.  The order of every sum is fixed
// by the sizes, so results repeat bit for bit.  The arithmetic runs on packed
// f32 pairs, and a vector whose channels share groups keeps their statistics
// once: 64 registers, so that two CTAs of 512 threads fit an SM.
#include <cooperative_groups.h>
#include "sc_attn_dev.cuh"
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

// Rows of a batch of loads (two are in flight, one while the other is used).
constexpr int kGnStatsBatch = 4, kGnApplyBatch = 2, kGnBwdBatch = 1;

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
  // last use of a line / a line nobody here reads again: first to leave L2, so
  // that the rows of the first pass stay for the second
  __device__ __forceinline__ void load_last(const T* p) { w = __ldcs(reinterpret_cast<const W*>(p)); }
  __device__ __forceinline__ void store(T* p) const { __stcs(reinterpret_cast<W*>(p), w); }
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
  int* err;
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

using F2 = unsigned long long;  // two f32

__device__ __forceinline__ F2 mul_f2(F2 a, F2 b) {
  F2 d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ F2 neg_f2(F2 a) { return a ^ 0x8000000080000000ull; }

// 1 / (1 + e^-z) of a pair, with one reciprocal for both: the special function
// unit is what this arithmetic waits for.  e^-z is cut at 2^60, so that the
// product of both denominators stays finite: sigmoid >= 2^-60, which below
// z = -41 puts silu(z) off by at most 2^-60 |z|.
__device__ __forceinline__ F2 sigmoid_f2(F2 z) {
  float a, b;
  f2_split(mul_f2(z, f2(-1.4426950408889634f, -1.4426950408889634f)), a, b);
  f2_split(add_f2(f2(ex2_ftz(fminf(a, 60.f)), ex2_ftz(fminf(b, 60.f))), f2(1.f, 1.f)), a, b);
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(a * b));
  return mul_f2(f2(r, r), f2(b, a));
}

// Pair i of a vector (the last of an odd vector twice) / a pair back into it.
template <typename T, int V>
__device__ __forceinline__ F2 get_pair(const Pack<T, V>& v, int i) {
  if constexpr (sizeof(T) == 4) {
    return f2(v.t[2 * i], v.t[V > 1 ? 2 * i + 1 : 0]);
  } else if constexpr (std::is_same_v<T, __nv_bfloat16> && V > 1) {
    const uint32_t w = reinterpret_cast<const uint32_t*>(&v.w)[i];
    return f2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  } else {
    return f2(Cvt<T>::to_f(v.t[2 * i]), Cvt<T>::to_f(v.t[V > 1 ? 2 * i + 1 : 0]));
  }
}
template <typename T, int V>
__device__ __forceinline__ void put_pair(Pack<T, V>& v, int i, F2 x) {
  float a, b;
  f2_split(x, a, b);
  if constexpr (sizeof(T) == 2 && V > 1) {
    reinterpret_cast<uint32_t*>(&v.w)[i] = pack2<T>(a, b);
  } else {
    v.t[2 * i] = Cvt<T>::from_f(a);
    if constexpr (V > 1) v.t[2 * i + 1] = Cvt<T>::from_f(b);
  }
}

// Statistics of the groups that a vector of V channels meets: GS consecutive
// channels share a group (GS even), or each channel has its own (GS = 1).
template <int V, int GS>
struct Span {
  static constexpr int NP = (V + 1) / 2;                 // pairs of the vector
  static constexpr int NR = GS > 1 ? V / GS : NP;        // pairs of statistics
  static __device__ __forceinline__ int of(int i) { return GS > 1 ? 2 * i / GS : i; }
  // s[group] of the vector's channels, times f
  static __device__ __forceinline__ void load(const float* s, int stride, int c0, int cg, F2 (&out)[NR]) {
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      const float a = s[(c0 + (GS > 1 ? r * GS : 2 * r)) / cg * stride];
      out[r] = f2(a, GS > 1 || V == 1 ? a : s[(c0 + 2 * r + 1) / cg * stride]);
    }
  }
};

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
  // rank's share of one sequence
  __device__ __forceinline__ Chunk(const SeqRec& r, int rank, int chunk)
      : row0(r.q0 + static_cast<int64_t>(rank) * chunk),
        rows(static_cast<int>(max(int64_t(0), min(static_cast<int64_t>(chunk), r.q1 - row0)))),
        seq(r.aux), first_item(0), seq_items(0), seq_rows(r.q1 - r.q0) {}
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

__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_release() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// The thread's rows of the chunk in batches of U, the loads of a batch ahead of
// the use of the one before: load(k, row) into slot k of 2 U, use(k, row).
template <int U, typename L, typename F>
__device__ __forceinline__ void for_rows(int rows, const Place& at, L&& load, F&& use) {
  const int step = U * at.TY;
  auto all = [&](int base, int r, auto&& f) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (r + u * at.TY < rows) f(base + u, r + u * at.TY);
  };
  all(0, at.ty, load);
  for (int r = at.ty; r < rows; r += 2 * step) {
    all(U, r + step, load);
    all(0, r, use);
    all(0, r + 2 * step, load);
    all(U, r + step, use);
  }
}

// The same rows through shared memory: blocks of 4 TY consecutive rows (at most
// 32 KB; of two arrays: 2 TY rows each) arrive by bulk copies in a ring of three,
// so the bytes in flight cost no registers: 96 KB a CTA.  Dense rows of 16-byte
// vectors only.  `last_first` walks the chunk's blocks from its end: the rows
// that the pass before read last are the ones still in L2.  use(pack of array 0,
// pack of array 1, row).
constexpr int kGnRing = 3, kGnRows = 4, kGnBlock = kGnRows * 8 * 1024, kGnRingSmem = kGnRing * kGnBlock + 16 * kGnRing + 128;
template <int ARRAYS, typename T, int V, typename F>
__device__ __forceinline__ void ring_rows(const GnParams& p, const Chunk& ch, const Place& at, float* sm, const void* a0,
                                          const void* a1, bool last_first, F&& use) {
  const uint32_t base = (smem_u32(sm) + 127u) & ~127u;
  uint8_t* ring = reinterpret_cast<uint8_t*>(sm) + (base - smem_u32(sm));
  const uint32_t full0 = base + kGnRing * kGnBlock, empty0 = full0 + 8 * kGnRing;
  const int row_bytes = p.c * static_cast<int>(sizeof(T)), per = kGnRows / ARRAYS * at.TY;
  const int blocks = (ch.rows + per - 1) / per;
  const char* src[2] = {static_cast<const char*>(a0) + ch.row0 * row_bytes,
                        static_cast<const char*>(a1) + ch.row0 * row_bytes};
  if (threadIdx.x == 0) {
    for (int i = 0; i < kGnRing; ++i) {
      mbar_init(full0 + 8 * i, 1);
      mbar_init(empty0 + 8 * i, kGnWarps);
    }
    fence_mbar_init();
  }
  __syncthreads();
  auto issue = [&](int k) {
    const int b = last_first ? blocks - 1 - k : k, s = k % kGnRing;
    const uint32_t bytes = static_cast<uint32_t>(min(per, ch.rows - b * per)) * row_bytes;
    mbar_arrive_expect_tx(full0 + 8 * s, ARRAYS * bytes);
    for (int i = 0; i < ARRAYS; ++i)
      bulk_load(base + s * kGnBlock + i * (kGnBlock / 2), src[i] + static_cast<int64_t>(b) * per * row_bytes, bytes,
                full0 + 8 * s);
  };
  int issued = min(blocks, kGnRing - 1);  // thread 0's
  if (threadIdx.x == 0)
    for (int k = 0; k < issued; ++k) issue(k);
  int s = 0, turn = 0, k = 0;
  for (; k < blocks; ++k) {
    if (threadIdx.x == 0 && issued < blocks && issued == k + kGnRing - 1) {
      // the slot of block k - 1, once every warp has left it; none is asked for after a wait that gave up
      if (k == 0 || mbar_wait(empty0 + 8 * ((k - 1) % kGnRing), ((k - 1) / kGnRing) & 1, p.err)) issue(issued++);
    }
    __syncwarp();
    // a warp goes on or leaves as one: its lanes meet again below
    if (!__all_sync(0xffffffffu, mbar_wait(full0 + 8 * s, turn, p.err))) break;
    const int b = last_first ? blocks - 1 - k : k, rows = min(per, ch.rows - b * per);
    if (at.live) {
#pragma unroll
      for (int u = 0; u < kGnRows / ARRAYS; ++u) {
        const int r = at.ty + u * at.TY;
        if (r < rows) {
          Pack<T, V> v, g;
          v.load(reinterpret_cast<const T*>(ring + s * kGnBlock + r * row_bytes) + at.tx * V);
          if (ARRAYS == 2) g.load(reinterpret_cast<const T*>(ring + s * kGnBlock + kGnBlock / 2 + r * row_bytes) + at.tx * V);
          use(v, g, b * per + r);
        }
      }
    }
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(empty0 + 8 * s);
    if (++s == kGnRing) s = 0, turn ^= 1;
  }
  // after a wait that gave up: the copies end before sm is used again
  if (threadIdx.x == 0)
    for (; k < issued; ++k) mbar_wait(full0 + 8 * (k % kGnRing), (k / kGnRing) & 1, p.err);
  __syncthreads();  // sm may be used again
}

// (mean, M2) of every group of the chunk, to dst[g * stride].  sm: [TY][C]
// means, then [TY][C] M2.
template <typename T, int V, bool RING = false>
__device__ __forceinline__ void gn_chunk_stats(const GnParams& p, const Chunk& ch, float* sm, float2* dst,
                                               int64_t stride) {
  constexpr int NP = (V + 1) / 2;
  const int nvec = p.c / V;
  const Place at(nvec);
  float* s_mean = sm;
  float* s_m2 = sm + at.TY * p.c;
  const T* x = static_cast<const T*>(p.x);
  if (at.live || RING) {  // the ring's barriers want every thread
    for (int cv = RING ? min(at.tx, nvec - 1) : at.tx; cv < nvec; cv += RING ? nvec : at.TX) {
      F2 nmean[NP], m2[NP];  // the running means, negated
#pragma unroll
      for (int i = 0; i < NP; ++i) nmean[i] = m2[i] = 0ull;
      const T* px = x + ch.row0 * p.xs + cv * V;
      float n = 0.f;
      auto add = [&](const Pack<T, V>& v) {
        n += 1.f;
        const float ninv = __fdividef(-1.f, n);
        const F2 ninv2 = f2(ninv, ninv);
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          const F2 f = get_pair<T, V>(v, i), d = add_f2(f, nmean[i]);
          nmean[i] = fma_f2(d, ninv2, nmean[i]);
          m2[i] = fma_f2(d, add_f2(f, nmean[i]), m2[i]);
        }
      };
      if constexpr (RING) {
        ring_rows<1, T, V>(p, ch, at, sm, p.x, nullptr, false,
                           [&](const Pack<T, V>& v, const Pack<T, V>&, int) { add(v); });
      } else {
        Pack<T, V> v[2 * kGnStatsBatch];
        for_rows<kGnStatsBatch>(
            ch.rows, at, [&](int u, int r) { v[u].load(px + static_cast<int64_t>(r) * p.xs); },
            [&](int u, int) { add(v[u]); });
      }
      if (at.live)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        float a, b;
        f2_split(nmean[e / 2], a, b);
        s_mean[at.ty * p.c + cv * V + e] = e & 1 ? -b : -a;
        f2_split(m2[e / 2], a, b);
        s_m2[at.ty * p.c + cv * V + e] = e & 1 ? b : a;
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
    if (lane == 0) dst[g * stride] = make_float2(mean, q);
  }
}

// y of the chunk's rows from s_mean / s_rstd [G].
template <typename T, int V, int GS, bool RING = false>
__device__ __forceinline__ void gn_chunk_apply(const GnParams& p, const Chunk& ch, const float* s_mean,
                                               const float* s_rstd, float* ring = nullptr) {
  using S = Span<V, GS>;
  const int nvec = p.c / V;
  const Place at(nvec);
  if (!at.live && !RING) return;
  const T* x = static_cast<const T*>(p.x);
  T* y = static_cast<T*>(p.y);
  for (int cv = RING ? min(at.tx, nvec - 1) : at.tx; cv < nvec; cv += RING ? nvec : at.TX) {
    F2 nmean[S::NR], a[S::NP], b[S::NP];
    S::load(s_mean, 1, cv * V, p.cg, nmean);
#pragma unroll
    for (int r = 0; r < S::NR; ++r) nmean[r] = neg_f2(nmean[r]);
    {
      F2 rstd[S::NR];
      S::load(s_rstd, 1, cv * V, p.cg, rstd);
#pragma unroll
      for (int i = 0; i < S::NP; ++i) {
        const int c = cv * V + 2 * i, d = V > 1 ? c + 1 : c;
        a[i] = mul_f2(rstd[S::of(i)], f2(load_w(p.w, p.wdtype, c, 1.f), load_w(p.w, p.wdtype, d, 1.f)));
        b[i] = f2(load_w(p.b, p.wdtype, c, 0.f), load_w(p.b, p.wdtype, d, 0.f));
      }
    }
    const T* px = x + ch.row0 * p.xs + cv * V;
    T* py = y + ch.row0 * p.c + cv * V;
    auto put = [&](const Pack<T, V>& v, int r) {
      Pack<T, V> o;
#pragma unroll
      for (int i = 0; i < S::NP; ++i) {
        F2 z = fma_f2(add_f2(get_pair<T, V>(v, i), nmean[S::of(i)]), a[i], b[i]);
        if (p.silu) z = mul_f2(z, sigmoid_f2(z));
        put_pair<T, V>(o, i, z);
      }
      o.store(py + static_cast<int64_t>(r) * p.c);
    };
    if constexpr (RING) {
      ring_rows<1, T, V>(p, ch, at, ring, p.x, nullptr, true,
                         [&](const Pack<T, V>& v, const Pack<T, V>&, int r) { put(v, r); });
    } else {
      Pack<T, V> v[2 * kGnApplyBatch];
      for_rows<kGnApplyBatch>(
          ch.rows, at, [&](int u, int r) { v[u].load_last(px + static_cast<int64_t>(r) * p.xs); },
          [&](int u, int r) { put(v[u], r); });
    }
  }
}

template <typename T, int V, bool RING>
__global__ void __launch_bounds__(kGnThreads, 2)
    k_gn_stats(const GnParams p, const __grid_constant__ SeqPlan plan) {
  extern __shared__ float sm[];
  grid_release();
  const Chunk ch(plan, blockIdx.x, p.chunk);
  gn_chunk_stats<T, V, RING>(p, ch, sm, p.part + blockIdx.x, p.items);
}

// Mean and rstd of every group of a sequence from its chunks' (mean, M2):
// part(i, g) for chunk i of `chunks`, chunk_rows rows each but the last.
template <typename P>
__device__ __forceinline__ void gn_combine(const GnParams& p, int64_t rows, int chunks, int64_t chunk_rows, P&& part,
                                           float* s_mean, float* s_rstd) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const float n = static_cast<float>(rows) * p.cg;
  for (int g = warp; g < p.groups; g += kGnWarps) {
    float s = 0.f;
    for (int i = lane; i < chunks; i += 32)
      s = fmaf(static_cast<float>(max(int64_t(0), min(chunk_rows, rows - i * chunk_rows))) * p.cg, part(i, g).x, s);
    const float mean = warp_sum(s) / n;
    float q = 0.f;
    for (int i = lane; i < chunks; i += 32) {
      const float ni = static_cast<float>(max(int64_t(0), min(chunk_rows, rows - i * chunk_rows))) * p.cg;
      const float2 v = part(i, g);
      q += fmaf(ni * (v.x - mean), v.x - mean, v.y);
    }
    const float rstd = rsqrtf(warp_sum(q) / n + p.eps);
    if (lane == 0) {
      s_mean[g] = mean;
      s_rstd[g] = rstd;
    }
  }
}

__device__ __forceinline__ void gn_keep_stats(const GnParams& p, int seq, const float* s_mean, const float* s_rstd) {
  for (int g = threadIdx.x; g < p.groups; g += kGnThreads) {
    float* st = p.stats + (static_cast<int64_t>(seq) * p.groups + g) * 2;
    st[0] = s_mean[g];
    st[1] = s_rstd[g];
  }
}

template <typename T, int V, int GS, bool RING>
__global__ void __launch_bounds__(kGnThreads, 2)
    k_gn_apply(const GnParams p, const __grid_constant__ SeqPlan plan) {
  extern __shared__ float sm[];
  float* s_mean = sm;
  float* s_rstd = sm + p.groups;
  const int item = p.items - 1 - blockIdx.x;
  const Chunk ch(plan, item, p.chunk);
  grid_wait();
  gn_combine(p, ch.seq_rows, ch.seq_items, p.chunk,
             [&](int i, int g) { return p.part[static_cast<int64_t>(g) * p.items + ch.first_item + i]; }, s_mean, s_rstd);
  __syncthreads();
  if (p.stats && item == ch.first_item) gn_keep_stats(p, ch.seq, s_mean, s_rstd);
  gn_chunk_apply<T, V, GS, RING>(p, ch, s_mean, s_rstd, s_rstd + p.groups);
}

// One cluster per sequence (records: one item each); rank r takes the rows
// [r chunk, (r + 1) chunk) of it.
template <typename T, int V, int GS>
__global__ void __launch_bounds__(kGnThreads, 2)
    k_gn_cluster(const GnParams p, const __grid_constant__ SeqPlan plan, int ranks) {
  extern __shared__ float sm[];
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = static_cast<int>(cluster.block_rank());
  const SeqRec& rec = plan.at(blockIdx.x / ranks);
  const int64_t rows = rec.q1 - rec.q0, chunk_rows = (rows + ranks - 1) / ranks;
  Chunk ch(rec, rank, static_cast<int>(chunk_rows));
  float2* s_part = reinterpret_cast<float2*>(sm);
  float* s_mean = sm + 2 * p.groups;
  float* s_rstd = s_mean + p.groups;
  if (ch.rows > 0) gn_chunk_stats<T, V>(p, ch, s_rstd + p.groups, s_part, 1);
  else for (int g = threadIdx.x; g < p.groups; g += kGnThreads) s_part[g] = make_float2(0.f, 0.f);
  cluster.sync();
  gn_combine(p, rows, ranks, chunk_rows, [&](int i, int g) { return cluster.map_shared_rank(s_part, i)[g]; }, s_mean,
             s_rstd);
  cluster.sync();  // every rank has read the others' before any leaves
  if (p.stats && rank == 0) gn_keep_stats(p, rec.aux, s_mean, s_rstd);
  if (ch.rows > 0) gn_chunk_apply<T, V, GS>(p, ch, s_mean, s_rstd);
}

// dz of a pair: x -> xhat, and the gradient through the activation.
__device__ __forceinline__ F2 gn_dz(F2 x, F2 dy, F2 nmean, F2 rstd, F2 w, F2 b, int silu, F2& xhat) {
  xhat = mul_f2(add_f2(x, nmean), rstd);
  if (!silu) return dy;
  const F2 one = f2(1.f, 1.f), z = fma_f2(xhat, w, b), s = sigmoid_f2(z);
  return mul_f2(mul_f2(dy, s), fma_f2(z, fma_f2(s, f2(-1.f, -1.f), one), one));
}

template <typename T, int V, int GS, bool RING>
__global__ void __launch_bounds__(kGnThreads, 2)
    k_gn_bwd_sums(const GnParams p, const __grid_constant__ SeqPlan plan) {
  extern __shared__ float sm[];  // [TY][C] A, then [TY][C] B
  using S = Span<V, GS>;
  grid_release();
  const int nvec = p.c / V;
  const Place at(nvec);
  const Chunk ch(plan, blockIdx.x, p.chunk);
  float* s_a = sm;
  float* s_b = sm + at.TY * p.c;
  const T* x = static_cast<const T*>(p.x);
  const T* dy = static_cast<const T*>(p.dy);
  const float* stats = p.stats + static_cast<int64_t>(ch.seq) * p.groups * 2;
  if (at.live || RING) {
    for (int cv = RING ? min(at.tx, nvec - 1) : at.tx; cv < nvec; cv += RING ? nvec : at.TX) {
      F2 nmean[S::NR], rstd[S::NR], w[S::NP], b[S::NP], sa[S::NP], sb[S::NP];
      S::load(stats, 2, cv * V, p.cg, nmean);
#pragma unroll
    for (int r = 0; r < S::NR; ++r) nmean[r] = neg_f2(nmean[r]);
      S::load(stats + 1, 2, cv * V, p.cg, rstd);
#pragma unroll
      for (int i = 0; i < S::NP; ++i) {
        const int c = cv * V + 2 * i, d = V > 1 ? c + 1 : c;
        w[i] = f2(load_w(p.w, p.wdtype, c, 1.f), load_w(p.w, p.wdtype, d, 1.f));
        b[i] = f2(load_w(p.b, p.wdtype, c, 0.f), load_w(p.b, p.wdtype, d, 0.f));
        sa[i] = sb[i] = 0ull;
      }
      const T* px = x + ch.row0 * p.xs + cv * V;
      const T* pd = dy + ch.row0 * p.c + cv * V;
      auto add = [&](const Pack<T, V>& v, const Pack<T, V>& g) {
#pragma unroll
        for (int i = 0; i < S::NP; ++i) {
          F2 xhat;
          const F2 dz = gn_dz(get_pair<T, V>(v, i), get_pair<T, V>(g, i), nmean[S::of(i)], rstd[S::of(i)], w[i], b[i],
                              p.silu, xhat);
          sa[i] = add_f2(sa[i], dz);
          sb[i] = fma_f2(dz, xhat, sb[i]);
        }
      };
      if constexpr (RING) {
        ring_rows<2, T, V>(p, ch, at, sm, p.x, p.dy, false,
                           [&](const Pack<T, V>& v, const Pack<T, V>& g, int) { add(v, g); });
      } else {
        Pack<T, V> v[2 * kGnBwdBatch], g[2 * kGnBwdBatch];
        for_rows<kGnBwdBatch>(
            ch.rows, at,
            [&](int u, int r) {
              v[u].load(px + static_cast<int64_t>(r) * p.xs);
              g[u].load(pd + static_cast<int64_t>(r) * p.c);
            },
            [&](int u, int) { add(v[u], g[u]); });
      }
      if (at.live)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        float lo, hi;
        f2_split(sa[e / 2], lo, hi);
        s_a[at.ty * p.c + cv * V + e] = e & 1 ? hi : lo;
        f2_split(sb[e / 2], lo, hi);
        s_b[at.ty * p.c + cv * V + e] = e & 1 ? hi : lo;
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

// CTAs [0, chan_ctas) sum dw and db over the items; the others write dx.
template <typename T, int V, int GS, bool RING>
__global__ void __launch_bounds__(kGnThreads, 2)
    k_gn_bwd_apply(const GnParams p, const __grid_constant__ SeqPlan plan, int chan_ctas) {
  extern __shared__ float sm[];
  using S = Span<V, GS>;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  grid_wait();
  if (static_cast<int>(blockIdx.x) < chan_ctas) {
    const int c = blockIdx.x * kGnChanBlock + lane;
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
  const int item = p.items - 1 - (blockIdx.x - chan_ctas);
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
      s_m1[g] = -a * inv_n;
      s_m2[g] = -b * inv_n;
    }
  }
  __syncthreads();
  const int nvec = p.c / V;
  const Place at(nvec);
  if (!at.live && !RING) return;
  const T* x = static_cast<const T*>(p.x);
  const T* dy = static_cast<const T*>(p.dy);
  T* dx = static_cast<T*>(p.dx);
  const float* stats = p.stats + static_cast<int64_t>(ch.seq) * p.groups * 2;
  for (int cv = RING ? min(at.tx, nvec - 1) : at.tx; cv < nvec; cv += RING ? nvec : at.TX) {
    F2 nmean[S::NR], rstd[S::NR], m1[S::NR], m2[S::NR], w[S::NP], b[S::NP];
    S::load(stats, 2, cv * V, p.cg, nmean);
#pragma unroll
    for (int r = 0; r < S::NR; ++r) nmean[r] = neg_f2(nmean[r]);
    S::load(stats + 1, 2, cv * V, p.cg, rstd);
    S::load(s_m1, 1, cv * V, p.cg, m1);
    S::load(s_m2, 1, cv * V, p.cg, m2);
#pragma unroll
    for (int i = 0; i < S::NP; ++i) {
      const int c = cv * V + 2 * i, d = V > 1 ? c + 1 : c;
      w[i] = f2(load_w(p.w, p.wdtype, c, 1.f), load_w(p.w, p.wdtype, d, 1.f));
      b[i] = f2(load_w(p.b, p.wdtype, c, 0.f), load_w(p.b, p.wdtype, d, 0.f));
    }
    const T* px = x + ch.row0 * p.xs + cv * V;
    const T* pd = dy + ch.row0 * p.c + cv * V;
    T* po = dx + ch.row0 * p.c + cv * V;
    auto put = [&](const Pack<T, V>& v, const Pack<T, V>& g, int r) {
      Pack<T, V> o;
#pragma unroll
      for (int i = 0; i < S::NP; ++i) {
        F2 xhat;
        const int k = S::of(i);
        const F2 dz = gn_dz(get_pair<T, V>(v, i), get_pair<T, V>(g, i), nmean[k], rstd[k], w[i], b[i], p.silu, xhat);
        put_pair<T, V>(o, i, mul_f2(rstd[k], fma_f2(xhat, m2[k], fma_f2(w[i], dz, m1[k]))));
      }
      o.store(po + static_cast<int64_t>(r) * p.c);
    };
    if constexpr (RING) {
      ring_rows<2, T, V>(p, ch, at, s_m2 + p.groups, p.x, p.dy, true, put);
    } else {
      Pack<T, V> v[2 * kGnBwdBatch], g[2 * kGnBwdBatch];
      for_rows<kGnBwdBatch>(
          ch.rows, at,
          [&](int u, int r) {
            v[u].load_last(px + static_cast<int64_t>(r) * p.xs);
            g[u].load_last(pd + static_cast<int64_t>(r) * p.c);
          },
          [&](int u, int r) { put(v[u], g[u], r); });
    }
  }
}

// Rows per chunk: two CTAs per SM in one wave (a chunk more would be a second
// one), and at least four rows per row lane.
int gn_chunk(const Handle* h, const int32_t* cu, int batch, int nvec) {
  const int ty = kGnThreads / std::min(nvec, kGnThreads);
  const int64_t slots = 2ll * h->num_sms;
  int64_t chunk = std::max<int64_t>((cu[batch] + slots - 1) / slots, 4ll * ty);
  for (int tries = 0; tries < 16; ++tries, chunk += (chunk + 63) / 64) {
    int64_t items = 0, seqs = 0;
    for (int s = 0; s < batch; ++s) {
      const int64_t len = static_cast<int64_t>(cu[s + 1]) - cu[s];
      items += (len + chunk - 1) / chunk;
      seqs += len > 0;
    }
    if (items <= slots || seqs > slots / 2) break;
  }
  return static_cast<int>(std::min<int64_t>(chunk, 0x7fffffff));
}

struct GnCall {
  SeqPlan plan;
  DevBuf table, ws;
  int items = 0;
  explicit GnCall(Handle* h) : table(h), ws(h) {}
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
  return make_plan(h, recs, &call->plan, &call->table.p);
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

// Launches `kernel` so that it may start before the stream's kernels before it
// end; it waits for them itself (grid_wait).  Or with clusters of `ranks`.
template <typename... P, typename... A>
cudaError_t launch_ex(Handle* h, void (*kernel)(P...), int grid, size_t smem, int ranks, A... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(kGnThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = h->stream;
  cudaLaunchAttribute at[1];
  if (ranks > 0) {
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = static_cast<unsigned>(ranks);
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  } else {
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
  }
  cfg.attrs = at;
  cfg.numAttrs = 1;
  ++h->launches;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// Whether the rows go through the ring of bulk copies: dense, in 16-byte
// vectors, no row longer than half a block, and blocks enough per chunk.
template <typename T, int V>
bool gn_ring(const GnParams& p) {
  const int nvec = p.c / V;
  return V * sizeof(T) == 16 && p.xs == p.c && nvec <= kGnThreads && p.chunk >= 8 * (kGnThreads / nvec);
}

// The limit belongs to the kernel, not to the handle: always the largest that a
// launch may need, so that calls of other threads do not lower it in between.
template <typename... P>
cudaError_t gn_allow_smem(void (*kernel)(P...), size_t bytes) {
  return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
}

// Sequences up to this many bytes per CTA of a cluster of eight take one kernel.
constexpr int64_t kGnClusterBytes = 128 * 1024;
constexpr int kGnClusterMax = 8;
constexpr size_t kGnClusterSmem = 32 * 1024 + 4 * sizeof(float) * 4096;  // sums, then four floats a group

template <typename T, int V, int GS>
sc_status gn_forward_v(Handle* h, GnParams p, const int32_t* cu, int batch) {
  int64_t longest = 0;
  for (int s = 0; s < batch; ++s) longest = std::max<int64_t>(longest, static_cast<int64_t>(cu[s + 1]) - cu[s]);
  const int64_t bytes = longest * p.c * static_cast<int64_t>(sizeof(T));
  const int ty = kGnThreads / std::min(p.c / V, kGnThreads);
  GnCall call(h);
  cudaError_t e;
  if (bytes <= kGnClusterMax * kGnClusterBytes) {
    std::vector<SeqRec> recs;
    for (int s = 0; s < batch; ++s)
      if (cu[s + 1] > cu[s])
        recs.push_back(SeqRec{cu[s], cu[s + 1], 0, 0, static_cast<int32_t>(recs.size()), s});
    sc_status st = make_plan(h, recs, &call.plan, &call.table.p);
    if (st != SC_OK) return st;
    // a rank for every eight rows of a row lane
    int ranks = 1;
    while (ranks < kGnClusterMax && longest > 8ll * ty * ranks) ranks *= 2;
    const size_t smem = gn_sum_smem(p.c, p.c / V) + sizeof(float) * 4 * p.groups;
    e = smem > 48 * 1024 ? gn_allow_smem(k_gn_cluster<T, V, GS>, kGnClusterSmem) : cudaSuccess;
    if (e == cudaSuccess)
      e = launch_ex(h, k_gn_cluster<T, V, GS>, static_cast<int>(recs.size()) * ranks, smem, ranks, p, call.plan, ranks);
  } else {
    p.chunk = gn_chunk(h, cu, batch, p.c / V);
    sc_status st = gn_plan(h, cu, batch, p.chunk, &call);
    if (st != SC_OK) return st;
    p.items = call.items;
    e = dev_alloc(h, &call.ws.p, sizeof(float2) * p.groups * p.items);
    if (e != cudaSuccess) return cuda_error(h, e, "group norm workspace");
    p.part = static_cast<float2*>(call.ws.p);
    const size_t sums = gn_sum_smem(p.c, p.c / V), norms = sizeof(float) * 2 * p.groups;
    ++h->launches;
    if (gn_ring<T, V>(p)) {
      if constexpr (V * sizeof(T) == 16) {
        e = gn_allow_smem(k_gn_stats<T, V, true>, kGnRingSmem);
        if (e == cudaSuccess) e = gn_allow_smem(k_gn_apply<T, V, GS, true>, kGnRingSmem + 2 * sizeof(float) * 4096);
        if (e == cudaSuccess) {
          k_gn_stats<T, V, true><<<p.items, kGnThreads, kGnRingSmem, h->stream>>>(p, call.plan);
          e = launch_ex(h, k_gn_apply<T, V, GS, true>, p.items, kGnRingSmem + norms, 0, p, call.plan);
        }
      }
    } else {
      k_gn_stats<T, V, false><<<p.items, kGnThreads, sums, h->stream>>>(p, call.plan);
      e = launch_ex(h, k_gn_apply<T, V, GS, false>, p.items, norms, 0, p, call.plan);
    }
  }
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? SC_OK : cuda_error(h, e, "group norm launch");
}

template <typename T, int V, int GS>
sc_status gn_backward_v(Handle* h, GnParams p, const int32_t* cu, int batch) {
  p.chunk = gn_chunk(h, cu, batch, p.c / V);
  GnCall call(h);
  sc_status st = gn_plan(h, cu, batch, p.chunk, &call);
  if (st != SC_OK) return st;
  p.items = call.items;
  const size_t part = (sizeof(float2) * p.groups * p.items + 255) / 256 * 256;
  cudaError_t e = dev_alloc(h, &call.ws.p, part + sizeof(float) * 2 * p.c * p.items);
  if (e != cudaSuccess) return cuda_error(h, e, "group norm workspace");
  p.part = static_cast<float2*>(call.ws.p);
  p.chan = reinterpret_cast<float*>(static_cast<char*>(call.ws.p) + part);
  const int dx_items = p.dx ? p.items : 0;
  const int chan_ctas = p.dw || p.db ? (p.c + kGnChanBlock - 1) / kGnChanBlock : 0;
  const size_t sums = gn_sum_smem(p.c, p.c / V), norms = sizeof(float) * 2 * std::max(p.groups, kGnThreads);
  ++h->launches;
  if (gn_ring<T, V>(p)) {
    if constexpr (V * sizeof(T) == 16) {
      e = gn_allow_smem(k_gn_bwd_sums<T, V, GS, true>, kGnRingSmem);
      if (e == cudaSuccess) e = gn_allow_smem(k_gn_bwd_apply<T, V, GS, true>, kGnRingSmem + 2 * sizeof(float) * 4096);
      if (e == cudaSuccess) {
        k_gn_bwd_sums<T, V, GS, true><<<p.items, kGnThreads, kGnRingSmem, h->stream>>>(p, call.plan);
        e = launch_ex(h, k_gn_bwd_apply<T, V, GS, true>, dx_items + chan_ctas, kGnRingSmem + norms, 0, p, call.plan,
                      chan_ctas);
      }
    }
  } else {
    k_gn_bwd_sums<T, V, GS, false><<<p.items, kGnThreads, sums, h->stream>>>(p, call.plan);
    e = launch_ex(h, k_gn_bwd_apply<T, V, GS, false>, dx_items + chan_ctas, norms, 0, p, call.plan, chan_ctas);
  }
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? SC_OK : cuda_error(h, e, "group norm backward launch");
}

// Channels of a vector that share a group: the whole vector, four of eight, or
// each its own.  Eight channels with statistics of their own spill registers:
// such rows go by vectors of four.
template <typename T, int V>
sc_status gn_run(Handle* h, const GnParams& p, const int32_t* cu, int batch, bool backward) {
  if constexpr (V >= 4)
    if (p.cg % V == 0) return backward ? gn_backward_v<T, V, V>(h, p, cu, batch) : gn_forward_v<T, V, V>(h, p, cu, batch);
  if constexpr (V == 8) {
    if (p.cg % 4 == 0) return backward ? gn_backward_v<T, V, 4>(h, p, cu, batch) : gn_forward_v<T, V, 4>(h, p, cu, batch);
    return gn_run<T, 4>(h, p, cu, batch, backward);
  } else {
    return backward ? gn_backward_v<T, V, 1>(h, p, cu, batch) : gn_forward_v<T, V, 1>(h, p, cu, batch);
  }
}

template <typename T>
sc_status gn_dispatch(Handle* h, const GnParams& p, const int32_t* cu, int batch, bool backward) {
  const void* ptrs[4] = {p.x, backward ? p.dy : p.y, backward ? p.dx : p.y, nullptr};
  const int v = gn_vec<T>(p.c, p.xs, ptrs, 3);
  if constexpr (sizeof(T) == 2)
    if (v == 8) return gn_run<T, 8>(h, p, cu, batch, backward);
  if (v == 4) return gn_run<T, 4>(h, p, cu, batch, backward);
  if (v == 2) return gn_run<T, 2>(h, p, cu, batch, backward);
  return gn_run<T, 1>(h, p, cu, batch, backward);
}

}  // namespace

sc_status group_norm(Handle* h, const void* x, int64_t x_stride, const void* weight, const void* bias, void* y,
                     float* stats, const int32_t* cu, int batch, int c, int groups, float eps, int silu,
                     sc_dtype dtype, sc_dtype wdtype) {
  GnParams p{};
  p.x = x; p.xs = x_stride; p.w = weight; p.b = bias; p.wdtype = wdtype; p.y = y; p.stats = stats;
  p.c = c; p.groups = groups; p.cg = c / groups; p.eps = eps; p.silu = silu; p.err = h->derr;
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
  p.c = c; p.groups = groups; p.cg = c / groups; p.silu = silu; p.err = h->derr;
  if (dtype == SC_F32) return gn_dispatch<float>(h, p, cu, batch, true);
  if (dtype == SC_BF16) return gn_dispatch<__nv_bfloat16>(h, p, cu, batch, true);
  return gn_dispatch<__half>(h, p, cu, batch, true);
}

}  // namespace sc
