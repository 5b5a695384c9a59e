// Varlen differential attention, backward.
//
// With P_m the softmax maps, recomputed from the forward's log-sum-exps, and
// dP = dO V^T, delta_m = rowsum(dO o O_m):
//   dS_1 = P_1 o (dP - delta_1),  dS_2 = -lam P_2 o (dP - delta_2),
//   dV = (P_1 - lam P_2)^T dO,  dQ_m = scale dS_m K_m,  dK_m = scale dS_m^T Q_m,
//   dlam_h = -sum_rows delta_2,
// dK and dV summed over the heads that share a key / value head.  O_1 and O_2
// are kept by the forward in f32.  Every sum has one fixed order.
//
// Two kernels of one shape (k_da_bwd): a CTA holds 128 rows X (queries for dQ,
// keys for dK and dV) and walks tiles of the other side Y.  Both maps share dP,
// and dV takes one product with the combined weights, so a pair of rows costs
// 768 flops in the dQ kernel and 1024 in the other.  Accumulating dQ in the
// dK / dV kernel instead would save the second recomputation (1,280 in all).  It
// was not tried: dQ would be summed across CTAs, in a fixed order only if each
// waits for its turn at a query tile, and its products have no tensor memory left
// there (Cfg).
//   warp 0     TMA producer: X's Q / K pair and its dO / V once, then Y's tiles
//              (and, for keys, the queries' statistics) into a ring
//   warp 1     issues S_m = X_m Y_m^T and dP into tensor memory
//   warp 3     issues the accumulations dX_m += dS_m Y_m, dV += P dO with dS and
//              P as A operands in tensor memory, Y MN-major
//   warp 2     zeroes Y rows behind the last visible one (0 * NaN)
//   warps 4-7, 8-11  the elementwise part, one row per thread: group 0 takes the
//              even steps, group 1 the odd ones
// Every buffer in tensor memory is single (S_1 S_2 dP P dS_1 dS_2 of 48 columns
// beside the accumulators fill it), but a group takes its row of S, then of dP,
// into registers at once, which frees them for the other group's step; so one
// group's exponentials run beside the other's products.
// Where X are keys, lse and delta belong to the columns.  Read from shared
// memory they cost 48 16-byte loads per thread and step beside the products'
// operands (565 of 1,274 us at 8,192 + 2,777 tokens and 8 heads), so the tensor
// cores add them: each statistic is split into three values of the input type
// (24 bits and more) and enters as one more K step of its product, against rows
// of a constant: S_m - lse_m / c and dP - delta_1 come out of tensor memory, and
// so does delta_1 - delta_2 for the 32 columns that still fit.
// P, dS_1 and dS_2 are rounded once to the input type, as operands of the last
// products, which f32 operands would halve in rate at least: dq is off by 0.0026
// relative in bf16 (2^-8 an element, averaged by the sum), 0.0017 in f32 with a
// rounded result.  Scores, statistics and accumulators stay f32.
// f16 has 2^-24 to 65,504 where weights of n keys are about 1 / n and score
// gradients less, so there the operands are scaled by powers of two, taken out
// of the f32 sums again.  With |dP - delta| <= 2 |dO_i| max_j |V_j| (O is a mean
// of V rows), a query's dS in the dQ kernel get the factor that takes this bound
// times max(1, |lam|) below 2^15; in the dK / dV kernel, whose rows sum over
// queries, dS get one for the sequence and its key / value head, and P - lam P_2
// one that takes 1 + |lam| there.  The factors of P are added to its exponent.
// k_da_top takes the norms' maxima.  8,192 keys, dO of 2^-14: dq is off by 0.067
// relative without the factors, with them by the rounding of its result (0.0074).
// Few CTAs: the walk is cut into ranges whose f32 sums k_da_bwd_join adds in order.
// Every mbarrier wait is bounded (SC_ETIMEOUT).
#include "sc_diffattn_dev.cuh"

#include <algorithm>
#include <vector>

namespace sc {
namespace {

constexpr int kX = 128;                   // rows per CTA
constexpr int kThreads = 384;
constexpr int kXBytes = kX * kDaD * 2;    // 16 KB
constexpr int kOffX = 0;                  // X_1, X_2, halves of the 128-wide one
constexpr int kOffY = 4 * kXBytes;
constexpr uint32_t kTmem = 512;

template <bool KV>
struct Cfg {
  static constexpr int kY = 48;                        // rows of Y per step
  static constexpr int kStages = 5;
  static constexpr int kYBytes = kY * kDaD * 2;
  // Y_1, Y_2, halves of the 128-wide one; statistics: 16-byte rows for S_1, S_2
  // and dP (kY each) and of delta_1 - delta_2 (kDiff), and the rest of it in f32
  static constexpr int kDiff = 32, kStatBytes = 16 * kY, kDiffBytes = 16 * kDiff, kRestBytes = 4 * (kY - kDiff);
  static constexpr int kStage = 4 * kYBytes + (KV ? 3 * 1024 : 0);
  static_assert(3 * kStatBytes + kDiffBytes + kRestBytes <= 3 * 1024, "stage");
  // constant rows against the split statistics (128 of 16 bytes), and zeros
  static constexpr int kOffOnes = kOffY + kStages * kStage, kOffZero = kOffOnes + kX * 16;
  static constexpr int kOffBar = kOffZero + kX * 16;
  static constexpr int kSmem = kOffBar + 256 + 1024;
  // tensor memory columns: S_1 S_2 dP [delta_1 - delta_2, P] dS_1 dS_2, then the accumulators
  static constexpr uint32_t kS = 0, kDp = 2 * kY, kD = 3 * kY, kP = kD + kDiff, kDs = KV ? kP + kY / 2 : 3 * kY,
                            kAcc = 256, kV = 384;
  static_assert(kDs + kY <= kAcc, "tensor memory");
};

struct DaBwd {
  LamRef lam;
  const float* lse;    // [2][heads][nq]
  const float* maps;   // [nq][heads][2][128]
  const void* dout;
  float* st;           // [5][heads][np]: -lse_1, -lse_2, -delta_1, -delta_2, delta_1 - delta_2; f16: a sixth, the
                       // exponent of the row's factor
  uint4* split;        // [4][heads][np] rows of eight values: -lse_m / c, -delta_1, delta_1 - delta_2 in three parts
  int64_t np;          // rows of st and split: sequences start at multiples of 4
  const float* top;    // f16: [2][batch][kv_heads] largest |V_j|^2 and |dO_i|^2 (records: part0 = batch entry)
  int batch;
  void *dq, *dk, *dv, *dlam;
  float* part;         // [splits][rows of X][heads of X][dX_1 dX_2 (dV)], when the walk is cut
  int64_t nx;          // rows of X in all
  int64_t nq;
  int heads, kv_heads, rep, causal;
  float scale, scale_log2;
  int* err;
};

__device__ __forceinline__ float warp_add(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ unsigned long long mul_f2(unsigned long long a, unsigned long long b) {
  unsigned long long d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
// Whether score gradients and weights are scaled into the type's range.
template <typename T> constexpr bool kScaled = std::is_same_v<T, __half>;
// A statistic v as three values of T, v = k0 a + k1 b + k2 c.  bf16 has f32's
// range.  f16: up to 65,504 * 1,024, in steps of 2^-34; a log-sum-exp over the
// scale or a delta beyond that (scores of 6.7e7 before the scale) becomes NaN, as
// does one that is no finite number, and so the gradients that it is part of.
template <typename T> struct Split {
  static constexpr float k0 = 1.f, k1 = 1.f, k2 = 1.f, kMost = 1e38f;
};
template <> struct Split<__half> {
  static constexpr float k0 = 1024.f, k1 = 1.f, k2 = 1.f / 1024.f, kMost = 65504.f * 1024.f;
};
template <typename T>
__device__ __forceinline__ uint4 split3(float v) {
  using S = Split<T>;
  v = fabsf(v) <= S::kMost ? v : NAN;
  const float a = Cvt<T>::to_f(Cvt<T>::from_f(v / S::k0)), r = v - a * S::k0, b = Cvt<T>::to_f(Cvt<T>::from_f(r / S::k1));
  return make_uint4(pack2<T>(a, b), pack2<T>((r - b * S::k1) / S::k2, 0.f), 0u, 0u);
}

// Whole e with 2^e bound < 2^want (and no less than half of it); `none` where
// bound is zero, infinite or NaN.
__device__ __forceinline__ int pow2_to(float bound, int want, int none) {
  if (!(bound > 0.f && bound < INFINITY)) return none;
  return max(-100, min(100, want - (__float_as_int(bound) >> 23) + 126));
}
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }

template <typename T>
__device__ __forceinline__ float4 load_f4(const T* p) {
  const uint2 raw = *reinterpret_cast<const uint2*>(p);
  const T* t = reinterpret_cast<const T*>(&raw);
  return make_float4(Cvt<T>::to_f(t[0]), Cvt<T>::to_f(t[1]), Cvt<T>::to_f(t[2]), Cvt<T>::to_f(t[3]));
}

// Largest squared norm of the 128-wide rows of each sequence and key / value
// head: top[sequence][group], zero before.  One CTA per (kTopRows rows, head),
// records: item0 counts such blocks, aux = the sequence.  The maximum of the
// bits of numbers that are not negative is theirs, NaN on top.
constexpr int kTopRows = 64;
template <typename T>
__global__ void __launch_bounds__(256) k_da_top(const T* x, int64_t stride, int rep, int groups, float* top,
                                                const __grid_constant__ SeqPlan plan) {
  __shared__ int s[8];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const SeqRec& r = plan.at(plan.find(blockIdx.x));
  const int64_t lo = r.q0 + static_cast<int64_t>(blockIdx.x - r.item0) * kTopRows;
  const int64_t hi = min(lo + kTopRows, static_cast<int64_t>(r.q1));
  float4 v[kTopRows / 8];  // every load ahead of the first use
#pragma unroll
  for (int k = 0; k < kTopRows / 8; ++k) {
    const int64_t i = lo + warp + 8 * k;
    v[k] = i < hi ? load_f4(x + i * stride + blockIdx.y * kDaDv + 4 * lane) : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  int most = 0;
#pragma unroll
  for (int k = 0; k < kTopRows / 8; ++k) {
    const float n = warp_add(fmaf(v[k].x, v[k].x, v[k].y * v[k].y) + fmaf(v[k].z, v[k].z, v[k].w * v[k].w));
    most = max(most, __float_as_int(n) & 0x7fffffff);
  }
  if (lane == 0) s[warp] = most;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 8; ++w) most = max(most, s[w]);
    atomicMax(reinterpret_cast<int*>(top) + static_cast<int64_t>(r.aux) * groups + blockIdx.y / rep, most);
  }
}

// Statistics of every (row, head), one warp each.  Records: aux = the
// sequence's first row in st.
template <typename T>
__global__ void __launch_bounds__(256) k_da_stats(const DaBwd p, const __grid_constant__ SeqPlan plan) {
  const int64_t at = blockIdx.x * 8ll + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (at >= p.nq * p.heads) return;
  const int row = static_cast<int>(at / p.heads), h = static_cast<int>(at % p.heads);
  const SeqRec& r = plan.at(plan.find(row));
  const float4 o1 = reinterpret_cast<const float4*>(p.maps + at * 2 * kDaDv)[lane];
  const float4 o2 = reinterpret_cast<const float4*>(p.maps + at * 2 * kDaDv + kDaDv)[lane];
  const float4 g = load_f4(static_cast<const T*>(p.dout) + at * kDaDv + 4 * lane);
  const float d1 = warp_add(fmaf(g.x, o1.x, g.y * o1.y) + fmaf(g.z, o1.z, g.w * o1.w));
  const float d2 = warp_add(fmaf(g.x, o2.x, g.y * o2.y) + fmaf(g.z, o2.z, g.w * o2.w));
  if constexpr (kScaled<T>) {
    const float n = warp_add(fmaf(g.x, g.x, g.y * g.y) + fmaf(g.z, g.z, g.w * g.w));
    const float v = p.top[static_cast<int64_t>(r.part0) * p.kv_heads + h / p.rep];
    if (lane == 0)
      p.st[(5ll * p.heads + h) * p.np + r.aux + (row - r.q0)] =
          static_cast<float>(pow2_to(2.f * sqrtf(n * v) * fmaxf(1.f, fabsf(p.lam.get(h))), 15, 0));
  }
  if (lane < 5) {
    const float l = lane < 2 ? p.lse[(static_cast<int64_t>(lane) * p.heads + h) * p.nq + row] : 0.f;
    const float v = lane < 2 ? -l : lane == 2 ? -d1 : lane == 3 ? -d2 : d1 - d2;
    const int64_t at_st = (static_cast<int64_t>(lane) * p.heads + h) * p.np + r.aux + (row - r.q0);
    p.st[at_st] = v;
    if (row == r.q1 - 1)  // up to three rows between sequences
      for (int i = 1; (r.aux + row - r.q0 + i) & 3; ++i) p.st[at_st + i] = 0.f;
  }
  if (lane < 4) {
    const float l = lane < 2 ? p.lse[(static_cast<int64_t>(lane) * p.heads + h) * p.nq + row] : 0.f;
    // l = +inf: a row without keys, which none of its columns is used for
    p.split[(static_cast<int64_t>(lane) * p.heads + h) * p.np + r.aux + (row - r.q0)] =
        split3<T>(lane < 2 ? (l == INFINITY ? 0.f : -l / p.scale_log2) : lane == 2 ? -d1 : d1 - d2);
  }
}

// dlam: one CTA per entry of lam sums -delta_2 over its heads' rows.
__global__ void __launch_bounds__(1024) k_da_dlam(const DaBwd p, int64_t rows) {
  __shared__ float s[32];
  const int heads = p.lam.count == 1 ? p.heads : 1;
  float a = 0.f;
  for (int k = 0; k < heads; ++k) {
    const float* d = p.st + (3ll * p.heads + blockIdx.x + k) * p.np;
    for (int64_t i = threadIdx.x; i < rows; i += 1024) a += d[i];
  }
  a = warp_add(a);
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = a;
  __syncthreads();
  if (threadIdx.x < 32) {
    a = warp_add(s[threadIdx.x]);
    if (threadIdx.x == 0) {
      if (p.lam.dtype == SC_F32) static_cast<float*>(p.dlam)[blockIdx.x] = a;
      else if (p.lam.dtype == SC_BF16) static_cast<__nv_bfloat16*>(p.dlam)[blockIdx.x] = __float2bfloat16_rn(a);
      else static_cast<__half*>(p.dlam)[blockIdx.x] = __float2half_rn(a);
    }
  }
}

// KV false: X = queries of one head, Y = keys; writes dQ.  KV true: X = keys of
// one key / value head, Y = the queries of each of its heads in turn; writes
// dK and dV.  tmX / tmXw: the 64- and 128-wide rows of X in boxes of 128; tmY /
// tmYw likewise in boxes of kY.  Records: item0 counts tiles of X, aux = the
// sequence's first row in st.  blockIdx.z: range of the walk.
template <typename T, bool KV>
__global__ void __launch_bounds__(kThreads, 1)
    k_da_bwd(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmXw,
             const __grid_constant__ CUtensorMap tmY, const __grid_constant__ CUtensorMap tmYw, const DaBwd p,
             const __grid_constant__ SeqPlan plan) {
  using C = Cfg<KV>;
  constexpr int kY = C::kY, kStages = C::kStages, kYBytes = C::kYBytes;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kOffBar);
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(bars + 28);
  const uint32_t x_full = smem_u32(bars);
  const uint32_t y_full0 = x_full + 8, y_empty0 = y_full0 + 8 * kStages;
  // per group (the step's parity): S written, dP written, the step's products done
  const uint32_t s_full0 = y_empty0 + 8 * kStages, dp_full0 = s_full0 + 16, p_free0 = dp_full0 + 16;
  // every step in turn: S read, dP read, P and dS written
  const uint32_t s_free = p_free0 + 16, dp_free = s_free + 8, ds_full = dp_free + 8;
  // rows to zero: asked for (warp 1), zeroed (warp 2), seen (warp 3)
  const uint32_t y_req = ds_full + 8, y_fixed = y_req + 8, y_ack = y_fixed + 8, done_bar = y_ack + 8;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const SeqRec& rec = plan.at(plan.find(blockIdx.x));
  const int lq = rec.q1 - rec.q0, lk = rec.k1 - rec.k0;
  const int ntiles = ((KV ? lk : lq) + kX - 1) / kX;
  int xt = blockIdx.x - rec.item0;
  if (!KV) xt = ntiles - 1 - xt;  // causal: the longest first
  const int x0 = xt * kX, nx = min(kX, (KV ? lk : lq) - x0);
  const int g = KV ? blockIdx.y : blockIdx.y / p.rep;
  // rows [y0, y1) of Y in ny tiles, for each of nh heads; this CTA takes steps [t0, t0 + n)
  const int y1 = KV ? lq : key_limit(rec, x0 + nx - 1, p.causal);
  const int y0 = KV && p.causal ? max(0, x0 - lk + lq) / kY * kY : 0;
  const int ny = y1 > y0 ? (y1 - y0 + kY - 1) / kY : 0;
  const int64_t all = static_cast<int64_t>(ny) * (KV ? p.rep : 1);
  const int t0 = static_cast<int>(all * blockIdx.z / gridDim.z);
  const int n = static_cast<int>(all * (blockIdx.z + 1) / gridDim.z) - t0;
  const bool ragged = (y1 - y0) % kY != 0;
  auto partial = [&](int j) { return ragged && (t0 + j) % ny == ny - 1; };  // the step's tile has rows that are not seen

  if (threadIdx.x == 0) {
    mbar_init(x_full, 1);
    for (int st = 0; st < kStages; ++st) {
      mbar_init(y_full0 + 8 * st, 1);
      mbar_init(y_empty0 + 8 * st, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(s_full0 + 8 * i, 1);
      mbar_init(dp_full0 + 8 * i, 1);
      mbar_init(p_free0 + 8 * i, 1);
    }
    mbar_init(s_free, 4);
    mbar_init(dp_free, 4);
    mbar_init(ds_full, 4);
    mbar_init(y_req, 1);
    mbar_init(y_fixed, 1);
    mbar_init(y_ack, 1);
    mbar_init(done_bar, 2);  // both issuers
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(s_tmem), kTmem);
    tmem_relinquish();
  }
  if (KV) {
    uint4* ones = reinterpret_cast<uint4*>(smem + C::kOffOnes);
    for (int i = threadIdx.x; i < 2 * kX; i += kThreads)
      ones[i] = i < kX ? make_uint4(pack2<T>(Split<T>::k0, Split<T>::k1), pack2<T>(Split<T>::k2, 0.f), 0u, 0u)
                       : make_uint4(0u, 0u, 0u, 0u);
    fence_proxy_async_smem();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *s_tmem;

  if (warp < 4) {
    regs_release();
    if (warp == 0) {
      // --------------------------------------------------------- producer
      if (n > 0 && elect_one()) {
        const int xrow = (KV ? rec.k0 : rec.q0) + x0, xh = blockIdx.y;
        mbar_arrive_expect_tx(x_full, 4 * kXBytes);
        tma_load_3d(sbase + kOffX, &tmX, 0, 2 * xh, xrow, x_full);
        tma_load_3d(sbase + kOffX + kXBytes, &tmX, 0, 2 * xh + 1, xrow, x_full);
        tma_load_3d(sbase + kOffX + 2 * kXBytes, &tmXw, 0, xh, xrow, x_full);
        tma_load_3d(sbase + kOffX + 3 * kXBytes, &tmXw, 64, xh, xrow, x_full);
        int ty = t0 % ny, yh = KV ? g * p.rep + t0 / ny : g, st = 0, use = 0, j = 0;
        for (; j < n; ++j) {
          if (!mbar_wait(y_empty0 + 8 * st, (use & 1) ^ 1, p.err)) break;
          const uint32_t yb = sbase + kOffY + st * C::kStage, bar = y_full0 + 8 * st;
          const int yr = y0 + ty * kY, yrow = (KV ? rec.q0 : rec.k0) + yr;
          mbar_arrive_expect_tx(bar, 4 * kYBytes + (KV ? 3 * C::kStatBytes + C::kDiffBytes + C::kRestBytes : 0));
          tma_load_3d(yb, &tmY, 0, 2 * yh, yrow, bar);
          tma_load_3d(yb + kYBytes, &tmY, 0, 2 * yh + 1, yrow, bar);
          tma_load_3d(yb + 2 * kYBytes, &tmYw, 0, yh, yrow, bar);
          tma_load_3d(yb + 3 * kYBytes, &tmYw, 64, yh, yrow, bar);
          if (KV) {  // st rows start at multiples of 4: 16-byte aligned; both go on behind their last row
            const int64_t at = static_cast<int64_t>(yh) * p.np + rec.aux + yr, step = static_cast<int64_t>(p.heads) * p.np;
            const uint32_t sb = yb + 4 * kYBytes;
            for (int k = 0; k < 3; ++k) bulk_load(sb + k * C::kStatBytes, p.split + k * step + at, C::kStatBytes, bar);
            bulk_load(sb + 3 * C::kStatBytes, p.split + 3 * step + at, C::kDiffBytes, bar);
            bulk_load(sb + 3 * C::kStatBytes + C::kDiffBytes, p.st + 4 * step + at + C::kDiff, C::kRestBytes, bar);
          }
          if (++ty == ny) ty = 0, yh += KV ? 1 : 0;
          if (++st == kStages) st = 0, ++use;
        }
        // the copies end before the CTA does, also where a wait has given up
        mbar_wait(x_full, 0, p.err);
        for (int i = max(0, j - kStages); i < j; ++i) mbar_wait(y_full0 + 8 * (i % kStages), (i / kStages) & 1, p.err);
      }
    } else if (warp == 1) {
      // ------------------------------------------------- S and dP of every step
      if (n > 0 && elect_one()) {
        const uint32_t id_s = idesc_f16(128, kY, std::is_same_v<T, __nv_bfloat16>);
        const uint64_t x1 = smem_desc(sbase + kOffX, 1024, 2), xw = x1 + 2 * kXBytes / 16;
        const uint64_t y1d = smem_desc(sbase + kOffY, 1024, 2);
        const uint32_t id_d = idesc_f16(128, C::kDiff, std::is_same_v<T, __nv_bfloat16>);
        // constant rows, and a tile's statistics; the second half of their K step is zeros
        const uint64_t one = smem_desc_plain(sbase + C::kOffOnes, C::kOffZero - C::kOffOnes, 128);
        auto stat_desc = [&](uint32_t a) { return smem_desc_plain(a, sbase + C::kOffZero - a, 128); };
        auto place = [&](uint64_t yd) { return static_cast<uint32_t>(yd - y1d) * 16u; };  // of a tile in the ring
        int ty = t0 % ny, st = 0, use = 0, asked = 0;  // tile and ring place of the next step to land; tiles to zero
        auto land = [&]() {
          bool r = mbar_wait(y_full0 + 8 * st, use & 1, p.err);
          if (r && ragged && ty == ny - 1) {
            if (asked > 0) r = mbar_wait(y_ack, (asked - 1) & 1, p.err);
            mbar_arrive(y_req);
            ++asked;
          }
          if (++ty == ny) ty = 0;
          if (++st == kStages) st = 0, ++use;
          return r;
        };
        auto issue_s = [&](int j, uint64_t yd) {
#pragma unroll
          for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int k = 0; k < kDaD / 16; ++k)  // 32 bytes a step, in units of 16
              tc_mma_f16(tmem + C::kS + kY * m, x1 + m * (kXBytes / 16) + 2 * k, yd + m * (kYBytes / 16) + 2 * k, id_s,
                         k > 0 ? 1u : 0u);
          if (KV) {
            const uint32_t sb = sbase + kOffY + place(yd) + 4 * kYBytes;
#pragma unroll
            for (int m = 0; m < 2; ++m)
              tc_mma_f16(tmem + C::kS + kY * m, one, stat_desc(sb + m * C::kStatBytes), id_s, 1u);
          }
          tc_commit(s_full0 + 8u * (j & 1));
        };
        auto issue_dp = [&](int j, uint64_t yd) {
#pragma unroll
          for (int k = 0; k < kDaDv / 16; ++k)
            tc_mma_f16(tmem + C::kDp, xw + (k / 4) * (kXBytes / 16) + 2 * (k % 4),
                       yd + (2 + k / 4) * (kYBytes / 16) + 2 * (k % 4), id_s, k > 0 ? 1u : 0u);
          if (KV) {
            const uint32_t sb = sbase + kOffY + place(yd) + 4 * kYBytes;
            tc_mma_f16(tmem + C::kDp, one, stat_desc(sb + 2 * C::kStatBytes), id_s, 1u);
            tc_mma_f16(tmem + C::kD, one, stat_desc(sb + 3 * C::kStatBytes), id_d, 0u);
          }
          tc_commit(dp_full0 + 8u * (j & 1));
        };
        bool ok = mbar_wait(x_full, 0, p.err) && land();
        if (ok) {
          tc_fence_after();
          issue_s(0, y1d);
          issue_dp(0, y1d);
        }
        // scores and dP of step j + 1 as soon as those of step j are in registers
        for (int j = 0; ok && j + 1 < n; ++j) {
          const uint64_t yd = y1d + static_cast<uint32_t>(st) * (C::kStage / 16);
          ok = land() && mbar_wait(s_free, j & 1, p.err);
          if (!ok) break;
          tc_fence_after();
          issue_s(j + 1, yd);
          ok = mbar_wait(dp_free, j & 1, p.err);
          if (!ok) break;
          tc_fence_after();
          issue_dp(j + 1, yd);
        }
        tc_commit(done_bar);  // every product ends before its tensor memory is released
        mbar_wait(done_bar, 0, p.err);
      }
    } else if (warp == 3) {
      // ------------------------------------------------------- the accumulations
      if (n > 0 && elect_one()) {
        const bool bf16 = std::is_same_v<T, __nv_bfloat16>;
        const uint32_t id_x = idesc_f16(128, 64, bf16) | (1u << 16), id_v = idesc_f16(128, 128, bf16) | (1u << 16);
        const uint64_t y1d = smem_desc_mn(sbase + kOffY, kYBytes);
        int ty = t0 % ny, st = 0, fixed = 0;
        bool ok = true;
        for (int j = 0; ok && j < n; ++j) {
          if (ragged && ty == ny - 1) {
            ok = mbar_wait(y_fixed, fixed++ & 1, p.err);
            mbar_arrive(y_ack);
          }
          ok = ok && mbar_wait(ds_full, j & 1, p.err);
          if (!ok) break;
          tc_fence_after();
          const uint64_t yd = y1d + static_cast<uint32_t>(st) * (C::kStage / 16);
          const uint32_t acc = j > 0 ? 1u : 0u;
#pragma unroll
          for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int k = 0; k < kY / 16; ++k)  // 16 rows of 128 bytes a step
              tc_mma_f16_tmem_a(tmem + C::kAcc + 64u * m, tmem + C::kDs + kY / 2 * m + 8u * k,
                                yd + m * (kYBytes / 16) + 128 * k, id_x, k > 0 ? 1u : acc);
          if (KV) {
#pragma unroll
            for (int k = 0; k < kY / 16; ++k)
              tc_mma_f16_tmem_a(tmem + C::kV, tmem + C::kP + 8u * k, yd + 2 * (kYBytes / 16) + 128 * k, id_v,
                                k > 0 ? 1u : acc);
          }
          tc_commit(p_free0 + 8u * (j & 1));
          tc_commit(y_empty0 + 8 * st);
          if (++ty == ny) ty = 0;
          if (++st == kStages) st = 0;
        }
        tc_commit(done_bar);
        mbar_wait(done_bar, 0, p.err);
      }
    } else if (warp == 2) {
      // ---------------------------------------- Y rows behind the last visible one
      if (ragged) {
        const uint32_t valid = (y1 - y0) - (ny - 1) * kY;
        int fixed = 0;
        for (int j = 0; j < n; ++j) {
          if (!partial(j)) continue;
          int w = 1;
          if (lane == 0) w = mbar_wait(y_req, fixed++ & 1, p.err) ? 1 : 0;
          if (__shfl_sync(0xffffffffu, w, 0) == 0) break;
          const uint32_t yb = sbase + kOffY + (j % kStages) * C::kStage;
          for (uint32_t a = 128u * valid + 16u * lane; a < static_cast<uint32_t>(kYBytes); a += 512u)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(yb + k * kYBytes + a), "r"(0u) : "memory");
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(y_fixed);
        }
      }
    }
  } else {
    // ------------------------------------------------- weights and score gradients
    regs_take();
    const int grp = (warp - 4) >> 2, row = (warp & 3) * 32 + lane, x = x0 + row;  // x: row of the sequence
    const uint32_t lane_base = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const bool live = row < nx;
    // this row sees the Y rows [lo, hi)
    const int lo = KV && p.causal ? x - lk + lq : 0;
    const int hi = KV ? lq : (live ? key_limit(rec, x, p.causal) : y1);
    const int lo_max = __reduce_max_sync(0xffffffffu, lo), hi_min = __reduce_min_sync(0xffffffffu, hi);
    float nl[2] = {0.f, 0.f}, nd[2] = {0.f, 0.f};
    // factors out of the accumulators; where X are keys, into P (2^lift) and into dP - delta (fac)
    float out_x = p.scale, out_v = 1.f, lift = 0.f, fac = 1.f;
    if (!KV && live) {
      const int64_t at = static_cast<int64_t>(blockIdx.y) * p.np + rec.aux + x, step = static_cast<int64_t>(p.heads) * p.np;
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        nl[m] = p.st[m * step + at];
        nd[m] = p.st[(2 + m) * step + at];
      }
      if constexpr (kScaled<T>) {
        const float e = p.st[5 * step + at];
        nl[0] += e;
        nl[1] += e;
        out_x *= pow2(-static_cast<int>(e));
      }
    }
    if constexpr (KV && kScaled<T>) {
      float most = 1.f;
      for (int i = 0; i < (p.lam.count == 1 || !p.lam.p ? 1 : p.rep); ++i) most = fmaxf(most, fabsf(p.lam.get(g * p.rep + i)));
      const float* top = p.top + static_cast<int64_t>(rec.part0) * p.kv_heads + g;
      const int b = pow2_to(1.f + most, 15, 0);
      const int f = pow2_to(2.f * sqrtf(top[0] * top[static_cast<int64_t>(p.batch) * p.kv_heads]) * most, 15 - b, -b);
      lift = static_cast<float>(b);
      fac = pow2(f);
      out_v = pow2(-b);
      out_x *= out_v * pow2(-f);
    }
    bool ok = true;
    const unsigned long long sc2 = f2(p.scale_log2, p.scale_log2);
    // tile and head of the group's step, its place in the ring
    int ty = n > 0 ? (t0 + grp) % ny : 0, head = KV ? g * p.rep + (n > 0 ? (t0 + grp) / ny : 0) : blockIdx.y;
    int place = grp, use = 0;
    float nlam = n > grp ? -p.lam.get(head) : 0.f;
    for (int j = grp; j < n; j += 2) {
      if (j > grp) {
        ty += 2;
        place += 2;
        if (place >= kStages) place -= kStages, use ^= 1;
        while (ty >= ny) {
          ty -= ny;
          if (KV) nlam = -p.lam.get(++head);
        }
      }
      const int c0 = y0 + ty * kY;
      const uint32_t turn = (j >> 1) & 1;
      const bool full = c0 >= lo_max && c0 + kY <= hi_min;
      const float4* rest = reinterpret_cast<const float4*>(smem + kOffY + place * C::kStage + 4 * kYBytes +
                                                           3 * C::kStatBytes + C::kDiffBytes);
      ok = warp_wait(s_full0 + 8u * grp, turn, p.err);
      // the statistics landed with the tile: the MMA thread has seen that, this one has not
      if (KV) ok = ok && warp_wait(y_full0 + 8 * place, use, p.err);
      if (!ok) break;
      tc_fence_after();
      float w[2][kY], dp[kY];
      tmem_ld48x2(lane_base + C::kS, lane_base + C::kS + kY, w[0], w[1]);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(s_free);
      auto weights = [&](int m) {
#pragma unroll
        for (int i = 0; i < kY; i += 2) {
          const unsigned long long x2 = f2(w[m][i], w[m][i + 1]);
          float a, b;
          f2_split(!KV             ? fma_f2(x2, sc2, f2(nl[m], nl[m]))
                   : kScaled<T> ? fma_f2(x2, sc2, f2(lift, lift))
                                : mul_f2(x2, sc2),
                   a, b);
          w[m][i] = ex2_ftz(a);
          w[m][i + 1] = ex2_ftz(b);
        }
      };
      weights(0);
      ok = warp_wait(dp_full0 + 8u * grp, turn, p.err);
      if (!ok) break;
      tc_fence_after();
      tmem_ld48(lane_base + C::kDp, dp);
      float diff[kY];  // delta_1 - delta_2 (of the columns; where X are queries, of the row)
      if constexpr (KV) {
        float d[C::kDiff];
        tmem_ld32(lane_base + C::kD, d);
#pragma unroll
        for (int i = 0; i < kY; i += 4) {
          const float4 r4 = i < C::kDiff ? make_float4(d[i], d[i + 1], d[i + 2], d[i + 3]) : rest[(i - C::kDiff) / 4];
          diff[i] = r4.x;
          diff[i + 1] = r4.y;
          diff[i + 2] = r4.z;
          diff[i + 3] = r4.w;
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(dp_free);
      weights(1);
      if (!full) {  // weight 0, and 0 * NaN of a row that is not seen
#pragma unroll
        for (int i = 0; i < kY; ++i) {
          const bool see = c0 + i >= lo && c0 + i < hi;
          w[0][i] = see ? w[0][i] : 0.f;
          w[1][i] = see ? w[1][i] : 0.f;
          dp[i] = see ? dp[i] : 0.f;
          if (KV) diff[i] = see ? diff[i] : 0.f;
        }
      }
      const unsigned long long nlam2 = f2(nlam, nlam);
      uint32_t pk[kY / 16][8], k1[kY / 16][8], k2[kY / 16][8];
#pragma unroll
      for (int e = 0; e < kY; e += 2) {
        // dP - delta_1 and dP - delta_2
        unsigned long long d1 = f2(dp[e], dp[e + 1]), d2;
        if (KV && kScaled<T>) {
          d1 = mul_f2(d1, f2(fac, fac));
          d2 = fma_f2(f2(diff[e], diff[e + 1]), f2(fac, fac), d1);
        } else if (KV) {
          d2 = add_f2(d1, f2(diff[e], diff[e + 1]));
        } else {
          d2 = add_f2(d1, f2(nd[1], nd[1]));
          d1 = add_f2(d1, f2(nd[0], nd[0]));
        }
        const unsigned long long w1 = f2(w[0][e], w[0][e + 1]);
        const unsigned long long w2 = mul_f2(nlam2, f2(w[1][e], w[1][e + 1]));  // -lam P_2
        float a, b;
        f2_split(mul_f2(w1, d1), a, b);
        k1[e / 16][e % 16 / 2] = pack2<T>(a, b);
        f2_split(mul_f2(w2, d2), a, b);
        k2[e / 16][e % 16 / 2] = pack2<T>(a, b);
        if (KV) {
          f2_split(add_f2(w1, w2), a, b);
          pk[e / 16][e % 16 / 2] = pack2<T>(a, b);
        }
      }
      // the columns of the step before are read: only these stores and the
      // products stand between one step's wait here and the next one's.  (A try
      // ahead of need would suspend the warp: 902 against 757 us for dk and dv.)
      if (j > 0) ok = warp_wait(p_free0 + 8u * (grp ^ 1), ((j - 1) >> 1) & 1, p.err);
      if (!ok) break;
      tc_fence_after();
#pragma unroll
      for (int c = 0; c < kY / 16; ++c) {
        if (KV) tmem_st8(lane_base + C::kP + 8 * c, pk[c]);
        tmem_st8(lane_base + C::kDs + 8 * c, k1[c]);
        tmem_st8(lane_base + C::kDs + kY / 2 + 8 * c, k2[c]);
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(ds_full);
    }
    ok = ok && n > 0 && warp_wait(done_bar, 0, p.err);
    tc_fence_after();
    // group 0 writes dX_1, group 1 dX_2, and each its half of dV's columns
    const int xheads = KV ? p.kv_heads : p.heads;
    const int64_t at = (static_cast<int64_t>(KV ? rec.k0 : rec.q0) + x) * xheads + blockIdx.y;
    T* dx = static_cast<T*>(KV ? p.dk : p.dq);
    T* dv = static_cast<T*>(p.dv);
    constexpr int kWide = KV ? 256 : 128;
#pragma unroll
    for (int part = 0; part < (KV ? 2 : 1); ++part)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float o[32];
        __syncwarp();
        if (n > 0) tmem_ld32(lane_base + (part ? C::kV : C::kAcc) + 64u * grp + 32u * c, o);
        const int col = 64 * grp + 32 * c;
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = ok ? o[i] * (part ? out_v : out_x) : 0.f;
        if (live && p.part) {
          float4* dst = reinterpret_cast<float4*>(p.part + (blockIdx.z * p.nx * xheads + at) * kWide + 128 * part + col);
#pragma unroll
          for (int i = 0; i < 8; ++i) dst[i] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
        } else if (live && (part ? dv : dx)) {
          uint4* dst = reinterpret_cast<uint4*>((part ? dv : dx) + at * 128 + col);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            dst[i] = make_uint4(pack2<T>(o[8 * i], o[8 * i + 1]), pack2<T>(o[8 * i + 2], o[8 * i + 3]),
                                pack2<T>(o[8 * i + 4], o[8 * i + 5]), pack2<T>(o[8 * i + 6], o[8 * i + 7]));
        }
      }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmem);
  }
}

// Adds the ranges' sums in order: [splits][rows][wide] f32 -> the first 128
// columns to dx, the others to dv (each may be null), four columns a thread.
template <typename T>
__global__ void __launch_bounds__(256) k_da_bwd_join(const float* part, int splits, int64_t rows, int wide, T* dx, T* dv) {
  const int64_t i = blockIdx.x * 256ll + threadIdx.x;
  const int64_t row = i / (wide / 4);
  if (row >= rows) return;
  const int col = static_cast<int>(i % (wide / 4)) * 4;
  T* out = col < 128 ? dx : dv;
  if (!out) return;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int k = 0; k < splits; ++k) {
    const float4 v = *reinterpret_cast<const float4*>(part + (k * rows + row) * wide + col);
    s = make_float4(s.x + v.x, s.y + v.y, s.z + v.z, s.w + v.w);
  }
  *reinterpret_cast<uint2*>(out + row * 128 + (col & 127)) = make_uint2(pack2<T>(s.x, s.y), pack2<T>(s.z, s.w));
}

bool box_map(CUtensorMap* m, bool bf16, const void* base, int width, int heads, int64_t rows, int64_t stride,
             int box_rows) {
  const uint64_t d[3] = {static_cast<uint64_t>(width), static_cast<uint64_t>(heads),
                         static_cast<uint64_t>(std::max<int64_t>(rows, 1))};
  const uint64_t s[2] = {static_cast<uint64_t>(width) * 2, static_cast<uint64_t>(stride) * 2};
  const uint32_t b[3] = {64, 1, static_cast<uint32_t>(box_rows)};
  return make_map_nd(m, bf16, base, 3, d, s, b);
}

template <typename T, bool KV>
sc_status launch_bwd(Handle* h, const DaArgs& a, DaBwd p, const std::vector<int32_t>& st_row) {
  constexpr int kY = Cfg<KV>::kY;
  const bool bf16 = std::is_same_v<T, __nv_bfloat16>;
  const int64_t nq = a.cu_q[a.batch], nkv = a.cu_kv[a.batch];
  std::vector<SeqRec> recs;
  for (int b = 0; b < a.batch; ++b)
    if (KV ? a.cu_kv[b + 1] > a.cu_kv[b] : a.cu_q[b + 1] > a.cu_q[b])
      recs.push_back(SeqRec{a.cu_q[b], a.cu_q[b + 1], a.cu_kv[b], a.cu_kv[b + 1], 0, st_row[b], b});
  if (recs.empty()) return SC_OK;
  // the longest walks first: the tail of the launch is made of short CTAs
  std::stable_sort(recs.begin(), recs.end(), [](const SeqRec& x, const SeqRec& y) {
    return KV ? x.q1 - x.q0 > y.q1 - y.q0 : x.k1 - x.k0 > y.k1 - y.k0;
  });
  int64_t items = 0, steps = 0;
  const int xheads = KV ? a.kv_heads : a.heads;
  for (SeqRec& r : recs) {
    const int64_t tiles = ((KV ? r.k1 - r.k0 : r.q1 - r.q0) + kX - 1) / kX;
    r.item0 = static_cast<int32_t>(items);
    items += tiles;
    steps += tiles * (((KV ? r.q1 - r.q0 : r.k1 - r.k0) + kY - 1) / kY) * (KV ? p.rep : 1);
  }
  // Fewer CTAs than SMs: the walks are cut so that two CTAs a SM have work, in
  // ranges of eight steps at least (their sums cost a write and a read).
  int64_t splits = 1;
  if (items * xheads < h->num_sms)
    splits = std::max<int64_t>(1, std::min<int64_t>({2ll * h->num_sms / (items * xheads), steps / items / 8, 32}));
  // a side without rows is never read, but its maps want an address
  const void* some = nq > 0 ? a.q : a.k;
  const void *q = nq > 0 ? a.q : some, *go = nq > 0 ? a.dout : some, *k = nkv > 0 ? a.k : some,
             *v = nkv > 0 ? a.v : some;
  const int64_t dense = 128ll * a.heads;
  const int64_t qs = nq > 0 ? a.qs : dense, ks = nkv > 0 ? a.ks : 128ll * a.kv_heads,
                vs = nkv > 0 ? a.vs : 128ll * a.kv_heads;
  CUtensorMap mq, mo, mk, mv;
  if (!box_map(&mq, bf16, q, kDaD, 2 * a.heads, nq, qs, KV ? kY : kX) ||
      !box_map(&mo, bf16, go, kDaDv, a.heads, nq, dense, KV ? kY : kX) ||
      !box_map(&mk, bf16, k, kDaD, 2 * a.kv_heads, nkv, ks, KV ? kX : kY) ||
      !box_map(&mv, bf16, v, kDaDv, a.kv_heads, nkv, vs, KV ? kX : kY))
    return set_error(h, SC_ECUDA, "cuTensorMapEncodeTiled failed (differential attention backward)");
  SeqPlan plan;
  DevBuf table(h), part(h);
  const sc_status st = make_plan(h, recs, &plan, &table.p);
  if (st != SC_OK) return st;
  cudaError_t e = cudaSuccess;
  p.nx = KV ? nkv : nq;
  const int wide = KV ? 256 : 128;
  if (splits > 1) {
    e = dev_alloc(h, &part.p, sizeof(float) * splits * p.nx * xheads * wide);
    if (e != cudaSuccess) return cuda_error(h, e, "differential attention workspace");
    p.part = static_cast<float*>(part.p);
  }
  e = cudaFuncSetAttribute(k_da_bwd<T, KV>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<KV>::kSmem);
  if (e == cudaSuccess) {
    ++h->launches;
    const dim3 grid(static_cast<unsigned>(items), xheads, static_cast<unsigned>(splits));
    if (KV) k_da_bwd<T, KV><<<grid, kThreads, Cfg<KV>::kSmem, h->stream>>>(mk, mv, mq, mo, p, plan);
    else k_da_bwd<T, KV><<<grid, kThreads, Cfg<KV>::kSmem, h->stream>>>(mq, mo, mk, mv, p, plan);
    if (splits > 1) {
      ++h->launches;
      const int64_t rows = p.nx * xheads;
      k_da_bwd_join<T><<<static_cast<unsigned>((rows * (wide / 4) + 255) / 256), 256, 0, h->stream>>>(
          p.part, static_cast<int>(splits), rows, wide, static_cast<T*>(KV ? p.dk : p.dq),
          static_cast<T*>(KV ? p.dv : nullptr));
    }
    e = cudaGetLastError();
  }
  return e == cudaSuccess ? SC_OK : cuda_error(h, e, "differential attention backward launch");
}

// top[sequence][group] of the rows of x (k_da_top), `heads` of them a token.
template <typename T>
sc_status launch_top(Handle* h, const void* x, int64_t stride, const int32_t* cu, int batch, int heads, int groups,
                     float* top) {
  std::vector<SeqRec> recs;
  int64_t items = 0;
  for (int b = 0; b < batch; ++b) {
    if (cu[b + 1] == cu[b]) continue;
    recs.push_back(SeqRec{cu[b], cu[b + 1], 0, 0, static_cast<int32_t>(items), b});
    items += (cu[b + 1] - cu[b] + kTopRows - 1) / kTopRows;
  }
  if (recs.empty()) return SC_OK;
  SeqPlan plan;
  DevBuf table(h);
  const sc_status st = make_plan(h, recs, &plan, &table.p);
  if (st != SC_OK) return st;
  ++h->launches;
  k_da_top<T><<<dim3(static_cast<unsigned>(items), heads), 256, 0, h->stream>>>(static_cast<const T*>(x), stride,
                                                                              heads / groups, groups, top, plan);
  return SC_OK;
}

template <typename T>
sc_status run_backward(Handle* h, const DaArgs& a) {
  const int64_t nq = a.cu_q[a.batch];
  DaBwd p{};
  p.lam = LamRef{a.lam, a.lam_count, a.lam_dtype, a.lam_value};
  p.lse = a.lse;
  p.maps = a.maps;
  p.dout = a.dout;
  p.dq = a.dq;
  p.dk = a.dk;
  p.dv = a.dv;
  p.dlam = a.dlam;
  p.nq = nq;
  p.heads = a.heads;
  p.kv_heads = a.kv_heads;
  p.rep = a.heads / a.kv_heads;
  p.causal = a.causal;
  p.scale = a.scale;
  p.scale_log2 = a.scale * kLog2e;
  p.err = h->derr;
  // statistics rows: every sequence starts at a multiple of 4 (16-byte bulk copies)
  std::vector<int32_t> st_row(a.batch);
  std::vector<SeqRec> recs;
  int64_t rows = 0;
  for (int b = 0; b < a.batch; ++b) {
    st_row[b] = static_cast<int32_t>(rows);
    if (a.cu_q[b + 1] == a.cu_q[b]) continue;
    recs.push_back(SeqRec{a.cu_q[b], a.cu_q[b + 1], 0, 0, a.cu_q[b], st_row[b], b});
    rows += (a.cu_q[b + 1] - a.cu_q[b] + 3) / 4 * 4;
    if (rows > 0x7fffff00) return set_error(h, SC_EINVAL, "differential attention backward: too many rows");
  }
  p.np = rows + Cfg<true>::kY;  // a tile's copy may reach behind the last row
  const size_t per = static_cast<size_t>(a.heads) * p.np;
  DevBuf buf(h);
  const size_t tops = kScaled<T> ? static_cast<size_t>(a.batch) * a.kv_heads : 0;
  cudaError_t e = dev_alloc(h, &buf.p, per * (4 * sizeof(uint4) + (kScaled<T> ? 6 : 5) * sizeof(float)) +
                                           2 * tops * sizeof(float));
  p.split = static_cast<uint4*>(buf.p);
  if (e != cudaSuccess) return cuda_error(h, e, "differential attention workspace");
  p.st = reinterpret_cast<float*>(p.split + 4 * per);
  p.batch = a.batch;
  sc_status st = SC_OK;
  if constexpr (kScaled<T>) {
    float* top = p.st + 6 * per;
    p.top = top;
    e = cudaMemsetAsync(top, 0, 2 * tops * sizeof(float), h->stream);
    if (e != cudaSuccess) return cuda_error(h, e, "differential attention workspace");
    st = launch_top<T>(h, a.v, a.vs, a.cu_kv, a.batch, a.kv_heads, a.kv_heads, top);
    if (st == SC_OK) st = launch_top<T>(h, a.dout, 128ll * a.heads, a.cu_q, a.batch, a.heads, a.kv_heads, top + tops);
  }
  if (st == SC_OK && nq > 0) {
    SeqPlan plan;
    DevBuf table(h);
    st = make_plan(h, recs, &plan, &table.p);
    if (st == SC_OK) {
      ++h->launches;
      k_da_stats<T><<<static_cast<unsigned>((nq * a.heads + 7) / 8), 256, 0, h->stream>>>(p, plan);
    }
  }
  if (st == SC_OK && a.dlam) {
    ++h->launches;
    k_da_dlam<<<a.lam_count, 1024, 0, h->stream>>>(p, rows);
  }
  if (st == SC_OK && (a.dk || a.dv)) st = launch_bwd<T, true>(h, a, p, st_row);
  if (st == SC_OK && a.dq) st = launch_bwd<T, false>(h, a, p, st_row);
  e = cudaGetLastError();
  if (st != SC_OK) return st;
  return e == cudaSuccess ? SC_OK : cuda_error(h, e, "differential attention backward launch");
}

}  // namespace

sc_status diff_attention_backward(Handle* h, const DaArgs& a) {
  return a.dtype == SC_BF16 ? run_backward<__nv_bfloat16>(h, a) : run_backward<__half>(h, a);
}

}  // namespace sc
