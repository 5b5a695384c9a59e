// Varlen differential attention, forward.
//
// For every sequence, head h and query row i
//   out[i, h] = O_1 - lam_h O_2,  O_m = softmax_j(scale Q_m[i] . K_m[j]) V[j],
// Q_m = q[:, 2h + m], K_m = k[:, 2g + m], V = v[:, g], g = h / (heads / kv_heads).
// Sums and softmax statistics are f32; the weights are rounded to the input
// type for the second product (f32 weights would halve its rate at least; the
// output's own rounding is as large).  NaN and +inf scores, and rows whose scores
// are all -inf, give NaN as softmax does; rows without keys are zero.
//
// One CTA per (tile of 128 rows, key / value head, range of keys).  A row is a
// (token, head) pair: the heads that share a key / value head lie side by side
// in a tile, so its keys and values are read once for all of them.  The two
// maps share V, so a CTA runs both over the same key tiles (step i = tile i / 2,
// map i % 2).  Tensor memory: O_1 and O_2 (128 columns each), one score buffer
// of 128 columns that the maps use in turn, and 64 columns of weights per map.
// A softmax thread takes its whole row of scores into registers at once, which
// frees the buffer for the next step's scores long before the weights of this
// step are done; with a score buffer per map that the weights overwrote, a map
// waited for its P V and the scores behind it every tile (746 TFLOP/s).
//   warp 0     TMA producer: Q_1, Q_2 once, then K_1, K_2 and V of a 128-key
//              tile (64 KB) into a ring of three; Q and the first three tiles
//              are asked for with the barriers, before tensor memory is there
//   warp 1     issues the products: S of step i + 1 when the scores of step i
//              are read, O_m += P_m V of step i when its weights are written (P
//              as the A operand in tensor memory, V from shared memory, MN-major)
//   warp 2     zeroes V rows behind the last key that any row of the tile sees
//              (their weights are 0, but 0 * NaN would be NaN)
//   warps 4-7, 8-11  softmax of map 1 / map 2, one row per thread: running
//              maximum and sum, P = 2^(s scale log2 e - max); O is rescaled in
//              tensor memory only when the maximum grows by more than 2^8
// Then out = O_1 / l_1 - lam O_2 / l_2, each group taking half of the columns.
//
// Few rows against many keys: the keys are cut into ranges, each CTA keeps its
// unnormalised f32 O_m with (max, sum), and k_da_join combines them in order.
// k_da_join is launched early and waits for the ranges on the device (7 us for 24
// single tokens of 16 heads, beside 98 us of k_da_fwd).
// Every mbarrier wait is bounded (SC_ETIMEOUT).
#include "sc_diffattn_dev.cuh"

#include <algorithm>
#include <vector>

namespace sc {
namespace {

constexpr int kTile = 128;                 // rows per CTA, keys per step
constexpr int kStages = 3;
constexpr int kThreads = 384;
constexpr int kQBytes = kTile * kDaD * 2;  // 16 KB: Q_m, K_m or half of V
constexpr int kStageBytes = 4 * kQBytes;   // K_1, K_2, V[:, :64], V[:, 64:]
constexpr int kOffQ = 0;
constexpr int kOffKV = 2 * kQBytes;
constexpr int kOffBar = kOffKV + kStages * kStageBytes;
constexpr int kSmem = kOffBar + 256 + 1024;
constexpr uint32_t kTmem = 512;            // S | P_1 | P_2 | O_1 | O_2
constexpr uint32_t kColP = 128, kColO = 256;  // + 64 m, + 128 m
constexpr float kRescale = 8.f;            // log2
// f16 weights are written 2^7 times larger, between 2^7 and 2^15 where they are
// largest: f16 has steps of 2^-24 at least, so unlifted it drops keys below 2^-25
// of the row's largest weight, of which 100,000 can make 0.3% of a row.
template <typename T> constexpr float kLift = std::is_same_v<T, __half> ? 7.f : 0.f;

struct DaFwd {
  LamRef lam;
  void* out;
  float* lse;
  float* maps;
  float* part_o;    // [part rows][heads][2][128], unnormalised: row part0 + range * rows + row of a cut sequence
  float4* part_ml;  // [part rows][heads] (max_1, sum_1, max_2, sum_2)
  int64_t nq;
  int heads, rep, pack, tokens;  // rep = heads / kv_heads; heads and tokens of a tile (pack * tokens rows)
  int causal;
  int split_keys;   // keys per range (the last may be short and fills gaps), a multiple of 128
  float scale_log2;
  int* err;
};

struct DaTile {
  int32_t tok0, ntok;    // tokens [tok0, tok0 + ntok), tok0 counted in the sequence
  int32_t key0, key1;    // keys [key0, key1) of the sequence that this CTA reads
  int split, nsplit;
  __device__ __forceinline__ DaTile(const SeqRec& r, int local, const DaFwd& p) {
    const int tiles = r.aux, lk = r.k1 - r.k0, lq = r.q1 - r.q0;
    nsplit = max(1, (lk + p.split_keys - 1) / p.split_keys);
    split = local / tiles;
    const int t = tiles - 1 - local % tiles;  // causal: the tiles that see the most keys first
    tok0 = t * p.tokens;
    ntok = min(p.tokens, lq - tok0);
    key0 = split * p.split_keys;
    key1 = min(min(lk, key0 + p.split_keys), key_limit(r, tok0 + ntok - 1, p.causal));
  }
};

template <typename T>
__global__ void __launch_bounds__(kThreads, 1)
    k_da_fwd(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
             const __grid_constant__ CUtensorMap tmV, const DaFwd p, const __grid_constant__ SeqPlan plan) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kOffBar);
  float2* s_row = reinterpret_cast<float2*>(smem + kOffQ);  // (max, sum) per map and row, once Q is no longer read
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(bars + 24);
  const uint32_t q_full = smem_u32(bars);
  const uint32_t kv_full0 = q_full + 8, kv_empty0 = kv_full0 + 8 * kStages;
  const uint32_t s_full0 = kv_empty0 + 8 * kStages, p_full0 = s_full0 + 16, o_done0 = p_full0 + 16;  // per map
  const uint32_t s_free = o_done0 + 16, done_bar = s_free + 8, v_req = done_bar + 8, v_fixed = v_req + 8;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const SeqRec& rec = plan.at(plan.find(blockIdx.x));
  const DaTile tile(rec, blockIdx.x - rec.item0, p);
  const int g = blockIdx.y, h0 = g * p.pack;
  const int nk = tile.key1 > tile.key0 ? (tile.key1 - tile.key0 + kTile - 1) / kTile : 0;
  const bool last_partial = nk > 0 && tile.key1 - tile.key0 < nk * kTile;
  const int rows = tile.ntok * p.pack;

  const int gk = h0 / p.rep;  // key / value head
  auto load_tile = [&](int j) {
    const uint32_t kb = sbase + kOffKV + (j % kStages) * kStageBytes, bar = kv_full0 + 8 * (j % kStages);
    const int row = rec.k0 + tile.key0 + j * kTile;
    mbar_arrive_expect_tx(bar, kStageBytes);
    tma_load_3d(kb, &tmK, 0, 2 * gk, row, bar);
    tma_load_3d(kb + kQBytes, &tmK, 0, 2 * gk + 1, row, bar);
    tma_load_3d(kb + 2 * kQBytes, &tmV, 0, gk, row, bar);
    tma_load_3d(kb + 3 * kQBytes, &tmV, 64, gk, row, bar);
  };
  // the barriers, and at once the loads that wait for nothing
  if (warp == 0 && elect_one()) {
    mbar_init(q_full, 1);
    for (int st = 0; st < kStages; ++st) {
      mbar_init(kv_full0 + 8 * st, 1);
      mbar_init(kv_empty0 + 8 * st, 1);
    }
    for (int m = 0; m < 2; ++m) {
      mbar_init(s_full0 + 8 * m, 1);
      mbar_init(p_full0 + 8 * m, (rows + 31) / 32);  // one arrival per warp with rows
      mbar_init(o_done0 + 8 * m, 1);
    }
    mbar_init(s_free, (rows + 31) / 32);
    mbar_init(done_bar, 1);
    mbar_init(v_req, 1);
    mbar_init(v_fixed, 1);
    fence_mbar_init();
    if (nk > 0) {
      mbar_arrive_expect_tx(q_full, 2 * p.pack * p.tokens * 128);
      for (int m = 0; m < 2; ++m)
        tma_load_4d(sbase + kOffQ + m * kQBytes, &tmQ, 0, m, h0, rec.q0 + tile.tok0, q_full);
      for (int j = 0; j < min(nk, kStages); ++j) load_tile(j);
    }
  }
  __syncwarp();
  if (warp == 1) {
    tmem_alloc(smem_u32(s_tmem), kTmem);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *s_tmem;

  if (warp < 4) {
    regs_release();
    if (warp == 0) {
    // ----------------------------------------------------------- producer
    if (nk > 0 && elect_one()) {
      int j = min(nk, kStages);
      for (; j < nk; ++j) {
        if (!mbar_wait(kv_empty0 + 8 * (j % kStages), ((j / kStages) & 1) ^ 1, p.err)) break;
        load_tile(j);
      }
      // the copies end before the CTA does, also where a wait has given up
      mbar_wait(q_full, 0, p.err);
      for (int i = max(0, j - kStages); i < j; ++i)
        mbar_wait(kv_full0 + 8 * (i % kStages), (i / kStages) & 1, p.err);
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------- MMA issuer
    if (nk > 0 && elect_one()) {
      const bool bf16 = std::is_same_v<T, __nv_bfloat16>;
      const uint32_t id_s = idesc_f16(128, 128, bf16), id_o = idesc_f16(128, 128, bf16) | (1u << 16);  // V MN-major
      auto issue_s = [&](int i) {
        const int m = i & 1, j = i >> 1;
        const uint64_t q = smem_desc(sbase + kOffQ + m * kQBytes, 1024, 2);
        const uint64_t kd = smem_desc(sbase + kOffKV + (j % kStages) * kStageBytes + m * kQBytes, 1024, 2);
#pragma unroll
        for (int k = 0; k < kDaD / 16; ++k)  // 32 bytes a step, in units of 16
          tc_mma_f16(tmem, q + 2 * k, kd + 2 * k, id_s, k > 0 ? 1u : 0u);
        tc_commit(s_full0 + 8u * m);
      };
      auto issue_o = [&](int i) {  // O_m (+)= P_m V_j
        const int m = i & 1, j = i >> 1;
        const uint64_t v = smem_desc_mn(sbase + kOffKV + (j % kStages) * kStageBytes + 2 * kQBytes, kQBytes);
#pragma unroll
        for (int k = 0; k < kTile / 16; ++k)  // 16 keys of 128 bytes a step
          tc_mma_f16_tmem_a(tmem + kColO + 128u * m, tmem + kColP + 64u * m + 8u * k, v + 128 * k, id_o,
                            (j > 0 || k > 0) ? 1u : 0u);
        tc_commit(o_done0 + 8u * m);
        if (m == 1) tc_commit(kv_empty0 + 8 * (j % kStages));  // K_j and V_j are read
      };
      auto landed = [&](int j) {
        const bool r = mbar_wait(kv_full0 + 8 * (j % kStages), (j / kStages) & 1, p.err);
        if (r && j == nk - 1 && last_partial) mbar_arrive(v_req);
        return r;
      };
      bool ok = mbar_wait(q_full, 0, p.err) && landed(0);
      if (ok) {
        tc_fence_after();
        issue_s(0);
      }
      const int steps = 2 * nk;
      for (int i = 0; ok && i <= steps; ++i) {
        if (i + 1 < steps) {  // scores of step i + 1, once those of step i are in registers
          if ((i + 1) % 2 == 0) ok = landed((i + 1) / 2);
          ok = ok && mbar_wait(s_free, i & 1, p.err);
          if (!ok) break;
          tc_fence_after();
          issue_s(i + 1);
        }
        if (i > 0) {  // weights of step i - 1
          const int k = i - 1;
          ok = mbar_wait(p_full0 + 8u * (k & 1), (k >> 1) & 1, p.err);
          if (ok && k == steps - 2 && last_partial) ok = mbar_wait(v_fixed, 0, p.err);
          if (!ok) break;
          tc_fence_after();
          issue_o(k);
        }
      }
      tc_commit(done_bar);  // every product ends before its tensor memory is released
      mbar_wait(done_bar, 0, p.err);
    }
  } else if (warp == 2) {
    // -------------------------------------- V rows that no row of the tile sees
    if (last_partial) {
      int w = 1;
      if (lane == 0) w = mbar_wait(v_req, 0, p.err) ? 1 : 0;
      if (__shfl_sync(0xffffffffu, w, 0) != 0) {
        const int valid = tile.key1 - (tile.key0 + (nk - 1) * kTile);
        const uint32_t vb = sbase + kOffKV + ((nk - 1) % kStages) * kStageBytes + 2 * kQBytes;
        for (uint32_t a = 128u * valid + 16u * lane; a < static_cast<uint32_t>(kQBytes); a += 512u) {
          asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(vb + a), "r"(0u) : "memory");
          asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(vb + kQBytes + a), "r"(0u) : "memory");
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(v_fixed);
      }
    }
    }
  } else {
    // ------------------------------------------------------------ softmax
    regs_take();
    const int m = (warp - 4) >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lane_base = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t pa = lane_base + kColP + 64u * m, oa = lane_base + kColO + 128u * m;
    const bool live = row < rows;
    const int tok = tile.tok0 + row / p.pack;  // in the sequence
    const int limit = live ? min(tile.key1, key_limit(rec, tok, p.causal)) : 0;
    float mx = -INFINITY, l = 0.f;
    bool ok = nk > 0;
    if ((warp & 3) * 32 < rows) {
      const int least = __reduce_min_sync(0xffffffffu, live ? limit : 0x7fffffff);
      for (int j = 0; j < nk; ++j) {
        const int valid = limit - (tile.key0 + j * kTile);  // this row sees the first `valid` columns
        const bool full = least - (tile.key0 + j * kTile) >= kTile;
        if (!warp_wait(s_full0 + 8u * m, j & 1, p.err)) {
          ok = false;
          break;
        }
        tc_fence_after();
        float s[2][64];
        tmem_ld64x2(lane_base, lane_base + 64u, s[0], s[1]);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(s_free);
        if (!full) {
#pragma unroll
          for (int i = 0; i < kTile; ++i) s[i / 64][i % 64] = i < valid ? s[i / 64][i % 64] : -INFINITY;  // 2^-inf = 0
        }
        float mv[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) mv[k] = fmaxf(s[0][2 * k], s[0][2 * k + 1]);
#pragma unroll
        for (int i = 16; i < kTile; i += 2) mv[(i >> 1) & 7] = max3(mv[(i >> 1) & 7], s[i / 64][i % 64], s[i / 64][i % 64 + 1]);
        const float top = fmaxf(fmaxf(fmaxf(mv[0], mv[1]), fmaxf(mv[2], mv[3])),
                                fmaxf(fmaxf(mv[4], mv[5]), fmaxf(mv[6], mv[7]))) * p.scale_log2;
        const bool move = top > mx + kLift<T> + kRescale;  // true for the first visible key (mx = -inf)
        const float m_new = move ? top - kLift<T> : mx;
        const float alpha = move ? ex2_ftz(mx - m_new) : 1.f;
        // the product of this map's last step: O_m is complete and P_m is read
        if (j > 0) {
          if (!warp_wait(o_done0 + 8u * m, (j - 1) & 1, p.err)) {
            ok = false;
            break;
          }
          tc_fence_after();
          if (__any_sync(0xffffffffu, move)) {
#pragma unroll
            for (int q = 0; q < kDaDv / 16; ++q) {
              float o[16];
              uint32_t w[16];
              tmem_ld16(oa + q * 16, o);
#pragma unroll
              for (int i = 0; i < 16; ++i) w[i] = __float_as_uint(o[i] * alpha);
              tmem_st16(oa + q * 16, w);
            }
          }
        }
        unsigned long long sumv[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) sumv[k] = 0ull;
        const float base = m_new == -INFINITY ? 0.f : -m_new;  // no key seen yet: every weight is 2^-inf = 0
        const unsigned long long sc2 = f2(p.scale_log2, p.scale_log2), neg_m2 = f2(base, base);
#pragma unroll
        for (int c = 0; c < kTile / 32; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            float x0, x1;
            f2_split(fma_f2(f2(s[c / 2][32 * (c % 2) + i], s[c / 2][32 * (c % 2) + i + 1]), sc2, neg_m2), x0, x1);
            const float p0 = ex2_ftz(x0), p1 = ex2_ftz(x1);
            sumv[(i >> 1) & 3] = add_f2(sumv[(i >> 1) & 3], f2(p0, p1));
            pk[i / 2] = pack2<T>(p0, p1);
          }
          tmem_st16(pa + 16u * c, pk);
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full0 + 8u * m);
        float a, b;
        f2_split(add_f2(add_f2(sumv[0], sumv[1]), add_f2(sumv[2], sumv[3])), a, b);
        l = fmaf(l, alpha, a + b);
        mx = m_new;
      }
      ok = ok && warp_wait(o_done0 + 8u * m, (nk - 1) & 1, p.err);
      // the last product of a map is issued after every score product, so Q's
      // shared memory is free (warps without rows come here at once: they may not write)
      s_row[m * kTile + row] = make_float2(ok ? mx : -INFINITY, ok ? l : 0.f);
    }
    // each group writes half of the columns of both maps
    tc_fence_before();
    named_bar_sync(1, 256);
    tc_fence_after();
    const float2 r1 = s_row[row], r2 = s_row[kTile + row];
    if ((warp & 3) * 32 < rows) {
      const int head = h0 + row % p.pack;
      const int64_t qrow = static_cast<int64_t>(rec.q0) + tok;
      const int64_t at = live ? qrow * p.heads + head : 0;
      const bool join = tile.nsplit > 1;
      const int64_t part = (rec.part0 + static_cast<int64_t>(tile.split) * (rec.q1 - rec.q0) + tok) * p.heads + head;
      // a sum of 0: no key, or scores of -inf alone, which have no softmax; a NaN sum goes through
      const float none = live && !join && key_limit(rec, tok, p.causal) > 0 ? NAN : 0.f;
      const float i1 = join ? 1.f : 1.f / r1.y, i2 = join ? 1.f : 1.f / r2.y;
      const float lam = live ? p.lam.get(head) : 0.f;
      if (live && join && m == 0)
        p.part_ml[part] = make_float4(r1.x, r1.y, r2.x, r2.y);
      if (live && !join && p.lse) {
        const float2 r = m ? r2 : r1;
        p.lse[(static_cast<int64_t>(m) * p.heads + head) * p.nq + qrow] =
            r.y != 0.f ? r.x + log2f(r.y) : none != 0.f ? NAN : INFINITY;
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float o1[32], o2[32];
        __syncwarp();
        if (nk > 0) {
          tmem_ld32(lane_base + kColO + 64u * m + 32u * c, o1);
          tmem_ld32(lane_base + kColO + 128u + 64u * m + 32u * c, o2);
        }
        const int d = 64 * m + 32 * c;
        // without a sum the columns may never have been written
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          o1[i] = r1.y != 0.f ? o1[i] * i1 : none;
          o2[i] = r2.y != 0.f ? o2[i] * i2 : none;
        }
        float* f32 = join ? p.part_o + part * (2 * kDaDv) : p.maps ? p.maps + at * (2 * kDaDv) : nullptr;
        if (live && f32) {
          float4* dst = reinterpret_cast<float4*>(f32 + d);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            dst[i] = make_float4(o1[4 * i], o1[4 * i + 1], o1[4 * i + 2], o1[4 * i + 3]);
            dst[kDaDv / 4 + i] = make_float4(o2[4 * i], o2[4 * i + 1], o2[4 * i + 2], o2[4 * i + 3]);
          }
        }
        if (live && !join) {
          uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(p.out) + at * kDaDv + d);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int e = 8 * i + 2 * k;
              w[k] = pack2<T>(fmaf(-lam, o2[e], o1[e]), fmaf(-lam, o2[e + 1], o1[e + 1]));
            }
            dst[i] = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
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

// Joins the key ranges of the rows whose sequence was cut: one warp per
// (row, head), ranges in ascending order.
template <typename T>
__global__ void __launch_bounds__(128) k_da_join(const DaFwd p, const __grid_constant__ SeqPlan plan, int nrec) {
  const int64_t at = blockIdx.x * 4ll + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (at >= p.nq * p.heads) return;
  const int row = static_cast<int>(at / p.heads), h = static_cast<int>(at % p.heads);
  asm volatile("griddepcontrol.wait;" ::: "memory");  // launched before k_da_fwd ends
  int rec = 0;
  for (int base = 0; base < nrec; base += 32) {  // records are sorted by key count, not by row
    const int i = base + lane;
    const bool hit = i < nrec && plan.at(i).q0 <= row && row < plan.at(i).q1;
    const unsigned who = __ballot_sync(0xffffffffu, hit);
    if (who) {
      rec = base + __ffs(who) - 1;
      break;
    }
  }
  const SeqRec& r = plan.at(rec);
  const int nsplit = max(1, (r.k1 - r.k0 + p.split_keys - 1) / p.split_keys);
  if (nsplit == 1) return;
  const int64_t step = static_cast<int64_t>(r.q1 - r.q0) * p.heads;
  const int64_t part = (r.part0 + static_cast<int64_t>(row - r.q0)) * p.heads + h;
  float m1 = -INFINITY, m2 = -INFINITY, l1 = 0.f, l2 = 0.f, o1[4] = {}, o2[4] = {};
  for (int s0 = 0; s0 < nsplit; s0 += 32) {  // lane = range
    const int ns = min(32, nsplit - s0);
    const float4 ml = lane < ns ? p.part_ml[(s0 + lane) * step + part] : make_float4(-INFINITY, 0.f, -INFINITY, 0.f);
    float t1 = ml.x, t2 = ml.z;
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) {
      t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, x));
      t2 = fmaxf(t2, __shfl_xor_sync(0xffffffffu, t2, x));
    }
    const float n1 = fmaxf(m1, t1), n2 = fmaxf(m2, t2);
    const float a1 = m1 > -INFINITY ? exp2f(m1 - n1) : 0.f, a2 = m2 > -INFINITY ? exp2f(m2 - n2) : 0.f;
    // a range without a sum has weight 0; a NaN sum goes through
    const float w1 = ml.y != 0.f ? exp2f(ml.x - n1) : 0.f, w2 = ml.w != 0.f ? exp2f(ml.z - n2) : 0.f;
    float s1 = w1 * ml.y, s2 = w2 * ml.w;
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) {
      s1 += __shfl_xor_sync(0xffffffffu, s1, x);
      s2 += __shfl_xor_sync(0xffffffffu, s2, x);
    }
    l1 = fmaf(l1, a1, s1);
    l2 = fmaf(l2, a2, s2);
    m1 = n1;
    m2 = n2;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      o1[e] *= a1;
      o2[e] *= a2;
    }
#pragma unroll 4
    for (int s = 0; s < ns; ++s) {
      const float* o = p.part_o + ((s0 + s) * step + part) * (2 * kDaDv) + 4 * lane;
      const float4 a = *reinterpret_cast<const float4*>(o), b = *reinterpret_cast<const float4*>(o + kDaDv);
      const float u1 = __shfl_sync(0xffffffffu, w1, s), u2 = __shfl_sync(0xffffffffu, w2, s);
      const float av[4] = {a.x, a.y, a.z, a.w}, bv[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        o1[e] = fmaf(u1, av[e], o1[e]);
        o2[e] = fmaf(u2, bv[e], o2[e]);
      }
    }
  }
  // a sum of 0: no key, or scores of -inf alone, which have no softmax
  const float none = key_limit(r, row - r.q0, p.causal) > 0 ? NAN : 0.f;
  const float i1 = l1 != 0.f ? 1.f / l1 : none, i2 = l2 != 0.f ? 1.f / l2 : none, lam = p.lam.get(h);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    o1[e] *= i1;
    o2[e] *= i2;
  }
  if (p.lse && lane < 2) {
    const float l = lane ? l2 : l1;
    p.lse[(static_cast<int64_t>(lane) * p.heads + h) * p.nq + row] =
        l != 0.f ? (lane ? m2 : m1) + log2f(l) : none != 0.f ? NAN : INFINITY;
  }
  if (p.maps) {
    float* dst = p.maps + at * (2 * kDaDv) + 4 * lane;
    *reinterpret_cast<float4*>(dst) = make_float4(o1[0], o1[1], o1[2], o1[3]);
    *reinterpret_cast<float4*>(dst + kDaDv) = make_float4(o2[0], o2[1], o2[2], o2[3]);
  }
  uint2 w;
  w.x = pack2<T>(fmaf(-lam, o2[0], o1[0]), fmaf(-lam, o2[1], o1[1]));
  w.y = pack2<T>(fmaf(-lam, o2[2], o1[2]), fmaf(-lam, o2[3], o1[3]));
  reinterpret_cast<uint2*>(static_cast<T*>(p.out) + at * kDaDv)[lane] = w;
}

template <typename T>
sc_status run_forward(Handle* h, const DaArgs& a) {
  const bool bf16 = std::is_same_v<T, __nv_bfloat16>;
  const int64_t nq = a.cu_q[a.batch], nkv = a.cu_kv[a.batch];
  const int rep = a.heads / a.kv_heads;
  DaFwd p{};
  p.lam = LamRef{a.lam, a.lam_count, a.lam_dtype, a.lam_value};
  p.out = a.out;
  p.lse = a.lse;
  p.maps = a.maps;
  p.nq = nq;
  p.heads = a.heads;
  p.rep = rep;
  p.pack = rep <= kTile ? rep : 1;
  p.tokens = kTile / p.pack;
  p.causal = a.causal;
  p.scale_log2 = a.scale * kLog2e;
  p.err = h->derr;
  const int groups = a.heads / p.pack;
  // Work in key tiles; keys are cut into ranges only where whole tiles of rows
  // would leave SMs without a CTA.  About two ranges per SM: at 24 single tokens
  // against 513 to 16,084 keys 1 / 2 / 3 / 4 / 8 took 109 / 100 / 103 / 110 / 128 us.
  std::vector<SeqRec> recs;
  int64_t tiles = 0, work = 0;
  int32_t longest = 0;
  for (int b = 0; b < a.batch; ++b) {
    const int32_t lq = a.cu_q[b + 1] - a.cu_q[b], lk = a.cu_kv[b + 1] - a.cu_kv[b];
    if (lq == 0) continue;
    const int32_t t = (lq + p.tokens - 1) / p.tokens;
    recs.push_back(SeqRec{a.cu_q[b], a.cu_q[b + 1], a.cu_kv[b], a.cu_kv[b + 1], 0, t});
    tiles += static_cast<int64_t>(t) * groups;
    work += static_cast<int64_t>(t) * groups * ((lk + kTile - 1) / kTile);
    longest = std::max(longest, lk);
  }
  p.split_keys = std::max(kTile, (longest + kTile - 1) / kTile * kTile);
  if (tiles < 2 * h->num_sms) {
    const int64_t want = (work + 2ll * h->num_sms - 1) / (2ll * h->num_sms);
    // four tiles at least: a shorter range costs less than the join
    p.split_keys = static_cast<int>(std::min<int64_t>(p.split_keys, std::max<int64_t>(4, want) * kTile));
  }
  // the longest first: the tail of the launch is made of short CTAs
  std::stable_sort(recs.begin(), recs.end(),
                   [](const SeqRec& x, const SeqRec& y) { return x.k1 - x.k0 > y.k1 - y.k0; });
  int64_t items = 0, parts = 0;
  for (SeqRec& r : recs) {
    const int64_t s = std::max(1, (r.k1 - r.k0 + p.split_keys - 1) / p.split_keys);
    r.item0 = static_cast<int32_t>(items);
    r.part0 = static_cast<int32_t>(parts);
    items += r.aux * s;
    if (s > 1) parts += s * (r.q1 - r.q0);
  }
  if (items > 0x7fffffff || parts > 0x7fffffff || groups > 65535) return set_error(h, SC_EINVAL, "differential attention: too many tiles");
  // q as [64][2 maps][heads][tokens], k as [64][2 kv heads][tokens], v as [128][kv heads][tokens]
  CUtensorMap tq, tk, tv;
  const uint64_t one = 1;
  const uint64_t dq[4] = {kDaD, 2, static_cast<uint64_t>(a.heads), static_cast<uint64_t>(std::max<int64_t>(nq, 1))};
  const uint64_t sq[3] = {kDaD * 2, kDaD * 4, static_cast<uint64_t>(a.qs) * 2};
  const uint32_t bq[4] = {kDaD, 1, static_cast<uint32_t>(p.pack), static_cast<uint32_t>(p.tokens)};
  const uint64_t rk = std::max<uint64_t>(static_cast<uint64_t>(nkv), one);
  const uint64_t dk[3] = {kDaD, 2ull * a.kv_heads, rk}, dv[3] = {kDaDv, static_cast<uint64_t>(a.kv_heads), rk};
  const uint64_t none = 128ull * a.kv_heads;  // without keys: any stride a map takes
  const uint64_t sk[2] = {kDaD * 2, (nkv > 0 ? static_cast<uint64_t>(a.ks) : none) * 2},
                 sv[2] = {kDaDv * 2, (nkv > 0 ? static_cast<uint64_t>(a.vs) : none) * 2};
  const uint32_t bk[3] = {kDaD, 1, kTile};
  // without keys no tile of them is read, but the maps want an address
  const void* k = nkv > 0 ? a.k : a.q;
  const void* v = nkv > 0 ? a.v : a.q;
  if (!make_map_nd(&tq, bf16, a.q, 4, dq, sq, bq) || !make_map_nd(&tk, bf16, k, 3, dk, sk, bk) ||
      !make_map_nd(&tv, bf16, v, 3, dv, sv, bk))
    return set_error(h, SC_ECUDA, "cuTensorMapEncodeTiled failed (differential attention)");
  SeqPlan plan;
  DevBuf table(h), ws(h);
  const sc_status st = make_plan(h, recs, &plan, &table.p);
  if (st != SC_OK) return st;
  cudaError_t e = cudaSuccess;
  if (parts > 0) {
    const size_t n = static_cast<size_t>(parts) * a.heads;
    e = dev_alloc(h, &ws.p, n * (2 * kDaDv * sizeof(float) + sizeof(float4)));
    if (e != cudaSuccess) return cuda_error(h, e, "differential attention workspace");
    p.part_o = static_cast<float*>(ws.p);
    p.part_ml = reinterpret_cast<float4*>(static_cast<char*>(ws.p) + n * 2 * kDaDv * sizeof(float));
  }
  e = cudaFuncSetAttribute(k_da_fwd<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
  if (e == cudaSuccess) {
    ++h->launches;
    k_da_fwd<T><<<dim3(static_cast<unsigned>(items), groups), kThreads, kSmem, h->stream>>>(tq, tk, tv, p, plan);
    if (parts > 0) {
      ++h->launches;
      cudaLaunchConfig_t cfg{};
      cfg.gridDim = dim3(static_cast<unsigned>((nq * a.heads + 3) / 4));
      cfg.blockDim = dim3(128);
      cfg.stream = h->stream;
      cudaLaunchAttribute at[1];
      at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
      at[0].val.programmaticStreamSerializationAllowed = 1;
      cfg.attrs = at;
      cfg.numAttrs = 1;
      e = cudaLaunchKernelEx(&cfg, k_da_join<T>, p, plan, static_cast<int>(recs.size()));
    }
    if (e == cudaSuccess) e = cudaGetLastError();
  }
  return e == cudaSuccess ? SC_OK : cuda_error(h, e, "differential attention launch");
}

}  // namespace

sc_status diff_attention(Handle* h, const DaArgs& a) {
  return a.dtype == SC_BF16 ? run_forward<__nv_bfloat16>(h, a) : run_forward<__half>(h, a);
}

}  // namespace sc
