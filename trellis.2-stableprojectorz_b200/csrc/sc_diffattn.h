// Differential attention: arguments shared by its translation units.
#pragma once
#include <cstdint>
#include "sc_internal.h"

namespace sc {

constexpr int kDaD = 64;    // query / key dims of one map
constexpr int kDaDv = 128;  // value dims

// One call.  Rows are tokens; strides are in elements between tokens.  Head h
// reads key / value head g = h / (heads / kv_heads); its two maps are q rows
// 2h, 2h + 1 against k rows 2g, 2g + 1.
struct DaArgs {
  const void *q, *k, *v;
  int64_t qs, ks, vs;
  const void* lam;        // [lam_count] in lam_dtype, or null: lam_value
  int lam_count;          // 1 (every head) or heads
  int lam_dtype;
  float lam_value;
  void* out;              // [Nq, heads, 128]
  float* lse;             // [2][heads][Nq] or null: log2 sum 2^(s log2 e) of every row and map, +inf without
                          // keys, NaN where a score is NaN or +inf or every one is -inf
  float* maps;            // [Nq, heads, 2, 128] or null: O_1 and O_2 of every row.  f32: dO . O_m is subtracted from
                          // every score gradient of its row, and with O_m rounded to bf16 that one error, common to
                          // the row's keys, made up most of dq's (0.0039 relative at 8,192 keys, 0.0017 without)
  const int32_t *cu_q, *cu_kv;  // host
  int batch, heads, kv_heads;
  float scale;
  int causal;             // query i of a sequence sees keys j <= i + len_kv - len_q
  sc_dtype dtype;
  // backward
  const void* dout;       // [Nq, heads, 128]
  void *dq, *dk, *dv;     // dense, or null
  void* dlam;             // [lam_count] in lam_dtype, or null
};

sc_status diff_attention(Handle* h, const DaArgs& a);           // sc_diffattn.cu
sc_status diff_attention_backward(Handle* h, const DaArgs& a);  // sc_diffattn_bwd.cu

}  // namespace sc
