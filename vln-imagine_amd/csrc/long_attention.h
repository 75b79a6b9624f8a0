// Shared by the long_attention*.hip files: one instance of the kernels per type, the entry points in long_attention.hip.
#pragma once
#include <type_traits>

#include "common.h"

constexpr float LA_LOG2E = 1.4426950408889634f;
constexpr float LA_MOST = 1e30f;             // finite masks beyond +- this count as this
constexpr float LA_EXACT = 1048576.f;        // a row whose maximum is larger than this rounds its scores before the maximum is taken off them
constexpr float LA_FOLD = 64.f;              // a row whose maximum (in units of log2) is larger than this keeps 1 / sum apart from it
constexpr int LA_PAD = 96;                   // a 32 x 64 piece that touches distance R reaches at most 94 beyond it
constexpr int LA_MAXB = 64;                  // buckets per side

struct LaP {
  const void *q, *k, *v, *dout;
  long q_b, q_s, q_h, k_b, k_s, k_h, v_b, v_s, v_h, d_b, d_s, d_h;      // strides in elements
  void *out, *low;             // [B, Sq, nh, D] each: the result, and what its rounding to 16 bits took (null: nobody wants it)
  float* lse; float* rl;       // [B, nh, Sq] each: see the masks' comment in long_attention_impl.inc
  float* delta;                // [B, nh, Sq] (float16: times la_range's factor of the sample and key head)
  float* range;                // [2][B, nkv][nch]: largest |v| and |dout| by piece of the positions; float16 only
  const float* kml;            // [B, SkP] mask in units of log2, -inf behind Sk; null without a mask
  const int* kind;             // [B, SkP / 64]: 0 no mask in these 64 keys, 1 finite values, 2 nothing but -inf, 3 some -inf
  const float* bvec;           // [nh, BL] bias by distance in units of log2, saturated LA_PAD beyond +-R; null without a bias
  float* part; float* part_ml; // split launches: float32 partial results; running (maximum, sum)
  void *dq, *dk, *dv;
  float* rowsum;               // [splits][5][B, nh, Sq] sums of a row's dS and P (see la_dq_kernel), null without a table gradient
  float* dbpart;               // [nh][B * row blocks][BL] sums of dS by distance
  int B, Sq, Sk, SkP, nh, nkv, D, causal, PG, R, BL, nblk, nsplit, zrow, nch;
  float c1, scale;             // c1 = scale log2(e)
};


// what: 0 forward, 1 (float16: ranges) dQ + delta + dS by distance, 2 dK + dV; each with the join of its splits
int la_run_bf16(const LaP& p, int what, hipStream_t st);
int la_run_f16(const LaP& p, int what, hipStream_t st);
int la_run_f32(const LaP& p, int what, hipStream_t st);
