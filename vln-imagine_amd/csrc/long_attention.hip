// Entry points of attention over long sequences (ops.long_attention), its mask / bias preparation and the bfloat16 instances.
// The kernels and the mathematics are in long_attention_impl.inc.
#include <limits.h>
#include <math.h>

#include "../../include/vlni.h"
#include "long_attention.h"

#include "long_attention_impl.inc"

int la_run_bf16(const LaP& p, int what, hipStream_t st) { return la_run<__bf16>(p, what, st); }

namespace {

// first[b]: smallest distance of a side's bucket b; table rows [0, n) for keys at or before the query, [n, 2 n) for keys behind it (two sides)
struct LaBuckets {
  int n, sides, first[LA_MAXB];
};
__device__ __forceinline__ int la_bucket(const LaBuckets& k, int rel) {
  const int d = rel < 0 ? -rel : k.sides == 2 ? rel : 0;
  int b = 0;
  for (int e = 1; e < k.n; ++e) b += d >= k.first[e];
  return b + (k.sides == 2 && rel > 0 ? k.n : 0);
}

// blocks [0, B SkP / 64): 64 keys of the mask to units of log2, and their kind; the rest: the bias by distance, one block = 64 distances of a head
__global__ __launch_bounds__(64) void la_prep_kernel(const float* kmask, const float* table, float* kml, int* kind, float* bvec, LaBuckets k, int B,
                                                     int Sk, int SkP, int nh, int R, int BL) {
  const int nmask = kmask ? B * (SkP >> 6) : 0, lane = threadIdx.x;
  if ((int)blockIdx.x < nmask) {
    const int b = blockIdx.x / (SkP >> 6), j = (blockIdx.x % (SkP >> 6)) * 64 + lane;
    float v = -INFINITY;
    if (j < Sk) {
      v = kmask[(long)b * Sk + j];
      if (fabsf(v) != INFINITY) v = (v < -LA_MOST ? -LA_MOST : v > LA_MOST ? LA_MOST : v) * LA_LOG2E;      // (NaN stays)
    }
    kml[(long)b * SkP + j] = v;
    const bool none = __all(v == 0.f), all = __all(v == -INFINITY), some = __any(v == -INFINITY);
    if (lane == 0) kind[blockIdx.x] = none ? 0 : all ? 2 : some ? 3 : 1;
  } else {
    const int per = (BL + 63) / 64, w = blockIdx.x - nmask, h = w / per, e = (w % per) * 64 + lane;
    if (e >= BL) return;
    const int rel = max(-R, min(R, e - R - LA_PAD));
    bvec[(long)h * BL + e] = table[(long)la_bucket(k, rel) * nh + h] * LA_LOG2E;
  }
}

// dtable[bucket][head] = sum of dS over the bucket's distances and all partial rows of the head; block = one (bucket, head), in a
// fixed order and in 64 bits
__global__ __launch_bounds__(256) void la_dtable_kernel(const float* part, float* dtable, LaBuckets k, int nh, int R, int BL, int nparts) {
  const int b = blockIdx.x, h = blockIdx.y, side = b / k.n, bb = b % k.n;
  const int d0 = k.first[bb], d1 = bb + 1 < k.n ? k.first[bb + 1] - 1 : INT_MAX;       // distances d0 .. d1 (none: d1 < d0)
  int e0, e1;                                                                          // entries of this bucket, e = rel + R + LA_PAD
  if (k.sides == 2 && side == 1) {
    e0 = R + LA_PAD + max(d0, 1);
    e1 = d1 == INT_MAX ? BL - 1 : min(BL - 1, R + LA_PAD + d1);
  } else {
    e0 = d1 == INT_MAX ? 0 : max(0, R + LA_PAD - d1);
    e1 = k.sides == 1 && d0 == 0 && d1 >= 0 ? BL - 1 : R + LA_PAD - d0;
  }
  double a = 0.0;
  const int lg = e1 - e0 >= 128 ? 8 : e1 - e0 >= 64 ? 7 : e1 - e0 >= 32 ? 6 : 5;       // 2^lg distances side by side
  for (int e = e0 + (threadIdx.x & ((1 << lg) - 1)); e <= e1; e += 1 << lg) {
    const float* col = part + (long)h * nparts * BL + e;
#pragma unroll 8
    for (int q = threadIdx.x >> lg; q < nparts; q += 256 >> lg) a += (double)col[(long)q * BL];
  }
  __shared__ double s[256];
  s[threadIdx.x] = a;
  __syncthreads();
  for (int o = 128; o > 0; o >>= 1) {
    if ((int)threadIdx.x < o) s[threadIdx.x] += s[threadIdx.x + o];
    __syncthreads();
  }
  if (threadIdx.x == 0) dtable[(long)b * nh + h] = (float)s[0];
}

int la_fill(const VlniLongAttnArgs* a, LaP& p, LaBuckets& k) {
  VLNI_CHECK(a && a->dtype >= VLNI_F32 && a->dtype <= VLNI_F16, VLNI_EINVAL, "long_attn: dtype %d", a ? a->dtype : -1);
  VLNI_CHECK(a->B > 0 && a->Sq > 0 && a->Sk > 0 && a->nh > 0 && a->nkv > 0, VLNI_EINVAL, "long_attn: B=%d Sq=%d Sk=%d nh=%d nkv=%d", a->B, a->Sq,
             a->Sk, a->nh, a->nkv);
  VLNI_CHECK(a->Sq <= (1 << 24) && a->Sk <= (1 << 24), VLNI_EUNSUP, "long_attn: Sq=%d Sk=%d (at most 2^24)", a->Sq, a->Sk);
  VLNI_CHECK(a->nh % a->nkv == 0 && a->nh <= 1024, VLNI_EINVAL, "long_attn: nh=%d is not a multiple of nkv=%d (at most 1024 heads)", a->nh, a->nkv);
  VLNI_CHECK(a->D >= 8 && a->D <= 128 && a->D % 8 == 0, VLNI_EUNSUP, "long_attn: head size %d (a multiple of 8 up to 128)", a->D);
  VLNI_CHECK(a->scale > 0.f && a->scale < 1e6f, VLNI_EINVAL, "long_attn: scale %g", (double)a->scale);
  p = LaP{};
  k = LaBuckets{};
  p.B = a->B; p.Sq = a->Sq; p.Sk = a->Sk; p.SkP = (a->Sk + 63) & ~63; p.nh = a->nh; p.nkv = a->nkv; p.D = a->D; p.causal = a->causal != 0;
  p.scale = a->scale; p.c1 = a->scale * LA_LOG2E;
  if (a->rel_table) {
    k.n = a->rel_n; k.sides = a->rel_sides;
    VLNI_CHECK((k.sides == 1 || k.sides == 2) && k.n >= 1 && k.n <= LA_MAXB && a->rel_first, VLNI_EINVAL, "long_attn: %d buckets on %d sides", k.n, k.sides);
    for (int e = 0; e < k.n; ++e) {
      k.first[e] = a->rel_first[e];
      VLNI_CHECK(e == 0 ? k.first[e] == 0 : k.first[e] >= k.first[e - 1], VLNI_EINVAL, "long_attn: bucket %d begins at %d", e, k.first[e]);
    }
    p.R = k.first[k.n - 1] < 1 ? 1 : k.first[k.n - 1];
    VLNI_CHECK(p.R <= 1024, VLNI_EUNSUP, "long_attn: the last bucket begins at distance %d (at most 1024)", p.R);
    p.BL = 2 * p.R + 1 + 2 * LA_PAD;
  }
  // float16: pieces of la_range_kernel, at most one a lane and at least 1024 reads of 16 bytes each
  const long reads = (a->Sk > (long)a->Sq * (a->nh / a->nkv) ? a->Sk : (long)a->Sq * (a->nh / a->nkv)) * (a->D / 8);
  p.nch = a->dtype != VLNI_F16 ? 0 : reads >= 65536 ? 64 : reads <= 1024 ? 1 : (int)(reads / 1024);
  // a few rows that share keys are worked on side by side (row = position x head of the group): one pass over K and V instead of one per head.
  // A bias differs by head, so its launches keep the heads apart.
  p.PG = !a->rel_table && (long)a->Sq * (a->nh / a->nkv) <= 128 ? a->nh / a->nkv : 1;
  return VLNI_OK;
}

// Splits of a launch along its loop, by what they cost and save. `blocks` blocks walk up to `chain` tiles each; a tile costs a CU `us` microseconds where
// other blocks fill its waits, and `alone` pass before a block begins its next one.
// Without a causal border all blocks are alike and run in rounds of one block a CU - two where a few rows leave the loads of K and V as the bound
// (latency: a second block's loads fly under the first one's). With one, the chip works through half of the tiles on average (`part`) but waits for the
// end of the longest chain. Splits cost a launch and their partial results, float32, written and read again at 4.5 TB/s.
// Measured (heads of 64, whole -> split, with what joins them): dK / dV of a causal 4 k pass with four key heads, 256 blocks: 406 us -> in four 129 + 11;
// 3 x 1501 causal positions of 8 heads with a bias, 288 blocks, forward: 42 -> in three 27 + 9; 1024 positions of 12 heads, 96 blocks, forward: 25 -> in
// four 15 + 5; 2 x 512: 14 -> in two 12 + 5, so not split. A token over 8 k keys, 64 blocks of heads of 128: in eight 45 + 5, in 25 71.
int la_split(double blocks, double chain, double part, bool few, const double (&tile)[2], double floats) {
  int best = 1;
  double least = 1e300;
  const double us = tile[0], alone = tile[1], slots = few ? 512.0 : 256.0;
  for (int n = 1; n <= 32 && (n == 1 || chain / n >= 2.0); ++n) {
    const double one = ceil(chain / n), all = us * (part < 1.0 ? blocks * n * one * part / 256.0 + 0.3 * one : slots / 256.0 * ceil(blocks * n / slots) * one);
    const double t = (!few && alone * one > all ? alone * one : all) + (n > 1 ? 5.0 + n * floats * 8.0 / 4.5e6 : 0.0);
    if (t < 0.98 * least) { best = n; least = t; }
  }
  return best;
}
int la_kt_of(const VlniLongAttnArgs* a) { return a->dtype == VLNI_F32 && a->D > 64 ? 32 : 64; }
// `us` and `alone` of a tile, for rows (forward, dQ) or keys (dK / dV): measured at D = 64 and, in 16 bits, half of it with a head's size; float32's
// products leave other blocks nothing to fill
void la_tile(const VlniLongAttnArgs* a, bool keys, double (&tile)[2]) {
  const int dp = (a->D + 31) / 32 * 32;
  if (a->dtype == VLNI_F32) tile[0] = tile[1] = (keys ? 10.5 : 6.0) * dp / 64 * la_kt_of(a) / 64;
  else {
    tile[0] = (keys ? 1.2 : 0.72) * (64 + dp) / 128;
    tile[1] = (keys ? 2.4 : 1.7) * (64 + dp) / 128;
  }
}
double la_part(const LaP& p) { return p.causal && p.PG == 1 && p.Sq > 64 ? (p.Sk - 0.5 * (p.Sq < p.Sk ? p.Sq : p.Sk)) / p.Sk : 1.0; }
void la_grid_rows(const VlniLongAttnArgs* a, LaP& p) {
  double tile[2];
  la_tile(a, false, tile);
  p.nblk = cdiv((long)p.Sq * p.PG, 128);
  p.nsplit = la_split((double)p.nblk * p.B * (p.nh / p.PG), cdiv(p.Sk, la_kt_of(a)), la_part(p), p.Sq * p.PG <= 32, tile, (double)p.B * p.Sq * p.nh * p.D);
}
void la_grid_keys(const VlniLongAttnArgs* a, LaP& p) {
  double tile[2];
  la_tile(a, true, tile);
  p.nblk = cdiv(p.Sk, 128);
  p.nsplit = la_split((double)p.nblk * p.B * p.nkv, (double)cdiv((long)p.Sq * p.PG, la_kt_of(a)) * (p.nh / p.nkv / p.PG), la_part(p), false, tile,
                      2.0 * p.B * p.Sk * p.nkv * p.D);
}
long la_prep_floats(const VlniLongAttnArgs* a, const LaP& p) {
  return (a->kmask ? (long)p.B * p.SkP + (long)p.B * (p.SkP >> 6) : 0) + (a->rel_table ? (long)p.nh * p.BL : 0);
}
void la_prep_pointers(const VlniLongAttnArgs* a, LaP& p) {
  float* f = (float*)a->prep;
  if (a->kmask) {
    p.kml = f;
    p.kind = (const int*)(f + (long)p.B * p.SkP);
    f += (long)p.B * p.SkP + (long)p.B * (p.SkP >> 6);
  }
  if (a->rel_table) p.bvec = f;
}
// floats of workspace: forward: split results; backward: delta, ranges (float16), row sums, sums by distance, split results (of dQ, then of dK and dV)
long la_fwd_work(const VlniLongAttnArgs* a, LaP p) {
  la_grid_rows(a, p);
  const long n = (long)p.B * p.Sq * p.nh;
  return p.nsplit > 1 ? p.nsplit * n * (p.D + 2) : 0;
}
long la_bwd_work(const VlniLongAttnArgs* a, LaP p, long* o_rs, long* o_db, long* o_part) {
  const long n = (long)p.B * p.Sq * p.nh;
  long f = (n + 3) & ~3L;
  f += 2L * p.nch * p.B * p.nkv;
  f = (f + 3) & ~3L;
  la_grid_rows(a, p);
  *o_rs = f;
  if (a->rel_table) f += 5 * p.nsplit * n;
  *o_db = f;
  if (a->rel_table) f += (long)p.nh * p.B * p.nblk * p.BL;
  f = (f + 3) & ~3L;
  *o_part = f;
  long part = p.nsplit > 1 ? p.nsplit * n * p.D : 0;
  la_grid_keys(a, p);
  if (p.nsplit > 1) {
    const long kv = 2L * p.nsplit * p.B * p.Sk * p.nkv * p.D;
    part = part > kv ? part : kv;
  }
  return f + part;
}
int la_operand(const char* what, const void* ptr, const long* s, int dtype) {
  const int al = dtype == VLNI_F32 ? 4 : 8;
  VLNI_CHECK(ptr && (uintptr_t)ptr % 16 == 0, VLNI_EINVAL, "long_attn: %s is %s", what, ptr ? "not 16-byte aligned" : "null");
  VLNI_CHECK(s[0] % al == 0 && s[1] % al == 0 && s[2] % al == 0, VLNI_EINVAL, "long_attn: strides %ld, %ld, %ld of %s are not multiples of 16 bytes", s[0],
             s[1], s[2], what);
  return VLNI_OK;
}
// a launch has less than 2^32 threads: 2^24 blocks of 256 rows' or keys' work, of the joins, and of 64 for the mask
int la_limits(const VlniLongAttnArgs* a, LaP p) {
  la_grid_rows(a, p);
  const long rows = (long)p.nblk * p.nsplit * p.B * (p.nh / p.PG), row4 = p.nsplit > 1 ? (long)p.B * p.Sq * p.nh * p.D / 4 : 0;
  la_grid_keys(a, p);
  const long keys = (long)p.nblk * p.nsplit * p.B * p.nkv, key4 = p.nsplit > 1 ? (long)p.B * p.Sk * p.nkv * p.D / 2 : 0;
  const long prep = (a->kmask ? (long)p.B * (p.SkP >> 6) : 0) + (a->rel_table ? (long)p.nh * cdiv(p.BL, 64) : 0);
  VLNI_CHECK(rows < (1L << 24) && keys < (1L << 24) && prep < (1L << 26) && row4 < 0xFFFFFF00L && key4 < 0xFFFFFF00L, VLNI_EUNSUP,
             "long_attn: B=%d Sq=%d Sk=%d nh=%d nkv=%d is more than one launch holds (%ld and %ld blocks, at most 2^24 - 1)", p.B, p.Sq, p.Sk, p.nh, p.nkv,
             rows, keys);
  return VLNI_OK;
}
int la_go(const VlniLongAttnArgs* a, const LaP& p, int what, hipStream_t st) {
  return a->dtype == VLNI_F32 ? la_run_f32(p, what, st) : a->dtype == VLNI_BF16 ? la_run_bf16(p, what, st) : la_run_f16(p, what, st);
}
}  // namespace

#define LA_TRY(x) do { const int rc_ = (x); if (rc_ != VLNI_OK) return rc_; } while (0)

extern "C" int vlni_long_attn_sizes(const VlniLongAttnArgs* a, long* sizes) {
  LaP p; LaBuckets k;
  LA_TRY(la_fill(a, p, k));
  LA_TRY(la_limits(a, p));
  long o1, o2, o3;
  sizes[0] = la_prep_floats(a, p);
  sizes[1] = la_fwd_work(a, p);
  sizes[2] = la_bwd_work(a, p, &o1, &o2, &o3);
  return VLNI_OK;
}

extern "C" int vlni_long_attn_fwd(const VlniLongAttnArgs* a, void* stream) {
  LaP p; LaBuckets k;
  LA_TRY(la_fill(a, p, k));
  LA_TRY(la_limits(a, p));
  LA_TRY(la_operand("q", a->q, a->q_stride, a->dtype));
  LA_TRY(la_operand("k", a->k, a->k_stride, a->dtype));
  LA_TRY(la_operand("v", a->v, a->v_stride, a->dtype));
  VLNI_CHECK(a->out && a->stat && ((uintptr_t)a->out | (uintptr_t)a->out_low) % 16 == 0, VLNI_EINVAL, "long_attn: out %p, out_low %p, stat %p", a->out,
             a->out_low, (void*)a->stat);
  const long n = (long)p.B * p.Sq * p.nh;
  const long need = la_prep_floats(a, p), work = la_fwd_work(a, p);
  VLNI_CHECK(!need || (a->prep && a->prep_floats >= need), VLNI_EINVAL, "long_attn: prep holds %ld floats, %ld are needed", a->prep ? a->prep_floats : 0, need);
  VLNI_CHECK(!work || (a->work && a->work_floats >= work && (uintptr_t)a->work % 16 == 0), VLNI_EINVAL, "long_attn: work holds %ld floats, %ld are needed",
             a->work ? a->work_floats : 0, work);
  const hipStream_t st = (hipStream_t)stream;
  la_prep_pointers(a, p);
  if (need) {
    const long blocks = (a->kmask ? (long)p.B * (p.SkP >> 6) : 0) + (a->rel_table ? (long)p.nh * cdiv(p.BL, 64) : 0);
    hipLaunchKernelGGL(la_prep_kernel, dim3((unsigned)blocks), dim3(64), 0, st, a->kmask, a->rel_table, (float*)p.kml, (int*)p.kind, (float*)p.bvec, k, p.B,
                       p.Sk, p.SkP, p.nh, p.R, p.BL);
    VLNI_LAUNCH_CHECK();
  }
  p.q = a->q; p.k = a->k; p.v = a->v;
  p.q_b = a->q_stride[0]; p.q_s = a->q_stride[1]; p.q_h = a->q_stride[2];
  p.k_b = a->k_stride[0]; p.k_s = a->k_stride[1]; p.k_h = a->k_stride[2];
  p.v_b = a->v_stride[0]; p.v_s = a->v_stride[1]; p.v_h = a->v_stride[2];
  p.out = a->out; p.low = a->dtype == VLNI_F32 ? nullptr : a->out_low; p.lse = a->stat; p.rl = a->stat + n;
  la_grid_rows(a, p);
  p.part = (float*)a->work;
  p.part_ml = p.part + (long)p.nsplit * n * p.D;
  return la_go(a, p, 0, st);
}

extern "C" int vlni_long_attn_bwd(const VlniLongAttnArgs* a, void* stream) {
  LaP p; LaBuckets k;
  LA_TRY(la_fill(a, p, k));
  LA_TRY(la_limits(a, p));
  LA_TRY(la_operand("q", a->q, a->q_stride, a->dtype));
  LA_TRY(la_operand("k", a->k, a->k_stride, a->dtype));
  LA_TRY(la_operand("v", a->v, a->v_stride, a->dtype));
  LA_TRY(la_operand("dout", a->dout, a->do_stride, a->dtype));
  VLNI_CHECK(a->out && a->stat && ((uintptr_t)a->out | (uintptr_t)a->out_low) % 16 == 0, VLNI_EINVAL, "long_attn: out %p, out_low %p, stat %p", a->out,
             a->out_low, (void*)a->stat);
  VLNI_CHECK(a->dq && a->dk && a->dv && ((uintptr_t)a->dq | (uintptr_t)a->dk | (uintptr_t)a->dv) % 16 == 0, VLNI_EINVAL, "long_attn: dq %p, dk %p, dv %p",
             a->dq, a->dk, a->dv);
  VLNI_CHECK(!a->dtable || a->rel_table, VLNI_EINVAL, "long_attn: a table gradient without a table");
  const long n = (long)p.B * p.Sq * p.nh, need = la_prep_floats(a, p);
  long o_rs, o_db, o_part;
  const long work = la_bwd_work(a, p, &o_rs, &o_db, &o_part);
  VLNI_CHECK(!need || (a->prep && a->prep_floats >= need), VLNI_EINVAL, "long_attn: prep holds %ld floats, %ld are needed", a->prep ? a->prep_floats : 0, need);
  VLNI_CHECK(a->work && a->work_floats >= work && (uintptr_t)a->work % 16 == 0, VLNI_EINVAL, "long_attn: work holds %ld floats, %ld are needed",
             a->work ? a->work_floats : 0, work);
  const hipStream_t st = (hipStream_t)stream;
  la_prep_pointers(a, p);
  p.q = a->q; p.k = a->k; p.v = a->v; p.dout = a->dout;
  p.q_b = a->q_stride[0]; p.q_s = a->q_stride[1]; p.q_h = a->q_stride[2];
  p.k_b = a->k_stride[0]; p.k_s = a->k_stride[1]; p.k_h = a->k_stride[2];
  p.v_b = a->v_stride[0]; p.v_s = a->v_stride[1]; p.v_h = a->v_stride[2];
  p.d_b = a->do_stride[0]; p.d_s = a->do_stride[1]; p.d_h = a->do_stride[2];
  p.out = a->out; p.low = a->dtype == VLNI_F32 ? nullptr : a->out_low; p.lse = a->stat; p.rl = a->stat + n;
  p.dq = a->dq; p.dk = a->dk; p.dv = a->dv;
  float* f = (float*)a->work;
  p.delta = f;
  p.range = f + ((n + 3) & ~3L);
  p.rowsum = a->dtable ? f + o_rs : nullptr;
  p.dbpart = f + o_db;
  p.part = f + o_part;
  la_grid_rows(a, p);
  LA_TRY(la_go(a, p, 1, st));
  if (a->dtable) {
    hipLaunchKernelGGL(la_dtable_kernel, dim3(k.n * k.sides, p.nh), dim3(256), 0, st, p.dbpart, a->dtable, k, p.nh, p.R, p.BL, p.B * p.nblk);
    VLNI_LAUNCH_CHECK();
  }
  la_grid_keys(a, p);
  return la_go(a, p, 2, st);
}
