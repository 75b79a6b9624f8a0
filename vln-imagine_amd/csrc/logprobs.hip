// Log probabilities of given tokens with the entropy of their rows and the most likely alternatives, and their gradient (ops.token_logprobs).
//
//   m = max x, l = sum exp(x - m), s = sum exp(x - m)(x - m);  logp_t = x_t - m - log l;  H = log l - s / l     (differences from m: no cancellation
//   dx_v = g ([v = t] - p_v) - h p_v (log p_v + H)                                                              of large offsets)
//
// Bound by memory: forward reads the logits once - a thread keeps its own running (m, l, s), merged over the row at the end -, backward reads
// them once and writes the gradient; nothing else of the logits' size is made. Rows start at any element (30522 16-bit columns are no multiple
// of 16 bytes): vectors are laid on the row's 16-byte boundaries, and the partial ones at its ends are read and written element by element.
//
// Alternatives: the row's threads form 16 groups; the top-th largest of the groups' maxima is a lower bound of the top-th largest element, so only
// elements not below it (a dozen on ordinary logits) are candidates. They meet in LDS as 64-bit keys (order-preserving bits of x, then the
// complement of the index: one comparison means "larger value, then lower index") and are ranked by counting. Where ties make more than 48 of them, the
// best is taken out `top` times instead.
#include <limits.h>

#include "../../include/vlni.h"
#include "common.h"

namespace {

constexpr int LP_MAXTOP = 16, LP_MANY = 1024;
constexpr float LP_LOG2E = 1.4426950408889634f, LP_LN2 = 0.6931471805599453f;
typedef unsigned long long u64;

struct LpP {
  const void* x; long ld;
  const long* target; long ignore;
  float *logp, *ent, *stat;            // stat [rows][3]: m, log l, H
  float* top_logp; long* top_idx;
  int rows, V, top;
  int* bad;                            // counter of targets outside [0, V), or null
  // backward
  const float *g, *h;                  // gradients of logp and of the entropy (either null)
  void* dx; long lddx;
};

__device__ __forceinline__ unsigned lp_order(float x) {                      // monotone: -inf < ... < +inf (-0 = 0)
  const unsigned u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float lp_value(u64 key) {
  const unsigned o = (unsigned)(key >> 32);
  return __uint_as_float(o & 0x80000000u ? o & 0x7FFFFFFFu : ~o);
}
__device__ __forceinline__ u64 lp_wave_max(u64 k) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const u64 other = ((u64)(unsigned)__shfl_xor((int)(k >> 32), o, 64) << 32) | (unsigned)__shfl_xor((int)k, o, 64);
    k = other > k ? other : k;
  }
  return k;
}
// (m, l, s) of two parts of a row; a part without elements has m = -inf, l = s = 0
__device__ __forceinline__ void lp_merge(float& m, float& l, float& s, float m2, float l2, float s2) {
  const float mn = fmaxf(m, m2), mu = mn == -INFINITY ? 0.f : mn;
  const float d1 = fmaxf(m - mu, -1e30f), d2 = fmaxf(m2 - mu, -1e30f);       // an empty part's weight is 0, not 0 * inf
  const float w1 = __builtin_amdgcn_exp2f(d1 * LP_LOG2E), w2 = __builtin_amdgcn_exp2f(d2 * LP_LOG2E);
  s = (s + l * d1) * w1 + (s2 + l2 * d2) * w2;
  l = l * w1 + l2 * w2;
  m = mn;
}

// 16 / sizeof(T) elements of a row from element e on; those outside [0, V) are -inf. Only whole vectors inside the row are read as vectors.
template <typename T, int VEC> __device__ __forceinline__ void lp_load(float (&x)[VEC], const T* row, long e, int V) {
  if constexpr (VEC == 1) {
    x[0] = e < V ? (float)row[e] : -INFINITY;
  } else {
    if (e >= 0 && e + VEC <= V) {
      typedef T vec __attribute__((ext_vector_type(VEC)));
      const vec v = *(const vec*)(row + e);
#pragma unroll
      for (int j = 0; j < VEC; ++j) x[j] = (float)v[j];
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) x[j] = e + j >= 0 && e + j < V ? (float)row[e + j] : -INFINITY;
    }
  }
}
template <typename T> __device__ __forceinline__ int lp_head(const T* row) {      // elements between the 16-byte boundary below the row and the row
  return (int)(((uintptr_t)row & 15) / sizeof(T));
}
// the threads of a row: a wave (its LDS operations are in order: nothing but the compiler has to be held) or the block
template <int NW> __device__ __forceinline__ void lp_sync() {
  if constexpr (NW == 1) {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  } else {
    __syncthreads();
  }
}

constexpr int LP_CAND = 48;
struct LpTop {
  u64 list[16], cand[LP_CAND], wbest[16];
  float gmax[16];
  int count;
};

// TPB threads per row (64: four rows a block), N vectors of VEC elements a thread and pass
template <typename T, int TPB, int VEC, int N, bool TOP, int WPE>
__global__ __launch_bounds__(TPB < 256 ? 256 : TPB, WPE) void lp_fwd_kernel(LpP p) {
  constexpr int NW = TPB / 64, RPB = TPB < 256 ? 256 / TPB : 1, GL = TPB / 16;       // waves and rows, threads of a group
  __shared__ LpTop tops[TOP ? RPB : 1];
  __shared__ float red[3][16];
  const int tid = threadIdx.x % TPB, lane = threadIdx.x & 63, wave = NW == 1 ? 0 : tid >> 6;
  const long row_i = NW == 1 ? (long)blockIdx.x * 4 + (threadIdx.x >> 6) : blockIdx.x;
  if (NW == 1 && row_i >= p.rows) return;
  LpTop& q = tops[TOP && NW == 1 ? threadIdx.x >> 6 : 0];
  const T* row = (const T*)p.x + row_i * p.ld;
  // whole vectors [first, first + full VEC), up to VEC - 1 elements on either side of them: one more element for the first 2 VEC threads
  const int first = VEC == 1 ? 0 : (VEC - lp_head(row)) % VEC, full = VEC == 1 ? p.V : (p.V - first) / VEC;
  float m = -INFINITY, l = 0.f, s = 0.f;
  if (TOP) {
    if (tid < 16) q.list[tid] = 0;
    if (tid == 0) q.count = 0;
    lp_sync<NW>();
  }
  for (int v0 = 0; v0 < full; v0 += TPB * N) {
    typedef T vec __attribute__((ext_vector_type(VEC)));
    float x[N][VEC], xe = -INFINITY;
    int ie = -1;
    {
      vec raw[N];
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const long v = min(v0 + n * TPB + tid, full - 1);          // (unconditional: the loads are in flight together)
        if constexpr (VEC == 1) raw[n][0] = row[v];
        else raw[n] = *(const vec*)(row + first + v * VEC);
      }
      if (VEC > 1 && v0 == 0) {
        if (tid < first) ie = tid;
        else if (tid >= VEC && first + full * VEC + tid - VEC < p.V && tid < 2 * VEC) ie = first + full * VEC + tid - VEC;
        if (ie >= 0) xe = (float)row[ie];
      }
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int j = 0; j < VEC; ++j) x[n][j] = v0 + n * TPB + tid < full ? (float)raw[n][j] : -INFINITY;
    }
    float mt = xe;
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int j = 0; j < VEC; ++j) mt = fmaxf(mt, x[n][j]);
    const float mu = mt == -INFINITY ? 0.f : mt;
    float lt, st;
    {
      const float d = xe - mu;
      lt = __builtin_amdgcn_exp2f(d * LP_LOG2E);
      st = lt * fmaxf(d, -1e30f);
    }
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float d = x[n][j] - mu, e = __builtin_amdgcn_exp2f(d * LP_LOG2E);
        lt += e;
        st += e * fmaxf(d, -1e30f);
      }
    lp_merge(m, l, s, mt, lt, st);
    if constexpr (TOP) {
      // what may be among the `top` best of the row: nothing below the list's last, or - while the list is not full, its last then 0 - below the
      // top-th largest of the groups' maxima
      const u64 last = q.list[p.top - 1];
      float tau;
      if (last) {                                                  // (uniform)
        tau = lp_value(last);
      } else {
        float gm = mt;
#pragma unroll
        for (int o = GL / 2; o > 0; o >>= 1) gm = fmaxf(gm, __shfl_xor(gm, o, 64));
        if (tid % GL == 0) q.gmax[tid / GL] = gm;
        lp_sync<NW>();
        const float own = q.gmax[lane & 15];
        int rank = 0;
#pragma unroll
        for (int g = 0; g < 16; ++g) {
          const float o = q.gmax[g];
          rank += o > own || (o == own && g < (lane & 15));
        }
        tau = __shfl(own, (int)__builtin_ctzll(__ballot(rank == p.top - 1) | (1ull << 63)), 64);
      }
      auto key = [&](float v, int e) { return ((u64)lp_order(v) << 32) | (0xFFFFFFFFu - (unsigned)e); };
      auto push = [&](float v, int e) {
        const int slot = atomicAdd(&q.count, 1);
        if (slot < LP_CAND) q.cand[slot] = key(v, e);
      };
      if (mt >= tau) {
        if (ie >= 0 && xe >= tau) push(xe, ie);
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
          for (int j = 0; j < VEC; ++j)
            if (x[n][j] >= tau && v0 + n * TPB + tid < full) push(x[n][j], first + (v0 + n * TPB + tid) * VEC + j);
      }
      lp_sync<NW>();
      const int count = q.count;
      if (count <= LP_CAND) {
        if (wave == 0) {
          // lanes 0 - 47 hold the candidates, 48 - 63 what is in the list; keys are unique, 0 stands for nothing
          const u64 mine = lane < count ? q.cand[lane] : lane >= 48 && lane - 48 < p.top ? q.list[lane - 48] : 0;
          int r = 0;
          for (int i = 0; i < count; ++i) r += q.cand[i] > mine;
          for (int i = 0; i < p.top; ++i) r += q.list[i] > mine;
          lp_sync<1>();
          if (mine && r < p.top) q.list[r] = mine;
          if (lane == 0) q.count = 0;
        }
        lp_sync<NW>();
      } else {
        unsigned taken = 0;                                        // of this thread's vectors; the single element: out
        bool out = ie < 0;
        auto best = [&]() {                                        // largest value first, then its lowest index: no 64-bit key per element
          float v = out ? -INFINITY : xe;
          int e = out ? INT_MAX : ie;
#pragma unroll
          for (int n = 0; n < N; ++n)
#pragma unroll
            for (int j = 0; j < VEC; ++j) v = (taken >> (n * VEC + j)) & 1 ? v : fmaxf(v, x[n][j]);
          if (!out && xe != v) e = INT_MAX;
#pragma unroll
          for (int n = 0; n < N; ++n)
#pragma unroll
            for (int j = 0; j < VEC; ++j)
              if (x[n][j] == v && !((taken >> (n * VEC + j)) & 1) && v0 + n * TPB + tid < full) e = min(e, first + (v0 + n * TPB + tid) * VEC + j);
          return e == INT_MAX ? 0 : key(v, e);
        };
        u64 mine = best(), wmax = lp_wave_max(mine);
        while (true) {
          lp_sync<NW>();
          if (lane == 0) q.wbest[wave] = wmax;
          lp_sync<NW>();
          const u64 k = lp_wave_max(lane < NW ? q.wbest[lane] : 0);
          if (k <= q.list[p.top - 1]) break;                       // (uniform) used up, or nothing beats the last one
          const u64 cur = q.list[lane & 15], prev = (lane & 15) ? q.list[(lane & 15) - 1] : ~0ull;
          lp_sync<NW>();
          if (wave == 0 && lane < p.top && cur < k) q.list[lane] = prev > k ? k : prev;
          if (wmax == k) {
            if (mine == k) {
              const int e = (int)(0xFFFFFFFFu - (unsigned)k);
              if (e == ie) {
                out = true;
              } else {
                const int i = (e - first) - v0 * VEC;
                taken |= 1u << ((i / VEC / TPB) * VEC + i % VEC);
              }
              mine = best();
            }
            wmax = lp_wave_max(mine);
          }
        }
        if (tid == 0) q.count = 0;             // (behind the loop's barriers: every wave has read it and taken this branch)
        lp_sync<NW>();
      }
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const float m2 = __shfl_xor(m, o, 64), l2 = __shfl_xor(l, o, 64), s2 = __shfl_xor(s, o, 64);
    lp_merge(m, l, s, m2, l2, s2);
  }
  if (NW > 1) {
    if (lane == 0) { red[0][wave] = m; red[1][wave] = l; red[2][wave] = s; }
    __syncthreads();
    m = red[0][0]; l = red[1][0]; s = red[2][0];
    for (int w = 1; w < NW; ++w) lp_merge(m, l, s, red[0][w], red[1][w], red[2][w]);
  }
  const bool dead = m == -INFINITY && l == 0.f;                                  // nothing but -inf
  const float logl = dead ? 0.f : __builtin_amdgcn_logf(l) * LP_LN2, H = dead ? 0.f : logl - s / l;
  if (tid == 0) {
    const long t = p.target[row_i];
    float lp = 0.f;
    if (t >= 0 && t < p.V) lp = dead ? -INFINITY : ((float)row[t] - m) - logl;
    else if (t != p.ignore && p.bad) atomicAdd(p.bad, 1);
    p.logp[row_i] = t == p.ignore ? 0.f : lp;
    p.ent[row_i] = H;
    p.stat[3 * row_i] = m;
    p.stat[3 * row_i + 1] = logl;
    p.stat[3 * row_i + 2] = H;
  }
  if (TOP && wave == 0 && lane < p.top) {
    const u64 k = q.list[lane];
    p.top_idx[row_i * p.top + lane] = k ? (long)(0xFFFFFFFFu - (unsigned)k) : lane;        // (a row of NaN has no largest elements)
    p.top_logp[row_i * p.top + lane] = dead ? -INFINITY : (lp_value(k) - m) - logl;        // (0 is the key of a NaN)
  }
}

// grid = (rows / rows a block, parts of a row); TPB threads per row and part
template <typename T, int TPB, int VEC, int N>
__global__ __launch_bounds__(256) void lp_bwd_kernel(LpP p) {
  const int tid = threadIdx.x % TPB;
  const long row_i = (long)blockIdx.x * (256 / TPB) + threadIdx.x / TPB;
  if (row_i >= p.rows) return;
  const T* row = (const T*)p.x + row_i * p.ld;
  T* out = (T*)p.dx + row_i * p.lddx;
  const long e0 = VEC == 1 ? 0 : -lp_head(row);
  const bool same = VEC > 1 && lp_head(row) == lp_head(out);
  const float m = p.stat[3 * row_i], logl = p.stat[3 * row_i + 1], H = p.stat[3 * row_i + 2];
  const long t = p.target[row_i];
  const bool dead = m == -INFINITY && logl == 0.f, scored = t >= 0 && t < p.V && t != p.ignore;
  const float g = p.g && scored && !dead ? p.g[row_i] : 0.f, h = p.h ? p.h[row_i] : 0.f;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const long e = e0 + (long)blockIdx.y * TPB * N * VEC + ((long)n * TPB + tid) * VEC;
    if (e >= p.V) break;
    float x[VEC];
    lp_load<T, VEC>(x, row, e, p.V);
    T v[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const float lp = (x[j] - m) - logl, pr = __builtin_amdgcn_exp2f(lp * LP_LOG2E);
      float d = -pr * (g + h * (fmaxf(lp, -200.f) + H));              // (below -104 p is 0: no infinity may stand beside it, however large h)
      if (e + j == t) d += g;
      v[j] = (T)(dead ? 0.f : d);
    }
    if constexpr (VEC > 1) {
      if (same && e >= 0 && e + VEC <= p.V) {
        typedef T vec __attribute__((ext_vector_type(VEC)));
        vec w;
#pragma unroll
        for (int j = 0; j < VEC; ++j) w[j] = v[j];
        *(vec*)(out + e) = w;
        continue;
      }
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j)
      if (e + j >= 0 && e + j < p.V) out[e + j] = v[j];
  }
}

template <typename T, bool TOP> int lp_fwd_launch(const LpP& p, hipStream_t st) {
  constexpr int CE = 16 / (int)sizeof(T);
  // a wave per row while a row fits its registers; short rows element by element (their vectors would be mostly partial); long rows of a launch that
  // fills the chip a block of 256 each, of a small one a block of 1024 (8 x 30522 float32, top 5: 12.6 us, with 256: 17.7). The alternatives' kernel at
  // five waves a SIMD: what it waits for are its own barriers, and 15 registers in memory cost less than the fourth wave's place (2048 x 30522 bf16,
  // top 8: 88 -> 58 us; 53 - 58 since passes are held against the list's last)
  if (p.V <= 512) hipLaunchKernelGGL((lp_fwd_kernel<T, 64, 1, 8, TOP, 1>), dim3(cdiv(p.rows, 4)), dim3(256), 0, st, p);
  else if (p.V <= 2048) hipLaunchKernelGGL((lp_fwd_kernel<T, 64, CE, 32 / CE, TOP, 1>), dim3(cdiv(p.rows, 4)), dim3(256), 0, st, p);
  else if (p.rows >= LP_MANY || p.V <= 8192) hipLaunchKernelGGL((lp_fwd_kernel<T, 256, CE, 32 / CE, TOP, TOP ? 5 : 1>), dim3(p.rows), dim3(256), 0, st, p);
  else hipLaunchKernelGGL((lp_fwd_kernel<T, 1024, CE, 32 / CE, TOP, 4>), dim3(p.rows), dim3(1024), 0, st, p);
  VLNI_LAUNCH_CHECK();
  return VLNI_OK;
}
template <typename T> int lp_bwd_launch(const LpP& p, hipStream_t st) {
  constexpr int CE = 16 / (int)sizeof(T);
  if (p.V <= 512) hipLaunchKernelGGL((lp_bwd_kernel<T, 64, 1, 8>), dim3(cdiv(p.rows, 4), 1), dim3(256), 0, st, p);
  else if (p.V <= 2048 - CE) hipLaunchKernelGGL((lp_bwd_kernel<T, 64, CE, 32 / CE>), dim3(cdiv(p.rows, 4), 1), dim3(256), 0, st, p);
  else hipLaunchKernelGGL((lp_bwd_kernel<T, 256, CE, 32 / CE>), dim3(p.rows, cdiv((long)p.V + CE, 8192)), dim3(256), 0, st, p);
  VLNI_LAUNCH_CHECK();
  return VLNI_OK;
}
// a launch has less than 2^32 threads: 256 a row, 64 where four rows share a block (in both directions)
bool lp_fits(int rows, int V) { return rows < (V <= 2040 ? 1 << 26 : 1 << 24); }
}  // namespace

extern "C" int vlni_token_logprobs_fwd(int dtype, const void* logits, long ld, const long* target, long ignore_index, float* logp, float* entropy,
                                       float* stat, float* top_logp, long* top_index, int top, int rows, int V, void* stream) {
  VLNI_CHECK(dtype >= VLNI_F32 && dtype <= VLNI_F16, VLNI_EINVAL, "token_logprobs: dtype %d", dtype);
  VLNI_CHECK(rows > 0 && V > 0 && V <= (1 << 28) && ld >= V, VLNI_EINVAL, "token_logprobs: rows=%d V=%d ld=%ld", rows, V, ld);
  VLNI_CHECK(lp_fits(rows, V), VLNI_EUNSUP, "token_logprobs: %d rows of %d (at most 2^26 - 1 up to 2040 columns, 2^24 - 1 beyond)", rows, V);
  VLNI_CHECK(top >= 0 && top <= LP_MAXTOP && top <= V, VLNI_EUNSUP, "token_logprobs: top=%d of %d (at most %d)", top, V, LP_MAXTOP);
  VLNI_CHECK(logits && target && logp && entropy && stat && (!top || (top_logp && top_index)), VLNI_EINVAL, "token_logprobs: null pointer");
  LpP p{};
  p.x = logits; p.ld = ld; p.target = target; p.ignore = ignore_index; p.logp = logp; p.ent = entropy; p.stat = stat; p.top_logp = top_logp;
  p.top_idx = top_index; p.rows = rows; p.V = V; p.top = top; p.bad = vlni_index_error_counter();
  const hipStream_t st = (hipStream_t)stream;
#define LP_GO(T) (top ? lp_fwd_launch<T, true>(p, st) : lp_fwd_launch<T, false>(p, st))
  return dtype == VLNI_F32 ? LP_GO(float) : dtype == VLNI_BF16 ? LP_GO(__bf16) : LP_GO(_Float16);
#undef LP_GO
}

extern "C" int vlni_token_logprobs_bwd(int dtype, const float* dlogp, const float* dentropy, const void* logits, long ld, const long* target,
                                       long ignore_index, const float* stat, void* dlogits, long lddl, int rows, int V, void* stream) {
  VLNI_CHECK(dtype >= VLNI_F32 && dtype <= VLNI_F16, VLNI_EINVAL, "token_logprobs: dtype %d", dtype);
  VLNI_CHECK(rows > 0 && V > 0 && V <= (1 << 28) && ld >= V && lddl >= V, VLNI_EINVAL, "token_logprobs: rows=%d V=%d ld=%ld lddl=%ld", rows, V, ld, lddl);
  VLNI_CHECK(lp_fits(rows, V), VLNI_EUNSUP, "token_logprobs: %d rows of %d (at most 2^26 - 1 up to 2040 columns, 2^24 - 1 beyond)", rows, V);
  VLNI_CHECK(logits && target && stat && dlogits, VLNI_EINVAL, "token_logprobs: null pointer");
  LpP p{};
  p.x = logits; p.ld = ld; p.target = target; p.ignore = ignore_index; p.stat = (float*)stat; p.rows = rows; p.V = V; p.g = dlogp; p.h = dentropy;
  p.dx = dlogits; p.lddx = lddl;
  const hipStream_t st = (hipStream_t)stream;
  return dtype == VLNI_F32 ? lp_bwd_launch<float>(p, st) : dtype == VLNI_BF16 ? lp_bwd_launch<__bf16>(p, st) : lp_bwd_launch<_Float16>(p, st);
}
