// logits.hip — objectives on the log-probabilities of taken classes: log softmax at a target, its backward pass, sums over packed
// sequences, a paired preference loss and a clipped policy loss with a KL term (gfx950).
//
// A row z of V logits with target y:   M = max z,  s = sum exp(z - M),  log p(y) = z_y - M - log s,
//                                      d log p(y) / dz_j = [j = y] - exp(z_j - M) / s.
// Every objective here reaches the logits through log p(y) alone, so a row's gradient is one number c times that vector.
//
// Precision: a row's sum is collected in fp64 from fp32 sums of 8 exponentials, log p(y) and what follows from it (a ratio that is compared
// with a border, exp(d) - 1 - d of a small d) in fp64: a handful of operations per row.
#include "rs_common.h"
#include <math.h>

namespace {

struct Rows {
  const void *z;
  long long rows, ld;
  int classes, sequences;
  const long long *target;
  long long ignore;
  const int *offset;
  int *bad;
};

struct Policy {
  const float *old_logp, *adv, *ref;
  int adv_per_sequence, token_mean;
  double lo, hi, kl;
  const int *counts;          // rows that count, per sequence (or of all), in `splits` parts
  int splits;
  float *coef;                // d loss / d log p(y) per row
  double *partial;            // per workgroup: loss, KL, cut-off rows
};

constexpr int LG_VEC = 8;
// 8 consecutive logits as the words they come in: two to a register in 16 bits
template <typename T> struct Vec { unsigned w[LG_VEC * sizeof(T) / 4]; };
__device__ __forceinline__ float lg_get(const Vec<float> &v, int i) { return __uint_as_float(v.w[i]); }
__device__ __forceinline__ float lg_get(const Vec<__bf16> &v, int i) { return __uint_as_float(i & 1 ? v.w[i >> 1] & 0xFFFF0000u : v.w[i >> 1] << 16); }
__device__ __forceinline__ float lg_get(const Vec<_Float16> &v, int i) {
  return (float)__builtin_bit_cast(_Float16, (unsigned short)(i & 1 ? v.w[i >> 1] >> 16 : v.w[i >> 1]));
}
// aligned to one logit: global loads and stores of this device need no more
template <typename T>
__device__ __forceinline__ Vec<T> lg_load(const T *p, int left) {
  Vec<T> v;
  if (left >= LG_VEC) __builtin_memcpy(&v, p, sizeof(v));
  else {
    T x[LG_VEC];
#pragma unroll
    for (int i = 0; i < LG_VEC; ++i) x[i] = i < left ? p[i] : (T)-INFINITY;
    __builtin_memcpy(&v, x, sizeof(v));
  }
  return v;
}
template <typename T>
__device__ __forceinline__ void lg_store(T *p, int left, const float *x) {
  T v[LG_VEC];
#pragma unroll
  for (int i = 0; i < LG_VEC; ++i) v[i] = (T)x[i];
  if (left >= LG_VEC) __builtin_memcpy(p, v, sizeof(v));
  else {
#pragma unroll
    for (int i = 0; i < LG_VEC; ++i) if (i < left) p[i] = v[i];
  }
}
template <typename T>
__device__ __forceinline__ float lg_top(const Vec<T> &v, float m) {
#pragma unroll
  for (int i = 0; i < LG_VEC; ++i) m = fmaxf(m, lg_get(v, i));
  return m;
}

// exp(x).  log2 e in two parts: its fp32 rounding alone would shift every row's sum the same way (1.3e-8 |x|), and a sequence's log-probability
// adds thousands of rows
__device__ __forceinline__ float lg_exp(float x) {
  return __builtin_amdgcn_exp2f(rs_fma(x, 1.44269502162933349609f, x * 1.92596299112661746887e-8f));
}
template <typename T>
__device__ __forceinline__ double lg_sum(const Vec<T> &v, float base) {
  float e[LG_VEC];
#pragma unroll
  for (int i = 0; i < LG_VEC; ++i) e[i] = lg_exp(lg_get(v, i) - base);
  return (double)(((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7])));
}
// c ([j = y] - exp(z_j - base) inv), scale = -c inv; j: the index of v's first logit
template <typename T>
__device__ __forceinline__ void lg_gradient(T *p, int left, const Vec<T> &v, float base, float scale, float c, int j, int y) {
  float g[LG_VEC];
#pragma unroll
  for (int i = 0; i < LG_VEC; ++i) g[i] = lg_exp(lg_get(v, i) - base) * scale;
  if ((unsigned)(y - j) < (unsigned)LG_VEC) {
#pragma unroll
    for (int i = 0; i < LG_VEC; ++i) g[i] += j + i == y ? c : 0.f;
  }
  lg_store(p, left, g);
}
template <typename T>
__device__ __forceinline__ void lg_fill(T *p, int left, float x) {
  float g[LG_VEC];
#pragma unroll
  for (int i = 0; i < LG_VEC; ++i) g[i] = x;
  lg_store(p, left, g);
}
// The compiler must not keep what it formed of v (conversions, exponentials) past this point: in fp32 that is twice the registers of a
// row in 16 bits, and a kernel that holds rows would spill.
template <typename T>
__device__ __forceinline__ void lg_forget(Vec<T> &v) {
#pragma unroll
  for (int i = 0; i < (int)(sizeof(v) / 4); ++i) asm volatile("" : "+v"(v.w[i]));
}
// the value that exponents are taken against: of a row that holds nothing but -infinity, 0 (exp(-inf - 0) = 0, and 0 / 0 follows)
__device__ __forceinline__ float lg_base(float m) { return m == -INFINITY ? 0.f : m; }

// over LANES neighbouring lanes, the result in each of them
template <int LANES>
__device__ __forceinline__ float lg_lanes_max(float x) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor(x, o));
  return x;
}
template <int LANES>
__device__ __forceinline__ double lg_lanes_sum(double x) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) x += __shfl_xor(x, o);
  return x;
}

// the sequence of a row: the first whose end exceeds it; `sequences` for the rows behind the last one
__device__ __forceinline__ int lg_owner(const int *offset, int sequences, long long row) {
  int lo = 0, hi = sequences;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (row >= (long long)offset[mid]) lo = mid + 1; else hi = mid;
  }
  return lo;
}

// exp, log and exp(d) - 1 - d in fp64, in a chain of few registers: they run while a row waits in the others.  exp(x) = 2^k exp(r), |r| <= ln 2 / 2,
// as its Taylor sum to r^13 / 13! (r^14 / 14!: 4e-18); log s = y + log(s exp(-y)) from fp32's y, whose rest is below 1e-6.
__device__ __forceinline__ double lg_taylor(double r, double from) {      // sum of r^i / (i + 2)!, the exponential without its first two terms over r^2
  double t = 1.0 / 6227020800.0;
  t = fma(t, r, 1.0 / 479001600.0); t = fma(t, r, 1.0 / 39916800.0); t = fma(t, r, 1.0 / 3628800.0); t = fma(t, r, 1.0 / 362880.0);
  t = fma(t, r, 1.0 / 40320.0); t = fma(t, r, 1.0 / 5040.0); t = fma(t, r, 1.0 / 720.0); t = fma(t, r, 1.0 / 120.0); t = fma(t, r, 1.0 / 24.0);
  t = fma(t, r, 1.0 / 6.0);
  return fma(t, r, from);
}
__device__ __forceinline__ double lg_exp64(double x) {
  const double lim = fmin(fmax(x, -1100.0), 1100.0);                  // (infinite arguments; not-a-numbers are put back below)
  const double k = rint(lim * 1.4426950408889634074);
  const double r = fma(-k, 2.3190468138462995584e-17, fma(-k, 0.69314718055994528623, lim));
  const double e = fma(fma(lg_taylor(r, 0.5), r, 1.0), r, 1.0);
  return x != x ? x : ldexp(e, (int)k);
}
__device__ __forceinline__ double lg_log64(double s) {                  // of a sum: at least 1, or infinite, or no number
  const double y = (double)(__builtin_amdgcn_logf((float)s) * 0.69314718055994530942f);
  const double q = fma(s, lg_exp64(-y), -1.0);
  return s < INFINITY ? y + fma(-0.5 * q, q, q) : s;
}
__device__ __forceinline__ double lg_rest(double d, double *slope) {     // exp(d) - 1 - d, and its slope exp(d) - 1 (each by itself: d may be -infinity)
  if (fabs(d) <= 0.35) {
    const double e = d * d * lg_taylor(d, 0.5);
    *slope = e + d;
    return e;
  }
  *slope = lg_exp64(d) - 1.0;
  return *slope - d;
}

// d loss / d log p(y) of the policy loss for one row, and its three contributions
__device__ __forceinline__ double lg_policy(const Policy &P, double w, double logp, double old, double a, double ref, double *add) {
  const double r = lg_exp64(logp - old);
  const bool cut = a >= 0.0 ? r > P.hi : r < P.lo;             // the cut-off ratio is the smaller term: no gradient through it
  double each = -(cut ? (a >= 0.0 ? P.hi : P.lo) : r) * a, c = cut ? 0.0 : -a * r;
  if (r != r || a != a) each = c = r + a;
  if (P.ref) {
    double slope;
    const double e = lg_rest(ref - logp, &slope);              // not negative, and its mean over the policy's own draws is the KL
    each += P.kl * e;
    c -= P.kl * slope;
    add[1] += w * e;
  }
  add[0] += w * each;
  add[2] += cut ? w : 0.0;
  return w * c;
}
__device__ __forceinline__ double lg_weight(const Rows &R, const Policy &P, int owner) {
  int n = 0;
  const int first = P.token_mean ? 0 : owner * P.splits;
  for (int k = 0; k < P.splits; ++k) n += P.counts[first + k];
  return 1.0 / (double)n / (P.token_mean ? 1.0 : (double)R.sequences);
}

enum { LG_LOGP = 0, LG_POLICY = 1, LG_BACK = 2 };

// what a row is, before any of its logits is read
struct Row {
  long long at, y;
  int owner;
  bool counts, bad;
};
__device__ __forceinline__ Row lg_row(const Rows &R, long long row) {
  Row w;
  w.at = row;
  w.y = R.target[row];
  w.owner = R.offset ? lg_owner(R.offset, R.sequences, row) : 0;
  w.counts = w.y != R.ignore && (!R.offset || w.owner < R.sequences);
  w.bad = w.counts && (w.y < 0 || w.y >= R.classes);
  return w;
}

struct Outs {                 // what a kernel writes of a row; null: not wanted
  float *logp;
  double *logp64;
  float2 *stat;               // M, 1 / s
  void *dz;
  const float *coef, *up;     // LG_BACK: coefficients of rows (of sequences with offsets, unless row_coef), and a factor for all of them
  int skip_unit, row_coef;
};

// LG_BACK: a row's coefficient.  With offsets too where every row has its own: they tell which rows lie behind the last sequence.
__device__ __forceinline__ float lg_coef(const Rows &R, const Outs &O, const Row &w) {
  return O.coef[R.offset && !O.row_coef ? (long long)w.owner : w.at];
}

// one that does not count, or whose target is no class: 0, or not a number; none of its logits is read
__device__ __forceinline__ float lg_void(const Rows &R, const Policy &P, const Outs &O, const Row &w, bool first, int policy, double *add) {
  const float fill = w.bad ? __uint_as_float(0x7FC00000u) : 0.f;
  if (first) {
    if (O.logp) O.logp[w.at] = fill;
    if (O.logp64) O.logp64[w.at] = (double)fill;
    if (O.stat) O.stat[w.at] = make_float2(fill, 0.f);
    if (w.bad && R.bad) atomicAdd(R.bad, 1);
    if (policy) {
      if (P.coef) P.coef[w.at] = fill;
      if (w.bad) { add[0] += (double)fill; add[1] += (double)fill; add[2] += (double)fill; }
    }
  }
  return fill;
}
// what the policy loss needs beside a row's logits: asked for before them
struct Pre {
  double w;
  float old, adv, ref;
};
__device__ __forceinline__ Pre lg_pre(const Rows &R, const Policy &P, const Row &w) {
  return Pre{lg_weight(R, P, w.owner), P.old_logp[w.at], P.adv[P.adv_per_sequence ? (long long)w.owner : w.at], P.ref ? P.ref[w.at] : 0.f};
}
// what follows from a row's M and s; `first`: the lane that writes it down
__device__ __forceinline__ float lg_finish(const Policy &P, const Outs &O, long long row, const Pre &pre, float zy, float M, double s, bool first, int policy,
                                           double *add) {
  const double lp = (double)zy - (double)M - lg_log64(s);
  float c = 0.f;
  double mine[3] = {0.0, 0.0, 0.0};
  if (policy) c = (float)lg_policy(P, pre.w, lp, (double)pre.old, (double)pre.adv, (double)pre.ref, mine);
  if (first) {
    if (O.logp) O.logp[row] = (float)lp;
    if (O.logp64) O.logp64[row] = lp;
    if (O.stat) O.stat[row] = make_float2(M, 1.f / (float)s);
    if (policy) {
      if (P.coef) P.coef[row] = c;
      add[0] += mine[0]; add[1] += mine[1]; add[2] += mine[2];
    }
  }
  return c;
}

// the policy loss's sums of a workgroup, in the order of its threads
template <int THREADS>
__device__ __forceinline__ void lg_partial(const Policy &P, const double *add, int block) {
  __shared__ double red[3][THREADS / 64];
  for (int k = 0; k < 3; ++k) {
    const double t = lg_lanes_sum<64>(add[k]);
    if ((threadIdx.x & 63) == 0) red[k][threadIdx.x >> 6] = t;
  }
  __syncthreads();
  if (threadIdx.x < 3) {
    double t = 0.0;
    for (int i = 0; i < THREADS / 64; ++i) t += red[threadIdx.x][i];
    P.partial[(long long)block * 3 + threadIdx.x] = t;
  }
}

// Rows of up to 4096 classes: LANES neighbouring lanes hold a row in NV vectors of 8 per lane; one read, one write.  A team takes SUB rows
// before the fp64 steps, which its first SUB lanes then do for a row each: with 13 classes (2 lanes, 2 rows) every lane of a wave works
// on a row of its own.  The policy loss is bound by those steps (some 300 instructions in fp64) and by the registers that its rows stay
// in; four waves per SIMD and SUB * NV = 4 measured best over all lengths (SUB * NV = 8 with two waves: 13..18 % slower).  Against a workgroup
// per row (long_kernel): 2048 classes 171 against 294 us, 4096 152 against 167 (65536 and 32768 rows in bf16), so the border is the 8
// vectors that a lane can hold (in fp32 4096 classes are the other way round, 273 against 255).  Measured: policy loss, fp32, 65536 x 2048
// 246 us = 4.4 TB/s, 1048576 x 40 169 us; backward 2097152 x 13 81 us = 2.7 TB/s (rows of 52 bytes, two lanes each); log-probabilities
// 32768 x 4096 in bf16 46 us = 5.9 TB/s.
// What four waves cost: in fp32 the policy loss spills 40 registers at <64, 8>, 17 at <64, 1>, 4 to 8 at <4..32, 1> (in 16 bits 2 at
// <64, 8>); with three waves none does.  Three against four: 32768 x 4096 239 and 273 us, 262144 x 500 443 and 483 -- but 262144 x 250
// 229 and 196, 524288 x 100 221 and 188, 524288 x 64 120 and 108, 131072 x 1000 330 and 287.
template <typename T, int MODE, int LANES, int NV>
__global__ void __launch_bounds__(256, MODE == LG_POLICY ? 4 : 1)
short_kernel(Rows R, Policy P, Outs O) {
  constexpr int TEAMS = 256 / LANES;
  constexpr int ROOM = MODE == LG_POLICY && NV < 4 ? 4 / NV : 1, SUB = LANES < ROOM ? LANES : ROOM;
  const float up = MODE == LG_BACK && O.up ? *O.up : 1.f;
  if (MODE == LG_BACK && O.skip_unit && up == 1.f) return;
  const int team = (int)threadIdx.x / LANES, lane = (int)threadIdx.x % LANES, V = R.classes;
  double add[3] = {0.0, 0.0, 0.0};
  for (long long first = (long long)blockIdx.x * (TEAMS * SUB); first < R.rows; first += (long long)gridDim.x * (TEAMS * SUB)) {
    Vec<T> v[SUB][NV];
    Row w[SUB];
    bool in[SUB];
    float zy[SUB];
    Row mine{0, 0, 0, false, false};                           // the row whose fp64 steps this lane does
#pragma unroll
    for (int q = 0; q < SUB; ++q) {
      const long long row = first + q * TEAMS + team;
      w[q] = Row{row, 0, 0, false, false};
      if (row < R.rows) w[q] = lg_row(R, row);                 // (all lanes take part in the exchanges below)
      in[q] = w[q].counts && !w[q].bad;
      const T *__restrict__ z = (const T *)R.z + row * R.ld;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int j = (k * LANES + lane) * LG_VEC;
        v[q][k] = lg_load(z + j, in[q] ? V - j : 0);
      }
      zy[q] = MODE != LG_BACK && in[q] ? (float)z[w[q].y] : 0.f;
      if (lane == q) mine = w[q];
    }
    float M[SUB], inv[SUB], c[SUB];
    if (MODE == LG_BACK) {
#pragma unroll
      for (int q = 0; q < SUB; ++q) {
        c[q] = 0.f; M[q] = 0.f; inv[q] = 0.f;
        if (w[q].counts) c[q] = w[q].bad ? __uint_as_float(0x7FC00000u) : lg_coef(R, O, w[q]) * up;
        if (in[q]) { const float2 st = O.stat[w[q].at]; M[q] = st.x; inv[q] = st.y; }
      }
    } else {
      const bool live = lane < SUB && mine.counts && !mine.bad;
      Pre pre{1.0, 0.f, 0.f, 0.f};
      if (MODE == LG_POLICY && live) pre = lg_pre(R, P, mine);
      float my_m = 0.f, my_zy = 0.f;
      double my_s = 1.0;
#pragma unroll
      for (int q = 0; q < SUB; ++q) {
        float m = -INFINITY;
#pragma unroll
        for (int k = 0; k < NV; ++k) { m = lg_top(v[q][k], m); if (SUB * NV > 1) lg_forget(v[q][k]); }
        M[q] = lg_lanes_max<LANES>(m);
        double s = 0.0;
#pragma unroll
        for (int k = 0; k < NV; ++k) { s += lg_sum(v[q][k], lg_base(M[q])); if (SUB * NV > 1) lg_forget(v[q][k]); }
        s = lg_lanes_sum<LANES>(s);
        inv[q] = 1.f / (float)s;
        if (lane == q) { my_m = M[q]; my_s = s; my_zy = zy[q]; }
      }
      float my_c = 0.f;
      if (live) my_c = lg_finish(P, O, mine.at, pre, my_zy, my_m, my_s, true, MODE == LG_POLICY, add);
      else if (lane < SUB && mine.at < R.rows) my_c = lg_void(R, P, O, mine, true, MODE == LG_POLICY, add);
#pragma unroll
      for (int q = 0; q < SUB; ++q) c[q] = __shfl(my_c, q, LANES);
    }
    if (MODE != LG_LOGP && O.dz) {
#pragma unroll
      for (int q = 0; q < SUB; ++q) {
        if (w[q].at >= R.rows) continue;
        T *__restrict__ dz = (T *)O.dz + w[q].at * V;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
          const int j = (k * LANES + lane) * LG_VEC;
          if (j >= V) continue;
          if (in[q] && c[q] == c[q]) lg_gradient(dz + j, V - j, v[q][k], lg_base(M[q]), -c[q] * inv[q], c[q], j, (int)w[q].y);
          else lg_fill(dz + j, V - j, c[q]);
        }
      }
    }
  }
  if (MODE == LG_POLICY) lg_partial<256>(P, add, (int)blockIdx.x);
}

// The logits z[0, left) of a workgroup's THREADS threads, 8 to a thread and step.  The first `full` steps are whole: their loads ask no
// question and leave in one go, from an address that the workgroup shares and a thread's offset in it.  The step behind them, where each
// thread asks, is `tail`.
template <typename T, int THREADS>
__device__ __forceinline__ void lg_step(const T *__restrict__ z, int k, unsigned off, bool there, Vec<T> &v) {
  if (there) __builtin_memcpy(&v, (const char *)(z + (long long)k * (THREADS * LG_VEC)) + off, sizeof(v));
  else __builtin_memset(&v, 0, sizeof(v));                   // (never looked at; left undefined, it would be carried from row to row)
}
template <typename T, int THREADS>
__device__ __forceinline__ void lg_step_out(T *__restrict__ dz, int k, unsigned off, int tid, const Vec<T> &v, float base, float scale, float c, int y) {
  T *at = (T *)((char *)(dz + (long long)k * (THREADS * LG_VEC)) + off);
  lg_gradient(at, LG_VEC, v, base, scale, c, (k * THREADS + tid) * LG_VEC, y);
}

// The logits in front of a row's first 16-byte border, one for each of the first threads: the vectors of rows of an odd number of classes
// would straddle cache lines otherwise (bf16, 8192 x 50001: log-probabilities 172 us without, 139 us with heads, policy loss 363 and 333).
template <typename T>
__device__ __forceinline__ int lg_head(const T *z, int V) {
  const int n = (int)((16 - ((size_t)z & 15)) & 15) / (int)sizeof(T);
  return n < V ? n : V;
}

// Long rows, one workgroup each, LDS for what its waves tell each other.  HELD (the policy loss): the row stays in registers between its
// sum and its gradient, at most NV steps of 8 logits per thread and a tail.  Otherwise chunks of NV steps are taken in turn: their loads
// are all in flight before the first is used, and the running maximum is corrected once per chunk.
// Bound by memory: policy loss in bf16 8192 x 32768 219 us, 8192 x 65536 433 us, 8192 x 50001 333 us (4.9..5.0 TB/s), fp32 8192 x 32768 425 us
// (5.1); log-probabilities 8192 x 65536 in bf16 183 us = 5.9 TB/s.  256 threads leave room for two or three rows on a CU, whose loads, sums
// and stores overlap (1024 threads, one row: 395, 574 and 519 us, 529 in fp32); at 131072 classes one row is all that fits (4096 rows 557 us,
// 3.9 TB/s).  Held against read twice (HELD false: 263, 500 and 396 us, 494 in fp32, 604 at 131072; 262144 classes, which are always read
// twice, 3.4 TB/s), a row costs a third less traffic.
// (WAVES per SIMD bound the registers: left alone, the compiler interleaves the steps until two waves are all that fits)
template <typename T, int MODE, int THREADS, int NV, bool HELD, int WAVES>
__global__ void __launch_bounds__(THREADS, WAVES)
long_kernel(Rows R, Policy P, Outs O) {
  constexpr int W = THREADS / 64, STEP = THREADS * LG_VEC;
  __shared__ float red_m[2][W];
  __shared__ double red_s[2][W];
  __shared__ float red_c[2];
  const int tid = (int)threadIdx.x, wave = tid >> 6;
  const unsigned off = (unsigned)tid * (LG_VEC * sizeof(T));
  double add[3] = {0.0, 0.0, 0.0};
  int turn = 0;                       // scratch of two rows in turn: a row's last reader is a barrier ahead of the next but one's writer
  for (long long row = blockIdx.x; row < R.rows; row += gridDim.x) {
    const Row w = lg_row(R, row);
    const T *__restrict__ z = (const T *)R.z + row * R.ld;
    T *__restrict__ dz = O.dz ? (T *)O.dz + row * R.classes : nullptr;
    if (!w.counts || w.bad) {
      const float fill = lg_void(R, P, O, w, tid == 0, MODE == LG_POLICY, add);
      if (MODE == LG_POLICY && dz)
        for (int j = tid * LG_VEC; j < R.classes; j += STEP) lg_fill(dz + j, R.classes - j, fill);
      continue;
    }
    turn ^= 1;
    Vec<T> v[NV], tail;
    float M;
    double s = 0.0;
    Pre pre{1.0, 0.f, 0.f, 0.f};
    const float zy = (float)z[w.y];
    const int head = lg_head(z, R.classes), V = R.classes - head;          // from here on, V logits from z + head
    const float first = tid < head ? (float)z[tid] : -INFINITY;
    z += head;
    const int full = V / STEP, last = full * STEP + tid * LG_VEC;          // whole steps, and the thread's first logit behind them
    if (MODE == LG_POLICY && wave == 0) pre = lg_pre(R, P, w);
    float m = HELD ? first : -INFINITY;
    if (HELD) {
#pragma unroll
      for (int k = 0; k < NV; ++k) lg_step<T, THREADS>(z, k, off, k < full, v[k]);
      tail = lg_load(z + last, V - last);
#pragma unroll
      for (int k = 0; k < NV; ++k) if (k < full) { m = lg_top(v[k], m); lg_forget(v[k]); }
      m = lg_top(tail, m);
      lg_forget(tail);
    } else {
      int k0 = 0;
      for (; k0 + NV <= full; k0 += NV) {
#pragma unroll
        for (int k = 0; k < NV; ++k) lg_step<T, THREADS>(z, k0 + k, off, true, v[k]);
        float top = m;
#pragma unroll
        for (int k = 0; k < NV; ++k) top = lg_top(v[k], top);
        if (top > m) { s *= (double)lg_exp(m - top); m = top; }          // (m = -inf at first: s is 0)
#pragma unroll
        for (int k = 0; k < NV; ++k) s += lg_sum(v[k], lg_base(m));
      }
#pragma unroll
      for (int k = 0; k < NV; ++k) lg_step<T, THREADS>(z, k0 + k, off, k0 + k < full, v[k]);
      tail = lg_load(z + last, V - last);
      float top = lg_top(tail, fmaxf(m, first));
#pragma unroll
      for (int k = 0; k < NV; ++k) if (k0 + k < full) top = lg_top(v[k], top);
      if (top > m) { s *= (double)lg_exp(m - top); m = top; }
#pragma unroll
      for (int k = 0; k < NV; ++k) if (k0 + k < full) s += lg_sum(v[k], lg_base(m));
      s += lg_sum(tail, lg_base(m)) + (double)lg_exp(first - lg_base(m));
    }
    M = lg_lanes_max<64>(m);
    if ((tid & 63) == 0) red_m[turn][wave] = M;
    __syncthreads();
    M = red_m[turn][0];
#pragma unroll
    for (int k = 1; k < W; ++k) M = fmaxf(M, red_m[turn][k]);
    const float base = lg_base(M);
    if (HELD) {
#pragma unroll
      for (int k = 0; k < NV; ++k) if (k < full) { s += lg_sum(v[k], base); lg_forget(v[k]); }
      s += lg_sum(tail, base) + (double)lg_exp(first - base);
      lg_forget(tail);
    } else if (m != -INFINITY) s *= (double)lg_exp(m - base);
    s = lg_lanes_sum<64>(s);
    if ((tid & 63) == 0) red_s[turn][wave] = s;
    __syncthreads();
    s = red_s[turn][0];
#pragma unroll
    for (int k = 1; k < W; ++k) s += red_s[turn][k];
    float c = 0.f;
    if (wave == 0) {
      c = lg_finish(P, O, row, pre, zy, M, s, tid == 0, MODE == LG_POLICY, add);
      if (tid == 0) red_c[turn] = c;
    }
    if (MODE == LG_POLICY && dz) {
      __syncthreads();
      c = red_c[turn];
      const float scale = -c * (1.f / (float)s);
      const int y = (int)w.y - head;
      if (c != c) {
        for (int j = tid * LG_VEC; j < R.classes; j += STEP) lg_fill(dz + j, R.classes - j, c);
        continue;
      }
      if (tid < head) dz[tid] = (T)(lg_exp(first - base) * scale + (tid == (int)w.y ? c : 0.f));
      dz += head;
      if (HELD) {
#pragma unroll
        for (int k = 0; k < NV; ++k) if (k < full) lg_step_out<T, THREADS>(dz, k, off, tid, v[k], base, scale, c, y);
      } else {
        int k0 = 0;
        for (; k0 + NV <= full; k0 += NV) {
#pragma unroll
          for (int k = 0; k < NV; ++k) lg_step<T, THREADS>(z, k0 + k, off, true, v[k]);
#pragma unroll
          for (int k = 0; k < NV; ++k) lg_step_out<T, THREADS>(dz, k0 + k, off, tid, v[k], base, scale, c, y);
        }
        for (; k0 < full; ++k0) {
          lg_step<T, THREADS>(z, k0, off, true, v[0]);
          lg_step_out<T, THREADS>(dz, k0, off, tid, v[0], base, scale, c, y);
        }
        tail = lg_load(z + last, V - last);
      }
      if (last < V) lg_gradient(dz + last, V - last, tail, base, scale, c, last, y);
    }
  }
  if (MODE == LG_POLICY) lg_partial<THREADS>(P, add, (int)blockIdx.x);
}

// backward pass of long rows: a workgroup takes 256 * 8 * NV logits of a row at a time, whatever row they are of.  Bound by memory: 8192 x
// 65536 in bf16 373 us = 5.8 TB/s, fp32 8192 x 32768 382 us = 5.6 TB/s
template <typename T, int NV>
__global__ void __launch_bounds__(256, 7)
long_back_kernel(Rows R, Outs O, int parts) {
  constexpr int STEP = 256 * LG_VEC;
  const float up = O.up ? *O.up : 1.f;
  if (O.skip_unit && up == 1.f) return;
  const int tid = (int)threadIdx.x, V = R.classes;
  const unsigned off = (unsigned)tid * (LG_VEC * sizeof(T));
  for (long long row = blockIdx.y; row < R.rows; row += gridDim.y) {
    const Row w = lg_row(R, row);
    float c = 0.f;
    if (w.counts) c = w.bad ? __uint_as_float(0x7FC00000u) : lg_coef(R, O, w) * up;
    const T *__restrict__ z = (const T *)R.z + row * R.ld;
    T *__restrict__ dz = (T *)O.dz + row * V;
    if (c == 0.f || c != c) {
      for (int j = ((int)blockIdx.x * 256 + tid) * LG_VEC; j < V; j += (int)gridDim.x * STEP) lg_fill(dz + j, V - j, c);
      continue;
    }
    const int head = lg_head(z, V);
    for (int part = blockIdx.x; part < parts; part += gridDim.x) {
      const int j0 = head + part * (STEP * NV), left = V - j0, y = (int)w.y - j0;
      const int full = left <= 0 ? 0 : (left / STEP < NV ? left / STEP : NV);
      Vec<T> v[NV];
#pragma unroll
      for (int k = 0; k < NV; ++k) lg_step<T, 256>(z + j0, k, off, k < full, v[k]);
      const float2 st = O.stat[row];
      const float base = lg_base(st.x), scale = -c * st.y;
      if (part == 0 && tid < head) dz[tid] = (T)(lg_exp((float)z[tid] - base) * scale + (tid == (int)w.y ? c : 0.f));
#pragma unroll
      for (int k = 0; k < NV; ++k) if (k < full) lg_step_out<T, 256>(dz + j0, k, off, tid, v[k], base, scale, c, y);
      const int last = full * STEP + tid * LG_VEC;
      if (full < NV && last < left) lg_gradient(dz + j0 + last, left - last, lg_load(z + j0 + last, left - last), base, scale, c, last, y);
    }
  }
}

// Few long rows: a row in `parts` pieces, (M, s) of each ...  (one row of 100001 classes in bf16: 3.3 + 2.0 us, against 9.5 us by one
// workgroup; the launches' own time bounds both)
template <typename T, int NV>
__global__ void __launch_bounds__(256)
part_kernel(Rows R, int parts, int piece, float *__restrict__ part_m, double *__restrict__ part_s) {
  __shared__ float red_m[4];
  __shared__ double red_s[4];
  const int tid = (int)threadIdx.x;
  const long long row = blockIdx.y;
  const Row w = lg_row(R, row);
  if (!w.counts || w.bad) return;
  const int from = (int)blockIdx.x * piece, to = min(R.classes, from + piece);
  const T *__restrict__ z = (const T *)R.z + row * R.ld;
  float m = -INFINITY;
  double s = 0.0;
  for (int j0 = from; j0 < to; j0 += 256 * LG_VEC * NV) {
    Vec<T> v[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) { const int j = j0 + (k * 256 + tid) * LG_VEC; v[k] = lg_load(z + j, to - j); }
    float top = m;
#pragma unroll
    for (int k = 0; k < NV; ++k) top = lg_top(v[k], top);
    if (top > m) { s *= (double)lg_exp(m - top); m = top; }
#pragma unroll
    for (int k = 0; k < NV; ++k) s += lg_sum(v[k], lg_base(m));
  }
  float M = lg_lanes_max<64>(m);
  if ((tid & 63) == 0) red_m[tid >> 6] = M;
  __syncthreads();
  M = fmaxf(fmaxf(red_m[0], red_m[1]), fmaxf(red_m[2], red_m[3]));
  if (m != -INFINITY) s *= (double)lg_exp(m - lg_base(M));
  s = lg_lanes_sum<64>(s);
  if ((tid & 63) == 0) red_s[tid >> 6] = s;
  __syncthreads();
  if (tid == 0) {
    part_m[row * parts + blockIdx.x] = M;
    part_s[row * parts + blockIdx.x] = (red_s[0] + red_s[1]) + (red_s[2] + red_s[3]);
  }
}
// ... and their join, a wave per row: what long_kernel does after its last barrier
template <typename T, int MODE>
__global__ void __launch_bounds__(64)
join_kernel(Rows R, Policy P, Outs O, int parts, const float *__restrict__ part_m, const double *__restrict__ part_s) {
  double add[3] = {0.0, 0.0, 0.0};
  const int lane = (int)threadIdx.x;
  const long long row = blockIdx.x;
  const Row w = lg_row(R, row);
  if (!w.counts || w.bad) lg_void(R, P, O, w, lane == 0, MODE == LG_POLICY, add);
  else {
    const float zy = (float)((const T *)R.z + row * R.ld)[w.y];
    Pre pre{1.0, 0.f, 0.f, 0.f};
    if (MODE == LG_POLICY) pre = lg_pre(R, P, w);
    const float m = lane < parts ? part_m[row * parts + lane] : -INFINITY;
    const float M = lg_lanes_max<64>(m);
    double s = lane < parts ? part_s[row * parts + lane] : 0.0;
    if (m != -INFINITY) s *= (double)lg_exp(m - lg_base(M));
    s = lg_lanes_sum<64>(s);
    lg_finish(P, O, row, pre, zy, M, s, lane == 0, MODE == LG_POLICY, add);
  }
  if (MODE == LG_POLICY) lg_partial<64>(P, add, (int)blockIdx.x);
}

// rows that count, of sequence blockIdx.y (of all rows without offsets), in gridDim.x parts: known before the first gradient is written.  4 us
// for 65536 rows, a launch's own time.
__global__ void __launch_bounds__(256)
count_kernel(long long rows, const int *__restrict__ offset, const long long *__restrict__ target, long long ignore, int *__restrict__ counts) {
  __shared__ int red[4];
  const int q = (int)blockIdx.y;
  long long a = 0, b = rows;
  if (offset && gridDim.y > 1) { a = q ? offset[q - 1] : 0; b = offset[q]; }
  else if (offset) b = offset[0];
  if (a < 0) a = 0;
  if (b > rows) b = rows;
  int n = 0;
  for (long long i = a + (long long)blockIdx.x * 256 + threadIdx.x; i < b; i += (long long)gridDim.x * 256) n += target[i] != ignore;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = n;
  __syncthreads();
  if (threadIdx.x == 0) counts[(long long)q * gridDim.x + blockIdx.x] = red[0] + red[1] + red[2] + red[3];
}

template <int WAVES>
__device__ __forceinline__ double lg_block_sum(double x, double *red) {
  x = lg_lanes_sum<64>(x);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
  __syncthreads();
  x = red[0];
#pragma unroll
  for (int k = 1; k < WAVES; ++k) x += red[k];
  return x;
}

// the workgroups' sums in a fixed order; one workgroup, 2.4 us for 1024 of them, 7 us for 8192 (why there are no more)
__global__ void __launch_bounds__(1024)
policy_sum_kernel(int n, const double *__restrict__ partial, float *__restrict__ loss, float *__restrict__ stats) {
  __shared__ double red[16];
  double a = 0.0, b = 0.0, c = 0.0;
#pragma unroll 4
  for (int i = threadIdx.x; i < n; i += 1024) { a += partial[3 * i]; b += partial[3 * i + 1]; c += partial[3 * i + 2]; }
  a = lg_block_sum<16>(a, red); b = lg_block_sum<16>(b, red); c = lg_block_sum<16>(c, red);
  if (threadIdx.x == 0) { *loss = (float)a; stats[0] = (float)b; stats[1] = (float)c; }
}

// per sequence: the sum of its rows' log-probabilities, and 1 or (average) one over the rows that count; 5..6 us for 16 sequences of 3000 rows, a
// workgroup's chain of reads
__global__ void __launch_bounds__(256)
sequence_kernel(Rows R, const double *__restrict__ logp, int average, double *__restrict__ sums, float *__restrict__ out, float *__restrict__ each) {
  __shared__ double red[4];
  const int q = (int)blockIdx.x;
  long long a = q ? R.offset[q - 1] : 0, b = R.offset[q];
  if (a < 0) a = 0;
  if (b > R.rows) b = R.rows;
  double s = 0.0, n = 0.0;
  for (long long i = a + threadIdx.x; i < b; i += 256) { s += logp[i]; n += R.target[i] != R.ignore ? 1.0 : 0.0; }
  s = lg_block_sum<4>(s, red);
  n = lg_block_sum<4>(n, red);
  if (threadIdx.x == 0) {
    const double k = average ? 1.0 / fmax(n, 1.0) : 1.0;
    if (sums) sums[q] = s * k;
    if (out) out[q] = (float)(s * k);
    if (each) each[q] = (float)k;
  }
}

// (one workgroup, 2.3 us: the mean over the pairs needs them all)
// pairs: h = beta ((chosen - its reference) - (rejected - its reference)), loss = -(1 - e) log sigmoid(h) - e log sigmoid(-h)
__global__ void __launch_bounds__(256)
pairs_kernel(int pairs, const double *__restrict__ sums, const float *__restrict__ each, const float *__restrict__ ref, double beta, double smooth,
             float *__restrict__ loss, float *__restrict__ rewards, float *__restrict__ coef) {
  __shared__ double red[4];
  double t = 0.0;
  for (int i = threadIdx.x; i < pairs; i += 256) {
    const double a = beta * (sums[i] - (double)ref[i]), b = beta * (sums[pairs + i] - (double)ref[pairs + i]), h = a - b;
    const double e = exp(-fabs(h)), tail = log1p(e);           // -log sigmoid(+-h) = tail + max(-+h, 0)
    t += (1.0 - smooth) * (tail + fmax(-h, 0.0)) + (smooth > 0.0 ? smooth * (tail + fmax(h, 0.0)) : 0.0);   // (h may be infinite)
    // smooth - sigmoid(-h), from the exponential that does not overflow: sigmoid(h) - 1 would lose what is left of a pair far apart
    const double slope = (smooth - (h >= 0.0 ? e : 1.0) / (1.0 + e)) * beta / pairs;
    rewards[i] = (float)a;
    rewards[pairs + i] = (float)b;
    coef[i] = (float)(slope * each[i]);
    coef[pairs + i] = (float)(-slope * each[pairs + i]);
  }
  t = lg_block_sum<4>(t, red);
  if (threadIdx.x == 0) *loss = (float)(t / pairs);
}

int check_rows(const rs_logits *l, const char *name) {
  RS_REQUIRE(l && l->rows >= 0 && l->classes > 0 && l->classes <= 1 << 30 && l->ld >= l->classes && l->type >= 0 && l->type <= 2, "%s: bad size or type", name);
  RS_REQUIRE(l->sequences >= 0 && (!l->offset) == (l->sequences == 0), "%s: offsets and their number do not match", name);
  RS_REQUIRE(l->rows == 0 || (l->logits && l->target), "%s: null pointer", name);
  RS_REQUIRE(l->rows < (1LL << 31), "%s: %lld rows (offsets and counts have 32 bits)", name, l->rows);
  return RS_OK;
}
Rows rows_of(const rs_logits *l) {
  return Rows{l->logits, l->rows, l->ld, l->classes, l->sequences, l->target, l->ignore_index, l->offset, l->bad_labels};
}

constexpr int LG_GRID = 2048;             // 8 workgroups of 256 threads on each of 256 CUs, for rows that are much alike
// Long rows get a workgroup each: some cost nothing (prompts), and 6208 rows dealt to 2048 workgroups beforehand leave a third of the chip idle
// at the end.  The policy loss's stop where its partial sums would cost more.
constexpr int LG_LONG_GRID = 1 << 20;
constexpr int LG_SHORT = 4096;            // classes of the longest row that a wave holds
constexpr int LG_FEW = 256, LG_PARTS = 64;
static_assert(LG_PARTS == RS_LOGITS_PARTS && LG_FEW == RS_LOGITS_FEW_ROWS, "room of the callers' scratch");

int lesser(long long a, long long b) { return (int)(a < b ? a : b); }

// Few long rows are cut so that about 512 workgroups share them, in pieces of 2048 logits at least; 1: not cut
int parts_of(const rs_logits *l) {
  if (l->rows > LG_FEW || l->classes <= 8192) return 1;
  const int room = l->classes / 2048 < LG_PARTS ? l->classes / 2048 : LG_PARTS, want = (int)((512 + l->rows - 1) / l->rows);
  return want < room ? want : room;
}

template <typename T, int MODE>
int launch_rows(const rs_logits *l, const Rows &R, const Policy &P, const Outs &O, hipStream_t st) {
  const int V = R.classes;
#define LG_RUN_SHORT(L, N) { const int room = MODE == LG_POLICY && N < 4 ? 4 / N : 1, per = 256 / L * (L < room ? L : room), g = lesser((R.rows + per - 1) / per, LG_GRID); hipLaunchKernelGGL((short_kernel<T, MODE, L, N>), dim3(g), dim3(256), 0, st, R, P, O); return g; }
  if (V <= 16) LG_RUN_SHORT(2, 1)
  if (V <= 32) LG_RUN_SHORT(4, 1)
  if (V <= 64) LG_RUN_SHORT(8, 1)
  if (V <= 128) LG_RUN_SHORT(16, 1)
  if (V <= 256) LG_RUN_SHORT(32, 1)
  if (V <= 512) LG_RUN_SHORT(64, 1)
  if (V <= 1024) LG_RUN_SHORT(64, 2)
  if (V <= 2048) LG_RUN_SHORT(64, 4)
  if (V <= LG_SHORT) LG_RUN_SHORT(64, 8)
#undef LG_RUN_SHORT
  if constexpr (MODE == LG_BACK) {
    constexpr int NV = 4;
    const int parts = (V + 256 * LG_VEC * NV - 1) / (256 * LG_VEC * NV), across = lesser(parts, LG_GRID);
    // (a launch that most often finds nothing to do is kept small: 63 000 workgroups that leave at once take 26 us)
    hipLaunchKernelGGL((long_back_kernel<T, NV>), dim3(across, lesser(R.rows, O.skip_unit ? 2 * LG_GRID / across : 65535)), dim3(256), 0, st, R, O, parts);
    return 0;
  } else {
#define LG_RUN_LONG(TH, N, H, WV) { const int g = lesser(R.rows, MODE == LG_POLICY ? RS_POLICY_GROUPS : LG_LONG_GRID); hipLaunchKernelGGL((long_kernel<T, MODE, TH, N, H, WV>), dim3(g), dim3(TH), 0, st, R, P, O); return g; }
    if constexpr (MODE == LG_POLICY) {       // (without a gradient too: the loss has the same bits either way)
      constexpr int K = sizeof(T) / 2;       // 8 logits: 4 or 8 registers of a thread
      // (in 16 bits 128 threads to a row while 16 steps hold it: two waves share its fp64 steps and barriers, not four.  Against 256 threads:
      // 32768 x 5000 198 and 264 us, 16384 x 8192 128 and 141, 16384 x 16000 229 and 242; with 32 steps 8192 x 32768 255 and 219.
      // They spill 7 to 9 registers for it.)
      if constexpr (K == 1) {
        if (V < 9216) LG_RUN_LONG(128, 8, true, 5)
        if (V < 17408) LG_RUN_LONG(128, 16, true, 4)
      } else {
        if (V < 5120) LG_RUN_LONG(128, 4, true, 5)        // 16384 x 5000 156 us against 168; with 8 steps 16384 x 8192 229 against 218
        if (V < 10240) LG_RUN_LONG(256, 4, true, 4)
        if (V < 18432) LG_RUN_LONG(256, 8, true, 3)
      }
      if (V < 34816) LG_RUN_LONG(256, 16, true, K == 1 ? 3 : 2)
      if constexpr (K == 1) {
        if (V < 51200) LG_RUN_LONG(256, 24, true, 3)      // three rows on a CU, with 32 steps two: 8192 x 40001 267 us against 304, x 50001 333 against 355
        if (V < 67584) LG_RUN_LONG(256, 32, true, 2)
        if (V < 135168) LG_RUN_LONG(512, 32, true, 2)
      } else {
        if (V < 69632) LG_RUN_LONG(512, 16, true, 2)
      }
    }
    LG_RUN_LONG(256, 4, false, MODE == LG_POLICY ? 4 : 6)
#undef LG_RUN_LONG
  }
}

#define LG_TYPE(K, ...)                                     \
  do {                                                      \
    if (K == 0) { typedef float T; __VA_ARGS__; }           \
    else if (K == 1) { typedef __bf16 T; __VA_ARGS__; }     \
    else { typedef _Float16 T; __VA_ARGS__; }               \
  } while (0)

// rows of any kind, cut or not; returns the number of workgroups that left partial sums
template <int MODE>
int run_rows(const rs_logits *l, const Policy &P, const Outs &O, void *scratch, hipStream_t st) {
  const Rows R = rows_of(l);
  const int parts = scratch ? parts_of(l) : 1;
  int n = 0;
  if (parts > 1) {
    const int piece = ((l->classes + parts - 1) / parts + LG_VEC - 1) / LG_VEC * LG_VEC;
    const int cut = (l->classes + piece - 1) / piece;
    double *part_s = (double *)scratch;
    float *part_m = (float *)(part_s + l->rows * cut);
    LG_TYPE(l->type, hipLaunchKernelGGL((part_kernel<T, 2>), dim3(cut, (int)l->rows), dim3(256), 0, st, R, cut, piece, part_m, part_s);
            hipLaunchKernelGGL((join_kernel<T, MODE>), dim3((int)l->rows), dim3(64), 0, st, R, P, O, cut, part_m, part_s));
    n = (int)l->rows;
    if (MODE == LG_POLICY && O.dz) {
      Outs B = O;
      B.coef = P.coef; B.row_coef = 1;
      LG_TYPE(l->type, (launch_rows<T, LG_BACK>(l, R, P, B, st)));
    }
  } else {
    LG_TYPE(l->type, n = (launch_rows<T, MODE>(l, R, P, O, st)));
  }
  return n;
}

}  // namespace

extern "C" int rs_token_logprobs(const rs_logits *l, float *logp, double *logp64, float *stat, void *scratch, void *stream) {
  const int rc = check_rows(l, "rs_token_logprobs");
  if (rc != RS_OK) return rc;
  if (l->rows == 0) return RS_OK;
  RS_REQUIRE(logp || logp64, "rs_token_logprobs: null pointer");
  run_rows<LG_LOGP>(l, Policy{}, Outs{logp, logp64, (float2 *)stat, nullptr, nullptr, nullptr, 0, 0}, scratch, (hipStream_t)stream);
  RS_CHECK_LAUNCH("rs_token_logprobs");
  return RS_OK;
}

extern "C" int rs_token_logprobs_backward(const rs_logits *l, const float *stat, const float *coef, const float *gout, int flags, void *dlogits,
                                          void *stream) {
  const int rc = check_rows(l, "rs_token_logprobs_backward");
  if (rc != RS_OK) return rc;
  if (l->rows == 0) return RS_OK;
  RS_REQUIRE(stat && coef && dlogits, "rs_token_logprobs_backward: null pointer");
  RS_REQUIRE(!(flags & ~(RS_BACKWARD_SKIP_UNIT | RS_BACKWARD_ROW_COEF)), "rs_token_logprobs_backward: flags=%d", flags);
  const Outs O{nullptr, nullptr, (float2 *)stat, dlogits, coef, gout, flags & RS_BACKWARD_SKIP_UNIT, flags & RS_BACKWARD_ROW_COEF};
  LG_TYPE(l->type, (launch_rows<T, LG_BACK>(l, rows_of(l), Policy{}, O, (hipStream_t)stream)));
  RS_CHECK_LAUNCH("rs_token_logprobs_backward");
  return RS_OK;
}

extern "C" int rs_sequence_sums(const rs_logits *l, const double *logp64, int average, double *sums, float *out, float *each, void *stream) {
  const int rc = check_rows(l, "rs_sequence_sums");
  if (rc != RS_OK) return rc;
  RS_REQUIRE(l->offset && (l->rows == 0 || logp64), "rs_sequence_sums: null pointer");
  hipLaunchKernelGGL(sequence_kernel, dim3(l->sequences), dim3(256), 0, (hipStream_t)stream, rows_of(l), logp64, average, sums, out, each);
  RS_CHECK_LAUNCH("rs_sequence_sums");
  return RS_OK;
}

extern "C" int rs_preference_pairs(int pairs, const double *sums, const float *each, const float *ref, double beta, double smoothing, float *loss,
                                   float *rewards, float *coef, void *stream) {
  RS_REQUIRE(smoothing >= 0.0 && smoothing <= 0.5, "rs_preference_pairs: smoothing=%g (0 to 0.5)", smoothing);
  RS_REQUIRE(pairs > 0 && sums && each && ref && loss && rewards && coef, "rs_preference_pairs: null pointer or no pairs");
  hipLaunchKernelGGL(pairs_kernel, dim3(1), dim3(256), 0, (hipStream_t)stream, pairs, sums, each, ref, beta, smoothing, loss, rewards, coef);
  RS_CHECK_LAUNCH("rs_preference_pairs");
  return RS_OK;
}

extern "C" int rs_policy_loss(const rs_logits *l, const rs_policy *p, void *stream) {
  const int rc = check_rows(l, "rs_policy_loss");
  if (rc != RS_OK) return rc;
  RS_REQUIRE(p && p->loss && p->stats && p->partial && p->counts, "rs_policy_loss: null pointer");
  RS_REQUIRE(l->rows == 0 || (p->old_logp && p->advantages), "rs_policy_loss: null pointer");
  RS_REQUIRE(!p->dlogits == !p->coef && !p->coef == !p->stat, "rs_policy_loss: dlogits, coef and stat go together");
  RS_REQUIRE(l->offset || (p->token_mean && !p->advantages_per_sequence), "rs_policy_loss: sequences need offsets");
  hipStream_t st = (hipStream_t)stream;
  const int parts = p->token_mean ? 1 : l->sequences;
  long long splits = (l->rows / parts + 4095) / 4096;
  splits = splits < 1 ? 1 : (splits > 64 ? 64 : splits);
  RS_REQUIRE((long long)parts * splits <= p->counts_room, "rs_policy_loss: room for %d counts, %lld are needed", p->counts_room, parts * splits);
  RS_REQUIRE(parts <= 65535, "rs_policy_loss: %d sequences (at most 65535)", parts);
  RS_REQUIRE(p->partial_room >= 3 * lesser(l->rows, RS_POLICY_GROUPS), "rs_policy_loss: room for %d partial sums, %d are needed", p->partial_room,
             3 * lesser(l->rows, RS_POLICY_GROUPS));
  static_assert(RS_POLICY_GROUPS >= LG_GRID && RS_POLICY_GROUPS >= LG_FEW, "every workgroup leaves partial sums");
  // (all rows of a token mean: those of the offsets' last sequence end them)
  hipLaunchKernelGGL(count_kernel, dim3((int)splits, parts), dim3(256), 0, st, l->rows,
                     l->offset ? (p->token_mean ? l->offset + l->sequences - 1 : l->offset) : nullptr, l->target, l->ignore_index, p->counts);
  int n = 0;
  if (l->rows > 0) {
    const Policy P{p->old_logp, p->advantages, p->ref_logp, p->advantages_per_sequence, p->token_mean, p->low, p->high, p->kl_coef, p->counts, (int)splits,
                   p->coef, p->partial};
    n = run_rows<LG_POLICY>(l, P, Outs{p->logp, nullptr, (float2 *)p->stat, p->dlogits, nullptr, nullptr, 0, 0}, p->scratch, st);
  }
  hipLaunchKernelGGL(policy_sum_kernel, dim3(1), dim3(1024), 0, st, n, p->partial, p->loss, p->stats);
  RS_CHECK_LAUNCH("rs_policy_loss");
  return RS_OK;
}
