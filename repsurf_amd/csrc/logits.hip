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

template <typename T> __device__ __forceinline__ float lg_wide(T x) { return (float)x; }

constexpr int LG_VEC = 8;
template <typename T> struct Vec { T x[LG_VEC]; };
// 8 consecutive logits, aligned to one of them: global loads and stores of this device need no more
template <typename T>
__device__ __forceinline__ void lg_load(const T *p, int left, float *x) {
  if (left >= LG_VEC) {
    Vec<T> v;
    __builtin_memcpy(&v, p, sizeof(v));
#pragma unroll
    for (int i = 0; i < LG_VEC; ++i) x[i] = lg_wide(v.x[i]);
  } else {
#pragma unroll
    for (int i = 0; i < LG_VEC; ++i) x[i] = i < left ? lg_wide(p[i]) : -INFINITY;
  }
}
template <typename T>
__device__ __forceinline__ void lg_store(T *p, int left, const float *x) {
  if (left >= LG_VEC) {
    Vec<T> v;
#pragma unroll
    for (int i = 0; i < LG_VEC; ++i) v.x[i] = (T)x[i];
    __builtin_memcpy(p, &v, sizeof(v));
  } else {
#pragma unroll
    for (int i = 0; i < LG_VEC; ++i) if (i < left) p[i] = (T)x[i];
  }
}

__device__ __forceinline__ float lg_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896340736f); }
// the value that exponents are taken against: of a row that holds nothing but -infinity, 0 (exp(-inf - 0) = 0, and 0 / 0 follows)
__device__ __forceinline__ float lg_base(float m) { return m == -INFINITY ? 0.f : m; }

__device__ __forceinline__ float lg_wave_max(float x) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor(x, o));
  return x;
}
__device__ __forceinline__ double lg_wave_sum(double x) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o);
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

enum { LG_LOGP = 0, LG_POLICY = 1 };

// d loss / d log p(y) of the policy loss for one row, and its three contributions
__device__ __forceinline__ double lg_policy(const Policy &P, double w, double logp, double old, double a, bool has_ref, double ref, double *add) {
  const double r = exp(logp - old);
  const bool cut = a >= 0.0 ? r > P.hi : r < P.lo;             // the cut-off ratio is the smaller term: no gradient through it
  double each = -(cut ? (a >= 0.0 ? P.hi : P.lo) : r) * a, c = cut ? 0.0 : -a * r;
  if (r != r || a != a) each = c = r + a;
  if (has_ref) {
    const double d = ref - logp, e = expm1(d);                 // exp(d) - 1 - d: not negative, and its mean over the policy's own draws is the KL
    each += P.kl * (e - d);
    c -= P.kl * e;
    add[1] += w * (e - d);
  }
  add[0] += w * each;
  add[2] += cut ? w : 0.0;
  return w * c;
}

// One team of WAVES waves per row, `4 / WAVES` (at least 1) teams per workgroup, rows taken in turn by the grid's teams.
//   LG_LOGP:   logp / logp64 / stat of every row
//   LG_POLICY: the policy loss's contributions, logp, and -- with dlogits -- the gradient and coef / stat for a later backward pass
template <typename T, int MODE, int WAVES>
__global__ void __launch_bounds__(WAVES < 4 ? 256 : WAVES * 64)
rows_kernel(Rows R, Policy P, float *__restrict__ logp_out, double *__restrict__ logp64, float2 *__restrict__ stat, T *__restrict__ dz) {
  constexpr int TEAMS = WAVES < 4 ? 4 / WAVES : 1;
  constexpr int LANES = WAVES * 64;
  __shared__ float red_m[WAVES];
  __shared__ double red_s[WAVES];
  __shared__ float row_c;
  __shared__ double sums[3][TEAMS];
  static_assert(WAVES == 1 || TEAMS == 1, "a team of several waves is the workgroup: its barriers are the workgroup's");
  const int team = (int)threadIdx.x / LANES, lane = (int)threadIdx.x % LANES, wave = lane >> 6;
  double add[3] = {0.0, 0.0, 0.0};
  const int V = R.classes;
  for (long long row = (long long)blockIdx.x * TEAMS + team; row < R.rows; row += (long long)gridDim.x * TEAMS) {
    const T *__restrict__ z = (const T *)R.z + row * R.ld;
    const long long y = R.target[row];
    int owner = 0;
    if (R.offset) owner = lg_owner(R.offset, R.sequences, row);
    const bool counts = y != R.ignore && (!R.offset || owner < R.sequences);
    const bool bad = counts && (y < 0 || y >= V);
    if (!counts || bad) {               // nothing of the row is read
      const float fill = bad ? __uint_as_float(0x7FC00000u) : 0.f;
      if (lane == 0) {
        if (logp_out) logp_out[row] = fill;
        if (logp64) logp64[row] = (double)fill;
        if (stat) stat[row] = make_float2(fill, 0.f);
        if (bad && R.bad) atomicAdd(R.bad, 1);
        if (MODE == LG_POLICY) {
          if (P.coef) P.coef[row] = fill;
          if (bad) { add[0] += (double)fill; add[1] += (double)fill; add[2] += (double)fill; }
        }
      }
      if (MODE == LG_POLICY && dz) {
        float x[LG_VEC];
#pragma unroll
        for (int i = 0; i < LG_VEC; ++i) x[i] = fill;
        for (int j = lane * LG_VEC; j < V; j += LANES * LG_VEC) lg_store(dz + row * V + j, V - j, x);
      }
      continue;
    }
    float m = -INFINITY;
    double s = 0.0;
    for (int j = lane * LG_VEC; j < V; j += LANES * LG_VEC) {
      float x[LG_VEC];
      lg_load(z + j, V - j, x);
      float top = x[0];
#pragma unroll
      for (int i = 1; i < LG_VEC; ++i) top = fmaxf(top, x[i]);
      if (top > m) { s *= (double)lg_exp(m - top); m = top; }       // (m = -inf at first: s is 0)
      const float base = lg_base(m);
      float e = 0.f;
#pragma unroll
      for (int i = 0; i < LG_VEC; ++i) e += lg_exp(x[i] - base);
      s += (double)e;
    }
    float M = lg_wave_max(m);
    if (WAVES > 1) {
      __syncthreads();                  // (the row before this one is done with the scratch)
      if ((lane & 63) == 0) red_m[wave] = M;
      __syncthreads();
      M = red_m[0];
      for (int k = 1; k < WAVES; ++k) M = fmaxf(M, red_m[k]);
    }
    s = lg_wave_sum(m == -INFINITY ? s : s * (double)lg_exp(m - lg_base(M)));
    if (WAVES > 1) {
      if ((lane & 63) == 0) red_s[wave] = s;
      __syncthreads();
      s = 0.0;
      for (int k = 0; k < WAVES; ++k) s += red_s[k];
    }
    const float inv = (float)(1.0 / s);
    float c = 0.f;
    if (lane == 0) {
      const double lp = (double)lg_wide(z[y]) - (double)M - log(s);
      if (logp_out) logp_out[row] = (float)lp;
      if (logp64) logp64[row] = lp;
      if (stat) stat[row] = make_float2(M, inv);
      if (MODE == LG_POLICY) {
        int n = 0;
        const int first = P.token_mean ? 0 : owner * P.splits;
        for (int k = 0; k < P.splits; ++k) n += P.counts[first + k];
        const double w = 1.0 / (double)n / (P.token_mean ? 1.0 : (double)R.sequences);
        c = (float)lg_policy(P, w, lp, (double)P.old_logp[row], (double)P.adv[P.adv_per_sequence ? (long long)owner : row], P.ref != nullptr,
                             P.ref ? (double)P.ref[row] : 0.0, add);
        if (P.coef) P.coef[row] = c;
      }
    }
    if (MODE == LG_POLICY && dz) {
      if (WAVES > 1) {
        if (lane == 0) row_c = c;
        __syncthreads();
        c = row_c;
      } else c = __shfl(c, 0);
      const float base = lg_base(M), scale = -c * inv;
      for (int j = lane * LG_VEC; j < V; j += LANES * LG_VEC) {
        float x[LG_VEC];
        lg_load(z + j, V - j, x);
#pragma unroll
        for (int i = 0; i < LG_VEC; ++i) x[i] = rs_fma(lg_exp(x[i] - base), scale, j + i == (int)y ? c : 0.f);
        lg_store(dz + row * V + j, V - j, x);
      }
    }
  }
  if (MODE == LG_POLICY) {
    if (lane == 0) { sums[0][team] = add[0]; sums[1][team] = add[1]; sums[2][team] = add[2]; }
    __syncthreads();
    if (threadIdx.x == 0)
      for (int k = 0; k < 3; ++k) {
        double t = 0.0;
        for (int i = 0; i < TEAMS; ++i) t += sums[k][i];
        P.partial[(long long)blockIdx.x * 3 + k] = t;
      }
  }
}

// dz = c ([j = y] - exp(z_j - M) / s) with the rows' saved M and 1 / s; c = coef of the row (or of its sequence) times *gout
template <typename T, int WAVES>
__global__ void __launch_bounds__(WAVES < 4 ? 256 : WAVES * 64)
rows_backward_kernel(Rows R, const float2 *__restrict__ stat, const float *__restrict__ coef, const float *__restrict__ gout, int skip_unit,
                     T *__restrict__ dz) {
  constexpr int TEAMS = WAVES < 4 ? 4 / WAVES : 1;
  constexpr int LANES = WAVES * 64;
  const float up = gout ? *gout : 1.f;
  if (skip_unit && up == 1.f) return;
  const int team = (int)threadIdx.x / LANES, lane = (int)threadIdx.x % LANES;
  const int V = R.classes;
  for (long long row = (long long)blockIdx.x * TEAMS + team; row < R.rows; row += (long long)gridDim.x * TEAMS) {
    const T *__restrict__ z = (const T *)R.z + row * R.ld;
    const long long y = R.target[row];
    int owner = 0;
    if (R.offset) owner = lg_owner(R.offset, R.sequences, row);
    const bool counts = y != R.ignore && (!R.offset || owner < R.sequences);
    float c = 0.f;
    if (counts) c = coef[R.offset ? (long long)owner : row] * up;
    if (counts && (y < 0 || y >= V)) c = __uint_as_float(0x7FC00000u);
    if (!counts || c == 0.f || c != c) {
      float x[LG_VEC];
#pragma unroll
      for (int i = 0; i < LG_VEC; ++i) x[i] = c;
      for (int j = lane * LG_VEC; j < V; j += LANES * LG_VEC) lg_store(dz + row * V + j, V - j, x);
      continue;
    }
    const float2 st = stat[row];
    const float base = lg_base(st.x), scale = -c * st.y;
    for (int j = lane * LG_VEC; j < V; j += LANES * LG_VEC) {
      float x[LG_VEC];
      lg_load(z + j, V - j, x);
#pragma unroll
      for (int i = 0; i < LG_VEC; ++i) x[i] = rs_fma(lg_exp(x[i] - base), scale, j + i == (int)y ? c : 0.f);
      lg_store(dz + row * V + j, V - j, x);
    }
  }
}

// rows that count, of sequence blockIdx.y (of all rows without offsets), in gridDim.x parts
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

__device__ __forceinline__ double lg_block_sum(double x, double *red) {
  x = lg_wave_sum(x);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
  __syncthreads();
  return (red[0] + red[1]) + (red[2] + red[3]);
}

__global__ void __launch_bounds__(256)
policy_sum_kernel(int n, const double *__restrict__ partial, float *__restrict__ loss, float *__restrict__ stats) {
  __shared__ double red[4];
  double a = 0.0, b = 0.0, c = 0.0;
  for (int i = threadIdx.x; i < n; i += 256) { a += partial[3 * i]; b += partial[3 * i + 1]; c += partial[3 * i + 2]; }
  a = lg_block_sum(a, red); b = lg_block_sum(b, red); c = lg_block_sum(c, red);
  if (threadIdx.x == 0) { *loss = (float)a; stats[0] = (float)b; stats[1] = (float)c; }
}

// per sequence: the sum of its rows' log-probabilities, and 1 or (average) one over the rows that count
__global__ void __launch_bounds__(256)
sequence_kernel(Rows R, const double *__restrict__ logp, int average, double *__restrict__ sums, float *__restrict__ out, float *__restrict__ each) {
  __shared__ double red[4];
  const int q = (int)blockIdx.x;
  long long a = q ? R.offset[q - 1] : 0, b = R.offset[q];
  if (a < 0) a = 0;
  if (b > R.rows) b = R.rows;
  double s = 0.0, n = 0.0;
  for (long long i = a + threadIdx.x; i < b; i += 256) { s += logp[i]; n += R.target[i] != R.ignore ? 1.0 : 0.0; }
  s = lg_block_sum(s, red);
  n = lg_block_sum(n, red);
  if (threadIdx.x == 0) {
    const double k = average ? 1.0 / fmax(n, 1.0) : 1.0;
    if (sums) sums[q] = s * k;
    if (out) out[q] = (float)(s * k);
    if (each) each[q] = (float)k;
  }
}

// pairs: h = beta ((chosen - its reference) - (rejected - its reference)), loss = -(1 - e) log sigmoid(h) - e log sigmoid(-h)
__global__ void __launch_bounds__(256)
pairs_kernel(int pairs, const double *__restrict__ sums, const float *__restrict__ each, const float *__restrict__ ref, double beta, double smooth,
             float *__restrict__ loss, float *__restrict__ rewards, float *__restrict__ coef) {
  __shared__ double red[4];
  double t = 0.0;
  for (int i = threadIdx.x; i < pairs; i += 256) {
    const double a = beta * (sums[i] - (double)ref[i]), b = beta * (sums[pairs + i] - (double)ref[pairs + i]), h = a - b;
    const double tail = log1p(exp(-fabs(h)));                  // -log sigmoid(+-h) = tail + max(-+h, 0)
    t += (1.0 - smooth) * (tail + fmax(-h, 0.0)) + (smooth > 0.0 ? smooth * (tail + fmax(h, 0.0)) : 0.0);   // (h may be infinite)
    const double slope = (1.0 / (1.0 + exp(-h)) - (1.0 - smooth)) * beta / pairs;
    rewards[i] = (float)a;
    rewards[pairs + i] = (float)b;
    coef[i] = (float)(slope * each[i]);
    coef[pairs + i] = (float)(-slope * each[pairs + i]);
  }
  t = lg_block_sum(t, red);
  if (threadIdx.x == 0) *loss = (float)(t / pairs);
}

constexpr int LG_GRID = 2048;

int check_rows(const rs_logits *l, const char *name) {
  RS_REQUIRE(l && l->rows >= 0 && l->classes > 0 && l->classes <= 1 << 30 && l->ld >= l->classes && l->type >= 0 && l->type <= 2, "%s: bad size or type", name);
  RS_REQUIRE(l->sequences >= 0 && (!l->offset) == (l->sequences == 0), "%s: offsets and their number do not match", name);
  RS_REQUIRE(l->rows == 0 || (l->logits && l->target), "%s: null pointer", name);
  RS_REQUIRE(!l->offset || l->rows < (1LL << 31), "%s: too many rows for 32-bit offsets", name);
  return RS_OK;
}
Rows rows_of(const rs_logits *l) {
  return Rows{l->logits, l->rows, l->ld, l->classes, l->sequences, l->target, l->ignore_index, l->offset, l->bad_labels};
}

// waves of a row's team: one up to 1024 classes, a workgroup of 4 or 16 above
int waves_of(int classes) { return classes <= 1024 ? 1 : (classes <= 16384 ? 4 : 16); }
int grid_of(long long rows, int waves) {
  const long long need = waves == 1 ? (rows + 3) / 4 : rows;
  return (int)(need < LG_GRID ? need : LG_GRID);
}

#define LG_WAVES(W, ...)                                    \
  do {                                                      \
    if (W == 1) { constexpr int WAVES = 1; __VA_ARGS__; }   \
    else if (W == 4) { constexpr int WAVES = 4; __VA_ARGS__; } \
    else { constexpr int WAVES = 16; __VA_ARGS__; }         \
  } while (0)
#define LG_TYPE(K, ...)                                     \
  do {                                                      \
    if (K == 0) { typedef float T; __VA_ARGS__; }           \
    else if (K == 1) { typedef __bf16 T; __VA_ARGS__; }     \
    else { typedef _Float16 T; __VA_ARGS__; }               \
  } while (0)

}  // namespace

extern "C" int rs_token_logprobs(const rs_logits *l, float *logp, double *logp64, float *stat, void *stream) {
  const int rc = check_rows(l, "rs_token_logprobs");
  if (rc != RS_OK) return rc;
  if (l->rows == 0) return RS_OK;
  RS_REQUIRE(logp || logp64, "rs_token_logprobs: null pointer");
  const int w = waves_of(l->classes);
  LG_TYPE(l->type, LG_WAVES(w, hipLaunchKernelGGL((rows_kernel<T, LG_LOGP, WAVES>), dim3(grid_of(l->rows, w)), dim3(WAVES < 4 ? 256 : WAVES * 64), 0,
                                                  (hipStream_t)stream, rows_of(l), Policy{}, logp, logp64, (float2 *)stat, (T *)nullptr)));
  RS_CHECK_LAUNCH("rs_token_logprobs");
  return RS_OK;
}

extern "C" int rs_token_logprobs_backward(const rs_logits *l, const float *stat, const float *coef, const float *gout, int skip_unit, void *dlogits,
                                          void *stream) {
  const int rc = check_rows(l, "rs_token_logprobs_backward");
  if (rc != RS_OK) return rc;
  if (l->rows == 0) return RS_OK;
  RS_REQUIRE(stat && coef && dlogits, "rs_token_logprobs_backward: null pointer");
  const int w = waves_of(l->classes);
  LG_TYPE(l->type, LG_WAVES(w, hipLaunchKernelGGL((rows_backward_kernel<T, WAVES>), dim3(grid_of(l->rows, w)), dim3(WAVES < 4 ? 256 : WAVES * 64), 0,
                                                  (hipStream_t)stream, rows_of(l), (const float2 *)stat, coef, gout, skip_unit, (T *)dlogits)));
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
  const int w = waves_of(l->classes), n = grid_of(l->rows, w);
  RS_REQUIRE(3 * n <= p->partial_room, "rs_policy_loss: room for %d partial sums, %d are needed", p->partial_room, 3 * n);
  // (all rows of a token mean: those of the offsets' last sequence end them)
  hipLaunchKernelGGL(count_kernel, dim3((int)splits, parts), dim3(256), 0, st, l->rows,
                     l->offset ? (p->token_mean ? l->offset + l->sequences - 1 : l->offset) : nullptr, l->target, l->ignore_index, p->counts);
  if (l->rows > 0) {
    Policy P{p->old_logp, p->advantages, p->ref_logp, p->advantages_per_sequence, p->token_mean, p->low, p->high, p->kl_coef, p->counts, (int)splits,
             p->coef, p->partial};
    LG_TYPE(l->type, LG_WAVES(w, hipLaunchKernelGGL((rows_kernel<T, LG_POLICY, WAVES>), dim3(n), dim3(WAVES < 4 ? 256 : WAVES * 64), 0, st, rows_of(l), P,
                                                    p->logp, (double *)nullptr, (float2 *)p->stat, (T *)p->dlogits)));
  }
  hipLaunchKernelGGL(policy_sum_kernel, dim3(1), dim3(256), 0, st, n, p->partial, p->loss, p->stats);
  RS_CHECK_LAUNCH("rs_policy_loss");
  return RS_OK;
}
