// adamw.hip — AdamW over a list of fp32 or bf16 tensors at once, with its two moments in 32 or in 8 bits (gfx950).
//
//   m += (g - m)(1 - b1);   v = b2 v + (1 - b2) g^2;   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// The moments of a parameter group live in flat buffers in which every tensor starts at a multiple of 256 elements, so a 256-element
// block belongs to one tensor and one wave takes a block at a time, four consecutive elements per lane.
//
// 8-bit moments: the elements of a block share one exponent E, the exponent field of the block's largest finite |x|.  With
// y = |x| 2^(F - E), which puts that element into exponent field F of an fp32 word, a code is the top of y's word: (bits(y) + r) >> 20,
// three mantissa bits, and the linear spacing at the bottom is fp32's own denormal range.  exp_avg has a sign and four exponent bits
// (F = 14, 16 powers of two below the largest), exp_avg_sq five exponent bits (F = 30): the square root of its range is that of
// exp_avg.  r spreads 16 random bits over the 20 that are cut off, so a value is rounded up with the probability of its cut-off part:
// rounded to nearest, b2 v would round back to v (a step of the code is 6..12 %, 1 - b2 is 0.1 %) and a second moment could never
// decay.  A positive v keeps at least the smallest code, so a moment m never meets a vanished v.  Code 127 of m stands for NaN, code
// 255 of v for infinity.
//
// bf16 parameters: the fp32 master's upper half, rounded, IS the parameter; `low` keeps what the rounding cut off (16 signed bits), so
// master bits = (parameter bits << 16) + low and a parameter that is written from outside moves its master with it.
//
// Bound by memory: every value is read and written once.  A workgroup takes one chunk of 2048 elements of one tensor, all of its loads in
// flight at once; workgroups that loop over chunks (2048 of them) were 8..16 % slower, 4096 elements a chunk no faster.  Measured: 100.7 M fp32
// parameters with fp32 moments 498 us (28 bytes each, 5.7 TB/s), 59.6 M bf16 parameters 272 us (26 bytes, 5.7 TB/s), 268 M fp32 parameters
// with 8-bit moments 763 us (16 bytes, 5.6 TB/s), 100.7 M bf16 parameters with 8-bit moments 239 us (14 bytes, 5.9 TB/s); 1.48 M in 67
// tensors 9.3 us, most of it the launch, two dependent reads and the counting of finished workgroups (1.2 us).
#include "rs_common.h"
#include <math.h>

namespace {

constexpr int AW_THREADS = 256;
constexpr int AW_BLOCK = 256;             // elements that share an exponent
constexpr int AW_UNROLL = 2;              // blocks a wave has in flight
constexpr int AW_CHUNK = AW_BLOCK * (AW_THREADS / RS_WAVE) * AW_UNROLL;
constexpr int AW_SQ_CHUNK = 8192;         // gradients a workgroup squares at a time
constexpr int AW_MAX = 80;                // tensors per launch: the table rides in the kernel arguments
constexpr int AW_COUNTS = RS_ADAMW_DONE / 16 - 1;      // counters of finished workgroups, below the one of all
constexpr int AW_FIELD_M = 14, AW_FIELD_V = 30;
constexpr float AW_EPS = 1e-9f;           // (1e-19 over sqrt(1 - b2^t), 3e-18 at b2 = 0.999, is below half a unit of what is larger)

struct AwTable {
  void *p[AW_MAX];
  const void *g[AW_MAX];
  long long n[AW_MAX];
  long long at[AW_MAX];
  int slot[AW_MAX];
  int blk_end[AW_MAX];                    // running number of chunks up to and including tensor i
  int count;
};

struct AwArgs {
  void *m, *v;                            // flat moments: fp32, or codes
  unsigned char *me, *ve;                 // 8 bits: one exponent field per block
  short *low;
  int *step, *done;
  const double *hyper_dev;                // captured launches read their hyper-parameters from device memory
  double hyper[7];                        // lr, beta1, beta2, eps, weight_decay, ln beta1, ln beta2
  const float *clip;                      // a factor for every gradient, or null
  unsigned seed;
};

static_assert(sizeof(AwTable) + sizeof(AwArgs) + 16 <= 4096, "the tables ride in the kernel arguments (4 KB)");

// 32-bit integer hash; the odd factors are the fractions of the square roots of 2 and 3
__device__ __forceinline__ unsigned aw_mix(unsigned x) {
  x = (x ^ (x >> 16)) * 0x6A09E667u;
  x = (x ^ (x >> 15)) * 0xBB67AE85u;
  return x ^ (x >> 16);
}
constexpr unsigned AW_PHI = 0x9E3779B9u;  // 2^32 / golden ratio

__device__ __forceinline__ unsigned aw_encode(float x, int shift, unsigned dither16, unsigned top) {
  const unsigned y = __float_as_uint(ldexpf(fabsf(x), shift));
  return min((y + ((dither16 << 4) | 8u)) >> 20, top);
}
__device__ __forceinline__ unsigned aw_encode_m(float x, int e, unsigned d) {
  return aw_encode(x, AW_FIELD_M - e, d, 127u) | ((__float_as_uint(x) >> 24) & 0x80u);
}
__device__ __forceinline__ unsigned aw_encode_v(float x, int e, unsigned d) {
  return max(aw_encode(x, AW_FIELD_V - e, d, 255u), x > 0.f ? 1u : 0u);
}
__device__ __forceinline__ float aw_decode_m(unsigned c, int e) {
  const float a = (c & 127u) == 127u ? __uint_as_float(0x7FC00000u) : ldexpf(__uint_as_float((c & 127u) << 20), e - AW_FIELD_M);
  return __uint_as_float(__float_as_uint(a) | ((c & 0x80u) << 24));
}
__device__ __forceinline__ float aw_decode_v(unsigned c, int e) {
  return c == 255u ? __uint_as_float(0x7F800000u) : ldexpf(__uint_as_float(c << 20), e - AW_FIELD_V);
}
// exponent field of |x|; 0 for what is not finite: it must not move the other elements' grid
__device__ __forceinline__ unsigned aw_field(float x) {
  const unsigned f = (__float_as_uint(x) >> 23) & 255u;
  return f == 255u ? 0u : f;
}

// (a word that is no number without its parameter being none: +-0 and infinity never carry a remainder of that sign, such a parameter
// was written from outside, and its remainder is dropped)
__device__ __forceinline__ float aw_master(unsigned p_high, int low) {
  const float x = __uint_as_float(p_high + (unsigned)low);
  return x != x ? __uint_as_float(p_high) : x;
}
// the master's word as it is kept: its upper half rounded is the parameter, its lower half, as a signed number, the remainder
__device__ __forceinline__ unsigned aw_word(float x) { return x != x ? 0x7FC00000u : __float_as_uint(x); }

// The tensor of a chunk: as many as have their running number at or below it.  All of the table's numbers are asked for at once, one per
// lane (a bisection is seven reads, each waiting for the one before).
struct AwFind {
  int a, b;
  __device__ __forceinline__ explicit AwFind(const AwTable &T) {
    const int lane = (int)threadIdx.x & 63;
    a = lane < T.count ? T.blk_end[lane] : 0x7FFFFFFF;
    b = 64 + lane < T.count ? T.blk_end[64 + lane < AW_MAX ? 64 + lane : 0] : 0x7FFFFFFF;
  }
  __device__ __forceinline__ int operator()(int chunk) const { return (int)(__popcll(__ballot(chunk >= a)) + __popcll(__ballot(chunk >= b))); }
};

template <bool BF16> struct AwType { typedef float T; };
template <> struct AwType<true> { typedef unsigned short T; };

// four consecutive elements as the words they come in; `left` of them exist.  The address is aligned to the element only: global loads and
// stores of this device need no more.
template <typename T> struct Four { unsigned w[sizeof(T)]; };
template <typename T>
__device__ __forceinline__ Four<T> aw_load(const T *p, long long left) {
  Four<T> r;
  if (left >= 4) { __builtin_memcpy(&r, p, sizeof(r)); return r; }
  T x[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = i < left ? p[i] : T(0);
  __builtin_memcpy(&r, x, sizeof(r));
  return r;
}
template <typename T>
__device__ __forceinline__ void aw_store(T *p, const Four<T> &r, long long left) {
  if (left >= 4) { __builtin_memcpy(p, &r, sizeof(r)); return; }
  T x[4];
  __builtin_memcpy(x, &r, sizeof(r));
#pragma unroll
  for (int i = 0; i < 4; ++i) if (i < left) p[i] = x[i];
}
__device__ __forceinline__ float aw_get(const Four<float> &r, int i) { return __uint_as_float(r.w[i]); }
__device__ __forceinline__ unsigned aw_high(const Four<unsigned short> &r, int i) { return i & 1 ? r.w[i >> 1] & 0xFFFF0000u : r.w[i >> 1] << 16; }
__device__ __forceinline__ float aw_get(const Four<unsigned short> &r, int i) { return __uint_as_float(aw_high(r, i)); }      // bf16
__device__ __forceinline__ int aw_get(const Four<short> &r, int i) { return i & 1 ? (int)r.w[i >> 1] >> 16 : (int)(r.w[i >> 1] << 16) >> 16; }
__device__ __forceinline__ unsigned aw_get(const Four<unsigned char> &r, int i) { return (r.w[0] >> (8 * i)) & 255u; }
// the larger of two pairs of 16-bit numbers, each half by itself, over a wave
__device__ __forceinline__ unsigned aw_pair_max(unsigned a, unsigned b) {
  typedef unsigned short us2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(us2, a), __builtin_bit_cast(us2, b)));
}
__device__ __forceinline__ unsigned aw_wave_pair_max(unsigned v) {
  v = aw_pair_max(v, rs_dpp<RS_DPP_QUAD_XOR1>(v));
  v = aw_pair_max(v, rs_dpp<RS_DPP_QUAD_XOR2>(v));
  v = aw_pair_max(v, rs_dpp<RS_DPP_ROW_HALF_MIRROR>(v));
  v = aw_pair_max(v, rs_dpp<RS_DPP_ROW_MIRROR>(v));
  auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = aw_pair_max((unsigned)r[0], (unsigned)r[1]);
  auto s = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return rs_uniform((int)aw_pair_max((unsigned)s[0], (unsigned)s[1]));
}

// what a launch's elements share, and what a tensor's do
struct AwShared {
  float eps, decay, omb1, b2, omb2, clip;
  float step_size, inv_bc2;
  unsigned key;
};

// N blocks of a wave from element `b` of a tensor on.  WHOLE: all of their elements exist, so the loads ask no question and leave in one go.
template <bool BF16, int BITS, int N, bool WHOLE>
struct AwBlocks {
  typedef typename AwType<BF16>::T PT;
  Four<PT> p[N], g[N];
  Four<short> low[N];
  Four<float> m[N], v[N];
  Four<unsigned char> mc[N], vc[N];
  int em[N], ev[N];

  __device__ __forceinline__ void load(const AwArgs &A, const PT *__restrict__ pp, const PT *__restrict__ gp, long long at, long long b, int lane, long long n) {
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const long long e = b + u * AW_BLOCK + lane * 4, left = WHOLE ? 4 : n - e;
      p[u] = aw_load(pp + e, left);
      g[u] = aw_load(gp + e, left);
      if constexpr (BF16) low[u] = aw_load((const short *)A.low + at + e, 4);
      if constexpr (BITS == 32) {         // (the flat buffers have the block's tail, as zeros)
        m[u] = aw_load((const float *)A.m + at + e, 4);
        v[u] = aw_load((const float *)A.v + at + e, 4);
      } else {
        mc[u] = aw_load((const unsigned char *)A.m + at + e, 4);
        vc[u] = aw_load((const unsigned char *)A.v + at + e, 4);
        em[u] = A.me[(at + b + u * AW_BLOCK) >> 8];
        ev[u] = A.ve[(at + b + u * AW_BLOCK) >> 8];
      }
    }
  }
  __device__ __forceinline__ void update(const AwArgs &A, const AwShared &S, PT *__restrict__ pp, long long at, long long b, int lane, long long n) {
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const long long e = b + u * AW_BLOCK + lane * 4, left = WHOLE ? 4 : n - e;
      const long long block = (at + b + u * AW_BLOCK) >> 8;
      unsigned fields = 0u, word[4];
      float mi[4], vi[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float x, gi = aw_get(g[u], i);
        if constexpr (BF16) x = aw_master(aw_high(p[u], i), aw_get(low[u], i)); else x = aw_get(p[u], i);
        if constexpr (BITS == 8) { mi[i] = aw_decode_m(aw_get(mc[u], i), em[u]); vi[i] = aw_decode_v(aw_get(vc[u], i), ev[u]); }
        else { mi[i] = aw_get(m[u], i); vi[i] = aw_get(v[u], i); }
        gi *= S.clip;
        // Each operation of the moments is rounded by itself, as the formula is written: an 8-bit moment next to a border of its grid then falls
        // to the side that the elementary operations choose, and a step larger or smaller by an eighth does not hang on a fused rounding.
        mi[i] = mi[i] + (gi - mi[i]) * S.omb1;
        vi[i] = vi[i] * S.b2 + (S.omb2 * gi) * gi;
        // The device's own root and reciprocal, each off by one unit: the correctly rounded ones are 25 instructions for an error that lr
        // scales away.  The root takes denormals as zero, so v is raised to the smallest normal number (1e-19 beside eps); beside an eps that
        // does not cover that, denormals are taken 2^64 higher (a vanished v is the smallest of them: no gradient and no eps is no step).
        float root;
        if (S.eps < AW_EPS) {
          const bool small = vi[i] < 1.17549435e-38f;
          root = __builtin_amdgcn_sqrtf(small ? fmaxf(vi[i], 1.40129846e-45f) * 0x1p64f : vi[i]) * (small ? 0x1p-32f : 1.f);
        } else root = __builtin_amdgcn_sqrtf(fmaxf(vi[i], 1.17549435e-38f));
        x = rs_fma(-S.step_size, mi[i] * __builtin_amdgcn_rcpf(rs_fma(root, S.inv_bc2, S.eps)), x * S.decay);
        if (!WHOLE && i >= left) mi[i] = vi[i] = x = 0.f;
        if constexpr (BF16) word[i] = aw_word(x); else p[u].w[i] = __float_as_uint(x);
        if constexpr (BITS == 8) fields = aw_pair_max(fields, aw_field(mi[i]) << 16 | aw_field(vi[i]));
        else { m[u].w[i] = __float_as_uint(mi[i]); v[u].w[i] = __float_as_uint(vi[i]); }
      }
      if constexpr (BF16) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          p[u].w[i] = ((word[2 * i + 1] + 0x8000u) & 0xFFFF0000u) | ((word[2 * i] + 0x8000u) >> 16);
          low[u].w[i] = (word[2 * i + 1] << 16) | (word[2 * i] & 0xFFFFu);
        }
      }
      aw_store(pp + e, p[u], left);
      if constexpr (BF16) aw_store(A.low + at + e, low[u], 4);
      if constexpr (BITS == 32) {
        aw_store((float *)A.m + at + e, m[u], 4);
        aw_store((float *)A.v + at + e, v[u], 4);
      } else {
        fields = aw_wave_pair_max(fields);
        const int fm = (int)(fields >> 16), fv = (int)(fields & 255u);
        const unsigned k = aw_mix(S.key + (unsigned)block) + (unsigned)(lane * 4) * AW_PHI;
        unsigned a = 0u, c = 0u;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const unsigned r = aw_mix(k + i * AW_PHI);
          a |= aw_encode_m(mi[i], fm, r >> 16) << (8 * i);
          c |= aw_encode_v(vi[i], fv, r & 0xFFFFu) << (8 * i);
        }
        mc[u].w[0] = a;
        vc[u].w[0] = c;
        aw_store((unsigned char *)A.m + at + e, mc[u], 4);
        aw_store((unsigned char *)A.v + at + e, vc[u], 4);
        if (lane == 0) { A.me[block] = (unsigned char)fm; A.ve[block] = (unsigned char)fv; }
      }
    }
  }
};

template <bool BF16, int BITS>
__global__ void __launch_bounds__(AW_THREADS)
adamw_kernel(AwTable T, AwArgs A) {
  typedef typename AwType<BF16>::T PT;
  double lr = A.hyper[0], beta1 = A.hyper[1], beta2 = A.hyper[2], eps64 = A.hyper[3], wd = A.hyper[4], lnb1 = A.hyper[5], lnb2 = A.hyper[6];
  if (A.hyper_dev) {
    lr = A.hyper_dev[0]; beta1 = A.hyper_dev[1]; beta2 = A.hyper_dev[2]; eps64 = A.hyper_dev[3]; wd = A.hyper_dev[4];
    lnb1 = A.hyper_dev[5]; lnb2 = A.hyper_dev[6];
  }
  AwShared S{(float)eps64, (float)(1.0 - lr * wd), (float)(1.0 - beta1), (float)beta2, (float)(1.0 - beta2), 1.f, 0.f, 1.f, 0u};
  if (A.clip) S.clip = *A.clip;
  const int wave = rs_uniform((int)threadIdx.x >> 6), lane = (int)threadIdx.x & 63;

  const int c = (int)blockIdx.x, ti = AwFind(T)(c);
  const long long n = T.n[ti], at = T.at[ti];
  const long long b = (long long)(c - (ti ? T.blk_end[ti - 1] : 0)) * AW_CHUNK + wave * (AW_BLOCK * AW_UNROLL);
  PT *__restrict__ p = (PT *)T.p[ti];
  const PT *__restrict__ g = (const PT *)T.g[ti];
  const bool whole = b + AW_BLOCK * AW_UNROLL <= n;
  AwBlocks<BF16, BITS, AW_UNROLL, true> W;
  if (whole) W.load(A, p, g, at, b, lane, n);                 // (in front of the step count, which the loads do not need)
  const int t = A.step[T.slot[ti]] + 1;
  // 1 - beta^t as -expm1(t ln beta): fp32 loses nothing where beta^t is near 1
  S.step_size = (float)(lr / (double)-expm1f((float)(lnb1 * t)));
  S.inv_bc2 = 1.f / sqrtf(-expm1f((float)(lnb2 * t)));
  S.key = aw_mix(A.seed + (unsigned)t * AW_PHI);
  if (whole) W.update(A, S, p, at, b, lane, n);
  else {
    for (int u = 0; u < AW_UNROLL && b + u * AW_BLOCK < n; ++u) {
      AwBlocks<BF16, BITS, 1, false> E;
      E.load(A, p, g, at, b + u * AW_BLOCK, lane, n);
      E.update(A, S, p, at, b + u * AW_BLOCK, lane, n);
    }
  }
  // The last workgroup advances the counters of this launch's tensors: every workgroup has read them by then (its reads feed its
  // stores, in front of the barrier and the count).  No fence: nothing written here is read before the next launch.  Counted in two
  // levels, in cache lines of their own: hundreds of workgroups that end together do not queue for one word.
  __shared__ int last;
  __syncthreads();
  if (threadIdx.x == 0) {
    const int k = (int)blockIdx.x % AW_COUNTS, mine = ((int)gridDim.x - 1 - k) / AW_COUNTS + 1, groups = min((int)gridDim.x, AW_COUNTS);
    last = 0;
    if (atomicAdd(A.done + 16 * (k + 1), 1) == mine - 1) {
      A.done[16 * (k + 1)] = 0;
      last = atomicAdd(A.done, 1) == groups - 1;
    }
  }
  __syncthreads();
  if (last) {
    if ((int)threadIdx.x < T.count) A.step[T.slot[threadIdx.x]] += 1;
    if (threadIdx.x == 0) *A.done = 0;
  }
}

// ---- the gradients' common norm -------------------------------------------------------------------------------------
// Bound by memory: 100.7 M fp32 gradients 101 us = 4.0 TB/s (what the step before wrote is still on its way to memory), bf16 45 us.
// partial[b] = sum of the squares of workgroup b's chunks, in fp64 and in an order that the sizes fix: the norm is the correctly rounded one but
// for a few cases in a thousand million, and the factor that every gradient is multiplied by hangs on no order.
template <bool BF16>
__global__ void __launch_bounds__(AW_THREADS)
grad_sq_kernel(AwTable T, double *__restrict__ partial) {
  typedef typename AwType<BF16>::T PT;
  constexpr int E = 16 / sizeof(PT), U = AW_SQ_CHUNK / (AW_THREADS * E);      // 16 bytes of a thread at a time
  __shared__ double red[AW_THREADS];
  const int chunks = T.blk_end[T.count - 1];
  double s = 0.0;
  const AwFind find(T);
  for (int c = (int)blockIdx.x; c < chunks; c += (int)gridDim.x) {
    const int ti = find(c);
    const long long left = T.n[ti] - (long long)(c - (ti ? T.blk_end[ti - 1] : 0)) * AW_SQ_CHUNK;
    const PT *__restrict__ g = (const PT *)T.g[ti] + (T.n[ti] - left);
    if (left >= AW_SQ_CHUNK) {
      unsigned w[U][4];
#pragma unroll
      for (int u = 0; u < U; ++u) __builtin_memcpy(w[u], g + (u * AW_THREADS + (int)threadIdx.x) * E, 16);
      double a[2] = {0.0, 0.0};
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (BF16) {
            const double x = (double)__uint_as_float(w[u][i] << 16), y = (double)__uint_as_float(w[u][i] & 0xFFFF0000u);
            a[0] = fma(x, x, a[0]);
            a[1] = fma(y, y, a[1]);
          } else {
            const double x = (double)__uint_as_float(w[u][i]);
            a[i & 1] = fma(x, x, a[i & 1]);
          }
        }
      s += a[0] + a[1];
    } else {
      for (int e = (int)threadIdx.x; e < (int)left; e += AW_THREADS) {
        float x;
        if constexpr (BF16) x = __uint_as_float((unsigned)g[e] << 16); else x = g[e];
        s = fma((double)x, (double)x, s);
      }
    }
  }
  red[threadIdx.x] = s;
  __syncthreads();
  for (int off = AW_THREADS / 2; off > 0; off >>= 1) {
    if ((int)threadIdx.x < off) red[threadIdx.x] += red[threadIdx.x + off];
    __syncthreads();
  }
  if (threadIdx.x == 0) partial[blockIdx.x] = red[0];
}

// the norm of all, and the factor of torch.nn.utils.clip_grad_norm_: max_norm / (norm + 1e-6), at most 1; a norm that is no number stays none
__global__ void __launch_bounds__(AW_THREADS)
grad_norm_kernel(int n, const double *__restrict__ partial, float max_norm, float *__restrict__ out) {
  __shared__ double red[AW_THREADS];
  double s = 0.0;
#pragma unroll 4
  for (int i = threadIdx.x; i < n; i += AW_THREADS) s += partial[i];
  red[threadIdx.x] = s;
  __syncthreads();
  for (int off = AW_THREADS / 2; off > 0; off >>= 1) {
    if ((int)threadIdx.x < off) red[threadIdx.x] += red[threadIdx.x + off];
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    const float norm = (float)sqrt(red[0]), c = (1.f / (norm + 1e-6f)) * max_norm;      // (a quotient by a tensor is its reciprocal's product there)
    out[0] = norm;
    out[1] = c > 1.f ? 1.f : c;
  }
}

// ---- 8-bit moments <-> values, flat (bound by memory: 268 M pairs to bf16 276 us = 5.8 TB/s) ---------------------------------------------------------------------------------
__global__ void __launch_bounds__(AW_THREADS)
adamw_pack_kernel(long long blocks, const float *__restrict__ m, const float *__restrict__ v, unsigned char *__restrict__ mc,
                  unsigned char *__restrict__ vc, unsigned char *__restrict__ me, unsigned char *__restrict__ ve) {
  const int lane = (int)threadIdx.x & 63;
  for (long long b = (long long)blockIdx.x * 4 + ((int)threadIdx.x >> 6); b < blocks; b += (long long)gridDim.x * 4) {
    const long long e = b * AW_BLOCK + lane * 4;
    const Four<float> x = aw_load(m + e, 4), y = aw_load(v + e, 4);
    unsigned fm = 0u, fv = 0u;
#pragma unroll
    for (int i = 0; i < 4; ++i) { fm = max(fm, aw_field(aw_get(x, i))); fv = max(fv, aw_field(aw_get(y, i))); }
    fm = rs_wave_max_u32(fm);
    fv = rs_wave_max_u32(fv);
    Four<unsigned char> a{{0u}}, c{{0u}};
#pragma unroll
    for (int i = 0; i < 4; ++i) {         // to nearest: a dither of one half
      a.w[0] |= aw_encode_m(aw_get(x, i), (int)fm, 0x8000u) << (8 * i);
      c.w[0] |= aw_encode_v(aw_get(y, i), (int)fv, 0x8000u) << (8 * i);
    }
    aw_store(mc + e, a, 4);
    aw_store(vc + e, c, 4);
    if (lane == 0) { me[b] = (unsigned char)fm; ve[b] = (unsigned char)fv; }
  }
}

__device__ __forceinline__ void aw_out(float *p, const float *x) { __builtin_memcpy(p, x, 16); }
__device__ __forceinline__ void aw_out(__bf16 *p, const float *x) {      // to nearest even: exact for a code's value
  __bf16 r[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = (__bf16)x[i];
  __builtin_memcpy(p, r, sizeof(r));
}
template <typename O>
__global__ void __launch_bounds__(AW_THREADS)
adamw_unpack_kernel(long long blocks, const unsigned char *__restrict__ mc, const unsigned char *__restrict__ vc,
                    const unsigned char *__restrict__ me, const unsigned char *__restrict__ ve, O *__restrict__ m, O *__restrict__ v) {
  const int lane = (int)threadIdx.x & 63;
  for (long long b = (long long)blockIdx.x * 4 + ((int)threadIdx.x >> 6); b < blocks; b += (long long)gridDim.x * 4) {
    const long long e = b * AW_BLOCK + lane * 4;
    const Four<unsigned char> a = aw_load(mc + e, 4), c = aw_load(vc + e, 4);
    const int em = me[b], ev = ve[b];
    float x[4], y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) { x[i] = aw_decode_m(aw_get(a, i), em); y[i] = aw_decode_v(aw_get(c, i), ev); }
    aw_out(m + e, x);
    aw_out(v + e, y);
  }
}

// masters of bf16 parameters into a flat fp32 buffer, zeros up to the next tensor
__global__ void __launch_bounds__(AW_THREADS)
adamw_masters_kernel(AwTable T, const short *__restrict__ low, float *__restrict__ out) {
  const int c = (int)blockIdx.x, ti = AwFind(T)(c);
  const long long n = T.n[ti], at = T.at[ti];
  const long long base = (long long)(c - (ti ? T.blk_end[ti - 1] : 0)) * AW_CHUNK;
  const unsigned short *__restrict__ p = (const unsigned short *)T.p[ti];
#pragma unroll
  for (int u = 0; u < AW_CHUNK / (4 * AW_THREADS); ++u) {
    const long long e = base + (u * AW_THREADS + (int)threadIdx.x) * 4, left = n - e;
    if (e >= (n + AW_BLOCK - 1) / AW_BLOCK * AW_BLOCK) continue;
    const Four<unsigned short> r = aw_load(p + e, left);
    const Four<short> l = aw_load(low + at + e, 4);
    Four<float> x;
#pragma unroll
    for (int i = 0; i < 4; ++i) x.w[i] = i < left ? __float_as_uint(aw_master(aw_high(r, i), aw_get(l, i))) : 0u;
    aw_store(out + at + e, x, 4);
  }
}

constexpr long long AW_CHUNKS = (1LL << 24) - 1;      // workgroups of 256 threads: a launch holds fewer than 2^32 threads
constexpr int AW_GRID = 1 << 22;

// calls f(table, chunks) for runs of at most AW_MAX tensors and AW_CHUNKS chunks
template <typename F>
int aw_tables(const rs_adamw_list *l, const char *name, int chunk, F f) {
  RS_REQUIRE(l && l->count >= 0 && (l->count == 0 || (l->p && l->g && l->n && l->at && l->slot)), "%s: null pointer", name);
  for (int k = 0; k < l->count; ++k) {
    RS_REQUIRE(l->p[k] && l->g[k] && l->n[k] > 0 && l->at[k] >= 0 && l->at[k] % AW_BLOCK == 0 && l->slot[k] >= 0,
               "%s: tensor %d: null pointer, empty, or not at a multiple of %d elements", name, k, AW_BLOCK);
    RS_REQUIRE((l->n[k] + chunk - 1) / chunk <= AW_CHUNKS, "%s: tensor %d has %lld elements, at most %lld are served", name, k, l->n[k], AW_CHUNKS * chunk);
  }
  for (int k = 0; k < l->count;) {
    AwTable T;
    long long chunks = 0;
    int i = 0;
    for (; i < AW_MAX && k < l->count; ++i, ++k) {
      const long long more = (l->n[k] + chunk - 1) / chunk;
      if (chunks + more > AW_CHUNKS) break;
      T.p[i] = l->p[k]; T.g[i] = l->g[k]; T.n[i] = l->n[k]; T.at[i] = l->at[k]; T.slot[i] = l->slot[k];
      T.blk_end[i] = (int)(chunks += more);
    }
    T.count = i;
    const int rc = f(T, (int)chunks);
    if (rc != RS_OK) return rc;
  }
  return RS_OK;
}

}  // namespace

extern "C" int rs_adamw_step(const rs_adamw_list *l, const rs_adamw_args *a, void *stream) {
  RS_REQUIRE(a && a->exp_avg && a->exp_avg_sq && a->step && a->done, "rs_adamw_step: null pointer");
  RS_REQUIRE(a->bits == 32 || (a->bits == 8 && a->exp_avg_exponent && a->exp_avg_sq_exponent), "rs_adamw_step: bits=%d (32, or 8 with exponents)", a->bits);
  RS_REQUIRE(!a->bf16 || a->low, "rs_adamw_step: bf16 parameters need the masters' low halves");
  AwArgs A;
  A.m = a->exp_avg; A.v = a->exp_avg_sq; A.me = a->exp_avg_exponent; A.ve = a->exp_avg_sq_exponent; A.low = a->low;
  A.step = a->step; A.done = a->done; A.hyper_dev = a->hyper_dev;
  for (int i = 0; i < 7; ++i) A.hyper[i] = a->hyper[i];
  A.clip = a->clip; A.seed = a->seed;
  return aw_tables(l, "rs_adamw_step", AW_CHUNK, [&](const AwTable &T, int chunks) {
    const dim3 grid(chunks), block(AW_THREADS);
    hipStream_t st = (hipStream_t)stream;
    if (a->bf16) {
      if (a->bits == 8) hipLaunchKernelGGL((adamw_kernel<true, 8>), grid, block, 0, st, T, A);
      else hipLaunchKernelGGL((adamw_kernel<true, 32>), grid, block, 0, st, T, A);
    } else {
      if (a->bits == 8) hipLaunchKernelGGL((adamw_kernel<false, 8>), grid, block, 0, st, T, A);
      else hipLaunchKernelGGL((adamw_kernel<false, 32>), grid, block, 0, st, T, A);
    }
    RS_CHECK_LAUNCH("rs_adamw_step");
    return RS_OK;
  });
}

extern "C" int rs_grad_square_sums(const rs_adamw_list *l, int bf16, double *partial, int room, int *used, void *stream) {
  RS_REQUIRE(partial && used && room >= 0, "rs_grad_square_sums: null pointer");
  *used = 0;
  return aw_tables(l, "rs_grad_square_sums", AW_SQ_CHUNK, [&](const AwTable &T, int chunks) {
    const int blocks = chunks < RS_GRAD_SQUARE_SUMS ? chunks : RS_GRAD_SQUARE_SUMS;
    RS_REQUIRE(*used + blocks <= room, "rs_grad_square_sums: room for %d sums, more are needed", room);
    if (bf16) hipLaunchKernelGGL((grad_sq_kernel<true>), dim3(blocks), dim3(AW_THREADS), 0, (hipStream_t)stream, T, partial + *used);
    else hipLaunchKernelGGL((grad_sq_kernel<false>), dim3(blocks), dim3(AW_THREADS), 0, (hipStream_t)stream, T, partial + *used);
    RS_CHECK_LAUNCH("rs_grad_square_sums");
    *used += blocks;
    return RS_OK;
  });
}

extern "C" int rs_grad_norm(int n, const double *partial, float max_norm, float *out, void *stream) {
  RS_REQUIRE(n > 0 && partial && out, "rs_grad_norm: null pointer or no sums");
  RS_REQUIRE(max_norm > 0.f, "rs_grad_norm: max_norm=%g", max_norm);
  hipLaunchKernelGGL(grad_norm_kernel, dim3(1), dim3(AW_THREADS), 0, (hipStream_t)stream, n, partial, max_norm, out);
  RS_CHECK_LAUNCH("rs_grad_norm");
  return RS_OK;
}

extern "C" int rs_adamw_masters(const rs_adamw_list *l, const short *low, float *out, void *stream) {
  RS_REQUIRE(low && out, "rs_adamw_masters: null pointer");
  return aw_tables(l, "rs_adamw_masters", AW_CHUNK, [&](const AwTable &T, int chunks) {
    hipLaunchKernelGGL(adamw_masters_kernel, dim3(chunks), dim3(AW_THREADS), 0, (hipStream_t)stream, T, low, out);
    RS_CHECK_LAUNCH("rs_adamw_masters");
    return RS_OK;
  });
}

extern "C" int rs_adamw_pack(long long n, const float *m, const float *v, unsigned char *mc, unsigned char *vc, unsigned char *me,
                             unsigned char *ve, void *stream) {
  RS_REQUIRE(n >= 0 && n % AW_BLOCK == 0, "rs_adamw_pack: n=%lld is no multiple of %d", n, AW_BLOCK);
  if (n == 0) return RS_OK;
  RS_REQUIRE(m && v && mc && vc && me && ve, "rs_adamw_pack: null pointer");
  const long long blocks = n / AW_BLOCK, wgs = (blocks + 3) / 4;
  hipLaunchKernelGGL(adamw_pack_kernel, dim3((int)(wgs < AW_GRID ? wgs : AW_GRID)), dim3(AW_THREADS), 0, (hipStream_t)stream, blocks, m, v, mc, vc, me, ve);
  RS_CHECK_LAUNCH("rs_adamw_pack");
  return RS_OK;
}

extern "C" int rs_adamw_unpack(long long n, const unsigned char *mc, const unsigned char *vc, const unsigned char *me, const unsigned char *ve,
                               int out_bf16, void *m, void *v, void *stream) {
  RS_REQUIRE(n >= 0 && n % AW_BLOCK == 0, "rs_adamw_unpack: n=%lld is no multiple of %d", n, AW_BLOCK);
  if (n == 0) return RS_OK;
  RS_REQUIRE(m && v && mc && vc && me && ve, "rs_adamw_unpack: null pointer");
  const long long blocks = n / AW_BLOCK, wgs = (blocks + 3) / 4;
  const dim3 grid((int)(wgs < AW_GRID ? wgs : AW_GRID));
  if (out_bf16) hipLaunchKernelGGL((adamw_unpack_kernel<__bf16>), grid, dim3(AW_THREADS), 0, (hipStream_t)stream, blocks, mc, vc, me, ve, (__bf16 *)m, (__bf16 *)v);
  else hipLaunchKernelGGL((adamw_unpack_kernel<float>), grid, dim3(AW_THREADS), 0, (hipStream_t)stream, blocks, mc, vc, me, ve, (float *)m, (float *)v);
  RS_CHECK_LAUNCH("rs_adamw_unpack");
  return RS_OK;
}
