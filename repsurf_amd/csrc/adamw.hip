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
#include "rs_common.h"
#include <math.h>

namespace {

constexpr int AW_THREADS = 256;
constexpr int AW_BLOCK = 256;             // elements that share an exponent
constexpr int AW_UNROLL = 2;              // blocks a wave has in flight
constexpr int AW_CHUNK = AW_BLOCK * (AW_THREADS / RS_WAVE) * AW_UNROLL;
constexpr int AW_MAX = 80;                // tensors per launch: the table rides in the kernel arguments
constexpr int AW_FIELD_M = 14, AW_FIELD_V = 30;

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
  const double *partial;                  // sums of squares of the gradients, or null
  int npartial;
  float max_norm;
  float *norm;
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

__device__ __forceinline__ float aw_master(unsigned short p, short low) {
  const unsigned a = p & 0x7FFFu;
  // +-0 and infinity never carry a remainder of this sign: such a parameter was written from outside, and its word would wrap to a NaN
  const int l = (a == 0u && low < 0) || (a >= 0x7F80u && low > 0) ? 0 : (int)low;
  return __uint_as_float(((unsigned)p << 16) + (unsigned)l);
}
__device__ __forceinline__ void aw_split(float x, unsigned short &p, short &low) {
  const unsigned b = __float_as_uint(x);
  const bool nan = (b & 0x7FFFFFFFu) > 0x7F800000u;
  p = nan ? (unsigned short)0x7FC0u : (unsigned short)((b + 0x8000u) >> 16);
  low = nan ? (short)0 : (short)(b - ((unsigned)p << 16));
}

template <bool BF16> struct AwType { typedef float T; };
template <> struct AwType<true> { typedef unsigned short T; };

// four consecutive elements; `left` of them exist.  The address is aligned to the element only: global loads of this device need no more.
template <typename T> struct Four { T x[4]; };
template <typename T>
__device__ __forceinline__ Four<T> aw_load(const T *p, long long left) {
  Four<T> r;
  if (left >= 4) { __builtin_memcpy(&r, p, sizeof(r)); return r; }
#pragma unroll
  for (int i = 0; i < 4; ++i) r.x[i] = i < left ? p[i] : T(0);
  return r;
}
template <typename T>
__device__ __forceinline__ void aw_store(T *p, const Four<T> &r, long long left) {
  if (left >= 4) { __builtin_memcpy(p, &r, sizeof(r)); return; }
#pragma unroll
  for (int i = 0; i < 4; ++i) if (i < left) p[i] = r.x[i];
}

// max(1, ...) of torch.nn.utils.clip_grad_norm_: max_norm / (norm + 1e-6), at most 1; a norm that is not a number stays one
__device__ __forceinline__ float aw_clip(const double *partial, int n, float max_norm, float *norm_out, double *red) {
  double s = 0.0;
  for (int i = threadIdx.x; i < n; i += AW_THREADS) s += partial[i];
  red[threadIdx.x] = s;
  __syncthreads();
  for (int off = AW_THREADS / 2; off > 0; off >>= 1) {
    if ((int)threadIdx.x < off) red[threadIdx.x] += red[threadIdx.x + off];
    __syncthreads();
  }
  const float norm = (float)sqrt(red[0]);
  if (blockIdx.x == 0 && threadIdx.x == 0) *norm_out = norm;
  const float c = max_norm / (norm + 1e-6f);
  return c > 1.f ? 1.f : c;
}

template <bool BF16, int BITS>
__global__ void __launch_bounds__(AW_THREADS)
adamw_kernel(AwTable T, AwArgs A) {
  typedef typename AwType<BF16>::T PT;
  __shared__ double red[AW_THREADS];
  double lr = A.hyper[0], beta1 = A.hyper[1], beta2 = A.hyper[2], eps64 = A.hyper[3], wd = A.hyper[4], lnb1 = A.hyper[5], lnb2 = A.hyper[6];
  if (A.hyper_dev) {
    lr = A.hyper_dev[0]; beta1 = A.hyper_dev[1]; beta2 = A.hyper_dev[2]; eps64 = A.hyper_dev[3]; wd = A.hyper_dev[4];
    lnb1 = A.hyper_dev[5]; lnb2 = A.hyper_dev[6];
  }
  const float eps = (float)eps64, decay = (float)(1.0 - lr * wd);
  const float omb1 = (float)(1.0 - beta1), b2 = (float)beta2, omb2 = (float)(1.0 - beta2);
  const float clip = A.partial ? aw_clip(A.partial, A.npartial, A.max_norm, A.norm, red) : 1.f;
  const int wave = rs_uniform((int)threadIdx.x >> 6), lane = (int)threadIdx.x & 63;
  const int chunks = T.blk_end[T.count - 1];

  int ti = 0, seen = -1;
  float step_size = 0.f, inv_bc2 = 1.f;
  unsigned key = 0u;
  for (int c = (int)blockIdx.x; c < chunks; c += (int)gridDim.x) {
    // the tensor of this chunk: the first whose running count exceeds c, by bisection above the last one (chunks only grow)
    int lo = ti, hi = T.count - 1;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (c >= T.blk_end[mid]) lo = mid + 1; else hi = mid;
    }
    ti = lo;
    if (ti != seen) {
      seen = ti;
      const int t = A.step[T.slot[ti]] + 1;
      // 1 - beta^t as -expm1(t ln beta): fp32 loses nothing where beta^t is near 1
      step_size = (float)(lr / (double)-expm1f((float)(lnb1 * t)));
      inv_bc2 = 1.f / sqrtf(-expm1f((float)(lnb2 * t)));
      key = aw_mix(A.seed + (unsigned)t * AW_PHI);
    }
    const long long n = T.n[ti], at = T.at[ti];
    const long long base = (long long)(c - (ti ? T.blk_end[ti - 1] : 0)) * AW_CHUNK + wave * (AW_BLOCK * AW_UNROLL);
    PT *__restrict__ p = (PT *)T.p[ti];
    const PT *__restrict__ g = (const PT *)T.g[ti];
    Four<PT> pv[AW_UNROLL], gv[AW_UNROLL];
    Four<short> lv[AW_UNROLL];
    Four<float> mv[AW_UNROLL], vv[AW_UNROLL];
    Four<unsigned char> mc[AW_UNROLL], vc[AW_UNROLL];
    int em[AW_UNROLL], ev[AW_UNROLL];
#pragma unroll
    for (int u = 0; u < AW_UNROLL; ++u) {
      const long long b = base + u * AW_BLOCK, e = b + lane * 4, left = n - e;
      if (b >= n) continue;
      pv[u] = aw_load(p + e, left);
      gv[u] = aw_load(g + e, left);
      if constexpr (BF16) lv[u] = aw_load((const short *)A.low + at + e, 4);
      if constexpr (BITS == 32) {         // (the flat buffers have the block's tail, as zeros)
        mv[u] = aw_load((const float *)A.m + at + e, 4);
        vv[u] = aw_load((const float *)A.v + at + e, 4);
      } else {
        mc[u] = aw_load((const unsigned char *)A.m + at + e, 4);
        vc[u] = aw_load((const unsigned char *)A.v + at + e, 4);
        em[u] = A.me[(at + b) >> 8];
        ev[u] = A.ve[(at + b) >> 8];
      }
    }
#pragma unroll
    for (int u = 0; u < AW_UNROLL; ++u) {
      const long long b = base + u * AW_BLOCK, e = b + lane * 4, left = n - e;
      if (b >= n) continue;
      unsigned fm = 0u, fv = 0u;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float x, gi;
        if constexpr (BF16) {
          x = aw_master(pv[u].x[i], lv[u].x[i]);
          gi = __uint_as_float((unsigned)gv[u].x[i] << 16);
        } else { x = pv[u].x[i]; gi = gv[u].x[i]; }
        if constexpr (BITS == 8) { mv[u].x[i] = aw_decode_m(mc[u].x[i], em[u]); vv[u].x[i] = aw_decode_v(vc[u].x[i], ev[u]); }
        gi *= clip;
        const float m = rs_fma(gi - mv[u].x[i], omb1, mv[u].x[i]);
        const float v = rs_fma(omb2 * gi, gi, vv[u].x[i] * b2);
        x = rs_fma(-step_size, m / rs_fma(sqrtf(v), inv_bc2, eps), x * decay);
        const bool in = i < left;
        mv[u].x[i] = in ? m : 0.f;
        vv[u].x[i] = in ? v : 0.f;
        if constexpr (BF16) aw_split(x, pv[u].x[i], lv[u].x[i]); else pv[u].x[i] = x;
        if constexpr (BF16) { if (!in) lv[u].x[i] = 0; }
        if constexpr (BITS == 8) { fm = max(fm, aw_field(mv[u].x[i])); fv = max(fv, aw_field(vv[u].x[i])); }
      }
      aw_store(p + e, pv[u], left);
      if constexpr (BF16) aw_store(A.low + at + e, lv[u], 4);
      if constexpr (BITS == 32) {
        aw_store((float *)A.m + at + e, mv[u], 4);
        aw_store((float *)A.v + at + e, vv[u], 4);
      } else {
        fm = rs_wave_max_u32(fm);
        fv = rs_wave_max_u32(fv);
        const unsigned k = aw_mix(key + (unsigned)((at + b) >> 8)) + (unsigned)(lane * 4) * AW_PHI;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const unsigned r = aw_mix(k + i * AW_PHI);
          mc[u].x[i] = (unsigned char)aw_encode_m(mv[u].x[i], (int)fm, r >> 16);
          vc[u].x[i] = (unsigned char)aw_encode_v(vv[u].x[i], (int)fv, r & 0xFFFFu);
        }
        aw_store((unsigned char *)A.m + at + e, mc[u], 4);
        aw_store((unsigned char *)A.v + at + e, vc[u], 4);
        if (lane == 0) { A.me[(at + b) >> 8] = (unsigned char)fm; A.ve[(at + b) >> 8] = (unsigned char)fv; }
      }
    }
  }
  // The last workgroup advances the counters of this launch's tensors: every workgroup has read them by then (its reads feed its
  // stores, in front of the barrier and the count).  No fence: nothing written here is read before the next launch.
  __shared__ int last;
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(A.done, 1) == (int)gridDim.x - 1;
  __syncthreads();
  if (last) {
    if ((int)threadIdx.x < T.count) A.step[T.slot[threadIdx.x]] += 1;
    if (threadIdx.x == 0) *A.done = 0;
  }
}

// ---- the gradients' common norm -------------------------------------------------------------------------------------
// partial[b] = sum of the squares of workgroup b's chunks.  A lane's 8 squares of a chunk are added in fp32, everything above in
// fp64, in an order that the sizes fix.
template <bool BF16>
__global__ void __launch_bounds__(AW_THREADS)
grad_sq_kernel(AwTable T, double *__restrict__ partial) {
  typedef typename AwType<BF16>::T PT;
  __shared__ double red[AW_THREADS];
  const int chunks = T.blk_end[T.count - 1];
  double s = 0.0;
  int ti = 0;
  for (int c = (int)blockIdx.x; c < chunks; c += (int)gridDim.x) {
    int lo = ti, hi = T.count - 1;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (c >= T.blk_end[mid]) lo = mid + 1; else hi = mid;
    }
    ti = lo;
    const long long n = T.n[ti];
    const long long base = (long long)(c - (ti ? T.blk_end[ti - 1] : 0)) * AW_CHUNK;
    const PT *__restrict__ g = (const PT *)T.g[ti];
    float a = 0.f;
#pragma unroll
    for (int u = 0; u < AW_CHUNK / (4 * AW_THREADS); ++u) {
      const long long e = base + (u * AW_THREADS + (int)threadIdx.x) * 4;
      const Four<PT> r = aw_load(g + e, n - e);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float x;
        if constexpr (BF16) x = __uint_as_float((unsigned)r.x[i] << 16); else x = r.x[i];
        a = rs_fma(x, x, a);
      }
    }
    s += (double)a;
  }
  red[threadIdx.x] = s;
  __syncthreads();
  for (int off = AW_THREADS / 2; off > 0; off >>= 1) {
    if ((int)threadIdx.x < off) red[threadIdx.x] += red[threadIdx.x + off];
    __syncthreads();
  }
  if (threadIdx.x == 0) partial[blockIdx.x] = red[0];
}

// ---- 8-bit moments <-> values, flat ---------------------------------------------------------------------------------
__global__ void __launch_bounds__(AW_THREADS)
adamw_pack_kernel(long long blocks, const float *__restrict__ m, const float *__restrict__ v, unsigned char *__restrict__ mc,
                  unsigned char *__restrict__ vc, unsigned char *__restrict__ me, unsigned char *__restrict__ ve) {
  const int lane = (int)threadIdx.x & 63;
  for (long long b = (long long)blockIdx.x * 4 + ((int)threadIdx.x >> 6); b < blocks; b += (long long)gridDim.x * 4) {
    const long long e = b * AW_BLOCK + lane * 4;
    const Four<float> x = aw_load(m + e, 4), y = aw_load(v + e, 4);
    unsigned fm = 0u, fv = 0u;
#pragma unroll
    for (int i = 0; i < 4; ++i) { fm = max(fm, aw_field(x.x[i])); fv = max(fv, aw_field(y.x[i])); }
    fm = rs_wave_max_u32(fm);
    fv = rs_wave_max_u32(fv);
    Four<unsigned char> a, c;
#pragma unroll
    for (int i = 0; i < 4; ++i) {         // to nearest: a dither of one half
      a.x[i] = (unsigned char)aw_encode_m(x.x[i], (int)fm, 0x8000u);
      c.x[i] = (unsigned char)aw_encode_v(y.x[i], (int)fv, 0x8000u);
    }
    aw_store(mc + e, a, 4);
    aw_store(vc + e, c, 4);
    if (lane == 0) { me[b] = (unsigned char)fm; ve[b] = (unsigned char)fv; }
  }
}

__device__ __forceinline__ void aw_out(float *p, const float *x) { __builtin_memcpy(p, x, 16); }
__device__ __forceinline__ void aw_out(unsigned short *p, const float *x) {      // to bf16, to nearest even (exact for a code's value)
  Four<unsigned short> r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const unsigned b = __float_as_uint(x[i]);
    r.x[i] = (b & 0x7FFFFFFFu) > 0x7F800000u ? 0x7FC0u : (unsigned short)((b + 0x7FFFu + ((b >> 16) & 1u)) >> 16);
  }
  __builtin_memcpy(p, &r, sizeof(r));
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
    for (int i = 0; i < 4; ++i) { x[i] = aw_decode_m(a.x[i], em); y[i] = aw_decode_v(c.x[i], ev); }
    aw_out(m + e, x);
    aw_out(v + e, y);
  }
}

// masters of bf16 parameters into a flat fp32 buffer (its tails are left as they are)
__global__ void __launch_bounds__(AW_THREADS)
adamw_masters_kernel(AwTable T, const short *__restrict__ low, float *__restrict__ out) {
  const int chunks = T.blk_end[T.count - 1];
  int ti = 0;
  for (int c = (int)blockIdx.x; c < chunks; c += (int)gridDim.x) {
    int lo = ti, hi = T.count - 1;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (c >= T.blk_end[mid]) lo = mid + 1; else hi = mid;
    }
    ti = lo;
    const long long n = T.n[ti], at = T.at[ti];
    const long long base = (long long)(c - (ti ? T.blk_end[ti - 1] : 0)) * AW_CHUNK;
    const unsigned short *__restrict__ p = (const unsigned short *)T.p[ti];
#pragma unroll
    for (int u = 0; u < AW_CHUNK / (4 * AW_THREADS); ++u) {
      const long long e = base + (u * AW_THREADS + (int)threadIdx.x) * 4, left = n - e;
      if (left <= 0) continue;
      const Four<unsigned short> r = aw_load(p + e, left);
      const Four<short> l = aw_load(low + at + e, 4);
      Four<float> x;
#pragma unroll
      for (int i = 0; i < 4; ++i) x.x[i] = aw_master(r.x[i], l.x[i]);
      aw_store(out + at + e, x, left);
    }
  }
}

constexpr int AW_GRID = 2048;             // 8 workgroups on each of 256 CUs

// calls f(table, chunks) for runs of at most AW_MAX tensors
template <typename F>
int aw_tables(const rs_adamw_list *l, const char *name, F f) {
  RS_REQUIRE(l && l->count >= 0 && (l->count == 0 || (l->p && l->g && l->n && l->at && l->slot)), "%s: null pointer", name);
  for (int first = 0; first < l->count; first += AW_MAX) {
    AwTable T;
    T.count = l->count - first < AW_MAX ? l->count - first : AW_MAX;
    long long chunks = 0;
    for (int i = 0; i < T.count; ++i) {
      const int k = first + i;
      RS_REQUIRE(l->p[k] && l->g[k] && l->n[k] > 0 && l->at[k] >= 0 && l->at[k] % AW_BLOCK == 0 && l->slot[k] >= 0,
                 "%s: tensor %d: null pointer, empty, or not at a multiple of %d elements", name, k, AW_BLOCK);
      T.p[i] = l->p[k]; T.g[i] = l->g[k]; T.n[i] = l->n[k]; T.at[i] = l->at[k]; T.slot[i] = l->slot[k];
      chunks += (l->n[k] + AW_CHUNK - 1) / AW_CHUNK;
      RS_REQUIRE(chunks < (1LL << 31), "%s: too many elements in one launch", name);
      T.blk_end[i] = (int)chunks;
    }
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
  RS_REQUIRE(!a->partial || (a->npartial > 0 && a->norm && a->max_norm > 0.f), "rs_adamw_step: partial sums without their number, a norm or a bound");
  AwArgs A;
  A.m = a->exp_avg; A.v = a->exp_avg_sq; A.me = a->exp_avg_exponent; A.ve = a->exp_avg_sq_exponent; A.low = a->low;
  A.step = a->step; A.done = a->done; A.hyper_dev = a->hyper_dev;
  for (int i = 0; i < 7; ++i) A.hyper[i] = a->hyper[i];
  A.partial = a->partial; A.npartial = a->npartial; A.max_norm = a->max_norm; A.norm = a->norm; A.seed = a->seed;
  return aw_tables(l, "rs_adamw_step", [&](const AwTable &T, int chunks) {
    const dim3 grid(chunks < AW_GRID ? chunks : AW_GRID), block(AW_THREADS);
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
  return aw_tables(l, "rs_grad_square_sums", [&](const AwTable &T, int chunks) {
    const int blocks = chunks < RS_GRAD_SQUARE_SUMS ? chunks : RS_GRAD_SQUARE_SUMS;
    RS_REQUIRE(*used + blocks <= room, "rs_grad_square_sums: room for %d sums, more are needed", room);
    if (bf16) hipLaunchKernelGGL((grad_sq_kernel<true>), dim3(blocks), dim3(AW_THREADS), 0, (hipStream_t)stream, T, partial + *used);
    else hipLaunchKernelGGL((grad_sq_kernel<false>), dim3(blocks), dim3(AW_THREADS), 0, (hipStream_t)stream, T, partial + *used);
    RS_CHECK_LAUNCH("rs_grad_square_sums");
    *used += blocks;
    return RS_OK;
  });
}

extern "C" int rs_adamw_masters(const rs_adamw_list *l, const short *low, float *out, void *stream) {
  RS_REQUIRE(low && out, "rs_adamw_masters: null pointer");
  return aw_tables(l, "rs_adamw_masters", [&](const AwTable &T, int chunks) {
    hipLaunchKernelGGL(adamw_masters_kernel, dim3(chunks < AW_GRID ? chunks : AW_GRID), dim3(AW_THREADS), 0, (hipStream_t)stream, T, low, out);
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
  if (out_bf16) hipLaunchKernelGGL((adamw_unpack_kernel<unsigned short>), grid, dim3(AW_THREADS), 0, (hipStream_t)stream, blocks, mc, vc, me, ve, (unsigned short *)m, (unsigned short *)v);
  else hipLaunchKernelGGL((adamw_unpack_kernel<float>), grid, dim3(AW_THREADS), 0, (hipStream_t)stream, blocks, mc, vc, me, ve, (float *)m, (float *)v);
  RS_CHECK_LAUNCH("rs_adamw_unpack");
  return RS_OK;
}
