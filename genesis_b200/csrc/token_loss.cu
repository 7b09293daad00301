// Losses on a language model's logits that need only the log-probability of one token per row: log-probabilities
// themselves, the clipped policy objective with its KL term, the loss of paired log ratios.
//
//   row:         m near max z,  s = sum exp((z - m) / T),  lp = (z[t] - m) / T - log s
//   policy:      r = exp(lp - old),  l = max(-A r, -A clamp(r, 1 - c, 1 + c')) + k (exp(ref - lp) - (ref - lp) - 1)
//                dl/dlp = (-A r where the unclipped term is the larger, else 0) + k (1 - exp(ref - lp))
//   preference:  S = sum lp over an answer,  h = beta ((S_c - ref_c) - (S_r - ref_r)),
//                l = -(1 - e) log sigmoid(h) - e log sigmoid(-h),  dl/dh = e - sigmoid(-h)
//   logits:      dz[j] = g / T ([j = t] - exp((z[j] - m) / T) / s)
//
// Three kinds of kernels: one reads every row that counts once and keeps m and s (16-bit logits: log2 s) of it; one block joins the rows
// into the loss, in a fixed order and in 64 bits (the sum of an answer's log-probabilities runs into the thousands, its
// difference to the reference's is of order one; there the log-probabilities too are kept in 64 bits); one writes the
// gradient.  Nothing of the size of the logits is kept between the two passes but the logits.  A row that does not count (its
// token is the ignored index) is not read, so whatever it holds reaches nothing, and its gradient is zero.
#include <cooperative_groups.h>
#include "sm100_ptx.cuh"
#include "common.cuh"

namespace gb {
namespace tl {

namespace cg = cooperative_groups;

constexpr int SITE_TOKEN = 7;                      // where a bad index was found (native.py: _raise_status)

// Row r of the logits starts at z + (r / inner) * s_outer + (r % inner) * s_inner elements: a [B, T, V] slice is read in place.
struct RowMap {
  long long inner, s_outer, s_inner;
  __device__ __forceinline__ long long at(long long r) const { return (r / inner) * s_outer + (r % inner) * s_inner; }
};

struct Policy {
  const float* old;            // [rows]; null: log-probabilities alone are wanted
  const float* adv;            // one per `adv_div` rows
  const float* ref;            // [rows] or null
  float* loss;                 // [rows]
  float* coef;                 // [rows] dl/dlp
  long long adv_div;
  float lo, hi, kl;            // 1 - c, 1 + c', k
  double* wide;                // [rows] log-probabilities as they are before they are rounded, in place of lp; or null
};

struct MaxSum { float m, s; };

// log2(e) / T as the sum of two floats: rounded to one, it would shift every log-probability the same way, by 1.3e-8 of
// (z - m) / T, and the sum of an answer's log-probabilities by their number times that.  The high part is rounded down, so
// that the low one is positive and -inf times either is -inf.
struct Scale {
  float hi, lo, inv, slack;    // inv: 1 / T; slack: what a factor of 2 is among the logits
  explicit Scale(double temperature) {
    const double c = 1.4426950408889634 / temperature;
    hi = (float)c;
    if ((double)hi >= c) hi = nextafterf(hi, 0.f);
    lo = (float)(c - (double)hi);
    inv = (float)(1.0 / temperature);
    slack = (float)(1.0 / c);
  }
  __device__ __forceinline__ float operator()(float d) const { return fmaf(d, hi, d * lo); }
};

// A part's sum relative to the maximum m of the whole; a part of -inf alone (or of nothing) is (-inf, 0).  expf here: the
// hardware's exponential is 5e-8 of its result too small on average, and a sum passes through several of these.
__device__ __forceinline__ float rescale(MaxSum a, float m, float temperature) {
  return a.m == m || m == -INFINITY ? a.s : a.s * expf((a.m - m) / temperature);       // (a NaN sum stays one)
}

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

template <typename T> struct Two;
template <> struct Two<__nv_bfloat16> {
  typedef __nv_bfloat162 P;
  static __device__ __forceinline__ float2 f(P a) { return __bfloat1622float2(a); }
  static __device__ __forceinline__ uint32_t pack(float a, float b) { return pack2c<true>(a, b); }
};
template <> struct Two<__half> {
  typedef __half2 P;
  static __device__ __forceinline__ float2 f(P a) { return __half22float2(a); }
  static __device__ __forceinline__ uint32_t pack(float a, float b) { return pack2c<false>(a, b); }
};

// 16 bytes of a row as floats, in pairs
template <typename T>
__device__ __forceinline__ void unpack(const uint4& v, float2 (&f)[8 / sizeof(T)]) {
  if constexpr (sizeof(T) == 4) {
    f[0] = make_float2(__uint_as_float(v.x), __uint_as_float(v.y));
    f[1] = make_float2(__uint_as_float(v.z), __uint_as_float(v.w));
  } else {
    const typename Two<T>::P* p = reinterpret_cast<const typename Two<T>::P*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = Two<T>::f(p[i]);
  }
}

template <typename T>
__device__ __forceinline__ float vec_max(const uint4& v) {
  if constexpr (sizeof(T) == 4) {
    return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)), fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
  } else {
    const typename Two<T>::P* p = reinterpret_cast<const typename Two<T>::P*>(&v);
    const float2 f = Two<T>::f(__hmax2(__hmax2(p[0], p[1]), __hmax2(p[2], p[3])));
    return fmaxf(f.x, f.y);
  }
}

// What thread `t` of `G` sees of the `n` elements at p: running maximum and sum, U vectors of 16 bytes at a time.  Elements
// before the first 16-byte boundary and behind the last are taken one by one, so rows of odd length cost no more than
// aligned ones.
template <typename T, int G, int U>
__device__ __forceinline__ MaxSum scan(const T* p, int n, const Scale& c, int t) {
  constexpr int V = 16 / sizeof(T), H = V / 2;
  MaxSum a{-INFINITY, 0.f};
  // The maximum follows when a term passes 2: that is seldom after a thread's first vectors.
  auto raise = [&](float mx) {
    if (mx > a.m + c.slack) { a.s *= expf((a.m - mx) * c.inv); a.m = mx; }   // (see rescale)
  };
  auto one = [&](T x) {
    const float z = Cvt<T>::to_f(x);
    raise(z);
    if (z != -INFINITY) a.s += ex2(c(z - a.m));                    // (NaN comes through: NaN - m)
  };
  // The hardware's exponential is 5e-8 of its result too small on average for negative arguments (2e-8 above -1) and 3.4e-8 too
  // large for positive ones (above 1).  So one of two neighbours is taken times 2^6: the errors of a sum cancel, where
  // they shifted the log-probabilities of rows of 151936 by 2.8e-8 each, all the same way.
  const float2 hi = make_float2(c.hi, c.hi), lo = make_float2(c.lo, c.lo);
  auto add = [&](const uint4& v) {
    float2 f[H], sum = make_float2(0.f, 0.f);
    unpack<T>(v, f);
    const float m = a.m == -INFINITY ? 0.f : a.m;                  // (all -inf so far: they add nothing to a sum of 0)
    const float2 nm = make_float2(-m, -m);
#pragma unroll
    for (int i = 0; i < H; ++i) {
      const float2 d = add2(f[i], nm);
      float2 e = fma2(d, hi, mul2(d, lo));
      e.y += 6.f;
      e.x = ex2(e.x); e.y = ex2(e.y);
      sum = add2(sum, e);
    }
    a.s += fmaf(sum.y, 0.015625f, sum.x);
  };
  const int mis = (int)((reinterpret_cast<uintptr_t>(p) & 15) / sizeof(T));
  int head = mis ? V - mis : 0;
  if (head > n) head = n;
  const uint4* v = reinterpret_cast<const uint4*>(p + head);
  const int nv = (n - head) / V, rest = head + nv * V + t;
  if (t < head) one(p[t]);
  int i = t;
  for (; i + (U - 1) * G < nv; i += U * G) {
    uint4 x[U];
    float mx = -INFINITY;
#pragma unroll
    for (int k = 0; k < U; ++k) x[k] = v[i + k * G];
#pragma unroll
    for (int k = 0; k < U; ++k) mx = fmaxf(mx, vec_max<T>(x[k]));
    raise(mx);
#pragma unroll
    for (int k = 0; k < U; ++k) add(x[k]);
  }
  for (; i < nv; i += G) {
    const uint4 x = v[i];
    raise(vec_max<T>(x));
    add(x);
  }
  if (rest < n) one(p[rest]);
  return a;
}

// (max, sum) of the warp's parts, in every lane
__device__ __forceinline__ MaxSum warp_join(MaxSum a, float temperature) {
  const float m = warp_max(a.m);
  return MaxSum{m, warp_sum(rescale(a, m, temperature))};
}

// The token of a row; false where the row does not count.  A token outside the vocabulary is reported and does not count.
template <typename TI>
__device__ __forceinline__ bool counts(const TI* tokens, long long r, long long cols, long long ignore, long long& t) {
  t = (long long)tokens[r];
  return t != ignore && t >= 0 && t < cols;
}

// One row's results, by one thread
template <typename T, typename TI>
__device__ __forceinline__ void finish_row(MaxSum a, const T* p, long long t, long long r, long long rows, double temperature,
                                           float* lp_out, float* stats, const Policy& q) {
  // In 64 bits and rounded once; the temperature too, which rounded would shift every row by up to 6e-8 of its exponent.
  // Differences come before products: z[t] - m is small where the token is likely.
  const double wide = ((double)Cvt<T>::to_f(p[t]) - (double)a.m) / temperature - log((double)a.s);
  const float lp = (float)wide;
  if (q.wide != nullptr) q.wide[r] = wide;
  else lp_out[r] = lp;
  stats[r] = a.m;
  stats[rows + r] = sizeof(T) == 4 ? a.s : log2f(a.s);             // (see grad_part)
  if (q.old != nullptr) {
    const float A = q.adv[r / q.adv_div];
    const float ratio = expf(lp - q.old[r]);
    const float plain = -A * ratio, clipped = -A * fminf(fmaxf(ratio, q.lo), q.hi);
    float loss = fmaxf(plain, clipped), coef = plain >= clipped ? plain : 0.f;
    if (plain != plain || clipped != clipped) { loss = plain + clipped; coef = loss; }      // NaN stays NaN
    if (q.ref != nullptr) {
      const float d = q.ref[r] - lp, e1 = expm1f(d);               // (exp(d) - 1 would lose what a small d adds)
      loss += q.kl * (e1 - d);
      coef -= q.kl * e1;
    }
    q.loss[r] = loss;
    q.coef[r] = coef;
  }
}

__device__ __forceinline__ void skip_row(long long r, long long rows, float* lp_out, float* stats, const Policy& q) {
  if (q.wide != nullptr) q.wide[r] = 0.0;
  else lp_out[r] = 0.f;
  stats[r] = 0.f;
  stats[rows + r] = 0.f;
  if (q.old != nullptr) { q.loss[r] = 0.f; q.coef[r] = 0.f; }
}

// Rows of up to a few KB: one warp each.
template <typename T, typename TI>
__global__ void __launch_bounds__(256)
token_rows_warp_kernel(const T* __restrict__ z, RowMap map, const TI* __restrict__ tokens, float* __restrict__ lp,
                       float* __restrict__ stats, long long rows, int cols, long long ignore, double temperature, Scale c,
                       Policy q, int* status) {
  const int lane = threadIdx.x & 31;
  const long long r = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (r >= rows) return;
  long long t;
  if (!counts(tokens, r, cols, ignore, t)) {
    if (lane == 0) {
      if (t != ignore) report_error(status, GB_ERR_BAD_INDEX, SITE_TOKEN, (int)t);
      skip_row(r, rows, lp, stats, q);
    }
    return;
  }
  const T* p = z + map.at(r);
  const MaxSum a = warp_join(scan<T, 32, 4>(p, cols, c, lane), (float)temperature);
  if (lane == 0) finish_row<T, TI>(a, p, t, r, rows, temperature, lp, stats, q);
}

// Longer rows: one CTA of G threads each, or, where rows are few, the CTAs of a cluster share one and rank 0 joins their
// parts through distributed shared memory.  A thread has U vectors in flight; OCC CTAs fit an SM.
template <typename T, typename TI, int G, int U, int OCC>
__global__ void __launch_bounds__(G, OCC)
token_rows_kernel(const T* __restrict__ z, RowMap map, const TI* __restrict__ tokens, float* __restrict__ lp,
                  float* __restrict__ stats, long long rows, int cols, long long ignore, double temperature, Scale c,
                  Policy q, int* status, int parts) {
  __shared__ float2 sh[G / 32];
  __shared__ float2 mine;
  const long long r = blockIdx.x / parts;
  const int part = blockIdx.x % parts;
  long long t;
  if (!counts(tokens, r, cols, ignore, t)) {                       // (alike in all CTAs of the cluster)
    if (part == 0 && threadIdx.x == 0) {
      if (t != ignore) report_error(status, GB_ERR_BAD_INDEX, SITE_TOKEN, (int)t);
      skip_row(r, rows, lp, stats, q);
    }
    return;
  }
  const T* p = z + map.at(r);
  int lo = 0, n = cols;
  if (parts > 1) {
    const int step = ((cols + parts - 1) / parts + 7) & ~7;
    lo = min(part * step, cols);
    n = min(step, cols - lo);
  }
  MaxSum a = warp_join(scan<T, G, U>(p + lo, n, c, threadIdx.x), (float)temperature);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = make_float2(a.m, a.s);
  __syncthreads();
  if (threadIdx.x < 32) {
    a = MaxSum{-INFINITY, 0.f};
    if (threadIdx.x < G / 32) a = MaxSum{sh[threadIdx.x].x, sh[threadIdx.x].y};
    a = warp_join(a, (float)temperature);
  }
  if (parts > 1) {
    cg::cluster_group cl = cg::this_cluster();
    if (threadIdx.x == 0) mine = make_float2(a.m, a.s);
    cl.sync();
    if (part == 0 && threadIdx.x == 0) {
      float m = a.m;
      for (int k = 1; k < parts; ++k) m = fmaxf(m, cl.map_shared_rank(&mine, k)->x);
      float sum = rescale(a, m, (float)temperature);
      for (int k = 1; k < parts; ++k) {
        const float2 o = *cl.map_shared_rank(&mine, k);
        sum += rescale(MaxSum{o.x, o.y}, m, (float)temperature);
      }
      a = MaxSum{m, sum};
    }
    cl.sync();                                                     // nobody leaves while its part may still be read
  }
  if (part == 0 && threadIdx.x == 0) finish_row<T, TI>(a, p, t, r, rows, temperature, lp, stats, q);
}

__device__ __forceinline__ double block_sum64(double v, double* sh) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  v = (threadIdx.x & 31) < (blockDim.x >> 5) ? sh[threadIdx.x & 31] : 0.0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// *out = sum of the rows' losses (over the number of rows that count), *factor = the factor of every row's gradient
template <typename TI>
__global__ void __launch_bounds__(1024)
policy_sum_kernel(const float* __restrict__ loss, const TI* __restrict__ tokens, long long rows, long long cols,
                  long long ignore, int mean, float* __restrict__ out, float* __restrict__ factor) {
  __shared__ double sh[32];
  double sum = 0.0, n = 0.0;
  for (long long r = threadIdx.x; r < rows; r += 1024) {
    long long t;
    if (counts(tokens, r, cols, ignore, t)) { sum += (double)loss[r]; n += 1.0; }
  }
  sum = block_sum64(sum, sh);
  n = block_sum64(n, sh);
  if (threadIdx.x == 0) {
    const double f = mean && n > 0.0 ? 1.0 / n : 1.0;
    *out = (float)(sum * f);
    *factor = (float)f;
  }
}

// Pair i: answers i (chosen) and pairs + i (rejected) of `len` rows each.  loss_each [pairs] or null; out[0] = their sum
// (or mean); rewards [2 pairs] = beta (S - ref), ref in 32 or 64 bits; gseq [2 pairs] = dl/dS.  Everything is in 64 bits until it goes out: rewards
// may be large where their difference is of order one, so that is formed from `wide` [2 pairs], rewards before they are rounded.
__global__ void __launch_bounds__(1024)
preference_kernel(const double* __restrict__ lp, const void* __restrict__ ref, int ref_f64, long long pairs, long long len, double beta,
                  double smooth, int mean, float* __restrict__ loss_each, float* __restrict__ out, float* __restrict__ rewards,
                  double* __restrict__ wide, float* __restrict__ gseq) {
  __shared__ double sh[32];
  const int lane = threadIdx.x & 31;
  for (long long s = threadIdx.x >> 5; s < 2 * pairs; s += 32) {
    const double* p = lp + s * len;
    double sum = 0.0;
    for (long long i = lane; i < len; i += 32) sum += p[i];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) {
      wide[s] = beta * (sum - (ref_f64 ? reinterpret_cast<const double*>(ref)[s] : (double)reinterpret_cast<const float*>(ref)[s]));
      rewards[s] = (float)wide[s];
    }
  }
  __syncthreads();
  double total = 0.0;
  for (long long i = threadIdx.x; i < pairs; i += 1024) {
    const double h = wide[i] - wide[pairs + i];
    // log(1 + exp(-|h|)) is common to both signs: -log sigmoid(h) = max(-h, 0) + it
    const double l1 = log1p(exp(-fabs(h)));
    // a side of weight 0 is left out: h is infinite where an answer holds a token of probability 0
    double loss = h != h ? h : 0.0;
    if (smooth < 1.0) loss += (1.0 - smooth) * (fmax(-h, 0.0) + l1);
    if (smooth > 0.0) loss += smooth * (fmax(h, 0.0) + l1);
    const float g = (float)(beta * (smooth - 1.0 / (1.0 + exp(h))));
    gseq[i] = g;
    gseq[pairs + i] = -g;
    if (loss_each != nullptr) loss_each[i] = (float)loss;
    total += loss;
  }
  total = block_sum64(total, sh);
  if (threadIdx.x == 0) out[0] = (float)(mean && pairs > 0 ? total / (double)pairs : total);
}

// A row's factor: base[r / base_div] * g[r / g_div % g_mod] * *dev_scale * scale, each pointer null for 1
struct Factor {
  const float* base; const float* g; const float* dev_scale;
  long long base_div, g_div, g_mod;
  float scale;
  __device__ __forceinline__ float at(long long r) const {
    float f = scale;
    if (dev_scale != nullptr) f *= *dev_scale;
    if (g != nullptr) f *= g[(r / g_div) % g_mod];
    if (base != nullptr) f *= base[r / base_div];
    return f;
  }
};

constexpr int BWD_THREADS = 256;

// Gradient of `n` elements of a row by `G` threads; `t` counts from the first of them.
template <typename T, int G>
__device__ __forceinline__ void grad_part(const T* p, T* d, int n, long long t, float m, float stat, const Scale& c, float f, int tid) {
  constexpr int V = 16 / sizeof(T), H = V / 2, U = 4;
  // Probabilities of 32-bit logits: the exponential of an argument formed with both parts of log2(e) / T, over s.  With log2 s
  // in the exponent instead, rounded to 32 bits, all of a row of 151936 would be off by up to 6.6e-7 of themselves, the same
  // way; 16-bit gradients, rounded to 5e-4 and more, do not show that, and take one instruction where this takes three.
  constexpr bool EXACT = sizeof(T) == 4;
  const float hi = c.hi + c.lo, ls = stat, rs = EXACT ? 1.f / stat : 1.f;
  auto one = [&](int j) {
    const float x = Cvt<T>::to_f(p[j]) - m;
    const float e = EXACT ? ex2(c(x)) * rs : ex2(fmaf(x, hi, -ls));
    d[j] = Cvt<T>::from_f(f * ((j == t ? 1.f : 0.f) - e));
  };
  const int mis = (int)((reinterpret_cast<uintptr_t>(d) & 15) / sizeof(T));
  int head = mis ? V - mis : 0;
  if (head > n) head = n;
  const bool same = ((reinterpret_cast<uintptr_t>(p) ^ reinterpret_cast<uintptr_t>(d)) & 15) == 0;
  const int nv = same ? (n - head) / V : 0;
  const uint4* src = reinterpret_cast<const uint4*>(p + head);
  uint4* dst = reinterpret_cast<uint4*>(d + head);
  const float2 nm = make_float2(-m, -m), nf = make_float2(-f, -f), nl = make_float2(-ls, -ls), r2 = make_float2(rs, rs);
  const float2 c2 = EXACT ? make_float2(c.hi, c.hi) : make_float2(hi, hi), lo = make_float2(c.lo, c.lo);
  const long long tv = t < head ? -1 : (t - head) / V;             // the vector that holds the token
  auto vec = [&](const uint4& x, int i) {
    float2 e[H];
    unpack<T>(x, e);
#pragma unroll
    for (int k = 0; k < H; ++k) {
      const float2 x = add2(e[k], nm);
      e[k] = fma2(x, c2, EXACT ? mul2(x, lo) : nl);
      e[k].x = ex2(e[k].x); e[k].y = ex2(e[k].y);
      if constexpr (EXACT) e[k] = mul2(e[k], r2);
    }
    if (i == tv) {
      const int at = (int)((t - head) % V);
#pragma unroll
      for (int k = 0; k < H; ++k) {
        if (2 * k == at) e[k].x -= 1.f;
        if (2 * k + 1 == at) e[k].y -= 1.f;
      }
    }
    uint4 o;
    uint32_t* w = reinterpret_cast<uint32_t*>(&o);
#pragma unroll
    for (int k = 0; k < H; ++k) {
      e[k] = mul2(e[k], nf);
      if constexpr (sizeof(T) == 4) { w[2 * k] = __float_as_uint(e[k].x); w[2 * k + 1] = __float_as_uint(e[k].y); }
      else w[k] = Two<T>::pack(e[k].x, e[k].y);
    }
    dst[i] = o;
  };
  if (same) {
    if (tid < head) one(tid);
    int i = tid;
    for (; i + (U - 1) * G < nv; i += U * G) {
      uint4 x[U];
#pragma unroll
      for (int k = 0; k < U; ++k) x[k] = src[i + k * G];
#pragma unroll
      for (int k = 0; k < U; ++k) vec(x[k], i + k * G);
    }
    for (; i < nv; i += G) vec(src[i], i);
    const int rest = head + nv * V + tid;
    if (rest < n) one(rest);
  } else {
    for (int j = tid; j < n; j += G) one(j);
  }
}

template <typename T, int G>
__device__ __forceinline__ void zero_part(T* d, int n, int tid) {
  constexpr int V = 16 / sizeof(T);
  const int mis = (int)((reinterpret_cast<uintptr_t>(d) & 15) / sizeof(T));
  int head = mis ? V - mis : 0;
  if (head > n) head = n;
  const int nv = (n - head) / V;
  if (tid < head) d[tid] = Cvt<T>::from_f(0.f);
  uint4* dst = reinterpret_cast<uint4*>(d + head);
  for (int i = tid; i < nv; i += G) dst[i] = make_uint4(0, 0, 0, 0);
  const int rest = head + nv * V + tid;
  if (rest < n) d[rest] = Cvt<T>::from_f(0.f);
}

// `G` threads per item; an item is `chunk` elements of one row.  Rows run from the last to the first: the forward pass
// has left the last ones in L2.
template <typename T, typename TI, int G>
__global__ void __launch_bounds__(BWD_THREADS)
token_grad_kernel(const T* __restrict__ z, RowMap map, const TI* __restrict__ tokens, const float* __restrict__ stats,
                  T* __restrict__ dz, long long rows, int cols, long long ignore, Scale c, Factor fac,
                  int chunk, int chunks) {
  const int tid = threadIdx.x % G;
  const long long item = (long long)blockIdx.x * (BWD_THREADS / G) + threadIdx.x / G;
  if (item >= rows * chunks) return;
  const long long r = rows - 1 - item / chunks;
  const int lo = (int)(item % chunks) * chunk;
  const int n = min(chunk, cols - lo);
  T* d = dz + r * cols + lo;
  long long t;
  const float f = counts(tokens, r, cols, ignore, t) ? fac.at(r) * c.inv : 0.f;
  if (f == 0.f) { zero_part<T, G>(d, n, tid); return; }
  grad_part<T, G>(z + map.at(r) + lo, d, n, t - lo, stats[r], stats[rows + r], c, f, tid);
}

template <typename T, typename TI>
static int rows_forward(const void* z, RowMap map, const void* tokens, float* lp, float* stats, long long rows, int cols,
                        long long ignore, double temperature, const Policy& q, int* status, cudaStream_t st) {
  const Scale c(temperature);
  const long long bytes = (long long)cols * sizeof(T), sms = sm_count();
  // A warp a row up to 8 KB, 128 threads up to 32 KB, as long as these fill the device
  if (bytes <= 2048 || (bytes <= 8192 && rows >= 32 * sms)) {
    token_rows_warp_kernel<T, TI><<<(unsigned)((rows + 7) / 8), 256, 0, st>>>(
        (const T*)z, map, (const TI*)tokens, lp, stats, rows, cols, ignore, temperature, c, q, status);
    return (int)cudaGetLastError();
  }
  int parts = 1;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  auto run = [&](auto kernel, int threads) {
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = parts; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3((unsigned)(rows * parts)); cfg.blockDim = dim3(threads); cfg.stream = st;
    cfg.attrs = attr; cfg.numAttrs = parts > 1 ? 1 : 0;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, (const T*)z, map, (const TI*)tokens, lp, stats, rows, cols, ignore,
                                             temperature, c, q, status, parts);
    return e == cudaSuccess ? (int)cudaGetLastError() : (int)e;
  };
  if (bytes <= 8192 || (bytes <= 32768 && rows >= 8 * sms)) return run(token_rows_kernel<T, TI, 128, 4, 8>, 128);
  // Up to two rows an SM: as many threads and vectors in flight as a row can use.  Clusters pay up to one CTA an SM, in parts
  // that are worth their barriers.  Rows of 151936 bf16, one CTA / clusters of 4, us: 16 rows 18.4 / 12.3, 40 18.4 / 14.3,
  // 74 18.4 / 20.5; of 24000 8.2 / 10.2.  256 threads instead, 148 rows: 26.7 for 20.5.
  if (rows <= 2 * sms) {
    while (parts < 8 && rows * parts * 2 <= sms && cols / (parts * 2) >= 16384) parts *= 2;
    return run(token_rows_kernel<T, TI, 512, 4, 2>, 512);
  }
  // More rows: smaller CTAs, so that fewer threads wait for a row's slowest warp and the last rows spread better.  Of 151936
  // bf16, 512 / 256 threads: 1000 rows 75.8 / 71.7, 6973 rows 367 / 352.  16-bit rows are bound by the exponentials as much as by
  // memory: five CTAs of 48 registers 354 (6.0 TB/s), four of 60 385, eight of 32, which spill, with two vectors 363; of 50257
  // fp16, 1250 rows 41.0 / 45.0 / 47.1.  32-bit rows, 2000 of 65536, in the same order: 100, 104, 107, and 1000 of 151936 125, 115, 127.
  return run(token_rows_kernel<T, TI, 256, 4, sizeof(T) == 2 ? 5 : 4>, 256);
}

template <typename T, typename TI>
static int rows_backward(const void* z, RowMap map, const void* tokens, const float* stats, void* dz, long long rows, int cols,
                         long long ignore, double temperature, const Factor& fac, cudaStream_t st) {
  const Scale c(temperature);
  if ((long long)cols * sizeof(T) <= 8192 && (cols <= 1024 || rows >= 32ll * sm_count())) {
    token_grad_kernel<T, TI, 32><<<(unsigned)((rows + 7) / 8), BWD_THREADS, 0, st>>>(
        (const T*)z, map, (const TI*)tokens, stats, (T*)dz, rows, cols, ignore, c, fac, cols, 1);
    return (int)cudaGetLastError();
  }
  const int chunk = 16384 / (int)sizeof(T) * 2;
  const int chunks = (cols + chunk - 1) / chunk;
  if (rows * chunks > 0x7fffffffll) return -3;
  token_grad_kernel<T, TI, BWD_THREADS><<<(unsigned)(rows * chunks), BWD_THREADS, 0, st>>>(
      (const T*)z, map, (const TI*)tokens, stats, (T*)dz, rows, cols, ignore, c, fac, chunk, chunks);
  return (int)cudaGetLastError();
}

static int rows_any(const void* z, const void* tokens, float* lp, float* stats, long long rows, long long cols, RowMap map,
                    long long ignore, double temperature, const Policy& q, int dt, int token_i64, int* status, cudaStream_t st) {
  if (rows == 0) return 0;
  if (cols < 1 || cols > 0x40000000ll || rows > 0x0fffffffll || map.inner < 1 || !(temperature >= 1e-6 && temperature <= 1e20)) return -3;
  if (token_i64) GB_DISPATCH_FLOAT(dt, T, return (rows_forward<T, long long>(z, map, tokens, lp, stats, rows, (int)cols, ignore, temperature, q, status, st)));
  GB_DISPATCH_FLOAT(dt, T, return (rows_forward<T, int>(z, map, tokens, lp, stats, rows, (int)cols, ignore, temperature, q, status, st)));
}

}  // namespace tl
}  // namespace gb

using namespace gb;

// Log-probabilities lp [rows] of `tokens` and what gb_token_grad needs of the rows in stats [2, rows].  Rows: see RowMap.
extern "C" int gb_token_rows(const void* z, const void* tokens, float* lp, float* stats, long long rows, long long cols,
                             long long inner, long long s_outer, long long s_inner, long long ignore, double temperature,
                             int dt, int token_i64, int* status, cudaStream_t st) {
  return tl::rows_any(z, tokens, lp, stats, rows, cols, tl::RowMap{inner, s_outer, s_inner}, ignore, temperature, tl::Policy{},
                      dt, token_i64, status, st);
}

// The same, and every row's clipped policy loss [rows] and its derivative by lp, coef [rows]; out (or null) receives the sum
// of the losses (over the number of rows that count with `mean`), factor that of their gradients.
extern "C" int gb_policy_loss(const void* z, const void* tokens, float* lp, float* stats, long long rows, long long cols,
                              long long inner, long long s_outer, long long s_inner, long long ignore, double temperature,
                              const float* old, const float* adv, const float* ref, float* loss, float* coef, long long adv_div,
                              float lo, float hi, float kl, float* out, float* factor, int mean, int dt, int token_i64, int* status,
                              cudaStream_t st) {
  if (adv_div < 1) return -3;
  const tl::Policy q{old, adv, ref, loss, coef, adv_div, lo, hi, kl};
  if (const int e = tl::rows_any(z, tokens, lp, stats, rows, cols, tl::RowMap{inner, s_outer, s_inner}, ignore, temperature, q,
                                 dt, token_i64, status, st)) return e;
  if (out == nullptr) return 0;
  if (token_i64) tl::policy_sum_kernel<long long><<<1, 1024, 0, st>>>(loss, (const long long*)tokens, rows, cols, ignore, mean, out, factor);
  else tl::policy_sum_kernel<int><<<1, 1024, 0, st>>>(loss, (const int*)tokens, rows, cols, ignore, mean, out, factor);
  return (int)cudaGetLastError();
}

// Log-probabilities as gb_token_rows gives them, but in 64 bits, and the loss of `pairs` pairs of answers of rows / (2 pairs)
// rows each, in 64 bits too (`wide` [2 pairs] is room for them): see preference_kernel.
extern "C" int gb_preference_loss(const void* z, const void* tokens, double* lp, float* stats, long long rows, long long cols,
                                  long long inner, long long s_outer, long long s_inner, long long ignore, const void* ref, int ref_f64,
                                  long long pairs, double beta, double smooth, int mean, float* loss_each, float* out,
                                  float* rewards, double* wide, float* gseq, int dt, int token_i64, int* status, cudaStream_t st) {
  tl::Policy q{};
  q.wide = lp;
  if (const int e = tl::rows_any(z, tokens, nullptr, stats, rows, cols, tl::RowMap{inner, s_outer, s_inner}, ignore, 1.0, q, dt,
                                 token_i64, status, st)) return e;
  tl::preference_kernel<<<1, 1024, 0, st>>>(lp, ref, ref_f64, pairs, pairs > 0 ? rows / (2 * pairs) : 0, beta, smooth, mean, loss_each, out,
                                            rewards, wide, gseq);
  return (int)cudaGetLastError();
}

// Gradient dz [rows, cols] (contiguous); a row's factor: see Factor.
extern "C" int gb_token_grad(const void* z, const void* tokens, const float* stats, void* dz, long long rows, long long cols,
                             long long inner, long long s_outer, long long s_inner, long long ignore, double temperature,
                             const float* base, long long base_div, const float* g, long long g_div, long long g_mod,
                             const float* dev_scale, float scale, int dt, int token_i64, cudaStream_t st) {
  if (rows == 0) return 0;
  if (cols < 1 || cols > 0x40000000ll || rows > 0x0fffffffll || inner < 1 || base_div < 1 || g_div < 1 || g_mod < 1 ||
      !(temperature >= 1e-6 && temperature <= 1e20)) return -3;
  const tl::RowMap map{inner, s_outer, s_inner};
  const tl::Factor fac{base, g, dev_scale, base_div, g_div, g_mod, scale};
  if (token_i64) GB_DISPATCH_FLOAT(dt, T, return (tl::rows_backward<T, long long>(z, map, tokens, stats, dz, rows, (int)cols, ignore, temperature, fac, st)));
  GB_DISPATCH_FLOAT(dt, T, return (tl::rows_backward<T, int>(z, map, tokens, stats, dz, rows, (int)cols, ignore, temperature, fac, st)));
}
