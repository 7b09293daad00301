// Writing keys and values into the pages of a cache, with the rotation of a fused q | k | v projection where there is one, and
// reading them back.
//
//   write : a row of D numbers for every (token, KV head), K and V, in the cache's type; e4m3 rows get the power of two of
//           their largest magnitude (paged_common.cuh), found in the registers that hold the row.
//   rotate: x1 cos - x2 sin, x2 cos + x1 sin over the halves of a head, at the token's position in its sequence; rotated keys
//           are rounded once, to the cache's type.
//   read  : rows of the pages as dense [B, L, Hkv, D], zeros behind each sequence's end.
//   bound : bytes; every one of these reads its input once and writes its output once.
#include "paged_common.cuh"

namespace gb {

struct Rows {              // [B, S, heads, D], the last dimension dense
  const void* p;
  long long sb, ss, sh;
};

struct PutArgs {
  Rows q, k, v;
  void* q_out;             // [B, S, Hq, D]
  void *kpool, *vpool;
  uint8_t *kscale, *vscale;
  const float *cosb, *sinb;     // [positions, D], halves equal (null where positions is 0)
  int positions, Hq;            // Hq = 0: keys and values only, not rotated
};

// N numbers (4 or 8) in 32 bits into a pool, in its type; e4m3 under the power of two 1 / inv, with infinities and NaN among them as
// NaN where they are `odd`
template <int CDT, int N>
__device__ __forceinline__ void store_numbers(void* pool, long long at, const float (&x)[N], float inv, bool odd) {
  if constexpr (CDT == DT_F32) {
#pragma unroll
    for (int j = 0; j < N; j += 4) *reinterpret_cast<float4*>(reinterpret_cast<float*>(pool) + at + j) = make_float4(x[j], x[j + 1], x[j + 2], x[j + 3]);
  } else if constexpr (CDT == DT_E4M3) {
    uint32_t w[N / 4];
#pragma unroll
    for (int j = 0; j < N; j += 4)
      w[j / 4] = (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(x[j] * inv, x[j + 1] * inv), __NV_SATFINITE, __NV_E4M3) |
                 (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(x[j + 2] * inv, x[j + 3] * inv), __NV_SATFINITE, __NV_E4M3) << 16;
    if (odd) {
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (!(fabsf(x[j]) < INFINITY)) w[j / 4] |= 0x7fu << j % 4 * 8;
    }
    if constexpr (N == 8) *reinterpret_cast<uint2*>(reinterpret_cast<uint8_t*>(pool) + at) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint32_t*>(reinterpret_cast<uint8_t*>(pool) + at) = w[0];
  } else {
    uint32_t w[N / 2];
#pragma unroll
    for (int j = 0; j < N; j += 2) w[j / 2] = pack2c<CDT == DT_BF16>(x[j], x[j + 1]);
    if constexpr (N == 8) *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(pool) + at) = make_uint4(w[0], w[1], w[2], w[3]);
    else *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(pool) + at) = make_uint2(w[0], w[1]);
  }
}

__device__ __forceinline__ float max_or_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Rows (token, head) lie one after another: a group of 2^log lanes takes a row, 16 bytes of each of its halves a lane, so the
// partner of a rotation is in the same registers and a row's largest magnitude a few shuffles away.  The row is asked for before
// it is known where its token stands.  One row a thread: with two, 8 x 2048 tokens of 14 / 2 heads of 64 took 21.5 us for 17.3 (of
// 11.8 that their bytes need), 8 x 4096 keys and values of 4 x 128 into 16 bits 28.8 for 25.7.
template <typename T, int CDT, bool ROPE>
__global__ void __launch_bounds__(256) paged_put_rows_kernel(const PutArgs a, const Paged c, const Div heads, const Div tokens, int rows, int log) {
  constexpr int V = 16 / sizeof(T);
  const int ch = threadIdx.x & ((1 << log) - 1), half = c.D / 2;
  const int Hq = ROPE ? a.Hq : 0, Hk = Hq + c.Hkv;
  const int r = (int)blockIdx.x * (256 >> log) + (threadIdx.x >> log);
  const int token = heads.by(r), h = r - token * heads.d, b = tokens.by(token), s = token - b * tokens.d;
  const bool there = r < rows, isq = h < Hq, isk = !isq && h < Hk;
  const int hh = isq ? h : isk ? h - Hq : h - Hk;
  float x[V], y[V];
#pragma unroll
  for (int j = 0; j < V; ++j) x[j] = y[j] = 0.f;
  int pos = -1;                        // -1: no token, or one without a rotation
  long long row = -1;                  // of the pool; -1: nowhere
  if (there) {
    const Rows& src = isq ? a.q : isk ? a.k : a.v;
    const T* p = reinterpret_cast<const T*>(src.p) + b * src.sb + s * src.ss + hh * src.sh + ch * V;
    const Vec16<T> lo = ld16(p), hi = ld16(p + half);
    const int n = c.count(b);
    pos = c.length(b) - n + s;
    if (s >= n || pos < 0) pos = -1;
    if (ROPE && pos >= a.positions) {
      report_error(c.status, GB_ERR_BAD_INDEX, SITE_POSITION, pos);
      pos = -1;
    }
    if (pos >= 0) {
      if (!isq) row = c.row(b, pos, hh);
#pragma unroll
      for (int j = 0; j < V; ++j) { x[j] = Cvt<T>::to_f(lo.v[j]); y[j] = Cvt<T>::to_f(hi.v[j]); }
      if (ROPE && (isq || isk)) {
        const float* cp = a.cosb + (long long)pos * c.D + ch * V;
        const float* sp = a.sinb + (long long)pos * c.D + ch * V;
        auto turn = [](float& p, float& q, float co, float si) { const float z = p * co - q * si; q = q * co + p * si; p = z; };
#pragma unroll
        for (int j = 0; j < V; j += 4) {
          const float4 cs = *reinterpret_cast<const float4*>(cp + j), sn = *reinterpret_cast<const float4*>(sp + j);
          turn(x[j], y[j], cs.x, sn.x); turn(x[j + 1], y[j + 1], cs.y, sn.y);
          turn(x[j + 2], y[j + 2], cs.z, sn.z); turn(x[j + 3], y[j + 3], cs.w, sn.w);
        }
      }
    }
  }
  int e = 0;
  bool odd = false;
  if constexpr (CDT == DT_E4M3) {
    float top = 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j) top = max_or_nan(max_or_nan(top, fabsf(x[j])), fabsf(y[j]));
    odd = !(top < INFINITY);           // infinities or NaN
    uint32_t m = __float_as_uint(top);
    if (odd) {
      m = 0;
#pragma unroll
      for (int j = 0; j < V; ++j) m = max(m, max(finite_bits(x[j]), finite_bits(y[j])));
    }
    for (int o = 1 << log >> 1; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    e = e4m3_exponent(m);
  }
  if (!there) return;
  if (isq) {
    Vec16<T> p, q;
#pragma unroll
    for (int j = 0; j < V; ++j) { p.v[j] = Cvt<T>::from_f(x[j]); q.v[j] = Cvt<T>::from_f(y[j]); }
    T* o = reinterpret_cast<T*>(a.q_out) + ((long long)token * Hq + h) * c.D + ch * V;
    st16(o, p);
    st16(o + half, q);
  } else if (row >= 0) {
    void* pool = isk ? a.kpool : a.vpool;
    const float inv = CDT == DT_E4M3 ? exp2i(-e) : 1.f;
    store_numbers<CDT, V>(pool, row * c.D + ch * V, x, inv, odd);
    store_numbers<CDT, V>(pool, row * c.D + ch * V + half, y, inv, odd);
    if (CDT == DT_E4M3 && ch == 0) (isk ? a.kscale : a.vscale)[row] = (uint8_t)(e + 127);
  }
}

// Any head size and any alignment: a warp takes a row, once for its largest magnitude and once to write it.
template <typename T, int CDT>
__global__ void paged_put_any_kernel(const PutArgs a, const Paged c) {
  const int lane = threadIdx.x & 31, Ht = a.Hq + 2 * c.Hkv, half = c.D / 2;
  const long long total = (long long)c.B * c.S * Ht, step = (long long)gridDim.x * (blockDim.x / 32);
  for (long long i = (long long)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32; i < total; i += step) {
    const int h = (int)(i % Ht), s = (int)(i / Ht % c.S), b = (int)(i / Ht / c.S);
    const bool isq = h < a.Hq, isk = !isq && h < a.Hq + c.Hkv;
    const int hh = isq ? h : isk ? h - a.Hq : h - a.Hq - c.Hkv;
    const Rows& r = isq ? a.q : isk ? a.k : a.v;
    const T* x = reinterpret_cast<const T*>(r.p) + b * r.sb + s * r.ss + hh * r.sh;
    const int n = c.count(b);
    const long long pos = (long long)c.length(b) - n + s;
    bool live = s < n && pos >= 0;
    const bool rot = a.Hq > 0 && (isq || isk);
    if (live && a.Hq > 0 && pos >= a.positions) {
      if (lane == 0) report_error(c.status, GB_ERR_BAD_INDEX, SITE_POSITION, (int)pos);
      live = false;
    }
    auto value = [&](int d) {
      const float v = Cvt<T>::to_f(x[d]);
      if (!rot) return v;
      const int o = d < half ? d + half : d - half;
      const float cs = a.cosb[pos * c.D + d], sn = a.sinb[pos * c.D + d], w = Cvt<T>::to_f(x[o]);
      return d < half ? v * cs - w * sn : v * cs + w * sn;
    };
    if (isq) {
      T* o = reinterpret_cast<T*>(a.q_out) + (((long long)b * c.S + s) * a.Hq + h) * c.D;
      for (int d = lane; d < c.D; d += 32) o[d] = Cvt<T>::from_f(live ? value(d) : 0.f);
      continue;
    }
    if (!live) continue;
    const long long row = c.row(b, (int)pos, hh);
    if (row < 0) continue;
    void* pool = isk ? a.kpool : a.vpool;
    if constexpr (CDT != DT_E4M3) {
      for (int d = lane; d < c.D; d += 32) store_from_float(pool, CDT, row * c.D + d, value(d));
    } else {
      uint32_t m = 0;
      for (int d = lane; d < c.D; d += 32) m = max(m, finite_bits(value(d)));
      m = __reduce_max_sync(0xffffffffu, m);
      const int e = e4m3_exponent(m);
      const float inv = exp2i(-e);
      uint8_t* o = reinterpret_cast<uint8_t*>(pool) + row * c.D;
      for (int d = lane; d < c.D; d += 32) o[d] = (uint8_t)to_e4m3x2(value(d) * inv, 0.f);
      if (lane == 0) (isk ? a.kscale : a.vscale)[row] = (uint8_t)(e + 127);
    }
  }
}

// One thread a number of the output.
template <typename T, int CDT>
__global__ void paged_read_any_kernel(const void* kpool, const void* vpool, const uint8_t* kscale, const uint8_t* vscale,
                                      void* kout, void* vout, int L, const Paged c) {
  const long long total = (long long)c.B * L * c.Hkv * c.D, step = (long long)gridDim.x * blockDim.x;
  for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += step) {
    const int d = (int)(i % c.D), h = (int)(i / c.D % c.Hkv), pos = (int)(i / c.D / c.Hkv % L), b = (int)(i / c.D / c.Hkv / L);
    float k = 0.f, v = 0.f;
    if (pos < c.length(b)) {
      const long long row = c.row(b, pos, h);
      if (row >= 0) {
        if constexpr (CDT == DT_E4M3) {
          k = from_e4m3x2(reinterpret_cast<const uint8_t*>(kpool)[row * c.D + d]).x * __uint_as_float((uint32_t)kscale[row] << 23);
          v = from_e4m3x2(reinterpret_cast<const uint8_t*>(vpool)[row * c.D + d]).x * __uint_as_float((uint32_t)vscale[row] << 23);
        } else {
          k = load_as_float(kpool, CDT, row * c.D + d);
          v = load_as_float(vpool, CDT, row * c.D + d);
        }
      }
    }
    reinterpret_cast<T*>(kout)[i] = Cvt<T>::from_f(k);
    reinterpret_cast<T*>(vout)[i] = Cvt<T>::from_f(v);
  }
}

// A block takes 16 positions of a sequence, which lie in one page: per KV head its rows are contiguous there.  A thread takes 8
// numbers of K and of V, so that it stores 16 contiguous bytes of 16 bits (8 x 4096 of 4 x 128 from 8 bits: 16.7 us, of 15.7 that the
// bytes need; 19.1 with 16 numbers a thread, 20.8 with two such rows asked for at once).
template <typename T, int CDT>
__global__ void __launch_bounds__(256) paged_read_rows_kernel(const void* __restrict__ kpool, const void* __restrict__ vpool,
                                                              const uint8_t* __restrict__ kscale, const uint8_t* __restrict__ vscale,
                                                              void* __restrict__ kout, void* __restrict__ vout, int L, int log,
                                                              const Paged c) {
  constexpr int N = 8;
  const int b = blockIdx.y, p0 = blockIdx.x * 16, groups = 1 << log;      // groups of N numbers in a row
  const int end = min(L, c.length(b));
  // (the page is asked for before the length is known)
  const int in_table = c.in_page.by(p0), id = in_table < c.per ? c.table[(size_t)b * c.per + in_table] : -1;
  long long row0 = -1;
  if (p0 < end) {
    if ((unsigned)id < (unsigned)c.pages) row0 = (long long)id * c.Hkv * c.page + p0 - in_table * c.page;
    else c.row(b, p0, 0);              // (records what is wrong)
  }
  const int there = row0 < 0 ? 0 : end - p0;
  for (int i = threadIdx.x; i < c.Hkv * 16 << log; i += 256) {
    const int g = i & (groups - 1), t = i >> log & 15, h = i >> log >> 4;
    if (p0 + t >= L) continue;
    const long long row = row0 + (long long)h * c.page + t, at = row * c.D + g * N;
    const long long out = (((long long)b * L + p0 + t) * c.Hkv + h) * c.D + g * N;
    float x[2][N];
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
      for (int j = 0; j < N; ++j) x[w][j] = 0.f;
    if (t < there) {
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const void* pool = w ? vpool : kpool;
        if constexpr (CDT == DT_E4M3) {
          alignas(8) uint32_t v[N / 4];
          *reinterpret_cast<uint2*>(v) = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint8_t*>(pool) + at);
          const float sc = __uint_as_float((uint32_t)(w ? vscale : kscale)[row] << 23);
#pragma unroll
          for (int j = 0; j < N / 4; ++j) {
            uint32_t lo, hi;
            e4m3x4_to_f16(v[j], lo, hi);
            const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&lo)), q = __half22float2(*reinterpret_cast<const __half2*>(&hi));
            x[w][4 * j] = p.x * sc; x[w][4 * j + 1] = p.y * sc; x[w][4 * j + 2] = q.x * sc; x[w][4 * j + 3] = q.y * sc;
          }
        } else if constexpr (CDT == DT_F32) {
#pragma unroll
          for (int j = 0; j < N; j += 4) {
            const float4 v = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(pool) + at + j);
            x[w][j] = v.x; x[w][j + 1] = v.y; x[w][j + 2] = v.z; x[w][j + 3] = v.w;
          }
        } else {
          alignas(16) uint16_t v[8];
          *reinterpret_cast<uint4*>(v) = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(pool) + at);
#pragma unroll
          for (int j = 0; j < 8; ++j) x[w][j] = half_bits_to_float(v[j], CDT);
        }
      }
    }
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      T* o = reinterpret_cast<T*>(w ? vout : kout) + out;
      constexpr int V = 16 / sizeof(T);
#pragma unroll
      for (int j = 0; j < N; j += V) {
        Vec16<T> v;
#pragma unroll
        for (int k = 0; k < V; ++k) v.v[k] = Cvt<T>::from_f(x[w][j + k]);
        st16(o + j, v);
      }
    }
  }
}

// exponent of a power of two; -1: none
static inline int log2_of(int x) {
  int l = 0;
  while (x > 1 << l) ++l;
  return x == 1 << l ? l : -1;
}

}  // namespace gb

using namespace gb;

static int paged_put(const PutArgs& a, const Paged& c, const PagedPools& p, int dt, cudaStream_t st) {
  const int Ht = a.Hq + 2 * p.Hkv;
  const long long tokens = (long long)c.B * c.S;
  const int V = dt == DT_F32 ? 4 : 8, log = p.D % (2 * V) == 0 ? log2_of(p.D / (2 * V)) : -1;
  auto wide = [&](const Rows& r) { return ((uintptr_t)r.p & 15) == 0 && r.sb % V == 0 && r.ss % V == 0 && r.sh % V == 0; };
  const long long rows = tokens * Ht;
  if (log >= 0 && log <= 5 && wide(a.k) && wide(a.v) && (a.Hq == 0 || wide(a.q)) && (((uintptr_t)a.cosb | (uintptr_t)a.sinb) & 15) == 0 && rows < 1 << 30) {
    const int each = 256 >> log;
    const unsigned grid = (unsigned)((rows + each - 1) / each);
    const Div heads(Ht), per(c.S);
    if (a.Hq > 0) GB_DISPATCH_FLOAT(dt, T, GB_DISPATCH_CACHE(p.type, C, paged_put_rows_kernel<T, C, true><<<grid, 256, 0, st>>>(a, c, heads, per, (int)rows, log)));
    else GB_DISPATCH_FLOAT(dt, T, GB_DISPATCH_CACHE(p.type, C, paged_put_rows_kernel<T, C, false><<<grid, 256, 0, st>>>(a, c, heads, per, (int)rows, log)));
    return (int)cudaGetLastError();
  }
  GB_DISPATCH_FLOAT(dt, T, GB_DISPATCH_CACHE(p.type, C, paged_put_any_kernel<T, C><<<gb_grid(rows, 8), 256, 0, st>>>(a, c)));
  return (int)cudaGetLastError();
}

// k, v: [B, S, Hkv, D] through strides of elements, the last dimension dense.  Tokens of one call that share a slot of the cache are
// written in no order.
extern "C" int gb_paged_write(const void* pools, const void* k, long long kb, long long ks, long long kh, const void* v, long long vb,
                              long long vs, long long vh, const int* table, const int* lengths, const int* counts, int B, int S,
                              int per, int dt, int* status, cudaStream_t st) {
  const PagedPools& p = *reinterpret_cast<const PagedPools*>(pools);
  if (B <= 0 || S <= 0 || p.Hkv <= 0 || p.D <= 0) return 0;
  const PutArgs a{{nullptr, 0, 0, 0}, {k, kb, ks, kh}, {v, vb, vs, vh}, nullptr, p.k, p.v, p.kscale, p.vscale, nullptr, nullptr, 0, 0};
  return paged_put(a, Paged{table, lengths, counts, status, B, S, p.Hkv, p.D, p.page, p.pages, per, Div(p.page)}, p, dt, st);
}

// y: [B, S, (Hq + 2 Hkv) D] through the strides yb and ys; rotated queries go to q_out [B, S, Hq, D], rotated keys and values to the
// pages.
extern "C" int gb_paged_qkv_rope(const void* pools, const void* y, long long yb, long long ys, void* q_out, const float* cosb,
                                 const float* sinb, int positions, const int* table, const int* lengths, const int* counts, int B,
                                 int S, int Hq, int per, int dt, int* status, cudaStream_t st) {
  const PagedPools& p = *reinterpret_cast<const PagedPools*>(pools);
  if (B <= 0 || S <= 0 || p.Hkv <= 0 || p.D <= 0 || Hq <= 0) return 0;
  const long long head = (long long)p.D * (dt == DT_F32 ? 4 : 2);
  const char* x = reinterpret_cast<const char*>(y);
  const PutArgs a{{x, yb, ys, p.D}, {x + Hq * head, yb, ys, p.D}, {x + (Hq + p.Hkv) * head, yb, ys, p.D}, q_out,
                  p.k, p.v, p.kscale, p.vscale, cosb, sinb, positions, Hq};
  return paged_put(a, Paged{table, lengths, counts, status, B, S, p.Hkv, p.D, p.page, p.pages, per, Div(p.page)}, p, dt, st);
}

extern "C" int gb_paged_read(const void* pools, void* kout, void* vout, const int* table, const int* lengths, int B, int L, int per,
                             int dt, int* status, cudaStream_t st) {
  const PagedPools& p = *reinterpret_cast<const PagedPools*>(pools);
  if (B <= 0 || L <= 0 || p.Hkv <= 0 || p.D <= 0) return 0;
  const Paged c{table, lengths, nullptr, status, B, 0, p.Hkv, p.D, p.page, p.pages, per, Div(p.page)};
  const int log = p.D % 8 == 0 ? log2_of(p.D / 8) : -1;
  if (log >= 0 && p.page % 16 == 0 && B <= 65535 && (long long)p.Hkv * 16 << log < 1 << 30) {
    const dim3 grid((L + 15) / 16, B);
    GB_DISPATCH_FLOAT(dt, T, GB_DISPATCH_CACHE(p.type, C, paged_read_rows_kernel<T, C><<<grid, 256, 0, st>>>(
        p.k, p.v, p.kscale, p.vscale, kout, vout, L, log, c)));
    return (int)cudaGetLastError();
  }
  const long long total = (long long)B * L * p.Hkv * p.D;
  GB_DISPATCH_FLOAT(dt, T, GB_DISPATCH_CACHE(p.type, C, paged_read_any_kernel<T, C><<<gb_grid(total, 256), 256, 0, st>>>(
      p.k, p.v, p.kscale, p.vscale, kout, vout, L, c)));
  return (int)cudaGetLastError();
}
