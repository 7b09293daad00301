// Attention of a sequence's newest tokens over the pages of its key / value cache, forward only, for sm_100a.
//
//   o[b, s, h] = sum_j p_j v_j,  p = softmax of scale * q . k_j over the j < lengths[b] - counts[b] + s + 1
//
// with K and V of KV head h / (Hq / Hkv), and zeros for a row that sees no key (a token that is none, or scores that are -inf
// throughout).  One pass over the keys with a running maximum and sum in 32 bits; keys behind the end are neither read nor
// multiplied, so what the rest of a page holds does not matter.
#include "paged_common.cuh"

namespace gb {

struct AttendArgs {
  const void* q;                     // [B, S, Hq, D]
  void* o;
  const void *kpool, *vpool;
  const uint8_t *kscale, *vscale;
  int Hq;
  float scale;
};

constexpr int PA_WARPS = 4, PA_MAX_D = 256;

// Any type and head size: a CTA takes a row of queries, its warps every fourth key, their lanes a share of the head.
template <typename T, int CDT>
__global__ void __launch_bounds__(PA_WARPS * 32) paged_attend_any_kernel(const AttendArgs a, const Paged c) {
  constexpr int N = PA_MAX_D / 32;
  __shared__ float sm_o[PA_WARPS][PA_MAX_D], sm_m[PA_WARPS], sm_l[PA_WARPS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int h = blockIdx.x % a.Hq, s = blockIdx.x / a.Hq % c.S, b = blockIdx.x / a.Hq / c.S;
  const int kvh = h / (a.Hq / c.Hkv), n = c.count(b);
  long long end = s < n ? (long long)c.length(b) - n + s + 1 : 0;
  if (end > c.capacity()) {
    if (threadIdx.x == 0) report_error(c.status, GB_ERR_BAD_INDEX, SITE_POSITION, (int)end - 1);
    end = c.capacity();
  }
  const T* q = reinterpret_cast<const T*>(a.q) + (((long long)b * c.S + s) * a.Hq + h) * c.D;
  float qv[N], o[N], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int d = i * 32 + lane;
    qv[i] = d < c.D ? Cvt<T>::to_f(q[d]) * a.scale : 0.f;
    o[i] = 0.f;
  }
  auto load = [&](const void* pool, long long e) {
    if constexpr (CDT == DT_E4M3) return from_e4m3x2(reinterpret_cast<const uint8_t*>(pool)[e]).x;
    else return load_as_float(pool, CDT, e);
  };
  for (int j = warp; j < end; j += PA_WARPS) {
    const long long row = c.row(b, j, kvh);
    if (row < 0) continue;
    float x = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i * 32 + lane < c.D) x += qv[i] * load(a.kpool, row * c.D + i * 32 + lane);
    x = warp_sum(x);
    float vs = 1.f;
    if constexpr (CDT == DT_E4M3) {
      x *= __uint_as_float((uint32_t)a.kscale[row] << 23);
      vs = __uint_as_float((uint32_t)a.vscale[row] << 23);
    }
    const float mn = fmaxf(m, x), base = mn == -INFINITY ? 0.f : mn;
    const float alpha = expf(m - base), p = expf(x - base);
    m = mn;
    l = l * alpha + p;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i * 32 + lane < c.D) o[i] = o[i] * alpha + p * vs * load(a.vpool, row * c.D + i * 32 + lane);
  }
#pragma unroll
  for (int i = 0; i < N; ++i) sm_o[warp][i * 32 + lane] = o[i];
  if (lane == 0) { sm_m[warp] = m; sm_l[warp] = l; }
  __syncthreads();
  float mc = -INFINITY, lc = 0.f;
  for (int w = 0; w < PA_WARPS; ++w) mc = fmaxf(mc, sm_m[w]);
  const float base = mc == -INFINITY ? 0.f : mc;
  for (int w = 0; w < PA_WARPS; ++w) lc += sm_l[w] * expf(sm_m[w] - base);
  for (int d = threadIdx.x; d < c.D; d += PA_WARPS * 32) {
    float acc = 0.f;
    for (int w = 0; w < PA_WARPS; ++w) acc += sm_o[w][d] * expf(sm_m[w] - base);
    reinterpret_cast<T*>(a.o)[(((long long)b * c.S + s) * a.Hq + h) * c.D + d] = Cvt<T>::from_f(lc == 0.f ? 0.f : acc / lc);
  }
}

#define GB_DISPATCH_CACHE(cdt, C, ...)                                    \
  do {                                                                    \
    if ((cdt) == DT_F32) { constexpr int C = DT_F32; __VA_ARGS__; }       \
    else if ((cdt) == DT_F16) { constexpr int C = DT_F16; __VA_ARGS__; }  \
    else if ((cdt) == DT_BF16) { constexpr int C = DT_BF16; __VA_ARGS__; } \
    else if ((cdt) == DT_E4M3) { constexpr int C = DT_E4M3; __VA_ARGS__; } \
    else return -2;                                                       \
  } while (0)

}  // namespace gb

using namespace gb;

extern "C" int gb_paged_attention(const void* q, void* o, const void* kpool, const void* vpool, const void* kscale,
                                  const void* vscale, const int* table, const int* lengths, const int* counts, int B, int S,
                                  int Hq, int Hkv, int D, int page, int pages, int per, float scale, int dt, int cdt,
                                  int* status, cudaStream_t st) {
  if (B <= 0 || S <= 0 || Hq <= 0 || D <= 0) return 0;
  if (D > PA_MAX_D || Hkv <= 0 || Hq % Hkv) return -3;
  AttendArgs a{q, o, kpool, vpool, (const uint8_t*)kscale, (const uint8_t*)vscale, Hq, scale};
  Paged c{table, lengths, counts, status, B, S, Hkv, D, page, pages, per};
  const long long rows = (long long)B * S * Hq;
  if (rows > 0x7fffffff) return -4;
  GB_DISPATCH_FLOAT(dt, T, GB_DISPATCH_CACHE(cdt, C, paged_attend_any_kernel<T, C><<<(unsigned)rows, PA_WARPS * 32, 0, st>>>(a, c)));
  return (int)cudaGetLastError();
}
