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
  const float *cosb, *sinb;     // [positions, D], halves equal; null: no rotation, Hq = 0
  int positions, Hq;
};

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
    const bool rot = a.cosb != nullptr && (isq || isk);
    if (live && rot && pos >= a.positions) {
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

// q, k, v: [B, S, heads, D] through strides of elements, the last dimension dense; q and the tables null for a write without
// rotation.  Tokens of one call that share a slot of the cache are written in no order.
extern "C" int gb_paged_put(const void* q, long long qb, long long qs, long long qh, const void* k, long long kb, long long ks,
                            long long kh, const void* v, long long vb, long long vs, long long vh, void* q_out,
                            const float* cosb, const float* sinb, int positions, void* kpool, void* vpool, void* kscale,
                            void* vscale, const int* table, const int* lengths, const int* counts, int B, int S, int Hq,
                            int Hkv, int D, int page, int pages, int per, int dt, int cdt, int* status, cudaStream_t st) {
  if (B <= 0 || S <= 0 || Hkv <= 0 || D <= 0) return 0;
  PutArgs a{{q, qb, qs, qh}, {k, kb, ks, kh}, {v, vb, vs, vh}, q_out, kpool, vpool, (uint8_t*)kscale, (uint8_t*)vscale,
            cosb, sinb, positions, Hq};
  Paged c{table, lengths, counts, status, B, S, Hkv, D, page, pages, per};
  const long long rows = (long long)B * S * (Hq + 2 * Hkv);
  GB_DISPATCH_FLOAT(dt, T, GB_DISPATCH_CACHE(cdt, C, paged_put_any_kernel<T, C><<<gb_grid(rows, 8), 256, 0, st>>>(a, c)));
  return (int)cudaGetLastError();
}

extern "C" int gb_paged_read(const void* kpool, const void* vpool, const void* kscale, const void* vscale, void* kout,
                             void* vout, const int* table, const int* lengths, int B, int L, int Hkv, int D, int page,
                             int pages, int per, int dt, int cdt, int* status, cudaStream_t st) {
  if (B <= 0 || L <= 0 || Hkv <= 0 || D <= 0) return 0;
  Paged c{table, lengths, nullptr, status, B, 0, Hkv, D, page, pages, per};
  const long long total = (long long)B * L * Hkv * D;
  GB_DISPATCH_FLOAT(dt, T, GB_DISPATCH_CACHE(cdt, C, paged_read_any_kernel<T, C><<<gb_grid(total, 256), 256, 0, st>>>(
      kpool, vpool, (const uint8_t*)kscale, (const uint8_t*)vscale, kout, vout, L, c)));
  return (int)cudaGetLastError();
}
