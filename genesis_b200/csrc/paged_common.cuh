// What the kernels over a paged key / value cache share: where a token stands, and e4m3 rows with a power of two each.
//
// K and V are pools [pages, Hkv, page, D]; table [B, per] names the pages of each sequence in order.  lengths[b] counts the
// tokens of sequence b with those of the call, of whose S tokens the first counts[b] are real (all S without counts): token s
// stands at position lengths[b] - counts[b] + s.  A negative position is no token: a slot of the batch that is not in use has
// length 0.  Pages outside the pool and positions behind the table are skipped and recorded in the status word.
#pragma once
#include <cuda_fp8.h>
#include "common.cuh"
#include "sm100_ptx.cuh"

namespace gb {

constexpr int DT_E4M3 = 8;
constexpr int SITE_PAGE = 8, SITE_POSITION = 9;

// n / d for n < 2^31: a division by a number that the host knows is a multiplication
struct Div {
  unsigned mul, shift, d;
  explicit Div(unsigned x = 1) : d(x) {
    shift = 0;
    while (1ull << shift < x) ++shift;
    mul = (unsigned)(((1ull << 32) * ((1ull << shift) - x)) / x + 1);
  }
  __device__ __forceinline__ int by(int n) const { return (int)((__umulhi(mul, (unsigned)n) + (unsigned)n) >> shift); }
};

struct Paged {
  const int* table;
  const int* lengths;
  const int* counts;
  int* status;
  int B, S, Hkv, D;
  int page, pages, per;
  Div in_page;             // by page

  // tokens of sequence b that the table has room for, and how many of this call's S are real
  __device__ __forceinline__ int length(int b) const {
    const int n = lengths[b];
    return n < 0 ? 0 : n;
  }
  __device__ __forceinline__ int count(int b) const {
    const int c = counts != nullptr ? counts[b] : S;
    return c < 0 ? 0 : c > S ? S : c;
  }
  // (the last positions of 2^31 are left out, so that keys can be counted in whole chunks, and one chunk ahead, in 31 bits)
  __device__ __forceinline__ int capacity() const {
    const long long c = (long long)per * page;
    return c > 0x7fffff00 ? 0x7fffff00 : (int)c;
  }
  // row of the pool [pages * Hkv * page] that token `pos` of sequence b has at KV head h; -1 (recorded) where there is none
  __device__ __forceinline__ long long row(int b, int pos, int h) const {
    if (pos >= capacity()) { report_error(status, GB_ERR_BAD_INDEX, SITE_POSITION, pos); return -1; }
    const int i = in_page.by(pos), id = table[(size_t)b * per + i];
    if (id < 0 || id >= pages) { report_error(status, GB_ERR_BAD_INDEX, SITE_PAGE, id); return -1; }
    return ((long long)id * Hkv + h) * page + (pos - i * page);
  }
};

// One layer's pools, as the caller keeps them (`Pools` in genesis_b200/ops/paged.py has the same fields).
struct PagedPools {
  void *k, *v;
  uint8_t *kscale, *vscale;
  int pages, Hkv, page, D, type;
};

// The exponent of a row of e4m3 numbers, from the bits of its largest finite magnitude: the smallest e >= -126 with
// magnitude <= 448 * 2^e (448 = 1.75 * 2^8).  A power of two loses nothing against magnitude / 448 (the format's relative
// step is the same everywhere above its subnormals), makes x * 2^-e exact, so that an element is rounded once, and what the
// row stands for exact in bf16.
__device__ __forceinline__ int e4m3_exponent(uint32_t magnitude_bits) {
  const int e = (int)(magnitude_bits >> 23) - 127 - ((magnitude_bits & 0x7fffffu) > 0x600000u ? 7 : 8);
  return e < -126 ? -126 : e;
}
__device__ __forceinline__ float exp2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }   // -126 <= e <= 127

__device__ __forceinline__ uint32_t finite_bits(float x) {        // |x| as ordered bits, 0 for infinities and NaN
  const uint32_t a = __float_as_uint(x) & 0x7fffffffu;
  return a < 0x7f800000u ? a : 0u;
}
// two numbers as e4m3, rounded to nearest; infinities and NaN as NaN
__device__ __forceinline__ uint32_t to_e4m3x2(float a, float b) {
  uint32_t r = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  if (!(fabsf(a) <= 448.f)) r |= 0x7fu;
  if (!(fabsf(b) <= 448.f)) r |= 0x7f00u;
  return r;
}
__device__ __forceinline__ float2 from_e4m3x2(uint32_t v) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)v, __NV_E4M3);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// four e4m3 numbers as two pairs of fp16
__device__ __forceinline__ void e4m3x4_to_f16(uint32_t v, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
      : "=r"(lo), "=r"(hi) : "r"(v));
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
