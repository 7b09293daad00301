// Attention of a sequence's newest tokens over the pages of its key / value cache, forward only, for sm_100a.
//
//   o[b, s, h] = sum_j p_j v_j,  p = softmax of scale * q . k_j over the j < lengths[b] - counts[b] + s + 1
//
// with K and V of KV head h / (Hq / Hkv), and zeros for a row that sees no key (a token that is none, or scores that are -inf
// throughout).  One pass over the keys with a running maximum and sum in 32 bits.  Tiles of 16 keys are read whole; scores and values
// of keys behind the end are cleared in the last one, so what the rest of a page holds does not matter.
//
// Work is shared out by the lengths on the device, so that a captured launch stays right as sequences grow and a long sequence
// does not leave the GPU to one SM: the chunks of keys of all items (sequence, KV head, tile of query rows) are numbered in
// order, every warp takes an equal run of them, the warps of a CTA join what they have of an item through shared memory, and
// a second small kernel joins the items that CTAs share (parts in a fixed order: the same call gives the same bits).
//   rows     : the query rows of a KV head's group (tokens x heads) are the 8 columns of mma.sync.m16n8k16, 16 keys its rows:
//              S^T = K Q^T, O^T = V^T P^T.  K and V are read once per 8 or 16 rows.
//   layout   : tiles of 16 keys come by TMA into a ring of each warp (no barrier between warps in the loop), the next chunk's K as
//              soon as this one's is read, its V behind it.  Fragments are read 16 bytes at a time: the contraction over d may go in any
//              order that K and Q share, so a lane takes contiguous bytes of its key's row; for V a lane takes contiguous d of four
//              keys and pairs the keys' numbers with byte permutes.  P^T comes from S^T by movmatrix.
//   bound    : the bytes of K and V where sequences are long: 64 x 4096 keys, 32 / 4 heads of 128, bf16: 95 us, 5.65 TB/s (6.1 less the 8
//              that 500 keys take).  In 8 bits 59 us, 4.6 TB/s, where nothing is at its limit (DRAM 49 %, issue slots 54 %): 16 warps an SM
//              with one chunk in flight wait for it, at 128 registers of which some are spilled.  8 us of a call are two launches,
//              finding the share, one round of latencies and the join.
//   other ways that were measured: fragments by plain loads (bf16 93 us, 8 bits 70), by cp.async (109, 70); fetching ahead into L2 with
//              plain loads (99 to 110).
//   precision: P enters its product as two 16-bit numbers (rounded, and what the rounding lost), or rounding it once to the
//              type of V would double the error that the output's rounding makes; with 8-bit V it is fp16, whose 11 bits suffice
//              below a bf16 output.  fp16 P is scaled by 2^7 on top of a maximum that may lag 2^8 behind, so that 2^-31 of the
//              largest probability is still a number.  e4m3 becomes fp16 exactly; a bf16 q does under a power of two for each
//              row.  K's powers of two multiply scores, V's multiply P, relative to the largest seen so far.
//   infinities and NaN among queries, keys and values come out as the definition has them (a key of score -inf weighs nothing, one
//              with any weight gives its infinity): a warp that meets some works its share over once more.
#include "attention_common.cuh"
#include "paged_common.cuh"
#include <type_traits>

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

// The chunks of all items: items[b] = n(b) * per_seq, in the order of b, then KV head and row tile.
struct AttendPlan {
  int per_seq;          // items of a sequence: Hkv * row tiles
  int tiles;            // row tiles
  int grid;             // CTAs launched
  Div seq, tile, group, page;      // by per_seq, tiles, Hq / Hkv, tiles of keys in a page
  float* parts;         // [grid][2][R][D] sums, then [grid][2][R] maxima and normalisers: of an item that comes from the CTA before,
                        // and of one that begins in the CTA and goes on behind it
  float* spill;         // [grid][PA_WARPS][R][D] sums: pieces that a warp leaves behind before it goes on
  int4* spans;          // [grid][2]: that item (-1: none), the first and the last CTA that have it
};

// Keys of a chunk: 4 KB of K and of V, but a tile of 16 at least and two of them at most: with four of 64 numbers in 8 bits, registers are
// spilled (64 x 4096, 14 / 2 heads: 45 us for 28.5), with one of 128 the rounds are short (8 x 4096, 32 / 4 heads: 20.3 us for 18.0; only
// runs of 32768 gain, 57.3 for 58.3).
static constexpr int attend_chunk(int D, int bytes) { return 4096 / (D * bytes) < 16 ? 16 : 4096 / (D * bytes) > 32 ? 32 : 4096 / (D * bytes); }

// CTAs on an SM, by registers: four, three where numbers are split in two or added up apart, two for two operands of rows over 128
// numbers of 8 bits.  (Three instead of four, 32 / 4 heads of 128: 64 x 4096 bf16 98.7 us for 95.2, in 8 bits 60.7 for 59.2; 8 x 4096 25.3
// for 23.0, in 8 bits 20.5 for 18.0; 8 x 32768 in 8 bits 57.3 for 58.3.)  Chunks in flight of a warp, by what shared memory is left; one
// where the spilled registers are many, which need the L1 that a larger ring takes (32 x 4096, drafts of 4: 144 us with two, 93 with one).
// (29 of the 38 kernels spill, 4 to 292 bytes a thread; those of two operands over 16 bits the most.)
static constexpr int attend_ctas(int dt, int cdt, int D, int R) {
  return R == 16 ? (cdt == DT_E4M3 && D == 128 ? 2 : 3) : cdt == DT_F32 || (cdt == DT_E4M3 && dt == DT_F16) ? 3 : 4;
}
static constexpr int attend_stages(int dt, int cdt, int D, int R) {
  return cdt == DT_E4M3 && D == 64 ? 3 : (cdt == DT_F32 && D == 128) || (R == 16 && cdt != DT_E4M3) ? 1 : 5 - attend_ctas(dt, cdt, D, R);
}

template <typename T, int CDT, int D_, int NQ_>
struct PA {
  static constexpr int D = D_, NQ = NQ_, R = 8 * NQ;
  static constexpr bool E8 = CDT == DT_E4M3, BF = CDT == DT_BF16, F32 = CDT == DT_F32;
  static constexpr bool OBF = std::is_same<T, __nv_bfloat16>::value;
  static constexpr int DT = F32 ? DT_F32 : OBF ? DT_BF16 : DT_F16;
  static constexpr bool SPLIT = !(E8 && OBF);           // P in two numbers
  // The tensor cores cut sums off towards zero (2^-24 of them a step on average).  Over thousands of steps that would show in an
  // output of 11 bits and more, so there a chunk's products are added up apart and then to the accumulators, rounded.
  static constexpr bool FRESH = !OBF;
  static constexpr int ES = E8 ? 1 : F32 ? 4 : 2;
  static constexpr int KT = attend_chunk(D, ES);        // keys of a chunk
  static constexpr int NS = KT / 16;                    // tiles of 16 keys
  static constexpr int KL = D * ES / 64;                // 16-byte loads of a lane's share of a key's row
  static constexpr int VW = D * ES / 32;                // words of a lane's share of a value's row
  static constexpr int MT = D / 16;                     // 16-row tiles of O^T
  static constexpr int QS = F32 ? D / 8 : D / 16;       // steps of the contraction over d
  static constexpr int GP = F32 ? 2 : 1;                // ... and of a tile's over its keys
  static constexpr int PIECE = R * D;
  static constexpr int RB = D * ES, BOX = RB < 128 ? RB : 128;      // bytes of a row, and of a column of the ring's boxes
  static constexpr int KB = KT * RB, SB = E8 ? NS * 32 : 0;          // a stage: K, V; powers of two (behind all rings)
  static constexpr int ST = attend_stages(DT, CDT, D, R), RING = ST * 2 * KB;
  static constexpr int SMEM = PA_WARPS * (RING + ST * SB) + 1024;   // (boxes start on 1024 bytes)
  static_assert(PIECE * 4 <= RING, "a warp's last piece takes its ring's place");
  static constexpr int CTAS = attend_ctas(DT, CDT, D, R);
  // first of the two columns d that a lane has of tile mt
  static __device__ __forceinline__ int column(int g, int mt) {
    if (E8) return g * (D / 8) + mt * 2;
    if (F32) return (g + 8 * (mt >> 1)) * 4 + (mt & 1) * 2;
    return (g + 8 * (mt >> 2)) * 8 + (mt & 3) * 2;
  }
  // Row r of an operand of 16 keys is key r ^ 4 where r is odd: then the eight lanes that read shared memory at a time meet eight
  // different 16-byte units of the swizzled boxes (16 rows of 128 bytes, unit u of row r at u ^ r % 8), for K and for V.
  static __device__ __forceinline__ int key_of(int r) { return r ^ ((r & 1) << 2); }
  // where a lane's share of K's row g starts in a tile, and of the first of the four rows whose values it reads (2t, 2t + 1, and 8
  // on; t, t + 4, t + 8, t + 12 for 32 bits); the others follow by constants
  static __device__ __forceinline__ int k_unit(int g, int t) {
    const int key = key_of(g);
    return RB == 64 ? key * 64 + ((t ^ (key >> 1 & 3)) << 4) : key * 128 + ((t ^ key) << 4);
  }
  static __device__ __forceinline__ int first_key(int t) { return F32 ? key_of(t) : 2 * t; }
  static __device__ __forceinline__ int v_unit(int g, int t) {
    const int key = first_key(t);
    return RB == 64 ? key * 64 + (((g >> 1) ^ (key >> 1 & 3)) << 4) + (g & 1) * 8 : key * 128 + ((g ^ key) << 4);
  }
  static constexpr int ODD_KEY = F32 ? 4 : 5;           // the second row's key is the first's ^ this: 4, or (2t + 1) ^ 4
  static constexpr int ODD_UNIT = RB == 64 ? 5 * 64 ^ 2 << 4 : ODD_KEY * 128 ^ ODD_KEY << 4;
};

// 16 bytes to shared memory by a bulk copy
__device__ __forceinline__ void bulk_copy_16(uint32_t dst, const void* src, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], 16, [%2];" ::"r"(dst), "l"(src), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ uint32_t transposed_8x8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
template <bool BF>
__device__ __forceinline__ float2 unpack2(uint32_t v) {
  if (BF) return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&v));
}
template <bool BF>
__device__ __forceinline__ void mma_k16(float (&c)[4], const uint32_t a0, const uint32_t a1, const uint32_t a2, const uint32_t a3, uint32_t b0, uint32_t b1) {
  if (BF)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
  asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
// 32 bits as two numbers of 11 bits: what is cut off, rounded (2^-22 at most is lost); nothing of an infinity or NaN
template <int N>
__device__ __forceinline__ void split_tf32(const uint32_t (&x)[N], uint32_t (&hi)[N], uint32_t (&lo)[N]) {
#pragma unroll
  for (int k = 0; k < N; ++k) {
    hi[k] = x[k] & 0xffffe000u;
    lo[k] = (x[k] & 0x7f800000u) == 0x7f800000u ? 0u : (__float_as_uint(__uint_as_float(x[k]) - __uint_as_float(hi[k])) + 0x1000u) & 0xffffe000u;
  }
}
// hi + lo += a b in 32 bits: the three larger of four products, the small ones in a sum of their own
__device__ __forceinline__ void mma_f32(float (&hi)[4], float (&lo)[4], const uint32_t (&a)[4], const uint32_t (&bh)[2], const uint32_t (&bl)[2]) {
  uint32_t ah[4], al[4];
  split_tf32(a, ah, al);
  mma_tf32(lo, al, bh);
  mma_tf32(lo, ah, bl);
  mma_tf32(hi, ah, bh);
}
// O^T += V^T P^T of a step: P as high and low part
template <class C>
__device__ __forceinline__ void mma_pv(float (&acc)[4], const uint32_t (&v)[4], const uint32_t (&hi)[2], const uint32_t (&lo)[2]) {
  if constexpr (C::F32) {
    mma_f32(acc, acc, v, hi, lo);
  } else {
    mma_k16<C::BF>(acc, v[0], v[1], v[2], v[3], hi[0], hi[1]);
    if constexpr (C::SPLIT) mma_k16<C::BF>(acc, v[0], v[1], v[2], v[3], lo[0], lo[1]);
  }
}
// Bits of a word of V that are infinities or NaN, as a mask.
template <class C>
__device__ __forceinline__ uint32_t not_finite(uint32_t w) {
  if constexpr (C::F32) return (w & 0x7f800000u) == 0x7f800000u ? 0xffffffffu : 0u;
  else if constexpr (C::E8) return __vcmpeq4(w & 0x7f7f7f7fu, 0x7f7f7f7fu);
  else return __vcmpeq2(w & (C::BF ? 0x7f807f80u : 0x7c007c00u), C::BF ? 0x7f807f80u : 0x7c007c00u);
}
__device__ __forceinline__ float pow2_of(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// weight of a part whose maximum is m against the common maximum
__device__ __forceinline__ float part_weight(float m, float common) { return m == -INFINITY ? 0.f : pow2_of(m - common); }

// keys that are read of sequence b (none where the call has no token of it), and chunks of KT of them, at least one: an item
// without keys writes zeros
__device__ __forceinline__ int attend_keys(const Paged& c, int b) {
  if (c.count(b) == 0) return 0;
  const int n = c.length(b), cap = c.capacity();
  return n < cap ? n : cap;
}
__device__ __forceinline__ int attend_chunks(int keys, int kt) { return keys == 0 ? 1 : (keys + kt - 1) / kt; }

// o / l of row r (0 .. S * group - 1) of a group, 4 columns from d on
template <typename T>
__device__ __forceinline__ void store_row4(const AttendArgs& a, const Paged& c, const Div& group, int b, int kvh, int r, int d, float4 o, float l) {
  const int s = group.by(r);
  if (l == 0.f) o = make_float4(0.f, 0.f, 0.f, 0.f);       // (scores of -inf throughout, whatever the values hold)
  const float inv = l == 0.f ? 0.f : 1.f / l;
  T* p = reinterpret_cast<T*>(a.o) + (((long long)b * c.S + s) * a.Hq + kvh * group.d + r - s * group.d) * c.D + d;
  if constexpr (std::is_same<T, float>::value) {
    *reinterpret_cast<float4*>(p) = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
  } else {
    constexpr bool BF = std::is_same<T, __nv_bfloat16>::value;
    *reinterpret_cast<uint2*>(p) = make_uint2(pack2c<BF>(o.x * inv, o.y * inv), pack2c<BF>(o.z * inv, o.w * inv));
  }
}

// A warp's share once more, number by number in 32 bits: where keys, values or queries are infinite, what the loop over the
// tensor cores has made of them is put right, in a run's sums (the last in the ring, others in `spill`, maxima and normalisers
// at m and l) or in the output.  Only rows and columns that are not finite, or were not to be, are replaced.  A row whose scores are
// NaN stays so, and is not followed to its end.  About two microseconds a key of the share, which only such numbers pay for (an infinity
// among the values, 64 x 4096, 32 / 4 heads of 128, bf16: 0.9 ms for 0.1); that the code is there costs others 0 to 0.3 us a call.
template <typename T, int CDT, int D, int R, int KT>
__device__ __noinline__ void redo_share(const AttendArgs& a, const Paged& c, const AttendPlan& plan, unsigned u, unsigned u_end, float* ring,
                                        float* spill, float* m, float* l) {
  constexpr int N = D / 32, G = 8;     // columns of a lane, rows at a time
  const int lane = threadIdx.x & 31, rows = c.S * (int)plan.group.d;
  const float sl2 = a.scale * 1.4426950408889634f;
  int b = 0, slot = 0;
  unsigned seq_start = 0;
  auto load = [](const void* pool, long long at) {
    if constexpr (CDT == DT_E4M3) return from_e4m3x2(reinterpret_cast<const uint8_t*>(pool)[at]).x;
    else return load_as_float(pool, CDT, at);
  };
  auto finite = [](float x) { return fabsf(x) < INFINITY; };
  while (u < u_end) {
    const int keys = attend_keys(c, b), n = attend_chunks(keys, KT);
    if (u - seq_start >= (unsigned)n * plan.per_seq) {
      seq_start += (unsigned)n * plan.per_seq;
      if (++b >= c.B) break;
      continue;
    }
    const int idx = (int)((u - seq_start) / (unsigned)n);
    const int c0 = (int)(u - seq_start - (unsigned)idx * n), c1 = min(n, c0 + (int)(u_end - u));
    const int kvh = plan.tile.by(idx), row0 = (idx - kvh * plan.tiles) * R, cnt = c.count(b), len = c.length(b);
    const bool whole = c0 == 0 && c1 == n;
    float* const sums = u + (c1 - c0) == u_end ? ring : spill;
    auto line = [&](int r) {           // of row r in q and o
      const int s = plan.group.by(r);
      return (((long long)b * c.S + s) * a.Hq + kvh * plan.group.d + r - s * plan.group.d) * D;
    };
    for (int r0 = 0; r0 < R && row0 + r0 < rows; r0 += G) {
      float q[G][N], o[G][N], rm[G], rl[G];
      int end[G], last = 0;
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const int r = row0 + r0 + g, s = plan.group.by(r);
        end[g] = r < rows && s < cnt ? min(min(c1 * KT, keys), len - cnt + s + 1) : 0;
        last = max(last, end[g]);
        rm[g] = -INFINITY;
        rl[g] = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          q[g][i] = end[g] > 0 ? Cvt<T>::to_f(reinterpret_cast<const T*>(a.q)[line(r) + i * 32 + lane]) : 0.f;
          o[g][i] = 0.f;
        }
      }
      for (int key = c0 * KT; key < last; ++key) {
        const int i = c.in_page.by(key), page = c.table[(size_t)b * c.per + i];
        if ((unsigned)page >= (unsigned)c.pages) continue;
        const long long row = ((long long)page * c.Hkv + kvh) * c.page + key - i * c.page;
        float k[N], v[N], ks = sl2;
#pragma unroll
        for (int j = 0; j < N; ++j) {
          k[j] = load(a.kpool, row * D + j * 32 + lane);
          v[j] = load(a.vpool, row * D + j * 32 + lane);
        }
        if constexpr (CDT == DT_E4M3) {
          ks *= __uint_as_float((uint32_t)a.kscale[row] << 23);
#pragma unroll
          for (int j = 0; j < N; ++j) v[j] *= __uint_as_float((uint32_t)a.vscale[row] << 23);
        }
        bool on = false;
#pragma unroll
        for (int g = 0; g < G; ++g) {
          if (key >= end[g]) continue;
          float x = 0.f;
#pragma unroll
          for (int j = 0; j < N; ++j) x = fmaf(q[g][j], k[j], x);
          x = warp_sum(x) * ks;
          const float mn = fmaxf(rm[g], x), base = mn == -INFINITY ? 0.f : mn, w = part_weight(rm[g], base), p = pow2_of(x - base);
          rm[g] = mn;
          rl[g] = rl[g] * w + p;
#pragma unroll
          for (int j = 0; j < N; ++j) o[g][j] = o[g][j] * w + p * v[j];
          on |= rl[g] == rl[g];
        }
        if (!on) break;                // (NaN in all rows that see this key; the others have ended)
      }
#pragma unroll
      for (int g = 0; g < G; ++g) {
        if (end[g] <= 0) continue;
        const int r = r0 + g;
        if (whole) {
          T* out = reinterpret_cast<T*>(a.o) + line(row0 + r);
#pragma unroll
          for (int j = 0; j < N; ++j) {
            const float x = rl[g] == 0.f ? 0.f : o[g][j] / rl[g];
            if (!finite(x) || !finite(Cvt<T>::to_f(out[j * 32 + lane]))) out[j * 32 + lane] = Cvt<T>::from_f(x);
          }
        } else {
          float &pm = m[slot * R + r], &pl = l[slot * R + r];
          const bool all = !finite(pl);
          const float unit = all ? 1.f : pow2_of(rm[g] - pm);
          __syncwarp();                // (all have read them)
#pragma unroll
          for (int j = 0; j < N; ++j) {
            float& x = sums[r * D + j * 32 + lane];
            if (all || !finite(o[g][j]) || !finite(x)) x = o[g][j] * unit;
          }
          if (all && lane == 0) { pm = rm[g]; pl = rl[g]; }
        }
      }
    }
    slot += !whole;
    u += c1 - c0;
  }
}

// MULTI: several tokens a sequence, whose rows end at different keys
template <typename T, int CDT, int D, int NQ, bool MULTI>
__global__ void __launch_bounds__(PA_WARPS * 32, PA<T, CDT, D, NQ>::CTAS)
paged_attend_kernel(const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv, const __grid_constant__ AttendArgs a,
                    const __grid_constant__ Paged c, const __grid_constant__ AttendPlan plan) {
  using C = PA<T, CDT, D, NQ>;
  constexpr int R = C::R, KT = C::KT, NS = C::NS, KL = C::KL, VW = C::VW, MT = C::MT, QS = C::QS, GP = C::GP, W = PA_WARPS;
  extern __shared__ __align__(1024) uint8_t shared[];              // [W][RING], [W][ST][SB]
  __shared__ uint64_t landed[W][2][C::ST];                         // K's and V's copies of a stage have landed
  __shared__ int abort_word[W];
  uint8_t* const rings = shared + (1024 - (smem_u32(shared) & 1023)) % 1024;
  __shared__ const float* piece_at[2 * W];                         // [R][D] sums: in the ring of the warp, or in the workspace
  __shared__ float piece_m[2 * W][R], piece_l[2 * W][R];
  __shared__ int piece_item[2 * W], piece_flags[2 * W];
  __shared__ unsigned piece_start[2 * W], piece_end[2 * W];
  __shared__ int again[W];             // a run of the warp has to be worked over once more
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");       // (the join waits for the end of this kernel)

  // ---- the share of this warp: every warp finds it by itself ----------------------------------------------------------------
  if (lane < 2) piece_item[2 * warp + lane] = -1;
  if (lane == 0) {
    abort_word[warp] = again[warp] = 0;
    for (int i = 0; i < C::ST * 2; ++i) mbar_init(&landed[warp][0][0] + i, 1);
    mbar_fence_init();
    tma_prefetch_desc(&tmk);
    tma_prefetch_desc(&tmv);
  }
  __syncwarp();
  const int each = (c.B + 31) / 32, b0 = min(c.B, lane * each), b1 = min(c.B, b0 + each);
  unsigned mine = 0;                   // (the host has seen to it that all chunks are less than 2^31)
  for (int b = b0; b < b1; ++b) mine += attend_chunks(attend_keys(c, b), KT);
  mine *= plan.per_seq;
  unsigned upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned x = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += x;
  }
  const unsigned total = __shfl_sync(0xffffffffu, upto, 31);
  // the first `rest` warps have a chunk more than the others
  const int cta = blockIdx.x, ctas = min((unsigned)plan.grid, (total + W - 1) / W);
  const unsigned workers = ctas * W, share = total / workers, rest = total - share * workers;
  auto start_of = [&](unsigned worker) { return share * worker + min(worker, rest); };
  auto cta_of = [&](unsigned chunk) {
    const unsigned more = rest * (share + 1);
    return (int)((chunk < more ? chunk / (share + 1) : rest + (chunk - more) / share) / W);
  };
  if (cta >= ctas) {
    if (threadIdx.x < 2) plan.spans[2 * cta + threadIdx.x] = make_int4(-1, 0, 0, 0);
    return;
  }
  unsigned u = start_of(cta * W + warp);
  const unsigned u_end = start_of(cta * W + warp + 1);
  // the sequence that it begins in (a warp without a share finds one too, or sequence 0)
  const int owner = max(0, __ffs(__ballot_sync(0xffffffffu, u < upto)) - 1);
  int b = owner * each;
  unsigned seq_start = __shfl_sync(0xffffffffu, upto - mine, owner);
  int slot = 0;
  const int k_at = C::k_unit(g, t), v_at = C::v_unit(g, t), gk = C::key_of(g);
  volatile int* const abort_flag = &abort_word[warp];
  uint8_t* const ring = rings + warp * C::RING;
  uint8_t* const powers = rings + W * C::RING + warp * C::ST * C::SB;
  int put = 0, use = 0, use_phase = 0;                             // stage of the next chunk that is copied and of the one that is worked on
  unsigned k_copies = 0, v_copies = 0;                             // so far
  const float sl2 = a.scale * 1.4426950408889634f;
  const int rows = c.S * plan.group.d;

  while (u < u_end) {
    // ---- an item's run of chunks ------------------------------------------------------------------------------------
    const int keys = attend_keys(c, b), n = attend_chunks(keys, KT);
    if (u - seq_start >= (unsigned)n * plan.per_seq) {
      seq_start += (unsigned)n * plan.per_seq;
      if (++b >= c.B) break;           // (lengths that change under the kernel's hands give wrong sums, and nothing worse)
      continue;
    }
    const int idx = plan.per_seq == 1 ? 0 : (int)((u - seq_start) / (unsigned)n);
    const int c0 = (int)(u - seq_start - (unsigned)idx * n);
    const int c1 = min(n, c0 + (int)(u_end - u));
    const int kvh = plan.tile.by(idx), row0 = (idx - kvh * plan.tiles) * R;
    const int cnt = c.count(b), len = c.length(b);
    if (len > keys && cnt > 0 && c0 == 0 && lane == 0) report_error(c.status, GB_ERR_BAD_INDEX, SITE_POSITION, len - 1);

    // ---- copies -----------------------------------------------------------------------------------------------------
    const int* pages = c.table + (size_t)b * c.per;
    const int tpp = plan.page.d;
    int tile = c0 * NS, pg = plan.page.by(tile), sub = tile - pg * tpp;    // the next tile whose page is asked for
    int id[NS], place[NS];
    auto ask = [&]() {
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        place[i] = -1;
        if (tile * 16 < keys) { id[i] = pages[pg]; place[i] = sub * 16; }
        ++tile;
        if (++sub == tpp) { sub = 0; ++pg; }
      }
    };
    ask();
    // queries as the B operand: row g, the d that this lane has of a key's row
    uint32_t qf[NQ][QS][2];
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
      const int r = row0 + q * 8 + g, s = plan.group.by(r);
      const T* p = reinterpret_cast<const T*>(a.q) + (((long long)b * c.S + s) * a.Hq + kvh * plan.group.d + r - s * plan.group.d) * D;
      constexpr int H = C::E8 ? 2 : 1, E = 16 / sizeof(T);     // 16-byte loads that go with one of a key's row, numbers of each
#pragma unroll
      for (int i = 0; i < KL * H; ++i) {
        uint4 v = make_uint4(0, 0, 0, 0);
        if (r < rows) v = __ldg(reinterpret_cast<const uint4*>(p + ((i / H) * 4 + t) * E * H + (i % H) * E));
        qf[q][2 * i][0] = v.x; qf[q][2 * i][1] = v.y;
        qf[q][2 * i + 1][0] = v.z; qf[q][2 * i + 1][1] = v.w;
      }
    }
    long long row[NS];                 // of the pool, of the chunk that is copied; -1: no such tile
    float factor[NQ][2];               // of the scores of queries 2t, 2t + 1
    int end[NQ][2];                    // keys that they see (without MULTI: all, or it is no row)
    // running maximum m (may lag 2^8 behind), what the exponents are taken off by, normaliser: of this lane's keys
    float o[NQ][MT][4], m[NQ][2], off[NQ][2], l[NQ][2];
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[q][i][e] = 0.f;
#pragma unroll
      for (int e = 0; e < 2; ++e) { m[q][e] = -INFINITY; off[q][e] = 0.f; l[q][e] = 0.f; }
    }
    constexpr float LIFT = !C::E8 && !C::BF && !C::F32 ? 7.f : 0.f;      // fp16 P without a scale of its own
    int vtop = -1000;                  // the power of two of V that the accumulators are relative to, as stored
    bool left_out = false;             // values of keys that not all tokens see
    const int full = MULTI ? min(keys, max(0, len - cnt + 1)) : keys;      // keys that every token sees

    // one round: scores of chunk ch, then K of chunk ch + ST into its place; probabilities and products of ch, then V of ch + ST.
    uint32_t gone_later = 0;           // tiles that are not there, of the chunks in flight
    for (int ch = c0 - C::ST; ch < c1; ++ch) {
      const bool now = ch >= c0, more = ch + C::ST < c1;
      uint8_t* const sk = ring + use * 2 * C::KB;
      // ---- S^T = K Q^T ----------------------------------------------------------------------------------------------
      float s[NS][NQ][4];
      float ks[NS][2];
      int ve[NS][2];
      const uint32_t gone = gone_later & ((1u << NS) - 1);
      gone_later >>= NS;
      if (ch == c0) {
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
          float fq = 1.f;
          if constexpr (C::E8 && C::OBF) {   // bf16 -> fp16 with the row's largest in [2^14, 2^15)
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const float2 x = unpack2<true>(qf[q][i][h]);
                top = max(top, max(finite_bits(x.x), finite_bits(x.y)));
              }
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
            int e = (int)(top >> 23) - 127 - 14;
            e = e < -100 ? -100 : e;
            const float inv = exp2i(-e);
            fq = exp2i(e);
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const float2 x = unpack2<true>(qf[q][i][h]);
                qf[q][i][h] = pack2c<false>(x.x * inv, x.y * inv);
              }
          }
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            factor[q][e] = sl2 * __shfl_sync(0xffffffffu, fq, (2 * t + e) * 4);
            if constexpr (MULTI) {
              const int rr = row0 + q * 8 + 2 * t + e, s = plan.group.by(rr);
              end[q][e] = rr < rows && s < cnt ? min(keys, max(0, len - cnt + s + 1)) : 0;
            } else {
              end[q][e] = keys;
            }
          }
        }
      }
      if (now) {
        if (!__all_sync(0xffffffffu, mbar_wait(&landed[warp][0][use], use_phase, abort_flag, c.status, 81))) break;
#pragma unroll
        for (int i = 0; i < NS; ++i) {
          float small[NQ][4] = {};
#pragma unroll
          for (int q = 0; q < NQ; ++q)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[i][q][e] = 0.f;
#pragma unroll
          for (int j = 0; j < KL; ++j) {
            const uint8_t* x = sk + i * 16 * C::RB + (j >> 1) * 2048 + (k_at ^ (j & 1) * 64);
            const uint4 klo = *reinterpret_cast<const uint4*>(x), khi = *reinterpret_cast<const uint4*>(x + 8 * C::BOX);
            const uint32_t lo[4] = {klo.x, klo.y, klo.z, klo.w}, hi[4] = {khi.x, khi.y, khi.z, khi.w};
            if constexpr (C::F32) {
#pragma unroll
              for (int q = 0; q < NQ; ++q) {
                float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                  const uint32_t x[4] = {lo[2 * h], hi[2 * h], lo[2 * h + 1], hi[2 * h + 1]};
                  uint32_t bh[2], bl[2];
                  split_tf32(qf[q][2 * j + h], bh, bl);
                  mma_f32(sum, small[q], x, bh, bl);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) s[i][q][e] += sum[e];
              }
            } else if constexpr (!C::E8) {
#pragma unroll
              for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int q = 0; q < NQ; ++q)
                  mma_k16<C::BF>(s[i][q], lo[2 * h], hi[2 * h], lo[2 * h + 1], hi[2 * h + 1], qf[q][2 * j + h][0], qf[q][2 * j + h][1]);
            } else {
#pragma unroll
              for (int h = 0; h < 4; ++h) {
                uint32_t a0, a1, a2, a3;
                e4m3x4_to_f16(lo[h], a0, a2);
                e4m3x4_to_f16(hi[h], a1, a3);
#pragma unroll
                for (int q = 0; q < NQ; ++q) mma_k16<false>(s[i][q], a0, a1, a2, a3, qf[q][4 * j + h][0], qf[q][4 * j + h][1]);
              }
            }
          }
          if constexpr (C::F32) {
#pragma unroll
            for (int q = 0; q < NQ; ++q)
#pragma unroll
              for (int e = 0; e < 4; ++e) s[i][q][e] += small[q][e];
          }
          if constexpr (C::E8) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint8_t* e = powers + use * C::SB + i * 32 + gk + 8 * h;
              ks[i][h] = __uint_as_float((uint32_t)e[0] << 23);
              ve[i][h] = e[16];
            }
          }
        }
      }
      __syncwarp();                    // all have read
      if (more) {
        uint64_t* const bar = &landed[warp][0][put];
        uint8_t* const dk = ring + put * 2 * C::KB;
        int tiles = 0;
#pragma unroll
        for (int i = 0; i < NS; ++i) {
          row[i] = -1;
          if (place[i] >= 0) {
            if ((unsigned)id[i] >= (unsigned)c.pages) { if (lane == 0) report_error(c.status, GB_ERR_BAD_INDEX, SITE_PAGE, id[i]); }
            else row[i] = ((long long)id[i] * c.Hkv + kvh) * c.page + place[i];
          }
          if (row[i] < 0) gone_later |= 1u << (NS * (C::ST - 1) + i);
          else ++tiles;
        }
        if (lane == 0) {
          mbar_expect_tx(bar, tiles * (16 * C::RB + (C::E8 ? 32 : 0)));
#pragma unroll
          for (int i = 0; i < NS; ++i) {
            if (row[i] < 0) continue;
#pragma unroll
            for (int x = 0; x < C::RB / C::BOX; ++x) tma_load_2d(dk + i * 16 * C::RB + x * 2048, &tmk, bar, x * (C::BOX / C::ES), (int)row[i]);
            if constexpr (C::E8) {
              bulk_copy_16(smem_u32(powers) + put * C::SB + i * 32, a.kscale + row[i], bar);
              bulk_copy_16(smem_u32(powers) + put * C::SB + i * 32 + 16, a.vscale + row[i], bar);
            }
          }
        }
        ++k_copies;
        ask();
      }
      if (now) {
        // ---- probabilities ------------------------------------------------------------------------------------------
        const bool tail = gone != 0 || (ch + 1) * KT > full;
#pragma unroll
        for (int i = 0; i < NS; ++i)
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int q = 0; q < NQ; ++q)
#pragma unroll
              for (int e = 0; e < 2; ++e) s[i][q][2 * h + e] *= C::E8 ? factor[q][e] * ks[i][h] : factor[q][e];
        if (tail) {
#pragma unroll
          for (int i = 0; i < NS; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int key = gone >> i & 1 ? 0x7fffffff : (ch * NS + i) * 16 + gk + 8 * h;
              if (C::E8 && key >= keys) ve[i][h] = 0;
#pragma unroll
              for (int q = 0; q < NQ; ++q)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                  if (key >= end[q][e]) s[i][q][2 * h + e] = -INFINITY;
            }
        }
        float top[NQ][2];
        bool grow = false;
#pragma unroll
        for (int q = 0; q < NQ; ++q)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            top[q][e] = fmaxf(s[0][q][e], s[0][q][2 + e]);
#pragma unroll
            for (int i = 1; i < NS; ++i) top[q][e] = fmaxf(top[q][e], fmaxf(s[i][q][e], s[i][q][2 + e]));
            grow |= top[q][e] > m[q][e] + 8.f;
          }
        int power = 0;                 // V's largest power of two here, as stored
        if constexpr (C::E8) {
#pragma unroll
          for (int i = 0; i < NS; ++i) power = max(power, max(ve[i][0], ve[i][1]));
          grow |= power > vtop;
        }
        if (__any_sync(0xffffffffu, grow)) {
          float vscale = 1.f;
          if constexpr (C::E8) {
            const int e = __reduce_max_sync(0xffffffffu, max(power, vtop));
            vscale = vtop - e < -126 ? 0.f : exp2i(vtop - e);
            vtop = e;
          }
#pragma unroll
          for (int q = 0; q < NQ; ++q)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float x = fmaxf(m[q][e], top[q][e]);
#pragma unroll
              for (int w = 4; w < 32; w <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, w));
              const float alpha = part_weight(m[q][e], x);
              m[q][e] = x;
              off[q][e] = x == -INFINITY ? 0.f : x - LIFT;
              l[q][e] *= alpha;
#pragma unroll
              for (int i = 0; i < MT; ++i) {
                o[q][i][e] *= alpha * vscale;
                o[q][i][2 + e] *= alpha * vscale;
              }
            }
        }
        uint32_t ph[NS][NQ][GP][2], pl[NS][NQ][GP][2];
        // 32-bit numbers of keys g (lane's row) and queries 2t, 2t + 1 as the operand of 8 keys: keys t and t + 4 of query g
        auto turned = [&](float x, float y, uint32_t (&out)[2]) {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const float p = __shfl_sync(0xffffffffu, x, (t + 4 * k) * 4 + (g >> 1)), q = __shfl_sync(0xffffffffu, y, (t + 4 * k) * 4 + (g >> 1));
            out[k] = __float_as_uint(g & 1 ? q : p);
          }
        };
#pragma unroll
        for (int i = 0; i < NS; ++i)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float vs = C::E8 ? __uint_as_float((uint32_t)max(ve[i][h] - vtop + 134, 1) << 23) : 1.f;
#pragma unroll
            for (int q = 0; q < NQ; ++q) {
              float p[2];
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                p[e] = pow2_of(s[i][q][2 * h + e] - off[q][e]);
                l[q][e] += p[e];
                if constexpr (C::E8) p[e] *= vs;
              }
              if constexpr (C::F32) {
                uint32_t x[2];
                turned(p[0], p[1], x);
                split_tf32(x, ph[i][q][h % GP], pl[i][q][h % GP]);
              } else {
                const uint32_t w = pack2c<C::BF>(p[0], p[1]);
                ph[i][q][0][h] = transposed_8x8(w);
                if constexpr (C::SPLIT) {
                  const float2 r = unpack2<C::BF>(w);
                  pl[i][q][0][h] = transposed_8x8(pack2c<C::BF>(p[0] - r.x, p[1] - r.y));
                }
              }
            }
          }
        // ---- O^T += V^T P^T -----------------------------------------------------------------------------------------
        constexpr int TW = C::E8 ? 2 : 1;              // tiles of O^T that a word of V has numbers of
        alignas(16) uint32_t vr[NS][4][4];
        uint32_t bad = 0;
        if (!__all_sync(0xffffffffu, mbar_wait(&landed[warp][1][use], use_phase, abort_flag, c.status, 82))) break;
#pragma unroll
        for (int j = 0; j < VW; j += C::F32 ? 2 : 1) {
          constexpr int VN = VW == 2 ? 2 : 4;         // words that a lane has of a key side by side
          if (j % VN == 0) {
#pragma unroll
            for (int i = 0; i < NS; ++i)
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const uint8_t* x = sk + C::KB + i * 16 * C::RB + j / VN * 2048 + (k >> 1) * 8 * C::BOX + (k & 1 ? v_at ^ C::ODD_UNIT : v_at);
                if constexpr (VN == 2) *reinterpret_cast<uint2*>(vr[i][k]) = *reinterpret_cast<const uint2*>(x);
                else *reinterpret_cast<uint4*>(vr[i][k]) = *reinterpret_cast<const uint4*>(x);
              }
            // What stands behind the end of a sequence or in a tile that is not there is none of it.  With several tokens, a key that
            // one row sees and another does not is multiplied by a probability of 0 there, which an infinity or NaN among its values
            // would turn into NaN: those are left out here, and the rows that see them get them in the end.
            if (tail) {
#pragma unroll
              for (int i = 0; i < NS; ++i)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                  const int key = (ch * NS + i) * 16 + (k >> 1) * 8 + (k & 1 ? C::first_key(t) ^ C::ODD_KEY : C::first_key(t));
                  const bool there = !(gone >> i & 1) && key < keys;
#pragma unroll
                  for (int w = 0; w < VN; ++w) {
                    if (!there) vr[i][k][w] = 0;
                    if constexpr (MULTI) {
                      const uint32_t f = not_finite<C>(vr[i][k][w]);
                      bad |= f;
                      vr[i][k][w] &= ~f;
                    }
                  }
                }
            }
          }
          float sum[TW][NQ][4] = {};
#pragma unroll
          for (int i = 0; i < NS; ++i) {
            uint32_t v[TW * GP][4];
            const int w = j % VN;
            if constexpr (C::F32) {
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                v[k][0] = vr[i][2 * k][w]; v[k][1] = vr[i][2 * k][w + 1];
                v[k][2] = vr[i][2 * k + 1][w]; v[k][3] = vr[i][2 * k + 1][w + 1];
              }
            } else if constexpr (!C::E8) {
              v[0][0] = __byte_perm(vr[i][0][w], vr[i][1][w], 0x5410);
              v[0][1] = __byte_perm(vr[i][0][w], vr[i][1][w], 0x7632);
              v[0][2] = __byte_perm(vr[i][2][w], vr[i][3][w], 0x5410);
              v[0][3] = __byte_perm(vr[i][2][w], vr[i][3][w], 0x7632);
            } else {
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                e4m3x4_to_f16(__byte_perm(vr[i][0][w], vr[i][1][w], h ? 0x7362 : 0x5140), v[h][0], v[h][1]);
                e4m3x4_to_f16(__byte_perm(vr[i][2][w], vr[i][3][w], h ? 0x7362 : 0x5140), v[h][2], v[h][3]);
              }
            }
#pragma unroll
            for (int h = 0; h < TW; ++h)
#pragma unroll
              for (int q = 0; q < NQ; ++q)
#pragma unroll
                for (int gp = 0; gp < GP; ++gp) {
                  if constexpr (C::FRESH) mma_pv<C>(sum[h][q], v[h + gp], ph[i][q][gp], pl[i][q][gp]);
                  else mma_pv<C>(o[q][j * TW + h], v[h], ph[i][q][gp], pl[i][q][gp]);
                }
          }
          if constexpr (C::FRESH) {
#pragma unroll
            for (int h = 0; h < TW; ++h)
#pragma unroll
              for (int q = 0; q < NQ; ++q)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[q][C::F32 ? j / 2 : j * TW + h][e] += sum[h][q][e];
          }
        }
        if constexpr (MULTI) {
          left_out |= bad != 0;
        }
      }
      __syncwarp();
      if (more) {
        if (lane == 0) {
          uint64_t* const bar = &landed[warp][1][put];
          uint8_t* const dv = ring + put * 2 * C::KB + C::KB;
          int tiles = 0;
#pragma unroll
          for (int i = 0; i < NS; ++i) tiles += row[i] >= 0;
          mbar_expect_tx(bar, tiles * 16 * C::RB);
#pragma unroll
          for (int i = 0; i < NS; ++i) {
            if (row[i] < 0) continue;
#pragma unroll
            for (int x = 0; x < C::RB / C::BOX; ++x) tma_load_2d(dv + i * 16 * C::RB + x * 2048, &tmv, bar, x * (C::BOX / C::ES), (int)row[i]);
          }
        }
        ++v_copies;
        if (++put == C::ST) put = 0;
      }
      if (now && ++use == C::ST) { use = 0; use_phase ^= 1; }
    }
    if (__any_sync(0xffffffffu, *abort_flag)) {      // gave up: the copies in flight land first, and nothing is kept
      drain_copies(&landed[warp][0][0], C::ST, k_copies);
      drain_copies(&landed[warp][1][0], C::ST, v_copies);
      __syncwarp();
      break;
    }

    // ---- the run's result ---------------------------------------------------------------------------------------------
    const float unit = !C::E8 ? 1.f : vtop >= 8 ? exp2i(vtop - 134) : vtop > 0 ? __uint_as_float(1u << (vtop + 15)) : 0.f;
    if constexpr (MULTI) {             // rows that are no tokens (chunks that all tokens see are not masked)
#pragma unroll
      for (int q = 0; q < NQ; ++q)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          if (end[q][e] == 0) {
            m[q][e] = -INFINITY;
            l[q][e] = 0.f;
#pragma unroll
            for (int i = 0; i < MT; ++i) o[q][i][e] = o[q][i][2 + e] = 0.f;
          }
    }
#pragma unroll
    for (int q = 0; q < NQ; ++q)
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int w = 4; w < 32; w <<= 1) l[q][e] += __shfl_xor_sync(0xffffffffu, l[q][e], w);
    const bool whole = c0 == 0 && c1 == n;
    const int piece = 2 * warp + slot;
    // a piece that ends the warp's share stays in its ring's place; one that others follow goes to the workspace
    __syncwarp();
    float* const sums = u + (c1 - c0) == u_end ? reinterpret_cast<float*>(ring) : plan.spill + ((size_t)cta * W + warp) * C::PIECE;
    if (!whole) {
      ++slot;
      if (lane == 0) {
        piece_at[piece] = sums;
        piece_item[piece] = b * plan.per_seq + idx;
        piece_flags[piece] = (c0 == 0 ? 1 : 0) | (c1 == n ? 2 : 0);
        piece_start[piece] = seq_start + (unsigned)idx * n;
        piece_end[piece] = seq_start + (unsigned)(idx + 1) * n;
      }
    }
#pragma unroll
    for (int q = 0; q < NQ; ++q)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = q * 8 + 2 * t + e;
        if (!whole && g == 0) { piece_m[piece][r] = m[q][e] - LIFT; piece_l[piece][r] = l[q][e]; }
#pragma unroll
        for (int i = 0; i < MT; i += 2) {
          const float4 v = make_float4(o[q][i][e] * unit, o[q][i][2 + e] * unit, o[q][i + 1][e] * unit, o[q][i + 1][2 + e] * unit);
          const int d = C::column(g, i);
          if (!whole) *reinterpret_cast<float4*>(sums + r * D + d) = v;
          else if (row0 + r < rows) store_row4<T>(a, c, plan.group, b, kvh, row0 + r, d, v, l[q][e]);
        }
      }
    // What is not finite may have met a part of 0 or of the other sign where P, or a number of 32 bits, is split in two.
    if constexpr (MULTI || !C::E8) {
      bool odd = left_out;
      if constexpr (!C::E8) {
#pragma unroll
        for (int q = 0; q < NQ; ++q)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float probe = 0.f;
#pragma unroll
            for (int i = 0; i < MT; ++i) probe = fmaf(o[q][i][2 + e], 0.f, fmaf(o[q][i][e], 0.f, probe));
            odd |= probe != 0.f && (C::F32 || l[q][e] > 0.f);
          }
      }
      if (odd) again[warp] = 1;
    }
    u += c1 - c0;
  }
  if constexpr (MULTI || !C::E8) {
    __syncwarp();
    if (again[warp] != 0 && *abort_flag == 0)
      redo_share<T, CDT, D, R, KT>(a, c, plan, start_of(cta * W + warp), u_end, reinterpret_cast<float*>(ring),
                                   plan.spill + ((size_t)cta * W + warp) * C::PIECE, piece_m[2 * warp], piece_l[2 * warp]);
  }
  __syncthreads();

  // ---- the warps' pieces, item by item ----------------------------------------------------------------------------------
  int4 span[2] = {make_int4(-1, 0, 0, 0), make_int4(-1, 0, 0, 0)};
  for (int p = 0; p < 2 * W;) {
    const int item = piece_item[p];
    if (item < 0) { ++p; continue; }
    int last = p;
    for (int k = p + 1; k < 2 * W; ++k) {
      if (piece_item[k] == item) last = k;
      else if (piece_item[k] >= 0) break;
    }
    const bool begins = piece_flags[p] & 1, ends = piece_flags[last] & 2;
    const int bb = plan.seq.by(item), idx = item - bb * plan.per_seq, kvh = plan.tile.by(idx), row0 = (idx - kvh * plan.tiles) * R;
    const size_t part = (size_t)cta * 2 + (begins ? 1 : 0);
    for (int e = threadIdx.x; e < R * D / 4; e += W * 32) {
      const int r = e / (D / 4), d = e % (D / 4) * 4;
      float mc = -INFINITY, lc = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int k = p; k <= last; ++k)
        if (piece_item[k] == item) mc = fmaxf(mc, piece_m[k][r]);
      for (int k = p; k <= last; ++k) {
        if (piece_item[k] != item) continue;
        const float w = part_weight(piece_m[k][r], mc);
        const float4 v = *reinterpret_cast<const float4*>(piece_at[k] + r * D + d);
        acc.x += w * v.x; acc.y += w * v.y; acc.z += w * v.z; acc.w += w * v.w;
        lc += w * piece_l[k][r];
      }
      if (begins && ends) {
        if (row0 + r < rows) store_row4<T>(a, c, plan.group, bb, kvh, row0 + r, d, acc, lc);
      } else {
        *reinterpret_cast<float4*>(plan.parts + (part * R + r) * D + d) = acc;
        if (d == 0) {
          float* st = plan.parts + (size_t)plan.grid * 2 * R * D + (part * R + r) * 2;
          st[0] = mc;
          st[1] = lc;
        }
      }
    }
    if (!(begins && ends)) {
      const int4 x = make_int4(item, cta_of(piece_start[p]), cta_of(piece_end[p] - 1), 0);
      if (begins) span[1] = x;
      else span[0] = x;
    }
    p = last + 1;
  }
  if (threadIdx.x == 0) { plan.spans[2 * cta] = span[0]; plan.spans[2 * cta + 1] = span[1]; }
}

// Joins the items that several CTAs have parts of.  CTA i takes its share of the columns of each item that CTA i of the kernel
// above has a part of, so that many parts of one item are read by as many CTAs; groups of threads share the parts.
constexpr int PJ_THREADS = 256;
template <typename T, int D, int R>
__global__ void __launch_bounds__(PJ_THREADS) paged_join_kernel(const AttendArgs a, const Paged c, const AttendPlan plan) {
  static_assert(R * D / 4 <= 2 * PJ_THREADS, "two CTAs have an item's columns among them");
  __shared__ float4 sum[PJ_THREADS];
  __shared__ float2 stat[PJ_THREADS];
  const int cta = blockIdx.x, tid = threadIdx.x;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const float2* stats = reinterpret_cast<const float2*>(plan.parts + (size_t)plan.grid * 2 * R * D);
  for (int which = 0; which < 2; ++which) {
    const int4 span = plan.spans[2 * cta + which];
    if (span.x < 0) continue;
    const int first = span.y, parts = span.z - first + 1;
    const int b = plan.seq.by(span.x), idx = span.x - b * plan.per_seq, kvh = plan.tile.by(idx), row0 = (idx - kvh * plan.tiles) * R;
    const int slots = min(R, c.S * (int)plan.group.d - row0) * (D / 4), each = (slots + parts - 1) / parts, s0 = (cta - first) * each;
    const int mine = min(each, slots - s0);
    if (mine <= 0) continue;
    const int P = mine <= 1 ? 1 : 1 << (32 - __clz(mine - 1)), G = PJ_THREADS / P;
    const int slot = tid & (P - 1), group = tid / P, r = (s0 + slot) / (D / 4), d = (s0 + slot) % (D / 4) * 4;
    float m = -INFINITY, l = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    auto merge = [&](float2 st, float4 v) {
      const float mn = fmaxf(m, st.x), wa = part_weight(m, mn), wb = part_weight(st.x, mn);
      acc.x = acc.x * wa + v.x * wb; acc.y = acc.y * wa + v.y * wb; acc.z = acc.z * wa + v.z * wb; acc.w = acc.w * wa + v.w * wb;
      l = l * wa + st.y * wb;
      m = mn;
    };
    if (slot < mine) {
#pragma unroll 2
      for (int k = group; k < parts; k += G) {
        const size_t part = (size_t)(first + k) * 2 + (k == 0 ? 1 : 0);
        merge(stats[part * R + r], *reinterpret_cast<const float4*>(plan.parts + (part * R + r) * D + d));
      }
    }
    for (int h = G / 2; h >= 1; h >>= 1) {
      __syncthreads();
      sum[tid] = acc;
      stat[tid] = make_float2(m, l);
      __syncthreads();
      if (group < h) merge(stat[tid + h * P], sum[tid + h * P]);
    }
    if (group == 0 && slot < mine) store_row4<T>(a, c, plan.group, b, kvh, row0 + r, d, acc, l);
  }
}

// A pool's rows [pages * Hkv * page, D] in boxes of 16 rows and `box` bytes
static int pool_map(CUtensorMap* out, const void* pool, const Paged& c, int cdt, int box) {
  EncodeTiledFn4 enc = encode4();
  if (enc == nullptr) return -1;
  const int es = cdt == DT_E4M3 ? 1 : cdt == DT_F32 ? 4 : 2;
  const cuuint64_t dims[2] = {(cuuint64_t)c.D, (cuuint64_t)c.pages * c.Hkv * c.page}, strides[1] = {(cuuint64_t)c.D * es};
  const cuuint32_t boxes[2] = {(cuuint32_t)(box / es), 16}, steps[2] = {1, 1};
  const CUtensorMapDataType type = cdt == DT_E4M3 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : cdt == DT_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : cdt == DT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  return (int)enc(out, type, 2, const_cast<void*>(pool), dims, strides, boxes, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  box == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
}

template <typename T, int CDT, int D, int NQ, bool MULTI>
static int launch_attend(const AttendArgs& a, const Paged& c, float* parts, int4* spans, int grid, cudaStream_t st) {
  using C = PA<T, CDT, D, NQ>;
  static unsigned long long cfg = 0;
  int r;
  if ((r = smem_opt_in(paged_attend_kernel<T, CDT, D, NQ, MULTI>, C::SMEM, cfg)) != 0) return r;
  AttendPlan plan;
  plan.tiles = (c.S * (a.Hq / c.Hkv) + C::R - 1) / C::R;
  plan.per_seq = plan.tiles * c.Hkv;
  plan.grid = grid;
  plan.seq = Div(plan.per_seq);
  plan.tile = Div(plan.tiles);
  plan.group = Div(a.Hq / c.Hkv);
  plan.page = Div(c.page / 16);
  plan.parts = parts;
  plan.spans = spans;
  plan.spill = reinterpret_cast<float*>(spans + 2 * (size_t)grid);
  CUtensorMap tmk, tmv;
  if ((r = pool_map(&tmk, a.kpool, c, CDT, C::BOX)) != 0 || (r = pool_map(&tmv, a.vpool, c, CDT, C::BOX)) != 0) return 20000 + r;
  paged_attend_kernel<T, CDT, D, NQ, MULTI><<<grid, PA_WARPS * 32, C::SMEM, st>>>(tmk, tmv, a, c, plan);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return (int)e;
  cudaLaunchConfig_t lc{};
  lc.gridDim = dim3(grid);
  lc.blockDim = dim3(PJ_THREADS);
  lc.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  lc.attrs = at;
  lc.numAttrs = 1;
  e = cudaLaunchKernelEx(&lc, paged_join_kernel<T, D, C::R>, a, c, plan);
  return e != cudaSuccess ? (int)e : (int)cudaGetLastError();
}

// Any type and head size: a CTA takes a row of queries and one of `splits` runs of keys, its warps every fourth key, their lanes a
// share of the head.  Runs are joined below.
template <typename T, int CDT>
__global__ void __launch_bounds__(PA_WARPS * 32) paged_attend_any_kernel(const AttendArgs a, const Paged c, int splits, float* parts) {
  constexpr int N = PA_MAX_D / 32;
  __shared__ float sm_o[PA_WARPS][PA_MAX_D], sm_m[PA_WARPS], sm_l[PA_WARPS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int line = blockIdx.x / splits, split = blockIdx.x - line * splits;
  const int h = line % a.Hq, s = line / a.Hq % c.S, b = line / a.Hq / c.S;
  const int kvh = h / (a.Hq / c.Hkv), n = c.count(b);
  long long end = s < n ? (long long)c.length(b) - n + s + 1 : 0;
  if (end > c.capacity()) {
    if (threadIdx.x == 0 && split == 0) report_error(c.status, GB_ERR_BAD_INDEX, SITE_POSITION, (int)end - 1);
    end = c.capacity();
  }
  const int from = (int)(end * split / splits);
  end = end * (split + 1) / splits;
  const T* q = reinterpret_cast<const T*>(a.q) + (long long)line * c.D;
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
  for (int j = from + warp; j < end; j += PA_WARPS) {
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
    if (splits > 1) parts[(size_t)blockIdx.x * (c.D + 2) + d] = acc;
    else reinterpret_cast<T*>(a.o)[(long long)line * c.D + d] = Cvt<T>::from_f(lc == 0.f ? 0.f : acc / lc);
  }
  if (splits > 1 && threadIdx.x == 0) {
    parts[(size_t)blockIdx.x * (c.D + 2) + c.D] = mc;
    parts[(size_t)blockIdx.x * (c.D + 2) + c.D + 1] = lc;
  }
}

template <typename T>
__global__ void __launch_bounds__(PA_WARPS * 32) paged_join_any_kernel(void* o, int D, int splits, const float* parts) {
  const float* p = parts + (size_t)blockIdx.x * splits * (D + 2);
  float m = -INFINITY;
  for (int k = 0; k < splits; ++k) m = fmaxf(m, p[k * (D + 2) + D]);
  const float base = m == -INFINITY ? 0.f : m;
  for (int d = threadIdx.x; d < D; d += PA_WARPS * 32) {
    float acc = 0.f, l = 0.f;
    for (int k = 0; k < splits; ++k) {
      const float w = expf(p[k * (D + 2) + D] - base);
      acc += w * p[k * (D + 2) + d];
      l += w * p[k * (D + 2) + D + 1];
    }
    reinterpret_cast<T*>(o)[(long long)blockIdx.x * D + d] = Cvt<T>::from_f(l == 0.f ? 0.f : acc / l);
  }
}

// Runs of keys of the kernel for any type: until each SM has sixteen CTAs, of 64 keys at least.
static int any_splits(long long rows, int page, int per) {
  const long long keys = (long long)page * per, most = 16ll * sm_count() / (rows > 0 ? rows : 1);
  const long long n = keys / 64 < most ? keys / 64 : most;
  return n < 1 ? 1 : n > 256 ? 256 : (int)n;
}

}  // namespace gb

using namespace gb;

// Which kernel a call takes: query rows of an item and CTAs (0: the kernel for any type).  The tensor cores take heads of 64 or 128
// over caches of the queries' type, or of 8 bits below 16-bit queries; what remains (other head sizes, types that differ, more
// than 2^31 chunks of keys or rows of the pool) is worked on number by number.
//   rows: two operands of 8 read K and V half as often, and leave half as many chunks to share out.  By what the page table has
//   room for, two where each warp then has four chunks and more: 32 x 4096, drafts of 4, 32 / 4 heads of 128: 93 us (146 with one), 14 / 2
//   of 64, drafts of 2: 25.6 (28.7); 8 x 2000, drafts of 8, 12 / 2 of 128: 26.6 with two, 22.9 with one; 4 x 2000, drafts of 5: 17.6, 15.8.
//   The sequences' own lengths are known on the device only.  A table with room for 32768 over 8 sequences of 200 (drafts of 4, 32 / 4 of
//   128) takes two operands for one and 15.8 us for 14.0; single tokens 11.7 for 11.2; over 32 of 2000 nothing changes.
struct AttendChoice { int R, grid; };
static AttendChoice attend_choice(int B, int S, int Hq, int Hkv, int D, int page, int pages, int per, int dt, int cdt) {
  if ((D != 64 && D != 128) || (cdt != dt && !(cdt == DT_E4M3 && dt != DT_F32)) || page % 16) return {8, 0};
  const int rows = S * (Hq / Hkv), kt = attend_chunk(D, cdt == DT_E4M3 ? 1 : cdt == DT_F32 ? 4 : 2);
  const long long keys = (long long)per * page, run = keys <= 0 ? 1 : (keys + kt - 1) / kt;
  auto chunks = [&](int R) { return (long long)B * Hkv * ((rows + R - 1) / R) * run; };
  // (numbers of 32 bits and 128 have no registers for two)
  const int R = rows <= 8 || (cdt == DT_F32 && D == 128) || chunks(16) < 4ll * 12 * sm_count() ? 8 : 16;
  if (chunks(R) > 0x7fffffff || (long long)pages * Hkv * page > 0x7fffffff) return {8, 0};       // (counted in 32 bits)
  const long long want = (chunks(R) + PA_WARPS - 1) / PA_WARPS, most = (long long)sm_count() * attend_ctas(dt, cdt, D, R);
  return {R, (int)(want < most ? want : most)};
}

// 32-bit words of workspace that a call needs
extern "C" int gb_paged_attention_workspace(int B, int S, int Hq, int Hkv, int D, int page, int pages, int per, int dt, int cdt) {
  if (B <= 0 || S <= 0 || Hq <= 0 || Hkv <= 0) return 0;
  const AttendChoice x = attend_choice(B, S, Hq, Hkv, D, page, pages, per, dt, cdt);
  if (x.grid == 0) {
    const long long rows = (long long)B * S * Hq;
    const int splits = any_splits(rows, page, per);
    return splits == 1 ? 0 : (int)(rows * splits * (D + 2));
  }
  return x.grid * (2 * (x.R * (D + 2) + 4) + PA_WARPS * x.R * D);
}

extern "C" int gb_paged_attention(const void* pools, const void* q, void* o, const int* table, const int* lengths, const int* counts,
                                  int B, int S, int Hq, int per, float scale, int dt, float* workspace, int* status,
                                  cudaStream_t st) {
  const PagedPools& p = *reinterpret_cast<const PagedPools*>(pools);
  const int Hkv = p.Hkv, D = p.D, page = p.page, pages = p.pages, cdt = p.type;
  if (B <= 0 || S <= 0 || Hq <= 0 || D <= 0) return 0;
  if (D > PA_MAX_D || Hkv <= 0 || Hq % Hkv) return -3;
  AttendArgs a{q, o, p.k, p.v, p.kscale, p.vscale, Hq, scale};
  Paged c{table, lengths, counts, status, B, S, Hkv, D, page, pages, per, Div(page)};
  const long long rows = (long long)B * S * Hq;
  if (rows > 0x7fffffff) return -4;
  const AttendChoice x = attend_choice(B, S, Hq, Hkv, D, page, pages, per, dt, cdt);
  if (x.grid > 0) {
    const int R = x.R, grid = x.grid;
    int4* spans = reinterpret_cast<int4*>(workspace + (size_t)grid * 2 * R * (D + 2));
#define GB_ATTEND_(T, C, D_, NQ_) (S > 1 ? launch_attend<T, C, D_, NQ_, true>(a, c, workspace, spans, grid, st) : launch_attend<T, C, D_, NQ_, false>(a, c, workspace, spans, grid, st))
#define GB_ATTEND(T, C) (D == 64 ? (R == 8 ? GB_ATTEND_(T, C, 64, 1) : GB_ATTEND_(T, C, 64, 2)) : (R == 8 ? GB_ATTEND_(T, C, 128, 1) : GB_ATTEND_(T, C, 128, 2)))
    if (dt == DT_BF16) return cdt == DT_E4M3 ? GB_ATTEND(__nv_bfloat16, DT_E4M3) : GB_ATTEND(__nv_bfloat16, DT_BF16);
    if (dt == DT_F16) return cdt == DT_E4M3 ? GB_ATTEND(__half, DT_E4M3) : GB_ATTEND(__half, DT_F16);
    if (D == 128) return GB_ATTEND_(float, DT_F32, 128, 1);
    return R == 8 ? GB_ATTEND_(float, DT_F32, 64, 1) : GB_ATTEND_(float, DT_F32, 64, 2);
#undef GB_ATTEND
#undef GB_ATTEND_
  }
  const int splits = any_splits(rows, page, per);
  GB_DISPATCH_FLOAT(dt, T, GB_DISPATCH_CACHE(cdt, C, paged_attend_any_kernel<T, C><<<(unsigned)(rows * splits), PA_WARPS * 32, 0, st>>>(a, c, splits, workspace)));
  if (splits > 1) GB_DISPATCH_FLOAT(dt, T, paged_join_any_kernel<T><<<(unsigned)rows, PA_WARPS * 32, 0, st>>>(o, D, splits, workspace));
  return (int)cudaGetLastError();
}
