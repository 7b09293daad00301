// Newton-Schulz orthogonalisation of weight updates: the singular values of a matrix are driven to about one by
//
//   X = G / (|G|_F + eps),   repeated:  A = X X^T,  B = b A + c A A,  X <- (a I + B) X           (X: m x n, m <= n)
//
// i.e. every singular value s goes to a s + b s^3 + c s^5.  A tall G is handled as its transpose.
//
// Steps are made one by one, with products of X, A X; or, for long and many matrices, in blocks (see one_by_one).
//
// Products of m x m matrices in place of m x n ones, in a block.  With P = a I + B, the next A is P A P, so a block of steps needs X
// only at its ends: A = X X^T once, then per step  B = b A + c A A,  W = a A + B A,  A <- a W + B W,  and the product of the
// P's, kept as s I + Q:  Q <- a Q + s B + B Q.  At the end of the block X <- s X + Q X.  All but the last are symmetric.
// For 896 x 4864 and five steps in blocks of three and two that is 33 GFLOP for the 62 of five products with X each way, and
// X passes through memory twice instead of five times; for square matrices it is as many operations.  A rounding of A grows
// by a^2 a step, so blocks are of three at most: five in one lose a digit (256 x 1024, simulated, Gaussian and rank 8 plus noise:
// 5e-6 and 21e-6), and matrices of few rows, which have few roundings else, go without (see one_by_one).
//
// Arithmetic.  The iteration amplifies: with the usual coefficients a small singular value grows by a factor of
// 3.44 a step, 485 over five, and so does every rounding of X in its direction.  So X, A and W are kept in 32 bits, and enter
// the tensor cores as two fp16 terms, x 2^k = hi + lo, which hold 22 of its 24 bits (k keeps the largest entry near the top
// of fp16's range, so that lo stays clear of its subnormals: an entry is at most the largest eigenvalue, which the host
// bounds from the coefficients).  Each product is three of fp16 with fp32 accumulation, hi hi + hi lo + lo hi; a X, a A and a W
// are added in 32 bits from the matrices themselves.  One fp16 term alone loses three digits (1.7e-3).
//
// Work.  Of symmetric results only tiles on and below the diagonal are computed, the rest is written as their mirror image by
// the same epilogue.  A product is one launch over all matrices of a batch (W and Q of a block's step together; for m <= 128, A and B
// of a step, which then is two launches), on persistent CTAs:
//   warp 0 TMA producer, warp 1 issues tcgen05.mma, warps 4-11 epilogue; accumulators in all of tensor memory.
// A block of 64 elements of the contraction brings both terms of both operands and feeds three products.  Tiles too few to
// fill the GPU are shared by clusters of up to 8 CTAs, each with a part of the contraction; many large ones are worked on by
// CTA pairs, which read two thirds of the bytes.
//
// Sums.  The tensor cores round their accumulator towards zero, by 0.5 to 0.8 of a unit in the last place for every 16
// elements of the contraction: 13 units of a sum of 256 positive terms, 65 of 1024.  In A that shortens the diagonal, and steps
// with A amplify it.  So in symmetric products an accumulator takes up 64 elements of the contraction where a cluster shares
// it (matrices with few rows for their length, which lose most, are there; 896 x 4864 267 for 262 us with 128), else 128, the
// small products of each block of 64 first, and is then added, rounded to nearest, to the sums that the epilogue's warps hold
// in registers; in the products with X, 256.  The products go on in the next accumulator meanwhile.  Measured error
// of the result against 64 bits, in blocks, with 64 / 128 / 256 elements throughout (and of fp32 products): rank 8 plus noise, 16 x 5000
// 3.6 / 6.3 / 9.6e-6 (0.8e-6), 1024 x 4096 1.9 / 1.7 / 1.7e-6 (3.2e-6); Gaussian, 400 x 4000 1.5 / 2.2 / 3.3e-5 (0.5e-5), 1024 x 1024
// 7.5 / 7.6 / 9.9e-6 (3.1e-6); time of 24 of 4864 x 896 3866 / 3669 / 3592 us.
#include "sm100_ptx.cuh"
#include "sm100_pair.cuh"
#include "common.cuh"

namespace gb {

int make_tmap_3d(CUtensorMap* out, const void* base, int dtype, long long inner, long long outer, long long batch,
                 long long ld_elems, long long batch_stride_elems, int box_outer);

namespace ns {

constexpr int BM = 128, BK = 64;
constexpr int A_BYTES = BM * 128;                     // 128 rows of 64 fp16
constexpr int RING_BYTES = 4 * 48 * 1024;
constexpr int CHUNK_BYTES = 32 * 32 * 4;              // 32 x 32 results in fp32
constexpr int SLAB_OFFSET = RING_BYTES;               // one chunk per epilogue warp
constexpr int BARRIER_OFFSET = SLAB_OFFSET + 8 * CHUNK_BYTES;
constexpr int SMEM_TOTAL = BARRIER_OFFSET + 256;
constexpr int THREADS = 384;                          // warps 0 TMA, 1 MMA, 2 and 3 idle, 4-11 epilogue
constexpr int PARTS = 256;                            // most partial sums of squares per matrix

enum Mode : int { SYM = 0, APPLY = 1, APPLY_LAST = 2 };

// m x m matrices of a batch live in slots: terms [SLOTS][batch][hi, lo][m][lda] and, where they are needed, the matrices
// themselves in 32 bits [SLOTS][batch][m][lda], on and below the diagonal only.
constexpr int SLOTS = 5;

// out = f_acc L R + f1 M1 + f2 M2, symmetric
struct Problem {
  int left, right;             // slots of L and R (GRAM: X both)
  int out;                     // slot
  int m1, m2;                  // slots of M1, M2 or -1
  int keep;                    // the result in 32 bits is kept too
  float f_acc, f1, f2;
  float scale;                 // 2^k of the result's terms
};

struct Params {
  int* status;
  int m, n, batch;             // X [batch, m, n]
  int k;                       // elements of the contraction
  int ldx, lda;                // pitch of X and of m x m matrices in elements (multiples of 8)
  int problems;                // SYM: one or two for every matrix of the batch
  Problem prob[2];             // APPLY: prob[0].left is Q, X <- f_acc Q X + f1 X
  __half* terms;               // slots
  float* whole;
  __half* dst;                 // APPLY: terms of the next X [batch][hi, lo][m][ldx]
  float* x;                    // X in 32 bits [batch][m][ldx]
  // APPLY_LAST: out[batch] in `out_dtype`, or the weights of an optimizer step through `weights`
  void* out;
  int out_dtype, tall;         // tall: the result goes out transposed, [n, m]
  const long long* weights;    // [batch] addresses of fp32 weights (+ 1 where the weight is tall), or null
  float lr, decay, tall_scale; // w <- w (1 - lr decay) - lr o, or tall_scale lr o where it is tall
  const float* dyn_lr;
  const float* found_inf;
  int splits;                  // CTAs of a cluster that share a tile's contraction (1: whole tiles, persistent CTAs)
};

// Terms of four numbers, x = hi + lo to 22 bits: (hi0 hi1, hi2 hi3, lo0 lo1, lo2 lo3)
__device__ __forceinline__ uint4 split4(float a, float b, float c, float d) {
  uint4 t;
  t.x = pack2c<false>(a, b);
  t.y = pack2c<false>(c, d);
  const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&t.x)), y = __half22float2(*reinterpret_cast<const __half2*>(&t.y));
  t.z = pack2c<false>(a - x.x, b - x.y);
  t.w = pack2c<false>(c - y.x, d - y.y);
  return t;
}
__device__ __forceinline__ void prefetch_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }

// Byte offset of 16-byte unit `u` of row `r` of a 32 x 32 chunk in shared memory.  Eight neighbouring rows, and the eight
// rows r, r + 4, .., put a unit into eight different bank groups: rows written lane by lane, read unit by unit, and
// columns read four rows apart are all free of conflicts.
__device__ __forceinline__ int chunk_at(int r, int u) { return r * 128 + ((u ^ r ^ (r >> 3)) & 7) * 16; }

__device__ __forceinline__ float4 ld_peer(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
// A launch of this chain may start while the one before it runs; nothing that it wrote is touched before this returns.
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// What becomes of a 32 x 32 chunk of accumulators (rows row0.., columns col0.. of matrix z).  A lane takes four neighbouring
// columns of a row, eight lanes a row, so that memory sees whole 128-byte lines (64 of fp16): acc[i] is row 4 i + lane / 8,
// columns 4 (lane % 8)...  `chunk` is the warp's shared memory, for what goes out transposed.  What a chunk reads is fetched
// while the chunk before it is worked on: with the loads of a row behind the stores of the row before it, each row waited
// for its own, and an epilogue took twice as long as the products of its tile.
template <int MODE>
struct Epilogue {
  const Params& p;
  int lane;
  float keep, step;
  bool skip, vec;              // vec: four elements of the result at a time
  __device__ __forceinline__ Epilogue(const Params& q) : p(q), lane(threadIdx.x & 31), keep(1.f), step(0.f), skip(false), vec(false) {
    if constexpr (MODE == APPLY_LAST) {
      const float lr = p.dyn_lr != nullptr ? *p.dyn_lr : p.lr;
      keep = 1.f - lr * p.decay;
      step = lr;
      skip = p.found_inf != nullptr && *p.found_inf != 0.f;
      // rows of n, or m, elements start on a boundary of four, and end on one
      vec = ((p.tall ? p.m : p.n) & 3) == 0 && (reinterpret_cast<uintptr_t>(p.out) & 15) == 0;
    }
  }
  // symmetric results: blocks of 128 below the diagonal are written twice, those above it not at all
  __device__ __forceinline__ bool outside(int row0, int col0) const {
    return row0 >= p.m || col0 >= (MODE == SYM ? p.m : p.n) || (MODE == SYM && col0 / BM > row0 / BM);
  }
  // four elements of row `row` of the 32-bit matrix in slot `slot` of matrix z
  __device__ __forceinline__ float* whole(int slot, int z, int row, int col) const {
    return p.whole + (((size_t)slot * p.batch + z) * p.m + row) * p.lda + col;
  }
  // What a chunk's results are made from besides its sums: X, or M1
  __device__ __forceinline__ void fetch(float4 (&in)[8], int z, int row0, int col0) const {
    const int r0 = lane >> 3, col = col0 + 4 * (lane & 7);
    int rows = outside(row0, col0) || col >= (MODE == SYM ? p.m : p.n) ? 0 : p.m - row0 - r0;
    const float* src;
    size_t pitch;
    if constexpr (MODE == SYM) {
      const Problem& q = p.prob[z >= p.batch];
      if (q.m1 < 0) rows = 0;
      src = whole(q.m1, z >= p.batch ? z - p.batch : z, row0 + r0, col);
      pitch = 4 * (size_t)p.lda;
    } else {
      src = p.x + ((size_t)z * p.m + row0 + r0) * p.ldx + col;
      pitch = 4 * (size_t)p.ldx;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
      in[i] = 4 * i < rows ? *reinterpret_cast<const float4*>(src + i * pitch) : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  __device__ __forceinline__ void run(const float4 (&acc)[8], const float4 (&in)[8], uint8_t* chunk, int z, int row0, int col0) const {
    const int cols = MODE == SYM ? p.m : p.n;
    if (outside(row0, col0)) return;
    const int u = lane & 7, r0 = lane >> 3, col = col0 + 4 * u;
    const int rows = col < cols ? p.m - row0 - r0 : 0;           // (rows 4 i of this lane below it are inside the matrix)
    const Problem& q = p.prob[MODE == SYM && z >= p.batch];
    float4 v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = axpby(acc[i], q.f_acc, in[i], q.f1);
    if constexpr (MODE == SYM) {
      if (z >= p.batch) z -= p.batch;
      const bool mirror = col0 / BM < row0 / BM;
      const size_t pitch = 4 * (size_t)p.lda;
      if (q.m2 >= 0) {
        const float* src = whole(q.m2, z, row0 + r0, col);
        float4 w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = 4 * i < rows ? *reinterpret_cast<const float4*>(src + i * pitch) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = axpby(w[i], q.f2, v[i], 1.f);
      }
      if (q.keep) {
        float* dst = whole(q.out, z, row0 + r0, col);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (4 * i < rows) *reinterpret_cast<float4*>(dst + i * pitch) = v[i];
      }
      const size_t plane = (size_t)p.m * p.lda;
      __half* base = p.terms + ((size_t)q.out * p.batch + z) * 2 * plane;
      uint4 t[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) t[i] = split4(v[i].x * q.scale, v[i].y * q.scale, v[i].z * q.scale, v[i].w * q.scale);
      if (mirror) {
        // both terms of an element in the place of its sum; then columns are read as rows
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 8; ++i)
          *reinterpret_cast<uint4*>(chunk + chunk_at(4 * i + r0, u)) =
              make_uint4(__byte_perm(t[i].x, t[i].z, 0x5410), __byte_perm(t[i].x, t[i].z, 0x7632),
                         __byte_perm(t[i].y, t[i].w, 0x5410), __byte_perm(t[i].y, t[i].w, 0x7632));
        __syncwarp();
      }
      __half* dst = base + (size_t)(row0 + r0) * p.lda + col;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (4 * i < rows) put(dst + i * pitch, plane, t[i]);
      if (mirror) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          uint32_t w[4];
          column(chunk, 4 * i + r0, u, w);
          t[i] = make_uint4(__byte_perm(w[0], w[1], 0x5410), __byte_perm(w[2], w[3], 0x5410), __byte_perm(w[0], w[1], 0x7632),
                            __byte_perm(w[2], w[3], 0x7632));
        }
        const int j = row0 + 4 * u, left = j < p.m ? p.m - col0 - r0 : 0;
        __half* out = base + (size_t)(col0 + r0) * p.lda + j;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (4 * i < left) put(out + i * pitch, plane, t[i]);
      }
    } else {
      if constexpr (MODE == APPLY) {
        float* x = p.x + ((size_t)z * p.m + row0 + r0) * p.ldx + col;
        const size_t pitch = 4 * (size_t)p.ldx, plane = (size_t)p.m * p.ldx;
        __half* dst = p.dst + (size_t)z * 2 * plane + (size_t)(row0 + r0) * p.ldx + col;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (4 * i < rows) {
            *reinterpret_cast<float4*>(x + i * pitch) = v[i];
            put(dst + i * pitch, plane, split4(v[i].x * q.scale, v[i].y * q.scale, v[i].z * q.scale, v[i].w * q.scale));
          }
        }
      } else {
        const bool across = p.weights != nullptr ? (p.weights[z] & 1) != 0 : p.tall != 0;     // the result is the transpose
        if (across) {
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 8; ++i) *reinterpret_cast<float4*>(chunk + chunk_at(4 * i + r0, u)) = v[i];
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            uint32_t w[4];
            column(chunk, 4 * i + r0, u, w);
            v[i] = make_float4(__uint_as_float(w[0]), __uint_as_float(w[1]), __uint_as_float(w[2]), __uint_as_float(w[3]));
          }
        }
        const int i0 = across ? col0 : row0, j = across ? row0 + 4 * u : col;
        const int ld = across ? p.m : p.n, count = ld - j;       // elements of a row from here on
        const int left = count > 0 ? (across ? p.n : p.m) - i0 - r0 : 0;
        const size_t at = (size_t)(i0 + r0) * ld + j, lp = 4 * (size_t)ld;
        if (p.weights != nullptr) {
          if (!skip) apply(reinterpret_cast<float*>(p.weights[z] & ~1ll) + at, lp, left, count, ld, across ? step * p.tall_scale : step, v);
        } else if (p.out_dtype == DT_F32) {
          float* o = reinterpret_cast<float*>(p.out) + (size_t)z * p.m * p.n + at;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            if (4 * i >= left) continue;
            if (vec) *reinterpret_cast<float4*>(o + i * lp) = v[i];
            else {
              o[i * lp] = v[i].x;
              if (count > 1) o[i * lp + 1] = v[i].y;
              if (count > 2) o[i * lp + 2] = v[i].z;
              if (count > 3) o[i * lp + 3] = v[i].w;
            }
          }
        } else {
          uint16_t* o = reinterpret_cast<uint16_t*>(p.out) + (size_t)z * p.m * p.n + at;
          const bool bf = p.out_dtype == DT_BF16;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            if (4 * i >= left) continue;
            uint2 w;
            if (bf) { w.x = pack2c<true>(v[i].x, v[i].y); w.y = pack2c<true>(v[i].z, v[i].w); }
            else { w.x = pack2c<false>(v[i].x, v[i].y); w.y = pack2c<false>(v[i].z, v[i].w); }
            if (vec) *reinterpret_cast<uint2*>(o + i * lp) = w;
            else {
              o[i * lp] = (uint16_t)w.x;
              if (count > 1) o[i * lp + 1] = (uint16_t)(w.x >> 16);
              if (count > 2) o[i * lp + 2] = (uint16_t)w.y;
              if (count > 3) o[i * lp + 3] = (uint16_t)(w.y >> 16);
            }
          }
        }
      }
    }
  }
  // rows 4 i of the weights from `w` on, `left` of them below, `count` elements each from here on
  __device__ __forceinline__ void apply(float* w, size_t pitch, int left, int count, int ld, float st, const float4 (&v)[8]) const {
    if ((ld & 3) == 0 && (reinterpret_cast<uintptr_t>(w) & 15) == 0) {
      float4 o[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (4 * i < left) o[i] = *reinterpret_cast<const float4*>(w + i * pitch);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (4 * i < left)
          *reinterpret_cast<float4*>(w + i * pitch) = make_float4(fmaf(o[i].x, keep, -st * v[i].x), fmaf(o[i].y, keep, -st * v[i].y),
                                                                  fmaf(o[i].z, keep, -st * v[i].z), fmaf(o[i].w, keep, -st * v[i].w));
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (4 * i >= left) continue;
        float* q = w + i * pitch;
        q[0] = fmaf(q[0], keep, -st * v[i].x);
        if (count > 1) q[1] = fmaf(q[1], keep, -st * v[i].y);
        if (count > 2) q[2] = fmaf(q[2], keep, -st * v[i].z);
        if (count > 3) q[3] = fmaf(q[3], keep, -st * v[i].w);
      }
    }
  }
  __device__ __forceinline__ float4 axpby(const float4& a, float f, const float4& b, float g) const {
    return make_float4(fmaf(a.x, f, b.x * g), fmaf(a.y, f, b.y * g), fmaf(a.z, f, b.z * g), fmaf(a.w, f, b.w * g));
  }
  // four rows 4 u .. of column `c` of the chunk
  __device__ __forceinline__ void column(const uint8_t* chunk, int c, int u, uint32_t (&v)[4]) const {
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = *reinterpret_cast<const uint32_t*>(chunk + chunk_at(4 * u + k, c >> 2) + (c & 3) * 4);
  }
  // (the pitch is a multiple of 8, so what lies past the last column is padding)
  __device__ __forceinline__ void put(__half* hi, size_t plane, const uint4& t) const {
    *reinterpret_cast<uint2*>(hi) = make_uint2(t.x, t.y);
    *reinterpret_cast<uint2*>(hi + plane) = make_uint2(t.z, t.w);
  }
  // What this lane's warp will read of a chunk at its end is fetched into L2 while the products run: one line a lane
  __device__ __forceinline__ void prefetch(int z, int row0, int col0) const {
    if constexpr (MODE != SYM) {
      if (row0 + lane < p.m && col0 < p.n) prefetch_l2(p.x + ((size_t)z * p.m + row0 + lane) * p.ldx + col0);
      if constexpr (MODE == APPLY_LAST) {
        if (p.weights != nullptr) {
          const float* w = reinterpret_cast<const float*>(p.weights[z] & ~1ll);
          if (p.weights[z] & 1) { if (col0 + lane < p.n && row0 < p.m) prefetch_l2(w + (size_t)(col0 + lane) * p.m + row0); }
          else if (row0 + lane < p.m && col0 < p.n) prefetch_l2(w + (size_t)(row0 + lane) * p.n + col0);
        }
      }
    }
  }
};

// How CTAs work on tiles: each on whole ones; the CTAs of a cluster each on a part of the contraction of one tile; two CTAs
// on a tile of twice the rows, through the tensor instructions of CTA pairs.
enum Kind : int { WHOLE = 0, SPLIT = 1, PAIR = 2 };

// Tiles of `rows` x BN: for the symmetric modes those that hold a block of 128 x 128 on or below the diagonal, row by row
__host__ __device__ constexpr long long tiles_of(bool sym, long long m, long long n, int rows, int bn) {
  const long long tm = (m + rows - 1) / rows;
  if (!sym) return tm * ((n + bn - 1) / bn);
  return bn == rows ? tm * (tm + 1) / 2 : (tm + 1) / 2 * (tm + 1 - (tm + 1) / 2);
}

template <int MODE, int BN, int KIND>
__global__ void __launch_bounds__(THREADS, 1)
ns_product_kernel(const __grid_constant__ CUtensorMap tmapA, const __grid_constant__ CUtensorMap tmapB,
                  const __grid_constant__ Params p) {
  constexpr bool B_MN = MODE != SYM;                           // X as the right operand: its rows run along the contraction
  constexpr int TM = KIND == PAIR ? 2 * BM : BM;        // rows of a tile
  constexpr int BNC = KIND == PAIR ? BN / 2 : BN;       // columns of the right operand that a CTA loads
  // Ring of half stages: the high terms of both operands for a block of the contraction, then the low ones.  The products of
  // a block run in the order hi lo, lo hi, hi hi: while the small ones are summed the accumulator is small and loses little,
  // and the low terms are free before the block is done.
  constexpr int HALF_BYTES = A_BYTES + BNC * 128, HALVES = RING_BYTES / HALF_BYTES / 2 * 2;
  constexpr int ACCS = 512 / BN;                        // accumulators in tensor memory
  // blocks of BK that one accumulator takes up: see the header
  constexpr int DRAIN = MODE != SYM ? 4 : KIND == SPLIT ? 1 : 2;
  constexpr int CHUNKS = BN / 64;                       // of 32 x 32 results, per epilogue warp
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + BARRIER_OFFSET);       // (a pair: those of CTA 0 count both CTAs' loads)
  uint64_t* empty_bar = full_bar + HALVES;
  uint64_t* tmem_full = empty_bar + HALVES;
  uint64_t* tmem_empty = tmem_full + ACCS;                                       // (a pair: those of CTA 0 count both epilogues)
  uint32_t* tmem_base_slot = reinterpret_cast<uint32_t*>(tmem_empty + ACCS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_base_slot + 1);
  uint32_t* poison_slot = tmem_base_slot + 2;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
  const int lane = threadIdx.x & 31;
  const int rank = KIND == WHOLE ? 0 : (int)g2::cta_rank_in_cluster();

  if (threadIdx.x == 0) {
    for (int s = 0; s < HALVES; ++s) { mbar_init(&full_bar[s], 1); mbar_init(&empty_bar[s], 1); }
    for (int a = 0; a < ACCS; ++a) { mbar_init(&tmem_full[a], 1); mbar_init(&tmem_empty[a], KIND == PAIR ? 16 : 8); }
    // after an error no work is done, but every CTA of a cluster comes to its barriers
    const bool aligned = (smem_u32(smem) & 1023) == 0;
    if (!aligned) report_error(p.status, GB_ERR_BAD_ARG, 5, 0);
    *abort_flag = !aligned || status_poisoned(p.status) ? 1 : 0;
    *poison_slot = (uint32_t)*abort_flag;
    mbar_fence_init();
    tma_prefetch_desc(&tmapA);
    tma_prefetch_desc(&tmapB);
  }
  if (warp == 1) {
    if constexpr (KIND == PAIR) { g2::tmem_alloc2(tmem_base_slot, 512); g2::tmem_relinquish2(); }
    else { tmem_alloc(tmem_base_slot, 512); tmem_relinquish(); }
  }
  tc_fence_before_sync();
  __syncthreads();
  if constexpr (KIND == PAIR) {
    // the two decide alike whether they work
    g2::cluster_sync_all();
    const uint32_t other = g2::ld_cluster_u32(g2::map_to_cta(smem_u32(poison_slot), rank ^ 1));
    if (threadIdx.x == 0 && other != 0) *abort_flag = 1;
    __syncthreads();
  }
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_base_slot;
  let_next_start();
  wait_for_previous();

  const int tm = (p.m + TM - 1) / TM;
  const int per = (int)tiles_of(MODE == SYM, p.m, p.n, TM, BN);
  const long long total = (long long)per * p.batch * p.problems;
  const int kblocks = (p.k + BK - 1) / BK;
  // this CTA's tiles and its part of their contraction, in blocks of BK
  const int splits = KIND == SPLIT ? p.splits : 1, group = KIND == PAIR ? 2 : splits;
  const long long first = blockIdx.x / group, stride = gridDim.x / group;
  const int kb0 = KIND == SPLIT ? kblocks * rank / splits : 0, kb1 = KIND == SPLIT ? kblocks * (rank + 1) / splits : kblocks;
  const int row_in_tile = KIND == PAIR ? rank * BM : 0;
  // tile of matrix z: (mi, ni)
  auto decode = [&](long long t, int& mi, int& ni, int& z) {
    z = (int)(t / per);
    const int r = (int)(t % per);
    if constexpr (MODE == SYM) {
      if constexpr (BN == TM) {
        mi = (int)((sqrtf(8.f * (float)r + 1.f) - 1.f) * 0.5f);
        while (mi * (mi + 1) / 2 > r) --mi;
        while ((mi + 1) * (mi + 2) / 2 <= r) ++mi;
        ni = r - mi * (mi + 1) / 2;
      } else {
        // rows 2 g and 2 g + 1 have g + 1 tiles each; g (g + 1) tiles lie before row 2 g
        int g = (int)((sqrtf(4.f * (float)r + 1.f) - 1.f) * 0.5f);
        while (g * (g + 1) > r) --g;
        while ((g + 1) * (g + 2) <= r) ++g;
        const int o = r - g * (g + 1);
        mi = 2 * g + (o > g ? 1 : 0);
        ni = o > g ? o - g - 1 : o;
      }
    } else {
      ni = r / tm;
      mi = r % tm;
    }
  };
  // a role that gives up takes the pair with it
  auto give_up = [&]() {
    if constexpr (KIND == PAIR) g2::st_cluster_u32(g2::map_to_cta(smem_u32(const_cast<int*>(abort_flag)), rank ^ 1), 1u);
  };

  // The sums of a 128 x 256 tile take 128 registers of every epilogue thread: of 384 x 168 at launch, the first four warps
  // keep 56 each and the others get 224 (128 x 56 + 256 x 224 = 384 x 168).
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp == 0) {
      // =========================== TMA producer ===========================
      if (elect_one()) {
        uint32_t it = 0;
        for (long long t = first; t < total && !*abort_flag; t += stride) {
          int mi, ni, z;
          decode(t, mi, ni, z);
          const int m0 = mi * TM + row_in_tile, n0 = ni * BN + (KIND == PAIR ? rank * BNC : 0);
          // planes of the operands: two for every matrix of a slot
          const Problem& pr = p.prob[z >= p.batch];
          const int zz = z >= p.batch ? z - p.batch : z;
          const int za = 2 * (pr.left * p.batch + zz), zb = 2 * (pr.right * p.batch + zz);
          bool ok = true;
          for (int kh = 2 * kb0; kh < 2 * kb1; ++kh, ++it) {
            const int s = it % HALVES, k0 = (kh >> 1) * BK, h = kh & 1;      // h: 0 = high terms, 1 = low
            if (!mbar_wait(&empty_bar[s], ((it / HALVES) & 1) ^ 1, abort_flag, p.status, 110)) { ok = false; break; }
            uint8_t* sa = smem + s * HALF_BYTES;
            uint8_t* sb = sa + A_BYTES;
            if constexpr (KIND == PAIR) {
              const uint32_t bar = g2::map_to_cta(smem_u32(&full_bar[s]), 0);
              if (rank == 0) mbar_expect_tx(&full_bar[s], 2 * HALF_BYTES);
              g2::tma2_load_3d(sa, &tmapA, bar, k0, m0, za + h);
              if constexpr (!B_MN) {
                g2::tma2_load_3d(sb, &tmapB, bar, k0, n0, zb + h);
              } else {
#pragma unroll
                for (int c = 0; c < BNC / 64; ++c) g2::tma2_load_3d(sb + c * (BK * 128), &tmapB, bar, n0 + c * 64, k0, zb + h);
              }
            } else {
              mbar_expect_tx(&full_bar[s], HALF_BYTES);
              tma_load_3d(sa, &tmapA, &full_bar[s], k0, m0, za + h);
              if constexpr (!B_MN) {
#pragma unroll
                for (int c = 0; c < BNC / 128; ++c)
                  tma_load_3d(sb + c * A_BYTES, &tmapB, &full_bar[s], k0, n0 + c * 128, zb + h);
              } else {
#pragma unroll
                for (int c = 0; c < BNC / 64; ++c) tma_load_3d(sb + c * (BK * 128), &tmapB, &full_bar[s], n0 + c * 64, k0, zb + h);
              }
            }
          }
          if (!ok) { give_up(); break; }
        }
        if (*abort_flag && (KIND != PAIR || rank == 0)) drain_copies(full_bar, HALVES, it);
      }
      __syncwarp();
    } else if (warp == 1 && (KIND != PAIR || rank == 0)) {
      // =========================== MMA issuer (converged warp, one elected lane) ===========================
      const uint32_t idesc = make_idesc(0u, 0u, B_MN ? 1u : 0u, TM, BN);
      uint32_t it = 0, drains = 0;
      bool ok = __all_sync(0xffffffffu, *abort_flag == 0);
      auto b_desc = [&](uint32_t addr) { return B_MN ? make_smem_desc(addr, BK * 128, 1024) : make_smem_desc(addr, 16, 1024); };
      auto multiply = [&](uint32_t d, uint64_t a, uint64_t b, bool fresh) {
#pragma unroll
        for (int kk = 0; kk < BK / 16; ++kk) {                               // (descriptors count 16-byte units)
          const uint64_t bk = b + (B_MN ? kk * 128 : kk * 2);
          if constexpr (KIND == PAIR) g2::umma2_f16(d, a + kk * 2, bk, idesc, fresh && kk == 0 ? 0u : 1u);
          else umma_f16(d, a + kk * 2, bk, idesc, fresh && kk == 0 ? 0u : 1u);
        }
      };
      auto commit = [&](uint64_t* bar) {                                     // (in both CTAs of a pair)
        if constexpr (KIND == PAIR) {
          g2::umma2_commit(smem_u32(bar));
          g2::umma2_commit(g2::map_to_cta(smem_u32(bar), 1));
        } else {
          umma_commit(bar);
        }
      };
      for (long long t = first; t < total && ok; t += stride) {
        for (int kb = kb0; kb < kb1 && ok; kb += DRAIN, ++drains) {
          const uint32_t acc = drains % ACCS;
          if (!__all_sync(0xffffffffu, mbar_wait(&tmem_empty[acc], ((drains / ACCS) & 1) ^ 1, abort_flag, p.status, 210))) { ok = false; break; }
          tc_fence_after_sync();
          const uint32_t d_tmem = tmem_base + acc * BN;
          const int end = min(kb + DRAIN, kb1);
          for (int k = kb; k < end; ++k, it += 2) {
            const int s = it % HALVES;                                       // (even: HALVES is)
            const uint32_t ph = (it / HALVES) & 1;
            if (!__all_sync(0xffffffffu, mbar_wait(&full_bar[s], ph, abort_flag, p.status, 211) &&
                                             mbar_wait(&full_bar[s + 1], ph, abort_flag, p.status, 212))) { ok = false; break; }
            tc_fence_after_sync();
            const uint32_t x_addr = smem_u32(smem + s * HALF_BYTES), y_addr = x_addr + HALF_BYTES;
            const uint64_t a_hi = make_smem_desc(x_addr, 16, 1024), b_hi = b_desc(x_addr + A_BYTES);
            const uint64_t a_lo = make_smem_desc(y_addr, 16, 1024), b_lo = b_desc(y_addr + A_BYTES);
            if (elect_one()) {
              multiply(d_tmem, a_hi, b_lo, k == kb);
              multiply(d_tmem, a_lo, b_hi, false);
              commit(&empty_bar[s + 1]);
              multiply(d_tmem, a_hi, b_hi, false);
              commit(&empty_bar[s]);
            }
            __syncwarp();
          }
          if (ok) {
            if (elect_one()) commit(&tmem_full[acc]);
            __syncwarp();
          }
        }
      }
      if (!ok && lane == 0) give_up();
      __syncwarp();
    }
    if constexpr (KIND == SPLIT) {                       // (the epilogue's three barriers, see there)
      tc_fence_before_sync();
      __syncthreads();
      g2::cluster_sync_all();
      g2::cluster_sync_all();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
    // =========================== epilogue: 8 warps, 32 rows x BN / 2 columns each ===========================
    const int q = warp & 3, half = (warp - 4) >> 2;
    uint8_t* slab = smem + SLAB_OFFSET + (warp - 4) * CHUNK_BYTES;
    const Epilogue<MODE> epi(p);
    const uint32_t empty0 = KIND == PAIR ? g2::map_to_cta(smem_u32(&tmem_empty[0]), 0) : 0u;
    uint32_t drains = 0;
    bool ok = true;
    for (long long t = first; t < total; t += stride) {
      int mi, ni, z;
      decode(t, mi, ni, z);
      const int row0 = mi * TM + row_in_tile + q * 32, col0 = ni * BN + half * (BN / 2);
      float v[CHUNKS][32];
#pragma unroll
      for (int h = 0; h < CHUNKS; ++h)
#pragma unroll
        for (int j = 0; j < 32; ++j) v[h][j] = 0.f;
      float4 in[8];
      if constexpr (KIND != SPLIT)
        for (int h = 0; h < CHUNKS; ++h) epi.prefetch(z, row0, col0 + h * 32);
      for (int kb = kb0; kb < kb1; kb += DRAIN, ++drains) {
        const uint32_t acc = drains % ACCS;
        if (!__all_sync(0xffffffffu, mbar_wait(&tmem_full[acc], (drains / ACCS) & 1, abort_flag, p.status, 310))) { ok = false; break; }
        tc_fence_after_sync();
        const uint32_t at = tmem_base + ((uint32_t)(q * 32) << 16) + acc * BN + half * (BN / 2);
        if (kb + DRAIN >= kb1 && KIND != SPLIT) epi.fetch(in, z, row0, col0);
#pragma unroll
        for (int h = 0; h < CHUNKS; ++h) {
          uint32_t r[32];
          tmem_ld_32x32b_x32(at + 32 * h, r);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 32; ++j) v[h][j] += __uint_as_float(r[j]);
        }
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) {
          if constexpr (KIND == PAIR) g2::mbar_arrive_cluster(empty0 + acc * 8);
          else mbar_arrive(&tmem_empty[acc]);
        }
      }
      if (!ok) {
        if (lane == 0) give_up();
        break;
      }
#pragma unroll
      for (int h = 0; h < CHUNKS; ++h) {
        // a part of the contraction waits in this CTA's ring, which all products have been read from by now
        uint8_t* at = KIND == SPLIT ? smem + ((warp - 4) * CHUNKS + h) * CHUNK_BYTES : slab;
        __syncwarp();                                   // (the chunk before has been read)
#pragma unroll
        for (int u = 0; u < 8; ++u)
          *reinterpret_cast<float4*>(at + chunk_at(lane, u)) = make_float4(v[h][4 * u], v[h][4 * u + 1], v[h][4 * u + 2], v[h][4 * u + 3]);
        __syncwarp();
        if constexpr (KIND != SPLIT) {
          float4 acc[8];
          float4 now[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) { acc[i] = *reinterpret_cast<const float4*>(slab + chunk_at(4 * i + (lane >> 3), lane & 7)); now[i] = in[i]; }
          if (h + 1 < CHUNKS) epi.fetch(in, z, row0, col0 + (h + 1) * 32);
          epi.run(acc, now, slab, z, row0, col0 + h * 32);
        }
      }
    }
    if constexpr (KIND == SPLIT) {
      // the parts of a tile meet: rank k adds up chunks k, k + splits, .., one warp each at a time, its own part first and
      // the others' in turn (a fixed order for every chunk, and not all ranks at one CTA's shared memory)
      tc_fence_before_sync();
      __syncthreads();
      g2::cluster_sync_all();
      if (!*abort_flag) {
        int mi, ni, z;
        decode(first, mi, ni, z);
        for (int c = rank + (warp - 4) * splits; c < 8 * CHUNKS; c += 8 * splits) {
          __syncwarp();
          const int w = c / CHUNKS;                      // the warp whose chunk this was, and where its rows and columns are
          const int row0 = mi * BM + (w & 3) * 32, col0 = ni * BN + (w >> 2) * (BN / 2) + (c % CHUNKS) * 32;
          float4 in[8];
          epi.fetch(in, z, row0, col0);
          float4 sum[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) sum[i] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
          for (int k = 0; k < splits; ++k) {
            const uint32_t peer = g2::map_to_cta(smem_u32(smem) + c * CHUNK_BYTES, (rank + k) & (splits - 1));
            float4 o[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i] = ld_peer(peer + chunk_at(4 * i + (lane >> 3), lane & 7));
#pragma unroll
            for (int i = 0; i < 8; ++i) { sum[i].x += o[i].x; sum[i].y += o[i].y; sum[i].z += o[i].z; sum[i].w += o[i].w; }
          }
          epi.run(sum, in, slab, z, row0, col0);
        }
      }
      g2::cluster_sync_all();                            // nobody leaves while its part may still be read
    }
  }

  tc_fence_before_sync();
  __syncthreads();
  if constexpr (KIND == PAIR) g2::cluster_sync_all();    // nobody leaves (or frees tensor memory) while the other may still signal it
  if (warp == 1) {
    tc_fence_after_sync();
    if constexpr (KIND == PAIR) g2::tmem_dealloc2(tmem_base, 512);
    else tmem_dealloc(tmem_base, 512);
  }
}

// B = b A + c A A for m <= 128, and often A = X X^T before it, in one launch: one CTA per matrix, A in its shared memory.  Launched one
// by one the two take 8 us each, of which the products are one or two.  Three slots hold terms, [two halves of the columns][hi, lo]
// [128 rows of 128 bytes], swizzled as the tensor cores read them: blocks of X in turn, then A in the first.  A thread keeps a
// quarter of a row of A in 32 bits in registers.  Rows and columns past m are zero throughout.
constexpr int GRAM_THREADS = 512;
constexpr int GRAM_SLOT = 4 * 128 * 128;
constexpr int GRAM_BARRIERS = 3 * GRAM_SLOT;
constexpr int GRAM_SMEM = GRAM_BARRIERS + 64;

struct Gram {
  int* status;
  int m, batch, lda;
  int blocks;                  // X in blocks of 128 columns, from which A is formed here; 0: A is there
  float gram, gram_scale;      // A = gram X X^T, 2^k of its terms
  float b_acc, b_a, b_scale;   // B = b_acc A A + b_a A, 2^k of its terms
  const float* a;              // A in 32 bits (slot 0)
  __half* b;                   // terms of B [batch][hi, lo][m][lda]
};

__global__ void __launch_bounds__(GRAM_THREADS, 1)
ns_gram_kernel(const __grid_constant__ CUtensorMap tmapA, const __grid_constant__ CUtensorMap tmapX,
                const __grid_constant__ Gram p) {
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* loaded = reinterpret_cast<uint64_t*>(smem + GRAM_BARRIERS);
  uint64_t* done = loaded + 3;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int z = blockIdx.x;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 5; ++i) mbar_init(&loaded[i], 1);
    const bool aligned = (smem_u32(smem) & 1023) == 0;
    if (!aligned) report_error(p.status, GB_ERR_BAD_ARG, 6, 0);
    *abort_flag = !aligned || status_poisoned(p.status) ? 1 : 0;
    mbar_fence_init();
    tma_prefetch_desc(p.blocks > 0 ? &tmapX : &tmapA);
  }
  if (warp == 0) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  const bool work = *abort_flag == 0;
  let_next_start();
  wait_for_previous();

  const int row = (warp & 3) * 32 + lane, col0 = (warp >> 2) * 32;       // this thread's part of a row
  float whole[32];
  const uint32_t idesc = make_idesc(0u, 0u, 0u, 128, 128);
  uint32_t phase = 0;                                    // of done[0]
  bool ok = work;
  // accumulators `buf` = S S^T for a slot S, by warp 0 (A is its own transpose)
  auto issue = [&](const uint8_t* slot, int buf) {
    const uint64_t l = make_smem_desc(smem_u32(slot), 16, 1024), r = l;
    const uint32_t acc = tmem + buf * 256;
    if (elect_one()) {
      // the small products and half of the large ones in one accumulator, the others in a second one
      constexpr uint64_t LO = 1024;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint64_t at = (uint64_t)((k >> 2) * 2048 + (k & 3) * 2);      // (16-byte units; 32 KB a half)
        umma_f16(acc, l + at, r + at + LO, idesc, k == 0 ? 0u : 1u);
        umma_f16(acc, l + at + LO, r + at, idesc, 1u);
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint64_t at = (uint64_t)((k >> 2) * 2048 + (k & 3) * 2);
        umma_f16(acc + (k >> 2) * 128, l + at, r + at, idesc, k == 4 ? 0u : 1u);
      }
      umma_commit(&done[buf]);
    }
    __syncwarp();
  };
  // the thread's part of accumulators `buf`
  auto take = [&](float (&r)[32], int buf) {
    uint32_t a[32], b[32];
    const uint32_t at = tmem + buf * 256 + ((uint32_t)((warp & 3) * 32) << 16) + col0;
    tmem_ld_32x32b_x32(at, a);
    tmem_ld_32x32b_x32(at + 128, b);
    tmem_ld_wait();
#pragma unroll
    for (int j = 0; j < 32; ++j) r[j] = __uint_as_float(a[j]) + __uint_as_float(b[j]);
  };
  // the terms of 8 columns from 8 u on of the thread's part of a row, as they lie in memory: hi, lo
  auto terms = [&](const float (&v)[32], int u, float scale, uint4& hi, uint4& lo) {
    const uint4 s = split4(v[8 * u] * scale, v[8 * u + 1] * scale, v[8 * u + 2] * scale, v[8 * u + 3] * scale);
    const uint4 t = split4(v[8 * u + 4] * scale, v[8 * u + 5] * scale, v[8 * u + 6] * scale, v[8 * u + 7] * scale);
    hi = make_uint4(s.x, s.y, t.x, t.y);
    lo = make_uint4(s.z, s.w, t.z, t.w);
  };
  if (p.blocks > 0) {
    // A = X X^T: the slots are a ring of blocks of X; while one is multiplied, the products of the last are added up
    auto load = [&](int d) {
      const int i = d % 3;
      mbar_expect_tx(&loaded[i], GRAM_SLOT);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        tma_load_3d(smem + i * GRAM_SLOT + k * 16384, &tmapX, &loaded[i], d * 128 + (k >> 1) * 64, 0, 2 * z + (k & 1));
    };
    int issued = 0;
    if (work && threadIdx.x == 0)
      for (; issued < 3 && issued < p.blocks; ++issued) load(issued);
#pragma unroll
    for (int j = 0; j < 32; ++j) whole[j] = 0.f;
    for (int d = 0; d <= p.blocks; ++d) {
      if (warp == 0 && d < p.blocks && ok) {
        ok = __all_sync(0xffffffffu, mbar_wait(&loaded[d % 3], (d / 3) & 1, abort_flag, p.status, 411));
        if (ok) issue(smem + d % 3 * GRAM_SLOT, d & 1);
      }
      if (d > 0) {
        const int e = d - 1;
        if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&done[e & 1], (e >> 1) & 1, abort_flag, p.status, 412));
        if (ok) {
          if (threadIdx.x == 0 && issued < p.blocks) load(issued++);      // into the slot that block e has left
          __syncwarp();
          tc_fence_after_sync();
          float r[32];
          take(r, e & 1);
#pragma unroll
          for (int j = 0; j < 32; ++j) whole[j] += r[j];
          tc_fence_before_sync();
        }
      }
      ok = __syncthreads_and(ok);
      tc_fence_after_sync();
      if (!ok) break;
    }
    if (work && !ok && threadIdx.x == 0) drain_copies(loaded, 3, issued);
    phase = ((p.blocks + 1) / 2) & 1;
#pragma unroll
    for (int j = 0; j < 32; ++j) whole[j] *= p.gram;
    // A's terms into the first slot: every product has been waited for
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      uint4 hi, lo;
      terms(whole, u, p.gram_scale, hi, lo);
      uint8_t* at = smem + (warp >> 3) * 32768 + row * 128 + ((((warp >> 2) & 1) * 4 + u) ^ (row & 7)) * 16;
      *reinterpret_cast<uint4*>(at) = hi;
      *reinterpret_cast<uint4*>(at + 16384) = lo;
    }
  } else {
    if (work && threadIdx.x == 0) {
      mbar_expect_tx(loaded, GRAM_SLOT);
#pragma unroll
      for (int i = 0; i < 4; ++i) tma_load_3d(smem + i * 16384, &tmapA, loaded, (i >> 1) * 64, 0, 2 * z + (i & 1));
    }
    const float* a = p.a + ((size_t)z * p.m + row) * p.lda + col0;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const float4 v = row < p.m && col0 + 4 * u < p.m ? *reinterpret_cast<const float4*>(a + 4 * u) : make_float4(0.f, 0.f, 0.f, 0.f);
      // (elements of the last vector past m are padding, whatever it holds)
      whole[4 * u] = v.x;
      whole[4 * u + 1] = col0 + 4 * u + 1 < p.m ? v.y : 0.f;
      whole[4 * u + 2] = col0 + 4 * u + 2 < p.m ? v.z : 0.f;
      whole[4 * u + 3] = col0 + 4 * u + 3 < p.m ? v.w : 0.f;
    }
    if (ok) ok = mbar_wait(loaded, 0, abort_flag, p.status, 413);
    ok = __syncthreads_and(ok);
    if (work && !ok && threadIdx.x == 0) drain_copies(loaded, 1, 1);
  }
  fence_proxy_async_smem();
  tc_fence_before_sync();
  __syncthreads();                                       // A is there, the last accumulator has been read
  tc_fence_after_sync();
  if (warp == 0 && ok) issue(smem, 0);
  if (ok) ok = mbar_wait(&done[0], phase, abort_flag, p.status, 410);
  ok = __syncthreads_and(ok);
  tc_fence_after_sync();
  float r[32];
  take(r, 0);
#pragma unroll
  for (int j = 0; j < 32; ++j) whole[j] = fmaf(r[j], p.b_acc, whole[j] * p.b_a);
  if (ok && row < p.m) {
    __half* b = p.b + ((size_t)z * 2 * p.m + row) * p.lda + col0;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (col0 + 8 * u < p.m) {                          // (elements of the last vector past m are zero, and padding)
        uint4 hi, lo;
        terms(whole, u, p.b_scale, hi, lo);
        *reinterpret_cast<uint4*>(b + 8 * u) = hi;
        *reinterpret_cast<uint4*>(b + (size_t)p.m * p.lda + 8 * u) = lo;
      }
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, 512);
  }
}

__device__ __forceinline__ double block_sum256(double v, double* sh) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.0;
#pragma unroll
  for (int i = 0; i < 8; ++i) v += sh[i];
  return v;
}

__device__ __forceinline__ float4 load4(const void* p, int dt, size_t i) {
  if (dt == DT_F32) return *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + i);
  const uint2 w = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(p) + i);
  return make_float4(half_bits_to_float((uint16_t)w.x, dt), half_bits_to_float((uint16_t)(w.x >> 16), dt),
                     half_bits_to_float((uint16_t)w.y, dt), half_bits_to_float((uint16_t)(w.y >> 16), dt));
}
__device__ __forceinline__ bool aligned4(const void* p, int dt) {
  return (reinterpret_cast<uintptr_t>(p) & (dt == DT_F32 ? 15 : 7)) == 0;
}
// (the squares in 64 bits: 32 would overflow or vanish at half the exponent range of the elements)
__device__ __forceinline__ double square4(float4 v) {
  return ((double)v.x * v.x + (double)v.y * v.y) + ((double)v.z * v.z + (double)v.w * v.w);
}

// Partial sums of squares of every matrix: gridDim.x of them, in an order that depends on the sizes alone
__global__ void __launch_bounds__(256)
ns_norm_kernel(const void* __restrict__ src, int dt, long long numel, double* __restrict__ partial) {
  __shared__ double sh[8];
  const void* p = reinterpret_cast<const uint8_t*>(src) + (size_t)blockIdx.y * numel * (dt == DT_F32 ? 4 : 2);
  const long long step = 256ll * gridDim.x, me = (long long)blockIdx.x * 256 + threadIdx.x;
  double s = 0.0;
  const long long nv = aligned4(p, dt) ? numel / 4 : 0;
  long long i = me;
  for (; i + 3 * step < nv; i += 4 * step) {
    float4 v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = load4(p, dt, 4 * (i + k * step));
#pragma unroll
    for (int k = 0; k < 4; ++k) s += square4(v[k]);
  }
  for (; i < nv; i += step) s += square4(load4(p, dt, 4 * i));
  for (i = 4 * nv + me; i < numel; i += step) {
    const double x = (double)load_as_float(p, dt, i);
    s += x * x;
  }
  s = block_sum256(s, sh);
  if (threadIdx.x == 0) partial[blockIdx.y * PARTS + blockIdx.x] = s;
}

// Momentum of every matrix of a batch and the update that goes on to the iteration:
//   u <- mu u + nu g,   y = mu u + nu g (Nesterov) or u,   nu = 1 - mu, formed in 64 bits: from mu rounded to 32 it would be
// 2.4e-7 of itself off at mu = 0.9 or 0.95, and with it every momentum
// table: addresses of gradients, then of momenta [2, batch]; y [batch, numel], and the partial sums of its squares.
__global__ void __launch_bounds__(256)
muon_momentum_kernel(const long long* __restrict__ table, int batch, int grad_dt, long long numel, float mu, float nu, int nesterov,
                     const float* __restrict__ grad_scale, const float* __restrict__ found_inf, float* __restrict__ y,
                     double* __restrict__ partial) {
  __shared__ double sh[8];
  const int z = blockIdx.y;
  const void* g = reinterpret_cast<const void*>(table[z]);
  float* u = reinterpret_cast<float*>(table[batch + z]);
  float* yz = y + (size_t)z * numel;
  const float gs = grad_scale != nullptr ? *grad_scale : 1.f;
  const bool skip = found_inf != nullptr && *found_inf != 0.f;      // the step is cancelled: momentum stays as it is
  double s = 0.0;
  const long long step = 256ll * gridDim.x, me = (long long)blockIdx.x * 256 + threadIdx.x;
  auto update = [&](float g1, float& u1) {
    const float gi = g1 * gs;
    u1 = mu * u1 + nu * gi;
    return nesterov ? mu * u1 + nu * gi : u1;
  };
  const bool vec = aligned4(g, grad_dt) && ((reinterpret_cast<uintptr_t>(u) | reinterpret_cast<uintptr_t>(yz)) & 15) == 0;
  const long long nv = skip ? 0 : (vec ? numel / 4 : 0), n = skip ? 0 : numel;
  auto four = [&](float4 gv, float4 uv, long long i) {
    float4 o;
    o.x = update(gv.x, uv.x); o.y = update(gv.y, uv.y); o.z = update(gv.z, uv.z); o.w = update(gv.w, uv.w);
    *reinterpret_cast<float4*>(u + 4 * i) = uv;
    *reinterpret_cast<float4*>(yz + 4 * i) = o;
    s += square4(o);
  };
  long long i = me;
  for (; i + step < nv; i += 2 * step) {
    const float4 g0 = load4(g, grad_dt, 4 * i), g1 = load4(g, grad_dt, 4 * (i + step));
    const float4 u0 = *reinterpret_cast<const float4*>(u + 4 * i), u1 = *reinterpret_cast<const float4*>(u + 4 * (i + step));
    four(g0, u0, i);
    four(g1, u1, i + step);
  }
  if (i < nv) four(load4(g, grad_dt, 4 * i), *reinterpret_cast<const float4*>(u + 4 * i), i);
  for (i = 4 * nv + me; i < n; i += step) {
    float ui = u[i];
    const float yi = update(load_as_float(g, grad_dt, i), ui);
    u[i] = ui;
    yz[i] = yi;
    s += (double)yi * (double)yi;
  }
  s = block_sum256(s, sh);
  if (threadIdx.x == 0) partial[z * PARTS + blockIdx.x] = s;
}

// X = G / (|G| + eps), in 32 bits and as fp16 terms; a tall G [n, m] is transposed on the way.  A block: 32 x 128 of X.
__global__ void __launch_bounds__(256)
ns_prepare_kernel(const void* __restrict__ src, int dt, int m, int n, int tall, const long long* __restrict__ weights,
                  const double* __restrict__ partial, int parts, double eps, float scale, float* __restrict__ x,
                  __half* __restrict__ planes, int ldx) {
  __shared__ float tile[128][33];
  __shared__ double sh[8];
  const int z = blockIdx.z, i0 = blockIdx.y * 32, j0 = blockIdx.x * 128;
  let_next_start();
  wait_for_previous();
  const double inv = 1.0 / (sqrt(block_sum256((int)threadIdx.x < parts ? partial[z * PARTS + threadIdx.x] : 0.0, sh)) + eps);
  const void* g = reinterpret_cast<const uint8_t*>(src) + (size_t)z * m * n * (dt == DT_F32 ? 4 : 2);
  if (weights != nullptr) tall = (int)(weights[z] & 1);
  const size_t plane = (size_t)m * ldx;
  float* xz = x + (size_t)z * plane;
  __half* hi = planes + (size_t)z * 2 * plane;
  const int u = threadIdx.x & 31, w = threadIdx.x >> 5;
  auto put = [&](int i, int j, float4 v) {               // (the pitch is a multiple of 8: four elements stay inside it)
    const size_t o = (size_t)i * ldx + j;
    *reinterpret_cast<float4*>(xz + o) = v;
    const uint4 t = split4(v.x * scale, v.y * scale, v.z * scale, v.w * scale);
    *reinterpret_cast<uint2*>(hi + o) = make_uint2(t.x, t.y);
    *reinterpret_cast<uint2*>(hi + plane + o) = make_uint2(t.z, t.w);
  };
  auto norm = [&](float a) { return (float)((double)a * inv); };
  if (!tall) {
    const bool vec = (n & 3) == 0 && aligned4(g, dt);
    const int j = j0 + 4 * u;
    float4 v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = i0 + w + 8 * k;
      v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (i < m && j < n) {
        const size_t o = (size_t)i * n + j;
        if (vec) v[k] = load4(g, dt, o);
        else {
          v[k].x = load_as_float(g, dt, o);
          if (j + 1 < n) v[k].y = load_as_float(g, dt, o + 1);
          if (j + 2 < n) v[k].z = load_as_float(g, dt, o + 2);
          if (j + 3 < n) v[k].w = load_as_float(g, dt, o + 3);
        }
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = i0 + w + 8 * k;
      if (i < m && j < n) put(i, j, make_float4(norm(v[k].x), norm(v[k].y), norm(v[k].z), norm(v[k].w)));
    }
  } else {
    float v[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      const int j = j0 + w + 8 * k, i = i0 + u;
      v[k] = i < m && j < n ? load_as_float(g, dt, (size_t)j * m + i) : 0.f;
    }
#pragma unroll
    for (int k = 0; k < 16; ++k) tile[w + 8 * k][u] = v[k];
    __syncthreads();
    const int j = j0 + 4 * u;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int r = w + 8 * k, i = i0 + r;
      if (i < m && j < n)
        put(i, j, make_float4(norm(tile[4 * u][r]), norm(tile[4 * u + 1][r]), norm(tile[4 * u + 2][r]), norm(tile[4 * u + 3][r])));
    }
  }
}

// How many partial sums a matrix gets: 16 K elements each, up to 256
static inline int norm_parts(long long numel) {
  const long long p = (numel + 16383) / 16384;
  return (int)(p < PARTS ? p : PARTS);
}

template <int MODE, int BN, int KIND>
static int launch(const CUtensorMap& ta, const CUtensorMap& tb, const Params& p, int grid, cudaStream_t st) {
  static unsigned long long configured = 0;
  if (int r = smem_opt_in(ns_product_kernel<MODE, BN, KIND>, SMEM_TOTAL, configured)) return r;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = KIND == PAIR ? 2 : p.splits; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
  cfg.gridDim = dim3((unsigned)grid); cfg.blockDim = dim3(THREADS); cfg.dynamicSmemBytes = SMEM_TOTAL; cfg.stream = st;
  cfg.attrs = attr; cfg.numAttrs = KIND == WHOLE ? 1 : 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, ns_product_kernel<MODE, BN, KIND>, ta, tb, p);
  return e == cudaSuccess ? (int)cudaGetLastError() : (int)e;
}

// How many clusters of 2, 4, 8 CTAs of this size the device holds at once: a cluster stays inside one group of SMs, and
// groups differ in size, so it is less than the number of SMs allows (asked for once per device).
static int max_clusters(int size) {
  static int known[64][4] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  int& n = known[dev & 63][size == 2 ? 1 : size == 4 ? 2 : 3];
  if (n == 0) {
    auto kern = ns_product_kernel<SYM, 128, SPLIT>;
    static unsigned long long configured = 0;
    if (smem_opt_in(kern, SMEM_TOTAL, configured)) return 1;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = size; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3(size); cfg.blockDim = dim3(THREADS); cfg.dynamicSmemBytes = SMEM_TOTAL; cfg.attrs = attr; cfg.numAttrs = 1;
    int got = 0;
    if (cudaOccupancyMaxActiveClusters(&got, kern, &cfg) != cudaSuccess || got < 1) { cudaGetLastError(); got = 1; }
    n = got;
  }
  return n;
}

// How a product is worked on: tiles of 128 x 128 or 128 x 256, whole or shared by the CTAs of a cluster, or of 256 x 256 on
// pairs: whatever has the fewest clocks on its longest CTA.  A block of the contraction takes 1080 clocks with 128 columns and
// 1700 with 256, bound by shared memory (213 and 160 bytes a clock at the full tensor rate, of 128), or 2100 where all SMs
// together read more than L2 gives (11 TB/s); pairs read two thirds of that and take 1600.  The epilogue of the last tile,
// which no products hide, takes 6500 for each chunk of a warp; the parts of a cluster 4000 to meet and 5000 a chunk.
struct Plan { int kind, bn, splits, grid; long long clocks; };
static Plan plan(bool sym, int m, int n, int k, long long matrices) {
  const long long sms = sm_count(), kblocks = (k + BK - 1) / BK;
  Plan best{WHOLE, 128, 1, 0, -1};
  auto offer = [&](long long clocks, int kind, int width, int splits, long long ctas) {
    if (best.clocks < 0 || clocks < best.clocks) best = Plan{kind, width, splits, (int)ctas, clocks};
  };
  for (int width = 128; width <= 256; width += 128) {
    const long long total = tiles_of(sym, m, n, BM, width) * matrices, waves = (total + sms - 1) / sms;
    const long long block = width == 128 ? 1080 : total >= sms ? 2100 : 1700, chunks = width / 64;
    offer(waves * kblocks * block + chunks * 6500, WHOLE, width, 1, total < sms ? total : sms);
    for (int s = 2; s <= 8 && kblocks >= 2 * s && total <= max_clusters(s); s *= 2)      // (one tile each: a single wave)
      offer((kblocks + s - 1) / s * (width == 128 ? 1080 : 1700) + (chunks + s - 1) / s * 5000 + 4000, SPLIT, width, s, total * s);
  }
  const long long pairs = tiles_of(sym, m, n, 2 * BM, 256) * matrices, at_once = max_clusters(2);
  offer((pairs + at_once - 1) / at_once * kblocks * 1600 + 4 * 6500, PAIR, 256, 1, 2 * (pairs < at_once ? pairs : at_once));
  return best;
}

template <int MODE>
static int product(const CUtensorMap& ta, const CUtensorMap& tb, Params p, cudaStream_t st) {
  const Plan c = plan(MODE == SYM, p.m, p.n, p.k, (long long)p.batch * p.problems);
  p.splits = c.splits;
  if (c.kind == PAIR) return launch<MODE, 256, PAIR>(ta, tb, p, c.grid, st);
  if (c.kind == SPLIT)
    return c.bn == 256 ? launch<MODE, 256, SPLIT>(ta, tb, p, c.grid, st) : launch<MODE, 128, SPLIT>(ta, tb, p, c.grid, st);
  return c.bn == 256 ? launch<MODE, 256, WHOLE>(ta, tb, p, c.grid, st) : launch<MODE, 128, WHOLE>(ta, tb, p, c.grid, st);
}

// The clocks of a program's products (see gb_newton_schulz), each a launch with 10000 to start and to end.
static long long clocks(const double* program, int count, int m, int n, int batch) {
  long long total = 0;
  for (int i = 0; i < count; ++i) {
    const int kind = (int)program[12 * i], problems = kind == 2 && i + 1 < count ? 2 : 1;
    total += plan(kind != 3, m, n, kind == 0 ? n : m, (long long)batch * problems).clocks + 10000;
    i += problems - 1;
  }
  return total;
}

// Whether steps are made one by one, not in blocks.  One by one they are as exact as 32-bit products: X X^T is formed anew for each.
// In blocks it is carried on, and its roundings with it.  Error over that of 32-bit products, one by one / in blocks, for gradients of
// a few strong directions over small ones and for Gaussian matrices: 16 x 5000 1.0 / 5.1 and 1.2 / 2.6, 128 x 896 1.0 / 1.7 and 1.0 / 4.5,
// batches of 200 x 3000 1.0 / 1.7 and 0.9 / 3.6, of 320 x 2000 0.9 / 1.2 and 1.0 / 5.1, of 512 x 2048 0.7 / 0.9 and 1.1 / 4.4, of 896 x 4864
// 0.5 / 0.6 and 0.9 / 3.1 (1.2e-5 of the norm).  So blocks are for more than 320 rows, and where they save a tenth of the time:
// long or many matrices, where operations count.  One by one / in blocks, us: 128 x 896 124 / 83, 256 x 1024 154 / 175, 64 of them
// 521 / 440, 896 x 896 200 / 219, eight of them 506 / 608, 896 x 4864 316 / 272, 24 of them 4810 / 3242.
static bool one_by_one(const double* blocks, int blocks_count, const double* single, int single_count, int m, int n, int batch) {
  return m <= 320 || clocks(single, single_count, m, n, batch) * 9 <= clocks(blocks, blocks_count, m, n, batch) * 10;
}

// Whether ns_gram_kernel forms A = X X^T itself: its one CTA takes 2700 clocks for 128 columns of X; a launch of its own 1080
// for 64 of them, shared by as many CTAs as there are SMs to a matrix, 8 at most, and 21000 besides (its start, the parts' meeting
// and A's way through memory).  Five steps, own launch / here, us: 128 x 128 128 / 85, 128 x 896 140 / 124, 128 x 2048 145 / 184,
// 100 of 128 x 4864 1316 / 1253.
static bool folds(int n, int batch) {
  const long long kblocks = (n + BK - 1) / BK;
  int s = 1;
  while (s < 8 && kblocks >= 4 * s && (long long)batch * s * 2 <= sm_count()) s *= 2;
  return (n + 127) / 128 * 2700ll <= kblocks * 1080 / s + 21000;
}

static int gram(const CUtensorMap& ta, const CUtensorMap& tx, const Gram& c, cudaStream_t st) {
  static unsigned long long configured = 0;
  if (int r = smem_opt_in(ns_gram_kernel, GRAM_SMEM, configured)) return r;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3((unsigned)c.batch); cfg.blockDim = dim3(GRAM_THREADS); cfg.dynamicSmemBytes = GRAM_SMEM; cfg.stream = st;
  cfg.attrs = attr; cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, ns_gram_kernel, ta, tx, c);
  return e == cudaSuccess ? (int)cudaGetLastError() : (int)e;
}

static inline long long up256(long long b) { return (b + 255) & ~255ll; }

struct Workspace {
  double* partial; float* y; float* x; __half* xp[2]; __half* terms; float* whole;
  long long bytes;
  Workspace(uint8_t* base, long long m, long long n, long long batch, bool with_y) {
    const long long ldx = (n + 7) & ~7ll, lda = (m + 7) & ~7ll;
    long long at = 0;
    auto take = [&](long long b) { uint8_t* p = base + at; at += up256(b); return p; };
    partial = (double*)take(batch * PARTS * 8);
    y = (float*)take(with_y ? batch * m * n * 4 : 0);
    x = (float*)take(batch * m * ldx * 4);
    xp[0] = (__half*)take(batch * m * ldx * 4);
    xp[1] = (__half*)take(batch * m * ldx * 4);
    terms = (__half*)take(SLOTS * batch * m * lda * 4);
    whole = (float*)take(SLOTS * batch * m * lda * 4);
    bytes = at;
  }
};

}  // namespace ns
}  // namespace gb

using namespace gb;

// Bytes of workspace that `batch` matrices m x n, m <= n, need (with_y: an optimizer step, which keeps its updates there)
extern "C" int gb_ns_workspace(long long m, long long n, long long batch, int with_y, long long* bytes) {
  *bytes = ns::Workspace(nullptr, m, n, batch, with_y != 0).bytes;
  return 0;
}

// What `plan` chooses on this device for a product with a contraction of k, in which `problems` results are wanted of each of
// `batch` matrices [m, n]: kind (0 whole tiles, 1 shared by a cluster, 2 CTA pairs), columns of a tile, CTAs that share one
extern "C" int gb_ns_plan(int sym, int m, int n, int k, int batch, int problems, int* out) {
  if (m < 1 || n < m || k < 1 || batch < 1 || problems < 1) return -3;
  const ns::Plan c = ns::plan(sym != 0, m, n, k, (long long)batch * problems);
  out[0] = c.kind; out[1] = c.bn; out[2] = c.splits;
  return 0;
}

// Whether gb_newton_schulz takes the second program
extern "C" int gb_ns_one_by_one(const double* blocks, int blocks_count, const double* single, int single_count, int m, int n,
                                int batch) {
  return ns::one_by_one(blocks, blocks_count, single, single_count, m, n, batch) ? 1 : 0;
}

// First half of an optimizer step: see muon_momentum_kernel.  The update and its partial sums stay in the workspace.
extern "C" int gb_muon_momentum(const long long* table, int batch, int grad_dt, int m, int n, double mu, int nesterov,
                                const float* grad_scale, const float* found_inf, void* workspace, cudaStream_t st) {
  if (batch <= 0 || m <= 0 || n <= 0) return 0;
  if (batch > 32767 || m > n || n > (1 << 30)) return -3;
  const ns::Workspace w((uint8_t*)workspace, m, n, batch, true);
  const long long numel = (long long)m * n;
  ns::muon_momentum_kernel<<<dim3(ns::norm_parts(numel), batch), 256, 0, st>>>(table, batch, grad_dt, numel, (float)mu, (float)(1.0 - mu), nesterov,
                                                                               grad_scale, found_inf, w.y, w.partial);
  return (int)cudaGetLastError();
}

// Orthogonalises `batch` matrices [m, n], or [n, m] (tall), m <= n.  `src` (contiguous, dtype dt) with `out` of the same type;
// or src null for the updates that gb_muon_momentum has left in the workspace, which go into the weights whose addresses
// `weights` [batch] holds (+ 1 for a tall one).
// The products to be made are rows of 12 numbers, in two programs for the same steps: `blocks` of steps, and steps `single`, one by
// one, which are taken where one_by_one says so, and always for m <= 128.  A row: kind (0 X X^T, 1 symmetric, 2 the same and to be
// launched together with the next row, 3 X <- Q X + ..), left, right and out slots, M1 and M2 slots or -1, whether the result
// is kept in 32 bits, f_acc, f1, f2, the power of two of the result's terms, 0.  The first row's last number: the power of
// two of the first X's terms.  The last row is of kind 3.
extern "C" int gb_newton_schulz(const void* src, void* out, int dt, int m, int n, int tall, int batch, const double* blocks,
                                int blocks_count, const double* single, int single_count, double eps, const long long* weights, float lr, float decay, float tall_scale,
                                const float* dyn_lr, const float* found_inf, void* workspace, int* status, cudaStream_t st) {
  if (batch <= 0 || m <= 0 || n <= 0) return 0;
  if (batch > 6000 || m > n || n > (1 << 30) || blocks_count < 2 || single_count < 2 || (src == nullptr) != (weights != nullptr) ||
      (reinterpret_cast<uintptr_t>(workspace) & 255) != 0) return -3;
  const bool one = ns::one_by_one(blocks, blocks_count, single, single_count, m, n, batch);
  const double* program = one ? single : blocks;
  const int count = one ? single_count : blocks_count;
  const int ldx = (n + 7) & ~7, lda = (m + 7) & ~7;
  const ns::Workspace w((uint8_t*)workspace, m, n, batch, src == nullptr);
  const int parts = ns::norm_parts((long long)m * n);
  const dim3 grid((n + 127) / 128, (m + 31) / 32, batch);
  if (grid.y > 65535) return -3;
  if (src != nullptr) ns::ns_norm_kernel<<<dim3(parts, batch), 256, 0, st>>>(src, dt, (long long)m * n, w.partial);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = grid; cfg.blockDim = dim3(256); cfg.stream = st; cfg.attrs = attr; cfg.numAttrs = 1;
  const void* g = src != nullptr ? src : (const void*)w.y;
  const int g_dt = src != nullptr ? dt : (int)DT_F32;
  if (const cudaError_t e = cudaLaunchKernelEx(&cfg, ns::ns_prepare_kernel, g, g_dt, m, n, tall, weights, (const double*)w.partial,
                                               parts, eps, (float)program[11], w.x, w.xp[0], ldx)) return (int)e;
  // maps: X as left or right operand of X X^T, X as right operand of Q X (64 rows of the contraction at a time), the slots
  CUtensorMap mx[2], mxr[2], ms;
  int r;
  for (int i = 0; i < 2; ++i) {
    if ((r = make_tmap_3d(&mx[i], w.xp[i], DT_F16, n, m, 2ll * batch, ldx, (long long)m * ldx, 128)) != 0) return 10000 + r;
    if ((r = make_tmap_3d(&mxr[i], w.xp[i], DT_F16, n, m, 2ll * batch, ldx, (long long)m * ldx, 64)) != 0) return 20000 + r;
  }
  if ((r = make_tmap_3d(&ms, w.terms, DT_F16, m, m, 2ll * batch * ns::SLOTS, lda, (long long)m * lda, 128)) != 0) return 30000 + r;
  ns::Params p = {};
  p.status = status; p.m = m; p.n = n; p.batch = batch; p.ldx = ldx; p.lda = lda; p.x = w.x; p.terms = w.terms; p.whole = w.whole;
  p.out = out; p.out_dtype = dt; p.tall = tall; p.weights = weights; p.lr = lr; p.decay = decay; p.tall_scale = tall_scale;
  p.dyn_lr = dyn_lr; p.found_inf = found_inf;
  int cur = 0;
  bool fold = false;
  for (int i = 0; i < count; ++i) {
    const int kind = (int)program[12 * i];
    p.problems = kind == 2 && i + 1 < count ? 2 : 1;
    for (int j = 0; j < p.problems; ++j) {
      const double* o = program + 12 * (i + j);
      for (int k = 1; k <= 5; ++k)
        if (!(o[k] >= (k > 3 ? -1 : 0) && o[k] < ns::SLOTS)) return -3;
      p.prob[j] = ns::Problem{(int)o[1], (int)o[2], (int)o[3], (int)o[4], (int)o[5], (int)o[6], (float)o[7], (float)o[8], (float)o[9],
                              (float)o[10]};
    }
    i += p.problems - 1;
    if (kind == 3) {
      p.k = m;
      p.prob[0].right = 0;
      p.dst = w.xp[cur ^ 1];
      r = i + 1 < count ? ns::product<ns::APPLY>(ms, mxr[cur], p, st) : ns::product<ns::APPLY_LAST>(ms, mxr[cur], p, st);
      cur ^= 1;
    } else {
      p.k = kind == 0 ? n : m;
      if (kind == 0) p.prob[0].left = p.prob[0].right = 0;
      fold = kind == 0 && m <= 128 && ns::folds(n, batch);
      r = fold ? 0 : kind == 0 ? ns::product<ns::SYM>(mx[cur], mx[cur], p, st) : ns::product<ns::SYM>(ms, ms, p, st);
    }
    if (r != 0) return r;
    if (kind == 0 && m <= 128) {
      // the next row, B, from A in the same launch, or in one of its own kind
      if (++i >= count || program[12 * i] != 1.0 || program[12 * i + 1] != 0.0 || program[12 * i + 2] != 0.0) return -3;
      const double* o = program + 12 * i;
      if (!(o[3] >= 1 && o[3] < ns::SLOTS)) return -3;
      ns::Gram c = {};
      c.status = status; c.m = m; c.batch = batch; c.lda = lda; c.a = w.whole;
      c.blocks = fold ? (n + 127) / 128 : 0; c.gram = p.prob[0].f_acc; c.gram_scale = p.prob[0].scale;
      c.b_acc = (float)o[7]; c.b_a = (float)o[8]; c.b_scale = (float)o[10];
      c.b = w.terms + (size_t)o[3] * batch * 2 * m * lda;
      if ((r = ns::gram(ms, mx[cur], c, st)) != 0) return r;
    }
  }
  return 0;
}
