// Newton-Schulz orthogonalisation of weight updates: the singular values of a matrix are driven to about one by
//
//   X = G / (|G|_F + eps),   repeated:  A = X X^T,  B = b A + c A A,  X <- a X + B X          (X: m x n, m <= n)
//
// i.e. every singular value s goes to a s + b s^3 + c s^5.  A tall G is handled as its transpose.
//
// Arithmetic.  The iteration amplifies: with the usual coefficients a small singular value grows by a factor of
// 3.44 a step, 485 over five, and so does every rounding of X in its direction.  So X is kept in 32 bits, and enters the
// tensor cores as two fp16 terms, x 2^k = hi + lo, which hold 22 of its 24 bits (k keeps the largest entry near the top
// of fp16's range, so that lo stays clear of its subnormals: |x_ij| is at most the spectral norm, which the host bounds
// from the coefficients).  Each product is three of fp16 with fp32 accumulation, hi hi + hi lo + lo hi; a X is added in
// 32 bits from X itself.  Errors measured against 64 bits (256 x 1024, Gaussian / rank 8 plus noise): 9e-7 / 6e-7, of the
// products in fp32 1.7e-7 / 5.9e-7, with one fp16 term 1.7e-3, with terms but without X in 32 bits 7e-7 / 4e-6.
//
// Work.  A and B are symmetric: only tiles on and below the diagonal are computed, the rest is written as their mirror
// image by the same epilogue.  A step is three launches over all matrices of a batch, 128 x 128 tiles on persistent CTAs:
//   warp 0 TMA producer, warp 1 issues tcgen05.mma, warps 2-9 epilogue; two accumulators in tensor memory.
// A stage holds both terms of both operands for 64 elements of the contraction (64 KB) and feeds three products, so an SM
// reads 85 bytes a clock from L2 at the full tensor rate, as the single-product GEMM with tiles of 128 x 256 does.
#include "sm100_ptx.cuh"
#include "common.cuh"

namespace gb {

int make_tmap_3d(CUtensorMap* out, const void* base, int dtype, long long inner, long long outer, long long batch,
                 long long ld_elems, long long batch_stride_elems, int box_outer);

namespace ns {

constexpr int BM = 128, BN = 128, BK = 64, STAGES = 3;
constexpr int TILE_BYTES = 128 * 128;                 // 128 rows of 64 fp16, or 64 rows of 2 x 64
constexpr int STAGE_BYTES = 4 * TILE_BYTES;           // hi and lo of both operands
constexpr int BARRIER_OFFSET = STAGES * STAGE_BYTES;
constexpr int SMEM_TOTAL = BARRIER_OFFSET + 1024;
constexpr int PARTS = 64;                             // partial sums of squares per matrix
constexpr int ACC_STRIDE = BN;

enum Mode : int { GRAM = 0, SQUARE = 1, APPLY = 2, APPLY_LAST = 3 };

struct Params {
  int* status;
  int m, n, batch;             // X [batch, m, n]
  int ldx, lda;                // pitch of X and of A, B in elements (multiples of 8)
  __half* dst;                 // GRAM: A, SQUARE: B, APPLY: the next X; planes [batch][hi, lo][m][ld]
  const __half* a_planes;      // SQUARE: A
  float* x;                    // APPLY: X in 32 bits [batch][m][ldx]
  float f_acc, f_a;            // result = f_acc * accumulator + f_a * (SQUARE: A as stored; APPLY: X)
  float next_scale;            // APPLY: 2^k of the next X
  // APPLY_LAST: out[batch] in `out_dtype`, or the weights of an optimizer step through `weights`
  void* out;
  int out_dtype, tall;         // tall: the result goes out transposed, [n, m]
  const long long* weights;    // [batch] addresses of fp32 weights, or null
  float lr, decay, scale;      // w <- w (1 - lr decay) - lr scale o
  const float* dyn_lr;
  const float* found_inf;
};

__device__ __forceinline__ void split(float x, __half& hi, __half& lo) {
  hi = __float2half_rn(x);
  lo = __float2half_rn(x - __half2float(hi));
}

template <int MODE>
__global__ void __launch_bounds__(320, 1)
ns_product_kernel(const __grid_constant__ CUtensorMap tmapA, const __grid_constant__ CUtensorMap tmapB, const Params p) {
  constexpr bool SYM = MODE == GRAM || MODE == SQUARE;
  constexpr bool B_MN = !SYM;                           // X as the right operand: its rows run along the contraction
  extern __shared__ __align__(1024) uint8_t smem[];
  if (status_poisoned(p.status)) return;
  if ((reinterpret_cast<uintptr_t>(smem) & 1023) != 0) {
    if (threadIdx.x == 0) report_error(p.status, GB_ERR_BAD_ARG, 5, 0);
    return;
  }
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + BARRIER_OFFSET);
  uint64_t* empty_bar = full_bar + STAGES;
  uint64_t* tmem_full = empty_bar + STAGES;
  uint64_t* tmem_empty = tmem_full + 2;
  uint32_t* tmem_base_slot = reinterpret_cast<uint32_t*>(tmem_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_base_slot + 1);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
  const int lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) { mbar_init(&full_bar[s], 1); mbar_init(&empty_bar[s], 1); }
    for (int a = 0; a < 2; ++a) { mbar_init(&tmem_full[a], 1); mbar_init(&tmem_empty[a], 8); }
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tmapA);
    tma_prefetch_desc(&tmapB);
  }
  if (warp == 1) {
    tmem_alloc(tmem_base_slot, 2 * ACC_STRIDE);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_base_slot;

  const int tm = (p.m + BM - 1) / BM, tn = (p.n + BN - 1) / BN;
  const int per = SYM ? tm * (tm + 1) / 2 : tm * tn;
  const long long total = (long long)per * p.batch;
  const int K = MODE == GRAM ? p.n : p.m;
  // tile of matrix z: (mi, ni); the symmetric modes walk the lower triangle row by row
  auto decode = [&](long long t, int& mi, int& ni, int& z) {
    z = (int)(t / per);
    const int r = (int)(t % per);
    if constexpr (SYM) {
      mi = (int)((sqrtf(8.f * (float)r + 1.f) - 1.f) * 0.5f);
      while (mi * (mi + 1) / 2 > r) --mi;
      while ((mi + 1) * (mi + 2) / 2 <= r) ++mi;
      ni = r - mi * (mi + 1) / 2;
    } else {
      ni = r / tm;
      mi = r % tm;
    }
  };

  if (warp == 0) {
    // =========================== TMA producer ===========================
    if (elect_one()) {
      uint32_t it = 0;
      for (long long t = blockIdx.x; t < total && !*abort_flag; t += gridDim.x) {
        int mi, ni, z;
        decode(t, mi, ni, z);
        for (int k0 = 0; k0 < K; k0 += BK, ++it) {
          const int s = it % STAGES;
          if (!mbar_wait(&empty_bar[s], ((it / STAGES) & 1) ^ 1, abort_flag, p.status, 110)) break;
          uint8_t* st = smem + s * STAGE_BYTES;
          mbar_expect_tx(&full_bar[s], STAGE_BYTES);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            tma_load_3d(st + h * TILE_BYTES, &tmapA, &full_bar[s], k0, mi * BM, 2 * z + h);
            uint8_t* sb = st + (2 + h) * TILE_BYTES;
            if constexpr (!B_MN) {
              tma_load_3d(sb, &tmapB, &full_bar[s], k0, ni * BN, 2 * z + h);
            } else {
#pragma unroll
              for (int c = 0; c < BN / 64; ++c)
                tma_load_3d(sb + c * (BK * 128), &tmapB, &full_bar[s], ni * BN + c * 64, k0, 2 * z + h);
            }
          }
        }
      }
      if (*abort_flag) drain_copies(full_bar, STAGES, it);
    }
  } else if (warp == 1) {
    // =========================== MMA issuer (converged warp, one elected lane) ===========================
    const uint32_t idesc = make_idesc(0u, 0u, B_MN ? 1u : 0u, BM, BN);
    uint32_t it = 0, tile_no = 0;
    for (long long t = blockIdx.x; t < total; t += gridDim.x) {
      const uint32_t acc = tile_no & 1, acc_ph = (tile_no >> 1) & 1;
      if (!__all_sync(0xffffffffu, mbar_wait(&tmem_empty[acc], acc_ph ^ 1, abort_flag, p.status, 210))) break;
      tc_fence_after_sync();
      const uint32_t d_tmem = tmem_base + acc * ACC_STRIDE;
      bool ok = true;
      for (int k0 = 0; k0 < K; k0 += BK, ++it) {
        const int s = it % STAGES;
        if (!__all_sync(0xffffffffu, mbar_wait(&full_bar[s], (it / STAGES) & 1, abort_flag, p.status, 211))) { ok = false; break; }
        tc_fence_after_sync();
        const uint32_t a_addr = smem_u32(smem + s * STAGE_BYTES), b_addr = a_addr + 2 * TILE_BYTES;
        const uint64_t da = make_smem_desc(a_addr, 16, 1024);
        const uint64_t db = B_MN ? make_smem_desc(b_addr, BK * 128, 1024) : make_smem_desc(b_addr, 16, 1024);
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < BK / 16; ++kk) {
            const uint64_t a = da + kk * 2, b = db + (B_MN ? kk * 128 : kk * 2);      // (16-byte units)
            constexpr uint64_t LO = TILE_BYTES / 16;
            umma_f16(d_tmem, a, b, idesc, (k0 == 0 && kk == 0) ? 0u : 1u);
            umma_f16(d_tmem, a, b + LO, idesc, 1u);
            umma_f16(d_tmem, a + LO, b, idesc, 1u);
          }
          umma_commit(&empty_bar[s]);
        }
        __syncwarp();
      }
      if (!ok) break;
      if (elect_one()) umma_commit(&tmem_full[acc]);
      __syncwarp();
      ++tile_no;
    }
    __syncwarp();
  } else {
    // =========================== epilogue: 8 warps, 32 rows x 64 columns each ===========================
    const int q = warp & 3, half = (warp - 2) >> 2;
    uint32_t tile_no = 0;
    float keep = 0.f, step = 0.f;
    bool skip = false;
    if constexpr (MODE == APPLY_LAST) {
      const float lr = p.dyn_lr != nullptr ? *p.dyn_lr : p.lr;
      keep = 1.f - lr * p.decay;
      step = lr * p.scale;
      skip = p.found_inf != nullptr && *p.found_inf != 0.f;
    }
    for (long long t = blockIdx.x; t < total && !*abort_flag; t += gridDim.x) {
      int mi, ni, z;
      decode(t, mi, ni, z);
      const uint32_t acc = tile_no & 1, acc_ph = (tile_no >> 1) & 1;
      if (!__all_sync(0xffffffffu, mbar_wait(&tmem_full[acc], acc_ph, abort_flag, p.status, 310))) break;
      tc_fence_after_sync();
      const int row = mi * BM + q * 32 + lane;
      const int cols = SYM ? p.m : p.n;
#pragma unroll 1
      for (int c = half * 64; c < half * 64 + 64; c += 32) {
        const int col0 = ni * BN + c;
        __syncwarp();                                   // (the lanes part below where rows or columns end)
        uint32_t r[32];
        tmem_ld_32x32b_x32(tmem_base + ((uint32_t)(q * 32) << 16) + acc * ACC_STRIDE + c, r);
        tmem_ld_wait();
        if (row >= p.m || col0 >= cols) continue;
        float v[32];
        if constexpr (SYM) {
          const size_t plane = (size_t)p.m * p.lda, base = (size_t)z * 2 * plane;
          __half* hi = p.dst + base;
          __half* lo = hi + plane;
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]) * p.f_acc;
          if constexpr (MODE == SQUARE) {
            const __half* ah = p.a_planes + base + (size_t)row * p.lda + col0;
            const __half* al = ah + plane;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              if (col0 + 8 * g < cols) {
                const uint4 x = *reinterpret_cast<const uint4*>(ah + 8 * g), y = *reinterpret_cast<const uint4*>(al + 8 * g);
                const __half2* xh = reinterpret_cast<const __half2*>(&x);
                const __half2* yh = reinterpret_cast<const __half2*>(&y);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                  const float2 f = __half22float2(xh[k]), e = __half22float2(yh[k]);
                  v[8 * g + 2 * k] = fmaf(f.x + e.x, p.f_a, v[8 * g + 2 * k]);
                  v[8 * g + 2 * k + 1] = fmaf(f.y + e.y, p.f_a, v[8 * g + 2 * k + 1]);
                }
              }
            }
          }
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            if (col0 + 8 * g < cols) {                  // (the pitch is a multiple of 8: whole vectors fit)
              uint4 oh, ol;
              __half* h8 = reinterpret_cast<__half*>(&oh);
              __half* l8 = reinterpret_cast<__half*>(&ol);
#pragma unroll
              for (int k = 0; k < 8; ++k) split(v[8 * g + k], h8[k], l8[k]);
              *reinterpret_cast<uint4*>(hi + (size_t)row * p.lda + col0 + 8 * g) = oh;
              *reinterpret_cast<uint4*>(lo + (size_t)row * p.lda + col0 + 8 * g) = ol;
              if (mi != ni) {
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                  if (col0 + 8 * g + k < cols) {
                    hi[(size_t)(col0 + 8 * g + k) * p.lda + row] = h8[k];
                    lo[(size_t)(col0 + 8 * g + k) * p.lda + row] = l8[k];
                  }
                }
              }
            }
          }
        } else {
          float* x = p.x + ((size_t)z * p.m + row) * p.ldx + col0;
#pragma unroll
          for (int g = 0; g < 8; ++g) {
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
            if (col0 + 4 * g < cols) o = *reinterpret_cast<const float4*>(x + 4 * g);
            v[4 * g] = fmaf(__uint_as_float(r[4 * g]), p.f_acc, o.x * p.f_a);
            v[4 * g + 1] = fmaf(__uint_as_float(r[4 * g + 1]), p.f_acc, o.y * p.f_a);
            v[4 * g + 2] = fmaf(__uint_as_float(r[4 * g + 2]), p.f_acc, o.z * p.f_a);
            v[4 * g + 3] = fmaf(__uint_as_float(r[4 * g + 3]), p.f_acc, o.w * p.f_a);
          }
          if constexpr (MODE == APPLY) {
            const size_t plane = (size_t)p.m * p.ldx;
            __half* hi = p.dst + (size_t)z * 2 * plane + (size_t)row * p.ldx + col0;
            __half* lo = hi + plane;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              if (col0 + 8 * g < cols) {
                uint4 oh, ol;
                __half* h8 = reinterpret_cast<__half*>(&oh);
                __half* l8 = reinterpret_cast<__half*>(&ol);
#pragma unroll
                for (int k = 0; k < 8; ++k) split(v[8 * g + k] * p.next_scale, h8[k], l8[k]);
                *reinterpret_cast<uint4*>(hi + 8 * g) = oh;
                *reinterpret_cast<uint4*>(lo + 8 * g) = ol;
                *reinterpret_cast<float4*>(x + 8 * g) = make_float4(v[8 * g], v[8 * g + 1], v[8 * g + 2], v[8 * g + 3]);
                *reinterpret_cast<float4*>(x + 8 * g + 4) = make_float4(v[8 * g + 4], v[8 * g + 5], v[8 * g + 6], v[8 * g + 7]);
              }
            }
          } else {
            // element (row, col) of X is (col, row) of a tall result
            const size_t si = p.tall ? 1 : p.n, sj = p.tall ? p.m : 1;
            const size_t at = (size_t)row * si + (size_t)col0 * sj;
            if (p.weights != nullptr) {
              float* w = reinterpret_cast<float*>(p.weights[z]) + at;
              if (!skip) {
#pragma unroll
                for (int j = 0; j < 32; ++j)
                  if (col0 + j < cols) w[j * sj] = fmaf(w[j * sj], keep, -step * v[j]);
              }
            } else {
              const size_t o = (size_t)z * p.m * p.n + at;
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (col0 + j < cols) store_from_float(p.out, p.out_dtype, o + j * sj, v[j]);
            }
          }
        }
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&tmem_empty[acc]);
      ++tile_no;
    }
  }

  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, 2 * ACC_STRIDE);
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

// Partial sums of squares, in 64 bits: 32 would overflow or vanish at half the exponent range of the elements
__global__ void __launch_bounds__(256)
ns_norm_kernel(const void* __restrict__ src, int dt, long long numel, double* __restrict__ partial) {
  __shared__ double sh[8];
  const size_t base = (size_t)blockIdx.y * numel;
  double s = 0.0;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < numel; i += 256 * PARTS) {
    const double x = (double)load_as_float(src, dt, base + i);
    s += x * x;
  }
  s = block_sum256(s, sh);
  if (threadIdx.x == 0) partial[blockIdx.y * PARTS + blockIdx.x] = s;
}

// Momentum of every matrix of a batch and the update that goes on to the iteration:
//   u <- mu u + (1 - mu) g,   y = mu u + (1 - mu) g (Nesterov) or u
// table: addresses of gradients, then of momenta [2, batch]; y [batch, numel], and the partial sums of its squares.
__global__ void __launch_bounds__(256)
muon_momentum_kernel(const long long* __restrict__ table, int batch, int grad_dt, long long numel, float mu, int nesterov,
                     const float* __restrict__ grad_scale, const float* __restrict__ found_inf, float* __restrict__ y,
                     double* __restrict__ partial) {
  __shared__ double sh[8];
  const int z = blockIdx.y;
  const void* g = reinterpret_cast<const void*>(table[z]);
  float* u = reinterpret_cast<float*>(table[batch + z]);
  const float gs = grad_scale != nullptr ? *grad_scale : 1.f;
  const bool skip = found_inf != nullptr && *found_inf != 0.f;      // the step is cancelled: momentum stays as it is
  double s = 0.0;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < numel; i += 256 * PARTS) {
    const float gi = skip ? 0.f : load_as_float(g, grad_dt, i) * gs;
    const float ui = mu * u[i] + (1.f - mu) * gi;
    if (!skip) u[i] = ui;
    const float yi = nesterov ? mu * ui + (1.f - mu) * gi : ui;
    y[(size_t)z * numel + i] = yi;
    s += (double)yi * (double)yi;
  }
  s = block_sum256(s, sh);
  if (threadIdx.x == 0) partial[z * PARTS + blockIdx.x] = s;
}

// X = G / (|G| + eps), in 32 bits and as fp16 terms, transposed where G [rows, cols] is tall
__global__ void __launch_bounds__(256)
ns_prepare_kernel(const void* __restrict__ src, int dt, int rows, int cols, int tall, const double* __restrict__ partial,
                  double eps, float scale, float* __restrict__ x, __half* __restrict__ planes, int ldx) {
  __shared__ float tile[32][33];
  __shared__ double inv;
  const int z = blockIdx.z;
  if (threadIdx.x == 0) {
    double s = 0.0;
    for (int i = 0; i < PARTS; ++i) s += partial[z * PARTS + i];
    inv = 1.0 / (sqrt(s) + eps);
  }
  __syncthreads();
  const int r0 = blockIdx.y * 32, c0 = blockIdx.x * 32;
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
#pragma unroll
  for (int k = 0; k < 32; k += 8) {
    const int r = r0 + ty + k, c = c0 + tx;
    if (r < rows && c < cols)
      tile[ty + k][tx] = (float)((double)load_as_float(src, dt, ((size_t)z * rows + r) * cols + c) * inv);
  }
  __syncthreads();
  const int m = tall ? cols : rows;
  const size_t plane = (size_t)m * ldx;
#pragma unroll
  for (int k = 0; k < 32; k += 8) {
    int i, j;
    float v;
    if (tall) { i = c0 + ty + k; j = r0 + tx; v = tile[tx][ty + k]; if (i >= cols || j >= rows) continue; }
    else { i = r0 + ty + k; j = c0 + tx; v = tile[ty + k][tx]; if (i >= rows || j >= cols) continue; }
    const size_t o = (size_t)i * ldx + j;
    __half hi, lo;
    split(v * scale, hi, lo);
    x[(size_t)z * plane + o] = v;
    planes[(size_t)z * 2 * plane + o] = hi;
    planes[(size_t)z * 2 * plane + plane + o] = lo;
  }
}

template <int MODE>
static int product(const CUtensorMap& ta, const CUtensorMap& tb, const Params& p, cudaStream_t st) {
  static unsigned long long configured = 0;
  if (int e = smem_opt_in(ns_product_kernel<MODE>, SMEM_TOTAL, configured)) return e;
  const int tm = (p.m + BM - 1) / BM, tn = (p.n + BN - 1) / BN;
  const long long total = (long long)(MODE == GRAM || MODE == SQUARE ? tm * (tm + 1) / 2 : tm * tn) * p.batch;
  const int sms = sm_count();
  ns_product_kernel<MODE><<<(unsigned)(total < sms ? total : sms), 320, SMEM_TOTAL, st>>>(ta, tb, p);
  return (int)cudaGetLastError();
}

static inline long long up256(long long b) { return (b + 255) & ~255ll; }

struct Workspace {
  double* partial; float* y; float* x; __half* xp[2]; __half* a; __half* b;
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
    a = (__half*)take(batch * m * lda * 4);
    b = (__half*)take(batch * m * lda * 4);
    bytes = at;
  }
};

}  // namespace ns
}  // namespace gb

using namespace gb;

// Bytes of workspace that a batch of `batch` matrices needs (with_y: an optimizer step, which keeps its update there)
extern "C" int gb_ns_workspace(long long rows, long long cols, long long batch, int with_y, long long* bytes) {
  *bytes = ns::Workspace(nullptr, rows < cols ? rows : cols, rows < cols ? cols : rows, batch, with_y != 0).bytes;
  return 0;
}

// First half of an optimizer step: see muon_momentum_kernel.  The update and its partial sums stay in the workspace.
extern "C" int gb_muon_momentum(const long long* table, int batch, int grad_dt, int rows, int cols, float mu, int nesterov,
                                const float* grad_scale, const float* found_inf, void* workspace, cudaStream_t st) {
  if (batch <= 0 || rows <= 0 || cols <= 0) return 0;
  if (batch > 65535) return -3;
  const ns::Workspace w((uint8_t*)workspace, rows < cols ? rows : cols, rows < cols ? cols : rows, batch, true);
  ns::muon_momentum_kernel<<<dim3(ns::PARTS, batch), 256, 0, st>>>(table, batch, grad_dt, (long long)rows * cols, mu, nesterov,
                                                                   grad_scale, found_inf, w.y, w.partial);
  return (int)cudaGetLastError();
}

// Orthogonalises `batch` matrices [rows, cols].  `src` (contiguous, dtype dt) with `out` of the same type, or null for the
// update that gb_muon_momentum has left in the workspace, which goes into the weights at `weights` [batch].
// exponents [3 steps]: powers of two by which X, A and B of each step are scaled in fp16 (host: from the coefficients).
extern "C" int gb_newton_schulz(const void* src, void* out, int dt, int rows, int cols, int batch, int steps, float a, float b,
                                float c, double eps, const int* exponents, const long long* weights, float lr, float decay,
                                float scale, const float* dyn_lr, const float* found_inf, void* workspace, int* status,
                                cudaStream_t st) {
  if (batch <= 0 || rows <= 0 || cols <= 0) return 0;
  if (batch > 32767 || steps < 1 || (src == nullptr) != (weights != nullptr) || (reinterpret_cast<uintptr_t>(workspace) & 255) != 0)
    return -3;
  const int tall = rows > cols, m = tall ? cols : rows, n = tall ? rows : cols;
  const int ldx = (n + 7) & ~7, lda = (m + 7) & ~7;
  const ns::Workspace w((uint8_t*)workspace, m, n, batch, src == nullptr);
  if (src != nullptr) ns::ns_norm_kernel<<<dim3(ns::PARTS, batch), 256, 0, st>>>(src, dt, (long long)rows * cols, w.partial);
  const dim3 grid((cols + 31) / 32, (rows + 31) / 32, batch);
  if (grid.y > 65535) return -3;
  ns::ns_prepare_kernel<<<grid, 256, 0, st>>>(src != nullptr ? src : w.y, src != nullptr ? dt : (int)DT_F32, rows, cols, tall,
                                              w.partial, eps, ldexpf(1.f, exponents[0]), w.x, w.xp[0], ldx);
  if (const int e = (int)cudaGetLastError()) return e;
  // maps: X as left or right operand of X X^T (rows of the contraction), X as right operand of B X, A, B
  CUtensorMap mx[2], mxr[2], ma, mb;
  int r;
  for (int i = 0; i < 2; ++i) {
    if ((r = make_tmap_3d(&mx[i], w.xp[i], DT_F16, n, m, 2ll * batch, ldx, (long long)m * ldx, 128)) != 0) return 10000 + r;
    if ((r = make_tmap_3d(&mxr[i], w.xp[i], DT_F16, n, m, 2ll * batch, ldx, (long long)m * ldx, 64)) != 0) return 20000 + r;
  }
  if ((r = make_tmap_3d(&ma, w.a, DT_F16, m, m, 2ll * batch, lda, (long long)m * lda, 128)) != 0) return 30000 + r;
  if ((r = make_tmap_3d(&mb, w.b, DT_F16, m, m, 2ll * batch, lda, (long long)m * lda, 128)) != 0) return 40000 + r;
  ns::Params p = {};
  p.status = status; p.m = m; p.n = n; p.batch = batch; p.ldx = ldx; p.lda = lda; p.x = w.x; p.a_planes = w.a;
  p.out = out; p.out_dtype = dt; p.tall = tall; p.weights = weights; p.lr = lr; p.decay = decay; p.scale = scale;
  p.dyn_lr = dyn_lr; p.found_inf = found_inf;
  for (int k = 0; k < steps; ++k) {
    const int sx = exponents[3 * k], sa = exponents[3 * k + 1], sb = exponents[3 * k + 2], cur = k & 1;
    p.dst = w.a; p.f_acc = ldexpf(1.f, sa - 2 * sx); p.f_a = 0.f;
    if ((r = ns::product<ns::GRAM>(mx[cur], mx[cur], p, st)) != 0) return r;
    p.dst = w.b; p.f_acc = ldexpf(c, sb - 2 * sa); p.f_a = ldexpf(b, sb - sa);
    if ((r = ns::product<ns::SQUARE>(ma, ma, p, st)) != 0) return r;
    p.dst = w.xp[cur ^ 1]; p.f_acc = ldexpf(1.f, -sb - sx); p.f_a = a;
    p.next_scale = k + 1 < steps ? ldexpf(1.f, exponents[3 * k + 3]) : 1.f;
    r = k + 1 < steps ? ns::product<ns::APPLY>(mb, mxr[cur], p, st) : ns::product<ns::APPLY_LAST>(mb, mxr[cur], p, st);
    if (r != 0) return r;
  }
  return 0;
}
