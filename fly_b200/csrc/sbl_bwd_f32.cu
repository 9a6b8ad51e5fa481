// Generic kernels of the SBLocal gradients: any E, D <= 128, r, w, T != S,
// ragged key lengths, fp32 accuracy with fp32 or bf16 storage (eps = 0).
//
// With n_i the log-normaliser of row i, p_is = exp(tau q_i.k_s - n_i) inside the
// window, a_is = psi_i.phi_s outside it (phi_s = phi(k_s) as in the forward,
// psi_i = phi(q_i) over the row's normaliser) and g_is = dout_i.v_s - delta_i,
// delta_i = dout_i.out_i:
//
//   dq_i = tau sum_in p g k_s    + through(psi_i, sum_out g phi_s)
//   dk_s = tau sum_in p g q_i    + through(phi_s, sum_out g psi_i)
//   dv_s = sum_in (p - psi.phi) dout_i + phi_s . sum_i psi_i dout_i
//   sum_out g phi_s = [KV dout_i - delta_i sum phi] - sum_in g phi_s   (and the same for keys)
//   through(f, df) = ((f df)_+ - (f df)_-) Wt - tau x sum f df
//
// Kernels: row statistics; the features of the forward, once more for the
// queries; a summary per side; per side `dfeat` (f df for 64 rows and 128
// features) and `dx` (the window part and the projection back); `dv`.
//
// Products.  Three TF32 products of a split operand pair (x = hi + lo with 11
// bits each: lo hi' + hi lo' + hi hi', fp32 accumulation) keep 22 bits of every
// factor; an operand stored in bf16 is its own hi and saves its lo products.
// mma.sync.m16n8k8 runs at 512 multiply-adds per clock and SM, three of them at
// 171 against 124 measured for FFMA, with a twentieth of the instructions.  (The
// tcgen05 path would need both terms of every operand in shared memory as
// swizzled tiles, padded to its shapes; this path takes any shape.)
// A warp owns 16 rows.  It leaves g or p g in the registers of the first
// product's accumulator and feeds them to the second as A operand: column pair
// (2t, 2t + 1) of an 8-column step plays k = t and t + 4 on both operands.
#include "sbl_f32_tile.cuh"

namespace sbl {
namespace {

size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }

constexpr int LK = 68;     // row pitch of a 64-wide operand tile: 4 mod 32 words, so fragment loads meet no bank twice
constexpr int LW = 132;    // row pitch of a 128-wide one
constexpr int FT = 128;    // features per dfeat block
constexpr int WARPS = 4, NT = 32 * WARPS;   // 64 rows

// ---- TF32 fragments -----------------------------------------------------------
struct Split {
  uint32_t hi, lo;
};
__device__ __forceinline__ uint32_t tf32(float x) {
  uint32_t r;
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(x));
  return r;
}
template <bool EXACT>
__device__ __forceinline__ Split split(float x) {
  Split s;
  if (EXACT) {
    s.hi = __float_as_uint(x);
    s.lo = 0u;
  } else {
    s.hi = tf32(x);
    s.lo = tf32(x - __uint_as_float(s.hi));
  }
  return s;
}
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// c[n0 .. n0 + COUNT) += a b to fp32 accuracy; the products of one accumulator are COUNT instructions apart
template <bool AX, bool BX, int COUNT, int N>
__device__ __forceinline__ void mma3(float (&c)[N][4], int n0, const Split (&a)[4], const Split (&b)[COUNT][2]) {
  if (!AX) {
#pragma unroll
    for (int n = 0; n < COUNT; ++n) mma(c[n0 + n], a[0].lo, a[1].lo, a[2].lo, a[3].lo, b[n][0].hi, b[n][1].hi);
  }
  if (!BX) {
#pragma unroll
    for (int n = 0; n < COUNT; ++n) mma(c[n0 + n], a[0].hi, a[1].hi, a[2].hi, a[3].hi, b[n][0].lo, b[n][1].lo);
  }
#pragma unroll
  for (int n = 0; n < COUNT; ++n) mma(c[n0 + n], a[0].hi, a[1].hi, a[2].hi, a[3].hi, b[n][0].hi, b[n][1].hi);
}

// The tensor core cuts the bits that fall off its accumulator instead of rounding them: a chain of products is off by
// up to a unit of 2^-24 per link, all in one direction.  So every product below sums 64 terms in a fresh
// accumulator (24 links) and adds it to the running one in fp32.

// c (16 x 8 N) += A (16 x 64) B^T, A and B [rows][k] of pitch LK; A points at the warp's first row
template <int N, bool AX, bool BX>
__device__ __forceinline__ void product_nt(float (&c)[N][4], const float* A, const float* B) {
  const int g = (threadIdx.x % 32) / 4, t = threadIdx.x % 4;
#pragma unroll
  for (int nb = 0; nb < N; nb += 8) {
    float part[8][4] = {};
#pragma unroll 2
    for (int k = 0; k < 64; k += 8) {
      Split a[4];
      a[0] = split<AX>(A[g * LK + k + t]);
      a[1] = split<AX>(A[(g + 8) * LK + k + t]);
      a[2] = split<AX>(A[g * LK + k + t + 4]);
      a[3] = split<AX>(A[(g + 8) * LK + k + t + 4]);
#pragma unroll
      for (int n4 = 0; n4 < 8; n4 += 4) {
        Split b[4][2];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          b[n][0] = split<BX>(B[(8 * (nb + n4 + n) + g) * LK + k + t]);
          b[n][1] = split<BX>(B[(8 * (nb + n4 + n) + g) * LK + k + t + 4]);
        }
        mma3<AX, BX>(part, n4, a, b);
      }
    }
#pragma unroll
    for (int n = 0; n < 8; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) c[nb + n][j] += part[n][j];
  }
}
// c (16 x 8 N) += A (16 x 64) B, A [rows][k] of pitch LK, B [k][n] of pitch PITCH (4 mod 32)
template <int N, int PITCH, bool BX>
__device__ __forceinline__ void product_nn(float (&c)[N][4], const float* A, const float* B) {
  const int g = (threadIdx.x % 32) / 4, t = threadIdx.x % 4;
#pragma unroll
  for (int nb = 0; nb < N; nb += 8) {
    float part[8][4] = {};
#pragma unroll 2
    for (int k = 0; k < 64; k += 8) {
      // (k = 2t and 2t + 1 in the places of t and t + 4, on both sides: no bank conflicts in B)
      Split a[4];
      a[0] = split<false>(A[g * LK + k + 2 * t]);
      a[1] = split<false>(A[(g + 8) * LK + k + 2 * t]);
      a[2] = split<false>(A[g * LK + k + 2 * t + 1]);
      a[3] = split<false>(A[(g + 8) * LK + k + 2 * t + 1]);
#pragma unroll
      for (int n4 = 0; n4 < 8; n4 += 4) {
        Split b[4][2];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          b[n][0] = split<BX>(B[(k + 2 * t) * PITCH + 8 * (nb + n4 + n) + g]);
          b[n][1] = split<BX>(B[(k + 2 * t + 1) * PITCH + 8 * (nb + n4 + n) + g]);
        }
        mma3<false, BX>(part, n4, a, b);
      }
    }
#pragma unroll
    for (int n = 0; n < 8; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) c[nb + n][j] += part[n][j];
  }
}
// c (16 x 8 N) += P B, P (16 x 64) in the accumulators of an earlier product
template <int N, int PITCH, bool BX>
__device__ __forceinline__ void product_acc(float (&c)[N][4], const float (&p)[8][4], const float* B) {
  const int g = (threadIdx.x % 32) / 4, t = threadIdx.x % 4;
#pragma unroll
  for (int nb = 0; nb < N; nb += 8) {
    float part[8][4] = {};
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      Split a[4];
      a[0] = split<false>(p[k][0]);
      a[1] = split<false>(p[k][2]);
      a[2] = split<false>(p[k][1]);
      a[3] = split<false>(p[k][3]);
#pragma unroll
      for (int n4 = 0; n4 < 8; n4 += 4) {
        Split b[4][2];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          b[n][0] = split<BX>(B[(8 * k + 2 * t) * PITCH + 8 * (nb + n4 + n) + g]);
          b[n][1] = split<BX>(B[(8 * k + 2 * t + 1) * PITCH + 8 * (nb + n4 + n) + g]);
        }
        mma3<false, BX>(part, n4, a, b);
      }
    }
#pragma unroll
    for (int n = 0; n < 8; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) c[nb + n][j] += part[n][j];
  }
}

__device__ __forceinline__ float4 ld4(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ float4 ld4(const __nv_bfloat16* p) {
  const uint2 v = *reinterpret_cast<const uint2*>(p);
  return make_float4(__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u), __uint_as_float(v.y << 16),
                     __uint_as_float(v.y & 0xffff0000u));
}

// dst [rows][PITCH] <- src (row stride ld, `nrow` x `ncol` valid), zeros elsewhere; COLS of them are written.
// Four at a time, all loads of a thread in flight, where the source allows it.
template <int ROWS, int COLS, int PITCH, typename T>
__device__ __forceinline__ void stage(float* dst, const T* src, int64_t ld, int nrow, int ncol) {
  constexpr int Q = COLS / 4, PER = ROWS * Q / NT;
  if ((reinterpret_cast<uintptr_t>(src) & (4 * sizeof(T) - 1)) == 0 && ld % 4 == 0 && (ncol % 4 == 0 || ncol >= COLS)) {
#pragma unroll
    for (int u0 = 0; u0 < PER; u0 += 8) {
      float4 v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int i = threadIdx.x + (u0 + u) * NT, r = i / Q, c = 4 * (i % Q);
        v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (r < nrow && c < ncol) v[u] = ld4(src + (int64_t)r * ld + c);
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int i = threadIdx.x + (u0 + u) * NT, r = i / Q, c = 4 * (i % Q);
        *reinterpret_cast<float4*>(dst + r * PITCH + c) = v[u];
      }
    }
    return;
  }
#pragma unroll 8
  for (int i = threadIdx.x; i < ROWS * COLS; i += NT) {
    const int r = i / COLS, c = i % COLS;
    dst[r * PITCH + c] = r < nrow && c < ncol ? ldf(src + (int64_t)r * ld + c) : 0.f;
  }
}

// ---- shared arguments ---------------------------------------------------------
// Which side the 64 rows of a block belong to.
enum { QUERIES = 0, KEYS = 1 };

struct SideArgs {
  const void *x, *y;              // rows: q or k (width E) | dout or v (width D)
  int64_t xb, xr, xh, yb, yr, yh; // strides: batch, row, head
  int rows;
};
struct GradArgs {
  SideArgs side[2];               // QUERIES, KEYS
  const int64_t* lengths;
  const float *lognorm, *delta;   // (BH, T)
  const float* feat[2];           // psi (BH,T,m), phi (BH,S,m)
  const float* sum[2];            // summaries over the queries, over the keys (BH,m,D)
  const float* sum1[2];           // their extra columns: sum delta psi, sum phi (BH,m)
  float* h;
  const float* Wt;
  void* dx; int64_t dxb, dxr, dxh;
  float* partial; int nsplit, split_rows;
  int H, E, D, r, w;
  float tau;
};

// first and last column a tile of rows can meet, and the mask
template <int SIDE>
struct Window {
  int lo, hi;         // columns, inclusive
  int len;            // real keys
  int hw, w;
  __device__ Window(const GradArgs& a, int b, int row0, int nrows) {
    len = a.side[KEYS].rows;
    if (a.lengths) {
      const int64_t l = a.lengths[b];
      len = l < 0 ? 0 : (l < len ? (int)l : len);
    }
    hw = a.w / 2;
    w = a.w;
    if (SIDE == QUERIES) {
      lo = row0 - hw;
      hi = min(row0 + nrows - 1 - hw + w - 1, len - 1);
    } else {
      lo = row0 + hw - w + 1;
      hi = row0 >= len ? -1 : min(row0 + nrows - 1 + hw, a.side[QUERIES].rows - 1);
    }
    lo = max(lo, 0);
  }
  // (row and column exist)
  __device__ bool in(int row, int col) const {
    const int i = SIDE == QUERIES ? row : col, s = SIDE == QUERIES ? col : row;
    return s >= i - hw && s <= i - hw + w - 1 && s < len;
  }
};

template <typename T>
__device__ __forceinline__ const T* side_x(const SideArgs& s, int b, int h, int row) {
  return static_cast<const T*>(s.x) + b * s.xb + h * s.xh + row * s.xr;
}
template <typename T>
__device__ __forceinline__ const T* side_y(const SideArgs& s, int b, int h, int row) {
  return static_cast<const T*>(s.y) + b * s.yb + h * s.yh + row * s.yr;
}
template <typename T>
struct IsExact {
  static constexpr bool value = false;
};
template <>
struct IsExact<__nv_bfloat16> {
  static constexpr bool value = true;
};

// c (64 rows x 64 columns) = A B^T over K, in slices of 64 through sA and sB (free before and after)
template <typename TA, typename TB>
__device__ __forceinline__ void tile_product(float (&c)[8][4], const TA* A, int64_t lda, int na, const TB* B, int64_t ldb,
                                             int nb, int K, float* sA, float* sB) {
#pragma unroll
  for (int n = 0; n < 8; ++n)
#pragma unroll
    for (int j = 0; j < 4; ++j) c[n][j] = 0.f;
  for (int k0 = 0; k0 < K; k0 += 64) {
    __syncthreads();
    stage<64, 64, LK>(sA, A + k0, lda, na, K - k0);
    stage<64, 64, LK>(sB, B + k0, ldb, nb, K - k0);
    __syncthreads();
    product_nt<8, IsExact<TA>::value, IsExact<TB>::value>(c, sA + (threadIdx.x / 32) * 16 * LK, sB);
  }
}

// ---- rows ---------------------------------------------------------------------
// One warp per query row: delta = dout . out, the log-normaliser, and that minus beta.
template <typename T>
__global__ void __launch_bounds__(256) row_kernel(SblParams p, SblGrads g, const float* beta, float* lognorm,
                                                  float* scale, float* delta) {
  const int64_t rows = (int64_t)p.B * p.H * p.T;
  const int64_t i = (int64_t)blockIdx.x * 8 + threadIdx.x / 32;
  if (i >= rows) return;
  const int lane = threadIdx.x % 32;
  const int64_t bh = i / p.T;
  const int t = (int)(i - bh * p.T), b = (int)(bh / p.H), h = (int)(bh % p.H);
  const T* o = static_cast<const T*>(p.out) + b * p.o_stride_b + t * p.o_stride_t + h * p.o_stride_h;
  const T* d = static_cast<const T*>(g.dout) + b * g.do_stride_b + t * g.do_stride_t + h * g.do_stride_h;
  float s = 0.f;
  for (int e = lane; e < p.D; e += 32) s = fmaf(ldf(o + e), ldf(d + e), s);
#pragma unroll
  for (int k = 16; k > 0; k >>= 1) s += __shfl_xor_sync(0xffffffffu, s, k);
  if (lane == 0) {
    const float n = g.row_stats[i] + logf(g.row_stats[rows + i]);
    lognorm[i] = n;
    // (a batch without keys: no features over the floor of the normaliser, whose sums could leave the fp32 range)
    scale[i] = p.key_lengths && p.key_lengths[b] <= 0 ? INFINITY : n - beta[bh];
    delta[i] = s;
  }
}

// ---- summary --------------------------------------------------------------------
// partial[bh][split] (m x (D + 1)) = sum over the split's rows of feature x [y | 1] (keys) or [y | delta] (queries).
// Block: 64 features, 8 N >= D + 1 columns.
template <typename T, int SIDE, int N>
__global__ void __launch_bounds__(NT) summary_kernel(GradArgs a) {
  extern __shared__ __align__(16) float smem[];
  constexpr int P = 8 * N + (N % 4 == 0 ? 4 : (N % 4 == 1 ? 28 : (N % 4 == 2 ? 20 : 12)));   // 4 mod 32
  float *sF = smem, *sY = smem + 64 * LK;      // [64 rows][64 features], [64 rows][8 N]
  const int warp = threadIdx.x / 32, g = (threadIdx.x % 32) / 4, t = threadIdx.x % 4;
  const int bh = blockIdx.z, b = bh / a.H, h = bh % a.H;
  const int m = 2 * a.r, f0 = blockIdx.x * 64, rows = a.side[SIDE].rows, D1 = a.D + 1;
  const int lo = blockIdx.y * a.split_rows, hi = min(rows, lo + a.split_rows);
  float c[N][4] = {};
  for (int r0 = lo; r0 < hi; r0 += 64) {
    const int nr = min(64, hi - r0);
    __syncthreads();
    stage<64, 64, LK>(sF, a.feat[SIDE] + ((int64_t)bh * rows + r0) * m + f0, (int64_t)m, nr, m - f0);
    const T* y = side_y<T>(a.side[SIDE], b, h, r0);
    constexpr int MAIN = N / 9 * 64, TAIL = 8 * N - MAIN;     // whole 64s, and the columns that may hold the extra one
    stage<64, MAIN, P>(sY, y, a.side[SIDE].yr, nr, a.D);
    if (a.D < MAIN) __syncthreads();                          // (the extra column lies among them)
    for (int i = threadIdx.x; i < 64 * (TAIL + 1); i += NT) {
      const int r = i / (TAIL + 1), j = i % (TAIL + 1);
      const int d = j < TAIL ? MAIN + j : a.D;
      if (j == TAIL && a.D >= MAIN) continue;
      float v = 0.f;
      if (r < nr && d < a.D) v = ldf(y + (int64_t)r * a.side[SIDE].yr + d);
      else if (r < nr && d == a.D) v = SIDE == KEYS ? 1.f : a.delta[(int64_t)bh * rows + r0 + r];
      sY[r * P + d] = v;
    }
    __syncthreads();
    float part[N][4] = {};
#pragma unroll 1
    for (int k = 0; k < 64; k += 8) {
      // A = features^T: row f, k = row 2t or 2t + 1
      const float* F = sF + k * LK + 16 * warp + g;
      Split s[4];
      s[0] = split<false>(F[2 * t * LK]);
      s[1] = split<false>(F[2 * t * LK + 8]);
      s[2] = split<false>(F[(2 * t + 1) * LK]);
      s[3] = split<false>(F[(2 * t + 1) * LK + 8]);
      constexpr int CH = 3;         // N = 9 or 18
#pragma unroll
      for (int n0 = 0; n0 < N; n0 += CH) {
        Split e[CH][2];
#pragma unroll
        for (int n = 0; n < CH; ++n) {
          e[n][0] = split<false>(sY[(k + 2 * t) * P + 8 * (n0 + n) + g]);
          e[n][1] = split<false>(sY[(k + 2 * t + 1) * P + 8 * (n0 + n) + g]);
        }
        mma3<false, false>(part, n0, s, e);
      }
    }
    // one partial per 64 rows: the rounding error grows with the number of partials
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) c[n][j] += part[n][j];
  }
  float* out = a.partial + ((int64_t)bh * a.nsplit + blockIdx.y) * m * D1;
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int f = f0 + 16 * warp + g + (j >= 2 ? 8 : 0), d = 8 * n + 2 * t + (j & 1);
      if (f < m && d < D1) out[(int64_t)f * D1 + d] = c[n][j];
    }
}

__global__ void combine_kernel(const float* partial, int nsplit, int m, int D, int64_t n, float* sum, float* sum1) {
  const int D1 = D + 1;
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;   // over BH * m * (D + 1)
  if (i >= n) return;
  const int d = (int)(i % D1);
  const int64_t bf = i / D1, bh = bf / m, f = bf % m;
  float s = 0.f;
  for (int k = 0; k < nsplit; ++k) s += partial[((bh * nsplit + k) * m + f) * D1 + d];
  if (d < D) sum[bf * D + d] = s;
  else sum1[bf] = s;
}

// ---- f df -------------------------------------------------------------------------
// h = f * (sum over the columns outside the window of g * f_other), for 64 rows and FT features
template <typename T, int SIDE>
__global__ void __launch_bounds__(NT, 3) dfeat_kernel(GradArgs a) {
  extern __shared__ __align__(16) float smem[];
  float *sA = smem, *sB = sA + 64 * LK, *sF = sB + 64 * LK;   // [64][64], [64][64], [64 columns][FT] or [FT][64]
  constexpr int OTHER = 1 - SIDE;
  const int warp = threadIdx.x / 32, g = (threadIdx.x % 32) / 4, t = threadIdx.x % 4;
  const int bh = blockIdx.z, b = bh / a.H, h = bh % a.H;
  const int row0 = blockIdx.x * 64, rows = a.side[SIDE].rows, cols = a.side[OTHER].rows;
  const int nr = min(64, rows - row0);
  const int m = 2 * a.r, f0 = blockIdx.y * FT;
  const T* y = side_y<T>(a.side[SIDE], b, h, row0);
  const float* delta = a.delta + (int64_t)bh * a.side[QUERIES].rows;
  const float* fo = a.feat[OTHER] + (int64_t)bh * cols * m + f0;
  const Window<SIDE> win(a, b, row0, nr);
  const int ra = row0 + 16 * warp + g, rb = ra + 8;           // this thread's two rows
  float da = 1.f, db = 1.f;
  if (SIDE == QUERIES) {
    da = ra < rows ? delta[ra] : 0.f;
    db = rb < rows ? delta[rb] : 0.f;
  }

  float acc[16][4] = {};
  for (int c0 = win.lo; c0 <= win.hi; c0 += 64) {
    const int nc = min(64, win.hi - c0 + 1);
    float p[8][4];
    tile_product(p, y, a.side[SIDE].yr, nr, side_y<T>(a.side[OTHER], b, h, c0), a.side[OTHER].yr, nc, a.D, sA, sB);
    stage<64, FT, LW>(sF, fo + (int64_t)c0 * m, (int64_t)m, nc, m - f0);
    // minus g inside the window
#pragma unroll
    for (int n = 0; n < 8; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int row = j >= 2 ? rb : ra, cj = 8 * n + 2 * t + (j & 1);
        const bool in = row < rows && cj < nc && win.in(row, c0 + cj);
        const float d = SIDE == QUERIES ? (j >= 2 ? db : da) : (in ? delta[c0 + cj] : 0.f);
        p[n][j] = in ? d - p[n][j] : 0.f;
      }
    __syncthreads();
    product_acc<16, LW, false>(acc, p, sF);
  }
  // the same sum over all columns: y . summary^T - delta * extra (queries), y . summary^T - extra (keys)
  const float* sum = a.sum[OTHER] + ((int64_t)bh * m + f0) * a.D;
  for (int k0 = 0; k0 < a.D; k0 += 64) {
    __syncthreads();
    stage<64, 64, LK>(sA, y + k0, a.side[SIDE].yr, nr, a.D - k0);
    stage<FT, 64, LK>(sF, sum + k0, (int64_t)a.D, m - f0, a.D - k0);
    __syncthreads();
    product_nt<16, IsExact<T>::value, false>(acc, sA + warp * 16 * LK, sF);
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int row = j ? rb : ra;
    if (row >= rows) continue;
    const float d = j ? db : da;
    const float* f = a.feat[SIDE] + ((int64_t)bh * rows + row) * m;
    float* out = a.h + ((int64_t)bh * rows + row) * m;
#pragma unroll
    for (int n = 0; n < 16; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int col = f0 + 8 * n + 2 * t + e;
        if (col < m) out[col] = f[col] * (acc[n][2 * j + e] - d * a.sum1[OTHER][(int64_t)bh * m + col]);
      }
  }
}

// ---- dq, dk -----------------------------------------------------------------------
// tau sum_in p g x' + (h_+ - h_-) Wt - tau x sum h; 64 rows, 64 NC columns of E
template <typename T, int SIDE, int NC>
__global__ void __launch_bounds__(NT, 3) dx_kernel(GradArgs a) {
  constexpr int P = NC == 1 ? LK : LW;
  extern __shared__ __align__(16) float smem[];
  float *sA = smem, *sB = sA + 64 * LK, *sX = sB + 64 * LK;   // ..., [64][64 NC]
  float* sH = sX + 64 * P;                                    // [64] sum of h per row
  constexpr int OTHER = 1 - SIDE;
  const int warp = threadIdx.x / 32, g = (threadIdx.x % 32) / 4, t = threadIdx.x % 4;
  const int bh = blockIdx.z, b = bh / a.H, h = bh % a.H;
  const int row0 = blockIdx.x * 64, rows = a.side[SIDE].rows, T_ = a.side[QUERIES].rows;
  const int nr = min(64, rows - row0);
  const int e0 = blockIdx.y * 64 * NC, m = 2 * a.r;
  const T* x = side_x<T>(a.side[SIDE], b, h, row0);
  const T* y = side_y<T>(a.side[SIDE], b, h, row0);
  const float* delta = a.delta + (int64_t)bh * T_;
  const float* lognorm = a.lognorm + (int64_t)bh * T_;
  const Window<SIDE> win(a, b, row0, nr);
  const int ra = row0 + 16 * warp + g, rb = ra + 8;

  float acc[8 * NC][4] = {};
  for (int c0 = win.lo; c0 <= win.hi; c0 += 64) {
    const int nc = min(64, win.hi - c0 + 1);
    const T* xo = side_x<T>(a.side[OTHER], b, h, c0);
    float s[8][4], p[8][4];
    tile_product(s, x, a.side[SIDE].xr, nr, xo, a.side[OTHER].xr, nc, a.E, sA, sB);
    tile_product(p, y, a.side[SIDE].yr, nr, side_y<T>(a.side[OTHER], b, h, c0), a.side[OTHER].yr, nc, a.D, sA, sB);
    stage<64, 64 * NC, P>(sX, xo + e0, a.side[OTHER].xr, nc, a.E - e0);
#pragma unroll
    for (int n = 0; n < 8; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int row = j >= 2 ? rb : ra, cj = 8 * n + 2 * t + (j & 1);
        const bool in = row < rows && cj < nc && win.in(row, c0 + cj);
        float v = 0.f;
        if (in) {
          const int q = SIDE == QUERIES ? row : c0 + cj;
          v = a.tau * (expf(a.tau * s[n][j] - lognorm[q]) * (p[n][j] - delta[q]));
        }
        p[n][j] = v;
      }
    __syncthreads();
    product_acc<8 * NC, P, IsExact<T>::value>(acc, p, sX);
  }
  // through the projection
  const float* hrow = a.h + ((int64_t)bh * rows + row0) * m;
  {
    const int row = threadIdx.x / 2, part = threadIdx.x % 2;
    float s = 0.f;
    if (row < nr)
      for (int f = part; f < m; f += 2) s += hrow[(int64_t)row * m + f];
    s += __shfl_xor_sync(0xffffffffu, s, 1);
    if (part == 0) sH[row] = s;
  }
  for (int k0 = 0; k0 < a.r; k0 += 64) {
    __syncthreads();
#pragma unroll 8
    for (int i = threadIdx.x; i < 64 * 64; i += NT) {
      const int row = i / 64, k = i % 64;
      sA[row * LK + k] = row < nr && k0 + k < a.r
                             ? hrow[(int64_t)row * m + k0 + k] - hrow[(int64_t)row * m + a.r + k0 + k] : 0.f;
    }
    stage<64, 64 * NC, P>(sX, a.Wt + (int64_t)k0 * a.E + e0, (int64_t)a.E, a.r - k0, a.E - e0);
    __syncthreads();
    product_nn<8 * NC, P, false>(acc, sA + warp * 16 * LK, sX);
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int row = j ? rb : ra;
    if (row >= rows) continue;
    T* out = static_cast<T*>(a.dx) + b * a.dxb + h * a.dxh + (int64_t)row * a.dxr;
    const T* xr = x + (int64_t)(row - row0) * a.side[SIDE].xr;
    const float hs = a.tau * sH[row - row0];
#pragma unroll
    for (int n = 0; n < 8 * NC; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int e = e0 + 8 * n + 2 * t + c;
        if (e < a.E) stf(out + e, acc[n][2 * j + c] - hs * ldf(xr + e));
      }
  }
}

// ---- dv ---------------------------------------------------------------------------
// sum_in (p - psi.phi) dout + phi . QG; 64 key rows, 64 NC columns of D
template <typename T, int NC>
__global__ void __launch_bounds__(NT, 3) dv_kernel(GradArgs a) {
  constexpr int P = NC == 1 ? LK : LW;
  extern __shared__ __align__(16) float smem[];
  float *sA = smem, *sB = sA + 64 * LK, *sX = sB + 64 * LK;   // ..., [64][64 NC]
  const int warp = threadIdx.x / 32, g = (threadIdx.x % 32) / 4, t = threadIdx.x % 4;
  const int bh = blockIdx.z, b = bh / a.H, h = bh % a.H;
  const int row0 = blockIdx.x * 64, rows = a.side[KEYS].rows, T_ = a.side[QUERIES].rows;
  const int nr = min(64, rows - row0);
  const int m = 2 * a.r;
  const T* x = side_x<T>(a.side[KEYS], b, h, row0);
  const float* lognorm = a.lognorm + (int64_t)bh * T_;
  const float* phi = a.feat[KEYS] + ((int64_t)bh * rows + row0) * m;
  const float* psi = a.feat[QUERIES] + (int64_t)bh * T_ * m;
  const Window<KEYS> win(a, b, row0, nr);
  const int ra = row0 + 16 * warp + g, rb = ra + 8;

  float acc[8 * NC][4] = {};
  for (int c0 = win.lo; c0 <= win.hi; c0 += 64) {
    const int nc = min(64, win.hi - c0 + 1);
    float s[8][4], l[8][4];
    tile_product(s, x, a.side[KEYS].xr, nr, side_x<T>(a.side[QUERIES], b, h, c0), a.side[QUERIES].xr, nc, a.E, sA, sB);
    tile_product(l, phi, (int64_t)m, nr, psi + (int64_t)c0 * m, (int64_t)m, nc, m, sA, sB);
    stage<64, 64 * NC, P>(sX, side_y<T>(a.side[QUERIES], b, h, c0), a.side[QUERIES].yr, nc, a.D);
#pragma unroll
    for (int n = 0; n < 8; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int row = j >= 2 ? rb : ra, cj = 8 * n + 2 * t + (j & 1);
        const bool in = row < rows && cj < nc && win.in(row, c0 + cj);
        l[n][j] = in ? expf(a.tau * s[n][j] - lognorm[c0 + cj]) - l[n][j] : 0.f;
      }
    __syncthreads();
    product_acc<8 * NC, P, IsExact<T>::value>(acc, l, sX);
  }
  const float* sum = a.sum[QUERIES] + (int64_t)bh * m * a.D;
  for (int f0 = 0; f0 < m; f0 += 64) {
    __syncthreads();
    stage<64, 64, LK>(sA, phi + f0, (int64_t)m, nr, m - f0);
    stage<64, 64 * NC, P>(sX, sum + (int64_t)f0 * a.D, (int64_t)a.D, m - f0, a.D);
    __syncthreads();
    product_nn<8 * NC, P, false>(acc, sA + warp * 16 * LK, sX);
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int row = j ? rb : ra;
    if (row >= rows) continue;
    T* out = static_cast<T*>(a.dx) + b * a.dxb + h * a.dxh + (int64_t)row * a.dxr;
#pragma unroll
    for (int n = 0; n < 8 * NC; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int d = 8 * n + 2 * t + c;
        if (d < a.D) stf(out + d, acc[n][2 * j + c]);
      }
  }
}

// ---- host -------------------------------------------------------------------------
template <typename K>
cudaError_t run(K kernel, dim3 grid, size_t floats, const GradArgs& a, cudaStream_t st) {
  const size_t smem = floats * sizeof(float);
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  kernel<<<grid, NT, smem, st>>>(a);
  return cudaGetLastError();
}

template <typename T, int SIDE>
cudaError_t summary(const SblParams& p, GradArgs a, const BwdWorkspace& ws, char* base, cudaStream_t st) {
  const unsigned bh = (unsigned)(p.B * p.H), m = 2 * (unsigned)p.r;
  a.partial = reinterpret_cast<float*>(base + ws.partial);
  a.nsplit = ws.nsplit[SIDE];
  a.split_rows = ws.split_rows[SIDE];
  const dim3 grid((unsigned)div_up(m, 64), (unsigned)a.nsplit, bh);
  // 72 or 144 columns hold D + 1
  cudaError_t e = p.D < 72 ? run(summary_kernel<T, SIDE, 9>, grid, 64 * LK + 64 * 100, a, st)
                           : run(summary_kernel<T, SIDE, 18>, grid, 64 * LK + 64 * 164, a, st);
  if (e != cudaSuccess) return e;
  const int64_t n = (int64_t)bh * m * (p.D + 1);
  combine_kernel<<<(unsigned)div_up(n, 256), 256, 0, st>>>(a.partial, a.nsplit, (int)m, p.D, n,
                                                          const_cast<float*>(a.sum[SIDE]),
                                                          const_cast<float*>(a.sum1[SIDE]));
  return cudaGetLastError();
}

template <typename T, int SIDE>
cudaError_t side_grads(const SblParams& p, const GradArgs& a, cudaStream_t st) {
  const unsigned tiles = (unsigned)div_up(a.side[SIDE].rows, 64), bh = (unsigned)(p.B * p.H);
  cudaError_t e = run(dfeat_kernel<T, SIDE>, dim3(tiles, (unsigned)div_up(2 * p.r, FT), bh), 128 * LK + FT * LK, a, st);
  if (e != cudaSuccess) return e;
  if (p.E <= 64) return run(dx_kernel<T, SIDE, 1>, dim3(tiles, 1, bh), 192 * LK + 64, a, st);
  return run(dx_kernel<T, SIDE, 2>, dim3(tiles, (unsigned)div_up(p.E, 128), bh), 128 * LK + 64 * LW + 64, a, st);
}

template <typename T>
cudaError_t grads(const SblParams& p, const SblGrads& g, GradArgs a, const BwdWorkspace& ws, char* base, cudaStream_t st) {
  const unsigned bh = (unsigned)(p.B * p.H);
  cudaError_t e;
  const bool dq = !(g.skip & SBL_SKIP_DQ), dk = !(g.skip & SBL_SKIP_DK), dv = !(g.skip & SBL_SKIP_DV);
  if (dq && (e = summary<T, KEYS>(p, a, ws, base, st)) != cudaSuccess) return e;
  if ((dk || dv) && (e = summary<T, QUERIES>(p, a, ws, base, st)) != cudaSuccess) return e;
  if (dv) {
    a.dx = g.dv; a.dxb = g.dv_stride_b; a.dxr = g.dv_stride_s; a.dxh = g.dv_stride_h;
    const dim3 grid((unsigned)div_up(p.S, 64), 1, bh);
    e = p.D <= 64 ? run(dv_kernel<T, 1>, grid, 192 * LK, a, st) : run(dv_kernel<T, 2>, grid, 128 * LK + 64 * LW, a, st);
    if (e != cudaSuccess) return e;
  }
  a.dx = g.dq; a.dxb = g.dq_stride_b; a.dxr = g.dq_stride_t; a.dxh = g.dq_stride_h;
  if (dq && (e = side_grads<T, QUERIES>(p, a, st)) != cudaSuccess) return e;
  if (!dk) return cudaSuccess;
  a.dx = g.dk; a.dxb = g.dk_stride_b; a.dxr = g.dk_stride_s; a.dxh = g.dk_stride_h;
  return side_grads<T, KEYS>(p, a, st);
}

__global__ void row_stats_kernel(const float* lognorm, float* stats, int64_t n) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i < n) {
    stats[i] = lognorm[i];
    stats[n + i] = 1.f;
  }
}

}  // namespace

cudaError_t f32_row_stats(const SblParams& p, const Workspace& ws, char* base, float* row_stats, cudaStream_t st) {
  const int64_t n = (int64_t)p.B * p.H * p.T;
  row_stats_kernel<<<(unsigned)div_up(n, 256), 256, 0, st>>>(reinterpret_cast<const float*>(base + ws.lognorm),
                                                             row_stats, n);
  return cudaGetLastError();
}

void f32_plan_backward(const SblParams& p, BwdWorkspace* ws) {
  const size_t BH = (size_t)p.B * p.H, m = 2 * (size_t)p.r, T = p.T, S = p.S;
  size_t off = 0;
  auto take = [&](size_t bytes) {
    const size_t at = off;
    off = up256(off + bytes);
    return at;
  };
  Workspace& f = ws->fwd;
  f = Workspace{};
  f.tensor = false;
  f.wt = take((size_t)p.r * p.E * 4);
  f.phik = take(BH * S * m * 4);
  ws->lognorm = take(BH * T * 4);
  ws->scale = take(BH * T * 4);
  ws->delta = take(BH * T * 4);
  ws->psi = take(BH * T * m * 4);
  size_t partial = 0;
  for (int s = 0; s < 2; ++s) {
    ws->sum[s] = take(BH * m * p.D * 4);
    ws->sum1[s] = take(BH * m * 4);
    // at least 256 rows each, and no more splits than give every SM four blocks
    const int rows = s == QUERIES ? p.T : p.S;
    const int64_t units = (int64_t)BH * div_up(m, 64);
    int64_t n = div_up(148 * 4, units);
    n = n < div_up(rows, 256) ? n : div_up(rows, 256);
    ws->split_rows[s] = (int)(div_up(div_up(rows, n), 64) * 64);
    ws->nsplit[s] = (int)div_up(rows, ws->split_rows[s]);
    const size_t bytes = BH * ws->nsplit[s] * m * (p.D + 1) * 4;
    partial = bytes > partial ? bytes : partial;
  }
  ws->h = take(BH * (T > S ? T : S) * m * 4);
  ws->partial = take(partial);
  f.total = ws->total = off;
}

cudaError_t f32_backward(const SblParams& p, const SblGrads& g, const BwdWorkspace& ws, char* base, cudaStream_t st) {
  const float* beta = g.row_stats + 2 * (int64_t)p.B * p.H * p.T;
  float* phi = reinterpret_cast<float*>(base + ws.fwd.phik);
  float* lognorm = reinterpret_cast<float*>(base + ws.lognorm);
  float* scale = reinterpret_cast<float*>(base + ws.scale);
  float* delta = reinterpret_cast<float*>(base + ws.delta);
  float* psi = reinterpret_cast<float*>(base + ws.psi);
  cudaError_t e;
  if ((e = f32_prepare_projection(p, ws.fwd, base, st)) != cudaSuccess) return e;
  if ((e = f32_key_features(p, ws.fwd, base, beta, phi, st)) != cudaSuccess) return e;
  const unsigned blocks = (unsigned)div_up((int64_t)p.B * p.H * p.T, 8);
  if (p.dtype == SBL_DTYPE_F32) row_kernel<float><<<blocks, 256, 0, st>>>(p, g, beta, lognorm, scale, delta);
  else row_kernel<__nv_bfloat16><<<blocks, 256, 0, st>>>(p, g, beta, lognorm, scale, delta);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  if ((e = f32_query_features_over(p, ws.fwd, base, scale, psi, st)) != cudaSuccess) return e;
  GradArgs a{};
  a.side[QUERIES] = {p.q, g.dout, p.q_stride_b, p.q_stride_t, p.q_stride_h, g.do_stride_b, g.do_stride_t,
                     g.do_stride_h, p.T};
  a.side[KEYS] = {p.k, p.v, p.k_stride_b, p.k_stride_s, p.k_stride_h, p.v_stride_b, p.v_stride_s, p.v_stride_h, p.S};
  a.lengths = p.key_lengths;
  a.lognorm = lognorm;
  a.delta = delta;
  a.feat[QUERIES] = psi;
  a.feat[KEYS] = phi;
  for (int s = 0; s < 2; ++s) {
    a.sum[s] = reinterpret_cast<float*>(base + ws.sum[s]);
    a.sum1[s] = reinterpret_cast<float*>(base + ws.sum1[s]);
  }
  a.h = reinterpret_cast<float*>(base + ws.h);
  a.Wt = reinterpret_cast<const float*>(base + ws.fwd.wt);
  a.H = p.H; a.E = p.E; a.D = p.D; a.r = p.r;
  // a window wider than both sequences sees everything: keeps the index arithmetic far from 2^31
  const int64_t most = 2 * (int64_t)(p.T > p.S ? p.T : p.S) + 2;
  a.w = (int)(p.w < most ? p.w : most);
  a.tau = p.softmax_temp;
  return p.dtype == SBL_DTYPE_F32 ? grads<float>(p, g, a, ws, base, st) : grads<__nv_bfloat16>(p, g, a, ws, base, st);
}

}  // namespace sbl
