// Generic SIMT kernels of the SBLocal gradients: any E, D <= 128, r, w, T != S,
// ragged key lengths, fp32 arithmetic with fp32 or bf16 storage (eps = 0).
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
// Kernels: row statistics; the features and summaries of the forward, once more
// for the queries; per side `dfeat` (f df for a tile of rows and 128 features)
// and `dx` (the window part and the projection back); `dv`.  Every product is a
// 64-row block tile with 4x4 to 4x8 outputs per thread, so the FP32 pipe bounds
// them; sums over windows are one partial per 64 columns.
#include "sbl_f32_tile.cuh"

namespace sbl {
namespace {

size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }

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
    scale[i] = n - beta[bh];
    delta[i] = s;
  }
}

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
  const float* sum[2];            // summary over the OTHER side: KV for queries, QG for keys (BH,m,D)
  const float* sum1[2];           // its extra column: sum phi, sum delta psi
  float* h;
  const float* Wt;
  void* dx; int64_t dxb, dxr, dxh;
  int H, E, D, r, w;
  float tau;
};

// first and last column a tile of rows can meet, and the mask
template <int SIDE>
struct Window {
  int64_t lo, hi;     // columns, inclusive
  int64_t len;        // real keys
  int64_t hw, w;
  __device__ Window(const GradArgs& a, int b, int64_t row0, int nrows) {
    len = a.side[KEYS].rows;
    if (a.lengths && a.lengths[b] < len) len = a.lengths[b];
    hw = a.w / 2;
    w = a.w;
    if (SIDE == QUERIES) {
      lo = row0 - hw;
      hi = row0 + nrows - 1 - hw + w - 1;
      if (hi > len - 1) hi = len - 1;
    } else {
      lo = row0 + hw - w + 1;
      hi = row0 + nrows - 1 + hw;
      if (hi > a.side[QUERIES].rows - 1) hi = a.side[QUERIES].rows - 1;
      if (row0 >= len) hi = -1;
    }
    if (lo < 0) lo = 0;
  }
  __device__ bool in(int64_t row, int64_t col) const {
    const int64_t i = SIDE == QUERIES ? row : col, s = SIDE == QUERIES ? col : row;
    return s >= i - hw && s <= i - hw + w - 1 && s < len;
  }
};

template <typename T>
__device__ __forceinline__ const T* side_x(const SideArgs& s, int b, int h, int64_t row) {
  return static_cast<const T*>(s.x) + b * s.xb + h * s.xh + row * s.xr;
}
template <typename T>
__device__ __forceinline__ const T* side_y(const SideArgs& s, int b, int h, int64_t row) {
  return static_cast<const T*>(s.y) + b * s.yb + h * s.yh + row * s.yr;
}

constexpr int FT = 128;   // features per dfeat block

// acc (64 x 64 NC) += A^T B: A [64 k][68] holds the 64 rows of this tile per k, B [64 k][64 NC] the columns.
// Column c of a thread: 64 (c / 4) + 4 tx + c % 4.
template <int NC>
__device__ __forceinline__ void tile_tn(float (&acc)[4][4 * NC], const float (*A)[LDT], const float* B, float sign) {
  const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
  float part[4][4 * NC] = {};
#pragma unroll 4
  for (int k = 0; k < TILE; ++k) {
    const float4 a4 = *reinterpret_cast<const float4*>(&A[k][ty * 4]);
    const float av[4] = {a4.x, a4.y, a4.z, a4.w};
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const float4 b4 = *reinterpret_cast<const float4*>(B + k * 64 * NC + 64 * c + 4 * tx);
      const float bv[4] = {b4.x, b4.y, b4.z, b4.w};
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) part[i][4 * c + j] = fmaf(av[i], bv[j], part[i][4 * c + j]);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4 * NC; ++j) acc[i][j] = fmaf(sign, part[i][j], acc[i][j]);
}

// h = f * (sum over the columns outside the window of g * f_other), for 64 rows and FT features
template <typename T, int SIDE>
__global__ void __launch_bounds__(NTHR) dfeat_kernel(GradArgs a) {
  extern __shared__ __align__(16) float smem[];
  float(*sA)[LDT] = reinterpret_cast<float(*)[LDT]>(smem);
  float(*sB)[LDT] = sA + KS;
  float(*sG)[LDT] = sB + KS;                   // [64 columns][64 rows]: g^T, masked
  float* sF = &sG[TILE][0];                    // [64 columns][FT]
  constexpr int OTHER = 1 - SIDE;
  const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
  const int bh = blockIdx.z, b = bh / a.H, h = bh % a.H;
  const int64_t row0 = (int64_t)blockIdx.x * TILE;
  const int rows = a.side[SIDE].rows, cols = a.side[OTHER].rows;
  const int nr = (int)min((int64_t)TILE, rows - row0);
  const int m = 2 * a.r, f0 = blockIdx.y * FT, nf = min(FT, m - f0);
  const T* y = side_y<T>(a.side[SIDE], b, h, row0);
  const float* delta = a.delta + (int64_t)bh * a.side[QUERIES].rows;
  const float* fo = a.feat[OTHER] + (int64_t)bh * cols * m + f0;
  const Window<SIDE> win(a, b, row0, nr);

  float acc[4][8] = {};
  for (int64_t c0 = win.lo; c0 <= win.hi; c0 += TILE) {
    const int nc = (int)min((int64_t)TILE, win.hi - c0 + 1);
    float g[4][4] = {};
    tile_nt(g, y, a.side[SIDE].yr, nr, side_y<T>(a.side[OTHER], b, h, c0), a.side[OTHER].yr, nc, a.D, sA, sB);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int ri = ty * 4 + i, cj = tx * 4 + j;
        const bool in = ri < nr && cj < nc && win.in(row0 + ri, c0 + cj);
        sG[cj][ri] = in ? g[i][j] - delta[SIDE == QUERIES ? row0 + ri : c0 + cj] : 0.f;
      }
    for (int i = threadIdx.x; i < TILE * FT; i += NTHR) {
      const int k = i / FT, f = i % FT;
      sF[i] = k < nc && f < nf ? fo[(c0 + k) * m + f] : 0.f;
    }
    __syncthreads();
    tile_tn<2>(acc, sG, sF, -1.f);
    __syncthreads();
  }
  // the same sum over all columns: y . summary^T - delta * extra (queries), y . summary^T - extra (keys)
  float all[4][8];
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    float t[4][4] = {};
    const int f = f0 + 64 * c;
    tile_nt(t, y, a.side[SIDE].yr, nr, a.sum[SIDE] + ((int64_t)bh * m + f) * a.D, (int64_t)a.D, m - f, a.D, sA, sB);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) all[i][4 * c + j] = t[i][j];
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t row = row0 + ty * 4 + i;
    if (row >= rows) continue;
    const float d = SIDE == QUERIES ? delta[row] : 1.f;
    const float* f = a.feat[SIDE] + ((int64_t)bh * rows + row) * m;
    float* out = a.h + ((int64_t)bh * rows + row) * m;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int col = f0 + 64 * (j / 4) + 4 * tx + j % 4;
      if (col < m) out[col] = f[col] * ((all[i][j] - d * a.sum1[SIDE][(int64_t)bh * m + col]) + acc[i][j]);
    }
  }
}

// dq or dk: tau sum_in p g x' + (h_+ - h_-) Wt - tau x sum h; 64 rows, 64 NC columns of E
template <typename T, int SIDE, int NC>
__global__ void __launch_bounds__(NTHR) dx_kernel(GradArgs a) {
  extern __shared__ __align__(16) float smem[];
  float(*sA)[LDT] = reinterpret_cast<float(*)[LDT]>(smem);
  float(*sB)[LDT] = sA + KS;
  float(*sG)[LDT] = sB + KS;
  float* sX = &sG[TILE][0];                    // [64][64 NC]
  float* sH = sX + TILE * 64 * NC;             // [64] sum of h per row
  constexpr int OTHER = 1 - SIDE;
  const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
  const int bh = blockIdx.z, b = bh / a.H, h = bh % a.H;
  const int64_t row0 = (int64_t)blockIdx.x * TILE;
  const int rows = a.side[SIDE].rows, T_ = a.side[QUERIES].rows;
  const int nr = (int)min((int64_t)TILE, rows - row0);
  const int e0 = blockIdx.y * 64 * NC, m = 2 * a.r;
  const T* x = side_x<T>(a.side[SIDE], b, h, row0);
  const T* y = side_y<T>(a.side[SIDE], b, h, row0);
  const float* delta = a.delta + (int64_t)bh * T_;
  const float* lognorm = a.lognorm + (int64_t)bh * T_;
  const Window<SIDE> win(a, b, row0, nr);

  float acc[4][4 * NC] = {};
  for (int64_t c0 = win.lo; c0 <= win.hi; c0 += TILE) {
    const int nc = (int)min((int64_t)TILE, win.hi - c0 + 1);
    const T* xo = side_x<T>(a.side[OTHER], b, h, c0);
    float s[4][4] = {}, g[4][4] = {};
    tile_nt(s, x, a.side[SIDE].xr, nr, xo, a.side[OTHER].xr, nc, a.E, sA, sB);
    tile_nt(g, y, a.side[SIDE].yr, nr, side_y<T>(a.side[OTHER], b, h, c0), a.side[OTHER].yr, nc, a.D, sA, sB);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int ri = ty * 4 + i, cj = tx * 4 + j;
        float v = 0.f;
        if (ri < nr && cj < nc && win.in(row0 + ri, c0 + cj)) {
          const int64_t q = SIDE == QUERIES ? row0 + ri : c0 + cj;
          v = expf(a.tau * s[i][j] - lognorm[q]) * (g[i][j] - delta[q]);
        }
        sG[cj][ri] = v;
      }
    for (int i = threadIdx.x; i < TILE * 64 * NC; i += NTHR) {
      const int k = i / (64 * NC), e = e0 + i % (64 * NC);
      sX[i] = k < nc && e < a.E ? ldf(xo + k * a.side[OTHER].xr + e) : 0.f;
    }
    __syncthreads();
    tile_tn<NC>(acc, sG, sX, a.tau);
    __syncthreads();
  }
  // through the projection
  const float* hrow = a.h + ((int64_t)bh * rows + row0) * m;
  {
    const int row = threadIdx.x / 4, part = threadIdx.x % 4;
    float s = 0.f;
    if (row < nr)
      for (int f = part; f < m; f += 4) s += hrow[(int64_t)row * m + f];
    s += __shfl_xor_sync(0xffffffffu, s, 1);
    s += __shfl_xor_sync(0xffffffffu, s, 2);
    if (part == 0) sH[row] = s;
  }
  for (int k0 = 0; k0 < a.r; k0 += TILE) {
    __syncthreads();
    for (int i = threadIdx.x; i < TILE * TILE; i += NTHR) {
      const int row = i / TILE, k = i % TILE;
      sG[k][row] = row < nr && k0 + k < a.r
                       ? hrow[(int64_t)row * m + k0 + k] - hrow[(int64_t)row * m + a.r + k0 + k] : 0.f;
    }
    for (int i = threadIdx.x; i < TILE * 64 * NC; i += NTHR) {
      const int k = i / (64 * NC), e = e0 + i % (64 * NC);
      sX[i] = k0 + k < a.r && e < a.E ? a.Wt[(int64_t)(k0 + k) * a.E + e] : 0.f;
    }
    __syncthreads();
    tile_tn<NC>(acc, sG, sX, 1.f);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int ri = ty * 4 + i;
    if (ri >= nr) continue;
    T* out = static_cast<T*>(a.dx) + b * a.dxb + h * a.dxh + (row0 + ri) * a.dxr;
    const float hs = a.tau * sH[ri];
#pragma unroll
    for (int j = 0; j < 4 * NC; ++j) {
      const int e = e0 + 64 * (j / 4) + 4 * tx + j % 4;
      if (e < a.E) stf(out + e, acc[i][j] - hs * ldf(x + ri * a.side[SIDE].xr + e));
    }
  }
}

// dv: sum_in (p - psi.phi) dout + phi . QG; 64 key rows, 64 NC columns of D
template <typename T, int NC>
__global__ void __launch_bounds__(NTHR) dv_kernel(GradArgs a) {
  extern __shared__ __align__(16) float smem[];
  float(*sA)[LDT] = reinterpret_cast<float(*)[LDT]>(smem);
  float(*sB)[LDT] = sA + KS;
  float(*sG)[LDT] = sB + KS;
  float* sX = &sG[TILE][0];                    // [64][64 NC]
  const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
  const int bh = blockIdx.z, b = bh / a.H, h = bh % a.H;
  const int64_t row0 = (int64_t)blockIdx.x * TILE;
  const int rows = a.side[KEYS].rows, T_ = a.side[QUERIES].rows;
  const int nr = (int)min((int64_t)TILE, rows - row0);
  const int m = 2 * a.r;
  const T* x = side_x<T>(a.side[KEYS], b, h, row0);
  const float* lognorm = a.lognorm + (int64_t)bh * T_;
  const float* phi = a.feat[KEYS] + ((int64_t)bh * rows + row0) * m;
  const float* psi = a.feat[QUERIES] + (int64_t)bh * T_ * m;
  const Window<KEYS> win(a, b, row0, nr);

  float acc[4][4 * NC] = {};
  for (int64_t c0 = win.lo; c0 <= win.hi; c0 += TILE) {
    const int nc = (int)min((int64_t)TILE, win.hi - c0 + 1);
    float s[4][4] = {}, l[4][4] = {};
    tile_nt(s, x, a.side[KEYS].xr, nr, side_x<T>(a.side[QUERIES], b, h, c0), a.side[QUERIES].xr, nc, a.E, sA, sB);
    tile_nt(l, phi, (int64_t)m, nr, psi + c0 * m, (int64_t)m, nc, m, sA, sB);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int ri = ty * 4 + i, cj = tx * 4 + j;
        const bool in = ri < nr && cj < nc && win.in(row0 + ri, c0 + cj);
        sG[cj][ri] = in ? expf(a.tau * s[i][j] - lognorm[c0 + cj]) - l[i][j] : 0.f;
      }
    const T* y = side_y<T>(a.side[QUERIES], b, h, c0);
    for (int i = threadIdx.x; i < TILE * 64 * NC; i += NTHR) {
      const int k = i / (64 * NC), d = i % (64 * NC);
      sX[i] = k < nc && d < a.D ? ldf(y + k * a.side[QUERIES].yr + d) : 0.f;
    }
    __syncthreads();
    tile_tn<NC>(acc, sG, sX, 1.f);
    __syncthreads();
  }
  for (int f0 = 0; f0 < m; f0 += TILE) {
    __syncthreads();
    for (int i = threadIdx.x; i < TILE * TILE; i += NTHR) {
      const int row = i / TILE, k = i % TILE;
      sG[k][row] = row < nr && f0 + k < m ? phi[(int64_t)row * m + f0 + k] : 0.f;
    }
    for (int i = threadIdx.x; i < TILE * 64 * NC; i += NTHR) {
      const int k = i / (64 * NC), d = i % (64 * NC);
      sX[i] = f0 + k < m && d < a.D ? a.sum[KEYS][((int64_t)bh * m + f0 + k) * a.D + d] : 0.f;
    }
    __syncthreads();
    tile_tn<NC>(acc, sG, sX, 1.f);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int ri = ty * 4 + i;
    if (ri >= nr) continue;
    T* out = static_cast<T*>(a.dx) + b * a.dxb + h * a.dxh + (row0 + ri) * a.dxr;
#pragma unroll
    for (int j = 0; j < 4 * NC; ++j) {
      const int d = 64 * (j / 4) + 4 * tx + j % 4;
      if (d < a.D) stf(out + d, acc[i][j]);
    }
  }
}

constexpr size_t smem_of(int cols) { return sizeof(float) * (2 * KS * LDT + TILE * LDT + TILE * cols + TILE); }

template <typename K>
cudaError_t run(K kernel, dim3 grid, int cols, const GradArgs& a, cudaStream_t st) {
  const size_t smem = smem_of(cols);
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  kernel<<<grid, NTHR, smem, st>>>(a);
  return cudaGetLastError();
}

template <typename T, int SIDE>
cudaError_t side_grads(const SblParams& p, GradArgs a, cudaStream_t st) {
  const unsigned tiles = (unsigned)div_up(a.side[SIDE].rows, TILE), bh = (unsigned)(p.B * p.H);
  cudaError_t e = run(dfeat_kernel<T, SIDE>, dim3(tiles, (unsigned)div_up(2 * p.r, FT), bh), FT, a, st);
  if (e != cudaSuccess) return e;
  if (p.E <= 64) return run(dx_kernel<T, SIDE, 1>, dim3(tiles, 1, bh), 64, a, st);
  return run(dx_kernel<T, SIDE, 2>, dim3(tiles, (unsigned)div_up(p.E, 128), bh), 128, a, st);
}

template <typename T>
cudaError_t grads(const SblParams& p, const SblGrads& g, GradArgs a, cudaStream_t st) {
  const unsigned bh = (unsigned)(p.B * p.H);
  a.dx = g.dv; a.dxb = g.dv_stride_b; a.dxr = g.dv_stride_s; a.dxh = g.dv_stride_h;
  const dim3 grid((unsigned)div_up(p.S, TILE), 1, bh);
  cudaError_t e = p.D <= 64 ? run(dv_kernel<T, 1>, grid, 64, a, st) : run(dv_kernel<T, 2>, grid, 128, a, st);
  if (e != cudaSuccess) return e;
  a.dx = g.dq; a.dxb = g.dq_stride_b; a.dxr = g.dq_stride_t; a.dxh = g.dq_stride_h;
  if ((e = side_grads<T, QUERIES>(p, a, st)) != cudaSuccess) return e;
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
  auto split = [](int rows, int* per) {   // at most 64 splits, at least 256 rows each (as in the forward)
    *per = 256;
    while (div_up(rows, *per) > 64) *per *= 2;
    return (int)div_up(rows, *per);
  };
  f.nsplit = split(p.S, &f.split_rows);
  ws->nsplit = split(p.T, &ws->split_rows);
  f.wt = take((size_t)p.r * p.E * 4);
  f.phik = take(BH * S * m * 4);
  f.beta = take(BH * 4);
  f.kv = take(BH * m * p.D * 4);
  f.ksum = take(BH * m * 4);
  f.partial = take(BH * f.nsplit * m * (p.D + 1) * 4);
  ws->lognorm = take(BH * T * 4);
  ws->scale = take(BH * T * 4);
  ws->delta = take(BH * T * 4);
  ws->psi = take(BH * T * m * 4);
  ws->qg = take(BH * m * p.D * 4);
  ws->qd = take(BH * m * 4);
  ws->h = take(BH * (T > S ? T : S) * m * 4);
  ws->partial = take(BH * ws->nsplit * m * (p.D + 1) * 4);
  f.total = ws->total = off;
}

cudaError_t f32_backward(const SblParams& p, const SblGrads& g, const BwdWorkspace& ws, char* base, cudaStream_t st) {
  float* beta = reinterpret_cast<float*>(base + ws.fwd.beta);
  float* phi = reinterpret_cast<float*>(base + ws.fwd.phik);
  float* kv = reinterpret_cast<float*>(base + ws.fwd.kv);
  float* ksum = reinterpret_cast<float*>(base + ws.fwd.ksum);
  float* lognorm = reinterpret_cast<float*>(base + ws.lognorm);
  float* scale = reinterpret_cast<float*>(base + ws.scale);
  float* delta = reinterpret_cast<float*>(base + ws.delta);
  float* psi = reinterpret_cast<float*>(base + ws.psi);
  float* qg = reinterpret_cast<float*>(base + ws.qg);
  float* qd = reinterpret_cast<float*>(base + ws.qd);
  cudaError_t e;
  if ((e = f32_prepare_projection(p, ws.fwd, base, st)) != cudaSuccess) return e;
  if ((e = f32_key_logscale(p, ws.fwd, base, beta, st)) != cudaSuccess) return e;
  if ((e = f32_key_features(p, ws.fwd, base, beta, phi, st)) != cudaSuccess) return e;
  if ((e = f32_key_summary(p, ws.fwd, base, phi, kv, ksum, st)) != cudaSuccess) return e;
  const unsigned blocks = (unsigned)div_up((int64_t)p.B * p.H * p.T, 8);
  if (p.dtype == SBL_DTYPE_F32) row_kernel<float><<<blocks, 256, 0, st>>>(p, g, beta, lognorm, scale, delta);
  else row_kernel<__nv_bfloat16><<<blocks, 256, 0, st>>>(p, g, beta, lognorm, scale, delta);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  if ((e = f32_query_features_over(p, ws.fwd, base, scale, psi, st)) != cudaSuccess) return e;
  if ((e = f32_query_summary(p, g, psi, delta, ws.split_rows, ws.nsplit, reinterpret_cast<float*>(base + ws.partial),
                             qg, qd, st)) != cudaSuccess)
    return e;
  GradArgs a{};
  a.side[QUERIES] = {p.q, g.dout, p.q_stride_b, p.q_stride_t, p.q_stride_h, g.do_stride_b, g.do_stride_t,
                     g.do_stride_h, p.T};
  a.side[KEYS] = {p.k, p.v, p.k_stride_b, p.k_stride_s, p.k_stride_h, p.v_stride_b, p.v_stride_s, p.v_stride_h, p.S};
  a.lengths = p.key_lengths;
  a.lognorm = lognorm;
  a.delta = delta;
  a.feat[QUERIES] = psi;
  a.feat[KEYS] = phi;
  a.sum[QUERIES] = kv;
  a.sum[KEYS] = qg;
  a.sum1[QUERIES] = ksum;
  a.sum1[KEYS] = qd;
  a.h = reinterpret_cast<float*>(base + ws.h);
  a.Wt = reinterpret_cast<const float*>(base + ws.fwd.wt);
  a.H = p.H; a.E = p.E; a.D = p.D; a.r = p.r; a.w = p.w;
  a.tau = p.softmax_temp;
  return p.dtype == SBL_DTYPE_F32 ? grads<float>(p, g, a, st) : grads<__nv_bfloat16>(p, g, a, st);
}

}  // namespace sbl
