// bf16 tensor-core path of the SBLocal gradients for sm_100a: E = D = 64,
// r = 128 (m = 256) and E = D = 128, r = 256 (m = 512), eps = 0, any T, S, w and
// key lengths.  The formulas are those at the top of sbl_bwd_f32.cu.
//
// Kernels (rows = the side a CTA's 128-row tiles belong to, columns = the other)
//   rows      delta = dout . out and the log-normaliser (base 2) of every query
//   feat      per (split, block of 128 features, b*h): U = X Wt^T, the features
//             phi (keys) or psi (queries, over the row's normaliser) -> bf16 to the
//             workspace, and the summary phi^T [V | 1] or psi^T [dout | delta]
//   combine   sums the splits -> summary in bf16, its extra column in fp32
//   window    (head dim 128) exact part of dq or dk: S = X X'^T, G = Y Y'^T, p (G - delta) -> bf16,
//             dx += (p g) X', over the 64-column steps of the window -> fp32
//   dvalue    S = K Q^T -> p, minus phi psi^T (same buffer, A operand negated),
//             packed, dv += (p - a) dout; dv += phi QG
//   grad      G = Y Y'^T - delta -> bf16, df -= G f' over the window (256 features at a time in tensor
//             memory), df += Y summary^T; U = X Wt^T, du = (f df)_+ - (f df)_-, dx += du Wt; writes dq or dk.
//             Head dim 64: the exact part too (S beside G, dx += (p g) X'); 128: adds the window kernel's
//
// Measured, us: B2 H16 N16384 d64 w256 | B1 H8 N32768 d128 w512
//   rows 30 | 26   feat, queries and keys 101 + 94 | 169 + 163   combine 2 x 3.5 | 2 x 8   window - | 179 + 189
//   dvalue 215 | 307   grad, queries and keys 268 + 300 | 371 + 390
// The tensor core is busy for 20 (feat) to 43 % (grad) of that; what bounds each kernel stands beside it.
//
// Numerics.  Products take bf16 operands and accumulate in fp32.  Rounded to bf16
// (half a step, 2^-9 on average): phi and psi as operands, g, p g, p - a.  Carried
// as two bf16 terms (16 bits): the projection, the summaries and du -- each alone
// would add as much to the error of dq and dk as the features do.  The own
// features of a row are formed again in fp32 for du instead of being read back.
//
// Where a tile's columns are few (`whole`), df is summed over the columns
// OUTSIDE the window directly instead of all - inside: a short sequence lies
// inside its windows almost entirely, and the difference of two sums of bf16
// products would leave their rounding where the exact value is next to nothing.
//
// Feature order: block of 128 = "+" features of 64 projections, then their "-".
// All waits are bounded (mbar_wait, wait_inline): a wait that runs out sets the first word of
// the workspace and the kernel runs to its end.
#include "sbl_common.cuh"
#include "sbl_tc_dev.cuh"
#include "sbl_tc_host.cuh"
#include "sbl_bwd_walk.cuh"

namespace sbl {
namespace {

using namespace ptx;
using namespace tcdev;
using namespace tch;

__device__ __forceinline__ uint32_t bits(int lo, int hi) {   // bits lo..hi of a word, clipped
  lo = max(lo, 0);
  hi = min(hi, 31);
  return hi >= lo ? (0xFFFFFFFFu >> (31 - (hi - lo))) << lo : 0u;
}
// Which of the 32 columns from c on row `row` has in its window; with `whole`, the real ones outside it.
template <int SIDE>
__device__ __forceinline__ uint32_t seen(const Geom& g, const RowTile& t, int row, int c, bool whole) {
  const int hw = g.w / 2;
  if (SIDE == QUERIES) {
    const uint32_t real = bits(0, t.len - 1 - c);
    const uint32_t in = bits(row - hw - c, row - hw + g.w - 1 - c) & real;
    return whole ? real & ~in : in;
  }
  const uint32_t real = row < t.len ? bits(0, g.T - 1 - c) : 0u;
  const uint32_t in = bits(row + hw - g.w + 1 - c, row + hw - c) & real;
  return whole ? real & ~in : in;
}

__device__ __forceinline__ uint8_t* align1024(uint8_t* p) {
  return reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(p) + 1023) & ~(uintptr_t)1023);
}
// Whether a phase is over, without waiting.
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.b32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
// mbar_wait without the call.  A call makes the issuing warp rebuild every matrix descriptor behind it: about 130
// cycles per group of four MMAs (256 cycles of work at N = 128), 30 with the loop in line.  The loop stays a loop: the
// compiler unrolls it by four at some forty waits of a kernel, a sixth of the code, and what does not fit the
// instruction cache is paid for in every tile (grad 293 + 325 -> 273 + 300 us, dvalue 226 -> 215).
__device__ __forceinline__ void wait_inline(uint64_t* bar, uint32_t parity, int* status, int code) {
  uint32_t n = 0;
#pragma unroll 1
  while (!mbar_try_wait(bar, parity)) {
    ++n;
    if (n >= kWaitLimit || ((n & 255u) == 255u && *reinterpret_cast<volatile int*>(status) != 0)) {
      atomicCAS(status, 0, code);
      break;
    }
  }
}
// untiled bulk copy to shared memory: both addresses and the size are multiples of 16 bytes
__device__ __forceinline__ void bulk_load(void* smem, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(smem)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
// ---------------------------------------------------------------------------
// Per query row: (log-normaliser * log2(e), delta = dout . out), (BH, Tp); zero in the padding rows.  Head dim 128:
// delta once more by itself.
// A block owns 32 positions of up to 16 heads: it reads them heads innermost, as they lie in memory, D / 8 lanes per row
// and four rows per group of lanes with all their loads in flight, and writes the results by head through shared
// memory, 256 bytes at a time.  (Written one by one, a plane apart: 46 us where this takes 30, B2 H16 N16384.)
constexpr int kRowHeads = 16, kRowSpan = 32;
template <int D>
__global__ void __launch_bounds__(256) bwd_rows_kernel(const __nv_bfloat16* out, int64_t ob, int64_t ot, int64_t oh,
                                                       const __nv_bfloat16* dout, int64_t db, int64_t dt, int64_t dh,
                                                       const float* stats, int B, int H, int T, int Tp, float2* nd,
                                                       float* delta) {
  constexpr int LPR = D / 8, RPB = 256 / LPR;
  __shared__ float s_delta[kRowHeads][kRowSpan + 1];
  const int sub = threadIdx.x % LPR, slot = threadIdx.x / LPR;
  const int t0 = blockIdx.x * kRowSpan, h0 = blockIdx.y * kRowHeads, b = blockIdx.z;
  const int nh = min(kRowHeads, H - h0), n = nh * kRowSpan;
  out += b * ob;
  dout += b * db;
  for (int base = 0; base < n; base += 4 * RPB) {
    uint4 x[4], y[4];
    int h[4], t[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = base + u * RPB + slot;
      t[u] = i / nh;
      h[u] = i - t[u] * nh;
      x[u] = y[u] = make_uint4(0, 0, 0, 0);
      if (i < n && t0 + t[u] < T) {
        x[u] = __ldg(reinterpret_cast<const uint4*>(out + (t0 + t[u]) * ot + (h0 + h[u]) * oh) + sub);
        y[u] = __ldg(reinterpret_cast<const uint4*>(dout + (t0 + t[u]) * dt + (h0 + h[u]) * dh) + sub);
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const uint32_t xw[4] = {x[u].x, x[u].y, x[u].z, x[u].w}, yw[4] = {y[u].x, y[u].y, y[u].z, y[u].w};
      float s = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s = fmaf(bf16_lo(xw[j]), bf16_lo(yw[j]), s);
        s = fmaf(bf16_hi(xw[j]), bf16_hi(yw[j]), s);
      }
#pragma unroll
      for (int o = 1; o < LPR; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      if (sub == 0 && base + u * RPB + slot < n) s_delta[h[u]][t[u]] = s;
    }
  }
  __syncthreads();
  const int64_t rows = (int64_t)B * H * T;
  for (int i = threadIdx.x; i < n; i += 256) {
    const int h = i / kRowSpan, t = t0 + i % kRowSpan;      // (t < Tp, a multiple of kRowSpan)
    const int64_t bh = (int64_t)b * H + h0 + h;
    const float s = s_delta[h][i % kRowSpan];
    float m = 0.f;
    if (t < T) m = stats[bh * T + t] * kLog2e + log2f(stats[rows + bh * T + t]);
    nd[bh * Tp + t] = make_float2(m, s);
    if (D == 128) delta[bh * Tp + t] = s;
  }
}

// ---------------------------------------------------------------------------
// Features and summary of one side.
struct FeatArgs {
  CUtensorMap tm_x, tm_y, tm_hi, tm_lo, tm_f;
  const int64_t* lengths;
  const float* beta;                // (BH)
  const float2* nd;                 // (BH, Tp): log-normaliser (base 2) and delta of every query row
  float* off;                       // (BH, rows padded to tiles): exponent offset (base 2) of every row, -inf if padding
  float* partial;                   // (BH, nsplit, m, D + 4)
  int* status;
  int H, rows, Tp, nsplit;
  float tau, half_log_m;
};

template <int D>
struct FeatCfg {
  static constexpr int NB = D / 64, M = 4 * D, XD = D == 64 ? 2 : 1;
  static constexpr uint32_t WB = NB * 8192;              // one bf16 term of 64 projections
  static constexpr uint32_t XB = NB * 16384, YB = (NB + 1) * 16384;
  static constexpr uint32_t OFF_W = 0, OFF_X = 2 * WB, OFF_Y = OFF_X + XD * XB, OFF_A = OFF_Y + 2 * YB;
  static constexpr uint32_t OFF_BAR = OFF_A + 2 * 32768;
  static constexpr uint32_t SMEM = OFF_BAR + 256 + 1024;
  // Groups of eight warps that take the tiles in turn.  Head dim 64: two (110 and 94 us for queries and keys, with one 127
  // and 100: B2 H16 N16384).  128 has room for one X tile only and waits for that: 169 and 163 us with one, 171 and 170
  // with two (B1 H8 N32768).
  static constexpr int GROUPS = D == 64 ? 2 : 1;
  static constexpr int NFEAT = 256 * GROUPS, NTHR = NFEAT + 64, W_LOAD = NFEAT / 32, W_MMA = W_LOAD + 1;
  static constexpr uint32_t T_U = 0, T_SUM = 128;        // 2 x 64 | D + 16
  static_assert(GROUPS <= XD, "a group sees every phase of the X slots it reads");
  static_assert(SMEM <= 232448, "dynamic shared memory of one CTA");
};

template <int SIDE, int D>
__global__ void __launch_bounds__(FeatCfg<D>::NTHR, 1) bwd_feat_kernel(const __grid_constant__ FeatArgs a) {
  using C = FeatCfg<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align1024(smem_raw);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  uint64_t *bar_w = bars, *bar_done = bars + 1, *x_full = bars + 2, *x_free = bars + 4, *y_full = bars + 6,
           *y_free = bars + 8, *u_full = bars + 10, *u_free = bars + 12, *a_full = bars + 14, *a_free = bars + 16;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 18);
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int fb = blockIdx.x % (C::M / 128), split = blockIdx.x / (C::M / 128);
  const int bh = blockIdx.y, b = bh / a.H, h = bh % a.H;
  const int ntiles = (a.rows + TR - 1) / TR;
  const int t_lo = (int)((int64_t)ntiles * split / a.nsplit), t_hi = (int)((int64_t)ntiles * (split + 1) / a.nsplit);
  const int nt = t_hi - t_lo;

  if (tid == 0) {
    mbar_init(bar_w, 1);
    mbar_init(bar_done, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(x_full + i, 1);
      mbar_init(x_free + i, 8);
      mbar_init(y_full + i, 1);
      mbar_init(y_free + i, 1);
      mbar_init(u_full + i, 1);
      mbar_init(u_free + i, 8);
      mbar_init(a_full + i, 8);
      mbar_init(a_free + i, 2);
    }
    fence_mbar_init();
  }
  if (warp == C::W_LOAD) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  // the extra summary column's operand behind each Y slot: ones (keys), or delta per row, written with the features
  for (int i = tid; i < 2 * 8192; i += C::NTHR)
    reinterpret_cast<__nv_bfloat16*>(smem + C::OFF_Y + (i / 8192) * C::YB + C::NB * 16384)[i % 8192] =
        __float2bfloat16(SIDE == KEYS ? 1.f : 0.f);
  fence_async_smem();
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  constexpr uint32_t tb = 0;   // the CTA owns all 512 tensor-memory columns of its SM
  if (tid == 0 && *tmem_slot != 0) atomicCAS(a.status, 0, 241);

  if (warp == C::W_LOAD) {
    const bool leader = elect_one();
    if (leader) {
      mbar_expect_tx(bar_w, 2 * C::WB);
      for (int j = 0; j < C::NB; ++j) {
        tma_load_2d(smem + C::OFF_W + j * 8192, &a.tm_hi, bar_w, 64 * j, 64 * fb);
        tma_load_2d(smem + C::OFF_W + C::WB + j * 8192, &a.tm_lo, bar_w, 64 * j, 64 * fb);
      }
    }
    // X runs one tile ahead of Y: a Y slot is freed by the summary of two tiles back, an X slot long before
    for (int i = 0; i <= nt; ++i) {
      if (i < nt) {
        const int xs = i % C::XD;
        if (i >= C::XD) wait_inline(x_free + xs, ((i / C::XD) - 1) & 1, a.status, 201);
        if (leader) {
          mbar_expect_tx(x_full + xs, C::XB);
          for (int j = 0; j < C::NB; ++j)
            tma_load_4d(smem + C::OFF_X + xs * C::XB + j * 16384, &a.tm_x, x_full + xs, 64 * j, (t_lo + i) * TR, h, b);
        }
      }
      if (i >= 1) {
        const int y = i - 1, s = y & 1;
        if (y >= 2) wait_inline(y_free + s, ((y >> 1) - 1) & 1, a.status, 202);
        if (leader) {
          mbar_expect_tx(y_full + s, C::XB);
          for (int j = 0; j < C::NB; ++j)
            tma_load_4d(smem + C::OFF_Y + s * C::YB + j * 16384, &a.tm_y, y_full + s, 64 * j, (t_lo + y) * TR, h, b);
        }
      }
    }
    __syncwarp();
  } else if (warp == C::W_MMA) {
    const bool leader = elect_one();
    constexpr uint32_t id_u = idesc_bf16(128, 64, false, false);
    constexpr uint32_t id_s = idesc_bf16(128, D + 16, true, true);
    const uint64_t dW = smem_desc_sw128(smem_u32(smem + C::OFF_W), 16, 1024);
    const uint64_t dX = smem_desc_sw128(smem_u32(smem + C::OFF_X), 16, 1024);
    const uint64_t dY = smem_desc_sw128(smem_u32(smem + C::OFF_Y), 16384, 1024);
    const uint64_t dA = smem_desc_sw128(smem_u32(smem + C::OFF_A), 16384, 1024);
    auto summary = [&](int u) {
      const int s = u & 1;
      wait_inline(a_full + s, (u >> 1) & 1, a.status, 203);
      wait_inline(y_full + s, (u >> 1) & 1, a.status, 204);
      tc_fence_after_sync();
      if (leader) {
        tma_store_3d(&a.tm_f, smem + C::OFF_A + s * 32768, 128 * fb, (t_lo + u) * TR, bh);
        tma_store_3d(&a.tm_f, smem + C::OFF_A + s * 32768 + 16384, 128 * fb + 64, (t_lo + u) * TR, bh);
        tma_store_commit();
#pragma unroll
        for (int k = 0; k < 8; ++k)
          mma_ss(tb + C::T_SUM, dA + (uint64_t)(s * (32768 >> 4) + k * 128), dY + (uint64_t)(s * (C::YB >> 4) + k * 128),
                 id_s, u > 0 || k > 0);
        mma_commit(a_free + s);
        mma_commit(y_free + s);
        // the previous tile's bulk store has read its buffer once at most one group is pending
        if (u >= 1) {
          tma_store_wait_read1();
          mbar_arrive(a_free + (s ^ 1));
        }
      }
      __syncwarp();
    };
    wait_inline(bar_w, 0, a.status, 205);
    for (int i = 0; i < nt; ++i) {
      const int s = i & 1, xs = i % C::XD;
      wait_inline(x_full + xs, (i / C::XD) & 1, a.status, 206);
      if (i >= 2) wait_inline(u_free + s, ((i >> 1) - 1) & 1, a.status, 207);
      tc_fence_after_sync();
      if (leader) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int k = 0; k < D / 16; ++k)
            mma_ss(tb + C::T_U + 64 * s, dX + (uint64_t)(xs * (C::XB >> 4)) + kmajor(k, 16384),
                   dW + (uint64_t)(t * (C::WB >> 4)) + kmajor(k, 8192), id_u, t > 0 || k > 0);
        mma_commit(u_full + s);
      }
      __syncwarp();
      if (i >= 1) summary(i - 1);
    }
    if (nt > 0) summary(nt - 1);
    if (leader) {
      mma_commit(bar_done);
      tma_store_wait_all();
    }
    __syncwarp();
  } else {
    // a thread owns a row and 32 of the block's 64 projections
    const int grp = warp >> 3, qd = warp & 3, cq = (warp >> 2) & 1;
    const int row = qd * 32 + lane;
    const uint32_t lane_base = tb + ((uint32_t)(qd * 32) << 16);
    const float beta = a.beta[bh];
    // Padded keys have no features.  Nor have the queries of a batch without keys: over the floor of their normaliser
    // (1e-37) they would be so large that their sums leave the fp32 range, and zero weights do not hide that.
    int len = a.rows;
    if (a.lengths) {
      const int64_t l = a.lengths[b];
      if (l <= 0) len = 0;
      else if (SIDE == KEYS && l < a.rows) len = (int)l;
    }
    const float2* nd = a.nd + (int64_t)bh * a.Tp;
    for (int i = grp; i < nt; i += C::GROUPS) {
      const int s = i & 1, xs = i % C::XD;
      const int r = (t_lo + i) * TR + row;
      float2 own = make_float2(0.f, 0.f);
      if (SIDE == QUERIES) own = __ldg(nd + r);   // r < Tp: the row arrays are padded to whole tiles
      mbar_wait(x_full + xs, (i / C::XD) & 1, a.status, 208);
      float sq = 0.f;
#pragma unroll
      for (int j = 0; j < C::NB; ++j) sq += row_sumsq_sw128(smem + C::OFF_X + xs * C::XB + j * 16384, row);
      const float g = 0.5f * a.tau * sq;
      const bool live = r < len;
      float off, dl = 0.f;
      if (SIDE == KEYS) {
        off = (-g - a.half_log_m - beta) * kLog2e;
      } else {
        off = (-g - a.half_log_m + beta) * kLog2e - own.x;
        dl = own.y;
      }
      if (fb == 0 && cq == 0) a.off[((int64_t)bh * ntiles + t_lo + i) * TR + row] = live ? off : -INFINITY;
      mbar_wait(u_full + s, (i >> 1) & 1, a.status, 209);   // U computed: the X tile has been read too
      tc_fence_after_sync();
      warp_arrive(x_free + xs, lane);
      uint32_t u[32];
      tmem_ld32(lane_base + C::T_U + 64 * s + 32 * cq, u);
      tmem_ld_wait();
      tc_fence_before_sync();
      warp_arrive(u_free + s, lane);
      uint32_t p1[16], p2[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const float x = __uint_as_float(u[2 * j]), y = __uint_as_float(u[2 * j + 1]);
        const uint32_t e = pack_bf16(ex2(fmaf(x, kLog2e, off)), ex2(fmaf(y, kLog2e, off)));
        const uint32_t f = pack_bf16(ex2(fmaf(x, -kLog2e, off)), ex2(fmaf(y, -kLog2e, off)));
        p1[j] = live ? e : 0u;
        p2[j] = live ? f : 0u;
      }
      // the MMAs and the bulk store two tiles back are done with this buffer (and with the Y slot's extra column)
      if (i >= 2) mbar_wait(a_free + s, ((i >> 1) - 1) & 1, a.status, 210);
      uint8_t* line = smem + C::OFF_A + s * 32768 + row * 128;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const uint32_t at = (uint32_t)(((4 * cq + c) ^ (row & 7)) << 4);
        *reinterpret_cast<uint4*>(line + at) = make_uint4(p1[4 * c], p1[4 * c + 1], p1[4 * c + 2], p1[4 * c + 3]);
        *reinterpret_cast<uint4*>(line + 16384 + at) = make_uint4(p2[4 * c], p2[4 * c + 1], p2[4 * c + 2], p2[4 * c + 3]);
      }
      if (SIDE == QUERIES) {
        // delta in two bf16 terms: columns 0, 2, .. the high one, 1, 3, .. the low one
        const float hi = __bfloat162float(__float2bfloat16_rn(dl));
        const uint32_t w = pack_bf16(hi, dl - hi);
        *reinterpret_cast<uint4*>(smem + C::OFF_Y + s * C::YB + C::NB * 16384 + row * 128 + ((cq ^ (row & 7)) << 4)) =
            make_uint4(w, w, w, w);
      }
      fence_async_smem();
      warp_arrive(a_full + s, lane);
    }
    mbar_wait(bar_done, 0, a.status, 211);
    tc_fence_after_sync();
    float* prow = a.partial + (((int64_t)bh * a.nsplit + split) * C::M + 128 * fb + row) * (D + 4);
#pragma unroll
    for (int j = 0; j < D / (32 * C::GROUPS); ++j) {
      uint32_t r[16];
      const int c = (D / (2 * C::GROUPS)) * (2 * grp + cq) + 16 * j;
      tmem_ld16(lane_base + C::T_SUM + c, r);
      tmem_ld_wait();
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<uint4*>(prow + c + 4 * q) = nt ? make_uint4(r[4 * q], r[4 * q + 1], r[4 * q + 2], r[4 * q + 3])
                                                         : make_uint4(0, 0, 0, 0);
    }
    uint32_t r[16];
    tmem_ld16(lane_base + C::T_SUM + D, r);
    tmem_ld_wait();
    if (cq == 0 && grp == 0) prow[D] = nt == 0 ? 0.f : __uint_as_float(r[0]) + (SIDE == QUERIES ? __uint_as_float(r[1]) : 0.f);
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == C::W_LOAD) {
    __syncwarp();
    tmem_dealloc(tb, 512);
  }
}

// summary (BH, m, D) in two bf16 terms and its extra column (BH, m) fp32 = sums over the splits
template <int D>
__global__ void __launch_bounds__(256) bwd_combine_kernel(const float* partial, int nsplit, int64_t rows, int m,
                                                          __nv_bfloat16* sum, __nv_bfloat16* sum_lo, float* sum1) {
  constexpr int G = D / 4 + 1;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= rows * G) return;
  const int64_t row = i / G, bh = row / m;
  const int g = (int)(i % G);
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int k = 0; k < nsplit; ++k) {
    const float* p = partial + ((bh * nsplit + k) * m + row % m) * (D + 4) + 4 * g;
    if (g < D / 4) {
      const float4 x = *reinterpret_cast<const float4*>(p);
      v.x += x.x; v.y += x.y; v.z += x.z; v.w += x.w;
    } else {
      v.x += *p;
    }
  }
  if (g < D / 4) {
    const uint2 hi = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
    *reinterpret_cast<uint2*>(sum + row * D + 4 * g) = hi;
    *reinterpret_cast<uint2*>(sum_lo + row * D + 4 * g) =
        make_uint2(pack_bf16(v.x - bf16_lo(hi.x), v.y - bf16_hi(hi.x)), pack_bf16(v.z - bf16_lo(hi.y), v.w - bf16_hi(hi.y)));
  } else {
    sum1[row] = v.x;
  }
}

// ---------------------------------------------------------------------------
// Exact part of dq or dk.
struct WinArgs {
  CUtensorMap tm_x, tm_y, tm_xo, tm_yo;   // own side (128 rows), other side (64 rows)
  Geom g;
  const float2* nd;                       // (BH, Tp)
  float* part;                            // (tiles, D / 4, 128 rows) float4
  int* status;
  int Tp;
  float tau;
};

template <int D>
struct WinCfg {
  static_assert(D == 128, "head dim 64 has its exact part in the gradient kernel");
  static constexpr int NB = D / 64, NS = 3;
  static constexpr uint32_t TB = NB * 16384, SLOT = 2 * NB * 8192;
  static constexpr uint32_t OFF_X = 0, OFF_Y = 2 * TB, OFF_RING = 4 * TB, OFF_BAR = OFF_RING + NS * SLOT;
  static constexpr uint32_t SMEM = OFF_BAR + 512 + 1024;
  static constexpr int NTHR = 576, W_LOAD = 16, W_MMA = 17;
  static constexpr uint32_t T_DX = 256;   // buffers: S at 128 b, G at 128 b + 64; dx at 256 + D b
  enum { XY_FULL = 0, XY_FREE = 2, R_FULL = 4, R_FREE = R_FULL + NS, ST_FULL = R_FREE + NS, DS_DONE = ST_FULL + 2,
         DX_FULL = DS_DONE + 2, DX_FREE = DX_FULL + 2, COUNT = DX_FREE + 2 };
  static_assert(SMEM <= 232448 && COUNT <= 60, "shared memory of one CTA");
};

// Bound: the chain of a step (S and G -> p g -> dx) over two buffers, 2.3 k cycles per step with 1.1 k of products; the
// 32 KB that a step brings in take 0.8 k.
template <int SIDE, int D>
__global__ void __launch_bounds__(576, 1) bwd_window_kernel(const __grid_constant__ WinArgs a) {
  using C = WinCfg<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align1024(smem_raw);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + C::COUNT);
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  if (tid == 0) {
    for (int i = 0; i < C::COUNT; ++i)
      mbar_init(bars + i, i >= C::DX_FREE ? 16 : (i >= C::DS_DONE && i < C::DX_FULL ? 8 : 1));
    fence_mbar_init();
  }
  if (warp == C::W_LOAD) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  constexpr uint32_t tb = 0;
  if (tid == 0 && *tmem_slot != 0) atomicCAS(a.status, 0, 241);
  const int step = gridDim.x;

  if (warp == C::W_LOAD) {
    const bool leader = elect_one();
    int n = 0, ne = 0;
    for (int tile = blockIdx.x; tile < a.g.ntiles; tile += step) {
      const RowTile t = row_tile<SIDE, 64>(a.g, tile, false);
      if (t.n == 0) continue;
      const int buf = ne & 1;
      if (ne >= 2) wait_inline(bars + C::XY_FREE + buf, ((ne >> 1) - 1) & 1, a.status, 221);
      if (leader) {
        mbar_expect_tx(bars + C::XY_FULL + buf, 2 * C::TB);
        for (int j = 0; j < C::NB; ++j) {
          tma_load_4d(smem + C::OFF_X + buf * C::TB + j * 16384, &a.tm_x, bars + C::XY_FULL + buf, 64 * j, t.r0, t.h, t.b);
          tma_load_4d(smem + C::OFF_Y + buf * C::TB + j * 16384, &a.tm_y, bars + C::XY_FULL + buf, 64 * j, t.r0, t.h, t.b);
        }
      }
      ++ne;
      for (int s = 0; s < t.n; ++s, ++n) {
        const int slot = n % C::NS;
        if (n >= C::NS) wait_inline(bars + C::R_FREE + slot, ((n / C::NS) - 1) & 1, a.status, 222);
        if (leader) {
          uint8_t* dst = smem + C::OFF_RING + slot * C::SLOT;
          mbar_expect_tx(bars + C::R_FULL + slot, C::SLOT);
          for (int j = 0; j < C::NB; ++j) {
            tma_load_4d(dst + j * 8192, &a.tm_xo, bars + C::R_FULL + slot, 64 * j, t.c0 + 64 * s, t.h, t.b);
            tma_load_4d(dst + (C::NB + j) * 8192, &a.tm_yo, bars + C::R_FULL + slot, 64 * j, t.c0 + 64 * s, t.h, t.b);
          }
        }
      }
    }
    __syncwarp();
  } else if (warp == C::W_MMA) {
    const bool leader = elect_one();
    constexpr uint32_t id_st = idesc_bf16(128, 64, false, false);
    constexpr uint32_t id_dx = idesc_bf16(128, D, false, true);
    const uint64_t dX = smem_desc_sw128(smem_u32(smem + C::OFF_X), 16, 1024);
    const uint64_t dY = smem_desc_sw128(smem_u32(smem + C::OFF_Y), 16, 1024);
    const uint64_t dR = smem_desc_sw128(smem_u32(smem + C::OFF_RING), 16, 1024);
    const uint64_t dRt = smem_desc_sw128(smem_u32(smem + C::OFF_RING), 8192, 1024);
    // Two cursors over the same stream of steps: `st` runs two steps ahead of `dx`.
    struct Cursor {
      int tile, s, n, ne;
    };
    auto seek = [&](Cursor& c) {   // to the first step of the next tile that has one
      while (c.tile < a.g.ntiles && (c.n = row_tile<SIDE, 64>(a.g, c.tile, false).n) == 0) c.tile += step;
      c.s = 0;
      ++c.ne;
    };
    auto next = [&](Cursor& c) {
      if (++c.s == c.n) {
        c.tile += step;
        seek(c);
      }
    };
    Cursor st{(int)blockIdx.x, 0, 0, -1};
    seek(st);
    Cursor dx = st;
    int gs = 0;
    auto issue_st = [&]() {
      if (st.tile >= a.g.ntiles) return;
      const int buf = gs & 1, xb = st.ne & 1, slot = gs % C::NS;
      if (st.s == 0) wait_inline(bars + C::XY_FULL + xb, (st.ne >> 1) & 1, a.status, 223);
      wait_inline(bars + C::R_FULL + slot, (gs / C::NS) & 1, a.status, 224);
      tc_fence_after_sync();
      if (leader) {
        const uint64_t x = dX + (uint64_t)(xb * (C::TB >> 4)), y = dY + (uint64_t)(xb * (C::TB >> 4));
        const uint64_t o = dR + (uint64_t)(slot * (C::SLOT >> 4));
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          mma_ss(tb + 128 * buf, x + kmajor(k, 16384), o + kmajor(k, 8192), id_st, k > 0);
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          mma_ss(tb + 128 * buf + 64, y + kmajor(k, 16384), o + (uint64_t)(C::NB * (8192 >> 4)) + kmajor(k, 8192), id_st,
                 k > 0);
        mma_commit(bars + C::ST_FULL + buf);
        if (st.s == st.n - 1) mma_commit(bars + C::XY_FREE + xb);
      }
      __syncwarp();
      ++gs;
      next(st);
    };
    issue_st();
    issue_st();
    for (int g = 0; dx.tile < a.g.ntiles; ++g, next(dx)) {
      const int buf = g & 1, db = dx.ne & 1, slot = g % C::NS;
      wait_inline(bars + C::DS_DONE + buf, (g >> 1) & 1, a.status, 225);
      if (dx.s == 0 && dx.ne >= 2) wait_inline(bars + C::DX_FREE + db, ((dx.ne >> 1) - 1) & 1, a.status, 226);
      tc_fence_after_sync();
      if (leader) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          mma_ts(tb + C::T_DX + D * db, tb + 128 * buf + packed(k),
                 dRt + (uint64_t)(slot * (C::SLOT >> 4) + k * 128), id_dx, dx.s > 0 || k > 0);
        mma_commit(bars + C::R_FREE + slot);
        if (dx.s == dx.n - 1) mma_commit(bars + C::DX_FULL + db);
      }
      __syncwarp();
      issue_st();
    }
  } else {
    // two groups of eight warps, one per buffer; a thread owns a row and 32 of the step's 64 columns
    const int grp = warp >> 3, qd = warp & 3, cq = (warp >> 2) & 1;
    const int row = qd * 32 + lane;
    const uint32_t lane_base = tb + ((uint32_t)(qd * 32) << 16);
    const float sc = a.tau * kLog2e;
    int g = 0, ne = 0;
    for (int tile = blockIdx.x; tile < a.g.ntiles; tile += step) {
      const RowTile t = row_tile<SIDE, 64>(a.g, tile, false);
      const int r = t.r0 + row;
      const float2* nd = a.nd + (int64_t)t.bh * a.Tp;
      float2 own = make_float2(0.f, 0.f);
      if (SIDE == QUERIES) own = __ldg(nd + r);
      for (int s = 0; s < t.n; ++s, ++g) {
        if ((g & 1) != grp) continue;
        const int c = t.c0 + 64 * s + 32 * cq;
        const uint32_t vis = seen<SIDE>(a.g, t, r, c, false);
        const uint32_t ts = lane_base + 128 * grp + 32 * cq;
        uint32_t o[16];
        mbar_wait(bars + C::ST_FULL + grp, (g >> 1) & 1, a.status, 227);
        tc_fence_after_sync();
        if (__any_sync(0xffffffffu, vis != 0u)) {
          uint32_t x[32], y[32];
          tmem_ld32(ts, x);
          tmem_ld32(ts + 64, y);
          tmem_ld_wait();
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            float4 n01 = make_float4(own.x, own.y, own.x, own.y), n23 = n01;
            if (SIDE == KEYS) {
              // c < Tp: the row arrays are padded to whole tiles
              n01 = __ldg(reinterpret_cast<const float4*>(nd + c) + 2 * q);
              n23 = __ldg(reinterpret_cast<const float4*>(nd + c) + 2 * q + 1);
            }
            const float nn[4] = {n01.x, n01.z, n23.x, n23.z}, dd[4] = {n01.y, n01.w, n23.y, n23.w};
            float v[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float p = ex2(fmaf(__uint_as_float(x[4 * q + j]), sc, -nn[j]));
              v[j] = keep_if_bit(p * (__uint_as_float(y[4 * q + j]) - dd[j]), vis, 4 * q + j);
            }
            o[2 * q] = pack_bf16(v[0], v[1]);
            o[2 * q + 1] = pack_bf16(v[2], v[3]);
          }
        } else {
#pragma unroll
          for (int j = 0; j < 16; ++j) o[j] = 0u;
        }
        tmem_st16(ts, o);
        tmem_st_wait();
        tc_fence_before_sync();
        warp_arrive(bars + C::DS_DONE + grp, lane);
      }
      // this thread's quarter of the row's D sums
      constexpr int NC = D / 4;
      const int c = NC * (2 * grp + cq);
      uint32_t v[32];
      if (t.n > 0) {
        const int db = ne & 1;
        mbar_wait(bars + C::DX_FULL + db, (ne >> 1) & 1, a.status, 228);
        tc_fence_after_sync();
        tmem_ld32(lane_base + C::T_DX + D * db + c, v);
        tmem_ld_wait();
        tc_fence_before_sync();
        warp_arrive(bars + C::DX_FREE + db, lane);
        ++ne;
      } else {
#pragma unroll
        for (int j = 0; j < NC; ++j) v[j] = 0u;
      }
      // part: per tile (D / 4 groups of four columns) x 128 rows, so that a warp writes whole lines
      float4* dst = reinterpret_cast<float4*>(a.part) + ((int64_t)tile * (D / 4) + c / 4) * TR + row;
#pragma unroll
      for (int j = 0; j < NC / 4; ++j)
        dst[j * TR] = make_float4(a.tau * __uint_as_float(v[4 * j]), a.tau * __uint_as_float(v[4 * j + 1]),
                                  a.tau * __uint_as_float(v[4 * j + 2]), a.tau * __uint_as_float(v[4 * j + 3]));
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == C::W_LOAD) {
    __syncwarp();
    tmem_dealloc(tb, 512);
  }
}

// ---------------------------------------------------------------------------
// dq or dk.  Head dim 64: both parts; head dim 128 (no tensor memory left for S): the low-rank part, and adds the
// exact part that the window kernel left.
struct GradArgs {
  CUtensorMap tm_x, tm_y, tm_xo, tm_yo, tm_fo, tm_sum, tm_sum_lo, tm_hi, tm_lo, tm_dx;
  Geom g;
  const float2* nd;                        // (BH, Tp)
  const float* delta;                      // (BH, Tp): the second of nd
  const float* off;                        // (BH, rows padded): exponent offsets of the own features
  const float* sum1;                       // (BH, m): extra column of the other side's summary
  const float* part;                       // head dim 128: (tiles, D / 4, 128 rows) float4
  int* status;
  int Tp, whole;
  float tau;
};

// A unit is a (tile, pass of 256 features); head dim 128 takes two passes.  The steps of all units form one stream,
// gg = 0, 1, ..
//
// Tensor memory: df 256 | dx D | G 64 | (head dim 64) S 64 | packed operands 64.  A step's G and S are read at once,
// which frees both for the next step; what is made of them, g and p g, goes to the packed columns (head dim 64: 32 of
// g and 32 of p g of one step; 128: g of two steps).  After the last step U of the own features takes 128 columns from
// G on.  Every compute warp loads its U before it waits for df, so that the next tile's first G and S form meanwhile;
// the group whose turn it is packs that step before it finishes the tile.
//
// Bound: two chains beside the stream into shared memory.  A step's (G and S -> read -> packed -> df, dx) takes 1.4 k
// cycles, because there is no room for a second G and S beside df; a tile's (last step -> df -> du -> dx -> stored)
// 5 k.  With six steps 18 to 20 k cycles a tile at head dim 64 and w = 256, of which products take 8.7 k.  A step's 64
// columns are 32 KB of features and 16 KB of X' and Y'; with the summary and the own rows 368 KB per tile, 8.8 k
// cycles at the 41.7 B/clk that one SM's TMA loads sustain.
template <int D>
struct GradCfg {
  static constexpr bool FUSE = D == 64;
  static constexpr int NB = D / 64, M = 4 * D, PASS = M / 256, XBUF = FUSE ? 2 : 1, NF = 2, NC = FUSE ? 3 : 2;
  static constexpr uint32_t TB = NB * 16384;             // own tile of X or Y
  static constexpr uint32_t AUX = 512 * D;               // 256 features x D of the summary; 2 terms x 128 x D of Wt
  static constexpr uint32_t CSLOT = 16384;               // Y' of a step, and X' (head dim 64)
  static constexpr uint32_t OFF_X = 0, OFF_Y = XBUF * TB, OFF_SUM = OFF_Y + TB;
  static constexpr uint32_t OFF_W = FUSE ? OFF_SUM + AUX : OFF_SUM;   // head dim 128: one buffer for both, in turn
  static constexpr uint32_t OFF_F = OFF_W + AUX, OFF_C = OFF_F + NF * 32768;
  // per step, 64 columns of (n2, delta); head dim 128: of delta, in four slots, because there a column tile is freed
  // when G has been formed, with G itself still to be read (the load of step g + 4 is behind the products of step g)
  static constexpr int NND = FUSE ? NC : 4;
  static constexpr uint32_t NDB = FUSE ? 512 : 256;
  static constexpr uint32_t OFF_ND = OFF_C + NC * CSLOT, OFF_S1 = OFF_ND + NND * NDB;   // then sum1 of the unit
  static constexpr uint32_t OFF_BAR = OFF_S1 + 1024, SMEM = OFF_BAR + 320;   // (the base is 1024-byte aligned)
  static constexpr int NCOMP = 512, NTHR = NCOMP + 128, W_LOAD = 16, W_STORE = 17, W_MMA_A = 18, W_MMA_B = 19;
  static constexpr uint32_t T_DF = 0, T_DX = 256, T_G = FUSE ? 320 : 384, T_S = T_G + 64, T_P = 448;
  enum { X_FULL = 0, X_FREE = 2, Y_FULL = 4, Y_FREE, SUM_FULL, SUM_FREE, W_FULL, W_FREE, F_FULL, F_FREE = F_FULL + NF,
         C_FULL = F_FREE + NF, C_FREE = C_FULL + NC, T_FULL = C_FREE + NC, P_FREE = T_FULL + 2, T_READ = P_FREE + 2,
         G_DONE = T_READ + 2, U_FULL = G_DONE + 2, U_READ, DF_FULL, DU_DONE, DX_FULL, DX_FREE, H_READ, STAGED, ND_FULL,
         COUNT = ND_FULL + (FUSE ? 0 : NND) };
  static_assert(SMEM <= 232448 && COUNT * 8 + 4 <= 320, "shared memory of one CTA");
};

template <int SIDE, int D>
__global__ void __launch_bounds__(640, 1) bwd_grad_kernel(const __grid_constant__ GradArgs a) {
  using C = GradCfg<D>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + C::COUNT);
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  if (tid == 0) {
    for (int i = 0; i < C::COUNT; ++i) {
      const bool group = i >= C::T_READ && i < C::U_FULL;
      const bool all = i == C::U_READ || i == C::DU_DONE || i == C::DX_FREE || i == C::H_READ || i == C::STAGED;
      const bool both = i == C::Y_FREE;                      // one commit of either issuing warp
      mbar_init(bars + i, group ? 8 : all ? 16 : both ? 2 : 1);
    }
    fence_mbar_init();
  }
  if (warp == C::W_LOAD) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  constexpr uint32_t tb = 0;
  if (tid == 0 && (*tmem_slot != 0 || (smem_u32(smem) & 1023) != 0)) atomicCAS(a.status, 0, 241);
  const int step = gridDim.x;
  const bool whole = a.whole != 0;
  const int n_it = (a.g.ntiles - (int)blockIdx.x + step - 1) / step, n_u = n_it * C::PASS;

  if (warp == C::W_LOAD) {
    const bool leader = elect_one();
    int nf = 0, nc = 0, ns = 0;     // loads so far: features, column tiles, summary terms
    for (int u = 0; u < n_u; ++u) {
      const int it = u / C::PASS, pass = u % C::PASS;
      const RowTile t = row_tile<SIDE, 64>(a.g, blockIdx.x + it * step, whole);
      auto load_x = [&]() {
        const int buf = it % C::XBUF;
        if (it >= C::XBUF) wait_inline(bars + C::X_FREE + buf, ((it / C::XBUF) - 1) & 1, a.status, 261);
        if (leader) {
          mbar_expect_tx(bars + C::X_FULL + buf, C::TB);
          for (int j = 0; j < C::NB; ++j)
            tma_load_4d(smem + C::OFF_X + buf * C::TB + j * 16384, &a.tm_x, bars + C::X_FULL + buf, 64 * j, t.r0, t.h, t.b);
        }
      };
      auto load_c = [&](int s) {
        const int slot = nc % C::NC;
        if (nc >= C::NC) wait_inline(bars + C::C_FREE + slot, ((nc / C::NC) - 1) & 1, a.status, 262);
        ++nc;
        if (leader) {
          uint8_t* dst = smem + C::OFF_C + slot * C::CSLOT;
          mbar_expect_tx(bars + C::C_FULL + slot, C::CSLOT + (SIDE == KEYS && C::FUSE ? C::NDB : 0));
          if (SIDE == KEYS) {
            const int d = (nc - 1) % C::NND;
            uint64_t* bar = bars + (C::FUSE ? C::C_FULL + slot : C::ND_FULL + d);
            if (!C::FUSE) mbar_expect_tx(bar, C::NDB);
            // c0 + 64 s + 63 < Tp: the row arrays are padded to whole tiles
            const int64_t at = (int64_t)t.bh * a.Tp + t.c0 + 64 * s;
            bulk_load(smem + C::OFF_ND + d * C::NDB,
                      C::FUSE ? static_cast<const void*>(a.nd + at) : static_cast<const void*>(a.delta + at), C::NDB, bar);
          }
          for (int j = 0; j < C::NB; ++j)
            tma_load_4d(dst + j * 8192, &a.tm_yo, bars + C::C_FULL + slot, 64 * j, t.c0 + 64 * s, t.h, t.b);
          if (C::FUSE) tma_load_4d(dst + 8192, &a.tm_xo, bars + C::C_FULL + slot, 0, t.c0 + 64 * s, t.h, t.b);
        }
      };
      auto load_f = [&](int s) {
        const int slot = nf % C::NF;
        if (nf >= C::NF) wait_inline(bars + C::F_FREE + slot, ((nf / C::NF) - 1) & 1, a.status, 263);
        ++nf;
        if (leader) {
          uint8_t* dst = smem + C::OFF_F + slot * 32768;
          mbar_expect_tx(bars + C::F_FULL + slot, 32768);
          for (int j = 0; j < 4; ++j)
            tma_load_3d(dst + j * 8192, &a.tm_fo, bars + C::F_FULL + slot, 256 * pass + 64 * j, t.c0 + 64 * s, t.bh);
        }
      };
      // Head dim 64: the summary's terms take turns in a buffer of their own and Wt stays.  Head dim 128: they and
      // Wt of the unit take turns in one (term, its product, term, its product, Wt, its products, next unit).
      auto load_sum = [&](int term) {
        if (term == 0 && !C::FUSE) {
          if (u >= 1) wait_inline(bars + C::W_FREE, (u - 1) & 1, a.status, 264);
        } else if (ns >= 1) {
          wait_inline(bars + C::SUM_FREE, (ns - 1) & 1, a.status, 265);
        }
        ++ns;
        if (leader) {
          mbar_expect_tx(bars + C::SUM_FULL, C::AUX);
          for (int j = 0; j < C::NB; ++j)
            for (int f = 0; f < 2; ++f)
              tma_load_3d(smem + C::OFF_SUM + j * 32768 + f * 16384, term ? &a.tm_sum_lo : &a.tm_sum, bars + C::SUM_FULL,
                          64 * j, 256 * pass + 128 * f, t.bh);
        }
      };
      auto load_w = [&]() {
        if (C::FUSE && u > 0) return;
        if (!C::FUSE) {
          if (!whole) wait_inline(bars + C::SUM_FREE, (ns - 1) & 1, a.status, 266);
          else if (u >= 1) wait_inline(bars + C::W_FREE, (u - 1) & 1, a.status, 267);
        }
        if (leader) {
          mbar_expect_tx(bars + C::W_FULL, C::AUX);
          for (int j = 0; j < C::NB; ++j) {
            tma_load_2d(smem + C::OFF_W + j * 16384, &a.tm_hi, bars + C::W_FULL, 64 * j, 128 * pass);
            tma_load_2d(smem + C::OFF_W + C::AUX / 2 + j * 16384, &a.tm_lo, bars + C::W_FULL, 64 * j, 128 * pass);
          }
        }
      };
      if (pass == 0) {
        if (it >= 1) wait_inline(bars + C::Y_FREE, (it - 1) & 1, a.status, 268);
        if (leader) {
          mbar_expect_tx(bars + C::Y_FULL, C::TB);
          for (int j = 0; j < C::NB; ++j)
            tma_load_4d(smem + C::OFF_Y + j * 16384, &a.tm_y, bars + C::Y_FULL, 64 * j, t.r0, t.h, t.b);
        }
        if (C::FUSE) load_x();
      }
      // Column tiles run one step ahead of the features; the summary's terms behind steps 0 and 1, Wt behind step 2.
      // (Each load has one place in the code: see `wait_inline` on its size.)
      int sums = whole ? 2 : 0;
      bool w = false;
#pragma unroll 1
      for (int s = -1; s < t.n || !w; ++s) {
        if (s + 1 < t.n) load_c(s + 1);
        if (s >= 0 && s < t.n) load_f(s);
        if (s >= 0 && sums < 2) load_sum(sums++);
        if (!w && (s == 2 || (s >= t.n - 1 && sums == 2))) {
          load_w();
          w = true;
        }
      }
      if (!C::FUSE && pass == 0) load_x();
    }
    __syncwarp();
  } else if (warp == C::W_MMA_A) {
    // ---- issuer A: G, S, U.  (Two issuing warps: each spends as long on waits and descriptors as on its products.)
    const bool leader = elect_one();
    constexpr uint32_t id_t = idesc_bf16(128, 64, false, false);
    constexpr uint32_t id_u = idesc_bf16(128, 128, false, false);
    const uint64_t dX = smem_desc_sw128(smem_u32(smem + C::OFF_X), 16, 1024);
    const uint64_t dY = smem_desc_sw128(smem_u32(smem + C::OFF_Y), 16, 1024);
    const uint64_t dC = smem_desc_sw128(smem_u32(smem + C::OFF_C), 16, 1024);
    const uint64_t dW = smem_desc_sw128(smem_u32(smem + C::OFF_W), 16, 1024);
    int gg = 0;                     // number of the step in the CTA's stream
    for (int u = 0; u < n_u; ++u) {
      const int it = u / C::PASS, pass = u % C::PASS, xb = it % C::XBUF;
      const int n = row_tile<SIDE, 64>(a.g, blockIdx.x + it * step, whole).n;
      const uint64_t x = dX + (uint64_t)(xb * (C::TB >> 4));
      if (pass == 0) wait_inline(bars + C::Y_FULL, it & 1, a.status, 274);
      if (C::FUSE) wait_inline(bars + C::X_FULL + xb, (it / C::XBUF) & 1, a.status, 275);
      for (int s = 0; s < n; ++s, ++gg) {
        const int slot = gg % C::NC;
        wait_inline(bars + C::C_FULL + slot, (gg / C::NC) & 1, a.status, 271);
        // the step before has been read, or U of the unit before
        if (s > 0) wait_inline(bars + C::T_READ + ((gg - 1) & 1), ((gg - 1) >> 1) & 1, a.status, 276);
        else if (u > 0) wait_inline(bars + C::U_READ, (u - 1) & 1, a.status, 273);
        // (head dim 128: seen for every step, because U waits for the last two and phases are told apart by parity)
        if (!C::FUSE && gg >= 2) wait_inline(bars + C::P_FREE + (gg & 1), ((gg >> 1) - 1) & 1, a.status, 275);
        tc_fence_after_sync();
        if (leader) {
          const uint64_t o = dC + (uint64_t)(slot * (C::CSLOT >> 4));
#pragma unroll
          for (int k = 0; k < D / 16; ++k) mma_ss(tb + C::T_G, dY + kmajor(k, 16384), o + kmajor(k, 8192), id_t, k > 0);
          if (C::FUSE) {
#pragma unroll
            for (int k = 0; k < D / 16; ++k)
              mma_ss(tb + C::T_S, x + kmajor(k, 16384), o + 512 + kmajor(k, 8192), id_t, k > 0);
          }
          mma_commit(bars + C::T_FULL + (gg & 1));
          if (!C::FUSE) mma_commit(bars + C::C_FREE + slot);
        }
        __syncwarp();
      }
      // U of the own features, from the columns of G on: the last step has been read (without steps: U of the unit
      // before); head dim 128: and the products that read the packed columns are done
      if (n > 0) wait_inline(bars + C::T_READ + ((gg - 1) & 1), ((gg - 1) >> 1) & 1, a.status, 277);
      else if (u > 0) wait_inline(bars + C::U_READ, (u - 1) & 1, a.status, 278);
      if (!C::FUSE)
        for (int g = gg - 2 > 0 ? gg - 2 : 0; g < gg; ++g)
          wait_inline(bars + C::P_FREE + (g & 1), (g >> 1) & 1, a.status, 272);
      wait_inline(bars + C::W_FULL, C::FUSE ? 0 : u & 1, a.status, 279);
      if (!C::FUSE && pass == 0) wait_inline(bars + C::X_FULL + xb, (it / C::XBUF) & 1, a.status, 280);
      tc_fence_after_sync();
      if (leader) {
        if (pass == C::PASS - 1) mma_commit(bars + C::Y_FREE);
#pragma unroll 1
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int k = 0; k < D / 16; ++k)
            mma_ss(tb + C::T_G, x + kmajor(k, 16384), dW + (uint64_t)(t * (C::AUX >> 5)) + kmajor(k, 16384), id_u,
                   t > 0 || k > 0);
        mma_commit(bars + C::U_FULL);
      }
      __syncwarp();
    }
  } else if (warp == C::W_MMA_B) {
    // ---- issuer B: df, dx
    const bool leader = elect_one();
    // The packed operands hold delta - y.y' and p times that.  Bit 13 negates A: df takes -g inside the window, g
    // outside it (`whole`), dx takes p g.
    const uint32_t id_df = idesc_bf16(128, 256, false, true) | (whole ? 1u << 13 : 0u);
    constexpr uint32_t id_sum = idesc_bf16(128, 256, false, false);
    constexpr uint32_t id_dx = idesc_bf16(128, D, false, true);
    const uint64_t dY = smem_desc_sw128(smem_u32(smem + C::OFF_Y), 16, 1024);
    const uint64_t dCt = smem_desc_sw128(smem_u32(smem + C::OFF_C + 8192), 8192, 1024);   // X', MN-major
    const uint64_t dF = smem_desc_sw128(smem_u32(smem + C::OFF_F), 8192, 1024);
    const uint64_t dSum = smem_desc_sw128(smem_u32(smem + C::OFF_SUM), 16, 1024);
    const uint64_t dWt = smem_desc_sw128(smem_u32(smem + C::OFF_W), 16384, 1024);
    int g0 = 0, ns = 0;             // number of the unit's first step; summary terms so far
    for (int u = 0; u < n_u; ++u) {
      const int it = u / C::PASS, pass = u % C::PASS;
      const int n = row_tile<SIDE, 64>(a.g, blockIdx.x + it * step, whole).n;
      bool fresh = true;            // df of this unit has not been written to
      int sums = whole ? 2 : 0;
      auto issue_sum = [&]() {      // df += Y summary^T, one term
        if (pass == 0 && sums == 0) wait_inline(bars + C::Y_FULL, it & 1, a.status, 291);
        wait_inline(bars + C::SUM_FULL, ns & 1, a.status, 292);
        ++ns;
        tc_fence_after_sync();
        if (leader) {
#pragma unroll
          for (int k = 0; k < D / 16; ++k)
            mma_ss(tb + C::T_DF, dY + kmajor(k, 16384), dSum + kmajor(k, 32768), id_sum, !fresh || k > 0);
          mma_commit(bars + C::SUM_FREE);
        }
        __syncwarp();
        fresh = false;
        ++sums;
      };
      // what lies in df of the previous tile: the operands of dx are through, the sums beside them have been read
      if (pass == 0 && it >= 1) {
        wait_inline(bars + C::DX_FULL, (it - 1) & 1, a.status, 293);
        wait_inline(bars + C::H_READ, (it - 1) & 1, a.status, 299);
      }
      // The previous tile's dx has been read.  df of the first step and a term of the summary are issued before this is
      // waited for: the tensor core has them while the group that packed the step finishes the previous tile.
      bool dx_seen = pass > 0 || it == 0;
      auto dx_ready = [&]() {
        if (!dx_seen) wait_inline(bars + C::DX_FREE, (it - 1) & 1, a.status, 298);
        dx_seen = true;
      };
#pragma unroll 1
      for (int s = 0; s < n || sums < 2; ++s) {
        const int gg = g0 + s, slot = gg % C::NF;
        if (s < n) {
          wait_inline(bars + C::F_FULL + slot, (gg / C::NF) & 1, a.status, 294);
          wait_inline(bars + C::G_DONE + (gg & 1), (gg >> 1) & 1, a.status, 278);
          tc_fence_after_sync();
          if (leader) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              mma_ts(tb + C::T_DF, tb + C::T_P + (C::FUSE ? 0 : 32 * (gg & 1)) + 8 * k, dF + (uint64_t)(slot * 2048 + k * 128),
                     id_df, !fresh || k > 0);
            mma_commit(bars + C::F_FREE + slot);
            if (!C::FUSE) mma_commit(bars + C::P_FREE + (gg & 1));
          }
          __syncwarp();
          fresh = false;
        }
        if (sums < 2) issue_sum();
        if (C::FUSE && s < n) {
          if (s == 0) {
            dx_ready();
            tc_fence_after_sync();
          }
          if (leader) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              mma_ts(tb + C::T_DX, tb + C::T_P + 32 + 8 * k, dCt + (uint64_t)((gg % C::NC) * (C::CSLOT >> 4) + k * 128),
                     id_dx | (1u << 13), s > 0 || k > 0);
            mma_commit(bars + C::C_FREE + gg % C::NC);
            mma_commit(bars + C::P_FREE + (gg & 1));
          }
          __syncwarp();
        }
      }
      g0 += n;
      if (leader) {
        if (pass == C::PASS - 1) mma_commit(bars + C::Y_FREE);
        mma_commit(bars + C::DF_FULL);
      }
      __syncwarp();
      wait_inline(bars + C::W_FULL, C::FUSE ? 0 : u & 1, a.status, 295);
      wait_inline(bars + C::DU_DONE, u & 1, a.status, 281);
      const bool first = pass == 0 && !(C::FUSE && n > 0);   // nothing of this tile is in dx yet
      dx_ready();
      tc_fence_after_sync();
      if (leader) {
        // du Wt: high x high, high x low, low x high; du's low term lies behind its high one
#pragma unroll 1
        for (int t = 0; t < 3; ++t)
#pragma unroll
          for (int k = 0; k < 8; ++k)
            mma_ts(tb + C::T_DX, tb + C::T_DF + 128 * (k >> 2) + packed(k & 3) + (t == 2 ? 16 : 0),
                   dWt + (uint64_t)((t == 1 ? (C::AUX >> 5) : 0) + k * 128), id_dx, !first || t > 0 || k > 0);
        mma_commit(bars + C::W_FREE);
        if (pass == C::PASS - 1) mma_commit(bars + C::DX_FULL);
      }
      __syncwarp();
    }
  } else if (warp == C::W_STORE) {
    // the staged dx (over the X rows) -> memory; rows past the end are clipped by the tensor map
    const bool leader = elect_one();
    for (int it = 0; it < n_it; ++it) {
      const RowTile t = row_tile<SIDE, 64>(a.g, blockIdx.x + it * step, whole);
      const int buf = it % C::XBUF;
      wait_inline(bars + C::STAGED, it & 1, a.status, 283);
      if (leader) {
        for (int j = 0; j < C::NB; ++j)
          tma_store_4d(&a.tm_dx, smem + C::OFF_X + buf * C::TB + j * 16384, 64 * j, t.r0, t.h, t.b);
        tma_store_commit();
        tma_store_wait_read0();
        mbar_arrive(bars + C::X_FREE + buf);
      }
      __syncwarp();
    }
    if (leader) tma_store_wait_all();
    __syncwarp();
  } else {
    // Two groups of eight warps take the steps in turn; a thread owns a row and 32 of a step's 64 columns.  For du the
    // groups take a block of 128 features each, for dx every thread a quarter of the row.
    const int grp = warp >> 3, qd = warp & 3, cq = (warp >> 2) & 1;
    const int row = qd * 32 + lane;
    const uint32_t lane_base = tb + ((uint32_t)(qd * 32) << 16);
    float* s_s1 = reinterpret_cast<float*>(smem + C::OFF_S1);
    const float sc = a.tau * kLog2e;
    const float lt = log2f(a.tau);
    // a tile, and what a thread needs of its row
    RowTile t = row_tile<SIDE, 64>(a.g, blockIdx.x, whole);
    float off, rn = 0.f, rd = 0.f;
    auto fetch_row = [&]() {
      const int r = t.r0 + row;     // (the row arrays are padded to whole tiles)
      off = __ldg(a.off + (int64_t)t.bh * a.g.ntr * TR + r);
      if (SIDE == QUERIES) {
        const float2 v = __ldg(a.nd + (int64_t)t.bh * a.Tp + r);   // (r < Tp)
        rn = lt - v.x;              // tau p = 2^(S sc + (log2 tau - n2))
        rd = v.y;
      }
    };
    // Step s of tile t, number gg of the stream: G, S -> delta - y.y' and p times that, packed.
    auto pack_step = [&](int s, int gg) {
      const int c = t.c0 + 64 * s + 32 * cq, r = t.r0 + row;
      const uint32_t in = seen<SIDE>(a.g, t, r, c, false);
      const uint32_t out = whole ? seen<SIDE>(a.g, t, r, c, true) : 0u;
      mbar_wait(bars + C::T_FULL + grp, (gg >> 1) & 1, a.status, 286);
      tc_fence_after_sync();
      uint32_t x[32], y[32];
      tmem_ld32(lane_base + C::T_G + 32 * cq, y);
      if (C::FUSE) tmem_ld32(lane_base + C::T_S + 32 * cq, x);
      const float4* nd = reinterpret_cast<const float4*>(smem + C::OFF_ND + (gg % C::NND) * C::NDB + cq * (C::NDB / 2));
      // head dim 64: landed with the step's tile, which is held until its products are done
      if (SIDE == KEYS && C::FUSE) mbar_wait(bars + C::C_FULL + gg % C::NC, (gg / C::NC) & 1, a.status, 285);
      if (SIDE == KEYS && !C::FUSE) mbar_wait(bars + C::ND_FULL + (gg & 3), (gg >> 2) & 1, a.status, 283);
      tmem_ld_wait();
      tc_fence_before_sync();
      warp_arrive(bars + C::T_READ + grp, lane);
      uint32_t o[16], e[16];
#pragma unroll
      for (int q = 0; q < 16; ++q) {
        float2 dd = make_float2(rd, rd), nn = make_float2(rn, rn);
        if (SIDE == KEYS && C::FUSE) {
          const float4 v = nd[q];
          dd = make_float2(v.y, v.w);
          nn = make_float2(lt - v.x, lt - v.z);
        } else if (SIDE == KEYS) {
          dd = reinterpret_cast<const float2*>(nd)[q];
        }
        const float2 d = fma2(make_float2(__uint_as_float(y[2 * q]), __uint_as_float(y[2 * q + 1])), make_float2(-1.f, -1.f), dd);
        float2 g = make_float2(keep_if_bit(d.x, in, 2 * q), keep_if_bit(d.y, in, 2 * q + 1));
        if (C::FUSE) {
          // (hidden columns: a weight that is finite, times zero)
          const float2 arg = fma2(make_float2(__uint_as_float(x[2 * q]), __uint_as_float(x[2 * q + 1])), make_float2(sc, sc), nn);
          const float2 w = mul2(make_float2(ex2(fminf(arg.x, 126.f)), ex2(fminf(arg.y, 126.f))), g);
          e[q] = pack_bf16(w.x, w.y);
        }
        if (whole) g = make_float2(keep_if_bit(d.x, out, 2 * q), keep_if_bit(d.y, out, 2 * q + 1));
        o[q] = pack_bf16(g.x, g.y);
      }
      // the products that read the packed columns before
      if (C::FUSE) {
        if (gg >= 1) mbar_wait(bars + C::P_FREE + (grp ^ 1), ((gg - 1) >> 1) & 1, a.status, 284);
        tmem_st16(lane_base + C::T_P + 16 * cq, o);
        tmem_st16(lane_base + C::T_P + 32 + 16 * cq, e);
      } else {
        if (gg >= 2) mbar_wait(bars + C::P_FREE + grp, ((gg >> 1) - 1) & 1, a.status, 284);
        tmem_st16(lane_base + C::T_P + 32 * grp + 16 * cq, o);
      }
      tmem_st_wait();
      tc_fence_before_sync();
      warp_arrive(bars + C::G_DONE + grp, lane);
    };
    fetch_row();
    int gg = 0;                     // number of the unit's first step
    float hs = 0.f, hsum = 0.f;
    // One unit more than there are: the last tile's dx.
#pragma unroll 1
    for (int u = 0; u <= n_u; ++u) {
      const int it = u / C::PASS, pass = u % C::PASS;
      const int n = u < n_u ? t.n : 0;
      float sum1 = 0.f;
      if (tid < 256 && u < n_u) sum1 = __ldg(a.sum1 + (int64_t)t.bh * C::M + 256 * pass + tid);
      const bool none = whole && n == 0;
      const bool last = pass == C::PASS - 1;
      // This group's steps, and the previous tile's dx: behind step 0 in the group that packs it (its G and S are there
      // as soon as U has been read), in front of the steps in the other.  One place in the code for each.
      bool pend = pass == 0 && it > 0;
      int s = (gg ^ grp) & 1;
#pragma unroll 1
      while (pend || s < n) {
        if (s < n && (!pend || s == 0)) {
          pack_step(s, gg + s);
          s += 2;
          continue;
        }
        pend = false;
        const int pi = it - 1;
        constexpr int NQ = D / 4;
        const int c = NQ * (2 * grp + cq), buf = pi % C::XBUF;
        uint8_t* xs = smem + C::OFF_X + buf * C::TB + (c >> 6) * 16384 + row * 128;
        float4 e[C::FUSE ? 1 : NQ / 4];
        if (!C::FUSE) {
          const float4* part = reinterpret_cast<const float4*>(a.part) + ((int64_t)(blockIdx.x + pi * step) * (D / 4) + c / 4) * TR + row;
#pragma unroll
          for (int j = 0; j < NQ / 4; ++j) e[j] = __ldg(part + j * TR);
        }
        mbar_wait(bars + C::X_FULL + buf, (pi / C::XBUF) & 1, a.status, 288);
        mbar_wait(bars + C::DX_FULL, pi & 1, a.status, 289);
        tc_fence_after_sync();
        uint32_t v[NQ / 16][16];
#pragma unroll
        for (int q = 0; q < NQ / 16; ++q) tmem_ld16(lane_base + C::T_DX + c + 16 * q, v[q]);
        tmem_ld_wait();
        tc_fence_before_sync();
        warp_arrive(bars + C::DX_FREE, lane);
#pragma unroll
        for (int j = 0; j < NQ / 8; ++j) {
          // eight entries: 16 bytes of the row's swizzled line, dx over x
          uint4* at = reinterpret_cast<uint4*>(xs + ((((c & 63) >> 3) + j) ^ (row & 7)) * 16);
          const uint4 xv = *at;
          const uint32_t xw[4] = {xv.x, xv.y, xv.z, xv.w};
          float z[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) z[k] = __uint_as_float(v[j >> 1][8 * (j & 1) + k]);
          if (!C::FUSE) {
            const float4 e0 = e[2 * j], e1 = e[2 * j + 1];
            z[0] += e0.x; z[1] += e0.y; z[2] += e0.z; z[3] += e0.w;
            z[4] += e1.x; z[5] += e1.y; z[6] += e1.z; z[7] += e1.w;
          }
          uint32_t w[4];
#pragma unroll
          for (int k = 0; k < 4; ++k)
            w[k] = pack_bf16(fmaf(-hsum, bf16_lo(xw[k]), z[2 * k]), fmaf(-hsum, bf16_hi(xw[k]), z[2 * k + 1]));
          *at = make_uint4(w[0], w[1], w[2], w[3]);
        }
        fence_async_smem();
        warp_arrive(bars + C::STAGED, lane);
      }
      if (u == n_u) break;
      gg += n;
      if (tid < 256) {
        // (every reader of the unit before is through; head dim 64: a tile has one unit, and its dx was waited for)
        if (!C::FUSE && u >= 1) mbar_wait(bars + C::DU_DONE, (u - 1) & 1, a.status, 283);
        s_s1[tid] = sum1;
      }
      if (pass == 0) hs = 0.f;
      asm volatile("bar.sync 1, 512;" ::: "memory");
      // df -> du of this thread's 32 projections: du = f+ df+ - f- df-, in two bf16 terms
      const float nd1 = whole ? 0.f : (SIDE == QUERIES ? -rd : -1.f);
      const float o1 = off;
      const float* s1 = s_s1 + 128 * grp + 32 * cq;
      const uint32_t td = lane_base + C::T_DF + 128 * grp + 32 * cq;
      mbar_wait(bars + C::U_FULL, u & 1, a.status, 290);
      tc_fence_after_sync();
      uint32_t uu[32];
      tmem_ld32(lane_base + C::T_G + 64 * grp + 32 * cq, uu);
      tmem_ld_wait();
      tc_fence_before_sync();
      warp_arrive(bars + C::U_READ, lane);
      // the next tile's row, on its way while df is waited for
      if (last && it + 1 < n_it) {
        t = row_tile<SIDE, 64>(a.g, blockIdx.x + (it + 1) * step, whole);
        fetch_row();
      }
      mbar_wait(bars + C::DF_FULL, u & 1, a.status, 287);
      tc_fence_after_sync();
      float2 hs2 = make_float2(0.f, 0.f);
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        uint32_t p[16], m[16], hi[8], lo[8];
        tmem_ld16(td + 16 * hf, p);
        tmem_ld16(td + 64 + 16 * hf, m);
        tmem_ld_wait();
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          const float2 sp = *reinterpret_cast<const float2*>(s1 + 16 * hf + 2 * q);
          const float2 sm = *reinterpret_cast<const float2*>(s1 + 64 + 16 * hf + 2 * q);
          const float2 uv = make_float2(__uint_as_float(uu[16 * hf + 2 * q]), __uint_as_float(uu[16 * hf + 2 * q + 1]));
          float2 dp = make_float2(__uint_as_float(p[2 * q]), __uint_as_float(p[2 * q + 1]));
          float2 dm = make_float2(__uint_as_float(m[2 * q]), __uint_as_float(m[2 * q + 1]));
          if (none) dp = dm = make_float2(0.f, 0.f);
          dp = fma2(make_float2(nd1, nd1), sp, dp);
          dm = fma2(make_float2(nd1, nd1), sm, dm);
          const float2 ap = fma2(uv, make_float2(kLog2e, kLog2e), make_float2(o1, o1));
          const float2 am = fma2(uv, make_float2(-kLog2e, -kLog2e), make_float2(o1, o1));
          const float2 hp = mul2(make_float2(ex2(ap.x), ex2(ap.y)), dp);
          const float2 hm = mul2(make_float2(ex2(am.x), ex2(am.y)), dm);
          hs2 = add2(hs2, add2(hp, hm));
          const float2 d = fma2(hm, make_float2(-1.f, -1.f), hp);
          const uint32_t h2 = pack_bf16(d.x, d.y);
          const float2 l = fma2(make_float2(bf16_lo(h2), bf16_hi(h2)), make_float2(-1.f, -1.f), d);
          hi[q] = h2;
          lo[q] = pack_bf16(l.x, l.y);
        }
        // high terms over the thread's first 16 "+" columns, low ones over the next 16: of the second half these are
        // read before the first half's are written
        if (hf == 0) {
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            uu[q] = hi[q];
            uu[8 + q] = lo[q];
          }
        } else {
          uint32_t h0[8], l0[8];
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            h0[q] = uu[q];
            l0[q] = uu[8 + q];
          }
          tmem_st8(td, h0);
          tmem_st8(td + 8, hi);
          tmem_st8(td + 16, l0);
          tmem_st8(td + 24, lo);
        }
      }
      hs += hs2.x + hs2.y;
      if (last) tmem_st1(td + 64, __float_as_uint(hs));   // ... and the sum over the first of its "-" columns
      tmem_st_wait();
      tc_fence_before_sync();
      warp_arrive(bars + C::DU_DONE, lane);
      if (!last) continue;
      mbar_wait(bars + C::DU_DONE, u & 1, a.status, 300);
      tc_fence_after_sync();
      const uint32_t h0 = tmem_ld1(lane_base + C::T_DF + 64), h1 = tmem_ld1(lane_base + C::T_DF + 96);
      const uint32_t h2 = tmem_ld1(lane_base + C::T_DF + 192), h3 = tmem_ld1(lane_base + C::T_DF + 224);
      tmem_ld_wait();
      tc_fence_before_sync();
      warp_arrive(bars + C::H_READ, lane);
      hsum = a.tau * ((__uint_as_float(h0) + __uint_as_float(h1)) + (__uint_as_float(h2) + __uint_as_float(h3)));
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == C::W_LOAD) {
    __syncwarp();
    tmem_dealloc(tb, 512);
  }
}

// ---------------------------------------------------------------------------
// dv (the walk, the loading and the issuing lane: sbl_bwd_walk.cuh).
template <int D>
__global__ void __launch_bounds__(576, 1) bwd_value_kernel(const __grid_constant__ ValArgs a) {
  using C = ValCfg<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align1024(smem_raw);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + C::COUNT);
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  if (tid == 0) {
    for (int i = 0; i < C::COUNT; ++i)
      mbar_init(bars + i, (i >= C::E_DONE && i < C::P_FULL) || (i >= C::D_DONE && i < C::DV_FULL) || i == C::DV_FREE ? 8 : 1);
    fence_mbar_init();
  }
  if (warp == C::W_LOAD) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  constexpr uint32_t tb = 0;
  if (tid == 0 && *tmem_slot != 0) atomicCAS(a.status, 0, 241);
  const int step = gridDim.x;

  if (warp == C::W_LOAD) {
    if (elect_one()) {
      ValLoader<D> v{a, smem, bars};
      walk_values(a.g, v);
    }
    __syncwarp();
  } else if (warp == C::W_MMA) {
    if (elect_one()) {
      ValIssuer<D> v{a, bars, smem_desc_sw128(smem_u32(smem + C::OFF_K), 16, 1024),
                     smem_desc_sw128(smem_u32(smem + C::OFF_F), 16, 1024),
                     smem_desc_sw128(smem_u32(smem + C::OFF_RING), 16, 1024),
                     smem_desc_sw128(smem_u32(smem + C::OFF_RING), 16384, 1024)};
      walk_values(a.g, v);
    }
    __syncwarp();
  } else {
    // exponential group (warps 0-7): S -> p in place; packing group (warps 8-15): p - a -> bf16, epilogue.
    // A thread owns a row and 64 columns, in two chunks of 32.
    const bool exp_group = warp < 8;
    const int qd = warp & 3, cq = (warp >> 2) & 1;
    const int row = qd * 32 + lane;
    const uint32_t lane_base = tb + ((uint32_t)(qd * 32) << 16);
    const float sc = a.tau * kLog2e;
    int g = 0, it = 0;
    for (int tile = blockIdx.x; tile < a.g.ntiles; tile += step, ++it) {
      const RowTile t = row_tile<KEYS, 128>(a.g, tile, false);
      const int r = t.r0 + row;
      const float2* nd = a.nd + (int64_t)t.bh * a.Tp;
      for (int s = 0; s < t.n; ++s, ++g) {
        const int buf = g % 3;
        mbar_wait(bars + (exp_group ? C::S_FULL : C::P_FULL) + buf, (g / 3) & 1, a.status, exp_group ? 291 : 292);
        tc_fence_after_sync();
#pragma unroll 1
        for (int ch = 0; ch < 2; ++ch) {
          const int c = t.c0 + 128 * s + 64 * cq + 32 * ch;
          const uint32_t vis = seen<KEYS>(a.g, t, r, c, false);
          const bool any = __any_sync(0xffffffffu, vis != 0u);
          const uint32_t tc = lane_base + 128 * buf + 64 * cq + 32 * ch;
          if (exp_group) {
            if (!any) continue;   // hidden columns keep what they hold: the packing group writes zeros for them
            uint32_t x[32];
            tmem_ld32(tc, x);
            tmem_ld_wait();
#pragma unroll
            for (int q = 0; q < 8; ++q) {
              const float4 n01 = __ldg(reinterpret_cast<const float4*>(nd + c) + 2 * q);
              const float4 n23 = __ldg(reinterpret_cast<const float4*>(nd + c) + 2 * q + 1);
              x[4 * q] = __float_as_uint(ex2(fmaf(__uint_as_float(x[4 * q]), sc, -n01.x)));
              x[4 * q + 1] = __float_as_uint(ex2(fmaf(__uint_as_float(x[4 * q + 1]), sc, -n01.z)));
              x[4 * q + 2] = __float_as_uint(ex2(fmaf(__uint_as_float(x[4 * q + 2]), sc, -n23.x)));
              x[4 * q + 3] = __float_as_uint(ex2(fmaf(__uint_as_float(x[4 * q + 3]), sc, -n23.z)));
            }
            tmem_st32(tc, x);
          } else {
            uint32_t o[16];
            if (any) {
              uint32_t x[32];
              tmem_ld32(tc, x);
              tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 16; ++j)
                o[j] = pack_bf16(keep_if_bit(__uint_as_float(x[2 * j]), vis, 2 * j),
                                 keep_if_bit(__uint_as_float(x[2 * j + 1]), vis, 2 * j + 1));
            } else {
#pragma unroll
              for (int j = 0; j < 16; ++j) o[j] = 0u;
            }
            tmem_st16(tc, o);
          }
        }
        tmem_st_wait();
        tc_fence_before_sync();
        warp_arrive(bars + (exp_group ? C::E_DONE : C::D_DONE) + buf, lane);
      }
      if (!exp_group) {
        mbar_wait(bars + C::DV_FULL, it & 1, a.status, 293);
        tc_fence_after_sync();
        __nv_bfloat16* dst = a.dv + t.b * a.vb + t.h * a.vh + (int64_t)r * a.vs;
#pragma unroll
        for (int q = 0; q < D / 32; ++q) {
          const int c = (D / 2) * cq + 16 * q;
          uint32_t v[16];
          tmem_ld16(lane_base + C::T_DV + c, v);
          tmem_ld_wait();
          uint32_t o[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) o[j] = pack_bf16(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1]));
          if (row < t.nr) {
            reinterpret_cast<uint4*>(dst + c)[0] = make_uint4(o[0], o[1], o[2], o[3]);
            reinterpret_cast<uint4*>(dst + c)[1] = make_uint4(o[4], o[5], o[6], o[7]);
          }
        }
        tc_fence_before_sync();
        warp_arrive(bars + C::DV_FREE, lane);
      }
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == C::W_LOAD) {
    __syncwarp();
    tmem_dealloc(tb, 512);
  }
}

// ---------------------------------------------------------------------------
// host side
bool map_rows(CUtensorMap* m, const void* base, int64_t width, int64_t rows, int BH, uint32_t box_rows) {
  const uint64_t dims[3] = {(uint64_t)width, (uint64_t)rows, (uint64_t)BH};
  const uint64_t str[2] = {(uint64_t)width * 2, (uint64_t)(rows * width) * 2};
  const uint32_t box[3] = {64, box_rows, 1};
  return cached_tmap(m, base, 3, dims, str, box);
}
bool map_w(CUtensorMap* m, const void* base, int D, uint32_t box_rows) {
  const uint64_t dims[2] = {(uint64_t)D, (uint64_t)(2 * D)};
  const uint64_t str[1] = {(uint64_t)D * 2};
  const uint32_t box[2] = {64, box_rows};
  return cached_tmap(m, base, 2, dims, str, box);
}

// Raises the kernel's shared-memory limit once per device.
template <typename K>
cudaError_t allow_smem(K kernel, uint32_t bytes, bool* done) {
  if (*done) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e == cudaSuccess) *done = true;
  return e;
}

struct Side {
  const void *x, *y;
  int64_t xb, xr, xh, yb, yr, yh;
  int rows;
};
struct Host {
  const SblParams& p;
  const SblGrads& g;
  const TcBwdWorkspace& ws;
  char* base;
  cudaStream_t st;
  DeviceInfo* dev;
  Side side[2];
  template <typename T>
  T* at(size_t off) const { return reinterpret_cast<T*>(base + off); }
  bool map_x(CUtensorMap* m, int s, uint32_t box) const {
    const Side& d = side[s];
    return map_bthe(m, d.x, p.B, d.rows, p.H, p.E, d.xb, d.xr, d.xh, box);
  }
  bool map_y(CUtensorMap* m, int s, uint32_t box) const {
    const Side& d = side[s];
    return map_bthe(m, d.y, p.B, d.rows, p.H, p.E, d.yb, d.yr, d.yh, box);
  }
  Geom geom(int s) const {
    Geom gm;
    gm.lengths = p.key_lengths;
    gm.H = p.H;
    gm.T = p.T;
    gm.S = p.S;
    // a window wider than both sequences sees everything: keeps the index arithmetic far from 2^31
    const int64_t most = 2 * (int64_t)(p.T > p.S ? p.T : p.S) + 2;
    gm.w = (int)(p.w < most ? p.w : most);
    gm.ntr = (int)div_up(side[s].rows, TR);
    gm.ntiles = gm.ntr * p.B * p.H;
    gm.by_ntr = divisor(gm.ntr);
    gm.by_h = divisor(p.H);
    return gm;
  }
};

template <int SIDE, int D>
cudaError_t launch_feat(const Host& h) {
  using C = FeatCfg<D>;
  FeatArgs a{};
  const int BH = h.p.B * h.p.H, rows = h.side[SIDE].rows;
  if (!h.map_x(&a.tm_x, SIDE, 128) || !h.map_y(&a.tm_y, SIDE, 128) || !map_w(&a.tm_hi, h.at<void>(h.ws.fwd.phiq), D, 64) ||
      !map_w(&a.tm_lo, h.at<void>(h.ws.wlo), D, 64) || !map_rows(&a.tm_f, h.at<void>(h.ws.feat[SIDE]), C::M, rows, BH, 128))
    return cudaErrorInvalidValue;
  a.lengths = h.p.key_lengths;
  a.beta = h.g.row_stats + 2 * (int64_t)BH * h.p.T;
  a.nd = h.at<float2>(h.ws.nd);
  a.off = h.at<float>(h.ws.off[SIDE]);
  a.partial = h.at<float>(h.ws.partial);
  a.status = h.at<int>(h.ws.fwd.status);
  a.H = h.p.H;
  a.rows = rows;
  a.Tp = h.ws.Tp;
  a.nsplit = h.ws.nsplit[SIDE];
  a.tau = h.p.softmax_temp;
  a.half_log_m = (float)(log((double)C::M) / 2.0);
  cudaError_t e = allow_smem(bwd_feat_kernel<SIDE, D>, C::SMEM, &h.dev->attr_bwd[D == 128][0][SIDE]);
  if (e != cudaSuccess) return e;
  bwd_feat_kernel<SIDE, D><<<dim3((unsigned)(a.nsplit * (C::M / 128)), (unsigned)BH), C::NTHR, C::SMEM, h.st>>>(a);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  const int64_t n = (int64_t)BH * C::M;
  bwd_combine_kernel<D><<<(unsigned)div_up(n * (D / 4 + 1), 256), 256, 0, h.st>>>(
      a.partial, a.nsplit, n, C::M, h.at<__nv_bfloat16>(h.ws.sum[SIDE]), h.at<__nv_bfloat16>(h.ws.sum_lo[SIDE]),
      h.at<float>(h.ws.sum1[SIDE]));
  return cudaGetLastError();
}

template <int SIDE, int D>
cudaError_t launch_side(const Host& h, void* dx, int64_t ob, int64_t orow, int64_t oh) {
  constexpr int OTHER = 1 - SIDE;
  const int BH = h.p.B * h.p.H;
  cudaError_t e;
  if constexpr (D == 128) {
    using C = WinCfg<D>;
    WinArgs a{};
    if (!h.map_x(&a.tm_x, SIDE, 128) || !h.map_y(&a.tm_y, SIDE, 128) || !h.map_x(&a.tm_xo, OTHER, 64) ||
        !h.map_y(&a.tm_yo, OTHER, 64))
      return cudaErrorInvalidValue;
    a.g = h.geom(SIDE);
    a.nd = h.at<float2>(h.ws.nd);
    a.part = h.at<float>(h.ws.part);
    a.status = h.at<int>(h.ws.fwd.status);
    a.Tp = h.ws.Tp;
    a.tau = h.p.softmax_temp;
    if ((e = allow_smem(bwd_window_kernel<SIDE, D>, C::SMEM, &h.dev->attr_bwd[1][1][SIDE])) != cudaSuccess) return e;
    bwd_window_kernel<SIDE, D><<<(unsigned)(a.g.ntiles < h.dev->sms ? a.g.ntiles : h.dev->sms), C::NTHR, C::SMEM, h.st>>>(a);
    if ((e = cudaGetLastError()) != cudaSuccess) return e;
  }
  using C = GradCfg<D>;
  GradArgs a{};
  if (!h.map_x(&a.tm_x, SIDE, 128) || !h.map_y(&a.tm_y, SIDE, 128) || !h.map_x(&a.tm_xo, OTHER, 64) ||
      !h.map_y(&a.tm_yo, OTHER, 64) || !map_rows(&a.tm_fo, h.at<void>(h.ws.feat[OTHER]), C::M, h.side[OTHER].rows, BH, 64) ||
      !map_rows(&a.tm_sum, h.at<void>(h.ws.sum[OTHER]), D, C::M, BH, 128) ||
      !map_rows(&a.tm_sum_lo, h.at<void>(h.ws.sum_lo[OTHER]), D, C::M, BH, 128) ||
      !map_w(&a.tm_hi, h.at<void>(h.ws.fwd.phiq), D, 128) || !map_w(&a.tm_lo, h.at<void>(h.ws.wlo), D, 128) ||
      !map_bthe(&a.tm_dx, dx, h.p.B, h.side[SIDE].rows, h.p.H, D, ob, orow, oh, 128))
    return cudaErrorInvalidValue;
  a.g = h.geom(SIDE);
  a.nd = h.at<float2>(h.ws.nd);
  a.delta = h.at<float>(h.ws.delta);
  a.off = h.at<float>(h.ws.off[SIDE]);
  a.sum1 = h.at<float>(h.ws.sum1[OTHER]);
  a.part = D == 128 ? h.at<float>(h.ws.part) : nullptr;
  a.status = h.at<int>(h.ws.fwd.status);
  a.Tp = h.ws.Tp;
  // Few columns: the sum over those outside the window instead of all - inside (accuracy, see the top).  It visits
  // every column, so it is used while that is at most the window's own steps and four more.
  a.whole = div_up(h.side[OTHER].rows, 64) <= div_up((int64_t)a.g.w + TR, 64) + 4;
  a.tau = h.p.softmax_temp;
  if ((e = allow_smem(bwd_grad_kernel<SIDE, D>, C::SMEM, &h.dev->attr_bwd[D == 128][2][SIDE])) != cudaSuccess) return e;
  bwd_grad_kernel<SIDE, D><<<(unsigned)(a.g.ntiles < h.dev->sms ? a.g.ntiles : h.dev->sms), C::NTHR, C::SMEM, h.st>>>(a);
  return cudaGetLastError();
}

template <int D>
cudaError_t launch_value(const Host& h) {
  using C = ValCfg<D>;
  const SblParams& p = h.p;
  const SblGrads& g = h.g;
  const int BH = p.B * p.H;
  cudaError_t e;
  ValArgs a{};
  if (!h.map_x(&a.tm_k, KEYS, 128) || !h.map_x(&a.tm_q, QUERIES, 128) || !h.map_y(&a.tm_do, QUERIES, 128) ||
      !map_rows(&a.tm_phi, h.at<void>(h.ws.feat[KEYS]), C::M, p.S, BH, 128) ||
      !map_rows(&a.tm_psi, h.at<void>(h.ws.feat[QUERIES]), C::M, p.T, BH, 128) ||
      !map_rows(&a.tm_sum, h.at<void>(h.ws.sum[QUERIES]), D, C::M, BH, 128))
    return cudaErrorInvalidValue;
  a.g = h.geom(KEYS);
  a.nd = h.at<float2>(h.ws.nd);
  a.dv = static_cast<__nv_bfloat16*>(g.dv);
  a.vb = g.dv_stride_b; a.vs = g.dv_stride_s; a.vh = g.dv_stride_h;
  a.status = h.at<int>(h.ws.fwd.status);
  a.Tp = h.ws.Tp;
  a.tau = p.softmax_temp;
  if ((e = allow_smem(bwd_value_kernel<D>, C::SMEM, &h.dev->attr_bwd[D == 128][3][0])) != cudaSuccess) return e;
  bwd_value_kernel<D><<<(unsigned)(a.g.ntiles < h.dev->sms ? a.g.ntiles : h.dev->sms), C::NTHR, C::SMEM, h.st>>>(a);
  return cudaGetLastError();
}

template <int D>
cudaError_t backward(const Host& h) {
  const SblParams& p = h.p;
  const SblGrads& g = h.g;
  cudaError_t e;
  if ((e = tc_prepare_projection(p, h.ws.fwd, h.base, h.st, true, nullptr, h.at<__nv_bfloat16>(h.ws.wlo))) != cudaSuccess)
    return e;
  bwd_rows_kernel<D><<<dim3((unsigned)(h.ws.Tp / kRowSpan), (unsigned)div_up(p.H, kRowHeads), (unsigned)p.B), 256, 0, h.st>>>(
      static_cast<const __nv_bfloat16*>(p.out), p.o_stride_b, p.o_stride_t, p.o_stride_h,
      static_cast<const __nv_bfloat16*>(g.dout), g.do_stride_b, g.do_stride_t, g.do_stride_h, g.row_stats, p.B, p.H, p.T,
      h.ws.Tp, h.at<float2>(h.ws.nd), h.at<float>(h.ws.delta));
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  if ((e = launch_feat<KEYS, D>(h)) != cudaSuccess) return e;
  if ((e = launch_feat<QUERIES, D>(h)) != cudaSuccess) return e;
  if (!(g.skip & SBL_SKIP_DV) && (e = launch_value<D>(h)) != cudaSuccess) return e;
  if (!(g.skip & SBL_SKIP_DQ) &&
      (e = launch_side<QUERIES, D>(h, g.dq, g.dq_stride_b, g.dq_stride_t, g.dq_stride_h)) != cudaSuccess)
    return e;
  if (g.skip & SBL_SKIP_DK) return cudaSuccess;
  return launch_side<KEYS, D>(h, g.dk, g.dk_stride_b, g.dk_stride_s, g.dk_stride_h);
}

}  // namespace

const char* tc_backward_strides(const SblGrads& g, const SblParams& p) {
  struct { const char* name; const void* ptr; int skip, rows; int64_t b, r, h; } t[] = {
      {"dout", g.dout, 0, p.T, g.do_stride_b, g.do_stride_t, g.do_stride_h},
      {"dq", g.dq, SBL_SKIP_DQ, p.T, g.dq_stride_b, g.dq_stride_t, g.dq_stride_h},
      {"dk", g.dk, SBL_SKIP_DK, p.S, g.dk_stride_b, g.dk_stride_s, g.dk_stride_h},
      {"dv", g.dv, SBL_SKIP_DV, p.S, g.dv_stride_b, g.dv_stride_s, g.dv_stride_h}};
  for (const auto& x : t) {
    if (g.skip & x.skip) continue;
    if (!aligned16(x.ptr)) return x.name;
    // a size-1 axis may carry any stride
    for (int64_t s : {p.B > 1 ? x.b : 8, x.rows > 1 ? x.r : 8, p.H > 1 ? x.h : 8})
      if (s % 8 != 0 || s <= 0) return x.name;
    if (x.rows > 1 && x.r < p.E) return x.name;
  }
  return nullptr;
}

void tc_plan_backward(const SblParams& p, TcBwdWorkspace* ws) {
  const size_t BH = (size_t)p.B * p.H, m = 2 * (size_t)p.r, D = p.D, T = p.T, S = p.S;
  size_t off = 0;
  auto take = [&](size_t bytes) {
    const size_t at = off;
    off = (off + bytes + 255) & ~(size_t)255;
    return at;
  };
  Workspace& f = ws->fwd;
  f = Workspace{};
  f.tensor = true;
  f.status = take(64);                       // first: hosts read the words without asking where they are
  f.wt = take((size_t)p.r * p.E * 4);
  f.phiq = take((size_t)p.r * p.E * 2);      // the projection's first bf16 term
  ws->wlo = take((size_t)p.r * p.E * 2);     // ... and its second
  ws->Tp = (int)(div_up(p.T, TR) * TR);
  ws->nd = take(BH * ws->Tp * 8);
  ws->delta = p.E == 128 ? take(BH * ws->Tp * 4) : off;
  ws->feat[QUERIES] = take(BH * T * m * 2);
  ws->feat[KEYS] = take(BH * S * m * 2);
  size_t partial = 0;
  for (int s = 0; s < 2; ++s) {
    ws->sum[s] = take(BH * m * D * 2);
    ws->sum_lo[s] = take(BH * m * D * 2);
    ws->sum1[s] = take(BH * m * 4);
    ws->off[s] = take(BH * div_up(s == QUERIES ? p.T : p.S, TR) * TR * 4);
    // one CTA per SM at a time: the fewest rounds of tiles over whole waves of CTAs; a CTA's prologue and its partial
    // summary cost about as much as three tiles
    const int ntiles = (int)div_up(s == QUERIES ? p.T : p.S, TR);
    const size_t units = BH * (m / 128);
    int best = 1;
    int64_t least = INT64_MAX;
    for (int ns = 1; ns <= 16 && ns <= ntiles; ++ns) {
      const int64_t cost = div_up((int64_t)units * ns, 148) * (div_up(ntiles, ns) + 3);
      if (cost < least) {
        least = cost;
        best = ns;
      }
    }
    ws->nsplit[s] = best;
    const size_t bytes = BH * ws->nsplit[s] * m * (D + 4) * 4;
    partial = bytes > partial ? bytes : partial;
  }
  ws->partial = take(partial);
  ws->part = p.E == 128 ? take(BH * div_up(T > S ? T : S, TR) * TR * D * 4) : off;
  f.total = off;
}

cudaError_t tc_backward(const SblParams& p, const SblGrads& g, const TcBwdWorkspace& ws, char* base, cudaStream_t st) {
  DeviceInfo* dev = nullptr;
  cudaError_t e = device_info(&dev);
  if (e != cudaSuccess) return e;
  Host h{p, g, ws, base, st, dev,
         {{p.q, g.dout, p.q_stride_b, p.q_stride_t, p.q_stride_h, g.do_stride_b, g.do_stride_t, g.do_stride_h, p.T},
          {p.k, p.v, p.k_stride_b, p.k_stride_s, p.k_stride_h, p.v_stride_b, p.v_stride_s, p.v_stride_h, p.S}}};
  return p.E == 64 ? backward<64>(h) : backward<128>(h);
}

}  // namespace sbl
