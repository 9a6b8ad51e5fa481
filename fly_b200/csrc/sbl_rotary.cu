// Root-mean-square norm of query and key heads with a learned weight, followed
// by the rotation of pairs of entries, forward and backward, in one pass over
// the data (declared in include/sblocal_b200.h).
//
//   r = 1 / sqrt(mean(x^2) + eps),  u = r x,  z = u * weight,  y = R(pos) z
//   dz = R(pos)^T dy,  dweight = sum_rows dz * u,
//   dx = r (dz * weight - u * mean(dz * weight * u))
//
// Bound by memory (forward 2 and backward 3 passes over the rows), close behind
// it by issuing: a warp owns the tokens it visits and loops over their heads, so
// the angles of a token (one fp64 product, a reduction to a fraction of a turn
// and one sincospi per pair) are formed once per token and shared through 8
// bytes per pair of shared memory; with equal positions once for queries and
// keys.  Arithmetic goes in packed fp32 pairs.
//
// B2 N16384 H16 E64 bf16: forward 55 us, backward 82 us, 4.9 TB/s both (74 % of
// a plain copy); B1 N32768 H8 E128: 67 and 87 us.  Steps that led there, at
// the first size: 97 / 134 us with plain loads in front of their use; 71 / 91
// with the ring; 64 / 86 with packed arithmetic and the weights folded into the
// angles; 58 / 85 with the angles shared by both sides; 55 / 82 without the
// divisions of every token.  Eight stages in the ring instead of four, alone:
// no difference.
//
// Two layouts.  `vec`: a row is held by LPR lanes with 8 consecutive entries
// each (16-byte copies of bf16, two of fp32), several rows per warp; pairs of
// halves meet through one shuffle of the raw words.  It needs E % 8 == 0,
// E <= 256, rotary % 16 == 0 (halves), 16-byte aligned rows.  `scalar`: one row
// per warp, entry lane + 32 j per lane, partners re-read through L1; any E up to
// 512 and any stride.
#include <cmath>

#include "sbl_common.cuh"
#include "sbl_tc_dev.cuh"

namespace sbl {
namespace {

using namespace tcdev;

constexpr int kWarps = 4;                               // warps per block
constexpr int kMaxPairs = SBL_NORM_ROTARY_MAX_E / 2;

struct RotaryArgs {
  SblNormRotarySide side[2];
  int B, E, rotary, wbf16;
  int joint;                                            // vec: both sides in one warp
  int side0;                                            // otherwise the side of blockIdx.z = 0
  float eps;
  float* partial;                                       // backward: (2, blocks, E), null = no weight gradients
  double rate[kMaxPairs];                               // turns per position of pair i
};

__device__ __forceinline__ float weight_at(const void* w, int bf16, int e) {
  if (!w) return 1.f;
  return bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(w)[e]) : static_cast<const float*>(w)[e];
}

// cos and sin of position * rate turns.  The product keeps 53 bits and the whole turns are taken off before the
// rounding to fp32, so positions of millions cost no accuracy.
__device__ __forceinline__ float2 turn(double pos, double rate) {
  const double a = pos * rate;
  float2 cs;
  sincospif(2.f * (float)(a - rint(a)), &cs.y, &cs.x);
  return cs;
}

__device__ __forceinline__ double position_of(const SblNormRotarySide& s, int b, int t) {
  return (double)(s.positions ? s.positions[b * s.pos_stride_b + t * s.pos_stride_t] : s.pos0 + t);
}

// 8 consecutive entries of a row into shared memory, asynchronously
template <typename T>
__device__ __forceinline__ void copy_row8(T* dst, const T* src) {
  const uint32_t d = (uint32_t)__cvta_generic_to_shared(dst);
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d + 16 * i), "l"(reinterpret_cast<const char*>(src) + 16 * i)
                 : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// 8 consecutive entries as raw words
template <typename T>
struct Raw8;
template <>
struct Raw8<__nv_bfloat16> {
  uint32_t w[4];
  __device__ void load(const __nv_bfloat16* p) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  }
  __device__ void zero() { w[0] = w[1] = w[2] = w[3] = 0u; }
  __device__ void exchange(const Raw8& o, int src) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __shfl_sync(0xffffffffu, o.w[i], src);
  }
  __device__ float2 pair(int i) const { return make_float2(bf16_lo(w[i]), bf16_hi(w[i])); }
  static __device__ void store(__nv_bfloat16* p, const float (&v)[8]) {
    uint4 o;
    __nv_bfloat162 h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
    o.x = *reinterpret_cast<uint32_t*>(&h[0]); o.y = *reinterpret_cast<uint32_t*>(&h[1]);
    o.z = *reinterpret_cast<uint32_t*>(&h[2]); o.w = *reinterpret_cast<uint32_t*>(&h[3]);
    *reinterpret_cast<uint4*>(p) = o;
  }
};
template <>
struct Raw8<float> {
  float w[8];
  __device__ void load(const float* p) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w; w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
  }
  __device__ void zero() {
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = 0.f;
  }
  __device__ void exchange(const Raw8& o, int src) {
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = __shfl_sync(0xffffffffu, o.w[i], src);
  }
  __device__ float2 pair(int i) const { return make_float2(w[2 * i], w[2 * i + 1]); }
  static __device__ void store(float* p, const float (&v)[8]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  }
};

template <int LPR>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int o = 1; o < LPR; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// grid (blocks over tokens, parts of the heads, sides or 1).  With one part per side a warp takes a token's heads of both
// sides one after the other (`RotaryArgs::joint`: same tokens, same positions): the angles, a third of the instructions
// at 16 heads of 64 entries, are formed once for both.
template <typename T, int LPR, bool BWD, bool INTER>
__global__ void __launch_bounds__(32 * kWarps, BWD ? 4 : 6) vec_kernel(const __grid_constant__ RotaryArgs a) {
  constexpr int RPW = 32 / LPR;                         // rows per warp
  constexpr int EP = 8 * LPR;                           // entries held
  constexpr int kStages = sizeof(T) == 4 ? 4 : 8;        // 16 KB per block, 32 KB backward
  __shared__ double s_rate[kMaxPairs / 2];              // E <= 256: 128 pairs
  __shared__ float2 s_turn[kWarps][kMaxPairs / 2];
  __shared__ __align__(16) float s_w[2][EP];
  __shared__ float s_dw[BWD ? kWarps : 1][BWD ? 2 : 1][BWD ? EP : 1];
  // The warp's steps, RPW rows of a token each, form one stream.  Rows travel kStages - 1 steps ahead through a ring in
  // shared memory; a lane reads back what it copied itself, so that nothing but its own copies is waited for.
  __shared__ __align__(16) T s_ring[kWarps][kStages][BWD ? 2 : 1][32 * 8];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int sub = lane % LPR, grp = lane / LPR;
  const int e0 = 8 * sub, E = a.E, half = a.rotary / 2;
  const bool held = e0 < E;
  const int side_lo = a.joint ? 0 : a.side0 + blockIdx.z, side_hi = a.joint ? 2 : side_lo + 1;
  for (int i = threadIdx.x; i < half; i += 32 * kWarps) s_rate[i] = a.rate[i];
  for (int i = threadIdx.x; i < 2 * EP; i += 32 * kWarps)
    s_w[i / EP][i % EP] = i % EP < E ? weight_at(a.side[i / EP].weight, a.wbf16, i % EP) : 0.f;
  __syncthreads();
  // Halves: entry e is turned with e + half, `half / 8` lanes up (the low one) or down.  rotary % 16 == 0 here.
  const bool low = e0 < half, turned = e0 < a.rotary;
  const int src = INTER || !turned ? lane : (low ? lane + half / 8 : lane - half / 8);
  const int ep0 = INTER || !turned ? e0 : (low ? e0 + half : e0 - half);
  const float inv_e = 1.f / (float)E;
  const uint32_t T_ = (uint32_t)a.side[side_lo].T, hop = gridDim.x * kWarps, first = blockIdx.x * kWarps + warp;
  const uint32_t hop_b = T_ ? hop / T_ : 0, hop_t = T_ ? hop % T_ : 0;
  struct Cursor { uint32_t b, t; int side, h, end; };
  // this block's part of either side's heads
  const int per0 = (a.side[0].H + gridDim.y - 1) / gridDim.y, per1 = (a.side[1].H + gridDim.y - 1) / gridDim.y;
  const int lo0 = blockIdx.y * per0, lo1 = blockIdx.y * per1;
  const int hi0 = min(a.side[0].H, lo0 + per0), hi1 = min(a.side[1].H, lo1 + per1);
  auto heads = [&](Cursor& c) {
    c.h = c.side ? lo1 : lo0;
    c.end = c.side ? hi1 : hi0;
  };
  Cursor at = {T_ ? first / T_ : 0, T_ ? first % T_ : 0, side_lo, 0, 0};
  heads(at);
  const uint32_t none = (uint32_t)a.B;
  if (T_ == 0 || at.h >= at.end) at.b = none;           // (joint: one part, which is never empty)
  auto advance = [&](Cursor& c) {                       // true: another side or token
    c.h += RPW;
    if (c.h < c.end) return false;
    if (++c.side == side_hi) {
      c.side = side_lo;
      c.b += hop_b;
      c.t += hop_t;                                     // (both below 2^31)
      if (c.t >= T_) {
        c.t -= T_;
        ++c.b;
      }
    }
    heads(c);
    return true;
  };
  Cursor ahead = at;
  const T *x, *dy;
  int64_t x_hop, dy_hop;
  auto seek = [&]() {                                   // the lane's row of the step `ahead`
    const SblNormRotarySide& s = a.side[ahead.side];
    const int64_t h = ahead.h + grp;
    x = static_cast<const T*>(s.x) + ahead.b * s.x_stride_b + ahead.t * s.x_stride_t + h * s.x_stride_h + e0;
    x_hop = RPW * s.x_stride_h;
    if (BWD) {
      dy = static_cast<const T*>(s.dy) + ahead.b * s.dy_stride_b + ahead.t * s.dy_stride_t + h * s.dy_stride_h + e0;
      dy_hop = RPW * s.dy_stride_h;
    }
  };
  T* const ring = &s_ring[warp][0][0][8 * lane];
  constexpr int SLOT = (BWD ? 2 : 1) * 32 * 8;
  auto fetch = [&](int slot) {
    if (ahead.b < none) {
      if (held && ahead.h + grp < ahead.end) {
        copy_row8(ring + slot * SLOT, x);
        if (BWD) copy_row8(ring + slot * SLOT + 32 * 8, dy);
      }
      if (advance(ahead)) {
        seek();
      } else {
        x += x_hop;
        if (BWD) dy += dy_hop;
      }
    }
    copies_commit();
  };
  seek();
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) fetch(i);
  // y = r (x * cs + x_partner * sn), the weights in them; backward: dz = dy * cs - dy_partner * sn without
  float2 cs[4], sn[4], wt[4], dw[4], dw_other[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) dw[i] = dw_other[i] = make_float2(0.f, 0.f);
  T* y = nullptr;
  int64_t y_hop = 0;
  bool fresh = true;
  for (uint32_t step = 0; at.b < none; ++step) {
    const int slot = (int)(step % kStages);
    // into the slot of the step before, whose rows are in registers or stored
    fetch((int)((step + kStages - 1) % kStages));
    if (fresh) {
      const SblNormRotarySide& s = a.side[at.side];
      if (half > 0 && at.side == side_lo) {
        const double pos = position_of(s, at.b, at.t);
        __syncwarp();
        for (int i = lane; i < half; i += 32) s_turn[warp][i] = turn(pos, s_rate[i]);
        __syncwarp();
      }
      float c[8], n[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        c[i] = 1.f;
        n[i] = 0.f;
        if (INTER) {
          if (e0 + i < a.rotary) {
            const float2 t = s_turn[warp][(e0 + i) / 2];
            c[i] = t.x;
            n[i] = (i & 1) ? t.y : -t.y;
          }
        } else if (turned) {
          const float2 t = s_turn[warp][low ? e0 + i : e0 + i - half];
          c[i] = t.x;
          n[i] = low ? -t.y : t.y;
        }
      }
      const float2* w = reinterpret_cast<const float2*>(&s_w[at.side][e0]);
      const float2* wp = reinterpret_cast<const float2*>(&s_w[at.side][ep0]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        cs[i] = make_float2(c[2 * i], c[2 * i + 1]);
        sn[i] = make_float2(n[2 * i], n[2 * i + 1]);
        if (!BWD) {
          const float2 p = wp[i];
          cs[i] = mul2(cs[i], w[i]);
          sn[i] = mul2(sn[i], INTER ? make_float2(p.y, p.x) : p);
        } else {
          sn[i] = make_float2(-sn[i].x, -sn[i].y);      // the inverse turn
          wt[i] = w[i];
        }
        if (BWD && a.joint && step > 0) {               // the other side's sums
          const float2 d = dw[i];
          dw[i] = dw_other[i];
          dw_other[i] = d;
        }
      }
      y = static_cast<T*>(s.y) + at.b * s.y_stride_b + at.t * s.y_stride_t + (int64_t)(at.h + grp) * s.y_stride_h + e0;
      y_hop = RPW * s.y_stride_h;
    }
    const bool row = held && at.h + grp < at.end;
    copies_wait<kStages - 1>();
    Raw8<T> rx, rd;
    rx.zero();
    if (row) rx.load(ring + slot * SLOT);
    if (BWD) {
      rd.zero();
      if (row) rd.load(ring + slot * SLOT + 32 * 8);
    }
    float2 v[4], sq = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = rx.pair(i);
      sq = fma2(v[i], v[i], sq);
    }
    // what is turned: x forward, dy backward; its partner is the other half, or the other entry of the pair
    const Raw8<T>& raw = BWD ? rd : rx;
    Raw8<T> rp;
    if (!INTER) rp.exchange(raw, src);
    float2 z[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 m = BWD ? raw.pair(i) : v[i];
      const float2 p = INTER ? make_float2(m.y, m.x) : rp.pair(i);
      z[i] = fma2(p, sn[i], mul2(m, cs[i]));
    }
    const float r = rsqrtf(row_sum<LPR>(sq.x + sq.y) * inv_e + a.eps);
    const float2 r2 = make_float2(r, r);
    float o[8];
    if (!BWD) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 t = mul2(z[i], r2);
        o[2 * i] = t.x;
        o[2 * i + 1] = t.y;
      }
    } else {
      float2 zw[4], dot = make_float2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        zw[i] = mul2(z[i], wt[i]);
        dot = fma2(zw[i], v[i], dot);
        dw[i] = fma2(z[i], mul2(v[i], r2), dw[i]);
      }
      const float c = -row_sum<LPR>(dot.x + dot.y) * r * r * inv_e;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 t = mul2(r2, fma2(v[i], make_float2(c, c), zw[i]));
        o[2 * i] = t.x;
        o[2 * i + 1] = t.y;
      }
    }
    if (row) Raw8<T>::store(y, o);
    y += y_hop;
    fresh = advance(at);
  }
  if (BWD && a.partial) {
    // Lane groups, then warps, in a fixed order.  A joint warp has ended with the second side in `dw` (one without
    // tokens has zeros in both).
#pragma unroll
    for (int i = 0; i < 8; ++i) {
#pragma unroll
      for (int side = 0; side < 2; ++side) {
        const float2 p = side == 0 ? dw[i / 2] : dw_other[i / 2];
        float d = (i & 1) ? p.y : p.x;
#pragma unroll
        for (int o = LPR; o < 32; o <<= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
        if (grp == 0) s_dw[warp][a.joint ? 1 - side : side][e0 + i] = d;
      }
    }
    __syncthreads();
    for (int side = side_lo; side < side_hi; ++side) {
      const int64_t block = ((int64_t)side * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x;
      for (int e = threadIdx.x; e < E; e += 32 * kWarps) {
        float sum = 0.f;
        for (int w = 0; w < kWarps; ++w) sum += s_dw[w][a.joint ? side : 0][e];
        a.partial[block * E + e] = sum;
      }
    }
  }
}

__device__ __forceinline__ float ld1(const float* p) { return *p; }
__device__ __forceinline__ float ld1(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void st1(float* p, float v) { *p = v; }
__device__ __forceinline__ void st1(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// NJ entries per lane: E <= 32 NJ
template <typename T, int NJ, bool BWD>
__global__ void __launch_bounds__(32 * kWarps) scalar_kernel(const __grid_constant__ RotaryArgs a, int interleaved) {
  __shared__ float s_dw[BWD ? kWarps : 1][BWD ? 32 * NJ : 1];
  const int side = a.side0 + blockIdx.z;
  const SblNormRotarySide& s = a.side[side];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int E = a.E, half = a.rotary / 2;
  float wt[NJ], wp[NJ], dw[NJ];
  int ep[NJ];
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const int e = lane + 32 * j;
    ep[j] = e >= a.rotary ? e : (interleaved ? (e ^ 1) : (e < half ? e + half : e - half));
    wt[j] = e < E ? weight_at(s.weight, a.wbf16, e) : 0.f;
    wp[j] = e < E ? weight_at(s.weight, a.wbf16, ep[j]) : 0.f;
    dw[j] = 0.f;
  }
  const int H = s.H, per = (H + gridDim.y - 1) / gridDim.y;
  const int h_lo = blockIdx.y * per, h_hi = min(H, h_lo + per);
  const int64_t tokens = (int64_t)a.B * s.T;
  const float inv_e = 1.f / (float)E;
  for (int64_t tok = (int64_t)blockIdx.x * kWarps + warp; tok < tokens; tok += (int64_t)gridDim.x * kWarps) {
    const int b = (int)(tok / s.T), t = (int)(tok - (int64_t)b * s.T);
    float cs[NJ], sn[NJ];
    const double pos = half > 0 ? position_of(s, b, t) : 0.0;
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int e = lane + 32 * j;
      cs[j] = 1.f;
      sn[j] = 0.f;
      if (e < a.rotary) {
        const float2 c = turn(pos, a.rate[interleaved ? e / 2 : (e < half ? e : e - half)]);
        cs[j] = c.x;
        sn[j] = (interleaved ? (e & 1) == 0 : e < half) ? -c.y : c.y;
      }
    }
    for (int h = h_lo; h < h_hi; ++h) {
      const T* x = static_cast<const T*>(s.x) + b * s.x_stride_b + t * s.x_stride_t + h * s.x_stride_h;
      T* y = static_cast<T*>(s.y) + b * s.y_stride_b + t * s.y_stride_t + h * s.y_stride_h;
      float v[NJ], sq = 0.f;
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int e = lane + 32 * j;
        v[j] = e < E ? ld1(x + e) : 0.f;
        sq = fmaf(v[j], v[j], sq);
      }
      if (!BWD) {
        const float r = rsqrtf(row_sum<32>(sq) * inv_e + a.eps);
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          const int e = lane + 32 * j;
          if (e < E) {
            float o = (v[j] * r * wt[j]) * cs[j];
            if (e < a.rotary) o += (ld1(x + ep[j]) * r * wp[j]) * sn[j];
            st1(y + e, o);
          }
        }
      } else {
        const T* dy = static_cast<const T*>(s.dy) + b * s.dy_stride_b + t * s.dy_stride_t + h * s.dy_stride_h;
        float dz[NJ], dot = 0.f;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          const int e = lane + 32 * j;
          dz[j] = 0.f;
          if (e < E) {
            dz[j] = ld1(dy + e) * cs[j];
            if (e < a.rotary) dz[j] -= ld1(dy + ep[j]) * sn[j];
          }
          dot = fmaf(dz[j] * wt[j], v[j], dot);
        }
        const float r = rsqrtf(row_sum<32>(sq) * inv_e + a.eps);
        const float c = row_sum<32>(dot) * r * r * inv_e;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          const int e = lane + 32 * j;
          dw[j] = fmaf(dz[j], v[j] * r, dw[j]);
          if (e < E) st1(y + e, r * (dz[j] * wt[j] - v[j] * c));
        }
      }
    }
  }
  if (BWD && a.partial) {
#pragma unroll
    for (int j = 0; j < NJ; ++j) s_dw[warp][lane + 32 * j] = dw[j];
    __syncthreads();
    const int64_t block = ((int64_t)side * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x;
    for (int e = threadIdx.x; e < E; e += 32 * kWarps) {
      float sum = 0.f;
      for (int w = 0; w < kWarps; ++w) sum += s_dw[w][e];
      a.partial[block * E + e] = sum;
    }
  }
}

// dweight[side][e] = sum over the blocks' partials, in a fixed order; grid (E / 32, sides), 32 x 32 threads
__global__ void __launch_bounds__(1024) weight_grad_kernel(const float* partial, int blocks, int E, void* d0, void* d1,
                                                           int wbf16) {
  __shared__ float s[32][33];
  void* out = blockIdx.y ? d1 : d0;
  const int e = blockIdx.x * 32 + threadIdx.x;
  float sum = 0.f;
  if (out && e < E)
    for (int k = threadIdx.y; k < blocks; k += 32) sum += partial[((int64_t)blockIdx.y * blocks + k) * E + e];
  s[threadIdx.y][threadIdx.x] = sum;
  __syncthreads();
  if (threadIdx.y == 0 && out && e < E) {
    for (int k = 1; k < 32; ++k) sum += s[k][threadIdx.x];
    if (wbf16) static_cast<__nv_bfloat16*>(out)[e] = __float2bfloat16_rn(sum);
    else static_cast<float*>(out)[e] = sum;
  }
}

bool fits16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

bool side_is_vec(const SblNormRotarySide& s, bool bwd) {
  if ((int64_t)s.T * s.H == 0) return true;
  int64_t all = s.x_stride_b | s.x_stride_t | s.x_stride_h | s.y_stride_b | s.y_stride_t | s.y_stride_h;
  bool ok = fits16(s.x) && fits16(s.y);
  if (bwd) {
    all |= s.dy_stride_b | s.dy_stride_t | s.dy_stride_h;
    ok = ok && fits16(s.dy);
  }
  return ok && all % 8 == 0;
}

// Blocks over tokens and over heads.  Heads are split only while there are too few tokens to give every SM 16 warps
// (a handful of decoded tokens: one step of rows per warp instead of a loop).
// Over tokens no more blocks than an SM holds at once (registers), so that all of them end together.
void plan(const SblNormRotary& p, int rpw, bool bwd, unsigned* gx, unsigned* gy, bool* joint) {
  const int64_t tokens = (int64_t)p.B * (p.side[0].T > p.side[1].T ? p.side[0].T : p.side[1].T);
  const int H = p.side[0].H > p.side[1].H ? p.side[0].H : p.side[1].H;
  const int64_t steps = div_up(H, rpw);
  int64_t parts = 1;
  while (parts * 2 <= steps && tokens * parts * 2 <= 148 * 16) parts *= 2;
  int64_t bx = tokens > 0 ? div_up(tokens, kWarps) : 1;
  const SblNormRotarySide &q = p.side[0], &k = p.side[1];
  *joint = parts == 1 && q.T == k.T && q.positions == k.positions && q.pos0 == k.pos0 &&
           (!q.positions || (q.pos_stride_b == k.pos_stride_b && q.pos_stride_t == k.pos_stride_t));
  const int64_t most = 148 * (bwd ? 4 : 6) / (*joint ? 1 : 2);
  if (bx > most) bx = most;
  *gx = (unsigned)bx;
  *gy = (unsigned)parts;
}

template <typename T, bool BWD>
cudaError_t launch(const SblNormRotary& p, RotaryArgs& a, cudaStream_t st) {
  const bool inter = p.interleaved != 0;
  const bool vec = p.E % 8 == 0 && p.E <= 256 && (inter || p.rotary % 16 == 0) && side_is_vec(p.side[0], BWD) &&
                   side_is_vec(p.side[1], BWD);
  // A side whose gradients nobody needs has no blocks.  The plan is that of both, so that the other side's sums keep
  // their order.
  const bool skip0 = BWD && !p.side[0].y && !p.side[0].dweight, skip1 = BWD && !p.side[1].y && !p.side[1].dweight;
  if (skip0 && skip1) return cudaSuccess;
  a.side0 = skip0;
  const unsigned sides = skip0 || skip1 ? 1 : 2;
  unsigned gx, gy;
  bool joint;
  if (vec) {
    const int lpr = p.E <= 32 ? 4 : p.E <= 64 ? 8 : p.E <= 128 ? 16 : 32;
    plan(p, 32 / lpr, BWD, &gx, &gy, &joint);
    a.joint = joint && sides == 2;
    const dim3 grid(gx, gy, a.joint ? 1 : sides);
#define SBL_VEC(L)                                                                                  \
  (inter ? vec_kernel<T, L, BWD, true><<<grid, 32 * kWarps, 0, st>>>(a)                             \
         : vec_kernel<T, L, BWD, false><<<grid, 32 * kWarps, 0, st>>>(a))
    if (lpr == 4) SBL_VEC(4);
    else if (lpr == 8) SBL_VEC(8);
    else if (lpr == 16) SBL_VEC(16);
    else SBL_VEC(32);
#undef SBL_VEC
  } else {
    plan(p, 1, BWD, &gx, &gy, &joint);
    const dim3 grid(gx, gy, sides);
    if (p.E <= 128) scalar_kernel<T, 4, BWD><<<grid, 32 * kWarps, 0, st>>>(a, inter);
    else scalar_kernel<T, 16, BWD><<<grid, 32 * kWarps, 0, st>>>(a, inter);
  }
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || !BWD || !a.partial) return e;
  const int blocks = (int)(gx * gy);
  weight_grad_kernel<<<dim3((unsigned)div_up(p.E, 32), 2), dim3(32, 32), 0, st>>>(
      a.partial, blocks, p.E, p.side[0].dweight, p.side[1].dweight, a.wbf16);
  return cudaGetLastError();
}

}  // namespace

size_t norm_rotary_partial_bytes(const SblNormRotary& p) {
  // an upper bound of what plan() may ask for: blocks over tokens x parts of the heads, two sides
  unsigned gx, gy, best = 0;
  bool joint;
  for (int rpw = 1; rpw <= 8; rpw *= 2) {
    plan(p, rpw, true, &gx, &gy, &joint);
    if (gx * gy > best) best = gx * gy;
  }
  return (size_t)best * 2 * p.E * sizeof(float);
}

cudaError_t norm_rotary(const SblNormRotary& p, bool backward, float* partial, cudaStream_t st) {
  RotaryArgs a;
  a.side[0] = p.side[0];
  a.side[1] = p.side[1];
  a.B = p.B;
  a.E = p.E;
  a.rotary = p.rotary;
  a.wbf16 = p.weight_dtype == SBL_DTYPE_BF16;
  a.eps = (float)p.eps;
  a.partial = partial;
  const double turns = 1.0 / (2.0 * 3.14159265358979323846);
  for (int i = 0; i < p.rotary / 2; ++i) a.rate[i] = pow(p.theta, -2.0 * i / p.rotary) * turns;
  if (p.dtype == SBL_DTYPE_BF16)
    return backward ? launch<__nv_bfloat16, true>(p, a, st) : launch<__nv_bfloat16, false>(p, a, st);
  return backward ? launch<float, true>(p, a, st) : launch<float, false>(p, a, st);
}

}  // namespace sbl
