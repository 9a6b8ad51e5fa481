// Root-mean-square norm of query and key heads with a learned weight, followed
// by the rotation of pairs of entries, forward and backward, in one pass over
// the data (declared in include/sblocal_b200.h).
//
//   r = 1 / sqrt(mean(x^2) + eps),  u = r x,  z = u * weight,  y = R(pos) z
//   dz = R(pos)^T dy,  dweight = sum_rows dz * u,
//   dx = r (dz * weight - u * mean(dz * weight * u))
//
// Bound by memory: forward 2 and backward 3 passes over the rows.  A warp owns
// the tokens it visits and loops over their heads, so the angles of a token
// (one fp64 product, a reduction to a fraction of a turn and one sincospi per
// pair) are formed once per token, shared through 8 bytes per pair of shared
// memory, and cost about a tenth of the row work at 16 heads.
//
// Two layouts.  `vec`: a row is held by LPR lanes with 8 consecutive entries
// each (16-byte accesses of bf16, two of fp32), several rows per warp; pairs of
// halves meet through one shuffle of the raw words.  It needs E % 8 == 0,
// E <= 256, rotary % 16 == 0 (halves), 16-byte aligned rows.  `scalar`: one row
// per warp, entry lane + 32 j per lane, partners re-read through L1; any E up to
// 512 and any stride.
#include <cmath>

#include "sbl_common.cuh"

namespace sbl {
namespace {

constexpr int kWarps = 4;                               // warps per block
constexpr int kStages = 4;                              // row steps in the ring of a warp
constexpr int kMaxPairs = SBL_NORM_ROTARY_MAX_E / 2;

struct RotaryArgs {
  SblNormRotarySide side[2];
  int B, E, rotary, wbf16;
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
  __device__ float at(int i) const { return __uint_as_float((i & 1) ? (w[i >> 1] & 0xffff0000u) : (w[i >> 1] << 16)); }
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
  __device__ float at(int i) const { return w[i]; }
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

// grid (blocks over tokens, parts of the heads, sides)
template <typename T, int LPR, bool BWD, bool INTER>
__global__ void __launch_bounds__(32 * kWarps) vec_kernel(const __grid_constant__ RotaryArgs a) {
  constexpr int RPW = 32 / LPR;                         // rows per warp
  __shared__ double s_rate[kMaxPairs / 2];              // E <= 256: 128 pairs
  __shared__ float2 s_turn[kWarps][kMaxPairs / 2];
  __shared__ float s_dw[BWD ? kWarps : 1][BWD ? 8 * LPR : 1];
  const SblNormRotarySide& s = a.side[blockIdx.z];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int sub = lane % LPR, grp = lane / LPR;
  const int e0 = 8 * sub, E = a.E, half = a.rotary / 2;
  const bool held = e0 < E;
  for (int i = threadIdx.x; i < half; i += 32 * kWarps) s_rate[i] = a.rate[i];
  __syncthreads();
  // Halves: entry e is turned with e + half, `half / 8` lanes up (the low one) or down.  rotary % 16 == 0 here.
  const bool low = e0 < half, turned = e0 < a.rotary;
  const int src = INTER || !turned ? lane : (low ? lane + half / 8 : lane - half / 8);
  float wt[8], wp[8], dw[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int e = e0 + i, ep = INTER || !turned ? e : (low ? e + half : e - half);
    wt[i] = held ? weight_at(s.weight, a.wbf16, e) : 0.f;
    wp[i] = held ? weight_at(s.weight, a.wbf16, ep) : 0.f;
    dw[i] = 0.f;
  }
  const int H = s.H, per = (H + gridDim.y - 1) / gridDim.y;
  const int h_lo = blockIdx.y * per, h_hi = min(H, h_lo + per);
  const float inv_e = 1.f / (float)E;
  // The warp's steps, RPW rows of a token each, form one stream.  Rows travel kStages - 1 steps ahead through a ring in
  // shared memory; a lane reads back what it copied itself, so that nothing but its own copies is waited for.
  __shared__ __align__(16) T s_ring[kWarps][kStages][BWD ? 2 : 1][32 * 8];
  const uint32_t T_ = (uint32_t)s.T, hop = gridDim.x * kWarps, first = blockIdx.x * kWarps + warp;
  const uint32_t hop_b = T_ ? hop / T_ : 0, hop_t = T_ ? hop % T_ : 0;
  struct Cursor { uint32_t b, t; int h; };
  Cursor at = {T_ ? first / T_ : 0, T_ ? first % T_ : 0, h_lo};
  const uint32_t none = (uint32_t)a.B;
  if (T_ == 0 || h_lo >= h_hi) at.b = none;
  auto advance = [&](Cursor& c) {
    c.h += RPW;
    if (c.h >= h_hi) {
      c.h = h_lo;
      c.b += hop_b;
      c.t += hop_t;                                     // (both below 2^31)
      if (c.t >= T_) {
        c.t -= T_;
        ++c.b;
      }
    }
  };
  Cursor ahead = at;
  auto fetch = [&](int slot) {
    if (ahead.b < none) {
      if (held && ahead.h + grp < h_hi) {
        const int64_t h = ahead.h + grp;
        copy_row8(&s_ring[warp][slot][0][8 * lane],
                  static_cast<const T*>(s.x) + ahead.b * s.x_stride_b + ahead.t * s.x_stride_t + h * s.x_stride_h + e0);
        if (BWD)
          copy_row8(&s_ring[warp][slot][BWD ? 1 : 0][8 * lane],
                    static_cast<const T*>(s.dy) + ahead.b * s.dy_stride_b + ahead.t * s.dy_stride_t + h * s.dy_stride_h + e0);
      }
      advance(ahead);
    }
    copies_commit();
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) fetch(i);
  float cs[8], sn[8];                                   // y = z * cs + z_partner * sn
  T* y = nullptr;
  for (uint32_t step = 0; at.b < none; ++step, advance(at)) {
    const int slot = (int)(step % kStages);
    // into the slot of the step before, whose rows are in registers or stored
    fetch((int)((step + kStages - 1) % kStages));
    if (at.h == h_lo) {
      if (half > 0) {
        const double pos = position_of(s, at.b, at.t);
        __syncwarp();
        for (int i = lane; i < half; i += 32) s_turn[warp][i] = turn(pos, s_rate[i]);
        __syncwarp();
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        cs[i] = 1.f;
        sn[i] = 0.f;
        if (INTER) {
          if (e0 + i < a.rotary) {
            const float2 c = s_turn[warp][(e0 + i) / 2];
            cs[i] = c.x;
            sn[i] = (i & 1) ? c.y : -c.y;
          }
        } else if (turned) {
          const float2 c = s_turn[warp][low ? e0 + i : e0 + i - half];
          cs[i] = c.x;
          sn[i] = low ? -c.y : c.y;
        }
      }
      y = static_cast<T*>(s.y) + at.b * s.y_stride_b + at.t * s.y_stride_t + e0;
    }
    {
      const int64_t h = at.h + grp;
      const bool row = held && h < h_hi;
      copies_wait<kStages - 1>();
      Raw8<T> rx, rp;
      rx.zero();
      if (row) rx.load(&s_ring[warp][slot][0][8 * lane]);
      float v[8], sq = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[i] = rx.at(i);
        sq = fmaf(v[i], v[i], sq);
      }
      if (!BWD) {
        const float r = rsqrtf(row_sum<LPR>(sq) * inv_e + a.eps);
        float o[8];
        if (INTER) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            o[i] = (v[i] * r * wt[i]) * cs[i] + (v[i ^ 1] * r * wt[i ^ 1]) * sn[i];
        } else {
          rp.exchange(rx, src);
#pragma unroll
          for (int i = 0; i < 8; ++i) o[i] = (v[i] * r * wt[i]) * cs[i] + (rp.at(i) * r * wp[i]) * sn[i];
        }
        if (row) Raw8<T>::store(y + h * s.y_stride_h, o);
      } else {
        Raw8<T> rd;
        rd.zero();
        if (row) rd.load(&s_ring[warp][slot][1][8 * lane]);
        float dz[8], dot = 0.f;
        // the inverse turn: the sign of the sine flips
        if (INTER) {
#pragma unroll
          for (int i = 0; i < 8; ++i) dz[i] = rd.at(i) * cs[i] - rd.at(i ^ 1) * sn[i];
        } else {
          rp.exchange(rd, src);
#pragma unroll
          for (int i = 0; i < 8; ++i) dz[i] = rd.at(i) * cs[i] - rp.at(i) * sn[i];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) dot = fmaf(dz[i] * wt[i], v[i], dot);
        const float r = rsqrtf(row_sum<LPR>(sq) * inv_e + a.eps);
        const float c = row_sum<LPR>(dot) * r * r * inv_e;
        float o[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float u = v[i] * r;
          dw[i] = fmaf(dz[i], u, dw[i]);
          o[i] = r * (dz[i] * wt[i] - v[i] * c);
        }
        if (row) Raw8<T>::store(y + h * s.y_stride_h, o);
      }
    }
  }
  if (BWD && a.partial) {
    // lane groups, then warps, in a fixed order
#pragma unroll
    for (int i = 0; i < 8; ++i) {
#pragma unroll
      for (int o = LPR; o < 32; o <<= 1) dw[i] += __shfl_xor_sync(0xffffffffu, dw[i], o);
      if (grp == 0) s_dw[warp][e0 + i] = dw[i];
    }
    __syncthreads();
    const int64_t block = ((int64_t)blockIdx.z * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x;
    for (int e = threadIdx.x; e < E; e += 32 * kWarps) {
      float sum = 0.f;
      for (int w = 0; w < kWarps; ++w) sum += s_dw[w][e];
      a.partial[block * E + e] = sum;
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
  const SblNormRotarySide& s = a.side[blockIdx.z];
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
    const int64_t block = ((int64_t)blockIdx.z * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x;
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
void plan(const SblNormRotary& p, int rpw, bool bwd, unsigned* gx, unsigned* gy) {
  const int64_t tokens = (int64_t)p.B * (p.side[0].T > p.side[1].T ? p.side[0].T : p.side[1].T);
  const int H = p.side[0].H > p.side[1].H ? p.side[0].H : p.side[1].H;
  const int64_t steps = div_up(H, rpw);
  int64_t parts = 1;
  while (parts * 2 <= steps && tokens * parts * 2 <= 148 * 16) parts *= 2;
  int64_t bx = tokens > 0 ? div_up(tokens, kWarps) : 1;
  const int64_t most = bwd ? 148 * 4 : 148 * 8;   // per side: the backward's blocks each leave a row of partials
  if (bx > most) bx = most;
  *gx = (unsigned)bx;
  *gy = (unsigned)parts;
}

template <typename T, bool BWD>
cudaError_t launch(const SblNormRotary& p, RotaryArgs& a, cudaStream_t st) {
  const bool inter = p.interleaved != 0;
  const bool vec = p.E % 8 == 0 && p.E <= 256 && (inter || p.rotary % 16 == 0) && side_is_vec(p.side[0], BWD) &&
                   side_is_vec(p.side[1], BWD);
  unsigned gx, gy;
  if (vec) {
    const int lpr = p.E <= 32 ? 4 : p.E <= 64 ? 8 : p.E <= 128 ? 16 : 32;
    plan(p, 32 / lpr, BWD, &gx, &gy);
    const dim3 grid(gx, gy, 2);
#define SBL_VEC(L)                                                                                  \
  (inter ? vec_kernel<T, L, BWD, true><<<grid, 32 * kWarps, 0, st>>>(a)                             \
         : vec_kernel<T, L, BWD, false><<<grid, 32 * kWarps, 0, st>>>(a))
    if (lpr == 4) SBL_VEC(4);
    else if (lpr == 8) SBL_VEC(8);
    else if (lpr == 16) SBL_VEC(16);
    else SBL_VEC(32);
#undef SBL_VEC
  } else {
    plan(p, 1, BWD, &gx, &gy);
    const dim3 grid(gx, gy, 2);
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
  for (int rpw = 1; rpw <= 8; rpw *= 2) {
    plan(p, rpw, true, &gx, &gy);
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
