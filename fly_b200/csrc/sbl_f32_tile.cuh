// Helpers of the generic fp32 kernels: the loads and stores of either storage
// type, which forward (sbl_f32.cu) and backward (sbl_bwd_f32.cu) share, and the
// forward's 64x64 register-tiled products, fed from shared memory in K-slices of
// 16 with the next slice prefetched into registers.
#pragma once

#include "sbl_common.cuh"

namespace sbl {
namespace {

constexpr int TILE = 64;       // block tile edge
constexpr int KS = 16;         // K slice
constexpr int LDT = TILE + 4;  // shared leading dimension (keeps float4 rows 16-byte aligned)
constexpr int NTHR = 256;
constexpr int PER_THR = TILE * KS / NTHR;  // slice elements per thread = 4

__device__ __forceinline__ float ldf(const float* p) { return *p; }
__device__ __forceinline__ float ldf(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void stf(float* p, float x) { *p = x; }
__device__ __forceinline__ void stf(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

// atomic max on a float through its ordered integer image
__device__ __forceinline__ void atomic_max_float(float* addr, float v) {
  if (v >= 0.f) atomicMax(reinterpret_cast<int*>(addr), __float_as_int(v));
  else atomicMin(reinterpret_cast<unsigned int*>(addr), __float_as_uint(v));
}

// Fetches this thread's share of a TILE x KS slice (rows of a row-major
// matrix, K-contiguous) into registers; out-of-range elements read as 0.
template <typename T>
__device__ __forceinline__ void fetch_slice(float (&reg)[PER_THR], const T* base, int64_t ld, int nrows,
                                            int k0, int K) {
#pragma unroll
  for (int i = 0; i < PER_THR; ++i) {
    const int idx = threadIdx.x + i * NTHR;
    const int row = idx / KS, kk = idx % KS;
    reg[i] = (row < nrows && k0 + kk < K) ? ldf(base + (int64_t)row * ld + k0 + kk) : 0.f;
  }
}
__device__ __forceinline__ void stash_slice(float (*s)[LDT], const float (&reg)[PER_THR]) {
#pragma unroll
  for (int i = 0; i < PER_THR; ++i) {
    const int idx = threadIdx.x + i * NTHR;
    s[idx % KS][idx / KS] = reg[i];
  }
}

// acc(64x64) += A(64 x K) * B(64 x K)^T, both operands K-contiguous in global
// memory.  Thread (ty,tx) owns rows ty*4.., cols tx*4...
template <typename TA, typename TB>
__device__ __forceinline__ void tile_nt(float (&acc)[4][4], const TA* A, int64_t lda, int na, const TB* B,
                                        int64_t ldb, int nb, int K, float (*sA)[LDT], float (*sB)[LDT]) {
  const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
  float ra[PER_THR], rb[PER_THR];
  fetch_slice(ra, A, lda, na, 0, K);
  fetch_slice(rb, B, ldb, nb, 0, K);
  for (int k0 = 0; k0 < K; k0 += KS) {
    __syncthreads();
    stash_slice(sA, ra);
    stash_slice(sB, rb);
    __syncthreads();
    if (k0 + KS < K) {
      fetch_slice(ra, A, lda, na, k0 + KS, K);
      fetch_slice(rb, B, ldb, nb, k0 + KS, K);
    }
    // two-level sum: one partial per K slice, so the rounding error grows with K/16, not K
    // (the feature dimension can be tens of thousands)
    float part[4][4] = {};
#pragma unroll
    for (int kk = 0; kk < KS; ++kk) {
      const float4 a = *reinterpret_cast<const float4*>(&sA[kk][ty * 4]);
      const float4 b = *reinterpret_cast<const float4*>(&sB[kk][tx * 4]);
      const float av[4] = {a.x, a.y, a.z, a.w};
      const float bv[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) part[i][j] = fmaf(av[i], bv[j], part[i][j]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] += part[i][j];
  }
}

__device__ __forceinline__ float group16_max(float v) {
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float group16_sum(float v) {
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

}  // namespace
}  // namespace sbl
