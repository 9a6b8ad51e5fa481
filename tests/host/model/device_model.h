// What the tensor-core kernels need of a GPU, on the host: CUDA's spellings for a thread of a block, and the PTX wrappers of
// sbl_tc_ptx.cuh and sbl_tc_dev.cuh over the models of device_model.cpp.  The kernels' own source is compiled against
// this (translate.py), block by block, and run under a random schedule.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <functional>

#undef __launch_bounds__
#define __launch_bounds__(...)
#undef __grid_constant__
#define __grid_constant__
#undef __shared__
#define __shared__ static
#undef __global__
#define __global__
#undef __device__
#define __device__
#undef __host__
#define __host__
#undef __forceinline__
#define __forceinline__ inline
#undef __noinline__
#define __noinline__
#undef __align__
#define __align__(x) alignas(x)

namespace model {

struct Index {
  unsigned x, y, z;
};
extern Index block_index, grid_size, block_size;
extern uint8_t* smem;                 // dynamic shared memory of the block
extern uint32_t tmem[128][512];
extern int sms;                       // what the host side takes for the number of SMs
Index& thread_index();

void seed(unsigned s);                // of the schedules that follow
void launch(dim3 grid, dim3 block, size_t smem_bytes, std::function<void()> body);

// A thread may be put aside here, so that others come in between.
void pause();
void barrier_sync(int id, int threads);
enum Op { SYNC, ANY, ALL, XOR, FROM, WAIT };
uint64_t collective(Op op, uint64_t value, int arg);

void mbar_init(uint64_t* bar, uint32_t count);
void mbar_arrive(uint64_t* bar);
void mbar_expect_tx(uint64_t* bar, uint32_t bytes);
bool mbar_test(uint64_t* bar, uint32_t parity);
void mbar_wait(uint64_t* bar, uint32_t parity, int code);

void load(void* dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z, int u);
void load_bytes(void* dst, const void* src, uint32_t bytes, uint64_t* bar);
void store(const CUtensorMap* map, const void* src, int x, int y, int z, int u);
void store_commit();
void store_wait(int groups);

void mma(uint32_t d, uint64_t a, bool a_in_tmem, uint64_t b, uint32_t idesc, bool accumulate);
void mma_commit(uint64_t* bar);

[[noreturn]] void fail(const char* what);

}  // namespace model

#define threadIdx (model::thread_index())
#define blockIdx (model::block_index)
#define gridDim (model::grid_size)
#define blockDim (model::block_size)
#define __syncthreads() model::barrier_sync(0, model::block_size.x* model::block_size.y)
#define cudaGetLastError() cudaSuccess
#define cudaFuncSetAttribute(...) cudaSuccess

inline void __syncwarp(unsigned = ~0u) { model::collective(model::SYNC, 0, 0); }
inline int __any_sync(unsigned, int p) { return (int)model::collective(model::ANY, p != 0, 0); }
inline int __all_sync(unsigned, int p) { return (int)model::collective(model::ALL, p != 0, 0); }
template <typename T>
T shuffle(model::Op op, T v, int lane) {
  uint64_t bits = 0;
  memcpy(&bits, &v, sizeof v);
  bits = model::collective(op, bits, lane);
  memcpy(&v, &bits, sizeof v);
  return v;
}
template <typename T>
T __shfl_xor_sync(unsigned, T v, int mask) { return shuffle(model::XOR, v, mask); }
template <typename T>
T __shfl_sync(unsigned, T v, int lane) { return shuffle(model::FROM, v, lane); }
template <typename T>
T __ldg(const T* p) { return *p; }
template <typename To, typename From>
To as(From v) {
  To r;
  static_assert(sizeof r == sizeof v, "");
  memcpy(&r, &v, sizeof r);
  return r;
}
inline float __uint_as_float(uint32_t u) { return as<float>(u); }
inline uint32_t __float_as_uint(float f) { return as<uint32_t>(f); }
inline int __float_as_int(float f) { return as<int>(f); }
inline int atomicCAS(int* p, int expected, int v) {
  const int old = *p;
  if (old == expected) *p = v;
  return old;
}
inline int min(int a, int b) { return a < b ? a : b; }
inline int max(int a, int b) { return a > b ? a : b; }
inline int64_t min(int64_t a, int64_t b) { return a < b ? a : b; }
inline int64_t max(int64_t a, int64_t b) { return a > b ? a : b; }

namespace sbl {

namespace ptx {

inline uint32_t smem_u32(const void* p) { return (uint32_t)(static_cast<const uint8_t*>(p) - model::smem); }
inline bool elect_one() {
  __syncwarp();
  return threadIdx.x % 32 == 0;
}
inline void mbar_init(uint64_t* bar, uint32_t count) { model::mbar_init(bar, count); }
inline void mbar_arrive(uint64_t* bar) { model::mbar_arrive(bar); }
inline void mbar_expect_tx(uint64_t* bar, uint32_t bytes) { model::mbar_expect_tx(bar, bytes); }
inline bool mbar_wait(uint64_t* bar, uint32_t parity, int*, int code) {
  model::mbar_wait(bar, parity, code);
  return true;
}
inline void fence_mbar_init() {}
inline void fence_async_smem() {}
inline void tc_fence_before_sync() {}
inline void tc_fence_after_sync() {}
inline void prefetch_tmap(const CUtensorMap*) {}
inline void tma_prefetch_4d(const CUtensorMap*, int, int, int, int) {}
inline void tma_prefetch_3d(const CUtensorMap*, int, int, int) {}
inline void tma_load_2d(void* s, const CUtensorMap* m, uint64_t* b, int x, int y) { model::load(s, m, b, x, y, 0, 0); }
inline void tma_load_3d(void* s, const CUtensorMap* m, uint64_t* b, int x, int y, int z) {
  model::load(s, m, b, x, y, z, 0);
}
inline void tma_load_4d(void* s, const CUtensorMap* m, uint64_t* b, int x, int y, int z, int u) {
  model::load(s, m, b, x, y, z, u);
}
inline void tmem_alloc(uint32_t* slot, uint32_t) {
  if (threadIdx.x % 32 == 0) *slot = 0;
}
inline void tmem_relinquish() {}
inline void tmem_dealloc(uint32_t, uint32_t) {}
inline uint64_t smem_desc_sw128(uint32_t addr, uint32_t lbo, uint32_t sbo) {
  return (uint64_t)((addr & 0x3FFFF) >> 4) | (uint64_t)((lbo >> 4) & 0x3FFF) << 16 | (uint64_t)((sbo >> 4) & 0x3FFF) << 32;
}
constexpr uint32_t idesc_bf16(int m, int n, bool a_mn, bool b_mn) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) |
         ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
inline void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, bool acc) { model::mma(d, a, false, b, id, acc); }
inline void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, bool acc) { model::mma(d, a, true, b, id, acc); }
inline void mma_commit(uint64_t* bar) { model::mma_commit(bar); }

// a warp reaches the 32 lanes of its quarter
inline uint32_t* tmem_words(uint32_t addr) {
  const uint32_t lanes = addr >> 16;
  if (lanes != 32 * (threadIdx.x / 32 % 4)) model::fail("tensor memory of another warp's lanes");
  return &model::tmem[lanes + threadIdx.x % 32][addr & 0xFFFF];
}
template <int N>
void tmem_ld(uint32_t addr, uint32_t (&r)[N]) {
  model::pause();
  memcpy(r, tmem_words(addr), sizeof r);
}
template <int N>
void tmem_st(uint32_t addr, const uint32_t (&r)[N]) {
  memcpy(tmem_words(addr), r, sizeof r);
  model::pause();
}
inline void tmem_ld16(uint32_t a, uint32_t (&r)[16]) { tmem_ld(a, r); }
inline void tmem_ld32(uint32_t a, uint32_t (&r)[32]) { tmem_ld(a, r); }
inline void tmem_st8(uint32_t a, const uint32_t (&r)[8]) { tmem_st(a, r); }
inline void tmem_st16(uint32_t a, const uint32_t (&r)[16]) { tmem_st(a, r); }
inline void tmem_st32(uint32_t a, const uint32_t (&r)[32]) { tmem_st(a, r); }
inline void tmem_st1(uint32_t a, uint32_t v) { tmem_st<1>(a, {v}); }
inline uint32_t tmem_ld1(uint32_t a) {
  uint32_t r[1];
  tmem_ld(a, r);
  return r[0];
}
inline void tmem_ld_wait() { model::pause(); }
inline void tmem_st_wait() { model::pause(); }
inline uint32_t pack_bf16(float lo, float hi) { return as<uint32_t>(__floats2bfloat162_rn(lo, hi)); }

}  // namespace ptx

namespace tcdev {

using namespace ptx;

constexpr float kLog2e = 1.4426950408889634f;

inline float ex2(float x) { return exp2f(x); }
inline float bf16_lo(uint32_t v) { return __uint_as_float(v << 16); }
inline float bf16_hi(uint32_t v) { return __uint_as_float(v & 0xFFFF0000u); }
inline void atomic_max_float(float* p, float v) { *p = std::max(*p, v); }
inline float2 fma2(float2 a, float2 b, float2 c) { return make_float2(fmaf(a.x, b.x, c.x), fmaf(a.y, b.y, c.y)); }
inline float2 add2(float2 a, float2 b) { return make_float2(a.x + b.x, a.y + b.y); }
inline float2 mul2(float2 a, float2 b) { return make_float2(a.x * b.x, a.y * b.y); }
inline void warp_arrive(uint64_t* bar, int lane) {
  __syncwarp();
  if (lane == 0) mbar_arrive(bar);
}
inline float keep_if_bit(float v, uint32_t mask, int k) { return (mask >> k) & 1 ? v : 0.f; }
inline float row_sumsq_sw128(const uint8_t* tile, int row) {
  float s = 0.f;
  for (int c = 0; c < 8; ++c) {
    uint32_t w[4];
    memcpy(w, tile + row * 128 + ((c ^ (row & 7)) << 4), sizeof w);
    for (uint32_t x : w) s = fmaf(bf16_hi(x), bf16_hi(x), fmaf(bf16_lo(x), bf16_lo(x), s));
  }
  return s;
}
inline void tma_store_3d(const CUtensorMap* m, const void* s, int x, int y, int z) { model::store(m, s, x, y, z, 0); }
inline void tma_store_4d(const CUtensorMap* m, const void* s, int x, int y, int z, int u) {
  model::store(m, s, x, y, z, u);
}
inline void tma_store_commit() { model::store_commit(); }
inline void tma_store_wait_read0() { model::store_wait(0); }
inline void tma_store_wait_read1() { model::store_wait(1); }
inline void tma_store_wait_all() { model::store_wait(0); }

}  // namespace tcdev

bool encode_tmap_bf16(CUtensorMap* map, const void* base, int rank, const uint64_t* dims, const uint64_t* strides_bytes,
                      const uint32_t* box);

}  // namespace sbl
