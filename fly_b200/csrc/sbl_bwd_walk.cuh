// What the roles of the gradient kernels agree on without exchanging it: the
// column steps of a row tile, and the order of the dv kernel's loads and
// products with what its loading and its issuing lane wait for.  The including
// file defines the two waits declared here; a host test brings models of them
// and of the PTX wrappers and replays both lanes.
#pragma once

#include <cstdint>

namespace sbl {
namespace {

using namespace ptx;

__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity);
__device__ __forceinline__ void wait_inline(uint64_t* bar, uint32_t parity, int* status, int code);

enum { QUERIES = 0, KEYS = 1 };
constexpr int TR = 128;        // rows of a tile

// n / d for n < 2^31 without a division: floor(n * ceil(2^p / d) / 2^p), p = 31 + ceil(log2 d)
struct Divisor {
  uint32_t mul;
  int p;
};
inline Divisor divisor(int d) {
  if (d < 1) d = 1;               // (no tiles: nobody asks)
  Divisor v{0, 31};
  while ((int64_t)1 << (v.p - 31) < d) ++v.p;
  v.mul = (uint32_t)((((uint64_t)1 << v.p) + d - 1) / d);
  return v;
}
__device__ __forceinline__ int quotient(int n, const Divisor& d) { return (int)(((uint64_t)(uint32_t)n * d.mul) >> d.p); }

struct Geom {
  const int64_t* lengths;
  int H, T, S, w, ntr, ntiles;   // ntr: row tiles per (b,h)
  Divisor by_ntr, by_h;
};
struct RowTile {
  int bh, b, h, r0, nr, len, c0, n;   // n column steps from c0 on
};

// The column steps of width STEP (a power of two) that a row tile meets; all real columns with `whole`.  In line and
// without divisions: every role of a kernel asks for every tile, and behind a call (with the parameters read through
// a pointer, two divisions and the answer in local memory) each answer took 1.2 to 1.6 k cycles of a tile's 18 to 22 k.
template <int SIDE, int STEP>
__device__ __forceinline__ RowTile row_tile(const Geom& g, int tile, bool whole) {
  RowTile t;
  t.bh = quotient(tile, g.by_ntr);
  t.r0 = (tile - t.bh * g.ntr) * TR;
  t.b = quotient(t.bh, g.by_h);
  t.h = t.bh - t.b * g.H;
  t.len = g.S;
  if (g.lengths) {
    const int64_t l = __ldg(g.lengths + t.b);
    t.len = l < 0 ? 0 : (l < g.S ? (int)l : g.S);
  }
  const int hw = g.w / 2;
  int lo, hi;
  if (SIDE == QUERIES) {
    t.nr = min(TR, g.T - t.r0);
    lo = t.r0 - hw;
    hi = t.r0 + t.nr - 1 - hw + g.w - 1;
    if (whole) { lo = 0; hi = t.len; }
    hi = min(hi, t.len - 1);
  } else {
    t.nr = min(TR, g.S - t.r0);
    lo = t.r0 + hw - g.w + 1;
    hi = t.r0 + t.nr - 1 + hw;
    if (whole) { lo = 0; hi = g.T; }
    hi = t.r0 < t.len ? min(hi, g.T - 1) : -1;
  }
  lo = max(lo, 0);
  t.c0 = lo & ~(STEP - 1);
  t.n = hi >= lo ? (hi - t.c0) / STEP + 1 : 0;
  return t;
}

// The issuing lane asks for a barrier before it issues the products that come before the wait (`seen`), and waits only
// where the answer was no.  A wait in front of a group of four products costs 30 cycles on an idle SM and 150 to 230
// beside busy warps, in which the tensor core runs dry; asked ahead, by one lane that runs the whole loop, it costs
// none (64.4 cycles per N = 128 product, its full rate; 72 to 124 with the wait in place).
__device__ __forceinline__ void wait_unless(bool seen, uint64_t* bar, uint32_t parity, int* status, int code) {
  if (!seen) wait_inline(bar, parity, status, code);
}

// start-address steps (in 16-byte units) of K step k inside a K-major operand of [rows][64] pieces
__device__ __forceinline__ uint64_t kmajor(int k, uint32_t piece_bytes) {
  return (uint64_t)((uint32_t)(k >> 2) * (piece_bytes >> 4) + (uint32_t)(k & 3) * 2);
}
// tensor-memory column of K step k of a packed operand that lies over the first half of every 32 columns
__device__ __forceinline__ uint32_t packed(int k) { return 32u * (uint32_t)(k >> 1) + 8u * (uint32_t)(k & 1); }

// ---------------------------------------------------------------------------
// dv.
struct ValArgs {
  CUtensorMap tm_k, tm_q, tm_do, tm_phi, tm_psi, tm_sum;
  Geom g;
  const float2* nd;                        // (BH, Tp)
  __nv_bfloat16* dv; int64_t vb, vs, vh;
  int* status;
  int Tp;
  float tau;
};

template <int D>
struct ValCfg {
  static constexpr int NB = D / 64, M = 4 * D, KBUF = D == 64 ? 2 : 1, NS = 4;
  static constexpr uint32_t KB = NB * 16384, FB = (M / 64) * 16384;
  static constexpr uint32_t OFF_K = 0, OFF_F = KBUF * KB, OFF_RING = OFF_F + KBUF * FB, OFF_BAR = OFF_RING + NS * 16384;
  static constexpr uint32_t SMEM = OFF_BAR + 512 + 1024;
  static constexpr int NTHR = 576, W_LOAD = 16, W_MMA = 17;
  static constexpr uint32_t T_DV = 384;    // buffers at 128 b, b < 3
  enum { K_FULL = 0, K_FREE = 2, F_FULL = 4, F_FREE = 6, R_FULL = 8, R_FREE = R_FULL + NS, S_FULL = R_FREE + NS,
         E_DONE = S_FULL + 3, P_FULL = E_DONE + 3, D_DONE = P_FULL + 3, DV_FULL = D_DONE + 3, DV_FREE, COUNT };
  static_assert(SMEM <= 232448 && COUNT <= 60, "shared memory of one CTA");
};

// S = K Q^T -> p (exponential group, in place) -> p - phi psi^T (accumulated onto p) -> bf16 (packing group, in place)
// -> dv += (p - a) dO; then dv += phi summary.
//
// Bound: one lane issues and one loads, in 16-KB pieces of four or eight products: 25 pieces and 14.5 k cycles a tile
// at head dim 64 and w = 256, of which the products take 5.4 k and the stream into shared memory 10.4 k.  Two issuing
// warps with a ring and a loader of their own each took 264 us for 226, because that leaves room for one phi tile
// instead of two (head dim 128: 395 for 325); log-normalisers through shared memory instead of __ldg cost a fifth:
// its whole bandwidth goes to products with both operands there (8 KB in 64 cycles at N = 128).
//
// The order in which the tensor core consumes what the producer loads; both walk it.  Column steps (128 queries) are
// numbered g = 0, 1, .. over the CTA's tiles and use buffer g % 3.  The visitor's calls:
//   score(tile t, first, ke, g)   S of step g; t is where it belongs, ke the number of that tile among those with steps
//   begin(t, it), minus(t, it, s, g, pending), value(t, it, s, g, first, last), rank(t, it, first, alone)
// `pending`: the value product of step g - 1 comes next.  A tile without steps has that product issued before the next
// tile begins, and the one behind the following step's difference is then the step's own.
template <typename V>
__device__ __forceinline__ void walk_values(const Geom& g, V& v) {
  const int stride = gridDim.x;
  int sc_tile = blockIdx.x, sc_s = 0, sc_g = 0, sc_ke = 0;
  RowTile sc{};
  auto seek = [&]() {
    sc.n = 0;
    while (sc_tile < g.ntiles) {
      sc = row_tile<KEYS, 128>(g, sc_tile, false);
      if (sc.n > 0) break;
      sc_tile += stride;
    }
    sc_s = 0;
  };
  auto score = [&]() {
    if (sc_tile >= g.ntiles) return;
    v.score(sc, sc_s, sc_ke, sc_g);
    ++sc_g;
    if (++sc_s == sc.n) {
      sc_tile += stride;
      ++sc_ke;
      seek();
    }
  };
  seek();
  score();
  score();
  int n = 0;                        // steps so far
  RowTile pend{};                   // tile and step of the value product that is still to come
  int pend_s = -1;
  int it = 0;
  for (int tile = blockIdx.x; tile < g.ntiles; tile += stride, ++it) {
    const RowTile t = row_tile<KEYS, 128>(g, tile, false);
    v.begin(t, it);
    bool fresh = true;              // nothing of this tile is in dv yet
    for (int s = 0; s < t.n; ++s, ++n) {
      v.minus(t, it, s, n, pend_s >= 0);
      if (pend_s >= 0) {
        const bool own = s > 0;
        v.value(pend, own ? it : it - 1, pend_s, n - 1, own && fresh, pend_s == pend.n - 1);
        if (own) fresh = false;
      }
      score();
      pend = t;
      pend_s = s;
    }
    if (t.n == 0 && pend_s >= 0) {
      v.value(pend, it - 1, pend_s, n - 1, false, true);
      pend_s = -1;
    }
    v.rank(t, it, fresh, t.n == 0);
    if (t.n == 0) pend_s = -1;
  }
  if (pend_s >= 0) v.value(pend, it - 1, pend_s, n - 1, false, true);
}

template <int D>
struct ValLoader {
  using C = ValCfg<D>;
  const ValArgs& a;
  uint8_t* smem;
  uint64_t* bars;
  int n = 0, loaded = 0;           // ring pieces, phi tiles
  bool seen = true;                // the next piece's place is free

  __device__ uint8_t* piece() {
    const int slot = n % C::NS;
    wait_unless(seen, bars + C::R_FREE + slot, ((n / C::NS) - 1) & 1, a.status, 281);
    mbar_expect_tx(bars + C::R_FULL + slot, 16384);
    return smem + C::OFF_RING + slot * 16384;
  }
  __device__ uint64_t* full() {
    uint64_t* bar = bars + C::R_FULL + (n++ % C::NS);
    seen = n < C::NS || mbar_test(bars + C::R_FREE + n % C::NS, ((n / C::NS) - 1) & 1);
    return bar;
  }
  __device__ void phi(const RowTile& t, int it) {
    const int buf = it % C::KBUF;
    if (it >= C::KBUF) wait_inline(bars + C::F_FREE + buf, ((it / C::KBUF) - 1) & 1, a.status, 282);
    mbar_expect_tx(bars + C::F_FULL + buf, C::FB);
    for (int j = 0; j < C::M / 64; ++j)
      tma_load_3d(smem + C::OFF_F + buf * C::FB + j * 16384, &a.tm_phi, bars + C::F_FULL + buf, 64 * j, t.r0, t.bh);
    loaded = it + 1;
  }
  __device__ void score(const RowTile& t, int s, int ke, int) {
    if (s == 0) {
      const int buf = ke % C::KBUF;
      if (ke >= C::KBUF) wait_inline(bars + C::K_FREE + buf, ((ke / C::KBUF) - 1) & 1, a.status, 283);
      mbar_expect_tx(bars + C::K_FULL + buf, C::KB);
      for (int j = 0; j < C::NB; ++j)
        tma_load_4d(smem + C::OFF_K + buf * C::KB + j * 16384, &a.tm_k, bars + C::K_FULL + buf, 64 * j, t.r0, t.h, t.b);
    }
    for (int j = 0; j < C::NB; ++j) {
      uint8_t* dst = piece();
      uint64_t* bar = full();
      tma_load_4d(dst, &a.tm_q, bar, 64 * j, t.c0 + 128 * s, t.h, t.b);
    }
  }
  __device__ void begin(const RowTile& t, int it) {
    if (loaded <= it) phi(t, it);
  }
  __device__ void minus(const RowTile& t, int it, int s, int, bool) {
    for (int j = 0; j < C::M / 64; ++j) {
      uint8_t* dst = piece();
      uint64_t* bar = full();
      tma_load_3d(dst, &a.tm_psi, bar, 64 * j, t.c0 + 128 * s, t.bh);
    }
    // two phi buffers: the next tile's features come in behind this tile's first step (the previous tile's last
    // product with its buffer was issued before this tile began)
    if (C::KBUF == 2 && s == 0) {
      const int tile = blockIdx.x + (it + 1) * (int)gridDim.x;
      if (tile < a.g.ntiles) phi(row_tile<KEYS, 128>(a.g, tile, false), it + 1);
    }
  }
  __device__ void value(const RowTile& t, int, int s, int, bool, bool) {
    for (int j = 0; j < C::NB; ++j) {
      uint8_t* dst = piece();
      uint64_t* bar = full();
      tma_load_4d(dst, &a.tm_do, bar, 64 * j, t.c0 + 128 * s, t.h, t.b);
    }
  }
  __device__ void rank(const RowTile& t, int, bool, bool) {
    for (int f = 0; f < C::M / 128; ++f)
      for (int j = 0; j < C::NB; ++j) {
        uint8_t* dst = piece();
        uint64_t* bar = full();
        tma_load_3d(dst, &a.tm_sum, bar, 64 * j, 128 * f, t.bh);
      }
  }
};

template <int D>
struct ValIssuer {
  using C = ValCfg<D>;
  const ValArgs& a;
  uint64_t* bars;
  uint64_t dK, dF, dR, dRt;
  int n = 0, m = 0;                // ring pieces, differences
  bool r_seen = false, e_seen = false, d_seen = false;

  __device__ int take() {          // the next ring piece, landed
    const int slot = n % C::NS;
    wait_unless(r_seen, bars + C::R_FULL + slot, (n / C::NS) & 1, a.status, 284);
    ++n;
    r_seen = mbar_test(bars + C::R_FULL + n % C::NS, (n / C::NS) & 1);
    return slot;
  }
  __device__ void score(const RowTile& t, int s, int ke, int g) {
    const int kb = ke % C::KBUF;
    if (s == 0) wait_inline(bars + C::K_FULL + kb, (ke / C::KBUF) & 1, a.status, 285);
    constexpr uint32_t id = idesc_bf16(128, 128, false, false);
#pragma unroll
    for (int j = 0; j < C::NB; ++j) {
      const int slot = take();
      if (j == C::NB - 1) e_seen = mbar_test(bars + C::E_DONE + m % 3, (m / 3) & 1);
      tc_fence_after_sync();
#pragma unroll
      for (int k = 0; k < 4; ++k)
        mma_ss(128 * (g % 3), dK + (uint64_t)(kb * (C::KB >> 4) + j * 1024 + 2 * k), dR + (uint64_t)(slot * 1024 + 2 * k), id,
               j > 0 || k > 0);
      mma_commit(bars + C::R_FREE + slot);
    }
    mma_commit(bars + C::S_FULL + g % 3);
    if (s == t.n - 1) mma_commit(bars + C::K_FREE + kb);
  }
  __device__ void begin(const RowTile&, int it) {
    wait_inline(bars + C::F_FULL + it % C::KBUF, (it / C::KBUF) & 1, a.status, 286);
  }
  __device__ void minus(const RowTile&, int it, int, int g, bool pending) {
    wait_unless(e_seen, bars + C::E_DONE + g % 3, (g / 3) & 1, a.status, 287);
    m = g + 1;
    e_seen = false;
    constexpr uint32_t id = idesc_bf16(128, 128, false, false) | (1u << 13);   // bit 13 negates A
    const int fb = it % C::KBUF;
#pragma unroll
    for (int j = 0; j < C::M / 64; ++j) {
      const int slot = take();
      // (asked about the step whose product takes the answer: kept for another one it would hide that one's wait)
      if (j == C::M / 64 - 1 && pending) d_seen = mbar_test(bars + C::D_DONE + (g - 1) % 3, ((g - 1) / 3) & 1);
      tc_fence_after_sync();
#pragma unroll
      for (int k = 0; k < 4; ++k)
        mma_ss(128 * (g % 3), dF + (uint64_t)(fb * (C::FB >> 4) + j * 1024 + 2 * k), dR + (uint64_t)(slot * 1024 + 2 * k), id,
               true);
      mma_commit(bars + C::R_FREE + slot);
    }
    mma_commit(bars + C::P_FULL + g % 3);
  }
  __device__ void value(const RowTile&, int it, int, int g, bool first, bool last) {
    wait_unless(d_seen, bars + C::D_DONE + g % 3, (g / 3) & 1, a.status, 288);
    d_seen = false;
    if (first && it >= 1) wait_inline(bars + C::DV_FREE, (it - 1) & 1, a.status, 289);
    constexpr uint32_t id = idesc_bf16(128, 64, false, true);
#pragma unroll
    for (int j = 0; j < C::NB; ++j) {
      const int slot = take();
      tc_fence_after_sync();
#pragma unroll
      for (int k = 0; k < 8; ++k)
        mma_ts(C::T_DV + 64 * j, 128 * (g % 3) + packed(k), dRt + (uint64_t)(slot * 1024 + k * 128), id, !first || k > 0);
      mma_commit(bars + C::R_FREE + slot);
    }
    if (last) mma_commit(bars + C::DV_FULL);
  }
  __device__ void rank(const RowTile&, int it, bool first, bool alone) {
    if (first && it >= 1) wait_inline(bars + C::DV_FREE, (it - 1) & 1, a.status, 290);
    constexpr uint32_t id = idesc_bf16(128, 64, false, true);
    const int fb = it % C::KBUF;
    for (int f = 0; f < C::M / 128; ++f)
#pragma unroll
      for (int j = 0; j < C::NB; ++j) {
        const int slot = take();
        tc_fence_after_sync();
#pragma unroll
        for (int k = 0; k < 8; ++k)
          mma_ss(C::T_DV + 64 * j, dF + (uint64_t)(fb * (C::FB >> 4) + 2 * f * 1024) + kmajor(k, 16384),
                 dRt + (uint64_t)(slot * 1024 + k * 128), id, !first || f > 0 || k > 0);
        mma_commit(bars + C::R_FREE + slot);
      }
    mma_commit(bars + C::F_FREE + fb);
    if (alone) mma_commit(bars + C::DV_FULL);
  }
};

}  // namespace
}  // namespace sbl
