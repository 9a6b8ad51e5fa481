// What the roles of the head-dim-64 band kernel agree on without exchanging it:
// its barriers, the key tiles of a query tile, and which phi(K) tile lies in
// which shared-memory slot, with what its producer waits for.  A host test
// brings models of the PTX wrappers and replays the producer.
#pragma once

#include "sblocal_b200.h"

namespace sbl {
namespace {

using namespace ptx;

struct BandArgs {
  CUtensorMap tm_q, tm_k, tm_v, tm_w, tm_phik, tm_kv, tm_out;
  SblParams p;
  const float* beta;
  const float* ksum;     // (BH, 256) fp32, reference feature order
  const float* wmax;     // [1]: max_f |sqrt(tau) w_f| of the bf16 projection
  int* status;
  float* row_stats;      // (2,BH,T): query + key log-scale and normaliser of every row, for the gradients; or null
  int ntq;               // query tiles per (b,h)
  int ntiles;            // ntq * B * H
};

namespace band {
constexpr int BQ = 128, KT = 128;
constexpr int NSOFT = 512;                 // softmax threads: two groups of 256, warp w owns rows 32*(w%4)..
constexpr int WSOFT = NSOFT / 32;          // softmax warps
constexpr int WGRP = WSOFT / 2;            // warps per softmax group (exponential group, packing group)
constexpr int W_LOADKV = WSOFT;            // producer: K, V, phi(K) tiles; output stores
constexpr int W_LOADQ = WSOFT + 1;         // producer: Q tiles, halves of Wt, halves of KV
constexpr int W_MMA_A = WSOFT + 2;         // MMA issuer: U halves, S
constexpr int W_MMA_B = WSOFT + 3;         // MMA issuer: P
constexpr int W_MMA_C = WSOFT + 4;         // MMA issuer: low-rank, O
constexpr int NTHREADS = NSOFT + 160;
constexpr uint32_t OFF_Q = 0;              // 2 x 16 KB [128 q][64 e]: current and next query tile
constexpr uint32_t OFF_W = 32768;          // 8 KB [64 r][64 e]: one half of Wt at a time
constexpr uint32_t OFF_KVH = 40960;        // 16 KB [128 f][64 d]: one feature half of KV at a time
constexpr uint32_t OFF_K = 57344;          // 16 KB [128 keys][64 e]
constexpr uint32_t OFF_V = OFF_K + 16384;  // 16 KB [128 keys][64 d]; also the staging buffer of the output tile
constexpr uint32_t OFF_PK = OFF_V + 16384; // 2 x 64 KB: phi(K) tiles, each 4 blocks [128 keys][64 f]
constexpr uint32_t OFF_MISC = OFF_PK + 2 * 65536;    // ksum fp32[256] + (L, Z) exchange fp32[2][2][256] + sum D fp32[2][256]
constexpr uint32_t OFF_BAR = OFF_MISC + 1024 + 12 * NSOFT;
constexpr uint32_t SMEM_BYTES = OFF_BAR + 512 + 1024;
static_assert(SMEM_BYTES <= 232448, "dynamic shared memory of one CTA");
// tensor memory columns (512): three 64-column feature-half slots, two 128-column S/E/D buffers, O
__device__ __forceinline__ constexpr uint32_t hq_col(int slot) { return slot == 0 ? 0u : (slot == 1 ? 64u : 384u); }
constexpr uint32_t T_BUF = 128;    // 2 x 128: S of a key tile, then E, then D = E - P (fp32), then D packed bf16 in place
constexpr uint32_t T_O = 448;      // 64
// barrier indices
enum {
  B_QFULL = 0,                    // [2] Q tile landed                                   (by query tile parity)
  B_QFREE = B_QFULL + 2,          // [2] Q buffer reusable: last MMA reading it + one arrival per softmax warp
  B_WFULL = B_QFREE + 2,          // half of Wt landed                                   (per load)
  B_WFREE,                        // U half computed: the Wt buffer is reusable
  B_KVFULL,                       // half of KV landed                                   (per load)
  B_KVFREE,                       // low-rank product done with it
  B_UQFULL,                       // [3] U half computed into the slot
  B_PHIFULL = B_UQFULL + 3,       // [3] features formed in the slot (one arrival per softmax warp)
  B_HQFREE = B_PHIFULL + 3,       // [3] slot reusable: issuer A (low-rank) and issuer B (last P) both done
  B_KFULL = B_HQFREE + 3, B_KEMPTY, B_VFULL, B_VEMPTY,   // per key tile, single buffers
  B_PKFULL,                                              // [2] phi(K) tile landed in the slot
  B_SFULL = B_PKFULL + 2,         // [2] by buffer
  B_ADONE = B_SFULL + 2,          // [2] one arrival per softmax warp
  B_PFULL = B_ADONE + 2,          // [2]
  B_BDONE = B_PFULL + 2,          // [2] one arrival per softmax warp
  B_BUFFREE = B_BDONE + 2,        // [2] O += D V done: the buffer may take the next S
  B_OFREE = B_BUFFREE + 2,        // O read by the epilogue (one arrival per softmax warp)
  B_DONE,                         // all MMAs of the query tile done
  B_OFULL,                        // output tile staged in shared memory (one arrival per softmax warp)
  B_OSTORED,                      // the bulk store of the staged tile has read the staging buffer
  B_LZFULL,                       // [2] L and Z of a query tile published by the exponential group (by tile parity)
  B_XFREE = B_LZFULL + 2,         // [2] ... and read by the packing group
  B_COUNT = B_XFREE + 2
};
static_assert(B_COUNT <= 60, "barriers and the tensor-memory slot share 512 bytes");
}  // namespace band

// Geometry of one 128-query tile: which key tiles it visits.
struct BandTile {
  int bh, b, h, i0, nq, len_b, j0, nt;
};
// A CTA walks consecutive tiles: (b*h, query tile) advance without dividing by the tile count.
struct TileCursor {
  int bh, qt;
  __device__ TileCursor(const BandArgs& a, int tile_id) : bh(tile_id / a.ntq), qt(tile_id % a.ntq) {}
  __device__ void next(const BandArgs& a) {
    if (++qt == a.ntq) {
      qt = 0;
      ++bh;
    }
  }
};
// Not inlined: every warp role needs it once per tile, and the kernel's instruction footprint is what limits it.
__device__ __noinline__ BandTile band_tile(const BandArgs& a, const TileCursor& c) {
  const SblParams& p = a.p;
  BandTile t;
  t.bh = c.bh;
  t.b = t.bh / p.H;
  t.h = t.bh - t.b * p.H;
  t.i0 = c.qt * band::BQ;
  t.nq = min(band::BQ, p.T - t.i0);
  t.len_b = (int)(p.key_lengths ? min(p.key_lengths[t.b], p.S_total) : p.S_total);
  const int hw = p.w / 2;
  // key buffer rows any query of this tile can see, clipped to the buffer and to the key length
  int lo = (int)(p.q_pos0 + t.i0 - hw - p.k_pos0);
  int hi = (int)(p.q_pos0 + t.i0 + t.nq - 1 - hw + p.w - 1 - p.k_pos0);
  lo = max(lo, 0);
  hi = min(hi, min(p.S - 1, t.len_b - 1 - (int)p.k_pos0));
  t.j0 = (lo / band::KT) * band::KT;
  t.nt = hi >= lo ? (hi - t.j0) / band::KT + 1 : 0;
  return t;
}

// Which phi(K) tile each of the two shared-memory slots holds.  Key tile kt of a (b,h) lives in slot
// kt & 1; consecutive query tiles of a run share two of their three key tiles, so only the new one is
// loaded.  The producer and the P-issuing warp walk the same sequence and keep identical copies.
struct PkTrack {
  int bh0 = -1, bh1 = -1, kt0 = -1, kt1 = -1;
  int fills0 = 0, fills1 = 0;   // completed or pending loads per slot
  int last0 = -1, last1 = -1;   // number of the latest key tile whose P product reads the slot
  __device__ bool resident(int slot, int b, int k) const {
    return slot ? (bh1 == b && kt1 == k) : (bh0 == b && kt0 == k);
  }
  __device__ int fills(int slot) const { return slot ? fills1 : fills0; }
  __device__ int last(int slot) const { return slot ? last1 : last0; }
  __device__ void filled(int slot, int b, int k) {
    if (slot) { bh1 = b; kt1 = k; ++fills1; } else { bh0 = b; kt0 = k; ++fills0; }
  }
  __device__ void used(int slot, int g) {
    if (slot) last1 = g; else last0 = g;
  }
};

// Slot of key tile number g, tile kt of (b,h): true if it has to be filled, after waiting until no product reads what it
// holds.  P products run in order, and those up to g - 3 are done: the K tile before this one has been freed by S(g - 1),
// which was issued behind the value product of g - 3.  So there is something to wait for only where the slot's latest
// product is that of g - 2 or g - 1, and then its own barrier tells: the one before it on that barrier is done, the one
// behind it needs this key tile.  (A barrier per slot does not: two products that follow one another on a slot, key tiles
// of query tiles with one each, are two phases, and waiting for the second passes while the first is still running.)
__device__ __forceinline__ bool pk_claim(PkTrack& pk, int slot, int bh, int kt, int g, uint64_t* bars, int* status) {
  const bool fill = !pk.resident(slot, bh, kt);
  if (fill) {
    const int last = pk.last(slot);
    if (last >= 0 && last >= g - 2) mbar_wait(bars + band::B_PFULL + (last & 1), (last >> 1) & 1, status, 22);
    pk.filled(slot, bh, kt);
  }
  pk.used(slot, g);
  return fill;
}

}  // namespace
}  // namespace sbl
