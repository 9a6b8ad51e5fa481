// Replays the phi(K) producer of the head-dim-64 band kernel (sbl_band_walk.cuh) on the host over models of the barriers
// and checks that no slot is filled while a product that reads it may still run.
//
// Before key tile g is loaded the producer has seen S(g - 1) issued, which waited for the value product of g - 3: the P
// products up to g - 3 are done, those of g - 2 and g - 1 may or may not be.  A wait returns if the phase before the
// current one has the asked parity; otherwise the products behind it finish one by one until it does.
#include <algorithm>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <random>
#include <string>
#include <vector>

#define __device__
#define __noinline__
#define __forceinline__ inline
using std::max;
using std::min;
struct CUtensorMap { int id; };

namespace model {
constexpr int BARS = 64;
uint64_t bars[BARS];
std::vector<int> slots;            // slot of the P product of key tile g, in order
int done;                          // products 0 .. done - 1 are complete
int phases(int bar);               // complete phases of a barrier
std::string fault;
void fail(const std::string& s) {
  if (fault.empty()) fault = s;
}
}  // namespace model

namespace sbl {
namespace {
namespace ptx {
inline bool mbar_wait(uint64_t* bar, uint32_t parity, int*, int code) {
  const int b = (int)(bar - model::bars);
  while ((uint32_t)(model::phases(b) & 1) == parity) {
    if (model::done == (int)model::slots.size()) {
      model::fail("wait " + std::to_string(code) + " never ends");
      break;
    }
    ++model::done;
  }
  return true;
}
}  // namespace ptx
}  // namespace
}  // namespace sbl

#include "sbl_band_walk.cuh"

using namespace sbl;

int model::phases(int bar) {
  int n = 0;
  for (int g = 0; g < done; ++g) n += bar == band::B_PFULL + (g & 1);
  return n;
}

std::string replay(const BandArgs& a, int ctas, int cta, int mode, std::mt19937& rng) {
  const int lo = (int)((int64_t)a.ntiles * cta / ctas), n_it = (int)((int64_t)a.ntiles * (cta + 1) / ctas) - lo;
  model::fault.clear();
  model::slots.clear();
  model::done = 0;
  PkTrack pk;
  TileCursor cur(a, lo);
  int g = 0;
  for (int it = 0; it < n_it; ++it, cur.next(a)) {
    const BandTile T = band_tile(a, cur);
    for (int t = 0; t < T.nt; ++t, ++g) {
      const int kt = T.j0 / band::KT + t, slot = kt & 1;
      // at least the products up to g - 3, at most all
      const int least = max(0, g - 2), more = mode == 0 ? 0 : mode == 1 ? 2 : (int)(rng() % 3);
      model::done = max(model::done, min(g, least + more));
      if (pk_claim(pk, slot, T.bh, kt, g, model::bars, nullptr))
        for (int u = model::done; u < g; ++u)
          if (model::slots[u] == slot)
            model::fail("key tile " + std::to_string(g) + " over the one that product " + std::to_string(u) + " reads");
      model::slots.push_back(slot);
    }
  }
  return model::fault;
}

// band_walk CTAS B H T S W [lengths...]: one problem; band_walk random N: small ones
int main(int argc, char** argv) {
  int bad = 0, runs = 0;
  std::mt19937 rng(11);
  auto problem = [&](int ctas, int B, int H, int T, int S, int w, const std::vector<int64_t>& lengths) {
    BandArgs a{};
    a.p.B = B; a.p.H = H; a.p.T = T; a.p.S = S; a.p.w = w; a.p.S_total = S;
    a.p.key_lengths = lengths.empty() ? nullptr : lengths.data();
    a.ntq = (T + band::BQ - 1) / band::BQ;
    a.ntiles = a.ntq * B * H;
    ctas = min(ctas, a.ntiles);
    for (int mode = 0; mode < 3; ++mode)
      for (int cta = 0; cta < ctas; ++cta, ++runs) {
        const std::string f = replay(a, ctas, cta, mode, rng);
        if (!f.empty() && bad++ < 5)
          printf("CTA %d of %d, B %d H %d T %d S %d w %d: %s\n", cta, ctas, B, H, T, S, w, f.c_str());
      }
  };
  if (argc > 2 && std::string(argv[1]) == "random") {
    auto pick = [&](int lo, int hi) { return (int)(lo + rng() % (unsigned)(hi - lo + 1)); };
    for (int i = 0; i < atoi(argv[2]); ++i) {
      const int B = pick(1, 12), H = pick(1, 3), T = pick(1, 900), S = pick(1, pick(1, 900)), w = pick(1, pick(1, 900));
      std::vector<int64_t> lengths;
      if (pick(0, 2)) for (int b = 0; b < B; ++b) lengths.push_back(pick(0, 2) ? pick(1, S) : 0);
      problem(pick(1, 6), B, H, T, S, w, lengths);
    }
  } else if (argc >= 7) {
    const int B = atoi(argv[2]);
    std::vector<int64_t> given, lengths;
    for (int i = 7; i < argc; ++i) given.push_back(atoi(argv[i]));
    for (int b = 0; b < B && !given.empty(); ++b) lengths.push_back(given[b % given.size()]);
    problem(atoi(argv[1]), B, atoi(argv[3]), atoi(argv[4]), atoi(argv[5]), atoi(argv[6]), lengths);
  }
  printf("%d of %d runs at fault\n", bad, runs);
  return bad || !runs;
}
