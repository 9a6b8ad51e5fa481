// Replays the loading and the issuing lane of the dv kernel (sbl_bwd_walk.cuh) on the host, over models of the barriers
// and the products, and checks that every product waited for what it reads and overwrites.
//
// A barrier is the number of phases that its lane knows to be complete.  Waiting for a parity tells of the next phase, or
// of nothing new; asking (mbar_test) may tell of it as soon as it can be complete, by a coin.  A phase can be complete
// when whatever the other roles wait for has been committed.
#include <algorithm>
#include <cstdio>
#include <cstdint>
#include <cstdlib>
#include <random>
#include <string>
#include <vector>

#define __device__
#define __forceinline__ inline
using std::max;
using std::min;
template <typename T>
T __ldg(const T* p) { return *p; }
struct { unsigned x; } blockIdx, gridDim;
struct float2 { float x, y; };
struct __nv_bfloat16 { uint16_t v; };
struct CUtensorMap { int id; };

namespace model {
constexpr int BARS = 64, NONE = 1 << 30;
uint64_t bars[BARS];
int known[BARS], commits[BARS];
int (*possible)(int bar);           // phases that can be complete
std::mt19937 rng;
double eager;                       // how often a question about a complete phase is answered yes
std::string fault;
void fail(const std::string& what) {
  if (fault.empty()) fault = what;
}
int index(uint64_t* bar) { return (int)(bar - bars); }
int can(int b) {
  const int p = possible(b);
  if (p != NONE && p > known[b] + 1) fail("barrier " + std::to_string(b) + " ran ahead: parities cannot be told apart");
  return p;
}
struct Product { char kind; int buf; };
std::vector<Product> open;          // products since the last commit of a piece
void product(char kind, int buf, bool accumulate);
void committed(int bar);
struct Load { int map; int bar; };
void loaded(const Load& l);
}  // namespace model

namespace sbl {
namespace {
namespace ptx {
constexpr uint32_t idesc_bf16(int m, int n, bool, bool) { return (uint32_t)(n << 17 | m << 4) & ~(1u << 13); }
inline void tc_fence_after_sync() {}
inline void mbar_expect_tx(uint64_t*, uint32_t) {}
inline void tma_load_3d(void*, const CUtensorMap* m, uint64_t* bar, int, int, int) { model::loaded({m->id, model::index(bar)}); }
inline void tma_load_4d(void*, const CUtensorMap* m, uint64_t* bar, int, int, int, int) {
  model::loaded({m->id, model::index(bar)});
}
inline void mma_commit(uint64_t* bar) { model::committed(model::index(bar)); }
void mma_ss(uint32_t d, uint64_t, uint64_t, uint32_t idesc, bool accumulate);
void mma_ts(uint32_t d, uint32_t a, uint64_t, uint32_t, bool accumulate);
}  // namespace ptx
}  // namespace
}  // namespace sbl

#include "sbl_bwd_walk.cuh"

namespace sbl {
namespace {
bool mbar_test(uint64_t* bar, uint32_t parity) {
  const int b = model::index(bar), p = model::can(b);
  if (parity != (uint32_t)(model::known[b] & 1)) return true;       // complete before
  if (p <= model::known[b] || std::uniform_real_distribution<>()(model::rng) >= model::eager) return false;
  ++model::known[b];
  return true;
}
void wait_inline(uint64_t* bar, uint32_t parity, int*, int code) {
  const int b = model::index(bar), p = model::can(b);
  if (parity != (uint32_t)(model::known[b] & 1)) return;
  if (p <= model::known[b]) model::fail("wait " + std::to_string(code) + " never ends");
  ++model::known[b];
}
namespace ptx {
constexpr uint32_t kDv = 384;
void mma_ss(uint32_t d, uint64_t, uint64_t, uint32_t idesc, bool accumulate) {
  if (d >= kDv) model::product('r', (int)(d - kDv) / 64, accumulate);
  else model::product(idesc & (1u << 13) ? 'm' : 's', (int)d / 128, accumulate);
}
void mma_ts(uint32_t d, uint32_t a, uint64_t, uint32_t, bool accumulate) {
  if (d < kDv) model::fail("value product outside dv");
  if (!accumulate) model::product('0', (int)(d - kDv) / 64, false);
  model::product('v', (int)a / 128, accumulate);
}
}  // namespace ptx

enum { K, Q, DO, PHI, PSI, SUM };
const char* kKinds = "_sv_mr";        // the product that takes a piece of each map

template <int D>
struct Replay {
  using C = ValCfg<D>;
  static std::string order;         // of the ring pieces: kinds of the products they are for
  static size_t taken;
  static int pieces, values[3];

  static int of(int first, int n, int b) { return b >= first && b < first + n ? b - first : -1; }
  static int issuer_possible(int b) {
    int i;
    if ((i = of(C::E_DONE, 3, b)) >= 0) return model::commits[C::S_FULL + i];
    if ((i = of(C::D_DONE, 3, b)) >= 0) return model::commits[C::P_FULL + i];
    if (b == C::DV_FREE) return model::commits[C::DV_FULL];
    return model::NONE;               // loads: the loader runs as far ahead as it may
  }
  static int loader_possible(int) { return model::NONE; }

  static std::string run(const Geom& g, double eager) {
    ValArgs a{};
    a.g = g;
    a.tm_k.id = K; a.tm_q.id = Q; a.tm_do.id = DO; a.tm_phi.id = PHI; a.tm_psi.id = PSI; a.tm_sum.id = SUM;
    model::fault.clear();
    model::eager = eager;
    auto reset = [] {
      std::fill(model::known, model::known + model::BARS, 0);
      std::fill(model::commits, model::commits + model::BARS, 0);
    };
    reset();
    order.clear();
    pieces = 0;
    model::possible = loader_possible;
    ValLoader<D> l{a, nullptr, model::bars};
    walk_values(a.g, l);
    reset();
    taken = 0;
    values[0] = values[1] = values[2] = 0;
    model::open.clear();
    model::possible = issuer_possible;
    ValIssuer<D> v{a, model::bars, 0, 0, 0, 0};
    walk_values(a.g, v);
    if (taken != order.size()) model::fail("pieces loaded and not used");
    int tiles = 0;
    for (int t = blockIdx.x; t < g.ntiles; t += gridDim.x) ++tiles;
    if (model::commits[C::DV_FULL] != tiles) model::fail("tiles without dv");
    for (int b = 0; b < 3; ++b)
      if (values[b] != model::commits[C::P_FULL + b] * C::NB * 8) model::fail("steps without their value product");
    return model::fault;
  }
  static void loaded(const model::Load& l) {
    if (l.map == K || l.map == PHI) return;
    const int slot = pieces % C::NS;
    if (l.bar != C::R_FULL + slot) model::fail("a piece in the wrong place");
    if (model::known[C::R_FREE + slot] != pieces / C::NS) model::fail("a piece over one in use");
    order += kKinds[l.map];
    ++pieces;
  }
  static void product(char kind, int buf, bool accumulate) {
    const int *known = model::known, *commits = model::commits;
    if (kind == 's' && !accumulate && values[buf] != commits[C::S_FULL + buf] * C::NB * 8)
      model::fail("a score over a step in use");
    if (kind == 'm' && known[C::E_DONE + buf] != commits[C::S_FULL + buf]) model::fail("a difference before its weights");
    if (kind == 'v' && known[C::D_DONE + buf] != commits[C::P_FULL + buf])
      model::fail("a value product that did not wait for its step");
    if ((kind == '0' || (kind == 'r' && !accumulate)) && known[C::DV_FREE] != commits[C::DV_FULL])
      model::fail("dv over a tile that has not been read");
    if (kind == 'v') ++values[buf];
    if (kind != '0') model::open.push_back({kind, buf});
  }
  static void committed(int b) {
    ++model::commits[b];
    const int slot = of(C::R_FREE, C::NS, b);
    if (slot < 0) return;
    // one piece: products of one kind, out of the place that is next
    if (slot != (int)(taken % C::NS)) model::fail("pieces out of order");
    if (model::known[C::R_FULL + slot] != (int)(taken / C::NS) + 1) model::fail("a piece used before it landed");
    for (const auto& p : model::open)
      if (taken >= order.size() || p.kind != order[taken]) model::fail("a piece meant for another product");
    model::open.clear();
    ++taken;
  }
};
template <int D> std::string Replay<D>::order;
template <int D> size_t Replay<D>::taken;
template <int D> int Replay<D>::pieces;
template <int D> int Replay<D>::values[3];

int g_dim;
}  // namespace
}  // namespace sbl

void model::product(char kind, int buf, bool acc) {
  sbl::g_dim == 64 ? sbl::Replay<64>::product(kind, buf, acc) : sbl::Replay<128>::product(kind, buf, acc);
}
void model::committed(int b) { sbl::g_dim == 64 ? sbl::Replay<64>::committed(b) : sbl::Replay<128>::committed(b); }
void model::loaded(const Load& l) { sbl::g_dim == 64 ? sbl::Replay<64>::loaded(l) : sbl::Replay<128>::loaded(l); }

// value_walk CTAS B H T S W [lengths...]: one problem; value_walk random N: small ones
int main(int argc, char** argv) {
  using namespace sbl;
  int bad = 0, lanes = 0;
  auto problem = [&](int ctas, int B, int H, int T, int S, int w, const std::vector<int64_t>& lengths) {
    Geom g{};
    g.lengths = lengths.empty() ? nullptr : lengths.data();
    g.H = H; g.T = T; g.S = S;
    g.w = (int)min<int64_t>(w, 2 * (int64_t)max(T, S) + 2);
    g.ntr = (S + TR - 1) / TR;
    g.ntiles = g.ntr * B * H;
    g.by_ntr = divisor(g.ntr);
    g.by_h = divisor(H);
    gridDim.x = min(ctas, g.ntiles);
    for (g_dim = 64; g_dim <= 128; g_dim += 64)
      for (double eager : {1.0, 0.0, 0.5})
        for (blockIdx.x = 0; blockIdx.x < gridDim.x; ++blockIdx.x, ++lanes) {
          const std::string f = g_dim == 64 ? Replay<64>::run(g, eager) : Replay<128>::run(g, eager);
          if (!f.empty() && bad++ < 5)
            printf("d %d CTA %u of %u, B %d H %d T %d S %d w %d, eager %.1f: %s\n", g_dim, blockIdx.x, gridDim.x, B, H, T, S,
                   w, eager, f.c_str());
        }
  };
  if (argc > 2 && std::string(argv[1]) == "random") {
    std::mt19937 rng(7);
    auto pick = [&](int lo, int hi) { return (int)(lo + rng() % (unsigned)(hi - lo + 1)); };
    for (int i = 0; i < atoi(argv[2]); ++i) {
      const int B = pick(1, 12), H = pick(1, 3), T = pick(1, 400), S = pick(1, 900), w = pick(1, pick(1, 500));
      std::vector<int64_t> lengths;
      if (pick(0, 3)) for (int b = 0; b < B; ++b) lengths.push_back(pick(0, 2) ? pick(0, S) : 0);
      problem(pick(1, 4), B, H, T, S, w, lengths);
    }
  } else if (argc >= 7) {
    const int B = atoi(argv[2]);
    std::vector<int64_t> given, lengths;
    for (int i = 7; i < argc; ++i) given.push_back(atoi(argv[i]));
    for (int b = 0; b < B && !given.empty(); ++b) lengths.push_back(given[b % given.size()]);
    problem(atoi(argv[1]), B, atoi(argv[3]), atoi(argv[4]), atoi(argv[5]), atoi(argv[6]), lengths);
  }
  printf("%d of %d lanes at fault\n", bad, lanes);
  return bad || !lanes;
}
