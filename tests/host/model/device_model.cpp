// Models of what runs beside a block's warps, and the random schedule over all of them.
//
// Threads are fibers.  A step of the schedule runs one warp until its lanes are put aside, or one item of an engine: the
// next product of a thread's queue (products and commits of one thread in order, those of different threads in any), a
// bulk load (in any order), the next bulk store of a thread.  Every warp and engine gets a random speed per block, over
// three orders of magnitude, so that each of them runs far ahead of, or far behind, the others in some schedule.
//
// Loads take their bytes when they are issued and write them when they complete; products read both memories when they
// are run; stores read shared memory when they are run.  Whatever a missing wait lets happen too early or too late
// therefore ends in the results, which must not depend on the schedule.  Both memories start as not-a-numbers.
#include "device_model.h"

#include <deque>
#include <map>
#include <random>
#include <vector>

// Saves the callee-saved registers on this stack and goes on with another one (x86-64).
extern "C" void switch_stack(void** from, void* to);
asm(R"(
.text
.globl switch_stack
switch_stack:
  pushq %rbp
  pushq %rbx
  pushq %r12
  pushq %r13
  pushq %r14
  pushq %r15
  movq %rsp, (%rdi)
  movq %rsi, %rsp
  popq %r15
  popq %r14
  popq %r13
  popq %r12
  popq %rbx
  popq %rbp
  ret
)");

namespace model {

struct TensorMap {                    // what encode_tmap_bf16 leaves in a CUtensorMap
  uint8_t* base;
  int rank;
  uint64_t dims[4], strides[3];
  uint32_t box[4];
};
static_assert(sizeof(TensorMap) <= sizeof(CUtensorMap), "");

Index block_index, grid_size, block_size;
uint8_t* smem;
uint32_t tmem[128][512];
int sms = 1;

namespace {

struct Barrier {
  uint32_t count = 0, pending = 0, phase = 0;
  int64_t bytes = 0;
  void settle() {
    if (pending == 0 && bytes == 0 && count > 0) {
      ++phase;
      pending = count;
    }
  }
  void arrive() {
    if (pending == 0) fail("more arrivals than a barrier expects");
    --pending;
    settle();
  }
  bool passed(uint32_t parity) const { return (phase & 1) != parity; }
};
struct Warp;
struct Store {
  TensorMap map;
  const uint8_t* src;
  int at[4], group;
};
enum State { RUNS, PARKED, AT_MBARRIER, AT_BARRIER, AT_STORES, ENDED };
struct Thread {
  void* sp;
  Index id;
  State state = RUNS;
  Warp* warp;
  Barrier* bar = nullptr;             // waited for, with this parity; the wait's code
  uint32_t parity = 0;
  int code = 0;
  Op op = SYNC;                       // collective: what, and its operands
  uint64_t value = 0, result = 0;
  int arg = 0;
  int barrier = 0;
  std::deque<Store> stores;
  int groups = 0, allowed = 0;        // store groups committed; how many may be pending where the thread waits
  int pending_groups() const { return stores.empty() ? 0 : groups - stores.front().group; }
};
struct Warp {
  Thread* lanes[32];
  int parked = 0;
  double speed;
};
struct Product {
  Barrier* commit;                    // null: a product
  uint32_t d;
  uint64_t a;
  bool a_in_tmem;
  uint64_t b;
  uint32_t idesc;
  bool accumulate;
};
struct Load {
  uint8_t* dst;
  std::vector<uint8_t> bytes;
  Barrier* bar;
};
struct Queue {
  std::deque<Product> items;
  double speed;
};

constexpr size_t kStack = 96 << 10, kThreads = 1024, kSmem = 400 << 10;
std::mt19937 rng;
std::vector<Thread> threads;
std::vector<Warp> warps;
std::map<uint64_t*, Barrier> barriers;
std::map<Thread*, Queue> queues;
std::vector<Load> loads;
std::map<int, int> at_barrier;
std::function<void()> body;
Thread* current;
void* scheduler_sp;
double load_speed, store_speed, pause_rate;

double uniform() { return std::uniform_real_distribution<>()(rng); }
double any_speed() { return std::pow(10.0, -3 * uniform()); }
void put_aside() {
  Thread* t = current;
  switch_stack(&t->sp, scheduler_sp);
}
void enter() {
  body();
  current->state = ENDED;
  put_aside();
  abort();
}
void resume(Thread* t) {
  current = t;
  switch_stack(&scheduler_sp, t->sp);
}

template <typename F>
void each_chunk(const TensorMap& m, const int (&at)[4], F&& f) {   // f(offset in the tile, place in memory or null)
  for (int r = 0; r < (int)m.box[1]; ++r)
    for (int q = 0; q < 8; ++q) {
      const int64_t c[4] = {at[0] + 8 * q, at[1] + r, at[2], at[3]};
      bool inside = c[0] >= 0 && c[0] + 8 <= (int64_t)m.dims[0];
      int64_t offset = 2 * c[0];
      for (int i = 1; i < m.rank; ++i) {
        inside = inside && c[i] >= 0 && c[i] < (int64_t)m.dims[i];
        offset += c[i] * (int64_t)m.strides[i - 1];
      }
      f(r * 128 + ((q ^ (r & 7)) << 4), inside ? m.base + offset : nullptr);
    }
}

// rows x 16 of an operand in shared memory, as its descriptor says
void gather(float* out, uint64_t desc, bool mn_major, int rows) {
  const uint32_t start = (uint32_t)(desc & 0x3FFF) << 4, lbo = (uint32_t)(desc >> 16 & 0x3FFF) << 4,
                 sbo = (uint32_t)(desc >> 32 & 0x3FFF) << 4;
  for (int r = 0; r < rows; ++r)
    for (int k = 0; k < 16; ++k) {
      uint32_t at = mn_major ? start + r / 64 * lbo + k / 8 * sbo + k % 8 * 128 + r % 64 * 2
                             : start + r / 8 * sbo + r % 8 * 128 + k * 2;
      at ^= (at >> 7 & 7) << 4;
      uint16_t h;
      memcpy(&h, smem + at, 2);
      out[r * 16 + k] = __uint_as_float((uint32_t)h << 16);
    }
}
void run(const Product& p) {
  const int n = (int)(p.idesc >> 17 & 63) * 8;
  const float sign = p.idesc >> 13 & 1 ? -1.f : 1.f;
  static float a[128 * 16], b[256 * 16], bt[16 * 256], sum[256];
  if (p.a_in_tmem) {
    for (int r = 0; r < 128; ++r)
      for (int k = 0; k < 16; ++k) {
        const uint32_t w = tmem[r][(uint32_t)p.a + k / 2];
        a[r * 16 + k] = __uint_as_float(k & 1 ? w & 0xFFFF0000u : w << 16);
      }
  } else {
    gather(a, p.a, p.idesc >> 15 & 1, 128);
  }
  gather(b, p.b, p.idesc >> 16 & 1, n);
  for (int j = 0; j < n; ++j)
    for (int k = 0; k < 16; ++k) bt[k * n + j] = b[j * 16 + k];
  for (int r = 0; r < 128; ++r) {
    std::fill(sum, sum + n, 0.f);
    for (int k = 0; k < 16; ++k) {
      const float x = sign * a[r * 16 + k];
      for (int j = 0; j < n; ++j) sum[j] += x * bt[k * n + j];
    }
    for (int j = 0; j < n; ++j) {
      uint32_t& d = tmem[r][p.d + j];
      d = __float_as_uint((p.accumulate ? __uint_as_float(d) : 0.f) + sum[j]);
    }
  }
}
void next_product(Queue& q) {
  const Product p = q.items.front();
  q.items.pop_front();
  if (p.commit) p.commit->arrive();
  else run(p);
}
void any_load() {
  const size_t i = rng() % loads.size();
  Load l = std::move(loads[i]);
  loads[i] = std::move(loads.back());
  loads.pop_back();
  memcpy(l.dst, l.bytes.data(), l.bytes.size());
  l.bar->bytes -= (int64_t)l.bytes.size();
  l.bar->settle();
}
void next_store(Thread& t) {
  const Store s = t.stores.front();
  t.stores.pop_front();
  each_chunk(s.map, s.at, [&](int offset, uint8_t* to) {
    if (to) memcpy(to, s.src + offset, 16);
  });
}

void start_threads() {
  static uint8_t* stacks = static_cast<uint8_t*>(aligned_alloc(4096, kStack * kThreads));
  const unsigned n = block_size.x * block_size.y;
  threads.assign(n, Thread{});
  warps.assign(n / 32, Warp{});
  barriers.clear();
  queues.clear();
  loads.clear();
  at_barrier.clear();
  for (unsigned i = 0; i < n; ++i) {
    Thread& t = threads[i];
    t.id = {i % block_size.x, i / block_size.x, 0};
    t.warp = &warps[i / 32];
    t.warp->lanes[i % 32] = &t;
    void** sp = reinterpret_cast<void**>(stacks + kStack * (i + 1) - 64);
    *--sp = nullptr;
    *--sp = reinterpret_cast<void*>(&enter);
    for (int k = 0; k < 6; ++k) *--sp = nullptr;
    t.sp = sp;
  }
  for (auto& w : warps) w.speed = any_speed();
  load_speed = 3 * any_speed();
  store_speed = any_speed();
  pause_rate = uniform() < 0.3 ? 0 : 0.3 * uniform() * uniform();
}

void run_block() {
  start_threads();
  struct Choice {
    double speed;
    Warp* warp;
    Queue* queue;
  };
  std::vector<Choice> choices;
  std::vector<Thread*> storing;
  for (;;) {
    choices.clear();
    storing.clear();
    bool alive = false;
    for (auto& w : warps) {
      bool ready = false;
      for (Thread* t : w.lanes) {
        if ((t->state == AT_MBARRIER && t->bar->passed(t->parity)) ||
            (t->state == AT_STORES && t->pending_groups() <= t->allowed))
          t->state = RUNS;
        ready |= t->state == RUNS;
        alive |= t->state != ENDED;
      }
      if (ready) choices.push_back({w.speed, &w, nullptr});
    }
    for (auto& q : queues)
      if (!q.second.items.empty()) choices.push_back({q.second.speed, nullptr, &q.second});
    for (auto& t : threads)
      if (!t.stores.empty()) storing.push_back(&t);
    double total = (loads.empty() ? 0 : load_speed) + (storing.empty() ? 0 : store_speed);
    for (const auto& c : choices) total += c.speed;
    if (total == 0 && !alive) return;
    if (total == 0) {
      std::string s = "nothing can go on; waits by warp:";
      for (const auto& w : warps) s += " " + std::to_string(w.lanes[0]->code);
      fail(s.c_str());
    }
    double x = uniform() * total;
    const Choice* chosen = nullptr;
    for (const auto& c : choices)
      if ((x -= c.speed) < 0) {
        chosen = &c;
        break;
      }
    if (chosen && chosen->warp) {
      for (Thread* t : chosen->warp->lanes)
        if (t->state == RUNS) resume(t);
    } else if (chosen) {
      next_product(*chosen->queue);
    } else if (!loads.empty() && ((x -= load_speed) < 0 || storing.empty())) {
      any_load();
    } else if (!storing.empty()) {
      next_store(*storing[rng() % storing.size()]);
    }
  }
}

}  // namespace

void fail(const char* what) {
  printf("FAULT in block %u: %s\n", block_index.x, what);
  fflush(stdout);
  exit(3);
}
void seed(unsigned s) { rng.seed(s); }
Index& thread_index() { return current->id; }
void pause() {
  if (uniform() < pause_rate) put_aside();
}

void launch(dim3 grid, dim3 block, size_t, std::function<void()> kernel) {
  static std::vector<uint8_t> memory(kSmem);
  body = std::move(kernel);
  grid_size = {grid.x, grid.y, grid.z};
  block_size = {block.x, block.y, block.z};
  smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(memory.data()) + 1023) & ~(uintptr_t)1023);
  Index& b = block_index;
  for (b.z = 0; b.z < grid.z; ++b.z)
    for (b.y = 0; b.y < grid.y; ++b.y)
      for (b.x = 0; b.x < grid.x; ++b.x) {
        std::fill(memory.begin(), memory.end(), 0xff);
        memset(tmem, 0xff, sizeof tmem);
        run_block();
      }
}

void barrier_sync(int id, int count) {
  if (++at_barrier[id] == count) {
    at_barrier[id] = 0;
    for (auto& t : threads)
      if (t.state == AT_BARRIER && t.barrier == id) t.state = RUNS;
    return;
  }
  current->state = AT_BARRIER;
  current->barrier = id;
  put_aside();
}

// All 32 lanes of a warp meet.  A wait for an mbarrier is one too, since a warp comes together behind its loop; but
// lanes may wait while the others are parked at the next __syncwarp (an elected lane that runs a loop of its own).
uint64_t collective(Op op, uint64_t value, int arg) {
  Thread* t = current;
  Warp* w = t->warp;
  t->op = op;
  t->value = value;
  t->arg = arg;
  t->state = PARKED;
  if (++w->parked < 32) {
    put_aside();
    return t->result;
  }
  bool waits = false, same = true;
  for (Thread* x : w->lanes) {
    waits |= x->op == WAIT;
    same &= x->op == op;
  }
  if (waits) {
    for (Thread* x : w->lanes) {
      if (x->op == WAIT) {
        x->state = x->bar->passed(x->parity) ? RUNS : AT_MBARRIER;
        --w->parked;
      } else if (x->op != SYNC) {
        fail("a collective of some lanes only");
      }
    }
  } else {
    if (!same) fail("different collectives in one warp");
    w->parked = 0;
    uint64_t any = 0, all = 1, values[32];
    for (int i = 0; i < 32; ++i) {
      values[i] = w->lanes[i]->value;
      any |= values[i];
      all &= values[i];
    }
    for (int i = 0; i < 32; ++i) {
      Thread* x = w->lanes[i];
      x->state = RUNS;
      x->result = op == ANY ? any : op == ALL ? all : op == XOR ? values[i ^ x->arg] : op == FROM ? values[x->arg & 31] : 0;
    }
  }
  if (t->state != RUNS) put_aside();
  return t->result;
}

void mbar_init(uint64_t* bar, uint32_t count) {
  Barrier b;
  b.count = b.pending = count;
  barriers[bar] = b;
}
void mbar_arrive(uint64_t* bar) {
  barriers[bar].arrive();
  pause();
}
void mbar_expect_tx(uint64_t* bar, uint32_t bytes) {
  barriers[bar].bytes += bytes;
  barriers[bar].arrive();
  pause();
}
bool mbar_test(uint64_t* bar, uint32_t parity) {
  pause();
  return barriers[bar].passed(parity);
}
void mbar_wait(uint64_t* bar, uint32_t parity, int code) {
  pause();
  current->bar = &barriers[bar];
  current->parity = parity;
  current->code = code;
  collective(WAIT, 0, 0);
}

void load(void* dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z, int u) {
  TensorMap m;
  memcpy(&m, map, sizeof m);
  if (x % 8 != 0) fail("a tile that begins off a 16-byte boundary");
  if (sbl::ptx::smem_u32(dst) % 1024 != 0) fail("a swizzled tile off a 1024-byte boundary");
  Load l{static_cast<uint8_t*>(dst), std::vector<uint8_t>(m.box[1] * 128, 0), &barriers[bar]};
  each_chunk(m, {x, y, z, u}, [&](int offset, uint8_t* from) {
    if (from) memcpy(&l.bytes[offset], from, 16);
  });
  loads.push_back(std::move(l));
  pause();
}
void load_bytes(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  const uint8_t* s = static_cast<const uint8_t*>(src);
  if (reinterpret_cast<uintptr_t>(s) % 16 != 0 || bytes % 16 != 0) fail("a bulk copy off a 16-byte boundary");
  loads.push_back({static_cast<uint8_t*>(dst), std::vector<uint8_t>(s, s + bytes), &barriers[bar]});
  pause();
}
void store(const CUtensorMap* map, const void* src, int x, int y, int z, int u) {
  Store s{{}, static_cast<const uint8_t*>(src), {x, y, z, u}, current->groups};
  memcpy(&s.map, map, sizeof s.map);
  current->stores.push_back(s);
  pause();
}
void store_commit() { ++current->groups; }
void store_wait(int groups) {
  current->allowed = groups;
  if (current->pending_groups() > groups) {
    current->state = AT_STORES;
    put_aside();
  }
}

static Queue& own_queue() {
  const auto at = queues.find(current);
  if (at != queues.end()) return at->second;
  return queues[current] = {{}, 3 * any_speed()};
}
void mma(uint32_t d, uint64_t a, bool a_in_tmem, uint64_t b, uint32_t idesc, bool accumulate) {
  own_queue().items.push_back({nullptr, d, a, a_in_tmem, b, idesc, accumulate});
  pause();
}
void mma_commit(uint64_t* bar) {
  own_queue().items.push_back({&barriers[bar], 0, 0, false, 0, 0, false});
  pause();
}

}  // namespace model

namespace sbl {

bool encode_tmap_bf16(CUtensorMap* map, const void* base, int rank, const uint64_t* dims, const uint64_t* strides,
                      const uint32_t* box) {
  model::TensorMap m{};
  m.base = static_cast<uint8_t*>(const_cast<void*>(base));
  m.rank = rank;
  for (int i = 0; i < rank; ++i) {
    m.dims[i] = dims[i];
    m.box[i] = box[i];
    if (i > 0) m.strides[i - 1] = strides[i - 1];
  }
  if (box[0] != 64) return false;
  memset(map, 0, sizeof *map);
  memcpy(map, &m, sizeof m);
  return true;
}

}  // namespace sbl
