/* Clusters for the SIMT emulator: the CTAs of a cluster take turns, each running
 * its fibers (simt_runtime.cpp) until all of them wait, with the barrier and
 * shuffle state of its own swapped in. Shared memory beyond a CTA's own is
 * reached through shared_of(). */
#include "simt_emul.h"

namespace simt {
typedef void (*Body)(void *);

unsigned cluster_rank = 0;
static char *arena = nullptr;
static const size_t SHARED = 256 * 1024;
char *shared_of(unsigned rank) {
  if (arena == nullptr) arena = (char *)calloc(16, SHARED);
  return arena + rank * SHARED;
}

static unsigned long long arrived, phase_threads;
static unsigned long long *waits_for; /* per thread of the cluster: arrivals it waits for */
static unsigned per_cta;

void cluster_arrive() {
  const unsigned me = cluster_rank * per_cta + cur->linear;
  waits_for[me] += phase_threads;
  arrived++;
}
void cluster_wait() {
  const unsigned me = cluster_rank * per_cta + cur->linear;
  while (arrived < waits_for[me]) yield();
}

struct State {
  unsigned live, count, gen, wcount[64], wgen[64];
  unsigned long long slot[64][32];
};
static void take(const State &s) {
  live_threads = s.live;
  cta_count = s.count;
  cta_gen = s.gen;
  memcpy(warp_count, s.wcount, sizeof(s.wcount));
  memcpy(warp_gen, s.wgen, sizeof(s.wgen));
  memcpy(warp_slot, s.slot, sizeof(s.slot));
}
static void keep(State &s) {
  s.live = live_threads;
  s.count = cta_count;
  s.gen = cta_gen;
  memcpy(s.wcount, warp_count, sizeof(s.wcount));
  memcpy(s.wgen, warp_gen, sizeof(s.wgen));
  memcpy(s.slot, warp_slot, sizeof(s.slot));
}

static Body body_of;
static void *arg_of;
static void start() {
  body_of(arg_of);
  cur->done = 1;
  swapcontext(&cur->ctx, &sched);
}

void run_clusters(Body body, void *arg, simt_dim3 grid, simt_dim3 block, unsigned size) {
  const unsigned n = block.x * block.y * block.z, total = n * size;
  const size_t stack = 64 * 1024;
  Fiber *f = (Fiber *)calloc(total, sizeof(Fiber));
  State *st = (State *)calloc(size, sizeof(State));
  waits_for = (unsigned long long *)calloc(total, sizeof(*waits_for));
  for (unsigned t = 0; t < total; t++) f[t].stack = (char *)malloc(stack);
  body_of = body;
  arg_of = arg;
  grid_dim = grid;
  block_dim = block;
  per_cta = n;
  phase_threads = total;
  for (unsigned by = 0; by < grid.y; by++)
    for (unsigned b0 = 0; b0 < grid.x; b0 += size) {
      arrived = 0;
      memset(waits_for, 0, total * sizeof(*waits_for));
      memset(st, 0, size * sizeof(State));
      for (unsigned c = 0; c < size; c++) memset(shared_of(c), 0x5a, SHARED);
      for (unsigned t = 0; t < total; t++) {
        const unsigned l = t % n;
        st[t / n].live = n;
        f[t].done = 0;
        f[t].linear = l;
        f[t].tid = simt_dim3{l % block.x, (l / block.x) % block.y, l / (block.x * block.y)};
        getcontext(&f[t].ctx);
        f[t].ctx.uc_stack.ss_sp = f[t].stack;
        f[t].ctx.uc_stack.ss_size = stack;
        f[t].ctx.uc_link = &sched;
        makecontext(&f[t].ctx, start, 0);
      }
      unsigned left = total;
      while (left)
        for (unsigned c = 0; c < size; c++) {
          take(st[c]);
          cluster_rank = c;
          block_idx = simt_dim3{b0 + c, by, 0};
          for (unsigned t = c * n; t < (c + 1) * n; t++) {
            if (f[t].done) continue;
            cur = &f[t];
            swapcontext(&sched, &cur->ctx);
            if (f[t].done == 1) {
              f[t].done = 2;
              left--;
            }
          }
          keep(st[c]);
        }
    }
  cluster_rank = 0;
  for (unsigned t = 0; t < total; t++) free(f[t].stack);
  free(f);
  free(st);
  free(waits_for);
}
}  // namespace simt
