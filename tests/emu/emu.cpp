// The emulated device: coroutines, checks of memory, and counts of stores.
#include "hip/hip_runtime.h"

#include <sanitizer/asan_interface.h>
#include <sanitizer/common_interface_defs.h>
#include <sys/mman.h>
#include <ucontext.h>
#include <unistd.h>
#include <string>
#include <vector>

dim3 threadIdx, blockIdx, blockDim, gridDim;

namespace emu {
namespace {
constexpr size_t kStack = 1 << 19;
enum State { kReady, kAtBarrier, kAtExchange, kEnded };
// A coroutine starts by setcontext, once; after that they switch by the builtins, which make no
// system call and are not intercepted.
struct Fiber {
  void* at[5];
  char* stack = nullptr;
  void* fake = nullptr;
  State state = kEnded;
  unsigned tid = 0;
};
std::vector<Fiber> fibers(1024);
void* scheduler[5];
void* scheduler_fake;
const void* scheduler_stack;
size_t scheduler_size;
Fiber* current;
const std::function<void()>* body;
std::string kernel;
uint64_t slots[16][2][64], live_lanes[16];
int side[16];
char* dynamic;
hipError_t last_error_ = hipSuccess;

__attribute__((noinline)) void jump(void** to) { __builtin_longjmp(to, 1); }
__attribute__((noinline)) void yield() {
  Fiber* f = current;
  __sanitizer_start_switch_fiber(&f->fake, scheduler_stack, scheduler_size);
  if (!__builtin_setjmp(f->at)) jump(scheduler);
  __sanitizer_finish_switch_fiber(current->fake, &scheduler_stack, &scheduler_size);
}
void entry() {
  __sanitizer_finish_switch_fiber(nullptr, &scheduler_stack, &scheduler_size);
  for (;;) {
    (*body)();
    current->state = kEnded;
    yield();
  }
}
void start(Fiber& f) {
  static ucontext_t ctx;
  getcontext(&ctx);
  ctx.uc_stack.ss_sp = f.stack;
  ctx.uc_stack.ss_size = kStack;
  ctx.uc_link = nullptr;
  makecontext(&ctx, entry, 0);
  setcontext(&ctx);
}
__attribute__((noinline)) void resume(Fiber& f) {
  current = &f;
  threadIdx = dim3(f.tid, 0, 0);
  f.state = kReady;
  const bool fresh = !f.stack;
  if (fresh)
    f.stack = (char*)mmap(nullptr, kStack, PROT_READ | PROT_WRITE, MAP_PRIVATE | MAP_ANONYMOUS | MAP_NORESERVE, -1, 0);
  __sanitizer_start_switch_fiber(&scheduler_fake, f.stack, kStack);
  if (!__builtin_setjmp(scheduler)) {
    if (fresh) start(f);
    jump(f.at);
  }
  __sanitizer_finish_switch_fiber(scheduler_fake, nullptr, nullptr);
}
void run_block(unsigned threads) {
  for (unsigned t = 0; t < threads; ++t) {
    fibers[t].tid = t;
    fibers[t].state = kReady;
  }
  const unsigned waves = (threads + 63) / 64;
  for (;;) {
    unsigned ended = 0, waiting = 0;
    for (unsigned w = 0; w < waves; ++w) {
      const unsigned t0 = w * 64, t1 = std::min(threads, t0 + 64);
      for (;;) {  // the wave's lanes up to a barrier or their end
        for (unsigned t = t0; t < t1; ++t)
          if (fibers[t].state == kReady) resume(fibers[t]);
        uint64_t live = 0;
        for (unsigned t = t0; t < t1; ++t)
          if (fibers[t].state == kAtExchange) live |= 1ull << (t - t0);
        if (!live) break;
        for (unsigned t = t0; t < t1; ++t)
          if (fibers[t].state == kAtBarrier) die("a lane waits at a barrier while others exchange values", w);
        live_lanes[w] = live;
        side[w] ^= 1;
        memset(slots[w][side[w]], 0, sizeof slots[w][0]);
        for (unsigned t = t0; t < t1; ++t)
          if (fibers[t].state == kAtExchange) fibers[t].state = kReady;
      }
      for (unsigned t = t0; t < t1; ++t) {
        ended += fibers[t].state == kEnded;
        waiting += fibers[t].state == kAtBarrier;
      }
    }
    if (ended == threads) return;
    if (ended + waiting != threads) die("a thread neither waits nor ended");
    for (unsigned t = 0; t < threads; ++t)
      if (fibers[t].state == kAtBarrier) fibers[t].state = kReady;
  }
}
struct Counted {
  const char* base;
  std::vector<uint8_t> n;
};
std::vector<Counted> counted;
}  // namespace

void die(const char* what, long long a, long long b) {
  printf("%s (%lld, %lld) in %s, block %u of %u, thread %u\n", what, a, b, kernel.c_str(), blockIdx.x, gridDim.x,
         threadIdx.x);
  fflush(stdout);
  _exit(3);
}
void barrier() {
  current->state = kAtBarrier;
  yield();
}
const uint64_t* exchange(uint64_t v, uint64_t* live) {
  const int w = current->tid / 64;
  slots[w][side[w] ^ 0][current->tid % 64] = v;
  // read after every live lane wrote: the scheduler flips the side, so the values stay
  const int mine = side[w];
  current->state = kAtExchange;
  yield();
  if (live) *live = live_lanes[w];
  return slots[w][mine];
}
void* dynamic_lds() { return dynamic; }
void touch(const void* p, size_t n, bool) {
  if (void* bad = __asan_region_is_poisoned(const_cast<void*>(p), n)) {
    printf("kernel %s, block %u, thread %u\n", kernel.c_str(), blockIdx.x, threadIdx.x);
    __asan_describe_address(bad);
    die("out of bounds", (long long)(intptr_t)bad, (long long)n);
  }
}
void run(const char* name, dim3 grid, dim3 block, size_t lds, const std::function<void()>& f) {
  kernel = name;
  if ((uint64_t)grid.x * block.x >= (1ull << 32) || !grid.x || !grid.y || grid.y > 65535 || block.x > 1024) {
    last_error_ = hipErrorInvalidConfiguration;
    return;
  }
  body = &f;
  gridDim = grid;
  blockDim = block;
  for (unsigned y = 0; y < grid.y; ++y)
    for (unsigned x = 0; x < grid.x; ++x) {
      blockIdx = dim3(x, y, 0);
      dynamic = (char*)malloc(lds ? lds : 1);
      run_block(block.x);
      free(dynamic);
    }
}
void count_stores(const void* base, size_t bytes) { counted.push_back({(const char*)base, std::vector<uint8_t>(bytes / 16)}); }
const std::vector<uint8_t>& stores_of(const void* base) {
  for (auto& c : counted)
    if (c.base == base) return c.n;
  die("not counted");
}
void forget_counts() { counted.clear(); }
void count_store(const void* p) {
  for (auto& c : counted) {
    const size_t i = ((const char*)p - c.base) / 16;
    if ((const char*)p >= c.base && i < c.n.size()) c.n[i] += c.n[i] < 255;
  }
}
}  // namespace emu
hipError_t hipGetLastError() {
  const hipError_t e = emu::last_error_;
  emu::last_error_ = hipSuccess;
  return e;
}
