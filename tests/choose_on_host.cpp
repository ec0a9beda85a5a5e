// choose_best of csrc/pfa_choose.h on the host: a fiber a lane, lanes of a wave
// held together at their exchanges, and the waves run one behind the other, in an
// order that the caller gives, each as far as its next barrier.  That is one of the
// orders that a GPU may take, and the one in which a wave that is ahead does most
// harm to what waves behind it have still to read.
#include <stdint.h>
#include <string.h>
#include <ucontext.h>

#include <vector>

#define __device__
#define __host__
#define __forceinline__ inline
#define __shared__ static

namespace {

struct Dim {
  unsigned x;
};
Dim threadIdx;

enum State { kReady, kLanes, kBarrier, kDone };
struct Fiber {
  ucontext_t at;
  State state;
  uint32_t out[2];  // what a lane gives to an exchange, this one's and the next's
  int turn;
};
std::vector<Fiber> fibers;
ucontext_t scheduler;
void (*body)();

void yield(State s) {
  Fiber& f = fibers[threadIdx.x];
  f.state = s;
  swapcontext(&f.at, &scheduler);
}
void enter() {
  body();
  fibers[threadIdx.x].state = kDone;
}
void __syncthreads() { yield(kBarrier); }
uint32_t exchange(uint32_t x, int from) {
  const int tid = threadIdx.x;
  const int turn = fibers[tid].turn ^= 1;
  fibers[tid].out[turn] = x;
  yield(kLanes);
  return fibers[(tid & ~63) + from].out[turn];
}
template <typename T>
T __shfl_xor(T x, int mask) {
  return (T)exchange((uint32_t)x, (threadIdx.x & 63) ^ mask);
}
template <typename T>
T __shfl_up(T x, int by) {
  const int lane = threadIdx.x & 63;
  return (T)exchange((uint32_t)x, lane < by ? lane : lane - by);
}
int __clz(int x) { return x ? __builtin_clz((unsigned)x) : 32; }
int atomicAdd(int* p, int x) {
  const int old = *p;
  *p += x;
  return old;
}

// One workgroup.  False where a wave ends, or waits for its lanes, while another
// waits at a barrier: on a GPU that would not end.
bool run(int threads, const int* order, void (*f)()) {
  body = f;
  fibers.assign(threads, Fiber{});
  const size_t size = 1 << 16;
  static std::vector<char> stacks;
  if (stacks.size() < size * threads) stacks.resize(size * threads);
  for (int t = 0; t < threads; ++t) {
    getcontext(&fibers[t].at);
    fibers[t].at.uc_stack.ss_sp = &stacks[size * t];
    fibers[t].at.uc_stack.ss_size = size;
    fibers[t].at.uc_link = &scheduler;
    makecontext(&fibers[t].at, enter, 0);
  }
  while (true) {
    int done = 0, barrier = 0;
    for (int i = 0; i < threads / 64; ++i) {
      const int t0 = order[i] * 64;
      while (true) {  // the wave, to its next barrier or its end
        int n[4] = {};
        for (int t = t0; t < t0 + 64; ++t) {
          if (fibers[t].state == kReady) {
            threadIdx.x = t;
            swapcontext(&scheduler, &fibers[t].at);
          }
          ++n[fibers[t].state];
        }
        if (n[kLanes] == 0 && (n[kBarrier] == 0 || n[kDone] == 0)) {
          done += n[kDone], barrier += n[kBarrier];
          break;
        }
        if (n[kLanes] != 64) return false;
        for (int t = t0; t < t0 + 64; ++t) fibers[t].state = kReady;
      }
    }
    if (done == threads) return true;
    if (barrier != threads) return false;
    for (auto& x : fibers) x.state = kReady;
  }
}

}  // namespace

namespace pfa {
constexpr int kWave = 64;
}
#include "choose.h"  // csrc/pfa_choose.h without its includes

namespace {

const uint32_t* keys;
int n_keys, count_;
int32_t* chosen;

template <int THREADS, int K, bool HELD>
void choose() {
  auto fetch = [&](int r, uint32_t(&x)[K]) {
    for (int i = 0; i < K; ++i) {
      const int p = (r * THREADS + (int)threadIdx.x) * K + i;
      x[i] = p < n_keys ? keys[p] : pfa::paged::kNone;
    }
  };
  pfa::paged::choose_best<THREADS, K, HELD>(0, HELD ? 1 : (n_keys + THREADS * K - 1) / (THREADS * K), count_, fetch,
                                            [&](int i, int entry) {
                                              if (i >= 0 && i < count_) chosen[i] = entry;
                                            });
}

}  // namespace

// The forms that the kernels use.  0: done; 1: the waves do not meet.
extern "C" int choose_on_host(int form, const uint32_t* k, int n, int count, const int* order, int32_t* out) {
  keys = k, n_keys = n, count_ = count, chosen = out;
  switch (form) {
    case 0: return !run(256, order, choose<256, 2, true>);
    case 1: return !run(256, order, choose<256, 4, true>);
    case 2: return !run(1024, order, choose<1024, 4, true>);
    case 3: return !run(1024, order, choose<1024, 8, true>);
    case 4: return !run(1024, order, choose<1024, 16, true>);
    default: return !run(1024, order, choose<1024, 16, false>);
  }
}
