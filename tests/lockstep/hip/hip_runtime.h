// HIP's names on the CPU, for tests that follow a kernel's source thread by thread: as much as kernels without matrix products use.
//
// Every thread of a workgroup is a fiber of one host thread.  Lanes meet at the cross-lane operations of their wavefront, wavefronts at
// __syncthreads alone: between two of these one wavefront runs as far as it gets before the next one starts, in an order that the
// test gives.  What a kernel reads without a barrier behind another wavefront's write is then read wrongly every time.
#pragma once
#include <ucontext.h>

#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <functional>
#include <memory>
#include <vector>

#define __global__
#define __device__
#define __host__
#define __forceinline__ inline
#define __launch_bounds__(...)
#define __shared__ static

struct dim3 {
  uint32_t x = 1, y = 1, z = 1;
  dim3() = default;
  dim3(uint32_t x_, uint32_t y_ = 1, uint32_t z_ = 1) : x(x_), y(y_), z(z_) {}
};
struct uint2 { uint32_t x, y; };
struct uint4 { uint32_t x, y, z, w; };
struct float2 { float x, y; };
struct float4 { float x, y, z, w; };

namespace lockstep {

constexpr int kWave = 64, kStack = 64 << 10;
enum State { kReady, kLanes, kBarrier, kDone };

struct Fiber {
  ucontext_t at;
  std::unique_ptr<char[]> stack;
  State state = kReady;
  int value = 0;
};

struct Group {
  std::vector<Fiber> fibers;
  ucontext_t home;
  int now = 0;
  std::function<void()> body;
};

inline Group* group = nullptr;
inline int order = 0;                         // which wavefront starts: 0 the first, -1 the last and downwards, else rotated by it
inline dim3 thread_at, block_at, block_size, grid_size;

inline const char* error = nullptr;           // of the launches so far: the workgroup that it is found in ends there

inline void enter() {
  group->body();
  group->fibers[group->now].state = kDone;
  swapcontext(&group->fibers[group->now].at, &group->home);
}

inline void wait(State s) {
  Fiber& f = group->fibers[group->now];
  f.state = s;
  swapcontext(&f.at, &group->home);
}

[[noreturn]] inline void fail(const char* what) {
  error = what;
  for (;;) wait(kDone);
}

// One wavefront until it waits at a barrier or is done
inline void run_wave(int w, int threads) {
  const int first = w * kWave, end = first + kWave < threads ? first + kWave : threads;
  for (;;) {
    for (int i = first; i < end; ++i) {
      Fiber& f = group->fibers[i];
      if (f.state != kReady) continue;
      group->now = i;
      thread_at = dim3(i, 0, 0);
      swapcontext(&group->home, &f.at);
    }
    int lanes = 0, other = 0;
    for (int i = first; i < end; ++i) {
      lanes += group->fibers[i].state == kLanes;
      other += group->fibers[i].state != kLanes;
    }
    if (lanes && other) error = "lanes of a wavefront parted at a cross-lane operation";
    if (!lanes || error) return;
    for (int i = first; i < end; ++i) group->fibers[i].state = kReady;
  }
}

inline void run_block(int threads, std::function<void()> body) {
  Group g;
  g.fibers = std::vector<Fiber>(threads);
  g.body = std::move(body);
  group = &g;
  for (Fiber& f : g.fibers) {
    f.stack.reset(new char[kStack]);
    getcontext(&f.at);
    f.at.uc_stack.ss_sp = f.stack.get();
    f.at.uc_stack.ss_size = kStack;
    f.at.uc_link = nullptr;
    makecontext(&f.at, enter, 0);
  }
  const int waves = (threads + kWave - 1) / kWave;
  for (;;) {
    for (int w = 0; w < waves && !error; ++w) run_wave(order < 0 ? waves - 1 - w : (w + order) % waves, threads);
    int done = 0;
    for (Fiber& f : g.fibers) done += f.state == kDone;
    if (!error && done && done < threads) error = "a barrier that some threads have passed by";
    if (error || done == threads) break;
    for (Fiber& f : g.fibers) f.state = kReady;
  }
  group = nullptr;
}

template <class K, class... A>
void launch(K&& kernel, dim3 grid, dim3 block, A... args) {
  grid_size = grid;
  block_size = block;
  for (uint32_t y = 0; y < grid.y; ++y)
    for (uint32_t x = 0; x < grid.x && !error; ++x) {
      block_at = dim3(x, y);
      run_block(block.x, [&] { kernel(args...); });
    }
}

// Every lane's value to all of its wavefront: what lane `from` put there
inline int exchange(int x, int from) {
  const int base = group->now / kWave * kWave;
  group->fibers[group->now].value = x;
  wait(kLanes);
  const int y = group->fibers[base + from].value;
  wait(kLanes);
  return y;
}

}  // namespace lockstep

#define threadIdx lockstep::thread_at
#define blockIdx lockstep::block_at
#define blockDim lockstep::block_size
#define gridDim lockstep::grid_size

inline void __syncthreads() { lockstep::wait(lockstep::kBarrier); }
inline int __shfl_xor(int x, int o) { return lockstep::exchange(x, (lockstep::group->now % 64) ^ o); }
inline int __shfl_up(int x, int o) { const int l = lockstep::group->now % 64; return lockstep::exchange(x, l >= o ? l - o : l); }

// one fiber at a time
inline int atomicAdd(int* p, int v) { const int x = *p; *p = x + v; return x; }
inline int atomicSub(int* p, int v) { const int x = *p; *p = x - v; return x; }
inline int atomicOr(int* p, int v) { const int x = *p; *p = x | v; return x; }
inline int atomicMin(int* p, int v) { const int x = *p; *p = v < x ? v : x; return x; }

typedef void* hipStream_t;
typedef int hipError_t;
constexpr hipError_t hipSuccess = 0;
inline hipError_t hipGetLastError() { return hipSuccess; }
inline const char* hipGetErrorString(hipError_t) { return ""; }
#define hipLaunchKernelGGL(kernel, grid, block, lds, stream, ...) lockstep::launch(kernel, grid, block, __VA_ARGS__)

// named by helpers of the shared headers that no kernel followed here calls
inline uint32_t __float_as_uint(float x) { uint32_t y; memcpy(&y, &x, 4); return y; }
inline float __uint_as_float(uint32_t x) { float y; memcpy(&y, &x, 4); return y; }
inline uint64_t unused_on_the_cpu() { lockstep::fail("an operation that this header leaves out"); }
inline int __popcll(uint64_t x) { return __builtin_popcountll(x); }
#define __builtin_amdgcn_ballot_w64(x) ((void)(x), unused_on_the_cpu())
#define __builtin_amdgcn_readfirstlane(x) ((void)(x), static_cast<int>(unused_on_the_cpu()))
#define __builtin_amdgcn_sqrtf(x) sqrtf(x)
