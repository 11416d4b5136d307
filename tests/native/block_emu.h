// block_emu.h — a block of 256 threads (four waves of 64) on the host, for device
// code of integers: every thread is a fibre, and what goes between lanes waits
// for the wave's others. Between two of a block's barriers the waves run in the
// order asked for, each as far as it gets, so code that lacks a barrier meets
// every order of its waves' reads and writes.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>
#include <ucontext.h>

#include <algorithm>
#include <functional>
#include <vector>

namespace emu {

constexpr int kThreads = 256, kLanes = 64, kWaves = kThreads / kLanes;

struct Thread {
  ucontext_t at;
  std::vector<char> stack = std::vector<char>(64 << 10);
  bool done;
  uint64_t exchanges, barriers;  // entered
};
struct Block {
  Thread threads[kThreads];
  ucontext_t main;
  int now;
  uint64_t words[kWaves][2][kLanes];  // of exchanges in turn: none is written before all have read the one two before
  int arrived[kWaves], waiting;
  uint64_t exchanged[kWaves], passed;  // complete
  const std::function<void()>* body;
};
inline Block block;
inline dim3 thread, block_id;

inline void pause() { swapcontext(&block.threads[block.now].at, &block.main); }

// Every lane's word.
inline const uint64_t* exchange(uint64_t word) {
  const int w = block.now / kLanes;
  Thread& t = block.threads[block.now];
  uint64_t* const words = block.words[w][t.exchanges & 1];
  words[block.now % kLanes] = word;
  ++t.exchanges;
  if (++block.arrived[w] == kLanes) block.arrived[w] = 0, ++block.exchanged[w];
  if (block.exchanged[w] < t.exchanges) pause();
  return words;
}
inline void barrier() {
  Thread& t = block.threads[block.now];
  ++t.barriers;
  ++block.waiting;
  pause();
}
inline void enter() {
  (*block.body)();
  block.threads[block.now].done = true;
  pause();
}
inline bool runs(int i) {
  const Thread& t = block.threads[i];
  return !t.done && t.exchanges <= block.exchanged[i / kLanes] && t.barriers <= block.passed;
}

// Runs body in every thread; waves: which goes first of those that can. False:
// some wait for others for ever, or passed another number of barriers.
inline bool run(const int (&waves)[kWaves], const std::function<void()>& body) {
  block.body = &body;
  block.waiting = 0;
  block.passed = 0;
  for (int w = 0; w < kWaves; ++w) block.arrived[w] = 0, block.exchanged[w] = 0;
  for (Thread& t : block.threads) {
    t.done = false;
    t.exchanges = t.barriers = 0;
    getcontext(&t.at);
    t.at.uc_stack.ss_sp = t.stack.data();
    t.at.uc_stack.ss_size = t.stack.size();
    t.at.uc_link = nullptr;
    makecontext(&t.at, enter, 0);
  }
  for (;;) {
    bool any = false;
    for (int w : waves) {
      for (int i = w * kLanes; i < (w + 1) * kLanes; ++i) {
        if (!runs(i)) continue;
        any = true;
        block.now = i;
        thread.x = i;
        swapcontext(&block.main, &block.threads[i].at);
      }
      if (any) break;
    }
    if (any) continue;
    const int alive = (int)std::count_if(block.threads, block.threads + kThreads, [](const Thread& t) { return !t.done; });
    if (!alive) break;
    if (block.waiting != alive) return false;
    block.waiting = 0;
    ++block.passed;
  }
  for (const Thread& t : block.threads)
    if (t.barriers != block.threads[0].barriers) return false;
  return true;
}

}  // namespace emu

#define threadIdx ::emu::thread
#define blockIdx ::emu::block_id
#define __builtin_amdgcn_readlane(v, l) ((int)::emu::exchange((uint32_t)(v))[l])
#define __builtin_amdgcn_readfirstlane(v) ((uint32_t)::emu::exchange((uint32_t)(v))[0])

namespace smoe {

using std::max;
using std::min;
constexpr int kWave = 64;
inline void __syncthreads() { ::emu::barrier(); }
inline uint64_t __ballot(bool p) {
  const uint64_t* const w = ::emu::exchange(p);
  uint64_t m = 0;
  for (int i = 0; i < 64; ++i) m |= w[i] << i;
  return m;
}
inline int __shfl_up(int v, unsigned by, int) {
  const unsigned lane = threadIdx.x & 63;
  return (int)::emu::exchange((uint32_t)v)[lane < by ? lane : lane - by];
}
inline unsigned long long wave_scan_u64(unsigned long long v) {
  const uint64_t* const w = ::emu::exchange(v);
  unsigned long long sum = 0;
  for (unsigned i = 0; i <= (threadIdx.x & 63); ++i) sum += w[i];
  return sum;
}

}  // namespace smoe
