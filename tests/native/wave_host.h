// Device code of waves of 64 lanes, run on the host: every lane is a context of its own that runs until it reaches an
// operation of the whole wave (a ballot, a permutation, a fence) or of its block (a barrier), and goes on once all lanes
// have reached the same one.  Between two of them the lanes run one after the other, so what one lane leaves in LDS for
// another without a fence between comes out wrong, and lanes that part ways end the program.  Compiled with
// AddressSanitizer, every access outside its array does too.
#pragma once

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <functional>
#include <type_traits>
#include <vector>

struct dim3 { unsigned x, y, z; };
static dim3 threadIdx, blockIdx, blockDim, gridDim;
struct int4 { int x, y, z, w; } __attribute__((aligned(16)));

namespace host {

// Goes on where the stack `to` was left, and leaves this one at *from (x86-64).
extern "C" void host_switch(void** from, void* to);
asm(".text\n.globl host_switch\nhost_switch:\n"
    "pushq %rbp\npushq %rbx\npushq %r12\npushq %r13\npushq %r14\npushq %r15\n"
    "movq %rsp, (%rdi)\nmovq %rsi, %rsp\n"
    "popq %r15\npopq %r14\npopq %r13\npopq %r12\npopq %rbx\npopq %rbp\nret\n");

enum State { kReady, kAtWave, kAtBlock, kDone };
struct Lane {
  char* stack = nullptr;
  void* at = nullptr;                 // where it goes on
  State state = kReady;
  int site = 0, turn = 0;
};
static std::vector<Lane> lanes;
static void* scheduler;
static int current;
static uint64_t left[2][1024];        // what lanes leave for each other, two sets in turn
static std::function<void()> body;
constexpr size_t kStack = 1 << 18;

[[noreturn]] inline void fail(const char* what, int site) {
  fprintf(stderr, "%s (line %d)\n", what, site);
  fflush(stderr);
  _Exit(2);
}

static void run_lane() {
  body();
  lanes[current].state = kDone;
  host_switch(&lanes[current].at, scheduler);
}

// Leaves `v` for the other lanes of the wave and returns what all 64 of them left.
inline const uint64_t* meet(State at, int site, uint64_t v) {
  const int me = current;
  Lane& l = lanes[me];
  const int turn = l.turn;
  l.turn ^= 1;
  left[turn][me] = v;
  l.state = at;
  l.site = site;
  host_switch(&l.at, scheduler);
  return left[turn] + me / 64 * 64;
}

// Whether the lanes [first, last) all wait for each other at one place; they go on if so.
inline bool release(int first, int last, State at, const char* part) {
  int n = 0;
  for (int i = first; i < last; ++i) n += lanes[i].state == at;
  if (!n) return false;
  for (int i = first; i < last; ++i)
    if (lanes[i].state != at || lanes[i].site != lanes[first].site) fail(part, lanes[i].site);
  for (int i = first; i < last; ++i) lanes[i].state = kReady;
  return true;
}

template <class F>
void launch(unsigned grid, unsigned block, F f) {
  const int n = (int)block;
  lanes.resize(std::max<size_t>(lanes.size(), n));
  gridDim = {grid, 1, 1}, blockDim = {block, 1, 1};
  body = f;
  for (unsigned b = 0; b < grid; ++b) {
    blockIdx = {b, 0, 0};
    for (int i = 0; i < n; ++i) {
      Lane& l = lanes[i];
      if (!l.stack) l.stack = (char*)malloc(kStack);
      l.state = kReady, l.turn = 0;
      void** top = (void**)(((uintptr_t)l.stack + kStack) / 16 * 16) - 1;
      *--top = (void*)run_lane;       // behind six saved registers
      l.at = top - 6;
    }
    for (;;) {
      bool ran = false;
      for (int i = 0; i < n; ++i)
        if (lanes[i].state == kReady) {
          current = i;
          threadIdx = {(unsigned)i, 0, 0};
          host_switch(&scheduler, lanes[i].at);
          ran = true;
        }
      for (int w = 0; w < n; w += 64) ran |= release(w, w + 64, kAtWave, "the lanes of a wave part ways");
      if (!ran && !release(0, n, kAtBlock, "the threads of a block part ways")) break;
    }
  }
}

inline unsigned long long ballot(bool p, int site) {
  const uint64_t* all = meet(kAtWave, site, p);
  unsigned long long m = 0;
  for (int i = 0; i < 64; ++i) m |= (unsigned long long)all[i] << i;
  return m;
}
template <class T>
T from_lane(T v, int lane, int site) {
  uint64_t bits = 0;
  memcpy(&bits, &v, sizeof v);
  bits = meet(kAtWave, site, bits)[lane & 63];
  memcpy(&v, &bits, sizeof v);
  return v;
}
// The permutations within 16 lanes that the reductions use.
inline int permuted(int v, int control, int site) {
  const int lane = current & 63;
  switch (control) {
    case 0xB1: return from_lane(v, lane ^ 1, site);
    case 0x4E: return from_lane(v, lane ^ 2, site);
    case 0x141: return from_lane(v, lane ^ 7, site);
    case 0x140: return from_lane(v, lane ^ 15, site);
  }
  fail("a permutation that is not known here", site);
}
inline unsigned below(unsigned mask, int lanes_before) {
  return lanes_before <= 0 ? 0 : __builtin_popcount(lanes_before >= 32 ? mask : mask & ((1u << lanes_before) - 1));
}
template <class To, class From>
To bits(From v) {
  To t;
  static_assert(sizeof t == sizeof v, "");
  memcpy(&t, &v, sizeof v);
  return t;
}

}  // namespace host

#define __device__
#define __global__
#define __forceinline__ inline
#define __launch_bounds__(...)
#define __shared__ static
#define __align__(n) __attribute__((aligned(n)))
#define __ballot(p) host::ballot(p, __LINE__)
#define __popcll(m) __builtin_popcountll(m)
#define __shfl_xor(v, m, w) host::from_lane(v, (host::current & 63) ^ (m), __LINE__)
#define __syncthreads() host::meet(host::kAtBlock, __LINE__, 0)
#define __builtin_amdgcn_update_dpp(o, v, c, r, b, z) host::permuted(v, c, __LINE__)
#define __builtin_amdgcn_fence(o, s) host::meet(host::kAtWave, __LINE__, 0)
#define __builtin_amdgcn_mbcnt_lo(m, c) (host::below(m, host::current & 63) + (c))
#define __builtin_amdgcn_mbcnt_hi(m, c) (host::below(m, (host::current & 63) - 32) + (c))
#define __builtin_amdgcn_exp2f(v) exp2f(v)
#define __float_as_int(v) host::bits<int>((float)(v))
#define __int_as_float(v) host::bits<float>((int)(v))
#define __float_as_uint(v) host::bits<unsigned>((float)(v))
#define __uint_as_float(v) host::bits<float>((unsigned)(v))
#define __double_as_longlong(v) host::bits<long long>((double)(v))
#define __longlong_as_double(v) host::bits<double>((long long)(v))
