// A block of CUDA threads on the host: each a context of its own, switched at barriers and shuffles, so that a kernel's code that uses no more than these runs
// as it stands. For functions at the head of a kernel that lay out work, whose results must not depend on how many threads lay them out.
#pragma once
#include <algorithm>
#include <climits>
#include <cmath>
#include <cstddef>
#include <cstdint>
#include <cstdlib>
#include <cstring>
#include <functional>
#include <ucontext.h>
#include <vector>

#define __device__
#define __host__
#define __global__
#define __forceinline__ inline
#define __shared__ static
#define __restrict__

struct float2 { float x, y; };
struct int4 { int x, y, z, w; };
struct longlong2 { long long x, y; };
inline float2 make_float2(float x, float y) { return {x, y}; }
inline int4 make_int4(int x, int y, int z, int w) { return {x, y, z, w}; }
inline longlong2 make_longlong2(long long x, long long y) { return {x, y}; }
struct Dim { int x; };
static Dim threadIdx, blockIdx, blockDim;
using std::max;
using std::min;

namespace host_block {

struct Thread { ucontext_t at; std::vector<char> stack; bool done; };
struct Warp { uint64_t word[2][32]; int count, turn; };
static std::vector<Thread> threads;
static std::vector<Warp> warps;
static ucontext_t home;
static int here, count, turn, any[2];
static std::function<void()> work;

inline void enter() { work(); threads[here].done = true; swapcontext(&threads[here].at, &home); }
inline void yield() { swapcontext(&threads[here].at, &home); threadIdx.x = here; }

inline void run(int n, std::function<void()> f)
{
    work = f;
    threads.resize(n);
    warps.assign((n + 31) / 32, Warp{});
    count = turn = any[0] = any[1] = 0;
    blockDim.x = n;
    for (int i = 0; i < n; ++i) {
        Thread &t = threads[i];
        t.stack.resize(64 << 10);
        t.done = false;
        getcontext(&t.at);
        t.at.uc_stack.ss_sp = t.stack.data();
        t.at.uc_stack.ss_size = t.stack.size();
        t.at.uc_link = nullptr;
        makecontext(&t.at, enter, 0);
    }
    for (int left = n; left;) {
        left = 0;
        for (here = 0; here < n; ++here)
            if (!threads[here].done) { ++left; threadIdx.x = here; swapcontext(&home, &threads[here].at); }
    }
}
inline int barrier(int x)
{
    const int mine = turn;
    any[mine & 1] |= x;
    if (++count == blockDim.x) { count = 0; ++turn; any[turn & 1] = 0; }
    while (turn == mine) yield();
    return any[mine & 1];
}
template <typename T> T shuffle(T v, int from)
{
    Warp &w = warps[here / 32];
    const int mine = w.turn, lane = here % 32;
    w.word[mine & 1][lane] = 0;
    memcpy(&w.word[mine & 1][lane], &v, sizeof(T));
    if (++w.count == 32) { w.count = 0; ++w.turn; }
    while (w.turn == mine) yield();
    memcpy(&v, &w.word[mine & 1][from], sizeof(T));
    return v;
}

}  // namespace host_block

inline void __syncthreads() { host_block::barrier(0); }
inline int __syncthreads_or(int x) { return host_block::barrier(x != 0); }
template <typename T> T __shfl_sync(unsigned, T v, int lane) { return host_block::shuffle(v, lane); }
template <typename T> T __shfl_up_sync(unsigned, T v, int by) { const int lane = host_block::here % 32; return host_block::shuffle(v, lane >= by ? lane - by : lane); }
inline unsigned __umulhi(unsigned a, unsigned b) { return (unsigned)((uint64_t)a * b >> 32); }
inline float __fdividef(float a, float b) { return a / b; }
inline int __clz(int x) { return x ? __builtin_clz(x) : 32; }
inline int __clzll(long long x) { return x ? __builtin_clzll(x) : 64; }
inline void atomicOr(unsigned *at, unsigned bits) { *at |= bits; }
