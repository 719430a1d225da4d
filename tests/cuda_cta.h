// One CTA's threads as threads of the host, for device code that needs no more of CUDA than barriers, warp votes and exchanges, and integer
// built-ins.  Shared memory is static memory (one CTA at a time); every __syncthreads is a barrier of all threads and every warp-wide built-in one of
// 32, so that what the code leaves unordered is unordered here, too: a thread sanitizer reports it, and a warp that is held up behind a barrier
// (hold_up) sees what the others have written meanwhile.
#pragma once

#include <pthread.h>
#include <stdint.h>
#include <unistd.h>

#include <algorithm>
#include <functional>
#include <thread>
#include <vector>

#define __device__
#define __forceinline__ inline
#define __shared__ static

struct Dim3 {
    uint32_t x;
};
inline thread_local Dim3 threadIdx;

namespace cta {

inline pthread_barrier_t all, warps[32];
inline uint32_t lanes[32][32];
inline uint32_t held_up = ~0u;   // this warp sleeps behind each of its first barriers
inline thread_local uint32_t barriers = 0;

inline uint32_t warp() { return threadIdx.x / 32; }
inline uint32_t lane() { return threadIdx.x % 32; }
inline void join() { pthread_barrier_wait(&warps[warp()]); }

// Every lane's word, seen by all of them.
template <typename F>
uint32_t exchange(uint32_t mine, F f) {
    lanes[warp()][lane()] = mine;
    join();
    const uint32_t r = f(lanes[warp()]);
    join();
    return r;
}

inline void run(uint32_t threads, const std::function<void()> &body) {
    pthread_barrier_init(&all, nullptr, threads);
    for (uint32_t w = 0; w < threads / 32; ++w) pthread_barrier_init(&warps[w], nullptr, 32);
    std::vector<std::thread> ts;
    for (uint32_t t = 0; t < threads; ++t)
        ts.emplace_back([&, t] {
            threadIdx.x = t;
            barriers = 0;
            body();
        });
    for (auto &t : ts) t.join();
}

}  // namespace cta

inline void __syncthreads() {
    pthread_barrier_wait(&cta::all);
    if (cta::warp() == cta::held_up && cta::barriers++ < 2) usleep(20000);
}
inline uint32_t __reduce_min_sync(uint32_t, uint32_t v) {
    return cta::exchange(v, [](const uint32_t *w) { return *std::min_element(w, w + 32); });
}
inline uint32_t __reduce_max_sync(uint32_t, uint32_t v) {
    return cta::exchange(v, [](const uint32_t *w) { return *std::max_element(w, w + 32); });
}
inline uint32_t __shfl_sync(uint32_t, uint32_t v, int src) {
    return cta::exchange(v, [&](const uint32_t *w) { return w[src]; });
}
inline uint32_t __shfl_up_sync(uint32_t, uint32_t v, int by) {
    return cta::exchange(v, [&](const uint32_t *w) { return (int)cta::lane() >= by ? w[cta::lane() - by] : v; });
}
inline uint32_t __ballot_sync(uint32_t, bool p) {
    return cta::exchange(p, [](const uint32_t *w) {
        uint32_t b = 0;
        for (int i = 0; i < 32; ++i) b |= w[i] << i;
        return b;
    });
}
inline int warp_sum_i(int v) {
    return (int)cta::exchange((uint32_t)v, [](const uint32_t *w) {
        uint32_t s = 0;
        for (int i = 0; i < 32; ++i) s += w[i];
        return s;
    });
}
inline uint32_t atomicAdd(uint32_t *p, uint32_t v) { return __atomic_fetch_add(p, v, __ATOMIC_RELAXED); }
inline int __popc(uint32_t v) { return __builtin_popcount(v); }
inline int __clz(uint32_t v) { return v ? __builtin_clz(v) : 32; }
using std::max;
using std::min;
