// The picking half of the choice of pages, run as threads of the host: its lists against a sort, with one warp after the other held up behind the first
// barriers.  Built with a thread sanitizer, it also reports what no barrier orders.  Exits with 0, 1 (a wrong list), 66 (the sanitizer's report) or
// by the alarm, when threads wait at different barriers for good.
#include "cuda_cta.h"

#include "../orangu_b200/csrc/pages_pick.cuh"

#include <cstdio>
#include <numeric>
#include <random>

namespace {

template <uint32_t THREADS>
int check(const char *what, const std::vector<uint32_t> &keys, uint32_t n_select, uint32_t held_up) {
    const uint32_t n = (uint32_t)keys.size(), forced = (uint32_t)std::count(keys.begin(), keys.end(), ob::SEL_FORCED);
    std::vector<int32_t> out(n_select + 1, -7), order(n);
    std::iota(order.begin(), order.end(), 0);
    std::stable_sort(order.begin(), order.end(), [&](int a, int b) { return keys[a] > keys[b]; });
    order.resize(n_select);
    std::sort(order.begin(), order.end());
    order.push_back(-7);  // nothing behind the list
    cta::held_up = held_up;
    cta::run(THREADS, [&] {
        uint32_t lo = 0xffffffffu, hi = 0;
        for (uint32_t i = threadIdx.x; i < n; i += THREADS)
            if (keys[i] != ob::SEL_FORCED) lo = min(lo, keys[i]), hi = max(hi, keys[i]);
        ob::pick<THREADS>(n_select - forced, keys.data(), n, lo, hi, out.data());
    });
    if (out == order) return 0;
    std::printf("%s, %u of %u, warp %d held up: wrong list\n", what, n_select, n, (int)held_up);
    return 1;
}

template <uint32_t THREADS>
int all(uint32_t held_up) {
    std::mt19937 r(THREADS + held_up);
    int bad = 0;
    for (uint32_t n : {3u, 70u, 300u}) {
        std::vector<uint32_t> keys(n, 0x80000000u);  // scores of zero: a padded row, or a cache of zeros
        bad += check<THREADS>("all equal", keys, n / 2 + 1, held_up);
        keys[0] = keys[n - 1] = ob::SEL_FORCED;
        if (n > 3) bad += check<THREADS>("equal but the first and the last, which are kept", keys, n / 3, held_up);
        for (auto &k : keys) k = 0x80000000u + r() % 5;
        bad += check<THREADS>("few values", keys, n / 2, held_up);
        for (auto &k : keys) k = r() >> 1;
        bad += check<THREADS>("many values", keys, n / 2, held_up);
    }
    return bad;
}

}  // namespace

int main() {
    alarm(240);
    int bad = 0;
    for (uint32_t w : {~0u, 0u, 3u, 7u}) bad += all<256>(w);
    bad += all<1024>(31);
    return bad != 0;
}
