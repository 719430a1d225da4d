// Pages in 4 bits: how the keys and values of a page of one key/value head lie together, and how codes become f16 numbers.
//
// 32 entries of a position's key or value share a unit d, an f16 number of 7 significant bits and at most 896: entry = c d, c from -8 to 7, kept as c + 8.
// Then c d has at most 10 significant bits, and every entry is an f16 number exactly: products with queries and weights are those of an f16 cache.
// 72 d is one, too (10 bits, at most 64512), which is what makes an entry one fused multiply-add of its code: 64 + (c + 8) is the f16 number 0x5400 | (c + 8) << 4,
// and (64 + c + 8) d - 72 d = c d is not rounded.
//
// A word of 32 bits is eight entries e0 .. e7 in order: nibble j of the low half is e_2j, nibble j of the high half e_2j+1, so that a mask takes
// two neighbours at a time.  A block (page, head) is 9 HD bytes, HD / 2 a position and then the units:
//
//   keys    position p's words in order at p HD / 2; units [position][32 entries]
//   values  position p at slot(p) HD / 2, slot = p / 2 % 4 + p % 2 * 4 + p / 8 * 8; units [32 entries][position].  With HD = 128 the two halves of every other
//           pair of slots are exchanged.  Four lanes then read four positions two apart, eight lanes the dimensions, without bank conflicts.
#pragma once

#include <cuda_fp16.h>
#include <stdint.h>

#include "common.cuh"

namespace ob {

constexpr uint32_t Q4_GROUP = 32;           // entries of a unit
constexpr float Q4_LARGEST = 7168.0f;       // what larger entries count as: 8 units of 896

template <int HD>
struct Q4Block {
    static constexpr uint32_t ROW = HD / 2, CODES = KV_PAGE * ROW, GROUPS = HD / Q4_GROUP, BYTES = CODES + KV_PAGE * GROUPS * 2;
    static_assert(BYTES == 9 * HD, "9 bits for two entries");
    static __host__ __device__ __forceinline__ uint32_t slot(uint32_t p) { return (p >> 1 & 3) | (p & 1) << 2 | (p & 8); }
    // Byte of word w (eight entries) of a position, and of the unit of group g.
    static __host__ __device__ __forceinline__ uint32_t word(bool value, uint32_t p, uint32_t w) {
        if (!value) return p * ROW + 4 * w;
        const uint32_t s = slot(p);
        return s * ROW + 4 * (HD == 128 && (s & 2) ? w ^ 8 : w);
    }
    static __host__ __device__ __forceinline__ uint32_t unit(bool value, uint32_t p, uint32_t g) { return CODES + 2 * (value ? g * KV_PAGE + p : p * GROUPS + g); }
};

// Field j of a word: the entries whose nibbles are j of both halves, times their units.  d: the units, n: -72 times them.
__device__ __forceinline__ uint32_t q4_field(uint32_t w, int j, uint32_t d, uint32_t n) {
    const uint32_t x = j == 0 ? w << 4 : w >> (4 * j - 4);
    uint32_t u, r;
    asm("lop3.b32 %0, %1, 0x00f000f0, 0x54005400, 0xea;" : "=r"(u) : "r"(x));  // (x & mask) | 64
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(u), "r"(d), "r"(n));
    return r;
}
__device__ __forceinline__ uint32_t q4_offset(uint32_t d) {  // -72 d, exact
    uint32_t n;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(n) : "r"(d), "r"(0xd480d480u));
    return n;
}

}  // namespace ob
