// Pages in 4 bits: how the keys and values of a page of one key/value head lie together, and how codes become f16 numbers.
//
// 32 entries of a position's key or value share a unit d, an f16 number of 7 significant bits and at most 896: entry = c d, c from -8 to 7, kept as c + 8.
// Then c d has at most 10 significant bits, and every entry is an f16 number exactly: products with queries and weights are those of an f16 cache.
// 72 d is one, too (10 bits, at most 64512), which is what makes an entry one fused multiply-add of its code: 64 + (c + 8) is the f16 number 0x5400 | (c + 8) << 4,
// and (64 + c + 8) d - 72 d = c d is not rounded.
//
// Eight entries e0 .. e7 are two halves of 16 bits: nibble j of the first is e_2j, nibble j of the second e_2j+1.  As one word, a mask takes two neighbours at a
// time.  A block (page, head) is 9 HD bytes, HD / 2 a position and then the units:
//
//   keys    position p's words in order at p HD / 2; units [position][32 entries]
//   values  positions 2 r and 2 r + 1 lie together, HD bytes: for each eight entries the first halves of both in a word, then the second ones, so that a mask takes
//           the same entry of two positions; units [32 entries][position].  The places of the eights are exchanged by a mask that depends on r, so that four lanes with
//           four pairs of positions and eight lanes with an eighth of the dimensions each read without bank conflicts.
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
    // Byte of a key's entries 8 w .. 8 w + 7 (a word); of a value's (two halves, four bytes apart); and of the unit of group g.
    static __host__ __device__ __forceinline__ uint32_t key(uint32_t p, uint32_t w) { return p * ROW + 4 * w; }
    static __host__ __device__ __forceinline__ uint32_t eight(uint32_t r, uint32_t w) { return w ^ (HD == 128 ? (r & 3) << 2 : (r & 2) << 1); }  // place of eight w in pair r, and back
    static __host__ __device__ __forceinline__ uint32_t value(uint32_t p, uint32_t w) { return (p >> 1) * HD + 8 * eight(p >> 1, w) + 2 * (p & 1); }
    static __host__ __device__ __forceinline__ uint32_t unit(bool value, uint32_t p, uint32_t g) { return CODES + 2 * (value ? g * KV_PAGE + p : p * GROUPS + g); }
};

// Field j of a word: the entries whose nibbles are j of both halves, times their units.  d: the units, n: -72 times them.  Nibbles 1 and 3 (after a shift by 8 for
// both 2 and 3) are taken where they make 64 + c + 8; 0 and 2 where they make 1024 + c + 8, from which 1032 is taken first: that costs a fused
// multiply-add more and a shift less, of which an SM does half as many.
__device__ __forceinline__ uint32_t q4_field(uint32_t w, int j, uint32_t d, uint32_t n) {
    const uint32_t x = j < 2 ? w : w >> 8;
    uint32_t u, r;
    if (j & 1) {
        asm("lop3.b32 %0, %1, 0x00f000f0, 0x54005400, 0xea;" : "=r"(u) : "r"(x));  // (x & mask) | 64
        asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(u), "r"(d), "r"(n));
    } else {
        asm("lop3.b32 %0, %1, 0x000f000f, 0x64006400, 0xea;" : "=r"(u) : "r"(x));  // (x & mask) | 1024
        asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(u) : "r"(u), "r"(0x64086408u));
        asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(u), "r"(d));
    }
    return r;
}
__device__ __forceinline__ uint32_t q4_offset(uint32_t d) {  // -72 d, exact
    uint32_t n;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(n) : "r"(d), "r"(0xd480d480u));
    return n;
}

__device__ __forceinline__ uint32_t lds32(uint32_t at) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(at));
    return v;
}
__device__ __forceinline__ uint32_t lds16(uint32_t at) {
    uint16_t v;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(at));
    return v;
}
template <int N> __device__ __forceinline__ void lds_words(uint32_t (&v)[N], uint32_t at) {
    if constexpr (N == 4) asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(at));
    else asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v[0]), "=r"(v[1]) : "r"(at));
}

}  // namespace ob
