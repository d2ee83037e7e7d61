// Numbers held in four bits: how the codes of weights and of cached keys and values lie in memory, and how they become bfloat16 pairs.
//
// A word holds eight codes, the lowest bits first.  `pair(w, i)` is codes i and i + 4 of it as the bfloat16 numbers 128 + code: a code in the low bits of
// the mantissa of 128 (0x4300, whose last bit is worth 1) is that number, so a pair costs a shift and one logical operation.
//
// Weights [n, k] lie in tiles of 128 x 128 codes, a row 16 words: word 4 t + w holds columns 32 w + 8 t + (0..7).  The lane of column t of a tensor-core fragment so finds in
// sixteen bytes a word of each 32 columns, and products of one word belong to one group of 32, 64 or 128 columns that share a scale.
//
// The cache is [pages, kv_heads, 2 (keys, values), page_size * (d / 2 + d / 16)] bytes: the codes of the page's places, d / 2 bytes each, then for each place and group of 64
// features its step and its lowest value, two bfloat16 numbers.  Word 8 j + 4 h + t of a key (j the group) lies at (t, j, h), word 8 j + g of a value at (g, j): each lane
// of a fragment finds what it needs of a place side by side.
#pragma once

#include "common.cuh"

namespace lily {
namespace four {

constexpr int GROUP = 64;                    // features of a head that share a step and a lowest value

// codes i and i + 4 (0 <= i < 4) as bfloat16 numbers 128 + code
__device__ __forceinline__ uint32_t pair(uint32_t w, int i) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(w >> (4 * i)), "r"(0x000F000Fu), "r"(0x43004300u));      // (a & b) | c
    return r;
}
__device__ __forceinline__ uint32_t bits(__nv_bfloat162 v) { return *reinterpret_cast<uint32_t*>(&v); }
__device__ __forceinline__ __nv_bfloat162 two(uint32_t v) { return *reinterpret_cast<__nv_bfloat162*>(&v); }
__device__ __forceinline__ float low(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float high(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }

__host__ __device__ __forceinline__ size_t row_bytes(int d) { return d / 2 + d / 16; }       // a place of one head, keys or values
// Where word `l` of a place's codes lies among its d / 8.
__device__ __forceinline__ int key_word(int l, int groups) { return (l & 3) * 2 * groups + 2 * (l >> 3) + ((l >> 2) & 1); }
__device__ __forceinline__ int value_word(int l, int groups) { return (l & 7) * groups + (l >> 3); }

}  // namespace four
}  // namespace lily
