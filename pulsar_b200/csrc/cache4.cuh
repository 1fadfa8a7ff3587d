// Keys and values held in 4 bits.
//
// For every token, kv head and group of 32 neighbouring channels x_0 .. x_31 a cache holds a least value m, a step s (both bfloat16) and
// codes c_i of 4 bits; the value that they stand for is m + s c_i in float32:
//
//   m = the largest bfloat16 <= min x        s = the smallest bfloat16 >= (max x - m) / 15        c_i = round((x_i - m) / s), halves to even
//
// Both are rounded outwards, so that every x_i lies between m and m + 15 s and is off by s / 2 at most; bfloat16 has float32's range, so
// small and large heads keep their relative precision (float16 steps would end at 6e-8 and 65,504).  A group that holds a NaN or anything
// beyond bfloat16's range has m = s = NaN.
//
// A pool is [pages, heads, page, width]: codes in bytes, D / 2 a row, and steps, D / 16 bfloat16 a row (s and m of group 0, of group 1, ...).
// In a row of codes the 16-bit word r * G + g, r < 8, G = D / 32 groups, holds channels 32 g + 4 r .. + 3, the first in the lowest bits.  The
// lanes of a quad of a matrix instruction then find what they need of all groups side by side, and every step of 16 channels lies inside one group.
#pragma once

#include <string.h>

#include "common.cuh"

namespace pb {

constexpr int kGroup4 = 32;
constexpr float kMost4 = 3.38953139e38f;          // the largest bfloat16

struct Pool4 {
    uint8_t* codes;             // [pages, heads, page, D / 2]
    __nv_bfloat16* steps;       // [pages, heads, page, D / 16]
};

// A page of a block table as the kernels of this cache take it: -1 where it is not a page of the pool (nothing is read or written there).
__device__ __forceinline__ int page_or_none(int page, int n_pages) { return (unsigned)page < (unsigned)n_pages ? page : -1; }

// Whether a word of a step and a least value holds a NaN or an infinity.
__device__ __forceinline__ bool no_number(uint32_t word) { return (word & 0x7f80u) == 0x7f80u || (word & 0x7f800000u) == 0x7f800000u; }

// The arguments of the entry points of this cache come as one row of 64-bit words (a pointer, a whole number or a double each), which the host fills in
// a sixth of the time that as many arguments of a call take it.
struct Words4 {
    const long long* at;
    template <typename P> P* ptr() { return reinterpret_cast<P*>(*at++); }
    int num() { return (int)*at++; }
    double real() {
        double v;
        memcpy(&v, at++, 8);
        return v;
    }
};

}  // namespace pb
