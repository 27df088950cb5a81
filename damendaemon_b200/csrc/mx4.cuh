// Microscaled 4-bit matrices: how they lie in memory, and the pieces that the kernels which read them share.
//
// 32 neighbouring elements of a row, a block, share a power of two; an element is sign, two bits of exponent and one of
// mantissa (e2m1: 0, 0.5, 1, 1.5, 2, 3, 4, 6). Four blocks, a group of 128 elements, are sixteen 32-bit words: word 4 t + b holds
// elements 8 t .. 8 t + 7 of block b, so that one 16-byte load gives lane t of four its eighth of every block of the group. In a word
// elements 0, 2, 4, 6 lie in bits 0 .. 15 and 1, 3, 5, 7 in bits 16 .. 31, so that one mask cuts out two neighbours at once. A row is
// padded with zeros to whole groups. A block's scale is a byte s for 2^(s - 127), four bytes a group; s = 255 marks a block
// that had no finite numbers.
#pragma once
#include <stdint.h>

namespace mx4 {
constexpr int BLOCK = 32, GROUP = 128, GROUP_BYTES = 64;

// The eight elements of a word as bfloat16 pairs (0,1) (2,3) (4,5) (6,7), each element times 2^-126: exponent and mantissa
// bits moved to the low end of bfloat16's exponent. 0.5 becomes a subnormal, which the tensor cores take as it is.
__device__ __forceinline__ void pairs(uint32_t w, uint32_t* v) {
    constexpr uint32_t SIGN = 0x80008000u, SIZE = 0x01C001C0u;
    v[0] = ((w << 12) & SIGN) | ((w << 6) & SIZE);
    v[1] = ((w << 8) & SIGN) | ((w << 2) & SIZE);
    v[2] = ((w << 4) & SIGN) | ((w >> 2) & SIZE);
    v[3] = (w & SIGN) | ((w >> 6) & SIZE);
}
// The elements themselves as bfloat16 pairs in that order: products with rows of any size then stay clear of float32's ends. (With the
// pairs above and rows times 2^64 instead, rows from 2^64 on were not finite and those below 2^-64 lost; the time is the same: 6,400 x 1,600
// by one row 4.65 us, 1,600 x 6,400 by eight 6.5, before 6.65.)
__device__ __forceinline__ void whole_pairs(uint32_t w, uint32_t* v) {
    pairs(w, v);
#pragma unroll
    for (int i = 0; i < 4; ++i) asm("mul.rn.bf16x2 %0, %0, %1;" : "+r"(v[i]) : "r"(0x7E807E80u));        // 2^126
}
// pairs() with multiplications for the shifts to the left: masks and multiply-adds then take two pipes by turns. The powers of two come
// from the launch (a constant would be made a shift again).
struct Shifts { uint32_t by4, by16, by64, by256, by4096; };
constexpr Shifts SHIFTS = {4, 16, 64, 256, 4096};
__device__ __forceinline__ void pairs(uint32_t w, const Shifts& m, uint32_t* v) {
    const uint32_t down = w >> 6;
    v[0] = (w & 0x00080008u) * m.by4096 + (w & 0x00070007u) * m.by64;
    v[1] = (w & 0x00800080u) * m.by256 + (w & 0x00700070u) * m.by4;
    v[2] = ((w & 0x08000800u) | (down & 0x001C001Cu)) * m.by16;
    v[3] = (w & 0x80008000u) | (down & 0x01C001C0u);
}
// The eight elements of a word as float16 pairs (0,2) (4,6) (1,3) (5,7), one instruction a pair. (83 elements a clock and SM, the
// bfloat16 pairs above 45.)
__device__ __forceinline__ void pairs_f16(uint32_t w, uint32_t* v) {
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\tmov.b32 {b0, b1, b2, b3}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, b0;\n\tcvt.rn.f16x2.e2m1x2 %1, b1;\n\tcvt.rn.f16x2.e2m1x2 %2, b2;\n\tcvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(w));
}
// 2^(s - 127) of block b of a group's four scale bytes (s = 0: a subnormal number); s = 255 as infinity.
__device__ __forceinline__ float scale(uint32_t four, int b) {
    const uint32_t moved = b == 0 ? four << 23 : b == 1 ? four << 15 : b == 2 ? four << 7 : four >> 1;
    return __uint_as_float(max(moved & 0x7f800000u, 0x00400000u));
}
}  // namespace mx4
