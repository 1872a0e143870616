// The 8-bit KV page: e4m3 codes (OCP: 4 exponent bits, 3 of mantissa, no
// infinities) of 16 tokens x 128 dims of one kv head, 2 KiB, and one scale 2^E
// per (block, kv head), K and V apart; a value is code * 2^E.
//
// E is the least whole number with top <= 448 * 2^E, top being the largest
// finite magnitude among the block's values when they were written, and
// kF8LeastExp at least. It is a power of two so that a block whose later token
// needs a larger scale can be re-encoded: the old codes lose their low bits
// only where they become subnormal (2^-15 of the block's top and less),
// however often the scale grows, where a scale of 24 bits would round every
// code again each time. The codes' relative error (2^-4 at most) is the same
// for any scale.
//
// Byte of (token t, dim d) within a page:
//   K: (d / 64) * 1024 + (d / 8 % 4) * 256 + t * 16 + (d / 32 % 2) * 8 + d % 8
//   V: (d / 64) * 1024 + (t / 4) * 256 + (d % 16) * 16 + (d / 16 % 4) * 4 + t % 4
// Each 1 KiB half is one 64-lane x 16 B load: K gives lane (t, d / 8 % 4) the
// eight codes of two 32-dim MFMA steps, V gives lane (d % 16, t / 4) four keys
// of four 16-dim blocks; widened to bf16 they are the operands that two
// loads of the bf16 page hold.
#pragma once

#include "launch.hpp"

#include <hip/hip_runtime.h>

#include <cstdint>

namespace llaisys::kernels {

constexpr int kF8LeastExp = -100; // blocks with a top under 2^-92 share this scale
constexpr int kF8MostExp = 120;   // that of the largest bf16
constexpr int kF8PageBytes = kPageTokens * kHeadDim;
// An append refuses a block's second run where its rows come up to this many
// rows after the first one's (one run writes a block).
constexpr int kF8LookBack = 32;

__host__ __device__ constexpr int kF8Index(int t, int d) {
    return (d >> 6) * 1024 + ((d >> 3) & 3) * 256 + t * 16 + ((d >> 5) & 1) * 8 + (d & 7);
}
__host__ __device__ constexpr int vF8Index(int t, int d) {
    return (d >> 6) * 1024 + (t >> 2) * 256 + (d & 15) * 16 + ((d >> 4) & 3) * 4 + (t & 3);
}

// E of a block whose largest finite magnitude has the bf16 bits `top` (sign
// cleared): 448 is 1.75 * 2^8, so E is top's exponent - 8, and one more where
// its significand is past 1.75.
__host__ __device__ inline int f8ExpOf(int top) {
    const int e = (top >> 7) - 127 - 8 + ((top & 0x7f) > 0x60 ? 1 : 0);
    return e > kF8LeastExp ? e : kF8LeastExp;
}
// E of a stored scale (its exponent; a block never written may hold anything).
__host__ __device__ inline int f8ExpOfScale(float scale) {
    const int e = int((__builtin_bit_cast(uint32_t, scale) >> 23) & 0xff) - 127;
    return e < kF8LeastExp ? kF8LeastExp : e > kF8MostExp ? kF8MostExp : e;
}
// 2^e for -126 <= e <= 127.
__host__ __device__ inline float f8Exp2(int e) { return __builtin_bit_cast(float, uint32_t(e + 127) << 23); }

} // namespace llaisys::kernels
