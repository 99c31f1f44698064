// A cache of keys and values in 8 bits, as its kernels see it.
//
// Pages of `page_size` tokens.  A block is 16 tokens of a page, the whole page where 16 does not divide its size.  Of a (block, kv
// head) the keys have one scale and the values one, powers of two: s = 2^e with the least e >= LEAST for which every finite |x| that
// the block holds is at most 448 s (448: the largest e4m3 number).  A byte is the e4m3 number nearest to x / s, ties to even (with e = 120, the
// greatest, of those up to 240: 256 s is no float32 number any more, and less than 256 s is off by less than 2^-4 of itself); what is not finite
// is kept as NaN, and a block whose values hold one says so by a negative scale.
//   keys   [page, head, token, channel]
//   values [page, head, block, channel, token]   16 bytes: a channel's tokens of a block, a matrix-core operand's own order
//   scales [page, head, block, (key, value)]     float32
// A power of two: bytes of earlier tokens move to a larger scale by their exponents alone (exact unless they end below the smallest
// normal e4m3 number, 2^-6 s), and the matrix cores' operands take it in the conversion to bfloat16, which has a place for it.
#pragma once

#include "common.h"

namespace cache8 {

constexpr int LEAST = -118;        // 2^-118 and 2^118 are normal float32 numbers, and 2^-118 times the smallest e4m3 number is none that matters
constexpr int MOST = 120;          // of the largest float32 numbers
constexpr int BLOCK = 16;

__host__ __device__ inline int block_tokens(int page_size) { return page_size % BLOCK == 0 ? BLOCK : page_size; }

// 2^e, -126 <= e <= 127
__device__ __forceinline__ float pow2(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

// The least e >= LEAST with amax <= 448 * 2^e (amax finite, >= 0): 448 = 1.75 * 2^8.
__device__ __forceinline__ int exponent_for(float amax) {
    const uint32_t b = __float_as_uint(amax);
    const int e = static_cast<int>(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
    return e > LEAST ? e : LEAST;
}
__device__ __forceinline__ int exponent_of(float scale) { return static_cast<int>((__float_as_uint(scale) >> 23) & 0xff) - 127; }

__device__ __forceinline__ bool finite(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }

// Two float32 numbers, |x| <= 448 or not finite, to two e4m3 bytes (round to nearest even; what is not finite to NaN).
__device__ __forceinline__ uint32_t to_e4m3x2(float lo, float hi) {
    const uint32_t both = static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(finite(lo) ? lo : 0.f, finite(hi) ? hi : 0.f, 0, false)) & 0xffffu;
    return both | (finite(lo) ? 0u : 0x7fu) | (finite(hi) ? 0u : 0x7f00u);
}
__device__ __forceinline__ uint32_t to_e4m3x4(float a, float b, float c, float d) { return to_e4m3x2(a, b) | (to_e4m3x2(c, d) << 16); }

// Bytes of a block of exponent e: 240 where 256 (0x78, the largest there) would stand, if 256 * 2^e is no float32 number.
__device__ __forceinline__ uint32_t at_exponent(int e, uint32_t w) {
    if (e < MOST) return w;
    const uint32_t apart = (w & 0x7f7f7f7fu) ^ 0x78787878u;
    return w - ((~(apart + 0x7f7f7f7fu) & 0x80808080u) >> 7);
}

// What four bytes stand for, before the scale.
__device__ __forceinline__ void from_e4m3x4(uint32_t b, float (&out)[4]) {
    typedef __attribute__((ext_vector_type(2))) float f32x2;
    const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(b), false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(b), true);
    out[0] = lo[0];
    out[1] = lo[1];
    out[2] = hi[0];
    out[3] = hi[1];
}
__device__ __forceinline__ float from_e4m3(uint8_t b) { return __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(b), 0); }

// Four bytes at a scale 2^by times as large (by >= 0); NaN stays.
__device__ __forceinline__ uint32_t moved(uint32_t b, float down) {
    float x[4];
    from_e4m3x4(b, x);
    return to_e4m3x4(x[0] * down, x[1] * down, x[2] * down, x[3] * down);
}

// a / b and a % b for 0 <= a < 2^31 by a multiplication, without a branch: with L the least number for which 2^L >= b and
// m = floor(2^(31 + L) / b) + 1 (less than 2^32), a m / 2^(31 + L) exceeds a / b by less than 1 / b.
struct Div {
    int b;
    uint32_t m, shift;
    __device__ __forceinline__ int over(int a) const { return static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(a)) * m) >> shift); }
    __device__ __forceinline__ int rest(int a) const { return a - over(a) * b; }
};
inline Div div_by(int b) {
    uint32_t bits = 0;
    while ((1ll << bits) < b) ++bits;
    return {b, static_cast<uint32_t>((1ull << (31 + bits)) / static_cast<uint32_t>(b) + 1), 31 + bits};
}

}  // namespace cache8
