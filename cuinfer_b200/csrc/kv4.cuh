// The paged cache that holds keys and values in 4 bits.
//
// A group is 32 neighbouring values of a head's key (normed and rotated) or value.  It shares one 16-bit word: a bfloat16 step with
// four significant bits (sign 0, 8 bits of exponent, the upper 3 of the 7 bits of mantissa) whose low four bits hold the zero point.
// A value is step * (code - zero), code and zero in 0..15: four significant bits times four, so it is exact in bfloat16 and every
// kernel, whatever it multiplies in, works on the same numbers.  4.5 bits a value.
//
//   lo = min(0, x), hi = max(0, x) over the group        (zero is always one of the values, so the zero point fits four bits)
//   step = (hi - lo) / 15 rounded up to four significant bits, at least 2^-120
//   zero = rint(-lo / step),  code = clamp(rint(x / step) + zero, 0, 15)
//
// A value comes back within step / 2: the range is at most 15 steps, so where rounding both ends up asks for code 16, clamping
// it to 15 leaves half a step as well.  All of it is 32-bit arithmetic rounded to nearest, operation by operation, so the
// codes do not depend on who computes them.  A group with a value that is not finite, or whose magnitude is 2^127 or more, reads
// back as NaN.
//
// 16 tokens of one key head are one block of 18 * D bytes; cache [page][kv head][page_size / 16][18 D].  The order inside is that of
// the operand fragments of mma.m16n8k16, so that a warp's loads of codes are 16 bytes a lane and consecutive:
//   key codes    8 D bytes   32-bit words [token 16][quarter 4][group]: values 32 group + 8 quarter + e, e = 0..7, in bits 4 (e / 2) + 16 (e % 2)
//   key words    D bytes     16-bit words [token 16][group]
//   value codes  8 D bytes   32-bit words [half 2][eighth 8][pair 4][group]: values 32 group + 4 eighth + e, e = 0..3, of token 8 half + 2 pair
//                            in bits 4 e and of the token after it in bits 16 + 4 e (a token's codes are whole 16-bit words: tokens
//                            are appended without reading what is there)
//   value words  D bytes     16-bit words [pair 8][group][token of the pair]
#pragma once

#include "common.cuh"

namespace cib {
namespace kv4 {

constexpr int kGroup = 32;
constexpr int kBlock = 16;
constexpr int kMaxHeadDim = 256;
constexpr uint32_t kNanWord = 0x7ff0u;

__host__ __device__ constexpr int block_bytes(int d) { return 18 * d; }
__host__ __device__ constexpr int key_words_at(int d) { return 8 * d; }
__host__ __device__ constexpr int value_codes_at(int d) { return 9 * d; }
__host__ __device__ constexpr int value_words_at(int d) { return 17 * d; }

// the step of a word in the low half of `w`
__device__ __forceinline__ float step_of(uint32_t w) { return __uint_as_float((w & 0xfff0u) << 16); }

// The block that holds `slot` of head `kvh`; nullptr where the slot is none (below zero or beyond the pool).
__device__ __forceinline__ unsigned char* block_of(unsigned char* cache, int slot, int num_pages, int page_size, int nkv, int kvh, int d) {
    if (slot < 0) return nullptr;
    const int page = slot / page_size;
    if (page >= num_pages) return nullptr;
    const int block = (slot - page * page_size) / kBlock;
    return cache + (((size_t)page * nkv + kvh) * (page_size / kBlock) + block) * (size_t)block_bytes(d);
}

// x / s rounded to nearest, from r = 1 / s rounded to nearest: the quotient's remainder is exact in a fused multiply-add, and adding it times r
// rounds correctly (P. Markstein, "Computation of elementary functions on the IBM RISC System/6000 processor", IBM J. Res. Dev. 34, 1990).
// Where it underflows, |x| is far below a step and the code does not depend on it.
__device__ __forceinline__ float quotient(float x, float s, float r) {
    const float q = __fmul_rn(x, r);
    return __fmaf_rn(__fmaf_rn(-q, s, x), r, q);
}

struct Scale {
    float step, inverse, zero;
    uint32_t word;
};

// lo <= 0 <= hi; `bad`: a value of the group is not finite or too large
__device__ __forceinline__ Scale scale_of(float lo, float hi, bool bad) {
    Scale s;
    const float t = fmaxf(quotient(__fsub_rn(hi, lo), 15.f, 1.f / 15.f), 7.5231638452626401e-37f);      // 2^-120
    s.step = __uint_as_float((__float_as_uint(t) + 0xfffffu) & ~0xfffffu);
    s.inverse = __frcp_rn(s.step);
    s.zero = rintf(quotient(-lo, s.step, s.inverse));
    s.word = bad ? kNanWord : (__float_as_uint(s.step) >> 16) | (uint32_t)s.zero;
    return s;
}
__device__ __forceinline__ uint32_t code_of(float x, const Scale& s, bool bad) {
    return bad ? 0u : (uint32_t)fminf(fmaxf(rintf(quotient(x, s.step, s.inverse)) + s.zero, 0.f), 15.f);
}
// (false for NaN)
__device__ __forceinline__ bool holds(float x) { return fabsf(x) < 1.7014118346046923e38f; }     // 2^127

// Every entry point's checks of the cache's geometry.
inline bool sizes_ok(int d, int page_size) { return d > 0 && d % kGroup == 0 && d <= kMaxHeadDim && page_size > 0 && page_size % kBlock == 0; }

}  // namespace kv4
}  // namespace cib
