// The cache of keys and values in 4 bits.
//
// 32 neighbouring features of one token and kv head are a group with two bfloat16 numbers: S = (hi - lo) 16 / 15 and B = lo - S of its
// largest and smallest feature, each rounded once.  A code c of 0 to 15 stands for the bfloat16 nearest to B + S (1 + c / 16): 1 + c / 16 is a
// bfloat16 whose four upper mantissa bits are c, so a shift, a mask and one fused multiply-add of two numbers give two values, and B,
// rounded at about S's size, misses lo by no more than half of its own last bit.  A feature x takes the code nearest to 16 (x - B) / S - 16 (ties to even).
// A group whose S would be below 2^-100 holds B = lo and codes of 0 (S = 0).  A group is not finite where a feature is an infinity or a NaN, where bfloat16 cannot
// hold S or B, or where B + S (1 + 15 / 16) rounds to an infinity (S and B are finite then, hi is within a few steps of bfloat16's largest number).  A token whose key
// or value (of one kv head) has such a group has NaN for all S and B of that key, and zeros for the groups of its value that are not finite: a query that sees the
// token gets NaN, and one that does not meets finite values only.
//
// A page of a kv head is one run of page_size * D * 5 / 8 bytes: the codes of all its tokens (D / 2 bytes each, byte j feature 2j in
// the low half and 2j + 1 in the high one), then their groups' (S, B) pairs (D / 8 bytes each).  Codes and pairs lie apart, so that a
// warp which takes eight tokens' codes, or their pairs, reads runs without gaps.
#pragma once

#include "common.cuh"

namespace {

constexpr int kGroup = 32;

__host__ __device__ constexpr size_t kv4_block_bytes(int page_size, int D) { return (size_t)page_size * D / 8 * 5; }

// two codes at bits 3-6 of both halves of w -> two values; S and B twice each
__device__ __forceinline__ uint32_t kv4_fma(uint32_t w, uint32_t S2, uint32_t B2) {
    uint32_t one, v;
    asm("lop3.b32 %0, %1, 0x00780078, 0x3f803f80, 0xea;" : "=r"(one) : "r"(w));  // (w & mask) | 1.0
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(v) : "r"(one), "r"(S2), "r"(B2));
    return v;
}
// the eight codes of a word as values: out[p] = features (p, p + 4) of the word
__device__ __forceinline__ void kv4_word(uint32_t w, uint32_t S2, uint32_t B2, uint32_t (&out)[4]) {
    uint32_t up;  // w << 3, in the multiplier's pipe: the logic pipe, at half of the issue rate, is what bounds a kernel that does little else than unpack
    asm("mad.lo.u32 %0, %1, 8, 0;" : "=r"(up) : "r"(w));
    out[0] = kv4_fma(up, S2, B2);
    out[1] = kv4_fma(w >> 1, S2, B2);
    out[2] = kv4_fma(w >> 5, S2, B2);
    out[3] = kv4_fma(w >> 9, S2, B2);
}
// a group's pair (S in the low half) as S twice and B twice
__device__ __forceinline__ void kv4_pair(uint32_t pair, uint32_t& S2, uint32_t& B2) {
    S2 = __byte_perm(pair, pair, 0x1010);
    B2 = __byte_perm(pair, pair, 0x3232);
}
// a word's eight values in the features' order
__device__ __forceinline__ uint4 kv4_in_order(uint32_t w, uint32_t pair) {
    uint32_t S2, B2, p[4];
    kv4_pair(pair, S2, B2);
    kv4_word(w, S2, B2, p);
    return make_uint4(__byte_perm(p[0], p[1], 0x5410), __byte_perm(p[2], p[3], 0x5410), __byte_perm(p[0], p[1], 0x7632), __byte_perm(p[2], p[3], 0x7632));
}
__device__ __forceinline__ float2 kv4_floats(uint32_t v) { return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u)); }

}  // namespace
