// A cache of keys and values held in 4 bits: microscaled floating point, 32 neighbouring elements of a row with one scale.
//
// An element is a code of 4 bits (sign, 2 bits of exponent, 1 of fraction: 0, 0.5, 1, 1.5, 2, 3, 4, 6), a scale a byte s that
// stands for 2^(s - 127); 255 stands for NaN, as which a block with an infinity or a NaN is held.  A block's s - 127 is
// floor(log2(largest magnitude)) - 2, so that its largest element lies in [4, 8) of its steps (beyond 6 it is held as 6), and
// at least -124: every value that is not zero is then a normal bfloat16.
//
// A page's part of one kv head holds 64 tokens of head size 32 m in 68 * 32 m bytes, one block of memory: codes of the keys
// [64 tokens][16 m bytes], their scales [16][m][4], codes of the values [8][4 m][8 tokens][4 bytes], their scales
// [8][m][8 tokens].  The low half of a byte comes first.  The orders are the matrix instructions' operands:
//  * S^T = K Q^T takes keys as rows of A: a lane reads neighbouring codes of one token.  Row c of 16-row tile j of a page is token
//    32 (j / 2) + 8 (c / 4) + 4 (j % 2) + c % 4, so that the lane's scores of two tiles are 8 neighbouring tokens; the scales of a lane's
//    rows in the page's four tiles are one 4-byte word.
//  * O^T = V^T P^T takes values as columns: 8 neighbouring tokens of 8 channels are 32 bytes, their 8 scales 8 bytes.
#pragma once
#include "common.h"

#define KV4_PAGE 64

// Offsets in a head's part of a page, M = head size / 32
template <int M> struct kv4_layout {
    static constexpr int HD = 32 * M;
    static constexpr int KC = 0, KS = 1024 * M, VC = 1088 * M, VS = 2112 * M, BYTES = 2176 * M;
};
__device__ __forceinline__ int kv4_key_scale(int t, int blk, int m) {       // place of a key's scale behind KS
    return ((4 * ((t & 31) >> 3) + (t & 3)) * m + blk) * 4 + 2 * (t >> 5) + ((t >> 2) & 1);
}

typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

// 2^(s - 127) as a float; 255 gives infinity, which the conversions below take as NaN (as they do NaN).  They look at the exponent of
// their scale only: what stands in its sign and fraction does not matter (65,536 words of random bits), so that a byte of a
// word of scales needs a shift and no mask.
__device__ __forceinline__ float kv4_scale(unsigned s) { return __uint_as_float(s << 23); }

__device__ __forceinline__ float kv4_scale_of(unsigned word, int byte) { return __uint_as_float(byte < 3 ? word << (23 - 8 * byte) : word >> 1); }

// 8 codes of a word as bfloat16, times `scale`
__device__ __forceinline__ bf16x8 kv4_to_bf16(unsigned w, float scale) {
    bf16x8 v;
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3);
    v[0] = a[0]; v[1] = a[1]; v[2] = b[0]; v[3] = b[1]; v[4] = c[0]; v[5] = c[1]; v[6] = d[0]; v[7] = d[1];
    return v;
}

// Byte B of a word (two channels of one token) and of the next token's word, each with its token's scale -> the two
// channels' values of both tokens, pairs along the tokens: lo = channel 0 of (a, b), hi = channel 1.
template <int B>
__device__ __forceinline__ void kv4_pair(unsigned a, float sa, unsigned b, float sb, unsigned& lo, unsigned& hi) {
    const unsigned x = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(a, sa, B));
    const unsigned y = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(b, sb, B));
    lo = __builtin_amdgcn_perm(y, x, 0x05040100u);
    hi = __builtin_amdgcn_perm(y, x, 0x07060302u);
}
