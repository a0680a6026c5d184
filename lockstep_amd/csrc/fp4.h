// Pages of keys and values held in 4 bits: their layout, and the way from codes to values.
//
// A head's key or value of one token is cut into groups of 32 elements.  A group whose largest magnitude is a has the scale
// 2^e, e = floor(log2 a) - 2 (at least -125, so that the smallest value stays a normal number), held as the byte e + 127;
// an element x is held as the code of x / 2^e rounded to the nearest of 0, 1/2, 1, 3/2, 2, 3, 4, 6 (ties to the even code;
// what lies beyond 6 becomes 6), the sign in the fourth bit.  These are the element and the scale of the open
// microscaling format with blocks of 32, which gfx950 converts two elements an instruction; every value has two
// significant bits, so it is exact in bfloat16.  A group with an infinity or a NaN has the scale byte 255, and all of it
// reads as NaN.
//
//   key codes     [pages][kv heads][tokens][d / 2]           two elements a byte, the lower one in the low half
//   key scales    [pages][kv heads][tokens][d / 32]
//   value codes   [pages][kv heads][tokens / 4][d / 8][4][4]  blocks of four tokens by eight elements: four bytes a token
//   value scales  [pages][kv heads][tokens / 4][d / 32][4]
//
// A product over the keys' elements wants a run of elements of one token in a lane, one over the tokens wants the same
// element of several tokens: with these blocks both read 16 bytes a lane, 1 KiB in a row for 16 tokens of a head of 128,
// and no tile passes through LDS.
#pragma once

#include "common.h"

namespace ls {

constexpr int kFp4Group = 32;
constexpr unsigned int kFp4Nan = 255u;  // scale byte of a group that is not finite

typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
typedef __attribute__((ext_vector_type(2))) float f32x2_t;

struct Fp4Pool {  // strides in bytes
  const unsigned char* k_codes;
  const unsigned char* k_scales;
  const unsigned char* v_codes;
  const unsigned char* v_scales;
  int pages, page_shift, kv_heads;
};

// The float whose value is that of a scale byte (0: 0, beyond what a write leaves).
__device__ __forceinline__ float fp4_scale(unsigned int byte) { return __uint_as_float(byte << 23); }

// Elements 2 B and 2 B + 1 of eight codes.
template <int B> __device__ __forceinline__ unsigned int fp4_pair(unsigned int codes, float scale) {
  return __builtin_bit_cast(unsigned int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, B));
}

}  // namespace ls
