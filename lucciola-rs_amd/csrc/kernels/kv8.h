// The 8-bit K/V cache: layout and arithmetic shared by its append, reads, attention and page selection.
//
// Values.  A value is code * scale, the code in e4m3 (largest 448, subnormals from 2^-9, no infinities).  The
// tokens of a page share, for one kv head, one scale of K and one of V: powers of two, the smallest that bring the
// page's largest value to at most 448.  A float code's relative precision is the same under any scale, so
// powers of two lose nothing, a page whose scale grows only moves its codes' exponents (exact but for
// subnormals), and to 16 bits a code goes in one v_cvt_scalef32_pk_*_fp8, scale included.
//
// Pools.  [page][layer][kv head] slabs of 16 * D bytes, in the operand order of v_mfma_f32_16x16x32 (f16, bf16):
//   K (A operand, a lane holds dimensions of one token): [16 tokens][D].
//   V (A operand of the transposed product, a lane holds tokens of one dimension): [4 fours of tokens][D][4 tokens],
//     so that a dword is four tokens of one dimension and 16 bytes of a lane four dimensions.
// Scales [page][layer][kv head][K, V] in f32.  Key bounds [page][layer][kv head][largest, smallest][D]: by
// dimension, of the codes that the page took in since it began (a NaN counts as 0).
#pragma once
#include "luc_common.h"

namespace luc {

constexpr float kKv8Limit = 60000.0f;  // K and V beyond it are stored as it: code * scale stays below fp16's 65504
constexpr int kKv8LeastExp = -64;      // of a scale: 2^-73, its smallest value, is far from bf16's subnormals

template <int D> struct Kv8 {
  static constexpr int kSlab = 16 * D;  // bytes of a (page, layer, kv head)
  // K, dimension i of token t; V, dimension i of tokens 4 q .. 4 q + 3
  __device__ static inline int k_at(int t, int i) { return t * D + i; }
  __device__ static inline int v_at(int q, int i) { return (q * D + i) * 4; }
};

__device__ inline float pow2f(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
__device__ inline int exp2of(float x) { return (int)(__float_as_uint(x) >> 23 & 0xff) - 127; }  // of a power of two

// The smallest e with amax <= 448 * 2^e (1.75 * 2^8; amax finite, not negative), at least kKv8LeastExp.
__device__ inline int kv8_exponent(float amax) {
  const uint32_t u = __float_as_uint(amax);
  return max((int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0), kKv8LeastExp);
}

// Four values to codes, nearest even, and back.
__device__ inline uint32_t kv8_encode4(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
  return (uint32_t)w;
}
__device__ inline float4 kv8_decode4(uint32_t w) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  return make_float4(lo[0], lo[1], hi[0], hi[1]);
}
// Codes of a page whose scale grew by 2^-less: f = 2^less.
__device__ inline uint32_t kv8_rescale4(uint32_t w, float f) {
  const float4 x = kv8_decode4(w);
  return kv8_encode4(x.x * f, x.y * f, x.z * f, x.w * f);
}
// Codes 2 i, 2 i + 1 of a dword times a scale, as two 16-bit values.
template <int DT, bool HI>
__device__ inline uint32_t kv8_pair(uint32_t w, float scale) {
  if constexpr (DT == kF16)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, HI));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, HI));
}

}  // namespace luc
