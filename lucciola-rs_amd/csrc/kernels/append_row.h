// A new token's head on its way to a paged cache: what the appends share (gfx950).
#pragma once
#include "luc_common.h"

namespace luc {

struct NormAppendArgs {
  const uint16_t* q;  // row r at q + r * row_stride, likewise k, v
  const uint16_t* k;
  const uint16_t* v;
  int64_t row_stride;
  const uint16_t* q_bias;
  const uint16_t* k_bias;
  const uint16_t* v_bias;
  const uint16_t* q_norm;  // [D], both or neither
  const uint16_t* k_norm;
  const float* cos_t;      // [max_pos][D / 2]
  const float* sin_t;
  const int32_t* positions;
  const int64_t* slots;
  uint16_t* q_out;
  int64_t q_out_stride;
  uint16_t* k_out;         // or null
  uint16_t* v_out;         // 4 bits only, or null
  int64_t kv_out_stride;
  void* k_pool;
  void* v_pool;
  int64_t num_slots;
  float eps;
  int32_t rows, max_pos, layer, num_layers, hq, hkv;
};

// Sum, minimum and maximum over the 4 or 8 lanes of a head, alike in each.
template <int LANES>
__device__ inline float head_sum(float x) {
  x += dpp_mov<kDppQuadXor1>(x);
  x += dpp_mov<kDppQuadXor2>(x);
  if (LANES == 8) x += dpp_mov<kDppHalfMirror>(x);
  return x;
}
__device__ inline float quad_min(float x) {
  x = fminf(x, dpp_mov<kDppQuadXor1>(x));
  return fminf(x, dpp_mov<kDppQuadXor2>(x));
}
__device__ inline float quad_max(float x) {
  x = fmaxf(x, dpp_mov<kDppQuadXor1>(x));
  return fmaxf(x, dpp_mov<kDppQuadXor2>(x));
}

template <int DT>
__device__ inline void unpack8(const uint4& v, float* x) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = St<DT>::lo(w[i]);
    x[2 * i + 1] = St<DT>::hi(w[i]);
  }
}
template <int DT>
__device__ inline uint4 pack8(const float* x) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (DT == kBF16) {
      typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
      const bf16x2 p = {(__bf16)x[2 * i], (__bf16)x[2 * i + 1]};
      w[i] = __builtin_bit_cast(uint32_t, p);
    } else {
      const half2_t p = {(_Float16)x[2 * i], (_Float16)x[2 * i + 1]};
      w[i] = __builtin_bit_cast(uint32_t, p);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// a, b or c by kind 0, 1, 2 (by value: an address chosen per lane would put the arguments in
// scratch)
template <class T>
__device__ inline T* pick(int kind, T* a, T* b, T* c) {
  uint64_t r = (uint64_t)a;
  r = kind == 1 ? (uint64_t)b : r;
  r = kind == 2 ? (uint64_t)c : r;
  asm("" : "+v"(r));
  return (T*)r;
}

// Row `row`'s head hh of q, k or v (kind 0, 1, 2): the lane's elements 8 c .. 8 c + 7 and the same plus D / 2,
// with bias, norm and rotation at position pos, in f32.  Each product and sum of the rotation is rounded by
// itself (contraction off).
template <int DT, int D>
__device__ __attribute__((always_inline)) inline void append_head(const NormAppendArgs& A, int kind, int row, int hh, int c, int pos, float (&x)[16]) {
#pragma clang fp contract(off)
  constexpr int LANES = D / 16;
  const uint16_t* src = pick(kind, A.q, A.k, A.v);
  const uint16_t* const bias = pick(kind, A.q_bias, A.k_bias, A.v_bias);
  src += row * A.row_stride + hh * D;
  const uint4 r1 = *(const uint4*)(src + 8 * c), r2 = *(const uint4*)(src + D / 2 + 8 * c);
  unpack8<DT>(r1, x);
  unpack8<DT>(r2, x + 8);
  if (bias) {
    float b[16];
    unpack8<DT>(*(const uint4*)(bias + hh * D + 8 * c), b);
    unpack8<DT>(*(const uint4*)(bias + hh * D + D / 2 + 8 * c), b + 8);
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] = x[e] + b[e];
  }
  if (kind != 2) {
    const uint16_t* const norm = pick(kind, A.q_norm, A.k_norm, A.k_norm);
    if (norm) {
      float s = 0.0f;
#pragma unroll
      for (int e = 0; e < 16; ++e) s = fmaf(x[e], x[e], s);
      s = head_sum<LANES>(s);
      const float inv = 1.0f / sqrtf(s / (float)D + A.eps);
      float w[16];
      unpack8<DT>(*(const uint4*)(norm + 8 * c), w);
      unpack8<DT>(*(const uint4*)(norm + D / 2 + 8 * c), w + 8);
#pragma unroll
      for (int e = 0; e < 16; ++e) x[e] = (x[e] * inv) * w[e];
    }
    const float4* const cr = (const float4*)(A.cos_t + (int64_t)pos * (D / 2) + 8 * c);
    const float4* const sr = (const float4*)(A.sin_t + (int64_t)pos * (D / 2) + 8 * c);
    const float4 c0 = cr[0], c1 = cr[1], s0 = sr[0], s1 = sr[1];
    const float cs[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
    const float sn[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float p = x[e] * cs[e], r = x[e + 8] * sn[e];
      const float m = x[e] * sn[e], n = x[e + 8] * cs[e];
      x[e] = p - r;
      x[e + 8] = m + n;
    }
  }
}

}  // namespace luc
