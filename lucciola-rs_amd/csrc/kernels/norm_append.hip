// RMS norm of q's and k's heads, RoPE and the paged cache write of one row per new token, in
// one pass (gfx950), into a 16-bit pool or a 4-bit one:
//   x = q or k head (+ bias), f32
//   y = (x * inv) * w,  inv = 1 / sqrt(mean(x^2) + eps)       (norms given; else y = x)
//   q_out, k = round(y1 c - y2 s | y1 s + y2 c)               (halves y1, y2; cos, sin of the position)
//   v = round(v + bias)
// and k, v to the slot of the row.  The rotation rounds each product and the sum separately
// (contraction off): without norms q_out and a 16-bit pool get the bits of luc_rope_append
// (the reference's rope, src/kernels/rope.cu:31-52, and update_kv_cache_kernel,
// src/kernels/kv_cache.cu:3-59).  The norm is of f32 values and nothing is rounded between it and
// the rotation's result.
//
// 4 bits: of a group's 32 (16-bit) values, clamped to +-kKv4Limit,
//   m = fp16(min), s = fp16((max - m) / 15), n = rint((x - m) / s) in 0 .. 15,
// all in f32 with IEEE divisions, so that n is a function of the 16-bit values; s = m = NaN where a
// value is NaN.  k_out and v_out get n * s + m.
//
// Lanes.  A head takes D / 16 lanes; a lane has elements 8 c .. 8 c + 7 and the same plus
// D / 2 (a rotation's partners), and four lanes a group of the low and one of the high half: sums and
// extremes of a head are DPP steps inside 4 or 8 lanes, no LDS.
//
// Order.  All of q, row by row; then k, then v, head by head: a wave has one kind, so that only those
// of k and v encode, and the rows of a page, which are mostly neighbours, write V's two bytes a token
// side by side.  4100 rows of 14 + 2 x 2 heads of 64 into 4 bits: 7.8 us, 11.0 head by head of a row.
//
// What bounds it.  8191 rows of 28 + 2 x 4 heads of 128, 16 bits: 35 us for 155 MB from HBM (4.4 TB/s; a copy of as
// many bytes 31), 26.7 on buffers that the last-level cache holds from call to call (the copy 22);
// 32 rows of 14 + 2 x 2 of 64: 3.4 us, 64 rows of 28 + 2 x 4 of 128 into 4 bits 4.9 us, the latency
// of a launch and of position -> row of the table -> slot.
#include "kv4.h"

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

// A group of 32 values, 8 a lane over a quad: n in one dword (element i in bits 4 i), (s, m) as two
// fp16 in another, x the values that they stand for.
__device__ inline void kv4_encode(float* x, uint32_t& n, uint32_t& sm) {
#pragma clang fp contract(off)
  float lo = kKv4Limit, hi = -kKv4Limit;
  float nan = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if (__builtin_isnan(x[e])) nan = 1.0f;
    x[e] = fminf(fmaxf(x[e], -kKv4Limit), kKv4Limit);
    lo = fminf(lo, x[e]);
    hi = fmaxf(hi, x[e]);
  }
  nan = quad_max(nan);
  lo = quad_min(lo);
  hi = quad_max(hi);
  const _Float16 mh = (_Float16)lo;
  const float m = (float)mh;
  const _Float16 sh = (_Float16)fmaxf((hi - m) / 15.0f, 0.0f);
  const float s = (float)sh;
  n = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float q = s > 0.0f ? rintf((x[e] - m) / s) : 0.0f;
    const float c = fminf(fmaxf(q, 0.0f), 15.0f);
    n |= (uint32_t)c << (4 * e);
    x[e] = c * s + m;
  }
  sm = (uint32_t)__builtin_bit_cast(uint16_t, sh) | (uint32_t)__builtin_bit_cast(uint16_t, mh) << 16;
  if (nan != 0.0f) {
    n = 0;
    sm = 0x7e007e00u;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = __builtin_nanf("");
  }
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

template <int DT, int D, bool POOL4>
__device__ void norm_append_impl(const NormAppendArgs& A) {
#pragma clang fp contract(off)
  constexpr int LANES = D / 16;
  uint32_t unit = (blockIdx.x * blockDim.x + threadIdx.x) / LANES;  // (the grid's threads fit 32 bits)
  const int c = threadIdx.x % LANES;
  const uint32_t nq = (uint32_t)A.rows * A.hq, nk = (uint32_t)A.rows * A.hkv;
  if (unit >= nq + 2 * nk) return;
  const int kind = unit < nq ? 0 : unit < nq + nk ? 1 : 2;  // q, k, v
  int row, hh;
  if (kind == 0) {
    row = unit / A.hq;
    hh = unit % A.hq;
  } else {
    unit -= kind == 1 ? nq : nq + nk;
    hh = unit / A.rows;
    row = unit % A.rows;
  }
  const int pos = A.positions[row];
  if (pos < 0 || pos >= A.max_pos) return;
  const uint16_t* src = pick(kind, A.q, A.k, A.v);
  const uint16_t* const bias = pick(kind, A.q_bias, A.k_bias, A.v_bias);
  src += row * A.row_stride + hh * D;
  const uint4 r1 = *(const uint4*)(src + 8 * c), r2 = *(const uint4*)(src + D / 2 + 8 * c);
  float x[16];
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
  uint4 o1 = pack8<DT>(x), o2 = pack8<DT>(x + 8);
  if (kind == 0) {
    uint16_t* const o = A.q_out + row * A.q_out_stride + hh * D;
    *(uint4*)(o + 8 * c) = o1;
    *(uint4*)(o + D / 2 + 8 * c) = o2;
    return;
  }
  const int64_t slot = A.slots[row];
  const bool write = slot >= 0 && slot < A.num_slots;
  const int t = (int)(slot & (kPage - 1));
  const int64_t slab = ((slot >> 4) * A.num_layers + A.layer) * A.hkv + hh;
  if constexpr (!POOL4) {
    if (write) {
      uint16_t* const p = (uint16_t*)pick(kind, A.k_pool, A.k_pool, A.v_pool) + slab * (kPage * D) + t * D;
      *(uint4*)(p + 8 * c) = o1;
      *(uint4*)(p + D / 2 + 8 * c) = o2;
    }
  } else {
    // of the 16-bit values
    unpack8<DT>(o1, x);
    unpack8<DT>(o2, x + 8);
    uint32_t n1, n2, sm1, sm2;
    kv4_encode(x, n1, sm1);
    kv4_encode(x + 8, n2, sm2);
    if (write) {
      char* const p = (char*)pick(kind, A.k_pool, A.k_pool, A.v_pool) + slab * Kv4<D>::kSlab;
      const int g1 = c / 4, g2 = g1 + Kv4<D>::kGroups / 2;
      if (kind == 1) {
        *(uint32_t*)(p + Kv4<D>::k_row(t) + 4 * c) = n1;
        *(uint32_t*)(p + Kv4<D>::k_row(t) + 4 * c + D / 4) = n2;
        if (c % 4 == 0) {
          *(uint32_t*)(p + Kv4<D>::k_scale(t, g1)) = sm1;
          *(uint32_t*)(p + Kv4<D>::k_scale(t, g2)) = sm2;
        }
      } else {
        *(uint16_t*)(p + Kv4<D>::v_quad(t, 2 * c)) = (uint16_t)n1;
        *(uint16_t*)(p + Kv4<D>::v_quad(t, 2 * c + 1)) = (uint16_t)(n1 >> 16);
        *(uint16_t*)(p + Kv4<D>::v_quad(t, 2 * c + D / 8)) = (uint16_t)n2;
        *(uint16_t*)(p + Kv4<D>::v_quad(t, 2 * c + D / 8 + 1)) = (uint16_t)(n2 >> 16);
        if (c % 4 == 0) {
          char* const a = p + Kv4<D>::v_scale(t >> 3, g1) + (t & 7) * 2;
          char* const b = p + Kv4<D>::v_scale(t >> 3, g2) + (t & 7) * 2;
          *(uint16_t*)a = (uint16_t)sm1;
          *(uint16_t*)(a + 16) = (uint16_t)(sm1 >> 16);
          *(uint16_t*)b = (uint16_t)sm2;
          *(uint16_t*)(b + 16) = (uint16_t)(sm2 >> 16);
        }
      }
    }
    o1 = pack8<DT>(x);
    o2 = pack8<DT>(x + 8);
  }
  uint16_t* o = pick(kind, A.k_out, A.k_out, A.v_out);
  if (o) {
    o += row * A.kv_out_stride + hh * D;
    *(uint4*)(o + 8 * c) = o1;
    *(uint4*)(o + D / 2 + 8 * c) = o2;
  }
}

}  // namespace luc

#define LUC_NORM_APPEND(DTN, DT, D)                                                             \
  extern "C" __global__ __launch_bounds__(256) void luc_norm_append_##DTN##_d##D(               \
      luc::NormAppendArgs a) {                                                                  \
    luc::norm_append_impl<luc::DT, D, false>(a);                                                \
  }                                                                                             \
  extern "C" __global__ __launch_bounds__(256) void luc_norm_append4_##DTN##_d##D(              \
      luc::NormAppendArgs a) {                                                                  \
    luc::norm_append_impl<luc::DT, D, true>(a);                                                 \
  }
LUC_NORM_APPEND(bf16, kBF16, 64)
LUC_NORM_APPEND(bf16, kBF16, 128)
LUC_NORM_APPEND(f16, kF16, 64)
LUC_NORM_APPEND(f16, kF16, 128)
