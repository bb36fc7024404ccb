// The 4-bit K/V cache: layout and arithmetic shared by the append and attention kernels.
//
// Values.  32 consecutive dimensions of one token's head are a group with a step s and a
// minimum m, both fp16; a value is n * s + m with n in 0 .. 15.
//
// Pools.  [page][layer][kv head] slabs of 10 * D bytes: 16 tokens, 8 * D bytes of n, then 2 * D
// bytes of (s, m).  The attention kernels read whole slabs with loads of 8 and 16 bytes a lane,
// straight into the operand layout of v_mfma_f32_16x16x32_f16:
//   K (A operand, a lane holds dimensions of one token): n as [16 tokens][D / 2 bytes], dimension
//     2 i in the low half of byte i; (s, m) as [16 tokens][D / 32][2].
//   V (A operand of the transposed product, a lane holds 8 tokens of 4 dimensions): n as
//     [2 octets of tokens][D / 4][8 tokens][2 bytes]: dword i of a 16-byte load is tokens 2 i and 2 i + 1
//     in its halves, four dimensions each; (s, m) as [2 octets][D / 32][s, m][8 tokens], so
//     that a pair of tokens is one packed fp16 operand.
// A token's bytes of n and its scales are whole bytes of its own in both: rows that are
// appended side by side never share one.
#pragma once
#include "luc_common.h"

namespace luc {

constexpr int kKv4Group = 32;
// K and V beyond it are stored as it: 15 s + m stays below fp16's 65504 with s rounded up
constexpr float kKv4Limit = 60000.0f;

template <int D> struct Kv4 {
  static constexpr int kSlab = 10 * D;   // bytes of a (page, layer, kv head)
  static constexpr int kScales = 8 * D;  // offset of (s, m)
  static constexpr int kGroups = D / kKv4Group;
  // K, token t of the page
  __device__ static inline int k_row(int t) { return t * (D / 2); }
  __device__ static inline int k_scale(int t, int g) { return kScales + (t * kGroups + g) * 4; }
  // V, token t: four dimensions from 4 j on
  __device__ static inline int v_quad(int t, int j) { return ((t >> 3) * (D / 4) + j) * 16 + (t & 7) * 2; }
  // V, octet o of tokens: s of its 8 tokens, 16 bytes on their m
  __device__ static inline int v_scale(int o, int g) { return kScales + (o * kGroups + g) * 32; }
};

}  // namespace luc
