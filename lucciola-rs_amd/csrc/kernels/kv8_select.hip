// The pages of a long context that a new row attends to, chosen by a score over the key bounds of kv8.h
// (gfx950): of one row each of a batch of sequences, for every kv head, the `budget` pages that score highest, the first
// `first` and the last `recent` pages always among them, equal scores to the lower page; ascending.
//
// Score.  Of a page's keys k, q . k = sum_i q_i k_i is at most sum_i (q_i > 0 ? q_i max_i : q_i min_i).  q in 8 bits: of
// every 32 dimensions j of a head, n = rint(q 2^-e_j) with the smallest e_j that brings them to at most 127; the bounds in
// whole code units, |max|, |min| <= 448.  A group's sum over its 32 dimensions is then a whole number below
// 32 * 127 * 448 < 2^21, exact on the matrix unit in any order; and
//   score = max over the group's heads of (((S_0 2^e_0 + S_1 2^e_1) + S_2 2^e_2) + S_3 2^e_3) * scale_K
// rounds its few sums in f32, in that order: the choice is a function of the inputs, whatever computes it.
//
// A workgroup scores 128 pages of one (sequence, kv head); the last of them to arrive picks.  Lane (n, g) of a wave loads
// bounds 64 i + 16 g .. + 15 of page n of 16; those belong to group 2 i + g / 2, so of the 16 columns of
// v_mfma_f32_16x16x32_f16 the lower 8 take the heads' even groups (q is 0 in lanes of the odd ones) and the upper
// 8 the same heads' odd groups.
//
// The pick.  Scores become whole numbers of the same order (keys).  The budget'th largest is found 8 bits at a time by
// a histogram in LDS; then every wave goes through its quarter of the pages in order and writes those above, and of those
// equal to it the first, to their places.
#include "kv8.h"
#include "kv_split.h"

namespace luc {

struct Kv8SelectArgs {
  const uint16_t* q;
  int64_t q_stride;
  const uint8_t* bounds;
  const float2* scales;
  const int32_t* tables;
  int64_t table_stride;
  const int32_t* cu_seqlens;  // or null: row b is sequence b's
  const int32_t* start_pos;
  int32_t* pages;             // [batch][hkv][budget]
  int32_t* ws_cnt;
  uint32_t* ws_key;           // [batch][hkv][max_pages]
  int32_t batch, total_rows, max_rows, max_ctx, layer, num_layers, hkv, group, num_blocks;
  int32_t budget, first, recent, chunks, max_pages;
};

constexpr int kSelWaves = 4;
constexpr int kSelTiles = 2;                                 // of 16 pages a wave
constexpr int kSelChunk = kSelWaves * kSelTiles * 16;        // pages of a workgroup
constexpr int kSelLdsKeys = 8192;                            // keys of a pick that LDS holds

// Whole numbers as packed fp16: codes rounded to units.  |x| <= 448, and from 1024 to 2048 fp16 has no fractions.
__device__ inline uint32_t whole2(uint32_t w) {
  const half2_t big = {(_Float16)1536.0f, (_Float16)1536.0f};
  half2_t x = __builtin_bit_cast(half2_t, w);
  x = x + big;
  asm("" : "+v"(x));  // (not folded)
  return __builtin_bit_cast(uint32_t, (half2_t)(x - big));
}
__device__ inline uint4 whole8(uint32_t a, uint32_t b) {
  return make_uint4(whole2(kv8_pair<kF16, false>(a, 1.0f)), whole2(kv8_pair<kF16, true>(a, 1.0f)),
                    whole2(kv8_pair<kF16, false>(b, 1.0f)), whole2(kv8_pair<kF16, true>(b, 1.0f)));
}
__device__ inline f32x4_t mfma_f16(uint4 a, uint4 b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// A score's place in the order of whole numbers, below the highest one, which belongs to pages that are always chosen.
__device__ inline uint32_t score_key(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);  // (-0 is 0)
  const uint32_t k = u ^ (u >> 31 ? ~0u : 0x80000000u);
  return __builtin_isnan(x) ? 0u : k;
}

template <int DT, int D>
__device__ void kv8_select_impl(const Kv8SelectArgs& A) {
  constexpr int H = D / 64;
  __shared__ uint32_t s_key[kSelLdsKeys];
  __shared__ uint32_t s_hist[256];
  __shared__ uint32_t s_pick[4];  // bits of the key so far, how many are wanted among those that share them
  __shared__ int s_count[kSelWaves][2], s_last;
  // neighbours on one XCD (block x runs on XCD x % 8): the kv heads of the same pages, whose bounds lie side by side
  const int units = A.batch * A.chunks;  // (padded to whole eights)
  const int u = blockIdx.x / (8 * A.hkv) * 8 + blockIdx.x % 8, kvh = blockIdx.x / 8 % A.hkv;
  if (u >= units) return;
  const int b = u % A.batch, chunk = u / A.batch;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const KvSeq S = kv_seq(A, b);
  int32_t* const out = A.pages + ((int64_t)b * A.hkv + kvh) * A.budget;
  const int count = S.ctx == 0 || S.rows == 0 ? 0 : S.start / kPage + 1;  // pages of the context
  if (count <= A.budget) {  // all of them, or none
    if (chunk == 0)
      for (int i = threadIdx.x; i < A.budget; i += 64 * kSelWaves) out[i] = i < count ? i : -1;
    return;
  }
  const int chunks = (count + kSelChunk - 1) / kSelChunk;
  if (chunk >= chunks) return;
  uint32_t* const keys = A.ws_key + ((int64_t)b * A.hkv + kvh) * A.max_pages;

  // ---- scores of 16 pages at a time
  {
    const int n = lane & 15, g = lane >> 4, p0 = chunk * kSelChunk + w * (16 * kSelTiles);
    const int32_t* const table = A.tables + (int64_t)b * A.table_stride;
    const int64_t base = (int64_t)A.layer * A.hkv + kvh;
    const int64_t stride = (int64_t)A.num_layers * A.hkv;
    int page[kSelTiles];
#pragma unroll
    for (int t = 0; t < kSelTiles; ++t) page[t] = p0 + 16 * t + n < count ? table[p0 + 16 * t + n] : 0;
    // q of head n % 8, dimensions 64 i + 16 g + 8 k .. + 7
    const int head = n & 7;
    const bool on = head < A.group;
    const uint16_t* const src = A.q + (int64_t)S.row0 * A.q_stride + ((int64_t)kvh * A.group + (on ? head : 0)) * D + 16 * g;
    uint4 raw[H][2];
#pragma unroll
    for (int i = 0; i < H; ++i)
#pragma unroll
      for (int k = 0; k < 2; ++k) raw[i][k] = on ? *(const uint4*)(src + 64 * i + 8 * k) : make_uint4(0, 0, 0, 0);
    bool bad[kSelTiles];
    uint4 hi[kSelTiles][H], lo[kSelTiles][H];
    float scale[kSelTiles];
#pragma unroll
    for (int t = 0; t < kSelTiles; ++t) {
      // a page outside the pool is never an address: page 0 is read instead, and the page comes last
      bad[t] = page[t] < 0 || page[t] >= A.num_blocks;
      const int64_t at = (int64_t)(bad[t] ? 0 : page[t]) * stride + base;
      const uint8_t* const p = A.bounds + at * (2 * D) + 16 * g;
#pragma unroll
      for (int i = 0; i < H; ++i) {
        hi[t][i] = *(const uint4*)(p + 64 * i);
        lo[t][i] = *(const uint4*)(p + D + 64 * i);
      }
      scale[t] = A.scales[at].x;
    }
    uint4 qp[H][2], qn[H][2];  // n where it is positive, and where it is negative
    float unit[H];             // of the lane's column: group 2 i + n / 8
    const bool mine = (g >> 1) == (n >> 3);
#pragma unroll
    for (int i = 0; i < H; ++i) {
      float x[16], top = 0.0f;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const uint32_t ww[4] = {raw[i][k].x, raw[i][k].y, raw[i][k].z, raw[i][k].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[8 * k + 2 * e] = St<DT>::lo(ww[e]);
          x[8 * k + 2 * e + 1] = St<DT>::hi(ww[e]);
        }
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        x[e] = __builtin_isnan(x[e]) ? 0.0f : fminf(fmaxf(x[e], -kKv8Limit), kKv8Limit);
        top = fmaxf(top, fabsf(x[e]));
      }
      top = fmaxf(top, __shfl_xor(top, 16));  // lanes g and g ^ 1: a group of 32 dimensions
      const uint32_t bits = __float_as_uint(top);  // the smallest e with top <= 127 * 2^e (1.984375 * 2^6)
      const int e = max((int)(bits >> 23) - 127 - 6 + ((bits & 0x7fffffu) > 0x7e0000u ? 1 : 0), kKv8LeastExp);
      const float down = pow2f(-e);
      unit[i] = __shfl(pow2f(e), (lane & 15) | (n >> 3) << 5);  // of the column's group: lanes g = 0, 1 or 2, 3
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        uint32_t wp[4], wn[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float y = rintf(x[8 * k + 2 * r] * down), z = rintf(x[8 * k + 2 * r + 1] * down);
          const half2_t pos = {(_Float16)fmaxf(y, 0.0f), (_Float16)fmaxf(z, 0.0f)};
          const half2_t neg = {(_Float16)fminf(y, 0.0f), (_Float16)fminf(z, 0.0f)};
          wp[r] = mine ? __builtin_bit_cast(uint32_t, pos) : 0u;
          wn[r] = mine ? __builtin_bit_cast(uint32_t, neg) : 0u;
        }
        qp[i][k] = make_uint4(wp[0], wp[1], wp[2], wp[3]);
        qn[i][k] = make_uint4(wn[0], wn[1], wn[2], wn[3]);
      }
    }
#pragma unroll
    for (int t = 0; t < kSelTiles; ++t) {
      f32x4_t sum[H];
#pragma unroll
      for (int i = 0; i < H; ++i) {
        sum[i] = (f32x4_t){0, 0, 0, 0};
        sum[i] = mfma_f16(whole8(hi[t][i].x, hi[t][i].y), qp[i][0], sum[i]);
        sum[i] = mfma_f16(whole8(hi[t][i].z, hi[t][i].w), qp[i][1], sum[i]);
        sum[i] = mfma_f16(whole8(lo[t][i].x, lo[t][i].y), qn[i][0], sum[i]);
        sum[i] = mfma_f16(whole8(lo[t][i].z, lo[t][i].w), qn[i][1], sum[i]);
      }
      // rows 4 g + r are pages; columns n < 8 the even groups' sums, n >= 8 the odd ones'
      float best[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float score = 0.0f;
#pragma unroll
        for (int i = 0; i < H; ++i) {
          const float own = sum[i][r] * unit[i], other = __shfl_xor(own, 8);
          const float even = n < 8 ? own : other, odd = n < 8 ? other : own;
          score = i == 0 ? even + odd : (score + even) + odd;
        }
        best[r] = on ? score : -INFINITY;
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) best[r] = row_max16(best[r]);
      // lane n < 4 of a row stores page 4 g + n
      const int r = n & 3, at = 4 * g + r, p = p0 + 16 * t + at;
      const float top = r == 0 ? best[0] : r == 1 ? best[1] : r == 2 ? best[2] : best[3];
      const float s = __shfl(scale[t], at);
      const bool none = __shfl((int)bad[t], at);
      if (n < 4 && p < count) {
        const bool always = p < A.first || p >= count - A.recent;
        __hip_atomic_store(keys + p, always ? ~0u : none ? 0u : score_key(top * s), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
    }
  }
  // ---- the last workgroup of the (sequence, kv head) to arrive picks
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0) {
    int32_t* const cnt = A.ws_cnt + b * A.hkv + kvh;
    s_last = __hip_atomic_fetch_add(cnt, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == chunks - 1;
    if (s_last) __hip_atomic_store(cnt, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    s_pick[0] = 0;
    s_pick[1] = A.budget;
  }
  __syncthreads();
  if (!s_last) return;
  const bool lds = count <= kSelLdsKeys;
  auto key = [&](int i) __attribute__((always_inline)) {
    return lds ? s_key[i] : __hip_atomic_load(keys + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  };
  if (lds) {
    for (int i = threadIdx.x; i < count; i += 64 * kSelWaves)
      s_key[i] = __hip_atomic_load(keys + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
  }
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = threadIdx.x; i < 256; i += 64 * kSelWaves) s_hist[i] = 0;
    __syncthreads();
    const uint32_t above = s_pick[0], mask = shift == 24 ? 0u : ~0u << (shift + 8);
    for (int i = threadIdx.x; i < count; i += 64 * kSelWaves) {
      const uint32_t k = key(i);
      if ((k & mask) == above) atomicAdd(&s_hist[k >> shift & 255], 1u);
    }
    __syncthreads();
    if (w == 0) {  // lane l: digits 255 - 4 l and the three below it
      const uint32_t want = s_pick[1];
      uint32_t c[4], sum = 0;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        c[r] = s_hist[255 - 4 * lane - r];
        sum += c[r];
      }
      uint32_t up = sum;  // of the lane's digits and all above
#pragma unroll
      for (int k = 1; k < 64; k <<= 1) {
        const uint32_t y = __shfl_up(up, k);
        if (lane >= k) up += y;
      }
      uint32_t before = up - sum;
      if (before < want && up >= want) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if (before < want && before + c[r] >= want) {
            s_pick[0] = above | (uint32_t)(255 - 4 * lane - r) << shift;
            s_pick[1] = want - before;
            before = want;  // (found)
          } else {
            before += c[r];
          }
        }
      }
    }
    __syncthreads();
  }
  const uint32_t bar = s_pick[0];
  const int want = (int)s_pick[1];  // of those equal to it
  const int span = ((count + kSelWaves - 1) / kSelWaves + 63) / 64 * 64;
  const int from = w * span, to = min(count, from + span);
  int over = 0, same = 0;
  for (int i = from; i < to; i += 64) {
    const uint32_t k = i + lane < to ? key(i + lane) : 0u;
    over += __builtin_popcountll(__ballot(i + lane < to && k > bar));
    same += __builtin_popcountll(__ballot(i + lane < to && k == bar));
  }
  if (lane == 0) {
    s_count[w][0] = over;
    s_count[w][1] = same;
  }
  __syncthreads();
  over = same = 0;
  for (int k = 0; k < w; ++k) {
    over += s_count[k][0];
    same += s_count[k][1];
  }
  const uint64_t below = lane ? ~0ull >> (64 - lane) : 0ull;
  for (int i = from; i < to; i += 64) {
    const uint32_t k = i + lane < to ? key(i + lane) : 0u;
    const uint64_t o = __ballot(i + lane < to && k > bar), e = __ballot(i + lane < to && k == bar);
    const int o_at = over + __builtin_popcountll(o & below), e_at = same + __builtin_popcountll(e & below);
    const bool take = i + lane < to && (k > bar || (k == bar && e_at < want));
    const int to_at = o_at + min(e_at, want);
    if (take) out[to_at] = i + lane;
    over += __builtin_popcountll(o);
    same += __builtin_popcountll(e);
  }
}

}  // namespace luc

#define LUC_KV8_SELECT(DTN, DT, D)                                                               \
  extern "C" __global__ __launch_bounds__(256) void luc_kv8_select_##DTN##_d##D(luc::Kv8SelectArgs a) { \
    luc::kv8_select_impl<luc::DT, D>(a);                                                         \
  }
LUC_KV8_SELECT(bf16, kBF16, 64)
LUC_KV8_SELECT(bf16, kBF16, 128)
LUC_KV8_SELECT(f16, kF16, 64)
LUC_KV8_SELECT(f16, kF16, 128)
