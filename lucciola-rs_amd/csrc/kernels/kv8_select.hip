// The pages of a long context that a new row attends to, chosen by a score over the key bounds of kv8.h
// (gfx950): of one row each of a batch of sequences, for every kv head, the `budget` pages that score highest, the first
// `first` and the last `recent` pages always among them, equal scores to the lower page; ascending.
//
// Score.  Of a page's keys k, q . k = sum_i q_i k_i is at most sum_i (q_i > 0 ? q_i max_i : q_i min_i).  q in 8 bits: of
// every 32 dimensions j of a head, n = rint(q 2^-e_j) with the smallest e_j that brings them to at most 127; the bounds in
// whole code units, |max|, |min| <= 448.  A group's sum over its 32 dimensions is then a whole number below
// 32 * 127 * 448 < 2^21, exact on the matrix unit in any order; and
//   score = max over the group's heads of (((S_0 2^e_0 + S_1 2^e_1) + S_2 2^e_2) + S_3 2^e_3) * scale_K
// rounds its few sums in f32, in that order: the choice is a function of the inputs, whatever computes it.  Units are
// coarse where a page has dimensions of very different size, since its scale is that of the largest: of 2048 pages of normal keys the 128
// chosen are those that unrounded bounds choose, also where two dimensions lie at +-20; 91% of them at +-100, 79% at +-200 (7 heads of 128).
//
// A workgroup scores 64 pages of one (sequence, kv head) or more; the last of them to arrive picks.  Lane (n, g) of a wave loads
// bounds 64 i + 16 g .. + 15 of page n of 16; those belong to group 2 i + g / 2, so of the 16 columns of
// v_mfma_f32_16x16x32_f16 the lower 8 take the heads' even groups (q is 0 in lanes of the odd ones) and the upper
// 8 the same heads' odd groups.
//
// The pick.  Scores become whole numbers of the same order (keys).  A histogram in LDS over 1024 equal parts of
// the keys' range finds the part that the last chosen one lies in; the keys there, a few, are ranked by every wave for
// itself (many: another histogram over that part).  Then every thread writes those above, and of those equal to it the
// first, to their places, which sums over the threads before it give.
//
// What bounds it: round trips, then bytes and instructions alike.  One context of 32768 tokens, 2 kv heads of 128 (1 MB of
// bounds): 9.2 us, about 4 until the scores are stored (lengths and table beside each other, then bounds, products), 1.5
// for the arrival, 3.4 for the pick's passes and barriers.  64 contexts of 1024 to 16384, 4 heads: 17.9 us for
// 36 MB of bounds, of which 6.7 are the steps of the longest contexts; with codes rounded to units by additions and a
// reduction over the heads page by page 20.3, with streaming loads of the bounds 5 more; four tiles of bounds on their way are no
// better than one.  By shuffles and compare passes over the bits of the keys the pick alone took 11.
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
  uint32_t* ws_key;           // [batch][hkv][max_pages], that a multiple of 4
  int32_t batch, total_rows, max_rows, max_ctx, layer, num_layers, hkv, group, num_blocks;
  int32_t budget, first, recent, chunks, max_pages;
  int32_t tiles;  // of 16 pages a wave
};

constexpr int kSelWaves = 4;
constexpr int kDppRowRor8 = 0x128;
constexpr int kSelBatch = 4 * 64 * kSelWaves, kSelBatches = 4;  // keys that a pick reads at once
constexpr int kSelBinBits = 10, kSelBins = 1 << kSelBinBits;

// Codes as whole numbers of 2^-24, eight to an operand: fp16's subnormals are those, up to 1023, so the conversion itself
// rounds codes (448 at most) to units, ties to even.
constexpr float kWhole = 0x1p-24f;
__device__ inline uint4 whole8(uint32_t a, uint32_t b) {
  return make_uint4(kv8_pair<kF16, false>(a, kWhole), kv8_pair<kF16, true>(a, kWhole), kv8_pair<kF16, false>(b, kWhole),
                    kv8_pair<kF16, true>(b, kWhole));
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

// ---- the pick: of `count` keys the `budget` largest, equal ones from the lowest place on
struct SelectMem {
  uint32_t hist[kSelBins];
  uint32_t list[64];
  uint32_t part[kSelWaves][kSelBatches];
  uint32_t bin, before, length;
};

// x of the lanes that a DPP control names, `none` where it names no lane.
template <int CTRL, int ROWS>
__device__ inline uint32_t dpp_u32(uint32_t none, uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp((int)none, (int)x, CTRL, ROWS, 0xf, false);
}
// Inclusive f over the lanes before and of a lane: shifts inside rows of 16, then the rows' last lanes to those behind.
template <class F>
__device__ __attribute__((always_inline)) inline uint32_t wave_scan(uint32_t x, uint32_t none, F&& f) {
  x = f(x, dpp_u32<0x111, 0xf>(none, x));
  x = f(x, dpp_u32<0x112, 0xf>(none, x));
  x = f(x, dpp_u32<0x114, 0xf>(none, x));
  x = f(x, dpp_u32<0x118, 0xf>(none, x));
  x = f(x, dpp_u32<0x142, 0xa>(none, x));
  return f(x, dpp_u32<0x143, 0xc>(none, x));
}

// Inclusive sums over the threads of the workgroup, of N numbers; a barrier inside.  total: of all threads.
template <int N>
__device__ __attribute__((always_inline)) inline void block_scan(uint32_t (&x)[N], uint32_t (&total)[N], uint32_t (&part)[kSelWaves][kSelBatches]) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
  for (int n = 0; n < N; ++n) x[n] = wave_scan(x[n], 0, [](uint32_t a, uint32_t b) { return a + b; });
  if (lane == 63) {
#pragma unroll
    for (int n = 0; n < N; ++n) part[w][n] = x[n];
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < N; ++n) {
    total[n] = 0;
#pragma unroll
    for (int k = 0; k < kSelWaves; ++k) {
      const uint32_t y = part[k][n];
      x[n] += k < w ? y : 0u;
      total[n] += y;
    }
  }
}

// The threads' keys are read kSelBatch at a time, in kSelBatches rounds, four successive places a thread; as
// many stay in registers (HELD), more are read again by every pass.  (hist is 0, and so is length.)  fixed: how
// many of the keys are the highest one.
template <bool HELD>
__device__ __attribute__((always_inline)) inline void pick_pages(const uint32_t* keys, int count, int budget, int fixed, int32_t* out,
                                                                 SelectMem& s) {
  constexpr int NT = 64 * kSelWaves, EACH = kSelBins / NT, R = kSelBatches;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const __amdgpu_buffer_rsrc_t far = ws_rsrc((const float*)keys);  // (written on other XCDs)
  uint32_t k[R][4];
  auto read = [&](int base) __attribute__((always_inline)) {  // (the keys' room is whole fours)
#pragma unroll
    for (int u = 0; u < R; ++u) {
      const float4 x = ws_get4(far, min(base + u * kSelBatch + 4 * tid, (count - 1) & ~3));
      const u32x4_t y = __builtin_bit_cast(u32x4_t, x);
#pragma unroll
      for (int r = 0; r < 4; ++r) k[u][r] = y[r];
    }
  };
  // f(place, key) of every key, in rounds
  auto pass = [&](auto&& f) __attribute__((always_inline)) {
    for (int base = 0; base < (HELD ? 1 : count); base += R * kSelBatch) {
      if constexpr (!HELD) read(base);
#pragma unroll
      for (int u = 0; u < R; ++u) {
        if (base + u * kSelBatch >= count) break;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int at = base + u * kSelBatch + 4 * tid + r;
          f(at, at < count ? k[u][r] : 0u, at < count);
        }
      }
    }
  };
  if constexpr (HELD) read(0);
  // the range of the keys; those of pages that are always chosen (the highest key) stand apart
  uint32_t lo = ~0u, hi = 0;
  pass([&](int, uint32_t x, bool on) __attribute__((always_inline)) {
    lo = on ? min(lo, x) : lo;
    hi = x == ~0u ? hi : max(hi, x);
  });
  lo = wave_scan(lo, ~0u, [](uint32_t a, uint32_t b) { return min(a, b); });
  hi = wave_scan(hi, 0, [](uint32_t a, uint32_t b) { return max(a, b); });
  if (lane == 63) {
    s.list[w] = lo;
    s.list[kSelWaves + w] = hi;
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < kSelWaves; ++n) {
    lo = min(lo, s.list[n]);
    hi = max(hi, s.list[kSelWaves + n]);
  }
  // bar: the want'th largest of the others; in steps of kSelBins equal bins of what is left of the range
  uint32_t bar = ~0u, want = (uint32_t)(budget - fixed);
  while (want) {
    const int shift = max(32 - __builtin_clz((hi - lo) | 1) - kSelBinBits, 0);
    pass([&](int, uint32_t x, bool on) __attribute__((always_inline)) {
      if (on && x >= lo && x <= hi) atomicAdd(&s.hist[(x - lo) >> shift], 1u);
    });
    __syncthreads();
    uint32_t c[EACH], up[1] = {0}, all[1];  // bins from the top, EACH a thread
#pragma unroll
    for (int n = 0; n < EACH; ++n) {
      c[n] = s.hist[kSelBins - 1 - EACH * tid - n];
      up[0] += c[n];
    }
    const uint32_t sum = up[0];
    block_scan(up, all, s.part);
    uint32_t before = up[0] - sum;
    if (before < want && up[0] >= want) {
      int at = 0;
#pragma unroll
      for (int n = 0; n < EACH - 1; ++n)
        if (at == n && before + c[n] < want) {
          before += c[n];
          at = n + 1;
        }
      s.bin = kSelBins - 1 - EACH * tid - at;
      s.before = before;
    }
    __syncthreads();
    lo += s.bin << shift;
    hi = min(hi, lo + ((1u << shift) - 1));
    want -= s.before;
    if (shift == 0) {
      bar = lo;
      break;
    }
    // few keys are left: every wave ranks them by itself
    pass([&](int, uint32_t x, bool on) __attribute__((always_inline)) {
      if (on && x >= lo && x <= hi) {
        const uint32_t n = atomicAdd(&s.length, 1u);
        if (n < 64) s.list[n] = x;
      }
    });
#pragma unroll
    for (int n = 0; n < EACH; ++n) s.hist[tid + NT * n] = 0;
    __syncthreads();
    const uint32_t length = s.length;
    if (length <= 64) {
      const uint32_t mine = lane < (int)length ? s.list[lane] : 0u;
      uint32_t over = 0, same = 0;
      for (uint32_t n = 0; n < length; ++n) {
        const uint32_t x = (uint32_t)__builtin_amdgcn_readlane((int)mine, n);
        over += x > mine;
        same += x == mine;
      }
      const uint64_t at = __ballot(lane < (int)length && over < want && over + same >= want);
      const int l = __builtin_ctzll(at);
      bar = (uint32_t)__builtin_amdgcn_readlane((int)mine, l);
      want -= (uint32_t)__builtin_amdgcn_readlane((int)over, l);
      break;
    }
    __syncthreads();
    if (tid == 0) s.length = 0;
    __syncthreads();
  }
  // ---- places: behind those of earlier rounds, and of earlier threads in this one.  (Counts of a round fit 16 bits.)
  uint32_t over = 0, same = 0;  // of earlier rounds
  for (int base = 0; base < (HELD ? 1 : count); base += R * kSelBatch) {
    if constexpr (!HELD) read(base);
    uint32_t own[R], up[R], all[R];
#pragma unroll
    for (int u = 0; u < R; ++u) {
      own[u] = 0;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const bool on = base + u * kSelBatch + 4 * tid + r < count;
        const uint32_t x = k[u][r];
        own[u] += on ? (x > bar || x == ~0u ? 1u : x == bar ? 1u << 16 : 0u) : 0u;
      }
      up[u] = own[u];
    }
    __syncthreads();  // (part)
    block_scan(up, all, s.part);
#pragma unroll
    for (int u = 0; u < R; ++u) {
      if (base + u * kSelBatch >= count) break;
      const uint32_t before = up[u] - own[u];
      uint32_t o = over + (before & 0xffffu), e = same + (before >> 16);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int at = base + u * kSelBatch + 4 * tid + r;
        const uint32_t x = k[u][r];
        const bool on = at < count, high = on && (x > bar || x == ~0u), equal = on && !high && x == bar;
        if (high || (equal && e < want)) out[o + min(e, want)] = at;
        o += high;
        e += equal;
      }
      over += all[u] & 0xffffu;
      same += all[u] >> 16;
    }
  }
}

template <int DT, int D>
__device__ void kv8_select_impl(const Kv8SelectArgs& A) {
  constexpr int H = D / 64;
  __shared__ SelectMem s;
  __shared__ int s_last;
  // neighbours on one XCD (block x runs on XCD x % 8): the kv heads of the same pages, whose bounds lie side by side
  const int units = A.batch * A.chunks;  // (padded to whole eights)
  const int u = blockIdx.x / (8 * A.hkv) * 8 + blockIdx.x % 8, kvh = blockIdx.x / 8 % A.hkv;
  if (u >= units) return;
  const int b = u % A.batch, chunk = u / A.batch;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int chunk_pages = 16 * kSelWaves * A.tiles;
  const int p0 = chunk * chunk_pages + w * (16 * A.tiles);
  const int32_t* const table = A.tables + (int64_t)b * A.table_stride;
  int pages = table[min(p0 + lane, (A.max_ctx - 1) / kPage)];  // of the wave's next 64 (on their way beside the lengths)
  const KvSeq S = kv_seq(A, b);
  int32_t* const out = A.pages + ((int64_t)b * A.hkv + kvh) * A.budget;
  const int count = S.ctx == 0 || S.rows == 0 ? 0 : S.start / kPage + 1;  // pages of the context
  if (count <= A.budget) {  // all of them, or none
    if (chunk == 0)
      for (int i = threadIdx.x; i < A.budget; i += 64 * kSelWaves) out[i] = i < count ? i : -1;
    return;
  }
  const int chunks = (count + chunk_pages - 1) / chunk_pages;
  if (chunk >= chunks) return;
  uint32_t* const keys = A.ws_key + ((int64_t)b * A.hkv + kvh) * A.max_pages;
  for (int i = threadIdx.x; i < kSelBins; i += 64 * kSelWaves) s.hist[i] = 0;
  if (threadIdx.x == 0) s.length = 0;

  // ---- scores of 16 pages at a time, their bounds one step ahead
  {
    const int n = lane & 15, g = lane >> 4;
    const int last = min(count, p0 + 16 * A.tiles);
    const int64_t base = (int64_t)A.layer * A.hkv + kvh;
    const int64_t stride = (int64_t)A.num_layers * A.hkv;
    // q of head n % 8, dimensions 64 i + 16 g + 8 k .. + 7
    const int head = n & 7;
    const bool on = head < A.group;
    const uint16_t* const src = A.q + (int64_t)S.row0 * A.q_stride + ((int64_t)kvh * A.group + (on ? head : 0)) * D + 16 * g;
    uint4 raw[H][2];
#pragma unroll
    for (int i = 0; i < H; ++i)
#pragma unroll
      for (int k = 0; k < 2; ++k) raw[i][k] = on ? *(const uint4*)(src + 64 * i + 8 * k) : make_uint4(0, 0, 0, 0);
    struct Step {
      uint4 hi[H], lo[H];
      float scale;
      bool bad;
    };
    auto load = [&](Step& T, int tile) __attribute__((always_inline)) {
      if (tile && tile % 4 == 0) pages = table[min(p0 + 16 * tile + lane, last - 1)];
      const int page = __shfl(pages, 16 * (tile & 3) + n);
      // a page outside the pool is never an address: page 0 is read instead, and the page comes last
      T.bad = page < 0 || page >= A.num_blocks;
      const int64_t at = (int64_t)(T.bad ? 0 : page) * stride + base;
      const uint8_t* const p = A.bounds + at * (2 * D) + 16 * g;
#pragma unroll
      for (int i = 0; i < H; ++i) {
        T.hi[i] = *(const uint4*)(p + 64 * i);
        T.lo[i] = *(const uint4*)(p + D + 64 * i);
      }
      T.scale = A.scales[at].x;
    };
    Step T[2];
    if (p0 < last) load(T[0], 0);
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
      unit[i] = __shfl(pow2f(e) / kWhole, (lane & 15) | (n >> 3) << 5);  // of the column's group: lanes g = 0, 1 or 2, 3
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
    auto score = [&](const Step& T, int tile) __attribute__((always_inline)) {
      f32x4_t sum[H];
#pragma unroll
      for (int i = 0; i < H; ++i) {
        sum[i] = (f32x4_t){0, 0, 0, 0};
        sum[i] = mfma_f16(whole8(T.hi[i].x, T.hi[i].y), qp[i][0], sum[i]);
        sum[i] = mfma_f16(whole8(T.hi[i].z, T.hi[i].w), qp[i][1], sum[i]);
        sum[i] = mfma_f16(whole8(T.lo[i].x, T.lo[i].y), qn[i][0], sum[i]);
        sum[i] = mfma_f16(whole8(T.lo[i].z, T.lo[i].w), qn[i][1], sum[i]);
      }
      // rows 4 g + r are pages; columns n < 8 the even groups' sums, n >= 8 the odd ones'.  Lanes n < 8 go on with pages
      // r = 0 and 1, their partners n ^ 8 with 2 and 3
      float all[2];
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int i = 0; i < H; ++i) {
          const float own = (n < 8 ? sum[i][r] : sum[i][r + 2]) * unit[i];
          const float other = dpp_mov<kDppRowRor8>((n < 8 ? sum[i][r + 2] : sum[i][r]) * unit[i]);
          if (i == 0) all[r] = own + other;
          else all[r] = (all[r] + (n < 8 ? own : other)) + (n < 8 ? other : own);
        }
      // the largest over the eight heads: of two pages over a quad, of one over both quads of the eight
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        all[r] = on ? all[r] : -INFINITY;
        all[r] = fmaxf(all[r], dpp_mov<kDppQuadXor1>(all[r]));
        all[r] = fmaxf(all[r], dpp_mov<kDppQuadXor2>(all[r]));
      }
      const bool second = n & 4;
      const float top = fmaxf(second ? all[1] : all[0], dpp_mov<kDppHalfMirror>(second ? all[0] : all[1]));
      // the first lane of a quad stores page 4 g + n / 4
      const int at = 4 * g + (n >> 2), p = p0 + 16 * tile + at;
      const float sk = __shfl(T.scale, at);
      const bool none = __shfl((int)T.bad, at);
      if ((n & 3) == 0 && p < count) {
        const bool always = p < A.first || p >= count - A.recent;
        __hip_atomic_store(keys + p, always ? ~0u : none ? 0u : score_key(top * sk), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
    };
    const int steps = (last - p0 + 15) / 16;  // (none: below 1)
    for (int i = 0; i < steps; i += 2) {
      if (i + 1 < steps) load(T[1], i + 1);
      score(T[0], i);
      if (i + 2 < steps) load(T[0], i + 2);
      if (i + 1 < steps) score(T[1], i + 1);
    }
  }
  // ---- the last workgroup of the (sequence, kv head) to arrive picks
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0) {
    int32_t* const cnt = A.ws_cnt + b * A.hkv + kvh;
    s_last = __hip_atomic_fetch_add(cnt, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == chunks - 1;
    if (s_last) __hip_atomic_store(cnt, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!s_last) return;
  if (count <= kSelBatch * kSelBatches) pick_pages<true>(keys, count, A.budget, A.first + A.recent, out, s);
  else pick_pages<false>(keys, count, A.budget, A.first + A.recent, out, s);
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
