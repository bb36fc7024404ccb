// Appends into the 8-bit paged cache of kv8.h, and its tokens back in 16 bits (gfx950).
//
// Append: bias, head norms and RoPE as norm_append.hip has them (append_row.h); q in 16 bits to q_out; of k and v, as
// they would go to a 16-bit pool, codes, scales and key bounds to the pages of the rows' slots:
//   e = max(the page's exponent, the smallest that holds the new rows),   code = e4m3(x 2^-e)
// A page begins anew with its first token: then only the new rows count.  Where a page's exponent grows, the
// codes that it holds are rounded again, and its bounds with them (rounding keeps order, so the bounds stay those
// of the codes).
//
// Runs.  A wave has one run of K or of V of one head: the rows of the call that go to one page, up to 16, D / 16
// lanes a row.  Its extremes are a reduction of the wave; the codes take their places by way of LDS, and 16 bytes a lane
// go out side by side.  A page's rows are one run wherever they lie in the call, and the wave of the first of them has
// it: two runs of a page would each write its codes, scale and bounds as if the other were not.  A wave is launched for every
// row, and those whose page an earlier row has end at once; or, of many rows, for every 16, among which it looks for the
// beginnings of runs.  Rows of one page are sought among the 64 around the run's first, where packed sequences have
// them; the slots of the other rows are compared with the page too, and only where one is of it (token by token orders)
// is the run put together from all rows.  That costs calls of up to 64 rows nothing, 512 single rows of 28 + 2 x 4
// heads of 128 7.3 us instead of 6.7, a prompt of 1000 rows 7.5 for 6.9, 2000 rows of 4 a sequence 25.1 for 23.1, 8191 single rows
// 112 for 95; it grows with the rows times the pages that are not whole: 64 prompts of 2047 rows 607 for 507.  With a span's
// heads side by side, so that a workgroup seeks one span's pages for four heads, those take 535, but 8191 rows 29.8.
//
// What bounds it.  8191 rows of 28 + 2 x 4 heads of 128 (bf16): 28.4 us for 147 MB, as a copy of them takes; 54 with a wave
// a row, 73 with the blocks of runs every eighth (all on one XCD), 36.9 with streamed loads of qkv.  A bound of
// registers for 5 or 6 waves a SIMD spills and is slower.  32 rows of 14 + 2 x 2 of 64: 6.1 us, of which a launch and the
// chain slots -> rows of the page -> position -> cos, row -> scale, slab.  The read, 32701 rows of 4 heads of 128: 18.7
// us for 101 MB, 5.4 TB/s; 333 of 2 of 64 2.7, a launch and slots -> scale, codes.
#include "append_row.h"
#include "kv8.h"

namespace luc {

struct Kv8AppendArgs : NormAppendArgs {  // (k_out, v_out unused)
  float* scales;
  uint8_t* bounds;  // or null
  uint32_t every;   // a block of runs comes first of so many
};

constexpr int kAppendWaves = 4;
constexpr int kManyRows = 512;   // calls of more are of many rows (kAppendManyRows of luc_kv8.cpp)
constexpr int kSpan = 16;        // rows of which a wave of such a call has the runs
constexpr int kBefore = 31;      // rows before a run's first that are in the 64 looked at first
constexpr int kFarChunks = 16;   // slots of the others that a wave reads at once, in 64s

// A run: lane j < len has its j'th row, its position and its place in the page.
struct AppendRun {
  int row, pos, place, len;
};

// Adds the members of the run of row `row` in page `page` among 64 rows from lo on: a lane has the slot and position of
// row lo + lane, -1 where that is none of the call's, or none of those rows.  False if the run's first row is another.
__device__ __attribute__((always_inline)) inline bool append_members(const Kv8AppendArgs& A, int lo, int64_t slot, int pos, int row,
                                                                     int64_t page, AppendRun& run) {
  const int lane = threadIdx.x & 63;
  // (rows without a position belong to no run)
  const bool member = slot >> 4 == page && pos >= 0 && pos < A.max_pos;
  const uint64_t in = __ballot(member);
  if (!in) return true;
  if (run.len == 0 && lo + __builtin_ctzll(in) != row) return false;
  const int rank = run.len + __builtin_popcountll(in & (lane ? ~0ull >> (64 - lane) : 0ull));
  const int from = __builtin_amdgcn_ds_permute((member ? min(rank, 63) : 63) * 4, lane);
  const int p = __shfl(pos, from), o = __shfl((int)(slot & (kPage - 1)), from);
  const int end = min(run.len + __builtin_popcountll(in), kPage);  // (more of them name a slot twice)
  if (lane >= run.len && lane < end) {
    run.row = lo + from;
    run.pos = p;
    run.place = o;
  }
  run.len = end;
  return true;
}

// ---- of many rows: what the waves of a workgroup seek together.  A wave's runs begin in rows row0 + 1 .. row0 + kSpan.
struct AppendFar {
  uint32_t low[kAppendWaves * kSpan];  // of a row's slot
  uint32_t open[kAppendWaves], far[kAppendWaves];  // bit i: row row0 + 1 + i
  int row0[kAppendWaves];
};

// Lane i has the slot of row row0 + i, or -1.  Of the lanes `begins`, 1 .. kSpan, those whose page a row may have that none of
// them looks at first: 15 rows before row0 to 33 behind are.  (All of a page, in order, from a lane on: no.)  The waves
// share the call's slots and compare them with the pages of the workgroup's rows; more than a few pages stand in a table, N bytes,
// by a hash, where the second one in a place may be anywhere.  1024 single rows of 14 + 2 x 2 heads of 64: 57 us by
// comparisons, 48 by the table, whose barriers make it slower for few pages: a prompt of 1000 rows 5.8 and 7.9.
// Barriers inside, one behind the last use of the table.
constexpr int kFewPages = 8;
template <int N>
__device__ __attribute__((always_inline)) inline uint64_t append_far(const Kv8AppendArgs& A, int w, int row0, int64_t slot,
                                                                     uint64_t begins, AppendFar& s, uint8_t* table) {
  const int lane = threadIdx.x & 63;
  uint64_t follows = __ballot(slot - __shfl_up(slot, 1) == 1 && lane > 0);
  follows &= follows >> 1;
  follows &= follows >> 2;
  follows &= follows >> 4;
  follows &= follows >> 7;  // 15 of them from here on
  const uint64_t open = begins & ~(__ballot((slot & (kPage - 1)) == 0) & follows >> 1);
  const int id = w * kSpan + lane - 1;
  if (lane >= 1 && lane <= kSpan) s.low[id] = (uint32_t)slot & ~(kPage - 1u);  // (a page by its low bits, which another may share)
  if (lane == 0) {
    s.open[w] = (uint32_t)(open >> 1);
    s.far[w] = 0;
    s.row0[w] = row0;
  }
  __syncthreads();
  static_assert(kAppendWaves * kSpan == 64, "a lane a row");
  const uint64_t all = __ballot(s.open[lane / kSpan] >> (lane % kSpan) & 1);
  if (!all) return 0;
  const uint32_t low = s.low[lane];
  const int near = s.row0[lane / kSpan] - 15;
  const bool few = __builtin_popcountll(all) <= kFewPages, mine = all >> lane & 1 && lane / kSpan == w;
  auto place = [](uint32_t x) { return (x >> 4) * 0x9e3779b1u >> (32 - __builtin_ctz(N)); };
  if (!few) {
#pragma unroll
    for (int i = 0; i < N / (16 * 64 * kAppendWaves); ++i) ((uint4*)table)[threadIdx.x + 64 * kAppendWaves * i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    if (mine) table[place(low)] = (uint8_t)(lane + 1);
    __syncthreads();
    if (mine && table[place(low)] != lane + 1) atomicOr(&s.far[w], 1u << (lane % kSpan));
  }
  for (int lo = 0; lo < A.rows; lo += 64 * kAppendWaves * kFarChunks) {
    uint32_t y[kFarChunks];
    auto chunk = [&](int u) { return min(lo + 64 * (kAppendWaves * u + w), A.rows - 64); };  // (behind the rows the last again)
#pragma unroll
    for (int u = 0; u < kFarChunks; ++u) y[u] = (uint32_t)A.slots[chunk(u) + (int64_t)lane];
    if (few) {
      for (uint64_t left = all; left; left &= left - 1) {
        const int i = __builtin_ctzll(left);
        const uint32_t page = (uint32_t)__builtin_amdgcn_readlane((int)low, i);
        const int from = __builtin_amdgcn_readlane(near, i);
        uint32_t least = ~0u;
#pragma unroll
        for (int u = 0; u < kFarChunks; ++u) least = min(least, (uint32_t)(chunk(u) + lane - from) < 49u ? ~0u : y[u] ^ page);
        if (__any(least < (uint32_t)kPage) && lane == 0) atomicOr(&s.far[i / kSpan], 1u << (i % kSpan));
      }
    } else {
      int at[kFarChunks];
#pragma unroll
      for (int u = 0; u < kFarChunks; ++u) at[u] = table[place(y[u])];
#pragma unroll
      for (int u = 0; u < kFarChunks; ++u) {
        if (!__any(at[u])) continue;
        const int j = max(at[u] - 1, 0), v = j / kSpan;
        if (at[u] && (s.low[j] ^ y[u]) < (uint32_t)kPage && (uint32_t)(chunk(u) + lane - (s.row0[v] - 15)) >= 49u)
          atomicOr(&s.far[v], 1u << (j % kSpan));
      }
    }
  }
  __syncthreads();
  return (uint64_t)s.far[w] << 1;
}

// The run that row `row` of a head of k (is_v 0) or v begins, if it does.  image: a slab of LDS, the wave's.  MANY: the
// call is of many rows, and `far` says that a row outside the 64 around this one may have its page.
template <int DT, int D, bool MANY>
__device__ __attribute__((always_inline)) inline void append_run(const Kv8AppendArgs& A, int row, int hh, int is_v, bool far, uint8_t* image) {
#pragma clang fp contract(off)
  constexpr int LANES = D / 16;
  constexpr int ROWS = 64 / LANES, PASSES = 16 / ROWS;  // rows of a pass
  constexpr int CHUNKS = D / 64;                        // 16 bytes of a slab a lane
  const int lane = threadIdx.x & 63;
  const int near = !MANY && A.rows <= 64 ? 0 : row - kBefore;  // lane i: row near + i
  int64_t slot = -1;
  int pos = -1;
  if (near + lane >= 0 && near + lane < A.rows) {
    slot = A.slots[near + lane];
    pos = A.positions[near + lane];
  }
  constexpr int MOST = kManyRows / 64;
  uint32_t y[MOST];  // all slots of more than 64 rows
  auto chunk = [&](int u) { return min(64 * u, A.rows - 64); };
  if (!MANY && A.rows > 64) {
#pragma unroll
    for (int u = 0; u < MOST; ++u) {
      y[u] = ~0u;
      if (64 * u < A.rows) y[u] = (uint32_t)A.slots[chunk(u) + lane];
    }
  }
  const int64_t first = __shfl(slot, row - near);
  if (first < 0 || first >= A.num_slots) return;
  const int64_t page = first >> 4;
  AppendRun run = {0, 0, 0, 0};
  if (!(MANY && far) && !append_members(A, near, slot, pos, row, page, run)) return;
  if (!MANY && A.rows > 64) {
    uint32_t least = ~0u;
#pragma unroll
    for (int u = 0; u < MOST; ++u)
      least = min(least, (uint32_t)(chunk(u) + lane - near) < 64u ? ~0u : y[u] ^ ((uint32_t)first & ~(kPage - 1u)));
    far = __any(least < (uint32_t)kPage);
    if (far) run.len = 0;
  }
  if (far) {  // all of the call's rows
    for (int from = 0; from < A.rows; from += 64 * 8) {
      int64_t s[8];
      int p[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int at = min(from + 64 * u + lane, A.rows - 1);
        s[u] = A.slots[at];
        p[u] = A.positions[at];
      }
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (!append_members(A, from + 64 * u, from + 64 * u + lane < A.rows ? s[u] : -1, p[u], row, page, run)) return;
    }
  }
  if (run.len == 0) return;  // (a row without a position)
  const int len = run.len;
  uint32_t tokens = lane < len ? 1u << run.place : 0u;  // the page's tokens that are new
#pragma unroll
  for (int k = 1; k < kPage; k <<= 1) tokens |= (uint32_t)__shfl_xor((int)tokens, k);
  tokens = (uint32_t)__builtin_amdgcn_readfirstlane((int)tokens);
  const bool joins = !(tokens & 1);  // what the page holds
  const int64_t head = ((first >> 4) * A.num_layers + A.layer) * A.hkv + hh;
  uint8_t* const slab = (uint8_t*)(is_v ? A.v_pool : A.k_pool) + head * Kv8<D>::kSlab;
  float* const scale_at = A.scales + head * 2 + is_v;
  const int held = joins ? max(exp2of(*scale_at), kKv8LeastExp) : kKv8LeastExp;
  // new tokens of the lane's chunks, a mask of bytes; where some bytes stay, they are read first
  uint32_t fresh[CHUNKS];
  uint4 old[CHUNKS];
#pragma unroll
  for (int i = 0; i < CHUNKS; ++i) {
    const int b = 16 * (lane + 64 * i);
    if (is_v) {
      fresh[i] = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (tokens >> (b / (4 * D) * 4 + k) & 1) fresh[i] |= 0xffu << (8 * k);
      }
    } else {
      fresh[i] = tokens >> (b / D) & 1 ? ~0u : 0u;
    }
    old[i] = make_uint4(0, 0, 0, 0);
    if (fresh[i] != 0 && fresh[i] != ~0u) old[i] = *(const uint4*)(slab + b);
  }
  // ---- the rows' values, in 16 bits and back
  const int c = lane % LANES, kind = 1 + is_v;
  uint4 x[PASSES][2];
  int place[PASSES];  // of the lane's row in the page
  float top = 0.0f;
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const int j = p * ROWS + lane / LANES;
    const int from = __shfl(run.row, j), pj = __shfl(run.pos, j);
    place[p] = __shfl(run.place, j);
    if (j >= len) continue;
    float y[16];
    append_head<DT, D>(A, kind, from, hh, c, pj, y);
    x[p][0] = pack8<DT>(y);
    x[p][1] = pack8<DT>(y + 8);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      unpack8<DT>(x[p][h], y);
#pragma unroll
      for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(y[e]));  // (a NaN is passed over)
    }
    asm volatile("" : "+v"(x[p][0].x), "+v"(x[p][1].x)::"memory");
  }
  top = fminf(top, kKv8Limit);
  const int e = max(kv8_exponent(wave_max(top)), held);
  const float up = pow2f(-e), less = pow2f(held - e);
  const bool grown = joins && e != held;
  // ---- codes by way of LDS
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const int j = p * ROWS + lane / LANES, t = place[p];
    if (j >= len) continue;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float y[8];
      unpack8<DT>(x[p][h], y);
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = __builtin_isnan(y[e]) ? y[e] : fminf(fmaxf(y[e], -kKv8Limit), kKv8Limit) * up;
      const uint32_t code[2] = {kv8_encode4(y[0], y[1], y[2], y[3]), kv8_encode4(y[4], y[5], y[6], y[7])};
      const int i = D / 2 * h + 8 * c;
      if (is_v) {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          image[Kv8<D>::v_at(t >> 2, i + k) + (t & 3)] = (uint8_t)(code[k >> 2] >> (8 * (k & 3)));
      } else {
        *(uint2*)(image + Kv8<D>::k_at(t, i)) = make_uint2(code[0], code[1]);
      }
    }
  }
  wave_lds_sync();
#pragma unroll
  for (int i = 0; i < CHUNKS; ++i) {
    const int b = 16 * (lane + 64 * i);
    uint32_t o[4] = {old[i].x, old[i].y, old[i].z, old[i].w};
    if (grown && fresh[i] != ~0u) {
      const uint4 y = *(const uint4*)(slab + b);
      o[0] = kv8_rescale4(y.x, less); o[1] = kv8_rescale4(y.y, less);
      o[2] = kv8_rescale4(y.z, less); o[3] = kv8_rescale4(y.w, less);
    }
    if (fresh[i] == 0 && !grown) continue;
    const uint4 n = *(const uint4*)(image + b);
    const uint32_t f = fresh[i];
    *(uint4*)(slab + b) = make_uint4((n.x & f) | (o[0] & ~f), (n.y & f) | (o[1] & ~f), (n.z & f) | (o[2] & ~f),
                                     (n.w & f) | (o[3] & ~f));
  }
  if (lane == 0) *scale_at = pow2f(e);
  if (is_v || !A.bounds) return;
  // ---- key bounds: a lane has 4 dimensions of every 256 / D'th token
  constexpr int QUADS = D / 4, SETS = 64 / QUADS;
  const int quad = lane % QUADS, set = lane / QUADS;
  float hi[4], lo[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    hi[k] = -INFINITY;
    lo[k] = INFINITY;
  }
  uint8_t* const bound = A.bounds + head * (2 * D) + 4 * quad;
  auto take = [&](uint32_t word, uint32_t word_lo, float f) __attribute__((always_inline)) {
    const float4 a = kv8_decode4(word), b = kv8_decode4(word_lo);
    const float ya[4] = {a.x, a.y, a.z, a.w}, yb[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      hi[k] = fmaxf(hi[k], __builtin_isnan(ya[k]) ? 0.0f : ya[k] * f);
      lo[k] = fminf(lo[k], __builtin_isnan(yb[k]) ? 0.0f : yb[k] * f);
    }
  };
  if (joins && set == 0)  // (rounded again, as the codes are)
    take(kv8_rescale4(*(const uint32_t*)bound, less), kv8_rescale4(*(const uint32_t*)(bound + D), less), 1.0f);
#pragma unroll
  for (int t0 = 0; t0 < kPage; t0 += SETS) {
    const int t = t0 + set;
    if (!(tokens >> t & 1)) continue;
    const uint32_t y = *(const uint32_t*)(image + Kv8<D>::k_at(t, 4 * quad));
    take(y, y, 1.0f);
  }
#pragma unroll
  for (int k = 0; k < 4; ++k)
#pragma unroll
    for (int s = QUADS; s < 64; s <<= 1) {
      hi[k] = fmaxf(hi[k], __shfl_xor(hi[k], s));
      lo[k] = fminf(lo[k], __shfl_xor(lo[k], s));
    }
  if (set == 0) {
    *(uint32_t*)bound = kv8_encode4(hi[0], hi[1], hi[2], hi[3]);
    *(uint32_t*)(bound + D) = kv8_encode4(lo[0], lo[1], lo[2], lo[3]);
  }
}

// MANY: a wave has the runs that begin in 16 rows, else in one.
template <int DT, int D, bool MANY>
__device__ void kv8_append_impl(const Kv8AppendArgs& A) {
  constexpr int LANES = D / 16, SPAN = MANY ? kSpan : 1;
  __shared__ __attribute__((aligned(16))) uint8_t s_image[kAppendWaves][Kv8<D>::kSlab];
  const uint32_t nq = (uint32_t)A.rows * A.hq;
  const uint32_t spans = ((uint32_t)A.rows + SPAN - 1) / SPAN;
  // blocks of runs among those of q, evenly: they wait more than they move
  const uint32_t run_blocks = (2u * A.hkv * spans + kAppendWaves - 1) / kAppendWaves;
  const uint32_t turn = blockIdx.x / A.every, before = min(turn + (blockIdx.x % A.every != 0), run_blocks);
  if (blockIdx.x % A.every != 0 || turn >= run_blocks) {
    const uint32_t unit = ((blockIdx.x - before) * 256 + threadIdx.x) / LANES;
    const int c = threadIdx.x % LANES;
    if (unit >= nq) return;
    const int row = unit / A.hq, hh = unit % A.hq;
    const int pos = A.positions[row];
    if (pos < 0 || pos >= A.max_pos) return;
    float x[16];
    append_head<DT, D>(A, 0, row, hh, c, pos, x);
    uint16_t* const o = A.q_out + row * A.q_out_stride + hh * D;
    const uint4 o1 = pack8<DT>(x), o2 = pack8<DT>(x + 8);
    if constexpr (MANY) {
      // q is more than the caches keep beside the pools.  8191 rows of 28 + 2 x 4 heads of 128: 29.1 us,
      // 38.6 with ordinary stores (the attention behind it then finds q nearer: of both together, 189 and 187)
      __builtin_nontemporal_store(__builtin_bit_cast(u32x4_t, o1), (u32x4_t*)(o + 8 * c));
      __builtin_nontemporal_store(__builtin_bit_cast(u32x4_t, o2), (u32x4_t*)(o + D / 2 + 8 * c));
    } else {
      *(uint4*)(o + 8 * c) = o1;
      *(uint4*)(o + D / 2 + 8 * c) = o2;
    }
    return;
  }
  // ---- the runs of one head of k or v that begin in SPAN rows
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const uint32_t unit = turn * kAppendWaves + w;  // (the grid's threads fit 32 bits)
  const bool none = unit >= 2u * A.hkv * spans;
  const int row0 = (int)(unit % spans) * SPAN;
  const int hh = unit / spans % A.hkv, is_v = unit / spans / A.hkv;
  if constexpr (!MANY) {
    if (!none) append_run<DT, D, false>(A, row0, hh, is_v, false, s_image[w]);
  } else {
    // lane i: row row0 - 1 + i; one that follows another of its page begins no run
    __shared__ AppendFar s_far;
    const int at = row0 - 1 + lane;
    const bool on = at >= 0 && at < A.rows;
    const int64_t slot = on ? A.slots[at] : -1;
    const int pos = on ? A.positions[at] : -1;
    const int64_t page = pos >= 0 && pos < A.max_pos ? slot >> 4 : -1;  // (rows without a position belong to no run)
    const int64_t before = __shfl_up(page, 1);
    uint64_t begins = none ? 0 : __ballot(lane > 0 && lane <= SPAN && page >= 0 && page != before);
    const uint64_t far = append_far<sizeof(s_image)>(A, w, row0 - 1, page < 0 ? -1 : slot, begins, s_far, s_image[0]);
    while (begins) {
      const int i = __builtin_ctzll(begins);
      begins &= begins - 1;
      wave_lds_sync();  // (the image again)
      asm volatile("" ::: "memory");  // (norms and biases stay loads of every run: held in registers they cost occupancy)
      append_run<DT, D, true>(A, row0 - 1 + i, hh, is_v, far >> i & 1, s_image[w]);
    }
  }
}

// ---- tokens back in 16 bits: a thread has 8 dimensions of K or V of a row's head
struct Kv8ReadArgs {
  uint16_t* k_out;
  uint16_t* v_out;
  int64_t out_stride;
  const int64_t* slots;
  const uint8_t* k_pool;
  const uint8_t* v_pool;
  const float* scales;
  int64_t num_slots;
  int32_t rows, layer, num_layers, hkv;
};

template <int DT, int D>
__device__ void kv8_read_impl(const Kv8ReadArgs& A) {
  constexpr int T = D / 8;  // threads of a head
  const uint32_t each = (uint32_t)A.rows * A.hkv * T;  // (twice that fits 32 bits)
  uint32_t i = blockIdx.x * 256 + threadIdx.x;
  const bool is_v = i >= each;
  if (is_v) i -= each;
  if (i >= each) return;
  const int c = i % T, hh = i / T % A.hkv, row = i / T / A.hkv;
  const int64_t slot = A.slots[row];
  if (slot < 0 || slot >= A.num_slots) return;
  const int t = (int)(slot & (kPage - 1));
  const int64_t head = ((slot >> 4) * A.num_layers + A.layer) * A.hkv + hh;
  const float scale = A.scales[head * 2 + is_v];
  uint32_t a, b;
  if (is_v) {
    const uint4* const p = (const uint4*)(A.v_pool + head * Kv8<D>::kSlab + Kv8<D>::v_at(t >> 2, 8 * c));
    const uint4 u = p[0], v = p[1];
    // byte t % 4 of every dword: of two dwords (selectors 0 .. 3 the second operand's, 4 .. 7 the first's), then of four
    const uint32_t s = (uint32_t)(t & 3), sel = s | (s + 4) << 8;
    a = __builtin_amdgcn_perm(u.y, u.x, sel) & 0xffffu;
    a |= __builtin_amdgcn_perm(u.w, u.z, sel) << 16;
    b = __builtin_amdgcn_perm(v.y, v.x, sel) & 0xffffu;
    b |= __builtin_amdgcn_perm(v.w, v.z, sel) << 16;
  } else {
    const uint2 u = *(const uint2*)(A.k_pool + head * Kv8<D>::kSlab + Kv8<D>::k_at(t, 8 * c));
    a = u.x;
    b = u.y;
  }
  uint16_t* const o = (is_v ? A.v_out : A.k_out) + row * A.out_stride + hh * D + 8 * c;
  // (streamed: 32701 rows of 4 heads of 128 take 19.3 us, 23.8 with ordinary stores)
  const uint4 y = make_uint4(kv8_pair<DT, false>(a, scale), kv8_pair<DT, true>(a, scale), kv8_pair<DT, false>(b, scale),
                          kv8_pair<DT, true>(b, scale));
  __builtin_nontemporal_store(__builtin_bit_cast(u32x4_t, y), (u32x4_t*)o);
}

}  // namespace luc

#define LUC_KV8_APPEND(DTN, DT, D)                                                              \
  extern "C" __global__ __launch_bounds__(256) void luc_kv8_append_##DTN##_d##D(                \
      luc::Kv8AppendArgs a) {                                                                   \
    luc::kv8_append_impl<luc::DT, D, false>(a);                                                 \
  }                                                                                             \
  extern "C" __global__ __launch_bounds__(256) void luc_kv8_append_many_##DTN##_d##D(           \
      luc::Kv8AppendArgs a) {                                                                   \
    luc::kv8_append_impl<luc::DT, D, true>(a);                                                  \
  }                                                                                             \
  extern "C" __global__ __launch_bounds__(256) void luc_kv8_read_##DTN##_d##D(luc::Kv8ReadArgs a) { \
    luc::kv8_read_impl<luc::DT, D>(a);                                                          \
  }
LUC_KV8_APPEND(bf16, kBF16, 64)
LUC_KV8_APPEND(bf16, kBF16, 128)
LUC_KV8_APPEND(f16, kF16, 64)
LUC_KV8_APPEND(f16, kF16, 128)
