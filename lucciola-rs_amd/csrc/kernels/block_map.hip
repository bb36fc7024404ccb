// Pages for the rows of a batch, dealt on the GPU (gfx950): the block tables of
// luc_blocks (the reference's free list and prepare_for_step,
// src/layers/kv_cache.rs:73-76, 106-122) kept on the device, so that a loop with no
// host work per step, or a captured one, can grow and shrink its sequences.
//
// extend.  Sequence i of B holds L_i tokens in held_i = ceil(L_i / 16) pages and gets n_i
// more: need_i = ceil((L_i + n_i) / 16) - held_i pages, off the top of the free list (F
// entries) in the order of the sequences.  With P_i = sum of need_j and c_i = sum of n_j
// over j < i, row r of the packed new rows belongs to the last i with c_i <= r, at position
// p = L_i + r - c_i, in page
//   p / 16 <  held_i: table[i][p / 16]
//   p / 16 >= held_i: free[F - 1 - (P_i + p / 16 - held_i)]   (the page's first row writes it
//                                                              to the table)
// All or nothing: with too few pages, rows or table entries nothing is taken.
//
// truncate is extend's inverse: pages ceil(keep_i / 16) .. held_i - 1 go back on top, the last
// sequence's first and its last page first, so that the pages of an extend that is
// undone lie where they lay.
//
// Work split.  Every workgroup scans the lengths itself (at most kMaxSeqs, 4 a thread: one
// round trip to L2 against a second launch) and then takes its share of rows (or
// pages).  Lengths and the free count change only when the last workgroup has read them: each
// counts itself in, the last one to arrive writes them.  What bounds it is that chain of
// dependent round trips (a launch, lengths, table or free list, the arrival), not bytes: extend
// 3.9 us for 8 rows of 8 sequences, 8.0 us for some 120,000 of 64 (1.4 MB written); truncate 3.4 and
// 6.0 us.  Scans in LDS by ds_bpermute and a release fence at the arrival took 5.5, 11.6, 4.0
// and 7.0.
#include "luc_common.h"

namespace luc {

constexpr int kMapThreads = 1024;
constexpr int kMapPer = 4;                          // sequences per thread
constexpr int kMaxSeqs = kMapThreads * kMapPer;     // luc_kv4.cpp: kMaxMapBatch
// words of the state, and the bits of its status
enum : int { kStFree = 0, kStStatus = 1, kStArrived = 2 };
enum : int { kMapNoPages = 1, kMapTableFull = 2, kMapBadLength = 4, kMapNoRows = 8 };

struct MapArgs {
  const int32_t* count;    // extend: new tokens; truncate: tokens to keep
  int32_t* lens;
  int32_t* tables;
  int64_t table_stride;
  int32_t* free_list;
  int32_t* state;
  int64_t* slots;          // extend only, from here on
  int32_t* positions;
  int32_t* cu_seqlens;
  int32_t* start_pos;
  int32_t batch, num_blocks, rows;
};

// Sums stop at 2^32 - 1, so that no counts wrap around: more than any limit that a total is held to.
__device__ inline uint32_t map_add(uint32_t x, uint32_t y) { return __builtin_elementwise_add_sat(x, y); }

// One step of a scan over the wave: adds the value that DPP control CTRL brings from a lower lane, in
// the rows of the mask.
template <int CTRL, int ROWS>
__device__ inline uint32_t map_step(uint32_t x) {
  return map_add(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, false));
}
__device__ inline uint32_t map_wave_scan(uint32_t x) {
  x = map_step<0x111, 0xf>(x);  // row_shr 1, 2, 4, 8
  x = map_step<0x112, 0xf>(x);
  x = map_step<0x114, 0xf>(x);
  x = map_step<0x118, 0xf>(x);
  x = map_step<0x142, 0xa>(x);  // row_bcast 15, 31
  return map_step<0x143, 0xc>(x);
}

// Over the workgroup, of one a and b and some bits per thread: inclusive scans, totals, the bits that
// any thread has set.
struct MapScan {
  uint32_t a, b, all_a, all_b;
  int bits;
};
__device__ inline MapScan map_scan(uint32_t a, uint32_t b, int bits) {
  constexpr int WAVES = kMapThreads / 64;
  __shared__ uint32_t s_a[WAVES], s_b[WAVES];
  __shared__ int s_bits[WAVES];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  MapScan r{map_wave_scan(a), map_wave_scan(b), 0, 0, 0};
  int any = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) any |= __any(bits >> k & 1) ? 1 << k : 0;
  if (lane == 63) {
    s_a[w] = r.a;
    s_b[w] = r.b;
    s_bits[w] = any;
  }
  __syncthreads();
  uint32_t before_a = 0, before_b = 0;
#pragma unroll
  for (int i = 0; i < WAVES; ++i) {
    if (i == w) {
      before_a = r.all_a;
      before_b = r.all_b;
    }
    r.all_a = map_add(r.all_a, s_a[i]);
    r.all_b = map_add(r.all_b, s_b[i]);
    r.bits |= s_bits[i];
  }
  r.a = map_add(r.a, before_a);
  r.b = map_add(r.b, before_b);
  return r;
}

// Counts this workgroup in; whether it is the last, once every other one has read what the caller
// is about to write (reads only, and those have arrived where their values were used: no fence, which
// would write an L2 back).
__device__ inline bool map_last(int32_t* state) {
  if (gridDim.x == 1) return true;
  __shared__ int s_last;
  __syncthreads();
  if (threadIdx.x == 0)
    s_last = __hip_atomic_fetch_add(state + kStArrived, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
             (int)gridDim.x - 1;
  __syncthreads();
  return s_last;
}

// last i in [0, n) with a[i] <= x  (a ascending, a[0] <= x)
__device__ inline int map_find(const int32_t* a, int n, int x) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a[mid] <= x) lo = mid; else hi = mid - 1;
  }
  return lo;
}

__device__ void extend_impl(const MapArgs& A) {
  __shared__ int32_t s_cu[kMaxSeqs], s_page[kMaxSeqs], s_len[kMaxSeqs];
  const int t = threadIdx.x;
  const int64_t room = A.table_stride * kPage;  // tokens of a table row
  const int F = A.state[kStFree];
  int len[kMapPer], cnt[kMapPer], need[kMapPer];
  int bad = F < 0 || F > A.num_blocks ? kMapBadLength : 0;
  uint32_t rows = 0, pages = 0;
#pragma unroll
  for (int k = 0; k < kMapPer; ++k) {
    const int i = t * kMapPer + k;
    len[k] = i < A.batch ? A.lens[i] : 0;
    cnt[k] = i < A.batch ? A.count[i] : 0;
    const int64_t sum = (int64_t)len[k] + cnt[k];
    if (len[k] < 0 || cnt[k] < 0 || len[k] > room) bad |= kMapBadLength;
    else if (sum > room) bad |= kMapTableFull;
    need[k] = (int)((sum + kPage - 1) / kPage - ((int64_t)len[k] + kPage - 1) / kPage);
    rows = map_add(rows, max(cnt[k], 0));
    pages = map_add(pages, max(need[k], 0));
  }
  const MapScan S = map_scan(rows, pages, bad);
  int verdict = S.bits;
  if (S.all_a > (uint32_t)A.rows) verdict |= kMapNoRows;
  if (S.all_b > (uint32_t)max(F, 0)) verdict |= kMapNoPages;
  // sums of rejected lengths mean nothing: only the lengths' own bits are told
  if (verdict & (kMapBadLength | kMapTableFull)) verdict &= kMapBadLength | kMapTableFull;
  if (verdict) {
    for (uint32_t r = blockIdx.x * kMapThreads + t; r < (uint32_t)A.rows; r += gridDim.x * kMapThreads) {
      A.slots[r] = -1;
      A.positions[r] = -1;
    }
    if (blockIdx.x == 0) {
#pragma unroll
      for (int k = 0; k < kMapPer; ++k) {
        const int i = t * kMapPer + k;
        if (i < A.batch) {
          A.start_pos[i] = len[k];
          A.cu_seqlens[i + 1] = 0;
        }
      }
      if (t == 0) {
        A.cu_seqlens[0] = 0;
        A.state[kStStatus] |= verdict;
      }
    }
    return;
  }
  {
    int c = (int)(S.a - rows), p = (int)(S.b - pages);
#pragma unroll
    for (int k = 0; k < kMapPer; ++k) {
      const int i = t * kMapPer + k;
      s_cu[i] = c;
      s_page[i] = p;
      s_len[i] = len[k];
      c += cnt[k];
      p += need[k];
      if (blockIdx.x == 0 && i < A.batch) {
        A.start_pos[i] = len[k];
        A.cu_seqlens[i + 1] = c;
      }
    }
    if (blockIdx.x == 0 && t == 0) A.cu_seqlens[0] = 0;
  }
  __syncthreads();
  // (32 unsigned bits: the last step may pass 2^31)
  const int total = (int)S.all_a;
  for (uint32_t x = blockIdx.x * kMapThreads + t; x < (uint32_t)A.rows; x += gridDim.x * kMapThreads) {
    const int r = (int)x;
    int64_t slot = -1;
    int pos = -1;
    if (r < total) {
      const int i = map_find(s_cu, A.batch, r);
      pos = s_len[i] + r - s_cu[i];
      const int held = (s_len[i] + kPage - 1) / kPage, pg = pos / kPage;
      int32_t* const entry = A.tables + i * A.table_stride + pg;
      int id;
      if (pg < held) {
        id = *entry;
      } else {
        id = A.free_list[F - 1 - (s_page[i] + pg - held)];
        if (pos % kPage == 0) *entry = id;
      }
      // a page outside the pool is never a slot
      if (id >= 0 && id < A.num_blocks) slot = (int64_t)id * kPage + pos % kPage;
    }
    A.slots[r] = slot;
    A.positions[r] = pos;
  }
  if (!map_last(A.state)) return;
#pragma unroll
  for (int k = 0; k < kMapPer; ++k) {
    const int i = t * kMapPer + k;
    if (i < A.batch) A.lens[i] = len[k] + cnt[k];
  }
  if (t == 0) {
    A.state[kStFree] = F - (int)S.all_b;
    A.state[kStArrived] = 0;
  }
}

__device__ void truncate_impl(const MapArgs& A) {
  __shared__ int32_t s_gone[kMaxSeqs], s_left[kMaxSeqs];
  const int t = threadIdx.x;
  const int64_t room = A.table_stride * kPage;
  const int F = A.state[kStFree];
  int keep[kMapPer], left[kMapPer], gone[kMapPer];
  int bad = F < 0 || F > A.num_blocks ? kMapBadLength : 0;
  uint32_t pages = 0;
#pragma unroll
  for (int k = 0; k < kMapPer; ++k) {
    const int i = t * kMapPer + k;
    const int len = i < A.batch ? A.lens[i] : 0;
    const int want = i < A.batch ? A.count[i] : 0;
    if (len < 0 || len > room || want < 0) bad |= kMapBadLength;
    keep[k] = min(len, want);
    left[k] = (int)(((int64_t)keep[k] + kPage - 1) / kPage);
    gone[k] = (int)(((int64_t)len + kPage - 1) / kPage) - left[k];
    pages = map_add(pages, max(gone[k], 0));
  }
  const MapScan S = map_scan(pages, 0, bad);
  int verdict = S.bits;
  if (F + (int64_t)S.all_a > A.num_blocks) verdict |= kMapBadLength;  // more pages than the pool has
  if (verdict) {
    if (blockIdx.x == 0 && t == 0) A.state[kStStatus] |= verdict;
    return;
  }
  {
    int g = (int)(S.a - pages);
#pragma unroll
    for (int k = 0; k < kMapPer; ++k) {
      s_gone[t * kMapPer + k] = g;  // pages given back by the sequences before it
      s_left[t * kMapPer + k] = left[k];
      g += gone[k];
    }
  }
  __syncthreads();
  const int all = (int)S.all_a;
  for (uint32_t x = blockIdx.x * kMapThreads + t; x < (uint32_t)all; x += gridDim.x * kMapThreads) {
    const int e = (int)x;
    const int i = map_find(s_gone, A.batch, e);
    int32_t* const entry = A.tables + i * A.table_stride + s_left[i] + (e - s_gone[i]);
    // entry e of the pages in table order is the (all - 1 - e)-th to go back
    A.free_list[F + all - 1 - e] = *entry;
    *entry = 0;
  }
  if (!map_last(A.state)) return;
#pragma unroll
  for (int k = 0; k < kMapPer; ++k) {
    const int i = t * kMapPer + k;
    if (i < A.batch) A.lens[i] = keep[k];
  }
  if (t == 0) {
    A.state[kStFree] = F + all;
    A.state[kStArrived] = 0;
  }
}

}  // namespace luc

extern "C" __global__ __launch_bounds__(1024) void luc_block_extend(luc::MapArgs a) {
  luc::extend_impl(a);
}
extern "C" __global__ __launch_bounds__(1024) void luc_block_truncate(luc::MapArgs a) {
  luc::truncate_impl(a);
}
