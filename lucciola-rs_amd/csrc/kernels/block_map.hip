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
// dependent round trips, not bytes.
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

// Inclusive scan over the workgroup of one value per thread; total of all.
__device__ inline int64_t map_scan(int64_t x, int64_t* s_part, int64_t& total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
  for (int k = 1; k < 64; k <<= 1) {
    const int64_t y = __shfl_up((long long)x, k);
    if (lane >= k) x += y;
  }
  if (lane == 63) s_part[w] = x;
  __syncthreads();
  int64_t before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < kMapThreads / 64; ++i) {
    const int64_t y = s_part[i];
    if (i < w) before += y;
    total += y;
  }
  __syncthreads();  // s_part is free again
  return x + before;
}

// The bits that any thread has set.
__device__ inline int map_or(int bits) {
  __shared__ int s_bits;
  if (threadIdx.x == 0) s_bits = 0;
  __syncthreads();
  if (bits) atomicOr(&s_bits, bits);
  __syncthreads();
  return s_bits;
}

// Counts this workgroup in; whether it is the last, once every other one has read
// what the caller is about to write.
__device__ inline bool map_last(int32_t* state) {
  if (gridDim.x == 1) return true;
  __shared__ int s_last;
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    s_last = atomicAdd(state + kStArrived, 1) == (int)gridDim.x - 1;
  }
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
  __shared__ int64_t s_part[kMapThreads / 64];
  const int t = threadIdx.x;
  const int64_t room = A.table_stride * kPage;  // tokens of a table row
  const int F = A.state[kStFree];
  int len[kMapPer], cnt[kMapPer], need[kMapPer];
  int bad = F < 0 || F > A.num_blocks ? kMapBadLength : 0;
  int64_t rows = 0, pages = 0;
#pragma unroll
  for (int k = 0; k < kMapPer; ++k) {
    const int i = t * kMapPer + k;
    len[k] = i < A.batch ? A.lens[i] : 0;
    cnt[k] = i < A.batch ? A.count[i] : 0;
    const int64_t sum = (int64_t)len[k] + cnt[k];
    if (len[k] < 0 || cnt[k] < 0 || len[k] > room) bad |= kMapBadLength;
    else if (sum > room) bad |= kMapTableFull;
    need[k] = (int)((sum + kPage - 1) / kPage - ((int64_t)len[k] + kPage - 1) / kPage);
    rows += cnt[k];
    pages += need[k];
  }
  int64_t all_rows, all_pages;
  const int64_t r_end = map_scan(rows, s_part, all_rows);
  const int64_t p_end = map_scan(pages, s_part, all_pages);
  if (all_rows > A.rows) bad |= kMapNoRows;
  if (all_pages > F) bad |= kMapNoPages;
  int verdict = map_or(bad);
  // sums of rejected lengths mean nothing: only the lengths' own bits are told
  if (verdict & (kMapBadLength | kMapTableFull)) verdict &= kMapBadLength | kMapTableFull;
  if (verdict) {
    for (int r = blockIdx.x * kMapThreads + t; r < A.rows; r += gridDim.x * kMapThreads) {
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
    int c = (int)(r_end - rows), p = (int)(p_end - pages);
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
  const int total = (int)all_rows;
  for (int r = blockIdx.x * kMapThreads + t; r < A.rows; r += gridDim.x * kMapThreads) {
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
    A.state[kStFree] = F - (int)all_pages;
    A.state[kStArrived] = 0;
  }
}

__device__ void truncate_impl(const MapArgs& A) {
  __shared__ int32_t s_gone[kMaxSeqs], s_left[kMaxSeqs];
  __shared__ int64_t s_part[kMapThreads / 64];
  const int t = threadIdx.x;
  const int64_t room = A.table_stride * kPage;
  const int F = A.state[kStFree];
  int keep[kMapPer], left[kMapPer], gone[kMapPer];
  int bad = F < 0 || F > A.num_blocks ? kMapBadLength : 0;
  int64_t pages = 0;
#pragma unroll
  for (int k = 0; k < kMapPer; ++k) {
    const int i = t * kMapPer + k;
    const int len = i < A.batch ? A.lens[i] : 0;
    const int want = i < A.batch ? A.count[i] : 0;
    if (len < 0 || len > room || want < 0) bad |= kMapBadLength;
    keep[k] = min(len, want);
    left[k] = (int)(((int64_t)keep[k] + kPage - 1) / kPage);
    gone[k] = (int)(((int64_t)len + kPage - 1) / kPage) - left[k];
    pages += gone[k];
  }
  int64_t all;
  const int64_t end = map_scan(pages, s_part, all);
  if (F + all > A.num_blocks) bad |= kMapBadLength;  // more pages than the pool has
  const int verdict = map_or(bad);
  if (verdict) {
    if (blockIdx.x == 0 && t == 0) A.state[kStStatus] |= verdict;
    return;
  }
  {
    int g = (int)(end - pages);
#pragma unroll
    for (int k = 0; k < kMapPer; ++k) {
      s_gone[t * kMapPer + k] = g;  // pages given back by the sequences before it
      s_left[t * kMapPer + k] = left[k];
      g += gone[k];
    }
  }
  __syncthreads();
  for (int e = blockIdx.x * kMapThreads + t; e < all; e += gridDim.x * kMapThreads) {
    const int i = map_find(s_gone, A.batch, e);
    int32_t* const entry = A.tables + i * A.table_stride + s_left[i] + (e - s_gone[i]);
    // entry e of the pages in table order is the (all - 1 - e)-th to go back
    A.free_list[F + (int)all - 1 - e] = *entry;
    *entry = 0;
  }
  if (!map_last(A.state)) return;
#pragma unroll
  for (int k = 0; k < kMapPer; ++k) {
    const int i = t * kMapPer + k;
    if (i < A.batch) A.lens[i] = keep[k];
  }
  if (t == 0) {
    A.state[kStFree] = F + (int)all;
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
