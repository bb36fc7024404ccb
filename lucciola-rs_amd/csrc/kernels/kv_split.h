// What the attention kernels over quantised caches share (gfx950): a batch's sequences, the order
// of their splits, accesses of the workspace of partial results and the merge of a columns launch's.  Args:
// the kernels' argument structs, whose fields of one name are one thing.
#pragma once
#include "luc_common.h"

namespace luc {

typedef float f32x4_t __attribute__((ext_vector_type(4)));

// A sequence's rows, the position of the first, and its context: 0 where that is longer, or the
// rows are more, than the call allows, or the position is none.
struct KvSeq {
  int row0, rows, start, ctx;
};
template <class Args>
__device__ inline KvSeq kv_seq(const Args& A, int b) {
  KvSeq s;
  s.row0 = A.cu_seqlens ? A.cu_seqlens[b] : b;
  const int end = A.cu_seqlens ? A.cu_seqlens[b + 1] : b + 1;
  s.row0 = min(max(s.row0, 0), A.total_rows);
  s.rows = max(min(end, A.total_rows) - s.row0, 0);
  s.start = A.start_pos[b];
  const int64_t ctx = (int64_t)s.start + s.rows;
  s.ctx = s.start >= 0 && ctx <= A.max_ctx && s.rows <= A.max_rows ? (int)ctx : 0;
  return s;
}
// The rows of a sequence without a context: NaN.
template <int DT, int D, class Args>
__device__ inline void kv_no_context(const Args& A, const KvSeq& S, int kvh) {
  const int width = A.group * D;
  for (int64_t i = threadIdx.x; i < (int64_t)S.rows * width; i += blockDim.x)
    A.out[(S.row0 + i / width) * A.out_stride + (int64_t)kvh * width + i % width] = St<DT>::store(__builtin_nanf(""));
}

// (agent scope: read by a workgroup of another XCD)
__device__ inline void ws_put(float* p, float x) {
  __hip_atomic_store(p, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ inline float ws_get(const float* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// 16-byte agent-scope accesses of the workspace (sc1, as the scoped atomics above).
__device__ inline __amdgpu_buffer_rsrc_t ws_rsrc(const float* p) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, 0x7fffffff, 0x00020000);
}
constexpr int kAuxSc1 = 16;
__device__ inline float4 ws_get4(__amdgpu_buffer_rsrc_t r, int at) {  // at: floats
  return __builtin_bit_cast(float4, __builtin_amdgcn_raw_buffer_load_b128(r, at * 4, 0, kAuxSc1));
}
__device__ inline void ws_put4(__amdgpu_buffer_rsrc_t r, int at, float4 x) {
  __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_t, x), r, at * 4, 0, kAuxSc1);
}

constexpr int kTokWaves = 4;
constexpr int kTokCols = 8;   // columns of a workgroup
constexpr int kTokMaxSplits = 256;

// The work of workgroup blockIdx.x where there are more than fit the chip at once: full splits
// first, then the sequences' last ones, longest first, so that the launch does not end on full splits
// that started late (plain order deals a split of every sequence in turn).  At most 64 sequences, one a
// lane; one tile a sequence.  False: no work.
template <class Args>
__device__ inline bool kv_longest_first(const Args& A, KvSeq& S, int& split, int& b, int& kvh) {
  const int lane = threadIdx.x & 63;
  KvSeq own{};
  if (lane < A.batch) own = kv_seq(A, lane);
  const int full = own.rows ? own.ctx / A.split_tokens : 0;
  // (no context: the rows still get their NaN, from split 0)
  const int rest = own.rows && (own.ctx == 0 || own.ctx % A.split_tokens) ? own.ctx % A.split_tokens : -1;
  int end = full * A.hkv;
#pragma unroll
  for (int k = 1; k < 64; k <<= 1) {
    const int y = __shfl_up(end, k);
    if (lane >= k) end += y;
  }
  int i = blockIdx.x;
  const int all = __builtin_amdgcn_readlane(end, 63);
  if (i < all) {
    b = __builtin_ctzll(__ballot(i < end));
    i -= __builtin_amdgcn_readlane(end - full * A.hkv, b);
    split = i / A.hkv;
  } else {
    i -= all;
    int rank = 0;
    for (int k = 0; k < A.batch; ++k) {
      const int r = __builtin_amdgcn_readlane(rest, k);
      rank += r > rest || (r == rest && k < lane);
    }
    const uint64_t at = __ballot(rest >= 0 && rank == i / A.hkv);
    if (!at) return false;
    b = __builtin_ctzll(at);
    split = __builtin_amdgcn_readlane(full, b);
  }
  kvh = i % A.hkv;
  S.row0 = __builtin_amdgcn_readlane(own.row0, b);
  S.rows = __builtin_amdgcn_readlane(own.rows, b);
  S.start = __builtin_amdgcn_readlane(own.start, b);
  S.ctx = __builtin_amdgcn_readlane(own.ctx, b);
  return true;
}

// The partials of a columns launch: D / 4 lanes a (row, head).
template <int DT, int D, class Args>
__device__ void kv_merge_impl(const Args& A) {
  constexpr int LANES = D / 4;
  const int hq = A.hkv * A.group;
  const int64_t item = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) / LANES;
  const int d = threadIdx.x % LANES * 4;
  if (item >= (int64_t)A.total_rows * hq) return;
  const int row = (int)(item / hq), head = (int)(item % hq);
  int b = row;
  if (A.cu_seqlens) {
    int lo = 0, hi = A.batch - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (A.cu_seqlens[mid] <= row) lo = mid; else hi = mid - 1;
    }
    b = lo;
  }
  const KvSeq S = kv_seq(A, b);
  const int r = row - S.row0;
  if (r < 0 || r >= S.rows || S.ctx == 0) return;  // no sequence's row, or written already
  const int nsplit = min(A.splits, (S.start + r) / A.split_tokens + 1);
  const int64_t step = (int64_t)A.total_rows * hq;
  float M = -3.4028235e38f, L = 0.0f;
  float4 o = make_float4(0, 0, 0, 0);
  // eight splits' loads under way at once (those past the last read the last again, times 0)
  for (int s0 = 0; s0 < nsplit; s0 += 8) {
    float2 ml[8];
    float4 x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t at = item + min(s0 + i, nsplit - 1) * step;
      ml[i] = *(const float2*)(A.ws_ml + at * 2);
      x[i] = *(const float4*)(A.ws_o + at * D + d);
    }
    float top = M;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = fmaxf(top, ml[i].x);
    const float a = __builtin_amdgcn_exp2f(M - top);
    M = top;
    L *= a;
    o.x *= a; o.y *= a; o.z *= a; o.w *= a;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float e = s0 + i < nsplit ? __builtin_amdgcn_exp2f(ml[i].x - M) : 0.0f;
      L = fmaf(e, ml[i].y, L);
      o.x = fmaf(e, x[i].x, o.x); o.y = fmaf(e, x[i].y, o.y); o.z = fmaf(e, x[i].z, o.z); o.w = fmaf(e, x[i].w, o.w);
    }
  }
  const float inv = 1.0f / L;
  const uint32_t a0 = St<DT>::store(o.x * inv) | (uint32_t)St<DT>::store(o.y * inv) << 16;
  const uint32_t a1 = St<DT>::store(o.z * inv) | (uint32_t)St<DT>::store(o.w * inv) << 16;
  *(uint2*)(A.out + row * A.out_stride + (int64_t)head * D + d) = make_uint2(a0, a1);
}

}  // namespace luc
