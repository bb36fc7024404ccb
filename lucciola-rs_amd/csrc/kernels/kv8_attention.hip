// Attention of new rows over the 8-bit paged cache of kv8.h (gfx950):
//   o = sum_t softmax_t(sm_scale q . k_t) v_t,  t = 0 .. the row's own position,
// for the rows of a batch of sequences: one row each (a decode step; the reference's flash_decoding
// kernel, src/kernels/attention.cu:4-240, over its 16-bit cache) or packed prompts; or, for one row
// each, over the tokens of chosen pages (kv8_select.hip).
//
// Columns.  The (row, head of the group) pairs of one sequence and kv head are the columns of
// the products: S^T = K Q^T and O^T += V^T P^T on v_mfma_f32_16x16x32_{f16,bf16}, 16 columns a fragment.
// In the accumulators a lane has one column throughout (column lane % 16), so maxima, sums and
// rescaling are lane-local up to the four lanes that share it, and the scores of two pages are
// already the operand of the second product: lane l holds four tokens of either.  Codes become 16-bit values, scale
// included, in one conversion a pair, exactly (fp16: where the value is one; below 2^-14 it rounds to fp16's 2^-24).
// Weights are rounded to the rows' type, which the matrix unit takes, and summed as rounded, and held times a power of two,
// far above fp16's smallest.  That is all of the error beyond the output's own rounding (2.3e-4 of fp16's outputs for 2.1e-4
// with weights in f32, 1.9e-3 for 1.7e-3 of bf16's); a second part for what the rounding takes away would double V's
// products.  The running maximum moves only when a score passes it by some powers of two, so most tiles
// rescale nothing.
//
// NaN.  Tokens that no column of a tile sees, and tokens that only some see, have weight 0 there, and 0 times what
// is not finite would reach the columns that do not see it: in tiles with a limit inside, such values of V are
// taken out, and a product of their places with the columns' view puts NaN where one is seen.
//
// Two kernels:
//   tokens: 8 columns a workgroup; its 4 waves take stages of tokens in turn and merge in LDS.  Few
//     columns a sequence (decode): every wave streams its own part of the cache into registers, in operand order.
//   columns: 128 (D = 64) or 256 columns a workgroup, every wave walks all tokens of its columns'
//     contexts.  Prompts: a tile of K and V in 16 bits serves all of them.
// Either may cut the context into splits over workgroups, whose partial (m, l, o) go to the
// workspace; tokens: the last workgroup of a (sequence, kv head, column tile) to arrive
// merges them; columns: a second launch does.
//
// What bounds them (us).  Tokens: HBM where contexts are long: 64 rows over 1024 to 16384 tokens, 4 kv heads of 128, 110 for
// 612 MB, 5.6 TB/s; a gather of the same slabs without arithmetic takes 96, a copy's rate 120.  Loads marked as
// streamed: 110, 120 without.  No slower with two workgroups a CU than with three; K by 1 KB a wave
// in another slab order 108.  The first 512 workgroups read 6.7 TB/s, the tail from 75 us on is what is lost.  Few tokens: a
// chain of round trips, lengths -> table -> scale, K -> products -> merge of the waves, and of splits by way of the
// workspace: 5.6 for 512 tokens, 11 for 32 rows over up to 4096, 21.6 for 96 chosen pages of each of 64 contexts (100 MB).
// Columns: issue.  512 rows after 8000, 12 / 2 heads of 128 (fp16): 36.6 and 7.7 for the merge of ten splits, 31 MB each
// way; four prompts of 1531 to 2048, 14 / 2 heads of 64 (bf16): 40.4; matrix instructions busy 38% and 32% of the SIMDs'
// time, VALU instructions, two thirds of their cycles exponentials, 47% and 64%: the two hardly run at once whatever the
// waves.  1024 rows at the end of 32768 tokens, 28 / 4 heads of 128: 455, 1040 TFLOP/s; with the two waves of a SIMD a phase
// apart by barriers, one's products beside the other's softmax, 475.  Both halves of a tile at a time spill (53 for the first
// case), wave priorities changed nothing; chunks of columns in serpentine order of their lengths 40.4, in plain order 42.6.
#include "kv8.h"
#include "kv_split.h"

namespace luc {

struct Kv8AttnArgs {
  const uint16_t* q;
  int64_t q_stride;
  uint16_t* out;
  int64_t out_stride;
  const char* k_pool;
  const char* v_pool;
  const float2* scales;       // of K and V
  const int32_t* tables;
  int64_t table_stride;
  const int32_t* cu_seqlens;  // or null: row b is sequence b's one row
  const int32_t* start_pos;   // position of a sequence's first row
  const int32_t* chosen;      // tokens over chosen pages: [batch][hkv][budget] pages of the context, ascending
  int32_t* ws_cnt;
  float* ws_ml;
  float* ws_o;
  int32_t batch, total_rows, max_rows, max_ctx, layer, num_layers, hkv, group, num_blocks, budget;
  int32_t tiles;         // column tiles (chunks) per (sequence, kv head)
  int32_t splits, split_tokens;
  int32_t longest_first;
  float qk_scale_log2;
};

// The running maximum moves when a score (in powers of two) passes it by this, and weights are held times 2^lift:
// 2^15 at most.
constexpr float kKv8TokLazy = 3.0f, kKv8TokLift = 12.0f;
constexpr float kKv8ColsLazy = kLazyMax, kKv8ColsLift = 15.0f - kLazyMax;
// What a largest score (in powers of two) makes the running maximum, less the lift: none where a rounding of the
// score itself is as much as the room that the lift leaves below 2^16.
__device__ inline float kv8_reference(float score, float lift) {
  return fabsf(score) < 0x1p23f ? score - lift : score;
}

template <int DT>
__device__ inline f32x4_t mfma16(uint4 a, uint4 b, f32x4_t c) {
  if constexpr (DT == kF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
// Two values rounded to the type, nearest even; 1.0 twice.
template <int DT>
__device__ inline uint32_t pack2(float a, float b) {
  if constexpr (DT == kF16) return __builtin_bit_cast(uint32_t, (half2_t){(_Float16)a, (_Float16)b});
  else return __builtin_bit_cast(uint32_t, (bf162_t){(__bf16)a, (__bf16)b});
}
template <int DT> constexpr uint32_t kOnes = DT == kF16 ? 0x3c003c00u : 0x3f803f80u;

// Of a pair, the halves that are not finite: all ones.
template <int DT>
__device__ inline uint32_t not_finite(uint32_t w) {
  const uint32_t t = ((w & 0x7fff7fffu) + (DT == kF16 ? 0x04000400u : 0x00800080u)) & 0x80008000u;
  return (t >> 15) * 0xffffu;
}
template <int DT>
__device__ inline uint4 not_finite4(uint4 a) {
  return make_uint4(not_finite<DT>(a.x), not_finite<DT>(a.y), not_finite<DT>(a.z), not_finite<DT>(a.w));
}

// max3 that is NaN where one is.  (fmaxf, which passes over it, would first quiet every operand.)
__device__ inline float max3(float a, float b, float c) {
  return __builtin_elementwise_maximum(__builtin_elementwise_maximum(a, b), c);
}

// Eight codes times their scale: an operand.
template <int DT>
__device__ inline uint4 expand8(uint32_t a, uint32_t b, float scale) {
  return make_uint4(kv8_pair<DT, false>(a, scale), kv8_pair<DT, true>(a, scale), kv8_pair<DT, false>(b, scale),
                    kv8_pair<DT, true>(b, scale));
}

// q of a lane's column as the operand of a score: step j is dimensions 64 (j / 2) + 16 g + 8 (j % 2) .. + 7.  The
// scale's sign goes to q, so that the largest product is the largest score.
template <int D>
__device__ inline void load_q(const Kv8AttnArgs& A, int64_t row, int head, int g, bool on, uint4 (&q)[D / 32]) {
  const uint16_t* const src = A.q + row * A.q_stride + (int64_t)head * D + 16 * g;
  const uint32_t flip = A.qk_scale_log2 < 0.0f ? 0x80008000u : 0u;
#pragma unroll
  for (int j = 0; j < D / 32; ++j) {
    const uint4 w = on ? *(const uint4*)(src + 64 * (j >> 1) + 8 * (j & 1)) : make_uint4(0, 0, 0, 0);
    q[j] = make_uint4(w.x ^ flip, w.y ^ flip, w.z ^ flip, w.w ^ flip);
  }
}
__device__ inline float score_scale(const Kv8AttnArgs& A) {
  const float s = fabsf(A.qk_scale_log2);
  return s == 0.0f ? 1e-37f : s;  // (a masked product, -inf, times 0 is NaN)
}

// ---- stages: what a wave takes at once, 8 KB of 32 (D = 128) or 64 (D = 64) tokens, in operand order: K token n of
// the page, dimensions 64 h + 16 g .. + 15; V dimensions 64 h + 4 n .. + 3 of tokens 4 g .. 4 g + 3.
template <int D> struct Kv8Stage {
  static constexpr int SUB = D == 128 ? 1 : 2;  // 32-token sub-tiles
  static constexpr int TOKENS = 32 * SUB, PAGES = 2 * SUB, H = D / 64;
};
// Numbers that are alike in all lanes come by the scalar cache, past the queue of the cache's own loads.
typedef __attribute__((address_space(4))) const int32_t scalar_i32;
typedef __attribute__((address_space(4))) const float scalar_f32;

// One wave's 8 columns over stages.  Of a fragment's 16 columns the lower 8 take the first page's tokens
// and the upper 8, the same rows and heads again, the second's: a lane has 4 tokens of one column, and
// softmax costs half of what 16 columns would.  The two halves of a column are partial results
// like those of two waves.
template <int DT, int D> struct Kv8Row {
  using Stage = Kv8Stage<D>;
  static constexpr int KS = D / 32, NF = D / 16, H = D / 64, SUB = Stage::SUB, PAGES = Stage::PAGES;
  uint4 q[KS];
  f32x4_t acc[NF];  // O^T: row 4 g + r of fragment 4 h + c is dimension 64 h + 16 g + 4 r + c
  float s[SUB][4];  // scores of the stage
  float m, l, scale;  // m: less the lift
  float bar;          // products above it move m
  int limit;
  int n, g;
  uint32_t mask[2];   // of the first and the second page's tokens in P: the lane's or 0

  __device__ __attribute__((always_inline)) inline void begin(const Kv8AttnArgs& A, int64_t row0, int kvh, int start, int ctx, int col0,
                                                              int ncols) {
    const int lane = threadIdx.x & 63;
    n = lane & 15;
    g = lane >> 4;
    mask[0] = n >> 3 ? 0 : ~0u;
    mask[1] = ~mask[0];
    const int col = col0 + (n & 7);
    const bool on = col < ncols;
    const int r = on ? col / A.group : 0, hd = on ? col % A.group : 0;
    limit = on ? start + r : ctx - 1;
    load_q<D>(A, row0 + r, kvh * A.group + hd, g, on, q);
    scale = score_scale(A);
    m = -3.4028235e38f;
    bar = -INFINITY;
    l = 0.0f;
#pragma unroll
    for (int i = 0; i < NF; ++i) acc[i] = (f32x4_t){0, 0, 0, 0};
  }

  // Products with a stage's K; sk: its pages' scales.
  __device__ __attribute__((always_inline)) inline void score(const uint4 (&k)[PAGES][H], const float (&sk)[PAGES]) {
#pragma unroll
    for (int u = 0; u < SUB; ++u) {
      f32x4_t x[2];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        x[b] = (f32x4_t){0, 0, 0, 0};
#pragma unroll
        for (int h = 0; h < H; ++h) {
          const uint4 w = k[2 * u + b][h];
          x[b] = mfma16<DT>(expand8<DT>(w.x, w.y, sk[2 * u + b]), q[2 * h], x[b]);
          x[b] = mfma16<DT>(expand8<DT>(w.z, w.w, sk[2 * u + b]), q[2 * h + 1], x[b]);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) s[u][i] = mask[0] ? x[0][i] : x[1][i];
    }
  }

  // The lane's tokens up to this one of sub-tile u are seen (tok0: the stage's first).
  __device__ inline int room(int tok0, int u) const { return limit - tok0 - 32 * u - 4 * g - (mask[0] ? 0 : kPage); }

  // Softmax and the products with a stage's V; sv: its pages' scales.  EDGE: some column's limit lies before the
  // stage's last token.
  template <bool EDGE>
  __device__ __attribute__((always_inline)) inline void add(const uint4 (&v)[PAGES][H], const float (&sv)[PAGES], int tok0) {
    if constexpr (EDGE) {
#pragma unroll
      for (int u = 0; u < SUB; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[u][i] = i <= room(tok0, u) ? s[u][i] : -INFINITY;
    }
    float top = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3]));
    if constexpr (SUB == 2) top = fmaxf(top, fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
    if (__any(top > bar)) {
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      const float mn = fmaxf(m, kv8_reference(top * scale, kKv8TokLift));
      const float a = __builtin_amdgcn_exp2f(m - mn);
      bar = fmaxf(bar, top + kKv8TokLazy / scale);
      m = mn;
      l *= a;
#pragma unroll
      for (int i = 0; i < NF; ++i) acc[i] *= a;
    }
    uint4 p[SUB];
#pragma unroll
    for (int u = 0; u < SUB; ++u) {
      uint32_t w[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        w[i] = pack2<DT>(__builtin_amdgcn_exp2f(fmaf(s[u][2 * i], scale, -m)), __builtin_amdgcn_exp2f(fmaf(s[u][2 * i + 1], scale, -m)));
        l = St<DT>::dot2(w[i], kOnes<DT>, l);
      }
      p[u] = make_uint4(w[0] & mask[0], w[1] & mask[0], w[0] & mask[1], w[1] & mask[1]);
    }
#pragma unroll
    for (int u = 0; u < SUB; ++u)
#pragma unroll
      for (int h = 0; h < H; ++h) {
        const uint4 wa = v[2 * u][h], wb = v[2 * u + 1][h];
        const uint32_t a[4] = {wa.x, wa.y, wa.z, wa.w}, b[4] = {wb.x, wb.y, wb.z, wb.w};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint4 vv = make_uint4(kv8_pair<DT, false>(a[c], sv[2 * u]), kv8_pair<DT, true>(a[c], sv[2 * u]),
                                kv8_pair<DT, false>(b[c], sv[2 * u + 1]), kv8_pair<DT, true>(b[c], sv[2 * u + 1]));
          if constexpr (EDGE) {
            const uint4 bad = not_finite4<DT>(vv);
            if (__any((bad.x | bad.y | bad.z | bad.w) != 0)) {
              const int r = room(tok0, u);
              const uint32_t lo = (0 <= r ? kOnes<DT> & 0xffffu : 0u) | (1 <= r ? kOnes<DT> & 0xffff0000u : 0u);
              const uint32_t hi = (2 <= r ? kOnes<DT> & 0xffffu : 0u) | (3 <= r ? kOnes<DT> & 0xffff0000u : 0u);
              const uint4 seen = make_uint4(lo & mask[0], hi & mask[0], lo & mask[1], hi & mask[1]);
              const f32x4_t t = mfma16<DT>(make_uint4(bad.x & kOnes<DT>, bad.y & kOnes<DT>, bad.z & kOnes<DT>, bad.w & kOnes<DT>),
                                           seen, (f32x4_t){0, 0, 0, 0});
#pragma unroll
              for (int i = 0; i < 4; ++i) acc[4 * h + c][i] = t[i] > 0.0f ? __builtin_nanf("") : acc[4 * h + c][i];
              vv = make_uint4(vv.x & ~bad.x, vv.y & ~bad.y, vv.z & ~bad.z, vv.w & ~bad.w);
            }
          }
          acc[4 * h + c] = mfma16<DT>(vv, p[u], acc[4 * h + c]);
        }
      }
  }

  // After the last stage: l over the lanes of a column, NaN where it saw a page outside the pool
  // (bad_at: the first one's position).
  __device__ __attribute__((always_inline)) inline void finish(int bad_at) {
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (limit >= bad_at) l = __builtin_nanf("");
  }
};

// ---- the end of a tokens kernel: kTokWaves waves with partial results of up to kTokCols columns each, twice
// (a wave's columns col and col + kTokCols are parts of one).  mem (kTokMergeBytes of LDS, 16-byte aligned):
// the waves' o, [wave][column][D + 4]; s_m and s_l their maxima and sums.  All of it written, and a
// barrier behind.  The columns of a unit that has one split go out; others go to the workspace, and the last
// workgroup of the unit to arrive merges its splits.  (kv4_attention.hip has the same lines in its kernels, and those of
// kv_columns_out: what is wrong in one is wrong in both.  Through a function they take its tokens kernel of 64 dimensions from 142 to
// 189 registers, and its columns kernels of bf16 spill.)
template <int D> constexpr int kTokMergeBytes = kTokWaves * 2 * kTokCols * (D + 4) * 4;

template <int DT, int D, class Args>
__device__ __attribute__((always_inline)) inline void kv_tokens_finish(const Args& A, const KvSeq& S, int kvh, int unit, int split,
                                                                       int nsplit, int col0, int here, int w, char* mem,
                                                                       float (&s_m)[kTokWaves][2 * kTokCols],
                                                                       float (&s_l)[kTokWaves][2 * kTokCols], int& s_last) {
  constexpr int NW = kTokWaves, NT = 64 * NW, TC = kTokCols;
  constexpr int OS = D + 4;  // floats of a column's row in LDS
  constexpr int Q = D / 4;   // float4s of a column
  float (*const s_o)[2 * TC][OS] = (float (*)[2 * TC][OS])mem;
  // then, in the merge of the splits, the sets' o and the splits' weights
  float4* const s_x = (float4*)mem;
  float (*const s_w)[TC] = (float (*)[TC])(mem + NT * 16);
  static_assert(NT * 16 + kTokMaxSplits * TC * 4 <= kTokMergeBytes<D>, "fits");
  auto store = [&](int col, int d, float4 o, float L) __attribute__((always_inline)) {
    const int c = col0 + col;
    uint16_t* const dst = A.out + (int64_t)(S.row0 + c / A.group) * A.out_stride + ((int64_t)kvh * A.group + c % A.group) * D + d;
    const uint32_t a0 = St<DT>::store(o.x / L) | (uint32_t)St<DT>::store(o.y / L) << 16;
    const uint32_t a1 = St<DT>::store(o.z / L) | (uint32_t)St<DT>::store(o.w / L) << 16;
    *(uint2*)dst = make_uint2(a0, a1);
  };
  // ---- the workgroup's columns
  const int64_t part = (int64_t)unit * A.splits * TC;  // (split, column) records
  const __amdgpu_buffer_rsrc_t po = ws_rsrc(A.ws_o + part * D);
  for (int i = threadIdx.x; i < here * Q; i += NT) {
    const int col = i / Q, d = i % Q * 4;
    float M = fmaxf(s_m[0][col], s_m[0][col + TC]);
#pragma unroll
    for (int k = 1; k < NW; ++k) M = fmaxf(M, fmaxf(s_m[k][col], s_m[k][col + TC]));
    float L = 0.0f;
    float4 o = make_float4(0, 0, 0, 0);
#pragma unroll
    for (int k = 0; k < 2 * NW; ++k) {
      const int c = col + (k & 1) * TC;
      const float e = __builtin_amdgcn_exp2f(s_m[k >> 1][c] - M);
      const float4 x = *(const float4*)&s_o[k >> 1][c][d];
      L = fmaf(e, s_l[k >> 1][c], L);
      o.x = fmaf(e, x.x, o.x); o.y = fmaf(e, x.y, o.y); o.z = fmaf(e, x.z, o.z); o.w = fmaf(e, x.w, o.w);
    }
    if (nsplit == 1) {
      store(col, d, o, L);
    } else {
      ws_put4(po, (split * TC + col) * D + d, o);
      if (d == 0) {
        float* const pm = A.ws_ml + (part + split * TC + col) * 2;
        ws_put(pm, M);
        ws_put(pm + 1, L);
      }
    }
  }
  if (nsplit == 1) return;
  // ---- the last workgroup of the unit to arrive merges its splits
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0)
    s_last = __hip_atomic_fetch_add(A.ws_cnt + unit, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == nsplit - 1;
  __syncthreads();
  if (!s_last) return;
  if (threadIdx.x == 0) __hip_atomic_store(A.ws_cnt + unit, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  // (m, l): lane s of wave w has splits s, s + 64, ... of columns w, w + NW, ...; weights 2^(m_s - M)
  // and l
  constexpr int CW = TC / NW, SL = kTokMaxSplits / 64;
  const int lane = threadIdx.x & 63;
  float mv[CW][SL], lv[CW][SL];
#pragma unroll
  for (int c = 0; c < CW; ++c)
#pragma unroll
    for (int k = 0; k < SL; ++k) {
      const int s = lane + 64 * k;
      const bool on = s < nsplit && w + NW * c < here;
      const float* const pm = A.ws_ml + (part + (on ? s * TC + w + NW * c : 0)) * 2;
      mv[c][k] = on ? ws_get(pm) : -INFINITY;
      lv[c][k] = on ? ws_get(pm + 1) : 0.0f;
    }
  // o: columns x Q float4s, the splits dealt to as many sets of threads as there are; NB loads
  // of a thread under way (the rounds of loads are what a merge takes)
  const int items = here * Q;
  const int sets = max(NT / items, 1);
  constexpr int NB = 8;
  for (int i0 = 0; i0 < items; i0 += NT) {
    const int item = sets > 1 ? threadIdx.x % items : i0 + threadIdx.x;
    const int set = sets > 1 ? threadIdx.x / items : 0;
    const bool on = item < items && set < sets;
    const int col = on ? item / Q : 0, d = on ? item % Q * 4 : 0;
    float4 x[NB];
#pragma unroll
    for (int k = 0; k < NB; ++k) x[k] = ws_get4(po, (min(set + k * sets, nsplit - 1) * TC + col) * D + d);
    if (i0 == 0) {
#pragma unroll
      for (int c = 0; c < CW; ++c) {
        float M = mv[c][0];
#pragma unroll
        for (int k = 1; k < SL; ++k) M = fmaxf(M, mv[c][k]);
        M = wave_max(M);
        float L = 0.0f, e[SL];
#pragma unroll
        for (int k = 0; k < SL; ++k) {
          e[k] = __builtin_amdgcn_exp2f(mv[c][k] - M);
          if (lane + 64 * k < nsplit) L = fmaf(e[k], lv[c][k], L);
        }
        L = wave_sum(L);
        if (w + NW * c < here) {
#pragma unroll
          for (int k = 0; k < SL; ++k)
            if (lane + 64 * k < nsplit) s_w[lane + 64 * k][w + NW * c] = e[k];
          if (lane == 0) s_l[0][w + NW * c] = L;
        }
      }
      __syncthreads();
    }
    float4 o = make_float4(0, 0, 0, 0);
    for (int s0 = set; s0 < nsplit; s0 += NB * sets) {
      if (s0 != set) {
#pragma unroll
        for (int k = 0; k < NB; ++k) x[k] = ws_get4(po, (min(s0 + k * sets, nsplit - 1) * TC + col) * D + d);
      }
#pragma unroll
      for (int k = 0; k < NB; ++k) {
        const int s = s0 + k * sets;
        if (s < nsplit) {
          const float e = s_w[s][col];
          o.x = fmaf(e, x[k].x, o.x); o.y = fmaf(e, x[k].y, o.y); o.z = fmaf(e, x[k].z, o.z); o.w = fmaf(e, x[k].w, o.w);
        }
      }
    }
    if (sets > 1) {  // (one round)
      if (on && set) s_x[set * items + item] = o;
      __syncthreads();
      if (on && !set)
        for (int k = 1; k < sets; ++k) {
          const float4 y = s_x[k * items + item];
          o.x += y.x; o.y += y.y; o.z += y.z; o.w += y.w;
        }
    }
    if (on && !set) store(col, d, o, s_l[0][col]);
  }
}


// ---- waves split tokens: one workgroup per (split, sequence, kv head, 8-column tile).  CHOSEN: a sequence's tokens are
// those of its chosen pages, side by side, the last of them its row's own page.
constexpr int kAuxNt = 2;  // streamed: nothing of it is read again

template <int DT, int D, bool CHOSEN>
__device__ void kv8_tokens_impl(const Kv8AttnArgs& A) {
  constexpr int NW = kTokWaves, TC = kTokCols;
  using Stage = Kv8Stage<D>;
  constexpr int OS = D + 4;  // floats of a column's row in LDS
  __shared__ __attribute__((aligned(16))) char s_mem[kTokMergeBytes<D>];
  __shared__ float s_m[NW][2 * TC], s_l[NW][2 * TC];
  __shared__ int s_last;
  float (*const s_o)[2 * TC][OS] = (float (*)[2 * TC][OS])s_mem;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int split, tile, b, kvh;
  KvSeq S;
  if (!CHOSEN && A.longest_first) {
    if (!kv_longest_first(A, S, split, b, kvh)) return;
    tile = 0;
  } else {
    const int units = A.batch * A.hkv * A.tiles;
    split = blockIdx.x / units;
    const int u = blockIdx.x % units;
    // the tiles of a (sequence, kv head) lie whole pairs apart: where there are eight, on one XCD, whose L2 has the pages
    // for all but the first (two tiles over 16 x 4096 tokens of 8 heads of 128: 39.0 us, side by side 48.2)
    const int pairs = A.batch * A.hkv;
    tile = u / pairs;
    b = u % pairs / A.hkv;
    kvh = u % A.hkv;
    S = kv_seq(A, b);
  }
  const int unit = (b * A.hkv + kvh) * A.tiles + tile;
  const int col0 = tile * TC, ncols = S.rows * A.group;
  const int here = min(TC, ncols - col0);
  if (S.ctx == 0) {
    if (split == 0 && tile == 0) kv_no_context<DT, D>(A, S, kvh);
    return;
  }
  if (here <= 0) return;
  const int own_page = S.start / kPage;  // (CHOSEN: of the one row)
  if constexpr (CHOSEN) {  // positions among the chosen tokens
    S.start = (min(own_page + 1, A.budget) - 1) * kPage + S.start % kPage;
    S.ctx = S.start + 1;
  }
  const int last_row = (col0 + here - 1) / A.group;
  const int last = S.start + last_row;  // the last position that a column here sees
  const int begin = split * A.split_tokens;
  const int nsplit = min(A.splits, last / A.split_tokens + 1);
  if (begin > last) return;
  const int end = min(last + 1, begin + A.split_tokens);

  // ---- the wave's stages: w, w + NW, ... of the split
  Kv8Row<DT, D> W;
  W.begin(A, S.row0, kvh, S.start, S.ctx, col0, ncols);
  constexpr int PAGES = Stage::PAGES, H = Stage::H;
  const uint32_t page_stride = (uint32_t)(A.num_layers * A.hkv) * Kv8<D>::kSlab;
  const int64_t base = (int64_t)A.layer * A.hkv + kvh;
  const char* const kp = A.k_pool + base * Kv8<D>::kSlab;
  const char* const vp = A.v_pool + base * Kv8<D>::kSlab;
  scalar_f32* const sp = (scalar_f32*)(A.scales + base);
  scalar_i32* const table = (scalar_i32*)(A.tables + (int64_t)b * A.table_stride);
  scalar_i32* const chosen = CHOSEN ? (scalar_i32*)(A.chosen + ((int64_t)b * A.hkv + kvh) * A.budget) : nullptr;
  const int stages = (end - begin + Stage::TOKENS - 1) / Stage::TOKENS;
  const int count = stages > w ? (stages - w + NW - 1) / NW : 0;
  const int min_limit = S.start + col0 / A.group;
  const int last_page = (end - 1) / kPage;
  int bad_at = 0x7fffffff;
  auto first_of = [&](int i) __attribute__((always_inline)) { return begin + (i * NW + w) * Stage::TOKENS; };
  // Numbers of a stage's pages in the context, and in the pool (those behind the last: the last again).  All of
  // these are loads of the scalar cache, whose results are used a stage later.
  auto list = [&](int i, int (&at)[PAGES]) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < PAGES; ++k) {
      const int p = min(first_of(min(i, count - 1)) / kPage + k, last_page);
      at[k] = CHOSEN ? chosen[p] : p;
    }
  };
  auto look_up = [&](int i, const int (&at)[PAGES], int (&id)[PAGES]) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < PAGES; ++k) {
      int p = at[k];
      if constexpr (CHOSEN) {
        // a list that does not ascend to the row's own page is no selection
        const int j = min(first_of(min(i, count - 1)) / kPage + k, last_page);
        const bool ok = j == last / kPage ? p == own_page : p >= 0 && p < own_page;
        if (!ok) {
          p = 0;
          bad_at = 0;
        }
      }
      id[k] = table[p];
    }
  };
  // a page outside the pool is never an address: page 0 is read instead
  auto check = [&](int i, int (&id)[PAGES]) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < PAGES; ++k)
      if (id[k] < 0 || id[k] >= A.num_blocks) {
        id[k] = 0;
        bad_at = min(bad_at, min(first_of(min(i, count - 1)) / kPage + k, last_page) * kPage);
      }
  };
  const int lane = threadIdx.x & 63;
  const int k_off = Kv8<D>::k_at(lane & 15, 16 * (lane >> 4)), v_off = Kv8<D>::v_at(lane >> 4, 4 * (lane & 15));
  // loads of no bytes where there is no stage (on: 0): a branch around them would make every wait for them one for all
  auto load = [&](uint4 (&x)[PAGES][H], const char* pool, int off, int step, const int (&id)[PAGES], bool on) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < PAGES; ++k) {
      const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(
          (void*)(pool + (uint64_t)(uint32_t)id[k] * page_stride), 0, on ? Kv8<D>::kSlab : 0, 0x00020000);
#pragma unroll
      for (int h = 0; h < H; ++h)
        x[k][h] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(r, off + step * h, 0, kAuxNt));
    }
  };
  auto scales_of = [&](const int (&id)[PAGES], float (&sk)[PAGES], float (&sv)[PAGES]) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < PAGES; ++k) {
      scalar_f32* const x = sp + (int64_t)id[k] * (2 * A.num_layers * A.hkv);
      sk[k] = x[0];
      sv[k] = x[1];
    }
  };
  if (count) {
    uint4 K[PAGES][H], V[PAGES][H];
    int at[PAGES], id[PAGES], next[PAGES];
    float sk[PAGES], sv[PAGES];
    list(0, at);
    look_up(0, at, id);
    list(1, at);
    look_up(1, at, next);
    check(0, id);
    load(K, kp, k_off, 64, id, true);
    __builtin_amdgcn_sched_barrier(0);  // (K's before V's, here as below)
    load(V, vp, v_off, 256, id, true);
    __builtin_amdgcn_sched_barrier(0);
    scales_of(id, sk, sv);
    list(2, at);
    check(1, next);
    for (int i = 0; i < count; ++i) {
      // of the next stage its scales, of the one behind it its pages, on their way while this one is worked on
      float sk2[PAGES], sv2[PAGES];
      int after[PAGES];
      scales_of(next, sk2, sv2);
      look_up(i + 2, at, after);
      list(i + 3, at);
      W.score(K, sk);
      __builtin_amdgcn_sched_barrier(0);
      load(K, kp, k_off, 64, next, i + 1 < count);
      __builtin_amdgcn_sched_barrier(0);
      const int tok0 = first_of(i);
      if (tok0 + Stage::TOKENS - 1 > min_limit) W.template add<true>(V, sv, tok0);
      else W.template add<false>(V, sv, tok0);
      __builtin_amdgcn_sched_barrier(0);
      load(V, vp, v_off, 256, next, i + 1 < count);
      __builtin_amdgcn_sched_barrier(0);
      check(i + 2, after);
#pragma unroll
      for (int k = 0; k < PAGES; ++k) {
        next[k] = after[k];
        sk[k] = sk2[k];
        sv[k] = sv2[k];
      }
    }
  }
  W.finish(bad_at);
  const int n = W.n, g = W.g;
  if (g == 0) {
    s_m[w][n] = W.m;
    s_l[w][n] = W.l;
  }
#pragma unroll
  for (int h = 0; h < D / 64; ++h)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      *(float4*)&s_o[w][n][64 * h + 16 * g + 4 * r] =
          make_float4(W.acc[4 * h][r], W.acc[4 * h + 1][r], W.acc[4 * h + 2][r], W.acc[4 * h + 3][r]);
  __syncthreads();
  kv_tokens_finish<DT, D>(A, S, kvh, unit, split, nsplit, col0, here, w, s_mem, s_m, s_l, s_last);
}

// ---- waves split columns: one workgroup per (chunk of columns, sequence, kv head, split) ----
//
// The waves expand a tile of 64 tokens together into LDS in operand order (a lane's 16 bytes
// of every operand side by side: reads without conflicts), one tile ahead of the products and with
// the loads of another under way; one barrier a tile.  A wave has 32 columns; all of K's and V's reads of 32
// tokens are under way before the products and the softmax that need them.
template <int D> struct Kv8Tile {
  static constexpr int KS = D / 32;   // k steps of a score
  static constexpr int NF = D / 16;   // output fragments
  uint4 k[4][KS][64];                 // [page][step][lane]
  uint4 v[2][NF][64];                 // [half][fragment of dimensions][lane]
};
template <int D> struct Kv8Cols {
  static constexpr int WAVES = D == 128 ? 8 : 4;
  // Fragments of a wave.  Four of D = 64 read LDS half as often, with 246 registers: 1024 rows on 32768 tokens (14 / 2 heads)
  // 136 us, 171 with two, but 512 on 8512 41.5 and 37.6, 8192 on themselves 199 and 139: longer chains that end later.
  static constexpr int F = 2;
  static constexpr int N = WAVES * F * 16;
};

// What a wave loads of a tile and makes of it: of page w % 4, 64 dimensions (the w / 4'th) of K and V, 16
// bytes of each a lane.  One page: its address is scalar.
template <int DT, int D> struct Kv8Expand {
  uint4 k, v;
  const char* kp;  // page 0
  const char* vp;
  int ko, vo;      // of the lane in a page
  int page, part;

  __device__ __attribute__((always_inline)) inline void begin(const char* k_pool, const char* v_pool, int wave) {
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    page = wave & 3;
    part = wave >> 2;
    kp = k_pool;
    vp = v_pool;
    ko = Kv8<D>::k_at(n, 64 * part + 16 * g);
    vo = Kv8<D>::v_at(g, 64 * part + 4 * n);
  }
  // p (alike in all lanes): the page.
  __device__ __attribute__((always_inline)) inline void load(int p, uint32_t page_stride) {
    const uint64_t at = (uint64_t)(uint32_t)p * page_stride;
    k = *(const uint4*)(kp + at + ko);
    v = *(const uint4*)(vp + at + vo);
  }
  __device__ __attribute__((always_inline)) inline void store(Kv8Tile<D>& T, float2 scale) {
    const int lane = threadIdx.x & 63;
    T.k[page][2 * part][lane] = expand8<DT>(k.x, k.y, scale.x);
    T.k[page][2 * part + 1][lane] = expand8<DT>(k.z, k.w, scale.x);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int c = 0; c < 4; ++c)
      ((uint2*)&T.v[page >> 1][4 * part + c][lane])[page & 1] =
          make_uint2(kv8_pair<DT, false>(w[c], scale.y), kv8_pair<DT, true>(w[c], scale.y));
  }
};

// One wave's F fragments of 16 columns over tiles.
template <int DT, int D> struct Kv8Chunk {
  static constexpr int F = Kv8Cols<D>::F, KS = D / 32, NF = D / 16;
  uint4 q[F][KS];
  f32x4_t acc[F][NF], l[F];
  float m[F], bar[F], scale;  // m: less kKv8ColsLift
  int limit[F];  // last position that the lane's column sees
  int lane, n, g;

  // Columns col0 + 16 f + n of a sequence with ncols of them whose first row is at `start`.
  __device__ __attribute__((always_inline)) inline void begin(const Kv8AttnArgs& A, int64_t row0, int kvh, int start, int ctx, int col0,
                                                              int ncols) {
    lane = threadIdx.x & 63;
    n = lane & 15;
    g = lane >> 4;
    scale = score_scale(A);
#pragma unroll
    for (int f = 0; f < F; ++f) {
      const int col = col0 + 16 * f + n;
      const bool on = col < ncols;
      const int r = on ? col / A.group : 0, hd = on ? col % A.group : 0;
      limit[f] = on ? start + r : ctx - 1;
      load_q<D>(A, row0 + r, kvh * A.group + hd, g, on, q[f]);
      m[f] = -3.4028235e38f;
      bar[f] = -INFINITY;
      l[f] = (f32x4_t){0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < NF; ++i) acc[f][i] = (f32x4_t){0, 0, 0, 0};
    }
  }

  // Half `half` of a tile: tokens tok0 .. tok0 + 31.  edge (alike in all lanes): some column's limit
  // lies before its end.
  __device__ __attribute__((always_inline)) inline void step(const Kv8Tile<D>& T, int half, int tok0, bool edge) {
    const f32x4_t zero = {0, 0, 0, 0};
    float s[F][8];  // tokens 4 g .. 4 g + 3 of either page
    // all of K's reads under way before the first product, all of V's before the softmax
    uint4 kk[2][KS];
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int j = 0; j < KS; ++j) kk[b][j] = T.k[2 * half + b][j][lane];
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      f32x4_t t[F];
#pragma unroll
      for (int j = 0; j < KS; ++j)
#pragma unroll
        for (int f = 0; f < F; ++f) t[f] = mfma16<DT>(kk[b][j], q[f][j], j == 0 ? zero : t[f]);
#pragma unroll
      for (int f = 0; f < F; ++f)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[f][4 * b + i] = t[f][i];
    }
    uint4 vv[NF];
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < NF; ++i) vv[i] = T.v[half][i][lane];
    __builtin_amdgcn_sched_barrier(0);
    if (edge) {
#pragma unroll
      for (int f = 0; f < F; ++f) {
        const int room = limit[f] - tok0 - 4 * g;
#pragma unroll
        for (int i = 0; i < 8; ++i) s[f][i] = 16 * (i >> 2) + (i & 3) <= room ? s[f][i] : -INFINITY;
      }
    }
    float top[F];
    bool over = false;
#pragma unroll
    for (int f = 0; f < F; ++f) {
      top[f] = max3(max3(s[f][0], s[f][1], s[f][2]), max3(s[f][3], s[f][4], s[f][5]), max3(s[f][6], s[f][7], s[f][7]));
      over |= top[f] > bar[f];
    }
    if (__any(over)) {
#pragma unroll
      for (int f = 0; f < F; ++f) {
        float t = fmaxf(top[f], __shfl_xor(top[f], 16));
        t = fmaxf(t, __shfl_xor(t, 32));
        const float mn = fmaxf(m[f], kv8_reference(t * scale, kKv8ColsLift));
        const float a = __builtin_amdgcn_exp2f(m[f] - mn);
        bar[f] = fmaxf(bar[f], t + kKv8ColsLazy / scale);
        m[f] = mn;
        l[f] *= a;
#pragma unroll
        for (int i = 0; i < NF; ++i) acc[f][i] *= a;
      }
    }
    uint4 p[F];
#pragma unroll
    for (int f = 0; f < F; ++f) {
      uint32_t o[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        o[i] = pack2<DT>(__builtin_amdgcn_exp2f(fmaf(s[f][2 * i], scale, -m[f])),
                         __builtin_amdgcn_exp2f(fmaf(s[f][2 * i + 1], scale, -m[f])));
      p[f] = make_uint4(o[0], o[1], o[2], o[3]);
    }
    if (edge) {
      uint32_t any = 0;
#pragma unroll
      for (int i = 0; i < NF; ++i) {
        const uint4 bad = not_finite4<DT>(vv[i]);
        any |= bad.x | bad.y | bad.z | bad.w;
      }
      if (__any(any != 0)) unseen(vv, tok0);
    }
    const uint4 ones = make_uint4(kOnes<DT>, kOnes<DT>, kOnes<DT>, kOnes<DT>);
#pragma unroll
    for (int f = 0; f < F; ++f) l[f] = mfma16<DT>(ones, p[f], l[f]);
#pragma unroll
    for (int i = 0; i < NF; ++i)
#pragma unroll
      for (int f = 0; f < F; ++f) acc[f][i] = mfma16<DT>(vv[i], p[f], acc[f][i]);
  }

  // Values of V that are not finite out of the operands, and NaN to the columns that see them.
  __device__ __attribute__((always_inline)) inline void unseen(uint4 (&vv)[NF], int tok0) {
    uint4 seen[F];
#pragma unroll
    for (int f = 0; f < F; ++f) {
      const int room = limit[f] - tok0 - 4 * g;
      uint32_t o[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int t = 16 * (i >> 1) + 2 * (i & 1);
        o[i] = (t <= room ? kOnes<DT> & 0xffffu : 0u) | (t + 1 <= room ? kOnes<DT> & 0xffff0000u : 0u);
      }
      seen[f] = make_uint4(o[0], o[1], o[2], o[3]);
    }
#pragma unroll
    for (int i = 0; i < NF; ++i) {
      const uint4 bad = not_finite4<DT>(vv[i]);
      const uint4 at = make_uint4(bad.x & kOnes<DT>, bad.y & kOnes<DT>, bad.z & kOnes<DT>, bad.w & kOnes<DT>);
#pragma unroll
      for (int f = 0; f < F; ++f) {
        const f32x4_t t = mfma16<DT>(at, seen[f], (f32x4_t){0, 0, 0, 0});
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[f][i][r] = t[r] > 0.0f ? __builtin_nanf("") : acc[f][i][r];
      }
      vv[i] = make_uint4(vv[i].x & ~bad.x, vv[i].y & ~bad.y, vv[i].z & ~bad.z, vv[i].w & ~bad.w);
    }
  }

  // After the last tile: NaN where a column saw a page outside the pool (bad_at: the first one's position).
  __device__ __attribute__((always_inline)) inline void finish(int bad_at) {
#pragma unroll
    for (int f = 0; f < F; ++f)
      if (limit[f] >= bad_at) l[f][0] = __builtin_nanf("");
  }
};

// ---- the end of a columns kernel.  A lane holds 16 dimensions (of each 64) of its wave's F fragments' columns;
// by way of the wave's share of LDS (turn, 4 * D float4s) D / 4 lanes write a column side by side: to the output,
// or as partial results.  W: m, l, acc of a fragment f; dimension 64 h + 16 g + 4 r + c is acc[f][4 h + c][r].
template <int DT, int D, int F, class Args, class W_t>
__device__ __attribute__((always_inline)) inline void kv_columns_out(const Args& A, const KvSeq& S, int kvh, int split, int col0, int ncols,
                                                                     const W_t& W, float4* turn) {
  const int hq = A.hkv * A.group;
#pragma unroll
  for (int f = 0; f < F; ++f) {
    const float inv = A.splits == 1 ? 1.0f / W.l[f][0] : 1.0f;
#pragma unroll
    for (int h = 0; h < D / 64; ++h)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        turn[W.n * (D / 4) + ((16 * h + 4 * W.g + r) ^ W.n)] =
            make_float4(W.acc[f][4 * h][r] * inv, W.acc[f][4 * h + 1][r] * inv, W.acc[f][4 * h + 2][r] * inv,
                        W.acc[f][4 * h + 3][r] * inv);
    if (A.splits > 1 && W.g == 0 && col0 + 16 * f + W.n < ncols) {
      const int col = col0 + 16 * f + W.n;
      const int64_t at = ((int64_t)split * A.total_rows + S.row0 + col / A.group) * hq + kvh * A.group + col % A.group;
      *(float2*)(A.ws_ml + at * 2) = make_float2(W.m[f], W.l[f][0]);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // (lanes read what others wrote)
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      const int c = (64 / (D / 4)) * i + W.lane / (D / 4), part = W.lane % (D / 4);
      const int col = col0 + 16 * f + c;
      const float4 x = turn[c * (D / 4) + (part ^ c)];
      if (col >= ncols) continue;
      const int64_t row = S.row0 + col / A.group;
      const int head = kvh * A.group + col % A.group;
      if (A.splits == 1) {
        const uint32_t a0 = St<DT>::store(x.x) | (uint32_t)St<DT>::store(x.y) << 16;
        const uint32_t a1 = St<DT>::store(x.z) | (uint32_t)St<DT>::store(x.w) << 16;
        *(uint2*)(A.out + row * A.out_stride + (int64_t)head * D + 4 * part) = make_uint2(a0, a1);
      } else {
        *(float4*)(A.ws_o + (((int64_t)split * A.total_rows + row) * hq + head) * D + 4 * part) = x;
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

template <int DT, int D>
__device__ void kv8_columns_impl(const Kv8AttnArgs& A) {
  using C = Kv8Cols<D>;
  constexpr int F = C::F;
  __shared__ Kv8Tile<D> s_tile[2];
  __shared__ int s_bad;  // the first position of a page outside the pool
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // The chunks that see the longest contexts first, and split 0, which every chunk has, before the
  // others; neighbours of a pair on different XCDs (block x runs on XCD x % 8).
  const int pairs = A.batch * A.hkv;
  const int split = blockIdx.x / (pairs * A.tiles);
  int rest = blockIdx.x % (pairs * A.tiles);
  // Every other 256 of them (a workgroup a CU) in reverse, so that the longest of one lot meet the shortest of
  // the next: 4 x 1531..2048 rows, 14 and 2 heads of 64, 40.6 us, 42.6 without
  if ((rest >> 8 & 1) && (rest | 255) < pairs * A.tiles) rest ^= 248;
  const int chunk = A.tiles - 1 - rest / pairs, bh = (rest + rest / pairs) % pairs;
  const int b = bh / A.hkv, kvh = bh % A.hkv;
  const KvSeq S = kv_seq(A, b);
  if (S.ctx == 0) {
    if (split == 0 && chunk == 0) kv_no_context<DT, D>(A, S, kvh);
    return;
  }
  const int ncols = S.rows * A.group;
  const int all0 = chunk * C::N, all = min(C::N, ncols - all0);  // the workgroup's columns
  if (all <= 0) return;
  const int all_last = S.start + (all0 + all - 1) / A.group;
  const int begin = split * A.split_tokens;  // (splits x split_tokens fits: luc_kv8.cpp)
  if (begin > all_last) return;
  const int end = A.splits == 1 ? all_last + 1 : min(all_last + 1, begin + A.split_tokens);
  const int col0 = all0 + w * (16 * F);
  const int here = min(16 * F, ncols - col0);  // the wave's, or none
  const int last = here > 0 ? S.start + (col0 + here - 1) / A.group : -1;
  const int min_limit = S.start + col0 / A.group;
  if (threadIdx.x == 0) s_bad = 0x7fffffff;

  const uint32_t page_stride = (uint32_t)(A.num_layers * A.hkv) * Kv8<D>::kSlab;
  const int64_t base = (int64_t)A.layer * A.hkv + kvh;
  const float2* const sp = A.scales + base;
  const int32_t* const table = A.tables + (int64_t)b * A.table_stride;
  Kv8Expand<DT, D> E;
  E.begin(A.k_pool + base * Kv8<D>::kSlab, A.v_pool + base * Kv8<D>::kSlab, w);
  const int count = (end - begin + 63) / 64;  // tiles
  int bad_at = 0x7fffffff;  // of the wave's pages
  int pages = 0;            // the wave's of tile i + lane, and their scales
  float2 scales;
  float2 scale;             // of the tile under way
  auto load = [&](int i) __attribute__((always_inline)) {
    if ((i & 63) == 0) {
      const int64_t at = begin + (int64_t)(i + (threadIdx.x & 63)) * 64 + 16 * E.page;
      pages = at < end ? table[at / kPage] : 0;
      // a page outside the pool is never an address: page 0 is read instead
      const bool bad = pages < 0 || pages >= A.num_blocks;
      if (__any(bad)) {
        int first = bad ? (int)at : 0x7fffffff;
#pragma unroll
        for (int k = 1; k < 64; k <<= 1) first = min(first, __shfl_xor(first, k));
        if (bad_at == 0x7fffffff && (threadIdx.x & 63) == 0) atomicMin(&s_bad, first);
        bad_at = min(bad_at, first);
        pages = bad ? 0 : pages;
      }
      scales = sp[(int64_t)pages * (A.num_layers * A.hkv)];
    }
    E.load(__builtin_amdgcn_readlane(pages, i & 63), page_stride);
    scale = make_float2(readlane(scales.x, i & 63), readlane(scales.y, i & 63));
  };
  __syncthreads();  // s_bad
  load(0);
  Kv8Chunk<DT, D> W;
  W.begin(A, S.row0, kvh, S.start, S.ctx, min(col0, ncols - 1), ncols);
  E.store(s_tile[0], scale);
  if (count > 1) load(1);
  __syncthreads();
  for (int i = 0; i < count; ++i) {
    const int tok0 = begin + 64 * i;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int t = tok0 + 32 * half;
      if (t <= last) W.step(s_tile[i & 1], half, t, t + 31 > min_limit);
    }
    // (every wave is done with the other tile since the last barrier)
    if (i + 1 < count) {
      E.store(s_tile[(i + 1) & 1], scale);
      if (i + 2 < count) load(i + 2);
      __syncthreads();
    }
  }
  W.finish(s_bad);
  __syncthreads();  // no wave reads the tiles any more
  static_assert(sizeof(s_tile) >= C::WAVES * 4 * D * sizeof(float4), "a share holds 16 columns");
  kv_columns_out<DT, D, F>(A, S, kvh, split, col0, ncols, W, (float4*)s_tile + w * (4 * D));
}

}  // namespace luc

#define LUC_KV8_ATTENTION(DTN, DT, D)                                                            \
  extern "C" __global__ __launch_bounds__(256, D == 64 ? 4 : 3) void luc_kv8_tokens_##DTN##_d##D(luc::Kv8AttnArgs a) {  \
    luc::kv8_tokens_impl<luc::DT, D, false>(a);                                                  \
  }                                                                                              \
  extern "C" __global__ __launch_bounds__(256, D == 64 ? 4 : 3) void luc_kv8_chosen_##DTN##_d##D(luc::Kv8AttnArgs a) {  \
    luc::kv8_tokens_impl<luc::DT, D, true>(a);                                                   \
  }                                                                                              \
  extern "C" __global__ __launch_bounds__(64 * luc::Kv8Cols<D>::WAVES, D == 128 ? 2 : 3) void luc_kv8_columns_##DTN##_d##D(luc::Kv8AttnArgs a) { \
    luc::kv8_columns_impl<luc::DT, D>(a);                                                        \
  }                                                                                              \
  extern "C" __global__ __launch_bounds__(256) void luc_kv8_merge_##DTN##_d##D(luc::Kv8AttnArgs a) {      \
    luc::kv_merge_impl<luc::DT, D>(a);                                                           \
  }
LUC_KV8_ATTENTION(bf16, kBF16, 64)
LUC_KV8_ATTENTION(bf16, kBF16, 128)
LUC_KV8_ATTENTION(f16, kF16, 64)
LUC_KV8_ATTENTION(f16, kF16, 128)
