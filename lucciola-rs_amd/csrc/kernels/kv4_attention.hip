// Attention of new rows over a 4-bit paged cache (gfx950):
//   o = sum_t softmax_t(sm_scale q . k_t) v_t,  t = 0 .. the row's own position,
// with k_t and v_t the values n * s + m of kv4.h, for the rows of a batch of sequences: one
// row each (a decode step; the reference's flash_decoding kernel, src/kernels/attention.cu:4-240,
// over its 16-bit cache) or packed prompts.
//
// Columns.  The (row, head of the group) pairs of one sequence and kv head are the columns of
// the products: S^T = K Q^T and O^T += V^T P^T on v_mfma_f32_16x16x32_f16, 16 columns a fragment.
// In the accumulators a lane has one column throughout (column lane % 16), so maxima, sums and
// rescaling are lane-local up to the four lanes that share it, and the scores of a tile of
// 32 tokens are already the operand of the second product: lane l holds rows 4 (l / 16) .. + 3 of two
// 16-token fragments, whose tokens are dealt so that those 8 are tokens 8 (l / 16) .. + 7.
//
// Operands.  A lane expands n to fp16 in registers: four n of a dword at a time fall in place of
// the low bits of 1024.0 (or 16 n in those), one packed add or FMA makes them whole, one
// packed FMA applies s and m: 13 VALU instructions for 8 values, no LDS.  K and V are rounded to fp16
// there (2^-11 of the value at most, against a step of 1/15 of the group's range); q is taken to fp16 after
// a power of two brings its largest element into [1, 2), exactly unless an element is 2^-14 of that.
// P is fp16 in (0, 2^kLazyMax], and l sums the rounded P.
//
// Two work splits:
//   tokens: 16 columns a workgroup; its 4 waves take 32-token tiles in turn and merge in LDS.
//     Few columns a sequence (decode): every wave streams its own part of the cache.
//   columns: 64 columns a wave, 4 waves, every wave walks all tiles of its context.  Prompts: an
//     expanded tile serves 4 fragments.
// Either may cut the context into splits over workgroups, whose partial (m, l, o) go to the
// workspace; tokens: the last workgroup of a (sequence, kv head, column tile) to arrive
// merges them; columns: a second launch does.
#include "kv4.h"

namespace luc {

struct Kv4AttnArgs {
  const uint16_t* q;
  int64_t q_stride;
  uint16_t* out;
  int64_t out_stride;
  const char* k_pool;
  const char* v_pool;
  const int32_t* tables;
  int64_t table_stride;
  const int32_t* cu_seqlens;  // or null: row b is sequence b's one row
  const int32_t* start_pos;   // position of a sequence's first row
  int32_t* ws_cnt;
  float* ws_ml;
  float* ws_o;
  int32_t batch, total_rows, max_rows, max_ctx, layer, num_layers, hkv, group, num_blocks;
  int32_t tiles;         // column tiles (chunks) per (sequence, kv head)
  int32_t splits, split_tokens;
  float qk_scale_log2;
};

typedef float f32x4_t __attribute__((ext_vector_type(4)));

__device__ inline f32x4_t mfma16(uint4 a, uint4 b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

__device__ inline half2_t as_h2(uint32_t x) { return __builtin_bit_cast(half2_t, x); }
__device__ inline uint32_t as_u(half2_t x) { return __builtin_bit_cast(uint32_t, x); }

// The four pairs (n i, n i + 4) of a dword's n, times s plus m, as packed fp16.
__device__ inline void expand8(uint32_t w, half2_t s, half2_t m, uint32_t* o) {
  constexpr uint32_t kBig = 0x64006400u;  // 1024.0 twice
  const half2_t big = {(_Float16)1024.0f, (_Float16)1024.0f};
  const half2_t sixteenth = {(_Float16)0.0625f, (_Float16)0.0625f}, less = {(_Float16)-64.0f, (_Float16)-64.0f};
  const uint32_t v = w >> 8;
  const half2_t n0 = as_h2((w & 0x000f000fu) | kBig) - big;
  const half2_t n1 = __builtin_elementwise_fma(as_h2((w & 0x00f000f0u) | kBig), sixteenth, less);
  const half2_t n2 = as_h2((v & 0x000f000fu) | kBig) - big;
  const half2_t n3 = __builtin_elementwise_fma(as_h2((v & 0x00f000f0u) | kBig), sixteenth, less);
  o[0] = as_u(__builtin_elementwise_fma(n0, s, m));
  o[1] = as_u(__builtin_elementwise_fma(n1, s, m));
  o[2] = as_u(__builtin_elementwise_fma(n2, s, m));
  o[3] = as_u(__builtin_elementwise_fma(n3, s, m));
}

// Of a pair of tokens' s and m, bit 15 or 31 where a token's is NaN (the format has no
// infinities: an exponent of all ones is NaN).
__device__ inline uint32_t kv4_nan(uint32_t s, uint32_t m) {
  return (((s & 0x7c007c00u) + 0x04000400u) | ((m & 0x7c007c00u) + 0x04000400u)) & 0x80008000u;
}

// What a lane loads of a 32-token tile.
template <int D> struct Kv4Tile {
  static constexpr int KW = D / 32;  // dwords of K per token (16 or 32 dimensions)
  static constexpr int H = D / 64;   // V quads per lane
  uint32_t k[2][KW];                 // fragments a and b
  uint32_t ksm[2];
  uint4 v[H], vs[H], vm[H];
};

// One wave's walk over tiles for F fragments of 16 columns.
template <int DT, int D, int F> struct Kv4Wave {
  static constexpr int KS = D / 32;  // k steps of a score
  static constexpr int NF = D / 16;  // output fragments: 4 a quad of V
  static constexpr int H = D / 64;

  uint4 q[F][KS];
  f32x4_t acc[F][NF];
  float m[F], l[F], scale[F];
  int limit[F];  // last position that the lane's column sees
  int nan_at[H];  // first NaN value (of a tile at an edge) in the group of the lane's outputs
  int lane, n, g;

  // Columns col0 + 16 f + n of a sequence with ncols of them whose first row is at `start`.
  __device__ __attribute__((always_inline)) inline void begin(const Kv4AttnArgs& A, int64_t row0, int kvh, int start, int ctx, int col0,
                               int ncols) {
    lane = threadIdx.x & 63;
    n = lane & 15;
    g = lane >> 4;
#pragma unroll
    for (int h = 0; h < H; ++h) nan_at[h] = 0x7fffffff;
#pragma unroll
    for (int f = 0; f < F; ++f) {
      const int col = col0 + 16 * f + n;
      const bool on = col < ncols;
      const int r = on ? col / A.group : 0, hd = on ? col % A.group : 0;
      limit[f] = on ? start + r : ctx - 1;
      const uint16_t* const src = A.q + (row0 + r) * A.q_stride + ((int64_t)kvh * A.group + hd) * D + g * (D / 4);
      // the lane's D / 4 dimensions: those of its K loads
      float x[D / 4];
      float top = 0.0f;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        const uint4 w = on ? *(const uint4*)(src + 8 * i) : make_uint4(0, 0, 0, 0);
        const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[8 * i + 2 * e] = St<DT>::lo(ww[e]);
          x[8 * i + 2 * e + 1] = St<DT>::hi(ww[e]);
          top = fmaxf(top, fmaxf(fabsf(x[8 * i + 2 * e]), fabsf(x[8 * i + 2 * e + 1])));
        }
      }
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      // 2^-e of the largest element (infinities and NaN stay what they are)
      const int e = min(max((int)(__float_as_uint(top) >> 23), 1), 253);
      const float down = __uint_as_float((uint32_t)(254 - e) << 23);
      scale[f] = A.qk_scale_log2 * __uint_as_float((uint32_t)e << 23);
#pragma unroll
      for (int j = 0; j < KS; ++j) {
        uint32_t o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const half2_t p = {(_Float16)(x[8 * j + i] * down), (_Float16)(x[8 * j + i + 4] * down)};
          o[i] = as_u(p);
        }
        q[f][j] = make_uint4(o[0], o[1], o[2], o[3]);
      }
      m[f] = -3.4028235e38f;
      l[f] = 0.0f;
#pragma unroll
      for (int i = 0; i < NF; ++i) acc[f][i] = (f32x4_t){0, 0, 0, 0};
    }
  }

  // Byte offsets of the lane's loads within slabs; page: which of the tile's two.
  struct Offsets {
    int k, ksm, v, vs;
    bool kpage, vpage;
  };
  __device__ __attribute__((always_inline)) inline Offsets offsets() const {
    // fragment a's row n is token 8 (n / 4) + n % 4 of the tile, b's 4 further
    const int tok = 8 * (n >> 2) + (n & 3), t = tok & 15;
    Offsets o;
    o.kpage = tok >= 16;
    o.k = Kv4<D>::k_row(t) + g * (D / 8);
    o.ksm = Kv4<D>::k_scale(t, D == 128 ? g : g >> 1);
    o.vpage = g >= 2;
    o.v = Kv4<D>::v_quad(8 * (g & 1), n);
    o.vs = Kv4<D>::v_scale(g & 1, n >> 3);
    return o;
  }
  __device__ __attribute__((always_inline)) inline void load(Kv4Tile<D>& t, const Offsets& o, const char* kp, const char* vp, int64_t page_stride,
                              int p0, int p1) const {
    const char* const kb = kp + (o.kpage ? p1 : p0) * page_stride;
    const char* const vb = vp + (o.vpage ? p1 : p0) * page_stride;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      if constexpr (D == 128) {
        const uint4 x = *(const uint4*)(kb + o.k + b * 4 * (D / 2));
        t.k[b][0] = x.x; t.k[b][1] = x.y; t.k[b][2] = x.z; t.k[b][3] = x.w;
      } else {
        const uint2 x = *(const uint2*)(kb + o.k + b * 4 * (D / 2));
        t.k[b][0] = x.x; t.k[b][1] = x.y;
      }
      t.ksm[b] = *(const uint32_t*)(kb + o.ksm + b * 4 * Kv4<D>::kGroups * 4);
    }
#pragma unroll
    for (int h = 0; h < H; ++h) {
      t.v[h] = *(const uint4*)(vb + o.v + h * 256);       // 16 quads on
      t.vs[h] = *(const uint4*)(vb + o.vs + h * 64);      // two groups on
      t.vm[h] = *(const uint4*)(vb + o.vs + h * 64 + 16);
    }
  }

  // One tile of tokens tok0 .. tok0 + 31.  edge (alike in all lanes): some column's limit lies
  // before its end.
  __device__ __attribute__((always_inline)) inline void step(Kv4Tile<D>& t, int tok0, int ctx, bool edge) {
    // ---- scores
    uint4 ka[2][KS];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const half2_t sm = as_h2(t.ksm[b]);
      const half2_t s = {sm.x, sm.x}, mm = {sm.y, sm.y};
#pragma unroll
      for (int j = 0; j < KS; ++j) {
        uint32_t o[4];
        expand8(t.k[b][j], s, mm, o);
        ka[b][j] = make_uint4(o[0], o[1], o[2], o[3]);
      }
    }
    const int first = tok0 + 8 * g;  // the lane's 8 tokens
    uint4 p[F];
#pragma unroll
    for (int f = 0; f < F; ++f) {
      float s[8];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        f32x4_t c = {0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < KS; ++j) c = mfma16(ka[b][j], q[f][j], c);
#pragma unroll
        for (int i = 0; i < 4; ++i) s[4 * b + i] = c[i] * scale[f];
      }
      if (edge) {
#pragma unroll
        for (int i = 0; i < 8; ++i) s[i] = first + i <= limit[f] ? s[i] : -INFINITY;
      }
      float top = fmaxf(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])), fmaxf(fmaxf(s[4], s[5]), fmaxf(s[6], s[7])));
      if (__any(top > m[f] + kLazyMax)) {
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        const float mn = fmaxf(m[f], top);
        const float a = __builtin_amdgcn_exp2f(m[f] - mn);
        m[f] = mn;
        l[f] *= a;
#pragma unroll
        for (int i = 0; i < NF; ++i) acc[f][i] *= a;
      }
      uint32_t o[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = __builtin_amdgcn_exp2f(s[2 * i] - m[f]), y = __builtin_amdgcn_exp2f(s[2 * i + 1] - m[f]);
        const half2_t h = __builtin_bit_cast(half2_t, __builtin_amdgcn_cvt_pkrtz(x, y));
        o[i] = as_u(h);
        l[f] = __builtin_amdgcn_fdot2(h, (half2_t){(_Float16)1.0f, (_Float16)1.0f}, l[f], false);
      }
      p[f] = make_uint4(o[0], o[1], o[2], o[3]);
    }
    // ---- output
    if (edge) {
      // Tokens that no column sees hold anything: their s and m become 0.  A NaN value that
      // only some columns see must not reach the others through 0 * NaN: it becomes 0 too, and
      // the columns that see it get their NaN in finish().
      uint32_t any = 0;
#pragma unroll
      for (int h = 0; h < H; ++h) {
        uint32_t sw[4] = {t.vs[h].x, t.vs[h].y, t.vs[h].z, t.vs[h].w};
        uint32_t mw[4] = {t.vm[h].x, t.vm[h].y, t.vm[h].z, t.vm[h].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t keep = (first + 2 * i < ctx ? 0xffffu : 0u) | (first + 2 * i + 1 < ctx ? 0xffff0000u : 0u);
          sw[i] &= keep;
          mw[i] &= keep;
          any |= kv4_nan(sw[i], mw[i]);
        }
        t.vs[h] = make_uint4(sw[0], sw[1], sw[2], sw[3]);
        t.vm[h] = make_uint4(mw[0], mw[1], mw[2], mw[3]);
      }
      if (__any(any != 0)) {
#pragma unroll
        for (int h = 0; h < H; ++h) {
          uint32_t sw[4] = {t.vs[h].x, t.vs[h].y, t.vs[h].z, t.vs[h].w};
          uint32_t mw[4] = {t.vm[h].x, t.vm[h].y, t.vm[h].z, t.vm[h].w};
          int at = 0x7fffffff;
#pragma unroll
          for (int i = 3; i >= 0; --i) {
            const uint32_t nan = kv4_nan(sw[i], mw[i]);
            if (nan & 0x80000000u) at = first + 2 * i + 1;
            if (nan & 0x8000u) at = first + 2 * i;
            const uint32_t keep = (nan & 0x8000u ? 0u : 0xffffu) | (nan & 0x80000000u ? 0u : 0xffff0000u);
            sw[i] &= keep;
            mw[i] &= keep;
          }
          t.vs[h] = make_uint4(sw[0], sw[1], sw[2], sw[3]);
          t.vm[h] = make_uint4(mw[0], mw[1], mw[2], mw[3]);
          // first such token of group 2 h + n / 8; the lane's outputs are of group 2 h + g / 2
          at = min(at, __shfl_xor(at, 16));
          at = min(at, __shfl_xor(at, 32));
          nan_at[h] = min(nan_at[h], __shfl(at, 8 * (g >> 1)));
        }
      }
    }
#pragma unroll
    for (int h = 0; h < H; ++h) {
      const uint32_t vw[4] = {t.v[h].x, t.v[h].y, t.v[h].z, t.v[h].w};
      const uint32_t sw[4] = {t.vs[h].x, t.vs[h].y, t.vs[h].z, t.vs[h].w};
      const uint32_t mw[4] = {t.vm[h].x, t.vm[h].y, t.vm[h].z, t.vm[h].w};
      uint32_t o[4][4];  // [pair of tokens][dimension]
#pragma unroll
      for (int i = 0; i < 4; ++i) expand8(vw[i], as_h2(sw[i]), as_h2(mw[i]), o[i]);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const uint4 va = make_uint4(o[0][c], o[1][c], o[2][c], o[3][c]);
#pragma unroll
        for (int f = 0; f < F; ++f) acc[f][4 * h + c] = mfma16(va, p[f], acc[f][4 * h + c]);
      }
    }
  }

  // The sums of the columns after the last tile: l over the lanes of a column, NaN where the
  // column saw a page outside the pool (bad_at: the first one's position) or a NaN value.
  __device__ __attribute__((always_inline)) inline void finish(int bad_at) {
#pragma unroll
    for (int f = 0; f < F; ++f) {
      l[f] += __shfl_xor(l[f], 16);
      l[f] += __shfl_xor(l[f], 32);
      if (limit[f] >= bad_at) l[f] = __builtin_nanf("");
#pragma unroll
      for (int h = 0; h < H; ++h)
        if (limit[f] >= nan_at[h]) {
#pragma unroll
          for (int c = 0; c < 4; ++c) acc[f][4 * h + c] = (f32x4_t)__builtin_nanf("");
        }
    }
  }
};

// Page numbers of the pair of pages of up to 64 tiles, one tile a lane.
struct Kv4Pages {
  int p0, p1;
  // tile of lane i: base + i * step; tokens at and past ctx have none
  __device__ __attribute__((always_inline)) inline void load(const int32_t* table, int tile0, int step, int ctx, int num_blocks, int& bad_at) {
    const int lane = threadIdx.x & 63;
    const int64_t tok = ((int64_t)tile0 + (int64_t)lane * step) * 32;
    p0 = tok < ctx ? table[tok / kPage] : 0;
    p1 = tok + kPage < ctx ? table[tok / kPage + 1] : 0;
    // a page outside the pool is never an address: page 0 is read instead
    int bad = 0x7fffffff;
    if (p1 < 0 || p1 >= num_blocks) { bad = (int)tok + kPage; p1 = 0; }
    if (p0 < 0 || p0 >= num_blocks) { bad = (int)tok; p0 = 0; }
#pragma unroll
    for (int k = 1; k < 64; k <<= 1) bad = min(bad, __shfl_xor(bad, k));
    bad_at = min(bad_at, bad);
  }
};

// Tiles tile0, tile0 + step, ... < tile_end of the sequence, for one wave.
template <int DT, int D, int F>
__device__ __attribute__((always_inline)) inline void kv4_walk(const Kv4AttnArgs& A, Kv4Wave<DT, D, F>& W, const int32_t* table, int kvh, int tile0, int tile_end,
                                int step, int ctx, int min_limit, int& bad_at) {
  const int64_t page_stride = (int64_t)A.num_layers * A.hkv * Kv4<D>::kSlab;
  const int64_t base = ((int64_t)A.layer * A.hkv + kvh) * Kv4<D>::kSlab;
  const char* const kp = A.k_pool + base;
  const char* const vp = A.v_pool + base;
  const auto off = W.offsets();
  for (int t0 = tile0; t0 < tile_end; t0 += 64 * step) {
    Kv4Pages pages;
    pages.load(table, t0, step, ctx, A.num_blocks, bad_at);
    const int count = min(64, (tile_end - t0 + step - 1) / step);
    auto at = [&](Kv4Tile<D>& t, int i) __attribute__((always_inline)) {
      W.load(t, off, kp, vp, page_stride, __builtin_amdgcn_readlane(pages.p0, i),
             __builtin_amdgcn_readlane(pages.p1, i));
    };
    Kv4Tile<D> cur, next;
    at(cur, 0);
    for (int i = 0; i < count; ++i) {
      at(next, min(i + 1, count - 1));
      const int tok0 = (t0 + i * step) * 32;
      W.step(cur, tok0, ctx, tok0 + 31 > min_limit);
      cur = next;
    }
  }
}

// A sequence's rows, the position of the first, and its context: 0 where that is longer, or the
// rows are more, than the call allows, or the position is none.
struct Kv4Seq {
  int row0, rows, start, ctx;
};
__device__ inline Kv4Seq kv4_seq(const Kv4AttnArgs& A, int b) {
  Kv4Seq s;
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
template <int DT, int D>
__device__ inline void kv4_no_context(const Kv4AttnArgs& A, const Kv4Seq& S, int kvh) {
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

constexpr int kTokWaves = 4;
constexpr int kTokMaxSplits = 64;

// ---- waves split tokens: one workgroup per (split, sequence, kv head, 16-column tile) ----
template <int DT, int D>
__device__ void kv4_tokens_impl(const Kv4AttnArgs& A) {
  constexpr int NW = kTokWaves;
  constexpr int OS = D + 4;  // floats of a column's row in LDS
  __shared__ float s_o[NW][16][OS];
  __shared__ float s_m[NW][16], s_l[NW][16];
  __shared__ float s_w[kTokMaxSplits][16];
  __shared__ int s_last;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int units = A.batch * A.hkv * A.tiles;
  const int split = blockIdx.x / units, unit = blockIdx.x % units;
  const int tile = unit % A.tiles, bh = unit / A.tiles;
  const int b = bh / A.hkv, kvh = bh % A.hkv;
  const Kv4Seq S = kv4_seq(A, b);
  const int col0 = tile * 16, ncols = S.rows * A.group;
  const int here = min(16, ncols - col0);
  if (S.ctx == 0) {
    if (split == 0 && tile == 0) kv4_no_context<DT, D>(A, S, kvh);
    return;
  }
  if (here <= 0) return;
  const int last_row = (col0 + here - 1) / A.group;
  const int last = S.start + last_row;  // the last position that a column here sees
  const int begin = split * A.split_tokens;
  const int nsplit = min(A.splits, last / A.split_tokens + 1);
  if (begin > last) return;
  const int end = min(last + 1, begin + A.split_tokens);

  Kv4Wave<DT, D, 1> W;
  W.begin(A, S.row0, kvh, S.start, S.ctx, col0, ncols);
  int bad_at = 0x7fffffff;
  kv4_walk<DT, D, 1>(A, W, A.tables + (int64_t)b * A.table_stride, kvh, begin / 32 + w, (end + 31) / 32, NW,
                     S.ctx, S.start + col0 / A.group, bad_at);
  const int n = W.n, g = W.g;
  W.finish(bad_at);
  if (g == 0) {
    s_m[w][n] = W.m[0];
    s_l[w][n] = W.l[0];
  }
#pragma unroll
  for (int h = 0; h < D / 64; ++h)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      *(float4*)&s_o[w][n][64 * h + 16 * g + 4 * r] =
          make_float4(W.acc[0][4 * h][r], W.acc[0][4 * h + 1][r], W.acc[0][4 * h + 2][r], W.acc[0][4 * h + 3][r]);
  __syncthreads();
  // ---- the workgroup's columns
  constexpr int Q = D / 4;  // float4s of a column
  const int64_t part = (int64_t)unit * A.splits;
  for (int i = threadIdx.x; i < here * Q; i += 64 * NW) {
    const int col = i / Q, d = i % Q * 4;
    float M = s_m[0][col];
#pragma unroll
    for (int k = 1; k < NW; ++k) M = fmaxf(M, s_m[k][col]);
    float L = 0.0f;
    float4 o = make_float4(0, 0, 0, 0);
#pragma unroll
    for (int k = 0; k < NW; ++k) {
      const float e = __builtin_amdgcn_exp2f(s_m[k][col] - M);
      const float4 x = *(const float4*)&s_o[k][col][d];
      L = fmaf(e, s_l[k][col], L);
      o.x = fmaf(e, x.x, o.x); o.y = fmaf(e, x.y, o.y); o.z = fmaf(e, x.z, o.z); o.w = fmaf(e, x.w, o.w);
    }
    if (nsplit == 1) {
      const int c = col0 + col;
      uint16_t* const dst = A.out + (int64_t)(S.row0 + c / A.group) * A.out_stride + ((int64_t)kvh * A.group + c % A.group) * D + d;
      const uint32_t a0 = St<DT>::store(o.x / L) | (uint32_t)St<DT>::store(o.y / L) << 16;
      const uint32_t a1 = St<DT>::store(o.z / L) | (uint32_t)St<DT>::store(o.w / L) << 16;
      *(uint2*)dst = make_uint2(a0, a1);
    } else {
      float* const po = A.ws_o + ((part + split) * 16 + col) * D + d;
      ws_put(po, o.x); ws_put(po + 1, o.y); ws_put(po + 2, o.z); ws_put(po + 3, o.w);
      if (d == 0) {
        float* const pm = A.ws_ml + ((part + split) * 16 + col) * 2;
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
    s_last = __hip_atomic_fetch_add(A.ws_cnt + unit, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == nsplit - 1;
  __syncthreads();
  if (!s_last) return;
  if (threadIdx.x == 0) __hip_atomic_store(A.ws_cnt + unit, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  // weights 2^(m_s - M) and their sums (s_l's first row)
  for (int col = threadIdx.x; col < here; col += 64 * NW) {
    const float* const pm = A.ws_ml + (part * 16 + col) * 2;
    float M = -INFINITY;
    for (int s = 0; s < nsplit; ++s) M = fmaxf(M, ws_get(pm + (int64_t)s * 32));
    float L = 0.0f;
    for (int s = 0; s < nsplit; ++s) {
      const float e = __builtin_amdgcn_exp2f(ws_get(pm + (int64_t)s * 32) - M);
      L = fmaf(e, ws_get(pm + (int64_t)s * 32 + 1), L);
      s_w[s][col] = e;
    }
    s_l[0][col] = L;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < here * Q; i += 64 * NW) {
    const int col = i / Q, d = i % Q * 4;
    const float* const po = A.ws_o + (part * 16 + col) * D + d;
    float4 o = make_float4(0, 0, 0, 0);
    for (int s = 0; s < nsplit; ++s) {
      const float e = s_w[s][col];
      const float* const x = po + (int64_t)s * 16 * D;
      o.x = fmaf(e, ws_get(x), o.x); o.y = fmaf(e, ws_get(x + 1), o.y);
      o.z = fmaf(e, ws_get(x + 2), o.z); o.w = fmaf(e, ws_get(x + 3), o.w);
    }
    const float L = s_l[0][col];
    const int c = col0 + col;
    uint16_t* const dst = A.out + (int64_t)(S.row0 + c / A.group) * A.out_stride + ((int64_t)kvh * A.group + c % A.group) * D + d;
    const uint32_t a0 = St<DT>::store(o.x / L) | (uint32_t)St<DT>::store(o.y / L) << 16;
    const uint32_t a1 = St<DT>::store(o.z / L) | (uint32_t)St<DT>::store(o.w / L) << 16;
    *(uint2*)dst = make_uint2(a0, a1);
  }
}

// ---- waves split columns: one workgroup per (chunk of columns, sequence, kv head, split) ----
constexpr int kColWaves = 4;
template <int D> struct Kv4Cols {
  static constexpr int F = D == 64 ? 4 : 2;  // fragments of a wave
  static constexpr int N = kColWaves * F * 16;
};

template <int DT, int D>
__device__ void kv4_columns_impl(const Kv4AttnArgs& A) {
  constexpr int F = Kv4Cols<D>::F;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // the chunks that see the longest contexts first
  const int pairs = A.batch * A.hkv;
  const int split = blockIdx.x % A.splits, rest = blockIdx.x / A.splits;
  const int chunk = A.tiles - 1 - rest / pairs, bh = rest % pairs;
  const int b = bh / A.hkv, kvh = bh % A.hkv;
  const Kv4Seq S = kv4_seq(A, b);
  const int ncols = S.rows * A.group;
  const int col0 = chunk * Kv4Cols<D>::N + w * (16 * F);
  const int here = min(16 * F, ncols - col0);
  const int hq = A.hkv * A.group;
  if (S.ctx == 0) {
    if (split == 0 && chunk == 0) kv4_no_context<DT, D>(A, S, kvh);
    return;
  }
  if (here <= 0) return;  // (no barrier follows)
  const int last = S.start + (col0 + here - 1) / A.group;
  const int begin = split * A.split_tokens;  // (splits x split_tokens fits: luc_kv4.cpp)
  if (begin > last) return;
  const int end = A.splits == 1 ? last + 1 : min(last + 1, begin + A.split_tokens);
  Kv4Wave<DT, D, F> W;
  W.begin(A, S.row0, kvh, S.start, S.ctx, col0, ncols);
  int bad_at = 0x7fffffff;
  kv4_walk<DT, D, F>(A, W, A.tables + (int64_t)b * A.table_stride, kvh, begin / 32, (end + 31) / 32, 1, S.ctx,
                     S.start + col0 / A.group, bad_at);
  W.finish(bad_at);
#pragma unroll
  for (int f = 0; f < F; ++f) {
    const float l = W.l[f];
    const int col = col0 + 16 * f + W.n;
    if (col >= ncols) continue;
    const int64_t row = S.row0 + col / A.group;
    const int head = kvh * A.group + col % A.group;
    if (A.splits == 1) {
      uint16_t* const dst = A.out + row * A.out_stride + (int64_t)head * D + 16 * W.g;
      const float inv = 1.0f / l;
#pragma unroll
      for (int h = 0; h < D / 64; ++h)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const uint32_t a0 = St<DT>::store(W.acc[f][4 * h][r] * inv) | (uint32_t)St<DT>::store(W.acc[f][4 * h + 1][r] * inv) << 16;
          const uint32_t a1 = St<DT>::store(W.acc[f][4 * h + 2][r] * inv) | (uint32_t)St<DT>::store(W.acc[f][4 * h + 3][r] * inv) << 16;
          *(uint2*)(dst + 64 * h + 4 * r) = make_uint2(a0, a1);
        }
    } else {
      const int64_t at = ((int64_t)split * A.total_rows + row) * hq + head;
      if (W.g == 0) *(float2*)(A.ws_ml + at * 2) = make_float2(W.m[f], l);
      float* const po = A.ws_o + at * D + 16 * W.g;
#pragma unroll
      for (int h = 0; h < D / 64; ++h)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          *(float4*)(po + 64 * h + 4 * r) = make_float4(W.acc[f][4 * h][r], W.acc[f][4 * h + 1][r], W.acc[f][4 * h + 2][r],
                                                        W.acc[f][4 * h + 3][r]);
    }
  }
}

// The partials of a columns launch: D / 4 lanes a (row, head).
template <int DT, int D>
__device__ void kv4_merge_impl(const Kv4AttnArgs& A) {
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
  const Kv4Seq S = kv4_seq(A, b);
  const int r = row - S.row0;
  if (r < 0 || r >= S.rows || S.ctx == 0) return;  // no sequence's row, or written already
  const int nsplit = min(A.splits, (S.start + r) / A.split_tokens + 1);
  const int64_t step = (int64_t)A.total_rows * hq;
  float M = -INFINITY;
  for (int s = 0; s < nsplit; ++s) M = fmaxf(M, A.ws_ml[(item + s * step) * 2]);
  float L = 0.0f;
  float4 o = make_float4(0, 0, 0, 0);
  for (int s = 0; s < nsplit; ++s) {
    const float2 ml = *(const float2*)(A.ws_ml + (item + s * step) * 2);
    const float e = __builtin_amdgcn_exp2f(ml.x - M);
    const float4 x = *(const float4*)(A.ws_o + (item + s * step) * D + d);
    L = fmaf(e, ml.y, L);
    o.x = fmaf(e, x.x, o.x); o.y = fmaf(e, x.y, o.y); o.z = fmaf(e, x.z, o.z); o.w = fmaf(e, x.w, o.w);
  }
  const float inv = 1.0f / L;
  const uint32_t a0 = St<DT>::store(o.x * inv) | (uint32_t)St<DT>::store(o.y * inv) << 16;
  const uint32_t a1 = St<DT>::store(o.z * inv) | (uint32_t)St<DT>::store(o.w * inv) << 16;
  *(uint2*)(A.out + row * A.out_stride + (int64_t)head * D + d) = make_uint2(a0, a1);
}

}  // namespace luc

#define LUC_KV4_ATTENTION(DTN, DT, D)                                                            \
  extern "C" __global__ __launch_bounds__(256, 2) void luc_kv4_tokens_##DTN##_d##D(luc::Kv4AttnArgs a) {  \
    luc::kv4_tokens_impl<luc::DT, D>(a);                                                         \
  }                                                                                              \
  extern "C" __global__ __launch_bounds__(256, 2) void luc_kv4_columns_##DTN##_d##D(luc::Kv4AttnArgs a) { \
    luc::kv4_columns_impl<luc::DT, D>(a);                                                        \
  }                                                                                              \
  extern "C" __global__ __launch_bounds__(256) void luc_kv4_merge_##DTN##_d##D(luc::Kv4AttnArgs a) {      \
    luc::kv4_merge_impl<luc::DT, D>(a);                                                          \
  }
LUC_KV4_ATTENTION(bf16, kBF16, 64)
LUC_KV4_ATTENTION(bf16, kBF16, 128)
LUC_KV4_ATTENTION(f16, kF16, 64)
LUC_KV4_ATTENTION(f16, kF16, 128)
