// Attention of new rows over a 4-bit paged cache (gfx950):
//   o = sum_t softmax_t(sm_scale q . k_t) v_t,  t = 0 .. the row's own position,
// with k_t and v_t the values n * s + m of kv4.h, for the rows of a batch of sequences: one
// row each (a decode step; the reference's flash_decoding kernel, src/kernels/attention.cu:4-240,
// over its 16-bit cache) or packed prompts.
//
// Columns.  The (row, head of the group) pairs of one sequence and kv head are the columns of
// the products: S^T = K Q^T and O^T += V^T P^T on v_mfma_f32_16x16x32_f16, 16 columns a fragment.
// In the accumulators a lane has one column throughout (column lane % 16), so maxima, sums and
// rescaling are lane-local up to the four lanes that share it, and the scores of 32 tokens are
// already the operand of the second product: lane l holds four tokens of either 16-token fragment.
// q is taken to fp16 after a power of two brings its largest element to [1, 2) (columns) or [2^14, 2^15)
// (tokens, whose n are fp16 subnormals), exactly unless an element is below 2^-14 or 2^-24 of that.  The
// running maximum moves only when a score passes it by some powers of two, so most tiles rescale nothing.
// Weights are held times a power of two, far above fp16's smallest.
//
// Two kernels:
//   tokens: 8 columns a workgroup; its 4 waves take stages of tokens in turn and merge in LDS.  Few
//     columns a sequence (decode): every wave streams its own part of the cache, n goes to the
//     matrix unit as it is, and s and m are applied to sums.
//   columns: 128 (D = 64) or 256 columns a workgroup, every wave walks all tokens of its columns'
//     contexts.  Prompts: an expanded tile of n s + m serves all of them.
// Either may cut the context into splits over workgroups, whose partial (m, l, o) go to the
// workspace; tokens: the last workgroup of a (sequence, kv head, column tile) to arrive
// merges them; columns: a second launch does.
#include "kv4.h"
#include "kv_split.h"

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
  int32_t longest_first;
  float qk_scale_log2;
};

// The running maximum moves when a score (in powers of two) passes it by this: weights are at most
// 8 times what the largest had when it moved.
constexpr float kKv4Lazy = 3.0f;
// tokens: weights are held times 2^lift, so that neither those of a long tail nor their products with a
// small step of V get lost below fp16's smallest, 2^-24.  A product is below 2^(12 - lift) 2^(3 + lift) = 2^15
// for steps below 2^(12 - lift), and below 2^16 whatever the rounding of large scores adds: a column that meets a
// longer step lowers its lift (-1 holds every s of the format, 8000 at most).
constexpr int kKv4Lift = 12, kKv4LeastLift = -1;
__device__ inline uint32_t kv4_steps(int lift) { return (uint32_t)(27 - lift) << 10; }  // fp16 bits of 2^(12 - lift)

// columns: weights, at most 2^kLazyMax of that, are held times this power of two, 2^15 at most.  (V is
// multiplied in the matrix unit.)
constexpr float kKv4ColsLift = 15.0f - kLazyMax;
// What a largest score (in powers of two) makes the running maximum, less the lift: none where a rounding of the
// score itself is as much as the room that the lift leaves below 2^16.
__device__ inline float kv4_reference(float score, float lift) {
  return fabsf(score) < 0x1p23f ? score - lift : score;
}

__device__ inline f32x4_t mfma16(uint4 a, uint4 b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

__device__ inline half2_t as_h2(uint32_t x) { return __builtin_bit_cast(half2_t, x); }
__device__ inline uint32_t as_u(half2_t x) { return __builtin_bit_cast(uint32_t, x); }

// The four pairs (n i, n i + 4) of a dword's n, times s plus m, as packed fp16.
__device__ inline void expand8(uint32_t w, half2_t s, half2_t m, uint32_t* o) {
  uint32_t kBig = 0x64006400u;  // 1024.0 twice
  asm("" : "+v"(kBig));         // in a VGPR: v_and_or_b32 takes one scalar operand, the mask
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

// The four pairs as they are.
__device__ inline void whole8(uint32_t w, uint32_t* o) {
  uint32_t kBig = 0x64006400u;
  asm("" : "+v"(kBig));
  const half2_t big = {(_Float16)1024.0f, (_Float16)1024.0f};
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = as_u(as_h2((w >> (4 * i) & 0x000f000fu) | kBig) - big);
}
// NaN where one is.  (fmaxf, which passes over it, would first quiet every operand.)
__device__ inline float max3(float a, float b, float c) {
  return __builtin_elementwise_maximum(__builtin_elementwise_maximum(a, b), c);
}

// Of a pair of tokens' s and m, bit 15 or 31 where a token's is NaN (the format has no
// infinities: an exponent of all ones is NaN).
__device__ inline uint32_t kv4_nan(uint32_t s, uint32_t m) {
  return (((s & 0x7c007c00u) + 0x04000400u) | ((m & 0x7c007c00u) + 0x04000400u)) & 0x80008000u;
}

// Of the two halves of a dword.
typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));
__device__ inline uint32_t max_u16(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2_t, a), __builtin_bit_cast(u16x2_t, b)));
}
__device__ inline uint32_t sub_sat_u16(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_sub_sat(__builtin_bit_cast(u16x2_t, a), __builtin_bit_cast(u16x2_t, b)));
}

__device__ inline int pick2(bool c, int a, int b) {
  int r = c ? a : b;
  asm("" : "+v"(r));
  return r;
}

// ---- stages: what a wave keeps in LDS of the tokens ahead ------------------------------
//
// A stage is 5 KB: the slabs of 32 (D = 128) or 64 (D = 64) tokens, in 320 chunks of 16 bytes,
// five loads of 64 lanes straight into LDS.  A lane's source is free, its place in LDS is not, so
// chunks are dealt such that the reads below are conflict-free:
//   K n      [sub-tile][fragment][group][token of the fragment]
//   V n      [sub-tile][group][octet][quad of the group]
//   K (s, m) [sub-tile][token of the octet (pairs, D = 64)][octet]
//   V s, V m [sub-tile][group][octet]
template <int D> struct Kv4Stage {
  static constexpr int SUB = D == 128 ? 1 : 2;  // 32-token sub-tiles
  static constexpr int TOKENS = 32 * SUB;
  static constexpr int PAGES = 2 * SUB;
  static constexpr int LOADS = 5;
  static constexpr int BYTES = 1024 * LOADS;

  const char* src[3];  // of the lane, in page 0: K n, V n, scales

  __device__ __attribute__((always_inline)) inline void begin(const char* k_pool, const char* v_pool) {
    const int l = threadIdx.x & 63;
    const int n = l & 15;
    // K: D = 128 fragment i, group l / 16; D = 64 sub-tile i, fragment l / 32, group (l / 16) % 2
    const int tok = 8 * (n >> 2) + (n & 3) + (D == 128 ? 0 : 4 * (l >> 5));
    src[0] = k_pool + Kv4<D>::k_row(tok & 15) + 16 * (D == 128 ? l >> 4 : (l >> 4) & 1);
    // V: D = 128 groups 2 i and 2 i + 1; D = 64 sub-tile i
    src[1] = v_pool + Kv4<D>::v_quad(l & 8, 8 * (l >> 5) + (l & 7));
    if (l < 32) {
      const int o = l & 3;
      src[2] = k_pool + Kv4<D>::k_scale(D == 128 ? (8 * o + (l >> 2)) & 15 : 8 * (o & 1) + 2 * ((l >> 2) & 3), 0);
    } else {
      const int x = l & 15;
      src[2] = v_pool + Kv4<D>::v_scale(x & 1, D == 128 ? x >> 2 : (x >> 2) & 1) + (l < 48 ? 0 : 16);
    }
  }
  // The loads of a stage.  p0 ..: its pages (alike in all lanes; scalars, since an array indexed
  // by lane would go through memory).
  __device__ __attribute__((always_inline)) inline void issue(char* lds, int p0, int p1, int p2, int p3, uint32_t page_stride) const {
    // the second page of two by a bit of the lane, as begin() deals tokens and octets
    const int l = threadIdx.x & 63;
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      const bool odd = l & (v ? 16 : 8);
      const char* const a = src[v] + (uint64_t)(uint32_t)pick2(odd, p1, p0) * page_stride;
      to_lds(a, lds + 2048 * v);
      // four rows of K on; 16 quads of V on
      to_lds(D == 128 ? a + 256 : src[v] + (uint64_t)(uint32_t)pick2(odd, p3, p2) * page_stride, lds + 2048 * v + 1024);
    }
    int id = pick2(l & 2, p1, p0);
    if constexpr (PAGES == 4) id = pick2(l < 32 ? l & 16 : l & 8, pick2(l & 2, p3, p2), id);
    to_lds(src[2] + (uint64_t)(uint32_t)id * page_stride, lds + 4096);
  }
  __device__ static inline void to_lds(const char* a, char* lds) {
    __builtin_amdgcn_global_load_lds(a, (__attribute__((address_space(3))) void*)lds, 16, 0, 0);
  }
};

// LDS reads of a sub-tile with their wait: the compiler would wait for every load into LDS
// that is under way before a read that it can see.
template <int D> struct Kv4Reads;
template <> struct Kv4Reads<128> {
  typedef uint32_t pair __attribute__((ext_vector_type(2)));
  pair kw[4];       // K n: fragment a groups 0 1, 2 3, fragment b
  uint32_t am[2];   // (s, m) of the fragments' tokens for the m term
  u32x4_t sm[4];    // (s, m) of the lane's 4 tokens, a dword a group
  u32x4_t v[4], vm;  // a group each: the lane's quads of it; m of group n
  pair vs[4];        // s of the lane's 4 tokens
  __device__ __attribute__((always_inline)) inline void read_k(uint32_t kw_at, uint32_t sm_at, uint32_t am_at, int) {
    asm volatile(
        "ds_read2st64_b32 %0, %10 offset1:1\n\tds_read2st64_b32 %1, %10 offset0:2 offset1:3\n\t"
        "ds_read2st64_b32 %2, %10 offset0:4 offset1:5\n\tds_read2st64_b32 %3, %10 offset0:6 offset1:7\n\t"
        "ds_read_b32 %4, %12 offset:4096\n\tds_read_b32 %5, %12 offset:4352\n\t"
        "ds_read_b128 %6, %11 offset:4096\n\tds_read_b128 %7, %11 offset:4160\n\t"
        "ds_read_b128 %8, %11 offset:4224\n\tds_read_b128 %9, %11 offset:4288\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(kw[0]), "=&v"(kw[1]), "=&v"(kw[2]), "=&v"(kw[3]), "=&v"(am[0]), "=&v"(am[1]), "=&v"(sm[0]), "=&v"(sm[1]), "=&v"(sm[2]),
          "=&v"(sm[3])
        : "v"(kw_at), "v"(sm_at), "v"(am_at)
        : "memory");
  }
  __device__ __attribute__((always_inline)) inline void read_v(uint32_t v_at, uint32_t vs_at, uint32_t vm_at, int) {
    asm volatile(
        "ds_read_b128 %0, %9 offset:2048\n\tds_read_b128 %1, %9 offset:2560\n\t"
        "ds_read_b128 %2, %9 offset:2048+1024\n\tds_read_b128 %3, %9 offset:3584\n\t"
        "ds_read_b64 %4, %10 offset:4608\n\tds_read_b64 %5, %10 offset:4672\n\t"
        "ds_read_b64 %6, %10 offset:4736\n\tds_read_b64 %7, %10 offset:4800\n\t"
        "ds_read_b128 %8, %11 offset:4864\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]), "=&v"(vs[0]), "=&v"(vs[1]), "=&v"(vs[2]), "=&v"(vs[3]), "=&v"(vm)
        : "v"(v_at), "v"(vs_at), "v"(vm_at)
        : "memory");
  }
  __device__ inline uint32_t k(int b, int j) const { return kw[2 * b + (j >> 1)][j & 1]; }
  __device__ inline uint32_t scale(int i, int j) const { return sm[i][j]; }
};
template <> struct Kv4Reads<64> {
  typedef uint32_t pair __attribute__((ext_vector_type(2)));
  pair kw[2];
  uint32_t am[2];
  u32x4_t sm[2];    // two tokens each, two groups
  u32x4_t v[2], vm;
  pair vs[2];
  __device__ __attribute__((always_inline)) inline void read_k(uint32_t kw_at, uint32_t sm_at, uint32_t am_at, int u) {
    asm volatile(
        "ds_read2st64_b32 %0, %6 offset1:1\n\tds_read2st64_b32 %1, %6 offset0:2 offset1:3\n\t"
        "ds_read_b32 %2, %8 offset:4096\n\tds_read_b32 %3, %8 offset:4224\n\t"
        "ds_read_b128 %4, %7 offset:4096\n\tds_read_b128 %5, %7 offset:4160\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(kw[0]), "=&v"(kw[1]), "=&v"(am[0]), "=&v"(am[1]), "=&v"(sm[0]), "=&v"(sm[1])
        : "v"(kw_at + u * 1024), "v"(sm_at + u * 256), "v"(am_at + u * 256)
        : "memory");
  }
  __device__ __attribute__((always_inline)) inline void read_v(uint32_t v_at, uint32_t vs_at, uint32_t vm_at, int u) {
    asm volatile(
        "ds_read_b128 %0, %5 offset:2048\n\tds_read_b128 %1, %5 offset:2560\n\t"
        "ds_read_b64 %2, %6 offset:4608\n\tds_read_b64 %3, %6 offset:4672\n\t"
        "ds_read_b128 %4, %7 offset:4864\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(v[0]), "=&v"(v[1]), "=&v"(vs[0]), "=&v"(vs[1]), "=&v"(vm)
        : "v"(v_at + u * 1024), "v"(vs_at + u * 128), "v"(vm_at + u * 128)
        : "memory");
  }
  __device__ inline uint32_t k(int b, int j) const { return kw[b][j]; }
  __device__ inline uint32_t scale(int i, int j) const { return sm[i >> 1][2 * (i & 1) + j]; }
};

// One wave's 8 columns over stages.  Of a fragment's 16 columns the lower 8 take fragment a's tokens
// and the upper 8, the same rows and heads again, fragment b's: q is zero in the others' places, so
// both fragments' products add up in one accumulator, a lane has 4 tokens of one column, and
// softmax costs half of what 16 columns would.  The two halves of a column are partial results
// like those of two waves.
template <int DT, int D> struct Kv4Row {
  static constexpr int NG = D / 32;  // groups of 32 dimensions
  static constexpr bool HILO = DT == kF16;  // weights in two fp16 parts: see step()

  uint4 q[2][NG];  // [fragment]; group j's dimensions 8 g .. + 7 of it, pairs (i, i + 4), i odd divided by 16
  uint32_t qsum;   // k = 8 g, 8 g + 1: the sum of group g's dimensions times 2^-9, high and low part
  // O^T: [group][c], rows 4 g + i of it are dimensions 16 (g % 2) + 4 i + 2 (g / 2) + c of the group, in
  // units of 2^-20; and the m term, whose rows are groups
  f32x4_t acc[NG][2], acc_m;
  float m, l, scale;  // m: less the column's lift
  float bar;       // products above it move m
  int limit;
  int lift;        // of the column, see kKv4Lift
  int lane, n, g;
  uint32_t mask[2];  // of the pairs of fragment a's and b's tokens in P: the lane's or 0
  uint32_t kw_at, sm_at, am_at, v_at, vs_at, vm_at;  // LDS offsets of the lane's reads in a stage

  __device__ __attribute__((always_inline)) inline void begin(const Kv4AttnArgs& A, int64_t row0, int kvh, int start, int ctx, int col0,
                                                              int ncols) {
    lane = threadIdx.x & 63;
    n = lane & 15;
    g = lane >> 4;
    const int half = n >> 3;
    kw_at = n * 16 + g * 4;
    sm_at = g * 16 + half * (D == 128 ? 256 : 128);
    am_at = D == 128 ? ((n & 3) * 4 + (n >> 2)) * 16 + g * 4
                     : (((n & 3) >> 1) * 4 + (n >> 2)) * 16 + (n & 1) * 8 + (g & 1) * 4;
    v_at = (g * 8 + (n & 7)) * 16;
    vs_at = g * 16 + half * 8;
    vm_at = ((n & (NG - 1)) * 4 + g) * 16;
    mask[0] = half ? 0 : ~0u;
    mask[1] = ~mask[0];
    const int col = col0 + (n & 7);
    const bool on = col < ncols;
    const int r = on ? col / A.group : 0, hd = on ? col % A.group : 0;
    limit = on ? start + r : ctx - 1;
    const uint16_t* const src = A.q + (row0 + r) * A.q_stride + ((int64_t)kvh * A.group + hd) * D + 8 * g;
    float x[NG][8];
    float top = 0.0f;
#pragma unroll
    for (int j = 0; j < NG; ++j) {
      const uint4 w = on ? *(const uint4*)(src + 32 * j) : make_uint4(0, 0, 0, 0);
      const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[j][2 * e] = St<DT>::lo(ww[e]);
        x[j][2 * e + 1] = St<DT>::hi(ww[e]);
        top = fmaxf(top, fmaxf(fabsf(x[j][2 * e]), fabsf(x[j][2 * e + 1])));
      }
    }
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
    // a power of two takes the largest element into [2^14, 2^15) (infinities and NaN stay so)
    const int e = min(max((int)(__float_as_uint(top) >> 23), 15), 253);
    const float up = copysignf(__uint_as_float((uint32_t)(268 - e) << 23), A.qk_scale_log2);
    // n is 2^-24 n in the products: 2^(e - 127) 2^-14 2^24.  The scale's sign goes to q, so that
    // the largest product is the largest score.
    scale = fabsf(A.qk_scale_log2) * 1024.0f * __uint_as_float((uint32_t)e << 23);
    if (scale == 0.0f) scale = 1e-37f;  // (a masked product, -inf, times 0 is NaN)
    float mine = 0.0f;
#pragma unroll
    for (int j = 0; j < NG; ++j) {
      uint32_t o[4];
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float f = i & 1 ? up * 0.0625f : up;
        const half2_t p = {(_Float16)(x[j][i] * f), (_Float16)(x[j][i + 4] * f)};
        o[i] = as_u(p);
        sum += x[j][i] * up + x[j][i + 4] * up;
      }
#pragma unroll
      for (int b = 0; b < 2; ++b) q[b][j] = make_uint4(o[0] & mask[b], o[1] & mask[b], o[2] & mask[b], o[3] & mask[b]);
      sum += __shfl_xor(sum, 16);
      sum += __shfl_xor(sum, 32);
      mine = g == j ? sum : mine;
    }
    mine *= 0x1p-9f;  // (at most 2^11; times 2^-24 the low part would be mostly lost below fp16's smallest)
    const _Float16 hi = (_Float16)mine;
    const half2_t parts = {hi, (_Float16)(mine - (float)hi)};
    qsum = as_u(parts);
    lift = kKv4Lift;
    m = -3.4028235e38f;
    bar = -INFINITY;
    l = 0.0f;
#pragma unroll
    for (int j = 0; j < NG; ++j) acc[j][0] = acc[j][1] = (f32x4_t){0, 0, 0, 0};
    acc_m = (f32x4_t){0, 0, 0, 0};
  }

  // Sub-tile u of the stage at LDS address lds: tokens tok0 .. tok0 + 31.
  __device__ __attribute__((always_inline)) inline void step(uint32_t lds, int u, int tok0, int ctx, bool edge) {
    Kv4Reads<D> R;
    R.read_k(lds + kw_at, lds + sm_at, lds + am_at, u);
    // ---- products with the tokens' K: sum over groups of s (n . q), and the m term by itself
    f32x4_t x[2], c[NG];
#pragma unroll
    for (int j = 0; j < NG; ++j) c[j] = (f32x4_t){0, 0, 0, 0};
#pragma unroll
    for (int b = 0; b < 2; ++b) {
#pragma unroll
      for (int j = 0; j < NG; ++j) {
        const uint32_t w = R.k(b, j), v = w >> 8;
        // fp16 subnormals: n 2^-24, and 16 n 2^-24 for the odd ones
        c[j] = mfma16(make_uint4(w & 0x000f000fu, w & 0x00f000f0u, v & 0x000f000fu, v & 0x00f000f0u), q[b][j], c[j]);
      }
      const uint32_t mm = R.am[b] >> 16 | (R.am[b] & 0xffff0000u);
      x[b] = mfma16(make_uint4(D == 128 || g < 2 ? mm : 0, 0, 0, 0), make_uint4(qsum, 0, 0, 0), (f32x4_t){0, 0, 0, 0});
    }
    float s[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s[i] = (mask[0] ? x[0][i] : x[1][i]) * 0x1p-15f;  // (not a sum: m may be NaN in the other fragment)
#pragma unroll
      for (int j = 0; j < NG; ++j) s[i] = fmaf((float)as_h2(R.scale(i, j)).x, c[j][i], s[i]);
    }
    const int first = tok0 + 8 * g;  // the 8 tokens of the lane's V
    const int own = first + (n >> 3) * 4;  // and the 4 of its column
    if (edge) {
      asm volatile("" ::: "memory");  // (stays a branch)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[i] = own + i <= limit ? s[i] : -INFINITY;
    }
    float top = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
    if (__any(top > bar)) {
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      const float mn = fmaxf(m, kv4_reference(top * scale, (float)lift));
      const float a = __builtin_amdgcn_exp2f(m - mn);
      bar = fmaxf(bar, top + kKv4Lazy / scale);
      m = mn;
      l *= a;
#pragma unroll
      for (int j = 0; j < NG; ++j) {
        acc[j][0] *= a;
        acc[j][1] *= a;
      }
      acc_m *= a;
    }
    // fp16 rows get P in two parts, whose own rounding would show in their outputs; bf16 rows
    // one, and l the sum of the same truncated weights: errors of 1.74e-3 of the output against 1.72e-3 of
    // its rounding alone, 25.7 and 89.6 us for 8 x 32768 and 64 x 1024..16384 against 26.5 and 90.4 in two parts
    uint32_t ph[2], pl[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float y = __builtin_amdgcn_exp2f(fmaf(s[2 * i], scale, -m));
      const float z = __builtin_amdgcn_exp2f(fmaf(s[2 * i + 1], scale, -m));
      const half2_t h = __builtin_bit_cast(half2_t, __builtin_amdgcn_cvt_pkrtz(y, z));
      ph[i] = as_u(h);
      if constexpr (HILO) {
        pl[i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(y - (float)h.x, z - (float)h.y));
        l += y + z;
      } else {
        l = __builtin_amdgcn_fdot2(h, (half2_t){(_Float16)1.0f, (_Float16)1.0f}, l, false);
      }
    }
    // ---- output: the weights times s are the operand of each group's n, as fp16 subnormals, and the
    // weights that of m
    R.read_v(lds + v_at, lds + vs_at, lds + vm_at, u);
    if (edge) {
      asm volatile("" ::: "memory");
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int t = own + 2 * i;
        const uint32_t seen = (t <= limit ? 0xffffu : 0u) | (t + 1 <= limit ? 0xffff0000u : 0u);
#pragma unroll
        for (int j = 0; j < NG; ++j) R.vs[j][i] &= seen;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // of tokens that the column does not see nothing may come through, NaN neither: their s
        // is 0; and m's operand is shared by all columns, so what is NaN (s is, too) or belongs
        // to no token is 0 there
        const int t = first + 2 * i;
        const uint32_t live = (t < ctx ? 0xffffu : 0u) | (t + 1 < ctx ? 0xffff0000u : 0u);
        const uint32_t nan = ((R.vm[i] & 0x7c007c00u) + 0x04000400u) & 0x80008000u;
        R.vm[i] &= live & ~((nan >> 15) * 0xffffu);
      }
    }
    uint32_t longest = R.vs[0][0];  // of the steps that the column sees, two fp16
#pragma unroll
    for (int j = 0; j < NG; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i) longest = max_u16(longest, R.vs[j][i]);
    const uint32_t most = kv4_steps(lift) - 1;
    if (__any(sub_sat_u16(longest, most | most << 16))) lower(R, ph, pl);
    uint32_t p[4] = {ph[0] & mask[0], ph[1] & mask[0], ph[0] & mask[1], ph[1] & mask[1]};
    uint32_t p2[4];
    if constexpr (HILO) {
      p2[0] = pl[0] & mask[0]; p2[1] = pl[1] & mask[0]; p2[2] = pl[0] & mask[1]; p2[3] = pl[1] & mask[1];
    }
    const uint32_t groups = n < NG ? ~0u : 0u;
    const uint4 vm = make_uint4(R.vm[0] & groups, R.vm[1] & groups, R.vm[2] & groups, R.vm[3] & groups);
    acc_m = mfma16(vm, make_uint4(p[0], p[1], p[2], p[3]), acc_m);
    if constexpr (HILO) acc_m = mfma16(vm, make_uint4(p2[0], p2[1], p2[2], p2[3]), acc_m);
    // lanes 8 .. 15 of a row have the same quads' upper two dimensions
    const uint32_t shift = n & 8, turn = shift ? 4 : 28;
#pragma unroll
    for (int j = 0; j < NG; ++j) {
      uint32_t w[4], w2[4], a0[4], a1[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const half2_t s2 = as_h2(R.vs[j][i & 1]);  // (one half of p is 0)
        const half2_t ps = as_h2(p[i]) * s2;
        w[i] = as_u(ps);
        // what the product's rounding left out (n s is many times a value near 0), and the
        // weights' second part
        half2_t rest = __builtin_elementwise_fma(as_h2(p[i]), s2, -ps);
        if constexpr (HILO) rest = __builtin_elementwise_fma(as_h2(p2[i]), s2, rest);
        w2[i] = as_u(rest);
        // 16 n 2^-24: the matrix unit aligns a subnormal's products by 2^-14, its nominal
        // exponent, and n 2^-24 would lose 4 more bits (n s against m: near-zero values showed it)
        a0[i] = __builtin_amdgcn_alignbit(R.v[j][i], R.v[j][i], turn) & 0x00f000f0u;
        a1[i] = R.v[j][i] >> shift & 0x00f000f0u;
      }
      const uint4 b = make_uint4(w[0], w[1], w[2], w[3]);
      const uint4 x0 = make_uint4(a0[0], a0[1], a0[2], a0[3]), x1 = make_uint4(a1[0], a1[1], a1[2], a1[3]);
      acc[j][0] = mfma16(x0, b, acc[j][0]);
      acc[j][1] = mfma16(x1, b, acc[j][1]);
      const uint4 b2 = make_uint4(w2[0], w2[1], w2[2], w2[3]);
      acc[j][0] = mfma16(x0, b2, acc[j][0]);
      acc[j][1] = mfma16(x1, b2, acc[j][1]);
    }
  }

  // The column's lift down to what V's steps of its tokens allow, and with it what it has summed and the weights at
  // hand.  (Steps that are NaN say nothing of the other groups.)
  __device__ __attribute__((always_inline)) inline void lower(const Kv4Reads<D>& R, uint32_t (&ph)[2], uint32_t (&pl)[2]) {
    uint32_t longest = 0;
#pragma unroll
    for (int j = 0; j < NG; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i) longest = max_u16(longest, R.vs[j][i] & ~((kv4_nan(R.vs[j][i], 0) >> 15) * 0xffffu));
    uint32_t s = max(longest & 0xffffu, longest >> 16);
    s = max(s, (uint32_t)__shfl_xor((int)s, 16));
    s = max(s, (uint32_t)__shfl_xor((int)s, 32));
    const int down = max(lift - max(26 - (int)(s >> 10), kKv4LeastLift), 0);
    lift -= down;
    m += (float)down;
    const float a = __uint_as_float((uint32_t)(127 - down) << 23);
    l *= a;
#pragma unroll
    for (int j = 0; j < NG; ++j) {
      acc[j][0] *= a;
      acc[j][1] *= a;
    }
    acc_m *= a;
    const half2_t a2 = {(_Float16)a, (_Float16)a};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      ph[i] = as_u(as_h2(ph[i]) * a2);
      if constexpr (HILO) pl[i] = as_u(as_h2(pl[i]) * a2);
    }
  }

  // After the last stage: l over the lanes of a column, NaN where it saw a page outside the pool
  // (bad_at: the first one's position); o[4 j + i][c] its dimensions 32 j + 16 (g % 2) + 4 i +
  // 2 (g / 2) + c.
  __device__ __attribute__((always_inline)) inline void finish(int bad_at, float (&o)[4 * NG][2]) {
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (limit >= bad_at) l = __builtin_nanf("");
#pragma unroll
    for (int j = 0; j < NG; ++j) {
      const float mt = __shfl(acc_m[j], n);  // row j: lanes 0 .. 15
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        o[4 * j + i][0] = fmaf(acc[j][0][i], 0x1p20f, mt);
        o[4 * j + i][1] = fmaf(acc[j][1][i], 0x1p20f, mt);
      }
    }
  }
};

constexpr int kTokRing = 2;  // stages of a wave

// ---- waves split tokens: one workgroup per (split, sequence, kv head, 8-column tile) ----
//
// What bounds it, us a launch:
//   64 sequences of 1024..16384, 28 and 4 heads of 128: 90 for 383 MB, 4.2 TB/s of the 5.2 that a large copy
//     reaches; the stream alone takes 74, the rest is products that do not hide behind it
//   8 of 32768, 12 and 2 of 128: 26.6 for 81 MB (which the last-level cache holds from call to call): stream 14,
//     products 5.5, the waves' merge 1.4, partials and their arrival 2.4, the merge of 32 splits 3.7
//   32 of 128..4096, 14 and 2 of 64: 13.1 for 13 MB; one of 512: 7.0: the chain of lengths, pages, stages and
//     arrivals, not bytes
// Tried: equal runs of stages over all units (104..119 at the first; the prologue of every run), eight
// waves a workgroup (24.8 at the second, slower elsewhere), a ring of three at less occupancy (103),
// V in fp16 before the product (equal, less exact), K and V in rings of their own (100).
template <int DT, int D>
__device__ void kv4_tokens_impl(const Kv4AttnArgs& A) {
  constexpr int NW = kTokWaves, NT = 64 * NW, R = kTokRing;
  using Stage = Kv4Stage<D>;
  constexpr int OS = D + 4;  // floats of a column's row in LDS
  constexpr int Q = D / 4;   // float4s of a column
  __shared__ __attribute__((aligned(16))) char s_ring[NW][R][Stage::BYTES];
  constexpr int TC = kTokCols;
  __shared__ float s_m[NW][2 * TC], s_l[NW][2 * TC];
  __shared__ int s_last;
  // the ring's memory after the last stage: the waves' o; then, in the merge of the splits, the sets' o
  // and the splits' weights (what follows the stages is kv_tokens_finish of kv8_attention.hip too, in all but NB)
  float (*const s_o)[2 * TC][OS] = (float (*)[2 * TC][OS])s_ring;
  float4* const s_x = (float4*)s_ring;
  float (*const s_w)[TC] = (float (*)[TC])((char*)s_ring + NT * 16);
  static_assert(NW * 2 * TC * OS * 4 <= (int)sizeof(s_ring) && NT * 16 + kTokMaxSplits * TC * 4 <= (int)sizeof(s_ring), "fits");
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int split, tile, b, kvh;
  KvSeq S;
  if (A.longest_first) {
    if (!kv_longest_first(A, S, split, b, kvh)) return;
    tile = 0;
  } else {
    const int units = A.batch * A.hkv * A.tiles;
    split = blockIdx.x / units;
    const int u = blockIdx.x % units;
    tile = u % A.tiles;
    b = u / A.tiles / A.hkv;
    kvh = u / A.tiles % A.hkv;
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
  const int last_row = (col0 + here - 1) / A.group;
  const int last = S.start + last_row;  // the last position that a column here sees
  const int begin = split * A.split_tokens;
  const int nsplit = min(A.splits, last / A.split_tokens + 1);
  if (begin > last) return;
  const int end = min(last + 1, begin + A.split_tokens);

  // ---- the wave's stages: w, w + NW, ... of the split
  const uint32_t page_stride = (uint32_t)(A.num_layers * A.hkv) * Kv4<D>::kSlab;
  const int64_t base = ((int64_t)A.layer * A.hkv + kvh) * Kv4<D>::kSlab;
  Stage st;
  st.begin(A.k_pool + base, A.v_pool + base);
  const int32_t* const table = A.tables + (int64_t)b * A.table_stride;
  const int stages = (end - begin + Stage::TOKENS - 1) / Stage::TOKENS;
  const int count = stages > w ? (stages - w + NW - 1) / NW : 0;
  const int min_limit = S.start + col0 / A.group;
  int bad_at = 0x7fffffff;
  int pages[Stage::PAGES];  // of stage chunk + lane
  auto load_pages = [&](int chunk) __attribute__((always_inline)) {
    const int lane = threadIdx.x & 63;
    const int64_t tok = begin + ((int64_t)(chunk + lane) * NW + w) * Stage::TOKENS;
    int bad = 0x7fffffff;
#pragma unroll
    for (int i = Stage::PAGES - 1; i >= 0; --i) {
      const int64_t at = tok + i * kPage;
      pages[i] = at < end ? table[at / kPage] : 0;
      // a page outside the pool is never an address: page 0 is read instead
      if (pages[i] < 0 || pages[i] >= A.num_blocks) {
        bad = (int)at;
        pages[i] = 0;
      }
    }
    if (__any(bad != 0x7fffffff)) {
#pragma unroll
      for (int k = 1; k < 64; k <<= 1) bad = min(bad, __shfl_xor(bad, k));
      bad_at = min(bad_at, bad);
    }
  };
  auto issue = [&](int i) __attribute__((always_inline)) {
    const int p0 = __builtin_amdgcn_readlane(pages[0], i & 63), p1 = __builtin_amdgcn_readlane(pages[1], i & 63);
    int p2 = 0, p3 = 0;
    if constexpr (Stage::PAGES == 4) {
      p2 = __builtin_amdgcn_readlane(pages[2], i & 63);
      p3 = __builtin_amdgcn_readlane(pages[3], i & 63);
    }
    st.issue(s_ring[w][i % R], p0, p1, p2, p3, page_stride);
  };
  if (count) load_pages(0);
#pragma unroll
  for (int i = 0; i < R; ++i)
    if (i < count) issue(i);
  Kv4Row<DT, D> W;
  W.begin(A, S.row0, kvh, S.start, S.ctx, col0, ncols);
  for (int i = 0; i < count; ++i) {
    static_assert(R == 2, "at most one stage is under way behind this one");
    if (i + 1 < count) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(Stage::LOADS) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    const int tok0 = begin + (i * NW + w) * Stage::TOKENS;
    const uint32_t lds = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char*)s_ring[w][i % R];
#pragma unroll
    for (int u = 0; u < Stage::SUB; ++u) {
      const int t = tok0 + 32 * u;
      if (t <= last) W.step(lds, u, t, S.ctx, t + 31 > min_limit);
    }
    const int nx = i + R;
    if (nx < count) {
      if ((nx & 63) == 0) load_pages(nx);
      issue(nx);
    }
  }
  float o_wave[D / 8][2];
  W.finish(bad_at, o_wave);
  const int n = W.n, g = W.g;
  if (g == 0) {
    s_m[w][n] = W.m;
    s_l[w][n] = W.l;
  }
  __syncthreads();  // every wave is done with its ring
#pragma unroll
  for (int k = 0; k < D / 8; ++k)
    *(float2*)&s_o[w][n][32 * (k >> 2) + 16 * (g & 1) + 4 * (k & 3) + 2 * (g >> 1)] = make_float2(o_wave[k][0], o_wave[k][1]);
  __syncthreads();
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
  constexpr int NB = 16;
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

// ---- waves split columns: one workgroup per (chunk of columns, sequence, kv head, split) ----
//
// The waves expand a tile of 64 tokens together into LDS in operand order (a lane's 16 bytes
// of every operand side by side: reads without conflicts), one tile ahead of the products and with
// the loads of another under way; one barrier a tile.  A k step of a score is a group of 32
// dimensions.  A wave has 32 columns; all of K's and V's reads of 32 tokens are under way before the products and
// the softmax that need them.
//
// What bounds it: issue.  A product of 16 x 16 x 32 keeps a SIMD's VALU from issuing for about 8 of its
// 16 cycles, and 32 tokens of 16 columns take (128 dimensions, bf16) 17 products and some 60 VALU
// instructions: the softmax's 34, the column's share of the expansion, masks and loop.
//   16 prompts of 1531..2048, 14 and 2 heads of 64, bf16: 141 us, 650 TFLOP/s; fp16: 208 (28 products and 32
//     more FMAs: EXACT); 12 and 2 of 128, bf16: 224 us, 700 TFLOP/s
//   4 of them: 47.4, the longest columns' chain of 32 tiles at the end
//   512 rows after 8000, 12 and 2 of 128: fp16 65.7 with 7.6 in the merge of ten splits; bf16 45
// Tried, us for bf16 rows of 4 such prompts at 64 dimensions, at 128, and the 512 rows (47.6, 68, 45.6 as it
// is): 16 waves of one fragment (two at 64) 71.6, 70, 47.2; 4 waves of four fragments at 64 65; 8 of one
// there 52.8; reads of LDS as they are needed 48.3, 77, 47; products of 32 x 32 x 16 in three forms
// 50.0..52.7, 69.8..74.7, 48.2..52.0, and with the softmax between the products of the next 32
// tokens 52.5, 70, 48; a raised wave priority around the products no gain; expansion by every wave for
// itself 105 at the first.
//   bf16 rows: K and V are n s + m in fp16, one rounding of 2^-12, far below the output's 2^-9 (and an eighth of
//     what K in bf16 is off by).  Where a group of K lies far from 0 and q takes that out of the scores, what the
//     rounding leaves is seen: 2.5e-3 of the output with the group at 10, 8e-3 at 50; n and m apart, as fp16 rows
//     have them, would be 11 products for 9 of 32 tokens at 64 dimensions, 19 for 17 at 128.
//   fp16 rows (EXACT): that rounding of K and P's own would each add an error as large as the output's.
//     K is n, and a group's products are scaled by s in 32 bits; the group's sum of q times m, q's sums
//     in two fp16 parts, are a product of their own.  P is two fp16 parts.  V stays n s + m in one fp16: a
//     second part would be 8 more products than the 28 of 32 tokens at 128 dimensions and as much LDS again, for
//     errors of 2.1e-4 at most (the output's own rounding) in place of 2.8e-4.
template <int DT, int D> struct Kv4Tile {
  static constexpr bool EXACT = DT == kF16;
  static constexpr int KS = D / 32;   // k steps of a score
  static constexpr int NF = D / 16;   // output fragments: 4 a quad of V
  uint4 k[4][KS][64];                 // [fragment of 16 tokens][step][lane]
  uint4 v[2][NF][64];                 // [half][fragment of dimensions][lane]
  uint16_t ks[EXACT ? 4 : 1][16][KS]; // s by token and group
  uint4 km[EXACT ? 4 : 1][16];        // m by token: the groups', repeated to 8
};
template <int D> struct Kv4Cols {
  static constexpr int WAVES = D == 128 ? 8 : 4;
  static constexpr int F = 2;  // fragments of a wave
  static constexpr int N = WAVES * F * 16;
};

// What a wave loads of a tile and makes of it: of page w % 4, C dwords of K a lane, and V's quads n + 16 h
// for HW halves h of the dimensions, four tokens a lane (two dwords).  One page: its address is scalar.
template <int DT, int D> struct Kv4Expand {
  static constexpr bool EXACT = DT == kF16;
  static constexpr int KS = D / 32, C = D / 8 / Kv4Cols<D>::WAVES, HW = C / 2;
  uint32_t k[C], ksm;
  uint2 v[HW], vs[HW], vm[HW];
  const char* kp;  // page 0
  const char* vp;
  int ko, kso, vo, vso;  // of the lane in a page
  int n, g, page, part;  // part: of the lane's D / 32 dwords of K, or of V's halves

  __device__ __attribute__((always_inline)) inline void begin(const char* k_pool, const char* v_pool, int wave) {
    const int lane = threadIdx.x & 63;
    n = lane & 15;
    g = lane >> 4;
    page = wave & 3;
    part = wave >> 2;
    kp = k_pool;
    vp = v_pool;
    ko = (int)Kv4<D>::k_row(n) + g * (D / 8) + part * C * 4;
    kso = (int)Kv4<D>::k_scale(n, D == 128 ? g : g >> 1);
    vo = (int)Kv4<D>::v_quad(8 * (g >> 1), n + 16 * HW * part) + 8 * (g & 1);
    vso = (int)Kv4<D>::v_scale(g >> 1, (n >> 3) + 2 * HW * part) + 8 * (g & 1);
  }
  // p (alike in all lanes): the page.
  __device__ __attribute__((always_inline)) inline void load(int p, uint32_t page_stride) {
    const uint64_t at = (uint64_t)(uint32_t)p * page_stride;
    const char* const ka = kp + at;
    const char* const va = vp + at;
    if constexpr (C == 4) {
      const uint4 y = *(const uint4*)(ka + ko);
      k[0] = y.x; k[1] = y.y; k[2] = y.z; k[3] = y.w;
    } else {
      const uint2 y = *(const uint2*)(ka + ko);
      k[0] = y.x; k[1] = y.y;
    }
    ksm = *(const uint32_t*)(ka + kso);
#pragma unroll
    for (int h = 0; h < HW; ++h) {
      v[h] = *(const uint2*)(va + vo + 256 * h);
      vs[h] = *(const uint2*)(va + vso + 64 * h);
      vm[h] = *(const uint2*)(va + vso + 64 * h + 16);
    }
  }
  // What tokens from `end` on hold is unknown, and no column that is kept sees it: their s and m of
  // V become 0.  So do NaN ones', since 0 * NaN would reach columns that do not see them: nan_at, by
  // group, keeps the first position.
  __device__ __attribute__((always_inline)) inline void store(Kv4Tile<DT, D>& T, int tok0, int end, int* nan_at) {
    const int lane = threadIdx.x & 63;
    const half2_t sm = as_h2(ksm);
    const half2_t ks = {sm.x, sm.x}, km = {sm.y, sm.y};
#pragma unroll
    for (int j = 0; j < C; ++j) {
      uint32_t o[4];
      if constexpr (EXACT) whole8(k[j], o); else expand8(k[j], ks, km, o);
      // the lane's dword i of dimensions 8 (D / 32 g + i) and the next 7
      const int i = D / 32 * g + part * C + j;
      T.k[page][i >> 2][16 * (i & 3) + n] = make_uint4(o[0], o[1], o[2], o[3]);
    }
    if constexpr (EXACT) {
      const int group = D == 128 ? g : g >> 1;
      if (part == 0 && (D == 128 || !(g & 1))) {
        T.ks[page][n][group] = (uint16_t)ksm;
        uint16_t* const to = (uint16_t*)&T.km[page][n] + group;
#pragma unroll
        for (int r = 0; r < 8; r += KS) to[r] = (uint16_t)(ksm >> 16);
      }
    }
    const int first = tok0 + 16 * page + 4 * g;  // of the lane's four tokens
    if (tok0 + 64 > end) {
      const uint32_t lo = (first < end ? 0xffffu : 0u) | (first + 1 < end ? 0xffff0000u : 0u);
      const uint32_t hi = (first + 2 < end ? 0xffffu : 0u) | (first + 3 < end ? 0xffff0000u : 0u);
#pragma unroll
      for (int h = 0; h < HW; ++h) {
        vs[h].x &= lo; vs[h].y &= hi;
        vm[h].x &= lo; vm[h].y &= hi;
      }
    }
    // 0 times s and m: NaN where one is not finite (the format has no infinities)
    half2_t any = {(_Float16)0.0f, (_Float16)0.0f};
    const half2_t zero = any;
#pragma unroll
    for (int h = 0; h < HW; ++h) {
      any = __builtin_elementwise_fma(as_h2(vs[h].x), zero, any);
      any = __builtin_elementwise_fma(as_h2(vs[h].y), zero, any);
      any = __builtin_elementwise_fma(as_h2(vm[h].x), zero, any);
      any = __builtin_elementwise_fma(as_h2(vm[h].y), zero, any);
    }
    if (__any((as_u(any) & 0x7fff7fffu) != 0)) {
#pragma unroll
      for (int h = 0; h < HW; ++h) {
        const uint32_t lo = kv4_nan(vs[h].x, vm[h].x), hi = kv4_nan(vs[h].y, vm[h].y);
        const uint32_t keep_lo = (lo & 0x8000u ? 0u : 0xffffu) | (lo & 0x80000000u ? 0u : 0xffff0000u);
        const uint32_t keep_hi = (hi & 0x8000u ? 0u : 0xffffu) | (hi & 0x80000000u ? 0u : 0xffff0000u);
        vs[h].x &= keep_lo; vm[h].x &= keep_lo;
        vs[h].y &= keep_hi; vm[h].y &= keep_hi;
        if (lo | hi)
          atomicMin(nan_at + (n >> 3) + 2 * (HW * part + h),
                    first + (lo & 0x8000u ? 0 : lo ? 1 : hi & 0x8000u ? 2 : 3));
      }
    }
#pragma unroll
    for (int h = 0; h < HW; ++h) {
      uint32_t o[2][4];  // [pair of tokens][dimension]
      expand8(v[h].x, as_h2(vs[h].x), as_h2(vm[h].x), o[0]);
      expand8(v[h].y, as_h2(vs[h].y), as_h2(vm[h].y), o[1]);
#pragma unroll
      for (int c = 0; c < 4; ++c)
        ((uint2*)&T.v[page >> 1][4 * (HW * part + h) + c][lane])[page & 1] = make_uint2(o[0][c], o[1][c]);
    }
  }
};

// One wave's F fragments of 16 columns over tiles.
template <int DT, int D> struct Kv4Chunk {
  static constexpr bool EXACT = DT == kF16;
  static constexpr int F = Kv4Cols<D>::F, KS = D / 32, NF = D / 16, H = D / 64;
  static constexpr bool AHEAD = !EXACT || D == 128;  // V is read before the softmax, where registers allow
  uint4 q[F][KS], qsum[EXACT ? F : 1];
  f32x4_t acc[F][NF], l[F];
  float m[F], scale[F], bar[F];  // m: less kKv4ColsLift
  int limit[F];  // last position that the lane's column sees
  int lane, n, g;

  // Columns col0 + 16 f + n of a sequence with ncols of them whose first row is at `start`.
  __device__ __attribute__((always_inline)) inline void begin(const Kv4AttnArgs& A, int64_t row0, int kvh, int start, int ctx, int col0,
                                                              int ncols) {
    lane = threadIdx.x & 63;
    n = lane & 15;
    g = lane >> 4;
#pragma unroll
    for (int f = 0; f < F; ++f) {
      const int col = col0 + 16 * f + n;
      const bool on = col < ncols;
      const int r = on ? col / A.group : 0, hd = on ? col % A.group : 0;
      limit[f] = on ? start + r : ctx - 1;
      const uint16_t* const src = A.q + (row0 + r) * A.q_stride + ((int64_t)kvh * A.group + hd) * D + 8 * g;
      float x[KS][8];
      float top = 0.0f;
#pragma unroll
      for (int j = 0; j < KS; ++j) {
        const uint4 w = on ? *(const uint4*)(src + 32 * j) : make_uint4(0, 0, 0, 0);
        const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[j][2 * e] = St<DT>::lo(ww[e]);
          x[j][2 * e + 1] = St<DT>::hi(ww[e]);
          top = fmaxf(top, fmaxf(fabsf(x[j][2 * e]), fabsf(x[j][2 * e + 1])));
        }
      }
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      // a power of two takes the largest element into [1, 2) (infinities and NaN stay so), and the
      // scale's sign goes to q, so that the largest product is the largest score
      const int e = min(max((int)(__float_as_uint(top) >> 23), 1), 253);
      const float down = copysignf(__uint_as_float((uint32_t)(254 - e) << 23), A.qk_scale_log2);
      scale[f] = fabsf(A.qk_scale_log2) * __uint_as_float((uint32_t)e << 23);
      if (scale[f] == 0.0f) scale[f] = 1e-37f;  // (a masked product, -inf, times 0 is NaN)
      uint32_t sums[KS];  // of q by group: two fp16 parts
#pragma unroll
      for (int j = 0; j < KS; ++j) {
        uint32_t o[4];
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const half2_t p = {(_Float16)(x[j][i] * down), (_Float16)(x[j][i + 4] * down)};
          o[i] = as_u(p);
          sum += (float)p.x + (float)p.y;
        }
        q[f][j] = make_uint4(o[0], o[1], o[2], o[3]);
        sum += __shfl_xor(sum, 16);
        sum += __shfl_xor(sum, 32);
        const _Float16 hi = (_Float16)sum;
        sums[j] = as_u((half2_t){hi, (_Float16)(sum - (float)hi)});
      }
      if constexpr (EXACT) {
        // k slots 0 .. KS - 1 of lanes 0 .. 15: first parts; KS .. 2 KS - 1: second parts
        auto pair = [](uint32_t a, uint32_t b, bool second) __attribute__((always_inline)) {
          return second ? (a >> 16) | (b & 0xffff0000u) : (a & 0xffffu) | b << 16;
        };
        if constexpr (KS == 4)
          qsum[f] = make_uint4(pair(sums[0], sums[1], false), pair(sums[2], sums[3], false),
                               pair(sums[0], sums[1], true), pair(sums[2], sums[3], true));
        else
          qsum[f] = make_uint4(pair(sums[0], sums[1], false), pair(sums[0], sums[1], true), 0, 0);
        if (g != 0) qsum[f] = make_uint4(0, 0, 0, 0);
      }
      m[f] = -3.4028235e38f;
      bar[f] = -INFINITY;
      l[f] = (f32x4_t){0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < NF; ++i) acc[f][i] = (f32x4_t){0, 0, 0, 0};
    }
  }

  // Half `half` of a tile: tokens tok0 .. tok0 + 31.  edge (alike in all lanes): some column's limit
  // lies before its end.
  __device__ __attribute__((always_inline)) inline void step(const Kv4Tile<DT, D>& T, int half, int tok0, bool edge) {
    const f32x4_t zero = {0, 0, 0, 0};
    float s[F][8];  // tokens 4 g .. 4 g + 3 of either page
    // all of K's reads under way before the first product, all of V's before the softmax
    uint4 kk[2][KS], km[2], ks[2][KS / 2];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
#pragma unroll
      for (int j = 0; j < KS; ++j) kk[b][j] = T.k[2 * half + b][j][lane];
      if constexpr (EXACT) {
        km[b] = T.km[2 * half + b][n];
#pragma unroll
        for (int i = 0; i < KS / 2; ++i) ks[b][i] = ((const uint4*)T.ks[2 * half + b][4 * g])[i];  // 4 tokens' s
      }
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      f32x4_t t[F];
      if constexpr (EXACT) {
        uint32_t sc[2 * KS];
#pragma unroll
        for (int i = 0; i < KS / 2; ++i) {
          sc[4 * i] = ks[b][i].x; sc[4 * i + 1] = ks[b][i].y; sc[4 * i + 2] = ks[b][i].z; sc[4 * i + 3] = ks[b][i].w;
        }
#pragma unroll
        for (int f = 0; f < F; ++f) t[f] = mfma16(km[b], qsum[f], zero);
#pragma unroll
        for (int j = 0; j < KS; ++j)
#pragma unroll
          for (int f = 0; f < F; ++f) {
            const f32x4_t c = mfma16(kk[b][j], q[f][j], zero);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const half2_t sj = as_h2(sc[(i * KS + j) / 2]);
              t[f][i] = fmaf(c[i], (float)(j & 1 ? sj.y : sj.x), t[f][i]);
            }
          }
      } else {
#pragma unroll
        for (int j = 0; j < KS; ++j)
#pragma unroll
          for (int f = 0; f < F; ++f) t[f] = mfma16(kk[b][j], q[f][j], j == 0 ? zero : t[f]);
      }
#pragma unroll
      for (int f = 0; f < F; ++f)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[f][4 * b + i] = t[f][i];
    }
    uint4 vv[NF];
    if constexpr (AHEAD) {
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < NF; ++i) vv[i] = T.v[half][i][lane];
      __builtin_amdgcn_sched_barrier(0);
    } else {
      asm volatile("" ::: "memory");  // (no read of V moves up)
    }
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
        const float mn = fmaxf(m[f], kv4_reference(t * scale[f], kKv4ColsLift));
        const float a = __builtin_amdgcn_exp2f(m[f] - mn);
        bar[f] = fmaxf(bar[f], t + kLazyMax / scale[f]);
        m[f] = mn;
        l[f] *= a;
#pragma unroll
        for (int i = 0; i < NF; ++i) acc[f][i] *= a;
      }
    }
    float less = -1.0f;
    asm("" : "+s"(less));  // (times a fp16, plus an fp32: one instruction)
    uint4 p[F], p2[EXACT ? F : 1];
#pragma unroll
    for (int f = 0; f < F; ++f) {
      uint32_t o[4], o2[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = __builtin_amdgcn_exp2f(fmaf(s[f][2 * i], scale[f], -m[f]));
        const float y = __builtin_amdgcn_exp2f(fmaf(s[f][2 * i + 1], scale[f], -m[f]));
        o[i] = as_u((half2_t){(_Float16)x, (_Float16)y});
        if constexpr (EXACT) {
          asm("" : "+v"(o[i]));  // (converted once, as a pair)
          const half2_t h = as_h2(o[i]);
          o2[i] = as_u((half2_t){(_Float16)fmaf((float)h.x, less, x), (_Float16)fmaf((float)h.y, less, y)});
        }
      }
      p[f] = make_uint4(o[0], o[1], o[2], o[3]);
      if constexpr (EXACT) p2[f] = make_uint4(o2[0], o2[1], o2[2], o2[3]);
    }
    const uint4 ones = make_uint4(0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u);
#pragma unroll
    for (int f = 0; f < F; ++f) {
      l[f] = mfma16(ones, p[f], l[f]);
      if constexpr (EXACT) l[f] = mfma16(ones, p2[f], l[f]);
    }
    if constexpr (!AHEAD) {
#pragma unroll
      for (int i = 0; i < NF; ++i) vv[i] = T.v[half][i][lane];
    }
#pragma unroll
    for (int i = 0; i < NF; ++i)
#pragma unroll
      for (int f = 0; f < F; ++f) {
        acc[f][i] = mfma16(vv[i], p[f], acc[f][i]);
        if constexpr (EXACT) acc[f][i] = mfma16(vv[i], p2[f], acc[f][i]);
      }
  }

  // After the last tile: NaN where a column saw a page outside the pool
  // (bad_at: the first one's position) or a NaN value (nan_at, by group; a lane's outputs of half h
  // are of group 2 h + g / 2).
  __device__ __attribute__((always_inline)) inline void finish(int bad_at, const int* nan_at) {
#pragma unroll
    for (int f = 0; f < F; ++f) {
      if (limit[f] >= bad_at) l[f][0] = __builtin_nanf("");
#pragma unroll
      for (int h = 0; h < H; ++h)
        if (limit[f] >= nan_at[2 * h + (g >> 1)]) {
#pragma unroll
          for (int c = 0; c < 4; ++c) acc[f][4 * h + c] = (f32x4_t)__builtin_nanf("");
        }
    }
  }
};

template <int DT, int D>
__device__ void kv4_columns_impl(const Kv4AttnArgs& A) {
  using C = Kv4Cols<D>;
  constexpr int F = C::F;
  __shared__ Kv4Tile<DT, D> s_tile[2];
  __shared__ int s_nan[D / 32 + 1];  // and the first position of a page outside the pool
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // The chunks that see the longest contexts first, and split 0, which every chunk has, before the
  // others; neighbours of a pair on different XCDs (block x runs on XCD x % 8).
  const int pairs = A.batch * A.hkv;
  const int split = blockIdx.x / (pairs * A.tiles), rest = blockIdx.x % (pairs * A.tiles);
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
  const int begin = split * A.split_tokens;  // (splits x split_tokens fits: luc_kv4.cpp)
  if (begin > all_last) return;
  const int end = A.splits == 1 ? all_last + 1 : min(all_last + 1, begin + A.split_tokens);
  const int col0 = all0 + w * (16 * F);
  const int here = min(16 * F, ncols - col0);  // the wave's, or none
  const int last = here > 0 ? S.start + (col0 + here - 1) / A.group : -1;
  const int min_limit = S.start + col0 / A.group;
  if (threadIdx.x <= D / 32) s_nan[threadIdx.x] = 0x7fffffff;

  const uint32_t page_stride = (uint32_t)(A.num_layers * A.hkv) * Kv4<D>::kSlab;
  const int64_t base = ((int64_t)A.layer * A.hkv + kvh) * Kv4<D>::kSlab;
  const int32_t* const table = A.tables + (int64_t)b * A.table_stride;
  Kv4Expand<DT, D> E;
  E.begin(A.k_pool + base, A.v_pool + base, w);
  const int count = (end - begin + 63) / 64;  // tiles
  int bad_at = 0x7fffffff;  // of the wave's pages
  int pages = 0;            // the wave's of tile i + lane
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
        if (bad_at == 0x7fffffff && (threadIdx.x & 63) == 0) atomicMin(s_nan + D / 32, first);
        bad_at = min(bad_at, first);
        pages = bad ? 0 : pages;
      }
    }
    E.load(__builtin_amdgcn_readlane(pages, i & 63), page_stride);
  };
  __syncthreads();  // s_nan
  load(0);
  Kv4Chunk<DT, D> W;
  W.begin(A, S.row0, kvh, S.start, S.ctx, min(col0, ncols - 1), ncols);
  E.store(s_tile[0], begin, min(end, bad_at), s_nan);
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
      E.store(s_tile[(i + 1) & 1], tok0 + 64, min(end, bad_at), s_nan);
      if (i + 2 < count) load(i + 2);
      __syncthreads();
    }
  }
  W.finish(s_nan[D / 32], s_nan);
  // A lane holds 16 dimensions of a column.  By way of the wave's share of the tiles, which no wave
  // reads any more, D / 4 lanes write a column side by side.  (kv_columns_out of kv8_attention.hip too.)
  __syncthreads();
  const int hq = A.hkv * A.group;
  float4* const turn = (float4*)s_tile + w * (4 * D);  // [16 columns][D / 4], swizzled
  static_assert(sizeof(s_tile) >= C::WAVES * 4 * D * sizeof(float4), "a share holds 16 columns");
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

}  // namespace luc

#define LUC_KV4_ATTENTION(DTN, DT, D)                                                            \
  extern "C" __global__ __launch_bounds__(256, 2) void luc_kv4_tokens_##DTN##_d##D(luc::Kv4AttnArgs a) {  \
    luc::kv4_tokens_impl<luc::DT, D>(a);                                                         \
  }                                                                                              \
  extern "C" __global__ __launch_bounds__(64 * luc::Kv4Cols<D>::WAVES, D == 128 ? 2 : 3) void luc_kv4_columns_##DTN##_d##D(luc::Kv4AttnArgs a) { \
    luc::kv4_columns_impl<luc::DT, D>(a);                                                        \
  }                                                                                              \
  extern "C" __global__ __launch_bounds__(256) void luc_kv4_merge_##DTN##_d##D(luc::Kv4AttnArgs a) {      \
    luc::kv_merge_impl<luc::DT, D>(a);                                                          \
  }
LUC_KV4_ATTENTION(bf16, kBF16, 64)
LUC_KV4_ATTENTION(bf16, kBF16, 128)
LUC_KV4_ATTENTION(f16, kF16, 64)
LUC_KV4_ATTENTION(f16, kF16, 128)
