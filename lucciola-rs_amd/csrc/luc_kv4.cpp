// luc_kv4.cpp -- host side of the page maps on the GPU, the normed appends and the
// 4-bit cache (include/luc_attn.h, "Serving over a paged cache held on the GPU"): argument checks, work
// splits and launches of block_map.hip, norm_append.hip and kv4_attention.hip.  Nothing here
// allocates device memory or synchronises.
#include "luc_internal.h"

#include <algorithm>

using namespace luc_internal;

namespace {

const char* dt_name(int dtype) { return dtype == LUC_F16 ? "f16" : "bf16"; }

constexpr int kGroup4 = 32;             // values of a 4-bit group (kernels/kv4.h)
constexpr int kMaxMapBatch = 4096;      // block_map.hip: kMaxSeqs
constexpr int kMaxTableStride = 1 << 26;  // positions stay below 2^30

constexpr int kMaxHeads = 1 << 20;        // rows of heads stay within 32 bits

int64_t align256(int64_t n) { return ceil_div(n, 256) * 256; }

// luc::MapArgs of block_map.hip: the same fields in the same order.
struct MapArgs {
  const int32_t* count;
  int32_t* lens;
  int32_t* tables;
  int64_t table_stride;
  int32_t* free_list;
  int32_t* state;
  int64_t* slots;
  int32_t* positions;
  int32_t* cu_seqlens;
  int32_t* start_pos;
  int32_t batch, num_blocks, rows;
};

int check_map(const luc_ctx* ctx, const MapArgs& a, int table_stride) {
  if (!ctx) return fail(LUC_E_INVALID, "null context");
  if (a.batch < 0) return fail(LUC_E_INVALID, "batch %d < 0", a.batch);
  if (a.batch > kMaxMapBatch)
    return fail(LUC_E_UNSUPPORTED, "batch %d above %d sequences", a.batch, kMaxMapBatch);
  if (table_stride <= 0 || table_stride > kMaxTableStride)
    return fail(LUC_E_INVALID, "table_stride %d outside [1, %d]", table_stride, kMaxTableStride);
  if (a.num_blocks < 1) return fail(LUC_E_INVALID, "num_blocks %d < 1", a.num_blocks);
  if ((a.batch && (!a.count || !a.lens || !a.tables)) || !a.free_list || !a.state)
    return fail(LUC_E_INVALID, "null counts, lengths, tables, free list or state");
  return LUC_OK;
}

// luc::NormAppendArgs of norm_append.hip: the same fields in the same order.
struct NormAppendArgs {
  const void* q;
  const void* k;
  const void* v;
  int64_t row_stride;
  const void* q_bias;
  const void* k_bias;
  const void* v_bias;
  const void* q_norm;
  const void* k_norm;
  const float* cos_t;
  const float* sin_t;
  const int32_t* positions;
  const int64_t* slots;
  void* q_out;
  int64_t q_out_stride;
  void* k_out;
  void* v_out;
  int64_t kv_out_stride;
  void* k_pool;
  void* v_pool;
  int64_t num_slots;
  float eps;
  int32_t rows, max_pos, layer, num_layers, hq, hkv;
};

int check_sizes(const luc_ctx* ctx, int dtype, int hq, int hkv, int head_dim, int block_size, int layer,
                int num_layers, int num_blocks) {
  if (!ctx) return fail(LUC_E_INVALID, "null context");
  if (dtype != LUC_BF16 && dtype != LUC_F16) return fail(LUC_E_INVALID, "bad dtype %d", dtype);
  if (head_dim != 64 && head_dim != 128)
    return fail(LUC_E_UNSUPPORTED, "unsupported head_dim %d (64 or 128)", head_dim);
  if (hq <= 0 || hkv <= 0) return fail(LUC_E_INVALID, "head counts must be positive");
  if (hq > kMaxHeads) return fail(LUC_E_INVALID, "num_q_heads %d above %d", hq, kMaxHeads);
  if (hq % hkv) return fail(LUC_E_INVALID, "num_q_heads %d not a multiple of num_kv_heads %d", hq, hkv);
  if (hq / hkv > 8) return fail(LUC_E_UNSUPPORTED, "group size %d > 8", hq / hkv);
  if (block_size != LUC_BLOCK_SIZE)
    return fail(LUC_E_UNSUPPORTED, "block_size %d (only %d)", block_size, LUC_BLOCK_SIZE);
  if (num_layers <= 0 || layer < 0 || layer >= num_layers)
    return fail(LUC_E_INVALID, "layer %d outside [0, %d)", layer, num_layers);
  if (num_blocks < 1) return fail(LUC_E_INVALID, "num_blocks %d < 1", num_blocks);
  return LUC_OK;
}

int norm_append(luc_ctx* ctx, void* stream, int dtype, const char* kind, NormAppendArgs& a, int num_blocks,
                int head_dim, int block_size) {
  if (int rc = check_sizes(ctx, dtype, a.hq, a.hkv, head_dim, block_size, a.layer, a.num_layers, num_blocks))
    return rc;
  if (a.rows < 0) return fail(LUC_E_INVALID, "num_tokens %d < 0", a.rows);
  if (a.max_pos < 1) return fail(LUC_E_INVALID, "max_pos %d < 1", a.max_pos);
  if ((a.rows && (!a.q || !a.k || !a.v || !a.q_out || !a.positions || !a.slots)) || !a.cos_t || !a.sin_t ||
      !a.k_pool || !a.v_pool)
    return fail(LUC_E_INVALID, "null q, k, v, q_out, rope table, positions, slots or pool");
  if (!a.q_norm != !a.k_norm) return fail(LUC_E_INVALID, "one of q_norm and k_norm without the other");
  // (a row of q, k and v each starts 16-byte loads)
  const int q_row = a.hq * head_dim, kv_row = a.hkv * head_dim;
  if (a.row_stride < q_row || a.q_out_stride < q_row ||
      ((a.k_out || a.v_out) && a.kv_out_stride < kv_row))
    return fail(LUC_E_INVALID, "row stride smaller than a row (%d, %d)", q_row, kv_row);
  if (a.row_stride % 8 || a.q_out_stride % 8 || ((a.k_out || a.v_out) && a.kv_out_stride % 8))
    return fail(LUC_E_INVALID, "row strides must be multiples of 8 elements");
  for (const void* p : {a.q, a.k, a.v, a.q_bias, a.k_bias, a.v_bias, a.q_norm, a.k_norm, (const void*)a.cos_t,
                        (const void*)a.sin_t, (const void*)a.q_out, (const void*)a.k_out, (const void*)a.v_out,
                        (const void*)a.k_pool, (const void*)a.v_pool})
    if (!aligned(p, 16)) return fail(LUC_E_INVALID, "operands must be 16-byte aligned");
  if (!aligned(a.slots, 8) || !aligned(a.positions, 4))
    return fail(LUC_E_INVALID, "slots must be 8-byte aligned, positions 4-byte");
  a.num_slots = (int64_t)num_blocks * LUC_BLOCK_SIZE;
  if (a.rows == 0) return LUC_OK;
  if (int rc = check_device(ctx)) return rc;
  hipFunction_t fn;
  if (int rc = get_fn(ctx, std::string(kind) + dt_name(dtype) + "_d" + std::to_string(head_dim), &fn)) return rc;
  const int64_t lanes = (int64_t)a.rows * (a.hq + 2 * a.hkv) * (head_dim / 16);
  const int64_t grid = ceil_div(lanes, 256);
  if (grid * 256 > UINT32_MAX) return fail(LUC_E_INVALID, "too many rows for one launch");
  void* args[] = {&a};
  return launch(fn, dim3((unsigned)grid), dim3(256), stream, args);
}

// luc::Kv4AttnArgs of kv4_attention.hip: the same fields in the same order.
struct Kv4AttnArgs {
  const void* q;
  int64_t q_stride;
  void* out;
  int64_t out_stride;
  const void* k_pool;
  const void* v_pool;
  const int32_t* tables;
  int64_t table_stride;
  const int32_t* cu_seqlens;
  const int32_t* start_pos;
  int32_t* ws_cnt;
  float* ws_ml;
  float* ws_o;
  int32_t batch, total_rows, max_rows, max_ctx, layer, num_layers, hkv, group, num_blocks;
  int32_t tiles, splits, split_tokens, longest_first;
  float qk_scale_log2;
};

constexpr int kCUs = 256;
constexpr int kTokCols = 8;                   // columns of a workgroup
constexpr int kTokMaxSplits = 256;            // kv4_attention.hip
constexpr int kTokSlots = 2 * kCUs;           // workgroups that a launch is planned for: two a CU (128 dimensions
                                              // hold two, 64 three, by their registers)
// Split lengths of a tokens launch: what fills the chip once, but not shorter than is worth a merge
// and not longer than lets mixed contexts end together.  us at fixed lengths (of one build, up to 2% below
// the present one's), batch x context, heads:
//   8 x 32768, 12 and 2 of 128: 40.3 at 512, 25.6 at 1024 (the rule's) and 2048
//   32 x 128..4096, 14 and 2 of 64: 13.9 at 256, 13.2 at 512 (the rule's), 13.7 at 1024
//   64 x 1024..16384, 28 and 4 of 128: 104 at 1024, 87.6 at 2048 (the rule's), 90.9 at 4096;
//     all of 8192: 74.8, 69.9 at 4096, 66.8 whole
//   256 x 1000, 14 and 2 of 64: 24.1 at 256, 20.8 at 512, 15.4 whole (the rule's)
//   1 x 32768, 14 and 2 of 64: 12.9 at 512 (the rule's), 13.1 at 1024
//   4 x 4000, 28 and 4 of 128: 16.9 at 128, 13.3 at 256 and 512 (the rule's), 16.0 at 1024
// More than one round of workgroups starts with the longest (64 x 1024..16384: 87.5, in plain order
// 93.8).
constexpr int kTokMinSplit = 512, kTokMaxSplit = 2048;
constexpr int kTokRounds = 8;  // rounds of workgroups balance any contexts: longer splits beyond
// Up to 16 columns go to the tokens kernel, which reads the cache once for each 8; up to 48 while its
// tiles leave the chip room.  us, tokens and columns kernel, sequences x rows at 1000..2000 tokens:
//   14 and 2 heads of 64: 1 x 6 of 8000 12.6, 18.2; 16 x 6 17.4, 18.2; 64 x 3 21.1, 19.6;
//     64 x 6 (768 tiles) 26.6, 23.0; 256 x 3 of 100..200 (1536) 15.5, 11.0
//   12 and 2 of 128: 1 x 8 of 8000 15.3, 22.5; 64 x 4 30.5, 38.2; 64 x 8 (768 tiles) 45.7, 41.4
constexpr int kTokMostCols = 48;
// Columns of a workgroup of the columns kernel (Kv4Cols).
constexpr int kColsOf64 = 128, kColsOf128 = 256;
// Its splits fill the chip once, planned as a workgroup a CU (128) or two (64, whose registers hold three), but
// are not shorter than pays for their partials.  us:
//   512 rows after 8000, 12 and 2 of 128: 44.3 at 832 and 45.0 at 896 (the rule's), 71 at 768, where a
//     second round begins; 64 rows: 26.0 at 256 (the rule's), 29.8 at 512
//   14 and 2 of 64, 512 rows after 8000: 45.2 at 576, 36.5 at 640, 36.7 at 960 (the rule's), 38.4 at
//     1088; 128 rows: 21.7 at 256, 20.6 at 512 (the rule's), 27.7 at 1024
//   4 x 1531..2048 rows, 14 and 2 of 64: 67 at 1024, 47.6 whole (the rule's)
constexpr int kColsMinSplit64 = 512, kColsMinSplit128 = 256, kColsMaxSplits = 32;
constexpr int64_t kMaxArrivals = 1 << 16;     // (sequence, kv head, column tile)
constexpr int kMaxCtx = 1 << 30;

struct Kv4Plan {
  bool tokens = false;  // waves split tokens, else columns
  int tiles = 0;        // per (sequence, kv head)
  int splits = 1;
  int split_tokens = 0;
  bool longest_first = false;
};

// Depends only on the arguments, so that the workspace size agrees with the launch.
Kv4Plan kv4_plan(int batch, int total_rows, int max_rows, int max_ctx, int hkv, int group, int head_dim) {
  Kv4Plan p;
  const int64_t cols = (int64_t)std::min(max_rows, total_rows) * group;
  const int64_t pairs = (int64_t)batch * hkv;
  const int64_t units = pairs * ceil_div(cols, kTokCols);
  p.tokens = units <= kMaxArrivals && (cols <= 2 * kTokCols || (cols <= kTokMostCols && units <= kTokSlots));
  if (p.tokens) {
    p.tiles = (int)ceil_div(cols, kTokCols);
    // a stage for each of 4 waves
    const int round = head_dim == 64 ? 256 : 128;
    const int64_t fill = units * max_ctx / kTokSlots;
    int64_t st = std::min<int64_t>(std::max<int64_t>(fill, kTokMinSplit), kTokMaxSplit);
    st = std::max({st, fill / kTokRounds, ceil_div(max_ctx, kTokMaxSplits)});
    p.split_tokens = (int)(ceil_div(st, round) * round);
    p.longest_first = p.tiles == 1 && batch <= 64 && units * ceil_div(max_ctx, p.split_tokens) > kTokSlots;
  } else {
    p.tiles = (int)ceil_div(cols, head_dim == 64 ? kColsOf64 : kColsOf128);
    const int64_t wgs = pairs * p.tiles;
    const int64_t want = std::min<int64_t>(std::max<int64_t>((head_dim == 64 ? 2 : 1) * kCUs / wgs, 1), kColsMaxSplits);
    const int64_t least = head_dim == 64 ? kColsMinSplit64 : kColsMinSplit128;
    // whole tiles of 64 tokens
    p.split_tokens = (int)(ceil_div(std::max(ceil_div(max_ctx, want), least), 64) * 64);
  }
  p.splits = (int)ceil_div(max_ctx, p.split_tokens);
  return p;
}

// Workspace: [arrivals: int32 x kMaxArrivals, zero between launches][(m, l)][o].  The counters come
// first at a fixed size, so that calls of other sizes never find partials in their place.
int64_t kv4_partials(const Kv4Plan& p, int batch, int total_rows, int hkv, int group) {
  return p.tokens ? (int64_t)batch * hkv * p.tiles * p.splits * kTokCols : (int64_t)p.splits * total_rows * hkv * group;
}
size_t kv4_workspace_bytes(const Kv4Plan& p, int batch, int total_rows, int hkv, int group, int head_dim) {
  if (p.splits <= 1) return 0;
  const int64_t n = kv4_partials(p, batch, total_rows, hkv, group);
  return (size_t)(kMaxArrivals * 4 + align256(n * 8) + n * head_dim * 4);
}

}  // namespace

namespace luc_internal {
std::vector<std::string> kv4_kernel_names() {
  std::vector<std::string> names = {"luc_block_extend", "luc_block_truncate"};
  for (const char* dt : {"bf16", "f16"})
    for (const char* d : {"_d64", "_d128"})
      for (const char* kind : {"luc_norm_append_", "luc_norm_append4_", "luc_kv4_tokens_", "luc_kv4_columns_",
                               "luc_kv4_merge_"})
        names.push_back(std::string(kind) + dt + d);
  return names;
}
}  // namespace luc_internal

extern "C" {

int luc_block_extend(luc_ctx* ctx, void* stream, int batch, const int32_t* new_tokens, int32_t* lens,
                     int32_t* block_tables, int table_stride, int32_t* free_list, int32_t* state,
                     int num_blocks, int rows, int64_t* slots, int32_t* positions, int32_t* cu_seqlens,
                     int32_t* start_pos) {
  MapArgs a{new_tokens, lens,  block_tables, table_stride, free_list, state,      slots,
            positions,  cu_seqlens, start_pos, batch,      num_blocks, rows};
  if (int rc = check_map(ctx, a, table_stride)) return rc;
  if (rows < 0) return fail(LUC_E_INVALID, "rows %d < 0", rows);
  if ((batch && (!cu_seqlens || !start_pos)) || (rows && (!slots || !positions)))
    return fail(LUC_E_INVALID, "null slots, positions, cu_seqlens or start_pos");
  if (!aligned(slots, 8)) return fail(LUC_E_INVALID, "slots must be 8-byte aligned");
  if (batch == 0) return LUC_OK;
  if (int rc = check_device(ctx)) return rc;
  hipFunction_t fn;
  if (int rc = get_fn(ctx, "luc_block_extend", &fn)) return rc;
  const int64_t grid = std::min<int64_t>(std::max<int64_t>(ceil_div(rows, 2048), 1), 64);
  void* args[] = {&a};
  return launch(fn, dim3((unsigned)grid), dim3(1024), stream, args);
}

int luc_block_truncate(luc_ctx* ctx, void* stream, int batch, const int32_t* keep, int32_t* lens,
                       int32_t* block_tables, int table_stride, int32_t* free_list, int32_t* state,
                       int num_blocks) {
  MapArgs a{keep, lens, block_tables, table_stride, free_list, state, nullptr, nullptr, nullptr, nullptr, batch,
            num_blocks, 0};
  if (int rc = check_map(ctx, a, table_stride)) return rc;
  if (batch == 0) return LUC_OK;
  if (int rc = check_device(ctx)) return rc;
  hipFunction_t fn;
  if (int rc = get_fn(ctx, "luc_block_truncate", &fn)) return rc;
  const int64_t most = std::min<int64_t>((int64_t)batch * table_stride, num_blocks);
  const int64_t grid = std::min<int64_t>(std::max<int64_t>(ceil_div(most, 4096), 1), 16);
  void* args[] = {&a};
  return launch(fn, dim3((unsigned)grid), dim3(1024), stream, args);
}

int luc_qk_norm_rope_append(luc_ctx* ctx, void* stream, int dtype, const void* q, const void* k, const void* v,
                            int64_t row_stride, const void* q_bias, const void* k_bias, const void* v_bias,
                            const void* q_norm, const void* k_norm, float eps, const float* cos_table,
                            const float* sin_table, int max_pos, const int32_t* positions, const int64_t* slots,
                            int num_tokens, void* q_out, int64_t q_out_stride, void* k_out, int64_t k_out_stride,
                            void* k_pool, void* v_pool, int num_blocks, int layer, int num_layers,
                            int num_q_heads, int num_kv_heads, int head_dim, int block_size) {
  NormAppendArgs a{q, k, v, row_stride, q_bias, k_bias, v_bias, q_norm, k_norm, cos_table, sin_table, positions,
                   slots, q_out, q_out_stride, k_out, nullptr, k_out_stride, k_pool, v_pool, 0, eps, num_tokens,
                   max_pos, layer, num_layers, num_q_heads, num_kv_heads};
  return norm_append(ctx, stream, dtype, "luc_norm_append_", a, num_blocks, head_dim, block_size);
}

size_t luc_kv4_page_bytes(int head_dim) {
  return head_dim == 64 || head_dim == 128 ? (size_t)LUC_BLOCK_SIZE * (head_dim / 2 + head_dim / kGroup4 * 4) : 0;
}

int luc_kv4_append(luc_ctx* ctx, void* stream, int dtype, const void* q, const void* k, const void* v,
                   int64_t row_stride, const void* q_bias, const void* k_bias, const void* v_bias,
                   const void* q_norm, const void* k_norm, float eps, const float* cos_table,
                   const float* sin_table, int max_pos, const int32_t* positions, const int64_t* slots,
                   int num_tokens, void* q_out, int64_t q_out_stride, void* k_out, void* v_out,
                   int64_t kv_out_stride, void* k_pool, void* v_pool, int num_blocks, int layer, int num_layers,
                   int num_q_heads, int num_kv_heads, int head_dim, int block_size) {
  NormAppendArgs a{q, k, v, row_stride, q_bias, k_bias, v_bias, q_norm, k_norm, cos_table, sin_table, positions,
                   slots, q_out, q_out_stride, k_out, v_out, kv_out_stride, k_pool, v_pool, 0, eps, num_tokens,
                   max_pos, layer, num_layers, num_q_heads, num_kv_heads};
  return norm_append(ctx, stream, dtype, "luc_norm_append4_", a, num_blocks, head_dim, block_size);
}

size_t luc_kv4_workspace_size(int batch, int total_rows, int max_rows, int max_ctx, int num_q_heads,
                              int num_kv_heads, int head_dim) {
  if (batch <= 0 || total_rows <= 0 || max_rows <= 0 || max_ctx <= 0 || max_ctx > kMaxCtx || num_q_heads <= 0 ||
      num_kv_heads <= 0 || num_q_heads > kMaxHeads || num_q_heads % num_kv_heads ||
      num_q_heads / num_kv_heads > 8 || (int64_t)total_rows * num_q_heads > INT32_MAX ||
      (head_dim != 64 && head_dim != 128))
    return 0;
  const int group = num_q_heads / num_kv_heads;
  return kv4_workspace_bytes(kv4_plan(batch, total_rows, max_rows, max_ctx, num_kv_heads, group, head_dim), batch,
                             total_rows, num_kv_heads, group, head_dim);
}

int luc_kv4_attention(luc_ctx* ctx, void* stream, int dtype, void* out, int64_t out_row_stride, const void* q,
                      int64_t q_row_stride, const void* k_pool, const void* v_pool, const int32_t* block_tables,
                      int table_stride, int num_blocks, const int32_t* cu_seqlens, const int32_t* start_pos,
                      int batch, int total_rows, int max_rows, int max_ctx, int layer, int num_layers,
                      int num_q_heads, int num_kv_heads, int head_dim, int block_size, float sm_scale,
                      void* workspace, size_t workspace_bytes) {
  if (int rc = check_sizes(ctx, dtype, num_q_heads, num_kv_heads, head_dim, block_size, layer, num_layers, num_blocks))
    return rc;
  if (batch < 0 || total_rows < 0) return fail(LUC_E_INVALID, "batch %d / total_rows %d < 0", batch, total_rows);
  if (!cu_seqlens && total_rows != batch)
    return fail(LUC_E_INVALID, "no cu_seqlens: one row a sequence, not %d for %d", total_rows, batch);
  if (max_ctx <= 0 || max_ctx > kMaxCtx) return fail(LUC_E_INVALID, "max_ctx %d outside [1, %d]", max_ctx, kMaxCtx);
  if ((total_rows && (!out || !q)) || !k_pool || !v_pool || (batch && (!block_tables || !start_pos)))
    return fail(LUC_E_INVALID, "null out, q, pool, block table or start_pos");
  const int row = num_q_heads * head_dim;
  if (q_row_stride < row || out_row_stride < row)
    return fail(LUC_E_INVALID, "q/out row stride smaller than a row (%d)", row);
  if (!aligned(q, 16) || q_row_stride % 8 || !aligned(out, 8) || out_row_stride % 4)
    return fail(LUC_E_INVALID, "q must be 16-byte aligned with a row stride that is a multiple of 8, out 8-byte and 4");
  if (!aligned(k_pool, 16) || !aligned(v_pool, 16)) return fail(LUC_E_INVALID, "KV pools must be 16-byte aligned");
  if (table_stride <= 0 || (int64_t)table_stride * LUC_BLOCK_SIZE < max_ctx)
    return fail(LUC_E_INVALID, "table_stride %d pages cannot hold max_ctx %d", table_stride, max_ctx);
  if (batch == 0 || total_rows == 0) return LUC_OK;
  if (max_rows < 1) return fail(LUC_E_INVALID, "max_rows %d < 1", max_rows);
  if ((int64_t)total_rows * num_q_heads > INT32_MAX)
    return fail(LUC_E_INVALID, "total_rows x num_q_heads too large");
  const int group = num_q_heads / num_kv_heads;
  const Kv4Plan plan = kv4_plan(batch, total_rows, max_rows, max_ctx, num_kv_heads, group, head_dim);
  const size_t need = kv4_workspace_bytes(plan, batch, total_rows, num_kv_heads, group, head_dim);
  if (need && (!workspace || workspace_bytes < need))
    return fail(LUC_E_WORKSPACE, "workspace %zu bytes, %zu needed", workspace_bytes, need);
  if (need && !aligned(workspace, 256)) return fail(LUC_E_INVALID, "workspace must be 256-byte aligned");
  const int64_t units = (int64_t)batch * num_kv_heads * plan.tiles;
  if ((int64_t)num_layers * num_kv_heads * 10 * head_dim > UINT32_MAX)
    return fail(LUC_E_INVALID, "num_layers x num_kv_heads too large");
  const int64_t threads = !plan.tokens && head_dim == 128 ? 512 : 256;
  const int64_t items = (int64_t)total_rows * num_q_heads;  // of the merge, head_dim / 4 threads each
  if (units * plan.splits * threads > UINT32_MAX || (!plan.tokens && plan.splits > 1 && items * (head_dim / 4) > UINT32_MAX))
    return fail(LUC_E_INVALID, "batch x kv heads x rows too large");
  if (int rc = check_device(ctx)) return rc;
  Kv4AttnArgs a{q, q_row_stride, out, out_row_stride, k_pool, v_pool, block_tables, table_stride, cu_seqlens,
                start_pos, nullptr, nullptr, nullptr, batch, total_rows, max_rows, max_ctx, layer, num_layers,
                num_kv_heads, group, num_blocks, plan.tiles, plan.splits, plan.split_tokens,
                plan.longest_first, sm_scale * 1.4426950408889634f};
  if (need) {
    char* ws = static_cast<char*>(workspace);
    a.ws_cnt = reinterpret_cast<int32_t*>(ws);
    a.ws_ml = reinterpret_cast<float*>(ws + kMaxArrivals * 4);
    a.ws_o = reinterpret_cast<float*>(
        ws + kMaxArrivals * 4 + align256(kv4_partials(plan, batch, total_rows, num_kv_heads, group) * 8));
  }
  const std::string suffix = std::string(dt_name(dtype)) + "_d" + std::to_string(head_dim);
  hipFunction_t fn, merge;
  if (int rc = get_fn(ctx, (plan.tokens ? "luc_kv4_tokens_" : "luc_kv4_columns_") + suffix, &fn)) return rc;
  if (int rc = get_fn(ctx, "luc_kv4_merge_" + suffix, &merge)) return rc;
  void* args[] = {&a};
  if (int rc = launch(fn, dim3((unsigned)(units * plan.splits)), dim3((unsigned)threads), stream, args)) return rc;
  if (plan.tokens || plan.splits == 1) return LUC_OK;
  return launch(merge, dim3((unsigned)ceil_div(items, 1024 / head_dim)), dim3(256), stream, args);
}

}  // extern "C"
