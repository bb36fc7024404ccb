// luc_kv8.cpp -- host side of the 8-bit cache (include/luc_attn.h, "The 8-bit cache"): argument checks, work
// splits and launches of kv8_append.hip, kv8_attention.hip and kv8_select.hip.  Nothing here allocates
// device memory or synchronises.
#include "luc_internal.h"

#include <algorithm>
#include <cmath>

using namespace luc_internal;

namespace {

// luc::Kv8AppendArgs of kv8_append.hip: the same fields in the same order.
struct Kv8AppendArgs : NormAppendArgs {
  float* scales;
  void* bounds;
  uint32_t every;
};

// luc::Kv8ReadArgs of kv8_append.hip: the same fields in the same order.
struct Kv8ReadArgs {
  void* k_out;
  void* v_out;
  int64_t out_stride;
  const int64_t* slots;
  const void* k_pool;
  const void* v_pool;
  const float* scales;
  int64_t num_slots;
  int32_t rows, layer, num_layers, hkv;
};

// luc::Kv8AttnArgs of kv8_attention.hip: the same fields in the same order.
struct Kv8AttnArgs {
  const void* q;
  int64_t q_stride;
  void* out;
  int64_t out_stride;
  const void* k_pool;
  const void* v_pool;
  const float* scales;
  const int32_t* tables;
  int64_t table_stride;
  const int32_t* cu_seqlens;
  const int32_t* start_pos;
  const int32_t* chosen;
  int32_t* ws_cnt;
  float* ws_ml;
  float* ws_o;
  int32_t batch, total_rows, max_rows, max_ctx, layer, num_layers, hkv, group, num_blocks, budget;
  int32_t tiles, splits, split_tokens, longest_first;
  float qk_scale_log2;
};

// luc::Kv8SelectArgs of kv8_select.hip: the same fields in the same order.
struct Kv8SelectArgs {
  const void* q;
  int64_t q_stride;
  const void* bounds;
  const float* scales;
  const int32_t* tables;
  int64_t table_stride;
  const int32_t* cu_seqlens;
  const int32_t* start_pos;
  int32_t* pages;
  int32_t* ws_cnt;
  uint32_t* ws_key;
  int32_t batch, total_rows, max_rows, max_ctx, layer, num_layers, hkv, group, num_blocks;
  int32_t budget, first, recent, chunks, max_pages, tiles;
};

constexpr int kCUs = 256;
// Rows up to which a wave of an append has the runs of one row and the slots of all in registers, and beyond which it has those of
// 16.  28 + 2 x 4 heads of 128, us by either: a prompt of 256 rows 6.3 and 6.4, of 512 7.0 and 6.5; 512 single rows 7.4
// and 49, one run after the other.
constexpr int kAppendManyRows = 512;  // kManyRows of kv8_append.hip
constexpr int kTokCols = 8;          // columns of a workgroup
constexpr int kTokMaxSplits = 256;   // kv_split.h
// Workgroups that a launch is planned for: one a CU.  Short splits of a launch planned for two cost more by their merge than
// they gain: of 4 kv heads of 128, 64 contexts of 1536 18.1 us and 21.2, 8 of 4096 11.2 and 13.3; of 2 of 64, 64 mixed ones up
// to 4096 12.9 and 12.1, 128 of 2048 11.8 and 14.0; long ones alike.
constexpr int kTokSlots = kCUs;
constexpr int kTokAtOnce = 2 * kCUs;  // more of them go longest first (512 of one length each: 17.3 us, 20.3 so)
// Split lengths of a tokens launch: what fills the chip once, but not longer than lets mixed contexts end together (64
// contexts of 8192, 7 heads of 64 a group: 24.3 us, 28.1 of splits to 1024; 128 mixed up to 8192, 7 of 128: 107.8,
// 111.8 to 1024, 111.5 to 4096), nor shorter than is worth a merge.  A workgroup takes 0.0048 us a token, a
// merge 0.13 us a split, so a single context is quickest in splits of sqrt(26 ctx): of 32768 tokens 11.0 us, 16.0 in splits of
// 256; of 8192 9.9, 10.7 in 256, 11.4 in 1024; of 2048 8.1, 9.0 in 512.  Up to 512 tokens a second split costs more
// than it saves: 6.3 us, 7.8 in two.
constexpr int kTokOneSplit = 512, kTokMaxSplit = 2048, kTokSplitRate = 26;
// Beyond so many rounds of workgroups splits grow again: any contexts balance (200 mixed contexts up to 8192, 8 kv heads of
// 128: 288 us, 290 without; 4 and 16 lie between).
constexpr int kTokRounds = 8;
// Up to 16 columns go to the tokens kernel, which reads the cache once for each 8, and more of them while it reads at
// most this: 5.4 TB/s from the L2 of an XCD, or 5.6 ns a workgroup, as many bytes as kTokLeastBytes, where contexts are
// short.  The columns kernel reads the cache once, and takes 6 to 10 us more to begin.  28 / 4 heads of 128, us by tokens
// and by columns: 64 rows of a context of 64 5.3 and 12.5, 256 of 256 11.2 and 18.1, 64 of 2048 (112 MiB) 17.9
// and 22.0, 3 of each of 16 x 4096 (192 MiB) 36 and 30.7, 8 sequences of 64 rows (168) 14.4 and 13.0, 32 of 16 13.8 and 9.9.
constexpr int64_t kTokMostBytes = 128 << 20, kTokLeastBytes = 96 << 10;
// Columns of a workgroup of the columns kernel (Kv8Cols).
constexpr int kColsOf64 = 128, kColsOf128 = 256;
// Its splits fill the chip once, planned as a workgroup a CU (128) or two (64, whose registers hold three), but
// are not shorter than pays for their partials: of 64, 200 rows at the end of each of 4 x 1024 tokens 19.4 us, 21.0
// in splits of 256 and of 1024; of 128, 512 rows on 4096 47.7, 48.6 in 512.  No more than 32: 128 rows on 16384
// 46.5, 69.5 with 8, 46.5 with 128.
constexpr int kColsMinSplit64 = 512, kColsMinSplit128 = 256, kColsMaxSplits = 32;
constexpr int64_t kMaxArrivals = 1 << 16;  // (sequence, kv head, column tile)
constexpr int kSelPages = 4 * 16;          // pages of a workgroup's waves at once (kv8_select.hip)
// Workgroups of a selection before they take more pages each, up to 16 times kSelPages.  64 contexts of 1024 to 16384
// tokens, 4 kv heads of 128, selection and attention over 96 pages: 39.1 us; planned for 256 42.6, for 1024 39.0, but 8 of
// 65536 then take 21.8 instead of 19.5 to choose from.
constexpr int kSelWorkgroups = 2 * kCUs;

struct Kv8Plan {
  bool tokens = false;  // waves split tokens, else columns
  int tiles = 0;        // per (sequence, kv head)
  int splits = 1;
  int split_tokens = 0;
  bool longest_first = false;
};

// Depends only on the arguments, so that the workspace size agrees with the launch.
Kv8Plan kv8_plan(int batch, int total_rows, int max_rows, int max_ctx, int hkv, int group, int head_dim) {
  Kv8Plan p;
  const int64_t cols = (int64_t)std::min(max_rows, total_rows) * group;
  const int64_t pairs = (int64_t)batch * hkv;
  const int64_t units = pairs * ceil_div(cols, kTokCols);
  p.tokens = units <= kMaxArrivals && (cols <= 2 * kTokCols || units * std::max((int64_t)max_ctx * 2 * head_dim, kTokLeastBytes) <= kTokMostBytes);
  if (p.tokens) {
    p.tiles = (int)ceil_div(cols, kTokCols);
    // a stage for each of 4 waves
    const int round = head_dim == 64 ? 256 : 128;
    const int64_t fill = units * max_ctx / kTokSlots;
    int64_t st = max_ctx <= kTokOneSplit ? kTokOneSplit : (int64_t)std::sqrt((double)kTokSplitRate * max_ctx);
    st = std::min<int64_t>(std::max(fill, st), kTokMaxSplit);
    st = std::max({st, fill / kTokRounds, ceil_div(max_ctx, kTokMaxSplits)});
    st = std::min<int64_t>(st, max_ctx);  // (the rounds of the largest calls ask for more than 32 bits)
    p.split_tokens = (int)(ceil_div(st, round) * round);
    p.longest_first = p.tiles == 1 && batch <= 64 && units * ceil_div(max_ctx, p.split_tokens) > kTokAtOnce;
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

// Workspace: [arrivals: int32 x kMaxArrivals, zero between launches][(m, l)][o], or [arrivals][keys].  The
// counters come first at a fixed size, so that calls of other sizes never find partials in their place.
int64_t kv8_partials(const Kv8Plan& p, int batch, int total_rows, int hkv, int group) {
  return p.tokens ? (int64_t)batch * hkv * p.tiles * p.splits * kTokCols : (int64_t)p.splits * total_rows * hkv * group;
}
size_t kv8_workspace_bytes(const Kv8Plan& p, int batch, int total_rows, int hkv, int group, int head_dim) {
  if (p.splits <= 1) return 0;
  const int64_t n = kv8_partials(p, batch, total_rows, hkv, group);
  return (size_t)(kMaxArrivals * 4 + align256(n * 8) + n * head_dim * 4);
}
// Of a selection: scores are needed where a context may have more pages than the budget.
size_t select_workspace_bytes(int batch, int max_ctx, int budget, int hkv) {
  const int64_t pages = ceil_div(max_ctx, LUC_BLOCK_SIZE);
  return pages <= budget ? 0 : (size_t)(kMaxArrivals * 4 + (int64_t)batch * hkv * ceil_div(pages, 4) * 16);
}
// Positions among the chosen pages' tokens.
int chosen_ctx(int max_ctx, int budget) { return (int)std::min<int64_t>(max_ctx, (int64_t)budget * LUC_BLOCK_SIZE); }

// The kernels of a type and head dimension, in this order.
enum Kernel { kAppend, kAppendMany, kRead, kTokens, kChosen, kColumns, kMerge, kSelect, kKernels };
constexpr const char* kKernelNames[kKernels] = {"append", "append_many", "read", "tokens", "chosen", "columns", "merge", "select"};
// (by place: looking up their names would be a tenth of a launch)
hipFunction_t kernel(const luc_ctx* ctx, Kernel k, int dtype, int head_dim) {
  return ctx->kv8[((dtype == LUC_F16) * 2 + (head_dim == 128)) * kKernels + k];
}

bool sizes_fit(int hq, int hkv, int head_dim) {
  return hq > 0 && hkv > 0 && hq <= kMaxHeads && hq % hkv == 0 && hq / hkv <= 8 && (head_dim == 64 || head_dim == 128);
}

int check_pools(const void* k_pool, const void* v_pool, const void* scales, int num_layers, int hkv, int head_dim) {
  if (!k_pool || !v_pool || !scales) return fail(LUC_E_INVALID, "null pool or scales");
  if (!aligned(k_pool, 16) || !aligned(v_pool, 16) || !aligned(scales, 8))
    return fail(LUC_E_INVALID, "KV pools must be 16-byte aligned, scales 8-byte");
  if ((int64_t)num_layers * hkv * 16 * head_dim > UINT32_MAX)
    return fail(LUC_E_INVALID, "num_layers x num_kv_heads too large");
  return LUC_OK;
}

// What attention and selection check of a batch's rows.
int check_rows(const void* q, int64_t q_row_stride, const int32_t* block_tables, int table_stride,
               const int32_t* cu_seqlens, const int32_t* start_pos, int batch, int total_rows, int max_ctx, int hq,
               int head_dim) {
  if (batch < 0 || total_rows < 0) return fail(LUC_E_INVALID, "batch %d / total_rows %d < 0", batch, total_rows);
  if (!cu_seqlens && total_rows != batch)
    return fail(LUC_E_INVALID, "no cu_seqlens: one row a sequence, not %d for %d", total_rows, batch);
  if (max_ctx <= 0 || max_ctx > kMaxCtx) return fail(LUC_E_INVALID, "max_ctx %d outside [1, %d]", max_ctx, kMaxCtx);
  if ((total_rows && !q) || (batch && (!block_tables || !start_pos)))
    return fail(LUC_E_INVALID, "null q, block table or start_pos");
  const int64_t row = (int64_t)hq * head_dim;
  if (q_row_stride < row) return fail(LUC_E_INVALID, "q row stride smaller than a row (%lld)", (long long)row);
  if (!aligned(q, 16) || q_row_stride % 8)
    return fail(LUC_E_INVALID, "q must be 16-byte aligned with a row stride that is a multiple of 8");
  if (table_stride <= 0 || (int64_t)table_stride * LUC_BLOCK_SIZE < max_ctx)
    return fail(LUC_E_INVALID, "table_stride %d pages cannot hold max_ctx %d", table_stride, max_ctx);
  if ((int64_t)total_rows * hq > INT32_MAX) return fail(LUC_E_INVALID, "total_rows x num_q_heads too large");
  return LUC_OK;
}
int check_out(const void* out, int64_t out_row_stride, int total_rows, int hq, int head_dim) {
  if (total_rows && !out) return fail(LUC_E_INVALID, "null out");
  const int64_t row = (int64_t)hq * head_dim;
  if (out_row_stride < row) return fail(LUC_E_INVALID, "out row stride smaller than a row (%lld)", (long long)row);
  if (!aligned(out, 8) || out_row_stride % 4)
    return fail(LUC_E_INVALID, "out must be 8-byte aligned with a row stride that is a multiple of 4");
  return LUC_OK;
}
int check_workspace(const void* workspace, size_t bytes, size_t need) {
  if (need && (!workspace || bytes < need)) return fail(LUC_E_WORKSPACE, "workspace %zu bytes, %zu needed", bytes, need);
  if (need && !aligned(workspace, 256)) return fail(LUC_E_INVALID, "workspace must be 256-byte aligned");
  return LUC_OK;
}

// a: everything but the workspace's parts and the plan's fields.
int attend(luc_ctx* ctx, void* stream, int dtype, int head_dim, const Kv8Plan& plan, Kv8AttnArgs& a, void* workspace,
           size_t workspace_bytes) {
  const size_t need = kv8_workspace_bytes(plan, a.batch, a.total_rows, a.hkv, a.group, head_dim);
  if (int rc = check_workspace(workspace, workspace_bytes, need)) return rc;
  const int64_t units = (int64_t)a.batch * a.hkv * plan.tiles;
  const int64_t threads = !plan.tokens && head_dim == 128 ? 512 : 256;
  const int64_t items = (int64_t)a.total_rows * a.hkv * a.group;  // of the merge, head_dim / 4 threads each
  if (units > UINT32_MAX / (plan.splits * threads) || (!plan.tokens && plan.splits > 1 && items * (head_dim / 4) > UINT32_MAX))
    return fail(LUC_E_INVALID, "batch x kv heads x rows too large");
  if (int rc = check_device(ctx)) return rc;
  a.tiles = plan.tiles;
  a.splits = plan.splits;
  a.split_tokens = plan.split_tokens;
  a.longest_first = plan.longest_first;
  if (need) {
    char* ws = static_cast<char*>(workspace);
    a.ws_cnt = reinterpret_cast<int32_t*>(ws);
    a.ws_ml = reinterpret_cast<float*>(ws + kMaxArrivals * 4);
    a.ws_o = reinterpret_cast<float*>(
        ws + kMaxArrivals * 4 + align256(kv8_partials(plan, a.batch, a.total_rows, a.hkv, a.group) * 8));
  }
  const hipFunction_t fn = kernel(ctx, a.chosen ? kChosen : plan.tokens ? kTokens : kColumns, dtype, head_dim);
  void* args[] = {&a};
  if (int rc = launch(fn, dim3((unsigned)(units * plan.splits)), dim3((unsigned)threads), stream, args)) return rc;
  if (plan.tokens || plan.splits == 1) return LUC_OK;
  return launch(kernel(ctx, kMerge, dtype, head_dim), dim3((unsigned)ceil_div(items, 1024 / head_dim)), dim3(256), stream, args);
}

constexpr float kLog2e = 1.4426950408889634f;

}  // namespace

namespace luc_internal {
std::vector<std::string> kv8_kernel_names() {
  std::vector<std::string> names;
  for (const char* dt : {"bf16", "f16"})
    for (const char* d : {"_d64", "_d128"})
      for (const char* kind : kKernelNames) names.push_back(std::string("luc_kv8_") + kind + "_" + dt + d);
  return names;
}
}  // namespace luc_internal

extern "C" {

int luc_kv8_append(luc_ctx* ctx, void* stream, int dtype, const void* q, const void* k, const void* v,
                   int64_t row_stride, const void* q_bias, const void* k_bias, const void* v_bias,
                   const void* q_norm, const void* k_norm, float eps, const float* cos_table,
                   const float* sin_table, int max_pos, const int32_t* positions, const int64_t* slots,
                   int num_tokens, void* q_out, int64_t q_out_stride, void* k_pool, void* v_pool, float* scales,
                   void* bounds, int num_blocks, int layer, int num_layers, int num_q_heads, int num_kv_heads,
                   int head_dim, int block_size) {
  Kv8AppendArgs a{{q, k, v, row_stride, q_bias, k_bias, v_bias, q_norm, k_norm, cos_table, sin_table, positions,
                   slots, q_out, q_out_stride, nullptr, nullptr, 0, k_pool, v_pool, 0, eps, num_tokens, max_pos,
                   layer, num_layers, num_q_heads, num_kv_heads},
                  scales, bounds, 1};
  if (int rc = check_append(ctx, dtype, a, num_blocks, head_dim, block_size)) return rc;
  if (int rc = check_pools(k_pool, v_pool, scales, num_layers, num_kv_heads, head_dim)) return rc;
  if (!aligned(bounds, 16)) return fail(LUC_E_INVALID, "bounds must be 16-byte aligned");
  if (num_tokens == 0) return LUC_OK;
  // q: head_dim / 16 lanes a head; a wave for every row, or 16, of every k and v head
  const bool many = num_tokens > kAppendManyRows;
  const int64_t runs = ceil_div(ceil_div(num_tokens, many ? 16 : 1) * num_kv_heads * 2, 4);
  const int64_t grid = ceil_div((int64_t)num_tokens * num_q_heads, 4096 / head_dim) + runs;
  // the blocks of runs evenly among q's, an odd number apart (block x runs on XCD x % 8), and all of them in the first half:
  // they take longest
  a.every = (uint32_t)std::min<int64_t>((grid / runs / 2) | 1, 1 << 30);
  if (grid * 256 > UINT32_MAX) return fail(LUC_E_INVALID, "too many rows for one launch");
  if (int rc = check_device(ctx)) return rc;
  const hipFunction_t fn = kernel(ctx, many ? kAppendMany : kAppend, dtype, head_dim);
  void* args[] = {&a};
  return launch(fn, dim3((unsigned)grid), dim3(256), stream, args);
}

int luc_kv8_read(luc_ctx* ctx, void* stream, int dtype, void* k_out, void* v_out, int64_t out_row_stride,
                 const int64_t* slots, int num_tokens, const void* k_pool, const void* v_pool, const float* scales,
                 int num_blocks, int layer, int num_layers, int num_kv_heads, int head_dim, int block_size) {
  if (int rc = check_sizes(ctx, dtype, num_kv_heads, num_kv_heads, head_dim, block_size, layer, num_layers, num_blocks))
    return rc;
  if (num_tokens < 0) return fail(LUC_E_INVALID, "num_tokens %d < 0", num_tokens);
  if (int rc = check_pools(k_pool, v_pool, scales, num_layers, num_kv_heads, head_dim)) return rc;
  if (num_tokens && (!k_out || !v_out || !slots)) return fail(LUC_E_INVALID, "null k_out, v_out or slots");
  if (out_row_stride < (int64_t)num_kv_heads * head_dim || out_row_stride % 8)
    return fail(LUC_E_INVALID, "row stride smaller than a row (%d), or not a multiple of 8", num_kv_heads * head_dim);
  if (!aligned(k_out, 16) || !aligned(v_out, 16) || !aligned(slots, 8))
    return fail(LUC_E_INVALID, "k_out and v_out must be 16-byte aligned, slots 8-byte");
  if (num_tokens == 0) return LUC_OK;
  const int64_t threads = (int64_t)num_tokens * num_kv_heads * (head_dim / 8) * 2;
  if (threads + 256 > UINT32_MAX) return fail(LUC_E_INVALID, "too many rows for one launch");
  if (int rc = check_device(ctx)) return rc;
  const hipFunction_t fn = kernel(ctx, kRead, dtype, head_dim);
  Kv8ReadArgs a{k_out, v_out, out_row_stride, slots, k_pool, v_pool, scales, (int64_t)num_blocks * LUC_BLOCK_SIZE,
                num_tokens, layer, num_layers, num_kv_heads};
  void* args[] = {&a};
  return launch(fn, dim3((unsigned)ceil_div(threads, 256)), dim3(256), stream, args);
}

size_t luc_kv8_workspace_size(int batch, int total_rows, int max_rows, int max_ctx, int num_q_heads,
                              int num_kv_heads, int head_dim) {
  if (batch <= 0 || total_rows <= 0 || max_rows <= 0 || max_ctx <= 0 || max_ctx > kMaxCtx ||
      !sizes_fit(num_q_heads, num_kv_heads, head_dim) || (int64_t)total_rows * num_q_heads > INT32_MAX)
    return 0;
  const int group = num_q_heads / num_kv_heads;
  return kv8_workspace_bytes(kv8_plan(batch, total_rows, max_rows, max_ctx, num_kv_heads, group, head_dim), batch,
                             total_rows, num_kv_heads, group, head_dim);
}

int luc_kv8_attention(luc_ctx* ctx, void* stream, int dtype, void* out, int64_t out_row_stride, const void* q,
                      int64_t q_row_stride, const void* k_pool, const void* v_pool, const float* scales,
                      const int32_t* block_tables, int table_stride, int num_blocks, const int32_t* cu_seqlens,
                      const int32_t* start_pos, int batch, int total_rows, int max_rows, int max_ctx, int layer,
                      int num_layers, int num_q_heads, int num_kv_heads, int head_dim, int block_size, float sm_scale,
                      void* workspace, size_t workspace_bytes) {
  if (int rc = check_sizes(ctx, dtype, num_q_heads, num_kv_heads, head_dim, block_size, layer, num_layers, num_blocks))
    return rc;
  if (int rc = check_rows(q, q_row_stride, block_tables, table_stride, cu_seqlens, start_pos, batch, total_rows, max_ctx,
                          num_q_heads, head_dim))
    return rc;
  if (int rc = check_out(out, out_row_stride, total_rows, num_q_heads, head_dim)) return rc;
  if (int rc = check_pools(k_pool, v_pool, scales, num_layers, num_kv_heads, head_dim)) return rc;
  if (batch == 0 || total_rows == 0) return LUC_OK;
  if (max_rows < 1) return fail(LUC_E_INVALID, "max_rows %d < 1", max_rows);
  const int group = num_q_heads / num_kv_heads;
  const Kv8Plan plan = kv8_plan(batch, total_rows, max_rows, max_ctx, num_kv_heads, group, head_dim);
  Kv8AttnArgs a{q, q_row_stride, out, out_row_stride, k_pool, v_pool, scales, block_tables, table_stride, cu_seqlens,
                start_pos, nullptr, nullptr, nullptr, nullptr, batch, total_rows, max_rows, max_ctx, layer, num_layers,
                num_kv_heads, group, num_blocks, 0, 0, 0, 0, 0, sm_scale * kLog2e};
  return attend(ctx, stream, dtype, head_dim, plan, a, workspace, workspace_bytes);
}

size_t luc_kv8_sparse_workspace_size(int batch, int max_ctx, int budget, int num_q_heads, int num_kv_heads,
                                     int head_dim) {
  if (batch <= 0 || max_ctx <= 0 || max_ctx > kMaxCtx || budget <= 0 || !sizes_fit(num_q_heads, num_kv_heads, head_dim) ||
      (int64_t)batch * num_q_heads > INT32_MAX)
    return 0;
  const int group = num_q_heads / num_kv_heads;
  const Kv8Plan plan = kv8_plan(batch, batch, 1, chosen_ctx(max_ctx, budget), num_kv_heads, group, head_dim);
  return std::max(kv8_workspace_bytes(plan, batch, batch, num_kv_heads, group, head_dim),
                  select_workspace_bytes(batch, max_ctx, budget, num_kv_heads));
}

int luc_kv8_select(luc_ctx* ctx, void* stream, int dtype, int32_t* pages, int budget, int first, int recent,
                   const void* q, int64_t q_row_stride, const void* bounds, const float* scales,
                   const int32_t* block_tables, int table_stride, int num_blocks, const int32_t* cu_seqlens,
                   const int32_t* start_pos, int batch, int total_rows, int max_ctx, int layer, int num_layers,
                   int num_q_heads, int num_kv_heads, int head_dim, int block_size, void* workspace,
                   size_t workspace_bytes) {
  if (int rc = check_sizes(ctx, dtype, num_q_heads, num_kv_heads, head_dim, block_size, layer, num_layers, num_blocks))
    return rc;
  if (int rc = check_rows(q, q_row_stride, block_tables, table_stride, cu_seqlens, start_pos, batch, total_rows, max_ctx,
                          num_q_heads, head_dim))
    return rc;
  if (int rc = check_pools(bounds, bounds, scales, num_layers, num_kv_heads, head_dim)) return rc;
  if (first < 0 || recent < 1 || (int64_t)first + recent > budget)
    return fail(LUC_E_INVALID, "first %d and recent %d (1 or more) of a budget of %d pages", first, recent, budget);
  if ((batch && !pages) || !aligned(pages, 4)) return fail(LUC_E_INVALID, "null or misaligned pages");
  if ((int64_t)batch * num_kv_heads > kMaxArrivals)
    return fail(LUC_E_UNSUPPORTED, "batch x kv heads above %d", (int)kMaxArrivals);
  if (batch == 0) return LUC_OK;
  const size_t need = select_workspace_bytes(batch, max_ctx, budget, num_kv_heads);
  if (int rc = check_workspace(workspace, workspace_bytes, need)) return rc;
  const int max_pages = (int)ceil_div(max_ctx, 4 * LUC_BLOCK_SIZE) * 4;
  int tiles = 1;
  while (tiles < 16 && (int64_t)batch * num_kv_heads * ceil_div(max_pages, kSelPages * tiles) > kSelWorkgroups) tiles *= 2;
  const int64_t chunks = need ? ceil_div(max_pages, kSelPages * tiles) : 1;
  const int64_t grid = ceil_div(batch * chunks, 8) * 8 * num_kv_heads;
  if (grid * 256 > UINT32_MAX) return fail(LUC_E_INVALID, "batch x kv heads x max_ctx too large");
  if (int rc = check_device(ctx)) return rc;
  Kv8SelectArgs a{q, q_row_stride, bounds, scales, block_tables, table_stride, cu_seqlens, start_pos, pages, nullptr,
                  nullptr, batch, total_rows, 1, max_ctx, layer, num_layers, num_kv_heads, num_q_heads / num_kv_heads,
                  num_blocks, budget, first, recent, (int)chunks, max_pages, tiles};
  if (need) {
    a.ws_cnt = static_cast<int32_t*>(workspace);
    a.ws_key = reinterpret_cast<uint32_t*>(static_cast<char*>(workspace) + kMaxArrivals * 4);
  }
  const hipFunction_t fn = kernel(ctx, kSelect, dtype, head_dim);
  void* args[] = {&a};
  return launch(fn, dim3((unsigned)grid), dim3(256), stream, args);
}

int luc_kv8_sparse_attention(luc_ctx* ctx, void* stream, int dtype, void* out, int64_t out_row_stride, const void* q,
                             int64_t q_row_stride, const void* k_pool, const void* v_pool, const float* scales,
                             const int32_t* block_tables, int table_stride, int num_blocks, const int32_t* pages,
                             int budget, const int32_t* cu_seqlens, const int32_t* start_pos, int batch,
                             int total_rows, int max_ctx, int layer, int num_layers, int num_q_heads,
                             int num_kv_heads, int head_dim, int block_size, float sm_scale, void* workspace,
                             size_t workspace_bytes) {
  if (int rc = check_sizes(ctx, dtype, num_q_heads, num_kv_heads, head_dim, block_size, layer, num_layers, num_blocks))
    return rc;
  if (int rc = check_rows(q, q_row_stride, block_tables, table_stride, cu_seqlens, start_pos, batch, total_rows, max_ctx,
                          num_q_heads, head_dim))
    return rc;
  if (int rc = check_out(out, out_row_stride, total_rows, num_q_heads, head_dim)) return rc;
  if (int rc = check_pools(k_pool, v_pool, scales, num_layers, num_kv_heads, head_dim)) return rc;
  if (budget < 1) return fail(LUC_E_INVALID, "budget %d < 1", budget);
  if ((batch && !pages) || !aligned(pages, 4)) return fail(LUC_E_INVALID, "null or misaligned pages");
  if ((int64_t)batch * num_kv_heads > kMaxArrivals)
    return fail(LUC_E_UNSUPPORTED, "batch x kv heads above %d", (int)kMaxArrivals);
  if (batch == 0 || total_rows == 0) return LUC_OK;
  const int group = num_q_heads / num_kv_heads;
  // (the plan is of one row a sequence, whatever total_rows says: as the workspace's size has it)
  const Kv8Plan plan = kv8_plan(batch, batch, 1, chosen_ctx(max_ctx, budget), num_kv_heads, group, head_dim);
  Kv8AttnArgs a{q, q_row_stride, out, out_row_stride, k_pool, v_pool, scales, block_tables, table_stride, cu_seqlens,
                start_pos, pages, nullptr, nullptr, nullptr, batch, total_rows, 1, max_ctx, layer, num_layers,
                num_kv_heads, group, num_blocks, budget, 0, 0, 0, 0, sm_scale * kLog2e};
  return attend(ctx, stream, dtype, head_dim, plan, a, workspace, workspace_bytes);
}

}  // extern "C"
