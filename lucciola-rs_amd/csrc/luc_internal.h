// luc_internal.h -- what the translation units of liblucattn.so share: the
// context, error reporting and the launch helpers of luc_attn.cpp.
#pragma once
#include "luc_attn.h"

#include <hip/hip_runtime_api.h>

#include <cstdint>
#include <string>
#include <unordered_map>
#include <vector>

struct luc_ctx {
  int device = 0;
  int num_cus = 0;
  void* scratch = nullptr;  // this device's copy of the library scratch (luc_scratch.hip)
  std::vector<hipModule_t> modules;
  std::unordered_map<std::string, hipFunction_t> fns;
  std::vector<hipFunction_t> kv8;  // of kv8_kernel_names(), in its order
};

namespace luc_internal {
int scratch_setup(int device, void** out);
// Sets the thread's error message and returns `code`.
int fail(int code, const char* fmt, ...);
// A kernel that luc_init has resolved.
int get_fn(const luc_ctx* ctx, const std::string& name, hipFunction_t* fn);
// LUC_E_INVALID unless the context's device is the current one.
int check_device(const luc_ctx* ctx);
int launch(hipFunction_t fn, dim3 grid, dim3 block, void* stream, void** args);
// Names of the kernels that luc_kv4.cpp and luc_kv8.cpp launch, for luc_init to resolve.
std::vector<std::string> kv4_kernel_names();
std::vector<std::string> kv8_kernel_names();

inline bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }
inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline int64_t align256(int64_t n) { return ceil_div(n, 256) * 256; }
inline const char* dt_name(int dtype) { return dtype == LUC_F16 ? "f16" : "bf16"; }

// ---- what the appends and attention over quantised caches share (luc_kv4.cpp)
constexpr int kMaxHeads = 1 << 20;  // rows of heads stay within 32 bits
constexpr int kMaxCtx = 1 << 30;

// luc::NormAppendArgs of append_row.h: the same fields in the same order.
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
                int num_layers, int num_blocks);
// The arguments of an append; sets a.num_slots.
int check_append(const luc_ctx* ctx, int dtype, NormAppendArgs& a, int num_blocks, int head_dim, int block_size);
}  // namespace luc_internal
