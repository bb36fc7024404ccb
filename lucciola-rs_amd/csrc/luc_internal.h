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
// Names of the kernels that luc_kv4.cpp launches, for luc_init to resolve.
std::vector<std::string> kv4_kernel_names();

inline bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }
inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
}  // namespace luc_internal
