// fm_ops.hpp -- host side shared by the policy-head operators (fm_norm.hip, fm_sample.hip, fm_distill.hip) and their
// CPU backend (fm_ops_cpu.cpp): argument checks and the error report.
#pragma once
#include <cmath>
#include <cstdint>

#include "../../include/factorysim.h"

namespace fm {
int report(int code, const char* msg) noexcept;  // fm_api.hip: sets fm_last_error's text, returns code

inline int type_size(int t) { return t == FM_DTYPE_F64 || t == FM_DTYPE_I64 ? 8 : t == FM_DTYPE_F32 || t == FM_DTYPE_I32
    ? 4 : 2; }
inline bool is_float_type(int t) { return t == FM_DTYPE_F32 || t == FM_DTYPE_F16 || t == FM_DTYPE_BF16; }
inline bool aligned(const void* p, int bytes) { return ((uintptr_t)p % (uintptr_t)bytes) == 0; }
// rows x cols elements and every row offset stay below 2^60
inline bool fits(int64_t rows, int64_t cols, int64_t stride) {
  const int64_t most = (int64_t)1 << 60;
  return rows <= most / (cols > 0 ? cols : 1) && (stride == 0 || rows <= most / stride);
}
// Every entry point returns through this: nothing thrown crosses the C ABI.
template <typename F>
int guarded(F&& f) noexcept {
  try {
    return f();
  } catch (...) {
    return report(FM_ENOMEM, "out of host memory");
  }
}

int check_norm(const fm_layer_norm_args* a, bool backward);
int check_sample(const fm_sample_args* a);
int check_distill(const fm_distill_args* a, bool backward);

// the CPU backend (device = -1)
void cpu_norm_forward(const fm_layer_norm_args& a);
void cpu_norm_backward(const fm_layer_norm_args& a);
void cpu_sample(const fm_sample_args& a);
void cpu_distill_forward(const fm_distill_args& a);
void cpu_distill_backward(const fm_distill_args& a);
}  // namespace fm
