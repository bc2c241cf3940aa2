// fm_ops_dev.hpp -- device side shared by the policy-head operators: element types, wave and block reductions, the
// launch guard.
#pragma once
#include <hip/hip_runtime.h>

#include <string>

#include "fm_ops.hpp"

namespace fm {
typedef _Float16 f16;
typedef __bf16 bf16;

template <typename T>
__device__ __forceinline__ float to_f32(T v) {
  return (float)v;
}
template <typename T>
__device__ __forceinline__ T from_f32(float v) {
  return (T)v;  // to the nearest, ties to even
}

// what a wave's lanes wrote before is there for its other lanes after
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// sums and maxima over groups of G lanes (a power of two up to 64); every lane gets the result, the order is fixed
template <int G, typename V>
__device__ __forceinline__ V group_sum(V v) {
#pragma unroll
  for (int m = G / 2; m; m >>= 1) v += __shfl_xor(v, m);
  return v;
}
template <int G>
__device__ __forceinline__ float group_max(float v) {
#pragma unroll
  for (int m = G / 2; m; m >>= 1) v = fmaxf(v, __shfl_xor(v, m));
  return v;
}

// over a block of NT threads; `buf` holds NT / 64 values and may be used again after the next barrier
template <int NT, typename V>
__device__ __forceinline__ V block_sum(V v, V* buf) {
  v = group_sum<64>(v);
  if (NT == 64) return v;
  if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = v;
  __syncthreads();
  V s = buf[0];
#pragma unroll
  for (int i = 1; i < NT / 64; i++) s += buf[i];
  return s;
}
template <int NT>
__device__ __forceinline__ float block_max(float v, float* buf) {
  v = group_max<64>(v);
  if (NT == 64) return v;
  if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = buf[0];
#pragma unroll
  for (int i = 1; i < NT / 64; i++) s = fmaxf(s, buf[i]);
  return s;
}

// Makes `device` current for one call's launches and restores the caller's; status() reports what the launches did.
struct OnDevice {
  int before = -1;
  hipError_t err;
  explicit OnDevice(int device) {
    err = hipGetDevice(&before);
    if (err == hipSuccess && before != device)
      err = hipSetDevice(device);
    else
      before = -1;
  }
  ~OnDevice() {
    if (before >= 0) (void)hipSetDevice(before);
  }
  int status(const char* what) {
    if (err == hipSuccess) err = hipGetLastError();
    if (err == hipSuccess) return FM_OK;
    try {
      return report(FM_EDEVICE, (std::string(what) + ": " + hipGetErrorString(err)).c_str());
    } catch (...) {
      return report(FM_EDEVICE, what);
    }
  }
};

// f(element type tag) for a dtype code that the checks have let through
template <typename T>
struct Tag {
  typedef T type;
};
template <typename F>
void with_type(int dtype, F&& f) {
  if (dtype == FM_DTYPE_F16)
    f(Tag<f16>());
  else if (dtype == FM_DTYPE_BF16)
    f(Tag<bf16>());
  else
    f(Tag<float>());
}
}  // namespace fm
