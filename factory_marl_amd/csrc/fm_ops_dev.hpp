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

// Exchanges between lanes without LDS: within rows of 16 lanes by data-parallel moves, between them by the row and half swaps.
// A value of 4 or 8 bytes goes a word at a time.
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ uint32_t move_word(uint32_t v) {  // lanes that nothing comes to get 0
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, true);
}
template <int M>
__device__ __forceinline__ uint32_t xor_word(uint32_t v) {  // the word of lane number ^ M
  if constexpr (M == 1) {
    return move_word<0xB1>(v);  // quads: 1 0 3 2
  } else if constexpr (M == 2) {
    return move_word<0x4E>(v);  // quads: 2 3 0 1
  } else if constexpr (M == 4) {
    return move_word<0x141>(move_word<0x1B>(v));  // quads reversed (^ 3), then eights (^ 7)
  } else if constexpr (M == 8) {
    return move_word<0x140>(move_word<0x141>(v));  // eights reversed (^ 7), then rows (^ 15)
  } else if constexpr (M == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);  // [0] even rows' words twice, [1] odd rows'
    return threadIdx.x & 16 ? r[0] : r[1];
  } else {
    static_assert(M == 32, "");
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);  // [0] the lower half's words twice, [1] the upper's
    return threadIdx.x & 32 ? r[0] : r[1];
  }
}
template <typename V, typename F>
__device__ __forceinline__ V by_words(V v, F&& f) {
  static_assert(sizeof(V) == 4 || sizeof(V) == 8, "");
  uint32_t w[sizeof(V) / 4];
  __builtin_memcpy(w, &v, sizeof(V));
#pragma unroll
  for (unsigned i = 0; i < sizeof(V) / 4; i++) w[i] = f(w[i]);
  __builtin_memcpy(&v, w, sizeof(V));
  return v;
}
template <int M, typename V>
__device__ __forceinline__ V lane_xor(V v) {
  return by_words(v, [](uint32_t w) { return xor_word<M>(w); });
}

// sums and maxima over groups of G lanes (a power of two up to 64); every lane gets the result, the order is fixed
template <int G, int M = 1, typename V>
__device__ __forceinline__ V group_sum(V v) {
  if constexpr (M < G)
    return group_sum<G, 2 * M>(v + lane_xor<M>(v));
  else
    return v;
}
template <int G, int M = 1>
__device__ __forceinline__ float group_max(float v) {
  if constexpr (M < G)
    return group_max<G, 2 * M>(fmaxf(v, lane_xor<M>(v)));
  else
    return v;
}
// sum over this lane and the ones before it, of G; j: the lane's number among them
template <int G, typename V>
__device__ __forceinline__ V sum_lanes(V v, int j) {
  if constexpr (G > 1) {
    const V q = by_words(v, [](uint32_t w) { return move_word<0x111>(w); });
    if (j >= 1) v += q;
  }
  if constexpr (G > 2) {
    const V q = by_words(v, [](uint32_t w) { return move_word<0x112>(w); });
    if (j >= 2) v += q;
  }
  if constexpr (G > 4) {
    const V q = by_words(v, [](uint32_t w) { return move_word<0x114>(w); });
    if (j >= 4) v += q;
  }
  if constexpr (G > 8) {
    const V q = by_words(v, [](uint32_t w) { return move_word<0x118>(w); });
    if (j >= 8) v += q;
  }
  // the last lane's of the row before to rows 1 and 3, then of the lower half to rows 2 and 3
  if constexpr (G > 16) v += by_words(v, [](uint32_t w) { return move_word<0x142, 0xa>(w); });
  if constexpr (G > 32) v += by_words(v, [](uint32_t w) { return move_word<0x143, 0xc>(w); });
  return v;
}

// over a block of NT > 64 threads; `buf` holds NT / 64 values and may be used again after the next barrier
template <int NT, typename V>
__device__ __forceinline__ V block_sum(V v, V* buf) {
  v = group_sum<64>(v);
  if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = v;
  __syncthreads();
  return group_sum<NT / 64>(buf[threadIdx.x % (NT / 64)]);
}
template <int NT>
__device__ __forceinline__ float block_max(float v, float* buf) {
  v = group_max<64>(v);
  if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = v;
  __syncthreads();
  return group_max<NT / 64>(buf[threadIdx.x % (NT / 64)]);
}

// n blocks as a grid that holds any number of them: a grid's line is limited to 2^32 threads
inline dim3 grid_of(int64_t n) {
  return dim3((unsigned)(n < (1 << 20) ? n : 1 << 20), (unsigned)((n + (1 << 20) - 1) >> 20));
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
