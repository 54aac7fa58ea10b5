// What the kernels of the local training step share: element types, vectors
// of one memory transaction, wave reductions, activations, host-side checks.
#pragma once

#include <hip/hip_runtime.h>
#include <ATen/ATen.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/utils/pybind.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <cstdint>

namespace mm {

using at::Tensor;
namespace py = pybind11;
using OptTensor = c10::optional<Tensor>;

struct bf16 {
  unsigned short v;
};

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(bf16 x) {
  return __uint_as_float(((unsigned int)x.v) << 16);
}

// round to nearest even: the compiler turns this into v_cvt_pk_bf16_f32
__device__ __forceinline__ bf16 round_bf16(float f) {
  __bf16 b = (__bf16)f;
  bf16 r;
  __builtin_memcpy(&r, &b, 2);
  return r;
}

template <typename T>
__device__ __forceinline__ T from_float(float f);
template <>
__device__ __forceinline__ float from_float<float>(float f) { return f; }
template <>
__device__ __forceinline__ bf16 from_float<bf16>(float f) { return round_bf16(f); }

template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
  T e[V];
};

// a parameter that is held in the activations' type or in fp32
__device__ __forceinline__ float load_param(const void* p, int64_t i, bool is_float, float none) {
  if (p == nullptr) return none;
  return is_float ? ((const float*)p)[i] : to_float(((const bf16*)p)[i]);
}
__device__ __forceinline__ void store_param(void* p, int64_t i, bool is_float, float v) {
  if (is_float)
    ((float*)p)[i] = v;
  else
    ((bf16*)p)[i] = round_bf16(v);
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}

// ------------------------------------------------------------- activations
enum Act { ACT_NONE = 0, ACT_RELU = 1, ACT_SILU = 2, ACT_GELU = 3 };

// act(z). A NaN stays one in each of them.
template <int ACT>
__device__ __forceinline__ float act_fwd(float z) {
  if constexpr (ACT == ACT_RELU) return z < 0.f ? 0.f : z;
  if constexpr (ACT == ACT_SILU) return z / (1.f + __expf(-z));
  if constexpr (ACT == ACT_GELU) return 0.5f * z * (1.f + erff(z * 0.70710678118654752f));
  return z;
}

// dy * act'(z)
template <int ACT>
__device__ __forceinline__ float act_bwd(float dy, float z) {
  if constexpr (ACT == ACT_RELU) return z <= 0.f ? 0.f : dy;
  if constexpr (ACT == ACT_SILU) {
    const float s = 1.f / (1.f + __expf(-z));
    return dy * s * (1.f + z * (1.f - s));
  }
  if constexpr (ACT == ACT_GELU) {
    const float cdf = 0.5f * (1.f + erff(z * 0.70710678118654752f));
    return dy * (cdf + z * (__expf(-0.5f * z * z) * 0.39894228040143268f));
  }
  return dy;
}

// ---------------------------------------------------------------- host side
inline hipStream_t stream_of(const Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

inline bool is_float_type(const Tensor& t) {
  return t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16;
}

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

inline void check_launch(const char* what) {
  const hipError_t e = hipGetLastError();
  TORCH_CHECK(e == hipSuccess, what, ": launch failed: ", hipGetErrorString(e));
}

#define MM_DISPATCH_TYPE(TENSOR, ...)             \
  if ((TENSOR).scalar_type() == at::kFloat) {     \
    using T = float;                              \
    __VA_ARGS__;                                  \
  } else {                                        \
    using T = mm::bf16;                           \
    __VA_ARGS__;                                  \
  }

#define MM_DISPATCH_ACT(ACT_VALUE, ...)                        \
  switch (ACT_VALUE) {                                         \
    case mm::ACT_RELU: { constexpr int ACT = mm::ACT_RELU; __VA_ARGS__; } break; \
    case mm::ACT_SILU: { constexpr int ACT = mm::ACT_SILU; __VA_ARGS__; } break; \
    case mm::ACT_GELU: { constexpr int ACT = mm::ACT_GELU; __VA_ARGS__; } break; \
    default: { constexpr int ACT = mm::ACT_NONE; __VA_ARGS__; } break;           \
  }

}  // namespace mm
