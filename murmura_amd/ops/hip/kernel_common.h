// What the kernels of the local training step share: element types, vectors
// of one memory transaction, wave reductions, activations, host-side checks.
#pragma once

#include <hip/hip_runtime.h>
#include <ATen/ATen.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/jit/frontend/tracer.h>
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

// V values as they lie in memory, two bf16 a register. (Arrays of 16-bit values take a register
// each as soon as they are looked at.)
template <typename T, int V>
struct Packed {
  static constexpr int W = V * sizeof(T) / 4;
  unsigned int w[W];
  static constexpr int ALIGNED = sizeof(T) * V < 16 ? sizeof(T) * V : 16;
  __device__ __forceinline__ void load(const T* p) {
    *this = *(const Packed*)__builtin_assume_aligned(p, ALIGNED);
  }
  __device__ __forceinline__ void store(T* p) const {
    *(Packed*)__builtin_assume_aligned(p, ALIGNED) = *this;
  }
  __device__ __forceinline__ float get(int i) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
    else return __uint_as_float(i & 1 ? w[i / 2] & 0xFFFF0000u : w[i / 2] << 16);
  }
  // values 2i and 2i + 1
  __device__ __forceinline__ void set2(int i, float a, float b) {
    if constexpr (sizeof(T) == 4) {
      w[2 * i] = __float_as_uint(a);
      w[2 * i + 1] = __float_as_uint(b);
    } else {
      typedef float f2 __attribute__((ext_vector_type(2)));
      typedef __bf16 h2 __attribute__((ext_vector_type(2)));
      w[i] = __builtin_bit_cast(unsigned int, __builtin_convertvector((f2){a, b}, h2));
    }
  }
};

// a parameter that is held in the activations' type or in fp32
__device__ __forceinline__ float load_param(const void* p, int64_t i, bool is_float, float none) {
  if (p == nullptr) return none;
  return is_float ? ((const float*)p)[i] : to_float(((const bf16*)p)[i]);
}
// V of them from i on; `whole`: i and p allow whole vectors
template <int V>
__device__ __forceinline__ void load_params(const void* p, int64_t i, bool is_float, bool whole, float none,
                                            float (&out)[V]) {
#pragma unroll
  for (int v = 0; v < V; ++v) out[v] = none;
  if (p == nullptr) return;
  if (whole && is_float) {
    Packed<float, V> q;
    q.load((const float*)p + i);
#pragma unroll
    for (int v = 0; v < V; ++v) out[v] = q.get(v);
  } else if (whole) {
    Packed<bf16, V> q;
    q.load((const bf16*)p + i);
#pragma unroll
    for (int v = 0; v < V; ++v) out[v] = q.get(v);
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) out[v] = load_param(p, i + v, is_float, none);
  }
}
__device__ __forceinline__ void store_param(void* p, int64_t i, bool is_float, float v) {
  if (is_float)
    ((float*)p)[i] = v;
  else
    ((bf16*)p)[i] = round_bf16(v);
}

// v of the lane that is `DPP`'s move away
template <int DPP>
__device__ __forceinline__ float moved(float v) {
  return __uint_as_float((unsigned int)__builtin_amdgcn_mov_dpp((int)__float_as_uint(v), DPP, 0xF, 0xF, true));
}

// Sum over the lanes that are alike in the low log2 `lanes` bits of their number, in all of them:
// rows of 16 by the adder's own lane moves (turned by 8 and 4, then within quads), rows by swapping
// them.
__device__ __forceinline__ float lanes_sum(float v, int lanes) {
  if (lanes < 4) v += moved<0x128>(v);  // turned by 8
  if (lanes < 3) v += moved<0x124>(v);  // by 4
  if (lanes < 2) v += moved<0x4E>(v);   // 2 3 0 1
  if (lanes < 1) v += moved<0xB1>(v);   // 1 0 3 2
  if (lanes < 5) {
    const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(s[0]) + __uint_as_float(s[1]);
  }
  if (lanes < 6) {
    const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(s[0]) + __uint_as_float(s[1]);
  }
  return v;
}

__device__ __forceinline__ float wave_sum(float v) { return lanes_sum(v, 0); }

// a / d for a < 2^16 and 0 < d < 2^16, by ceil(2^32 / d) (0 stands for 2^32)
__device__ __forceinline__ int divided(int a, unsigned int magic) {
  return magic ? (int)__umulhi((unsigned int)a, magic) : a;
}

// ------------------------------------------------------------- activations
enum Act { ACT_NONE = 0, ACT_RELU = 1, ACT_SILU = 2, ACT_GELU = 3 };

// Exponential and reciprocal are the hardware's, within one unit in the last place. For fp32 what
// the exponent's rounding cuts off is put back, so that the whole stays within 2^-22; for bf16, where a
// result is rounded by 2^-8 of itself, exp(-x) may be off by 2^-24 |x|.
__device__ __forceinline__ float exp2_of(float y, float rest) {  // 2^(y + rest)
  return __builtin_amdgcn_exp2f(y) * __builtin_fmaf(rest, 0.69314718055994531f, 1.f);
}
template <typename T>
__device__ __forceinline__ float exp_neg(float x) {  // exp(-x)
  constexpr float C = -1.44269504088896341f, LOW = -1.92596299e-8f;  // C in fp32 and its rest
  if constexpr (sizeof(T) == 4) {
    x = __builtin_amdgcn_fmed3f(x, -104.f, 104.f);  // beyond, it is infinite or zero
    const float y = x * C;
    return exp2_of(y, __builtin_fmaf(x, LOW, __builtin_fmaf(x, C, -y)));
  }
  return __builtin_amdgcn_exp2f(x * C);
}
template <typename T>
__device__ __forceinline__ float sigmoid(float z) {
  return __builtin_amdgcn_rcpf(1.f + exp_neg<T>(z));
}
// The normal distribution at z, and exp(-z*z/2), which its density shares with it.
//
// For fp32: erfc(a) = t P(t) exp(-a*a) with t = 1 / (1 + 0.3 a) and P of degree 8, fitted to least
// relative error over 0 <= a <= 10, 2.0e-8. The square's rounding is left: gelu is within 9 + z*z/2
// times 2^-24 of itself, its rms error over normal z 4.2e-8 (by erf in fp32 3.7e-8).
// For bf16: erfc by Abramowitz and Stegun, 7.1.26, within 1.5e-7 (5e-5 of itself at z = -3), with which
// fp32 would have 8.6e-8. Group norm over 64x128x56x56 in fp32 with gelu takes 50 us forward and 94 back,
// with that form 46 and 93, with the math library's erfc and exp 66 and 130; with silu 2% more than
// by the short exponential.
template <typename T>
__device__ __forceinline__ float normal_cdf(float z, float& e) {
  float half;
  if constexpr (sizeof(T) == 4) {
    constexpr float C = -0.72134752044448170f;  // -log2(e)/2
    const float a = fminf(fabsf(z), 15.f);  // beyond, it is 0 or 1
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(a, 0.212132034f, 1.f));
    const float square = a * a, y = square * C;
    e = exp2_of(y, __builtin_fmaf(square, C, -y));
    float p = -0.0647613704f;  // P / 2
    p = __builtin_fmaf(p, t, 0.242781207f);
    p = __builtin_fmaf(p, t, -0.256138206f);
    p = __builtin_fmaf(p, t, 0.273859084f);
    p = __builtin_fmaf(p, t, -0.0473247133f);
    p = __builtin_fmaf(p, t, 0.107462756f);
    p = __builtin_fmaf(p, t, 0.0741696581f);
    p = __builtin_fmaf(p, t, 0.0853576064f);
    p = __builtin_fmaf(p, t, 0.0845940039f);
    half = p * t * e;
  } else {
    const float a = fabsf(z) * 0.70710678118654752f;
    const float t = __builtin_amdgcn_rcpf(1.f + 0.3275911f * a);
    e = exp_neg<T>(a * a);
    const float poly =
        t * (0.254829592f + t * (-0.284496736f + t * (1.421413741f + t * (-1.453152027f + t * 1.061405429f))));
    half = 0.5f * poly * e;
  }
  return z < 0.f ? half : 1.f - half;
}

// act(z), for results of type T. A NaN stays one in each of them.
template <typename T, int ACT>
__device__ __forceinline__ float act_fwd(float z) {
  if constexpr (ACT == ACT_RELU) return z < 0.f ? 0.f : z;
  if constexpr (ACT == ACT_SILU) return z * sigmoid<T>(z);
  if constexpr (ACT == ACT_GELU) {
    float e;
    return z * normal_cdf<T>(z, e);
  }
  return z;
}

// dy * act'(z)
template <typename T, int ACT>
__device__ __forceinline__ float act_bwd(float dy, float z) {
  if constexpr (ACT == ACT_RELU) return z <= 0.f ? 0.f : dy;
  if constexpr (ACT == ACT_SILU) {
    const float s = sigmoid<T>(z);
    return dy * (s * (1.f + z * (1.f - s)));
  }
  if constexpr (ACT == ACT_GELU) {
    float e;
    const float cdf = normal_cdf<T>(z, e);
    return dy * (cdf + z * (e * 0.39894228040143268f));
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

// A tensor that carries a derivative going forward would lose it without a word: the kernels know
// none.
inline void refuse_forward_mode(std::initializer_list<const Tensor*> inputs, const char* what) {
  for (const Tensor* t : inputs)
    TORCH_CHECK(!t->defined() || !t->_fw_grad(0).defined(), what,
                ": no derivative going forward (forward-mode differentiation)");
}

// A trace would hold the result's memory and not the kernels that fill it.
inline void refuse_tracing(const char* what) {
  TORCH_CHECK(!torch::jit::tracer::isTracing(), what, ": not to be traced (torch.jit.trace)");
}

inline unsigned int magic_of(int64_t d) {
  return (unsigned int)(((1LL << 32) + d - 1) / d);  // d = 1 gives 0
}

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// a grid of so many blocks: its threads are counted in 32 bits
inline unsigned grid_of(int64_t blocks, int64_t threads, const char* what) {
  TORCH_CHECK(blocks > 0 && blocks * threads < (1LL << 32), what, ": too many values for one launch");
  return (unsigned)blocks;
}

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
