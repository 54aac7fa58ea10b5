// Matrix product with bias, residual and activation in its epilogue, and the
// products of its backward pass (K18).
//
//   z = x W^T + b (+ res),  y = act(z)          x [M, K], W [N, K]
//   dz = dy * act'(z),  dres = dz,  db = sum dz,  dx = dz W,  dW = dz^T x
//
// All three products are one shape to the kernels: out[r, c] = sum_k A(r, k)
// B(c, k), where an operand lies either with k along its rows (x and W going
// forward) or with k across them (W in dx, both in dW). Products of bf16 are
// exact in fp32 and are summed there by the matrix cores; fp32 operands go
// through the fp32 matrix instructions, not through narrower ones.

#include "kernel_common.h"

namespace mm {
namespace {

constexpr int NT = 256;

typedef float f4 __attribute__((ext_vector_type(4)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));

struct Operand {
  const void* p;
  int64_t ld;  // values from one row in memory to the next
  bool whole;  // rows and base allow 16-byte loads
};

struct Epilogue {
  const void* bias;  // [cols], or null
  bool bias_float;
  const void* res;  // [rows, cols] without gaps, or null
  void* z;          // what the activation is taken of, or null
  void* out;
  int act;
};

__device__ __forceinline__ float activate(float z, int act) {
  switch (act) {
    case ACT_RELU: return act_fwd<ACT_RELU>(z);
    case ACT_SILU: return act_fwd<ACT_SILU>(z);
    case ACT_GELU: return act_fwd<ACT_GELU>(z);
    default: return z;
  }
}

template <typename T>
__device__ __forceinline__ void finish(const Epilogue& e, int64_t at, int64_t col, float v) {
  float z = v + load_param(e.bias, col, e.bias_float, 0.f);
  if (e.res) z += to_float(((const T*)e.res)[at]);
  if (e.z) ((T*)e.z)[at] = from_float<T>(z);
  ((T*)e.out)[at] = from_float<T>(activate(z, e.act));
}

template <typename T>
struct Tile;
template <>
struct Tile<bf16> {
  static constexpr int BK = 32, P = 8, LD = BK + 8;
};
template <>
struct Tile<float> {
  static constexpr int BK = 16, P = 4, LD = BK + 4;
};

// One pack of P values of an operand's tile, zeros where it ends.
template <typename T, bool ACROSS>
__device__ __forceinline__ Vec<T, Tile<T>::P> load_pack(const Operand& o, int64_t r, int64_t k,
                                                        int64_t R, int64_t Kd) {
  constexpr int P = Tile<T>::P;
  const int64_t major = ACROSS ? k : r, minor = ACROSS ? r : k;
  const int64_t majors = ACROSS ? Kd : R, minors = ACROSS ? R : Kd;
  const T* p = (const T*)o.p + major * o.ld + minor;
  Vec<T, P> v;
  if (o.whole && major < majors && minor + P <= minors) {
    v = *(const Vec<T, P>*)p;
  } else {
#pragma unroll
    for (int i = 0; i < P; ++i)
      v.e[i] = major < majors && minor + i < minors ? p[i] : from_float<T>(0.f);
  }
  return v;
}

// One operand's tile of ROWS x BK: through registers into LDS, k along the rows there.
template <typename T, bool ACROSS, int ROWS>
struct Stage {
  static constexpr int P = Tile<T>::P, BK = Tile<T>::BK, LD = Tile<T>::LD;
  static constexpr int PACKS = ROWS * BK / P / NT;
  Vec<T, P> v[PACKS];

  __device__ __forceinline__ static void where(int i, int& r, int& k) {
    const int q = threadIdx.x + i * NT;
    if (ACROSS) {
      r = q % (ROWS / P) * P;
      k = q / (ROWS / P);
    } else {
      r = q / (BK / P);
      k = q % (BK / P) * P;
    }
  }
  __device__ __forceinline__ void load(const Operand& o, int64_t r0, int64_t k0, int64_t R,
                                       int64_t Kd) {
#pragma unroll
    for (int i = 0; i < PACKS; ++i) {
      int r, k;
      where(i, r, k);
      v[i] = load_pack<T, ACROSS>(o, r0 + r, k0 + k, R, Kd);
    }
  }
  __device__ __forceinline__ void store(T* lds) {
#pragma unroll
    for (int i = 0; i < PACKS; ++i) {
      int r, k;
      where(i, r, k);
      if (ACROSS) {
#pragma unroll
        for (int j = 0; j < P; ++j) lds[(r + j) * LD + k] = v[i].e[j];
      } else {
        *(Vec<T, P>*)(lds + r * LD + k) = v[i];
      }
    }
  }
};

// Four waves side by side two by two, each with (BM/2) x (BN/2) of the tile in 16x16 blocks. A
// lane holds 4 rows of one column of each block.
template <typename T, bool AX, bool BX, int BM, int BN>
__global__ __launch_bounds__(NT) void gemm_kernel(Operand a, Operand b, int64_t M, int64_t N,
                                                  int64_t Kd, int64_t k_part, int64_t col_tiles,
                                                  Epilogue e, float* __restrict__ ws) {
  constexpr int BK = Tile<T>::BK, LD = Tile<T>::LD;
  constexpr int FM = BM / 32, FN = BN / 32;
  __shared__ __attribute__((aligned(16))) T as[BM * LD];
  __shared__ __attribute__((aligned(16))) T bs[BN * LD];
  const int64_t m0 = blockIdx.x / col_tiles * BM, n0 = blockIdx.x % col_tiles * BN;
  const int64_t kb = blockIdx.y * k_part, ke = min(Kd, kb + k_part);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wm = (wave >> 1) * (BM / 2), wn = (wave & 1) * (BN / 2);
  f4 acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = {0.f, 0.f, 0.f, 0.f};
  Stage<T, AX, BM> sa;
  Stage<T, BX, BN> sb;
  if (kb < ke) {
    sa.load(a, m0, kb, M, ke);
    sb.load(b, n0, kb, N, ke);
  }
  for (int64_t k0 = kb; k0 < ke; k0 += BK) {
    sa.store(as);
    sb.store(bs);
    __syncthreads();
    if (k0 + BK < ke) {
      sa.load(a, m0, k0 + BK, M, ke);
      sb.load(b, n0, k0 + BK, N, ke);
    }
    if constexpr (sizeof(T) == 2) {
      b8 fa[FM], fb[FN];
#pragma unroll
      for (int i = 0; i < FM; ++i)
        fa[i] = *(const b8*)(as + (wm + i * 16 + (lane & 15)) * LD + (lane >> 4) * 8);
#pragma unroll
      for (int j = 0; j < FN; ++j)
        fb[j] = *(const b8*)(bs + (wn + j * 16 + (lane & 15)) * LD + (lane >> 4) * 8);
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fa[i], fb[j], acc[i][j], 0, 0, 0);
    } else {
#pragma unroll
      for (int s = 0; s < BK; s += 4) {
        float fa[FM], fb[FN];
#pragma unroll
        for (int i = 0; i < FM; ++i) fa[i] = as[(wm + i * 16 + (lane & 15)) * LD + s + (lane >> 4)];
#pragma unroll
        for (int j = 0; j < FN; ++j) fb[j] = bs[(wn + j * 16 + (lane & 15)) * LD + s + (lane >> 4)];
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
          for (int j = 0; j < FN; ++j)
            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(fa[i], fb[j], acc[i][j], 0, 0, 0);
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int64_t r = m0 + wm + i * 16 + (lane >> 4) * 4 + q;
        const int64_t c = n0 + wn + j * 16 + (lane & 15);
        if (r >= M || c >= N) continue;
        if (ws)
          ws[(blockIdx.y * M + r) * N + c] = acc[i][j][q];
        else
          finish<T>(e, r * N + c, c, acc[i][j][q]);
      }
}

// joins the parts of a split sum, in their order
template <typename T>
__global__ __launch_bounds__(NT) void join_kernel(const float* __restrict__ ws, int parts,
                                                  int64_t total, int64_t N, Epilogue e) {
  const int64_t at = (int64_t)blockIdx.x * NT + threadIdx.x;
  if (at >= total) return;
  float v = 0.f;
  for (int s = 0; s < parts; ++s) v += ws[s * total + at];
  finish<T>(e, at, at % N, v);
}

// dz = dy * act'(z) and, for each chunk of rows, its sum over them. 64 columns a block, a wave a
// row. A relu's z is told by y = relu(z) as well: they are above zero together.
template <typename T, int ACT>
__global__ __launch_bounds__(NT) void act_bwd_kernel(const T* __restrict__ dy,
                                                     const T* __restrict__ z, int64_t M, int64_t N,
                                                     int64_t col_tiles, int64_t chunk,
                                                     T* __restrict__ dz, float* __restrict__ ws) {
  __shared__ float part[NT / 64][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t c = blockIdx.x % col_tiles * 64 + lane, k = blockIdx.x / col_tiles;
  const int64_t end = min(M, (k + 1) * chunk);
  float s = 0.f;
  if (c < N) {
    for (int64_t r = k * chunk + wave; r < end; r += NT / 64) {
      const int64_t at = r * N + c;
      float d = to_float(dy[at]);
      if constexpr (ACT != ACT_NONE) {
        d = act_bwd<ACT>(d, to_float(z[at]));
        dz[at] = from_float<T>(d);
      }
      s += d;
    }
  }
  part[wave][lane] = s;
  __syncthreads();
  if (ws && wave == 0 && c < N) {
#pragma unroll
    for (int w = 1; w < NT / 64; ++w) s += part[w][lane];
    ws[k * N + c] = s;
  }
}

__global__ __launch_bounds__(NT) void bias_grad_kernel(const float* __restrict__ ws, int64_t chunks,
                                                       int64_t N, bool is_float, void* db) {
  __shared__ float part[NT / 64][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t c = (int64_t)blockIdx.x * 64 + lane;
  float s = 0.f;
  if (c < N)
    for (int64_t k = wave; k < chunks; k += NT / 64) s += ws[k * N + c];
  part[wave][lane] = s;
  __syncthreads();
  if (wave == 0 && c < N) {
#pragma unroll
    for (int w = 1; w < NT / 64; ++w) s += part[w][lane];
    store_param(db, c, is_float, s);
  }
}

// ------------------------------------------------------------------ host
const void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

Operand operand(const Tensor& t) {
  const int64_t size = t.element_size();
  return {t.data_ptr(), t.stride(0), t.stride(0) * size % 16 == 0 && (uintptr_t)t.data_ptr() % 16 == 0};
}

template <typename T, bool AX, bool BX, int B>
void launch_gemm(const Operand& a, const Operand& b, int64_t M, int64_t N, int64_t Kd, int64_t parts,
                 const Epilogue& e, float* ws, hipStream_t st) {
  const int64_t rows = ceil_div(M, B), cols = ceil_div(N, B);
  TORCH_CHECK(rows * cols < (1LL << 31), "linear_act: too many tiles");
  const int64_t part = ceil_div(ceil_div(Kd, parts), Tile<T>::BK) * Tile<T>::BK;
  gemm_kernel<T, AX, BX, B, B><<<dim3((unsigned)(rows * cols), (unsigned)parts), NT, 0, st>>>(
      a, b, M, N, Kd, part, cols, e, ws);
}

// out [M, N] = A B^T over Kd, A and B with k along (or across) their rows in memory
template <bool AX, bool BX>
void gemm(const Tensor& a, const Tensor& b, int64_t M, int64_t N, int64_t Kd, const Epilogue& e,
          const Tensor& like) {
  if (M == 0 || N == 0) return;
  const hipStream_t st = stream_of(like);
  const bool large = ceil_div(M, 128) * ceil_div(N, 128) >= 256;
  const int64_t B = large ? 128 : 64;
  const int64_t tiles = ceil_div(M, B) * ceil_div(N, B);
  // few tiles: the sum is split over k, 128 values a part at least
  const int64_t parts = std::max<int64_t>(1, std::min(ceil_div(512, tiles), Kd / 128));
  Tensor ws;
  if (parts > 1) ws = at::empty({parts * M * N}, like.options().dtype(at::kFloat));
  float* wp = parts > 1 ? ws.data_ptr<float>() : nullptr;
  const Operand oa = operand(a), ob = operand(b);
  MM_DISPATCH_TYPE(like, {
    if (large) launch_gemm<T, AX, BX, 128>(oa, ob, M, N, Kd, parts, e, wp, st);
    else launch_gemm<T, AX, BX, 64>(oa, ob, M, N, Kd, parts, e, wp, st);
    if (parts > 1) {
      TORCH_CHECK(ceil_div(M * N, NT) < (1LL << 31), "linear_act: too many values");
      join_kernel<T><<<(unsigned)ceil_div(M * N, NT), NT, 0, st>>>(wp, (int)parts, M * N, N, e);
    }
  });
  check_launch("linear_act");
}

// a matrix whose rows have no gaps within: copied only if they have
Tensor rows_whole(const Tensor& t) { return t.stride(1) == 1 || t.size(1) == 1 ? t : t.contiguous(); }

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }

struct Forward {
  Tensor y, x, w, keep;  // the result, the matrices, and what the activation's gradient needs
};

Forward forward_of(const Tensor& x, const Tensor& weight, const Tensor& bias, const Tensor& residual,
                   int64_t act, bool differentiable) {
  const int64_t N = weight.size(0), Kd = weight.size(1);
  std::vector<int64_t> sizes = x.sizes().vec();
  sizes.back() = N;
  int64_t M = 1;
  for (size_t i = 0; i + 1 < sizes.size(); ++i) M *= sizes[i];
  Forward f;
  f.x = rows_whole(x.dim() == 2 ? x : x.reshape({M, Kd}));
  f.w = rows_whole(weight);
  const Tensor b = bias.defined() ? bias.contiguous() : bias;
  const Tensor res = residual.defined() ? residual.contiguous() : residual;
  f.y = at::empty(sizes, x.options());
  // silu and gelu have to see z again. It is kept in the operands' type, as a layer that writes
  // it out would keep it.
  const bool keep_z = differentiable && (act == ACT_SILU || act == ACT_GELU);
  if (keep_z) f.keep = at::empty(sizes, x.options());
  Epilogue e{ptr(b), b.defined() && b.scalar_type() == at::kFloat, ptr(res), (void*)ptr(f.keep),
             f.y.data_ptr(), (int)act};
  gemm<false, false>(f.x, f.w, M, N, Kd, e, x);
  if (differentiable && act == ACT_RELU) f.keep = f.y;
  return f;
}

class LinearAct : public torch::autograd::Function<LinearAct> {
 public:
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight,
                        const OptTensor& bias, const OptTensor& residual, int64_t act) {
    at::AutoDispatchBelowADInplaceOrView guard;
    const Tensor b = bias.value_or(Tensor()), res = residual.value_or(Tensor());
    const bool need_x = x.requires_grad(), need_w = weight.requires_grad();
    const Forward f = forward_of(x, weight, b, res, act, true);
    ctx->save_for_backward({need_w ? f.x : Tensor(), need_x ? f.w : Tensor(), f.keep});
    ctx->saved_data["act"] = act;
    ctx->saved_data["needs"] = (int64_t)(need_x | need_w << 1 | wants_grad(b) << 2 | wants_grad(res) << 3);
    ctx->saved_data["x"] = x.sizes().vec();
    ctx->saved_data["n"] = weight.size(0);
    ctx->saved_data["bias_float"] = b.defined() && b.scalar_type() == at::kFloat;
    return f.y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(),
                "linear_act has no second derivative (create_graph=True)");
    const auto saved = ctx->get_saved_variables();
    const int64_t needs = ctx->saved_data["needs"].toInt(), act = ctx->saved_data["act"].toInt();
    const std::vector<int64_t> sizes = ctx->saved_data["x"].toIntVector();
    const c10::DeviceGuard guard(grads[0].device());
    const Tensor dy = grads[0].contiguous();
    const int64_t Kd = sizes.back(), N = ctx->saved_data["n"].toInt();
    int64_t M = 1;
    for (size_t i = 0; i + 1 < sizes.size(); ++i) M *= sizes[i];
    const hipStream_t st = stream_of(dy);
    Tensor dz = act == ACT_NONE ? dy : at::empty_like(dy), db;
    const bool need_b = needs & 4;
    if (need_b)
      db = at::empty({N}, dy.options().dtype(ctx->saved_data["bias_float"].toBool() ? at::kFloat
                                                                                    : dy.scalar_type()));
    if (M * N == 0) {
      if (need_b) db.zero_();
    } else if (need_b || act != ACT_NONE) {
      const int64_t cols = ceil_div(N, 64);
      const int64_t chunk = std::max<int64_t>(16, ceil_div(M, std::max<int64_t>(1, 2048 / cols)));
      const int64_t chunks = ceil_div(M, chunk);
      TORCH_CHECK(cols * chunks < (1LL << 31), "linear_act: too many blocks");
      Tensor ws;
      if (need_b) ws = at::empty({chunks * N}, dy.options().dtype(at::kFloat));
      float* wp = need_b ? ws.data_ptr<float>() : nullptr;
      MM_DISPATCH_TYPE(dy, MM_DISPATCH_ACT(act, {
        act_bwd_kernel<T, ACT><<<(unsigned)(cols * chunks), NT, 0, st>>>(
            (const T*)ptr(dy), (const T*)ptr(saved[2]), M, N, cols, chunk, (T*)dz.data_ptr(), wp);
      }));
      if (need_b)
        bias_grad_kernel<<<(unsigned)cols, NT, 0, st>>>(wp, chunks, N, db.scalar_type() == at::kFloat,
                                                       db.data_ptr());
      check_launch("linear_act backward");
    }
    const Tensor dzm = dz.view({M, N});
    Tensor dx, dw;
    if (needs & 1) {
      dx = at::empty(sizes, dy.options());
      Epilogue e{nullptr, false, nullptr, nullptr, dx.data_ptr(), ACT_NONE};
      gemm<false, true>(dzm, saved[1], M, Kd, N, e, dy);
    }
    if (needs & 2) {
      dw = at::empty({N, Kd}, dy.options());
      Epilogue e{nullptr, false, nullptr, nullptr, dw.data_ptr(), ACT_NONE};
      gemm<true, true>(dzm, saved[0], N, Kd, M, e, dy);
    }
    return {dx, dw, db, needs & 8 ? dz : Tensor(), Tensor()};
  }
};

Tensor linear_act(const Tensor& x, const Tensor& weight, const OptTensor& bias, int64_t act,
                  const OptTensor& res) {
  TORCH_CHECK(x.is_cuda() && is_float_type(x), "linear_act: x must be fp32 or bf16 on a GPU");
  TORCH_CHECK(x.dim() >= 1 && weight.dim() == 2 && weight.size(1) == x.size(-1) &&
                  weight.device() == x.device() && weight.scalar_type() == x.scalar_type(),
              "linear_act: weight must be [N, K] for x [..., K], of its type and device");
  TORCH_CHECK(act >= 0 && act <= 3, "linear_act: unknown activation");
  const int64_t N = weight.size(0);
  if (bias.has_value())
    TORCH_CHECK(bias->device() == x.device() && bias->dim() == 1 && bias->size(0) == N &&
                    (bias->scalar_type() == at::kFloat || bias->scalar_type() == x.scalar_type()),
                "linear_act: bias must be [N], fp32 or of x's type, on its device");
  if (res.has_value()) {
    std::vector<int64_t> sizes = x.sizes().vec();
    sizes.back() = N;
    TORCH_CHECK(res->device() == x.device() && res->scalar_type() == x.scalar_type() &&
                    res->sizes() == at::IntArrayRef(sizes),
                "linear_act: res must be [..., N], of x's type and device");
  }
  const c10::DeviceGuard guard(x.device());
  const Tensor b = bias.value_or(Tensor()), r = res.value_or(Tensor());
  if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(weight) || wants_grad(b) || wants_grad(r)))
    return LinearAct::apply(x, weight, bias, res, act);
  return forward_of(x, weight, b, r, act, false).y;
}

}  // namespace

void bind_linear_act(pybind11::module_& m) {
  m.def("linear_act", &linear_act,
        "K18: act(x W^T + bias + res), differentiable", py::arg("x"), py::arg("weight"),
        py::arg("bias") = py::none(), py::arg("act") = 0, py::arg("res") = py::none());
}

}  // namespace mm
