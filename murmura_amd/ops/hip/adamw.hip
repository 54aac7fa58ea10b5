// AdamW over all tensors of a model in one launch (K17).
//
// t is the number of the step. For every parameter p with gradient g:
//
//   m = b1*m + (1-b1)*g          v = b2*v + (1-b2)*g*g
//   p = p*(1 - lr*decay) - lr/(1-b1^t) * m / (sqrt(v)/sqrt(1-b2^t) + eps)
//
// The moments lie in the order of the parameters, as one vector of P values
// each, either in fp32 or in 8 bits. A block of 256 values in 8 bits shares a
// power of two over its largest value (held as the exponent field e of that
// value: the scale is 2^(e-126)), and a value below it is kept as
//
//   m: sign, 4 bits of exponent, 3 of mantissa   (1+M/8)*2^(E-15), 2^-17 at least
//   v: 5 bits of exponent, 3 of mantissa         (1+M/8)*2^(E-31), 2^-33 at least
//
// with exponent 0 for what has no leading one and all bits set for a NaN (an
// infinity is kept as one: neither comes back from there in 32 bits either).
// m and sqrt(v) so have the same range. Codes are rounded up with the
// probability of what is cut off: 1-b2 of v is a thousandth of it, and steps of
// an eighth rounded to nearest would never see it. A v above zero never becomes
// zero, which would make m/sqrt(v) boundless. Parameters in bf16 are rounded
// the same way, for steps below half of their last bit. The random bits are a
// hash of (seed, step, place), so a run repeats bit for bit.
//
// Every operation is rounded by itself (no contraction): an element's result
// does not depend on which path, vector width or compiler it went through, and
// the moments are those of elementary fp32 operations bit for bit.

#include "kernel_common.h"

#include <algorithm>

#pragma clang fp contract(off)

namespace mm {
namespace {

constexpr int NT = 256;
constexpr int QB = 256;  // values that share a scale
// Blocks walk over the vector, so that the step's constants, 150 operations in 64 bits, are worked
// out a few times a CU. bf16 with 8-bit moments: 11M values take 31 us in 1024 blocks, 36 in 2048, 70
// in 8192; 100M 216, 209 and 203 us.
constexpr int64_t FEW_BLOCKS = 1024, MANY_BLOCKS = 2048;

struct Segment {
  void* p;
  const void* g;
  int64_t start;  // place of its first value in the whole vector
};

// The table travels in the launch's arguments: a captured step needs no copy,
// and the 4 KB that a launch can carry hold 160 tensors. More take more launches.
constexpr int MAX_SEGMENTS = 160;
struct Table {
  int count;
  int64_t begin, end;  // the places of this launch
  bool last;           // the step ends with it
  Segment s[MAX_SEGMENTS];
};

struct Moments {  // fp32, or codes and exponents
  void* m;
  void* v;
  unsigned char* me;
  unsigned char* ve;
  bool whole;  // on 16 bytes (codes: on 8)
};

struct Hyper {
  double log_b1, log_b2;
  float b1, b1c, b2, b2c, eps;
  double lr, decay;
  const float* lr_dev;  // in place of lr, where the caller keeps it on the device
  unsigned int seed;
  int64_t* step;  // steps done before this one, fewer than 2^32
};

// what is the same for all elements of a step
struct Now {
  float keep, c1, c2;
  unsigned int key, t;
};

__device__ __forceinline__ Now now_of(const Hyper& h) {
  const unsigned int t = *(const unsigned int*)h.step + 1;
  const double lr = h.lr_dev ? (double)*h.lr_dev : h.lr;
  Now n;
  n.keep = (float)(1.0 - lr * h.decay);
  n.c1 = (float)(lr / -expm1((double)t * h.log_b1));
  n.c2 = (float)(1.0 / sqrt(-expm1((double)t * h.log_b2)));
  n.key = (h.seed * 0x9E3779B1u) ^ (t * 0x85A308D3u + 0x3C6EF372u);
  n.t = t;
  return n;
}

__device__ __forceinline__ unsigned int hash_of(unsigned int place, unsigned int key) {
  unsigned int x = place * 0x9E3779B1u + key;
  x = (x ^ (x >> 16)) * 0x6A09E667u;
  x = (x ^ (x >> 15)) * 0xBB67AE85u;
  return x ^ (x >> 16);
}

// FIRST: sign + 4 + 3 bits, TOP 15; else 5 + 3 bits, TOP 31
template <bool FIRST>
struct Code {
  static constexpr int TOP = FIRST ? 15 : 31;
  static constexpr unsigned int NAN_CODE = 8 * TOP + 7;

  // A code's bits at the place of a float's: the exponent then is off by 127 - TOP, and what has no
  // leading one is a denormal float. One ldexp puts both right, either way. What is not finite is
  // looked for in several values at once (odd_codes, the largest bits) and put right apart.
  __device__ static __forceinline__ float decode(unsigned int c, int e) {
    const float v = ldexpf(__uint_as_float((FIRST ? c & 127u : c) << 20), 127 - TOP + e - 126);
    return FIRST ? __uint_as_float(__float_as_uint(v) | (c & 128u) << 24) : v;
  }
  __device__ static __forceinline__ bool is_nan(unsigned int c) {
    return (FIRST ? c & 127u : c) == NAN_CODE;
  }
  // whether one of four codes is a NaN (or, seldom, the code after one): a byte without its
  // complement is zero
  __device__ static __forceinline__ bool odd_codes(unsigned int c4) {
    const unsigned int x = FIRST ? ~c4 & 0x7F7F7F7Fu : ~c4;
    return ((x - 0x01010101u) & ~x & 0x80808080u) != 0;
  }
  __device__ static __forceinline__ unsigned int encode(float x, int e, unsigned int dither) {
    const unsigned int bits = __float_as_uint(x), a = bits & 0x7FFFFFFFu;
    const float s = ldexpf(__uint_as_float(a), 126 - e - (127 - TOP));
    unsigned int c = (__float_as_uint(s) + (dither << 4 | 8u)) >> 20;
    if (!FIRST) c = max(c, min(a, 1u));
    return FIRST ? c | (bits >> 31) << 7 : c;
  }
};

// Keeps the compiler from working a seldom branch out for everybody.
#define MM_SELDOM() asm volatile("")

constexpr unsigned int INF_BITS = 0x7F800000u;
__device__ __forceinline__ unsigned int abs_bits(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }

// the segment that holds a place, the last that starts at or before it: a wave looks at 64 of
// them at once
__device__ __forceinline__ int segment_of(const Segment* s, int count, int64_t place) {
  const int lane = threadIdx.x & 63;
  int n = 0;
  for (int base = 0; base < count; base += 64)
    n += __popcll(__ballot(base + lane < count && s[base + lane].start <= place));
  return n - 1;
}

// the largest of 32 lanes, in all of them: within quads, halves and rows of 16 by the adder's own
// lane moves, across the two rows through LDS
__device__ __forceinline__ unsigned int max32(unsigned int x) {
  x = max(x, (unsigned int)__builtin_amdgcn_mov_dpp((int)x, 0xB1, 0xF, 0xF, true));   // 1 0 3 2
  x = max(x, (unsigned int)__builtin_amdgcn_mov_dpp((int)x, 0x4E, 0xF, 0xF, true));   // 2 3 0 1
  x = max(x, (unsigned int)__builtin_amdgcn_mov_dpp((int)x, 0x141, 0xF, 0xF, true));  // half mirror
  x = max(x, (unsigned int)__builtin_amdgcn_mov_dpp((int)x, 0x140, 0xF, 0xF, true));  // mirror
  return max(x, (unsigned int)__shfl_xor((int)x, 16, 64));
}

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&f)[8]) {
  constexpr int V = 16 / sizeof(T);
#pragma unroll
  for (int i = 0; i < 8; i += V) {
    const Vec<T, V> v = *(const Vec<T, V>*)(p + i);
#pragma unroll
    for (int j = 0; j < V; ++j) f[i + j] = to_float(v.e[j]);
  }
}

// A thread takes 8 values in a row, 32 threads the 256 of one scale, a block 2048 at a time. Where
// the 8 lie in one tensor, on 16 bytes, they are moved as a whole, else one by one; the arithmetic
// is the same.
template <typename T, typename GT, bool EIGHT>
__global__ __launch_bounds__(NT) void adamw_kernel(Table t, Moments st, Hyper h, int64_t chunks) {
  // the table in LDS: a lane's look into the launch's arguments goes out to the host's memory
  __shared__ Segment segs[MAX_SEGMENTS];
  for (int i = threadIdx.x; i < t.count; i += NT) segs[i] = t.s[i];
  const Now now = now_of(h);
  __syncthreads();
  for (int64_t chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x) {
    const int64_t first = t.begin + (chunk * NT + threadIdx.x) * 8;
    const int n = (int)max((int64_t)0, min((int64_t)8, t.end - first));
    int seg = t.count == 1 ? 0 : segment_of(segs, t.count, t.begin + (chunk * NT + (threadIdx.x & ~63)) * 8);
    float p[8], g[8], m[8], v[8];
    T* pp = nullptr;
    bool whole = false;
    alignas(8) unsigned int cm[2], cv[2];
    int me = 0, ve = 0;
    if (n > 0) {
      while (seg + 1 < t.count && segs[seg + 1].start <= first) ++seg;
      const int64_t at = first - segs[seg].start;
      pp = (T*)segs[seg].p + at;
      const GT* gp = (const GT*)segs[seg].g + at;
      whole = n == 8 && st.whole && (seg + 1 == t.count || segs[seg + 1].start >= first + 8) &&
              ((uintptr_t)pp | (uintptr_t)gp) % 16 == 0;
      if (EIGHT) {
        me = st.me[first / QB];
        ve = st.ve[first / QB];
      }
      if (whole) {
        load8(pp, p);
        load8(gp, g);
        if (EIGHT) {
          *(uint2*)cm = *(const uint2*)((const unsigned char*)st.m + first);
          *(uint2*)cv = *(const uint2*)((const unsigned char*)st.v + first);
        } else {
          load8((const float*)st.m + first, m);
          load8((const float*)st.v + first, v);
        }
      } else {
        cm[0] = cm[1] = cv[0] = cv[1] = 0;
        int sg = seg;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          p[i] = g[i] = m[i] = v[i] = 0.f;
          if (i >= n) continue;
          while (sg + 1 < t.count && segs[sg + 1].start <= first + i) ++sg;
          const int64_t place = first + i - segs[sg].start;
          p[i] = to_float(((const T*)segs[sg].p)[place]);
          g[i] = to_float(((const GT*)segs[sg].g)[place]);
          if (EIGHT) {
            cm[i / 4] |= (unsigned int)((const unsigned char*)st.m)[first + i] << (i % 4 * 8);
            cv[i / 4] |= (unsigned int)((const unsigned char*)st.v)[first + i] << (i % 4 * 8);
          } else {
            m[i] = ((const float*)st.m)[first + i];
            v[i] = ((const float*)st.v)[first + i];
          }
        }
      }
    }
    if (n == 0) {
#pragma unroll
      for (int i = 0; i < 8; ++i) m[i] = v[i] = p[i] = g[i] = 0.f;
      cm[0] = cm[1] = cv[0] = cv[1] = 0;
    }
    if (EIGHT) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        m[i] = Code<true>::decode(cm[i / 4] >> (i % 4 * 8) & 255u, me);
        v[i] = Code<false>::decode(cv[i / 4] >> (i % 4 * 8) & 255u, ve);
      }
      if (Code<true>::odd_codes(cm[0]) || Code<true>::odd_codes(cm[1]) ||
          Code<false>::odd_codes(cv[0]) || Code<false>::odd_codes(cv[1])) {
        MM_SELDOM();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (Code<true>::is_nan(cm[i / 4] >> (i % 4 * 8) & 255u)) m[i] = __uint_as_float(0x7FC00000u);
          if (Code<false>::is_nan(cv[i / 4] >> (i % 4 * 8) & 255u)) v[i] = __uint_as_float(0x7FC00000u);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      m[i] = h.b1 * m[i] + h.b1c * g[i];
      v[i] = h.b2 * v[i] + h.b2c * (g[i] * g[i]);
      // root and reciprocal are within one unit in the last place: a step of 1e-3 of a parameter
      // needs no more, and the exact ones took a quarter of all instructions
      const float root = __builtin_amdgcn_sqrtf(v[i]);
      p[i] = p[i] * now.keep - now.c1 * (m[i] * __builtin_amdgcn_rcpf(root * now.c2 + h.eps));
    }
    bool odd = false;
    if (EIGHT) {
      unsigned int ma = 0, va = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        ma = max(ma, abs_bits(m[i]));
        va = max(va, abs_bits(v[i]));
      }
      odd = max(ma, va) >= INF_BITS;
      if (odd) {  // the largest of what is finite
        MM_SELDOM();
        ma = va = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          ma = max(ma, abs_bits(m[i]) < INF_BITS ? abs_bits(m[i]) : 0u);
          va = max(va, abs_bits(v[i]) < INF_BITS ? abs_bits(v[i]) : 0u);
        }
      }
      me = (int)(max32(ma) >> 23);
      ve = (int)(max32(va) >> 23);
    }
    if (n == 0) continue;
    if (EIGHT && (threadIdx.x & 31) == 0) {
      st.me[first / QB] = (unsigned char)me;
      st.ve[first / QB] = (unsigned char)ve;
    }
    // The codes, and the parameters in bf16: what the dither carries into stays. Values that are not
    // finite are taken along and put right afterwards.
    alignas(16) T q[8];
    unsigned int most = 0, cut = 0;
    cm[0] = cm[1] = cv[0] = cv[1] = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (EIGHT || sizeof(T) == 2) cut = hash_of((unsigned int)first + i, now.key);
      if constexpr (sizeof(T) == 2) {
        most = max(most, abs_bits(p[i]));
        q[i].v = (unsigned short)((__float_as_uint(p[i]) + (cut * 0xA54FF53Bu >> 16)) >> 16);
      } else {
        q[i] = p[i];
      }
      if (EIGHT) {
        cm[i / 4] |= Code<true>::encode(m[i], me, cut & 0xFFFFu) << (i % 4 * 8);
        cv[i / 4] |= Code<false>::encode(v[i], ve, cut >> 16) << (i % 4 * 8);
      }
    }
    if (EIGHT && odd) {
      MM_SELDOM();
      cm[0] = cm[1] = cv[0] = cv[1] = 0;
      for (int i = 0; i < 8; ++i) {
        const unsigned int x = hash_of((unsigned int)first + i, now.key);
        const unsigned int a = abs_bits(m[i]) < INF_BITS ? Code<true>::encode(m[i], me, x & 0xFFFFu)
                                                         : Code<true>::NAN_CODE;
        const unsigned int b = abs_bits(v[i]) < INF_BITS ? Code<false>::encode(v[i], ve, x >> 16)
                                                         : Code<false>::NAN_CODE;
        cm[i / 4] |= (a | __float_as_uint(m[i]) >> 31 << 7) << (i % 4 * 8);
        cv[i / 4] |= b << (i % 4 * 8);
      }
    }
    if constexpr (sizeof(T) == 2) {
      if (most >= INF_BITS) {
        MM_SELDOM();
        for (int i = 0; i < 8; ++i)
          if (abs_bits(p[i]) >= INF_BITS) q[i] = round_bf16(p[i]);
      }
    }
    if (whole) {
      constexpr int V = 16 / sizeof(T);
#pragma unroll
      for (int i = 0; i < 8; i += V) *(Vec<T, V>*)(pp + i) = *(const Vec<T, V>*)(q + i);
      if (EIGHT) {
        *(uint2*)((unsigned char*)st.m + first) = *(const uint2*)cm;
        *(uint2*)((unsigned char*)st.v + first) = *(const uint2*)cv;
      } else {
#pragma unroll
        for (int i = 0; i < 8; i += 4) {
          *(float4*)((float*)st.m + first + i) = make_float4(m[i], m[i + 1], m[i + 2], m[i + 3]);
          *(float4*)((float*)st.v + first + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (i >= n) continue;
        while (seg + 1 < t.count && segs[seg + 1].start <= first + i) ++seg;
        ((T*)segs[seg].p)[first + i - segs[seg].start] = q[i];
        if (EIGHT) {
          ((unsigned char*)st.m)[first + i] = (unsigned char)(cm[i / 4] >> (i % 4 * 8));
          ((unsigned char*)st.v)[first + i] = (unsigned char)(cv[i / 4] >> (i % 4 * 8));
        } else {
          ((float*)st.m)[first + i] = m[i];
          ((float*)st.v)[first + i] = v[i];
        }
      }
    }
  }
  // The block that ends last counts the step. The high half of the count tells how many blocks of
  // the last launch have read it, and is zero again when the launch ends.
  if (!t.last) return;
  __syncthreads();
  if (threadIdx.x == 0) {
    unsigned int* halves = (unsigned int*)h.step;
    if (atomicAdd(halves + 1, 1u) == gridDim.x - 1)
      atomicExch((unsigned long long*)h.step, (unsigned long long)(now.t));
  }
}

// The values of 8 codes.
template <typename O, bool FIRST>
__device__ __forceinline__ void decode8(const unsigned char* __restrict__ c,
                                        const unsigned char* __restrict__ e, int64_t first, int64_t P,
                                        bool whole, O* __restrict__ out) {
  const int ex = e[first / QB];
  const int n = (int)min((int64_t)8, P - first);
  alignas(8) unsigned int in[2] = {0, 0};
  alignas(16) O o[8];
  if (whole && n == 8)
    *(uint2*)in = *(const uint2*)(c + first);
  else
    for (int i = 0; i < n; ++i) in[i / 4] |= (unsigned int)c[first + i] << (i % 4 * 8);
#pragma unroll
  for (int i = 0; i < 8; ++i)
    o[i] = from_float<O>(Code<FIRST>::decode(in[i / 4] >> (i % 4 * 8) & 255u, ex));
  if (Code<FIRST>::odd_codes(in[0]) || Code<FIRST>::odd_codes(in[1])) {
    MM_SELDOM();
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (Code<FIRST>::is_nan(in[i / 4] >> (i % 4 * 8) & 255u))
        o[i] = from_float<O>(__uint_as_float(0x7FC00000u));
  }
  if (n == 8) {
    constexpr int V = 16 / sizeof(O);
#pragma unroll
    for (int i = 0; i < 8; i += V) *(Vec<O, V>*)(out + first + i) = *(const Vec<O, V>*)(o + i);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) out[first + i] = o[i];
  }
}

// Both moments, 8 values of one a thread: blockIdx.y tells which.
template <typename O>
__global__ __launch_bounds__(NT) void adamw_decode_kernel(Moments st, int64_t P, O* __restrict__ m,
                                                          O* __restrict__ v) {
  const int64_t first = ((int64_t)blockIdx.x * NT + threadIdx.x) * 8;
  if (first >= P) return;
  if (blockIdx.y == 0)
    decode8<O, true>((const unsigned char*)st.m, st.me, first, P, st.whole, m);
  else
    decode8<O, false>((const unsigned char*)st.v, st.ve, first, P, st.whole, v);
}

void check_state(const std::vector<Tensor>& s, int64_t P, const at::Device& d) {
  TORCH_CHECK(s.size() == 1 || s.size() == 2, "adamw_step: a moment is one tensor or two");
  for (const Tensor& t : s)
    TORCH_CHECK(t.device() == d && t.is_contiguous(), "adamw_step: moments must be contiguous, "
                "on the parameters' device");
  TORCH_CHECK(s[0].numel() == P, "adamw_step: a moment must have a value for each parameter");
  if (s.size() == 1) {
    TORCH_CHECK(s[0].scalar_type() == at::kFloat, "adamw_step: a moment of one tensor is fp32");
  } else {
    TORCH_CHECK(s[0].scalar_type() == at::kByte && s[1].scalar_type() == at::kByte &&
                    s[1].numel() == ceil_div(P, QB),
                "adamw_step: an 8-bit moment is codes [P] and exponents [ceil(P/256)], uint8");
  }
}

void adamw_step(const std::vector<Tensor>& params, std::vector<Tensor> grads,
                const std::vector<Tensor>& exp_avg, const std::vector<Tensor>& exp_avg_sq,
                const Tensor& step, double lr, const OptTensor& lr_tensor, double b1, double b2,
                double eps, double decay, int64_t seed) {
  TORCH_CHECK(!params.empty() && params.size() == grads.size(),
              "adamw_step: as many gradients as parameters are wanted");
  const at::Device dev = params[0].device();
  const auto type = params[0].scalar_type(), gtype = grads[0].scalar_type();
  TORCH_CHECK(dev.is_cuda() && is_float_type(params[0]), "adamw_step: fp32 or bf16 on a GPU");
  TORCH_CHECK(gtype == type || gtype == at::kFloat, "adamw_step: gradients are of the parameters' "
              "type or fp32");
  const c10::DeviceGuard guard(dev);
  int64_t P = 0;
  std::vector<std::pair<const char*, const char*>> spans(params.size());
  for (size_t i = 0; i < params.size(); ++i) {
    const Tensor& p = params[i];
    TORCH_CHECK(p.device() == dev && grads[i].device() == dev && p.scalar_type() == type &&
                    grads[i].scalar_type() == gtype,
                "adamw_step: all parameters, and all gradients, must be of one type and device");
    TORCH_CHECK(p.sizes() == grads[i].sizes(), "adamw_step: a gradient must have its parameter's shape");
    TORCH_CHECK(p.is_non_overlapping_and_dense(), "adamw_step: a parameter must have no gaps");
    if (p.strides() != grads[i].strides())  // the same values in the parameter's order
      grads[i] = at::empty_strided(p.sizes(), p.strides(), grads[i].options()).copy_(grads[i]);
    spans[i] = {(const char*)p.data_ptr(), (const char*)p.data_ptr() + p.nbytes()};
    P += p.numel();
  }
  std::sort(spans.begin(), spans.end());
  for (size_t i = 1; i < spans.size(); ++i)
    TORCH_CHECK(spans[i - 1].second <= spans[i].first || spans[i].first == spans[i].second,
                "adamw_step: parameters share memory: pass each once");
  check_state(exp_avg, P, dev);
  check_state(exp_avg_sq, P, dev);
  TORCH_CHECK(exp_avg.size() == exp_avg_sq.size(), "adamw_step: both moments in the same bits");
  TORCH_CHECK(step.device() == dev && step.scalar_type() == at::kLong && step.numel() == 1,
              "adamw_step: step is one int64 on the parameters' device");
  TORCH_CHECK(b1 >= 0 && b1 < 1 && b2 >= 0 && b2 < 1, "adamw_step: betas lie in [0, 1)");
  if (lr_tensor.has_value())
    TORCH_CHECK(lr_tensor->device() == dev && lr_tensor->scalar_type() == at::kFloat &&
                    lr_tensor->numel() == 1,
                "adamw_step: lr on the device is one fp32 value");
  const hipStream_t st = stream_of(step);
  const bool eight = exp_avg.size() == 2;
  Moments mo{exp_avg[0].data_ptr(), exp_avg_sq[0].data_ptr(), nullptr, nullptr, false};
  mo.whole = ((uintptr_t)mo.m | (uintptr_t)mo.v) % (eight ? 8 : 16) == 0;
  if (eight) {
    mo.me = (unsigned char*)exp_avg[1].data_ptr();
    mo.ve = (unsigned char*)exp_avg_sq[1].data_ptr();
  }
  Hyper h;
  h.log_b1 = log(b1);
  h.log_b2 = log(b2);
  h.b1 = (float)b1;
  h.b1c = (float)(1 - b1);
  h.b2 = (float)b2;
  h.b2c = (float)(1 - b2);
  h.eps = (float)eps;
  h.lr = lr;
  h.decay = decay;
  h.lr_dev = lr_tensor.has_value() ? lr_tensor->data_ptr<float>() : nullptr;
  h.seed = (unsigned int)seed;
  h.step = step.data_ptr<int64_t>();
  // What a launch takes from place `begin` on, where params[next] holds it and starts at `start`. 256
  // values with one scale must lie within one launch: a tensor that ends inside of them is listed
  // again at the head of the next table.
  const auto table_from = [&](int64_t begin, size_t& next, int64_t& start) {
    Table t;
    t.count = 0;
    t.begin = begin;
    int64_t at = start;
    size_t i = next;
    for (; i < params.size() && t.count < MAX_SEGMENTS; ++i) {
      if (params[i].numel() == 0) continue;
      t.s[t.count++] = {params[i].data_ptr(), grads[i].data_ptr(), at};
      at += params[i].numel();
    }
    const int64_t unit = eight ? QB : 8;  // and a launch starts on whole vectors of the moments
    t.end = i == params.size() ? P : at / unit * unit;
    t.last = t.end == P;
    while (next < i && start + params[next].numel() <= t.end) start += params[next++].numel();
    return t;
  };
  // all that can be refused is refused before the first launch: a step is done as a whole or not at all
  if (eight && params.size() > MAX_SEGMENTS) {
    size_t next = 0;
    int64_t start = 0;
    for (int64_t begin = 0; begin < P;) {
      const int64_t end = table_from(begin, next, start).end;
      TORCH_CHECK(end > begin, "adamw_step: over ", MAX_SEGMENTS, " tensors within ", QB,
                  " values of 8-bit moments: pass them as one");
      begin = end;
    }
  }
  // a graph that saved a parameter must not be gone back through with its new values
  for (const Tensor& p : params)
    if (!p.is_inference()) p.unsafeGetTensorImpl()->bump_version();
  size_t next = 0;
  int64_t start = 0;
  for (int64_t begin = 0; begin < P;) {
    const Table t = table_from(begin, next, start);
    begin = t.end;
    const int64_t chunks = ceil_div(t.end - t.begin, (int64_t)NT * 8);
    const int64_t blocks = std::min(chunks, chunks < (1 << 14) ? FEW_BLOCKS : MANY_BLOCKS);
    MM_DISPATCH_TYPE(params[0], {
      if (gtype == type) {
        if (eight) adamw_kernel<T, T, true><<<(unsigned)blocks, NT, 0, st>>>(t, mo, h, chunks);
        else adamw_kernel<T, T, false><<<(unsigned)blocks, NT, 0, st>>>(t, mo, h, chunks);
      } else {
        if (eight) adamw_kernel<T, float, true><<<(unsigned)blocks, NT, 0, st>>>(t, mo, h, chunks);
        else adamw_kernel<T, float, false><<<(unsigned)blocks, NT, 0, st>>>(t, mo, h, chunks);
      }
    });
    check_launch("adamw_step");
  }
  if (P == 0) step.add_(1);
}

std::tuple<Tensor, Tensor> adamw_decode(const std::vector<Tensor>& exp_avg,
                                        const std::vector<Tensor>& exp_avg_sq, bool half) {
  TORCH_CHECK(exp_avg.size() == 2 && exp_avg_sq.size() == 2 && exp_avg[0].is_cuda(),
              "adamw_dequantize: 8-bit moments on a GPU are wanted");
  const int64_t P = exp_avg[0].numel();
  check_state(exp_avg, P, exp_avg[0].device());
  check_state(exp_avg_sq, P, exp_avg[0].device());
  const c10::DeviceGuard guard(exp_avg[0].device());
  const auto options = exp_avg[0].options().dtype(half ? at::kBFloat16 : at::kFloat);
  Tensor m = at::empty({P}, options), v = at::empty({P}, options);
  if (P == 0) return {m, v};
  const int64_t blocks = ceil_div(P, (int64_t)NT * 8);
  Moments mo{exp_avg[0].data_ptr(), exp_avg_sq[0].data_ptr(), (unsigned char*)exp_avg[1].data_ptr(),
             (unsigned char*)exp_avg_sq[1].data_ptr(), false};
  mo.whole = ((uintptr_t)mo.m | (uintptr_t)mo.v) % 8 == 0;
  MM_DISPATCH_TYPE(m, {
    adamw_decode_kernel<T><<<dim3(grid_of(blocks, NT, "adamw_dequantize"), 2), NT, 0, stream_of(m)>>>(
        mo, P, (T*)m.data_ptr(), (T*)v.data_ptr());
  });
  check_launch("adamw_dequantize");
  return {m, v};
}

}  // namespace

void bind_adamw(pybind11::module_& m) {
  m.def("adamw_step", &adamw_step, "K17: AdamW over many tensors, moments in fp32 or 8 bits",
        py::arg("params"), py::arg("grads"), py::arg("exp_avg"), py::arg("exp_avg_sq"),
        py::arg("step"), py::arg("lr"), py::arg("lr_tensor"), py::arg("b1"), py::arg("b2"),
        py::arg("eps"), py::arg("decay"), py::arg("seed"));
  m.def("adamw_decode", &adamw_decode, "K17: the values of 8-bit moments", py::arg("exp_avg"),
        py::arg("exp_avg_sq"), py::arg("half"));
}

}  // namespace mm
