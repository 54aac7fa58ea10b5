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
  bool words;  // or 4-byte ones
  const void* rest;  // what p's values were rounded by, laid out like them, or null
};

struct Epilogue {
  const void* bias;  // [cols], or null
  bool bias_float;
  const void* res;  // [rows, cols] without gaps, or null
  void* z;          // what the activation is taken of, or null
  void* out;
  int act;
  bool whole;  // 8 columns of a row lie on 16 bytes, in all of these
};

// What a store may overwrite is not loaded ahead of it: a caller with several values loads bias and
// residual for all of them first.
template <typename T, int ACT>
__device__ __forceinline__ void finish(const Epilogue& e, int64_t at, float v, float bias, float res) {
  const float z = v + bias + res;
  if (e.z) ((T*)e.z)[at] = from_float<T>(z);
  ((T*)e.out)[at] = from_float<T>(act_fwd<T, ACT>(z));
}

template <typename T>
struct Eight {  // 8 values that lie on 16 bytes
  static constexpr int V = 16 / sizeof(T);
  Vec<T, V> v[8 / V];
  __device__ __forceinline__ T& operator[](int i) { return v[i / V].e[i % V]; }
  __device__ __forceinline__ void load(const void* p, int64_t at) {
#pragma unroll
    for (int i = 0; i < 8 / V; ++i) v[i] = ((const Vec<T, V>*)((const T*)p + at))[i];
  }
  __device__ __forceinline__ void store(void* p, int64_t at) const {
#pragma unroll
    for (int i = 0; i < 8 / V; ++i) ((Vec<T, V>*)((T*)p + at))[i] = v[i];
  }
};

// 8 columns of a row, which lie on 16 bytes
template <typename T, int ACT>
__device__ __forceinline__ void finish8(const Epilogue& e, int64_t at, const float (&bias)[8],
                                        Eight<T>& res, const float* v) {
  float z[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) z[i] = v[i] + bias[i];
  Eight<T> o;
  if (e.res) {
#pragma unroll
    for (int i = 0; i < 8; ++i) z[i] += to_float(res[i]);
  }
  if (e.z) {
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = from_float<T>(z[i]);
    o.store(e.z, at);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) o[i] = from_float<T>(act_fwd<T, ACT>(z[i]));
  o.store(e.out, at);
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
// lane holds 4 rows of one column of each block. HALVES: how often the sum is gone over, twice where A
// comes in two halves, of which the rest is the second.
template <typename T, bool AX, bool BX, int ACT, int BM, int BN, int HALVES>
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
  for (int half = 0; half < HALVES; ++half) {
    const Operand now{half ? a.rest : a.p, a.ld, a.whole, a.words, nullptr};
    if (kb < ke) {
      sa.load(now, m0, kb, M, ke);
      sb.load(b, n0, kb, N, ke);
    }
    for (int64_t k0 = kb; k0 < ke; k0 += BK) {
      sa.store(as);
      sb.store(bs);
      __syncthreads();
      if (k0 + BK < ke) {
        sa.load(now, m0, k0 + BK, M, ke);
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
          finish<T, ACT>(e, r * N + c, acc[i][j][q], load_param(e.bias, c, e.bias_float, 0.f),
                         e.res ? to_float(((const T*)e.res)[r * N + c]) : 0.f);
      }
}

// ------------------------------------------------------------ large products
//
// A block of WM x WN waves takes a tile of BM x BN, over 128 bytes of k at a time (64 values in bf16,
// on which the text below counts, 32 in fp32). The operands' tiles go
// from memory to LDS without registers between, into two buffers in turn. A wave multiplies a step
// in four quarters and reads the fragments of the next quarter beside the products of this one:
//
//   1  upper rows, k 0..31      read A's upper rows and B, k 32..63
//      wait, barrier X: A's upper rows and B are read; the lower rows have to be there
//   2  upper rows, k 32..63     load A's upper rows and B of two steps ahead over them
//                               read the lower rows, k 0..31
//   3  lower rows, k 0..31      read the lower rows, k 32..63
//      wait, barrier Y: the lower rows are read; the next step's upper rows and B have to be there
//   4  lower rows, k 32..63     load the lower rows of two steps ahead; read the next step's first
//
// Upper and lower rows are halves of each wave's own, and lie in buffers of their own. So every load
// has six quarters until it is waited for, with two buffers, and lines of 128 bytes are loaded whole.
// (One barrier a step, and loads a step ahead, reached 1030 to 1130 TFLOP/s at 8192x4096x12288, tiles
// of 32 of k four steps ahead 990 with half lines and 1180 with whole ones.)
//
// The loads are written in assembly, and waited for by count: the compiler would wait for all of
// them before each transposing read. They have no result in registers, and a wait that it counts
// without them only waits for more.
//
// LDS holds what a wave loaded in lane order, so the order that spares bank conflicts is made where
// lanes choose what they load:
// (A fragment is 16 bytes of each of 16 rows' k for 4 groups of 16 lanes: one bf16 product over 32 of
// k, or four fp32 ones over 4 each, of which group q takes k = 4q + j in the j-th.)
//   k along the rows:  [row][64], 16-byte chunk c of a row stands at c ^ (row / 2 & 7): 16 rows of
//                      one chunk, which are read at once, lie in the 16 places of 256 bytes
//   k across the rows: [k][rows], 16 columns of row k stand at their place ^ g(k); the fragments
//                      come through the transposing read, 4 rows of k for 16 lanes, or value by
//                      value in fp32
// Rows behind the operand's end repeat its last ones (their results are not stored); the k behind
// its end are zeros, put there through registers in a step of their own.
typedef short s4 __attribute__((ext_vector_type(4)));
typedef unsigned int u4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(3))) s4 lds_s4;

constexpr int ROW_BYTES = 128;

// ROWS rows of an operand: HR of each STRIDE, from the first on
// (LB bytes a lane and load: 16 where rows and their ends lie on 16 bytes, else 4)
template <typename T, bool ACROSS, int ROWS, int THREADS, int HR, int STRIDE, int LB>
struct Direct {
  static constexpr int E = 16 / sizeof(T), FK = ROW_BYTES / sizeof(T);  // values of a chunk, of a row
  static constexpr int U = LB / sizeof(T), PARTS = E / U;  // values of a load, loads of a chunk
  static constexpr int LOADS = ROWS * (FK / U) / THREADS;
  static constexpr int SIZE = ROWS * FK;
  static constexpr int CH = ROWS / E;        // chunks of a row of k
  static constexpr int PAIRS = ROWS / 16;    // 16 columns of it
  static constexpr int LOW = PAIRS < 4 ? PAIRS - 1 : 3, HIGH = PAIRS < 4 ? 0 : PAIRS / 4 - 1;
  const T* base;        // the tile, the same for all lanes
  unsigned at[LOADS];   // a lane's places from there, in bytes
  int64_t step;

  __device__ __forceinline__ static int g_of(int k) {
    return sizeof(T) == 4 ? (k >> 2) & LOW : (k & LOW) | ((k >> 3) & HIGH) << 2;
  }
  __device__ __forceinline__ static void slot(int i, int& r, int& k) {
    const int s = (i * THREADS + threadIdx.x) / PARTS, part = threadIdx.x % PARTS * U;
    if (ACROSS) {
      k = s / CH;
      r = ((s % CH) ^ g_of(k) * (16 / E)) * E + part;
    } else {
      r = s / 8;
      k = ((s % 8) ^ (r >> 1 & 7)) * E + part;
    }
  }
  __device__ __forceinline__ void init(const Operand& o, int64_t r0, int64_t k0, int64_t R) {
    step = ACROSS ? FK * o.ld : FK;
    r0 = min(r0, R - (ACROSS ? U : 1));  // rows that start behind the end
    base = (const T*)o.p + (ACROSS ? k0 * o.ld + r0 : r0 * o.ld + k0);
    const int last = (int)min(R - r0, (int64_t)(ROWS / HR * STRIDE)) - (ACROSS ? U : 1);
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      int r, k;
      slot(i, r, k);
      r = min(r / HR * STRIDE + r % HR, last);
      at[i] = (unsigned)(ACROSS ? k * o.ld + r : r * o.ld + k) * sizeof(T);
    }
  }
  // `wave` the same for all lanes. m0, which the load reads and the compiler sets for its own uses
  // alone, is told as overwritten; that it is not kept for anybody is what the warning says.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
  __device__ __forceinline__ void load(T* lds, int wave) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const unsigned to = (unsigned)(uintptr_t)(lds_void*)(lds + (i * THREADS + wave * 64) * U);
      if constexpr (LB == 16)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                     :
                     : "s"(to), "v"(at[i]), "s"(base)
                     : "memory", "m0");
      else
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2"
                     :
                     : "s"(to), "v"(at[i]), "s"(base)
                     : "memory", "m0");
    }
    base += step;
  }
#pragma clang diagnostic pop
  // the `left` values of k behind `steps` whole tiles, `away` from here
  __device__ __forceinline__ void load_tail(T* lds, int64_t steps, int left, int64_t away = 0) const {
    const T* p = base + away + steps * step;
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      int r, k;
      slot(i, r, k);
      const T* from = p + at[i] / sizeof(T);
      Vec<T, U> v = {};
      if ((ACROSS ? k + 1 : k + U) <= left) {
        v = *(const Vec<T, U>*)from;
      } else if (!ACROSS) {
#pragma unroll
        for (int j = 0; j < U; ++j)
          if (k + j < left) v.e[j] = from[j];
      }
      *(Vec<T, U>*)(lds + (i * THREADS + threadIdx.x) * U) = v;
    }
  }
  // 16 rows from `row`, half ks of the step's k: lane l has row l % 16, chunk l / 16 of the half
  __device__ __forceinline__ static u4 fragment(const T* lds, int row, int ks) {
    const int lane = threadIdx.x & 63, l = lane & 15, q = lane >> 4;
    if constexpr (!ACROSS) {
      return *(const u4*)(lds + (row + l) * FK + (((ks * 4 + q) ^ (l >> 1 & 7)) * E));
    } else if constexpr (sizeof(T) == 2) {
      const int g = ((l >> 2) & LOW) | (q & HIGH) << 2;
      const T* p = lds + (ks * 32 + q * 8 + (l >> 2)) * ROWS + ((row >> 4) ^ g) * 16 + (l & 3) * 4;
      union {
        s4 h[2];
        u4 v;
      } f;
      f.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)p);
      f.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(p + 4 * ROWS));
      return f.v;
    } else {
      const T* p = lds + (ks * 16 + q * 4) * ROWS + ((row >> 4) ^ (q & LOW)) * 16 + l;
      u4 f;
#pragma unroll
      for (int j = 0; j < 4; ++j) f[j] = __float_as_uint(p[j * ROWS]);
      return f;
    }
  }
};

template <typename T>
__device__ __forceinline__ f4 product(u4 a, u4 b, f4 c) {
  if constexpr (sizeof(T) == 2) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[j]), __uint_as_float(b[j]), c, 0, 0, 0);
    return c;
  }
}

// which tile a block takes: blocks of one XCD (every eighth) take neighbours, 8 tiles down before
// the next column, so that what they share stays in that XCD's L2
__device__ __forceinline__ void tile_of(int64_t b, int64_t rows, int64_t cols, int64_t& r, int64_t& c) {
  const int64_t total = rows * cols, each = total / 8, rest = total % 8, x = b % 8;
  const int64_t t = x * each + min(x, rest) + b / 8;
  const int64_t band = 8 * cols, top = t / band * 8, height = min((int64_t)8, rows - top);
  r = top + t % band % height;
  c = t % band / height;
}

// HALVES as in gemm_kernel. (A kernel for both takes up to 5% longer where there is one.)
template <typename T, bool AX, bool BX, int ACT, int BM, int BN, int WM, int WN, int LB, int HALVES>
__global__ __launch_bounds__(64 * WM * WN, 2) void gemm_large_kernel(
    Operand a, Operand b, int64_t M, int64_t N, int64_t Kd, int64_t a_end, int64_t b_end, int64_t k_part,
    int64_t row_tiles, int64_t col_tiles, Epilogue e, float* __restrict__ ws) {
  constexpr int THREADS = 64 * WM * WN, FM = BM / WM / 16, FN = BN / WN / 16, H = FM / 2;
  using A = Direct<T, AX, BM / 2, THREADS, H * 16, FM * 16, LB>;  // the upper rows, or the lower ones
  using B = Direct<T, BX, BN, THREADS, BN, BN, LB>;
  constexpr int FK = A::FK;
  __shared__ __attribute__((aligned(1024))) T lds[2 * (2 * A::SIZE + B::SIZE)];
  // per buffer: upper rows, lower rows, B
  const auto up = [&](int at) { return lds + at * (2 * A::SIZE + B::SIZE); };
  const auto low = [&](int at) { return up(at) + A::SIZE; };
  const auto bs = [&](int at) { return up(at) + 2 * A::SIZE; };
  if constexpr (AX || BX) e.bias = e.res = nullptr, e.z = nullptr;  // going back there are none
  int64_t tr, tc;
  tile_of(blockIdx.x, row_tiles, col_tiles, tr, tc);
  const int64_t m0 = tr * BM, n0 = tc * BN;
  const int64_t kb = blockIdx.y * k_part, ke = min(Kd, kb + k_part);
  const int tiles = (int)((max(ke, kb) - kb) / FK), left = (int)((max(ke, kb) - kb) % FK);
  const int64_t away = HALVES == 2 ? (const T*)a.rest - (const T*)a.p : 0;
  const int lead = left > 0 ? HALVES : 0;  // what is left over of k comes first, of both halves
  const int steps = HALVES * tiles + lead;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN * (BM / WM), wn = wave % WN * (BN / WN);
  A du, dl;
  B db;
  du.init(a, m0, kb, a_end);
  dl.init(a, m0 + H * 16, kb, a_end);
  db.init(b, n0, kb, b_end);
  for (int s = 0; s < lead; ++s) {
    du.load_tail(up(s), tiles, left, s * away);
    dl.load_tail(low(s), tiles, left, s * away);
    db.load_tail(bs(s), tiles, left);
  }
  // before step s is loaded: whether it is the second half's first, for which B starts again
  const auto turn = [&](int s) {
    if (HALVES == 1 || s != lead + tiles) return;
    du.base += away - tiles * du.step;
    dl.base += away - tiles * dl.step;
    db.base -= tiles * db.step;
  };
  for (int s = lead; s < min(steps, 2); ++s) {
    turn(s);
    du.load(up(s), wave);
    db.load(bs(s), wave);
    dl.load(low(s), wave);
  }
  f4 acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = {0.f, 0.f, 0.f, 0.f};
  u4 a0[H], a1[H], b0[FN], b1[FN];
  const auto read_a = [&](u4 (&f)[H], const T* tile, int ks) {
#pragma unroll
    for (int i = 0; i < H; ++i) f[i] = A::fragment(tile, wave / WN * (H * 16) + i * 16, ks);
  };
  const auto read_b = [&](u4 (&f)[FN], const T* tile, int ks) {
#pragma unroll
    for (int j = 0; j < FN; ++j) f[j] = B::fragment(tile, wn + j * 16, ks);
  };
  const auto multiply = [&](const u4 (&fa)[H], const u4 (&fb)[FN], int half) {
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < H; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j)
        acc[half * H + i][j] = product<T>(fb[j], fa[i], acc[half * H + i][j]);
    __builtin_amdgcn_sched_barrier(0);
  };
  // A step's loads but the oldest of them may still be on their way at a barrier; at the sum's end,
  // where nothing new is loaded, all are waited for.
  constexpr int AHEAD = 2 * A::LOADS + B::LOADS;
  static_assert(AHEAD < 64, "the count of outstanding loads has 6 bits");
  const auto barrier = [&](bool all) {
    if (all)
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    else
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(AHEAD) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  barrier(true);
  read_b(b0, bs(0), 0);
  read_a(a0, up(0), 0);
#pragma unroll 1
  for (int s = 0; s < steps; ++s) {
    const int at = s & 1;
    const bool more = s + 2 < steps;
    read_b(b1, bs(at), 1);
    read_a(a1, up(at), 1);
    multiply(a0, b0, 0);
    barrier(!more);
    read_a(a0, low(at), 0);
    if (more) {
      turn(s + 2);
      du.load(up(at), wave);
      db.load(bs(at), wave);
    }
    multiply(a1, b1, 0);
    read_a(a1, low(at), 1);
    multiply(a0, b0, 1);
    barrier(!more);
    // the last step reads on, into a tile that nobody needs
    read_b(b0, bs(at ^ 1), 0);
    read_a(a0, up(at ^ 1), 0);
    if (more) dl.load(low(at), wave);
    multiply(a1, b1, 1);
  }
  // A lane has 4 neighbouring columns of a row in each block.
  if (ws) {
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      const int64_t r = m0 + wm + i * 16 + (lane & 15);
      float* row = ws + (blockIdx.y * M + r) * N;
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        const int64_t c = n0 + wn + j * 16 + (lane >> 4) * 4;
        if (r >= M) continue;
        if (N % 4 == 0 && c < N) {
          *(f4*)(row + c) = acc[i][j];
        } else {
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (c + q < N) row[c + q] = acc[i][j][q];
        }
      }
    }
    return;
  }
  // Through LDS, a wave 32 of its rows at a time, so that each lane finishes 8 columns of one row
  // and rows leave in whole lines. 4 floats more a row keep 8 rows' writes in different banks.
  constexpr int COLS = BN / WN, PITCH = COLS + 4, LANES = COLS / 8, DOWN = 64 / LANES;
  static_assert(64 % COLS == 0 && FM % 2 == 0 && WM * WN * 32 * PITCH * 4 <= sizeof(lds), "");
  __syncthreads();
  float* mine = (float*)lds + wave * 32 * PITCH;
  const bool inside = e.whole && m0 + BM <= M && n0 + BN <= N;
  const int64_t c = n0 + wn + lane % LANES * 8;
  float bias[8];
#pragma unroll
  for (int q = 0; q < 8; ++q) bias[q] = c + q < N ? load_param(e.bias, c + q, e.bias_float, 0.f) : 0.f;
#pragma unroll
  for (int i = 0; i < FM; i += 2) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < FN; ++j)
        *(f4*)(mine + (h * 16 + (lane & 15)) * PITCH + j * 16 + (lane >> 4) * 4) = acc[i + h][j];
    __builtin_amdgcn_wave_barrier();
    const float* row = mine + lane / LANES * PITCH + lane % LANES * 8;
    const int64_t r = m0 + wm + i * 16 + lane / LANES;
    if (inside) {
      Eight<T> res[32 / DOWN];
      if (e.res) {
#pragma unroll
        for (int k = 0; k < 32 / DOWN; ++k) res[k].load(e.res, (r + k * DOWN) * N + c);
      }
#pragma unroll
      for (int k = 0; k < 32 / DOWN; ++k)
        finish8<T, ACT>(e, (r + k * DOWN) * N + c, bias, res[k], row + k * DOWN * PITCH);
    } else {  // a row at a time, a value a lane, the residuals of eight rows ahead
      constexpr int NEXT = 64 / COLS;
      const int64_t one = n0 + wn + lane % COLS, top = m0 + wm + i * 16 + lane / COLS;
      const float shift = one < N ? load_param(e.bias, one, e.bias_float, 0.f) : 0.f;
#pragma unroll 1
      for (int k = 0; k < 32; k += 8 * NEXT) {
        float res[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          const int64_t down = top + k + q * NEXT;
          res[q] = e.res && down < M && one < N ? to_float(((const T*)e.res)[down * N + one]) : 0.f;
        }
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          const int64_t down = top + k + q * NEXT;
          if (down < M && one < N)
            finish<T, ACT>(e, down * N + one,
                           mine[(k + q * NEXT + lane / COLS) * PITCH + lane % COLS], shift, res[q]);
        }
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// joins the parts of a split sum, in their order
template <typename T, int ACT>
__global__ __launch_bounds__(NT) void join_kernel(const float* __restrict__ ws, int parts,
                                                  int64_t total, int64_t N, Epilogue e) {
  const int64_t at = (int64_t)blockIdx.x * NT + threadIdx.x;
  if (at >= total) return;
  float v = 0.f;
  for (int s = 0; s < parts; ++s) v += ws[s * total + at];
  finish<T, ACT>(e, at, v, load_param(e.bias, at % N, e.bias_float, 0.f),
                 e.res ? to_float(((const T*)e.res)[at]) : 0.f);
}

// dz = dy * act'(z) and, for each chunk of rows, its sum over them (of a single chunk: the bias's
// gradient). 64 columns a block, a wave a row. A relu's z is told by y = relu(z) as well: they are above zero together.
// dz is rounded to the operands' type, which the matrix instructions of dx and dW take; its sum is of
// what it was before. In bf16 that is half a step a value, and with silu or gelu, whose dz is no copy
// of dy, dx and dW would be 1.44 times as far from their formula as with dz in fp32 (2.4e-3 against
// 1.7e-3, relative; 1.0 to 2.2 times where they have some dozen values). What it is rounded by goes to
// `rest`, in bf16 too, and through the products beside it: 16 bits of dz are kept. All of a pass with
// gradients takes 1.1 times as long for it at 64x3136x2048 (37 us, 41), 1.5 at 2048x2048x2048 (89, 132)
// and 1.56 at 8192x4096x12288 (2.04 ms, 3.18).
template <typename T, int ACT>
constexpr bool HAS_REST = sizeof(T) == 2 && ACT >= ACT_SILU;
template <typename T>
__device__ __forceinline__ float rest_of(float d) {  // of what is not finite there is none
  const float kept = to_float(from_float<T>(d));
  return fabsf(kept) < __builtin_inff() ? d - kept : 0.f;
}

template <typename T, int ACT>
__global__ __launch_bounds__(NT) void act_bwd_kernel(const T* __restrict__ dy,
                                                     const T* __restrict__ z, int64_t M, int64_t N,
                                                     int64_t col_tiles, int64_t chunk,
                                                     T* __restrict__ dz, T* __restrict__ rest, int64_t ld,
                                                     float* __restrict__ ws, void* __restrict__ db,
                                                     bool is_float) {
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
        d = act_bwd<T, ACT>(d, to_float(z[at]));
        dz[r * ld + c] = from_float<T>(d);
        if constexpr (HAS_REST<T, ACT>)
          if (rest) rest[r * ld + c] = from_float<T>(rest_of<T>(d));
      }
      s += d;
    }
  }
  part[wave][lane] = s;
  __syncthreads();
  if ((ws || db) && wave == 0 && c < N) {
#pragma unroll
    for (int w = 1; w < NT / 64; ++w) s += part[w][lane];
    if (db)
      store_param(db, c, is_float, s);
    else
      ws[k * N + c] = s;
  }
}

// The same by vectors of 16 bytes, 32 side by side and 8 rows a block, four of a thread's rows ahead:
// 8192x12288 in bf16 takes 111 us, 5.4 TB/s; by values 160.
template <typename T, int ACT>
__global__ __launch_bounds__(NT) void act_bwd_vector_kernel(const T* __restrict__ dy,
                                                            const T* __restrict__ z, int64_t M,
                                                            int64_t N, int64_t col_tiles, int64_t chunk,
                                                            T* __restrict__ dz, T* __restrict__ rest,
                                                            int64_t ld, float* __restrict__ ws,
                                                            void* __restrict__ db, bool is_float) {
  constexpr int V = 16 / sizeof(T), WIDE = 32 * V, AHEAD = 4;
  __shared__ float part[8][WIDE];
  const int64_t c0 = blockIdx.x % col_tiles * WIDE, c = c0 + threadIdx.x % 32 * V;
  const int64_t k = blockIdx.x / col_tiles, end = min(M, (k + 1) * chunk);
  float s[V] = {};
  if (c < N) {
    for (int64_t r = k * chunk + threadIdx.x / 32; r < end; r += 8 * AHEAD) {
      Packed<T, V> d[AHEAD], x[AHEAD];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i)
        if (r + 8 * i < end) {
          d[i].load(dy + (r + 8 * i) * N + c);
          if constexpr (ACT != ACT_NONE) x[i].load(z + (r + 8 * i) * N + c);
        }
#pragma unroll
      for (int i = 0; i < AHEAD; ++i)
        if (r + 8 * i < end) {
          float g[V];
#pragma unroll
          for (int v = 0; v < V; ++v) {
            g[v] = d[i].get(v);
            if constexpr (ACT != ACT_NONE) g[v] = act_bwd<T, ACT>(g[v], x[i].get(v));
            s[v] += g[v];
          }
          if constexpr (ACT != ACT_NONE) {
#pragma unroll
            for (int v = 0; v < V / 2; ++v) d[i].set2(v, g[2 * v], g[2 * v + 1]);
            d[i].store(dz + (r + 8 * i) * ld + c);
            if constexpr (HAS_REST<T, ACT>)
              if (rest) {
#pragma unroll
                for (int v = 0; v < V / 2; ++v)
                  d[i].set2(v, rest_of<T>(g[2 * v]), rest_of<T>(g[2 * v + 1]));
                d[i].store(rest + (r + 8 * i) * ld + c);
              }
          }
        }
    }
  }
  if (!ws && !db) return;
#pragma unroll
  for (int v = 0; v < V; ++v) part[threadIdx.x / 32][threadIdx.x % 32 * V + v] = s[v];
  __syncthreads();
  if (threadIdx.x < WIDE && c0 + threadIdx.x < N) {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += part[i][threadIdx.x];
    if (db)
      store_param(db, c0 + threadIdx.x, is_float, sum);
    else
      ws[k * N + c0 + threadIdx.x] = sum;
  }
}

__global__ __launch_bounds__(1024) void bias_grad_kernel(const float* __restrict__ ws, int64_t chunks,
                                                         int64_t N, bool is_float, void* db) {
  __shared__ float part[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t c = (int64_t)blockIdx.x * 64 + lane;
  float s = 0.f;
  if (c < N)
    for (int64_t k = wave; k < chunks; k += 16) s += ws[k * N + c];
  part[wave][lane] = s;
  __syncthreads();
  if (wave == 0 && c < N) {
#pragma unroll
    for (int w = 1; w < 16; ++w) s += part[w][lane];
    store_param(db, c, is_float, s);
  }
}

// ------------------------------------------------------------------ host
const void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

Operand operand(const Tensor& t) {
  const int64_t size = t.element_size(), ld = t.size(0) > 1 ? t.stride(0) : 0;
  const uintptr_t at = (uintptr_t)t.data_ptr();
  return {t.data_ptr(), ld, ld * size % 16 == 0 && at % 16 == 0, ld * size % 4 == 0 && at % 4 == 0, nullptr};
}

bool rows_of_8(int64_t N, std::initializer_list<const void*> ptrs) {
  if (N % 8) return false;
  for (const void* p : ptrs)
    if ((uintptr_t)p % 16) return false;
  return true;
}

// Up to two matrices, copied so that each row starts on 16 bytes, with zeros behind the values and
// in the rows behind `full`.
struct Pad {
  Operand from;
  int64_t full, cols;  // rows and columns that there are
  int64_t rows, ld;    // and with those behind them
  void* to;
};

template <typename T>
__global__ __launch_bounds__(NT) void pad_kernel(Pad a, Pad b) {
  for (int64_t i = blockIdx.x; i < a.rows + b.rows; i += gridDim.x) {
    const bool second = i >= a.rows;
    const Pad& p = second ? b : a;
    const int64_t row = second ? i - a.rows : i;
    const T* from = (const T*)p.from.p + row * p.from.ld;
    T* to = (T*)p.to + row * p.ld;
    for (int64_t c = threadIdx.x; c < p.ld; c += NT) to[c] = row < p.full && c < p.cols ? from[c] : T{};
  }
}

struct Choice {
  int tile;
  int64_t parts;
};

struct TileShape {
  int bm, bn, per_cu;
  // microseconds that a step of 128 bytes of k takes on a CU with 1, 2, 3 such blocks
  double bf16_us[4], fp32_us[4];
};
constexpr TileShape TILES[] = {
    {256, 256, 1, {1.80}, {7.0}},
    {256, 128, 1, {0.97}, {3.6}},
    {128, 128, 2, {0.67, 1.03}, {1.85, 3.6}},
    {64, 64, 4, {0.45, 0.50, 0.70, 0.90}, {0.60, 0.95, 1.40, 1.85}},
};

// Which tile, and into how many parts the sum is split: the least of an estimate. A tile's steps are
// measured at 4096 and 8192 rows and columns with all CUs busy, and with one block a CU, where what
// it waits for shows. A split costs its parts' writing and reading at 5 TB/s and a launch; and no
// choice is faster than memory, which some hundred blocks are needed to keep busy. The choice is
// within 15% of the best of all tiles and splits over 22 products that were measured, from 33x200x40
// on. bf16, M x K x N: 2048x12288x4096 takes 278 us in tiles of 256x256 and 205 in two parts, 184 in
// 256x128, 198 in 128x128; 1024x1024x1024 14 in 128x128, 9 in 64x64; 64x3136x2048 19 in 64x64 whole,
// 8.5 in 8 parts; 1x4096x12288 39 whole, 19 in 2 parts, 22 in 8.
// `halves`: 2 where A comes in two, and the sum is gone over twice.
Choice choose(int64_t M, int64_t N, int64_t Kd, int64_t elem, bool by_words, int halves) {
  Choice best{0, 1};
  double least = 1e30;
  const int64_t steps = ceil_div(Kd * elem, ROW_BYTES);
  const double bytes = (double)(halves * M * Kd + N * Kd + M * N) * elem;
  for (int t = by_words ? 2 : 0; t < 4; ++t) {
    const TileShape& s = TILES[t];
    const int64_t tiles = ceil_div(M, s.bm) * ceil_div(N, s.bn);
    for (int64_t parts = 1; parts <= 64 && (parts == 1 || (steps >= 2 * parts && tiles * parts <= 1536));
         parts *= 2) {
      const int64_t a_cu = ceil_div(tiles * parts, 256), full = a_cu / s.per_cu, rest = a_cu % s.per_cu;
      const double* us = elem == 2 ? s.bf16_us : s.fp32_us;
      const double part = (double)(halves * ceil_div(steps, parts));
      const double last = 2 + 1.5e-4 * s.bm * s.bn * s.per_cu;  // and the tile's way out
      double cost = full * (part * us[s.per_cu - 1] + last) + (rest ? part * us[rest - 1] + last : 0);
      cost = std::max(cost, bytes / 5e6 * std::max(1.0, 256.0 / (tiles * parts)));
      if (parts > 1) cost += 6 + (double)M * N * 8 * parts / 5e6;
      if (cost < least) {
        least = cost;
        best = {t, parts};
      }
    }
  }
  return best;
}

// only going back, in bf16, does A come in two halves
template <typename T, bool BX>
constexpr bool MAY_HALVE = BX && sizeof(T) == 2;

template <typename T, bool AX, bool BX, int ACT, int BM, int BN, int WM, int WN, int LB = 16>
void launch_large(const Operand& a, const Operand& b, int64_t M, int64_t N, int64_t Kd, int64_t Ma,
                  int64_t Nb, int64_t parts, const Epilogue& e, float* ws, hipStream_t st) {
  const int64_t rows = ceil_div(M, BM), cols = ceil_div(N, BN), values = ROW_BYTES / sizeof(T);
  const int64_t part = ceil_div(ceil_div(Kd, parts), values) * values;
  const dim3 grid(grid_of(rows * cols, 64 * WM * WN, "linear_act"), (unsigned)parts);
  if constexpr (MAY_HALVE<T, BX>)
    if (a.rest) {
      gemm_large_kernel<T, AX, BX, ACT, BM, BN, WM, WN, LB, 2>
          <<<grid, 64 * WM * WN, 0, st>>>(a, b, M, N, Kd, Ma, Nb, part, rows, cols, e, ws);
      return;
    }
  gemm_large_kernel<T, AX, BX, ACT, BM, BN, WM, WN, LB, 1>
      <<<grid, 64 * WM * WN, 0, st>>>(a, b, M, N, Kd, Ma, Nb, part, rows, cols, e, ws);
}

template <typename T, bool AX, bool BX, int ACT>
void launch_small(const Operand& a, const Operand& b, int64_t M, int64_t N, int64_t Kd, int64_t parts,
                  const Epilogue& e, float* ws, hipStream_t st) {
  const int64_t rows = ceil_div(M, 64), cols = ceil_div(N, 64);
  const int64_t part = ceil_div(ceil_div(Kd, parts), Tile<T>::BK) * Tile<T>::BK;
  const dim3 grid(grid_of(rows * cols, NT, "linear_act"), (unsigned)parts);
  if constexpr (MAY_HALVE<T, BX>)
    if (a.rest) {
      gemm_kernel<T, AX, BX, ACT, 64, 64, 2><<<grid, NT, 0, st>>>(a, b, M, N, Kd, part, cols, e, ws);
      return;
    }
  gemm_kernel<T, AX, BX, ACT, 64, 64, 1><<<grid, NT, 0, st>>>(a, b, M, N, Kd, part, cols, e, ws);
}

// Rows off the 16 bytes. Where they lie on 4, as fp32 always does, lanes load 4 bytes each: fp32
// 509x561x250 takes 15 us so and 14 through registers, 2000x999x1003 48 and 92, copied 52;
// 4001x4003x4099 1033, 2600 and 1074. bf16 needs more loads a product and is copied from PAD_WORDS
// multiplications on: 2002^3 takes 49 us by words and 46 copied, 3002^3 130 and 107, 4002^3 205 and
// 152. Rows of bf16 off the 4 bytes go through registers, and are copied from PAD_ODD on: 509x561x250
// takes 13 us so and 21 copied, 2000x561x250 20 and 22, 1000x1001x999 43 and 17, 4001x4003x4099 2435
// and 198.
constexpr double PAD_WORDS = 8e9, PAD_ODD = 8e8;

// out [M, N] = A B^T over Kd, A and B with k along (or across) their rows in memory; A plus `rest`,
// where there is one, and then A's rows are whole vectors
template <bool AX, bool BX>
void gemm(const Tensor& a, const Tensor& b, int64_t M, int64_t N, int64_t Kd, const Epilogue& e,
          const Tensor& like, const Tensor& rest = Tensor()) {
  if (M == 0 || N == 0) return;
  const hipStream_t st = stream_of(like);
  Operand oa = operand(a), ob = operand(b);
  oa.rest = ptr(rest);
  const int halves = oa.rest ? 2 : 1;
  const int64_t elem = like.element_size(), E = 16 / elem;
  int64_t Ma = AX && oa.rest ? ceil_div(M, E) * E : M, Nb = N;  // rows that may be read
  // offsets within a tile are 32 bits
  bool large = Kd > 0 && std::max(oa.ld, ob.ld) * 256 * elem < (1LL << 32);
  const bool fits_a = oa.whole && (!AX || Ma % E == 0), fits_b = ob.whole && (!BX || N % E == 0);
  const bool words = oa.words && ob.words && (!AX || Ma * elem % 4 == 0) && (!BX || N * elem % 4 == 0);
  bool by_words = false;
  Tensor padded;
  if (large && !(fits_a && fits_b)) {
    const double work = (double)M * N * Kd * halves;
    by_words = words && (elem == 4 || work < PAD_WORDS);
    large = by_words || work >= PAD_ODD;
    if (large && !by_words) {
      // k is filled up to whole steps with zeros, the rows that a product goes over to whole vectors
      const int64_t step = ROW_BYTES / elem;
      const auto pad = [&](const Tensor& t, const Operand& o, bool fits, bool across) {
        if (fits) return Pad{o, 0, 0, 0, 0, nullptr};
        return Pad{o, t.size(0), t.size(1), across ? ceil_div(t.size(0), step) * step : t.size(0),
                   across ? ceil_div(t.size(1), E) * E : ceil_div(t.size(1), step) * step, nullptr};
      };
      Pad pa = pad(a, oa, fits_a, AX), pb = pad(b, ob, fits_b, BX);
      padded = at::empty({pa.rows * pa.ld + pb.rows * pb.ld}, like.options());
      pa.to = padded.data_ptr();
      pb.to = (char*)pa.to + pa.rows * pa.ld * elem;
      // a block a row, as far as a launch has blocks
      const unsigned rows = (unsigned)std::min<int64_t>(pa.rows + pb.rows, 1 << 20);
      MM_DISPATCH_TYPE(like, (pad_kernel<T><<<rows, NT, 0, st>>>(pa, pb)));
      if (!fits_a) oa = {pa.to, pa.ld, true, true, nullptr}, Ma = AX ? pa.ld : M;
      if (!fits_b) ob = {pb.to, pb.ld, true, true, nullptr}, Nb = BX ? pb.ld : N;
      if (!fits_a && !fits_b) Kd = ceil_div(Kd, step) * step;
    }
  }
  Choice c{0, 1};
  if (large) {
    c = choose(M, N, Kd, elem, by_words, halves);
  } else {
    // few tiles: the sum is split over k, 128 values a part at least
    c.parts = std::max<int64_t>(1, std::min(ceil_div(512, ceil_div(M, 64) * ceil_div(N, 64)), Kd / 128));
  }
  Tensor ws;
  if (c.parts > 1) ws = at::empty({c.parts * M * N}, like.options().dtype(at::kFloat));
  float* wp = c.parts > 1 ? ws.data_ptr<float>() : nullptr;
  MM_DISPATCH_TYPE(like, {
    MM_DISPATCH_ACT((AX || BX) ? 0 : e.act, {
      if constexpr (ACT == ACT_NONE || !(AX || BX)) {  // only the forward product has an epilogue
        if (!large)
          launch_small<T, AX, BX, ACT>(oa, ob, M, N, Kd, c.parts, e, wp, st);
        else if (by_words && c.tile == 2)
          launch_large<T, AX, BX, ACT, 128, 128, 2, 2, 4>(oa, ob, M, N, Kd, Ma, Nb, c.parts, e, wp, st);
        else if (by_words)
          launch_large<T, AX, BX, ACT, 64, 64, 2, 2, 4>(oa, ob, M, N, Kd, Ma, Nb, c.parts, e, wp, st);
        else if (c.tile == 0)
          launch_large<T, AX, BX, ACT, 256, 256, 2, 4>(oa, ob, M, N, Kd, Ma, Nb, c.parts, e, wp, st);
        else if (c.tile == 1)
          launch_large<T, AX, BX, ACT, 256, 128, 4, 2>(oa, ob, M, N, Kd, Ma, Nb, c.parts, e, wp, st);
        else if (c.tile == 2)
          launch_large<T, AX, BX, ACT, 128, 128, 2, 2>(oa, ob, M, N, Kd, Ma, Nb, c.parts, e, wp, st);
        else
          launch_large<T, AX, BX, ACT, 64, 64, 2, 2>(oa, ob, M, N, Kd, Ma, Nb, c.parts, e, wp, st);
        if (c.parts > 1) {
          join_kernel<T, ACT>
              <<<grid_of(ceil_div(M * N, NT), NT, "linear_act"), NT, 0, st>>>(wp, (int)c.parts, M * N, N, e);
        }
      }
    });
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
  // it out would keep it: in bf16, dx, dW and db are 1.06 times as far from their formula as with z in
  // fp32 (1.0 to 1.3 times where they have some dozen values), for half of its memory.
  const bool keep_z = differentiable && (act == ACT_SILU || act == ACT_GELU);
  if (keep_z) f.keep = at::empty(sizes, x.options());
  Epilogue e{ptr(b), b.defined() && b.scalar_type() == at::kFloat, ptr(res), (void*)ptr(f.keep),
             f.y.data_ptr(), (int)act, rows_of_8(N, {ptr(res), ptr(f.keep), ptr(f.y)})};
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
    // x itself and not the matrix that was made of it: a view made in here counts its changes by
    // itself, and one in place would go unseen
    const Tensor kept_x = f.x.is_alias_of(x) ? x : f.x;
    ctx->save_for_backward({need_w ? kept_x : Tensor(), need_x ? f.w : Tensor(), f.keep});
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
    // [M, N]; in two halves its rows are filled up to whole vectors, with what nobody reads
    const bool halves = act >= ACT_SILU && dy.scalar_type() == at::kBFloat16 && (needs & 3);
    const int64_t ld = halves ? ceil_div(N, 8) * 8 : N;
    Tensor dz = act == ACT_NONE ? dy.view({M, N}) : at::empty({M, ld}, dy.options()).narrow(1, 0, N), db;
    const Tensor rest = halves ? at::empty({M, ld}, dy.options()) : Tensor();
    const bool need_b = needs & 4;
    if (need_b)
      db = at::empty({N}, dy.options().dtype(ctx->saved_data["bias_float"].toBool() ? at::kFloat
                                                                                    : dy.scalar_type()));
    if (M * N == 0) {
      if (need_b) db.zero_();
    } else if (need_b || act != ACT_NONE) {
      const bool vectors = N * dy.element_size() % 16 == 0 && (uintptr_t)dy.data_ptr() % 16 == 0 &&
                           (uintptr_t)dz.data_ptr() % 16 == 0 && (uintptr_t)ptr(rest) % 16 == 0 &&
                           (uintptr_t)ptr(saved[2]) % 16 == 0;
      const int64_t cols = ceil_div(N, vectors ? 512 / dy.element_size() : 64);
      // up to 128 rows one chunk, which needs no second launch; else as many as fill the CUs, and
      // 256 at most, which 16 waves join in 16 steps
      const int64_t most = std::min<int64_t>(256, std::max<int64_t>(1, 2048 / cols));
      const int64_t chunk = M <= 128 ? M : std::max<int64_t>(16, ceil_div(M, most));
      const int64_t chunks = ceil_div(M, chunk);
      Tensor ws;
      const bool bias_float = need_b && db.scalar_type() == at::kFloat;
      if (need_b && chunks > 1) ws = at::empty({chunks * N}, dy.options().dtype(at::kFloat));
      float* wp = ws.defined() ? ws.data_ptr<float>() : nullptr;
      void* once = need_b && chunks == 1 ? db.data_ptr() : nullptr;
      MM_DISPATCH_TYPE(dy, MM_DISPATCH_ACT(act, {
        const auto kernel = vectors ? &act_bwd_vector_kernel<T, ACT> : &act_bwd_kernel<T, ACT>;
        kernel<<<grid_of(cols * chunks, NT, "linear_act"), NT, 0, st>>>(
            (const T*)ptr(dy), (const T*)ptr(saved[2]), M, N, cols, chunk, (T*)dz.data_ptr(),
            (T*)ptr(rest), ld, wp, once, bias_float);
      }));
      if (wp)
        bias_grad_kernel<<<grid_of(ceil_div(N, 64), 1024, "linear_act"), 1024, 0, st>>>(wp, chunks, N, bias_float, db.data_ptr());
      check_launch("linear_act backward");
    }
    Tensor dx, dw;
    if (needs & 1) {
      dx = at::empty(sizes, dy.options());
      Epilogue e{nullptr, false, nullptr, nullptr, dx.data_ptr(), ACT_NONE, rows_of_8(Kd, {ptr(dx)})};
      gemm<false, true>(dz, saved[1], M, Kd, N, e, dy, rest);
    }
    if (needs & 2) {
      dw = at::empty({N, Kd}, dy.options());
      Epilogue e{nullptr, false, nullptr, nullptr, dw.data_ptr(), ACT_NONE, rows_of_8(Kd, {ptr(dw)})};
      gemm<true, true>(dz, saved[0].dim() == 2 ? saved[0] : saved[0].reshape({M, Kd}), N, Kd, M, e, dy, rest);
    }
    return {dx, dw, db, needs & 8 ? dz.view(dy.sizes()) : Tensor(), Tensor()};
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
  refuse_forward_mode({&x, &weight, &b, &r}, "linear_act");
  refuse_tracing("linear_act");
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
