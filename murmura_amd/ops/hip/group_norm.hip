// Group norm with residual and activation over channels-last images (K16).
//
// x is [N, R, C] in memory, R pixels of C channels; group g of sample n holds
// R * C/G values. With mean, rstd over a group and xhat = (x - mean) * rstd:
//
//   z = xhat * gamma + beta (+ res),  y = act(z)
//   dz = dy * act'(z),  dres = dz,  dbeta = sum dz,  dgamma = sum dz * xhat
//   dx = rstd * (dz*gamma - avg(dz*gamma) - xhat * avg(dz*gamma*xhat))
//
// A thread owns V channels (one memory transaction) and walks over rows, so
// that every load is whole and the channels' sums stay in registers. Sums run
// rows of a thread -> lanes of a wave -> waves of a block -> chunks, always in
// the same order: no atomics, the same bits on every run. All statistics are
// fp32; a variance is taken around its own mean, chunks are joined by their
// counts, so that a level far above the spread costs no digits.

#include "kernel_common.h"

namespace mm {
namespace {

constexpr int NT = 256;          // threads of a block
constexpr int NW = NT / 64;      // its waves
constexpr int K = 8;             // rows that a thread holds
constexpr int MAX_TILE = 64 * 8; // channels of a tile: 64 lanes of 8

struct Shape {
  int64_t R;    // pixels of a sample
  int C, G, Cg; // channels, groups, channels of a group
  int lanes;    // log2 of the lanes that lie side by side along the channels
  int tiles;    // channel tiles of (1 << lanes) * V
  int S;        // row chunks of (NT >> lanes) * K
};

struct Place {
  int64_t n, row0, rows;  // sample; first row of the chunk; rows in it
  int tile, chunk, col, c, lane_row, step;
  bool active;
};

template <int V>
__device__ __forceinline__ Place place_of(const Shape& s) {
  Place p;
  const int64_t b = blockIdx.x;
  p.chunk = (int)(b % s.S);
  p.tile = (int)((b / s.S) % s.tiles);
  p.n = b / ((int64_t)s.S * s.tiles);
  p.step = NT >> s.lanes;
  p.row0 = (int64_t)p.chunk * p.step * K;
  p.rows = min((int64_t)p.step * K, s.R - p.row0);
  p.col = threadIdx.x & ((1 << s.lanes) - 1);
  p.lane_row = threadIdx.x >> s.lanes;
  p.c = (p.tile * (1 << s.lanes) + p.col) * V;
  p.active = p.c < s.C;
  return p;
}

// Sums `acc` over the rows of the block; part[wave][channel of the tile] holds
// what the waves have, the caller adds them after the barrier.
template <int V>
__device__ __forceinline__ void rows_to_waves(float (&acc)[V], int lanes, int col, float* part) {
#pragma unroll
  for (int v = 0; v < V; ++v) acc[v] = lanes_sum(acc[v], lanes);
  const int tile = (1 << lanes) * V;
  if ((threadIdx.x & 63) < (1 << lanes)) {
#pragma unroll
    for (int v = 0; v < V; ++v) part[(threadIdx.x >> 6) * tile + col * V + v] = acc[v];
  }
}

__device__ __forceinline__ float over_waves(const float* part, int tile, int c) {
  float s = 0.f;
#pragma unroll
  for (int w = 0; w < NW; ++w) s += part[w * tile + c];
  return s;
}

// (mean, sum of squares around it) of each channel over a chunk of rows
template <typename T, int V>
__global__ __launch_bounds__(NT) void gn_stats_kernel(const T* __restrict__ x, Shape s,
                                                      float2* __restrict__ ws) {
  __shared__ float part[NW * MAX_TILE];
  __shared__ float mean[MAX_TILE];
  const Place p = place_of<V>(s);
  const int tile = (1 << s.lanes) * V;
  const float inv = 1.f / (float)p.rows;
  Vec<T, V> val[K];
  float acc[V] = {};
#pragma unroll
  for (int i = 0; i < K; ++i) {
    const int64_t r = p.lane_row + i * p.step;
    if (p.active && r < p.rows) {
      val[i] = *(const Vec<T, V>*)(x + (p.n * s.R + p.row0 + r) * s.C + p.c);
#pragma unroll
      for (int v = 0; v < V; ++v) acc[v] += to_float(val[i].e[v]);
    }
  }
  rows_to_waves<V>(acc, s.lanes, p.col, part);
  __syncthreads();
  for (int c = threadIdx.x; c < tile; c += NT) mean[c] = over_waves(part, tile, c) * inv;
  __syncthreads();
#pragma unroll
  for (int v = 0; v < V; ++v) acc[v] = 0.f;
#pragma unroll
  for (int i = 0; i < K; ++i) {
    const int64_t r = p.lane_row + i * p.step;
    if (p.active && r < p.rows) {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float d = to_float(val[i].e[v]) - mean[p.col * V + v];
        acc[v] += d * d;
      }
    }
  }
  rows_to_waves<V>(acc, s.lanes, p.col, part);
  __syncthreads();
  for (int c = threadIdx.x; c < tile; c += NT) {
    const int cc = p.tile * tile + c;
    if (cc < s.C)
      ws[(p.n * s.S + p.chunk) * s.C + cc] = make_float2(mean[c], over_waves(part, tile, c));
  }
}

__device__ __forceinline__ float block_sum(float v, float* lds) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int w = 0; w < NW; ++w) s += lds[w];
  return s;
}

// joins the chunks' statistics, a block a group
__global__ __launch_bounds__(NT) void gn_join_stats_kernel(const float2* __restrict__ ws, Shape s,
                                                           int64_t all, float eps,
                                                           float* __restrict__ mean,
                                                           float* __restrict__ rstd) {
  __shared__ float lds[NW];
  const int64_t chunk_rows = (int64_t)(NT >> s.lanes) * K;
  const int64_t entries = (int64_t)s.S * s.Cg;
  for (int64_t b = blockIdx.x; b < all; b += gridDim.x) {
    const float2* w = ws + b / s.G * s.S * s.C + b % s.G * s.Cg;
    float sum = 0.f;
    for (int64_t e = threadIdx.x; e < entries; e += NT) {
      const int64_t k = e / s.Cg;
      sum += w[k * s.C + e % s.Cg].x * (float)min(chunk_rows, s.R - k * chunk_rows);
    }
    const float inv = 1.f / ((float)s.R * (float)s.Cg);
    const float mu = block_sum(sum, lds) * inv;
    float m2 = 0.f;
    for (int64_t e = threadIdx.x; e < entries; e += NT) {
      const int64_t k = e / s.Cg;
      const float2 q = w[k * s.C + e % s.Cg];
      const float d = q.x - mu;
      m2 += q.y + d * d * (float)min(chunk_rows, s.R - k * chunk_rows);
    }
    m2 = block_sum(m2, lds);
    if (threadIdx.x == 0) {
      mean[b] = mu;
      rstd[b] = 1.f / sqrtf(m2 * inv + eps);
    }
  }
}

// the affine map of a thread's channels
template <int V>
struct Affine {
  float mu[V], rs[V], ga[V], be[V];
  __device__ __forceinline__ void load(const Shape& s, const Place& p, const float* mean,
                                       const float* rstd, const void* gamma, const void* beta,
                                       bool wf) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int g = (p.c + v) / s.Cg;
      mu[v] = mean[p.n * s.G + g];
      rs[v] = rstd[p.n * s.G + g];
      ga[v] = load_param(gamma, p.c + v, wf, 1.f);
      be[v] = load_param(beta, p.c + v, wf, 0.f);
    }
  }
  __device__ __forceinline__ float xhat(float x, int v) const { return (x - mu[v]) * rs[v]; }
};

template <typename T, int V, int ACT>
__global__ __launch_bounds__(NT) void gn_apply_kernel(
    const T* __restrict__ x, const T* __restrict__ res, Shape s, const float* __restrict__ mean,
    const float* __restrict__ rstd, const void* __restrict__ gamma, const void* __restrict__ beta,
    bool wf, T* __restrict__ y) {
  const Place p = place_of<V>(s);
  if (!p.active) return;
  Affine<V> a;
  a.load(s, p, mean, rstd, gamma, beta, wf);
#pragma unroll
  for (int i = 0; i < K; ++i) {
    const int64_t r = p.lane_row + i * p.step;
    if (r >= p.rows) break;
    const int64_t at = (p.n * s.R + p.row0 + r) * s.C + p.c;
    const Vec<T, V> xv = *(const Vec<T, V>*)(x + at);
    Vec<T, V> rv, yv;
    if (res) rv = *(const Vec<T, V>*)(res + at);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float z = a.xhat(to_float(xv.e[v]), v) * a.ga[v] + a.be[v];
      if (res) z += to_float(rv.e[v]);
      yv.e[v] = from_float<T>(act_fwd<T, ACT>(z));
    }
    *(Vec<T, V>*)(y + at) = yv;
  }
}

// (sum dz, sum dz * xhat) of each channel over a chunk of rows; dres = dz
template <typename T, int V, int ACT>
__global__ __launch_bounds__(NT) void gn_bwd_sums_kernel(
    const T* __restrict__ x, const T* __restrict__ dy, const T* __restrict__ res, Shape s,
    const float* __restrict__ mean, const float* __restrict__ rstd, const void* __restrict__ gamma,
    const void* __restrict__ beta, bool wf, T* __restrict__ dres, float2* __restrict__ ws) {
  __shared__ float part[2][NW * MAX_TILE];
  const Place p = place_of<V>(s);
  const int tile = (1 << s.lanes) * V;
  float sz[V] = {}, sx[V] = {};
  if (p.active) {
    Affine<V> a;
    a.load(s, p, mean, rstd, gamma, beta, wf);
#pragma unroll
    for (int i = 0; i < K; ++i) {
      const int64_t r = p.lane_row + i * p.step;
      if (r >= p.rows) break;
      const int64_t at = (p.n * s.R + p.row0 + r) * s.C + p.c;
      const Vec<T, V> xv = *(const Vec<T, V>*)(x + at);
      const Vec<T, V> dv = *(const Vec<T, V>*)(dy + at);
      Vec<T, V> rv, dr;
      if (res) rv = *(const Vec<T, V>*)(res + at);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float xh = a.xhat(to_float(xv.e[v]), v);
        float z = xh * a.ga[v] + a.be[v];
        if (res) z += to_float(rv.e[v]);
        const float dz = act_bwd<T, ACT>(to_float(dv.e[v]), z);
        sz[v] += dz;
        sx[v] += dz * xh;
        dr.e[v] = from_float<T>(dz);
      }
      if (dres) *(Vec<T, V>*)(dres + at) = dr;
    }
  }
  rows_to_waves<V>(sz, s.lanes, p.col, part[0]);
  rows_to_waves<V>(sx, s.lanes, p.col, part[1]);
  __syncthreads();
  for (int c = threadIdx.x; c < tile; c += NT) {
    const int cc = p.tile * tile + c;
    if (cc < s.C)
      ws[(p.n * s.S + p.chunk) * s.C + cc] =
          make_float2(over_waves(part[0], tile, c), over_waves(part[1], tile, c));
  }
}

// avg(dz*gamma), avg(dz*gamma*xhat), a block a group
__global__ __launch_bounds__(NT) void gn_join_sums_kernel(const float2* __restrict__ ws, Shape s,
                                                          int64_t all,
                                                          const void* __restrict__ gamma, bool wf,
                                                          float2* __restrict__ avg) {
  __shared__ float lds[NW];
  const int64_t entries = (int64_t)s.S * s.Cg;
  for (int64_t b = blockIdx.x; b < all; b += gridDim.x) {
    const int g = (int)(b % s.G);
    const float2* w = ws + b / s.G * s.S * s.C + g * s.Cg;
    float sz = 0.f, sx = 0.f;
    for (int64_t e = threadIdx.x; e < entries; e += NT) {
      const int64_t k = e / s.Cg;
      const int c = (int)(e % s.Cg);
      const float2 q = w[k * s.C + c];
      const float ga = load_param(gamma, g * s.Cg + c, wf, 1.f);
      sz += q.x * ga;
      sx += q.y * ga;
    }
    const float inv = 1.f / ((float)s.R * (float)s.Cg);
    sz = block_sum(sz, lds) * inv;
    sx = block_sum(sx, lds) * inv;
    if (threadIdx.x == 0) avg[b] = make_float2(sz, sx);
  }
}

template <typename T, int V, int ACT>
__global__ __launch_bounds__(NT) void gn_bwd_dx_kernel(
    const T* __restrict__ x, const T* __restrict__ dy, const T* __restrict__ res, Shape s,
    const float* __restrict__ mean, const float* __restrict__ rstd, const float2* __restrict__ avg,
    const void* __restrict__ gamma, const void* __restrict__ beta, bool wf, T* __restrict__ dx) {
  const Place p = place_of<V>(s);
  if (!p.active) return;
  Affine<V> a;
  a.load(s, p, mean, rstd, gamma, beta, wf);
  float2 m[V];
#pragma unroll
  for (int v = 0; v < V; ++v) m[v] = avg[p.n * s.G + (p.c + v) / s.Cg];
#pragma unroll
  for (int i = 0; i < K; ++i) {
    const int64_t r = p.lane_row + i * p.step;
    if (r >= p.rows) break;
    const int64_t at = (p.n * s.R + p.row0 + r) * s.C + p.c;
    const Vec<T, V> xv = *(const Vec<T, V>*)(x + at);
    const Vec<T, V> dv = *(const Vec<T, V>*)(dy + at);
    Vec<T, V> rv, out;
    if (res) rv = *(const Vec<T, V>*)(res + at);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float xh = a.xhat(to_float(xv.e[v]), v);
      float z = xh * a.ga[v] + a.be[v];
      if (res) z += to_float(rv.e[v]);
      const float dz = act_bwd<T, ACT>(to_float(dv.e[v]), z);
      out.e[v] = from_float<T>(a.rs[v] * (dz * a.ga[v] - m[v].x - xh * m[v].y));
    }
    *(Vec<T, V>*)(dx + at) = out;
  }
}

// dgamma, dbeta: 64 channels a block, its waves over the rows of ws [rows, C]
__global__ __launch_bounds__(1024) void gn_bwd_params_kernel(const float2* __restrict__ ws,
                                                             int64_t rows, int C, bool wf,
                                                             void* __restrict__ dgamma,
                                                             void* __restrict__ dbeta) {
  __shared__ float2 lds[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c = blockIdx.x * 64 + lane;
  float sz = 0.f, sx = 0.f;
  if (c < C) {
    for (int64_t r = wave; r < rows; r += 16) {
      const float2 q = ws[r * C + c];
      sz += q.x;
      sx += q.y;
    }
  }
  lds[wave][lane] = make_float2(sz, sx);
  __syncthreads();
  if (wave == 0 && c < C) {
    for (int w = 1; w < 16; ++w) {
      sz += lds[w][lane].x;
      sx += lds[w][lane].y;
    }
    if (dgamma) store_param(dgamma, c, wf, sx);
    if (dbeta) store_param(dbeta, c, wf, sz);
  }
}

// --------------------------------------------- a tile of groups in registers
//
// Where all pixels of some whole groups fit into a block's registers, the block reads them once:
// it has their mean, their variance and the result (going back: the sums and dx) without looking at
// memory again. Blocks that share lines of memory, the tiles of one sample, run on one XCD.
struct Tile {
  int64_t R;
  int C, G, Cg;
  int groups;     // of the tile
  int lanes;      // log2 of the lanes along the channels, the last of which may be idle
  int tiles;      // of a sample
  int64_t blocks;
  unsigned int magic;  // for division by Cg
  bool params;         // gamma and beta lie on 16 bytes
};

constexpr int MAX_WAVES = 16;
constexpr int MAX_CHANNELS = 512;
constexpr int FWD_ROWS = 16, BWD_ROWS = 14;  // of a thread, at most

struct Spot {
  int64_t n;
  int tile, c0, col, row, step;  // first channel; the lane's first in the tile; first row, rows a pass
  bool active;
};

template <int V>
__device__ __forceinline__ Spot spot_of(const Tile& t) {
  Spot p;
  const int64_t each = t.blocks / 8, rest = t.blocks % 8, x = blockIdx.x % 8;
  const int64_t b = x * each + min(x, rest) + blockIdx.x / 8;
  p.n = b / t.tiles;
  p.tile = (int)(b % t.tiles);
  p.c0 = p.tile * t.groups * t.Cg;
  p.col = (threadIdx.x & ((1 << t.lanes) - 1)) * V;
  p.row = threadIdx.x >> t.lanes;
  p.step = blockDim.x >> t.lanes;
  p.active = p.col < t.groups * t.Cg;
  return p;
}

// Sums of `part` [waves][pitch] over the waves and the channels of each group: a row of 16 lanes a
// group, each lane over every 16th of its values.
__device__ __forceinline__ void over_groups(const float* part, const Tile& t, int pitch, float* to) {
  const int waves = blockDim.x >> 6, lane = threadIdx.x & 15, entries = waves * t.Cg;
  for (int g = threadIdx.x >> 4; g < t.groups; g += blockDim.x >> 4) {
    float s = 0.f;
    for (int e = lane; e < entries; e += 16) {
      const int w = divided(e, t.magic);
      s += part[w * pitch + g * t.Cg + e - w * t.Cg];
    }
    s += moved<0x128>(s);
    s += moved<0x124>(s);
    s += moved<0x4E>(s);
    s += moved<0xB1>(s);
    if (lane == 0) to[g] = s;
  }
}

// The tile's means and 1/deviations, to memory and the latter to `spread` in the sums' place.
__device__ __forceinline__ void tell_groups(const Tile& t, const Spot& p, float inv, float eps,
                                            const float* group, float* spread, float* mean, float* rstd) {
  for (int i = threadIdx.x; i < t.groups; i += blockDim.x) {
    const int64_t at = p.n * t.G + p.tile * t.groups + i;
    const float r = 1.f / sqrtf(spread[i] * inv + eps);
    mean[at] = group[i] * inv;
    rstd[at] = r;
    spread[i] = r;
  }
  __syncthreads();
}

template <typename T, int V, int ACT, int KR>
__global__ __launch_bounds__(1024) void gn_tile_kernel(
    const T* __restrict__ x, const T* __restrict__ res, Tile t, float eps, const void* __restrict__ gamma,
    const void* __restrict__ beta, bool wf, T* __restrict__ y, float* __restrict__ mean,
    float* __restrict__ rstd) {
  __shared__ float part[MAX_WAVES * 64 * V];
  __shared__ float group[MAX_CHANNELS], spread[MAX_CHANNELS];
  const Spot p = spot_of<V>(t);
  const int pitch = V << t.lanes;
  const float inv = 1.f / ((float)t.R * (float)t.Cg);
  const int64_t first = (p.n * t.R + p.row) * t.C + p.c0 + p.col, stride = (int64_t)p.step * t.C;
  int g[V];
#pragma unroll
  for (int v = 0; v < V; ++v) g[v] = p.active ? divided(p.col + v, t.magic) : 0;
  Packed<T, V> val[KR];
  float acc[V] = {}, ga[V], be[V];
#pragma unroll
  for (int i = 0; i < KR; ++i)
    if (p.active && p.row + i * p.step < t.R) val[i].load(x + first + i * stride);
  if (p.active) {
    load_params<V>(gamma, p.c0 + p.col, wf, t.params, 1.f, ga);
    load_params<V>(beta, p.c0 + p.col, wf, t.params, 0.f, be);
  }
#pragma unroll
  for (int i = 0; i < KR; ++i)
    if (p.active && p.row + i * p.step < t.R) {
#pragma unroll
      for (int v = 0; v < V; ++v) acc[v] += val[i].get(v);
    }
  rows_to_waves<V>(acc, t.lanes, p.col / V, part);
  __syncthreads();
  over_groups(part, t, pitch, group);
  __syncthreads();
  float mu[V];
#pragma unroll
  for (int v = 0; v < V; ++v) mu[v] = group[g[v]] * inv, acc[v] = 0.f;
#pragma unroll
  for (int i = 0; i < KR; ++i)
    if (p.active && p.row + i * p.step < t.R) {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float d = val[i].get(v) - mu[v];
        acc[v] += d * d;
      }
    }
  rows_to_waves<V>(acc, t.lanes, p.col / V, part);
  __syncthreads();
  over_groups(part, t, pitch, spread);
  __syncthreads();
  tell_groups(t, p, inv, eps, group, spread, mean, rstd);
  if (!p.active) return;
#pragma unroll
  for (int v = 0; v < V; ++v) ga[v] *= spread[g[v]];
#pragma unroll
  for (int i = 0; i < KR; ++i)
    if (p.row + i * p.step < t.R) {
      Packed<T, V> r = {}, o;
      if (res) r.load(res + first + i * stride);
      float z[V];
#pragma unroll
      for (int v = 0; v < V; ++v)
        z[v] = act_fwd<T, ACT>((val[i].get(v) - mu[v]) * ga[v] + be[v] + r.get(v));
#pragma unroll
      for (int v = 0; v < V / 2; ++v) o.set2(v, z[2 * v], z[2 * v + 1]);
      o.store(y + first + i * stride);
    }
}

// The block's sums of dz and dz * xhat: to ws, a sample's part of the parameters' gradients, and times
// gamma over each group to `group`.
template <int V>
__device__ __forceinline__ void join_sums(float (&sz)[V], float (&sx)[V], const Tile& t, const Spot& p,
                                          const void* gamma, bool wf, float* part_z, float* part_x,
                                          float (*group)[MAX_CHANNELS], float2* ws, bool groups) {
  const int pitch = V << t.lanes, waves = blockDim.x >> 6;
  rows_to_waves<V>(sz, t.lanes, p.col / V, part_z);
  rows_to_waves<V>(sx, t.lanes, p.col / V, part_x);
  __syncthreads();
  for (int c = threadIdx.x; c < t.groups * t.Cg; c += blockDim.x) {
    float z = 0.f, xs = 0.f;
    for (int w = 0; w < waves; ++w) {
      z += part_z[w * pitch + c];
      xs += part_x[w * pitch + c];
    }
    ws[p.n * t.C + p.c0 + c] = make_float2(z, xs);
    const float a = load_param(gamma, p.c0 + c, wf, 1.f);
    part_z[c] = z * a;  // nobody else reads this place
    part_x[c] = xs * a;
  }
  if (!groups) return;
  __syncthreads();
  const int lane = threadIdx.x & 15;
  for (int k = threadIdx.x >> 4; k < t.groups; k += blockDim.x >> 4) {
    float z = 0.f, xs = 0.f;
    for (int c = lane; c < t.Cg; c += 16) {
      z += part_z[k * t.Cg + c];
      xs += part_x[k * t.Cg + c];
    }
    z += moved<0x128>(z), xs += moved<0x128>(xs);
    z += moved<0x124>(z), xs += moved<0x124>(xs);
    z += moved<0x4E>(z), xs += moved<0x4E>(xs);
    z += moved<0xB1>(z), xs += moved<0xB1>(xs);
    if (lane == 0) group[0][k] = z, group[1][k] = xs;
  }
  __syncthreads();
}

template <typename T, int V, int ACT, int KR>
__global__ __launch_bounds__(512) void gn_tile_bwd_kernel(
    const T* __restrict__ x, const T* __restrict__ dy, const T* __restrict__ res, Tile t,
    const float* __restrict__ mean, const float* __restrict__ rstd, const void* __restrict__ gamma,
    const void* __restrict__ beta, bool wf, T* __restrict__ dx, T* __restrict__ dres,
    float2* __restrict__ ws) {
  __shared__ float part[2][8 * 64 * V];
  __shared__ float group[2][MAX_CHANNELS];
  const Spot p = spot_of<V>(t);
  const int64_t first = (p.n * t.R + p.row) * t.C + p.c0 + p.col, stride = (int64_t)p.step * t.C;
  // x as it lies in memory, and where dy was, dz in fp32: the activation is gone through once
  Packed<T, V> xv[KR];
  float dz[KR][V];
#pragma unroll
  for (int i = 0; i < KR; ++i)
    if (p.active && p.row + i * p.step < t.R) {
      xv[i].load(x + first + i * stride);
      Packed<T, V> d;
      d.load(dy + first + i * stride);
#pragma unroll
      for (int v = 0; v < V; ++v) dz[i][v] = d.get(v);
    }
  int g[V];
  float mu[V], rs[V], ga[V], sz[V] = {}, sx[V] = {};
  {
    float be[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      g[v] = p.active ? divided(p.col + v, t.magic) : 0;
      const int64_t at = p.n * t.G + p.tile * t.groups + g[v];
      mu[v] = mean[at];
      rs[v] = rstd[at];
    }
    if (p.active) {
      load_params<V>(gamma, p.c0 + p.col, wf, t.params, 1.f, ga);
      load_params<V>(beta, p.c0 + p.col, wf, t.params, 0.f, be);
    }
#pragma unroll
    for (int i = 0; i < KR; ++i)
      if (p.active && p.row + i * p.step < t.R) {
        Packed<T, V> r = {}, o;
        if (res) r.load(res + first + i * stride);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float xh = (xv[i].get(v) - mu[v]) * rs[v];
          dz[i][v] = act_bwd<T, ACT>(dz[i][v], xh * ga[v] + be[v] + r.get(v));
          sz[v] += dz[i][v];
          sx[v] += dz[i][v] * xh;
        }
        if (dres) {
#pragma unroll
          for (int v = 0; v < V / 2; ++v) o.set2(v, dz[i][2 * v], dz[i][2 * v + 1]);
          o.store(dres + first + i * stride);
        }
      }
  }
  join_sums<V>(sz, sx, t, p, gamma, wf, part[0], part[1], group, ws, dx != nullptr);
  if (!dx || !p.active) return;
  // dx = rs*ga * dz - rs*rs*avg(dz*ga*xhat) * (x - mu) - rs*avg(dz*ga)
  const float inv = 1.f / ((float)t.R * (float)t.Cg);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    sz[v] = rs[v] * (group[0][g[v]] * inv);
    sx[v] = rs[v] * rs[v] * (group[1][g[v]] * inv);
    ga[v] *= rs[v];
  }
#pragma unroll
  for (int i = 0; i < KR; ++i)
    if (p.row + i * p.step < t.R) {
      Packed<T, V> o;
#pragma unroll
      for (int v = 0; v < V; ++v)
        dz[i][v] = dz[i][v] * ga[v] - (xv[i].get(v) - mu[v]) * sx[v] - sz[v];
#pragma unroll
      for (int v = 0; v < V / 2; ++v) o.set2(v, dz[i][2 * v], dz[i][2 * v + 1]);
      o.store(dx + first + i * stride);
    }
}

// Groups of more pixels than registers hold: the block goes over its rows twice. A thread's mean and
// variance grow by four rows at a time, each four around their own mean, and are joined by counts.
template <typename T, int V, int ACT>
__global__ __launch_bounds__(512, 4) void gn_stream_kernel(
    const T* __restrict__ x, const T* __restrict__ res, Tile t, float eps, const void* __restrict__ gamma,
    const void* __restrict__ beta, bool wf, T* __restrict__ y, float* __restrict__ mean,
    float* __restrict__ rstd) {
  constexpr int KR = 4;
  __shared__ float part[8 * 64 * V];
  __shared__ float group[MAX_CHANNELS], spread[MAX_CHANNELS];
  const Spot p = spot_of<V>(t);
  const int pitch = V << t.lanes;
  const float inv = 1.f / ((float)t.R * (float)t.Cg);
  const int64_t first = (p.n * t.R + p.row) * t.C + p.c0 + p.col, stride = (int64_t)p.step * t.C;
  float mu[V] = {}, m2[V] = {}, seen = 0.f;
  if (p.active)
    for (int64_t r = p.row, at = first; r < t.R; r += KR * p.step, at += KR * stride) {
      Packed<T, V> val[KR];
#pragma unroll
      for (int i = 0; i < KR; ++i)
        if (r + i * p.step < t.R) val[i].load(x + at + i * stride);
      const float n = (float)min((int64_t)KR, (t.R - r + p.step - 1) / p.step);
      const float share = 1.f / n, all = 1.f / (seen + n);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float s = 0.f, q = 0.f;
#pragma unroll
        for (int i = 0; i < KR; ++i)
          if (r + i * p.step < t.R) s += val[i].get(v);
        s *= share;
#pragma unroll
        for (int i = 0; i < KR; ++i)
          if (r + i * p.step < t.R) {
            const float d = val[i].get(v) - s;
            q += d * d;
          }
        const float d = s - mu[v];
        mu[v] += d * (n * all);
        m2[v] += q + d * d * (seen * n * all);
      }
      seen += n;
    }
  float acc[V];
#pragma unroll
  for (int v = 0; v < V; ++v) acc[v] = mu[v] * seen;
  rows_to_waves<V>(acc, t.lanes, p.col / V, part);
  __syncthreads();
  over_groups(part, t, pitch, group);
  __syncthreads();
  int g[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    g[v] = p.active ? divided(p.col + v, t.magic) : 0;
    const float d = mu[v] - group[g[v]] * inv;
    acc[v] = m2[v] + d * d * seen;
  }
  rows_to_waves<V>(acc, t.lanes, p.col / V, part);
  __syncthreads();
  over_groups(part, t, pitch, spread);
  __syncthreads();
  tell_groups(t, p, inv, eps, group, spread, mean, rstd);
  if (!p.active) return;
  float be[V];
  load_params<V>(gamma, p.c0 + p.col, wf, t.params, 1.f, m2);
  load_params<V>(beta, p.c0 + p.col, wf, t.params, 0.f, be);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    mu[v] = group[g[v]] * inv;
    m2[v] *= spread[g[v]];
  }
  for (int64_t r = p.row, at = first; r < t.R; r += KR * p.step, at += KR * stride) {
    Packed<T, V> val[KR], rv[KR] = {};
#pragma unroll
    for (int i = 0; i < KR; ++i)
      if (r + i * p.step < t.R) {
        val[i].load(x + at + i * stride);
        if (res) rv[i].load(res + at + i * stride);
      }
#pragma unroll
    for (int i = 0; i < KR; ++i)
      if (r + i * p.step < t.R) {
        float z[V];
#pragma unroll
        for (int v = 0; v < V; ++v)
          z[v] = act_fwd<T, ACT>((val[i].get(v) - mu[v]) * m2[v] + be[v] + rv[i].get(v));
#pragma unroll
        for (int v = 0; v < V / 2; ++v) val[i].set2(v, z[2 * v], z[2 * v + 1]);
        val[i].store(y + at + i * stride);
      }
  }
}

// And back: the sums, then dx, the second time while the caches still have some of the rows.
template <typename T, int V, int ACT>
__global__ __launch_bounds__(512, 4) void gn_stream_bwd_kernel(
    const T* __restrict__ x, const T* __restrict__ dy, const T* __restrict__ res, Tile t,
    const float* __restrict__ mean, const float* __restrict__ rstd, const void* __restrict__ gamma,
    const void* __restrict__ beta, bool wf, T* __restrict__ dx, T* __restrict__ dres,
    float2* __restrict__ ws) {
  constexpr int KR = 2;
  __shared__ float part[2][8 * 64 * V];
  __shared__ float group[2][MAX_CHANNELS];
  const Spot p = spot_of<V>(t);
  const int64_t first = (p.n * t.R + p.row) * t.C + p.c0 + p.col, stride = (int64_t)p.step * t.C;
  int g[V];
  float mu[V], rs[V], ga[V], be[V], sz[V] = {}, sx[V] = {};
#pragma unroll
  for (int v = 0; v < V; ++v) {
    g[v] = p.active ? divided(p.col + v, t.magic) : 0;
    const int64_t at = p.n * t.G + p.tile * t.groups + g[v];
    mu[v] = mean[at];
    rs[v] = rstd[at];
  }
  if (p.active) {
    load_params<V>(gamma, p.c0 + p.col, wf, t.params, 1.f, ga);
    load_params<V>(beta, p.c0 + p.col, wf, t.params, 0.f, be);
  }
  // `with` gets each vector's place, xhat and dz
  const auto rows = [&](auto with) {
    if (!p.active) return;
    for (int64_t r = p.row, at = first; r < t.R; r += KR * p.step, at += KR * stride) {
      Packed<T, V> xv[KR], dv[KR], rv[KR] = {};
#pragma unroll
      for (int i = 0; i < KR; ++i)
        if (r + i * p.step < t.R) {
          xv[i].load(x + at + i * stride);
          dv[i].load(dy + at + i * stride);
          if (res) rv[i].load(res + at + i * stride);
        }
#pragma unroll
      for (int i = 0; i < KR; ++i)
        if (r + i * p.step < t.R) {
          float xh[V], dz[V];
#pragma unroll
          for (int v = 0; v < V; ++v) {
            xh[v] = (xv[i].get(v) - mu[v]) * rs[v];
            dz[v] = act_bwd<T, ACT>(dv[i].get(v), xh[v] * ga[v] + be[v] + rv[i].get(v));
          }
          with(at + i * stride, xh, dz);
        }
    }
  };
  rows([&](int64_t at, const float (&xh)[V], const float (&dz)[V]) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      sz[v] += dz[v];
      sx[v] += dz[v] * xh[v];
    }
    if (dres) {
      Packed<T, V> o;
#pragma unroll
      for (int v = 0; v < V / 2; ++v) o.set2(v, dz[2 * v], dz[2 * v + 1]);
      o.store(dres + at);
    }
  });
  join_sums<V>(sz, sx, t, p, gamma, wf, part[0], part[1], group, ws, dx != nullptr);
  if (!dx) return;
  const float inv = 1.f / ((float)t.R * (float)t.Cg);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    sz[v] = group[0][g[v]] * inv;
    sx[v] = group[1][g[v]] * inv;
  }
  rows([&](int64_t at, const float (&xh)[V], const float (&dz)[V]) {
    Packed<T, V> o;
    float d[V];
#pragma unroll
    for (int v = 0; v < V; ++v) d[v] = rs[v] * (dz[v] * ga[v] - sz[v] - xh[v] * sx[v]);
#pragma unroll
    for (int v = 0; v < V / 2; ++v) o.set2(v, d[2 * v], d[2 * v + 1]);
    o.store(dx + at);
  });
}

// ------------------------------------------------------------------ host
struct Image {
  int64_t N, R;
  int C;
};

Image image_of(const Tensor& x) {
  return {x.size(0), x.dim() == 4 ? x.size(2) * x.size(3) : 1, (int)x.size(1)};
}

Tensor channels_last(const Tensor& t) {
  return t.dim() == 4 ? t.contiguous(at::MemoryFormat::ChannelsLast) : t.contiguous();
}

Tensor like(const Tensor& t) {
  return at::empty_like(
      t, t.options(), t.dim() == 4 ? at::MemoryFormat::ChannelsLast : at::MemoryFormat::Contiguous);
}

void check_args(const Tensor& x, int64_t groups, const Tensor& w, const Tensor& b, const Tensor& res,
                int64_t act) {
  TORCH_CHECK(x.is_cuda() && is_float_type(x), "group_norm_act: x must be fp32 or bf16 on a GPU");
  TORCH_CHECK(x.dim() == 2 || x.dim() == 4, "group_norm_act: x must be [N, C] or [N, C, H, W]");
  const int64_t C = x.size(1);
  TORCH_CHECK(groups > 0 && C > 0 && C % groups == 0 && C < (1 << 24),
              "group_norm_act: num_groups must divide the channels");
  TORCH_CHECK(act >= 0 && act <= 3, "group_norm_act: unknown activation");
  for (const Tensor* p : {&w, &b}) {
    if (!p->defined()) continue;
    TORCH_CHECK(p->device() == x.device() && p->dim() == 1 && p->size(0) == C,
                "group_norm_act: weight and bias must be [C] on x's device");
    TORCH_CHECK(p->scalar_type() == at::kFloat || p->scalar_type() == x.scalar_type(),
                "group_norm_act: weight and bias must be fp32 or of x's type");
  }
  TORCH_CHECK(!w.defined() || !b.defined() || w.scalar_type() == b.scalar_type(),
              "group_norm_act: weight and bias must be of one type");
  if (res.defined())
    TORCH_CHECK(res.device() == x.device() && res.scalar_type() == x.scalar_type() &&
                    res.sizes() == x.sizes(),
                "group_norm_act: res must be like x");
}

bool aligned(std::initializer_list<const void*> ptrs, size_t to) {
  for (const void* p : ptrs)
    if ((uintptr_t)p % to) return false;
  return true;
}

// channels of one transaction: 16 bytes where the rows and all pointers allow it, else 8 or 4
// bytes (two values), else one value
int vector_of(int C, int64_t elem, std::initializer_list<const void*> ptrs) {
  for (int64_t v = 16 / elem; v > 1; v >>= 1)
    if (C % v == 0 && aligned(ptrs, v * elem)) return (int)v;
  return 1;
}

Shape shape_of(const Image& im, int64_t groups, int V) {
  Shape s;
  s.R = im.R;
  s.C = im.C;
  s.G = (int)groups;
  s.Cg = im.C / s.G;
  s.lanes = 0;
  while (s.lanes < 6 && (1 << s.lanes) * V < s.C) ++s.lanes;
  s.tiles = (int)ceil_div(s.C, (int64_t)(1 << s.lanes) * V);
  const int64_t S = ceil_div(s.R, (int64_t)(NT >> s.lanes) * K);
  grid_of(im.N * s.tiles * S, NT, "group_norm_act");
  s.S = (int)S;
  return s;
}

struct Plan {
  Tile t;
  int threads = 0;  // of a block; 0: chunks of rows for many blocks, statistics joined between kernels
  int rows = 0;     // of a thread; 0: any number, read twice
};

// Which groups a block takes, and whether it holds their pixels: as few idle lanes, as long pieces of
// memory and as many blocks as go together, by the penalties below. Measured, going back:
// 128x256x56x56 in bf16 250 us held, in pieces of 32 bytes, and 233 and 220 read twice in 128 and 256;
// 128x128x112x112 830 us by chunks, 600, 491 and 425 read twice in pieces of 32, 64 and 128;
// 64x256x28x28 33 us held in 128, 53 read twice. Forward, 64x64x32x32: 11.4 us in pieces of 32 bytes
// and 256 blocks, 13.5 in 16 and 512, 12.8 in 64 and 128; 128x256x56x56 141 held in 64, 198 in 32.
Plan plan_of(const Image& im, int64_t groups, int V, int64_t elem, bool params, int max_threads, int most,
             double twice) {
  Plan best;
  double least = 1e30;
  const int G = (int)groups, Cg = im.C / G;
  if (V * elem < 8) return best;
  for (int k = 1; k <= G; ++k) {
    const int c = k * Cg;
    if (G % k || c % V || c > MAX_CHANNELS || c > 64 * V) continue;
    int lanes = 0;
    while ((1 << lanes) * V < c) ++lanes;
    const int64_t blocks = im.N * (G / k);
    if (blocks * max_threads >= (1LL << 32)) continue;
    // four rows a thread keep enough loads on their way; `most` are what registers hold
    int threads = 64;
    while (threads < max_threads && (threads >> lanes) * 4 < im.R) threads *= 2;
    int rows = (int64_t)(threads >> lanes) * 4 >= im.R ? 4 : (int64_t)(threads >> lanes) * most >= im.R ? most : 0;
    const double piece = c * elem, idle = (double)(V << lanes) / c;
    const double cost = idle * (piece >= 128 ? 1.0 : piece >= 64 ? 1.05 : piece >= 32 ? 1.3 : 1.8) *
                        std::max(1.0, 256.0 / blocks) * (rows ? 1.0 : twice);
    if (cost < least) {
      least = cost;
      best.t = {im.R, im.C, G, Cg, k, lanes, G / k, blocks, magic_of(Cg), params};
      best.threads = rows ? threads : 512;
      best.rows = rows;
    }
  }
  // few blocks with much to read: one image of 64x256x256 in bf16 would be 8 blocks of a megabyte
  if (best.threads && best.t.blocks < 128 && im.N * im.R * im.C * elem / best.t.blocks > (256 << 10))
    best.threads = 0;
  return best;
}

// kernels for vectors of 8 bytes and more, 4 or 16 rows a thread
#define GN_DISPATCH_ROWS(ROWS, MOST, ...)                         \
  if ((ROWS) == 4) { constexpr int KR = 4; __VA_ARGS__; }         \
  else if ((ROWS) == (MOST)) { constexpr int KR = MOST; __VA_ARGS__; } \
  else { constexpr int KR = 0; __VA_ARGS__; }
#define GN_DISPATCH_TILE(V_VALUE, ROWS, MOST, ...)                                                       \
  switch (V_VALUE) {                                                                                     \
    case 8: { constexpr int V = sizeof(T) == 2 ? 8 : 4; GN_DISPATCH_ROWS(ROWS, MOST, __VA_ARGS__) } break; \
    case 4: { constexpr int V = 4; GN_DISPATCH_ROWS(ROWS, MOST, __VA_ARGS__) } break;                    \
    default: { constexpr int V = sizeof(T) == 2 ? 4 : 2; GN_DISPATCH_ROWS(ROWS, MOST, __VA_ARGS__) }      \
  }

template <typename T, int V, int ACT, int KR>
auto tile_of() {
  if constexpr (KR) return &gn_tile_kernel<T, V, ACT, KR>;
  else return &gn_stream_kernel<T, V, ACT>;
}
template <typename T, int V, int ACT, int KR>
auto tile_bwd_of() {
  if constexpr (KR) return &gn_tile_bwd_kernel<T, V, ACT, KR>;
  else return &gn_stream_bwd_kernel<T, V, ACT>;
}

#define GN_DISPATCH_VEC(V_VALUE, ...)                                      \
  switch (V_VALUE) {                                                       \
    case 8: { constexpr int V = sizeof(T) == 2 ? 8 : 4; __VA_ARGS__; } break; \
    case 4: { constexpr int V = 4; __VA_ARGS__; } break;                   \
    case 2: { constexpr int V = 2; __VA_ARGS__; } break;                   \
    default: { constexpr int V = 1; __VA_ARGS__; } break;                  \
  }

const void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

struct Forward {
  Tensor y, x, w, b, res, mean, rstd;  // the result, and what the backward pass reads
};

void normalise(Forward& f, int64_t groups, double eps, int64_t act) {
  const Tensor &x = f.x, &w = f.w, &b = f.b, &res = f.res;
  const Image im = image_of(x);
  Tensor& y = f.y = like(x);
  Tensor& mean = f.mean = at::empty({im.N, groups}, x.options().dtype(at::kFloat));
  Tensor& rstd = f.rstd = at::empty_like(mean);
  if (x.numel() == 0) return;
  const bool wf = (w.defined() ? w : b.defined() ? b : x).scalar_type() == at::kFloat;
  const int vec = vector_of(im.C, x.element_size(), {ptr(x), ptr(res), ptr(y)});
  const hipStream_t st = stream_of(x);
  const Plan plan = plan_of(im, groups, vec, x.element_size(), aligned({ptr(w), ptr(b)}, 16), 1024, FWD_ROWS, 1.5);
  if (plan.threads) {
    MM_DISPATCH_TYPE(x, GN_DISPATCH_TILE(vec, plan.rows, FWD_ROWS, MM_DISPATCH_ACT(act, (
        tile_of<T, V, ACT, KR>()<<<(unsigned)plan.t.blocks, plan.threads, 0, st>>>(
            (const T*)ptr(x), (const T*)ptr(res), plan.t, (float)eps, ptr(w), ptr(b), wf,
            (T*)y.data_ptr(), mean.data_ptr<float>(), rstd.data_ptr<float>())))));
    check_launch("group_norm_act");
    return;
  }
  const Shape s = shape_of(im, groups, vec);
  Tensor ws = at::empty({im.N * s.S * s.C * 2}, mean.options());
  const unsigned blocks = (unsigned)(im.N * s.tiles * s.S);
  MM_DISPATCH_TYPE(x, GN_DISPATCH_VEC(vec, {
    gn_stats_kernel<T, V><<<blocks, NT, 0, st>>>((const T*)ptr(x), s, (float2*)ws.data_ptr());
    gn_join_stats_kernel<<<(unsigned)std::min<int64_t>(im.N * groups, 1 << 20), NT, 0, st>>>(
        (const float2*)ws.data_ptr(), s, im.N * groups, (float)eps, mean.data_ptr<float>(), rstd.data_ptr<float>());
    MM_DISPATCH_ACT(act, (gn_apply_kernel<T, V, ACT><<<blocks, NT, 0, st>>>(
        (const T*)ptr(x), (const T*)ptr(res), s, mean.data_ptr<float>(), rstd.data_ptr<float>(),
        ptr(w), ptr(b), wf, (T*)y.data_ptr())));
  }));
  check_launch("group_norm_act");
}

struct Grads {
  Tensor dx, dw, db, dres;
};

Grads backward_of(const Tensor& dy, const Tensor& x, int64_t groups, const Tensor& w,
                  const Tensor& b, int64_t act, const Tensor& res, const Tensor& mean,
                  const Tensor& rstd, bool need_dx, bool need_dw, bool need_db, bool need_dres) {
  const Image im = image_of(x);
  Grads g;
  if (need_dx) g.dx = like(x);
  if (need_dw) g.dw = at::empty_like(w);
  if (need_db) g.db = at::empty_like(b);
  if (need_dres) g.dres = like(x);
  if (x.numel() == 0) {
    if (need_dw) g.dw.zero_();
    if (need_db) g.db.zero_();
    return g;
  }
  const bool wf = (w.defined() ? w : b.defined() ? b : x).scalar_type() == at::kFloat;
  const int vec = vector_of(im.C, x.element_size(),
                            {ptr(x), ptr(dy), ptr(res), ptr(g.dx), ptr(g.dres)});
  const hipStream_t st = stream_of(x);
  const Plan plan = plan_of(im, groups, vec, x.element_size(), aligned({ptr(w), ptr(b)}, 16), 512, BWD_ROWS, 1.15);
  Tensor ws;
  int64_t rows;  // of ws: what each sample, or each chunk of it, adds to the parameters' gradients
  if (plan.threads) {
    ws = at::empty({im.N * im.C * 2}, mean.options());
    rows = im.N;
    MM_DISPATCH_TYPE(x, GN_DISPATCH_TILE(vec, plan.rows, BWD_ROWS, MM_DISPATCH_ACT(act, (
        tile_bwd_of<T, V, ACT, KR>()<<<(unsigned)plan.t.blocks, plan.threads, 0, st>>>(
            (const T*)ptr(x), (const T*)ptr(dy), (const T*)ptr(res), plan.t, mean.data_ptr<float>(),
            rstd.data_ptr<float>(), ptr(w), ptr(b), wf, (T*)ptr(g.dx), (T*)ptr(g.dres),
            (float2*)ws.data_ptr())))));
  } else {
    const Shape s = shape_of(im, groups, vec);
    ws = at::empty({im.N * s.S * s.C * 2}, mean.options());
    rows = im.N * s.S;
    Tensor avg = at::empty({im.N * groups * 2}, mean.options());
    const unsigned blocks = (unsigned)(im.N * s.tiles * s.S);
  MM_DISPATCH_TYPE(x, GN_DISPATCH_VEC(vec, {
    MM_DISPATCH_ACT(act, (gn_bwd_sums_kernel<T, V, ACT><<<blocks, NT, 0, st>>>(
        (const T*)ptr(x), (const T*)ptr(dy), (const T*)ptr(res), s, mean.data_ptr<float>(),
        rstd.data_ptr<float>(), ptr(w), ptr(b), wf, (T*)ptr(g.dres), (float2*)ws.data_ptr())));
    if (need_dx) {
      gn_join_sums_kernel<<<(unsigned)std::min<int64_t>(im.N * groups, 1 << 20), NT, 0, st>>>(
          (const float2*)ws.data_ptr(), s, im.N * groups, ptr(w), wf, (float2*)avg.data_ptr());
      MM_DISPATCH_ACT(act, (gn_bwd_dx_kernel<T, V, ACT><<<blocks, NT, 0, st>>>(
          (const T*)ptr(x), (const T*)ptr(dy), (const T*)ptr(res), s, mean.data_ptr<float>(),
          rstd.data_ptr<float>(), (const float2*)avg.data_ptr(), ptr(w), ptr(b), wf,
          (T*)g.dx.data_ptr())));
    }
  }));
  }
  if (need_dw || need_db)
    gn_bwd_params_kernel<<<(unsigned)ceil_div(im.C, 64), 1024, 0, st>>>(
        (const float2*)ws.data_ptr(), rows, im.C, wf, (void*)ptr(g.dw), (void*)ptr(g.db));
  check_launch("group_norm_act backward");
  return g;
}

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }

Forward forward_of(const Tensor& x, const Tensor& w, const Tensor& b, const Tensor& res,
                   int64_t groups, double eps, int64_t act) {
  Forward f;
  f.x = channels_last(x);
  f.w = w.defined() ? w.contiguous() : w;
  f.b = b.defined() ? b.contiguous() : b;
  f.res = res.defined() ? channels_last(res) : res;
  normalise(f, groups, eps, act);
  return f;
}

class GroupNormAct : public torch::autograd::Function<GroupNormAct> {
 public:
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& weight,
                        const OptTensor& bias, const OptTensor& residual, int64_t groups,
                        double eps, int64_t act) {
    at::AutoDispatchBelowADInplaceOrView guard;
    const Tensor w = weight.value_or(Tensor()), b = bias.value_or(Tensor()),
                 res = residual.value_or(Tensor());
    const Forward f = forward_of(x, w, b, res, groups, eps, act);
    // without an activation the backward pass never looks at the residual
    ctx->save_for_backward(
        {f.x, f.w, f.b, act == ACT_NONE ? Tensor() : f.res, f.mean, f.rstd});
    ctx->saved_data["groups"] = groups;
    ctx->saved_data["act"] = act;
    ctx->saved_data["needs"] = (int64_t)(x.requires_grad() | wants_grad(w) << 1 |
                                         wants_grad(b) << 2 | wants_grad(res) << 3);
    return f.y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(),
                "group_norm_act has no second derivative (create_graph=True)");
    const auto saved = ctx->get_saved_variables();
    const int64_t needs = ctx->saved_data["needs"].toInt();
    const c10::DeviceGuard guard(saved[0].device());
    Grads g = backward_of(channels_last(grads[0]), saved[0], ctx->saved_data["groups"].toInt(),
                          saved[1], saved[2], ctx->saved_data["act"].toInt(), saved[3], saved[4],
                          saved[5], needs & 1, needs & 2, needs & 4, needs & 8);
    return {g.dx, g.dw, g.db, g.dres, Tensor(), Tensor(), Tensor()};
  }
};

Tensor group_norm_act(const Tensor& x, int64_t groups, const OptTensor& weight,
                      const OptTensor& bias, double eps, int64_t act, const OptTensor& residual) {
  const Tensor w = weight.value_or(Tensor()), b = bias.value_or(Tensor()),
               res = residual.value_or(Tensor());
  check_args(x, groups, w, b, res, act);
  refuse_forward_mode({&x, &w, &b, &res}, "group_norm_act");
  refuse_tracing("group_norm_act");
  const c10::DeviceGuard guard(x.device());
  if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(w) || wants_grad(b) || wants_grad(res)))
    return GroupNormAct::apply(x, weight, bias, residual, groups, eps, act);
  return forward_of(x, w, b, res, groups, eps, act).y;
}

}  // namespace

void bind_group_norm(pybind11::module_& m) {
  m.def("group_norm_act", &group_norm_act,
        "K16: channels-last group norm (+residual) (+activation), differentiable",
        py::arg("x"), py::arg("num_groups"), py::arg("weight") = py::none(),
        py::arg("bias") = py::none(), py::arg("eps") = 1e-5, py::arg("act") = 0,
        py::arg("res") = py::none());
}

}  // namespace mm
