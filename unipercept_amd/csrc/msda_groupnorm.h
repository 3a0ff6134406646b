// Group normalisation of a flattened pyramid (gfx950): x (N, S, C), channels last; every level is a
// run of rows of every sample with statistics of its own, an activation follows.
//
//   per (n, level, group): mu = mean x, s = 1 / sqrt(mean (x - mu)^2 + eps) over the level's rows
//   and the group's C / G channels;  u = (x - mu) * s,  z = u * w + b,  y = act(z)
//   with dz = dy * act'(z):  db = sum dz,  dw = sum dz * u  (over samples and rows),
//   dx = s * (w dz - m1 - u * m2),  m1 = mean (w dz),  m2 = mean (w dz u)  (over rows and group)
//
// A level's rows are cut into chunks, a workgroup each.  Threads lie along the channels (16 bytes a
// thread) and then along the rows, so a thread keeps its channels for the whole chunk and sums per
// channel in registers; groups are formed from channels once per chunk.  Two launches a direction:
// the first leaves partial sums per chunk, every workgroup of the second joins the partial sums of
// its level (the same numbers in the same order everywhere) and writes its chunk.
#pragma once

#include "msda_vec.h"

namespace msda {

enum GnAct { kGnNone = 0, kGnRelu = 1, kGnSilu = 2, kGnGelu = 3 };

struct GnLevels {
  int levels, chunks, rows_per_chunk, param_levels;
  int row_start[kMaxNormLevels + 1];
  int chunk_start[kMaxNormLevels + 1];
};

struct GnChunk {
  int level, rows;
  int64_t first_row;  // within the tensor
  int64_t n;
};

__device__ __forceinline__ GnChunk gn_chunk(const GnLevels& lv, int block) {
  GnChunk c;
  c.n = block / lv.chunks;
  const int chunk = block - static_cast<int>(c.n) * lv.chunks;
  c.level = 0;
  while (c.level + 1 < lv.levels && chunk >= lv.chunk_start[c.level + 1]) ++c.level;
  const int row = lv.row_start[c.level] + (chunk - lv.chunk_start[c.level]) * lv.rows_per_chunk;
  c.rows = min(lv.rows_per_chunk, lv.row_start[c.level + 1] - row);
  c.first_row = c.n * lv.row_start[lv.levels] + row;
  return c;
}

// rows of a chunk of `rows` that row lane r of `lanes` handles
__device__ __forceinline__ int gn_lane_rows(int rows, int r, int lanes) {
  return r < rows ? (rows - r + lanes - 1) / lanes : 0;
}

// (count, mean, M2) of a union of two sets (T. F. Chan, G. H. Golub, R. J. LeVeque 1979)
template <typename CT>
struct Moments {
  CT n, mean, m2;
  __device__ __forceinline__ void add(CT on, CT omean, CT om2) {
    const CT total = n + on;
    if (total > CT(0)) {
      const CT d = omean - mean, f = on / total;
      mean += d * f;
      m2 += om2 + (d * n) * (d * f);  // (an empty side adds 0 whatever d is)
      n = total;
    }
  }
};

// over the `width` lanes of a team (a power of two up to the wave)
template <typename CT>
__device__ __forceinline__ void team_moments(Moments<CT>& m, int width) {
  for (int off = 1; off < width; off <<= 1) {
    const CT on = __shfl_xor(m.n, off, 64), omean = __shfl_xor(m.mean, off, 64),
             om2 = __shfl_xor(m.m2, off, 64);
    // both lanes of a pair join in the same order, so that all lanes hold the same bits
    const bool low = (threadIdx.x & off) == 0;
    Moments<CT> a{low ? m.n : on, low ? m.mean : omean, low ? m.m2 : om2};
    a.add(low ? on : m.n, low ? omean : m.mean, low ? om2 : m.m2);
    m = a;
  }
}

// ---- activation -----------------------------------------------------------------------------------
__device__ __forceinline__ float gn_sigmoid(float z) { return 1.f / (1.f + __expf(-z)); }
__device__ __forceinline__ double gn_sigmoid(double z) { return 1.0 / (1.0 + exp(-z)); }

template <int ACT, typename CT>
__device__ __forceinline__ CT gn_act(CT z) {
  if constexpr (ACT == kGnRelu) return z <= CT(0) ? CT(0) : z;  // NaN stays
  if constexpr (ACT == kGnSilu) return z * gn_sigmoid(z);
  if constexpr (ACT == kGnGelu) return CT(0.5) * z * (CT(1) + erf(z * CT(0.70710678118654752440)));
  return z;
}

template <int ACT, typename CT>
__device__ __forceinline__ CT gn_slope(CT z) {
  if constexpr (ACT == kGnRelu) return z <= CT(0) ? CT(0) : CT(1);
  if constexpr (ACT == kGnSilu) {
    const CT s = gn_sigmoid(z);
    return s * (CT(1) + z * (CT(1) - s));
  }
  if constexpr (ACT == kGnGelu) {
    const CT below = CT(0.5) * (CT(1) + erf(z * CT(0.70710678118654752440)));
    return below + z * exp(z * z * CT(-0.5)) * CT(0.39894228040143267794);
  }
  return CT(1);
}

// ---- forward ----------------------------------------------------------------------------------------
// partial[(n * chunks + chunk) * G + g] = (mean, M2) of the chunk's rows of group g.
// Thread-level sums are taken about the first value that the thread reads of each channel: at most
// rows_per_chunk additions each, so an outlying first value costs at most that many roundings of
// what it adds to the variance itself.
// Dynamic LDS: 2 * row lanes * C values.
template <typename T>
__global__ __launch_bounds__(1024) void gn_stats_kernel(
    const T* __restrict__ x, typename Elem<T>::compute_t* __restrict__ partial, GnLevels lv, int C,
    int G, int team_width) {
  using ct = typename Elem<T>::compute_t;
  constexpr int VE = 16 / sizeof(T);
  extern __shared__ __align__(16) char gn_lds[];
  const int tc = (C + VE - 1) / VE, lanes = blockDim.x / tc;
  ct* lds_mean = reinterpret_cast<ct*>(gn_lds);
  ct* lds_m2 = lds_mean + lanes * C;
  const GnChunk ch = gn_chunk(lv, blockIdx.x);
  const int r0 = threadIdx.x / tc, c0 = (threadIdx.x - r0 * tc) * VE;
  const int count = min(VE, C - c0);
  if (r0 < lanes) {
    const T* src = x + ch.first_row * C + c0;
    ct pivot[VE], s[VE], q[VE];
#pragma unroll
    for (int i = 0; i < VE; ++i) pivot[i] = s[i] = q[i] = 0;
    if (r0 < ch.rows) {
      Pack<T, VE> p;
      p.load(src + static_cast<int64_t>(r0) * C, count);
      p.unpack(pivot);
    }
#pragma unroll 4
    for (int r = r0 + lanes; r < ch.rows; r += lanes) {
      Pack<T, VE> p;
      p.load(src + static_cast<int64_t>(r) * C, count);
      ct v[VE];
      p.unpack(v);
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        const ct d = v[i] - pivot[i];
        s[i] += d;
        q[i] += d * d;
      }
    }
    const int n = gn_lane_rows(ch.rows, r0, lanes);
    const ct inv = n > 0 ? ct(1) / static_cast<ct>(n) : ct(0);
#pragma unroll
    for (int i = 0; i < VE; ++i)
      if (i < count) {
        lds_mean[r0 * C + c0 + i] = pivot[i] + s[i] * inv;
        const ct m2 = q[i] - s[i] * s[i] * inv;
        lds_m2[r0 * C + c0 + i] = m2 < ct(0) ? ct(0) : m2;  // (NaN stays)
      }
  }
  __syncthreads();
  const int cpg = C / G, teams = blockDim.x / team_width;
  const int j = threadIdx.x & (team_width - 1);
  for (int g = threadIdx.x / team_width; g < G; g += teams) {
    Moments<ct> m{0, 0, 0};
    for (int e = j; e < lanes * cpg; e += team_width) {
      const int r = e / cpg, at = r * C + g * cpg + (e - r * cpg);
      m.add(static_cast<ct>(gn_lane_rows(ch.rows, r, lanes)), lds_mean[at], lds_m2[at]);
    }
    team_moments(m, team_width);
    if (j == 0) {
      ct* dst = partial + (static_cast<int64_t>(blockIdx.x) * G + g) * 2;
      dst[0] = m.mean;
      dst[1] = m.m2;
    }
  }
}

// mean and M2 of every group of the block's level, from the chunks' partial sums
template <typename CT>
__device__ __forceinline__ void gn_join_stats(const CT* __restrict__ partial, const GnLevels& lv,
                                              const GnChunk& ch, int cpg, int G, int team_width,
                                              CT eps, CT* lds_mean, CT* lds_rstd) {
  const int begin = lv.chunk_start[ch.level], end = lv.chunk_start[ch.level + 1];
  const int rows = lv.row_start[ch.level + 1] - lv.row_start[ch.level];
  const int teams = blockDim.x / team_width, j = threadIdx.x & (team_width - 1);
  for (int g = threadIdx.x / team_width; g < G; g += teams) {
    Moments<CT> m{0, 0, 0};
    for (int k = begin + j; k < end; k += team_width) {
      const CT* src = partial + ((ch.n * lv.chunks + k) * G + g) * 2;
      const int in = min(lv.rows_per_chunk, rows - (k - begin) * lv.rows_per_chunk);
      m.add(static_cast<CT>(in) * static_cast<CT>(cpg), src[0], src[1]);
    }
    team_moments(m, team_width);
    if (j == 0) {
      lds_mean[g] = m.mean;
      lds_rstd[g] = CT(1) / sqrt(m.m2 / (static_cast<CT>(rows) * static_cast<CT>(cpg)) + eps);
    }
  }
}

// mean and rstd (N, levels, G) may be NULL (no gradient wanted).  Dynamic LDS: 2 G values.
template <typename T, int ACT>
__global__ __launch_bounds__(1024) void gn_apply_kernel(
    const T* __restrict__ x, const typename Elem<T>::compute_t* __restrict__ partial,
    const void* __restrict__ weight, const void* __restrict__ bias, T* __restrict__ out,
    typename Elem<T>::compute_t* __restrict__ mean, typename Elem<T>::compute_t* __restrict__ rstd,
    GnLevels lv, int C, int G, int team_width, typename Elem<T>::compute_t eps, int wide) {
  using ct = typename Elem<T>::compute_t;
  constexpr int VE = 16 / sizeof(T);
  extern __shared__ __align__(16) char gn_lds[];
  ct* lds_mean = reinterpret_cast<ct*>(gn_lds);
  ct* lds_rstd = lds_mean + G;
  const GnChunk ch = gn_chunk(lv, blockIdx.x);
  const int cpg = C / G;
  gn_join_stats(partial, lv, ch, cpg, G, team_width, eps, lds_mean, lds_rstd);
  __syncthreads();
  const int chunk = blockIdx.x % lv.chunks;
  if (mean != nullptr && chunk == lv.chunk_start[ch.level]) {
    for (int g = threadIdx.x; g < G; g += blockDim.x) {
      const int64_t at = (ch.n * lv.levels + ch.level) * G + g;
      mean[at] = lds_mean[g];
      rstd[at] = lds_rstd[g];
    }
  }
  const int tc = (C + VE - 1) / VE, lanes = blockDim.x / tc;
  const int r0 = threadIdx.x / tc, c0 = (threadIdx.x - r0 * tc) * VE;
  if (r0 >= lanes) return;
  const int count = min(VE, C - c0);
  const int64_t pl = lv.param_levels > 1 ? static_cast<int64_t>(ch.level) * C : 0;
  ct mu[VE], a[VE], b[VE];
#pragma unroll
  for (int i = 0; i < VE; ++i) {
    mu[i] = a[i] = b[i] = 0;
    if (i < count) {
      const int g = (c0 + i) / cpg;
      mu[i] = lds_mean[g];
      a[i] = lds_rstd[g] * load_param<T>(weight, pl + c0 + i, wide != 0);
      b[i] = load_param<T>(bias, pl + c0 + i, wide != 0);
    }
  }
  const int64_t base = ch.first_row * C + c0;
#pragma unroll 4
  for (int r = r0; r < ch.rows; r += lanes) {
    Pack<T, VE> p;
    p.load(x + base + static_cast<int64_t>(r) * C, count);
    ct v[VE];
    p.unpack(v);
#pragma unroll
    for (int i = 0; i < VE; ++i) v[i] = gn_act<ACT>((v[i] - mu[i]) * a[i] + b[i]);
    p.pack(v);
    p.store(out + base + static_cast<int64_t>(r) * C, count);
  }
}

// ---- gradient ---------------------------------------------------------------------------------------
// Per chunk: partial_c[(block * 2 + k) * C + c] = sum over rows of dz * u (k = 0) and dz (k = 1), for
// the parameters; partial_g[(block * G + g) * 2 + k] = sum over the group of w dz (k = 0) and
// w dz u (k = 1), for dx.  partial_c may be NULL.  Dynamic LDS: 2 * row lanes * C values.
template <typename T, int ACT>
__global__ __launch_bounds__(1024) void gn_bwd_stats_kernel(
    const T* __restrict__ grad_out, const T* __restrict__ x, const void* __restrict__ weight,
    const void* __restrict__ bias, const typename Elem<T>::compute_t* __restrict__ mean,
    const typename Elem<T>::compute_t* __restrict__ rstd,
    typename Elem<T>::compute_t* __restrict__ partial_c,
    typename Elem<T>::compute_t* __restrict__ partial_g, GnLevels lv, int C, int G, int team_width,
    int wide) {
  using ct = typename Elem<T>::compute_t;
  constexpr int VE = 16 / sizeof(T);
  extern __shared__ __align__(16) char gn_lds[];
  const int tc = (C + VE - 1) / VE, lanes = blockDim.x / tc;
  ct* lds_dw = reinterpret_cast<ct*>(gn_lds);
  ct* lds_db = lds_dw + lanes * C;
  const GnChunk ch = gn_chunk(lv, blockIdx.x);
  const int r0 = threadIdx.x / tc, c0 = (threadIdx.x - r0 * tc) * VE;
  const int count = min(VE, C - c0), cpg = C / G;
  const int64_t pl = lv.param_levels > 1 ? static_cast<int64_t>(ch.level) * C : 0;
  const int64_t sg = (ch.n * lv.levels + ch.level) * G;
  if (r0 < lanes) {
    ct mu[VE], s[VE], w[VE], b[VE], dw[VE], db[VE];
#pragma unroll
    for (int i = 0; i < VE; ++i) {
      mu[i] = s[i] = w[i] = b[i] = dw[i] = db[i] = 0;
      if (i < count) {
        const int g = (c0 + i) / cpg;
        mu[i] = mean[sg + g];
        s[i] = rstd[sg + g];
        if (ACT != kGnNone) {
          w[i] = load_param<T>(weight, pl + c0 + i, wide != 0);
          b[i] = load_param<T>(bias, pl + c0 + i, wide != 0);
        }
      }
    }
    const int64_t base = ch.first_row * C + c0;
#pragma unroll 4
    for (int r = r0; r < ch.rows; r += lanes) {
      Pack<T, VE> px, pg;
      px.load(x + base + static_cast<int64_t>(r) * C, count);
      pg.load(grad_out + base + static_cast<int64_t>(r) * C, count);
      ct xv[VE], gv[VE];
      px.unpack(xv);
      pg.unpack(gv);
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        const ct u = (xv[i] - mu[i]) * s[i];
        const ct dz = ACT == kGnNone ? gv[i] : gv[i] * gn_slope<ACT>(u * w[i] + b[i]);
        dw[i] += dz * u;
        db[i] += dz;
      }
    }
#pragma unroll
    for (int i = 0; i < VE; ++i)
      if (i < count) {
        lds_dw[r0 * C + c0 + i] = dw[i];
        lds_db[r0 * C + c0 + i] = db[i];
      }
  }
  __syncthreads();
  for (int c = threadIdx.x; c < C; c += blockDim.x) {
    ct dw = 0, db = 0;
    for (int r = 0; r < lanes; ++r) {
      dw += lds_dw[r * C + c];
      db += lds_db[r * C + c];
    }
    if (partial_c != nullptr) {
      ct* dst = partial_c + static_cast<int64_t>(blockIdx.x) * 2 * C;
      dst[c] = dw;
      dst[C + c] = db;
    }
    const ct w = load_param<T>(weight, pl + c, wide != 0);
    lds_dw[c] = dw * w;  // row lane 0's place of column c: read and written by this thread only
    lds_db[c] = db * w;
  }
  __syncthreads();
  const int teams = blockDim.x / team_width, j = threadIdx.x & (team_width - 1);
  for (int g = threadIdx.x / team_width; g < G; g += teams) {
    ct m1 = 0, m2 = 0;
    for (int e = j; e < cpg; e += team_width) {
      m1 += lds_db[g * cpg + e];
      m2 += lds_dw[g * cpg + e];
    }
    for (int off = 1; off < team_width; off <<= 1) {
      m1 += __shfl_xor(m1, off, 64);
      m2 += __shfl_xor(m2, off, 64);
    }
    if (j == 0) {
      ct* dst = partial_g + (static_cast<int64_t>(blockIdx.x) * G + g) * 2;
      dst[0] = m1;
      dst[1] = m2;
    }
  }
}

// Dynamic LDS: 2 G values.
template <typename T, int ACT>
__global__ __launch_bounds__(1024) void gn_bwd_apply_kernel(
    const T* __restrict__ grad_out, const T* __restrict__ x, const void* __restrict__ weight,
    const void* __restrict__ bias, const typename Elem<T>::compute_t* __restrict__ mean,
    const typename Elem<T>::compute_t* __restrict__ rstd,
    const typename Elem<T>::compute_t* __restrict__ partial_g, T* __restrict__ grad_x, GnLevels lv,
    int C, int G, int team_width, int wide) {
  using ct = typename Elem<T>::compute_t;
  constexpr int VE = 16 / sizeof(T);
  extern __shared__ __align__(16) char gn_lds[];
  ct* lds_m1 = reinterpret_cast<ct*>(gn_lds);
  ct* lds_m2 = lds_m1 + G;
  const GnChunk ch = gn_chunk(lv, blockIdx.x);
  const int cpg = C / G;
  const int teams = blockDim.x / team_width, j = threadIdx.x & (team_width - 1);
  const int rows = lv.row_start[ch.level + 1] - lv.row_start[ch.level];
  const ct inv = ct(1) / (static_cast<ct>(rows) * static_cast<ct>(cpg));
  for (int g = threadIdx.x / team_width; g < G; g += teams) {
    ct m1 = 0, m2 = 0;
    for (int k = lv.chunk_start[ch.level] + j; k < lv.chunk_start[ch.level + 1]; k += team_width) {
      const ct* src = partial_g + ((ch.n * lv.chunks + k) * G + g) * 2;
      m1 += src[0];
      m2 += src[1];
    }
    for (int off = 1; off < team_width; off <<= 1) {
      m1 += __shfl_xor(m1, off, 64);
      m2 += __shfl_xor(m2, off, 64);
    }
    if (j == 0) {
      lds_m1[g] = m1 * inv;
      lds_m2[g] = m2 * inv;
    }
  }
  __syncthreads();
  const int tc = (C + VE - 1) / VE, lanes = blockDim.x / tc;
  const int r0 = threadIdx.x / tc, c0 = (threadIdx.x - r0 * tc) * VE;
  if (r0 >= lanes) return;
  const int count = min(VE, C - c0);
  const int64_t pl = lv.param_levels > 1 ? static_cast<int64_t>(ch.level) * C : 0;
  const int64_t sg = (ch.n * lv.levels + ch.level) * G;
  ct mu[VE], s[VE], w[VE], b[VE], m1[VE], m2[VE];
#pragma unroll
  for (int i = 0; i < VE; ++i) {
    mu[i] = s[i] = w[i] = b[i] = m1[i] = m2[i] = 0;
    if (i < count) {
      const int g = (c0 + i) / cpg;
      mu[i] = mean[sg + g];
      s[i] = rstd[sg + g];
      w[i] = load_param<T>(weight, pl + c0 + i, wide != 0);
      if (ACT != kGnNone) b[i] = load_param<T>(bias, pl + c0 + i, wide != 0);
      m1[i] = lds_m1[g];
      m2[i] = lds_m2[g];
    }
  }
  const int64_t base = ch.first_row * C + c0;
#pragma unroll 4
  for (int r = r0; r < ch.rows; r += lanes) {
    Pack<T, VE> px, pg;
    px.load(x + base + static_cast<int64_t>(r) * C, count);
    pg.load(grad_out + base + static_cast<int64_t>(r) * C, count);
    ct xv[VE], gv[VE];
    px.unpack(xv);
    pg.unpack(gv);
#pragma unroll
    for (int i = 0; i < VE; ++i) {
      const ct u = (xv[i] - mu[i]) * s[i];
      const ct dz = ACT == kGnNone ? gv[i] : gv[i] * gn_slope<ACT>(u * w[i] + b[i]);
      gv[i] = s[i] * (w[i] * dz - m1[i] - u * m2[i]);
    }
    pg.pack(gv);
    pg.store(grad_x + base + static_cast<int64_t>(r) * C, count);
  }
}

}  // namespace msda
