// Group normalisation of a flattened pyramid (gfx950): x (N, S, C), channels last; every level is a
// run of rows of every sample with statistics of its own, an activation follows.
//
//   per (n, level, group): mu = mean x, s = 1 / sqrt(mean (x - mu)^2 + eps) over the level's rows
//   and the group's C / G channels;  u = (x - mu) * s,  z = u * w + b,  y = act(z)
//   with dz = dy * act'(z):  db = sum dz,  dw = sum dz * u  (over samples and rows),
//   dx = s * (w dz - m1 - u * m2),  m1 = mean (w dz),  m2 = mean (w dz u)  (over rows and group)
//
// Three launches a direction: sums per chunk of rows, a join of the chunks' sums per level, and the
// pass that writes.  Threads lie along the channels (16 bytes a thread) and then along the rows, so a
// thread keeps its channels for the whole chunk and sums per channel in registers; groups are formed
// from channels once per chunk.  The passes that write take short chunks (a workgroup a few rows a
// thread, all their loads in flight at once), which need the level's joined sums and not its chunks'.
#pragma once

#include "msda_vec.h"

namespace msda {

enum GnAct { kGnNone = 0, kGnRelu = 1, kGnSilu = 2, kGnGelu = 3 };

constexpr int kGnThreads = 256;
constexpr int kGnRowsAhead = 4;  // rows of a thread whose loads are in flight together

// The rows of every sample cut into levels and the levels into chunks.
struct GnCut {
  int levels, chunks, rows_per_chunk;
  int row_start[kMaxNormLevels + 1];
  int chunk_start[kMaxNormLevels + 1];
};

struct GnChunk {
  int level, rows;
  int n;
  int64_t first_row;  // within the tensor
};

__device__ __forceinline__ GnChunk gn_chunk(const GnCut& cut, int block) {
  GnChunk c;
  c.n = block / cut.chunks;
  const int chunk = block - c.n * cut.chunks;
  c.level = 0;
  while (c.level + 1 < cut.levels && chunk >= cut.chunk_start[c.level + 1]) ++c.level;
  const int row = cut.row_start[c.level] + (chunk - cut.chunk_start[c.level]) * cut.rows_per_chunk;
  c.rows = min(cut.rows_per_chunk, cut.row_start[c.level + 1] - row);
  c.first_row = static_cast<int64_t>(c.n) * cut.row_start[cut.levels] + row;
  return c;
}

// row lanes of a workgroup for rows of `vecs` vectors
__host__ __device__ inline int gn_lanes(int vecs) { return vecs < kGnThreads ? kGnThreads / vecs : 1; }

// rows of a chunk of `rows` that row lane r of `lanes` handles
__device__ __forceinline__ int gn_lane_rows(int rows, int r, int lanes) {
  return r < rows ? (rows - r + lanes - 1) / lanes : 0;
}

// Calls f(Pack (&)[K], rows r0, r0 + lanes, ...) for the thread's rows with the loads of
// kGnRowsAhead rows issued before the first is used.  `load` fills one row's packs.
template <typename P, typename Load, typename Use>
__device__ __forceinline__ void gn_rows(int r0, int rows, int lanes, Load load, Use use) {
  constexpr int U = kGnRowsAhead;
  int r = r0;
  for (; r + (U - 1) * lanes < rows; r += U * lanes) {
    P p[U];
#pragma unroll
    for (int k = 0; k < U; ++k) load(p[k], r + k * lanes);
#pragma unroll
    for (int k = 0; k < U; ++k) use(p[k], r + k * lanes);
  }
  for (; r < rows; r += lanes) {
    P p;
    load(p, r);
    use(p, r);
  }
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
template <typename CT>
__device__ __forceinline__ void team_add2(CT& a, CT& b, int width) {
  for (int off = 1; off < width; off <<= 1) {
    a += __shfl_xor(a, off, 64);
    b += __shfl_xor(b, off, 64);
  }
}

// lanes that join the sums of one group in a workgroup of `threads`
__host__ __device__ inline int gn_team_width(int threads, int G) {
  int w = 1;
  while (w < 64 && w * 2 * G <= threads) w *= 2;
  return w;
}

// the VE values of `src` (one a group) that belong to the columns of a span
template <int VE, int MODE, typename CT>
__device__ __forceinline__ void gn_spread(const CT* __restrict__ src, const Span<VE, MODE>& sp, int cpg,
                                          CT* v) {
  int g = sp.c / cpg, at = sp.c - g * cpg;
#pragma unroll
  for (int i = 0; i < VE; ++i) {
    v[i] = i < sp.count ? src[g] : CT(0);
    if (++at == cpg) {
      at = 0;
      ++g;
    }
  }
}

// ---- activation -----------------------------------------------------------------------------------
// (v_rcp_f32 is within one step of 1 / x: a division would cost ten instructions more an element)
__device__ __forceinline__ float gn_sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + __expf(-z)); }
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
// partial[(block * G + g) * 2] = (mean, M2) of the chunk's rows of group g.
// Thread-level sums are taken about the first value that the thread reads of each channel, so a
// common offset of the values costs nothing; an outlying first value costs at most a rounding per
// row of what it adds to the variance itself.
// Dynamic LDS: 2 * row lanes * C values.
template <typename T, int MODE>
__global__ __launch_bounds__(kGnThreads) void gn_stats_kernel(
    const T* __restrict__ x, typename Elem<T>::compute_t* __restrict__ partial, GnCut cut, int C,
    int G) {
  using ct = typename Elem<T>::compute_t;
  constexpr int VE = 16 / sizeof(T);
  using P = Pack<T, VE>;
  extern __shared__ __align__(16) char gn_lds[];
  const int vecs = (C + VE - 1) / VE, lanes = gn_lanes(vecs);
  ct* lds_mean = reinterpret_cast<ct*>(gn_lds);
  ct* lds_m2 = lds_mean + lanes * C;
  const GnChunk ch = gn_chunk(cut, blockIdx.x);
  const T* src = x + ch.first_row * C;
  const int r0 = vecs < kGnThreads ? threadIdx.x / vecs : 0;
  for (int k = threadIdx.x - r0 * vecs; k < vecs && r0 < lanes; k += kGnThreads) {
    const auto sp = Span<VE, MODE>::at(k, C);
    ct pivot[VE], s[VE], q[VE];
#pragma unroll
    for (int i = 0; i < VE; ++i) pivot[i] = s[i] = q[i] = 0;
    if (r0 < ch.rows) {
      P p;
      sp.load(p, src + static_cast<int64_t>(r0) * C);
      p.unpack(pivot);
    }
    gn_rows<P>(
        r0 + lanes, ch.rows, lanes,
        [&](P& p, int r) { sp.load(p, src + static_cast<int64_t>(r) * C); },
        [&](P& p, int) {
          ct v[VE];
          p.unpack(v);
#pragma unroll
          for (int i = 0; i < VE; ++i) {
            const ct d = v[i] - pivot[i];
            s[i] += d;
            q[i] += d * d;
          }
        });
    const int n = gn_lane_rows(ch.rows, r0, lanes);
    const ct inv = n > 0 ? ct(1) / static_cast<ct>(n) : ct(0);
#pragma unroll
    for (int i = 0; i < VE; ++i)
      if (sp.owns(i)) {
        const ct m2 = q[i] - s[i] * s[i] * inv;
        lds_mean[r0 * C + sp.c + i] = pivot[i] + s[i] * inv;
        lds_m2[r0 * C + sp.c + i] = m2 < ct(0) ? ct(0) : m2;  // (NaN stays)
      }
  }
  __syncthreads();
  const int cpg = C / G, width = gn_team_width(kGnThreads, G), teams = kGnThreads / width;
  const int j = threadIdx.x & (width - 1);
  for (int g = threadIdx.x / width; g < G; g += teams) {
    Moments<ct> m{0, 0, 0};
    for (int e = j; e < lanes * cpg; e += width) {
      const int r = e / cpg, at = r * C + g * cpg + (e - r * cpg);
      m.add(static_cast<ct>(gn_lane_rows(ch.rows, r, lanes)), lds_mean[at], lds_m2[at]);
    }
    team_moments(m, width);
    if (j == 0) {
      ct* dst = partial + (static_cast<int64_t>(blockIdx.x) * G + g) * 2;
      dst[0] = m.mean;
      dst[1] = m.m2;
    }
  }
}

// mean and rstd (N, levels, G) from the chunks' sums: the mean of the means, then M2 about it
// (sum of the chunks' M2 and of n_k (mean_k - mean)^2; the second reading comes from the cache).
// blockIdx.x: (sample, level), blockIdx.y: tile of kGnJoinGroups groups.
constexpr int kGnJoinGroups = 8;
template <typename CT>
__global__ __launch_bounds__(kGnThreads) void gn_join_kernel(const CT* __restrict__ partial,
                                                             CT* __restrict__ mean,
                                                             CT* __restrict__ rstd, GnCut cut, int cpg,
                                                             int G, CT eps) {
  constexpr int WIDTH = kGnThreads / kGnJoinGroups;
  const int n = blockIdx.x / cut.levels, level = blockIdx.x - n * cut.levels;
  const int chunks = cut.chunk_start[level + 1] - cut.chunk_start[level];
  const int rows = cut.row_start[level + 1] - cut.row_start[level];
  const int j = threadIdx.x % WIDTH, g = blockIdx.y * kGnJoinGroups + threadIdx.x / WIDTH;
  if (g >= G) return;
  const CT* src =
      partial + ((static_cast<int64_t>(n) * cut.chunks + cut.chunk_start[level]) * G + g) * 2;
  const CT share = CT(1) / static_cast<CT>(rows);
  auto chunk_rows = [&](int k) {
    return static_cast<CT>(min(cut.rows_per_chunk, rows - k * cut.rows_per_chunk));
  };
  // about the first chunk's mean, so that a common offset costs nothing
  const CT pivot = src[0];
  CT mu = 0;
#pragma unroll 4
  for (int k = j; k < chunks; k += WIDTH)
    mu += chunk_rows(k) * share * (src[static_cast<int64_t>(k) * G * 2] - pivot);
  for (int off = 1; off < WIDTH; off <<= 1) mu += __shfl_xor(mu, off, 64);
  CT m2 = 0;
#pragma unroll 4
  for (int k = j; k < chunks; k += WIDTH) {
    const CT* at = src + static_cast<int64_t>(k) * G * 2;
    const CT d = at[0] - pivot - mu;
    m2 += at[1] + chunk_rows(k) * static_cast<CT>(cpg) * d * d;
  }
  for (int off = 1; off < WIDTH; off <<= 1) m2 += __shfl_xor(m2, off, 64);
  if (j == 0) {
    const int64_t at = static_cast<int64_t>(blockIdx.x) * G + g;
    mean[at] = pivot + mu;
    rstd[at] = CT(1) / sqrt(m2 / (static_cast<CT>(rows) * static_cast<CT>(cpg)) + eps);
  }
}

// blockIdx.y: tile of kGnThreads vectors of a row
template <typename T, int ACT, int MODE>
__global__ __launch_bounds__(kGnThreads) void gn_apply_kernel(
    const T* __restrict__ x, const typename Elem<T>::compute_t* __restrict__ mean,
    const typename Elem<T>::compute_t* __restrict__ rstd, const void* __restrict__ weight,
    const void* __restrict__ bias, T* __restrict__ out, GnCut cut, int C, int G, int param_levels,
    int wide) {
  using ct = typename Elem<T>::compute_t;
  constexpr int VE = 16 / sizeof(T);
  using P = Pack<T, VE>;
  const int vecs = (C + VE - 1) / VE, lanes = gn_lanes(vecs), cpg = C / G;
  const GnChunk ch = gn_chunk(cut, blockIdx.x);
  const int r0 = vecs < kGnThreads ? threadIdx.x / vecs : 0;
  const int k = threadIdx.x - r0 * vecs + blockIdx.y * kGnThreads;
  if (r0 >= lanes || k >= vecs) return;
  const auto sp = Span<VE, MODE>::at(k, C);
  const int64_t pl = param_levels > 1 ? static_cast<int64_t>(ch.level) * C : 0;
  const int64_t sg = (static_cast<int64_t>(ch.n) * cut.levels + ch.level) * G;
  ct mu[VE], a[VE], b[VE], w[VE];
  gn_spread(mean + sg, sp, cpg, mu);
  gn_spread(rstd + sg, sp, cpg, a);
  load_params<T>(weight, pl, sp, wide != 0, w);
  load_params<T>(bias, pl, sp, wide != 0, b);
#pragma unroll
  for (int i = 0; i < VE; ++i) a[i] *= w[i];
  const T* src = x + ch.first_row * C;
  T* dst = out + ch.first_row * C;
  gn_rows<P>(
      r0, ch.rows, lanes, [&](P& p, int r) { sp.load(p, src + static_cast<int64_t>(r) * C); },
      [&](P& p, int r) {
        ct v[VE];
        p.unpack(v);
#pragma unroll
        for (int i = 0; i < VE; ++i) v[i] = gn_act<ACT>((v[i] - mu[i]) * a[i] + b[i]);
        p.pack(v);
        sp.store(p, dst + static_cast<int64_t>(r) * C);
      });
}

// ---- gradient ---------------------------------------------------------------------------------------
template <typename T, int VE>
struct GnPair {
  Pack<T, VE> x, g;
};

// Per chunk: partial_c[(block * 2 + k) * C + c] = sum over rows of dz * u (k = 0) and dz (k = 1), for
// the parameters; partial_g[(block * G + g) * 2 + k] = sum over the group of w dz (k = 0) and
// w dz u (k = 1), for dx.  partial_c may be NULL.  Dynamic LDS: 2 * row lanes * C values.
template <typename T, int ACT, int MODE>
__global__ __launch_bounds__(kGnThreads) void gn_bwd_stats_kernel(
    const T* __restrict__ grad_out, const T* __restrict__ x, const void* __restrict__ weight,
    const void* __restrict__ bias, const typename Elem<T>::compute_t* __restrict__ mean,
    const typename Elem<T>::compute_t* __restrict__ rstd,
    typename Elem<T>::compute_t* __restrict__ partial_c,
    typename Elem<T>::compute_t* __restrict__ partial_g, GnCut cut, int C, int G, int param_levels,
    int wide) {
  using ct = typename Elem<T>::compute_t;
  constexpr int VE = 16 / sizeof(T);
  using P = GnPair<T, VE>;
  extern __shared__ __align__(16) char gn_lds[];
  const int vecs = (C + VE - 1) / VE, lanes = gn_lanes(vecs), cpg = C / G;
  ct* lds_dw = reinterpret_cast<ct*>(gn_lds);
  ct* lds_db = lds_dw + lanes * C;
  const GnChunk ch = gn_chunk(cut, blockIdx.x);
  const int64_t pl = param_levels > 1 ? static_cast<int64_t>(ch.level) * C : 0;
  const int64_t sg = (static_cast<int64_t>(ch.n) * cut.levels + ch.level) * G;
  const T* sx = x + ch.first_row * C;
  const T* sd = grad_out + ch.first_row * C;
  const int r0 = vecs < kGnThreads ? threadIdx.x / vecs : 0;
  for (int k = threadIdx.x - r0 * vecs; k < vecs && r0 < lanes; k += kGnThreads) {
    const auto sp = Span<VE, MODE>::at(k, C);
    ct mu[VE], s[VE], w[VE], b[VE], dw[VE], db[VE];
    gn_spread(mean + sg, sp, cpg, mu);
    gn_spread(rstd + sg, sp, cpg, s);
    if constexpr (ACT != kGnNone) {
      load_params<T>(weight, pl, sp, wide != 0, w);
      load_params<T>(bias, pl, sp, wide != 0, b);
    }
#pragma unroll
    for (int i = 0; i < VE; ++i) dw[i] = db[i] = 0;
    gn_rows<P>(
        r0, ch.rows, lanes,
        [&](P& p, int r) {
          sp.load(p.x, sx + static_cast<int64_t>(r) * C);
          sp.load(p.g, sd + static_cast<int64_t>(r) * C);
        },
        [&](P& p, int) {
          ct xv[VE], gv[VE];
          p.x.unpack(xv);
          p.g.unpack(gv);
#pragma unroll
          for (int i = 0; i < VE; ++i) {
            const ct u = (xv[i] - mu[i]) * s[i];
            ct dz = gv[i];
            if constexpr (ACT != kGnNone) dz *= gn_slope<ACT>(u * w[i] + b[i]);
            dw[i] += dz * u;
            db[i] += dz;
          }
        });
#pragma unroll
    for (int i = 0; i < VE; ++i)
      if (sp.owns(i)) {
        lds_dw[r0 * C + sp.c + i] = dw[i];
        lds_db[r0 * C + sp.c + i] = db[i];
      }
  }
  __syncthreads();
  for (int c = threadIdx.x; c < C; c += kGnThreads) {
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
  const int width = gn_team_width(kGnThreads, G), teams = kGnThreads / width;
  const int j = threadIdx.x & (width - 1);
  for (int g = threadIdx.x / width; g < G; g += teams) {
    ct m1 = 0, m2 = 0;
    for (int e = j; e < cpg; e += width) {
      m1 += lds_db[g * cpg + e];
      m2 += lds_dw[g * cpg + e];
    }
    team_add2(m1, m2, width);
    if (j == 0) {
      ct* dst = partial_g + (static_cast<int64_t>(blockIdx.x) * G + g) * 2;
      dst[0] = m1;
      dst[1] = m2;
    }
  }
}

// Joins what the chunks left, in one launch: the first `groups` workgroups (one a (sample, level) and
// tile of 32 groups) write m1 and m2 (N, levels, G), the others the parameters' gradients.
template <typename T>
__global__ __launch_bounds__(1024) void gn_bwd_join_kernel(
    const typename Elem<T>::compute_t* __restrict__ partial_g,
    const typename Elem<T>::compute_t* __restrict__ partial_c,
    typename Elem<T>::compute_t* __restrict__ m1, typename Elem<T>::compute_t* __restrict__ m2,
    void* __restrict__ grad_weight, void* __restrict__ grad_bias, GnCut cut, ColumnRuns runs, int groups,
    int C, int G, int wide) {
  using ct = typename Elem<T>::compute_t;
  if (static_cast<int>(blockIdx.x) >= groups) {
    const int tiles = (C + 15) / 16, b = blockIdx.x - groups;
    column_sums<T>(partial_c, grad_weight, grad_bias, runs, C, wide != 0, b % tiles,
                   (b / tiles) & 1, b / tiles / 2);
    return;
  }
  const int tiles = (G + 31) / 32, cell = blockIdx.x / tiles;
  const int n = cell / cut.levels, level = cell - n * cut.levels;
  const int chunks = cut.chunk_start[level + 1] - cut.chunk_start[level];
  const int rows = cut.row_start[level + 1] - cut.row_start[level];
  const ct inv = ct(1) / (static_cast<ct>(rows) * static_cast<ct>(C / G));
  const int j = threadIdx.x & 31, g = (blockIdx.x - cell * tiles) * 32 + (threadIdx.x >> 5);
  if (g >= G) return;
  const ct* src =
      partial_g + ((static_cast<int64_t>(n) * cut.chunks + cut.chunk_start[level]) * G + g) * 2;
  ct a = 0, b = 0;
#pragma unroll 4
  for (int k = j; k < chunks; k += 32) {
    a += src[static_cast<int64_t>(k) * G * 2];
    b += src[static_cast<int64_t>(k) * G * 2 + 1];
  }
  team_add2(a, b, 32);
  if (j == 0) {
    m1[static_cast<int64_t>(cell) * G + g] = a * inv;
    m2[static_cast<int64_t>(cell) * G + g] = b * inv;
  }
}

template <typename T, int ACT, int MODE>
__global__ __launch_bounds__(kGnThreads) void gn_bwd_apply_kernel(
    const T* __restrict__ grad_out, const T* __restrict__ x, const void* __restrict__ weight,
    const void* __restrict__ bias, const typename Elem<T>::compute_t* __restrict__ mean,
    const typename Elem<T>::compute_t* __restrict__ rstd,
    const typename Elem<T>::compute_t* __restrict__ m1,
    const typename Elem<T>::compute_t* __restrict__ m2, T* __restrict__ grad_x, GnCut cut, int C, int G,
    int param_levels, int wide) {
  using ct = typename Elem<T>::compute_t;
  constexpr int VE = 16 / sizeof(T);
  using P = GnPair<T, VE>;
  const int vecs = (C + VE - 1) / VE, lanes = gn_lanes(vecs), cpg = C / G;
  const GnChunk ch = gn_chunk(cut, blockIdx.x);
  const int r0 = vecs < kGnThreads ? threadIdx.x / vecs : 0;
  const int k = threadIdx.x - r0 * vecs + blockIdx.y * kGnThreads;
  if (r0 >= lanes || k >= vecs) return;
  const auto sp = Span<VE, MODE>::at(k, C);
  const int64_t pl = param_levels > 1 ? static_cast<int64_t>(ch.level) * C : 0;
  const int64_t sg = (static_cast<int64_t>(ch.n) * cut.levels + ch.level) * G;
  ct mu[VE], s[VE], w[VE], b[VE], a1[VE], a2[VE];
  gn_spread(mean + sg, sp, cpg, mu);
  gn_spread(rstd + sg, sp, cpg, s);
  gn_spread(m1 + sg, sp, cpg, a1);
  gn_spread(m2 + sg, sp, cpg, a2);
  load_params<T>(weight, pl, sp, wide != 0, w);
  if constexpr (ACT != kGnNone) load_params<T>(bias, pl, sp, wide != 0, b);
  const T* sx = x + ch.first_row * C;
  const T* sd = grad_out + ch.first_row * C;
  T* dst = grad_x + ch.first_row * C;
  gn_rows<P>(
      r0, ch.rows, lanes,
      [&](P& p, int r) {
        sp.load(p.x, sx + static_cast<int64_t>(r) * C);
        sp.load(p.g, sd + static_cast<int64_t>(r) * C);
      },
      [&](P& p, int r) {
        ct xv[VE], gv[VE];
        p.x.unpack(xv);
        p.g.unpack(gv);
#pragma unroll
        for (int i = 0; i < VE; ++i) {
          const ct u = (xv[i] - mu[i]) * s[i];
          ct dz = gv[i];
          if constexpr (ACT != kGnNone) dz *= gn_slope<ACT>(u * w[i] + b[i]);
          gv[i] = s[i] * (w[i] * dz - a1[i] - u * a2[i]);
        }
        p.g.pack(gv);
        sp.store(p.g, dst + static_cast<int64_t>(r) * C);
      });
}

}  // namespace msda
