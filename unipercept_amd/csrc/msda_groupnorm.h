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
//
// Bound by HBM, which every tensor but the last crosses twice a direction (MI355X, 8 x 43008 rows of
// 256 fp32 channels, 352 MB a tensor): sums 56 us, 6.3 TB/s; forward pass 113 us, 6.2 TB/s; sums of
// the gradient 115 us, 6.1 TB/s; its pass 162 us, 6.5 TB/s; the joins 5 and 6 us.
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

// Walks the thread's rows r0, r0 + lanes, ... of a chunk in steps of kGnRowsAhead rows, and of one row
// for the rest: load(p, r) for every row of a step, then use(p, r) with the array of the step's rows.
template <typename P, typename Load, typename Use>
__device__ __forceinline__ void gn_row_steps(int r0, int rows, int lanes, Load load, Use use) {
  constexpr int U = kGnRowsAhead;
  int r = r0;
  for (; r + (U - 1) * lanes < rows; r += U * lanes) {
    P p[U];
#pragma unroll
    for (int k = 0; k < U; ++k) load(p[k], r + k * lanes);
    use(p, r);
  }
  for (; r < rows; r += lanes) {
    P p[1];
    load(p[0], r);
    use(p, r);
  }
}
// the same with use(p, r) for one row at a time
template <typename P, typename Load, typename Use>
__device__ __forceinline__ void gn_rows(int r0, int rows, int lanes, Load load, Use use) {
  gn_row_steps<P>(r0, rows, lanes, load, [&](auto& p, int r) {
    constexpr int K = sizeof(p) / sizeof(P);
#pragma unroll
    for (int k = 0; k < K; ++k) use(p[k], r + k * lanes);
  });
}

// sums of two values over the `width` lanes of a team (a power of two up to the wave)
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

// Normal distribution function Phi(z) and, with it, exp(-z^2 / 2).  In fp32
//   1 - Phi(a) = exp(-a^2 / 2) * R(t),  t = 1 / (1 + 0.46 a),  a = |z|,
// with a polynomial R of degree 7 without constant term, fitted to sqrt(2 pi)^-1 times Mills' ratio over
// a = 0 .. 8.  With these constants as fp32 holds them the product is off by at most 8.4e-9 (at a = 0.74),
// 0.28 of fp32's rounding of a Phi next to 1.  (Parameters' gradients add this error up with one sign: a
// form that is off by 1.5e-7 shows there.)
// One exponential serves the function and its density.
__device__ __forceinline__ float gn_phi(float z, float& e) {
  const float a = fabsf(z);
  const float t = __builtin_amdgcn_rcpf(1.f + 0.46f * a);
  e = __expf(-0.5f * (a * a));
  float r = -0.0406047851f;
  r = r * t + 0.224280536f;
  r = r * t - 0.46577087f;
  r = r * t + 0.355322272f;
  r = r * t + 0.0418243669f;
  r = r * t + 0.202958718f;
  r = r * t + 0.181989759f;
  const float upper = r * t * e;  // 1 - Phi(|z|)
  return z < 0.f ? upper : 1.f - upper;
}
__device__ __forceinline__ double gn_phi(double z, double& e) {
  e = exp(z * z * -0.5);
  return 0.5 * erfc(z * -0.70710678118654752440);
}

template <int ACT, typename CT>
__device__ __forceinline__ CT gn_act(CT z) {
  if constexpr (ACT == kGnRelu) return z <= CT(0) ? CT(0) : z;  // NaN stays
  if constexpr (ACT == kGnSilu) return z * gn_sigmoid(z);
  if constexpr (ACT == kGnGelu) {
    CT e;
    return z * gn_phi(z, e);
  }
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
    CT e;
    const CT phi = gn_phi(z, e);
    return phi + z * e * CT(0.39894228040143267794);
  }
  return CT(1);
}

// 1 / n of a count of rows, n >= 1 (v_rcp_f32 is within one step of it)
__device__ __forceinline__ float gn_inverse(float n) { return __builtin_amdgcn_rcpf(n); }
__device__ __forceinline__ double gn_inverse(double n) { return 1.0 / n; }

// ---- the normalised value ---------------------------------------------------------------------------
// z = (x - mean) * (rstd * weight) + bias decides the ReLU's gate, and an element whose z is a rounding
// away from 0 has to be open in all of y, dx, dw and db or in none.  So every pass of both directions
// forms z and what it is made of by these functions alone, whose roundings the compiler may not change.
template <typename CT>
__device__ __forceinline__ CT gn_times(CT a, CT b) {
#pragma clang fp contract(off)
  return a * b;
}
template <typename CT>
__device__ __forceinline__ CT gn_centred(CT x, CT mean) {
#pragma clang fp contract(off)
  return x - mean;
}
__device__ __forceinline__ float gn_affine(float d, float scale, float bias) { return fmaf(d, scale, bias); }
__device__ __forceinline__ double gn_affine(double d, double scale, double bias) { return fma(d, scale, bias); }
// 1 / sqrt(sum / count + eps), inv = 1 / count
__device__ __forceinline__ float gn_rstd(float sum, float inv, float eps) { return 1.f / sqrtf(fmaf(sum, inv, eps)); }

// ---- forward ----------------------------------------------------------------------------------------
// partial[(block * G + g) * 2] = (mean, M2) of the chunk's rows of group g.
// A thread keeps the mean and M2 of the rows that it has read, per channel, and merges the next step's
// k rows about that mean: with d_i = x_i - mean, D = sum d_i and n rows so far,
//   mean += D / (n + k),  M2 += sum d_i^2 - D^2 / (n + k)
// (k = 1 is Welford's recurrence).  D^2 / (n + k) takes away at most half of sum d_i^2, in the first step
// (about its first row) three quarters, so nothing cancels: a common offset of the values costs nothing,
// and an outlying value costs roundings of its own share of M2.  (Sums about the first value alone lose
// about n^2 / 2 roundings where that value is the outlier.)
// Where a vector lies in one group, a thread joins its VE channels before the workgroup does (10752 bf16
// rows of 256 channels 5.4 us, 348160 rows 32.3; 1.3 and 1.8 us more where the workgroup joins them).
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
  const bool whole = MODE == kRowEven && C / G % VE == 0;
  const int joined = whole ? VE : 1;  // channels of a part in LDS
  for (int k = threadIdx.x - r0 * vecs; k < vecs && r0 < lanes; k += kGnThreads) {
    const auto sp = Span<VE, MODE>::at(k, C);
    ct mean[VE], m2[VE];
#pragma unroll
    for (int i = 0; i < VE; ++i) mean[i] = m2[i] = 0;
    int n = 0;
    gn_row_steps<P>(
        r0, ch.rows, lanes, [&](P& p, int r) { sp.load(p, src + static_cast<int64_t>(r) * C); },
        [&](auto& p, int) {
          constexpr int K = sizeof(p) / sizeof(P);
          ct v[K][VE];
#pragma unroll
          for (int k = 0; k < K; ++k) p[k].unpack(v[k]);
          if (n == 0) {  // (the first step is taken about its first row)
#pragma unroll
            for (int i = 0; i < VE; ++i) mean[i] = v[0][i];
          }
          n += K;
          const ct inv = gn_inverse(static_cast<ct>(n));
#pragma unroll
          for (int i = 0; i < VE; ++i) {
            ct sum = v[0][i] - mean[i];
            m2[i] += sum * sum;
#pragma unroll
            for (int k = 1; k < K; ++k) {
              const ct d = v[k][i] - mean[i];
              sum += d;
              m2[i] += d * d;
            }
            const ct move = sum * inv;
            m2[i] -= sum * move;
            mean[i] += move;
          }
        });
#pragma unroll
    for (int i = 0; i < VE; ++i) m2[i] = m2[i] < ct(0) ? ct(0) : m2[i];  // (NaN stays)
    if (whole) {
      ct d = 0, all = 0;
#pragma unroll
      for (int i = 1; i < VE; ++i) d += mean[i] - mean[0];
      d *= ct(1) / VE;
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        const ct e = mean[i] - mean[0] - d;
        all += m2[i] + static_cast<ct>(n) * e * e;
      }
      lds_mean[r0 * vecs + k] = mean[0] + d;
      lds_m2[r0 * vecs + k] = all;
    } else {
#pragma unroll
      for (int i = 0; i < VE; ++i)
        if (sp.owns(i)) {
          lds_mean[r0 * C + sp.c + i] = mean[i];
          lds_m2[r0 * C + sp.c + i] = m2[i];
        }
    }
  }
  __syncthreads();
  // groups: the mean of the parts' means, then M2 about it (sum of the parts' M2 and of
  // n_r (mean_r - mean)^2), all about one part's mean so that a common offset costs nothing
  const int pitch = C / joined, cpg = pitch / G;  // parts of a row lane, of its groups
  const int width = gn_team_width(kGnThreads, G), teams = kGnThreads / width;
  const int j = threadIdx.x & (width - 1), parts = min(lanes, ch.rows) * cpg;
  const ct share = ct(1) / (static_cast<ct>(ch.rows) * static_cast<ct>(cpg));
  const int full = ch.rows / lanes, rest = ch.rows - full * lanes;  // rows of lane r: full, or one more
  const int step_r = width / cpg, step_c = width - step_r * cpg, r_at = j / cpg, c_at = j - r_at * cpg;
  for (int g = threadIdx.x / width; g < G; g += teams) {
    const ct pivot = lds_mean[g * cpg];
    // visits part e = j, j + width, ... as (row lane, column), without a division each
    auto visit = [&](auto f) {
      int r = r_at, c = c_at;
      for (int e = j; e < parts; e += width) {
        f(r * pitch + g * cpg + c, static_cast<ct>(full + (r < rest ? 1 : 0)));
        r += step_r;
        c += step_c;
        if (c >= cpg) {
          c -= cpg;
          ++r;
        }
      }
    };
    ct mu = 0, m2 = 0;
    visit([&](int at, ct n) { mu += n * share * (lds_mean[at] - pivot); });
    for (int off = 1; off < width; off <<= 1) mu += __shfl_xor(mu, off, 64);
    visit([&](int at, ct n) {
      const ct d = lds_mean[at] - pivot - mu;
      m2 += lds_m2[at] + n * static_cast<ct>(joined) * d * d;
    });
    for (int off = 1; off < width; off <<= 1) m2 += __shfl_xor(m2, off, 64);
    if (j == 0) {
      ct* dst = partial + (static_cast<int64_t>(blockIdx.x) * G + g) * 2;
      dst[0] = pivot + mu;
      dst[1] = m2;
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
  for (int i = 0; i < VE; ++i) a[i] = gn_times(a[i], w[i]);
  const T* src = x + ch.first_row * C;
  T* dst = out + ch.first_row * C;
  gn_rows<P>(
      r0, ch.rows, lanes, [&](P& p, int r) { sp.load(p, src + static_cast<int64_t>(r) * C); },
      [&](P& p, int r) {
        ct v[VE];
        p.unpack(v);
#pragma unroll
        for (int i = 0; i < VE; ++i) v[i] = gn_act<ACT>(gn_affine(gn_centred(v[i], mu[i]), a[i], b[i]));
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
    // d = x - mu, z = d * (s w) + b; s * sum dz d is the sum of dz u
    ct mu[VE], s[VE], a[VE] = {}, b[VE] = {}, dw[VE], db[VE];
    gn_spread(mean + sg, sp, cpg, mu);
    gn_spread(rstd + sg, sp, cpg, s);
    if constexpr (ACT != kGnNone) {
      load_params<T>(weight, pl, sp, wide != 0, a);
      load_params<T>(bias, pl, sp, wide != 0, b);
    }
#pragma unroll
    for (int i = 0; i < VE; ++i) {
      a[i] = gn_times(s[i], a[i]);
      dw[i] = db[i] = 0;
    }
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
            const ct d = gn_centred(xv[i], mu[i]);
            ct dz = gv[i];
            if constexpr (ACT != kGnNone) dz *= gn_slope<ACT>(gn_affine(d, a[i], b[i]));
            dw[i] += dz * d;
            db[i] += dz;
          }
        });
#pragma unroll
    for (int i = 0; i < VE; ++i)
      if (sp.owns(i)) {
        lds_dw[r0 * C + sp.c + i] = dw[i] * s[i];
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
  ct mu[VE], s[VE], w[VE], b[VE], sw[VE], a1[VE], a2[VE];
  gn_spread(mean + sg, sp, cpg, mu);
  gn_spread(rstd + sg, sp, cpg, s);
  gn_spread(m1 + sg, sp, cpg, a1);
  gn_spread(m2 + sg, sp, cpg, a2);
  load_params<T>(weight, pl, sp, wide != 0, w);
  if constexpr (ACT != kGnNone) load_params<T>(bias, pl, sp, wide != 0, b);
#pragma unroll
  for (int i = 0; i < VE; ++i) sw[i] = gn_times(s[i], w[i]);
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
          const ct d = gn_centred(xv[i], mu[i]), u = d * s[i];
          ct dz = gv[i];
          if constexpr (ACT != kGnNone) dz *= gn_slope<ACT>(gn_affine(d, sw[i], b[i]));
          gv[i] = s[i] * (w[i] * dz - a1[i] - u * a2[i]);
        }
        p.g.pack(gv);
        sp.store(p.g, dst + static_cast<int64_t>(r) * C);
      });
}

// ---- small levels: one launch --------------------------------------------------------------------
// Where every level of the call fits the registers of a workgroup per slab of whole groups, the
// workgroup reads its slab once, forms the sums and writes: one launch instead of three and one
// reading instead of two.  A thread holds up to kGnHold vectors of x, in the gradient kGnHoldBwd of
// each tensor (four spill some registers there and lose to three launches); statistics are taken in
// two passes over them (mean, then squares about it).
// Slabs are whole vectors wide.  blockDim.x is chosen by the host (up to 1024).
constexpr int kGnHold = 4, kGnHoldBwd = 2;
constexpr int kGnSlabChannels = 256;  // widest slab: no more channels than threads

struct GnSlab {
  int groups, channels, vecs;  // of a slab
  int slabs;                   // of a row
};

struct GnSmall {
  int n, level, slab, rows, lanes, r0, count;
  int64_t base;  // of the thread's first vector
};

__device__ __forceinline__ GnSmall gn_small(const GnCut& cut, const GnSlab& sl, int C, int VE) {
  GnSmall s;
  const int cell = blockIdx.x / sl.slabs;
  s.slab = blockIdx.x - cell * sl.slabs;
  s.n = cell / cut.levels;
  s.level = cell - s.n * cut.levels;
  s.rows = cut.row_start[s.level + 1] - cut.row_start[s.level];
  s.lanes = blockDim.x / sl.vecs;
  s.r0 = threadIdx.x / sl.vecs;
  s.count = s.r0 < s.lanes ? gn_lane_rows(s.rows, s.r0, s.lanes) : 0;
  const int64_t row = static_cast<int64_t>(s.n) * cut.row_start[cut.levels] + cut.row_start[s.level] + s.r0;
  s.base = row * C + s.slab * sl.channels + (threadIdx.x - s.r0 * sl.vecs) * VE;
  return s;
}

// Sum over rows of what every thread holds per channel of the slab, in two steps: the threads' VE
// values to LDS (`lanes` rows of channels + 1: the odd pitch keeps columns off one bank), then
// blockDim / channels threads a column.  Leaves gn_small_parts() rows of sums at the start of `lds`,
// which the caller adds up after the last barrier.
__device__ __forceinline__ int gn_small_parts(const GnSmall& s, const GnSlab& sl) {
  return min(static_cast<int>(blockDim.x) / sl.channels, min(s.lanes, s.rows));
}
template <int VE>
__device__ __forceinline__ void gn_small_columns(const float (&v)[VE], const GnSmall& s, const GnSlab& sl,
                                                 float* lds) {
  const int pitch = sl.channels + 1, c0 = (threadIdx.x - s.r0 * sl.vecs) * VE;
  if (s.r0 < s.lanes) {
#pragma unroll
    for (int i = 0; i < VE; ++i) lds[s.r0 * pitch + c0 + i] = v[i];
  }
  __syncthreads();
  const int parts = gn_small_parts(s, sl), part = threadIdx.x / sl.channels;
  const int c = threadIdx.x - part * sl.channels, used = min(s.lanes, s.rows);
  float sum = 0;
  if (part < parts)
    for (int r = part; r < used; r += parts) sum += lds[r * pitch + c];
  __syncthreads();
  if (part < parts) lds[part * pitch + c] = sum;
  __syncthreads();
}

// per group; `totals` (groups of the slab) receives the sums
template <int VE>
__device__ __forceinline__ void gn_small_sum(const float (&v)[VE], const GnSmall& s, const GnSlab& sl,
                                             int cpg, float* lds, float* totals) {
  gn_small_columns<VE>(v, s, sl, lds);
  const int pitch = sl.channels + 1, parts = gn_small_parts(s, sl);
  const int width = gn_team_width(blockDim.x, sl.groups), teams = blockDim.x / width;
  const int j = threadIdx.x & (width - 1);
  for (int g = threadIdx.x / width; g < sl.groups; g += teams) {
    float sum = 0;
    for (int q = j; q < parts; q += width)
      for (int c = 0; c < cpg; ++c) sum += lds[q * pitch + g * cpg + c];
    for (int off = 1; off < width; off <<= 1) sum += __shfl_xor(sum, off, 64);
    if (j == 0) totals[g] = sum;
  }
  __syncthreads();
}

// The same where every vector lies in one group and a wave holds whole rows of the slab: one value a
// thread, shuffles over the wave's rows, one barrier.  Returns the sum of the thread's own group
// (m vectors a group).  `lds`: waves * vecs values of its own: nobody may still read what they held.
// 512 bf16 rows of 256 channels take 6.9 us where the general sum takes 9.9.  (The gradient's sums are
// per channel: 16 values a thread, and exchanging those by shuffles took 13.0 us for 16 x 256 rows
// against 10.5 through LDS.)
__device__ __forceinline__ float gn_small_sum_whole(float v, int m, const GnSlab& sl, float* lds) {
  for (int off = sl.vecs; off < 64; off <<= 1) v += __shfl_xor(v, off, 64);
  const int lane = threadIdx.x & 63, waves = blockDim.x >> 6;
  if (lane < sl.vecs) lds[(threadIdx.x >> 6) * sl.vecs + lane] = v;
  __syncthreads();
  const int first = lane % sl.vecs / m * m;
  float sum = 0;
  for (int q = 0; q < m; ++q)
    for (int w = 0; w < waves; ++w) sum += lds[w * sl.vecs + first + q];
  return sum;
}

// mean and rstd (N, levels, G) may be NULL.  Dynamic LDS: lanes * (channels + 1) + 2 * groups values.
template <typename T, int ACT>
__global__ __launch_bounds__(1024) void gn_small_kernel(
    const T* __restrict__ x, const void* __restrict__ weight, const void* __restrict__ bias,
    T* __restrict__ out, float* __restrict__ mean, float* __restrict__ rstd, GnCut cut, GnSlab sl, int C,
    int G, int param_levels, float eps, int wide) {
  constexpr int VE = 16 / sizeof(T);
  extern __shared__ __align__(16) char gn_lds[];
  float* lds = reinterpret_cast<float*>(gn_lds);
  const GnSmall s = gn_small(cut, sl, C, VE);
  const int cpg = C / G;
  const int64_t step = static_cast<int64_t>(s.lanes) * C;
  Pack<T, VE> p[kGnHold];
#pragma unroll
  for (int i = 0; i < kGnHold; ++i)
    if (i < s.count) p[i].template load<false>(x + s.base + i * step);
  const Span<VE, kRowEven> sp = {static_cast<int>((threadIdx.x - s.r0 * sl.vecs) * VE), 0, VE};
  const int64_t pc = (param_levels > 1 ? static_cast<int64_t>(s.level) * C : 0) + s.slab * sl.channels;
  float sum[VE], mu[VE], a[VE], w[VE], b[VE];
  load_params<T>(weight, pc, sp, wide != 0, w);
  load_params<T>(bias, pc, sp, wide != 0, b);
#pragma unroll
  for (int e = 0; e < VE; ++e) sum[e] = 0;
#pragma unroll
  for (int i = 0; i < kGnHold; ++i)
    if (i < s.count) {
      float v[VE];
      p[i].unpack(v);
#pragma unroll
      for (int e = 0; e < VE; ++e) sum[e] += v[e];
    }
  const float inv = 1.f / (static_cast<float>(s.rows) * static_cast<float>(cpg));
  const bool whole = cpg % VE == 0 && 64 % sl.vecs == 0;
  const int m = whole ? cpg / VE : 1;
  float* totals = lds + s.lanes * (sl.channels + 1);
  float* squares = totals + sl.groups;
  if (whole) {
    float t = 0;
#pragma unroll
    for (int e = 0; e < VE; ++e) t += sum[e];
    t = gn_times(gn_small_sum_whole(t, m, sl, lds), inv);
#pragma unroll
    for (int e = 0; e < VE; ++e) mu[e] = t;
  } else {
    gn_small_sum<VE>(sum, s, sl, cpg, lds, totals);
    gn_spread(totals, sp, cpg, mu);
#pragma unroll
    for (int e = 0; e < VE; ++e) mu[e] = gn_times(mu[e], inv);
  }
#pragma unroll
  for (int e = 0; e < VE; ++e) sum[e] = 0;
#pragma unroll
  for (int i = 0; i < kGnHold; ++i)
    if (i < s.count) {
      float v[VE];
      p[i].unpack(v);
#pragma unroll
      for (int e = 0; e < VE; ++e) sum[e] += (v[e] - mu[e]) * (v[e] - mu[e]);
    }
  const int64_t cell = (static_cast<int64_t>(s.n) * cut.levels + s.level) * G + s.slab * sl.groups;
  if (whole) {
    float t = 0;
#pragma unroll
    for (int e = 0; e < VE; ++e) t += sum[e];
    // (behind the first sum's values, which other waves may still read; 2 * waves * vecs <= lanes *
    // channels, as a slab has vecs <= 64 and four channels or more a vector)
    t = gn_rstd(gn_small_sum_whole(t, m, sl, lds + (blockDim.x >> 6) * sl.vecs), inv, eps);
#pragma unroll
    for (int e = 0; e < VE; ++e) a[e] = t;
    const int kv = sp.c / VE;
    if (mean != nullptr && s.r0 == 0 && kv % m == 0) {
      mean[cell + kv / m] = mu[0];
      rstd[cell + kv / m] = t;
    }
  } else {
    gn_small_sum<VE>(sum, s, sl, cpg, lds, squares);
    if (mean != nullptr)
      for (int g = threadIdx.x; g < sl.groups; g += blockDim.x) {
        mean[cell + g] = gn_times(totals[g], inv);
        rstd[cell + g] = gn_rstd(squares[g], inv, eps);
      }
    gn_spread(squares, sp, cpg, a);
#pragma unroll
    for (int e = 0; e < VE; ++e) a[e] = gn_rstd(a[e], inv, eps);
  }
#pragma unroll
  for (int e = 0; e < VE; ++e) a[e] = gn_times(a[e], w[e]);
#pragma unroll
  for (int i = 0; i < kGnHold; ++i)
    if (i < s.count) {
      float v[VE];
      p[i].unpack(v);
#pragma unroll
      for (int e = 0; e < VE; ++e) v[e] = gn_act<ACT>(gn_affine(gn_centred(v[e], mu[e]), a[e], b[e]));
      p[i].pack(v);
      p[i].template store<false>(out + s.base + i * step);
    }
}

// partial (one row of 2 C sums per (sample, level): dz * u, then dz) or, with `direct`, the gradients
// themselves (one sample, parameters per level); grad_weight NULL: neither.  grad_x may be NULL.
template <typename T, int ACT>
__global__ __launch_bounds__(1024) void gn_small_bwd_kernel(
    const T* __restrict__ grad_out, const T* __restrict__ x, const void* __restrict__ weight,
    const void* __restrict__ bias, const float* __restrict__ mean, const float* __restrict__ rstd,
    T* __restrict__ grad_x, float* __restrict__ partial, void* __restrict__ grad_weight,
    void* __restrict__ grad_bias, GnCut cut, GnSlab sl, int C, int G, int param_levels, int wide) {
  constexpr int VE = 16 / sizeof(T), HOLD = kGnHoldBwd;
  extern __shared__ __align__(16) char gn_lds[];
  float* lds = reinterpret_cast<float*>(gn_lds);
  const GnSmall s = gn_small(cut, sl, C, VE);
  const int cpg = C / G, pitch = sl.channels + 1;
  float* columns = lds + s.lanes * pitch;  // dw, db of the slab's channels
  float* totals = columns + 2 * sl.channels;
  const int64_t step = static_cast<int64_t>(s.lanes) * C;
  Pack<T, VE> px[HOLD], pg[HOLD];
#pragma unroll
  for (int i = 0; i < HOLD; ++i)
    if (i < s.count) {
      px[i].template load<false>(x + s.base + i * step);
      pg[i].template load<false>(grad_out + s.base + i * step);
    }
  const int c0 = (threadIdx.x - s.r0 * sl.vecs) * VE;
  const Span<VE, kRowEven> sp = {c0, 0, VE};
  const int64_t cell = (static_cast<int64_t>(s.n) * cut.levels + s.level) * G + s.slab * sl.groups;
  const int64_t pc = (param_levels > 1 ? static_cast<int64_t>(s.level) * C : 0) + s.slab * sl.channels;
  float mu[VE], r[VE], w[VE], b[VE], rw[VE], sums[2][VE];
  gn_spread(mean + cell, sp, cpg, mu);
  gn_spread(rstd + cell, sp, cpg, r);
  load_params<T>(weight, pc, sp, wide != 0, w);
  load_params<T>(bias, pc, sp, wide != 0, b);
#pragma unroll
  for (int e = 0; e < VE; ++e) {
    rw[e] = gn_times(r[e], w[e]);
    sums[0][e] = sums[1][e] = 0;
  }
#pragma unroll
  for (int i = 0; i < HOLD; ++i)
    if (i < s.count) {
      float xv[VE], gv[VE];
      px[i].unpack(xv);
      pg[i].unpack(gv);
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        const float d = gn_centred(xv[e], mu[e]), u = d * r[e];
        float dz = gv[e];
        if constexpr (ACT != kGnNone) dz *= gn_slope<ACT>(gn_affine(d, rw[e], b[e]));
        sums[0][e] += dz * u;
        sums[1][e] += dz;
      }
    }
  const int parts = gn_small_parts(s, sl);
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    gn_small_columns<VE>(sums[k], s, sl, lds);
    for (int c = threadIdx.x; c < sl.channels; c += blockDim.x) {
      float sum = 0;
      for (int q = 0; q < parts; ++q) sum += lds[q * pitch + c];
      columns[k * sl.channels + c] = sum;
    }
    __syncthreads();
  }
  const int64_t slot = static_cast<int64_t>(s.n) * cut.levels + s.level;
  if (grad_weight != nullptr)
    for (int c = threadIdx.x; c < sl.channels; c += blockDim.x) {
      if (partial != nullptr) {
        partial[slot * 2 * C + s.slab * sl.channels + c] = columns[c];
        partial[(slot * 2 + 1) * C + s.slab * sl.channels + c] = columns[sl.channels + c];
      } else {
        store_param<T>(grad_weight, pc + c, columns[c], wide != 0);
        store_param<T>(grad_bias, pc + c, columns[sl.channels + c], wide != 0);
      }
    }
  if (grad_x == nullptr) return;
  const float inv = 1.f / (static_cast<float>(s.rows) * static_cast<float>(cpg));
  for (int g = threadIdx.x; g < sl.groups; g += blockDim.x) {
    float m1 = 0, m2 = 0;
    for (int c = g * cpg; c < (g + 1) * cpg; ++c) {
      const float wc = load_param<T>(weight, pc + c, wide != 0);
      m1 += columns[sl.channels + c] * wc;
      m2 += columns[c] * wc;
    }
    totals[g] = m1 * inv;
    totals[sl.groups + g] = m2 * inv;
  }
  __syncthreads();
  float m1[VE], m2[VE];
  gn_spread(totals, sp, cpg, m1);
  gn_spread(totals + sl.groups, sp, cpg, m2);
#pragma unroll
  for (int i = 0; i < HOLD; ++i)
    if (i < s.count) {
      float xv[VE], gv[VE];
      px[i].unpack(xv);
      pg[i].unpack(gv);
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        const float d = gn_centred(xv[e], mu[e]), u = d * r[e];
        float dz = gv[e];
        if constexpr (ACT != kGnNone) dz *= gn_slope<ACT>(gn_affine(d, rw[e], b[e]));
        gv[e] = r[e] * (w[e] * dz - m1[e] - u * m2[e]);
      }
      pg[i].pack(gv);
      pg[i].template store<false>(grad_x + s.base + i * step);
    }
}

}  // namespace msda
