// out = LayerNorm(residual + dropout(x)) * weight + bias and its gradient (gfx950): the epilogue
// behind the attention and behind the feed-forward network of an encoder layer.
//
//   h = r + keep * x * scale,  mu = mean_c h,  s = 1 / sqrt(mean_c (h - mu)^2 + eps)
//   y = (h - mu) * s * w + b
//   with u = (h - mu) * s and g = dy * w:
//   dh = s * (g - mean_c g - u * mean_c (g u)),  dr = dh,  dx = keep * scale * dh,
//   dw = sum_rows dy * u,  db = sum_rows dy
//
// Both directions read and write every element once.  The gradient recomputes h from x and r
// (and the dropout mask from its counters) instead of storing h: one tensor more to read there, one
// less to write in the forward, and no rounding of h to 16 bits.
//
// A team of TS lanes owns a row; each lane holds NV vectors of VE = 16 bytes (of the wider type) in
// registers, so the variance is taken about the mean in a second pass over registers.  Statistics,
// h and all sums are in 32 bits (64 for fp64).
//
// Bound by HBM where rows are many (MI355X, 344064 rows of 256 fp32 columns, dropout 0.1): forward
// 1.06 GB in 168 us, 6.3 TB/s; backward 1.78 GB in 293 us, 6.1 TB/s, and 15 us for the column sums.
#pragma once

#include "msda_dropout.h"
#include "msda_vec.h"

namespace msda {

template <typename XT, typename RT>
struct AddNormTypes {
  static constexpr int VE = 16 / static_cast<int>(sizeof(RT));  // RT is at least as wide as XT
  using ct = typename Elem<RT>::compute_t;
};

// Sums of K values over a team; teams of 256 lanes go through LDS (2 * K * waves values; all
// threads of the workgroup reach the call the same number of times).
template <int TS, int K, typename CT>
__device__ __forceinline__ void team_sums(CT (&v)[K], CT* lds) {
  constexpr int W = TS < 64 ? TS : 64;
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = wave_team_sum<W>(v[k]);
  if constexpr (TS > 64) {
    constexpr int WAVES = TS / 64;
    __syncthreads();  // the previous call's values have been read
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int k = 0; k < K; ++k) lds[(threadIdx.x >> 6) * K + k] = v[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
      v[k] = lds[k];
#pragma unroll
      for (int i = 1; i < WAVES; ++i) v[k] += lds[i * K + k];
    }
  }
}

// A team takes NR rows a step: their loads are in flight together and the chains of their sums
// overlap (64 lanes x 1 vector, one, two, four rows: 179, 166, 169 us for 344064 rows of 256 fp32
// columns).
template <typename XT, typename RT, int TS, int NV, int NR, int MODE>
__global__ __launch_bounds__(256) void add_norm_fwd_kernel(
    const XT* __restrict__ x, const RT* __restrict__ res, const void* __restrict__ weight,
    const void* __restrict__ bias, RT* __restrict__ out,
    typename Elem<RT>::compute_t* __restrict__ mean, typename Elem<RT>::compute_t* __restrict__ rstd,
    const int64_t* __restrict__ rng_state, int64_t rows, int C, uint32_t threshold,
    typename Elem<RT>::compute_t scale, uint32_t site, typename Elem<RT>::compute_t eps, int wide) {
  using ct = typename Elem<RT>::compute_t;
  constexpr int VE = AddNormTypes<XT, RT>::VE, TEAMS = 256 / TS;
  __shared__ ct lds[4 * NR];
  const int lane = threadIdx.x % TS, team = threadIdx.x / TS;
  DropKey key{};
  if (threshold) key = load_drop_key(rng_state);
  const ct inv_c = ct(1) / static_cast<ct>(C);
  for (int64_t row0 = (static_cast<int64_t>(blockIdx.x) * TEAMS + team) * NR; row0 < rows;
       row0 += static_cast<int64_t>(gridDim.x) * TEAMS * NR) {
    Pack<XT, VE> px[NR][NV];
    Pack<RT, VE> pr[NR][NV];
#pragma unroll
    for (int k = 0; k < NR; ++k) {
      const int64_t row = row0 + k < rows ? row0 + k : row0;  // (a row too many is not stored)
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const auto sp = Span<VE, MODE>::at(v * TS + lane, C);
        sp.load(px[k][v], x + row * C);
        sp.load(pr[k][v], res + row * C);
      }
    }
    ct h[NR][NV][VE], sum[NR];
#pragma unroll
    for (int k = 0; k < NR; ++k) {
      sum[k] = 0;
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const auto sp = Span<VE, MODE>::at(v * TS + lane, C);
        ct xv[VE];
        px[k][v].unpack(xv);
        pr[k][v].unpack(h[k][v]);
        uint32_t keep = 0xFFFFFFFFu;
        if (threshold) keep = keep_bits<VE, MODE == kRowEven>(key, (row0 + k) * C + sp.c, site, threshold);
#pragma unroll
        for (int i = 0; i < VE; ++i) {
          h[k][v][i] += (keep >> i) & 1u ? xv[i] * scale : ct(0);
          if (sp.owns(i)) sum[k] += h[k][v][i];
        }
      }
    }
    team_sums<TS, NR>(sum, lds);
    ct sq[NR];
#pragma unroll
    for (int k = 0; k < NR; ++k) {
      sum[k] *= inv_c;
      sq[k] = 0;
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const auto sp = Span<VE, MODE>::at(v * TS + lane, C);
#pragma unroll
        for (int i = 0; i < VE; ++i) {
          h[k][v][i] -= sum[k];
          if (sp.owns(i)) sq[k] += h[k][v][i] * h[k][v][i];
        }
      }
    }
    team_sums<TS, NR>(sq, lds);
#pragma unroll
    for (int k = 0; k < NR; ++k) {
      sq[k] = ct(1) / sqrt(sq[k] * inv_c + eps);
      if (mean != nullptr && lane == 0 && row0 + k < rows) {
        mean[row0 + k] = sum[k];
        rstd[row0 + k] = sq[k];
      }
    }
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const auto sp = Span<VE, MODE>::at(v * TS + lane, C);
      ct w[VE], b[VE];
      load_params<RT>(weight, 0, sp, wide != 0, w);
      load_params<RT>(bias, 0, sp, wide != 0, b);
#pragma unroll
      for (int k = 0; k < NR; ++k) {
        if (row0 + k >= rows) continue;
#pragma unroll
        for (int i = 0; i < VE; ++i) h[k][v][i] = h[k][v][i] * sq[k] * w[i] + b[i];
        Pack<RT, VE> po;
        po.pack(h[k][v]);
        sp.store(po, out + (row0 + k) * C);
      }
    }
  }
}

// grad_x or grad_res may be NULL (not wanted, or equal to the other); `partial` (one row of
// 2 C sums per workgroup: dy * u, then dy) may be NULL.
// A workgroup of THREADS takes `steps` times NR rows a team and ends: where 1024 workgroups walked
// all rows instead, the same traffic ran at 5.1 TB/s against 5.9 (the phases of long-lived
// workgroups fall into step; short ones keep reads and writes mixed).
template <typename XT, typename RT, int TS, int NV, int NR, int THREADS, int MODE>
__global__ __launch_bounds__(THREADS) void add_norm_bwd_kernel(
    const RT* __restrict__ grad_out, const XT* __restrict__ x, const RT* __restrict__ res,
    const void* __restrict__ weight, const typename Elem<RT>::compute_t* __restrict__ mean,
    const typename Elem<RT>::compute_t* __restrict__ rstd, XT* __restrict__ grad_x,
    RT* __restrict__ grad_res, typename Elem<RT>::compute_t* __restrict__ partial,
    const int64_t* __restrict__ rng_state, int64_t rows, int C, int steps, uint32_t threshold,
    typename Elem<RT>::compute_t scale, uint32_t site, int wide) {
  using ct = typename Elem<RT>::compute_t;
  constexpr int VE = AddNormTypes<XT, RT>::VE, TEAMS = THREADS / TS;
  __shared__ ct lds[THREADS * VE];
  const int lane = threadIdx.x % TS, team = threadIdx.x / TS;
  DropKey key{};
  if (threshold) key = load_drop_key(rng_state);
  ct w[NV][VE], dw[NV][VE], db[NV][VE];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    load_params<RT>(weight, 0, Span<VE, MODE>::at(v * TS + lane, C), wide != 0, w[v]);
#pragma unroll
    for (int i = 0; i < VE; ++i) dw[v][i] = db[v][i] = 0;
  }
  const ct inv_c = ct(1) / static_cast<ct>(C);
  const int64_t begin = static_cast<int64_t>(blockIdx.x) * TEAMS * NR * steps;
  for (int step = 0; step < steps; ++step) {
    const int64_t row0 = begin + (static_cast<int64_t>(step) * TEAMS + team) * NR;
    if (row0 >= rows && TS <= 64) break;  // (a whole workgroup a row: all or none of it, below)
    if (TS > 64 && begin + static_cast<int64_t>(step) * TEAMS * NR >= rows) break;
    Pack<XT, VE> px[NR][NV];
    Pack<RT, VE> pr[NR][NV], pg[NR][NV];
    ct mu[NR], s[NR];
#pragma unroll
    for (int k = 0; k < NR; ++k) {
      const int64_t row = row0 + k < rows ? row0 + k : rows - 1;  // (a row too many counts nowhere)
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const auto sp = Span<VE, MODE>::at(v * TS + lane, C);
        sp.load(px[k][v], x + row * C);
        sp.load(pr[k][v], res + row * C);
        sp.load(pg[k][v], grad_out + row * C);
      }
      mu[k] = mean[row];
      s[k] = rstd[row];
    }
    ct u[NR][NV][VE], g[NR][NV][VE];
    uint32_t keep[NR][NV];
    ct sums[2 * NR];  // of g, of g * u
#pragma unroll
    for (int k = 0; k < NR; ++k) {
      const bool in = row0 + k < rows;
      sums[2 * k] = sums[2 * k + 1] = 0;
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const auto sp = Span<VE, MODE>::at(v * TS + lane, C);
        ct xv[VE];
        px[k][v].unpack(xv);
        pr[k][v].unpack(u[k][v]);
        pg[k][v].unpack(g[k][v]);
        keep[k][v] = 0xFFFFFFFFu;
        if (threshold)
          keep[k][v] = keep_bits<VE, MODE == kRowEven>(key, (row0 + k) * C + sp.c, site, threshold);
#pragma unroll
        for (int i = 0; i < VE; ++i) {
          const ct h = u[k][v][i] + ((keep[k][v] >> i) & 1u ? xv[i] * scale : ct(0));
          u[k][v][i] = (h - mu[k]) * s[k];
          const ct dy = g[k][v][i];
          g[k][v][i] = dy * w[v][i];
          if (sp.owns(i)) {
            if (in) {
              dw[v][i] += dy * u[k][v][i];
              db[v][i] += dy;
            }
            sums[2 * k] += g[k][v][i];
            sums[2 * k + 1] += g[k][v][i] * u[k][v][i];
          }
        }
      }
    }
    team_sums<TS, 2 * NR>(sums, lds);
#pragma unroll
    for (int k = 0; k < NR; ++k) {
      if (row0 + k >= rows) continue;
      const ct m1 = sums[2 * k] * inv_c, m2 = sums[2 * k + 1] * inv_c;
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const auto sp = Span<VE, MODE>::at(v * TS + lane, C);
#pragma unroll
        for (int i = 0; i < VE; ++i) g[k][v][i] = s[k] * (g[k][v][i] - m1 - u[k][v][i] * m2);
        if (grad_res != nullptr) {
          Pack<RT, VE> po;
          po.pack(g[k][v]);
          sp.store(po, grad_res + (row0 + k) * C);
        }
        if (grad_x != nullptr) {
#pragma unroll
          for (int i = 0; i < VE; ++i)
            g[k][v][i] = (keep[k][v] >> i) & 1u ? g[k][v][i] * scale : ct(0);
          Pack<XT, VE> po;
          po.pack(g[k][v]);
          sp.store(po, grad_x + (row0 + k) * C);
        }
      }
    }
  }
  if (partial == nullptr) return;
  // sums over the workgroup's teams, one vector slot at a time: columns [v * TS * VE, ...)
  ct* dst = partial + static_cast<int64_t>(blockIdx.x) * 2 * C;
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const auto sp = Span<VE, MODE>::at(v * TS + lane, C);
      __syncthreads();
#pragma unroll
      for (int i = 0; i < VE; ++i)
        if (sp.owns(i)) lds[team * TS * VE + sp.c + i - v * TS * VE] = k == 0 ? dw[v][i] : db[v][i];
      __syncthreads();
      for (int j = threadIdx.x; j < TS * VE; j += THREADS) {
        const int c = v * TS * VE + j;
        if (c < C) {
          ct acc = 0;
          for (int t = 0; t < TEAMS; ++t) acc += lds[t * TS * VE + j];
          dst[static_cast<int64_t>(k) * C + c] = acc;
        }
      }
    }
}

}  // namespace msda
