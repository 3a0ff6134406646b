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
#pragma once

#include "msda_dropout.h"
#include "msda_vec.h"

namespace msda {

template <typename XT, typename RT>
struct AddNormTypes {
  static constexpr int VE = 16 / static_cast<int>(sizeof(RT));  // RT is at least as wide as XT
  using ct = typename Elem<RT>::compute_t;
};

// sums of two values over a team; teams of 256 lanes go through LDS (all threads of the workgroup
// reach the call the same number of times)
template <int TS, typename CT>
__device__ __forceinline__ void team_sum2(CT& a, CT& b, CT* lds) {
  constexpr int W = TS < 64 ? TS : 64;
  a = wave_team_sum<W>(a);
  b = wave_team_sum<W>(b);
  if constexpr (TS > 64) {
    constexpr int WAVES = TS / 64;
    __syncthreads();  // the previous call's values have been read
    if ((threadIdx.x & 63) == 0) {
      lds[(threadIdx.x >> 6) * 2] = a;
      lds[(threadIdx.x >> 6) * 2 + 1] = b;
    }
    __syncthreads();
    a = lds[0];
    b = lds[1];
#pragma unroll
    for (int i = 1; i < WAVES; ++i) {
      a += lds[2 * i];
      b += lds[2 * i + 1];
    }
  }
}

// EVEN: C is a multiple of VE, i.e. every vector lies whole inside its row and starts at an element
// index that is a multiple of VE.
template <typename XT, typename RT, int TS, int NV, bool EVEN>
__global__ __launch_bounds__(256) void add_norm_fwd_kernel(
    const XT* __restrict__ x, const RT* __restrict__ res, const void* __restrict__ weight,
    const void* __restrict__ bias, RT* __restrict__ out,
    typename Elem<RT>::compute_t* __restrict__ mean, typename Elem<RT>::compute_t* __restrict__ rstd,
    const int64_t* __restrict__ rng_state, int64_t rows, int C, uint32_t threshold,
    typename Elem<RT>::compute_t scale, uint32_t site, typename Elem<RT>::compute_t eps, int wide) {
  using ct = typename Elem<RT>::compute_t;
  constexpr int VE = AddNormTypes<XT, RT>::VE, TEAMS = 256 / TS;
  __shared__ ct lds[8];
  const int lane = threadIdx.x % TS, team = threadIdx.x / TS;
  DropKey key{};
  if (threshold) key = load_drop_key(rng_state);
  int count[NV];
  ct w[NV][VE], b[NV][VE];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int c = (v * TS + lane) * VE;
    count[v] = EVEN ? (c < C ? VE : 0) : min(max(C - c, 0), VE);
#pragma unroll
    for (int i = 0; i < VE; ++i) {
      const bool in = i < count[v];
      w[v][i] = in ? load_param<RT>(weight, c + i, wide != 0) : ct(0);
      b[v][i] = in ? load_param<RT>(bias, c + i, wide != 0) : ct(0);
    }
  }
  const ct inv_c = ct(1) / static_cast<ct>(C);
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * TEAMS + team; row < rows;
       row += static_cast<int64_t>(gridDim.x) * TEAMS) {
    const int64_t base = row * C;
    Pack<XT, VE> px[NV];
    Pack<RT, VE> pr[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int64_t at = base + (v * TS + lane) * VE;
      if (count[v] > 0) {
        px[v].load(x + at, EVEN ? VE : count[v]);
        pr[v].load(res + at, EVEN ? VE : count[v]);
      } else {
        px[v].zero();
        pr[v].zero();
      }
    }
    ct h[NV][VE];
    ct sum = 0, unused = 0;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      ct xv[VE];
      px[v].unpack(xv);
      pr[v].unpack(h[v]);
      uint32_t keep = 0xFFFFFFFFu;
      if (threshold)
        keep = keep_bits<VE, EVEN>(key, base + (v * TS + lane) * VE, site, threshold);
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        h[v][i] += (keep >> i) & 1u ? xv[i] * scale : ct(0);
        sum += h[v][i];
      }
    }
    team_sum2<TS>(sum, unused, lds);
    const ct mu = sum * inv_c;
    ct sq = 0;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        h[v][i] -= mu;
        if (i < count[v]) sq += h[v][i] * h[v][i];
      }
    team_sum2<TS>(sq, unused, lds);
    const ct s = ct(1) / sqrt(sq * inv_c + eps);
    if (mean != nullptr && lane == 0) {
      mean[row] = mu;
      rstd[row] = s;
    }
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      if (count[v] == 0) continue;
#pragma unroll
      for (int i = 0; i < VE; ++i) h[v][i] = h[v][i] * s * w[v][i] + b[v][i];
      Pack<RT, VE> po;
      po.pack(h[v]);
      po.store(out + base + (v * TS + lane) * VE, EVEN ? VE : count[v]);
    }
  }
}

// grad_x or grad_res may be NULL (not wanted, or equal to the other); `partial` (one row of
// 2 C sums per workgroup: dy * u, then dy) may be NULL.
template <typename XT, typename RT, int TS, int NV, bool EVEN>
__global__ __launch_bounds__(256) void add_norm_bwd_kernel(
    const RT* __restrict__ grad_out, const XT* __restrict__ x, const RT* __restrict__ res,
    const void* __restrict__ weight, const typename Elem<RT>::compute_t* __restrict__ mean,
    const typename Elem<RT>::compute_t* __restrict__ rstd, XT* __restrict__ grad_x,
    RT* __restrict__ grad_res, typename Elem<RT>::compute_t* __restrict__ partial,
    const int64_t* __restrict__ rng_state, int64_t rows, int C, uint32_t threshold,
    typename Elem<RT>::compute_t scale, uint32_t site, int wide) {
  using ct = typename Elem<RT>::compute_t;
  constexpr int VE = AddNormTypes<XT, RT>::VE, TEAMS = 256 / TS;
  __shared__ ct lds[256 * VE];
  const int lane = threadIdx.x % TS, team = threadIdx.x / TS;
  DropKey key{};
  if (threshold) key = load_drop_key(rng_state);
  int count[NV];
  ct w[NV][VE], dw[NV][VE], db[NV][VE];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int c = (v * TS + lane) * VE;
    count[v] = EVEN ? (c < C ? VE : 0) : min(max(C - c, 0), VE);
#pragma unroll
    for (int i = 0; i < VE; ++i) {
      w[v][i] = i < count[v] ? load_param<RT>(weight, c + i, wide != 0) : ct(0);
      dw[v][i] = db[v][i] = 0;
    }
  }
  const ct inv_c = ct(1) / static_cast<ct>(C);
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * TEAMS + team; row < rows;
       row += static_cast<int64_t>(gridDim.x) * TEAMS) {
    const int64_t base = row * C;
    Pack<XT, VE> px[NV];
    Pack<RT, VE> pr[NV], pg[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int64_t at = base + (v * TS + lane) * VE;
      if (count[v] > 0) {
        const int n = EVEN ? VE : count[v];
        px[v].load(x + at, n);
        pr[v].load(res + at, n);
        pg[v].load(grad_out + at, n);
      } else {
        px[v].zero();
        pr[v].zero();
        pg[v].zero();
      }
    }
    const ct mu = mean[row], s = rstd[row];
    ct u[NV][VE], g[NV][VE];
    uint32_t keep[NV];
    ct sum_g = 0, sum_gu = 0;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      ct xv[VE];
      px[v].unpack(xv);
      pr[v].unpack(u[v]);
      pg[v].unpack(g[v]);
      keep[v] = 0xFFFFFFFFu;
      if (threshold)
        keep[v] = keep_bits<VE, EVEN>(key, base + (v * TS + lane) * VE, site, threshold);
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        const ct h = u[v][i] + ((keep[v] >> i) & 1u ? xv[i] * scale : ct(0));
        u[v][i] = (h - mu) * s;
        // columns behind the row hold g = 0: they add nothing to any sum
        if (i < count[v]) {
          dw[v][i] += g[v][i] * u[v][i];
          db[v][i] += g[v][i];
          g[v][i] *= w[v][i];
          sum_g += g[v][i];
          sum_gu += g[v][i] * u[v][i];
        }
      }
    }
    team_sum2<TS>(sum_g, sum_gu, lds);
    const ct m1 = sum_g * inv_c, m2 = sum_gu * inv_c;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      if (count[v] == 0) continue;
      const int64_t at = base + (v * TS + lane) * VE;
      const int n = EVEN ? VE : count[v];
#pragma unroll
      for (int i = 0; i < VE; ++i) g[v][i] = s * (g[v][i] - m1 - u[v][i] * m2);
      if (grad_res != nullptr) {
        Pack<RT, VE> po;
        po.pack(g[v]);
        po.store(grad_res + at, n);
      }
      if (grad_x != nullptr) {
#pragma unroll
        for (int i = 0; i < VE; ++i) g[v][i] = (keep[v] >> i) & 1u ? g[v][i] * scale : ct(0);
        Pack<XT, VE> po;
        po.pack(g[v]);
        po.store(grad_x + at, n);
      }
    }
  }
  if (partial == nullptr) return;
  // sums over the workgroup's teams, one vector slot at a time
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < VE; ++i)
        lds[(team * VE + i) * TS + lane] = k == 0 ? dw[v][i] : db[v][i];
      __syncthreads();
      for (int j = threadIdx.x; j < TS * VE; j += 256) {
        const int c = v * TS * VE + j;  // column; held by lane j / VE at place j % VE
        if (c < C) {
          ct acc = 0;
          for (int t = 0; t < TEAMS; ++t) acc += lds[(t * VE + j % VE) * TS + j / VE];
          partial[(static_cast<int64_t>(blockIdx.x) * 2 + k) * C + c] = acc;
        }
      }
    }
}

}  // namespace msda
