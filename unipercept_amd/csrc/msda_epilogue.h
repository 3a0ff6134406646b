// C ABI of the operators around the attention: argument checks, launch geometry, dispatch.
#pragma once

#include <math.h>

#include <initializer_list>

#include "msda_addnorm.h"
#include "msda_common.h"
#include "msda_dropout.h"
#include "msda_groupnorm.h"

namespace msda {

// ---- dropout ------------------------------------------------------------------------------------
struct DropArgs {
  uint32_t threshold;  // 0: nothing is dropped, 65536: everything
  double scale;
};

inline bool drop_args(double p, DropArgs* a) {
  if (!(p >= 0.0 && p <= 1.0)) return false;
  double t = nearbyint(p * 65536.0);
  if (p > 0.0 && t < 1.0) t = 1.0;  // only p = 0 drops nothing, only p = 1 everything
  if (p < 1.0 && t > 65535.0) t = 65535.0;
  a->threshold = static_cast<uint32_t>(t);
  a->scale = a->threshold < 65536u ? 65536.0 / (65536.0 - t) : 0.0;
  return true;
}

constexpr int64_t kMaxDropElements = static_cast<int64_t>(1) << 35;  // 32-bit block counter

// Workgroups of a pass over `items` steps of `per_block` a workgroup: one step each, so that loads
// of the next workgroups overlap the stores of the last (a copy of 352 MB, one vector a thread and
// step: 6.8 TB/s so with the streaming hint and 6.1 without, 5.7 and 5.0 with 2048 workgroups that
// loop); more than a launch holds are looped over.
inline unsigned pass_grid(int64_t items, int per_block) {
  const int64_t blocks = (items + per_block - 1) / per_block;
  return static_cast<unsigned>(blocks < (1 << 23) ? blocks : (1 << 23));
}

template <typename T>
int dropout_forward(const void* x, void* out, const int64_t* rng_state, int64_t numel,
                    const DropArgs& d, uint32_t site, bool relu, hipStream_t stream) {
  using ct = typename Elem<T>::compute_t;
  Launches run;
  constexpr int VE = 16 / sizeof(T);
  const dim3 grid(pass_grid((numel + VE - 1) / VE, 256));
#define MSDA_DROP(RELU, DROP)                                                                  \
  run((dropout_kernel<T, RELU, DROP>), grid, dim3(256), 0, stream, static_cast<const T*>(x),   \
      static_cast<T*>(out), rng_state, numel, d.threshold, static_cast<ct>(d.scale), site)
  if (d.threshold) {
    if (relu) MSDA_DROP(true, true);
    else MSDA_DROP(false, true);
  } else {
    if (relu) MSDA_DROP(true, false);
    else MSDA_DROP(false, false);
  }
#undef MSDA_DROP
  return run.rc;
}

template <typename T>
int dropout_relu_backward(const void* grad_out, const void* out, void* grad_x, int64_t numel,
                          const DropArgs& d, hipStream_t stream) {
  Launches run;
  constexpr int VE = 16 / sizeof(T);
  run((dropout_relu_bwd_kernel<T>), dim3(pass_grid((numel + VE - 1) / VE, 256)), dim3(256), 0, stream,
      static_cast<const T*>(grad_out), static_cast<const T*>(out), static_cast<T*>(grad_x), numel,
      static_cast<typename Elem<T>::compute_t>(d.scale));
  return run.rc;
}

// ---- dropout + residual + layer norm ------------------------------------------------------------
constexpr int64_t kMaxNormRowBytes = 16384;  // 256 lanes x 4 vectors x 16 bytes

inline bool add_norm_types(int dtype_x, int dtype_res, int dtype_param) {
  if (elem_size(dtype_x) == 0 || elem_size(dtype_res) == 0) return false;
  const bool half = dtype_x == MSDA_BF16 || dtype_x == MSDA_F16;
  if (dtype_res != dtype_x && !(half && dtype_res == MSDA_F32)) return false;
  return dtype_param == dtype_res || (half && dtype_param == MSDA_F32);
}

inline int add_norm_check(int64_t rows, int C, double p, int site, int dtype_x, int dtype_res,
                          int dtype_param, DropArgs* d) {
  if (rows < 1 || C < 1 || rows > INT32_MAX || site < 0) return MSDA_ESHAPE;
  if (!add_norm_types(dtype_x, dtype_res, dtype_param)) return MSDA_EDTYPE;
  if (C * static_cast<int64_t>(elem_size(dtype_res)) > kMaxNormRowBytes) return MSDA_ESHAPE;
  if (!drop_args(p, d)) return MSDA_ESHAPE;
  if (d->threshold && rows * C > kMaxDropElements) return MSDA_ESHAPE;
  return MSDA_OK;
}

// Lanes of a row's team and vectors of a lane, for rows of `vecs` vectors.  Few lanes with several
// vectors spend less on sums over lanes; rows of more than 256 vectors take four waves.  Measured on
// MI355X, 344064 rows of 256 columns, dropout 0.1, forward / backward in us:
//   fp32 (64 vectors)   64 x 1: 172 / 303   32 x 2: 168 / 316   16 x 4: 168 / 328
//   bf16 with fp32 res. 64 x 1: 149 / 251   32 x 2: 139 / 252   16 x 4: 141 / 264
//   bf16 (32 vectors)   32 x 1: 106 / 161   16 x 2:  91 / 178
// (the backward keeps more of a row in registers and gains less from the shorter sums).
// Rows between two shapes take one that leaves few lanes empty (fp16, forward, 21502 rows of 520
// columns, 65 vectors: 64 x 2 19.0, 32 x 3 15.9; of 1030, 129 vectors: 64 x 4 48, 64 x 3 34; of 258,
// 33 vectors: 64 x 1 15.5, 16 x 3 11.0).  16 x 3, 32 x 3, 64 x 3 and 64 x 4 were chosen by these times of
// the forward and serve the backward too, where no other shape was timed (fp16, 21502 rows with the column
// sums: 16 x 3, 258 columns 38 us; 32 x 3, 515 columns 50; 64 x 3, 1030 columns 75; 64 x 4, 1537 columns
// 153 where 1536 take 77: on odd 16-bit rows that one uses all 256 registers and spills about 20).
struct AddNormTeam {
  int TS, NV;
};
inline AddNormTeam add_norm_team(int vecs, bool f64, bool backward) {
  if (f64) return vecs <= 64 ? AddNormTeam{64, 1} : vecs <= 256 ? AddNormTeam{64, 4} : AddNormTeam{256, 4};
  if (vecs <= 16) return {16, 1};
  if (vecs <= 32) return backward ? AddNormTeam{32, 1} : AddNormTeam{16, 2};
  if (vecs <= 48) return {16, 3};
  if (vecs <= 64) return backward ? AddNormTeam{64, 1} : AddNormTeam{32, 2};
  if (vecs <= 96) return {32, 3};
  if (vecs <= 128) return {64, 2};
  if (vecs <= 192) return {64, 3};
  if (vecs <= 256) return {64, 4};
  if (vecs <= 512) return {256, 2};
  return {256, 4};
}
// threads of a workgroup and rows in flight of a team in the backward
constexpr int add_norm_bwd_threads(int TS) { return TS > 64 ? 256 : 512; }
constexpr int add_norm_bwd_rows(int NV) { return NV == 1 ? 2 : 1; }

// Steps of a workgroup of the backward (NR rows a team each): up to kBwdTeamRows rows a team where
// there are many rows, one step where there are few, so that they spread over the chip.  Longer
// workgroups leave fewer partial rows and run slower (344064 rows of 256 fp32 columns, 8 teams of 64
// lanes, kernel and column sums: 2 rows a team 320 + 21 us, 4 rows 296 + 15, 8 rows 310 + 14, 16 rows
// 330 + 9).
constexpr int kBwdTeamRows = 4;
struct AddNormGrid {
  int steps;
  int64_t blocks;
};
inline AddNormGrid add_norm_bwd_grid(int64_t rows, int C, int dtype_res) {
  const int VE = 16 / static_cast<int>(elem_size(dtype_res)), vecs = (C + VE - 1) / VE;
  const AddNormTeam team = add_norm_team(vecs, dtype_res == MSDA_F64, true);
  const int NR = add_norm_bwd_rows(team.NV);
  const int64_t per_step = static_cast<int64_t>(add_norm_bwd_threads(team.TS) / team.TS) * NR;
  const int most = kBwdTeamRows / NR;
  int64_t steps = rows / (per_step * 512);
  steps = steps < 1 ? 1 : steps > most ? most : steps;
  while ((rows + per_step * steps - 1) / (per_step * steps) > (1 << 22)) steps *= 2;
  return {static_cast<int>(steps), (rows + per_step * steps - 1) / (per_step * steps)};
}

// Partial rows that one workgroup a tile of columns adds up; more are added in segments first (11 MB
// of partial rows: 14 us in one step, 8 in two; 22 MB: 26 and 15).
constexpr int kColumnSplit = 1024, kColumnSegments = 16;

struct AddNormCall {
  const void *grad_out, *x, *res, *weight, *bias;
  void *out, *mean, *rstd, *grad_x, *grad_res, *grad_weight, *grad_bias, *partial;
  const int64_t* rng_state;
  int64_t rows;
  int C, dtype_res;
  DropArgs drop;
  uint32_t site;
  double eps;
  bool wide;
  hipStream_t stream;
};

template <typename XT, typename RT, int TS, int NV, int MODE>
int add_norm_forward(const AddNormCall& a) {
  using ct = typename Elem<RT>::compute_t;
  Launches run;
  constexpr int NR = NV == 1 ? 2 : 1;
  run((add_norm_fwd_kernel<XT, RT, TS, NV, NR, MODE>), dim3(pass_grid(a.rows, 256 / TS * NR)),
      dim3(256), 0, a.stream, static_cast<const XT*>(a.x), static_cast<const RT*>(a.res), a.weight,
      a.bias, static_cast<RT*>(a.out), static_cast<ct*>(a.mean), static_cast<ct*>(a.rstd),
      a.rng_state, a.rows, a.C, a.drop.threshold, static_cast<ct>(a.drop.scale), a.site,
      static_cast<ct>(a.eps), a.wide ? 1 : 0);
  return run.rc;
}

template <typename XT, typename RT, int TS, int NV, int MODE>
int add_norm_backward(const AddNormCall& a) {
  using ct = typename Elem<RT>::compute_t;
  Launches run;
  constexpr int THREADS = add_norm_bwd_threads(TS), NR = add_norm_bwd_rows(NV);
  const AddNormGrid grid = add_norm_bwd_grid(a.rows, a.C, a.dtype_res);
  run((add_norm_bwd_kernel<XT, RT, TS, NV, NR, THREADS, MODE>),
      dim3(static_cast<unsigned>(grid.blocks)), dim3(THREADS), 0, a.stream,
      static_cast<const RT*>(a.grad_out), static_cast<const XT*>(a.x),
      static_cast<const RT*>(a.res), a.weight, static_cast<const ct*>(a.mean),
      static_cast<const ct*>(a.rstd), static_cast<XT*>(a.grad_x), static_cast<RT*>(a.grad_res),
      static_cast<ct*>(a.partial), a.rng_state, a.rows, a.C, grid.steps, a.drop.threshold,
      static_cast<ct>(a.drop.scale), a.site, a.wide ? 1 : 0);
  if (a.partial != nullptr) {
    const dim3 tiles((a.C + 15) / 16, 2, 1);
    const ct* src = static_cast<const ct*>(a.partial);
    ct* next = static_cast<ct*>(a.partial) + grid.blocks * 2 * a.C;
    int total = static_cast<int>(grid.blocks);
    if (total > kColumnSplit) {
      run((column_sums_kernel<RT>), dim3(tiles.x, 2, kColumnSegments), dim3(1024), 0, a.stream, src,
          next, nullptr, nullptr, total, a.C, 1);
      src = next;
      total = kColumnSegments;
    }
    run((column_sums_kernel<RT>), tiles, dim3(1024), 0, a.stream, src, nullptr, a.grad_weight,
        a.grad_bias, total, a.C, a.wide ? 1 : 0);
  }
  return run.rc;
}

template <typename XT, typename RT, int MODE>
int add_norm_width(const AddNormCall& a, bool backward) {
  const int vecs = (a.C + AddNormTypes<XT, RT>::VE - 1) / AddNormTypes<XT, RT>::VE;
  const AddNormTeam team = add_norm_team(vecs, sizeof(RT) == 8, backward);
#define MSDA_TEAM(TS, NV)                                                  \
  case TS * 8 + NV:                                                        \
    return backward ? add_norm_backward<XT, RT, TS, NV, MODE>(a)           \
                    : add_norm_forward<XT, RT, TS, NV, MODE>(a)
  if constexpr (sizeof(RT) == 8) {
    switch (team.TS * 8 + team.NV) {
      MSDA_TEAM(64, 1);
      MSDA_TEAM(64, 4);
      MSDA_TEAM(256, 4);
    }
  } else {
    switch (team.TS * 8 + team.NV) {
      MSDA_TEAM(16, 1);
      MSDA_TEAM(16, 3);
      MSDA_TEAM(32, 3);
      MSDA_TEAM(64, 2);
      MSDA_TEAM(64, 3);
      MSDA_TEAM(64, 4);
      MSDA_TEAM(256, 2);
      MSDA_TEAM(256, 4);
      case 16 * 8 + 2: return add_norm_forward<XT, RT, 16, 2, MODE>(a);
      case 32 * 8 + 1: return add_norm_backward<XT, RT, 32, 1, MODE>(a);
      case 32 * 8 + 2: return add_norm_forward<XT, RT, 32, 2, MODE>(a);
      case 64 * 8 + 1: return add_norm_backward<XT, RT, 64, 1, MODE>(a);
    }
  }
#undef MSDA_TEAM
  return MSDA_ESHAPE;  // (a team that add_norm_team does not name)
}

template <typename XT, typename RT>
int add_norm_run(const AddNormCall& a, bool backward) {
  switch (row_mode(a.C, AddNormTypes<XT, RT>::VE)) {
    case kRowEven: return add_norm_width<XT, RT, kRowEven>(a, backward);
    case kRowOdd: return add_norm_width<XT, RT, kRowOdd>(a, backward);
    default: {
      constexpr int TS = sizeof(RT) == 8 ? 64 : 16;
      return backward ? add_norm_backward<XT, RT, TS, 1, kRowShort>(a)
                      : add_norm_forward<XT, RT, TS, 1, kRowShort>(a);
    }
  }
}

inline int add_norm_dispatch(const AddNormCall& a, int dtype_x, int dtype_res, bool backward) {
  switch (dtype_x) {
    case MSDA_F32: return add_norm_run<float, float>(a, backward);
    case MSDA_F64: return add_norm_run<double, double>(a, backward);
    case MSDA_BF16:
      return dtype_res == MSDA_F32 ? add_norm_run<bf16_t, float>(a, backward)
                                   : add_norm_run<bf16_t, bf16_t>(a, backward);
    default:
      return dtype_res == MSDA_F32 ? add_norm_run<f16_t, float>(a, backward)
                                   : add_norm_run<f16_t, f16_t>(a, backward);
  }
}

// ---- group norm ---------------------------------------------------------------------------------
struct GnPlan {
  GnCut sums, writes;  // chunks of the passes that sum and of those that write
  int param_levels, lanes, tiles;
  int64_t cells;  // (sample, level, group)
};

inline void gn_cut(const int64_t* level_rows, int L, int64_t rows_per_chunk, GnCut* cut) {
  cut->levels = L;
  cut->rows_per_chunk = static_cast<int>(rows_per_chunk);
  cut->row_start[0] = cut->chunk_start[0] = 0;
  for (int l = 0; l < L; ++l) {
    cut->row_start[l + 1] = cut->row_start[l] + static_cast<int>(level_rows[l]);
    cut->chunk_start[l + 1] =
        cut->chunk_start[l] + static_cast<int>((level_rows[l] + rows_per_chunk - 1) / rows_per_chunk);
  }
  cut->chunks = cut->chunk_start[L];
}

inline int gn_plan(const int64_t* level_rows, int N, int S, int C, int G, int L, int param_levels,
                   int activation, int dtype, int dtype_param, GnPlan* plan) {
  if (N < 1 || S < 1 || C < 1 || G < 1 || L < 1 || C % G != 0) return MSDA_ESHAPE;
  if (L > kMaxNormLevels) return MSDA_ELEVELS;
  // threads of a launch: 32 bits
  if (static_cast<int64_t>(N) * L * ((G + 31) / 32) > (1 << 21)) return MSDA_ESHAPE;
  if (param_levels != 1 && param_levels != L) return MSDA_ESHAPE;
  const int64_t e = static_cast<int64_t>(elem_size(dtype));
  if (e == 0 || activation < kGnNone || activation > kGnGelu) return MSDA_EDTYPE;
  if (dtype_param != dtype && !(e == 2 && dtype_param == MSDA_F32)) return MSDA_EDTYPE;
  if (C * e > kMaxNormRowBytes || static_cast<int64_t>(N) * S > INT32_MAX) return MSDA_ESHAPE;
  int64_t sum = 0, longest = 0;
  for (int l = 0; l < L; ++l) {
    if (level_rows[l] < 1 || level_rows[l] > S) return MSDA_ESHAPE;
    sum += level_rows[l];
    longest = level_rows[l] > longest ? level_rows[l] : longest;
  }
  if (sum != S) return MSDA_ESHAPE;
  const int vecs = static_cast<int>((C * e + 15) / 16);
  plan->lanes = gn_lanes(vecs);
  plan->tiles = (vecs + kGnThreads - 1) / kGnThreads;
  plan->param_levels = param_levels;
  plan->cells = static_cast<int64_t>(N) * L * G;
  // Sums: about 2048 workgroups in the call (8 a CU) of at least kGnRowsAhead rows a thread.
  // Writes: the rows that a thread has in flight (twice or four times as many: 165 -> 167, 179 us
  // for the gradient of 344064 rows of 256 fp32 columns).
  const int64_t step = static_cast<int64_t>(kGnRowsAhead) * plan->lanes;
  auto up = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
  int64_t r = up(up(static_cast<int64_t>(N) * S, 2048), step) * step;
  gn_cut(level_rows, L, r < longest ? r : longest, &plan->sums);
  r = step;
  while (static_cast<int64_t>(N) * up(S, r) > (1 << 22)) r *= 2;
  gn_cut(level_rows, L, r < longest ? r : longest, &plan->writes);
  return MSDA_OK;
}

inline size_t gn_compute_size(int dtype) { return dtype == MSDA_F64 ? 8 : 4; }

// values in the workspace: forward: sums of every chunk, and the statistics where the caller has no
// room for them; backward: sums of every chunk per group and per channel, m1 and m2
inline int64_t gn_workspace_values(const GnPlan& plan, int N, int C, int G, bool backward) {
  const int64_t chunks = static_cast<int64_t>(N) * plan.sums.chunks;
  return chunks * 2 * (G + (backward ? C : 0)) + 2 * plan.cells;
}

struct GnCall {
  const void *grad_out, *x, *weight, *bias;
  void *out, *mean, *rstd, *grad_x, *grad_weight, *grad_bias, *workspace;
  int N, C, G;
  double eps;
  bool wide;
  hipStream_t stream;
};

template <typename T, int ACT, int MODE>
int gn_forward(const GnCall& a, const GnPlan& plan) {
  using ct = typename Elem<T>::compute_t;
  const int chunks = a.N * plan.sums.chunks;
  ct* partial = static_cast<ct*>(a.workspace);
  ct* mean = static_cast<ct*>(a.mean);
  ct* rstd = static_cast<ct*>(a.rstd);
  if (mean == nullptr) {
    mean = partial + static_cast<int64_t>(chunks) * 2 * a.G;
    rstd = mean + plan.cells;
  }
  Launches run;
  run((gn_stats_kernel<T, MODE>), dim3(chunks), dim3(kGnThreads), 2 * sizeof(ct) * plan.lanes * a.C,
      a.stream, static_cast<const T*>(a.x), partial, plan.sums, a.C, a.G);
  run((gn_join_kernel<ct>), dim3(a.N * plan.sums.levels, (a.G + kGnJoinGroups - 1) / kGnJoinGroups),
      dim3(kGnThreads), 0, a.stream,
      static_cast<const ct*>(partial), mean, rstd, plan.sums, a.C / a.G, a.G, static_cast<ct>(a.eps));
  run((gn_apply_kernel<T, ACT, MODE>), dim3(a.N * plan.writes.chunks, plan.tiles), dim3(kGnThreads), 0,
      a.stream, static_cast<const T*>(a.x), static_cast<const ct*>(mean), static_cast<const ct*>(rstd),
      a.weight, a.bias, static_cast<T*>(a.out), plan.writes, a.C, a.G, plan.param_levels,
      a.wide ? 1 : 0);
  return run.rc;
}

template <typename T, int ACT, int MODE>
int gn_backward(const GnCall& a, const GnPlan& plan) {
  using ct = typename Elem<T>::compute_t;
  const int chunks = a.N * plan.sums.chunks;
  ct* m1 = static_cast<ct*>(a.workspace);
  ct* m2 = m1 + plan.cells;
  ct* partial_g = m2 + plan.cells;
  ct* partial_c = a.grad_weight != nullptr ? partial_g + static_cast<int64_t>(chunks) * a.G * 2 : nullptr;
  const ct* mean = static_cast<const ct*>(a.mean);
  const ct* rstd = static_cast<const ct*>(a.rstd);
  Launches run;
  run((gn_bwd_stats_kernel<T, ACT, MODE>), dim3(chunks), dim3(kGnThreads),
      2 * sizeof(ct) * plan.lanes * a.C, a.stream, static_cast<const T*>(a.grad_out),
      static_cast<const T*>(a.x), a.weight, a.bias, mean, rstd, partial_c, partial_g, plan.sums, a.C,
      a.G, plan.param_levels, a.wide ? 1 : 0);
  ColumnRuns runs{};
  runs.outer = a.N;
  runs.pitch = plan.sums.chunks;
  if (plan.param_levels == 1) {
    runs.end[0] = plan.sums.chunks;
  } else {
    for (int l = 0; l < plan.sums.levels; ++l) {
      runs.begin[l] = plan.sums.chunk_start[l];
      runs.end[l] = plan.sums.chunk_start[l + 1];
    }
  }
  const int groups = a.grad_x != nullptr ? a.N * plan.sums.levels * ((a.G + 31) / 32) : 0;
  const int columns = partial_c != nullptr ? (a.C + 15) / 16 * 2 * plan.param_levels : 0;
  if (groups + columns > 0)
    run((gn_bwd_join_kernel<T>), dim3(groups + columns), dim3(1024), 0, a.stream,
        static_cast<const ct*>(partial_g), static_cast<const ct*>(partial_c), m1, m2, a.grad_weight,
        a.grad_bias, plan.sums, runs, groups, a.C, a.G, a.wide ? 1 : 0);
  if (a.grad_x != nullptr)
    run((gn_bwd_apply_kernel<T, ACT, MODE>), dim3(a.N * plan.writes.chunks, plan.tiles),
        dim3(kGnThreads), 0, a.stream, static_cast<const T*>(a.grad_out), static_cast<const T*>(a.x),
        a.weight, a.bias, mean, rstd, static_cast<const ct*>(m1), static_cast<const ct*>(m2),
        static_cast<T*>(a.grad_x), plan.writes, a.C, a.G, plan.param_levels, a.wide ? 1 : 0);
  return run.rc;
}

// A slab of whole groups for the one-launch kernels, and the threads of its workgroup; false where a
// level does not fit `hold` vectors a thread or the call is too large for slabs of 64 bytes a row (they
// use half of each cache line).  One launch against three (MI355X, 256 bf16 channels, us): forward 512
// rows 6.9 against 11.2, 64 x 256 rows 8.0 / 13.9, 8 x 1024 rows (four vectors a thread) 8.7 / 11.7;
// gradient 512 rows 10.3 / 12.6, 64 x 256 rows 16.0 / 17.9.  The gradient with four vectors a thread
// loses (8 x 1024 rows 16.9 / 14.3), so does a slab of 32 bytes (17.5 for the latter), and so do
// 128 x 1024 rows of 512 channels (118 + 184 / 74 + 130).
constexpr int64_t kGnSmallBytes = 16 << 20;
inline bool gn_small_plan(const GnPlan& plan, int N, int C, int G, size_t esize, int hold,
                          GnSlab* sl, int* threads) {
  const int VE = 16 / static_cast<int>(esize), cpg = C / G, S = plan.sums.row_start[plan.sums.levels];
  if (static_cast<int64_t>(N) * S * C * static_cast<int64_t>(esize) > kGnSmallBytes) return false;
  int longest = 0;
  for (int l = 0; l < plan.sums.levels; ++l) {
    const int rows = plan.sums.row_start[l + 1] - plan.sums.row_start[l];
    longest = rows > longest ? rows : longest;
  }
  int best = 0;
  for (int k = 1; k <= G && static_cast<int64_t>(k) * cpg <= kGnSlabChannels && best == 0; ++k) {
    const int vecs = k * cpg / VE;
    if (G % k == 0 && k * cpg % VE == 0 && (vecs >= 4 || k == G)) best = k;
  }
  if (best == 0 || longest > 1024 / (best * cpg / VE) * hold ||
      static_cast<int64_t>(N) * plan.sums.levels * (G / best) > (1 << 21))
    return false;
  *sl = {best, best * cpg, best * cpg / VE, G / best};
  *threads = 1024;
  for (int t = 256; t < 1024; t *= 2)
    if (longest <= t / sl->vecs * 2) {  // (two vectors a thread: more rows a thread were no faster)
      *threads = t;
      break;
    }
  return true;
}

template <typename T, int ACT>
int gn_small_forward(const GnCall& a, const GnPlan& plan, const GnSlab& sl, int threads) {
  Launches run;
  const size_t lds = (static_cast<size_t>(threads / sl.vecs) * (sl.channels + 1) + 2 * sl.groups) * 4;
  run((gn_small_kernel<T, ACT>), dim3(a.N * plan.sums.levels * sl.slabs), dim3(threads), lds, a.stream,
      static_cast<const T*>(a.x), a.weight, a.bias, static_cast<T*>(a.out), static_cast<float*>(a.mean),
      static_cast<float*>(a.rstd), plan.sums, sl, a.C, a.G, plan.param_levels, static_cast<float>(a.eps),
      a.wide ? 1 : 0);
  return run.rc;
}

template <typename T, int ACT>
int gn_small_backward(const GnCall& a, const GnPlan& plan, const GnSlab& sl, int threads) {
  Launches run;
  const bool params = a.grad_weight != nullptr;
  const bool direct = a.N == 1 && plan.param_levels == plan.sums.levels;
  float* partial = params && !direct ? static_cast<float*>(a.workspace) : nullptr;
  const size_t lds = (static_cast<size_t>(threads / sl.vecs) * (sl.channels + 1) + 2 * sl.channels +
                      2 * sl.groups) * 4;
  run((gn_small_bwd_kernel<T, ACT>), dim3(a.N * plan.sums.levels * sl.slabs), dim3(threads), lds, a.stream,
      static_cast<const T*>(a.grad_out), static_cast<const T*>(a.x), a.weight, a.bias,
      static_cast<const float*>(a.mean), static_cast<const float*>(a.rstd), static_cast<T*>(a.grad_x),
      partial, a.grad_weight, a.grad_bias, plan.sums, sl, a.C, a.G, plan.param_levels, a.wide ? 1 : 0);
  if (partial != nullptr) {
    // partial rows lie sample by sample, level by level
    ColumnRuns runs{};
    runs.outer = a.N;
    runs.pitch = plan.sums.levels;
    if (plan.param_levels == 1) {
      runs.end[0] = plan.sums.levels;
    } else {
      for (int l = 0; l < plan.sums.levels; ++l) {
        runs.begin[l] = l;
        runs.end[l] = l + 1;
      }
    }
    run((gn_bwd_join_kernel<T>), dim3((a.C + 15) / 16 * 2 * plan.param_levels), dim3(1024), 0, a.stream,
        static_cast<const float*>(nullptr), static_cast<const float*>(partial),
        static_cast<float*>(nullptr), static_cast<float*>(nullptr), a.grad_weight, a.grad_bias, plan.sums,
        runs, 0, a.C, a.G, a.wide ? 1 : 0);
  }
  return run.rc;
}

template <typename T, int ACT>
int gn_act_run(const GnCall& a, const GnPlan& plan, bool backward) {
  // (fp64 is for checking gradients: it takes the general kernels)
  if constexpr (sizeof(T) <= 4) {
    GnSlab sl;
    int threads;
    if (gn_small_plan(plan, a.N, a.C, a.G, sizeof(T), backward ? kGnHoldBwd : kGnHold, &sl,
                      &threads))
      return backward ? gn_small_backward<T, ACT>(a, plan, sl, threads)
                      : gn_small_forward<T, ACT>(a, plan, sl, threads);
  }
  switch (row_mode(a.C, 16 / static_cast<int>(sizeof(T)))) {
    case kRowEven:
      return backward ? gn_backward<T, ACT, kRowEven>(a, plan) : gn_forward<T, ACT, kRowEven>(a, plan);
    case kRowOdd:
      return backward ? gn_backward<T, ACT, kRowOdd>(a, plan) : gn_forward<T, ACT, kRowOdd>(a, plan);
    default:
      return backward ? gn_backward<T, ACT, kRowShort>(a, plan) : gn_forward<T, ACT, kRowShort>(a, plan);
  }
}

template <typename T>
int gn_run(const GnCall& a, const GnPlan& plan, int activation, bool backward) {
  switch (activation) {
    case kGnRelu: return gn_act_run<T, kGnRelu>(a, plan, backward);
    case kGnSilu: return gn_act_run<T, kGnSilu>(a, plan, backward);
    case kGnGelu: return gn_act_run<T, kGnGelu>(a, plan, backward);
    default: return gn_act_run<T, kGnNone>(a, plan, backward);
  }
}

inline int gn_dispatch(const GnCall& a, const GnPlan& plan, int activation, int dtype, bool backward) {
  switch (dtype) {
    case MSDA_F32: return gn_run<float>(a, plan, activation, backward);
    case MSDA_F64: return gn_run<double>(a, plan, activation, backward);
    case MSDA_BF16: return gn_run<bf16_t>(a, plan, activation, backward);
    default: return gn_run<f16_t>(a, plan, activation, backward);
  }
}

inline bool all_aligned(size_t a, std::initializer_list<const void*> ptrs) {
  for (const void* p : ptrs)
    if (p != nullptr && !aligned(p, a)) return false;
  return true;
}

}  // namespace msda

extern "C" {

int msda_dropout_forward(const void* x, void* out, const int64_t* rng_state, int64_t numel,
                         double p, int site, int activation, int dtype, void* hip_stream) {
  using namespace msda;
  DropArgs d;
  if (!x || !out) return MSDA_ENULL;
  if (numel < 1 || site < 0 || !drop_args(p, &d)) return MSDA_ESHAPE;
  const size_t e = elem_size(dtype);
  if (e == 0 || (activation != MSDA_ACT_NONE && activation != MSDA_ACT_RELU)) return MSDA_EDTYPE;
  if (d.threshold && !rng_state) return MSDA_ENULL;
  if (d.threshold && numel > kMaxDropElements) return MSDA_ESHAPE;
  if (!all_aligned(e, {x, out}) || !all_aligned(8, {rng_state})) return MSDA_EALIGN;
  const bool relu = activation == MSDA_ACT_RELU;
  const uint32_t s = static_cast<uint32_t>(site);
  hipStream_t stream = static_cast<hipStream_t>(hip_stream);
  switch (dtype) {
    case MSDA_F32: return dropout_forward<float>(x, out, rng_state, numel, d, s, relu, stream);
    case MSDA_F64: return dropout_forward<double>(x, out, rng_state, numel, d, s, relu, stream);
    case MSDA_BF16: return dropout_forward<bf16_t>(x, out, rng_state, numel, d, s, relu, stream);
    default: return dropout_forward<f16_t>(x, out, rng_state, numel, d, s, relu, stream);
  }
}

int msda_dropout_backward(const void* grad_out, const void* out, void* grad_x,
                          const int64_t* rng_state, int64_t numel, double p, int site,
                          int activation, int dtype, void* hip_stream) {
  using namespace msda;
  if (activation == MSDA_ACT_NONE)  // the same mask and scale on the gradient
    return msda_dropout_forward(grad_out, grad_x, rng_state, numel, p, site, activation, dtype,
                                hip_stream);
  DropArgs d;
  if (!grad_out || !out || !grad_x) return MSDA_ENULL;
  if (numel < 1 || site < 0 || !drop_args(p, &d)) return MSDA_ESHAPE;
  const size_t e = elem_size(dtype);
  if (e == 0 || activation != MSDA_ACT_RELU) return MSDA_EDTYPE;
  if (!all_aligned(e, {grad_out, out, grad_x})) return MSDA_EALIGN;
  hipStream_t stream = static_cast<hipStream_t>(hip_stream);
  switch (dtype) {
    case MSDA_F32: return dropout_relu_backward<float>(grad_out, out, grad_x, numel, d, stream);
    case MSDA_F64: return dropout_relu_backward<double>(grad_out, out, grad_x, numel, d, stream);
    case MSDA_BF16: return dropout_relu_backward<bf16_t>(grad_out, out, grad_x, numel, d, stream);
    default: return dropout_relu_backward<f16_t>(grad_out, out, grad_x, numel, d, stream);
  }
}

int msda_dropout_add_norm_forward(const void* x, const void* residual, const void* weight,
                                  const void* bias, void* out, void* mean, void* rstd,
                                  const int64_t* rng_state, int64_t rows, int C, double p, int site,
                                  double eps, int dtype_x, int dtype_residual, int dtype_param,
                                  void* hip_stream) {
  using namespace msda;
  AddNormCall a{};
  if (!x || !residual || !weight || !bias || !out || !mean != !rstd) return MSDA_ENULL;
  const int rc = add_norm_check(rows, C, p, site, dtype_x, dtype_residual, dtype_param, &a.drop);
  if (rc != MSDA_OK) return rc;
  if (!(eps >= 0.0)) return MSDA_ESHAPE;
  if (a.drop.threshold && !rng_state) return MSDA_ENULL;
  const size_t ce = dtype_residual == MSDA_F64 ? 8 : 4;
  if (!all_aligned(elem_size(dtype_x), {x}) || !all_aligned(elem_size(dtype_residual), {residual, out}) ||
      !all_aligned(elem_size(dtype_param), {weight, bias}) || !all_aligned(ce, {mean, rstd}) ||
      !all_aligned(8, {rng_state}))
    return MSDA_EALIGN;
  a.x = x;
  a.res = residual;
  a.weight = weight;
  a.bias = bias;
  a.out = out;
  a.mean = mean;
  a.rstd = rstd;
  a.rng_state = rng_state;
  a.rows = rows;
  a.C = C;
  a.dtype_res = dtype_residual;
  a.site = static_cast<uint32_t>(site);
  a.eps = eps;
  a.wide = dtype_param != MSDA_BF16 && dtype_param != MSDA_F16;
  a.stream = static_cast<hipStream_t>(hip_stream);
  return add_norm_dispatch(a, dtype_x, dtype_residual, false);
}

size_t msda_dropout_add_norm_workspace_bytes(int64_t rows, int C, int dtype_x, int dtype_residual) {
  using namespace msda;
  DropArgs d;
  if (add_norm_check(rows, C, 0.0, 0, dtype_x, dtype_residual, dtype_residual, &d) != MSDA_OK) return 0;
  const int64_t blocks = add_norm_bwd_grid(rows, C, dtype_residual).blocks;
  return static_cast<size_t>(blocks + (blocks > kColumnSplit ? kColumnSegments : 0)) * 2 * C *
         (dtype_residual == MSDA_F64 ? 8 : 4);
}

int msda_dropout_add_norm_backward(const void* grad_out, const void* x, const void* residual,
                                   const void* weight, const void* mean, const void* rstd,
                                   void* grad_x, void* grad_residual, void* grad_weight,
                                   void* grad_bias, void* workspace, size_t workspace_bytes,
                                   const int64_t* rng_state, int64_t rows, int C, double p,
                                   int site, int dtype_x, int dtype_residual, int dtype_param,
                                   void* hip_stream) {
  using namespace msda;
  AddNormCall a{};
  if (!grad_out || !x || !residual || !weight || !mean || !rstd || !grad_weight != !grad_bias)
    return MSDA_ENULL;
  const int rc = add_norm_check(rows, C, p, site, dtype_x, dtype_residual, dtype_param, &a.drop);
  if (rc != MSDA_OK) return rc;
  if (a.drop.threshold && !rng_state) return MSDA_ENULL;
  const size_t ce = dtype_residual == MSDA_F64 ? 8 : 4;
  if (!all_aligned(elem_size(dtype_x), {x, grad_x}) ||
      !all_aligned(elem_size(dtype_residual), {grad_out, residual, grad_residual}) ||
      !all_aligned(elem_size(dtype_param), {weight, grad_weight, grad_bias}) ||
      !all_aligned(ce, {mean, rstd}) || !all_aligned(8, {rng_state}))
    return MSDA_EALIGN;
  if (grad_weight != nullptr &&
      (!workspace || !aligned(workspace, 8) ||
       workspace_bytes < msda_dropout_add_norm_workspace_bytes(rows, C, dtype_x, dtype_residual)))
    return MSDA_EWORKSPACE;
  a.grad_out = grad_out;
  a.x = x;
  a.res = residual;
  a.weight = weight;
  a.mean = const_cast<void*>(mean);
  a.rstd = const_cast<void*>(rstd);
  a.grad_x = grad_x;
  a.grad_res = grad_residual;
  a.grad_weight = grad_weight;
  a.grad_bias = grad_bias;
  a.partial = grad_weight != nullptr ? workspace : nullptr;
  a.rng_state = rng_state;
  a.rows = rows;
  a.C = C;
  a.dtype_res = dtype_residual;
  a.site = static_cast<uint32_t>(site);
  a.wide = dtype_param != MSDA_BF16 && dtype_param != MSDA_F16;
  a.stream = static_cast<hipStream_t>(hip_stream);
  return add_norm_dispatch(a, dtype_x, dtype_residual, true);
}

size_t msda_group_norm_workspace_bytes(const int64_t* level_rows_host, int N, int S, int C, int G,
                                       int L, int dtype, int backward) {
  using namespace msda;
  GnPlan plan;
  if (level_rows_host == nullptr ||
      gn_plan(level_rows_host, N, S, C, G, L, 1, kGnNone, dtype, dtype, &plan) != MSDA_OK)
    return 0;
  return static_cast<size_t>(gn_workspace_values(plan, N, C, G, backward != 0)) * gn_compute_size(dtype);
}

int msda_group_norm_forward(const void* x, const void* weight, const void* bias, void* out,
                            void* mean, void* rstd, void* workspace, size_t workspace_bytes,
                            const int64_t* level_rows_host, int N, int S, int C, int G, int L,
                            int param_levels, double eps, int activation, int dtype,
                            int dtype_param, void* hip_stream) {
  using namespace msda;
  if (!x || !weight || !bias || !out || !level_rows_host || !mean != !rstd) return MSDA_ENULL;
  GnPlan plan;
  const int rc = gn_plan(level_rows_host, N, S, C, G, L, param_levels, activation, dtype,
                         dtype_param, &plan);
  if (rc != MSDA_OK) return rc;
  if (!(eps >= 0.0)) return MSDA_ESHAPE;
  if (!all_aligned(elem_size(dtype), {x, out}) ||
      !all_aligned(elem_size(dtype_param), {weight, bias}) ||
      !all_aligned(gn_compute_size(dtype), {mean, rstd}))
    return MSDA_EALIGN;
  if (!workspace || !aligned(workspace, 8) ||
      workspace_bytes < msda_group_norm_workspace_bytes(level_rows_host, N, S, C, G, L, dtype, 0))
    return MSDA_EWORKSPACE;
  GnCall a{};
  a.x = x;
  a.weight = weight;
  a.bias = bias;
  a.out = out;
  a.mean = mean;
  a.rstd = rstd;
  a.workspace = workspace;
  a.N = N;
  a.C = C;
  a.G = G;
  a.eps = eps;
  a.wide = dtype_param != MSDA_BF16 && dtype_param != MSDA_F16;
  a.stream = static_cast<hipStream_t>(hip_stream);
  return gn_dispatch(a, plan, activation, dtype, false);
}

int msda_group_norm_backward(const void* grad_out, const void* x, const void* weight,
                             const void* bias, const void* mean, const void* rstd, void* grad_x,
                             void* grad_weight, void* grad_bias, void* workspace,
                             size_t workspace_bytes, const int64_t* level_rows_host, int N, int S,
                             int C, int G, int L, int param_levels, int activation, int dtype,
                             int dtype_param, void* hip_stream) {
  using namespace msda;
  if (!grad_out || !x || !weight || !bias || !mean || !rstd || !level_rows_host ||
      !grad_weight != !grad_bias)
    return MSDA_ENULL;
  GnPlan plan;
  const int rc = gn_plan(level_rows_host, N, S, C, G, L, param_levels, activation, dtype,
                         dtype_param, &plan);
  if (rc != MSDA_OK) return rc;
  if (!all_aligned(elem_size(dtype), {grad_out, x, grad_x}) ||
      !all_aligned(elem_size(dtype_param), {weight, bias, grad_weight, grad_bias}) ||
      !all_aligned(gn_compute_size(dtype), {mean, rstd}))
    return MSDA_EALIGN;
  if (!workspace || !aligned(workspace, 8) ||
      workspace_bytes < msda_group_norm_workspace_bytes(level_rows_host, N, S, C, G, L, dtype, 1))
    return MSDA_EWORKSPACE;
  GnCall a{};
  a.grad_out = grad_out;
  a.x = x;
  a.weight = weight;
  a.bias = bias;
  a.mean = const_cast<void*>(mean);
  a.rstd = const_cast<void*>(rstd);
  a.grad_x = grad_x;
  a.grad_weight = grad_weight;
  a.grad_bias = grad_bias;
  a.workspace = workspace;
  a.N = N;
  a.C = C;
  a.G = G;
  a.wide = dtype_param != MSDA_BF16 && dtype_param != MSDA_F16;
  a.stream = static_cast<hipStream_t>(hip_stream);
  return gn_dispatch(a, plan, activation, dtype, true);
}

}  // extern "C"
