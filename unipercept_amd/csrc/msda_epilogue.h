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

// Workgroups of a pass over `items` thread steps of 256: enough of them to fill the chip several
// times over (2048 hold 8 on every CU), each thread looping over what is left.
inline unsigned pass_grid(int64_t items) {
  const int64_t blocks = (items + 255) / 256;
  return static_cast<unsigned>(blocks < 4096 ? blocks : 4096);
}

template <typename T>
int dropout_forward(const void* x, void* out, const int64_t* rng_state, int64_t numel,
                    const DropArgs& d, uint32_t site, bool relu, hipStream_t stream) {
  using ct = typename Elem<T>::compute_t;
  Launches run;
  const dim3 grid(pass_grid((numel + 7) / 8));
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
  run((dropout_relu_bwd_kernel<T>), dim3(pass_grid((numel + VE - 1) / VE)), dim3(256), 0, stream,
      static_cast<const T*>(grad_out), static_cast<const T*>(out), static_cast<T*>(grad_x), numel,
      static_cast<typename Elem<T>::compute_t>(d.scale));
  return run.rc;
}

// ---- column sums --------------------------------------------------------------------------------
template <typename T>
void column_sums(Launches& run, const void* partial, void* dst0, void* dst1, const ColumnRuns& runs,
                 int levels, int C, bool wide, hipStream_t stream) {
  using ct = typename Elem<T>::compute_t;
  run((column_sums_kernel<T>), dim3((C + 15) / 16, 2, levels), dim3(1024), 0, stream,
      static_cast<const ct*>(partial), dst0, dst1, runs, C, wide ? 1 : 0);
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

// workgroups of the backward: each leaves one row of partial parameter gradients
inline int64_t add_norm_bwd_blocks(int64_t rows) { return rows < 1024 ? rows : 1024; }

struct AddNormCall {
  const void *grad_out, *x, *res, *weight, *bias;
  void *out, *mean, *rstd, *grad_x, *grad_res, *grad_weight, *grad_bias, *partial;
  const int64_t* rng_state;
  int64_t rows;
  int C;
  DropArgs drop;
  uint32_t site;
  double eps;
  bool wide;
  hipStream_t stream;
};

template <typename XT, typename RT, int TS, int NV, bool EVEN>
int add_norm_launch(const AddNormCall& a, bool backward) {
  using ct = typename Elem<RT>::compute_t;
  constexpr int TEAMS = 256 / TS;
  const int64_t need = (a.rows + TEAMS - 1) / TEAMS;
  Launches run;
  if (!backward) {
    run((add_norm_fwd_kernel<XT, RT, TS, NV, EVEN>),
        dim3(static_cast<unsigned>(need < 4096 ? need : 4096)), dim3(256), 0, a.stream,
        static_cast<const XT*>(a.x), static_cast<const RT*>(a.res), a.weight, a.bias,
        static_cast<RT*>(a.out), static_cast<ct*>(a.mean), static_cast<ct*>(a.rstd), a.rng_state,
        a.rows, a.C, a.drop.threshold, static_cast<ct>(a.drop.scale), a.site,
        static_cast<ct>(a.eps), a.wide ? 1 : 0);
    return run.rc;
  }
  const int64_t most = add_norm_bwd_blocks(a.rows);
  const int blocks = static_cast<int>(need < most ? need : most);
  run((add_norm_bwd_kernel<XT, RT, TS, NV, EVEN>), dim3(blocks), dim3(256), 0, a.stream,
      static_cast<const RT*>(a.grad_out), static_cast<const XT*>(a.x),
      static_cast<const RT*>(a.res), a.weight, static_cast<const ct*>(a.mean),
      static_cast<const ct*>(a.rstd), static_cast<XT*>(a.grad_x), static_cast<RT*>(a.grad_res),
      static_cast<ct*>(a.partial), a.rng_state, a.rows, a.C, a.drop.threshold,
      static_cast<ct>(a.drop.scale), a.site, a.wide ? 1 : 0);
  if (a.partial != nullptr) {
    ColumnRuns runs{};
    runs.outer = 1;
    runs.end[0] = blocks;
    column_sums<RT>(run, a.partial, a.grad_weight, a.grad_bias, runs, 1, a.C, a.wide, a.stream);
  }
  return run.rc;
}

// The narrowest team whose lanes cover a row: a wave or less per row needs no barrier; rows of up
// to four vectors a lane of one wave stay there, longer ones go to the whole workgroup.
template <typename XT, typename RT, bool EVEN>
int add_norm_width(const AddNormCall& a, bool backward) {
  const int vecs = (a.C + AddNormTypes<XT, RT>::VE - 1) / AddNormTypes<XT, RT>::VE;
  if (vecs <= 16) return add_norm_launch<XT, RT, 16, 1, EVEN>(a, backward);
  if (vecs <= 32) return add_norm_launch<XT, RT, 32, 1, EVEN>(a, backward);
  if (vecs <= 64) return add_norm_launch<XT, RT, 64, 1, EVEN>(a, backward);
  if (vecs <= 128) return add_norm_launch<XT, RT, 64, 2, EVEN>(a, backward);
  if (vecs <= 256) return add_norm_launch<XT, RT, 64, 4, EVEN>(a, backward);
  if (vecs <= 512) return add_norm_launch<XT, RT, 256, 2, EVEN>(a, backward);
  return add_norm_launch<XT, RT, 256, 4, EVEN>(a, backward);
}

template <typename XT, typename RT>
int add_norm_run(const AddNormCall& a, bool backward) {
  return a.C % AddNormTypes<XT, RT>::VE == 0 ? add_norm_width<XT, RT, true>(a, backward)
                                             : add_norm_width<XT, RT, false>(a, backward);
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
  GnLevels lv;
  int threads, lanes, team_width;
  int64_t blocks;
};

inline int gn_plan(const int64_t* level_rows, int N, int S, int C, int G, int L, int param_levels,
                   int activation, int dtype, int dtype_param, GnPlan* plan) {
  if (N < 1 || S < 1 || C < 1 || G < 1 || L < 1 || C % G != 0) return MSDA_ESHAPE;
  if (L > kMaxNormLevels) return MSDA_ELEVELS;
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
  const int tc = static_cast<int>((C * e + 15) / 16);
  plan->threads = tc <= 256 ? 256 : (tc + 63) / 64 * 64;
  plan->lanes = plan->threads / tc;
  // lanes that join the sums of one group
  int w = 1;
  while (w < 64 && w * 2 * G <= plan->threads) w *= 2;
  plan->team_width = w;
  // Rows of a chunk: about 2048 workgroups in the call (8 a CU), at most 128 chunks in a level
  // (every workgroup of the second launch reads all partial sums of its level), and at least four
  // rows a thread.
  auto up = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
  int64_t r = up(static_cast<int64_t>(N) * S, 2048);
  if (r < up(longest, 128)) r = up(longest, 128);
  r = up(r, 4 * plan->lanes) * 4 * plan->lanes;
  if (r > longest) r = longest;
  GnLevels& lv = plan->lv;
  lv.levels = L;
  lv.param_levels = param_levels;
  lv.rows_per_chunk = static_cast<int>(r);
  lv.row_start[0] = lv.chunk_start[0] = 0;
  for (int l = 0; l < L; ++l) {
    lv.row_start[l + 1] = lv.row_start[l] + static_cast<int>(level_rows[l]);
    lv.chunk_start[l + 1] = lv.chunk_start[l] + static_cast<int>(up(level_rows[l], r));
  }
  lv.chunks = lv.chunk_start[L];
  plan->blocks = static_cast<int64_t>(N) * lv.chunks;
  if (plan->blocks > INT32_MAX) return MSDA_ESHAPE;
  return MSDA_OK;
}

inline size_t gn_compute_size(int dtype) { return dtype == MSDA_F64 ? 8 : 4; }

struct GnCall {
  const void *grad_out, *x, *weight, *bias;
  void *out, *mean, *rstd, *grad_x, *grad_weight, *grad_bias, *workspace;
  int C, G;
  double eps;
  bool wide;
  hipStream_t stream;
};

template <typename T, int ACT>
int gn_forward(const GnCall& a, const GnPlan& plan) {
  using ct = typename Elem<T>::compute_t;
  const dim3 grid(static_cast<unsigned>(plan.blocks)), block(plan.threads);
  ct* partial = static_cast<ct*>(a.workspace);
  Launches run;
  run((gn_stats_kernel<T>), grid, block, 2 * sizeof(ct) * plan.lanes * a.C, a.stream,
      static_cast<const T*>(a.x), partial, plan.lv, a.C, a.G, plan.team_width);
  run((gn_apply_kernel<T, ACT>), grid, block, 2 * sizeof(ct) * a.G, a.stream,
      static_cast<const T*>(a.x), static_cast<const ct*>(partial), a.weight, a.bias,
      static_cast<T*>(a.out), static_cast<ct*>(a.mean), static_cast<ct*>(a.rstd), plan.lv, a.C, a.G,
      plan.team_width, static_cast<ct>(a.eps), a.wide ? 1 : 0);
  return run.rc;
}

template <typename T, int ACT>
int gn_backward(const GnCall& a, const GnPlan& plan) {
  using ct = typename Elem<T>::compute_t;
  const dim3 grid(static_cast<unsigned>(plan.blocks)), block(plan.threads);
  ct* partial_g = static_cast<ct*>(a.workspace);
  ct* partial_c = a.grad_weight != nullptr ? partial_g + plan.blocks * a.G * 2 : nullptr;
  Launches run;
  run((gn_bwd_stats_kernel<T, ACT>), grid, block, 2 * sizeof(ct) * plan.lanes * a.C, a.stream,
      static_cast<const T*>(a.grad_out), static_cast<const T*>(a.x), a.weight, a.bias,
      static_cast<const ct*>(a.mean), static_cast<const ct*>(a.rstd), partial_c, partial_g, plan.lv,
      a.C, a.G, plan.team_width, a.wide ? 1 : 0);
  if (partial_c != nullptr) {
    ColumnRuns runs{};
    runs.outer = static_cast<int>(plan.blocks / plan.lv.chunks);
    runs.pitch = plan.lv.chunks;
    if (plan.lv.param_levels == 1) {
      runs.end[0] = plan.lv.chunks;
    } else {
      for (int l = 0; l < plan.lv.levels; ++l) {
        runs.begin[l] = plan.lv.chunk_start[l];
        runs.end[l] = plan.lv.chunk_start[l + 1];
      }
    }
    column_sums<T>(run, partial_c, a.grad_weight, a.grad_bias, runs, plan.lv.param_levels, a.C,
                   a.wide, a.stream);
  }
  if (a.grad_x != nullptr)
    run((gn_bwd_apply_kernel<T, ACT>), grid, block, 2 * sizeof(ct) * a.G, a.stream,
        static_cast<const T*>(a.grad_out), static_cast<const T*>(a.x), a.weight, a.bias,
        static_cast<const ct*>(a.mean), static_cast<const ct*>(a.rstd),
        static_cast<const ct*>(partial_g), static_cast<T*>(a.grad_x), plan.lv, a.C, a.G,
        plan.team_width, a.wide ? 1 : 0);
  return run.rc;
}

template <typename T>
int gn_run(const GnCall& a, const GnPlan& plan, int activation, bool backward) {
  switch (activation) {
    case kGnRelu: return backward ? gn_backward<T, kGnRelu>(a, plan) : gn_forward<T, kGnRelu>(a, plan);
    case kGnSilu: return backward ? gn_backward<T, kGnSilu>(a, plan) : gn_forward<T, kGnSilu>(a, plan);
    case kGnGelu: return backward ? gn_backward<T, kGnGelu>(a, plan) : gn_forward<T, kGnGelu>(a, plan);
    default: return backward ? gn_backward<T, kGnNone>(a, plan) : gn_forward<T, kGnNone>(a, plan);
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
  return static_cast<size_t>(add_norm_bwd_blocks(rows)) * 2 * C * (dtype_residual == MSDA_F64 ? 8 : 4);
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
  return static_cast<size_t>(plan.blocks) * 2 * (G + (backward ? C : 0)) * gn_compute_size(dtype);
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
  a.C = C;
  a.G = G;
  a.wide = dtype_param != MSDA_BF16 && dtype_param != MSDA_F16;
  a.stream = static_cast<hipStream_t>(hip_stream);
  return gn_dispatch(a, plan, activation, dtype, true);
}

}  // extern "C"
