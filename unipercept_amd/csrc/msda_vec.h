// 16-byte vector accesses at any element alignment, team sums and parameter loads shared by the
// kernels around the attention (dropout, residual + layer norm, group norm).
#pragma once

#include "msda_common.h"

namespace msda {

// Raw words of a vector access.  The types only promise the element's alignment: rows of odd
// widths start anywhere.  The hardware takes one 16-byte access at any byte address (unaligned
// access mode of the HSA ABI), so aligned and odd rows run the same instruction.
template <int BYTES, int ALIGN>
struct RawWords;
#define MSDA_RAW_WORDS(BYTES, COUNT, ALIGN)                                              \
  template <>                                                                            \
  struct RawWords<BYTES, ALIGN> {                                                        \
    typedef uint32_t type __attribute__((ext_vector_type(COUNT), aligned(ALIGN), may_alias)); \
  };
MSDA_RAW_WORDS(16, 4, 2)
MSDA_RAW_WORDS(16, 4, 4)
MSDA_RAW_WORDS(16, 4, 8)
MSDA_RAW_WORDS(8, 2, 2)
#undef MSDA_RAW_WORDS

// VE consecutive elements as they lie in memory.  STREAM: with the streaming (nontemporal) hint, for
// tensors that are read or written once in whole cache lines: a copy of 352 MB goes from 6.1 to
// 6.7 TB/s with it (MI355X, one vector a thread).  Where neighbouring accesses share a line the hint
// costs the line a second transfer (odd rows: 37 -> 48 us), so those go without.
template <typename T, int VE>
struct Pack {
  static constexpr int kBytes = VE * static_cast<int>(sizeof(T));
  using raw_t = typename RawWords<kBytes, static_cast<int>(sizeof(T))>::type;
  using ct = typename Elem<T>::compute_t;
  uint32_t w[kBytes / 4];

  template <bool STREAM>
  __device__ __forceinline__ void load(const T* p) {
    const raw_t* q = reinterpret_cast<const raw_t*>(p);
    raw_t r;
    if constexpr (STREAM) {
      r = __builtin_nontemporal_load(q);
    } else {
      r = *q;
    }
#pragma unroll
    for (int i = 0; i < kBytes / 4; ++i) w[i] = r[i];
  }
  // the first `count` elements only; the others read as zero
  __device__ __forceinline__ void load_part(const T* p, int count) {
    T tmp[VE] = {};
#pragma unroll
    for (int i = 0; i < VE; ++i)
      if (i < count) tmp[i] = p[i];
    __builtin_memcpy(w, tmp, kBytes);
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < kBytes / 4; ++i) w[i] = 0;
  }
  template <bool STREAM>
  __device__ __forceinline__ void store(T* p) const {
    raw_t r;
#pragma unroll
    for (int i = 0; i < kBytes / 4; ++i) r[i] = w[i];
    raw_t* q = reinterpret_cast<raw_t*>(p);
    if constexpr (STREAM) {
      __builtin_nontemporal_store(r, q);
    } else {
      *q = r;
    }
  }
  __device__ __forceinline__ void store_part(T* p, int count) const {
    T tmp[VE];
    __builtin_memcpy(tmp, w, kBytes);
#pragma unroll
    for (int i = 0; i < VE; ++i)
      if (i < count) p[i] = tmp[i];
  }
  __device__ __forceinline__ void unpack(ct* v) const {
    T tmp[VE];
    __builtin_memcpy(tmp, w, kBytes);
#pragma unroll
    for (int i = 0; i < VE; ++i) v[i] = Elem<T>::load(&tmp[i]);
  }
  __device__ __forceinline__ void pack(const ct* v) {
    T tmp[VE];
#pragma unroll
    for (int i = 0; i < VE; ++i) Elem<T>::store(&tmp[i], v[i]);
    __builtin_memcpy(w, tmp, kBytes);
  }
};

// How a row of C columns lies in vectors of VE columns.
enum RowMode {
  kRowEven = 0,   // C is a multiple of VE
  kRowOdd = 1,    // it is not, C > VE
  kRowShort = 2,  // C < VE: one vector, partly filled
};

inline int row_mode(int C, int VE) { return C % VE == 0 ? kRowEven : C < VE ? kRowShort : kRowOdd; }

// Columns of one vector of a row.  Vector k starts at column k * VE; the last one of an odd row is
// moved back to end with the row: its first `skip` columns belong to its neighbour too and stay out
// of the sums (both write the same bits).  So odd rows move in whole vectors like even ones; only
// short rows go element by element.  (Partial vectors for the ends of odd rows cost 204 registers
// instead of 50 and three times the time: rows of 515 fp16 columns 45 us, 512 columns 15 us.)
template <int VE, int MODE>
struct Span {
  int c, skip, count;

  __device__ __forceinline__ static Span at(int k, int C) {
    const int first = k * VE;
    if constexpr (MODE == kRowEven) return {first, 0, first < C ? VE : 0};
    if constexpr (MODE == kRowShort) return {0, 0, k == 0 ? C : 0};
    const int c = min(first, C - VE);
    return {c, first - c, first < C ? VE : 0};
  }
  __device__ __forceinline__ bool active() const { return count > 0; }
  // element i belongs to this vector's share of the sums
  __device__ __forceinline__ bool owns(int i) const {
    if constexpr (MODE == kRowEven) return count > 0;
    if constexpr (MODE == kRowShort) return i < count;
    return count > 0 && i >= skip;
  }

  template <typename T>
  __device__ __forceinline__ void load(Pack<T, VE>& p, const T* row) const {
    if constexpr (MODE == kRowShort) {
      p.load_part(row, count);
    } else if (count > 0) {
      p.template load<MODE == kRowEven>(row + c);
    } else {
      p.zero();
    }
  }
  template <typename T>
  __device__ __forceinline__ void store(const Pack<T, VE>& p, T* row) const {
    if constexpr (MODE == kRowShort) {
      p.store_part(row, count);
    } else if (count > 0) {
      p.template store<MODE == kRowEven>(row + c);
    }
  }
};

// Parameters (weight, bias) come in the activations' type or, next to 16-bit activations, in fp32.
template <typename T>
__device__ __forceinline__ typename Elem<T>::compute_t load_param(const void* p, int64_t i, bool wide) {
  using ct = typename Elem<T>::compute_t;
  return wide ? static_cast<const ct*>(p)[i] : Elem<T>::load(static_cast<const T*>(p) + i);
}
template <typename T>
__device__ __forceinline__ void store_param(void* p, int64_t i, typename Elem<T>::compute_t v, bool wide) {
  using ct = typename Elem<T>::compute_t;
  if (wide) {
    static_cast<ct*>(p)[i] = v;
  } else {
    Elem<T>::store(static_cast<T*>(p) + i, v);
  }
}

// VE parameters of a vector; columns outside the row read as zero
template <typename T, int VE, int MODE>
__device__ __forceinline__ void load_params(const void* p, int64_t row, const Span<VE, MODE>& s, bool wide,
                                            typename Elem<T>::compute_t* v) {
  using ct = typename Elem<T>::compute_t;
  if constexpr (MODE == kRowShort) {
#pragma unroll
    for (int i = 0; i < VE; ++i) v[i] = i < s.count ? load_param<T>(p, row + i, wide) : ct(0);
  } else if (!s.active()) {
#pragma unroll
    for (int i = 0; i < VE; ++i) v[i] = ct(0);
  } else if (wide) {
    constexpr int WE = 16 / sizeof(ct);
#pragma unroll
    for (int i = 0; i < VE; i += WE) {
      Pack<ct, WE> q;
      q.template load<false>(static_cast<const ct*>(p) + row + s.c + i);
      q.unpack(v + i);
    }
  } else {
    Pack<T, VE> q;
    q.template load<false>(static_cast<const T*>(p) + row + s.c);
    q.unpack(v);
  }
}

// Sum over the TS lanes of a team (TS a power of two up to the wave), the same bits in every lane.
// In fp32 by data-parallel moves inside rows of 16 lanes and by the row exchanges of gfx950 between
// them: no trip through LDS.
template <int TS>
__device__ __forceinline__ float wave_team_sum(float v) {
#define MSDA_DPP_ADD(CTRL)                                                                     \
  v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(                                  \
                                     0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true))
  if constexpr (TS >= 2) MSDA_DPP_ADD(0xB1);    // quad_perm [1, 0, 3, 2]
  if constexpr (TS >= 4) MSDA_DPP_ADD(0x4E);    // quad_perm [2, 3, 0, 1]
  if constexpr (TS >= 8) MSDA_DPP_ADD(0x141);   // row_half_mirror: the other four of eight
  if constexpr (TS >= 16) MSDA_DPP_ADD(0x140);  // row_mirror: the other eight of sixteen
#undef MSDA_DPP_ADD
  if constexpr (TS >= 32) {
    const uint32_t bits = __builtin_bit_cast(uint32_t, v);
    const auto r = __builtin_amdgcn_permlane16_swap(bits, bits, false, false);
    const uint32_t low = r[0], high = r[1];  // (scalars: a bit cast of r[1] itself reads r[0])
    v = __builtin_bit_cast(float, low) + __builtin_bit_cast(float, high);
  }
  if constexpr (TS >= 64) {
    const uint32_t bits = __builtin_bit_cast(uint32_t, v);
    const auto r = __builtin_amdgcn_permlane32_swap(bits, bits, false, false);
    const uint32_t low = r[0], high = r[1];  // (scalars: a bit cast of r[1] itself reads r[0])
    v = __builtin_bit_cast(float, low) + __builtin_bit_cast(float, high);
  }
  return v;
}
template <int TS>
__device__ __forceinline__ double wave_team_sum(double v) {
#pragma unroll
  for (int off = TS / 2; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}

// ---- column sums -------------------------------------------------------------------------------
// Second stage of a sum over rows whose first stage left one row of partial sums per workgroup:
// dst_k[level * C + c] = sum over the level's partial rows r of src[(r * 2 + k) * C + c], k = 0, 1.
// The partial rows of a level are `outer` runs of rows [begin, end) at a distance of `pitch` rows.
// The order of the additions is fixed by the sizes.
constexpr int kMaxNormLevels = 16;
struct ColumnRuns {
  int outer, pitch;
  int begin[kMaxNormLevels], end[kMaxNormLevels];
};

// One tile of 16 columns by a workgroup of 1024 threads: 16 bytes a thread and row, so that all
// partial rows are on their way in a few steps.
template <typename T>
__device__ __forceinline__ void column_sums(const typename Elem<T>::compute_t* __restrict__ src,
                                            void* __restrict__ dst0, void* __restrict__ dst1,
                                            const ColumnRuns& runs, int C, bool wide, int tile, int k,
                                            int level) {
  using ct = typename Elem<T>::compute_t;
  constexpr int VE = 16 / sizeof(ct), ACROSS = 16 / VE, LANES = 1024 / ACROSS;
  __shared__ ct part[LANES][17];
  const int at = (threadIdx.x % ACROSS) * VE, lane = threadIdx.x / ACROSS;
  const int c = tile * 16 + at, count = min(VE, C - c);
  const int inner = runs.end[level] - runs.begin[level], total = runs.outer * inner;
  ct sum[VE];
#pragma unroll
  for (int i = 0; i < VE; ++i) sum[i] = 0;
  if (count > 0) {
#pragma unroll 8
    for (int i = lane; i < total; i += LANES) {
      const int o = i / inner;
      const int64_t r = static_cast<int64_t>(o) * runs.pitch + runs.begin[level] + (i - o * inner);
      const ct* row = src + (r * 2 + k) * C + c;
      Pack<ct, VE> p;
      if (count == VE) {
        p.template load<false>(row);
      } else {
        p.load_part(row, count);
      }
      ct v[VE];
      p.unpack(v);
#pragma unroll
      for (int e = 0; e < VE; ++e) sum[e] += v[e];
    }
  }
#pragma unroll
  for (int i = 0; i < VE; ++i) part[lane][at + i] = sum[i];
  __syncthreads();
  // 16 columns x 64 groups of LANES / 64 lanes, then the groups
  const int col = threadIdx.x & 15, group = threadIdx.x >> 4;
  ct acc = 0;
#pragma unroll
  for (int i = 0; i < LANES / 64; ++i) acc += part[group + 64 * i][col];
  __syncthreads();
  part[group][col] = acc;
  __syncthreads();
  if (threadIdx.x < 16 && tile * 16 + col < C) {
    ct four[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 64; ++i) four[i & 3] += part[i][col];
    store_param<T>(k == 0 ? dst0 : dst1, static_cast<int64_t>(level) * C + tile * 16 + col,
                   (four[0] + four[1]) + (four[2] + four[3]), wide);
  }
}

// The sums of `total` partial rows.  blockIdx.z: one of gridDim.z segments of the rows; with more than
// one, every segment leaves a partial row of its own in `next` (for a second call), else the results
// go to dst0 and dst1.
template <typename T>
__global__ __launch_bounds__(1024) void column_sums_kernel(
    const typename Elem<T>::compute_t* __restrict__ src,
    typename Elem<T>::compute_t* __restrict__ next, void* __restrict__ dst0, void* __restrict__ dst1,
    int total, int C, int wide) {
  using ct = typename Elem<T>::compute_t;
  ColumnRuns runs;
  runs.outer = 1;
  runs.pitch = 0;
  const int share = (total + gridDim.z - 1) / gridDim.z;
  runs.begin[0] = min(static_cast<int>(blockIdx.z) * share, total);
  runs.end[0] = min(runs.begin[0] + share, total);
  if (gridDim.z > 1) {
    ct* row = next + static_cast<int64_t>(blockIdx.z) * 2 * C;
    column_sums<T>(src, row, row + C, runs, C, true, blockIdx.x, blockIdx.y, 0);
  } else {
    column_sums<T>(src, dst0, dst1, runs, C, wide != 0, blockIdx.x, blockIdx.y, 0);
  }
}

}  // namespace msda
