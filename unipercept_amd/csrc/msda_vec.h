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

// VE consecutive elements as they lie in memory
template <typename T, int VE>
struct Pack {
  static constexpr int kBytes = VE * static_cast<int>(sizeof(T));
  using raw_t = typename RawWords<kBytes, static_cast<int>(sizeof(T))>::type;
  using ct = typename Elem<T>::compute_t;
  uint32_t w[kBytes / 4];

  __device__ __forceinline__ void load(const T* p) {
    const raw_t r = *reinterpret_cast<const raw_t*>(p);
#pragma unroll
    for (int i = 0; i < kBytes / 4; ++i) w[i] = r[i];
  }
  // the first `count` elements only (the end of a row); the others read as zero
  __device__ __forceinline__ void load_part(const T* p, int count) {
    T tmp[VE] = {};
#pragma unroll
    for (int i = 0; i < VE; ++i)
      if (i < count) tmp[i] = p[i];
    __builtin_memcpy(w, tmp, kBytes);
  }
  __device__ __forceinline__ void load(const T* p, int count) {
    if (count >= VE) {
      load(p);
    } else {
      load_part(p, count);
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < kBytes / 4; ++i) w[i] = 0;
  }
  __device__ __forceinline__ void store(T* p) const {
    raw_t r;
#pragma unroll
    for (int i = 0; i < kBytes / 4; ++i) r[i] = w[i];
    *reinterpret_cast<raw_t*>(p) = r;
  }
  __device__ __forceinline__ void store(T* p, int count) const {
    if (count >= VE) {
      store(p);
    } else {
      T tmp[VE];
      __builtin_memcpy(tmp, w, kBytes);
#pragma unroll
      for (int i = 0; i < VE; ++i)
        if (i < count) p[i] = tmp[i];
    }
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

// sum over the TS lanes of a team (TS a power of two up to the wave)
template <int TS, typename CT>
__device__ __forceinline__ CT wave_team_sum(CT v) {
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

template <typename T>
__global__ __launch_bounds__(1024) void column_sums_kernel(
    const typename Elem<T>::compute_t* __restrict__ src, void* __restrict__ dst0,
    void* __restrict__ dst1, ColumnRuns runs, int C, int wide) {
  using ct = typename Elem<T>::compute_t;
  __shared__ ct part[64][17];
  const int col = threadIdx.x & 15, lane = threadIdx.x >> 4;
  const int c = blockIdx.x * 16 + col, k = blockIdx.y, level = blockIdx.z;
  const int inner = runs.end[level] - runs.begin[level];
  const int64_t total = static_cast<int64_t>(runs.outer) * inner;
  ct sum = 0;
  if (c < C) {
#pragma unroll 4
    for (int64_t i = lane; i < total; i += 64) {
      const int64_t o = i / inner;
      const int64_t r = o * runs.pitch + runs.begin[level] + (i - o * inner);
      sum += src[(r * 2 + k) * C + c];
    }
  }
  part[lane][col] = sum;
  __syncthreads();
  if (threadIdx.x < 16 && c < C) {
    ct acc[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 64; ++i) acc[i & 3] += part[i][col];
    store_param<T>(k == 0 ? dst0 : dst1, static_cast<int64_t>(level) * C + c,
                   (acc[0] + acc[1]) + (acc[2] + acc[3]), wide != 0);
  }
}

}  // namespace msda
