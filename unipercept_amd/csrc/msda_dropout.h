// Dropout from a counter-based generator (gfx950): the mask is a function of (seed, offset, site,
// element index) and is computed where it is needed, never stored.
//
//   u(i)  16 random bits of element i (flat index in the contiguous order of the tensor):
//         Philox4x32 with 7 rounds (J. K. Salmon, M. A. Moraes, R. O. Dror, D. E. Shaw, "Parallel
//         random numbers: as easy as 1, 2, 3", SC 2011; 7 rounds is the fewest that their tests
//         accept), counter (i / 8, site, offset low, offset high), key (seed low, seed high);
//         element 8 j + e takes the low (even e) or high half of word e / 2.
//   keep  u(i) >= t with t = round(p * 65536); kept elements are scaled by 65536 / (65536 - t).
//
// Sixteen bits an element: one generator call serves 8 elements.  A whole word an element would
// double the arithmetic, which is what bounds the 16-bit cases next; p moves by at most 2^-17, and
// the scale belongs to the p that is used, so expectations stay exact.
#pragma once

#include "msda_vec.h"

namespace msda {

struct DropKey {
  uint32_t k0, k1, o0, o1;
};

__device__ __forceinline__ DropKey load_drop_key(const int64_t* __restrict__ rng_state) {
  const uint64_t seed = static_cast<uint64_t>(rng_state[0]);
  const uint64_t offset = static_cast<uint64_t>(rng_state[1]);
  return {static_cast<uint32_t>(seed), static_cast<uint32_t>(seed >> 32),
          static_cast<uint32_t>(offset), static_cast<uint32_t>(offset >> 32)};
}

__device__ __forceinline__ uint4 drop_words(const DropKey& key, uint32_t block, uint32_t site) {
  uint32_t c0 = block, c1 = site, c2 = key.o0, c3 = key.o1, k0 = key.k0, k1 = key.k1;
#pragma unroll
  for (int r = 0; r < 7; ++r) {
    const uint64_t p0 = static_cast<uint64_t>(c0) * 0xD2511F53u;
    const uint64_t p1 = static_cast<uint64_t>(c2) * 0xCD9E8D57u;
    c0 = static_cast<uint32_t>(p1 >> 32) ^ c1 ^ k0;
    c1 = static_cast<uint32_t>(p1);
    c2 = static_cast<uint32_t>(p0 >> 32) ^ c3 ^ k1;
    c3 = static_cast<uint32_t>(p0);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return {c0, c1, c2, c3};
}

// keep bits of two elements of one generator word
__device__ __forceinline__ uint32_t keep_pair(uint32_t word, uint32_t threshold) {
  return ((word & 0xFFFFu) >= threshold ? 1u : 0u) | ((word >> 16) >= threshold ? 2u : 0u);
}
__device__ __forceinline__ uint32_t keep_block(const DropKey& key, uint32_t block, uint32_t site,
                                               uint32_t threshold) {
  const uint4 w = drop_words(key, block, site);
  return keep_pair(w.x, threshold) | keep_pair(w.y, threshold) << 2 |
         keep_pair(w.z, threshold) << 4 | keep_pair(w.w, threshold) << 6;
}

// Keep bits of elements [first, first + VE), VE <= 8.  ALIGNED: first is a multiple of VE, so that
// the vector lies in one generator block.
template <int VE, bool ALIGNED>
__device__ __forceinline__ uint32_t keep_bits(const DropKey& key, uint64_t first, uint32_t site,
                                              uint32_t threshold) {
  const uint32_t block = static_cast<uint32_t>(first >> 3), at = static_cast<uint32_t>(first & 7);
  uint32_t bits = keep_block(key, block, site, threshold);
  if constexpr (!ALIGNED) {
    if (at + VE > 8) bits |= keep_block(key, block + 1, site, threshold) << 8;
  }
  return VE == 8 && ALIGNED ? bits : bits >> at;
}

// One vector of 16 bytes per thread and step: with fp32 two lanes share a generator block and both
// compute it, which leaves the arithmetic per byte that of the 16-bit types (two vectors a lane
// instead leave every access half a line: 54 MB in 44 us against 20).  RELU: y = max(x, 0) first
// (NaN stays); a dropped element is 0 whatever x holds.
// Bound by HBM: 344064 x 1024 bf16 with ReLU and dropout, 1.41 GB in 234 us, 6.0 TB/s; the generator
// fills 0.6 of the VALU's time beside it (86 M wave instructions).
template <typename T, bool RELU, bool DROP>
__global__ __launch_bounds__(256) void dropout_kernel(const T* __restrict__ x, T* __restrict__ out,
                                                      const int64_t* __restrict__ rng_state,
                                                      int64_t numel, uint32_t threshold,
                                                      typename Elem<T>::compute_t scale,
                                                      uint32_t site) {
  using ct = typename Elem<T>::compute_t;
  constexpr int VE = 16 / sizeof(T);
  const DropKey key = DROP ? load_drop_key(rng_state) : DropKey{};
  const int64_t vecs = (numel + VE - 1) / VE;
  for (int64_t b = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; b < vecs;
       b += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t first = b * VE, left = numel - first;
    Pack<T, VE> p;
    if (left >= VE) {
      p.template load<true>(x + first);
    } else {
      p.load_part(x + first, static_cast<int>(left));
    }
    const uint32_t keep = DROP ? keep_bits<VE, true>(key, first, site, threshold) : 0xFFu;
    ct v[VE];
    p.unpack(v);
#pragma unroll
    for (int i = 0; i < VE; ++i) {
      bool on = (keep >> i) & 1u;
      if (RELU) on = on && !(v[i] <= ct(0));
      v[i] = on ? v[i] * scale : ct(0);
    }
    p.pack(v);
    if (left >= VE) {
      p.template store<true>(out + first);
    } else {
      p.store_part(out + first, static_cast<int>(left));
    }
  }
}

// Gradient of ReLU + dropout from the stored output: y is 0 exactly where the element was dropped
// or the ReLU closed (x * scale cannot underflow, scale >= 1), so the mask needs no generator.
// Bound by HBM: the same tensors, 2.11 GB in 323 us, 6.5 TB/s.
template <typename T>
__global__ __launch_bounds__(256) void dropout_relu_bwd_kernel(
    const T* __restrict__ grad_out, const T* __restrict__ y, T* __restrict__ grad_x, int64_t numel,
    typename Elem<T>::compute_t scale) {
  using ct = typename Elem<T>::compute_t;
  constexpr int VE = 16 / sizeof(T);
  const int64_t vecs = (numel + VE - 1) / VE;
  for (int64_t b = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; b < vecs;
       b += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t first = b * VE, left = numel - first;
    Pack<T, VE> g, o;
    if (left >= VE) {
      g.template load<true>(grad_out + first);
      o.template load<true>(y + first);
    } else {
      g.load_part(grad_out + first, static_cast<int>(left));
      o.load_part(y + first, static_cast<int>(left));
    }
    ct gv[VE], ov[VE];
    g.unpack(gv);
    o.unpack(ov);
#pragma unroll
    for (int i = 0; i < VE; ++i) gv[i] = ov[i] <= ct(0) ? ct(0) : gv[i] * scale;
    g.pack(gv);
    if (left >= VE) {
      g.template store<true>(grad_x + first);
    } else {
      g.store_part(grad_x + first, static_cast<int>(left));
    }
  }
}

}  // namespace msda
