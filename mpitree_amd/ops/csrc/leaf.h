// Shared pieces of the operators over a tree's leaves (leaf_route.hip, leaf_embed.hip,
// leaf_linear.hip): element types, the grid of many small blocks and the route's search.
#pragma once
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include <string.h>

#include <algorithm>

#include "common.h"

namespace mt {

// element types as the bindings number them
enum LeafType { kLeafF32 = 0, kLeafF16 = 1, kLeafBF16 = 2 };

// A launch of `total` blocks of up to 1024 threads: a grid's x has to stay below 2^32 threads, so
// more blocks go to y; kernels number them with leaf_block() and leave past `total`.
inline dim3 leaf_grid(int64_t total) {
  constexpr int64_t kX = 1 << 21;
  if (total <= kX) return dim3((unsigned)total);
  const int64_t y = (total + kX - 1) / kX;
  if (y > 65535) throw std::runtime_error("leaf operator: too many blocks for one launch");
  return dim3((unsigned)kX, (unsigned)y);
}
__device__ __forceinline__ int64_t leaf_block() {
  return (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
}

// conversions to and from 32 bits; narrowing rounds to nearest even
struct f16_t {
  uint16_t u;
};
struct bf16_t {
  uint16_t u;
};
__device__ __forceinline__ float leaf_f32(float v) { return v; }
__device__ __forceinline__ float leaf_f32(f16_t v) {
  return (float)__builtin_bit_cast(_Float16, v.u);
}
__device__ __forceinline__ float leaf_f32(bf16_t v) {
  return __uint_as_float((uint32_t)v.u << 16);
}
template <typename T>
__device__ __forceinline__ T leaf_from(float v);
template <>
__device__ __forceinline__ float leaf_from<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ f16_t leaf_from<f16_t>(float v) {
  return f16_t{__builtin_bit_cast(uint16_t, (_Float16)v)};
}
template <>
__device__ __forceinline__ bf16_t leaf_from<bf16_t>(float v) {
  return bf16_t{__builtin_bit_cast(uint16_t, (__bf16)v)};
}

// W elements moved at once
template <typename T, int W>
struct alignas(sizeof(T) * W) LeafVec {
  T v[W];
};

// The route numbers tiles of `BM` rows without a scan: group g's tiles take the numbers from
// s(g) = off[g] / BM + g on. s grows by at least ceil(rows(g) / BM) from g to g + 1, so no number
// has two owners; some have none. This finds the last g in [0, G) with s(g) <= t: 64 probes a
// round, one per lane, so G <= 64 takes one load and 2^18 groups three. Every lane of the wave
// has to take part.
__device__ __forceinline__ int leaf_find_group(const int32_t* __restrict__ off, int G, int bm_shift,
                                               int64_t t) {
  const int lane = lane_id();
  int lo = 0, hi = G;
  while (hi - lo > 1) {
    const int step = (hi - lo + kWave - 1) / kWave;
    const int64_t g = (int64_t)lo + (int64_t)step * lane;
    const bool le = g < hi && ((int64_t)(off[g] >> bm_shift) + g) <= t;
    const int c = __popcll(__ballot(le));  // lane 0 always holds: s(0) = 0, s(lo) <= t
    lo += step * (c - 1);
    hi = min(hi, lo + step);
  }
  return lo;
}

}  // namespace mt
