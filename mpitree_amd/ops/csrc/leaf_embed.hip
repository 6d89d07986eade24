// Embedding by leaf: y[i] = scale * table[leaf(i)], and its gradient summed by sorted leaves.
//
// Forward: a row without a leaf (its index outside [0, V)) gets zeros. Each row's vector is read
// and written once by a group of lanes, up to 16 bytes a lane.
//
// Gradient: dtable[v] = scale * sum of dy over the rows of leaf v, for every v (zeros where no row
// is). The rows are sorted by leaf first (leaf_route.hip), so a leaf's rows are a run of `order`,
// and every sum has one fixed order: the result does not depend on the launch. A leaf with at most
// kLeRun rows is summed by one group of lanes. A leaf with more is cut at the multiples of kLeRun
// of the sorted positions: each piece is summed by one workgroup into a partial row, and a second
// launch adds a leaf's partial rows. A chunk of kLeRun positions meets at most two such leaves
// (one that reaches into it, one that reaches out of it), so two partial rows a chunk suffice.
//
// Sums are held in 32 bits for 16-bit types and in 64 bits for f32: a leaf may hold most of a
// million rows, and a 64-bit add costs no more than a 32-bit one here, where memory is the bound.
#include "leaf.h"

namespace mt {

constexpr int kLeThreads = 256;
constexpr int kLeRun = 64;
constexpr int kLeUnroll = 4;

template <typename T>
struct LeAcc {
  using type = float;
};
template <>
struct LeAcc<float> {
  using type = double;
};

// Columns of a lane: NC vectors of W elements, a vector every `tpr` lanes of the column block.
struct LeCols {
  int tpr_shift;   // lanes of a row's group: 1 << tpr_shift, at most 64
  int col_blocks;  // column blocks of tpr * NC * W columns
};

template <typename T, int W, int NC, bool kScale, bool kWide>
__global__ __launch_bounds__(kLeThreads) void le_forward_kernel(
    const void* __restrict__ ids, const T* __restrict__ table, int64_t stride, int64_t n,
    int64_t V, int D, float scale, LeCols lc, T* __restrict__ y) {
  const int tpr = 1 << lc.tpr_shift, rpb = kLeThreads >> lc.tpr_shift;
  const int sub = threadIdx.x >> lc.tpr_shift, lr = threadIdx.x & (tpr - 1);
  const int64_t blk = leaf_block();
  const int64_t r0 = (blk / lc.col_blocks) * (rpb * kLeUnroll) + sub;
  const int c0 = ((int)(blk % lc.col_blocks) * NC * tpr + lr) * W;
  int64_t id[kLeUnroll];
#pragma unroll
  for (int u = 0; u < kLeUnroll; ++u) {
    const int64_t r = r0 + (int64_t)u * rpb;
    id[u] = -1;
    if (r < n) id[u] = kWide ? ((const int64_t*)ids)[r] : (int64_t)((const int32_t*)ids)[r];
  }
#pragma unroll
  for (int q = 0; q < NC; ++q) {
    const int c = c0 + q * tpr * W;
    if (c >= D) break;
    LeafVec<T, W> v[kLeUnroll];
#pragma unroll
    for (int u = 0; u < kLeUnroll; ++u) {
      v[u] = LeafVec<T, W>{};
      if ((uint64_t)id[u] < (uint64_t)V)
        v[u] = *(const LeafVec<T, W>*)(table + id[u] * stride + c);
    }
#pragma unroll
    for (int u = 0; u < kLeUnroll; ++u) {
      const int64_t r = r0 + (int64_t)u * rpb;
      if (r >= n) break;
      if constexpr (kScale) {
#pragma unroll
        for (int e = 0; e < W; ++e) v[u].v[e] = leaf_from<T>(leaf_f32(v[u].v[e]) * scale);
      }
      *(LeafVec<T, W>*)(y + r * D + c) = v[u];
    }
  }
}

// acc += dy[order[p]] for p = a, a + step, ... below b; the columns of one lane
template <typename T, int W, int NC, typename A>
__device__ __forceinline__ void le_sum_rows(const T* __restrict__ dy, int D, int c0, int tpr,
                                            const int32_t* __restrict__ order, int64_t a, int64_t b,
                                            int step, A (&acc)[NC][W]) {
  for (int64_t p = a; p < b; p += (int64_t)step * kLeUnroll) {
    int32_t row[kLeUnroll];
#pragma unroll
    for (int u = 0; u < kLeUnroll; ++u) {
      const int64_t pu = p + (int64_t)u * step;
      row[u] = pu < b ? order[pu] : -1;
    }
#pragma unroll
    for (int q = 0; q < NC; ++q) {
      const int c = c0 + q * tpr * W;
      if (c >= D) break;
      LeafVec<T, W> v[kLeUnroll];
#pragma unroll
      for (int u = 0; u < kLeUnroll; ++u) {
        v[u] = LeafVec<T, W>{};
        if (row[u] >= 0) v[u] = *(const LeafVec<T, W>*)(dy + (int64_t)row[u] * D + c);
      }
#pragma unroll
      for (int u = 0; u < kLeUnroll; ++u)
#pragma unroll
        for (int e = 0; e < W; ++e) acc[q][e] += (A)leaf_f32(v[u].v[e]);
    }
  }
}

// the sums of the block's row groups, added in their order; group 0's lanes hold the result
template <int W, int NC, typename A>
__device__ __forceinline__ void le_block_sum(A (&acc)[NC][W], int tpr_shift, A* s_acc) {
  const int tpr = 1 << tpr_shift, rpb = kLeThreads >> tpr_shift;
  const int sub = threadIdx.x >> tpr_shift, lr = threadIdx.x & (tpr - 1);
  // pairwise: groups [half, 2 half) hand theirs to groups [0, half)
  for (int half = rpb >> 1; half > 0; half >>= 1) {
    if (sub >= half && sub < 2 * half) {
#pragma unroll
      for (int q = 0; q < NC; ++q)
#pragma unroll
        for (int e = 0; e < W; ++e)
          s_acc[((q * W + e) * half + (sub - half)) * tpr + lr] = acc[q][e];
    }
    __syncthreads();
    if (sub < half) {
#pragma unroll
      for (int q = 0; q < NC; ++q)
#pragma unroll
        for (int e = 0; e < W; ++e) acc[q][e] += s_acc[((q * W + e) * half + sub) * tpr + lr];
    }
    __syncthreads();
  }
}

template <typename T, int W, int NC, typename A>
__device__ __forceinline__ void le_store(T* __restrict__ out, int D, int c0, int tpr, float scale,
                                         const A (&acc)[NC][W]) {
#pragma unroll
  for (int q = 0; q < NC; ++q) {
    const int c = c0 + q * tpr * W;
    if (c >= D) break;
    LeafVec<T, W> v;
#pragma unroll
    for (int e = 0; e < W; ++e) v.v[e] = leaf_from<T>((float)(acc[q][e] * (A)scale));
    *(LeafVec<T, W>*)(out + c) = v;
  }
}

// Blocks below `light`: the leaves with at most kLeRun rows. Blocks from there on: chunk pieces of
// the leaves with more, into `part` ([2 * chunks][D]).
template <typename T, int W, int NC>
__global__ __launch_bounds__(kLeThreads) void le_backward_kernel(
    const T* __restrict__ dy, const int32_t* __restrict__ order, const uint32_t* __restrict__ keys,
    const int32_t* __restrict__ off, int64_t V, int D, float scale, LeCols lc, int64_t light,
    T* __restrict__ dtable, typename LeAcc<T>::type* __restrict__ part) {
  using A = typename LeAcc<T>::type;
  __shared__ A s_acc[NC * W * kLeThreads / 2];
  const int tpr = 1 << lc.tpr_shift, rpb = kLeThreads >> lc.tpr_shift;
  const int sub = threadIdx.x >> lc.tpr_shift, lr = threadIdx.x & (tpr - 1);
  int64_t blk = leaf_block();
  const int c0 = ((int)(blk % lc.col_blocks) * NC * tpr + lr) * W;
  blk /= lc.col_blocks;
  if (blk < light) {
    const int64_t v = blk * rpb + sub;
    if (v >= V) return;
    const int64_t a = off[v], b = off[v + 1];
    if (b - a > kLeRun) return;
    A acc[NC][W] = {};
    le_sum_rows<T, W, NC, A>(dy, D, c0, tpr, order, a, b, 1, acc);
    le_store<T, W, NC, A>(dtable + v * D, D, c0, tpr, scale, acc);
    return;
  }
  const int64_t c = blk - light, m = off[V];
  const int64_t a = c * kLeRun, b = min<int64_t>(a + kLeRun, m);
  if (a >= m) return;
  const int64_t k0 = keys[a], k1 = keys[b - 1];
  const int64_t e0 = off[k0 + 1], s1 = off[k1];
#pragma unroll 1
  for (int which = 0; which < 2; ++which) {
    if (which == 0 && e0 - off[k0] <= kLeRun) continue;
    if (which == 1 && (k1 == k0 || off[k1 + 1] - s1 <= kLeRun)) continue;
    A acc[NC][W] = {};
    const int64_t pa = which == 0 ? a : s1, pb = which == 0 ? min<int64_t>(b, e0) : b;
    le_sum_rows<T, W, NC, A>(dy, D, c0, tpr, order, pa + sub, pb, rpb, acc);
    le_block_sum<W, NC, A>(acc, lc.tpr_shift, s_acc);
    if (sub == 0) {
      A* out = part + (2 * c + which) * D;
#pragma unroll
      for (int q = 0; q < NC; ++q) {
        const int col = c0 + q * tpr * W;
        if (col >= D) break;
#pragma unroll
        for (int e = 0; e < W; ++e) out[col + e] = acc[q][e];
      }
    }
  }
}

// One block (and column block) per chunk; it works if a leaf with more than kLeRun rows starts in
// the chunk, and adds that leaf's partial rows.
template <typename T, int W, int NC>
__global__ __launch_bounds__(kLeThreads) void le_join_kernel(
    const typename LeAcc<T>::type* __restrict__ part, const uint32_t* __restrict__ keys,
    const int32_t* __restrict__ off, int64_t V, int D, float scale, LeCols lc,
    T* __restrict__ dtable) {
  using A = typename LeAcc<T>::type;
  __shared__ A s_acc[NC * W * kLeThreads / 2];
  const int tpr = 1 << lc.tpr_shift, rpb = kLeThreads >> lc.tpr_shift;
  const int sub = threadIdx.x >> lc.tpr_shift, lr = threadIdx.x & (tpr - 1);
  int64_t c = leaf_block();
  const int c0 = ((int)(c % lc.col_blocks) * NC * tpr + lr) * W;
  c /= lc.col_blocks;
  const int64_t m = off[V], a = c * kLeRun, b = min<int64_t>(a + kLeRun, m);
  if (a >= m) return;
  const int64_t k0 = keys[a], k1 = keys[b - 1];
  const int64_t s1 = off[k1], e1 = off[k1 + 1];
  if (s1 < a || e1 - s1 <= kLeRun) return;
  A acc[NC][W] = {};
  const int64_t last = (e1 - 1) / kLeRun;
  for (int64_t p = c + sub; p <= last; p += rpb) {
    const A* in = part + (2 * p + (p == c && k1 != k0 ? 1 : 0)) * D;
#pragma unroll
    for (int q = 0; q < NC; ++q) {
      const int col = c0 + q * tpr * W;
      if (col >= D) break;
#pragma unroll
      for (int e = 0; e < W; ++e) acc[q][e] += in[col + e];
    }
  }
  le_block_sum<W, NC, A>(acc, lc.tpr_shift, s_acc);
  if (sub == 0) le_store<T, W, NC, A>(dtable + k1 * D, D, c0, tpr, scale, acc);
}

static LeCols le_cols(int D, int W, int NC) {
  const int vecs = (D + W - 1) / W;
  LeCols lc;
  lc.tpr_shift = 0;
  while (lc.tpr_shift < 6 && (1 << lc.tpr_shift) < vecs) ++lc.tpr_shift;
  const int per = NC << lc.tpr_shift;
  lc.col_blocks = (vecs + per - 1) / per;
  return lc;
}

// The widest vectors that every row's address and the width allow: 16 bytes, for 16-bit types also
// 4, else one element.
static int le_width(int elem, int D, int64_t stride, const void* a, const void* b) {
  const uintptr_t at = (uintptr_t)a | (uintptr_t)b;
  for (int bytes : {16, 4}) {
    const int w = bytes / elem;
    if (w >= 1 && D % w == 0 && stride % w == 0 && at % bytes == 0) return w;
  }
  return 1;
}

template <typename F>
static void le_dispatch_16(int W, F f) {
  if (W == 8)
    f(std::integral_constant<int, 8>{});
  else if (W == 2)
    f(std::integral_constant<int, 2>{});
  else
    f(std::integral_constant<int, 1>{});
}
template <typename F>
static void le_dispatch_32(int W, F f) {
  if (W == 4)
    f(std::integral_constant<int, 4>{});
  else
    f(std::integral_constant<int, 1>{});
}

template <typename T, bool kScale, int W>
static void le_forward(hipStream_t s, const void* ids, bool wide, const T* table, int64_t stride,
                       int64_t n, int64_t V, int D, float scale, T* y) {
  // wide rows: four vectors a lane while that leaves no lane idle
  const bool four = D >= 4 * kWave * W;
  const LeCols lc = le_cols(D, W, four ? 4 : 1);
  const int rows = (kLeThreads >> lc.tpr_shift) * kLeUnroll;
  const dim3 grid = leaf_grid((n + rows - 1) / rows * lc.col_blocks);
  auto go = [&](auto kern) {
    hipLaunchKernelGGL(kern, grid, dim3(kLeThreads), 0, s, ids, table, stride, n, V, D, scale, lc,
                       y);
    MT_HIP_CHECK(hipGetLastError());
  };
  if (four)
    wide ? go(le_forward_kernel<T, W, 4, kScale, true>)
         : go(le_forward_kernel<T, W, 4, kScale, false>);
  else
    wide ? go(le_forward_kernel<T, W, 1, kScale, true>)
         : go(le_forward_kernel<T, W, 1, kScale, false>);
}

void launch_leaf_embed(hipStream_t s, int type, const void* ids, bool wide, const void* table,
                       int64_t stride, int64_t n, int64_t V, int D, float scale, void* y) {
  if (n <= 0 || D <= 0) return;
  const int elem = type == kLeafF32 || type == kLeafRaw32 ? 4 : 2;
  const int W = le_width(elem, D, stride, table, y);
  if (type == kLeafF32)
    le_dispatch_32(W, [&](auto w) {
      le_forward<float, true, w()>(s, ids, wide, (const float*)table, stride, n, V, D, scale,
                                   (float*)y);
    });
  else if (type == kLeafRaw32)
    le_dispatch_32(W, [&](auto w) {
      le_forward<uint32_t, false, w()>(s, ids, wide, (const uint32_t*)table, stride, n, V, D, scale,
                                       (uint32_t*)y);
    });
  else if (type == kLeafF16)
    le_dispatch_16(W, [&](auto w) {
      le_forward<f16_t, true, w()>(s, ids, wide, (const f16_t*)table, stride, n, V, D, scale,
                                   (f16_t*)y);
    });
  else
    le_dispatch_16(W, [&](auto w) {
      le_forward<bf16_t, true, w()>(s, ids, wide, (const bf16_t*)table, stride, n, V, D, scale,
                                    (bf16_t*)y);
    });
}

// bytes of scratch for the partial rows
int64_t leaf_embed_grad_bytes(int type, int64_t n, int D) {
  if (n <= kLeRun) return 0;
  return 2 * ((n + kLeRun - 1) / kLeRun) * D * (type == kLeafF32 ? 8 : 4);
}

template <typename T, int W>
static void le_backward(hipStream_t s, const T* dy, const int32_t* order, const uint32_t* keys,
                        const int32_t* off, int64_t n, int64_t V, int D, float scale, T* dtable,
                        void* work) {
  using A = typename LeAcc<T>::type;
  const bool four = D >= 4 * kWave * W;
  const LeCols lc = le_cols(D, W, four ? 4 : 1);
  const int rpb = kLeThreads >> lc.tpr_shift;
  const int64_t light = (V + rpb - 1) / rpb;
  const int64_t chunks = n > kLeRun ? (n + kLeRun - 1) / kLeRun : 0;
  const dim3 grid = leaf_grid((light + chunks) * lc.col_blocks);
  auto go = [&](auto kern, auto join) {
    hipLaunchKernelGGL(kern, grid, dim3(kLeThreads), 0, s, dy, order, keys, off, V, D, scale, lc,
                       light, dtable, (A*)work);
    MT_HIP_CHECK(hipGetLastError());
    if (chunks > 0) {
      hipLaunchKernelGGL(join, leaf_grid(chunks * lc.col_blocks), dim3(kLeThreads), 0, s,
                         (const A*)work, keys, off, V, D, scale, lc, dtable);
      MT_HIP_CHECK(hipGetLastError());
    }
  };
  if (four)
    go(le_backward_kernel<T, W, 4>, le_join_kernel<T, W, 4>);
  else
    go(le_backward_kernel<T, W, 1>, le_join_kernel<T, W, 1>);
}

void launch_leaf_embed_grad(hipStream_t s, int type, const void* dy, const int32_t* order,
                            const uint32_t* keys, const int32_t* off, int64_t n, int64_t V, int D,
                            float scale, void* dtable, void* work) {
  if (D <= 0) return;
  const int W = le_width(type == kLeafF32 ? 4 : 2, D, D, dy, dtable);
  if (type == kLeafF32)
    le_dispatch_32(W, [&](auto w) {
      le_backward<float, w()>(s, (const float*)dy, order, keys, off, n, V, D, scale,
                              (float*)dtable, work);
    });
  else if (type == kLeafF16)
    le_dispatch_16(W, [&](auto w) {
      le_backward<f16_t, w()>(s, (const f16_t*)dy, order, keys, off, n, V, D, scale,
                              (f16_t*)dtable, work);
    });
  else
    le_dispatch_16(W, [&](auto w) {
      le_backward<bf16_t, w()>(s, (const bf16_t*)dy, order, keys, off, n, V, D, scale,
                               (bf16_t*)dtable, work);
    });
}

}  // namespace mt
