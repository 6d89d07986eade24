// Embedding by leaf: y[i] = scale * table[leaf(i)], and its gradient summed by sorted leaves.
//
// Forward: a row without a leaf (its index outside [0, V)) gets zeros. Each row's vector is read
// and written once by a group of lanes, up to 16 bytes a lane.
//
// Gradient: dtable[v] = scale * sum of dy over the rows of leaf v, for every v (zeros where no row
// is). The rows are sorted by leaf first (leaf_route.hip), so a leaf's rows are a run of `order`,
// and every sum has one fixed order: the result does not depend on the launch. The sorted positions
// are cut into chunks, one for a group of lanes, which streams its chunk's rows (their numbers are
// known at once, so a batch of rows is in flight) and writes out a sum where the leaf changes. A
// leaf that reaches over a chunk's end leaves partial rows there, at most two a chunk, and a second
// launch adds a leaf's partial rows. Leaves without rows are found through the offsets.
//
// Sums are held in 32 bits for 16-bit types and in 64 bits for f32: a leaf may hold most of a
// million rows, and a 64-bit add costs no more than a 32-bit one here, where memory is the bound.
//
// Both are bound by memory where rows are wide. Launches on four sets of operands in turn, where a
// copy reaches 4.9 TB/s: 200k rows of 2048 f16 in 120000 leaves (87000 of them met) forward 264 us
// (4.45 TB/s), gradient 291 us (4.5 TB/s). 1M rows of 63 f32 in 64 leaves 57 us (4.5 TB/s) and 70
// us (3.7 TB/s); on one set, which the last-level cache holds in part, 45 and 65; inside a training
// pass, where the gradient comes behind the forward pass's writes, 60 and 95. 1M rows of 16 f32 in
// 93500 leaves, random 64-byte reads, 22 us (3.5 TB/s) and 100 us.
#include "leaf.h"

namespace mt {

constexpr int kLeThreads = 256;
// Rows of a group in flight, in the forward pass and in the gradient. Each takes dependent loads
// (number, row), so narrow vectors need more of them. us, 1M rows of 63 columns of f32 with 4 / 16
// / 32 forward 62 / 57 / 83, gradient 80 / 70 / 76; 200k rows of 2048 columns of f16 with 4 / 8
// forward 264 / 269, with 4 / 8 / 16 gradient 294 / 291 / 290.
constexpr int le_unroll(int bytes) { return bytes >= 16 ? 4 : 16; }
constexpr int le_batch(int bytes) { return bytes >= 16 ? 8 : 16; }
// Leaves that a group looks over for missing rows; a gradient's us with 4 / 16 / 32: 16384 rows, 1M
// leaves, 63 columns of f32 75 / 59 / 60, 16 columns 15.7 / 16.7 / 17.3; 2000 rows, 200k leaves, 64
// columns 13.4 / 14.9 / 15.4.
constexpr int kLeEmpty = 16;

template <typename T>
struct LeAcc {
  using type = float;
};
template <>
struct LeAcc<float> {
  using type = double;
};

// Columns of a lane: one vector of W elements. (Several, with the row's number read once for all of
// them, take longer: 2048 columns of f16 290 us with four, 261 with one.)
struct LeCols {
  int tpr_shift;   // lanes of a row's group: 1 << tpr_shift, at most 64
  int col_blocks;  // column blocks of tpr * W columns
};

// kWave: a row's group is a whole wave, so the row's number and address are scalars (63 columns of
// f32: the 64-bit address arithmetic of every lane bound the kernel before).
template <bool kWave>
__device__ __forceinline__ int32_t le_same(int32_t v) {
  return kWave ? __builtin_amdgcn_readfirstlane(v) : v;
}
template <bool kWave>
__device__ __forceinline__ int64_t le_same(int64_t v) {
  if constexpr (!kWave) return v;
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)v);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)((uint64_t)v >> 32));
  return (int64_t)(((uint64_t)hi << 32) | lo);
}

template <typename T, int W, bool kWide, bool kWave>
__global__ __launch_bounds__(kLeThreads) void le_forward_kernel(
    const void* __restrict__ ids, const T* __restrict__ table, int64_t stride, int64_t n,
    int64_t V, int D, float scale, LeCols lc, T* __restrict__ y) {
  constexpr int kUnroll = le_unroll(W * (int)sizeof(T));
  const int tpr = 1 << lc.tpr_shift, rpb = kLeThreads >> lc.tpr_shift;
  const int sub = le_same<kWave>((int32_t)(threadIdx.x >> lc.tpr_shift));
  const int lr = threadIdx.x & (tpr - 1);
  const int64_t blk = leaf_block();
  const int64_t r0 = (blk / lc.col_blocks) * (rpb * kUnroll) + sub;
  const int c = ((int)(blk % lc.col_blocks) * tpr + lr) * W;
  int64_t id[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int64_t r = r0 + (int64_t)u * rpb;
    id[u] = -1;
    if (r < n) id[u] = kWide ? ((const int64_t*)ids)[r] : (int64_t)((const int32_t*)ids)[r];
    id[u] = le_same<kWave>(id[u]);
  }
  if (c >= D) return;
  LeafVec<T, W> v[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    v[u] = LeafVec<T, W>{};
    if ((uint64_t)id[u] < (uint64_t)V)
      v[u] = *(const LeafVec<T, W>*)(table + id[u] * stride + c);
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int64_t r = r0 + (int64_t)u * rpb;
    if (r >= n) break;
#pragma unroll
    for (int e = 0; e < W; ++e) v[u].v[e] = leaf_from<T>(leaf_f32(v[u].v[e]) * scale);
    *(LeafVec<T, W>*)(y + r * D + c) = v[u];
  }
}

// the sums of the block's row groups, added in their order; group 0's lanes hold the result
template <int W, int THREADS, typename A>
__device__ __forceinline__ void le_block_sum(A (&acc)[W], int tpr_shift, A* s_acc) {
  const int tpr = 1 << tpr_shift, rpb = THREADS >> tpr_shift;
  const int sub = threadIdx.x >> tpr_shift, lr = threadIdx.x & (tpr - 1);
  // pairwise: groups [half, 2 half) hand theirs to groups [0, half)
  for (int half = rpb >> 1; half > 0; half >>= 1) {
    if (sub >= half && sub < 2 * half) {
#pragma unroll
      for (int e = 0; e < W; ++e) s_acc[(e * half + (sub - half)) * tpr + lr] = acc[e];
    }
    __syncthreads();
    if (sub < half) {
#pragma unroll
      for (int e = 0; e < W; ++e) acc[e] += s_acc[(e * half + sub) * tpr + lr];
    }
    __syncthreads();
  }
}

template <typename T, int W, typename A>
__device__ __forceinline__ void le_store(T* __restrict__ out, float scale, const A (&acc)[W]) {
  LeafVec<T, W> v;
#pragma unroll
  for (int e = 0; e < W; ++e) v.v[e] = leaf_from<T>((float)(acc[e] * (A)scale));
  *(LeafVec<T, W>*)out = v;
}

// Blocks below `chunk_blocks`: a chunk of 1 << run_shift sorted positions for each group of lanes,
// partial rows into `part` ([2 * chunks][D]: of the leaf that reaches into the chunk, of the one
// that starts in it and reaches out; open[chunk]: that one's number + 1, or 0). Blocks from there
// on: zeros for the leaves without rows.
template <typename T, int W, bool kWave>
__global__ __launch_bounds__(kLeThreads) void le_backward_kernel(
    const T* __restrict__ dy, int64_t stride, const int32_t* __restrict__ order,
    const uint32_t* __restrict__ keys, const int32_t* __restrict__ off, int64_t V, int D,
    float scale, LeCols lc, int run_shift, int64_t chunks, int64_t chunk_blocks,
    T* __restrict__ dtable, typename LeAcc<T>::type* __restrict__ part,
    uint32_t* __restrict__ open) {
  using A = typename LeAcc<T>::type;
  constexpr int kBatch = le_batch(W * (int)sizeof(T));
  const int tpr = 1 << lc.tpr_shift, rpb = kLeThreads >> lc.tpr_shift;
  const int sub = le_same<kWave>((int32_t)(threadIdx.x >> lc.tpr_shift));
  const int lr = threadIdx.x & (tpr - 1);
  const int64_t blk = leaf_block();
  if (blk >= chunk_blocks) {
    const int64_t v0 = ((blk - chunk_blocks) * rpb + sub) * kLeEmpty;
    uint32_t none = 0;
#pragma unroll
    for (int i = 0; i < kLeEmpty; ++i)
      if (v0 + i < V && off[v0 + i] == off[v0 + i + 1]) none |= 1u << i;
    while (none) {
      const int i = __ffs((int)none) - 1;
      none &= none - 1;
      for (int c = lr * W; c < D; c += tpr * W)
        *(LeafVec<T, W>*)(dtable + (v0 + i) * D + c) = LeafVec<T, W>{};
    }
    return;
  }
  const int64_t chunk = blk / lc.col_blocks * rpb + sub, m = off[V];
  const int c0 = ((int)(blk % lc.col_blocks) * tpr + lr) * W;
  const int64_t a = chunk << run_shift, b = min<int64_t>(a + (1 << run_shift), m);
  if (a >= m || c0 >= D) {
    if (c0 == 0 && chunk < chunks) open[chunk] = 0;
    return;
  }
  const bool into = a > 0 && keys[a - 1] == keys[a];
  const bool out_of = b < m && keys[b] == keys[b - 1];
  if (c0 == 0) open[chunk] = out_of && !(into && keys[a] == keys[b - 1]) ? keys[b - 1] + 1 : 0;
  A acc[W] = {};
  uint32_t cur = (uint32_t)le_same<kWave>((int32_t)keys[a]);
  bool first = true;
  auto partial = [&](int which) {
    A* const to = part + (2 * chunk + which) * D + c0;
#pragma unroll
    for (int e = 0; e < W; ++e) to[e] = acc[e];
  };
  for (int64_t p = a; p < b; p += kBatch) {
    uint32_t key[kBatch];
    LeafVec<T, W> v[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int64_t pu = min(p + u, b - 1);
      key[u] = (uint32_t)le_same<kWave>((int32_t)keys[pu]);
      v[u] = *(const LeafVec<T, W>*)(dy + le_same<kWave>(order[pu]) * stride + c0);
    }
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      if (p + u >= b) break;
      if (key[u] != cur) {
        if (first && into)
          partial(0);
        else
          le_store<T, W, A>(dtable + (int64_t)cur * D + c0, scale, acc);
        first = false;
        cur = key[u];
#pragma unroll
        for (int e = 0; e < W; ++e) acc[e] = 0;
      }
#pragma unroll
      for (int e = 0; e < W; ++e) acc[e] += (A)leaf_f32(v[u].v[e]);
    }
  }
  if (first && into)
    partial(0);
  else if (out_of)
    partial(1);
  else
    le_store<T, W, A>(dtable + (int64_t)cur * D + c0, scale, acc);
}

// Adds the partial rows of the leaves that reach over a chunk's end. One block (and column block)
// for each leaf (kByLeaf), or for each chunk in which such a leaf may start, whichever are fewer.
// Few leaves have many partial rows each, so their blocks are larger (16384 rows of one leaf, 1024
// columns of bf16: a gradient takes 36 us, 48 with 256 threads; 1M rows, 64 columns of f32 222 and
// 677).
template <bool kByLeaf>
constexpr int kLeJoinThreads = kByLeaf ? 1024 : kLeThreads;
template <typename T, int W, bool kByLeaf>
__global__ __launch_bounds__(kLeJoinThreads<kByLeaf>) void le_join_kernel(
    const typename LeAcc<T>::type* __restrict__ part, const uint32_t* __restrict__ open,
    const int32_t* __restrict__ off, int64_t count, int D, float scale, LeCols lc, int run_shift,
    T* __restrict__ dtable) {
  using A = typename LeAcc<T>::type;
  constexpr int kThreads = kLeJoinThreads<kByLeaf>;
  __shared__ A s_acc[W * kThreads / 2];
  const int64_t blk = leaf_block(), i = blk / lc.col_blocks;
  if (i >= count) return;
  int64_t k, chunk;
  if constexpr (kByLeaf) {
    k = i, chunk = off[k] >> run_shift;
    if (off[k + 1] <= (chunk + 1) << run_shift) return;
  } else {
    chunk = i, k = (int64_t)open[chunk] - 1;
    if (k < 0) return;
  }
  const int tpr = 1 << lc.tpr_shift, rpb = kThreads >> lc.tpr_shift;
  const int sub = threadIdx.x >> lc.tpr_shift, lr = threadIdx.x & (tpr - 1);
  const int c0 = ((int)(blk % lc.col_blocks) * tpr + lr) * W;
  const int64_t last = (off[k + 1] - 1) >> run_shift;
  A acc[W] = {};
  if (c0 < D) {
#pragma unroll 8
    for (int64_t p = chunk + sub; p <= last; p += rpb) {
      const A* const in = part + (2 * p + (p == chunk ? 1 : 0)) * D + c0;
#pragma unroll
      for (int e = 0; e < W; ++e) acc[e] += in[e];
    }
  }
  le_block_sum<W, kThreads, A>(acc, lc.tpr_shift, s_acc);
  if (sub == 0 && c0 < D) le_store<T, W, A>(dtable + (int64_t)k * D + c0, scale, acc);
}

static LeCols le_cols(int D, int W) {
  const int vecs = (D + W - 1) / W;
  LeCols lc;
  lc.tpr_shift = 0;
  while (lc.tpr_shift < 6 && (1 << lc.tpr_shift) < vecs) ++lc.tpr_shift;
  lc.col_blocks = (vecs + (1 << lc.tpr_shift) - 1) >> lc.tpr_shift;
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

template <typename T, int W>
static void le_forward(hipStream_t s, const void* ids, bool wide, const T* table, int64_t stride,
                       int64_t n, int64_t V, int D, float scale, T* y) {
  const LeCols lc = le_cols(D, W);
  const int rows = (kLeThreads >> lc.tpr_shift) * le_unroll(W * (int)sizeof(T));
  const dim3 grid = leaf_grid((n + rows - 1) / rows * lc.col_blocks);
  auto go = [&](auto kern) {
    hipLaunchKernelGGL(kern, grid, dim3(kLeThreads), 0, s, ids, table, stride, n, V, D, scale, lc,
                       y);
    MT_HIP_CHECK(hipGetLastError());
  };
  if (lc.tpr_shift == 6)
    wide ? go(le_forward_kernel<T, W, true, true>) : go(le_forward_kernel<T, W, false, true>);
  else
    wide ? go(le_forward_kernel<T, W, true, false>) : go(le_forward_kernel<T, W, false, false>);
}

void launch_leaf_embed(hipStream_t s, int type, const void* ids, bool wide, const void* table,
                       int64_t stride, int64_t n, int64_t V, int D, float scale, void* y) {
  if (n <= 0 || D <= 0) return;
  const int W = le_width(type == kLeafF32 ? 4 : 2, D, stride, table, y);
  if (type == kLeafF32)
    le_dispatch_32(W, [&](auto w) {
      le_forward<float, w()>(s, ids, wide, (const float*)table, stride, n, V, D, scale,
                             (float*)y);
    });
  else if (type == kLeafF16)
    le_dispatch_16(W, [&](auto w) {
      le_forward<f16_t, w()>(s, ids, wide, (const f16_t*)table, stride, n, V, D, scale,
                             (f16_t*)y);
    });
  else
    le_dispatch_16(W, [&](auto w) {
      le_forward<bf16_t, w()>(s, ids, wide, (const bf16_t*)table, stride, n, V, D, scale,
                              (bf16_t*)y);
    });
}

// Sorted positions of a chunk: 16 to 256, so few that the chunks make about 4096 waves (16 on each
// CU) of 16-byte vectors, 2048 of narrower ones; longer chunks leave fewer partial rows. us with
// half / these / two / four times as many: 1M rows, 63 columns of f32 70 / 70 / 78 / 80, 300k rows
// 47 / 32 / 31 / 32; 200k rows, 2048 columns of f16 302 / 291 / 293 / 302.
static int le_run_shift(int64_t n, const LeCols& lc, int bytes) {
  const int64_t waves = bytes >= 16 ? 4096 : 2048;
  int shift = 8;
  while (shift > 4 && ((n >> shift) * lc.col_blocks << lc.tpr_shift) / kWave < waves) --shift;
  return shift;
}

// bytes of scratch for the partial rows, whichever width is taken
int64_t leaf_embed_grad_bytes(int type, int64_t n, int D) {
  const int elem = type == kLeafF32 ? 4 : 2;
  int shift = 8;
  for (int W : {8, 4, 2, 1}) shift = std::min(shift, le_run_shift(n, le_cols(D, W), W * elem));
  return ((n >> shift) + 1) * (2 * (int64_t)D * (type == kLeafF32 ? 8 : 4) + 4);
}

template <typename T, int W>
static void le_backward(hipStream_t s, const T* dy, int64_t stride, const int32_t* order,
                        const uint32_t* keys, const int32_t* off, int64_t n, int64_t V, int D,
                        float scale, T* dtable, void* work) {
  using A = typename LeAcc<T>::type;
  const LeCols lc = le_cols(D, W);
  const int rpb = kLeThreads >> lc.tpr_shift, shift = le_run_shift(n, lc, W * (int)sizeof(T));
  const int64_t chunks = (n + (1 << shift) - 1) >> shift;
  const int64_t chunk_blocks = (chunks + rpb - 1) / rpb * lc.col_blocks;
  const int64_t empty = (V + rpb * kLeEmpty - 1) / (rpb * kLeEmpty);
  A* const part = (A*)work;
  uint32_t* const open = (uint32_t*)(part + 2 * chunks * D);
  auto go = [&](auto kern) {
    hipLaunchKernelGGL(kern, leaf_grid(chunk_blocks + empty), dim3(kLeThreads), 0, s, dy, stride,
                       order, keys, off, V, D, scale, lc, shift, chunks, chunk_blocks, dtable, part,
                       open);
    MT_HIP_CHECK(hipGetLastError());
  };
  lc.tpr_shift == 6 ? go(le_backward_kernel<T, W, true>) : go(le_backward_kernel<T, W, false>);
  if (chunks > 1) {
    const int64_t count = std::min(V, chunks - 1);
    auto join = [&](auto kern, int threads) {
      hipLaunchKernelGGL(kern, leaf_grid(count * lc.col_blocks), dim3(threads), 0, s, part, open,
                         off, count, D, scale, lc, shift, dtable);
      MT_HIP_CHECK(hipGetLastError());
    };
    V < chunks ? join(le_join_kernel<T, W, true>, kLeJoinThreads<true>)
               : join(le_join_kernel<T, W, false>, kLeJoinThreads<false>);
  }
}

void launch_leaf_embed_grad(hipStream_t s, int type, const void* dy, int64_t stride,
                            const int32_t* order, const uint32_t* keys, const int32_t* off,
                            int64_t n, int64_t V, int D, float scale, void* dtable, void* work) {
  if (D <= 0) return;
  const int W = le_width(type == kLeafF32 ? 4 : 2, D, stride, dy, dtable);
  if (type == kLeafF32)
    le_dispatch_32(W, [&](auto w) {
      le_backward<float, w()>(s, (const float*)dy, stride, order, keys, off, n, V, D, scale,
                              (float*)dtable, work);
    });
  else if (type == kLeafF16)
    le_dispatch_16(W, [&](auto w) {
      le_backward<f16_t, w()>(s, (const f16_t*)dy, stride, order, keys, off, n, V, D, scale,
                              (f16_t*)dtable, work);
    });
  else
    le_dispatch_16(W, [&](auto w) {
      le_backward<bf16_t, w()>(s, (const bf16_t*)dy, stride, order, keys, off, n, V, D, scale,
                               (bf16_t*)dtable, work);
    });
}

}  // namespace mt
