// The route of rows to leaves: a stable sort of the row numbers by leaf, and where each
// leaf's rows begin.
//
//   order[p]            the row at sorted position p; rows of a leaf keep their order
//   keys[p]             its leaf; a row whose leaf is outside [0, G) has no leaf and key G
//   offsets[g], g <= G  the first position of leaf g (of the rows without a leaf: g = G)
//   offsets[G + 1]      n
//
// A fitted tree sends its rows to leaves once (apply); the gradients of what the leaves hold are
// sums over each leaf's rows, and the grouped products need a leaf's rows side by side. Sums in
// sorted order do not depend on the launch, which sums by atomics would.
//
// The sort is an LSD radix sort with 8-bit digits: ceil(bits(G) / 8) stable passes, so one up to
// 255 leaves and three up to 2^24. Up to kLrTile rows one workgroup runs all passes in LDS (one
// launch; 16384 rows so: 22 us a pass, 12 with the tiles); beyond, a pass is a count of every
// tile's digits and a scatter that takes its own prefix over the earlier tiles (two launches; with
// more than kLrSelfTiles tiles a scan between them, since every scatter block reads all counts).
// It moves 8 to 16 bytes a row and pass; at a million rows it is bound by its launches and the
// latency inside them, not by memory: 19 us with 64 leaves, 41 with 4096; 100k rows of 1500 leaves
// 25.
#include "leaf.h"

namespace mt {

constexpr int kLrThreads = 1024;
constexpr int kLrItems = 4;
constexpr int kLrTile = kLrThreads * kLrItems;  // 4096 rows
constexpr int kLrWaves = kLrThreads / kWave;
// Leaves a row up to which the one workgroup fills the offsets too. us so / with a launch that
// searches: 4096 rows, 200 leaves 7.3 / 9.9, 16000 leaves 15.3 / 16.5; 1000 rows, 16000 leaves 20.8
// / 11.8.
constexpr int kLrFillLeaves = 4;
// Tiles up to which a scatter sums the earlier tiles' counts itself. us of a sort of 64 leaves so /
// with a scan: 500k rows (123 tiles) 14.4 / 17.9, 1M 19.0 / 23.8, 2M (489) 33.8 / 39.0, 4M (977)
// 72.7 / 71.3; of 4096 leaves 33.5 / 40.4, 41.8 / 51.7, 72.7 / 82.3, 151 / 146.
constexpr int kLrSelfTiles = 512;
// Offsets a lane fills by itself before the wave helps; us of a sort with 4 / 16 / 64: 100k rows in
// 1M leaves 43.9 / 42.1 / 43.1, 20k rows in few of 200k 48.3 / 48.1 / 47.3.
constexpr int kLrOwn = 16;

__device__ __forceinline__ uint32_t lr_key(const void* ids, bool wide, int64_t i, int G) {
  const int64_t v = wide ? ((const int64_t*)ids)[i] : (int64_t)((const int32_t*)ids)[i];
  return (uint64_t)v < (uint64_t)G ? (uint32_t)v : (uint32_t)G;
}

// lanes of the wave that hold the same digit (8 ballots), among those with `in`
__device__ __forceinline__ unsigned long long lr_match(uint32_t d, bool in) {
  unsigned long long m = __ballot(in);
#pragma unroll
  for (int b = 0; b < 8; ++b) {
    const bool bit = (d >> b) & 1u;
    const unsigned long long bb = __ballot(bit);
    m &= bit ? bb : ~bb;
  }
  return m;
}

// Ranks the tile's keys by digit. Item k of lane l of wave w is tile entry w * 256 + k * 64 + l.
// On return rk holds each item's rank among the wave's equal digits, s_wh the waves' counts.
__device__ __forceinline__ void lr_rank(const uint32_t (&key)[kLrItems], uint32_t (&rk)[kLrItems],
                                        int cnt, int shift, uint32_t (*s_wh)[256]) {
  const int lane = lane_id(), w = threadIdx.x / kWave;
  const unsigned long long lt = (1ull << lane) - 1ull;
#pragma unroll
  for (int k = 0; k < kLrItems; ++k) {
    const bool in = w * (kWave * kLrItems) + k * kWave + lane < cnt;
    const uint32_t d = (key[k] >> shift) & 255u;
    const unsigned long long m = lr_match(d, in);
    const uint32_t c = s_wh[w][d];
    rk[k] = c + (uint32_t)__popcll(m & lt);
    // (the wave's reads come before its writes, and those before the next item's reads)
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (in && (m & lt) == 0ull) s_wh[w][d] = c + (uint32_t)__popcll(m);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
}

// threads 0..255: the waves' counts -> their exclusive prefixes per digit; returns the digit's sum
__device__ __forceinline__ uint32_t lr_wave_prefix(uint32_t (*s_wh)[256]) {
  uint32_t s = 0;
#pragma unroll
  for (int q = 0; q < kLrWaves; ++q) {
    const uint32_t v = s_wh[q][threadIdx.x];
    s_wh[q][threadIdx.x] = s;
    s += v;
  }
  return s;
}

// exclusive prefix of v over threads 0..255 (the other threads pass 0 and ignore the result)
__device__ __forceinline__ uint32_t lr_digit_prefix(uint32_t v, uint32_t* s_w4) {
  const uint32_t incl = wave_incl_scan_u32(v);
  if (lane_id() == kWave - 1 && threadIdx.x < 256) s_w4[threadIdx.x / kWave] = incl;
  __syncthreads();
  uint32_t before = 0;
  for (int q = 0; q < (int)(threadIdx.x / kWave) && q < 4; ++q) before += s_w4[q];
  return before + incl - v;
}

// Position i starts every leaf after the key before it, up to its own; a run of more than kLrOwn
// leaves without rows is filled by the whole wave, all of whose lanes have to come here. i == n:
// the end, i > n: nothing.
__device__ __forceinline__ void lr_fill(int64_t i, int64_t n, int64_t prev, int64_t cur, int G,
                                        int32_t* __restrict__ offsets) {
  if (i == n) offsets[G + 1] = (int32_t)n;
  const bool wide = cur - prev > kLrOwn;
  if (!wide)
    for (int64_t g = prev + 1; g <= cur; ++g) offsets[g] = (int32_t)i;
  unsigned long long big = __ballot(wide);
  while (big) {
    const int src = __ffsll((long long)big) - 1;
    big &= big - 1;
    const int a = __shfl((int)prev, src, kWave), b = __shfl((int)cur, src, kWave);
    const int v = __shfl((int)i, src, kWave);
    for (int64_t g = (int64_t)a + 1 + lane_id(); g <= b; g += kWave) offsets[g] = v;
  }
}

// ---- up to kLrTile rows: all passes in one workgroup. offsets: null, or filled here.
__global__ __launch_bounds__(kLrThreads) void lr_small_kernel(const void* __restrict__ ids,
                                                              bool wide, int n, int G, int passes,
                                                              int32_t* __restrict__ order,
                                                              uint32_t* __restrict__ keys,
                                                              int32_t* __restrict__ offsets) {
  __shared__ uint32_t s_key[kLrTile], s_row[kLrTile];
  __shared__ uint32_t s_wh[kLrWaves][256];
  __shared__ uint32_t s_base[256], s_w4[4];
  const int tid = threadIdx.x, lane = lane_id(), w = tid / kWave;
  uint32_t key[kLrItems], row[kLrItems], rk[kLrItems];
#pragma unroll
  for (int k = 0; k < kLrItems; ++k) {
    const int i = w * (kWave * kLrItems) + k * kWave + lane;
    key[k] = i < n ? lr_key(ids, wide, i, G) : 0u;
    row[k] = (uint32_t)i;
  }
  for (int p = 0; p < passes; ++p) {
    const int shift = 8 * p;
    for (int i = tid; i < kLrWaves * 256; i += kLrThreads) (&s_wh[0][0])[i] = 0u;
    __syncthreads();
    lr_rank(key, rk, n, shift, s_wh);
    __syncthreads();
    const uint32_t tot = tid < 256 ? lr_wave_prefix(s_wh) : 0u;
    const uint32_t base = lr_digit_prefix(tot, s_w4);
    if (tid < 256) s_base[tid] = base;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kLrItems; ++k) {
      const int i = w * (kWave * kLrItems) + k * kWave + lane;
      if (i < n) {
        const uint32_t d = (key[k] >> shift) & 255u;
        const uint32_t to = s_base[d] + s_wh[w][d] + rk[k];
        s_key[to] = key[k];
        s_row[to] = row[k];
      }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kLrItems; ++k) {
      const int i = w * (kWave * kLrItems) + k * kWave + lane;
      if (i < n) {
        key[k] = s_key[i];
        row[k] = s_row[i];
      }
    }
  }
#pragma unroll
  for (int k = 0; k < kLrItems; ++k) {
    const int i = w * (kWave * kLrItems) + k * kWave + lane;
    if (i < n) {
      order[i] = (int32_t)row[k];
      keys[i] = key[k];
    }
  }
  if (offsets == nullptr) return;
#pragma unroll
  for (int k = 0; k < kLrItems; ++k) {
    const int i = w * (kWave * kLrItems) + k * kWave + lane;
    lr_fill(i, n, i > 0 && i <= n ? (int64_t)s_key[i - 1] : i == 0 ? -1 : 0,
            i < n ? (int64_t)key[k] : i == n ? (int64_t)G : 0, G, offsets);
  }
  // (all positions taken by rows: the end is one more)
  if (n == kLrTile && w == kLrWaves - 1)
    lr_fill(n + lane, n, lane == 0 ? (int64_t)s_key[n - 1] : 0, lane == 0 ? (int64_t)G : 0, G,
            offsets);
}

// ---- one pass over many tiles. kFirst: keys come from the leaf indices, rows are 0..n-1
template <bool kFirst>
__device__ __forceinline__ void lr_load(const void* ids, bool wide, const uint32_t* kin, int64_t p0,
                                        int cnt, int G, uint32_t (&key)[kLrItems]) {
  const int lane = lane_id(), w = threadIdx.x / kWave;
#pragma unroll
  for (int k = 0; k < kLrItems; ++k) {
    const int i = w * (kWave * kLrItems) + k * kWave + lane;
    if constexpr (kFirst)
      key[k] = i < cnt ? lr_key(ids, wide, p0 + i, G) : 0u;
    else
      key[k] = i < cnt ? kin[p0 + i] : 0u;
  }
}

template <bool kFirst>
__global__ __launch_bounds__(kLrThreads) void lr_count_kernel(const void* __restrict__ ids,
                                                              bool wide,
                                                              const uint32_t* __restrict__ kin,
                                                              int64_t n, int G, int shift,
                                                              uint32_t* __restrict__ counts) {
  __shared__ uint32_t s_wh[kLrWaves][256];
  const int w = threadIdx.x / kWave;
  for (int i = threadIdx.x; i < kLrWaves * 256; i += kLrThreads) (&s_wh[0][0])[i] = 0u;
  const int64_t p0 = (int64_t)blockIdx.x * kLrTile;
  const int cnt = (int)min<int64_t>(kLrTile, n - p0);
  uint32_t key[kLrItems];
  lr_load<kFirst>(ids, wide, kin, p0, cnt, G, key);
  __syncthreads();
  // counts alone do not depend on the order of these adds
#pragma unroll
  for (int k = 0; k < kLrItems; ++k)
    if (w * (kWave * kLrItems) + k * kWave + lane_id() < cnt)
      atomicAdd(&s_wh[w][(key[k] >> shift) & 255u], 1u);
  __syncthreads();
  if (threadIdx.x < 256) {
    uint32_t s = 0;
#pragma unroll
    for (int q = 0; q < kLrWaves; ++q) s += s_wh[q][threadIdx.x];
    counts[(int64_t)blockIdx.x * 256 + threadIdx.x] = s;
  }
}

// counts[t][d] -> the prefix over earlier tiles, in place; totals[d]. One block per 64 digits,
// 16 groups of tiles (many tiles only).
__global__ __launch_bounds__(1024) void lr_scan_kernel(uint32_t* __restrict__ counts, int T,
                                                       uint32_t* __restrict__ totals) {
  __shared__ uint32_t s_g[16][kWave];
  const int dl = threadIdx.x & (kWave - 1), g = threadIdx.x / kWave;
  const int d = blockIdx.x * kWave + dl;
  const int per = (T + 15) / 16;
  const int t0 = min(T, g * per), t1 = min(T, t0 + per);
  uint32_t sum = 0;
  for (int t = t0; t < t1; ++t) sum += counts[(int64_t)t * 256 + d];
  s_g[g][dl] = sum;
  __syncthreads();
  uint32_t run = 0;
  for (int q = 0; q < g; ++q) run += s_g[q][dl];
  for (int t = t0; t < t1; ++t) {
    const uint32_t v = counts[(int64_t)t * 256 + d];
    counts[(int64_t)t * 256 + d] = run;
    run += v;
  }
  if (g == 15) totals[d] = run;
}

template <bool kFirst, bool kSelf>
__global__ __launch_bounds__(kLrThreads) void lr_scatter_kernel(
    const void* __restrict__ ids, bool wide, const uint32_t* __restrict__ kin,
    const uint32_t* __restrict__ rin, int64_t n, int T, int G, int shift,
    const uint32_t* __restrict__ counts, const uint32_t* __restrict__ totals,
    uint32_t* __restrict__ kout, uint32_t* __restrict__ rout, int32_t* __restrict__ offsets) {
  __shared__ uint32_t s_wh[kLrWaves][256];
  __shared__ uint32_t s_pre[kLrWaves][256], s_tot[kLrWaves][256];
  __shared__ uint32_t s_base[256], s_w4[4];
  const int tid = threadIdx.x, lane = lane_id(), w = tid / kWave;
  for (int i = tid; i < kLrWaves * 256; i += kLrThreads) (&s_wh[0][0])[i] = 0u;
  const int64_t p0 = (int64_t)blockIdx.x * kLrTile;
  const int cnt = (int)min<int64_t>(kLrTile, n - p0);
  uint32_t key[kLrItems], row[kLrItems], rk[kLrItems];
  lr_load<kFirst>(ids, wide, kin, p0, cnt, G, key);
#pragma unroll
  for (int k = 0; k < kLrItems; ++k) {
    const int i = w * (kWave * kLrItems) + k * kWave + lane;
    if constexpr (kFirst)
      row[k] = (uint32_t)(p0 + i);
    else
      row[k] = i < cnt ? rin[p0 + i] : 0u;
  }
  if constexpr (kSelf) {
    // wave w sums the counts of tiles w, w + 16, ...: four digits a lane
    uint4 pre = make_uint4(0, 0, 0, 0), tot = make_uint4(0, 0, 0, 0);
#pragma unroll 4
    for (int t = w; t < T; t += kLrWaves) {
      const uint4 c = ((const uint4*)(counts + (int64_t)t * 256))[lane];
      const uint32_t m = t < (int)blockIdx.x ? 0xffffffffu : 0u;
      pre.x += c.x & m, pre.y += c.y & m, pre.z += c.z & m, pre.w += c.w & m;
      tot.x += c.x, tot.y += c.y, tot.z += c.z, tot.w += c.w;
    }
    ((uint4*)s_pre[w])[lane] = pre;
    ((uint4*)s_tot[w])[lane] = tot;
  }
  __syncthreads();
  lr_rank(key, rk, cnt, shift, s_wh);
  __syncthreads();
  uint32_t pre = 0, tot = 0;
  if (tid < 256) {
    lr_wave_prefix(s_wh);
    if constexpr (kSelf) {
#pragma unroll
      for (int q = 0; q < kLrWaves; ++q) pre += s_pre[q][tid], tot += s_tot[q][tid];
    } else {
      pre = counts[(int64_t)blockIdx.x * 256 + tid];
      tot = totals[tid];
    }
  }
  const uint32_t base = lr_digit_prefix(tot, s_w4);
  if (tid < 256) {
    s_base[tid] = base + pre;
    // a single pass: the digits are the leaves
    if (offsets != nullptr && blockIdx.x == 0) {
      if (tid <= G) offsets[tid] = (int32_t)base;
      if (tid == 0) offsets[G + 1] = (int32_t)n;
    }
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kLrItems; ++k) {
    const int i = w * (kWave * kLrItems) + k * kWave + lane;
    if (i < cnt) {
      const uint32_t d = (key[k] >> shift) & 255u;
      const uint32_t to = s_base[d] + s_wh[w][d] + rk[k];
      kout[to] = key[k];
      rout[to] = row[k];
    }
  }
}

// ---- offsets from the sorted keys. Few rows: every leaf searches a copy of the keys in LDS.
__global__ __launch_bounds__(256) void lr_offsets_search_kernel(const uint32_t* __restrict__ keys,
                                                                int n, int G,
                                                                int32_t* __restrict__ offsets) {
  __shared__ uint32_t s_key[kLrTile];
  for (int i = threadIdx.x; i < n; i += 256) s_key[i] = keys[i];
  __syncthreads();
  const int64_t g = leaf_block() * 256 + threadIdx.x;
  if (g > (int64_t)G + 1) return;
  int lo = 0, hi = n;
  if (g == (int64_t)G + 1) lo = n;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (s_key[mid] < (uint32_t)g)
      lo = mid + 1;
    else
      hi = mid;
  }
  offsets[g] = lo;
}

// Many rows: lr_fill for every position.
__global__ __launch_bounds__(256) void lr_offsets_fill_kernel(const uint32_t* __restrict__ keys,
                                                              int64_t n, int G,
                                                              int32_t* __restrict__ offsets) {
  const int64_t i = leaf_block() * 256 + threadIdx.x;
  int64_t prev = 0, cur = 0;
  if (i <= n) {
    prev = i > 0 ? (int64_t)keys[i - 1] : -1;
    cur = i < n ? (int64_t)keys[i] : (int64_t)G;
  }
  lr_fill(i, n, prev, cur, G, offsets);
}

int leaf_route_passes(int G) {
  int bits = 1;
  while (bits < 31 && (1ll << bits) <= (int64_t)G) ++bits;  // keys 0..G
  return (bits + 7) / 8;
}

// 32-bit words of scratch a sort of n rows needs: a second keys + rows buffer, the tiles' counts
int64_t leaf_route_words(int64_t n, int G) {
  if (n <= kLrTile) return 0;
  const int64_t T = (n + kLrTile - 1) / kLrTile;
  return (leaf_route_passes(G) > 1 ? 2 * n : 0) + 256 * T + 256 + 3;
}

void launch_leaf_route(hipStream_t stream, const void* ids, bool wide, int64_t n, int G,
                       int32_t* order, uint32_t* keys, int32_t* offsets, uint32_t* work) {
  const int passes = leaf_route_passes(G);
  if (n <= kLrTile) {
    const bool fill = G <= kLrFillLeaves * n;
    if (n > 0) {
      hipLaunchKernelGGL(lr_small_kernel, dim3(1), dim3(kLrThreads), 0, stream, ids, wide, (int)n,
                         G, passes, order, keys, fill ? offsets : nullptr);
      MT_HIP_CHECK(hipGetLastError());
    }
    if (!fill) {
      hipLaunchKernelGGL(lr_offsets_search_kernel, leaf_grid(((int64_t)G + 2 + 255) / 256),
                         dim3(256), 0, stream, keys, (int)n, G, offsets);
      MT_HIP_CHECK(hipGetLastError());
    }
    return;
  }
  const int T = (int)((n + kLrTile - 1) / kLrTile);
  const bool self = T <= kLrSelfTiles;
  uint32_t* counts = work;  // first: 16-byte loads of it
  uint32_t* totals = counts + 256 * (int64_t)T;
  uint32_t* k2 = totals + 256;
  uint32_t* r2 = k2 + n;
  uint32_t* const r1 = (uint32_t*)order;
  for (int p = 0; p < passes; ++p) {
    // the last pass ends in keys / order: passes alternate towards it
    const bool to_out = ((passes - 1 - p) & 1) == 0;
    uint32_t* ko = to_out ? keys : k2;
    uint32_t* ro = to_out ? r1 : r2;
    const uint32_t* ki = to_out ? k2 : keys;
    const uint32_t* ri = to_out ? r2 : r1;
    int32_t* off = passes == 1 ? offsets : nullptr;
    const dim3 g(T), b(kLrThreads);
    if (p == 0)
      hipLaunchKernelGGL(lr_count_kernel<true>, g, b, 0, stream, ids, wide, ki, n, G, 8 * p,
                         counts);
    else
      hipLaunchKernelGGL(lr_count_kernel<false>, g, b, 0, stream, ids, wide, ki, n, G, 8 * p,
                         counts);
    MT_HIP_CHECK(hipGetLastError());
    if (!self) {
      hipLaunchKernelGGL(lr_scan_kernel, dim3(4), dim3(1024), 0, stream, counts, T, totals);
      MT_HIP_CHECK(hipGetLastError());
    }
    auto go = [&](auto kern) {
      hipLaunchKernelGGL(kern, g, b, 0, stream, ids, wide, ki, ri, n, T, G, 8 * p, counts, totals,
                         ko, ro, off);
      MT_HIP_CHECK(hipGetLastError());
    };
    if (p == 0)
      self ? go(lr_scatter_kernel<true, true>) : go(lr_scatter_kernel<true, false>);
    else
      self ? go(lr_scatter_kernel<false, true>) : go(lr_scatter_kernel<false, false>);
  }
  if (passes > 1) {
    hipLaunchKernelGGL(lr_offsets_fill_kernel, leaf_grid((n + 1 + 255) / 256), dim3(256), 0, stream,
                       keys, n, G, offsets);
    MT_HIP_CHECK(hipGetLastError());
  }
}

}  // namespace mt
