// Products grouped by leaf: y[i] = W[g] x[i] + b[g] for the leaf g of row i, and the gradients
//   dx[i] = W[g]^T dy[i],   dW[g] = sum over g's rows of dy[i] x[i]^T.
// (db[g], the sum of dy over g's rows, is the embedding's gradient: leaf_embed.hip.)
//
// x is [n, K], W is [G, N, K], rows of a leaf are found through the route's `order` and `offsets`
// (leaf_route.hip). Rows are gathered while a tile is loaded and scattered when it is stored, so
// no sorted copy of x or y is made. A row without a leaf gets zeros in y and dx.
//
// All products run on the matrix cores with 32-bit accumulators (f32 inputs: the f32 MFMA, no
// rounding of inputs). The A operand of every MFMA is the side whose index runs along the output's
// columns, so a lane ends with four neighbouring columns of one row and stores them together.
#include "leaf.h"

namespace mt {

constexpr int kLlThreads = 256;
constexpr int kLlWaves = kLlThreads / kWave;
constexpr int kLlSmallRows = 64;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));

template <typename T>
struct Ll {
  static constexpr int kEpc = 16 / (int)sizeof(T);     // elements of a 16-byte chunk
  static constexpr int kDepth = 128 / (int)sizeof(T);  // contraction depth of an LDS tile
};

// 16 x 16 products over 4 chunks' worth of depth: lane l holds row l % 16 and the kEpc elements of
// chunk l / 16 of either operand. 16-bit types: one MFMA over 32; f32: four over 4, whose lanes'
// k run 4 (l / 16) + u -- any order of k serves as long as both operands share it.
template <typename T>
__device__ __forceinline__ f32x4 ll_mma(uint4 a, uint4 b, f32x4 c) {
  if constexpr (sizeof(T) == 4) {
    const f32x4 av = __builtin_bit_cast(f32x4, a), bv = __builtin_bit_cast(f32x4, b);
#pragma unroll
    for (int u = 0; u < 4; ++u)
      c = __builtin_amdgcn_mfma_f32_16x16x4f32(av[u], bv[u], c, 0, 0, 0);
    return c;
  } else if constexpr (std::is_same_v<T, f16_t>) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h16x8, a),
                                                  __builtin_bit_cast(h16x8, b), c, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b16x8, a),
                                                   __builtin_bit_cast(b16x8, b), c, 0, 0, 0);
  }
}

// `valid` (may be <= 0) leading elements of the chunk at p, zeros behind them. kAligned: chunks are
// 16-byte aligned and either whole or empty.
template <typename T, bool kAligned>
__device__ __forceinline__ uint4 ll_chunk(const T* p, int valid) {
  constexpr int E = Ll<T>::kEpc;
  uint4 v = make_uint4(0, 0, 0, 0);
  if (valid >= E) {
    if constexpr (kAligned)
      v = *(const uint4*)p;
    else
      __builtin_memcpy(&v, p, 16);
  } else if (!kAligned && valid > 0) {
    T e[E] = {};
#pragma unroll
    for (int i = 0; i < E; ++i)
      if (i < valid) e[i] = p[i];
    __builtin_memcpy(&v, e, 16);
  }
  return v;
}

// ---- LDS tiles of 128 bytes of depth for ROWS rows ("flat": depth contiguous) or of kDepth rows
// of ROWS columns ("turned": depth is the row). Both hold ROWS * 8 chunks.
//
// Flat: row r's chunk c lies at r * 8 + (c ^ (r & 7)), so the 16 rows a fragment reads at one c
// spread over the banks.
// Turned: columns come in slabs of 16, row k's slab s lies at s ^ f(k), for the same reason.
template <typename T>
__device__ __forceinline__ int ll_flat_chunk(int r, int c) {
  return r * 8 + (c ^ (r & 7));
}
template <typename T, int COLS>
__device__ __forceinline__ int ll_turn_slab(int k, int slab) {
  const int f = sizeof(T) == 4 ? (k >> 2) & 3 : (k & 3) | ((k >> 3) & 1) << 2;
  return slab ^ (f & (COLS / 16 - 1));
}
template <typename T, int COLS>
__device__ __forceinline__ int ll_turn_chunk(int k, int c) {  // chunk c of row k
  constexpr int kPer = 16 * (int)sizeof(T) / 16;              // chunks of a slab
  constexpr int kRow = COLS * (int)sizeof(T) / 16;
  return k * kRow + ll_turn_slab<T, COLS>(k, c / kPer) * kPer + c % kPer;
}

// fragment (row r0 + l % 16, chunk 4 * step + l / 16) of a flat tile
template <typename T>
__device__ __forceinline__ uint4 ll_frag_flat(const uint4* s, int r0, int step) {
  const int l = lane_id();
  return s[ll_flat_chunk<T>(r0 + (l & 15), 4 * step + (l >> 4))];
}

// the same fragment of a turned tile: column c0 + l % 16, depth (4 * step + l / 16) * kEpc on
template <typename T, int COLS>
__device__ __forceinline__ uint4 ll_frag_turn(const uint4* s, int c0, int step) {
  const int l = lane_id();
  if constexpr (sizeof(T) == 4) {
    const float* f = (const float*)s;
    uint4 v;
    uint32_t* e = (uint32_t*)&v;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int k = 16 * step + 4 * (l >> 4) + u;
      e[u] = __float_as_uint(f[k * COLS + ll_turn_slab<T, COLS>(k, c0 >> 4) * 16 + (l & 15)]);
    }
    return v;
  } else {
    // ds_read_b64_tr_b16: 16 lanes read 4 rows of 16 columns, 8 bytes each, and lane i of them
    // gets column i of the 4 rows
    const uint16_t* h = (const uint16_t*)s;
    s16x4 part[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int k = 32 * step + 8 * (l >> 4) + 4 * u + ((l & 15) >> 2);
      const uint16_t* p =
          h + k * COLS + ll_turn_slab<T, COLS>(k, c0 >> 4) * 16 + (l & 3) * 4;
      part[u] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (__attribute__((address_space(3))) s16x4*)p);
    }
    uint4 v;
    __builtin_memcpy(&v, &part[0], 8);
    __builtin_memcpy((char*)&v + 8, &part[1], 8);
    return v;
  }
}

// four neighbouring columns of one output row
template <typename T>
__device__ __forceinline__ void ll_store4(T* p, f32x4 v, int left, bool vec) {
  if (vec && left >= 4) {
    LeafVec<T, 4> o;
#pragma unroll
    for (int e = 0; e < 4; ++e) o.v[e] = leaf_from<T>(v[e]);
    *(LeafVec<T, 4>*)p = o;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < left) p[e] = leaf_from<T>(v[e]);
  }
}

struct LlTile {
  const void* src;  // x (forward) or dy (kDx): rows of `depth` elements
  const void* w;    // [G, N, K]
  const void* bias;
  void* out;  // y or dx: rows of `cols` elements
  const int32_t* order;
  const int32_t* off;
  int64_t src_stride, w_stride;  // elements between src rows; between leaves' matrices
  int G, depth, cols, w_row;     // w_row: elements of a row of W (K)
  int col_tiles, bj_shift;
  int64_t tiles;
};

// One tile of BJ rows of one leaf by BI output columns. Forward: A = W's rows, flat; kDx: A = W
// with its rows as depth, turned. B = gathered rows of src, flat.
template <typename T, bool kDx, int BJ, int BI, int WJ, bool kAligned>
__global__ __launch_bounds__(kLlThreads) void ll_tile_kernel(LlTile a) {
  constexpr int E = Ll<T>::kEpc, KD = Ll<T>::kDepth;
  constexpr int WI = kLlWaves / WJ;
  constexpr int SJ = BJ / WJ / 16, SI = BI / WI / 16;
  constexpr int QJ = (BJ * 8 + kLlThreads - 1) / kLlThreads;
  constexpr int QI = (BI * 8 + kLlThreads - 1) / kLlThreads;
  static_assert(SJ >= 1 && SI >= 1, "a wave needs a subtile");
  __shared__ uint4 s_j[BJ * 8], s_i[BI * 8];
  const int64_t blk = leaf_block();
  if (blk >= a.tiles) return;
  const int tid = threadIdx.x, l = lane_id(), w = tid / kWave;
  const int wj = w / WI * (SJ * 16), wi = w % WI * (SI * 16);
  const int64_t slot = blk / a.col_tiles;
  const int i0 = (int)(blk % a.col_tiles) * BI;
  const int g = leaf_find_group(a.off, a.G + 1, a.bj_shift, slot);
  const int64_t m0 = a.off[g] + ((slot - ((a.off[g] >> a.bj_shift) + (int64_t)g)) << a.bj_shift);
  const int64_t m1 = a.off[g + 1];
  if (m0 >= m1) return;
  const int rows = (int)min<int64_t>(BJ, m1 - m0);
  T* const out = (T*)a.out;
  const bool vec = a.cols % 4 == 0 && (uintptr_t)a.out % (4 * sizeof(T)) == 0;

  int32_t out_row[SJ];
#pragma unroll
  for (int j = 0; j < SJ; ++j) {
    const int r = wj + j * 16 + (l & 15);
    out_row[j] = r < rows ? a.order[m0 + r] : -1;
  }
  f32x4 acc[SJ][SI] = {};
  if (g < a.G) {
    const T* const src = (const T*)a.src;
    const T* const wg = (const T*)a.w + (int64_t)g * a.w_stride;
    const T* jp[QJ];
#pragma unroll
    for (int q = 0; q < QJ; ++q) {
      const int r = (q * kLlThreads + tid) >> 3;
      jp[q] = r < rows ? src + (int64_t)a.order[m0 + r] * a.src_stride : nullptr;
    }
    uint4 vj[QJ], vi[QI];
    auto load = [&](int k0) {
#pragma unroll
      for (int q = 0; q < QJ; ++q) {
        const int id = q * kLlThreads + tid, r = id >> 3;
        const int k = k0 + ((id & 7) ^ (r & 7)) * E;
        vj[q] = ll_chunk<T, kAligned>(jp[q] + k, jp[q] != nullptr ? a.depth - k : 0);
      }
#pragma unroll
      for (int q = 0; q < QI; ++q) {
        const int id = q * kLlThreads + tid;
        if constexpr (!kDx) {
          const int r = id >> 3;
          const int k = k0 + ((id & 7) ^ (r & 7)) * E;
          const bool in = BI * 8 % kLlThreads == 0 || r < BI;
          vi[q] = ll_chunk<T, kAligned>(wg + (int64_t)(i0 + r) * a.w_row + k,
                                        in && i0 + r < a.cols ? a.depth - k : 0);
        } else {
          constexpr int kRow = BI / E;
          const int k = id / kRow, c = id % kRow;
          const bool in = BI * 8 % kLlThreads == 0 || k < KD;
          vi[q] = ll_chunk<T, kAligned>(wg + (int64_t)(k0 + k) * a.w_row + i0 + c * E,
                                        in && k0 + k < a.depth ? a.cols - i0 - c * E : 0);
        }
      }
    };
    load(0);
    for (int k0 = 0; k0 < a.depth; k0 += KD) {
#pragma unroll
      for (int q = 0; q < QJ; ++q) {
        const int id = q * kLlThreads + tid;
        if (BJ * 8 % kLlThreads == 0 || id < BJ * 8) s_j[id] = vj[q];
      }
#pragma unroll
      for (int q = 0; q < QI; ++q) {
        const int id = q * kLlThreads + tid;
        if (BI * 8 % kLlThreads == 0 || id < BI * 8) {
          if constexpr (!kDx)
            s_i[id] = vi[q];
          else
            s_i[ll_turn_chunk<T, BI>(id / (BI / E), id % (BI / E))] = vi[q];
        }
      }
      __syncthreads();
      if (k0 + KD < a.depth) load(k0 + KD);
#pragma unroll
      for (int step = 0; step < 2; ++step) {
        uint4 fj[SJ], fi[SI];
#pragma unroll
        for (int j = 0; j < SJ; ++j) fj[j] = ll_frag_flat<T>(s_j, wj + j * 16, step);
#pragma unroll
        for (int i = 0; i < SI; ++i) {
          if constexpr (!kDx)
            fi[i] = ll_frag_flat<T>(s_i, wi + i * 16, step);
          else
            fi[i] = ll_frag_turn<T, BI>(s_i, wi + i * 16, step);
        }
#pragma unroll
        for (int j = 0; j < SJ; ++j)
#pragma unroll
          for (int i = 0; i < SI; ++i) acc[j][i] = ll_mma<T>(fi[i], fj[j], acc[j][i]);
      }
      __syncthreads();
    }
    if (a.bias != nullptr) {
      const T* const bg = (const T*)a.bias + (int64_t)g * a.cols;
#pragma unroll
      for (int i = 0; i < SI; ++i) {
        const int c = i0 + wi + i * 16 + 4 * (l >> 4);
        f32x4 b = {};
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (c + e < a.cols) b[e] = leaf_f32(bg[c + e]);
#pragma unroll
        for (int j = 0; j < SJ; ++j) acc[j][i] += b;
      }
    }
  }
#pragma unroll
  for (int j = 0; j < SJ; ++j) {
    if (out_row[j] < 0) continue;
    T* const o = out + (int64_t)out_row[j] * a.cols;
#pragma unroll
    for (int i = 0; i < SI; ++i) {
      const int c = i0 + wi + i * 16 + 4 * (l >> 4);
      ll_store4<T>(o + c, acc[j][i], a.cols - c, vec);
    }
  }
}

// ---- dW. A unit is a leaf with at most `run` rows (units below G), or a leaf's piece of a chunk of
// `run` sorted positions into a partial matrix (as in leaf_embed.hip: at most two pieces a chunk).
struct LlGrad {
  const void* x;
  const void* dy;
  void* dw;
  float* part;  // [2 * chunks][N][K]
  const int32_t* order;
  const uint32_t* keys;
  const int32_t* off;
  int64_t x_stride, dy_stride;
  int G, N, K, k_tiles, n_tiles;
  int64_t run, units;
};

// One BJ x BI tile (rows of W, columns of W) of one unit: both operands are gathered rows with the
// rows as depth, turned.
template <typename T, int BJ, int BI, int WJ, bool kAligned>
__global__ __launch_bounds__(kLlThreads) void ll_grad_kernel(LlGrad a) {
  constexpr int E = Ll<T>::kEpc, KD = Ll<T>::kDepth;
  constexpr int WI = kLlWaves / WJ;
  constexpr int SJ = BJ / WJ / 16, SI = BI / WI / 16;
  constexpr int QJ = (BJ * 8 + kLlThreads - 1) / kLlThreads;
  constexpr int QI = (BI * 8 + kLlThreads - 1) / kLlThreads;
  __shared__ uint4 s_j[BJ * 8], s_i[BI * 8];
  const int64_t blk = leaf_block();
  const int tiles = a.n_tiles * a.k_tiles;
  const int64_t unit = blk / tiles;
  if (unit >= a.units) return;
  const int t = (int)(blk % tiles);
  const int j0 = t / a.k_tiles * BJ, i0 = t % a.k_tiles * BI;
  const int tid = threadIdx.x, l = lane_id(), w = tid / kWave;
  const int wj = w / WI * (SJ * 16), wi = w % WI * (SI * 16);

  int64_t pa, pb;
  if (unit < a.G) {
    pa = a.off[unit], pb = a.off[unit + 1];
    if (pb - pa > a.run) return;
  } else {
    const int64_t c = (unit - a.G) >> 1, m = a.off[a.G];
    const int64_t ca = c * a.run, cb = min<int64_t>(ca + a.run, m);
    if (ca >= m) return;
    const int64_t k0 = a.keys[ca], k1 = a.keys[cb - 1];
    if (((unit - a.G) & 1) == 0) {
      if (a.off[k0 + 1] - a.off[k0] <= a.run) return;
      pa = ca, pb = min<int64_t>(cb, a.off[k0 + 1]);
    } else {
      if (k1 == k0 || a.off[k1 + 1] - a.off[k1] <= a.run) return;
      pa = a.off[k1], pb = cb;
    }
  }

  f32x4 acc[SJ][SI] = {};
  const T* const x = (const T*)a.x;
  const T* const dy = (const T*)a.dy;
  uint4 vj[QJ], vi[QI];
  auto load = [&](int64_t p0) {
#pragma unroll
    for (int q = 0; q < QJ; ++q) {
      constexpr int kRow = BJ / E;
      const int id = q * kLlThreads + tid, k = id / kRow, c = id % kRow;
      const bool in = (BJ * 8 % kLlThreads == 0 || k < KD) && p0 + k < pb;
      const int64_t row = in ? a.order[p0 + k] : 0;
      vj[q] = ll_chunk<T, kAligned>(dy + row * a.dy_stride + j0 + c * E,
                                    in ? a.N - j0 - c * E : 0);
    }
#pragma unroll
    for (int q = 0; q < QI; ++q) {
      constexpr int kRow = BI / E;
      const int id = q * kLlThreads + tid, k = id / kRow, c = id % kRow;
      const bool in = (BI * 8 % kLlThreads == 0 || k < KD) && p0 + k < pb;
      const int64_t row = in ? a.order[p0 + k] : 0;
      vi[q] = ll_chunk<T, kAligned>(x + row * a.x_stride + i0 + c * E, in ? a.K - i0 - c * E : 0);
    }
  };
  if (pa < pb) load(pa);
  for (int64_t p0 = pa; p0 < pb; p0 += KD) {
#pragma unroll
    for (int q = 0; q < QJ; ++q) {
      const int id = q * kLlThreads + tid;
      if (BJ * 8 % kLlThreads == 0 || id < BJ * 8)
        s_j[ll_turn_chunk<T, BJ>(id / (BJ / E), id % (BJ / E))] = vj[q];
    }
#pragma unroll
    for (int q = 0; q < QI; ++q) {
      const int id = q * kLlThreads + tid;
      if (BI * 8 % kLlThreads == 0 || id < BI * 8)
        s_i[ll_turn_chunk<T, BI>(id / (BI / E), id % (BI / E))] = vi[q];
    }
    __syncthreads();
    if (p0 + KD < pb) load(p0 + KD);
#pragma unroll
    for (int step = 0; step < 2; ++step) {
      uint4 fj[SJ], fi[SI];
#pragma unroll
      for (int j = 0; j < SJ; ++j) fj[j] = ll_frag_turn<T, BJ>(s_j, wj + j * 16, step);
#pragma unroll
      for (int i = 0; i < SI; ++i) fi[i] = ll_frag_turn<T, BI>(s_i, wi + i * 16, step);
#pragma unroll
      for (int j = 0; j < SJ; ++j)
#pragma unroll
        for (int i = 0; i < SI; ++i) acc[j][i] = ll_mma<T>(fi[i], fj[j], acc[j][i]);
    }
    __syncthreads();
  }

  const bool whole = unit < a.G;
  const bool vec = a.K % 4 == 0 && (uintptr_t)a.dw % (4 * sizeof(T)) == 0;
#pragma unroll
  for (int j = 0; j < SJ; ++j) {
    const int r = j0 + wj + j * 16 + (l & 15);
    if (r >= a.N) continue;
#pragma unroll
    for (int i = 0; i < SI; ++i) {
      const int c = i0 + wi + i * 16 + 4 * (l >> 4);
      if (whole)
        ll_store4<T>((T*)a.dw + ((int64_t)unit * a.N + r) * a.K + c, acc[j][i], a.K - c, vec);
      else
        ll_store4<float>(a.part + ((unit - a.G) * a.N + r) * a.K + c, acc[j][i], a.K - c,
                         a.K % 4 == 0);
    }
  }
}

// Adds the partial matrices of the leaves with more than `run` rows: one block per chunk in which
// such a leaf starts and per kLlThreads elements, in 64 bits for f32.
template <typename T>
__global__ __launch_bounds__(kLlThreads) void ll_join_kernel(LlGrad a, int64_t blocks_per_chunk,
                                                             int64_t chunks) {
  using A = std::conditional_t<sizeof(T) == 4, double, float>;
  const int64_t blk = leaf_block();
  const int64_t c = blk / blocks_per_chunk, m = a.off[a.G];
  const int64_t ca = c * a.run, cb = min<int64_t>(ca + a.run, m);
  if (c >= chunks || ca >= m) return;
  const int64_t k0 = a.keys[ca], k1 = a.keys[cb - 1];
  const int64_t s1 = a.off[k1], e1 = a.off[k1 + 1];
  if (s1 < ca || e1 - s1 <= a.run) return;
  const int64_t size = (int64_t)a.N * a.K;
  const int64_t e = (blk % blocks_per_chunk) * kLlThreads + threadIdx.x;
  if (e >= size) return;
  const int64_t last = (e1 - 1) / a.run;
  A sum = 0;
  for (int64_t p = c; p <= last; ++p)
    sum += (A)a.part[(2 * p + (p == c && k1 != k0 ? 1 : 0)) * size + e];
  ((T*)a.dw)[k1 * size + e] = leaf_from<T>((float)sum);
}

// ---- forward of at most 64 rows, straight from the leaf indices (no route). Each wave holds all of
// them, one a lane. Block (column tile, row i): row i leads the tile of up to 16 rows of its leaf
// that start with it; rows that follow another row of their leaf inside its 16 leave. So a leaf's
// matrix is read once for 16 rows. The waves split the depth, from memory straight into fragments,
// and their sums meet in LDS.
struct LlSmall {
  const void* x;
  const void* ids;
  const void* w;
  const void* bias;
  void* y;
  int64_t x_stride;
  int n, G, K, N, col_tiles;
  bool wide;
};

template <typename T, bool kAligned>
__global__ __launch_bounds__(kLlThreads) void ll_small_kernel(LlSmall a) {
  constexpr int E = Ll<T>::kEpc, kStep = 4 * E, kUnroll = 4;
  __shared__ f32x4 s_acc[kLlWaves][kWave];
  const int l = lane_id(), w = threadIdx.x / kWave;
  const int i = blockIdx.x / a.col_tiles, c0 = (blockIdx.x % a.col_tiles) * 16;
  int64_t id = -1;
  if (l < a.n) id = a.wide ? ((const int64_t*)a.ids)[l] : (int64_t)((const int32_t*)a.ids)[l];
  const int key = (uint64_t)id < (uint64_t)a.G ? (int)id : -1;
  const int g = __builtin_amdgcn_readlane(key, i);
  T* const y = (T*)a.y;
  if (g < 0) {
    const int c = c0 + (int)threadIdx.x;
    if (threadIdx.x < 16 && c < a.N) y[(int64_t)i * a.N + c] = leaf_from<T>(0.f);
    return;
  }
  unsigned long long same = __ballot(key == g);
  const unsigned long long before = (1ull << i) - 1ull;
  if (__popcll(same & before) & 15) return;
  same &= ~before;
  for (int j = 0; j < (l & 15); ++j) same &= same - 1;  // the (l % 16)-th row from i on
  const int row = same ? __ffsll((long long)same) - 1 : -1;

  const T* const xr = (const T*)a.x + (int64_t)max(row, 0) * a.x_stride;
  const int col = c0 + (l & 15);
  const T* const wr = (const T*)a.w + ((int64_t)g * a.N + min(col, a.N - 1)) * a.K;
  const int steps = (a.K + kStep - 1) / kStep;
  const int per = (steps + kLlWaves - 1) / kLlWaves;
  const int s0 = w * per, s1 = min(steps, s0 + per);
  f32x4 acc = {};
  for (int s = s0; s < s1; s += kUnroll) {
    uint4 fw[kUnroll], fx[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int k = (s + u) * kStep + (l >> 4) * E;
      const int left = s + u < s1 ? a.K - k : 0;
      fw[u] = ll_chunk<T, kAligned>(wr + k, col < a.N ? left : 0);
      fx[u] = ll_chunk<T, kAligned>(xr + k, row >= 0 ? left : 0);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) acc = ll_mma<T>(fw[u], fx[u], acc);
  }
  s_acc[w][l] = acc;
  __syncthreads();
  if (w > 0) return;
#pragma unroll
  for (int q = 1; q < kLlWaves; ++q) acc += s_acc[q][l];
  const int c = c0 + 4 * (l >> 4);
  if (row < 0 || c >= a.N) return;
  if (a.bias != nullptr) {
    const T* const bg = (const T*)a.bias + (int64_t)g * a.N;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (c + e < a.N) acc[e] += leaf_f32(bg[c + e]);
  }
  const bool vec = a.N % 4 == 0 && (uintptr_t)a.y % (4 * sizeof(T)) == 0;
  ll_store4<T>(y + (int64_t)row * a.N + c, acc, a.N - c, vec);
}

// ---------------------------------------------------------------------------- launches
template <typename T>
static bool ll_aligned(std::initializer_list<const void*> ptrs,
                       std::initializer_list<int64_t> sizes) {
  for (const void* p : ptrs)
    if ((uintptr_t)p % 16) return false;
  for (int64_t s : sizes)
    if (s % Ll<T>::kEpc) return false;
  return true;
}

template <typename F>
static void ll_dispatch_type(int type, F f) {
  if (type == kLeafF32)
    f(float{});
  else if (type == kLeafF16)
    f(f16_t{});
  else
    f(bf16_t{});
}

int leaf_linear_small_rows() { return kLlSmallRows; }

void launch_leaf_linear_small(hipStream_t s, int type, const void* x, int64_t x_stride,
                              const void* ids, bool wide, int n, int G, const void* w,
                              const void* bias, int K, int N, void* y) {
  if (n <= 0) return;
  LlSmall a{x, ids, w, bias, y, x_stride, n, G, K, N, (N + 15) / 16, wide};
  if (n > kLlSmallRows || (int64_t)a.col_tiles * n > (1 << 22))
    throw std::runtime_error("leaf_linear: too large for the small form");
  ll_dispatch_type(type, [&](auto t) {
    using T = decltype(t);
    auto go = [&](auto kern) {
      hipLaunchKernelGGL(kern, dim3(a.col_tiles * n), dim3(kLlThreads), 0, s, a);
      MT_HIP_CHECK(hipGetLastError());
    };
    ll_aligned<T>({x, w}, {K, x_stride}) ? go(ll_small_kernel<T, true>)
                                        : go(ll_small_kernel<T, false>);
  });
}

// forward (dx false: src = x, depth = K, cols = N) or dx (src = dy, depth = N, cols = K)
void launch_leaf_linear_tile(hipStream_t s, int type, bool dx, const void* src, int64_t src_stride,
                             const int32_t* order, const int32_t* off, int64_t n, int G,
                             const void* w, const void* bias, int K, int N, void* out) {
  if (n <= 0) return;
  LlTile a{};
  a.src = src, a.w = w, a.bias = bias, a.out = out, a.order = order, a.off = off;
  a.src_stride = src_stride, a.w_stride = (int64_t)N * K;
  a.G = G, a.depth = dx ? N : K, a.cols = dx ? K : N, a.w_row = K;
  ll_dispatch_type(type, [&](auto t) {
    using T = decltype(t);
    const bool al = ll_aligned<T>({src, w}, {K, src_stride, dx ? N : K});
    auto go = [&](auto bj, auto bi, auto wj) {
      a.bj_shift = __builtin_ctz((unsigned)bj());
      a.col_tiles = (a.cols + bi() - 1) / bi();
      a.tiles = ((n >> a.bj_shift) + G + 1) * a.col_tiles;
      const dim3 grid = leaf_grid(a.tiles);
      auto run = [&](auto kern) {
        hipLaunchKernelGGL(kern, grid, dim3(kLlThreads), 0, s, a);
        MT_HIP_CHECK(hipGetLastError());
      };
      if (dx)
        al ? run(ll_tile_kernel<T, true, bj(), bi(), wj(), true>)
           : run(ll_tile_kernel<T, true, bj(), bi(), wj(), false>);
      else
        al ? run(ll_tile_kernel<T, false, bj(), bi(), wj(), true>)
           : run(ll_tile_kernel<T, false, bj(), bi(), wj(), false>);
    };
    using std::integral_constant;
    using c1 = integral_constant<int, 1>;
    using c2 = integral_constant<int, 2>;
    using c4 = integral_constant<int, 4>;
    using c16 = integral_constant<int, 16>;
    using c64 = integral_constant<int, 64>;
    using c128 = integral_constant<int, 128>;
    const int64_t mean = n / G;
    if (a.cols <= 16)
      go(c64{}, c16{}, c4{});
    else if (mean < 32)
      go(c16{}, c64{}, c1{});
    else if (mean < 128 || a.cols <= 64)
      go(c64{}, c64{}, c2{});
    else
      go(c128{}, c128{}, c2{});
  });
}

// rows a dW unit may have: a power of two, small enough that about 1024 tiles run at once
static int64_t ll_grad_run(int64_t n, int64_t tiles) {
  int64_t run = 256;
  while (run < (1 << 20) && n / run * tiles > 2048) run <<= 1;
  return run;
}
static int ll_grad_tile(int N, int K) { return N > 64 && K > 64 ? 128 : 64; }
static int64_t ll_grad_tiles(int N, int K) {
  const int b = ll_grad_tile(N, K);
  return (int64_t)((N + b - 1) / b) * ((K + b - 1) / b);
}

int64_t leaf_linear_grad_bytes(int64_t n, int K, int N) {
  const int64_t run = ll_grad_run(n, ll_grad_tiles(N, K));
  if (n <= run) return 0;
  return 2 * ((n + run - 1) / run) * (int64_t)N * K * 4;
}

void launch_leaf_linear_grad(hipStream_t s, int type, const void* x, int64_t x_stride,
                             const void* dy, int64_t dy_stride, const int32_t* order,
                             const uint32_t* keys, const int32_t* off, int64_t n, int G, int K,
                             int N, void* dw, void* work) {
  LlGrad a{};
  a.x = x, a.dy = dy, a.dw = dw, a.part = (float*)work;
  a.order = order, a.keys = keys, a.off = off;
  a.x_stride = x_stride, a.dy_stride = dy_stride;
  a.G = G, a.N = N, a.K = K;
  const int64_t tiles = ll_grad_tiles(N, K);
  a.run = ll_grad_run(n, tiles);
  const int64_t chunks = n > a.run ? (n + a.run - 1) / a.run : 0;
  a.units = G + 2 * chunks;
  ll_dispatch_type(type, [&](auto t) {
    using T = decltype(t);
    const bool al = ll_aligned<T>({x, dy}, {K, N, x_stride, dy_stride});
    auto go = [&](auto b) {
      a.n_tiles = (N + b() - 1) / b(), a.k_tiles = (K + b() - 1) / b();
      const dim3 grid = leaf_grid(a.units * tiles);
      auto run = [&](auto kern) {
        hipLaunchKernelGGL(kern, grid, dim3(kLlThreads), 0, s, a);
        MT_HIP_CHECK(hipGetLastError());
      };
      al ? run(ll_grad_kernel<T, b(), b(), 2, true>) : run(ll_grad_kernel<T, b(), b(), 2, false>);
    };
    if (ll_grad_tile(N, K) == 128)
      go(std::integral_constant<int, 128>{});
    else
      go(std::integral_constant<int, 64>{});
    if (chunks > 0) {
      const int64_t per = ((int64_t)N * K + kLlThreads - 1) / kLlThreads;
      hipLaunchKernelGGL(ll_join_kernel<T>, leaf_grid(chunks * per), dim3(kLlThreads), 0, s, a, per,
                         chunks);
      MT_HIP_CHECK(hipGetLastError());
    }
  });
}

}  // namespace mt
