// Products grouped by leaf: y[i] = W[g] x[i] + b[g] for the leaf g of row i, and the gradients
//   dx[i] = W[g]^T dy[i],   dW[g] = sum over g's rows of dy[i] x[i]^T,
// and db[g], the sum of dy over g's rows, which comes from the same tiles of dy as dW; without dW,
// and beside its largest tiles, it is the embedding's gradient (leaf_embed.hip).
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

int64_t leaf_embed_grad_bytes(int, int64_t, int);
void launch_leaf_embed_grad(hipStream_t, int, const void*, int64_t, const int32_t*, const uint32_t*,
                            const int32_t*, int64_t, int64_t, int, float, void*, void*);

constexpr int kLlThreads = 256;
constexpr int kLlWaves = kLlThreads / kWave;
// Rows of the form without a route, one a lane. us so / by tiles with a kept route / and with the
// sort, 2048 -> 1024 bf16: 64 rows of 64 leaves 36 / 45 / 49, of one 13 / 29 / 35; 4 rows 6 / 18 /
// 24.
constexpr int kLlSmallRows = 64;
constexpr int kLlBigRows = 256;  // rows a leaf on average from which on 256-row tiles are taken

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

// What a lane adds to a fragment's address, once for all fragments: the swizzles depend on the lane
// alone, so the rest of an address is an immediate (turned tiles: and the slab).
template <typename T>
struct LlLane {
  int flat[2];  // chunk index inside 16 rows of a flat tile, by step
  int turn_k;   // first depth row of a turned tile
  int turn_c;   // element inside the slab
  int turn_f;   // the slab's swizzle
  __device__ __forceinline__ LlLane() {
    const int l = lane_id();
    flat[0] = ll_flat_chunk<T>(l & 15, l >> 4);
    flat[1] = ll_flat_chunk<T>(l & 15, 4 + (l >> 4));
    if constexpr (sizeof(T) == 4) {
      turn_k = 4 * (l >> 4), turn_c = l & 15;
    } else {
      turn_k = 8 * (l >> 4) + ((l & 15) >> 2), turn_c = (l & 3) * 4;
    }
    turn_f = ll_turn_slab<T, 1024>(turn_k, 0);
  }
};

// fragment (row r0 + l % 16, chunk 4 * step + l / 16) of a flat tile
template <typename T>
__device__ __forceinline__ uint4 ll_frag_flat(const uint4* s, const LlLane<T>& ln, int r0,
                                              int step) {
  return s[r0 * 8 + ln.flat[step]];
}

// the same fragment of a turned tile: column 16 slab + l % 16, depth (4 * step + l / 16) * kEpc on
template <typename T, int COLS>
__device__ __forceinline__ uint4 ll_frag_turn(const uint4* s, const LlLane<T>& ln, int slab,
                                              int step) {
  const int at = ln.turn_k * COLS + ln.turn_c + (slab ^ (ln.turn_f & (COLS / 16 - 1))) * 16;
  uint4 v;
  if constexpr (sizeof(T) == 4) {
    const float* f = (const float*)s + at + 16 * step * COLS;
    uint32_t* e = (uint32_t*)&v;
#pragma unroll
    for (int u = 0; u < 4; ++u) e[u] = __float_as_uint(f[u * COLS]);
  } else {
    // ds_read_b64_tr_b16: 16 lanes read 4 rows of 16 columns, 8 bytes each, and lane i of them
    // gets column i of the 4 rows
    const uint16_t* h = (const uint16_t*)s + at + 32 * step * COLS;
    s16x4 part[2];
#pragma unroll
    for (int u = 0; u < 2; ++u)
      part[u] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (__attribute__((address_space(3))) s16x4*)(h + 4 * u * COLS));
    __builtin_memcpy(&v, &part[0], 8);
    __builtin_memcpy((char*)&v + 8, &part[1], 8);
  }
  return v;
}

// four neighbouring columns of one output row, `left` of them inside. kVec: rows are so aligned
// that all four are inside, or none, and one store takes them.
template <bool kVec, typename T>
__device__ __forceinline__ void ll_store4(T* p, f32x4 v, int left) {
  if constexpr (kVec) {
    LeafVec<T, 4> o;
#pragma unroll
    for (int e = 0; e < 4; ++e) o.v[e] = leaf_from<T>(v[e]);
    if (left > 0) *(LeafVec<T, 4>*)p = o;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < left) p[e] = leaf_from<T>(v[e]);
  }
}

// 16 bytes a lane from memory straight into LDS: lane l's chunk lands at lds[l] (lds: one address
// for the wave).
__device__ __forceinline__ void ll_dma(const void* g, void* lds) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)g,
                                   (__attribute__((address_space(3))) void*)lds, 16, 0, 0);
}
// The same through a buffer descriptor, address = base + lane_off + off. In assembly, because the
// compiler orders every later LDS read behind the builtin's writes: ll_dma_wait orders them.
typedef int i32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ i32x4 ll_rsrc(const void* base) {
  const uint64_t p = (uint64_t)base;
  return i32x4{(int)(uint32_t)p, (int)(uint32_t)(p >> 32), -1, 0x00027000};
}
__device__ __forceinline__ void ll_dma_buffer(i32x4 rsrc, uint32_t lane_off, uint32_t off,
                                              const void* lds) {
  const uint32_t to = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)lds;
  asm volatile(
      "s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
      :
      : "s"(to), "v"(lane_off), "s"(rsrc), "s"(off)
      : "memory", "m0");
}
// ... from any address of a lane
__device__ __forceinline__ void ll_dma_at(const void* g, const void* lds) {
  const uint32_t to = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)lds;
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
               :
               : "s"(to), "v"(g)
               : "memory", "m0");
}
// Every fetch of this wave has landed, and every wave has come here. (__syncthreads() does not do:
// it waits for a wave's own reads and writes of LDS, not for its fetches into LDS.)
__device__ __forceinline__ void ll_dma_wait() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}
// what the chunks behind the end of the depth are read from
__device__ const uint4 kLlZeros[1] = {};

// *p, or zeros, read either way; from the global address space, which a choice of two plain
// pointers would leave
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
template <typename V>
__device__ __forceinline__ V ll_load_or_zeros(bool there, const void* p) {
  using U = std::conditional_t<sizeof(V) == 16, u32x4,
                               std::conditional_t<sizeof(V) == 4, uint32_t, uint16_t>>;
  const U u = *(const __attribute__((address_space(1))) U*)(there ? (uintptr_t)p
                                                                  : (uintptr_t)kLlZeros);
  return __builtin_bit_cast(V, u);
}

// Blocks go to the 8 XCDs in turn, and each XCD has its own L2: runs of kLlXcdRun tiles stay on one
// XCD, so that neighbours share the panels they read; runs go round, so that a stretch of tiles
// without rows does not leave an XCD idle. us with runs of 4 / 32 / 128, bf16: 32768 rows, 32
// leaves, 2048 -> 4096 forward 656 / 656 / 776, dx 624 / 648 / 986, dW 702 / 717 / 826; 65536 rows,
// 64 leaves, 2048 -> 2048 652 / 645 / 769, 654 / 647 / 807, 715 / 797 / 834.
constexpr int kLlXcds = 8, kLlXcdRun = 32;
__device__ __forceinline__ int64_t ll_xcd_order(int64_t blk) {
  const int64_t i = blk / kLlXcds;
  return ((i / kLlXcdRun) * kLlXcds + blk % kLlXcds) * kLlXcdRun + i % kLlXcdRun;
}
static int64_t ll_xcd_blocks(int64_t tiles) {  // blocks that ll_xcd_order maps onto all tiles
  constexpr int64_t kRound = kLlXcds * kLlXcdRun;
  return (tiles + kRound - 1) / kRound * kRound;
}

struct LlTile {
  const void* src;  // x (forward) or dy (kDx): rows of `depth` elements
  const void* w;    // [G, N, K]
  const void* bias;
  void* out;  // y or dx: rows of `cols` elements
  const int32_t* order;
  const int32_t* off;
  int64_t src_stride, w_stride;  // elements between src rows; between leaves' matrices
  int G, depth, cols, w_row;     // w_row: elements of a row of W (K, or more of a packed one)
  int col_tiles, bj_shift;
  int64_t tiles;              // a bound
  const int2* plan;           // the tiles' leaves and positions, or null: found through off
  const int32_t* plan_count;  // how many there are
};

// The tiles of kBig rows in order of their leaves, {leaf, first sorted position}, and how many
// there are: with many column tiles, tiles without rows between them would keep neighbours from
// sharing what they read. One workgroup; a leaf has at least kLlBigRows rows on average here.
constexpr int kLlPlanThreads = 1024;
__global__ __launch_bounds__(kLlPlanThreads) void ll_plan_kernel(const int32_t* __restrict__ off,
                                                                 int G, int bj_shift,
                                                                 int2* __restrict__ plan,
                                                                 int32_t* __restrict__ count) {
  __shared__ uint32_t s_w[kLlPlanThreads / kWave];
  const int w = threadIdx.x / kWave, lane = lane_id();
  uint32_t before = 0;
  for (int g0 = 0; g0 <= G; g0 += kLlPlanThreads) {
    const int g = g0 + threadIdx.x;
    const int a = g <= G ? off[g] : 0, b = g <= G ? off[g + 1] : 0;
    const uint32_t mine = (uint32_t)(((int64_t)b - a + (1 << bj_shift) - 1) >> bj_shift);
    const uint32_t incl = wave_incl_scan_u32(mine);
    if (lane == kWave - 1) s_w[w] = incl;
    __syncthreads();
    uint32_t at = before, all = 0;
    for (int q = 0; q < kLlPlanThreads / kWave; ++q) {
      at += q < w ? s_w[q] : 0u;
      all += s_w[q];
    }
    at += incl - mine;
    for (uint32_t k = 0; k < mine; ++k) plan[at + k] = make_int2(g, a + (int)(k << bj_shift));
    before += all;
    __syncthreads();
  }
  if (threadIdx.x == 0) *count = (int32_t)before;
}

// which rows and columns a tile is
struct LlPlace {
  int g, i0, rows;  // leaf (G: the rows without one), first column, rows (<= 0: no such tile)
  int64_t m0;       // first sorted position
};
__device__ __forceinline__ LlPlace ll_place(const LlTile& a, int64_t blk, int bi) {
  // bands of 8 column tiles: neighbours share rows of src and panels of W alike
  LlPlace at;
  at.rows = 0;
  const int64_t slots = a.plan != nullptr ? *a.plan_count : a.tiles / a.col_tiles;
  const int band = (int)(blk / (slots * 8));
  const int wide = min(8, a.col_tiles - band * 8);
  if (wide <= 0) return at;
  const int64_t in_band = blk - (int64_t)band * slots * 8;
  const int64_t slot = in_band / wide;
  if (slot >= slots) return at;  // (the list may be shorter than the bound that was launched)
  at.i0 = (band * 8 + (int)(in_band % wide)) * bi;
  if (a.plan != nullptr) {
    const int2 p = a.plan[slot];
    at.g = p.x, at.m0 = p.y;
  } else {
    at.g = leaf_find_group(a.off, a.G + 1, a.bj_shift, slot);
    const int64_t first = a.off[at.g];
    at.m0 = first + ((slot - ((first >> a.bj_shift) + (int64_t)at.g)) << a.bj_shift);
  }
  at.rows = (int)max<int64_t>(-1, min<int64_t>(1 << a.bj_shift, a.off[at.g + 1] - at.m0));
  return at;
}

// acc[j][i] holds row kStep j + l % 16 and columns 16 i + 4 (l / 16) .. + 3 of the wave's part
template <typename T, int SJ, int SI>
__device__ __forceinline__ void ll_add_bias(f32x4 (&acc)[SJ][SI], const LlTile& a, int g, int c0) {
  if (a.bias == nullptr) return;
  const T* const bg = (const T*)a.bias + (int64_t)g * a.cols;
#pragma unroll
  for (int i = 0; i < SI; ++i) {
    const int c = c0 + i * 16 + 4 * (lane_id() >> 4);
    f32x4 b = {};
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (c + e < a.cols) b[e] = leaf_f32(bg[c + e]);
#pragma unroll
    for (int j = 0; j < SJ; ++j) acc[j][i] += b;
  }
}

template <typename T, int kStep, int SJ, int SI>
__device__ __forceinline__ void ll_store_rows(const f32x4 (&acc)[SJ][SI], const LlTile& a,
                                              const LlPlace& at, int wj, int wi) {
  const int l = lane_id();
  auto store = [&](auto kvec) {
#pragma unroll
    for (int j = 0; j < SJ; ++j) {
      const int r = wj + j * kStep + (l & 15);
      if (r >= at.rows) continue;
      T* const o = (T*)a.out + (int64_t)a.order[at.m0 + r] * a.cols;
#pragma unroll
      for (int i = 0; i < SI; ++i) {
        const int c = at.i0 + wi + i * 16 + 4 * (l >> 4);
        ll_store4<kvec()>(o + c, acc[j][i], a.cols - c);
      }
    }
  };
  const bool vec = a.cols % 4 == 0 && (uintptr_t)a.out % (4 * sizeof(T)) == 0;
  vec ? store(std::true_type{}) : store(std::false_type{});
}

// One tile of BJ rows of one leaf by BI output columns, NW waves, WJ of them along the rows.
// Forward: A = W's rows, flat; kDx: A = W with its rows as depth, turned. B = gathered rows of src,
// flat. Rows past the leaf's last and columns past the last repeat the last one: their products
// are not stored. Depth past the end is zeros in both operands.
//
// kAligned: the next tile of depth goes from memory straight into the LDS buffer that is not read;
// one barrier a tile. Otherwise chunks go through registers, whose loads wait until the tile's
// products are issued. One tile of depth is on its way at a time, about 1.1 us each, which bounds
// short depths: 10007 rows in 12 leaves, 1000 -> 600 f16 27 us (445 TFLOP/s), 4096 -> 1280 169 us
// (620). f32 is bound by its products: 65536 rows in 64 leaves, 1024 -> 1024 forward 1209 us, dx
// 1216 us (113 TFLOP/s; one library product of that size 142).
template <typename T, bool kDx, int BJ, int BI, int WJ, int NW, bool kAligned>
__global__ __launch_bounds__(NW* kWave) void ll_tile_kernel(LlTile a) {
  constexpr int E = Ll<T>::kEpc, KD = Ll<T>::kDepth, NT = NW * kWave;
  constexpr int WI = NW / WJ;
  constexpr int SJ = BJ / WJ / 16, SI = BI / WI / 16;
  constexpr int QJ = (BJ * 8 + NT - 1) / NT;
  constexpr int QI = (BI * 8 + NT - 1) / NT;
  static_assert(SJ >= 1 && SI >= 1, "a wave needs a subtile");
  __shared__ uint4 s_j0[BJ * 8], s_i0[BI * 8];
  __shared__ uint4 s_j1[kAligned ? BJ * 8 : 1], s_i1[kAligned ? BI * 8 : 1];
  const int64_t blk = ll_xcd_order(leaf_block());
  if (blk >= a.tiles) return;
  const int tid = threadIdx.x, l = lane_id(), w = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int wj = w / WI * (SJ * 16), wi = w % WI * (SI * 16);
  const LlPlace at = ll_place(a, blk, BI);
  if (at.rows <= 0) return;
  const int rows = at.rows, i0 = at.i0, g = at.g;
  f32x4 acc[SJ][SI] = {};
  const LlLane<T> ln;
  if (g < a.G) {
    const T* const src = (const T*)a.src;
    const T* const wg = (const T*)a.w + (int64_t)g * a.w_stride;
    const T* jp[QJ];
#pragma unroll
    for (int q = 0; q < QJ; ++q) {
      const int r = (q * NT + tid) >> 3;
      jp[q] = src + (int64_t)a.order[at.m0 + min(r, rows - 1)] * a.src_stride;
    }
    auto products = [&](const uint4* sj, const uint4* si) {
      if (wj >= rows) return;
#pragma unroll
      for (int step = 0; step < 2; ++step) {
        uint4 fj[SJ], fi[SI];
#pragma unroll
        for (int j = 0; j < SJ; ++j) fj[j] = ll_frag_flat<T>(sj, ln, wj + j * 16, step);
#pragma unroll
        for (int i = 0; i < SI; ++i) {
          if constexpr (!kDx)
            fi[i] = ll_frag_flat<T>(si, ln, wi + i * 16, step);
          else
            fi[i] = ll_frag_turn<T, BI>(si, ln, wi / 16 + i, step);
        }
#pragma unroll
        for (int j = 0; j < SJ; ++j)
#pragma unroll
          for (int i = 0; i < SI; ++i) acc[j][i] = ll_mma<T>(fi[i], fj[j], acc[j][i]);
      }
    };
    if constexpr (kAligned) {
      auto load = [&](uint4* sj, uint4* si, int k0) {
#pragma unroll
        for (int q = 0; q < QJ; ++q) {
          const int id = q * NT + tid, r = id >> 3;
          if (BJ * 8 % NT != 0 && q * NT + w * kWave >= BJ * 8) break;
          const int k = k0 + ((id & 7) ^ (r & 7)) * E;
          const void* p = jp[q] + k;
          if (k >= a.depth) p = kLlZeros;
          ll_dma(p, sj + q * NT + w * kWave);
        }
#pragma unroll
        for (int q = 0; q < QI; ++q) {
          const int id = q * NT + tid;
          if (BI * 8 % NT != 0 && q * NT + w * kWave >= BI * 8) break;
          const void* p;
          if constexpr (!kDx) {
            const int r = id >> 3;
            const int k = k0 + ((id & 7) ^ (r & 7)) * E;
            p = wg + (int64_t)min(i0 + r, a.cols - 1) * a.w_row + k;
            if (k >= a.depth) p = kLlZeros;
          } else {
            constexpr int kRow = BI / E;
            const int k = id / kRow;
            const int c = ll_turn_chunk<T, BI>(k, id % kRow) - k * kRow;
            p = wg + (int64_t)(k0 + k) * a.w_row + min(i0 + c * E, a.w_row - E);
            if (k0 + k >= a.depth) p = kLlZeros;
          }
          ll_dma(p, si + q * NT + w * kWave);
        }
      };
      load(s_j0, s_i0, 0);
      for (int k0 = 0; k0 < a.depth; k0 += 2 * KD) {
        ll_dma_wait();
        if (k0 + KD < a.depth) load(s_j1, s_i1, k0 + KD);
        products(s_j0, s_i0);
        if (k0 + KD >= a.depth) break;
        ll_dma_wait();
        if (k0 + 2 * KD < a.depth) load(s_j0, s_i0, k0 + 2 * KD);
        products(s_j1, s_i1);
      }
    } else {
      uint4 vj[QJ], vi[QI];
      auto load = [&](int k0) {
#pragma unroll
        for (int q = 0; q < QJ; ++q) {
          const int id = q * NT + tid, r = id >> 3;
          const int k = k0 + ((id & 7) ^ (r & 7)) * E;
          vj[q] = ll_chunk<T, false>(jp[q] + k, a.depth - k);
        }
#pragma unroll
        for (int q = 0; q < QI; ++q) {
          const int id = q * NT + tid;
          if constexpr (!kDx) {
            const int r = id >> 3;
            const int k = k0 + ((id & 7) ^ (r & 7)) * E;
            vi[q] = ll_chunk<T, false>(wg + (int64_t)min(i0 + r, a.cols - 1) * a.w_row + k,
                                       a.depth - k);
          } else {
            constexpr int kRow = BI / E;
            const int k = id / kRow, c = id % kRow;
            const bool in = BI * 8 % NT == 0 || k < KD;
            vi[q] = ll_chunk<T, false>(wg + (int64_t)(k0 + k) * a.w_row + i0 + c * E,
                                       in && k0 + k < a.depth ? a.cols - i0 - c * E : 0);
          }
        }
      };
      load(0);
      for (int k0 = 0; k0 < a.depth; k0 += KD) {
#pragma unroll
        for (int q = 0; q < QJ; ++q) {
          const int id = q * NT + tid;
          if (BJ * 8 % NT == 0 || id < BJ * 8) s_j0[id] = vj[q];
        }
#pragma unroll
        for (int q = 0; q < QI; ++q) {
          const int id = q * NT + tid;
          if (BI * 8 % NT == 0 || id < BI * 8) {
            if constexpr (!kDx)
              s_i0[id] = vi[q];
            else
              s_i0[ll_turn_chunk<T, BI>(id / (BI / E), id % (BI / E))] = vi[q];
          }
        }
        __syncthreads();
        if (k0 + KD < a.depth) load(k0 + KD);
        products(s_j0, s_i0);
        __syncthreads();
      }
    }
    ll_add_bias<T, SJ, SI>(acc, a, g, i0 + wi);
  }
  ll_store_rows<T, 16, SJ, SI>(acc, a, at, wj, wi);
}

// ---- short rows: at most 256 bytes of depth, so a wave holds its columns of the leaf's matrix
// in registers and streams the leaf's rows past them, from memory straight into fragments, without
// LDS or barriers. A wave takes up to kRowsTile rows of one leaf and SI * 16 columns. Bound by
// memory latency and the f32 products: 1M rows, 64 -> 64 f32 in 4096 leaves 152 us (3.4 TB/s, 54 us
// of them products).
// Rows of a wave's tile; us with 64 / 128 / 256: that forward pass 171 / 153 / 211, its dx 186 /
// 170 / 161; 100k rows in 1500 leaves, 32 -> 1 f32 7.6 / 8.4 / 11.7; 500k rows in 2000 leaves,
// 64 -> 64 bf16 38.5 / 37.8 / 42.5.
constexpr int kRowsTile = 128, kRowsShift = 7;

template <typename T, bool kDx, int STEPS, int SI, bool kAligned>
__global__ __launch_bounds__(kLlThreads) void ll_rows_kernel(LlTile a) {
  constexpr int E = Ll<T>::kEpc;
  const int l = lane_id();
  const int64_t tile = leaf_block() * kLlWaves +
                       __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  if (tile >= a.tiles) return;
  const int64_t slot = tile / a.col_tiles;
  const int i0 = (int)(tile % a.col_tiles) * SI * 16;
  const int g = leaf_find_group(a.off, a.G + 1, kRowsShift, slot);
  const int64_t first = a.off[g];
  const int64_t m0 = first + ((slot - ((first >> kRowsShift) + (int64_t)g)) << kRowsShift);
  const int rows = (int)max<int64_t>(-1, min<int64_t>(kRowsTile, a.off[g + 1] - m0));
  if (rows <= 0) return;
  // 16 rows at a time; the row of this lane in the j-th 16 (past the last one: that one)
  constexpr int kOrd = kRowsTile / kWave;
  int32_t ord[kOrd];
#pragma unroll
  for (int i = 0; i < kOrd; ++i) ord[i] = a.order[m0 + min(i * kWave + l, rows - 1)];
  auto row_of = [&](int j) {
    int32_t o = ord[0];
#pragma unroll
    for (int i = 1; i < kOrd; ++i) o = j >= 4 * i ? ord[i] : o;
    return __shfl(o, ((16 * j) & (kWave - 1)) + (l & 15), kWave);
  };
  const bool vec = a.cols % 4 == 0 && (uintptr_t)a.out % (4 * sizeof(T)) == 0;
  const int c0 = i0 + 4 * (l >> 4);
  // whole: all 16 rows and all columns are there, and aligned
  auto store = [&](auto whole, int j, int32_t row, const f32x4 (&acc)[SI]) {
    T* const o = (T*)a.out + (int64_t)row * a.cols;
    if constexpr (whole()) {
#pragma unroll
      for (int i = 0; i < SI; ++i) ll_store4<true>(o + c0 + i * 16, acc[i], 4);
    } else {
      if (16 * j + (l & 15) >= rows) return;
#pragma unroll
      for (int i = 0; i < SI; ++i) {
        const int c = c0 + i * 16;
        ll_store4<false>(o + c, acc[i], a.cols - c);
      }
    }
  };
  constexpr std::true_type kYes{};
  constexpr std::false_type kNo{};
  if (g == a.G) {  // rows without a leaf
    const f32x4 zero[SI] = {};
    for (int j = 0; 16 * j < rows; ++j) store(kNo, j, row_of(j), zero);
    return;
  }
  const T* const src = (const T*)a.src;
  auto load = [&](int32_t row, uint4 (&f)[STEPS]) {
    const T* const p = src + row * a.src_stride;
#pragma unroll
    for (int t = 0; t < STEPS; ++t) {
      const int k = (4 * t + (l >> 4)) * E;
      if constexpr (kAligned)
        f[t] = ll_load_or_zeros<uint4>(k < a.depth, p + k);
      else
        f[t] = ll_chunk<T, false>(p + k, a.depth - k);
    }
  };
  uint4 f0[STEPS], f1[STEPS];
  load(row_of(0), f0);
  const T* const wg = (const T*)a.w + (int64_t)g * a.w_stride;
  uint4 fw[SI][STEPS];
#pragma unroll
  for (int i = 0; i < SI; ++i) {
    const int col = min(i0 + i * 16 + (l & 15), a.cols - 1);  // (past the last: not stored)
#pragma unroll
    for (int t = 0; t < STEPS; ++t) {
      const int k = (4 * t + (l >> 4)) * E;
      if constexpr (kDx) {
        T e[E];
#pragma unroll
        for (int u = 0; u < E; ++u) {
          e[u] = ll_load_or_zeros<T>(k + u < a.depth, wg + (int64_t)(k + u) * a.w_row + col);
        }
        __builtin_memcpy(&fw[i][t], e, 16);
      } else {
        const T* const p = wg + (int64_t)col * a.w_row + k;
        if constexpr (kAligned)
          fw[i][t] = ll_load_or_zeros<uint4>(k < a.depth, p);
        else
          fw[i][t] = ll_chunk<T, false>(p, a.depth - k);
      }
    }
  }
  f32x4 bias[SI] = {};
  if (a.bias != nullptr) {
    const T* const bg = (const T*)a.bias + (int64_t)g * a.cols;
#pragma unroll
    for (int i = 0; i < SI; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) bias[i][e] = leaf_f32(bg[min(c0 + i * 16 + e, a.cols - 1)]);
  }
  auto step = [&](auto whole, int j, const uint4 (&f)[STEPS], uint4 (&next)[STEPS]) {
    load(row_of(j + 1), next);
    f32x4 acc[SI];
#pragma unroll
    for (int i = 0; i < SI; ++i) acc[i] = bias[i];
#pragma unroll
    for (int t = 0; t < STEPS; ++t)
#pragma unroll
      for (int i = 0; i < SI; ++i) acc[i] = ll_mma<T>(fw[i][t], f[t], acc[i]);
    store(whole, j, row_of(j), acc);
  };
  int j = 0;
  if (vec && i0 + SI * 16 <= a.cols) {
    for (; 16 * (j + 2) <= rows; j += 2) {
      step(kYes, j, f0, f1);
      step(kYes, j + 1, f1, f0);
    }
  }
  for (; 16 * j < rows; j += 2) {
    step(kNo, j, f0, f1);
    if (16 * (j + 1) < rows) step(kNo, j + 1, f1, f0);
  }
}

// ---- 256 x 256 tiles of 16-bit types, where rows and columns fill them: 8 waves of 128 x 64.
//
// A tile of depth is multiplied in two halves. While one half is multiplied, the other's
// fragments are read -- past the barrier, those of the next tile -- each row fragment into the
// registers that the products have just left. The tile after next is fetched into the buffer that
// has been read: it has one tile's products to arrive. Operands are fetched through buffer
// descriptors: a lane's 32-bit offset is fixed and the depth is a scalar, so a fetch costs no
// vector arithmetic; an operand has to lie within 4 GiB for that.
// (Behind the last tile the same happens with zeros, which nothing uses.)
// One leaf, 8192 x 8192 x 8192 bf16: forward 1391, row gradient 1378, weight gradient 1157 TFLOP/s
// (the library's products of the same operands 1611, 1396, 1211);
// 1024 of depth take 23 us, a tile's start and end 12.
//
// A turned operand's depth rows lie in pairs, kPair bytes apart: 512 bytes a row and 32 to spare,
// and the odd row's slabs lie at s ^ 2. So the four rows that 16 lanes read at once, and those of
// the next 16 lanes, are in different banks, and a fragment's address is one of two lane constants
// plus an immediate.
constexpr int kBig = 256, kBigWaves = 8, kBigThreads = kBigWaves * kWave;
constexpr int kBigPair = 2 * 512 + 32;
constexpr int kBigFlatBytes = kBig * 128, kBigTurnBytes = 32 * kBigPair;
constexpr int kBigQ = kBig * 8 / kBigThreads;  // fetches of a thread per operand and tile

struct LlBigLane {
  int e[2];  // by the slab's bit 1
  __device__ __forceinline__ LlBigLane() {
    const int l = lane_id(), k = 8 * (l >> 4) + ((l & 15) >> 2), odd = k & 1;
    const int at = (k >> 1) * kBigPair + odd * 512 + (l & 3) * 8;
    e[0] = at + odd * 64, e[1] = at - odd * 64;
  }
};
// slab0: a multiple of 4, the same for the wave
__device__ __forceinline__ uint4 ll_big_turn(const char* s, const LlBigLane& ln, int slab0, int i,
                                             int step) {
  s16x4 part[2];
#pragma unroll
  for (int u = 0; u < 2; ++u)
    part[u] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) s16x4*)(s + ln.e[(i >> 1) & 1] + slab0 * 32 + i * 32 +
                                                   (16 * step + 2 * u) * kBigPair));
  uint4 v;
  __builtin_memcpy(&v, &part[0], 8);
  __builtin_memcpy((char*)&v + 8, &part[1], 8);
  return v;
}
// where fetch q of this wave lands, and which depth row (0..63) and column chunk this lane brings
__device__ __forceinline__ int ll_big_turn_to(int w, int q) {
  return (q * kBigWaves + w) * kBigPair;
}
__device__ __forceinline__ int ll_big_turn_row(int w, int q) {
  return 2 * (q * kBigWaves + w) + (lane_id() >> 5);
}
__device__ __forceinline__ int ll_big_turn_col() {
  const int l = lane_id();
  return (l & 31) ^ ((l >> 5) * 4);
}

template <typename T, bool kDx>
__global__ __launch_bounds__(kBigThreads, 2) void ll_big_kernel(LlTile a) {
  constexpr int E = Ll<T>::kEpc, KD = Ll<T>::kDepth;
  constexpr int SJ = 8, SI = 4;
  static_assert(sizeof(T) == 2, "the buffers' layout is for 16-bit types");
  constexpr int kBytes = kBigFlatBytes + (kDx ? kBigTurnBytes : kBigFlatBytes);
  __shared__ alignas(16) char s0[kBytes], s1[kBytes];  // rows, then columns
  const int64_t blk = ll_xcd_order(leaf_block());
  if (blk >= a.tiles) return;
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid / kWave);
  // rows of 16 go to the two halves of the waves in turn, so that a tile with fewer rows costs less
  const int wj = w / 4 * 16, wi = w % 4 * (SI * 16);
  const LlPlace at = ll_place(a, blk, kBig);
  if (at.rows <= 0) return;
  const int rows = at.rows, i0 = at.i0;
  f32x4 acc[SJ][SI] = {};
  if (at.g < a.G) {
    const LlLane<T> ln;
    const LlBigLane lt;
    const T* const src = (const T*)a.src;
    const T* const wg = (const T*)a.w + (int64_t)at.g * a.w_stride;
    const i32x4 src_rsrc = ll_rsrc(src), w_rsrc = ll_rsrc(wg);
    const int kc = ((tid & 7) ^ ((tid >> 3) & 7)) * E;  // a flat chunk's place in the depth
    uint32_t jo[kBigQ], wo[kBigQ];
#pragma unroll
    for (int q = 0; q < kBigQ; ++q) {
      const int r = (q * kBigThreads + tid) >> 3;
      jo[q] = (uint32_t)(a.order[at.m0 + min(r, rows - 1)] * a.src_stride + kc) * sizeof(T);
      if constexpr (!kDx)
        wo[q] = ((uint32_t)min(i0 + r, a.cols - 1) * a.w_row + kc) * sizeof(T);
      else
        wo[q] = ((uint32_t)ll_big_turn_row(w, q) * a.w_row +
                 min(i0 + ll_big_turn_col() * E, a.w_row - E)) * sizeof(T);
    }
    // tail: the tile may reach past the depth
    auto load = [&](auto tail, char* s, int k0) {
      const uint32_t ko = (uint32_t)k0 * sizeof(T);
      const uint32_t kw = kDx ? ko * a.w_row : ko;
#pragma unroll
      for (int q = 0; q < kBigQ; ++q) {
        char* const to = s + (q * kBigThreads + w * kWave) * 16;
        if constexpr (!tail())
          ll_dma_buffer(src_rsrc, jo[q], ko, to);
        else
          ll_dma_at(k0 + kc < a.depth ? (const char*)src + jo[q] + ko : (const char*)kLlZeros, to);
      }
#pragma unroll
      for (int q = 0; q < kBigQ; ++q) {
        char* const to = s + kBigFlatBytes +
                         (kDx ? ll_big_turn_to(w, q) : (q * kBigThreads + w * kWave) * 16);
        const int k = kDx ? ll_big_turn_row(w, q) : kc;
        if constexpr (!tail())
          ll_dma_buffer(w_rsrc, wo[q], kw, to);
        else
          ll_dma_at(k0 + k < a.depth ? (const char*)wg + wo[q] + kw : (const char*)kLlZeros, to);
      }
    };
    uint4 fj[SJ], fi0[SI], fi1[SI];
    auto read_j = [&](const char* s, int j, int step) {
      return ll_frag_flat<T>((const uint4*)s, ln, wj + j * 32, step);
    };
    auto read_i = [&](uint4 (&fi)[SI], const char* s, int step) {
#pragma unroll
      for (int i = 0; i < SI; ++i) {
        if constexpr (!kDx)
          fi[i] = ll_frag_flat<T>((const uint4*)(s + kBigFlatBytes), ln, wi + i * 16, step);
        else
          fi[i] = ll_big_turn(s + kBigFlatBytes, lt, wi / 16, i, step);
      }
    };
    const int nj = (rows - wj + 31) / 32;  // subtiles of this wave that hold rows (<= 0: none)
    // all: nj == SJ
    auto half = [&](auto all, const uint4 (&fi)[SI], uint4 (&fn)[SI], const char* next, int step) {
      read_i(fn, next, step);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int j = 0; j < SJ; ++j) {
        if (all() || j < nj) {
          __builtin_amdgcn_s_setprio(1);
#pragma unroll
          for (int i = 0; i < SI; ++i) acc[j][i] = ll_mma<T>(fi[i], fj[j], acc[j][i]);
          __builtin_amdgcn_s_setprio(0);
          fj[j] = read_j(next, j, step);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    auto pair = [&](auto all, auto tail, int k0) {
      half(all, fi0, fi1, s0, 1);
      ll_dma_wait();
      load(tail, s0, k0 + 2 * KD);
      half(all, fi1, fi0, s1, 0);
      half(all, fi0, fi1, s1, 1);
      ll_dma_wait();
      load(tail, s1, k0 + 3 * KD);
      half(all, fi1, fi0, s0, 0);
    };
    constexpr std::true_type kYes{};
    constexpr std::false_type kNo{};
    load(kYes, s0, 0);
    ll_dma_wait();
    load(kYes, s1, KD);
#pragma unroll
    for (int j = 0; j < SJ; ++j) fj[j] = read_j(s0, j, 0);
    read_i(fi0, s0, 0);
    int k0 = 0;
    if (nj == SJ) {
      for (; k0 + 4 * KD <= a.depth; k0 += 2 * KD) pair(kYes, kNo, k0);
    } else {
      for (; k0 + 4 * KD <= a.depth; k0 += 2 * KD) pair(kNo, kNo, k0);
    }
    for (; k0 < a.depth; k0 += 2 * KD) pair(kNo, kYes, k0);
    ll_dma_wait();  // (the fetches behind the last tile, before the workgroup's LDS goes)
    ll_add_bias<T, SJ, SI>(acc, a, at.g, i0 + wi);
  }
  ll_store_rows<T, 32, SJ, SI>(acc, a, at, wj, wi);
}

// ---- dW. A unit is a leaf with at most `run` rows (units below G), or a leaf's piece of a chunk
// of `run` sorted positions into a partial matrix (as in leaf_embed.hip: at most two pieces a
// chunk).
struct LlGrad {
  const void* x;
  const void* dy;
  void* dw;
  void* db;        // null: not made here
  const void* w;   // with dx: W
  void* dx;        // rows of K
  float* part;     // [2 * chunks][N][K]
  double* part_b;  // [2 * chunks][N]
  const int32_t* order;
  const uint32_t* keys;
  const int32_t* off;
  int64_t x_stride, dy_stride;
  int G, N, K, k_tiles, n_tiles;
  int n_row, k_row;  // elements of a row of dy and x: N and K, or more of packed ones
  int64_t run, units;
};

// the unit of the i-th blocks: pieces come first, so that no long one is left for the end
__device__ __forceinline__ int64_t ll_grad_unit(const LlGrad& a, int64_t i) {
  const int64_t pieces = a.units - a.G;
  return i < pieces ? a.G + i : i - pieces;
}

// sorted positions [pa, pb) of a unit; false: there is no such unit
__device__ __forceinline__ bool ll_grad_rows(const LlGrad& a, int64_t unit, int64_t& pa,
                                             int64_t& pb) {
  if (unit < a.G) {
    pa = a.off[unit], pb = a.off[unit + 1];
    return pb - pa <= a.run;
  }
  const int64_t c = (unit - a.G) >> 1, m = a.off[a.G];
  const int64_t ca = c * a.run, cb = min<int64_t>(ca + a.run, m);
  if (ca >= m) return false;
  const int64_t k0 = a.keys[ca], k1 = a.keys[cb - 1];
  if (((unit - a.G) & 1) == 0) {
    pa = ca, pb = min<int64_t>(cb, a.off[k0 + 1]);
    return a.off[k0 + 1] - a.off[k0] > a.run;
  }
  pa = a.off[k1], pb = cb;
  return k1 != k0 && a.off[k1 + 1] - a.off[k1] > a.run;
}

// acc[j][i] holds row 16 j + l % 16 and columns 16 i + 4 (l / 16) .. + 3 from (r0, c0) on
template <typename T, int SJ, int SI>
__device__ __forceinline__ void ll_grad_store(const f32x4 (&acc)[SJ][SI], const LlGrad& a,
                                              int64_t unit, int r0, int c0) {
  const int l = lane_id();
  auto store = [&](auto kvec, auto* to) {
#pragma unroll
    for (int j = 0; j < SJ; ++j) {
      const int r = r0 + j * 16 + (l & 15);
      if (r >= a.N) continue;
#pragma unroll
      for (int i = 0; i < SI; ++i) {
        const int c = c0 + i * 16 + 4 * (l >> 4);
        ll_store4<kvec()>(to + (int64_t)r * a.K + c, acc[j][i], a.K - c);
      }
    }
  };
  const bool vec = a.K % 4 == 0 && (uintptr_t)a.dw % (4 * sizeof(T)) == 0;
  const int64_t size = (int64_t)a.N * a.K;
  if (unit < a.G) {
    T* const to = (T*)a.dw + unit * size;
    vec ? store(std::true_type{}, to) : store(std::false_type{}, to);
  } else {
    float* const to = a.part + (unit - a.G) * size;
    vec ? store(std::true_type{}, to) : store(std::false_type{}, to);
  }
}

// column c of the sum of a unit's rows of dy
template <typename T>
__device__ __forceinline__ void ll_store_sum(const LlGrad& a, int64_t unit, int c, double sum) {
  if (unit < a.G)
    ((T*)a.db)[unit * a.N + c] = leaf_from<T>((float)sum);
  else
    a.part_b[(unit - a.G) * a.N + c] = sum;
}

// zeros to dx of the rows without a leaf: 16 bytes a lane, block `part` of kLlZeroBlocks. us of a
// gradient with 8 / 64 / 512 of them, 1M rows of 4096 leaves, 64 x 64 f32: a twentieth of the rows
// without a leaf 406 / 304 / 303, half of them 2027 / 380 / 221.
constexpr int kLlZeroBlocks = 64;
template <typename T>
__device__ __forceinline__ void ll_grad_zeros(const LlGrad& a, int64_t part) {
  const int per = a.K / Ll<T>::kEpc;
  const int64_t first = a.off[a.G], chunks = (a.off[a.G + 1] - first) * per;
  for (int64_t i = part * kLlThreads + threadIdx.x; i < chunks; i += kLlZeroBlocks * kLlThreads)
    ((uint4*)((T*)a.dx + (int64_t)a.order[first + i / per] * a.K))[i % per] =
        make_uint4(0, 0, 0, 0);
}

// One B x B tile (rows of W, columns of W) of one unit: both operands are gathered rows with the
// rows as depth, turned. The row numbers of a tile of depth are fetched a tile ahead of the rows.
// The sums of dy (db) fall out of its fragments, in 64 bits for f32. kAligned: as in
// ll_tile_kernel.
//
// kDx (one tile holds all of W): dx is made of the same tiles of dy, read once for both. Each wave
// holds 16 columns of the leaf's W and multiplies all rows of a tile with them (B = 32: half of
// them). Blocks behind the units' write the zeros of the rows without a leaf. 1M rows, 64 x 64 f32
// in 4096 leaves: 305 us (2.5 TB/s), dW alone 168 (3.05 TB/s), both with the join.
template <typename T, int B, bool kAligned, bool kDx = false>
__global__ __launch_bounds__(kLlThreads) void ll_grad_kernel(LlGrad a) {
  static_assert(!kDx || (B <= 64 && kAligned), "");
  using A = std::conditional_t<sizeof(T) == 4, double, float>;
  constexpr int E = Ll<T>::kEpc, KD = Ll<T>::kDepth, kRow = B / E;
  constexpr int S = B / 2 / 16, Q = B * 8 / kLlThreads;  // 2 x 2 waves
  __shared__ uint4 s_j0[B * 8], s_i0[B * 8];
  __shared__ uint4 s_j1[kAligned ? B * 8 : 1], s_i1[kAligned ? B * 8 : 1];
  __shared__ A s_sum[kLlWaves][S * 16];
  const int64_t blk = leaf_block();
  const int tiles = a.n_tiles * a.k_tiles;
  if (blk >= a.units * tiles) {
    if constexpr (kDx) ll_grad_zeros<T>(a, blk - a.units);
    return;
  }
  const int64_t unit = ll_grad_unit(a, blk / tiles);
  const int t = (int)(blk % tiles);
  const int j0 = t / a.k_tiles * B, i0 = t % a.k_tiles * B;
  const int tid = threadIdx.x, l = lane_id(), w = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int wj = w / 2 * (S * 16), wi = w % 2 * (S * 16);
  int64_t pa, pb;
  if (!ll_grad_rows(a, unit, pa, pb)) return;
  const int rows = (int)(pb - pa);
  const int32_t* const order = a.order + pa;

  f32x4 acc[S][S] = {};
  A sum[S] = {};
  // two waves hold the same rows of dy: each sums one half of the depth
  const bool sums = a.db != nullptr && i0 == 0;
  const LlLane<T> ln;
  auto products = [&](const uint4* sj, const uint4* si) {
#pragma unroll
    for (int step = 0; step < 2; ++step) {
      uint4 fj[S], fi[S];
#pragma unroll
      for (int j = 0; j < S; ++j) fj[j] = ll_frag_turn<T, B>(sj, ln, wj / 16 + j, step);
#pragma unroll
      for (int i = 0; i < S; ++i) fi[i] = ll_frag_turn<T, B>(si, ln, wi / 16 + i, step);
#pragma unroll
      for (int j = 0; j < S; ++j)
#pragma unroll
        for (int i = 0; i < S; ++i) acc[j][i] = ll_mma<T>(fi[i], fj[j], acc[j][i]);
      if (sums && step == (w & 1)) {
#pragma unroll
        for (int j = 0; j < S; ++j) {
          T e[E];
          __builtin_memcpy(e, &fj[j], 16);
          A four[2] = {};
#pragma unroll
          for (int u = 0; u < E; ++u) four[u & 1] += (A)leaf_f32(e[u]);
          sum[j] += four[0] + four[1];
        }
      }
    }
  };
  // dx: this wave's columns of W (zeros past its last row), where in a tile a lane's chunks lie
  constexpr int CW = kDx ? B / 16 : kLlWaves, RJ = KD / 16 * CW / kLlWaves;
  constexpr int DT = kDx ? (B + 4 * E - 1) / (4 * E) : 1;
  const int dc = w % CW * 16, dr = w / CW * (RJ * 16);
  uint4 fw[DT];
  int at_c[DT];
  if constexpr (kDx) {
    const int64_t g = unit < a.G ? unit : (int64_t)a.keys[pa];
    const T* const wg = (const T*)a.w + g * a.N * a.K + min(dc + (l & 15), a.K - 1);
#pragma unroll
    for (int t = 0; t < DT; ++t) {
      T e[E];
#pragma unroll
      for (int u = 0; u < E; ++u) {
        const int k = (4 * t + (l >> 4)) * E + u;
        e[u] = ll_load_or_zeros<T>(rows > 0 && k < a.N, wg + (int64_t)k * a.K);
      }
      __builtin_memcpy(&fw[t], e, 16);
      at_c[t] = ll_turn_chunk<T, B>(dr + (l & 15), 4 * t + (l >> 4));
    }
  }
  auto dx_rows = [&](const uint4* sj, int p0, const int32_t (&to)[RJ]) {
#pragma unroll
    for (int j = 0; j < RJ; ++j) {
      f32x4 d = {};
#pragma unroll
      for (int t = 0; t < DT; ++t) d = ll_mma<T>(fw[t], sj[j * 16 * kRow + at_c[t]], d);
      const int c = dc + 4 * (l >> 4);
      if (p0 + dr + j * 16 + (l & 15) < rows)
        ll_store4<true>((T*)a.dx + (int64_t)to[j] * a.K + c, d, a.K - c);
    }
  };
  if (rows > 0) {
    const T* const x = (const T*)a.x;
    const T* const dy = (const T*)a.dy;
    int32_t row[Q];  // of the next tile to fetch
    auto next_rows = [&](int p0) {
#pragma unroll
      for (int q = 0; q < Q; ++q)
        row[q] = order[min(p0 + (q * kLlThreads + tid) / kRow, rows - 1)];
    };
    if constexpr (kAligned) {
      int32_t to0[RJ], to1[RJ];  // dx: the rows of this lane in either buffer
      auto load = [&](uint4* sj, uint4* si, int p0, int32_t (&to)[RJ]) {
        if constexpr (kDx) {
#pragma unroll
          for (int j = 0; j < RJ; ++j) to[j] = order[min(p0 + dr + j * 16 + (l & 15), rows - 1)];
        }
#pragma unroll
        for (int q = 0; q < Q; ++q) {
          const int id = q * kLlThreads + tid, k = id / kRow;
          const int c = ll_turn_chunk<T, B>(k, id % kRow) - k * kRow;
          const bool in = p0 + k < rows;
          const T* const pj = dy + row[q] * a.dy_stride + min(j0 + c * E, a.n_row - E);
          const T* const pi = x + row[q] * a.x_stride + min(i0 + c * E, a.k_row - E);
          // (dx sums over dy's columns: zeros behind the last)
          ll_dma(in && (!kDx || c * E < a.N) ? (const void*)pj : kLlZeros,
                 sj + q * kLlThreads + w * kWave);
          ll_dma(in ? (const void*)pi : kLlZeros, si + q * kLlThreads + w * kWave);
        }
        next_rows(p0 + KD);
      };
      next_rows(0);
      load(s_j0, s_i0, 0, to0);
      for (int p0 = 0; p0 < rows; p0 += 2 * KD) {
        ll_dma_wait();
        if (p0 + KD < rows) load(s_j1, s_i1, p0 + KD, to1);
        products(s_j0, s_i0);
        if constexpr (kDx) dx_rows(s_j0, p0, to0);
        if (p0 + KD >= rows) break;
        ll_dma_wait();
        if (p0 + 2 * KD < rows) load(s_j0, s_i0, p0 + 2 * KD, to0);
        products(s_j1, s_i1);
        if constexpr (kDx) dx_rows(s_j1, p0 + KD, to1);
      }
    } else {
      uint4 vj[Q], vi[Q];
      auto load = [&](int p0) {
#pragma unroll
        for (int q = 0; q < Q; ++q) {
          const int id = q * kLlThreads + tid, k = id / kRow, c = id % kRow;
          const bool in = p0 + k < rows;
          vj[q] = ll_chunk<T, false>(dy + row[q] * a.dy_stride + j0 + c * E,
                                     in ? a.N - j0 - c * E : 0);
          vi[q] = ll_chunk<T, false>(x + row[q] * a.x_stride + i0 + c * E,
                                     in ? a.K - i0 - c * E : 0);
        }
        next_rows(p0 + KD);
      };
      next_rows(0);
      load(0);
      for (int p0 = 0; p0 < rows; p0 += KD) {
#pragma unroll
        for (int q = 0; q < Q; ++q) {
          const int id = q * kLlThreads + tid;
          s_j0[ll_turn_chunk<T, B>(id / kRow, id % kRow)] = vj[q];
          s_i0[ll_turn_chunk<T, B>(id / kRow, id % kRow)] = vi[q];
        }
        __syncthreads();
        if (p0 + KD < rows) load(p0 + KD);
        products(s_j0, s_i0);
        __syncthreads();
      }
    }
  }
  if (sums) {
#pragma unroll
    for (int j = 0; j < S; ++j) {
      sum[j] += __shfl_xor(sum[j], 16, kWave);
      sum[j] += __shfl_xor(sum[j], 32, kWave);
      if (l < 16) s_sum[w][j * 16 + l] = sum[j];
    }
    __syncthreads();
    const int c = tid % B, q = c / (S * 16) * 2;
    if (tid < B && j0 + c < a.N)
      ll_store_sum<T>(a, unit, j0 + c,
                      (double)s_sum[q][c % (S * 16)] + (double)s_sum[q + 1][c % (S * 16)]);
  }
  ll_grad_store<T, S, S>(acc, a, unit, j0 + wj, i0 + wi);
}

// The same on 256 x 256 tiles of 16-bit types (see ll_big_kernel): both operands turned.
template <typename T>
__global__ __launch_bounds__(kBigThreads, 2) void ll_big_grad_kernel(LlGrad a) {
  constexpr int E = Ll<T>::kEpc, KD = Ll<T>::kDepth;
  constexpr int SJ = 8, SI = 4;
  static_assert(sizeof(T) == 2, "the buffers' layout is for 16-bit types");
  __shared__ alignas(16) char s0[2 * kBigTurnBytes], s1[2 * kBigTurnBytes];  // dy, then x
  const int64_t blk = ll_xcd_order(leaf_block());
  const int tiles = a.n_tiles * a.k_tiles;
  if (blk >= a.units * tiles) return;
  const int64_t unit = ll_grad_unit(a, blk / tiles);
  const int t = (int)(blk % tiles);
  const int j0 = t / a.k_tiles * kBig, i0 = t % a.k_tiles * kBig;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int wj = w / 4 * (SJ * 16), wi = w % 4 * (SI * 16);
  int64_t pa, pb;
  if (!ll_grad_rows(a, unit, pa, pb)) return;
  const int rows = (int)(pb - pa);
  const int32_t* const order = a.order + pa;

  f32x4 acc[SJ][SI] = {};
  if (rows > 0) {
    const LlBigLane lt;
    const i32x4 dy_rsrc = ll_rsrc(a.dy), x_rsrc = ll_rsrc(a.x);
    const uint32_t jc = (uint32_t)min(j0 + ll_big_turn_col() * E, a.n_row - E) * sizeof(T);
    const uint32_t ic = (uint32_t)min(i0 + ll_big_turn_col() * E, a.k_row - E) * sizeof(T);
    const uint32_t js = (uint32_t)a.dy_stride * sizeof(T), is = (uint32_t)a.x_stride * sizeof(T);
    int32_t row[kBigQ];  // of the next tile to fetch
    auto next_rows = [&](int p0) {
#pragma unroll
      for (int q = 0; q < kBigQ; ++q) row[q] = order[min(p0 + ll_big_turn_row(w, q), rows - 1)];
    };
    // tail: the tile may reach past the rows
    auto load = [&](auto tail, char* s, int p0) {
      // the row numbers have arrived with the barrier; told here, the compiler waits for none of
      // them between the fetches, where it would wait for the fetches too
      static_assert(kBigQ == 4, "");
      asm volatile("" : "+v"(row[0]), "+v"(row[1]), "+v"(row[2]), "+v"(row[3]));
#pragma unroll
      for (int q = 0; q < kBigQ; ++q) {
        char* const to = s + ll_big_turn_to(w, q);
        const uint32_t jo = (uint32_t)row[q] * js + jc, io = (uint32_t)row[q] * is + ic;
        if constexpr (!tail()) {
          ll_dma_buffer(dy_rsrc, jo, 0, to);
          ll_dma_buffer(x_rsrc, io, 0, to + kBigTurnBytes);
        } else {
          const bool in = p0 + ll_big_turn_row(w, q) < rows;
          ll_dma_at(in ? (const char*)a.dy + jo : (const char*)kLlZeros, to);
          ll_dma_at(in ? (const char*)a.x + io : (const char*)kLlZeros, to + kBigTurnBytes);
        }
      }
      next_rows(p0 + KD);
    };
    uint4 fj[SJ], fi0[SI], fi1[SI];
    auto read_j = [&](const char* s, int j, int step) {
      return ll_big_turn(s, lt, wj / 16, j, step);
    };
    auto read_i = [&](uint4 (&fi)[SI], const char* s, int step) {
#pragma unroll
      for (int i = 0; i < SI; ++i) fi[i] = ll_big_turn(s + kBigTurnBytes, lt, wi / 16, i, step);
    };
    auto half = [&](const uint4 (&fi)[SI], uint4 (&fn)[SI], const char* next, int step) {
      read_i(fn, next, step);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int j = 0; j < SJ; ++j) {
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int i = 0; i < SI; ++i) acc[j][i] = ll_mma<T>(fi[i], fj[j], acc[j][i]);
        __builtin_amdgcn_s_setprio(0);
        fj[j] = read_j(next, j, step);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    auto pair = [&](auto tail, int p0) {
      half(fi0, fi1, s0, 1);
      ll_dma_wait();
      load(tail, s0, p0 + 2 * KD);
      half(fi1, fi0, s1, 0);
      half(fi0, fi1, s1, 1);
      ll_dma_wait();
      load(tail, s1, p0 + 3 * KD);
      half(fi1, fi0, s0, 0);
    };
    constexpr std::true_type kYes{};
    constexpr std::false_type kNo{};
    next_rows(0);
    load(kYes, s0, 0);
    ll_dma_wait();
    load(kYes, s1, KD);
#pragma unroll
    for (int j = 0; j < SJ; ++j) fj[j] = read_j(s0, j, 0);
    read_i(fi0, s0, 0);
    int p0 = 0;
    for (; p0 + 4 * KD <= rows; p0 += 2 * KD) pair(kNo, p0);
    for (; p0 < rows; p0 += 2 * KD) pair(kYes, p0);
    ll_dma_wait();  // (the fetches behind the last tile, before the workgroup's LDS goes)
  }
  ll_grad_store<T, SJ, SI>(acc, a, unit, j0 + wj, i0 + wi);
}

// Adds the partial matrices of the leaves with more than `run` rows, in 64 bits for f32 (and their
// partial sums of dy, where the kernel above made them). Such leaves are looked for among the
// leaves, or, if these are fewer, among the chunks in which they start: `per` blocks each, which
// take a leaf's elements in turn, 4 a lane. The WAVES share a leaf's pieces and meet in LDS, so
// that many pieces of a small matrix are not one chain of loads (1M rows of one leaf, 64 x 64 f32:
// a weight gradient takes 197 to 218 us with 16 waves, 342 with none sharing).
template <typename T, int WAVES>
__global__ __launch_bounds__(WAVES* kWave) void ll_join_kernel(LlGrad a, bool by_leaf, int per) {
  using A = std::conditional_t<sizeof(T) == 4, double, float>;
  __shared__ A s_sum[WAVES][4][kWave];
  __shared__ double s_b[WAVES][kWave];
  const int64_t blk = leaf_block(), i0 = blk / per, m = a.off[a.G];
  int64_t k1 = i0;
  if (by_leaf) {
    if (i0 >= a.G) return;
  } else {
    if (i0 * a.run >= m) return;
    k1 = a.keys[min<int64_t>((i0 + 1) * a.run, m) - 1];
  }
  const int64_t s1 = a.off[k1], e1 = a.off[k1 + 1];
  if (e1 - s1 <= a.run || (!by_leaf && s1 < i0 * a.run)) return;
  const int64_t c = s1 / a.run, k0 = a.keys[c * a.run];
  const int64_t size = (int64_t)a.N * a.K;
  const int pieces = (int)((e1 - 1) / a.run - c) + 1;
  // piece i's place in the partial matrices
  auto place = [&](int i) { return i == 0 ? 2 * c + (k1 != k0 ? 1 : 0) : 2 * (c + i); };
  int share = 1;  // waves that share the pieces of the same elements
  while (share < WAVES && 2 * share <= pieces) share <<= 1;
  const int l = lane_id(), w = threadIdx.x / kWave, q = w & (share - 1), sub = w / share;
  const int64_t step = (int64_t)(WAVES / share) * kWave * 4;
  for (int64_t b0 = (blk % per) * step; b0 < size; b0 += per * step) {
    const int64_t e = b0 + (sub * kWave + l) * 4;
    A sum[4] = {};
    if (e < size) {
      if (size % 4 == 0) {
#pragma unroll 8
        for (int i = q; i < pieces; i += share) {
          const f32x4 v = *(const f32x4*)(a.part + place(i) * size + e);
#pragma unroll
          for (int u = 0; u < 4; ++u) sum[u] += (A)v[u];
        }
      } else {
        for (int i = q; i < pieces; i += share)
          for (int u = 0; u < 4 && e + u < size; ++u) sum[u] += (A)a.part[place(i) * size + e + u];
      }
    }
    if (share > 1) {
#pragma unroll
      for (int u = 0; u < 4; ++u) s_sum[w][u][l] = sum[u];
      __syncthreads();
      if (q == 0) {
        for (int i = 1; i < share; ++i)
#pragma unroll
          for (int u = 0; u < 4; ++u) sum[u] += s_sum[w + i][u][l];
      }
      __syncthreads();
    }
    if (q == 0 && e < size) {
      T* const to = (T*)a.dw + k1 * size + e;
      if (size % 4 == 0) {
        LeafVec<T, 4> o;
#pragma unroll
        for (int u = 0; u < 4; ++u) o.v[u] = leaf_from<T>((float)sum[u]);
        *(LeafVec<T, 4>*)to = o;
      } else {
        for (int u = 0; u < 4 && e + u < size; ++u) to[u] = leaf_from<T>((float)sum[u]);
      }
    }
  }
  if (a.db == nullptr || blk % per != 0) return;
  for (int n0 = 0; n0 < a.N; n0 += WAVES / share * kWave) {
    const int n = n0 + sub * kWave + l;
    double sum = 0;
    if (n < a.N) {
#pragma unroll 8
      for (int i = q; i < pieces; i += share) sum += a.part_b[place(i) * a.N + n];
    }
    s_b[w][l] = sum;
    __syncthreads();
    if (q == 0 && n < a.N) {
      for (int i = 1; i < share; ++i) sum += s_b[w + i][l];
      ((T*)a.db)[k1 * a.N + n] = leaf_from<T>((float)sum);
    }
    __syncthreads();
  }
}

// ---- forward of at most 64 rows, straight from the leaf indices (no route). Each wave holds all
// of them, one a lane. Block (column tile, row i): row i leads the tile of up to 16 rows of its
// leaf that start with it; rows that follow another row of their leaf inside its 16 leave. So a
// leaf's matrix is read once for 16 rows. The waves split the depth, from memory straight into
// fragments, and their sums meet in LDS. 64 rows of 64 leaves, 2048 -> 1024 bf16: 36 us, 4.7 TB/s.
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
  T* const to = y + (int64_t)row * a.N + c;
  vec ? ll_store4<true>(to, acc, a.N - c) : ll_store4<false>(to, acc, a.N - c);
}

// Rows of `cols` elements as rows of whole 16-byte chunks, zeros behind the last column: what the
// tiles that fetch straight into LDS can read. One chunk a thread; memory is the bound (10007 rows
// of 601 f16 6 us).
template <typename T>
__global__ __launch_bounds__(kLlThreads) void ll_pack_kernel(const T* __restrict__ src,
                                                             int64_t stride, int64_t rows, int cols,
                                                             int chunks, uint4* __restrict__ dst) {
  const int64_t i = leaf_block() * kLlThreads + threadIdx.x;
  if (i >= rows * chunks) return;
  const int64_t r = i / chunks;
  const int c = (int)(i - r * chunks) * Ll<T>::kEpc;
  dst[i] = ll_chunk<T, false>(src + r * stride + c, cols - c);
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

template <int N>
using LlInt = std::integral_constant<int, N>;

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

// Rows short enough for ll_rows_kernel. 500k rows in 2000 leaves, us of it / of the tiles: f32 64
// deep, 16 columns 36 / 32, 32: 47 / 68, 64: 82 / 92, 128: 153 / 167; bf16 64 deep, 64 columns 38 /
// 44, 128: 67 / 73; bf16 128 deep, 128 columns 121 / 108, its row gradient 143 / 106.
static bool ll_short_rows(int elem, int depth, int cols) {
  if (cols > 128) return false;
  return depth * elem <= 128 || (elem == 4 && depth * elem <= 256 && cols > 16);
}

// ---- operands whose rows do not start on 16 bytes, or whose width is no multiple of them
static bool ll_rows_aligned(int type, const void* p, int64_t stride, int width) {
  const int e = type == kLeafF32 ? 4 : 8;
  return (uintptr_t)p % 16 == 0 && stride % e == 0 && width % e == 0;
}
static int ll_packed_width(int type, int width) {
  const int e = type == kLeafF32 ? 4 : 8;
  return (width + e - 1) / e * e;
}
static int64_t ll_packed_bytes(int type, int64_t rows, int width) {
  return rows * ll_packed_width(type, width) * (type == kLeafF32 ? 4 : 2);
}
static const void* ll_pack(hipStream_t s, int type, const void* src, int64_t stride, int64_t rows,
                           int width, void*& work) {
  void* const to = work;
  work = (char*)work + ll_packed_bytes(type, rows, width);
  ll_dispatch_type(type, [&](auto t) {
    using T = decltype(t);
    const int chunks = (int)(ll_packed_width(type, width) / Ll<T>::kEpc);
    const int64_t blocks = (rows * chunks + kLlThreads - 1) / kLlThreads;
    hipLaunchKernelGGL(ll_pack_kernel<T>, leaf_grid(blocks), dim3(kLlThreads), 0, s, (const T*)src,
                       stride, rows, width, chunks, (uint4*)to);
    MT_HIP_CHECK(hipGetLastError());
  });
  return to;
}

// Which operands a pass copies into whole chunks first.
struct LlPacks {
  bool x = false, dy = false, w = false;
  bool any() const { return x || dy || w; }
  int64_t bytes(int type, int64_t n, int G, int K, int N) const {
    return (x ? ll_packed_bytes(type, n, K) : 0) + (dy ? ll_packed_bytes(type, n, N) : 0) +
           (w ? ll_packed_bytes(type, (int64_t)G * N, K) : 0);
  }
};
// Such a copy is two passes over an operand and lets the products fetch straight into LDS. us
// without / with, a forward pass, a row gradient, all gradients, bf16 and f16 unless noted:
//   65536 rows, 64 leaves, 2047 -> 2049: 1466 / 1169, 1760 / 1118, 5032 / 2443
//   20000 rows, 300 leaves, 511 -> 513: 104 / 166, 155 / 158, 414 / 349; 100 leaves: 77 / 77 (no
//     copy), 101 / 73, 250 / 174; 20 leaves: 63 / 59, 88 / 58, 226 / 134; 30 leaves, f32 498 / 456
//   10007 rows, 12 leaves, 1001 -> 601: 45 / 50, 66 / 56, 162 / 130
//   300000 rows, 100 leaves, 301 -> 199: 265 / 294, 325 / 428, 1026 / 806; 129 -> 127: 104 / 160,
//     176 / 152, 459 / 298
//   1500 rows, 2 leaves, 511 -> 513: 23 / 23, 35 / 26, 70 / 54
//   below kLlPackRows, 2 leaves, 511 -> 513, a row gradient, all: 500 rows 39 / 22, 61 / 41; 1000
//     rows 39 / 25, 69 / 46 (a lower bound would serve)
// So gradients copy from widths of about 64 on, the row gradient alone from about 256 on, a forward
// pass where the largest tiles follow; W, which a leaf's rows have to pay for, from 64 rows a leaf
// on with dW and 192 without, 384 in a forward pass, and not in f32, whose products are slower.
constexpr int kLlPackRows = 1024;
static LlPacks ll_forward_packs(int type, const void* x, int64_t x_stride, const void* w, int64_t n,
                                int G, int K, int N) {
  LlPacks p;
  const bool xa = ll_rows_aligned(type, x, x_stride, K), wa = ll_rows_aligned(type, w, K, K);
  if ((xa && wa) || type == kLeafF32 || K < 512 || n / G < 384) return p;
  if ((n >> 8) * ((N + kBig - 1) / kBig) < 256) return p;
  p.x = !xa, p.w = !wa;
  return p;
}
static LlPacks ll_grad_packs(int type, const void* x, int64_t x_stride, const void* dy,
                             int64_t dy_stride, const void* w, int64_t n, int G, int K, int N,
                             bool dx, bool dw) {
  LlPacks p;
  const bool xa = ll_rows_aligned(type, x, x_stride, K), wa = ll_rows_aligned(type, w, K, K);
  const bool ya = ll_rows_aligned(type, dy, dy_stride, N);
  const int64_t width = (int64_t)K * N / (K + N);  // half of it where both are the same
  if (width < (dw ? 32 : 128) || n / G < 32 || n < kLlPackRows) return p;
  if (dw) p.x = !xa, p.dy = !ya;
  if (dx && (wa || (type != kLeafF32 && n / G >= (dw ? 64 : 192)))) p.dy = !ya, p.w = !wa;
  return p;
}

// scratch for the tile list
static int64_t ll_plan_bytes(int64_t n, int G) {
  return n / G >= kLlBigRows ? 8 + 8 * ((n >> 8) + G + 1) : 0;
}

// forward (dx false: src = x, depth = K, cols = N) or dx (src = dy, depth = N, cols = K). Rows of
// src and W may be wider than that, with zeros behind (src_width, w_row).
static void ll_launch_tile(hipStream_t s, int type, bool dx, const void* src, int64_t src_stride,
                           int src_width, const int32_t* order, const int32_t* off, int64_t n,
                           int G, const void* w, int w_row, const void* bias, int K, int N,
                           void* out, void* work) {
  LlTile a{};
  a.src = src, a.w = w, a.bias = bias, a.out = out, a.order = order, a.off = off;
  a.src_stride = src_stride, a.w_stride = (int64_t)N * w_row;
  a.G = G, a.depth = dx ? N : w_row, a.cols = dx ? K : N, a.w_row = w_row;
  ll_dispatch_type(type, [&](auto t) {
    using T = decltype(t);
    const bool al = ll_aligned<T>({src, w}, {w_row, src_stride, src_width});
    auto go = [&](auto bj, auto bi, auto wj, auto nw) {
      a.bj_shift = __builtin_ctz((unsigned)bj());
      a.col_tiles = (a.cols + bi() - 1) / bi();
      a.tiles = ((n >> a.bj_shift) + G + 1) * a.col_tiles;
      const dim3 grid = leaf_grid(ll_xcd_blocks(a.tiles));
      auto run = [&](auto kern) {
        hipLaunchKernelGGL(kern, grid, dim3(nw() * kWave), 0, s, a);
        MT_HIP_CHECK(hipGetLastError());
      };
      if (dx)
        al ? run(ll_tile_kernel<T, true, bj(), bi(), wj(), nw(), true>)
           : run(ll_tile_kernel<T, true, bj(), bi(), wj(), nw(), false>);
      else
        al ? run(ll_tile_kernel<T, false, bj(), bi(), wj(), nw(), true>)
           : run(ll_tile_kernel<T, false, bj(), bi(), wj(), nw(), false>);
    };
    const int64_t mean = n / G;
    // 256 x 256 tiles from 256 of them on (16384 rows in 16 leaves, 1024 -> 1024 bf16: 41 us, 57
    // with 128 x 128; 8192 rows: 44 and 39), and leaves that fill them (128 rows a leaf, 2048 ->
    // 2048: 364 and 329; 256 rows, 1024 -> 1024: 44 and 49)
    const bool big = sizeof(T) == 2 && al && mean >= kLlBigRows &&
                     (n >> 8) * ((a.cols + kBig - 1) / kBig) >= 256 &&
                     (n * src_stride + a.depth) * (int64_t)sizeof(T) < (1ll << 32) &&
                     a.w_stride * (int64_t)sizeof(T) < (1ll << 32);
    if (ll_short_rows(sizeof(T), a.depth, a.cols)) {
      const int si = a.cols <= 16 ? 1 : a.cols <= 32 ? 2 : 4;  // fragments of columns a wave holds
      a.col_tiles = (a.cols + si * 16 - 1) / (si * 16);
      a.tiles = ((n >> kRowsShift) + G + 1) * a.col_tiles;
      auto rows = [&](auto steps, auto cols) {
        auto run = [&](auto kern) {
          hipLaunchKernelGGL(kern, leaf_grid((a.tiles + kLlWaves - 1) / kLlWaves), dim3(kLlThreads),
                             0, s, a);
          MT_HIP_CHECK(hipGetLastError());
        };
        if (dx)
          al ? run(ll_rows_kernel<T, true, steps(), cols(), true>)
             : run(ll_rows_kernel<T, true, steps(), cols(), false>);
        else
          al ? run(ll_rows_kernel<T, false, steps(), cols(), true>)
             : run(ll_rows_kernel<T, false, steps(), cols(), false>);
      };
      [[maybe_unused]] const bool half = a.depth * (int)sizeof(T) <= 128;
      if constexpr (sizeof(T) == 4) {
        if (half)
          si == 1   ? rows(LlInt<2>{}, LlInt<1>{})
          : si == 2 ? rows(LlInt<2>{}, LlInt<2>{})
                    : rows(LlInt<2>{}, LlInt<4>{});
        else
          si == 2 ? rows(LlInt<4>{}, LlInt<2>{}) : rows(LlInt<4>{}, LlInt<4>{});
      } else {
        si == 1   ? rows(LlInt<2>{}, LlInt<1>{})
        : si == 2 ? rows(LlInt<2>{}, LlInt<2>{})
                  : rows(LlInt<2>{}, LlInt<4>{});
      }
    } else if (a.cols <= 16)
      go(LlInt<64>{}, LlInt<16>{}, LlInt<4>{}, LlInt<4>{});
    // Rows of a tile by the mean rows of a leaf; 16384 rows, 1024 -> 1024 bf16, us with 16 / 64 /
    // 128 rows: mean 8: 757 / 792 / 827, mean 16: 412 / 429 / 430, mean 32: 262 / 236 / 234, mean
    // 64: 192 / 133 / 128, mean 256: 127 / 67 / 49. 512 -> 512 f32: mean 16: 219 / 259 / 509, mean
    // 32: 139 / 143 / 267, mean 64: 116 / 99 / 142, mean 128: 114 / 93 / 82.
    else if (mean < (sizeof(T) == 4 ? 48 : 24))
      go(LlInt<16>{}, LlInt<64>{}, LlInt<1>{}, LlInt<4>{});
    else if ((sizeof(T) == 4 && mean < 96) || a.cols <= 64)
      go(LlInt<64>{}, LlInt<64>{}, LlInt<2>{}, LlInt<4>{});
    else if (!big)
      go(LlInt<128>{}, LlInt<128>{}, LlInt<2>{}, LlInt<4>{});
    else if constexpr (sizeof(T) == 2) {
      a.bj_shift = 8;
      a.col_tiles = (a.cols + kBig - 1) / kBig;
      a.tiles = ((n >> 8) + G + 1) * a.col_tiles;
      auto run = [&](auto kern) {
        hipLaunchKernelGGL(kern, leaf_grid(ll_xcd_blocks(a.tiles)), dim3(kBigThreads), 0, s,
                           a);
        MT_HIP_CHECK(hipGetLastError());
      };
      int2* const plan = (int2*)((int32_t*)work + 2);
      a.plan = plan, a.plan_count = (const int32_t*)work;
      hipLaunchKernelGGL(ll_plan_kernel, dim3(1), dim3(kLlPlanThreads), 0, s, off, G, a.bj_shift,
                         plan, (int32_t*)work);
      MT_HIP_CHECK(hipGetLastError());
      dx ? run(ll_big_kernel<T, true>) : run(ll_big_kernel<T, false>);
    }
  });
}

// Rows a dW unit may have, a power of two; leaves with more are cut, and a cut costs a partial
// matrix in 32 bits, written and read. Where whole leaves make 2048 tiles, only those above four
// times the mean are cut (us with 1, 2, 4, 8 times: 1M rows of 4096 leaves, 64 x 64 f32 227, 189,
// 176, 192; 65536 rows of 64 leaves, 2048 x 2048 bf16 1452, 953, 830, 891). Otherwise pieces make
// up to 1024 tiles of 32, 512 of 64 and 128, 256 of 256 (500k rows of 2000 leaves, 32 x 32 f32 38
// with 512, 33 with 1024, 43 with 2048; 1M rows of 64 leaves, 64 x 64 bf16 75 with 512, 81 with
// 1024; 16384 rows of one leaf, 1024 x 1024 bf16 55 with 256, 77 with 512).
static int64_t ll_grad_run(int64_t n, int G, int b, int64_t tiles) {
  int64_t run = 256;
  if (G * tiles >= 2048) {
    while (run < 4 * (n / G)) run <<= 1;
  } else {
    const int most = b == 32 ? 1024 : b == kBig ? 256 : 512;
    while (run < (1 << 20) && n / run * tiles > most) run <<= 1;
  }
  return run;
}
// Tile edge of dW; direct: operands are 16-byte aligned and lie within 4 GiB. 256 where leaves are
// long and fill the GPU, whole or in pieces; bf16 1024 x 1024, us with 256 / 128: 4096 rows in 4
// leaves 39 / 22, in 16 25 / 31, in 64 68 / 57; 16384 rows in 1 55 / 61, in 16 44 / 62, in 64 81 /
// 90. 32 for short rows (500k rows of 2000 leaves, 32 x 32 f32 37, 83 with 64).
static int ll_grad_tile(int type, bool direct, int64_t n, int G, int K, int N) {
  const int64_t big = (int64_t)((N + kBig - 1) / kBig) * ((K + kBig - 1) / kBig);
  if (type != kLeafF32 && direct && N > 128 && K > 128 && n / G >= 256 &&
      (G * big >= 256 || (n / 256) * big >= 1024))
    return kBig;
  return N > 64 && K > 64 ? 128 : N > 32 || K > 32 ? 64 : 32;
}
static int64_t ll_grad_tiles(int b, int K, int N) {
  return (int64_t)((N + b - 1) / b) * ((K + b - 1) / b);
}

// dx together with dW, where one tile holds W and there are leaves enough; us together / apart: 1M
// rows, 64 x 64: 4096 leaves f32 294 / 350, bf16 146 / 177, 64 leaves f32 374 / 352, bf16 164 /
// 148; 500k rows, 32 x 32: 2000 leaves f32 57 / 68, 50 leaves 69 / 66, bf16 30 leaves 43 / 51.
static bool ll_fuse_dx(int b, int G, int K, int N) {
  return N <= b && K <= b && (b == 32 || (b == 64 && G >= 2048));
}

// scratch for the partial matrices (and sums), whichever tile is taken
static int64_t ll_part_bytes(int type, int64_t n, int G, int K, int N) {
  int64_t chunks = 0;
  for (bool direct : {false, true}) {
    const int b = ll_grad_tile(type, direct, n, G, K, N);
    const int64_t run = ll_grad_run(n, G, b, ll_grad_tiles(b, K, N));
    if (n > run) chunks = std::max(chunks, (n + run - 1) / run);
  }
  return 2 * chunks * ((int64_t)N * K * 4 + 8 * N + 8);
}

// dW, and dx and db where they are asked for (not null); whether they were made here. Rows of x and
// dy may be wider than K and N, with zeros behind (k_row, n_row).
struct LlMade {
  bool dx, db;
};
static LlMade ll_launch_grad(hipStream_t s, int type, const void* x, int64_t x_stride, int k_row,
                             const void* dy, int64_t dy_stride, int n_row, const int32_t* order,
                             const uint32_t* keys, const int32_t* off, int64_t n, int G,
                             const void* w, int K, int N, void* dx, void* dw, void* db,
                             void* work) {
  LlGrad a{};
  a.x = x, a.dy = dy, a.dw = dw, a.part = (float*)work;
  a.order = order, a.keys = keys, a.off = off;
  a.x_stride = x_stride, a.dy_stride = dy_stride;
  a.G = G, a.N = N, a.K = K, a.n_row = n_row, a.k_row = k_row;
  const int64_t elem = type == kLeafF32 ? 4 : 2;
  const bool al = (elem == 4 ? ll_aligned<float> : ll_aligned<f16_t>)(
      {x, dy}, {k_row, n_row, x_stride, dy_stride});
  const bool direct =
      al && (n * std::max(x_stride, dy_stride) + std::max(k_row, n_row)) * elem < (1ll << 32);
  const int b = ll_grad_tile(type, direct, n, G, K, N);
  const int64_t tiles = ll_grad_tiles(b, K, N);
  a.n_tiles = (N + b - 1) / b, a.k_tiles = (K + b - 1) / b;
  a.run = ll_grad_run(n, G, b, tiles);
  const int64_t chunks = n > a.run ? (n + a.run - 1) / a.run : 0;
  a.units = G + 2 * chunks;
  ll_dispatch_type(type, [&](auto t) {
    using T = decltype(t);
    auto run = [&](auto kern, int64_t blocks, int threads) {
      hipLaunchKernelGGL(kern, leaf_grid(blocks), dim3(threads), 0, s, a);
      MT_HIP_CHECK(hipGetLastError());
    };
    const int64_t all = a.units * tiles;
    if (b != kBig) a.db = db;
    a.part_b = (double*)((char*)work + (2 * chunks * (int64_t)N * K * 4 + 7) / 8 * 8);
    auto tile = [&](auto edge) {
      if constexpr (edge() <= 64) {
        if (a.dx != nullptr)
          return run(ll_grad_kernel<T, edge(), true, true>, all + kLlZeroBlocks, kLlThreads);
      }
      al ? run(ll_grad_kernel<T, edge(), true>, all, kLlThreads)
         : run(ll_grad_kernel<T, edge(), false>, all, kLlThreads);
    };
    if (dx != nullptr && al && ll_aligned<T>({dx}, {}) && ll_fuse_dx(b, G, K, N))
      a.w = w, a.dx = dx;
    if (b == kBig) {
      if constexpr (sizeof(T) == 2) run(ll_big_grad_kernel<T>, ll_xcd_blocks(all), kBigThreads);
    } else {
      b == 128  ? tile(LlInt<128>{})
      : b == 64 ? tile(LlInt<64>{})
                : tile(LlInt<32>{});
    }
    if (chunks > 0) {
      // A block that finds nothing to do costs 5 ns with 16 waves, a quarter of that with 4, which
      // large matrices take: they have few pieces (65536 rows, 64 leaves, 2048 x 2048: 33 / 12 us).
      const int64_t starts = std::min<int64_t>(G, chunks), size = (int64_t)N * K;
      auto join = [&](auto waves, int64_t blocks) {
        const int64_t per = std::clamp<int64_t>(blocks / starts, 1,
                                                std::min<int64_t>(512, (size + 255) / 256));
        hipLaunchKernelGGL((ll_join_kernel<T, waves()>), leaf_grid(starts * per),
                           dim3(waves() * kWave), 0, s, a, G <= chunks, (int)per);
      };
      size < 65536 ? join(LlInt<16>{}, 1024)
                   : join(LlInt<4>{}, std::max<int64_t>(4096, size / 128));
      MT_HIP_CHECK(hipGetLastError());
    }
  });
  return LlMade{a.dx != nullptr, a.db != nullptr};
}

// ---- a forward and a backward pass
int64_t leaf_linear_bytes(int type, const void* x, int64_t x_stride, const void* w, int64_t n,
                          int G, int K, int N) {
  const LlPacks p = ll_forward_packs(type, x, x_stride, w, n, G, K, N);
  return p.bytes(type, n, G, K, N) + ll_plan_bytes(n, G);
}

void launch_leaf_linear(hipStream_t s, int type, const void* x, int64_t x_stride,
                        const int32_t* order, const int32_t* off, int64_t n, int G, const void* w,
                        const void* bias, int K, int N, void* y, void* work) {
  if (n <= 0) return;
  const LlPacks p = ll_forward_packs(type, x, x_stride, w, n, G, K, N);
  const int k_row = p.any() ? ll_packed_width(type, K) : K;
  if (p.x) x = ll_pack(s, type, x, x_stride, n, K, work), x_stride = k_row;
  if (p.w) w = ll_pack(s, type, w, K, (int64_t)G * N, K, work);
  ll_launch_tile(s, type, false, x, x_stride, k_row, order, off, n, G, w, k_row, bias, K, N, y,
                 work);
}

int64_t leaf_linear_grad_bytes(int type, const void* x, int64_t x_stride, const void* dy,
                               int64_t dy_stride, const void* w, int64_t n, int G, int K, int N,
                               bool dx, bool dw, bool db) {
  const LlPacks p = ll_grad_packs(type, x, x_stride, dy, dy_stride, w, n, G, K, N, dx, dw);
  return p.bytes(type, n, G, K, N) + std::max({dx ? ll_plan_bytes(n, G) : 0,
                                               dw ? ll_part_bytes(type, n, G, K, N) : 0,
                                               db ? leaf_embed_grad_bytes(type, n, N) : 0});
}

// dx, dw and db, each where it is not null; their scratch is used by one after the other
void launch_leaf_linear_grad(hipStream_t s, int type, const void* x, int64_t x_stride,
                             const void* dy, int64_t dy_stride, const int32_t* order,
                             const uint32_t* keys, const int32_t* off, int64_t n, int G,
                             const void* w, int K, int N, void* dx, void* dw, void* db,
                             void* work) {
  const LlPacks p = ll_grad_packs(type, x, x_stride, dy, dy_stride, w, n, G, K, N, dx != nullptr,
                                  dw != nullptr);
  int k_row = K, n_row = N, w_row = K;
  const void* const dy0 = dy;
  const int64_t dy0_stride = dy_stride;
  if (p.x) {
    k_row = ll_packed_width(type, K);
    x = ll_pack(s, type, x, x_stride, n, K, work), x_stride = k_row;
  }
  if (p.dy) {
    n_row = ll_packed_width(type, N);
    dy = ll_pack(s, type, dy, dy_stride, n, N, work), dy_stride = n_row;
  }
  if (p.w) {
    w_row = ll_packed_width(type, K);
    w = ll_pack(s, type, w, K, (int64_t)G * N, K, work);
  }
  LlMade made{};
  if (dw != nullptr)
    made = ll_launch_grad(s, type, x, x_stride, k_row, dy, dy_stride, n_row, order, keys, off, n,
                          G, w, K, N, dx, dw, db, work);
  if (dx != nullptr && !made.dx && n > 0)
    ll_launch_tile(s, type, true, dy, dy_stride, n_row, order, off, n, G, w, w_row, nullptr, K, N,
                   dx, work);
  if (db != nullptr && !made.db)
    launch_leaf_embed_grad(s, type, dy0, dy0_stride, order, keys, off, n, G, N, 1.f, db, work);
}

}  // namespace mt
