// Batched inference on gfx950 (binning lives in binning.hip).
//
// predict: replaces the reference's per-row recursive Python ``walk`` driven
// by ``np.apply_along_axis`` (mpitree/tree/decision_tree.py:208-227) with one
// thread per row walking the flat pre-order tree arrays (root-to-leaf loads of
// 16-B node records stay in L1/L2; the raw feature value is compared in fp64,
// so ``x <= threshold`` is decided exactly as on the host).

#include "common.h"

namespace mt {

struct NodeRec {
  int32_t feature;  // -1 leaf
  int32_t left;
  int32_t right;
  int32_t number;  // of a leaf, among the leaves
};

// kNumber: writes the leaf's number among the leaves instead of its node index
template <typename XT, bool kNumber>
__global__ __launch_bounds__(256) void predict_kernel(const XT* __restrict__ X, int64_t n, int F,
                                                      const NodeRec* __restrict__ nodes,
                                                      const double* __restrict__ thr,
                                                      int32_t* __restrict__ leaf) {
  const int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x;
  if (i >= n) return;
  const XT* x = X + i * F;
  int32_t node = 0;
  NodeRec r = nodes[0];
  while (r.feature >= 0) {
    node = ((double)x[r.feature] <= thr[node]) ? r.left : r.right;
    r = nodes[node];
  }
  leaf[i] = kNumber ? r.number : node;
}

void launch_predict(hipStream_t stream, const void* X, bool x64, int64_t n, int F,
                    const void* nodes, const double* thr, int32_t* leaf, bool number) {
  if (n <= 0) return;
  dim3 grid((unsigned)((n + 255) / 256));
  auto go = [&](auto kern, auto* x) {
    hipLaunchKernelGGL(kern, grid, dim3(256), 0, stream, x, n, F, (const NodeRec*)nodes, thr,
                       leaf);
    MT_HIP_CHECK(hipGetLastError());
  };
  if (x64)
    number ? go(predict_kernel<double, true>, (const double*)X)
           : go(predict_kernel<double, false>, (const double*)X);
  else
    number ? go(predict_kernel<float, true>, (const float*)X)
           : go(predict_kernel<float, false>, (const float*)X);
}

}  // namespace mt
