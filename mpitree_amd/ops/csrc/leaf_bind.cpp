// pybind11 entry points of the operators over a tree's leaves (part of ``mpitree_amd._hip``).
#include <hip/hip_runtime.h>

#include <pybind11/pybind11.h>

#include "common.h"

namespace py = pybind11;

namespace mt {

int64_t leaf_route_words(int64_t, int);
void launch_leaf_route(hipStream_t, const void*, bool, int64_t, int, int32_t*, uint32_t*, int32_t*,
                       uint32_t*);
void launch_leaf_embed(hipStream_t, int, const void*, bool, const void*, int64_t, int64_t, int64_t,
                       int, float, void*);
int64_t leaf_embed_grad_bytes(int, int64_t, int);
void launch_leaf_embed_grad(hipStream_t, int, const void*, const int32_t*, const uint32_t*,
                            const int32_t*, int64_t, int64_t, int, float, void*, void*);
int leaf_linear_small_rows();
void launch_leaf_linear_small(hipStream_t, int, const void*, int64_t, const void*, bool, int, int,
                              const void*, const void*, int, int, void*);
void launch_leaf_linear_tile(hipStream_t, int, bool, const void*, int64_t, const int32_t*,
                             const int32_t*, int64_t, int, const void*, const void*, int, int,
                             void*, void*);
int64_t leaf_linear_tile_bytes(int64_t, int);
int64_t leaf_linear_grad_bytes(int, int64_t, int, int, int);
void launch_leaf_linear_grad(hipStream_t, int, const void*, int64_t, const void*, int64_t,
                             const int32_t*, const uint32_t*, const int32_t*, int64_t, int, int,
                             int, void*, void*);

namespace {
hipStream_t S(uintptr_t s) { return reinterpret_cast<hipStream_t>(s); }
template <typename T>
T* P(uintptr_t p) {
  return reinterpret_cast<T*>(p);
}
}  // namespace

void bind_leaf(py::module_& m) {
  m.def("leaf_route_words", &leaf_route_words);
  m.def("leaf_route", [](uintptr_t s, uintptr_t ids, bool wide, int64_t n, int G, uintptr_t order,
                         uintptr_t keys, uintptr_t off, uintptr_t work) {
    launch_leaf_route(S(s), P<void>(ids), wide, n, G, P<int32_t>(order), P<uint32_t>(keys),
                      P<int32_t>(off), P<uint32_t>(work));
  });
  m.def("leaf_embed", [](uintptr_t s, int type, uintptr_t ids, bool wide, uintptr_t table,
                         int64_t stride, int64_t n, int64_t V, int D, float scale, uintptr_t y) {
    launch_leaf_embed(S(s), type, P<void>(ids), wide, P<void>(table), stride, n, V, D, scale,
                      P<void>(y));
  });
  m.def("leaf_embed_grad_bytes", &leaf_embed_grad_bytes);
  m.def("leaf_embed_grad", [](uintptr_t s, int type, uintptr_t dy, uintptr_t order, uintptr_t keys,
                              uintptr_t off, int64_t n, int64_t V, int D, float scale,
                              uintptr_t dtable, uintptr_t work) {
    launch_leaf_embed_grad(S(s), type, P<void>(dy), P<int32_t>(order), P<uint32_t>(keys),
                           P<int32_t>(off), n, V, D, scale, P<void>(dtable), P<void>(work));
  });
  m.def("leaf_linear_small_rows", &leaf_linear_small_rows);
  m.def("leaf_linear_small", [](uintptr_t s, int type, uintptr_t x, int64_t x_stride, uintptr_t ids,
                                bool wide, int n, int G, uintptr_t w, uintptr_t bias, int K, int N,
                                uintptr_t y) {
    launch_leaf_linear_small(S(s), type, P<void>(x), x_stride, P<void>(ids), wide, n, G,
                             P<void>(w), P<void>(bias), K, N, P<void>(y));
  });
  m.def("leaf_linear_tile", [](uintptr_t s, int type, bool dx, uintptr_t src, int64_t src_stride,
                               uintptr_t order, uintptr_t off, int64_t n, int G, uintptr_t w,
                               uintptr_t bias, int K, int N, uintptr_t out, uintptr_t work) {
    launch_leaf_linear_tile(S(s), type, dx, P<void>(src), src_stride, P<int32_t>(order),
                            P<int32_t>(off), n, G, P<void>(w), P<void>(bias), K, N, P<void>(out),
                            P<void>(work));
  });
  m.def("leaf_linear_tile_bytes", &leaf_linear_tile_bytes);
  m.def("leaf_linear_grad_bytes", &leaf_linear_grad_bytes);
  m.def("leaf_linear_grad", [](uintptr_t s, int type, uintptr_t x, int64_t x_stride, uintptr_t dy,
                               int64_t dy_stride, uintptr_t order, uintptr_t keys, uintptr_t off,
                               int64_t n, int G, int K, int N, uintptr_t dw, uintptr_t work) {
    launch_leaf_linear_grad(S(s), type, P<void>(x), x_stride, P<void>(dy), dy_stride,
                            P<int32_t>(order), P<uint32_t>(keys), P<int32_t>(off), n, G, K, N,
                            P<void>(dw), P<void>(work));
  });
}

}  // namespace mt
