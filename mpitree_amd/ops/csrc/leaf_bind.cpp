// pybind11 entry points of the operators over a tree's leaves (part of ``mpitree_amd._hip``).
#include <hip/hip_runtime.h>

#include <pybind11/pybind11.h>

#include <algorithm>
#include <initializer_list>

#include "leaf.h"

namespace py = pybind11;

namespace mt {

int64_t leaf_route_words(int64_t, int);
void launch_leaf_route(hipStream_t, const void*, bool, int64_t, int, int32_t*, uint32_t*, int32_t*,
                       uint32_t*);
void launch_leaf_embed(hipStream_t, int, const void*, bool, const void*, int64_t, int64_t, int64_t,
                       int, float, void*);
int64_t leaf_embed_grad_bytes(int, int64_t, int);
void launch_leaf_embed_grad(hipStream_t, int, const void*, int64_t, const int32_t*, const uint32_t*,
                            const int32_t*, int64_t, int64_t, int, float, void*, void*);
int leaf_linear_small_rows();
void launch_leaf_linear_small(hipStream_t, int, const void*, int64_t, const void*, bool, int, int,
                              const void*, const void*, int, int, void*);
int64_t leaf_linear_bytes(int, const void*, int64_t, const void*, int64_t, int, int, int);
void launch_leaf_linear(hipStream_t, int, const void*, int64_t, const int32_t*, const int32_t*,
                        int64_t, int, const void*, const void*, int, int, void*, void*);
int64_t leaf_linear_grad_bytes(int, const void*, int64_t, const void*, int64_t, const void*,
                               int64_t, int, int, int, bool, bool, bool);
void launch_leaf_linear_grad(hipStream_t, int, const void*, int64_t, const void*, int64_t,
                             const int32_t*, const uint32_t*, const int32_t*, int64_t, int,
                             const void*, int, int, void*, void*, void*, void*);

namespace {
hipStream_t S(uintptr_t s) { return reinterpret_cast<hipStream_t>(s); }
template <typename T>
T* P(uintptr_t p) {
  return reinterpret_cast<T*>(p);
}
}  // namespace

// Launches go to the current device: the operands' one, for the length of a call.
class OnDevice {
 public:
  explicit OnDevice(int dev) : dev_(dev) {
    MT_HIP_CHECK(hipGetDevice(&was_));
    if (was_ != dev_) MT_HIP_CHECK(hipSetDevice(dev_));
  }
  ~OnDevice() {
    if (was_ != dev_) (void)hipSetDevice(was_);
  }

 private:
  int dev_, was_ = 0;
};

// Operands that a launch of `n` rows reads or writes. A tensor without memory of its own (a wrapper
// of another one) has the address 0.
void need(int64_t n, std::initializer_list<uintptr_t> operands) {
  if (n > 0)
    for (const uintptr_t p : operands)
      if (p == 0) throw std::runtime_error("leaf operator: an operand has no memory of its own");
}

// A route in one int32 buffer: order [n], keys [n], offsets [G + 2].
struct Route {
  int32_t* order;
  uint32_t* keys;
  int32_t* off;
  Route(uintptr_t buf, int64_t n)
      : order(P<int32_t>(buf)), keys(P<uint32_t>(buf) + n), off(P<int32_t>(buf) + 2 * n) {}
};
int64_t route_len(int64_t n, int64_t G) { return 2 * n + G + 2; }
int64_t pad16(int64_t bytes) { return (bytes + 15) / 16 * 16; }

void bind_leaf(py::module_& m) {
  m.def("leaf_route_len", &route_len);      // int32 words of a route
  m.def("leaf_route_words", &leaf_route_words);  // ... of the scratch of its sort
  m.def("leaf_route", [](int dev, uintptr_t s, uintptr_t ids, bool wide, int64_t n, int G,
                         uintptr_t buf, uintptr_t work) {
    need(1, {buf});
    need(n, {ids});
    const OnDevice on(dev);
    const Route r(buf, n);
    launch_leaf_route(S(s), P<void>(ids), wide, n, G, r.order, r.keys, r.off, P<uint32_t>(work));
  });
  m.def("leaf_embed", [](int dev, uintptr_t s, int type, uintptr_t ids, bool wide, uintptr_t table,
                         int64_t stride, int64_t n, int64_t V, int D, float scale, uintptr_t y) {
    need(n, {ids, table, y});
    const OnDevice on(dev);
    launch_leaf_embed(S(s), type, P<void>(ids), wide, P<void>(table), stride, n, V, D, scale,
                      P<void>(y));
  });
  // the sums of dy by leaf; ids: they are sorted first, into `work`; else `route` holds the sort
  m.def("leaf_embed_grad_bytes", [](int type, int64_t n, int G, int D, bool routed) {
    return leaf_embed_grad_bytes(type, n, D) +
           (routed ? 0 : pad16(4 * leaf_route_words(n, G)) + pad16(4 * route_len(n, G)));
  });
  m.def("leaf_embed_grad", [](int dev, uintptr_t s, int type, uintptr_t dy, int64_t dy_stride,
                              uintptr_t ids, bool wide, uintptr_t route, int64_t n, int G, int D,
                              float scale, uintptr_t dtable, uintptr_t work) {
    need(1, {dtable, work});
    need(n, {dy, route | ids});
    const OnDevice on(dev);
    if (route == 0) {
      route = work + pad16(4 * leaf_route_words(n, G));
      const Route r(route, n);
      launch_leaf_route(S(s), P<void>(ids), wide, n, G, r.order, r.keys, r.off,
                        P<uint32_t>(work));
      work = route + pad16(4 * route_len(n, G));
    }
    const Route r(route, n);
    launch_leaf_embed_grad(S(s), type, P<void>(dy), dy_stride, r.order, r.keys, r.off, n, G, D,
                           scale, P<void>(dtable), P<void>(work));
  });
  m.attr("LEAF_LINEAR_SMALL_ROWS") = leaf_linear_small_rows();
  m.def("leaf_linear_small", [](int dev, uintptr_t s, int type, uintptr_t x, int64_t x_stride,
                                uintptr_t ids, bool wide, int n, int G, uintptr_t w,
                                uintptr_t bias, int K, int N, uintptr_t y) {
    need(n, {x, ids, w, y});
    const OnDevice on(dev);
    launch_leaf_linear_small(S(s), type, P<void>(x), x_stride, P<void>(ids), wide, n, G,
                             P<void>(w), P<void>(bias), K, N, P<void>(y));
  });
  // ids != 0: the rows are sorted into `route` first; else it holds the sort (routed)
  m.def("leaf_linear_bytes", [](int type, uintptr_t x, int64_t x_stride, uintptr_t w, int64_t n,
                                int G, int K, int N, bool routed) {
    return std::max(routed ? 0 : 4 * leaf_route_words(n, G),
                    leaf_linear_bytes(type, P<void>(x), x_stride, P<void>(w), n, G, K, N));
  });
  m.def("leaf_linear", [](int dev, uintptr_t s, int type, uintptr_t x, int64_t x_stride,
                          uintptr_t ids, bool wide, uintptr_t route, int64_t n, int G, uintptr_t w,
                          uintptr_t bias, int K, int N, uintptr_t y, uintptr_t work) {
    need(n, {x, route, w, y});
    const OnDevice on(dev);
    const Route r(route, n);
    if (ids != 0)
      launch_leaf_route(S(s), P<void>(ids), wide, n, G, r.order, r.keys, r.off,
                        P<uint32_t>(work));
    launch_leaf_linear(S(s), type, P<void>(x), x_stride, r.order, r.off, n, G, P<void>(w),
                       P<void>(bias), K, N, P<void>(y), P<void>(work));
  });
  // dx, dw and db, each where its address is not 0
  m.def("leaf_linear_grad_bytes", [](int type, uintptr_t x, int64_t x_stride, uintptr_t dy,
                                     int64_t dy_stride, uintptr_t w, int64_t n, int G, int K, int N,
                                     bool dx, bool dw, bool db) {
    return leaf_linear_grad_bytes(type, P<void>(x), x_stride, P<void>(dy), dy_stride, P<void>(w), n,
                                  G, K, N, dx, dw, db);
  });
  m.def("leaf_linear_grad", [](int dev, uintptr_t s, int type, uintptr_t x, int64_t x_stride,
                               uintptr_t dy, int64_t dy_stride, uintptr_t route, int64_t n, int G,
                               uintptr_t w, int K, int N, uintptr_t dx, uintptr_t dw, uintptr_t db,
                               uintptr_t work) {
    need(1, {route});
    need(n, {x, dy, w});
    const OnDevice on(dev);
    const Route r(route, n);
    launch_leaf_linear_grad(S(s), type, P<void>(x), x_stride, P<void>(dy), dy_stride, r.order,
                            r.keys, r.off, n, G, P<void>(w), K, N, P<void>(dx), P<void>(dw),
                            P<void>(db), P<void>(work));
  });
}

}  // namespace mt
