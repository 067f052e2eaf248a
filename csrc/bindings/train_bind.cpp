// Bindings of the training ops on torch tensors (oap_mllib_amd/ops/training.py): addresses, sizes
// and the caller's stream; device -1 is host memory.  Nothing here allocates or synchronises, so
// a call can be captured into a graph.
#include <pybind11/pybind11.h>

#include <cmath>
#include <string>

#include "bindings/bindings.h"
#include "drivers/train_host.h"
#include "runtime/common.h"

namespace py = pybind11;
using namespace oap;

namespace {

// The tensors' device for the duration of a call
class DeviceGuard {
 public:
  explicit DeviceGuard(int device) {
    OAP_HIP_CHECK(hipGetDevice(&prev_));
    if (prev_ != device) {
      OAP_HIP_CHECK(hipSetDevice(device));
      changed_ = true;
    }
  }
  ~DeviceGuard() {
    if (changed_) (void)hipSetDevice(prev_);
  }
  DeviceGuard(const DeviceGuard&) = delete;
  DeviceGuard& operator=(const DeviceGuard&) = delete;

 private:
  int prev_ = 0;
  bool changed_ = false;
};

kern::Elem elem_of(const std::string& s) {
  if (s == "f32") return kern::Elem::F32;
  if (s == "bf16") return kern::Elem::BF16;
  if (s == "f16") return kern::Elem::F16;
  throw ConfigError("unknown element type '" + s + "'");
}

template <typename T>
T* at(uintptr_t p) {
  return reinterpret_cast<T*>(p);
}

// `gpu(stream)` on the device, or `host()`
template <typename G, typename H>
void on(int device, uintptr_t stream, kern::Elem e, G&& gpu, H&& host) {
  py::gil_scoped_release release;
  if (device < 0) {
    OAP_CHECK(e == kern::Elem::F32, "the host engine takes f32");
    host();
    return;
  }
  DeviceGuard guard(device);
  gpu(reinterpret_cast<hipStream_t>(stream));
}

kern::CeArgs ce_args(const std::string& elem, uintptr_t x, int64_t ldx, uintptr_t w, int64_t ldw,
                     uintptr_t bias, uintptr_t target, int64_t ignore, int64_t n, int64_t classes,
                     int64_t dim) {
  kern::CeArgs a = {};
  a.elem = elem_of(elem);
  a.x = at<const void>(x);
  a.ldx = ldx;
  a.w = at<const void>(w);
  a.ldw = ldw;
  a.bias = at<const float>(bias);
  a.target = at<const int64_t>(target);
  a.ignore = ignore;
  a.n = n;
  a.classes = classes;
  OAP_CHECK(dim >= 1 && dim <= (1 << 20), "softmax_cross_entropy: 1 to 2^20 features");
  a.dim = int(dim);
  return a;
}

}  // namespace

void register_train(py::module_& m) {
  m.def(
      "dropout",
      [](int device, uintptr_t stream, const std::string& elem, uintptr_t x, uintptr_t residual,
         uintptr_t y, int64_t n, uint64_t offset, uint64_t seed, uintptr_t seed_ptr, double p) {
        OAP_CHECK(p >= 0.0 && p <= 1.0, "dropout: p must lie in [0, 1]");
        kern::DropoutArgs a = {};
        a.x = at<const void>(x);
        a.residual = at<const void>(residual);
        a.y = at<void>(y);
        a.n = n;
        a.offset = offset;
        a.seed = seed;
        a.seed_ptr = at<const int64_t>(seed_ptr);
        a.threshold = uint64_t(std::nearbyint(p * 4294967296.0));
        a.scale = p < 1.0 ? float(1.0 / (1.0 - p)) : 0.f;
        const kern::Elem e = elem_of(elem);
        on(device, stream, e, [&](hipStream_t s) { kern::dropout(e, a, s); },
           [&] { dropout_host(a); });
      },
      py::arg("device"), py::arg("stream"), py::arg("elem"), py::arg("x"), py::arg("residual"),
      py::arg("y"), py::arg("n"), py::arg("offset"), py::arg("seed"), py::arg("seed_ptr"),
      py::arg("p"));

  m.attr("route_max_experts") = kern::kRouteMaxExperts;
  m.attr("route_max_k") = kern::kRouteMaxK;
  m.attr("route_max_groups") = kern::kRouteMaxGroups;
  m.def("route_partial_bytes", &kern::route_partial_bytes, py::arg("tokens"), py::arg("experts"));
  m.def(
      "route",
      [](int device, uintptr_t stream, const std::string& elem, uintptr_t logits, int64_t ld,
         uintptr_t bias, int64_t tokens, int experts, int k, int groups, int top_groups,
         bool sigmoid, bool renormalize, float scale, uintptr_t weights, uintptr_t indices,
         uintptr_t counts, uintptr_t partial) {
        kern::RouteArgs a = {};
        a.logits = at<const void>(logits);
        a.ld = ld;
        a.bias = at<const float>(bias);
        a.tokens = tokens;
        a.experts = experts;
        a.k = k;
        a.groups = groups;
        a.top_groups = top_groups;
        a.sigmoid = sigmoid;
        a.renormalize = renormalize;
        a.scale = scale;
        a.weights = at<float>(weights);
        a.indices = at<int32_t>(indices);
        a.counts = at<int32_t>(counts);
        a.partial = at<int32_t>(partial);
        const kern::Elem e = elem_of(elem);
        on(device, stream, e, [&](hipStream_t s) { kern::route(e, a, s); },
           [&] { route_host(a); });
      },
      py::arg("device"), py::arg("stream"), py::arg("elem"), py::arg("logits"), py::arg("ld"),
      py::arg("bias"), py::arg("tokens"), py::arg("experts"), py::arg("k"), py::arg("groups"),
      py::arg("top_groups"), py::arg("sigmoid"), py::arg("renormalize"), py::arg("scale"),
      py::arg("weights"), py::arg("indices"), py::arg("counts"), py::arg("partial"));
  m.def(
      "route_grad",
      [](int device, uintptr_t stream, const std::string& elem, uintptr_t logits, int64_t ld,
         uintptr_t weights, uintptr_t indices, uintptr_t grad, int64_t tokens, int experts, int k,
         bool sigmoid, bool renormalize, float scale, uintptr_t grad_logits) {
        kern::RouteGradArgs a = {};
        a.logits = at<const void>(logits);
        a.ld = ld;
        a.weights = at<const float>(weights);
        a.indices = at<const int32_t>(indices);
        a.grad = at<const float>(grad);
        a.tokens = tokens;
        a.experts = experts;
        a.k = k;
        a.sigmoid = sigmoid;
        a.renormalize = renormalize;
        a.scale = scale;
        a.grad_logits = at<void>(grad_logits);
        const kern::Elem e = elem_of(elem);
        on(device, stream, e, [&](hipStream_t s) { kern::route_grad(e, a, s); },
           [&] { route_grad_host(a); });
      },
      py::arg("device"), py::arg("stream"), py::arg("elem"), py::arg("logits"), py::arg("ld"),
      py::arg("weights"), py::arg("indices"), py::arg("grad"), py::arg("tokens"),
      py::arg("experts"), py::arg("k"), py::arg("sigmoid"), py::arg("renormalize"),
      py::arg("scale"), py::arg("grad_logits"));

  // workspace bytes (the addresses decide whether an operand is read in place)
  m.def("softmax_ce_forward_bytes",
        [](const std::string& elem, uintptr_t x, int64_t ldx, uintptr_t w, int64_t ldw,
           uintptr_t bias, int64_t n, int64_t classes, int64_t dim, bool train) {
          kern::CeArgs a = ce_args(elem, x, ldx, w, ldw, bias, 0, 0, n, classes, dim);
          a.train = train;
          return kern::ce_forward_bytes(a);
        });
  m.def("softmax_ce_backward_bytes",
        [](const std::string& elem, uintptr_t x, int64_t ldx, uintptr_t w, int64_t ldw,
           uintptr_t bias, int64_t n, int64_t classes, int64_t dim, bool want_dx, bool want_dw,
           bool want_db) {
          return kern::ce_backward_bytes(
              ce_args(elem, x, ldx, w, ldw, bias, 0, 0, n, classes, dim), want_dx, want_dw,
              want_db);
        });
  // (rows of a turn, classes of a piece, fp32 operands split): how a call is divided
  m.def("softmax_ce_plan",
        [](const std::string& elem, uintptr_t x, int64_t ldx, uintptr_t w, int64_t ldw,
           uintptr_t bias, int64_t n, int64_t classes, int64_t dim, bool grad) {
          const kern::CePlan p =
              kern::ce_plan(ce_args(elem, x, ldx, w, ldw, bias, 0, 0, n, classes, dim), grad);
          return py::make_tuple(p.rows, p.classes, p.split);
        });
  m.def("softmax_ce_forward",
        [](int device, uintptr_t stream, const std::string& elem, uintptr_t x, int64_t ldx,
           uintptr_t w, int64_t ldw, uintptr_t bias, uintptr_t target, int64_t ignore, int64_t n,
           int64_t classes, int64_t dim, bool train, uintptr_t loss, uintptr_t stat,
           uintptr_t miss, uintptr_t total, bool mean, uintptr_t work) {
          kern::CeArgs a = ce_args(elem, x, ldx, w, ldw, bias, target, ignore, n, classes, dim);
          a.train = train;
          on(device, stream, a.elem,
             [&](hipStream_t s) {
               kern::ce_forward(a, at<float>(loss), at<float2>(stat), at<float>(miss),
                                at<float>(total), mean, at<void>(work), s);
             },
             [&] {
               ce_forward_host(a, at<float>(loss), at<float2>(stat), at<float>(total), mean);
             });
        });
  m.def("softmax_ce_backward",
        [](int device, uintptr_t stream, const std::string& elem, uintptr_t x, int64_t ldx,
           uintptr_t w, int64_t ldw, uintptr_t bias, uintptr_t target, int64_t ignore, int64_t n,
           int64_t classes, int64_t dim, uintptr_t stat, uintptr_t miss, uintptr_t grad,
           bool per_row, bool mean, uintptr_t dx, uintptr_t dw, uintptr_t db, uintptr_t work) {
          const kern::CeArgs a =
              ce_args(elem, x, ldx, w, ldw, bias, target, ignore, n, classes, dim);
          on(device, stream, a.elem,
             [&](hipStream_t s) {
               kern::ce_backward(a, at<const float2>(stat), at<const float>(miss),
                                 at<const float>(grad), per_row, mean, at<void>(dx), at<void>(dw),
                                 at<float>(db), at<void>(work), s);
             },
             [&] {
               ce_backward_host(a, at<const float2>(stat), at<const float>(grad), per_row, mean,
                                at<float>(dx), at<float>(dw), at<float>(db));
             });
        });
}
