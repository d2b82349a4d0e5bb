// py_rust.cpp — the `basalto._rust` extension module.
//
// Same Python surface as the reference's PyO3 module (crates/basalto-tree/src/interceptor.rs:
// 527-580): class PyBasaltoInterceptor() with
//   compile_and_execute(op, dtype, shape, strides, job_id, device_ptr_x, device_ptr_y,
//                       device_ptr_z)
// which releases the GIL and raises RuntimeError on failure.  Keyword-only extras of this
// build: custom_coeffs (the Rust-level `custom_coeffs`), program (a packed bst_program)
// and stream (a cudaStream_t as int).  Without stream the call is synchronous, as the
// reference's launch is; with one (0 included: torch's default stream) it is queued on that
// stream and returns at once.  The layer operators' entry points of the C ABI are bound here too, as
// functions of plain numbers: a call from Python costs less than through ctypes structures.
#include <pybind11/pybind11.h>
#include <pybind11/stl.h>

#include <optional>
#include <stdexcept>
#include <string>
#include <vector>

#include "../../include/basalto_b200.h"

namespace py = pybind11;

static void check(int rc) {
  if (rc != BST_OK) throw std::runtime_error(bst_last_error());
}

class PyBasaltoInterceptor {
 public:
  PyBasaltoInterceptor() { check(bst_interceptor_create(&h_)); }
  ~PyBasaltoInterceptor() { bst_interceptor_destroy(h_); }
  PyBasaltoInterceptor(const PyBasaltoInterceptor&) = delete;
  PyBasaltoInterceptor& operator=(const PyBasaltoInterceptor&) = delete;

  void compile_and_execute(const std::string& op, const std::string& dtype, const std::vector<int64_t>& shape,
                           const std::vector<int64_t>& strides, std::optional<std::string> job_id,
                           uint64_t device_ptr_x, uint64_t device_ptr_y, uint64_t device_ptr_z,
                           std::optional<std::vector<double>> custom_coeffs, std::optional<py::bytes> program,
                           std::optional<uint64_t> stream) {
    if (shape.empty() || shape.size() > 3)
      throw std::runtime_error("only 1-D, 2-D and 3-D are supported (shape has " + std::to_string(shape.size()) +
                               " dims)");
    if (shape.size() != strides.size()) throw std::runtime_error("shape and strides must have the same length");
    std::string prog_bytes;
    if (program) {
      prog_bytes = std::string(*program);
      if (prog_bytes.size() != sizeof(bst_program))
        throw std::runtime_error("program must be a packed bst_program of " + std::to_string(sizeof(bst_program)) +
                                 " bytes");
    }
    // A null stream makes the C ABI synchronous; the legacy default stream given explicitly (handle
    // 0, as torch reports it) is passed as CUDA's own handle for it, cudaStreamLegacy = 0x1.
    void* st = nullptr;
    if (stream) st = reinterpret_cast<void*>(*stream == 0 ? uint64_t(0x1) : *stream);
    const double* cc = custom_coeffs ? custom_coeffs->data() : nullptr;
    const int64_t nc = custom_coeffs ? int64_t(custom_coeffs->size()) : 0;
    int rc;
    {
      py::gil_scoped_release nogil;
      rc = bst_interceptor_compile_and_execute(
          h_, op.c_str(), dtype.c_str(), int32_t(shape.size()), shape.data(), strides.data(),
          job_id ? job_id->c_str() : nullptr, device_ptr_x, device_ptr_y, device_ptr_z, cc, nc,
          program ? reinterpret_cast<const bst_program*>(prog_bytes.data()) : nullptr, st);
    }
    check(rc);
  }

  int64_t cache_size() const { return bst_interceptor_cache_size(h_); }
  int64_t cache_hits() const { return bst_interceptor_cache_hits(h_); }
  std::string last_cache_key() const {
    char k[65] = {0};
    check(bst_interceptor_last_key(h_, k));
    return k;
  }

 private:
  bst_interceptor* h_ = nullptr;
};

// ---- layer operators: the C ABI with its descriptions unpacked into numbers ----------------
// Each returns the bst_status (the caller raises); addresses are integers, 0 = absent.
namespace {
using addr = uint64_t;
template <typename T = void>
T* at(addr p) {
  return reinterpret_cast<T*>(p);
}
using f32 = float;
using ints = std::vector<int64_t>;

// Fills the int64 fields of a description, in order, from a sequence.
template <typename D>
void fill(D& d, int64_t* first, const ints& v) {
  const size_t room = (reinterpret_cast<char*>(&d + 1) - reinterpret_cast<char*>(first)) / sizeof(int64_t);
  if (v.size() > room) throw std::runtime_error("too many fields");
  for (size_t i = 0; i < v.size(); ++i) first[i] = v[i];
}

bst_norm_desc norm_desc(int dtype, int param, const ints& v, double eps) {
  bst_norm_desc d{};
  d.dtype = dtype, d.param_dtype = param;
  if (v.size() > 6) throw std::runtime_error("too many fields");
  fill(d, &d.rows, v);
  d.eps = eps;
  return d;
}
bst_conv_desc conv_desc(int dtype, int param, int width, int silu, int lines, const ints& v) {
  bst_conv_desc d{};
  d.dtype = dtype, d.param_dtype = param, d.width = width, d.silu = silu, d.lines = lines;
  fill(d, &d.batch, v);
  return d;
}
bst_scan_desc scan_desc(int dtype, int softplus, const ints& v) {
  bst_scan_desc d{};
  d.dtype = dtype, d.softplus = softplus;
  fill(d, &d.batch, v);
  return d;
}

int64_t norm_workspace(int dtype, int param, const ints& v, double eps) {
  const bst_norm_desc d = norm_desc(dtype, param, v, eps);
  int64_t n = 0;
  check(bst_layer_norm_workspace(&d, &n));
  return n;
}
int norm_forward(int dtype, int param, const ints& v, double eps, addr x, addr w, addr b, addr y, addr mean,
                 addr rstd, addr stream) {
  const bst_norm_desc d = norm_desc(dtype, param, v, eps);
  return bst_layer_norm_forward(&d, at(x), at(w), at(b), at(y), at<f32>(mean), at<f32>(rstd), at(stream));
}
int norm_backward(int dtype, int param, const ints& v, double eps, addr x, addr w, addr dy, addr mean, addr rstd,
                  addr dx, addr dw, addr db, addr ws, int64_t bytes, addr stream) {
  const bst_norm_desc d = norm_desc(dtype, param, v, eps);
  return bst_layer_norm_backward(&d, at(x), at(w), at(dy), at<f32>(mean), at<f32>(rstd), at(dx), at(dw), at(db),
                                 at(ws), bytes, at(stream));
}
int64_t conv_workspace(int dtype, int param, int width, int silu, int lines, const ints& v) {
  const bst_conv_desc d = conv_desc(dtype, param, width, silu, lines, v);
  int64_t n = 0;
  check(bst_causal_conv_workspace(&d, &n));
  return n;
}
int conv_forward(int dtype, int param, int width, int silu, int lines, const ints& v, addr x, addr w, addr b,
                 addr init, addr lengths, addr y, addr final_state, addr stream) {
  const bst_conv_desc d = conv_desc(dtype, param, width, silu, lines, v);
  return bst_causal_conv_forward(&d, at(x), at(w), at(b), at(init), at<int32_t>(lengths), at(y), at(final_state),
                                 at(stream));
}
int conv_backward(int dtype, int param, int width, int silu, int lines, const ints& v, addr x, addr w, addr b,
                  addr init, addr lengths, addr dy, addr dfinal, addr dx, addr dw, addr db, addr dinit, addr ws,
                  int64_t bytes, addr stream) {
  const bst_conv_desc d = conv_desc(dtype, param, width, silu, lines, v);
  return bst_causal_conv_backward(&d, at(x), at(w), at(b), at(init), at<int32_t>(lengths), at(dy), at(dfinal), at(dx),
                                  at(dw), at(db), at(dinit), at(ws), bytes, at(stream));
}
int conv_step(int dtype, int param, int width, int silu, int64_t batch, int64_t channels, int64_t x_batch,
              int64_t y_batch, addr x, addr state, int64_t state_batch, addr w, addr b, addr y, addr out,
              int64_t out_batch, addr stream) {
  bst_conv_desc d{};
  d.dtype = dtype, d.param_dtype = param, d.width = width, d.silu = silu;
  d.batch = batch, d.length = 1, d.channels = channels, d.x_batch = x_batch, d.y_batch = y_batch;
  return bst_causal_conv_step(&d, at(x), at(state), state_batch, at(w), at(b), at(y), at(out), out_batch, at(stream));
}
int64_t scan_workspace(int dtype, int softplus, const ints& v, int what) {
  const bst_scan_desc d = scan_desc(dtype, softplus, v);
  int64_t n = 0;
  check(bst_scan_workspace(&d, what, &n));
  return n;
}
int scan_forward(int dtype, int softplus, const ints& v, addr u, addr delta, addr A, addr B, addr C, addr D, addr z,
                 addr bias, addr init, addr lengths, addr y, addr final_state, addr saved, addr stream) {
  const bst_scan_desc d = scan_desc(dtype, softplus, v);
  return bst_scan_forward(&d, at(u), at(delta), at<f32>(A), at(B), at(C), at<f32>(D), at(z), at<f32>(bias),
                          at<f32>(init), at<int32_t>(lengths), at(y), at<f32>(final_state), at(saved), at(stream));
}
int scan_backward(int dtype, int softplus, const ints& v, addr u, addr delta, addr A, addr B, addr C, addr D, addr z,
                  addr bias, addr lengths, addr dy, addr dfinal, addr saved, addr du, addr ddelta, addr dA, addr dB,
                  addr dC, addr dD, addr dz, addr dbias, addr dinit, addr ws, int64_t bytes, addr stream) {
  const bst_scan_desc d = scan_desc(dtype, softplus, v);
  return bst_scan_backward(&d, at(u), at(delta), at<f32>(A), at(B), at(C), at<f32>(D), at(z), at<f32>(bias),
                           at<int32_t>(lengths), at(dy), at<f32>(dfinal), at(saved), at(du), at(ddelta), at<f32>(dA),
                           at(dB), at(dC), at<f32>(dD), at(dz), at<f32>(dbias), at<f32>(dinit), at(ws), bytes,
                           at(stream));
}
int scan_step(int dtype, int softplus, int64_t batch, int64_t channels, int64_t states, int64_t groups, int64_t ub,
              int64_t db, int64_t zb, int64_t yb, int64_t Bb, int64_t Bg, int64_t Cb, int64_t Cg, addr u, addr delta,
              addr A, addr B, addr C, addr D, addr z, addr bias, addr state, int64_t sb, int64_t sc, addr y, addr out,
              int64_t ob, int64_t oc, addr stream) {
  bst_scan_desc d{};
  d.dtype = dtype, d.softplus = softplus;
  d.batch = batch, d.length = 1, d.channels = channels, d.states = states, d.groups = groups;
  d.u_batch = ub, d.delta_batch = db, d.z_batch = zb, d.y_batch = yb;
  d.B_batch = Bb, d.B_group = Bg, d.C_batch = Cb, d.C_group = Cg;
  return bst_scan_step(&d, at(u), at(delta), at<f32>(A), at(B), at(C), at<f32>(D), at(z), at<f32>(bias),
                       at<f32>(state), sb, sc, at(y), at<f32>(out), ob, oc, at(stream));
}
}  // namespace

PYBIND11_MODULE(_rust, m) {
  m.doc() = "B200-native Basalto interceptor (C++ host over sm_100a stencil kernels)";
  py::class_<PyBasaltoInterceptor>(m, "PyBasaltoInterceptor")
      .def(py::init<>())
      .def("compile_and_execute", &PyBasaltoInterceptor::compile_and_execute, py::arg("op"), py::arg("dtype"),
           py::arg("shape"), py::arg("strides"), py::arg("job_id"), py::arg("device_ptr_x"),
           py::arg("device_ptr_y"), py::arg("device_ptr_z"), py::kw_only(), py::arg("custom_coeffs") = py::none(),
           py::arg("program") = py::none(), py::arg("stream") = py::none())
      .def("cache_size", &PyBasaltoInterceptor::cache_size)
      .def("cache_hits", &PyBasaltoInterceptor::cache_hits)
      .def("last_cache_key", &PyBasaltoInterceptor::last_cache_key);
  m.def("abi_version", &bst_abi_version);
  m.def("launch_count", &bst_launch_count);
  m.def("extract_radius", [](const std::string& op) { return bst_extract_radius(op.c_str()); });
  m.def("layer_norm_workspace", &norm_workspace);
  m.def("layer_norm_forward", &norm_forward);
  m.def("layer_norm_backward", &norm_backward);
  m.def("causal_conv_workspace", &conv_workspace);
  m.def("causal_conv_forward", &conv_forward);
  m.def("causal_conv_backward", &conv_backward);
  m.def("causal_conv_step", &conv_step);
  m.def("scan_workspace", &scan_workspace);
  m.def("scan_forward", &scan_forward);
  m.def("scan_backward", &scan_backward);
  m.def("scan_step", &scan_step);
  m.attr("PROGRAM_NBYTES") = py::int_(sizeof(bst_program));
}
