// Host side of the MXFP4 operators (lumen/ops/mxfp4.py): results, streams and autograd of the launchers in seqmix/mx*.hip.
//
// A call on few rows takes less time on the GPU than on the host, and a gradient runs on a thread of its own, where interpreted
// code finds cold caches.  So what happens on every call stands here: from Python a product of 16 rows took 7.8 us of host time,
// it and its gradient 90.  The launchers are in another library (lumen/_C_seqmix.so), whose loader hands their addresses over once.
#include <torch/extension.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime.h>

#include <array>
#include <optional>
#include <string>
#include <vector>

namespace {

using at::Tensor;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

typedef hipError_t (*QuantizeFn)(int, const void*, long long, void*, void*, int, int, hipStream_t);
typedef hipError_t (*DequantizeFn)(int, const void*, const void*, void*, int, int, hipStream_t);
typedef hipError_t (*LinearFn)(int, const void*, long long, const void*, const void*, const void*, void*, int, int, int, int, int, hipStream_t);
typedef hipError_t (*GradFn)(int, const void*, long long, const void*, const void*, void*, int, int, int, int, hipStream_t);
typedef hipError_t (*MatmulFn)(int, const void*, const void*, const void*, const void*, const void*, void*, int, int, int, int, int, hipStream_t);

enum Launcher { kQuantize, kDequantize, kLinear, kRows, kGrad, kRowsGrad, kMatmul, kRowsMatmul, kLaunchers };
std::array<void*, kLaunchers> launcher{};

void mx_launchers(const std::vector<long long>& addresses) {
  TORCH_CHECK(addresses.size() == kLaunchers, "mx_launchers: ", int(kLaunchers), " addresses");
  for (int i = 0; i < kLaunchers; ++i) launcher[i] = reinterpret_cast<void*>(addresses[i]);
}

template <typename F> F fn(Launcher which) {
  TORCH_CHECK(launcher[which], "MXFP4: the kernel library is not loaded");
  return reinterpret_cast<F>(launcher[which]);
}

void done(hipError_t e, const char* what) { TORCH_CHECK(e == hipSuccess, what, ": HIP error ", int(e), " (", hipGetErrorString(e), ")"); }

int code_of(at::ScalarType t, const char* what) {
  switch (t) {
    case at::kFloat: return 0;
    case at::kHalf: return 1;
    case at::kBFloat16: return 2;
    default: TORCH_CHECK_VALUE(false, what, ": ", toString(t), " is no type of its kernels");
  }
}

// the current stream of a device, which is the current device for as long as this lives
struct On {
  std::optional<c10::DeviceGuard> guard;
  hipStream_t stream;
  explicit On(const c10::Device& d) {
    if (d.index() != c10::hip::current_device()) guard.emplace(d);
    stream = c10::hip::getCurrentHIPStream(d.index()).stream();
  }
};

// codes and scales of a matrix [R, K] that lies in `data`
struct Packed {
  char *codes, *scales;
  Packed(const Tensor& data, int64_t R, int64_t K) {
    const int64_t rows = (K + 127) / 128 * R;
    TORCH_CHECK_VALUE(data.is_cuda() && data.scalar_type() == at::kByte && data.is_contiguous() && data.numel() == rows * 68,
                      "MXFP4: the data is no matrix of ", R, " x ", K);
    codes = static_cast<char*>(data.data_ptr());
    scales = codes + rows * 64;
  }
};

// x itself where its rows are contiguous and at 16-byte addresses, else a copy
struct Rows {
  Tensor t;
  const void* p;
  long long ld;
  Rows(const Tensor& x, int64_t unit, int64_t most) : t(x), p(x.data_ptr()), ld(x.size(0) == 1 ? x.size(1) : x.stride(0)) {
    if (x.stride(1) != 1 || reinterpret_cast<uintptr_t>(p) % 16 || ld % unit || ld < x.size(1) || ld > most || x.is_neg()) {
      at::NoGradGuard none;
      t = x.resolve_neg().clone(at::MemoryFormat::Contiguous);
      p = t.data_ptr(), ld = x.size(1);
    }
  }
};

constexpr int64_t kMaxLd = 1 << 22, kMaxRows = 1 << 24;
typedef std::array<int, 3> Form;          // tiles or few rows, and their two sizes (lumen/ops/mxfp4.py)

void need(const Tensor& x, const char* what) {
  TORCH_CHECK_VALUE(x.is_cuda() && x.dim() == 2 && x.size(0) <= kMaxRows, what, ": no GPU rows (at most ", kMaxRows, ")");
  TORCH_CHECK_VALUE(!x._fw_grad(0).defined(), what, ": no forward-mode derivative");
}

// 16-bit rows of K values beside the weight's data (whose size cannot tell two K of one number of panels apart); the code of their type
int need_rows(const Tensor& x, const Tensor& data, int64_t K, const char* what) {
  need(x, what);
  TORCH_CHECK_VALUE(x.size(1) == K, what, ": rows of ", x.size(1), " values against a weight of ", K);
  TORCH_CHECK_VALUE(K <= kMaxLd, what, ": rows of ", K, " values (at most ", kMaxLd, ")");
  TORCH_CHECK_VALUE(x.device() == data.device(), what, ": rows on ", x.device(), ", weight on ", data.device());
  TORCH_CHECK_VALUE(x.scalar_type() == at::kHalf || x.scalar_type() == at::kBFloat16, what, ": rows of ", toString(x.scalar_type()),
                    " (bf16 or fp16)");
  return code_of(x.scalar_type(), what);
}

// a bias [N] as the kernels read it, undefined where there is none
Tensor need_bias(const std::optional<Tensor>& bias, const Tensor& data, int64_t N, at::ScalarType type, const char* what) {
  if (!bias) return Tensor();
  TORCH_CHECK_VALUE(bias->device() == data.device() && bias->numel() == N && bias->scalar_type() == type, what, ": the bias is not [", N,
                    "] values of ", toString(type), " on ", data.device());
  return bias->resolve_neg().contiguous();
}

Tensor quantize(const Tensor& x) {
  need(x, "mxfp4_quantize");
  const int dt = code_of(x.scalar_type(), "mxfp4_quantize");
  const int64_t R = x.size(0), K = x.size(1);
  Tensor data = at::empty({(K + 127) / 128 * R * 68}, x.options().dtype(at::kByte));
  if (R) {
    const On on(x.device());
    const Packed q(data, R, K);
    const Rows r(x, dt ? 8 : 4, int64_t(1) << 40);
    done(fn<QuantizeFn>(kQuantize)(dt, r.p, r.ld, q.codes, q.scales, int(R), int(K), on.stream), "mxfp4_quantize");
  }
  return data;
}

Tensor dequantize(const Tensor& data, int64_t R, int64_t K, at::ScalarType type) {
  const Packed q(data, R, K);
  const int dt = code_of(type, "mxfp4_dequantize");
  Tensor y = at::empty({R, K}, data.options().dtype(type));
  if (R) {
    const On on(data.device());
    done(fn<DequantizeFn>(kDequantize)(dt, q.codes, q.scales, y.data_ptr(), int(R), int(K), on.stream), "mxfp4_dequantize");
  }
  return y;
}

Tensor linear(const Tensor& x, const Tensor& data, int64_t N, int64_t K, const std::optional<Tensor>& bias, const Form& f) {
  const int dt = need_rows(x, data, K, "mxfp4_linear");
  const Packed w(data, N, K);
  const Tensor b = need_bias(bias, data, N, x.scalar_type(), "mxfp4_linear");
  const int64_t M = x.size(0);
  Tensor y = at::empty({M, N}, x.options());
  if (M && N) {
    const On on(x.device());
    const Rows r(x, 8, kMaxLd);
    done(fn<LinearFn>(f[0] ? kLinear : kRows)(dt, r.p, r.ld, w.codes, w.scales, bias ? b.data_ptr() : nullptr, y.data_ptr(), int(M), int(N),
                                              int(K), f[1], f[2], on.stream), "mxfp4_linear");
  }
  return y;
}

Tensor grad(const Tensor& dy, const Tensor& data, int64_t N, int64_t K, const Form& f) {
  const int dt = need_rows(dy, data, N, "gradient of mxfp4_linear");
  const Packed w(data, N, K);
  const int64_t M = dy.size(0);
  if (!M || !N) return at::zeros({M, K}, dy.options());
  const On on(dy.device());
  Tensor dx = at::empty({M, K}, dy.options()), rows = dy;
  if (N % 8) {                             // (rows at 16-byte addresses, zeros behind them)
    at::NoGradGuard none;
    rows = at::constant_pad_nd(dy, {0, 8 - N % 8});
  }
  const Rows r(rows, 8, kMaxLd);
  done(fn<GradFn>(f[0] ? kGrad : kRowsGrad)(dt, r.p, r.ld, w.codes, w.scales, dx.data_ptr(), int(M), int(N), int(K), f[1], on.stream),
       "gradient of mxfp4_linear");
  return dx;
}

Tensor tracked(const Tensor& in, const Tensor& data, int64_t N, int64_t K, const std::optional<Tensor>& bias, const Form& f, const Form& g,
               bool back);

// y = x w^T, whose gradient is dx = dy w, and the other way round; either's gradient may be differentiated again
struct Product : torch::autograd::Node {
  SavedVariable data;
  int64_t N = 0, K = 0;
  Form f, g;
  bool back = false;                       // this node's own forward was dx = dy w
  variable_list apply(variable_list&& in) override {
    if (!in[0].defined()) return {Tensor()};
    refuse_foreign_accumulation(in[0].device());
    Tensor d;
    {
      const std::lock_guard<std::mutex> lock(mutex_);
      d = data.unpack();
    }
    return {tracked(in[0], d, N, K, std::nullopt, f, g, !back)};
  }
  void release_variables() override {
    const std::lock_guard<std::mutex> lock(mutex_);
    data.reset_data();
  }
  // A leaf's accumulation node belongs to the stream of the first of its graphs that are alive.  If that is the default stream, the engine
  // makes it wait for the capture, which no capture survives (and an error there ends the process).
  void refuse_foreign_accumulation(const c10::Device& device) const {
    const auto ours = c10::hip::getCurrentHIPStream(device.index());
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    done(hipStreamIsCapturing(ours.stream(), &status), "gradient of mxfp4_linear");
    if (status == hipStreamCaptureStatusNone) return;
    auto* node = next_edge(0).function.get();
    while (node && node->num_outputs() == 1) node = node->next_edge(0).function.get();       // (views of the leaf)
    auto* sum = dynamic_cast<torch::autograd::AccumulateGrad*>(node);
    const auto theirs = sum ? sum->stream() : std::nullopt;
    TORCH_CHECK_VALUE(!theirs || theirs->id() != 0, "gradient of mxfp4_linear: the captured pass ends at a leaf whose graph from before the "
                      "capture is alive on the default stream; drop that graph first");
  }
  std::string name() const override { return "Mxfp4LinearBackward"; }
};

Tensor tracked(const Tensor& in, const Tensor& data, int64_t N, int64_t K, const std::optional<Tensor>& bias, const Form& f, const Form& g,
               bool back) {
  Tensor out = back ? grad(in, data, N, K, g) : linear(in, data, N, K, bias, f);
  if (at::GradMode::is_enabled() && in.requires_grad()) {
    std::shared_ptr<Product> node(new Product(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(in));
    node->data = SavedVariable(data, false);
    node->N = N, node->K = K, node->f = f, node->g = g, node->back = back;
    torch::autograd::set_history(out, node);
  }
  return out;
}

Tensor mx_linear(const Tensor& x, const Tensor& data, int64_t N, int64_t K, const std::optional<Tensor>& bias, int f0, int f1, int f2) {
  return linear(x, data, N, K, bias, {f0, f1, f2});
}

Tensor mx_grad(const Tensor& dy, const Tensor& data, int64_t N, int64_t K, int g0, int g1, int g2) {
  return grad(dy, data, N, K, {g0, g1, g2});
}

Tensor mx_linear_tracked(const Tensor& x, const Tensor& data, int64_t N, int64_t K, const std::optional<Tensor>& bias, int f0, int f1, int f2,
                         int g0, int g1, int g2) {
  return tracked(x, data, N, K, bias, {f0, f1, f2}, {g0, g1, g2}, false);
}

Tensor mx_matmul(const Tensor& x, const Tensor& data, int64_t M, int64_t N, int64_t K, const std::optional<Tensor>& bias, at::ScalarType type,
                 int f0, int f1, int f2) {
  TORCH_CHECK_VALUE(x.device() == data.device(), "mxfp4_matmul: rows on ", x.device(), ", weight on ", data.device());
  const Packed a(x, M, K), w(data, N, K);
  const int dt = code_of(type, "mxfp4_matmul");
  const Tensor b = need_bias(bias, data, N, type, "mxfp4_matmul");
  Tensor y = at::empty({M, N}, x.options().dtype(type));
  if (M && N) {
    const On on(x.device());
    done(fn<MatmulFn>(f0 ? kMatmul : kRowsMatmul)(dt, a.codes, a.scales, w.codes, w.scales, bias ? b.data_ptr() : nullptr, y.data_ptr(), int(M),
                                                  int(N), int(K), f1, f2, on.stream), "mxfp4_matmul");
  }
  return y;
}

}  // namespace

void bind_mx_calls(pybind11::module_& m) {
  m.def("mx_launchers", &mx_launchers);
  m.def("mx_quantize", &quantize);
  m.def("mx_dequantize", &dequantize);
  m.def("mx_linear", &mx_linear);
  m.def("mx_linear_tracked", &mx_linear_tracked);
  m.def("mx_grad", &mx_grad);
  m.def("mx_matmul", &mx_matmul);
}
