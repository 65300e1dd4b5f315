// module.cpp -- pybind11/torch binding of libgicc (opengda_b200._C).
// Tensors are validated here; the kernels themselves live in libgicc.so.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/CUDAGraphsUtils.cuh>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <unordered_set>
#include <vector>

#include "gicc/config.hpp"
#include "gicc/error.hpp"
#include "gicc/ops.hpp"

namespace {

cudaStream_t cur_stream() { return at::cuda::getCurrentCUDAStream().stream(); }

void check_cuda_bf16(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK(t.scalar_type() == at::kBFloat16, name, " must be bfloat16");
  TORCH_CHECK(t.dim() == 2, name, " must be 2-D");
  TORCH_CHECK(t.stride(1) == 1, name, " must be row-major (stride(1) == 1)");
}

at::Tensor gemm(const at::Tensor& A, const at::Tensor& B, c10::optional<at::Tensor> out, double alpha, bool out_f32,
                int64_t bn) {
  check_cuda_bf16(A, "A");
  check_cuda_bf16(B, "B");
  TORCH_CHECK(A.size(1) == B.size(1), "A[M,K] and B[N,K] must share K");
  const c10::cuda::CUDAGuard g(A.device());
  const int64_t M = A.size(0), N = B.size(0), K = A.size(1);
  at::Tensor C;
  if (out.has_value()) {
    C = *out;
    TORCH_CHECK(C.is_cuda() && C.dim() == 2 && C.size(0) == M && C.size(1) == N && C.stride(1) == 1, "bad out");
    TORCH_CHECK(C.scalar_type() == (out_f32 ? at::kFloat : at::kBFloat16), "out dtype mismatch");
  } else {
    C = at::empty({M, N}, A.options().dtype(out_f32 ? at::kFloat : at::kBFloat16));
  }
  gicc::ops::gemm_bf16(A.data_ptr(), B.data_ptr(), C.data_ptr(), (int)M, (int)N, (int)K, A.stride(0), B.stride(0),
                       C.stride(0), out_f32, (float)alpha, (int)bn, cur_stream());
  return C;
}

at::Tensor gemm_fp32(const at::Tensor& A, const at::Tensor& B, c10::optional<at::Tensor> out, double alpha,
                     int64_t bn) {
  TORCH_CHECK(A.is_cuda() && B.is_cuda() && A.scalar_type() == at::kFloat && B.scalar_type() == at::kFloat &&
                  A.dim() == 2 && B.dim() == 2 && A.stride(1) == 1 && B.stride(1) == 1,
              "A[M,K], B[N,K]: fp32 CUDA matrices with unit column stride");
  TORCH_CHECK(A.size(1) == B.size(1), "A[M,K] and B[N,K] must share K");
  const c10::cuda::CUDAGuard g(A.device());
  const int64_t M = A.size(0), N = B.size(0), K = A.size(1);
  at::Tensor C;
  if (out.has_value()) {
    C = *out;
    TORCH_CHECK(C.is_cuda() && C.dim() == 2 && C.size(0) == M && C.size(1) == N && C.stride(1) == 1 &&
                    C.scalar_type() == at::kFloat, "bad out");
  } else {
    C = at::empty({M, N}, A.options());
  }
  at::Tensor work = at::empty({(M + N) * 3 * K}, A.options());
  gicc::ops::gemm_fp32(A.data_ptr<float>(), B.data_ptr<float>(), C.data_ptr<float>(), (int)M, (int)N, (int)K,
                       A.stride(0), B.stride(0), C.stride(0), (float)alpha, work.data_ptr<float>(), cur_stream(),
                       (int)bn);
  return C;
}

void gemm_tile_done_selftest(const at::Tensor& A, const at::Tensor& B, const at::Tensor& counters, int64_t skew_ns) {
  check_cuda_bf16(A, "A");
  check_cuda_bf16(B, "B");
  TORCH_CHECK(A.is_contiguous() && B.is_contiguous() && A.size(1) == B.size(1), "A[M,K], B[N,K] contiguous");
  TORCH_CHECK(counters.is_cuda() && counters.scalar_type() == at::kInt && counters.is_contiguous(), "int32 counters");
  const c10::cuda::CUDAGuard g(A.device());
  gicc::ops::gemm_tile_done_selftest(A.data_ptr(), B.data_ptr(), (int)A.size(0), (int)B.size(0), (int)A.size(1),
                                     static_cast<uint32_t*>(counters.data_ptr()), (uint32_t)skew_ns, cur_stream());
}

// ---- projections (ffn.cu, lora.cu) ----
int fmt_of(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf, name, " must be bfloat16 or float16");
  return t.scalar_type() == at::kBFloat16 ? 1 : 0;
}
// A row-major matrix of `like`'s type and device with 16-byte aligned rows.
void check_rows(const at::Tensor& t, const char* name, const at::Tensor& like) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK(t.device() == like.device(), name, " must be on the inputs' device");
  TORCH_CHECK(t.scalar_type() == like.scalar_type(), name, " must have the inputs' dtype");
  TORCH_CHECK(t.dim() == 2, name, " must be 2-D");
  TORCH_CHECK(t.size(0) <= INT32_MAX && t.size(1) <= INT32_MAX / 2, name, " is too large");
  TORCH_CHECK(t.size(1) <= 1 || t.stride(1) == 1, name, " must be row-major (stride(1) == 1)");
  TORCH_CHECK(t.size(0) <= 1 || t.stride(0) >= t.size(1), name, " must have rows that do not overlap");
}
// The row pitch; a single row's stride says nothing, so it counts as dense.
long long pitch_of(const at::Tensor& t) { return t.size(0) <= 1 ? std::max<int64_t>((t.size(1) + 7) / 8 * 8, 8) : t.stride(0); }

// Whether `out` (row-major matrix) may share memory with `in`: their address ranges meet, and they
// are not column ranges of one buffer that lie side by side.
bool may_overlap(const at::Tensor& out, const at::Tensor& in) {
  auto bytes = [](const at::Tensor& t) {
    int64_t last = 0;
    for (int64_t d = 0; d < t.dim(); ++d) last += (t.size(d) - 1) * t.stride(d);
    return (last + 1) * (int64_t)t.element_size();
  };
  if (out.numel() == 0 || in.numel() == 0) return false;
  const char *a = static_cast<const char*>(out.data_ptr()), *b = static_cast<const char*>(in.data_ptr());
  if (a + bytes(out) <= b || b + bytes(in) <= a) return false;
  if (out.dim() == 2 && in.dim() == 2 && out.size(0) > 1 && in.size(0) > 1 && out.stride(0) == in.stride(0)) {
    const int64_t pitch = out.stride(0) * (int64_t)out.element_size();
    const int64_t at = ((a - b) % pitch + pitch) % pitch;  // out's first byte within a row of in's
    return at < in.size(1) * (int64_t)in.element_size() || at + out.size(1) * (int64_t)out.element_size() > pitch;
  }
  return true;
}

at::Tensor out_or_empty(const c10::optional<at::Tensor>& out, int64_t rows, int64_t cols, const at::Tensor& like,
                        std::initializer_list<at::Tensor> inputs) {
  if (!out.has_value()) return at::empty({rows, cols}, like.options());
  check_rows(*out, "out", like);
  TORCH_CHECK(out->size(0) == rows && out->size(1) == cols, "out has the wrong shape");
  for (const auto& t : inputs) TORCH_CHECK(!may_overlap(*out, t), "out must not overlap an input");
  return *out;
}

// Callers that would lose the launch or a derivative without a word.  torch.jit.trace records the
// allocation of the output and not what fills it.  A dual tensor does not require a gradient and has a
// valid pointer: its tangent would be dropped.
void check_caller(const char* who, std::initializer_list<at::Tensor> tensors) {
  TORCH_CHECK(!torch::jit::tracer::isTracing(), who, " cannot be traced: torch.jit.trace would record an empty result");
  for (const auto& t : tensors)
    TORCH_CHECK(!t.defined() || !t._fw_grad(0).defined(), who, " has no forward-mode derivative: an argument carries a tangent");
}

std::tuple<at::Tensor, at::Tensor> gated_linear(const at::Tensor& x, const at::Tensor& w_gate, const at::Tensor& w_up,
                                                int64_t kind, bool save, c10::optional<at::Tensor> out, int64_t tile) {
  check_caller("gated_linear", {x, w_gate, w_up, out.value_or(at::Tensor())});
  const int fmt = fmt_of(x, "x");
  check_rows(x, "x", x);
  check_rows(w_gate, "w_gate", x);
  check_rows(w_up, "w_up", x);
  const int64_t T = x.size(0), H = x.size(1), I = w_gate.size(0);
  TORCH_CHECK(w_gate.size(1) == H && w_up.size(1) == H && w_up.size(0) == I,
              "x[T,H], w_gate[I,H], w_up[I,H] must share H and I");
  const c10::cuda::CUDAGuard g(x.device());
  at::Tensor h = out_or_empty(out, T, I, x, {x, w_gate, w_up});
  at::Tensor saved;
  if (save)
    saved = at::empty({T > 0 ? (int64_t)gicc::ops::gated_saved_floats((int)T, (int)I) : 0}, x.options().dtype(at::kFloat));
  if (T > 0)
    gicc::ops::gated_linear(x.data_ptr(), w_gate.data_ptr(), w_up.data_ptr(), h.data_ptr(), (int)T, (int)H, (int)I,
                            pitch_of(x), pitch_of(w_gate), pitch_of(w_up), T == 1 ? std::max<int64_t>(I, h.stride(0)) : h.stride(0),
                            (int)kind, fmt, save ? saved.data_ptr<float>() : nullptr, (int)tile, cur_stream());
  return {h, saved};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> gated_linear_backward(const at::Tensor& dh, const at::Tensor& x,
                                                                     const at::Tensor& w_gate, const at::Tensor& w_up,
                                                                     const at::Tensor& saved, int64_t kind, bool need_dx,
                                                                     bool need_dw, int64_t tile) {
  check_caller("gated_linear_backward", {dh, x, w_gate, w_up, saved});
  const int fmt = fmt_of(x, "x");
  check_rows(x, "x", x);
  check_rows(dh, "dh", x);
  check_rows(w_gate, "w_gate", x);
  check_rows(w_up, "w_up", x);
  const int64_t T = x.size(0), H = x.size(1), I = w_gate.size(0);
  TORCH_CHECK(w_gate.size(1) == H && w_up.size(1) == H && w_up.size(0) == I && dh.size(0) == T && dh.size(1) == I,
              "dh[T,I], x[T,H], w_gate[I,H], w_up[I,H] must share T, H and I");
  TORCH_CHECK(saved.is_cuda() && saved.device() == x.device() && saved.scalar_type() == at::kFloat && saved.is_contiguous() &&
                  saved.numel() == (T > 0 ? (int64_t)gicc::ops::gated_saved_floats((int)T, (int)I) : 0),
              "saved must be what gated_linear_forward kept for these shapes");
  const c10::cuda::CUDAGuard g(x.device());
  at::Tensor dx, dwg, dwu;
  if (need_dx) dx = at::empty({T, H}, x.options());
  if (need_dw) {  // apart: one weight's gradient may be freed or overwritten while the other's lives
    dwg = T > 0 ? at::empty({I, H}, x.options()) : at::zeros({I, H}, x.options());
    dwu = T > 0 ? at::empty({I, H}, x.options()) : at::zeros({I, H}, x.options());
  }
  if (T > 0 && (need_dx || need_dw)) {
    at::Tensor work = at::empty({(int64_t)gicc::ops::gated_grad_bytes((int)T, (int)I)},
                                 x.options().dtype(at::kByte));
    gicc::ops::gated_linear_backward(dh.data_ptr(), x.data_ptr(), w_gate.data_ptr(), w_up.data_ptr(), saved.data_ptr<float>(),
                                     work.data_ptr(), need_dx ? dx.data_ptr() : nullptr, need_dw ? dwg.data_ptr() : nullptr,
                                     need_dw ? dwu.data_ptr() : nullptr, (int)T, (int)H, (int)I,
                                     T == 1 ? std::max<int64_t>(I, dh.stride(0)) : dh.stride(0), pitch_of(x),
                                     pitch_of(w_gate), pitch_of(w_up), H, H, (int)kind, fmt, (int)tile, cur_stream());
  }
  return {dx, dwg, dwu};
}

// The autograd node (C++, so that neither pass takes the interpreter's lock for its own work).
struct GatedLinearFn : public torch::autograd::Function<GatedLinearFn> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x, const at::Tensor& w_gate,
                            const at::Tensor& w_up, int64_t kind) {
    auto hs = gated_linear(x, w_gate, w_up, kind, true, c10::nullopt, 0);
    ctx->save_for_backward({x, w_gate, w_up, std::get<1>(hs)});
    ctx->saved_data["kind"] = kind;
    return std::get<0>(hs);
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const bool need_x = ctx->needs_input_grad(0), need_g = ctx->needs_input_grad(1), need_u = ctx->needs_input_grad(2);
    torch::autograd::variable_list out(4);
    if (!grads[0].defined()) return out;
    std::tuple<at::Tensor, at::Tensor, at::Tensor> d;
    {
      const at::AutoGradMode off(false);
      d = gated_linear_backward(grads[0].contiguous(), saved[0], saved[1], saved[2], saved[3], ctx->saved_data["kind"].toInt(),
                                need_x, need_g || need_u, 0);
    }
    if (need_x) out[0] = std::get<0>(d);
    if (need_g) out[1] = std::get<1>(d);
    if (need_u) out[2] = std::get<2>(d);
    if (at::GradMode::is_enabled()) {  // create_graph: there is no second derivative to go through
      torch::autograd::variable_list defined;
      for (const auto& t : out)
        if (t.defined()) defined.push_back(t.detach().requires_grad_(true));
      torch::autograd::DelayedError error("gated_linear: the backward pass is not differentiable", defined.size());
      defined = error.apply(std::move(defined));
      size_t k = 0;
      for (auto& t : out)
        if (t.defined()) t = defined[k++];
    }
    return out;
  }
};

// During a capture: refuses inputs whose autograd graph has a node made on the default stream, as it is for
// a parameter (given itself, or as the source of an input) while a graph from outside the capture is alive.
// The engine would run that node there, and a default stream that waits for a captured one breaks the
// capture half way through.  Nodes of other streams (a warm-up's, as in torch.cuda.make_graphed_callables) are
// joined by the engine.
void check_captured_graph(std::initializer_list<at::Tensor> inputs) {
  using torch::autograd::Node;
  std::vector<std::shared_ptr<Node>> roots;
  for (const auto& t : inputs)
    if (t.requires_grad()) {
      auto node = t.is_leaf() ? torch::autograd::impl::try_get_grad_accumulator(t) : t.grad_fn();
      if (node) roots.push_back(std::move(node));
    }
  std::vector<Node*> todo;
  std::unordered_set<Node*> seen;
  for (const auto& n : roots)
    if (seen.insert(n.get()).second) todo.push_back(n.get());
  while (!todo.empty()) {
    Node* n = todo.back();
    todo.pop_back();
    const auto stream = n->stream();
    TORCH_CHECK(!stream.has_value() || *stream != at::cuda::getDefaultCUDAStream(stream->device_index()).unwrap(),
                "gated_linear: an autograd graph of this parameter from the default stream is still alive; free it "
                "first, detach the input, or capture gated_linear_forward and gated_linear_backward");
    for (const auto& e : n->next_edges())
      if (e.function && seen.insert(e.function.get()).second) todo.push_back(e.function.get());
  }
}

at::Tensor gated_linear_autograd(const at::Tensor& x, const at::Tensor& w_gate, const at::Tensor& w_up, int64_t kind) {
  check_caller("gated_linear", {x, w_gate, w_up});
  if (at::cuda::currentStreamCaptureStatusMayInitCtx() != at::cuda::CaptureStatus::None) check_captured_graph({x, w_gate, w_up});
  return GatedLinearFn::apply(x, w_gate, w_up, kind);
}

at::Tensor lora_linear(const at::Tensor& x, const at::Tensor& w, const at::Tensor& lora_a, const at::Tensor& lora_b,
                       const at::Tensor& adapter, const c10::optional<at::Tensor>& scale, c10::optional<at::Tensor> out,
                       int64_t tile) {
  check_caller("lora_linear", {x, w, lora_a, lora_b, scale.value_or(at::Tensor()), out.value_or(at::Tensor())});
  const int fmt = fmt_of(x, "x");
  check_rows(x, "x", x);
  check_rows(w, "w", x);
  const int64_t T = x.size(0), K = x.size(1), N = w.size(0);
  TORCH_CHECK(w.size(1) == K, "x[T,K] and w[N,K] must share K");
  for (const auto* t : {&lora_a, &lora_b})
    TORCH_CHECK(t->is_cuda() && t->device() == x.device() && t->scalar_type() == x.scalar_type() && t->dim() == 3 &&
                    t->is_contiguous(),
                "lora_a[L,r,K] and lora_b[L,N,r] must be contiguous, of x's dtype and on its device");
  const int64_t L = lora_a.size(0), r = lora_a.size(1);
  TORCH_CHECK(lora_a.size(2) == K && lora_b.size(0) == L && lora_b.size(1) == N && lora_b.size(2) == r,
              "lora_a[L,r,K] and lora_b[L,N,r] must share L and r, and K and N with w[N,K]");
  TORCH_CHECK(adapter.is_cuda() && adapter.device() == x.device() && adapter.scalar_type() == at::kInt && adapter.dim() == 1 &&
                  adapter.size(0) == T && adapter.is_contiguous(),
              "adapter must be a contiguous int32 tensor with one index per row of x, on its device");
  const c10::cuda::CUDAGuard g(x.device());
  const float* sp = nullptr;
  if (scale.has_value()) {
    const at::Tensor& s = *scale;
    TORCH_CHECK(s.is_cuda() && s.device() == x.device() && s.scalar_type() == at::kFloat && s.dim() == 1 && s.size(0) == L &&
                    s.is_contiguous(),
                "scale must be a contiguous float32 tensor with one factor per adapter, on x's device");
    sp = s.data_ptr<float>();
  }
  at::Tensor y = out_or_empty(out, T, N, x, {x, w, lora_a, lora_b, adapter});
  TORCH_CHECK(!out.has_value() || !scale.has_value() || !may_overlap(y, *scale), "out must not overlap an input");
  TORCH_CHECK(L >= 1 && r >= 1, "at least one adapter of rank 8 or more");
  if (T > 0) {
    at::Tensor work = at::empty({(int64_t)gicc::ops::lora_work_bytes((int)T, (int)L, (int)r)}, x.options().dtype(at::kByte));
    gicc::ops::lora_linear(x.data_ptr(), w.data_ptr(), lora_a.data_ptr(), lora_b.data_ptr(), adapter.data_ptr<int>(),
                           sp, y.data_ptr(), work.data_ptr(), (int)T, (int)K, (int)N, (int)L, (int)r,
                           pitch_of(x), pitch_of(w), T == 1 ? std::max<int64_t>(N, y.stride(0)) : y.stride(0), fmt, (int)tile,
                           cur_stream());
  }
  return y;
}

py::dict read_errors(bool clear) {
  gicc::ErrorRecord r = gicc::read_error_record(clear);
  py::dict d;
  d["code"] = r.code;
  d["status"] = gicc::status_name(r.code);
  d["where"] = gicc::where_name(r.where);
  d["rank"] = r.rank;
  d["peer"] = r.peer;
  d["value"] = r.value;
  d["expected"] = r.expected;
  d["count"] = r.count;
  return d;
}

at::ScalarType dtype_from_name(const std::string& n) {
  if (n == "bfloat16") return at::kBFloat16;
  if (n == "float16") return at::kHalf;
  if (n == "float32") return at::kFloat;
  if (n == "float64") return at::kDouble;
  if (n == "int32") return at::kInt;
  if (n == "int64") return at::kLong;
  if (n == "uint8") return at::kByte;
  if (n == "int8") return at::kChar;
  throw std::runtime_error("tensor_from_ptr: unsupported dtype " + n);
}

// Zero-copy tensor view of device memory owned elsewhere (symmetric buffers, peer
// mappings, multicast addresses).  The caller keeps the owner alive.
at::Tensor tensor_from_ptr(uint64_t ptr, std::vector<int64_t> shape, const std::string& dtype, int device) {
  auto opts = at::TensorOptions().dtype(dtype_from_name(dtype)).device(at::kCUDA, device);
  return at::from_blob(reinterpret_cast<void*>(static_cast<uintptr_t>(ptr)), shape, opts);
}

}  // namespace

void bind_runtime(py::module_& m);  // runtime.cpp

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.doc() = "opengda_b200 native ops (sm_100a)";
  m.def("set_gemm_tuning", [](int group_m, int l2_hint, int pair_group_m, int pair_l2_hint, int pair_prefetch,
                              int pair_tma_store) {
    gicc::ops::GemmTuning t;
    t.group_m = group_m;
    t.l2_hint = l2_hint;
    t.pair_group_m = pair_group_m;
    t.pair_l2_hint = pair_l2_hint;
    t.pair_prefetch = pair_prefetch;
    t.pair_tma_store = pair_tma_store;
    gicc::ops::set_gemm_tuning(t);
  }, py::arg("group_m") = 16, py::arg("l2_hint") = 0, py::arg("pair_group_m") = 16, py::arg("pair_l2_hint") = 0,
     py::arg("pair_prefetch") = 0, py::arg("pair_tma_store") = 1);
  m.def("gemm_tuning", []() {
    const auto t = gicc::ops::gemm_tuning();
    py::dict d;
    d["group_m"] = t.group_m;
    d["l2_hint"] = t.l2_hint;
    d["pair_group_m"] = t.pair_group_m;
    d["pair_l2_hint"] = t.pair_l2_hint;
    d["pair_prefetch"] = t.pair_prefetch;
    d["pair_tma_store"] = t.pair_tma_store;
    return d;
  });
  m.def("gemm", &gemm, py::arg("A"), py::arg("B"), py::arg("out") = py::none(), py::arg("alpha") = 1.0,
        py::arg("out_f32") = false, py::arg("bn") = 0, "C = alpha * A @ B^T with the tcgen05 GEMM");
  m.def("gemm_fp32", &gemm_fp32, py::arg("A"), py::arg("B"), py::arg("out") = py::none(), py::arg("alpha") = 1.0,
        py::arg("bn") = 0,
        "fp32 C = alpha * A @ B^T on the tensor cores (three tf32 products)");
  m.def("gated_linear", &gated_linear, py::arg("x"), py::arg("w_gate"), py::arg("w_up"), py::arg("act") = 0,
        py::arg("save") = false, py::arg("out") = py::none(), py::arg("tile") = 0,
        "h = act(x w_gate^T) * (x w_up^T); (h, what the backward pass needs)");
  m.def("gated_linear_tile", &gicc::ops::gated_linear_tile, py::arg("T"), py::arg("H"), py::arg("I"),
        "the tile that gated_linear picks for these sizes on the current device");
  m.def("lora_linear_tile", &gicc::ops::lora_linear_tile, py::arg("T"), py::arg("K"), py::arg("N"), py::arg("r"),
        "the tile that lora_linear picks for these sizes on the current device");
  m.def("gated_linear_autograd", &gated_linear_autograd, py::arg("x"), py::arg("w_gate"), py::arg("w_up"), py::arg("act") = 0,
        "gated_linear as a node of the autograd graph");
  m.def("gated_linear_backward", &gated_linear_backward, py::arg("dh"), py::arg("x"), py::arg("w_gate"), py::arg("w_up"),
        py::arg("saved"), py::arg("act") = 0, py::arg("need_dx") = true, py::arg("need_dw") = true, py::arg("tile") = 0,
        "gradients of gated_linear: (dx, dw_gate, dw_up)");
  m.def("lora_linear", &lora_linear, py::arg("x"), py::arg("w"), py::arg("lora_a"), py::arg("lora_b"), py::arg("adapter"),
        py::arg("scale") = py::none(), py::arg("out") = py::none(), py::arg("tile") = 0,
        "y = x w^T plus each row's low-rank adapter");
  m.def("gemm_tile_done_selftest", &gemm_tile_done_selftest, py::arg("A"), py::arg("B"), py::arg("counters"),
        py::arg("skew_ns") = 20000, "run the GEMM core with an epilogue that checks the tile-done ordering");
  m.def("config", [] {
    const gicc::Config c = gicc::config();
    py::dict d;
    d["timeout_ms"] = c.timeout_ms;
    d["bootstrap_timeout_ms"] = c.bootstrap_timeout_ms;
    d["log_level"] = c.log_level;
    d["checks"] = c.checks;
    d["disable_nvls"] = c.disable_nvls;
    d["debug_puts"] = c.debug_puts;
    d["signal_heap_bytes"] = c.signal_heap_bytes;
    return d;
  }, "the GICC_* environment, parsed and range checked (raises ValueError on a bad value)");
  m.def("config_summary", [] { return gicc::config().summary(); });
  m.def("log", [](int level, const std::string& msg) { gicc::log(level, "%s", msg.c_str()); });
  m.def("read_errors", &read_errors, py::arg("clear") = true, "read (and clear) the device error record");
  m.def("default_timeout_ns", &gicc::default_timeout_ns);
  m.def("tensor_from_ptr", &tensor_from_ptr, py::arg("ptr"), py::arg("shape"), py::arg("dtype"), py::arg("device"));
  bind_runtime(m);
}
