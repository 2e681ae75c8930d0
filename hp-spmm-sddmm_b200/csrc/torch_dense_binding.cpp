// PyTorch operators of the dense operands by index (tables, groups of rows, teachers): registration, autograd formulas,
// stream and memory handling.  Arithmetic stays in libhpspmm.so.
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/extension.h>

#include <memory>
#include <mutex>
#include <vector>

#include "hpspmm.h"

namespace {

using at::Tensor;

// One context for each device, for its error text: these operators keep nothing in it.  Calls that share one are kept apart
// on the host.  Contexts live as long as the process, as a graph that holds such calls may.
struct DeviceContext {
  std::mutex use;
  hpspmm_ctx* ctx = nullptr;
};

DeviceContext& context_of(const at::Device& device) {
  static std::mutex mutex;
  static auto* all = new std::vector<std::unique_ptr<DeviceContext>>();
  const size_t index = (size_t)device.index();
  std::lock_guard<std::mutex> lock(mutex);
  if (all->size() <= index) all->resize(index + 1);
  auto& c = (*all)[index];
  if (!c) {
    // a first call may be a captured one: the context's 256 bytes are allocated outside the capture
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    cudaThreadExchangeStreamCaptureMode(&mode);
    auto made = std::make_unique<DeviceContext>();
    const int st = hpspmm_ctx_create((int)index, &made->ctx);
    cudaThreadExchangeStreamCaptureMode(&mode);
    TORCH_CHECK(st == HPSPMM_OK, "hpspmm_ctx_create failed with status ", st, ": ", hpspmm_status_string(st));
    c = std::move(made);
  }
  return *c;
}

template <typename F>
void call(const at::Device& device, const char* what, F&& f) {
  const c10::cuda::CUDAGuard guard(device);
  DeviceContext& c = context_of(device);
  std::lock_guard<std::mutex> lock(c.use);
  const int st = f(c.ctx, (hpspmm_stream)c10::cuda::getCurrentCUDAStream().stream());
  TORCH_CHECK(st == HPSPMM_OK, what, " failed with status ", st, ": ", hpspmm_last_error(c.ctx));
}

int type_of(const Tensor& t, const char* what) {
  TORCH_CHECK(t.is_cuda(), "hpspmm: ", what, " must be a CUDA tensor (there is no CPU path)");
  switch (t.scalar_type()) {
    case at::kFloat: return HPSPMM_TYPE_F32;
    case at::kHalf: return HPSPMM_TYPE_F16;
    case at::kBFloat16: return HPSPMM_TYPE_BF16;
    default: TORCH_CHECK(false, "hpspmm: ", what, " must be float32, float16 or bfloat16, got ", t.scalar_type());
  }
}

Tensor ids_of(const Tensor& t, const at::Device& device, const char* what) {
  TORCH_CHECK((t.scalar_type() == at::kInt || t.scalar_type() == at::kLong) && t.device() == device, "hpspmm: ", what,
              " must be int32 or int64 on ", device, ", got ", t.scalar_type(), " on ", t.device());
  return t.contiguous();
}

// Elements of a row next to each other, rows a stride of at least their width apart, as the kernels read them.
Tensor rows_of(const Tensor& t) {
  const bool dense = t.size(1) <= 1 || t.stride(1) == 1;
  const bool apart = t.size(0) <= 1 || t.stride(0) >= t.size(1);
  return dense && apart ? t : t.contiguous();
}
int64_t stride_of(const Tensor& rows) { return rows.size(0) <= 1 ? rows.size(1) : rows.stride(0); }

// ---- rows of a table -------------------------------------------------------------------------------------------

Tensor embedding(const Tensor& ids_, const Tensor& table_, double scale) {
  const int type = type_of(table_, "table");
  TORCH_CHECK(table_.dim() == 2, "hpspmm: table must have two dimensions, got ", table_.sizes());
  const Tensor ids = ids_of(ids_, table_.device(), "ids"), table = rows_of(table_);
  auto shape = ids.sizes().vec();
  shape.push_back(table.size(1));
  Tensor out = at::empty(shape, table.options());
  call(table.device(), "hpspmm_embedding_forward", [&](hpspmm_ctx* ctx, hpspmm_stream stream) {
    return hpspmm_embedding_forward(ctx, ids.numel(), table.size(0), table.size(1), type, ids.const_data_ptr(),
                                    (int)ids.element_size(), table.const_data_ptr(), stride_of(table), (float)scale,
                                    out.mutable_data_ptr(), stream);
  });
  return out;
}

Tensor embedding_backward(const Tensor& grad, const Tensor& ids_, int64_t rows, double scale) {
  const int type = type_of(grad, "the gradient");
  TORCH_CHECK(grad.dim() >= 1 && grad.dim() == ids_.dim() + 1 && grad.sizes().slice(0, ids_.dim()) == ids_.sizes(),
              "hpspmm: a gradient of shape ", grad.sizes(), " for ids of shape ", ids_.sizes());
  TORCH_CHECK(rows >= 0, "hpspmm: a negative number of rows");
  const Tensor ids = ids_of(ids_, grad.device(), "ids");
  const int64_t T = ids.numel(), K = grad.size(-1);
  const Tensor dout = rows_of(grad.reshape({T, K}));
  Tensor dtable = at::empty({rows, K}, grad.options());
  const int64_t bytes = hpspmm_embedding_backward_workspace(T, rows, K);
  TORCH_CHECK(bytes >= 0, "hpspmm: a table or batch of more than 2^31 - 2 rows");
  const Tensor workspace = at::empty({bytes}, grad.options().dtype(at::kByte));
  call(grad.device(), "hpspmm_embedding_backward", [&](hpspmm_ctx* ctx, hpspmm_stream stream) {
    return hpspmm_embedding_backward(ctx, T, rows, K, type, ids.const_data_ptr(), (int)ids.element_size(),
                                     dout.const_data_ptr(), stride_of(dout), (float)scale, dtable.mutable_data_ptr(),
                                     workspace.mutable_data_ptr(), (size_t)bytes, stream);
  });
  return dtable;
}

// ---- products of groups of rows ---------------------------------------------------------------------------------

Tensor offsets_of(const Tensor& t, const at::Device& device, int64_t groups) {
  TORCH_CHECK(t.scalar_type() == at::kInt && t.device() == device && t.dim() == 1 && t.numel() == groups + 1,
              "hpspmm: offsets must be ", groups + 1, " int32 values on ", device, ", got ", t.scalar_type(), " ", t.sizes(),
              " on ", t.device());
  return t.contiguous();
}

// Whether the matrices of W [G, K, N] are stored transposed.
bool out_first(const Tensor& W) { return !W.is_contiguous() && W.transpose(1, 2).is_contiguous(); }

Tensor grouped_product(const Tensor& X, const Tensor& W, const Tensor& offsets_) {
  const int type = type_of(X, "X");
  TORCH_CHECK(X.dim() == 2 && W.dim() == 3 && W.size(1) == X.size(1) && W.scalar_type() == X.scalar_type() &&
                  W.device() == X.device(), "hpspmm: X [R, K] and W [G, K, N] must agree in K, type and device, got ",
              X.sizes(), " ", X.scalar_type(), " on ", X.device(), " and ", W.sizes(), " ", W.scalar_type(), " on ", W.device());
  const Tensor offsets = offsets_of(offsets_, X.device(), W.size(0)), x = rows_of(X);
  const bool t = out_first(W);
  const Tensor w = t ? W : W.contiguous();
  Tensor Y = at::empty({x.size(0), w.size(2)}, x.options());
  call(x.device(), "hpspmm_grouped_product", [&](hpspmm_ctx* ctx, hpspmm_stream stream) {
    return hpspmm_grouped_product(ctx, x.size(0), w.size(0), x.size(1), w.size(2), type, x.const_data_ptr(), stride_of(x),
                                  w.const_data_ptr(), t, offsets.const_data_ptr<int>(), Y.mutable_data_ptr(), stream);
  });
  return Y;
}

Tensor grouped_weight_grad(const Tensor& X, const Tensor& dY, const Tensor& offsets_, bool transposed) {
  const int type = type_of(X, "X");
  TORCH_CHECK(X.dim() == 2 && dY.dim() == 2 && X.size(0) == dY.size(0) && X.scalar_type() == dY.scalar_type() &&
                  X.device() == dY.device(), "hpspmm: X [R, K] and dY [R, N] must agree in R, type and device, got ", X.sizes(),
              " ", X.scalar_type(), " on ", X.device(), " and ", dY.sizes(), " ", dY.scalar_type(), " on ", dY.device());
  TORCH_CHECK(offsets_.dim() == 1 && offsets_.numel() >= 1, "hpspmm: offsets must hold at least one value");
  const int64_t groups = offsets_.numel() - 1;
  const Tensor offsets = offsets_of(offsets_, X.device(), groups), x = rows_of(X), dy = rows_of(dY);
  const int64_t K = x.size(1), N = dy.size(1);
  Tensor dW = transposed ? at::empty({groups, N, K}, x.options()) : at::empty({groups, K, N}, x.options());
  const int64_t bytes = hpspmm_grouped_weight_grad_workspace(x.size(0), groups, K, N, type, transposed);
  TORCH_CHECK(bytes >= 0, "hpspmm: more than 2^31 - 1026 rows or columns, or 2^20 groups");
  const Tensor workspace = at::empty({bytes}, x.options().dtype(at::kByte));
  call(x.device(), "hpspmm_grouped_weight_grad", [&](hpspmm_ctx* ctx, hpspmm_stream stream) {
    return hpspmm_grouped_weight_grad(ctx, x.size(0), groups, K, N, type, x.const_data_ptr(), stride_of(x),
                                      dy.const_data_ptr(), stride_of(dy), offsets.const_data_ptr<int>(),
                                      dW.mutable_data_ptr(), transposed, workspace.mutable_data_ptr(), (size_t)bytes, stream);
  });
  return transposed ? dW.transpose(1, 2) : dW;
}

// ---- loss against a teacher's entries ------------------------------------------------------------------------------

struct Teacher {
  Tensor logits, ids, values;   // rows of each, flattened over the leading dimensions
};
Teacher teacher_of(const Tensor& logits, const Tensor& ids, const Tensor& values) {
  TORCH_CHECK(logits.dim() >= 1 && ids.dim() == logits.dim() && ids.sizes() == values.sizes() &&
                  ids.sizes().slice(0, ids.dim() - 1) == logits.sizes().slice(0, logits.dim() - 1),
              "hpspmm: logits [..., V] and the teacher's ids and logits [..., k] must agree, got ", logits.sizes(), ", ",
              ids.sizes(), " and ", values.sizes());
  type_of(values, "teacher_logits");
  TORCH_CHECK(values.device() == logits.device(), "hpspmm: teacher_logits must be on ", logits.device());
  const int64_t V = logits.size(-1), k = ids.size(-1);
  int64_t T = 1;
  for (int64_t d = 0; d + 1 < logits.dim(); ++d) T *= logits.size(d);
  return {rows_of(logits.reshape({T, V})), ids_of(ids, logits.device(), "teacher_ids").reshape({T, k}),
          values.to(at::kFloat).contiguous().reshape({T, k})};
}

std::tuple<Tensor, Tensor> topk_distill(const Tensor& logits, const Tensor& ids, const Tensor& values, double temperature) {
  const int type = type_of(logits, "logits");
  const Teacher t = teacher_of(logits, ids, values);
  const int64_t T = t.logits.size(0);
  Tensor loss = at::empty(logits.sizes().slice(0, logits.dim() - 1), logits.options().dtype(at::kFloat));
  Tensor stats = at::empty({T, 2}, loss.options());
  call(logits.device(), "hpspmm_topk_distill_forward", [&](hpspmm_ctx* ctx, hpspmm_stream stream) {
    return hpspmm_topk_distill_forward(ctx, T, t.logits.size(1), t.ids.size(1), type, t.logits.const_data_ptr(),
                                       stride_of(t.logits), t.ids.const_data_ptr(), (int)t.ids.element_size(),
                                       t.values.const_data_ptr<float>(), (float)temperature, loss.mutable_data_ptr<float>(),
                                       stats.mutable_data_ptr<float>(), stream);
  });
  return {loss, stats};
}

Tensor topk_distill_backward(const Tensor& dloss_, const Tensor& logits, const Tensor& ids, const Tensor& values,
                             const Tensor& stats_, double temperature) {
  const int type = type_of(logits, "logits");
  const Teacher t = teacher_of(logits, ids, values);
  const int64_t T = t.logits.size(0);
  TORCH_CHECK(dloss_.scalar_type() == at::kFloat && dloss_.device() == logits.device() && dloss_.numel() == T &&
                  stats_.scalar_type() == at::kFloat && stats_.device() == logits.device() && stats_.numel() == 2 * T,
              "hpspmm: the gradient of the loss and the row statistics must be float32 for ", T, " rows on ", logits.device());
  const Tensor dloss = dloss_.reshape({T}), stats = stats_.contiguous();
  Tensor dz = at::empty(logits.sizes(), logits.options());
  call(logits.device(), "hpspmm_topk_distill_backward", [&](hpspmm_ctx* ctx, hpspmm_stream stream) {
    return hpspmm_topk_distill_backward(ctx, T, t.logits.size(1), t.ids.size(1), type, t.logits.const_data_ptr(),
                                        stride_of(t.logits), t.ids.const_data_ptr(), (int)t.ids.element_size(),
                                        t.values.const_data_ptr<float>(), (float)temperature,
                                        stats.const_data_ptr<float>(), dloss.const_data_ptr<float>(),
                                        T <= 1 ? 1 : dloss.stride(0), dz.mutable_data_ptr(), stream);
  });
  return dz;
}

// ---- the registered operators, for calls that go through the dispatcher ---------------------------------------------

template <typename F>
c10::TypedOperatorHandle<F> find(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}
#define HPSPMM_OP(NAME)                                                          \
  const c10::TypedOperatorHandle<decltype(NAME)>& op_##NAME() {                  \
    static const auto op = find<decltype(NAME)>("hpspmm::" #NAME);               \
    return op;                                                                   \
  }
HPSPMM_OP(embedding)
HPSPMM_OP(embedding_backward)
HPSPMM_OP(grouped_product)
HPSPMM_OP(grouped_weight_grad)
HPSPMM_OP(topk_distill)
HPSPMM_OP(topk_distill_backward)

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// A lookup is linear in the table, so the two operators are each other's derivative.
struct EmbeddingFunction : public torch::autograd::Function<EmbeddingFunction> {
  static Tensor forward(AutogradContext* ctx, const Tensor& ids, const Tensor& table, double scale) {
    ctx->save_for_backward({ids});
    ctx->saved_data["rows"] = table.dim() > 0 ? table.size(0) : 0;
    ctx->saved_data["scale"] = scale;
    at::AutoDispatchBelowADInplaceOrView below;
    return op_embedding().call(ids, table, scale);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    Tensor d;
    if (grads[0].defined() && ctx->needs_input_grad(1))
      d = op_embedding_backward().call(grads[0], ctx->get_saved_variables()[0], ctx->saved_data["rows"].toInt(),
                                       ctx->saved_data["scale"].toDouble());
    return {Tensor(), d, Tensor()};
  }
};
struct EmbeddingBackwardFunction : public torch::autograd::Function<EmbeddingBackwardFunction> {
  static Tensor forward(AutogradContext* ctx, const Tensor& grad, const Tensor& ids, int64_t rows, double scale) {
    ctx->save_for_backward({ids});
    ctx->saved_data["scale"] = scale;
    at::AutoDispatchBelowADInplaceOrView below;
    return op_embedding_backward().call(grad, ids, rows, scale);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    Tensor d;
    if (grads[0].defined() && ctx->needs_input_grad(0))
      d = op_embedding().call(ctx->get_saved_variables()[0], grads[0], ctx->saved_data["scale"].toDouble());
    return {d, Tensor(), Tensor(), Tensor()};
  }
};

// Bilinear in X and W: every derivative is one of the two operators again.
struct GroupedProductFunction : public torch::autograd::Function<GroupedProductFunction> {
  static Tensor forward(AutogradContext* ctx, const Tensor& X, const Tensor& W, const Tensor& offsets) {
    ctx->save_for_backward({X, W, offsets});
    at::AutoDispatchBelowADInplaceOrView below;
    return op_grouped_product().call(X, W, offsets);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    Tensor dX, dW;
    if (grads[0].defined()) {
      const auto saved = ctx->get_saved_variables();
      if (ctx->needs_input_grad(0)) dX = op_grouped_product().call(grads[0], saved[1].transpose(1, 2), saved[2]);
      if (ctx->needs_input_grad(1)) dW = op_grouped_weight_grad().call(saved[0], grads[0], saved[2], out_first(saved[1]));
    }
    return {dX, dW, Tensor()};
  }
};
struct GroupedWeightGradFunction : public torch::autograd::Function<GroupedWeightGradFunction> {
  static Tensor forward(AutogradContext* ctx, const Tensor& X, const Tensor& dY, const Tensor& offsets, bool transposed) {
    ctx->save_for_backward({X, dY, offsets});
    at::AutoDispatchBelowADInplaceOrView below;
    return op_grouped_weight_grad().call(X, dY, offsets, transposed);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    Tensor dX, ddY;
    if (grads[0].defined()) {
      const auto saved = ctx->get_saved_variables();
      if (ctx->needs_input_grad(0)) dX = op_grouped_product().call(saved[1], grads[0].transpose(1, 2), saved[2]);
      if (ctx->needs_input_grad(1)) ddY = op_grouped_product().call(saved[0], grads[0], saved[2]);
    }
    return {dX, ddY, Tensor(), Tensor()};
  }
};

struct TopkDistillFunction : public torch::autograd::Function<TopkDistillFunction> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& ids, const Tensor& values,
                               double temperature) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto out = op_topk_distill().call(logits, ids, values, temperature);
    ctx->save_for_backward({logits, ids, values, std::get<1>(out)});
    ctx->saved_data["temperature"] = temperature;
    ctx->mark_non_differentiable({std::get<1>(out)});
    return {std::get<0>(out), std::get<1>(out)};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    Tensor d;
    if (grads[0].defined() && ctx->needs_input_grad(0)) {
      const auto saved = ctx->get_saved_variables();
      d = op_topk_distill_backward().call(grads[0], saved[0], saved[1], saved[2], saved[3],
                                          ctx->saved_data["temperature"].toDouble());
    }
    return {d, Tensor(), Tensor(), Tensor()};
  }
};
struct NoDerivativeOfDistill : public torch::autograd::Function<NoDerivativeOfDistill> {
  static Tensor forward(AutogradContext*, const Tensor& dloss, const Tensor& logits, const Tensor& ids, const Tensor& values,
                        const Tensor& stats, double temperature) {
    at::AutoDispatchBelowADInplaceOrView below;
    return op_topk_distill_backward().call(dloss, logits, ids, values, stats, temperature);
  }
  static variable_list backward(AutogradContext*, variable_list) {
    TORCH_CHECK(false, "hpspmm: no derivative of hpspmm::topk_distill_backward is implemented (a second derivative of the loss)");
  }
};

Tensor embedding_autograd(const Tensor& ids, const Tensor& table, double scale) {
  return EmbeddingFunction::apply(ids, table, scale);
}
Tensor embedding_backward_autograd(const Tensor& grad, const Tensor& ids, int64_t rows, double scale) {
  return EmbeddingBackwardFunction::apply(grad, ids, rows, scale);
}
Tensor grouped_product_autograd(const Tensor& X, const Tensor& W, const Tensor& offsets) {
  return GroupedProductFunction::apply(X, W, offsets);
}
Tensor grouped_weight_grad_autograd(const Tensor& X, const Tensor& dY, const Tensor& offsets, bool transposed) {
  return GroupedWeightGradFunction::apply(X, dY, offsets, transposed);
}
std::tuple<Tensor, Tensor> topk_distill_autograd(const Tensor& logits, const Tensor& ids, const Tensor& values,
                                                 double temperature) {
  TORCH_CHECK(!(at::GradMode::is_enabled() && values.requires_grad()),
              "hpspmm: the loss has no gradient of teacher_logits: detach them");
  auto out = TopkDistillFunction::apply(logits, ids, values, temperature);
  return {out[0], out[1]};
}
Tensor topk_distill_backward_autograd(const Tensor& dloss, const Tensor& logits, const Tensor& ids, const Tensor& values,
                                      const Tensor& stats, double temperature) {
  if (at::GradMode::is_enabled() && (dloss.requires_grad() || logits.requires_grad()))
    return NoDerivativeOfDistill::apply(dloss, logits, ids, values, stats, temperature);
  at::AutoDispatchBelowADInplaceOrView below;
  return op_topk_distill_backward().call(dloss, logits, ids, values, stats, temperature);
}

TORCH_LIBRARY_FRAGMENT(hpspmm, m) {
  m.def("embedding(Tensor ids, Tensor table, float scale) -> Tensor");
  m.def("embedding_backward(Tensor grad, Tensor ids, int rows, float scale) -> Tensor");
  m.def("grouped_product(Tensor X, Tensor W, Tensor offsets) -> Tensor");
  m.def("grouped_weight_grad(Tensor X, Tensor dY, Tensor offsets, bool transposed) -> Tensor");
  m.def("topk_distill(Tensor logits, Tensor teacher_ids, Tensor teacher_logits, float temperature) -> (Tensor, Tensor)");
  m.def("topk_distill_backward(Tensor dloss, Tensor logits, Tensor teacher_ids, Tensor teacher_logits, Tensor stats, "
        "float temperature) -> Tensor");
}
// a CPU tensor reaches the same functions, which refuse it by name
#define HPSPMM_DENSE_IMPL(KEY)                             \
  TORCH_LIBRARY_IMPL(hpspmm, KEY, m) {                     \
    m.impl("embedding", embedding);                        \
    m.impl("embedding_backward", embedding_backward);      \
    m.impl("grouped_product", grouped_product);            \
    m.impl("grouped_weight_grad", grouped_weight_grad);    \
    m.impl("topk_distill", topk_distill);                  \
    m.impl("topk_distill_backward", topk_distill_backward); \
  }
HPSPMM_DENSE_IMPL(CUDA)
HPSPMM_DENSE_IMPL(CPU)
TORCH_LIBRARY_IMPL(hpspmm, Autograd, m) {
  m.impl("embedding", embedding_autograd);
  m.impl("embedding_backward", embedding_backward_autograd);
  m.impl("grouped_product", grouped_product_autograd);
  m.impl("grouped_weight_grad", grouped_weight_grad_autograd);
  m.impl("topk_distill", topk_distill_autograd);
  m.impl("topk_distill_backward", topk_distill_backward_autograd);
}

}  // namespace

// The operators without the Python dispatcher's share.
void bind_dense_operators(py::module_& m) {
  m.def("timeouts", [](int device) {
    DeviceContext& c = context_of(at::Device(at::kCUDA, (c10::DeviceIndex)device));
    int64_t n = 0;
    std::lock_guard<std::mutex> lock(c.use);
    const int st = hpspmm_ctx_timeouts(c.ctx, &n);
    TORCH_CHECK(st == HPSPMM_OK, "hpspmm_ctx_timeouts failed with status ", st, ": ", hpspmm_last_error(c.ctx));
    return n;
  }, py::call_guard<py::gil_scoped_release>());
  m.def("embedding", [](const Tensor& ids, const Tensor& table, double scale) { return op_embedding().call(ids, table, scale); },
        py::call_guard<py::gil_scoped_release>());
  m.def("grouped_product",
        [](const Tensor& X, const Tensor& W, const Tensor& offsets) { return op_grouped_product().call(X, W, offsets); },
        py::call_guard<py::gil_scoped_release>());
  m.def("topk_distill",
        [](const Tensor& logits, const Tensor& ids, const Tensor& values, double temperature) {
          return std::get<0>(op_topk_distill().call(logits, ids, values, temperature));
        },
        py::call_guard<py::gil_scoped_release>());
}
