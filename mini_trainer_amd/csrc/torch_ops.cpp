// Autograd nodes and allocations of the operators whose calls are short, in C++: the
// same calls of the C ABI (include/mt_flce.h) as from Python, without its interpreter in
// the engine's thread (an embedding of 192 tokens, forward and backward, 75 -> 46 us;
// an empty Python function's backward alone takes 30).
//
// The module links no library of this package: bind() is handed the addresses that
// _lib.py has loaded, once the versions of both agree.  Checks of arguments stay in
// Python.  Streams: a node's backward runs on the stream of its forward, which the engine
// makes the current one and waits for.
#include <torch/extension.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include <stdexcept>
#include <string>

#include "../../include/mt_flce.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Api {
  decltype(&mt_flce_last_error) last_error;
  decltype(&mt_embed_forward) embed_forward;
  decltype(&mt_embed_backward_workspace_bytes) embed_bytes;
  decltype(&mt_embed_backward) embed_backward;
  decltype(&mt_layer_norm_forward) norm_forward;
  decltype(&mt_layer_norm_backward_workspace_bytes) norm_bytes;
  decltype(&mt_layer_norm_backward) norm_backward;
  decltype(&mt_orthogonalize_workspace_bytes) orthogonalize_bytes;
  decltype(&mt_orthogonalize) orthogonalize;
  int (*stream_is_capturing)(mt_stream_t, int*);  // hipStreamIsCapturing
} api;

struct Error : std::runtime_error {
  using std::runtime_error::runtime_error;
};
PyObject* error_class = nullptr;  // what it is in Python

// f(), an Error as the exception that it is in Python: what a node's backward throws gets
// there by way of the engine, where the module's translation does not reach.
template <class F>
variable_list in_engine(F f) {
  try {
    return f();
  } catch (const Error& e) {
    const py::gil_scoped_acquire gil;
    PyErr_SetString(error_class ? error_class : PyExc_RuntimeError, e.what());
    python_error raised;
    raised.persist();
    throw raised;
  }
}

void check(int status, const char* what) {
  if (status == MT_OK) return;
  const char* names[] = {"", "MT_ERR_INVALID_ARGUMENT", "MT_ERR_WORKSPACE_TOO_SMALL", "MT_ERR_UNSUPPORTED",
                         "MT_ERR_HIP"};
  throw Error(std::string(what) + ": " + (status > 0 && status < 5 ? names[status] : "?") + ": " +
                           api.last_error());
}

int dtype_code(const Tensor& t) { return t.scalar_type() == at::kBFloat16 ? MT_DTYPE_BF16 : MT_DTYPE_F32; }

// [T, H] with unit stride along H and rows that do not overlap.
Tensor rows(const Tensor& t) {
  if (t.dim() != 2) return rows(t.reshape({-1, t.size(-1)}));
  if (t.is_contiguous()) return t;
  if ((t.size(1) > 1 && t.stride(1) != 1) || (t.size(0) > 1 && t.stride(0) < t.size(1)))
    return t.clone(at::MemoryFormat::Contiguous);
  return t;
}
int64_t pitch(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }
void* at_or_null(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
mt_stream_t stream_of(int64_t handle) { return reinterpret_cast<mt_stream_t>(handle); }

Tensor workspace(size_t bytes, const Tensor& like) {
  return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : Tensor();
}

// Gradients that cannot be differentiated again: where a graph of them is asked for, one
// that says so.
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  auto refuse = std::make_shared<torch::autograd::DelayedError>(
      "trying to differentiate twice a function that was marked with @once_differentiable", (int64_t)grads.size());
  for (Tensor& g : grads)
    if (g.defined()) g = g.detach().requires_grad_(true);
  return (*refuse)(std::move(grads));
}

// A leaf's gradient node belongs to the stream on which it was made, and lives as long as
// any graph that uses the leaf.  A captured backward that reached one of an eager graph
// would make that graph's stream wait for the capture, and the process ends; it is refused
// here, before the node's result goes on.
void refuse_foreign_leaves(const at::Device& device, int64_t stream) {
  int capturing = 0;
  if (api.stream_is_capturing(stream_of(stream), &capturing) != 0 || !capturing) return;
  const auto node = torch::autograd::get_current_node();
  const c10::Stream here = c10::impl::VirtualGuardImpl(device.type()).getStream(device);
  for (const auto& edge : node->next_edges()) {
    const auto* leaf = dynamic_cast<torch::autograd::AccumulateGrad*>(edge.function.get());
    if (leaf == nullptr) continue;
    const auto made = edge.function->stream();
    if (made && *made != here)
      throw Error("a captured backward reaches a leaf that a graph made on another stream still uses: "
                  "drop that graph's outputs before the capture");
  }
}

struct Embedding : torch::autograd::Function<Embedding> {
  static Tensor forward(AutogradContext* ctx, const Tensor& ids, const Tensor& weight, double scale, int64_t padding,
                        const Tensor* accumulator, const Tensor* status, int64_t stream) {
    const Tensor w = rows(weight), flat = ids.reshape({-1}).contiguous();
    auto shape = ids.sizes().vec();
    shape.push_back(w.size(1));
    Tensor out = at::empty(shape, weight.options());
    mt_embed_args a{};
    a.ids = flat.data_ptr();
    a.weight = w.data_ptr();
    a.out = out.data_ptr();
    a.status = status->defined() ? status->data_ptr<int32_t>() : nullptr;
    a.weight_t = pitch(w);
    a.T = flat.numel(), a.V = w.size(0), a.H = w.size(1);
    a.padding_idx = padding;
    a.scale = (float)scale;
    a.dtype = dtype_code(w), a.ids_bytes = (int)flat.element_size();
    check(api.embed_forward(&a, stream_of(stream)), "mt_embed_forward");
    ctx->save_for_backward({flat});
    ctx->saved_data["V"] = a.V;
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["padding"] = padding;
    ctx->saved_data["stream"] = stream;
    if (accumulator->defined()) ctx->saved_data["accumulator"] = *accumulator;
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    return in_engine([&] { return gradients(ctx, grads); });
  }

  static variable_list gradients(AutogradContext* ctx, const variable_list& grads) {
    variable_list none(7);
    if (!ctx->needs_input_grad(1) || !grads[0].defined()) return none;
    const Tensor ids = ctx->get_saved_variables()[0].contiguous(), d = rows(grads[0]);  // (as below)
    const auto found = ctx->saved_data.find("accumulator");
    const bool add = found != ctx->saved_data.end();
    const int64_t V = ctx->saved_data["V"].toInt(), T = ids.numel(), H = d.size(1);
    const c10::DeviceGuard guard(d.device());
    refuse_foreign_leaves(d.device(), ctx->saved_data["stream"].toInt());
    Tensor dw = add ? found->second.toTensor() : at::empty({V, H}, d.options());
    mt_embed_args a{};
    a.ids = ids.data_ptr();
    a.dout = d.data_ptr();
    a.dweight = dw.data_ptr();
    a.dout_t = pitch(d), a.dweight_t = pitch(dw);
    a.T = T, a.V = V, a.H = H;
    a.padding_idx = ctx->saved_data["padding"].toInt();
    a.scale = (float)ctx->saved_data["scale"].toDouble();
    a.dtype = dtype_code(d), a.ids_bytes = (int)ids.element_size();
    a.accumulate = add;
    const size_t bytes = api.embed_bytes(T, V, H);
    const Tensor ws = workspace(bytes, d);
    check(api.embed_backward(&a, at_or_null(ws), bytes, stream_of(ctx->saved_data["stream"].toInt())),
          "mt_embed_backward");
    if (add) {
      dw.unsafeGetTensorImpl()->bump_version();
      return none;
    }
    none[1] = dw;
    return once(std::move(none));
  }
};

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  using Maybe = std::optional<Tensor>;

  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Maybe& residual, const Maybe& weight,
                               const Maybe& bias, double eps, double block_scale, double residual_scale, bool record,
                               int64_t stream) {
    ctx->set_materialize_grads(false);
    const Tensor x2 = rows(x), r2 = residual ? rows(*residual) : Tensor();
    const Tensor w = weight ? weight->contiguous() : Tensor(), b = bias ? bias->contiguous() : Tensor();
    const int64_t T = x2.size(0), H = x2.size(1);
    Tensor normed = at::empty(x.sizes(), x.options()), h, kept;
    if (r2.defined()) h = at::empty(x.sizes(), x.options());
    // one buffer: 8 bytes a row, and behind them (whole 16 bytes) the low byte of each
    // element of a bf16 sum
    int64_t low = 0;
    if (record) {
      low = (T + 1) / 2 * 16;
      const bool bytes = h.defined() && x.scalar_type() == at::kBFloat16;
      kept = at::empty({low + (bytes ? T * H : 0)}, x.options().dtype(at::kByte));
      if (!bytes) low = 0;
    }
    mt_layer_norm_args a{};
    a.x = x2.data_ptr();
    a.residual = at_or_null(r2);
    a.weight = at_or_null(w);
    a.bias = at_or_null(b);
    a.normed = normed.data_ptr();
    a.new_residual = at_or_null(h);
    a.stat = static_cast<float*>(at_or_null(kept));
    a.residual_lo = low ? kept.data_ptr<uint8_t>() + low : nullptr;
    a.x_t = pitch(x2), a.residual_t = r2.defined() ? pitch(r2) : 0;
    a.T = T, a.H = H;
    a.eps = (float)eps, a.block_scale = (float)block_scale, a.residual_scale = (float)residual_scale;
    a.has_residual = h.defined(), a.dtype = dtype_code(x);
    check(api.norm_forward(&a, stream_of(stream)), "mt_layer_norm_forward");
    ctx->save_for_backward({h.defined() ? h : x2, w, kept});
    auto& data = ctx->saved_data;
    data["shape"] = x.sizes().vec();
    data["low"] = low;
    data["eps"] = eps;
    data["block_scale"] = block_scale;
    data["residual_scale"] = residual_scale;
    data["residual"] = h.defined();
    data["bias"] = b.defined();
    data["stream"] = stream;
    if (h.defined()) return {normed, h};
    return {normed};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    return in_engine([&] { return gradients(ctx, grads); });
  }

  static variable_list gradients(AutogradContext* ctx, const variable_list& grads) {
    variable_list none(9);
    const bool second = grads.size() > 1 && grads[1].defined();
    if (!grads[0].defined() && !second) return none;
    const auto saved = ctx->get_saved_variables();
    auto& data = ctx->saved_data;
    const auto shape = data["shape"].toIntVector();
    const bool residual = data["residual"].toBool();
    const double block_scale = data["block_scale"].toDouble(), residual_scale = data["residual_scale"].toDouble();
    const int64_t low = data["low"].toInt();
    const c10::DeviceGuard guard(saved[0].device());
    // (a hook on saved tensors may hand them back in another layout)
    const Tensor h = residual ? saved[0].contiguous() : rows(saved[0]);
    const Tensor w = saved[1].defined() ? saved[1].contiguous() : Tensor(), kept = saved[2].contiguous();
    refuse_foreign_leaves(h.device(), data["stream"].toInt());
    const Tensor dn = rows(grads[0].defined() ? grads[0] : at::zeros(shape, h.options()));
    const Tensor dh = second ? rows(grads[1]) : Tensor();
    const int64_t T = dn.size(0), H = dn.size(1);
    // (the node's edges count only the tensors that were there)
    int edge = 0;
    const bool need_x = ctx->needs_input_grad(edge++), need_r = residual && ctx->needs_input_grad(edge++);
    const bool need_w = w.defined() && ctx->needs_input_grad(edge++);
    const bool need_b = data["bias"].toBool() && ctx->needs_input_grad(edge);
    // where both are the same number the two inputs share one gradient, as an addition's do
    const bool same = need_x && need_r && block_scale == residual_scale;
    Tensor dr = need_r ? at::empty(shape, h.options()) : Tensor();
    Tensor dx = need_x && !same ? at::empty(shape, h.options()) : Tensor();
    Tensor dw = need_w ? at::empty({H}, h.options()) : Tensor();
    Tensor db = need_b ? at::empty({H}, h.options()) : Tensor();
    mt_layer_norm_args a{};
    if (residual) a.new_residual = h.data_ptr();
    else a.x = h.data_ptr();
    a.weight = at_or_null(w);
    a.stat = static_cast<float*>(kept.data_ptr());
    a.residual_lo = low ? kept.data_ptr<uint8_t>() + low : nullptr;
    a.dnormed = dn.data_ptr();
    a.dresidual_out = at_or_null(dh);
    a.dx = at_or_null(dx);
    a.dresidual = at_or_null(dr);
    a.dweight = at_or_null(dw);
    a.dbias = at_or_null(db);
    a.x_t = residual ? H : pitch(h);
    a.dnormed_t = pitch(dn), a.dresidual_out_t = dh.defined() ? pitch(dh) : H;
    a.T = T, a.H = H;
    a.eps = (float)data["eps"].toDouble();
    a.block_scale = (float)block_scale, a.residual_scale = (float)residual_scale;
    a.has_residual = residual, a.dtype = dtype_code(h);
    const size_t bytes = api.norm_bytes(T, H);
    const Tensor ws = workspace(bytes, h);
    check(api.norm_backward(&a, at_or_null(ws), bytes, stream_of(data["stream"].toInt())), "mt_layer_norm_backward");
    if (T == 0) {
      if (dw.defined()) dw.zero_();
      if (db.defined()) db.zero_();
    }
    none[0] = same ? dr : dx, none[1] = dr, none[2] = dw, none[3] = db;
    return once(std::move(none));
  }
};

Tensor embedding(const Tensor& ids, const Tensor& weight, double scale, int64_t padding,
                 const std::optional<Tensor>& accumulator, const std::optional<Tensor>& status, int64_t stream) {
  const c10::DeviceGuard guard(weight.device());
  const Tensor acc = accumulator.value_or(Tensor()), st = status.value_or(Tensor());
  return Embedding::apply(ids, weight, scale, padding, &acc, &st, stream);
}

variable_list layer_norm(const Tensor& x, const std::optional<Tensor>& residual, const std::optional<Tensor>& weight,
                         const std::optional<Tensor>& bias, double eps, double block_scale, double residual_scale,
                         bool record, int64_t stream) {
  const c10::DeviceGuard guard(x.device());
  return LayerNorm::apply(x, residual, weight, bias, eps, block_scale, residual_scale, record, stream);
}

// The coefficients: the address of 3 steps doubles.
Tensor orthogonalize(const Tensor& update, int64_t coefficients, int64_t steps, double eps, int64_t stream) {
  const at::NoGradGuard no_grad;
  const c10::DeviceGuard guard(update.device());
  Tensor out = at::empty(update.sizes(), update.options());
  if (out.numel() == 0) return out;
  const int64_t m = update.size(-2), n = update.size(-1);
  Tensor x = update.dim() == 3 ? update : update.reshape({-1, m, n});
  if ((n > 1 && x.stride(2) != 1) || (m > 1 && x.stride(1) < n)) x = x.clone(at::MemoryFormat::Contiguous);
  mt_orthogonalize_args a{};
  a.in = x.data_ptr();
  a.out = out.data_ptr();
  a.coefficients = reinterpret_cast<const double*>(coefficients);
  a.eps = eps;
  a.batch = x.size(0), a.m = m, a.n = n;
  a.in_row = m > 1 ? x.stride(1) : n, a.in_batch = a.batch > 1 ? x.stride(0) : 0;
  a.steps = (int)steps, a.dtype = dtype_code(x);
  const size_t bytes = api.orthogonalize_bytes(&a);
  const Tensor ws = workspace(bytes, x);
  check(api.orthogonalize(&a, at_or_null(ws), bytes, stream_of(stream)), "mt_orthogonalize");
  return out;
}

// The addresses of the functions, in Api's order, and the class that Error becomes.
void bind(const std::vector<int64_t>& at, const py::object& error) {
  error_class = error.inc_ref().ptr();
  int k = 0;
  const auto take = [&](auto& f) { f = reinterpret_cast<std::decay_t<decltype(f)>>(at.at(k++)); };
  take(api.last_error), take(api.embed_forward), take(api.embed_bytes), take(api.embed_backward);
  take(api.norm_forward), take(api.norm_bytes), take(api.norm_backward);
  take(api.orthogonalize_bytes), take(api.orthogonalize), take(api.stream_is_capturing);
}

}  // namespace

PYBIND11_MODULE(_mt_torch, m) {
  py::register_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const Error& e) {
      PyErr_SetString(error_class ? error_class : PyExc_RuntimeError, e.what());
    }
  });
  // what _lib.py compares before it binds
  m.attr("abi_version") = MT_FLCE_ABI_VERSION;
  m.attr("torch_version") = MT_TORCH_VERSION;
  m.def("bind", &bind);
  m.def("embedding", &embedding);
  m.def("layer_norm", &layer_norm);
  m.def("orthogonalize", &orthogonalize);
}
