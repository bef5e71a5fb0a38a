// The token operators as torch sees them: tensors in, tensors out, gradients.  Host code only - every kernel is behind the C entries of
// omnihd_hip.h, whose addresses omnihd_amd/_lib.py hands over (so there is one loaded library, whichever it is).
//
// Why not the ctypes path of the other wrappers: these operators are called between the blocks of a model, often on a few rows, where
// a training pass is bound by the host.  A pass through ctypes and a Python autograd function took 105 us (embedding), 160 us (join) on a
// box where a bare autograd pass takes 40.  Argument checks with their messages stay in Python (omnihd_amd/ops).
#include <torch/extension.h>
#include <ATen/SavedTensorHooks.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include "omnihd_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;
typedef std::optional<Tensor> Maybe;

struct Api {
  decltype(&omnihd_last_error) last_error;
  decltype(&omnihd_token_embed_fwd) token_embed_fwd;
  decltype(&omnihd_token_embed_bwd_workspace_bytes) token_embed_bwd_workspace_bytes;
  decltype(&omnihd_token_embed_bwd) token_embed_bwd;
  decltype(&omnihd_block_join_fwd) block_join_fwd;
  decltype(&omnihd_block_join_bwd_workspace_bytes) block_join_bwd_workspace_bytes;
  decltype(&omnihd_block_join_bwd) block_join_bwd;
  decltype(&omnihd_topk_distill_workspace_bytes) topk_distill_workspace_bytes;
  decltype(&omnihd_topk_distill) topk_distill;
} api;

void bind(const py::dict& at) {
  auto set = [&](auto& f, const char* name) { f = reinterpret_cast<std::decay_t<decltype(f)>>(at[name].cast<uintptr_t>()); };
  set(api.last_error, "omnihd_last_error");
  set(api.token_embed_fwd, "omnihd_token_embed_fwd");
  set(api.token_embed_bwd_workspace_bytes, "omnihd_token_embed_bwd_workspace_bytes");
  set(api.token_embed_bwd, "omnihd_token_embed_bwd");
  set(api.block_join_fwd, "omnihd_block_join_fwd");
  set(api.block_join_bwd_workspace_bytes, "omnihd_block_join_bwd_workspace_bytes");
  set(api.block_join_bwd, "omnihd_block_join_bwd");
  set(api.topk_distill_workspace_bytes, "omnihd_topk_distill_workspace_bytes");
  set(api.topk_distill, "omnihd_topk_distill");
}

void check(int status, const char* what) {
  TORCH_CHECK(status == OMNIHD_OK, what, " failed with status ", status, ": ", api.last_error());
}

int code(const Tensor& t) { return t.scalar_type() == at::kFloat ? 0 : t.scalar_type() == at::kBFloat16 ? 1 : 2; }
int code(at::ScalarType t) { return t == at::kFloat ? 0 : t == at::kBFloat16 ? 1 : 2; }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
// tensors kept for the backward go somewhere else or are computed again (save_on_cpu, checkpointing)
bool saved_elsewhere() { return !at::SavedTensorDefaultHooks::get_tls_state().stack.empty(); }
bool capturing() { return c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None; }

// (..., dim) as rows with one pitch between them: the tensor as it lies where the strides allow it, else a copy
struct Rows {
  void* p = nullptr;
  long long pitch = 0;
  Tensor keep;
};
Rows rows_of(const Tensor& t, int64_t dim) {
  Rows r;
  if (!t.defined()) return r;
  r.keep = t;
  r.pitch = dim;
  bool fits = t.is_contiguous();
  if (!fits && (dim == 1 || t.stride(-1) == 1)) {
    fits = true;
    int64_t step = -1, inner = 1;                   // of the leading dimensions with more than one entry: the innermost's stride, their product
    for (int64_t k = t.dim() - 2; k >= 0 && fits; --k) {
      if (t.size(k) == 1) continue;
      if (step < 0) step = t.stride(k);
      fits = t.stride(k) == step * inner;
      inner *= t.size(k);
    }
    if (step >= 0) r.pitch = step;
    fits = fits && r.pitch >= dim;
  }
  if (!fits) {
    r.keep = t.contiguous();
    r.pitch = dim;
  }
  r.p = r.keep.data_ptr();
  return r;
}

Tensor dense_like(const Tensor& t) { return at::empty(t.sizes(), t.options()); }
Tensor workspace(size_t bytes, const Tensor& like) { return at::empty({(int64_t)std::max<size_t>(bytes, 256)}, like.options().dtype(at::kByte)); }
void no_second_order(const char* what) {
  TORCH_CHECK(!at::GradMode::is_enabled(), what, ": second derivatives (create_graph=True) are not supported");
}
// What follows a call by torch's own operations sees no kernel: an output would come without the tangent of a forward-mode dual tensor (its
// directional derivative silently zero), a traced function would hold the allocation of an output and nothing that fills it.  Both are refused.
void seen_by_autograd_alone(const char* what, std::initializer_list<Tensor> ts) {
  namespace mode = c10::impl;
  const bool recorded = mode::TorchDispatchModeTLS::any_modes_set() &&
                        mode::TorchDispatchModeTLS::get_mode(mode::TorchDispatchModeKey::PROXY).has_value();
  TORCH_CHECK_NOT_IMPLEMENTED(!recorded && !torch::jit::tracer::isTracing(), what, ": cannot be traced (torch.jit.trace, make_fx); capture a graph instead");
  for (const Tensor& t : ts)
    TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(0).defined(), what, ": forward-mode derivatives (dual tensors) are not supported");
}
Tensor of(const Maybe& t) { return t.has_value() ? *t : Tensor(); }
bool wants_grad(std::initializer_list<Tensor> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor& t : ts)
    if (t.defined() && t.requires_grad()) return true;
  return false;
}

// ---- embedding ----------------------------------------------------------------------------------------------------------------
Tensor embed_forward(const Tensor& ids, const Tensor& table, double scale, at::ScalarType out_type) {
  std::vector<int64_t> shape = ids.sizes().vec();
  shape.push_back(table.size(1));
  Tensor out = at::empty(shape, table.options().dtype(out_type));
  if (out.numel()) {
    c10::DeviceGuard guard(table.device());
    check(api.token_embed_fwd(ids.data_ptr(), ids.scalar_type() == at::kLong, ids.numel(), table.data_ptr(), code(table),
                              table.size(0) > 1 ? table.stride(0) : table.size(1), table.size(0), table.size(1), scale, out.data_ptr(),
                              code(out_type), stream_of(table)), "omnihd_token_embed_fwd");
  }
  return out;
}

struct Embed : public Function<Embed> {
  static Tensor forward(AutogradContext* ctx, Tensor table, Tensor ids, double scale, int64_t padding, int64_t out_type) {
    ctx->save_for_backward({ids});
    ctx->saved_data["vocab"] = table.size(0);
    ctx->saved_data["dim"] = table.size(1);
    ctx->saved_data["type"] = (int64_t)table.scalar_type();
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["padding"] = padding;
    return embed_forward(ids, table, scale, (at::ScalarType)out_type);
  }
  static variable_list backward(AutogradContext* ctx, variable_list ups) {
    no_second_order("token_embedding");
    const Tensor ids = ctx->get_saved_variables()[0], g = ups[0];
    const int64_t vocab = ctx->saved_data["vocab"].toInt(), dim = ctx->saved_data["dim"].toInt();
    const auto type = (at::ScalarType)ctx->saved_data["type"].toInt();
    c10::DeviceGuard guard(g.device());
    const Rows r = rows_of(g, dim);
    Tensor grad = at::empty({vocab, dim}, g.options().dtype(type));
    Tensor ws = workspace(api.token_embed_bwd_workspace_bytes(ids.numel(), vocab, dim), g);
    check(api.token_embed_bwd(ids.data_ptr(), ids.scalar_type() == at::kLong, ids.numel(), r.p, code(g), r.pitch, vocab, dim,
                              ctx->saved_data["scale"].toDouble(), ctx->saved_data["padding"].toInt(), grad.data_ptr(), code(type), ws.data_ptr(),
                              ws.numel(), stream_of(g)), "omnihd_token_embed_bwd");
    return {grad, Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor token_embedding(const Tensor& ids, const Tensor& table, double scale, int64_t padding, py::object out_type) {
  const auto type = torch::python::detail::py_object_to_dtype(out_type);
  seen_by_autograd_alone("token_embedding", {table});
  const Tensor dense = ids.contiguous();
  return wants_grad({table}) ? Embed::apply(table, dense, scale, padding, (int64_t)type) : embed_forward(dense, table, scale, type);
}

// ---- block norms ----------------------------------------------------------------------------------------------------------------
struct Join {                                       // what the forward and the backward share
  double scale, eps;
  int64_t kind, per_gate;
  at::ScalarType act;
};
struct JoinRows {
  Rows x, y, gate;
  Tensor post, next;
  int64_t dim, rows;
};
JoinRows join_rows(const Tensor& x, const Tensor& y, const Tensor& post, const Tensor& gate, const Tensor& next, const Join& j) {
  JoinRows r;
  r.dim = x.size(-1);
  r.rows = x.numel() / r.dim;
  r.x = rows_of(x, r.dim);
  r.y = rows_of(y, r.dim);
  r.gate = j.kind == 2 ? rows_of(gate, 1) : rows_of(gate, r.dim);
  if (j.kind == 2 && r.gate.pitch != 1) r.gate = rows_of(gate.contiguous(), 1);      // (one number a row: dense)
  if (post.defined()) r.post = post.contiguous();
  if (next.defined()) r.next = next.contiguous();
  return r;
}

variable_list join_forward(const Tensor& x, const Tensor& y, const Tensor& post, const Tensor& gate, const Tensor& next, const Join& j, Tensor* stats) {
  c10::DeviceGuard guard(x.device());
  const JoinRows r = join_rows(x, y, post, gate, next, j);
  Tensor out, h;
  if (y.defined()) out = dense_like(x);
  if (next.defined()) h = at::empty(x.sizes(), x.options().dtype(j.act));
  if (stats) *stats = at::empty({r.rows, 2}, x.options().dtype(at::kFloat));
  if (r.rows)
    check(api.block_join_fwd(r.x.p, r.x.pitch, code(x), r.y.p, r.y.pitch, code(j.act), ptr(r.post), post.defined() ? code(post) : 0, r.gate.p,
                             gate.defined() ? code(gate) : 0, (int)j.kind, r.gate.pitch, j.per_gate, ptr(r.next), next.defined() ? code(next) : 0, j.scale,
                             j.eps, r.rows, r.dim, ptr(out), ptr(h), stats ? static_cast<float*>(stats->data_ptr()) : nullptr, stream_of(x)),
          "omnihd_block_join_fwd");
  variable_list got;
  if (out.defined()) got.push_back(out);
  if (h.defined()) got.push_back(h);
  return got;
}

struct BlockJoin : public Function<BlockJoin> {
  static variable_list forward(AutogradContext* ctx, Tensor x, Maybe y_, Maybe post_, Maybe gate_, Maybe next_, double scale, double eps,
                               int64_t kind, int64_t per_gate, int64_t act) {
    const Tensor y = of(y_), post = of(post_), gate = of(gate_), next = of(next_);
    Tensor stats;
    variable_list got = join_forward(x, y, post, gate, next, Join{scale, eps, kind, per_gate, (at::ScalarType)act}, &stats);
    ctx->save_for_backward({x, y, post, gate, next, stats});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["kind"] = kind;
    ctx->saved_data["per_gate"] = per_gate;
    ctx->saved_data["act"] = act;
    ctx->set_materialize_grads(false);
    return got;
  }
  static variable_list backward(AutogradContext* ctx, variable_list ups) {
    no_second_order("block_join");
    variable_list grads(10);
    const variable_list in = ctx->get_saved_variables();
    const Tensor &x = in[0], &y = in[1], &post = in[2], &gate = in[3], &next = in[4], &stats = in[5];
    const Tensor d_out = y.defined() ? ups[0] : Tensor(), d_h = next.defined() ? ups[y.defined() ? 1 : 0] : Tensor();
    if (!d_out.defined() && !d_h.defined()) return grads;
    const Join j{ctx->saved_data["scale"].toDouble(), 0., ctx->saved_data["kind"].toInt(), ctx->saved_data["per_gate"].toInt(),
                 (at::ScalarType)ctx->saved_data["act"].toInt()};
    c10::DeviceGuard guard(x.device());
    const JoinRows r = join_rows(x, y, post, gate, next, j);
    size_t given = 0;                               // (autograd counts the tensors that were given)
    for (int k = 0; k < 5; ++k)
      if (in[k].defined() && ctx->needs_input_grad(given++)) grads[k] = r.rows ? dense_like(in[k]) : at::zeros(in[k].sizes(), in[k].options());
    if (r.rows == 0) return grads;
    const Rows go = rows_of(d_out, r.dim), gh = rows_of(d_h, r.dim);
    Tensor ws = workspace(api.block_join_bwd_workspace_bytes(r.rows, r.dim, (int)j.kind, j.per_gate, y.defined()), x);
    check(api.block_join_bwd(r.x.p, r.x.pitch, code(x), r.y.p, r.y.pitch, code(j.act), ptr(r.post), post.defined() ? code(post) : 0, r.gate.p,
                             gate.defined() ? code(gate) : 0, (int)j.kind, r.gate.pitch, j.per_gate, ptr(r.next), next.defined() ? code(next) : 0, j.scale,
                             r.rows, r.dim, static_cast<const float*>(stats.data_ptr()), go.p, go.pitch, gh.p, gh.pitch, ptr(grads[0]), ptr(grads[1]),
                             ptr(grads[2]), ptr(grads[3]), ptr(grads[4]), ws.data_ptr(), ws.numel(), stream_of(x)), "omnihd_block_join_bwd");
    return grads;
  }
};

variable_list block_join(const Tensor& x, const Maybe& y, const Maybe& post, const Maybe& gate, const Maybe& next, double scale, double eps,
                         int64_t kind, int64_t per_gate, py::object act) {
  const auto type = torch::python::detail::py_object_to_dtype(act);
  const Tensor y_ = of(y), post_ = of(post), gate_ = of(gate), next_ = of(next);
  seen_by_autograd_alone(y_.defined() ? "block_join" : "block_norm", {x, y_, post_, gate_, next_});
  if (wants_grad({x, y_, post_, gate_, next_})) return BlockJoin::apply(x, y, post, gate, next, scale, eps, kind, per_gate, (int64_t)type);
  return join_forward(x, y_, post_, gate_, next_, Join{scale, eps, kind, per_gate, type}, nullptr);
}

// ---- distillation ----------------------------------------------------------------------------------------------------------------
// one launch over the rows: the loss (one number, or one a row; `loss` unset: not wanted) and / or the gradient into `grad`
void distill_run(const Tensor& z, const Tensor& t, const Tensor& ids, const Tensor& weight, const Tensor& avg, double temperature, double factor,
                 bool per_row, Tensor* loss, const Tensor& grad, const Tensor& up, bool skip_if_one) {
  c10::DeviceGuard guard(z.device());
  const int64_t vocab = z.size(-1), top = t.size(-1), rows = z.numel() / vocab;
  const Rows zr = rows_of(z, vocab), tr = rows_of(t, top), ir = rows_of(ids, top);
  Tensor ws;
  if (loss) {
    *loss = at::empty(per_row ? z.sizes().slice(0, z.dim() - 1) : at::IntArrayRef(), z.options().dtype(at::kFloat));
    if (!per_row) ws = workspace(api.topk_distill_workspace_bytes(rows, vocab, top, code(z)), z);
  }
  float* to = loss ? static_cast<float*>(loss->data_ptr()) : nullptr;
  check(api.topk_distill(zr.p, code(z), zr.pitch, tr.p, code(t), tr.pitch, ir.p, ids.scalar_type() == at::kLong, ir.pitch,
                         static_cast<const float*>(ptr(weight)), rows, vocab, top, temperature, factor, static_cast<const float*>(ptr(avg)),
                         static_cast<const float*>(ptr(up)), up.defined() && per_row, skip_if_one, ptr(grad), vocab, per_row ? to : nullptr,
                         per_row ? nullptr : to, ptr(ws), ws.defined() ? ws.numel() : 0, stream_of(z)), "omnihd_topk_distill");
}

// The forward of a summed loss writes the logits' gradient too, while the row is in registers; the backward returns it, after a launch that
// writes it again where the gradient arriving at the loss is not 1.  That second form alone (two passes instead of one and a half) serves
// per-row losses, whose upstream gradient is not known in the forward, stream capture, whose replays may be of the backward alone,
// every further backward pass over the same forward, and forwards under saved-tensor hooks: the gradient is no saved tensor, so that the hooks could
// not take it off the device, and one of the logits' size would be held from the forward that they are meant to relieve.
struct Distill : public Function<Distill> {
  static Tensor forward(AutogradContext* ctx, Tensor z, Tensor t, Tensor ids, Maybe weight_, Maybe avg_, double temperature, double factor,
                        bool per_row) {
    const Tensor weight = of(weight_), avg = of(avg_);
    c10::DeviceGuard guard(z.device());             // (whether a stream is captured is asked of the logits' device)
    const bool fresh = !per_row && !saved_elsewhere() && !capturing();
    Tensor loss, grad;
    if (fresh) grad = dense_like(z);
    distill_run(z, t, ids, weight, avg, temperature, factor, per_row, &loss, grad, Tensor(), false);
    ctx->save_for_backward({z, t, ids, weight, avg});
    ctx->saved_data["temperature"] = temperature;
    ctx->saved_data["factor"] = factor;
    ctx->saved_data["per_row"] = per_row;
    if (fresh) ctx->saved_data["grad"] = grad;      // (not among the saved variables: its next holder may write to it)
    return loss;
  }
  static variable_list backward(AutogradContext* ctx, variable_list ups) {
    no_second_order("topk_distill_loss");
    const variable_list in = ctx->get_saved_variables();
    Tensor grad;
    const auto kept = ctx->saved_data.find("grad");
    if (kept != ctx->saved_data.end()) {
      if (!capturing()) grad = kept->second.toTensor();
      ctx->saved_data.erase(kept);                  // (a captured backward has no use for it)
    }
    const bool in_place = grad.defined();
    if (!in_place) grad = dense_like(in[0]);
    distill_run(in[0], in[1], in[2], in[3], in[4], ctx->saved_data["temperature"].toDouble(), ctx->saved_data["factor"].toDouble(),
                ctx->saved_data["per_row"].toBool(), nullptr, grad, ups[0].contiguous(), in_place);
    variable_list grads(8);
    grads[0] = grad;
    return grads;
  }
};

Tensor topk_distill(const Tensor& z, const Tensor& t, const Tensor& ids, const Maybe& weight, const Maybe& avg, double temperature, double factor,
                    bool per_row) {
  const Tensor teacher = t.detach(), w = of(weight), a = of(avg);
  seen_by_autograd_alone("topk_distill_loss", {z, t, w, a});
  if (wants_grad({z})) return Distill::apply(z, teacher, ids, weight, avg, temperature, factor, per_row);
  Tensor loss;
  distill_run(z, teacher, ids, w, a, temperature, factor, per_row, &loss, Tensor(), Tensor(), false);
  return loss;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("bind", &bind);
  m.def("token_embedding", &token_embedding);
  m.def("block_join", &block_join);
  m.def("topk_distill", &topk_distill);
}
