// Autograd nodes of the training operators around the mixers (row norms, dropout, cross entropy from hidden
// states), over the C ABI of libmotif_hip.so.  In C++ because a step calls them by the dozen: as
// Python Functions a norm's forward and backward kept the host 106 us (64 x 768; torch's own op beside it 60), most of
// it in Python on the engine's thread; so they keep it 59.  Arguments are checked by the callers in
// motif/ops; here they are tensors of one device with features beside each other.
#include <torch/extension.h>

#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/graph_task.h>

#include <unordered_set>

#include "../../include/motif_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> OptTensor;

int dtype_code(const Tensor &t) {
  switch (t.scalar_type()) {
    case at::kFloat: return MOTIF_F32;
    case at::kBFloat16: return MOTIF_BF16;
    default: return MOTIF_F16;
  }
}

void *stream_of(const Tensor &t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

void check(int rc, const char *what) {
  if (rc == MOTIF_OK) return;
  const std::string msg = std::string(what) + ": " + motif_last_error();
  TORCH_CHECK_VALUE(rc != MOTIF_ERR_INVALID, msg);
  TORCH_CHECK_NOT_IMPLEMENTED(rc != MOTIF_ERR_UNSUPPORTED, msg);
  TORCH_CHECK(false, msg);
}

// Refuses a backward that is captured while a gradient of it would be summed up on the default stream.  A leaf's
// summing node lives as long as any graph of that leaf and keeps the stream that it was made on: where an eager
// loss of the same leaves is still held, the engine would make the default stream wait for the capturing one, which
// breaks the capture and can end the process.  So this runs before a gradient is handed on, over the nodes that the pass will
// reach, and only while capturing.
void refuse_stale_leaves(const char *what) {
  using namespace torch::autograd;
  if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
  const auto *wanted = get_current_graph_task_exec_info();  // (empty: every node)
  std::vector<Node *> next = {get_current_node().get()};
  std::unordered_set<Node *> seen;
  while (!next.empty()) {
    Node *node = next.back();
    next.pop_back();
    if (!node || !seen.insert(node).second) continue;
    if (seen.size() > 1 && wanted && !wanted->empty()) {
      const auto it = wanted->find(node);
      if (it == wanted->end() || !it->second.should_execute()) continue;
    }
    if (dynamic_cast<AccumulateGrad *>(node)) {
      const auto stream = node->stream();
      TORCH_CHECK(!stream || stream->id() != 0, what, ": this backward is being captured while a loss of the same leaves, made on the "
                  "default stream, is still held: delete it (and what else holds its graph) before the capture");
    }
    for (const auto &edge : node->next_edges()) next.push_back(edge.function.get());
  }
}

// A gradient that came in with a forward-mode tangent, which the kernels would lose
bool has_tangent(const Tensor &t) { return t._fw_grad(/*level=*/0).defined(); }

// Null for an argument left out, and for nothing else: subclasses without memory of their own (distributed tensors, fake
// ones) have null pointers too.
void *ptr(const Tensor &t) {
  if (!t.defined()) return nullptr;
  void *p = t.data_ptr();
  TORCH_CHECK_VALUE(p || t.numel() == 0, "the kernels take tensors with memory of their own: this one has no memory (a distributed or fake tensor)");
  return p;
}
Tensor given(const OptTensor &t) { return t.has_value() ? *t : Tensor(); }

// t as it lies in memory: torch's negative views (the imaginary part of a conjugate, say) hold their sign beside it, its
// zero tensors (which come up in derivatives) have no memory
Tensor plain(const Tensor &t) {
  if (!t.defined()) return t;
  return t._is_zerotensor() ? t.clone() : t.is_neg() ? t.resolve_neg() : t;
}

// ------------------------------------------------------------ row norms
// x as rows of D: its stride where the leading dimensions lie regularly, else a contiguous copy
struct Rows {
  Tensor t;
  int64_t n, D, stride;
  explicit Rows(const Tensor &x) : t(x), D(x.size(-1)) {
    n = x.numel() / D;
    stride = D;
    const auto ok = [&] {
      if (D > 1 && x.stride(-1) != 1) return false;
      int64_t inner = -1;  // stride that a row further out has to have
      for (int64_t i = x.dim() - 2; i >= 0; --i) {
        if (x.size(i) == 1) continue;
        if (inner < 0) stride = x.stride(i);
        else if (x.stride(i) != inner) return false;
        inner = x.stride(i) * x.size(i);
      }
      return true;
    };
    if (!x.is_contiguous() && !ok()) t = x.contiguous(), stride = D;
  }
};

void norm_forward(const Rows &r, const Tensor &w, const Tensor &b, const Tensor &y, const Tensor &stats, double eps, bool layer) {
  if (r.n == 0) return;
  float *rstd = stats.defined() ? stats.data_ptr<float>() : nullptr;
  check(motif_row_norm_fwd(ptr(r.t), r.stride, ptr(w), ptr(b), y.data_ptr(), r.D, rstd, layer && rstd ? rstd + r.n : nullptr,
                           static_cast<int>(r.n), static_cast<int>(r.D), static_cast<float>(eps), layer, dtype_code(y), stream_of(y)),
        "motif_row_norm_fwd");
}

// The gradients in torch ops, all in fp32: where they have to carry a graph of their own (create_graph) or a tangent, which
// the kernels' do not, and for several gradients at once (is_grads_batched), which have no memory for a kernel to read.
variable_list norm_grads_torch(const Tensor &x, const Tensor &w, const Tensor &grad, double eps, bool layer, const bool (&need)[3]) {
  Tensor h = x.to(at::kFloat);
  if (layer) h = h - h.mean(-1, true);
  const Tensor r = (h.square().mean(-1, true) + eps).rsqrt(), dy = grad.to(at::kFloat);
  h = h * r;
  variable_list out(5);
  if (need[0]) {
    const Tensor g = w.defined() ? dy * w.to(at::kFloat) : dy;
    Tensor dx = g - h * (g * h).mean(-1, true);
    if (layer) dx = dx - g.mean(-1, true);
    out[0] = (dx * r).to(x.scalar_type());
  }
  const auto rows = [&](const Tensor &t) { return t.reshape({-1, x.size(-1)}).sum(0).to(x.scalar_type()); };
  if (need[1]) out[1] = rows(dy * h);
  if (need[2]) out[2] = rows(dy);
  return out;
}

struct RowNorm : torch::autograd::Function<RowNorm> {
  static Tensor forward(AutogradContext *ctx, const Tensor &x, const OptTensor &weight, const OptTensor &bias, double eps, bool layer) {
    const c10::DeviceGuard guard(x.device());
    const Rows r(x);
    const Tensor w = given(weight), b = given(bias), y = at::empty(x.sizes(), x.options());
    const Tensor stats = at::empty({(layer ? 2 : 1) * r.n}, x.options().dtype(at::kFloat));
    norm_forward(r, w, b, y, stats, eps, layer);
    ctx->save_for_backward({x, w, b, stats});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["layer"] = layer;
    return y;
  }

  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &b = saved[2], &stats = saved[3];
    const bool layer = ctx->saved_data["layer"].toBool();
    // (the inputs are counted without the absent ones)
    const bool need[3] = {ctx->needs_input_grad(0), w.defined() && ctx->needs_input_grad(1),
                          b.defined() && ctx->needs_input_grad(w.defined() ? 2 : 1)};
    if (!grads[0].defined()) return variable_list(5);
    refuse_stale_leaves("row norm");
    if (at::GradMode::is_enabled() || !grads[0].has_storage() || has_tangent(grads[0]))
      return norm_grads_torch(x, w, grads[0], ctx->saved_data["eps"].toDouble(), layer, need);
    const c10::DeviceGuard guard(x.device());
    const Rows r(x), dy(plain(grads[0]));
    const Tensor dx = need[0] ? at::empty(x.sizes(), x.options()) : Tensor();
    const Tensor dw = need[1] ? at::empty({r.D}, x.options()) : Tensor(), db = need[2] ? at::empty({r.D}, x.options()) : Tensor();
    if (r.n == 0) {
      if (need[1]) dw.zero_();
      if (need[2]) db.zero_();
      return {dx, dw, db, Tensor(), Tensor()};
    }
    Tensor ws;
    size_t bytes = 0;
    if (need[1] || need[2]) {
      bytes = motif_row_norm_bwd_workspace_bytes(static_cast<int>(r.n), static_cast<int>(r.D), layer);
      ws = at::empty({static_cast<int64_t>(bytes / 4)}, stats.options());
    }
    const float *rstd = stats.data_ptr<float>();
    check(motif_row_norm_bwd(ptr(dy.t), dy.stride, ptr(r.t), r.stride, ptr(w), rstd, layer ? rstd + r.n : nullptr, ptr(dx),
                             r.D, ptr(dw), ptr(db), static_cast<int>(r.n), static_cast<int>(r.D), layer, ptr(ws), bytes,
                             dtype_code(x), stream_of(x)),
          "motif_row_norm_bwd");
    return {dx, dw, db, Tensor(), Tensor()};
  }
};

bool wants_grad(std::initializer_list<const Tensor *> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor *t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

Tensor row_norm(const Tensor &input, const OptTensor &weight, const OptTensor &bias, double eps, bool layer) {
  const Tensor x = plain(input), w = weight ? plain(weight->contiguous()) : Tensor(), b = bias ? plain(bias->contiguous()) : Tensor();
  if (wants_grad({&x, &w, &b}))
    return RowNorm::apply(x, w.defined() ? OptTensor(w) : OptTensor(), b.defined() ? OptTensor(b) : OptTensor(), eps, layer);
  const c10::DeviceGuard guard(x.device());
  const Tensor y = at::empty(x.sizes(), x.options());
  norm_forward(Rows(x), w, b, y, Tensor(), eps, layer);
  return y;
}

// ------------------------------------------------------------ dropout
Tensor dropout_launch(const Tensor &x, const Tensor &residual, double p, int64_t seed, const Tensor &seed_dev) {
  const Tensor y = at::empty(x.sizes(), x.options());
  const double t = std::nearbyint(p * 4294967296.0);  // (half to even, as Python's round)
  const bool none = t >= 4294967296.0;  // (no word is as large: a scale of 0 drops every element)
  check(motif_dropout_add(ptr(x), ptr(residual), ptr(y), x.numel(), none ? 0 : static_cast<uint32_t>(t), none ? 0.f : static_cast<float>(1 / (1 - p)),
                          static_cast<uint64_t>(seed), static_cast<const int64_t *>(ptr(seed_dev)), dtype_code(x), stream_of(x)),
        "motif_dropout_add");
  return y;
}

struct DropoutAdd : torch::autograd::Function<DropoutAdd> {
  static Tensor forward(AutogradContext *ctx, const Tensor &x, const OptTensor &residual, double p, int64_t seed, const OptTensor &seed_dev) {
    const c10::DeviceGuard guard(x.device());
    ctx->save_for_backward({given(seed_dev)});
    ctx->saved_data["p"] = p;
    ctx->saved_data["seed"] = seed;
    ctx->saved_data["added"] = residual.has_value();
    return dropout_launch(x.contiguous(), residual ? residual->contiguous() : Tensor(), p, seed, given(seed_dev));
  }

  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "dropout_add has no second derivatives");
    const Tensor seed_dev = ctx->get_saved_variables()[0];
    const Tensor &dy = grads[0];
    variable_list out(5);
    if (!dy.defined()) return out;
    TORCH_CHECK_NOT_IMPLEMENTED(!has_tangent(dy), "dropout_add: no forward-mode derivatives");
    refuse_stale_leaves("dropout_add");
    const c10::DeviceGuard guard(dy.device());
    if (ctx->needs_input_grad(0))
      out[0] = dropout_launch(plain(dy.contiguous()), Tensor(), ctx->saved_data["p"].toDouble(), ctx->saved_data["seed"].toInt(), seed_dev);
    if (ctx->saved_data["added"].toBool() && ctx->needs_input_grad(1)) out[1] = dy;
    return out;
  }
};

Tensor dropout_add(const Tensor &x, const OptTensor &residual, double p, int64_t seed, const OptTensor &seed_dev) {
  return DropoutAdd::apply(plain(x), residual ? OptTensor(plain(*residual)) : OptTensor(), p, seed,
                           seed_dev ? OptTensor(plain(*seed_dev)) : OptTensor());
}

// ------------------------------------------------------------ cross entropy
// x [N, d] with features beside each other, weight [V, d] with rows that do not overlap, labels [N].  Kept for the
// backward: the labelled rows of x (a copy), the weight and 16 bytes a row.
struct LinearCE : torch::autograd::Function<LinearCE> {
  static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &weight, const Tensor &labels, int64_t ignore, int64_t reduction) {
    const c10::DeviceGuard guard(x.device());
    const int N = static_cast<int>(x.size(0)), d = static_cast<int>(x.size(1)), V = static_cast<int>(weight.size(0));
    const int code = dtype_code(x);
    const auto bytes = x.options().dtype(at::kByte);
    const Tensor rows = at::empty({static_cast<int64_t>(motif_linear_ce_rows_bytes(N, d, code))}, bytes);
    const Tensor kept = at::empty({4 * int64_t(N) + 1}, x.options().dtype(at::kInt));
    const Tensor loss = reduction == 0 ? at::empty({N}, x.options().dtype(at::kFloat)) : at::empty({}, x.options().dtype(at::kFloat));
    const size_t need = motif_linear_ce_workspace_bytes(N, d, ptr(weight), weight.stride(0), V, code, 0);
    const Tensor ws = at::empty({static_cast<int64_t>(need)}, bytes);
    check(motif_linear_ce_fwd(ptr(x), x.stride(0), ptr(weight), weight.stride(0), static_cast<const int64_t *>(ptr(labels)),
                              labels.stride(0), ignore, N, d, V, static_cast<int>(reduction), rows.data_ptr(), kept.data_ptr<int>(),
                              loss.data_ptr<float>(), ws.data_ptr(), need, code, stream_of(x)),
          "motif_linear_ce_fwd");
    if (ctx) {
      ctx->save_for_backward({rows, weight, kept});
      ctx->saved_data["d"] = int64_t(d);
      ctx->saved_data["N"] = int64_t(N);
      ctx->saved_data["reduction"] = reduction;
    }
    return loss;
  }

  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "linear_cross_entropy has no second derivatives");
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &rows = saved[0], &weight = saved[1], &kept = saved[2];
    const Tensor dloss = plain(grads[0]);
    variable_list out(5);
    if (!dloss.defined()) return out;
    TORCH_CHECK_NOT_IMPLEMENTED(!has_tangent(dloss), "linear_cross_entropy: no forward-mode derivatives");
    refuse_stale_leaves("linear_cross_entropy");
    const c10::DeviceGuard guard(weight.device());
    const int64_t N = ctx->saved_data["N"].toInt(), d = ctx->saved_data["d"].toInt(), V = weight.size(0);
    const int reduction = static_cast<int>(ctx->saved_data["reduction"].toInt()), code = dtype_code(weight);
    const Tensor dx = ctx->needs_input_grad(0) ? at::empty({N, d}, weight.options()) : Tensor();
    const Tensor dw = ctx->needs_input_grad(1) ? at::empty({V, d}, weight.options()) : Tensor();
    const size_t need = motif_linear_ce_workspace_bytes(static_cast<int>(N), static_cast<int>(d), ptr(weight), weight.stride(0),
                                                        static_cast<int>(V), code, 1);
    const Tensor ws = at::empty({static_cast<int64_t>(need)}, weight.options().dtype(at::kByte));
    check(motif_linear_ce_bwd(rows.data_ptr(), ptr(weight), weight.stride(0), kept.data_ptr<int>(), static_cast<const float *>(ptr(dloss)),
                              reduction == 0 ? dloss.stride(0) : 0, static_cast<int>(N), static_cast<int>(d), static_cast<int>(V),
                              reduction, ptr(dx), ptr(dw), ws.data_ptr(), need, code, stream_of(weight)),
          "motif_linear_ce_bwd");
    out[0] = dx;
    out[1] = dw;
    return out;
  }
};

Tensor linear_ce(const Tensor &states, const Tensor &vocabulary, const Tensor &targets, int64_t ignore, int64_t reduction) {
  const Tensor x = plain(states), weight = plain(vocabulary), labels = plain(targets);
  if (wants_grad({&x, &weight})) return LinearCE::apply(x, weight, labels, ignore, reduction);
  return LinearCE::forward(nullptr, x, weight, labels, ignore, reduction);
}

}  // namespace

PYBIND11_MODULE(_autograd_nodes, m) {
  const auto release = pybind11::call_guard<pybind11::gil_scoped_release>();
  m.def("row_norm", &row_norm, release);
  m.def("dropout_add", &dropout_add, release);
  m.def("linear_ce", &linear_ce, release);
}
