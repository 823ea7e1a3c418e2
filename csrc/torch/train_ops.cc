// train_ops.cc — torch bindings and autograd of the training-step kernels:
// embedding, gated residual norm, 8-bit activation checkpoints.
//
// Arguments are checked in the order type, shape, size, device, so that a
// wrong call is refused the same way with or without a GPU.  Kernels run on
// the current stream of their tensors' device; workspaces and saved tensors
// come from torch's allocator, so calls may be captured into a graph.

#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <algorithm>
#include <array>
#include <memory>
#include <mutex>
#include <optional>
#include <tuple>
#include <vector>

#include "../hip/train_kernels.h"

namespace baguanet {
namespace {

using torch::Tensor;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

constexpr int64_t kMaxRows = int64_t(1) << 30;

hipStream_t stream_of(const Tensor& t) {
  return (hipStream_t)c10::cuda::getCurrentCUDAStream(t.get_device()).stream();
}

void check_launch(hipError_t e, const char* what) {
  TORCH_CHECK(e == hipSuccess, what, ": ", hipGetErrorString(e));
}

bool is_act_type(at::ScalarType t) {
  return t == at::kFloat || t == at::kBFloat16 || t == at::kHalf;
}

ElemType elem(at::ScalarType t) {
  return t == at::kFloat      ? ElemType::kF32
         : t == at::kBFloat16 ? ElemType::kBF16
                              : ElemType::kF16;
}

// A recorder would see the tensors that are made here and not the kernels that
// fill them: its recording would give whatever their memory holds.
void check_not_recorded(const char* op) {
  using c10::impl::TorchDispatchModeKey;
  bool recorded = torch::jit::tracer::isTracing() ||
                  c10::impl::tls_is_dispatch_key_included(
                      c10::DispatchKey::PreDispatch);
  if (c10::impl::dispatch_mode_enabled())
    for (const auto key : {TorchDispatchModeKey::FAKE,
                           TorchDispatchModeKey::PROXY,
                           TorchDispatchModeKey::FUNCTIONAL})
      recorded |= c10::impl::TorchDispatchModeTLS::get_mode(key).has_value();
  TORCH_CHECK(!recorded, op, ": cannot be recorded by a tracer");
}

// Kernels read a tensor's memory: it has to be there, and to hold the values
// themselves.  Wrappers of other tensors and tensors that only stand for zeros
// have none, and a storage may have been freed or cut under its tensor.
bool has_memory(const Tensor& t) {
  if (t.numel() == 0) return true;
  int64_t last = t.storage_offset();
  for (int64_t d = 0; d < t.dim(); d++) last += (t.size(d) - 1) * t.stride(d);
  const c10::Storage& s = t.storage();
  return s.data() != nullptr &&
         (size_t)(last + 1) * t.element_size() <= s.nbytes();
}

void check_plain(const Tensor& t, const char* op, const char* name) {
  TORCH_CHECK(t.layout() == at::kStrided, op, ": ", name, " must be dense");
  TORCH_CHECK(!t.is_neg(), op, ": ", name,
              " is a view that stands for its negative; resolve_neg() it");
  TORCH_CHECK(has_memory(t), op, ": ", name, " holds no values of its own");
}

void check_act(const Tensor& t, const char* op, const char* name) {
  TORCH_CHECK(t.defined(), op, ": ", name, " is missing");
  TORCH_CHECK(is_act_type(t.scalar_type()), op, ": ", name,
              " must be float32, bfloat16 or float16, not ", t.scalar_type());
  check_plain(t, op, name);
}

void check_device(const Tensor& t, const Tensor& on, const char* op,
                  const char* name) {
  TORCH_CHECK(t.is_cuda(), op, ": ", name, " must be on the GPU");
  TORCH_CHECK(t.device() == on.device(), op, ": ", name, " is on ",
              t.device(), ", expected ", on.device());
}

// Whether a gradient will be asked of any of these.  Without one an operator
// runs alone, keeps nothing and makes no graph.
bool wants_grad(const char* op, std::initializer_list<const Tensor*> tensors) {
  for (const Tensor* t : tensors)
    TORCH_CHECK(!t || !t->defined() || !t->_fw_grad(0).defined(), op,
                ": no forward-mode gradient");
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : tensors)
    if (t && t->defined() && t->requires_grad()) return true;
  return false;
}

const Tensor* get(const OptTensor& t) { return t ? &*t : nullptr; }

// A tensor that autograd gives, with its values in memory as they are.
Tensor plain(const Tensor& given) {
  if (given._is_zerotensor()) return at::zeros(given.sizes(), given.options());
  TORCH_CHECK(has_memory(given),
              "a gradient or a kept tensor holds no values of its own");
  return given.resolve_neg();
}

// An operator's backward pass: a node of the graph that keeps N tensors.  As a
// node of its own it has its numbers as members; through torch's Function, with
// its context of named values, a call with a gradient took 5 us longer.
template <size_t N>
class OpNode : public torch::autograd::Node {
 public:
  // Only once t has been written: a hook may copy it here.
  void keep(size_t i, const Tensor& t) {
    saved_[i] = torch::autograd::SavedVariable(t, false);
    if (t.defined())
      saved_as_[i] = {t.scalar_type(), t.device(), t.is_contiguous(),
                      is_aligned(t), at::DimVector(t.sizes())};
  }

  void release_variables() override {
    const std::lock_guard<std::mutex> lock(mutex_);
    for (auto& s : saved_) s.reset_data();
  }

 protected:
  std::array<Tensor, N> kept(const char* op) {
    check_not_recorded(op);
    TORCH_CHECK(!at::GradMode::is_enabled(), op,
                ": its gradient cannot be differentiated again");
    const std::lock_guard<std::mutex> lock(mutex_);
    std::array<Tensor, N> t;
    for (size_t i = 0; i < N; i++) {
      t[i] = saved_[i].unpack();
      if (t[i].defined()) t[i] = as_saved(op, t[i], saved_as_[i]);
    }
    return t;
  }

 private:
  struct Meta {
    at::ScalarType type = at::kByte;
    at::Device device = at::kCPU;
    bool contiguous = false, aligned = false;
    at::DimVector sizes;
  };

  // A kept tensor as it was kept.  A hook may give another one back, and a
  // parameter's data may have been exchanged (a module's half(), its move to
  // another device) without counting as a change in place; but the kernels read
  // it by the type, place and sizes that it had, weights and codes without gaps
  // and codes in whole words.
  static Tensor as_saved(const char* op, const Tensor& t, const Meta& m) {
    TORCH_CHECK(t.layout() == at::kStrided && t.scalar_type() == m.type &&
                    t.device() == m.device && t.sizes() == m.sizes,
                op, ": a kept tensor has become ", t.scalar_type(), " ",
                t.sizes(), " on ", t.device(), " from ", m.type, " ",
                at::IntArrayRef(m.sizes), " on ", m.device);
    Tensor own = plain(t);
    if (m.contiguous) own = own.contiguous();
    return m.aligned && !is_aligned(own) ? own.clone() : own;
  }

  static bool is_aligned(const Tensor& t) {
    return ((uintptr_t)t.const_data_ptr() & 15) == 0;
  }

  std::array<torch::autograd::SavedVariable, N> saved_;
  std::array<Meta, N> saved_as_;
};

// A node that gives gradients to `inputs`, in their order.
template <typename Op, typename... T>
std::shared_ptr<Op> make_node(const T&... inputs) {
  std::shared_ptr<Op> node(new Op(), torch::autograd::deleteNode);
  node->set_next_edges(torch::autograd::collect_next_edges(inputs...));
  return node;
}

// A tensor as rows of its last dimension: unit stride within a row and one
// stride between rows.  Others are copied.
struct Rows {
  Tensor t;
  int64_t stride;
};

Rows as_rows(const Tensor& given) {
  const Tensor t = plain(given);
  const int64_t dim = t.size(-1);
  bool ok = dim <= 1 || t.stride(-1) == 1;
  int64_t stride = dim, next = -1;
  for (int64_t d = t.dim() - 2; d >= 0 && ok; d--) {
    if (t.size(d) == 1) continue;
    if (next < 0)
      stride = t.stride(d);
    else
      ok = t.stride(d) == next;
    next = t.stride(d) * t.size(d);
  }
  if (ok) return {t, stride};
  return {t.contiguous(), dim};
}

int64_t rows_of(const Tensor& t) {
  int64_t r = 1;
  for (int64_t d = 0; d < t.dim() - 1; d++) r *= t.size(d);
  return r;
}

Tensor empty_bytes(size_t bytes, const Tensor& like) {
  return at::empty({(int64_t)bytes}, like.options().dtype(at::kByte));
}

// ---------------------------------------------------------------------------
// embedding

Tensor lookup(const Tensor& weight, const Tensor& tok, double scale,
              at::ScalarType out_type) {
  const c10::OptionalDeviceGuard guard(weight.device());
  const Tensor w = weight.stride(-1) == 1 ? weight : weight.contiguous();
  c10::SmallVector<int64_t, 6> sizes(tok.sizes().begin(), tok.sizes().end());
  sizes.push_back(weight.size(1));
  Tensor out = at::empty(sizes, weight.options().dtype(out_type));
  EmbeddingFwd a = {};
  a.weight = w.data_ptr();
  a.tokens = tok.data_ptr();
  a.out = out.data_ptr();
  a.vocab = w.size(0);
  a.dim = w.size(1);
  a.n = tok.numel();
  a.wstride = w.stride(0);
  a.scale = (float)scale;
  a.tok64 = tok.scalar_type() == at::kLong;
  a.wtype = elem(w.scalar_type());
  a.otype = elem(out_type);
  check_launch(embedding_forward(a, stream_of(w)), "embedding");
  return out;
}

struct EmbeddingNode : OpNode<1> {
  int64_t vocab, padding;
  double scale;
  at::ScalarType type;

  std::string name() const override { return "EmbeddingBackward"; }

  variable_list apply(variable_list&& grads) override {
    const Tensor tok = kept("embedding")[0];
    if (!grads[0].defined()) return {Tensor()};
    const Rows dout = as_rows(grads[0]);
    const c10::OptionalDeviceGuard guard(dout.t.device());
    EmbeddingBwd a = {};
    a.vocab = vocab;
    a.dim = dout.t.size(-1);
    a.n = tok.numel();
    Tensor dw = at::empty({a.vocab, a.dim}, dout.t.options().dtype(type));
    const Tensor ws =
        empty_bytes(embedding_workspace(a.vocab, a.dim, a.n), dout.t);
    a.dout = dout.t.data_ptr();
    a.tokens = tok.data_ptr();
    a.dweight = dw.data_ptr();
    a.workspace = ws.data_ptr();
    a.dstride = dout.stride;
    a.padding = padding;
    a.scale = (float)scale;
    a.tok64 = tok.scalar_type() == at::kLong;
    a.dtype = elem(dout.t.scalar_type());
    a.wtype = elem(type);
    check_launch(embedding_backward(a, stream_of(dw)), "embedding backward");
    return {dw};
  }
};

Tensor embedding(const Tensor& weight, const Tensor& tokens, double scale,
                 std::optional<int64_t> padding_idx,
                 std::optional<at::ScalarType> out_dtype) {
  const char* op = "embedding";
  check_not_recorded(op);
  check_act(weight, op, "weight");
  TORCH_CHECK(tokens.scalar_type() == at::kLong ||
                  tokens.scalar_type() == at::kInt,
              op, ": tokens must be int64 or int32, not ",
              tokens.scalar_type());
  check_plain(tokens, op, "tokens");
  const at::ScalarType out = out_dtype ? *out_dtype : weight.scalar_type();
  TORCH_CHECK(is_act_type(out), op,
              ": out_dtype must be float32, bfloat16 or float16, not ", out);
  TORCH_CHECK(weight.dim() == 2, op, ": weight must be [vocab, dim], not ",
              weight.sizes());
  const int64_t vocab = weight.size(0);
  TORCH_CHECK(vocab <= kMaxRows && tokens.numel() <= kMaxRows, op,
              ": at most 2^30 rows and tokens");
  const bool grad = at::GradMode::is_enabled() && weight.requires_grad();
  TORCH_CHECK(!grad || vocab == 0 ||
                  weight.size(1) < kEmbeddingMaxGrad / vocab,
              op, ": a table with a gradient has fewer than 2^35 elements");
  int64_t padding = -1;
  if (padding_idx) {
    padding = *padding_idx < 0 ? *padding_idx + vocab : *padding_idx;
    TORCH_CHECK(padding >= 0 && padding < vocab, op, ": padding_idx ",
                *padding_idx, " is outside a table of ", vocab, " rows");
  }
  check_device(weight, weight, op, "weight");
  check_device(tokens, weight, op, "tokens");
  const Tensor tok = tokens.contiguous();
  if (!wants_grad(op, {&weight})) return lookup(weight, tok, scale, out);
  const auto node = make_node<EmbeddingNode>(weight);
  node->vocab = vocab;
  node->padding = padding;
  node->scale = scale;
  node->type = weight.scalar_type();
  node->keep(0, tok);
  const at::NoGradGuard no_grad;
  Tensor y = lookup(weight, tok, scale, out);
  torch::autograd::set_history(y, node);
  return y;
}

// ---------------------------------------------------------------------------
// gated residual norm

// What a gate's gradient is summed over: the kernels give one value for each
// row or element, and the gate has fewer.  In fp32, so that it is rounded once.
struct Repeated {
  std::vector<int64_t> sizes;  // of the kernels' gate, or empty: as it is
  int64_t outer, rows, inner;  // the sizes merged, `rows` to be summed
  // several dimensions apart from each other: the others first, then those
  std::vector<int64_t> order;
};

struct NormArgs {
  Tensor x, branch, gate, post, pre;  // undefined where not given
  double residual_scale, branch_scale, eps;
  Gate gmode;
  int64_t group_rows;
  bool want_h;
  Tensor gate_leaf;  // as it was given: it takes the gradient
  Repeated repeated;
};

// A gate of the sizes `own` in the place of one of `to`, with as many
// dimensions (leading ones of 1 stand for those that it lacks).
Repeated repeated_over(const std::vector<int64_t>& own,
                       const std::vector<int64_t>& to) {
  Repeated r = {};
  if (own == to) return r;
  r.sizes = to;
  r.outer = r.rows = r.inner = 1;
  bool split = false;  // an own dimension between two repeated ones
  for (size_t d = 0; d < to.size(); d++) {
    if (to[d] == 1) continue;
    if (own[d] == to[d]) {
      (r.rows == 1 ? r.outer : r.inner) *= to[d];
    } else {
      split |= r.inner != 1;
      r.rows *= to[d];
    }
  }
  if (!split) return r;
  for (const bool repeat : {false, true})
    for (size_t d = 0; d < to.size(); d++)
      if ((own[d] != to[d]) == repeat) r.order.push_back((int64_t)d);
  r.outer *= r.inner;
  r.inner = 1;
  return r;
}

// The gate's gradient from that of each row or element.
Tensor sum_repeated(const Repeated& r, const Tensor& each, const Tensor& out) {
  const Tensor in = r.order.empty() ? each : each.permute(r.order).contiguous();
  GateSum a = {};
  a.in = in.data_ptr<float>();
  a.out = out.data_ptr();
  a.outer = r.outer;
  a.rows = r.rows;
  a.inner = r.inner;
  a.type = elem(out.scalar_type());
  if (in.numel() == 0) out.zero_();
  const Tensor ws = empty_bytes(norm_gate_workspace(a), in);
  a.workspace = (float*)ws.data_ptr();
  check_launch(norm_gate_sum(a, stream_of(in)), "residual norm backward");
  return out;
}

// y (where there is a branch) and h (where it is wanted); `stats`: [2, rows],
// the reciprocals that the backward pass takes, or undefined.
std::tuple<Tensor, Tensor> run_norm(const NormArgs& n, const Tensor& stats) {
  const c10::OptionalDeviceGuard guard(n.x.device());
  const Rows xr = as_rows(n.x);
  NormFwd a = {};
  a.rows = rows_of(n.x);
  a.dim = n.x.size(-1);
  a.x = xr.t.data_ptr();
  a.xstride = xr.stride;
  a.type = elem(n.x.scalar_type());
  a.residual_scale = (float)n.residual_scale;
  a.branch_scale = (float)n.branch_scale;
  a.eps = (float)n.eps;
  a.gmode = n.gmode;
  a.group_rows = n.group_rows;
  float* kept = stats.defined() ? stats.data_ptr<float>() : nullptr;
  Tensor y, h;
  Rows br;
  if (n.branch.defined()) {
    br = as_rows(n.branch);
    a.branch = br.t.data_ptr();
    a.bstride = br.stride;
    y = at::empty(n.x.sizes(), n.x.options());
    a.y = y.data_ptr();
    if (n.gate.defined()) {
      a.gate = n.gate.data_ptr();
      a.gate32 = n.gate.scalar_type() == at::kFloat;
    }
    if (n.post.defined()) {
      a.post = n.post.data_ptr();
      a.post32 = n.post.scalar_type() == at::kFloat;
      a.rbranch = kept;
    }
  }
  if (n.want_h) {
    h = at::empty(n.x.sizes(), n.x.options());
    a.h = h.data_ptr();
    a.ry = kept ? kept + a.rows : nullptr;
    if (n.pre.defined()) {
      a.pre = n.pre.data_ptr();
      a.pre32 = n.pre.scalar_type() == at::kFloat;
    }
  }
  check_launch(norm_forward(a, stream_of(n.x)), "residual norm");
  return {y, h};
}

struct NormNode : OpNode<6> {
  double residual_scale, branch_scale;
  Gate gmode;
  int64_t group_rows;
  std::vector<int64_t> gate_sizes;
  Repeated repeated;

  std::string name() const override { return "GatedResidualNormBackward"; }

  variable_list apply(variable_list&& grads) override {
    const auto saved = kept("residual norm");
    variable_list out(5);
    const Tensor &x = saved[0], &branch = saved[1], &gate = saved[2],
                 &post = saved[3], &pre = saved[4];
    const float* stats = saved[5].data_ptr<float>();
    Tensor dy, dh;
    if (branch.defined()) {
      dy = grads[0];
      if (grads.size() > 1) dh = grads[1];
    } else {
      dh = grads[0];
    }
    if (!dy.defined() && !dh.defined()) return out;
    const Tensor& some = dy.defined() ? dy : dh;
    const c10::OptionalDeviceGuard guard(some.device());
    NormBwd a = {};
    a.rows = rows_of(some);
    a.dim = some.size(-1);
    a.type = elem(some.scalar_type());
    a.residual_scale = (float)residual_scale;
    a.branch_scale = (float)branch_scale;
    a.gmode = gmode;
    a.group_rows = group_rows;
    Rows xr, br, dyr, dhr;
    Tensor dx = at::empty(some.sizes(), some.options());
    a.dx = dx.data_ptr();
    Tensor dbranch, dgate, dpost, dpre;
    Tensor each;  // dgate, before its sum over what it is repeated over
    if (dy.defined()) {
      dyr = as_rows(dy);
      a.dy = dyr.t.data_ptr();
      a.dystride = dyr.stride;
    }
    if (dh.defined()) {
      xr = as_rows(x);
      dhr = as_rows(dh);
      a.x = xr.t.data_ptr();
      a.xstride = xr.stride;
      a.dh = dhr.t.data_ptr();
      a.dhstride = dhr.stride;
      a.ry = stats + a.rows;
      if (pre.defined()) {
        a.pre = pre.data_ptr();
        a.pre32 = pre.scalar_type() == at::kFloat;
        if (task_should_compute_output(4)) {
          dpre = at::empty(pre.sizes(), pre.options());
          a.dpre = dpre.data_ptr();
        }
      }
    }
    if (branch.defined()) {
      br = as_rows(branch);
      a.branch = br.t.data_ptr();
      a.bstride = br.stride;
      dbranch = at::empty(some.sizes(), some.options());
      a.dbranch = dbranch.data_ptr();
      if (gate.defined()) {
        a.gate = gate.data_ptr();
        a.gate32 = gate.scalar_type() == at::kFloat;
        if (task_should_compute_output(2)) {
          dgate = at::empty(gate_sizes, gate.options());
          each = dgate;
          if (!repeated.sizes.empty())
            each = at::empty(repeated.sizes, gate.options().dtype(at::kFloat));
          a.dgate = each.data_ptr();
          a.dgate32 = each.scalar_type() == at::kFloat;
        }
      }
      if (post.defined()) {
        a.post = post.data_ptr();
        a.post32 = post.scalar_type() == at::kFloat;
        a.rbranch = stats;
        if (task_should_compute_output(3)) {
          dpost = at::empty(post.sizes(), post.options());
          a.dpost = dpost.data_ptr();
        }
      }
    }
    if (a.rows == 0 || a.dim == 0) {
      for (Tensor* t : {&each, &dpost, &dpre})
        if (t->defined()) t->zero_();
    }
    const Tensor ws = empty_bytes(norm_workspace(a), dx);
    a.workspace = ws.data_ptr();
    check_launch(norm_backward(a, stream_of(dx)), "residual norm backward");
    if (each.defined() && !repeated.sizes.empty())
      sum_repeated(repeated, each, dgate);
    out[0] = dx;
    out[1] = dbranch;
    out[2] = dgate;
    out[3] = dpost;
    out[4] = dpre;
    return out;
  }
};

// y and h as run_norm gives them, with their place in the graph.
std::tuple<Tensor, Tensor> norm_with_grad(const NormArgs& n) {
  const auto node = make_node<NormNode>(n.x, n.branch, n.gate_leaf, n.post,
                                       n.pre);
  node->residual_scale = n.residual_scale;
  node->branch_scale = n.branch_scale;
  node->gmode = n.gmode;
  node->group_rows = n.group_rows;
  if (n.gate_leaf.defined()) node->gate_sizes = n.gate_leaf.sizes().vec();
  node->repeated = n.repeated;
  const at::NoGradGuard no_grad;
  const Tensor stats =
      at::empty({2, rows_of(n.x)}, n.x.options().dtype(at::kFloat));
  auto [y, h] = run_norm(n, stats);
  if (n.want_h) node->keep(0, n.x);
  node->keep(1, n.branch);
  node->keep(2, n.gate);
  node->keep(3, n.post);
  node->keep(4, n.pre);
  node->keep(5, stats);
  if (y.defined()) torch::autograd::set_history(y, node);
  if (h.defined()) torch::autograd::set_history(h, node);
  return {y, h};
}

void check_norm_input(const Tensor& x, const char* op, const char* name) {
  check_act(x, op, name);
  TORCH_CHECK(x.dim() >= 1, op, ": ", name, " must have rows, not be a scalar");
  TORCH_CHECK(x.size(-1) <= kNormMaxDim, op, ": rows of at most ", kNormMaxDim,
              " columns, not ", x.size(-1));
  TORCH_CHECK(rows_of(x) <= kMaxRows, op, ": at most 2^30 rows");
}

void check_norm_weight(const OptTensor& w, const Tensor& x, const char* op,
                       const char* name) {
  if (!w) return;
  check_act(*w, op, name);
  TORCH_CHECK(w->scalar_type() == at::kFloat ||
                  w->scalar_type() == x.scalar_type(),
              op, ": ", name, " must be float32 or of x's type, not ",
              w->scalar_type());
  TORCH_CHECK(w->dim() == 1 && w->size(0) == x.size(-1), op, ": ", name,
              " must be [", x.size(-1), "], not ", w->sizes());
}

Tensor contiguous(const OptTensor& t) {  // undefined where it is not given
  return t ? t->contiguous() : Tensor();
}

Tensor rms_norm(const Tensor& x, const OptTensor& weight, double eps) {
  const char* op = "rms_norm";
  check_not_recorded(op);
  check_norm_input(x, op, "x");
  check_norm_weight(weight, x, op, "weight");
  TORCH_CHECK(eps >= 0, op, ": eps must not be negative");
  check_device(x, x, op, "x");
  if (weight) check_device(*weight, x, op, "weight");
  const NormArgs n = {x,   {},  {},          {}, contiguous(weight), 1.0,
                      1.0, eps, Gate::kNone, 1,  true,               {},
                      {}};
  return std::get<1>(wants_grad(op, {&x, &n.pre}) ? norm_with_grad(n)
                                              : run_norm(n, Tensor()));
}

std::tuple<Tensor, OptTensor> gated_residual_norm(
    const Tensor& x, const Tensor& branch, const OptTensor& gate,
    const OptTensor& post_weight, const OptTensor& pre_weight,
    double residual_scale, double branch_scale, double eps) {
  const char* op = "gated_residual_norm";
  check_not_recorded(op);
  check_norm_input(x, op, "x");
  check_act(branch, op, "branch");
  TORCH_CHECK(branch.scalar_type() == x.scalar_type(), op,
              ": branch must have x's type ", x.scalar_type(), ", not ",
              branch.scalar_type());
  TORCH_CHECK(branch.sizes() == x.sizes(), op, ": branch must have x's shape ",
              x.sizes(), ", not ", branch.sizes());
  check_norm_weight(post_weight, x, op, "post_weight");
  check_norm_weight(pre_weight, x, op, "pre_weight");
  TORCH_CHECK(eps >= 0, op, ": eps must not be negative");
  const int64_t dim = x.size(-1), rows = rows_of(x);
  Gate mode = Gate::kNone;
  int64_t group_rows = rows > 0 ? rows : 1;
  Tensor g;
  Repeated repeated = {};
  if (gate) {
    const at::NoGradGuard no_grad;  // its gradient comes from the node
    check_act(*gate, op, "gate");
    TORCH_CHECK(gate->scalar_type() == at::kFloat ||
                    gate->scalar_type() == x.scalar_type(),
                op, ": gate must be float32 or of x's type, not ",
                gate->scalar_type());
    bool fits = gate->dim() <= x.dim();
    for (int64_t d = 1; fits && d <= gate->dim(); d++)
      fits = gate->size(-d) == 1 || gate->size(-d) == x.size(-d);
    TORCH_CHECK(fits, op, ": gate ", gate->sizes(),
                " cannot be broadcast to x ", x.sizes());
    // x's leading dimensions that the gate has too, then those it lacks
    std::vector<int64_t> lead(x.dim() - 1, 1);
    for (int64_t d = 0; d < gate->dim() - 1; d++)
      lead[lead.size() - 1 - d] = gate->size(gate->dim() - 2 - d);
    const bool wide = gate->dim() > 0 && gate->size(-1) == dim;
    size_t own = 0;
    while (own < lead.size() && lead[own] == x.size(own)) own++;
    bool prefix = true;
    for (size_t d = own; d < lead.size(); d++) prefix &= lead[d] == 1;
    Tensor t = *gate;
    if (wide && prefix) {
      group_rows = 1;
      for (size_t d = own; d < lead.size(); d++) group_rows *= x.size(d);
      mode = group_rows == 1 && rows > 1 ? Gate::kFull : Gate::kGroup;
      if (group_rows == 0) group_rows = 1;
    } else {
      // one value for each row, or any other pattern element by element
      auto to = x.sizes().vec();
      mode = wide ? Gate::kFull : Gate::kRow;
      if (!wide) to.back() = 1;
      lead.push_back(to.back());
      repeated = repeated_over(lead, to);
      t = t.expand(to);
    }
    g = t.contiguous();
  }
  check_device(x, x, op, "x");
  check_device(branch, x, op, "branch");
  if (gate) check_device(*gate, x, op, "gate");
  if (post_weight) check_device(*post_weight, x, op, "post_weight");
  if (pre_weight) check_device(*pre_weight, x, op, "pre_weight");
  const NormArgs n = {x,
                      branch,
                      g,
                      contiguous(post_weight),
                      contiguous(pre_weight),
                      residual_scale,
                      branch_scale,
                      eps,
                      mode,
                      group_rows,
                      pre_weight.has_value(),
                      gate ? *gate : Tensor(),
                      repeated};
  auto [y, h] = wants_grad(op, {&x, &branch, get(gate), &n.post, &n.pre})
                    ? norm_with_grad(n)
                    : run_norm(n, Tensor());
  return {y, n.want_h ? OptTensor(h) : OptTensor()};
}

// ---------------------------------------------------------------------------
// 8-bit activation checkpoints

int64_t pitch_of(int64_t cols) {
  return (cols + kAct8Group - 1) / kAct8Group * kAct8Group;
}

void check_act8_input(const Tensor& x, const char* op, const char* name) {
  check_act(x, op, name);
  TORCH_CHECK(x.dim() >= 1, op, ": ", name, " must have rows, not be a scalar");
  TORCH_CHECK(rows_of(x) <= kMaxRows && x.size(-1) <= kMaxRows, op,
              ": at most 2^30 rows and columns");
}

std::tuple<Tensor, Tensor> pack_rows(const Tensor& x) {
  const c10::OptionalDeviceGuard guard(x.device());
  const Rows xr = as_rows(x);
  Act8Move a = {};
  a.rows = rows_of(x);
  a.cols = x.size(-1);
  a.pitch = pitch_of(a.cols);
  const auto bytes = x.options().dtype(at::kByte);
  Tensor codes = at::empty({a.rows, a.pitch}, bytes);
  Tensor exps = at::empty({a.rows, a.pitch / kAct8Group}, bytes);
  a.x = xr.t.data_ptr();
  a.xstride = xr.stride;
  a.codes = codes.data_ptr<uint8_t>();
  a.exps = exps.data_ptr<uint8_t>();
  a.type = elem(x.scalar_type());
  check_launch(act8_pack(a, stream_of(x)), "act8_pack");
  return {codes, exps};
}

std::tuple<Tensor, Tensor> act8_pack_op(const Tensor& x) {
  check_not_recorded("act8_pack");
  check_act8_input(x, "act8_pack", "x");
  check_device(x, x, "act8_pack", "x");
  at::NoGradGuard no_grad;
  return pack_rows(x.detach());
}

// A checkpoint's parts against the rows and columns they stand for.
void check_codes(const Tensor& codes, const Tensor& exps, int64_t rows,
                 int64_t cols, const char* op) {
  const int64_t pitch = pitch_of(cols);
  TORCH_CHECK(codes.scalar_type() == at::kByte &&
                  exps.scalar_type() == at::kByte,
              op, ": codes and exponents must be bytes");
  check_plain(codes, op, "codes");
  check_plain(exps, op, "exponents");
  TORCH_CHECK(codes.dim() == 2 && codes.size(0) == rows &&
                  codes.size(1) == pitch && codes.is_contiguous(),
              op, ": codes must be contiguous [", rows, ", ", pitch, "], not ",
              codes.sizes());
  TORCH_CHECK(exps.dim() == 2 && exps.size(0) == rows &&
                  exps.size(1) == pitch / kAct8Group && exps.is_contiguous(),
              op, ": exponents must be contiguous [", rows, ", ",
              pitch / kAct8Group, "], not ", exps.sizes());
}

void check_wgrad_size(int64_t n, int64_t k, const char* op) {
  constexpr int64_t most = kAct8MaxCols - kAct8Group;
  TORCH_CHECK(n <= most && k <= most, op, ": at most ", most, " columns");
}

void check_codes_aligned(const Tensor& codes, const char* op) {
  TORCH_CHECK(((uintptr_t)codes.data_ptr() & 15) == 0, op,
              ": codes must be aligned to 16 bytes");
}

Tensor act8_unpack_op(const Tensor& codes, const Tensor& exps,
                      const std::vector<int64_t>& shape,
                      at::ScalarType dtype) {
  const char* op = "act8_unpack";
  check_not_recorded(op);
  TORCH_CHECK(is_act_type(dtype), op,
              ": dtype must be float32, bfloat16 or float16, not ", dtype);
  TORCH_CHECK(!shape.empty(), op, ": the shape must have rows");
  for (const int64_t n : shape)
    TORCH_CHECK(n >= 0, op, ": a shape of ", at::IntArrayRef(shape));
  const auto lead = at::IntArrayRef(shape).slice(0, shape.size() - 1);
  int64_t rows = std::find(lead.begin(), lead.end(), 0) == lead.end();
  for (const int64_t n : lead) {
    TORCH_CHECK(rows == 0 || n <= kMaxRows / rows, op, ": at most 2^30 rows");
    rows *= n;
  }
  TORCH_CHECK(shape.back() <= kMaxRows, op, ": at most 2^30 columns");
  check_codes(codes, exps, rows, shape.back(), op);
  check_device(codes, codes, op, "codes");
  check_device(exps, codes, op, "exponents");
  check_codes_aligned(codes, op);
  const c10::OptionalDeviceGuard guard(codes.device());
  Tensor x = at::empty(shape, codes.options().dtype(dtype));
  Act8Move a = {};
  a.x = x.data_ptr();
  a.codes = codes.data_ptr<uint8_t>();
  a.exps = exps.data_ptr<uint8_t>();
  a.rows = rows;
  a.cols = a.xstride = shape.back();
  a.pitch = pitch_of(a.cols);
  a.type = elem(dtype);
  check_launch(act8_unpack(a, stream_of(x)), op);
  return x;
}

Tensor bias_rows(const Tensor& dy);

std::tuple<Tensor, Tensor> wgrad_rows(const Tensor& dy, const Tensor& codes,
                                      const Tensor& exps, int64_t k,
                                      bool bias) {
  const c10::OptionalDeviceGuard guard(dy.device());
  const Rows dr = as_rows(dy);
  Act8Wgrad a = {};
  a.m = rows_of(dy);
  a.n = dy.size(-1);
  a.k = k;
  a.pitch = pitch_of(k);
  Tensor dw = at::empty({a.n, a.k}, dy.options());
  Tensor db = bias ? at::empty({a.n}, dy.options()) : Tensor();
  if (a.m == 0) {
    dw.zero_();
    if (bias) db.zero_();
  } else if (bias && a.k == 0) {
    db = bias_rows(dy);
  }
  a.dy = dr.t.data_ptr();
  a.dstride = dr.stride;
  a.codes = codes.data_ptr<uint8_t>();
  a.exps = exps.data_ptr<uint8_t>();
  a.dw = dw.data_ptr();
  a.db = bias ? db.data_ptr() : nullptr;
  a.type = elem(dy.scalar_type());
  const Tensor ws = empty_bytes(act8_wgrad_workspace(a), dy);
  a.workspace = ws.data_ptr();
  check_launch(act8_wgrad(a, stream_of(dy)), "act8_wgrad");
  return {dw, db};
}

// The sum of dy's rows alone, beside a product with one column of zeros.
// (torch's sum clears memory in a way that a captured graph does not repeat
// reliably on this hardware.)
Tensor bias_rows(const Tensor& dy) {
  const auto bytes = dy.options().dtype(at::kByte);
  const int64_t rows = rows_of(dy);
  return std::get<1>(wgrad_rows(dy, at::zeros({rows, kAct8Group}, bytes),
                                at::zeros({rows, 1}, bytes), 1, true));
}

std::tuple<Tensor, OptTensor> act8_wgrad_op(const Tensor& dy,
                                            const Tensor& codes,
                                            const Tensor& exps,
                                            const std::vector<int64_t>& shape,
                                            at::ScalarType dtype, bool bias) {
  const char* op = "act8_wgrad";
  check_not_recorded(op);
  check_act8_input(dy, op, "dy");
  TORCH_CHECK(dy.scalar_type() == dtype, op, ": dy must have the kept input's "
              "type ", dtype, ", not ", dy.scalar_type());
  TORCH_CHECK((size_t)dy.dim() == shape.size(), op, ": dy ", dy.sizes(),
              " does not have the rows of the kept input ",
              at::IntArrayRef(shape));
  for (size_t d = 0; d + 1 < shape.size(); d++)
    TORCH_CHECK(dy.size(d) == shape[d], op, ": dy ", dy.sizes(),
                " does not have the rows of the kept input ",
                at::IntArrayRef(shape));
  check_wgrad_size(dy.size(-1), shape.back(), op);
  check_codes(codes, exps, rows_of(dy), shape.back(), op);
  check_device(dy, dy, op, "dy");
  check_device(codes, dy, op, "codes");
  check_device(exps, dy, op, "exponents");
  check_codes_aligned(codes, op);
  at::NoGradGuard no_grad;
  auto [dw, db] = wgrad_rows(dy.detach(), codes, exps, shape.back(), bias);
  return {dw, bias ? OptTensor(db) : OptTensor()};
}

// One product of matrices whatever x's layout: as batches of small ones with
// a transposed operand, which the library makes of some layouts, it has
// faulted on this hardware.
Tensor flat_linear(const Tensor& x, const Tensor& weight,
                   const OptTensor& bias) {
  auto sizes = x.sizes().vec();
  sizes.back() = weight.size(0);
  return at::_unsafe_view(
      at::linear(x.reshape({rows_of(x), x.size(-1)}), weight, bias), sizes);
}

// A linear layer whose input is kept in 8 bits.  Its two plain products, y
// and dx, are the library's, as in torch.nn.Linear; the weight gradient is
// taken from the codes.
struct LinearAct8Node : OpNode<3> {
  int64_t k;

  std::string name() const override { return "LinearAct8Backward"; }

  variable_list apply(variable_list&& grads) override {
    const c10::impl::ExcludeDispatchKeyGuard own_types(
        c10::autocast_dispatch_keyset);
    const auto saved = kept("linear_act8");
    variable_list out(3);
    if (!grads[0].defined()) return out;
    const Tensor dy = plain(grads[0]);
    const c10::OptionalDeviceGuard guard(dy.device());
    if (task_should_compute_output(0)) {
      auto sizes = dy.sizes().vec();
      sizes.back() = saved[0].size(1);
      out[0] = at::mm(dy.reshape({rows_of(dy), dy.size(-1)}), saved[0])
                   .view(sizes);
    }
    const bool bias = task_should_compute_output(2);
    if (task_should_compute_output(1))
      std::tie(out[1], out[2]) =
          wgrad_rows(dy, saved[1], saved[2], k, bias);
    else if (bias)
      out[2] = bias_rows(dy);
    return out;
  }
};

Tensor linear_act8(const Tensor& x, const Tensor& weight,
                   const OptTensor& bias) {
  const char* op = "linear_act8";
  check_not_recorded(op);
  check_act8_input(x, op, "x");
  check_act(weight, op, "weight");
  TORCH_CHECK(weight.scalar_type() == x.scalar_type(), op,
              ": weight must have x's type ", x.scalar_type(), ", not ",
              weight.scalar_type());
  TORCH_CHECK(weight.dim() == 2 && weight.size(1) == x.size(-1), op,
              ": weight must be [out, ", x.size(-1), "], not ",
              weight.sizes());
  check_wgrad_size(weight.size(0), weight.size(1), op);
  if (bias) {
    check_act(*bias, op, "bias");
    TORCH_CHECK(bias->scalar_type() == x.scalar_type(), op,
                ": bias must have x's type ", x.scalar_type(), ", not ",
                bias->scalar_type());
    TORCH_CHECK(bias->dim() == 1 && bias->size(0) == weight.size(0), op,
                ": bias must be [", weight.size(0), "], not ", bias->sizes());
  }
  check_device(x, x, op, "x");
  check_device(weight, x, op, "weight");
  if (bias) check_device(*bias, x, op, "bias");
  // the products are in the arguments' type, under autocast too: the codes
  // and the gradients go with it
  const c10::impl::ExcludeDispatchKeyGuard own_types(
      c10::autocast_dispatch_keyset);
  const c10::OptionalDeviceGuard guard(x.device());
  if (!wants_grad(op, {&x, &weight, get(bias)}))
    return flat_linear(x, weight, bias);
  const auto node = make_node<LinearAct8Node>(x, weight, bias);
  node->k = x.size(-1);
  const at::NoGradGuard no_grad;
  if (x.requires_grad()) node->keep(0, weight);
  if (weight.requires_grad()) {
    const auto [codes, exps] = pack_rows(x);
    node->keep(1, codes);
    node->keep(2, exps);
  }
  Tensor y = flat_linear(x, weight, bias);
  torch::autograd::set_history(y, node);
  return y;
}

// silu(a) * b, and the copies of a and b where they are defined.
Tensor run_silu(const Tensor& x, const Tensor& codes, const Tensor& exps) {
  const c10::OptionalDeviceGuard guard(x.device());
  const Rows xr = as_rows(x);
  SiluAct8 p = {};
  p.rows = rows_of(x);
  p.cols = x.size(-1) / 2;
  p.pitch = pitch_of(p.cols);
  p.x = xr.t.data_ptr();
  p.xstride = xr.stride;
  p.type = elem(x.scalar_type());
  c10::SmallVector<int64_t, 6> sizes(x.sizes().begin(), x.sizes().end());
  sizes.back() = p.cols;
  Tensor out = at::empty(sizes, x.options());
  p.out = out.data_ptr();
  if (codes.defined()) {
    p.codes = codes.data_ptr<uint8_t>();
    p.exps = exps.data_ptr<uint8_t>();
  }
  check_launch(silu_act8_forward(p, stream_of(x)), "silu_mul_act8");
  return out;
}

struct SiluAct8Node : OpNode<2> {
  std::string name() const override { return "SiluMulAct8Backward"; }

  variable_list apply(variable_list&& grads) override {
    const auto saved = kept("silu_mul_act8");
    if (!grads[0].defined()) return {Tensor()};
    const Rows dr = as_rows(grads[0]);
    const c10::OptionalDeviceGuard guard(dr.t.device());
    SiluAct8 p = {};
    p.rows = rows_of(dr.t);
    p.cols = dr.t.size(-1);
    p.pitch = pitch_of(p.cols);
    p.dout = dr.t.data_ptr();
    p.dstride = dr.stride;
    p.type = elem(dr.t.scalar_type());
    auto sizes = dr.t.sizes().vec();
    sizes.back() = 2 * p.cols;
    Tensor dx = at::empty(sizes, dr.t.options());
    p.dx = dx.data_ptr();
    p.codes = saved[0].data_ptr<uint8_t>();
    p.exps = saved[1].data_ptr<uint8_t>();
    check_launch(silu_act8_backward(p, stream_of(dx)),
                 "silu_mul_act8 backward");
    return {dx};
  }
};

Tensor silu_mul_act8(const Tensor& x) {
  const char* op = "silu_mul_act8";
  check_not_recorded(op);
  check_act8_input(x, op, "x");
  TORCH_CHECK(x.size(-1) % 2 == 0, op,
              ": x must hold two halves in its last dimension, not ",
              x.size(-1), " columns");
  check_device(x, x, op, "x");
  if (!wants_grad(op, {&x})) return run_silu(x, Tensor(), Tensor());
  const auto node = make_node<SiluAct8Node>(x);
  const at::NoGradGuard no_grad;
  const c10::OptionalDeviceGuard guard(x.device());
  const int64_t rows = rows_of(x), pitch = pitch_of(x.size(-1) / 2);
  const auto bytes = x.options().dtype(at::kByte);
  const Tensor codes = at::empty({rows, 2 * pitch}, bytes);
  const Tensor exps = at::empty({rows, 2 * pitch / kAct8Group}, bytes);
  Tensor out = run_silu(x, codes, exps);
  node->keep(0, codes);
  node->keep(1, exps);
  torch::autograd::set_history(out, node);
  return out;
}

}  // namespace

void bind_train_ops(pybind11::module& m) {
  namespace py = pybind11;
  m.def("embedding", &embedding, "scaled lookup of table rows",
        py::arg("weight"), py::arg("tokens"), py::arg("scale"),
        py::arg("padding_idx"), py::arg("out_dtype"));
  m.def("rms_norm", &rms_norm, "norm before a block", py::arg("x"),
        py::arg("weight"), py::arg("eps"));
  m.def("gated_residual_norm", &gated_residual_norm,
        "norm after a block, gate, residual scale and the next block's norm",
        py::arg("x"), py::arg("branch"), py::arg("gate"),
        py::arg("post_weight"), py::arg("pre_weight"),
        py::arg("residual_scale"), py::arg("branch_scale"), py::arg("eps"));
  m.def("act8_pack", &act8_pack_op, "8-bit copy of an activation");
  m.def("act8_unpack", &act8_unpack_op, "the values an 8-bit copy stands for");
  m.def("act8_wgrad", &act8_wgrad_op,
        "a linear layer's weight gradient from its input's 8-bit copy");
  m.def("linear_act8", &linear_act8, "linear layer, its input kept in 8 bits",
        py::arg("x"), py::arg("weight"), py::arg("bias"));
  m.def("silu_mul_act8", &silu_mul_act8,
        "silu(a) * b, its inputs kept in 8 bits");
}

}  // namespace baguanet
