// PyTorch-ROCm extension module `lm_ops`: the host work of the operators around
// a matrix-valued state -- linear attention for prompts, training and single
// tokens, the embedding and its gradient, gradient clipping -- over the C ABI of
// libssm_mamba_hip.so, with their autograd functions (a short prompt's or a small
// embedding's kernels take less time than a Python function of autograd).
#include "ext_common.h"

#include <ATen/MemoryOverlap.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <algorithm>
#include <array>
#include <vector>

namespace {

using namespace ssm_ext;

int dtype_code(const at::Tensor& x, const char* name) {
  TORCH_CHECK(x.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK(x.scalar_type() == at::kFloat || x.scalar_type() == at::kBFloat16, name,
              " must be float32 or bfloat16 tensor");
  return x.scalar_type() == at::kBFloat16 ? SSM_BF16 : SSM_F32;
}

// written through its address: what autograd saved of it is out of date
void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// A trace would hold the results' allocations and not the kernels that fill them.
void not_traced(const char* name) {
  TORCH_CHECK(!torch::jit::tracer::isTracing(), name, " cannot be traced by torch.jit.trace");
}

// as the step's kernel reads it: any strides, the last one 1
at::Tensor rows(const at::Tensor& x, at::ScalarType t) {
  at::Tensor y = x.scalar_type() == t ? x : x.to(t);
  return y.stride(-1) == 1 || y.size(-1) == 1 ? y : y.contiguous();
}

// (batch, tokens, heads, size) as the chunk kernels read it: in place where its rows
// are adjacent elements, 16-byte aligned and whole 16 bytes long; else a copy whose
// rows are
at::Tensor whole_rows(const at::Tensor& x, at::ScalarType t) {
  at::Tensor y = x.scalar_type() == t ? x : x.to(t);
  const int64_t dim = y.size(3), piece = 16 / y.element_size();
  bool ok = y.stride(3) == 1 && dim % piece == 0 && reinterpret_cast<uintptr_t>(y.data_ptr()) % 16 == 0 &&
            (y.size(1) == 1 || (y.stride(1) >= dim && y.stride(1) <= (1 << 22)));
  for (int d = 0; d < 3; ++d) ok = ok && (y.size(d) == 1 || y.stride(d) % piece == 0);
  if (ok || y.numel() == 0) return y;
  at::Tensor buf = at::empty({y.size(0), y.size(1), y.size(2), (dim + piece - 1) / piece * piece}, y.options());
  at::Tensor view = buf.narrow(3, 0, dim);
  view.copy_(y);
  return view;
}

// decays with heads adjacent; one per head expanded over tokens becomes a tensor of
// its own (strides of 0, 0 mean one per head to the kernels)
at::Tensor decays(const at::Tensor& g_) {
  at::Tensor g = g_.scalar_type() == at::kFloat ? g_ : g_.to(at::kFloat);
  const bool adjacent = g.stride(-1) == 1 || g.size(-1) == 1;
  return adjacent && !(g.dim() == 3 && g.stride(0) == 0 && g.stride(1) == 0) ? g : g.contiguous();
}

// what the chunk kernels and their backward are called with
struct LaArgs {
  at::Tensor q, k, v, g;
  OptT h_init, length;
  double scale;
  bool right;
  int io;
  int64_t batch, seqlen, heads, groups, key, value;

  void sizes() {
    batch = v.size(0), seqlen = v.size(1), heads = v.size(2), value = v.size(3);
    groups = q.size(2), key = q.size(3);
    io = v.scalar_type() == at::kBFloat16 ? SSM_BF16 : SSM_F32;
  }
  int64_t g_sb() const { return g.dim() == 1 ? 0 : g.stride(0); }
  int64_t g_st() const { return g.dim() == 1 ? 0 : g.stride(1); }
  at::Tensor state() const { return at::empty({batch, heads, key, value}, v.options().dtype(at::kFloat)); }
};

void check_state(const at::Tensor& t, const LaArgs& a, const char* name) {
  TORCH_CHECK(t.device() == a.v.device() && t.scalar_type() == at::kFloat && t.is_contiguous() &&
                  t.sizes() == at::IntArrayRef({a.batch, a.heads, a.key, a.value}),
              name, " must be a contiguous float32 (batch, heads, key, value) tensor on v's device");
}

void check_qkv(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& g) {
  const int64_t lead = v.dim() - 2;
  (void)dtype_code(q, "q");
  (void)dtype_code(k, "k");
  (void)dtype_code(v, "v");
  TORCH_CHECK(q.sizes() == k.sizes(), "q and k must have the same shape");
  TORCH_CHECK(q.sizes().slice(0, lead) == v.sizes().slice(0, lead),
              "q, k and v must have the same leading sizes");
  const int64_t heads = v.size(lead), groups = q.size(lead);
  TORCH_CHECK(heads >= 1 && groups >= 1 && heads % groups == 0,
              "the number of value heads must be a multiple of the number of query and key heads");
  TORCH_CHECK(q.size(-1) >= 1 && v.size(-1) >= 1, "key and value sizes must be >= 1");
  TORCH_CHECK(g.sizes() == at::IntArrayRef({heads}) || g.sizes() == v.sizes().slice(0, lead + 1),
              "g must have shape (heads,) or v's shape without its last size");
  for (const at::Tensor* t : {&q, &k, &g})
    TORCH_CHECK(t->device() == v.device(), "all tensors must be on one device");
}

// {out, last state or undefined, the segments' starts or undefined}
std::array<at::Tensor, 3> la_forward(const LaArgs& a, bool want_last) {
  at::Tensor out = at::empty(a.v.sizes(), a.v.options()), last, states, ws;
  if (want_last) last = a.state();
  if (a.batch == 0 || a.seqlen == 0) {  // nothing to read: the state stays what it was
    if (want_last) {
      if (a.h_init) last.copy_(*a.h_init);
      else last.zero_();
    }
    return {out, last, states};
  }
  const int64_t segs = ssm_linear_attention_segments(a.batch, a.seqlen, a.heads, a.groups, a.key, a.value, a.io);
  size_t bytes = 0;
  if (segs > 1) {
    states = at::empty({segs, a.batch, a.heads, a.key, a.value}, a.v.options().dtype(at::kFloat));
    bytes = ssm_linear_attention_fwd_workspace_bytes(a.batch, a.seqlen, a.heads, a.groups, a.key, a.value, a.io);
    ws = at::empty({(int64_t)bytes}, a.v.options().dtype(at::kByte));
  }
  int64_t s[9];
  const at::Tensor* t[3] = {&a.q, &a.k, &a.v};
  for (int i = 0; i < 9; ++i) s[i] = t[i / 3]->stride(i % 3);
  ok(ssm_linear_attention_fwd(a.batch, a.seqlen, a.heads, a.groups, a.key, a.value, a.io, a.q.data_ptr(),
                              a.k.data_ptr(), a.v.data_ptr(), s, a.g.data_ptr<float>(), a.g_sb(), a.g_st(),
                              (float)a.scale, ptr<float>(opt(a.h_init)), ptr<int64_t>(opt(a.length)),
                              a.right ? 1 : 0, out.data_ptr(), last.defined() ? last.data_ptr<float>() : nullptr,
                              states.defined() ? states.data_ptr<float>() : nullptr,
                              ws.defined() ? ws.data_ptr() : nullptr, bytes, stream_of(a.v)));
  return {out, last, states};
}

// gradients of q, k, v, g and the first state, those that `need` asks for
std::array<at::Tensor, 5> la_backward(const LaArgs& a, const at::Tensor& states, const at::Tensor& last,
                                      const at::Tensor& dout, const at::Tensor& dlast,
                                      const std::array<bool, 5>& need) {
  // the decays' gradient is summed up from dq's and dk's, the first state's is dk's last
  const bool dg_ = need[3], dh_ = need[4];
  at::Tensor dq, dk, dv, dg, dh;
  if (need[0] || dg_) dq = at::empty(a.q.sizes(), a.q.options());
  if (need[1] || dg_ || dh_) dk = at::empty(a.k.sizes(), a.k.options());
  if (need[2]) dv = at::empty(a.v.sizes(), a.v.options());
  if (dg_) dg = at::empty(a.g.sizes(), a.g.options());
  if (dh_) dh = a.state();
  const auto p = [](const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; };
  const auto f = [](const at::Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; };
  if (a.batch == 0 || a.seqlen == 0) {
    if (dg_) dg.zero_();
    if (dh_) {
      if (dlast.defined()) dh.copy_(dlast);
      else dh.zero_();
    }
  } else {
    const size_t bytes = ssm_linear_attention_bwd_workspace_bytes(a.batch, a.seqlen, a.heads, a.groups, a.key, a.value, a.io);
    at::Tensor ws = at::empty({(int64_t)bytes}, a.v.options().dtype(at::kByte));
    int64_t s[12];
    const at::Tensor* t[4] = {&a.q, &a.k, &a.v, &dout};
    for (int i = 0; i < 12; ++i) s[i] = t[i / 3]->stride(i % 3);
    ok(ssm_linear_attention_bwd(a.batch, a.seqlen, a.heads, a.groups, a.key, a.value, a.io, a.q.data_ptr(),
                                a.k.data_ptr(), a.v.data_ptr(), dout.data_ptr(), s, a.g.data_ptr<float>(),
                                a.g_sb(), a.g_st(), (float)a.scale, ptr<float>(opt(a.h_init)),
                                ptr<int64_t>(opt(a.length)), a.right ? 1 : 0, f(states), f(last), f(dlast),
                                p(dq), p(dk), p(dv), f(dg), f(dh), ws.data_ptr(), bytes, stream_of(a.v)));
  }
  return {need[0] ? dq : at::Tensor(), need[1] ? dk : at::Tensor(), dv, dg, dh};
}

LaArgs la_args(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& g,
               const OptT& h_init, const OptT& length, double scale, bool right) {
  LaArgs a;
  a.q = whole_rows(q, v.scalar_type());
  a.k = whole_rows(k, v.scalar_type());
  a.v = whole_rows(v, v.scalar_type());
  a.g = decays(g);
  a.h_init = h_init;
  a.length = length;
  a.scale = scale;
  a.right = right;
  a.sizes();
  return a;
}

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// whether a call is to be differentiated: backwards, or forwards, which is in force
// under no_grad too and which the autograd functions refuse
bool differentiated(std::initializer_list<const at::Tensor*> inputs) {
  const bool grad = at::GradMode::is_enabled();
  for (const at::Tensor* t : inputs)
    if ((grad && t->requires_grad()) || t->_fw_grad(0).defined()) return true;
  return false;
}

// The gradients that a backward made with create_graph, `by` those of its results:
// functions of them and of the node's inputs that raise if differentiated again.
void once(const char* name, variable_list& grads, const variable_list& by) {
  using namespace torch::autograd;
  edge_list from = get_current_node()->next_edges();
  for (const at::Tensor& t : by)
    if (t.defined() && t.requires_grad()) from.push_back(impl::gradient_edge(t));
  const auto error = std::make_shared<Error>(
      std::string(name) + " is differentiable once: its gradients cannot be differentiated", std::move(from));
  for (at::Tensor& t : grads)
    if (t.defined()) impl::set_gradient_edge(t = t.detach(), {error, error->add_input_metadata(t)});
}

struct LinearAttentionFn : torch::autograd::Function<LinearAttentionFn> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k,
                               const at::Tensor& v, const at::Tensor& g, const OptT& h_init,
                               const OptT& length, double scale, bool right, bool want_last) {
    const LaArgs a = la_args(q, k, v, g, h_init, length, scale, right);
    auto [out, last, states] = la_forward(a, want_last);
    ctx->set_materialize_grads(false);  // an unused last state's gradient stays undefined
    ctx->save_for_backward({a.q, a.k, a.v, a.g, h_init.value_or(at::Tensor()), length.value_or(at::Tensor()),
                            states, last});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["right"] = right;
    if (!want_last) return {out};
    return {out, last};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    LaArgs a;
    a.q = saved[0], a.k = saved[1], a.v = saved[2], a.g = saved[3];
    if (saved[4].defined()) a.h_init = saved[4];
    if (saved[5].defined()) a.length = saved[5];
    a.scale = ctx->saved_data["scale"].toDouble();
    a.right = ctx->saved_data["right"].toBool();
    a.sizes();
    c10::hip::HIPGuard guard(a.v.get_device());
    at::Tensor dout = grads[0].defined() ? whole_rows(grads[0], a.v.scalar_type())
                                         : whole_rows(at::zeros(a.v.sizes(), a.v.options()), a.v.scalar_type());
    at::Tensor dlast;
    if (grads.size() > 1 && grads[1].defined()) dlast = grads[1].to(at::kFloat).contiguous();
    std::array<bool, 5> need;
    for (int i = 0; i < 5; ++i) need[i] = (i < 4 || a.h_init) && ctx->needs_input_grad(i);
    auto [dq, dk, dv, dg, dh] = la_backward(a, saved[6], saved[7], dout, dlast, need);
    variable_list res{dq, dk, dv, dg, dh};
    if (at::GradMode::is_enabled()) once("linear_attention_fn", res, grads);
    res.resize(9);
    return res;
  }
};

variable_list linear_attention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                               const at::Tensor& g, double scale, const OptT& h_init_, const OptT& length_,
                               const std::string& padding_side, bool want_last) {
  not_traced("linear_attention_fn");
  check_dim(q, 4, "q");
  check_dim(k, 4, "k");
  check_dim(v, 4, "v");
  check_qkv(q, k, v, g);
  TORCH_CHECK(padding_side == "left" || padding_side == "right", "padding_side must be 'left' or 'right'");
  c10::hip::HIPGuard guard(v.get_device());
  OptT h_init, length;
  LaArgs a;
  a.q = q, a.v = v;
  a.sizes();
  if (const at::Tensor* t = opt(h_init_)) {
    h_init = t->to(at::kFloat).contiguous();
    check_state(*h_init, a, "h_init");
  }
  if (const at::Tensor* t = opt(length_)) {
    TORCH_CHECK(t->scalar_type() == at::kLong && t->sizes() == at::IntArrayRef({a.batch}) &&
                    t->device() == v.device(),
                "length must be an int64 (batch,) tensor on v's device");
    length = t->contiguous();
  }
  const bool right = padding_side == "right";
  if (differentiated({&q, &k, &v, &g}) || (h_init && differentiated({&*h_init})))
    return LinearAttentionFn::apply(q, k, v, g, h_init, length, scale, right, want_last);
  auto [out, last, states] = la_forward(la_args(q, k, v, g, h_init, length, scale, right), want_last);
  return {out, last};
}

at::Tensor linear_attention_step(const at::Tensor& state, const at::Tensor& q_, const at::Tensor& k_,
                                 const at::Tensor& v_, const at::Tensor& g_, double scale) {
  not_traced("linear_attention_step");
  check_dim(q_, 3, "q");
  check_dim(k_, 3, "k");
  check_dim(v_, 3, "v");
  check_qkv(q_, k_, v_, g_);
  const int io = dtype_code(v_, "v");
  const auto type = v_.scalar_type();
  const int64_t batch = v_.size(0), heads = v_.size(1), value = v_.size(2);
  const int64_t groups = q_.size(1), key = q_.size(2);
  TORCH_CHECK(state.device() == v_.device(), "all tensors must be on one device");
  TORCH_CHECK(state.scalar_type() == at::kFloat && state.is_contiguous() &&
                  state.sizes() == at::IntArrayRef({batch, heads, key, value}),
              "state must be a contiguous float32 (batch, heads, key, value) tensor on v's device "
              "(it is updated in place)");
  TORCH_CHECK(!(state.requires_grad() && at::GradMode::is_enabled()),
              "state is updated in place and must not require a gradient");
  c10::hip::HIPGuard guard(v_.get_device());
  const at::Tensor q = rows(q_, type), k = rows(k_, type), v = rows(v_, type), g = rows(g_, at::kFloat);
  at::Tensor out = at::empty({batch, heads, value}, v.options());
  if (batch == 0) return out;
  const int64_t strides[6] = {q.stride(0), q.stride(1), k.stride(0),
                              k.stride(1), v.stride(0), v.stride(1)};
  ok(ssm_linear_attention_step(batch, heads, groups, key, value, io, state.data_ptr<float>(),
                               q.data_ptr(), k.data_ptr(), v.data_ptr(), strides, g.data_ptr<float>(),
                               g.dim() == 1 ? 0 : g.stride(0), (float)scale, out.data_ptr(),
                               stream_of(v)));
  written(state);
  return out;
}

void check_ids(const at::Tensor& ids, const at::Tensor& w) {
  TORCH_CHECK(ids.scalar_type() == at::kLong || ids.scalar_type() == at::kInt,
              "ids must be an int64 or int32 tensor");
  TORCH_CHECK(ids.device() == w.device(), "all tensors must be on one device");
}

// a tensor as the kernels read it, without the dispatcher where it is so already
at::Tensor plain(const at::Tensor& t, at::ScalarType type) {
  at::Tensor x = t.scalar_type() == type ? t : t.to(type);
  return x.is_contiguous() ? x : x.contiguous();
}

at::Tensor embedding(const at::Tensor& ids_, const at::Tensor& weight, double scale) {
  check_dim(weight, 2, "weight");
  const int io = dtype_code(weight, "weight");
  check_ids(ids_, weight);
  c10::hip::HIPGuard guard(weight.get_device());
  const at::Tensor ids = plain(ids_, at::kLong), w = plain(weight, weight.scalar_type());
  c10::SmallVector<int64_t, 6> shape(ids.sizes().begin(), ids.sizes().end());
  shape.push_back(w.size(1));
  at::Tensor out = at::empty(shape, w.options());
  if (out.numel() == 0) return out;
  ok(ssm_embedding_fwd(ids.numel(), w.size(0), w.size(1), io, ids.data_ptr<int64_t>(), w.data_ptr(),
                       (float)scale, out.data_ptr(), stream_of(w)));
  return out;
}

// the gradient of a (vocab, dout.size(-1)) weight, in dout's type
at::Tensor embedding_backward(const at::Tensor& ids_, const at::Tensor& dout_, int64_t vocab, double scale,
                              int64_t padding_idx) {
  const int io = dtype_code(dout_, "dout");
  check_ids(ids_, dout_);
  c10::hip::HIPGuard guard(dout_.get_device());
  const int64_t dim = dout_.size(-1);
  const at::Tensor ids = plain(ids_, at::kLong), dout = plain(dout_, dout_.scalar_type());
  TORCH_CHECK(dout.numel() == ids.numel() * dim, "dout must be like the output");
  if (ids.numel() == 0 || dim == 0) return at::zeros({vocab, dim}, dout.options());
  at::Tensor dw = at::empty({vocab, dim}, dout.options());
  if (vocab == 0) return dw;
  const size_t bytes = ssm_embedding_bwd_workspace_bytes(ids.numel(), vocab, dim);
  at::Tensor ws = at::empty({(int64_t)bytes}, dout.options().dtype(at::kByte));
  ok(ssm_embedding_bwd(ids.numel(), vocab, dim, io, ids.data_ptr<int64_t>(), dout.data_ptr(),
                       (float)scale, padding_idx, dw.data_ptr(), ws.data_ptr(), bytes,
                       stream_of(dout)));
  return dw;
}

at::Tensor embedding_fn(const at::Tensor& ids, const at::Tensor& weight, double scale,
                        std::optional<int64_t> padding_idx);

// The weight's gradient as a function of the output's, where that is to be
// differentiated again: it is linear, with the lookup for its derivative.
struct EmbeddingGradFn : torch::autograd::Function<EmbeddingGradFn> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& ids, const at::Tensor& dout,
                            int64_t vocab, double scale, int64_t padding_idx) {
    ctx->save_for_backward({ids});
    ctx->saved_data["sizes"] = std::vector<int64_t>{vocab, padding_idx};
    ctx->saved_data["scale"] = scale;
    return embedding_backward(ids, dout, vocab, scale, padding_idx);
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list res(5);
    if (!grads[0].defined()) return res;
    const at::Tensor ids = ctx->get_saved_variables()[0];
    const auto sizes = ctx->saved_data["sizes"].toIntVector();
    const at::Tensor none = ids.lt(0).logical_or(ids.ge(sizes[0])).logical_or(ids.eq(sizes[1]));
    const auto pad = sizes[1] < 0 ? std::nullopt : std::optional<int64_t>(sizes[1]);
    res[1] = embedding_fn(ids, grads[0], ctx->saved_data["scale"].toDouble(), pad)
                 .masked_fill(none.unsqueeze(-1), 0);
    return res;
  }
};

struct EmbeddingFn : torch::autograd::Function<EmbeddingFn> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& ids, const at::Tensor& weight,
                            double scale, int64_t padding_idx) {
    at::Tensor out = embedding(ids, weight, scale);
    ctx->save_for_backward({ids});
    ctx->saved_data["sizes"] = std::vector<int64_t>{weight.size(0), (int64_t)weight.scalar_type(), padding_idx};
    ctx->saved_data["scale"] = scale;
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined()) return {at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
    const auto sizes = ctx->saved_data["sizes"].toIntVector();
    const at::Tensor ids = ctx->get_saved_variables()[0];
    const at::Tensor dout = plain(grads[0], (at::ScalarType)sizes[1]);
    const double scale = ctx->saved_data["scale"].toDouble();
    at::Tensor dw = differentiated({&dout}) ? EmbeddingGradFn::apply(ids, dout, sizes[0], scale, sizes[2])
                                            : embedding_backward(ids, dout, sizes[0], scale, sizes[2]);
    return {at::Tensor(), dw, at::Tensor(), at::Tensor()};
  }
};

at::Tensor embedding_fn(const at::Tensor& ids, const at::Tensor& weight, double scale,
                        std::optional<int64_t> padding_idx) {
  not_traced("embedding_fn");
  check_dim(weight, 2, "weight");
  (void)dtype_code(weight, "weight");
  check_ids(ids, weight);
  const int64_t vocab = weight.size(0);
  int64_t pad = -1;
  if (padding_idx) {
    TORCH_CHECK(*padding_idx >= -vocab && *padding_idx < vocab, "padding_idx must be within the vocabulary");
    pad = *padding_idx < 0 ? *padding_idx + vocab : *padding_idx;
  }
  return differentiated({&weight}) ? EmbeddingFn::apply(ids, weight, scale, pad)
                                   : embedding(ids, weight, scale);
}

struct Range {
  const char *lo, *hi;
  size_t owner;
  bool written;
};

Range range_of(const at::Tensor& t, size_t owner, bool written) {
  const char* p = static_cast<const char*>(t.data_ptr());
  return {p, p + t.numel() * t.element_size(), owner, written};
}

// The norm of all gradients; gradient i times its coefficient into outs[i], or
// in place where there are no outs.
at::Tensor clip_grad_norm(const std::vector<at::Tensor>& grads, const std::vector<at::Tensor>& outs,
                          double max_norm) {
  not_traced("clip_grad_norm_");
  TORCH_CHECK(max_norm >= 0, "max_norm must be >= 0");
  TORCH_CHECK(!grads.empty(), "no gradients");
  const bool inplace = outs.empty();
  TORCH_CHECK(inplace || outs.size() == grads.size(), "out must have one tensor for each parameter");
  const size_t n = grads.size();
  const at::Device dev = grads[0].device();
  std::vector<at::Tensor> src(n), dst(n);
  std::vector<const void*> gp(n);
  std::vector<void*> op(n);
  std::vector<int64_t> sizes(n);
  std::vector<int> gt(n), ot(n);
  std::vector<Range> ranges;
  ranges.reserve(2 * n);
  std::vector<const void*> copied;  // tensors that are written through a copy
  for (size_t i = 0; i < n; ++i) {
    const at::Tensor& g = grads[i];
    TORCH_CHECK(g.layout() == at::kStrided, "gradients must be dense tensors");
    gt[i] = dtype_code(g, "every gradient");
    TORCH_CHECK(g.device() == dev, "all tensors must be on one device");
    const at::Tensor& o = inplace ? g : outs[i];
    if (!inplace) {
      TORCH_CHECK(o.layout() == at::kStrided && o.sizes() == g.sizes(),
                  "every out must have its gradient's shape");
      TORCH_CHECK(o.device() == dev, "all tensors must be on one device");
    }
    ot[i] = inplace ? gt[i] : dtype_code(o, "every out");
    // dense in any order of dimensions is one stretch of memory; other layouts
    // go through a copy
    const bool dense = g.is_non_overlapping_and_dense() && (inplace || o.strides() == g.strides());
    src[i] = dense ? g : g.contiguous();
    dst[i] = dense ? o : inplace ? src[i] : at::empty(g.sizes(), o.options());
    gp[i] = src[i].data_ptr();
    op[i] = dst[i].data_ptr();
    sizes[i] = g.numel();
    if (sizes[i] == 0) continue;
    TORCH_CHECK(dense || at::has_internal_overlap(o) != at::MemOverlap::Yes,
                "a gradient that is scaled in place, or an out, has elements that share memory");
    if (!dense) copied.push_back(o.data_ptr());
    ranges.push_back(range_of(dst[i], i, true));
    if (!inplace && gp[i] != op[i]) ranges.push_back(range_of(src[i], i, false));
  }
  std::sort(ranges.begin(), ranges.end(), [](const Range& a, const Range& b) { return a.lo < b.lo; });
  std::sort(copied.begin(), copied.end());
  TORCH_CHECK(std::adjacent_find(copied.begin(), copied.end()) == copied.end(),
              "gradients (or outs) overlap: a tensor that is written must be listed once");
  const char* end = nullptr;       // of all ranges so far
  const char* written_end = nullptr;
  for (const Range& r : ranges) {
    TORCH_CHECK(!(written_end && r.lo < written_end) && !(r.written && end && r.lo < end),
                "gradients (or outs) overlap: a tensor that is written must be listed once");
    end = std::max(end, r.hi);
    if (r.written) written_end = std::max(written_end, r.hi);
  }
  c10::hip::HIPGuard guard(dev.index());
  const auto f32 = grads[0].options().dtype(at::kFloat);
  at::Tensor norm = at::empty({}, f32);
  const size_t bytes = ssm_grad_clip_workspace_bytes((int64_t)n, sizes.data());
  at::Tensor ws = at::empty({(int64_t)bytes}, f32.dtype(at::kByte));
  ok(ssm_grad_clip((int64_t)n, gp.data(), op.data(), sizes.data(), gt.data(), ot.data(), (float)max_norm,
                   norm.data_ptr<float>(), ws.data_ptr(), bytes, stream_of(norm)));
  for (size_t i = 0; i < n; ++i) {
    const at::Tensor& o = inplace ? grads[i] : outs[i];
    if (!dst[i].is_same(o)) o.copy_(dst[i]);
    else written(o);
  }
  return norm;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  namespace py = pybind11;
  m.doc() = "MI355X operators around a matrix-valued state (HIP, gfx950)";
  m.def("linear_attention_step", &linear_attention_step, py::arg("state"), py::arg("q"), py::arg("k"),
        py::arg("v"), py::arg("g"), py::arg("scale"));
  m.def("linear_attention", &linear_attention, py::arg("q"), py::arg("k"), py::arg("v"), py::arg("g"),
        py::arg("scale"), py::arg("h_init"), py::arg("length"), py::arg("padding_side"), py::arg("want_last"));
  m.def("embedding_fn", &embedding_fn, py::arg("ids"), py::arg("weight"), py::arg("scale"),
        py::arg("padding_idx"));
  m.def("embedding", &embedding, py::arg("ids"), py::arg("weight"), py::arg("scale"));
  m.def("embedding_backward", &embedding_backward, py::arg("ids"), py::arg("dout"), py::arg("vocab"),
        py::arg("scale"), py::arg("padding_idx"));
  m.def("clip_grad_norm", &clip_grad_norm, py::arg("grads"), py::arg("outs"), py::arg("max_norm"));
}
