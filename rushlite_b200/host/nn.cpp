// Operators of a transformer's training step: layer norm, causal attention
// over packed sequences, AdamW.  Each is one call of the C ABI; none is
// recorded lazily, so pending inputs are realized first.
#include <algorithm>
#include <cmath>
#include <mutex>
#include <unordered_set>

#include "lamp.hpp"

namespace lmp {
namespace tensor {

namespace {

// Handles whose owner went away while a graph was capturing on its thread,
// where device memory cannot be freed.
std::mutex g_released_mu;
std::vector<lmpb_sequences>& released() {
  static auto* v = new std::vector<lmpb_sequences>();
  return *v;
}

void release_pending() {
  std::vector<lmpb_sequences> take;
  {
    std::lock_guard<std::mutex> lk(g_released_mu);
    take.swap(released());
  }
  for (lmpb_sequences h : take) lmpb_sequences_release(h);
}

}  // namespace

Sequences::Sequences(const std::vector<int64_t>& lens) : lengths(lens) {
  LMP_CHECK(!capturing_graph(), "Sequences: create them before the capture, which cannot record their table's upload");
  LMP_CHECK(lens.size() <= (size_t)INT32_MAX, "Sequences: too many");
  release_pending();
  LMPB_OK_OR_THROW(lmpb_sequences_create(lens.data(), (int)lens.size(), &handle));
  for (int64_t n : lens) tokens += n;
}

Sequences::~Sequences() {
  if (capturing_graph()) {
    std::lock_guard<std::mutex> lk(g_released_mu);
    released().push_back(handle);
    return;
  }
  lmpb_sequences_release(handle);
  release_pending();
}

}  // namespace tensor

namespace autograd {

using tensor::ImplPtr;
using tensor::LazyNode;
using tensor::TensorImpl;

namespace {

// `extra`: bytes behind the values, for what belongs to them.
Tensor empty(const std::vector<size_t>& shape, DataType dt, size_t extra = 0) {
  auto p = std::make_shared<TensorImpl>();
  p->shape = shape;
  p->dtype = dt;
  p->device = DeviceType::CUDA;
  p->storage = tensor::make_storage(p->nbytes() + extra, p->device);
  return Tensor(p);
}

void* ptr(const Tensor& t) { return t.impl()->data(); }

bool on_cuda(const Variable& v) { return v.data().device() == DeviceType::CUDA; }

bool floating(DataType d) { return d == DataType::Float32 || d == DataType::Float64; }

// Where a kernel writes a gradient: straight into the gradient's own buffer
// while that is the untouched zero (as gemm_accumulate does), else into a new
// tensor that add() accumulates.  Without add(), as when the call fails, the
// gradient is the zero that it was.
class GradOut {
 public:
  explicit GradOut(Variable* v) : v_(v && v->requires_grad() ? v : nullptr) {
    if (!v_) return;
    const ImplPtr& gi = v_->grad_slot().impl();
    if (!v_->impl()->grad_shared && gi->device == DeviceType::CUDA && gi->dtype == v_->data().type() &&
        gi->lazy && gi->lazy->kind == LazyNode::kConst && gi->lazy->p0 == 0.0) {
      if (!gi->storage || gi->storage->bytes < gi->nbytes()) gi->storage = tensor::make_storage(gi->nbytes(), gi->device);
      zero_.swap(gi->lazy);  // taken: another place of the same Variable gets a tensor of its own
      t_ = Tensor(gi);
    } else {
      t_ = empty(v_->data().shape(), v_->data().type());
    }
  }
  GradOut(const GradOut&) = delete;
  GradOut& operator=(const GradOut&) = delete;
  ~GradOut() {
    if (zero_) t_.impl()->lazy = zero_;
  }
  bool wanted() const { return v_ != nullptr; }
  void* get() const { return v_ ? ptr(t_) : nullptr; }
  // After the kernel that writes get() is queued.
  void add() {
    if (!v_) return;
    if (!zero_) return v_->incr_grad(t_);
    zero_ = nullptr;
    if (v_->impl()->grad_hook) v_->impl()->grad_hook();
  }

 private:
  Variable* v_;
  std::shared_ptr<LazyNode> zero_;  // what the gradient was, while its buffer is being written
  Tensor t_;
};

bool records(const variable_list& in) {
  if (!is_grad_enabled()) return false;
  return std::any_of(in.begin(), in.end(), [](const Variable& v) { return v.requires_grad(); });
}

Variable output(const Tensor& t, bool rg, std::shared_ptr<Function> fn, variable_list in) {
  Variable out(t, rg);
  if (rg) {
    fn->saved_inputs = std::make_shared<variable_list>(std::move(in));
    out.set_grad_fn(std::move(fn));
  }
  return out;
}

struct LayerNormBackward : Function {
  tensor::Storage buffer;  // of the next two
  void *mean = nullptr, *rstd = nullptr;
  bool has_weight = false, has_bias = false;
  void apply(const Variable& out) override {
    variable_list& in = *saved_inputs;
    const Tensor& x = in[0].data();
    const Tensor& g = out.grad();
    const void* pg = ptr(g);
    const void* px = ptr(x);
    const void* pw = has_weight ? ptr(in[1].data()) : nullptr;
    GradOut dx(&in[0]), dw(has_weight ? &in[1] : nullptr), db(has_bias ? &in.back() : nullptr);
    const int64_t f = (int64_t)x.shape().back();
    LMPB_OK_OR_THROW(lmpb_layer_norm_backward((int)x.type(), px, pw, mean, rstd, pg,
                                              (int64_t)x.numel() / f, f, dx.get(), dw.get(), db.get(), tensor::current_stream()));
    dx.add(), dw.add(), db.add();
  }
};

struct AttentionBackward : Function {
  tensor::Storage buffer;  // out's, with lse behind it
  float* lse = nullptr;
  std::shared_ptr<tensor::Sequences> seqs;
  float scale = 1.f;
  void apply(const Variable& out) override {
    variable_list& in = *saved_inputs;
    const Tensor &q = in[0].data(), &k = in[1].data(), &v = in[2].data();
    const float* pg = static_cast<const float*>(ptr(out.grad()));
    const float *pq = (const float*)ptr(q), *pk = (const float*)ptr(k), *pv = (const float*)ptr(v);
    GradOut dq(&in[0]), dk(&in[1]), dv(&in[2]);
    // the kernel computes dk and dv together: one that nobody asked for goes to a scratch tensor
    Tensor scratch;
    float *pdk = (float*)dk.get(), *pdv = (float*)dv.get();
    if (dk.wanted() != dv.wanted()) {
      scratch = empty(k.shape(), k.type());
      (pdk ? pdv : pdk) = (float*)ptr(scratch);
    }
    const std::vector<size_t>& s = q.shape();
    if (tensor::Graph* g = tensor::capturing_graph()) g->keep(seqs);
    LMPB_OK_OR_THROW(lmpb_attention_backward(pq, pk, pv, (const float*)ptr(out.data()), lse, pg,
                                             (float*)dq.get(), pdk, pdv, (int64_t)s[0], (int)s[1], (int)k.shape()[1],
                                             (int)s[2], scale, seqs->handle, tensor::current_stream()));
    dq.add(), dk.add(), dv.add();
  }
};

}  // namespace

namespace ops {

Variable layer_norm(const Variable& x, const Variable* weight, const Variable* bias, Scalar eps) {
  const std::vector<size_t>& s = x.data().shape();
  LMP_CHECK(on_cuda(x), "layer_norm: this backend computes on CUDA tensors; move the tensor with .to(device.cuda)");
  LMP_CHECK(floating(x.data().type()), "layer_norm: float32 or float64 only");
  LMP_CHECK(!s.empty() && s.back() >= 1, "layer_norm: needs a last dimension of at least 1");
  LMP_CHECK(std::isfinite(eps) && eps >= 0, "layer_norm: eps must be finite and not negative");
  variable_list in{x};
  for (const Variable* p : {weight, bias}) {
    if (!p) continue;
    const char* name = p == weight ? "weight" : "bias";
    LMP_CHECK(on_cuda(*p) && p->data().type() == x.data().type(), "layer_norm: " << name << " must have x's device and dtype");
    LMP_CHECK(p->data().shape() == std::vector<size_t>{s.back()}, "layer_norm: " << name << " must have shape [" << s.back() << "]");
    in.push_back(*p);
  }
  const bool rg = records(in);
  const DataType dt = x.data().type();
  const void* px = ptr(x.data());
  const void* pw = weight ? ptr(weight->data()) : nullptr;
  const void* pb = bias ? ptr(bias->data()) : nullptr;
  size_t values = 1;
  for (size_t n : s) values *= n;
  const size_t rows = values / s.back(), size = dtype_size(dt), stats = rg ? 2 * rows * size : 0;
  // The statistics go behind a small y, which then lives as long as they do, and save an allocation (1.5 of 17 us
  // forward and backward); a large y does not have to.
  const bool behind = values * size <= size_t(1) << 20;
  Tensor y = empty(s, dt, behind ? stats : 0);
  auto fn = std::make_shared<LayerNormBackward>();
  if (rg) {
    fn->buffer = behind ? y.impl()->storage : tensor::make_storage(stats, DeviceType::CUDA);
    fn->mean = static_cast<char*>(fn->buffer->ptr) + (behind ? values * size : 0);
    fn->rstd = static_cast<char*>(fn->mean) + rows * size;
    fn->has_weight = weight != nullptr;
    fn->has_bias = bias != nullptr;
  }
  LMPB_OK_OR_THROW(lmpb_layer_norm((int)dt, px, pw, pb, (int64_t)rows, (int64_t)s.back(), eps, ptr(y), fn->mean, fn->rstd,
                                   tensor::current_stream()));
  return output(y, rg, fn, std::move(in));
}

Variable causal_attention(const Variable& q, const Variable& k, const Variable& v,
                          const std::shared_ptr<tensor::Sequences>& seqs, const Scalar* scale) {
  for (const Variable* x : {&q, &k, &v}) {
    LMP_CHECK(on_cuda(*x), "causal_attention: this backend computes on CUDA tensors; move the tensor with .to(device.cuda)");
    LMP_CHECK(x->data().type() == DataType::Float32, "causal_attention: float32 only");
    LMP_CHECK(x->data().shape().size() == 3, "causal_attention: q, k and v are [tokens, heads, head_dim]");
  }
  LMP_CHECK(seqs, "causal_attention: no sequences");
  const std::vector<size_t>&s = q.data().shape(), &t = k.data().shape();
  LMP_CHECK(t == v.data().shape(), "causal_attention: k and v must have the same shape");
  LMP_CHECK(s[0] == t[0] && s[2] == t[2], "causal_attention: q and k differ in tokens or head_dim");
  LMP_CHECK(s[1] >= 1 && t[1] >= 1 && s[1] % t[1] == 0,
            "causal_attention: " << s[1] << " heads are not a multiple of " << t[1] << " key/value heads");
  LMP_CHECK(s[1] <= 65535, "causal_attention: at most 65535 heads");
  LMP_CHECK(s[2] >= 1 && s[2] <= 128, "causal_attention: head_dim must lie in [1, 128], got " << s[2]);
  LMP_CHECK((size_t)seqs->tokens <= s[0], "causal_attention: the sequences have " << seqs->tokens << " tokens, q has " << s[0]);
  const float sc = scale ? (float)*scale : (float)(1.0 / std::sqrt((double)s[2]));
  LMP_CHECK(sc > 0 && sc <= 0x1p64f, "causal_attention: scale must be positive and at most 2^64");
  variable_list in{q, k, v};
  const bool rg = records(in);
  const float *pq = (const float*)ptr(q.data()), *pk = (const float*)ptr(k.data()), *pv = (const float*)ptr(v.data());
  Tensor out = empty(s, DataType::Float32, s[0] * s[1] * sizeof(float));
  auto fn = std::make_shared<AttentionBackward>();
  fn->buffer = out.impl()->storage;
  fn->lse = (float*)ptr(out) + out.numel();
  fn->seqs = seqs;
  fn->scale = sc;
  if (tensor::Graph* g = tensor::capturing_graph()) g->keep(seqs);
  LMPB_OK_OR_THROW(lmpb_attention(pq, pk, pv, (float*)ptr(out), fn->lse, (int64_t)s[0], (int)s[1], (int)t[1],
                                  (int)s[2], sc, seqs->handle, tensor::current_stream()));
  return output(out, rg, fn, std::move(in));
}

}  // namespace ops

void adamw_step(const std::vector<Variable>& params, const std::vector<Tensor>& exp_avg,
                const std::vector<Tensor>& exp_avg_sq, const Tensor& step, Scalar lr, Scalar beta1, Scalar beta2,
                Scalar eps, Scalar weight_decay) {
  LMP_CHECK(exp_avg.size() == params.size() && exp_avg_sq.size() == params.size(),
            "adamw_step: " << params.size() << " parameters, " << exp_avg.size() << " and " << exp_avg_sq.size() << " moments");
  LMP_CHECK(step.defined() && step.device() == DeviceType::CUDA && step.type() == DataType::Int64 && step.numel() == 2,
            "adamw_step: step must be a CUDA int64 tensor of 2 values");
  std::vector<lmpb_adamw_tensor> ts;
  std::unordered_set<void*> seen;
  DataType dt = DataType::Float32;
  for (size_t i = 0; i < params.size(); ++i) {
    const Variable& p = params[i];
    LMP_CHECK(p.defined() && on_cuda(p) && floating(p.data().type()), "adamw_step: parameter " << i << " must be a float32 or float64 CUDA tensor");
    if (i == 0) dt = p.data().type();
    LMP_CHECK(p.data().type() == dt, "adamw_step: all parameters must have one dtype");
    LMP_CHECK(p.requires_grad(), "adamw_step: parameter " << i << " does not require a gradient");
    for (const Tensor* t : {&exp_avg[i], &exp_avg_sq[i], &p.grad()})
      LMP_CHECK(t->defined() && t->device() == DeviceType::CUDA && t->type() == dt && t->shape() == p.data().shape(),
                "adamw_step: the moments and the gradient must match parameter " << i << " in shape, dtype and device");
  }
  std::vector<ImplPtr> pending;  // gradients still pending: one batch, so that they share kernels
  for (const Variable& p : params) pending.push_back(p.grad().impl());
  tensor::realize_all(pending);
  for (size_t i = 0; i < params.size(); ++i) {
    const Variable& p = params[i];
    const int64_t n = (int64_t)p.data().numel();
    if (n == 0) continue;
    const lmpb_adamw_tensor t{ptr(p.data()), ptr(p.grad()), ptr(exp_avg[i]), ptr(exp_avg_sq[i]), n};
    for (void* x : {t.param, t.exp_avg, t.exp_avg_sq})
      LMP_CHECK(seen.insert(x).second, "adamw_step: parameter " << i << " or its moments appear twice");
    ts.push_back(t);
  }
  if (tensor::Graph* g = tensor::capturing_graph()) {  // the optimizer and the gradients may go before the recorded step
    for (const auto* list : {&exp_avg, &exp_avg_sq})
      for (const Tensor& t : *list) g->keep(t.impl());
    for (const Variable& p : params) {
      g->keep(p.data().impl());
      g->keep(p.grad().impl());
    }
    g->keep(step.impl());
  }
  LMPB_OK_OR_THROW(lmpb_adamw((int)dt, ts.data(), (int)ts.size(), lr, beta1, beta2, eps, weight_decay,
                              static_cast<int64_t*>(ptr(step)), tensor::current_stream()));
}

}  // namespace autograd
}  // namespace lmp
