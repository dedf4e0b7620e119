// Autograd nodes of the operators whose training step is bound by the host: attention over long rows, norm + rotation of queries and
// keys (no counterpart in the reference).  torch runs a node's backward on a thread of its own.  A Python function has to be entered
// there, with the interpreter's lock handed over twice, and runs on a core that has not seen it: with 128 rows of 21 tokens and 8
// heads (fp32) a step of forward and backward took 147 us, of which the kernels are busy for 46.  These nodes do the same without the
// interpreter: 70 us.  Arguments are checked in Python (ops.py), which also fills the argument struct; the C entry points of
// libmmt_amd.so are handed over as addresses, so that this file needs torch's headers and nothing of the library's.
// The entry points `plain_*` fill the struct themselves where nothing has to be said or copied, and return None otherwise, upon which the
// caller goes through the checks: a single token's call takes 8 us, 12 through the checks in Python, 16 with the node in Python too.
#include <ATen/FuncTorchTLS.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/extension.h>

#include "../../include/mmt_amd.h"

namespace {

using at::Tensor;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;
typedef std::optional<Tensor> Maybe;

struct Entries {
  decltype(&mmt_last_error) last_error;
  decltype(&mmt_long_attention_workspace_bytes) attention_workspace;
  decltype(&mmt_long_attention_fwd) attention_fwd;
  decltype(&mmt_long_attention_bwd) attention_bwd;
  decltype(&mmt_qk_norm_rope_fwd) rope_fwd;
  decltype(&mmt_qk_norm_rope_workspace_bytes) rope_workspace;
  decltype(&mmt_qk_norm_rope_bwd) rope_bwd;
} lib;

struct Failure : std::runtime_error {
  using std::runtime_error::runtime_error;
};
void check(int rc) {
  if (rc) throw Failure(lib.last_error());
}

void *stream_of(const Tensor &t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
Tensor like(const Tensor &t) { return at::empty(t.sizes(), at::TensorOptions().dtype(t.scalar_type()).device(t.device())); }
Tensor bytes(size_t n, const Tensor &beside) { return at::empty({(int64_t)n}, at::TensorOptions().dtype(at::kByte).device(beside.device())); }
template <typename T> const T *address(const Tensor &t) { return t.defined() ? (const T *)t.const_data_ptr() : nullptr; }

// What a tensor subclass, a lazily negated view or a lazy zero stands for is not what lies at its address (or it has none): such arguments
// go through the dispatcher, which turns them into plain ones
bool has_memory(const Tensor &t) { return !t.unsafeGetTensorImpl()->is_python_dispatch() && !t.is_neg() && !t._is_zerotensor(); }
// a gradient, or what saved-tensor hooks gave back, as plain memory
Tensor in_memory(const Tensor &t) {
  if (has_memory(t)) return t;
  if (t.unsafeGetTensorImpl()->is_python_dispatch()) throw Failure("a tensor subclass without memory of its own arrived in the backward pass");
  return t._is_zerotensor() ? at::zeros(t.sizes(), at::TensorOptions().dtype(t.scalar_type()).device(t.device())) : t.resolve_neg();
}

// Row strides of a (B, L, heads, dh) tensor as the kernels read them where it lies, of a copy where they cannot (ops._head_rows)
struct Rows {
  const void *p;
  int64_t b, r, h;
};
bool in_place(const Tensor &t, Rows &s) {
  const int64_t odd = 15 / t.element_size();
  s = {t.const_data_ptr(), t.size(0) > 1 ? t.stride(0) : 0, t.size(1) > 1 ? t.stride(1) : 0, t.size(2) > 1 ? t.stride(2) : 0};
  return !(t.stride(3) != 1 && t.size(3) > 1) && !((uintptr_t)s.p & 15) && !((s.b | s.r | s.h) & odd) && s.r * t.element_size() < (1 << 25);
}
Rows rows(Tensor &t) {
  Rows s;
  t = in_memory(t);
  for (int copies = 0; !in_place(t, s); ++copies) {
    TORCH_CHECK(copies < 2, "rows cannot be laid out for the kernels");
    t = copies ? t.clone(at::MemoryFormat::Contiguous) : t.contiguous();
  }
  return s;
}
// (0: none of them)
int element_type(const Tensor &t, int &type) {
  const auto s = t.scalar_type();
  type = s == at::kFloat ? MMT_F32 : s == at::kBFloat16 ? MMT_BF16 : MMT_F16;
  return s == at::kFloat || s == at::kBFloat16 || s == at::kHalf;
}
constexpr int64_t MOST = 1 << 30;
bool beside(const Tensor &t, const Tensor &q) { return t.defined() && t.is_cuda() && t.device() == q.device() && t.layout() == at::kStrided && has_memory(t); }
// an optional contiguous tensor beside q
bool side(const Maybe &t, const Tensor &q, at::ScalarType type, at::IntArrayRef shape) {
  return !t || (beside(*t, q) && t->scalar_type() == type && t->sizes() == shape && t->is_contiguous());
}
template <typename T> const T *address(const Maybe &t) { return t ? (const T *)t->const_data_ptr() : nullptr; }

// what these nodes do not support, of constants either, has to be an error, as with any other function of torch that does not
void supported(std::initializer_list<Tensor> inputs) {
  const auto &functorch = at::functorch::functorchTLSAccessor();
  if (functorch) functorch->checkSupportsCppAutogradFunction();
  for (const Tensor &t : inputs)
    if (t.defined() && t._fw_grad(0).defined()) throw Failure("forward-mode gradients are not supported");
}

// A leaf that an eager graph which still lives has brought its gradient accumulator into: the accumulator belongs to that graph's stream,
// and the captured backward pass would make this stream wait for the captured one, which ends the capture and the process with it.
void capturable(std::initializer_list<Tensor> inputs, c10::Device device) {
  if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
  const auto here = c10::hip::getCurrentHIPStream(device.index()).id();
  for (const Tensor &t : inputs) {
    if (!t.defined() || !t.requires_grad() || !t.is_leaf()) continue;
    const auto accumulator = torch::autograd::impl::try_get_grad_accumulator(t);
    if (accumulator && accumulator->stream() && accumulator->stream()->id() != here)
      throw Failure("a graph of this leaf on another stream still lives: capture the step on leaves that are made inside the capture");
  }
}

// the gradients have no history of their own: a second derivative is an error, not a silent zero
variable_list final_grads(variable_list &&g, const char *what) {
  if (!at::GradMode::is_enabled()) return std::move(g);
  for (Tensor &t : g)
    if (t.defined()) t.set_requires_grad(true);
  return torch::autograd::DelayedError(std::string(what) + ": there is no second derivative", (int64_t)g.size()).apply(std::move(g));
}

template <typename N> std::shared_ptr<N> node_for(std::initializer_list<Tensor> inputs) {
  std::shared_ptr<N> n(new N(), torch::autograd::deleteNode);
  torch::autograd::edge_list edges;
  for (const Tensor &t : inputs) edges.push_back(t.defined() ? torch::autograd::impl::gradient_edge(t) : torch::autograd::Edge());
  n->set_next_edges(std::move(edges));
  return n;
}

// ---- attention over long rows ----------------------------------------------------------------------------------------------
struct MmtLongAttentionBackward : public Node {
  mmt_long_attention a;
  SavedVariable out, lse, low, q, k, v, prefix, q_doc, k_doc, kv_len, slopes, rel_bias, rel_buckets;
  std::string name() const override { return "MmtLongAttentionBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (SavedVariable *s : {&out, &lse, &low, &q, &k, &v, &prefix, &q_doc, &k_doc, &kv_len, &slopes, &rel_bias, &rel_buckets}) s->reset_data();
  }
  variable_list apply(variable_list &&grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    Tensor dout = grads[0], dlse = grads[1];
    if (!dout.defined() && !dlse.defined()) return variable_list(4);
    const auto self = shared_from_this();
    const Tensor o = out.unpack(self), l = lse.unpack(self), lo = low.unpack(), pf = prefix.unpack(), qd = q_doc.unpack(), kd = k_doc.unpack(),
                 kl = kv_len.unpack(), sl = slopes.unpack(), rb = rel_bias.unpack(), ru = rel_buckets.unpack();
    Tensor qt = q.unpack(), kt = k.unpack(), vt = v.unpack();
    variable_list g(4);
    {
      c10::DeviceGuard device(qt.device());
      at::AutoDispatchBelowADInplaceOrView below;
      // (saved tensors may come back at other addresses)
      const Rows rq = rows(qt), rk = rows(kt), rv = rows(vt);
      a.q = rq.p, a.q_bs = rq.b, a.q_rs = rq.r, a.q_hs = rq.h;
      a.k = rk.p, a.k_bs = rk.b, a.k_rs = rk.r, a.k_hs = rk.h;
      a.v = rv.p, a.v_bs = rv.b, a.v_rs = rv.r, a.v_hs = rv.h;
      a.prefix = address<int32_t>(pf), a.q_doc = address<int32_t>(qd), a.k_doc = address<int32_t>(kd), a.kv_len = address<int32_t>(kl);
      a.slopes = address<float>(sl), a.rel_bias = address<float>(rb), a.rel_buckets = address<int32_t>(ru);
      if (!dout.defined()) dout = at::zeros_like(o);
      const Rows rd = rows(dout);
      if (dlse.defined()) dlse = in_memory(dlse).contiguous();
      g[0] = like(qt), g[1] = like(kt), g[2] = like(vt);
      if (rb.defined()) g[3] = like(rb);
      if ((int64_t)a.B * a.Lq * a.Lk == 0) {
        for (Tensor &t : g)
          if (t.defined()) t.zero_();
      } else {
        const size_t n = lib.attention_workspace(&a, 1);
        const Tensor ws = bytes(n, qt);
        check(lib.attention_bwd(&a, o.const_data_ptr(), lo.defined() ? lo.const_data_ptr() : nullptr, (const float *)l.const_data_ptr(), rd.p, rd.b, rd.r,
                                rd.h, address<float>(dlse), g[0].mutable_data_ptr(), g[1].mutable_data_ptr(), g[2].mutable_data_ptr(),
                                rb.defined() ? (float *)g[3].mutable_data_ptr() : nullptr, ws.mutable_data_ptr(), n, stream_of(qt)));
      }
    }
    return final_grads(std::move(g), "long_attention");
  }
};

// `args`: address of a checked mmt_long_attention that describes the tensors
std::tuple<Tensor, Tensor> long_attention(uintptr_t args, const Tensor &q, const Tensor &k, const Tensor &v, const Maybe &prefix, const Maybe &q_doc,
                                          const Maybe &k_doc, const Maybe &kv_len, const Maybe &slopes, const Maybe &rel_bias, const Maybe &rel_buckets) {
  const mmt_long_attention &a = *(const mmt_long_attention *)args;
  const Tensor table = rel_bias.value_or(Tensor());
  supported({q, k, v, table, slopes.value_or(Tensor())});
  const bool wanted = torch::autograd::compute_requires_grad(q, k, v, table);
  c10::DeviceGuard device(q.device());
  if (wanted) capturable({q, k, v, table}, q.device());
  Tensor out, lse, low;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    out = like(q);
    lse = at::empty({a.B, a.H, a.Lq}, at::TensorOptions().dtype(at::kFloat).device(q.device()));
    if (wanted && a.dtype != MMT_F32) low = like(q);
    if (!a.Lk) {
      out.zero_(), lse.fill_(-INFINITY);
      if (low.defined()) low.zero_();
    } else if (a.B && a.Lq) {
      const size_t n = lib.attention_workspace(&a, 0);
      const Tensor ws = n ? bytes(n, q) : Tensor();
      check(lib.attention_fwd(&a, out.mutable_data_ptr(), low.defined() ? low.mutable_data_ptr() : nullptr, (float *)lse.mutable_data_ptr(),
                              n ? ws.mutable_data_ptr() : nullptr, n, stream_of(q)));
    }
  }
  if (wanted) {
    auto node = node_for<MmtLongAttentionBackward>({q, k, v, table});
    node->a = a;
    torch::autograd::set_history({out, lse}, node);
    node->out = SavedVariable(out, true), node->lse = SavedVariable(lse, true), node->low = SavedVariable(low, false);
    node->q = SavedVariable(q, false), node->k = SavedVariable(k, false), node->v = SavedVariable(v, false);
    node->prefix = SavedVariable(prefix, false), node->q_doc = SavedVariable(q_doc, false), node->k_doc = SavedVariable(k_doc, false);
    node->kv_len = SavedVariable(kv_len, false), node->slopes = SavedVariable(slopes, false);
    node->rel_bias = SavedVariable(table, false), node->rel_buckets = SavedVariable(rel_buckets, false);
  }
  return {out, lse};
}

std::optional<std::tuple<Tensor, Tensor>> plain_long_attention(const Tensor &q, const Tensor &k, const Tensor &v, std::optional<double> scale, bool causal,
                                                               const Maybe &prefix, const Maybe &q_doc, const Maybe &k_doc, const Maybe &kv_len,
                                                               double softcap, const Maybe &slopes, const Maybe &rel_bias, const Maybe &rel_buckets) {
  mmt_long_attention a = {};
  if (!beside(q, q) || !element_type(q, a.dtype) || q.dim() != 4 || !beside(k, q) || !beside(v, q) || k.dim() != 4 ||
      k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type() || k.sizes() != v.sizes())
    return std::nullopt;
  const int64_t B = q.size(0), Lq = q.size(1), H = q.size(2), dh = q.size(3), Lk = k.size(1), Hk = k.size(2);
  if (k.size(0) != B || k.size(3) != dh || Hk < 1 || H < 1 || H % Hk || std::max({B, Lq, Lk, H}) > MOST) return std::nullopt;
  if ((prefix && !causal) || (softcap != 0. && (float)softcap == 0.f) || !q_doc != !k_doc || !rel_bias != !rel_buckets) return std::nullopt;
  if (slopes && slopes->requires_grad() && at::GradMode::is_enabled()) return std::nullopt;
  Rows rq, rk, rv;
  if (!in_place(q, rq) || !in_place(k, rk) || !in_place(v, rv)) return std::nullopt;
  if (!side(prefix, q, at::kInt, {B}) || !side(kv_len, q, at::kInt, {B}) || !side(q_doc, q, at::kInt, {B, Lq}) || !side(k_doc, q, at::kInt, {B, Lk}) ||
      !side(slopes, q, at::kFloat, {H}))
    return std::nullopt;
  if (rel_bias) {
    if (!beside(*rel_bias, q) || rel_bias->dim() != 2 || !beside(*rel_buckets, q) || rel_buckets->dim() != 1 || rel_buckets->numel() < 3 ||
        rel_buckets->numel() % 2 == 0 || rel_buckets->numel() > MOST || rel_bias->size(1) > MOST || !side(rel_bias, q, at::kFloat, {H, rel_bias->size(1)}) ||
        !side(rel_buckets, q, at::kInt, {rel_buckets->numel()}))
      return std::nullopt;
    a.n_buckets = (int)rel_bias->size(1), a.reach = (int)(rel_buckets->numel() / 2);
  }
  a.q = rq.p, a.k = rk.p, a.v = rv.p;
  a.q_bs = rq.b, a.q_rs = rq.r, a.q_hs = rq.h, a.k_bs = rk.b, a.k_rs = rk.r, a.k_hs = rk.h, a.v_bs = rv.b, a.v_rs = rv.r, a.v_hs = rv.h;
  a.B = (int)B, a.Lq = (int)Lq, a.Lk = (int)Lk, a.H = (int)H, a.Hk = (int)Hk, a.dh = (int)std::min(dh, MOST), a.causal = causal;
  a.scale = (float)(scale ? *scale : 1. / std::sqrt((double)dh)), a.softcap = (float)softcap;
  a.prefix = address<int32_t>(prefix), a.kv_len = address<int32_t>(kv_len), a.q_doc = address<int32_t>(q_doc), a.k_doc = address<int32_t>(k_doc);
  a.slopes = address<float>(slopes), a.rel_bias = address<float>(rel_bias), a.rel_buckets = address<int32_t>(rel_buckets);
  return long_attention((uintptr_t)&a, q, k, v, prefix, q_doc, k_doc, kv_len, slopes, rel_bias, rel_buckets);
}

// ---- norm + rotation of queries and keys -----------------------------------------------------------------------------------
struct MmtQkNormRopeBackward : public Node {
  mmt_qk_norm_rope a;
  SavedVariable q, k, q_weight, k_weight, inv_freq, positions;
  std::string name() const override { return "MmtQkNormRopeBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (SavedVariable *s : {&q, &k, &q_weight, &k_weight, &inv_freq, &positions}) s->reset_data();
  }
  variable_list apply(variable_list &&grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    Tensor dqo = grads[0], dko = grads[1];
    if (!dqo.defined() && !dko.defined()) return variable_list(4);
    Tensor qt = q.unpack(), kt = k.unpack();
    const Tensor qw = q_weight.unpack(), kw = k_weight.unpack(), fr = inv_freq.unpack(), ps = positions.unpack();
    variable_list g(4);
    {
      c10::DeviceGuard device(qt.device());
      at::AutoDispatchBelowADInplaceOrView below;
      const Rows rq = rows(qt), rk = rows(kt);
      a.q = rq.p, a.q_bs = rq.b, a.q_rs = rq.r, a.q_hs = rq.h;
      a.k = rk.p, a.k_bs = rk.b, a.k_rs = rk.r, a.k_hs = rk.h;
      a.q_weight = qw.const_data_ptr(), a.k_weight = kw.const_data_ptr();
      a.inv_freq = address<double>(fr), a.positions = address<int64_t>(ps);
      if (!dqo.defined()) dqo = at::zeros_like(qt);
      if (!dko.defined()) dko = at::zeros_like(kt);
      const Rows rdq = rows(dqo), rdk = rows(dko);
      g[0] = like(qt), g[1] = like(kt), g[2] = like(qw), g[3] = like(kw);
      if ((int64_t)a.B * a.L == 0) {
        g[2].zero_(), g[3].zero_();
      } else {
        const size_t n = lib.rope_workspace(&a);
        const Tensor ws = bytes(n, qt);
        check(lib.rope_bwd(&a, rdq.p, rdq.b, rdq.r, rdq.h, rdk.p, rdk.b, rdk.r, rdk.h, g[0].mutable_data_ptr(), g[1].mutable_data_ptr(),
                           g[2].mutable_data_ptr(), g[3].mutable_data_ptr(), ws.mutable_data_ptr(), n, stream_of(qt)));
      }
    }
    return final_grads(std::move(g), "qk_norm_rope");
  }
};

std::tuple<Tensor, Tensor> qk_norm_rope(uintptr_t args, const Tensor &q, const Tensor &k, const Tensor &q_weight, const Tensor &k_weight,
                                        const Tensor &inv_freq, const Maybe &positions) {
  const mmt_qk_norm_rope &a = *(const mmt_qk_norm_rope *)args;
  supported({q, k, q_weight, k_weight, inv_freq});
  const bool wanted = torch::autograd::compute_requires_grad(q, k, q_weight, k_weight);
  c10::DeviceGuard device(q.device());
  if (wanted) capturable({q, k, q_weight, k_weight}, q.device());
  Tensor qo, ko;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    qo = like(q), ko = like(k);
    if (a.B && a.L) check(lib.rope_fwd(&a, qo.mutable_data_ptr(), ko.mutable_data_ptr(), stream_of(q)));
  }
  if (wanted) {
    auto node = node_for<MmtQkNormRopeBackward>({q, k, q_weight, k_weight});
    node->a = a;
    torch::autograd::set_history({qo, ko}, node);
    node->q = SavedVariable(q, false), node->k = SavedVariable(k, false), node->q_weight = SavedVariable(q_weight, false);
    node->k_weight = SavedVariable(k_weight, false), node->inv_freq = SavedVariable(inv_freq, false), node->positions = SavedVariable(positions, false);
  }
  return {qo, ko};
}

std::optional<std::tuple<Tensor, Tensor>> plain_qk_norm_rope(const Tensor &q, const Tensor &k, const Tensor &q_weight, const Tensor &k_weight,
                                                             const Tensor &inv_freq, const Maybe &positions, double eps, bool interleaved) {
  mmt_qk_norm_rope a = {};
  if (!beside(q, q) || !element_type(q, a.dtype) || q.dim() != 4 || !beside(k, q) || k.dim() != 4 || k.scalar_type() != q.scalar_type())
    return std::nullopt;
  const int64_t B = q.size(0), L = q.size(1), H = q.size(2), dh = q.size(3), Hk = k.size(2);
  if (k.size(0) != B || k.size(1) != L || k.size(3) != dh || Hk < 1 || H < 1 || std::max({B, L, H, Hk}) > MOST) return std::nullopt;
  if (!beside(q_weight, q) || !element_type(q_weight, a.w_dtype) || (a.w_dtype != a.dtype && a.w_dtype != MMT_F32)) return std::nullopt;
  if (!side(q_weight, q, q_weight.scalar_type(), {dh}) || !side(k_weight, q, q_weight.scalar_type(), {dh})) return std::nullopt;
  if (!beside(inv_freq, q) || inv_freq.dim() != 1 || inv_freq.numel() > MOST / 2 || !side(inv_freq, q, at::kDouble, {inv_freq.numel()}) ||
      !side(positions, q, at::kLong, {B, L}) || (inv_freq.requires_grad() && at::GradMode::is_enabled()))
    return std::nullopt;
  Rows rq, rk;
  if (!in_place(q, rq) || !in_place(k, rk)) return std::nullopt;
  a.q = rq.p, a.k = rk.p, a.q_weight = q_weight.const_data_ptr(), a.k_weight = k_weight.const_data_ptr();
  a.q_bs = rq.b, a.q_rs = rq.r, a.q_hs = rq.h, a.k_bs = rk.b, a.k_rs = rk.r, a.k_hs = rk.h;
  a.inv_freq = address<double>(inv_freq), a.positions = address<int64_t>(positions);
  a.B = (int)B, a.L = (int)L, a.H = (int)H, a.Hk = (int)Hk, a.dh = (int)std::min(dh, MOST), a.rot = (int)(2 * inv_freq.numel());
  a.interleaved = interleaved, a.eps = (float)eps;
  return qk_norm_rope((uintptr_t)&a, q, k, q_weight, k_weight, inv_freq, positions);
}

}  // namespace

PYBIND11_MODULE(_autograd, m) {
  // entries: addresses in the order of struct Entries; error: the exception that a failed call raises
  // sizes: what the caller takes the argument structs' sizes for
  m.def("bind", [](const std::vector<uintptr_t> &entries, std::pair<size_t, size_t> sizes, py::object error) {
    TORCH_CHECK(sizes.first == sizeof(mmt_long_attention) && sizes.second == sizeof(mmt_qk_norm_rope), "bind: other argument structs");
    TORCH_CHECK(entries.size() * sizeof(uintptr_t) == sizeof(Entries), "bind: ", sizeof(Entries) / sizeof(uintptr_t), " entry points are needed");
    std::memcpy((void *)&lib, entries.data(), sizeof(Entries));
    static PyObject *raised = nullptr;
    if (!raised)
      py::register_exception_translator([](std::exception_ptr p) {
        try {
          if (p) std::rethrow_exception(p);
        } catch (const Failure &e) {
          PyErr_SetString(raised, e.what());
        }
      });
    raised = error.release().ptr();
  });
  m.def("long_attention", &long_attention, py::call_guard<py::gil_scoped_release>());
  m.def("qk_norm_rope", &qk_norm_rope, py::call_guard<py::gil_scoped_release>());
  m.def("plain_long_attention", &plain_long_attention, py::call_guard<py::gil_scoped_release>());
  m.def("plain_qk_norm_rope", &plain_qk_norm_rope, py::call_guard<py::gil_scoped_release>());
}
