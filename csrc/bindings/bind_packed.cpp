// Python bindings of the operators around whole prompts and packed texts (csrc/ops/packed.hpp).  As in bind_serving.cpp every function checks its operands,
// allocates through torch and launches on the current stream of the operands' device.  Those that models train with are autograd nodes of their own here: a
// Python node costs more host time than the kernels of a few thousand tokens take.
#include "../ops/ops.hpp"
#include "../ops/packed.hpp"
#include "../symm/cu_driver.hpp"
#include "bind.hpp"
#include "operand_checks.hpp"

#include <cmath>

namespace py = pybind11;

namespace mccl {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

namespace {

void need_no_tangent(const at::Tensor& t, const char* what) {
  MCCL_CHECK_TENSOR(!(c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(/*level=*/0).defined()), what << ": has no forward-mode derivative; a tangent would be lost");
}
// A backward pass that would itself be differentiated.
void need_first_order(const char* what) { MCCL_CHECK_TENSOR(!at::GradMode::is_enabled(), what << ": has no second derivative (create_graph)"); }

// As tensor maps and 16-byte accesses take them: gradients come in any strides and from any place on (contiguous() would leave one that only begins off a 16-byte boundary as it is).
at::Tensor rows_of_heads(const at::Tensor& t) { return vector_rows(t) && !repeated(t) ? t : t.clone(at::MemoryFormat::Contiguous); }

// The operands of a call as the kernels take them.
struct Attention {
  at::Tensor q, k, v, offsets, k_offsets;
  double scale;
  int64_t window, sinks;

  ops::PackedAttentionArgs args(const char* op) const {
    ops::PackedAttentionArgs a;
    a.type = half16(q, op);
    a.q = tokens_of(q, "packed_attention(q)");
    a.k = tokens_of(k, "packed_attention(k)");
    a.v = tokens_of(v, "packed_attention(v)");
    a.offsets = offsets.data_ptr<int>();
    a.k_offsets = k_offsets.data_ptr<int>();
    a.tokens = as_int(q.size(0), op);
    a.k_tokens = as_int(k.size(0), op);
    a.sequences = as_int(offsets.numel() - 1, op);
    a.heads = as_int(q.size(1), op);
    a.kv_heads = as_int(k.size(1), op);
    a.head_dim = as_int(q.size(2), op);
    a.scale = static_cast<float>(scale);
    const int64_t most = std::numeric_limits<int>::max();
    a.window = static_cast<int>(std::min(window, most));
    a.sinks = static_cast<int>(std::min(sinks, most));
    return a;
  }
};

// (o, lse [heads, tokens] or undefined, what rounding o left or undefined)
std::tuple<at::Tensor, at::Tensor, at::Tensor> attention_forward(const Attention& x, bool lse, bool rest) {
  const char* op = "packed_attention";
  ops::PackedAttentionArgs a = x.args(op);
  c10::cuda::CUDAGuard guard(x.q.device());
  at::Tensor o = empty_on(x.q, {x.q.size(0), x.q.size(1), x.q.size(2)}, x.q.scalar_type()), l, r;
  a.o = o.data_ptr();
  if (lse) {
    l = empty_on(x.q, {x.q.size(1), x.q.size(0)}, at::kFloat);
    a.lse = l.data_ptr<float>();
  }
  if (rest) {
    r = empty_on(x.q, o.sizes(), x.q.scalar_type());
    a.o_rest = r.data_ptr();
  }
  if (a.k_tokens == 0 || a.sequences == 0) {   // nothing to see
    o.zero_();
    if (lse) l.fill_(-std::numeric_limits<float>::infinity());
  } else {
    at::Tensor workspace;
    if (const size_t bytes = ops::packed_attention_workspace(a)) {
      workspace = empty_on(x.q, {static_cast<int64_t>(bytes)}, at::kByte);
      a.workspace = workspace.data_ptr();
    }
    CuDriver::get().ensure_context(x.q.get_device());   // (tensor maps)
    check_launch(ops::packed_attention(a, stream_of(x.q)), op);
  }
  return {o, l, r};
}

struct AttentionNode : torch::autograd::Function<AttentionNode> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& offsets, const at::Tensor& k_offsets, double scale,
                               int64_t window, int64_t sinks) {
    const auto [o, lse, rest] = attention_forward({q, k, v, offsets, k_offsets, scale, window, sinks}, true, true);
    ctx->save_for_backward({q, k, v, offsets, k_offsets, o, lse, rest});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["window"] = window;
    ctx->saved_data["sinks"] = sinks;
    ctx->mark_non_differentiable({lse});
    ctx->set_materialize_grads(false);   // (zeros for lse would be a launch of their own)
    return {o, lse};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const char* op = "packed_attention";
    need_first_order(op);
    if (!grads[0].defined()) return variable_list(8);
    const auto s = ctx->get_saved_variables();
    const Attention x{s[0], s[1], s[2], s[3], s[4], ctx->saved_data["scale"].toDouble(), ctx->saved_data["window"].toInt(), ctx->saved_data["sinks"].toInt()};
    const at::Tensor &o = s[5], &lse = s[6], &rest = s[7], d_o = rows_of_heads(grads[0]);
    c10::cuda::CUDAGuard guard(x.q.device());
    at::Tensor dq = empty_on(x.q, x.q.sizes(), at::kBFloat16), dk = empty_on(x.q, x.k.sizes(), at::kBFloat16), dv = empty_on(x.q, x.v.sizes(), at::kBFloat16);
    if (x.k.size(0) == 0 || x.q.numel() == 0 || x.offsets.numel() == 1) {
      dq.zero_();
      dk.zero_();
      dv.zero_();
    } else {
      ops::PackedAttentionGradArgs a;
      a.f = x.args(op);
      a.f.lse = lse.data_ptr<float>();
      a.f.o = o.data_ptr();
      a.f.o_rest = rest.data_ptr();
      a.d_o = tokens_of(d_o, "packed_attention(gradient)");
      a.dq = dq.data_ptr();
      a.dk = dk.data_ptr();
      a.dv = dv.data_ptr();
      at::Tensor delta = empty_on(x.q, lse.sizes(), at::kFloat);
      a.delta = delta.data_ptr<float>();
      CuDriver::get().ensure_context(x.q.get_device());
      check_launch(ops::packed_attention_grad(a, stream_of(x.q)), "packed_attention backward");
    }
    return {dq, dk, dv, at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

// Rotation tables and positions of a call.
struct Turn {
  at::Tensor cos, sin, positions;   // positions may be undefined
  bool halves;

  // (q, k or undefined) turned; with `inverse` the other way
  std::pair<at::Tensor, at::Tensor> operator()(const at::Tensor& q, const at::Tensor& k, bool inverse) const {
    const char* op = "rotary";
    ops::RotaryArgs a;
    a.type = half16(q, op);
    a.cos = cos.data_ptr<float>();
    a.sin = sin.data_ptr<float>();
    a.rope_rows = as_int(cos.size(0), op);
    a.width = as_int(cos.size(1), op);
    a.positions = positions.defined() ? positions.data_ptr<int>() : nullptr;
    a.tokens = as_int(q.size(0), op);
    a.head_dim = as_int(q.size(2), op);
    a.halves = halves;
    a.inverse = inverse;
    c10::cuda::CUDAGuard guard(q.device());
    at::Tensor out[2];
    const at::Tensor* in[2] = {&q, &k};
    ops::RotaryPart* part[2] = {&a.q, &a.k};
    for (int i = 0; i < 2; ++i) {
      if (!in[i]->defined()) continue;
      out[i] = empty_on(q, in[i]->sizes(), q.scalar_type());
      part[i]->x = tokens_of(*in[i], i == 0 ? "rotary(q)" : "rotary(k)");
      part[i]->out = out[i].data_ptr();
      part[i]->heads = as_int(in[i]->size(1), op);
    }
    check_launch(ops::rotary(a, stream_of(q)), op);
    return {out[0], out[1]};
  }
};

struct RotaryNode : torch::autograd::Function<RotaryNode> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& q, const c10::optional<at::Tensor>& k, const at::Tensor& cos, const at::Tensor& sin,
                               const c10::optional<at::Tensor>& positions, bool halves) {
    const at::Tensor at = positions.value_or(at::Tensor());
    ctx->save_for_backward({cos, sin, at});
    ctx->saved_data["halves"] = halves;
    ctx->saved_data["both"] = k.has_value();
    const auto [a, b] = Turn{cos, sin, at, halves}(q, k.value_or(at::Tensor()), false);
    return k.has_value() ? variable_list{a, b} : variable_list{a};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    need_first_order("rotary");
    const auto s = ctx->get_saved_variables();
    const bool both = ctx->saved_data["both"].toBool();
    const auto [a, b] = Turn{s[0], s[1], s[2], ctx->saved_data["halves"].toBool()}(rows_of_heads(grads[0]), both ? rows_of_heads(grads[1]) : at::Tensor(), true);
    return {a, b, at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

// A setting of a sampler: a number, or one per row.
template <typename T>
ops::RowSetting<T> row_setting(const py::object& value, const at::Tensor& logits, at::ScalarType dtype, const char* what, double low, double high) {
  ops::RowSetting<T> s;
  if (THPVariable_Check(value.ptr())) {
    const at::Tensor& t = THPVariable_Unpack(value.ptr());
    need_on(t, logits, what);
    MCCL_CHECK_TENSOR(t.scalar_type() == dtype && t.dim() == 1 && t.numel() == logits.size(0) && t.is_contiguous(),
                      what << ": expected a number or contiguous " << c10::toString(dtype) << " [" << logits.size(0) << "]");
    s.each = t.data_ptr<T>();
    return s;
  }
  const double v = value.cast<double>();
  MCCL_CHECK_TENSOR(v >= low && v <= high, what << ": " << v << " is out of range");
  MCCL_CHECK_TENSOR(std::is_floating_point<T>::value || v == std::floor(v), what << ": " << v << " is not a whole number");
  s.all = static_cast<T>(v);
  return s;
}

}  // namespace

void bind_packed(py::module_& m) {
  m.def(
      "rotary",
      [](const at::Tensor& q, const c10::optional<at::Tensor>& k, const at::Tensor& cos_t, const at::Tensor& sin_t, const c10::optional<at::Tensor>& positions,
         bool halves) -> std::pair<at::Tensor, c10::optional<at::Tensor>> {
        const char* op = "rotary";
        need_on(q, q, op);
        half16(q, op);
        MCCL_CHECK_TENSOR(q.dim() == 3 && q.size(2) > 0 && q.size(2) % 8 == 0, op << ": expected [tokens, heads, head_dim] with a head_dim that is a multiple of 8");
        MCCL_CHECK_TENSOR(q.size(0) < std::numeric_limits<int>::max(), op << ": 2^31 - 1 tokens or more");
        need_no_tangent(q, op);
        bool train = q.requires_grad();
        if (k.has_value()) {
          need_on(*k, q, "rotary(k)");
          need_no_tangent(*k, op);
          MCCL_CHECK_TENSOR(k->scalar_type() == q.scalar_type() && k->dim() == 3 && k->size(0) == q.size(0) && k->size(2) == q.size(2),
                            "rotary(k): another dtype, other tokens or another head_dim than q");
          train = train || k->requires_grad();
        }
        train = train && at::GradMode::is_enabled();
        for (const auto* t : {&cos_t, &sin_t}) {
          need_on(*t, q, "rotary(rope)");
          need_forward_only(*t, "rotary(rope)");
          MCCL_CHECK_TENSOR(t->scalar_type() == at::kFloat && t->dim() == 2 && t->is_contiguous() && reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 == 0,
                            "rotary(rope): cos and sin must be contiguous fp32 [positions, pairs] on a 16-byte boundary");
        }
        MCCL_CHECK_TENSOR(cos_t.sizes() == sin_t.sizes(), "rotary(rope): cos and sin of different sizes");
        MCCL_CHECK_TENSOR(cos_t.size(1) > 0 && cos_t.size(1) % 4 == 0 && 2 * cos_t.size(1) <= q.size(2),
                          "rotary(rope): " << cos_t.size(1) << " pairs for heads of " << q.size(2) << "; multiples of 4 up to half a head are possible");
        if (positions.has_value()) need_int32(*positions, q, q.size(0), "rotary(positions)");
        auto dense = [](const at::Tensor& t) { return repeated(t) ? t.contiguous() : t; };
        const at::Tensor q_ = dense(q);
        tokens_of(q_, "rotary(q)");
        c10::optional<at::Tensor> k_;
        if (k.has_value()) {
          k_ = dense(*k);
          tokens_of(*k_, "rotary(k)");
        }
        at::Tensor a, b;
        if (train) {
          const variable_list r = RotaryNode::apply(q_, k_, cos_t, sin_t, positions, halves);
          a = r[0];
          if (k_.has_value()) b = r[1];
        } else {
          std::tie(a, b) = Turn{cos_t, sin_t, positions.value_or(at::Tensor()), halves}(q_, k_.value_or(at::Tensor()), false);
        }
        if (!b.defined()) return {a, c10::nullopt};
        return {a, b};
      },
      py::arg("q"), py::arg("k"), py::arg("cos"), py::arg("sin"), py::arg("positions") = py::none(), py::arg("halves") = false);

  m.def(
      "sample",
      [](const at::Tensor& logits, const at::Tensor& uniform, const py::object& temperature, const py::object& top_k, const py::object& top_p, const py::object& min_p) {
        const char* op = "sample";
        need_on(logits, logits, op);
        const at::ScalarType type = logits.scalar_type();
        MCCL_CHECK_TENSOR(type == at::kBFloat16 || type == at::kHalf || type == at::kFloat, op << ": expected bf16, fp16 or fp32, got " << c10::toString(type));
        MCCL_CHECK_TENSOR(logits.dim() == 2 && logits.size(1) >= 1 && logits.size(1) <= (1 << 20), op << ": expected [rows, vocab] with 1 to 2^20 tokens");
        MCCL_CHECK_TENSOR(logits.size(1) == 1 || logits.stride(1) == 1, op << ": the logits of a row must be contiguous");
        need_on(uniform, logits, "sample(uniform)");
        MCCL_CHECK_TENSOR((uniform.scalar_type() == at::kFloat || uniform.scalar_type() == at::kDouble) && uniform.dim() == 1 && uniform.numel() == logits.size(0) && uniform.is_contiguous(),
                          "sample(uniform): expected contiguous fp32 or fp64 [" << logits.size(0) << "]");
        ops::SampleArgs a;
        a.logits = logits.data_ptr();
        a.stride = logits.stride(0);
        a.type = type == at::kBFloat16 ? ops::Logits::bf16 : (type == at::kHalf ? ops::Logits::fp16 : ops::Logits::fp32);
        a.rows = as_int(logits.size(0), op);
        a.vocab = as_int(logits.size(1), op);
        a.uniform = uniform.data_ptr();
        a.uniform64 = uniform.scalar_type() == at::kDouble;
        a.temperature = row_setting<float>(temperature, logits, at::kFloat, "sample(temperature)", 0.0, 3.4e38);
        a.top_k = row_setting<int>(top_k, logits, at::kInt, "sample(top_k)", 0.0, std::numeric_limits<int>::max());
        a.top_p = row_setting<float>(top_p, logits, at::kFloat, "sample(top_p)", 0.0, 1.0);
        a.min_p = row_setting<float>(min_p, logits, at::kFloat, "sample(min_p)", 0.0, 1.0);
        c10::cuda::CUDAGuard guard(logits.device());
        at::Tensor tokens = empty_on(logits, {logits.size(0)}, at::kLong);
        a.tokens = reinterpret_cast<long long*>(tokens.data_ptr<int64_t>());
        check_launch(ops::sample(a, stream_of(logits)), op);
        return tokens;
      },
      py::arg("logits"), py::arg("uniform"), py::arg("temperature"), py::arg("top_k"), py::arg("top_p"), py::arg("min_p"));

  m.def(
      "packed_attention",
      [](const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& offsets, const c10::optional<at::Tensor>& k_offsets, double scale, int64_t window,
         int64_t sinks, bool return_lse) -> std::pair<at::Tensor, c10::optional<at::Tensor>> {
        const char* op = "packed_attention";
        bool train = false;
        for (const auto* t : {&q, &k, &v}) {
          need_on(*t, q, op);
          need_no_tangent(*t, op);
          MCCL_CHECK_TENSOR(t->dim() == 3, op << ": expected [tokens, heads, head_dim]");
          MCCL_CHECK_TENSOR(t->scalar_type() == q.scalar_type(), op << ": q, k and v differ in dtype");
          train = train || t->requires_grad();
        }
        train = train && at::GradMode::is_enabled();
        half16(q, op);
        MCCL_CHECK_TENSOR(!train || q.scalar_type() == at::kBFloat16, op << ": gradients are computed in bf16 only (in fp16 the gradients of scores fall below its smallest numbers)");
        MCCL_CHECK_TENSOR(k.sizes() == v.sizes(), op << ": keys and values of different sizes");
        MCCL_CHECK_TENSOR(q.size(2) == k.size(2), op << ": q has head_dim " << q.size(2) << ", k " << k.size(2));
        MCCL_CHECK_TENSOR(q.size(2) > 0 && q.size(2) % 8 == 0 && q.size(2) <= 128, op << ": head_dim must be a multiple of 8 up to 128");
        MCCL_CHECK_TENSOR(k.size(1) > 0 && q.size(1) % k.size(1) == 0, op << ": " << q.size(1) << " query heads over " << k.size(1) << " heads of keys and values");
        MCCL_CHECK_TENSOR(std::max(q.size(0), k.size(0)) < (1 << 29), op << ": 2^29 tokens or more");
        MCCL_CHECK_TENSOR(offsets.dim() == 1 && offsets.numel() >= 1, op << ": offsets must be int32 [sequences + 1]");
        need_int32(offsets, q, offsets.numel(), "packed_attention(offsets)");
        if (k_offsets.has_value()) need_int32(*k_offsets, q, offsets.numel(), "packed_attention(k_offsets)");
        MCCL_CHECK_TENSOR(k_offsets.has_value() || q.size(0) == k.size(0), op << ": " << q.size(0) << " queries and " << k.size(0) << " keys without offsets of their own");
        MCCL_CHECK_TENSOR(std::isfinite(scale) && scale > 0 && static_cast<float>(scale) > 0, op << ": scale must be a positive number");
        MCCL_CHECK_TENSOR(window >= 0 && sinks >= 0, op << ": window and sinks must not be negative");
        // expanded tensors are copied; other strides than the kernels' are refused
        auto dense = [](const at::Tensor& t) { return repeated(t) ? t.contiguous() : t; };
        const at::Tensor q_ = dense(q), k_ = dense(k), v_ = dense(v), ko = k_offsets.value_or(offsets);
        for (const auto* t : {&q_, &k_, &v_}) tokens_of(*t, op);
        at::Tensor o, lse;
        if (train) {
          const variable_list r = AttentionNode::apply(q_, k_, v_, offsets, ko, scale, window, sinks);
          o = r[0];
          lse = r[1];
        } else {
          std::tie(o, lse, std::ignore) = attention_forward({q_, k_, v_, offsets, ko, scale, window, sinks}, return_lse, false);
        }
        if (!return_lse) return {o, c10::nullopt};
        return {o, lse.t()};
      },
      py::arg("q"), py::arg("k"), py::arg("v"), py::arg("offsets"), py::arg("k_offsets") = py::none(), py::arg("scale"), py::arg("window") = 0, py::arg("sinks") = 0,
      py::arg("return_lse") = false);
}

}  // namespace mccl
