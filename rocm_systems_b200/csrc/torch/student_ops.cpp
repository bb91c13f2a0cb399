// Autograd of the student decoder's operators (per-head norms with the rotation, windowed attention) and the distillation loss for Python.
//
// The kernels are the native library's; what is here checks arguments, allocates outputs and records the graph. It is C++ because these
// calls are short: an autograd function written in Python cost 150 us of host time for a forward and backward pass (4 heads, 128 tokens),
// several times what its kernels run.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <atomic>
#include <cmath>

extern "C" {
int b200ops_qk_norm_rope_fwd(const void*, const void*, const void*, int, const float*, void*, void*, long long, int, int, int, int, float, cudaStream_t);
long long b200ops_qk_norm_rope_bwd_scratch(int, int, int);
int b200ops_qk_norm_rope_bwd(const void*, const void*, const void*, const long long*, const void*, const void*, const void*, int, const float*, void*, float*, void*, void*,
                             long long, int, int, int, int, float, cudaStream_t);
int b200ops_window_attention_fwd(const void*, const void*, const void*, void*, float*, void*, const int*, const long long*, int, int, int, int, int, int, int, float,
                                 cudaStream_t);
long long b200ops_window_attention_bwd_scratch(int, int, int, int, int, int, int);
int b200ops_window_attention_bwd_launches(int, int, int, int, int, int, int);
int b200ops_window_attention_bwd(const void*, const void*, const void*, const void*, const void*, const void*, const float*, float*, void*, void*, void*, const int*,
                                 const long long*, int, int, int, int, int, int, int, float, cudaStream_t);
int b200ops_distill_loss(const void*, void*, const long long*, const void*, int, const void*, int, float*, long long, int, int, long long, long long, float, float, float,
                         cudaStream_t);
}

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

std::atomic<long long> gLaunches{0};

void need(bool ok, const char* what) {
  if (ok) return;
  PyErr_SetString(PyExc_AssertionError, what);
  throw py::error_already_set();
}
void check(int rc, const char* what, int launches) {
  if (rc != 0) throw std::runtime_error(std::string(what) + ": CUDA error " + std::to_string(rc));
  gLaunches += launches;
}
void once() { TORCH_CHECK(!at::GradMode::is_enabled(), "this operator's gradient is not itself differentiable (create_graph)"); }

// There is no forward-mode derivative here; without this a tangent would be dropped in silence, as its tensor need not require a gradient.
void noTangent(std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts) need(!t->_fw_grad(/*level=*/0).defined(), "forward-mode derivatives are not implemented (an input is a dual tensor)");
}

bool onOneDevice(const Tensor& t, std::initializer_list<const Tensor*> others) {
  for (const Tensor* o : others)
    if (o->device() != t.device()) return false;
  return t.is_cuda();
}

// `t` [.., .., .., D] if every row of its last dimension is dense and starts on a 16-byte boundary, and no two of them are the same memory;
// else a copy.
Tensor rows16(const Tensor& t) {
  bool fine = t.stride(3) == 1 && (reinterpret_cast<uintptr_t>(t.const_data_ptr()) & 15) == 0;
  for (int d = 0; d < 3; d++) fine = fine && (t.size(d) <= 1 || (t.stride(d) > 0 && t.stride(d) % 8 == 0));
  return fine ? t : t.clone(at::MemoryFormat::Contiguous);
}
// `t` if it is dense and starts on a 16-byte boundary; else a copy.
Tensor dense16(const Tensor& t) {
  return t.is_contiguous() && (reinterpret_cast<uintptr_t>(t.const_data_ptr()) & 15) == 0 ? t : t.clone(at::MemoryFormat::Contiguous);
}
// A hook on saved tensors promises equal values; in which memory they come back is its own affair.
void cameBack(const Tensor& t, at::IntArrayRef sizes, at::ScalarType type, const Tensor& grad) {
  TORCH_CHECK(t.defined() && t.sizes() == sizes && t.scalar_type() == type && t.device() == grad.device(), "a saved tensor came back as something else");
}
// (batch, head, position) strides of [B, heads, S, D] tensors in turn; of a dimension of one the stride is nothing.
template <size_t N> std::array<long long, 3 * N> strides(const std::array<const Tensor*, N>& ts) {
  std::array<long long, 3 * N> s{};
  for (size_t i = 0; i < N; i++)
    for (int d = 0; d < 3; d++) s[3 * i + d] = ts[i]->size(d) > 1 ? ts[i]->stride(d) : 0;
  return s;
}
// [B, heads, S, D] whose memory is [B, S, heads, D], the layout the projections read and write.
Tensor byToken(int64_t B, int64_t heads, int64_t S, int64_t D, const Tensor& like) {
  return at::empty_strided({B, heads, S, D}, {S * heads * D, D, heads * D, 1}, like.options());
}

const void* ptr(const Tensor& t) { return t.const_data_ptr(); }
void* out(const Tensor& t) { return t.mutable_data_ptr(); }
cudaStream_t stream() { return c10::cuda::getCurrentCUDAStream(); }

// ---- norms of queries and keys, rotation ------------------------------------------------------------------------
variable_list normForward(const Tensor& qkv, const Tensor& wq, const Tensor& wk, const Tensor& table, int64_t heads, int64_t kv, double eps) {
  const int64_t B = qkv.size(0), S = qkv.size(1), D = qkv.size(3);
  c10::cuda::OptionalCUDAGuard guard(qkv.device());
  Tensor q = byToken(B, heads, S, D, qkv), k = byToken(B, kv, S, D, qkv);
  check(b200ops_qk_norm_rope_fwd(ptr(qkv), ptr(wq), ptr(wk), wq.scalar_type() == at::kBFloat16, (const float*)ptr(table), out(q), out(k), B * S, (int)S, (int)heads, (int)kv,
                                 (int)D, (float)eps, stream()),
        "qk_norm_rope_fwd", 1);
  return {q, k, qkv.slice(2, heads + kv).transpose(1, 2)};
}

struct QkNormRope : torch::autograd::Function<QkNormRope> {
  static variable_list forward(AutogradContext* ctx, const Tensor& qkvIn, const Tensor& wqIn, const Tensor& wkIn, const Tensor& table, int64_t heads, int64_t kv, double eps) {
    const Tensor qkv = rows16(qkvIn).contiguous(), wq = wqIn.contiguous(), wk = wkIn.contiguous();
    ctx->save_for_backward({qkv, wq, wk, table});
    ctx->saved_data["heads"] = heads;
    ctx->saved_data["kv"] = kv;
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["wide"] = wq.scalar_type() == at::kFloat;
    return normForward(qkv, wq, wk, table, heads, kv, eps);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once();
    const auto saved = ctx->get_saved_variables();
    const int64_t heads = ctx->saved_data["heads"].toInt(), kv = ctx->saved_data["kv"].toInt(), B = grads[0].size(0), S = grads[0].size(2), D = grads[0].size(3);
    const auto weights = ctx->saved_data["wide"].toBool() ? at::kFloat : at::kBFloat16;
    cameBack(saved[0], {B, S, heads + 2 * kv, D}, at::kBFloat16, grads[0]);
    for (int i = 1; i < 3; i++) cameBack(saved[i], {D}, weights, grads[0]);
    cameBack(saved[3], {saved[3].size(0), D / 2, 2}, at::kFloat, grads[0]);
    TORCH_CHECK(saved[3].size(0) >= S, "a saved tensor came back as something else");
    c10::cuda::OptionalCUDAGuard guard(grads[0].device());
    const Tensor qkv = dense16(saved[0]), wq = saved[1].contiguous(), wk = saved[2].contiguous(), table = dense16(saved[3]);
    const Tensor dq = rows16(grads[0]), dk = rows16(grads[1]), dv = rows16(grads[2]);
    const Tensor dqkv = at::empty_like(qkv), dwq = at::empty_like(wq), dwk = at::empty_like(wk);
    const Tensor scratch = at::empty({(int64_t)b200ops_qk_norm_rope_bwd_scratch((int)D, (int)heads, (int)kv)}, qkv.options().dtype(at::kFloat));
    const auto st = strides<3>({&dq, &dk, &dv});
    check(b200ops_qk_norm_rope_bwd(ptr(dq), ptr(dk), ptr(dv), st.data(), ptr(qkv), ptr(wq), ptr(wk), wq.scalar_type() == at::kBFloat16, (const float*)ptr(table), out(dqkv),
                                   (float*)out(scratch), out(dwq), out(dwk), B * S, (int)S, (int)heads, (int)kv, (int)D, (float)ctx->saved_data["eps"].toDouble(), stream()),
          "qk_norm_rope_bwd", 2);
    return {dqkv, dwq, dwk, Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

std::tuple<Tensor, Tensor, Tensor> qkNormRope(const Tensor& qkv, const Tensor& wq, const Tensor& wk, const Tensor& table, int64_t heads, int64_t kv, double eps) {
  need(qkv.dim() == 4 && qkv.scalar_type() == at::kBFloat16, "qkv: [B, S, heads + 2 kv_heads, D] in bf16");
  need(qkv.numel() > 0, "qkv is empty");
  const int64_t S = qkv.size(1), D = qkv.size(3);
  need(heads > 0 && kv > 0 && qkv.size(2) == heads + 2 * kv, "qkv holds heads + 2 kv_heads heads per token");
  need(D % 8 == 0 && D <= 256, "head dimension: a multiple of 8 up to 256");
  need(wq.dim() == 1 && wk.dim() == 1 && wq.size(0) == D && wk.size(0) == D && wq.scalar_type() == wk.scalar_type(), "weights: [D], of one type");
  need(wq.scalar_type() == at::kBFloat16 || wq.scalar_type() == at::kFloat, "weights: bf16 or fp32");
  need(table.dim() == 3 && table.size(0) >= S && table.size(1) == D / 2 && table.size(2) == 2, "table: [at least S, D / 2, 2]");
  need(table.scalar_type() == at::kFloat && table.is_contiguous() && (reinterpret_cast<uintptr_t>(ptr(table)) & 15) == 0, "table: contiguous fp32");
  need(eps >= 0 && std::isfinite(eps), "eps: finite, not negative");
  need(qkv.size(0) * S < (1LL << 30) && heads + 2 * kv < (1LL << 14), "too many positions or heads");
  need(!at::GradMode::is_enabled() || !table.requires_grad(), "table: a gradient is not formed for it");
  noTangent({&qkv, &wq, &wk, &table});
  need(onOneDevice(qkv, {&wq, &wk, &table}), "tensors on one CUDA device expected");
  variable_list r;
  if (at::GradMode::is_enabled() && (qkv.requires_grad() || wq.requires_grad() || wk.requires_grad()))
    r = QkNormRope::apply(qkv, wq, wk, table, heads, kv, eps);
  else
    r = normForward(rows16(qkv).contiguous(), wq.contiguous(), wk.contiguous(), table, heads, kv, eps);
  return {r[0], r[1], r[2]};
}

// ---- attention with a window and sinks -------------------------------------------------------------------------
struct Numbers {
  int64_t window, sinks;
  double scale;
};

Tensor attend(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& lengths, const Numbers& n, const Tensor& lse, const Tensor& rest) {
  const int64_t B = q.size(0), H = q.size(1), S = q.size(2), D = q.size(3);
  const Tensor o = byToken(B, H, S, D, q);
  const auto st = strides<4>({&q, &k, &v, &o});
  check(b200ops_window_attention_fwd(ptr(q), ptr(k), ptr(v), out(o), lse.defined() ? (float*)out(lse) : nullptr, rest.defined() ? out(rest) : nullptr,
                                     lengths.defined() ? (const int*)ptr(lengths) : nullptr, st.data(), (int)B, (int)H, (int)k.size(1), (int)S, (int)D, (int)n.window,
                                     (int)n.sinks, (float)n.scale, stream()),
        "window_attention_fwd", 1);
  return o;
}

struct WindowAttention : torch::autograd::Function<WindowAttention> {
  static Tensor forward(AutogradContext* ctx, const Tensor& qIn, const Tensor& kIn, const Tensor& vIn, const std::optional<Tensor>& lengthsIn, int64_t window, int64_t sinks,
                        double scale) {
    c10::cuda::OptionalCUDAGuard guard(qIn.device());
    const Tensor q = rows16(qIn), k = rows16(kIn), v = rows16(vIn), lengths = lengthsIn.value_or(Tensor());
    const int64_t B = q.size(0), H = q.size(1), S = q.size(2), D = q.size(3);
    const Tensor lse = at::empty({B, H, (S + 127) / 128 * 128}, q.options().dtype(at::kFloat));
    const Tensor rest = at::empty({B, S, H, D}, q.options());  // what rounding took from the answer
    const Tensor o = attend(q, k, v, lengths, {window, sinks, scale}, lse, rest);
    variable_list kept{q, k, v, o, rest, lse};
    if (lengths.defined()) kept.push_back(lengths);
    ctx->save_for_backward(kept);
    ctx->saved_data["window"] = window;
    ctx->saved_data["sinks"] = sinks;
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["kv"] = k.size(1);
    return o;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once();
    const auto saved = ctx->get_saved_variables();
    const int B = (int)grads[0].size(0), H = (int)grads[0].size(1), KV = (int)ctx->saved_data["kv"].toInt(), S = (int)grads[0].size(2), D = (int)grads[0].size(3);
    for (int i = 0; i < 4; i++) cameBack(saved[i], {B, i == 1 || i == 2 ? KV : H, S, D}, at::kBFloat16, grads[0]);
    cameBack(saved[4], {B, S, H, D}, at::kBFloat16, grads[0]);
    cameBack(saved[5], {B, H, (S + 127) / 128 * 128}, at::kFloat, grads[0]);
    if (saved.size() > 6) cameBack(saved[6], {B}, at::kInt, grads[0]);
    const int window = (int)ctx->saved_data["window"].toInt(), sinks = (int)ctx->saved_data["sinks"].toInt();
    c10::cuda::OptionalCUDAGuard guard(grads[0].device());
    const Tensor q = rows16(saved[0]), k = rows16(saved[1]), v = rows16(saved[2]), o = rows16(saved[3]), rest = dense16(saved[4]), lse = dense16(saved[5]);
    const Tensor lengths = saved.size() > 6 ? saved[6].contiguous() : Tensor(), g = rows16(grads[0]);
    const Tensor dq = byToken(B, H, S, D, q), dk = byToken(B, KV, S, D, q), dv = byToken(B, KV, S, D, q);
    const Tensor scratch = at::empty({(int64_t)b200ops_window_attention_bwd_scratch(B, H, KV, S, D, window, sinks)}, lse.options());
    const auto st = strides<8>({&q, &k, &v, &o, &g, &dq, &dk, &dv});
    check(b200ops_window_attention_bwd(ptr(q), ptr(k), ptr(v), ptr(o), ptr(rest), ptr(g), (const float*)ptr(lse), (float*)out(scratch), out(dq), out(dk), out(dv),
                                       lengths.defined() ? (const int*)ptr(lengths) : nullptr, st.data(), B, H, KV, S, D, window, sinks,
                                       (float)ctx->saved_data["scale"].toDouble(), stream()),
          "window_attention_bwd", b200ops_window_attention_bwd_launches(B, H, KV, S, D, window, sinks));
    return {dq, dk, dv, Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor windowAttention(const Tensor& q, const Tensor& k, const Tensor& v, int64_t window, int64_t sinks, const std::optional<Tensor>& lengthsIn, std::optional<double> scaleIn) {
  need(q.dim() == 4 && k.dim() == 4 && k.sizes() == v.sizes(), "q [B, H, S, D], k and v [B, KV, S, D]");
  const int64_t B = q.size(0), H = q.size(1), S = q.size(2), D = q.size(3);
  need(k.size(0) == B && k.size(2) == S && k.size(3) == D, "q, k and v: the same batch, length and head dimension");
  need(q.numel() > 0 && k.size(1) > 0 && H % k.size(1) == 0, "query heads: a multiple of the key heads, nothing empty");
  need(D % 8 == 0 && D <= 128, "head dimension: a multiple of 8 up to 128");
  need(q.scalar_type() == at::kBFloat16 && k.scalar_type() == at::kBFloat16 && v.scalar_type() == at::kBFloat16, "bf16 tensors expected");
  need(window >= 0 && sinks >= 0, "window and sinks: not negative");
  need(!scaleIn || (*scaleIn >= 0 && std::isfinite(*scaleIn)), "scale: finite, not negative");
  need(!lengthsIn || (lengthsIn->dim() == 1 && lengthsIn->size(0) == B && lengthsIn->scalar_type() == at::kInt && lengthsIn->is_contiguous()),
       "lengths: contiguous int32 [B]");
  need(S < (1LL << 30) && B * k.size(1) < (1LL << 16) && B * H * ((S + 127) / 128) < (1LL << 31), "too many positions, heads or sequences");
  noTangent({&q, &k, &v});
  const Tensor lengths = lengthsIn.value_or(Tensor());
  need(onOneDevice(q, {&k, &v}) && (!lengths.defined() || lengths.device() == q.device()), "tensors on one CUDA device expected");
  const Numbers n{std::min(window, S), std::min(sinks, S), scaleIn ? *scaleIn : 1.0 / std::sqrt((double)D)};
  if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad()))
    return WindowAttention::apply(q, k, v, lengthsIn, n.window, n.sinks, n.scale);
  c10::cuda::OptionalCUDAGuard guard(q.device());
  return attend(rows16(q), rows16(k), rows16(v), lengths, n, Tensor(), Tensor());
}

// ---- distillation ------------------------------------------------------------------------------------------------
std::tuple<Tensor, Tensor> distillLoss(const Tensor& logits, const Tensor& targets, const Tensor& teacherIds, const Tensor& teacherLogits, double weight, double temperature,
                                       double gradScale, const std::optional<Tensor>& gradIn) {
  need(logits.dim() == 2 && logits.scalar_type() == at::kBFloat16 && (logits.stride(1) == 1 || logits.size(1) == 1), "logits: [T, V] in bf16 with dense rows");
  const int64_t T = logits.size(0), V = logits.size(1);
  need(V > 0 && (logits.stride(0) >= V || T <= 1), "logits: rows that do not overlap");
  need(targets.dim() == 1 && targets.size(0) == T && targets.scalar_type() == at::kLong && targets.is_contiguous(), "targets: contiguous int64 [T]");
  need(teacherIds.dim() == 2 && teacherIds.sizes() == teacherLogits.sizes() && teacherIds.size(0) == T, "teacher_ids and teacher_logits: [T, K]");
  const int64_t K = teacherIds.size(1);
  need(V <= 851968, "a vocabulary of up to 851,968");
  need(K >= 1 && K <= 1024, "1 to 1024 teacher entries per row");
  const auto it = teacherIds.scalar_type(), vt = teacherLogits.scalar_type();
  need((it == at::kLong || it == at::kInt) && (vt == at::kFloat || vt == at::kBFloat16), "int64 or int32 ids, fp32 or bf16 logits");
  need(weight >= 0 && weight <= 1 && temperature >= 0.01 && temperature <= 100 && std::isfinite(gradScale), "0 <= weight <= 1, temperature from 0.01 to 100");
  need(T < (1LL << 28), "too many rows");
  if (gradIn) {
    const Tensor& g = *gradIn;
    need(g.dim() == 2 && g.size(0) == T && g.size(1) == V && g.scalar_type() == at::kBFloat16 && (g.stride(1) == 1 || V == 1) && (g.stride(0) >= V || T <= 1),
         "grad: like logits");
    const auto from = [&](const Tensor& t) { return reinterpret_cast<uintptr_t>(ptr(t)); };
    const auto to = [&](const Tensor& t) { return from(t) + 2 * ((T - 1) * t.stride(0) + V); };
    if (T > 0 && !(from(g) == from(logits) && (T == 1 || g.stride(0) == logits.stride(0))))
      need(to(g) <= from(logits) || to(logits) <= from(g), "grad: logits itself, or memory apart from it");
  }
  noTangent({&logits, &teacherLogits});
  need(onOneDevice(logits, {&targets, &teacherIds, &teacherLogits}) && (!gradIn || gradIn->device() == logits.device()), "tensors on one CUDA device expected");
  c10::cuda::OptionalCUDAGuard guard(logits.device());
  const Tensor grad = gradIn ? *gradIn : at::empty({T, V}, logits.options());
  const Tensor ids = teacherIds.contiguous(), values = teacherLogits.contiguous(), loss = at::empty({T}, logits.options().dtype(at::kFloat));
  check(b200ops_distill_loss(ptr(logits), out(grad), (const long long*)ptr(targets), ptr(ids), (int)ids.element_size(), ptr(values), (int)values.element_size(),
                             (float*)out(loss), T, (int)V, (int)K, std::max(logits.stride(0), V), std::max(grad.stride(0), V), (float)weight, (float)temperature,
                             (float)gradScale, stream()),
        "distill_loss", T > 0);
  if (gradIn && !grad.is_inference()) grad.unsafeGetTensorImpl()->bump_version();  // written through its pointer: a graph that saved it has to notice
  return {loss, grad};
}

}  // namespace

void bindStudentOps(py::module_& m) {
  m.def("qk_norm_rope", &qkNormRope);
  m.def("window_attention", &windowAttention);
  m.def("distill_loss", [](const Tensor& logits, const Tensor& targets, const Tensor& ids, const Tensor& values, double weight, double temperature, double gradScale,
                           const std::optional<py::object>& grad) -> py::tuple {
    std::optional<Tensor> g;
    if (grad) g = grad->cast<Tensor>();
    auto [loss, dz] = distillLoss(logits, targets, ids, values, weight, temperature, gradScale, g);
    return py::make_tuple(loss, grad ? *grad : py::cast(dz));
  });
  m.def("student_launches", [] { return gLaunches.load(); });
}
