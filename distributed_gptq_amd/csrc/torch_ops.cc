// gptq::linear_rows, the dequant-GEMV/GEMM entry point as a native torch
// operator: what a decode step calls once per layer, where a Python
// implementation (operator wrapper, argument checks, ctypes marshalling) took
// 25 us around kernels of 5-15 us.  The caller has resolved the layer's
// layout (code width, contiguous groups); autograd and layouts with a group
// index go through gptq::linear.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/autograd_not_implemented_fallback.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/library.h>

#include <limits>

#include "gptq_hip.h"

namespace {

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return GPTQ_F32;
    case at::kHalf: return GPTQ_F16;
    case at::kBFloat16: return GPTQ_BF16;
    default: TORCH_CHECK_TYPE(false, "unsupported dtype ", t, "; expected float32, float16 or bfloat16");
  }
}

// y = x @ dequant(W)^T (+ bias), x (..., K): as gptq_linear_ws, on x's current stream
at::Tensor linear_rows(const at::Tensor& x, const at::Tensor& qweight, const at::Tensor& scales,
                       const at::Tensor& zeros, const std::optional<at::Tensor>& bias,
                       const std::optional<at::Tensor>& perm, int64_t bits, int64_t group_size, int64_t K) {
  // what is refused is a ValueError or a TypeError, which the caller leaves to
  // gptq::linear; everything else is a failure
  TORCH_CHECK_VALUE(x.is_cuda() && qweight.device() == x.device() && scales.device() == x.device() &&
                        zeros.device() == x.device() && (!bias || bias->device() == x.device()) &&
                        (!perm || perm->device() == x.device()),
                    "gptq::linear_rows: expected GPU tensors on one device");
  TORCH_CHECK_VALUE(K > 0 && x.dim() > 0 && x.size(-1) == K && qweight.dim() == 2 && scales.dim() == 2 &&
                        zeros.sizes() == scales.sizes() && scales.size(0) == qweight.size(0) &&
                        qweight.scalar_type() == at::kByte && qweight.is_contiguous() &&
                        qweight.size(1) == (bits == 0 ? K : (K * bits + 7) / 8) &&
                        (!bias || bias->numel() == qweight.size(0)),
                    "gptq::linear_rows: the shapes of x and the weight do not match in_features = ", K);
  const c10::DeviceGuard guard(x.device());
  const int64_t N = qweight.size(0);
  const at::Tensor x2 = x.reshape({-1, K}).contiguous();
  const int64_t M = x2.size(0);
  const at::Tensor s = scales.contiguous(), z = zeros.to(scales.scalar_type()).contiguous();
  at::Tensor b, p;
  if (bias) b = bias->contiguous();
  if (perm) {
    TORCH_CHECK_VALUE(perm->numel() == K, "perm has ", perm->numel(), " entries, in_features is ", K);
    p = perm->to(at::kInt).contiguous();
  }
  const int xt = dtype_code(x2.scalar_type());
  std::vector<int64_t> shape = x.sizes().vec();
  shape.back() = N;
  at::Tensor y = at::empty(shape, x2.options());
  // exactly the requested size, so that the kernel choice depends on the
  // shapes only; from the caching allocator, ordered on this stream
  const size_t bytes = gptq_linear_workspace_size(M, N, K, static_cast<int>(bits), static_cast<int>(group_size), xt, perm ? 1 : 0);
  at::Tensor ws;
  if (bytes) ws = at::empty({static_cast<int64_t>(bytes)}, x2.options().dtype(at::kByte));
  const int rc = gptq_linear_ws(
      x2.const_data_ptr(), xt, M, perm ? p.const_data_ptr<int32_t>() : nullptr, qweight.const_data_ptr<uint8_t>(),
      static_cast<int>(bits), s.const_data_ptr(), z.const_data_ptr(), dtype_code(s.scalar_type()), nullptr,
      static_cast<int>(group_size), s.size(1), bias ? b.const_data_ptr() : nullptr,
      bias ? dtype_code(b.scalar_type()) : 0, N, K, y.mutable_data_ptr(), bytes ? ws.mutable_data_ptr() : nullptr, bytes,
      c10::hip::getCurrentHIPStream(x.device().index()).stream());
  TORCH_CHECK_VALUE(rc != GPTQ_ERR_ARG && rc != GPTQ_ERR_SHAPE, "gptq_linear_ws: ", gptq_last_error());
  TORCH_CHECK_TYPE(rc != GPTQ_ERR_DTYPE, "gptq_linear_ws: ", gptq_last_error());
  TORCH_CHECK(rc == GPTQ_OK, "gptq_linear_ws failed (status ", rc, "): ", gptq_last_error());
  return y;
}

// ------------------------------------------------------------- attention ----

#define GPTQ_CALL(name, ...)                                                                        \
  do {                                                                                              \
    const int rc = name(__VA_ARGS__);                                                               \
    TORCH_CHECK_VALUE(rc != GPTQ_ERR_ARG && rc != GPTQ_ERR_SHAPE, gptq_last_error());               \
    TORCH_CHECK_TYPE(rc != GPTQ_ERR_DTYPE, gptq_last_error());                                      \
    TORCH_CHECK(rc == GPTQ_OK, #name " failed (status ", rc, "): ", gptq_last_error());             \
  } while (0)

gptq_stream_t stream_of(const at::Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

// whether t has contiguous, 16-byte aligned rows of whole 8s of values, as the
// kernels read them
bool rows_aligned(const at::Tensor& t) {
  bool ok = t.stride(-1) == 1 && reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0;
  for (int64_t i = 0; i + 1 < t.dim(); ++i) ok = ok && (t.stride(i) % 8 == 0 || t.size(i) <= 1);
  return ok;
}
// t (tokens, heads, values) with such rows, tokens below 2^28 values apart:
// itself wherever it has them already (a part of a fused projection)
at::Tensor aligned_rows(const at::Tensor& t) {
  if (rows_aligned(t) && (t.size(0) <= 1 || t.stride(0) < (int64_t{1} << 28))) return t;
  const at::Tensor c = t.contiguous();
  return reinterpret_cast<uintptr_t>(c.const_data_ptr()) % 16 == 0 ? c : c.clone();
}
// (a dimension of one row may have any stride)
int64_t stride_of(const at::Tensor& t, int64_t dim) { return t.size(dim) <= 1 ? 0 : t.stride(dim); }

at::Tensor int32_of(const at::Tensor& t, const at::Tensor& like, const char* name) {
  TORCH_CHECK_VALUE(t.device() == like.device(), name, " is on ", t.device(), ", the queries are on ", like.device());
  TORCH_CHECK_TYPE(t.scalar_type() == at::kInt || t.scalar_type() == at::kLong, name, " has to be int32 or int64");
  if (t.scalar_type() == at::kInt) return t.contiguous();
  // what 32 bits do not hold stays out of every range that the kernels check
  return t.clamp(std::numeric_limits<int32_t>::min(), std::numeric_limits<int32_t>::max()).to(at::kInt).contiguous();
}

void check_heads(const char* fn, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, int64_t dim) {
  TORCH_CHECK_VALUE(q.is_cuda() && k.device() == q.device() && v.device() == q.device(), fn,
                    ": expected GPU tensors on one device");
  TORCH_CHECK_TYPE(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(), fn,
                   ": q, k and v have different types");
  TORCH_CHECK_VALUE(q.dim() == 3 && k.dim() == dim && v.sizes() == k.sizes() && k.size(-1) == q.size(-1), fn,
                    ": shapes ", q.sizes(), ", ", k.sizes(), " and ", v.sizes(), " do not match");
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> attention_run(const at::Tensor& q_, const at::Tensor& k_,
                                                             const at::Tensor& v_,
                                                             const std::optional<at::Tensor>& cu_q,
                                                             const std::optional<at::Tensor>& cu_k, bool causal,
                                                             double scale, bool train) {
  check_heads("gptq::attention", q_, k_, v_, 3);
  TORCH_CHECK_VALUE(cu_q || !cu_k, "gptq::attention: offsets of the keys without offsets of the queries");
  TORCH_CHECK_VALUE(!cu_q || (cu_q->dim() == 1 && cu_q->numel() >= 2), "gptq::attention: cu_seqlens has to hold B + 1 offsets");
  TORCH_CHECK_VALUE(!cu_k || cu_k->sizes() == cu_q->sizes(),
                    "gptq::attention: cu_seqlens and cu_seqlens_k have different lengths");
  TORCH_CHECK_VALUE(!cu_q || cu_k || k_.size(0) == q_.size(0), "gptq::attention: ", q_.size(0), " queries and ",
                    k_.size(0), " keys need offsets of their own");
  const c10::DeviceGuard guard(q_.device());
  const at::Tensor q = aligned_rows(q_), k = aligned_rows(k_), v = aligned_rows(v_);
  at::Tensor cq, ck;
  if (cu_q) cq = int32_of(*cu_q, q, "cu_seqlens");
  if (cu_k) ck = int32_of(*cu_k, q, "cu_seqlens_k");
  const int64_t T = q.size(0), H = q.size(1), D = q.size(2);
  at::Tensor out = at::empty({T, H, D}, q.options());
  at::Tensor rest, lse;
  if (train) rest = at::empty({T, H, D}, q.options()), lse = at::empty({T, H}, q.options().dtype(at::kFloat));
  const int32_t* pq = cu_q ? cq.const_data_ptr<int32_t>() : nullptr;
  GPTQ_CALL(gptq_attention, q.const_data_ptr(), k.const_data_ptr(), v.const_data_ptr(), dtype_code(q.scalar_type()),
            stride_of(q, 0), stride_of(q, 1), stride_of(k, 0), stride_of(k, 1), stride_of(v, 0), stride_of(v, 1), pq,
            cu_k ? ck.const_data_ptr<int32_t>() : pq, cu_q ? cq.numel() - 1 : 1, T, k.size(0), H, k.size(1), D, causal,
            static_cast<float>(scale), out.mutable_data_ptr(), train ? rest.mutable_data_ptr() : nullptr,
            train ? lse.mutable_data_ptr<float>() : nullptr, stream_of(q));
  return {out, rest, lse};
}

at::Tensor attention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                     const std::optional<at::Tensor>& cu_q, const std::optional<at::Tensor>& cu_k, bool causal,
                     double scale) {
  return std::get<0>(attention_run(q, k, v, cu_q, cu_k, causal, scale, false));
}

// (out, out_rest, lse): what the gradient needs too
std::tuple<at::Tensor, at::Tensor, at::Tensor> attention_forward(const at::Tensor& q, const at::Tensor& k,
                                                                 const at::Tensor& v,
                                                                 const std::optional<at::Tensor>& cu_q,
                                                                 const std::optional<at::Tensor>& cu_k, bool causal,
                                                                 double scale) {
  return attention_run(q, k, v, cu_q, cu_k, causal, scale, true);
}

// (dq, dk, dv) of attention_forward's output
std::tuple<at::Tensor, at::Tensor, at::Tensor> attention_backward(
    const at::Tensor& grad_, const at::Tensor& q_, const at::Tensor& k_, const at::Tensor& v_, const at::Tensor& out_,
    const at::Tensor& rest_, const at::Tensor& lse_, const std::optional<at::Tensor>& cu_q, const std::optional<at::Tensor>& cu_k, bool causal,
    double scale) {
  check_heads("gptq::attention_backward", q_, k_, v_, 3);
  TORCH_CHECK_VALUE(grad_.sizes() == q_.sizes() && out_.sizes() == q_.sizes() && rest_.sizes() == q_.sizes() && lse_.dim() == 2 &&
                        lse_.size(0) == q_.size(0) && lse_.size(1) == q_.size(1) && grad_.device() == q_.device() &&
                        out_.device() == q_.device() && rest_.device() == q_.device() && lse_.device() == q_.device(),
                    "gptq::attention_backward: the gradient, output or lse do not match the queries");
  TORCH_CHECK_TYPE(grad_.scalar_type() == q_.scalar_type() && out_.scalar_type() == q_.scalar_type() &&
                       rest_.scalar_type() == q_.scalar_type() &&
                       lse_.scalar_type() == at::kFloat,
                   "gptq::attention_backward: the gradient, output or lse have another type");
  TORCH_CHECK_VALUE((cu_q || !cu_k) && (!cu_q || (cu_q->dim() == 1 && cu_q->numel() >= 2)) &&
                        (!cu_k || cu_k->sizes() == cu_q->sizes()) && (!cu_q || cu_k || k_.size(0) == q_.size(0)),
                    "gptq::attention_backward: the offsets do not match");
  const c10::DeviceGuard guard(q_.device());
  const at::Tensor grad = aligned_rows(grad_), q = aligned_rows(q_), k = aligned_rows(k_), v = aligned_rows(v_);
  const at::Tensor out = aligned_rows(out_.contiguous()), rest = aligned_rows(rest_.contiguous()), lse = lse_.contiguous();
  at::Tensor cq, ck;
  if (cu_q) cq = int32_of(*cu_q, q, "cu_seqlens");
  if (cu_k) ck = int32_of(*cu_k, q, "cu_seqlens_k");
  const int64_t T = q.size(0), H = q.size(1), D = q.size(2);
  at::Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options()),
             dv = at::empty(v.sizes(), v.options());
  const size_t bytes = gptq_attention_backward_workspace_size(cu_q ? cq.numel() - 1 : 1, T, k.size(0), H, k.size(1), D);
  at::Tensor ws = at::empty({static_cast<int64_t>(bytes)}, q.options().dtype(at::kByte));
  const int32_t* pq = cu_q ? cq.const_data_ptr<int32_t>() : nullptr;
  GPTQ_CALL(gptq_attention_backward, grad.const_data_ptr(), q.const_data_ptr(), k.const_data_ptr(), v.const_data_ptr(),
            out.const_data_ptr(), rest.const_data_ptr(), lse.const_data_ptr<float>(), dtype_code(q.scalar_type()), stride_of(grad, 0),
            stride_of(grad, 1), stride_of(q, 0), stride_of(q, 1), stride_of(k, 0), stride_of(k, 1), stride_of(v, 0),
            stride_of(v, 1), pq, cu_k ? ck.const_data_ptr<int32_t>() : pq, cu_q ? cq.numel() - 1 : 1, T, k.size(0), H,
            k.size(1), D, causal, static_cast<float>(scale), dq.mutable_data_ptr(), dk.mutable_data_ptr(),
            dv.mutable_data_ptr(), ws.mutable_data_ptr(), bytes, stream_of(q));
  return {dq, dk, dv};
}

at::Tensor paged_attention(const at::Tensor& q_, const at::Tensor& k_cache, const at::Tensor& v_cache,
                           const at::Tensor& block_table, const at::Tensor& context,
                           const std::optional<at::Tensor>& cu_q, double scale, int64_t max_context) {
  check_heads("gptq::paged_attention", q_, k_cache, v_cache, 4);
  TORCH_CHECK_VALUE(block_table.dim() == 2 && context.dim() == 1 && block_table.size(0) == context.size(0),
                    "gptq::paged_attention: a block table ", block_table.sizes(), " for ", context.sizes(), " contexts");
  const int64_t B = context.size(0), T = q_.size(0), H = q_.size(1), D = q_.size(2);
  TORCH_CHECK_VALUE(cu_q ? cu_q->dim() == 1 && cu_q->numel() == B + 1 : T == B, "gptq::paged_attention: ", T,
                    " new tokens of ", B, " sequences ", cu_q ? "need B + 1 offsets" : "without their offsets");
  const c10::DeviceGuard guard(q_.device());
  const at::Tensor q = aligned_rows(q_);
  // (a cache is never copied)
  TORCH_CHECK_VALUE(rows_aligned(k_cache) && rows_aligned(v_cache),
                    "gptq::paged_attention: the cache's heads have to be contiguous and 16-byte aligned");
  at::Tensor out = at::empty({T, H, D}, q.options());
  if (T == 0) return out;
  const at::Tensor table = int32_of(block_table, q, "block_table"), ctx = int32_of(context, q, "context_lens");
  at::Tensor cq;
  if (cu_q) cq = int32_of(*cu_q, q, "cu_seqlens");
  const int64_t Hk = k_cache.size(2);
  const size_t bytes = gptq_paged_attention_workspace_size(B, T, H, Hk, D, max_context);
  at::Tensor ws;
  if (bytes) ws = at::empty({static_cast<int64_t>(bytes)}, q.options().dtype(at::kByte));
  GPTQ_CALL(gptq_paged_attention, q.const_data_ptr(), k_cache.const_data_ptr(), v_cache.const_data_ptr(),
            dtype_code(q.scalar_type()), stride_of(q, 0), stride_of(q, 1), stride_of(k_cache, 0), stride_of(k_cache, 1),
            stride_of(k_cache, 2), stride_of(v_cache, 0), stride_of(v_cache, 1), stride_of(v_cache, 2),
            table.const_data_ptr<int32_t>(), table.size(1), table.size(1), k_cache.size(1), k_cache.size(0),
            ctx.const_data_ptr<int32_t>(), cu_q ? cq.const_data_ptr<int32_t>() : nullptr, B, T, H, Hk, D,
            static_cast<float>(scale), max_context, out.mutable_data_ptr(), bytes ? ws.mutable_data_ptr() : nullptr, bytes,
            stream_of(q));
  return out;
}

// ---------------------------------------------------------------- rotary ----

void check_table(const char* fn, const at::Tensor& q, const std::optional<at::Tensor>& table,
                 const std::optional<at::Tensor>& positions) {
  if (!table) return;
  TORCH_CHECK_TYPE(table->scalar_type() == at::kFloat, fn, ": the table has to be float32");
  TORCH_CHECK_VALUE(table->device() == q.device() && table->dim() == 3 && table->size(1) == 2 && table->size(0) >= 1 &&
                        2 * table->size(2) <= q.size(-1) && table->size(2) >= 1,
                    fn, ": a table ", table->sizes(), " does not hold (positions, 2, half the rotated channels) for heads of ",
                    q.size(-1));
  TORCH_CHECK_VALUE(positions && positions->dim() == 1 && positions->size(0) == q.size(0), fn,
                    ": one position a token is needed");
}

at::Tensor last_contiguous(const at::Tensor& t) { return t.stride(-1) == 1 ? t : t.contiguous(); }

// q and k turned by their positions' angles, or back
std::tuple<at::Tensor, at::Tensor> rotary(const at::Tensor& q_, const at::Tensor& k_, const at::Tensor& table_,
                                          const at::Tensor& positions_, bool interleaved, bool inverse) {
  check_heads("gptq::rotary", q_, k_, k_, 3);
  TORCH_CHECK_VALUE(k_.size(0) == q_.size(0), "gptq::rotary: ", q_.size(0), " queries and ", k_.size(0), " keys");
  check_table("gptq::rotary", q_, table_, positions_);
  const c10::DeviceGuard guard(q_.device());
  const at::Tensor q = last_contiguous(q_), k = last_contiguous(k_), table = table_.contiguous();
  const at::Tensor positions = int32_of(positions_, q, "positions");
  at::Tensor qo = at::empty(q.sizes(), q.options()), ko = at::empty(k.sizes(), k.options());
  GPTQ_CALL(gptq_rotary, q.const_data_ptr(), k.const_data_ptr(), dtype_code(q.scalar_type()), stride_of(q, 0),
            stride_of(q, 1), stride_of(k, 0), stride_of(k, 1), table.const_data_ptr<float>(), table.size(0),
            2 * table.size(2), positions.const_data_ptr<int32_t>(), interleaved, inverse, q.size(0), q.size(1), k.size(1),
            q.size(2), qo.mutable_data_ptr(), ko.mutable_data_ptr(), stream_of(q));
  return {qo, ko};
}

// the queries turned, the keys (turned) and values written into their slots
at::Tensor rotary_append(const at::Tensor& q_, const at::Tensor& k_, const at::Tensor& v_,
                         const std::optional<at::Tensor>& table_, const std::optional<at::Tensor>& positions_,
                         at::Tensor k_cache, at::Tensor v_cache, const at::Tensor& slots_, bool interleaved) {
  check_heads("gptq::rotary_append", q_, k_, v_, 3);
  check_heads("gptq::rotary_append", q_, k_cache, v_cache, 4);
  TORCH_CHECK_VALUE(k_.size(0) == q_.size(0) && k_cache.size(2) == k_.size(1) && slots_.dim() == 1 &&
                        slots_.size(0) == q_.size(0),
                    "gptq::rotary_append: queries ", q_.sizes(), ", keys ", k_.sizes(), ", slots ", slots_.sizes(),
                    " and a cache ", k_cache.sizes(), " do not match");
  TORCH_CHECK_VALUE(k_cache.stride(-1) == 1 && v_cache.stride(-1) == 1,
                    "gptq::rotary_append: the cache's heads have to be contiguous");
  check_table("gptq::rotary_append", q_, table_, positions_);
  const c10::DeviceGuard guard(q_.device());
  const at::Tensor q = last_contiguous(q_), k = last_contiguous(k_), v = last_contiguous(v_);
  at::Tensor table, positions;
  if (table_) table = table_->contiguous(), positions = int32_of(*positions_, q, "positions");
  const at::Tensor slots = int32_of(slots_, q, "slots");
  at::Tensor qo = at::empty(q.sizes(), q.options());
  if (k_cache.numel() == 0) TORCH_CHECK_VALUE(k.numel() == 0, "gptq::rotary_append: the cache has no pages");
  GPTQ_CALL(gptq_rotary_append, q.const_data_ptr(), k.const_data_ptr(), v.const_data_ptr(), dtype_code(q.scalar_type()),
            stride_of(q, 0), stride_of(q, 1), stride_of(k, 0), stride_of(k, 1), stride_of(v, 0), stride_of(v, 1),
            table_ ? table.const_data_ptr<float>() : nullptr, table_ ? table.size(0) : 0, table_ ? 2 * table.size(2) : 0,
            table_ ? positions.const_data_ptr<int32_t>() : nullptr, interleaved, slots.const_data_ptr<int32_t>(),
            k_cache.size(1), k_cache.size(0), q.size(0), q.size(1), k.size(1), q.size(2), qo.mutable_data_ptr(),
            k_cache.mutable_data_ptr(), stride_of(k_cache, 0), stride_of(k_cache, 1), stride_of(k_cache, 2),
            v_cache.mutable_data_ptr(), stride_of(v_cache, 0), stride_of(v_cache, 1), stride_of(v_cache, 2), stream_of(q));
  return qo;
}

// -------------------------------------------------------------- gradients ----

template <class F>
c10::TypedOperatorHandle<F> typed_op(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}

bool follows(std::initializer_list<const at::Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const at::Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// A tangent of forward-mode differentiation would be lost below autograd.
void no_tangents(const char* name, std::initializer_list<const at::Tensor*> ts) {
  for (const at::Tensor* t : ts)
    TORCH_CHECK(!t->defined() || !t->_fw_grad(0).defined(), name, " has no forward-mode derivative");
}

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// gradients that are differentiated again raise: these have no second derivative
variable_list once(variable_list grads, std::initializer_list<const at::Tensor*> of, const char* name) {
  if (!follows(of)) return grads;
  for (at::Tensor& g : grads) g = g.detach().set_requires_grad(true);
  auto error = std::make_shared<torch::autograd::DelayedError>(std::string(name) + " can be differentiated once only",
                                                               static_cast<int64_t>(grads.size()));
  return (*error)(std::move(grads));
}

at::Tensor or_none(const std::optional<at::Tensor>& t) { return t ? *t : at::Tensor(); }
std::optional<at::Tensor> or_null(const at::Tensor& t) {
  return t.defined() ? std::optional<at::Tensor>(t) : std::nullopt;
}

struct AttentionGrad : torch::autograd::Function<AttentionGrad> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                            const std::optional<at::Tensor>& cu_q, const std::optional<at::Tensor>& cu_k, bool causal,
                            double scale) {
    static const auto op = typed_op<decltype(attention_forward)>("gptq::attention_forward");
    at::AutoDispatchBelowADInplaceOrView below;
    auto [out, rest, lse] = op.call(q, k, v, cu_q, cu_k, causal, scale);
    ctx->save_for_backward({q, k, v, out, rest, lse, or_none(cu_q), or_none(cu_k)});
    ctx->saved_data["causal"] = causal;
    ctx->saved_data["scale"] = scale;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    static const auto op = typed_op<decltype(attention_backward)>("gptq::attention_backward");
    const auto s = ctx->get_saved_variables();
    no_tangents("gptq::attention", {&grads[0], &s[0], &s[1], &s[2]});
    at::Tensor dq, dk, dv;
    {
      at::AutoDispatchBelowADInplaceOrView below;
      std::tie(dq, dk, dv) = op.call(grads[0], s[0], s[1], s[2], s[3], s[4], s[5], or_null(s[6]), or_null(s[7]),
                                     ctx->saved_data["causal"].toBool(), ctx->saved_data["scale"].toDouble());
    }
    variable_list got = once({dq, dk, dv}, {&grads[0], &s[0], &s[1], &s[2]}, "gptq::attention");
    return {got[0], got[1], got[2], at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

at::Tensor attention_autograd(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                              const std::optional<at::Tensor>& cu_q, const std::optional<at::Tensor>& cu_k, bool causal,
                              double scale) {
  no_tangents("gptq::attention", {&q, &k, &v});
  if (follows({&q, &k, &v})) return AttentionGrad::apply(q, k, v, cu_q, cu_k, causal, scale);
  static const auto op = typed_op<decltype(attention)>("gptq::attention");
  at::AutoDispatchBelowADInplaceOrView below;
  return op.call(q, k, v, cu_q, cu_k, causal, scale);
}

struct RotaryGrad : torch::autograd::Function<RotaryGrad> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k, const at::Tensor& table,
                               const at::Tensor& positions, bool interleaved, bool inverse) {
    static const auto op = typed_op<decltype(rotary)>("gptq::rotary");
    at::AutoDispatchBelowADInplaceOrView below;
    auto [qo, ko] = op.call(q, k, table, positions, interleaved, inverse);
    ctx->save_for_backward({table, positions});
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["inverse"] = inverse;
    return {qo, ko};
  }
  // a rotation's transpose turns back (a table's factor stays in both)
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    static const auto op = typed_op<decltype(rotary)>("gptq::rotary");
    const auto s = ctx->get_saved_variables();
    auto [dq, dk] = op.call(grads[0], grads[1], s[0], s[1], ctx->saved_data["interleaved"].toBool(),
                            !ctx->saved_data["inverse"].toBool());
    return {dq, dk, at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

std::tuple<at::Tensor, at::Tensor> rotary_autograd(const at::Tensor& q, const at::Tensor& k, const at::Tensor& table,
                                                   const at::Tensor& positions, bool interleaved, bool inverse) {
  no_tangents("gptq::rotary", {&q, &k, &table});
  TORCH_CHECK(!follows({&table}), "gptq::rotary: the table gets no gradient: detach it");
  if (follows({&q, &k})) {
    const variable_list out = RotaryGrad::apply(q, k, table, positions, interleaved, inverse);
    return {out[0], out[1]};
  }
  static const auto op = typed_op<decltype(rotary)>("gptq::rotary");
  at::AutoDispatchBelowADInplaceOrView below;
  return op.call(q, k, table, positions, interleaved, inverse);
}

// Serving's operators have no gradient at all.
void no_gradient(const char* name, std::initializer_list<const at::Tensor*> ts) {
  no_tangents(name, ts);
  TORCH_CHECK(!follows(ts), name, " records no gradient: call it under torch.no_grad()");
}

at::Tensor rotary_append_autograd(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                  const std::optional<at::Tensor>& table, const std::optional<at::Tensor>& positions,
                                  at::Tensor k_cache, at::Tensor v_cache, const at::Tensor& slots, bool interleaved) {
  const at::Tensor angles = or_none(table);
  no_gradient("gptq::rotary_append", {&q, &k, &v, &angles, &k_cache, &v_cache});
  static const auto op = typed_op<decltype(rotary_append)>("gptq::rotary_append");
  at::AutoDispatchBelowADInplaceOrView below;
  return op.call(q, k, v, table, positions, std::move(k_cache), std::move(v_cache), slots, interleaved);
}

at::Tensor paged_attention_autograd(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache,
                                    const at::Tensor& block_table, const at::Tensor& context,
                                    const std::optional<at::Tensor>& cu_q, double scale, int64_t max_context) {
  no_gradient("gptq::paged_attention", {&q, &k_cache, &v_cache});
  static const auto op = typed_op<decltype(paged_attention)>("gptq::paged_attention");
  at::AutoDispatchBelowADInplaceOrView below;
  return op.call(q, k_cache, v_cache, block_table, context, cu_q, scale, max_context);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(gptq, m) {
  m.def("linear_rows(Tensor x, Tensor qweight, Tensor scales, Tensor zeros, Tensor? bias, Tensor? perm, int bits, "
        "int group_size, int in_features) -> Tensor");
  m.def("attention(Tensor q, Tensor k, Tensor v, Tensor? cu_seqlens, Tensor? cu_seqlens_k, bool causal, float scale) "
        "-> Tensor");
  m.def("attention_forward(Tensor q, Tensor k, Tensor v, Tensor? cu_seqlens, Tensor? cu_seqlens_k, bool causal, "
        "float scale) -> (Tensor, Tensor, Tensor)");
  m.def("attention_backward(Tensor grad, Tensor q, Tensor k, Tensor v, Tensor out, Tensor out_rest, Tensor lse, "
        "Tensor? cu_seqlens, Tensor? cu_seqlens_k, bool causal, float scale) -> (Tensor, Tensor, Tensor)");
  m.def("rotary(Tensor q, Tensor k, Tensor table, Tensor positions, bool interleaved, bool inverse) "
        "-> (Tensor, Tensor)");
  m.def("rotary_append(Tensor q, Tensor k, Tensor v, Tensor? table, Tensor? positions, Tensor(a!) k_cache, "
        "Tensor(b!) v_cache, Tensor slots, bool interleaved) -> Tensor");
  m.def("paged_attention(Tensor q, Tensor k_cache, Tensor v_cache, Tensor block_table, Tensor context_lens, "
        "Tensor? cu_seqlens, float scale, int max_context) -> Tensor");
}

TORCH_LIBRARY_IMPL(gptq, CUDA, m) {
  m.impl("linear_rows", linear_rows);
  m.impl("attention", attention);
  m.impl("attention_forward", attention_forward);
  m.impl("attention_backward", attention_backward);
  m.impl("paged_attention", paged_attention);
  m.impl("rotary", rotary);
  m.impl("rotary_append", rotary_append);
}

TORCH_LIBRARY_IMPL(gptq, Autograd, m) {
  m.impl("attention", attention_autograd);
  m.impl("rotary", rotary_autograd);
  m.impl("rotary_append", rotary_append_autograd);
  m.impl("paged_attention", paged_attention_autograd);
  // (parts of attention's own derivative)
  m.impl("attention_forward", torch::autograd::autogradNotImplementedFallback());
  m.impl("attention_backward", torch::autograd::autogradNotImplementedFallback());
}
