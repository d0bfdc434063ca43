// The package's per-layer calls for torch tensors, as one native call each:
// argument checks, output and workspace allocation, the C ABI call and the
// autograd node. The Python forms spend 20-50 us of interpreter time on each,
// more than the kernels take at small sizes. Forward and backward together,
// Python form -> native: norm + RoPE staging 152-190 -> 90 us (5120 rows, kernels
// 46 us), fp32 attention with its cache update 213 -> 103 us (320 queries),
// soft cross-entropy of 52 rows 117 -> 55 us, a 1387-row gated LoRA layer
// 176 -> 157 us, a chunk's cache bookkeeping 309 -> 270 us.
//
// Every entry returns None when the call is not of its plain form (a tensor
// that is not a dense GPU tensor, strides or types that need a copy or an error
// message, functorch transforms, forward-mode tangents, dispatch modes,
// tracing): the caller then takes the Python form, which handles or refuses it.
// Nothing has been launched or changed in that case. Apart from what the graph
// saves for a backward, nothing is kept from one call to the next.
//
// The C ABI is reached through function pointers that bind() receives, so both
// forms use the one library that the package has loaded; its errors are raised
// by the package's own Python function, with the same exception types.
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include "../../include/mtp_glora_amd.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;

#define MGA_API(X)                                                                                    \
  X(mga_header_hash) X(mga_kv_append) X(mga_attn_workspace_bytes) X(mga_attn_fwd_ws) X(mga_attn_bwd_ws) \
  X(mga_qk_norm_rope_stage_fwd) X(mga_qk_norm_rope_bwd) X(mga_gated_lora_workspace_bytes)             \
  X(mga_gated_lora_fwd) X(mga_gated_lora_bwd) X(mga_soft_ce_workspace_floats) X(mga_soft_ce_loss)     \
  X(mga_soft_ce_bwd) X(mga_top_logits) X(mga_top_logits_ce_workspace_floats) X(mga_top_logits_ce_fwd)  \
  X(mga_top_logits_ce_bwd) X(mga_top_logits_ce_step_workspace_floats) X(mga_top_logits_ce_step)          \
  X(mga_sample) X(mga_embedding_fwd) X(mga_embedding_workspace_bytes) X(mga_embedding_bwd) \
  X(mga_paged_append) X(mga_paged_attn_workspace_bytes) X(mga_paged_attn) \
  X(mga_adjust_logits)
struct Api {
#define X(f) decltype(&::f) f = nullptr;
  MGA_API(X)
#undef X
} g;

PyObject *g_raise = nullptr;   // raise(function name, code): owned for the life of the process

void bind_api(const std::map<std::string, int64_t> &addr, const py::object &raise) {
  // argument lists are compiled in: a library of another header must not be called
  const auto at = addr.find("mga_header_hash");
  if (at == addr.end() || reinterpret_cast<decltype(&::mga_header_hash)>(at->second)() != MGA_HEADER_HASH)
    throw std::runtime_error("_mga_torch.so and libmtp_glora_amd.so were built from different headers: build both "
                             "with `python __graft_entry__.py`");
#define X(f) g.f = reinterpret_cast<decltype(&::f)>(addr.at(#f));
  MGA_API(X)
#undef X
  Py_XDECREF(g_raise);
  g_raise = raise.inc_ref().ptr();
}

void check_rc(const char *fn, int rc) {
  if (rc == MGA_OK) return;
  py::gil_scoped_acquire gil;
  Py_XDECREF(PyObject_CallFunction(g_raise, "si", fn, rc));
  python_error e;
  e.persist();
  throw e;
}

// No transform, mode or trace is watching the calls.
bool eager() {
  return !c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerFrontMode) &&
         !c10::impl::TorchDispatchModeTLS::any_modes_set() && !torch::jit::tracer::isTracing();
}

bool plain(const Tensor &t) {
  static const c10::DispatchKeySet wrapped{c10::DispatchKey::Python,        c10::DispatchKey::FuncTorchBatched,
                                           c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::Functionalize,
                                           c10::DispatchKey::Conjugate,     c10::DispatchKey::Negative,
                                           c10::DispatchKey::ZeroTensor};
  return t.defined() && t.is_cuda() && t.layout() == at::kStrided && !t.key_set().has_any(wrapped) &&
         !t._fw_grad(0).defined();
}

int dtype_code(at::ScalarType t) {
  return t == at::kBFloat16 ? MGA_DTYPE_BF16 : t == at::kHalf ? MGA_DTYPE_F16 : t == at::kFloat ? MGA_DTYPE_F32 : -1;
}

bool same(const Tensor &a, const Tensor &b) { return a.scalar_type() == b.scalar_type() && a.device() == b.device(); }

void *stream(const Tensor &t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

bool aligned16(const Tensor &t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

// A captured backward joins the stream of the leaf's gradient accumulator. An eager
// graph that still lives has bound it to the default stream, which no capture may
// touch: torch's engine then ends the process. Refused while it can be said.
void check_capture(const std::string &fn, const Tensor &leaf) {
  if (!leaf.is_cuda() || !at::GradMode::is_enabled() || !leaf.requires_grad() || !leaf.is_leaf()) return;
  const at::DeviceGuard guard(leaf.device());
  if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
  const auto node = torch::autograd::impl::try_get_grad_accumulator(leaf);
  const auto stream = node ? node->stream() : std::nullopt;
  TORCH_CHECK(!stream || stream->id() != 0, fn, ": under graph capture, while an eager graph of the same leaf lives on "
              "the default stream; release that graph first");
}

// A gradient that is asked for with a graph of its own: differentiating it again is
// refused where that happens, since the backward leaves no graph.
Tensor once(const std::string &fn, const Tensor &g) {
  if (!at::GradMode::is_enabled()) return g;
  const auto refuse = std::make_shared<torch::autograd::DelayedError>(fn + ": no second derivatives", 1);
  return (*refuse)({g.detach().set_requires_grad(true)})[0];
}

// [1, H, S, D] with unit stride on D and 16-byte aligned rows
bool rows4(const Tensor &t) {
  const int64_t eb = t.element_size();
  return t.dim() == 4 && t.size(0) == 1 && t.stride(3) == 1 && t.stride(1) * eb % 16 == 0 && t.stride(2) * eb % 16 == 0 &&
         t.stride(1) >= 0 && t.stride(2) > 0 && t.stride(2) < (int64_t(1) << 23) && t.numel() > 0 && aligned16(t);
}

bool int32_on(const Tensor &t, const Tensor &like) {
  return plain(t) && t.scalar_type() == at::kInt && t.is_contiguous() && t.device() == like.device();
}

Tensor bytes(int64_t n, const Tensor &like) { return at::empty({n}, like.options().dtype(at::kByte)); }

// ---- cache rows --------------------------------------------------------------

bool kv_append(const Tensor &sk, const Tensor &sv, const Tensor &dk, const Tensor &dv, int64_t off,
               const std::optional<Tensor> &idx, std::optional<int64_t> n_rows) {
  if (!eager() || !plain(sk) || !plain(sv) || !plain(dk) || !plain(dv) || !rows4(sk) || !rows4(sv)) return false;
  if (!same(sk, sv) || !same(sk, dk) || !same(sk, dv) || sk.sizes() != sv.sizes() || sk.strides() != sv.strides())
    return false;
  if (dk.dim() != 3 || dk.sizes() != dv.sizes() || dk.strides() != dv.strides() || dk.stride(2) != 1 ||
      dk.size(0) != sk.size(1) || dk.size(2) != sk.size(3) || dtype_code(sk.scalar_type()) < 0)
    return false;
  if (idx && !int32_on(*idx, sk)) return false;
  const int64_t rows = n_rows ? *n_rows : idx ? idx->numel() : sk.size(2);
  if (rows < 0 || off < 0 || off + rows > dk.size(1) || (!idx && rows > sk.size(2))) return false;
  const at::DeviceGuard guard(sk.device());
  return g.mga_kv_append(sk.data_ptr(), sv.data_ptr(), sk.stride(1), sk.stride(2), sk.size(2),
                         idx ? idx->data_ptr<int32_t>() : nullptr, (int32_t)rows, dk.data_ptr(), dv.data_ptr(),
                         dk.stride(0), dk.stride(1), off, dk.size(1), (int32_t)dk.size(0), (int32_t)dk.size(2),
                         dtype_code(sk.scalar_type()), stream(sk)) == MGA_OK;
}

// Identity on the staged buffer view whose backward routes the rows of the
// chunk (the last ones) to the chunk's K or V and drops the detached prefix.
struct StageKV : public Function<StageKV> {
  static Tensor forward(AutogradContext *ctx, const Tensor &cur, const Tensor &full) {
    ctx->saved_data["P"] = full.size(2) - cur.size(2);
    return full.view_as(full);
  }
  static variable_list backward(AutogradContext *ctx, const variable_list &grad) {
    return {grad[0].slice(2, ctx->saved_data["P"].toInt()), Tensor()};
  }
};

bool at_row(const Tensor &t, const Tensor &buf, int64_t P) {
  return P < buf.size(1) && t.size(1) == buf.size(0) && t.stride(1) == buf.stride(0) && t.stride(2) == buf.stride(1) &&
         t.stride(3) == buf.stride(2) &&
         t.data_ptr() == static_cast<char *>(buf.data_ptr()) + P * buf.stride(1) * buf.element_size();
}

// The cache update's device side: the chunk's rows behind the prefix, unless
// they are there already (restage: the caller can write them again), and the
// views of prefix and chunk. (k, v, were there)
std::optional<std::tuple<Tensor, Tensor, bool>> update_kv(const Tensor &k, const Tensor &v, const Tensor &kb,
                                                          const Tensor &vb, int64_t P, bool restage) {
  if (!eager() || !plain(k) || !plain(v) || !plain(kb) || !plain(vb) || k.dim() != 4 || v.sizes() != k.sizes() ||
      !same(k, kb) || !same(v, vb) || kb.dim() != 3 || vb.sizes() != kb.sizes() ||
      kb.is_inference() || vb.is_inference())
    return std::nullopt;
  const bool in_place = at_row(k, kb, P);
  if (at_row(v, vb, P) != in_place || (in_place && !restage) ||
      (!in_place && !kv_append(k, v, kb, vb, P, std::nullopt, std::nullopt)))
    return std::nullopt;
  kb.unsafeGetTensorImpl()->bump_version();   // before the views: they record the version
  vb.unsafeGetTensorImpl()->bump_version();
  const int64_t L = P + k.size(2);
  Tensor kf = kb.unsqueeze(0).slice(2, 0, L), vf = vb.unsqueeze(0).slice(2, 0, L);
  if (k.requires_grad()) kf = StageKV::apply(k, kf);
  if (v.requires_grad()) vf = StageKV::apply(v, vf);
  return std::make_tuple(kf, vf, in_place);
}

// ---- attention ----------------------------------------------------------------

struct Mask {   // code, then the eight BlockMask tensors in the C ABI's order
  std::vector<Tensor> t;
  int64_t P;
  double scale;
  int64_t grad_start;
};

struct Attention : public Function<Attention> {
  // k_src, v_src receive the gradients of the rows from grad_start on
  static variable_list forward(AutogradContext *ctx, const Tensor &q, const Tensor &k_src, const Tensor &v_src,
                               const Tensor &k, const Tensor &v, const Mask &m) {
    const int64_t Hq = q.size(1), S = q.size(2), D = q.size(3), Hkv = k.size(1), L = k.size(2);
    const int dt = dtype_code(q.scalar_type());
    Tensor o = at::empty({1, S, Hq, D}, q.options().requires_grad(false));
    Tensor lse = at::empty({1, Hq, S}, q.options().requires_grad(false).dtype(at::kFloat));
    const int64_t wn = g.mga_attn_workspace_bytes((int32_t)S, (int32_t)L, (int32_t)Hq, (int32_t)Hkv, (int32_t)D, dt, 0, 0);
    Tensor ws;
    if (wn > 0) ws = bytes(wn, q);
    auto p = [&](int i) { return m.t[i].data_ptr<int32_t>(); };
    check_rc("mga_attn_fwd_ws",
             g.mga_attn_fwd_ws(q.data_ptr(), q.stride(1), q.stride(2), k.data_ptr(), k.stride(1), k.stride(2),
                               v.data_ptr(), v.stride(1), v.stride(2), o.data_ptr(), D, Hq * D, lse.data_ptr<float>(),
                               p(0), p(1), p(2), p(3), p(4), (int32_t)S, (int32_t)L, (int32_t)m.P, (int32_t)Hq,
                               (int32_t)Hkv, (int32_t)D, dt, (float)m.scale, wn > 0 ? ws.data_ptr() : nullptr, wn,
                               stream(q)));
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({q, k, v, o, lse});
    ctx->saved_data["mask"] = m.t;
    ctx->saved_data["P"] = m.P;
    ctx->saved_data["scale"] = m.scale;
    ctx->saved_data["grad_start"] = m.grad_start;
    return {o, lse};
  }

  static variable_list backward(AutogradContext *ctx, const variable_list &grad) {
    TORCH_CHECK_NOT_IMPLEMENTED(!grad[1].defined(),
                                "gradient through the attention LSE is not supported (the decoder layers discard it)");
    variable_list out(6);
    if (!grad[0].defined()) return out;
    const auto saved = ctx->get_saved_variables();
    const Tensor &q = saved[0], &k = saved[1], &v = saved[2], &o = saved[3], &lse = saved[4];
    const auto mask = ctx->saved_data["mask"].toTensorVector();
    const int64_t P = ctx->saved_data["P"].toInt();
    const double scale = ctx->saved_data["scale"].toDouble();
    const int64_t Hq = q.size(1), S = q.size(2), D = q.size(3), Hkv = k.size(1), L = k.size(2);
    const int dt = dtype_code(q.scalar_type());
    const at::DeviceGuard guard(q.device());
    const bool need_kv = ctx->needs_input_grad(1) || ctx->needs_input_grad(2);
    const int64_t gs = need_kv ? ctx->saved_data["grad_start"].toInt() : L, Lg = L - gs;
    Tensor d = grad[0];
    TORCH_CHECK(d.sizes() == o.sizes(), "grad_output shape ", d.sizes(), " != output shape ", o.sizes());
    if (d.scalar_type() != q.scalar_type()) d = d.to(q.scalar_type());
    const int64_t eb = d.element_size();
    // rows that the kernels do not read where they are: one row expanded, or rows too far apart
    if (d.stride(3) != 1 || d.stride(1) * eb % 16 || d.stride(2) * eb % 16 || d.stride(1) <= 0 ||
        d.stride(1) >= (int64_t(1) << 23) || !aligned16(d))
      d = d.clone(at::MemoryFormat::Contiguous);
    const auto opt = q.options().requires_grad(false);
    Tensor dq = at::empty({1, S, Hq, D}, opt), dk, dv;
    if (Lg > 0) {
      dk = at::empty({1, Lg, Hkv, D}, opt);
      dv = at::empty({1, Lg, Hkv, D}, opt);
    }
    Tensor delta = at::empty({MGA_BWD_WS_WORDS_PER_ROW * Hq * S}, opt.dtype(at::kFloat));
    const int64_t wn = g.mga_attn_workspace_bytes((int32_t)S, (int32_t)L, (int32_t)Hq, (int32_t)Hkv, (int32_t)D, dt, 1,
                                                  (int32_t)gs);
    Tensor ws;
    if (wn > 0) ws = bytes(wn, q);
    auto p = [&](int i) { return mask[i].data_ptr<int32_t>(); };
    check_rc("mga_attn_bwd_ws",
             g.mga_attn_bwd_ws(q.data_ptr(), q.stride(1), q.stride(2), k.data_ptr(), k.stride(1), k.stride(2),
                               v.data_ptr(), v.stride(1), v.stride(2), o.data_ptr(), o.stride(2), o.stride(1),
                               d.data_ptr(), d.stride(2), d.stride(1), lse.data_ptr<float>(), delta.data_ptr<float>(),
                               dq.data_ptr(), D, Hq * D, Lg > 0 ? dk.data_ptr() : nullptr, D, Hkv * D,
                               Lg > 0 ? dv.data_ptr() : nullptr, D, Hkv * D, (int32_t)gs, p(0), p(1), p(2), p(3), p(4),
                               p(5), p(6), p(7), p(8), (int32_t)S, (int32_t)L, (int32_t)P, (int32_t)Hq, (int32_t)Hkv,
                               (int32_t)D, dt, (float)scale, MGA_BWD_DQ | (need_kv ? MGA_BWD_DKDV : 0),
                               wn > 0 ? ws.data_ptr() : nullptr, wn, stream(q)));
    if (ctx->needs_input_grad(0)) out[0] = dq.transpose(1, 2);
    if (Lg > 0 && ctx->needs_input_grad(1)) out[1] = dk.transpose(1, 2);
    if (Lg > 0 && ctx->needs_input_grad(2)) out[2] = dv.transpose(1, 2);
    return out;
  }
};

// mask: code and the eight BlockMask tensors; (o [1, S, Hq, D], lse [1, Hq, S])
std::optional<std::tuple<Tensor, Tensor>> attention(const Tensor &q, const Tensor &k_src, const Tensor &v_src,
                                                    const Tensor &k, const Tensor &v, std::vector<Tensor> mask,
                                                    int64_t P, double scale, int64_t grad_start) {
  if (!eager() || !plain(q) || !plain(k_src) || !plain(v_src) || !plain(k) || !plain(v)) return std::nullopt;
  if (!rows4(q) || !rows4(k) || !rows4(v) || !same(q, k) || !same(q, v) || k.sizes() != v.sizes()) return std::nullopt;
  const int64_t D = q.size(3), Hkv = k.size(1);
  if (dtype_code(q.scalar_type()) < 0 || (D != 64 && D != 128) || k.size(3) != D || q.size(1) % Hkv ||
      k.size(2) != P + q.size(2) || P < 0 || !(scale > 0) || !std::isfinite((float)scale) || (float)scale <= 0.f ||
      grad_start < 0 || grad_start > k.size(2))
    return std::nullopt;
  if (mask.size() != 9 || k_src.size(2) != k.size(2) - grad_start) return std::nullopt;
  for (const auto &t : mask)
    if (!int32_on(t, q)) return std::nullopt;
  const at::DeviceGuard guard(q.device());
  const auto r = Attention::apply(q, k_src, v_src, k.detach(), v.detach(), Mask{std::move(mask), P, scale, grad_start});
  return std::make_tuple(r[0], r[1]);
}

// ---- q/k norm + RoPE into the cache rows --------------------------------------

// [1, S, H, D] with unit stride on D
bool heads4(const Tensor &t) { return t.dim() == 4 && t.size(0) == 1 && t.stride(3) == 1 && t.numel() > 0; }

// cos / sin [1, S, D] or [S, D]: row stride, or -1
int64_t table_stride(const Tensor &t, int64_t S, int64_t D) {
  const int64_t n = t.dim();
  if ((n != 2 && n != 3) || (n == 3 && t.size(0) != 1) || t.size(n - 2) != S || t.size(n - 1) != D || t.stride(n - 1) != 1)
    return -1;
  return t.stride(n - 2);
}

// a tensor on t's memory that is not an autograd view of it
Tensor rows_alias(const Tensor &t) {
  return at::empty({0}, t.options().requires_grad(false)).set_(t.storage(), t.storage_offset(), t.sizes(), t.strides());
}

struct NormRopeStage : public Function<NormRopeStage> {
  static variable_list forward(AutogradContext *ctx, const Tensor &q, const Tensor &k, const Tensor &v,
                               const Tensor &qw, const Tensor &kw, const Tensor &cos, const Tensor &sin, double eps,
                               const Tensor &kd, const Tensor &vd) {
    const int64_t S = q.size(1), Hq = q.size(2), D = q.size(3), Hkv = k.size(2);
    const auto opt = q.options().requires_grad(false);
    Tensor qo = at::empty({1, S, Hq, D}, opt);
    Tensor rstd = at::empty({S, Hq + Hkv}, opt.dtype(at::kFloat));
    check_rc("mga_qk_norm_rope_stage_fwd",
             g.mga_qk_norm_rope_stage_fwd(
                 q.data_ptr(), q.stride(1), q.stride(2), k.data_ptr(), k.stride(1), k.stride(2), v.data_ptr(),
                 v.stride(1), v.stride(2), qw.data_ptr(), kw.data_ptr(), cos.data_ptr(), sin.data_ptr(),
                 table_stride(cos, S, D), (float)eps, nullptr, 0, (int32_t)S, (int32_t)Hq, (int32_t)Hkv, (int32_t)D,
                 dtype_code(q.scalar_type()), qo.data_ptr(), qo.stride(1), qo.stride(2), kd.data_ptr(), kd.stride(2),
                 kd.stride(1), vd.data_ptr(), vd.stride(2), vd.stride(1), rstd.data_ptr<float>(), stream(q)));
    ctx->save_for_backward({q, k, qw, kw, cos, sin, rstd});
    return {qo.transpose(1, 2), rows_alias(kd), rows_alias(vd)};
  }

  static variable_list backward(AutogradContext *ctx, const variable_list &grad) {
    const auto s = ctx->get_saved_variables();
    const Tensor &q = s[0], &k = s[1], &qw = s[2], &kw = s[3], &cos = s[4], &sin = s[5], &rstd = s[6];
    const int64_t S = q.size(1), Hq = q.size(2), D = q.size(3), Hkv = k.size(2);
    const at::DeviceGuard guard(q.device());
    auto heads = [&](Tensor t) {
      t = t.to(q.scalar_type()).transpose(1, 2);
      return t.stride(3) == 1 ? t : t.contiguous();
    };
    variable_list out(10);
    if (ctx->needs_input_grad(0) || ctx->needs_input_grad(1)) {
      const Tensor gq = heads(grad[0]), gk = heads(grad[1]);
      const auto opt = q.options().requires_grad(false);
      Tensor dq = at::empty({1, S, Hq, D}, opt), dk = at::empty({1, S, Hkv, D}, opt);
      check_rc("mga_qk_norm_rope_bwd",
               g.mga_qk_norm_rope_bwd(q.data_ptr(), q.stride(1), q.stride(2), k.data_ptr(), k.stride(1), k.stride(2),
                                      qw.data_ptr(), kw.data_ptr(), cos.data_ptr(), sin.data_ptr(),
                                      table_stride(cos, S, D), rstd.data_ptr<float>(), (int32_t)S, (int32_t)Hq,
                                      (int32_t)Hkv, (int32_t)D, dtype_code(q.scalar_type()), gq.data_ptr(),
                                      gq.stride(1), gq.stride(2), gk.data_ptr(), gk.stride(1), gk.stride(2),
                                      dq.data_ptr(), dq.stride(1), dq.stride(2), dk.data_ptr(), dk.stride(1),
                                      dk.stride(2), stream(q)));
      if (ctx->needs_input_grad(0)) out[0] = dq;
      if (ctx->needs_input_grad(1)) out[1] = dk;
    }
    if (ctx->needs_input_grad(2)) out[2] = grad[2].transpose(1, 2);
    return out;
  }
};

std::optional<std::tuple<Tensor, Tensor, Tensor>> norm_rope_stage(const Tensor &q, const Tensor &k, const Tensor &v,
                                                                  const Tensor &qw, const Tensor &kw,
                                                                  const Tensor &cos, const Tensor &sin, double eps,
                                                                  const Tensor &kd, const Tensor &vd) {
  if (!eager()) return std::nullopt;
  for (const Tensor *t : {&q, &k, &v, &qw, &kw, &cos, &sin, &kd, &vd})
    if (!plain(*t) || !same(*t, q)) return std::nullopt;
  if (!heads4(q) || !heads4(k) || !heads4(v) || dtype_code(q.scalar_type()) < 0) return std::nullopt;
  const int64_t S = q.size(1), D = q.size(3), Hkv = k.size(2);
  if (k.size(1) != S || k.size(3) != D || v.sizes() != k.sizes() || D > 128 || D % 2) return std::nullopt;
  for (const Tensor *w : {&qw, &kw})
    if (w->dim() != 1 || w->size(0) != D || w->stride(0) != 1) return std::nullopt;
  if (table_stride(cos, S, D) < 0 || table_stride(cos, S, D) != table_stride(sin, S, D)) return std::nullopt;
  for (const Tensor *d : {&kd, &vd})
    if (d->dim() != 4 || d->size(0) != 1 || d->size(1) != Hkv || d->size(2) != S || d->size(3) != D || d->stride(3) != 1)
      return std::nullopt;
  const at::DeviceGuard guard(q.device());
  const auto r = NormRopeStage::apply(q, k, v, qw, kw, cos, sin, eps, kd, vd);
  return std::make_tuple(r[0], r[1], r[2]);
}

// ---- gated LoRA -----------------------------------------------------------------

// a [rows, cols] view that 16-byte vectors can read
bool rows2(const Tensor &t, int64_t cols) {
  return t.dim() == 2 && t.size(1) == cols && t.size(0) > 0 && t.stride(1) == 1 && t.stride(0) >= cols &&
         t.stride(0) % 8 == 0 && aligned16(t);
}

struct GatedLora : public Function<GatedLora> {
  static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &w, const Tensor &a, const Tensor &b,
                        const std::optional<Tensor> &gate, double scaling, double p, int64_t seed) {
    const int64_t N = w.size(0), K = w.size(1), rank = a.size(0), rp = (rank + 31) / 32 * 32;
    const Tensor x2 = x.detach().view({-1, K});
    const int64_t S = x2.size(0);
    const int dt = dtype_code(w.scalar_type());
    const auto opt = w.options().requires_grad(false);
    Tensor y = at::empty({S, N}, opt), t = at::empty({S, rp}, opt), h;
    if (p > 0 && (K % 128 || dt != MGA_DTYPE_BF16)) h = at::empty({S, K}, opt);
    const int64_t wn = g.mga_gated_lora_workspace_bytes((int32_t)S, (int32_t)K, (int32_t)N, (int32_t)rank);
    Tensor ws = bytes(wn, w);
    check_rc("mga_gated_lora_fwd",
             g.mga_gated_lora_fwd(x2.data_ptr(), x2.stride(0), w.data_ptr(), w.stride(0), a.data_ptr(), a.stride(0),
                                  b.data_ptr(), b.stride(0), gate ? gate->data_ptr<float>() : nullptr, (float)scaling, p, (uint64_t)seed, (int32_t)S, (int32_t)K, (int32_t)N, (int32_t)rank,
                                  y.data_ptr(), y.stride(0), t.data_ptr(), t.stride(0),
                                  h.defined() ? h.data_ptr() : nullptr, h.defined() ? h.stride(0) : 0, ws.data_ptr(),
                                  wn, dt, stream(w)));
    ctx->save_for_backward({x2, h, t, w, a, b, gate ? *gate : Tensor()});
    ctx->saved_data["scaling"] = scaling;
    ctx->saved_data["p"] = p;
    ctx->saved_data["seed"] = seed;
    ctx->saved_data["shape"] = x.sizes().vec();
    auto shape = x.sizes().vec();
    shape.back() = N;
    return y.view(shape);
  }

  static variable_list backward(AutogradContext *ctx, const variable_list &grad) {
    const auto s = ctx->get_saved_variables();
    const Tensor &x = s[0], &h = s[1], &t = s[2], &w = s[3], &a = s[4], &b = s[5], &gate = s[6];
    const int64_t N = w.size(0), K = w.size(1), rank = a.size(0), S = x.size(0);
    const int dt = dtype_code(w.scalar_type());
    const at::DeviceGuard guard(w.device());
    Tensor gy = grad[0].to(w.scalar_type()).reshape({-1, N});
    if (!rows2(gy, N)) gy = gy.contiguous();
    const auto opt = w.options().requires_grad(false);
    Tensor gx, ga, gb;
    if (ctx->needs_input_grad(0)) gx = at::empty({S, K}, opt);
    if (ctx->needs_input_grad(2)) ga = at::empty({rank, K}, opt);
    if (ctx->needs_input_grad(3)) gb = at::empty({N, rank}, opt);
    const int64_t wn = g.mga_gated_lora_workspace_bytes((int32_t)S, (int32_t)K, (int32_t)N, (int32_t)rank);
    Tensor ws = bytes(wn, w);
    auto ptr = [](const Tensor &v) { return v.defined() ? v.data_ptr() : nullptr; };
    auto rs = [](const Tensor &v) { return v.defined() ? v.stride(0) : 0; };
    check_rc("mga_gated_lora_bwd",
             g.mga_gated_lora_bwd(gy.data_ptr(), gy.stride(0), x.data_ptr(), x.stride(0), ptr(h), rs(h), w.data_ptr(),
                                  w.stride(0), a.data_ptr(), a.stride(0), b.data_ptr(), b.stride(0), t.data_ptr(),
                                  t.stride(0), gate.defined() ? gate.data_ptr<float>() : nullptr,
                                  (float)ctx->saved_data["scaling"].toDouble(), ctx->saved_data["p"].toDouble(),
                                  (uint64_t)ctx->saved_data["seed"].toInt(), (int32_t)S, (int32_t)K, (int32_t)N,
                                  (int32_t)rank, ptr(gx), rs(gx), ptr(ga), rs(ga), ptr(gb), rs(gb), ws.data_ptr(), wn,
                                  dt, stream(w)));
    variable_list out(8);
    if (gx.defined()) out[0] = gx.view(ctx->saved_data["shape"].toIntVector());
    out[2] = ga;
    out[3] = gb;
    return out;
  }
};

std::optional<Tensor> gated_lora(const Tensor &x, const Tensor &w, const Tensor &a, const Tensor &b,
                                 const std::optional<Tensor> &gate_mask, double scaling, double p, int64_t seed) {
  if (!eager()) return std::nullopt;
  for (const Tensor *t : {&x, &w, &a, &b})
    if (!plain(*t) || !same(*t, w)) return std::nullopt;
  if (gate_mask && (!plain(*gate_mask) || gate_mask->device() != w.device() || gate_mask->requires_grad()))
    return std::nullopt;
  if (dtype_code(w.scalar_type()) < 0 || w.dim() != 2 || a.dim() != 2 || b.dim() != 2 || !w.is_contiguous() ||
      !a.is_contiguous() || !b.is_contiguous() || x.dim() < 1 || x.numel() == 0 || w.numel() == 0 || a.numel() == 0)
    return std::nullopt;
  const int64_t K = w.size(1), N = w.size(0);
  if (x.size(-1) != K || a.size(1) != K || b.size(0) != N || b.size(1) != a.size(0) || K % 16 || !(p >= 0 && p < 1) ||
      !aligned16(a))
    return std::nullopt;
  const int64_t S = x.numel() / K;
  if (!x.is_contiguous() && x.dim() != 2) return std::nullopt;
  if (!rows2(x.detach().view({S, K}), K)) return std::nullopt;
  const at::DeviceGuard guard(w.device());
  std::optional<Tensor> gate;
  if (gate_mask) {
    if (gate_mask->numel() != S) return std::nullopt;
    gate = gate_mask->reshape({-1}).to(at::kFloat).contiguous();
  }
  return GatedLora::apply(x, w, a, b, gate, scaling, p, seed);
}

// ---- soft cross-entropy ------------------------------------------------------------

struct SoftCE : public Function<SoftCE> {
  static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &t) {
    const int32_t N = (int32_t)x.size(1), V = (int32_t)x.size(2);
    const auto opt = x.options().requires_grad(false).dtype(at::kFloat);
    Tensor loss = at::empty({N}, opt), stats = at::empty({4, N}, opt), total = at::empty({}, opt);
    Tensor ws = at::empty({g.mga_soft_ce_workspace_floats(N, V)}, opt);
    check_rc("mga_soft_ce_loss",
             g.mga_soft_ce_loss(x.data_ptr(), x.stride(1), t.data_ptr(), t.stride(1), N, V,
                                dtype_code(x.scalar_type()), loss.data_ptr<float>(), stats.data_ptr<float>(),
                                total.data_ptr<float>(), ws.data_ptr<float>(), stream(x)));
    ctx->save_for_backward({x.detach(), t.detach(), stats});
    return total;
  }
  static variable_list backward(AutogradContext *ctx, const variable_list &grad) {
    const auto s = ctx->get_saved_variables();
    const Tensor &x = s[0], &t = s[1], &stats = s[2];
    const at::DeviceGuard guard(x.device());
    const Tensor go = grad[0].detach().reshape({1}).to(x.device(), at::kFloat).contiguous();
    Tensor gx = at::empty(x.sizes(), x.options());
    check_rc("mga_soft_ce_bwd",
             g.mga_soft_ce_bwd(x.data_ptr(), x.stride(1), t.data_ptr(), t.stride(1), (int32_t)x.size(1),
                               (int32_t)x.size(2), dtype_code(x.scalar_type()), go.data_ptr<float>(),
                               stats.data_ptr<float>(), gx.data_ptr(), gx.stride(1), stream(x)));
    return {gx, Tensor()};
  }
};

std::optional<Tensor> soft_ce(const Tensor &x, const Tensor &t) {
  if (!eager() || !plain(x) || !plain(t) || !same(x, t) || dtype_code(x.scalar_type()) < 0) return std::nullopt;
  if (x.dim() != 3 || x.sizes() != t.sizes() || x.size(0) != 1 || x.numel() == 0 || x.stride(2) != 1 ||
      t.stride(2) != 1 || x.stride(1) < x.size(2) || t.stride(1) < x.size(2))
    return std::nullopt;
  const at::DeviceGuard guard(x.device());
  return SoftCE::apply(x, t);
}

// ---- vocabulary rows -----------------------------------------------------------------

// Rows of a [..., cols] tensor with unit stride on the last dimension; of every
// contiguous one with elements.
struct Rows {
  int64_t n = 1, stride = 0;
  int32_t cols = 0;
  void *data = nullptr;
};
std::optional<Rows> rows_of(const Tensor &t) {
  Rows r;
  const int64_t d = t.dim();
  if (d < 1 || t.numel() == 0 || t.size(d - 1) > INT32_MAX) return std::nullopt;
  if (t.size(d - 1) > 1 && t.stride(d - 1) != 1) return std::nullopt;   // one column may carry any stride
  r.cols = (int32_t)t.size(d - 1);
  for (int64_t i = d - 2; i >= 0; --i) {
    if (t.size(i) == 1) continue;
    if (r.n == 1) r.stride = t.stride(i);
    else if (t.stride(i) != r.stride * r.n) return std::nullopt;
    r.n *= t.size(i);
  }
  if (r.n == 1) r.stride = r.cols;
  if (r.stride < r.cols || r.n > INT32_MAX) return std::nullopt;
  r.data = t.data_ptr();
  return r;
}

constexpr int64_t kMaxTop = 1024, kMaxVocab = 1 << 20, kMaxCeVocab = 1 << 30;

std::optional<std::tuple<Tensor, Tensor, Tensor>> top_logits(const Tensor &x, int64_t k, double temperature) {
  if (!eager() || !plain(x) || dtype_code(x.scalar_type()) < 0) return std::nullopt;
  const auto r = rows_of(x);
  if (!r || k < 1 || k > kMaxTop || k > r->cols || r->cols > kMaxVocab) return std::nullopt;
  const at::DeviceGuard guard(x.device());
  auto lead = x.sizes().vec();
  lead.back() = k;
  const auto opt = x.options().requires_grad(false);
  Tensor values = at::empty(lead, opt), ids = at::empty(lead, opt.dtype(at::kInt));
  lead.pop_back();
  Tensor lse = at::empty(lead, opt.dtype(at::kFloat));
  check_rc("mga_top_logits",
           g.mga_top_logits(r->data, r->stride, (int32_t)r->n, r->cols, dtype_code(x.scalar_type()), (int32_t)k,
                            (float)temperature, values.data_ptr(), ids.data_ptr<int32_t>(), lse.data_ptr<float>(),
                            stream(x)));
  return std::make_tuple(values, ids, lse);
}

// The operands of a call against a teacher's top logits, of their plain form.
struct TopCe {
  Rows x, values, ids;
  int dtype, values_dtype;
  bool ids64;
  const float *lse = nullptr;
};
std::optional<TopCe> top_ce_operands(const Tensor &x, const Tensor &values, const Tensor &ids,
                                     const std::optional<Tensor> &lse) {
  if (!eager() || x.dim() < 1) return std::nullopt;
  for (const Tensor *t : {&x, &values, &ids})
    if (!plain(*t) || t->device() != x.device() || t->dim() != x.dim()) return std::nullopt;
  TopCe o;
  o.dtype = dtype_code(x.scalar_type());
  o.values_dtype = dtype_code(values.scalar_type());
  o.ids64 = ids.scalar_type() == at::kLong;
  if (o.dtype < 0 || o.values_dtype < 0 || (!o.ids64 && ids.scalar_type() != at::kInt) || values.sizes() != ids.sizes())
    return std::nullopt;
  const auto lead = x.sizes().slice(0, x.dim() - 1);
  if (values.sizes().slice(0, x.dim() - 1) != lead || values.size(-1) > kMaxTop) return std::nullopt;
  const auto rx = rows_of(x), rv = rows_of(values), ri = rows_of(ids);
  if (!rx || !rv || !ri || rx->cols > kMaxCeVocab) return std::nullopt;
  if (lse) {
    if (!plain(*lse) || lse->device() != x.device() || lse->scalar_type() != at::kFloat || lse->sizes() != lead ||
        !lse->is_contiguous())
      return std::nullopt;
    o.lse = lse->data_ptr<float>();
  }
  o.x = *rx;
  o.values = *rv;
  o.ids = *ri;
  return o;
}

struct TopLogitsCE : public Function<TopLogitsCE> {
  static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &values, const Tensor &ids,
                        const std::optional<Tensor> &lse, double tau) {
    const TopCe o = *top_ce_operands(x, values, ids, lse);
    const int32_t N = (int32_t)o.x.n, V = o.x.cols, K = o.ids.cols;
    const auto opt = x.options().requires_grad(false).dtype(at::kFloat);
    // what the backward reads, and what only this call does
    Tensor keep = at::empty({N * (3 + (int64_t)K)}, opt), total = at::empty({}, opt);
    Tensor ws = at::empty({g.mga_top_logits_ce_workspace_floats(N, V) + N}, opt);
    float *stats = keep.data_ptr<float>(), *w = ws.data_ptr<float>();
    check_rc("mga_top_logits_ce_fwd",
             g.mga_top_logits_ce_fwd(o.x.data, o.x.stride, o.values.data, o.values.stride, o.values_dtype, o.ids.data,
                                     o.ids.stride, o.ids64, o.lse, N, V, K, (float)tau, o.dtype, stats + 3 * (int64_t)N,
                                     stats, w + ws.numel() - N, total.data_ptr<float>(), w, stream(x)));
    ctx->save_for_backward({x.detach(), ids.detach(), keep});
    ctx->saved_data["tau"] = tau;
    return total;
  }
  static variable_list backward(AutogradContext *ctx, const variable_list &grad) {
    const auto s = ctx->get_saved_variables();
    const Tensor &x = s[0], &ids = s[1];
    const at::DeviceGuard guard(x.device());
    const Rows rx = *rows_of(x), ri = *rows_of(ids);
    const float *stats = s[2].data_ptr<float>();
    // of a scalar: one value, contiguous as it is
    const Tensor &g0 = grad[0];
    const Tensor go = g0.scalar_type() == at::kFloat && g0.device() == x.device() ? g0 : g0.detach().to(x.device(), at::kFloat);
    Tensor gx = at::empty(x.sizes(), x.options().requires_grad(false).memory_format(at::MemoryFormat::Contiguous));
    check_rc("mga_top_logits_ce_bwd",
             g.mga_top_logits_ce_bwd(rx.data, rx.stride, ri.data, ri.stride, ids.scalar_type() == at::kLong,
                                     stats + 3 * rx.n, stats, (int32_t)rx.n, rx.cols, ri.cols,
                                     (float)ctx->saved_data["tau"].toDouble(), dtype_code(x.scalar_type()),
                                     go.data_ptr<float>(), gx.data_ptr(), rx.cols, stream(x)));
    return {once("top_logits_cross_entropy", gx), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

std::optional<Tensor> top_logits_ce(const Tensor &x, const Tensor &values, const Tensor &ids,
                                    const std::optional<Tensor> &lse, double tau) {
  if (!top_ce_operands(x, values, ids, lse)) return std::nullopt;
  const at::DeviceGuard guard(x.device());
  check_capture("top_logits_cross_entropy", x);
  return TopLogitsCE::apply(x, values.detach(), ids, lse ? std::optional<Tensor>(lse->detach()) : lse, tau);
}

std::optional<std::tuple<Tensor, Tensor>> top_logits_step(const Tensor &x, const Tensor &values, const Tensor &ids,
                                                          const std::optional<Tensor> &lse, double tau, double scale) {
  const auto o = top_ce_operands(x, values, ids, lse);
  if (!o) return std::nullopt;
  const at::DeviceGuard guard(x.device());
  const int32_t N = (int32_t)o->x.n, V = o->x.cols, K = o->ids.cols;
  const auto opt = x.options().requires_grad(false);
  Tensor total = at::empty({}, opt.dtype(at::kFloat));
  Tensor gx = at::empty(x.sizes(), opt.memory_format(at::MemoryFormat::Contiguous));
  Tensor ws = at::empty({g.mga_top_logits_ce_step_workspace_floats(N, V, K) + N}, opt.dtype(at::kFloat));
  float *w = ws.data_ptr<float>();
  check_rc("mga_top_logits_ce_step",
           g.mga_top_logits_ce_step(o->x.data, o->x.stride, o->values.data, o->values.stride, o->values_dtype,
                                    o->ids.data, o->ids.stride, o->ids64, o->lse, N, V, K, (float)tau, (float)scale,
                                    o->dtype, w + ws.numel() - N, total.data_ptr<float>(), gx.data_ptr(), V, w,
                                    stream(x)));
  return std::make_tuple(total, gx);
}

// A sampling setting: a dense tensor with one value a row, or none (the number counts).
bool setting(const std::optional<Tensor> &t, const Tensor &x, int64_t n, at::ScalarType type) {
  return !t || (plain(*t) && t->device() == x.device() && t->scalar_type() == type && t->is_contiguous() &&
                t->numel() == n);
}

std::optional<Tensor> sample(const Tensor &x, const Tensor &u, const std::optional<Tensor> &temperature,
                             const std::optional<Tensor> &top_k, const std::optional<Tensor> &top_p,
                             const std::optional<Tensor> &min_p, double temperature_all, int64_t top_k_all,
                             double top_p_all, double min_p_all) {
  if (!eager() || !plain(x) || !plain(u) || dtype_code(x.scalar_type()) < 0) return std::nullopt;
  const auto r = rows_of(x);
  if (!r || r->cols > kMaxVocab || u.device() != x.device() || u.scalar_type() != at::kFloat || !u.is_contiguous() ||
      u.sizes() != x.sizes().slice(0, x.dim() - 1))
    return std::nullopt;
  if (!setting(temperature, x, r->n, at::kFloat) || !setting(top_k, x, r->n, at::kInt) ||
      !setting(top_p, x, r->n, at::kFloat) || !setting(min_p, x, r->n, at::kFloat))
    return std::nullopt;
  const at::DeviceGuard guard(x.device());
  Tensor token = at::empty(u.sizes(), x.options().requires_grad(false).dtype(at::kLong));
  auto f32 = [](const std::optional<Tensor> &t) { return t ? t->data_ptr<float>() : nullptr; };
  const int32_t k = (int32_t)std::max<int64_t>(-1, std::min(top_k_all, kMaxVocab));
  check_rc("mga_sample",
           g.mga_sample(r->data, r->stride, (int32_t)r->n, r->cols, dtype_code(x.scalar_type()), u.data_ptr<float>(),
                        f32(temperature), (float)temperature_all, top_k ? top_k->data_ptr<int32_t>() : nullptr, k,
                        f32(top_p), (float)top_p_all, f32(min_p), (float)min_p_all, token.data_ptr<int64_t>(),
                        stream(x)));
  return token;
}

// A list with the rows of x, or (shared) one for all of them.
struct RowList {
  const void *data = nullptr;
  int64_t stride = 0;
  int32_t n = 0;
  bool wide = false;
};
std::optional<RowList> row_list(const std::optional<Tensor> &t, const Tensor &x, bool shared) {
  RowList r;
  if (!t) return r;
  if (!plain(*t) || t->device() != x.device() || t->dim() < 1 || !t->is_contiguous() || t->numel() == 0 ||
      t->size(-1) > INT32_MAX)
    return std::nullopt;
  const bool one = t->dim() == 1 && x.dim() > 1;
  if (!(one && shared) && t->sizes().slice(0, t->dim() - 1) != x.sizes().slice(0, x.dim() - 1)) return std::nullopt;
  r.data = t->data_ptr();
  r.n = (int32_t)t->size(-1);
  r.stride = one ? 0 : r.n;
  r.wide = t->scalar_type() == at::kLong;
  return r;
}

std::optional<Tensor> adjust_logits(const Tensor &x, const std::optional<Tensor> &tokens, const std::optional<Tensor> &lengths,
                                    const std::optional<Tensor> &prompts, const std::optional<Tensor> &repetition,
                                    const std::optional<Tensor> &frequency, const std::optional<Tensor> &presence,
                                    double repetition_all, double frequency_all, double presence_all,
                                    const std::optional<Tensor> &bias_ids, const std::optional<Tensor> &bias,
                                    const std::optional<Tensor> &allowed, const std::optional<Tensor> &given) {
  if (!eager() || !plain(x) || dtype_code(x.scalar_type()) < 0 || given) return std::nullopt;
  const auto r = rows_of(x);
  if (!r) return std::nullopt;
  const auto tok = row_list(tokens, x, false), bid = row_list(bias_ids, x, true), val = row_list(bias, x, true),
             ok = row_list(allowed, x, true);
  if (!tok || !bid || !val || !ok || bid->n != val->n || (!tokens && (lengths || prompts))) return std::nullopt;
  for (const auto *t : {&tokens, &bias_ids})
    if (*t && (*t)->scalar_type() != at::kInt && (*t)->scalar_type() != at::kLong) return std::nullopt;
  if ((bias && bias->scalar_type() != at::kFloat) ||
      (allowed && (allowed->scalar_type() != at::kInt || ok->n != (r->cols + 31) / 32)))
    return std::nullopt;
  const auto lead = x.sizes().slice(0, x.dim() - 1);
  for (const auto *t : {&lengths, &prompts})
    if (*t && (!int32_on(**t, x) || (*t)->sizes() != lead)) return std::nullopt;
  if (!setting(repetition, x, r->n, at::kFloat) || !setting(frequency, x, r->n, at::kFloat) ||
      !setting(presence, x, r->n, at::kFloat))
    return std::nullopt;
  const at::DeviceGuard guard(x.device());
  Tensor out = at::empty(x.sizes(), x.options().requires_grad(false).memory_format(at::MemoryFormat::Contiguous));
  auto f32 = [](const std::optional<Tensor> &t) { return t ? t->data_ptr<float>() : nullptr; };
  auto i32 = [](const std::optional<Tensor> &t) { return t ? t->data_ptr<int32_t>() : nullptr; };
  check_rc("mga_adjust_logits",
           g.mga_adjust_logits(r->data, r->stride, (int32_t)r->n, r->cols, dtype_code(x.scalar_type()), tok->data, tok->wide,
                               tok->stride, tok->n, i32(lengths), i32(prompts), f32(repetition), (float)repetition_all,
                               f32(frequency), (float)frequency_all, f32(presence), (float)presence_all, bid->data,
                               bid->wide, bid->stride, (const float *)val->data, val->stride, bid->n,
                               (const int32_t *)ok->data, ok->stride, out.data_ptr(), r->cols, stream(x)));
  return out;
}

// ---- embedding -----------------------------------------------------------------------

struct Embedding : public Function<Embedding> {
  static Tensor forward(AutogradContext *ctx, const Tensor &ids, const Tensor &w, double scale, int64_t padding_idx) {
    auto shape = ids.sizes().vec();
    shape.push_back(w.size(1));
    Tensor out = at::empty(shape, w.options().requires_grad(false));
    check_rc("mga_embedding_fwd",
             g.mga_embedding_fwd(ids.data_ptr(), ids.scalar_type() == at::kLong, (int32_t)ids.numel(), w.data_ptr(),
                                 w.stride(0), (int32_t)w.size(0), (int32_t)w.size(1), (float)scale,
                                 dtype_code(w.scalar_type()), out.data_ptr(), w.size(1), stream(w)));
    ctx->save_for_backward({ids});
    ctx->saved_data["rows"] = w.size(0);
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["pad"] = padding_idx;
    return out;
  }
  static variable_list backward(AutogradContext *ctx, const variable_list &grad) {
    if (!ctx->needs_input_grad(1)) return {Tensor(), Tensor(), Tensor(), Tensor()};
    const auto s = ctx->get_saved_variables();
    const Tensor &ids = s[0];
    const at::DeviceGuard guard(ids.device());
    Tensor dy = grad[0].detach();
    auto r = rows_of(dy);
    if (!r) {
      dy = dy.contiguous();
      r = rows_of(dy);
    }
    const int64_t V = ctx->saved_data["rows"].toInt();
    const int32_t n = (int32_t)ids.numel(), H = r->cols;
    Tensor dw = at::empty({V, H}, dy.options().requires_grad(false).memory_format(at::MemoryFormat::Contiguous));
    const int64_t wn = g.mga_embedding_workspace_bytes(n, H);
    Tensor ws = bytes(wn, dy);
    check_rc("mga_embedding_bwd",
             g.mga_embedding_bwd(r->data, r->stride, ids.data_ptr(), ids.scalar_type() == at::kLong, n,
                                 (float)ctx->saved_data["scale"].toDouble(), ctx->saved_data["pad"].toInt(), (int32_t)V,
                                 H, dtype_code(dy.scalar_type()), dw.data_ptr(), H, dtype_code(dy.scalar_type()), 0,
                                 ws.data_ptr(), wn, stream(dy)));
    // linear in the output's gradient, of nothing else
    return {Tensor(), grad[0].requires_grad() ? once("scaled_embedding", dw) : dw, Tensor(), Tensor()};
  }
};

std::optional<Tensor> embedding(const Tensor &ids, const Tensor &w, double scale, int64_t padding_idx) {
  if (!eager() || !plain(ids) || !plain(w) || dtype_code(w.scalar_type()) < 0 || ids.device() != w.device())
    return std::nullopt;
  if ((ids.scalar_type() != at::kLong && ids.scalar_type() != at::kInt) || !ids.is_contiguous() || ids.numel() == 0 ||
      ids.numel() > INT32_MAX || w.dim() != 2 || w.numel() == 0 || w.stride(1) != 1 || w.stride(0) < w.size(1) ||
      w.size(0) > INT32_MAX || w.size(1) > INT32_MAX)
    return std::nullopt;
  const at::DeviceGuard guard(w.device());
  check_capture("scaled_embedding", w);
  return Embedding::apply(ids, w, scale, padding_idx);
}

// ---- paged cache -----------------------------------------------------------------------

// [tokens, heads, D] rows with unit stride on D
bool rows3(const Tensor &t, int64_t D, const Tensor &like) {
  return plain(t) && t.dim() == 3 && t.size(2) == D && t.stride(2) == 1 && t.stride(0) >= 0 && t.stride(1) >= 0 &&
         t.device() == like.device() && t.size(0) <= INT32_MAX;
}

bool aligned_rows3(const Tensor &t) {
  const int64_t eb = t.element_size();
  return t.stride(0) * eb % 16 == 0 && t.stride(1) * eb % 16 == 0 && aligned16(t);
}

struct Paged {
  int32_t n, Hkv, ps, D, B, width;
};

// Pages and batch of their plain form, contiguous.
std::optional<Paged> paged_operands(const Tensor &k, const Tensor &v, const Tensor &ks, const Tensor &vs,
                                    const Tensor &table, const Tensor &cu, const Tensor &lengths) {
  if (!eager()) return std::nullopt;
  for (const Tensor *t : {&k, &v, &ks, &vs})
    if (!plain(*t) || !t->is_contiguous() || t->device() != k.device()) return std::nullopt;
  for (const Tensor *t : {&table, &cu, &lengths})
    if (!int32_on(*t, k)) return std::nullopt;
  if (k.dim() != 4 || v.dim() != 4 || k.scalar_type() != at::kFloat8_e4m3fn || v.scalar_type() != at::kFloat8_e4m3fn ||
      ks.scalar_type() != at::kFloat || vs.scalar_type() != at::kFloat || table.dim() != 2 || table.numel() == 0)
    return std::nullopt;
  for (int64_t s : k.sizes())
    if (s <= 0 || s > INT32_MAX) return std::nullopt;
  const int64_t B = table.size(0);
  if (v.sizes() != at::IntArrayRef{k.size(0), k.size(1), k.size(3), k.size(2)} || ks.sizes() != k.sizes().slice(0, 2) ||
      vs.sizes() != k.sizes().slice(0, 2) || cu.sizes() != at::IntArrayRef{B + 1} || lengths.sizes() != at::IntArrayRef{B} ||
      B > INT32_MAX || table.size(1) > INT32_MAX)
    return std::nullopt;
  return Paged{(int32_t)k.size(0), (int32_t)k.size(1), (int32_t)k.size(2), (int32_t)k.size(3), (int32_t)B,
               (int32_t)table.size(1)};
}

// one tensor with a query, none without
std::optional<std::vector<Tensor>> paged_append(const Tensor &key, const Tensor &value, const Tensor &kp, const Tensor &vp,
                                                const Tensor &ks, const Tensor &vs, const Tensor &table, const Tensor &cu,
                                                const Tensor &lengths, const std::optional<Tensor> &query,
                                                const std::optional<Tensor> &cos, const std::optional<Tensor> &sin,
                                                const std::optional<Tensor> &qw, const std::optional<Tensor> &kw,
                                                double eps) {
  const auto p = paged_operands(kp, vp, ks, vs, table, cu, lengths);
  if (!p || !rows3(key, p->D, kp) || !rows3(value, p->D, kp) || dtype_code(key.scalar_type()) < 0 ||
      value.sizes() != key.sizes() || key.size(1) != p->Hkv || !same(key, value) || key.size(0) == 0)
    return std::nullopt;
  const int64_t T = key.size(0);
  if (query && (!rows3(*query, p->D, kp) || !same(*query, key) || query->size(0) != T || query->size(1) == 0))
    return std::nullopt;
  if (cos.has_value() != sin.has_value()) return std::nullopt;
  if (cos) {
    for (const Tensor *t : {&*cos, &*sin})
      if (!plain(*t) || t->dim() != 2 || t->size(0) != T || t->size(1) != p->D || t->stride(1) != 1 || t->stride(0) < 0 ||
          t->strides() != cos->strides() || !same(*t, *cos) || t->device() != kp.device() ||
          (t->scalar_type() != key.scalar_type() && t->scalar_type() != at::kFloat))
        return std::nullopt;
  }
  for (const auto *w : {&qw, &kw})
    if (*w && (!plain(**w) || !(*w)->is_contiguous() || (*w)->dim() != 1 || (*w)->size(0) != p->D || !same(**w, key)))
      return std::nullopt;
  const at::DeviceGuard guard(kp.device());
  std::vector<Tensor> out;
  if (query) out.push_back(at::empty(query->sizes(), query->options().requires_grad(false)));
  for (const Tensor *t : {&kp, &vp, &ks, &vs}) t->unsafeGetTensorImpl()->bump_version();
  auto ptr = [](const std::optional<Tensor> &t) { return t ? t->data_ptr() : nullptr; };
  auto st = [](const std::optional<Tensor> &t, int i) { return t ? t->stride(i) : 0; };
  check_rc("mga_paged_append",
           g.mga_paged_append(key.data_ptr(), key.stride(0), key.stride(1), value.data_ptr(), value.stride(0),
                              value.stride(1), ptr(query), st(query, 0), st(query, 1), ptr(qw), ptr(kw), ptr(cos), ptr(sin),
                              st(cos, 0), cos && cos->scalar_type() == at::kFloat, (float)eps, (int32_t)T, p->B,
                              query ? (int32_t)query->size(1) : 0, p->Hkv, p->D, dtype_code(key.scalar_type()),
                              kp.data_ptr(), vp.data_ptr(), ks.data_ptr<float>(), vs.data_ptr<float>(), p->n, p->ps,
                              table.data_ptr<int32_t>(), p->width, p->width, cu.data_ptr<int32_t>(),
                              lengths.data_ptr<int32_t>(), query ? out[0].data_ptr() : nullptr, query ? out[0].stride(0) : 0,
                              query ? out[0].stride(1) : 0, stream(kp)));
  return out;
}

std::optional<Tensor> paged_attention(const Tensor &q, const Tensor &kp, const Tensor &vp, const Tensor &ks,
                                      const Tensor &vs, const Tensor &table, const Tensor &cu, const Tensor &lengths,
                                      double scaling, const std::optional<Tensor> &given) {
  const auto p = paged_operands(kp, vp, ks, vs, table, cu, lengths);
  if (!p || given || !rows3(q, p->D, kp) || dtype_code(q.scalar_type()) < 0 || q.numel() == 0 || !aligned_rows3(q) ||
      q.size(1) > INT32_MAX || q.size(1) % p->Hkv)
    return std::nullopt;
  const at::DeviceGuard guard(kp.device());
  const int32_t T = (int32_t)q.size(0), Hq = (int32_t)q.size(1), code = dtype_code(q.scalar_type());
  Tensor out = at::empty(q.sizes(), q.options().requires_grad(false));
  const int64_t wn = g.mga_paged_attn_workspace_bytes(T, p->B, Hq, p->Hkv, p->D, p->ps, p->width, code);
  Tensor ws;
  if (wn) ws = bytes(wn, q);
  check_rc("mga_paged_attn",
           g.mga_paged_attn(q.data_ptr(), q.stride(0), q.stride(1), kp.data_ptr(), vp.data_ptr(), ks.data_ptr<float>(),
                            vs.data_ptr<float>(), p->n, p->ps, table.data_ptr<int32_t>(), p->width, p->width,
                            cu.data_ptr<int32_t>(), lengths.data_ptr<int32_t>(), T, p->B, Hq, p->Hkv, p->D, code,
                            (float)scaling, out.data_ptr(), out.stride(0), out.stride(1), 1, wn ? ws.data_ptr() : nullptr, wn, stream(q)));
  return out;
}

}  // namespace

#define MGA_DEF(f) m.def(#f, torch::wrap_pybind_function_no_gil(f))
PYBIND11_MODULE(_mga_torch, m) {
  m.def("bind", &bind_api);
  MGA_DEF(kv_append);
  MGA_DEF(update_kv);
  MGA_DEF(attention);
  MGA_DEF(norm_rope_stage);
  MGA_DEF(gated_lora);
  MGA_DEF(soft_ce);
  MGA_DEF(top_logits);
  MGA_DEF(top_logits_ce);
  MGA_DEF(top_logits_step);
  MGA_DEF(sample);
  MGA_DEF(adjust_logits);
  MGA_DEF(embedding);
  MGA_DEF(paged_append);
  MGA_DEF(paged_attention);
  MGA_DEF(check_capture);
  MGA_DEF(once);
}
