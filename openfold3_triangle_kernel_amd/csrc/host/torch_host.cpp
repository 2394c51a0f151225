// Host path of the operators for plain eager GPU tensors, in C++.
//
// The Python facades stay the definition of the operators: they validate,
// report and handle every form.  A small call is bound by what the host does
// around its launches (N = 128 attention, forward and backward: 45 us of
// kernels behind about 200 us of Python), so the common form is recognised and
// run here: the same checks, the same native calls with the same arguments,
// autograd through C++ nodes.  Everything else returns no value, before any
// launch, and the facade goes on in Python: other dtypes or devices, head
// dimensions that need padding, partially broadcast biases, misaligned
// storage, function transforms, forward-mode AD, dispatch modes.
#include <torch/extension.h>
#include <torch/version.h>

#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>

#include <torch/csrc/autograd/functions/basic_ops.h>

#include <atomic>
#include <cctype>
#include <cmath>
#include <cstdlib>
#include <optional>
#include <string>

#include "tpf_amd.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// Workspace budget of the attention backward (attention.set_sr_workspace_budget).
std::atomic<int64_t> g_budget{int64_t(8) << 30};

void check(int rc, const char* fn) {
  if (rc != TPF_OK)
    throw std::runtime_error(std::string(fn) + " failed (status " + std::to_string(rc) +
                             "): " + tpf_last_error());
}

void* stream() { return (void*)c10::hip::getCurrentHIPStream().stream(); }

// The policy variables as the facade reads them: the canonical name, then
// the older one, then "1"; surrounding blanks dropped.  Called with the GIL
// held: Python's os.environ assignments change the environment under it.
std::string env_flag(const char* canonical, const char* legacy) {
  const char* v = std::getenv(canonical);
  if (!v) v = std::getenv(legacy);
  std::string s = v ? v : "1";
  const char* ws = " \t\n\r\f\v";
  const size_t b = s.find_first_not_of(ws);
  if (b == std::string::npos) return "";
  return s.substr(b, s.find_last_not_of(ws) - b + 1);
}

bool transforms_active() {
  return c10::impl::tls_is_dispatch_key_included(at::DispatchKey::FuncTorchDynamicLayerFrontMode) ||
         c10::impl::dispatch_mode_enabled();
}

// An ordinary strided tensor on the current GPU.
bool plain(const Tensor& t, c10::DeviceIndex dev) {
  static const at::DispatchKeySet special{
      at::DispatchKey::FuncTorchBatched, at::DispatchKey::FuncTorchGradWrapper,
      at::DispatchKey::Functionalize,    at::DispatchKey::Python,
      at::DispatchKey::ZeroTensor,       at::DispatchKey::Conjugate,
      at::DispatchKey::Negative};
  return t.defined() && t.is_cuda() && t.device().index() == dev && t.layout() == at::kStrided &&
         !t.key_set().has_any(special) && !t._fw_grad(0).defined();
}

bool aligned16(const Tensor& t) { return (uintptr_t)t.const_data_ptr() % 16 == 0; }

// An upstream gradient as the kernels read it: bf16, contiguous, 16-byte aligned.
Tensor kernel_grad(const Tensor& g) {
  const Tensor t = g.to(at::kBFloat16).contiguous();
  return aligned16(t) ? t : t.clone();
}

at::TensorOptions like(const Tensor& t, at::ScalarType dtype) {
  return at::TensorOptions().device(t.device()).dtype(dtype);
}

// Whether `sizes`, aligned to the right of `prefix`, broadcasts to exactly it.
bool broadcasts(at::IntArrayRef sizes, at::IntArrayRef prefix) {
  if (sizes.size() > prefix.size()) return false;
  const size_t off = prefix.size() - sizes.size();
  for (size_t i = 0; i < sizes.size(); ++i)
    if (sizes[i] != 1 && sizes[i] != prefix[off + i]) return false;
  return true;
}

// ------------------------------------------------------------- attention

struct AttentionFn : torch::autograd::Function<AttentionFn> {
  // bias_k: the detached kernel bias; source_bias keeps the autograd edge.
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v,
                        const Tensor& mask, const Tensor& bias_k, const Tensor& source_bias,
                        int64_t layout, int64_t bias_batches, bool shadow) {
    const int64_t B = q.size(0), O = q.size(1), H = q.size(2), N = q.size(3), D = q.size(4);
    const double scale = 1.0 / std::sqrt((double)D);
    Tensor out = at::empty({B, O, N, H, D}, like(q, at::kBFloat16));
    Tensor lse = at::empty({B, O, H, N}, like(q, at::kFloat));
    const int64_t ws_bytes = tpf_attn_forward_workspace_bytes(B, H, N, bias_batches);
    Tensor ws = at::empty({ws_bytes}, like(q, at::kByte)), res;
    if (shadow) {
      res = at::empty_like(out);
      check(tpf_attn_forward_shadow_bf16(
                q.const_data_ptr(), k.const_data_ptr(), v.const_data_ptr(),
                (const float*)mask.const_data_ptr(), bias_k.const_data_ptr(), out.data_ptr(),
                (float*)lse.data_ptr(), res.data_ptr(), ws.data_ptr(), ws_bytes, B, O, H, N, D,
                (int)layout, bias_batches, scale, stream()),
            "tpf_attn_forward_shadow_bf16");
    } else {
      check(tpf_attn_forward_bf16(q.const_data_ptr(), k.const_data_ptr(), v.const_data_ptr(),
                                  (const float*)mask.const_data_ptr(), bias_k.const_data_ptr(),
                                  out.data_ptr(), (float*)lse.data_ptr(), ws.data_ptr(), ws_bytes,
                                  B, O, H, N, D, (int)layout, bias_batches, scale, stream()),
            "tpf_attn_forward_bf16");
    }
    ctx->save_for_backward({q, k, v, mask, bias_k, out, lse, res});
    ctx->saved_data["layout"] = layout;
    ctx->saved_data["batches"] = bias_batches;
    ctx->saved_data["shape"] = source_bias.sizes().vec();
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list s = ctx->get_saved_variables();
    const Tensor &q = s[0], &k = s[1], &v = s[2], &mask = s[3], &bias_k = s[4], &out = s[5],
                 &lse = s[6], &res = s[7];
    const int64_t layout = ctx->saved_data["layout"].toInt();
    const int64_t batches = ctx->saved_data["batches"].toInt();
    const int64_t B = q.size(0), O = q.size(1), H = q.size(2), N = q.size(3), D = q.size(4);
    const Tensor dout = kernel_grad(grads[0]);
    Tensor d[3];
    for (Tensor& t : d)
      t = layout & TPF_QKV_SEQ_MAJOR
              ? at::empty({B, O, N, H, D}, like(q, at::kBFloat16)).transpose(2, 3)
              : at::empty({B, O, H, N, D}, like(q, at::kBFloat16));
    // The fold writes the bf16 bias gradient in the bias's own storage order.
    Tensor dbias = at::empty({batches, H, N, N}, like(q, at::kBFloat16));
    const int64_t ws_bytes = tpf_attn_backward_workspace_bytes_budget(
        B, O, H, N, D, g_budget.load(std::memory_order_relaxed));
    Tensor ws = at::empty({ws_bytes}, like(q, at::kByte));
    check(tpf_attn_backward_fused_bf16(
              q.const_data_ptr(), k.const_data_ptr(), v.const_data_ptr(), dout.const_data_ptr(),
              out.const_data_ptr(), res.defined() ? res.const_data_ptr() : nullptr,
              (const float*)lse.const_data_ptr(), (const float*)mask.const_data_ptr(),
              bias_k.const_data_ptr(), d[0].data_ptr(), d[1].data_ptr(), d[2].data_ptr(),
              dbias.data_ptr(), ws.data_ptr(), ws_bytes, B, O, H, N, D,
              (int)layout | TPF_DBIAS_BF16, batches, 1.0 / std::sqrt((double)D), stream()),
          "tpf_attn_backward_fused_bf16");
    if (layout & TPF_BIAS_TRANSPOSED) dbias = dbias.transpose(-1, -2);
    return {d[0], d[1], d[2], Tensor(), Tensor(),
            dbias.reshape(ctx->saved_data["shape"].toIntVector()), Tensor(), Tensor(), Tensor()};
  }
};

// backward, shadow: the policy variables (env_flag).
std::optional<Tensor> attention(const Tensor& q, const Tensor& k, const Tensor& v,
                                const Tensor& res_mask, const Tensor& pair_bias,
                                const std::string& backward, const std::string& sh) {
  if (transforms_active() || !q.is_cuda()) return std::nullopt;
  const c10::DeviceIndex dev = c10::hip::current_device();
  for (const Tensor* t : {&q, &k, &v, &res_mask, &pair_bias})
    if (!plain(*t, dev)) return std::nullopt;
  const int64_t nd = q.dim();
  if (nd < 5 || q.numel() == 0 || k.sizes() != q.sizes() || v.sizes() != q.sizes())
    return std::nullopt;
  for (const Tensor* t : {&q, &k, &v})
    if (t->scalar_type() != at::kBFloat16) return std::nullopt;
  const at::IntArrayRef prefix = q.sizes().slice(0, nd - 4);
  const int64_t O = q.size(-4), H = q.size(-3), N = q.size(-2), D = q.size(-1);
  const int64_t B = c10::multiply_integers(prefix);
  if (D % 8 || D > 64 || H > 65535 || B * O > 65535) return std::nullopt;
  const auto mt = res_mask.scalar_type();
  if ((mt != at::kFloat && mt != at::kBFloat16 && mt != at::kHalf) || res_mask.requires_grad() ||
      res_mask.dim() < 4 || res_mask.size(-4) != O || res_mask.size(-3) != 1 ||
      res_mask.size(-2) != 1 || res_mask.size(-1) != N ||
      !broadcasts(res_mask.sizes().slice(0, res_mask.dim() - 4), prefix))
    return std::nullopt;
  const auto bt = pair_bias.scalar_type();
  if ((bt != at::kFloat && bt != at::kBFloat16) || pair_bias.dim() < 4 || pair_bias.size(-4) != 1 ||
      pair_bias.size(-3) != H || pair_bias.size(-2) != N || pair_bias.size(-1) != N)
    return std::nullopt;
  const at::IntArrayRef bp = pair_bias.sizes().slice(0, pair_bias.dim() - 4);
  const bool shared = c10::multiply_integers(bp) == 1 && bp.size() <= prefix.size();
  if (!shared && bp != prefix) return std::nullopt;
  if (backward == "0" || (sh != "0" && sh != "1")) return std::nullopt;

  // One storage order for q, k and v: contiguous, or the transposed view of a
  // contiguous [*B, O, N, H, D] projection.
  auto order = [](const Tensor& t) {
    if (t.is_contiguous()) return 0;
    return t.transpose(-2, -3).is_contiguous() && aligned16(t) ? 1 : 2;
  };
  const int oq = order(q);
  if (oq == 2 || order(k) != oq || order(v) != oq || !aligned16(q) || !aligned16(k) ||
      !aligned16(v))
    return std::nullopt;
  int64_t layout = (oq ? TPF_QKV_SEQ_MAJOR : 0) | (N % 64 ? TPF_ANY_N : 0);
  auto flat = [&](const Tensor& t) { return nd == 5 ? t : t.reshape({B, O, H, N, D}); };

  Tensor mask = res_mask;
  if (res_mask.dim() != 5 || res_mask.size(0) != B || mt != at::kFloat || nd != 5 ||
      !res_mask.is_contiguous()) {
    std::vector<int64_t> full = prefix.vec();
    full.insert(full.end(), {O, 1, 1, N});
    mask = res_mask.expand(full).reshape({B, O, N}).to(at::kFloat).contiguous();
  }
  const Tensor bias = bt == at::kFloat ? pair_bias.to(at::kBFloat16) : pair_bias;
  Tensor bias_k = bias.detach();
  if (!bias_k.is_contiguous()) {
    if (bias_k.transpose(-1, -2).is_contiguous()) layout |= TPF_BIAS_TRANSPOSED;
    else bias_k = bias_k.contiguous();
  }
  if (!aligned16(mask) || !aligned16(bias_k)) return std::nullopt;
  const bool grad = at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() ||
                                                   v.requires_grad() || bias.requires_grad());
  Tensor out = AttentionFn::apply(flat(q), flat(k), flat(v), mask, bias_k, bias, layout,
                                  shared ? 1 : B, sh == "1" && grad);
  if (nd == 5) return out;
  std::vector<int64_t> shape = prefix.vec();
  shape.insert(shape.end(), {O, N, H, D});
  return out.reshape(shape);
}

// ---------------------------------------------------------------- TriMul

int64_t a256(int64_t v) { return (v + 255) / 256 * 256; }

// The forward's state in one allocation: z_ln, gate, a, b, x (bf16), LN_in's
// statistics (f32) and, for a backward, xln (bf16) and LN_out's (f32).
struct TrimulState {
  char* p[10] = {};
  int64_t bytes;
  TrimulState(int64_t B, int64_t N, int64_t C, bool save, char* base) {
    const int64_t rows = a256(B * N * N * C * 2);
    const int64_t planes = a256(B * C * N * tpf_trimul_plane_pitch(N) * 2);
    const int64_t stat = a256(B * N * N * 4);
    const int64_t sizes[10] = {rows, rows, planes, planes, planes, stat, stat, rows, stat, stat};
    bytes = 0;
    for (int i = 0; i < (save ? 10 : 7); ++i) {
      p[i] = base + bytes;
      bytes += sizes[i];
    }
  }
};

// params: p_in [2C, C], g_in [2C, C], g_out [C, C], p_out [C, C], then the
// weight and bias of LN_in and LN_out.
Tensor trimul_forward(const Tensor& z, const Tensor& mask, const variable_list& w, bool outgoing,
                      const TrimulState& st) {
  const int64_t B = z.size(0), N = z.size(1), C = z.size(3), cc = C * C;
  Tensor out = at::empty({B, N, N, C}, like(z, at::kBFloat16));
  const int64_t ws_bytes = tpf_trimul_forward_workspace_bytes(C);
  Tensor ws = at::empty({ws_bytes}, like(z, at::kByte));
  auto f = [&](int i) { return (const float*)w[i].const_data_ptr(); };
  check(tpf_trimul_forward_bf16(
            z.const_data_ptr(), (const float*)mask.const_data_ptr(), f(0), f(1), f(0) + cc,
            f(1) + cc, f(2), f(3), f(4), f(5), f(6), f(7), outgoing ? 1 : 0, B, N, C,
            out.data_ptr(), st.p[0], st.p[1], st.p[2], st.p[3], st.p[4], st.p[7], (float*)st.p[5],
            (float*)st.p[6], (float*)st.p[8], (float*)st.p[9], ws.data_ptr(), ws_bytes, stream()),
        "tpf_trimul_forward_bf16");
  return out;
}

struct TrimulFn : torch::autograd::Function<TrimulFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& z, const Tensor& mask,
                        const Tensor& p_in, const Tensor& g_in, const Tensor& g_out,
                        const Tensor& p_out, const Tensor& n_in_w, const Tensor& n_in_b,
                        const Tensor& n_out_w, const Tensor& n_out_b, bool outgoing) {
    const int64_t B = z.size(0), N = z.size(1), C = z.size(3);
    Tensor state = at::empty({TrimulState(B, N, C, true, nullptr).bytes}, like(z, at::kByte));
    Tensor out = trimul_forward(z, mask, {p_in, g_in, g_out, p_out, n_in_w, n_in_b, n_out_w, n_out_b},
                                outgoing, TrimulState(B, N, C, true, (char*)state.data_ptr()));
    ctx->save_for_backward({z, mask, state, p_in, g_in, g_out, p_out, n_in_w, n_out_w});
    ctx->saved_data["outgoing"] = outgoing;
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list s = ctx->get_saved_variables();
    const Tensor &z = s[0], &mask = s[1], &state = s[2];
    const int64_t B = z.size(0), N = z.size(1), C = z.size(3), cc = C * C;
    const TrimulState st(B, N, C, true, (char*)state.data_ptr());
    const Tensor g = kernel_grad(grads[0]);
    const auto f32 = like(z, at::kFloat);
    Tensor dz = at::empty({B, N, N, C}, like(z, at::kBFloat16));
    Tensor dp = at::empty({2 * C, C}, f32), dg = at::empty({2 * C, C}, f32);
    Tensor dgo = at::empty({C, C}, f32), dpo = at::empty({C, C}, f32);
    Tensor dn[4];
    for (Tensor& t : dn) t = at::empty({C}, f32);
    const int64_t ws_bytes = tpf_trimul_backward_workspace_bytes(B, N, C);
    Tensor ws = at::empty({ws_bytes}, like(z, at::kByte));
    auto f = [&](int i) { return (const float*)s[i].const_data_ptr(); };
    auto o = [](const Tensor& t) { return (float*)t.data_ptr(); };
    check(tpf_trimul_backward_named_bf16(
              g.const_data_ptr(), z.const_data_ptr(), (const float*)mask.const_data_ptr(), f(3),
              f(4), f(3) + cc, f(4) + cc, f(5), f(6), f(7), f(8), st.p[0], st.p[1], st.p[2],
              st.p[3], st.p[4], st.p[7], (const float*)st.p[5], (const float*)st.p[6],
              (const float*)st.p[8], (const float*)st.p[9],
              ctx->saved_data["outgoing"].toBool() ? 1 : 0, B, N, C, dz.data_ptr(), o(dp), o(dg),
              o(dgo), o(dpo), o(dn[0]), o(dn[1]), o(dn[2]), o(dn[3]), ws.data_ptr(), ws_bytes,
              stream()),
          "tpf_trimul_backward_named_bf16");
    return {dz, Tensor(), dp, dg, dgo, dpo, dn[0], dn[1], dn[2], dn[3], Tensor()};
  }
};

std::optional<Tensor> trimul(const Tensor& z, const std::optional<Tensor>& mask_in,
                             const variable_list& w, bool outgoing) {
  if (transforms_active() || !z.is_cuda()) return std::nullopt;
  const c10::DeviceIndex dev = c10::hip::current_device();
  if (!plain(z, dev) || z.dim() < 3 || z.scalar_type() != at::kBFloat16 || z.numel() == 0 ||
      !z.is_contiguous() || !aligned16(z))
    return std::nullopt;
  const int64_t C = z.size(-1), N = z.size(-2);
  if (z.size(-3) != N) return std::nullopt;
  const int64_t B = z.numel() / (N * N * C);
  if (!tpf_trimul_shape_supported(B, N, C, 0)) return std::nullopt;
  for (size_t i = 0; i < w.size(); ++i) {
    const Tensor& t = w[i];
    if (!plain(t, dev) || t.scalar_type() != at::kFloat || !t.is_contiguous() || !aligned16(t))
      return std::nullopt;
    if (i < 4 ? (t.dim() != 2 || t.size(0) != (i < 2 ? 2 * C : C) || t.size(1) != C)
              : (t.dim() != 1 || t.size(0) != C))
      return std::nullopt;
  }
  Tensor mask;
  if (!mask_in.has_value()) {
    mask = at::ones({B, N, N}, like(z, at::kFloat));
  } else {
    mask = *mask_in;
    if (!plain(mask, dev) || mask.sizes() != z.sizes().slice(0, z.dim() - 1) ||
        !mask.is_contiguous() || mask.requires_grad())
      return std::nullopt;
    if (mask.scalar_type() != at::kFloat) mask = mask.to(at::kFloat);
  }
  bool grad = z.requires_grad();
  for (const Tensor& t : w) grad = grad || t.requires_grad();
  grad = grad && at::GradMode::is_enabled();
  if (grad && !tpf_trimul_shape_supported(B, N, C, 1)) return std::nullopt;
  const Tensor z4 = z.dim() == 4 ? z : z.view({B, N, N, C});
  Tensor out;
  if (grad) {
    out = TrimulFn::apply(z4, mask, w[0], w[1], w[2], w[3], w[4], w[5], w[6], w[7], outgoing);
  } else {
    Tensor scratch = at::empty({TrimulState(B, N, C, false, nullptr).bytes}, like(z, at::kByte));
    out = trimul_forward(z4, mask, w, outgoing, TrimulState(B, N, C, false, (char*)scratch.data_ptr()));
  }
  return z.dim() == 4 ? out : out.view(z.sizes());
}

// --------------------------------------------------------- shared by the below

// Gradients asked for with create_graph: as Python's once_differentiable,
// differentiating them again raises.
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list marked;
  for (const Tensor& g : grads) {
    Tensor t = g.defined() ? g.detach() : g;
    if (t.defined()) t.set_requires_grad(true);
    marked.push_back(t);
  }
  auto err = std::make_shared<torch::autograd::DelayedError>(
      "trying to differentiate twice a function that was marked with @once_differentiable",
      (int64_t)marked.size());
  return (*err)(std::move(marked));
}

const void* cptr(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* mptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
Tensor bytes(const Tensor& like_, int64_t n) {
  return n > 0 ? at::empty({n}, like(like_, at::kByte)) : Tensor();
}
int64_t type_code(at::ScalarType t) {
  return t == at::kBFloat16 ? TPF_BF16 : t == at::kHalf ? TPF_F16 : t == at::kFloat ? TPF_F32 : -1;
}

// ----------------------------------------------------------- cross attention

void strides3(const Tensor& t, int64_t* out) {
  for (int i = 0; i < 3; ++i) out[i] = t.size(i) > 1 ? t.stride(i) : 0;
}

// q [B, H, Nq, D], k and v [B, Hk, Nk, D] as the kernels read them.
tpf_xattn_shape xattn_shape(const Tensor& q, const Tensor& k, const Tensor& v, int64_t kind,
                            int64_t mask_stride) {
  tpf_xattn_shape s{q.size(0), q.size(1), k.size(1), q.size(2), k.size(2), q.size(3),
                    type_code(q.scalar_type()), kind, mask_stride, {}, {}, {}};
  strides3(q, s.q_stride);
  strides3(k, s.k_stride);
  strides3(v, s.v_stride);
  return s;
}

Tensor xattn_forward(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& mask,
                     int64_t kind, int64_t mask_stride, double scale, Tensor* lse, Tensor* res) {
  const tpf_xattn_shape s = xattn_shape(q, k, v, kind, mask_stride);
  Tensor out = at::empty({s.B, s.Nq, s.H, s.D}, q.options());
  if (lse) *lse = at::empty({kind == TPF_MASK_F32 ? 2 : 1, s.B, s.H, s.Nq}, like(q, at::kFloat));
  const int64_t n = tpf_xattn_forward_workspace_bytes(&s);
  const Tensor ws = bytes(q, n);
  if (res) {
    *res = at::empty_like(out);
    check(tpf_xattn_forward_shadow_bf16(cptr(q), cptr(k), cptr(v), cptr(mask), out.data_ptr(),
                                        (float*)lse->data_ptr(), res->data_ptr(), mptr(ws),
                                        n, &s, scale, stream()),
          "tpf_xattn_forward_shadow_bf16");
  } else {
    check(tpf_xattn_forward(cptr(q), cptr(k), cptr(v), cptr(mask), out.data_ptr(),
                            lse ? (float*)lse->data_ptr() : nullptr, mptr(ws), n, &s, scale,
                            stream()),
          "tpf_xattn_forward");
  }
  return out;
}

// A gradient in the operand's storage order, where that keeps its channels
// contiguous (a broadcast operand's order may not).
Tensor grad_like(const Tensor& t) {
  Tensor g = at::empty_like(t);
  bool fine = g.stride(3) == 1;
  for (int i = 0; i < 3; ++i) fine = fine && g.stride(i) % 8 == 0;
  return fine ? g : at::empty(t.sizes(), t.options());
}

struct XattnFn : torch::autograd::Function<XattnFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v,
                        const std::optional<Tensor>& mask_in, int64_t kind, int64_t mask_stride,
                        double scale, bool shadow) {
    const Tensor mask = mask_in.value_or(Tensor());
    Tensor lse, res;
    Tensor out = xattn_forward(q, k, v, mask, kind, mask_stride, scale, &lse, shadow ? &res : nullptr);
    ctx->save_for_backward({q, k, v, mask, out, lse, res});
    ctx->saved_data["kind"] = kind;
    ctx->saved_data["stride"] = mask_stride;
    ctx->saved_data["scale"] = scale;
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list sv = ctx->get_saved_variables();
    const Tensor &q = sv[0], &k = sv[1], &v = sv[2], &mask = sv[3], &out = sv[4], &lse = sv[5], &res = sv[6];
    const tpf_xattn_shape s = xattn_shape(q, k, v, ctx->saved_data["kind"].toInt(),
                                          ctx->saved_data["stride"].toInt());
    const Tensor dout = kernel_grad(grads[0]);
    Tensor d[3] = {grad_like(q), grad_like(k), grad_like(v)};
    int64_t gs[9];
    for (int i = 0; i < 3; ++i) strides3(d[i], gs + 3 * i);
    const int64_t n = tpf_xattn_backward_workspace_bytes(&s);
    const Tensor ws = bytes(q, n < 16 ? 16 : n);
    const double scale = ctx->saved_data["scale"].toDouble();
    if (res.defined())
      check(tpf_xattn_backward_shadow_bf16(cptr(q), cptr(k), cptr(v), cptr(mask), cptr(out), cptr(res),
                                           cptr(dout), (const float*)cptr(lse), mptr(d[0]), mptr(d[1]),
                                           mptr(d[2]), mptr(ws), n, &s, gs, scale, stream()),
            "tpf_xattn_backward_shadow_bf16");
    else
      check(tpf_xattn_backward_bf16(cptr(q), cptr(k), cptr(v), cptr(mask), cptr(out), cptr(dout),
                                    (const float*)cptr(lse), mptr(d[0]), mptr(d[1]), mptr(d[2]),
                                    mptr(ws), n, &s, gs, scale, stream()),
            "tpf_xattn_backward_bf16");
    return once({d[0], d[1], d[2], Tensor(), Tensor(), Tensor(), Tensor(), Tensor()});
  }
};

bool xattn_operand(const Tensor& t) {
  if (t.stride(3) != 1 || !aligned16(t)) return false;
  for (int i = 0; i < 3; ++i)
    if (t.size(i) > 1 && t.stride(i) % 8) return false;
  return t.size(2) <= 1 || t.stride(2) < (int64_t(1) << 23);
}

// sh: the policy variable of the shadow residual (env_flag).
std::optional<Tensor> cross_attention(const Tensor& q, const Tensor& k, const Tensor& v,
                                      const std::optional<Tensor>& mask_in,
                                      std::optional<double> scale_in, const std::string& sh) {
  if (transforms_active() || !q.is_cuda()) return std::nullopt;
  const c10::DeviceIndex dev = c10::hip::current_device();
  for (const Tensor* t : {&q, &k, &v})
    if (!plain(*t, dev) || t->dim() != 4 || t->numel() == 0 || t->scalar_type() != q.scalar_type())
      return std::nullopt;
  const auto type = q.scalar_type();
  const bool grad = at::GradMode::is_enabled() &&
                    (q.requires_grad() || k.requires_grad() || v.requires_grad());
  if (type != at::kBFloat16 && (type != at::kHalf || grad)) return std::nullopt;
  if (grad && sh != "0" && sh != "1") return std::nullopt;
  const int64_t B = q.size(0), D = q.size(3), Nk = k.size(2);
  if (k.sizes() != v.sizes() || k.size(0) != B || k.size(3) != D || D % 8 || D > 128 ||
      q.size(1) % k.size(1))
    return std::nullopt;
  for (const Tensor* t : {&q, &k, &v})
    if (!xattn_operand(*t)) return std::nullopt;
  const double scale = scale_in ? *scale_in : 1.0 / std::sqrt((double)D);
  if (!(scale > 1e-30 && scale < 1e30)) return std::nullopt;
  Tensor mask;
  int64_t kind = TPF_MASK_NONE, mask_stride = 0;
  if (mask_in) {
    mask = *mask_in;
    const auto mt = mask.scalar_type();
    if (!plain(mask, dev) || mask.requires_grad() || (mt != at::kBool && mt != at::kFloat) ||
        !mask.is_contiguous() || mask.dim() < 1 || mask.dim() > 2 || mask.size(-1) != Nk ||
        (mask.dim() == 2 && mask.size(0) != B && mask.size(0) != 1))
      return std::nullopt;
    kind = mt == at::kBool ? TPF_MASK_BYTES : TPF_MASK_F32;
    mask_stride = mask.dim() == 2 && mask.size(0) > 1 ? Nk : 0;
  }
  // Sizes that the launches do not hold (of the backward too, before the forward).
  const tpf_xattn_shape s = xattn_shape(q, k, v, kind, mask_stride);
  if (tpf_xattn_forward_workspace_bytes(&s) < 0 || (grad && tpf_xattn_backward_workspace_bytes(&s) < 0))
    return std::nullopt;
  if (grad) return XattnFn::apply(q, k, v, mask_in, kind, mask_stride, scale, sh == "1");
  return xattn_forward(q, k, v, mask, kind, mask_stride, scale, nullptr, nullptr);
}

// -------------------------------------------------------- norms and rotation

Tensor or_none(const std::optional<Tensor>& t) { return t.value_or(Tensor()); }

constexpr int64_t kMaxTokens = (1 << 26) - 32;  // of a launch

// Frequencies and weights as the kernels read them (D channels); nullopt-worthy ones are false.
bool rotation_plain(int64_t D, const std::optional<Tensor>& freq, const std::optional<Tensor>& qw,
                    const std::optional<Tensor>& kw, const std::optional<double>& eps,
                    c10::DeviceIndex dev) {
  if (freq && (!plain(*freq, dev) || freq->dim() != 1 || freq->numel() == 0 || 2 * freq->numel() > D ||
               freq->scalar_type() != at::kDouble || !freq->is_contiguous() || freq->requires_grad()))
    return false;
  if (eps ? !(*eps >= 0.0 && *eps < 1e30) : qw.has_value() || kw.has_value()) return false;
  for (const auto* w : {&qw, &kw})
    if (*w && (!plain(**w, dev) || (*w)->dim() != 1 || (*w)->size(0) != D || !(*w)->is_contiguous() ||
               type_code((*w)->scalar_type()) < 0))
      return false;
  return !(qw && kw) || qw->scalar_type() == kw->scalar_type();
}
at::ScalarType weight_type(const Tensor& qw, const Tensor& kw) {
  return qw.defined() ? qw.scalar_type() : kw.defined() ? kw.scalar_type() : at::kFloat;
}

// A new tensor in t's storage order, its channels contiguous.
Tensor rotary_like(const Tensor& t) {
  Tensor out = at::empty_like(t);
  return out.stride(3) == 1 ? out : at::empty(t.sizes(), t.options());
}

tpf_rotary_shape rotary_shape(const Tensor& q, const Tensor& k, const Tensor& out_q, const Tensor& out_k,
                              const Tensor& positions, const Tensor& freq, at::ScalarType wtype, bool norm,
                              bool interleaved) {
  tpf_rotary_shape s{};
  s.B = q.size(0); s.N = q.size(2); s.H = q.size(1); s.Hk = k.size(1); s.D = q.size(3);
  s.half = freq.defined() ? freq.numel() : 0;
  s.dtype = type_code(q.scalar_type());
  s.weight_dtype = type_code(wtype);
  s.norm = norm;
  s.interleaved = interleaved;
  s.position_bits = 64;
  if (positions.defined()) {
    s.position_bits = positions.scalar_type() == at::kLong ? 64 : 32;
    for (int i = 0; i < 2; ++i) s.position_stride[i] = positions.size(i) > 1 ? positions.stride(i) : 0;
  }
  strides3(q, s.q_stride);
  strides3(k, s.k_stride);
  strides3(out_q, s.out_q_stride);
  strides3(out_k, s.out_k_stride);
  return s;
}

variable_list rotary_forward(const Tensor& q, const Tensor& k, const Tensor& positions, const Tensor& freq,
                             const Tensor& qw, const Tensor& kw, const std::optional<double>& eps,
                             bool interleaved) {
  Tensor oq = rotary_like(q), ok = rotary_like(k);
  const tpf_rotary_shape s =
      rotary_shape(q, k, oq, ok, positions, freq, weight_type(qw, kw), eps.has_value(), interleaved);
  check(tpf_rotary_forward(cptr(q), cptr(k), cptr(positions), (const double*)cptr(freq), cptr(qw), cptr(kw),
                           eps.value_or(0.0), mptr(oq), mptr(ok), &s, stream()),
        "tpf_rotary_forward");
  return {oq, ok};
}

struct RotaryFn : torch::autograd::Function<RotaryFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k,
                               const std::optional<Tensor>& qw, const std::optional<Tensor>& kw,
                               const std::optional<Tensor>& positions, const std::optional<Tensor>& freq,
                               std::optional<double> eps, bool interleaved) {
    const Tensor p = or_none(positions), f = or_none(freq), wq = or_none(qw), wk = or_none(kw);
    variable_list out = rotary_forward(q, k, p, f, wq, wk, eps, interleaved);
    ctx->save_for_backward({eps ? q : Tensor(), eps ? k : Tensor(), p, f, wq, wk});
    ctx->saved_data["eps"] = eps.value_or(-1.0);
    ctx->saved_data["inter"] = interleaved;
    ctx->saved_data["want"] = (int64_t)((wq.defined() && wq.requires_grad() ? 1 : 0) |
                                        (wk.defined() && wk.requires_grad() ? 2 : 0));
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list sv = ctx->get_saved_variables();
    const Tensor &q = sv[0], &k = sv[1], &p = sv[2], &f = sv[3], &qw = sv[4], &kw = sv[5];
    const double eps = ctx->saved_data["eps"].toDouble();
    const int64_t want = ctx->saved_data["want"].toInt();
    Tensor dy[2], dx[2], dw[2];
    int64_t gs[6];
    for (int i = 0; i < 2; ++i) {
      const Tensor& g = grads[i];
      dy[i] = g.stride(3) == 1 || g.size(3) == 1 ? g : g.contiguous();
      dx[i] = rotary_like(sv[i].defined() ? sv[i] : dy[i]);
      strides3(dy[i], gs + 3 * i);
    }
    const auto wtype = weight_type(qw, kw);
    for (int i = 0; i < 2; ++i)
      if (want >> i & 1) dw[i] = at::empty({dx[0].size(3)}, like(dx[0], wtype));
    const tpf_rotary_shape s =
        rotary_shape(q.defined() ? q : dy[0], k.defined() ? k : dy[1], dx[0], dx[1], p, f, wtype, eps >= 0.0,
                     ctx->saved_data["inter"].toBool());
    const int64_t n = want ? tpf_rotary_backward_workspace_bytes(&s) : 0;
    const Tensor ws = bytes(dx[0], n);
    check(tpf_rotary_backward(cptr(q), cptr(k), cptr(dy[0]), cptr(dy[1]), cptr(p), (const double*)cptr(f),
                              cptr(qw), cptr(kw), eps >= 0.0 ? eps : 0.0, mptr(dx[0]), mptr(dx[1]),
                              mptr(dw[0]), mptr(dw[1]), mptr(ws), n, &s, gs, stream()),
          "tpf_rotary_backward");
    return once({dx[0], dx[1], dw[0], dw[1], Tensor(), Tensor(), Tensor(), Tensor()});
  }
};

std::optional<std::tuple<Tensor, Tensor>> qk_norm_rotary(
    const Tensor& q, const Tensor& k, const std::optional<Tensor>& positions_in,
    const std::optional<Tensor>& freq, const std::optional<Tensor>& qw, const std::optional<Tensor>& kw,
    std::optional<double> eps, bool interleaved) {
  if (transforms_active() || !q.is_cuda()) return std::nullopt;
  const c10::DeviceIndex dev = c10::hip::current_device();
  for (const Tensor* t : {&q, &k})
    if (!plain(*t, dev) || t->dim() != 4 || t->numel() == 0 || t->scalar_type() != q.scalar_type() ||
        t->stride(3) != 1)
      return std::nullopt;
  const int64_t B = q.size(0), N = q.size(2), D = q.size(3);
  if (type_code(q.scalar_type()) < 0 || k.size(0) != B || k.size(2) != N || k.size(3) != D || D > 256 ||
      q.size(1) > 65535 || k.size(1) > 65535 || B * N > kMaxTokens || !rotation_plain(D, freq, qw, kw, eps, dev))
    return std::nullopt;
  std::optional<Tensor> positions = positions_in;
  if (positions) {
    const auto pt = positions->scalar_type();
    if (!plain(*positions, dev) || (pt != at::kInt && pt != at::kLong) || !broadcasts(positions->sizes(), {B, N}))
      return std::nullopt;
    if (positions->dim() != 2 || positions->size(0) != B || positions->size(1) != N)
      positions = positions->expand({B, N});
  }
  bool grad = false;
  for (const Tensor* t : {&q, &k}) grad = grad || t->requires_grad();
  for (const auto* w : {&qw, &kw}) grad = grad || (*w && (*w)->requires_grad());
  const variable_list out =
      grad && at::GradMode::is_enabled()
          ? RotaryFn::apply(q, k, qw, kw, positions, freq, eps, interleaved)
          : rotary_forward(q, k, or_none(positions), or_none(freq), or_none(qw), or_none(kw), eps, interleaved);
  return std::make_tuple(out[0], out[1]);
}

// ---------------------------------------------------------- window attention

tpf_window_shape window_shape(const Tensor& q, const Tensor& k, const Tensor& v, int64_t mask_stride,
                              int64_t window, int64_t sinks) {
  tpf_window_shape s{q.size(0), q.size(1), k.size(1), q.size(2), q.size(3), type_code(q.scalar_type()),
                     window, sinks, mask_stride, {}, {}, {}};
  strides3(q, s.q_stride);
  strides3(k, s.k_stride);
  strides3(v, s.v_stride);
  return s;
}

Tensor window_forward(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& mask,
                      const tpf_window_shape& s, double scale, Tensor* lse, Tensor* res) {
  Tensor out = at::empty({s.B, s.N, s.H, s.D}, q.options());
  if (lse) *lse = at::empty({s.B, s.H, s.N}, like(q, at::kFloat));
  if (res) *res = at::empty_like(out);
  const int64_t n = tpf_window_forward_workspace_bytes(&s);
  const Tensor ws = bytes(q, n);
  check(tpf_window_forward(cptr(q), cptr(k), cptr(v), cptr(mask), out.data_ptr(),
                           lse ? (float*)lse->data_ptr() : nullptr, res ? res->data_ptr() : nullptr, mptr(ws), n,
                           &s, scale, stream()),
        "tpf_window_forward");
  return out;
}

struct WindowFn : torch::autograd::Function<WindowFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v,
                        const std::optional<Tensor>& mask_in, int64_t mask_stride, int64_t window,
                        int64_t sinks, double scale, bool shadow) {
    const Tensor mask = or_none(mask_in);
    Tensor lse, res;
    Tensor out = window_forward(q, k, v, mask, window_shape(q, k, v, mask_stride, window, sinks), scale, &lse,
                                shadow ? &res : nullptr);
    ctx->save_for_backward({q, k, v, mask, out, lse, res});
    ctx->saved_data["stride"] = mask_stride;
    ctx->saved_data["window"] = window;
    ctx->saved_data["sinks"] = sinks;
    ctx->saved_data["scale"] = scale;
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list sv = ctx->get_saved_variables();
    const Tensor &q = sv[0], &k = sv[1], &v = sv[2];
    const tpf_window_shape s =
        window_shape(q, k, v, ctx->saved_data["stride"].toInt(), ctx->saved_data["window"].toInt(),
                     ctx->saved_data["sinks"].toInt());
    const Tensor dout = kernel_grad(grads[0]);
    Tensor d[3] = {grad_like(q), grad_like(k), grad_like(v)};
    int64_t gs[9];
    for (int i = 0; i < 3; ++i) strides3(d[i], gs + 3 * i);
    const int64_t n = tpf_window_backward_workspace_bytes(&s);
    const Tensor ws = bytes(q, n < 16 ? 16 : n);
    check(tpf_window_backward_bf16(cptr(q), cptr(k), cptr(v), cptr(sv[3]), cptr(sv[4]), cptr(sv[6]), cptr(dout),
                                   (const float*)cptr(sv[5]), mptr(d[0]), mptr(d[1]), mptr(d[2]), mptr(ws), n,
                                   &s, gs, ctx->saved_data["scale"].toDouble(), stream()),
          "tpf_window_backward_bf16");
    return once({d[0], d[1], d[2], Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()});
  }
};

// window 0: none.  sh: the policy variable of the shadow residual (env_flag).
std::optional<Tensor> window_attention(const Tensor& q, const Tensor& k, const Tensor& v, int64_t window,
                                       int64_t sinks, const std::optional<Tensor>& mask,
                                       std::optional<double> scale_in, const std::string& sh) {
  if (transforms_active() || !q.is_cuda()) return std::nullopt;
  const c10::DeviceIndex dev = c10::hip::current_device();
  for (const Tensor* t : {&q, &k, &v})
    if (!plain(*t, dev) || t->dim() != 4 || t->numel() == 0 || t->scalar_type() != q.scalar_type())
      return std::nullopt;
  const auto type = q.scalar_type();
  const bool grad = at::GradMode::is_enabled() &&
                    (q.requires_grad() || k.requires_grad() || v.requires_grad());
  if (type != at::kBFloat16 && (type != at::kHalf || grad)) return std::nullopt;
  if (grad && sh != "0" && sh != "1") return std::nullopt;
  const int64_t B = q.size(0), N = q.size(2), D = q.size(3);
  if (k.sizes() != v.sizes() || k.size(0) != B || k.size(2) != N || k.size(3) != D || D % 8 || D > 128 ||
      q.size(1) % k.size(1))
    return std::nullopt;
  for (const Tensor* t : {&q, &k, &v})
    if (!xattn_operand(*t)) return std::nullopt;
  const double scale = scale_in ? *scale_in : 1.0 / std::sqrt((double)D);
  if (!(scale > 1e-30 && scale < 1e30)) return std::nullopt;
  int64_t mask_stride = 0;
  if (mask) {
    if (!plain(*mask, dev) || mask->scalar_type() != at::kBool || !mask->is_contiguous() || mask->dim() < 1 ||
        mask->dim() > 2 || mask->size(-1) != N ||
        (mask->dim() == 2 && mask->size(0) != B && mask->size(0) != 1))
      return std::nullopt;
    mask_stride = mask->dim() == 2 && mask->size(0) > 1 ? N : 0;
  }
  // Sizes that the launches do not hold (of the backward too, before the forward).
  const tpf_window_shape s = window_shape(q, k, v, mask_stride, window, sinks);
  if (tpf_window_forward_workspace_bytes(&s) < 0 || (grad && tpf_window_backward_workspace_bytes(&s) < 0))
    return std::nullopt;
  if (grad) return WindowFn::apply(q, k, v, mask, mask_stride, window, sinks, scale, sh == "1");
  return window_forward(q, k, v, or_none(mask), s, scale, nullptr, nullptr);
}

// -------------------------------------------------------------- paged cache

// The batch over a cache [pages, Hk, page, D] (checked when it was made) with T new tokens.
std::optional<tpf_paged_batch> paged_batch(const Tensor& ck, const Tensor& tables, const Tensor& starts,
                                           const Tensor& lengths, int64_t T, c10::DeviceIndex dev) {
  for (const Tensor* t : {&tables, &starts, &lengths})
    if (!plain(*t, dev) || t->scalar_type() != at::kInt || (t->numel() && t->stride(-1) != 1))
      return std::nullopt;
  if (tables.dim() != 2 || starts.dim() != 1 || lengths.dim() != 1) return std::nullopt;
  const int64_t S = lengths.size(0), width = tables.size(1);
  if (S < 1 || width < 1 || tables.size(0) != S || starts.size(0) != S + 1 || T < 1 || T > kMaxTokens ||
      width > (1 << 30) / ck.size(2))
    return std::nullopt;
  return tpf_paged_batch{(const int32_t*)cptr(tables), (const int32_t*)cptr(starts), (const int32_t*)cptr(lengths),
                         S, T, width, S > 1 ? tables.stride(0) : width, ck.size(2), ck.size(0)};
}
// New tokens [T, heads, D] of the cache's type that a call without gradients takes.
bool tokens_plain(const Tensor& t, const Tensor& ck, int64_t T, c10::DeviceIndex dev) {
  return plain(t, dev) && t.dim() == 3 && t.size(0) == T && t.size(1) > 0 && t.size(1) <= 65535 && t.size(2) == ck.size(3) &&
         t.scalar_type() == ck.scalar_type() && t.stride(2) == 1 &&
         !(t.requires_grad() && at::GradMode::is_enabled());
}
void strides2(const Tensor& t, int64_t* out) {
  for (int i = 0; i < 2; ++i) out[i] = t.size(i) > 1 ? t.stride(i) : 0;
}

std::optional<Tensor> append_kv(const Tensor& ck, const Tensor& cv, const Tensor& k, const Tensor& v,
                                const Tensor& tables, const Tensor& starts, const Tensor& lengths,
                                const std::optional<Tensor>& q, const std::optional<Tensor>& freq,
                                const std::optional<Tensor>& qw, const std::optional<Tensor>& kw,
                                std::optional<double> eps, bool interleaved) {
  if (transforms_active() || !k.is_cuda() || k.dim() != 3) return std::nullopt;
  const c10::DeviceIndex dev = c10::hip::current_device();
  const int64_t T = k.size(0), Hk = ck.size(1), D = ck.size(3);
  if (!plain(ck, dev) || !plain(cv, dev) || !tokens_plain(k, ck, T, dev) || !tokens_plain(v, ck, T, dev) ||
      k.size(1) != Hk || v.size(1) != Hk || (q && !tokens_plain(*q, ck, T, dev)) ||
      !rotation_plain(D, freq, qw, kw, eps, dev))
    return std::nullopt;
  for (const auto* w : {&qw, &kw})
    if (*w && (*w)->requires_grad() && at::GradMode::is_enabled()) return std::nullopt;
  const auto batch = paged_batch(ck, tables, starts, lengths, T, dev);
  if (!batch) return std::nullopt;
  const Tensor f = or_none(freq), wq = or_none(qw), wk = or_none(kw);
  const int64_t H = q ? q->size(1) : 0;
  Tensor out = at::empty({T, H, D}, k.options());
  tpf_append_shape s{H, Hk, D, f.defined() ? f.numel() : 0, type_code(k.scalar_type()),
                     type_code(weight_type(wq, wk)), eps.has_value(), interleaved, {}, {}, {}};
  if (q) strides2(*q, s.q_stride);
  strides2(k, s.k_stride);
  strides2(v, s.v_stride);
  check(tpf_paged_append(q ? cptr(*q) : nullptr, cptr(k), cptr(v), (const double*)cptr(f), cptr(wq), cptr(wk),
                         eps.value_or(0.0), out.data_ptr(), ck.data_ptr(), cv.data_ptr(), &s, &*batch, stream()),
        "tpf_paged_append");
  for (const Tensor* t : {&ck, &cv})
    if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
  return out;
}

// window 0: none.
std::optional<Tensor> paged_attention(const Tensor& q, const Tensor& ck, const Tensor& cv, const Tensor& tables,
                                      const Tensor& starts, const Tensor& lengths, int64_t window,
                                      int64_t sinks, std::optional<double> scale_in) {
  if (transforms_active() || !q.is_cuda() || q.dim() != 3) return std::nullopt;
  const c10::DeviceIndex dev = c10::hip::current_device();
  const int64_t T = q.size(0), Hk = ck.size(1), D = ck.size(3);
  if (!plain(ck, dev) || !plain(cv, dev) || !tokens_plain(q, ck, T, dev) || q.size(1) % Hk || !aligned16(q) ||
      (T > 1 && q.stride(0) % 8) || (q.size(1) > 1 && q.stride(1) % 8))
    return std::nullopt;
  const double scale = scale_in ? *scale_in : 1.0 / std::sqrt((double)D);
  if (!(scale > 1e-30 && scale < 1e30)) return std::nullopt;
  const auto batch = paged_batch(ck, tables, starts, lengths, T, dev);
  if (!batch) return std::nullopt;
  tpf_paged_shape s{q.size(1), Hk, D, type_code(q.scalar_type()), window, sinks, {}};
  strides2(q, s.q_stride);
  const int64_t n = tpf_paged_attention_workspace_bytes(&s, &*batch);
  if (n < 0) return std::nullopt;
  Tensor out = at::empty(q.sizes(), q.options());
  const Tensor ws = bytes(q, n);
  check(tpf_paged_attention(cptr(q), cptr(ck), cptr(cv), out.data_ptr(), mptr(ws), n, &s, &*batch, scale,
                            stream()),
        "tpf_paged_attention");
  return out;
}

// ---------------------------------------------------------------- layer norm

// Rows x2 [R, C]; what a backward needs of `keep` (0 nothing, 1 the rows, 2 the
// 8-bit form): mean, rstd, codes, scales.
Tensor norm_forward(const Tensor& x2, const Tensor& w, const Tensor& b, double eps, int keep,
                    Tensor* st) {
  const int64_t R = x2.size(0), C = x2.size(1), blocks = (C + 31) / 32;
  Tensor y = at::empty({R, C}, x2.options());
  if (keep == 1) st[0] = at::empty({R}, like(x2, at::kFloat));
  if (keep) st[1] = at::empty({R}, like(x2, at::kFloat));
  if (keep == 2) {
    st[2] = at::empty({R, blocks * 32}, like(x2, at::kByte));
    st[3] = at::empty({R, blocks}, like(x2, at::kByte));
  }
  const Tensor& p = w.defined() ? w : b;
  check(tpf_norm_forward(cptr(x2), R > 1 ? x2.stride(0) : C, R, C, type_code(x2.scalar_type()),
                         cptr(w), cptr(b), p.defined() ? type_code(p.scalar_type()) : 0, eps,
                         y.data_ptr(), (float*)mptr(st[0]), (float*)mptr(st[1]), mptr(st[2]),
                         mptr(st[3]), stream()),
        "tpf_norm_forward");
  return y;
}

struct NormFn : torch::autograd::Function<NormFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x2, const std::optional<Tensor>& weight,
                        const std::optional<Tensor>& bias, double eps, bool int8) {
    const Tensor w = weight.value_or(Tensor()), b = bias.value_or(Tensor());
    Tensor st[4];
    Tensor y = norm_forward(x2, w, b, eps, int8 ? 2 : 1, st);
    ctx->save_for_backward({int8 ? Tensor() : x2, st[0], st[1], st[2], st[3], w});
    ctx->saved_data["type"] = (int64_t)x2.scalar_type();
    ctx->saved_data["ptype"] =
        (int64_t)(w.defined() ? w.scalar_type() : b.defined() ? b.scalar_type() : at::kFloat);
    ctx->saved_data["want"] = (int64_t)((w.defined() && w.requires_grad() ? 1 : 0) |
                                        (b.defined() && b.requires_grad() ? 2 : 0));
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list s = ctx->get_saved_variables();
    const Tensor &x2 = s[0], &w = s[5];
    const auto type = (at::ScalarType)ctx->saved_data["type"].toInt();
    const auto ptype = (at::ScalarType)ctx->saved_data["ptype"].toInt();
    const int64_t want = ctx->saved_data["want"].toInt();
    const Tensor dy = grads[0].to(type).contiguous();
    const int64_t R = dy.size(0), C = dy.size(1);
    Tensor dx = at::empty({R, C}, dy.options()), dw, db, ws;
    if (want & 1) dw = at::empty({C}, like(dy, ptype));
    if (want & 2) db = at::empty({C}, like(dy, ptype));
    const int64_t n = want ? tpf_norm_backward_workspace_bytes(R, C) : 0;
    if (want) ws = bytes(dy, n);
    check(tpf_norm_backward(cptr(dy), cptr(x2), x2.defined() && R > 1 ? x2.stride(0) : C, cptr(s[3]),
                            cptr(s[4]), (const float*)cptr(s[1]), (const float*)cptr(s[2]), R, C,
                            type_code(type), cptr(w), type_code(ptype), dx.data_ptr(), C, mptr(dw),
                            mptr(db), mptr(ws), n, stream()),
          "tpf_norm_backward");
    return once({dx, dw, db, Tensor(), Tensor()});
  }
};

std::optional<Tensor> layer_norm(const Tensor& x, const std::optional<Tensor>& weight,
                                 const std::optional<Tensor>& bias, double eps, bool int8) {
  if (transforms_active() || !x.is_cuda()) return std::nullopt;
  const c10::DeviceIndex dev = c10::hip::current_device();
  if (!plain(x, dev) || x.dim() < 1 || x.numel() == 0 || type_code(x.scalar_type()) < 0 ||
      x.size(-1) > (1 << 24) || !(eps >= 0.0))
    return std::nullopt;
  const bool strided = x.dim() == 2 && x.stride(1) == 1;
  if (!strided && !x.is_contiguous()) return std::nullopt;
  const int64_t C = x.size(-1);
  const Tensor w = weight.value_or(Tensor()), b = bias.value_or(Tensor());
  for (const Tensor* p : {&w, &b})
    if (p->defined() && (!plain(*p, dev) || p->dim() != 1 || p->size(0) != C || !p->is_contiguous() ||
                         type_code(p->scalar_type()) < 0))
      return std::nullopt;
  if (w.defined() && b.defined() && w.scalar_type() != b.scalar_type()) return std::nullopt;
  const Tensor x2 = x.dim() == 2 ? x : x.view({-1, C});
  const bool grad = at::GradMode::is_enabled() &&
                    (x.requires_grad() || (w.defined() && w.requires_grad()) ||
                     (b.defined() && b.requires_grad()));
  Tensor st[4];
  const Tensor y = grad ? NormFn::apply(x2, weight, bias, eps, int8) : norm_forward(x2, w, b, eps, 0, st);
  return x.dim() == 2 ? y : y.view(x.sizes());
}

// ------------------------------------------------------- activations in 8 bits

std::optional<std::tuple<Tensor, Tensor>> act8_pack(const Tensor& x) {
  if (transforms_active() || !x.is_cuda()) return std::nullopt;
  if (!plain(x, c10::hip::current_device()) || x.dim() < 1 || x.numel() == 0 ||
      type_code(x.scalar_type()) < 0 || x.size(-1) > (1 << 24) ||
      !(x.is_contiguous() || (x.dim() == 2 && x.stride(1) == 1)))
    return std::nullopt;
  const int64_t C = x.size(-1), R = x.numel() / C, blocks = (C + 31) / 32;
  Tensor codes = at::empty({R, blocks * 32}, like(x, at::kByte));
  Tensor scales = at::empty({R, blocks}, like(x, at::kByte));
  check(tpf_act8_pack(cptr(x), x.dim() == 2 && R > 1 ? x.stride(0) : C, R, C,
                      type_code(x.scalar_type()), mptr(codes), mptr(scales), stream()),
        "tpf_act8_pack");
  return std::make_tuple(codes, scales);
}

std::optional<Tensor> act8_unpack(const Tensor& codes, const Tensor& scales,
                                  const std::vector<int64_t>& shape, at::ScalarType dtype) {
  const c10::DeviceIndex dev = c10::hip::current_device();
  if (transforms_active() || !plain(codes, dev) || !plain(scales, dev) || shape.empty() ||
      codes.numel() == 0 || type_code(dtype) < 0)
    return std::nullopt;
  const int64_t C = shape.back(), R = codes.size(0), blocks = (C + 31) / 32;
  if (C < 1 || c10::multiply_integers(shape) != R * C || codes.dim() != 2 || scales.dim() != 2 ||
      codes.scalar_type() != at::kByte || scales.scalar_type() != at::kByte ||
      codes.size(1) != 32 * blocks || scales.size(0) != R || scales.size(1) != blocks ||
      !codes.is_contiguous() || !scales.is_contiguous())
    return std::nullopt;
  Tensor out = at::empty(shape, like(codes, dtype));
  check(tpf_act8_unpack(cptr(codes), cptr(scales), R, C, out.data_ptr(), C, type_code(dtype), stream()),
        "tpf_act8_unpack");
  return out;
}

// -------------------------------------------------------------------- linear

// a [R, K] times b^T (b_kc: b [N, K]) or b [K, N], contiguous BF16.
Tensor row_gemm(const Tensor& a, const Tensor& b, bool b_kc) {
  const int64_t R = a.size(0), K = a.size(1), N = b_kc ? b.size(0) : b.size(1);
  Tensor out = at::empty({R, N}, a.options());
  check(tpf_row_gemm_bf16(cptr(a), K, cptr(b), b_kc ? 1 : 0, out.data_ptr(), R, N, K, stream()),
        "tpf_row_gemm_bf16");
  return out;
}

struct LinearFn : torch::autograd::Function<LinearFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w) {
    const int64_t R = x.size(0), K = x.size(1), blocks = (K + 31) / 32;
    Tensor codes, scales;
    if (w.requires_grad()) {
      codes = at::empty({R, blocks * 32}, like(x, at::kByte));
      scales = at::empty({R, blocks}, like(x, at::kByte));
      check(tpf_act8_pack(cptr(x), K, R, K, TPF_BF16, mptr(codes), mptr(scales), stream()),
            "tpf_act8_pack");
    }
    ctx->save_for_backward({w, codes, scales});
    ctx->saved_data["dx"] = x.requires_grad();
    return row_gemm(x, w, true);
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list s = ctx->get_saved_variables();
    const Tensor& w = s[0];
    const Tensor dy = kernel_grad(grads[0]);
    const int64_t R = dy.size(0), N = w.size(0), K = w.size(1);
    Tensor dx, dw;
    if (ctx->saved_data["dx"].toBool()) dx = row_gemm(dy, w, false);
    if (s[1].defined()) {
      dw = at::empty({N, K}, w.options());
      const int64_t n = tpf_wgrad_act8_workspace_bytes(R, N, K, N);
      const Tensor ws = bytes(dy, n);
      check(tpf_wgrad_act8(cptr(dy), N, cptr(s[1]), cptr(s[2]), R, N, K, dw.data_ptr(), TPF_BF16,
                           mptr(ws), n < 0 ? 0 : n, stream()),
            "tpf_wgrad_act8");
    }
    return once({dx, dw});
  }
};

// BF16 input and weight, the input kept in 8 bits.
std::optional<Tensor> linear(const Tensor& x, const Tensor& w) {
  if (transforms_active() || !x.is_cuda()) return std::nullopt;
  const c10::DeviceIndex dev = c10::hip::current_device();
  for (const Tensor* t : {&x, &w})
    if (!plain(*t, dev) || t->scalar_type() != at::kBFloat16 || t->numel() == 0 ||
        !t->is_contiguous() || !aligned16(*t))
      return std::nullopt;
  if (x.dim() < 1 || w.dim() != 2 || w.size(1) != x.size(-1)) return std::nullopt;
  const int64_t N = w.size(0), K = w.size(1), R = x.numel() / K, most = (int64_t(1) << 30) - 1;
  const int64_t wide = N > K ? N : K;
  if (N % 8 || K % 8 || wide > (1 << 23) || R > most / wide || N > most / K) return std::nullopt;
  const Tensor x2 = x.dim() == 2 ? x : x.view({R, K});
  const bool grad = at::GradMode::is_enabled() && (x.requires_grad() || w.requires_grad());
  const Tensor y = grad ? LinearFn::apply(x2, w) : row_gemm(x2, w, true);
  if (x.dim() == 2) return y;
  std::vector<int64_t> shape = x.sizes().vec();
  shape.back() = N;
  return y.view(shape);
}

}  // namespace

// Refuses the import beside another torch or C-ABI library than it was built
// with: both are called through their headers of that time.
void check_versions() {
  const auto torch = pybind11::module_::import("torch").attr("__version__").cast<std::string>();
  const std::string built = TORCH_VERSION;
  if (torch.compare(0, built.size(), built) != 0 ||
      (torch.size() > built.size() && std::isdigit((unsigned char)torch[built.size()])))
    throw pybind11::import_error("built for torch " + built + ", found " + torch);
  if (tpf_abi_version() != TPF_ABI_VERSION)
    throw pybind11::import_error("built for library ABI " + std::to_string(TPF_ABI_VERSION) +
                                 ", found " + std::to_string(tpf_abi_version()));
}

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  check_versions();
  m.def("attention", [](const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& res_mask,
                        const Tensor& pair_bias) {
    const std::string backward = env_flag("TURBOPAIRFORMER_SR_BACKWARD", "OPENFOLD3_SR_BACKWARD");
    const std::string shadow = env_flag("TURBOPAIRFORMER_SR_SHADOW", "OPENFOLD3_SR_SHADOW");
    pybind11::gil_scoped_release nogil;
    return attention(q, k, v, res_mask, pair_bias, backward, shadow);
  });
  m.def("trimul", &trimul, pybind11::call_guard<pybind11::gil_scoped_release>());
  m.def("cross_attention", [](const Tensor& q, const Tensor& k, const Tensor& v,
                              const std::optional<Tensor>& mask, std::optional<double> scale) {
    const std::string shadow = env_flag("TURBOPAIRFORMER_SR_SHADOW", "OPENFOLD3_SR_SHADOW");
    pybind11::gil_scoped_release nogil;
    return cross_attention(q, k, v, mask, scale, shadow);
  });
  m.def("window_attention", [](const Tensor& q, const Tensor& k, const Tensor& v, int64_t window,
                               int64_t sinks, const std::optional<Tensor>& mask,
                               std::optional<double> scale) {
    const std::string shadow = env_flag("TURBOPAIRFORMER_SR_SHADOW", "OPENFOLD3_SR_SHADOW");
    pybind11::gil_scoped_release nogil;
    return window_attention(q, k, v, window, sinks, mask, scale, shadow);
  });
  m.def("qk_norm_rotary", &qk_norm_rotary, pybind11::call_guard<pybind11::gil_scoped_release>());
  m.def("append_kv", &append_kv, pybind11::call_guard<pybind11::gil_scoped_release>());
  m.def("paged_attention", &paged_attention, pybind11::call_guard<pybind11::gil_scoped_release>());
  m.def("layer_norm", &layer_norm, pybind11::call_guard<pybind11::gil_scoped_release>());
  m.def("act8_pack", &act8_pack, pybind11::call_guard<pybind11::gil_scoped_release>());
  m.def("act8_unpack", &act8_unpack, pybind11::call_guard<pybind11::gil_scoped_release>());
  m.def("linear", &linear, pybind11::call_guard<pybind11::gil_scoped_release>());
  m.def("set_workspace_budget", [](int64_t bytes) { g_budget.store(bytes); });
}
