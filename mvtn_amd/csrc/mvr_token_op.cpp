// mvtn_amd/_mvr_token_op.so — host side of mvtn_amd/tokens.py: the operators on view tokens as torch operators with C++ autograd nodes,
// so that a call crosses from Python once and its backward runs on the autograd engine's thread without the interpreter lock (as Python
// autograd functions over ctypes, a forward and backward cost 110-160 us of host time, against 35-130 us on the GPU).
//
// Argument checks, allocation and the calls of the C ABI (include/mvr.h); no arithmetic.  The entry points' addresses are handed over
// by mvtn_amd/_lib.py: this file does not link against libmvr_hip.so, and that library stays free of torch types.  (libc10_hip: torch's current stream.)  What Python sees: ValueError
// for arguments that do not fit, RuntimeError for tensors that are not on the GPU and for errors of the library.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/library.h>

#include <cmath>
#include <cstring>
#include <vector>

#include "../../include/mvr.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef c10::optional<Tensor> MaybeTensor;

struct Entry {
  decltype(&mvr_rotate_tokens_forward) rotate = nullptr;
  decltype(&mvr_rotate_tokens_backward) rotate_backward = nullptr;
  decltype(&mvr_attend_tokens_workspace_bytes) attend_bytes = nullptr;
  decltype(&mvr_attend_tokens_forward_rest) attend = nullptr;
  decltype(&mvr_attend_tokens_backward_rest) attend_backward = nullptr;
  decltype(&mvr_add_norm_tokens_workspace_bytes) norm_bytes = nullptr;
  decltype(&mvr_add_norm_tokens_forward) norm = nullptr;
  decltype(&mvr_add_norm_tokens_backward) norm_backward = nullptr;
  decltype(&mvr_last_error) last_error = nullptr;
} g_entry;

void init(std::vector<int64_t> a) {
  TORCH_CHECK(a.size() * sizeof(void *) == sizeof(Entry), "mvr_tokens::init: ", sizeof(Entry) / sizeof(void *), " entry points expected");
  for (size_t k = 0; k < a.size(); ++k) std::memcpy(reinterpret_cast<char *>(&g_entry) + k * sizeof(void *), &a[k], sizeof(void *));
}

void check(int rc, const char *what) {
  if (rc == MVR_OK) return;
  const char *msg = g_entry.last_error ? g_entry.last_error() : nullptr;
  TORCH_CHECK(false, "mvr ", what, " failed (code ", rc, "): ", msg ? msg : "");
}

int type_of(const Tensor &t) {
  switch (t.scalar_type()) {
    case at::kFloat: return MVR_TYPE_FLOAT;
    case at::kHalf: return MVR_TYPE_HALF;
    case at::kBFloat16: return MVR_TYPE_BFLOAT;
    default: return -1;
  }
}

void same_device(const Tensor &first, std::initializer_list<const Tensor *> others) {
  TORCH_CHECK(first.is_cuda(), "mvtn_amd: tensors must live on the GPU (the HIP library is the only path; there is no CPU fallback)");
  for (const Tensor *t : others) {
    if (!t->defined()) continue;
    TORCH_CHECK(t->is_cuda(), "mvtn_amd: tensors must live on the GPU (the HIP library is the only path; there is no CPU fallback)");
    TORCH_CHECK(t->device() == first.device(), "mvtn_amd.tokens: all tensors must be on one GPU (", first.device(), " and ", t->device(), ")");
  }
}

void *ptr(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
float *fptr(const Tensor &t) { return t.defined() ? t.data_ptr<float>() : nullptr; }
Tensor or_none(const MaybeTensor &t) { return t.has_value() ? *t : Tensor(); }
MaybeTensor some(const Tensor &t) { return t.defined() ? MaybeTensor(t) : MaybeTensor(); }
Tensor packed(const Tensor &t) { return t.defined() ? t.contiguous() : t; }
// the last dimension's elements side by side (a copy only where they are not)
Tensor rows_packed(const Tensor &t) { return t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous(); }
bool wants_grad(std::initializer_list<const Tensor *> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor *t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}
// tangents would be dropped, the result's derivative taken for 0
void no_forward_mode(std::initializer_list<const Tensor *> ts) {
  for (const Tensor *t : ts)
    TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(/*level=*/0).defined(),
                                "mvtn_amd.tokens: these operators have no forward-mode derivative (the reverse mode has all of them)");
}
bool in_32_bits(const Tensor &t) {   // the C ABI's sizes
  for (int64_t n : t.sizes())
    if (n > 0x7FFFFFFF) return false;
  return true;
}
void strides(int64_t (&to)[3], const Tensor &t) {
  for (int k = 0; k < 3; ++k) to[k] = t.stride(k);
}
// the stream that is current on the tensor's GPU when the work is issued (in a backward: the forward's, as the engine makes it current)
mvr_stream_t stream_of(const Tensor &t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

// A gradient that somebody asks to differentiate again fails there, and not silently.  again: it depends on inputs that require grad, not on the
// incoming gradients alone
variable_list once(variable_list out, const variable_list &grads, bool again) {
  for (const Tensor &g : grads) again = again || (g.defined() && g.requires_grad());
  if (!at::GradMode::is_enabled() || !again) return out;
  variable_list in;
  for (Tensor &t : out) in.push_back(t.defined() ? t.detach().requires_grad_(true) : t);
  auto error = std::make_shared<torch::autograd::DelayedError>("mvtn_amd.tokens: the gradients of these operators cannot be differentiated again", (int64_t)in.size());
  return (*error)(std::move(in));
}

// ---- rotary positions -------------------------------------------------------------------------------------------------

mvr_rotary_params rotary_params(const Tensor &x, const Tensor &grad, const Tensor &positions, at::IntArrayRef sections, bool interleaved) {
  mvr_rotary_params p;
  std::memset(&p, 0, sizeof(p));
  p.batch = (int32_t)x.size(0), p.tokens = (int32_t)x.size(1), p.heads = (int32_t)x.size(2), p.dim = (int32_t)x.size(3);
  p.type = type_of(x), p.axes = (int32_t)sections.size(), p.interleaved = interleaved;
  for (size_t k = 0; k < sections.size(); ++k) p.sections[k] = (int32_t)sections[k];
  strides(p.x_stride, x);
  if (grad.defined()) strides(p.grad_stride, grad);
  p.position_stride[0] = positions.stride(0), p.position_stride[1] = positions.stride(1);
  return p;
}

Tensor rotate_forward(const Tensor &x_, const Tensor &positions_, const Tensor &turns, at::IntArrayRef sections, bool interleaved) {
  const c10::DeviceGuard guard(x_.device());
  Tensor out = at::empty(x_.sizes(), x_.options());
  if (out.numel() == 0) return out;
  const Tensor x = rows_packed(x_), positions = rows_packed(positions_);
  const mvr_rotary_params p = rotary_params(x, Tensor(), positions, sections, interleaved);
  check(g_entry.rotate(&p, turns.data_ptr<double>(), x.data_ptr(), positions.data_ptr<float>(), out.data_ptr(), stream_of(x)), "mvr_rotate_tokens_forward");
  return out;
}

struct Rotate : public torch::autograd::Function<Rotate> {
  static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &positions, const Tensor &turns, std::vector<int64_t> sections, bool interleaved) {
    Tensor out = rotate_forward(x, positions, turns, sections, interleaved);
    ctx->save_for_backward({positions.requires_grad() ? x : Tensor(), positions, turns});
    ctx->saved_data["sections"] = sections;
    ctx->saved_data["interleaved"] = interleaved;
    return out;
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor grad = rows_packed(grads[0]), positions = rows_packed(saved[1]), &turns = saved[2];
    const Tensor x = saved[0].defined() ? rows_packed(saved[0]) : Tensor();
    const c10::DeviceGuard guard(grad.device());
    Tensor gx = at::empty(grad.sizes(), grad.options()), gp;
    if (x.defined()) gp = at::empty(positions.sizes(), positions.options());
    if (gx.numel()) {
      const auto sections = ctx->saved_data["sections"].toIntVector();
      const mvr_rotary_params p = rotary_params(x.defined() ? x : grad, grad, positions, sections, ctx->saved_data["interleaved"].toBool());
      check(g_entry.rotate_backward(&p, turns.data_ptr<double>(), ptr(x), positions.data_ptr<float>(), grad.data_ptr(), gx.data_ptr(), fptr(gp), stream_of(grad)),
            "mvr_rotate_tokens_backward");
    } else if (gp.defined()) {
      gp.zero_();
    }
    return once({gx, gp, Tensor(), Tensor(), Tensor()}, grads, x.defined());   // (without the positions' a gradient is linear in dy)
  }
};

Tensor rotate_tokens(const Tensor &x, const Tensor &positions_, const Tensor &turns, std::vector<int64_t> sections, bool interleaved) {
  TORCH_CHECK_VALUE(x.dim() == 4, "x is (B, L, H, D)");
  const int64_t B = x.size(0), L = x.size(1), D = x.size(3), pairs = turns.numel(), axes = (int64_t)sections.size();
  TORCH_CHECK_VALUE(type_of(x) >= 0, "x must be float32, float16 or bfloat16, not ", x.scalar_type());
  TORCH_CHECK_VALUE(2 * pairs <= D && D <= 256 && !(interleaved && D % 2), pairs, " pairs do not fit a head of ", D, " (at most 256, even when interleaved)");
  TORCH_CHECK_VALUE(in_32_bits(x), "every size of x must be below 2^31");
  const int64_t dims = positions_.dim();
  TORCH_CHECK_VALUE((dims == 2 || dims == 3) && positions_.size(-2) == L && positions_.size(-1) == axes && (dims == 2 || positions_.size(0) == 1 || positions_.size(0) == B),
                    "positions are (B, L, axes), (1, L, axes) or (L, axes) with L = ", L, " and ", axes, " axes");
  no_forward_mode({&x, &positions_});
  same_device(x, {&positions_});
  const Tensor positions = positions_.to(at::kFloat).expand({B, L, axes});
  if (wants_grad({&x, &positions})) return Rotate::apply(x, positions, turns, sections, interleaved);
  return rotate_forward(x, positions, turns, sections, interleaved);
}

// ---- attention ---------------------------------------------------------------------------------------------------------

mvr_attend_params attend_params(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &keep, const Tensor &grad, double scale) {
  mvr_attend_params p;
  std::memset(&p, 0, sizeof(p));
  p.batch = (int32_t)q.size(0), p.queries = (int32_t)q.size(1), p.keys = (int32_t)k.size(1), p.heads = (int32_t)q.size(2), p.kv_heads = (int32_t)k.size(2);
  p.dim = (int32_t)q.size(3), p.type = type_of(q), p.keep_groups = keep.defined() ? (int32_t)keep.size(1) : 0, p.scale = (float)scale;
  strides(p.q_stride, q), strides(p.k_stride, k), strides(p.v_stride, v);
  if (grad.defined()) strides(p.grad_stride, grad);
  return p;
}

Tensor workspace(size_t bytes, const Tensor &like) { return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : Tensor(); }

// q, k, v with packed rows; rest, lse: undefined where no backward follows
Tensor attend_forward(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &keep, double scale, const Tensor &rest, const Tensor &lse) {
  Tensor out = at::empty(q.sizes(), q.options());
  if (k.size(1) == 0) return out.zero_();
  if (out.numel() == 0) return out;
  const mvr_attend_params p = attend_params(q, k, v, keep, Tensor(), scale);
  const size_t bytes = g_entry.attend_bytes(&p, 0);
  const Tensor ws = workspace(bytes, q);
  check(g_entry.attend(&p, q.data_ptr(), k.data_ptr(), v.data_ptr(), (const uint8_t *)ptr(keep), out.data_ptr(), ptr(rest), fptr(lse), ptr(ws), bytes, stream_of(q)),
        "mvr_attend_tokens_forward");
  return out;
}

struct Attend : public torch::autograd::Function<Attend> {
  static Tensor forward(AutogradContext *ctx, const Tensor &q_, const Tensor &k_, const Tensor &v_, const MaybeTensor &keep_, double scale) {
    const Tensor keep = or_none(keep_);
    const c10::DeviceGuard guard(q_.device());
    const Tensor q = rows_packed(q_), k = rows_packed(k_), v = rows_packed(v_);
    const Tensor lse = at::empty({q.size(0), q.size(2), q.size(1)}, q.options().dtype(at::kFloat));
    const Tensor rest = k.size(1) > 64 ? at::empty(q.sizes(), q.options()) : Tensor();   // (over so few keys the backward does without)
    Tensor out = attend_forward(q, k, v, keep, scale, rest, lse);
    ctx->save_for_backward({q, k, v, keep, out, lse, rest});
    ctx->saved_data["scale"] = scale;
    return out;
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    const Tensor &q = s[0], &k = s[1], &v = s[2], &keep = s[3], &out = s[4], &lse = s[5], &rest = s[6];
    const c10::DeviceGuard guard(q.device());
    Tensor gq = at::empty(q.sizes(), q.options()), gk = at::empty(k.sizes(), k.options()), gv = at::empty(v.sizes(), v.options());
    if (out.numel() && k.size(1)) {
      const Tensor grad = rows_packed(grads[0]);
      const mvr_attend_params p = attend_params(q, k, v, keep, grad, ctx->saved_data["scale"].toDouble());
      const size_t bytes = g_entry.attend_bytes(&p, 1);
      const Tensor ws = workspace(bytes, q);
      check(g_entry.attend_backward(&p, q.data_ptr(), k.data_ptr(), v.data_ptr(), (const uint8_t *)ptr(keep), out.data_ptr(), ptr(rest), lse.data_ptr<float>(),
                                    grad.data_ptr(), gq.data_ptr(), gk.data_ptr(), gv.data_ptr(), ptr(ws), bytes, stream_of(q)),
            "mvr_attend_tokens_backward");
    } else {
      gq.zero_(), gk.zero_(), gv.zero_();
    }
    return once({gq, gk, gv, Tensor(), Tensor()}, grads, q.requires_grad() || k.requires_grad());   // (v's alone is linear in dO)
  }
};

Tensor attend_tokens(const Tensor &q, const Tensor &k, const Tensor &v, const MaybeTensor &keep_, const c10::optional<double> &scale_) {
  TORCH_CHECK_VALUE(q.dim() == 4 && k.dim() == 4 && k.sizes() == v.sizes(), "q is (B, Lq, H, D), k and v are (B, Lk, Hkv, D)");
  const int64_t B = q.size(0), H = q.size(2), D = q.size(3), Lk = k.size(1), E = k.size(2);
  TORCH_CHECK_VALUE(k.size(0) == B && k.size(3) == D && D >= 1 && D <= 128, "q, k and v share the batch and a head size of 1 to 128");
  TORCH_CHECK_VALUE(E >= 1 && H >= 1 && H % E == 0, H, " heads are not a multiple of ", E, " key/value heads");
  TORCH_CHECK_VALUE((q.scalar_type() == at::kHalf || q.scalar_type() == at::kBFloat16) && k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(),
                    "q, k and v share one type of float16, bfloat16");
  TORCH_CHECK_VALUE(in_32_bits(q) && in_32_bits(k), "every size of q, k and v must be below 2^31");
  const double scale = scale_.has_value() ? *scale_ : 1.0 / std::sqrt((double)D);
  TORCH_CHECK_VALUE((float)scale > 0 && std::isfinite((float)scale), "scale must be positive and finite, in 32 bits too");
  Tensor keep = or_none(keep_);
  if (keep.defined()) {
    TORCH_CHECK_VALUE(keep.dim() == 2 && keep.size(0) == B && keep.size(1) >= 1 && Lk % keep.size(1) == 0, "keep is (B, G) with G a divisor of the ", Lk, " keys");
    TORCH_CHECK_VALUE(!keep.requires_grad(), "keep is a mask: it gets no gradient");
  }
  no_forward_mode({&q, &k, &v});
  same_device(q, {&k, &v, &keep});
  if (keep.defined()) keep = (keep.scalar_type() == at::kBool || keep.scalar_type() == at::kByte ? keep : keep.ne(0)).contiguous();
  if (wants_grad({&q, &k, &v})) return Attend::apply(q, k, v, some(keep), scale);
  const c10::DeviceGuard guard(q.device());
  return attend_forward(rows_packed(q), rows_packed(k), rows_packed(v), keep, scale, Tensor(), Tensor());
}

// ---- norms around a block ----------------------------------------------------------------------------------------------

struct Norm {
  Tensor residual, branch, weight, bias, post, gate, draws;
};

Tensor norm_forward(const mvr_norm_params &p, const Norm &t, Tensor &y, Tensor &z, bool training) {
  y = at::empty(t.residual.sizes(), t.residual.options()), z = at::empty(t.branch.sizes(), t.branch.options());
  const Tensor stats = training ? at::empty({p.rows, 4}, y.options().dtype(at::kFloat)) : Tensor();
  if (p.rows)
    check(g_entry.norm(&p, t.residual.data_ptr(), t.branch.data_ptr(), t.weight.data_ptr(), ptr(t.bias), ptr(t.post), ptr(t.gate), fptr(t.draws), y.data_ptr(),
                       z.data_ptr(), fptr(stats), stream_of(t.residual)),
          "mvr_add_norm_tokens_forward");
  return stats;
}

struct AddNorm : public torch::autograd::Function<AddNorm> {
  static variable_list forward(AutogradContext *ctx, const Tensor &residual, const Tensor &branch, const Tensor &weight, const MaybeTensor &bias_,
                               const MaybeTensor &post_, const MaybeTensor &gate_, const MaybeTensor &draws_, const std::string &params) {
    const Tensor bias = or_none(bias_), post = or_none(post_), gate = or_none(gate_), draws = or_none(draws_);
    mvr_norm_params p;
    std::memcpy(&p, params.data(), sizeof(p));
    const c10::DeviceGuard guard(residual.device());
    const Norm t{packed(residual), packed(branch), packed(weight), packed(bias), packed(post), packed(gate), draws};
    Tensor y, z;
    const Tensor stats = norm_forward(p, t, y, z, true);
    ctx->set_materialize_grads(false);
    // (y in 32 bits is what the backward needs; in 16 bits it would bring its rounding along, and the backward forms it again)
    ctx->save_for_backward({p.residual_type == MVR_TYPE_FLOAT ? y : t.residual, t.branch, t.weight, t.post, t.gate, draws, stats});
    ctx->saved_data["params"] = params;
    ctx->saved_data["need"] = std::vector<int64_t>{weight.requires_grad(), bias.defined() && bias.requires_grad(), post.defined() && post.requires_grad(),
                                                   gate.defined() && gate.requires_grad(),
                                                   // (weight's and bias' alone are linear in dz)
                                                   residual.requires_grad() || branch.requires_grad() || (post.defined() && post.requires_grad()) || (gate.defined() && gate.requires_grad())};
    return {y, z};
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    variable_list none(8);
    if (!grads[0].defined() && !grads[1].defined()) return none;
    const auto s = ctx->get_saved_variables();
    const Tensor &y = s[0] /* or the residual */, &branch = s[1], &weight = s[2], &post = s[3], &gate = s[4], &draws = s[5], &stats = s[6];
    const auto need = ctx->saved_data["need"].toIntVector();
    mvr_norm_params p;
    std::memcpy(&p, ctx->saved_data["params"].toStringRef().data(), sizeof(p));
    const c10::DeviceGuard guard(y.device());
    const Tensor gy = packed(grads[0]), gz = packed(grads[1]);
    const auto like = [](const Tensor &t, bool want) { return want ? at::empty(t.sizes(), t.options()) : Tensor(); };
    const Tensor gr = like(y, true), gb = like(branch, true), gw = like(weight, need[0]), gbias = like(weight, need[1]), gpost = like(post, need[2]),
                 ggate = like(gate, need[3]);
    if (p.rows) {
      const size_t bytes = need[0] || need[1] || need[2] || need[3] ? g_entry.norm_bytes(&p) : 0;
      const Tensor ws = workspace(bytes, y);
      check(g_entry.norm_backward(&p, y.data_ptr(), branch.data_ptr(), weight.data_ptr(), ptr(post), ptr(gate), fptr(draws), stats.data_ptr<float>(), ptr(gy), ptr(gz),
                                  gr.data_ptr(), gb.data_ptr(), ptr(gw), ptr(gbias), ptr(gpost), ptr(ggate), ptr(ws), bytes, stream_of(y)),
            "mvr_add_norm_tokens_backward");
    } else {
      for (const Tensor *t : {&gw, &gbias, &gpost, &ggate})
        if (t->defined()) t->zero_();
    }
    return once({gr, gb, gw, gbias, gpost, ggate, Tensor(), Tensor()}, grads, need[4]);
  }
};

std::vector<Tensor> add_norm_tokens(const Tensor &residual, const Tensor &branch, const Tensor &weight, const MaybeTensor &bias_, const MaybeTensor &post_,
                                    const MaybeTensor &gate_, const MaybeTensor &draws_, double number, bool layer, double eps) {
  const Tensor bias = or_none(bias_), post = or_none(post_), gate = or_none(gate_);
  Tensor draws = or_none(draws_);
  TORCH_CHECK_VALUE(residual.sizes() == branch.sizes() && residual.dim() >= 2, "residual and branch are of one shape (..., D)");
  const int64_t dims = residual.dim(), D = residual.size(-1);
  TORCH_CHECK_VALUE(D >= 1 && D <= 8192, "rows of 1 to 8192 elements");
  const int r = type_of(residual), b = type_of(branch);
  TORCH_CHECK_VALUE(r >= 0 && b >= 0 && (r == b || r == MVR_TYPE_FLOAT), "residual and branch share one type of float32, float16, bfloat16, or the residual is float32");
  TORCH_CHECK_VALUE(eps >= 0 && std::isfinite(eps), "eps must not be negative");
  for (const Tensor *t : {&weight, &bias, &post})
    TORCH_CHECK_VALUE(!t->defined() || (t->dim() == 1 && t->size(0) == D), "weight, bias and post_weight are (", D, ",)");
  const int64_t rows = residual.numel() / D;
  int64_t groups = 0;
  if (gate.defined()) {
    // one row per leading index, trailing ones left out
    int64_t lead = gate.dim() - 1;
    while (lead > 0 && gate.size(lead - 1) == 1) --lead;
    bool fits = gate.dim() >= 1 && gate.size(-1) == D && gate.dim() <= dims && (lead == 0 || lead < dims - 1);
    groups = 1;
    for (int64_t k = 0; fits && k < lead; ++k) fits = gate.size(k) == residual.size(k), groups *= gate.size(k);
    TORCH_CHECK_VALUE(fits, "gate is (D,), or has one row per leading index of the residual ((B, D) or (B, 1, D) for (B, L, D)); a gate of every element belongs into the branch");
    TORCH_CHECK_VALUE(groups <= 65000, "at most 65000 rows of gates");
  }
  for (const Tensor *t : {&weight, &bias, &post, &gate})
    TORCH_CHECK_VALUE(!t->defined() || (t->scalar_type() == weight.scalar_type() && type_of(*t) >= 0), "weight, bias, post_weight and gate share one type of float32, float16, bfloat16");
  if (draws.defined()) {
    TORCH_CHECK_VALUE(!draws.requires_grad(), "scale holds draws: it gets no gradient (put what is learned into gate)");
    TORCH_CHECK_VALUE(draws.numel() >= 1 && rows % draws.numel() == 0, "scale has ", draws.numel(), " draws, which do not divide the ", rows, " rows");
  }
  no_forward_mode({&residual, &branch, &weight, &bias, &post, &gate});
  same_device(residual, {&branch, &weight, &bias, &post, &gate, &draws});
  if (draws.defined()) draws = draws.to(at::kFloat).contiguous();
  mvr_norm_params p;
  std::memset(&p, 0, sizeof(p));
  p.rows = rows, p.dim = (int32_t)D, p.residual_type = r, p.branch_type = b, p.param_type = type_of(weight), p.kind = layer;
  p.gate_groups = groups, p.scale_groups = draws.defined() ? draws.numel() : 0, p.scale = (float)number, p.eps = (float)eps;
  if (wants_grad({&residual, &branch, &weight, &bias, &post, &gate}))
    return AddNorm::apply(residual, branch, weight, some(bias), some(post), some(gate), some(draws), std::string(reinterpret_cast<const char *>(&p), sizeof(p)));
  const c10::DeviceGuard guard(residual.device());
  Tensor y, z;
  norm_forward(p, Norm{packed(residual), packed(branch), packed(weight), packed(bias), packed(post), packed(gate), draws}, y, z, false);
  return {y, z};
}

}  // namespace

TORCH_LIBRARY(mvr_tokens, m) {
  m.def("init(int[] entry_points) -> ()", init);
  m.def("rotate(Tensor x, Tensor positions, Tensor turns, int[] sections, bool interleaved) -> Tensor");
  m.def("attend(Tensor q, Tensor k, Tensor v, Tensor? keep, float? scale) -> Tensor");
  m.def("add_norm(Tensor residual, Tensor branch, Tensor weight, Tensor? bias, Tensor? post_weight, Tensor? gate, Tensor? draws, float number, bool layer, "
        "float eps) -> Tensor[]");
}

// (the autograd nodes are built inside: each operator is registered for every backend key at once, as a composite)
TORCH_LIBRARY_IMPL(mvr_tokens, CompositeImplicitAutograd, m) {
  m.impl("rotate", rotate_tokens);
  m.impl("attend", attend_tokens);
  m.impl("add_norm", add_norm_tokens);
}
