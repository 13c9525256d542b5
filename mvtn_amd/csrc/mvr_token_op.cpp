// mvtn_amd/_mvr_token_op.so — host side of mvtn_amd/tokens.py: the operators on view tokens as torch operators with C++ autograd nodes,
// so that a call crosses from Python once and its backward runs on the autograd engine's thread without the interpreter lock (as Python
// autograd functions over ctypes, a forward and backward cost 110-160 us of host time, against 35-130 us on the GPU).
//
// Each operator is three or four: the one that Python calls (rotate, attend, add_norm: checks its arguments and brings them into the form of the next),
// its forward, the forward that keeps what a backward needs, and the backward.  The latter have a kernel for the GPU, one for autograd and one for shapes
// alone, so that tracers and compilers, which look below autograd or run on tensors without memory, find whole operators there.
//
// Argument checks, allocation and the calls of the C ABI (include/mvr.h); no arithmetic.  The entry points' addresses are handed over
// by mvtn_amd/_lib.py: this file does not link against libmvr_hip.so, and that library stays free of torch types.  (libc10_hip: torch's current stream.)  What Python sees: ValueError
// for arguments that do not fit, RuntimeError for tensors that are not on the GPU and for errors of the library.
#include <ATen/ATen.h>
#include <ATen/core/LegacyTypeDispatch.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/autograd_not_implemented_fallback.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/library.h>

#include <cmath>
#include <cstring>
#include <tuple>
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
// sizes and strides as numbers, where a compiler traces with symbols too
int64_t len(const Tensor &t, int64_t d) { return t.sym_size(d).guard_int(__FILE__, __LINE__); }
bool same_shape(const Tensor &a, const Tensor &b) {
  bool same = a.dim() == b.dim();
  for (int64_t d = 0; same && d < a.dim(); ++d) same = len(a, d) == len(b, d);
  return same;
}
// the last dimension's elements side by side (a copy only where they are not)
Tensor rows_packed(const Tensor &t) { return t.sym_stride(-1).guard_int(__FILE__, __LINE__) == 1 || len(t, -1) == 1 ? t : t.contiguous(); }
Tensor like(const Tensor &t) { return at::empty_symint(t.sym_sizes(), t.options()); }   // (contiguous)
Tensor none_of(const Tensor &t) { return at::empty({0}, t.options()); }   // in the place of a result that was not asked for
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
  for (int64_t d = 0; d < t.dim(); ++d)
    if (len(t, d) > 0x7FFFFFFF) return false;
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

// An operator by its name, with its GPU kernel's signature
#define MVR_OP(name, kernel) static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("mvr_tokens::" name, "").typed<decltype(kernel)>()

// ---- rotary positions -------------------------------------------------------------------------------------------------

typedef at::ArrayRef<double> Doubles;
typedef at::IntArrayRef Ints;

mvr_rotary_params rotary_params(const Tensor &x, const Tensor &grad, const Tensor &positions, Ints sections, bool interleaved) {
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

// What every way in has to hold: the C ABI reads `turns` by the sections' sum and the tensors by x's sizes
void check_rotary(const Tensor &x, const Tensor &positions, Doubles turns, Ints sections, bool interleaved) {
  TORCH_CHECK_VALUE(x.dim() == 4, "x is (B, L, H, D)");
  const int64_t B = len(x, 0), L = len(x, 1), D = len(x, 3), pairs = (int64_t)turns.size(), axes = (int64_t)sections.size();
  int64_t sum = 0;
  for (int64_t n : sections) sum += n;
  TORCH_CHECK_VALUE(axes >= 1 && axes <= 4 && sum == pairs, "one number of turns per pair of the 1 to 4 sections");
  TORCH_CHECK_VALUE(type_of(x) >= 0, "x must be float32, float16 or bfloat16, not ", x.scalar_type());
  TORCH_CHECK_VALUE(2 * pairs <= D && D <= 256 && !(interleaved && D % 2), pairs, " pairs do not fit a head of ", D, " (at most 256, even when interleaved)");
  TORCH_CHECK_VALUE(in_32_bits(x), "every size of x must be below 2^31");
  const int64_t dims = positions.dim();
  TORCH_CHECK_VALUE((dims == 2 || dims == 3) && len(positions, -2) == L && len(positions, -1) == axes && (dims == 2 || len(positions, 0) == 1 || len(positions, 0) == B),
                    "positions are (B, L, axes), (1, L, axes) or (L, axes) with L = ", L, " and ", axes, " axes");
}
// ... and the forms that only the inner operators are called with
void check_rotary_inner(const Tensor &x, const Tensor &positions, Doubles turns, Ints sections, bool interleaved) {
  check_rotary(x, positions, turns, sections, interleaved);
  same_device(x, {&positions});
  TORCH_CHECK_VALUE(positions.dim() == 3 && len(positions, 0) == len(x, 0) && positions.scalar_type() == at::kFloat, "positions are (B, L, axes) in float32 here");
}

Tensor rotate_forward_gpu(const Tensor &x_, const Tensor &positions_, Doubles turns, Ints sections, bool interleaved) {
  check_rotary_inner(x_, positions_, turns, sections, interleaved);
  const c10::DeviceGuard guard(x_.device());
  Tensor out = like(x_);
  if (out.numel() == 0) return out;
  const Tensor x = rows_packed(x_), positions = rows_packed(positions_);
  const mvr_rotary_params p = rotary_params(x, Tensor(), positions, sections, interleaved);
  check(g_entry.rotate(&p, turns.data(), x.data_ptr(), positions.data_ptr<float>(), out.data_ptr(), stream_of(x)), "mvr_rotate_tokens_forward");
  return out;
}
Tensor rotate_forward_shape(const Tensor &x, const Tensor &, Doubles, Ints, bool) { return like(x); }

std::tuple<Tensor, Tensor> rotate_backward_gpu(const Tensor &grad_, const MaybeTensor &x_, const Tensor &positions_, Doubles turns, Ints sections, bool interleaved) {
  check_rotary_inner(grad_, positions_, turns, sections, interleaved);
  const Tensor given = or_none(x_);
  if (given.defined()) {
    same_device(grad_, {&given});
    TORCH_CHECK_VALUE(same_shape(given, grad_) && given.scalar_type() == grad_.scalar_type(), "x and its gradient are alike");
  }
  const c10::DeviceGuard guard(grad_.device());
  Tensor gx = like(grad_), gp = given.defined() ? like(positions_) : none_of(positions_);
  if (gx.numel() == 0) {
    gp.zero_();
    return {gx, gp};
  }
  const Tensor grad = rows_packed(grad_), positions = rows_packed(positions_), x = given.defined() ? rows_packed(given) : given;
  const mvr_rotary_params p = rotary_params(x.defined() ? x : grad, grad, positions, sections, interleaved);
  check(g_entry.rotate_backward(&p, turns.data(), ptr(x), positions.data_ptr<float>(), grad.data_ptr(), gx.data_ptr(), x.defined() ? fptr(gp) : nullptr, stream_of(grad)),
        "mvr_rotate_tokens_backward");
  return {gx, gp};
}
std::tuple<Tensor, Tensor> rotate_backward_shape(const Tensor &grad, const MaybeTensor &x, const Tensor &positions, Doubles, Ints, bool) {
  return {like(grad), x.has_value() ? like(positions) : none_of(positions)};
}

struct Rotate : public torch::autograd::Function<Rotate> {
  static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &positions, std::vector<double> turns, std::vector<int64_t> sections, bool interleaved) {
    const at::AutoDispatchBelowADInplaceOrView below;
    MVR_OP("rotate_forward", rotate_forward_gpu);
    Tensor out = op.call(x, positions, turns, sections, interleaved);
    ctx->save_for_backward({positions.requires_grad() ? x : Tensor(), positions});
    ctx->saved_data["turns"] = std::move(turns);
    ctx->saved_data["sections"] = std::move(sections);
    ctx->saved_data["interleaved"] = interleaved;
    return out;
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &positions = saved[1];
    MVR_OP("rotate_backward", rotate_backward_gpu);
    std::tuple<Tensor, Tensor> out;
    {
      const at::AutoDispatchBelowADInplaceOrView below;
      out = op.call(grads[0], some(x), positions, ctx->saved_data["turns"].toDoubleVector(), ctx->saved_data["sections"].toIntVector(),
                    ctx->saved_data["interleaved"].toBool());
    }
    // (without the positions' a gradient is linear in dy)
    return once({std::get<0>(out), x.defined() ? std::get<1>(out) : Tensor(), Tensor(), Tensor(), Tensor()}, grads, x.defined());
  }
};

Tensor rotate_forward_autograd(const Tensor &x, const Tensor &positions, Doubles turns, Ints sections, bool interleaved) {
  no_forward_mode({&x, &positions});
  if (wants_grad({&x, &positions})) return Rotate::apply(x, positions, turns.vec(), sections.vec(), interleaved);
  const at::AutoDispatchBelowADInplaceOrView below;
  MVR_OP("rotate_forward", rotate_forward_gpu);
  return op.call(x, positions, turns, sections, interleaved);
}

Tensor rotate_tokens(const Tensor &x, const Tensor &positions, Doubles turns, Ints sections, bool interleaved) {
  check_rotary(x, positions, turns, sections, interleaved);
  no_forward_mode({&x, &positions});
  same_device(x, {&positions});
  return rotate_forward_autograd(rows_packed(x), positions.to(at::kFloat).expand_symint({x.sym_size(0), x.sym_size(1), (int64_t)sections.size()}), turns, sections, interleaved);
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

void check_attend(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &keep, double scale) {
  TORCH_CHECK_VALUE(q.dim() == 4 && k.dim() == 4 && same_shape(k, v), "q is (B, Lq, H, D), k and v are (B, Lk, Hkv, D)");
  const int64_t B = len(q, 0), H = len(q, 2), D = len(q, 3), Lk = len(k, 1), E = len(k, 2);
  TORCH_CHECK_VALUE(len(k, 0) == B && len(k, 3) == D && D >= 1 && D <= 128, "q, k and v share the batch and a head size of 1 to 128");
  TORCH_CHECK_VALUE(E >= 1 && H >= 1 && H % E == 0, H, " heads are not a multiple of ", E, " key/value heads");
  TORCH_CHECK_VALUE((q.scalar_type() == at::kHalf || q.scalar_type() == at::kBFloat16) && k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(),
                    "q, k and v share one type of float16, bfloat16");
  TORCH_CHECK_VALUE(in_32_bits(q) && in_32_bits(k), "every size of q, k and v must be below 2^31");
  TORCH_CHECK_VALUE((float)scale > 0 && std::isfinite((float)scale), "scale must be positive and finite, in 32 bits too");
  if (keep.defined()) {
    const int64_t groups = keep.dim() == 2 ? len(keep, 1) : 0;
    // (one entry per key of no keys: none)
    TORCH_CHECK_VALUE(keep.dim() == 2 && len(keep, 0) == B && (groups >= 1 ? Lk % groups == 0 : Lk == 0), "keep is (B, G) with G a divisor of the ", Lk, " keys");
    TORCH_CHECK_VALUE(!keep.requires_grad(), "keep is a mask: it gets no gradient");
  }
}
void check_attend_inner(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &keep, double scale) {
  check_attend(q, k, v, keep, scale);
  same_device(q, {&k, &v, &keep});
  TORCH_CHECK_VALUE(!keep.defined() || keep.scalar_type() == at::kBool || keep.scalar_type() == at::kByte, "keep is in bytes here");
}

// over so few keys the backward does without the output's rest
constexpr int64_t kFewKeys = 64;

void attend_into(const Tensor &q_, const Tensor &k_, const Tensor &v_, const Tensor &keep_, double scale, Tensor &out, const Tensor &rest, const Tensor &lse) {
  if (k_.size(1) == 0) out.zero_();
  if (k_.size(1) == 0 || out.numel() == 0) return;
  const Tensor q = rows_packed(q_), k = rows_packed(k_), v = rows_packed(v_), keep = packed(keep_);
  const mvr_attend_params p = attend_params(q, k, v, keep, Tensor(), scale);
  const size_t bytes = g_entry.attend_bytes(&p, 0);
  const Tensor ws = workspace(bytes, q);
  check(g_entry.attend(&p, q.data_ptr(), k.data_ptr(), v.data_ptr(), (const uint8_t *)ptr(keep), out.data_ptr(), ptr(rest), fptr(lse), ptr(ws), bytes, stream_of(q)),
        "mvr_attend_tokens_forward");
}

Tensor attend_forward_gpu(const Tensor &q, const Tensor &k, const Tensor &v, const MaybeTensor &keep_, double scale) {
  const Tensor keep = or_none(keep_);
  check_attend_inner(q, k, v, keep, scale);
  const c10::DeviceGuard guard(q.device());
  Tensor out = like(q);
  attend_into(q, k, v, keep, scale, out, Tensor(), Tensor());
  return out;
}
Tensor attend_forward_shape(const Tensor &q, const Tensor &, const Tensor &, const MaybeTensor &, double) { return like(q); }

typedef std::tuple<Tensor, Tensor, Tensor> Three;

// out, what its rounding left, lse
Three attend_training_shape(const Tensor &q, const Tensor &k, const Tensor &, const MaybeTensor &, double) {
  return {like(q), len(k, 1) > kFewKeys ? like(q) : none_of(q), at::empty_symint({q.sym_size(0), q.sym_size(2), q.sym_size(1)}, q.options().dtype(at::kFloat))};
}
Three attend_training_gpu(const Tensor &q, const Tensor &k, const Tensor &v, const MaybeTensor &keep_, double scale) {
  const Tensor keep = or_none(keep_);
  check_attend_inner(q, k, v, keep, scale);
  const c10::DeviceGuard guard(q.device());
  Three all = attend_training_shape(q, k, v, keep_, scale);
  attend_into(q, k, v, keep, scale, std::get<0>(all), k.size(1) > kFewKeys ? std::get<1>(all) : Tensor(), std::get<2>(all));
  return all;
}

Three attend_backward_gpu(const Tensor &grad_, const Tensor &q_, const Tensor &k_, const Tensor &v_, const MaybeTensor &keep_, const Tensor &out_, const Tensor &rest_,
                          const Tensor &lse_, double scale) {
  const Tensor unpacked = or_none(keep_);
  check_attend_inner(q_, k_, v_, unpacked, scale);
  same_device(q_, {&grad_, &out_, &rest_, &lse_});
  const bool few = k_.size(1) <= kFewKeys;
  TORCH_CHECK_VALUE(same_shape(grad_, q_) && same_shape(out_, q_) && (few || same_shape(rest_, q_)) && grad_.scalar_type() == q_.scalar_type() &&
                        out_.scalar_type() == q_.scalar_type() && rest_.scalar_type() == q_.scalar_type() && lse_.scalar_type() == at::kFloat &&
                        lse_.dim() == 3 && lse_.size(0) == q_.size(0) && lse_.size(1) == q_.size(2) && lse_.size(2) == q_.size(1),
                    "the gradient, out, rest and lse belong to q");
  const c10::DeviceGuard guard(q_.device());
  Tensor gq = like(q_), gk = like(k_), gv = like(v_);
  if (gq.numel() == 0 || gk.numel() == 0) return {gq.zero_(), gk.zero_(), gv.zero_()};
  const Tensor q = rows_packed(q_), k = rows_packed(k_), v = rows_packed(v_), keep = packed(unpacked), grad = rows_packed(grad_), out = packed(out_),
               rest = few ? Tensor() : packed(rest_), lse = packed(lse_);
  const mvr_attend_params p = attend_params(q, k, v, keep, grad, scale);
  const size_t bytes = g_entry.attend_bytes(&p, 1);
  const Tensor ws = workspace(bytes, q);
  check(g_entry.attend_backward(&p, q.data_ptr(), k.data_ptr(), v.data_ptr(), (const uint8_t *)ptr(keep), out.data_ptr(), ptr(rest), lse.data_ptr<float>(),
                                grad.data_ptr(), gq.data_ptr(), gk.data_ptr(), gv.data_ptr(), ptr(ws), bytes, stream_of(q)),
        "mvr_attend_tokens_backward");
  return {gq, gk, gv};
}
Three attend_backward_shape(const Tensor &, const Tensor &q, const Tensor &k, const Tensor &v, const MaybeTensor &, const Tensor &, const Tensor &, const Tensor &, double) {
  return {like(q), like(k), like(v)};
}

struct Attend : public torch::autograd::Function<Attend> {
  static Tensor forward(AutogradContext *ctx, const Tensor &q, const Tensor &k, const Tensor &v, const MaybeTensor &keep, double scale) {
    const at::AutoDispatchBelowADInplaceOrView below;
    MVR_OP("attend_training", attend_training_gpu);
    const Three all = op.call(q, k, v, keep, scale);
    ctx->save_for_backward({q, k, v, or_none(keep), std::get<0>(all), std::get<1>(all), std::get<2>(all)});
    ctx->saved_data["scale"] = scale;
    return std::get<0>(all);
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    MVR_OP("attend_backward", attend_backward_gpu);
    Three g;
    {
      const at::AutoDispatchBelowADInplaceOrView below;
      g = op.call(grads[0], s[0], s[1], s[2], some(s[3]), s[4], s[5], s[6], ctx->saved_data["scale"].toDouble());
    }
    // (v's alone is linear in dO)
    return once({std::get<0>(g), std::get<1>(g), std::get<2>(g), Tensor(), Tensor()}, grads, s[0].requires_grad() || s[1].requires_grad());
  }
};

Tensor attend_forward_autograd(const Tensor &q, const Tensor &k, const Tensor &v, const MaybeTensor &keep, double scale) {
  no_forward_mode({&q, &k, &v});
  if (wants_grad({&q, &k, &v})) return Attend::apply(q, k, v, keep, scale);
  const at::AutoDispatchBelowADInplaceOrView below;
  MVR_OP("attend_forward", attend_forward_gpu);
  return op.call(q, k, v, keep, scale);
}

Tensor attend_tokens(const Tensor &q, const Tensor &k, const Tensor &v, const MaybeTensor &keep_, const c10::optional<double> &scale_) {
  Tensor keep = or_none(keep_);
  const double scale = scale_.has_value() ? *scale_ : q.dim() == 4 && len(q, 3) > 0 ? 1.0 / std::sqrt((double)len(q, 3)) : 1.0;
  check_attend(q, k, v, keep, scale);
  no_forward_mode({&q, &k, &v});
  same_device(q, {&k, &v, &keep});
  if (keep.defined()) keep = (keep.scalar_type() == at::kBool || keep.scalar_type() == at::kByte ? keep : keep.ne(0)).contiguous();
  return attend_forward_autograd(rows_packed(q), rows_packed(k), rows_packed(v), some(keep), scale);
}

// ---- norms around a block ----------------------------------------------------------------------------------------------

// What goes along with the tensors: by number (in the operators' arguments), as the C ABI takes it
struct NormNumbers {
  double number;
  bool layer;
  double eps;
};

// how many rows of gates there are, 0 without; -1: they do not fit
int64_t gate_groups(const Tensor &gate, const Tensor &residual) {
  if (!gate.defined()) return 0;
  const int64_t dims = residual.dim(), D = len(residual, -1);
  // one row per leading index, trailing ones left out
  int64_t lead = gate.dim() - 1, groups = 1;
  while (lead > 0 && len(gate, lead - 1) == 1) --lead;
  bool fits = gate.dim() >= 1 && len(gate, -1) == D && gate.dim() <= dims && (lead == 0 || lead < dims - 1);
  for (int64_t k = 0; fits && k < lead; ++k) fits = len(gate, k) == len(residual, k), groups *= len(gate, k);
  return fits ? groups : -1;
}

mvr_norm_params check_norm(const Tensor &residual, const Tensor &branch, const Tensor &weight, const Tensor &bias, const Tensor &post, const Tensor &gate, const Tensor &draws,
                           const NormNumbers &n) {
  TORCH_CHECK_VALUE(same_shape(residual, branch) && residual.dim() >= 2, "residual and branch are of one shape (..., D)");
  const int64_t D = len(residual, -1);
  TORCH_CHECK_VALUE(D >= 1 && D <= 8192, "rows of 1 to 8192 elements");
  const int r = type_of(residual), b = type_of(branch);
  TORCH_CHECK_VALUE(r >= 0 && b >= 0 && (r == b || r == MVR_TYPE_FLOAT), "residual and branch share one type of float32, float16, bfloat16, or the residual is float32");
  TORCH_CHECK_VALUE(n.eps >= 0 && std::isfinite(n.eps), "eps must not be negative");
  for (const Tensor *t : {&weight, &bias, &post})
    TORCH_CHECK_VALUE(!t->defined() || (t->dim() == 1 && len(*t, 0) == D), "weight, bias and post_weight are (", D, ",)");
  int64_t rows = 1;
  for (int64_t k = 0; k + 1 < residual.dim(); ++k) rows *= len(residual, k);
  const int64_t groups = gate_groups(gate, residual);
  TORCH_CHECK_VALUE(groups >= 0, "gate is (D,), or has one row per leading index of the residual ((B, D) or (B, 1, D) for (B, L, D)); a gate of every element belongs into the branch");
  TORCH_CHECK_VALUE(groups <= 65000, "at most 65000 rows of gates");
  for (const Tensor *t : {&weight, &bias, &post, &gate})
    TORCH_CHECK_VALUE(!t->defined() || (t->scalar_type() == weight.scalar_type() && type_of(*t) >= 0), "weight, bias, post_weight and gate share one type of float32, float16, bfloat16");
  int64_t count = 0;
  if (draws.defined()) {
    TORCH_CHECK_VALUE(!draws.requires_grad(), "scale holds draws: it gets no gradient (put what is learned into gate)");
    count = 1;
    for (int64_t k = 0; k < draws.dim(); ++k) count *= len(draws, k);
    TORCH_CHECK_VALUE(count >= 1 ? rows % count == 0 : rows == 0, "scale has ", count, " draws, which do not divide the ", rows, " rows");
  }
  mvr_norm_params p;
  std::memset(&p, 0, sizeof(p));
  p.rows = rows, p.dim = (int32_t)D, p.residual_type = r, p.branch_type = b, p.param_type = type_of(weight), p.kind = n.layer;
  p.gate_groups = groups, p.scale_groups = count, p.scale = (float)n.number, p.eps = (float)n.eps;
  return p;
}
mvr_norm_params check_norm_inner(const Tensor &residual, const Tensor &branch, const Tensor &weight, const Tensor &bias, const Tensor &post, const Tensor &gate,
                                 const Tensor &draws, const NormNumbers &n) {
  const mvr_norm_params p = check_norm(residual, branch, weight, bias, post, gate, draws, n);
  same_device(residual, {&branch, &weight, &bias, &post, &gate, &draws});
  TORCH_CHECK_VALUE(!draws.defined() || draws.scalar_type() == at::kFloat, "scale is in float32 here");
  return p;
}

typedef std::tuple<Tensor, Tensor> Two;
typedef std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor> Six;
#define MVR_NORM_INPUTS                                                                                                                                \
  const Tensor &residual, const Tensor &branch, const Tensor &weight, const MaybeTensor &bias_, const MaybeTensor &post_, const MaybeTensor &gate_,   \
      const MaybeTensor &draws_, double number, bool layer, double eps

void norm_into(MVR_NORM_INPUTS, Tensor &y, Tensor &z, float *stats) {
  const Tensor bias = packed(or_none(bias_)), post = packed(or_none(post_)), gate = packed(or_none(gate_)), draws = packed(or_none(draws_));
  const mvr_norm_params p = check_norm_inner(residual, branch, weight, bias, post, gate, draws, {number, layer, eps});
  if (!p.rows) return;
  const Tensor r = packed(residual), b = packed(branch), w = packed(weight);
  check(g_entry.norm(&p, r.data_ptr(), b.data_ptr(), w.data_ptr(), ptr(bias), ptr(post), ptr(gate), fptr(draws), y.data_ptr(), z.data_ptr(), stats, stream_of(r)),
        "mvr_add_norm_tokens_forward");
}

Two norm_forward_shape(MVR_NORM_INPUTS) { return {like(residual), like(branch)}; }
Two norm_forward_gpu(MVR_NORM_INPUTS) {
  const c10::DeviceGuard guard(residual.device());
  Two out = {like(residual), like(branch)};
  norm_into(residual, branch, weight, bias_, post_, gate_, draws_, number, layer, eps, std::get<0>(out), std::get<1>(out), nullptr);
  return out;
}

// y, z, the rows' statistics
Three norm_training_shape(MVR_NORM_INPUTS) {
  c10::SymInt rows = 1;
  for (int64_t k = 0; k + 1 < residual.dim(); ++k) rows = rows * residual.sym_size(k);
  return {like(residual), like(branch), at::empty_symint({rows, 4}, residual.options().dtype(at::kFloat))};
}
Three norm_training_gpu(MVR_NORM_INPUTS) {
  const c10::DeviceGuard guard(residual.device());
  Three out = norm_training_shape(residual, branch, weight, bias_, post_, gate_, draws_, number, layer, eps);
  norm_into(residual, branch, weight, bias_, post_, gate_, draws_, number, layer, eps, std::get<0>(out), std::get<1>(out), fptr(std::get<2>(out)));
  return out;
}

// need: of weight, bias, post_weight and gate, whose gradients are wanted; the others come empty
Six norm_backward_shape(const MaybeTensor &, const MaybeTensor &, const Tensor &y, const Tensor &branch, const Tensor &weight, const MaybeTensor &post, const MaybeTensor &gate,
                        const MaybeTensor &, const Tensor &, Ints need, double, bool, double) {
  const auto wanted = [&](const Tensor &t, int k) { return need[k] ? like(t) : none_of(weight); };
  return {like(y), like(branch), wanted(weight, 0), wanted(weight, 1), wanted(or_none(post), 2), wanted(or_none(gate), 3)};
}
Six norm_backward_gpu(const MaybeTensor &grad_y, const MaybeTensor &grad_z, const Tensor &y_, const Tensor &branch_, const Tensor &weight_, const MaybeTensor &post_,
                      const MaybeTensor &gate_, const MaybeTensor &draws_, const Tensor &stats_, Ints need, double number, bool layer, double eps) {
  const Tensor y = packed(y_), branch = packed(branch_), weight = packed(weight_), post = packed(or_none(post_)), gate = packed(or_none(gate_)),
               draws = packed(or_none(draws_)), stats = packed(stats_), gy = packed(or_none(grad_y)), gz = packed(or_none(grad_z));
  const mvr_norm_params p = check_norm_inner(y, branch, weight, Tensor(), post, gate, draws, {number, layer, eps});
  same_device(y, {&stats, &gy, &gz});
  TORCH_CHECK_VALUE((gy.defined() || gz.defined()) && (!gy.defined() || (same_shape(gy, y) && gy.scalar_type() == y.scalar_type())) &&
                        (!gz.defined() || (same_shape(gz, branch) && gz.scalar_type() == branch.scalar_type())),
                    "the gradients are those of y and z, one of them at least");
  TORCH_CHECK_VALUE(stats.scalar_type() == at::kFloat && stats.dim() == 2 && stats.size(0) == p.rows && stats.size(1) == 4, "stats are (rows, 4) in float32");
  TORCH_CHECK_VALUE(need.size() == 4 && (!need[2] || post.defined()) && (!need[3] || gate.defined()), "a gradient of a parameter that is not there");
  const c10::DeviceGuard guard(y.device());
  Six out = norm_backward_shape(grad_y, grad_z, y, branch, weight, post_, gate_, draws_, stats, need, number, layer, eps);
  const bool columns = need[0] || need[1] || need[2] || need[3];
  const Tensor &gw = std::get<2>(out), &gbias = std::get<3>(out), &gpost = std::get<4>(out), &ggate = std::get<5>(out);
  if (!p.rows) {
    for (const Tensor *t : {&gw, &gbias, &gpost, &ggate}) t->zero_();
    return out;
  }
  const size_t bytes = columns ? g_entry.norm_bytes(&p) : 0;
  const Tensor ws = workspace(bytes, y);
  const auto to = [&](const Tensor &t, int k) { return need[k] ? t.data_ptr() : nullptr; };
  check(g_entry.norm_backward(&p, y.data_ptr(), branch.data_ptr(), weight.data_ptr(), ptr(post), ptr(gate), fptr(draws), stats.data_ptr<float>(), ptr(gy), ptr(gz),
                              std::get<0>(out).data_ptr(), std::get<1>(out).data_ptr(), to(gw, 0), to(gbias, 1), to(gpost, 2), to(ggate, 3), ptr(ws), bytes, stream_of(y)),
        "mvr_add_norm_tokens_backward");
  return out;
}

struct AddNorm : public torch::autograd::Function<AddNorm> {
  static variable_list forward(AutogradContext *ctx, MVR_NORM_INPUTS) {
    const at::AutoDispatchBelowADInplaceOrView below;
    MVR_OP("add_norm_training", norm_training_gpu);
    const Three all = op.call(residual, branch, weight, bias_, post_, gate_, draws_, number, layer, eps);
    const Tensor bias = or_none(bias_), post = or_none(post_), gate = or_none(gate_);
    ctx->set_materialize_grads(false);
    // (y in 32 bits is what the backward needs; in 16 bits it would bring its rounding along, and the backward forms it again)
    ctx->save_for_backward({residual.scalar_type() == at::kFloat ? std::get<0>(all) : residual, branch, weight, post, gate, or_none(draws_), std::get<2>(all)});
    ctx->saved_data["numbers"] = std::vector<double>{number, (double)layer, eps};
    const auto wants = [](const Tensor &t) { return t.defined() && t.requires_grad(); };
    ctx->saved_data["need"] = std::vector<int64_t>{wants(weight), wants(bias), wants(post), wants(gate),
                                                   // (weight's and bias' alone are linear in dz)
                                                   wants(residual) || wants(branch) || wants(post) || wants(gate)};
    return {std::get<0>(all), std::get<1>(all)};
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    variable_list none(10);
    if (!grads[0].defined() && !grads[1].defined()) return none;
    const auto s = ctx->get_saved_variables();
    const auto numbers = ctx->saved_data["numbers"].toDoubleVector();
    auto need = ctx->saved_data["need"].toIntVector();
    const bool again = need.back();
    need.pop_back();
    MVR_OP("add_norm_backward", norm_backward_gpu);
    Six g;
    {
      const at::AutoDispatchBelowADInplaceOrView below;
      g = op.call(some(grads[0]), some(grads[1]), s[0] /* y, or the residual */, s[1], s[2], some(s[3]), some(s[4]), some(s[5]), s[6], need, numbers[0], numbers[1] != 0, numbers[2]);
    }
    const auto wanted = [&](const Tensor &t, int k) { return need[k] ? t : Tensor(); };
    return once({std::get<0>(g), std::get<1>(g), wanted(std::get<2>(g), 0), wanted(std::get<3>(g), 1), wanted(std::get<4>(g), 2), wanted(std::get<5>(g), 3), Tensor(), Tensor(),
                 Tensor(), Tensor()},
                grads, again);
  }
};

Two norm_forward_autograd(MVR_NORM_INPUTS) {
  const Tensor bias = or_none(bias_), post = or_none(post_), gate = or_none(gate_);
  no_forward_mode({&residual, &branch, &weight, &bias, &post, &gate});
  if (wants_grad({&residual, &branch, &weight, &bias, &post, &gate})) {
    const variable_list out = AddNorm::apply(residual, branch, weight, bias_, post_, gate_, draws_, number, layer, eps);
    return {out[0], out[1]};
  }
  const at::AutoDispatchBelowADInplaceOrView below;
  MVR_OP("add_norm_forward", norm_forward_gpu);
  return op.call(residual, branch, weight, bias_, post_, gate_, draws_, number, layer, eps);
}

Two add_norm_tokens(MVR_NORM_INPUTS) {
  const Tensor bias = or_none(bias_), post = or_none(post_), gate = or_none(gate_);
  Tensor draws = or_none(draws_);
  check_norm(residual, branch, weight, bias, post, gate, draws, {number, layer, eps});
  no_forward_mode({&residual, &branch, &weight, &bias, &post, &gate});
  same_device(residual, {&branch, &weight, &bias, &post, &gate, &draws});
  if (draws.defined()) draws = draws.to(at::kFloat).contiguous();
  return norm_forward_autograd(residual, branch, weight, bias_, post_, gate_, some(draws), number, layer, eps);
}

}  // namespace

#define MVR_NORM_SCHEMA "(Tensor residual, Tensor branch, Tensor weight, Tensor? bias, Tensor? post_weight, Tensor? gate, Tensor? draws, float number, bool layer, float eps)"

TORCH_LIBRARY(mvr_tokens, m) {
  m.def("init(int[] entry_points) -> ()", init);
  m.def("rotate(Tensor x, Tensor positions, float[] turns, int[] sections, bool interleaved) -> Tensor");
  m.def("rotate_forward(Tensor x, Tensor positions, float[] turns, int[] sections, bool interleaved) -> Tensor");
  m.def("rotate_backward(Tensor grad, Tensor? x, Tensor positions, float[] turns, int[] sections, bool interleaved) -> (Tensor, Tensor)");
  m.def("attend(Tensor q, Tensor k, Tensor v, Tensor? keep, float? scale) -> Tensor");
  m.def("attend_forward(Tensor q, Tensor k, Tensor v, Tensor? keep, float scale) -> Tensor");
  m.def("attend_training(Tensor q, Tensor k, Tensor v, Tensor? keep, float scale) -> (Tensor, Tensor, Tensor)");
  m.def("attend_backward(Tensor grad, Tensor q, Tensor k, Tensor v, Tensor? keep, Tensor out, Tensor rest, Tensor lse, float scale) -> (Tensor, Tensor, Tensor)");
  m.def("add_norm" MVR_NORM_SCHEMA " -> (Tensor, Tensor)");
  m.def("add_norm_forward" MVR_NORM_SCHEMA " -> (Tensor, Tensor)");
  m.def("add_norm_training" MVR_NORM_SCHEMA " -> (Tensor, Tensor, Tensor)");
  m.def("add_norm_backward(Tensor? grad_y, Tensor? grad_z, Tensor y_or_residual, Tensor branch, Tensor weight, Tensor? post_weight, Tensor? gate, Tensor? draws, Tensor stats, "
        "int[] need, float number, bool layer, float eps) -> (Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(mvr_tokens, CompositeImplicitAutograd, m) {
  m.impl("rotate", rotate_tokens);
  m.impl("attend", attend_tokens);
  m.impl("add_norm", add_norm_tokens);
}

TORCH_LIBRARY_IMPL(mvr_tokens, CUDA, m) {   // (torch's name for HIP devices)
  m.impl("rotate_forward", rotate_forward_gpu);
  m.impl("rotate_backward", rotate_backward_gpu);
  m.impl("attend_forward", attend_forward_gpu);
  m.impl("attend_training", attend_training_gpu);
  m.impl("attend_backward", attend_backward_gpu);
  m.impl("add_norm_forward", norm_forward_gpu);
  m.impl("add_norm_training", norm_training_gpu);
  m.impl("add_norm_backward", norm_backward_gpu);
}

TORCH_LIBRARY_IMPL(mvr_tokens, Meta, m) {
  m.impl("rotate_forward", rotate_forward_shape);
  m.impl("rotate_backward", rotate_backward_shape);
  m.impl("attend_forward", attend_forward_shape);
  m.impl("attend_training", attend_training_shape);
  m.impl("attend_backward", attend_backward_shape);
  m.impl("add_norm_forward", norm_forward_shape);
  m.impl("add_norm_training", norm_training_shape);
  m.impl("add_norm_backward", norm_backward_shape);
}

TORCH_LIBRARY_IMPL(mvr_tokens, Autograd, m) {
  m.impl("rotate_forward", rotate_forward_autograd);
  m.impl("attend_forward", attend_forward_autograd);
  m.impl("add_norm_forward", norm_forward_autograd);
  // called below autograd by the nodes above; called otherwise, they refuse to be differentiated
  for (const char *name : {"rotate_backward", "attend_training", "attend_backward", "add_norm_training", "add_norm_backward"})
    m.impl(name, torch::autograd::autogradNotImplementedFallback());
}
