// Native torch kernels of the package's ops: the CUDA and AutogradCUDA entries
// that take a call of the usual form from the dispatcher to libanima_attn.so
// without entering Python.
//
// The ops themselves (schemas, fake kernels, the kernels of every other
// dispatch key) are registered in Python by torch.library.custom_op; attach()
// adds these two keys to one of them. Reached through Python, an op costs
// 25-30 us of host time per call, and a training step's autograd wiring 320 us
// for prologue + attention forward and backward, more than their kernels take
// at 1024 tokens (about 105 us); through here 8-15 and 78 us.
//
// A call that a kernel here does not take as it is (an odd stride or
// alignment that needs a copy, another dtype, a shape error) goes to the op's
// Python function, which owns every such case and its error message.
#include <torch/extension.h>

#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <algorithm>
#include <cmath>
#include <functional>
#include <initializer_list>
#include <map>
#include <memory>
#include <optional>
#include <string>
#include <tuple>
#include <unordered_set>
#include <utility>
#include <vector>

#include "../../include/anima_attn.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using T2 = std::tuple<Tensor, Tensor>;
using T3 = std::tuple<Tensor, Tensor, Tensor>;

// ---------------------------------------------------------------- fallback --

// The ops' Python functions. Never destroyed: ops may outlive the interpreter.
std::map<std::string, PyObject*>& python_impls() {
  static auto* m = new std::map<std::string, PyObject*>();
  return *m;
}

template <class R, class... A>
R python_impl(const char* name, const A&... args) {
  pybind11::gil_scoped_acquire gil;
  const pybind11::handle fn(python_impls().at(name));
  return fn(args...).template cast<R>();
}

// ------------------------------------------------------------------ helpers --

void* stream_of(const Tensor& t) {
  return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream();
}

bool aligned16(const Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0; }

// bf16 on the GPU of `like`.
bool bf16_on(const Tensor& t, const Tensor& like) {
  return t.scalar_type() == at::kBFloat16 && t.is_cuda() && t.device() == like.device();
}

// A [B, S, H, hd] view that the attention kernels read in place.
bool kernel_ready(const Tensor& t) {
  return t.stride(3) == 1 && t.stride(0) % 8 == 0 && t.stride(1) % 8 == 0 && t.stride(2) % 8 == 0 &&
         aligned16(t);
}

// True when done; false (nothing launched) sends the call to the Python
// function, which raises the library's message.
bool launched(int rc, const char* what) {
  if (rc == AA_OK) return true;
  TORCH_CHECK(rc != AA_EHIP, what, ": ", aa_last_error(), " (code ", rc, ")");
  return false;
}

void set_strides(int64_t (&dst)[3], const Tensor& t) {
  for (int i = 0; i < 3; ++i) dst[i] = t.stride(i);
}

Tensor f32(const Tensor& t) { return t.to(at::kFloat).contiguous(); }

// ---------------------------------------------------------------- attention --

bool attention_ready(const Tensor& q, const Tensor& k, const Tensor& v, int64_t hd) {
  return q.dim() == 4 && k.dim() == 4 && v.dim() == 4 && k.sizes() == v.sizes() &&
         q.size(0) == k.size(0) && q.size(2) == k.size(2) && q.size(3) == hd && k.size(3) == hd &&
         bf16_on(q, q) && bf16_on(k, q) && bf16_on(v, q) && q.numel() > 0 && k.numel() > 0 &&
         kernel_ready(q) && kernel_ready(k) && kernel_ready(v);
}

bool lengths_ready(const Tensor& t, const Tensor& q, at::ScalarType dtype) {
  return t.dim() == 1 && t.size(0) == q.size(0) && t.scalar_type() == dtype &&
         t.device() == q.device() && t.is_contiguous();
}

// out (and lse when wanted); false: for the Python function.
bool forward(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor* seqused,
             const Tensor* ln_pad, int64_t hd, Tensor& out, Tensor* lse) {
  if (!attention_ready(q, k, v, hd)) return false;
  if (seqused && !lengths_ready(*seqused, q, at::kInt)) return false;
  if (ln_pad && !lengths_ready(*ln_pad, q, at::kFloat)) return false;
  const c10::DeviceGuard guard(q.device());
  const int64_t B = q.size(0), Sq = q.size(1), H = q.size(2), Sk = k.size(1);
  out = at::empty({B, Sq, H, hd}, q.options());
  if (lse) *lse = at::empty({B, H, Sq}, q.options().dtype(at::kFloat));
  aa_attn_fwd_args a = {};
  a.q = q.data_ptr();
  a.k = k.data_ptr();
  a.v = v.data_ptr();
  a.out = out.data_ptr();
  a.lse = lse ? lse->data_ptr<float>() : nullptr;
  a.seqused_k = seqused ? seqused->data_ptr<int32_t>() : nullptr;
  a.ln_pad = ln_pad ? ln_pad->data_ptr<float>() : nullptr;
  set_strides(a.q_stride, q);
  set_strides(a.k_stride, k);
  set_strides(a.v_stride, v);
  set_strides(a.out_stride, out);
  a.B = B;
  a.Sq = Sq;
  a.Sk = Sk;
  a.H = H;
  a.hd = hd;
  a.softmax_scale = (float)(1.0 / std::sqrt((double)hd));
  a.dtype = AA_DTYPE_BF16;
  const size_t bytes = aa_attn_fwd_workspace(B, Sq, Sk, H, hd);
  Tensor ws;
  if (bytes) {
    ws = at::empty({(int64_t)bytes}, q.options().dtype(at::kByte));
    a.workspace = ws.data_ptr();
    a.workspace_bytes = bytes;
  }
  return launched(aa_attn_fwd(&a, stream_of(q)), "attn_fwd");
}

T2 fa_fwd(const Tensor& q, const Tensor& k, const Tensor& v) {
  Tensor out, lse;
  if (forward(q, k, v, nullptr, nullptr, 128, out, &lse)) return {out, lse};
  return python_impl<T2>("fa_fwd", q, k, v);
}

Tensor fa_fwd_nolse(const Tensor& q, const Tensor& k, const Tensor& v) {
  Tensor out;
  if (forward(q, k, v, nullptr, nullptr, 128, out, nullptr)) return out;
  return python_impl<Tensor>("fa_fwd_nolse", q, k, v);
}

T2 fa_fwd_k(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& seqused) {
  Tensor out, lse;
  if (forward(q, k, v, &seqused, nullptr, 128, out, &lse)) return {out, lse};
  return python_impl<T2>("fa_fwd_k", q, k, v, seqused);
}

Tensor fa_fwd_k_ctx(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& seqused,
                    const Tensor& ln_pad) {
  Tensor out;
  if (forward(q, k, v, &seqused, &ln_pad, 128, out, nullptr)) return out;
  return python_impl<Tensor>("fa_fwd_k_ctx", q, k, v, seqused, ln_pad);
}

Tensor attend_d384(const Tensor& q, const Tensor& k, const Tensor& v) {
  Tensor out;
  if (forward(q, k, v, nullptr, nullptr, 384, out, nullptr)) return out;
  return python_impl<Tensor>("attend_d384", q, k, v);
}

T3 fa_bwd(const Tensor& dout, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& out,
          const Tensor& lse) {
  const auto slow = [&] { return python_impl<T3>("fa_bwd", dout, q, k, v, out, lse); };
  if (!attention_ready(q, k, v, 128) || !dout.sizes().equals(q.sizes()) ||
      !out.sizes().equals(q.sizes()) || !bf16_on(dout, q) || !bf16_on(out, q) ||
      !dout.is_contiguous() || !aligned16(dout) || !kernel_ready(out))
    return slow();
  const int64_t B = q.size(0), Sq = q.size(1), H = q.size(2), Sk = k.size(1);
  if (lse.dim() != 3 || lse.size(0) != B || lse.size(1) != H || lse.size(2) != Sq ||
      lse.scalar_type() != at::kFloat || lse.device() != q.device() || !lse.is_contiguous())
    return slow();
  const c10::DeviceGuard guard(q.device());
  Tensor dq = at::empty_like(q), dk = at::empty_like(k), dv = at::empty_like(v);
  if (!kernel_ready(dq) || !kernel_ready(dk) || !kernel_ready(dv)) return slow();
  aa_attn_bwd_args a = {};
  a.dout = dout.data_ptr();
  a.q = q.data_ptr();
  a.k = k.data_ptr();
  a.v = v.data_ptr();
  a.out = out.data_ptr();
  a.lse = lse.data_ptr<float>();
  a.dq = dq.data_ptr();
  a.dk = dk.data_ptr();
  a.dv = dv.data_ptr();
  set_strides(a.dout_stride, dout);
  set_strides(a.q_stride, q);
  set_strides(a.k_stride, k);
  set_strides(a.v_stride, v);
  set_strides(a.out_stride, out);
  set_strides(a.dq_stride, dq);
  set_strides(a.dk_stride, dk);
  set_strides(a.dv_stride, dv);
  a.B = B;
  a.Sq = Sq;
  a.Sk = Sk;
  a.H = H;
  a.hd = 128;
  a.softmax_scale = (float)(1.0 / std::sqrt(128.0));
  a.dtype = AA_DTYPE_BF16;
  const size_t bytes = aa_attn_bwd_workspace(B, Sq, Sk, H, 128);
  const Tensor ws = at::empty({std::max<int64_t>((int64_t)bytes / 4, 1)}, q.options().dtype(at::kFloat));
  if (!launched(aa_attn_bwd(&a, ws.data_ptr(), bytes, stream_of(q)), "attn_bwd")) return slow();
  return {dq, dk, dv};
}

// ----------------------------------------------------------------- prologue --

bool on_gpu(const Tensor& t, const Tensor& like) { return t.device() == like.device(); }

bool qkv_ready(const Tensor& qkv, const Tensor& qw, const Tensor& kw, const Tensor& cos,
               const Tensor& sin, int64_t heads) {
  return qkv.dim() == 3 && bf16_on(qkv, qkv) && qkv.is_contiguous() && qkv.numel() > 0 &&
         cos.dim() == 2 && cos.size(1) == 64 && sin.sizes() == cos.sizes() &&
         cos.size(0) == qkv.size(1) && qkv.size(2) == 3 * heads * 128 && qw.numel() == 128 &&
         kw.numel() == 128 && on_gpu(qw, qkv) && on_gpu(kw, qkv) && on_gpu(cos, qkv) &&
         on_gpu(sin, qkv);
}

bool qkv_forward(const Tensor& qkv, const Tensor& qw, const Tensor& kw, const Tensor& cos,
                 const Tensor& sin, int64_t heads, double eps, Tensor& q, Tensor& k, Tensor* v) {
  if (!qkv_ready(qkv, qw, kw, cos, sin, heads)) return false;
  const c10::DeviceGuard guard(qkv.device());
  const int64_t B = qkv.size(0), S = qkv.size(1);
  q = at::empty({B, S, heads, 128}, qkv.options());
  k = at::empty_like(q);
  if (v) *v = at::empty_like(q);
  const Tensor qw32 = f32(qw), kw32 = f32(kw), c32 = f32(cos), s32 = f32(sin);
  return launched(aa_qkv_norm_rope_fwd(qkv.data_ptr(), q.data_ptr(), k.data_ptr(),
                                       v ? v->data_ptr() : nullptr, qw32.data_ptr<float>(),
                                       kw32.data_ptr<float>(), c32.data_ptr<float>(),
                                       s32.data_ptr<float>(), B, S, heads, 128, (float)eps,
                                       AA_DTYPE_BF16, stream_of(qkv)),
                  "qkv_norm_rope");
}

T2 qkv_norm_rope(const Tensor& qkv, const Tensor& qw, const Tensor& kw, const Tensor& cos,
                 const Tensor& sin, int64_t heads, double eps) {
  Tensor q, k;
  if (qkv_forward(qkv, qw, kw, cos, sin, heads, eps, q, k, nullptr)) return {q, k};
  return python_impl<T2>("qkv_norm_rope", qkv, qw, kw, cos, sin, heads, eps);
}

T3 qkv_norm_rope_v(const Tensor& qkv, const Tensor& qw, const Tensor& kw, const Tensor& cos,
                   const Tensor& sin, int64_t heads, double eps) {
  Tensor q, k, v;
  if (qkv_forward(qkv, qw, kw, cos, sin, heads, eps, q, k, &v)) return {q, k, v};
  return python_impl<T3>("qkv_norm_rope_v", qkv, qw, kw, cos, sin, heads, eps);
}

T3 qkv_norm_rope_bwd(const Tensor& qkv, const Tensor& dq_, const Tensor& dk_, const Tensor& dv_,
                     const Tensor& qw, const Tensor& kw, const Tensor& cos, const Tensor& sin,
                     int64_t heads, double eps) {
  const auto slow = [&] {
    return python_impl<T3>("qkv_norm_rope_bwd", qkv, dq_, dk_, dv_, qw, kw, cos, sin, heads, eps);
  };
  if (!qkv_ready(qkv, qw, kw, cos, sin, heads)) return slow();
  const int64_t B = qkv.size(0), S = qkv.size(1);
  for (const Tensor* t : {&dq_, &dk_, &dv_})
    if (!bf16_on(*t, qkv) || t->numel() != B * S * heads * 128) return slow();
  const c10::DeviceGuard guard(qkv.device());
  const Tensor dq = dq_.contiguous(), dk = dk_.contiguous(), dv = dv_.contiguous();
  Tensor dqkv = at::empty_like(qkv);
  const auto fopt = qkv.options().dtype(at::kFloat);
  Tensor dqw = at::empty({128}, fopt), dkw = at::empty({128}, fopt);
  const size_t bytes = aa_qkv_norm_rope_bwd_workspace(B, S, heads, 128);
  const Tensor ws = at::empty({std::max<int64_t>((int64_t)bytes / 4, 1)}, fopt);
  const Tensor qw32 = f32(qw), kw32 = f32(kw), c32 = f32(cos), s32 = f32(sin);
  if (!launched(aa_qkv_norm_rope_bwd(qkv.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                                     dqkv.data_ptr(), qw32.data_ptr<float>(),
                                     kw32.data_ptr<float>(), c32.data_ptr<float>(),
                                     s32.data_ptr<float>(), dqw.data_ptr<float>(),
                                     dkw.data_ptr<float>(), ws.data_ptr(), bytes, B, S, heads, 128,
                                     (float)eps, AA_DTYPE_BF16, stream_of(qkv)),
                "qkv_norm_rope_bwd"))
    return slow();
  return {dqkv, dqw.to(qw.scalar_type()), dkw.to(kw.scalar_type())};
}

bool head_norm_ready(const Tensor& x, const Tensor& w, int64_t heads) {
  return x.dim() == 3 && bf16_on(x, x) && x.is_contiguous() && x.numel() > 0 && w.numel() == 128 &&
         x.size(2) == heads * 128 && on_gpu(w, x);
}

Tensor head_norm(const Tensor& x, const Tensor& w, int64_t heads, double eps) {
  if (head_norm_ready(x, w, heads)) {
    const c10::DeviceGuard guard(x.device());
    const int64_t B = x.size(0), S = x.size(1);
    Tensor y = at::empty({B, S, heads, 128}, x.options());
    const Tensor w32 = f32(w);
    if (launched(aa_head_norm_fwd(x.data_ptr(), y.data_ptr(), w32.data_ptr<float>(), B, S, heads,
                                  128, (float)eps, AA_DTYPE_BF16, stream_of(x)),
                 "head_norm"))
      return y;
  }
  return python_impl<Tensor>("head_norm", x, w, heads, eps);
}

T2 head_norm_bwd(const Tensor& x, const Tensor& dy_, const Tensor& w, int64_t heads, double eps) {
  const auto slow = [&] { return python_impl<T2>("head_norm_bwd", x, dy_, w, heads, eps); };
  if (!head_norm_ready(x, w, heads) || !bf16_on(dy_, x) || dy_.numel() != x.numel()) return slow();
  const c10::DeviceGuard guard(x.device());
  const int64_t B = x.size(0), S = x.size(1);
  const Tensor dy = dy_.contiguous();
  Tensor dx = at::empty_like(x);
  const auto fopt = x.options().dtype(at::kFloat);
  Tensor dw = at::empty({128}, fopt);
  const size_t bytes = aa_head_norm_bwd_workspace(B, S, heads, 128);
  const Tensor ws = at::empty({std::max<int64_t>((int64_t)bytes / 4, 1)}, fopt);
  const Tensor w32 = f32(w);
  if (!launched(aa_head_norm_bwd(x.data_ptr(), dy.data_ptr(), dx.data_ptr(), w32.data_ptr<float>(),
                                 dw.data_ptr<float>(), ws.data_ptr(), bytes, B, S, heads, 128,
                                 (float)eps, AA_DTYPE_BF16, stream_of(x)),
                "head_norm_bwd"))
    return slow();
  return {dx, dw.to(w.scalar_type())};
}

// -------------------------------------------------------------- projections --

// [B, S, K] rows at one row stride (what the C ABI addresses) and a weight of
// `cols` rows; false for the forms that take one launch per batch item.
bool proj_ready(const Tensor& x, const Tensor& w, int64_t cols) {
  return x.dim() == 3 && bf16_on(x, x) && x.numel() > 0 && x.size(1) > 1 && x.stride(2) == 1 &&
         (x.size(0) == 1 || x.stride(0) == x.size(1) * x.stride(1)) && bf16_on(w, x) &&
         w.is_contiguous() && w.dim() == 2 && w.size(0) == cols && w.size(1) == x.size(2);
}

T3 qkv_proj_norm_rope(const Tensor& x, const Tensor& w, const Tensor& qw, const Tensor& kw,
                      const Tensor& cos, const Tensor& sin, int64_t heads, double eps) {
  if (proj_ready(x, w, 3 * heads * 128) && x.size(2) == heads * 128 && cos.dim() == 2 &&
      cos.size(1) == 64 && cos.size(0) == x.size(1) && sin.sizes() == cos.sizes() &&
      qw.numel() == 128 && kw.numel() == 128 && on_gpu(qw, x) && on_gpu(kw, x) && on_gpu(cos, x) &&
      on_gpu(sin, x)) {
    const c10::DeviceGuard guard(x.device());
    const int64_t B = x.size(0), S = x.size(1);
    Tensor q = at::empty({B, S, heads, 128}, x.options());
    Tensor k = at::empty_like(q), v = at::empty_like(q);
    const Tensor qw32 = f32(qw), kw32 = f32(kw), c32 = f32(cos), s32 = f32(sin);
    if (launched(aa_qkv_proj_norm_rope(x.data_ptr(), x.stride(1), w.data_ptr(), q.data_ptr(),
                                       k.data_ptr(), v.data_ptr(), qw32.data_ptr<float>(),
                                       kw32.data_ptr<float>(), c32.data_ptr<float>(),
                                       s32.data_ptr<float>(), B, S, heads, 128, (float)eps,
                                       AA_DTYPE_BF16, stream_of(x)),
                 "qkv_proj_norm_rope"))
      return {q, k, v};
  }
  return python_impl<T3>("qkv_proj_norm_rope", x, w, qw, kw, cos, sin, heads, eps);
}

Tensor proj_head_norm(const Tensor& x, const Tensor& w, const Tensor& nw, int64_t heads, double eps) {
  if (proj_ready(x, w, heads * 128) && nw.numel() == 128 && on_gpu(nw, x)) {
    const c10::DeviceGuard guard(x.device());
    const int64_t B = x.size(0), S = x.size(1);
    Tensor y = at::empty({B, S, heads, 128}, x.options());
    const Tensor nw32 = f32(nw);
    if (launched(aa_proj_head_norm(x.data_ptr(), x.stride(1), w.data_ptr(), x.size(2), y.data_ptr(),
                                   nw32.data_ptr<float>(), B, S, heads, 128, (float)eps,
                                   AA_DTYPE_BF16, stream_of(x)),
                 "proj_head_norm"))
      return y;
  }
  return python_impl<Tensor>("proj_head_norm", x, w, nw, heads, eps);
}

T2 kv_proj_norm(const Tensor& x, const Tensor& w, const Tensor& kw, int64_t heads, double eps) {
  if (proj_ready(x, w, 2 * heads * 128) && kw.numel() == 128 && on_gpu(kw, x)) {
    const c10::DeviceGuard guard(x.device());
    const int64_t B = x.size(0), S = x.size(1);
    Tensor k = at::empty({B, S, heads, 128}, x.options());
    Tensor v = at::empty_like(k);
    const Tensor kw32 = f32(kw);
    if (launched(aa_kv_proj_norm(x.data_ptr(), x.stride(1), w.data_ptr(), x.size(2), k.data_ptr(),
                                 v.data_ptr(), kw32.data_ptr<float>(), B, S, heads, 128, (float)eps,
                                 AA_DTYPE_BF16, stream_of(x)),
                 "kv_proj_norm"))
      return {k, v};
  }
  return python_impl<T2>("kv_proj_norm", x, w, kw, heads, eps);
}

// ------------------------------------------------------ norms of the block --

using T6 = std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor>;
using OptT = std::optional<Tensor>;

// Contiguous bf16 [B, S, D] at a 16-byte boundary, on the GPU of `like`.
bool rows_ready(const Tensor& t, const Tensor& like) {
  return t.dim() == 3 && bf16_on(t, like) && t.is_contiguous() && aligned16(t) && t.numel() > 0;
}

// Modulation rows [1 or B, D] that the kernels read in place, of mod0's dtype.
bool mod_ready(const Tensor& t, const Tensor& x, const Tensor& mod0) {
  const auto dtype = t.scalar_type();
  return t.dim() == 2 && t.size(1) == x.size(2) && (t.size(0) == 1 || t.size(0) == x.size(0)) &&
         dtype == mod0.scalar_type() && (dtype == at::kFloat || dtype == at::kBFloat16) && on_gpu(t, x) &&
         t.stride(1) == 1 && aligned16(t) &&
         (t.size(0) == 1 || (t.stride(0) * t.element_size() % 16 == 0 && t.stride(0) >= t.size(1)));
}

int64_t mod_stride(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : 0; }

bool adaln_ready(const Tensor& x, const Tensor* y, const Tensor* gate, const Tensor& scale, const OptT& weight) {
  return rows_ready(x, x) && (!y || (rows_ready(*y, x) && y->sizes() == x.sizes() && gate && mod_ready(*gate, x, scale))) &&
         mod_ready(scale, x, scale) &&
         (!weight || (weight->dim() == 1 && weight->size(0) == x.size(2) && on_gpu(*weight, x) &&
                      (weight->scalar_type() == at::kFloat || weight->scalar_type() == at::kBFloat16)));
}

// fp32 weight that lives until the launch.
Tensor f32_or_none(const OptT& weight) { return weight ? f32(*weight) : Tensor(); }
float* float_ptr(const Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }

// A tensor without elements, with x's type and a storage of its own (no two outputs of an op
// may share one), for what is not computed. (Through the dispatcher each would be a twentieth
// of the backward's host time.)
Tensor no_elements(const Tensor& x) {
  c10::Storage none(c10::Storage::use_byte_size_t(), 0, at::DataPtr(nullptr, x.device()), nullptr, false);
  return at::detail::make_tensor<c10::TensorImpl>(std::move(none), c10::DispatchKeySet(c10::DispatchKey::CUDA), x.dtype());
}

bool adaln_forward(const Tensor& x, const Tensor* y, const Tensor* gate, const Tensor& scale, const Tensor& shift,
                   const OptT& weight, double eps, double branch_scale, Tensor* r, Tensor* h, Tensor* q,
                   Tensor* qs, Tensor* stats) {
  if (!adaln_ready(x, y, gate, scale, weight) || !mod_ready(shift, x, scale)) return false;
  const c10::DeviceGuard guard(x.device());
  const int64_t B = x.size(0), S = x.size(1), D = x.size(2);
  const auto fopt = x.options().dtype(at::kFloat);
  const Tensor w = f32_or_none(weight);
  if (w.defined() && !aligned16(w)) return false;
  if (r) *r = at::empty(x.sizes(), x.options());
  if (h) *h = at::empty(x.sizes(), x.options());
  if (q) {
    *q = at::empty(x.sizes(), x.options().dtype(at::kChar));
    *qs = at::empty({B * S, 1}, fopt);
  }
  if (stats) *stats = at::empty({B * S, 4}, fopt);
  aa_adaln_args a = {};
  a.x = x.data_ptr();
  a.y = y ? y->data_ptr() : nullptr;
  a.gate = gate ? gate->data_ptr() : nullptr;
  a.scale = scale.data_ptr();
  a.shift = shift.data_ptr();
  a.gate_stride = gate ? mod_stride(*gate) : 0;
  a.scale_stride = mod_stride(scale);
  a.shift_stride = mod_stride(shift);
  a.weight = float_ptr(w);
  a.r = r ? r->data_ptr() : nullptr;
  a.h = h ? h->data_ptr() : nullptr;
  a.q = q ? q->data_ptr() : nullptr;
  a.q_scale = qs ? qs->data_ptr<float>() : nullptr;
  a.stats = stats ? stats->data_ptr<float>() : nullptr;
  a.B = B;
  a.S = S;
  a.D = D;
  a.eps = (float)eps;
  a.branch_scale = (float)branch_scale;
  a.dtype = AA_DTYPE_BF16;
  a.mod_dtype = scale.scalar_type() == at::kFloat ? AA_DTYPE_FP32 : AA_DTYPE_BF16;
  return launched(aa_adaln_fwd(&a, stream_of(x)), "adaln");
}

T3 residual_adaln(const Tensor& x, const Tensor& y, const Tensor& gate, const Tensor& scale, const Tensor& shift,
                  const OptT& weight, double eps, double branch_scale, bool want_stats) {
  Tensor r, h, stats;
  if (adaln_forward(x, &y, &gate, scale, shift, weight, eps, branch_scale, &r, &h, nullptr, nullptr,
                    want_stats ? &stats : nullptr)) {
    if (!want_stats) stats = at::empty({0, 4}, x.options().dtype(at::kFloat));
    return {r, h, stats};
  }
  return python_impl<T3>("residual_adaln", x, y, gate, scale, shift, weight, eps, branch_scale, want_stats);
}

T2 adaln(const Tensor& x, const Tensor& scale, const Tensor& shift, double eps, bool want_stats) {
  Tensor h, stats;
  if (adaln_forward(x, nullptr, nullptr, scale, shift, std::nullopt, eps, 1.0, nullptr, &h, nullptr, nullptr,
                    want_stats ? &stats : nullptr)) {
    if (!want_stats) stats = at::empty({0, 4}, x.options().dtype(at::kFloat));
    return {h, stats};
  }
  return python_impl<T2>("adaln", x, scale, shift, eps, want_stats);
}

T3 residual_adaln_int8(const Tensor& x, const Tensor& y, const Tensor& gate, const Tensor& scale,
                       const Tensor& shift, const OptT& weight, double eps, double branch_scale) {
  Tensor r, q, qs;
  if (adaln_forward(x, &y, &gate, scale, shift, weight, eps, branch_scale, &r, nullptr, &q, &qs, nullptr))
    return {r, q, qs};
  return python_impl<T3>("residual_adaln_int8", x, y, gate, scale, shift, weight, eps, branch_scale);
}

T6 adaln_bwd(const OptT& dr_, const OptT& dh_, const Tensor& x, const OptT& y, const OptT& gate, const Tensor& scale,
             const OptT& weight, const Tensor& stats, int64_t shift_rows, double branch_scale, bool mods) {
  const auto slow = [&] {
    return python_impl<T6>("adaln_bwd", dr_, dh_, x, y, gate, scale, weight, stats, shift_rows, branch_scale, mods);
  };
  if (!adaln_ready(x, y ? &*y : nullptr, gate ? &*gate : nullptr, scale, weight)) return slow();
  const int64_t B = x.size(0), S = x.size(1), D = x.size(2);
  if (stats.scalar_type() != at::kFloat || stats.dim() != 2 || stats.size(0) != B * S || stats.size(1) != 4 ||
      !stats.is_contiguous() || !on_gpu(stats, x) || y.has_value() != gate.has_value() ||
      (shift_rows != 1 && shift_rows != B))
    return slow();
  const c10::DeviceGuard guard(x.device());
  Tensor dr, dh;
  for (const auto& [from, to] : {std::make_pair(&dr_, &dr), std::make_pair(&dh_, &dh)}) {
    if (!*from) continue;
    if (!bf16_on(**from, x) || (*from)->sizes() != x.sizes()) return slow();
    *to = (*from)->contiguous();
    if (!aligned16(*to)) return slow();
  }
  const Tensor w = f32_or_none(weight);
  if (w.defined() && !aligned16(w)) return slow();
  Tensor dx = at::empty(x.sizes(), x.options());
  Tensor dy = y ? at::empty(x.sizes(), x.options()) : no_elements(x);
  Tensor dgate = mods && y ? at::empty(gate->sizes(), gate->options()) : no_elements(x);
  Tensor dscale = mods ? at::empty(scale.sizes(), scale.options()) : no_elements(x);
  Tensor dshift = mods ? at::empty({shift_rows, D}, scale.options()) : no_elements(x);
  Tensor dweight = mods && weight ? at::empty({D}, x.options().dtype(at::kFloat)) : no_elements(x);
  const auto ptr = [](const Tensor& t) { return t.numel() ? t.data_ptr() : nullptr; };
  aa_adaln_bwd_args a = {};
  a.dr = dr.defined() ? dr.data_ptr() : nullptr;
  a.dh = dh.defined() ? dh.data_ptr() : nullptr;
  a.x = x.data_ptr();
  a.y = y ? y->data_ptr() : nullptr;
  a.gate = gate ? gate->data_ptr() : nullptr;
  a.scale = scale.data_ptr();
  a.gate_stride = gate ? mod_stride(*gate) : 0;
  a.scale_stride = mod_stride(scale);
  a.weight = float_ptr(w);
  a.stats = stats.data_ptr<float>();
  a.dx = dx.data_ptr();
  a.dy = ptr(dy);
  a.dgate = ptr(dgate);
  a.dscale = ptr(dscale);
  a.dshift = ptr(dshift);
  a.dweight = (float*)ptr(dweight);
  a.gate_rows = gate ? gate->size(0) : 1;
  a.scale_rows = scale.size(0);
  a.shift_rows = shift_rows;
  a.B = B;
  a.S = S;
  a.D = D;
  a.branch_scale = (float)branch_scale;
  a.dtype = AA_DTYPE_BF16;
  a.mod_dtype = scale.scalar_type() == at::kFloat ? AA_DTYPE_FP32 : AA_DTYPE_BF16;
  const size_t bytes = aa_adaln_bwd_workspace(B, S, D, mods);
  Tensor ws;
  if (bytes) ws = at::empty({(int64_t)bytes / 4}, x.options().dtype(at::kFloat));
  if (!launched(aa_adaln_bwd(&a, bytes ? ws.data_ptr() : nullptr, bytes, stream_of(x)), "adaln_bwd")) return slow();
  return {dx, dy, dgate, dscale, dshift, dweight};
}

// ----------------------------------------------------------- int8 products --

T2 rowquant_int8(const Tensor& x, bool gelu) {
  if (rows_ready(x, x)) {
    const c10::DeviceGuard guard(x.device());
    const int64_t rows = x.size(0) * x.size(1);
    Tensor q = at::empty(x.sizes(), x.options().dtype(at::kChar));
    Tensor s = at::empty({rows, 1}, x.options().dtype(at::kFloat));
    if (launched(aa_rowquant_int8(x.data_ptr(), rows, x.size(2), gelu, q.data_ptr(), s.data_ptr<float>(),
                                  AA_DTYPE_BF16, stream_of(x)),
                 "rowquant_int8"))
      return {q, s};
  }
  return python_impl<T2>("rowquant_int8", x, gelu);
}

Tensor int8_linear(const Tensor& q, const Tensor& s, const Tensor& w, const Tensor& ws) {
  if (q.is_cuda() && q.dim() == 3 && w.dim() == 2 && q.scalar_type() == at::kChar && w.scalar_type() == at::kChar &&
      q.size(2) == w.size(1) && q.numel() > 0 && q.is_contiguous() && w.is_contiguous() && aligned16(q) && aligned16(w) &&
      on_gpu(w, q) && on_gpu(s, q) && on_gpu(ws, q) && s.scalar_type() == at::kFloat && ws.scalar_type() == at::kFloat &&
      s.numel() == q.size(0) * q.size(1) && ws.numel() == w.size(0) && s.is_contiguous() && ws.is_contiguous()) {
    const c10::DeviceGuard guard(q.device());
    Tensor y = at::empty({q.size(0), q.size(1), w.size(0)}, q.options().dtype(at::kBFloat16));
    if (launched(aa_int8_linear(q.data_ptr(), s.data_ptr<float>(), w.data_ptr(), ws.data_ptr<float>(), y.data_ptr(),
                                s.numel(), w.size(0), w.size(1), AA_DTYPE_BF16, stream_of(q)),
                 "int8_linear"))
      return y;
  }
  return python_impl<Tensor>("int8_linear", q, s, w, ws);
}

// ------------------------------------------------------- 8-bit checkpoints --

// Codes [rows, 32 G] and exponents of the given shape; empty without `keep`.
void kept(const Tensor& x, bool keep, int64_t e0, int64_t e1, Tensor* codes, Tensor* exps) {
  const int64_t K = x.size(2);
  *codes = at::empty({keep ? x.size(0) * x.size(1) : 0, (K + 31) / 32 * 32}, x.options().dtype(at::kChar));
  *exps = at::empty({keep ? e0 : 0, keep ? e1 : 0}, x.options().dtype(at::kByte));
}

T3 gelu8(const Tensor& x, bool keep) {
  if (rows_ready(x, x)) {
    const c10::DeviceGuard guard(x.device());
    const int64_t rows = x.size(0) * x.size(1), K = x.size(2);
    Tensor y = at::empty(x.sizes(), x.options()), codes, exps;
    kept(x, keep, rows, (K + 31) / 32, &codes, &exps);
    if (launched(aa_gelu8_fwd(x.data_ptr(), y.data_ptr(), keep ? codes.data_ptr() : nullptr,
                              keep ? exps.data_ptr() : nullptr, rows, K, AA_DTYPE_BF16, stream_of(x)),
                 "gelu8"))
      return {y, codes, exps};
  }
  return python_impl<T3>("gelu8", x, keep);
}

// The copy that the forward of `rows` rows of K channels made, with exponents [e0, e1].
bool kept_ready(const Tensor& codes, const Tensor& exps, const Tensor& like, int64_t rows, int64_t K, int64_t e0,
                int64_t e1) {
  const auto is = [&](const Tensor& t, at::ScalarType dtype, int64_t n0, int64_t n1) {
    return t.scalar_type() == dtype && on_gpu(t, like) && t.dim() == 2 && t.size(0) == n0 && t.size(1) == n1 &&
           t.is_contiguous() && aligned16(t);
  };
  return is(codes, at::kChar, rows, (K + 31) / 32 * 32) && is(exps, at::kByte, e0, e1);
}

Tensor gelu8_bwd(const Tensor& dy_, const Tensor& codes, const Tensor& exps) {
  if (dy_.dim() == 3 && bf16_on(dy_, dy_) && dy_.numel() > 0) {
    const c10::DeviceGuard guard(dy_.device());
    const Tensor dy = dy_.contiguous();
    const int64_t rows = dy.size(0) * dy.size(1), K = dy.size(2);
    if (aligned16(dy) && kept_ready(codes, exps, dy, rows, K, rows, (K + 31) / 32)) {
      Tensor dx = at::empty(dy.sizes(), dy.options());
      if (launched(aa_gelu8_bwd(dy.data_ptr(), codes.data_ptr(), exps.data_ptr(), dx.data_ptr(), rows, K,
                                AA_DTYPE_BF16, stream_of(dy)),
                   "gelu8_bwd"))
        return dx;
    }
  }
  return python_impl<Tensor>("gelu8_bwd", dy_, codes, exps);
}

bool down_ready(const Tensor& a, const Tensor& like) {
  return a.dim() == 2 && bf16_on(a, like) && a.is_contiguous() && aligned16(a) && a.numel() > 0;
}

T3 lora_down8(const Tensor& x, const Tensor& a, bool keep) {
  if (rows_ready(x, x) && down_ready(a, x) && a.size(1) == x.size(2)) {
    const c10::DeviceGuard guard(x.device());
    const int64_t rows = x.size(0) * x.size(1), K = x.size(2), R = a.size(0);
    Tensor t = at::empty({x.size(0), x.size(1), R}, x.options()), codes, exps;
    kept(x, keep, (K + 31) / 32, (rows + 15) / 16 * 16, &codes, &exps);
    const size_t bytes = aa_lora8_fwd_workspace(rows, K, R);
    Tensor ws;
    if (bytes) ws = at::empty({(int64_t)bytes / 4}, x.options().dtype(at::kFloat));
    if (launched(aa_lora8_fwd(x.data_ptr(), a.data_ptr(), t.data_ptr(), keep ? codes.data_ptr() : nullptr,
                              keep ? exps.data_ptr() : nullptr, bytes ? ws.data_ptr() : nullptr, bytes, rows, K, R,
                              AA_DTYPE_BF16, stream_of(x)),
                 "lora_down8"))
      return {t, codes, exps};
  }
  return python_impl<T3>("lora_down8", x, a, keep);
}

T2 lora_down8_bwd(const Tensor& dt_, const Tensor& a, const Tensor& codes, const Tensor& exps, bool need_x, bool need_a) {
  if (dt_.dim() == 3 && bf16_on(dt_, dt_) && dt_.numel() > 0 && down_ready(a, dt_) && dt_.size(2) == a.size(0)) {
    const c10::DeviceGuard guard(dt_.device());
    const Tensor dt = dt_.contiguous();
    const int64_t rows = dt.size(0) * dt.size(1), R = a.size(0), K = a.size(1);
    if (aligned16(dt) &&
        (!need_a || kept_ready(codes, exps, dt, rows, K, (K + 31) / 32, (rows + 15) / 16 * 16))) {
      Tensor dx = need_x ? at::empty({dt.size(0), dt.size(1), K}, dt.options()) : at::empty({0}, dt.options());
      Tensor da = need_a ? at::empty({R, K}, dt.options()) : at::empty({0}, dt.options());
      const size_t bytes = need_a ? aa_lora8_bwd_workspace(rows, K, R) : 0;
      Tensor ws;
      if (bytes) ws = at::empty({(int64_t)bytes / 4}, dt.options().dtype(at::kFloat));
      if (launched(aa_lora8_bwd(dt.data_ptr(), a.data_ptr(), need_a ? codes.data_ptr() : nullptr,
                                need_a ? exps.data_ptr() : nullptr, need_x ? dx.data_ptr() : nullptr,
                                need_a ? da.data_ptr() : nullptr, bytes ? ws.data_ptr() : nullptr, bytes, rows, K, R,
                                AA_DTYPE_BF16, stream_of(dt)),
                   "lora_down8_bwd"))
        return {dx, da};
    }
  }
  return python_impl<T2>("lora_down8_bwd", dt_, a, codes, exps, need_x, need_a);
}

// ----------------------------------------------------------------- autograd --

// The dispatcher's handle of one op, called below or above autograd.
template <class R, class... A>
struct Op {
  c10::TypedOperatorHandle<R(A...)> handle;
  explicit Op(const char* name)
      : handle(c10::Dispatcher::singleton().findSchemaOrThrow(name, "").template typed<R(A...)>()) {}
  R operator()(A... args) const { return handle.call(args...); }
  R below(A... args) const {
    at::AutoDispatchBelowADInplaceOrView guard;
    return handle.call(args...);
  }
};

#define ANIMA_OP(fn, name, ...)            \
  const Op<__VA_ARGS__>& fn() {            \
    static const Op<__VA_ARGS__> op(name); \
    return op;                             \
  }
using CT = const Tensor&;
ANIMA_OP(op_fa_fwd, "anima_flat::fa_fwd", T2, CT, CT, CT)
ANIMA_OP(op_fa_fwd_nolse, "anima_flat::fa_fwd_nolse", Tensor, CT, CT, CT)
ANIMA_OP(op_fa_fwd_k, "anima_flat::fa_fwd_k", T2, CT, CT, CT, CT)
ANIMA_OP(op_fa_bwd, "anima_flat::fa_bwd", T3, CT, CT, CT, CT, CT, CT)
ANIMA_OP(op_fa_fwd_k_ctx, "anima_flat_amd::fa_fwd_k_ctx", Tensor, CT, CT, CT, CT, CT)
ANIMA_OP(op_attend_d384, "anima_flat_amd::attend_d384", Tensor, CT, CT, CT)
ANIMA_OP(op_qkv_norm_rope, "anima_flat::qkv_norm_rope", T2, CT, CT, CT, CT, CT, int64_t, double)
ANIMA_OP(op_qkv_norm_rope_v, "anima_flat::qkv_norm_rope_v", T3, CT, CT, CT, CT, CT, int64_t, double)
ANIMA_OP(op_qkv_norm_rope_bwd, "anima_flat::qkv_norm_rope_bwd", T3, CT, CT, CT, CT, CT, CT, CT, CT,
         int64_t, double)
ANIMA_OP(op_head_norm, "anima_flat::head_norm", Tensor, CT, CT, int64_t, double)
ANIMA_OP(op_head_norm_bwd, "anima_flat::head_norm_bwd", T2, CT, CT, CT, int64_t, double)
ANIMA_OP(op_qkv_proj_norm_rope, "anima_flat_amd::qkv_proj_norm_rope", T3, CT, CT, CT, CT, CT, CT,
         int64_t, double)
ANIMA_OP(op_proj_head_norm, "anima_flat_amd::proj_head_norm", Tensor, CT, CT, CT, int64_t, double)
ANIMA_OP(op_kv_proj_norm, "anima_flat_amd::kv_proj_norm", T2, CT, CT, CT, int64_t, double)
using CO = const OptT&;
ANIMA_OP(op_residual_adaln, "anima_flat_amd::residual_adaln", T3, CT, CT, CT, CT, CT, CO, double, double, bool)
ANIMA_OP(op_adaln, "anima_flat_amd::adaln", T2, CT, CT, CT, double, bool)
ANIMA_OP(op_residual_adaln_int8, "anima_flat_amd::residual_adaln_int8", T3, CT, CT, CT, CT, CT, CO, double, double)
ANIMA_OP(op_adaln_bwd, "anima_flat_amd::adaln_bwd", T6, CO, CO, CT, CO, CO, CT, CO, CT, int64_t, double, bool)
ANIMA_OP(op_rowquant_int8, "anima_flat_amd::rowquant_int8", T2, CT, bool)
ANIMA_OP(op_int8_linear, "anima_flat_amd::int8_linear", Tensor, CT, CT, CT, CT)
ANIMA_OP(op_gelu8, "anima_flat_amd::gelu8", T3, CT, bool)
ANIMA_OP(op_gelu8_bwd, "anima_flat_amd::gelu8_bwd", Tensor, CT, CT, CT)
ANIMA_OP(op_lora_down8, "anima_flat_amd::lora_down8", T3, CT, CT, bool)
ANIMA_OP(op_lora_down8_bwd, "anima_flat_amd::lora_down8_bwd", T2, CT, CT, CT, CT, bool, bool)
#undef ANIMA_OP

// Whether a call is recorded for the backward; no op here has a forward-mode
// derivative.
template <class... A>
bool needs_grad(const A&... args) {
  const auto any = [&](auto pred) {
    const auto one = [&](const auto& a) {
      using A1 = std::decay_t<decltype(a)>;
      if constexpr (std::is_same_v<A1, Tensor>) return pred(a);
      else if constexpr (std::is_same_v<A1, OptT>) return a.has_value() && a->defined() && pred(*a);
      else return false;
    };
    return (one(args) || ...);
  };
  if (!c10::GradMode::is_enabled() || !any([](const Tensor& t) { return t.requires_grad(); }))
    return false;
  TORCH_CHECK_NOT_IMPLEMENTED(
      !any([](const Tensor& t) { return t._fw_grad(0).defined(); }),
      "You must implement the jvp function for custom autograd.Function to use it with forward "
      "mode AD.");
  return true;
}

// An op without a backward, reached with inputs that need one: its outputs
// need grad too, and asking for it raises what torch.library's own autograd
// kernel raises.
struct NoBackward : torch::autograd::Function<NoBackward> {
  static constexpr bool is_traceable = true;
  // The inputs are there for autograd to find (it does not look into lists).
  template <class... A>
  static variable_list forward(AutogradContext* ctx, const std::function<variable_list()>& run,
                               const std::string& name, const A&...) {
    ctx->saved_data["op"] = name;
    return run();
  }
  static variable_list backward(AutogradContext* ctx, const variable_list&) {
    TORCH_CHECK(false, "Trying to backward through ", ctx->saved_data["op"].toStringRef(),
                " but no autograd formula was registered. Please use register_autograd to add one.");
  }
};

variable_list as_list(const Tensor& t) { return {t}; }
variable_list as_list(const T2& t) { return {std::get<0>(t), std::get<1>(t)}; }
variable_list as_list(const T3& t) { return {std::get<0>(t), std::get<1>(t), std::get<2>(t)}; }
variable_list as_list(const T6& t) {
  return std::apply([](const auto&... v) { return variable_list{v...}; }, t);
}
void from_list(const variable_list& l, Tensor& t) { t = l[0]; }
void from_list(const variable_list& l, T6& t) { t = {l[0], l[1], l[2], l[3], l[4], l[5]}; }
void from_list(const variable_list& l, T2& t) { t = {l[0], l[1]}; }
void from_list(const variable_list& l, T3& t) { t = {l[0], l[1], l[2]}; }

// AutogradCUDA kernel of an op without a backward.
template <auto OpFn, class R, class... A>
struct Plain {
  static R call(A... args) {
    if (!needs_grad(args...)) return OpFn().below(args...);
    std::string name = OpFn().handle.operator_name().name;
    name.replace(name.find("::"), 2, ".");
    const std::function<variable_list()> run = [&] { return as_list(OpFn().below(args...)); };
    R result;
    from_list(NoBackward::apply(run, name + ".default", args...), result);
    return result;
  }
};

// One output: the LSE, which has no derivative, is handed past the node (a node
// with an output marked as such cannot be traced by compiled autograd).
struct FaFwd : torch::autograd::Function<FaFwd> {
  static constexpr bool is_traceable = true;
  static Tensor forward(AutogradContext* ctx, CT q, CT k, CT v, Tensor* lse) {
    Tensor out;
    std::tie(out, *lse) = op_fa_fwd().below(q, k, v);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({q, k, v, out, *lse});
    return out;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const variable_list s = ctx->get_saved_variables();
    if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
    variable_list g = as_list(op_fa_bwd()(grads[0], s[0], s[1], s[2], s[3], s[4]));
    g.emplace_back();
    return g;
  }
};

T2 fa_fwd_autograd(CT q, CT k, CT v) {
  if (!needs_grad(q, k, v)) return op_fa_fwd().below(q, k, v);
  Tensor lse;
  Tensor out = FaFwd::apply(q, k, v, &lse);
  return {out, lse};
}

struct QkvNormRopeV : torch::autograd::Function<QkvNormRopeV> {
  static constexpr bool is_traceable = true;
  static variable_list forward(AutogradContext* ctx, CT qkv, CT qw, CT kw, CT cos, CT sin,
                               int64_t heads, double eps) {
    auto [q, k, v] = op_qkv_norm_rope_v().below(qkv, qw, kw, cos, sin, heads, eps);
    ctx->save_for_backward({qkv, qw, kw, cos, sin});
    ctx->saved_data["heads"] = heads;
    ctx->saved_data["eps"] = eps;
    return {q, k, v};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& g) {
    const variable_list s = ctx->get_saved_variables();
    auto [dqkv, dqw, dkw] =
        op_qkv_norm_rope_bwd()(s[0], g[0], g[1], g[2], s[1], s[2], s[3], s[4],
                               ctx->saved_data["heads"].toInt(), ctx->saved_data["eps"].toDouble());
    return {dqkv, dqw, dkw, Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

T3 qkv_norm_rope_v_autograd(CT qkv, CT qw, CT kw, CT cos, CT sin, int64_t heads, double eps) {
  if (!needs_grad(qkv, qw, kw, cos, sin))
    return op_qkv_norm_rope_v().below(qkv, qw, kw, cos, sin, heads, eps);
  T3 r;
  from_list(QkvNormRopeV::apply(qkv, qw, kw, cos, sin, heads, eps), r);
  return r;
}

struct HeadNorm : torch::autograd::Function<HeadNorm> {
  static constexpr bool is_traceable = true;
  static Tensor forward(AutogradContext* ctx, CT x, CT w, int64_t heads, double eps) {
    Tensor y = op_head_norm().below(x, w, heads, eps);
    ctx->save_for_backward({x, w});
    ctx->saved_data["heads"] = heads;
    ctx->saved_data["eps"] = eps;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& g) {
    const variable_list s = ctx->get_saved_variables();
    auto [dx, dw] = op_head_norm_bwd()(s[0], g[0], s[1], ctx->saved_data["heads"].toInt(),
                                       ctx->saved_data["eps"].toDouble());
    return {dx, dw, Tensor(), Tensor()};
  }
};

Tensor head_norm_autograd(CT x, CT w, int64_t heads, double eps) {
  if (!needs_grad(x, w)) return op_head_norm().below(x, w, heads, eps);
  return HeadNorm::apply(x, w, heads, eps);
}

// Whether a node that the gradient of one of `inputs` goes to, or on to, was made by an
// eager graph on the default stream: a live accumulator of a leaf, or an operation
// ahead of this one. Every edge is followed; this runs in captures only.
bool reaches_default_stream(std::initializer_list<Tensor> inputs) {
  using torch::autograd::Node;
  std::vector<std::shared_ptr<Node>> roots;  // keep all nodes behind them alive
  std::vector<Node*> todo;
  std::unordered_set<Node*> seen;
  const auto add = [&](Node* node) {
    if (node && seen.insert(node).second) todo.push_back(node);
  };
  for (const Tensor& t : inputs) {
    if (!t.defined() || !t.requires_grad()) continue;
    roots.push_back(t.grad_fn() ? t.grad_fn() : torch::autograd::impl::try_get_grad_accumulator(t));
    add(roots.back().get());
  }
  while (!todo.empty()) {
    Node* node = todo.back();
    todo.pop_back();
    const auto stream = node->stream();
    if (stream && stream->device_type() == c10::DeviceType::CUDA &&
        *stream == c10::hip::getDefaultHIPStreamMasqueradingAsCUDA(stream->device_index()).unwrap())
      return true;
    for (const auto& edge : node->next_edges()) add(edge.function.get());
  }
  return false;
}
// The backward of a captured forward would make the default stream wait for captured
// work in such a place, which it cannot join: that ends the capture, and the process
// with it. (Any other stream joins the capture.)
template <class... T>
void check_capture(const Tensor& x, const T&... more) {
  if (c10::hip::device_count() == 0) return;  // fake tensors, on a machine that has no stream to ask for
  const hipStream_t stream = (hipStream_t)stream_of(x);
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  if (!stream || hipStreamIsCapturing(stream, &status) != hipSuccess || status == hipStreamCaptureStatusNone) return;
  TORCH_CHECK(!reaches_default_stream({x, more...}),
              "a forward with gradients is being captured while an eager graph of the same leaves lives: "
              "its nodes are on the default stream, which cannot join the capture; end that graph first");
}

// The statistics and 8-bit copies, which have no derivative, are handed past
// the node as the LSE is.
struct ResidualAdaln : torch::autograd::Function<ResidualAdaln> {
  static constexpr bool is_traceable = true;
  static variable_list forward(AutogradContext* ctx, CT x, CT y, CT gate, CT scale, CT shift, CO weight, double eps,
                               double branch_scale, bool mods, Tensor* stats) {
    auto [r, h, st] = op_residual_adaln().below(x, y, gate, scale, shift, weight, eps, branch_scale, true);
    *stats = st;
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({x, y, gate, scale, weight.value_or(Tensor()), st});
    ctx->saved_data["branch_scale"] = branch_scale;
    ctx->saved_data["shift_rows"] = shift.size(0);
    ctx->saved_data["mods"] = mods;
    return {r, h};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& g) {
    variable_list out(10);
    if (!g[0].defined() && !g[1].defined()) return out;
    const variable_list s = ctx->get_saved_variables();
    const auto opt = [](const Tensor& t) { return t.defined() ? OptT(t) : OptT(); };
    const bool mods = ctx->saved_data["mods"].toBool();
    auto [dx, dy, dgate, dscale, dshift, dweight] =
        op_adaln_bwd()(opt(g[0]), opt(g[1]), s[0], s[1], s[2], s[3], opt(s[4]), s[5],
                       ctx->saved_data["shift_rows"].toInt(), ctx->saved_data["branch_scale"].toDouble(), mods);
    out[0] = dx;
    out[1] = dy;
    if (mods) {
      out[2] = dgate;
      out[3] = dscale;
      out[4] = dshift;
      if (s[4].defined()) out[5] = dweight.to(s[4].scalar_type());
    }
    return out;
  }
};

T3 residual_adaln_autograd(CT x, CT y, CT gate, CT scale, CT shift, CO weight, double eps, double branch_scale,
                           bool want_stats) {
  if (!needs_grad(x, y, gate, scale, shift, weight))
    return op_residual_adaln().below(x, y, gate, scale, shift, weight, eps, branch_scale, want_stats);
  check_capture(x, y, gate, scale, shift, weight.value_or(Tensor()));
  const bool mods = gate.requires_grad() || scale.requires_grad() || shift.requires_grad() ||
                    (weight && weight->requires_grad());
  Tensor stats;
  const variable_list o = ResidualAdaln::apply(x, y, gate, scale, shift, weight, eps, branch_scale, mods, &stats);
  return {o[0], o[1], stats};
}

struct Adaln : torch::autograd::Function<Adaln> {
  static constexpr bool is_traceable = true;
  static Tensor forward(AutogradContext* ctx, CT x, CT scale, CT shift, double eps, bool mods, Tensor* stats) {
    auto [h, st] = op_adaln().below(x, scale, shift, eps, true);
    *stats = st;
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({x, scale, st});
    ctx->saved_data["shift_rows"] = shift.size(0);
    ctx->saved_data["mods"] = mods;
    return h;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& g) {
    variable_list out(6);
    if (!g[0].defined()) return out;
    const variable_list s = ctx->get_saved_variables();
    const bool mods = ctx->saved_data["mods"].toBool();
    const T6 r = op_adaln_bwd()(OptT(), g[0], s[0], OptT(), OptT(), s[1], OptT(), s[2],
                                ctx->saved_data["shift_rows"].toInt(), 1.0, mods);
    out[0] = std::get<0>(r);
    if (mods) {
      out[1] = std::get<3>(r);
      out[2] = std::get<4>(r);
    }
    return out;
  }
};

T2 adaln_autograd(CT x, CT scale, CT shift, double eps, bool want_stats) {
  if (!needs_grad(x, scale, shift)) return op_adaln().below(x, scale, shift, eps, want_stats);
  check_capture(x, scale, shift);
  Tensor stats;
  Tensor h = Adaln::apply(x, scale, shift, eps, scale.requires_grad() || shift.requires_grad(), &stats);
  return {h, stats};
}

struct Gelu8 : torch::autograd::Function<Gelu8> {
  static constexpr bool is_traceable = true;
  static Tensor forward(AutogradContext* ctx, CT x, Tensor* codes, Tensor* exps) {
    Tensor y;
    std::tie(y, *codes, *exps) = op_gelu8().below(x, true);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({*codes, *exps});
    return y;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& g) {
    variable_list out(3);
    if (!g[0].defined()) return out;
    const variable_list s = ctx->get_saved_variables();
    out[0] = op_gelu8_bwd()(g[0], s[0], s[1]);
    return out;
  }
};

T3 gelu8_autograd(CT x, bool keep) {
  if (!needs_grad(x)) return op_gelu8().below(x, keep);
  check_capture(x);
  Tensor codes, exps;
  Tensor y = Gelu8::apply(x, &codes, &exps);
  return {y, codes, exps};
}

struct LoraDown8 : torch::autograd::Function<LoraDown8> {
  static constexpr bool is_traceable = true;
  static Tensor forward(AutogradContext* ctx, CT x, CT a, bool need_x, bool need_a, Tensor* codes, Tensor* exps) {
    Tensor t;
    std::tie(t, *codes, *exps) = op_lora_down8().below(x, a, need_a);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({a, *codes, *exps});
    ctx->saved_data["need_x"] = need_x;
    ctx->saved_data["need_a"] = need_a;
    return t;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& g) {
    variable_list out(6);
    if (!g[0].defined()) return out;
    const variable_list s = ctx->get_saved_variables();
    const bool need_x = ctx->saved_data["need_x"].toBool(), need_a = ctx->saved_data["need_a"].toBool();
    auto [dx, da] = op_lora_down8_bwd()(g[0], s[0], s[1], s[2], need_x, need_a);
    if (need_x) out[0] = dx;
    if (need_a) out[1] = da;
    return out;
  }
};

T3 lora_down8_autograd(CT x, CT a, bool keep) {
  if (!needs_grad(x, a)) return op_lora_down8().below(x, a, keep);
  check_capture(x, a);
  Tensor codes, exps;
  Tensor t = LoraDown8::apply(x, a, x.requires_grad(), a.requires_grad(), &codes, &exps);
  return {t, codes, exps};
}

// ------------------------------------------------------------- registration --

// Registrations live as long as the process, as torch.library's do.
std::vector<std::unique_ptr<torch::Library>>& libraries() {
  static auto* v = new std::vector<std::unique_ptr<torch::Library>>();
  return *v;
}

template <class Cuda, class Autograd>
void add(const std::string& ns, const char* name, Cuda cuda, Autograd autograd) {
  for (const auto key : {c10::DispatchKey::CUDA, c10::DispatchKey::AutogradCUDA}) {
    libraries().push_back(std::make_unique<torch::Library>(torch::Library::IMPL, ns, key, __FILE__, __LINE__));
    if (key == c10::DispatchKey::CUDA) libraries().back()->impl(name, cuda);
    else libraries().back()->impl(name, autograd);
  }
}

#define ANIMA_ADD(fn, autograd) \
  if (name == #fn) return add(ns, #fn, TORCH_FN(fn), autograd)
#define ANIMA_PLAIN(fn, ...) \
  if (name == #fn) return add(ns, #fn, TORCH_FN(fn), &Plain<&op_##fn, __VA_ARGS__>::call)

void add_kernels(const std::string& ns, const std::string& name) {
  ANIMA_ADD(fa_fwd, &fa_fwd_autograd);
  ANIMA_ADD(qkv_norm_rope_v, &qkv_norm_rope_v_autograd);
  ANIMA_ADD(head_norm, &head_norm_autograd);
  ANIMA_PLAIN(fa_fwd_nolse, Tensor, CT, CT, CT);
  ANIMA_PLAIN(fa_fwd_k, T2, CT, CT, CT, CT);
  ANIMA_PLAIN(fa_bwd, T3, CT, CT, CT, CT, CT, CT);
  ANIMA_PLAIN(fa_fwd_k_ctx, Tensor, CT, CT, CT, CT, CT);
  ANIMA_PLAIN(attend_d384, Tensor, CT, CT, CT);
  ANIMA_PLAIN(qkv_norm_rope, T2, CT, CT, CT, CT, CT, int64_t, double);
  ANIMA_PLAIN(qkv_norm_rope_bwd, T3, CT, CT, CT, CT, CT, CT, CT, CT, int64_t, double);
  ANIMA_PLAIN(head_norm_bwd, T2, CT, CT, CT, int64_t, double);
  ANIMA_PLAIN(qkv_proj_norm_rope, T3, CT, CT, CT, CT, CT, CT, int64_t, double);
  ANIMA_PLAIN(proj_head_norm, Tensor, CT, CT, CT, int64_t, double);
  ANIMA_PLAIN(kv_proj_norm, T2, CT, CT, CT, int64_t, double);
  ANIMA_ADD(residual_adaln, &residual_adaln_autograd);
  ANIMA_ADD(adaln, &adaln_autograd);
  ANIMA_ADD(gelu8, &gelu8_autograd);
  ANIMA_ADD(lora_down8, &lora_down8_autograd);
  ANIMA_PLAIN(residual_adaln_int8, T3, CT, CT, CT, CT, CT, CO, double, double);
  ANIMA_PLAIN(adaln_bwd, T6, CO, CO, CT, CO, CO, CT, CO, CT, int64_t, double, bool);
  ANIMA_PLAIN(rowquant_int8, T2, CT, bool);
  ANIMA_PLAIN(int8_linear, Tensor, CT, CT, CT, CT);
  ANIMA_PLAIN(gelu8_bwd, Tensor, CT, CT, CT);
  ANIMA_PLAIN(lora_down8_bwd, T2, CT, CT, CT, CT, bool, bool);
  TORCH_CHECK(false, "no native kernels for ", ns, "::", name);
}

// Gives op ns::name its native CUDA and AutogradCUDA kernels; `impl` is the
// op's Python function, for the calls they do not take.
void attach(const std::string& qualname, pybind11::function impl) {
  const size_t at = qualname.find("::");
  TORCH_CHECK(at != std::string::npos, "expected ns::name, got ", qualname);
  const std::string ns = qualname.substr(0, at), name = qualname.substr(at + 2);
  python_impls()[name] = impl.release().ptr();
  add_kernels(ns, name);
}

}  // namespace

PYBIND11_MODULE(_anima_torch, m) {
  m.def("attach", &attach, "Native dispatcher kernels for one op of the package");
  // What this file's argument structs are laid out for; the library may be newer.
  m.def("abi_version", [] { return AA_ABI_VERSION; }, "Of the header it was compiled with");
  m.def("library_abi_version", &aa_abi_version, "Of the libanima_attn.so it is linked to");
}
