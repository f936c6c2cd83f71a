// Attention, layer norm and rotary positions for PyTorch: argument checks, allocation, autograd. The Python wrappers
// (ops/attention.py, ops/norm.py, ops/rotary.py) only fill in defaults; everything is here so that a call costs a few
// microseconds on the host. Shapes, types and values are checked before devices, so a wrong call says what is wrong
// with it on any machine. Kernels run on the current stream of the tensors' device; workspaces come from the caching
// allocator, call by call (a captured graph gets its own from its pool).
#include "block_ops.h"

#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <cmath>
#include <limits>
#include <optional>
#include <string>
#include <vector>

#include "kernels/launch.h"

namespace {

using OptT = std::optional<at::Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

hipStream_t stream() { return c10::hip::getCurrentHIPStream().stream(); }

void ok(int rc, const char* what) {
  TORCH_CHECK(rc != 2, what, ": too large for one launch");
  TORCH_CHECK(rc == 0, what, " failed (code ", rc, ")");
}

// also for a tangent of forward-mode derivatives: the autograd function refuses it, the plain call would drop it
bool wants_grad(std::initializer_list<const at::Tensor*> ts) {
  for (const at::Tensor* t : ts)
    if (t->defined() && t->_fw_grad(0).defined()) return true;
  if (!at::GradMode::is_enabled()) return false;
  for (const at::Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// The kernels write through pointers. What records calls (jit.trace, make_fx) would see an allocation only and return
// memory as it was found, what stands for a tensor without holding it (fake, functional, zero tensors) has no address.
void check_eager(const char* what, std::initializer_list<const at::Tensor*> ts) {
  using Modes = c10::impl::TorchDispatchModeTLS;
  using Key = c10::impl::TorchDispatchModeKey;
  bool eager = !torch::jit::tracer::isTracing();
  if (Modes::any_modes_set())
    for (const Key k : {Key::FAKE, Key::PROXY, Key::FUNCTIONAL}) eager = eager && !Modes::get_mode(k).has_value();
  for (const at::Tensor* t : ts)
    if (t->defined())
      eager = eager && t->has_storage() && !t->key_set().has(c10::DispatchKey::Functionalize) &&
              t->storage().device() == t->device() && (t->numel() == 0 || t->const_data_ptr() != nullptr);
  TORCH_CHECK_NOT_IMPLEMENTED(eager, what, ": runs on tensors in memory only; it cannot be traced, nor take fake, "
                              "functional or zero tensors");
}

// A backward pass that is itself recorded (create_graph=True) would be taken for a constant by the next derivative.
void check_backward(const char* what, const at::Tensor& g) {
  TORCH_CHECK_NOT_IMPLEMENTED(!at::GradMode::is_enabled(), what, ": the backward pass cannot be differentiated");
  check_eager(what, {&g});
}

// the values of a tensor with a pending sign (the imaginary part of a conjugate), which memory does not show
at::Tensor with_sign(const at::Tensor& t) { return t.defined() && t.is_neg() ? t.resolve_neg() : t; }

void check_device(const at::Tensor& t, const at::Tensor& like, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be a device tensor");
  TORCH_CHECK(t.device() == like.device(), name, " must be on ", like.device(), ", is on ", t.device());
}

// ---------------------------------------------------------------------------------------------------- attention
// A token tensor the kernels can read: channels contiguous, 16-byte rows, tile offsets in 31 bits; else a copy.
at::Tensor readable(const at::Tensor& t) {
  bool good = t.stride(3) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  for (int i = 0; i < 3; ++i)
    if (t.size(i) > 1) good = good && t.stride(i) % 8 == 0;
  if (t.size(1) > 1) good = good && t.stride(1) < (int64_t)1 << 23;
  if (t.size(2) > 1) good = good && t.stride(2) * t.size(2) < (int64_t)1 << 28;
  return good ? t : t.clone(at::MemoryFormat::Contiguous);
}

AttnTensor view(const at::Tensor& t) {
  auto st = [&](int i) { return t.size(i) > 1 ? t.stride(i) : 0; };
  return AttnTensor{t.data_ptr(), st(0), st(1), st(2)};
}

struct Shape {
  int64_t B, Sq, Sk, Hq, Hkv, D;
};

Shape check_attention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const OptT& mask,
                      const OptT& lengths, double scale) {
  TORCH_CHECK_VALUE(q.dim() == 4 && k.dim() == 4 && v.dim() == 4,
                    "attention: q, k and v must be (images, tokens, heads, channels), got ", q.sizes(), ", ",
                    k.sizes(), ", ", v.sizes());
  TORCH_CHECK_TYPE(q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kHalf,
                   "attention: q must be bfloat16 or float16, is ", q.scalar_type());
  TORCH_CHECK_TYPE(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(),
                   "attention: q, k and v must have one type, got ", q.scalar_type(), ", ", k.scalar_type(), ", ",
                   v.scalar_type());
  const Shape s{q.size(0), q.size(1), k.size(1), q.size(2), k.size(2), q.size(3)};
  TORCH_CHECK_VALUE(k.sizes() == v.sizes(), "attention: k and v must have one shape, got ", k.sizes(), ", ", v.sizes());
  TORCH_CHECK_VALUE(k.size(0) == s.B && k.size(3) == s.D, "attention: q ", q.sizes(), " does not fit k ", k.sizes());
  TORCH_CHECK_VALUE(s.D >= 8 && s.D <= 128 && s.D % 8 == 0,
                    "attention: head channels must be a multiple of 8 up to 128, got ", s.D);
  TORCH_CHECK_VALUE(s.Hkv >= 1 && s.Hq >= 1 && s.Hq % s.Hkv == 0, "attention: ", s.Hq,
                    " query heads cannot share ", s.Hkv, " key heads evenly");
  constexpr int64_t top = (int64_t)1 << 30;
  TORCH_CHECK_VALUE(s.Sq * (s.Hq / s.Hkv) < top && s.Sk < top && s.B * s.Hkv < top && s.Hq * s.D < ((int64_t)1 << 23),
                    "attention: too large: q ", q.sizes(), ", k ", k.sizes());
  TORCH_CHECK_VALUE((float)scale > 0 && std::isfinite(2 * (float)scale),    // the kernels take it times log2(e)
                    "attention: scale must be positive and finite in float32, got ", scale);
  if (mask) {
    TORCH_CHECK_TYPE(mask->scalar_type() == at::kBool, "attention: mask must be bool (True: may attend), is ",
                     mask->scalar_type());
    const int64_t full[4] = {s.B, s.Hq, s.Sq, s.Sk};
    bool fits = mask->dim() <= 4;
    for (int64_t i = 0; fits && i < mask->dim(); ++i) {
      const int64_t n = mask->size(mask->dim() - 1 - i);
      fits = n == 1 || n == full[3 - i];
    }
    TORCH_CHECK_VALUE(fits, "attention: mask ", mask->sizes(), " does not broadcast to ", at::IntArrayRef(full, 4));
  }
  if (lengths) {
    TORCH_CHECK_TYPE(lengths->scalar_type() == at::kInt, "attention: lengths must be int32, is ",
                     lengths->scalar_type());
    TORCH_CHECK_VALUE(lengths->dim() == 1 && lengths->size(0) == s.B, "attention: lengths must be (", s.B, ",), got ",
                      lengths->sizes());
  }
  const at::Tensor none;
  check_eager("attention", {&q, &k, &v, mask ? &*mask : &none, lengths ? &*lengths : &none});
  TORCH_CHECK(q.is_cuda(), "attention: q must be a device tensor");
  check_device(k, q, "attention: k");
  check_device(v, q, "attention: v");
  if (mask) check_device(*mask, q, "attention: mask");
  if (lengths) check_device(*lengths, q, "attention: lengths");
  return s;
}

// a boolean mask as words and classes, one int64 tensor: [words | classes]
struct PackedMask {
  at::Tensor buf;
  int64_t Bm = 1, Hm = 1, Im = 1, words = 0;
};

PackedMask pack_mask(const at::Tensor& mask, const Shape& s) {
  const at::Tensor m = mask.expand({s.B, s.Hq, s.Sq, s.Sk});
  PackedMask pm;
  auto kept = [&](int i) { return m.size(i) > 1 && m.stride(i) != 0 ? m.size(i) : (int64_t)1; };
  pm.Bm = kept(0);
  pm.Hm = kept(1);
  pm.Im = kept(2);
  pm.words = (s.Sk + 63) / 64;
  const int64_t nw = pm.Bm * pm.Hm * pm.Im * pm.words, nc = pm.Bm * pm.Hm * ((pm.Im + 31) / 32) * pm.words;
  pm.buf = at::empty({nw + (nc + 7) / 8}, mask.options().dtype(at::kLong));
  AttnMaskArgs a{};
  a.src = reinterpret_cast<const uint8_t*>(m.data_ptr());
  a.sb = m.stride(0);
  a.sh = m.stride(1);
  a.si = m.stride(2);
  a.sk = s.Sk > 1 ? m.stride(3) : 0;
  a.Bm = (int)pm.Bm;
  a.Hm = (int)pm.Hm;
  a.Im = (int)pm.Im;
  a.Sk = (int)s.Sk;
  a.words = (int)pm.words;
  a.bits = reinterpret_cast<unsigned long long*>(pm.buf.data_ptr());
  a.cls = reinterpret_cast<uint8_t*>(a.bits + nw);
  if (s.Sk > 0) ok(attn_mask_bits(a, stream()), "attention: mask");
  return pm;
}

AttnMask mask_view(const at::Tensor& buf, int64_t Bm, int64_t Hm, int64_t Im, int64_t words) {
  AttnMask m{};
  if (!buf.defined() || words == 0) return m;
  m.bits = reinterpret_cast<const unsigned long long*>(buf.data_ptr());
  m.cls = reinterpret_cast<const uint8_t*>(m.bits + Bm * Hm * Im * words);
  m.sb = Bm > 1 ? Hm * Im : 0;
  m.sh = Hm > 1 ? Im : 0;
  m.rows = (int)Im;
  m.words = (int)words;
  return m;
}

AttnParams params(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const Shape& s, bool causal,
                  double scale, const at::Tensor& lengths) {
  AttnParams p{};
  p.q = view(q);
  p.k = view(k);
  p.v = view(v);
  p.lengths = lengths.defined() ? lengths.data_ptr<int>() : nullptr;
  p.B = (int)s.B;
  p.Sq = (int)s.Sq;
  p.Sk = (int)s.Sk;
  p.Hq = (int)s.Hq;
  p.Hkv = (int)s.Hkv;
  p.G = (int)(s.Hq / s.Hkv);
  p.D = (int)s.D;
  p.M = p.Sq * p.G;
  p.causal = causal;
  p.fp16 = q.scalar_type() == at::kHalf;
  p.scale = (float)scale;
  p.div_g = fast_div(p.G);
  p.splits = p.kv_splits = 1;
  return p;
}

// blocks of different work (attention.h locate())
bool uneven(const AttnParams& p) {
  return p.lengths || p.mask.sb || p.causal;
}

// The forward call on readable tensors. lse2: defined -> filled.
void run_forward(AttnParams& p, const at::Tensor& out, const at::Tensor& lse2) {
  p.o = view(out);
  p.lse2 = lse2.defined() ? lse2.data_ptr<float>() : nullptr;
  p.splits = attn_splits(p.B, p.Hkv, p.M, p.Sk);
  at::Tensor ws;
  if (p.splits > 1) {
    const int64_t rows = (int64_t)p.splits * p.B * p.Hkv * p.M, dp = (p.D + 31) / 32 * 32;
    ws = at::empty({rows * (dp + 2)}, out.options().dtype(at::kFloat));
    p.ws_o = ws.data_ptr<float>();
    p.ws_ml = p.ws_o + rows * dp;
  }
  ok(attn_fwd(p, stream()), "attention");
}

// what the forward pass leaves for the backward pass, next to q, k, v and out
struct Saved {
  at::Tensor lse2, rest, bits, lengths;
  PackedMask pm;
};

at::Tensor forward(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const Shape& s, const OptT& mask,
                   const OptT& lengths, bool causal, double scale, bool lse, bool grad, Saved& sv) {
  at::Tensor out = at::empty({s.B, s.Sq, s.Hq, s.D}, q.options());
  if (grad) sv.rest = at::empty_like(out);
  if (lse || grad) sv.lse2 = at::empty({s.B, s.Hkv, s.Sq * (s.Hq / s.Hkv)}, q.options().dtype(at::kFloat));
  if (out.numel() == 0) return out;
  if (lengths) sv.lengths = lengths->contiguous();
  AttnParams p = params(q, k, v, s, causal, scale, sv.lengths);
  if (mask) {
    sv.pm = pack_mask(*mask, s);
    sv.bits = sv.pm.buf;
    p.mask = mask_view(sv.bits, sv.pm.Bm, sv.pm.Hm, sv.pm.Im, sv.pm.words);
  }
  p.uneven = uneven(p);
  p.o_rest = grad ? reinterpret_cast<bf16_t*>(sv.rest.data_ptr()) : nullptr;
  run_forward(p, out, sv.lse2);
  return out;
}

void backward(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& out,
              const at::Tensor& go_in, const Saved& sv, const Shape& s, bool causal, double scale,
              const at::Tensor& dq, const at::Tensor& dk, const at::Tensor& dv) {
  const at::Tensor go = readable(go_in);
  AttnParams p = params(q, k, v, s, causal, scale, sv.lengths);
  p.mask = mask_view(sv.bits, sv.pm.Bm, sv.pm.Hm, sv.pm.Im, sv.pm.words);
  p.uneven = uneven(p);
  p.o = view(out);
  p.o_rest = reinterpret_cast<bf16_t*>(sv.rest.data_ptr());
  p.go = view(go);
  // a softmax over one key is 1 whatever the score: no gradient, and not what the roundings of dp - delta leave
  p.grad_scale = s.Sk == 1 ? 0.f : p.scale;
  if (dq.defined()) p.dq = view(dq);
  if (dk.defined()) p.dk = view(dk);
  if (dv.defined()) p.dv = view(dv);
  const at::Tensor delta = at::empty_like(sv.lse2);
  attn_bwd_splits(p.B, p.Hkv, p.M, p.Sk, p.causal != 0, p.splits, p.kv_splits);
  const int64_t dp = (p.D + 31) / 32 * 32, bh = (int64_t)p.B * p.Hkv;
  const int64_t nq = p.splits > 1 ? p.splits * bh * p.M * dp : 0, nk = p.kv_splits > 1 ? 2 * p.kv_splits * bh * p.Sk * dp : 0;
  at::Tensor ws;
  if (nq + nk > 0) {
    ws = at::empty({nq + nk}, sv.lse2.options());
    p.ws_o = ws.data_ptr<float>();
    p.ws_kv = p.ws_o + nq;
  }
  p.lse2 = sv.lse2.data_ptr<float>();
  p.delta = delta.data_ptr<float>();
  ok(attn_bwd(p, stream()), "attention backward");
}

at::Tensor natural_lse(const at::Tensor& lse2, const Shape& s, bool fp16) {
  const int64_t G = s.Hq / s.Hkv;
  const at::Tensor t = lse2.view({s.B, s.Hkv, s.Sq, G}).permute({0, 1, 3, 2}).reshape({s.B, s.Hq, s.Sq});
  const double inf = std::numeric_limits<double>::infinity();
  return at::where(t == inf, at::scalar_tensor(-inf, t.options()),
                   (fp16 ? t + ATTN_FP16_P_UP : t) * 0.6931471805599453);
}

void put_meta(AutogradContext* ctx, const Shape& s, bool causal, double scale, const PackedMask& pm) {
  ctx->saved_data["shape"] = std::vector<int64_t>{s.B, s.Sq, s.Sk, s.Hq, s.Hkv, s.D, causal, pm.Bm, pm.Hm, pm.Im,
                                                  pm.words};
  ctx->saved_data["scale"] = scale;
}

void get_meta(AutogradContext* ctx, Shape& s, bool& causal, double& scale, PackedMask& pm) {
  const auto m = ctx->saved_data["shape"].toIntVector();
  s = Shape{m[0], m[1], m[2], m[3], m[4], m[5]};
  causal = m[6] != 0;
  pm.Bm = m[7];
  pm.Hm = m[8];
  pm.Im = m[9];
  pm.words = m[10];
  scale = ctx->saved_data["scale"].toDouble();
}

struct AttentionFn : torch::autograd::Function<AttentionFn> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                               const OptT& mask, const OptT& lengths, bool causal, double scale) {
    const Shape s{q.size(0), q.size(1), k.size(1), q.size(2), k.size(2), q.size(3)};
    const at::Tensor qr = readable(q), kr = readable(k), vr = readable(v);
    Saved sv;
    const at::Tensor out = ::forward(qr, kr, vr, s, mask, lengths, causal, scale, true, true, sv);
    ctx->save_for_backward({qr, kr, vr, out, sv.lse2, sv.rest, sv.bits, sv.lengths});
    put_meta(ctx, s, causal, scale, sv.pm);
    ctx->mark_non_differentiable({sv.lse2});
    return {out, sv.lse2};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    check_backward("attention", g[0]);
    const auto t = ctx->get_saved_variables();
    Shape s;
    bool causal;
    double scale;
    Saved sv;
    get_meta(ctx, s, causal, scale, sv.pm);
    sv.lse2 = t[4];
    sv.rest = t[5];
    sv.bits = t[6];
    sv.lengths = t[7];
    variable_list r(7);
    const c10::DeviceGuard guard(t[0].device());
    for (int i = 0; i < 3; ++i)
      if (ctx->needs_input_grad(i)) r[i] = at::empty(t[i].sizes(), t[i].options());
    if (t[3].numel() == 0) {
      for (int i = 0; i < 3; ++i)
        if (r[i].defined()) r[i].zero_();
      return r;
    }
    ::backward(t[0], t[1], t[2], t[3], g[0], sv, s, causal, scale, r[0], r[1], r[2]);
    return r;
  }
};

// q, k, v as one tensor (images, tokens, heads + 2 kv_heads, channels), its gradient as one
struct AttentionQkvFn : torch::autograd::Function<AttentionQkvFn> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& qkv, int64_t heads, int64_t kv,
                               const OptT& mask, const OptT& lengths, bool causal, double scale) {
    const at::Tensor t = readable(qkv);
    const Shape s{t.size(0), t.size(1), t.size(1), heads, kv, t.size(3)};
    Saved sv;
    const at::Tensor out = ::forward(t.narrow(2, 0, heads), t.narrow(2, heads, kv), t.narrow(2, heads + kv, kv), s,
                                     mask, lengths, causal, scale, true, true, sv);
    ctx->save_for_backward({t, out, sv.lse2, sv.rest, sv.bits, sv.lengths});
    put_meta(ctx, s, causal, scale, sv.pm);
    ctx->mark_non_differentiable({sv.lse2});
    return {out, sv.lse2};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    check_backward("attention_qkv", g[0]);
    const auto t = ctx->get_saved_variables();
    Shape s;
    bool causal;
    double scale;
    Saved sv;
    get_meta(ctx, s, causal, scale, sv.pm);
    sv.lse2 = t[2];
    sv.rest = t[3];
    sv.bits = t[4];
    sv.lengths = t[5];
    const c10::DeviceGuard guard(t[0].device());
    const at::Tensor d = at::empty(t[0].sizes(), t[0].options());
    if (d.numel() != 0) {
      auto part = [&](const at::Tensor& x, int i) {
        return x.narrow(2, i == 0 ? 0 : s.Hq + (i - 1) * s.Hkv, i == 0 ? s.Hq : s.Hkv);
      };
      ::backward(part(t[0], 0), part(t[0], 1), part(t[0], 2), t[1], g[0], sv, s, causal, scale, part(d, 0),
                 part(d, 1), part(d, 2));
    }
    variable_list r(7);
    r[0] = d;
    return r;
  }
};

py::object result(const at::Tensor& out, const at::Tensor& lse2, const Shape& s, bool return_lse) {
  if (!return_lse) return py::cast(out);
  return py::make_tuple(out, natural_lse(lse2, s, out.scalar_type() == at::kHalf));
}

py::object attention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const OptT& mask,
                     const OptT& lengths, bool causal, std::optional<double> scale, bool return_lse) {
  const double sc = scale ? *scale : q.dim() == 4 && q.size(3) > 0 ? 1.0 / std::sqrt((double)q.size(3)) : 1.0;
  const Shape s = check_attention(q, k, v, mask, lengths, sc);
  const c10::DeviceGuard guard(q.device());
  if (wants_grad({&q, &k, &v})) {
    const auto r = AttentionFn::apply(q, k, v, mask, lengths, causal, sc);
    return result(r[0], r[1], s, return_lse);
  }
  Saved sv;
  const at::Tensor out =
      forward(readable(q), readable(k), readable(v), s, mask, lengths, causal, sc, return_lse, false, sv);
  return result(out, sv.lse2, s, return_lse);
}

py::object attention_qkv(const at::Tensor& qkv, int64_t heads, std::optional<int64_t> kv_heads, const OptT& mask,
                         const OptT& lengths, bool causal, std::optional<double> scale, bool return_lse) {
  const int64_t kv = kv_heads ? *kv_heads : heads;
  TORCH_CHECK_VALUE(qkv.dim() == 4, "attention_qkv: qkv must be (images, tokens, heads, channels), got ", qkv.sizes());
  TORCH_CHECK_VALUE(heads >= 1 && kv >= 1 && qkv.size(2) == heads + 2 * kv, "attention_qkv: qkv ", qkv.sizes(),
                    " does not hold ", heads, " query and 2 x ", kv, " key and value heads");
  const double sc = scale ? *scale : qkv.size(3) > 0 ? 1.0 / std::sqrt((double)qkv.size(3)) : 1.0;
  check_eager("attention_qkv", {&qkv});
  const at::Tensor q = qkv.narrow(2, 0, heads), k = qkv.narrow(2, heads, kv), v = qkv.narrow(2, heads + kv, kv);
  const Shape s = check_attention(q, k, v, mask, lengths, sc);
  const c10::DeviceGuard guard(qkv.device());
  if (wants_grad({&qkv})) {
    const auto r = AttentionQkvFn::apply(qkv, heads, kv, mask, lengths, causal, sc);
    return result(r[0], r[1], s, return_lse);
  }
  Saved sv;
  const at::Tensor out =
      forward(readable(q), readable(k), readable(v), s, mask, lengths, causal, sc, return_lse, false, sv);
  return result(out, sv.lse2, s, return_lse);
}

// --------------------------------------------------------------------------------------------------- layer norm
int type_code(const at::Tensor& t, const char* what) {
  switch (t.scalar_type()) {
    case at::kFloat: return 0;
    case at::kBFloat16: return 1;
    case at::kHalf: return 2;
    default: TORCH_CHECK_TYPE(false, what, " must be float32, bfloat16 or float16, is ", t.scalar_type());
  }
  return -1;
}

// the rows of t as (row stride), or a contiguous copy
at::Tensor rows_of(const at::Tensor& t, int64_t C, int64_t& stride) {
  stride = C;
  bool good = t.stride(-1) == 1 || C == 1;
  int64_t step = -1, span = 1;                 // row stride; rows of the axes behind
  for (int64_t i = t.dim() - 2; good && i >= 0; --i) {
    if (t.size(i) == 1) continue;
    if (step < 0) step = t.stride(i);
    good = t.stride(i) == step * span;
    span *= t.size(i);
  }
  if (!good) return t.contiguous();
  if (step >= 0) stride = step;
  return t;
}

LayerNormParams ln_params(const at::Tensor& x, const at::Tensor& w, int64_t C, double eps) {
  LayerNormParams p{};
  p.x = x.data_ptr();
  p.w = w.defined() ? w.data_ptr<float>() : nullptr;
  p.rows = x.numel() / C;
  p.C = (int)C;
  p.eps = (float)eps;
  p.type = type_code(x, "layer_norm: x");
  return p;
}

at::Tensor ln_forward(const at::Tensor& x, const at::Tensor& w, const at::Tensor& b, double eps) {
  const int64_t C = x.size(-1);
  at::Tensor y = at::empty(x.sizes(), x.options());
  if (y.numel() == 0) return y;
  int64_t stride;
  const at::Tensor xr = rows_of(x, C, stride);
  LayerNormParams p = ln_params(xr, w, C, eps);
  p.x_stride = stride;
  p.b = b.defined() ? b.data_ptr<float>() : nullptr;
  p.y = y.data_ptr();
  ok(layer_norm_fwd(p, stream()), "layer_norm");
  return y;
}

struct LayerNormFn : torch::autograd::Function<LayerNormFn> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const OptT& w, const OptT& b, double eps) {
    const at::Tensor wc = w ? w->contiguous() : at::Tensor(), bc = b ? b->contiguous() : at::Tensor();
    ctx->save_for_backward({x, wc});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["w"] = w.has_value();
    ctx->saved_data["b"] = b.has_value();
    return ln_forward(x, wc, bc, eps);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    check_backward("layer_norm", g[0]);
    const auto t = ctx->get_saved_variables();
    const at::Tensor &x = t[0], &w = t[1];
    const int64_t C = x.size(-1);
    const c10::DeviceGuard guard(x.device());
    // needs_input_grad counts the tensors that were given
    const bool hw = ctx->saved_data["w"].toBool(), hb = ctx->saved_data["b"].toBool();
    const bool nx = ctx->needs_input_grad(0), nw = hw && ctx->needs_input_grad(1);
    const bool nb = hb && ctx->needs_input_grad(hw ? 2 : 1);
    variable_list r(4);
    if (nx) r[0] = at::empty(x.sizes(), x.options());
    const auto f32 = x.options().dtype(at::kFloat);
    if (nw) r[1] = at::empty({C}, f32);
    if (nb) r[2] = at::empty({C}, f32);
    if (x.numel() == 0) {
      if (nw) r[1].zero_();
      if (nb) r[2].zero_();
      return r;
    }
    int64_t xs, gs;
    const at::Tensor xr = rows_of(x, C, xs), gr = rows_of(with_sign(g[0]), C, gs);
    LayerNormParams p = ln_params(xr, w, C, ctx->saved_data["eps"].toDouble());
    p.x_stride = xs;
    p.gy = gr.data_ptr();
    p.gy_stride = gs;
    p.y = nx ? r[0].data_ptr() : nullptr;
    p.dw = nw ? r[1].data_ptr<float>() : nullptr;
    p.db = nb ? r[2].data_ptr<float>() : nullptr;
    p.blocks = layer_norm_bwd_blocks(p);
    at::Tensor ws;
    if ((nw || nb) && p.blocks > 1) {
      ws = at::empty({(int64_t)p.blocks * 2 * C}, f32);
      p.ws = ws.data_ptr<float>();
    }
    ok(layer_norm_bwd(p, stream()), "layer_norm backward");
    return r;
  }
};

at::Tensor layer_norm(const at::Tensor& x, OptT weight, OptT bias, double eps) {
  TORCH_CHECK_VALUE(x.dim() >= 1, "layer_norm: x must have at least one axis");
  type_code(x, "layer_norm: x");
  const int64_t C = x.size(-1);
  TORCH_CHECK_VALUE(C >= 1 && C <= LAYER_NORM_MAX_C, "layer_norm: the last axis must have 1 to ", LAYER_NORM_MAX_C,
                    " channels, has ", C);
  TORCH_CHECK_VALUE(std::isfinite(eps) && eps >= 0, "layer_norm: eps must be finite and not negative, got ", eps);
  for (const auto& [t, name] : {std::pair<const OptT&, const char*>(weight, "weight"), {bias, "bias"}})
    if (t) {
      TORCH_CHECK_TYPE(t->scalar_type() == at::kFloat, "layer_norm: ", name, " must be float32, is ",
                       t->scalar_type());
      TORCH_CHECK_VALUE(t->dim() == 1 && t->size(0) == C, "layer_norm: ", name, " must be (", C, ",), got ",
                        t->sizes());
    }
  const at::Tensor w = weight ? *weight : at::Tensor(), b = bias ? *bias : at::Tensor();
  check_eager("layer_norm", {&x, &w, &b});
  TORCH_CHECK(x.is_cuda(), "layer_norm: x must be a device tensor");
  if (weight) check_device(*weight, x, "layer_norm: weight");
  if (bias) check_device(*bias, x, "layer_norm: bias");
  const c10::DeviceGuard guard(x.device());
  if (weight) weight = with_sign(*weight);
  if (bias) bias = with_sign(*bias);
  if (wants_grad({&x, &w, &b})) return LayerNormFn::apply(with_sign(x), weight, bias, eps);
  return ln_forward(with_sign(x), weight ? weight->contiguous() : w, bias ? bias->contiguous() : b, eps);
}

// ------------------------------------------------------------------------------------------------------- rotary
struct RotaryPlan {
  int64_t half, end[4];
  double theta;
  bool joint, interleaved;
};

at::Tensor rotary_run(const at::Tensor& x, const at::Tensor& pos, const RotaryPlan& pl, bool inverse) {
  at::Tensor y = at::empty(x.sizes(), x.options());
  if (y.numel() == 0) return y;
  const at::Tensor xr = x.stride(3) == 1 || x.size(3) == 1 ? x : x.contiguous();
  RotaryParams p{};
  p.x = xr.data_ptr();
  p.y = y.data_ptr();
  p.pos = pos.data_ptr();
  p.B = (int)x.size(0);
  p.S = (int)x.size(1);
  p.H = (int)x.size(2);
  p.D = (int)x.size(3);
  auto st = [](const at::Tensor& t, int i) { return t.size(i) > 1 ? t.stride(i) : 0; };
  p.x_sb = st(xr, 0); p.x_ss = st(xr, 1); p.x_sh = st(xr, 2);
  p.y_sb = st(y, 0); p.y_ss = st(y, 1); p.y_sh = st(y, 2);
  p.p_sa = pos.stride(0);
  p.p_sb = pos.dim() == 3 && pos.size(1) > 1 ? pos.stride(1) : 0;
  p.p_ss = pos.stride(-1);
  p.half = (int)pl.half;
  for (int a = 0; a < 4; ++a) p.end[a] = (int)pl.end[a];
  p.log2_theta = std::log2(pl.theta);
  p.joint = pl.joint;
  p.interleaved = pl.interleaved;
  p.inverse = inverse;
  p.type = type_code(x, "rotary: x");
  p.pos_type = pos.scalar_type() == at::kInt ? 0 : pos.scalar_type() == at::kLong ? 1 : 2;
  ok(rotary_apply(p, stream()), "rotary");
  return y;
}

struct RotaryFn : torch::autograd::Function<RotaryFn> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& pos, const RotaryPlan& pl) {
    ctx->save_for_backward({pos});
    ctx->saved_data["plan"] = std::vector<int64_t>{pl.half, pl.end[0], pl.end[1], pl.end[2], pl.end[3], pl.joint,
                                                   pl.interleaved};
    ctx->saved_data["theta"] = pl.theta;
    return rotary_run(x, pos, pl, false);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    check_backward("rotary", g[0]);
    const auto t = ctx->get_saved_variables();
    const auto m = ctx->saved_data["plan"].toIntVector();
    const RotaryPlan pl{m[0], {m[1], m[2], m[3], m[4]}, ctx->saved_data["theta"].toDouble(), m[5] != 0, m[6] != 0};
    const c10::DeviceGuard guard(t[0].device());
    return {rotary_run(g[0], t[0], pl, true), at::Tensor(), at::Tensor()};
  }
};

at::Tensor rotary(const at::Tensor& x, const at::Tensor& pos, const std::vector<int64_t>& dims, double theta,
                  bool joint, bool interleaved) {
  TORCH_CHECK_VALUE(x.dim() == 4, "rotary: x must be (images, tokens, heads, channels), got ", x.sizes());
  type_code(x, "rotary: x");
  TORCH_CHECK_VALUE(dims.size() >= 1 && dims.size() <= 4, "rotary: one to four axes, got ", dims.size());
  RotaryPlan pl{};
  for (size_t a = 0; a < 4; ++a) {
    const int64_t n = a < dims.size() ? dims[a] : 0;
    TORCH_CHECK_VALUE(n >= 0 && n % 2 == 0, "rotary: the channels of an axis must be even, got ", dims);
    pl.half += n / 2;
    pl.end[a] = pl.half;
  }
  TORCH_CHECK_VALUE(pl.half >= 1 && 2 * pl.half <= x.size(3) && pl.half <= 2048, "rotary: dims ", dims,
                    " do not fit ", x.size(3), " channels");
  TORCH_CHECK_VALUE(std::isfinite(theta) && theta > 0, "rotary: theta must be positive and finite, got ", theta);
  TORCH_CHECK_TYPE(pos.scalar_type() == at::kInt || pos.scalar_type() == at::kLong || pos.scalar_type() == at::kFloat,
                   "rotary: positions must be int32, int64 or float32, are ", pos.scalar_type());
  const int64_t A = (int64_t)dims.size(), B = x.size(0), S = x.size(1);
  TORCH_CHECK_VALUE((pos.dim() == 2 && pos.size(0) == A && pos.size(1) == S) ||
                        (pos.dim() == 3 && pos.size(0) == A && (pos.size(1) == B || pos.size(1) == 1) &&
                         pos.size(2) == S),
                    "rotary: positions must be (", A, ", ", S, ") or (", A, ", ", B, ", ", S, "), got ", pos.sizes());
  TORCH_CHECK_VALUE(!pos.requires_grad() && !pos._fw_grad(0).defined(), "rotary: positions have no gradient");
  constexpr int64_t top = (int64_t)1 << 31;
  TORCH_CHECK_VALUE(B < top && S < top && x.size(2) < top && x.size(3) < top, "rotary: too large: x ", x.sizes());
  check_eager("rotary", {&x, &pos});
  TORCH_CHECK(x.is_cuda(), "rotary: x must be a device tensor");
  check_device(pos, x, "rotary: positions");
  pl.theta = theta;
  pl.joint = joint;
  pl.interleaved = interleaved;
  const c10::DeviceGuard guard(x.device());
  if (wants_grad({&x})) return RotaryFn::apply(x, with_sign(pos), pl);
  return rotary_run(x, with_sign(pos), pl, false);
}

}  // namespace

void bind_block_ops(py::module_& m) {
  m.def("attention", &attention, py::arg("q"), py::arg("k"), py::arg("v"), py::arg("mask"), py::arg("lengths"),
        py::arg("causal"), py::arg("scale"), py::arg("return_lse"));
  m.def("attention_qkv", &attention_qkv, py::arg("qkv"), py::arg("heads"), py::arg("kv_heads"), py::arg("mask"),
        py::arg("lengths"), py::arg("causal"), py::arg("scale"), py::arg("return_lse"));
  m.def("layer_norm", &layer_norm, py::arg("x"), py::arg("weight"), py::arg("bias"), py::arg("eps"));
  m.def("rotary", &rotary, py::arg("x"), py::arg("positions"), py::arg("dims"), py::arg("theta"), py::arg("joint"),
        py::arg("interleaved"));
}
