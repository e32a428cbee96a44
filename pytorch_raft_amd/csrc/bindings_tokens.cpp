// Torch registration of the token operators: attention (forward, backward), root-mean-square norm
// (forward, backward, 8-bit output), 8-bit integer product.  Same rules as bindings.cpp: every
// argument is checked on the host before a launch, kernels run on the current stream of the tensors'
// device, outputs and workspaces come from torch's allocator.
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>
#include <ATen/ATen.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <cmath>
#include <initializer_list>
#include <limits>
#include <vector>

#include "kernels/launchers.h"

namespace {

using at::Tensor;
typedef const std::optional<Tensor>& OptTensor;

hipStream_t cur_stream() { return c10::hip::getCurrentHIPStream().stream(); }

bool given(OptTensor t) { return t.has_value() && t->defined(); }

int dtype_code(const Tensor& t, const char* name) {
  const auto st = t.scalar_type();
  TORCH_CHECK(st == at::kBFloat16 || st == at::kHalf || st == at::kFloat, name,
              " must be bfloat16, float16 or float32, got ", st);
  return st == at::kBFloat16 ? 0 : (st == at::kHalf ? 1 : 2);
}

// (B, L, heads, D) whose rows the kernels can read in 16-byte pieces; anything else is copied once.
// heads: that one tile of rows spans (the backward walks the query heads of a group in one).
Tensor token_rows(const Tensor& t, int64_t heads = 1) {
  const int64_t es = t.element_size();
  bool ok = t.stride(3) == 1 && (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0;
  int64_t reach = 0;
  for (int d = 0; d < 3; ++d) {
    if (t.size(d) == 1) continue;
    ok = ok && t.stride(d) * es % 16 == 0 && t.stride(d) >= t.size(3);
    if (d == 1) reach += t.stride(d) * es * std::min<int64_t>(t.size(d), 72);
    if (d == 2) reach += t.stride(d) * es * (heads - 1);
  }
  ok = ok && reach < (int64_t(1) << 30);  // a tile's rows lie within a descriptor's 32-bit offsets
  // (.contiguous() alone would keep a dense tensor that starts off 16 bytes)
  return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}

// stride of a dimension of size 1 is never used: 0 keeps offsets small
int64_t stride_of(const Tensor& t, int d) { return t.size(d) == 1 ? 0 : t.stride(d); }

void check_ints(OptTensor t, const Tensor& like, int64_t n, const char* name) {
  if (!given(t)) return;
  TORCH_CHECK(t->device() == like.device() && t->scalar_type() == at::kInt && t->dim() == 1 &&
                  t->size(0) == n && t->is_contiguous(),
              name, " must be a contiguous int32 tensor of shape (", n, ",) on the device of q");
}

// scores are formed in fp32, in units of log 2: past its range, hidden places (-inf) would meet a factor of 0
// or a score of 0 one of infinity, and become NaN
bool scale_ok(double scale) {
  const double s = scale * 1.4426950408889634;
  return s > 0x1p-150 && s <= (double)std::numeric_limits<float>::max();
}

AttnArgs attn_args(const Tensor& q, const Tensor& k, const Tensor& v, double scale, bool causal,
                   OptTensor mask, OptTensor lengths, OptTensor q_offset) {
  TORCH_CHECK(q.is_cuda() && k.device() == q.device() && v.device() == q.device(),
              "q, k and v must be on one GPU");
  TORCH_CHECK(q.dim() == 4 && k.dim() == 4 && v.sizes() == k.sizes(),
              "q must be (B, Lq, H, D), k and v (B, Lk, Hkv, D)");
  TORCH_CHECK(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(),
              "q, k and v must have one dtype");
  TORCH_CHECK(k.size(0) == q.size(0) && k.size(3) == q.size(3), "q and k disagree on batch or head size");
  TORCH_CHECK(k.size(2) > 0 && q.size(2) > 0 && q.size(2) % k.size(2) == 0,
              "the query heads must be a multiple of the key heads");
  const int64_t B = q.size(0), Lq = q.size(1), H = q.size(2), D = q.size(3), Lk = k.size(1);
  TORCH_CHECK(D >= 8 && D <= 128 && D % 8 == 0, "head size must be a multiple of 8 up to 128, got ", D);
  TORCH_CHECK(scale_ok(scale), "scale must be positive and finite in fp32");
  const int64_t big = int64_t(1) << 26;
  // (grids: less than 2^24 workgroups of 256)
  TORCH_CHECK(B * H * std::max<int64_t>(Lq, 1) < big && B * k.size(2) * std::max<int64_t>(Lk, 1) < big * 16 && Lk < big * 16 &&
                  B * k.size(2) < big / 16,
              "attention: too many rows or heads for one call");
  AttnArgs a = {};
  a.dtype = dtype_code(q, "q");
  a.B = (int)B;
  a.Lq = (int)Lq;
  a.Lk = (int)Lk;
  a.Hkv = (int)k.size(2);
  a.G = (int)(H / k.size(2));
  a.D = (int)D;
  a.DP = (int)((D + 31) / 32 * 32);
  a.scale = (float)scale;
  a.scale_log2 = (float)(scale * 1.4426950408889634);
  a.causal = causal;
  a.q = q.data_ptr();
  a.q_sb = stride_of(q, 0), a.q_sl = stride_of(q, 1), a.q_sh = stride_of(q, 2);
  a.k = k.data_ptr();
  // (one key: a pitch past its row, so that a tile's places behind it read as zeros, not as the key again)
  const auto pitch = [](const Tensor& t) { return t.size(1) == 1 ? t.size(3) : t.stride(1); };
  a.k_sb = stride_of(k, 0), a.k_sl = pitch(k), a.k_sh = stride_of(k, 2);
  a.v = v.data_ptr();
  a.v_sb = stride_of(v, 0), a.v_sl = pitch(v), a.v_sh = stride_of(v, 2);
  check_ints(lengths, q, B, "lengths");
  check_ints(q_offset, q, B, "q_offset");
  a.lengths = given(lengths) ? lengths->data_ptr<int>() : nullptr;
  a.q_offset = given(q_offset) ? q_offset->data_ptr<int>() : nullptr;
  a.nsplit = 1;
  if (given(mask)) {
    const Tensor& m = *mask;
    TORCH_CHECK(m.device() == q.device() && m.scalar_type() == at::kBool && m.dim() == 4 && m.size(0) == B &&
                    m.size(1) == H && m.size(2) == Lq && m.size(3) == Lk,
                "mask must be a bool tensor expanded to (B, H, Lq, Lk) on the device of q");
    a.mask = reinterpret_cast<const uint8_t*>(m.data_ptr());
    a.m_sb = stride_of(m, 0), a.m_sh = stride_of(m, 1), a.m_sq = stride_of(m, 2), a.m_sk = stride_of(m, 3);
    a.mask_mode = a.m_sh == 0 && a.m_sq == 0 ? 1 : 2;
  }
  return a;
}

// -> {out (B, Lq, H, D), log2-sum-exp2 of the rows (B, Hkv, Lq * G) or empty, what out's rounding took away or empty}
std::vector<Tensor> attn_fwd(const Tensor& q0, const Tensor& k0, const Tensor& v0, double scale, bool causal,
                             OptTensor mask, OptTensor lengths, OptTensor q_offset, bool need_lse) {
  TORCH_CHECK(q0.dim() == 4 && k0.dim() == 4 && v0.dim() == 4, "q must be (B, Lq, H, D), k and v (B, Lk, Hkv, D)");
  c10::DeviceGuard g(q0.device());
  const Tensor q = token_rows(q0), k = token_rows(k0), v = token_rows(v0);
  AttnArgs a = attn_args(q, k, v, scale, causal, mask, lengths, q_offset);
  const auto f32 = q.options().dtype(at::kFloat);
  const int64_t R = (int64_t)a.G * a.Lq;
  if (a.B == 0 || a.Lq == 0 || a.Lk == 0)
    return {at::zeros(q.sizes(), q.options()),
            need_lse ? at::full({a.B, a.Hkv, R}, std::numeric_limits<float>::infinity(), f32) : at::empty({0}, f32), at::empty({0}, q.options())};
  Tensor out = at::empty(q.sizes(), q.options().memory_format(at::MemoryFormat::Contiguous));
  Tensor lse = need_lse ? at::empty({a.B, a.Hkv, R}, f32) : at::empty({0}, f32);
  const bool pair = need_lse && a.dtype != 2;
  Tensor lo = pair ? at::empty_like(out) : at::empty({0}, q.options());
  a.o = out.data_ptr();
  a.o_lo = pair ? lo.data_ptr() : nullptr;
  a.lse = need_lse ? lse.data_ptr<float>() : nullptr;
  attn_fwd_plan(a);
  Tensor part;
  if (a.nsplit > 1) {
    const int64_t n = (int64_t)a.B * a.Hkv * a.nsplit * R;
    part = at::empty({n * (a.DP + 2)}, f32);
    a.part = part.data_ptr<float>();
    a.part_ml = a.part + n * a.DP;
  }
  Tensor bits;
  if (const int64_t n = attn_bit_words(a, false)) {
    bits = at::empty({n}, q.options().dtype(at::kLong));
    a.row_bits = reinterpret_cast<uint64_t*>(bits.data_ptr<int64_t>());
  }
  launch_attn_fwd(a, cur_stream());
  return {out, lse, lo};
}

// -> {dq, dk, dv}, contiguous
std::vector<Tensor> attn_bwd(const Tensor& dout0, const Tensor& q0, const Tensor& k0, const Tensor& v0,
                             const Tensor& out, const Tensor& lse, const Tensor& lo, double scale, bool causal,
                             OptTensor mask, OptTensor lengths, OptTensor q_offset) {
  TORCH_CHECK(q0.dim() == 4 && k0.dim() == 4 && v0.dim() == 4, "q must be (B, Lq, H, D), k and v (B, Lk, Hkv, D)");
  c10::DeviceGuard g(q0.device());
  TORCH_CHECK(dout0.device() == q0.device() && dout0.scalar_type() == q0.scalar_type() && dout0.sizes() == q0.sizes(),
              "dout must match q");
  const int64_t group = k0.size(2) > 0 ? std::max<int64_t>(q0.size(2) / k0.size(2), 1) : 1;
  const Tensor q = token_rows(q0, group), k = token_rows(k0), v = token_rows(v0), dout = token_rows(dout0, group);
  AttnArgs a = attn_args(q, k, v, scale, causal, mask, lengths, q_offset);
  const int64_t R = (int64_t)a.G * a.Lq;
  TORCH_CHECK(out.device() == q.device() && out.scalar_type() == q.scalar_type() && out.sizes() == q.sizes() && out.is_contiguous(),
              "out must be the forward's");
  TORCH_CHECK(lse.device() == q.device() && lse.scalar_type() == at::kFloat && lse.is_contiguous() && lse.numel() == (int64_t)a.B * a.Hkv * R,
              "lse must be the forward's");
  TORCH_CHECK(lo.numel() == 0 || (lo.device() == q.device() && lo.scalar_type() == q.scalar_type() && lo.sizes() == q.sizes() && lo.is_contiguous()),
              "lo must be the forward's");
  Tensor dq = at::empty(q.sizes(), q.options().memory_format(at::MemoryFormat::Contiguous));
  Tensor dk = at::empty(k.sizes(), q.options().memory_format(at::MemoryFormat::Contiguous));
  Tensor dv = at::empty(k.sizes(), q.options().memory_format(at::MemoryFormat::Contiguous));
  if (a.B == 0 || a.Lq == 0 || a.Lk == 0) return {dq.zero_(), dk.zero_(), dv.zero_()};
  attn_bwd_plan(a);
  // one workspace: split parts (first: they want 16 bytes), delta, norms
  const int64_t n_kv = a.nsplit_kv > 1 ? 2 * a.nsplit_kv * dk.numel() : 0, n_q = a.nsplit_q > 1 ? a.nsplit_q * dq.numel() : 0;
  const int64_t n_rows = (int64_t)a.B * a.Hkv * R;
  Tensor ws = at::empty({n_kv + n_q + n_rows + (a.dtype == 1 ? 2 * a.nprep : 0)}, q.options().dtype(at::kFloat));
  a.part = ws.data_ptr<float>();
  a.part_q = a.part + n_kv;
  a.o = out.data_ptr();
  a.o_lo = lo.numel() ? lo.data_ptr() : nullptr;
  a.lse = lse.data_ptr<float>();
  a.dout = dout.data_ptr();
  a.d_sb = stride_of(dout, 0), a.d_sl = stride_of(dout, 1), a.d_sh = stride_of(dout, 2);
  a.delta = a.part_q + n_q;
  a.amax = reinterpret_cast<uint32_t*>(a.delta + n_rows);
  a.dq = dq.data_ptr();
  a.dk = dk.data_ptr();
  a.dv = dv.data_ptr();
  Tensor bits;
  if (const int64_t n = attn_bit_words(a, false)) {
    bits = at::empty({n + attn_bit_words(a, true)}, q.options().dtype(at::kLong));
    a.row_bits = reinterpret_cast<uint64_t*>(bits.data_ptr<int64_t>());
    a.key_bits = a.row_bits + n;
  }
  launch_attn_bwd(a, cur_stream());
  return {dq, dk, dv};
}

// ------------------------------------------------------------------ root-mean-square norm
RmsArgs rms_args(const Tensor& x, const Tensor& w, double eps) {
  TORCH_CHECK(x.is_cuda() && w.device() == x.device(), "x and weight must be on one GPU");
  TORCH_CHECK(x.dim() >= 1 && x.is_contiguous(), "x must be contiguous (..., C)");
  TORCH_CHECK(x.size(-1) >= 1 && x.size(-1) <= 16384, "rms norm takes 1 to 16384 channels, got ", x.size(-1));
  TORCH_CHECK(w.dim() == 1 && w.size(0) == x.size(-1) && w.is_contiguous() &&
                  (w.scalar_type() == at::kFloat || w.scalar_type() == x.scalar_type()),
              "weight must be contiguous (C,), float32 or the dtype of x");
  TORCH_CHECK(std::isfinite(eps) && eps >= 0, "eps must be finite and not negative");
  RmsArgs a = {};
  a.dtype = dtype_code(x, "x");
  a.rows = x.numel() / x.size(-1);
  a.C = (int)x.size(-1);
  a.eps = (float)eps;
  a.w = w.data_ptr();
  a.w_f32 = w.scalar_type() == at::kFloat;
  a.x = x.data_ptr();
  return a;
}
void check_like(const Tensor& t, const Tensor& x, const char* name) {
  TORCH_CHECK(t.device() == x.device() && t.scalar_type() == x.scalar_type() && t.sizes() == x.sizes() && t.is_contiguous(),
              name, " must match x (device, dtype, shape, contiguous)");
}

// -> {y, h (the sum; empty without a residual), 1 / rms (rows) or empty}
std::vector<Tensor> rms_fwd(const Tensor& x, const Tensor& w, OptTensor residual, double eps, bool need_rstd) {
  RmsArgs a = rms_args(x, w, eps);
  c10::DeviceGuard g(x.device());
  const auto f32 = x.options().dtype(at::kFloat);
  Tensor y = at::empty_like(x), h = given(residual) ? at::empty_like(x) : at::empty({0}, x.options());
  Tensor rstd = at::empty({need_rstd ? a.rows : 0}, f32);
  if (given(residual)) {
    check_like(*residual, x, "residual");
    a.r = residual->data_ptr();
    a.h = h.data_ptr();
  }
  a.y = y.data_ptr();
  a.rstd = need_rstd ? rstd.data_ptr<float>() : nullptr;
  if (a.rows > 0) launch_rms_fwd(a, cur_stream());
  return {y, h, rstd};
}

// -> {q int8, scale fp32 (rows), h or empty}
std::vector<Tensor> rms_fwd_int8(const Tensor& x, const Tensor& w, OptTensor residual, double eps) {
  RmsArgs a = rms_args(x, w, eps);
  c10::DeviceGuard g(x.device());
  Tensor q = at::empty(x.sizes(), x.options().dtype(at::kChar)), h = given(residual) ? at::empty_like(x) : at::empty({0}, x.options());
  Tensor scale = at::empty(x.sizes().slice(0, x.dim() - 1), x.options().dtype(at::kFloat));
  if (given(residual)) {
    check_like(*residual, x, "residual");
    a.r = residual->data_ptr();
    a.h = h.data_ptr();
  }
  a.y = q.data_ptr();
  a.rstd = scale.data_ptr<float>();
  if (a.rows > 0) launch_rms_int8(a, cur_stream());
  return {q, scale, h};
}

// h: the forward's sum (or x) -> {dx (also the residual's gradient), dw}
std::vector<Tensor> rms_bwd(const Tensor& dy, OptTensor dh, const Tensor& h, const Tensor& w, const Tensor& rstd) {
  RmsArgs a = rms_args(h, w, 0.0);
  c10::DeviceGuard g(h.device());
  check_like(dy, h, "dy");
  TORCH_CHECK(rstd.device() == h.device() && rstd.scalar_type() == at::kFloat && rstd.is_contiguous() && rstd.numel() == a.rows,
              "rstd must be the forward's");
  if (given(dh)) check_like(*dh, h, "dh");
  Tensor dx = at::empty_like(h), dw = at::empty_like(w);
  if (a.rows == 0) return {dx, dw.zero_()};
  a.parts = rms_parts(a.rows, a.C);
  Tensor part = at::empty({a.parts, (int64_t)a.C}, h.options().dtype(at::kFloat));
  a.h = h.data_ptr();
  a.dy = dy.data_ptr();
  a.dh = given(dh) ? dh->data_ptr() : nullptr;
  a.rstd = rstd.data_ptr<float>();
  a.dx = dx.data_ptr();
  a.dw = dw.data_ptr();
  a.part = part.data_ptr<float>();
  launch_rms_bwd(a, cur_stream());
  return {dx, dw};
}

// ------------------------------------------------------------------ 8-bit integer product
void check_vec(const Tensor& t, const Tensor& x, int64_t n, const char* name) {
  TORCH_CHECK(t.device() == x.device() && t.scalar_type() == at::kFloat && t.dim() == 1 && t.size(0) == n && t.is_contiguous(),
              name, " must be contiguous float32 of shape (", n, ",) on the device of x");
}

// out_dtype: 0 bf16, 1 fp16, 2 fp32
Tensor int8_mm(const Tensor& x, const Tensor& xs, const Tensor& w, const Tensor& ws, OptTensor bias, int64_t out_dtype) {
  TORCH_CHECK(x.is_cuda() && w.device() == x.device(), "x and w must be on one GPU");
  TORCH_CHECK(x.scalar_type() == at::kChar && w.scalar_type() == at::kChar, "x and w must be int8");
  TORCH_CHECK(x.dim() == 2 && w.dim() == 2 && x.size(1) == w.size(1) && x.is_contiguous() && w.is_contiguous(),
              "x must be contiguous (M, K), w contiguous (N, K)");
  TORCH_CHECK(out_dtype >= 0 && out_dtype <= 2, "out_dtype: 0 bf16, 1 fp16, 2 fp32");
  const int64_t M = x.size(0), K = x.size(1), N = w.size(0);
  TORCH_CHECK(K <= 131071, "int8_mm: K past 131071 could overflow the 32-bit sums");
  TORCH_CHECK(M < (int64_t(1) << 28) && N < (int64_t(1) << 26) && ((M + 63) / 64) * ((N + 63) / 64) < (int64_t(1) << 23),
              "int8_mm: too many outputs for one call");
  check_vec(xs, x, M, "xs");
  check_vec(ws, x, N, "ws");
  if (given(bias)) check_vec(*bias, x, N, "bias");
  c10::DeviceGuard g(x.device());
  Tensor out = at::empty({M, N}, x.options().dtype(out_dtype == 0 ? at::kBFloat16 : out_dtype == 1 ? at::kHalf : at::kFloat));
  if (M == 0 || N == 0) return out;
  Int8Args a = {};
  a.x = x.data_ptr<int8_t>();
  a.w = w.data_ptr<int8_t>();
  a.xs = xs.data_ptr<float>();
  a.ws = ws.data_ptr<float>();
  a.bias = given(bias) ? bias->data_ptr<float>() : nullptr;
  a.out = out.data_ptr();
  a.M = (int)M;
  a.N = (int)N;
  a.K = (int)K;
  a.dtype = (int)out_dtype;
  Tensor packed;
  if (const int64_t n = int8_packed_bytes(a)) {
    packed = at::empty({n}, x.options());
    a.packed = packed.data_ptr<int8_t>();
  }
  launch_int8_mm(a, cur_stream());
  return out;
}

// ------------------------------------------------------------------ the public operators
// Autograd nodes in C++: for the short launches of small batches the Python form of a node costs more
// host time than the kernels run (a norm's forward and backward: 140 us issued from Python nodes).
using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;

bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }

// the calls below go under autograd unless an input requires a gradient: a tangent would be lost there
void no_tangent(const char* name, std::initializer_list<Tensor> inputs) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  for (const Tensor& t : inputs)
    TORCH_CHECK(!t.defined() || !t._fw_grad(/*level=*/0).defined(), name, " has no forward-mode derivative");
}

// These functions call the kernels without passing the dispatcher again, so what its fallbacks would do is
// done here: a view with a pending negation gets memory of its own, a zero tensor without any is refused.
Tensor held(const Tensor& t) {
  if (!t.defined()) return t;
  TORCH_CHECK(!t._is_zerotensor(), "a zero tensor without memory (torch._efficientzerotensor): materialise it first");
  return t.is_neg() ? t.resolve_neg() : t;  // (resolve_neg passes the dispatcher whether it has work or not)
}
std::optional<Tensor> held(OptTensor t) { return given(t) ? std::optional<Tensor>(held(*t)) : std::nullopt; }

void once_only(const char* name) {
  TORCH_CHECK(!at::GradMode::is_enabled(), name, " has no second derivative (create_graph)");
}

struct AttentionNode : public torch::autograd::Function<AttentionNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, double scale, bool causal,
                        OptTensor mask, OptTensor lengths, OptTensor q_offset) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto r = attn_fwd(q, k, v, scale, causal, mask, lengths, q_offset, true);
    const auto opt = [](OptTensor t) { return given(t) ? *t : Tensor(); };
    ctx->save_for_backward({q, k, v, r[0], r[1], r[2], opt(mask), opt(lengths), opt(q_offset)});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["causal"] = causal;
    return r[0];
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once_only("attention");
    no_tangent("attention's backward", {grads[0]});
    grads[0] = held(grads[0]);
    const auto s = ctx->get_saved_variables();
    const auto opt = [](const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; };
    auto r = attn_bwd(grads[0], s[0], s[1], s[2], s[3], s[4], s[5], ctx->saved_data["scale"].toDouble(),
                      ctx->saved_data["causal"].toBool(), opt(s[6]), opt(s[7]), opt(s[8]));
    return {r[0], r[1], r[2], Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

// q (B, Lq, H, D), k, v (B, Lk, Hkv, D), mask broadcastable to (B, H, Lq, Lk); no scale given: D ** -0.5
Tensor attention(const Tensor& q_in, const Tensor& k_in, const Tensor& v_in, std::optional<double> scale0, bool causal, OptTensor mask0,
                 OptTensor lengths, OptTensor q_offset) {
  const Tensor q0 = held(q_in), k0 = held(k_in), v0 = held(v_in);
  TORCH_CHECK_VALUE(q0.dim() == 4 && k0.dim() == 4 && v0.sizes() == k0.sizes(), "q must be (B, Lq, H, D), k and v (B, Lk, Hkv, D); got ",
                    q0.sizes(), ", ", k0.sizes(), ", ", v0.sizes());
  TORCH_CHECK_TYPE(q0.scalar_type() == k0.scalar_type() && q0.scalar_type() == v0.scalar_type(),
                   "q, k and v must have one dtype, got ", q0.scalar_type(), ", ", k0.scalar_type(), ", ", v0.scalar_type());
  TORCH_CHECK_TYPE(q0.scalar_type() == at::kBFloat16 || q0.scalar_type() == at::kHalf || q0.scalar_type() == at::kFloat,
                   "attention runs in bf16, fp16 and fp32, got ", q0.scalar_type());
  const int64_t B = q0.size(0), Lq = q0.size(1), H = q0.size(2), D = q0.size(3), Lk = k0.size(1), Hkv = k0.size(2);
  TORCH_CHECK_VALUE(k0.size(0) == B && k0.size(3) == D, "q ", q0.sizes(), " and k ", k0.sizes(), " disagree on batch or head size");
  TORCH_CHECK_VALUE(Hkv > 0 && H > 0 && H % Hkv == 0, "the ", H, " query heads must be a multiple of the ", Hkv, " key heads");
  TORCH_CHECK_VALUE(D >= 1 && D <= 128, "head size must be 1 .. 128, got ", D);
  const double scale = scale0.has_value() ? *scale0 : 1.0 / std::sqrt((double)D);
  TORCH_CHECK_VALUE(scale_ok(scale), "scale must be positive and finite in fp32 (2^-150 .. 2^127), got ", scale);
  const auto on = [&](const Tensor& t, const char* name) {
    TORCH_CHECK_VALUE(t.device() == q0.device(), name, " is on ", t.device(), ", q on ", q0.device());
  };
  on(k0, "k"), on(v0, "v");
  const auto ints = [&](OptTensor t, const char* name) -> std::optional<Tensor> {
    if (!given(t)) return std::nullopt;
    on(*t, name);
    TORCH_CHECK_VALUE(t->scalar_type() == at::kInt && t->dim() == 1 && t->size(0) == B, name, " must be int32 of shape (", B, ",), got ",
                      t->scalar_type(), " ", t->sizes());
    return held(*t).contiguous();
  };
  const auto ln = ints(lengths, "lengths"), qo = ints(q_offset, "q_offset");
  std::optional<Tensor> mask;
  if (given(mask0)) {
    on(*mask0, "mask");
    TORCH_CHECK_TYPE(mask0->scalar_type() == at::kBool, "mask must be bool (True = seen), got ", mask0->scalar_type());
    const int64_t want[4] = {B, H, Lq, Lk}, nd = mask0->dim();
    bool fits = nd <= 4;
    for (int64_t d = 0; fits && d < nd; ++d) fits = mask0->size(nd - 1 - d) == 1 || mask0->size(nd - 1 - d) == want[3 - d];
    TORCH_CHECK_VALUE(fits, "mask ", mask0->sizes(), " does not broadcast to (", B, ", ", H, ", ", Lq, ", ", Lk, ")");
    mask = held(*mask0).expand({B, H, Lq, Lk});
  }
  no_tangent("attention", {q0, k0, v0});
  Tensor q = q0, k = k0, v = v0;
  const int64_t pad = (8 - D % 8) % 8;
  if (pad) q = at::constant_pad_nd(q, {0, pad}), k = at::constant_pad_nd(k, {0, pad}), v = at::constant_pad_nd(v, {0, pad});
  Tensor out;
  if (at::GradMode::is_enabled() && (wants_grad(q) || wants_grad(k) || wants_grad(v))) {
    out = AttentionNode::apply(q, k, v, scale, causal, mask, ln, qo);
  } else {
    at::AutoDispatchBelowADInplaceOrView below;
    out = attn_fwd(q, k, v, scale, causal, mask, ln, qo, false)[0];
  }
  return pad ? out.narrow(3, 0, D) : out;
}

void rms_check(const Tensor& x, const Tensor& w, OptTensor residual, double eps) {
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= 16384, "x must be (..., C) with 1 .. 16384 channels, got ", x.sizes());
  TORCH_CHECK_TYPE(x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf || x.scalar_type() == at::kFloat,
                   "rms_norm runs in bf16, fp16 and fp32, got ", x.scalar_type());
  TORCH_CHECK_VALUE(w.dim() == 1 && w.size(0) == x.size(-1), "weight ", w.sizes(), " does not match the channels of x ", x.sizes());
  TORCH_CHECK_TYPE(w.scalar_type() == at::kFloat || w.scalar_type() == x.scalar_type(), "weight must be float32 or ", x.scalar_type(),
                   ", got ", w.scalar_type());
  TORCH_CHECK_VALUE(w.device() == x.device(), "weight is on ", w.device(), ", x on ", x.device());
  if (given(residual)) {
    TORCH_CHECK_VALUE(residual->sizes() == x.sizes() && residual->scalar_type() == x.scalar_type(), "residual ", residual->scalar_type(),
                      " ", residual->sizes(), " does not match x ", x.scalar_type(), " ", x.sizes());
    TORCH_CHECK_VALUE(residual->device() == x.device(), "residual is on ", residual->device(), ", x on ", x.device());
  }
  TORCH_CHECK_VALUE(std::isfinite(eps) && eps >= 0, "eps must be finite and not negative, got ", eps);
}

OptTensor no_tensor = std::nullopt;
std::optional<Tensor> dense(OptTensor t) { return given(t) ? std::optional<Tensor>(t->contiguous()) : std::nullopt; }

struct RmsNormNode : public torch::autograd::Function<RmsNormNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, OptTensor residual, double eps) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto r = rms_fwd(x.contiguous(), w.contiguous(), dense(residual), eps, true);
    ctx->set_materialize_grads(false);
    const bool sum = given(residual);
    ctx->saved_data["sum"] = sum;
    ctx->save_for_backward({sum ? r[1] : x, w, r[2]});
    if (sum) return {r[0], r[1]};
    return {r[0]};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once_only("rms_norm");
    for (Tensor& t : grads) {
      no_tangent("rms_norm's backward", {t});
      t = held(t);
    }
    const auto s = ctx->get_saved_variables();
    const bool sum = ctx->saved_data["sum"].toBool();
    const Tensor dh = sum ? grads[1] : Tensor();
    if (!grads[0].defined()) return {dh, Tensor(), dh, Tensor()};
    auto r = rms_bwd(grads[0].contiguous(), dh.defined() ? std::optional<Tensor>(dh.contiguous()) : std::nullopt, s[0].contiguous(),
                     s[1].contiguous(), s[2]);
    return {r[0], r[1], sum ? r[0] : Tensor(), Tensor()};
  }
};

Tensor rms_norm(const Tensor& x_in, const Tensor& w_in, double eps) {
  const Tensor x = held(x_in), w = held(w_in);
  rms_check(x, w, no_tensor, eps);
  no_tangent("rms_norm", {x, w});
  if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(w))) return RmsNormNode::apply(x, w, std::optional<Tensor>(), eps)[0];
  at::AutoDispatchBelowADInplaceOrView below;
  return rms_fwd(x.contiguous(), w.contiguous(), no_tensor, eps, false)[0];
}

std::tuple<Tensor, Tensor> rms_norm_residual(const Tensor& x_in, const Tensor& w_in, const Tensor& residual_in, double eps) {
  const Tensor x = held(x_in), w = held(w_in), residual = held(residual_in);
  rms_check(x, w, residual, eps);
  no_tangent("rms_norm", {x, w, residual});
  if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(w) || wants_grad(residual))) {
    auto r = RmsNormNode::apply(x, w, std::optional<Tensor>(residual), eps);
    return {r[0], r[1]};
  }
  at::AutoDispatchBelowADInplaceOrView below;
  auto r = rms_fwd(x.contiguous(), w.contiguous(), residual.contiguous(), eps, false);
  return {r[0], r[1]};
}

// {q, scale} or {q, scale, h}
std::vector<Tensor> rms_norm_int8(const Tensor& x_in, const Tensor& w_in, OptTensor residual_in, double eps) {
  const Tensor x = held(x_in), w = held(w_in);
  const std::optional<Tensor> residual = held(residual_in);
  rms_check(x, w, residual, eps);
  TORCH_CHECK(!at::GradMode::is_enabled() || !(wants_grad(x) || wants_grad(w) || (given(residual) && wants_grad(*residual))),
              "rms_norm_int8 has no gradient: call it under torch.no_grad()");
  no_tangent("rms_norm_int8", {x, w, given(residual) ? *residual : Tensor()});
  at::AutoDispatchBelowADInplaceOrView below;
  auto r = rms_fwd_int8(x.contiguous(), w.contiguous(), dense(residual), eps);
  if (!given(residual)) r.pop_back();
  return r;
}

// x (..., K) int8, x_scale (...), w (N, K) int8, w_scale (N)
Tensor int8_linear(const Tensor& x_in, const Tensor& xs_in, const Tensor& w_in, const Tensor& ws_in, OptTensor bias_in, int64_t out_dtype) {
  const Tensor x = held(x_in), xs = held(xs_in), w = held(w_in), ws = held(ws_in);
  const std::optional<Tensor> bias = held(bias_in);
  TORCH_CHECK_TYPE(x.scalar_type() == at::kChar && w.scalar_type() == at::kChar, "x and w must be int8, got ", x.scalar_type(), " and ",
                   w.scalar_type());
  TORCH_CHECK_VALUE(x.dim() >= 1 && w.dim() == 2 && x.size(-1) == w.size(1), "x must be (..., K), w (N, K); got ", x.sizes(), ", ", w.sizes());
  TORCH_CHECK_VALUE(w.size(1) <= 131071, "K = ", w.size(1), " could overflow the 32-bit sums (at most 131071)");
  const auto lead = x.sizes().slice(0, x.dim() - 1);
  const auto vec = [&](const Tensor& t, at::IntArrayRef shape, const char* name) {
    TORCH_CHECK_VALUE(t.scalar_type() == at::kFloat && t.sizes() == shape, name, " must be float32 of shape ", shape, ", got ", t.scalar_type(),
                      " ", t.sizes());
    TORCH_CHECK(!at::GradMode::is_enabled() || !wants_grad(t), "int8_linear has no gradient (", name,
                " requires one): call it under torch.no_grad()");
    TORCH_CHECK_VALUE(t.device() == x.device(), name, " is on ", t.device(), ", x on ", x.device());
  };
  vec(xs, lead, "x_scale");
  vec(ws, {w.size(0)}, "w_scale");
  if (given(bias)) vec(*bias, {w.size(0)}, "bias");
  TORCH_CHECK_VALUE(w.device() == x.device(), "w is on ", w.device(), ", x on ", x.device());
  no_tangent("int8_linear", {xs, ws, given(bias) ? *bias : Tensor()});
  at::AutoDispatchBelowADInplaceOrView below;
  int64_t M = 1;
  for (const int64_t n : lead) M *= n;
  std::vector<int64_t> shape(lead.begin(), lead.end());
  shape.push_back(w.size(0));
  return int8_mm(x.contiguous().view({M, x.size(-1)}), xs.contiguous().view({M}), w.contiguous(), ws.contiguous(),
                 given(bias) ? std::optional<Tensor>(bias->contiguous()) : std::nullopt, out_dtype)
      .view(shape);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(raft_amd, m) {
  m.def("attention(Tensor q, Tensor k, Tensor v, float? scale, bool causal, Tensor? mask, Tensor? lengths, Tensor? q_offset) -> Tensor");
  m.def("rms_norm(Tensor x, Tensor w, float eps) -> Tensor");
  m.def("rms_norm_residual(Tensor x, Tensor w, Tensor residual, float eps) -> (Tensor, Tensor)");
  m.def("rms_norm_int8(Tensor x, Tensor w, Tensor? residual, float eps) -> Tensor[]");
  m.def("int8_linear(Tensor x, Tensor xs, Tensor w, Tensor ws, Tensor? bias, int out_dtype) -> Tensor");
  m.def("attn_fwd(Tensor q, Tensor k, Tensor v, float scale, bool causal, Tensor? mask, Tensor? lengths, Tensor? q_offset, bool need_lse) -> Tensor[]");
  m.def("attn_bwd(Tensor dout, Tensor q, Tensor k, Tensor v, Tensor out, Tensor lse, Tensor lo, float scale, bool causal, Tensor? mask, Tensor? lengths, Tensor? q_offset) -> Tensor[]");
  m.def("rms_fwd(Tensor x, Tensor w, Tensor? residual, float eps, bool need_rstd) -> Tensor[]");
  m.def("rms_fwd_int8(Tensor x, Tensor w, Tensor? residual, float eps) -> Tensor[]");
  m.def("rms_bwd(Tensor dy, Tensor? dh, Tensor h, Tensor w, Tensor rstd) -> Tensor[]");
  m.def("int8_mm(Tensor x, Tensor xs, Tensor w, Tensor ws, Tensor? bias, int out_dtype) -> Tensor");
}

TORCH_LIBRARY_IMPL(raft_amd, CUDA, m) {
  m.impl("attn_fwd", &attn_fwd);
  m.impl("attn_bwd", &attn_bwd);
  m.impl("rms_fwd", &rms_fwd);
  m.impl("rms_fwd_int8", &rms_fwd_int8);
  m.impl("rms_bwd", &rms_bwd);
  m.impl("int8_mm", &int8_mm);
  m.impl("attention", &attention);
  m.impl("rms_norm", &rms_norm);
  m.impl("rms_norm_residual", &rms_norm_residual);
  m.impl("rms_norm_int8", &rms_norm_int8);
  m.impl("int8_linear", &int8_linear);
}

TORCH_LIBRARY_IMPL(raft_amd, AutogradCUDA, m) {
  m.impl("attention", &attention);
  m.impl("rms_norm", &rms_norm);
  m.impl("rms_norm_residual", &rms_norm_residual);
  m.impl("rms_norm_int8", &rms_norm_int8);
  m.impl("int8_linear", &int8_linear);
}
