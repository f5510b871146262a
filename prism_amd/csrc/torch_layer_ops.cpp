// PyTorch operators of what runs around and beside the block-sparse attention
// (TORCH_LIBRARY_FRAGMENT(prism)): row norms, rotary positions and window
// attention.  As in torch_ops.cpp, each wraps one extern "C" entry point of
// include/prism_bsa.h, checks what the kernels assume, allocates its outputs
// and workspaces through the caching allocator and launches on the current HIP
// stream of its tensors' device.
//
// The gradients are autograd nodes in C++ (the Autograd kernels at the end): a
// training step of a small layer is bound by the host, and a node in Python
// costs the backward thread 27 us of it (rms_norm forward and backward of a few
// rows: 102 us against 75).
#include "torch_layer.h"

namespace {

// ------------------------------------------------------------------ row norms
Tensor rows_of(const Tensor& t) {  // [M, N] with adjacent columns
  const Tensor r = t.dim() == 2 ? t : t.numel() ? t.reshape({-1, t.size(-1)}) : t.new_empty({0, t.size(-1)});
  return unit_rows(r);
}
// x [.., N]: y, h (with a residual), scale (8-bit outputs), 1 / rms (on request)
Outputs rms_norm(const Tensor& x_, const OptT& r_, const OptT& w_, double eps,
                                                    int64_t out_code, bool want_inv) {
  on_gpu(x_, "x");
  same_device(x_, r_, "residual");
  same_device(x_, w_, "weight");
  TORCH_CHECK_VALUE(x_.dim() >= 1 && x_.size(-1) >= 1, "rms_norm: x must be [.., N]");
  const int dt = type_code(x_, "rms_norm");
  const int64_t N = x_.size(-1), M = x_.numel() / N;
  check_dtype(r_, x_.scalar_type(), "residual");
  if (r_) TORCH_CHECK_VALUE(r_->sizes() == x_.sizes(), "rms_norm: residual must have x's shape");
  if (w_) TORCH_CHECK_VALUE(w_->dim() == 1 && w_->size(0) == N, "rms_norm: weight must be [N]");
  const int wdt = w_ ? type_code(*w_, "rms_norm weight") : dt;
  const c10::DeviceGuard guard(x_.device());
  const Tensor x = rows_of(x_);
  const OptT r = r_ ? OptT(rows_of(*r_)) : OptT(), w = cont(w_);
  const at::ScalarType ot = out_code == PRISM_E4M3 ? at::kFloat8_e4m3fn : out_code == PRISM_I8 ? at::kChar : x.scalar_type();
  const bool quant = out_code == PRISM_E4M3 || out_code == PRISM_I8;
  Outputs out{at::empty(x_.sizes(), opts(x, ot))};
  Tensor h, scale, inv;
  if (r) out.push_back(h = at::empty(x_.sizes(), x.options()));
  if (quant) out.push_back(scale = at::empty(x_.sizes().slice(0, x_.dim() - 1), opts(x, at::kFloat)));
  if (want_inv) out.push_back(inv = at::empty({M}, opts(x, at::kFloat)));
  PRISM_TORCH_CALL(prism_rms_norm, x.data_ptr(), x.stride(0), p(r), r ? r->stride(0) : 0, p(w), wdt, dt, M,
                   small(N, "N"), (float)eps, r ? h.data_ptr() : nullptr, out[0].data_ptr(),
                   (int)(quant ? out_code : dt), quant ? scale.data_ptr<float>() : nullptr,
                   want_inv ? inv.data_ptr<float>() : nullptr, stream_of(x));
  return out;
}

// dx, and dw on request
Outputs rms_norm_bwd(const Tensor& dy_, const OptT& dh_, const Tensor& h_, const OptT& w_, const Tensor& inv_,
                     bool want_dw) {
  on_gpu(h_, "h");
  same_device(h_, dy_, "dy");
  same_device(h_, dh_, "dh");
  same_device(h_, w_, "weight");
  same_device(h_, inv_, "inv");
  TORCH_CHECK_VALUE(h_.dim() >= 1 && h_.size(-1) >= 1, "rms_norm_bwd: h must be [.., N]");
  const int dt = type_code(h_, "rms_norm_bwd");
  const int64_t N = h_.size(-1), M = h_.numel() / N;
  check_dtype(dy_, h_.scalar_type(), "dy");
  check_dtype(dh_, h_.scalar_type(), "dh");
  check_dtype(inv_, at::kFloat, "inv");
  TORCH_CHECK_VALUE(dy_.sizes() == h_.sizes() && (!dh_ || dh_->sizes() == h_.sizes()),
                    "rms_norm_bwd: gradients must have h's shape");
  TORCH_CHECK_VALUE(inv_.numel() == M, "rms_norm_bwd: inv must be [M]");
  if (w_) TORCH_CHECK_VALUE(w_->dim() == 1 && w_->size(0) == N, "rms_norm_bwd: weight must be [N]");
  TORCH_CHECK_VALUE(!want_dw || w_, "rms_norm_bwd: a weight gradient needs the weight");
  const int wdt = w_ ? type_code(*w_, "rms_norm weight") : dt;
  const c10::DeviceGuard guard(h_.device());
  const Tensor h = rows_of(h_), dy = rows_of(dy_), inv = inv_.contiguous();
  const OptT dh = dh_ ? OptT(rows_of(*dh_)) : OptT(), w = cont(w_);
  Tensor dx = at::empty(h_.sizes(), h.options());
  Outputs out{dx};
  Tensor dw, partial;
  if (want_dw) out.push_back(dw = M == 0 ? at::zeros({N}, w->options()) : at::empty({N}, w->options()));
  if (M == 0) return out;
  int parts = 0;
  check_rc(prism_rms_norm_parts(M, small(N, "N"), &parts));
  if (want_dw) partial = at::empty({parts, N}, opts(h, at::kFloat));
  PRISM_TORCH_CALL(prism_rms_norm_bwd, dy.data_ptr(), dy.stride(0), p(dh), dh ? dh->stride(0) : 0, h.data_ptr(),
                   h.stride(0), p(w), wdt, dt, M, small(N, "N"), inv.data_ptr<float>(), dx.data_ptr(),
                   want_dw ? partial.data_ptr<float>() : nullptr, parts, want_dw ? dw.data_ptr() : nullptr,
                   stream_of(h));
  return out;
}

// ------------------------------------------------------------------ rotary positions
// q', and k' where there is a k
Outputs rotary(const Tensor& q_, const OptT& k_, const Tensor& freqs_, const Tensor& pos_, c10::IntArrayRef axis_pairs,
               bool interleaved, double amplitude, bool inverse) {
  on_gpu(q_, "q");
  same_device(q_, k_, "k");
  same_device(q_, freqs_, "freqs");
  same_device(q_, pos_, "positions");
  TORCH_CHECK_VALUE(q_.dim() == 4, "rotary: q must be [B, H, S, D]");
  const int dt = type_code(q_, "rotary");
  check_dtype(freqs_, at::kDouble, "freqs");
  check_dtype(k_, q_.scalar_type(), "k");
  const int64_t B = q_.size(0), S = q_.size(2), D = q_.size(3);
  if (k_)
    TORCH_CHECK_VALUE(k_->dim() == 4 && k_->size(0) == B && k_->size(2) == S && k_->size(3) == D,
                      "rotary: k must be [B, Hk, S, D] with q's B, S and D");
  TORCH_CHECK_VALUE(freqs_.dim() == 1, "rotary: freqs must be [pairs]");
  TORCH_CHECK_TYPE(pos_.scalar_type() == at::kInt || pos_.scalar_type() == at::kLong,
                   "prism: positions must be int32 or int64, got ", pos_.scalar_type());
  // positions [S], [B, S], and with axes [S, A], [B, S, A]
  const int64_t A = axis_pairs.empty() ? 1 : (int64_t)axis_pairs.size();
  const bool has_axis = !axis_pairs.empty();
  const int64_t rank = pos_.dim() - (has_axis ? 1 : 0);
  TORCH_CHECK_VALUE((rank == 1 || rank == 2) && pos_.size(rank - 1) == S && (rank == 1 || pos_.size(0) == B || pos_.size(0) == 1) &&
                        (!has_axis || pos_.size(-1) == A),
                    "rotary: positions must be [S] or [B, S]", has_axis ? " with one entry per axis" : "", ", got ",
                    pos_.sizes());
  TORCH_CHECK_VALUE(A <= 4, "rotary: at most 4 axes");
  const c10::DeviceGuard guard(q_.device());
  const Tensor q = unit_rows(q_), freqs = freqs_.contiguous();
  const OptT k = k_ ? OptT(unit_rows(*k_)) : OptT();
  Tensor oq = like_layout(q_), ok;
  if (k_) ok = like_layout(*k_);
  int64_t strides[12] = {q.stride(0), q.stride(1), q.stride(2), oq.stride(0), oq.stride(1), oq.stride(2)};
  if (k) {
    const int64_t s[6] = {k->stride(0), k->stride(1), k->stride(2), ok.stride(0), ok.stride(1), ok.stride(2)};
    for (int i = 0; i < 6; ++i) strides[6 + i] = s[i];
  }
  const int64_t pos_strides[3] = {rank == 2 && pos_.size(0) > 1 ? pos_.stride(0) : 0, pos_.stride(rank - 1),
                                  has_axis ? pos_.stride(-1) : 0};
  int32_t axis_end[4] = {};
  int64_t at = 0;
  for (int64_t a = 0; a < A; ++a) {
    at += has_axis ? axis_pairs[a] : freqs.numel();
    TORCH_CHECK_VALUE(!has_axis || axis_pairs[a] >= 0, "rotary: negative axis size");
    axis_end[a] = small(at, "pairs");
  }
  PRISM_TORCH_CALL(prism_rotary, q.data_ptr(), p(k), dt, small(B, "B"), S, small(q.size(1), "heads"),
                   k ? small(k->size(1), "heads") : 0, small(D, "D"), small(2 * freqs.numel(), "rotary dim"), strides,
                   freqs.data_ptr<double>(), pos_.data_ptr(), pos_.scalar_type() == at::kLong, pos_strides, (int)A,
                   axis_end, interleaved, (float)amplitude, inverse, oq.data_ptr(), k ? ok.data_ptr() : nullptr,
                   stream_of(q));
  return k ? Outputs{oq, ok} : Outputs{oq};
}

// ------------------------------------------------------------------ window attention
// t as the window kernels take it: adjacent channels, 16-byte aligned rows at
// strides of whole 16-byte pieces; else a contiguous copy
Tensor win_rows(const Tensor& t) {
  bool ok = t.numel() == 0 || (t.stride(3) == 1 && (uintptr_t)t.data_ptr() % 16 == 0);
  for (int d = 0; d < 3 && ok; ++d) ok = t.size(d) <= 1 || t.stride(d) % 8 == 0;
  if (ok && t.size(2) > 1) ok = t.stride(2) < (1 << 24);
  return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}
void win_strides(const Tensor& t, int64_t* s) {
  for (int d = 0; d < 3; ++d) s[d] = t.size(d) > 1 ? t.stride(d) : 0;
}
// t's layout where that is dense, has adjacent channels and rows as near as the kernels take them
Tensor win_like(const Tensor& t) {
  Tensor o = at::empty_like(t);
  const bool ok = o.numel() == 0 || (o.stride(3) == 1 && (o.size(2) <= 1 || o.stride(2) < (1 << 24)));
  return ok ? o : at::empty(t.sizes(), t.options());
}

struct WinShape {
  int dt;
  int64_t B, Hq, Hk, Sq, Sk, D;
};
WinShape check_window(const Tensor& q, const Tensor& k, const Tensor& v, const OptT& q_lens, const OptT& kv_lens) {
  on_gpu(q, "q");
  same_device(q, k, "k");
  same_device(q, v, "v");
  same_device(q, q_lens, "q_lens");
  same_device(q, kv_lens, "kv_lens");
  TORCH_CHECK_TYPE(q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kHalf,
                   "prism: window attention takes bfloat16 or float16, got ", q.scalar_type());
  check_dtype(k, q.scalar_type(), "k");
  check_dtype(v, q.scalar_type(), "v");
  TORCH_CHECK_VALUE(q.dim() == 4 && k.dim() == 4 && k.sizes() == v.sizes() && k.size(0) == q.size(0) &&
                        k.size(3) == q.size(3),
                    "window attention: q must be [B, Hq, Sq, D], k and v [B, Hk, Sk, D], got ", q.sizes(), ", ",
                    k.sizes(), ", ", v.sizes());
  WinShape s{q.scalar_type() == at::kBFloat16 ? PRISM_BF16 : PRISM_F16, q.size(0), q.size(1), k.size(1), q.size(2),
             k.size(2), q.size(3)};
  for (const OptT* l : {&q_lens, &kv_lens}) {
    check_dtype(*l, at::kInt, "lengths");
    if (*l) TORCH_CHECK_VALUE((*l)->dim() == 1 && (*l)->size(0) == s.B, "window attention: lengths must be [B]");
  }
  return s;
}

// o, lse and what o's rounding left off on request
Outputs window_fwd(const Tensor& q_, const Tensor& k_, const Tensor& v_, int64_t window, int64_t sinks, bool causal,
                   const OptT& q_lens_, const OptT& kv_lens_, double sm_scale, bool want_lse, bool want_rest) {
  const WinShape s = check_window(q_, k_, v_, q_lens_, kv_lens_);
  const c10::DeviceGuard guard(q_.device());
  const Tensor q = win_rows(q_), k = win_rows(k_), v = win_rows(v_);
  const OptT q_lens = cont(q_lens_), kv_lens = cont(kv_lens_);
  Tensor o = win_like(q_);
  Tensor lse, rest;
  Outputs out{o};
  if (want_lse) out.push_back(lse = at::empty({s.B, s.Hq, s.Sq}, opts(q, at::kFloat)));
  if (want_rest) out.push_back(rest = at::empty_like(o));
  void* rp = want_rest ? rest.data_ptr() : nullptr;
  int64_t st[12];
  win_strides(q, st);
  win_strides(k, st + 3);
  win_strides(v, st + 6);
  win_strides(o, st + 9);
  float* lp = want_lse ? lse.data_ptr<float>() : nullptr;
  const int B = small(s.B, "B"), Hq = small(s.Hq, "heads"), Hk = small(s.Hk, "heads"), D = small(s.D, "D");
  int splits = 0;
  int64_t floats = 0;
  check_rc(prism_window_token_plan(B, Hq, Hk, s.Sq, s.Sk, window, sinks, causal, &splits, &floats));
  if (splits) {
    Tensor part;
    if (splits > 1) part = at::empty({floats * (s.D + 2)}, opts(q, at::kFloat));
    float* po = splits > 1 ? part.data_ptr<float>() : nullptr;
    PRISM_TORCH_CALL(prism_window_token, q.data_ptr(), k.data_ptr(), v.data_ptr(), s.dt, B, Hq, Hk, s.Sq, s.Sk, D, st,
                     window, sinks, causal, (const int32_t*)p(q_lens), (const int32_t*)p(kv_lens), (float)sm_scale,
                     o.data_ptr(), rp, lp, splits, po, po ? po + floats * s.D : nullptr, stream_of(q));
    return out;
  }
  check_rc(prism_window_fwd_plan(B, Hq, Hk, s.Sq, s.Sk, D, window, sinks, causal, &floats));
  Tensor part;
  if (floats) part = at::empty({floats}, opts(q, at::kFloat));
  PRISM_TORCH_CALL(prism_window_fwd, q.data_ptr(), k.data_ptr(), v.data_ptr(), s.dt, B, Hq, Hk, s.Sq, s.Sk, D, st,
                   window, sinks, causal, (const int32_t*)p(q_lens), (const int32_t*)p(kv_lens), (float)sm_scale,
                   o.data_ptr(), rp, lp, floats ? part.data_ptr<float>() : nullptr, stream_of(q));
  return out;
}

std::tuple<Tensor, Tensor, Tensor> window_bwd(const Tensor& do_, const Tensor& q_, const Tensor& k_, const Tensor& v_,
                                              const Tensor& o_, const OptT& rest_, const Tensor& lse_, int64_t window, int64_t sinks,
                                              bool causal, const OptT& q_lens_, const OptT& kv_lens_,
                                              double sm_scale) {
  const WinShape s = check_window(q_, k_, v_, q_lens_, kv_lens_);
  for (const auto& t : {std::make_pair(&do_, "do"), std::make_pair(&o_, "o")}) {
    same_device(q_, *t.first, t.second);
    check_dtype(*t.first, q_.scalar_type(), t.second);
    TORCH_CHECK_VALUE(t.first->sizes() == q_.sizes(), "window_bwd: ", t.second, " must have q's shape");
  }
  same_device(q_, rest_, "rest");
  check_dtype(rest_, q_.scalar_type(), "rest");
  if (rest_)
    TORCH_CHECK_VALUE(rest_->sizes() == o_.sizes() && rest_->strides() == o_.strides(),
                      "window_bwd: rest must have o's shape and strides");
  same_device(q_, lse_, "lse");
  check_dtype(lse_, at::kFloat, "lse");
  TORCH_CHECK_VALUE(lse_.numel() == s.B * s.Hq * s.Sq, "window_bwd: lse must be [B, Hq, Sq]");
  const c10::DeviceGuard guard(q_.device());
  const Tensor q = win_rows(q_), k = win_rows(k_), v = win_rows(v_), o = win_rows(o_), d = win_rows(do_);
  const OptT rest = rest_ ? OptT(win_rows(*rest_)) : OptT();
  if (rest)
    for (int x = 0; x < 4; ++x)
      TORCH_CHECK(rest->stride(x) == o.stride(x), "window_bwd: rest must be laid out like o");
  const Tensor lse = lse_.contiguous();
  const OptT q_lens = cont(q_lens_), kv_lens = cont(kv_lens_);
  Tensor dq = win_like(q_), dk = win_like(k_), dv = win_like(v_);
  int64_t st[24], floats = 0;
  const Tensor* all[8] = {&q, &k, &v, &o, &d, &dq, &dk, &dv};
  for (int i = 0; i < 8; ++i) win_strides(*all[i], st + 3 * i);
  const int B = small(s.B, "B"), Hq = small(s.Hq, "heads"), Hk = small(s.Hk, "heads"), D = small(s.D, "D");
  check_rc(prism_window_bwd_plan(B, Hq, Hk, s.Sq, s.Sk, D, window, sinks, causal, kv_lens.has_value(), &floats));
  Tensor work = at::empty({floats + 2 * s.B * s.Hq * s.Sq}, opts(q, at::kFloat));  // acc, then rows
  float* acc = work.data_ptr<float>();
  PRISM_TORCH_CALL(prism_window_bwd, d.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(),
                   p(rest), lse.data_ptr<float>(), s.dt, B, Hq, Hk, s.Sq, s.Sk, D, st, window, sinks, causal,
                   (const int32_t*)p(q_lens), (const int32_t*)p(kv_lens), (float)sm_scale, dq.data_ptr(), dk.data_ptr(),
                   dv.data_ptr(), acc + floats, floats ? acc : nullptr, stream_of(q));
  return {dq, dk, dv};
}

// ------------------------------------------------------------------ gradients
struct RmsNormGrad : torch::autograd::Function<RmsNormGrad> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const OptT& r, const OptT& w, double eps,
                               int64_t out_code, bool want_inv) {
    at::AutoDispatchBelowADInplaceOrView guard;
    ctx->set_materialize_grads(false);
    variable_list o = PRISM_OP(rms_norm).call(x, r, w, eps, out_code, true);  // y, h with a residual, inv
    ctx->save_for_backward({r ? o[1] : x, w ? *w : Tensor(), o.back()});
    ctx->saved_data["residual"] = r.has_value();
    ctx->saved_data["dw"] = w && w->requires_grad();
    // (what is only kept is no output of the node: each costs the host 2 us)
    if (want_inv) ctx->mark_non_differentiable({o.back()});
    else o.pop_back();
    return o;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const variable_list saved = ctx->get_saved_variables();
    const bool residual = ctx->saved_data["residual"].toBool();
    const Tensor dh = residual ? g[1] : Tensor();
    if (!g[0].defined() && !dh.defined()) return variable_list(6);
    const Outputs d = [&] {
      at::AutoDispatchBelowADInplaceOrView guard;
      const Tensor dy = g[0].defined() ? g[0] : at::zeros_like(dh);  // (only h went on)
      return PRISM_OP(rms_norm_bwd).call(dy, opt(dh), saved[0], opt(saved[1]), saved[2], ctx->saved_data["dw"].toBool());
    }();
    return once({d[0], residual ? d[0] : Tensor(), d.size() > 1 ? d[1] : Tensor(), Tensor(), Tensor(), Tensor()});
  }
};
Outputs rms_norm_autograd(const Tensor& x, const OptT& r, const OptT& w, double eps, int64_t out_code, bool want_inv) {
  check_no_tangents("rms_norm", x, r, w);
  if (!grads_wanted(x, r, w)) {
    at::AutoDispatchBelowADInplaceOrView guard;
    return PRISM_OP(rms_norm).call(x, r, w, eps, out_code, want_inv);
  }
  TORCH_CHECK_VALUE(out_code != PRISM_E4M3 && out_code != PRISM_I8, "rms_norm: 8-bit outputs have no gradient");
  return RmsNormGrad::apply(x, r, w, eps, out_code, want_inv);
}

struct RotaryGrad : torch::autograd::Function<RotaryGrad> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const OptT& k, const Tensor& freqs,
                               const Tensor& pos, std::vector<int64_t> axis_pairs, bool interleaved, double amplitude,
                               bool inverse) {
    at::AutoDispatchBelowADInplaceOrView guard;
    ctx->set_materialize_grads(false);
    const variable_list o = PRISM_OP(rotary).call(q, k, freqs, pos, axis_pairs, interleaved, amplitude, inverse);
    ctx->save_for_backward({freqs, pos});
    ctx->saved_data["axis_pairs"] = axis_pairs;
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["amplitude"] = amplitude;
    ctx->saved_data["inverse"] = inverse;
    return o;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    variable_list out(8);
    const Tensor dq = g[0], dk = g.size() > 1 ? g[1] : Tensor();
    if (!dq.defined() && !dk.defined()) return out;
    const variable_list saved = ctx->get_saved_variables();
    const bool both = dq.defined() && dk.defined();
    const Outputs d = [&] {
      at::AutoDispatchBelowADInplaceOrView guard;
      return PRISM_OP(rotary).call(dq.defined() ? dq : dk, both ? OptT(dk) : OptT(), saved[0], saved[1],
                    ctx->saved_data["axis_pairs"].toIntVector(), ctx->saved_data["interleaved"].toBool(),
                    ctx->saved_data["amplitude"].toDouble(), !ctx->saved_data["inverse"].toBool());
    }();
    if (dq.defined()) out[0] = d[0];
    if (dk.defined()) out[1] = d[both ? 1 : 0];
    return once(std::move(out));
  }
};
Outputs rotary_autograd(const Tensor& q, const OptT& k, const Tensor& freqs, const Tensor& pos,
                        c10::IntArrayRef axis_pairs, bool interleaved, double amplitude, bool inverse) {
  check_no_tangents("rotary", q, k, freqs);
  if (!grads_wanted(q, k)) {
    at::AutoDispatchBelowADInplaceOrView guard;
    return PRISM_OP(rotary).call(q, k, freqs, pos, axis_pairs, interleaved, amplitude, inverse);
  }
  return RotaryGrad::apply(q, k, freqs, pos, axis_pairs.vec(), interleaved, amplitude, inverse);
}

// prism_window_rest without fixing a length that is symbolic (a traced program): a
// window and sinks that reach 64 keys at most at any length, or a length of 64 at
// most, which as a bound serves all lengths on its side of it.
bool window_rest(const Tensor& k, int64_t window, int64_t sinks, bool causal) {
  return prism_window_rest(int64_t{1} << 40, window, sinks, causal) &&
         k.sym_size(2).sym_gt(64).guard_bool(__FILE__, __LINE__);
}

struct WindowGrad : torch::autograd::Function<WindowGrad> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, int64_t window,
                               int64_t sinks, bool causal, const OptT& q_lens, const OptT& kv_lens, double sm_scale,
                               bool want_lse, bool want_rest) {
    at::AutoDispatchBelowADInplaceOrView guard;
    ctx->set_materialize_grads(false);
    const bool use = window_rest(k, window, sinks, causal), keep = use || want_rest;
    const variable_list o = PRISM_OP(window_fwd).call(q, k, v, window, sinks, causal, q_lens, kv_lens, sm_scale, true, keep);
    ctx->save_for_backward({q, k, v, o[0], o[1], q_lens ? *q_lens : Tensor(), kv_lens ? *kv_lens : Tensor(),
                            use ? o[2] : Tensor()});
    ctx->saved_data["window"] = window;
    ctx->saved_data["sinks"] = sinks;
    ctx->saved_data["causal"] = causal;
    ctx->saved_data["sm_scale"] = sm_scale;
    variable_list out{o[0]};
    if (want_lse) out.push_back(o[1]);
    if (want_rest) out.push_back(o[2]);
    ctx->mark_non_differentiable(variable_list(out.begin() + 1, out.end()));
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    if (!g[0].defined()) return variable_list(11);
    const variable_list s = ctx->get_saved_variables();
    const auto [dq, dk, dv] = [&] {
      at::AutoDispatchBelowADInplaceOrView guard;
      return PRISM_OP(window_bwd).call(g[0], s[0], s[1], s[2], s[3], opt(s[7]), s[4], ctx->saved_data["window"].toInt(),
                        ctx->saved_data["sinks"].toInt(), ctx->saved_data["causal"].toBool(), opt(s[5]), opt(s[6]),
                        ctx->saved_data["sm_scale"].toDouble());
    }();
    variable_list out(11);
    out[0] = dq; out[1] = dk; out[2] = dv;
    return once(std::move(out));
  }
};
Outputs window_autograd(const Tensor& q, const Tensor& k, const Tensor& v, int64_t window, int64_t sinks, bool causal,
                        const OptT& q_lens, const OptT& kv_lens, double sm_scale, bool want_lse, bool want_rest) {
  check_no_tangents("window_fwd", q, k, v);
  if (!grads_wanted(q, k, v)) {
    at::AutoDispatchBelowADInplaceOrView guard;
    return PRISM_OP(window_fwd).call(q, k, v, window, sinks, causal, q_lens, kv_lens, sm_scale, want_lse, want_rest);
  }
  return WindowGrad::apply(q, k, v, window, sinks, causal, q_lens, kv_lens, sm_scale, want_lse, want_rest);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(prism, m) {
  m.def("rms_norm(Tensor x, Tensor? residual, Tensor? weight, float eps, int out_code, bool want_inv) "
        "-> Tensor[]");
  m.def("rms_norm_bwd(Tensor dy, Tensor? dh, Tensor h, Tensor? weight, Tensor inv, bool want_dw) -> Tensor[]");
  m.def("rotary(Tensor q, Tensor? k, Tensor freqs, Tensor positions, int[] axis_pairs, bool interleaved, "
        "float amplitude, bool inverse) -> Tensor[]");
  m.def("window_fwd(Tensor q, Tensor k, Tensor v, int window, int sinks, bool causal, Tensor? q_lens, "
        "Tensor? kv_lens, float sm_scale, bool want_lse, bool want_rest) -> Tensor[]");
  m.def("window_bwd(Tensor do, Tensor q, Tensor k, Tensor v, Tensor o, Tensor? rest, Tensor lse, int window, int sinks, bool causal, "
        "Tensor? q_lens, Tensor? kv_lens, float sm_scale) -> (Tensor, Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(prism, CUDA, m) {
  m.impl("rms_norm", &rms_norm);
  m.impl("rms_norm_bwd", &rms_norm_bwd);
  m.impl("rotary", &rotary);
  m.impl("window_fwd", &window_fwd);
  m.impl("window_bwd", &window_bwd);
}

TORCH_LIBRARY_IMPL(prism, AutogradCUDA, m) {
  m.impl("rms_norm", &rms_norm_autograd);
  m.impl("rotary", &rotary_autograd);
  m.impl("window_fwd", &window_autograd);
}
