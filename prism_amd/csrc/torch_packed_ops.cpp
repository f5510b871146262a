// PyTorch operators of packed batches and paged caches, and of the heads' norms
// before them (TORCH_LIBRARY_FRAGMENT(prism)); checks, allocation, streams and
// gradients as in torch_layer_ops.cpp.
#include "torch_layer.h"

namespace {

// ------------------------------------------------------------------ norms and positions of heads
// positions [S], [B, S], and with axes [S, A], [B, S, A], as the kernels take them
struct Places {
  int64_t strides[3];
  int32_t axis_end[4] = {};
  int axes;
  bool is64;
};
Places places_of(const char* op, const Tensor& pos, c10::IntArrayRef axis_pairs, int64_t B, int64_t S, int64_t pairs) {
  TORCH_CHECK_TYPE(pos.scalar_type() == at::kInt || pos.scalar_type() == at::kLong,
                   "prism: positions must be int32 or int64, got ", pos.scalar_type());
  const bool has_axis = !axis_pairs.empty();
  const int64_t A = has_axis ? (int64_t)axis_pairs.size() : 1, rank = pos.dim() - (has_axis ? 1 : 0);
  TORCH_CHECK_VALUE((rank == 1 || rank == 2) && pos.size(rank - 1) == S &&
                        (rank == 1 || pos.size(0) == B || pos.size(0) == 1) && (!has_axis || pos.size(-1) == A),
                    op, ": positions must be [S] or [B, S]", has_axis ? " with one entry per axis" : "", ", got ", pos.sizes());
  TORCH_CHECK_VALUE(A <= 4, op, ": at most 4 axes");
  Places p;
  p.strides[0] = rank == 2 && pos.size(0) > 1 ? pos.stride(0) : 0;
  p.strides[1] = pos.stride(rank - 1);
  p.strides[2] = has_axis ? pos.stride(-1) : 0;
  int64_t at = 0;
  for (int64_t a = 0; a < A; ++a) {
    at += has_axis ? axis_pairs[a] : pairs;
    TORCH_CHECK_VALUE(!has_axis || axis_pairs[a] >= 0, op, ": negative axis size");
    p.axis_end[a] = small(at, "pairs");
  }
  p.axes = (int)A;
  p.is64 = pos.scalar_type() == at::kLong;
  return p;
}

struct HeadCall {  // the checked arguments of both directions
  int dt, wdt;
  int64_t B, S, D, Hq, Hk;
};
HeadCall check_heads(const char* op, const Tensor& q, const OptT& k, const OptT& wq, const OptT& wk, const Tensor& freqs,
                     const Tensor& pos) {
  on_gpu(q, "q");
  same_device(q, k, "k");
  same_device(q, wq, "q_weight");
  same_device(q, wk, "k_weight");
  same_device(q, freqs, "freqs");
  same_device(q, pos, "positions");
  TORCH_CHECK_VALUE(q.dim() == 4, op, ": q must be [B, H, S, D]");
  HeadCall c;
  c.dt = type_code(q, op);
  check_dtype(k, q.scalar_type(), "k");
  check_dtype(freqs, at::kDouble, "freqs");
  TORCH_CHECK_VALUE(freqs.dim() == 1, op, ": freqs must be [pairs]");
  c.B = q.size(0); c.Hq = q.size(1); c.S = q.size(2); c.D = q.size(3);
  c.Hk = k ? k->size(1) : 0;
  if (k)
    TORCH_CHECK_VALUE(k->dim() == 4 && k->size(0) == c.B && k->size(2) == c.S && k->size(3) == c.D, op,
                      ": k must be [B, Hk, S, D] with q's B, S and D");
  TORCH_CHECK_VALUE(k || !wk, op, ": k_weight without k");
  c.wdt = wq ? type_code(*wq, "q_weight") : wk ? type_code(*wk, "k_weight") : c.dt;
  for (const OptT* w : {&wq, &wk})
    if (*w) {
      TORCH_CHECK_VALUE((*w)->dim() == 1 && (*w)->size(0) == c.D, op, ": weights must be [D]");
      TORCH_CHECK_TYPE(type_code(**w, "weight") == c.wdt, op, ": q_weight and k_weight must have one dtype");
    }
  return c;
}
void put_strides(const Tensor& t, int64_t* s) {
  for (int d = 0; d < 3; ++d) s[d] = t.stride(d);
}

// q', and k' where there is a k
Outputs qk_norm_rotary(const Tensor& q_, const OptT& k_, const OptT& wq_, const OptT& wk_, double eps, const Tensor& freqs_,
                       const Tensor& pos, c10::IntArrayRef axis_pairs, bool interleaved, double amplitude) {
  const HeadCall c = check_heads("qk_norm_rotary", q_, k_, wq_, wk_, freqs_, pos);
  const Places at = places_of("qk_norm_rotary", pos, axis_pairs, c.B, c.S, freqs_.numel());
  const c10::DeviceGuard guard(q_.device());
  const Tensor q = unit_rows(q_), freqs = freqs_.contiguous();
  const OptT k = k_ ? OptT(unit_rows(*k_)) : OptT(), wq = cont(wq_), wk = cont(wk_);
  Outputs out{like_layout(q_)};
  int64_t st[12] = {};
  put_strides(q, st);
  put_strides(out[0], st + 3);
  if (k) {
    out.push_back(like_layout(*k_));
    put_strides(*k, st + 6);
    put_strides(out[1], st + 9);
  }
  PRISM_TORCH_CALL(prism_qk_norm_rotary, q.data_ptr(), p(k), c.dt, small(c.B, "B"), c.S, small(c.Hq, "heads"),
                   small(c.Hk, "heads"), small(c.D, "D"), small(2 * freqs.numel(), "rotary dim"), st, p(wq), p(wk), c.wdt,
                   (float)eps, freqs.data_ptr<double>(), pos.data_ptr(), at.is64, at.strides, at.axes, at.axis_end,
                   interleaved, (float)amplitude, out[0].data_ptr(), k ? out[1].data_ptr() : nullptr, stream_of(q));
  return out;
}

// dq where there is a dyq, dk where there is a dyk, dwq and dwk on request
Outputs qk_norm_rotary_bwd(const OptT& dyq_, const OptT& dyk_, const Tensor& q_, const OptT& k_, const OptT& wq_,
                           const OptT& wk_, double eps, const Tensor& freqs_, const Tensor& pos,
                           c10::IntArrayRef axis_pairs, bool interleaved, double amplitude, bool want_dwq, bool want_dwk) {
  const HeadCall c = check_heads("qk_norm_rotary_bwd", q_, k_, wq_, wk_, freqs_, pos);
  const Places at = places_of("qk_norm_rotary_bwd", pos, axis_pairs, c.B, c.S, freqs_.numel());
  for (const auto& [g, x] : {std::make_pair(&dyq_, OptT(q_)), std::make_pair(&dyk_, k_)}) {
    same_device(q_, *g, "dy");
    check_dtype(*g, q_.scalar_type(), "dy");
    if (*g) TORCH_CHECK_VALUE(x && (*g)->sizes() == x->sizes(), "qk_norm_rotary_bwd: gradients must have their inputs' shape");
  }
  TORCH_CHECK_VALUE((!want_dwq || (dyq_ && wq_)) && (!want_dwk || (dyk_ && wk_)),
                    "qk_norm_rotary_bwd: a weight's gradient needs the weight and its heads' gradient");
  const c10::DeviceGuard guard(q_.device());
  const Tensor freqs = freqs_.contiguous();
  const OptT q = dyq_ ? OptT(unit_rows(q_)) : OptT(), k = dyk_ ? OptT(unit_rows(*k_)) : OptT();
  const OptT dyq = dyq_ ? OptT(unit_rows(*dyq_)) : OptT(), dyk = dyk_ ? OptT(unit_rows(*dyk_)) : OptT();
  const OptT wq = cont(wq_), wk = cont(wk_);
  Outputs out;
  Tensor dq, dk, dwq, dwk, partial;
  if (dyq) out.push_back(dq = like_layout(q_));
  if (dyk) out.push_back(dk = like_layout(*k_));
  const bool none = c.B * c.S == 0 || (dyq ? c.Hq : 0) + (dyk ? c.Hk : 0) == 0;
  auto weight_grad = [&](const OptT& w, bool heads) {  // (no rows: nothing writes it)
    out.push_back(none || !heads ? at::zeros_like(*w) : at::empty_like(*w));
    return out.back();
  };
  if (want_dwq) dwq = weight_grad(wq, c.Hq > 0);
  if (want_dwk) dwk = weight_grad(wk, c.Hk > 0);
  if (none) return out;
  int64_t st[18] = {};
  if (dyq) {
    put_strides(*dyq, st);
    put_strides(*q, st + 3);
    put_strides(dq, st + 6);
  }
  if (dyk) {
    put_strides(*dyk, st + 9);
    put_strides(*k, st + 12);
    put_strides(dk, st + 15);
  }
  if (want_dwq || want_dwk) partial = at::empty({2, PRISM_HEAD_PARTS, c.D}, opts(q_, at::kFloat));
  PRISM_TORCH_CALL(prism_qk_norm_rotary_bwd, p(dyq), p(dyk), p(q), p(k), c.dt, small(c.B, "B"), c.S,
                   dyq ? small(c.Hq, "heads") : 0, dyk ? small(c.Hk, "heads") : 0, small(c.D, "D"),
                   small(2 * freqs.numel(), "rotary dim"), st, p(wq), p(wk), c.wdt, (float)eps, freqs.data_ptr<double>(),
                   pos.data_ptr(), at.is64, at.strides, at.axes, at.axis_end, interleaved, (float)amplitude,
                   dyq ? dq.data_ptr() : nullptr, dyk ? dk.data_ptr() : nullptr,
                   partial.defined() ? partial.data_ptr<float>() : nullptr, want_dwq ? dwq.data_ptr() : nullptr,
                   want_dwk ? dwk.data_ptr() : nullptr, stream_of(q_));
  return out;
}

struct QkNormGrad : torch::autograd::Function<QkNormGrad> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const OptT& k, const OptT& wq, const OptT& wk,
                               double eps, const Tensor& freqs, const Tensor& pos, std::vector<int64_t> axis_pairs,
                               bool interleaved, double amplitude) {
    at::AutoDispatchBelowADInplaceOrView guard;
    ctx->set_materialize_grads(false);
    const variable_list o = PRISM_OP(qk_norm_rotary).call(q, k, wq, wk, eps, freqs, pos, axis_pairs, interleaved, amplitude);
    ctx->save_for_backward({q, k ? *k : Tensor(), wq ? *wq : Tensor(), wk ? *wk : Tensor(), freqs, pos});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["axis_pairs"] = axis_pairs;
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["amplitude"] = amplitude;
    ctx->saved_data["dwq"] = wants_grad(wq);
    ctx->saved_data["dwk"] = wants_grad(wk);
    return o;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    variable_list out(10);
    const Tensor dyq = g[0], dyk = g.size() > 1 ? g[1] : Tensor();
    if (!dyq.defined() && !dyk.defined()) return out;
    const variable_list s = ctx->get_saved_variables();
    const bool dwq = dyq.defined() && ctx->saved_data["dwq"].toBool(), dwk = dyk.defined() && ctx->saved_data["dwk"].toBool();
    const Outputs d = [&] {
      at::AutoDispatchBelowADInplaceOrView guard;
      return PRISM_OP(qk_norm_rotary_bwd).call(opt(dyq), opt(dyk), s[0], opt(s[1]), opt(s[2]), opt(s[3]),
                    ctx->saved_data["eps"].toDouble(), s[4], s[5], ctx->saved_data["axis_pairs"].toIntVector(),
                    ctx->saved_data["interleaved"].toBool(), ctx->saved_data["amplitude"].toDouble(), dwq, dwk);
    }();
    size_t at = 0;
    if (dyq.defined()) out[0] = d[at++];
    if (dyk.defined()) out[1] = d[at++];
    if (dwq) out[2] = d[at++];
    if (dwk) out[3] = d[at++];
    return once(std::move(out));
  }
};
Outputs qk_norm_rotary_autograd(const Tensor& q, const OptT& k, const OptT& wq, const OptT& wk, double eps,
                                const Tensor& freqs, const Tensor& pos, c10::IntArrayRef axis_pairs, bool interleaved,
                                double amplitude) {
  check_no_tangents("qk_norm_rotary", q, k, wq, wk, freqs);
  if (!grads_wanted(q, k, wq, wk)) {
    at::AutoDispatchBelowADInplaceOrView guard;
    return PRISM_OP(qk_norm_rotary).call(q, k, wq, wk, eps, freqs, pos, axis_pairs, interleaved, amplitude);
  }
  return QkNormGrad::apply(q, k, wq, wk, eps, freqs, pos, axis_pairs.vec(), interleaved, amplitude);
}

// ------------------------------------------------------------------ packed attention
// [T, H, D] as the kernels take it: adjacent channels, 16-byte aligned rows at strides of
// whole 16-byte pieces; else a contiguous copy
Tensor pack_rows(const Tensor& t) {
  bool ok = t.numel() == 0 || (t.stride(2) == 1 && (uintptr_t)t.data_ptr() % 16 == 0);
  for (int d = 0; d < 2 && ok; ++d) ok = t.size(d) <= 1 || t.stride(d) % 8 == 0;
  if (ok && t.size(0) > 1) ok = t.stride(0) < (1 << 24);
  return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}
void pack_strides(const Tensor& t, int64_t* s) {  // head, token
  s[0] = t.size(1) > 1 ? t.stride(1) : 0;
  s[1] = t.size(0) > 1 ? t.stride(0) : 0;
}
// t's layout where that is dense, has adjacent channels and rows as near as the kernels take them
Tensor pack_like(const Tensor& t) {
  Tensor o = at::empty_like(t);
  const bool ok = o.numel() == 0 || (o.stride(2) == 1 && (o.size(0) <= 1 || o.stride(0) < (1 << 24)));
  return ok ? o : at::empty(t.sizes(), t.options());
}

struct PackShape {
  int dt, B, Hq, Hk, D;
  int64_t Tq, Tk;
};
PackShape check_packed(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& cu_q, const Tensor& cu_k) {
  on_gpu(q, "q");
  same_device(q, k, "k");
  same_device(q, v, "v");
  same_device(q, cu_q, "cu_seqlens");
  same_device(q, cu_k, "cu_seqlens_k");
  TORCH_CHECK_TYPE(q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kHalf,
                   "prism: packed attention takes bfloat16 or float16, got ", q.scalar_type());
  check_dtype(k, q.scalar_type(), "k");
  check_dtype(v, q.scalar_type(), "v");
  check_dtype(cu_q, at::kInt, "cu_seqlens");
  check_dtype(cu_k, at::kInt, "cu_seqlens_k");
  TORCH_CHECK_VALUE(q.dim() == 3 && k.dim() == 3 && k.sizes() == v.sizes() && k.size(2) == q.size(2),
                    "packed attention: q must be [Tq, Hq, D], k and v [Tk, Hk, D], got ", q.sizes(), ", ", k.sizes(), ", ",
                    v.sizes());
  TORCH_CHECK_VALUE(cu_q.dim() == 1 && cu_q.size(0) >= 1 && cu_k.sizes() == cu_q.sizes(),
                    "packed attention: cu_seqlens must be [B + 1], got ", cu_q.sizes(), " and ", cu_k.sizes());
  return {q.scalar_type() == at::kBFloat16 ? PRISM_BF16 : PRISM_F16, small(cu_q.size(0) - 1, "B"), small(q.size(1), "heads"),
          small(k.size(1), "heads"), small(q.size(2), "D"), q.size(0), k.size(0)};
}

// o, lse and what o's rounding left off on request
Outputs packed_fwd(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& cu_q_, const Tensor& cu_k_,
                   bool causal, double sm_scale, bool want_lse, bool want_rest) {
  const PackShape s = check_packed(q_, k_, v_, cu_q_, cu_k_);
  const c10::DeviceGuard guard(q_.device());
  const Tensor q = pack_rows(q_), k = pack_rows(k_), v = pack_rows(v_), cu_q = cu_q_.contiguous(), cu_k = cu_k_.contiguous();
  Tensor o = pack_like(q_), lse, rest, work;
  Outputs out{o};
  if (want_lse) out.push_back(lse = at::empty({s.Hq, s.Tq}, opts(q, at::kFloat)));
  if (want_rest) out.push_back(rest = at::empty_like(o));
  int64_t st[8], ints = 0, floats = 0;
  const Tensor* all[4] = {&q, &k, &v, &o};
  for (int i = 0; i < 4; ++i) pack_strides(*all[i], st + 2 * i);
  check_rc(prism_packed_fwd_plan(s.B, s.Hq, s.Hk, s.Tq, s.Tk, s.D, &ints, &floats));
  if (ints + floats) work = at::empty({ints + floats}, opts(q, at::kFloat));  // (the list, then the parts)
  float* wp = ints + floats ? work.data_ptr<float>() : nullptr;
  PRISM_TORCH_CALL(prism_packed_fwd, q.data_ptr(), k.data_ptr(), v.data_ptr(), s.dt, s.B, s.Hq, s.Hk, s.Tq, s.Tk, s.D, st,
                   cu_q.data_ptr<int32_t>(), cu_k.data_ptr<int32_t>(), causal, (float)sm_scale, o.data_ptr(),
                   want_rest ? rest.data_ptr() : nullptr, want_lse ? lse.data_ptr<float>() : nullptr,
                   ints ? (int32_t*)wp : nullptr, floats ? wp + ints : nullptr, stream_of(q));
  return out;
}

std::tuple<Tensor, Tensor, Tensor> packed_bwd(const Tensor& do_, const Tensor& q_, const Tensor& k_, const Tensor& v_,
                                              const Tensor& o_, const Tensor& rest_, const Tensor& lse_, const Tensor& cu_q_,
                                              const Tensor& cu_k_, bool causal, double sm_scale) {
  const PackShape s = check_packed(q_, k_, v_, cu_q_, cu_k_);
  for (const auto& t : {std::make_pair(&do_, "do"), std::make_pair(&o_, "o"), std::make_pair(&rest_, "rest")}) {
    same_device(q_, *t.first, t.second);
    check_dtype(*t.first, q_.scalar_type(), t.second);
    TORCH_CHECK_VALUE(t.first->sizes() == q_.sizes(), "packed_bwd: ", t.second, " must have q's shape");
  }
  TORCH_CHECK_VALUE(rest_.strides() == o_.strides(), "packed_bwd: rest must have o's strides");
  same_device(q_, lse_, "lse");
  check_dtype(lse_, at::kFloat, "lse");
  TORCH_CHECK_VALUE(lse_.dim() == 2 && lse_.size(0) == s.Hq && lse_.size(1) == s.Tq, "packed_bwd: lse must be [Hq, Tq]");
  const c10::DeviceGuard guard(q_.device());
  const Tensor q = pack_rows(q_), k = pack_rows(k_), v = pack_rows(v_), o = pack_rows(o_), rest = pack_rows(rest_), d = pack_rows(do_);
  for (int x = 0; x < 3; ++x) TORCH_CHECK(rest.stride(x) == o.stride(x), "packed_bwd: rest must be laid out like o");
  const Tensor lse = lse_.contiguous(), cu_q = cu_q_.contiguous(), cu_k = cu_k_.contiguous();
  Tensor dq = pack_like(q_), dk = pack_like(k_), dv = pack_like(v_);
  int64_t st[16], ints = 0, floats = 0;
  const Tensor* all[8] = {&q, &k, &v, &o, &d, &dq, &dk, &dv};
  for (int i = 0; i < 8; ++i) pack_strides(*all[i], st + 2 * i);
  check_rc(prism_packed_bwd_plan(s.B, s.Hq, s.Hk, s.Tq, s.Tk, s.D, &ints, &floats));
  Tensor work = at::empty({ints + floats + 2 * s.Hq * s.Tq}, opts(q, at::kFloat));  // the lists, the parts, then rows
  float* wp = work.data_ptr<float>();
  PRISM_TORCH_CALL(prism_packed_bwd, d.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), rest.data_ptr(),
                   lse.data_ptr<float>(), s.dt, s.B, s.Hq, s.Hk, s.Tq, s.Tk, s.D, st, cu_q.data_ptr<int32_t>(),
                   cu_k.data_ptr<int32_t>(), causal, (float)sm_scale, dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                   wp + ints + floats, ints ? (int32_t*)wp : nullptr, floats ? wp + ints : nullptr, stream_of(q));
  return {dq, dk, dv};
}

struct PackedGrad : torch::autograd::Function<PackedGrad> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& cu_q,
                               const Tensor& cu_k, bool causal, double sm_scale, bool want_lse, bool want_rest) {
    at::AutoDispatchBelowADInplaceOrView guard;
    ctx->set_materialize_grads(false);
    const variable_list o = PRISM_OP(packed_fwd).call(q, k, v, cu_q, cu_k, causal, sm_scale, true, true);
    ctx->save_for_backward({q, k, v, o[0], o[2], o[1], cu_q, cu_k});
    ctx->saved_data["causal"] = causal;
    ctx->saved_data["sm_scale"] = sm_scale;
    variable_list out{o[0]};
    if (want_lse) out.push_back(o[1]);
    if (want_rest) out.push_back(o[2]);
    ctx->mark_non_differentiable(variable_list(out.begin() + 1, out.end()));
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    if (!g[0].defined()) return variable_list(9);
    const variable_list s = ctx->get_saved_variables();
    const auto [dq, dk, dv] = [&] {
      at::AutoDispatchBelowADInplaceOrView guard;
      return PRISM_OP(packed_bwd).call(g[0], s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7], ctx->saved_data["causal"].toBool(),
                        ctx->saved_data["sm_scale"].toDouble());
    }();
    variable_list out(9);
    out[0] = dq; out[1] = dk; out[2] = dv;
    return once(std::move(out));
  }
};
Outputs packed_autograd(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& cu_q, const Tensor& cu_k,
                        bool causal, double sm_scale, bool want_lse, bool want_rest) {
  check_no_tangents("packed_fwd", q, k, v);
  if (!grads_wanted(q, k, v)) {
    at::AutoDispatchBelowADInplaceOrView guard;
    return PRISM_OP(packed_fwd).call(q, k, v, cu_q, cu_k, causal, sm_scale, want_lse, want_rest);
  }
  return PackedGrad::apply(q, k, v, cu_q, cu_k, causal, sm_scale, want_lse, want_rest);
}

// ------------------------------------------------------------------ paged caches
// A cache as the kernels take it (it is written in place: nothing is copied to fit)
struct PagedCaches {
  int bits, page_size;
  int64_t pages, strides[6];
};
PagedCaches check_caches(const char* op, const Tensor& like, const Tensor& kc, const Tensor& vc, int64_t Hk, int64_t D) {
  same_device(like, kc, "k_cache");
  same_device(like, vc, "v_cache");
  const bool four = kc.scalar_type() == at::kByte;
  TORCH_CHECK_TYPE(vc.scalar_type() == kc.scalar_type() &&
                       (four || kc.scalar_type() == at::kBFloat16 || kc.scalar_type() == at::kHalf),
                   "prism: ", op, ": caches must be both bfloat16, float16 or uint8 (4 bits), got ", kc.scalar_type(), " and ",
                   vc.scalar_type());
  TORCH_CHECK_VALUE(D == 64 || D == 128, op, ": head_dim ", D, " unsupported (64, 128)");  // (a place's bytes divide below)
  PagedCaches c;
  c.bits = four ? 4 : 16;
  const int64_t place = D / 2 + D / 32;
  TORCH_CHECK_VALUE(kc.sizes() == vc.sizes() && kc.dim() == (four ? 3 : 4) && kc.size(1) == Hk &&
                        (four ? D % 32 == 0 && kc.size(2) % place == 0 : kc.size(3) == D),
                    op, ": caches must be [pages, ", Hk, ", ", four ? "page size (D / 2 + D / 32)]" : "page size, D]", ", got ",
                    kc.sizes(), " and ", vc.sizes());
  c.pages = kc.size(0);
  c.page_size = small(four ? kc.size(2) / place : kc.size(2), "page size");
  TORCH_CHECK_VALUE(kc.stride(-1) == 1 && vc.stride(-1) == 1, op, ": a cache's channels must be adjacent");
  int x = 0;
  for (const Tensor* t : {&kc, &vc}) {
    c.strides[x++] = t->size(0) > 1 ? t->stride(0) : 0;
    c.strides[x++] = t->size(1) > 1 ? t->stride(1) : 0;
    c.strides[x++] = four ? 0 : t->stride(2);
  }
  return c;
}
void check_table(const char* op, const Tensor& like, const Tensor& table, const OptT& lens) {
  same_device(like, table, "page_table");
  same_device(like, lens, "kv_lens");
  check_dtype(table, at::kInt, "page_table");
  check_dtype(lens, at::kInt, "kv_lens");
  TORCH_CHECK_VALUE(table.dim() == 2 && table.size(1) >= 1, op, ": page_table must be [B, pages of a sequence], got ", table.sizes());
  if (lens) TORCH_CHECK_VALUE(lens->dim() == 1 && lens->size(0) == table.size(0), op, ": kv_lens must be [B]");
}
Tensor unit_table(const Tensor& t) { return t.size(1) == 1 || t.stride(1) == 1 ? t : t.contiguous(); }

void paged_append(const Tensor& k_, const Tensor& v_, const Tensor& kc, const Tensor& vc, const Tensor& table_,
                  const Tensor& lens_, const OptT& cu_, const OptT& freqs_, const OptT& pos, c10::IntArrayRef axis_pairs,
                  bool interleaved, double amplitude) {
  on_gpu(k_, "k");
  same_device(k_, v_, "v");
  check_table("append_paged", k_, table_, lens_);
  same_device(k_, cu_, "cu_seqlens");
  same_device(k_, freqs_, "freqs");
  same_device(k_, pos, "positions");
  TORCH_CHECK_TYPE(k_.scalar_type() == at::kBFloat16 || k_.scalar_type() == at::kHalf,
                   "prism: append_paged takes bfloat16 or float16, got ", k_.scalar_type());
  check_dtype(v_, k_.scalar_type(), "v");
  check_dtype(cu_, at::kInt, "cu_seqlens");
  check_dtype(freqs_, at::kDouble, "freqs");
  TORCH_CHECK_VALUE(k_.dim() == 3 && k_.sizes() == v_.sizes(), "append_paged: k and v must be [T, Hk, D], got ", k_.sizes(), " and ",
                    v_.sizes());
  const int64_t T = k_.size(0), Hk = k_.size(1), D = k_.size(2), B = table_.size(0);
  const PagedCaches c = check_caches("append_paged", k_, kc, vc, Hk, D);
  if (c.bits == 16) check_dtype(kc, k_.scalar_type(), "k_cache");
  TORCH_CHECK_VALUE(!cu_ || (cu_->dim() == 1 && cu_->size(0) == B + 1), "append_paged: cu_seqlens must be [B + 1]");
  TORCH_CHECK_VALUE(cu_ || (B == 0 ? T == 0 : T % B == 0), "append_paged: ", T, " tokens do not share out over ", B, " sequences");
  TORCH_CHECK_VALUE(!freqs_ || freqs_->dim() == 1, "append_paged: freqs must be [pairs]");
  TORCH_CHECK_VALUE(freqs_ || !pos, "append_paged: positions without freqs");
  for (const Tensor* t : {&kc, &vc})
    TORCH_CHECK_VALUE(at::has_internal_overlap(*t) != at::MemOverlap::Yes,
                      "append_paged: a cache whose places share memory (expand) cannot be written");
  TORCH_CHECK_VALUE(kc.numel() == 0 || kc.data_ptr() != vc.data_ptr(),
                    "append_paged: k_cache and v_cache share memory: each place would hold the key, the value or pieces of both");
  const c10::DeviceGuard guard(k_.device());
  const Tensor k = pack_rows(k_), v = pack_rows(v_), table = unit_table(table_), lens = lens_.contiguous();
  const OptT cu = cont(cu_), freqs = cont(freqs_);
  int64_t st[4] = {k.stride(0), k.size(1) > 1 ? k.stride(1) : 0, v.stride(0), v.size(1) > 1 ? v.stride(1) : 0};
  if (T == 1) st[0] = st[2] = 0;
  Places at{};
  if (pos) at = places_of("append_paged", *pos, axis_pairs, 1, T, freqs->numel());
  PRISM_TORCH_CALL(prism_paged_append_f64, k.data_ptr(), v.data_ptr(), k.scalar_type() == at::kBFloat16 ? PRISM_BF16 : PRISM_F16, T,
                   small(Hk, "heads"), small(D, "D"), st, kc.data_ptr(), vc.data_ptr(), c.bits, c.pages, c.page_size, c.strides,
                   table.data_ptr<int32_t>(), table.size(0) > 1 ? table.stride(0) : 0, table.size(1), lens.data_ptr<int32_t>(),
                   small(B, "B"), (const int32_t*)p(cu), (const double*)p(freqs), freqs ? small(2 * freqs->numel(), "rotary dim") : 0,
                   interleaved, p(pos), pos ? at.is64 : false, at.strides + 1, at.axes, at.axis_end, amplitude, stream_of(k));
  // (torch's own record that the caches changed)
  for (const Tensor* t : {&kc, &vc})
    if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}

std::tuple<Tensor, Tensor> paged_gather(const Tensor& kc, const Tensor& vc, const Tensor& table_, const Tensor& cu_,
                                        int64_t total, int64_t heads, int64_t D, bool half) {
  on_gpu(kc, "k_cache");
  const PagedCaches c = check_caches("gather_paged", kc, kc, vc, heads, D);
  check_table("gather_paged", kc, table_, OptT());
  same_device(kc, cu_, "cu_seqlens");
  check_dtype(cu_, at::kInt, "cu_seqlens");
  TORCH_CHECK_VALUE(cu_.dim() == 1 && cu_.size(0) == table_.size(0) + 1, "gather_paged: cu_seqlens must be [B + 1]");
  TORCH_CHECK_VALUE(total >= 0, "gather_paged: total must not be negative");
  const c10::DeviceGuard guard(kc.device());
  const Tensor table = unit_table(table_), cu = cu_.contiguous();
  const at::ScalarType t = c.bits == 16 ? kc.scalar_type() : half ? at::kHalf : at::kBFloat16;
  Tensor k = at::empty({total, heads, D}, opts(kc, t)), v = at::empty({total, heads, D}, opts(kc, t));
  PRISM_TORCH_CALL(prism_paged_gather, kc.data_ptr(), vc.data_ptr(), t == at::kHalf ? PRISM_F16 : PRISM_BF16, c.bits, c.pages,
                   c.page_size, c.strides, table.data_ptr<int32_t>(), table.size(0) > 1 ? table.stride(0) : 0, table.size(1),
                   small(table.size(0), "B"), cu.data_ptr<int32_t>(), total, small(heads, "heads"), small(D, "D"), k.data_ptr(),
                   v.data_ptr(), stream_of(kc));
  return {k, v};
}

// o, and lse on request
Outputs paged_fwd(const Tensor& q_, const Tensor& kc, const Tensor& vc, const Tensor& table_, const Tensor& lens_, int64_t heads,
                  double sm_scale, bool want_lse) {
  on_gpu(q_, "q");
  TORCH_CHECK_TYPE(q_.scalar_type() == at::kBFloat16 || q_.scalar_type() == at::kHalf,
                   "prism: paged attention takes bfloat16 or float16, got ", q_.scalar_type());
  TORCH_CHECK_VALUE(q_.dim() == 3, "paged attention: q must be [T, Hq, D], got ", q_.sizes());
  const int64_t T = q_.size(0), Hq = q_.size(1), D = q_.size(2);
  const PagedCaches c = check_caches("flash_attn_paged", q_, kc, vc, heads, D);
  if (c.bits == 16) check_dtype(kc, q_.scalar_type(), "k_cache");
  check_table("flash_attn_paged", q_, table_, lens_);
  const int64_t B = table_.size(0);
  TORCH_CHECK_VALUE(B == 0 ? T == 0 : T % B == 0, "flash_attn_paged: ", T, " queries do not share out over ", B, " sequences");
  const int64_t n = B ? T / B : 0;
  const c10::DeviceGuard guard(q_.device());
  const Tensor q = pack_rows(q_), table = unit_table(table_), lens = lens_.contiguous();
  Tensor o = pack_like(q_), lse, part;
  Outputs out{o};
  if (want_lse) out.push_back(lse = at::empty({Hq, T}, opts(q, at::kFloat)));
  int64_t st[4], floats = 0;
  st[0] = T > 1 ? q.stride(0) : 0; st[1] = Hq > 1 ? q.stride(1) : 0;
  st[2] = T > 1 ? o.stride(0) : 0; st[3] = Hq > 1 ? o.stride(1) : 0;
  check_rc(prism_paged_plan(small(B, "B"), n, small(Hq, "heads"), small(heads, "heads"), small(D, "D"), c.bits,
                            table.size(1) * c.page_size, &floats));
  if (floats) part = at::empty({floats}, opts(q, at::kFloat));
  PRISM_TORCH_CALL(prism_paged_fwd, q.data_ptr(), q.scalar_type() == at::kBFloat16 ? PRISM_BF16 : PRISM_F16, (int)B, n, (int)Hq,
                   (int)heads, (int)D, st, kc.data_ptr(), vc.data_ptr(), c.bits, c.pages, c.page_size, c.strides,
                   table.data_ptr<int32_t>(), table.size(0) > 1 ? table.stride(0) : 0, table.size(1), lens.data_ptr<int32_t>(),
                   (float)sm_scale, o.data_ptr(), want_lse ? lse.data_ptr<float>() : nullptr,
                   floats ? part.data_ptr<float>() : nullptr, stream_of(q));
  return out;
}

// (no gradients and no tangents: refused here, where they would be lost without a word)
template <class... T>
void check_no_grads(const char* op, const T&... t) {
  check_no_tangents(op, t...);
  TORCH_CHECK_VALUE(!at::GradMode::is_enabled() || !(wants_grad(t) || ...), "prism: ", op,
                    " has no gradient: call it under torch.no_grad() or on detached tensors");
}
void paged_append_autograd(const Tensor& k, const Tensor& v, const Tensor& kc, const Tensor& vc, const Tensor& table,
                           const Tensor& lens, const OptT& cu, const OptT& freqs, const OptT& pos,
                           c10::IntArrayRef axis_pairs, bool interleaved, double amplitude) {
  check_no_grads("paged_append", k, v, kc, vc, freqs);
  at::AutoDispatchBelowADInplaceOrView guard;
  PRISM_OP(paged_append).call(k, v, kc, vc, table, lens, cu, freqs, pos, axis_pairs, interleaved, amplitude);
}
std::tuple<Tensor, Tensor> paged_gather_autograd(const Tensor& kc, const Tensor& vc, const Tensor& table, const Tensor& cu,
                                                 int64_t total, int64_t heads, int64_t D, bool half) {
  check_no_grads("paged_gather", kc, vc);
  at::AutoDispatchBelowADInplaceOrView guard;
  return PRISM_OP(paged_gather).call(kc, vc, table, cu, total, heads, D, half);
}
Outputs paged_fwd_autograd(const Tensor& q, const Tensor& kc, const Tensor& vc, const Tensor& table, const Tensor& lens,
                           int64_t heads, double sm_scale, bool want_lse) {
  check_no_grads("paged_fwd", q, kc, vc);
  at::AutoDispatchBelowADInplaceOrView guard;
  return PRISM_OP(paged_fwd).call(q, kc, vc, table, lens, heads, sm_scale, want_lse);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(prism, m) {
  m.def("paged_append(Tensor k, Tensor v, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor page_table, Tensor kv_lens, "
        "Tensor? cu_seqlens, Tensor? freqs, Tensor? positions, int[] axis_pairs, bool interleaved, float amplitude) -> ()");
  m.def("paged_gather(Tensor k_cache, Tensor v_cache, Tensor page_table, Tensor cu_seqlens, int total, int heads, "
        "int head_dim, bool half) -> (Tensor, Tensor)");
  m.def("paged_fwd(Tensor q, Tensor k_cache, Tensor v_cache, Tensor page_table, Tensor kv_lens, int heads, float sm_scale, "
        "bool want_lse) -> Tensor[]");
  m.def("packed_fwd(Tensor q, Tensor k, Tensor v, Tensor cu_q, Tensor cu_k, bool causal, float sm_scale, bool want_lse, "
        "bool want_rest) -> Tensor[]");
  m.def("packed_bwd(Tensor do, Tensor q, Tensor k, Tensor v, Tensor o, Tensor rest, Tensor lse, Tensor cu_q, Tensor cu_k, "
        "bool causal, float sm_scale) -> (Tensor, Tensor, Tensor)");
  m.def("qk_norm_rotary(Tensor q, Tensor? k, Tensor? q_weight, Tensor? k_weight, float eps, Tensor freqs, "
        "Tensor positions, int[] axis_pairs, bool interleaved, float amplitude) -> Tensor[]");
  m.def("qk_norm_rotary_bwd(Tensor? dyq, Tensor? dyk, Tensor q, Tensor? k, Tensor? q_weight, Tensor? k_weight, float eps, "
        "Tensor freqs, Tensor positions, int[] axis_pairs, bool interleaved, float amplitude, bool want_dwq, "
        "bool want_dwk) -> Tensor[]");
}

TORCH_LIBRARY_IMPL(prism, CUDA, m) {
  m.impl("qk_norm_rotary", &qk_norm_rotary);
  m.impl("qk_norm_rotary_bwd", &qk_norm_rotary_bwd);
  m.impl("packed_fwd", &packed_fwd);
  m.impl("packed_bwd", &packed_bwd);
  m.impl("paged_append", &paged_append);
  m.impl("paged_gather", &paged_gather);
  m.impl("paged_fwd", &paged_fwd);
}

TORCH_LIBRARY_IMPL(prism, AutogradCUDA, m) {
  m.impl("qk_norm_rotary", &qk_norm_rotary_autograd);
  m.impl("packed_fwd", &packed_autograd);
  m.impl("paged_append", &paged_append_autograd);
  m.impl("paged_gather", &paged_gather_autograd);
  m.impl("paged_fwd", &paged_fwd_autograd);
}
