// Native host path of the cache operators: outputs and workspaces from torch's allocator,
// parameter blocks, launches on torch's current stream.  The Python wrappers (cache.py) have
// checked shapes and types; their custom ops run the same functions.
#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/record_function.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>

#include <cmath>
#include <initializer_list>
#include <optional>
#include <tuple>
#include <vector>

#include "fa_host.h"

namespace fa_host {
namespace {

// Entry points of libfa2_4d_mask.so as the Python loader resolved them.
struct CacheApi {
  int (*prefix_plan)(const FaPrefixParams*, FaPrefixPlan*);
  int (*prefix_fwd)(const FaPrefixParams*);
  int (*mask_plan)(const FaMaskParams*, int64_t*);
  int (*mask_prepare)(const FaMaskParams*);
  int (*key_weights_plan)(const FaKeyWeightsParams*, int64_t*);
  int (*key_weights)(const FaKeyWeightsParams*);
  int (*evict)(const FaEvictParams*);
  int (*rotary)(const FaRotaryParams*);
  const char* (*last_error)();
};
CacheApi g_api{};
PyObject* g_general_backward = nullptr;   // cache.py's prefix backward, held for good

void check(int status, const char* what) {
  TORCH_CHECK(status == FA_OK, what, " failed with status ", status, ": ", g_api.last_error());
}

using MaybeTensor = std::optional<Tensor>;
Tensor get(const MaybeTensor& x) { return x.value_or(Tensor()); }
MaybeTensor get_opt(const Tensor& x) { return x.defined() ? MaybeTensor(x) : std::nullopt; }

// Columns the kernels are given of operands of D: D itself where they take it in place
// (multiples of 16), else padded with zeros to their own head dim.
int64_t columns(int64_t D) { return D % 16 == 0 ? D : kernel_head_dim(D); }

// What memory holds is x (not a view that stands for its negative).
Tensor as_held(const Tensor& x) { return x.is_neg() ? x.resolve_neg() : x; }

// x as the kernels can address it; copies only where that does not hold.
Tensor addressable(const Tensor& x, bool bhsd, int64_t W) {
  Tensor y = x.size(3) == W ? as_held(x) : at::constant_pad_nd(x, {0, W - x.size(3)});
  return in_place(y, operand(y, bhsd)) ? y : y.clone(at::MemoryFormat::Contiguous);
}

// [B, T, H, D] memory, viewed in the caller's layout.
Tensor token_major(int64_t B, int64_t T, int64_t H, int64_t D, const at::TensorOptions& o, bool bhsd) {
  const Tensor x = at::empty({B, T, H, D}, o);
  return bhsd ? x.transpose(1, 2) : x;
}
// The first D columns of such a tensor, in memory of their own.
Tensor first_columns(const Tensor& x, int64_t D, bool bhsd) {
  if (x.size(3) == D) return x;
  return bhsd ? x.narrow(3, 0, D).transpose(1, 2).contiguous().transpose(1, 2) : x.narrow(3, 0, D).contiguous();
}

// What the Python wrappers check, with their texts: nullptr, or why the operands do not fit.  The
// custom ops can be called without the wrappers, and plain calls come here first (the wrappers' own
// checks, 4 us a call, then only word the refusal).
using Why = const char*;
bool alike(const Tensor& x, const Tensor& first) {
  return x.dim() == 4 && x.device() == first.device() && x.scalar_type() == first.scalar_type();
}
Why operands_misfit(const Tensor& q, const Tensor& k, const Tensor& v) {
  if (!q.is_cuda() || (q.scalar_type() != at::kBFloat16 && q.scalar_type() != at::kHalf)) return "fp16 or bf16 GPU tensors expected";
  if (!alike(q, q) || !alike(k, q) || !alike(v, q)) return "rank-4 tensors of one type on one device expected";
  if (!v.sizes().equals(k.sizes()) || k.size(0) != q.size(0) || k.size(3) != q.size(3) || q.size(3) > 256)
    return "q, k and v do not fit together, or the head dimension exceeds 256";
  return nullptr;
}
Why lengths_misfit(const Tensor& n, const Tensor& first) {
  if (n.defined() && (n.scalar_type() != at::kInt || n.dim() != 1 || n.size(0) != first.size(0) || !n.is_contiguous() ||
                      n.device() != first.device()))
    return "lengths must be a contiguous int32 tensor of the batch size on the operands' device";
  return nullptr;
}
Why sums_misfit(const Tensor& w, const Tensor& k, bool bhsd) {
  if (w.defined() && (w.scalar_type() != at::kFloat || !w.sizes().equals({k.size(0), k.size(bhsd ? 1 : 2), k.size(bhsd ? 2 : 1)}) ||
                      w.device() != k.device()))
    return "key weights must be a float32 tensor [batch, key heads, keys] on the operands' device";
  return nullptr;
}
Why side_misfit(const Tensor& x, at::ScalarType t, const Tensor& q, const Tensor& k, bool bhsd) {
  if (x.defined() && (x.scalar_type() != t || x.dim() != 4 || (x.size(0) != 1 && x.size(0) != q.size(0)) ||
                      (x.size(1) != 1 && x.size(1) != q.size(bhsd ? 1 : 2)) || x.size(2) != q.size(bhsd ? 2 : 1) ||
                      x.size(3) != k.size(bhsd ? 2 : 1) || x.device() != q.device()))
    return "a bool mask or float32 score must be [batch or 1, heads or 1, rows, keys] on the operands' device";
  return nullptr;
}
Why attend_misfit(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& pk, const Tensor& pv, const Tensor& lengths,
                  const Tensor& mask, const Tensor& score, const Tensor& kw, bool bhsd) {
  const int t = bhsd ? 2 : 1, h = bhsd ? 1 : 2;
  if (const Why w = operands_misfit(q, k, v)) return w;
  if (k.size(h) == 0 || q.size(h) % k.size(h) != 0) return "the query heads must be a multiple of the key heads";
  if (pk.defined() != pv.defined()) return "pk and pv must be given together";
  if (pk.defined() && (!alike(pk, q) || !alike(pv, q) || !pv.sizes().equals(pk.sizes()) || pk.size(0) != 1 ||
                       pk.size(h) != k.size(h) || pk.size(3) != q.size(3)))
    return "pk and pv do not fit k";
  if (q.numel() == 0 || k.size(t) + (pk.defined() ? pk.size(t) : 0) == 0) return "no rows, or no keys at all";
  if (const Why w = lengths_misfit(lengths, q)) return w;
  if (const Why w = side_misfit(mask, at::kBool, q, k, bhsd)) return w;
  if (const Why w = side_misfit(score, at::kFloat, q, k, bhsd)) return w;
  return sums_misfit(kw, k, bhsd);
}
Why evict_misfit(const Tensor& k, const Tensor& v, const Tensor& kw, const Tensor& lengths, int64_t keep, int64_t recent, bool bhsd) {
  if (const Why w = operands_misfit(k, k, v)) return w;
  if (k.numel() == 0) return "no keys";
  if (const Why w = lengths_misfit(lengths, k)) return w;
  if (!kw.defined()) return "no key weights";
  if (const Why w = sums_misfit(kw, k, bhsd)) return w;
  if (keep < 1 || keep > k.size(bhsd ? 2 : 1)) return "keep must lie in [1, keys]";
  return recent < 0 || recent > keep ? "recent must lie in [0, keep]" : nullptr;
}
Why rotary_misfit(const Tensor& q, const Tensor& k, const Tensor& pos, const Tensor& freq, const std::vector<int64_t>& sections, bool bhsd) {
  const int t = bhsd ? 2 : 1, h = bhsd ? 1 : 2;
  if (const Why w = operands_misfit(q, k, k)) return w;
  if (k.size(t) != q.size(t) || q.size(h) == 0 || k.size(h) == 0 || q.size(3) < 2) return "q and k do not fit together";
  const int64_t axes = (int64_t)sections.size();
  if (pos.dim() != 3 || (pos.scalar_type() != at::kLong && pos.scalar_type() != at::kInt) || pos.device() != q.device() ||
      pos.size(0) != axes || (pos.size(1) != 1 && pos.size(1) != q.size(0)) || pos.size(2) != q.size(t))
    return "positions must be an int32 or int64 tensor [axes, batch or 1, tokens] on the operands' device";
  if (freq.dim() != 1 || freq.scalar_type() != at::kFloat || !freq.is_contiguous() || freq.device() != q.device() ||
      freq.size(0) < 1 || 2 * freq.size(0) > q.size(3))
    return "inv_freq must be a contiguous float32 vector on the operands' device";
  int64_t sum = 0;
  for (const int64_t x : sections) {
    if (x < 0 || x > freq.size(0)) return "a section is negative or too large";
    sum += x;
  }
  return axes < 1 || axes > FA_ROTARY_AXES || sum != freq.size(0) ? "the sections must add up to the pairs of inv_freq, on at most 8 axes" : nullptr;
}
bool wants_grad(std::initializer_list<Tensor> xs) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor& x : xs)
    if (x.defined() && x.requires_grad()) return true;
  return false;
}

// A mask or score [B|1, Hq|1, Tq, Tk] with a contiguous key axis.
Tensor side(const Tensor& x) {
  if (!x.defined()) return x;
  const Tensor y = as_held(x);
  return y.size(3) == 1 || y.stride(3) == 1 ? y : y.contiguous();
}

Tensor key_axis_contiguous(const Tensor& x_) {
  const Tensor x = as_held(x_);
  return x.size(2) == 1 || x.stride(2) == 1 ? x : x.contiguous();
}
Tensor columns_contiguous(const Tensor& x_) {
  const Tensor x = as_held(x_);
  return x.size(3) == 1 || x.stride(3) == 1 ? x : x.contiguous();
}
int64_t axis_stride(const Tensor& x, int i) { return x.size(i) == 1 ? 0 : x.stride(i); }

template <typename P> void set_sides(P& p, const Tensor& mask, const Tensor& score, const Tensor& lengths) {
  if (mask.defined()) {
    p.mask = (const uint8_t*)mask.const_data_ptr();
    p.mask_stride_b = side_stride(mask, 0); p.mask_stride_h = side_stride(mask, 1); p.mask_stride_q = side_stride(mask, 2);
  }
  if (score.defined()) {
    p.score = (const float*)score.const_data_ptr();
    p.score_stride_b = side_stride(score, 0); p.score_stride_h = side_stride(score, 1); p.score_stride_q = side_stride(score, 2);
  }
  if (lengths.defined()) p.lengths = (const int32_t*)lengths.const_data_ptr();
}

// kw [B, Hk, Tk] plus the sums of many rows' probabilities, from their LSE [B, Hq, Tq].
Tensor key_weights(const Tensor& q_, const Tensor& k_, const Tensor& lse_, const MaybeTensor& lengths_, const MaybeTensor& mask_,
                   const MaybeTensor& score_, const MaybeTensor& kw_, double scale, bool causal, bool bhsd) {
  at::AutoDispatchBelowADInplaceOrView below;
  const c10::DeviceGuard on_device(q_.device());
  const int64_t D = q_.size(3), W = columns(D);
  const Tensor q = addressable(q_, bhsd, W), k = addressable(k_, bhsd, W), lse = lse_.contiguous();
  const Operand oq = operand(q, bhsd), ok = operand(k, bhsd);
  const Tensor mask = get(mask_), score = get(score_), lengths = get(lengths_);
  FaKeyWeightsParams p{};
  set_sides(p, mask, score, lengths);
  p.q = oq.p; p.k = ok.p; p.lse = lse.const_data_ptr<float>();
  p.q_stride_b = oq.sb; p.q_stride_t = oq.st; p.q_stride_h = oq.sh;
  p.k_stride_b = ok.sb; p.k_stride_t = ok.st; p.k_stride_h = ok.sh;
  p.batch = (int32_t)oq.B; p.seqlen_q = (int32_t)oq.T; p.seqlen_k = (int32_t)ok.T;
  p.heads_q = (int32_t)oq.H; p.heads_k = (int32_t)ok.H;
  p.head_dim = kernel_head_dim(D);
  p.head_dim_in = (int32_t)W;
  p.scale = (float)scale;
  p.is_causal = causal;
  p.dtype = dtype_code(q);
  p.stream = stream_of(q);
  Tensor kw = get(kw_);
  if (kw.defined()) {
    kw = key_axis_contiguous(kw);
    p.kw_in = kw.const_data_ptr<float>();
    p.kw_stride_b = axis_stride(kw, 0); p.kw_stride_h = axis_stride(kw, 1);
  }
  const Tensor out = at::empty({ok.B, ok.H, ok.T}, q.options().dtype(at::kFloat));
  p.kw_out = out.data_ptr<float>();
  int64_t bytes = 0;
  check(g_api.key_weights_plan(&p, &bytes), "fa_key_weights_plan");
  Tensor ws;
  if (bytes) {
    ws = at::empty({bytes}, q.options().dtype(at::kByte));
    p.workspace = ws.data_ptr();
    p.workspace_bytes = bytes;
  }
  check(g_api.key_weights(&p), "fa_key_weights");
  return out;
}

// For kernels that take no lengths (a mask's or score's, the backward's) and read whole tiles: the own keys' mask with `lengths` as
// part of it (rows broadcast), and K or V with zeros past them (0 times what stands there
// would be NaN if that is no number).
Tensor existing_keys(const Tensor& lengths, int64_t B, int64_t Tk) { return at::arange(Tk, lengths.options()).lt(lengths.view({B, 1})); }
Tensor with_lengths(const Tensor& mask, const Tensor& there, int64_t B, int64_t Tq, int64_t Tk) {
  const Tensor keep = there.view({B, 1, 1, Tk}).expand({B, 1, Tq, Tk});
  return mask.defined() ? mask.logical_and(keep) : keep;
}
Tensor zeros_past(const Tensor& x, const Tensor& there, bool bhsd) {
  return at::where(bhsd ? there.view({there.size(0), 1, -1, 1}) : there.view({there.size(0), -1, 1, 1}), x, at::zeros({}, x.options()));
}

// A mask prepared for the kernels that take it so; empty dims are the caller's to exclude.
Tensor prepared_mask(FaMaskParams m, const at::TensorOptions& bytes) {
  int64_t n = 0;
  check(g_api.mask_plan(&m, &n), "fa_mask_plan");
  const Tensor ws = at::empty({n}, bytes);
  m.workspace = ws.data_ptr();
  check(g_api.mask_prepare(&m), "fa_mask_prepare");
  return ws;
}

// O (in the caller's layout), LSE [B, Hq, Tq], O's rounding residual and key weights [B, Hk, Tk]
// (none unless asked for).
std::tuple<Tensor, Tensor, MaybeTensor, MaybeTensor> attend(const Tensor& q_, const Tensor& k_, const Tensor& v_, const MaybeTensor& pk_,
                                                  const MaybeTensor& pv_, const MaybeTensor& lengths_, const MaybeTensor& mask_,
                                                  const MaybeTensor& score_, const MaybeTensor& kw_, double scale, bool causal,
                                                  bool weights, bool residual, bool bhsd) {
  at::AutoDispatchBelowADInplaceOrView below;
  const Why why = attend_misfit(q_, k_, v_, get(pk_), get(pv_), get(lengths_), get(mask_), get(score_), get(kw_), bhsd);
  TORCH_CHECK(!why, why);
  const c10::DeviceGuard on_device(q_.device());
  RECORD_FUNCTION("tilelang_fa2_4d_mask::prefix_fwd", c10::ArrayRef<const c10::IValue>());
  const int t = bhsd ? 2 : 1, h = bhsd ? 1 : 2;
  const int64_t B = q_.size(0), Tq = q_.size(t), Hq = q_.size(h), D = q_.size(3), Tk = k_.size(t), Hk = k_.size(h);
  const int64_t Tp = pk_ ? pk_->size(t) : 0, W = columns(D);
  FaPrefixParams p{};
  p.batch = (int32_t)B; p.seqlen_q = (int32_t)Tq; p.seqlen_p = (int32_t)Tp; p.seqlen_k = (int32_t)Tk;
  p.heads_q = (int32_t)Hq; p.heads_k = (int32_t)Hk;
  p.head_dim = kernel_head_dim(D);
  p.head_dim_in = (int32_t)W;
  p.scale = (float)scale;
  p.is_causal = causal;
  p.dtype = dtype_code(q_);
  p.stream = stream_of(q_);
  const Tensor own_mask = Tk ? side(get(mask_)) : Tensor();
  Tensor mask = own_mask, lengths = Tk ? get(lengths_) : Tensor();
  const Tensor score = Tk ? side(get(score_)) : Tensor();
  set_sides(p, mask, score, lengths);
  const bool kw_too = weights && Tk > 0;
  Tensor kw = get(kw_), kw_out;
  if (weights) kw_out = at::empty({B, Hk, Tk}, q_.options().dtype(at::kFloat));
  if (kw_too) p.kw_out = kw_out.data_ptr<float>();
  FaPrefixPlan plan{};
  check(g_api.prefix_plan(&p, &plan), "fa_prefix_plan");
  if (p.kw_out && !plan.few_rows) {   // the weights in a pass of their own, behind
    p.kw_out = nullptr;
    check(g_api.prefix_plan(&p, &plan), "fa_prefix_plan");
  }
  Tensor k_clean = k_, v_clean = v_;
  if (!plan.few_rows && lengths.defined() && (mask.defined() || score.defined())) {
    const Tensor there = existing_keys(lengths, B, Tk);
    mask = with_lengths(mask, there, B, Tq, Tk);
    k_clean = zeros_past(k_, there, bhsd);
    v_clean = zeros_past(v_, there, bhsd);
    p.lengths = nullptr;
    set_sides(p, mask, score, Tensor());
    check(g_api.prefix_plan(&p, &plan), "fa_prefix_plan");
  }

  const Tensor q = addressable(q_, bhsd, W), k = addressable(k_clean, bhsd, W), v = addressable(v_clean, bhsd, W);
  const Operand oq = operand(q, bhsd), ok = operand(k, bhsd), ov = operand(v, bhsd);
  p.q = oq.p; p.k = ok.p; p.v = ov.p;
  p.q_stride_b = oq.sb; p.q_stride_t = oq.st; p.q_stride_h = oq.sh;
  p.k_stride_b = ok.sb; p.k_stride_t = ok.st; p.k_stride_h = ok.sh;
  p.v_stride_b = ov.sb; p.v_stride_t = ov.st; p.v_stride_h = ov.sh;
  Tensor pk, pv;
  if (Tp > 0) {
    pk = addressable(*pk_, bhsd, W);
    pv = addressable(*pv_, bhsd, W);
    const Operand opk = operand(pk, bhsd), opv = operand(pv, bhsd);
    p.pk = opk.p; p.pv = opv.p;
    p.pk_stride_t = opk.st; p.pk_stride_h = opk.sh;
    p.pv_stride_t = opv.st; p.pv_stride_h = opv.sh;
  }
  const Tensor out = token_major(B, Tq, Hq, W, q.options(), bhsd), lse = at::empty({B, Hq, Tq}, q.options().dtype(at::kFloat));
  const Operand oo = operand(out, bhsd);
  p.o = const_cast<void*>(oo.p);
  p.o_stride_b = oo.sb; p.o_stride_t = oo.st; p.o_stride_h = oo.sh;
  p.lse = lse.data_ptr<float>();
  Tensor lo;
  if (residual) {
    lo = token_major(B, Tq, Hq, W, q.options(), bhsd);
    const Operand ol = operand(lo, bhsd);
    p.o_lo = const_cast<void*>(ol.p);
    p.o_lo_stride_b = ol.sb; p.o_lo_stride_t = ol.st; p.o_lo_stride_h = ol.sh;
  }
  if (p.kw_out && kw.defined()) {
    kw = key_axis_contiguous(kw);
    p.kw_in = kw.const_data_ptr<float>();
    p.kw_stride_b = axis_stride(kw, 0); p.kw_stride_h = axis_stride(kw, 1);
  }
  const auto bytes = q.options().dtype(at::kByte);
  Tensor mask_ws;
  if (plan.needs_mask_ws && mask.defined()) {
    FaMaskParams m{};
    m.mask = p.mask;
    m.mask_stride_b = p.mask_stride_b; m.mask_stride_h = p.mask_stride_h; m.mask_stride_q = p.mask_stride_q;
    m.batch = p.batch; m.seqlen_q = p.seqlen_q; m.seqlen_k = p.seqlen_k; m.heads_q = p.heads_q;
    m.is_causal = p.is_causal;
    m.stream = p.stream;
    mask_ws = prepared_mask(m, bytes);
    p.mask_ws = mask_ws.const_data_ptr();
  }
  const Tensor ws = at::empty({plan.workspace_bytes}, bytes);
  p.workspace = ws.data_ptr();
  p.workspace_bytes = plan.workspace_bytes;
  check(g_api.prefix_fwd(&p), "fa_prefix_fwd");
  if (kw_too && !p.kw_out) kw_out = key_weights(q, k, lse, get_opt(lengths), get_opt(own_mask), get_opt(score), kw_, scale, causal, bhsd);
  return {first_columns(out, D, bhsd), lse, residual ? MaybeTensor(first_columns(lo, D, bhsd)) : std::nullopt, get_opt(kw_out)};
}

// dQ, dK, dV, dKp, dVp of a shared prefix as cache.py's prefix_bwd makes them, for operands the
// kernels take as they lie in memory; false: not for this path.
bool prefix_backward(const Tensor& dout, const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& pk_, const Tensor& pv_,
                     const Tensor& lengths, const Tensor& mask_, const Tensor& score_, const Tensor& o_, const Tensor& lse,
                     const Tensor& lo_, double scale, bool causal, bool atomic, bool bhsd, Tensor* out) {
  for (const Tensor* x : {&q_, &k_, &v_, &pk_, &pv_, &o_, &lse, &lo_})   // (saved tensors come back through hooks)
    if (!plain(*x) || x->device() != q_.device()) return false;
  for (const Tensor* x : {&lengths, &mask_, &score_})
    if (x->defined() && (!plain(*x) || x->device() != q_.device())) return false;
  if (attend_misfit(q_, k_, v_, pk_, pv_, lengths, mask_, score_, Tensor(), bhsd) || q_.size(3) % 16 != 0 ||
      !dout.sizes().equals(q_.sizes()))
    return false;
  const c10::DeviceGuard on_device(q_.device());
  auto bthd = [&](const Tensor& x) { return bhsd ? x.transpose(1, 2) : x; };
  const Tensor d = bthd(dout), q = bthd(q_), k = bthd(k_), v = bthd(v_), pk = bthd(pk_), pv = bthd(pv_), o = bthd(o_), lo = bthd(lo_);
  const int64_t B = q.size(0), Tq = q.size(1), Hq = q.size(2), D = q.size(3), Tk = k.size(1), Tp = pk.size(1);
  const int64_t W = kernel_head_dim(D);
  const bool both = Tp > 0 && Tk > 0;
  // the sums laid out [Hq, B Tq, W], which is [B, Hq, Tq, W] by strides for the own keys
  const auto f32 = q.options().dtype(at::kFloat);
  const Tensor sums = both ? at::empty({Hq, B * Tq, W}, f32) : at::zeros({Hq, B * Tq, W}, f32);
  Gradients g;
  if (Tk > 0) {
    Tensor own_k = k, own_v = v, mask = mask_, mask_ws;
    if (lengths.defined()) {
      const Tensor there = existing_keys(lengths, B, Tk);
      mask = with_lengths(mask, there, B, Tq, Tk);
      own_k = zeros_past(k, there, false);
      own_v = zeros_past(v, there, false);
    }
    mask = side(mask);
    const Tensor score = side(score_);
    if (mask.defined()) {
      FaMaskParams m{};
      m.mask = (const uint8_t*)mask.const_data_ptr();
      m.mask_stride_b = side_stride(mask, 0); m.mask_stride_h = side_stride(mask, 1); m.mask_stride_q = side_stride(mask, 2);
      m.batch = (int32_t)B; m.seqlen_q = (int32_t)Tq; m.seqlen_k = (int32_t)Tk; m.heads_q = (int32_t)Hq;
      m.is_causal = causal;
      m.stream = stream_of(q);
      mask_ws = prepared_mask(m, q.options().dtype(at::kByte));
    }
    const DqSums to{sums, both ? FA_DQ_KEEP : FA_DQ_ADD, Tq * W, B * Tq * W};
    if (!backward(d, q, own_k, own_v, o, lse, mask, score, mask_ws, lo, scale, causal, atomic, false, &to, &g)) return false;
    out[0] = bthd(g.dq);
    out[1] = bthd(g.dk);
    out[2] = bthd(g.dv);
  } else {
    out[1] = at::zeros_like(k_);
    out[2] = at::zeros_like(v_);
  }
  if (Tp > 0) {   // the rows of the batch as one sequence
    auto one = [&](const Tensor& x) { return x.reshape({1, B * Tq, Hq, D}); };
    const Tensor lse1 = lse.transpose(0, 1).reshape({1, Hq, B * Tq}).contiguous();
    const DqSums to{sums, FA_DQ_ADD, 0, B * Tq * W};
    if (!backward(one(d), one(q), pk, pv, one(o), lse1, Tensor(), Tensor(), Tensor(), one(lo), scale, false, atomic, false, &to, &g))
      return false;
    out[0] = bthd(g.dq.view({B, Tq, Hq, D}));
    out[3] = bthd(g.dk);
    out[4] = bthd(g.dv);
  } else {
    out[3] = at::zeros_like(pk_);
    out[4] = at::zeros_like(pv_);
  }
  return true;
}

struct Attended {
  Tensor o, lse, lo, lengths, mask, score;   // the last three as given, undefined where not
};

struct Prefix : torch::autograd::Function<Prefix> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& pk,
                        const Tensor& pv, const Attended& done, double scale, bool causal, bool atomic, bool bhsd) {
    ctx->save_for_backward({q, k, v, pk, pv, done.lengths, done.mask, done.score, done.o, done.lse, done.lo});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["flags"] = (int64_t)(causal | atomic << 1 | bhsd << 2);
    ctx->set_materialize_grads(false);
    return done.o;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    torch::autograd::variable_list r(10);
    if (!grads[0].defined()) return r;   // the output does not reach the loss
    const auto s = ctx->get_saved_variables();
    const double scale = ctx->saved_data["scale"].toDouble();
    const int64_t flags = ctx->saved_data["flags"].toInt();
    const bool causal = flags & 1, atomic = flags >> 1 & 1, bhsd = flags >> 2 & 1;
    if (plain_backward(grads[0])) {
      at::AutoDispatchBelowADInplaceOrView below;
      if (prefix_backward(grads[0], s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7], s[8], s[9], s[10], scale, causal, atomic,
                          bhsd, r.data()))
        return r;
    }
    pybind11::gil_scoped_acquire gil;
    const auto g = pybind11::handle(g_general_backward)(grads[0], s[0], s[1], s[2], s[3], s[4], get_opt(s[5]), get_opt(s[6]),
                                                        get_opt(s[7]), s[8], s[9], s[10], scale, causal, atomic, bhsd)
                       .cast<std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor>>();
    std::tie(r[0], r[1], r[2], r[3], r[4]) = g;
    return r;
  }
};

// O of a shared prefix with its gradients to come.
Tensor attend_train(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& pk, const Tensor& pv, const MaybeTensor& lengths,
                    const MaybeTensor& mask, const MaybeTensor& score, double scale, bool causal, bool atomic, bool bhsd) {
  const bool some = pk.size(bhsd ? 2 : 1) > 0;
  const auto r = attend(q, k, v, some ? MaybeTensor(pk) : std::nullopt, some ? MaybeTensor(pv) : std::nullopt, lengths, mask, score,
                        std::nullopt, scale, causal, false, true, bhsd);
  return Prefix::apply(q, k, v, pk, pv, Attended{std::get<0>(r), std::get<1>(r), get(std::get<2>(r)), get(lengths), get(mask), get(score)},
                       scale, causal, atomic, bhsd);
}

// K, V and weights of the kept keys, and their indices.
std::tuple<Tensor, Tensor, Tensor, Tensor> evict(const Tensor& k_, const Tensor& v_, const Tensor& kw_, const MaybeTensor& lengths_,
                                                 int64_t keep, int64_t recent, bool bhsd) {
  at::AutoDispatchBelowADInplaceOrView below;
  const Why why = evict_misfit(k_, v_, kw_, get(lengths_), keep, recent, bhsd);
  TORCH_CHECK(!why, why);
  const c10::DeviceGuard on_device(k_.device());
  RECORD_FUNCTION("tilelang_fa2_4d_mask::evict", c10::ArrayRef<const c10::IValue>());
  const Tensor k = columns_contiguous(k_), v = columns_contiguous(v_), kw = key_axis_contiguous(kw_), lengths = get(lengths_);
  const Operand ok = operand(k, bhsd), ov = operand(v, bhsd);
  std::vector<int64_t> shape = k.sizes().vec();
  shape[bhsd ? 2 : 1] = keep;
  const Tensor ko = at::empty(shape, k.options()), vo = at::empty(shape, k.options());
  const Tensor kwo = at::empty({ok.B, ok.H, keep}, kw.options()), idx = at::empty({ok.B, ok.H, keep}, kw.options().dtype(at::kLong));
  const Operand oo = operand(ko, bhsd);
  FaEvictParams p{};
  p.k = ok.p; p.v = ov.p; p.kw = kw.const_data_ptr<float>();
  if (lengths.defined()) p.lengths = (const int32_t*)lengths.const_data_ptr();
  p.k_out = ko.data_ptr(); p.v_out = vo.data_ptr(); p.kw_out = kwo.data_ptr<float>(); p.index_out = idx.data_ptr<int64_t>();
  p.k_stride_b = ok.sb; p.k_stride_t = ok.st; p.k_stride_h = ok.sh;
  p.v_stride_b = ov.sb; p.v_stride_t = ov.st; p.v_stride_h = ov.sh;
  p.kw_stride_b = axis_stride(kw, 0); p.kw_stride_h = axis_stride(kw, 1);
  p.out_stride_b = oo.sb; p.out_stride_t = oo.st; p.out_stride_h = oo.sh;
  p.batch = (int32_t)ok.B; p.seqlen_k = (int32_t)ok.T; p.heads_k = (int32_t)ok.H; p.head_dim = (int32_t)ok.D;
  p.keep = (int32_t)keep; p.recent = (int32_t)recent;
  p.stream = stream_of(k);
  check(g_api.evict(&p), "fa_evict");
  return {ko, vo, kwo, idx};
}

using Pair = std::tuple<Tensor, Tensor>;

Pair rotary_run(const Tensor& q_, const Tensor& k_, const Tensor& pos, const Tensor& freq_, const std::vector<int64_t>& sections,
                bool adjacent, bool inverse, bool bhsd) {
  const Why why = rotary_misfit(q_, k_, pos, freq_, sections, bhsd);
  TORCH_CHECK(!why, why);
  const c10::DeviceGuard on_device(q_.device());
  RECORD_FUNCTION("tilelang_fa2_4d_mask::rotary", c10::ArrayRef<const c10::IValue>());
  const Tensor q = columns_contiguous(q_), k = columns_contiguous(k_), freq = as_held(freq_);
  const Operand oq = operand(q, bhsd), ok = operand(k, bhsd);
  const Tensor qo = token_major(oq.B, oq.T, oq.H, oq.D, q.options(), bhsd), ko = token_major(ok.B, ok.T, ok.H, ok.D, k.options(), bhsd);
  if (q.numel() == 0) return {qo, ko};
  const Operand wq = operand(qo, bhsd), wk = operand(ko, bhsd);
  FaRotaryParams p{};
  p.q = oq.p; p.k = ok.p; p.q_out = const_cast<void*>(wq.p); p.k_out = const_cast<void*>(wk.p);
  p.positions = pos.const_data_ptr();
  p.inv_freq = freq.const_data_ptr<float>();
  p.q_stride_b = oq.sb; p.q_stride_t = oq.st; p.q_stride_h = oq.sh;
  p.k_stride_b = ok.sb; p.k_stride_t = ok.st; p.k_stride_h = ok.sh;
  p.qo_stride_b = wq.sb; p.qo_stride_t = wq.st; p.qo_stride_h = wq.sh;
  p.ko_stride_b = wk.sb; p.ko_stride_t = wk.st; p.ko_stride_h = wk.sh;
  p.pos_stride_a = axis_stride(pos, 0); p.pos_stride_b = axis_stride(pos, 1); p.pos_stride_t = axis_stride(pos, 2);
  p.batch = (int32_t)oq.B; p.seqlen = (int32_t)oq.T; p.heads_q = (int32_t)oq.H; p.heads_k = (int32_t)ok.H;
  p.head_dim = (int32_t)oq.D;
  p.rotary = (int32_t)(2 * freq.numel());
  p.axes = (int32_t)sections.size();
  for (size_t i = 0; i < sections.size(); ++i) p.sections[i] = (int32_t)sections[i];
  p.positions_64 = pos.scalar_type() == at::kLong;
  p.adjacent = adjacent;
  p.sign = inverse ? -1 : 1;
  p.dtype = dtype_code(q);
  p.stream = stream_of(q);
  check(g_api.rotary(&p), "fa_rotary");
  return {qo, ko};
}

struct Rotary : torch::autograd::Function<Rotary> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& q, const Tensor& k,
                                                const Tensor& pos, const Tensor& freq, std::vector<int64_t> sections,
                                                bool adjacent, bool inverse, bool bhsd) {
    ctx->save_for_backward({pos, freq});
    ctx->saved_data["sections"] = sections;
    ctx->saved_data["flags"] = (int64_t)(adjacent | inverse << 1 | bhsd << 2);
    at::AutoDispatchBelowADInplaceOrView below;
    const Pair r = rotary_run(q, k, pos, freq, sections, adjacent, inverse, bhsd);
    return {std::get<0>(r), std::get<1>(r)};
  }
  // The rotation back of both gradients (one that does not reach the loss: zeros), itself
  // differentiable.
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list g) {
    const auto s = ctx->get_saved_variables();
    const int64_t flags = ctx->saved_data["flags"].toInt();
    const std::vector<int64_t> sections = ctx->saved_data["sections"].toIntVector();
    const bool adjacent = flags & 1, inverse = !(flags >> 1 & 1), bhsd = flags >> 2 & 1;
    torch::autograd::variable_list out(8);
    if (at::GradMode::is_enabled()) {
      auto r = Rotary::apply(g[0], g[1], s[0], s[1], sections, adjacent, inverse, bhsd);
      out[0] = r[0];
      out[1] = r[1];
    } else {
      at::AutoDispatchBelowADInplaceOrView below;
      std::tie(out[0], out[1]) = rotary_run(g[0], g[1], s[0], s[1], sections, adjacent, inverse, bhsd);
    }
    return out;
  }
};

Pair rotary(const Tensor& q, const Tensor& k, const Tensor& pos, const Tensor& freq, const std::vector<int64_t>& sections,
            bool adjacent, bool inverse, bool bhsd) {
  if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad())) {
    const auto r = Rotary::apply(q, k, pos, freq, sections, adjacent, inverse, bhsd);
    return {r[0], r[1]};
  }
  at::AutoDispatchBelowADInplaceOrView below;
  return rotary_run(q, k, pos, freq, sections, adjacent, inverse, bhsd);
}

// The wrappers' first try: plain calls whose operands fit and need no copies of lengths or score.
// None: for the wrappers' checks, and the custom ops.
using MaybeOutputs = std::optional<std::tuple<Tensor, MaybeTensor>>;
MaybeOutputs attend_plain(const MaybeTensor& q, const MaybeTensor& k, const MaybeTensor& v, const MaybeTensor& pk, const MaybeTensor& pv,
                          const MaybeTensor& lengths, const MaybeTensor& mask, const MaybeTensor& score, const MaybeTensor& kw,
                          std::optional<double> scale, bool causal, bool weights, bool bhsd) {
  if (!q || !k || !v || attend_misfit(*q, *k, *v, get(pk), get(pv), get(lengths), get(mask), get(score), get(kw), bhsd) ||
      wants_grad({*q, *k, *v, get(pk), get(pv), get(score), get(kw)}))
    return std::nullopt;
  const bool some = pk && pk->size(bhsd ? 2 : 1) > 0;
  const double by = scale ? *scale : std::pow((double)q->size(3), -0.5);
  auto r = attend(*q, *k, *v, some ? pk : std::nullopt, some ? pv : std::nullopt, lengths, mask, score, kw, by, causal, weights, false, bhsd);
  return std::make_tuple(std::get<0>(r), std::get<3>(r));
}
std::optional<std::tuple<Tensor, Tensor, Tensor, Tensor>> evict_plain(const MaybeTensor& k, const MaybeTensor& v, const MaybeTensor& kw,
                                                                      const MaybeTensor& lengths, int64_t keep, int64_t recent, bool bhsd) {
  if (!k || !v || evict_misfit(*k, *v, get(kw), get(lengths), keep, recent, bhsd) || wants_grad({*k, *v, get(kw)})) return std::nullopt;
  return evict(*k, *v, *kw, lengths, keep, recent, bhsd);
}
std::optional<Pair> rotary_plain(const MaybeTensor& q, const MaybeTensor& k, const MaybeTensor& pos, const MaybeTensor& freq,
                                 std::vector<int64_t> sections, bool adjacent, bool bhsd) {
  if (!q || !k || !pos || !freq) return std::nullopt;
  if (sections.empty()) sections = {freq->numel()};
  if (rotary_misfit(*q, *k, *pos, *freq, sections, bhsd) || wants_grad({*freq})) return std::nullopt;
  return rotary(*q, *k, *pos, *freq, sections, adjacent, false, bhsd);
}

void init_cache(const std::vector<uintptr_t>& fn, pybind11::object general) {
  TORCH_CHECK(fn.size() == 9, "nine entry points expected");
  g_api = CacheApi{(decltype(CacheApi::prefix_plan))fn[0],      (decltype(CacheApi::prefix_fwd))fn[1],
                   (decltype(CacheApi::mask_plan))fn[2],        (decltype(CacheApi::mask_prepare))fn[3],
                   (decltype(CacheApi::key_weights_plan))fn[4], (decltype(CacheApi::key_weights))fn[5],
                   (decltype(CacheApi::evict))fn[6],            (decltype(CacheApi::rotary))fn[7],
                   (decltype(CacheApi::last_error))fn[8]};
  g_general_backward = general.release().ptr();
}

}  // namespace

void bind_cache(pybind11::module_& m) {
  using release = pybind11::call_guard<pybind11::gil_scoped_release>;
  m.def("init_cache", &init_cache);
  m.def("attend", &attend, release());
  m.def("attend_train", &attend_train, release());
  m.def("attend_plain", &attend_plain, release());
  m.def("evict", &evict, release());
  m.def("evict_plain", &evict_plain, release());
  m.def("rotary", &rotary, release());
  m.def("rotary_plain", &rotary_plain, release());
}

}  // namespace fa_host
