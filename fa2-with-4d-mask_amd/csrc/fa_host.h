// Operands of the native host path (fa_host.cpp, fa_cache_host.cpp).
#pragma once

#include <torch/extension.h>

#include <c10/hip/HIPStream.h>

#include <cstdint>

#include "fa2_4d_mask.h"

namespace fa_host {

using at::Tensor;

// A dense device tensor that is its own memory: no batched, wrapped, negated,
// all-zero or subclass tensor (batched gradients reach a backward as such), whose
// data pointer is missing or means something else.
inline bool plain(const Tensor& x) {
  using K = c10::DispatchKey;
  constexpr c10::DispatchKeySet wrapped({K::Python, K::Negative, K::Conjugate, K::ZeroTensor, K::Batched, K::FuncTorchBatched,
                                         K::FuncTorchGradWrapper, K::Functionalize});
  const c10::DispatchKeySet keys = x.key_set();
  return keys.has(K::CUDA) && !keys.has_any(wrapped);
}

// The logical [B, T, H, D] view of a tensor given as [B, H, T, D] (bhsd) or
// [B, T, H, D]: sizes, and strides with those of size-1 axes 0.
struct Operand {
  int64_t B, T, H, D, sb, st, sh;
  const void* p;
};
inline Operand operand(const Tensor& x, bool bhsd) {
  const int t = bhsd ? 2 : 1, h = bhsd ? 1 : 2;
  auto st = [&](int i) { return x.size(i) == 1 ? (int64_t)0 : x.stride(i); };
  return {x.size(0), x.size(t), x.size(h), x.size(3), st(0), st(t), st(h), x.const_data_ptr()};
}
// Columns contiguous, rows 16-byte aligned (fa2.py _kernel_operand).
inline bool in_place(const Tensor& x, const Operand& o) {
  return (x.size(3) == 1 || x.stride(3) == 1) && o.sb % 8 == 0 && o.st % 8 == 0 && o.sh % 8 == 0 && (uintptr_t)o.p % 16 == 0;
}
inline int kernel_head_dim(int64_t D) { return D <= 64 ? 64 : (D <= 128 ? 128 : 256); }

// A mask / score the kernels read as it is (fa2.py _kernel_side).
inline bool side_ok(const Tensor& x, at::ScalarType dtype, const Tensor& q, int64_t B, int64_t Hq, int64_t Tq, int64_t Tk) {
  return x.dim() == 4 && x.scalar_type() == dtype && x.device() == q.device() && x.size(2) == Tq && x.size(3) == Tk &&
         (x.size(0) == 1 || x.size(0) == B) && (x.size(1) == 1 || x.size(1) == Hq) && (Tk == 1 || x.stride(3) == 1);
}
inline int64_t side_stride(const Tensor& x, int i) { return x.size(i) == 1 ? 0 : x.stride(i); }

inline int dtype_code(const Tensor& q) { return q.scalar_type() == at::kBFloat16 ? FA_DTYPE_BF16 : FA_DTYPE_FP16; }

inline void* stream_of(const Tensor& q) { return (void*)c10::hip::getCurrentHIPStream(q.device().index()).stream(); }

// ---- the attention's backward (fa_host.cpp) ----

struct Gradients {
  Tensor dq, dk, dv;   // in the caller's layout
};
// Where dQ is summed in fp32 over several key sets: the sums, FaDqMode, batch and head strides.
struct DqSums {
  Tensor sums;
  int mode;
  int64_t sb, sh;
};
// False: not for the native path.  With `sums` and FA_DQ_KEEP the dQ of `g` is not written.
bool backward(const Tensor& dout, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& out, const Tensor& lse,
              const Tensor& mask, const Tensor& score, const Tensor& mask_ws, const Tensor& o_lo, double scale, bool causal,
              bool atomic, bool bhsd, const DqSums* sums, Gradients* g);
// A backward that nothing traces, transforms or intercepts, and no setting that only the Python
// host path honours.
bool plain_backward(const Tensor& dout);

void bind_cache(pybind11::module_& m);   // fa_cache_host.cpp

}  // namespace fa_host
