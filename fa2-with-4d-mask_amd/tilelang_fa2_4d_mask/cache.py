"""Operators of a K/V cache beside the attention: prompts shared by a batch, the
weight every cached key receives, eviction by that weight, rotary positions.

* :func:`tilelang_rotary_embedding`: positions of one or several axes on queries
  and keys, before the keys go into a cache (differentiable);
* :func:`tilelang_shared_prefix_attention`: attention of a batch whose sequences
  share a prefix, computed once for all of them (differentiable);
* :func:`tilelang_attention_with_key_weights`: attention that adds up the
  probability each key received;
* :func:`tilelang_evict_keys`: the cache cut down to the keys with the largest
  such sums and the most recent ones.

The reference package has none of these.  They follow its wrappers' manner
(modeling_attention.py): rank-4 fp16 / bf16 tensors in ``layout="bhsd"`` (default)
or ``"bshd"``, ``ValueError`` for arguments that do not fit, launches on torch's
current stream, no state kept between calls (so they can be captured into a HIP
graph).  Plain eager calls go straight to the native host path
(csrc/fa_cache_host.cpp); traced and transformed ones through the custom ops
``tilelang_fa2_4d_mask::prefix_fwd`` / ``prefix_bwd`` / ``key_weights`` / ``evict`` /
``rotary``, which run the same functions.
"""

from __future__ import annotations

from typing import Optional, Sequence

import torch

from . import _ext
from . import fa2 as _fa2
from . import ops as _ops  # noqa: F401  (registers fwd / bwd)
from .modeling_attention import Layout, _broadcast_4d, _dims

_NS = "tilelang_fa2_4d_mask"


# ---- checks ------------------------------------------------------------------------


def _sizes_of(query, key, value, layout: str):
    """(batch, heads_q, heads_k, seqlen_q, seqlen_k, head_dim), checked."""
    if key.dim() == 4 and 0 in (key.shape[1 if layout == "bhsd" else 2], key.shape[3]):
        raise ValueError("key and value must have at least one head and one column")
    B, Hq, Tq, Tk, D = _dims(query, key, value, layout)
    if D > 256:
        raise ValueError(f"head dimension {D} is not supported (up to 256)")
    return B, Hq, key.shape[1 if layout == "bhsd" else 2], Tq, Tk, D


def _check_types(first: str, x: torch.Tensor, **others) -> None:
    if x.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"TileLang attention expects fp16 or bf16 inputs, got {x.dtype}")
    for name, y in others.items():
        if y is None:
            continue
        if y.dtype != x.dtype:
            raise ValueError(f"{first} and {name} must have the same dtype")
        if y.device != x.device:
            raise ValueError(f"{first} and {name} must be on the same device")


def _check_gpu(x: torch.Tensor) -> None:
    if not x.is_cuda:
        raise ValueError("inputs must be HIP/CUDA tensors: the operators run on the GPU")


def _check_lengths(lengths: Optional[torch.Tensor], B: int, device: torch.device) -> Optional[torch.Tensor]:
    if lengths is None:
        return None
    if lengths.dtype not in (torch.int32, torch.int64) or tuple(lengths.shape) != (B,):
        raise ValueError(f"lengths must be an int32 or int64 tensor of shape [{B}]")
    if lengths.device != device:
        raise ValueError(f"lengths must be on {device}, got {lengths.device}")
    # (clamped first: an int64 far out of range must not wrap into it)
    if lengths.dtype == torch.int64:
        lengths = lengths.clamp(0, 2 ** 31 - 1).to(torch.int32)
    return lengths.contiguous()


def _check_sides(mask, score, shape: dict, device: torch.device):
    if mask is not None:
        if mask.dtype != torch.bool:
            raise ValueError("mask must be a bool tensor with True for valid entries")
        if mask.device != device:
            raise ValueError(f"mask must be on {device}, got {mask.device}")
        _broadcast_4d(mask, name="mask", **shape)
    if score is not None:
        if not torch.is_floating_point(score):
            raise ValueError("score must be a floating-point tensor")
        score = score.to(device=device, dtype=torch.float32)
        _broadcast_4d(score, name="score", **shape)
    return mask, score


def _check_prefix(prefix_key, prefix_value, layout: str, Hk: int, D: int) -> None:
    for name, x in (("prefix_key", prefix_key), ("prefix_value", prefix_value)):
        if x.dim() != 4 or x.shape[0] != 1:
            raise ValueError(f"{name} must be a rank-4 tensor of batch size 1")
        if x.shape[1 if layout == "bhsd" else 2] != Hk:
            raise ValueError(f"{name} must have the {Hk} heads of key")
        if x.shape[3] != D:
            raise ValueError(f"{name} must have the head dimension {D}")
    if prefix_key.shape != prefix_value.shape:
        raise ValueError("prefix_key and prefix_value must have the same sequence length")


def _check_key_weights(kw, B: int, Hk: int, Tk: int, device: torch.device, name: str = "key_weights") -> None:
    if kw.dtype != torch.float32 or tuple(kw.shape) != (B, Hk, Tk):
        raise ValueError(f"{name} must be a float32 tensor of shape [{B}, {Hk}, {Tk}]")
    if kw.device != device:
        raise ValueError(f"{name} must be on {device}, got {kw.device}")


def _wants_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(x is not None and x.requires_grad for x in tensors)


def _host():
    return _ext.load_host()


def _plain(layout: str, first, *others) -> bool:
    """A plain eager call on GPU tensors: the native path tries it before any check here (it
    returns None unless the operands fit, as the checks here would have it)."""
    return getattr(first, "is_cuda", False) and layout in ("bhsd", "bshd") and _fa2._plain_eager(first, *others)


def _timed(entry: str, fn, *args):
    """fn(*args), recorded under the library entry's name where an event log is open
    (fa2.py record_kernel_events)."""
    log = _fa2._event_log
    if log is None:
        return fn(*args)
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    out = fn(*args)
    end.record()
    log.records.append((entry, start, end))
    return out


# ---- attention over a shared prefix and own keys --------------------------------------


def _sizes(q, k, pk, bhsd: bool):
    t, h = (2, 1) if bhsd else (1, 2)
    return q.shape[0], q.shape[t], 0 if pk is None else pk.shape[t], k.shape[t], q.shape[h], k.shape[h], q.shape[3]


def _bthd(x: torch.Tensor, bhsd: bool) -> torch.Tensor:
    return x.transpose(1, 2) if bhsd else x


def _own_mask(mask, lengths, B: int, Tq: int, Tk: int):
    """The bool mask of the attention kernels that take no lengths: rows broadcast."""
    if lengths is None:
        return mask
    keep = (torch.arange(Tk, device=lengths.device) < lengths.view(B, 1, 1, 1)).expand(B, 1, Tq, Tk)
    return keep if mask is None else mask & keep


def _existing(x: torch.Tensor, lengths) -> torch.Tensor:
    """A logical [B, T, H, D] cache with zeros past the lengths, for kernels that read whole
    tiles: 0 times what stands there would be NaN if that is no number."""
    if lengths is None:
        return x
    there = torch.arange(x.shape[1], device=x.device) < lengths.view(-1, 1)
    return torch.where(there[:, :, None, None], x, x.new_zeros(()))


def _one_sequence(x: torch.Tensor) -> torch.Tensor:
    """[B, T, H, D] -> [1, B T, H, D]: the rows of a batch against one key set."""
    return x.reshape(1, x.shape[0] * x.shape[1], x.shape[2], x.shape[3])


def _empty_attention(q, bhsd: bool):
    """No rows, or no key at all: as the attention answers an empty key set."""
    B, Tq, _, _, Hq, _, D = _sizes(q, q, None, bhsd)
    o = q.new_zeros((B, Tq, Hq, D))
    return (o.transpose(1, 2) if bhsd else o), q.new_full((B, Hq, Tq), float("-inf"), dtype=torch.float32)


def _attend(q, k, v, pk, pv, lengths, mask, score, kw, scale, causal, weights, residual, bhsd):
    """O, LSE, O's rounding residual (or None), key weights (or None)."""
    B, Tq, Tp, Tk, Hq, Hk, D = _sizes(q, k, pk, bhsd)
    if Tp == 0:
        pk = pv = None
    if B * Tq * Hq * D == 0 or Tp + Tk == 0:
        o, lse = _empty_attention(q, bhsd)
        if weights:
            return o, lse, None, q.new_zeros((B, Hk, Tk), dtype=torch.float32) if kw is None else kw.clone()
        return o, lse, None, None
    return _timed("fa_prefix_fwd", _host().attend, q, k, v, pk, pv, lengths, mask, score, kw, scale, causal, weights,
                  residual, bhsd)


@torch.library.custom_op(f"{_NS}::prefix_fwd", mutates_args=(), device_types="cuda")
def prefix_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, pk: Optional[torch.Tensor], pv: Optional[torch.Tensor],
               lengths: Optional[torch.Tensor], mask: Optional[torch.Tensor], score: Optional[torch.Tensor],
               scale: float, causal: bool, atomic: bool, residual: bool,
               bhsd: bool) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """O (layout of q), LSE [B, Hq, Tq] fp32, O's rounding residual (with ``residual``, else empty)."""
    o, lse, lo, _ = _attend(q, k, v, pk, pv, lengths, mask, score, None, scale, causal, False, residual, bhsd)
    return o, lse, q.new_empty((0,)) if lo is None else lo


def _like_output(q, bhsd: bool):
    B, Tq, _, _, Hq, _, D = _sizes(q, q, None, bhsd)
    o = q.new_empty((B, Tq, Hq, D))
    return o.transpose(1, 2) if bhsd else o


@prefix_fwd.register_fake
def _prefix_fwd_fake(q, k, v, pk, pv, lengths, mask, score, scale, causal, atomic, residual, bhsd):
    B, Tq, Tp, Tk, Hq, _, D = _sizes(q, k, pk, bhsd)
    some = residual and B * Tq * Hq * D > 0 and Tp + Tk > 0
    return (_like_output(q, bhsd), q.new_empty((B, Hq, Tq), dtype=torch.float32),
            _like_output(q, bhsd) if some else q.new_empty((0,)))


@torch.library.custom_op(f"{_NS}::prefix_bwd", mutates_args=(), device_types="cuda")
def prefix_bwd(do: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, pk: Optional[torch.Tensor],
               pv: Optional[torch.Tensor], lengths: Optional[torch.Tensor], mask: Optional[torch.Tensor],
               score: Optional[torch.Tensor], o: torch.Tensor, lse: torch.Tensor, o_lo: torch.Tensor, scale: float,
               causal: bool, atomic: bool,
               bhsd: bool) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """dQ, dK, dV, dKp, dVp of ``prefix_fwd`` (layout of q; empty where there is no prefix).

    With the LSE and Delta of the whole softmax, prefix and own keys are two independent
    backward passes.  Their dQ are summed in fp32 (they cancel where a row's weight lies on
    keys of both sets that point the same way); the prefix's pass takes the rows of the
    batch as one sequence, so that its dK and dV are summed over the batch in the kernel."""
    B, Tq, Tp, Tk, Hq, Hk, D = _sizes(q, k, pk, bhsd)

    def zeros(x):
        return _bthd(torch.zeros(_bthd(x, bhsd).shape, dtype=x.dtype, device=x.device), bhsd)

    none = [q.new_empty((0,)), q.new_empty((0,))]
    if B * Tq * Hq * D == 0 or Tp + Tk == 0:
        return zeros(q), zeros(k), zeros(v), *((zeros(pk), zeros(pv)) if Tp else none)
    do, q, k, v, o = (_bthd(x, bhsd) for x in (do, q, k, v, o))
    lo = _bthd(o_lo, bhsd) if o_lo.numel() else None
    _fa2._check_qkv(q, k, v)
    if any(x is not None and x.device != q.device for x in (o, lse, lo)) or o.dtype != q.dtype or lse.dtype != torch.float32:
        raise ValueError("o, lse and o_lo must be on the device of q, o and lse as prefix_fwd returned them")
    op = _fa2._kernel_operand
    W = _fa2.kernel_head_dim(D)
    # the sums laid out [Hq, B Tq, W], which is [B, Hq, Tq, W] by strides for the own keys
    both = Tp > 0 and Tk > 0
    sums = (torch.empty if both else torch.zeros)((Hq, B * Tq, W), dtype=torch.float32, device=q.device)
    dk = dv = None
    dpk, dpv = none
    if Tk > 0:
        m, mst = _fa2._kernel_side(_own_mask(mask, lengths, B, Tq, Tk), torch.bool, B, Hq, Tq, Tk, "mask", q.device)
        s, sst = _fa2._kernel_side(score, torch.float32, B, Hq, Tq, Tk, "score", q.device)
        dq, dk, dv = _fa2._backward_impl(
            do, op(q), op(_existing(k, lengths)), op(_existing(v, lengths)), op(o), lse.contiguous(), m, s, None, mst, sst, scale,
            causal, atomic, None if lo is None else op(lo), (sums, _ext.FA_DQ_KEEP if both else _ext.FA_DQ_ADD, Tq * W, B * Tq * W))
    if Tp > 0:
        pk, pv = _bthd(pk, bhsd), _bthd(pv, bhsd)
        _fa2._check_qkv(q, pk, pv)
        lse1 = lse.transpose(0, 1).reshape(1, Hq, B * Tq).contiguous()
        dq, dpk, dpv = _fa2._backward_impl(
            _one_sequence(do), op(_one_sequence(q)), op(pk), op(pv), op(_one_sequence(o)), lse1, None, None, None, (0, 0, 0),
            (0, 0, 0), scale, False, atomic, None if lo is None else op(_one_sequence(lo)),
            (sums, _ext.FA_DQ_ADD, 0, B * Tq * W))
        dq = dq.view(B, Tq, Hq, D)
        dpk, dpv = _bthd(dpk, bhsd), _bthd(dpv, bhsd)
    if dk is None:
        dk, dv = (torch.zeros(x.shape, dtype=x.dtype, device=x.device) for x in (k, v))
    return _bthd(dq, bhsd), _bthd(dk, bhsd), _bthd(dv, bhsd), dpk, dpv


@prefix_bwd.register_fake
def _prefix_bwd_fake(do, q, k, v, pk, pv, lengths, mask, score, o, lse, o_lo, scale, causal, atomic, bhsd):
    def like(x):
        return q.new_empty((0,)) if x is None or x.numel() == 0 else _bthd(_bthd(x, bhsd).new_empty(_bthd(x, bhsd).shape), bhsd)

    def own(x):
        return _bthd(x.new_empty(_bthd(x, bhsd).shape), bhsd)

    return own(q), own(k), own(v), like(pk), like(pv)


def _prefix_setup(ctx, inputs, output):
    q, k, v, pk, pv, lengths, mask, score, scale, causal, atomic, residual, bhsd = inputs
    O, LSE, lo = output
    ctx.save_for_backward(q, k, v, pk, pv, lengths, mask, score, O, LSE, lo)
    ctx.how = scale, causal, atomic, bhsd
    ctx.set_materialize_grads(False)


def _general_prefix_backward(dO, q, k, v, pk, pv, *rest):
    """The gradients through the custom op; the native node hands a backward back here that it does
    not take (a dS limit, the event log, gradients of gradients, operands to copy)."""
    g = torch.ops.tilelang_fa2_4d_mask.prefix_bwd(dO, q, k, v, pk, pv, *rest)
    dpk, dpv = (None if x is None else (y if x.numel() else torch.zeros_like(x)) for x, y in ((pk, g[3]), (pv, g[4])))
    return *g[:3], dpk, dpv


def _prefix_backward(ctx, dO, dLSE, dlo):
    if dO is None:
        return (None,) * 13
    return _general_prefix_backward(dO, *ctx.saved_tensors, *ctx.how) + (None,) * 8


prefix_fwd.register_autograd(_prefix_backward, setup_context=_prefix_setup)


@torch.library.custom_op(f"{_NS}::key_weights", mutates_args=(), device_types="cuda")
def key_weights(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, pk: Optional[torch.Tensor], pv: Optional[torch.Tensor],
                lengths: Optional[torch.Tensor], mask: Optional[torch.Tensor], score: Optional[torch.Tensor],
                kw: Optional[torch.Tensor], scale: float, causal: bool, bhsd: bool) -> tuple[torch.Tensor, torch.Tensor]:
    """O (layout of q) and kw [B, Hk, Tk] plus the probabilities' sums."""
    o, _, _, w = _attend(q, k, v, pk, pv, lengths, mask, score, kw, scale, causal, True, False, bhsd)
    return o, w


@key_weights.register_fake
def _key_weights_fake(q, k, v, pk, pv, lengths, mask, score, kw, scale, causal, bhsd):
    B, Tq, Tp, Tk, Hq, Hk, D = _sizes(q, k, pk, bhsd)
    return _like_output(q, bhsd), q.new_empty((B, Hk, Tk), dtype=torch.float32)


def tilelang_shared_prefix_attention(
    query: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    prefix_key: torch.Tensor,
    prefix_value: torch.Tensor,
    *,
    lengths: Optional[torch.Tensor] = None,
    mask: Optional[torch.Tensor] = None,
    score: Optional[torch.Tensor] = None,
    scale: Optional[float] = None,
    is_causal: bool = False,
    layout: Layout = "bhsd",
    use_atomic_backward: bool = True,
) -> torch.Tensor:
    """Attention of a batch whose sequences share a prefix:
    ``softmax([Q Kp^T, Q K^T + score] * scale) [Vp; V]``, one softmax over the prefix's
    keys and each sequence's own.  The prefix is read and multiplied once for the batch.

    query [B, Hq, Tq, D], key / value [B, Hk, Tk, D]: the own keys, Tk may be 0;
    prefix_key / prefix_value [1, Hk, Tp, D] (``layout="bshd"``: heads and tokens
    exchanged), fp16 / bf16, D up to 256, GQA/MQA as in :func:`tilelang_flash_attention`.
    Every row sees the whole prefix; the following concern the own keys:
    lengths: int32 / int64 [B], the first ``lengths[b]`` keys exist (values are clamped
    to [0, Tk]; memory past them may hold anything).  mask: bool [B|1, Hq|1, Tq, Tk], True
    keeps.  score: float [B|1, Hq|1, Tq, Tk], added before scaling.  is_causal: row i
    keeps own key j iff j <= i (top-left, as everywhere in this package; a row that
    decodes behind a cache needs lengths or a mask instead).  Keys that the mask or causality
    drops get probability 0, which times a value that is not finite is NaN, as in the formula.
    Rows that keep no key at all (no prefix) are NaN, as in the attention.
    Differentiable in query, key, value, prefix_key and prefix_value (the prefix's
    gradients are summed over the batch); ``use_atomic_backward`` as there.
    Returns the output in the input layout.
    """
    if _plain(layout, query, key, value, prefix_key, prefix_value, lengths, mask, score) and prefix_key is not None:
        r = _host().attend_plain(query, key, value, prefix_key, prefix_value, lengths, mask, score, None,
                                 None if scale is None else float(scale), bool(is_causal), False, layout == "bhsd")
        if r is not None:
            return r[0]
    B, Hq, Hk, Tq, Tk, D = _sizes_of(query, key, value, layout)
    _check_prefix(prefix_key, prefix_value, layout, Hk, D)
    _check_types("query", query, key=key, value=value, prefix_key=prefix_key, prefix_value=prefix_value)
    mask, score = _check_sides(mask, score, dict(batch=B, heads=Hq, seqlen_q=Tq, seqlen_k=Tk), query.device)
    lengths = _check_lengths(lengths, B, query.device)
    _check_gpu(query)
    scale = float(D ** -0.5 if scale is None else scale)
    causal, bhsd = bool(is_causal), layout == "bhsd"
    tensors = (query, key, value, prefix_key, prefix_value)
    grad = _wants_grad(*tensors)
    if _fa2._plain_eager(*tensors, lengths, mask, score):
        if not grad:
            return _attend(query, key, value, prefix_key, prefix_value, lengths, mask, score, None, scale, causal, False,
                           False, bhsd)[0]
        if query.numel() > 0 and key.numel() + prefix_key.numel() > 0:
            return _host().attend_train(query, key, value, prefix_key, prefix_value, lengths, mask, score, scale, causal,
                                        bool(use_atomic_backward), bhsd)
    # (the residual of O, for Delta: dQ and dK are sums over many keys and rows in which an error
    # of Delta adds up)
    return torch.ops.tilelang_fa2_4d_mask.prefix_fwd(query, key, value, prefix_key, prefix_value, lengths, mask, score,
                                                     scale, causal, bool(use_atomic_backward), grad, bhsd)[0]


def tilelang_attention_with_key_weights(
    query: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    *,
    key_weights: Optional[torch.Tensor] = None,
    prefix_key: Optional[torch.Tensor] = None,
    prefix_value: Optional[torch.Tensor] = None,
    lengths: Optional[torch.Tensor] = None,
    mask: Optional[torch.Tensor] = None,
    score: Optional[torch.Tensor] = None,
    scale: Optional[float] = None,
    is_causal: bool = False,
    layout: Layout = "bhsd",
) -> tuple[torch.Tensor, torch.Tensor]:
    """Attention that also adds up the weight each key received:
    ``weights[b, kvh, j] = key_weights[b, kvh, j] + sum over the rows i and the query
    heads of kvh's group of P[b, h, i, j]``, fp32 [B, Hk, Tk]; ``key_weights`` None: from 0.
    Keys that no row keeps, those past ``lengths`` among them, keep their value; rows that
    keep no key add nothing (their output is NaN, as in the attention).
    With ``prefix_key`` / ``prefix_value`` the keys stand behind a shared prefix (see
    :func:`tilelang_shared_prefix_attention`, also for the other arguments), which takes its
    share of every row's probability; the weights are those of the own keys.
    Returns (output in the input layout, weights as a new tensor).  For inference: there
    is no gradient, and inputs that ask for one are refused.
    """
    if _plain(layout, query, key, value, prefix_key, prefix_value, lengths, mask, score, key_weights):
        r = _host().attend_plain(query, key, value, prefix_key, prefix_value, lengths, mask, score, key_weights,
                                 None if scale is None else float(scale), bool(is_causal), True, layout == "bhsd")
        if r is not None:
            return r
    B, Hq, Hk, Tq, Tk, D = _sizes_of(query, key, value, layout)
    if (prefix_key is None) != (prefix_value is None):
        raise ValueError("prefix_key and prefix_value must be given together")
    if prefix_key is not None:
        _check_prefix(prefix_key, prefix_value, layout, Hk, D)
    _check_types("query", query, key=key, value=value, prefix_key=prefix_key, prefix_value=prefix_value)
    mask, score = _check_sides(mask, score, dict(batch=B, heads=Hq, seqlen_q=Tq, seqlen_k=Tk), query.device)
    lengths = _check_lengths(lengths, B, query.device)
    if key_weights is not None:
        _check_key_weights(key_weights, B, Hk, Tk, query.device)
    _check_gpu(query)
    tensors = (query, key, value, prefix_key, prefix_value, score, key_weights)
    if _wants_grad(*tensors):
        raise ValueError("attention with key weights has no gradient: call it under torch.no_grad()")
    scale = float(D ** -0.5 if scale is None else scale)
    causal, bhsd = bool(is_causal), layout == "bhsd"
    if _fa2._plain_eager(*tensors, lengths, mask):
        o, _, _, w = _attend(query, key, value, prefix_key, prefix_value, lengths, mask, score, key_weights, scale,
                             causal, True, False, bhsd)
        return o, w
    return torch.ops.tilelang_fa2_4d_mask.key_weights(query, key, value, prefix_key, prefix_value, lengths, mask, score,
                                                      key_weights, scale, causal, bhsd)


# ---- eviction ------------------------------------------------------------------------


def _evict(k, v, kw, lengths, keep, recent, bhsd):
    if k.shape[0] * k.shape[1 if bhsd else 2] == 0:
        shape = list(k.shape)
        shape[2 if bhsd else 1] = keep
        w = kw[:, :, :keep].clone()
        return k.new_empty(shape), v.new_empty(shape), w, torch.empty_like(w, dtype=torch.int64)
    return _timed("fa_evict", _host().evict, k, v, kw, lengths, keep, recent, bhsd)


@torch.library.custom_op(f"{_NS}::evict", mutates_args=(), device_types="cuda")
def evict(k: torch.Tensor, v: torch.Tensor, kw: torch.Tensor, lengths: Optional[torch.Tensor], keep: int, recent: int,
          bhsd: bool) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """K, V, weights and indices of the kept keys."""
    return _evict(k, v, kw, lengths, keep, recent, bhsd)


@evict.register_fake
def _evict_fake(k, v, kw, lengths, keep, recent, bhsd):
    shape = list(k.shape)
    shape[2 if bhsd else 1] = keep
    w = kw.new_empty((kw.shape[0], kw.shape[1], keep))
    return k.new_empty(shape), v.new_empty(shape), w, torch.empty_like(w, dtype=torch.int64)


def tilelang_evict_keys(
    key: torch.Tensor,
    value: torch.Tensor,
    key_weights: torch.Tensor,
    *,
    keep: int,
    recent: int = 0,
    lengths: Optional[torch.Tensor] = None,
    layout: Layout = "bhsd",
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """A K/V cache cut down to ``keep`` keys per sequence and head.

    Of a sequence's n keys (``lengths[b]``, clamped to [0, Tk]; Tk without lengths) every head
    keeps the last ``recent`` and, of the others, those with the largest ``key_weights``
    (fp32 [B, Hk, Tk]; ties go to the lowest index, NaN counts as the largest), ``keep`` in
    all; with n <= keep all of them.  key, value: [B, Hk, Tk, D] (``layout="bshd"``:
    [B, Tk, Hk, D]), fp16 / bf16, D up to 256; 1 <= keep <= Tk, 0 <= recent <= keep.
    Returns new tensors: key and value [B, Hk, keep, D] (or bshd) with the kept keys in
    their order, their weights [B, Hk, keep] and their indices in the old cache (int64).
    A sequence holds min(n, keep) keys afterwards; places behind them are zeros, index -1.
    """
    if _plain(layout, key, value, key_weights, lengths):
        r = _host().evict_plain(key, value, key_weights, lengths, int(keep), int(recent), layout == "bhsd")
        if r is not None:
            return r
    if key.dim() != 4 or value.dim() != 4:
        raise ValueError("key and value must be rank-4 tensors")
    if layout not in ("bhsd", "bshd"):
        raise ValueError(f"unsupported layout: {layout}")
    if key.shape != value.shape:
        raise ValueError("key and value must have the same shape")
    bhsd = layout == "bhsd"
    B, Hk, Tk = key.shape[0], key.shape[1 if bhsd else 2], key.shape[2 if bhsd else 1]
    if not 1 <= key.shape[3] <= 256:
        raise ValueError(f"head dimension {key.shape[3]} is not supported (1 to 256)")
    _check_types("key", key, value=value)
    keep, recent = int(keep), int(recent)
    if not 1 <= keep <= Tk:
        raise ValueError(f"keep must lie in [1, {Tk}], got {keep}")
    if not 0 <= recent <= keep:
        raise ValueError(f"recent must lie in [0, keep = {keep}], got {recent}")
    _check_key_weights(key_weights, B, Hk, Tk, key.device)
    lengths = _check_lengths(lengths, B, key.device)
    _check_gpu(key)
    if _wants_grad(key, value, key_weights):
        raise ValueError("eviction has no gradient: call it under torch.no_grad()")
    if _fa2._plain_eager(key, value, key_weights, lengths):
        return _evict(key, value, key_weights, lengths, keep, recent, bhsd)
    return torch.ops.tilelang_fa2_4d_mask.evict(key, value, key_weights, lengths, keep, recent, bhsd)


# ---- rotary positions ------------------------------------------------------------------


@torch.library.custom_op(f"{_NS}::rotary", mutates_args=(), device_types="cuda")
def rotary(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, sections: list[int],
           interleaved: bool, inverse: bool, bhsd: bool) -> tuple[torch.Tensor, torch.Tensor]:
    """q and k (their layout) turned by positions x inv_freq, or back (``inverse``)."""
    with torch.no_grad():
        return _timed("fa_rotary", _host().rotary, q, k, positions, inv_freq, sections, interleaved, inverse, bhsd)


@rotary.register_fake
def _rotary_fake(q, k, positions, inv_freq, sections, interleaved, inverse, bhsd):
    return _like_output(q, bhsd), _like_output(k, bhsd)


def _rotary_setup(ctx, inputs, output):
    q, k, positions, inv_freq, sections, interleaved, inverse, bhsd = inputs
    ctx.save_for_backward(positions, inv_freq)
    ctx.how = list(sections), interleaved, not inverse, bhsd


def _rotary_backward(ctx, dq, dk):
    positions, inv_freq = ctx.saved_tensors
    return (*torch.ops.tilelang_fa2_4d_mask.rotary(dq, dk, positions, inv_freq, *ctx.how),) + (None,) * 6


rotary.register_autograd(_rotary_backward, setup_context=_rotary_setup)


def tilelang_rotary_embedding(
    query: torch.Tensor,
    key: torch.Tensor,
    positions: torch.Tensor,
    inv_freq: torch.Tensor,
    *,
    sections: Optional[Sequence[int]] = None,
    interleaved: bool = False,
    layout: Layout = "bhsd",
) -> tuple[torch.Tensor, torch.Tensor]:
    """Rotary positions of one or several axes (time, height, width, ...).

    query [B, Hq, T, D], key [B, Hk, T, D] (``layout="bshd"``: heads and tokens exchanged),
    fp16 / bf16, D up to 256.  positions: int32 / int64 [axes, B|1, T], any integers.
    inv_freq: float32 [R / 2], R <= D the rotary columns; columns from R on are copied
    (entries of 2^30 and more, infinite ones and NaN turn their pair into NaN).
    sections: how many of the R / 2 pairs turn with each axis, in order (None: one axis).
    Pair i turns by ``positions[axis(i), b, t] * inv_freq[i]``, multiplied in 64-bit fixed
    point and reduced exactly (off by less than 2^-31 of a turn while |position| < 2^32); it
    is columns (i, i + R / 2), or (2 i, 2 i + 1) with ``interleaved``:
    ``(a, b) -> (a cos - b sin, b cos + a sin)``.
    Differentiable in query and key.  Returns new tensors (query, key) in the input layout.
    """
    sections = None if sections is None else [int(x) for x in sections]
    if sections != [] and _plain(layout, query, key, positions, inv_freq):
        r = _host().rotary_plain(query, key, positions, inv_freq, sections or [], bool(interleaved), layout == "bhsd")
        if r is not None:
            return r
    if query.dim() != 4 or key.dim() != 4:
        raise ValueError("query and key must be rank-4 tensors")
    if layout not in ("bhsd", "bshd"):
        raise ValueError(f"unsupported layout: {layout}")
    bhsd = layout == "bhsd"
    t = 2 if bhsd else 1
    B, T, D = query.shape[0], query.shape[t], query.shape[3]
    if key.shape[0] != B or key.shape[t] != T or key.shape[3] != D:
        raise ValueError("query and key must have the same batch size, sequence length and head dimension")
    if 0 in (query.shape[3 - t], key.shape[3 - t]):
        raise ValueError("query and key must have at least one head")
    if not 2 <= D <= 256:
        raise ValueError(f"head dimension {D} is not supported (2 to 256)")
    _check_types("query", query, key=key)
    if inv_freq.dim() != 1 or inv_freq.dtype != torch.float32 or inv_freq.device != query.device:
        raise ValueError(f"inv_freq must be a float32 vector on {query.device}")
    pairs = inv_freq.shape[0]
    if not 1 <= pairs <= D // 2:
        raise ValueError(f"inv_freq must have 1 to {D // 2} entries, got {pairs}")
    sections = [pairs] if sections is None else sections
    if not 1 <= len(sections) <= _ext.ROTARY_AXES or min(sections) < 0 or sum(sections) != pairs:
        raise ValueError(f"sections must be 1 to {_ext.ROTARY_AXES} counts that add up to the {pairs} pairs of inv_freq")
    if positions.dtype not in (torch.int32, torch.int64) or positions.dim() != 3:
        raise ValueError("positions must be an int32 or int64 tensor [axes, B or 1, T]")
    if positions.shape[0] != len(sections) or positions.shape[1] not in (1, B) or positions.shape[2] != T:
        raise ValueError(f"positions has shape {tuple(positions.shape)}, expected [{len(sections)}, {B} or 1, {T}]")
    if positions.device != query.device:
        raise ValueError(f"positions must be on {query.device}, got {positions.device}")
    _check_gpu(query)
    if _wants_grad(inv_freq):
        raise ValueError("inv_freq gets no gradient: give it detached")
    inv_freq = inv_freq.contiguous()
    if _fa2._plain_eager(query, key, positions, inv_freq):
        return _host().rotary(query, key, positions, inv_freq, sections, bool(interleaved), False, bhsd)
    return torch.ops.tilelang_fa2_4d_mask.rotary(query, key, positions, inv_freq, sections, bool(interleaved), False, bhsd)


__all__ = ["tilelang_shared_prefix_attention", "tilelang_attention_with_key_weights", "tilelang_evict_keys",
           "tilelang_rotary_embedding"]
