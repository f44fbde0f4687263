"""The cache operators (cache.py) on the GPU against their definitions in 64 bits
(oracle/cache.py, which also derives what each result may be off by)."""

import math

import pytest
import torch

import tilelang_fa2_4d_mask as api
from oracle import cache as OC

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


def _within(name, got, want, bound):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{name}: NaN in other places"
    fin = torch.isfinite(want)
    bound = bound.expand_as(want) if torch.is_tensor(bound) else torch.full_like(want, bound)
    off = ((got - want).abs() - bound)[fin]
    assert off.numel() == 0 or off.max().item() <= 0, f"{name}: {off.max().item():.3e} past the bound"


def _to(x, layout, dev, how="contiguous"):
    """A [B, H, T, D] CPU tensor on the GPU, in the layout, in memory as `how` says."""
    if x is None:
        return None
    y = x.to(dev)
    if how == "token_major":          # [B, T, H, D] memory whatever the layout
        y = y.transpose(1, 2).contiguous()
        return y if layout == "bshd" else y.transpose(1, 2)
    y = y if layout == "bhsd" else y.transpose(1, 2)
    if how == "contiguous":
        return y.contiguous()
    if how == "slice":                # rows apart, columns of a wider tensor, off 16 bytes
        wide = torch.zeros((*y.shape[:3], y.shape[3] + 5), dtype=y.dtype, device=dev)
        wide[..., 3:3 + y.shape[3]] = y
        return wide[..., 3:3 + y.shape[3]]
    raise AssertionError(how)


def _inputs(seed, B, Hq, Hk, D, Tq, Tp, Tk, dtype, lengths, mask, score, lean=0.0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    u = r(1, Hk, 1, D)
    q = (r(B, Hq, Tq, D) + lean * u.repeat_interleave(Hq // Hk, 1)).to(dtype)
    k = (r(B, Hk, Tk, D) + lean * u * r(B, Hk, Tk, 1)).to(dtype)
    v = r(B, Hk, Tk, D).to(dtype)
    pk = pv = n = m = s = None
    if Tp:
        pk = (r(1, Hk, Tp, D) + lean * u * r(1, Hk, Tp, 1)).to(dtype)
        pv = r(1, Hk, Tp, D).to(dtype)
    if lengths == "ragged":
        n = torch.tensor([(b * 7919 + Tk // 2) % (Tk + 1) for b in range(B)])
        n[0] = Tk
        if B > 1:
            n[1] = 0
        if B > 2:
            n[2] = 1
    elif lengths == "past":           # clamped: negative and past the end
        n = torch.tensor([Tk + 1000 if b % 2 else -3 for b in range(B)])
    if mask == "bernoulli":           # odd row stride (byte loads); a row that keeps nothing
        m = (torch.rand((B, Hq, Tq, Tk + 1), generator=g) < 0.6)[..., :Tk]
        m[0, 0, 0] = False
    elif mask == "rows":              # broadcast over heads and batch
        m = (torch.rand((1, 1, Tq, Tk), generator=g) < 0.7).contiguous()
        m[0, 0, Tq - 1] = False
    elif mask == "late":              # the first tiles of every row dropped
        m = (torch.arange(Tk) >= Tk - max(1, Tk // 5)).expand(B, 1, Tq, Tk).contiguous()
    if score == "normal":
        s = r(B, Hq, Tq, Tk)
    elif score == "lowest":           # a float mask: the type's lowest value, all of row 0
        s = torch.where(torch.rand((B, 1, Tq, Tk), generator=g) < 0.5, 0.0, float(torch.finfo(dtype).min))
        s[:, :, 0] = float(torch.finfo(dtype).min)
    elif score == "-inf":
        s = torch.where(torch.rand((B, 1, Tq, Tk), generator=g) < 0.5, 0.0, -math.inf)
    return q, k, v, pk, pv, n, m, s


def _spoil(k, v, n):
    """Anything past the lengths: NaN and infinities."""
    if n is None:
        return k, v
    gone = (torch.arange(k.shape[2]) >= n.clamp(0, k.shape[2]).view(-1, 1))[:, None, :, None]
    return k.masked_fill(gone, math.nan), v.masked_fill(gone, math.inf)


# B Hq Hk D Tq Tp Tk dtype lengths mask score causal scale layout memory
FORWARD = [
    (1, 1, 1, 64, 1, 1, 1, BF, None, None, None, False, None, "bhsd", "contiguous"),
    (1, 4, 2, 128, 1, 0, 1, FP, None, None, None, False, None, "bhsd", "contiguous"),
    (2, 4, 4, 64, 1, 1, 0, BF, None, None, None, False, None, "bshd", "contiguous"),
    (3, 8, 2, 128, 1, 31, 33, BF, "ragged", None, None, False, None, "bhsd", "token_major"),
    (5, 8, 1, 64, 1, 1000, 63, FP, "ragged", None, None, False, None, "bhsd", "slice"),
    (4, 8, 2, 128, 1, 4099, 517, BF, "ragged", None, None, False, -0.09, "bhsd", "contiguous"),
    (33, 32, 1, 128, 2, 129, 64, BF, "past", None, None, False, None, "bshd", "contiguous"),
    (2, 6, 2, 96, 11, 33, 40, FP, None, None, None, True, None, "bhsd", "contiguous"),
    (3, 6, 2, 80, 7, 65, 300, BF, "ragged", "bernoulli", None, False, None, "bshd", "token_major"),
    (2, 4, 2, 40, 3, 100, 70, BF, None, "rows", "normal", False, None, "bhsd", "contiguous"),
    (3, 4, 2, 64, 5, 0, 4133, BF, "ragged", "bernoulli", None, False, None, "bhsd", "contiguous"),
    (2, 4, 4, 128, 4, 50, 700, BF, None, None, "lowest", False, None, "bhsd", "contiguous"),
    (2, 4, 4, 128, 4, 0, 700, FP, None, None, "lowest", True, None, "bhsd", "contiguous"),
    (2, 4, 2, 64, 3, 0, 90, BF, None, "late", "-inf", False, None, "bhsd", "contiguous"),
    (2, 4, 2, 64, 32, 70, 90, BF, "ragged", "late", None, True, 0.0, "bhsd", "contiguous"),
    (3, 4, 1, 256, 1, 700, 300, BF, "ragged", None, None, False, None, "bhsd", "contiguous"),
    (2, 4, 2, 256, 40, 65, 100, FP, "ragged", "bernoulli", "normal", True, None, "bhsd", "contiguous"),
    (2, 2, 1, 200, 5, 33, 31, BF, None, None, None, True, None, "bshd", "contiguous"),
    # enough rows and prefix for the blocks of 128 rows (a last block of few rows, a last tile of few keys)
    (40, 32, 16, 64, 1, 4099, 33, BF, "ragged", None, None, False, None, "bhsd", "contiguous"),
    (17, 32, 8, 128, 2, 4097, 20, FP, None, "rows", None, False, -0.09, "bshd", "contiguous"),
    (23, 48, 16, 96, 1, 4160, 0, BF, None, None, None, False, None, "bhsd", "slice"),
    (65, 16, 16, 80, 1, 4095, 40, BF, "ragged", None, "normal", False, 0.0, "bhsd", "contiguous"),
    # one key set in more ranges than half of what the join takes; both
    (1, 4, 1, 64, 1, 0, 40001, BF, "past", None, None, False, None, "bhsd", "contiguous"),
    (1, 2, 1, 128, 1, 40000, 70, FP, None, None, None, False, None, "bhsd", "contiguous"),
    (1, 2, 1, 64, 1, 40000, 40000, BF, None, None, None, False, None, "bshd", "contiguous"),
    # more rows per head, on both sides of what decides for the 256-row blocks
    (2, 4, 2, 128, 33, 65, 100, BF, None, None, None, True, None, "bhsd", "token_major"),
    (2, 4, 2, 64, 257, 300, 257, FP, None, None, None, True, None, "bhsd", "contiguous"),
    (3, 4, 2, 128, 300, 0, 300, BF, "ragged", None, None, True, None, "bhsd", "contiguous"),
    (2, 4, 2, 96, 100, 1100, 0, BF, None, None, None, False, None, "bhsd", "slice"),
    (2, 4, 2, 128, 65, 513, 200, BF, "ragged", "bernoulli", "normal", False, -0.1, "bshd", "contiguous"),
    (2, 4, 4, 64, 130, 40, 130, FP, None, None, "lowest", True, None, "bhsd", "contiguous"),
    (1, 8, 8, 40, 70, 10, 70, BF, None, "rows", None, False, 0.0, "bhsd", "contiguous"),
    (2, 4, 2, 128, 64, 30, 100, BF, None, None, None, True, None, "bhsd", "contiguous"),
    (2, 4, 2, 64, 128, 100, 100, FP, "ragged", None, None, False, None, "bshd", "contiguous"),
    (2, 4, 2, 128, 133, 165, 140, BF, None, None, None, True, None, "bhsd", "token_major"),
    (2, 4, 2, 96, 150, 1100, 0, BF, None, None, None, False, None, "bhsd", "slice"),
    (2, 4, 2, 128, 129, 513, 200, BF, "ragged", "bernoulli", "normal", False, -0.1, "bshd", "contiguous"),
    (1, 8, 8, 40, 170, 180, 170, BF, None, "rows", None, False, 0.0, "bhsd", "contiguous"),
    (2, 4, 2, 64, 300, 77, 500, FP, "past", "late", None, True, None, "bhsd", "contiguous"),
    # lengths: ranges of one sequence that the next one does not have, none at all
    (5, 4, 2, 128, 260, 0, 700, BF, "ragged", None, None, False, None, "bhsd", "contiguous"),
    (5, 4, 2, 64, 200, 300, 900, FP, "ragged", None, None, True, None, "bshd", "token_major"),
    (3, 2, 2, 96, 150, 0, 2000, BF, "ragged", None, None, False, -0.1, "bhsd", "slice"),
    (20, 16, 4, 128, 257, 0, 300, BF, "ragged", None, None, True, None, "bhsd", "contiguous"),
    (20, 16, 4, 64, 270, 30, 300, BF, "past", None, None, False, 0.0, "bhsd", "contiguous"),
    # one range of one key set
    (2, 4, 2, 64, 70, 0, 200, BF, "ragged", "bernoulli", None, True, None, "bhsd", "contiguous"),
    (2, 4, 2, 128, 140, 0, 90, FP, None, None, "normal", False, None, "bshd", "slice"),
    (2, 4, 2, 128, 140, 0, 90, FP, None, None, "lowest", True, None, "bhsd", "contiguous"),
    (2, 16, 16, 96, 260, 0, 300, BF, "past", None, None, True, 0.0, "bhsd", "contiguous"),
    (2, 4, 1, 64, 270, 90, 0, BF, None, None, None, False, -0.1, "bshd", "token_major"),
]


def _id(c):
    return f"B{c[0]}H{c[1]}-{c[2]}D{c[3]}T{c[4]}-{c[5]}+{c[6]}{c[8] or ''}{c[9] or ''}{c[10] or ''}{'c' if c[11] else ''}"


def test_the_prefix_plan_of_the_cases(cuda):
    """Each way to run the prefix is among the cases: in blocks of 32 rows, of 128, of 256."""
    import ctypes

    from tilelang_fa2_4d_mask import _ext

    ways = set()
    for B, Hq, Hk, D, Tq, Tp, Tk, *_ in FORWARD:
        p, plan = _ext.FaPrefixParams(), _ext.FaPrefixPlan()
        p.batch, p.seqlen_q, p.seqlen_p, p.seqlen_k, p.heads_q, p.heads_k = B, Tq, Tp, Tk, Hq, Hk
        p.head_dim = 64 if D <= 64 else (128 if D <= 128 else 256)
        p.scale = 1.0
        _ext.check(_ext.load_library().fa_prefix_plan(ctypes.byref(p), ctypes.byref(plan)), "fa_prefix_plan")
        ways.add((plan.few_rows, plan.wide_rows, p.head_dim, plan.prefix_split > 1, plan.own_split > 1))
    assert {(few, wide, d) for few, wide, d in ((1, 0, 64), (1, 0, 128), (1, 0, 256), (1, 1, 64), (1, 1, 128), (0, 0, 64),
                                                (0, 0, 128))} <= {w[:3] for w in ways}
    assert {(1, True, False), (1, False, True), (0, True, False)} <= {(w[0], w[3], w[4]) for w in ways}


@pytest.mark.parametrize("case", FORWARD, ids=_id)
def test_prefix_forward(cuda, case):
    B, Hq, Hk, D, Tq, Tp, Tk, dtype, lengths, mask, score, causal, scale, layout, how = case
    print("case", case, flush=True)
    q, k, v, pk, pv, n, m, s = _inputs(1, *case[:7], dtype, lengths, mask, score)
    want = OC.Attention(q, k, v, pk, pv, n, m, s, scale, causal)
    ks, vs = _spoil(k, v, n)
    if pk is None:
        pk = pv = q.new_empty((1, Hk, 0, D))
    dev = [_to(x, layout, cuda, how) for x in (q, ks, vs, pk, pv)]
    on = lambda x: None if x is None else x.to(cuda)  # noqa: E731
    # (the mask keeps its odd row stride)
    md = None if m is None else (torch.zeros((*m.shape[:3], Tk + 1), dtype=torch.bool, device=cuda)[..., :Tk].copy_(m)
                                 if mask == "bernoulli" else on(m))
    out = api.tilelang_shared_prefix_attention(*dev, lengths=on(n), mask=md, score=on(s), scale=scale, is_causal=causal,
                                               layout=layout)
    out = out if layout == "bhsd" else out.transpose(1, 2)
    _within("out", out, want.o, want.out_bound(dtype))
    # through the custom op: LSE and O's residual
    o, lse, lo = torch.ops.tilelang_fa2_4d_mask.prefix_fwd(*dev, None if n is None else on(n).clamp(0, Tk).int(), md, on(s), want.scale, causal, False, True,
                                                           layout == "bhsd")
    dead = ~want.keep.any(3) | torch.isneginf(want.s).all(3)
    lse = lse.double().cpu()
    assert torch.equal(torch.isposinf(lse), dead)
    # the logits' error, and lse's own fp32 step
    off = (lse - want.lse2).abs() - (want.off[..., 0] / math.log(2) + 2.0 ** -23 * want.lse2.abs())
    assert off[~dead].numel() == 0 or off[~dead].max().item() <= 0
    both = o.double() + lo.double()
    both = both if layout == "bhsd" else both.transpose(1, 2)
    _within("out + residual", both, want.o, want.out_bound(dtype) - OC.U[dtype] * (1 - OC.U[dtype]) * want.o.abs())


# the gradients: B Hq Hk D Tq Tp Tk dtype lengths mask score causal scale layout memory
BACKWARD = [
    (1, 2, 1, 64, 1, 5, 3, BF, None, None, None, False, None, "bhsd", "contiguous"),
    (3, 8, 2, 128, 1, 100, 40, FP, "ragged", None, None, False, None, "bshd", "contiguous"),
    (2, 4, 2, 128, 64, 96, 64, BF, None, None, None, True, None, "bhsd", "token_major"),
    (3, 4, 2, 64, 65, 33, 65, FP, "ragged", None, None, True, None, "bhsd", "contiguous"),
    (2, 4, 4, 96, 40, 100, 50, BF, None, "rows", "normal", False, None, "bhsd", "contiguous"),
    (2, 4, 2, 40, 30, 20, 30, BF, None, "bernoulli", None, True, -0.1, "bhsd", "contiguous"),
    (2, 2, 1, 256, 33, 64, 40, BF, None, None, None, True, None, "bhsd", "contiguous"),
    (2, 2, 1, 200, 20, 40, 31, FP, "ragged", None, "normal", False, None, "bshd", "slice"),
    (2, 4, 2, 64, 20, 0, 20, BF, "ragged", None, None, True, None, "bhsd", "contiguous"),
    (2, 4, 2, 64, 20, 35, 0, BF, None, None, None, False, None, "bhsd", "contiguous"),
    (2, 16, 4, 128, 300, 700, 300, BF, None, None, None, True, None, "bhsd", "contiguous"),
    (1, 4, 2, 64, 40, 40, 40, BF, None, None, None, True, 0.0, "bhsd", "contiguous"),
    (3, 4, 2, 64, 131, 133, 131, FP, "ragged", None, None, True, None, "bhsd", "contiguous"),
    (2, 4, 2, 128, 140, 200, 150, BF, None, "rows", "normal", False, None, "bshd", "slice"),
    (2, 4, 2, 64, 140, 0, 140, BF, None, None, None, True, None, "bhsd", "contiguous"),
]


@pytest.mark.parametrize("atomic", [True, False])
@pytest.mark.parametrize("case", BACKWARD, ids=_id)
def test_prefix_backward(cuda, case, atomic):
    B, Hq, Hk, D, Tq, Tp, Tk, dtype, lengths, mask, score, causal, scale, layout, how = case
    print("case", case, flush=True)
    # keys that lean one way, so that rows lie on few keys and the two sets' dQ cancel
    q, k, v, pk, pv, n, m, s = _inputs(2, *case[:7], dtype, lengths, mask, score, lean=0.6)
    if lengths == "ragged" and Tp == 0:
        n = n.clamp(min=1)            # (rows without a key: the attention's own policy, tested there)
    want = OC.Attention(q, k, v, pk, pv, n, m, s, scale, causal)
    do = torch.randn(q.shape, generator=torch.Generator().manual_seed(3)).to(dtype)
    if pk is None:
        pk = pv = q.new_empty((1, Hk, 0, D))
    ks, vs = _spoil(k, v, n)
    dev = [_to(x, layout, cuda, how).detach().requires_grad_(True) for x in (q, ks, vs, pk, pv)]
    on = lambda x: None if x is None else x.to(cuda)  # noqa: E731
    out = api.tilelang_shared_prefix_attention(*dev, lengths=on(n), mask=on(m), score=on(s), scale=scale,
                                               is_causal=causal, layout=layout, use_atomic_backward=atomic)
    out.backward(_to(do, layout, cuda))
    got = [x.grad if layout == "bhsd" else x.grad.transpose(1, 2) for x in dev]
    for name, g, w, bound in zip(("dq", "dk", "dv", "dpk", "dpv"), got, want.grads(do), want.grad_bounds(do, dtype)):
        if w.numel():
            _within(name, g, w, bound)


@pytest.mark.parametrize("case", [
    ((2, 4, 2, 128, 70, 90, 70), None, None, None, "bhsd"), ((3, 4, 2, 64, 9, 40, 33), "ragged", "rows", "normal", "bshd"),
    ((2, 4, 2, 96, 33, 0, 40), None, "bernoulli", None, "bhsd"), ((2, 4, 2, 64, 20, 50, 0), None, None, None, "bhsd"),
    ((2, 4, 2, 40, 12, 20, 30), "ragged", None, None, "bshd"), ((2, 2, 1, 256, 12, 20, 30), "past", None, None, "bhsd")],
    ids=lambda c: str(c[0]))
def test_prefix_native_backward(cuda, case):
    """The native node and the custom ops give the same bits; so do a second backward, saved tensors
    that went through the host, and a gradient that is laid out otherwise."""
    from tilelang_fa2_4d_mask.fa2 import record_kernel_events

    shape, lengths, mask, score, layout = case
    q, k, v, pk, pv, n, m, s = _inputs(11, *shape, BF, lengths, mask, score)
    if pk is None:
        pk = pv = q.new_empty((1, shape[2], 0, shape[3]))
    on = lambda x: None if x is None else x.to(cuda)  # noqa: E731
    leaves = [_to(x, layout, cuda).requires_grad_(True) for x in (q, k, v, pk, pv)]
    do = _to(torch.randn(q.shape, generator=torch.Generator().manual_seed(12)).to(BF), layout, cuda)

    def call():
        return api.tilelang_shared_prefix_attention(*leaves, lengths=on(n), mask=on(m), score=on(s), layout=layout,
                                                    use_atomic_backward=False)

    def grads(out, do=do, **kw):
        return torch.autograd.grad(out, leaves, do, **kw)

    out = call()
    assert "Prefix" in out.grad_fn.name()
    want = grads(out, retain_graph=True)
    for x, leaf in zip(want, leaves):
        assert x.shape == leaf.shape and x.dtype == leaf.dtype
    other = do.transpose(1, 2).contiguous().transpose(1, 2)
    with record_kernel_events():
        op = call()
        by_op = grads(op)
    with torch.autograd.graph.save_on_cpu():
        far = call()
    for name, got in (("again", grads(out)), ("the ops", by_op), ("saved apart", grads(far)), ("other strides", grads(call(), other))):
        for x, y in zip(got, want):
            assert torch.equal(torch.nan_to_num(x), torch.nan_to_num(y)), name
    out = call()
    with torch.no_grad():
        out.add_(1)
    with pytest.raises(RuntimeError, match="inplace"):
        grads(out)


def test_ops_refuse_what_the_wrappers_would(cuda):
    """Called directly, the custom ops check what they are given before they launch."""
    q, k, v, pk, pv, n, m, s = (None if x is None else x.to(cuda) for x in
                                _inputs(9, 2, 4, 2, 64, 3, 5, 20, BF, "ragged", "rows", "normal"))
    ops = torch.ops.tilelang_fa2_4d_mask
    w, n = torch.zeros((2, 2, 20), device=cuda), n.int()
    good = [q, k, v, pk, pv, n, m, s]
    for i, bad in ((0, q.float()), (1, k[:, :, :, :32]), (2, v[:, :, :19]), (3, pk[:, :1]), (4, pv[..., :32]), (5, n.long()),
                   (5, n[:1]), (6, m[..., :19]), (7, s[:, :3]), (7, s.cpu())):
        args = list(good)
        args[i] = bad
        with pytest.raises(RuntimeError):
            ops.prefix_fwd(*args, 0.1, False, False, False, True)
        with pytest.raises(RuntimeError):
            ops.key_weights(*args, w, 0.1, False, True)
    for bad in (w[:, :, :19], w.half(), w[:, :1]):
        with pytest.raises(RuntimeError):
            ops.key_weights(*good, bad, 0.1, False, True)
        with pytest.raises(RuntimeError):
            ops.evict(k, v, bad, n, 5, 1, True)
    for keep, recent in ((0, 0), (21, 0), (5, 6), (5, -1)):
        with pytest.raises(RuntimeError):
            ops.evict(k, v, w, n, keep, recent, True)
    pos, freq = torch.zeros((1, 2, 3), dtype=torch.int64, device=cuda), torch.ones(32, device=cuda)
    kr = k[:, :, :3]
    for a in ((q, k, pos, freq, [32]), (q, kr, pos[:, :, :2], freq, [32]), (q, kr, pos, freq[::2], [16]),
              (q, kr, pos, torch.ones(33, device=cuda), [33]), (q, kr, pos, freq, [31]), (q, kr, pos.float(), freq, [32]),
              (q, kr, pos, freq.double(), [32])):
        with pytest.raises(RuntimeError):
            ops.rotary(*a, False, False, True)


def test_prefix_gradient_against_differences(cuda):
    """The gradients of sum(out * do) against central differences of the 64-bit definition,
    along random directions: they differ by at most the gradients' own bounds and h^2."""
    case = (2, 4, 2, 64, 9, 21, 13)
    q, k, v, pk, pv, n, m, s = _inputs(5, *case, BF, "ragged", "rows", "normal")
    g = torch.Generator().manual_seed(6)
    do = torch.randn(q.shape, generator=g).to(BF)
    dev = [x.to(cuda).requires_grad_(True) for x in (q, k, v, pk, pv)]
    api.tilelang_shared_prefix_attention(*dev, lengths=n.to(cuda), mask=m.to(cuda), score=s.to(cuda)).backward(do.to(cuda))
    base = [x.double() for x in (q, k, v, pk, pv)]
    bounds = OC.Attention(q, k, v, pk, pv, n, m, s).grad_bounds(do, BF)
    h = 1e-4
    loss = lambda xs: (OC.Attention(*xs, n, m, s).o * do.double()).sum().item()  # noqa: E731
    for i in range(5):
        d = torch.randn(base[i].shape, generator=g, dtype=torch.float64)
        up, down = (loss([x + sign * h * d if j == i else x for j, x in enumerate(base)]) for sign in (1, -1))
        got = (dev[i].grad.double().cpu() * d).sum().item()
        # third derivatives of a softmax of these logits: well below 10^3 of the values' sizes
        allowed = (bounds[i] * d.abs()).sum().item() + 1e3 * h * h
        assert abs(got - (up - down) / (2 * h)) <= allowed, i


def test_prefix_ds_limits_and_modes(cuda):
    """The routes of the backward (no dS tiles, slices, one piece) hold to the same bounds, and
    the non-atomic mode repeats bit by bit."""
    from tilelang_fa2_4d_mask import fa2

    case = (2, 8, 2, 128, 512, 640, 512)
    q, k, v, pk, pv, n, m, s = _inputs(7, *case, BF, None, None, None, lean=0.6)
    do = torch.randn(q.shape, generator=torch.Generator().manual_seed(8)).to(BF)
    want = OC.Attention(q, k, v, pk, pv, causal=True)
    grads, bounds = want.grads(do), want.grad_bounds(do, BF)

    def step(limit):
        old, fa2.DS_LIMIT_BYTES = fa2.DS_LIMIT_BYTES, limit
        try:
            dev = [x.to(cuda).requires_grad_(True) for x in (q, k, v, pk, pv)]
            api.tilelang_shared_prefix_attention(*dev, is_causal=True, use_atomic_backward=False).backward(do.to(cuda))
            return [x.grad for x in dev]
        finally:
            fa2.DS_LIMIT_BYTES = old

    for limit in (0, -1, 24 << 20, 8 << 20):
        a, b = step(limit), step(limit)
        for name, x, y, w, bound in zip(("dq", "dk", "dv", "dpk", "dpv"), a, b, grads, bounds):
            assert torch.equal(x, y), (limit, name)
            _within(f"{name} at limit {limit}", x, w, bound)


# ---- key weights ----------------------------------------------------------------------

WEIGHTS = [
    (1, 1, 1, 64, 1, 0, 1, BF, None, None, None, False, None, "bhsd", "contiguous"),
    (3, 8, 2, 128, 1, 0, 33, BF, "ragged", None, None, False, None, "bhsd", "contiguous"),
    (2, 8, 8, 64, 1, 0, 4097, FP, None, None, None, False, -0.125, "bshd", "contiguous"),
    (4, 32, 1, 128, 2, 77, 1030, BF, "past", None, None, False, None, "bhsd", "token_major"),
    (2, 6, 2, 96, 7, 33, 300, BF, "ragged", "bernoulli", None, True, None, "bhsd", "slice"),
    (2, 4, 2, 40, 5, 0, 200, FP, None, "rows", "normal", False, None, "bhsd", "contiguous"),
    (2, 4, 2, 64, 6, 0, 300, BF, "ragged", None, "lowest", False, None, "bhsd", "contiguous"),
    (2, 4, 2, 64, 6, 9, 100, BF, None, "late", "-inf", False, None, "bhsd", "contiguous"),
    (3, 4, 1, 256, 3, 20, 300, BF, "ragged", None, None, False, None, "bhsd", "contiguous"),
    (20, 32, 8, 128, 1, 8200, 77, BF, "ragged", None, None, False, None, "bhsd", "contiguous"),   # (128-row blocks)
    (1, 4, 2, 64, 1, 0, 45000, BF, None, None, None, False, None, "bhsd", "contiguous"),
    (2, 6, 2, 96, 5, 33, 300, BF, "ragged", "bernoulli", None, True, None, "bhsd", "slice"),
    (3, 16, 1, 128, 1, 40, 290, FP, "past", "rows", "normal", False, 0.0, "bshd", "contiguous"),
    # more rows: the sums in a pass of their own
    (2, 4, 2, 128, 40, 0, 40, BF, None, None, None, True, None, "bhsd", "token_major"),
    (2, 8, 2, 64, 257, 65, 300, FP, "ragged", None, None, False, None, "bshd", "contiguous"),
    (1, 16, 2, 96, 300, 0, 300, BF, None, "bernoulli", None, True, None, "bhsd", "contiguous"),
    (2, 4, 2, 128, 65, 0, 700, BF, "ragged", "rows", "normal", False, -0.09, "bhsd", "contiguous"),
    (2, 4, 2, 64, 70, 0, 200, BF, "ragged", None, "lowest", False, None, "bhsd", "contiguous"),
    (2, 4, 2, 64, 70, 30, 200, FP, None, "late", "lowest", True, None, "bhsd", "contiguous"),
    (1, 4, 4, 256, 50, 0, 300, BF, None, None, None, True, 0.0, "bhsd", "contiguous"),
    (1, 8, 1, 64, 1000, 0, 129, BF, None, None, None, False, None, "bhsd", "contiguous"),
    (2, 16, 1, 64, 5, 0, 129, FP, "ragged", None, "-inf", False, None, "bhsd", "contiguous"),
    (2, 4, 2, 64, 140, 30, 200, FP, None, "late", "lowest", True, None, "bhsd", "contiguous"),
    (2, 8, 2, 128, 131, 300, 299, BF, "ragged", None, None, True, None, "bshd", "contiguous"),
    (1, 6, 2, 128, 700, 0, 520, BF, None, None, None, True, None, "bhsd", "token_major"),
    (5, 4, 2, 128, 140, 0, 600, BF, "ragged", None, None, False, None, "bhsd", "contiguous"),
]


@pytest.mark.parametrize("prior", [False, True])
@pytest.mark.parametrize("case", WEIGHTS, ids=_id)
def test_key_weights(cuda, case, prior):
    B, Hq, Hk, D, Tq, Tp, Tk, dtype, lengths, mask, score, causal, scale, layout, how = case
    print("case", case, flush=True)
    q, k, v, pk, pv, n, m, s = _inputs(11, *case[:7], dtype, lengths, mask, score)
    want = OC.Attention(q, k, v, pk, pv, n, m, s, scale, causal)
    before = None
    if prior:                          # a slice of a wider tensor
        before = torch.rand((B, Hk, Tk + 3), generator=torch.Generator().manual_seed(4))[..., :Tk]
    ks, vs = _spoil(k, v, n)
    on = lambda x: None if x is None else x.to(cuda)  # noqa: E731
    dev = [_to(x, layout, cuda, how) for x in (q, ks, vs)]
    pd = [_to(x, layout, cuda, how) for x in (pk, pv)]
    wd = None if before is None else torch.zeros((B, Hk, Tk + 3), device=cuda)[..., :Tk].copy_(before)
    keep = None if wd is None else wd.clone()
    out, w = api.tilelang_attention_with_key_weights(*dev, key_weights=wd, prefix_key=pd[0], prefix_value=pd[1],
                                                     lengths=on(n), mask=on(m), score=on(s), scale=scale,
                                                     is_causal=causal, layout=layout)
    out = out if layout == "bhsd" else out.transpose(1, 2)
    _within("out", out, want.o, want.out_bound(dtype))
    _within("weights", w, want.weights(before), want.weights_bound(before))
    if keep is not None:
        assert torch.equal(wd, keep)   # the sums given stay as they were
        gone = ~OC.own_keep(B, Hq, Tq, Tk, n, m, causal).any(2).view(B, Hk, Hq // Hk, Tk).any(2)
        assert torch.equal(w.cpu()[gone], before[gone])


# ---- eviction -------------------------------------------------------------------------

EVICT = [
    # B Hk T D keep recent dtype layout lengths weights
    (1, 1, 1, 64, 1, 0, BF, "bhsd", None, "rand"),
    (1, 1, 1, 64, 1, 1, FP, "bhsd", None, "rand"),
    (2, 3, 65, 128, 64, 0, BF, "bhsd", None, "rand"),
    (3, 2, 1000, 96, 300, 100, FP, "bshd", "ragged", "rand"),
    (4, 2, 1025, 64, 1000, 999, BF, "bhsd", "ragged", "rand"),
    (2, 2, 2049, 20, 77, 0, BF, "bhsd", None, "zeros"),        # all equal: the first ones
    (2, 2, 3000, 24, 1500, 10, BF, "bshd", "ragged", "few"),   # many ties
    (3, 4, 500, 128, 500, 20, BF, "bhsd", "past", "rand"),     # everything fits
    (2, 2, 700, 128, 128, 128, BF, "bhsd", "ragged", "rand"),  # the most recent alone
    (2, 2, 600, 40, 100, 5, FP, "bhsd", None, "odd"),          # NaN, infinities, -0, negative, subnormal
    (1, 8, 9001, 256, 33, 1, BF, "bhsd", None, "close"),       # weights that differ in their last bits
    (2, 2, 33001, 24, 20000, 100, BF, "bhsd", "ragged", "few"),   # more weights than the LDS holds
]


@pytest.mark.parametrize("case", EVICT, ids=lambda c: f"B{c[0]}H{c[1]}T{c[2]}D{c[3]}k{c[4]}r{c[5]}{c[8] or ''}{c[9]}")
@pytest.mark.parametrize("how", ["contiguous", "token_major", "slice"])
def test_evict(cuda, case, how):
    B, H, T, D, keep, recent, dtype, layout, lengths, kind = case
    print("case", case, how, flush=True)
    g = torch.Generator().manual_seed(21)
    k, v = (torch.randn((B, H, T, D), generator=g).to(dtype) for _ in range(2))
    w = torch.rand((B, H, T + 2), generator=g)[..., :T] * 3
    if kind == "zeros":
        w = torch.zeros_like(w)
    elif kind == "few":
        w = torch.randint(0, 3, w.shape, generator=g).float()
    elif kind == "close":
        w = 1 + torch.randint(0, 200, w.shape, generator=g) * 2.0 ** -23
    elif kind == "odd":
        w = torch.randn(w.shape, generator=g)
        for i, x in enumerate((math.nan, math.inf, -math.inf, -0.0, 0.0, 1e-42, -1e-42)):
            w[:, :, 10 + i::50] = x
    n = None
    if lengths == "ragged":
        n = torch.tensor([[T, 0, 1, T // 2][b % 4] for b in range(B)])
    elif lengths == "past":
        n = torch.tensor([T + 9 if b % 2 else -1 for b in range(B)])
    want = OC.evict(k, v, w, keep, recent, n)
    wd = torch.zeros((B, H, T + 2), device=cuda)[..., :T].copy_(w)
    got = api.tilelang_evict_keys(_to(k, layout, cuda, how), _to(v, layout, cuda, how), wd, keep=keep, recent=recent,
                                  lengths=None if n is None else n.to(cuda), layout=layout)
    got = [x.cpu() for x in got]
    if layout == "bshd":
        got[0], got[1] = got[0].transpose(1, 2), got[1].transpose(1, 2)
    assert torch.equal(got[3], want[3])
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert torch.equal(torch.nan_to_num(got[2], nan=7.0), torch.nan_to_num(want[2], nan=7.0))


# ---- rotary positions -----------------------------------------------------------------

ROTARY = [
    # B T Hq Hk D sections interleaved dtype layout memory positions (first, type, batch) theta
    (1, 1, 1, 1, 2, (1,), False, BF, "bhsd", "contiguous", (0, torch.int64, 1), 1e4),
    (2, 1, 4, 2, 128, (16, 24, 24), False, BF, "bhsd", "contiguous", (100000, torch.int64, 2), 1e6),
    (3, 5, 8, 2, 64, (32,), False, FP, "bshd", "contiguous", (0, torch.int32, 1), 1e4),
    (2, 7, 3, 3, 80, (10, 10), True, FP, "bshd", "token_major", (-500, torch.int32, 2), 1e4),
    (2, 9, 4, 1, 96, (8, 0, 16, 24), True, BF, "bhsd", "slice", (0, torch.int64, 1), 1e4),
    (1, 3, 2, 2, 20, (3, 2), False, BF, "bhsd", "contiguous", (2 ** 31 - 5, torch.int64, 1), 1e4),
    (1, 4, 5, 5, 21, (4,), True, FP, "bhsd", "contiguous", (-2 ** 32 + 9, torch.int64, 1), 1e4),
    (2, 6, 4, 2, 256, (64, 32, 32), False, BF, "bhsd", "token_major", (2 ** 20, torch.int64, 1), 1e6),
    (2, 33, 4, 2, 128, (1,) * 8, False, BF, "bhsd", "slice", (0, torch.int32, 2), 1e4),
]


def _rotary_case(case, seed=31):
    B, T, Hq, Hk, D, sections, interleaved, dtype, layout, how, (first, ptype, pb), theta = case
    g = torch.Generator().manual_seed(seed)
    q, k = (torch.randn((B, H, T, D), generator=g).to(dtype) for H in (Hq, Hk))
    pairs = sum(sections)
    pos = torch.randint(first, first + 4, (len(sections), pb, T), generator=g, dtype=torch.int64) + torch.arange(T) * (
        -1 if first > 2 ** 30 else 3)
    freq = (theta ** (-torch.arange(pairs, dtype=torch.float64) / pairs)).float()
    angle = OC.angles(pos.expand(-1, B, -1), freq, sections)
    return q, k, pos.to(ptype), freq, angle


@pytest.mark.parametrize("case", ROTARY, ids=lambda c: f"B{c[0]}T{c[1]}H{c[2]}-{c[3]}D{c[4]}s{'_'.join(map(str, c[5]))}")
def test_rotary(cuda, case):
    B, T, Hq, Hk, D, sections, interleaved, dtype, layout, how, _, _ = case
    print("case", case, flush=True)
    q, k, pos, freq, angle = _rotary_case(case)
    g = torch.Generator().manual_seed(5)
    dq, dk = (torch.randn(x.shape, generator=g).to(dtype) for x in (q, k))
    qd, kd = (_to(x, layout, cuda, how).detach().requires_grad_(True) for x in (q, k))
    yq, yk = api.tilelang_rotary_embedding(qd, kd, pos.to(cuda), freq.to(cuda), sections=sections, interleaved=interleaved,
                                           layout=layout)
    torch.autograd.backward([yq, yk], [_to(x, layout, cuda) for x in (dq, dk)])
    R = 2 * sum(sections)
    for name, x, got, back in (("q", q, yq, False), ("k", k, yk, False), ("dq", dq, qd.grad, True), ("dk", dk, kd.grad, True)):
        got = got if layout == "bhsd" else got.transpose(1, 2)
        want = OC.turn(x, angle, interleaved, back)
        _within(name, got, want, OC.turn_bound(x, want, angle, interleaved, dtype))
        assert torch.equal(got.detach().cpu()[..., R:], x[..., R:])


def test_rotary_gradients_beyond_the_first(cuda):
    """One gradient alone, a gradient of the gradient (the rotation forward again), no grad mode."""
    case = ROTARY[1]
    q, k, pos, freq, angle = _rotary_case(case)
    args = (pos.to(cuda), freq.to(cuda))
    kw = dict(sections=case[5])
    qd, kd = (x.to(cuda).requires_grad_(True) for x in (q, k))
    yq, _ = api.tilelang_rotary_embedding(qd, kd, *args, **kw)
    w = torch.randn(q.shape, generator=torch.Generator().manual_seed(1)).to(BF).to(cuda).requires_grad_(True)
    gq, gk = torch.autograd.grad((yq * w).float().sum(), [qd, kd], create_graph=True, allow_unused=True)
    assert gk is None or not gk.any()
    want = OC.turn(w.detach().cpu(), angle, False, True)
    _within("dq", gq, want, OC.turn_bound(w.detach().cpu(), want, angle, False, BF))
    x = torch.randn(q.shape, generator=torch.Generator().manual_seed(2)).to(BF)
    (gw,) = torch.autograd.grad(gq, [w], x.to(cuda))
    want = OC.turn(x, angle, False)
    _within("dw", gw, want, OC.turn_bound(x, want, angle, False, BF))
    with torch.no_grad():
        y, _ = api.tilelang_rotary_embedding(qd, kd, *args, **kw)
    assert not y.requires_grad and torch.equal(y, yq)


def test_rotary_far_frequencies(cuda):
    """Frequencies that are none turn their pair into NaN, others leave theirs alone."""
    q = torch.ones((1, 1, 2, 8), dtype=BF, device=cuda)
    freq = torch.tensor([1.0, math.inf, 2.0 ** 31, 0.0], device=cuda)
    y, _ = api.tilelang_rotary_embedding(q, q, torch.tensor([[[0, 5]]], device=cuda), freq)
    bad = torch.isnan(y)[0, 0, 1]
    assert bad.tolist() == [False, True, True, False] * 2
    assert torch.equal(y[..., [3, 7]], q[..., [3, 7]])


def test_rotary_negative_frequencies(cuda):
    """Turns backwards, down to frequencies that a double of one turn cannot hold beside it."""
    g = torch.Generator().manual_seed(33)
    q = torch.randn((1, 2, 5, 16), generator=g).to(FP)
    freq = torch.tensor([-1.0, -0.37, -2.0 ** -20, -1e-9, -1e-18, -1e-30, -math.pi, 1e-18])
    pos = torch.tensor([[[0, 1, -7, 10 ** 9, -2 ** 31]]])
    angle = OC.angles(pos, freq, (8,))
    y, _ = api.tilelang_rotary_embedding(q.to(cuda), q.to(cuda), pos.to(cuda), freq.to(cuda))
    want = OC.turn(q, angle, False)
    _within("q", y, want, OC.turn_bound(q, want, angle, False, FP))


# ---- together, captured, on other streams ------------------------------------------------


def test_a_serving_run(cuda):
    """As they are used together: rotated prompt keys fill the caches of a batch, the prompt's
    attention gives the keys their weights, the caches are cut down, tokens are decoded behind
    a shared prefix while the weights grow, and the caches are cut down again."""
    g = torch.Generator().manual_seed(41)
    B, Hq, Hk, D, Tp, T, cap, keep, recent = 3, 8, 2, 64, 50, 90, 100, 40, 8
    dt, scale = BF, D ** -0.5
    r = lambda *s: torch.randn(s, generator=g).to(dt)  # noqa: E731
    sections, freq = (8, 12, 12), (1e4 ** (-torch.arange(32, dtype=torch.float64) / 32)).float()
    pk, pv = r(1, Hk, Tp, D), r(1, Hk, Tp, D)
    q, k, v = r(B, Hq, T, D), r(B, Hk, T, D), r(B, Hk, T, D)
    n = torch.tensor([90, 61, 30])
    on = lambda x: x.to(cuda)  # noqa: E731
    pos = torch.arange(Tp, Tp + T).expand(3, 1, T)
    angle = OC.angles(pos.expand(-1, B, -1), freq, sections)
    qd, kd = api.tilelang_rotary_embedding(on(q), on(k), on(pos), on(freq), sections=sections)
    for x, y in ((q, qd), (k, kd)):
        want = OC.turn(x, angle, False)
        _within("rotated", y, want, OC.turn_bound(x, want, angle, False, dt))
    kc, vc = (torch.zeros((B, Hk, cap, D), dtype=dt, device=cuda) for _ in range(2))
    kc[:, :, :T], vc[:, :, :T] = kd, on(v)
    out, w = api.tilelang_attention_with_key_weights(qd, kc[:, :, :T], vc[:, :, :T], prefix_key=on(pk), prefix_value=on(pv),
                                                     lengths=on(n), is_causal=True, scale=scale)
    want = OC.Attention(qd.cpu(), kd.cpu(), v, pk, pv, n, scale=scale, causal=True)
    _within("prompt out", out, want.o, want.out_bound(dt))
    _within("prompt weights", w, want.weights(), want.weights_bound())
    cut = api.tilelang_evict_keys(kc[:, :, :T], vc[:, :, :T], w, keep=keep, recent=recent, lengths=on(n))
    for x, y in zip(cut, OC.evict(kd.cpu(), v, w.cpu(), keep, recent, n)):
        assert torch.equal(x.cpu(), y)
    kc, vc, w, idx = cut
    length = n.clamp(max=keep)
    assert ((idx >= 0).sum(2).cpu() == length[:, None]).all()
    for step in range(4):
        # room for the new token behind the kept keys
        room = torch.zeros((B, Hk, 1, D), dtype=dt, device=cuda)
        kc, vc = torch.cat([kc, room], 2), torch.cat([vc, room], 2)
        w = torch.nn.functional.pad(w, (0, 1))
        qt, kt, vt = r(B, Hq, 1, D), r(B, Hk, 1, D), r(B, Hk, 1, D)
        at = (n + Tp + step).view(1, B, 1).expand(3, B, 1)
        qt, kt = api.tilelang_rotary_embedding(on(qt), on(kt), on(at), on(freq), sections=sections)
        row = on(length).view(B, 1, 1, 1).expand(B, Hk, 1, D)
        kc.scatter_(2, row, kt)
        vc.scatter_(2, row, on(vt))
        length = length + 1
        before = w
        out, w = api.tilelang_attention_with_key_weights(qt, kc, vc, key_weights=w, prefix_key=on(pk), prefix_value=on(pv),
                                                         lengths=on(length), scale=scale)
        want = OC.Attention(qt.cpu(), kc.cpu(), vc.cpu(), pk, pv, length, scale=scale)
        _within(f"token {step}", out, want.o, want.out_bound(dt))
        _within(f"weights {step}", w, want.weights(before.cpu()), want.weights_bound(before.cpu()))
        plain = api.tilelang_shared_prefix_attention(qt, kc, vc, on(pk), on(pv), lengths=on(length), scale=scale)
        _within(f"token {step} without weights", plain, want.o, want.out_bound(dt))
    cut = api.tilelang_evict_keys(kc, vc, w, keep=20, recent=4, lengths=on(length))
    for x, y in zip(cut, OC.evict(kc.cpu(), vc.cpu(), w.cpu(), 20, 4, length)):
        assert torch.equal(x.cpu(), y)


def _calls(cuda, seed=51, B=3, Tk=700):
    """One call of each operator on inputs of its own: (function, inputs to refill)."""
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g).to(BF).to(cuda)  # noqa: E731
    Hq, Hk, D, Tp = 8, 2, 128, 900
    q, k, v, pk, pv = r(B, Hq, 1, D), r(B, Hk, Tk, D), r(B, Hk, Tk, D), r(1, Hk, Tp, D), r(1, Hk, Tp, D)
    q2, w = r(B, Hq, 140, D), torch.rand((B, Hk, Tk), generator=g).to(cuda)
    n = torch.tensor([Tk, 1, Tk // 2], dtype=torch.int32, device=cuda)[:B]
    pos = torch.arange(140, device=cuda).expand(1, 1, 140).contiguous()
    freq = torch.logspace(0, -3, 64, device=cuda)
    return (q, k, v, pk, pv, q2, w, n, pos, freq), {
        "prefix": lambda: (api.tilelang_shared_prefix_attention(q, k, v, pk, pv, lengths=n),),
        "prefix_many": lambda: (api.tilelang_shared_prefix_attention(q2, k, v, pk, pv),),
        "prefix_many_lengths": lambda: (api.tilelang_shared_prefix_attention(q2, k, v, pk, pv, lengths=n),),
        "weights": lambda: api.tilelang_attention_with_key_weights(q, k, v, key_weights=w, lengths=n),
        "weights_many": lambda: api.tilelang_attention_with_key_weights(q2, k, v, key_weights=w, is_causal=True),
        "evict": lambda: api.tilelang_evict_keys(k, v, w, keep=100, recent=10, lengths=n),
        "rotary": lambda: api.tilelang_rotary_embedding(q2, q2, pos, freq),
    }


NAMES = ["prefix", "prefix_many", "prefix_many_lengths", "weights", "weights_many", "evict", "rotary"]


@pytest.mark.parametrize("name", NAMES)
@torch.no_grad()
def test_captured(cuda, name):
    """Two graphs of a call each, replayed in turn with eager work between: every replay equals the
    eager result of what the inputs hold then."""
    sides = [_calls(cuda, 51), _calls(cuda, 52)]
    graphs, outs = [], []
    s = torch.cuda.Stream()
    for inputs, calls in sides:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            calls[name]()
        torch.cuda.current_stream().wait_stream(s)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(calls[name]())
        graphs.append(g)
    for i in range(3):
        for (inputs, calls), g, out in zip(sides, graphs, outs):
            inputs[0].mul_(0.9)
            inputs[5].mul_(1.1)
            inputs[6].add_(0.25)
            inputs[7].copy_(torch.tensor([700 - i, 3 * i, 350 + i], dtype=torch.int32))
            g.replay()
        torch.cuda.synchronize()
        for (inputs, calls), out in zip(sides, outs):
            want = calls[name]()
            torch.cuda.synchronize()
            for a, b in zip(out, want):
                assert torch.equal(torch.nan_to_num(a), torch.nan_to_num(b)), (name, i)


@pytest.mark.parametrize("name", NAMES)
@torch.no_grad()
def test_on_another_stream(cuda, name):
    """Calls on two streams at once, each with its own inputs, equal those on the default one."""
    sides = [_calls(cuda, 61), _calls(cuda, 62)]
    want = [calls[name]() for _, calls in sides]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sides]
    got = [[], []]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(sides[i][1][name]())
    torch.cuda.synchronize()
    for w, runs in zip(want, got):
        for r in runs:
            for a, b in zip(r, w):
                assert torch.equal(torch.nan_to_num(a), torch.nan_to_num(b))


@torch.no_grad()
def test_negative_views(cuda):
    """Views that stand for the negative of what memory holds."""
    (q, k, v, pk, pv, _, w, _, pos, freq), _ = _calls(cuda, 75)
    neg = lambda x: torch._neg_view(-x)  # noqa: E731
    s = torch.randn((1, 1, 1, k.shape[2]), generator=torch.Generator().manual_seed(1)).to(cuda)
    call = api.tilelang_attention_with_key_weights
    for a, b in ((call(q, k, v, key_weights=w, score=s), call(neg(q), neg(k), neg(v), key_weights=neg(w), score=neg(s))),
                 ([api.tilelang_shared_prefix_attention(q, k, v, pk, pv)],
                  [api.tilelang_shared_prefix_attention(q, k, v, neg(pk), neg(pv))]),
                 (api.tilelang_evict_keys(k, v, w, keep=9), api.tilelang_evict_keys(neg(k), neg(v), neg(w), keep=9)),
                 (api.tilelang_rotary_embedding(k, v, torch.arange(700, device=cuda).view(1, 1, -1), freq),
                  api.tilelang_rotary_embedding(neg(k), neg(v), torch.arange(700, device=cuda).view(1, 1, -1), neg(freq)))):
        for x, y in zip(a, b):
            assert torch.equal(x, y.resolve_neg())


@pytest.mark.parametrize("name", NAMES)
@torch.no_grad()
def test_custom_ops_give_the_same(cuda, name):
    """Through the custom ops (here: an open event log), bit by bit, under their entries' names."""
    from tilelang_fa2_4d_mask.fa2 import record_kernel_events

    _, calls = _calls(cuda, 71)
    want = calls[name]()
    with record_kernel_events() as log:
        got = calls[name]()
    entry = {"p": "fa_prefix_fwd", "w": "fa_prefix_fwd", "e": "fa_evict", "r": "fa_rotary"}[name[0]]
    assert list(log.elapsed_ms()) == [entry]
    for a, b in zip(got, want):
        assert torch.equal(torch.nan_to_num(a), torch.nan_to_num(b)) and a.stride() == b.stride()


def test_compiled_training_step(cuda):
    """A compiled step through rotary positions and a shared prefix: one graph, eager's results."""
    torch._dynamo.reset()
    inputs, _ = _calls(cuda, 81)
    _, k, v, pk, pv, q, _, n, pos, freq = inputs

    def step(q, k, v, pk, pv):
        q, kr = api.tilelang_rotary_embedding(q, k[:, :, :140], pos, freq)
        return api.tilelang_shared_prefix_attention(q, kr, v[:, :, :140], pk, pv, is_causal=True, use_atomic_backward=False)

    leaves = [x.clone().requires_grad_(True) for x in (q, k, v, pk, pv)]
    out = step(*leaves)
    want = torch.autograd.grad(out, leaves, torch.ones_like(out))
    compiled = torch.compile(step, fullgraph=True, backend="aot_eager")
    out2 = compiled(*leaves)
    got = torch.autograd.grad(out2, leaves, torch.ones_like(out2))
    assert torch.equal(out, out2)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_captured_training_step(cuda):
    """Forward and backward captured together (no eager graph of the same leaves alive), replayed
    on changed inputs."""
    inputs, _ = _calls(cuda, 91)
    _, k, v, pk, pv, q, _, _, pos, freq = inputs
    static = [x.clone().requires_grad_(True) for x in (q, k[:, :, :140].contiguous(), v[:, :, :140].contiguous(), pk, pv)]
    do = torch.randn_like(q)

    def step(leaves):
        qr, kr = api.tilelang_rotary_embedding(leaves[0], leaves[1], pos, freq)
        out = api.tilelang_shared_prefix_attention(qr, kr, *leaves[2:], is_causal=True, use_atomic_backward=False)
        return [out.detach(), *torch.autograd.grad(out, leaves, do)]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(static)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = step(static)
    for i in range(3):
        with torch.no_grad():
            for x in static:
                x.mul_(0.95)
        g.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in outs]
        want = step([x.detach().clone().requires_grad_(True) for x in static])
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b), i
