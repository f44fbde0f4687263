"""The cache operators without a GPU: refusals of the Python entry points and of the C ABI
(every check runs before any HIP call), plans, struct layouts, fake implementations."""

import ctypes
import math
import shutil
import subprocess
from pathlib import Path

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import tilelang_fa2_4d_mask as api
from tilelang_fa2_4d_mask import _ext

HEADER = Path(__file__).resolve().parents[1] / "include" / "fa2_4d_mask.h"
FAKE = 0x100000   # 16-byte aligned, never dereferenced: validation fails first
BF = torch.bfloat16


@pytest.fixture(scope="module")
def lib():
    return _ext.load_library()


# ---- the Python entry points ----------------------------------------------------------


def _t(*shape, dtype=BF):
    return torch.zeros(shape, dtype=dtype)


def _attention_args(**over):
    a = dict(query=_t(2, 8, 3, 64), key=_t(2, 2, 5, 64), value=_t(2, 2, 5, 64), prefix_key=_t(1, 2, 7, 64),
             prefix_value=_t(1, 2, 7, 64))
    a.update(over)
    return a


ATTENTION_REFUSALS = [
    (dict(query=_t(8, 3, 64)), "rank-4"),
    (dict(layout="bsd"), "unsupported layout"),
    (dict(key=_t(3, 2, 5, 64), value=_t(3, 2, 5, 64)), "same batch size"),
    (dict(value=_t(2, 2, 6, 64)), "same sequence length"),
    (dict(value=_t(2, 4, 5, 64)), "same number of heads"),
    (dict(value=_t(2, 2, 5, 32)), "same head dimension"),
    (dict(key=_t(2, 3, 5, 64), value=_t(2, 3, 5, 64)), "divisible"),
    (dict(key=_t(2, 0, 5, 64), value=_t(2, 0, 5, 64)), "at least one head"),
    (dict(query=_t(2, 8, 3, 0), key=_t(2, 2, 5, 0), value=_t(2, 2, 5, 0)), "one column"),
    (dict(query=_t(2, 8, 3, 272), key=_t(2, 2, 5, 272), value=_t(2, 2, 5, 272)), "272 is not supported"),
    (dict(query=_t(2, 8, 3, 64, dtype=torch.float32)), "fp16 or bf16"),
    (dict(key=_t(2, 2, 5, 64, dtype=torch.float16)), "same dtype"),
    (dict(prefix_key=_t(2, 7, 64)), "rank-4 tensor of batch size 1"),
    (dict(prefix_key=_t(2, 2, 7, 64), prefix_value=_t(2, 2, 7, 64)), "batch size 1"),
    (dict(prefix_key=_t(1, 4, 7, 64)), "heads"),
    (dict(prefix_value=_t(1, 2, 7, 32)), "head dimension"),
    (dict(prefix_value=_t(1, 2, 8, 64)), "same sequence length"),
    (dict(prefix_value=_t(1, 2, 7, 64, dtype=torch.float16)), "same dtype"),
    (dict(mask=_t(2, 1, 3, 5)), "bool"),
    (dict(mask=_t(2, 1, 3, 12, dtype=torch.bool)), "trailing shape"),
    (dict(mask=_t(3, 1, 3, 5, dtype=torch.bool)), "batch dimension"),
    (dict(mask=_t(2, 2, 3, 5, dtype=torch.bool)), "head dimension"),
    (dict(score=_t(2, 1, 3, 5, dtype=torch.int32)), "floating-point"),
    (dict(score=_t(2, 1, 5, dtype=torch.float32)), "must have shape"),
    (dict(lengths=_t(2, dtype=torch.float32)), "lengths"),
    (dict(lengths=_t(3, dtype=torch.int32)), "lengths"),
    (dict(lengths=_t(2, 1, dtype=torch.int64)), "lengths"),
    (dict(), "HIP/CUDA"),
]


@pytest.mark.parametrize("over,text", ATTENTION_REFUSALS, ids=lambda x: x if isinstance(x, str) else ",".join(x))
def test_attention_refusals(over, text):
    a = _attention_args(**over)
    args = [a.pop(n) for n in ("query", "key", "value", "prefix_key", "prefix_value")]
    with pytest.raises(ValueError, match=text):
        api.tilelang_shared_prefix_attention(*args, **a)
    a = _attention_args(**over)
    args = [a.pop(n) for n in ("query", "key", "value")]
    with pytest.raises(ValueError, match=text):
        api.tilelang_attention_with_key_weights(*args, **a)


def test_key_weights_refusals():
    a = _attention_args()
    args = [a[n] for n in ("query", "key", "value")]
    with pytest.raises(ValueError, match="together"):
        api.tilelang_attention_with_key_weights(*args, prefix_key=a["prefix_key"])
    for bad in (_t(2, 2, 5), _t(2, 8, 5, dtype=torch.float32), _t(2, 2, 6, dtype=torch.float32)):
        with pytest.raises(ValueError, match="key_weights"):
            api.tilelang_attention_with_key_weights(*args, key_weights=bad)


def test_evict_refusals():
    k, w = _t(2, 3, 20, 64), _t(2, 3, 20, dtype=torch.float32)
    call = api.tilelang_evict_keys
    for over, text in (
        (dict(key=_t(3, 20, 64)), "rank-4"),
        (dict(layout="x"), "unsupported layout"),
        (dict(value=_t(2, 3, 19, 64)), "same shape"),
        (dict(key=_t(2, 3, 20, 64, dtype=torch.float32)), "fp16 or bf16"),
        (dict(value=_t(2, 3, 20, 64, dtype=torch.float16)), "same dtype"),
        (dict(key=_t(2, 3, 20, 0), value=_t(2, 3, 20, 0)), "head dimension"),
        (dict(key=_t(2, 3, 20, 264), value=_t(2, 3, 20, 264)), "264 is not supported"),
        (dict(keep=0), "keep"), (dict(keep=21), "keep"), (dict(recent=-1), "recent"), (dict(recent=11), "recent"),
        (dict(key_weights=_t(2, 3, 20)), "key_weights"),
        (dict(key_weights=_t(2, 20, 3, dtype=torch.float32)), "key_weights"),
        (dict(lengths=_t(3, dtype=torch.int32)), "lengths"),
        (dict(), "HIP/CUDA"),
    ):
        a = dict(key=k, value=k, key_weights=w, keep=10, recent=5)
        a.update(over)
        with pytest.raises(ValueError, match=text):
            call(a.pop("key"), a.pop("value"), a.pop("key_weights"), **a)


def test_rotary_refusals():
    q, k, pos, freq = _t(2, 8, 5, 64), _t(2, 2, 5, 64), _t(1, 2, 5, dtype=torch.int64), _t(32, dtype=torch.float32)
    for over, text in (
        (dict(query=_t(8, 5, 64)), "rank-4"),
        (dict(layout="x"), "unsupported layout"),
        (dict(key=_t(2, 2, 6, 64)), "same batch size"),
        (dict(key=_t(2, 2, 5, 32)), "same batch size"),
        (dict(query=_t(2, 0, 5, 64)), "at least one head"),
        (dict(key=_t(2, 0, 5, 64)), "at least one head"),
        (dict(query=_t(2, 8, 5, 258), key=_t(2, 2, 5, 258)), "not supported"),
        (dict(query=_t(2, 8, 5, 64, dtype=torch.float32)), "fp16 or bf16"),
        (dict(key=_t(2, 2, 5, 64, dtype=torch.float16)), "same dtype"),
        (dict(inv_freq=_t(32)), "float32 vector"),
        (dict(inv_freq=_t(1, 32, dtype=torch.float32)), "float32 vector"),
        (dict(inv_freq=_t(33, dtype=torch.float32)), "1 to 32"),
        (dict(inv_freq=_t(0, dtype=torch.float32)), "1 to 32"),
        (dict(sections=(16, 8)), "add up"), (dict(sections=(33, -1)), "add up"), (dict(sections=()), "add up"),
        (dict(sections=(4,) * 9), "add up"),
        (dict(positions=_t(1, 2, 5, dtype=torch.float32)), "int32 or int64"),
        (dict(positions=_t(2, 5, dtype=torch.int64)), "int32 or int64"),
        (dict(positions=_t(2, 2, 5, dtype=torch.int64)), "positions has shape"),
        (dict(positions=_t(1, 3, 5, dtype=torch.int64)), "positions has shape"),
        (dict(positions=_t(1, 2, 6, dtype=torch.int64)), "positions has shape"),
        (dict(), "HIP/CUDA"),
    ):
        a = dict(query=q, key=k, positions=pos, inv_freq=freq)
        a.update(over)
        with pytest.raises(ValueError, match=text):
            api.tilelang_rotary_embedding(**a)


def test_what_has_no_gradient_is_refused():
    with FakeTensorMode():
        g = lambda *s: torch.empty(s, dtype=BF, device="cuda", requires_grad=True)  # noqa: E731
        w = torch.empty((2, 3, 20), device="cuda")
        with pytest.raises(ValueError, match="no gradient"):
            api.tilelang_evict_keys(g(2, 3, 20, 64), g(2, 3, 20, 64), w, keep=10)
        with pytest.raises(ValueError, match="no gradient"):
            api.tilelang_attention_with_key_weights(g(2, 6, 1, 64), g(2, 3, 20, 64), g(2, 3, 20, 64), key_weights=w)
        with pytest.raises(ValueError, match="no gradient"):
            api.tilelang_rotary_embedding(g(2, 6, 1, 64), g(2, 3, 1, 64), torch.empty((1, 2, 1), dtype=torch.int64, device="cuda"),
                                          torch.empty(32, device="cuda", requires_grad=True))


@pytest.mark.parametrize("layout", ["bhsd", "bshd"])
@pytest.mark.parametrize("Tp,Tk", [(30, 20), (0, 20), (30, 0), (0, 0)])
def test_fake_implementations(layout, Tp, Tk):
    """Shapes, types and strides of traced calls."""
    B, Hq, Hk, Tq, D = 2, 8, 2, 5, 64
    bhsd = layout == "bhsd"

    def x(b, h, t):
        return torch.empty((b, h, t, D) if bhsd else (b, t, h, D), dtype=BF, device="cuda")

    with FakeTensorMode():
        q, k, pk = x(B, Hq, Tq), x(B, Hk, Tk), x(1, Hk, Tp)
        o = api.tilelang_shared_prefix_attention(q, k, k, pk, pk, layout=layout)
        assert o.shape == q.shape and o.dtype == BF
        assert o.stride() == ((Tq * Hq * D, D, Hq * D, 1) if bhsd else (Tq * Hq * D, Hq * D, D, 1))
        o, w = api.tilelang_attention_with_key_weights(q, k, k, prefix_key=pk, prefix_value=pk, layout=layout)
        assert o.shape == q.shape and w.shape == (B, Hk, Tk) and w.dtype == torch.float32
        if Tk:
            r = api.tilelang_evict_keys(k, k, w, keep=7, recent=2, layout=layout)
            assert r[0].shape == x(B, Hk, 7).shape == r[1].shape and r[2].shape == (B, Hk, 7) == r[3].shape
            assert r[3].dtype == torch.int64 and r[0].is_contiguous()
        # (the backward ops themselves: autograd's engine asks for a device)
        ns = torch.ops.tilelang_fa2_4d_mask
        o, lse, lo = ns.prefix_fwd(q, k, k, pk, pk, None, None, None, 0.1, True, False, True, bhsd)
        assert lse.shape == (B, Hq, Tq) and (lo.shape == q.shape if Tp + Tk else lo.numel() == 0)
        grads = ns.prefix_bwd(o, q, k, k, pk, pk, None, None, None, o, lse, lo, 0.1, True, False, bhsd)
        for y, g in zip((q, k, k, pk, pk), grads):
            assert g.shape == y.shape or (g.shape == (0,) and y.numel() == 0)
        kr = x(B, Hk, Tq)
        pos, freq = torch.empty((3, 1, Tq), dtype=torch.int32, device="cuda"), torch.empty(32, device="cuda")
        yq, yk = api.tilelang_rotary_embedding(q, kr, pos, freq, sections=(8, 12, 12), layout=layout)
        assert yq.shape == q.shape and yk.shape == kr.shape and yq.stride() == o.stride()


# ---- the C ABI ------------------------------------------------------------------------


def test_struct_layouts_match_the_header(tmp_path):
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("gcc not available")
    pairs = [(n, getattr(_ext, n)) for n in ("FaPrefixParams", "FaPrefixPlan", "FaKeyWeightsParams", "FaEvictParams",
                                              "FaRotaryParams", "FaBwdParams")]
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void) {"]
    for cname, cls in pairs:
        lines.append(f'printf("{cname} size %zu\\n", sizeof({cname}));')
        lines += [f'printf("{cname} {f} %zu\\n", offsetof({cname}, {f}));' for f, _ in cls._fields_]
    lines += [f'if (FA_ROTARY_AXES != {_ext.ROTARY_AXES} || FA_DQ_KEEP != {_ext.FA_DQ_KEEP} || FA_DQ_ADD != {_ext.FA_DQ_ADD}) return 1;',
              "return 0;", "}"]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines))
    subprocess.run([gcc, "-std=c99", str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout
    got = {tuple(x.split()[:2]): int(x.split()[2]) for x in out.splitlines()}
    for cname, cls in pairs:
        assert got[(cname, "size")] == ctypes.sizeof(cls), cname
        for f, _ in cls._fields_:
            assert got[(cname, f)] == getattr(cls, f).offset, (cname, f)


def _set(p, **kw):
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def prefix_params(**over):
    p = _ext.FaPrefixParams()
    for n in ("q", "pk", "pv", "k", "v", "o", "lse", "workspace"):
        setattr(p, n, FAKE)
    B, Tq, Tp, Tk, Hq, Hk, D = 16, 1, 8192, 512, 32, 8, 128
    _set(p, batch=B, seqlen_q=Tq, seqlen_p=Tp, seqlen_k=Tk, heads_q=Hq, heads_k=Hk, head_dim=D, scale=0.1,
         q_stride_b=Tq * Hq * D, q_stride_t=Hq * D, q_stride_h=D, o_stride_b=Tq * Hq * D, o_stride_t=Hq * D, o_stride_h=D,
         pk_stride_t=Hk * D, pk_stride_h=D, pv_stride_t=Hk * D, pv_stride_h=D, workspace_bytes=1 << 40)
    for n in "kv":
        _set(p, **{f"{n}_stride_b": Tk * Hk * D, f"{n}_stride_t": Hk * D, f"{n}_stride_h": D})
    return _set(p, **over)


PREFIX_REFUSALS = [
    (dict(batch=0), 2), (dict(seqlen_q=0), 2), (dict(seqlen_p=-1), 2), (dict(seqlen_p=0, seqlen_k=0), 2),
    (dict(heads_q=30), 2), (dict(batch=1 << 20, seqlen_q=1 << 8), 2), (dict(seqlen_p=1 << 30), 2),
    (dict(head_dim=96), 3), (dict(head_dim_in=24), 3), (dict(dtype=2), 4), (dict(scale=math.nan), 6),
    (dict(q=None), 1), (dict(pk=None), 1), (dict(v=None), 1), (dict(lse=None), 1), (dict(o=FAKE + 8), 5),
    (dict(pv_stride_t=100), 5), (dict(k_stride_t=1 << 24), 5), (dict(pk_stride_t=-8), 5),
    (dict(mask=FAKE, mask_stride_q=-1), 5), (dict(score=FAKE, score_stride_h=-4), 5),
    (dict(kw_in=FAKE, kw_out=FAKE, kw_stride_b=-1), 5), (dict(o_lo=FAKE, o_lo_stride_t=4), 5),
    (dict(workspace=None), 8), (dict(workspace_bytes=100), 8), (dict(workspace=FAKE + 8), 5),
    (dict(seqlen_q=129, kw_out=FAKE), 2), (dict(seqlen_q=129, lengths=FAKE, score=FAKE), 2),
    (dict(seqlen_q=20, kw_out=FAKE), 2),                       # 80 rows of a group: the weights in a pass of their own
    (dict(seqlen_q=129, mask=FAKE), 8), (dict(seqlen_q=129, mask=FAKE, mask_ws=FAKE + 16), 5),
    (dict(seqlen_q=129, score=FAKE, score_stride_q=1 << 26), 5),
]


@pytest.mark.parametrize("over,code", PREFIX_REFUSALS, ids=lambda x: str(x) if isinstance(x, int) else ",".join(x))
def test_prefix_refusals(lib, over, code):
    assert lib.fa_prefix_fwd(ctypes.byref(prefix_params(**over))) == code
    assert lib.fa_last_error() != b"no error"


def test_prefix_plans(lib):
    plan = _ext.FaPrefixPlan()

    def of(**over):
        p = prefix_params(**over)
        assert lib.fa_prefix_plan(ctypes.byref(p), ctypes.byref(plan)) == 0
        return plan.few_rows, plan.prefix_split, plan.own_split, plan.needs_mask_ws, plan.workspace_bytes

    few, nsp, nso, ws, n = of()
    assert few == 1 and ws == 0 and 1 <= nsp <= 64 and 1 <= nso <= 64
    rows = 16 * 32
    assert n == rows * (nsp + nso) * (128 + 4) * 4
    assert of(kw_out=FAKE)[4] == n + rows * 512 * 4          # and the logits of the own keys
    few, nsp, nso, _, n = of(kw_out=FAKE, seqlen_k=513)      # whole tiles of 32 keys
    assert n == rows * ((nsp + nso) * (128 + 4) + 544) * 4
    assert of(seqlen_p=0)[1] == 0 and of(seqlen_k=0)[2] == 0
    assert of(seqlen_q=129)[0] == 0 and of(seqlen_q=129)[3] == 1
    assert of(seqlen_q=20, kw_out=FAKE)[0] == 0 and of(seqlen_q=20)[0] == 1
    assert of(seqlen_q=4096, head_dim=256)[0] == 1           # head dim 256 is always packed
    assert lib.fa_prefix_plan(None, ctypes.byref(plan)) == 1
    assert lib.fa_prefix_plan(ctypes.byref(prefix_params()), None) == 1
    # a long cache: every range is covered, the slots stay within what the join holds
    for Tp in (1, 31, 33, 100000, 4000000):
        few, nsp, nso, _, _ = of(batch=1, seqlen_p=Tp)
        assert few and 1 <= nsp <= 64


def key_weights_params(**over):
    p = _ext.FaKeyWeightsParams()
    for n in ("q", "k", "lse", "kw_out", "workspace"):
        setattr(p, n, FAKE)
    B, T, Hq, Hk, D = 1, 2048, 32, 8, 128
    _set(p, batch=B, seqlen_q=T, seqlen_k=T, heads_q=Hq, heads_k=Hk, head_dim=D, scale=0.1, q_stride_b=T * Hq * D,
         q_stride_t=Hq * D, q_stride_h=D, k_stride_b=T * Hk * D, k_stride_t=Hk * D, k_stride_h=D, workspace_bytes=1 << 40)
    return _set(p, **over)


@pytest.mark.parametrize("over,code", [
    (dict(seqlen_k=0), 2), (dict(heads_k=5), 2), (dict(head_dim=32), 3), (dict(dtype=-1), 4), (dict(scale=math.inf), 6),
    (dict(q=None), 1), (dict(lse=None), 1), (dict(kw_out=None), 1), (dict(k=FAKE + 2), 5), (dict(k_stride_t=1 << 25), 5),
    (dict(mask=FAKE, mask_stride_b=-1), 5), (dict(score=FAKE, score_stride_b=-1), 5), (dict(kw_in=FAKE, kw_stride_h=-1), 5),
    (dict(workspace=None), 8), (dict(workspace_bytes=8), 8), (dict(workspace=FAKE + 4), 5),
], ids=lambda x: str(x) if isinstance(x, int) else ",".join(x))
def test_key_weights_abi_refusals(lib, over, code):
    assert lib.fa_key_weights(ctypes.byref(key_weights_params(**over))) == code


def test_key_weights_plan(lib):
    n = ctypes.c_int64(-1)
    assert lib.fa_key_weights_plan(ctypes.byref(key_weights_params()), ctypes.byref(n)) == 0
    assert n.value > 0 and n.value % (8 * 2048 * 4) == 0      # whole parts of the sums
    assert lib.fa_key_weights_plan(ctypes.byref(key_weights_params(batch=64)), ctypes.byref(n)) == 0 and n.value == 0
    assert lib.fa_key_weights_plan(ctypes.byref(key_weights_params(batch=64, score=FAKE)), ctypes.byref(n)) == 0
    assert n.value == 64 * 32 * 2048 * 2 * 4
    assert lib.fa_key_weights_plan(ctypes.byref(key_weights_params()), None) == 1


def evict_params(**over):
    p = _ext.FaEvictParams()
    for n in ("k", "v", "kw", "k_out", "v_out", "kw_out", "index_out"):
        setattr(p, n, FAKE)
    _set(p, batch=2, seqlen_k=100, heads_k=4, head_dim=64, keep=50, recent=10, kw_stride_b=400, kw_stride_h=100)
    for n, T in (("k", 100), ("v", 100), ("out", 50)):
        _set(p, **{f"{n}_stride_b": T * 256, f"{n}_stride_t": 256, f"{n}_stride_h": 64})
    return _set(p, **over)


@pytest.mark.parametrize("over,code", [
    (dict(batch=0), 2), (dict(seqlen_k=0), 2), (dict(keep=0), 2), (dict(keep=101), 2), (dict(recent=51), 2), (dict(recent=-1), 2),
    (dict(batch=1 << 21), 2), (dict(head_dim=0), 2), (dict(kw=None), 1), (dict(index_out=None), 1),
    (dict(k_stride_t=-1), 5), (dict(kw_stride_b=-1), 5), (dict(out_stride_h=-64), 5),
], ids=lambda x: str(x) if isinstance(x, int) else ",".join(x))
def test_evict_abi_refusals(lib, over, code):
    assert lib.fa_evict(ctypes.byref(evict_params(**over))) == code


def rotary_params(**over):
    p = _ext.FaRotaryParams()
    for n in ("q", "k", "q_out", "k_out", "positions", "inv_freq"):
        setattr(p, n, FAKE)
    _set(p, batch=1, seqlen=16, heads_q=8, heads_k=2, head_dim=128, rotary=128, axes=3, sign=1)
    p.sections[0], p.sections[1], p.sections[2] = over.pop("sections", (16, 24, 24))
    return _set(p, **over)


@pytest.mark.parametrize("over,code", [
    (dict(batch=0), 2), (dict(seqlen=0), 2), (dict(heads_q=0), 2), (dict(head_dim=257), 2), (dict(batch=1 << 25), 2),
    (dict(heads_q=1 << 16), 2), (dict(rotary=0), 3), (dict(rotary=127), 3), (dict(rotary=130), 3), (dict(axes=0), 2),
    (dict(axes=9), 2), (dict(sections=(16, 24, 23)), 2), (dict(sections=(80, -8, -8)), 2), (dict(sign=0), 2), (dict(dtype=3), 4),
    (dict(q=None), 1), (dict(k_out=None), 1), (dict(positions=None), 1), (dict(inv_freq=None), 1),
], ids=lambda x: str(x) if isinstance(x, int) else ",".join(x))
def test_rotary_abi_refusals(lib, over, code):
    assert lib.fa_rotary(ctypes.byref(rotary_params(**over))) == code


def test_every_entry_refuses_no_parameters(lib):
    for n in ("fa_prefix_fwd", "fa_key_weights", "fa_evict", "fa_rotary"):
        assert getattr(lib, n)(None) == 1


def test_dq_modes_of_the_backward(lib):
    """Plans and refusals of a backward that sums dQ over key sets."""
    import test_abi

    plan = _ext.FaBwdPlan()
    for mode in (1, 2, 3):
        for atomic in (0, 1):
            p = test_abi.bwd_params(dq_mode=mode, atomic_dq=atomic)
            assert lib.fa_bwd_plan(ctypes.byref(p), ctypes.byref(plan)) == 0
            assert plan.needs_dq_accum == 1 and plan.dq_accum_elems == 8192 * 32 * 128
        for fn in (lib.fa_bwd_preprocess, lib.fa_bwd, lib.fa_bwd_finalize):
            assert fn(ctypes.byref(test_abi.bwd_params(dq_mode=mode, dq_accum=None))) == 8
            assert fn(ctypes.byref(test_abi.bwd_params(dq_mode=mode, dq_accum=FAKE + 4))) == 5
            assert fn(ctypes.byref(test_abi.bwd_params(dq_mode=mode, dq_accum_stride_h=6))) == 5
    for fn in (lib.fa_bwd_preprocess, lib.fa_bwd, lib.fa_bwd_finalize):
        assert fn(ctypes.byref(test_abi.bwd_params(dq_mode=4))) == 2
    # dS as tile pairs: twice the workspace
    assert lib.fa_bwd_plan(ctypes.byref(test_abi.bwd_params(seqlen_q=1024, seqlen_k=1024)), ctypes.byref(plan)) == 0
    one = plan.ds_elems
    assert lib.fa_bwd_plan(ctypes.byref(test_abi.bwd_params(seqlen_q=1024, seqlen_k=1024, dq_mode=1)), ctypes.byref(plan)) == 0
    assert plan.ds_elems == 2 * one


def test_sizes_whose_products_overflow(lib):
    """2^31 - 1 of everything is refused, not multiplied."""
    most = 2 ** 31 - 1
    plan, n = _ext.FaPrefixPlan(), ctypes.c_int64()
    big = dict(batch=most, heads_q=most, heads_k=most, seqlen_k=most)
    p = prefix_params(seqlen_q=most, seqlen_p=most, **big)
    assert lib.fa_prefix_plan(ctypes.byref(p), ctypes.byref(plan)) == 2
    assert lib.fa_key_weights_plan(ctypes.byref(key_weights_params(seqlen_q=most, **big)), ctypes.byref(n)) == 2
    assert lib.fa_evict(ctypes.byref(evict_params(batch=most, heads_k=most, seqlen_k=most, keep=most))) == 2
    assert lib.fa_rotary(ctypes.byref(rotary_params(batch=most, seqlen=most, heads_q=most, heads_k=most))) == 2


@pytest.mark.parametrize("over,few", [
    (dict(seqlen_q=128), 1), (dict(seqlen_q=129), 0), (dict(seqlen_q=64, seqlen_p=100), 1), (dict(seqlen_q=65, seqlen_p=100), 0),
    (dict(seqlen_q=4000, head_dim=256), 1), (dict(seqlen_q=4, kw_out=FAKE), 1), (dict(seqlen_q=5, kw_out=FAKE), 0),
    (dict(seqlen_q=5, heads_q=8, kw_out=FAKE), 1),
])
def test_prefix_plan_rows(lib, over, few):
    """Which calls run packed, and keep the logits that key weights need."""
    plan = _ext.FaPrefixPlan()
    assert lib.fa_prefix_plan(ctypes.byref(prefix_params(**over)), ctypes.byref(plan)) == 0
    assert plan.few_rows == few and 1 <= plan.prefix_split + plan.own_split <= 128
