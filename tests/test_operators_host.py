"""The stand-alone operators' refusals, without a GPU: every call below must end in an error message before any launch."""
import ctypes as C

import pytest
import torch

import cora_amd as ca
from cora_amd import _lib

FAKE = 1 << 20       # an aligned address that is never read: the arguments are refused first


def _err():
    return _lib.load().cora_last_error(None).decode()


def rotary_args(**kw):
    a = dict(dtype=0, heads=2, head_dim=64, n_axes=3, axes_dim=(C.c_int32 * 4)(16, 16, 16, 0), interleaved=1, backward=0,
             theta=1e4, rows=8, pos_rows=8, pos=FAKE, x=FAKE, y=2 * FAKE, x_row=128, x_head=64, y_row=128, y_head=64)
    a.update(kw)
    return _lib.CoraRotaryArgs(**a)


@pytest.mark.parametrize("kw,word", [
    (dict(dtype=3), "dtype"), (dict(dtype=-1), "dtype"), (dict(heads=0), "heads"), (dict(head_dim=1), "head_dim"),
    (dict(n_axes=0), "n_axes"), (dict(n_axes=5), "n_axes"), (dict(axes_dim=(C.c_int32 * 4)(16, 15, 16, 0)), "axes_dim"),
    (dict(axes_dim=(C.c_int32 * 4)(16, 0, 16, 0)), "axes_dim"), (dict(axes_dim=(C.c_int32 * 4)(32, 32, 16, 0)), "channels"),
    (dict(head_dim=256, axes_dim=(C.c_int32 * 4)(64, 64, 32, 0)), "channels"), (dict(theta=0.0), "theta"),
    (dict(theta=float("inf")), "theta"), (dict(theta=float("nan")), "theta"), (dict(rows=-1), "rows"), (dict(pos_rows=0), "rows"),
    (dict(x=None), "NULL"), (dict(pos=None), "NULL"), (dict(x=FAKE + 2), "aligned"), (dict(x_row=-128), "negative"),
    (dict(y_row=64), "overlap"), (dict(y_head=32), "overlap"), (dict(y_row=0), "overlap"),
    (dict(y=FAKE, y_row=256), "in place"), (dict(rows=1 << 40), "rows"),
])
def test_rotary_refuses(kw, word):
    assert _lib.load().cora_rotary(C.byref(rotary_args(**kw)), 0, None) == -1
    assert word in _err() and "cora_rotary" in _err()


def test_no_rows_is_no_work():
    lib = _lib.load()
    assert lib.cora_rotary(C.byref(rotary_args(rows=0, x=None, y=None)), 0, None) == 0
    assert lib.cora_attention(C.byref(attn_args(rows=0, q=None)), 0, None) == 0
    assert lib.cora_attention(C.byref(attn_args(n_seq=0, q=None)), 0, None) == 0
    assert lib.cora_orthogonalize(0, None, 0, 5, coef(), 1e-7, None, 0, 0, None) == 0


def attn_args(**kw):
    a = dict(dtype=1, heads=4, kv_heads=2, head_dim=64, n_seq=2, seq_len=0, causal_block=1, scale=0.125, rows=100,
             cu_seqlens=FAKE, lse=FAKE, workspace=FAKE, workspace_bytes=1 << 20)
    for n, h in (("q", 4), ("k", 2), ("v", 2), ("out", 4), ("dout", 4), ("dq", 4), ("dk", 2), ("dv", 2)):
        a[n], a[n + "_row"], a[n + "_head"] = FAKE, 64 * h, 64
    a.update(kw)
    return _lib.CoraAttentionArgs(**a)


@pytest.mark.parametrize("kw,word", [
    (dict(dtype=7), "dtype"), (dict(heads=3), "multiple"), (dict(kv_heads=0), "multiple"), (dict(head_dim=0), "head_dim"),
    (dict(head_dim=20), "head_dim"), (dict(head_dim=136), "head_dim"), (dict(dtype=0, head_dim=6), "head_dim"),
    (dict(rows=-1), "rows"), (dict(rows=1 << 31), "rows"), (dict(n_seq=-1), "n_seq"), (dict(causal_block=-1), "causal_block"),
    (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"),
    (dict(cu_seqlens=None, seq_len=51), "seq_len"), (dict(cu_seqlens=None, seq_len=0), "seq_len"), (dict(q=None), "q is NULL"),
    (dict(k=FAKE + 8), "k must be 16-byte"), (dict(v_row=130), "v must be"), (dict(q_head=-64), "q must be"),
    (dict(k_row=1 << 24), "row stride"), (dict(out_row=128), "overlap"), (dict(out_head=0), "overlap"), (dict(lse=None), "lse"), (dict(cu_seqlens=FAKE + 2), "aligned"),
])
def test_attention_refuses(kw, word):
    lib = _lib.load()
    assert lib.cora_attention(C.byref(attn_args(**kw)), 0, None) == -1 and word in _err()
    if "overlap" not in word:       # the backward call reads out, it may have any strides there
        assert lib.cora_attention_backward(C.byref(attn_args(**kw)), 0, None) == -1 and word in _err()


@pytest.mark.parametrize("kw,word", [
    (dict(dout=None), "dout is NULL"), (dict(dq=None), "dq is NULL"), (dict(dk_row=64), "overlap"), (dict(dv_head=32), "overlap"),
    (dict(workspace=None), "workspace"), (dict(workspace=FAKE + 4), "workspace"), (dict(workspace_bytes=100), "workspace"),
])
def test_attention_backward_refuses(kw, word):
    assert _lib.load().cora_attention_backward(C.byref(attn_args(**kw)), 0, None) == -1 and word in _err()


def test_attention_refuses_outputs_that_are_inputs_and_launches_too_large():
    lib = _lib.load()
    apart = {n: FAKE * (i + 1) for i, n in enumerate(("q", "k", "v", "out", "dout", "dq", "dk", "dv", "workspace", "lse"))}
    for name, other in (("out", "q"), ("out", "k"), ("out", "v")):
        assert lib.cora_attention(C.byref(attn_args(**{**apart, name: apart[other]})), 0, None) == -1 and f"{name} is {other}" in _err()
    for name, other in (("dq", "q"), ("dk", "dout"), ("dv", "dk"), ("dk", "dv"), ("dq", "out")):
        a = attn_args(**{**apart, name: apart[other]})
        assert lib.cora_attention_backward(C.byref(a), 0, None) == -1 and " is " in _err()
    for kw in (dict(rows=1 << 30), dict(n_seq=1 << 22), dict(cu_seqlens=None, n_seq=1 << 22, seq_len=1, rows=1 << 22)):
        assert lib.cora_attention(C.byref(attn_args(**{**apart, **kw})), 0, None) == -1 and "too many tiles" in _err()


def test_orthogonalize_refuses_stacks_that_share_memory():
    lib = _lib.load()
    row = dict(x_mat=64, x_row=8, y_mat=64, y_row=8, count=1, rows=8, cols=8)
    for y0, y1 in ((3, 3), (2, 4), (4, 1), (3, 1)):
        s = (_lib.CoraMatrices * 2)(_lib.CoraMatrices(x=FAKE, y=y0 * FAKE, **row), _lib.CoraMatrices(x=2 * FAKE, y=y1 * FAKE, **row))
        assert lib.cora_orthogonalize(0, s, 2, 5, coef(), 1e-7, FAKE, 1 << 20, 0, None) == -1 and "is x or y of stack" in _err()
    big = (_lib.CoraMatrices * 1)(_lib.CoraMatrices(x=FAKE, y=FAKE, **{**row, "rows": 32768, "cols": 32768, "count": 16, "x_row": 32768, "y_row": 32768,
                                                                       "x_mat": 1 << 30, "y_mat": 1 << 30}))
    assert lib.cora_orthogonalize(0, big, 1, 5, coef(), 1e-7, FAKE, 1 << 20, 0, None) == -1 and "too many tiles" in _err()


def coef(*c):
    c = c or (3.4445, -4.775, 2.0315) * 5
    return (C.c_float * len(c))(*c)


def stack(**kw):
    a = dict(x=FAKE, y=2 * FAKE, x_mat=64 * 128, x_row=128, y_mat=64 * 128, y_row=128, count=2, rows=64, cols=128)
    a.update(kw)
    return (_lib.CoraMatrices * 1)(_lib.CoraMatrices(**a))


@pytest.mark.parametrize("kw,word", [
    (dict(count=-1), "count"), (dict(rows=0), "rows"), (dict(cols=40000), "cols"), (dict(count=65535, rows=32768, cols=32768), "tiles"),
    (dict(x=None), "NULL"), (dict(y=FAKE + 2), "aligned"), (dict(x_row=-1), "negative"), (dict(y_row=64), "overlap"),
    (dict(y_mat=64), "overlap"), (dict(y=FAKE, y_row=256, y_mat=64 * 256), "in place"),
])
def test_orthogonalize_refuses_stacks(kw, word):
    assert _lib.load().cora_orthogonalize(0, stack(**kw), 1, 5, coef(), 1e-7, FAKE, 1 << 40, 0, None) == -1
    assert word in _err()


@pytest.mark.parametrize("dtype,steps,c,eps,ws,word", [
    (4, 5, coef(), 1e-7, 1 << 40, "dtype"), (0, 0, coef(), 1e-7, 1 << 40, "steps"), (0, 33, coef(), 1e-7, 1 << 40, "steps"),
    (0, 5, None, 1e-7, 1 << 40, "coef"), (0, 5, coef(), -1.0, 1 << 40, "eps"), (0, 5, coef(), float("nan"), 1 << 40, "eps"),
    (0, 5, coef(), 1e-7, 1000, "workspace"), (0, 1, coef(9.0, 0.0, 0.0), 1e-7, 1 << 40, "out of range"),
    (0, 3, coef(*(3.0, 0.0, 0.0) * 3), 1e-7, 1 << 40, "out of range"), (0, 1, coef(float("nan"), 0.0, 0.0), 1e-7, 1 << 40, "out of range"),
])
def test_orthogonalize_refuses(dtype, steps, c, eps, ws, word):
    assert _lib.load().cora_orthogonalize(dtype, stack(), 1, steps, c, eps, FAKE, ws, 0, None) == -1
    assert word in _err()


def test_python_refuses_cpu_tensors_and_wrong_types():
    x = torch.zeros(4, 2, 16)
    with pytest.raises(ValueError, match="GPU"):
        ca.rotary(x, torch.zeros(4, 1, dtype=torch.int32), [16])
    with pytest.raises(ValueError, match="GPU"):
        ca.attention(x, x, x)
    with pytest.raises(ValueError, match="GPU"):
        ca.orthogonalize(torch.zeros(4, 4))
    with pytest.raises(TypeError):
        ca.orthogonalize([[1.0]])
    with pytest.raises(ValueError, match="steps"):
        ca.orthogonalize(torch.zeros(4, 4), steps=0)
    with pytest.raises(ValueError, match="triple"):
        ca.orthogonalize(torch.zeros(4, 4), steps=2, coefficients=[(1.0, 0.0, 0.0)] * 3)
