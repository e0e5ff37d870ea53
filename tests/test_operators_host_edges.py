"""Refusals of the stand-alone operators at the edges of their ranges, without a GPU: every call must end in its own error message
before a device is looked for."""
import ctypes as C

import pytest

from cora_amd import _lib
from tests.test_operators_host import FAKE, attn_args, coef, rotary_args, stack


def refused(call, word):
    assert call == -1
    err = _lib.load().cora_last_error(None).decode()
    assert word in err, err


APART = {n: FAKE * (i + 1) for i, n in enumerate(("q", "k", "v", "out", "dout", "dq", "dk", "dv", "workspace", "lse", "cu_seqlens"))}


@pytest.mark.parametrize("rows", [2 ** 31 - 1, 2 ** 31 - 127, 2 ** 31 - 128])
def test_attention_refuses_a_sequence_whose_tiles_overflow(rows):
    """seq_len + 127 passes 32 bits"""
    a = attn_args(**{**APART, "cu_seqlens": None}, heads=1, kv_heads=1, n_seq=1, seq_len=rows, rows=rows)
    refused(_lib.load().cora_attention(C.byref(a), 0, None), "too many tiles")


BASE = 1 << 30


def packed_args(rows=100, h=4, kv=2, d=64, **kw):
    """q, k, v of one packed projection (bf16), the other tensors apart"""
    a = {n: BASE * (2 + i) for i, n in enumerate(("out", "dout", "dq", "dk", "dv", "workspace", "lse", "cu_seqlens"))}
    row = (h + 2 * kv) * d
    a.update(q=BASE, k=BASE + 2 * h * d, v=BASE + 2 * (h + kv) * d, q_row=row, k_row=row, v_row=row, rows=rows)
    return attn_args(**{**a, **kw})


@pytest.mark.parametrize("kw,word", [
    (dict(out=BASE + 2 * 512, out_row=512), "out overlaps"),                             # one row behind q, the rows' stride
    (dict(out=BASE + 64 * 2, out_row=512), "out overlaps q"),                            # one head behind
    (dict(out=BASE + 16, out_row=512), "out overlaps q"),                                # eight channels behind
    (dict(out=BASE + 99 * 1024 + 16, out_row=512), "out overlaps"),                      # only the last row
    (dict(lse=BASE + 1024), "lse"), (dict(out=BASE * 8 - 4), "must be 16-byte"), (dict(out=BASE * 8 - 64, out_row=256), "out overlaps lse"),
    (dict(out=BASE * 9 - 1024, out_row=256), "out overlaps cu_seqlens"), (dict(lse=BASE * 9 - 4), "lse overlaps cu_seqlens"),
])
def test_attention_refuses_overlapping_outputs(kw, word):
    refused(_lib.load().cora_attention(C.byref(packed_args(**kw)), 0, None), word)


@pytest.mark.parametrize("kw,word", [
    (dict(dq=BASE + 1024 + 32, dq_row=512), "dq overlaps"), (dict(dk=BASE * 4 + 512, dk_row=256), "dq overlaps dk"), (dict(dv=BASE * 5 + 128 * 50), "overlaps"),
    (dict(dq=BASE * 2 + 64, dq_row=256), "dq overlaps out"), (dict(dq=BASE * 3 - 64, dq_row=256), "dq overlaps dout"),
    (dict(dv=BASE * 7 - 64), "dv overlaps workspace"), (dict(workspace=BASE + 64), "overlaps workspace"), (dict(dk=BASE * 8 - 64), "dk overlaps lse"),
    (dict(workspace=BASE * 8 - 64), "workspace overlaps lse"),
])
def test_attention_backward_refuses_overlapping_outputs(kw, word):
    refused(_lib.load().cora_attention_backward(C.byref(packed_args(workspace_bytes=1 << 20, **kw)), 0, None), word)


@pytest.mark.parametrize("kw", [
    dict(), dict(out=BASE + 1024, q_row=1024, k_row=1024, v_row=1024, out_row=1024),                # a fourth part of every row
    dict(out=BASE + 100 * 1024, out_row=256), dict(out=BASE - 100 * 512, out_row=256),              # right behind and right before
    dict(out=BASE + 512, q_row=256 * 3, out_row=256 * 3, k=BASE * 20, v=BASE * 21),                 # interleaved rows
    dict(q=BASE, q_row=64, q_head=64 * 100, out=BASE + 4 * 100 * 128, out_row=64, out_head=6400, k=BASE * 20, v=BASE * 21),    # head-major
    dict(q=BASE, q_row=64, q_head=64 * 300, out=BASE + 100 * 128, out_row=64, out_head=64 * 300, k=BASE * 20, v=BASE * 21),    # heads in turn
    dict(q=BASE, q_row=0, q_head=64, out=BASE + 512, out_row=256, k=BASE * 20, v=BASE * 21),        # one row, repeated
])
def test_views_of_one_buffer_that_do_not_overlap_are_taken(kw):
    """nothing but the missing device stops them"""
    import torch
    if torch.cuda.is_available():
        pytest.skip("addresses that must not be read")
    refused(_lib.load().cora_attention(C.byref(packed_args(**kw)), 0, None), "not available")


@pytest.mark.parametrize("kw,word", [
    (dict(x=BASE, y=BASE + 64), "y overlaps x"), (dict(x=BASE, y=BASE + 512), "y overlaps x"), (dict(x=BASE, y=BASE - 7 * 512 - 4), "y overlaps x"),
    (dict(x=BASE, y=BASE + 256, y_row=192, x_row=128), "y overlaps x"), (dict(pos=BASE + 100, y=BASE), "y overlaps pos"),
])
def test_rotary_refuses_overlapping_outputs(kw, word):
    refused(_lib.load().cora_rotary(C.byref(rotary_args(**kw)), 0, None), word)


def test_orthogonalize_refuses_overlapping_outputs():
    lib = _lib.load()
    row = dict(x_mat=64 * 256, x_row=256, y_mat=64 * 256, y_row=256, count=2, rows=64, cols=128)
    two = lambda a, b: (_lib.CoraMatrices * 2)(_lib.CoraMatrices(**{**row, **a}), _lib.CoraMatrices(**{**row, **b}))
    call = lambda s, n=2, ws=BASE * 50: lib.cora_orthogonalize(0, s, n, 5, coef(), 1e-7, ws, 1 << 40, 0, None)
    far = dict(x=BASE * 10, y=BASE * 11)
    refused(call(two(dict(x=BASE, y=BASE + 64), far)), "y of stack 0 overlaps x of stack 0")                 # columns 16 .. 143
    refused(call(two(dict(x=BASE, y=BASE + 1024), far)), "y of stack 0 overlaps x of stack 0")               # one row down
    refused(call(two(far, dict(x=BASE, y=BASE * 10 + 64 * 1024 + 4))), "y of stack 1 overlaps x of stack 0")
    refused(call(two(far, dict(x=BASE, y=BASE * 11 - 8))), "y of stack 0 overlaps y of stack 1")
    refused(call(two(far, dict(x=BASE, y=BASE * 2)), 2, BASE * 2 - 256), "workspace overlaps stack 1")
    import torch
    if not torch.cuda.is_available():
        refused(call(two(dict(x=BASE, y=BASE + 512), far)), "not available")                                 # the other half of every row
        refused(call(two(dict(x=BASE, y=BASE), far)), "not available")


def test_orthogonalize_refuses_coefficients_whose_products_leave_fp16():
    """b A + c A^2 is kept apart from a I for bfloat16 results and may be larger than their sum: 2000 in the second step here, where
    the planes, 64 times the value, hold 1023."""
    s = stack()
    refused(_lib.load().cora_orthogonalize(1, s, 1, 2, coef(0.001, 0.0, 0.0, 999.0, -1.99e9, 0.0), 1e-7, FAKE * 100, 1 << 40, 0, None), "out of range")
