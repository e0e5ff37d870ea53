"""Refusals of the stand-alone operators at the edges of their ranges, without a GPU: every call must end in its own error message
before a device is looked for."""
import ctypes as C

import pytest

from cora_amd import _lib
from tests.test_operators_host import FAKE, attn_args


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
