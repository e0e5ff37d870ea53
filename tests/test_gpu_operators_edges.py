"""Calls of the stand-alone operators that their documentation allows at its edges: repeated and overlapping rows, gradients of
very different sizes, values that are not finite, long sequences, launches of every tile size."""
import pytest
import torch

import cora_amd as ca
from tests.operator_bounds import attention_ref
from tests.test_gpu_operators import BF16, F16, F32, packed, randn, split, within

pytestmark = pytest.mark.gpu


def table(cu):
    return torch.tensor(cu, dtype=torch.int32, device="cuda")


def overlapping(rows, heads, d, step, dtype, seed):
    """rows that start `step` elements apart, less than they are long (0: one row, repeated)"""
    flat = randn(heads * ((rows - 1) * step + d), dtype=dtype, seed=seed)
    return flat.as_strided((rows, heads, d), (step, (rows - 1) * step + d, 1)), flat


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("lens", [[1], [33], [196], [1, 70, 31]])
@pytest.mark.parametrize("step", [0, 8])
@pytest.mark.parametrize("block", [0, 1, 20])
def test_attention_rows_that_repeat_or_overlap(lens, step, block, dtype):
    """The gradient of a sum over rows is one row, repeated; sliding windows overlap.  No row behind a sequence counts."""
    heads, d = 2, 32
    cu, qkv, dout = packed(lens, 0, heads, heads, d, dtype)
    rows = cu[-1]
    plain = dict(zip("qkv", split(qkv, heads, heads)), dout=dout)
    kw = dict(cu_seqlens=table(cu), causal_block=block)
    for names in (["dout"], ["q"], ["k"], ["v"], ["q", "k", "v", "dout"]):
        cpu, gpu = dict(plain), {n: t.cuda() for n, t in plain.items()}
        for i, n in enumerate(names):
            cpu[n], flat = overlapping(rows, heads, d, step, dtype, 50 + i)
            gpu[n] = flat.cuda().as_strided(cpu[n].shape, cpu[n].stride())
        ref, bound = attention_ref(cpu["q"], cpu["k"], cpu["v"], cu, block, d ** -0.5, cpu["dout"])
        out, lse = ca.attention(gpu["q"], gpu["k"], gpu["v"], **kw)
        within(out, ref["out"], bound["out"], (names, "out"))
        within(lse, ref["lse"], bound["lse"], (names, "lse"))
        for n, t in zip(("dq", "dk", "dv"), ca.attention_backward(gpu["dout"], gpu["q"], gpu["k"], gpu["v"], out, lse, **kw)):
            within(t, ref[n], bound[n], (names, n))
