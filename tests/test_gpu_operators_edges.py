"""Calls of the stand-alone operators that their documentation allows at its edges: repeated and overlapping rows, gradients of
very different sizes, values that are not finite, long sequences, launches of every tile size."""
import math

import pytest
import torch

import cora_amd as ca
from tests.operator_bounds import attention_ref, half_eps
from tests.test_gpu_operators import BF16, F16, F32, ortho_close, packed, randn, split, within

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


def by_key(q, k, v, cu, block, scale, dout):
    """attention_ref with the part of the fp16 gradients' bounds that belongs to small ds taken from what a key (dk) or a query (dq)
    itself sees, instead of the sequence's largest gradient: ds enters its products times a power of two that keeps the largest one
    of 32 at 2^-8 at least, where fp16 is off by 2^-25 absolutely: 2^-17 of the largest ds of the key or query."""
    ref, bound = attention_ref(q, k, v, cu, block, scale, dout)
    heads = q.shape[1]
    g, flat = heads // k.shape[1], 2.0 ** -24
    for b, e in zip(cu[:-1], cu[1:]):
        i = torch.arange(e - b)
        vis = i[None, :] // block <= i[:, None] // block if block else torch.ones(e - b, e - b, dtype=torch.bool)
        for h in range(heads):
            Q, K, V, G = q[b:e, h].double(), k[b:e, h // g].double(), v[b:e, h // g].double(), dout[b:e, h].double()
            p = torch.softmax(((Q @ K.T) * scale).masked_fill(~vis, -math.inf), 1)
            ds = (p * (G @ V.T - (G * (p @ V)).sum(1, keepdim=True))).abs()
            old = flat * G.abs().amax() * vis
            bound["dk"][b:e, h // g] += scale * (2.0 ** -17 * ds.amax(0)[:, None] * vis.T - old.T) @ Q.abs()
            bound["dq"][b:e, h] += scale * (2.0 ** -17 * ds.amax(1)[:, None] * vis - old) @ K.abs()
    return ref, bound


@pytest.mark.parametrize("lens,heads,kv,d,block", [([512], 2, 1, 64, 1), ([300, 97], 4, 2, 128, 1), ([700], 1, 1, 32, 50), ([200] * 40, 4, 4, 80, 1)])
@pytest.mark.parametrize("ratio", [2.0 ** 10, 2.0 ** 20])
def test_attention_fp16_dk_of_keys_that_large_gradients_do_not_see(lens, heads, kv, d, block, ratio):
    """The first token's gradient is far larger than the others'; keys that it does not see keep their precision."""
    cu, qkv, dout = packed(lens, 0, heads, kv, d, F16)
    dout = dout.float().clamp(-3, 3) * 8 / ratio
    dout[cu[:-1]] *= ratio
    dout = dout.to(F16)
    ref, bound = by_key(*split(qkv, heads, kv), cu, block, d ** -0.5, dout)
    q, k, v = split(qkv.cuda(), heads, kv)
    kw = dict(cu_seqlens=table(cu), causal_block=block)
    out, lse = ca.attention(q, k, v, **kw)
    dk = ca.attention_backward(dout.cuda(), q, k, v, out, lse, **kw)[1]
    hidden = torch.ones(cu[-1], dtype=torch.bool)
    for b in cu[:-1]:
        hidden[b:b + block] = False                       # the first token sees its own block
    within(dk[hidden.cuda()], ref["dk"][hidden], bound["dk"][hidden], "dk")
    assert bound["dk"][hidden].norm() < 0.1 * ref["dk"][hidden].norm()     # the bound would not let them be lost: reference values only
    within(dk, ref["dk"], bound["dk"], "all dk")


@pytest.mark.parametrize("lens,block", [([2] * 50, 0), ([2, 3, 200], 1), ([3000], 0)])
def test_attention_fp16_gradients_of_large_values(lens, block):
    """Large values, small gradients: their products fit fp16, the products with a gradient brought to 1 would not."""
    d = 128
    cu, qkv, dout = packed(lens, 0, 2, 2, d, F16)
    qkv[:, 4:] = (qkv[:, 4:].float() * 1.5e4).clamp(-6e4, 6e4).to(F16)
    dout = (dout.float() * 1e-3).to(F16)
    ref, bound = by_key(*split(qkv, 2, 2), cu, block, d ** -0.5, dout)
    q, k, v = split(qkv.cuda(), 2, 2)
    kw = dict(cu_seqlens=table(cu), causal_block=block)
    out, lse = ca.attention(q, k, v, **kw)
    for n, t in zip(("dq", "dk", "dv"), ca.attention_backward(dout.cuda(), q, k, v, out, lse, **kw)):
        assert ref[n].abs().max() < 6e4, n
        within(t, ref[n], bound[n], n)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n,heads", [(33, 1), (97, 2), (1025, 1), (600, 64)])
def test_attention_lse_of_rows_that_see_nan(n, heads, dtype):
    """The last key alone in its tile is NaN: so are the results and the softmax' denominators of all rows, and every gradient of a
    key that they see."""
    cu, qkv, dout = packed([n], 0, heads, heads, 32, dtype)
    q, k, v = (t.contiguous() for t in split(qkv.cuda(), heads, heads))
    k[-1] = float("nan")
    out, lse = ca.attention(q, k, v)
    assert torch.isnan(out).all() and torch.isnan(lse).all()
    assert all(torch.isnan(t).all() for t in ca.attention_backward(dout.cuda(), q, k, v, out, lse))


@pytest.mark.parametrize("n,block", [(98304, 0), (3000, 0), (98304, 49152)])
def test_attention_fp16_dv_of_long_sequences(n, block):
    """Queries of zero see all keys alike: p = 1 / n, which fp16 holds with 8 bits only at this length.  64 rows of dout are 1:
    dv = 64 p for every key (a key of the second block: from the rows of that block).  p and dv are rounded once each (2^-11), the sum's
    64 terms in fp32 (64 2^-24), exp2 of the logarithm of n is off by less than 1e-5."""
    d = 16
    q = torch.zeros(n, 1, d, dtype=F16, device="cuda")
    k, v = (randn(n, 1, d, dtype=F16, seed=i).cuda() for i in (1, 2))
    dout = torch.zeros_like(q)
    dout[-64:] = 1
    out, lse = ca.attention(q, k, v, causal_block=block)
    dv = ca.attention_backward(dout, q, k, v, out, lse, causal_block=block)[2].double().cpu()
    assert ((dv - 64 / n).abs() <= 64 / n * (2 * half_eps(F16) + 64 * 2.0 ** -24 + 1e-5)).all(), float((dv * n / 64 - 1).abs().max())


def test_tensors_with_a_tangent_or_a_gradient_are_refused():
    from torch.autograd import forward_ad
    x, pos = randn(8, 2, 32).cuda(), torch.zeros(8, 1, dtype=torch.int32, device="cuda")
    out, lse = ca.attention(x, x, x)
    calls = {"x": lambda t: ca.rotary(t, pos, [32]), "dout": lambda t: ca.rotary_backward(t, pos, [32]), "q": lambda t: ca.attention(t, x, x),
             "k": lambda t: ca.attention(x, t, x), "v": lambda t: ca.attention(x, x, t),
             "a gradient": lambda t: ca.attention_backward(t, x, x, x, out, lse), "m": lambda t: ca.orthogonalize([x[:, 0], t[:, 0]])}
    with forward_ad.dual_level():
        for name, call in calls.items():
            with pytest.raises(ValueError, match="tangent"):
                call(forward_ad.make_dual(x, torch.ones_like(x)))
            call(x)                                           # others are taken inside a level too
            call(forward_ad.unpack_dual(forward_ad.make_dual(x, torch.ones_like(x))).primal)
        with pytest.raises(ValueError, match="tangent"):
            ca.attention_backward(x, x, x, x, out, forward_ad.make_dual(lse, torch.ones_like(lse)))
    with pytest.raises(ValueError, match="requires a gradient"):
        ca.attention_backward(x, x, x, x, out, lse.clone().requires_grad_())


def test_numbers_past_32_bits_are_refused():
    """None of them may be taken for its lower 32 bits."""
    x, pos = randn(8, 2, 32, dtype=BF16).cuda(), torch.zeros(8, 1, dtype=torch.int32, device="cuda")
    for block in (2 ** 31, 2 ** 32, 2 ** 32 + 1, -2 ** 32 + 1):
        with pytest.raises(ValueError, match="causal_block"):
            ca.attention(x, x, x, causal_block=block)
    for axis in (2 ** 32 + 32, -2 ** 32 + 32):
        with pytest.raises(ValueError, match="axes_dim"):
            ca.rotary(x, pos, [axis])
    wide = x[:, :1].expand(8, 2 ** 32 + 2, 32)
    with pytest.raises(ValueError, match="2\\^31"):
        ca.rotary(wide, pos, [32], out=wide)
    with pytest.raises(ValueError, match="2\\^31"):
        ca.attention(wide, x, x, out=wide)
    one = torch.zeros(1, device="cuda")
    with pytest.raises(ValueError, match="32768"):
        ca.orthogonalize(one.expand(2 ** 32 + 8, 1), out=one.expand(2 ** 32 + 8, 1))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("count,rows,cols", [
    (6, 1030, 1300),        # P X on tiles of 256 (180 of them), the symmetric products on 128
    (5, 1300, 1030),        # the same, tall: the result is written transposed
    (11, 2309, 2051),       # the symmetric products on 256 too, tall, odd sizes
    (40, 390, 1030),        # the symmetric products on 64, P X on 128
    (40, 1031, 390),        # the same, tall
])
def test_orthogonalize_every_tile_size(count, rows, cols, dtype):
    """Stacks that are large enough for the wide tiles; the first and the last matrix against 64 bits."""
    G = torch.empty(count, rows, cols, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(rows + cols)
    G.normal_(generator=gen)
    G += torch.randn(count, rows, 4, device="cuda", generator=gen) @ torch.randn(count, 4, cols, device="cuda", generator=gen)
    G = (1e-3 * G).to(dtype)
    got = ca.orthogonalize(G, steps=3)
    assert torch.isfinite(got).all()
    for i in (0, count - 1):
        ortho_close(got[i], G[i].cpu(), steps=3)


def test_one_row_of_a_long_head_major_cache():
    """A dimension of size one has no stride that counts, however far its heads lie apart."""
    base = randn(16, 1, 128, dtype=BF16, seed=3)
    cache = torch.zeros(16, 2 ** 13 + 8, 128, dtype=BF16, device="cuda")
    cache[:, 5:6] = base.cuda()
    row = cache[:, 5:6].transpose(0, 1)                      # [1, 16, 128], heads 2^20 elements and more apart
    q = randn(1, 16, 128, dtype=BF16, seed=4)
    out, lse = ca.attention(q.cuda(), row, row)
    assert torch.equal(out, row) and out.shape == q.shape    # one key: its value
    ref, bound = attention_ref(q, base.transpose(0, 1), base.transpose(0, 1), [0, 1], 0, 128 ** -0.5, q)
    within(lse, ref["lse"], bound["lse"], "lse")
    for n, t in zip(("dq", "dk", "dv"), ca.attention_backward(q.cuda(), q.cuda(), row, row, out, lse)):
        within(t, ref[n], bound[n], n)
    turned = ca.rotary(row, torch.zeros(1, 1, dtype=torch.int32, device="cuda"), [128], out=row)
    assert torch.equal(turned, row)
    same = q.cuda()[:, :1].expand(1, 16, 128)                # one row of one head, repeated
    assert torch.equal(ca.attention(same, row, row)[0], row)


def rounding_ratio(got, exact):
    """error of a 16-bit result in units of what rounding the exact one would give"""
    exact = exact.double()
    rel = lambda t: float((t.double().cpu() - exact).norm() / exact.norm())
    return rel(got) / rel(exact.to(got.dtype))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("n,heads,d,block", [(155, 8, 80, 5), (155, 16, 32, 3), (300, 16, 64, 7)])
def test_attention_dq_of_rows_that_see_few_keys(n, heads, d, block, dtype):
    """The rounding of ds and of dq are each as large as the result's own: 1.41 of it together.  The rounding of out, through delta,
    would make it 1.6 and more in rows of 25 keys and less, so it must stay out of these.  1.52 leaves 7 % to the sample's spread
    (7000 elements and more; five seeds of the exact arithmetic gave 1.37 .. 1.50 with delta exact, 1.54 .. 1.82 without)."""
    cu, qkv, dout = packed([n], 0, heads, heads, d, dtype, seed=3)
    ref, _ = attention_ref(*split(qkv, heads, heads), cu, block, d ** -0.5, dout)
    q, k, v = split(qkv.cuda(), heads, heads)
    out, lse = ca.attention(q, k, v, causal_block=block)
    dq = ca.attention_backward(dout.cuda(), q, k, v, out, lse, causal_block=block)[0]
    assert rounding_ratio(dq[:25], ref["dq"][:25]) <= 1.52


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("lens,heads,kv,d,block", [([46], 2, 2, 16, 1), ([2, 3, 0, 2, 2, 3, 4], 3, 3, 48, 196), ([5, 17], 2, 2, 64, 64), ([7] * 9, 8, 2, 128, 0),
                                                   ([338], 8, 8, 16, 5), ([100] * 10, 4, 4, 16, 0), ([200, 50], 4, 4, 80, 1)])
def test_attention_gradients_of_small_calls(lens, heads, kv, d, block, dtype):
    """ds and p enter in two pieces, 2^-17 off and less, which leaves the results' own rounding (1) and that of out through delta (up to
    half as much, 1.12 together).  In one piece each would add 1 more: 1.41 .. 1.8.  Up to 1024 rows x heads, 4096 of heads up to 24."""
    cu, qkv, dout = packed(lens, 0, heads, kv, d, dtype, seed=11)
    ref, _ = attention_ref(*split(qkv, heads, kv), cu, block, d ** -0.5, dout)
    q, k, v = split(qkv.cuda(), heads, kv)
    kw = dict(cu_seqlens=table(cu), causal_block=block)
    out, lse = ca.attention(q, k, v, **kw)
    for n, t in zip(("dq", "dk", "dv"), ca.attention_backward(dout.cuda(), q, k, v, out, lse, **kw)):
        assert rounding_ratio(t, ref[n]) <= 1.25, n


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("lens,heads,d,block", [([2258, 257], 4, 16, 196), ([512] * 8, 8, 24, 1)])
def test_attention_dq_of_narrow_heads(lens, heads, d, block, dtype):
    cu, qkv, dout = packed(lens, 0, heads, heads, d, dtype, seed=12)
    ref, _ = attention_ref(*split(qkv, heads, heads), cu, block, d ** -0.5, dout)
    q, k, v = split(qkv.cuda(), heads, heads)
    kw = dict(cu_seqlens=table(cu), causal_block=block)
    out, lse = ca.attention(q, k, v, **kw)
    assert rounding_ratio(ca.attention_backward(dout.cuda(), q, k, v, out, lse, **kw)[0], ref["dq"]) <= 1.25


def rel(got, want):
    return float((got.double().cpu() - want).norm() / want.norm())


def test_attention_fp32_sums_of_long_walks():
    """A sum of N random terms whose every addition rounds by U / sqrt(3) (rms) of the sum so far is off by sqrt(N / 2) U / sqrt(3) of the
    result.  dk and dv of 4 heads' 2048 queries, out and dq of 8192 keys: in one chain, two products an instruction, 4096 roundings
    make 1.6e-6; sums apart for 32 rows leave 256 and 16: 4e-7.  p adds 5e-7: lse and the exponent's argument, 8 .. 16, are held to
    half of 2^-20 three times.  Together 6.5e-7, and half as much again for the sample, scores and exp: 1e-6."""
    heads, kv, d, n = 16, 4, 64, 2048
    cu, qkv, dout = packed([n] * 8, 0, heads, kv, d, F32)
    q, k, v = split(qkv.cuda(), heads, kv)
    out, lse = ca.attention(q, k, v, seq_len=n)
    _, dk, dv = ca.attention_backward(dout.cuda(), q, k, v, out, lse, seq_len=n)
    ref, _ = attention_ref(qkv[:n, :4], qkv[:n, heads:heads + 1], qkv[:n, heads + kv:heads + kv + 1], [0, n], 0, d ** -0.5, dout[:n, :4])
    for name, t in (("dk", dk), ("dv", dv)):
        assert rel(t[:n, :1], ref[name]) <= 1e-6, name
    n, d = 8192, 16
    cu, qkv, dout = packed([n], 0, 3, 3, d, F32)
    q, k, v = split(qkv.cuda(), 3, 3)
    out, lse = ca.attention(q, k, v)
    dq = ca.attention_backward(dout.cuda(), q, k, v, out, lse)[0]
    # the reference's first 256 rows
    Q, K, V, G = (t.double().transpose(0, 1) for t in (qkv[:256, :3], qkv[:, 3:6], qkv[:, 6:], dout[:256]))
    p = torch.softmax(Q @ K.transpose(1, 2) / 4, 2)
    O = p @ V
    ds = p * (G @ V.transpose(1, 2) - (G * O).sum(2, keepdim=True))
    assert rel(out[:256].transpose(0, 1), O) <= 1e-6
    assert rel(dq[:256].transpose(0, 1), ds @ K / 4) <= 1e-6


def test_refusals_name_what_is_wrong():
    x = torch.zeros(8, 2, 0, dtype=BF16, device="cuda")
    with pytest.raises(ca._lib.CoraError, match="head_dim"):
        ca.attention(x, x, x)
    with pytest.raises(TypeError, match="torch tensor"):
        ca.orthogonalize([torch.zeros(4, 4, device="cuda"), [[1.0]]])
