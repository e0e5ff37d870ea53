"""The stand-alone operators against their definitions in 64 bits (tests/operator_bounds.py derives the bounds)."""
import math

import pytest
import torch

import cora_amd as ca
from tests.operator_bounds import attention_ref, ortho_bound, ortho_ref, rotary_ref

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
COEF = (3.4445, -4.7750, 2.0315)


def within(got, ref, bound, what):
    got = got.double().cpu()
    bad = ~((got - ref).abs() <= bound)
    assert not bad.any(), (what, int(bad.sum()), float((got - ref).abs().max()), float(((got - ref).abs() / bound.clamp_min(1e-300)).max()))


def randn(*shape, dtype=F32, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (scale * torch.randn(*shape, generator=g)).to(dtype)


# ---- rotary ----------------------------------------------------------------------------------------------------------
ROTARY = [  # rows, positions, heads, head_dim, axes, interleaved
    (1, 1, 1, 2, [2], True), (1, 1, 1, 16, [16], False), (64, 64, 2, 64, [16, 16, 16], True), (48, 16, 3, 64, [16, 16, 16], False),
    (130, 65, 5, 48, [16, 16], True), (77, 77, 2, 80, [8, 40, 32], False), (33, 33, 7, 128, [32, 40, 40], True),
    (1000, 10, 1, 128, [64, 64], False), (19, 19, 4, 20, [6, 2, 4, 8], True), (19, 19, 4, 20, [6, 2, 4], False),
    (257, 257, 24, 96, [2, 30, 64], True), (5, 5, 300, 32, [32], False), (9, 9, 2, 200, [64, 64], True), (6, 6, 3, 7, [4, 2], True),
]


def positions(n, axes, seed, top):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-2, top, (n, axes), generator=g, dtype=torch.int32)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,n,heads,d,axes,inter", ROTARY)
def test_rotary(rows, n, heads, d, axes, inter, dtype):
    x = randn(rows, heads, d, dtype=dtype, seed=rows + d)
    pos = positions(n, len(axes), 3, 70)
    for theta, backward in ((1e4, False), (100.0, True)):
        f = ca.rotary_backward if backward else ca.rotary
        ref, bound = rotary_ref(x, pos, axes, theta, inter, backward)
        xg = x.cuda()
        y = f(xg, pos.cuda(), axes, theta=theta, interleaved=inter)
        within(y, ref, bound, (theta, backward))
        assert torch.equal(y[..., sum(axes):].cpu(), x[..., sum(axes):])
        assert f(xg, pos.cuda(), axes, theta=theta, interleaved=inter, out=xg) is xg     # in place
        assert torch.equal(xg, y)


@pytest.mark.parametrize("inter", [True, False])
def test_rotary_far_positions(inter):
    x = randn(64, 2, 64, seed=4)
    pos = torch.randint(-2**31, 2**31 - 1, (64, 2), generator=torch.Generator().manual_seed(5), dtype=torch.int64).to(torch.int32)
    ref, bound = rotary_ref(x, pos, [32, 32], 1e4, inter)
    within(ca.rotary(x.cuda(), pos.cuda(), [32, 32], interleaved=inter), ref, bound, "far")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shift", [0, 8, 3])
def test_rotary_strided(dtype, shift):
    """q and k of a packed projection, and a head-major layout; an offset of 3 elements breaks every vector's alignment."""
    base = randn(20, 7 * 32 + 11, dtype=dtype, seed=9).cuda()
    pos = positions(20, 2, 1, 30)
    x = base[:, shift:shift + 4 * 32].unflatten(1, (4, 32))
    ref, bound = rotary_ref(x.cpu(), pos, [16, 8], 1e4, True)
    keep = base.clone()
    within(ca.rotary(x, pos.cuda(), [16, 8]), ref, bound, "packed")
    out = torch.full((4, 20, 40), 7.0, dtype=dtype, device="cuda")
    ca.rotary(x, pos.cuda(), [16, 8], out=out.transpose(0, 1)[:, :, :32])
    within(out.transpose(0, 1)[:, :, :32], ref, bound, "head-major")
    assert (out[:, :, 32:] == 7).all()
    ca.rotary(x, pos.cuda(), [16, 8], out=x)
    keep[:, shift:shift + 128] = base[:, shift:shift + 128]
    assert torch.equal(keep, base)                       # nothing else of the projection changed
    same = x[:, :1].expand(20, 4, 32)                    # one head repeated
    within(ca.rotary(same, pos.cuda(), [16, 8]), *rotary_ref(same.cpu(), pos, [16, 8], 1e4, True), "repeated")


def test_rotary_is_the_transpose_of_its_backward():
    x, g = randn(40, 3, 64, seed=1).cuda(), randn(40, 3, 64, seed=2).cuda()
    pos = positions(40, 3, 1, 50).cuda()
    a = (ca.rotary(x, pos, [16, 16, 16]).double() * g.double()).sum()
    b = (x.double() * ca.rotary_backward(g, pos, [16, 16, 16]).double()).sum()
    assert abs(a - b) <= 12 * 2.0 ** -24 * float((x.double().abs() * 2).sum() * g.abs().max())


def test_rotary_offsets_past_32_bits():
    big = torch.empty(2 ** 32 + 4096, dtype=BF16, device="cuda")
    x = big.as_strided((3, 2, 64), (2 ** 31 + 512, 64, 1))
    x.copy_(randn(3, 2, 64, dtype=BF16, seed=3))
    pos = positions(3, 1, 1, 50)
    ref, bound = rotary_ref(x.cpu(), pos, [64], 1e4, True)
    ca.rotary(x, pos.cuda(), [64], out=x)
    within(x, ref, bound, "past 2^32")


def test_rotary_more_rows_than_a_launch_has_threads():
    rows = 2 ** 32 + 512
    x = torch.zeros(rows, 1, 2, dtype=F16, device="cuda")
    ends = [slice(0, 512), slice(2 ** 32 - 512, 2 ** 32), slice(2 ** 32, rows)]
    for i, e in enumerate(ends):
        x[e].copy_(randn(512, 1, 2, dtype=F16, seed=i))
    before = [x[e].cpu() for e in ends]
    pos = positions(512, 1, 7, 50)
    assert ca.rotary(x, pos.cuda(), [2], out=x) is x
    for e, b in zip(ends, before):
        ref, bound = rotary_ref(b, pos, [2], 1e4, True)
        within(x[e], ref, bound, e)


def test_rotary_no_rows():
    assert ca.rotary(torch.empty(0, 2, 16, device="cuda"), torch.zeros(1, 1, dtype=torch.int32, device="cuda"), [16]).shape == (0, 2, 16)


# ---- attention -------------------------------------------------------------------------------------------------------
ATTN = [  # lens, tail, heads, kv_heads, head_dim, causal block
    ([1], 0, 1, 1, 16, 0), ([1, 0, 2, 0, 0, 1], 3, 2, 1, 32, 1), ([64], 0, 1, 1, 64, 0), ([65, 31, 128], 0, 2, 2, 64, 1),
    ([200], 5, 4, 2, 48, 0), ([129, 1, 257], 70, 6, 2, 128, 1), ([130, 300], 0, 3, 3, 80, 64), ([127, 128, 129], 0, 2, 1, 96, 5),
    ([300] * 5 + [1, 260], 3, 12, 4, 48, 1), ([2100], 0, 2, 1, 64, 64), ([290, 300, 310], 0, 12, 6, 128, 0), ([33, 500], 0, 4, 1, 24, 7), ([400], 0, 8, 8, 16, 196), ([0, 0, 90], 0, 2, 2, 8, 1), ([256], 0, 5, 5, 112, 1000), ([192], 1, 2, 1, 128, 0),
]


def packed(lens, tail, heads, kv, d, dtype, seed=0):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    qkv = randn(cu[-1] + tail, heads + 2 * kv, d, dtype=dtype, seed=seed + sum(lens) + d)
    dout = randn(cu[-1] + tail, heads, d, dtype=dtype, seed=seed + 77 + d)
    return cu, qkv, dout


def split(qkv, heads, kv):
    return qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("lens,tail,heads,kv,d,block", ATTN)
def test_attention(lens, tail, heads, kv, d, block, dtype):
    cu, qkv, dout = packed(lens, tail, heads, kv, d, dtype)
    scale = 1 / math.sqrt(d)
    ref, bound = attention_ref(*split(qkv, heads, kv), cu, block, scale, dout)
    rows, total = qkv.shape[0], cu[-1]
    q, k, v = split(qkv.cuda(), heads, kv)
    kw = dict(cu_seqlens=torch.tensor(cu, dtype=torch.int32, device="cuda"), causal_block=block)
    out = torch.full((rows, heads, d), 3.0, dtype=dtype, device="cuda")
    lse = torch.full((heads, rows), 5.0, device="cuda")
    assert ca.attention(q, k, v, out=out, lse=lse, **kw)[0] is out
    within(out[:total], ref["out"][:total], bound["out"][:total], "out")
    within(lse[:, :total], ref["lse"][:, :total], bound["lse"][:, :total], "lse")
    assert (out[total:] == 3).all() and (lse[:, total:] == 5).all()         # rows of no sequence
    dqkv = torch.full(qkv.shape, 9.0, dtype=dtype, device="cuda")            # gradients straight into a packed projection's
    dq, dk, dv = split(dqkv, heads, kv)
    ca.attention_backward(dout.cuda(), q, k, v, out, lse, dq=dq, dk=dk, dv=dv, **kw)
    for n, t in (("dq", dq), ("dk", dk), ("dv", dv)):
        within(t[:total], ref[n][:total], bound[n][:total], n)
    assert (dqkv[total:] == 9).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_equal_lengths_without_a_table(dtype):
    cu, qkv, dout = packed([50] * 6, 0, 4, 2, 32, dtype)
    q, k, v = split(qkv.cuda(), 4, 2)
    a = ca.attention(q, k, v, seq_len=50, causal_block=10)
    b = ca.attention(q, k, v, cu_seqlens=torch.tensor(cu, dtype=torch.int32, device="cuda"), causal_block=10)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    ga = ca.attention_backward(dout.cuda(), q, k, v, *a, seq_len=50, causal_block=10)
    gb = ca.attention_backward(dout.cuda(), q, k, v, *a, cu_seqlens=torch.tensor(cu, dtype=torch.int32, device="cuda"), causal_block=10)
    assert all(torch.equal(x, y) for x, y in zip(ga, gb))
    one = ca.attention(q, k, v)                                             # all rows one sequence
    ref, bound = attention_ref(*split(qkv, 4, 2), [0, 300], 0, 1 / math.sqrt(32))
    within(one[0], ref["out"], bound["out"], "one sequence")


def test_attention_layouts_and_scale():
    """head-major tensors, a repeated key head (stride 0), another scale, outputs of another layout."""
    q0, kv0 = randn(3, 100, 64, dtype=BF16, seed=1), randn(100, 1, 64, dtype=BF16, seed=2)
    q, k = q0.cuda().transpose(0, 1), kv0.cuda().expand(100, 3, 64)
    ref, bound = attention_ref(q0.transpose(0, 1), k.cpu(), k.cpu(), [0, 100], 1, 0.3)
    out = torch.empty(3, 100, 64, dtype=BF16, device="cuda").transpose(0, 1)
    ca.attention(q, k, k, causal_block=1, scale=0.3, out=out)
    within(out, ref["out"], bound["out"], "head-major")


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_attention_large_scores(dtype):
    """Scores of some hundred, differing signs, and rows whose softmax is one-hot."""
    cu, qkv, dout = packed([150, 90], 0, 2, 2, 64, dtype, seed=5)
    qkv[:, :2] *= 8
    ref, bound = attention_ref(*split(qkv, 2, 2), cu, 1, 0.125, dout)
    q, k, v = split(qkv.cuda(), 2, 2)
    kw = dict(cu_seqlens=torch.tensor(cu, dtype=torch.int32, device="cuda"), causal_block=1)
    out, lse = ca.attention(q, k, v, **kw)
    within(out, ref["out"], bound["out"], "out")
    within(lse, ref["lse"], bound["lse"], "lse")
    for n, t in zip(("dq", "dk", "dv"), ca.attention_backward(dout.cuda(), q, k, v, out, lse, **kw)):
        within(t, ref[n], bound[n], n)


@pytest.mark.parametrize("size", [1e-7, 3e3])
def test_attention_fp16_gradients_keep_small_and_large_scales(size):
    cu, qkv, dout = packed([300], 0, 2, 1, 64, F16, seed=6)
    dout = (dout.float() * torch.logspace(0, -3, 300)[:, None, None] * size * (2.0 ** 10 if size < 1 else 1)).to(F16)
    ref, bound = attention_ref(*split(qkv, 2, 1), cu, 0, 0.125, dout)
    q, k, v = split(qkv.cuda(), 2, 1)
    out, lse = ca.attention(q, k, v)
    for n, t in zip(("dq", "dk", "dv"), ca.attention_backward(dout.cuda(), q, k, v, out, lse)):
        within(t, ref[n], bound[n], n)


def test_attention_gradients_against_differences():
    cu, qkv, dout = packed([37, 20], 0, 2, 1, 16, F32, seed=8)
    kw = dict(cu_seqlens=torch.tensor(cu, dtype=torch.int32, device="cuda"), causal_block=4)
    q, k, v = (t.cuda().contiguous() for t in split(qkv, 2, 1))
    out, lse = ca.attention(q, k, v, **kw)
    grads = ca.attention_backward(dout.cuda(), q, k, v, out, lse, **kw)
    g = dout.cuda().double()
    for i, t in enumerate((q, k, v)):
        step = randn(*t.shape, seed=20 + i).cuda()
        args = [q, k, v]
        f = []
        for s in (1, -1):
            args[i] = t + s * 2.0 ** -6 * step
            f.append((ca.attention(*args, **kw)[0].double() * g).sum())
        diff, exact = float((f[0] - f[1]) / 2.0 ** -5), float((grads[i].double() * step.double()).sum())
        # the difference quotient is off by its third derivative's h^2 / 6 (h = 2^-6: 4e-5 of directional terms of the size
        # below) and by fp32 results over 2 h (2^-24 * 2^5 of their size)
        size = float((g.abs() * out.double().abs()).sum() + (grads[i].double().abs() * step.double().abs()).sum())
        assert abs(diff - exact) <= 2e-3 * size, (i, diff, exact)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_attention_other_sequences_do_not_leak(dtype):
    """NaN and infinity in a neighbouring sequence, in rows of no sequence and before the first one stay there."""
    cu, qkv, dout = packed([70, 33, 140], 40, 2, 2, 64, dtype)
    cut = [70, 103]                                            # only the middle sequence
    for t in (qkv, dout):
        t[:70], t[103:] = float("nan"), float("inf")
    ref, bound = attention_ref(*split(qkv, 2, 2), cut, 1, 0.125, dout)
    q, k, v = split(qkv.cuda(), 2, 2)
    kw = dict(cu_seqlens=torch.tensor(cut, dtype=torch.int32, device="cuda"), causal_block=1)
    out, lse = ca.attention(q, k, v, **kw)
    within(out[70:103], ref["out"][70:103], bound["out"][70:103], "out")
    for n, t in zip(("dq", "dk", "dv"), ca.attention_backward(dout.cuda(), q, k, v, out, lse, **kw)):
        within(t[70:103], ref[n][70:103], bound[n][70:103], n)


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("lens,heads,kv,d,block", [([150, 3, 90], 4, 2, 64, 1), ([150, 90], 2, 2, 48, 50), ([300], 2, 1, 128, 7),
                                                   ([200] * 90, 4, 2, 32, 40), ([700] * 40, 2, 2, 96, 1)])
def test_attention_what_the_mask_hides_does_not_count(lens, heads, kv, d, block, dtype, value):
    """One token of every sequence has keys, values, queries or gradients that are not finite: what does not see it keeps its
    result.  Forward and dq repeat the untouched ones bit for bit (products with zero weights add zeros)."""
    cu, qkv, dout = packed(lens, 0, heads, kv, d, dtype)
    rows = cu[-1]
    lim, bad = torch.empty(rows, dtype=torch.long), torch.empty(rows, dtype=torch.long)
    for b, e in zip(cu, cu[1:]):
        i = torch.arange(e - b)
        lim[b:e], bad[b:e] = b + torch.clamp((i // block + 1) * block, max=e - b), b + (e - b) // 2
    at = torch.unique(bad)
    kw = dict(cu_seqlens=torch.tensor(cu, dtype=torch.int32, device="cuda"), causal_block=block)
    q, k, v = split(qkv.cuda(), heads, kv)
    g = dout.cuda()
    out, lse = ca.attention(q, k, v, **kw)
    dq, dk, dv = ca.attention_backward(g, q, k, v, out, lse, **kw)
    hides = (lim <= bad).cuda()                                      # rows that do not see the token's key
    assert hides.any()
    for name in ("k", "v"):
        t = {"k": k.clone(), "v": v.clone()}
        t[name][at, -1, d // 3] = value
        out2, lse2 = ca.attention(q, t["k"], t["v"], **kw)
        assert torch.equal(out2[hides], out[hides]) and torch.equal(lse2[:, hides], lse[:, hides]), name
        dq2 = ca.attention_backward(g, q, t["k"], t["v"], out2, lse2, **kw)[0]
        assert torch.equal(dq2[hides], dq[hides]), name
        if value != value:
            assert torch.isnan(out2[~hides][:, -1]).any(-1).all() and torch.isnan(dq2[~hides][:, -1]).any(-1).all(), name
    first = torch.arange(rows) >= lim[bad]                           # keys that the token's query does not see
    ref, bound = attention_ref(*split(qkv, heads, kv), cu, block, d ** -0.5, dout)
    for name in ("q", "dout"):
        t = {"q": q.clone(), "dout": g.clone()}
        t[name][at, -1, d // 3] = value
        out2, lse2 = ca.attention(t["q"], k, v, **kw)
        got = ca.attention_backward(t["dout"], t["q"], k, v, out2, lse2, **kw)
        for n, new, old in zip(("dk", "dv"), got[1:], (dk, dv)):
            within(new[first.cuda()], ref[n][first], bound[n][first], (name, n))
            if dtype is not F16:                                     # fp16: the rows' common exponent may have changed
                assert torch.equal(new[first.cuda()], old[first.cuda()]), (name, n)
        if value != value:
            assert torch.isnan(got[2][~first.cuda()][:, -1]).any(-1).all(), name


@pytest.mark.parametrize("n,seqs,heads,d,block,dtype", [(1024, 16, 1, 64, 64, F32), (700, 40, 2, 96, 1, BF16), (129, 130, 4, 32, 1, F16)])
def test_attention_many_causal_tiles_with_and_without_a_table(n, seqs, heads, d, block, dtype):
    """Enough tiles that the longest start first: where a tile runs changes no result."""
    cu, qkv, dout = packed([n] * seqs, 0, heads, heads, d, dtype)
    q, k, v = split(qkv.cuda(), heads, heads)
    results = []
    for kw in (dict(seq_len=n), dict(cu_seqlens=torch.tensor(cu, dtype=torch.int32, device="cuda"))):
        out, lse = ca.attention(q, k, v, causal_block=block, **kw)
        results.append((out, lse) + ca.attention_backward(dout.cuda(), q, k, v, out, lse, causal_block=block, **kw))
    for a, b in zip(*results):
        assert torch.equal(a, b)
    ref, bound = attention_ref(*split(qkv[:n], heads, heads), [0, n], block, d ** -0.5, dout[:n])
    for name, t in zip(("out", "dq", "dk", "dv"), (results[0][0],) + results[0][2:]):
        within(t[:n], ref[name], bound[name], name)


def test_attention_many_causal_tiles_with_empty_sequences():
    lens = [0, 1000, 0, 1, 700, 33, 2100, 0, 900, 1300, 31, 1024, 0]
    cu, qkv, dout = packed(lens, 40, 12, 4, 32, BF16)
    ref, bound = attention_ref(*split(qkv, 12, 4), cu, 16, 32 ** -0.5, dout)
    q, k, v = split(qkv.cuda(), 12, 4)
    kw = dict(cu_seqlens=torch.tensor(cu, dtype=torch.int32, device="cuda"), causal_block=16)
    out, lse = ca.attention(q, k, v, **kw)
    within(out[:cu[-1]], ref["out"][:cu[-1]], bound["out"][:cu[-1]], "out")
    for n, t in zip(("dq", "dk", "dv"), ca.attention_backward(dout.cuda(), q, k, v, out, lse, **kw)):
        within(t[:cu[-1]], ref[n][:cu[-1]], bound[n][:cu[-1]], n)


def test_attention_broken_tables_stay_in_bounds():
    """Descending and out-of-range bounds: rows outside [0, rows) are never touched and the call ends."""
    q = randn(50, 2, 32, dtype=BF16).cuda()
    for cu in ([0, 500], [-7, 20, 60], [30, 10, 50], [50, 50], [0, 0]):
        out = torch.zeros_like(q)
        out, lse = ca.attention(q, q, q, cu_seqlens=torch.tensor(cu, dtype=torch.int32, device="cuda"), out=out)
        ca.attention_backward(q, q, q, q, out, lse, cu_seqlens=torch.tensor(cu, dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()


def test_attention_repeats_bit_for_bit_and_on_another_stream():
    cu, qkv, dout = packed([300, 77, 513], 0, 4, 2, 64, BF16)
    q, k, v = split(qkv.cuda(), 4, 2)
    g, kw = dout.cuda(), dict(cu_seqlens=torch.tensor(cu, dtype=torch.int32, device="cuda"), causal_block=1)
    first = ca.attention(q, k, v, **kw)
    first += ca.attention_backward(g, q, k, v, *first, **kw)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        second = ca.attention(q, k, v, **kw)
        second += ca.attention_backward(g, q, k, v, *second, **kw)
    st.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, second))


def test_refusals_on_the_gpu():
    x = torch.zeros(8, 2, 32, device="cuda", dtype=BF16)
    pos = torch.zeros(8, 1, device="cuda", dtype=torch.int32)
    with pytest.raises(ValueError, match="multiple"):
        ca.attention(x, x[:, :1].expand(8, 3, 32), x[:, :1].expand(8, 3, 32))
    with pytest.raises(ValueError, match="expected torch.bfloat16"):
        ca.attention(x, x.float(), x)
    with pytest.raises(ValueError, match="contiguous"):
        ca.attention(torch.zeros(8, 2, 64, device="cuda", dtype=BF16)[..., ::2], x, x)
    with pytest.raises(ca._lib.CoraError, match="16-byte"):
        ca.attention(torch.zeros(8, 2, 40, device="cuda", dtype=BF16)[..., 1:33], x, x)
    with pytest.raises(ca._lib.CoraError, match="head_dim"):
        ca.attention(*[torch.zeros(8, 2, 20, device="cuda", dtype=BF16)] * 3)
    with pytest.raises(ValueError, match="int32"):
        ca.attention(x, x, x, cu_seqlens=torch.tensor([0, 8], device="cuda"))
    with pytest.raises(ValueError, match="seq_len"):
        ca.attention(x, x, x, seq_len=3)
    with pytest.raises(ValueError, match="not both"):
        ca.attention(x, x, x, seq_len=4, cu_seqlens=torch.tensor([0, 8], device="cuda", dtype=torch.int32))
    with pytest.raises(ValueError, match="lse"):
        ca.attention_backward(x, x, x, x, x, torch.zeros(8, 2, device="cuda"))
    with pytest.raises(ValueError, match="requires a gradient"):
        ca.attention(x.clone().requires_grad_(), x, x)
    with pytest.raises(ValueError, match="dtype"):
        ca.rotary(torch.zeros(8, 2, 32, device="cuda", dtype=torch.float64), pos, [32])
    with pytest.raises(ValueError, match="positions"):
        ca.rotary(x, pos.long(), [32])
    with pytest.raises(ValueError, match="multiple"):
        ca.rotary(x, pos[:3].contiguous(), [32])
    with pytest.raises(ca._lib.CoraError, match="overlap"):
        ca.rotary(x, pos, [32], out=torch.zeros(1, 2, 32, device="cuda", dtype=BF16).expand(8, 2, 32))
    with pytest.raises(ValueError, match="expected torch.bfloat16"):
        ca.orthogonalize([torch.zeros(4, 4, device="cuda", dtype=BF16), torch.zeros(4, 4, device="cuda")])
    with pytest.raises(ca._lib.CoraError, match="out of range"):
        ca.orthogonalize(torch.zeros(4, 4, device="cuda"), coefficients=(9.0, 0.0, 0.0))


# ---- orthogonalisation -----------------------------------------------------------------------------------------------
SHAPES = [(1, 1), (1, 70), (70, 1), (13, 22), (64, 64), (64, 256), (256, 64), (100, 37), (128, 128), (129, 200), (200, 320), (333, 130), (300, 520), (1030, 1100), (2100, 1025)]


def gradient(r, c, seed, scale=1e-3):
    return scale * (randn(r, c, seed=seed) + randn(r, 4, seed=seed + 1) @ randn(4, c, seed=seed + 2))


def ortho_close(got, G, steps=5, coef=COEF, eps=1e-7):
    ref, tol = ortho_ref(G, steps, coef, eps), ortho_bound(G, steps, coef, eps, G.dtype)
    got = got.double().cpu()
    assert torch.isfinite(got).all()
    err = float((got - ref).norm() / ref.norm())
    assert err <= tol, (tuple(G.shape), G.dtype, err, tol)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("r,c", SHAPES)
def test_orthogonalize(r, c, dtype):
    G = gradient(r, c, r * 7 + c).to(dtype)
    ortho_close(ca.orthogonalize(G.cuda()), G)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_orthogonalize_lists_stacks_views_and_in_place(dtype):
    mats = [gradient(64 * 3, 80, 1).unflatten(0, (3, 64)), gradient(40, 160, 2), gradient(2 * 150, 140, 3).unflatten(0, (2, 150)), gradient(64, 64, 4)]
    mats = [m.to(dtype) for m in mats]
    wide = torch.full((3, 64, 96), 5.0, dtype=dtype, device="cuda")
    wide[..., :80] = mats[0].cuda()
    args = [wide[..., :80]] + [m.cuda() for m in mats[1:]]
    got = ca.orthogonalize(args)
    for m, o in zip(mats, got):
        for a, b in (zip(m, o) if m.dim() == 3 else [(m, o)]):
            ortho_close(b, a)
    assert ca.orthogonalize(args, out=args)[0] is args[0]
    assert all(torch.equal(a, b) for a, b in zip(args, got)) and (wide[..., 80:] == 5).all()


def test_orthogonalize_many_stacks():
    mats = [gradient(8 + i, 30, i) for i in range(40)]                  # more stacks than one launch takes
    for m, o in zip(mats, ca.orthogonalize([m.cuda() for m in mats])):
        ortho_close(o, m)


@pytest.mark.parametrize("shape", [(48, 96), (150, 200)])
@pytest.mark.parametrize("scale", [1e-30, 1e15])
def test_orthogonalize_any_size_of_gradient(scale, shape):
    G = gradient(*shape, 5, scale)
    ortho_close(ca.orthogonalize(G.cuda(), eps=0.0), G, eps=0.0)


@pytest.mark.parametrize("shape", [(48, 96), (150, 200)])
def test_orthogonalize_zero_nan_steps_and_coefficients(shape):
    z = torch.zeros(2, *shape, device="cuda")
    z[1] = gradient(*shape, 6).cuda()
    out = ca.orthogonalize(z)
    assert (out[0] == 0).all()                                           # a parameter without gradient
    ortho_close(out[1], z[1].cpu())
    z[0, 3, 5] = float("nan")
    out = ca.orthogonalize(z)
    assert torch.isnan(out[0]).all()                                     # stays with its own matrix
    ortho_close(out[1], z[1].cpu())
    per_step = [(4.0, -6.5, 3.4), (3.0, -4.0, 1.9), (1.875, -1.25, 0.375)]
    with pytest.raises(ca._lib.CoraError, match="out of range"):          # 1 -> 0.9, but 0.57 -> 1.3 -> 2.1 -> above 8
        ca.orthogonalize(z[1], steps=3, coefficients=per_step)
    per_step = [(3.4445, -4.7750, 2.0315), (2.5, -2.25, 0.75), (1.875, -1.25, 0.375)]
    ortho_close(ca.orthogonalize(z[1], steps=3, coefficients=per_step), z[1].cpu(), 3, per_step)
    ortho_close(ca.orthogonalize(z[1], steps=1), z[1].cpu(), 1)
    assert ca.orthogonalize([]) == [] and ca.orthogonalize(torch.empty(0, 4, 4, device="cuda")).shape == (0, 4, 4)


# ---- as they are used together, and in graphs ------------------------------------------------------------------------
def sublayer(x, wq, pos, g, cu):
    """positions -> attention -> backward -> weight gradient -> orthogonal update of one projection (4 + 2 + 2 heads of 32)."""
    qkv = (x @ wq.T).unflatten(1, (8, 32))
    turned = ca.rotary(qkv[:, :6], pos, [8, 12, 12])
    q, k, v = turned[:, :4], turned[:, 4:], qkv[:, 6:]
    out, lse = ca.attention(q, k, v, cu_seqlens=cu, causal_block=16)
    d = torch.zeros_like(qkv)
    ca.attention_backward(g, q, k, v, out, lse, cu_seqlens=cu, causal_block=16, dq=d[:, :4], dk=d[:, 4:6], dv=d[:, 6:])
    ca.rotary_backward(d[:, :6], pos, [8, 12, 12], out=d[:, :6])
    dw = d.flatten(1).T @ x
    return out, dw, ca.orthogonalize(dw)


def test_a_training_sublayer():
    cu = [0, 48, 48, 128, 145]
    x, w, g = randn(145, 64, seed=1), randn(256, 64, seed=2, scale=0.1), randn(145, 4, 32, seed=3)
    pos = positions(145, 3, 4, 16)
    out, dw, update = sublayer(x.cuda(), w.cuda(), pos.cuda(), g.cuda(), torch.tensor(cu, dtype=torch.int32, device="cuda"))
    # the same with autograd in 64 bits
    W = w.double().requires_grad_()
    qkv = (x.double() @ W.T).unflatten(1, (8, 32))
    cols, start = [], 0
    for a, n in enumerate((8, 12, 12)):
        for i in range(n // 2):
            ang = pos[:, a].double()[:, None] * 1e4 ** (-2.0 * i / n)
            u, t = qkv[:, :6, start + 2 * i], qkv[:, :6, start + 2 * i + 1]
            cols += [u * ang.cos() - t * ang.sin(), u * ang.sin() + t * ang.cos()]
        start += n
    turned = torch.stack(cols, 2)
    outs = []
    for b, e in zip(cu[:-1], cu[1:]):
        for h in range(4):
            s = turned[b:e, h] @ turned[b:e, 4 + h // 2].T / math.sqrt(32)
            i = torch.arange(e - b) // 16
            outs.append((b, e, h, torch.softmax(s.masked_fill(i[None, :] > i[:, None], -math.inf), 1) @ qkv[b:e, 6 + h // 2]))
    total = sum((o * g[b:e, h].double()).sum() for b, e, h, o in outs)
    total.backward()
    ref = torch.zeros(145, 4, 32, dtype=torch.float64)
    for b, e, h, o in outs:
        ref[b:e, h] = o.detach()
    # fp32 throughout; the projections' sums of 64 and 145 terms dominate: (64 + 145 + 32) U of terms a few times the results
    assert float((out.double().cpu() - ref).norm() / ref.norm()) <= 241 * 2.0 ** -24 * 4
    assert float((dw.double().cpu() - W.grad).norm() / W.grad.norm()) <= 241 * 2.0 ** -24 * 8
    ortho_close(update, dw.cpu())


def test_operators_in_a_graph_with_eager_work_between():
    cu = torch.tensor([0, 48, 48, 128, 145], dtype=torch.int32, device="cuda")
    x, w, g = randn(145, 64, seed=1).cuda(), randn(256, 64, seed=2, scale=0.1).cuda(), randn(145, 4, 32, seed=3).cuda()
    pos = positions(145, 3, 4, 16).cuda()
    sublayer(x, w, pos, g, cu)                                    # loads the libraries' code before the capture
    graphs = []
    for _ in range(2):                                            # two graphs; their workspaces are their own
        graph = torch.cuda.CUDAGraph()
        xin = x.clone()
        with torch.cuda.graph(graph):
            res = sublayer(xin, w, pos, g, cu)
        graphs.append((graph, xin, res))
    for i in range(4):
        for n, (graph, xin, res) in enumerate(graphs):
            xin.copy_(x * (1 + i + 10 * n))
        for graph, _, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for graph, xin, res in graphs:
            eager = sublayer(xin, w, pos, g, cu)
            assert all(torch.equal(a, b) for a, b in zip(res, eager))
