"""The workloads on which the stand-alone operators of cora_amd are measured, with their plain forms.

Operators: `rotary` (rotary positions over several axes), `attention` / `attention_backward` (packed sequences,
frame-causal or bidirectional, grouped heads) and `orthogonalize` (Newton-Schulz orthogonalisation of weight updates).
`own` selects who computes: False, elementary torch operations in 32 bits (angles in 64); True, the framework's kernels.

A case is a dict of plain values:
  rotary     op, dtype, clips, grid (positions per axis of one clip), heads (those that turn), pass_heads (the v heads
             that share the rows with them), head_dim, axes (channels per axis), theta, interleaved, backward
  attention  op, dtype, lens (text: tokens of every packed sequence), tail (rows behind the last one), heads, kv_heads,
             head_dim, causal_block (0: bidirectional; b: a token sees its own and earlier blocks of b tokens), backward
  ortho      op, dtype, mats (text: "count x rows x cols" of every stack of matrices), steps
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
COEF = (3.4445, -4.7750, 2.0315)
EPS = 1e-7


def _lens(text):
    """"3*64,17" -> [64, 64, 64, 17]"""
    out = []
    for part in text.split(","):
        if "*" in part:
            n, length = part.split("*")
            out += [int(length)] * int(n)
        else:
            out.append(int(part))
    return out


def _mats(text):
    return [tuple(int(v) for v in part.split("x")) for part in text.split(",")]


def _case(name, op, **kw):
    return dict(name=name, op=op, **kw)


def listed():
    return [
        # q and k of one step of the 16-frame clips (batch 16, 16 x 8 x 8 patches, width 64, one head), forward
        _case("rotary_clips_f32", "rotary", dtype="f32", clips=16, grid="16x8x8", heads=2, pass_heads=1, head_dim=64,
              axes="16x16x16", theta=10000.0, interleaved=True, backward=False),
        # gradient of a long packed batch of clips with grouped heads; paired halves, channels left over per head
        _case("rotary_packed_bf16_bwd", "rotary", dtype="bf16", clips=5, grid="17x61x64", heads=20, pass_heads=4, head_dim=128,
              axes="32x40x40", theta=10000.0, interleaved=False, backward=True),
        # a handful of small images of different sizes answered at once: the call's latency counts
        _case("attn_few_images_bf16", "attention", dtype="bf16", lens="49,64,17,1,100", tail=0, heads=4, kv_heads=2, head_dim=32,
              causal_block=0, backward=False),
        # the 16-frame clips, a token sees its own and earlier frames: forward, 32 bits as the framework's default
        _case("attn_clips_f32", "attention", dtype="f32", lens="16*1024", tail=0, heads=1, kv_heads=1, head_dim=64,
              causal_block=64, backward=False),
        # a training step's attention on a batch of 224 x 224 images (14 x 14 patches, width 384, 8 heads)
        _case("attn_images_f32_train", "attention", dtype="f32", lens="64*196", tail=0, heads=8, kv_heads=8, head_dim=48,
              causal_block=0, backward=True),
        # packed clips of very different lengths, token-causal, grouped heads: forward
        _case("attn_packed_bf16", "attention", dtype="bf16",
              lens="4096,1000,1,333,2048,64,4095,129,3000,513,777,4097,255,31,2047,1024,3,1500,4096,600", tail=37,
              heads=16, kv_heads=4, head_dim=128, causal_block=1, backward=False),
        # images of mixed resolutions packed into one batch, bidirectional, a head size that is no power of two: training
        _case("attn_mixed_f16_train", "attention", dtype="f16",
              lens="1369,196,49,529,784,256,1,400,1024,961,81,676,144,1225,225,900,333,576,64,1089", tail=5,
              heads=12, kv_heads=12, head_dim=80, causal_block=0, backward=True),
        # packed clips, frames of 64 tokens, grouped heads: training
        _case("attn_packed_bf16_train", "attention", dtype="bf16",
              lens="1024,4096,320,2048,64,1088,3000,704,128,2560,64,1500", tail=0,
              heads=12, kv_heads=4, head_dim=64, causal_block=64, backward=True),
        # one long prompt of 16384 tokens, token-causal: training
        _case("attn_long_bf16_train", "attention", dtype="bf16", lens="16384", tail=0, heads=16, kv_heads=4, head_dim=128,
              causal_block=1, backward=True),
        # the weight step of the 6-block model (width 64): q, k, v, output and the two MLP matrices of every block
        _case("ortho_6block_f32", "ortho", dtype="f32", mats="18x64x64,6x64x64,6x256x64,6x64x256", steps=5),
        # the same for width 384 (224 x 224 images)
        _case("ortho_width384_f32", "ortho", dtype="f32", mats="18x384x384,6x384x384,6x1536x384,6x384x1536", steps=5),
        # wide layers with gradients kept in bf16; one stack is tall, one has odd sizes
        _case("ortho_wide_bf16", "ortho", dtype="bf16", mats="2x2048x8192,1x4096x2000,1x1111x2049", steps=5),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rotary", "attention", "attention", "attention", "ortho", "ortho"])
    if kind == "rotary":
        d = rng.choice([16, 32, 48, 64, 80, 96, 128])
        n = rng.choice([2, 3])
        grid = [_log(rng, 1, 32), _log(rng, 2, 64), _log(rng, 2, 64)][3 - n:]
        left, axes = d // 2, []
        for i in range(n):
            a = rng.randint(1, max(1, (left - (n - 1 - i)) if i < n - 1 else left))
            a = min(a, left - (n - 1 - i))
            axes.append(2 * a)
            left -= a
        heads, extra = rng.randint(1, 24), rng.randint(0, 8)
        clips = _log(rng, 1, max(1, min(256, 16_000_000 // (math.prod(grid) * (heads + extra) * d // 8))))
        return dict(op="rotary", dtype=rng.choice(["f32", "bf16", "f16"]), clips=clips, grid="x".join(map(str, grid)), heads=heads,
                    pass_heads=extra, head_dim=d, axes="x".join(map(str, axes)), theta=rng.choice([100.0, 10000.0]),
                    interleaved=rng.random() < 0.5, backward=rng.random() < 0.5)
    if kind == "attention":
        d = rng.choice([16, 24, 32, 48, 64, 80, 96, 128])
        kv = rng.choice([1, 2, 3, 4, 8])
        heads = kv * rng.choice([1, 1, 2, 3, 4])
        dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
        budget = 2.0e11 if dtype == "f32" else 8.0e11          # multiply-adds of the scores, forward
        top = _log(rng, 8, 8192)
        lens, cost = [], 0.0
        for _ in range(_log(rng, 1, 48)):
            n = rng.randint(0, 2) if rng.random() < 0.1 else _log(rng, max(1, top // 16), top)
            cost += n * n * heads * d
            if lens and cost > budget:
                break
            lens.append(n)
        if sum(lens) == 0:
            lens.append(top)
        return dict(op="attention", dtype=dtype, lens=",".join(map(str, lens)), tail=rng.choice([0, 0, 1, 70]), heads=heads, kv_heads=kv,
                    head_dim=d, causal_block=rng.choice([0, 1, 1, 5, 64, 196]), backward=rng.random() < 0.6)
    mats, cost = [], 0.0
    for _ in range(rng.randint(1, 4)):
        r, c = _log(rng, 8, 3000), _log(rng, 8, 3000)
        n = _log(rng, 1, max(1, min(24, int(4e10 / (min(r, c) ** 2 * max(r, c))))))
        mats.append(f"{n}x{r}x{c}")
    return dict(op="ortho", dtype=rng.choice(["f32", "f32", "bf16", "f16"]), mats=",".join(mats), steps=rng.choice([3, 5, 5, 6]))


# ---- inputs ---------------------------------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _grid_positions(text):
    dims = [int(v) for v in text.split("x")]
    axes = torch.meshgrid(*[torch.arange(n, device="cuda", dtype=torch.int32) for n in dims], indexing="ij")
    return torch.stack([a.reshape(-1) for a in axes], 1).contiguous()


def prepare(case, seed):
    g = _gen(seed)
    dt = DTYPES[case["dtype"]]
    s = dict(case)
    if case["op"] == "rotary":
        pos = _grid_positions(case["grid"])
        rows = case["clips"] * pos.shape[0]
        packed = torch.empty(rows, case["heads"] + case["pass_heads"], case["head_dim"], device="cuda", dtype=dt).normal_(generator=g)
        s.update(x=packed[:, :case["heads"]], pos=pos, axes_list=[int(v) for v in case["axes"].split("x")])
    elif case["op"] == "attention":
        lens = _lens(case["lens"])
        rows, h, kv, d = sum(lens) + case["tail"], case["heads"], case["kv_heads"], case["head_dim"]
        cu = [0]
        for n in lens:
            cu.append(cu[-1] + n)
        qkv = torch.empty(rows, h + 2 * kv, d, device="cuda", dtype=dt).normal_(generator=g)     # one projection's output
        s.update(q=qkv[:, :h], k=qkv[:, h:h + kv], v=qkv[:, h + kv:], cu=cu,
                 cu_dev=torch.tensor(cu, dtype=torch.int32, device="cuda"))
        if case["backward"]:
            s["dout"] = torch.empty(rows, h, d, device="cuda", dtype=dt).normal_(generator=g)
        if case["tail"]:
            # rows behind the last sequence stay as the caller left them, so such a caller brings its buffers
            s["buffers"] = dict(out=torch.zeros(rows, h, d, device="cuda", dtype=dt), lse=torch.zeros(h, rows, device="cuda"))
            s["grad_buffers"] = {n: torch.zeros(rows, m, d, device="cuda", dtype=dt) for n, m in (("dq", h), ("dk", kv), ("dv", kv))}
    else:
        mats = []
        for n, r, c in _mats(case["mats"]):
            # gradients of a layer: a few strong directions over a broad floor, of small size
            k = min(8, r, c)
            left = torch.empty(n, r, k, device="cuda").normal_(generator=g)
            right = torch.empty(n, k, c, device="cuda").normal_(generator=g)
            m = torch.empty(n, r, c, device="cuda").normal_(generator=g)
            mats.append((1e-3 * (m + torch.bmm(left, right))).to(dt))
        s["mats_list"] = mats
    return s


# ---- one pass -------------------------------------------------------------------------------------------------------

def run(state):
    op = state["op"]
    if own:
        import cora_amd as ca
        if op == "rotary":
            f = ca.rotary_backward if state["backward"] else ca.rotary
            return f(state["x"], state["pos"], state["axes_list"], theta=state["theta"], interleaved=state["interleaved"])
        if op == "attention":
            q, k, v = state["q"], state["k"], state["v"]
            kw = dict(cu_seqlens=state["cu_dev"], causal_block=state["causal_block"])
            out, lse = ca.attention(q, k, v, **kw, **state.get("buffers", {}))
            if not state["backward"]:
                return out, lse
            return (out,) + tuple(ca.attention_backward(state["dout"], q, k, v, out, lse, **kw, **state.get("grad_buffers", {})))
        return ca.orthogonalize(state["mats_list"], steps=state["steps"], coefficients=COEF, eps=EPS)
    if op == "rotary":
        return _plain_rotary(state)
    if op == "attention":
        return _plain_attention(state)
    return [_plain_ortho(m, state["steps"]) for m in state["mats_list"]]


def _plain_rotary(s):
    x, pos, d = s["x"], s["pos"], s["head_dim"]
    angles, first, second, start = [], [], [], 0
    for axis, n in enumerate(s["axes_list"]):
        i = torch.arange(n // 2, device="cuda", dtype=torch.float64)
        angles.append(pos[:, axis:axis + 1].double() * torch.pow(torch.tensor(s["theta"], device="cuda", dtype=torch.float64), -2.0 * i / n))
        i = torch.arange(n // 2, device="cuda")
        first.append(start + (2 * i if s["interleaved"] else i))
        second.append(start + (2 * i + 1 if s["interleaved"] else i + n // 2))
        start += n
    ang = torch.cat(angles, 1)
    sign = -1.0 if s["backward"] else 1.0
    clips = x.shape[0] // pos.shape[0]
    cos, sin = ang.cos().float().repeat(clips, 1)[:, None], (sign * ang.sin()).float().repeat(clips, 1)[:, None]
    ia, ib = torch.cat(first), torch.cat(second)
    y = x.float()
    a, b = y[..., ia], y[..., ib]
    out = y.clone()
    out[..., ia] = a * cos - b * sin
    out[..., ib] = a * sin + b * cos
    return out.to(x.dtype)


def _plain_attention(s):
    q, k, v, cu, block = s["q"], s["k"], s["v"], s["cu"], s["causal_block"]
    rows, h, d = q.shape
    kv = k.shape[1]
    scale = 1.0 / math.sqrt(d)
    out = torch.zeros(rows, h, d, device="cuda")
    lse = torch.zeros(h, rows, device="cuda")
    grads = None
    if s["backward"]:
        grads = [torch.zeros(t.shape, device="cuda") for t in (q, k, v)]
    for b, e in zip(cu[:-1], cu[1:]):
        n = e - b
        if n == 0:
            continue
        hidden = None
        if block:
            i = torch.arange(n, device="cuda") // block
            hidden = i[:, None] < i[None, :]
        # heads in groups whose score matrices fit comfortably
        step = max(1, min(kv, int(2e9 / (n * n * (h // kv)))))
        for k0 in range(0, kv, step):
            k1 = min(kv, k0 + step)
            g = h // kv
            qs = q[b:e, k0 * g:k1 * g].float().transpose(0, 1).contiguous()
            ks = k[b:e, k0:k1].float().transpose(0, 1).repeat_interleave(g, 0).contiguous()
            vs = v[b:e, k0:k1].float().transpose(0, 1).repeat_interleave(g, 0).contiguous()
            sc = torch.bmm(qs, ks.transpose(1, 2).contiguous()) * scale
            if hidden is not None:
                sc = sc.masked_fill(hidden, float("-inf"))
            m = sc.amax(2, keepdim=True)
            p = torch.exp(sc - m)
            del sc
            l = p.sum(2, keepdim=True)
            p = p / l
            lse[k0 * g:k1 * g, b:e] = (m + torch.log(l))[..., 0]
            o = torch.bmm(p, vs)
            out[b:e, k0 * g:k1 * g] = o.transpose(0, 1)
            if grads is None:
                continue
            do = s["dout"][b:e, k0 * g:k1 * g].float().transpose(0, 1).contiguous()
            dv = torch.bmm(p.transpose(1, 2).contiguous(), do)
            dp = torch.bmm(do, vs.transpose(1, 2).contiguous())
            ds = p * (dp - (do * o).sum(2, keepdim=True)) * scale
            del dp, p
            grads[0][b:e, k0 * g:k1 * g] = torch.bmm(ds, ks).transpose(0, 1)
            dk = torch.bmm(ds.transpose(1, 2).contiguous(), qs)
            grads[1][b:e, k0:k1] = dk.reshape(k1 - k0, g, n, d).sum(1).transpose(0, 1)
            grads[2][b:e, k0:k1] = dv.reshape(k1 - k0, g, n, d).sum(1).transpose(0, 1)
    out = out.to(q.dtype)
    return (out, lse) if grads is None else (out,) + tuple(t.to(q.dtype) for t in grads)


def _plain_ortho(m, steps):
    a, b, c = COEF
    x = m.float()
    x = x / (x.square().sum((1, 2), keepdim=True).sqrt() + EPS)
    tall = x.shape[1] > x.shape[2]
    if tall:
        x = x.transpose(1, 2).contiguous()
    for _ in range(steps):
        s = torch.bmm(x, x.transpose(1, 2).contiguous())
        x = a * x + torch.bmm(b * s + c * torch.bmm(s, s), x)
    return (x.transpose(1, 2).contiguous() if tall else x).to(m.dtype)


# ---- the same from the definitions, in 64 bits ----------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        x = s["x"]
        if x.numel() > 1_000_000_000:
            return None
        n_pos, off = s["pos"].shape[0], 0
        z = x.to(torch.float64).reshape(-1, n_pos, case["heads"], case["head_dim"])
        out = z.clone()
        for axis, n in enumerate(s["axes_list"]):
            for i in range(n // 2):
                ang = s["pos"][:, axis].to(torch.float64) * math.exp(-math.log(case["theta"]) * (2 * i) / n)
                if case["backward"]:
                    ang = -ang
                p0, p1 = (off + 2 * i, off + 2 * i + 1) if case["interleaved"] else (off + i, off + n // 2 + i)
                w = torch.polar(torch.ones_like(ang), ang)[None, :, None] * torch.complex(z[..., p0], z[..., p1])
                out[..., p0], out[..., p1] = w.real, w.imag
            off += n
        return out.reshape(x.shape)
    if case["op"] == "attention":
        return _exact_attention(s)
    if sum(n * min(r, c) ** 2 * max(r, c) for n, r, c in _mats(case["mats"])) * 30 > 2e14:
        return None
    res = []
    for stack in s["mats_list"]:
        done = []
        for g in stack.to(torch.float64):
            x = g / (torch.sqrt(torch.sum(g * g)) + EPS)
            for _ in range(case["steps"]):
                if x.shape[0] <= x.shape[1]:
                    t = x @ x.T
                    x = COEF[0] * x + COEF[1] * (t @ x) + COEF[2] * (t @ (t @ x))
                else:
                    t = x.T @ x
                    x = COEF[0] * x + COEF[1] * (x @ t) + COEF[2] * ((x @ t) @ t)
            done.append(x)
        res.append(torch.stack(done))
    return res


def _exact_attention(s):
    q, k, v = (s[n].to(torch.float64) for n in ("q", "k", "v"))
    rows, h, d = q.shape
    group = h // k.shape[1]
    if sum(float(n) ** 2 for n in _lens(s["lens"])) * h * d > 2e12:
        return None
    out, lse = torch.zeros_like(q), torch.zeros(h, rows, dtype=torch.float64, device="cuda")
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for b, e in zip(s["cu"][:-1], s["cu"][1:]):
        # whole blocks of a sequence share what they see; a chunk of rows at a time bounds the memory
        for head in range(h):
            kk, vv = k[b:e, head // group], v[b:e, head // group]
            for r0 in range(b, e, 8192):
                r1 = min(e, r0 + 8192)
                t = q[r0:r1, head] @ kk.T / math.sqrt(d)
                if s["causal_block"]:
                    last = (torch.arange(r0 - b, r1 - b, device="cuda") // s["causal_block"] + 1) * s["causal_block"]
                    t.masked_fill_(torch.arange(e - b, device="cuda")[None, :] >= last[:, None], -math.inf)
                z = torch.logsumexp(t, 1)
                lse[head, r0:r1] = z
                t = torch.exp(t - z[:, None])
                out[r0:r1, head] = t @ vv
                if s["backward"]:
                    go = s["dout"][r0:r1, head].to(torch.float64)
                    dv[b:e, head // group] += t.T @ go
                    t = t * (go @ vv.T - (go * out[r0:r1, head]).sum(1)[:, None]) / math.sqrt(d)
                    dq[r0:r1, head] = t @ kk
                    dk[b:e, head // group] += t.T @ q[r0:r1, head]
    return (out, dq, dk, dv) if s["backward"] else (out, lse)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------

def work(case):
    eb = BYTES[case["dtype"]]
    if case["op"] == "rotary":
        pos = math.prod(int(v) for v in case["grid"].split("x"))
        n = case["clips"] * pos * case["heads"] * case["head_dim"]
        return {"bytes": 2 * n * eb + pos * 4 * len(case["grid"].split("x")), "flops": 3 * n}
    if case["op"] == "attention":
        lens, h, kv, d, block = _lens(case["lens"]), case["heads"], case["kv_heads"], case["head_dim"], case["causal_block"]
        pairs = 0
        for n in lens:
            if block:
                full, rest = divmod(n, block)
                pairs += block * block * full * (full + 1) // 2 + rest * n
            else:
                pairs += n * n
        rows = sum(lens)
        nbytes = rows * d * (2 * h + 2 * kv) * eb + rows * h * 4
        flops = 4 * pairs * h * d
        if case["backward"]:
            nbytes += rows * d * (4 * h + 4 * kv) * eb      # q, k, v, dout read; dq, dk, dv written; out read again
            nbytes += rows * h * 4
            flops += 10 * pairs * h * d
        return {"bytes": nbytes, "flops": flops}
    nbytes = flops = 0
    for n, r, c in _mats(case["mats"]):
        lo, hi = min(r, c), max(r, c)
        nbytes += 2 * n * r * c * eb
        flops += n * case["steps"] * (3 * lo * lo * hi + lo ** 3)       # x x^T and its square are symmetric: half of each
    return {"bytes": nbytes, "flops": flops}
