"""Plain implementations in 64 bits of the stand-alone operators, with the error their kernels may make.

A rounding to type t is off by at most u = eps(t) / 2 of the value, an fp32 operation by U = 2^-24, exp2 / log2 and the
reciprocal by 2 U.  The bounds below follow these through the formulas element by element."""
import math

import torch

U = 2.0 ** -24


def half_eps(dtype):
    return torch.finfo(dtype).eps / 2


# ---- rotary ----------------------------------------------------------------------------------------------------------
def rotary_ref(x, pos, axes, theta, interleaved, backward=False):
    """(result, bound).  sin and cos: argument rounded (U) and evaluated to 2 ulp (4 U); each product one rounding, their
    sum one: 6 U (|a| + |b|) covers them; then the rounding of the result."""
    rows, heads, d = x.shape
    n = pos.shape[0]
    p = pos.double()[torch.arange(rows) % n]
    z = x.double()
    out, bound = z.clone(), torch.zeros_like(z)
    start = 0
    for a, w in enumerate(axes):
        for i in range(w // 2):
            c0, c1 = (start + 2 * i, start + 2 * i + 1) if interleaved else (start + i, start + w // 2 + i)
            turns = p[:, a] * (theta ** (-2.0 * i / w) / (2 * math.pi))
            ang = (turns - turns.round()) * 2 * math.pi
            # the angle of a far position is itself known to 2^-53 of its size only
            far = 2 * math.pi * turns.abs()[:, None] * 2.0 ** -50
            if backward:
                ang = -ang
            c, s = ang.cos()[:, None], ang.sin()[:, None]
            u, v = z[..., c0], z[..., c1]
            out[..., c0], out[..., c1] = u * c - v * s, u * s + v * c
            bound[..., c0] = bound[..., c1] = (6 * U + far) * (u.abs() + v.abs())
        start += w
    t = half_eps(x.dtype)
    return out, bound + t * out.abs() + (1e-40 if x.dtype == torch.float32 else 2.0 ** -25 if x.dtype == torch.float16 else 0.0)


# ---- attention -------------------------------------------------------------------------------------------------------
def visible(n, block):
    i = torch.arange(n)
    return torch.ones(n, n, dtype=torch.bool) if not block else i[None, :] // block <= i[:, None] // block


def attention_ref(q, k, v, cu, block, scale, dout=None):
    """dict of results and dict of bounds for out, lse (and dq, dk, dv), zeros outside the sequences.

    t_ij = scale q.k in fp32: off by (d + 2) U scale sum |q||k| =: dt, and U |t| for its scaling; p relative to its row's sum
    by e_p = 2 (dt + 4 U (1 + |t - lse|)) + (n + 8) U; p rounded to the inputs' type (u; fp16 additionally 2^-25, where it
    is denormal; fp32 not at all).  Sums of n terms add n U of the terms' absolute sum."""
    u = half_eps(q.dtype)
    up = 0.0 if q.dtype == torch.float32 else u
    ap = 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    tiny = {torch.float32: 1e-40, torch.bfloat16: 1e-40, torch.float16: 2.0 ** -25}[q.dtype]
    rows, heads, d = q.shape
    g = heads // k.shape[1]
    z = lambda t: torch.zeros(t.shape, dtype=torch.float64)
    r = dict(out=z(q), lse=torch.zeros(heads, rows, dtype=torch.float64))
    b = dict(out=z(q), lse=torch.zeros(heads, rows, dtype=torch.float64))
    if dout is not None:
        for n_, t in (("dq", q), ("dk", k), ("dv", v)):
            r[n_], b[n_] = z(t), z(t)
    for s0, s1 in zip(cu[:-1], cu[1:]):
        n = s1 - s0
        if n <= 0:
            continue
        vis = visible(n, block)
        for h in range(heads):
            Q, K, V = q[s0:s1, h].double(), k[s0:s1, h // g].double(), v[s0:s1, h // g].double()
            t = (Q @ K.T) * scale
            dt = (d + 2) * U * scale * (Q.abs() @ K.abs().T)
            t = t.masked_fill(~vis, -math.inf)
            lse = torch.logsumexp(t, 1)
            p = torch.exp(t - lse[:, None])
            away = torch.where(vis, (t - lse[:, None]).abs(), torch.zeros(()).double())
            big = torch.where(vis, t.abs(), torch.zeros(()).double()).amax(1, keepdim=True)
            dtm = torch.where(vis, dt, torch.zeros(()).double())
            ep = 2 * (dtm + dtm.amax(1, keepdim=True) + 4 * U * (1 + away + big)) + (n + 8) * U
            O = p @ V
            eo = u * O.abs() + (p * (ep + up) + ap * vis) @ V.abs() + (n + 4) * U * (p @ V.abs()) + tiny
            r["out"][s0:s1, h], b["out"][s0:s1, h] = O, eo
            r["lse"][h, s0:s1] = lse
            b["lse"][h, s0:s1] = dtm.amax(1) + (n + 16) * U + 4 * U * (big[:, 0] + lse.abs() + 1)
            if dout is None:
                continue
            G = dout[s0:s1, h].double()
            dp = G @ V.T
            delta = (G * O).sum(1, keepdim=True)
            ds = p * (dp - delta)
            edp = (d + 2) * U * (G.abs() @ V.abs().T)
            edl = (G.abs() * eo).sum(1, keepdim=True) + (d + 2) * U * (G * O).abs().sum(1, keepdim=True)
            floor = 2 * ap * G.abs().amax() * vis          # fp16 ds, in units of the largest gradient so far
            eds = (ds.abs() * (ep + up + 4 * U) + p * (edp + edl)) + floor
            r["dq"][s0:s1, h] = ds @ K * scale
            b["dq"][s0:s1, h] = u * r["dq"][s0:s1, h].abs() + scale * (eds @ K.abs() + (n + 4) * U * (ds.abs() @ K.abs())) + tiny
            r["dk"][s0:s1, h // g] += ds.T @ Q * scale
            b["dk"][s0:s1, h // g] += scale * (eds.T @ Q.abs() + (n * g + 4) * U * (ds.abs().T @ Q.abs())) + tiny
            r["dv"][s0:s1, h // g] += p.T @ G
            b["dv"][s0:s1, h // g] += (p * (ep + up) + ap * vis).T @ G.abs() + (n * g + 4) * U * (p.T @ G.abs()) + tiny
    if dout is not None:
        for n_ in ("dk", "dv"):
            b[n_] += u * r[n_].abs()
    return r, b


# ---- orthogonalisation -----------------------------------------------------------------------------------------------
def ortho_ref(G, steps, coef, eps):
    X = G.double()
    X = X / (X.square().sum().sqrt() + eps)
    tall = X.shape[0] > X.shape[1]
    X = X.T if tall else X
    for s in range(steps):
        a, b, c = coef[s] if hasattr(coef[0], "__len__") else coef
        A = X @ X.T
        X = a * X + (b * A + c * (A @ A)) @ X
    return X.T if tall else X


def ortho_bound(G, steps, coef, eps, dtype):
    """Relative Frobenius error the kernels may make: four times what independent errors of the size of every rounding they
    make do to the exact iteration, plus the result's own rounding.  Roundings: X, A, P to 22 bits (2^-22; lower halves
    times lower halves are left out, 2^-22 more of every product) and sums of K terms in fp32 (sqrt(K) U of the product of
    absolute values, as independent roundings add up); bfloat16 with min(rows, cols) >= 256: A from 11-bit X (2^-12 a factor),
    (b A + c A^2) X from 11-bit factors, a X from X itself."""
    gen = torch.Generator().manual_seed(1)
    noise = lambda t, rel: t * (1 + rel * (2 * torch.rand(t.shape, generator=gen, dtype=torch.float64) - 1))
    X = G.double()
    X = X / (X.square().sum().sqrt() + eps)
    X = X.T if X.shape[0] > X.shape[1] else X
    E = X.clone()
    m, n = X.shape
    eye = torch.eye(m, dtype=torch.float64)
    low = dtype == torch.bfloat16 and m >= 256

    def prod(L, R, rel):
        mag = (L.abs() @ R.abs()) * (2.0 ** -22 + math.sqrt(L.shape[1]) * U)
        return noise(L, rel) @ noise(R, rel) + mag * (2 * torch.rand(mag.shape, generator=gen, dtype=torch.float64) - 1)

    for s in range(steps):
        a, b, c = coef[s] if hasattr(coef[0], "__len__") else coef
        E = a * E + (b * (E @ E.T) + c * (E @ E.T) @ (E @ E.T)) @ E
        N = noise(X, 2.0 ** -22)
        A = prod(N, N.T, 2.0 ** -12 if low else 2.0 ** -22)
        A = noise((A + A.T) / 2, 2.0 ** -22)
        P = b * A + c * prod(A, A, 2.0 ** -22)
        X = a * N + prod(P, N, 2.0 ** -12) if low else prod(a * eye + P, N, 2.0 ** -22)
    norm = E.norm().clamp_min(1e-300)
    return 4 * float((X - E).norm() / norm) + half_eps(dtype) + 2.0 ** -22
