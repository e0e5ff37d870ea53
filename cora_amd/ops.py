"""Stand-alone operators on torch tensors of one GPU: rotary positions over several axes, attention over packed sequences
with its backward pass, and the Newton-Schulz orthogonalisation of weight updates.

They run the kernels a `TransformerDecoder` uses for `pos_encoding="rotary"`, `causal_frames=True` and the `muon` weight
optimiser, on the caller's own tensors.  The C entry points are `cora_rotary`, `cora_attention`, `cora_attention_backward`
and `cora_orthogonalize` of include/cora_hip.h, which states the formulas.  Types: float32, bfloat16, float16.  Launches go
to torch's current stream of the tensors' device and nothing is synchronised, so the calls can be captured into a graph.
There is no autograd: gradients come from the `*_backward` calls, and tensors that require one are refused while torch
records it.  The reference has none of these operators."""
from __future__ import annotations

import ctypes as C
import math
from typing import List, Optional, Sequence, Tuple, Union

from . import _lib

_DTYPES = {"torch.float32": 0, "torch.bfloat16": 1, "torch.float16": 2}


def _torch():
    import torch
    return torch


def _dtype(t, name: str) -> int:
    code = _DTYPES.get(str(t.dtype))
    if code is None:
        raise ValueError(f"{name}: dtype must be float32, bfloat16 or float16, got {t.dtype}")
    return code


def _check(t, name: str, like=None, shape=None):
    """A GPU tensor, on the device and of the dtype of `like`, of the given shape."""
    torch = _torch()
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch tensor")
    if t.device.type != "cuda":
        raise ValueError(f"{name} must be on a GPU, it is on {t.device}")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} requires a gradient: these operators are not recorded by autograd; use the *_backward "
                         "calls under torch.no_grad(), or detach it")
    if like is not None and (t.device != like.device or t.dtype != like.dtype):
        raise ValueError(f"{name} is {t.dtype} on {t.device}, expected {like.dtype} on {like.device}")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    return t


def _heads(t, name: str) -> Tuple[int, int, int]:
    """Pointer and (row, head) strides of [rows, heads, head_dim]."""
    rows, heads, d = t.shape
    if d > 1 and t.stride(2) != 1:
        raise ValueError(f"{name}: the last dimension must be contiguous")
    # strides of dimensions of size one carry no meaning; give the kernels the packed ones
    head = t.stride(1) if heads > 1 else d
    row = t.stride(0) if rows > 1 else heads * head
    return t.data_ptr(), row, head


def _stream(t) -> C.c_void_p:
    return C.c_void_p(_torch().cuda.current_stream(t.device).cuda_stream)


def _rotary(x, positions, axes_dim, theta, interleaved, out, backward):
    torch = _torch()
    _check(x, "x")
    if x.dim() != 3:
        raise ValueError(f"x must be [rows, heads, head_dim], got shape {tuple(x.shape)}")
    axes = [int(n) for n in axes_dim]
    if not 1 <= len(axes) <= 4:
        raise ValueError(f"axes_dim must name 1 to 4 axes, got {len(axes)}")
    _check(positions, "positions")
    if positions.dtype != torch.int32 or positions.device != x.device or positions.dim() != 2 or positions.shape[1] != len(axes) \
            or not positions.is_contiguous():
        raise ValueError(f"positions must be a contiguous int32 tensor [n, {len(axes)}] on {x.device}")
    rows, heads, d = x.shape
    n = positions.shape[0]
    if rows and (n == 0 or rows % n):
        raise ValueError(f"{rows} rows are not a multiple of {n} positions")
    code = _dtype(x, "x")
    out = torch.empty(x.shape, dtype=x.dtype, device=x.device) if out is None else _check(out, "out", x, x.shape)
    if rows == 0 or heads == 0:
        return out
    a = _lib.CoraRotaryArgs(dtype=code, heads=heads, head_dim=d, n_axes=len(axes), axes_dim=(C.c_int32 * 4)(*axes),
                            interleaved=int(bool(interleaved)), backward=backward, theta=float(theta), rows=rows, pos_rows=n,
                            pos=positions.data_ptr())
    a.x, a.x_row, a.x_head = _heads(x, "x")
    a.y, a.y_row, a.y_head = _heads(out, "out")
    _lib.check(_lib.load().cora_rotary(C.byref(a), x.device.index, _stream(x)))
    return out


def rotary(x, positions, axes_dim: Sequence[int], *, theta: float = 10000.0, interleaved: bool = True, out=None):
    """Turn x [rows, heads, head_dim] by its rows' positions.

    `axes_dim[a]` consecutive channels of every head belong to axis a and their pair i turns by the angle
    positions[r, a] * theta ** (-2 i / axes_dim[a]); pairs are neighbouring channels (`interleaved`) or half the axis'
    channels apart.  Channels behind the last axis are copied.  `positions` is int32 [n, axes]; with n < rows row r takes
    positions[r % n] (equal grids packed one after another).  `out` may be x itself."""
    return _rotary(x, positions, axes_dim, theta, interleaved, out, 0)


def rotary_backward(dout, positions, axes_dim: Sequence[int], *, theta: float = 10000.0, interleaved: bool = True, out=None):
    """Gradient with respect to `rotary`'s x, given the one with respect to its result: the rotation back."""
    return _rotary(dout, positions, axes_dim, theta, interleaved, out, 1)


def _attention_args(q, k, v, cu_seqlens, seq_len, causal_block, scale):
    torch = _torch()
    _check(q, "q")
    if q.dim() != 3:
        raise ValueError(f"q must be [rows, heads, head_dim], got shape {tuple(q.shape)}")
    rows, heads, d = q.shape
    _check(k, "k", q)
    if k.dim() != 3 or k.shape[0] != rows or k.shape[2] != d:
        raise ValueError(f"k has shape {tuple(k.shape)}, expected ({rows}, kv_heads, {d})")
    _check(v, "v", q, k.shape)
    kv = k.shape[1]
    if heads < 1 or kv < 1 or heads % kv:
        raise ValueError(f"{heads} query heads are not a multiple of {kv} key heads")
    a = _lib.CoraAttentionArgs(dtype=_dtype(q, "q"), heads=heads, kv_heads=kv, head_dim=d, rows=rows,
                               causal_block=int(causal_block), scale=1.0 / math.sqrt(d) if scale is None else float(scale))
    if cu_seqlens is not None:
        if seq_len is not None:
            raise ValueError("give cu_seqlens or seq_len, not both")
        _check(cu_seqlens, "cu_seqlens")
        if cu_seqlens.dtype != torch.int32 or cu_seqlens.dim() != 1 or cu_seqlens.numel() < 1 or cu_seqlens.device != q.device \
                or not cu_seqlens.is_contiguous():
            raise ValueError(f"cu_seqlens must be a contiguous int32 vector [sequences + 1] on {q.device}")
        a.cu_seqlens, a.n_seq = cu_seqlens.data_ptr(), cu_seqlens.numel() - 1
    else:
        n = rows if seq_len is None else int(seq_len)
        if rows and (n < 1 or rows % n):
            raise ValueError(f"{rows} rows are not a multiple of seq_len {n}")
        a.seq_len, a.n_seq = n, rows // n if rows else 0
    a.q, a.q_row, a.q_head = _heads(q, "q")
    a.k, a.k_row, a.k_head = _heads(k, "k")
    a.v, a.v_row, a.v_head = _heads(v, "v")
    return a


def _lse(lse, q):
    torch = _torch()
    _check(lse, "lse")
    if lse.dtype != torch.float32 or lse.device != q.device or tuple(lse.shape) != (q.shape[1], q.shape[0]) or not lse.is_contiguous():
        raise ValueError(f"lse must be a contiguous float32 tensor {(q.shape[1], q.shape[0])} on {q.device}")
    return lse


def attention(q, k, v, *, cu_seqlens=None, seq_len: Optional[int] = None, causal_block: int = 0,
              scale: Optional[float] = None, out=None, lse=None):
    """Attention over packed sequences; returns (out, lse).

    q [rows, heads, head_dim], k and v [rows, kv_heads, head_dim] (query head h reads key head h // (heads // kv_heads)),
    any strides with a contiguous last dimension and 16-byte aligned rows, so slices of one packed projection do.
    Sequence s owns rows cu_seqlens[s] .. cu_seqlens[s+1] - 1 (int32 on the GPU; lengths may differ, be 1 or 0), or every
    `seq_len` rows (default: all) are one.  `causal_block` 0: bidirectional; b: a token sees the tokens of its own and of
    earlier blocks of b tokens (1: causal; tokens per frame: frame-causal).  `scale` defaults to head_dim ** -0.5.
    `lse` [heads, rows] float32 is the log of the softmax' denominator.  Rows of no sequence are left as they were in
    `out` and `lse` (undefined in freshly allocated ones)."""
    torch = _torch()
    a = _attention_args(q, k, v, cu_seqlens, seq_len, causal_block, scale)
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device) if out is None else _check(out, "out", q, q.shape)
    lse = torch.empty(q.shape[1], q.shape[0], dtype=torch.float32, device=q.device) if lse is None else _lse(lse, q)
    a.out, a.out_row, a.out_head = _heads(out, "out")
    a.lse = lse.data_ptr()
    _lib.check(_lib.load().cora_attention(C.byref(a), q.device.index, _stream(q)))
    return out, lse


def attention_backward(dout, q, k, v, out, lse, *, cu_seqlens=None, seq_len: Optional[int] = None, causal_block: int = 0,
                       scale: Optional[float] = None, dq=None, dk=None, dv=None):
    """Gradients (dq, dk, dv) of `attention` for the gradient `dout` of its first result; `out`, `lse` and the options are
    the forward call's.  Gradients of shared key heads are summed over their query heads.  Rows of no sequence are left as
    they were in dq, dk and dv.  Results repeat bit for bit."""
    torch = _torch()
    a = _attention_args(q, k, v, cu_seqlens, seq_len, causal_block, scale)
    _check(dout, "dout", q, q.shape)
    _check(out, "out", q, q.shape)
    a.lse = _lse(lse, q).data_ptr()
    a.out, a.out_row, a.out_head = _heads(out, "out")
    a.dout, a.dout_row, a.dout_head = _heads(dout, "dout")
    new = lambda t, like, name: (torch.empty(like.shape, dtype=like.dtype, device=like.device) if t is None
                                 else _check(t, name, like, like.shape))
    dq, dk, dv = new(dq, q, "dq"), new(dk, k, "dk"), new(dv, v, "dv")
    a.dq, a.dq_row, a.dq_head = _heads(dq, "dq")
    a.dk, a.dk_row, a.dk_head = _heads(dk, "dk")
    a.dv, a.dv_row, a.dv_head = _heads(dv, "dv")
    lib = _lib.load()
    need = lib.cora_attention_workspace(C.byref(a))
    ws = torch.empty(need, dtype=torch.uint8, device=q.device)
    a.workspace, a.workspace_bytes = ws.data_ptr(), need
    _lib.check(lib.cora_attention_backward(C.byref(a), q.device.index, _stream(q)))
    return dq, dk, dv


def _coefficients(coefficients, steps: int):
    c = [tuple(float(v) for v in t) for t in coefficients] if hasattr(coefficients[0], "__len__") else \
        [tuple(float(v) for v in coefficients)] * steps
    if len(c) != steps or any(len(t) != 3 for t in c):
        raise ValueError("coefficients must be (a, b, c) or one such triple for every step")
    return (C.c_float * (3 * steps))(*[v for t in c for v in t])


def orthogonalize(x, *, steps: int = 5, coefficients=(3.4445, -4.7750, 2.0315), eps: float = 1e-7, out=None):
    """Newton-Schulz orthogonalisation of matrices: x [rows, cols], a stack [count, rows, cols], or a list of either (one
    dtype, one device, any sizes; all are worked on together).  X = x / (|x|_F + eps), then `steps` times
    X <- a X + (b A + c A^2) X with A = X X^T, which drives the singular values towards 1.  `coefficients` is (a, b, c) or a
    triple for every step.  Returns new tensors of the same shapes, or fills `out` (which may be x itself)."""
    torch = _torch()
    many = isinstance(x, (list, tuple))
    xs = list(x) if many else [x]
    steps = int(steps)
    if not 1 <= steps <= 32:
        raise ValueError("steps must be 1 to 32")
    coef = _coefficients(coefficients, steps)
    if out is not None and (isinstance(out, (list, tuple)) != many or (many and len(out) != len(xs))):
        raise ValueError("out must match x: a tensor, or a list of as many tensors")
    outs = [None] * len(xs) if out is None else (list(out) if many else [out])
    stacks = (_lib.CoraMatrices * max(1, len(xs)))()
    n = 0
    for i, t in enumerate(xs):
        _check(t, f"x[{i}]" if many else "x", xs[0])
        if t.dim() not in (2, 3):
            raise ValueError(f"matrices must be [rows, cols] or [count, rows, cols], got shape {tuple(t.shape)}")
        outs[i] = torch.empty(t.shape, dtype=t.dtype, device=t.device) if outs[i] is None else _check(outs[i], "out", t, t.shape)
        if t.numel() == 0:
            continue
        s = stacks[n]
        n += 1
        views = [m if m.dim() == 3 else m.unsqueeze(0) for m in (t, outs[i])]
        s.count, s.rows, s.cols = views[0].shape
        for m, name in zip(views, ("x", "out")):
            if s.cols > 1 and m.stride(2) != 1:
                raise ValueError(f"{name}: the last dimension must be contiguous")
            row = m.stride(1) if s.rows > 1 else s.cols
            mat = m.stride(0) if s.count > 1 else s.rows * row
            if name == "x":
                s.x, s.x_row, s.x_mat = m.data_ptr(), row, mat
            else:
                s.y, s.y_row, s.y_mat = m.data_ptr(), row, mat
    if n:
        code, lib = _dtype(xs[0], "x"), _lib.load()
        need = lib.cora_orthogonalize_workspace(code, stacks, n)
        ws = torch.empty(max(need, 256), dtype=torch.uint8, device=xs[0].device)
        _lib.check(lib.cora_orthogonalize(code, stacks, n, steps, coef, float(eps), ws.data_ptr(), ws.numel(),
                                          xs[0].device.index, _stream(xs[0])))
    return outs if many else outs[0]
