"""Stand-alone operators on torch tensors of one GPU: rotary positions over several axes, attention over packed sequences
with its backward pass, and the Newton-Schulz orthogonalisation of weight updates.

They run the kernels a `TransformerDecoder` uses for `pos_encoding="rotary"`, `causal_frames=True` and the `muon` weight
optimiser, on the caller's own tensors.  The C entry points are `cora_rotary`, `cora_attention`, `cora_attention_backward`
and `cora_orthogonalize` of include/cora_hip.h, which states the formulas.  Types: float32, bfloat16, float16.  Launches go
to torch's current stream of the tensors' device and nothing is synchronised, so the calls can be captured into a graph.
There is no autograd: gradients come from the `*_backward` calls, and tensors that require one while torch records it, or that
carry a forward-mode tangent, are refused.  The reference has none of these operators.

Small calls last some 5 us on the GPU, so the checks below are kept to a few lookups per tensor."""
from __future__ import annotations

import ctypes as C
from typing import Optional, Sequence

from . import _lib

_torch = None        # imported by the first call: the rest of the package works without torch
_codes = {}
_stream = None
_duals = None
_MOST = 2 ** 31 - 1  # of the C structures' 32-bit fields, which ctypes fills with a number's lower bits


def _load():
    global _torch, _stream, _duals
    import torch
    from torch.autograd import forward_ad
    _codes.update({torch.float32: 0, torch.bfloat16: 1, torch.float16: 2})
    _stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else \
        (lambda index: torch.cuda.current_stream(index).cuda_stream)
    _duals = forward_ad
    _torch = torch
    return torch


def _lead(t, name: str) -> int:
    """The call's first tensor: dtype code, if it is one these operators take."""
    torch = _torch or _load()
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be on a GPU, it is on {t.device}")
    code = _codes.get(t.dtype)
    if code is None:
        raise ValueError(f"{name}: dtype must be float32, bfloat16 or float16, got {t.dtype}")
    _no_grad(t, name)
    return code


def _no_grad(t, name: str) -> None:
    if t.requires_grad and _torch.is_grad_enabled():
        raise ValueError(f"{name} requires a gradient: these operators are not recorded by autograd; use the *_backward "
                         "calls under torch.no_grad(), or detach it")
    if _duals._current_level >= 0 and _duals.unpack_dual(t).tangent is not None:
        raise ValueError(f"{name} carries a tangent: these operators have no forward-mode derivative; take its primal")


def _like(t, name: str, lead, shape) -> None:
    """A further tensor: dtype and device of the first one, and the shape."""
    if not isinstance(t, _torch.Tensor):
        raise TypeError(f"{name} must be a torch tensor")
    if t.dtype is not lead.dtype or t.device != lead.device:
        raise ValueError(f"{name} is {t.dtype} on {t.device}, expected {lead.dtype} on {lead.device}")
    if t.shape != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    _no_grad(t, name)


def _table(t, name: str, lead, dtype, dims: int, what: str) -> None:
    """A contiguous index table or row statistic on the first tensor's device."""
    if not isinstance(t, _torch.Tensor) or t.dtype is not dtype or t.dim() != dims or t.device != lead.device or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {what} on {lead.device}")


def _heads(t, name: str):
    """(row, head) strides of [rows, heads, head_dim]."""
    rows, heads, d = t.shape
    row, head, last = t.stride()
    if last != 1 and d > 1:
        raise ValueError(f"{name}: the last dimension must be contiguous")
    # strides of dimensions of size one carry no meaning; give the kernels the packed ones
    if heads == 1:
        head = d
    if rows == 1:
        row = d
    return row, head


_axes = {}           # axes_dim -> its C array


def _axes_array(axes_dim):
    if not 1 <= len(axes_dim) <= 4:
        raise ValueError(f"axes_dim must name 1 to 4 axes, got {len(axes_dim)}")
    if not all(-_MOST <= n <= _MOST for n in axes_dim):
        raise ValueError(f"axes_dim must be positive, even and at most 128, got {axes_dim}")
    if len(_axes) >= 256:
        _axes.clear()
    return _axes.setdefault(axes_dim, (C.c_int32 * 4)(*axes_dim))


def _rotary(x, positions, axes_dim, theta, interleaved, out, backward):
    code = _lead(x, "x")
    if x.dim() != 3:
        raise ValueError(f"x must be [rows, heads, head_dim], got shape {tuple(x.shape)}")
    n_axes = len(axes_dim)
    axes = _axes.get(axes_dim := tuple(axes_dim)) or _axes_array(axes_dim)
    _table(positions, "positions", x, _torch.int32, 2, f"int32 tensor [n, {n_axes}]")
    rows, heads, d = x.shape
    if heads > _MOST or d > _MOST:
        raise ValueError(f"x has shape {tuple(x.shape)}: heads and head_dim must be below 2^31")
    n, width = positions.shape
    if width != n_axes:
        raise ValueError(f"positions must be a contiguous int32 tensor [n, {n_axes}], got {tuple(positions.shape)}")
    if rows and (n == 0 or rows % n):
        raise ValueError(f"{rows} rows are not a multiple of {n} positions")
    if out is None:
        out = _torch.empty((rows, heads, d), dtype=x.dtype, device=x.device)
    else:
        _like(out, "out", x, x.shape)
    if rows == 0 or heads == 0:
        return out
    xr, xh = _heads(x, "x")
    yr, yh = _heads(out, "out")
    a = _lib.CoraRotaryArgs(code, heads, d, n_axes, axes, 1 if interleaved else 0, backward, theta, rows, n,
                            positions.data_ptr(), x.data_ptr(), out.data_ptr(), xr, xh, yr, yh)
    index = x.get_device()
    _lib.check(_lib.load().cora_rotary(a, index, _stream(index)))
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


def _attention_inputs(q, k, v, cu_seqlens, seq_len, causal_block, scale):
    """The fields up to v of cora_attention_args, and the strides of q, k and v."""
    code = _lead(q, "q")
    if q.dim() != 3:
        raise ValueError(f"q must be [rows, heads, head_dim], got shape {tuple(q.shape)}")
    rows, heads, d = q.shape
    if not isinstance(k, _torch.Tensor) or k.dim() != 3 or k.shape[0] != rows or k.shape[2] != d:
        raise ValueError(f"k has shape {tuple(getattr(k, 'shape', ()))}, expected ({rows}, kv_heads, {d})")
    _like(k, "k", q, k.shape)
    _like(v, "v", q, k.shape)
    kv = k.shape[1]
    if heads < 1 or kv < 1 or heads % kv:
        raise ValueError(f"{heads} query heads are not a multiple of {kv} key heads")
    table = None
    if cu_seqlens is not None:
        if seq_len is not None:
            raise ValueError("give cu_seqlens or seq_len, not both")
        _table(cu_seqlens, "cu_seqlens", q, _torch.int32, 1, "int32 vector [sequences + 1]")
        n_seq, n, table = cu_seqlens.shape[0] - 1, 0, cu_seqlens.data_ptr()
        if n_seq < 0:
            raise ValueError("cu_seqlens must be a contiguous int32 vector [sequences + 1], it is empty")
    else:
        n = rows if seq_len is None else int(seq_len)
        if rows and (n < 1 or rows % n):
            raise ValueError(f"{rows} rows are not a multiple of seq_len {n}")
        n_seq = rows // n if rows else 0
    if heads > _MOST or kv > _MOST or d > _MOST or n_seq > _MOST:
        raise ValueError(f"heads {heads}, kv_heads {kv}, head_dim {d} and the number of sequences {n_seq} must be below 2^31")
    if not -_MOST <= causal_block <= _MOST:
        raise ValueError(f"causal_block must be 0 or positive and below 2^31, got {causal_block}")
    head = (code, heads, kv, d, n_seq, n, causal_block, (d or 1) ** -0.5 if scale is None else scale, rows, table,
            q.data_ptr(), k.data_ptr(), v.data_ptr())
    return head, _heads(q, "q") + _heads(k, "k") + _heads(v, "v")


def _check_lse(lse, q) -> None:
    _table(lse, "lse", q, _torch.float32, 2, f"float32 tensor {(q.shape[1], q.shape[0])}")
    _no_grad(lse, "lse")
    if lse.shape[0] != q.shape[1] or lse.shape[1] != q.shape[0]:
        raise ValueError(f"lse must be a contiguous float32 tensor {(q.shape[1], q.shape[0])}, got {tuple(lse.shape)}")


def attention(q, k, v, *, cu_seqlens=None, seq_len: Optional[int] = None, causal_block: int = 0,
              scale: Optional[float] = None, out=None, lse=None):
    """Attention over packed sequences; returns (out, lse).

    q [rows, heads, head_dim], k and v [rows, kv_heads, head_dim] (query head h reads key head h // (heads // kv_heads)),
    any strides with a contiguous last dimension and 16-byte aligned rows, so slices of one packed projection do.
    Sequence s owns rows cu_seqlens[s] .. cu_seqlens[s+1] - 1 (int32 on the GPU; lengths may differ, be 1 or 0), or every
    `seq_len` rows (default: all) are one.  `causal_block` 0: bidirectional; b: a token sees the tokens of its own and of
    earlier blocks of b tokens (1: causal; tokens per frame: frame-causal).  `scale` defaults to head_dim ** -0.5.
    What the mask hides does not count even if it is not finite; a row that sees a value that is not finite may come out as
    NaN in all its channels.  `lse` [heads, rows] float32 is the log of the softmax' denominator.  Rows of no sequence are left as they were in
    `out` and `lse` (undefined in freshly allocated ones)."""
    head, strides = _attention_inputs(q, k, v, cu_seqlens, seq_len, causal_block, scale)
    if out is None:
        out = _torch.empty(q.shape, dtype=q.dtype, device=q.device)
    else:
        _like(out, "out", q, q.shape)
    if lse is None:
        lse = _torch.empty((q.shape[1], q.shape[0]), dtype=_torch.float32, device=q.device)
    else:
        _check_lse(lse, q)
    a = _lib.CoraAttentionArgs(*head, out.data_ptr(), lse.data_ptr(), None, None, None, None, *strides, *_heads(out, "out"))
    index = q.get_device()
    _lib.check(_lib.load().cora_attention(a, index, _stream(index)))
    return out, lse


def attention_backward(dout, q, k, v, out, lse, *, cu_seqlens=None, seq_len: Optional[int] = None, causal_block: int = 0,
                       scale: Optional[float] = None, dq=None, dk=None, dv=None):
    """Gradients (dq, dk, dv) of `attention` for the gradient `dout` of its first result; `out`, `lse` and the options are
    the forward call's.  Gradients of shared key heads are summed over their query heads.  Rows of no sequence are left as
    they were in dq, dk and dv.  Results repeat bit for bit."""
    head, strides = _attention_inputs(q, k, v, cu_seqlens, seq_len, causal_block, scale)
    _like(dout, "dout", q, q.shape)
    _like(out, "out", q, q.shape)
    _check_lse(lse, q)

    def new(t, like, name):
        if t is None:
            return _torch.empty(like.shape, dtype=like.dtype, device=like.device)
        _like(t, name, like, like.shape)
        return t

    dq, dk, dv = new(dq, q, "dq"), new(dk, k, "dk"), new(dv, v, "dv")
    a = _lib.CoraAttentionArgs(*head, out.data_ptr(), lse.data_ptr(), dout.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                               *strides, *_heads(out, "out"), *_heads(dout, "dout"), *_heads(dq, "dq"), *_heads(dk, "dk"),
                               *_heads(dv, "dv"))
    lib, index = _lib.load(), q.get_device()
    need = lib.cora_attention_workspace(a)
    ws = _torch.empty(need, dtype=_torch.uint8, device=q.device)
    a.workspace, a.workspace_bytes = ws.data_ptr(), need
    _lib.check(lib.cora_attention_backward(a, index, _stream(index)))
    return dq, dk, dv


def _coefficients(coefficients, steps: int):
    c = [tuple(float(v) for v in t) for t in coefficients] if hasattr(coefficients[0], "__len__") else \
        [tuple(float(v) for v in coefficients)] * steps
    if len(c) != steps or any(len(t) != 3 for t in c):
        raise ValueError("coefficients must be (a, b, c) or one such triple for every step")
    return (C.c_float * (3 * steps))(*[v for t in c for v in t])


def _matrices(t, name: str):
    """(count, rows, cols, matrix stride, row stride) of [rows, cols] or [count, rows, cols]."""
    shape, strides = t.shape, t.stride()
    if len(shape) == 2:
        shape, strides = (1, *shape), (0, *strides)
    count, rows, cols = shape
    if strides[2] != 1 and cols > 1:
        raise ValueError(f"{name}: the last dimension must be contiguous")
    row = strides[1] if rows > 1 else cols
    return count, rows, cols, (strides[0] if count > 1 else rows * row), row


def orthogonalize(x, *, steps: int = 5, coefficients=(3.4445, -4.7750, 2.0315), eps: float = 1e-7, out=None):
    """Newton-Schulz orthogonalisation of matrices: x [rows, cols], a stack [count, rows, cols], or a list of either (one
    dtype, one device, any sizes; all are worked on together).  X = x / (|x|_F + eps), then `steps` times
    X <- a X + (b A + c A^2) X with A = X X^T, which drives the singular values towards 1.  `coefficients` is (a, b, c) or a
    triple for every step.  Returns new tensors of the same shapes, or fills `out` (which may be x itself)."""
    many = isinstance(x, (list, tuple))
    xs = x if many else [x]
    steps = int(steps)
    if not 1 <= steps <= 32:
        raise ValueError("steps must be 1 to 32")
    coef = _coefficients(coefficients, steps)
    if out is not None and (isinstance(out, (list, tuple)) != many or (many and len(out) != len(xs))):
        raise ValueError("out must match x: a tensor, or a list of as many tensors")
    outs = [None] * len(xs) if out is None else (list(out) if many else [out])
    if not xs:
        return outs
    code, first = _lead(xs[0], "x"), xs[0]
    stacks = []
    for i, t in enumerate(xs):
        _like(t, f"x[{i}]", first, getattr(t, "shape", None))
        if t.dim() not in (2, 3):
            raise ValueError(f"matrices must be [rows, cols] or [count, rows, cols], got shape {tuple(t.shape)}")
        if outs[i] is None:
            outs[i] = _torch.empty(t.shape, dtype=t.dtype, device=t.device)
        else:
            _like(outs[i], "out", t, t.shape)
        if t.numel():
            count, rows, cols, xm, xr = _matrices(t, "x")
            if count > _MOST or rows > _MOST or cols > _MOST:
                raise ValueError(f"x[{i}] has shape {tuple(t.shape)}: rows and columns must be at most 32768")
            ym, yr = _matrices(outs[i], "out")[3:]
            stacks.append((t.data_ptr(), outs[i].data_ptr(), xm, xr, ym, yr, count, rows, cols))
    if stacks:
        lib, index, n = _lib.load(), first.get_device(), len(stacks)
        table = (_lib.CoraMatrices * n)(*stacks)
        need = lib.cora_orthogonalize_workspace(code, table, n)
        ws = _torch.empty(max(need, 256), dtype=_torch.uint8, device=first.device)
        _lib.check(lib.cora_orthogonalize(code, table, n, steps, coef, eps, ws.data_ptr(), ws.numel(), index, _stream(index)))
    return outs if many else outs[0]
