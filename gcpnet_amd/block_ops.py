"""Operators of a residual block for fp32, bf16 and fp16 rows: a Linear with bias, activation and residual in its epilogue (`linear_act`), and
the norms before and after a block fused with its gate and residual scale (`residual_norm`).

As in `ops`: GPU tensors and libgcpnet_hip.so only, no fallback; the arithmetic between the loads and the stores is fp32."""
from __future__ import annotations

import contextlib
import ctypes as C
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import ACT, NORM, TYPE_BF16, TYPE_F16, TYPE_F32, BlockNorm, LinearDesc, check
from .ops import _stream

Tensor = torch.Tensor
TYPES = {torch.float32: TYPE_F32, torch.bfloat16: TYPE_BF16, torch.float16: TYPE_F16}


def _ptr(t: Optional[Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _on(t: Tensor):
    """The launches of an operator go to the device of its tensors, whatever the current one is."""
    return contextlib.nullcontext() if t.device.index == torch.cuda.current_device() else torch.cuda.device(t.device)


def _rows(t: Tensor) -> Tensor:
    """[..., d] as [rows, d] with unit column stride and any row stride; a copy only where no such view exists."""
    d = t.shape[-1]
    if t.dim() != 2:
        try:
            t = t.view(-1, d) if t.numel() else t.reshape(t.numel() // max(d, 1), d)
        except RuntimeError:
            t = t.contiguous().view(-1, d)
    return t if t.stride(1) == 1 or d == 1 else t.contiguous()


def _check(t, name: str, like: Tensor, shape=None, dtypes=None) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
    if t.device != like.device:
        raise _lib.GcpnetHipError(f"{name} is on {t.device}, not on {like.device}")
    if t.dtype not in (dtypes or (like.dtype,)):
        raise TypeError(f"{name} must be {' or '.join(str(d) for d in dtypes or (like.dtype,))}, got {t.dtype}")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")


def _check_first(x, name: str) -> None:
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{name} must be a tensor, got {type(x).__name__}")
    if not x.is_cuda:
        raise _lib.GcpnetHipError(f"{name} must live on the GPU: gcpnet_amd has no CPU path")
    if x.dtype not in TYPES:
        raise TypeError(f"{name} must be float32, bfloat16 or float16, got {x.dtype}")
    if x.dim() < 1:
        raise ValueError(f"{name} must have at least one dimension")


# ==============================================================================================================
# norms before and after a block, with its gate and residual scale
# ==============================================================================================================
class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, cfg, x, y, gate, post_w, post_b, pre_w, pre_b):
        post, pre, act, scale, slope, eps = cfg
        x2 = _rows(x)
        y2 = None if y is None else _rows(y)
        channel = gate is not None and gate.dim() == 1
        g2 = None if gate is None else gate.contiguous() if channel else _rows(gate)
        rows, d = x2.shape
        if g2 is not None and not channel and g2.stride(0) == 0 and rows > 1:
            g2 = g2.contiguous()
        ws = [None if w is None else w.contiguous() for w in (post_w, post_b, pre_w, pre_b)]
        need = any(ctx.needs_input_grad)
        n = BlockNorm()
        n.rows, n.d, n.type = rows, d, TYPES[x.dtype]
        n.param_type = next((TYPES[w.dtype] for w in ws if w is not None), n.type)
        n.x, n.y, n.gate = x2.data_ptr(), _ptr(y2), _ptr(g2)
        n.x_ld, n.y_ld, n.gate_ld = x2.stride(0), 0 if y2 is None else y2.stride(0), 0 if g2 is None or channel else d if rows == 1 else g2.stride(0)
        n.post_w, n.post_b, n.pre_w, n.pre_b = (_ptr(w) for w in ws)
        n.post, n.pre, n.act, n.scale, n.slope, n.eps = NORM[post], NORM[pre], ACT[act], scale, slope, eps
        with _on(x):
            s = x.new_empty(x.shape) if y is not None else None
            h = x.new_empty(x.shape) if pre is not None else None
            stats = torch.empty((rows, 4), dtype=torch.float32, device=x.device) if need and (post or pre) else None
            check(_lib.load().gcpnet_block_norm_forward(C.byref(n), _ptr(s), _ptr(h), _ptr(stats), _stream()), "residual_norm")
        if need:
            ctx.save_for_backward(y2, s if s is not None else x2, g2, stats, *ws)
            ctx.desc, ctx.channel = n, channel
            ctx.shapes = (x.shape, None if gate is None else gate.shape)
        ctx.set_materialize_grads(False)
        return s, h

    @staticmethod
    @once_differentiable
    def backward(ctx, ds, dh):
        y2, s, g2, stats, *ws = ctx.saved_tensors
        shape, gate_shape = ctx.shapes
        n = ctx.desc
        none = (None,) * 8
        if ds is None and dh is None:
            return none
        ds, dh = (None if g is None else g.contiguous() for g in (ds, dh))
        _, need_x, need_y, need_gate, *need_w = ctx.needs_input_grad
        s2 = s.view(n.rows, n.d) if s.is_contiguous() else s
        b = BlockNorm.from_buffer_copy(n)
        b.x, b.x_ld = None, s2.stride(0)
        lib = _lib.load()
        with _on(s):
            new = lambda want, like: torch.empty(like, dtype=s.dtype, device=s.device) if want else None  # noqa: E731
            dx, dy, dgate = new(need_x, shape), new(need_y and y2 is not None, shape), new(need_gate and g2 is not None, gate_shape)
            dws = [torch.empty_like(w) if w is not None and want else None for w, want in zip(ws, need_w)]
            scratch = None
            if any(w is not None for w in dws) or (dgate is not None and ctx.channel):
                scratch = torch.empty(max(1, int(lib.gcpnet_block_norm_backward_scratch(n.rows, n.d))), dtype=torch.float32, device=s.device)
            check(lib.gcpnet_block_norm_backward(C.byref(b), s2.data_ptr(), _ptr(stats), _ptr(ds), _ptr(dh), _ptr(dx), _ptr(dy), _ptr(dgate),
                                                 *(_ptr(w) for w in dws), _ptr(scratch), _stream()), "residual_norm backward")
        return (None, dx, dy, dgate, *dws)


def residual_norm(x: Tensor, y: Optional[Tensor] = None, gate: Optional[Tensor] = None, *, scale: float = 1.0, gate_act: Optional[str] = None,
                  slope: float = 1e-2, post: Optional[str] = None, post_weight: Optional[Tensor] = None, post_bias: Optional[Tensor] = None,
                  pre: Optional[str] = "layer", pre_weight: Optional[Tensor] = None, pre_bias: Optional[Tensor] = None,
                  eps: float = 1e-5) -> Tuple[Tensor, Optional[Tensor]]:
    """The end of one residual block and the norm that begins the next, in one launch each way:

        u = post(y);   s = x + scale * gate_act(gate) * u;   h = pre(s);   returns (s, h)

    x, y: [..., d] rows of fp32, bf16 or fp16, the residual stream and a block's output; without y, s is x (a norm alone).
    gate: [d], one value per channel, or of y's shape.  post / pre: "layer", "rms" or None (without pre, h is None), with optional weights
    and biases [d] of x's type or fp32 (all of one type).  d up to 16384.  Row strides are taken as they are, other layouts are copied.
    Gradients flow to every tensor; sums over rows are formed in a fixed order, so a run repeats bit for bit."""
    _check_first(x, "x")
    d = x.shape[-1]
    if d < 1 or d > 16384:
        raise ValueError(f"residual_norm: rows of 1 to 16384 elements, got {d}")
    if post not in NORM or pre not in NORM or gate_act not in ACT:
        raise ValueError(f"residual_norm: post and pre are 'layer', 'rms' or None and gate_act one of {sorted(k for k in ACT if k)}, "
                         f"got {post!r}, {pre!r}, {gate_act!r}")
    if not eps >= 0:
        raise ValueError(f"residual_norm: eps must not be negative, got {eps}")
    if y is None and (gate is not None or post is not None):
        raise ValueError("residual_norm: a gate or a post norm needs y")
    if y is None and pre is None:
        raise ValueError("residual_norm: nothing to do without y and without pre")
    if y is not None:
        _check(y, "y", x, x.shape)
    if gate is not None:
        _check(gate, "gate", x, (d,) if gate.dim() == 1 else x.shape)
    first = None
    for w, name, kind in ((post_weight, "post_weight", post), (post_bias, "post_bias", post), (pre_weight, "pre_weight", pre), (pre_bias, "pre_bias", pre)):
        if w is None:
            continue
        if kind is None:
            raise ValueError(f"residual_norm: {name} without its norm")
        _check(w, name, x, (d,), (x.dtype, torch.float32) if first is None else (first,))
        first = w.dtype
    s, h = _ResidualNorm.apply((post, pre, gate_act, float(scale), float(slope), float(eps)), x, y, gate, post_weight, post_bias, pre_weight, pre_bias)
    return (x if y is None else s), h


# ==============================================================================================================
# Linear with bias, activation and residual
# ==============================================================================================================
class _LinearAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, cfg, x, weight, bias, residual):
        act, slope = cfg
        x2, w2, r2 = _rows(x), _rows(weight), None if residual is None else _rows(residual)
        b2 = None if bias is None else bias.contiguous()
        rows, k = x2.shape
        n = w2.shape[0]
        need = any(ctx.needs_input_grad[1:4])
        q = LinearDesc()
        q.rows, q.k, q.n, q.type, q.act, q.slope = rows, k, n, TYPES[x.dtype], ACT[act], slope
        q.bias_type = q.type if b2 is None else TYPES[b2.dtype]
        q.x, q.w, q.bias, q.x_ld, q.w_ld = x2.data_ptr(), w2.data_ptr(), _ptr(b2), x2.stride(0), w2.stride(0)
        lib = _lib.load()
        with _on(x):
            y = torch.empty((*x.shape[:-1], n), dtype=x.dtype, device=x.device)
            z = torch.empty((rows, n), dtype=x.dtype, device=x.device) if need and act is not None else None
            space = int(lib.gcpnet_linear_act_workspace(rows, k, n, q.type, 0))
            ws = torch.empty(space, dtype=torch.float32, device=x.device) if space > 0 else None
            check(lib.gcpnet_linear_act_forward(C.byref(q), _ptr(r2), 0 if r2 is None else r2.stride(0), y.data_ptr(), _ptr(z), _ptr(ws), _stream()),
                  "linear_act")
        if need:
            ctx.save_for_backward(x2, w2, z)
            ctx.desc, ctx.shapes, ctx.bias_dtype = q, (x.shape, weight.shape), None if b2 is None else b2.dtype
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        _, need_x, need_w, need_b, need_r = ctx.needs_input_grad
        if not (need_x or need_w or need_b):
            return None, None, None, None, dy if need_r else None
        x2, w2, z = ctx.saved_tensors
        q = ctx.desc
        g2 = _rows(dy)
        lib = _lib.load()
        with _on(x2):
            new = lambda shape, dtype=x2.dtype: torch.empty(shape, dtype=dtype, device=x2.device)  # noqa: E731
            dx = new(ctx.shapes[0]) if need_x else None
            dw = new(ctx.shapes[1]) if need_w else None
            db = new((q.n,), ctx.bias_dtype) if need_b else None
            dz = None if z is None else new((q.rows, q.n))
            space = int(lib.gcpnet_linear_act_workspace(q.rows, q.k, q.n, q.type, 1))
            ws = new((space,), torch.float32) if space > 0 else None
            check(lib.gcpnet_linear_act_backward(C.byref(q), _ptr(z), g2.data_ptr(), g2.stride(0), _ptr(dz), _ptr(dx), _ptr(dw), _ptr(db), _ptr(ws),
                                                 _stream()), "linear_act backward")
        return None, dx, dw, db, dy if need_r else None


def linear_act(x: Tensor, weight: Tensor, bias: Optional[Tensor] = None, act: Optional[str] = None, residual: Optional[Tensor] = None,
               slope: float = 1e-2) -> Tensor:
    """act(x @ weight^T + bias) + residual, rounded once: [..., k] x [n, k] -> [..., n] in one launch (two where k is split).

    x, weight, residual: one type of fp32, bf16 and fp16; bias that type or fp32; act as in `get_nonlinearity` or None; any sizes from one row and
    one column on.  Sums are fp32 (fp32 operands on the fp32 matrix instructions: no shorter terms).  Row strides are taken as they are, other
    layouts are copied.  The backward keeps the pre-activation in x's type, and rounds its gradient to that type as an operand of the products for
    x and weight; the bias gradient is summed unrounded.  All sums have a fixed order, so a run repeats bit for bit."""
    _check_first(x, "x")
    _check(weight, "weight", x)
    if weight.dim() != 2 or weight.shape[1] != x.shape[-1] or weight.shape[0] < 1 or weight.shape[1] < 1:
        raise ValueError(f"linear_act: weight must be [n, {x.shape[-1]}] with at least one row and column, got {tuple(weight.shape)}")
    if act not in ACT:
        raise ValueError(f"linear_act: act is None or one of {sorted(k for k in ACT if k)}, got {act!r}")
    n = weight.shape[0]
    if bias is not None:
        _check(bias, "bias", x, (n,), (x.dtype, torch.float32))
    if residual is not None:
        _check(residual, "residual", x, (*x.shape[:-1], n))
    return _LinearAct.apply((act, float(slope)), x, weight, bias, residual)
