"""Operators of a residual block for fp32, bf16 and fp16 rows: a Linear with bias, activation and residual in its epilogue (`linear_act`), and
the norms before and after a block fused with its gate and residual scale (`residual_norm`).

As in `ops`: GPU tensors and libgcpnet_hip.so only, no fallback; the arithmetic between the loads and the stores is fp32."""
from __future__ import annotations

import contextlib
import ctypes as C
from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import ACT, NORM, TYPE_BF16, TYPE_F16, TYPE_F32, BlockNorm, LinearDesc, check
from .ops import _stream

Tensor = torch.Tensor
TYPES = {torch.float32: TYPE_F32, torch.bfloat16: TYPE_BF16, torch.float16: TYPE_F16}


def _ptr(t: Optional[Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


_HERE = contextlib.nullcontext()


def _on(t: Tensor):
    """The launches of an operator go to the device of its tensors, whatever the current one is.  (In a backward autograd has seen to it.)"""
    return _HERE if t.get_device() == torch._C._cuda_getDevice() else torch.cuda.device(t.device)


def _backward(body):
    """A backward that autograd may not differentiate again: with a graph asked for, the wrapper that makes such a use raise."""
    once = once_differentiable(body)

    def backward(ctx, *grads):
        _refuse_tangents(grads)
        return once(ctx, *grads) if torch.is_grad_enabled() else body(ctx, *grads)

    return staticmethod(backward)


def _refuse_tangents(tensors) -> None:
    """The kernels take values only: a tangent of forward mode would be lost without a word."""
    # (the level, a global of that module, is -1 outside forward mode: nothing to look for then)
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError("gcpnet_amd: linear_act and residual_norm have no forward-mode derivatives")


def _wants_grad(tensors) -> bool:
    _refuse_tangents(tensors)
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _rows(t: Tensor) -> Tensor:
    """[..., d] as [rows, d] with unit column stride and any row stride; a copy only where no such view exists."""
    if t.dim() != 2:
        d = t.shape[-1]
        try:
            t = t.view(-1, d) if t.numel() else t.reshape(t.numel() // max(d, 1), d)
        except RuntimeError:
            t = t.contiguous().view(-1, d)
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _check(t, name: str, like: Tensor, shape=None, also=None) -> None:
    """A tensor on like's device, of its type (or `also`) and of the given shape."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
    if t.get_device() != like.get_device():
        raise _lib.GcpnetHipError(f"{name} is on {t.device}, not on {like.device}")
    if t.dtype is not like.dtype and t.dtype is not also:
        raise TypeError(f"{name} must be {like.dtype}{'' if also is None else f' or {also}'}, got {t.dtype}")
    if shape is not None and t.shape != shape:
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
def _norm_forward(cfg, x, y, gate, weights, need):
    """The launch: s, h, and what a backward keeps."""
    post, pre, act, scale, slope, eps = cfg
    x2 = _rows(x)
    y2 = None if y is None else _rows(y)
    channel = gate is not None and gate.dim() == 1
    g2 = None if gate is None else gate.contiguous() if channel else _rows(gate)
    rows, d = x2.shape
    if g2 is not None and not channel and g2.stride(0) == 0 and rows > 1:
        g2 = g2.contiguous()
    ws = [None if w is None else w.contiguous() for w in weights]
    kind = TYPES[x.dtype]
    n = BlockNorm(rows, d, kind, next((TYPES[w.dtype] for w in ws if w is not None), kind), x2.data_ptr(), _ptr(y2), _ptr(g2), x2.stride(0),
                  0 if y2 is None else y2.stride(0), 0 if g2 is None or channel else d if rows == 1 else g2.stride(0), *map(_ptr, ws), NORM[post],
                  NORM[pre], ACT[act], scale, slope, eps)
    with _on(x):
        s = x.new_empty(x.shape) if y is not None else None
        h = x.new_empty(x.shape) if pre is not None else None
        stats = torch.empty((rows, 4), dtype=torch.float32, device=x.device) if need and (post or pre) else None
        check(_lib.load().gcpnet_block_norm_forward(C.byref(n), _ptr(s), _ptr(h), _ptr(stats), _stream()), "residual_norm")
    return s, h, (n, channel, (x2 if pre else None, y2, g2, stats, *ws))


def _norm_backward(ctx, ds, dh):
    x2, y2, g2, stats, *ws = ctx.saved_tensors
    shape, gate_shape = ctx.shapes
    n = ctx.desc
    if ds is None and dh is None:
        return (None,) * 8
    ds, dh = (None if g is None else g.contiguous() for g in (ds, dh))
    like = dh if ds is None else ds
    _, need_x, need_y, need_gate, *need_w = ctx.needs_input_grad
    # (addresses anew: what was saved may have been elsewhere meanwhile)
    b = BlockNorm(n.rows, n.d, n.type, n.param_type, _ptr(x2), _ptr(y2), _ptr(g2), 0 if x2 is None else x2.stride(0), 0 if y2 is None else y2.stride(0),
                  0 if g2 is None or ctx.channel else n.d if n.rows == 1 else g2.stride(0), *map(_ptr, ws), n.post, n.pre, n.act, n.scale, n.slope,
                  n.eps)
    lib = _lib.load()
    new = lambda want, size: like.new_empty(size) if want else None  # noqa: E731
    dx, dy = new(need_x, shape), new(need_y and y2 is not None, shape)
    need_gate = need_gate and g2 is not None
    dgate = new(need_gate and not ctx.channel, gate_shape)
    dws = [None] * 4
    wanted = [i for i in range(4) if need_w[i] and ws[i] is not None]
    dtype = ws[wanted[0]].dtype if wanted else like.dtype
    together = need_gate and ctx.channel and dtype == like.dtype  # (one allocation for the short ones)
    if wanted or together:
        short = iter(like.new_empty((len(wanted) + together, n.d), dtype=dtype).unbind())
        for i in wanted:
            dws[i] = next(short)
        if together:
            dgate = next(short)
    if need_gate and dgate is None:
        dgate = new(True, gate_shape)
    scratch = None
    if wanted or (dgate is not None and ctx.channel):
        scratch = torch.empty(max(1, int(lib.gcpnet_block_norm_backward_scratch(C.byref(b)))), dtype=torch.float32, device=like.device)
    check(lib.gcpnet_block_norm_backward(C.byref(b), _ptr(stats), _ptr(ds), _ptr(dh), _ptr(dx), _ptr(dy), _ptr(dgate),
                                         *map(_ptr, dws), _ptr(scratch), _stream()), "residual_norm backward")
    return (None, dx, dy, dgate, *dws)


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, cfg, x, y, gate, *weights):
        s, h, (ctx.desc, ctx.channel, keep) = _norm_forward(cfg, x, y, gate, weights, True)
        ctx.save_for_backward(*keep)
        ctx.shapes = (x.shape, None if gate is None else gate.shape)
        ctx.set_materialize_grads(False)
        return s, h

    backward = _backward(_norm_backward)


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
        _check(w, name, x, (d,), torch.float32)
        first = first or w.dtype
        if w.dtype is not first:
            raise TypeError(f"residual_norm: weights and biases of one type, got {first} and {w.dtype}")
    cfg, weights = (post, pre, gate_act, float(scale), float(slope), float(eps)), (post_weight, post_bias, pre_weight, pre_bias)
    if _wants_grad((x, y, gate, *weights)):
        s, h = _ResidualNorm.apply(cfg, x, y, gate, *weights)
    else:
        s, h, _ = _norm_forward(cfg, x, y, gate, weights, False)
    return (x if y is None else s), h


# ==============================================================================================================
# Linear with bias, activation and residual
# ==============================================================================================================
def _linear_forward(cfg, x, weight, bias, residual, need):
    """The launch: y, and what a backward keeps."""
    act, slope = cfg
    x2, w2, r2 = _rows(x), _rows(weight), None if residual is None else _rows(residual)
    b2 = None if bias is None else bias.contiguous()
    rows, k = x2.shape
    n = w2.shape[0]
    kind = TYPES[x.dtype]
    q = LinearDesc(rows, k, n, kind, kind if b2 is None else TYPES[b2.dtype], ACT[act], slope, x2.data_ptr(), w2.data_ptr(), _ptr(b2), x2.stride(0),
                   w2.stride(0))
    lib = _lib.load()
    with _on(x):
        y = x.new_empty((*x.shape[:-1], n))
        z = x.new_empty((rows, n)) if need and act is not None else None
        space = lib.gcpnet_linear_act_workspace(C.byref(q), 0)
        ws = torch.empty(space, dtype=torch.float32, device=x.device) if space > 0 else None
        check(lib.gcpnet_linear_act_forward(C.byref(q), _ptr(r2), 0 if r2 is None else r2.stride(0), y.data_ptr(), _ptr(z), _ptr(ws), _stream()),
              "linear_act")
    return y, q, (x2, w2, z)


def _linear_backward(ctx, dy):
    _, need_x, need_w, need_b, need_r = ctx.needs_input_grad
    if not (need_x or need_w or need_b):
        return None, None, None, None, dy if need_r else None
    x2, w2, z = ctx.saved_tensors
    d = ctx.desc  # (its addresses anew: what was saved may have been elsewhere meanwhile)
    q = LinearDesc(d.rows, d.k, d.n, d.type, d.bias_type, d.act, d.slope, x2.data_ptr(), w2.data_ptr(), None, x2.stride(0), w2.stride(0))
    g2 = _rows(dy)
    lib = _lib.load()
    dx = x2.new_empty(ctx.shapes[0]) if need_x else None
    dw = x2.new_empty(ctx.shapes[1]) if need_w else None
    db = x2.new_empty(q.n, dtype=ctx.bias_dtype) if need_b else None
    space = lib.gcpnet_linear_act_workspace(C.byref(q), 1)
    ws = x2.new_empty(space, dtype=torch.float32) if space > 0 else None
    check(lib.gcpnet_linear_act_backward(C.byref(q), _ptr(z), g2.data_ptr(), g2.stride(0), _ptr(dx), _ptr(dw), _ptr(db), _ptr(ws),
                                         _stream()), "linear_act backward")
    return None, dx, dw, db, dy if need_r else None


class _LinearAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, cfg, x, weight, bias, residual):
        y, ctx.desc, keep = _linear_forward(cfg, x, weight, bias, residual, any(ctx.needs_input_grad[1:4]))
        ctx.save_for_backward(*keep)
        ctx.shapes, ctx.bias_dtype = (x.shape, weight.shape), None if bias is None else bias.dtype
        return y

    backward = _backward(_linear_backward)


def linear_act(x: Tensor, weight: Tensor, bias: Optional[Tensor] = None, act: Optional[str] = None, residual: Optional[Tensor] = None,
               slope: float = 1e-2) -> Tensor:
    """act(x @ weight^T + bias) + residual, rounded once: [..., k] x [n, k] -> [..., n] in one launch (two where k is split).

    x, weight, residual: one type of fp32, bf16 and fp16; bias that type or fp32; act as in `get_nonlinearity` or None; any sizes from one row and
    one column on.  Sums are fp32 (fp32 operands on the fp32 matrix instructions: no shorter terms).  Row strides are taken as they are, other
    layouts are copied.  The backward keeps the pre-activation in x's type (held to its range), and rounds its gradient dz to that type as an operand
    of the products for x and weight, where it has the range of the type: in fp16 a |dz| from 65520 on is infinite, below 3e-8 zero.  The bias
    gradient is summed unrounded.  All sums have a fixed order, so a run repeats bit for bit."""
    _check_first(x, "x")
    _check(weight, "weight", x)
    if weight.dim() != 2 or weight.shape[1] != x.shape[-1] or weight.shape[0] < 1 or weight.shape[1] < 1:
        raise ValueError(f"linear_act: weight must be [n, {x.shape[-1]}] with at least one row and column, got {tuple(weight.shape)}")
    if act not in ACT:
        raise ValueError(f"linear_act: act is None or one of {sorted(k for k in ACT if k)}, got {act!r}")
    n = weight.shape[0]
    if bias is not None:
        _check(bias, "bias", x, (n,), torch.float32)
    if residual is not None:
        _check(residual, "residual", x, (*x.shape[:-1], n))
    if _wants_grad((x, weight, bias, residual)):
        return _LinearAct.apply((act, float(slope)), x, weight, bias, residual)
    return _linear_forward((act, float(slope)), x, weight, bias, residual, False)[0]
