"""The norms before and after a residual block, fused with the block's gate and its residual scale — host side of
csrc/block_norm.hip.

    y, h = residual_norm(x, f, ...)     u = N(f) * post_w + post_b;  y = x + scale * act(gate) * u;  h = N(y) * pre_w + pre_b
    h = norm_rows(x, w, b)              N(x) * w + b, the norm in front of the first block

x is the residual stream, f what a block made of the previous h; y is the new stream, h the next block's input.  N is the RMS norm
('rms': v / sqrt(mean(v^2) + eps)) or the layer norm ('layer'), over the last dimension; unlike BatchNorm's its statistics are one
row's own, so labelled and unlabelled samples do not mix in them.  With keep8 = True the backward pass keeps f and y in 8 bits
(act8.py) in place of the tensors themselves: normalised values are then those of the codes, with the statistics of the exact rows."""
import ctypes

import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from . import _lib
from .act8 import DTYPES, GROUP, _MAX, _device_of, _dtype_code, _on, _wants_grad, row_stride, rows_view

KINDS = {'rms': 0, 'layer': 1}
GATE_ACTS = {None: 0, 'none': 0, 'sigmoid': 1, 'tanh': 2}


def max_width():
    """Channels that a row may have."""
    return int(_lib.lib().dm_block_norm_max_width())


def _rows(t):
    """(rows tensor, address, pitch) of a (rows, width) operand"""
    r = rows_view(t)
    return r, r.data_ptr(), row_stride(r)


def _fill(meta, width, rows, dtype, gate, scale, post_w, post_b, pre_w, pre_b):
    """(the struct, what has to stay alive for the call)"""
    post, layer, act, eps, scale_host = meta[:5]
    q = _lib.BlockNorm()
    q.dtype, q.width, q.rows, q.layer, q.post, q.gate_act, q.eps = DTYPES[dtype], width, rows, layer, post, act, eps
    alive = []
    if gate is not None:
        gate, q.gate, q.ld_gate = _rows(gate)
        q.groups = gate.shape[0]
        alive.append(gate)
    for name, p in (('post_w', post_w), ('post_b', post_b), ('pre_w', pre_w), ('pre_b', pre_b)):
        if p is not None:
            p = p.contiguous()
            setattr(q, name, p.data_ptr())
            q.param_f32 = p.dtype == torch.float32
            alive.append(p)
    if scale is None:
        q.scale_host = scale_host
    else:
        q.scale, q.scale_f32 = scale.data_ptr(), scale.dtype == torch.float32
    return q, alive


def _kept_layout(rows, width, meta, has_f, pre, keep8):
    """[(field of the struct, offset)] and the size of the one buffer with statistics and codes."""
    post, layer = meta[:2]
    groups = (width + GROUP - 1) // GROUP
    codes = [('f', has_f), ('y', pre)] if keep8 else []
    out, at = [], 0
    for name, there in codes:
        if there:
            out.append((name + '_codes', at))
            at += rows * groups * GROUP
    for name, there in (('f_rstd', has_f and post), ('f_mean', has_f and post and layer), ('y_rstd', pre), ('y_mean', pre and layer)):
        if there:
            out.append((name, at))
            at += rows * 4
    for name, there in codes:
        if there:
            out.append((name + '_exps', at))
            at += rows * groups
    return out, at


def _point(q, kept, layout):
    base = kept.data_ptr()
    for name, at in layout:
        setattr(q, name, base + at)


def _forward(x, f, gate, scale, post_w, post_b, pre_w, pre_b, meta, pre, kept, layout):
    """(y, h) of x, f (rows, width); f None: the norm of x alone (y is None).  kept: the buffer for the backward pass, or None."""
    rows, width = x.shape
    y = torch.empty((rows, width), dtype=x.dtype, device=x.device) if f is not None else None
    h = torch.empty((rows, width), dtype=x.dtype, device=x.device) if pre else None
    if rows:
        q, alive = _fill(meta, width, rows, x.dtype, gate, scale, post_w, post_b, pre_w, pre_b)
        if kept is not None:
            _point(q, kept, layout)
        x, xp, ldx = _rows(x)
        fp = ldf = 0
        if f is not None:
            f, fp, ldf = _rows(f)
        _lib.check(_lib.lib().dm_block_norm_forward(ctypes.byref(q), xp, ldx, fp, ldf, _lib.ptr(y), _lib.ptr(h), _lib.stream()),
                   'dm_block_norm_forward')
    return y, h


class _ResidualNorm(Function):

    @staticmethod
    def forward(ctx, x, f, gate, scale, post_w, post_b, pre_w, pre_b, meta, pre, keep8):
        rows, width = x.shape
        layout, size = _kept_layout(rows, width, meta, f is not None, pre, keep8)
        with _on(x.device):
            kept = torch.empty(size, dtype=torch.uint8, device=x.device)
            y, h = _forward(x, f, gate, scale, post_w, post_b, pre_w, pre_b, meta, pre, kept, layout)
        exact = not keep8
        ctx.save_for_backward(gate, scale, post_w, post_b, pre_w, pre_b, f if exact else None,
                              (y if f is not None else x) if exact and pre else None, kept)
        ctx.rest = (rows, width, x.dtype, meta, layout, f is not None)
        ctx.set_materialize_grads(False)
        return y, h

    @staticmethod
    @once_differentiable
    def backward(ctx, gy, gh):
        saved = ctx.saved_tensors
        gate, scale, post_w, post_b, pre_w, pre_b, f, y, kept = saved
        rows, width, dtype, meta, layout, has_f = ctx.rest
        need = ctx.needs_input_grad
        if gy is None and gh is None:
            return (None,) * 11
        dev = kept.device
        with _on(dev):
            dx = torch.empty((rows, width), dtype=dtype, device=dev) if need[0] else None
            df = torch.empty((rows, width), dtype=dtype, device=dev) if need[1] else None
            out = [torch.empty(t.shape, dtype=t.dtype, device=dev) if wanted and t is not None else None
                   for t, wanted in zip(saved, need[2:8])]           # gate, scale, post_w, post_b, pre_w, pre_b
            if rows == 0 or gh is None:        # (without gh nothing came back through the second norm)
                for t in out if rows == 0 else out[4:]:
                    if t is not None:
                        t.zero_()
            if rows:
                L = _lib.lib()
                q, alive = _fill(meta, width, rows, dtype, gate, scale, post_w, post_b, pre_w, pre_b)
                _point(q, kept, layout)
                gyp = ldgy = ghp = ldgh = yp = ldy = fp = ldf = 0
                if gy is not None:
                    gy, gyp, ldgy = _rows(gy)
                pw = pb = None
                if gh is not None:
                    gh, ghp, ldgh = _rows(gh)
                    pw, pb = out[4], out[5]
                if y is not None:
                    y, yp, ldy = _rows(y)
                if f is not None:
                    f, fp, ldf = _rows(f)
                size = L.dm_block_norm_workspace_bytes(rows, width, q.groups)
                ws = torch.empty(size, dtype=torch.uint8, device=dev)
                _lib.check(L.dm_block_norm_backward(
                    ctypes.byref(q), gyp, ldgy, ghp, ldgh, yp, ldy, fp, ldf, _lib.ptr(dx), _lib.ptr(df), _lib.ptr(out[0]), _lib.ptr(pw),
                    _lib.ptr(pb), _lib.ptr(out[2]), _lib.ptr(out[3]), _lib.ptr(out[1]), ws.data_ptr(), size, _lib.stream()),
                    'dm_block_norm_backward')
        return (dx, df, *out, None, None, None)


def _apply(grad, x, f, gate, scale, post_w, post_b, pre_w, pre_b, meta, pre, keep8):
    if grad:
        return _ResidualNorm.apply(x, f, gate, scale, post_w, post_b, pre_w, pre_b, meta, pre, keep8)
    with _on(x.device):
        return _forward(x, f, gate, scale, post_w, post_b, pre_w, pre_b, meta, pre, None, None)


_WIDTH = []


def _check(x, f, gate, scale, post_w, post_b, pre_w, pre_b, kind, eps, gate_act, post):
    """What both entry points refuse; -> (rows, width, does the call go through the autograd function)"""
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError('x (..., channels) is wanted, got %s' % (tuple(x.shape),))
    dtype = x.dtype
    _dtype_code(x, 'x')
    width = x.shape[-1]
    rows = x.numel() // width
    if kind not in KINDS:
        raise ValueError('kind %r: one of %s' % (kind, sorted(KINDS)))
    if gate_act not in GATE_ACTS:
        raise ValueError("gate_act %r: None, 'sigmoid' or 'tanh'" % (gate_act,))
    if not eps >= 0:
        raise ValueError('eps %r' % (eps,))
    if rows > _MAX:
        raise ValueError('x has %d rows: up to %d' % (rows, _MAX))
    if f is not None:
        if f.dtype != dtype:
            raise TypeError('f is %s, x is %s: one type is wanted' % (f.dtype, dtype))
        if f.shape != x.shape:
            raise ValueError('f has shape %s, x %s' % (tuple(f.shape), tuple(x.shape)))
    if gate is not None:
        if gate.dtype != dtype:
            raise TypeError('gate is %s, x is %s: one type is wanted' % (gate.dtype, dtype))
        if gate.dim() < 1 or gate.shape[-1] != width:
            raise ValueError('gate has shape %s, x %s' % (tuple(gate.shape), tuple(x.shape)))
        groups = gate.numel() // width
        if groups < 1 and rows or groups and rows % groups:
            raise ValueError('%d rows do not divide into %d rows of gates' % (rows, groups))
    first = None
    for name, p in (('post_w', post_w), ('post_b', post_b), ('pre_w', pre_w), ('pre_b', pre_b)):
        if p is None:
            continue
        if p.dtype != (first or p.dtype) or (p.dtype != dtype and p.dtype != torch.float32):
            raise TypeError('%s is %s: all parameters float32 or all %s are wanted' % (name, p.dtype, dtype))
        first = p.dtype
        if p.dim() != 1 or p.shape[0] != width:
            raise ValueError('%s has shape %s: (%d,) is wanted' % (name, tuple(p.shape), width))
    if kind == 'rms' and (post_b is not None or pre_b is not None):
        raise ValueError('the RMS norm has no bias')
    if not post and (post_w is not None or post_b is not None):
        raise ValueError('post_w / post_b without post')
    if scale is not None:
        if scale.numel() != 1:
            raise ValueError('scale has %d elements: a number, or a tensor of one' % scale.numel())
        if scale.dtype != dtype and scale.dtype != torch.float32:
            raise TypeError('scale is %s: float32 or %s' % (scale.dtype, dtype))
    grad = _wants_grad(x, f, gate, scale, post_w, post_b, pre_w, pre_b)
    _device_of(x, f, gate, scale, post_w, post_b, pre_w, pre_b)
    if not _WIDTH:
        _WIDTH.append(max_width())
    if width > _WIDTH[0]:
        raise ValueError('%d channels: up to %d' % (width, _WIDTH[0]))
    return rows, width, grad


def residual_norm(x, f, scale=1.0, gate=None, gate_act=None, post=True, post_w=None, post_b=None, pre=True, pre_w=None, pre_b=None,
                  kind='rms', eps=1e-6, keep8=False):
    """(y, h) of the residual stream x (..., C) and a block's output f of the same shape and type (float32, bfloat16, float16):

        u = N(f) * post_w + post_b  (post = False: u = f)
        y = x + scale * act(gate) * u
        h = N(y) * pre_w + pre_b    (pre = False: h is None)

    scale: a number, or a tensor of one element (with a gradient).  gate: (C,) for all rows; (G, C) (any leading shape): each for
    rows / G consecutive rows, a sample's or (G = rows) a row's own; gate_act None, 'sigmoid' or 'tanh' of it.  (The backward pass is slow for G > 64
    groups of hundreds of rows: it walks each one after the other.)  Weights (C,) in x's type or float32; None: 1.  Biases with kind = 'layer' only.  Statistics and sums are fp32; h is the norm of y before y is rounded.
    keep8: keep f and y in 8 bits for the backward pass.  Differentiable once, in reverse mode; a forward-mode derivative is refused."""
    if f is None:
        raise ValueError('f is None: norm_rows is the norm alone')
    if not pre and (pre_w is not None or pre_b is not None):
        raise ValueError('pre_w / pre_b without pre')
    tensor, number = (scale, 0.0) if isinstance(scale, torch.Tensor) else (None, float(scale))
    rows, width, grad = _check(x, f, gate, tensor, post_w, post_b, pre_w, pre_b, kind, eps, gate_act, post)
    flat = x.dim() == 2
    y, h = _apply(grad, x if flat else x.reshape(rows, width), f if flat else f.reshape(rows, width),
                  gate if gate is None or gate.dim() == 2 else gate.reshape(-1, width), tensor, post_w, post_b, pre_w, pre_b,
                  (bool(post), KINDS[kind], GATE_ACTS[gate_act], float(eps), number), bool(pre), bool(keep8))
    return (y, h) if flat else (y.view(x.shape), None if h is None else h.view(x.shape))


def norm_rows(x, w=None, b=None, kind='rms', eps=1e-6, keep8=False):
    """N(x) * w + b over the last dimension of x (float32, bfloat16, float16); w, b (C,) in x's type or float32, or None."""
    rows, width, grad = _check(x, None, None, None, None, None, w, b, kind, eps, None, True)
    flat = x.dim() == 2
    _, h = _apply(grad, x if flat else x.reshape(rows, width), None, None, None, None, None, w, b, (False, KINDS[kind], 0, float(eps), 1.0), True,
                  bool(keep8))
    return h if flat else h.view(x.shape)
