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
from .act8 import DTYPES, GROUP, _MAX, _device_of, _dtype_code, row_stride, rows_view

KINDS = {'rms': 0, 'layer': 1}
GATE_ACTS = {None: 0, 'none': 0, 'sigmoid': 1, 'tanh': 2}


def max_width():
    """Channels that a row may have."""
    return int(_lib.lib().dm_block_norm_max_width())


def _codes(rows, width, dev):
    groups = (width + GROUP - 1) // GROUP
    return (torch.empty((rows, groups * GROUP), dtype=torch.uint8, device=dev),
            torch.empty((rows, groups), dtype=torch.uint8, device=dev))


def _rows(t):
    """(rows tensor, address, pitch) of an optional (rows, width) operand"""
    if t is None:
        return None, None, 0
    r = rows_view(t)
    return r, _lib.ptr(r), row_stride(r)


def _fill(meta, width, rows, dtype, gate, scale, scale_host, post_w, post_b, pre_w, pre_b):
    """(the struct, what has to stay alive for the call)"""
    post, layer, act, eps = meta
    q = _lib.BlockNorm()
    q.dtype, q.width, q.rows, q.layer, q.post, q.gate_act, q.eps = DTYPES[dtype], width, rows, layer, int(post), act, eps
    gate, q.gate, q.ld_gate = _rows(gate)
    q.groups = 0 if gate is None else gate.shape[0]
    params = [None if p is None else p.detach().contiguous() for p in (post_w, post_b, pre_w, pre_b)]
    q.post_w, q.post_b, q.pre_w, q.pre_b = (_lib.ptr(p) for p in params)
    q.param_f32 = int(any(p is not None and p.dtype == torch.float32 for p in params))
    q.scale_host, q.scale, q.scale_f32 = scale_host, _lib.ptr(scale), int(scale is not None and scale.dtype == torch.float32)
    return q, (gate, params)


class _ResidualNorm(Function):
    """x, f (rows, width); gate (groups, width).  f None: the norm of x alone (y is x itself and not returned)."""

    @staticmethod
    def forward(ctx, x, f, gate, scale, post_w, post_b, pre_w, pre_b, scale_host, meta, pre, keep8, grad):
        rows, width = x.shape
        post, layer, act, eps = meta
        dev, dtype = x.device, x.dtype
        train = grad and any(ctx.needs_input_grad)
        y = h = None
        stats, codes = [None] * 4, [None] * 4
        with torch.cuda.device(dev):
            xr, xp, ldx = _rows(x.detach())
            fr, fp, ldf = _rows(None if f is None else f.detach())
            if f is not None:
                y = torch.empty((rows, width), dtype=dtype, device=dev)
            if pre:
                h = torch.empty((rows, width), dtype=dtype, device=dev)
            if train:
                both = torch.empty((4, rows), dtype=torch.float32, device=dev)
                stats = [both[0] if f is not None and post and layer else None, both[1] if f is not None and post else None,
                         both[2] if pre and layer else None, both[3] if pre else None]
                if keep8:
                    if f is not None:
                        codes[:2] = _codes(rows, width, dev)
                    if pre:
                        codes[2:] = _codes(rows, width, dev)
            if rows:
                q, alive = _fill(meta, width, rows, dtype, None if gate is None else gate.detach(), None if scale is None else scale.detach(),
                                 scale_host, post_w, post_b, pre_w, pre_b)
                q.f_mean, q.f_rstd, q.y_mean, q.y_rstd = (_lib.ptr(t) for t in stats)
                q.f_codes, q.f_exps, q.y_codes, q.y_exps = (_lib.ptr(t) for t in codes)
                _lib.check(_lib.lib().dm_block_norm_forward(ctypes.byref(q), xp, ldx, fp, ldf, _lib.ptr(y), _lib.ptr(h), _lib.stream()),
                           'dm_block_norm_forward')
        if train:
            exact = not keep8
            ctx.save_for_backward(gate, scale, post_w, post_b, pre_w, pre_b, f if exact else None,
                                  (y if f is not None else x) if exact and pre else None, *stats, *codes)
            ctx.rest = (rows, width, dtype, scale_host, meta, pre, f is not None)
        ctx.set_materialize_grads(False)
        return y, h

    @staticmethod
    @once_differentiable
    def backward(ctx, gy, gh):
        gate, scale, post_w, post_b, pre_w, pre_b, f, y, *kept = ctx.saved_tensors
        rows, width, dtype, scale_host, meta, pre, has_f = ctx.rest
        post, layer, act, eps = meta
        need = ctx.needs_input_grad
        if gy is None and gh is None:
            return (None,) * 13
        dev = (gy if gy is not None else gh).device
        L = _lib.lib()

        def like(t, wanted):
            return torch.empty(t.shape, dtype=t.dtype, device=dev) if wanted and t is not None else None

        with torch.cuda.device(dev):
            dx = torch.empty((rows, width), dtype=dtype, device=dev) if need[0] else None
            df = torch.empty((rows, width), dtype=dtype, device=dev) if need[1] else None
            out = [like(gate, need[2]), like(scale, need[3]), like(post_w, need[4]), like(post_b, need[5]), like(pre_w, need[6]),
                   like(pre_b, need[7])]
            if gh is None:                     # nothing came back through the second norm
                for k in (4, 5):
                    if out[k] is not None:
                        out[k].zero_()
            if rows == 0:
                for t in out:
                    if t is not None:
                        t.zero_()
            else:
                q, alive = _fill(meta, width, rows, dtype, None if gate is None else gate.detach(), None if scale is None else scale.detach(),
                                 scale_host, post_w, post_b, pre_w, pre_b)
                q.f_mean, q.f_rstd, q.y_mean, q.y_rstd, q.f_codes, q.f_exps, q.y_codes, q.y_exps = (_lib.ptr(t) for t in kept)
                (gyr, gyp, ldgy), (ghr, ghp, ldgh) = _rows(gy), _rows(gh)
                (yr, yp, ldy), (fr, fp, ldf) = _rows(y), _rows(f)
                need_bytes = int(L.dm_block_norm_workspace_bytes(rows, width, q.groups))
                ws = torch.empty(need_bytes, dtype=torch.uint8, device=dev)
                pw, pb = (out[4], out[5]) if gh is not None else (None, None)
                _lib.check(L.dm_block_norm_backward(
                    ctypes.byref(q), gyp, ldgy, ghp, ldgh, yp, ldy, fp, ldf, _lib.ptr(dx), _lib.ptr(df), _lib.ptr(out[0]), _lib.ptr(pw),
                    _lib.ptr(pb), _lib.ptr(out[2]), _lib.ptr(out[3]), _lib.ptr(out[1]), _lib.ptr(ws), need_bytes, _lib.stream()),
                    'dm_block_norm_backward')
        return (dx, df, *out, None, None, None, None, None)


def _check(x, f, gate, scale, params, kind, eps, gate_act, post):
    """What both entry points refuse; -> (rows, width)"""
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError('x (..., channels) is wanted, got %s' % (tuple(x.shape),))
    _dtype_code(x, 'x')
    width, rows = x.shape[-1], x.numel() // x.shape[-1]
    if kind not in KINDS:
        raise ValueError('kind %r: one of %s' % (kind, sorted(KINDS)))
    if gate_act not in GATE_ACTS:
        raise ValueError("gate_act %r: None, 'sigmoid' or 'tanh'" % (gate_act,))
    if not eps >= 0:
        raise ValueError('eps %r' % (eps,))
    if rows > _MAX:
        raise ValueError('x has %d rows: up to %d' % (rows, _MAX))
    for name, t in (('f', f), ('gate', gate)):
        if t is not None and t.dtype != x.dtype:
            raise TypeError('%s is %s, x is %s: one type is wanted' % (name, t.dtype, x.dtype))
    if f is not None and f.shape != x.shape:
        raise ValueError('f has shape %s, x %s' % (tuple(f.shape), tuple(x.shape)))
    if gate is not None:
        if gate.dim() < 1 or gate.shape[-1] != width:
            raise ValueError('gate has shape %s, x %s' % (tuple(gate.shape), tuple(x.shape)))
        groups = gate.numel() // width
        if groups < 1 and rows or groups and rows % groups:
            raise ValueError('%d rows do not divide into %d rows of gates' % (rows, groups))
    kinds = {p.dtype for p in params.values() if p is not None}
    if len(kinds) > 1 or not kinds <= {torch.float32, x.dtype}:
        raise TypeError('parameters are %s: all float32 or all %s are wanted' % (sorted(map(str, kinds)), x.dtype))
    for name, p in params.items():
        if p is not None and tuple(p.shape) != (width,):
            raise ValueError('%s has shape %s: (%d,) is wanted' % (name, tuple(p.shape), width))
    if kind == 'rms' and any(p is not None for name, p in params.items() if name.endswith('b')):
        raise ValueError('the RMS norm has no bias')
    if not post and (params.get('post_w') is not None or params.get('post_b') is not None):
        raise ValueError('post_w / post_b without post')
    if isinstance(scale, torch.Tensor):
        if scale.numel() != 1:
            raise ValueError('scale has %d elements: a number, or a tensor of one' % scale.numel())
        if scale.dtype not in (torch.float32, x.dtype):
            raise TypeError('scale is %s: float32 or %s' % (scale.dtype, x.dtype))
    _device_of(x, f, gate, scale if isinstance(scale, torch.Tensor) else None, *params.values())
    if width > max_width():
        raise ValueError('%d channels: up to %d' % (width, max_width()))
    return rows, width


def residual_norm(x, f, scale=1.0, gate=None, gate_act=None, post=True, post_w=None, post_b=None, pre=True, pre_w=None, pre_b=None,
                  kind='rms', eps=1e-6, keep8=False):
    """(y, h) of the residual stream x (..., C) and a block's output f of the same shape and type (float32, bfloat16, float16):

        u = N(f) * post_w + post_b  (post = False: u = f)
        y = x + scale * act(gate) * u
        h = N(y) * pre_w + pre_b    (pre = False: h is None)

    scale: a number, or a tensor of one element (with a gradient).  gate: (C,) for all rows; (G, C) (any leading shape): each for
    rows / G consecutive rows, a sample's or (G = rows) a row's own; gate_act None, 'sigmoid' or 'tanh' of it.  Weights (C,) in x's type or
    float32; None: 1.  Biases with kind = 'layer' only.  Statistics and sums are fp32; h is the norm of y before y is rounded.
    keep8: keep f and y in 8 bits for the backward pass.  Differentiable once."""
    if f is None:
        raise ValueError('f is None: norm_rows is the norm alone')
    if not pre and (pre_w is not None or pre_b is not None):
        raise ValueError('pre_w / pre_b without pre')
    params = dict(post_w=post_w, post_b=post_b, pre_w=pre_w, pre_b=pre_b)
    rows, width = _check(x, f, gate, scale, params, kind, eps, gate_act, post)
    tensor = scale if isinstance(scale, torch.Tensor) else None
    y, h = _ResidualNorm.apply(
        x.reshape(rows, width), f.reshape(rows, width), None if gate is None else gate.reshape(-1, width), tensor, post_w, post_b, pre_w,
        pre_b, 0.0 if tensor is not None else float(scale), (bool(post), KINDS[kind], GATE_ACTS[gate_act], float(eps)), bool(pre), bool(keep8),
        torch.is_grad_enabled())
    return y.view(x.shape), None if h is None else h.view(x.shape)


def norm_rows(x, w=None, b=None, kind='rms', eps=1e-6, keep8=False):
    """N(x) * w + b over the last dimension of x (float32, bfloat16, float16); w, b (C,) in x's type or float32, or None."""
    rows, width = _check(x, None, None, 1.0, dict(pre_w=w, pre_b=b), kind, eps, None, True)
    _, h = _ResidualNorm.apply(x.reshape(rows, width), None, None, None, None, None, w, b, 1.0,
                               (False, KINDS[kind], 0, float(eps)), True, bool(keep8), torch.is_grad_enabled())
    return h.view(x.shape)
