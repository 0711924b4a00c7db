"""Activations kept in 8 bits for the backward pass — host side of csrc/act8.hip.

What a layer saves between its forward and its backward pass is most of the memory that a training step holds.  Here it is saved as
e4m3 codes with one power-of-two scale per 32 channels of a row: 1.03 bytes a value in place of 4 (fp32) or 2 (bf16, fp16),
off by at most 2^-4 of a value (half a step), or 2^-10 of the group's scale below its smallest normal code.

    kept = pack(x)              Act8: codes + exponents of x (..., C)
    x8 = unpack(kept)           the values that the codes stand for, in x's type

    y = linear(x, w, b, relu)   [relu](x w^T + b), with gradients; what waits for the backward pass is pack(x), one bit per
                                output behind a ReLU, and w

`pack` / `unpack` are plain functions (no gradient).  The forward pass and the input gradient of `linear` see x and w as they are;
only the weight gradient sees unpack(pack(x))."""
import torch
from torch.autograd import Function, forward_ad
from torch.autograd.function import once_differentiable

from . import _lib

GROUP = 32                                   # channels that share a scale
DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


class Act8(object):
    """The 8-bit form of a tensor of `shape` (..., C) and type `dtype`: codes (rows, 32 * groups) uint8, exps (rows, groups)
    uint8 = exponent + 127; value = code * 2^exponent."""
    __slots__ = ('codes', 'exps', 'shape', 'dtype')

    def __init__(self, codes, exps, shape, dtype):
        self.codes, self.exps, self.shape, self.dtype = codes, exps, torch.Size(shape), dtype

    @property
    def nbytes(self):
        return self.codes.numel() + self.exps.numel()

    def exponents(self):
        """(rows, groups) int32: the power of two that scales each group's codes."""
        return self.exps.to(torch.int32) - 127


class _Stay(object):
    """with _on(device) where the device is the current one already."""
    __slots__ = ()

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        return False


_STAY = _Stay()


def _on(dev):
    """A context with `dev` as the current device (launches and streams go by the current device)."""
    return _STAY if dev.index == torch._C._cuda_getDevice() else torch.cuda.device(dev)


def _device_of(*tensors):
    """The device that all tensors (or None) are on; raises unless it is one HIP device."""
    dev = None
    for t in tensors:
        if t is None:
            continue
        if dev is None:
            if not t.is_cuda:
                raise _lib.DetMatchHipError('detmatch_amd ops run on the MI355X only (got a %s tensor); there is no CPU path'
                                            % t.device)
            dev = t.device
        elif t.device != dev:
            if not t.is_cuda:
                raise _lib.DetMatchHipError('detmatch_amd ops run on the MI355X only (got a %s tensor); there is no CPU path'
                                            % t.device)
            raise ValueError('tensors on two devices: %s and %s' % (dev, t.device))
    return dev


def _refuse_trace():
    """Kernels called outside of an autograd function leave no trace: torch.jit.trace would record empty buffers in their place."""
    if torch._C._get_tracing_state() is not None:
        raise NotImplementedError('torch.jit.trace cannot record these operators where no input needs a gradient')


def _wants_grad(*tensors):
    """Does the call go through the autograd function?  Where it does not, what the function refuses by itself is refused here: forward-mode
    derivatives, which would be lost, and traces."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    if forward_ad._current_level >= 0:
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise NotImplementedError('these operators have no forward-mode derivatives')
    _refuse_trace()
    return False


def _dtype_code(t, what):
    code = DTYPES.get(t.dtype)
    if code is None:
        raise TypeError('%s is %s: float32, bfloat16 or float16 is wanted' % (what, t.dtype))
    return code


def rows_view(x):
    """x (..., C) as (rows, C) with unit stride along C and non-overlapping rows (a copy where it has neither)."""
    r = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    if r.is_contiguous():
        return r
    if (r.shape[1] > 1 and r.stride(1) != 1) or (r.shape[0] > 1 and r.stride(0) < r.shape[1]):
        r = r.contiguous()
    return r


def row_stride(r):
    """Elements between rows of rows_view's answer (a single row's stride means nothing)."""
    return r.stride(0) if r.shape[0] > 1 else r.shape[1]


def pack(x):
    """The 8-bit form of x (..., C), float32 / bfloat16 / float16, any row stride."""
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError('pack needs at least one channel, got shape %s' % (tuple(x.shape),))
    code = _dtype_code(x, 'x')
    _refuse_trace()
    dev = _device_of(x)
    with _on(dev):
        r = rows_view(x.detach() if x.requires_grad else x)
        rows, width = r.shape
        groups = (width + GROUP - 1) // GROUP
        codes = torch.empty((rows, groups * GROUP), dtype=torch.uint8, device=dev)
        exps = torch.empty((rows, groups), dtype=torch.uint8, device=dev)
        _lib.check(_lib.lib().dm_act8_pack(_lib.ptr(r), code, rows, width, row_stride(r), _lib.ptr(codes), _lib.ptr(exps),
                                           _lib.stream()), 'dm_act8_pack')
    return Act8(codes, exps, x.shape, x.dtype)


def unpack(kept, dtype=None):
    """The values of an Act8, in `dtype` (default: the type of the tensor that was packed), saturating at its largest finite
    value."""
    if not isinstance(kept, Act8):
        raise TypeError('unpack takes what pack returned, got %s' % type(kept).__name__)
    _refuse_trace()
    width = kept.shape[-1]
    rows, groups = kept.shape.numel() // width, (width + GROUP - 1) // GROUP
    for t, shape, name in ((kept.codes, (rows, groups * GROUP), 'codes'), (kept.exps, (rows, groups), 'exps')):
        if t.dtype != torch.uint8 or t.shape != shape or not t.is_contiguous():
            raise ValueError('%s: a contiguous uint8 tensor %s is wanted, got %s %s' % (name, shape, t.dtype, tuple(t.shape)))
    out = torch.empty(kept.shape, dtype=kept.dtype if dtype is None else dtype, device=kept.codes.device)
    code = _dtype_code(out, 'dtype')
    with _on(_device_of(kept.codes, kept.exps)):
        _lib.check(_lib.lib().dm_act8_unpack(_lib.ptr(kept.codes), _lib.ptr(kept.exps), rows, width,
                                             _lib.ptr(out), code, _lib.stream()), 'dm_act8_unpack')
    return out


# ---- fully connected layers ----------------------------------------------------------------------------------------------
_MAX = (1 << 31) - 1024                      # rows and channels are 32-bit numbers in the kernels


_COPY_FROM = 1 << 33                         # multiply-adds; see _operands


def _operand(r):
    """(tensor to keep alive, address, pitch) of rows as they lie."""
    r = rows_view(r)
    return r, r.data_ptr(), row_stride(r)


def _direct(o, width):
    return width % 8 == 0 and o[2] % 8 == 0 and o[1] % 16 == 0


def _masked(o, rows, width, bits, code):
    """A copy of an operand with a pitch of 8 elements and zeros behind its width, and 0 where a sign bit is not set."""
    r = o[0]
    pitch = (width + 7) // 8 * 8
    out = torch.empty((rows, pitch), dtype=r.dtype, device=r.device)
    at = out.data_ptr()
    _lib.check(_lib.lib().dm_act8_mask_rows(o[1], code, rows, width, o[2], bits, at, pitch,
                                            _lib.raw_stream()), 'dm_act8_mask_rows')
    return out, at, pitch


def _gemm(form, code, a, b, exps, bias, relu, m, n, k, out, bits=None, rowsum=None, masked=False):
    """One product; a, b: (what to keep alive, address, pitch); exps, bias, bits, rowsum: addresses or None; masked: a is _masked's."""
    padded = 1 if masked else 0
    if code and m * n * k >= _COPY_FROM:
        # Rows at any address go through registers, and through small tiles: for large products a copy at 16-byte pitch and the direct
        # path are faster.
        wide = m if form == 2 else k
        if not masked and not _direct(a, wide):
            a, padded = _masked(a, k if form == 2 else m, wide, None, code), 1
        wide = k if form == 0 else n
        if form != 2 and not _direct(b, wide):
            b, padded = _masked(b, n if form == 0 else k, wide, None, code), padded | 2
    L = _lib.lib()
    need = L.dm_act8_gemm_workspace_bytes(form, code, a[1], a[2], b[1], b[2], padded, m, n, k)
    # (a buffer of its own for every call: two streams, or two captured graphs, never share one)
    ws = torch.empty(need, dtype=torch.uint8, device=out.device) if need else None
    e = L.dm_act8_gemm(form, code, a[1], a[2], b[1], b[2], padded, exps, bias, relu, m, n, k, out.data_ptr(), bits, rowsum,
                       ws.data_ptr() if need else None, need, _lib.raw_stream())
    if e:
        _lib.check(e, 'dm_act8_gemm')
    return out


def _kept_layout(m, n, k, codes, bits):
    """Offsets of codes, exponents and sign bits in the one buffer that a layer keeps, and its size."""
    groups = (k + GROUP - 1) // GROUP
    at_exps = m * groups * GROUP if codes else 0
    at_bits = (at_exps + (m * groups if codes else 0) + 3) // 4 * 4
    return groups, at_exps, at_bits, at_bits + (m * ((n + 31) // 32) * 4 if bits else 0)


class _Linear8(Function):

    @staticmethod
    def forward(ctx, x, w, b, relu):
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        m, k = x.shape
        n = w.shape[0]
        dev, code = x.device, DTYPES[x.dtype]
        groups, at_exps, at_bits, size = _kept_layout(m, n, k, need_w, relu)
        with _on(dev):
            kept = torch.empty(size, dtype=torch.uint8, device=dev)
            y = torch.empty((m, n), dtype=x.dtype, device=dev)
            if m:
                base, xo = kept.data_ptr(), _operand(x)
                if need_w:
                    e = _lib.lib().dm_act8_pack(xo[1], code, m, k, xo[2], base, base + at_exps, _lib.raw_stream())
                    if e:
                        _lib.check(e, 'dm_act8_pack')
                bias = None if b is None else b.contiguous()
                _gemm(0, code, xo, _operand(w), None, None if b is None else bias.data_ptr(), relu, m, n, k, y,
                      base + at_bits if relu else None)
        ctx.save_for_backward(w if need_x else None, kept)
        ctx.rest = (m, n, k, relu)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, gy):
        w, kept = ctx.saved_tensors
        m, n, k, relu = ctx.rest
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        code, dtype, dev = DTYPES[gy.dtype], gy.dtype, gy.device
        gx = gw = gb = None
        with _on(dev):
            if m == 0:
                return (gy.new_zeros((0, k)) if need_x else None, gy.new_zeros((n, k)) if need_w else None,
                        gy.new_zeros(n) if need_b else None, None)
            groups, at_exps, at_bits, _ = _kept_layout(m, n, k, need_w, relu)
            base, g = kept.data_ptr(), _operand(gy)
            if relu:
                g = _masked(g, m, n, base + at_bits, code)
            if need_x:
                gx = _gemm(1, code, g, _operand(w), None, None, 0, m, k, n, torch.empty((m, k), dtype=dtype, device=dev), masked=relu)
            if need_b:
                gb = torch.empty(n, dtype=dtype, device=dev)
            if need_w:
                gw = _gemm(2, code, g, (kept, base, groups * GROUP), base + at_exps, None, 0, n, k, m,
                           torch.empty((n, k), dtype=dtype, device=dev), rowsum=gb.data_ptr() if need_b else None, masked=relu)
            elif need_b:                      # a bias alone: its sums ride on a product with one group of zeros
                zero = torch.zeros((2, m, GROUP), dtype=torch.uint8, device=dev)
                _gemm(2, code, g, (zero, zero.data_ptr(), GROUP), zero.data_ptr() + m * GROUP, None, 0, n, GROUP, m,
                      torch.empty((n, GROUP), dtype=dtype, device=dev), rowsum=gb.data_ptr(), masked=relu)
        return gx, gw, gb, None


def linear(x, w, b=None, relu=False):
    """[relu](x w^T + b) for x (..., in), w (out, in), b (out) of one type (float32, bfloat16 or float16), on csrc/act8_gemm.hip.

    Kept for the backward pass: pack(x) where w needs a gradient, one bit per output where there is a ReLU, w where x needs a
    gradient.  gw = g^T unpack(pack(x)), gx = g w, gb = sum of g over rows, g = the gradient behind the ReLU (0 where its output,
    as it is stored, is 0).  float32 operands are multiplied in pieces: a result in which an infinity takes part is nan, and less than
    2^-133 is lost of a value below 2^-109.
    x may be overwritten after the call.  Differentiable once, in reverse mode; a forward-mode derivative is refused."""
    if x.dim() < 1 or w.dim() != 2 or x.shape[-1] != w.shape[1]:
        raise ValueError('x (..., in) and w (out, in) are wanted, got %s and %s' % (tuple(x.shape), tuple(w.shape)))
    if b is not None and tuple(b.shape) != (w.shape[0],):
        raise ValueError('b has shape %s, w has %d rows' % (tuple(b.shape), w.shape[0]))
    if w.shape[0] < 1 or w.shape[1] < 1:
        raise ValueError('w %s has no elements' % (tuple(w.shape),))
    _dtype_code(x, 'x')
    for t, name in ((w, 'w'), (b, 'b')):
        if t is not None and t.dtype != x.dtype:
            raise TypeError('%s is %s, x is %s: one type is wanted' % (name, t.dtype, x.dtype))
    grad = _wants_grad(x, w, b)
    _device_of(x, w, b)
    x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    if max(x2.shape[0], w.shape[0], w.shape[1]) > _MAX:
        raise ValueError('sizes up to %d are wanted, got x %s, w %s' % (_MAX, tuple(x.shape), tuple(w.shape)))
    if grad:
        y = _Linear8.apply(x2, w, b, bool(relu))
    else:
        m, k = x2.shape
        n = w.shape[0]
        with _on(x.device):
            y = torch.empty((m, n), dtype=x.dtype, device=x.device)
            if m:
                bias = None if b is None else b.contiguous()
                _gemm(0, DTYPES[x.dtype], _operand(x2), _operand(w), None, None if b is None else bias.data_ptr(), bool(relu), m, n, k, y)
    return y if x.dim() == 2 else y.view(*x.shape[:-1], w.shape[0])
