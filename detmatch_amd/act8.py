"""Activations kept in 8 bits for the backward pass — host side of csrc/act8.hip.

What a layer saves between its forward and its backward pass is most of the memory that a training step holds.  Here it is saved as
e4m3 codes with one power-of-two scale per 32 channels of a row: 1.03 bytes a value in place of 4 (fp32) or 2 (bf16, fp16),
off by at most 2^-4 of a value (half a step), or 2^-10 of the group's scale below its smallest normal code.

    kept = pack(x)              Act8: codes + exponents of x (..., C)
    x8 = unpack(kept)           the values that the codes stand for, in x's type

`pack` / `unpack` are plain functions (no gradient)."""
import torch

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


def _device_of(*tensors):
    """The device that all tensors (or None) are on; raises unless it is one HIP device."""
    dev = None
    for t in tensors:
        if t is None:
            continue
        if not t.is_cuda:
            raise _lib.DetMatchHipError('detmatch_amd ops run on the MI355X only (got a %s tensor); there is no CPU path'
                                        % t.device)
        if dev is not None and t.device != dev:
            raise ValueError('tensors on two devices: %s and %s' % (dev, t.device))
        dev = t.device
    return dev


def _dtype_code(t, what):
    if t.dtype not in DTYPES:
        raise TypeError('%s is %s: float32, bfloat16 or float16 is wanted' % (what, t.dtype))
    return DTYPES[t.dtype]


def rows_view(x):
    """x (..., C) as (rows, C) with unit stride along C and non-overlapping rows (a copy where it has neither)."""
    r = x.reshape(-1, x.shape[-1]) if x.dim() != 2 else x
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
    dev = _device_of(x)
    with torch.cuda.device(dev):
        r = rows_view(x.detach())
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
    out = torch.empty(kept.shape, dtype=kept.dtype if dtype is None else dtype, device=kept.codes.device)
    code = _dtype_code(out, 'dtype')
    with torch.cuda.device(_device_of(kept.codes, kept.exps)):
        _lib.check(_lib.lib().dm_act8_unpack(_lib.ptr(kept.codes), _lib.ptr(kept.exps), kept.codes.shape[0], kept.shape[-1],
                                             _lib.ptr(out), code, _lib.stream()), 'dm_act8_unpack')
    return out
