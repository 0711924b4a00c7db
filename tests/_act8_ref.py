"""The 8-bit activation format by its definition, in float64 with numpy: every code's value is listed, a value takes the nearest one
(ties: the code with an even last bit)."""
import numpy as np
import torch


def _codes():
    """value of each of the 127 non-negative finite e4m3 codes."""
    out = []
    for c in range(127):
        exp, man = c >> 3, c & 7
        out.append(man * 2.0 ** -9 if exp == 0 else (8 + man) * 2.0 ** (exp - 10))
    return np.array(out)


CODES = _codes()


def exponent(top):
    """least e >= -127 with top <= 448 * 2^e, 0 for top == 0 (top: array of float64)."""
    e = np.full(top.shape, -127)
    for k in range(-127, 130):
        e = np.where(top > 448.0 * 2.0 ** (k - 0), k + 1, e)
    return np.where(top == 0, 0, e)


def pack(x):
    """x: torch tensor (rows, width) on any device -> (code bytes (rows, 32 * groups), exponents (rows, groups)) as numpy."""
    v = x.detach().cpu().double().numpy()
    rows, width = v.shape
    groups = (width + 31) // 32
    v = np.concatenate([v, np.zeros((rows, groups * 32 - width))], 1).reshape(rows, groups, 32)
    fine = np.isfinite(v)
    mag = np.abs(np.where(fine, v, 0.0))
    e = exponent(mag.max(2, initial=0.0))
    z = mag * 2.0 ** -e.astype(np.float64)[:, :, None]
    hi = np.searchsorted(CODES, z).clip(1, 126)
    lo = hi - 1
    dl, dh = z - CODES[lo], CODES[hi] - z
    code = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    code = np.where((e[:, :, None] >= 120) & (code > 0x77), 0x77, code)          # 240 * 2^120: 256 * 2^120 is no float
    code = np.where(fine, code | (np.signbit(v) * 128), 0x7f)
    return code.reshape(rows, groups * 32).astype(np.uint8), e


def unpack(code, e, width, dtype):
    """float64 values in `dtype`'s range (rows, width)."""
    c = code.astype(np.int64)
    mag = np.where((c & 127) == 127, np.nan, np.concatenate([CODES, [np.nan]])[c & 127])
    v = np.where(c >= 128, -mag, mag).reshape(code.shape[0], -1, 32) * 2.0 ** e.astype(np.float64)[:, :, None]
    v = v.reshape(code.shape)[:, :width]
    most = torch.finfo(dtype).max
    return torch.from_numpy(np.clip(v, -most, most)).to(dtype).double()
