"""act8.linear on the smallest numbers of each type, times large ones, so that results are ordinary numbers.

16-bit subnormal numbers take part as they are.  float32 operands are multiplied in bf16 pieces, and bf16 ends at 2^-133: of each value less than
2^-133 is lost, and of a code's value as much; a result is off by 2^-133 times the sum of what these are multiplied with, besides the bounds of
test_act8_linear_gpu.py.  Values from 2^-109 on are whole: 24 bits end at 2^-132 or above."""
import pytest
import torch

import test_act8_linear_gpu as lin
from detmatch_amd import act8

pytestmark = [pytest.mark.gpu, pytest.mark.timeout(300)]
M, K, N = 64, 96, 48
EXPONENTS = {torch.float16: (-10, -14, -16, -20, -24), torch.bfloat16: (-109, -126, -128, -130, -133),
             torch.float32: (-109, -112, -120, -126, -130, -133, -140)}


def _bound(small, large, want, dtype, codes, whole):
    """small (M, K) @ large (K, N), float64; whole: nothing of the small values is lost."""
    bound = lin._bound(small, large, want, dtype, codes)
    return bound if whole else bound + 2.0 ** -133 * large.abs().sum(0, keepdim=True)


@pytest.mark.parametrize('dtype,e', [(t, e) for t in lin.TYPES for e in EXPONENTS[t]])
def test_small_values(dev, dtype, e):
    g = torch.Generator().manual_seed(-e)
    up = 10 if dtype == torch.float16 else 60

    def small(*s):
        return ((torch.rand(*s, generator=g) + 1).double() * 2.0 ** e * torch.randn(*s, generator=g).sign()).to(dtype).to(dev)

    def large(*s):
        return ((torch.rand(*s, generator=g) + 1) * 2.0 ** up).to(dtype).to(dev)

    whole = dtype != torch.float32 or e >= -109
    x, w, gy = small(M, K).requires_grad_(True), large(N, K).requires_grad_(True), small(M, N)
    xd, wd, gd = (t.detach().double().cpu() for t in (x, w, gy))
    y = act8.linear(x, w)
    lin._inside(y.detach().cpu(), xd @ wd.t(), _bound(xd, wd.t(), xd @ wd.t(), dtype, False, whole), 'y')
    gx, = torch.autograd.grad(y, [x], gy)
    lin._inside(gx.cpu(), gd @ wd, _bound(gd, wd, gd @ wd, dtype, False, whole), 'gx')
    # weight gradient: small codes with large gradients, and the other way round
    gl = large(M, N)
    x8 = act8.unpack(act8.pack(x)).double().cpu()
    gw, = torch.autograd.grad(act8.linear(x, w), [w], gl)
    want = x8.t() @ gl.double().cpu()
    lin._inside(gw.t().cpu(), want, _bound(x8.t(), gl.double().cpu(), want, dtype, True, dtype != torch.float32), 'gw of small codes')
    xl = large(M, K)
    x8 = act8.unpack(act8.pack(xl)).double().cpu()
    gw, = torch.autograd.grad(act8.linear(xl, w), [w], gy)
    lin._inside(gw.cpu(), gd.t() @ x8, _bound(gd.t(), x8, gd.t() @ x8, dtype, True, whole), 'gw of small gradients')
