"""act8.linear where large tiles, copies of unaligned operands and 64-bit offsets come in, against float64 on the device."""
import pytest
import torch

import test_act8_linear_gpu as lin
from detmatch_amd import act8

pytestmark = [pytest.mark.gpu, pytest.mark.timeout(300)]


def _inside(got, a, b, dtype, codes, what, want=None):
    """lin._inside with the reference on the device."""
    want = a @ b if want is None else want
    far = (got.double() - want).abs() - lin._bound(a, b, want, dtype, codes)
    assert float(far.max()) <= 0, '%s: %g over its bound' % (what, float(far.max()))


def _check(x, w, gy, relu):
    x, w = x.requires_grad_(True), w.requires_grad_(True)
    y = act8.linear(x, w, relu=relu)
    gx, gw = torch.autograd.grad(y, (x, w), gy)
    x8 = act8.unpack(act8.pack(x)).double()
    xd, wd, gd, y = x.detach().double(), w.detach().double(), gy.double(), y.detach()
    z = xd @ wd.t()
    far = (y.double() - (z.clamp(min=0) if relu else z)).abs() - lin._bound(xd, wd.t(), z, x.dtype)
    assert float(far.max()) <= 0
    if relu:
        gd = gd * (y > 0)
    _inside(gx, gd, wd, x.dtype, False, 'gx')
    _inside(gw, gd.t(), x8, x.dtype, True, 'gw')


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
@pytest.mark.parametrize('relu', [False, True])
@pytest.mark.parametrize('m,k,n', [(3700, 3600, 3648), (3697, 3600, 4001), (4100, 520, 4608)])
def test_large_tiles(dev, dtype, relu, m, k, n):
    """200 tiles of 256 x 256 and more in each of the three products, at edges that are no tile's."""
    g = torch.Generator(device=dev).manual_seed(m + n)
    x = (torch.randn(m, k, generator=g, device=dev) * torch.exp(torch.randn(1, k, generator=g, device=dev))).to(dtype)
    w = (torch.randn(n, k, generator=g, device=dev) / k ** 0.5).to(dtype)
    gy = torch.randn(m, n, generator=g, device=dev).to(dtype)
    _check(x, w, gy, relu)


@pytest.mark.parametrize('dtype', lin.TYPES)
def test_copies_of_unaligned_operands(dev, dtype, monkeypatch):
    """What large products with rows at odd addresses do, at small sizes: the same results within the same bounds."""
    monkeypatch.setattr(act8, '_COPY_FROM', 0)
    g = torch.Generator().manual_seed(5)
    for m, k, n in ((129, 33, 77), (70, 1001, 515), (64, 64, 64)):
        x, w = torch.randn(m, k + 3, generator=g).to(dtype).to(dev)[:, 3:], torch.randn(n + 1, k, generator=g).to(dtype).to(dev)[1:]
        gy = torch.randn(m, n + 1, generator=g).to(dtype).to(dev)[:, 1:]
        for relu in (False, True):
            _check(x.detach(), w.detach(), gy, relu)


def test_offsets_behind_31_bits(dev):
    """x and the codes of x hold more than 2^31 elements, gx too."""
    m, k, n = 131200, 16384, 40
    x = torch.zeros(m, k, dtype=torch.bfloat16, device=dev)
    tail = torch.randn(48, k, device=dev).to(torch.bfloat16)
    x[-48:] = tail
    w = (torch.randn(n, k, device=dev) / 128).to(torch.bfloat16).requires_grad_(True)
    gy = torch.randn(m, n, device=dev).to(torch.bfloat16)
    x.requires_grad_(True)
    y = act8.linear(x, w)
    gx, gw = torch.autograd.grad(y, (x, w), gy)
    xd, wd, gd = tail.double(), w.detach().double(), gy[-48:].double()
    assert not bool(y[:-48].any())
    _inside(y[-48:].detach(), xd, wd.t(), torch.bfloat16, False, 'y')
    _inside(gx[-48:], gd, wd, torch.bfloat16, False, 'gx')
    x8 = act8.unpack(act8.pack(tail)).double()
    # (rows of zeros add nothing, but they are summed: the bound counts them)
    want = gd.t() @ x8
    bound = (m / 16 + 80) * 2.0 ** -23 * (gd.t().abs() @ x8.abs()) + 2.0 ** -8 * want.abs() * (1 + 1e-3) + 2.0 ** -120
    assert bool(((gw.double() - want).abs() <= bound).all())
