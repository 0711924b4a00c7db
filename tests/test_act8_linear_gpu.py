"""act8.linear (csrc/act8_gemm.hip) against float64.

Tolerances.  16-bit operands: products are exact in fp32; an instruction adds 16 of them, the K / 16 instructions (and at most 64 split
parts) follow one another, and each addition is off by at most 2^-23 of what it adds up to, which is at most S = sum |a b|: (K / 16 +
80) 2^-23 S, and half a step of the output's type on top.  fp32 operands: 6 (with codes 3) products an element, and the piece
products that are left out are at most 2 * 2^-22 + 2^-30 of |a b|: (6 K / 16 + 80) 2^-23 S + 2^-20.9 S.  A product or sum below
2^-126 may be lost whole: K + 80 of them."""
import numpy as np
import pytest
import torch

from detmatch_amd import act8

pytestmark = [pytest.mark.gpu, pytest.mark.timeout(300)]
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _requested():
    """Bytes that are asked for and alive (memory_allocated counts an allocator's blocks, which may be up to 1 MiB larger than asked for)."""
    return torch.cuda.memory_stats()['requested_bytes.all.current']


def _bound(a, b, want, dtype, codes=False):
    """elementwise bound of |got - want| for a (M, K) @ b (K, N), both float64"""
    s = a.abs() @ b.abs()
    k = a.shape[1]
    lost = (6 * k + 80) * 2.0 ** -126
    if dtype == torch.float32:
        return (k * (3 if codes else 6) / 16 + 80) * 2.0 ** -23 * s + (0 if codes else 2.0 ** -20.9) * s + lost
    return (k / 16 + 80) * 2.0 ** -23 * s + torch.finfo(dtype).eps / 2 * want.abs() * (1 + 1e-3) + torch.finfo(dtype).tiny + lost


def _inside(got, want, bound, what):
    far = (got.double().cpu() - want).abs() - bound
    assert got.shape == want.shape and bool((far <= 0).all()), '%s: %g over its bound' % (what, float(far.max()))


def _case(m, k, n, dtype, dev, bias, relu, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed + m * 7 + k * 3 + n)
    x = (torch.randn(m, k, generator=g) * torch.exp(torch.randn(1, k, generator=g)) * scale).to(dtype).to(dev)
    w = (torch.randn(n, k, generator=g) / k ** 0.5).to(dtype).to(dev)
    b = torch.randn(n, generator=g).to(dtype).to(dev) if bias else None
    gy = torch.randn(m, n, generator=g).to(dtype).to(dev)
    return x, w, b, gy


def _check(x, w, b, gy, relu):
    dtype = x.dtype
    leaves = [t.requires_grad_(True) for t in (x, w, b) if t is not None]
    y = act8.linear(x, w, b, relu=relu)
    grads = torch.autograd.grad(y, leaves, gy)
    x8 = act8.unpack(act8.pack(x)).double().cpu().reshape(-1, x.shape[-1])
    xd, wd, gd = (t.detach().double().cpu() for t in (x, w, gy))
    xd, gd, yd = xd.reshape(-1, xd.shape[-1]), gd.reshape(-1, gd.shape[-1]), y.detach().cpu().reshape(-1, y.shape[-1])
    z = xd @ wd.t() + (0 if b is None else b.detach().double().cpu())
    bound = _bound(xd, wd.t(), z, dtype) + (0 if b is None else 2.0 ** -23 * (z.abs() + b.detach().double().cpu().abs()))
    _inside(yd, z.clamp(min=0) if relu else z, bound, 'y')
    if relu:
        gd = gd * (yd > 0)                    # (the mask is the operator's own: a border is decided once)
    got = [t.detach().cpu() for t in grads]
    _inside(got[0].reshape(-1, wd.shape[1]), gd @ wd, _bound(gd, wd, gd @ wd, dtype), 'gx')
    gw = gd.t() @ x8
    _inside(got[1], gw, _bound(gd.t(), x8, gw, dtype, codes=True), 'gw')
    if b is not None:
        ones = torch.ones(gd.shape[0], 1, dtype=torch.float64)
        gb = gd.t() @ ones
        _inside(got[2][:, None], gb, _bound(gd.t(), ones, gb, dtype, codes=True), 'gb')
    assert all(g.dtype == dtype for g in grads) and y.dtype == dtype


SHAPES = [(1, 64, 64), (1, 1001, 515), (2, 32, 1), (7, 33, 8), (64, 64, 64), (128, 128, 128), (129, 136, 120), (257, 640, 130),
          (777, 1001, 515), (300, 2048, 256), (31, 8192, 96), (2049, 96, 72), (5000, 40, 24)]


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('m,k,n', SHAPES)
def test_forward_and_gradients(dev, m, k, n, dtype):
    x, w, b, gy = _case(m, k, n, dtype, dev, bias=(m + n) % 2 == 1, relu=False)
    _check(x, w, b, gy, False)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('m,k,n', [(1, 40, 33), (130, 256, 96), (777, 1001, 515), (40, 4096, 64)])
def test_relu_keeps_one_bit(dev, m, k, n, dtype):
    x, w, b, gy = _case(m, k, n, dtype, dev, bias=True, relu=True)
    _check(x, w, b, gy, True)


@pytest.mark.parametrize('dtype', TYPES)
def test_largest_and_smallest_values(dev, dtype):
    """Codes at both ends of the exponents: fp16's 65504 (its code stands for 2^16, which saturates), groups of tiny values."""
    top = {torch.float32: 1e30, torch.bfloat16: 1e30, torch.float16: 65504.0}[dtype]
    low = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 6e-8}[dtype]
    x, w, b, gy = _case(96, 128, 64, dtype, dev, True, False)
    x = x.detach()
    x[:, :32] = x[:, :32].sign() * top
    x[:, 32:64] = x[:, 32:64].sign() * low
    x[:, 64:96] = 0
    x[5] = 0
    # (forward: w must not turn the large columns into infinities)
    w = w.detach()
    w[:, :32] = 0
    gy = (gy.detach().float() * 2.0 ** -6).to(dtype)
    kept = act8.unpack(act8.pack(x)).double().cpu()
    gd = gy.double().cpu()
    want = gd.t() @ kept
    w.requires_grad_(True)
    y = act8.linear(x, w, None)
    gw, = torch.autograd.grad(y, [w], gy)
    _inside(gw.cpu(), want.clamp(-torch.finfo(dtype).max, torch.finfo(dtype).max) if dtype == torch.float16 else want,
            _bound(gd.t(), kept, want, dtype, codes=True), 'gw')


@pytest.mark.parametrize('dtype', TYPES)
def test_strided_and_batched_operands(dev, dtype):
    x, w, b, gy = _case(96, 200, 80, dtype, dev, True, False)
    wide_x, wide_w, wide_g = (torch.full((96, 304), float('nan'), device=dev, dtype=dtype) for _ in range(3))
    wide_x[:, 3:203], wide_w[:80, 8:208], wide_g[:, 1:81] = x.detach(), w.detach(), gy
    _check(wide_x[:, 3:203], wide_w[:80, 8:208], b, wide_g[:, 1:81], True)
    wide_x[:, 8:208] = x.detach()
    wide_x[:, 208:] = float('nan')
    # 195 of the contraction: the 16-byte piece at the end of a row also holds what does not belong to it
    _check(wide_x[:, 8:203].detach(), wide_w[:80, 8:203].detach(), b, wide_g[:, 1:81], False)
    _check(x.detach().view(4, 24, 200), w.detach(), b.detach(), gy.view(4, 24, 80), True)
    _check(x.detach().t().contiguous().t(), w.detach().t().contiguous().t(), b.detach(), gy.t().contiguous().t(), False)
    _check(x.detach(), w.detach(), b.detach(), gy[:1].expand(96, 80), True)


def test_every_subset_of_gradients(dev):
    for dtype in TYPES:
        x, w, b, gy = _case(70, 72, 40, dtype, dev, True, True)
        full = torch.autograd.grad(act8.linear(x.requires_grad_(True), w.requires_grad_(True), b.requires_grad_(True), True), [x, w, b], gy)
        for pick in range(1, 8):
            ts = [t.detach().requires_grad_(bool(pick >> i & 1)) for i, t in enumerate((x, w, b))]
            want = [f for i, f in enumerate(full) if pick >> i & 1]
            got = torch.autograd.grad(act8.linear(*ts, relu=True), [t for t in ts if t.requires_grad], gy)
            for a, c in zip(got, want):
                assert torch.equal(a, c)
        with torch.no_grad():
            assert torch.equal(act8.linear(x, w, b, True), act8.linear(x.detach(), w.detach(), b.detach(), True))


def test_no_rows(dev):
    x = torch.zeros(0, 24, device=dev, requires_grad=True)
    w = torch.zeros(8, 24, device=dev, requires_grad=True)
    y = act8.linear(x, w, None, relu=True)
    gx, gw = torch.autograd.grad(y, [x, w], torch.zeros(0, 8, device=dev))
    assert y.shape == (0, 8) and gx.shape == (0, 24) and gw.shape == (8, 24) and not gw.any()


def test_input_may_be_overwritten_and_what_is_kept_is_small(dev):
    x, w, b, gy = _case(512, 4096, 64, torch.float32, dev, True, False)
    w.requires_grad_(True)
    want, = torch.autograd.grad(act8.linear(x, w, b), [w], gy)
    torch.cuda.synchronize()
    before = _requested()
    y = act8.linear(x, w, b)
    held = _requested() - before - y.numel() * 4
    assert held <= 1.04 * x.numel() + 4096
    x.zero_()
    got, = torch.autograd.grad(y, [w], gy)
    assert torch.equal(got, want)


def test_gradients_are_those_of_differences(dev):
    """Central differences of the operator's own fp32 forward: the function is linear in each argument, so they hold up to rounding.
    gw is the gradient at the kept x."""
    x, w, b, gy = _case(50, 96, 40, torch.float32, dev, True, False)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    gx, gw, gb = torch.autograd.grad(act8.linear(*leaves), leaves, gy)
    g = torch.Generator().manual_seed(1)

    def loss(*a):
        with torch.no_grad():
            return float((act8.linear(*a).double() * gy.double()).sum())

    x8 = act8.unpack(act8.pack(x))
    for k, (at, grad) in enumerate((((x, w, b), gx), ((x8, w, b), gw), ((x, w, b), gb))):
        d = torch.randn(at[k].shape, generator=g).to(dev)
        at = [t.detach() for t in at]
        up, down = list(at), list(at)
        up[k], down[k] = at[k] + d, at[k] - d
        diff, want = (loss(*up) - loss(*down)) / 2, float((grad.double() * d.double()).sum())
        # 2000 outputs of size ~ 10, each off by (6 * 96 / 16 + 80) 2^-23 S, S ~ 30
        assert abs(diff - want) <= 2000 * (6 * 96 / 16 + 80) * 2.0 ** -23 * 30


def test_repeat_other_stream_and_two_graphs(dev):
    """Same inputs, same bits: eager, on a side stream, and from two captured graphs that are replayed in turn; the product is split
    (40 x 8192), so each call has a workspace."""
    x, w, b, gy = _case(40, 8192, 64, torch.bfloat16, dev, True, True)

    def step(xx):
        leaves = [t.detach().requires_grad_(True) for t in (xx, w, b)]
        y = act8.linear(*leaves, relu=True)
        return (y.detach(), *torch.autograd.grad(y, leaves, gy))

    want = step(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step(x)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, c) for a, c in zip(other, want))
    x2 = torch.randn_like(x)
    graphs = []
    for src in (x, x2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(src)
        graphs.append((graph, src, out))
    for k in range(3):
        for graph, src, out in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for graph, src, out in graphs:
            assert all(torch.equal(a, c) for a, c in zip(out, step(src)))
        x.copy_(torch.randn_like(x))


def test_not_a_number_and_infinity_reach_the_outputs(dev):
    for dtype in TYPES:
        x, w, b, gy = _case(40, 64, 32, dtype, dev, False, False)
        x[3, 5] = float('nan')
        x[4, 6] = float('inf')
        w.requires_grad_(True)
        y = act8.linear(x, w)
        assert y[3].isnan().all() and not y[4].isfinite().any() and y[5:].isfinite().all()
        gw, = torch.autograd.grad(y, [w], gy)
        assert gw[:, 5].isnan().all() and gw[:, 6].isnan().all() and gw[:, 7:].isfinite().all()


def test_relu_gradient_where_an_output_underflows_or_is_nan(dev):
    """The mask is that of the stored output: what is rounded to 0 has no gradient, its neighbours and a nan have."""
    for dtype, unit in ((torch.float16, 2.0 ** -24), (torch.bfloat16, 2.0 ** -133)):
        b = torch.tensor([unit, -unit, 3 * unit, 0.0, 1.0, float('nan')], dtype=dtype, device=dev)
        for split in (1, 4096):                # (the second: a split contraction, whose sums are joined by another kernel)
            # row 0 is b itself; rows 1 and 2 have a product of two small powers on top, half a unit of fp16
            xx = torch.zeros(3, split, dtype=dtype, device=dev)
            ww = torch.zeros(6, split, dtype=dtype, device=dev)
            xx[1, 0], xx[2, 0] = (2.0 ** -12, -2.0 ** -12) if dtype == torch.float16 else (2.0 ** -60, -2.0 ** -60)
            ww[:, 0] = 2.0 ** -13 if dtype == torch.float16 else 2.0 ** -65
            leaves = [t.requires_grad_(True) for t in (xx, ww, b.clone())]
            y = act8.linear(*leaves, relu=True)
            gy = torch.ones_like(y)
            gb, = torch.autograd.grad(y, leaves[2:], gy)
            want = (~(y.detach() <= 0)).double().sum(0)
            assert torch.equal(gb.double(), want), (dtype, split, gb, want, y)
            assert bool(y[:, 5].isnan().all()) and float(gb[5]) == 3 and float(gb[1]) <= 1 and float(gb[4]) == 3


def test_an_infinity_in_float32_is_nan_behind_a_relu_too(dev):
    x, w, b, _ = _case(40, 64, 32, torch.float32, dev, True, False)
    x[4, 6], x[5, 7] = float('inf'), -float('inf')
    y = act8.linear(x, w, b, relu=True)
    assert bool(y[4:6].isnan().all()) and bool(y[:4].isfinite().all()) and bool(y[6:].isfinite().all())
