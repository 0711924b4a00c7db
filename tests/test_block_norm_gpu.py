"""block_norm (csrc/block_norm.hip) against its formulas in float64.

Tolerances: an fp32 sum over C <= 16 384 channels is 16 additions in a thread and a tree of 6 + 16 more, statistics and each later
step add a few roundings; 256 * 2^-24 of a value's magnitude (the same formula over absolute values, tests/_block_norm_ref.py) covers
the forward pass, twice that dy, three times df; sums over rows add at most `rows` roundings.  16-bit results: half a step of the
type on top."""
import pytest
import torch

import _block_norm_ref as ref
from detmatch_amd import act8, block_norm

pytestmark = [pytest.mark.gpu, pytest.mark.timeout(300)]
TYPES = [torch.float32, torch.bfloat16, torch.float16]
U = 2.0 ** -24


def _requested():
    """Bytes that are asked for and alive (memory_allocated counts an allocator's blocks, which may be up to 1 MiB larger than asked for)."""
    return torch.cuda.memory_stats()['requested_bytes.all.current']


def _near(got, want, ulps, what):
    v, mag = want
    got = got.detach()
    half = 0.0 if got.dtype == torch.float32 else torch.finfo(got.dtype).eps / 2
    g = got.double().cpu().reshape(v.shape)
    far = (g - v).abs() - (ulps * U * mag + half * v.abs() * (1 + 1e-3) + torch.finfo(got.dtype).tiny)
    assert bool((far <= 0).all()), '%s: %g over its bound (of %g)' % (what, float(far.max()), float(v.abs().max()))


def _case(rows, width, dtype, dev, layer=False, groups=0, act='none', post=True, pre=True, params=None, tensor_scale=True, seed=0):
    g = torch.Generator().manual_seed(seed + rows * 13 + width)
    params = params or dtype

    def r(*s, t=dtype, scale=1.0, shift=0.0):
        return (torch.randn(*s, generator=g) * scale + shift).to(t).to(dev)

    size = torch.exp(torch.randn(1, width, generator=g)).to(dev)
    p = dict(x=r(rows, width), f=(r(rows, width).float() * size).to(dtype), gate=r(groups, width, scale=0.5, shift=0.5) if groups else None,
             scale=r(1, t=params, shift=1.0) if tensor_scale else 0.7, post=post, pre=pre,
             post_w=r(width, t=params, scale=0.2, shift=1.0) if post else None, post_b=r(width, t=params) if post and layer else None,
             pre_w=r(width, t=params, scale=0.2, shift=1.0) if pre else None, pre_b=r(width, t=params) if pre and layer else None)
    return p, dict(kind='layer' if layer else 'rms', gate_act=act, eps=1e-5), r(rows, width), r(rows, width)


def _as64(p, more):
    q = {k: v.detach().double().cpu() if isinstance(v, torch.Tensor) else v for k, v in p.items()}
    q['scale'] = float(q['scale'])
    q['x'], q['f'] = (q[k].reshape(-1, q[k].shape[-1]) if q.get(k) is not None else None for k in ('x', 'f'))
    if q.get('gate') is not None:
        q['gate'] = q['gate'].reshape(-1, q['x'].shape[1])
    return dict(q, layer=more['kind'] == 'layer', eps=more['eps'], act=more['gate_act'] or 'none')


def _seen(t, keep8):
    v = act8.unpack(act8.pack(t)) if keep8 else t
    return v.detach().double().cpu().reshape(-1, t.shape[-1])


def _check(p, more, gy, gh, keep8=False):
    rows = p['x'].numel() // p['x'].shape[-1]
    names = [k for k in ('x', 'f', 'gate', 'scale', 'post_w', 'post_b', 'pre_w', 'pre_b') if isinstance(p[k], torch.Tensor)]
    p = dict(p, **{k: p[k].detach().requires_grad_(True) for k in names})
    y, h = block_norm.residual_norm(keep8=keep8, **p, **more)
    q = _as64(p, more)
    want = ref.forward(q)
    _near(y, want['y'], 256, 'y')
    if p['pre']:
        _near(h, want['h'], 512, 'h')
    else:
        assert h is None
    outs, gs = ([y, h], [gy, gh]) if p['pre'] else ([y], [gy])
    grads = dict(zip(names, torch.autograd.grad(outs, [p[k] for k in names], gs)))
    flat = [None if t is None else t.double().cpu().reshape(rows, -1) for t in (gy, gh if p['pre'] else None)]
    want = ref.backward(q, *flat, _seen(p['f'], keep8), _seen(y, keep8))
    for k in names:
        assert grads[k].shape == p[k].shape and grads[k].dtype == p[k].dtype
        _near(grads[k], want[k], 512 if k == 'x' else 768 if k == 'f' else 1024 + rows * (p['x'].shape[-1] if k == 'scale' else 1), 'gradient of ' + k)
    return y, h, grads


WIDTHS = [1, 7, 8, 33, 64, 100, 256, 640, 1001, 2048, 2056, 4096, 5000, 8192, 12544]


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('layer', [False, True])
@pytest.mark.parametrize('width', WIDTHS)
def test_widths(dev, dtype, layer, width):
    if layer and width == 1:                 # one channel less its mean is 0: nothing is left to compare
        width = 2
    _check(*_case(19, width, dtype, dev, layer, groups=1, act='sigmoid'))


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('rows', [1, 2, 63, 1000])
@pytest.mark.parametrize('keep8', [False, True])
def test_rows(dev, dtype, rows, keep8):
    _check(*_case(rows, 320, dtype, dev, rows % 2 == 1, groups=1, act='tanh'), keep8=keep8)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('rows,width,groups', [(24, 72, 0), (24, 72, 1), (24, 72, 2), (24, 72, 24), (260, 72, 130), (260, 72, 65), (390, 1000, 130),
                                               (128, 2500, 64), (4096, 24, 4), (130, 4200, 130), (200, 520, 100)])
def test_gates(dev, dtype, rows, width, groups):
    for act in ('none', 'sigmoid', 'tanh'):
        _check(*_case(rows, width, dtype, dev, act == 'tanh', groups, act), keep8=act == 'sigmoid')


@pytest.mark.parametrize('dtype', TYPES)
def test_without_the_first_or_the_second_norm(dev, dtype):
    for layer in (False, True):
        for keep8 in (False, True):
            _check(*_case(40, 96, dtype, dev, layer, 2, 'sigmoid', post=False), keep8=keep8)
            _check(*_case(40, 96, dtype, dev, layer, 2, 'none', pre=False), keep8=keep8)
            _check(*_case(40, 96, dtype, dev, layer, 0, 'none', post=False, pre=False, tensor_scale=False), keep8=keep8)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
def test_fp32_parameters(dev, dtype):
    _check(*_case(50, 200, dtype, dev, True, 1, 'sigmoid', params=torch.float32))
    _check(*_case(50, 200, dtype, dev, False, 50, 'none', params=torch.float32), keep8=True)


@pytest.mark.parametrize('dtype', TYPES)
def test_no_weights(dev, dtype):
    p, more, gy, gh = _case(30, 130, dtype, dev)
    p['post_w'] = p['pre_w'] = None
    _check(p, more, gy, gh)


@pytest.mark.parametrize('dtype', TYPES)
def test_norm_rows(dev, dtype):
    for layer, keep8 in ((False, False), (True, True), (True, False)):
        p, more, _, gh = _case(37, 250, dtype, dev, layer)
        leaves = [p[k].requires_grad_(True) for k in ('x', 'pre_w', 'pre_b') if p[k] is not None]
        h = block_norm.norm_rows(*leaves, kind=more['kind'], eps=more['eps'], keep8=keep8)
        q = dict(_as64(p, more), f=None)
        _near(h, ref.forward(q)['h'], 512, 'h')
        grads = torch.autograd.grad(h, leaves, gh)
        want = ref.backward(q, None, gh.double().cpu(), None, _seen(p['x'], keep8))
        for t, k in zip(grads, ('x', 'pre_w', 'pre_b')):
            _near(t, want[k], 512 if k == 'x' else 1100, k)


@pytest.mark.parametrize('dtype', TYPES)
def test_strides_and_leading_dimensions(dev, dtype):
    p, more, gy, gh = _case(24, 104, dtype, dev, True, 2, 'sigmoid')
    wide = lambda t, at: torch.nn.functional.pad(t.detach(), (at, 200 - at), value=float('nan'))[:, at:at + 104]     # noqa: E731
    base = _check(p, more, gy, gh)
    for at in (0, 8, 3):
        out = _check(dict(p, x=wide(p['x'], at), f=wide(p['f'], at), gate=wide(p['gate'], at)), more, wide(gy, at), wide(gh, at))
        for a, b in zip((*base[:2], *base[2].values()), (*out[:2], *out[2].values())):
            assert torch.equal(a, b)
    col = lambda t: t.detach().t().contiguous().t()          # noqa: E731
    out = _check(dict(p, x=col(p['x']), f=col(p['f'])), more, col(gy), gh[:1].expand(24, 104))
    p3 = dict(p, x=p['x'].detach().view(2, 12, 104), f=p['f'].detach().view(2, 12, 104), gate=p['gate'].detach().view(2, 1, 104))
    _check(p3, more, gy.view(2, 12, 104), gh.view(2, 12, 104), keep8=True)


def test_a_gradient_for_one_output_alone(dev):
    """Only y, or only h, has a gradient; parameters of the unused norm get zeros; every subset of inputs gets what it gets together with the others."""
    p, more, gy, gh = _case(33, 72, torch.float32, dev, True, 3, 'sigmoid')
    names = [k for k in p if isinstance(p[k], torch.Tensor)]
    leaves = {k: p[k].requires_grad_(True) for k in names}
    for which in (0, 1):
        outs = block_norm.residual_norm(**dict(p, **leaves), **more)
        grads = dict(zip(names, torch.autograd.grad(outs[which], list(leaves.values()), (gy, gh)[which], allow_unused=True)))
        want = ref.backward(_as64(p, more), gy.double().cpu() if which == 0 else None, gh.double().cpu() if which == 1 else None,
                            _seen(p['f'], False), _seen(outs[0], False))
        for k in names:
            if which == 0 and k in ('pre_w', 'pre_b'):
                assert not grads[k].any()
            else:
                _near(grads[k], want[k], 1024 + 33 * (72 if k == 'scale' else 1), k)
    outs = block_norm.residual_norm(**dict(p, **leaves), **more)
    full = dict(zip(names, torch.autograd.grad(outs, list(leaves.values()), (gy, gh))))
    for k in names:
        only = {n: t.detach().requires_grad_(n == k) for n, t in leaves.items()}
        outs = block_norm.residual_norm(**dict(p, **only), **more)
        g, = torch.autograd.grad(outs, [only[k]], (gy, gh))
        assert torch.equal(g, full[k]), k


def test_what_is_kept(dev):
    """keep8: 2 x 1.03 bytes a value besides the outputs; without: x may still be overwritten (it is not kept)."""
    rows, width = 512, 2048
    p, more, gy, gh = _case(rows, width, torch.bfloat16, dev, tensor_scale=False)
    x = p.pop('x')
    for t in (x, p['f']):
        t.requires_grad_(True)
    torch.cuda.synchronize()
    before = _requested()
    y, h = block_norm.residual_norm(x, keep8=True, **p, **more)
    held = _requested() - before - 2 * 2 * rows * width
    assert held <= 2 * rows * width * (1 + 1 / 32) + 4 * 4 * rows + 8192
    with torch.no_grad():
        y2, h2 = block_norm.residual_norm(x, keep8=True, **p, **more)
    assert torch.equal(y, y2) and torch.equal(h, h2) and not y2.requires_grad


def test_no_rows(dev):
    x = torch.zeros(0, 24, device=dev, requires_grad=True)
    w = torch.ones(24, device=dev, requires_grad=True)
    y, h = block_norm.residual_norm(x, x * 1, pre_w=w)
    gx, gw = torch.autograd.grad((y, h), (x, w), (torch.zeros_like(y), torch.zeros_like(h)))
    assert y.shape == h.shape == gx.shape == (0, 24) and not gw.any()


def test_zero_rows_constant_rows_and_not_a_number(dev):
    """A row of zeros divides by sqrt(eps), a constant row has no deviation; a nan or inf stays in its own row (and in sums over rows)."""
    for dtype in TYPES:
        x = torch.randn(8, 64, device=dev).to(dtype)
        x[1] = 0
        x[2] = 3.0
        f = torch.zeros_like(x)
        for kind in ('rms', 'layer'):
            y, h = block_norm.residual_norm(x, f, kind=kind)
            assert torch.equal(y, x) and not h[1].any() and h.isfinite().all()
        assert not block_norm.norm_rows(x, kind='layer')[2].any()
        x[4, 7] = float('nan')
        x[5, 9] = float('inf')
        for keep8 in (False, True):
            xx, w = x.clone().requires_grad_(True), torch.ones(64, device=dev, dtype=dtype, requires_grad=True)
            y, h = block_norm.residual_norm(xx, f, pre_w=w, keep8=keep8)
            clean = [0, 1, 2, 3, 6, 7]
            assert h[4].isnan().all() and h[clean].isfinite().all()
            gx, gw = torch.autograd.grad((y, h), (xx, w), (torch.ones_like(y), torch.ones_like(h)))
            assert gx[clean].isfinite().all() and gx[4].isnan().all() and gw[7].isnan() and gw[9].isnan()


def test_more_rows_than_workgroups(dev):
    p, more, gy, gh = _case(70001, 16, torch.bfloat16, dev, False, 1, 'sigmoid')
    _check(p, more, gy, gh, keep8=True)
    p, more, gy, gh = _case(20000, 40, torch.float32, dev, True, 10000, 'tanh')
    _check(p, more, gy, gh)


def test_offsets_behind_32_bits(dev):
    """2^31 + elements a tensor: the last rows are those of a short call on them."""
    rows, width = 131080, 16384
    x = torch.zeros(rows, width, dtype=torch.bfloat16, device=dev)
    f = torch.zeros_like(x)
    x[-5:], f[-5:] = torch.randn(5, width, device=dev), torch.randn(5, width, device=dev)
    w = torch.rand(width, device=dev)
    with torch.no_grad():
        y, h = block_norm.residual_norm(x, f, 0.5, post_w=w, pre_w=w)
        y5, h5 = block_norm.residual_norm(x[-5:], f[-5:], 0.5, post_w=w, pre_w=w)
    assert torch.equal(y[-5:], y5) and torch.equal(h[-5:], h5) and not h[:-5].any()


def test_repeat_other_stream_and_two_graphs(dev):
    p, more, gy, gh = _case(1000, 600, torch.bfloat16, dev, True, 4, 'sigmoid')

    def step(x):
        q = {k: (x if k == 'x' else v).detach().requires_grad_(True) if isinstance(v, torch.Tensor) else v for k, v in p.items()}
        y, h = block_norm.residual_norm(keep8=True, **q, **more)
        return (y.detach(), h.detach(), *torch.autograd.grad((y, h), [v for v in q.values() if isinstance(v, torch.Tensor)], (gy, gh)))

    want = step(p['x'])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step(p['x'])
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(other, want))
    graphs = []
    for src in (p['x'].clone(), torch.randn_like(p['x'])):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(src)
        graphs.append((graph, src, out))
    for k in range(3):
        for graph, _, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for graph, src, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, step(src)))
            src.copy_(torch.randn_like(src))
