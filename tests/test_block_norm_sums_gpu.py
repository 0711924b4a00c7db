"""Sums over rows and walks over many rows in block_norm's backward pass, against float64.

Each workgroup walks at least three rows here, the last ones of some of them do not exist, and gradients lean towards what they are multiplied with, so
that sums over rows do not cancel: a bound is a small part of the sum itself (asserted), and a sum that lacks a row or adds one twice is outside of it.

Bounds, in units of 2^-24 of the magnitudes of tests/_block_norm_ref.py.  A term: normalised values of y 256, dy 512, what follows from it 768 (a
row's sum is 16 additions in a thread, a tree of 6 and 16 waves: 40; a deviation half of it and the rounding of what it is taken of; dy has
two of these and a product in it, what comes from dy three).  The sum: one rounding for each addition that a term goes through, as the kernel adds (see
_additions): the rows of one thread (for the scale times its channels), the teams of a workgroup, the workgroups in 32 slices, the slices."""
import pytest
import torch

import _block_norm_ref as ref
import test_block_norm_gpu as bn
from detmatch_amd import block_norm

pytestmark = [pytest.mark.gpu, pytest.mark.timeout(300)]
TERM = dict(x=512, f=768, gate=768, scale=768, post_w=768, post_b=512, pre_w=256, pre_b=1)


def _additions(rows, width, groups):
    """-> (trips of a team, {what: additions that a term may go through})"""
    chunks, t = -(-width // 8), 8
    while t < min(chunks, 512):
        t *= 2
    if chunks > t:
        t = 1024
    block = max(t, 512)
    teams, most, by_unit = block // t, 512 if block == 512 else 256, groups > 64
    units, y = (groups, 1) if by_unit else (rows // max(groups, 1), max(groups, 1))
    x = min(-(-units // teams), max(most // y, 1))
    trips = -(-units // (x * teams)) * (rows // groups if by_unit else 1)
    out = dict.fromkeys(('post_w', 'post_b', 'pre_w', 'pre_b'), trips + teams + -(-x * y // 32) + 32)
    out['gate'] = rows // groups if by_unit else trips + teams + -(-x // 32) + 32
    out['scale'] = trips * 8 * -(-chunks // t) + 6 + 16 + -(-x * y // 1024) + 32 + 5
    return trips, out


def _inputs(rows, width, dtype, dev, layer, groups, act, **form):
    """bn._case's, with gradients that lean towards f and y and have a mean."""
    p, more, gy, gh = bn._case(rows, width, dtype, dev, layer, groups, act, **form)
    if groups:
        p['gate'] = (p['gate'].float().abs() + 0.25).to(dtype)
    gy = (gy.float() + 0.5 * p['f'].float() + 0.5).to(dtype)
    gh = (gh.float() + 0.5 * p['x'].float() + 0.5).to(dtype)
    return p, more, gy, gh


def _bound(want, dtype, ulps):
    v, mag = want
    return ulps * bn.U * mag + (0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2 * (1 + 1e-3)) * v.abs() + torch.finfo(dtype).tiny


def _sharp(k, v, bound):
    """Most sums are at least 20 bounds large."""
    share = float((bound <= 0.05 * v.abs()).double().mean())
    assert share >= 0.8, '%s: the bound is as large as the sum itself at %.2f of the elements' % (k, 1 - share)


def _want(p, more, gy, gh, f_seen, y_seen, dev):
    """The reference's gradients, computed where the inputs are."""
    q = {k: v.detach().double() if isinstance(v, torch.Tensor) else v for k, v in p.items()}
    q.update(scale=float(q['scale']), layer=more['kind'] == 'layer', eps=more['eps'], act=more['gate_act'])
    with torch.device(dev):
        return ref.forward(q), ref.backward(q, gy.double(), None if gh is None else gh.double(), f_seen, y_seen)


def _check(p, more, gy, gh, keep8, dev):
    rows, width = p['x'].shape
    groups = p['gate'].shape[0] if p['gate'] is not None else 0
    trips, additions = _additions(rows, width, groups)
    assert trips >= 3
    names = [k for k in TERM if isinstance(p[k], torch.Tensor)]
    leaves = {k: p[k].detach().requires_grad_(True) for k in names}
    y, h = block_norm.residual_norm(**dict(p, **leaves), keep8=keep8, **more)
    outs, gs = ([y, h], [gy, gh]) if p['pre'] else ([y], [gy])
    got = dict(zip(names, torch.autograd.grad(outs, [leaves[k] for k in names], gs)), y=y.detach(), h=h.detach() if p['pre'] else None)
    seen = [bn.act8.unpack(bn.act8.pack(t.detach())).double() if keep8 else t.detach().double() for t in (p['f'], y)]
    out, want = _want(p, more, gy, gh if p['pre'] else None, *seen, dev)
    for k, v in {**out, **{k: want[k] for k in names}}.items():
        bound = _bound(v, got[k].dtype, dict(TERM, y=256, h=512)[k] + additions.get(k, 0))
        # (a value from the type's largest, M, plus half a step on is rounded to infinity, in fp16 from 65 520: both count as M)
        most = torch.finfo(got[k].dtype).max
        far = (got[k].double().reshape(v[0].shape).clamp(-most, most) - v[0].clamp(-most, most)).abs() - bound
        assert bool((far <= 0).all()), '%s (%s, keep8 %s): %g over its bound' % (k, more, keep8, float(far.max()))
        if k in additions and not (k == 'gate' and groups > 64):
            _sharp(k, v[0], bound)


CASES = [(1602, 2056, 0), (1602, 2056, 3), (1602, 2056, 1602), (1602, 4096, 0), (1602, 4096, 3), (1602, 4096, 1602), (801, 5000, 0), (801, 5000, 3),
         (801, 5000, 801), (801, 8192, 0), (801, 8192, 3), (801, 8192, 801), (600, 12544, 0), (600, 12544, 3), (600, 12544, 600),
         (70002, 16, 0), (70002, 16, 3), (70002, 16, 70002), (33000, 72, 66), (30000, 640, 1), (1200, 5000, 600), (1600, 1024, 100), (1200, 4096, 600)]


@pytest.mark.parametrize('dtype', bn.TYPES)
@pytest.mark.parametrize('rows,width,groups', CASES)
def test_many_rows_a_team(dev, dtype, rows, width, groups):
    for layer in (False, True):
        for keep8 in (False, True):
            _check(*_inputs(rows, width, dtype, dev, layer, groups, 'sigmoid' if layer else 'none'), keep8, dev)


@pytest.mark.parametrize('dtype', bn.TYPES)
@pytest.mark.parametrize('form', [dict(post=False), dict(pre=False), dict(post=False, pre=False), dict(tensor_scale=False), dict(params=torch.float32)],
                         ids=lambda f: '-'.join(f))
def test_other_forms_over_many_rows(dev, dtype, form):
    for groups in (0, 3):
        for layer in (False, True):
            for keep8 in (False, True):
                _check(*_inputs(6006, 520, dtype, dev, layer, groups, 'tanh', **form), keep8, dev)


def test_gradients_behind_32_bits(dev):
    """2^31 + elements a tensor, exact and in codes: the last rows' gradients are those of a short call on them, all others are 0."""
    rows, width = 131080, 16384
    x = torch.zeros(rows, width, dtype=torch.bfloat16, device=dev)
    x[-5:] = torch.randn(5, width, device=dev)
    f, gy, gh = x.flip(1), x * 0.5, x.roll(1, 1)
    w = torch.rand(width, device=dev) + 0.5
    for keep8 in (False, True):
        out = []
        for at in (0, rows - 5):
            leaves = [t[at:].detach().requires_grad_(True) for t in (x, f)]
            y, h = block_norm.residual_norm(*leaves, 0.5, post_w=w, pre_w=w, keep8=keep8)
            out.append(torch.autograd.grad((y, h), leaves, (gy[at:], gh[at:])))
            del y, h
        for whole, last in zip(*out):
            assert torch.equal(whole[-5:], last) and bool(last.any()) and not bool(whole[:-5].any())
        del out, whole, last
