"""Host side of the norms around a residual block: refusals, and the formulas of the tests themselves."""
import ctypes

import pytest
import torch

import _block_norm_ref as ref
from detmatch_amd import _lib, block_norm


def test_what_is_refused():
    x = torch.zeros(6, 16)
    call = block_norm.residual_norm
    with pytest.raises(_lib.DetMatchHipError):
        call(x, x)
    with pytest.raises(_lib.DetMatchHipError):
        block_norm.norm_rows(x)
    for bad in (dict(kind='batch'), dict(gate_act='relu'), dict(eps=-1.0), dict(eps=float('nan')), dict(post_w=torch.zeros(15)),
                dict(pre_w=torch.zeros(1, 16)), dict(pre_b=torch.zeros(16)), dict(post=False, post_w=torch.zeros(16)),
                dict(pre=False, pre_w=torch.zeros(16)), dict(gate=torch.zeros(15)), dict(gate=torch.zeros(4, 16)),
                dict(gate=torch.zeros(0, 16)), dict(scale=torch.zeros(2))):
        with pytest.raises(ValueError):
            call(x, x, **bad)
    for bad in (dict(gate=torch.zeros(16).half()), dict(pre_w=torch.zeros(16).half()), dict(scale=torch.zeros(1).double()),
                dict(pre_w=torch.zeros(16), post_w=torch.zeros(16).bfloat16())):
        with pytest.raises(TypeError):
            call(x, x, **bad)
    with pytest.raises(TypeError):
        call(x.bfloat16(), x.bfloat16(), pre_w=torch.zeros(16).bfloat16(), post_w=torch.zeros(16))
    with pytest.raises(TypeError):
        call(x.double(), x.double())
    with pytest.raises(TypeError):
        call(x, x.half())
    with pytest.raises(ValueError):
        call(x, torch.zeros(6, 15))
    with pytest.raises(ValueError):
        call(x, None)
    with pytest.raises(ValueError):
        call(torch.zeros(6, 0), torch.zeros(6, 0))
    with pytest.raises(ValueError):
        call(torch.zeros(()), torch.zeros(()))


def test_entry_points_check_their_arguments():
    L = _lib.lib()
    p, bad = 4096, 1
    q = _lib.BlockNorm()
    q.dtype, q.width, q.rows, q.post, q.eps, q.scale_host = 0, 16, 4, 1, 1e-6, 1.0
    assert L.dm_block_norm_max_width() == 16384

    def forward(x=p, ldx=16, f=p, ldf=16, y=p, h=p, **change):
        r = _lib.BlockNorm.from_buffer_copy(q)
        for k, v in change.items():
            setattr(r, k, v)
        return L.dm_block_norm_forward(ctypes.byref(r), x, ldx, f, ldf, y, h, None)

    assert forward(dtype=3) == bad and forward(width=0) == bad and forward(rows=-1) == bad and forward(width=16385, ldx=1 << 15) == 4
    assert forward(gate_act=3) == bad and forward(eps=-1.0) == bad and forward(groups=1) == bad and forward(gate=p) == bad
    assert forward(gate=p, groups=3, ld_gate=16) == bad and forward(gate=p, groups=2, ld_gate=8) == bad
    assert forward(x=None) == bad and forward(ldx=15) == bad and forward(ldf=15) == bad and forward(y=None) == bad
    assert forward(f=None) == bad and forward(f=None, y=None, h=None) == bad and forward(f_codes=p) == bad
    assert forward(f_codes=p + 4, f_exps=p) == bad and forward(layer=1, f_rstd=p) == bad
    assert forward(rows=0) == 0

    def backward(gy=p, gh=p, y=p, f=p, dgate=None, dpre_w=None, dpost_w=None, dpost_b=None, dscale=None, ws=p, nb=1 << 40, **change):
        r = _lib.BlockNorm.from_buffer_copy(q)
        r.f_rstd = r.y_rstd = p
        for k, v in change.items():
            setattr(r, k, v)
        return L.dm_block_norm_backward(ctypes.byref(r), gy, 16, gh, 16, y, 16, f, 16, None, None, dgate, dpre_w, None, dpost_w, dpost_b,
                                        dscale, ws, nb, None)

    assert backward(rows=0) == bad and backward(gy=None, gh=None) == bad and backward(y=None) == bad and backward(y_rstd=None) == bad
    assert backward(f_rstd=None) == bad and backward(layer=1) == bad and backward(f=None, dscale=p) == bad and backward(dgate=p) == bad
    assert backward(gh=None, dpre_w=p) == bad and backward(dpost_b=p) == bad and backward(post=0, dpost_w=p) == bad
    assert backward(f_codes=p, f_exps=p) == bad and backward(y_codes=p, y_exps=p) == bad       # codes of both, or of neither
    assert backward(ws=None) == 2 and backward(nb=16) == 2
    assert L.dm_block_norm_workspace_bytes(0, 16, 0) == 0 and L.dm_block_norm_workspace_bytes(4, 16385, 0) == 0
    assert L.dm_block_norm_workspace_bytes(4, 16, 0) >= 4 * (5 * 16 + 1)


@pytest.mark.parametrize('layer', [False, True])
@pytest.mark.parametrize('act,groups', [('none', 0), ('none', 1), ('sigmoid', 2), ('tanh', 6)])
@pytest.mark.parametrize('post', [True, False])
def test_formulas_are_autograds(layer, act, groups, post):
    """The tests' gradients are those of torch's autograd in float64, and of differences."""
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)      # noqa: E731
    p = dict(x=r(6, 10), f=r(6, 10), gate=r(groups, 10) if groups else None, scale=0.7, post=post, post_w=r(10) if post else None,
             post_b=r(10) if post and layer else None, pre_w=r(10), pre_b=r(10) if layer else None, layer=layer, eps=1e-3, act=act)
    gy, gh = r(6, 10), r(6, 10)
    names = [k for k in ('x', 'f', 'gate', 'post_w', 'post_b', 'pre_w', 'pre_b') if p[k] is not None]
    q = dict(p, **{k: p[k].clone().requires_grad_(True) for k in names}, scale=torch.tensor(0.7, dtype=torch.float64, requires_grad=True))
    out = ref.forward(q)
    want = torch.autograd.grad((out['y'][0] * gy).sum() + (out['h'][0] * gh).sum(), [q[k] for k in names] + [q['scale']])
    got = ref.backward(p, gy, gh, p['f'], ref.forward(p)['y'][0])
    for k, v in zip(names + ['scale'], want):
        torch.testing.assert_close(got[k][0].reshape(v.shape), v, rtol=1e-9, atol=1e-9)
        assert bool((got[k][0].abs() <= got[k][1] * (1 + 1e-9)).all())

    def loss(q):
        o = ref.forward(q)
        return float((o['y'][0] * gy).sum() + (o['h'][0] * gh).sum())

    for k in names:
        d = r(*p[k].shape)
        diff = (loss(dict(p, **{k: p[k] + 1e-5 * d})) - loss(dict(p, **{k: p[k] - 1e-5 * d}))) / 2e-5
        assert abs(diff - float((got[k][0] * d).sum())) < 1e-6 * (1 + abs(diff))
