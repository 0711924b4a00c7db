"""What torch's other ways of differentiating and recording would lose in silence is refused: tangents of forward-mode derivatives, traces
without gradients."""
import pytest
import torch
from torch.autograd import forward_ad

from detmatch_amd import _lib, act8, block_norm

ROWS, CHANNELS = 6, 16
SHAPES = dict(x=(ROWS, CHANNELS), f=(ROWS, CHANNELS), w=(8, CHANNELS), b=(8,), scale=(1,), gate=(2, CHANNELS), post_w=(CHANNELS,), pre_w=(CHANNELS,))


def _linear(q):
    return act8.linear(q['x'], q['w'], q['b'])


def _residual(q):
    return block_norm.residual_norm(q['x'], q['f'], q['scale'], q['gate'], 'sigmoid', post_w=q['post_w'], pre_w=q['pre_w'])


def _norm(q):
    return block_norm.norm_rows(q['x'], q['pre_w'])


CALLS = [(_linear, k) for k in ('x', 'w', 'b')] + [(_residual, k) for k in ('x', 'f', 'scale', 'gate', 'post_w', 'pre_w')] + [(_norm, k) for k in ('x', 'pre_w')]


@pytest.mark.parametrize('call,name', CALLS)
def test_a_tangent_is_refused(call, name):
    q = {k: torch.ones(s) for k, s in SHAPES.items()}
    with forward_ad.dual_level():
        with pytest.raises(_lib.DetMatchHipError):          # no tangent: as ever (host tensors are refused last)
            call(q)
        q[name] = forward_ad.make_dual(q[name], torch.ones_like(q[name]))
        with pytest.raises(NotImplementedError):
            call(q)
        with torch.no_grad(), pytest.raises(NotImplementedError):
            call(q)
    with pytest.raises(NotImplementedError):
        torch.func.jvp(lambda t: call(dict(q, **{name: t})), (torch.ones(SHAPES[name]),), (torch.ones(SHAPES[name]),))


@pytest.mark.parametrize('call', [_linear, _residual, _norm, lambda q: act8.unpack(act8.pack(q['x'])),
                                  lambda q: q['x'] + act8.unpack(act8.Act8(torch.zeros(6, 32, dtype=torch.uint8), torch.zeros(6, 1, dtype=torch.uint8),
                                                                           (6, 16), torch.float32))])
def test_a_trace_without_gradients_is_refused(call):
    q = {k: torch.ones(s) for k, s in SHAPES.items()}
    with pytest.raises(NotImplementedError):
        torch.jit.trace(lambda x: call(dict(q, x=x)), (q['x'],), check_trace=False)
