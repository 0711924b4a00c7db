"""Layers that keep their inputs in 8 bits and fused norms run together: residual_rows, the FC stacks of the heads, head modules.

A chain's result is its operators' results, bit for bit: the test walks the chain operator by operator on detached tensors, checks each
against float64 on the inputs and gradients that it has there (bounds: test_act8_linear_gpu.py, test_block_norm_gpu.py), and
demands that the module's outputs and gradients are the walk's.  So no tolerance is needed for the chain."""
import pytest
import torch
from torch import nn

import test_act8_linear_gpu as lin
import test_block_norm_gpu as bn
from detmatch_amd import act8, block_norm, configs
from detmatch_amd.bn_relu import fc_rows
from detmatch_amd.pcdet.config import ConfigDict
from detmatch_amd.residual_rows import ResidualRows

pytestmark = [pytest.mark.gpu, pytest.mark.timeout(300)]
KINDS = [('rms', None, False), ('rms', 'sigmoid', True), ('layer', 'tanh', True), ('layer', 'sigmoid', False)]


def _requested():
    """Bytes that are asked for and alive (memory_allocated counts an allocator's blocks, which may be up to 1 MiB larger than asked for)."""
    return torch.cuda.memory_stats()['requested_bytes.all.current']


def _module(channels, hidden, blocks, kind, gate, keep8, dtype, dev):
    torch.manual_seed(channels + hidden)
    m = ResidualRows(channels, hidden, blocks, kind, gate, 0.7, keep8=keep8)
    with torch.no_grad():
        for name, p in m.named_parameters():
            if 'fc' not in name or 'bias' in name:
                p.add_(torch.randn(p.shape) * 0.2)
    return m.to(dev, dtype)


def _leaf(t):
    return None if t is None else t.detach().clone().requires_grad_(True)


def _walk(m, x, gh):
    """The chain's result, its input's and its parameters' gradients, operator by operator, each checked against float64."""
    more = dict(kind=m.kind, eps=m.eps)
    steps, stream = [], x
    x0, w0, b0 = _leaf(x), _leaf(m.norm_w[0]), _leaf(m._bias(0))
    h0 = block_norm.norm_rows(x0, w0, b0, keep8=m.keep8, **more)
    h = h0.detach()
    for i, b in enumerate(m.blocks):
        p1, p2 = [[_leaf(t) for t in (a, fc.weight, fc.bias)] for a, fc in ((h, b.fc1), (h, b.fc2))]
        a1 = act8.linear(*p1, relu=True)
        p2[0] = _leaf(a1)
        f = act8.linear(*p2)
        q = dict(x=_leaf(stream), f=_leaf(f), gate=_leaf(b.gate), scale=_leaf(b.scale), post=True, pre=True, post_w=_leaf(b.post_w),
                 post_b=_leaf(b.post_b), pre_w=_leaf(m.norm_w[i + 1]), pre_b=_leaf(m._bias(i + 1)))
        y, h = block_norm.residual_norm(gate_act=m.gate, keep8=m.keep8, **q, **more)
        steps.append((p1, a1, p2, f, q, y, h))
        stream, h = y.detach(), h.detach()
    grads, gy = {}, None
    for i in reversed(range(len(steps))):
        p1, a1, p2, f, q, y, hh = steps[i]
        names = [k for k, v in q.items() if isinstance(v, torch.Tensor)]
        outs, gs = ([hh], [gh]) if gy is None else ([y, hh], [gy, gh])
        got = dict(zip(names, torch.autograd.grad(outs, [q[k] for k in names], gs)))
        bn._check({k: v.detach() if isinstance(v, torch.Tensor) else v for k, v in q.items()}, dict(gate_act=m.gate, **more),
                  torch.zeros_like(x) if gy is None else gy, gh, m.keep8)
        lin._check(*[t.detach().clone() for t in p2], got['f'], False)
        g2 = torch.autograd.grad(f, p2, got['f'])
        lin._check(*[t.detach().clone() for t in p1], g2[0], True)
        g1 = torch.autograd.grad(a1, p1, g2[0])
        for k in ('gate', 'scale', 'post_w', 'post_b'):
            grads['blocks.%d.%s' % (i, k)] = got.get(k)
        grads['norm_w.%d' % (i + 1)], grads['norm_b.%d' % (i + 1)] = got['pre_w'], got.get('pre_b')
        grads.update({'blocks.%d.fc1.weight' % i: g1[1], 'blocks.%d.fc1.bias' % i: g1[2], 'blocks.%d.fc2.weight' % i: g2[1],
                      'blocks.%d.fc2.bias' % i: g2[2]})
        gy, gh = got['x'], g1[0]
    leaves = [t for t in (x0, w0, b0) if t is not None]
    first = torch.autograd.grad(h0, leaves, gh)
    grads['norm_w.0'], grads['norm_b.0'] = first[1], first[2] if len(first) > 2 else None
    return h, gy + first[0], grads


@pytest.mark.parametrize('dtype', lin.TYPES)
@pytest.mark.parametrize('kind,gate,keep8', KINDS)
@pytest.mark.parametrize('rows,channels,hidden', [(37, 96, 200), (1, 256, 64), (300, 136, 33)])
def test_blocks_are_their_operators(dev, dtype, kind, gate, keep8, rows, channels, hidden):
    m = _module(channels, hidden, 2, kind, gate, keep8, dtype, dev)
    g = torch.Generator().manual_seed(rows)
    x, gh = (torch.randn(rows, channels, generator=g).to(dtype).to(dev) for _ in range(2))
    xr = x.clone().requires_grad_(True)
    h = m(xr)
    h.backward(gh)
    want, gx, grads = _walk(m, x, gh)
    assert torch.equal(h, want) and torch.equal(xr.grad, gx)
    for name, p in m.named_parameters():
        assert torch.equal(p.grad, grads[name]), name
    with torch.no_grad():                      # inference: the same rows, and each row by itself
        assert torch.equal(m(x), want)
        assert torch.equal(m(x.view(1, rows, channels))[0], want)


def test_rows_do_not_depend_on_their_batch(dev):
    m = _module(96, 64, 2, 'rms', 'sigmoid', True, torch.bfloat16, dev).eval()
    x = torch.randn(64, 96, device=dev).to(torch.bfloat16)
    with torch.no_grad():
        y = m(x)
        z = m(torch.cat([x[32:], x[:32] * 100]))
    assert torch.equal(y[32:], z[:32]) and m(x[:0]).shape == (0, 96)


def _roi_head(dev, **more):
    from detmatch_amd.pcdet.roi_heads import PVRCNNHead
    cfg = ConfigDict(configs.pvrcnn_kitti_model()['pcdet_model']).ROI_HEAD
    cfg.update(more)
    torch.manual_seed(0)
    return PVRCNNHead(input_channels=128, model_cfg=cfg, num_class=1).to(dev)


def test_roi_head_stacks(dev):
    """The stacks of the RoI head with 8-bit layers and residual blocks: the forward pass of a layer is a plain product, so the first
    layer's output is off by what two ways of multiplying in fp32 may differ; results do not change with what is kept."""
    head = _roi_head(dev, KEEP8=True, DP_RATIO=0.0, SHARED_RESIDUAL=dict(hidden=512, blocks=2, gate='sigmoid', keep8=True))
    assert head.keep8 and isinstance(list(head.shared_fc_layer)[-1], ResidualRows)
    x = torch.randn(96, 27648, device=dev).requires_grad_(True)
    first = act8.linear(x, head.shared_fc_layer[0].weight.squeeze(-1))
    xd, wd = x.detach().double().cpu(), head.shared_fc_layer[0].weight.detach().double().cpu().squeeze(-1).t()
    lin._inside(first.detach().cpu(), xd @ wd, lin._bound(xd, wd, xd @ wd, torch.float32), 'first layer')
    for train in (True, False):
        head.train(train)
        head.zero_grad()
        shared = fc_rows(head.shared_fc_layer, x, head.keep8)
        out = fc_rows(head.cls_layers, shared, head.keep8), fc_rows(head.reg_layers, shared, head.keep8)
        (out[0].square().mean() + out[1].square().mean()).backward()
        for name, p in head.named_parameters():
            if not name.startswith('roi_grid_pool'):
                assert p.grad is not None and bool(p.grad.isfinite().all()) and bool(p.grad.any()), name


def test_box_head_keeps_less(dev):
    from detmatch_amd.mm2d.faster_rcnn import Shared2FCBBoxHead
    cfg = dict(num_classes=3, bbox_coder=dict(target_means=[0.] * 4, target_stds=[0.1, 0.1, 0.2, 0.2]),
               loss_cls=dict(type='FocalLoss', use_sigmoid=True, loss_weight=1.0, gamma=2.0, alpha=0.5), loss_bbox=dict(type='L1Loss'))
    torch.manual_seed(0)
    plain = Shared2FCBBoxHead(**cfg).to(dev)
    small = Shared2FCBBoxHead(keep8=True, **cfg).to(dev)
    small.load_state_dict(plain.state_dict())
    kept = []
    feats = torch.randn(500, 256, 7, 7, device=dev)
    for head in (plain, small):
        for _ in range(2):                     # (the second time: what the library allocates once, and gradients, are there already)
            x = feats.clone().requires_grad_(True)
            torch.cuda.synchronize()
            before = _requested()
            y = head(x * 1.0)
            torch.cuda.synchronize()
            kept.append(_requested() - before)
            (y[0].sum() + y[1].square().sum()).backward()
            assert all(p.grad is not None and bool(p.grad.isfinite().all()) for p in head.parameters()) and bool(x.grad.isfinite().all())
            del y, x
    # 12 544 channels a row, fp32 -> 8 bits; the outputs of the two layers likewise
    assert kept[1] - kept[3] >= 0.99 * 500 * 12544 * (4 - 33 / 32)
    h = feats.flatten(1)
    with torch.no_grad():
        for fc in small.shared_fcs:
            h = act8.linear(h, fc.weight, fc.bias, relu=True)
        want = [act8.linear(h, fc.weight, fc.bias) for fc in (small.fc_cls, small.fc_reg)]
        assert all(torch.equal(a, b) for a, b in zip(small(feats), want))


def test_a_stack_without_the_option_is_what_it_was(dev):
    torch.manual_seed(0)
    seq = nn.Sequential(nn.Linear(64, 32, bias=False), nn.BatchNorm1d(32), nn.ReLU(), nn.Linear(32, 8)).to(dev)
    x = torch.randn(40, 64, device=dev)
    from detmatch_amd import _lib
    from detmatch_amd.bn_relu import bn_relu_rows
    with torch.no_grad():
        seq.eval()
        want = _lib.blas_linear(bn_relu_rows(_lib.blas_linear(x, seq[0].weight), seq[1], relu=True), seq[3].weight, seq[3].bias)
        assert torch.equal(fc_rows(seq, x), want)


def test_captured_while_an_eager_graph_of_the_same_leaves_lives(dev):
    """A training step captured into a graph, with an eager graph of the same parameters alive, replayed with eager work between."""
    m = _module(96, 64, 2, 'layer', 'tanh', True, torch.bfloat16, dev)
    params = list(m.parameters())
    x, gh = (torch.randn(50, 96, device=dev).to(torch.bfloat16) for _ in range(2))

    def step(x):
        leaves = [p.detach().requires_grad_(True) for p in params]       # (leaves of the step's own: gradients are its results)
        h = torch.func.functional_call(m, dict(zip([n for n, _ in m.named_parameters()], leaves)), (x,))
        return (h.detach(), *torch.autograd.grad(h, leaves, gh))

    alive = m(x.clone().requires_grad_(True))                            # an eager graph of m's own leaves
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(x)
    for _ in range(3):
        graph.replay()
        want = step(x)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
        x.copy_(torch.randn_like(x))
    alive.backward(gh)
    assert all(p.grad is not None for p in params)


def test_differentiable_once_and_weights_changed_in_place_are_noticed(dev):
    m = _module(64, 32, 1, 'rms', None, False, torch.float32, dev)
    x = torch.randn(8, 64, device=dev, requires_grad=True)
    g, = torch.autograd.grad(m(x).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    for p in (m.blocks[0].fc1.weight, m.blocks[0].post_w, m.blocks[0].scale):
        y = m(x)
        with torch.no_grad():
            p.mul_(2)
        with pytest.raises(RuntimeError):
            y.sum().backward()


def test_a_training_step_of_the_detector(dev, monkeypatch):
    """One iteration of the 3D detector's training with the options on: it runs, and every parameter of the head's stacks is reached."""
    from detmatch_amd.pcdet.workload import PretrainWorkload
    model = configs.pvrcnn_kitti_model

    def with_options(*args, **kw):
        cfg = model(*args, **kw)
        cfg['pcdet_model']['ROI_HEAD'].update(KEEP8=True, SHARED_RESIDUAL=dict(hidden=512, blocks=1, gate='sigmoid', keep8=True))
        return cfg

    monkeypatch.setattr(configs, 'pvrcnn_kitti_model', with_options)
    wl = PretrainWorkload(1, dev, recipe='pretrain_pvrcnn', iters_per_epoch=1, max_epochs=1)
    head = [m for m in wl.model.modules() if type(m).__name__ == 'PVRCNNHead'][0]
    assert head.keep8
    before = {n: p.detach().clone() for n, p in head.named_parameters() if 'fc_layer' in n}
    assert bool(torch.isfinite(torch.as_tensor(wl.run())).all())
    after = dict(head.named_parameters())
    assert all(bool(p.isfinite().all()) for p in after.values())
    assert all(not torch.equal(after[n], p) for n, p in before.items())
