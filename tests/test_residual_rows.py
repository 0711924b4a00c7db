"""Host side of residual blocks and of the heads' options for 8-bit layers."""
import pytest
import torch
from torch import nn

from detmatch_amd import _lib, configs
from detmatch_amd.bn_relu import fc_rows
from detmatch_amd.pcdet.config import ConfigDict
from detmatch_amd.residual_rows import ResidualRows


def test_what_is_refused():
    for kw in (dict(blocks=0), dict(kind='batch'), dict(gate='relu'), dict(gate='none')):
        with pytest.raises(ValueError):
            ResidualRows(16, 8, **kw)
    with pytest.raises(ValueError):
        ResidualRows(0, 8)
    with pytest.raises(ValueError):
        ResidualRows(16, 0)
    with pytest.raises(_lib.DetMatchHipError):
        ResidualRows(16, 8)(torch.zeros(2, 16))
    with pytest.raises(_lib.DetMatchHipError):
        fc_rows(nn.Sequential(nn.Linear(16, 8)), torch.zeros(2, 16), keep8=True)
    with pytest.raises(TypeError):
        fc_rows(nn.Sequential(nn.GELU()), torch.zeros(2, 16))


def test_parameters():
    names = set(ResidualRows(16, 8, 2).state_dict())
    block = {'fc1.weight', 'fc1.bias', 'fc2.weight', 'fc2.bias', 'post_w', 'scale'}
    assert names == {'blocks.%d.%s' % (i, n) for i in range(2) for n in block} | {'norm_w.0', 'norm_w.1', 'norm_w.2'}
    names = set(ResidualRows(16, 8, 1, 'layer', 'tanh').state_dict())
    assert names == {'blocks.0.' + n for n in block | {'post_b', 'gate'}} | {'norm_w.0', 'norm_w.1', 'norm_b.0', 'norm_b.1'}
    m = ResidualRows(16, 8, scale=0.25)
    assert float(m.blocks[0].scale.detach()) == 0.25


def _roi_head(**more):
    from detmatch_amd.pcdet.roi_heads import PVRCNNHead
    cfg = ConfigDict(configs.pvrcnn_kitti_model()['pcdet_model']).ROI_HEAD
    cfg.update(more)
    torch.manual_seed(0)
    return PVRCNNHead(input_channels=128, model_cfg=cfg, num_class=1)


def test_roi_head_options():
    plain, small = _roi_head(), _roi_head(KEEP8=True)
    assert not plain.keep8 and small.keep8
    a, b = plain.state_dict(), small.state_dict()
    assert list(a) == list(b) and all(torch.equal(a[k], b[k]) for k in a)
    more = _roi_head(SHARED_RESIDUAL=dict(hidden=64, blocks=3, kind='layer', gate='tanh')).state_dict()
    assert set(a) < set(more)
    last = len(plain.shared_fc_layer)
    assert all(k.startswith('shared_fc_layer.%d.' % last) for k in set(more) - set(a))
    with pytest.raises(TypeError):
        _roi_head(SHARED_RESIDUAL=dict(hidden=64, width=3))


def test_box_head_option():
    from detmatch_amd.mm2d.faster_rcnn import Shared2FCBBoxHead
    cfg = dict(in_channels=8, fc_out_channels=16, roi_feat_size=2, num_classes=3,
               bbox_coder=dict(target_means=[0.] * 4, target_stds=[0.1, 0.1, 0.2, 0.2]),
               loss_cls=dict(type='FocalLoss', use_sigmoid=True, loss_weight=1.0, gamma=2.0, alpha=0.5), loss_bbox=dict(type='L1Loss'))
    plain, small = Shared2FCBBoxHead(**cfg), Shared2FCBBoxHead(keep8=True, **cfg)
    assert not plain.keep8 and small.keep8 and list(plain.state_dict()) == list(small.state_dict())
    x = torch.randn(5, 8, 2, 2)
    assert plain(x)[0].shape == (5, 4)
    with pytest.raises(_lib.DetMatchHipError):
        small(x)
