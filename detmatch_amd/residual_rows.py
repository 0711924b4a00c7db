"""Residual blocks on rows of features: norm -> Linear -> ReLU -> Linear -> norm, times a gate and a scale, added to the stream.

    stream, h = x, N(x; norm[0])
    for each block i:  f = fc2(relu(fc1(h)));  stream, h = stream + scale * act(gate) * N(f; post),  N(that; norm[i + 1])

The last h is the result.  The two layers are act8.linear, everything between them and the next block's first layer is one pass of
block_norm.residual_norm: a block's forward pass is 3 launches at inference and 5 in training (each layer packs its input), and one more for
each layer whose contraction is split or whose rows are copied.  Unlike BatchNorm, no statistics are shared between rows: a row's result
does not depend on which rows, labelled or unlabelled, are in its batch (their number may choose another split of a product, and with
it another rounding), nor on training or evaluation mode."""
import torch
from torch import nn

from . import act8, block_norm


class ResidualBlock(nn.Module):
    """One block's parameters (ResidualRows runs them)."""

    def __init__(self, channels, hidden, layer, gate, scale):
        super().__init__()
        self.fc1, self.fc2 = nn.Linear(channels, hidden), nn.Linear(hidden, channels)
        for fc in (self.fc1, self.fc2):
            nn.init.xavier_uniform_(fc.weight)
            nn.init.zeros_(fc.bias)
        self.post_w = nn.Parameter(torch.ones(channels))
        self.post_b = nn.Parameter(torch.zeros(channels)) if layer else None
        self.gate = nn.Parameter(torch.zeros(channels)) if gate else None
        self.scale = nn.Parameter(torch.full((1,), float(scale)))


class ResidualRows(nn.Module):
    """`blocks` residual blocks on rows (..., channels) of float32, bfloat16 or float16 in the parameters' type.

    kind: 'rms' or 'layer'; gate: None, 'sigmoid' or 'tanh' of one learnt number per channel (0 at first: with 'tanh' a block adds
    nothing before it has learnt to); scale: the learnt factor's first value; keep8: the norms too keep 8 bits for the backward pass
    (the layers always do)."""

    def __init__(self, channels, hidden, blocks=1, kind='rms', gate=None, scale=1.0, eps=1e-6, keep8=False):
        super().__init__()
        if blocks < 1 or channels < 1 or hidden < 1:
            raise ValueError('blocks %r, channels %r, hidden %r: one at least is wanted of each' % (blocks, channels, hidden))
        if kind not in block_norm.KINDS:
            raise ValueError('kind %r: one of %s' % (kind, sorted(block_norm.KINDS)))
        if gate not in (None, 'sigmoid', 'tanh'):
            raise ValueError("gate %r: None, 'sigmoid' or 'tanh'" % (gate,))
        self.kind, self.gate, self.eps, self.keep8 = kind, gate, float(eps), bool(keep8)
        layer = kind == 'layer'
        self.blocks = nn.ModuleList([ResidualBlock(channels, hidden, layer, gate, scale) for _ in range(blocks)])
        self.norm_w = nn.ParameterList([nn.Parameter(torch.ones(channels)) for _ in range(blocks + 1)])
        self.norm_b = nn.ParameterList([nn.Parameter(torch.zeros(channels)) for _ in range(blocks + 1)]) if layer else None

    def _bias(self, i):
        return None if self.norm_b is None else self.norm_b[i]

    def forward(self, x):
        h = block_norm.norm_rows(x, self.norm_w[0], self._bias(0), self.kind, self.eps, self.keep8)
        for i, b in enumerate(self.blocks):
            f = act8.linear(act8.linear(h, b.fc1.weight, b.fc1.bias, relu=True), b.fc2.weight, b.fc2.bias)
            x, h = block_norm.residual_norm(x, f, b.scale, b.gate, self.gate, True, b.post_w, b.post_b, True, self.norm_w[i + 1],
                                            self._bias(i + 1), self.kind, self.eps, self.keep8)
        return h
