"""A nan or an infinity in one group of rows that share their gates stays out of every other group's results."""
import pytest
import torch

import test_block_norm_gpu as bn
from detmatch_amd import block_norm

pytestmark = [pytest.mark.gpu, pytest.mark.timeout(300)]


@pytest.mark.parametrize('dtype', bn.TYPES)
@pytest.mark.parametrize('keep8', [False, True])
@pytest.mark.parametrize('width', [72, 2056, 4096, 4200, 5000, 8192, 12544])
def test_a_nan_or_infinity_stays_in_its_group(dev, dtype, keep8, width):
    """2 x 130 and 3 x 90 rows do not divide the workgroups of a group: the last trip of most of them has no row of its own, and the numbers behind
    the group's end are the next group's.  The other groups' results are bit for bit those beside a clean group."""
    for groups, each in ((2, 130), (3, 90)):
        for layer in (False, True):
            p, more, gy, gh = bn._case(groups * each, width, dtype, dev, layer, groups, 'sigmoid')
            bad = dict(p, x=p['x'].clone(), f=p['f'].clone())
            at = (groups - 1) * each                      # the first rows of the last group
            for r in range(min(each, 40)):
                bad['x'][at + r, (7 * r + 3) % width] = float('nan')
                bad['f'][at + r, (5 * r + 9) % width] = float('inf')
            out = []
            for q in (p, bad):
                leaves = {k: q[k].detach().requires_grad_(True) for k in ('x', 'f', 'gate')}
                y, h = block_norm.residual_norm(**dict(q, **leaves), keep8=keep8, **more)
                out.append((y.detach(), h.detach(), *torch.autograd.grad((y, h), list(leaves.values()), (gy, gh))))
            for clean, seen in zip(*out):
                n = groups - 1 if clean.shape[0] == groups else at
                assert bool(clean.isfinite().all()) and torch.equal(clean[:n], seen[:n]), (groups, layer, tuple(clean.shape))
                assert not bool(seen[n:].isfinite().all())
