"""8-bit activations (csrc/act8.hip) against their definition in float64."""
import numpy as np
import pytest
import torch

import _act8_ref as ref
from detmatch_amd import act8

pytestmark = [pytest.mark.gpu, pytest.mark.timeout(300)]
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _check(x):
    """codes, exponents and values of pack(x) are the definition's, bit for bit (nan: any nan)."""
    kept = act8.pack(x)
    code, e = ref.pack(x.reshape(-1, x.shape[-1]))
    got = kept.codes.cpu().numpy()
    nan = (code & 127) == 127
    assert np.array_equal(kept.exponents().cpu().numpy(), e)
    assert np.array_equal((got & 127) == 127, nan)
    assert np.array_equal(got[~nan], code[~nan])
    want = ref.unpack(code, e, x.shape[-1], x.dtype)
    back = act8.unpack(kept)
    assert back.shape == x.shape and back.dtype == x.dtype
    torch.testing.assert_close(back.cpu().double().reshape(want.shape), want, rtol=0, atol=0, equal_nan=True)
    return kept


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('rows,width', [(1, 1), (1, 32), (3, 33), (7, 31), (256, 256), (5, 1001), (2, 27648), (130, 8), (64, 2080)])
def test_pack_and_unpack_are_the_definition(dev, dtype, rows, width):
    g = torch.Generator().manual_seed(rows * 31 + width)
    x = torch.randn(rows, width, generator=g) * torch.exp(2 * torch.randn(1, width, generator=g))
    _check(x.to(dtype).to(dev))


@pytest.mark.parametrize('dtype', TYPES)
def test_every_binade_and_every_tie(dev, dtype):
    """Rows whose largest value walks through the type's binades, with values on and beside the borders of two codes."""
    info = torch.finfo(dtype)
    lo, hi = int(np.floor(np.log2(info.tiny))) - 6, int(np.floor(np.log2(info.max)))
    rows = []
    for k in range(lo, hi + 1):
        for top in (1.0, 1.75, 1.7578125, 1.9921875):
            m = np.concatenate([[top], np.linspace(0.0, 1.0, 11), (ref.CODES[3:103:10] + ref.CODES[4:104:10]) / 2 / 448, [2.0 ** -15, 2.0 ** -17]])
            rows.append(np.pad(m, (0, 32 - len(m))) * 2.0 ** k)
    x = torch.from_numpy(np.array(rows)).clamp(max=info.max).to(dtype)
    _check(torch.cat([x, -x]).to(dev))


@pytest.mark.parametrize('dtype', TYPES)
def test_zeros_infinities_and_nan(dev, dtype):
    x = torch.zeros(6, 64)
    x[1] = float('nan')
    x[2, 3], x[2, 40] = float('inf'), -float('inf')
    x[2, 4] = 3.0
    x[3, 10] = torch.finfo(dtype).max
    x[3, 11] = -torch.finfo(dtype).max
    x[4, 5] = float('nan')
    x[4, 6] = 1e-3
    x[5] = -0.0
    kept = _check(x.to(dtype).to(dev))
    assert kept.exponents()[0].eq(0).all()


@pytest.mark.parametrize('dtype', TYPES)
def test_strides_and_alignment(dev, dtype):
    g = torch.Generator().manual_seed(5)
    big = torch.randn(40, 300, generator=g).to(dtype).to(dev)
    for x in (big[:, :256], big[:, 1:257], big[::3, 4:100], big[:, 7:8], big.t(), big[:1].expand(5, 300),
              big.view(4, 10, 300)[:, :, 8:72], big.view(4, 10, 300)[1:, 2:5]):
        _check(x)


def test_empty_and_other_types_of_output(dev):
    kept = act8.pack(torch.zeros(0, 40, device=dev))
    assert act8.unpack(kept).shape == (0, 40)
    x = torch.randn(9, 50, device=dev)
    kept = act8.pack(x)
    assert kept.nbytes == 9 * 66 and kept.shape == (9, 50)
    code, e = ref.pack(x)
    for t in TYPES:
        assert torch.equal(act8.unpack(kept, t).cpu().double(), ref.unpack(code, e, 50, t))
    # fp16 has no 2^16: what rounds up to it stays at 65504
    top = act8.pack(torch.full((1, 32), 65504.0, device=dev, dtype=torch.float16))
    assert torch.equal(act8.unpack(top), torch.full((1, 32), 65504.0, device=dev, dtype=torch.float16))
    with pytest.raises(TypeError):
        act8.unpack(kept, torch.float64)


def test_more_rows_than_a_grid_and_offsets_behind_32_bits(dev):
    """70 001 narrow rows (the grid strides), and a tensor of 2^31 + elements whose last rows are checked."""
    g = torch.Generator().manual_seed(9)
    _check(torch.randn(70001, 33, generator=g).to(dev))
    wide = torch.zeros(65552, 32768, dtype=torch.bfloat16, device=dev)          # 2^31 + 2^19 elements, 4.3 GB
    wide[-3:] = torch.randn(3, 32768, generator=g).to(torch.bfloat16).to(dev)
    kept = act8.pack(wide)
    code, e = ref.pack(wide[-3:])
    assert np.array_equal(kept.codes[-3:].cpu().numpy(), code) and np.array_equal(kept.exponents()[-3:].cpu().numpy(), e)
    assert int(kept.codes[:-3].max()) == 0
    back = act8.unpack(kept)
    assert torch.equal(back[-3:].cpu().double(), ref.unpack(code, e, 32768, torch.bfloat16))


def test_other_stream_and_graph_replay(dev):
    x = torch.randn(300, 200, device=dev)
    want = act8.unpack(act8.pack(x))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = act8.unpack(act8.pack(x))
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = act8.unpack(act8.pack(x))
    for k in range(3):
        x.copy_(torch.randn(300, 200, device=dev))
        graph.replay()
        assert torch.equal(out, act8.unpack(act8.pack(x)))
        torch.cuda.synchronize()
