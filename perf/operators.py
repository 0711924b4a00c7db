"""Operators of FC stacks that train with little memory, as they are measured: activations kept in 8 bits for the backward pass
(`detmatch_amd.act8`) and the norms around a residual block, fused with its gate and residual scale
(`detmatch_amd.block_norm`).

`run` computes an operator in elementary torch operations (`own = False`) or through the framework's entry points
(`own = True`); `exact` computes the same outputs from the definitions in 64 bits.
"""
import math

import torch

own = False

DTYPES = {'fp32': torch.float32, 'bf16': torch.bfloat16, 'fp16': torch.float16}
GROUP = 32          # channels that share one power-of-two scale
EPS = 1e-6


# ------------------------------------------------------------------------------------------------------------- cases
def _codec(name, rows, width, dtype):
    return dict(name=name, op='codec', rows=rows, width=width, dtype=dtype)


def _linear(name, rows, fan_in, fan_out, dtype, bias, relu):
    return dict(name=name, op='linear', rows=rows, fan_in=fan_in, fan_out=fan_out, dtype=dtype, bias=bias, relu=relu)


def _norm(name, rows, width, dtype, kind, gate, act, post, keep8, train):
    return dict(name=name, op='norm', rows=rows, width=width, dtype=dtype, kind=kind, gate=gate, act=act, post=post,
                keep8=keep8, train=train)


def listed():
    return [
        # RoI features of one small batch, the smallest tensor that is worth keeping in 8 bits: a latency
        _codec('codec 256x256 fp32', 256, 256, 'fp32'),
        # flattened 7 x 7 x 256 RoI features of a training batch
        _codec('codec 4096x12544 bf16', 4096, 12544, 'bf16'),
        # shared FC of the second stage over the pooled RoI grid (6 x 6 x 6 x 128): 256 RoIs, a skinny product
        _linear('linear roi grid fp32', 256, 27648, 256, 'fp32', False, False),
        # first shared FC of the 2D head, an odd number of proposals
        _linear('linear 1999x12544x1024 fp32', 1999, 12544, 1024, 'fp32', True, False),
        # the expanding FC of an ordinary block
        _linear('linear 4096x1024x4096 bf16', 4096, 1024, 4096, 'bf16', True, True),
        # the largest product: long batches of a wide block
        _linear('linear 16384x4096x4096 bf16', 16384, 4096, 4096, 'bf16', False, False),
        # nothing divides a tile, rows are not aligned to 16 bytes
        _linear('linear 777x1001x515 fp16', 777, 1001, 515, 'fp16', True, True),
        # one row at inference: the norms between two blocks, a latency
        _norm('norm 1x1024 bf16 infer', 1, 1024, 'bf16', 'rms', 'channel', 'none', True, False, False),
        # teacher pass over a batch of points, layer norm, no training
        _norm('norm 16384x640 fp32 infer', 16384, 640, 'fp32', 'layer', 'sample', 'sigmoid', True, False, False),
        # the ordinary training step of a block, kept in 8 bits
        _norm('norm 8192x2048 bf16 train', 8192, 2048, 'bf16', 'rms', 'channel', 'none', True, True, True),
        # the largest: a wide residual stream with a gate for each element
        _norm('norm 32768x4096 bf16 train', 32768, 4096, 'bf16', 'rms', 'row', 'sigmoid', True, True, True),
        # odd sizes, one gate vector a sample, exact copies kept
        _norm('norm 4098x1001 fp32 train', 4098, 1001, 'fp32', 'layer', 'sample', 'tanh', True, False, True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(['codec', 'linear', 'linear', 'norm', 'norm', 'norm'])
    dtype = rng.choice(['fp32', 'bf16', 'fp16'])
    if op == 'codec':
        while True:
            rows, width = _log(rng, 16, 32768), _log(rng, 33, 27648)
            if 10000 <= rows * width <= 4096 * 12544:
                return dict(op=op, rows=rows, width=width, dtype=dtype)
    if op == 'linear':
        while True:
            rows, fan_in, fan_out = _log(rng, 1, 16384), _log(rng, 33, 27648), _log(rng, 8, 4096)
            if rng.random() < 0.5:
                fan_in, fan_out = 64 * max(1, fan_in // 64), 64 * max(1, fan_out // 64)
            # (fp32 costs more: its largest is the listed 2D head's product)
            if rows * fan_in * fan_out <= (1999 * 12544 * 1024 if dtype == 'fp32' else 16384 * 4096 * 4096):
                break
        # in 32 bits a ReLU whose input is within rounding of 0 may open on one side only and is worth more than the tolerance
        relu = dtype != 'fp32' and rows >= 256 and rng.random() < 0.5
        return dict(op=op, rows=rows, fan_in=fan_in, fan_out=fan_out, dtype=dtype, bias=rng.random() < 0.5, relu=relu)
    while True:
        rows, width = _log(rng, 1, 32768), _log(rng, 33, 8192)
        if rows * width <= (8192 * 4096 if dtype == 'fp32' else 32768 * 4096):
            break
    train = rng.random() < 0.6
    gate = rng.choice(['none', 'channel', 'sample', 'row'])
    if gate == 'sample':
        rows = 2 * max(1, rows // 2)
    # (a value of 32 bits next to a border of two 8-bit codes may fall on either side: kept in 8 bits below 32 bits only)
    return dict(op=op, rows=rows, width=width, dtype=dtype, kind=rng.choice(['rms', 'layer']), gate=gate,
                act='none' if gate == 'none' else rng.choice(['none', 'sigmoid', 'tanh']), post=rng.random() < 0.75,
                keep8=train and dtype != 'fp32' and rng.random() < 0.5, train=train)


# ------------------------------------------------------------------------------------------------------------- inputs
def _activations(g, rows, width):
    """Rows as a network has them: channels of very different size, some of them closed by a ReLU, a few outliers."""
    size = torch.exp(torch.randn(width, generator=g, device='cuda') * 1.0)
    x = torch.randn(rows, width, generator=g, device='cuda') * size
    shut = torch.rand(rows, (width + 63) // 64, generator=g, device='cuda') < 0.1
    return x.masked_fill_(shut.repeat_interleave(64, 1)[:, :width], 0.0)


def prepare(case, seed):
    g = torch.Generator(device='cuda').manual_seed(seed)
    t = DTYPES[case['dtype']]

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device='cuda') * scale

    if case['op'] == 'codec':
        return dict(case, x=_activations(g, case['rows'], case['width']).to(t))
    if case['op'] == 'linear':
        m, k, n = case['rows'], case['fan_in'], case['fan_out']
        s = dict(case, x=_activations(g, m, k).to(t), w=normal(n, k, scale=k ** -0.5).to(t),
                 b=normal(n, scale=0.1).to(t) if case['bias'] else None, gy=normal(m, n, scale=0.1).to(t))
        for name in ('x', 'w', 'b'):
            if s[name] is not None:
                s[name].requires_grad_(True)
        return s
    m, c = case['rows'], case['width']
    groups = {'none': 0, 'channel': 1, 'sample': 2, 'row': m}[case['gate']]
    layer = case['kind'] == 'layer'
    x, f = normal(m, c).to(t), _activations(g, m, c).to(t)
    s = dict(case, x=x, f=f, scale=torch.full((1,), 0.7, device='cuda').to(t),
             gate=(0.5 + normal(groups, c, scale=0.3)).to(t) if groups else None,
             pre_w=(1 + normal(c, scale=0.1)).to(t), pre_b=normal(c, scale=0.1).to(t) if layer else None,
             post_w=(1 + normal(c, scale=0.1)).to(t) if case['post'] else None,
             post_b=normal(c, scale=0.1).to(t) if layer and case['post'] else None)
    if case['train']:
        # gradients that lean towards what they are gradients of, as those of a loss do
        s['gy'] = (normal(m, c) + 0.3 * f.float()).to(t)
        s['gh'] = (normal(m, c) + 0.3 * x.float()).to(t)
        for name in _LEAVES:
            if s[name] is not None:
                s[name].requires_grad_(True)
    return s


_LEAVES = ('x', 'f', 'scale', 'gate', 'pre_w', 'pre_b', 'post_w', 'post_b')


# ------------------------------------------------------------------------------------------------------------- run
def run(s):
    return _OWN[s['op']](s) if own else _PLAIN[s['op']](s)


def _own_codec(s):
    from detmatch_amd import act8
    kept = act8.pack(s['x'])
    return dict(values=act8.unpack(kept), exponents=kept.exponents())


def _own_linear(s):
    from detmatch_amd import act8
    y = act8.linear(s['x'], s['w'], s['b'], relu=s['relu'])
    leaves = [s[k] for k in ('x', 'w', 'b') if s[k] is not None]
    grads = torch.autograd.grad(y, leaves, s['gy'])
    return dict(zip(('y', 'gx', 'gw', 'gb'), (y, *grads)))


def _own_norm(s):
    from detmatch_amd import block_norm

    def forward():
        return block_norm.residual_norm(
            s['x'], s['f'], scale=s['scale'], gate=s['gate'], gate_act=s['act'], post=s['post'], post_w=s['post_w'],
            post_b=s['post_b'], pre_w=s['pre_w'], pre_b=s['pre_b'], kind=s['kind'], eps=EPS, keep8=s['keep8'])

    if not s['train']:
        with torch.no_grad():
            y, h = forward()
        return dict(y=y, h=h)
    y, h = forward()
    names = [k for k in _LEAVES if s[k] is not None]
    grads = torch.autograd.grad([y, h], [s[k] for k in names], [s['gy'], s['gh']])
    return dict(y=y, h=h, **dict(zip(('g_' + k for k in names), grads)))


_OWN = dict(codec=_own_codec, linear=_own_linear, norm=_own_norm)


def _power(e):
    """2^e in 64 bits."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _kept(x):
    """(the values that the 8-bit form of x (rows, width) stands for in x's type, as 32-bit numbers; exponents (rows, groups))."""
    rows, width = x.shape
    groups = (width + GROUP - 1) // GROUP
    v = torch.nn.functional.pad(x.detach().float(), (0, groups * GROUP - width)).view(rows, groups, GROUP)
    fine = torch.isfinite(v)
    top = torch.where(fine, v.abs(), 0.0).amax(2, keepdim=True)
    half, e = torch.frexp(top)                                  # top = half * 2^e, half in [1/2, 1)
    e = torch.where(top > 0, e - 9 + (half > 0.875), 0).clamp(min=-127)
    limit = torch.where(e >= 120, 240.0, 448.0)
    code = (v * _power(-e).float()).clamp(min=-limit, max=limit).to(torch.float8_e4m3fn).double()
    value = torch.where(fine, code, math.nan) * _power(e)
    most = torch.finfo(x.dtype).max
    value = value.clamp(-most, most).to(x.dtype).float()
    return value.view(rows, -1)[:, :width], e.view(rows, groups).to(torch.int32)


def _plain_codec(s):
    values, exponents = _kept(s['x'])
    return dict(values=values.to(s['x'].dtype), exponents=exponents)


def _plain_linear(s):
    t = s['x'].dtype
    x, w, gy = s['x'].detach().float(), s['w'].detach().float(), s['gy'].float()
    y = x @ w.t()
    if s['b'] is not None:
        y = y + s['b'].detach().float()
    if s['relu']:
        y = y.clamp(min=0)
        gy = gy * (y > 0)
    out = dict(y=y.to(t), gx=(gy @ w).to(t), gw=(gy.t() @ _kept(s['x'])[0]).to(t))
    if s['b'] is not None:
        out['gb'] = gy.sum(0).to(t)
    return out


def _stats(v, layer):
    mean = v.mean(1, keepdim=True) if layer else torch.zeros_like(v[:, :1])
    return mean, torch.rsqrt((v - mean).square().mean(1, keepdim=True) + EPS)


def _norm_back(d, hat, rstd, layer):
    """Gradient of a norm's input, from the gradient `d` of its normalised values."""
    d = d - hat * (d * hat).mean(1, keepdim=True) - (d.mean(1, keepdim=True) if layer else 0.0)
    return d * rstd


def _gate(s, rows, to):
    """(gate, its derivative) for all rows."""
    if s['gate'] is None:
        return 1.0, None
    z = to(s['gate'].detach())
    if s['act'] == 'sigmoid':
        g = torch.sigmoid(z)
        d = g * (1 - g)
    elif s['act'] == 'tanh':
        g = torch.tanh(z)
        d = 1 - g * g
    else:
        g, d = z, torch.ones_like(z)
    each = rows // g.shape[0]
    return g.repeat_interleave(each, 0), d


def _norm_by_formula(s, to, kept):
    """The norms around a block and their gradients; `to` casts to the precision that is computed in, kept(v, stored type)
    gives what the backward pass sees of a tensor that the forward pass kept."""
    layer, t = s['kind'] == 'layer', s['x'].dtype
    x, f = to(s['x'].detach()), to(s['f'].detach())
    rows = x.shape[0]
    scale = to(s['scale'].detach())
    pre_w = to(s['pre_w'].detach())
    g, dg = _gate(s, rows, to)
    u = f
    if s['post']:
        f_mean, f_rstd = _stats(f, layer)
        u = (f - f_mean) * f_rstd * to(s['post_w'].detach())
        u = u + to(s['post_b'].detach()) if layer else u
    y = x + scale * g * u
    mean, rstd = _stats(y, layer)
    h = (y - mean) * rstd * pre_w
    h = h + to(s['pre_b'].detach()) if layer else h
    out = dict(y=y, h=h)
    if not s['train']:
        return out
    gy, gh = to(s['gy']), to(s['gh'])
    y_hat = (kept(y.to(t)) - mean) * rstd
    dy = gy + _norm_back(gh * pre_w, y_hat, rstd, layer)
    out['g_pre_w'] = (gh * y_hat).sum(0)
    if layer:
        out['g_pre_b'] = gh.sum(0)
    out['g_x'] = dy
    v = f_hat = kept(s['f'].detach())
    if s['post']:
        f_hat = (v - f_mean) * f_rstd
        v = f_hat * to(s['post_w'].detach())
        v = v + to(s['post_b'].detach()) if layer else v
    d = dy * scale
    out['g_scale'] = (dy * g * v).sum().reshape(1)
    if s['gate'] is not None:
        out['g_gate'] = (d * v).view(dg.shape[0], -1, x.shape[1]).sum(1) * dg
    d = d * g
    if s['post']:
        out['g_post_w'] = (d * f_hat).sum(0)
        if layer:
            out['g_post_b'] = d.sum(0)
        d = _norm_back(d * to(s['post_w'].detach()), f_hat, f_rstd, layer)
    out['g_f'] = d
    return out


def _plain_norm(s):
    kept = (lambda v: _kept(v)[0]) if s['keep8'] else (lambda v: v.float())
    return {k: v.to(s['x'].dtype) for k, v in _norm_by_formula(s, lambda v: v.float(), kept).items()}


_PLAIN = dict(codec=_plain_codec, linear=_plain_linear, norm=_plain_norm)


# ------------------------------------------------------------------------------------------------------------- work
def work(case):
    size = 4 if case['dtype'] == 'fp32' else 2
    kept = 1 + 1.0 / GROUP                      # bytes of a value that is kept in 8 bits
    if case['op'] == 'codec':
        n = case['rows'] * case['width']
        return dict(bytes=2 * n * (size + kept), flops=4 * n)
    if case['op'] == 'linear':
        m, k, n = case['rows'], case['fan_in'], case['fan_out']
        # x, w, gy in; y, gx, gw out; x's codes out and in again; w a second time in the backward pass
        return dict(bytes=size * (2 * m * k + 3 * n * k + 2 * m * n) + 2 * kept * m * k, flops=6.0 * m * n * k)
    n = case['rows'] * case['width']
    gate = n * size if case['gate'] == 'row' else 0
    moved, flops = 4 * n * size + gate, 12 * n                   # x, f, y, h
    if case['train']:
        saved = kept if case['keep8'] else size
        # gy, gh, dx, df, the kept f and y (an exact copy is there already: read only), a gate for each element and its gradient
        moved += 4 * n * size + 2 * n * saved * (2 if case['keep8'] else 1) + 2 * gate
        flops += 30 * n
    return dict(bytes=moved, flops=flops)


# ------------------------------------------------------------------------------------------------------------- exact
def _exact_kept(x):
    """deq(pack(x)) by the definition in 64 bits: round to nearest, ties to even, 3 bits behind the leading one."""
    rows, width = x.shape
    v = x.detach().double()
    pad = -width % GROUP
    v = torch.cat([v, v.new_zeros(rows, pad)], 1) if pad else v
    v = v.reshape(rows, -1, GROUP)
    usable = v.isfinite()
    top = (v.abs() * usable).nan_to_num(0.0, 0.0, 0.0).max(2, keepdim=True).values
    e = torch.frexp(top).exponent.to(torch.int64) - 1            # floor(log2(top))
    e = e - 8 + (top > 1.75 * _power(e)).to(torch.int64)
    e = torch.where(top == 0, torch.zeros_like(e), e).clamp(min=-127)
    z = v * _power(-e)
    lead = (torch.frexp(z).exponent.to(torch.int64) - 1).clamp(min=-6)
    step = _power(lead - 3)
    z = torch.round(z / step) * step                             # torch.round: ties to even
    limit = torch.where(e >= 120, 240.0, 448.0).double()
    z = torch.minimum(torch.maximum(z, -limit), limit)
    z = torch.where(usable, z * _power(e), torch.full_like(z, math.nan))
    most = torch.finfo(x.dtype).max
    z = z.clamp(-most, most).to(x.dtype).double()
    return z.reshape(rows, -1)[:, :width], e[..., 0].to(torch.int32)


def exact(case, seed):
    s = prepare(case, seed)
    if case['op'] == 'codec':
        values, exponents = _exact_kept(s['x'])
        return dict(values=values, exponents=exponents)
    if case['op'] == 'linear':
        x, w, gy = s['x'].detach().double(), s['w'].detach().double(), s['gy'].double()
        y = torch.mm(x, w.t().contiguous())
        del x
        if s['b'] is not None:
            y += s['b'].detach().double()
        if s['relu']:
            y = torch.relu(y)
            gy = torch.where(y > 0, gy, torch.zeros_like(gy))
        out = dict(y=y, gx=torch.mm(gy, w))
        out['gw'] = torch.mm(gy.t().contiguous(), _exact_kept(s['x'])[0])
        if s['b'] is not None:
            out['gb'] = gy.sum(0)
        return out
    return _exact_norm(s)


def _exact_norm(s):
    """The definition of the norms in 64 bits; the gradients by torch's autograd of a function that is written so that its
    gradient is the operator's: the values that the backward pass sees take the place of those that the forward pass saw."""
    layer, t = s['kind'] == 'layer', s['x'].dtype
    leaf = {k: s[k].detach().double().requires_grad_(s['train']) for k in _LEAVES if s[k] is not None}

    class Norm(torch.autograd.Function):
        @staticmethod
        def forward(ctx, v, seen):
            mean = v.mean(1, keepdim=True) if layer else 0.0
            dev = torch.sqrt(((v - mean) ** 2).mean(1, keepdim=True) + EPS)
            ctx.save_for_backward((seen - mean) / dev, dev)
            return (v - mean) / dev

        @staticmethod
        def backward(ctx, d):
            hat, dev = ctx.saved_tensors
            rest = d - hat * torch.mean(d * hat, 1, True)
            return (rest - torch.mean(d, 1, True) if layer else rest) / dev, None

    class Seen(torch.autograd.Function):          # v * w, whose gradient for w sees `seen` in v's place
        @staticmethod
        def forward(ctx, v, w, seen):
            ctx.save_for_backward(w, seen)
            ctx.one = w.numel() == 1
            return v * w

        @staticmethod
        def backward(ctx, d):
            w, seen = ctx.saved_tensors
            return d * w, (d * seen).sum().reshape(1) if ctx.one else (d * seen).sum_to_size(w.shape), None

    def see(v):
        return _exact_kept(v)[0] if s['keep8'] else v.double()

    def hat_of(v, seen):                          # the normalised values that the backward pass sees
        mean = v.mean(1, keepdim=True) if layer else 0.0
        return (seen - mean) / torch.sqrt(((v - mean) ** 2).mean(1, keepdim=True) + EPS)

    with torch.set_grad_enabled(s['train']):
        f, seen = leaf['f'], see(s['f'].detach())
        u = f
        if s['post']:
            hat = hat_of(f.detach(), seen)
            u = Seen.apply(Norm.apply(f, seen), leaf['post_w'], hat)
            seen = hat * leaf['post_w'].detach()
            if layer:
                u, seen = u + leaf['post_b'], seen + leaf['post_b'].detach()
        if s['gate'] is not None:
            act = {'none': lambda z: z, 'sigmoid': torch.sigmoid, 'tanh': torch.tanh}[s['act']]
            each = s['x'].shape[0] // s['gate'].shape[0]
            g = act(leaf['gate'])
            g = g[:, None].expand(-1, each, -1).reshape(s['x'].shape)
            u = Seen.apply(u, g, seen)
            seen = seen * g.detach()
        y = leaf['x'] + Seen.apply(u, leaf['scale'], seen)
        stored = see(y.detach().to(t))
        h = Seen.apply(Norm.apply(y, stored), leaf['pre_w'], hat_of(y.detach(), stored))
        h = h + leaf['pre_b'] if layer else h
    out = dict(y=y.detach(), h=h.detach())
    if s['train']:
        names = [k for k in _LEAVES if s[k] is not None]
        grads = torch.autograd.grad([y, h], [leaf[k] for k in names], [s['gy'].double(), s['gh'].double()])
        out.update(zip(('g_' + k for k in names), grads))
    return out
