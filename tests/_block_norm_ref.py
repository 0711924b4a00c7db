"""The norms around a residual block in float64, by their formulas, with magnitudes for error bounds: every value is computed a second
time with absolute values in place of signed ones ("mag"), so that a result of fp32 arithmetic is off by a small multiple of
2^-24 of its magnitude."""
import torch

ACTS = {'none': lambda z: z, 'sigmoid': torch.sigmoid, 'tanh': torch.tanh}


def stats(v, layer, eps):
    mean = v.mean(1, keepdim=True) if layer else torch.zeros_like(v[:, :1])
    return mean, 1 / torch.sqrt(((v - mean) ** 2).mean(1, keepdim=True) + eps)


def norm(v, seen, layer, eps):
    """(normalised seen, its magnitude, rstd) with the statistics of v"""
    mean, rstd = stats(v, layer, eps)
    mean_mag = v.abs().mean(1, keepdim=True) if layer else 0.0
    return (seen - mean) * rstd, (seen.abs() + mean_mag) * rstd, rstd


def back(d, mag, hat, hat_mag, rstd, layer):
    out = d - hat * (d * hat).mean(1, keepdim=True) - (d.mean(1, keepdim=True) if layer else 0.0)
    out_mag = mag + hat_mag * (mag * hat_mag).mean(1, keepdim=True) + (mag.mean(1, keepdim=True) if layer else 0.0)
    return rstd * out, rstd * out_mag


def forward(p):
    """p: dict of float64 tensors x, f (or None), gate, scale (number), post, post_w, post_b, pre, pre_w, pre_b, layer, eps, act.
    -> dict of (value, magnitude): y, h"""
    out = {}
    one = torch.ones(p['x'].shape[1], dtype=torch.float64)
    zero = torch.zeros_like(one)
    w = lambda k: one if p.get(k) is None else p[k]           # noqa: E731
    b = lambda k: zero if p.get(k) is None else p[k]          # noqa: E731
    y, mag = p['x'], p['x'].abs()
    if p.get('f') is not None:
        u, u_mag = p['f'], p['f'].abs()
        if p['post']:
            hat, hat_mag, _ = norm(u, u, p['layer'], p['eps'])
            u, u_mag = hat * w('post_w') + b('post_b'), hat_mag * w('post_w').abs() + b('post_b').abs()
        g = gates(p)
        y, mag = y + p['scale'] * g * u, mag + abs(p['scale']) * g.abs() * u_mag
        out['y'] = y, mag
    if p.get('pre', True):
        hat, hat_mag, rstd = norm(y, y, p['layer'], p['eps'])
        # what y is off by moves its statistics too
        hat_mag = mag * rstd + hat_mag + hat.abs() * rstd * (mag ** 2).mean(1, keepdim=True).sqrt() + (rstd * mag.mean(1, keepdim=True) if p['layer'] else 0)
        out['h'] = hat * w('pre_w') + b('pre_b'), hat_mag * w('pre_w').abs() + b('pre_b').abs()
    return out


def gates(p):
    if p.get('gate') is None:
        return torch.ones_like(p['x'])
    return ACTS[p['act']](p['gate']).repeat_interleave(p['x'].shape[0] // p['gate'].shape[0], 0)


def backward(p, gy, gh, f_seen, y_seen):
    """Gradients; f_seen, y_seen: f and y as the backward pass has them.  -> dict of (value, magnitude)"""
    out = {}
    x = p['x']
    one = torch.ones(x.shape[1], dtype=torch.float64)
    w = lambda k: one if p.get(k) is None else p[k]           # noqa: E731
    dy, mag = torch.zeros_like(x), torch.zeros_like(x)
    if gy is not None:
        dy, mag = gy, gy.abs()
    if gh is not None:
        y = forward(p)['y'][0] if p.get('f') is not None else x
        hat, hat_mag, rstd = norm(y, y_seen, p['layer'], p['eps'])
        hat_mag = hat_mag + 2 * hat.abs()
        more, more_mag = back(gh * w('pre_w'), (gh * w('pre_w')).abs(), hat, hat_mag, rstd, p['layer'])
        dy, mag = dy + more, mag + more_mag
        out['pre_w'] = (gh * hat).sum(0), (gh.abs() * hat_mag).sum(0)
        out['pre_b'] = gh.sum(0), gh.abs().sum(0)
    out['x'] = dy, mag
    if p.get('f') is None:
        return out
    g, s = gates(p), p['scale']
    u, u_mag = f_seen, f_seen.abs()
    if p['post']:
        hat, hat_mag, rstd = norm(p['f'], f_seen, p['layer'], p['eps'])
        hat_mag = hat_mag + 2 * hat.abs()
        bias = p['post_b'] if p.get('post_b') is not None else torch.zeros_like(one)
        u, u_mag = hat * w('post_w') + bias, hat_mag * w('post_w').abs() + bias.abs()
    out['scale'] = (dy * g * u).sum().reshape(1), (mag * g.abs() * u_mag).sum().reshape(1)
    d, d_mag = dy * s, mag * abs(s)
    if p.get('gate') is not None:
        z = p['gate'].clone().requires_grad_(True)
        slope, = torch.autograd.grad(ACTS[p['act']](z).sum(), z)
        shape = (p['gate'].shape[0], -1, x.shape[1])
        out['gate'] = (d * u).view(shape).sum(1) * slope, (d_mag * u_mag).view(shape).sum(1) * (slope.abs() + 2.0 ** -20)
    t, t_mag = d * g, d_mag * g.abs()
    if p['post']:
        out['post_w'] = (t * hat).sum(0), (t_mag * hat_mag).sum(0)
        out['post_b'] = t.sum(0), t_mag.sum(0)
        t, t_mag = back(t * w('post_w'), t_mag * w('post_w').abs(), hat, hat_mag, rstd, p['layer'])
    out['f'] = t, t_mag
    return out
