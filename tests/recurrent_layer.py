"""
The state space scan, the short causal convolution and the root-mean-square norm written down in float64, token by token,
with torch's automatic differentiation for the gradients: what the kernels' tests compare with (test infrastructure).
"""
import math

import torch

E4M3_MAX = 448.0

TYPES = {'float32': torch.float32, 'float16': torch.float16, 'bfloat16': torch.bfloat16}
CODES = {'float32': 2, 'float16': 1, 'bfloat16': 32}


def half_step(dtype):
    """The largest relative error of one rounding to nearest."""
    return torch.finfo(dtype).eps / 2


def wide(t, grad=False):
    return None if t is None else t.detach().double().requires_grad_(grad)


def close(got, want, dtype, what, terms=1.0, scale=None):
    """Within one rounding to the type, plus float32 arithmetic: `terms` times 2^-22 of the largest magnitude (a handful of
    float32 roundings, which sums of values of either sign do not carry as a relative error), or of `scale`."""
    got, want = got.detach().cpu(), want.detach().double().cpu()
    assert got.shape == want.shape and got.dtype == dtype, what
    if scale is None:
        scale = float(want.abs().max() if want.numel() else 0.0)
    bound = half_step(dtype) * want.abs() * 1.001 + terms * 2.0 ** -22 * scale
    if dtype == torch.float16:
        bound = bound + 2.0 ** -25                 # half the distance of its subnormal numbers
    off = (got.double() - want).abs()
    if not off.numel():
        return
    assert bool((off <= bound).all()), '%s: off by %.3g where %.3g is allowed' % (
        what, float((off - bound).max()), float(bound.flatten()[(off - bound).argmax()]))


def scan(u, delta, A, B, C, D=None, z=None, delta_bias=None, softplus=False, state=None, lengths=None):
    """Float64 tensors in, (y, last) out; differentiable."""
    batch, length, channels = u.shape
    n = A.shape[1]
    if B.dim() == 3:
        B, C = B[:, :, None], C[:, :, None]
    per = channels // B.shape[2]
    dt = delta if delta_bias is None else delta + delta_bias
    if softplus:
        dt = torch.nn.functional.softplus(dt, threshold=700)
    ends = [length] * batch if lengths is None else [min(max(int(v), 0), length) for v in lengths.tolist()]
    ys, lasts = [], []
    for b in range(batch):
        h = torch.zeros(channels, n, dtype=u.dtype, device=u.device) if state is None else state[b]
        rows = []
        for t in range(ends[b]):
            h = torch.exp(dt[b, t, :, None] * A) * h + (dt[b, t] * u[b, t])[:, None] * B[b, t].repeat_interleave(per, 0)
            y = (h * C[b, t].repeat_interleave(per, 0)).sum(-1)
            if D is not None:
                y = y + D * u[b, t]
            if z is not None:
                y = y * z[b, t] * torch.sigmoid(z[b, t])
            rows.append(y)
        rows.append(torch.zeros(length - ends[b], channels, dtype=u.dtype, device=u.device))
        ys.append(torch.cat([r.view(-1, channels) for r in rows]))
        lasts.append(h)
    return torch.stack(ys), torch.stack(lasts)


def conv(x, weight, bias=None, activation=None, state=None, lengths=None):
    batch, length, channels = x.shape
    width = weight.shape[1]
    ends = [length] * batch if lengths is None else [min(max(int(v), 0), length) for v in lengths.tolist()]
    ys, lasts = [], []
    for b in range(batch):
        before = torch.zeros(width - 1, channels, dtype=x.dtype, device=x.device) if state is None else state[b]
        line = torch.cat([before, x[b, :ends[b]]])
        pre = torch.zeros(ends[b], channels, dtype=x.dtype, device=x.device)
        if bias is not None:
            pre = pre + bias
        for k in range(width):
            pre = pre + weight[:, k] * line[k:k + ends[b]]
        y = pre * torch.sigmoid(pre) if activation else pre
        ys.append(torch.cat([y, torch.zeros(length - ends[b], channels, dtype=x.dtype, device=x.device)]))
        lasts.append(line[ends[b]:])
    return torch.stack(ys), torch.stack(lasts)


def norm(s, weight, eps=1e-5):
    return s / torch.sqrt(s.square().mean(-1, keepdim=True) + eps) * weight


def norm_gradient_scale(s, weight, d_y, d_s=None, eps=1e-5):
    """The largest magnitude among the terms of the norm's gradient, d = r (t - n mean(t n)) + d_s with t = d_y w, n = s r.
    Each term is rounded on its own, so the error of d is a few units of 2^-24 times the largest TERM, however small their
    difference: with one column n^2 = s^2 / (s^2 + eps), so r (t - n (t n)) = r t (1 - n^2) = r t eps r^2, for s = -1 and t = 1
    a difference of 1e-5 between two terms of size 1, whose roundings of 6e-8 are 6e-3 of it."""
    s, t = s.double(), d_y.double() * weight.double()
    r = 1 / torch.sqrt(s.square().mean(-1, keepdim=True) + eps)
    n = s * r
    parts = [(r * t).abs().max(), (r * n * (t * n).mean(-1, keepdim=True)).abs().max()]
    return float(max(parts + ([] if d_s is None else [d_s.double().abs().max()])))


def scales_of(y, group=None):
    columns = y.shape[-1]
    parts = y.split(group or columns, -1)
    scale = torch.stack([p.abs().amax(-1) / E4M3_MAX for p in parts], -1)
    return torch.where(scale > 0, scale, torch.ones_like(scale))


def quantized(y, group=None):
    """The codes and scales that float32 results of the norm have to get, bit for bit: the largest magnitude divided by 448,
    at least 2^-126, and the quotients rounded to e4m3 (division and rounding of the CPU)."""
    y = y.detach().cpu()
    parts = y.split(group or y.shape[-1], -1)
    scales = torch.stack([p.abs().amax(-1) / E4M3_MAX for p in parts], -1).clamp(min=2.0 ** -126)
    scales = torch.where(torch.stack([p.abs().amax(-1) for p in parts], -1) > 0, scales, torch.ones_like(scales))
    each = scales.repeat_interleave(group or y.shape[-1], -1)[..., :y.shape[-1]]
    return (y / each).to(torch.float8_e4m3fn), scales


def middles(divisors):
    """For each of the divisors d (odd whole numbers of up to 19 bits) a row of 128 float32 weights whose results, for rows of
    ones without eps, are the weights themselves: 448 d, which makes the scale d, and then t d for numbers t in the middle of
    two neighbouring e4m3 numbers.  Both products are exact, so every quotient is such a middle and goes to the even one."""
    t = torch.tensor([(2 * m + 1) * 2.0 ** e for e in range(-4, 5) for m in range(8, 16)], dtype=torch.float64)
    t = torch.cat([torch.tensor([448.0], dtype=torch.float64), t[t < 448], torch.ones(128, dtype=torch.float64)])[:128]
    rows = torch.tensor(divisors, dtype=torch.float64)[:, None] * t
    assert torch.equal(rows.float().double(), rows)
    return rows.float(), t


def scan_inputs(seed, batch, length, channels, n, groups, dtype, gate=True, ragged=False, entering=True, device='cpu',
                softplus=True, skip=True, bias=True):
    """Inputs of the sizes a layer meets; softplus leaves time steps between 0.001 and 0.3."""
    g = torch.Generator()
    g.manual_seed(seed)

    def normal(*shape, scale=1.0):
        return torch.randn(shape, generator=g) * scale

    kind = TYPES[dtype]
    d = {}
    d['u'] = normal(batch, length, channels).to(kind)
    step = torch.exp(torch.rand(channels, generator=g) * math.log(100.0) + math.log(0.001))
    if softplus:
        d['delta'] = normal(batch, length, channels, scale=0.5).to(kind)
        d['delta_bias'] = step + torch.log(-torch.expm1(-step)) if bias else None
    else:
        d['delta'] = (step * torch.exp(normal(batch, length, channels, scale=0.3))).to(kind)
        d['delta_bias'] = normal(channels, scale=0.01).abs() if bias else None
    d['A'] = -(1 + torch.arange(n).float()) * torch.exp(normal(channels, n, scale=0.2))
    d['B'] = normal(batch, length, groups, n).to(kind)
    d['C'] = normal(batch, length, groups, n).to(kind)
    d['D'] = 1 + normal(channels, scale=0.1) if skip else None
    d['z'] = normal(batch, length, channels).to(kind) if gate else None
    d['state'] = normal(batch, channels, n) if entering else None
    d['lengths'] = None
    if ragged:
        lengths = torch.randint(0, length + 1, (batch,), generator=g).int()
        lengths[0] = 0
        lengths[-1] = length
        d['lengths'] = lengths
    d['softplus'] = softplus
    d['d_y'] = normal(batch, length, channels).to(kind)
    d['d_last'] = normal(batch, channels, n)
    if device != 'cpu':
        d = {k: v.to(device) if isinstance(v, torch.Tensor) else v for k, v in d.items()}
    return d


SCAN_NAMES = ('u', 'delta', 'A', 'B', 'C', 'D', 'z', 'delta_bias', 'state')


def scan_expected(d, with_last=True):
    """(y, last) and the gradients in the order of SCAN_NAMES, all float64."""
    leaves = {k: wide(d[k], True) for k in SCAN_NAMES}
    y, last = scan(softplus=d['softplus'], lengths=d['lengths'], **leaves)
    outs, ups = [y], [d['d_y'].double()]
    if with_last:
        outs, ups = outs + [last], ups + [d['d_last'].double()]
    present = [v for v in leaves.values() if v is not None]
    grads = iter(torch.autograd.grad(outs, present, ups, allow_unused=True))
    grads = [None if leaves[k] is None else next(grads) for k in SCAN_NAMES]
    grads = [torch.zeros_like(leaves[k]) if v is None and leaves[k] is not None else v for k, v in zip(SCAN_NAMES, grads)]
    return y.detach(), last.detach(), grads


def conv_inputs(seed, batch, length, channels, width, dtype, ragged=False, entering=True, bias=True, device='cpu'):
    g = torch.Generator()
    g.manual_seed(seed)

    def normal(*shape, scale=1.0):
        return torch.randn(shape, generator=g) * scale

    kind = TYPES[dtype]
    d = {'x': normal(batch, length, channels).to(kind), 'weight': normal(channels, width, scale=width ** -0.5),
         'bias': normal(channels, scale=0.1) if bias else None,
         'state': normal(batch, width - 1, channels).to(kind) if entering else None, 'lengths': None,
         'd_y': normal(batch, length, channels).to(kind), 'd_last': normal(batch, width - 1, channels).to(kind)}
    if ragged:
        lengths = torch.randint(0, length + 1, (batch,), generator=g).int()
        lengths[0] = 0
        lengths[-1] = length
        d['lengths'] = lengths
    if device != 'cpu':
        d = {k: v.to(device) if isinstance(v, torch.Tensor) else v for k, v in d.items()}
    return d


CONV_NAMES = ('x', 'weight', 'bias', 'state')


def conv_expected(d, activation, with_last=True):
    leaves = {k: wide(d[k], True) for k in CONV_NAMES}
    y, last = conv(activation=activation, lengths=d['lengths'], **leaves)
    outs, ups = [y], [d['d_y'].double()]
    if with_last and last.numel():
        outs, ups = outs + [last], ups + [d['d_last'].double()]
    # a sequence without tokens passes nothing on to some of the leaves
    present = [v for v in leaves.values() if v is not None]
    if not any(o.requires_grad for o in outs):
        grads = iter([torch.zeros_like(v) for v in present])
    else:
        keep = [(o, u) for o, u in zip(outs, ups) if o.requires_grad]
        grads = iter(torch.autograd.grad([o for o, _ in keep], present, [u for _, u in keep], allow_unused=True))
    grads = [None if leaves[k] is None else next(grads) for k in CONV_NAMES]
    grads = [torch.zeros_like(leaves[k]) if v is None and leaves[k] is not None else v for k, v in zip(CONV_NAMES, grads)]
    return y.detach(), last.detach(), grads
