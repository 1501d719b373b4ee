"""
What the operators of a state space block cost on a GPU: the recurrence along time whose decay, input and read-out
vectors depend on the token (``opveclib_amd.state_space.scan``), the short causal convolution in front of it
(``state_space.conv``) and the root-mean-square norm with the residual's addition that opens the block
(``opveclib_amd.rms_norm``), each for prompts, for training and for single tokens.

``run`` computes a case in plain torch operations, in 32 bits and rounded once at the end, or, with ``own`` set, through
the package's entry points.  ``exact`` computes the same in 64 bits: step by step along time instead of by doubling,
gradients by automatic differentiation instead of by formulas.
"""
import math

import torch

own = False

#: largest finite magnitude of torch.float8_e4m3fn
E4M3_MAX = 448.0
EPS = 1e-5

_TYPES = {'float32': torch.float32, 'float16': torch.float16, 'bfloat16': torch.bfloat16}


# ----------------------------------------------------------------------------------------------------------------------
# cases
# ----------------------------------------------------------------------------------------------------------------------
def _scan(name, op, dtype, batch, length, channels, state=16, groups=1, gate=True, ragged=False, entering=False):
    case = {'op': op, 'dtype': dtype, 'batch': batch, 'length': length, 'channels': channels, 'state': state,
            'groups': groups, 'gate': gate, 'ragged': ragged, 'entering': entering}
    return dict(case, name=name) if name else case


def _conv(name, op, dtype, batch, length, channels, width=4, activation=True, ragged=False, entering=False):
    case = {'op': op, 'dtype': dtype, 'batch': batch, 'length': length, 'channels': channels, 'width': width,
            'activation': activation, 'ragged': ragged, 'entering': entering}
    return dict(case, name=name) if name else case


def _norm(name, op, dtype, residual, rows, columns, group=0):
    case = {'op': op, 'dtype': dtype, 'residual': residual, 'rows': rows, 'columns': columns, 'group': group}
    return dict(case, name=name) if name else case


def listed():
    return [
        # one new token of a few conversations: nothing but latency
        _scan('scan token 2x1024', 'scan_step', 'bfloat16', 2, 1, 1024),
        # one new token of a full batch: the state is read and written once
        _scan('scan token 96x4096', 'scan_step', 'bfloat16', 96, 1, 4096),
        # one long prompt: few channels, so the length has to be split
        _scan('scan prompt 1x8192x2048', 'scan', 'bfloat16', 1, 8192, 2048),
        # prompts of unequal length in one padded batch, continuing from kept states, two groups of heads, odd sizes
        _scan('scan ragged 6x1500x1300', 'scan', 'float16', 6, 1500, 1300, groups=2, ragged=True, entering=True),
        # a small layer trained in float32 with the state carried from batch to batch
        _scan('scan train 3x333x650 float32', 'scan_train', 'float32', 3, 333, 650, state=8, entering=True),
        # a training batch of an ordinary layer
        _scan('scan train 4x2048x4096', 'scan_train', 'bfloat16', 4, 2048, 4096),
        # the convolution's new tokens
        _conv('conv token 64x4096', 'conv_step', 'bfloat16', 64, 1, 4096),
        # the convolution on the padded batch of prompts
        _conv('conv ragged 6x1500x1300', 'conv', 'float16', 6, 1500, 1300, width=3, ragged=True, entering=True),
        # the convolution of the training batch
        _conv('conv train 4x4096x8192', 'conv_train', 'bfloat16', 4, 4096, 8192),
        # the norm in front of an 8-bit projection: a few tokens, and a long prompt with a scale for each 128 columns
        _norm('norm e4m3 5x4096', 'norm_quantized', 'bfloat16', 'bfloat16', 5, 4096),
        _norm('norm e4m3 16384x8192', 'norm_quantized', 'bfloat16', 'bfloat16', 16384, 8192, group=128),
        # the norm of a training batch, the residual stream kept in float32
        _norm('norm train 8192x4096', 'norm_train', 'bfloat16', 'float32', 8192, 4096),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, spread over their logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(['scan_step', 'scan', 'scan', 'scan_train', 'scan_train', 'conv_step', 'conv', 'conv_train',
                     'norm_quantized', 'norm_quantized', 'norm_train'])
    dtype = rng.choice(['bfloat16', 'bfloat16', 'float16', 'float32'])
    if op.startswith('norm'):
        rows, columns = _spread(rng, 1, 16384), _spread(rng, 64, 16384)
        while rows * columns > (1 << 26 if op == 'norm_quantized' else 1 << 25):
            rows = (rows + 1) // 2
        return _norm(None, op, dtype, rng.choice(['none', 'float32', dtype]), rows, columns,
                     group=rng.choice([0, 128]) if op == 'norm_quantized' else 0)
    groups = rng.choice([1, 1, 2, 4])
    channels = groups * _spread(rng, 16, 8192 // groups)
    if op.endswith('step'):
        batch = _spread(rng, 1, 128)
        while batch * channels > 96 * 4096:
            batch = (batch + 1) // 2
        if op == 'conv_step':
            return _conv(None, op, dtype, batch, 1, channels, width=rng.choice([2, 3, 4]), activation=rng.random() < 0.8)
        return _scan(None, op, dtype, batch, 1, channels, state=rng.choice([8, 16, 16, 32]), groups=groups,
                     gate=rng.random() < 0.7)
    batch, length = _spread(rng, 1, 16), _spread(rng, 1, 8192)
    if op.startswith('conv'):
        while batch * length * channels > 4 * 4096 * 8192:
            batch, length = (batch + 1) // 2, (2 * length + 2) // 3
        return _conv(None, op, dtype, batch, length, channels, width=rng.choice([2, 3, 4]),
                     activation=rng.random() < 0.8, ragged=rng.random() < 0.4, entering=rng.random() < 0.4)
    state = rng.choice([4, 8, 16, 16, 16, 24, 32])
    while batch * length * channels * state > 1 << (28 if op == 'scan' else 28):
        batch, length = (batch + 1) // 2, (2 * length + 2) // 3
    return _scan(None, op, dtype, batch, length, channels, state=state, groups=groups, gate=rng.random() < 0.7,
                 ragged=rng.random() < 0.4, entering=rng.random() < 0.4)


# ----------------------------------------------------------------------------------------------------------------------
# inputs
# ----------------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device='cuda')
    g.manual_seed(seed)
    dtype = _TYPES[case['dtype']]
    op = case['op']
    train = op.endswith('train')

    def normal(*shape, scale=1.0, kind=torch.float32):
        return (torch.randn(shape, generator=g, device='cuda') * scale).to(kind)

    def leaf(t):
        return t.detach().requires_grad_(True) if train and t is not None else t

    s = {'op': op}
    if op.startswith('norm'):
        rows, columns = case['rows'], case['columns']
        s['x'] = leaf(normal(rows, columns, kind=dtype))
        s['weight'] = leaf(1 + normal(columns, scale=0.1))
        s['residual'] = None
        if case['residual'] != 'none':
            s['residual'] = leaf(normal(rows, columns, scale=3.0, kind=_TYPES[case['residual']]))
        if train:
            s['d_y'] = normal(rows, columns, kind=dtype)
            s['d_summed'] = None if s['residual'] is None else normal(rows, columns, kind=s['residual'].dtype)
        s['group'] = case['group'] or None
        return s

    batch, length, channels = case['batch'], case['length'], case['channels']
    s['lengths'] = None
    if case['ragged']:
        lengths = torch.randint(0, length + 1, (batch,), generator=g, device='cuda', dtype=torch.int32)
        lengths[0] = length
        s['lengths'] = lengths
    if op.startswith('conv'):
        width = case['width']
        # the convolution's input is one half of a projection
        wide = normal(batch, length, 2 * channels, kind=dtype)
        s['x'] = leaf(wide[..., :channels])
        s['weight'] = leaf(normal(channels, width, scale=width ** -0.5))
        s['bias'] = leaf(normal(channels, scale=0.1))
        s['activation'] = 'silu' if case['activation'] else None
        s['state'] = None
        if op == 'conv_step':
            s['x'] = s['x'][:, 0]
            s['state'] = normal(batch, width - 1, channels, kind=dtype)
        elif case['entering']:
            s['state'] = leaf(normal(batch, width - 1, channels, kind=dtype))
        if train:
            s['d_y'] = normal(batch, length, channels, kind=dtype)
            s['d_last'] = normal(batch, width - 1, channels, kind=dtype)
        return s

    n, groups = case['state'], case['groups']
    s['u'] = leaf(normal(batch, length, channels, kind=dtype))
    # the gate is the other half of the projection whose first half went through the convolution
    s['z'] = leaf(normal(batch, length, 2 * channels, kind=dtype)[..., channels:]) if case['gate'] else None
    s['delta'] = leaf(normal(batch, length, channels, scale=0.5, kind=dtype))
    # time steps between 0.001 and 0.1, spread over their logarithm: the bias is the inverse of log(1 + exp(.))
    step = torch.exp(torch.rand(channels, generator=g, device='cuda') * math.log(100.0) + math.log(0.001))
    s['delta_bias'] = leaf(step + torch.log(-torch.expm1(-step)))
    rates = torch.arange(1, n + 1, device='cuda', dtype=torch.float32)
    s['A'] = leaf(-rates * torch.exp(normal(channels, n, scale=0.2)))
    # the vectors B and C lie side by side behind the low rank part of another projection
    rank = 64
    mixed = normal(batch, length, rank + 2 * groups * n, kind=dtype)
    s['B'] = leaf(mixed[..., rank:rank + groups * n].unflatten(-1, (groups, n)))
    s['C'] = leaf(mixed[..., rank + groups * n:].unflatten(-1, (groups, n)))
    s['D'] = leaf(1 + normal(channels, scale=0.1))
    s['state'] = None
    if op == 'scan_step':
        for key in ('u', 'z', 'delta', 'B', 'C'):
            s[key] = s[key] if s[key] is None else s[key][:, 0]
        s['state'] = normal(batch, channels, n)
    elif case['entering']:
        s['state'] = leaf(normal(batch, channels, n))
    if train:
        s['d_y'] = normal(batch, length, channels, kind=dtype)
        s['d_last'] = normal(batch, channels, n)
    return s


# ----------------------------------------------------------------------------------------------------------------------
# one pass
# ----------------------------------------------------------------------------------------------------------------------
def run(s):
    if own:
        return _run_own(s)
    with torch.no_grad():
        return _PLAIN[s['op']](s)


def _run_own(s):
    from opveclib_amd import rms_norm, state_space
    op = s['op']
    if op == 'norm_quantized':
        return rms_norm.rms_norm_quantized(s['x'], s['weight'], EPS, residual=s['residual'], group=s['group'])
    if op == 'norm_train':
        if s['residual'] is None:
            y = rms_norm.rms_norm_torch(s['x'], s['weight'], EPS)
            return (y, *torch.autograd.grad(y, (s['x'], s['weight']), s['d_y']))
        out = rms_norm.rms_norm_torch(s['x'], s['weight'], EPS, residual=s['residual'])
        return (*out, *torch.autograd.grad(out, (s['x'], s['residual'], s['weight']), (s['d_y'], s['d_summed'])))
    if op.startswith('conv'):
        if op == 'conv_step':
            y = state_space.conv_step(s['x'], s['state'], s['weight'], s['bias'], activation=s['activation'])
            return y, s['state']
        more = {'activation': s['activation'], 'state': s['state'], 'lengths': s['lengths']}
        if op == 'conv':
            return state_space.conv(s['x'], s['weight'], s['bias'], **more)
        out = state_space.conv_torch(s['x'], s['weight'], s['bias'], **more)
        leaves = [s[k] for k in ('x', 'weight', 'bias', 'state') if s[k] is not None]
        return (*out, *torch.autograd.grad(out, leaves, (s['d_y'], s['d_last'])))
    if op == 'scan_step':
        y = state_space.scan_step(s['state'], s['u'], s['delta'], s['A'], s['B'], s['C'], D=s['D'], z=s['z'],
                                  delta_bias=s['delta_bias'], softplus=True)
        return y, s['state']
    call = state_space.scan if op == 'scan' else state_space.scan_torch
    out = call(s['u'], s['delta'], s['A'], s['B'], s['C'], D=s['D'], z=s['z'], delta_bias=s['delta_bias'],
               softplus=True, state=s['state'], lengths=s['lengths'])
    if op == 'scan':
        return out
    leaves = [s[k] for k in ('u', 'delta', 'A', 'B', 'C', 'D', 'z', 'delta_bias', 'state') if s[k] is not None]
    return (*out, *torch.autograd.grad(out, leaves, (s['d_y'], s['d_last'])))


# ----------------------------------------------------------------------------------------------------------------------
# the plain forms: 32 bits, rounded once at the end
# ----------------------------------------------------------------------------------------------------------------------
def _summed(s):
    """The sum with the residual as it is stored (in the residual's type): what the norm is taken of."""
    if s['residual'] is None:
        return s['x'], s['x'].float()
    summed = (s['x'].float() + s['residual'].float()).to(s['residual'].dtype)
    return summed, summed.float()


def _plain_norm_quantized(s):
    summed, x = _summed(s)
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * s['weight'].float()
    rows, columns = y.shape
    group = s['group'] or columns
    padded = torch.nn.functional.pad(y, (0, -columns % group)).view(rows, -1, group)
    largest = padded.abs().amax(-1)
    scale = torch.where(largest > 0, largest / E4M3_MAX, torch.ones_like(largest))
    q = (padded / scale[..., None]).clamp(-E4M3_MAX, E4M3_MAX).view(rows, -1)[:, :columns].to(torch.float8_e4m3fn)
    return (q, scale) if s['residual'] is None else (q, scale, summed)


def _plain_norm_train(s):
    summed, x = _summed(s)
    weight, d_y = s['weight'].float(), s['d_y'].float()
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    unit = x * r
    y = (unit * weight).to(s['x'].dtype)
    d_unit = d_y * weight
    d_x = r * (d_unit - unit * (d_unit * unit).mean(-1, keepdim=True))
    d_weight = (d_y * unit).sum(0).to(s['weight'].dtype)
    if s['residual'] is None:
        return y, d_x.to(s['x'].dtype), d_weight
    d_x = d_x + s['d_summed'].float()
    return y, summed, d_x.to(s['x'].dtype), d_x.to(s['residual'].dtype), d_weight


def _valid(s, length, device):
    """Which positions hold tokens, [batch, length, 1]; None where all do."""
    if s['lengths'] is None:
        return None
    return (torch.arange(length, device=device) < s['lengths'][:, None])[..., None]


def _kept(t, valid):
    return t if valid is None else torch.where(valid, t, torch.zeros((), dtype=t.dtype, device=t.device))


def _plain_conv_parts(s):
    x, weight, bias = s['x'], s['weight'].float(), s['bias'].float()
    batch, length, channels = x.shape
    width = weight.shape[1]
    valid = _valid(s, length, x.device)
    before = x.new_zeros(batch, width - 1, channels) if s['state'] is None else s['state']
    line = torch.cat([before.float(), _kept(x.float(), valid)], 1)
    windows = line.unfold(1, width, 1)                                   # [batch, length, channels, width]
    pre = (windows * weight).sum(-1) + bias
    y = pre * torch.sigmoid(pre) if s['activation'] else pre
    ends = torch.full((batch,), length, device=x.device) if s['lengths'] is None else s['lengths'].long()
    at = ends[:, None] + torch.arange(width - 1, device=x.device)        # rows of `line` that the next call needs
    last = torch.gather(line, 1, at[..., None].expand(-1, -1, channels))
    return windows, pre, _kept(y, valid), last, at, valid


def _plain_conv(s):
    _, _, y, last, _, _ = _plain_conv_parts(s)
    return y.to(s['x'].dtype), last.to(s['x'].dtype)


def _plain_conv_train(s):
    windows, pre, y, last, at, valid = _plain_conv_parts(s)
    dtype = s['x'].dtype
    d_pre = _kept(s['d_y'].float(), valid)
    if s['activation']:
        gate = torch.sigmoid(pre)
        d_pre = d_pre * gate * (1 + pre * (1 - gate))
    batch, length, channels = d_pre.shape
    weight = s['weight'].float()
    width = weight.shape[1]
    d_weight = (windows * d_pre[..., None]).sum((0, 1))
    d_bias = d_pre.sum((0, 1))
    # position p of `line` is read by the windows p - width + 1 .. p
    behind = torch.nn.functional.pad(d_pre, (0, 0, width - 1, width - 1)).unfold(1, width, 1)
    d_line = (behind * weight.flip(1)).sum(-1)
    d_line = d_line.scatter_add(1, at[..., None].expand(-1, -1, channels), s['d_last'].float())
    d_x = _kept(d_line[:, width - 1:], valid)
    out = [y.to(dtype), last.to(dtype), d_x.to(dtype), d_weight, d_bias]
    return out if s['state'] is None else out + [d_line[:, :width - 1].to(dtype)]


def _plain_conv_step(s):
    line = torch.cat([s['state'].float(), s['x'].float()[:, None]], 1)
    pre = (line * s['weight'].float().t()).sum(1) + s['bias'].float()
    y = pre * torch.sigmoid(pre) if s['activation'] else pre
    s['state'].copy_(line[:, 1:])
    return y.to(s['x'].dtype), s['state']


def _time_steps(s, valid):
    raw = s['delta'].float() + s['delta_bias'].float()
    return raw, _kept(torch.log1p(torch.exp(-raw.abs())) + raw.clamp(min=0), valid)


def _along_time(a, b):
    """h[t] = a[t] h[t-1] + b[t] with h[-1] = 0 along axis 1, by doubling: after the step of width w every position
    holds the composition of the w positions that end in it."""
    w = 1
    while w < a.shape[1]:
        b = torch.cat([b[:, :w], torch.addcmul(b[:, w:], a[:, w:], b[:, :-w])], 1)
        a = torch.cat([a[:, :w], a[:, w:] * a[:, :-w]], 1)
        w *= 2
    return b


def _plain_scan_parts(s):
    """Everything as [batch, length, groups, channels of a group, state]."""
    batch, length, groups, n = s['B'].shape
    valid = _valid(s, length, s['u'].device)

    def grouped(t):
        return t.unflatten(-1, (groups, -1))

    raw, dt = _time_steps(s, valid)
    u = _kept(s['u'].float(), valid)
    A = s['A'].float().unflatten(0, (groups, -1))
    B = _kept(s['B'].float(), None if valid is None else valid[..., None])[:, :, :, None]
    C = _kept(s['C'].float(), None if valid is None else valid[..., None])[:, :, :, None]
    a = torch.exp(grouped(dt)[..., None] * A)
    x = grouped(dt * u)[..., None]
    b = x * B
    before = torch.zeros_like(a[:, 0]) if s['state'] is None else s['state'].unflatten(1, (groups, -1))
    b[:, 0] += a[:, 0] * before
    h = _along_time(a, b)
    y = (h * C).sum(-1).flatten(2) + s['D'].float() * u
    return valid, raw, dt, u, A, B, C, a, x, before, h, y, grouped


def _gated(y, s, valid):
    if s['z'] is None:
        return _kept(y, valid)
    z = s['z'].float()
    return _kept(y * z * torch.sigmoid(z), valid)


def _plain_scan(s):
    valid, *_, h, y, _ = _plain_scan_parts(s)
    return _gated(y, s, valid).to(s['u'].dtype), h[:, -1].flatten(1, 2)


def _plain_scan_train(s):
    valid, raw, dt, u, A, B, C, a, x, before, h, y, grouped = _plain_scan_parts(s)
    dtype = s['u'].dtype
    d_out = _kept(s['d_y'].float(), valid)
    d_y = d_out
    d_z = None
    if s['z'] is not None:
        z = s['z'].float()
        gate = torch.sigmoid(z)
        d_y = _kept(d_out * z * gate, valid)
        d_z = _kept(d_out * y * gate * (1 + z * (1 - gate)), valid)
    d_yg = grouped(d_y)[..., None]
    # g[t] = C[t] dy[t] + a[t+1] g[t+1]: the same recurrence from the other end
    inner = d_yg * C
    inner[:, -1] += s['d_last'].unflatten(1, (A.shape[0], -1))
    later = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
    g = _along_time(later.flip(1), inner.flip(1)).flip(1)
    d_x = (g * B).sum(-1).flatten(2)
    through = g * a * torch.cat([before[:, None], h[:, :-1]], 1)
    d_dt = (through * A).sum(-1).flatten(2) + d_x * u
    d_delta = _kept(d_dt * torch.sigmoid(raw), valid)
    out = [_gated(y, s, valid).to(dtype), h[:, -1].flatten(1, 2),
           (d_x * dt + s['D'].float() * d_y).to(dtype), d_delta.to(dtype),
           (through * grouped(dt)[..., None]).sum((0, 1)).flatten(0, 1),
           (g * x).sum(3).to(dtype), (d_yg * h).sum(3).to(dtype), (d_y * u).sum((0, 1))]
    out += [] if d_z is None else [d_z.to(dtype)]
    out += [d_delta.sum((0, 1))]
    return out if s['state'] is None else out + [(a[:, 0] * g[:, 0]).flatten(1, 2)]


def _plain_scan_step(s):
    _, dt = _time_steps(s, None)
    batch, groups, n = s['B'].shape
    u = s['u'].float()
    state = s['state'].unflatten(1, (groups, -1))
    a = torch.exp(dt.unflatten(1, (groups, -1))[..., None] * s['A'].unflatten(0, (groups, -1)))
    h = a * state + (dt * u).unflatten(1, (groups, -1))[..., None] * s['B'].float()[:, :, None]
    y = (h * s['C'].float()[:, :, None]).sum(-1).flatten(1) + s['D'] * u
    if s['z'] is not None:
        z = s['z'].float()
        y = y * z * torch.sigmoid(z)
    s['state'].copy_(h.flatten(1, 2))
    return y.to(s['u'].dtype), s['state']


_PLAIN = {'norm_quantized': _plain_norm_quantized, 'norm_train': _plain_norm_train, 'conv': _plain_conv,
          'conv_train': _plain_conv_train, 'conv_step': _plain_conv_step, 'scan': _plain_scan,
          'scan_train': _plain_scan_train, 'scan_step': _plain_scan_step}


# ----------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ----------------------------------------------------------------------------------------------------------------------
def work(case):
    op = case['op']
    e = torch.finfo(_TYPES[case['dtype']]).bits // 8
    if op.startswith('norm'):
        rows, columns = case['rows'], case['columns']
        every = rows * columns
        r = 0 if case['residual'] == 'none' else torch.finfo(_TYPES[case['residual']]).bits // 8
        if op == 'norm_quantized':
            scales = rows * (-(-columns // case['group']) if case['group'] else 1)
            return {'bytes': every * (e + 2 * r + 1) + 4 * scales + 4 * columns, 'flops': every * 7}
        # x, residual, d_y, d_summed in; y, the sum, d_x and the residual's gradient out
        return {'bytes': every * (4 * e + 4 * r) + 8 * columns, 'flops': every * 14}
    batch, length, channels = case['batch'], case['length'], case['channels']
    tokens = batch * length
    if op.startswith('conv'):
        width = case['width']
        kept = batch * (width - 1) * channels * e
        entering = kept if case['entering'] or op == 'conv_step' else 0
        params = 4 * channels * (width + 1)
        per = 2 * width + (6 if case['activation'] else 0)
        if op == 'conv_train':
            return {'bytes': tokens * channels * 4 * e + 2 * kept + 2 * entering + 2 * params,
                    'flops': tokens * channels * (per + 4 * width + 8)}
        return {'bytes': tokens * channels * 2 * e + kept + entering + params, 'flops': tokens * channels * per}
    n, groups = case['state'], case['groups']
    z = 1 if case['gate'] else 0
    kept = 4 * batch * channels * n
    entering = kept if case['entering'] or op == 'scan_step' else 0
    params = 4 * channels * (n + 2)
    vectors = tokens * 2 * groups * n * e
    if op == 'scan_train':
        # u, delta, z, d_y and B, C in; y, their gradients out
        return {'bytes': tokens * channels * e * (6 + 2 * z) + 2 * vectors + 2 * kept + 2 * entering + 2 * params,
                'flops': tokens * channels * (24 * n + 40)}
    return {'bytes': tokens * channels * e * (3 + z) + vectors + kept + entering + params,
            'flops': tokens * channels * (7 * n + 20)}


# ----------------------------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ----------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    op = case['op']
    train = op.endswith('train')

    def wide(key):
        t = s[key]
        if t is None:
            return None
        t = t.detach().double()
        return t.requires_grad_(True) if train else t

    def gradients(outs, ups, leaves):
        return torch.autograd.grad(outs, [t for t in leaves if t is not None], [u.double() for u in ups])

    if op.startswith('norm'):
        x, residual, weight = wide('x'), wide('residual'), wide('weight')
        total, summed = x, None
        if residual is not None:
            # the norm is that of the sum as stored: its rounding is part of the definition, its gradient that of the sum
            summed = (x + residual).detach().to(s['residual'].dtype)
            total = x + residual + (summed.double() - (x + residual)).detach()
        y = weight * total / torch.sqrt(total.square().mean(-1, keepdim=True) + EPS)
        if op == 'norm_train':
            if residual is None:
                return (y.detach(), *gradients([y], [s['d_y']], [x, weight]))
            return (y.detach(), summed.double(), *gradients([y, x + residual], [s['d_y'], s['d_summed']], [x, residual, weight]))
        parts = y.split(s['group'] or y.shape[1], 1)
        scale = torch.stack([p.abs().max(1).values / E4M3_MAX for p in parts], 1)
        scale[scale == 0] = 1
        q = torch.cat([p / scale[:, i:i + 1] for i, p in enumerate(parts)], 1)
        return (q, scale) if residual is None else (q, scale, summed.double())

    batch, length, channels = case['batch'], case['length'], case['channels']
    ends = [length] * batch if s['lengths'] is None else s['lengths'].tolist()
    if op.startswith('conv'):
        x, weight, bias, state = wide('x'), wide('weight'), wide('bias'), wide('state')
        if op == 'conv_step':
            x = x[:, None]
        width = case['width']
        ys, lasts = [], []
        for b in range(batch):
            before = torch.zeros(width - 1, channels, dtype=torch.float64, device='cuda') if state is None else state[b]
            line = torch.cat([before, x[b, :ends[b]]])
            pre = bias.expand(ends[b], channels)
            for k in range(width):
                pre = pre + weight[:, k] * line[k:k + ends[b]]
            y = pre / (1 + torch.exp(-pre)) if s['activation'] else pre
            ys.append(torch.cat([y, torch.zeros(length - ends[b], channels, dtype=torch.float64, device='cuda')]))
            lasts.append(line[ends[b]:])
        y, last = torch.stack(ys), torch.stack(lasts)
        if op == 'conv_step':
            return y[:, 0], last
        if op == 'conv':
            return y, last
        return (y.detach(), last.detach(), *gradients([y, last], [s['d_y'], s['d_last']], [x, weight, bias, state]))

    u, delta, A, B, C, D = (wide(k) for k in ('u', 'delta', 'A', 'B', 'C', 'D'))
    z, bias, state = wide('z'), wide('delta_bias'), wide('state')
    leaves = [u, delta, A, B, C, D, z, bias, state]
    if op == 'scan_step':
        u, delta, B, C = u[:, None], delta[:, None], B[:, None], C[:, None]
        z = None if z is None else z[:, None]
    per = channels // case['groups']
    step = torch.nn.functional.softplus(delta + bias, threshold=50)
    zero = torch.zeros((), dtype=torch.float64, device='cuda')
    h = torch.zeros(batch, channels, case['state'], dtype=torch.float64, device='cuda') if state is None else state
    end = torch.tensor(ends, device='cuda')
    ys = []
    for t in range(length):
        on = (t < end)[:, None]
        moved = torch.exp(step[:, t, :, None] * A) * h + (step[:, t] * u[:, t])[..., None] * B[:, t].repeat_interleave(per, 1)
        h = moved if s['lengths'] is None else torch.where(on[..., None], moved, h)
        y = (h * C[:, t].repeat_interleave(per, 1)).sum(-1) + D * u[:, t]
        y = y if z is None else y * z[:, t] / (1 + torch.exp(-z[:, t]))
        ys.append(y if s['lengths'] is None else torch.where(on, y, zero))
    y = torch.stack(ys, 1)
    if op == 'scan_step':
        return y[:, 0], h
    if op == 'scan':
        return y, h
    return (y.detach(), h.detach(), *gradients([y, h], [s['d_y'], s['d_last']], leaves))
