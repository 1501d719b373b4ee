"""
The state space scan and the short causal convolution (include/ovl_ssm.h) on the GPU, against their definitions in float64:
types, sizes from one token and channel on, padded batches, strides, groups, long sequences that are split; gradients
against automatic differentiation and against differences; the one-token forms against the whole; streams, captured
graphs, large offsets; and a layer of them together with the norm.
"""
import math

import pytest
import torch

from opveclib_amd import rms_norm, state_space
from tests import recurrent_layer as ref
from tests.recurrent_layer import close

pytestmark = pytest.mark.gpu

F32 = torch.float32


def call_args(d):
    return {k: d[k] for k in ('D', 'z', 'delta_bias', 'softplus', 'state', 'lengths')}


def run_scan(d):
    return state_space.scan(d['u'], d['delta'], d['A'], d['B'], d['C'], **call_args(d))


def run_grad(d, with_last=True):
    return state_space.scan_grad(d['u'], d['delta'], d['A'], d['B'], d['C'], d['d_y'],
                                 d_last=d['d_last'] if with_last else None, **call_args(d))


def check_scan(d, terms=16):
    kind = d['u'].dtype
    y, last = run_scan(d)
    cpu = {k: v.cpu() if isinstance(v, torch.Tensor) else v for k, v in d.items()}
    want_y, want_last, want = ref.scan_expected(cpu)
    close(y, want_y, kind, 'y', terms)
    close(last, want_last, F32, 'last', terms)
    for name, got, w in zip(ref.SCAN_NAMES, run_grad(d), want):
        assert (got is None) == (w is None), name
        if w is not None:
            close(got, w, kind if name in ('u', 'delta', 'z', 'B', 'C') else F32, 'd_' + name, 4 * terms)


# batch, length, channels, state, groups
SIZES = [(1, 1, 1, 1, 1), (2, 1, 64, 16, 1), (3, 15, 65, 16, 5), (1, 16, 130, 8, 2), (2, 17, 63, 17, 1), (2, 50, 8, 3, 8),
         (1, 33, 20, 33, 2), (2, 31, 12, 64, 1), (5, 40, 100, 12, 2)]


@pytest.mark.parametrize('dtype', ['float32', 'float16', 'bfloat16'])
@pytest.mark.parametrize('size', SIZES, ids=str)
def test_scan_and_its_gradient(size, dtype):
    batch, length, channels, n, groups = size
    odd = (length + channels) % 2 == 1
    check_scan(ref.scan_inputs(hash(size) % 1000, batch, length, channels, n, groups, dtype, gate=not odd or n == 16,
                               ragged=batch > 1 and not odd, entering=odd, softplus=channels != 63, device='cuda'))


@pytest.mark.parametrize('absent', ['D', 'z', 'delta_bias', 'state', 'all'])
def test_optional_inputs(absent):
    d = ref.scan_inputs(3, 2, 37, 24, 16, 1, 'float32', device='cuda')
    for key in ('D', 'z', 'delta_bias', 'state') if absent == 'all' else (absent,):
        d[key] = None
    if d['delta_bias'] is None:
        d['softplus'] = False
        d['delta'] = d['delta'].abs() * 0.05
    check_scan(d)


@pytest.mark.parametrize('dtype', ['float32', 'bfloat16'])
@pytest.mark.parametrize('size', [(1, 300, 6, 16, 1), (3, 260, 70, 8, 2), (2, 1000, 3, 40, 1)], ids=str)
def test_long_sequences_are_split_without_a_trace(size, dtype):
    """Few channels: the tokens are worked on in chunks whose states are joined (checked by the size of the scratch
    memory); one sequence ends before the last chunks begin."""
    batch, length, channels, n, groups = size
    d = ref.scan_inputs(9, batch, length, channels, n, groups, dtype, ragged=batch > 1, device='cuda')
    if batch > 1:
        d['lengths'][0] = 40
    _, packed, _ = state_space._describe_scan(torch, d['u'], d['delta'], d['A'], d['B'], d['C'], d['D'], d['z'],
                                              d['delta_bias'], True, d['state'], d['lengths'])
    assert state_space.library().ovl_ssm_scan_workspace_bytes(packed, 0) > 0
    check_scan(d, terms=32)


@pytest.mark.parametrize('size', [(1, 2300, 2, 3, 1), (1, 170, 64 * 400, 2, 1), (2, 100, 64 * 300, 1, 2)], ids=str)
def test_splits_into_more_chunks_than_are_joined_at_once_and_into_unequal_ones(size):
    """144 chunks in both directions; 11 tiles in 6 resp. 9 chunks; enough channels for a split in one direction only."""
    batch, length, channels, n, groups = size
    d = ref.scan_inputs(10, batch, length, channels, n, groups, 'float32', ragged=batch > 1, device='cuda')
    check_scan(d, terms=32)


def test_slow_decay_over_a_long_sequence_keeps_its_precision():
    """Decays near one: the state is a sum over thousands of tokens."""
    d = ref.scan_inputs(11, 1, 3000, 2, 16, 1, 'float32', gate=False, entering=True, device='cuda')
    d['A'] = d['A'] * 1e-3
    y, last = run_scan(d)
    cpu = {k: v.cpu() if isinstance(v, torch.Tensor) else v for k, v in d.items()}
    with torch.no_grad():
        leaves = {k: ref.wide(cpu[k]) for k in ref.SCAN_NAMES}
        want_y, want_last = ref.scan(softplus=True, **leaves)
    # a state's roundings add up at random over the tokens that it remembers: sqrt(3000) = 55 of them
    close(y, want_y, F32, 'y', 64)
    close(last, want_last, F32, 'last', 64)


def test_groups_share_vectors_and_three_axes_mean_one_group():
    d = ref.scan_inputs(12, 2, 20, 12, 8, 1, 'float32', device='cuda')
    y, last = run_scan(d)
    flat = dict(d, B=d['B'][:, :, 0], C=d['C'][:, :, 0])
    y3, last3 = run_scan(flat)
    assert torch.equal(y, y3) and torch.equal(last, last3)
    grads = run_grad(flat)
    assert grads[3].shape == flat['B'].shape
    # four groups with the same vectors are one group; their gradients add up to its
    four = dict(d, B=d['B'].expand(2, 20, 4, 8), C=d['C'].expand(2, 20, 4, 8))
    y4, _ = run_scan(four)
    assert torch.equal(y, y4)
    close(run_grad(four)[3].sum(2), grads[3].double(), F32, 'd_B', 8)


def test_strides_and_broadcast_inputs():
    """Parts of wider tensors, a transposed sequence (which is copied), a token repeated by a stride of zero."""
    d = ref.scan_inputs(13, 3, 22, 18, 16, 1, 'bfloat16', device='cuda')
    want = run_scan(d) + tuple(run_grad(d))
    wide = torch.randn(3, 22, 50, device='cuda').bfloat16()
    wide[..., 5:23], wide[..., 30:48] = d['u'], d['z']
    moved = dict(d, u=wide[..., 5:23], z=wide[..., 30:48], delta=d['delta'].transpose(1, 2).contiguous().transpose(1, 2),
                 d_y=d['d_y'].transpose(0, 1).contiguous().transpose(0, 1))
    mixed = torch.randn(3, 22, 40, device='cuda').bfloat16()
    mixed[..., 1:17], mixed[..., 17:33] = d['B'][:, :, 0], d['C'][:, :, 0]
    moved.update(B=mixed[..., 1:17].unflatten(-1, (1, 16)), C=mixed[..., 17:33].unflatten(-1, (1, 16)),
                 A=d['A'].t().contiguous().t())
    for a, b in zip(want, run_scan(moved) + tuple(run_grad(moved))):
        assert torch.equal(a, b)
    same = dict(d, u=d['u'][:, :1].expand(3, 22, 18), B=d['B'][:1].expand(3, 22, 1, 16))
    full = dict(same, u=same['u'].contiguous(), B=same['B'].contiguous())
    for a, b in zip(run_scan(same) + tuple(run_grad(same)), run_scan(full) + tuple(run_grad(full))):
        assert torch.equal(a, b)


@pytest.mark.parametrize('op', ['scan', 'conv'])
def test_padding_is_not_looked_at(op):
    """What lies behind a sequence may be NaN or infinite; outputs and gradients there are zero; a sequence without tokens
    hands its state through, and lengths beyond either end are clamped."""
    lengths = torch.tensor([0, 7, 40, -3, 99], dtype=torch.int32, device='cuda')
    if op == 'scan':
        d = ref.scan_inputs(14, 5, 40, 33, 16, 1, 'float32', device='cuda')
        names, grad_names = ('u', 'delta', 'z', 'B', 'C', 'd_y'), (0, 1, 3, 4, 6)
        both = lambda v: run_scan(v) + tuple(run_grad(v))
    else:
        d = ref.conv_inputs(14, 5, 40, 33, 4, 'float32', device='cuda')
        names, grad_names = ('x', 'd_y'), (0,)
        both = lambda v: state_space.conv(v['x'], v['weight'], v['bias'], 'silu', v['state'], v['lengths']) + \
            state_space.conv_grad(v['x'], v['weight'], v['d_y'], v['bias'], 'silu', v['state'], v['lengths'], v['d_last'])
    d['lengths'] = lengths
    clean = both(d)
    for bad in (float('nan'), float('inf'), -float('inf'), torch.finfo(F32).min):
        dirty = dict(d)
        for name in names:
            dirty[name] = d[name].clone()
            for b, end in enumerate((0, 7, 40, 0, 40)):
                dirty[name][b, end:] = bad
        for a, b in zip(clean, both(dirty)):
            assert torch.equal(a, b)
    for which in (0,) + tuple(2 + g for g in grad_names):
        for b, end in enumerate((0, 7, 40, 0, 40)):
            assert not clean[which][b, end:].any()
    assert torch.equal(clean[1][0], d['state'][0]) and torch.equal(clean[1][3], d['state'][3])
    if op == 'scan':
        assert torch.equal(clean[-1][0], d['d_last'][0])
        check_scan(d)


def test_non_finite_values_stay_in_their_sequence_and_channel():
    d = ref.scan_inputs(15, 2, 30, 20, 16, 1, 'float32', gate=True, device='cuda')
    y, last = run_scan(d)
    d['u'][0, 11, 4] = float('nan')
    bad_y, bad_last = run_scan(d)
    assert torch.isnan(bad_y[0, 11:, 4]).all() and torch.isnan(bad_last[0, 4]).all()
    keep = torch.ones_like(y, dtype=torch.bool)
    keep[0, 11:, 4] = False
    assert torch.equal(y[keep], bad_y[keep])


@pytest.mark.parametrize('delta', [-200.0, -88.0, -20.0, -5.0, 0.0, 5.0, 30.0, 100.0])
def test_softplus_over_its_whole_range(delta):
    """One token from an empty state with A = 0: y = softplus(delta) when u, B, C are one."""
    one = torch.ones(1, 1, 8, device='cuda')
    value = torch.full((1, 1, 8), delta, device='cuda') + torch.linspace(-0.9, 0.9, 8, device='cuda')
    y, _ = state_space.scan(one, value, torch.zeros(8, 1, device='cuda'), one[..., :1], one[..., :1], softplus=True)
    want = torch.log1p(torch.exp(-value.double().abs())) + value.double().clamp(min=0)
    # float32 arithmetic (a few roundings), and results in its subnormal range are zero
    assert bool(((y.double() - want).abs() <= want * 2.0 ** -21 + 2.0 ** -126).all())


def test_gradient_against_differences():
    d = ref.scan_inputs(16, 2, 25, 10, 8, 2, 'float32', device='cuda')
    grads = dict(zip(ref.SCAN_NAMES, run_grad(d)))

    def loss(v):
        y, last = run_scan(v)
        return float((y.double() * d['d_y'].double()).sum() + (last.double() * d['d_last'].double()).sum())

    for name in ref.SCAN_NAMES:
        g = torch.Generator(device='cuda')
        g.manual_seed(1)
        way = torch.randn(d[name].shape, generator=g, device='cuda') * 1e-2
        slope = (loss(dict(d, **{name: d[name] + way})) - loss(dict(d, **{name: d[name] - way}))) / 2
        formula = float((grads[name].double() * way.double()).sum())
        # the step leaves a third-order term of about its square, 1e-4, and the outputs' roundings
        scale = float((grads[name].double() * way.double()).abs().sum())
        assert abs(slope - formula) <= 1e-3 * scale + 1e-5, (name, slope, formula)


@pytest.mark.parametrize('dtype', ['float32', 'float16', 'bfloat16'])
@pytest.mark.parametrize('size', [(1, 1, 1, 1), (3, 64, 16, 1), (130, 33, 16, 3), (2, 70, 24, 2), (5, 9, 64, 1), (4, 128, 8, 1),
                                  (2, 20, 32, 4)], ids=str)
def test_scan_step(size, dtype):
    batch, channels, n, groups = size
    d = ref.scan_inputs(17, batch, 1, channels, n, groups, dtype, gate=n != 24, device='cuda')
    cpu = {k: v.cpu() if isinstance(v, torch.Tensor) else v for k, v in d.items()}
    want_y, want_last, _ = ref.scan_expected(cpu)
    # the state is a part of a larger buffer whose rest stays as it is
    pool = torch.full((batch, channels + 4, n), 7.0, device='cuda')
    state = pool[:, :channels]
    state.copy_(d['state'])
    first = lambda k: None if d[k] is None else d[k][:, 0]
    y = state_space.scan_step(state, first('u'), first('delta'), d['A'], first('B'), first('C'), d['D'], first('z'),
                              d['delta_bias'], True)
    close(y, want_y[:, 0], d['u'].dtype, 'y', 16)
    close(state, want_last, F32, 'state', 16)
    assert bool((pool[:, channels:] == 7.0).all())


CONVS = [(1, 1, 1, 1), (2, 1, 8, 4), (3, 19, 24, 4), (2, 37, 10, 3), (4, 2, 7, 4), (2, 70, 130, 2), (1, 600, 16, 4), (5, 33, 260, 3)]


@pytest.mark.parametrize('dtype', ['float32', 'float16', 'bfloat16'])
@pytest.mark.parametrize('size', CONVS, ids=str)
def test_conv_and_its_gradient(size, dtype):
    batch, length, channels, width = size
    kind = ref.TYPES[dtype]
    for activation, ragged, entering, bias in ((None, False, False, False), ('silu', batch > 1, True, True)):
        d = ref.conv_inputs(18, batch, length, channels, width, dtype, ragged, entering, bias, device='cuda')
        cpu = {k: v.cpu() if isinstance(v, torch.Tensor) else v for k, v in d.items()}
        want_y, want_last, want = ref.conv_expected(cpu, activation)
        wide = torch.full((batch, length, channels + 3), float('nan'), dtype=kind, device='cuda')
        wide[..., :channels] = d['x']
        for x in (d['x'], wide[..., :channels], d['x'].transpose(1, 2).contiguous().transpose(1, 2)):
            y, last = state_space.conv(x, d['weight'], d['bias'], activation, d['state'], d['lengths'])
            close(y, want_y, kind, 'y', 4)
            assert torch.equal(last.double().cpu(), want_last)
            got = state_space.conv_grad(x, d['weight'], d['d_y'], d['bias'], activation, d['state'], d['lengths'],
                                        d['d_last'] if width > 1 else None)
            for name, g, w in zip(ref.CONV_NAMES, got, want):
                assert (g is None) == (w is None)
                if w is not None:
                    # the taps' gradients are sums over all tokens in float32, whose roundings add up at random
                    close(g, w, kind if name in ('x', 'state') else F32, 'd_' + name, 16 + math.sqrt(batch * length))


@pytest.mark.parametrize('width', [1, 2, 3, 4])
def test_conv_step_continues_a_sequence(width):
    """Prompts of unequal length in one call, then token by token: the same as everything at once."""
    d = ref.conv_inputs(19, 3, 30, 40, width, 'bfloat16', device='cuda')
    lengths = torch.tensor([0, 2, 21], dtype=torch.int32, device='cuda')
    _, state = state_space.conv(d['x'], d['weight'], d['bias'], 'silu', d['state'], lengths)
    for b, end in enumerate(lengths.tolist()):
        whole, last = state_space.conv(d['x'][b:b + 1], d['weight'], d['bias'], 'silu', d['state'][b:b + 1])
        own = state[b:b + 1].clone()
        for t in range(end, 30):
            y = state_space.conv_step(d['x'][b:b + 1, t], own, d['weight'], d['bias'], 'silu')
            assert torch.equal(y, whole[:, t])
        assert torch.equal(own, last)


def test_parameters_of_the_sequences_type():
    d = ref.conv_inputs(20, 2, 12, 16, 4, 'bfloat16', device='cuda')
    w, b = d['weight'].bfloat16(), d['bias'].bfloat16()
    y, _ = state_space.conv(d['x'], w, b)
    want, _ = state_space.conv(d['x'], w.float(), b.float())
    assert torch.equal(y, want)
    grads = state_space.conv_grad(d['x'], w, d['d_y'], b)
    assert grads[1].dtype == torch.bfloat16 and grads[2].dtype == torch.bfloat16


@pytest.mark.parametrize('dtype', ['bfloat16', 'float16'])
@pytest.mark.parametrize('channels,width', [(16, 4), (12, 3), (7, 4), (600, 2)])
def test_weights_of_the_sequences_type_are_widened(channels, width, dtype):
    """Bit for bit the call with the same weights in float32, also where only one of the two is narrow."""
    kind = ref.TYPES[dtype]
    d = ref.conv_inputs(22, 2, 33, channels, width, dtype, ragged=True, entering=True, device='cuda')
    w, b = d['weight'].to(kind), d['bias'].to(kind)

    def all_forms(w, b):
        y, last = state_space.conv(d['x'], w, b, 'silu', d['state'], d['lengths'])
        grads = state_space.conv_grad(d['x'], w, d['d_y'], b, 'silu', d['state'], d['lengths'], d['d_last'])
        own = d['state'].clone()
        return [y, last, state_space.conv_step(d['x'][:, 0].contiguous(), own, w, b, 'silu'), own] + list(grads)

    want = all_forms(w.float(), b.float())
    for weight, bias in ((w, b), (w, b.float()), (w.float(), b)):
        for got, expected in zip(all_forms(weight, bias), want):
            assert torch.equal(got, expected.to(got.dtype))


def test_autograd_functions_give_the_gradients():
    d = ref.scan_inputs(21, 2, 35, 12, 16, 1, 'float32', ragged=True, device='cuda')
    leaves = {k: d[k].clone().requires_grad_(True) for k in ref.SCAN_NAMES}
    args = [leaves[k] for k in ('u', 'delta', 'A', 'B', 'C')]
    more = {k: leaves[k] for k in ('D', 'z', 'delta_bias', 'state')}
    y, last = state_space.scan_torch(*args, softplus=True, lengths=d['lengths'], **more)
    plain_y, plain_last = run_scan(d)
    assert torch.equal(y, plain_y) and torch.equal(last, plain_last)
    got = torch.autograd.grad((y, last), list(leaves.values()), (d['d_y'], d['d_last']), retain_graph=True)
    for a, b in zip(got, run_grad(d)):
        assert torch.equal(a, b)
    # one output only; only some inputs
    got = torch.autograd.grad(y, [leaves['u'], leaves['A']], d['d_y'])
    want = run_grad(d, with_last=False)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[2])
    c = ref.conv_inputs(22, 2, 20, 12, 4, 'float32', device='cuda')
    leaves = {k: c[k].clone().requires_grad_(True) for k in ref.CONV_NAMES}
    out = state_space.conv_torch(leaves['x'], leaves['weight'], leaves['bias'], 'silu', leaves['state'])
    got = torch.autograd.grad(out, list(leaves.values()), (c['d_y'], c['d_last']))
    for a, b in zip(got, state_space.conv_grad(c['x'], c['weight'], c['d_y'], c['bias'], 'silu', c['state'], None, c['d_last'])):
        assert torch.equal(a, b)
    # a broadcast input: its gradient is summed over what it was repeated along
    row = d['u'][:, :1].clone().requires_grad_(True)
    y, _ = state_space.scan_torch(row.expand_as(d['u']), d['delta'], d['A'], d['B'], d['C'], softplus=True)
    grad, = torch.autograd.grad(y, row, d['d_y'])
    full = state_space.scan_grad(row.detach().expand_as(d['u']), d['delta'], d['A'], d['B'], d['C'], d['d_y'], softplus=True)[0]
    close(grad, full.double().sum(1, keepdim=True), F32, 'broadcast', 16)


def test_gradients_of_one_output_alone():
    d = ref.scan_inputs(30, 2, 21, 12, 16, 1, 'float32', device='cuda')
    c = ref.conv_inputs(30, 2, 21, 12, 4, 'float32', device='cuda')
    for op, names in (('scan', ref.SCAN_NAMES), ('conv', ref.CONV_NAMES)):
        v = d if op == 'scan' else c
        leaves = {k: v[k].clone().requires_grad_(True) for k in names}
        if op == 'scan':
            out = state_space.scan_torch(*[leaves[k] for k in ('u', 'delta', 'A', 'B', 'C')], softplus=True,
                                         **{k: leaves[k] for k in ('D', 'z', 'delta_bias', 'state')})
            grad = lambda d_y, d_last: run_grad(dict(v, d_y=d_y, d_last=d_last))
        else:
            out = state_space.conv_torch(leaves['x'], leaves['weight'], leaves['bias'], 'silu', leaves['state'])
            grad = lambda d_y, d_last: state_space.conv_grad(c['x'], c['weight'], d_y, c['bias'], 'silu', c['state'], None, d_last)
        zero_y, zero_last = torch.zeros_like(v['d_y']), torch.zeros_like(v['d_last'])
        for which, want in ((0, grad(v['d_y'], zero_last)), (1, grad(zero_y, v['d_last']))):
            got = torch.autograd.grad(out[which], list(leaves.values()), v['d_last' if which else 'd_y'], retain_graph=True)
            for a, b in zip(got, want):
                assert torch.equal(a, b)


def test_a_state_that_a_backward_pass_needs_is_not_overwritten_unnoticed():
    d = ref.scan_inputs(31, 2, 5, 12, 16, 1, 'float32', device='cuda')
    c = ref.conv_inputs(31, 2, 5, 12, 4, 'float32', device='cuda')
    u, x = d['u'].clone().requires_grad_(True), c['x'].clone().requires_grad_(True)
    y, _ = state_space.scan_torch(u, d['delta'], d['A'], d['B'], d['C'], softplus=True, state=d['state'])
    out, _ = state_space.conv_torch(x, c['weight'], c['bias'], 'silu', c['state'])
    state_space.scan_step(d['state'], d['u'][:, 0], d['delta'][:, 0], d['A'], d['B'][:, 0], d['C'][:, 0], softplus=True)
    state_space.conv_step(c['x'][:, 0], c['state'], c['weight'], c['bias'], 'silu')
    for result in (y, out):
        with pytest.raises(RuntimeError, match='modified by an inplace operation'):
            result.sum().backward()
    with torch.inference_mode():
        state = torch.zeros_like(d['state'])
        state_space.scan_step(state, d['u'][:, 0], d['delta'][:, 0], d['A'], d['B'][:, 0], d['C'][:, 0], softplus=True)


def test_sequences_without_tokens_and_batches_without_sequences():
    for batch, length in ((2, 0), (0, 5)):
        d = ref.scan_inputs(23, batch, length, 6, 4, 1, 'float32', device='cuda')
        y, last = run_scan(d)
        assert y.shape == (batch, length, 6) and torch.equal(last, d['state'])
        grads = run_grad(d)
        assert torch.equal(grads[8], d['d_last'])
        assert all(not g.any() for g in grads[:8])
        assert not state_space.scan(d['u'], d['delta'], d['A'], d['B'], d['C'])[1].any()
        c = ref.conv_inputs(23, batch, length, 6, 4, 'float32', device='cuda')
        y, last = state_space.conv(c['x'], c['weight'], c['bias'], None, c['state'])
        assert y.shape == (batch, length, 6) and torch.equal(last, c['state'])
        grads = state_space.conv_grad(c['x'], c['weight'], c['d_y'], c['bias'], None, c['state'], None, c['d_last'])
        assert torch.equal(grads[3], c['d_last']) and not grads[1].any() and not grads[2].any()
    empty = torch.empty(0, 6, device='cuda')
    assert state_space.scan_step(torch.empty(0, 6, 4, device='cuda'), empty, empty, torch.zeros(6, 4, device='cuda'),
                                 torch.empty(0, 4, device='cuda'), torch.empty(0, 4, device='cuda')).shape == (0, 6)
    assert state_space.conv_step(empty, torch.empty(0, 3, 6, device='cuda'), torch.zeros(6, 4, device='cuda')).shape == (0, 6)


def test_arguments_that_do_not_fit_are_refused():
    d = ref.scan_inputs(24, 2, 8, 12, 4, 1, 'float32', device='cuda')
    good = dict(u=d['u'], delta=d['delta'], A=d['A'], B=d['B'], C=d['C'])
    bad = [dict(u=d['u'][0]), dict(u=d['u'].double()), dict(delta=d['delta'][:, :7]), dict(delta=d['delta'].half()),
           dict(delta=d['delta'].cpu()), dict(A=d['A'][:11]), dict(A=d['A'].half()), dict(A=torch.zeros(12, 65, device='cuda')),
           dict(A=torch.zeros(12, 0, device='cuda')), dict(B=d['B'][..., :3]), dict(C=d['C'][:, :, 0]), dict(C=d['C'].half()),
           dict(B=d['B'].expand(2, 8, 5, 4), C=d['C'].expand(2, 8, 5, 4)), dict(D=d['D'].half()), dict(D=d['D'][:3]),
           dict(z=d['z'][:1]), dict(delta_bias=d['D'].cpu()), dict(state=d['state'].half()), dict(state=d['state'][:1]),
           dict(lengths=torch.zeros(2, device='cuda')), dict(lengths=torch.zeros(3, dtype=torch.int32, device='cuda')),
           dict(lengths=torch.zeros(2, dtype=torch.int32)), dict(lengths=[3, 4])]
    for change in bad:
        with pytest.raises(TypeError):
            state_space.scan(**dict(good, **change))
    with pytest.raises(TypeError):
        state_space.scan_grad(d_y=None, **good)
    with pytest.raises(TypeError):
        state_space.scan_grad(d_y=d['d_y'][:, :3], **good)
    with pytest.raises(TypeError):
        state_space.scan_grad(d_y=d['d_y'], saved=torch.zeros(5, device='cuda'), **good)
    step = dict(u=d['u'][:, 0], delta=d['delta'][:, 0], A=d['A'], B=d['B'][:, 0], C=d['C'][:, 0])
    state = d['state'].clone()
    overlapping = torch.zeros(1, 12, 4, device='cuda').expand(2, 12, 4)
    for wrong in (state.half(), state[:1], state.cpu(), overlapping, state.transpose(1, 2).contiguous().transpose(1, 2),
                  state.clone().requires_grad_(True), None):
        with pytest.raises(TypeError):
            state_space.scan_step(wrong, **step)
    c = ref.conv_inputs(24, 2, 8, 12, 4, 'float32', device='cuda')
    for change in (dict(x=c['x'][0]), dict(weight=torch.zeros(12, 5, device='cuda')), dict(weight=c['weight'][:3]),
                   dict(weight=c['weight'].half()), dict(bias=c['bias'][:3]), dict(state=c['state'][:, :2]),
                   dict(state=c['state'].half()), dict(lengths=torch.zeros(2, dtype=torch.int64, device='cuda'))):
        with pytest.raises(TypeError):
            state_space.conv(**dict(dict(x=c['x'], weight=c['weight']), **change))
    with pytest.raises(ValueError):
        state_space.conv(c['x'], c['weight'], activation='gelu')
    for wrong in (c['state'][:, :, :6], c['state'][:1].expand(2, 3, 12), c['state'].half(), None):
        with pytest.raises(TypeError):
            state_space.conv_step(c['x'][:, 0], wrong, c['weight'])


def test_equal_calls_give_equal_bits():
    d = ref.scan_inputs(25, 3, 500, 40, 16, 1, 'float32', device='cuda')
    first = run_scan(d) + run_grad(d)
    for _ in range(3):
        for a, b in zip(first, run_scan(d) + run_grad(d)):
            assert torch.equal(a, b)


def test_streams_of_their_own():
    """Two calls at once on two streams, each behind work of its stream."""
    sets = [ref.scan_inputs(s, 2, 400, 30, 16, 1, 'float32', device='cuda') for s in (26, 27)]
    want = [run_scan(d) + run_grad(d) for d in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    for _ in range(3):
        got = []
        for d, stream in zip(sets, streams):
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                d = dict(d, u=d['u'] * 2 * 0.5)
                got.append(run_scan(d) + run_grad(d))
        torch.cuda.synchronize()
    for a, b in zip(want, got):
        for x, y in zip(a, b):
            assert torch.equal(x, y)


def test_captured_graphs_replay():
    """A decoding step (convolution, scan, norm) and a forward and backward pass, captured and replayed on new inputs with
    eager work in between; two graphs captured one after the other do not share memory that they still use."""
    d = ref.scan_inputs(28, 4, 300, 24, 16, 1, 'float32', device='cuda')
    c = ref.conv_inputs(28, 4, 1, 24, 4, 'float32', device='cuda')
    w = torch.ones(24, device='cuda')
    x, state, kept = c['x'][:, 0].clone(), d['state'].clone(), c['state'].clone()

    def token(x, state, kept):
        h = state_space.conv_step(rms_norm.rms_norm(x, w), kept, c['weight'], c['bias'], 'silu')
        return state_space.scan_step(state, h, d['delta'][:, 0], d['A'], d['B'][:, 0], d['C'][:, 0], d['D'], h,
                                     d['delta_bias'], True)

    def whole(u):
        y, last = state_space.scan(u, d['delta'], d['A'], d['B'], d['C'], **call_args(d))
        return (y, last) + state_space.scan_grad(u, d['delta'], d['A'], d['B'], d['C'], d['d_y'], d_last=d['d_last'], **call_args(d))

    u = d['u'].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        token(x.clone(), state.clone(), kept.clone())
        whole(u)
    torch.cuda.current_stream().wait_stream(side)
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    with torch.cuda.graph(graphs[0]):
        y_graph = token(x, state, kept)
    with torch.cuda.graph(graphs[1]):
        whole_graph = whole(u)
    eager_state, eager_kept = d['state'].clone(), c['state'].clone()
    state.copy_(d['state'])
    kept.copy_(c['state'])
    for k in range(4):
        new = torch.randn(4, 24, device='cuda')
        new_u = torch.randn_like(u)
        x.copy_(new)
        u.copy_(new_u)
        graphs[0].replay()
        graphs[1].replay()
        want = token(new, eager_state, eager_kept)
        want_whole = whole(new_u)
        torch.cuda.synchronize()
        assert torch.equal(y_graph, want) and torch.equal(state, eager_state) and torch.equal(kept, eager_kept)
        for a, b in zip(whole_graph, want_whole):
            assert torch.equal(a, b)


def test_training_step_in_a_captured_graph():
    """Forward and backward through the autograd functions inside a capture, with gradients asked for by name (an eager
    graph of the same leaves lives beside it)."""
    d = ref.scan_inputs(29, 2, 40, 16, 16, 1, 'float32', device='cuda')
    leaves = {k: d[k].clone().requires_grad_(True) for k in ref.SCAN_NAMES}

    def step():
        y, last = state_space.scan_torch(*[leaves[k] for k in ('u', 'delta', 'A', 'B', 'C')], softplus=True,
                                         **{k: leaves[k] for k in ('D', 'z', 'delta_bias', 'state')})
        return torch.autograd.grad((y, last), list(leaves.values()), (d['d_y'], d['d_last']))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grads = step()
    for k in range(3):
        with torch.no_grad():
            leaves['u'].copy_(torch.randn_like(d['u']))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(grads, step()):
            assert torch.equal(a, b)


def test_offsets_beyond_32_bits():
    """Sequences whose parts lie more than 2^32 bytes apart, and outputs longer than that."""
    channels, length = 40, 20
    apart = 2 ** 31 + 64
    buffer = torch.zeros(apart + length * channels, dtype=torch.float16, device='cuda')
    far = buffer.as_strided((2, length, channels), (apart, channels, 1))
    d = ref.scan_inputs(30, 2, length, channels, 16, 1, 'float16', device='cuda')
    far.copy_(d['u'])
    want = run_scan(d) + run_grad(d)
    moved = dict(d, u=far)
    for a, b in zip(want, run_scan(moved) + run_grad(moved)):
        assert torch.equal(a, b)
    w = torch.randn(channels, 4, device='cuda')
    for a, b in zip(state_space.conv(d['u'], w), state_space.conv(far, w)):
        assert torch.equal(a, b)
    del buffer, far, moved
    tokens = 2 ** 31 // 4096 + 5
    x = torch.randn(1, 64, 4096, device='cuda').half().repeat(1, tokens // 64 + 1, 1)[:, :tokens]
    w = torch.randn(4096, 3, device='cuda')
    y, _ = state_space.conv(x, w, activation='silu')
    tail, _ = state_space.conv(x[:, -40:].contiguous(), w, activation='silu')
    assert torch.equal(y[:, -38:], tail[:, 2:])


class Layer(torch.nn.Module):
    """A layer as it is used: norm with the residual's addition, projection, convolution, projections of its output, scan
    with gate, projection back."""

    def __init__(self, width, inner, n, rank, seed, dtype):
        super().__init__()
        g = torch.Generator()
        g.manual_seed(seed)
        make = lambda *s, scale=1.0, kind=dtype: torch.nn.Parameter((torch.randn(s, generator=g) * scale).to(kind))
        self.inner, self.n, self.rank = inner, n, rank
        self.norm = make(width, kind=F32)
        self.into = make(2 * inner, width, scale=width ** -0.5)
        self.taps, self.taps_bias = make(inner, 4, scale=0.5, kind=F32), make(inner, scale=0.1, kind=F32)
        self.mix = make(rank + 2 * n, inner, scale=inner ** -0.5)
        self.steps = make(inner, rank, scale=rank ** -0.5)
        self.steps_bias = torch.nn.Parameter(torch.full((inner,), -3.0))
        self.A = torch.nn.Parameter(-(1 + torch.arange(n).float()).repeat(inner, 1))
        self.D = torch.nn.Parameter(torch.ones(inner))
        self.out = make(width, inner, scale=inner ** -0.5)

    def forward(self, x, residual, kept=None, state=None, lengths=None, one=False, ops=None):
        """ops: (norm, conv, scan) to be used in place of the package's."""
        if ops is None:
            if one:
                norm = lambda x, w, residual: rms_norm.rms_norm(x, w, residual=residual)
                conv = lambda x, *a: (state_space.conv_step(x, kept, *a, 'silu'), kept)
                scan = lambda u, *a, **k: (state_space.scan_step(state, u, *a, softplus=True, **k), state)
            else:
                norm = lambda x, w, residual: rms_norm.rms_norm_torch(x, w, residual=residual)
                conv = lambda x, *a: state_space.conv_torch(x, *a, 'silu', kept, lengths)
                scan = lambda u, *a, **k: state_space.scan_torch(u, *a, softplus=True, state=state, lengths=lengths, **k)
        else:
            norm, conv, scan = ops
        y, residual = norm(x, self.norm, residual)
        both = y @ self.into.t()
        u, kept = conv(both[..., :self.inner], self.taps, self.taps_bias)
        mixed = u @ self.mix.t()
        delta = mixed[..., :self.rank] @ self.steps.t()
        y, state = scan(u, delta, self.A, mixed[..., self.rank:self.rank + self.n], mixed[..., self.rank + self.n:], D=self.D,
                        z=both[..., self.inner:], delta_bias=self.steps_bias)
        return y @ self.out.t(), residual, kept, state


def test_layers_prompt_in_parts_and_token_by_token():
    """Two layers: a padded batch of prompts, then tokens one by one, against all tokens of a sequence at once (float32: the
    ways differ by the roundings of the products alone)."""
    layers = [Layer(32, 48, 16, 8, s, F32).cuda() for s in (1, 2)]
    g = torch.Generator(device='cuda')
    g.manual_seed(3)
    x = torch.randn(3, 30, 32, generator=g, device='cuda')
    lengths = torch.tensor([30, 11, 1], dtype=torch.int32, device='cuda')
    with torch.no_grad():
        h, residual, caches = x, torch.zeros_like(x), []
        for layer in layers:
            h, residual, kept, state = layer(h, residual, lengths=lengths)
            caches.append([kept, state])
        for b, end in enumerate(lengths.tolist()):
            whole, total = x[b:b + 1], torch.zeros_like(x[b:b + 1])
            for layer in layers:
                whole, total, _, _ = layer(whole, total)
            scale = float(whole.abs().max())
            # float32 products of 32 to 48 terms in other orders, through two layers: some tens of roundings
            assert float((whole[:, :end] - h[b:b + 1, :end]).abs().max()) <= 64 * 2.0 ** -24 * scale * 4
            own = [[k[b:b + 1].clone(), s[b:b + 1].clone()] for k, s in caches]
            for t in range(end, 30):
                one, total = x[b:b + 1, t], torch.zeros(1, 32, device='cuda')
                for layer, (kept, state) in zip(layers, own):
                    one, total, _, _ = layer(one, total, kept, state, one=True)
                assert float((whole[:, t] - one).abs().max()) <= 64 * 2.0 ** -24 * scale * 4


def test_layers_gradients():
    """Training through two layers in float32 against the same layers in float64 with the definitions."""
    layers = [Layer(24, 32, 8, 4, s, F32).cuda() for s in (4, 5)]
    wide = [Layer(24, 32, 8, 4, s, F32).double() for s in (4, 5)]
    g = torch.Generator()
    g.manual_seed(6)
    x = torch.randn(2, 21, 24, generator=g)
    up = torch.randn(2, 21, 24, generator=g)
    ops = (lambda x, w, residual: (ref.norm(x + residual, w), x + residual),
           lambda x, w, b: ref.conv(x, w, b, 'silu'),
           lambda u, delta, A, B, C, **k: ref.scan(u, delta, A, B, C, softplus=True, **k))

    def loss(layers, x, up, ops):
        h, residual = x, torch.zeros_like(x)
        for layer in layers:
            h, residual, _, _ = layer(h, residual, ops=ops)
        return ((h + residual) * up).sum()

    leaf, leaf_wide = x.cuda().requires_grad_(True), x.double().requires_grad_(True)
    params = [p for layer in layers for p in layer.parameters()]
    params_wide = [p for layer in wide for p in layer.parameters()]
    got = torch.autograd.grad(loss(layers, leaf, up.cuda(), None), [leaf] + params)
    want = torch.autograd.grad(loss(wide, leaf_wide, up.double(), ops), [leaf_wide] + params_wide)
    for k, (a, b) in enumerate(zip(got, want)):
        off = float((a.double().cpu() - b).norm() / b.norm())
        # some hundreds of float32 roundings at random along the way from the loss
        assert off <= 64 * 2.0 ** -24 * 4, (k, off)


def test_states_are_kept_only_where_a_backward_pass_can_follow():
    d = ref.scan_inputs(77, 4, 1024, 512, 16, 1, 'bfloat16', gate=True, device='cuda')
    d['A'] = torch.nn.Parameter(d['A'])
    args = [d['u'], d['delta'], d['A'], d['B'], d['C']]

    def most(call):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        out = call(*args, **call_args(d))
        return torch.cuda.max_memory_allocated() - before, out

    for call in (state_space.scan, state_space.scan_torch):         # (the first pass on a stream allocates more)
        call(*args, **call_args(d))
    with torch.no_grad():
        plain, (y, last) = most(state_space.scan)
        unrecorded, (y_2, last_2) = most(state_space.scan_torch)
    recorded, _ = most(state_space.scan_torch)
    assert unrecorded == plain and torch.equal(y, y_2) and torch.equal(last, last_2)
    # a state of float32 per channel and 16 tokens
    assert recorded >= plain + 4 * 1024 * 512 * 16 * 4 // 16


@pytest.mark.parametrize('length', [3, 64, 333])
def test_entries_that_forget_at_once(length):
    """A without bound, or beyond float32 with a factor: the decay is zero for every token, and tokens behind the sequence
    change nothing.  The gradients are those of decays that are zero in all bits, as for A = -1e6."""
    d = ref.scan_inputs(78, 3, length, 4, 9, 2, 'float32', ragged=True, device='cuda')
    d['A'][0, 0] = d['A'][3, 8] = -1e6
    cpu = {k: v.cpu() if isinstance(v, torch.Tensor) else v for k, v in d.items()}
    want_y, want_last, want = ref.scan_expected(cpu)
    d['A'][0, 0], d['A'][3, 8] = float('-inf'), -3.2e38
    y, last = run_scan(d)
    close(y, want_y, F32, 'y', 16)
    close(last, want_last, F32, 'last', 16)
    for name, got, w in zip(ref.SCAN_NAMES, run_grad(d), want):
        close(got, w, F32, 'd_' + name, 64)
    state = d['state'].clone()
    token = {k: d[k][:, 0].contiguous() for k in ('u', 'delta', 'z', 'B', 'C')}
    y = state_space.scan_step(state, token['u'], token['delta'], d['A'], token['B'], token['C'], D=d['D'], z=token['z'],
                              delta_bias=d['delta_bias'], softplus=True)
    first = {k: (v[:, :1] if k in token else v) for k, v in cpu.items()}
    want_y, want_last, _ = ref.scan_expected(dict(first, lengths=None, d_y=cpu['d_y'][:, :1]))
    close(y, want_y[:, 0], F32, 'y of the step', 16)
    close(state, want_last, F32, 'state of the step', 16)


def test_scans_whose_outputs_have_more_than_32_bits_of_bytes():
    """One sequence many times over: every one of the results is the first's."""
    batch, length, channels, n = 1040, 505, 4096, 3
    one = ref.scan_inputs(79, 1, length, channels, n, 1, 'bfloat16', device='cuda')
    every = {k: v.expand((batch,) + v.shape[1:]) if k in ('u', 'delta', 'z', 'B', 'C', 'state', 'd_y', 'd_last') else v
             for k, v in one.items()}
    assert batch * length * channels > 2 ** 31
    y, last = run_scan(every)
    want_y, want_last, want = ref.scan_expected({k: v.cpu() if isinstance(v, torch.Tensor) else v for k, v in one.items()})
    # A token's decay is off by a unit in its last place (2^-23) and its fused multiply-add by half of one: 0.75 times 2^-22 of
    # a state that forgets little in 505 tokens, at random sqrt(505) * 0.75 = 17 together, and 4.5 times that, 76, for the
    # largest of the 12288 states; the gradient that passes through the sequence likewise.
    terms = 80
    close(y[:1], want_y, torch.bfloat16, 'y', terms)
    close(last[:1], want_last, F32, 'last', terms)
    for part in y.split(130) + last.split(130):
        assert torch.equal(part, (y if part.dtype == y.dtype else last)[:1].expand_as(part))
    del y, last
    for name, got, w in zip(ref.SCAN_NAMES, run_grad(every), want):
        if got.shape[0] == batch:
            close(got[:1], w, got.dtype, 'd_' + name, terms)
            for part in got.split(130):
                assert torch.equal(part, got[:1].expand_as(part)), name
