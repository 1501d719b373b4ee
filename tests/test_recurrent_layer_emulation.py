"""
The state space and norm kernels on the CPU: csrc/ovl_ssm_scan.hip, ovl_ssm_conv.hip and ovl_norm.hip compiled as plain C++
with one host thread per GPU thread, run under AddressSanitizer on buffers of exactly the tensors' sizes, and compared
with the definitions in float64.  This checks index arithmetic, tails, barriers, lane moves, LDS layouts and that no access
leaves its tensor before anything runs on a GPU.
"""
import hashlib
import os

import numpy as np
import pytest
import torch

from opveclib_amd import local
from tests import host_emulation, recurrent_layer as ref
from tests.recurrent_layer import close

pytestmark = pytest.mark.skipif(not os.path.exists(host_emulation.CLANG), reason='needs the ROCm clang++ as host compiler')

NUMPY = {'float32': np.float32, 'float16': np.uint16, 'bfloat16': np.uint16}


@pytest.fixture(scope='module')
def program():
    parts = []
    for name in ('ovl_ssm_scan.hip', 'ovl_ssm_conv.hip', 'ovl_norm.hip'):
        with open(os.path.join(local.csrc_directory, name)) as f:
            parts.append(f.read())
    with open(os.path.join(host_emulation.SHIM, 'recurrent_layer_adapters.cpp')) as f:
        parts.append(f.read())
    headers = ''
    for path in (os.path.join(host_emulation.SHIM, 'ovl_lane.h'), os.path.join(local.csrc_directory, 'ovl_ssm_host.h')):
        with open(path) as f:
            headers += f.read()
    # the name of the program depends on the sources' text: the stand-in header is part of it
    parts[-1] += '\n// one stack per thread ' + hashlib.sha224(headers.encode('utf-8')).hexdigest() + '\n'
    include = os.path.normpath(os.path.join(local.csrc_directory, '..', '..', 'include'))
    # (one stack per thread: the sanitizer's second ones, for returned frames, exhaust the mappings a process may have)
    return host_emulation.build_source(parts, 'emu_recurrent_layer',
                                       ['-I' + include, '-fsanitize-address-use-after-return=never'])


def to_numpy(t):
    if t is None:
        return np.zeros(0, np.float32)
    t = t.detach().contiguous()
    if t.dtype in (torch.float16, torch.bfloat16):
        return t.view(torch.int16).numpy().view(np.uint16)
    return t.numpy()


def from_numpy(a, dtype):
    if dtype in (torch.float16, torch.bfloat16):
        return torch.from_numpy(a.view(np.int16).copy()).view(dtype)
    return torch.from_numpy(a.copy())


def run(program, settings, inputs, outputs):
    """inputs: tensors or None; outputs: (shape, torch dtype), an empty shape tuple entry for an absent one."""
    arrays = [np.array(settings, np.int64)] + [to_numpy(t) for t in inputs]
    in_types = [(0, a.dtype, a.shape) for a in arrays]
    out_types = [(0, {2: np.uint16, 4: np.float32, 1: np.uint8}[torch.empty(0, dtype=d).element_size()], s) for s, d in outputs]
    got = host_emulation.run_program(program, arrays, in_types, out_types)
    return [from_numpy(a, d) if d not in (torch.float8_e4m3fn,) else torch.from_numpy(a.copy()).view(d)
            for a, (_, d) in zip(got, outputs)]


def padded(t, more):
    """The sequence tensor inside rows that are `more` channels longer (filled with NaN)."""
    if t is None:
        return None
    wide = torch.full(t.shape[:2] + (t.shape[2] + more,), float('nan'), dtype=t.dtype)
    wide[:, :, :t.shape[2]] = t
    return wide


SCANS = [
    # batch, length, channels, state, groups, type, gate, ragged, entering, softplus
    (1, 1, 1, 1, 1, 'float32', False, False, False, True),
    (2, 19, 70, 16, 1, 'bfloat16', True, False, True, True),
    (3, 33, 10, 5, 2, 'float32', True, True, True, False),
    (2, 21, 6, 20, 3, 'float16', False, True, False, True),
    (1, 17, 3, 40, 1, 'float32', True, False, True, True),
    # long enough for a few channels to be split into chunks; the second with sequences that end before the last chunk
    (1, 230, 5, 16, 1, 'float32', True, False, True, True),
    (3, 209, 4, 8, 2, 'bfloat16', True, True, False, True),
]


def scan_settings(case, kind, more):
    batch, length, channels, n, groups, dtype, _, _, _, softplus = case
    wide = channels + more
    return [kind, batch, length, channels, n, groups, ref.CODES[dtype], int(softplus), length * wide, wide,
            length * groups * n, groups * n, n]


def scan_case(case, seed):
    batch, length, channels, n, groups, dtype, gate, ragged, entering, softplus = case
    return ref.scan_inputs(seed, batch, length, channels, n, groups, dtype, gate, ragged, entering, softplus=softplus)


@pytest.mark.parametrize('case', SCANS, ids=str)
def test_scan_forward(program, case):
    batch, length, channels, n, groups, dtype = case[:6]
    d = scan_case(case, 1)
    more = 3
    ins = [padded(d['u'], more), padded(d['delta'], more), padded(d['z'], more), d['B'], d['C'], d['A'], d['D'],
           d['delta_bias'], d['state'], d['lengths']]
    kind = ref.TYPES[dtype]
    y, last, _ = run(program, scan_settings(case, 0, more), ins,
                     [((batch, length, channels), kind), ((batch, channels, n), torch.float32), ((0,), torch.float32)])
    want_y, want_last, _ = ref.scan_expected(d)
    close(y, want_y, kind, 'y', 16)
    close(last, want_last, torch.float32, 'last', 16)


@pytest.mark.parametrize('case', SCANS, ids=str)
def test_scan_backward(program, case):
    batch, length, channels, n, groups, dtype = case[:6]
    d = scan_case(case, 2)
    more = 3
    ins = [padded(d['u'], more), padded(d['delta'], more), padded(d['z'], more), d['B'], d['C'], d['A'], d['D'],
           d['delta_bias'], d['state'], d['lengths'], padded(d['d_y'], more), d['d_last']]
    kind, f32 = ref.TYPES[dtype], torch.float32
    seq, vec, none = ((batch, length, channels), kind), ((batch, length, groups, n), kind), ((0,), f32)
    outs = [seq, seq, ((channels, n), f32), vec, vec, ((channels,), f32), seq if d['z'] is not None else ((0,), kind),
            ((channels,), f32), ((batch, channels, n), f32) if d['state'] is not None else none]
    got = run(program, scan_settings(case, 1, more), ins, outs)
    _, _, want = ref.scan_expected(d)
    for name, g, w in zip(ref.SCAN_NAMES, got, want):
        if w is not None:
            close(g, w, kind if name in ('u', 'delta', 'z', 'B', 'C') else f32, 'd_' + name, 32)


def forget_at_once(A):
    """Some decays exp(dt A) that are zero whatever the time step: A without bound, or beyond float32 with a factor."""
    A[0, 0], A[-1, -1] = float('-inf'), -3.2e38
    return A


@pytest.mark.parametrize('case', [(1, 13, 3, 5, 1, 'float32', True, False, True, True),
                                  (3, 24, 2, 16, 1, 'float32', False, True, True, False),
                                  (2, 230, 2, 8, 1, 'bfloat16', False, True, True, True)], ids=str)
def test_scan_forward_with_entries_that_forget_at_once(program, case):
    """Tokens behind the sequence change no state, also where nothing decays for them and everything for others."""
    batch, length, channels, n, groups, dtype = case[:6]
    d = scan_case(case, 9)
    forget_at_once(d['A'])
    ins = [d['u'], d['delta'], d['z'], d['B'], d['C'], d['A'], d['D'], d['delta_bias'], d['state'], d['lengths']]
    kind = ref.TYPES[dtype]
    y, last, _ = run(program, scan_settings(case, 0, 0), ins,
                     [((batch, length, channels), kind), ((batch, channels, n), torch.float32), ((0,), torch.float32)])
    want_y, want_last, _ = ref.scan_expected(d)
    close(y, want_y, kind, 'y', 16)
    close(last, want_last, torch.float32, 'last', 16)


def test_scan_backward_with_entries_that_forget_at_once(program):
    """Their gradients are those of decays that are zero in all bits (for A = -1e6: every time step is 1e-4 and more)."""
    case = (2, 21, 3, 5, 1, 'float32', True, True, True, True)
    batch, length, channels, n, groups, dtype = case[:6]
    d = scan_case(case, 10)
    _, _, want = ref.scan_expected(dict(d, A=torch.where(forget_at_once(d['A'].clone()) > -1e30, d['A'], -1e6)))
    forget_at_once(d['A'])
    ins = [d['u'], d['delta'], d['z'], d['B'], d['C'], d['A'], d['D'], d['delta_bias'], d['state'], d['lengths'], d['d_y'], d['d_last']]
    f32 = torch.float32
    outs = [((batch, length, channels), f32), ((batch, length, channels), f32), ((channels, n), f32), ((batch, length, groups, n), f32),
            ((batch, length, groups, n), f32), ((channels,), f32), ((batch, length, channels), f32), ((channels,), f32),
            ((batch, channels, n), f32)]
    for name, g, w in zip(ref.SCAN_NAMES, run(program, scan_settings(case, 1, 0), ins, outs), want):
        close(g, w, f32, 'd_' + name, 32)


@pytest.mark.parametrize('case', [(1, 1, 1, 1, 1, 'float32', False, False, True, True),
                                  (3, 1, 70, 16, 2, 'bfloat16', True, False, True, True),
                                  (2, 1, 21, 30, 3, 'float16', True, False, True, False),
                                  (2, 1, 9, 64, 1, 'float32', True, False, True, True)], ids=str)
def test_scan_step(program, case):
    batch, _, channels, n, groups, dtype = case[:6]
    d = scan_case(case, 3)
    ins = [d['u'], d['delta'], d['z'], d['B'], d['C'], d['A'], d['D'], d['delta_bias'], d['state'], None]
    kind = ref.TYPES[dtype]
    y, state = run(program, scan_settings(case, 2, 0), ins, [((batch, 1, channels), kind), ((batch, channels, n), torch.float32)])
    want_y, want_state, _ = ref.scan_expected(d)
    close(y, want_y, kind, 'y', 16)
    close(state, want_state, torch.float32, 'state', 16)


CONVS = [
    # batch, length, channels, width, type, silu, ragged, entering
    (1, 1, 1, 1, 'float32', False, False, False),
    (2, 19, 24, 4, 'bfloat16', True, False, True),
    (3, 37, 10, 3, 'float16', True, True, True),
    (2, 2, 7, 4, 'float32', False, True, True),
    (2, 70, 8, 2, 'float32', True, True, False),
    (1, 5, 600, 4, 'bfloat16', True, False, False),
]


@pytest.mark.parametrize('more', [0, 3])
@pytest.mark.parametrize('case', CONVS, ids=str)
def test_conv(program, case, more):
    batch, length, channels, width, dtype, silu, ragged, entering = case
    kind, f32 = ref.TYPES[dtype], torch.float32
    d = ref.conv_inputs(4, batch, length, channels, width, dtype, ragged, entering)
    wide = channels + more
    settings = [batch, length, channels, width, ref.CODES[dtype], int(silu), length * wide, wide]
    ins = [padded(d['x'], more), d['weight'], d['bias'], d['state'], d['lengths']]
    kept = ((batch, width - 1, channels), kind)
    want_y, want_last, want = ref.conv_expected(d, silu)
    y, last = run(program, [3] + settings, ins, [((batch, length, channels), kind), kept])
    close(y, want_y, kind, 'y', 4)
    assert torch.equal(last.double(), want_last)
    got = run(program, [4] + settings, ins + [padded(d['d_y'], more), d['d_last']],
              [((batch, length, channels), kind), ((channels, width), f32), ((channels,), f32),
               kept if entering else ((0,), kind)])
    for name, g, w in zip(ref.CONV_NAMES, got, want):
        if w is not None:
            close(g, w, kind if name in ('x', 'state') else f32, 'd_' + name, 16)


@pytest.mark.parametrize('case', [(3, 1, 24, 4, 'bfloat16', True), (2, 1, 7, 2, 'float32', False), (1, 1, 5, 1, 'float16', True)], ids=str)
def test_conv_step(program, case):
    batch, _, channels, width, dtype, silu = case
    kind = ref.TYPES[dtype]
    d = ref.conv_inputs(5, batch, 1, channels, width, dtype)
    y, state = run(program, [5, batch, 1, channels, width, ref.CODES[dtype], int(silu), channels, channels],
                   [d['x'], d['weight'], d['bias'], d['state'], None], [((batch, 1, channels), kind), ((batch, width - 1, channels), kind)])
    want_y, want_last, _ = ref.conv_expected(d, silu)
    close(y, want_y, kind, 'y', 4)
    assert torch.equal(state.double(), want_last)


@pytest.mark.parametrize('channels', [16, 7])
def test_conv_with_weights_of_the_sequences_type(program, channels):
    d = ref.conv_inputs(6, 2, 5, channels, 4, 'bfloat16')
    narrow = [d[n].bfloat16() for n in ('weight', 'bias')]
    results = []
    for own, (w, b) in enumerate(([t.float() for t in narrow], narrow)):
        results.append(run(program, [3, 2, 5, channels, 4, ref.CODES['bfloat16'], 1, 5 * channels, channels, own],
                           [d['x'], w, b, d['state'], None],
                           [((2, 5, channels), torch.bfloat16), ((2, 3, channels), torch.bfloat16)]))
    for wide, own in zip(*results):
        assert torch.equal(wide, own)


NORMS = [
    # rows, columns, type, residual's type or None, weight's type
    (1, 1, 'float32', None, 'float32'),
    (5, 200, 'bfloat16', 'bfloat16', 'float32'),
    (6, 515, 'float16', 'float32', 'float16'),
    (2, 2052, 'float32', 'float32', 'float32'),
    (2, 9001, 'bfloat16', 'float32', 'bfloat16'),
]


@pytest.mark.parametrize('case', NORMS, ids=str)
def test_norm(program, case):
    rows, columns, dtype, residual, weight_type = case
    g = torch.Generator()
    g.manual_seed(6)
    kind, f32 = ref.TYPES[dtype], torch.float32
    r_kind = kind if residual is None else ref.TYPES[residual]
    more = 5

    def matrix(kind):
        wide = torch.full((rows, columns + more), float('nan'), dtype=kind)
        wide[:, :columns] = torch.randn(rows, columns, generator=g).to(kind)
        return wide, wide[:, :columns]

    x_all, x = matrix(kind)
    r_all, r = matrix(r_kind) if residual is not None else (None, None)
    weight = (1 + 0.1 * torch.randn(columns, generator=g)).to(ref.TYPES[weight_type])
    settings = [rows, columns, ref.CODES[dtype], ref.CODES[residual or dtype], ref.CODES[weight_type], columns + more, columns + more]
    summed = x if r is None else (x.float() + r.float()).to(r_kind)
    s_out = ((rows, columns), r_kind) if residual is not None else ((0,), r_kind)
    want = ref.norm(summed.double(), weight.double())
    y, s = run(program, [6] + settings, [x_all, r_all, weight], [((rows, columns), kind), s_out])
    close(y, want, kind, 'y', 4)
    if residual is not None:
        assert torch.equal(s, summed)
    for group in (0, 128):
        scale_shape = (rows, -(-columns // 128) if group else 1)
        q, scales, s = run(program, [7] + settings + [group], [x_all, r_all, weight],
                           [((rows, columns), torch.float8_e4m3fn), (scale_shape, f32), s_out])
        want_scales = ref.scales_of(want, group or None)
        close(scales, want_scales, f32, 'scales', 4)
        each = want_scales.repeat_interleave(group or columns, 1)[:, :columns]
        # one rounding to four significant bits (2^-10 in the subnormal range), and float32 arithmetic before it
        assert bool(((q.double() - want / each).abs() <= (want / each).abs() * (2.0 ** -4 + 2.0 ** -20) + 2.0 ** -10).all())
    # gradient: the dense sum in front
    dy_all, dy = matrix(kind)
    ds = torch.randn(rows, columns, generator=g).to(r_kind)
    leaf, w_leaf = ref.wide(summed, True), ref.wide(weight, True)
    want = torch.autograd.grad([ref.norm(leaf, w_leaf), leaf * 1], [leaf, w_leaf], [dy.double(), ds.double()])
    settings[5] = columns
    d_x, d_r, d_w = run(program, [8] + settings, [summed.contiguous(), dy_all, weight, ds],
                        [((rows, columns), kind), ((rows, columns), r_kind), ((columns,), weight.dtype)])
    close(d_x, want[0], kind, 'd_x', 16)
    close(d_r, want[0], r_kind, 'd_residual', 16)
    close(d_w, want[1], weight.dtype, 'd_weight', 16)


@pytest.mark.parametrize('rows,columns', [(12, 120), (2, 515), (1, 2052)])
def test_norm_to_8_bits_divides_its_own_results(program, rows, columns):
    """Codes and scales are those of the float32 results, bit for bit, and rows of up to 128 columns get the same from both
    forms."""
    g = torch.Generator()
    g.manual_seed(7)
    x = torch.randn(rows, columns, generator=g)
    weight = torch.randn(columns, generator=g)
    settings = [rows, columns, 2, 2, 2, columns, columns]
    none = ((0,), torch.float32)
    y, _ = run(program, [6] + settings, [x, None, weight], [((rows, columns), torch.float32), none])
    for group in (0, 128):
        q, scales, _ = run(program, [7] + settings + [group], [x, None, weight],
                           [((rows, columns), torch.float8_e4m3fn), ((rows, -(-columns // 128) if group else 1), torch.float32), none])
        want, want_scales = ref.quantized(y, group or None)
        assert torch.equal(scales, want_scales)
        assert torch.equal(q.view(torch.uint8), want.view(torch.uint8))


def test_norm_to_8_bits_keeps_the_sign_of_zeros(program):
    x = torch.tensor([[0.0, -0.0, 3.0, -2.0] * 4, [-0.0, 0.0, -1.7, 2.0] * 4])
    for top in (3.0, 1.9, 1.1, 0.7):
        for group in (0, 128):
            q, _, _ = run(program, [7, 2, 16, 2, 2, 2, 16, 16, group], [x, None, torch.full((16,), top)],
                          [((2, 16), torch.float8_e4m3fn), ((2, 1), torch.float32), ((0,), torch.float32)])
            assert torch.equal(q.view(torch.uint8) >= 128, torch.signbit(x))


def test_norm_to_8_bits_sends_middles_to_the_even_number(program):
    weights, t = ref.middles([1, 3, 5, 7, 11, 49, 1021, 65537, 262657])
    ones = torch.ones(1, 128)
    for row in weights:
        for group in (0, 128):
            q, scales, _ = run(program, [7, 1, 128, 2, 2, 2, 128, 128, group, 1], [ones, None, row],
                               [((1, 128), torch.float8_e4m3fn), ((1, 1), torch.float32), ((0,), torch.float32)])
            assert scales.item() == row[0].item() / 448
            assert torch.equal(q.view(torch.uint8)[0], t.float().to(torch.float8_e4m3fn).view(torch.uint8))


@pytest.mark.parametrize('rows,columns', [(70, 24), (9, 2060), (5, 9001)])
def test_norm_in_several_launches(program, rows, columns):
    """The emulated device takes 2048 work items in a launch: 32, 8 and 2 rows of these."""
    g = torch.Generator()
    g.manual_seed(8)
    x, r = torch.randn(rows, columns, generator=g).bfloat16(), torch.randn(rows, columns + 3, generator=g)
    weight = torch.randn(columns, generator=g).bfloat16()
    b16, f32 = torch.bfloat16, torch.float32
    s = x.float() + r[:, :columns]
    want = ref.norm(s.double(), weight.double())
    settings = [rows, columns, ref.CODES['bfloat16'], ref.CODES['float32'], ref.CODES['bfloat16'], columns, columns + 3]
    y, summed = run(program, [6] + settings, [x, r, weight], [((rows, columns), b16), ((rows, columns), f32)])
    close(y, want, b16, 'y', 4)
    assert torch.equal(summed, s)
    for group in (0, 128):
        scale_shape = (rows, -(-columns // 128) if group else 1)
        q, scales, summed = run(program, [7] + settings + [group], [x, r, weight],
                                [((rows, columns), torch.float8_e4m3fn), (scale_shape, f32), ((rows, columns), f32)])
        assert torch.equal(summed, s)
        want_scales = ref.scales_of(want, group or None)
        close(scales, want_scales, f32, 'scales', 4)
        exact = want / want_scales.repeat_interleave(group or columns, 1)[:, :columns]
        # one rounding to four significant bits (2^-10 in the subnormal range), and float32 arithmetic before it
        assert bool(((q.double() - exact).abs() <= exact.abs() * (2.0 ** -4 + 2.0 ** -20) + 2.0 ** -10).all())


@pytest.mark.parametrize('power', [-115, 108])
def test_norm_to_8_bits_sends_middles_of_very_small_and_large_results_to_the_even_number(program, power):
    weights, t = ref.middles([1, 3, 7, 49, 511])
    ones = torch.ones(1, 128)
    for row in weights * 2.0 ** power:
        for group in (0, 128):
            q, scales, _ = run(program, [7, 1, 128, 2, 2, 2, 128, 128, group, 1], [ones, None, row],
                               [((1, 128), torch.float8_e4m3fn), ((1, 1), torch.float32), ((0,), torch.float32)])
            assert scales.item() == row[0].item() / 448
            assert torch.equal(q.view(torch.uint8)[0], t.float().to(torch.float8_e4m3fn).view(torch.uint8))
