"""
The root-mean-square norm (include/ovl_norm.h) on the GPU against its definition in float64: types, odd sizes and strides,
the residual's sum, the 8-bit output with its scales, gradients, streams and captured graphs.
"""
import math

import pytest
import torch

from opveclib_amd import rms_norm
from tests import recurrent_layer as ref
from tests.recurrent_layer import close

pytestmark = pytest.mark.gpu

F32 = torch.float32
KINDS = [('float32', None, 'float32'), ('float32', 'float32', 'float32'), ('float16', 'float16', 'float16'),
         ('bfloat16', 'float32', 'float32'), ('bfloat16', 'bfloat16', 'float32'), ('float16', None, 'float32')]
# one vector and less, a wavefront's row, four wavefronts', sixteen wavefronts'; whole and with a tail
SIZES = [(1, 1), (3, 7), (5, 128), (300, 200), (9, 1000), (70, 2048), (3, 2049), (17, 4096), (2, 8192), (3, 8200), (2, 20001),
         (1, 32768)]


def inputs(seed, shape, dtype, residual, weight):
    g = torch.Generator(device='cuda')
    g.manual_seed(seed)
    normal = lambda *s: torch.randn(s, generator=g, device='cuda')
    kind = ref.TYPES[dtype]
    x = normal(*shape).to(kind)
    r = None if residual is None else (3 * normal(*shape)).to(ref.TYPES[residual])
    w = (1 + 0.1 * normal(shape[-1])).to(ref.TYPES[weight])
    return x, r, w, normal(*shape).to(kind), None if r is None else normal(*shape).to(r.dtype)


def check_quantized(q, scales, want, group):
    columns = want.shape[-1]
    want_scales = ref.scales_of(want, group)
    close(scales, want_scales, F32, 'scales', 4)
    each = want_scales.repeat_interleave(group or columns, -1)[..., :columns]
    exact = want / each
    # one rounding to four significant bits (half of 2^-9 in the subnormal range), and float32 arithmetic before it
    assert bool(((q.double() - exact).abs() <= exact.abs() * (2.0 ** -4 + 2.0 ** -20) + 2.0 ** -10 + 2.0 ** -20).all())


@pytest.mark.parametrize('kind', KINDS, ids=str)
@pytest.mark.parametrize('size', SIZES, ids=str)
def test_norm_and_its_gradient(size, kind):
    x, r, w, d_y, d_s = inputs(1, size, *kind)
    s = x if r is None else (x.float() + r.float()).to(r.dtype)
    want = ref.norm(s.double(), w.double())
    out = rms_norm.rms_norm(x, w, residual=r)
    y = out if r is None else out[0]
    close(y, want, x.dtype, 'y', 4)
    if r is not None:
        assert torch.equal(out[1], s)
    for group in (None, 128):
        out = rms_norm.rms_norm_quantized(x, w, residual=r, group=group)
        check_quantized(out[0], out[1], want, group)
        if r is not None:
            assert torch.equal(out[2], s)
    leaf, w_leaf = ref.wide(s, True), ref.wide(w, True)
    outs, ups = [ref.norm(leaf, w_leaf)], [d_y.double()]
    if d_s is not None:
        outs, ups = outs + [leaf * 1], ups + [d_s.double()]
    want_s, want_w = torch.autograd.grad(outs, [leaf, w_leaf], ups)
    d_x, d_total, d_w = rms_norm.rms_norm_grad(s, w, d_y, d_s, both=True)
    terms = 16 + math.sqrt(size[0])          # roundings of a sum over the rows add up at random
    scale = ref.norm_gradient_scale(s, w, d_y, d_s)
    close(d_x, want_s, x.dtype, 'd_x', 16, scale)
    close(d_total, want_s, s.dtype, 'd_s', 16, scale)
    close(d_w, want_w, w.dtype, 'd_weight', terms)


def test_more_axes_strides_and_transposed_rows():
    x, r, w, d_y, d_s = inputs(2, (4, 6, 96), 'bfloat16', 'float32', 'float32')
    y, s = rms_norm.rms_norm(x, w, residual=r)
    flat_y, flat_s = rms_norm.rms_norm(x.view(24, 96), w, residual=r.view(24, 96))
    assert torch.equal(y.view(24, 96), flat_y) and torch.equal(s.view(24, 96), flat_s)
    wide = torch.full((24, 200), float('nan'), device='cuda').bfloat16()
    wide[:, 3:99] = x.view(24, 96)
    moved_y, moved_s = rms_norm.rms_norm(wide[:, 3:99], w, residual=r.view(24, 96).t().contiguous().t())
    assert torch.equal(flat_y, moved_y) and torch.equal(flat_s, moved_s)
    same = rms_norm.rms_norm(x.view(24, 96)[:1].expand(24, 96), w)
    assert torch.equal(same, flat_like(x, w))
    got = rms_norm.rms_norm_grad(s.transpose(0, 1), w, d_y.transpose(0, 1), d_s.transpose(0, 1))
    want = rms_norm.rms_norm_grad(s.transpose(0, 1).contiguous(), w, d_y.transpose(0, 1).contiguous(), d_s.transpose(0, 1).contiguous())
    assert torch.equal(got[0], want[0]) and torch.equal(got[2], want[2])


def flat_like(x, w):
    return rms_norm.rms_norm(x.view(-1, x.shape[-1])[:1], w).expand(24, 96)


def test_rows_of_zeros_and_rows_that_are_not_finite():
    x = torch.randn(6, 300, device='cuda')
    x[1] = 0
    x[2, 17] = float('nan')
    x[3, 5] = float('inf')
    x[4] *= 1e-22
    w = torch.ones(300, device='cuda')
    y = rms_norm.rms_norm(x, w)
    assert not y[1].any() and torch.isnan(y[2]).all() and torch.isnan(y[3, 5]) and not y[3, 6:].any()
    for group, width in ((None, 1), (128, 3)):
        q, scales = rms_norm.rms_norm_quantized(x, w, group=group)
        assert scales.shape == (6, width)
        assert bool((scales[1] == 1).all()) and not q[1].float().any()
        assert torch.isnan(q[2].float()).all() and torch.isnan(q[3].float()[5]) and not q[3].float()[6:].any()
        good = [0, 4, 5]
        check_quantized(q[good], scales[good], ref.norm(x[good].double(), w.double()), group)
    # the largest value of a row becomes the largest of the format
    assert bool((rms_norm.rms_norm_quantized(x, w)[0].float().abs().amax(1)[[0, 5]] == 448).all())


@pytest.mark.parametrize('group', [None, 128])
def test_scales_stay_normal_numbers(group):
    """Results so small that a 448th of them is subnormal, whose reciprocal would not be finite."""
    g = torch.Generator(device='cuda')
    g.manual_seed(5)
    x = torch.randn(3, 256, generator=g, device='cuda')
    x[0, 3] = 0
    w = torch.full((256,), 2.0 ** -124, device='cuda')
    q, scales = rms_norm.rms_norm_quantized(x, w, group=group)
    assert bool((scales == 2.0 ** -126).all()) and q[0, 3].item() == 0
    exact = ref.norm(x.double(), w.double()) * 2.0 ** 126
    # as in check_quantized; a result below 2^-126 may come out of float32 arithmetic as zero: up to 1 of the 448 steps
    off = (q.double() - exact).abs()
    assert bool(((off <= exact.abs() * (2.0 ** -4 + 2.0 ** -20) + 2.0 ** -10 + 2.0 ** -20) | ((q.float() == 0) & (exact.abs() < 1))).all())


def test_autograd_function():
    for kind in KINDS:
        x, r, w, d_y, d_s = inputs(3, (21, 260), *kind)
        leaves = [t.clone().requires_grad_(True) for t in (x, r, w) if t is not None]
        if r is None:
            y = rms_norm.rms_norm_torch(leaves[0], leaves[1])
            got = torch.autograd.grad(y, leaves, d_y)
            want = rms_norm.rms_norm_grad(x, w, d_y)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[2])
            continue
        y, s = rms_norm.rms_norm_torch(leaves[0], leaves[2], residual=leaves[1])
        got = torch.autograd.grad((y, s), leaves, (d_y, d_s), retain_graph=True)
        want = rms_norm.rms_norm_grad(s.detach(), w, d_y, d_s, both=True)
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        got = torch.autograd.grad(y, leaves, d_y, retain_graph=True)          # the sum is not used any further
        assert torch.equal(got[0], rms_norm.rms_norm_grad(s.detach(), w, d_y)[0])
        got = torch.autograd.grad(s, leaves, d_s)                             # nor the norm
        assert torch.equal(got[1], d_s) and not got[2].any()


def test_gradient_against_differences():
    x, r, w, d_y, d_s = inputs(4, (7, 50), 'float32', 'float32', 'float32')
    y, s = rms_norm.rms_norm(x, w, residual=r)
    d_x, _, d_w = rms_norm.rms_norm_grad(s, w, d_y, d_s)

    def loss(x, w):
        y, s = rms_norm.rms_norm(x, w, residual=r)
        return float((y.double() * d_y.double()).sum() + (s.double() * d_s.double()).sum())

    way, way_w = torch.randn_like(x) * 1e-2, torch.randn_like(w) * 1e-2
    for slope, formula in (((loss(x + way, w) - loss(x - way, w)) / 2, d_x.double() * way.double()),
                           ((loss(x, w + way_w) - loss(x, w - way_w)) / 2, d_w.double() * way_w.double())):
        # the step leaves a third-order term of about its square, 1e-4
        assert abs(slope - float(formula.sum())) <= 1e-3 * float(formula.abs().sum()) + 1e-5


def test_arguments_that_do_not_fit_are_refused():
    x, r, w, d_y, d_s = inputs(5, (4, 32), 'bfloat16', 'bfloat16', 'float32')
    for args, more in (((x.double(), w), {}), ((x, w.half()), {}), ((x, w[:31]), {}), ((x, w.cpu()), {}), ((x, w), {'residual': r[:3]}),
                       ((x, w), {'residual': r.half()}), ((x, w), {'residual': r.cpu()}), ((x[:, :0], w[:0]), {}),
                       ((torch.zeros(2, 32769, device='cuda'), torch.zeros(32769, device='cuda')), {}), ((x, None), {}),
                       ((torch.tensor(1.0, device='cuda'), w), {})):
        for call in (rms_norm.rms_norm, rms_norm.rms_norm_quantized):
            with pytest.raises(TypeError):
                call(*args, **more)
    for group in (0, 64, 256):
        with pytest.raises(ValueError):
            rms_norm.rms_norm_quantized(x, w, group=group)
    for args in ((r, w, d_y[:3]), (r.half(), w, d_y), (r, w, d_y, d_s.float()), (r, w, d_y, d_s[:2]), (r, w, None)):
        with pytest.raises(TypeError):
            rms_norm.rms_norm_grad(*args)
    none = torch.empty(0, 32, device='cuda')
    assert rms_norm.rms_norm(none, w).shape == (0, 32)
    assert rms_norm.rms_norm_quantized(none, w, group=128)[1].shape == (0, 1)
    assert not rms_norm.rms_norm_grad(none, w, none)[2].any()


def test_streams_and_captured_graphs():
    x, r, w, d_y, d_s = inputs(6, (33, 4096), 'bfloat16', 'float32', 'float32')

    def work(x, r):
        y, s = rms_norm.rms_norm(x, w, residual=r)
        return (y, s) + rms_norm.rms_norm_quantized(x, w, residual=r, group=128) + rms_norm.rms_norm_grad(s, w, d_y, d_s, both=True)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = work(x * 1, r * 1)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(other, work(x, r)):
        assert torch.equal(a.float(), b.float())
    x_in, r_in = x.clone(), r.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work(x_in, r_in)
    for k in range(4):
        x_in.copy_(torch.randn_like(x))
        graph.replay()
        want = work(x_in.clone(), r)
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a.float(), b.float())


def test_matrices_beyond_32_bits_of_bytes():
    rows, columns = 2 ** 31 // 16384 + 3, 16384
    x = torch.randn(64, columns, device='cuda').half().repeat(rows // 64 + 1, 1)[:rows]
    w = torch.randn(columns, device='cuda')
    y = rms_norm.rms_norm(x, w)
    q, scales = rms_norm.rms_norm_quantized(x, w)
    assert torch.equal(y[-64:], rms_norm.rms_norm(x[-64:].contiguous(), w))
    tail, tail_scales = rms_norm.rms_norm_quantized(x[-64:].contiguous(), w)
    assert torch.equal(q[-64:].view(torch.uint8), tail.view(torch.uint8)) and torch.equal(scales[-64:], tail_scales)
    d_x, _, _ = rms_norm.rms_norm_grad(x, w, y)
    assert torch.equal(d_x[-64:], rms_norm.rms_norm_grad(x[-64:].contiguous(), w, y[-64:].contiguous())[0])


@pytest.mark.parametrize('rows,columns', [(3000, 100), (700, 1000), (300, 4096), (40, 20001)])
def test_codes_and_scales_are_those_of_the_results(rows, columns):
    """Bit for bit: the results of rms_norm in float32 divided on the CPU, for both kinds of scales."""
    x, _, _, _, _ = inputs(7, (rows, columns), 'float32', None, 'float32')
    w = torch.randn(columns, device='cuda')
    y = rms_norm.rms_norm(x, w)
    for group in (None, 128):
        q, scales = rms_norm.rms_norm_quantized(x, w, group=group)
        want, want_scales = ref.quantized(y, group)
        assert torch.equal(scales.cpu(), want_scales)
        assert torch.equal(q.cpu().view(torch.uint8), want.view(torch.uint8))


def test_zeros_keep_their_sign_in_8_bits():
    x = torch.randn(500, 64, device='cuda')
    x[:, ::3] = 0
    x = torch.where(torch.rand_like(x) < 0.5, -x, x)
    w = 0.1 + torch.rand(64, device='cuda')
    for group in (None, 128):
        q, _ = rms_norm.rms_norm_quantized(x, w, group=group)
        assert torch.equal(q.view(torch.uint8) >= 128, torch.signbit(x))


def test_middles_of_two_8_bit_numbers_go_to_the_even_one():
    weights, t = ref.middles(list(range(1, 200, 2)) + [1021, 65537, 262657])
    want = t.float().to(torch.float8_e4m3fn).view(torch.uint8).cuda()
    ones = torch.ones(2, 128, device='cuda')
    for row in weights:
        for group in (None, 128):
            q, scales = rms_norm.rms_norm_quantized(ones, row.cuda(), eps=0.0, group=group)
            assert bool((scales == row[0].item() / 448).all())
            assert torch.equal(q.view(torch.uint8), want.expand(2, 128))


def test_more_rows_than_one_launch_takes():
    """2^26 rows of 64 work items."""
    rows, columns = 2 ** 26 + 5, 8
    x = torch.randn(1024, columns, device='cuda').bfloat16().repeat(rows // 1024 + 1, 1)[:rows]
    r = torch.randn(rows, columns, device='cuda').bfloat16()
    w = torch.randn(columns, device='cuda')
    y, s = rms_norm.rms_norm(x, w, residual=r)
    d_x, _, d_w = rms_norm.rms_norm_grad(s, w, x)
    for part in (slice(0, 300), slice(2 ** 26 - 8, 2 ** 26 + 5), slice(12345678, 12345700)):
        want_y, want_s = rms_norm.rms_norm(x[part].clone(), w, residual=r[part].clone())
        assert torch.equal(y[part], want_y) and torch.equal(s[part], want_s)
        assert torch.equal(d_x[part], rms_norm.rms_norm_grad(s[part].clone(), w, x[part].clone())[0])
    assert torch.equal(s, x + r)
    assert torch.isfinite(y).all() and torch.isfinite(d_w).all()
    for group in (None, 128):
        q, scales = rms_norm.rms_norm_quantized(s, w, group=group)
        want, want_scales = ref.quantized(rms_norm.rms_norm(s[-4000:].float(), w), group)
        assert torch.equal(scales[-4000:].cpu(), want_scales)
        assert torch.equal(q[-4000:].cpu().view(torch.uint8), want.view(torch.uint8))


def test_parts_of_a_projection_are_used_where_they_are():
    """Halves of [batch, length, 2 columns]: no copies, neither of the rows nor of their gradients."""
    batch, length, columns = 4, 256, 1000
    x, r, w, d_y, d_s = inputs(9, (batch, length, 2 * columns), 'bfloat16', 'float32', 'float32')
    w = w[:columns].contiguous()
    halves = [t[..., columns:] for t in (x, r, d_y, d_s)]
    dense = [t.contiguous() for t in halves]

    def work(x, r, d_y, d_s):
        y, s = rms_norm.rms_norm(x, w, residual=r)
        return (y, s) + rms_norm.rms_norm_quantized(x, w, residual=r, group=128) + rms_norm.rms_norm_grad(r, w, d_y, d_s, both=True)

    most = []
    for tensors in (dense, halves):
        got = work(*tensors)
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        again = work(*tensors)
        most.append(torch.cuda.max_memory_allocated() - before)
        if tensors is dense:
            want = got
    assert most[0] == most[1]
    for a, b, c in zip(want, got, again):
        assert torch.equal(a.float(), b.float()) and torch.equal(a.float(), c.float())


@pytest.mark.parametrize('power', [-115, 108])
def test_middles_of_very_small_and_large_results_go_to_the_even_one(power):
    weights, t = ref.middles(list(range(1, 200, 2)) + [509, 511])
    want = t.float().to(torch.float8_e4m3fn).view(torch.uint8).cuda()
    ones = torch.ones(2, 128, device='cuda')
    for row in weights * 2.0 ** power:
        for group in (None, 128):
            q, scales = rms_norm.rms_norm_quantized(ones, row.cuda(), eps=0.0, group=group)
            assert bool((scales == row[0].item() / 448).all())
            assert torch.equal(q.view(torch.uint8), want.expand(2, 128))
