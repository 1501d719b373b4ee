"""The state space and norm libraries without a GPU: headers and bindings agree, and bad arguments are refused, by the C
entry points before any GPU work and by the Python functions with the errors the other hand-written kernels use."""
import ctypes
import os
import re

import pytest
import torch

from opveclib_amd import rms_norm, state_space

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
EINVAL = 6


def declared_functions(header):
    text = open(os.path.join(ROOT, 'include', header)).read()
    text = re.sub(r'/\*.*?\*/', '', text, flags=re.S)
    return sorted(set(re.findall(r'\b(ovl_[a-z_0-9]+)\s*\(', text)))


@pytest.fixture(scope='module')
def libraries():
    for module in (state_space, rms_norm):
        if not os.path.exists(module.library_path):
            module.build()
    return state_space.library(), rms_norm.library()


def test_headers_and_bindings_agree(libraries):
    for header, module in (('ovl_ssm.h', state_space), ('ovl_norm.h', rms_norm)):
        assert declared_functions(header) == sorted(module.EXPORTED_SYMBOLS)
        raw = ctypes.CDLL(module.library_path)
        for name in declared_functions(header):
            assert hasattr(raw, name), name


def test_missing_libraries_are_loud_errors(monkeypatch):
    for module in (state_space, rms_norm):
        monkeypatch.setattr(module, '_lib', None)
        monkeypatch.setattr(module, 'library_path', '/nonexistent/lib.so')
        with pytest.raises(RuntimeError):
            module.library()


# addresses that no refused call looks at
P = 4096


def scan_struct(**changes):
    sequence = state_space.Sequence(P, 64, 8)
    vectors = state_space.Vectors(P, 64, 4, 4)
    s = state_space.Scan(2, 8, 8, 4, 1, 2, 1, sequence, sequence, state_space.Sequence(), vectors, vectors, P, P, P, None, None)
    for name, value in changes.items():
        setattr(s, name, value)
    return s


def test_scan_entry_points_refuse(libraries):
    lib, _ = libraries
    empty = state_space.Sequence()
    for changes, word in (({'batch': 0}, b'positive'), ({'length': 0}, b'positive'), ({'channels': 0}, b'positive'),
                          ({'state': 0}, b'positive'), ({'groups': 0}, b'positive'), ({'state': 65}, b'64 state'),
                          ({'groups': 3}, b'divide'), ({'dtype': 3}, b'element type'), ({'u': empty}, b'null'),
                          ({'delta': empty}, b'null'), ({'B': state_space.Vectors()}, b'null'),
                          ({'C': state_space.Vectors()}, b'null'), ({'A': None}, b'null'),
                          ({'length': (1 << 30) + 1}, b'2^30'), ({'batch': 1 << 30, 'channels': 1 << 20}, b'too many'),
                          ({'batch': 1 << 28, 'length': 1 << 30, 'state': 64}, b'too many')):
        s = scan_struct(**changes)
        ref = ctypes.byref(s)
        assert lib.ovl_ssm_scan_forward(ref, P, P, None, None, 0, None) == EINVAL, changes
        assert word in lib.ovl_ssm_last_error(), changes
        assert lib.ovl_ssm_scan_backward(ref, P, ctypes.byref(state_space.ScanGradients()), P, 1 << 40, None) == EINVAL
        assert lib.ovl_ssm_scan_workspace_bytes(ref, 0) == 0 and lib.ovl_ssm_scan_saved_bytes(ref) == 0
    s = scan_struct()
    ref = ctypes.byref(s)
    assert lib.ovl_ssm_scan_forward(None, P, P, None, None, 0, None) == EINVAL
    assert lib.ovl_ssm_scan_forward(ref, P, None, None, None, 0, None) == EINVAL
    assert lib.ovl_ssm_scan_forward(ref, None, None, None, None, 0, None) == EINVAL
    assert lib.ovl_ssm_scan_backward(ref, None, ctypes.byref(state_space.ScanGradients()), P, 1 << 40, None) == EINVAL
    assert lib.ovl_ssm_scan_backward(ref, P, ctypes.byref(state_space.ScanGradients()), P, 1 << 40, None) == EINVAL
    gradients = state_space.ScanGradients(state_space.Sequence(P, 64, 8), None, *([P] * 9))
    need = lib.ovl_ssm_scan_workspace_bytes(ref, 1)
    assert need > 0
    for workspace, size in ((None, need), (P, need - 1), (P + 4, need)):
        assert lib.ovl_ssm_scan_backward(ref, P, ctypes.byref(gradients), workspace, size, None) == EINVAL
        assert b'workspace' in lib.ovl_ssm_last_error()
    assert lib.ovl_ssm_scan_step(ref, P, 32, P, None) == EINVAL             # eight tokens are no step
    s.length = 1
    assert lib.ovl_ssm_scan_step(ref, None, 32, P, None) == EINVAL
    s.lengths = P
    assert lib.ovl_ssm_scan_step(ref, P, 32, P, None) == EINVAL
    long = scan_struct(batch=1, length=1 << 14)                             # split into chunks: needs scratch memory
    need = lib.ovl_ssm_scan_workspace_bytes(ctypes.byref(long), 0)
    assert need > 0
    assert lib.ovl_ssm_scan_forward(ctypes.byref(long), P, P, None, P, need - 1, None) == EINVAL


def test_conv_entry_points_refuse(libraries):
    lib, _ = libraries
    sequence = state_space.Sequence(P, 64, 8)

    def struct(**changes):
        s = state_space.Conv(2, 8, 8, 4, 2, 1, sequence, P, P, sequence, None)
        for name, value in changes.items():
            setattr(s, name, value)
        return s

    for changes in ({'batch': 0}, {'length': 0}, {'channels': 0}, {'width': 0}, {'width': 5}, {'dtype': 9},
                    {'x': state_space.Sequence()}, {'weight': None}, {'length': (1 << 30) + 1},
                    {'batch': 1 << 31, 'channels': 1 << 31}, {'batch': 1, 'length': 1, 'channels': (1 << 31) + 8}):
        ref = ctypes.byref(struct(**changes))
        assert lib.ovl_ssm_conv_forward(ref, P, P, None) == EINVAL, changes
        assert lib.ovl_ssm_conv_workspace_bytes(ref) == 0
        assert lib.ovl_ssm_conv_backward(ref, ctypes.byref(sequence), None, P, P, P, P, P, 1 << 40, None) == EINVAL
    s = struct()
    ref = ctypes.byref(s)
    assert lib.ovl_ssm_conv_forward(ref, None, P, None) == EINVAL
    assert lib.ovl_ssm_conv_forward(ref, P, None, None) == EINVAL
    need = lib.ovl_ssm_conv_workspace_bytes(ref)
    assert need > 0
    assert lib.ovl_ssm_conv_backward(ref, ctypes.byref(sequence), None, P, P, P, P, P, need - 1, None) == EINVAL
    assert lib.ovl_ssm_conv_backward(ref, None, None, P, P, P, P, P, need, None) == EINVAL
    assert lib.ovl_ssm_conv_step(ref, P, None) == EINVAL
    one = struct(length=1, kept=state_space.Sequence())
    assert lib.ovl_ssm_conv_step(ctypes.byref(one), P, None) == EINVAL


def test_norm_entry_points_refuse(libraries):
    _, lib = libraries

    def struct(**changes):
        s = rms_norm.Norm(4, 16, 32, 32, 2, 1e-5, P, 16, None, 0, P)
        for name, value in changes.items():
            setattr(s, name, value)
        return s

    for changes in ({'rows': 0}, {'columns': 0}, {'columns': 32769}, {'dtype': 3}, {'residual_dtype': 1}, {'weight_dtype': 1},
                    {'x': None}, {'weight': None}):
        ref = ctypes.byref(struct(**changes))
        assert lib.ovl_norm_forward(ref, P, P, None) == EINVAL, changes
        assert lib.ovl_norm_forward_quantized(ref, 0, P, P, P, None) == EINVAL, changes
        assert lib.ovl_norm_backward(ref, P, 16, None, 0, P, P, P, P, 1 << 40, None) == EINVAL, changes
        assert lib.ovl_norm_workspace_bytes(ref) == 0
    s = struct()
    ref = ctypes.byref(s)
    assert lib.ovl_norm_forward(None, P, P, None) == EINVAL
    assert lib.ovl_norm_forward(ref, None, None, None) == EINVAL
    assert lib.ovl_norm_forward_quantized(ref, 64, P, P, None, None) == EINVAL
    assert b'128' in lib.ovl_norm_last_error()
    assert lib.ovl_norm_forward_quantized(ref, 0, P, None, None, None) == EINVAL
    need = lib.ovl_norm_workspace_bytes(ref)
    assert lib.ovl_norm_backward(ref, P, 16, None, 0, P, P, P, P, need - 1, None) == EINVAL
    assert lib.ovl_norm_backward(ref, P, 16, None, 0, P, P, None, P, need, None) == EINVAL
    s.residual = P
    assert lib.ovl_norm_forward(ref, P, None, None) == EINVAL


def test_python_functions_refuse_host_tensors_and_other_things():
    u = torch.zeros(2, 4, 8)
    A = torch.zeros(8, 4)
    B = torch.zeros(2, 4, 4)
    with pytest.raises(RuntimeError):
        state_space.scan(u, u, A, B, B)
    with pytest.raises(RuntimeError):
        state_space.scan_step(torch.zeros(2, 8, 4), u[:, 0], u[:, 0], A, B[:, 0], B[:, 0])
    with pytest.raises(RuntimeError):
        state_space.conv(u, torch.zeros(8, 4))
    with pytest.raises(RuntimeError):
        rms_norm.rms_norm(u, torch.ones(8))
    for call in (lambda: state_space.scan(u.numpy(), u, A, B, B), lambda: state_space.conv(None, A),
                 lambda: rms_norm.rms_norm([1.0], A)):
        with pytest.raises(TypeError):
            call()
    with pytest.raises(ValueError):
        state_space._silu('relu')
    with pytest.raises(ValueError):
        rms_norm.rms_norm_quantized(u, torch.ones(8), group=64)


def test_calls_pack_their_structs_as_the_headers_lay_them_out():
    def same(packed, structure):
        expected = bytes(structure)
        assert len(packed) == len(expected) and packed == expected

    numbers = iter(range(1, 100))
    some = lambda count: [next(numbers) for _ in range(count)]
    v = some(29)
    same(state_space._pack_scan(*v), state_space.Scan(*v[:7], *[tuple(v[i:j]) for i, j in ((7, 10), (10, 13), (13, 16), (16, 20), (20, 24))],
                                                     *v[24:]))
    v = some(16)
    same(state_space._pack_conv(*v), state_space.Conv(*v[:6], tuple(v[6:9]), v[9], v[10], tuple(v[11:14]), *v[14:]))
    v = some(13)
    same(state_space._pack_gradients(*v), state_space.ScanGradients(tuple(v[:3]), *v[3:]))
    v = some(3)
    same(state_space._pack_sequence(*v), state_space.Sequence(*v))
    v = some(5) + [0.25] + some(5)
    same(rms_norm._pack(*v), rms_norm.Norm(*v))


def test_scan_torch_keeps_states_only_where_a_backward_pass_can_follow(monkeypatch):
    kept = []

    def scan_without_a_gpu(u, delta, A, B, C, D, z, delta_bias, softplus, state, lengths, keep):
        kept.append(keep)
        return u * 1, u.new_zeros(u.shape[0], u.shape[2], A.shape[1]), u.new_zeros(1) if keep else None

    monkeypatch.setattr(state_space, '_scan', scan_without_a_gpu)
    u, B, plain = torch.zeros(2, 4, 8), torch.zeros(2, 4, 3), torch.zeros(8, 3)
    A = torch.nn.Parameter(torch.zeros(8, 3))
    y, _ = state_space.scan_torch(u, u, A, B, B)
    assert kept.pop() and y.requires_grad
    for mode in (torch.no_grad, torch.inference_mode):
        with mode():
            y, _ = state_space.scan_torch(u, u, A, B, B)
        assert not kept.pop() and not y.requires_grad
    y, _ = state_space.scan_torch(u, u, plain, B, B)
    assert not kept.pop() and not y.requires_grad
    y, _ = state_space.scan_torch(u, u, plain, B, B, state=torch.zeros(2, 8, 3, requires_grad=True))
    assert kept.pop() and y.requires_grad


def test_norms_of_any_number_of_rows_are_taken(libraries):
    """Forward passes of many rows are several launches; the backward pass walks."""
    _, lib = libraries
    for rows in ((1 << 26) + 1, (1 << 31) + 1, (1 << 32) - 1):
        s = rms_norm.Norm(rows, 64, 32, 32, 2, 1e-5, P, 64, None, 0, P)
        assert lib.ovl_norm_workspace_bytes(ctypes.byref(s)) == 2048 * 64 * 4, rows


def test_calls_that_one_launch_does_not_take_are_refused(libraries):
    """A launch has fewer than 2^32 work items; what no kernel of a call could be launched for is refused before any is."""
    lib, _ = libraries
    vectors = state_space.Vectors(P, 4, 4, 4)
    gradients = state_space.ScanGradients(state_space.Sequence(P, 64, 8), None, *([P] * 9))

    def scan(batch, length, channels, state, groups=1):
        return ctypes.byref(scan_struct(batch=batch, length=length, channels=channels, state=state, groups=groups))

    # the forward pass: a wavefront for 64 channels of a sequence and group
    taken, much = scan((1 << 26) - 4, 1, 64, 4), scan((1 << 26) - 3, 1, 64, 4)
    assert lib.ovl_ssm_scan_saved_bytes(taken) > 0 and lib.ovl_ssm_scan_saved_bytes(much) == 0
    assert lib.ovl_ssm_scan_forward(much, P, P, None, None, 0, None) == EINVAL and b'too many' in lib.ovl_ssm_last_error()
    # the backward pass: a workgroup of 256; one result of dB and dC per thread; 1024 threads for 64 results of dA, dD, d_bias
    for taken, much in ((scan((1 << 24) - 1, 1, 64, 4), scan(1 << 24, 1, 64, 4)),
                        (scan(1, 1 << 24, 64, 64, 1), scan(4, 1 << 23, 64, 64, 1)),
                        (scan(1, 1, (1 << 22) - (1 << 18), 64), scan(1, 1, 1 << 22, 64))):
        assert lib.ovl_ssm_scan_workspace_bytes(taken, 1) > 0
        assert lib.ovl_ssm_scan_workspace_bytes(much, 1) == 0
        assert lib.ovl_ssm_scan_backward(much, P, ctypes.byref(gradients), P, 1 << 60, None) == EINVAL
        assert b'too many' in lib.ovl_ssm_last_error()
    # the step: a workgroup of 256 for 64 channels of a sequence
    assert lib.ovl_ssm_scan_step(scan(1 << 24, 1, 64, 4), P, 256, P, None) == EINVAL
    assert b'too many' in lib.ovl_ssm_last_error()

    def conv(batch, channels, odd=0):
        sequence = state_space.Sequence(P + odd, channels, channels)
        return ctypes.byref(state_space.Conv(batch, 1, channels, 4, 32, 1, sequence, P, P, sequence, None))

    # the convolution: a thread for the channels of an access
    for batch, odd in ((1 << 29, 2), ((1 << 32) - 1, 0)):
        much = conv(batch, 16, odd)
        assert lib.ovl_ssm_conv_forward(much, P, P, None) == EINVAL and b'too many' in lib.ovl_ssm_last_error()
        assert lib.ovl_ssm_conv_step(much, P, None) == EINVAL and b'too many' in lib.ovl_ssm_last_error()
    # its backward pass: at least 8 threads for the accesses of a sequence, and 1024 for 64 channels of a tap's sum
    d_y = ctypes.byref(state_space.Sequence(P, 64, 64))
    for much in (conv(1 << 30, 1), conv(2, 1 << 26)):
        assert lib.ovl_ssm_conv_backward(much, d_y, None, P, P, P, P, P, 1 << 60, None) == EINVAL
        assert b'too many' in lib.ovl_ssm_last_error()
    assert lib.ovl_ssm_conv_workspace_bytes(conv(2, 1 << 26)) == 0
    assert lib.ovl_ssm_conv_workspace_bytes(conv(2, 1 << 25)) > 0


def test_rows_at_one_distance_are_not_copied():
    t = torch.arange(2 * 3 * 4 * 40).view(2, 3, 4, 40).float()
    for rows, stride in ((t, 40), (t[..., 8:24], 40), (t[:1, ..., :16], 40), (t[:, :, :1, 8:], 160), (t[:, :1, 1, :8], 480),
                         (t[:, 1:2, :, 3:4], None), (t[0, 0, 0, 1:9], 8), (t[:, 1:2], None), (t[1:, 1:, ::2, 5:], 80),
                         (t[:1, :1, :1, ::40], 1), (t[0, 0, :, 3:4], 40), (t[..., :16].transpose(1, 2), None),
                         (t[0, 0, :1].expand(5, 40), 0), (t[0, 0, :1, :8].expand(3, 5, 8), 0), (t[0, 0, 0, ::2], None),
                         (t[:0, ..., 8:24], 16)):
        got, got_stride = rms_norm._rows(rows)
        copied = stride is None
        assert (got.data_ptr() != rows.data_ptr()) == copied, (rows.shape, rows.stride())
        columns = rows.shape[-1]
        assert got_stride == (columns if copied else stride)
        seen = torch.as_strided(got, (rows.numel() // columns, columns), (got_stride, 1), got.storage_offset())
        assert torch.equal(seen, rows.reshape(-1, columns))
