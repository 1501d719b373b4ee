"""
The hand-written state space kernels (``csrc/ovl_ssm_scan.hip``, ``csrc/ovl_ssm_conv.hip``, C ABI in
``include/ovl_ssm.h``) from Python: the selective state space scan and the short causal convolution in front of it.

Like the row scans (``row_scan``) and the LSTM cell (``lstm_cell``) these are recurrences with run-time shapes: nothing is
traced, generated or compiled when they are called.  Each comes as a plain call for whole sequences (:func:`scan`,
:func:`conv`), its gradient (:func:`scan_grad`, :func:`conv_grad`), a differentiable PyTorch function
(:func:`scan_torch`, :func:`conv_torch`) and a form for one new token per sequence that updates its state in place
(:func:`scan_step`, :func:`conv_step`).

Sequences are [batch, length, channels] tensors of one type - float32, float16 or bfloat16 - on one HIP device; their
channels lie side by side, the other strides are free (so halves of a projection are used where they are; a tensor with
other channel strides is copied first).  States, statistics and gradients of parameters are float32 throughout; outputs
are rounded once.  Launches go to the current PyTorch HIP stream and do not synchronise; equal calls give equal bits.

``lengths`` ([batch], int32, on the device) says how many tokens of a padded batch belong to each sequence (values are
clamped to 0 .. length): returned states are those after the last token, outputs and gradients behind it are zero, and
what the padding holds is not looked at.
"""

import contextlib
import ctypes
import os
import struct
import subprocess

from . import local

library_path = os.path.join(local.csrc_directory, 'libovl_ssm.so')
source_paths = [os.path.join(local.csrc_directory, n) for n in ('ovl_ssm_scan.hip', 'ovl_ssm_conv.hip')]
include_directory = os.path.normpath(os.path.join(local.csrc_directory, '..', '..', 'include'))

EXPORTED_SYMBOLS = ('ovl_ssm_scan_workspace_bytes', 'ovl_ssm_scan_saved_bytes', 'ovl_ssm_scan_forward',
                    'ovl_ssm_scan_backward', 'ovl_ssm_scan_step', 'ovl_ssm_conv_forward', 'ovl_ssm_conv_workspace_bytes',
                    'ovl_ssm_conv_backward', 'ovl_ssm_conv_step', 'ovl_ssm_last_error')

#: largest number of state entries per channel, and of taps of the convolution
MAX_STATE, MAX_WIDTH = 64, 4
#: largest token stride (in elements) the scan takes as it is; tensors with larger ones are copied
MAX_TOKEN_STRIDE = 1 << 25


def build(force=False):
    """Compile the library with hipcc next to its sources (same flags as generated operators); returns its path."""
    from .compiler import HIPCC_FLAGS
    headers = [os.path.join(local.csrc_directory, n) for n in ('ovl_lane.h', 'ovl_ssm_host.h')]
    headers.append(os.path.join(include_directory, 'ovl_ssm.h'))
    newest = max(os.path.getmtime(p) for p in source_paths + headers)
    if not force and os.path.exists(library_path) and os.path.getmtime(library_path) >= newest:
        return library_path
    tag = '.tmp.%d' % os.getpid()
    flags = [local.hipcc] + [f for f in HIPCC_FLAGS if f != '-shared'] + ['-I' + include_directory,
                                                                          '-I' + local.csrc_directory]
    objects = [p[:-len('.hip')] + tag + '.o' for p in source_paths]
    running = [subprocess.Popen(flags + ['-c', source, '-o', to], stdout=subprocess.PIPE, stderr=subprocess.STDOUT,
                                universal_newlines=True) for source, to in zip(source_paths, objects)]
    try:
        said = [p.communicate()[0] for p in running]
        if any(p.returncode != 0 for p in running):
            raise RuntimeError('hipcc failed for the state space library:\n' + '\n'.join(said))
        try:
            subprocess.check_output([local.hipcc, '--offload-arch=' + local.gpu_arch, '-shared'] + objects +
                                    ['-o', library_path + tag], stderr=subprocess.STDOUT, universal_newlines=True)
        except subprocess.CalledProcessError as exception:
            raise RuntimeError('hipcc failed for the state space library:\n' + exception.output)
    finally:
        for path in objects:
            if os.path.exists(path):
                os.remove(path)
    os.replace(library_path + tag, library_path)
    return library_path


class Sequence(ctypes.Structure):
    """``ovl_ssm_sequence``"""
    _fields_ = [('data', ctypes.c_void_p), ('batch_stride', ctypes.c_int64), ('token_stride', ctypes.c_int64)]


class Vectors(ctypes.Structure):
    """``ovl_ssm_vectors``"""
    _fields_ = [('data', ctypes.c_void_p), ('batch_stride', ctypes.c_int64), ('token_stride', ctypes.c_int64),
                ('group_stride', ctypes.c_int64)]


class Scan(ctypes.Structure):
    """``ovl_ssm_scan``"""
    _fields_ = [(n, ctypes.c_uint32) for n in ('batch', 'length', 'channels', 'state', 'groups')] + \
               [('dtype', ctypes.c_int32), ('softplus', ctypes.c_int32)] + \
               [(n, Sequence) for n in ('u', 'delta', 'z')] + [(n, Vectors) for n in ('B', 'C')] + \
               [(n, ctypes.c_void_p) for n in ('A', 'D', 'delta_bias', 'entering', 'lengths')]


class ScanGradients(ctypes.Structure):
    """``ovl_ssm_scan_gradients``"""
    _fields_ = [('d_y', Sequence)] + [(n, ctypes.c_void_p) for n in
                                      ('d_last', 'd_u', 'd_delta', 'd_z', 'd_B', 'd_C', 'd_A', 'd_D', 'd_delta_bias',
                                       'd_entering')]


class Conv(ctypes.Structure):
    """``ovl_ssm_conv``"""
    _fields_ = [(n, ctypes.c_uint32) for n in ('batch', 'length', 'channels', 'width')] + \
               [('dtype', ctypes.c_int32), ('silu', ctypes.c_int32), ('x', Sequence), ('weight', ctypes.c_void_p),
                ('bias', ctypes.c_void_p), ('kept', Sequence), ('lengths', ctypes.c_void_p),
                ('own_weights', ctypes.c_int32)]


# Packers of the structs above for the calls below: filling a ctypes structure costs ten times as much as packing its
# fields into a bytes object, and a call for one token has little else to do.
_pack_scan = struct.Struct('@7I4x22Q').pack
_pack_conv = struct.Struct('@6I9QI4x').pack
_pack_gradients = struct.Struct('@13Q').pack
_pack_sequence = struct.Struct('@3Q').pack


_lib = None


def library():
    """The loaded library (loads it on first use); there is no fallback when it has not been built."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(library_path):
        raise RuntimeError('The state space library ' + library_path + ' has not been built. '
                           'Run "python -m opveclib_amd.build" first.')
    lib = ctypes.CDLL(library_path)
    p, u64 = ctypes.c_void_p, ctypes.c_uint64
    lib.ovl_ssm_scan_workspace_bytes.argtypes = [p, ctypes.c_int32]
    lib.ovl_ssm_scan_saved_bytes.argtypes = [p]
    lib.ovl_ssm_scan_forward.argtypes = [p, p, p, p, p, u64, p]
    lib.ovl_ssm_scan_backward.argtypes = [p, p, p, p, u64, p]
    lib.ovl_ssm_scan_step.argtypes = [p, p, ctypes.c_int64, p, p]
    lib.ovl_ssm_conv_forward.argtypes = [p, p, p, p]
    lib.ovl_ssm_conv_workspace_bytes.argtypes = [p]
    lib.ovl_ssm_conv_backward.argtypes = [p, p, p, p, p, p, p, p, u64, p]
    lib.ovl_ssm_conv_step.argtypes = [p, p, p]
    for name in EXPORTED_SYMBOLS:
        getattr(lib, name).restype = u64 if name.endswith('_bytes') else ctypes.c_int
    lib.ovl_ssm_last_error.restype = ctypes.c_char_p
    _lib = lib
    return lib


class StateSpaceError(RuntimeError):
    def __init__(self, code, detail):
        RuntimeError.__init__(self, 'ovl_ssm error %d: %s' % (code, detail))
        self.code = code


def _call(code):
    if code != 0:
        raise StateSpaceError(code, library().ovl_ssm_last_error().decode('utf-8', 'replace'))


# ----------------------------------------------------------------------------------------------------------------------
# arguments
# ----------------------------------------------------------------------------------------------------------------------
_codes = {}


def _type_code(dtype):
    """The element type's code; only these three types have kernels."""
    if not _codes:
        import torch
        _codes.update({torch.float16: 1, torch.float32: 2, torch.bfloat16: 32})
    code = _codes.get(dtype)
    if code is None:
        raise TypeError('sequences must be float32, float16 or bfloat16, got ' + str(dtype))
    return code


class _Arguments(object):
    """Checks tensors of one call against its first one, and keeps those it had to copy alive until the launch.  Addresses
    of tensors that are not there are 0."""
    __slots__ = ('torch', 'Tensor', 'f32', 'index', 'dtype', 'code', 'kept')

    def __init__(self, torch, first, name):
        self.torch = torch
        self.Tensor = torch.Tensor
        self.f32 = torch.float32
        if not isinstance(first, torch.Tensor):
            raise TypeError(name + ' must be a torch tensor')
        if not first.is_cuda:
            raise RuntimeError('the state space kernels run on an AMD GPU: tensors must live on a HIP device')
        self.index = first.get_device()
        self.dtype = first.dtype
        self.code = _type_code(first.dtype)
        self.kept = []

    def tensor(self, t, name, shape, dtype):
        if not isinstance(t, self.Tensor):
            raise TypeError(name + ' must be a torch tensor')
        if t.get_device() != self.index:
            raise TypeError('%s is on %s, expected cuda:%d' % (name, t.device, self.index))
        if t.dtype != dtype:
            raise TypeError('%s must be %s, got %s' % (name, dtype, t.dtype))
        if t.shape != shape:
            raise TypeError('%s must be %s, got %s' % (name, list(shape), list(t.shape)))
        return t

    def copied(self, t):
        t = t.contiguous()
        self.kept.append(t)
        return t

    def dense(self, t):
        if not t.is_contiguous():
            t = self.copied(t)
        return t.data_ptr()

    def sequence(self, t, name, shape):
        """Address and strides of [batch, length, channels], or [batch, channels] for one token: channels side by side,
        tokens not too far apart."""
        if t is None:
            return 0, 0, 0
        self.tensor(t, name, shape, self.dtype)
        strides = t.stride()
        if len(strides) == 2:
            if strides[1] != 1 and shape[1] != 1:
                t = self.copied(t)
                strides = t.stride()
            return t.data_ptr(), strides[0], 0
        if (strides[2] != 1 and shape[2] != 1) or strides[1] > MAX_TOKEN_STRIDE:
            t = self.copied(t)
            strides = t.stride()
        return t.data_ptr(), strides[0], strides[1]

    def vectors(self, t, name, shape, token, grouped):
        """Address and strides of [batch, length, groups, state], or without the length for one token; without the groups
        if there is one."""
        self.tensor(t, name, shape, self.dtype)
        strides = t.stride()
        if (strides[-1] != 1 and shape[-1] != 1) or (not token and strides[1] > MAX_TOKEN_STRIDE):
            t = self.copied(t)
            strides = t.stride()
        return t.data_ptr(), strides[0], 0 if token else strides[1], strides[-2] if grouped else 0

    def parameter(self, t, name, shape):
        """A dense float32 tensor's address."""
        if t is None:
            return 0
        self.tensor(t, name, shape, self.f32)
        if not t.is_contiguous():
            t = self.copied(t)
        return t.data_ptr()

    def weights(self, weight, bias, width, channels):
        """(address of the taps, of the bias, whether they are of the sequences' type and not float32).  A call that mixes
        the types has the narrow one converted."""
        f32 = self.f32
        own = self.dtype != f32 and weight.dtype == self.dtype and (bias is None or bias.dtype == self.dtype)
        at = []
        for t, name, shape in ((weight, 'weight', (channels, width)), (bias, 'bias', (channels,))):
            if t is not None:
                if not own and t.dtype == self.dtype != f32:
                    t = t.detach().to(f32)
                    self.kept.append(t)
                at.append(self.dense(self.tensor(t, name, shape, self.dtype if own else f32)))
        return at[0], at[1] if bias is not None else 0, 1 if own else 0

    def lengths(self, t, batch):
        if t is None:
            return 0
        return self.dense(self.tensor(t, 'lengths', (batch,), self.torch.int32))

    def new(self, like):
        """A dense tensor of that shape and type for a result."""
        return self.torch.empty_like(like, memory_format=self.torch.contiguous_format)

    def scratch(self, like, nbytes):
        """Uninitialised device memory of that size: its address."""
        if nbytes == 0:
            return 0
        t = like.new_empty(nbytes, dtype=self.torch.uint8)
        self.kept.append(t)
        return t.data_ptr()

    def stream(self):
        return self.torch._C._cuda_getCurrentRawStream(self.index)

    def on(self):
        """The device of the call as the current one; without the cost of switching where it is already."""
        return _here if self.index == self.torch.cuda.current_device() else self.torch.cuda.device(self.index)


_here = contextlib.nullcontext()


# ----------------------------------------------------------------------------------------------------------------------
# the scan
# ----------------------------------------------------------------------------------------------------------------------
def _describe_scan(torch, u, delta, A, B, C, D, z, delta_bias, softplus, state, lengths, token=False):
    """(the checked arguments, ``ovl_ssm_scan`` as bytes, (batch, length, channels, state))"""
    args = _Arguments(torch, u, 'u')
    shape = u.shape
    if len(shape) != (2 if token else 3):
        raise TypeError('u must be %s, got %s' % ('[batch, channels]' if token else '[batch, length, channels]', list(shape)))
    batch, channels = shape[0], shape[-1]
    length = 1 if token else shape[1]
    if channels == 0:
        raise TypeError('u must have at least one channel')
    if not isinstance(A, torch.Tensor) or A.dim() != 2 or A.shape[0] != channels:
        raise TypeError('A must be [channels, state] with %d channels' % channels)
    n = A.shape[1]
    if not 1 <= n <= MAX_STATE:
        raise TypeError('A must have 1 to %d state entries per channel, got %d' % (MAX_STATE, n))
    if not isinstance(B, torch.Tensor):
        raise TypeError('B must be a torch tensor')
    groups, grouped = 1, B.dim() == len(shape) + 1
    if grouped:
        groups = B.shape[-2]
        if groups < 1 or channels % groups != 0:
            raise TypeError('the groups of B and C must divide the %d channels, got %d' % (channels, groups))
        vector_shape = (batch, groups, n) if token else (batch, length, groups, n)
    else:
        vector_shape = (batch, n) if token else (batch, length, n)
    scan_ = _pack_scan(batch, length, channels, n, groups, args.code, 1 if softplus else 0,
                       *args.sequence(u, 'u', shape), *args.sequence(delta, 'delta', shape), *args.sequence(z, 'z', shape),
                       *args.vectors(B, 'B', vector_shape, token, grouped),
                       *args.vectors(C, 'C', vector_shape, token, grouped),
                       args.parameter(A, 'A', (channels, n)), args.parameter(D, 'D', (channels,)),
                       args.parameter(delta_bias, 'delta_bias', (channels,)),
                       0 if token else args.parameter(state, 'state', (batch, channels, n)), args.lengths(lengths, batch))
    return args, scan_, (batch, length, channels, n)


def _scan(u, delta, A, B, C, D, z, delta_bias, softplus, state, lengths, keep):
    import torch
    args, scan_, (batch, length, channels, n) = _describe_scan(torch, u, delta, A, B, C, D, z, delta_bias, softplus, state,
                                                               lengths)
    y = args.new(u)
    last = u.new_empty((batch, channels, n), dtype=torch.float32)
    if batch == 0 or length == 0:
        return y, (last.zero_() if state is None else last.copy_(state.detach())), None
    lib = library()
    saved = None
    if keep:
        saved = u.new_empty(lib.ovl_ssm_scan_saved_bytes(scan_) // 4, dtype=torch.float32)
    need = lib.ovl_ssm_scan_workspace_bytes(scan_, 0)
    with args.on():
        _call(lib.ovl_ssm_scan_forward(scan_, y.data_ptr(), last.data_ptr(), None if saved is None else saved.data_ptr(),
                                       args.scratch(u, need), need, args.stream()))
    return y, last, saved


def scan(u, delta, A, B, C, D=None, z=None, delta_bias=None, softplus=False, state=None, lengths=None):
    """
    The selective state space scan: for every channel c, state entry n and token t

        dt = delta[t, c] + delta_bias[c], with ``softplus`` log(1 + exp(.)) of it
        h[t, n] = exp(dt * A[c, n]) * h[t - 1, n] + dt * u[t, c] * B[t, n]
        y[t, c] = sum over n of C[t, n] * h[t, n] + D[c] * u[t, c], times z[t, c] * sigmoid(z[t, c]) with a gate ``z``

    :param u, delta, z: [batch, length, channels]
    :param A: [channels, state], float32, up to 64 state entries
    :param B, C: [batch, length, state], or [batch, length, groups, state]: neighbouring channels / groups channels share
        the vectors of their group
    :param D, delta_bias: [channels], float32
    :param state: [batch, channels, state], float32: the state before the first token; zero if not given
    :return: (y [batch, length, channels], the state after the last token)
    """
    return _scan(u, delta, A, B, C, D, z, delta_bias, softplus, state, lengths, False)[:2]


def scan_grad(u, delta, A, B, C, d_y, D=None, z=None, delta_bias=None, softplus=False, state=None, lengths=None,
              d_last=None, saved=None):
    """
    Gradients of :func:`scan` given those of its outputs (``d_last`` may be left out).  The states inside the sequence are
    recomputed unless ``saved`` holds those that :func:`scan_torch` keeps.

    :return: (d_u, d_delta, d_A, d_B, d_C, d_D, d_z, d_delta_bias, d_state), None for what was not given
    """
    import torch
    args, scan_, (batch, length, channels, n) = _describe_scan(torch, u, delta, A, B, C, D, z, delta_bias, softplus, state,
                                                               lengths)
    state_shape = (batch, channels, n)
    if d_y is None:
        raise TypeError('d_y must be a torch tensor')
    d_y_at = args.sequence(d_y, 'd_y', u.shape)
    d_last_at = args.parameter(d_last, 'd_last', state_shape)
    out = (args.new(u), args.new(u), args.new(A), args.new(B), args.new(B), None if D is None else args.new(D),
           None if z is None else args.new(u), None if delta_bias is None else args.new(delta_bias),
           None if state is None else args.new(state))
    if batch == 0 or length == 0:
        for t in out:
            if t is not None:
                t.zero_()
        if out[8] is not None and d_last is not None:
            out[8].copy_(d_last.detach())
        return out
    d_u, d_delta, d_A, d_B, d_C, d_D, d_z, d_bias, d_state = [0 if t is None else t.data_ptr() for t in out]
    gradients = _pack_gradients(*d_y_at, d_last_at, d_u, d_delta, d_z, d_B, d_C, d_A, d_D, d_bias, d_state)
    lib = library()
    with args.on():
        stream = args.stream()
        need = lib.ovl_ssm_scan_saved_bytes(scan_)
        if saved is None:
            saved = u.new_empty(need // 4, dtype=torch.float32)
            work = lib.ovl_ssm_scan_workspace_bytes(scan_, 0)
            _call(lib.ovl_ssm_scan_forward(scan_, None, None, saved.data_ptr(), args.scratch(u, work), work, stream))
        else:
            args.tensor(saved, 'saved', (need // 4,), torch.float32)
            if not saved.is_contiguous():
                raise TypeError('saved must be contiguous')
        work = lib.ovl_ssm_scan_workspace_bytes(scan_, 1)
        _call(lib.ovl_ssm_scan_backward(scan_, saved.data_ptr(), gradients, args.scratch(u, work), work, stream))
    return out


def scan_step(state, u, delta, A, B, C, D=None, z=None, delta_bias=None, softplus=False):
    """
    :func:`scan` for one new token per sequence: ``u``, ``delta``, ``z`` are [batch, channels], ``B`` and ``C`` [batch,
    state] or [batch, groups, state].  ``state`` [batch, channels, state], float32, is updated in place; it may be a part
    of a larger buffer along its first axis (its other axes are dense, and its sequences do not overlap).

    :return: y [batch, channels]
    """
    import torch
    args, scan_, (batch, _, channels, n) = _describe_scan(torch, u, delta, A, B, C, D, z, delta_bias, softplus, None, None,
                                                          token=True)
    stride = _in_place(args, state, (batch, channels, n), torch.float32)[0]
    y = args.new(u)
    if batch == 0:
        return y
    with args.on():
        _call(library().ovl_ssm_scan_step(scan_, state.data_ptr(), stride, y.data_ptr(), args.stream()))
    torch.autograd.graph.increment_version(state)       # a backward pass that needs the state as it was raises
    return y


def _in_place(args, state, shape, dtype):
    """Strides of a [batch, .., ..] tensor that is overwritten: dense but for the first axis, whose parts lie apart."""
    args.tensor(state, 'state', shape, dtype)
    if state.requires_grad and args.torch.is_grad_enabled():
        raise TypeError('state is overwritten and must not require a gradient')
    strides = state.stride()
    inner = shape[1] * shape[2]
    if inner > 0 and not ((shape[2] == 1 or strides[2] == 1) and (shape[1] == 1 or strides[1] == shape[2])
                          and (shape[0] <= 1 or strides[0] >= inner)):
        raise TypeError('state is overwritten: its sequences must be dense and apart, got strides ' + str(strides))
    return strides[0], shape[2]


_functions = {}


def _differentiable(name):
    """The autograd functions, made on first use (torch is imported late)."""
    if _functions:
        return _functions[name]
    import torch
    once = torch.autograd.function.once_differentiable

    class _Scan(torch.autograd.Function):
        @staticmethod
        def forward(ctx, u, delta, A, B, C, D, z, delta_bias, state, lengths, softplus, recorded):
            # (needs_input_grad follows the tensors alone, also where nothing is recorded)
            y, last, saved = _scan(u, delta, A, B, C, D, z, delta_bias, softplus, state, lengths,
                                   recorded and any(ctx.needs_input_grad))
            ctx.softplus = softplus
            ctx.set_materialize_grads(False)
            ctx.save_for_backward(u, delta, A, B, C, D, z, delta_bias, state, lengths, saved)
            return y, last

        @staticmethod
        @once
        def backward(ctx, d_y, d_last):
            u, delta, A, B, C, D, z, delta_bias, state, lengths, saved = ctx.saved_tensors
            if d_y is None:
                d_y = torch.zeros_like(u)
            grads = scan_grad(u, delta, A, B, C, d_y, D, z, delta_bias, ctx.softplus, state, lengths, d_last, saved)
            return grads + (None, None, None)

    class _Conv(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, weight, bias, state, lengths, activation):
            ctx.activation = activation
            ctx.set_materialize_grads(False)
            ctx.save_for_backward(x, weight, bias, state, lengths)
            return conv(x, weight, bias, activation, state, lengths)

        @staticmethod
        @once
        def backward(ctx, d_y, d_last):
            x, weight, bias, state, lengths = ctx.saved_tensors
            if d_y is None:
                d_y = torch.zeros_like(x)
            grads = conv_grad(x, weight, d_y, bias, ctx.activation, state, lengths, d_last)
            return grads + (None, None)

    _functions.update(scan=_Scan, conv=_Conv)
    return _functions[name]


def scan_torch(u, delta, A, B, C, D=None, z=None, delta_bias=None, softplus=False, state=None, lengths=None):
    """:func:`scan` as a differentiable PyTorch function.  Where a backward pass can follow (an input requires a gradient,
    outside of ``torch.no_grad()`` and the like) the forward pass keeps the state before every 16th token for it: for each
    element of ``u`` 4 / 16 bytes times the state entries, counted as the next of 8, 16, 32 or 64."""
    import torch
    return _differentiable('scan').apply(u, delta, A, B, C, D, z, delta_bias, state, lengths, softplus,
                                         torch.is_grad_enabled())


# ----------------------------------------------------------------------------------------------------------------------
# the short causal convolution
# ----------------------------------------------------------------------------------------------------------------------
def _silu(activation):
    if activation not in (None, 'silu'):
        raise ValueError("activation must be None or 'silu', got " + repr(activation))
    return 0 if activation is None else 1


def _describe_conv(torch, x, weight, bias, activation, state, lengths, token=False):
    """(the checked arguments, ``ovl_ssm_conv`` as bytes, the shape of the state)"""
    args = _Arguments(torch, x, 'x')
    shape = x.shape
    if len(shape) != (2 if token else 3):
        raise TypeError('x must be %s, got %s' % ('[batch, channels]' if token else '[batch, length, channels]', list(shape)))
    batch, channels = shape[0], shape[-1]
    if channels == 0:
        raise TypeError('x must have at least one channel')
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2 or weight.shape[0] != channels:
        raise TypeError('weight must be [channels, width] with %d channels' % channels)
    width = weight.shape[1]
    if not 1 <= width <= MAX_WIDTH:
        raise TypeError('weight must have 1 to %d taps per channel, got %d' % (MAX_WIDTH, width))
    kept_shape = (batch, width - 1, channels)
    if token:
        strides = _in_place(args, state, kept_shape, x.dtype)
        kept = (state.data_ptr() if width > 1 else 0, strides[0], strides[1])
    else:
        kept = args.sequence(state, 'state', kept_shape)
        if width == 1:
            kept = (0, 0, 0)
    if bias is not None and not isinstance(bias, torch.Tensor):
        raise TypeError('bias must be a torch tensor')
    taps, more, own = args.weights(weight, bias, width, channels)
    conv_ = _pack_conv(batch, 1 if token else shape[1], channels, width, args.code, _silu(activation),
                       *args.sequence(x, 'x', shape), taps, more, *kept, args.lengths(lengths, batch), own)
    return args, conv_, kept_shape


def conv(x, weight, bias=None, activation=None, state=None, lengths=None):
    """
    Causal convolution of every channel with its own few taps: with ``line`` the ``width - 1`` tokens of ``state`` (zeros
    if not given) followed by ``x``,

        y[t, c] = bias[c] + sum over k of weight[c, k] * line[t + k, c], times its own sigmoid with activation 'silu'

    :param x: [batch, length, channels]
    :param weight: [channels, width], width 1 to 4; bias: [channels]; both float32 or of the type of ``x``
    :param state: [batch, width - 1, channels] of the type of ``x``: the tokens before the first
    :return: (y [batch, length, channels], the last width - 1 tokens, which a later call takes as ``state``)
    """
    import torch
    args, conv_, kept_shape = _describe_conv(torch, x, weight, bias, activation, state, lengths)
    y = args.new(x)
    last = x.new_empty(kept_shape)
    if y.numel() == 0:
        return y, (last.zero_() if state is None else last.copy_(state.detach()))
    with args.on():
        _call(library().ovl_ssm_conv_forward(conv_, y.data_ptr(), last.data_ptr(), args.stream()))
    return y, last


def conv_grad(x, weight, d_y, bias=None, activation=None, state=None, lengths=None, d_last=None):
    """
    Gradients of :func:`conv` given those of its outputs (``d_last`` may be left out); the convolution is recomputed.

    :return: (d_x, d_weight, d_bias, d_state), None for what was not given; d_weight and d_bias in their tensors' types
    """
    import torch
    args, conv_, kept_shape = _describe_conv(torch, x, weight, bias, activation, state, lengths)
    if d_y is None:
        raise TypeError('d_y must be a torch tensor')
    d_y_at = _pack_sequence(*args.sequence(d_y, 'd_y', x.shape))
    d_last_at = args.sequence(d_last, 'd_last', kept_shape)
    d_x = args.new(x)
    d_weight = x.new_empty(weight.shape, dtype=torch.float32)
    d_bias = None if bias is None else x.new_empty(bias.shape, dtype=torch.float32)
    d_state = None if state is None else args.new(state)
    if x.numel() == 0:
        d_weight.zero_()
        if d_bias is not None:
            d_bias.zero_()
        if d_state is not None:
            d_state.zero_() if d_last is None else d_state.copy_(d_last.detach())
    else:
        lib = library()
        need = lib.ovl_ssm_conv_workspace_bytes(conv_)
        with args.on():
            _call(lib.ovl_ssm_conv_backward(conv_, d_y_at, None if d_last_at[0] == 0 else _pack_sequence(*d_last_at),
                                            d_x.data_ptr(),
                                            0 if d_state is None or kept_shape[1] == 0 else d_state.data_ptr(),
                                            d_weight.data_ptr(), 0 if d_bias is None else d_bias.data_ptr(),
                                            args.scratch(x, need), need, args.stream()))
    return (d_x, d_weight.to(weight.dtype), None if d_bias is None else d_bias.to(bias.dtype), d_state)


def conv_step(x, state, weight, bias=None, activation=None):
    """
    :func:`conv` for one new token per sequence: ``x`` is [batch, channels]; ``state`` [batch, width - 1, channels] is
    updated in place; it may be a part of a larger buffer along its first axis (its other axes are dense, and its
    sequences do not overlap).

    :return: y [batch, channels]
    """
    import torch
    args, conv_, _ = _describe_conv(torch, x, weight, bias, activation, state, None, token=True)
    y = args.new(x)
    if y.numel() == 0:
        return y
    with args.on():
        _call(library().ovl_ssm_conv_step(conv_, y.data_ptr(), args.stream()))
    torch.autograd.graph.increment_version(state)       # a backward pass that needs the state as it was raises
    return y


def conv_torch(x, weight, bias=None, activation=None, state=None, lengths=None):
    """:func:`conv` as a differentiable PyTorch function (gradients through :func:`conv_grad`)."""
    return _differentiable('conv').apply(x, weight, bias, state, lengths, activation)
