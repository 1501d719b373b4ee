"""
The hand-written root-mean-square norm kernels (``csrc/ovl_norm.hip``, C ABI in ``include/ovl_norm.h``) from Python: the
norm over the last axis, with the residual's addition in front of it and with an 8-bit output and its scales.

As with the row scans and the LSTM cell the shape is a run-time argument: nothing is traced, generated or compiled when
they are called.  Inputs are float32, float16 or bfloat16 torch tensors on a HIP device; a residual may also be float32
beside rows of 16 bits.  Sums and statistics are float32.  Launches go to the current PyTorch HIP stream and do not
synchronise; equal calls give equal bits.
"""

import contextlib
import ctypes
import os
import struct
import subprocess

from . import local

library_path = os.path.join(local.csrc_directory, 'libovl_norm.so')
source_path = os.path.join(local.csrc_directory, 'ovl_norm.hip')
include_directory = os.path.normpath(os.path.join(local.csrc_directory, '..', '..', 'include'))

EXPORTED_SYMBOLS = ('ovl_norm_forward', 'ovl_norm_forward_quantized', 'ovl_norm_workspace_bytes', 'ovl_norm_backward',
                    'ovl_norm_last_error')

#: longest row, and the columns that share a scale where not all of a row do
MAX_COLUMNS, GROUP_COLUMNS = 32768, 128


def build(force=False):
    """Compile the library with hipcc next to its source (same flags as generated operators); returns its path."""
    from .compiler import HIPCC_FLAGS
    sources = (source_path, os.path.join(local.csrc_directory, 'ovl_lane.h'), os.path.join(include_directory, 'ovl_norm.h'))
    newest = max(os.path.getmtime(p) for p in sources)
    if not force and os.path.exists(library_path) and os.path.getmtime(library_path) >= newest:
        return library_path
    tmp = library_path + '.tmp.%d' % os.getpid()
    cmd = [local.hipcc] + list(HIPCC_FLAGS) + ['-I' + include_directory, '-I' + local.csrc_directory,
                                               source_path, '-o', tmp]
    try:
        subprocess.check_output(cmd, stderr=subprocess.STDOUT, universal_newlines=True)
    except subprocess.CalledProcessError as exception:
        raise RuntimeError('hipcc failed for the norm library:\n' + exception.output)
    os.replace(tmp, library_path)
    return library_path


class Norm(ctypes.Structure):
    """``ovl_norm``"""
    _fields_ = [('rows', ctypes.c_uint32), ('columns', ctypes.c_uint32), ('dtype', ctypes.c_int32),
                ('residual_dtype', ctypes.c_int32), ('weight_dtype', ctypes.c_int32), ('eps', ctypes.c_float),
                ('x', ctypes.c_void_p), ('x_stride', ctypes.c_int64), ('residual', ctypes.c_void_p),
                ('residual_stride', ctypes.c_int64), ('weight', ctypes.c_void_p)]


# Packer of the struct above for the calls below: filling a ctypes structure costs ten times as much as packing its fields
# into a bytes object.
_pack = struct.Struct('@5If5Q').pack


_lib = None


def library():
    """The loaded library (loads it on first use); there is no fallback when it has not been built."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(library_path):
        raise RuntimeError('The norm library ' + library_path + ' has not been built. '
                           'Run "python -m opveclib_amd.build" first.')
    lib = ctypes.CDLL(library_path)
    p, i64, u64 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_uint64
    lib.ovl_norm_forward.argtypes = [p, p, p, p]
    lib.ovl_norm_forward_quantized.argtypes = [p, ctypes.c_uint32, p, p, p, p]
    lib.ovl_norm_workspace_bytes.argtypes = [p]
    lib.ovl_norm_backward.argtypes = [p, p, i64, p, i64, p, p, p, p, u64, p]
    for name in EXPORTED_SYMBOLS:
        getattr(lib, name).restype = u64 if name.endswith('_bytes') else ctypes.c_int
    lib.ovl_norm_last_error.restype = ctypes.c_char_p
    _lib = lib
    return lib


class NormError(RuntimeError):
    def __init__(self, code, detail):
        RuntimeError.__init__(self, 'ovl_norm error %d: %s' % (code, detail))
        self.code = code


def _call(code):
    if code != 0:
        raise NormError(code, library().ovl_norm_last_error().decode('utf-8', 'replace'))


_codes = {}


def _type_code(dtype, name):
    if not _codes:
        import torch
        _codes.update({torch.float16: 1, torch.float32: 2, torch.bfloat16: 32})
    code = _codes.get(dtype)
    if code is None:
        raise TypeError('%s must be float32, float16 or bfloat16, got %s' % (name, dtype))
    return code


def _rows(t):
    """The tensor as rows of its last axis, columns side by side: (that tensor, row stride).  Copied only where its rows
    do not lie at one distance from each other."""
    columns = t.shape[-1]
    if t.is_contiguous():
        return t, columns
    shape, strides = t.shape, t.stride()
    if strides[-1] == 1 or columns == 1:
        distance, rows = None, 1                    # of the rows of the axes seen so far, of which there are that many
        for size, stride in zip(shape[-2::-1], strides[-2::-1]):
            if size != 1:
                if distance is None:
                    distance = stride
                elif stride != distance * rows:
                    return t.contiguous(), columns
                rows *= size
        return t, columns if distance is None else distance
    return t.contiguous(), columns


def _check(torch, t, name, index, dtype, wide):
    """A tensor of that type, or with ``wide`` of float32."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(name + ' must be a torch tensor')
    if t.get_device() != index:
        raise TypeError('%s is on %s, expected cuda:%d' % (name, t.device, index))
    if t.dtype != dtype and not (wide and t.dtype == torch.float32):
        raise TypeError('%s must be %s%s, got %s' % (name, dtype, ' or torch.float32' if wide else '', t.dtype))


def _describe(torch, x, weight, eps, residual, names=('x', 'residual')):
    """The numbers in front of the addresses in ``ovl_norm``, and (rows, row stride) of x, (rows, row stride) of the
    residual - (None, 0) without one - and the dense weight."""
    if not isinstance(x, torch.Tensor):
        raise TypeError(names[0] + ' must be a torch tensor')
    if not x.is_cuda:
        raise RuntimeError('the norm kernels run on an AMD GPU: tensors must live on a HIP device')
    dtype, shape, index = x.dtype, x.shape, x.get_device()
    code = _type_code(dtype, names[0])
    if not shape or not 1 <= shape[-1] <= MAX_COLUMNS:
        raise TypeError('%s must have 1 to %d columns, got %s' % (names[0], MAX_COLUMNS, list(shape)))
    columns = shape[-1]
    _check(torch, weight, 'weight', index, dtype, True)
    if weight.shape != (columns,):
        raise TypeError('weight must be [%d], got %s' % (columns, list(weight.shape)))
    other, other_code = (None, 0), code
    if residual is not None:
        _check(torch, residual, names[1], index, dtype, True)
        if residual.shape != shape:
            raise TypeError('%s must be %s, got %s' % (names[1], list(shape), list(residual.shape)))
        other = _rows(residual)
        other_code = _codes[residual.dtype]
    count = x.numel() // columns
    if count >= 1 << 32:
        raise TypeError('%s must have fewer than 2^32 rows, got %s' % (names[0], list(shape)))
    return (count, columns, code, other_code, _codes[weight.dtype], eps), _rows(x), other, weight.contiguous()


def _norm(numbers, rows, other, weight):
    """``ovl_norm`` as bytes."""
    return _pack(*numbers, rows[0].data_ptr(), rows[1], 0 if other[0] is None else other[0].data_ptr(), other[1],
                 weight.data_ptr())


_here = contextlib.nullcontext()


def _on(torch, index):
    """The device of the call as the current one; without the cost of switching where it is already."""
    return _here if index == torch.cuda.current_device() else torch.cuda.device(index)


def _new(torch, like):
    """A dense tensor of that shape and type for a result."""
    return torch.empty_like(like, memory_format=torch.contiguous_format)


def rms_norm(x, weight, eps=1e-5, residual=None):
    """
    ``y = s / sqrt(mean(s * s) + eps) * weight`` over the last axis, with s = x, or s = x + residual rounded to the
    residual's type (the norm is that of the sum as it is returned).

    :param x: [..., columns], at most 32768 columns; weight: [columns], float32 or of the type of ``x``
    :param residual: like ``x``, or float32
    :return: y like ``x``; with a residual (y, s)
    """
    import torch
    held = _describe(torch, x, weight, eps, residual)
    y = _new(torch, x)
    summed = None if residual is None else _new(torch, residual)
    if x.numel() > 0:
        with _on(torch, x.get_device()):
            _call(library().ovl_norm_forward(_norm(*held), y.data_ptr(), None if summed is None else summed.data_ptr(),
                                             torch._C._cuda_getCurrentRawStream(x.get_device())))
    return y if residual is None else (y, summed)


def rms_norm_quantized(x, weight, eps=1e-5, residual=None, group=None):
    """
    :func:`rms_norm` with its result in 8 bits: ``q = e4m3(y / scale)``, the float32 quotient of the float32 result y
    rounded to nearest, ties to even, where scale is the largest magnitude of y divided by 448 (the largest e4m3 value) - of
    the row, or with ``group=128`` of each 128 columns of it -, at least 2^-126 (the smallest normal number), and 1 where all
    of them are zero (NaN does not count).

    :return: (q, scales) with q a torch.float8_e4m3fn tensor like ``x`` and scales [..., 1] resp. [..., ceil(columns /
        128)] in float32; with a residual (q, scales, s)
    """
    import torch
    if group not in (None, GROUP_COLUMNS):
        raise ValueError('group must be None or %d, got %r' % (GROUP_COLUMNS, group))
    held = _describe(torch, x, weight, eps, residual)
    q = torch.empty_like(x, dtype=torch.float8_e4m3fn, memory_format=torch.contiguous_format)
    groups = 1 if group is None else -(-x.shape[-1] // group)
    scales = x.new_empty(x.shape[:-1] + (groups,), dtype=torch.float32)
    summed = None if residual is None else _new(torch, residual)
    if x.numel() > 0:
        with _on(torch, x.get_device()):
            _call(library().ovl_norm_forward_quantized(_norm(*held), group or 0, q.data_ptr(), scales.data_ptr(),
                                                       None if summed is None else summed.data_ptr(),
                                                       torch._C._cuda_getCurrentRawStream(x.get_device())))
    return (q, scales) if residual is None else (q, scales, summed)


def rms_norm_grad(s, weight, d_y, d_s=None, eps=1e-5, both=False):
    """
    Gradients of :func:`rms_norm`; the statistics of the rows are recomputed.

    :param s: what was normalised: ``x``, or the sum that the forward pass returned
    :param d_y: the gradient of y; d_s: that of the returned sum, like ``s`` (or None)
    :param both: whether the gradient is wanted in the type of s too where that is not the type of y
    :return: (the gradient of s in the type of ``d_y``, the same in the type of ``s``, d_weight); the first two are one
        tensor where the types are the same, and the second is None without ``both`` where they differ
    """
    import torch
    if not isinstance(s, torch.Tensor):
        raise TypeError('s must be a torch tensor')
    numbers, (d_y_rows, d_y_stride), s_rows, dense_weight = _describe(torch, d_y, weight, eps, s, ('d_y', 's'))
    # that describes d_y with s as residual: for the backward pass what was normalised stands in front
    norm = _norm(numbers, s_rows, (None, 0), dense_weight)
    same = s.dtype == d_y.dtype
    d_x = _new(torch, d_y)
    d_total = d_x if same else (_new(torch, s) if both else None)
    d_weight = _new(torch, weight)
    d_s_rows, d_s_stride = None, 0
    if d_s is not None:
        _check(torch, d_s, 'd_s', s.get_device(), s.dtype, False)
        if d_s.shape != s.shape:
            raise TypeError('d_s must be %s, got %s' % (list(s.shape), list(d_s.shape)))
        d_s_rows, d_s_stride = _rows(d_s)
    if s.numel() == 0:
        return d_x, d_total, d_weight.zero_()
    lib = library()
    need = lib.ovl_norm_workspace_bytes(norm)
    work = s.new_empty(need, dtype=torch.uint8)
    with _on(torch, s.get_device()):
        _call(lib.ovl_norm_backward(norm, d_y_rows.data_ptr(), d_y_stride,
                                    None if d_s_rows is None else d_s_rows.data_ptr(), d_s_stride, d_x.data_ptr(),
                                    None if same or d_total is None else d_total.data_ptr(), d_weight.data_ptr(),
                                    work.data_ptr(), need, torch._C._cuda_getCurrentRawStream(s.get_device())))
    return d_x, d_total, d_weight


_functions = {}


def _differentiable(name):
    """The autograd functions, made on first use (torch is imported late)."""
    if _functions:
        return _functions[name]
    import torch
    once = torch.autograd.function.once_differentiable

    class _Norm(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, weight, eps):
            ctx.eps = eps
            ctx.save_for_backward(x, weight)
            return rms_norm(x, weight, eps)

        @staticmethod
        @once
        def backward(ctx, d_y):
            x, weight = ctx.saved_tensors
            d_x, _, d_weight = rms_norm_grad(x, weight, d_y, None, ctx.eps)
            return d_x, d_weight, None

    class _ResidualNorm(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, residual, weight, eps):
            y, summed = rms_norm(x, weight, eps, residual)
            ctx.eps = eps
            ctx.dtype = x.dtype
            ctx.set_materialize_grads(False)
            ctx.save_for_backward(summed, weight)
            return y, summed

        @staticmethod
        @once
        def backward(ctx, d_y, d_summed):
            summed, weight = ctx.saved_tensors
            if d_y is None:
                d_y = torch.zeros(summed.shape, dtype=ctx.dtype, device=summed.device)
            d_x, d_residual, d_weight = rms_norm_grad(summed, weight, d_y, d_summed, ctx.eps, both=True)
            return d_x, d_residual, d_weight, None

    _functions.update(norm=_Norm, residual=_ResidualNorm)
    return _functions[name]


def rms_norm_torch(x, weight, eps=1e-5, residual=None):
    """:func:`rms_norm` as a differentiable PyTorch function."""
    if residual is None:
        return _differentiable('norm').apply(x, weight, eps)
    return _differentiable('residual').apply(x, residual, weight, eps)
