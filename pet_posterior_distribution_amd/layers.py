"""The dense layer on MI355X: forward, backward, and activations kept in 8 bits between them.

Keras layout (networks.py:529-537): ``y = act(x @ kernel + bias + residual)`` with x (..., k), kernel (k, n).  The
residual comes before the activation, as in the reference's ConvBlock (networks.py:679-691).  Everything runs in
libpetdiff.so (include/petdense.h) on the current stream of x's device; there is no CPU path.

Types: bfloat16, float16 or float32, one for x, kernel, residual and dy; sums are fp32 and every output is rounded
once.  In a 16-bit layer's backward pass the pre-activation's gradient is rounded to the layer's type before the two
products (exact for ReLU and linear layers); the bias gradient sums it unrounded.

Tensors may have any leading dimensions and row stride; a tensor whose rows are not contiguous is copied first.
No call synchronises, so each can be captured into a graph.  Autograd does not record them: the gradients are
``dense_backward``'s.  Where an input of ``dense`` requires a gradient, a backward pass through its result raises
RuntimeError; what ``dense_backward`` and checkpoints return has no history.

================================================  =============================================
reference (file:line)                             here
================================================  =============================================
Dense(units, activation)  networks.py:529-537     ``dense``
ConvBlock relu(conv + residual)  networks.py:679  ``dense`` over the im2col matrix, ``residual=``
tape.gradient of both  diffusion_model.py:580     ``dense_backward``
(no counterpart)                                  ``checkpoint_activations``: 8-bit saved inputs
================================================  =============================================
"""
from __future__ import annotations

import struct
from typing import NamedTuple, Optional

import torch

from . import _lib

BLOCK = 32                                     # PETDENSE_BLOCK: values of a row that share an exponent
ACTIVATIONS = {None: 0, 'none': 0, 'linear': 0, 'relu': 1, 'gelu': 2, 'silu': 3}
_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


class DenseGradients(NamedTuple):
    """Gradients of ``dense``: of x, the kernel, the bias and the residual (None where not asked for)."""
    x: Optional[torch.Tensor]
    kernel: Optional[torch.Tensor]
    bias: Optional[torch.Tensor]
    residual: Optional[torch.Tensor]


def _check(rc, what):
    if rc == _lib.PETDIFF_OK:
        return
    msg = f'{what}: ' + _lib.lib().petdense_last_error().decode(errors='replace')
    if rc == _lib.PETDIFF_ERR_INVALID:
        raise ValueError(msg)
    raise _lib.PetdiffError(msg)


def _activation(activation):
    act = ACTIVATIONS.get(activation) if activation is None or isinstance(activation, str) else None
    if act is None and isinstance(activation, str):
        act = ACTIVATIONS.get(activation.lower())
    if act is None:
        raise ValueError(f'activation must be one of {sorted(k for k in ACTIVATIONS if k)} or None, got {activation!r}')
    return act


def _lead(t, what):
    """(type code, device) of the call's leading operand."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f'{what} must be a CUDA tensor')
    dt = _TYPES.get(t.dtype)
    if dt is None:
        raise ValueError(f'{what} must be bfloat16, float16 or float32, got {t.dtype}')
    if t.dim() < 1 or t.shape[-1] < 1:
        raise ValueError(f'{what} must have a last dimension of at least 1, got shape {tuple(t.shape)}')
    return dt, t.device


def _operand(t, shape, dtype, dev, what):
    """t as rows (see _rows) after the checks that it is what the call's other operands ask for."""
    if not isinstance(t, torch.Tensor) or t.shape != shape or t.dtype != dtype or t.device != dev:
        _refuse(t, shape, dtype, dev, what)
    if t.is_contiguous():
        return t, shape[-1]
    return _rows(t)


def _refuse(t, shape, dtype, dev, what):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f'{what} must be a CUDA tensor')
    if t.device != dev:
        raise ValueError(f'{what} is on {t.device}, not on {dev}')
    if t.shape != shape:
        raise ValueError(f'{what} must have shape {tuple(shape)}, got {tuple(t.shape)}')
    raise ValueError(f'{what} must be {dtype}, got {t.dtype}')


def _rows(t):
    """(..., n) as rows that are contiguous and do not overlap (copied if they have to be), and their stride."""
    n = t.shape[-1]
    if t.is_contiguous():
        return t, n
    v = t if t.dim() <= 2 else t.reshape(-1, n)      # a view where the leading dimensions can be merged
    if v.dim() == 2 and (n == 1 or v.stride(1) == 1) and v.stride(0) >= n:
        return v, v.stride(0)
    return v.contiguous(), n


def _units(kernel, k):
    """n of a kernel (k, n)."""
    if not isinstance(kernel, torch.Tensor) or kernel.dim() != 2 or kernel.shape[0] != k or kernel.shape[1] < 1:
        got = tuple(kernel.shape) if isinstance(kernel, torch.Tensor) else type(kernel).__name__
        raise ValueError(f'kernel must be (k, n) with k = {k} and n >= 1, got {got}')
    return kernel.shape[1]


def _ptr(t):
    return 0 if t is None else t.data_ptr()


class _Unrecorded(torch.autograd.Function):
    """Outputs whose backward pass is refused.  The node hangs on a tensor of its own, not on the call's inputs, so it
    keeps nothing of theirs alive."""

    @staticmethod
    def forward(ctx, root, *outputs):
        ctx.mark_dirty(*outputs)
        return outputs

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError('dense is not recorded by autograd: take its gradients from dense_backward '
                           '(or call it under torch.no_grad())')


def _unrecorded(*outputs):
    return _Unrecorded.apply(torch.empty(0, requires_grad=True), *outputs)


def _new(shape, dtype, dev):
    """torch.empty; with strides given torch takes 0.4 us less, of which a small call would notice every one."""
    if len(shape) == 2:
        return torch.empty_strided(shape, (shape[1], 1), dtype=dtype, device=dev)
    return torch.empty(shape, dtype=dtype, device=dev)


# the C structs' bytes (petdense_forward_args, petdense_backward_args): packing them is quicker than filling fields
_FORWARD = struct.Struct('@6P8q4i')
_BACKWARD = struct.Struct('@9P11q3i4x')


def _run(entry, workspace, args, dev, what):
    """One call of the library on the current stream of `dev`, with its workspace."""
    if _current_device() != dev.index:
        with torch.cuda.device(dev):
            return _run(entry, workspace, args, dev, what)
    nb = workspace(args)
    # from the allocator of the current stream: two streams, and two captured graphs, never share one
    ws = torch.empty_strided((nb,), (1,), dtype=torch.uint8, device=dev) if nb else None
    rc = entry(args, _ptr(ws), nb, _stream(dev))
    if rc:
        _check(rc, what)


def _run_plain(entry, args, dev, what):
    """The same for entries without a workspace; the stream is their last argument."""
    if _current_device() != dev.index:
        with torch.cuda.device(dev):
            return _run_plain(entry, args, dev, what)
    rc = entry(*args, _stream(dev))
    if rc:
        _check(rc, what)


# the current device, and the current stream's handle; through torch's own accessors where it has them (a Stream object
# costs 2 us a call)
_current_device = getattr(torch._C, '_cuda_getDevice', None) or torch.cuda.current_device
_raw_stream = getattr(torch._C, '_cuda_getCurrentRawStream', None)


def _stream(dev):
    return _raw_stream(dev.index) if _raw_stream else torch.cuda.current_stream(dev).cuda_stream


def dense(x, kernel, bias=None, activation=None, residual=None, return_preactivation=False, out_dtype=None):
    """``act(x @ kernel + bias + residual)``.

    x (..., k), kernel (k, n), bias (n,) of x's type or float32, residual (..., n); activation None, 'relu', 'gelu'
    (erf) or 'silu'.  ``out_dtype``: x's type (default) or float32.  With ``return_preactivation`` also returns the
    value before the activation, in the output's type: what ``dense_backward`` wants saved for GELU and SiLU.  (It
    wants it in the layer's type: cast the float32 outputs of a 16-bit layer, and their gradient, to x's.)"""
    dt, dev = _lead(x, 'x')
    t = x.dtype
    shape = x.shape
    k = shape[-1]
    n = _units(kernel, k)
    out = (*shape[:-1], n)
    act = _activation(activation)
    if out_dtype is None:
        out_dtype = t
    elif out_dtype not in (t, torch.float32):
        raise ValueError(f'out_dtype must be {t} or float32, got {out_dtype}')
    bias_f32 = False
    if bias is not None:
        bias_f32 = isinstance(bias, torch.Tensor) and bias.dtype == torch.float32
        bias, _ = _operand(bias, (n,), torch.float32 if bias_f32 else t, dev, 'bias')
    dropped = torch.is_grad_enabled() and (x.requires_grad or kernel.requires_grad or
                                           bias is not None and bias.requires_grad or
                                           isinstance(residual, torch.Tensor) and residual.requires_grad)
    x, ldx = _rows(x)
    kernel, ldk = _operand(kernel, (k, n), t, dev, 'kernel')
    ldr = 0
    if residual is not None:
        residual, ldr = _operand(residual, out, t, dev, 'residual')
    y = _new(out, out_dtype, dev)
    pre = _new(out, out_dtype, dev) if return_preactivation else None
    L = _lib.lib()
    _run(L.petdense_forward, L.petdense_forward_workspace, _FORWARD.pack(
        x.data_ptr(), kernel.data_ptr(), _ptr(bias), _ptr(residual), y.data_ptr(), _ptr(pre), ldx, ldk, ldr, n, n,
        y.numel() // n, k, n, dt, act, bias_f32, out_dtype == torch.float32), dev, 'dense')
    if dropped:
        y, pre = _unrecorded(y, pre) if pre is not None else (_unrecorded(y)[0], None)
    return (y, pre) if return_preactivation else y


def dense_backward(dy, x, kernel, activation=None, saved=None, need_x=True, need_kernel=True, need_bias=True,
                   need_residual=False, grad_dtype=None):
    """Gradients of ``dense`` from its output's gradient dy (..., n).

    x: the layer's input (..., k), or its ``ActivationCheckpoint``.  saved (..., n): the pre-activation for 'gelu' and
    'silu', the pre-activation or the output for 'relu', of dy's type.  ``grad_dtype``: type of the kernel's and the
    bias's gradients, dy's (default) or float32; dx and the residual's gradient have dy's type.  It is the type that
    their sums are rounded to: a 16-bit layer's products take a pre-activation's gradient of 16 bits either way.
    Returns ``DenseGradients``."""
    dt, dev = _lead(dy, 'dy')
    t = dy.dtype
    shape = dy.shape
    lead, n = shape[:-1], shape[-1]
    act = _activation(activation)
    if grad_dtype is None:
        grad_dtype = t
    elif grad_dtype not in (t, torch.float32):
        raise ValueError(f'grad_dtype must be {t} or float32, got {grad_dtype}')
    exps, lde = None, 0
    if isinstance(x, ActivationCheckpoint):
        if x.dtype != t:
            raise ValueError(f'the checkpoint is of {x.dtype} activations, dy is {t}')
        k = x.codes.shape[-1]
        exps, lde = _operand(x.exponents, (*lead, -(-k // BLOCK)), torch.uint8, dev, "the checkpoint's exponents")
        x, ldx = _operand(x.codes, (*lead, k), x.codes.dtype, dev, 'the checkpoint')
    else:
        k = x.shape[-1] if isinstance(x, torch.Tensor) and x.dim() else 0
        x, ldx = _operand(x, (*lead, k), t, dev, 'x')
        if k < 1:
            raise ValueError('x must be (..., k) with k >= 1')
    if _units(kernel, k) != n:
        raise ValueError(f'kernel must be ({k}, {n}), got {tuple(kernel.shape)}')
    kernel, ldk = _operand(kernel, (k, n), t, dev, 'kernel')
    lds = 0
    if act:
        if saved is None:
            raise ValueError(f'activation {activation!r} needs saved=')
        saved, lds = _operand(saved, shape, t, dev, 'saved')
    else:
        saved = None
    m = dy.numel() // n
    dy, ldd = _rows(dy)
    gx = _new((*lead, k), t, dev) if need_x else None
    gk = _new((k, n), grad_dtype, dev) if need_kernel else None
    gb = torch.empty_strided((n,), (1,), dtype=grad_dtype, device=dev) if need_bias else None
    gr = _new(shape, t, dev) if need_residual else None
    L = _lib.lib()
    _run(L.petdense_backward, L.petdense_backward_workspace, _BACKWARD.pack(
        dy.data_ptr(), x.data_ptr(), _ptr(exps), kernel.data_ptr(), _ptr(saved), _ptr(gx), _ptr(gk), _ptr(gb),
        _ptr(gr), ldd, ldx, lde, ldk, lds, k, n, n, m, k, n, dt, act, grad_dtype == torch.float32), dev,
        'dense_backward')
    return DenseGradients(gx, gk, gb, gr)


class ActivationCheckpoint:
    """Activations of ``dtype`` kept in 8 bits: e4m3 ``codes`` (..., k) (torch.float8_e4m3fn) and one byte E + 127 per
    block of 32 along a row, ``exponents`` (..., ceil(k / 32)) (uint8).  A value is codes * 2^E.  8.25 bits a value;
    a value is off by at most 2^-4 of itself, or 2^-10 of its block's 2^E, a part in 2^17.8 of the block's largest."""

    def __init__(self, codes, exponents, dtype):
        if not isinstance(codes, torch.Tensor) or not codes.is_cuda:
            raise ValueError('codes must be a CUDA tensor')
        if codes.dtype not in (torch.float8_e4m3fn, torch.uint8) or codes.dim() < 1 or codes.shape[-1] < 1:
            raise ValueError('codes must be (..., k) of float8_e4m3fn, k >= 1')
        _operand(exponents, (*codes.shape[:-1], -(-codes.shape[-1] // BLOCK)), torch.uint8, codes.device, 'exponents')
        if dtype not in _TYPES:
            raise ValueError(f'dtype must be bfloat16, float16 or float32, got {dtype}')
        self.codes, self.exponents, self.dtype = codes, exponents, dtype

    @property
    def shape(self):
        return self.codes.shape

    @property
    def device(self):
        return self.codes.device

    @property
    def nbytes(self):
        return self.codes.numel() + self.exponents.numel()

    def restore(self):
        """The activations that the codes stand for (..., k), in ``dtype``."""
        codes, ldc = _rows(self.codes)
        exps, lde = _rows(self.exponents)
        dev, k = codes.device, codes.shape[-1]
        x = _new(self.codes.shape, self.dtype, dev)
        _run_plain(_lib.lib().petdense_restore, (codes.data_ptr(), ldc, exps.data_ptr(), lde, x.numel() // k, k,
                                                 _TYPES[self.dtype], x.data_ptr(), k), dev, 'restore')
        return x


def checkpoint_activations(x):
    """``ActivationCheckpoint`` of x (..., k): what a layer's backward pass needs of its input, in 8 bits."""
    dt, dev = _lead(x, 'x')
    shape = x.shape
    k = shape[-1]
    nb = -(-k // BLOCK)
    c = ActivationCheckpoint.__new__(ActivationCheckpoint)
    c.codes = codes = _new(shape, torch.float8_e4m3fn, dev)
    c.exponents = exps = _new((*shape[:-1], nb), torch.uint8, dev)
    c.dtype = x.dtype
    x, ldx = _rows(x)
    _run_plain(_lib.lib().petdense_checkpoint, (x.data_ptr(), ldx, codes.numel() // k, k, dt, codes.data_ptr(), k,
                                                exps.data_ptr(), nb), dev, 'checkpoint_activations')
    return c
