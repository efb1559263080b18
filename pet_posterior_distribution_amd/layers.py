"""The dense layer on MI355X: forward, backward, and activations kept in 8 bits between them.

Keras layout (networks.py:529-537): ``y = act(x @ kernel + bias + residual)`` with x (..., k), kernel (k, n).  The
residual comes before the activation, as in the reference's ConvBlock (networks.py:679-691).  Everything runs in
libpetdiff.so (include/petdense.h) on the current stream of x's device; there is no CPU path.

Types: bfloat16, float16 or float32, one for x, kernel, residual and dy; sums are fp32 and every output is rounded
once.  In a 16-bit layer's backward pass the pre-activation's gradient is rounded to the layer's type before the two
products (exact for ReLU and linear layers); the bias gradient sums it unrounded.

Tensors may have any leading dimensions and row stride; a tensor whose rows are not contiguous is copied first.
No call synchronises, so each can be captured into a graph.

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
    name = activation.lower() if isinstance(activation, str) else activation
    if name not in ACTIVATIONS:
        raise ValueError(f'activation must be one of {sorted(k for k in ACTIVATIONS if k)} or None, got {activation!r}')
    return ACTIVATIONS[name]


def _dtype(t, what):
    if t.dtype not in _TYPES:
        raise ValueError(f'{what} must be bfloat16, float16 or float32, got {t.dtype}')
    return _TYPES[t.dtype]


def _on(t, device, what):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f'{what} must be a CUDA tensor')
    if device is not None and t.device != device:
        raise ValueError(f'{what} is on {t.device}, x is on {device}')
    return t


def _rows(t, what):
    """(..., n) as rows that are contiguous and do not overlap (copied if they have to be), and their stride."""
    if t.is_contiguous():
        return t, t.shape[-1]
    n = t.shape[-1]
    v = t if t.dim() <= 2 else t.reshape(-1, n)      # a view where the leading dimensions can be merged
    if v.dim() == 2 and (n == 1 or v.stride(1) == 1) and v.stride(0) >= n:
        return v, v.stride(0)
    return v.contiguous(), n


def _same_rows(t, shape, dtype, device, what):
    _on(t, device, what)
    if t.shape != shape:
        raise ValueError(f'{what} must have shape {tuple(shape)}, got {tuple(t.shape)}')
    if t.dtype != dtype:
        raise ValueError(f'{what} must be {dtype}, got {t.dtype}')
    return _rows(t, what)


def _kernel(kernel, k, dtype, device):
    _on(kernel, device, 'kernel')
    shape = kernel.shape
    if len(shape) != 2 or shape[0] != k:
        raise ValueError(f'kernel must be (k, n) with k = {k}, got {tuple(shape)}')
    if kernel.dtype != dtype:
        raise ValueError(f'kernel must be {dtype}, got {kernel.dtype}')
    if shape[1] < 1:
        raise ValueError('kernel must not be empty')
    return _rows(kernel, 'kernel')


def _ptr(t):
    return 0 if t is None else t.data_ptr()


# the C structs' bytes (petdense_forward_args, petdense_backward_args): packing them is quicker than filling fields
_FORWARD = struct.Struct('@6P8q4i')
_BACKWARD = struct.Struct('@9P11q3i4x')


def _run(entry, workspace, args, dev, what):
    """One call of the library on the current stream of `dev`, with its workspace."""
    if torch.cuda.current_device() != dev.index:
        with torch.cuda.device(dev):
            return _run(entry, workspace, args, dev, what)
    nb = workspace(args)
    # from the allocator of the current stream: two streams, and two captured graphs, never share one
    ws = torch.empty(nb, dtype=torch.uint8, device=dev) if nb else None
    rc = entry(args, _ptr(ws), nb, _stream(dev))
    if rc:
        _check(rc, what)


def _run_plain(entry, args, dev, what):
    """The same for entries without a workspace; the stream is their last argument."""
    if torch.cuda.current_device() != dev.index:
        with torch.cuda.device(dev):
            return _run_plain(entry, args, dev, what)
    rc = entry(*args, _stream(dev))
    if rc:
        _check(rc, what)


# the current stream's handle; through torch's own accessor where it has one (a Stream object costs 2 us a call)
_raw_stream = getattr(torch._C, '_cuda_getCurrentRawStream', None)


def _stream(dev):
    return _raw_stream(dev.index) if _raw_stream else torch.cuda.current_stream(dev).cuda_stream


def dense(x, kernel, bias=None, activation=None, residual=None, return_preactivation=False, out_dtype=None):
    """``act(x @ kernel + bias + residual)``.

    x (..., k), kernel (k, n), bias (n,) of x's type or float32, residual (..., n); activation None, 'relu', 'gelu'
    (erf) or 'silu'.  ``out_dtype``: x's type (default) or float32.  With ``return_preactivation`` also returns the
    value before the activation, in the output's type (what ``dense_backward`` wants saved for GELU and SiLU)."""
    _on(x, None, 'x')
    dt = _dtype(x, 'x')
    dev = x.device
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError('x must be (..., k) with k >= 1')
    shape = x.shape
    k = shape[-1]
    w, ldk = _kernel(kernel, k, x.dtype, dev)
    n = kernel.shape[1]
    m = x.numel() // k
    out = (*shape[:-1], n)
    act = _activation(activation)
    out_dtype = x.dtype if out_dtype is None else out_dtype
    if out_dtype not in (x.dtype, torch.float32):
        raise ValueError(f'out_dtype must be {x.dtype} or float32, got {out_dtype}')
    if bias is not None:
        _on(bias, dev, 'bias')
        if tuple(bias.shape) != (n,) or bias.dtype not in (x.dtype, torch.float32):
            raise ValueError(f'bias must be ({n},) of {x.dtype} or float32, got {tuple(bias.shape)} of {bias.dtype}')
        bias = bias.contiguous()
    x2, ldx = _rows(x, 'x')
    r2, ldr = (None, 0) if residual is None else _same_rows(residual, out, x.dtype, dev, 'residual')
    y = torch.empty(out, dtype=out_dtype, device=dev)
    pre = torch.empty(out, dtype=out_dtype, device=dev) if return_preactivation else None
    L = _lib.lib()
    _run(L.petdense_forward, L.petdense_forward_workspace, _FORWARD.pack(
        _ptr(x2), _ptr(w), _ptr(bias), _ptr(r2), _ptr(y), _ptr(pre), ldx, ldk, ldr, n, n, m, k, n, dt, act,
        bias is not None and bias.dtype == torch.float32, out_dtype == torch.float32), dev, 'dense')
    return (y, pre) if return_preactivation else y


def dense_backward(dy, x, kernel, activation=None, saved=None, need_x=True, need_kernel=True, need_bias=True,
                   need_residual=False, grad_dtype=None):
    """Gradients of ``dense`` from its output's gradient dy (..., n).

    x: the layer's input (..., k), or its ``ActivationCheckpoint``.  saved (..., n): the pre-activation for 'gelu' and
    'silu', the pre-activation or the output for 'relu', of dy's type.  ``grad_dtype``: type of the kernel's and the
    bias's gradients, dy's (default) or float32; dx and the residual's gradient have dy's type.  Returns
    ``DenseGradients``."""
    _on(dy, None, 'dy')
    dt = _dtype(dy, 'dy')
    dev = dy.device
    if dy.dim() < 1 or dy.shape[-1] < 1:
        raise ValueError('dy must be (..., n) with n >= 1')
    shape = dy.shape
    lead, n = shape[:-1], shape[-1]
    act = _activation(activation)
    grad_dtype = dy.dtype if grad_dtype is None else grad_dtype
    if grad_dtype not in (dy.dtype, torch.float32):
        raise ValueError(f'grad_dtype must be {dy.dtype} or float32, got {grad_dtype}')
    exps, lde = None, 0
    if isinstance(x, ActivationCheckpoint):
        if x.dtype != dy.dtype:
            raise ValueError(f'the checkpoint is of {x.dtype} activations, dy is {dy.dtype}')
        k = x.shape[-1]
        if x.shape[:-1] != lead:
            raise ValueError(f'the checkpoint must have shape {(*lead, k)}, got {tuple(x.shape)}')
        _on(x.codes, dev, 'the checkpoint')
        x2, ldx = _rows(x.codes, 'codes')
        exps, lde = _rows(x.exponents, 'exponents')
    else:
        k = x.shape[-1] if isinstance(x, torch.Tensor) and x.dim() else 0
        x2, ldx = _same_rows(x, (*lead, k), dy.dtype, dev, 'x')
        if k < 1:
            raise ValueError('x must be (..., k) with k >= 1')
    w, ldk = _kernel(kernel, k, dy.dtype, dev)
    if kernel.shape[1] != n:
        raise ValueError(f'kernel must be ({k}, {n}), got {tuple(kernel.shape)}')
    s2, lds = None, 0
    if act:
        if saved is None:
            raise ValueError(f'activation {activation!r} needs saved=')
        s2, lds = _same_rows(saved, shape, dy.dtype, dev, 'saved')
    d2, ldd = _rows(dy, 'dy')

    gx = torch.empty((*lead, k), dtype=dy.dtype, device=dev) if need_x else None
    gk = torch.empty((k, n), dtype=grad_dtype, device=dev) if need_kernel else None
    gb = torch.empty((n,), dtype=grad_dtype, device=dev) if need_bias else None
    gr = torch.empty(shape, dtype=dy.dtype, device=dev) if need_residual else None
    L = _lib.lib()
    _run(L.petdense_backward, L.petdense_backward_workspace, _BACKWARD.pack(
        _ptr(d2), _ptr(x2), _ptr(exps), _ptr(w), _ptr(s2), _ptr(gx), _ptr(gk), _ptr(gb), _ptr(gr), ldd, ldx, lde, ldk,
        lds, k, n, n, dy.numel() // n, k, n, dt, act, grad_dtype == torch.float32), dev, 'dense_backward')
    return DenseGradients(gx, gk, gb, gr)


class ActivationCheckpoint:
    """Activations of ``dtype`` kept in 8 bits: e4m3 ``codes`` (..., k) (torch.float8_e4m3fn) and one byte E + 127 per
    block of 32 along a row, ``exponents`` (..., ceil(k / 32)) (uint8).  A value is codes * 2^E.  8.25 bits a value;
    a value is off by at most 2^-4 of itself, or 2^-10 of its block's 2^E, a part in 2^17.8 of the block's largest."""

    def __init__(self, codes, exponents, dtype):
        _on(codes, None, 'codes')
        if codes.dtype not in (torch.float8_e4m3fn, torch.uint8) or codes.dim() < 1 or codes.shape[-1] < 1:
            raise ValueError('codes must be (..., k) of float8_e4m3fn, k >= 1')
        want = (*codes.shape[:-1], -(-codes.shape[-1] // BLOCK))
        _on(exponents, codes.device, 'exponents')
        if tuple(exponents.shape) != want or exponents.dtype != torch.uint8:
            raise ValueError(f'exponents must be {want} of uint8, got {tuple(exponents.shape)} of {exponents.dtype}')
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
        c2, ldc = _rows(self.codes, 'codes')
        e2, lde = _rows(self.exponents, 'exponents')
        dev, k = self.codes.device, self.codes.shape[-1]
        x = torch.empty(self.codes.shape, dtype=self.dtype, device=dev)
        _run_plain(_lib.lib().petdense_restore, (_ptr(c2), ldc, _ptr(e2), lde, x.numel() // k, k, _TYPES[self.dtype],
                                                 _ptr(x), k), dev, 'restore')
        return x


def checkpoint_activations(x):
    """``ActivationCheckpoint`` of x (..., k): what a layer's backward pass needs of its input, in 8 bits."""
    _on(x, None, 'x')
    dt = _dtype(x, 'x')
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError('x must be (..., k) with k >= 1')
    x2, ldx = _rows(x, 'x')
    k = x.shape[-1]
    nb = -(-k // BLOCK)
    codes = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=x.device)
    exps = torch.empty((*x.shape[:-1], nb), dtype=torch.uint8, device=x.device)
    _run_plain(_lib.lib().petdense_checkpoint, (_ptr(x2), ldx, x.numel() // k, k, dt, _ptr(codes), k, _ptr(exps), nb),
               x.device, 'checkpoint_activations')
    return ActivationCheckpoint(codes, exps, x.dtype)
