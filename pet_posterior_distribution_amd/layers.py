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

import ctypes as C
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
    """(..., n) as (rows, n) with contiguous rows that do not overlap, copied if it has to be, and its row stride."""
    if t.dim() < 1:
        raise ValueError(f'{what} must have at least one dimension')
    n = t.shape[-1]
    if t.dim() == 1:
        v = t.reshape(1, n)
    elif t.dim() == 2:
        v = t
    else:
        m = 1
        for d in t.shape[:-1]:
            m *= d
        v = t.reshape(m, n)                    # a view where the leading dimensions can be merged
    if n > 0 and v.shape[0] > 0 and ((n > 1 and v.stride(1) != 1) or (v.shape[0] > 1 and v.stride(0) < n)):
        v = v.contiguous()
    return v, (v.stride(0) if v.shape[0] > 1 else n)


def _same_rows(t, lead, n, dtype, device, what):
    _on(t, device, what)
    if tuple(t.shape) != tuple(lead) + (n,):
        raise ValueError(f'{what} must have shape {tuple(lead) + (n,)}, got {tuple(t.shape)}')
    if t.dtype != dtype:
        raise ValueError(f'{what} must be {dtype}, got {t.dtype}')
    return _rows(t, what)


def _kernel(kernel, k, dtype, device):
    _on(kernel, device, 'kernel')
    if kernel.dim() != 2 or (k is not None and kernel.shape[0] != k):
        raise ValueError(f'kernel must be (k, n){f" with k = {k}" if k is not None else ""}, got {tuple(kernel.shape)}')
    if kernel.dtype != dtype:
        raise ValueError(f'kernel must be {dtype}, got {kernel.dtype}')
    if kernel.shape[1] < 1 or kernel.shape[0] < 1:
        raise ValueError('kernel must not be empty')
    return _rows(kernel, 'kernel')


def _ptr(t):
    return None if t is None else t.data_ptr()


def _stream(device):
    return C.c_void_p(torch.cuda.current_stream(device).cuda_stream)


def _workspace(nbytes, device):
    # from the allocator of the current stream: two streams, and two captured graphs, never share one
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


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
    lead, k = x.shape[:-1], x.shape[-1]
    w, ldk = _kernel(kernel, k, x.dtype, dev)
    n = w.shape[1]
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
    r2, ldr = (None, 0) if residual is None else _same_rows(residual, lead, n, x.dtype, dev, 'residual')
    y = torch.empty((*lead, n), dtype=out_dtype, device=dev)
    pre = torch.empty((*lead, n), dtype=out_dtype, device=dev) if return_preactivation else None
    a = _lib.PetdenseForwardArgs(
        _ptr(x2), _ptr(w), _ptr(bias), _ptr(r2), _ptr(y), _ptr(pre), ldx, ldk, ldr, n, n, x2.shape[0], k, n, dt, act,
        int(bias is not None and bias.dtype == torch.float32), int(out_dtype == torch.float32))
    L = _lib.lib()
    with torch.cuda.device(dev):
        nb = int(L.petdense_forward_workspace(C.byref(a)))
        ws = _workspace(nb, dev)
        _check(L.petdense_forward(C.byref(a), _ptr(ws), nb, _stream(dev)), 'dense')
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
    lead, n = dy.shape[:-1], dy.shape[-1]
    act = _activation(activation)
    grad_dtype = dy.dtype if grad_dtype is None else grad_dtype
    if grad_dtype not in (dy.dtype, torch.float32):
        raise ValueError(f'grad_dtype must be {dy.dtype} or float32, got {grad_dtype}')
    exps, lde = None, 0
    if isinstance(x, ActivationCheckpoint):
        if x.dtype != dy.dtype:
            raise ValueError(f'the checkpoint is of {x.dtype} activations, dy is {dy.dtype}')
        k = x.shape[-1]
        if tuple(x.shape[:-1]) != tuple(lead):
            raise ValueError(f'the checkpoint must have shape {tuple(lead) + (k,)}, got {tuple(x.shape)}')
        _on(x.codes, dev, 'the checkpoint')
        x2, ldx = _rows(x.codes, 'codes')
        exps, lde = _rows(x.exponents, 'exponents')
    else:
        k = x.shape[-1] if isinstance(x, torch.Tensor) and x.dim() else 0
        x2, ldx = _same_rows(x, lead, k, dy.dtype, dev, 'x')
        if k < 1:
            raise ValueError('x must be (..., k) with k >= 1')
    w, ldk = _kernel(kernel, k, dy.dtype, dev)
    if w.shape[1] != n:
        raise ValueError(f'kernel must be ({k}, {n}), got {tuple(kernel.shape)}')
    s2, lds = None, 0
    if act:
        if saved is None:
            raise ValueError(f'activation {activation!r} needs saved=')
        s2, lds = _same_rows(saved, lead, n, dy.dtype, dev, 'saved')
    d2, ldd = _rows(dy, 'dy')

    def out(need, shape, dtype):
        return torch.empty(shape, dtype=dtype, device=dev) if need else None

    gx = out(need_x, (*lead, k), dy.dtype)
    gk = out(need_kernel, (k, n), grad_dtype)
    gb = out(need_bias, (n,), grad_dtype)
    gr = out(need_residual, (*lead, n), dy.dtype)
    a = _lib.PetdenseBackwardArgs(
        _ptr(d2), _ptr(x2), _ptr(exps), _ptr(w), _ptr(s2), _ptr(gx), _ptr(gk), _ptr(gb), _ptr(gr), ldd, ldx, lde, ldk,
        lds, k, n, n, d2.shape[0], k, n, dt, act, int(grad_dtype == torch.float32))
    L = _lib.lib()
    with torch.cuda.device(dev):
        nb = int(L.petdense_backward_workspace(C.byref(a)))
        ws = _workspace(nb, dev)
        _check(L.petdense_backward(C.byref(a), _ptr(ws), nb, _stream(dev)), 'dense_backward')
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
        m, k = c2.shape
        x = torch.empty(self.codes.shape, dtype=self.dtype, device=self.device)
        with torch.cuda.device(self.device):
            _check(_lib.lib().petdense_restore(_ptr(c2), ldc, _ptr(e2), lde, m, k, _TYPES[self.dtype], _ptr(x), k,
                                               _stream(self.device)), 'restore')
        return x


def checkpoint_activations(x):
    """``ActivationCheckpoint`` of x (..., k): what a layer's backward pass needs of its input, in 8 bits."""
    _on(x, None, 'x')
    dt = _dtype(x, 'x')
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError('x must be (..., k) with k >= 1')
    x2, ldx = _rows(x, 'x')
    m, k = x2.shape
    nb = -(-k // BLOCK)
    codes = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=x.device)
    exps = torch.empty((*x.shape[:-1], nb), dtype=torch.uint8, device=x.device)
    with torch.cuda.device(x.device):
        _check(_lib.lib().petdense_checkpoint(_ptr(x2), ldx, m, k, dt, _ptr(codes), k, _ptr(exps), nb,
                                              _stream(x.device)), 'checkpoint_activations')
    return ActivationCheckpoint(codes, exps, x.dtype)
