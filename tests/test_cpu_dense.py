"""CPU tests of the dense layer's operators: every refused call is refused before the device is touched."""
import ctypes as C

import pytest
import torch

from pet_posterior_distribution_amd import _lib
from pet_posterior_distribution_amd import layers

L = _lib.lib()
INVALID = _lib.PETDIFF_ERR_INVALID


def forward_args(**kw):
    a = _lib.PetdenseForwardArgs(0x1000, 0x2000, None, None, 0x3000, None, 64, 32, 0, 32, 0, 100, 64, 32, 1, 0, 0, 0)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def backward_args(**kw):
    a = _lib.PetdenseBackwardArgs(0x1000, 0x2000, None, 0x3000, 0x4000, 0x5000, 0x6000, 0x7000, None, 32, 64, 0, 32,
                                  32, 64, 32, 0, 100, 64, 32, 1, 1, 0)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


BIG = 2 ** 31 - 100


@pytest.mark.parametrize('kw,says', [
    (dict(dtype=3), 'dtype'), (dict(dtype=-1), 'dtype'), (dict(activation=4), 'activation'),
    (dict(m=-1), 'm must be'), (dict(k=0), 'k and n'), (dict(n=0), 'k and n'), (dict(m=BIG), 'too large'),
    (dict(x=None), 'must be given'), (dict(kernel=None), 'must be given'), (dict(y=None), 'must be given'),
    (dict(ldx=63), 'stride'), (dict(ldk=31), 'stride'), (dict(ldy=31), 'stride'),
    (dict(residual=0x9000, ldr=31), 'stride'), (dict(pre=0x9000, ldp=31), 'stride'),
    (dict(y=0x1000), 'alias'), (dict(y=0x2000), 'alias'), (dict(pre=0x3000, ldp=32), 'alias'),
    (dict(residual=0x3000, ldr=40), 'residual only'), (dict(residual=0x3000, ldr=32, out_f32=1), 'residual only'),
    (dict(m=2 ** 30, n=2 ** 20, ldk=2 ** 20, ldy=2 ** 20), 'too many'),
])
def test_forward_refusals(kw, says):
    a = forward_args(**kw)
    assert L.petdense_forward_workspace(C.byref(a)) == 0
    assert L.petdense_forward(C.byref(a), None, 0, None) == INVALID
    assert says in L.petdense_last_error().decode()


@pytest.mark.parametrize('kw,says', [
    (dict(dtype=9), 'dtype'), (dict(activation=-1), 'activation'), (dict(m=-5), 'm must be'), (dict(k=0), 'k and n'),
    (dict(n=BIG), 'too large'), (dict(dy=None), 'dy'), (dict(lddy=31), 'dy'), (dict(saved=None), 'saved'),
    (dict(lds=31), 'saved'), (dict(kernel=None), 'dx needs'), (dict(ldk=31), 'dx needs'), (dict(lddx=63), 'dx needs'),
    (dict(x=None), 'dkernel needs'), (dict(ldx=63), 'dkernel needs'), (dict(lddk=31), 'stride'),
    (dict(x_exponents=0x8000, lde=1), 'exponents'), (dict(dresidual=0x8000, lddr=31), 'stride'),
    (dict(dx=0x1000), 'alias'), (dict(dkernel=0x2000), 'alias'), (dict(dresidual=0x4000, lddr=32), 'alias'),
])
def test_backward_refusals(kw, says):
    a = backward_args(**kw)
    assert L.petdense_backward_workspace(C.byref(a)) == 0
    assert L.petdense_backward(C.byref(a), None, 0, None) == INVALID
    assert says in L.petdense_last_error().decode()


def test_missing_small_and_unaligned_workspaces_are_refused():
    a = forward_args(m=32, k=8192, ldx=8192)
    need = L.petdense_forward_workspace(C.byref(a))
    assert need > 0                                    # a long contraction into few outputs is split
    for work, size in ((None, need), (0x10000, need - 1), (0x10010, need)):
        assert L.petdense_forward(C.byref(a), work, size, None) == INVALID
        assert 'workspace' in L.petdense_last_error().decode()
    b = backward_args(m=40000)                         # dP and the parts of its sums
    need = L.petdense_backward_workspace(C.byref(b))
    assert need > 0
    for work, size in ((None, need), (0x10000, need - 1), (0x10010, need)):
        assert L.petdense_backward(C.byref(b), work, size, None) == INVALID
        assert 'workspace' in L.petdense_last_error().decode()


def test_every_backward_pass_gets_a_plan():
    """With more tiles than one launch takes, dP goes through the workspace (a launch without a plan reads outside)."""
    for m, k, n in ((12288, 6144, 512), (8192, 8256, 24), (70000, 4096, 16), (16, 70000, 4096)):
        a = backward_args(m=m, k=k, n=n, lddy=n, ldx=k, ldk=n, lds=n, lddx=k, lddk=n)
        assert L.petdense_backward_workspace(C.byref(a)) >= m * n * 2


def test_null_arguments():
    assert L.petdense_forward(None, None, 0, None) == INVALID
    assert L.petdense_backward(None, None, 0, None) == INVALID
    assert L.petdense_forward_workspace(None) == 0 and L.petdense_backward_workspace(None) == 0


def test_no_rows_need_nothing():
    a = forward_args(m=0, x=None, y=None, kernel=None)
    assert L.petdense_forward_workspace(C.byref(a)) == 0
    assert L.petdense_forward(C.byref(a), None, 0, None) == 0


@pytest.mark.parametrize('kw,says', [
    (dict(dtype=5), 'dtype'), (dict(m=-1), 'm must be'), (dict(k=0), 'k >= 1'), (dict(ldx=99), 'stride'),
    (dict(ldc=99), 'stride'), (dict(lde=3), 'stride'), (dict(x=None), 'must be given'), (dict(codes=None), 'must be'),
    (dict(exps=None), 'must be given'),
])
def test_checkpoint_refusals(kw, says):
    v = dict(x=0x1000, ldx=100, m=10, k=100, dtype=1, codes=0x2000, ldc=100, exps=0x3000, lde=4)
    v.update(kw)
    rc = L.petdense_checkpoint(v['x'], v['ldx'], v['m'], v['k'], v['dtype'], v['codes'], v['ldc'], v['exps'], v['lde'],
                               None)
    assert rc == INVALID and says in L.petdense_last_error().decode()
    rc = L.petdense_restore(v['codes'], v['ldc'], v['exps'], v['lde'], v['m'], v['k'], v['dtype'], v['x'], v['ldx'],
                            None)
    assert rc == INVALID and says in L.petdense_last_error().decode()


def test_the_layers_refuse_cpu_tensors():
    x, w = torch.zeros(4, 8), torch.zeros(8, 3)
    for call in (lambda: layers.dense(x, w), lambda: layers.dense_backward(torch.zeros(4, 3), x, w),
                 lambda: layers.checkpoint_activations(x), lambda: layers.dense([1.0], w),
                 lambda: layers.ActivationCheckpoint(x.to(torch.float8_e4m3fn), torch.zeros(4, 1, dtype=torch.uint8),
                                                     torch.float32)):
        with pytest.raises(ValueError, match='CUDA'):
            call()


def test_packed_arguments_are_the_structs():
    f = _lib.PetdenseForwardArgs(*range(1, 19))
    assert bytes(f) == layers._FORWARD.pack(*range(1, 19))
    b = _lib.PetdenseBackwardArgs(*range(1, 24))
    assert bytes(b) == layers._BACKWARD.pack(*range(1, 24))


def test_row_views():
    def rows(t, what):
        return layers._rows(t)

    x = torch.zeros(6, 10)
    assert rows(x, 'x')[1] == 10 and rows(x[:, :4], 'x')[1] == 10 and rows(x[::2, :4], 'x')[1] == 20
    v, ld = rows(x.T, 'x')
    assert v.is_contiguous() and ld == 6
    v, ld = rows(torch.zeros(1, 4).expand(6, 4), 'x')          # rows that overlap are copied
    assert v.is_contiguous() and ld == 4
    assert rows(torch.zeros(2, 3, 4), 'x')[1] == 4 and rows(torch.zeros(5), 'x')[1] == 5
    v, ld = rows(torch.zeros(2, 3, 8)[:, :, :4], 'x')          # merged leading dimensions keep the row stride
    assert tuple(v.shape) == (6, 4) and ld == 8
    v, ld = rows(torch.zeros(2, 3, 4).transpose(0, 1), 'x')    # unmergeable ones are copied, in order
    assert tuple(v.shape) == (6, 4) and ld == 4
    v, ld = rows(torch.zeros(10)[::2], 'x')
    assert v.is_contiguous() and ld == 5
    assert rows(torch.zeros(0, 5), 'x')[1] == 5


def test_training_precisions_are_checked():
    from pet_posterior_distribution_amd.training import check_precision
    check_precision('float32', None)
    check_precision('bfloat16', None)
    check_precision('bfloat16', 'e4m3')
    for bad in (('float16', None), ('bf16', None), ('bfloat16', 'int8'), ('float32', 'e4m3')):
        with pytest.raises(ValueError):
            check_precision(*bad)
    assert L.pettrain_set_precision(None, 0, 0) == INVALID and L.pettrain_step_bytes(None) == 0


@pytest.mark.parametrize('kw', [
    dict(y=0x9000, bias=0x9000), dict(pre=0x2000, ldp=32), dict(pre=0x9000, ldp=32, bias=0x9000),
    dict(pre=0x9000, ldp=32, residual=0x9000, ldr=32), dict(pre=0x1000, ldp=32),
])
def test_forward_outputs_are_no_inputs(kw):
    a = forward_args(**kw)
    assert L.petdense_forward(C.byref(a), None, 0, None) == INVALID
    assert 'alias' in L.petdense_last_error().decode()


@pytest.mark.parametrize('kw', [
    dict(dx=0x8000, x_exponents=0x8000, lde=2), dict(dkernel=0x8000, x_exponents=0x8000, lde=2),
    dict(dresidual=0x5000, lddr=32), dict(dresidual=0x6000, lddr=32), dict(dbias=0x5000), dict(dbias=0x6000),
    dict(dkernel=0x5000), dict(dbias=0x4000), dict(dx=0x3000),
])
def test_backward_outputs_are_no_inputs_and_differ(kw):
    a = backward_args(**kw)
    assert L.petdense_backward(C.byref(a), None, 0, None) == INVALID
    assert 'alias' in L.petdense_last_error().decode()


@pytest.mark.parametrize('x,codes,exps', [(0x1000, 0x1000, 0x3000), (0x1000, 0x2000, 0x1000), (0x1000, 0x2000, 0x2000)])
def test_checkpoints_are_in_memory_of_their_own(x, codes, exps):
    assert L.petdense_checkpoint(x, 100, 10, 100, 1, codes, 100, exps, 4, None) == INVALID
    assert 'alias' in L.petdense_last_error().decode()
    if codes != exps:                       # two inputs may be one
        assert L.petdense_restore(codes, 100, exps, 4, 10, 100, 1, x, 100, None) == INVALID
        assert 'alias' in L.petdense_last_error().decode()


def test_the_largest_checkpoint_is_named():
    for m, k in ((BIG, 8), (8, BIG), (2 ** 31 - 65535, 8)):
        assert L.petdense_checkpoint(0x1000, BIG, m, k, 1, 0x2000, BIG, 0x3000, BIG, None) == INVALID
        assert '2^31 - 65536' in L.petdense_last_error().decode()
        assert L.petdense_restore(0x2000, BIG, 0x3000, BIG, m, k, 1, 0x1000, BIG, None) == INVALID
        assert '2^31 - 65536' in L.petdense_last_error().decode()


def test_a_gradient_through_an_output_is_refused():
    """Autograd does not record the layer: backward says so instead of leaving gradients out."""
    leaf = torch.ones(3, requires_grad=True)
    y, pre = layers._unrecorded(torch.zeros(3), torch.zeros(3))
    for out in (y, pre):
        with pytest.raises(RuntimeError, match='dense_backward'):
            (out * leaf).sum().backward()
    y = layers._unrecorded(torch.zeros(3))[0]
    y.mul_(2)                                           # written to like any other result
    dy, = torch.autograd.grad((y * leaf).sum(), y)      # what dense_backward takes
    assert torch.equal(dy, torch.ones(3)) and y.detach().numpy().shape == (3,)
