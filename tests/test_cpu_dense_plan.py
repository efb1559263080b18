"""CPU tests of the dense layer's plan: what its entries launch, from dense_api.cpp compiled for the host over launchers
that only write down what they are asked for (dense_plan.cpp), and the address rules that the kernels share with it."""
import ctypes as C
import os
import shutil
import subprocess

import pytest

from pet_posterior_distribution_amd import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, 'pet_posterior_distribution_amd', 'csrc')


@pytest.fixture(scope='module')
def plan(tmp_path_factory):
    hipcc = shutil.which('hipcc') or '/opt/rocm/bin/hipcc'
    out = str(tmp_path_factory.mktemp('plan') / 'libplan.so')
    subprocess.run([hipcc, '-x', 'hip', '--cuda-host-only', '-O1', '-std=c++17', '-fPIC', '-shared', '-I', CSRC, '-I',
                    os.path.join(ROOT, 'include'), os.path.join(ROOT, 'tests', 'dense_plan.cpp'),
                    os.path.join(CSRC, 'dense_api.cpp'), '-o', out], check=True, timeout=300)
    lib = C.CDLL(out)
    lib.plan_log.restype = lib.petdense_last_error.restype = C.c_char_p
    lib.plan_exponents_fit.argtypes = [C.c_int64]
    lib.plan_exponent_offset.argtypes = [C.c_int, C.c_int64, C.c_int]
    lib.plan_exponent_offset.restype = C.c_uint64
    for name in ('forward', 'backward'):
        w, f = getattr(lib, f'petdense_{name}_workspace'), getattr(lib, f'petdense_{name}')
        w.argtypes, w.restype = [C.c_void_p], C.c_size_t
        f.argtypes = [C.c_void_p, C.c_void_p, C.c_size_t, C.c_void_p]
    return lib


@pytest.mark.parametrize('bc', [64, 32])
def test_exponent_bytes_of_a_whole_step_are_reached_at_any_row_stride(plan, bc):
    """The exponents of a column slice keep the wide tensor's row stride: the step's last row then lies past what 32
    bits hold (65 rows of 70,000,000 bytes are enough), and the step has to be read by 64-bit offsets."""
    block = 3
    for lde in (4, 1 << 20, 1 << 23, 68174083, 68174084, 70000000, 1 << 28, (1 << 31) - 1, (1 << 31) + 5, 1 << 33):
        if not plan.plan_exponents_fit(lde):
            continue
        for r in range(bc):
            assert plan.plan_exponent_offset(r, lde, block) == r * lde + block, (lde, r)
    assert plan.plan_exponents_fit(128)          # dense exponents: the quick way


# ------------------------------------------------------------------------------------------------ the plan's launches
F32, BF16, F16 = 0, 1, 2
SIZE = {F32: 4, BF16: 2, F16: 2}
TILE = {0: 256, 1: 128, 2: 64, 3: 32, 4: 64}
FORWARD, INPUT_GRAD, KERNEL_GRAD = 0, 1, 2
DMA = 0


def launches(plan, name, args):
    """The launches of one call, as (kind, {field: number}); its workspace is an address that nothing reads."""
    need = getattr(plan, f'petdense_{name}_workspace')(C.byref(args))
    plan.plan_clear()
    rc = getattr(plan, f'petdense_{name}')(C.byref(args), 0x10000 if need else None, need, None)
    assert rc == 0, plan.petdense_last_error().decode()
    out = []
    for line in plan.plan_log().decode().splitlines():
        kind, *fields = line.split()
        out.append((kind, {k: int(v) for k, v in (f.split('=') for f in fields)}))
    return out


def forward(m, k, n, dtype, ldx=None, ldk=None, **kw):
    a = _lib.PetdenseForwardArgs(0x1000, 0x2000, 0x3000, None, 0x4000, None, ldx or k, ldk or n, 0, n, 0, m, k, n,
                                 dtype, 0, 0, 0)
    for key, v in kw.items():
        setattr(a, key, v)
    return a


def backward(m, k, n, dtype, activation=0, codes=False, **kw):
    a = _lib.PetdenseBackwardArgs(0x1000, 0x2000, 0x8000 if codes else None, 0x3000, 0x4000, 0x5000, 0x6000, 0x7000,
                                  None, n, k, -(-k // 32) if codes else 0, n, n, k, n, 0, m, k, n, dtype, activation, 0)
    for key, v in kw.items():
        setattr(a, key, v)
    return a


def check_products(log):
    """What DMA stages lies within the 31-bit offsets of a tile: its rows (contraction-contiguous), or the rows of one
    step (free-contiguous)."""
    seen = 0
    for kind, p in log:
        if kind not in ('product', 'pair') or p['loader'] != DMA:
            continue
        tile, size = TILE[p['tile']], SIZE[p['type']]
        step = 128 // size
        rows_a = step if p['layout'] == KERNEL_GRAD else tile
        rows_b = tile if p['layout'] == INPUT_GRAD else step
        if not p['q8']:                           # 8-bit inputs go through registers
            assert rows_a * p['lda'] * size < 2 ** 31, (kind, p)
            assert p['lda'] * size % 16 == 0, (kind, p)
        assert rows_b * p['ldb'] * size < 2 ** 31, (kind, p)
        assert p['ldb'] * size % 16 == 0, (kind, p)
        seen += 1
    return seen


@pytest.mark.parametrize('dtype', [BF16, F16, F32])
def test_what_dma_stages_lies_within_its_offsets(plan, dtype):
    """Contractions and layers longer than a DMA row may be: no copy of the same length either."""
    for k in (4_194_248, 4_300_000, 4_300_001, 5_000_000, 6_000_000, 2_097_144, 2_200_000, 2_200_001, 20_000_000):
        for m, n in ((1024, 1024), (512, 512), (70, 300), (3, 40)):
            check_products(launches(plan, 'forward', forward(m, k, n, dtype)))
    for n in (4_300_000, 4_300_001, 2_200_000, 2_200_003, 20_000_000, 20_000_003):
        for m, k in ((1024, 1024), (300, 64), (64, 72), (33, 9)):
            check_products(launches(plan, 'forward', forward(m, k, n, dtype)))
            for act in (0, 1, 2):
                for codes in (False, True):
                    check_products(launches(plan, 'backward', backward(m, k, n, dtype, act, codes)))
                    check_products(launches(plan, 'backward', backward(m, n, k, dtype, act, codes)))
                    check_products(launches(plan, 'backward', backward(m, k, n, dtype, act, codes, dresidual=0x9000,
                                                                       lddr=n)))
    # long strides of short rows are copied to short ones, and small rows are staged as they lie
    log = launches(plan, 'forward', forward(4096, 4096, 4096, dtype, ldx=30_000_000))
    assert check_products(log) == 1 and any(kind == 'pad' for kind, _ in log)
    assert check_products(launches(plan, 'forward', forward(4096, 4096, 4096, dtype))) == 1


@pytest.mark.parametrize('dtype', [BF16, F32])
def test_wide_layers_are_staged_by_dma(plan, dtype):
    """Free-contiguous operands are staged a step's rows at a time: theirs may be longer than a tile's rows."""
    n = 16_000_003 // SIZE[dtype]
    log = launches(plan, 'forward', forward(2048, 64, n, dtype))
    assert check_products(log) == 1 and any(kind == 'pad' for kind, _ in log)
    log = launches(plan, 'backward', backward(512, 64, n, dtype, 1))
    assert check_products(log) == 1                      # the kernel's gradient, from dP in the workspace


@pytest.mark.parametrize('dtype', [BF16, F32])
def test_column_sums_beside_a_join_leave_its_grid_in_bounds(plan, dtype):
    """A grid holds fewer than 2^32 threads, and 65,535 workgroups in y; a join of column sums by itself walks."""
    joined = 0
    for m, k, n in ((1, 1, 2 ** 28 + 8), (1, 1, 2 ** 27), (1376, 228, 34_629_222), (4, 3, 2 ** 26), (300, 256, 2 ** 25),
                    (2048, 256, 2 ** 24 + 64), (40, 48, 5000), (4096, 4096, 512)):
        for act in (0, 1):
            for kind, p in launches(plan, 'backward', backward(m, k, n, dtype, act)):
                if kind == 'join':
                    outputs = p['I'] * -(-p['J'] // 8) * (8 if p['splits'] > 2 else 1)
                    assert (-(-p['N'] // 16) + -(-outputs // 256)) * 256 < 2 ** 32, (m, k, n, p)
                elif kind == 'join_tiles':
                    row = p['b'] * p['b'] // 8 // 256
                    tiles = -(-p['I'] // p['b']) * -(-p['J'] // p['b']) - p['whole']
                    assert -(-p['N'] // (16 * row)) + tiles <= 65535, (m, k, n, p)
                joined += p.get('N') == n and kind in ('join', 'join_tiles', 'join_columns')
    assert joined


def test_outputs_that_are_not_asked_for_do_not_limit_a_call(plan):
    """2^23 tiles of 64 x 64 is the limit of an output that is asked for."""
    tall = dict(m=2 ** 29 + 100, k=64, n=8)                       # x's gradient would be too large
    assert launches(plan, 'backward', backward(**tall, dtype=BF16, dx=None))
    wide = dict(m=8, k=2 ** 20, n=2 ** 16)                        # the kernel's gradient would be
    assert launches(plan, 'backward', backward(**wide, dtype=BF16, dkernel=None))
    assert launches(plan, 'backward', backward(m=2, k=2 ** 20, n=2 ** 31 - 2 ** 17, dtype=BF16, dx=None, dkernel=None))
    for size, gone in ((tall, 'dkernel'), (wide, 'dx')):
        a = backward(**size, dtype=BF16, **{gone: None})
        assert plan.petdense_backward_workspace(C.byref(a)) == 0
        assert plan.petdense_backward(C.byref(a), None, 0, None) == _lib.PETDIFF_ERR_INVALID
        assert b'too many' in plan.petdense_last_error()


@pytest.mark.parametrize('dtype', [BF16, F32])
def test_copies_fit_one_launch(plan, dtype):
    """A copy's rows are filled up to whole pieces of 16 bytes: narrow rows move more than their values."""
    for m, k, n in ((2 ** 31 - 2 ** 17, 1, 1), (1_600_000_000, 1, 9), (1_000_000_000, 9, 17), (600_000_000, 3, 5)):
        for args in (backward(m, k, n, dtype, dx=None), backward(m, k, n, dtype, dx=None, codes=True)):
            pieces = sum(p['rows'] * (p['ldd'] * SIZE[dtype] // 16)
                         for kind, p in launches(plan, 'backward', args) if kind == 'pad')
            assert pieces + 256 < 2 ** 32, (m, k, n, pieces)
