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
    lib.plan_whole_step.argtypes = [C.c_int, C.c_int, C.c_int, C.c_int64, C.c_int64, C.c_int64]
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
    bits hold (65 rows of 70,000,000 bytes are enough), and the step has to be one that is read by 64-bit offsets."""
    block = 3
    for lde in (4, 1 << 20, 1 << 23, 68174083, 68174084, 70000000, 1 << 28, (1 << 31) - 1, (1 << 31) + 5, 1 << 33):
        if not plan.plan_whole_step(1, bc + 1, bc, 4096, 4096, lde):
            continue
        for r in range(bc):
            assert plan.plan_exponent_offset(r, lde, block) == r * lde + block, (lde, r)
    assert plan.plan_whole_step(1, bc + 1, bc, 4096, 4096, 128)          # dense exponents: the quick way
