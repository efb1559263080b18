"""GPU tests of the training step on the dense layer's operators (precision='bfloat16', activation_checkpoint).

Tolerances, from the number of roundings (2^-9 at most, 1.1e-3 in the mean square, each):
* activations: two operands a product, about ten products deep: 1.6e-3 sqrt(10) = 0.5 %.  The loss is 1 % off at most.
* gradients: as much again on the way back, and the units whose pre-activation lies within that 0.5 % of zero (a
  standard normal one: 0.2 % of them) switch their ReLU: sqrt(0.002) = 4.5 % of the gradient's 2-norm a layer, up to
  ten layers in quadrature: 14 %.  A variable's gradient is 20 % off at most in the 2-norm.
* 8-bit inputs of the kernel gradients: 2^-4 at most, 2^-4 / sqrt 3 = 3.6 % in the mean square a value; sums over
  positions keep the ratio: 6.25 % at most.  Nothing else reads them: every other gradient keeps its bits.
"""
import numpy as np
import pytest
import torch

from oracle import iddpm_ref as R
from oracle import train_ref as TR
from tests.test_gpu_train import batch, make, split

pytestmark = pytest.mark.gpu

S = R.schedule_tables(R.get_beta_schedule('cosine', 1000))


def trainer(precision, keep, seed=7, **kw):
    from pet_posterior_distribution_amd import Adam
    m = make(seed=seed, **kw)
    m.compile(optimizer=Adam(learning_rate=1e-3, clipnorm=1.5), precision=precision, activation_checkpoint=keep)
    return m, m._ensure_trainer()


def gradients(m, tr, data):
    x0, cond, t, noise = (torch.as_tensor(v, device=m.device) for v in data)
    loss = torch.empty(x0.shape[0], dtype=torch.float32, device=m.device)
    tr.compute_gradients(x0, cond, t, noise, loss=loss)
    return loss.cpu().numpy(), split(tr.gradients().cpu().numpy(), m.network.spec())


def far(a, b):
    return np.linalg.norm(a.astype(np.float64) - b) / (np.linalg.norm(b) + 1e-30)


@pytest.mark.parametrize('lv,param', [('learn_ranged', 'eps'), ('', 'x0')])
@pytest.mark.parametrize('keep', [None, 'e4m3'])
def test_loss_and_gradients_vs_oracle(lv, param, keep):
    m, tr = trainer('bfloat16', keep, learn_variance=lv, parameterization=param)
    P = {k: v.astype(np.float64) for k, v in m.network.weights.items()}
    data = batch(B=4)
    loss, g = gradients(m, tr, data)
    rl, _, _, G = TR.train_loss_and_grads(P, S, *data, learn_variance=lv, parameterization=param)
    assert np.abs(loss - rl).max() <= 0.01 * np.abs(rl).max()
    off = {k: far(g[k], G[k]) for k in G}
    assert max(off.values()) <= 0.2, {k: v for k, v in off.items() if v > 0.2}


def test_checkpoints_change_the_kernel_gradients_alone():
    data = batch(B=16, seed=4)
    (m1, t1), (m2, t2) = trainer('bfloat16', None), trainer('bfloat16', 'e4m3')
    l1, g1 = gradients(m1, t1, data)
    l2, g2 = gradients(m2, t2, data)
    np.testing.assert_array_equal(l1, l2)
    through = [k for k in g1 if k.endswith('.kernel') and ('conv' in k or 'res' in k or 'cond_enc' in k)]
    assert len(through) == 4 + 4 * 2 + 3 * 3
    for k in g1:
        if k in through:
            assert 0 < far(g2[k], g1[k]) <= 0.0625, (k, far(g2[k], g1[k]))
        else:
            np.testing.assert_array_equal(g1[k], g2[k], err_msg=k)


def test_less_memory():
    data = batch(B=64, seed=6)
    held = []
    for precision, keep in (('float32', None), ('bfloat16', None), ('bfloat16', 'e4m3')):
        m, tr = trainer(precision, keep)
        gradients(m, tr, data)
        held.append(tr.step_bytes)
    assert held[2] < held[1] < held[0], held


def test_a_change_of_precision_frees_what_the_other_one_held():
    from pet_posterior_distribution_amd import _lib
    L = _lib.lib()
    data = batch(B=16, seed=6)
    kinds = [('float32', None), ('bfloat16', None), ('bfloat16', 'e4m3')]
    code = {kinds[0]: (0, 0), kinds[1]: (1, 0), kinds[2]: (1, 1)}
    held = {}
    for kind in kinds:
        m, tr = trainer(*kind)
        gradients(m, tr, data)
        held[kind] = tr.step_bytes
    for before in kinds:
        for after in kinds:
            m, tr = trainer(*before)
            gradients(m, tr, data)
            assert L.pettrain_set_precision(tr.handle, *code[after]) == 0
            gradients(m, tr, data)
            assert tr.step_bytes == held[after], (before, after)


def test_runs_repeat_and_batches_may_change():
    """Growing and shrinking batches: the buffers and the workspace follow, and results do not depend on what ran
    before."""
    runs = []
    for sizes in ((3, 40, 5, 40), (40, 3, 5, 3, 40)):
        m, tr = trainer('bfloat16', 'e4m3', seed=9)
        out = {}
        for B in sizes:
            out[B] = gradients(m, tr, batch(B=B, seed=B))
        runs.append(out)
    for B in (3, 5, 40):
        np.testing.assert_array_equal(runs[0][B][0], runs[1][B][0])
        for k in runs[0][B][1]:
            np.testing.assert_array_equal(runs[0][B][1][k], runs[1][B][1][k], err_msg=k)


def test_precision_can_be_changed_and_fp32_keeps_its_results():
    data = batch(B=4, seed=8)
    m0, t0 = trainer('float32', None, seed=3)
    want = gradients(m0, t0, data)
    m, tr = trainer('bfloat16', 'e4m3', seed=3)
    first = gradients(m, tr, data)
    from pet_posterior_distribution_amd import _lib
    L = _lib.lib()
    assert L.pettrain_set_precision(tr.handle, 0, 1) == _lib.PETDIFF_ERR_INVALID      # e4m3 without bf16
    assert L.pettrain_set_precision(tr.handle, 2, 0) == _lib.PETDIFF_ERR_INVALID
    assert L.pettrain_set_precision(tr.handle, 0, 0) == 0
    got = gradients(m, tr, data)
    np.testing.assert_array_equal(got[0], want[0])
    for k in want[1]:
        np.testing.assert_array_equal(got[1][k], want[1][k], err_msg=k)
    assert L.pettrain_set_precision(tr.handle, 1, 1) == 0
    again = gradients(m, tr, data)
    for k in first[1]:
        np.testing.assert_array_equal(again[1][k], first[1][k], err_msg=k)


def test_fit_and_test_step_in_bf16():
    from pet_posterior_distribution_amd import Adam
    m = make(lr=1e-4)
    m.compile(optimizer=Adam(learning_rate=1e-4, clipnorm=1.5), precision='bfloat16', activation_checkpoint='e4m3')
    rng = np.random.default_rng(2)
    x0 = rng.standard_normal((48, 48, 2)).astype(np.float32)
    cond = np.abs(rng.standard_normal((48, 49, 54))).astype(np.float32)
    before = {k: v.copy() for k, v in m.network.weights.items()}
    hist = m.fit(x0, cond, batch_size=16, epochs=1, validation_split=0.34)
    assert np.isfinite(hist['loss']).all() and np.isfinite(hist['val_loss']).all()
    m._sync_trained_weights()
    assert any(not np.array_equal(before[k], m.network.weights[k]) for k in before)
    assert all(np.isfinite(v).all() for v in m.network.weights.values())
