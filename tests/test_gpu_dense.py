"""GPU tests of the dense layer's operators (petdense_*, layers.py) against their formulas in 64 bits.

Tolerances, elementwise and derived, with u = eps / 2 of the output's type and S = the sum of the magnitudes of the
terms of an output (from the 64-bit reference):
* a product of C terms in fp32: every addition is off by at most 2^-23 of a partial sum that S bounds, the terms
  themselves by 2^-24: (C + 4) 2^-23 S covers the sum, a split's join, bias and residual;
* activations have slope at most 1.13 (GELU) and are evaluated to 4e-7 (|v| + 1): A = 1.13 P + 4e-7 (|v| + 1);
* rounding the output: u |y|, and 2^-25 for fp16 outputs below its normal range;
* a 16-bit layer's dP is rounded once more before the products: u |dP| through |W| and |X|.
"""
import ctypes as C
import os
import subprocess
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
TYPES = [BF16, F16, F32]
ACTS = [None, 'relu', 'gelu', 'silu']
E23 = 2.0 ** -23

# one row and value, a few rows, odd sizes, sizes of whole tiles, a long contraction that is split, narrow outputs
SHAPES = [(1, 1, 1), (1, 54, 256), (2, 300, 33), (7, 129, 64), (8, 64, 6), (9, 65, 33), (64, 64, 64), (77, 40, 136),
          (130, 129, 257), (256, 256, 256), (257, 312, 128), (49 * 3, 33, 48), (40, 4100, 64), (24, 8000, 16),
          (300, 72, 6)]
# outputs of many tiles
WIDE = [(2048, 128, 2048), (2040, 72, 4104)]
# more tiles than one launch of the whole backward pass takes
MANY = [(8192, 8256, 24)]


def rand(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device='cuda').manual_seed(seed)
    return (torch.randn(*shape, generator=g, device='cuda') * scale).to(dtype)


def act64(p, act):
    if act == 'relu':
        return torch.where(p < 0, torch.zeros_like(p), p)
    if act == 'gelu':
        return p * torch.special.ndtr(p)
    if act == 'silu':
        return p * torch.sigmoid(p)
    return p


def act_grad64(v, act):
    if act == 'relu':
        return torch.where(v <= 0, torch.zeros_like(v), torch.ones_like(v))
    if act == 'gelu':
        return torch.special.ndtr(v) + v * torch.exp(-v * v / 2) / (2 * torch.pi) ** 0.5
    if act == 'silu':
        s = torch.sigmoid(v)
        return s * (1 + v * (1 - s))
    return torch.ones_like(v)


def half_step(t):
    return torch.finfo(t).eps / 2


def close(got, ref, tol, what):
    tol = tol + half_step(got.dtype) * (ref.abs() + tol) + (2.0 ** -25 if got.dtype == F16 else 1e-37)
    err = (got.double() - ref).abs()
    worst = (err / tol).max().item() if err.numel() else 0.0
    assert worst <= 1.0, f'{what}: {worst:.3g} of its tolerance, max error {err.max().item():.3g}'


def check_forward(x, w, b, act, r, pre, out_dtype=None):
    from pet_posterior_distribution_amd import dense
    got = dense(x, w, b, activation=act, residual=r, return_preactivation=pre, out_dtype=out_dtype)
    y, p_got = got if pre else (got, None)
    x64, w64 = x.double().reshape(-1, x.shape[-1]), w.double()
    n, k = w.shape[1], w.shape[0]
    p, s = x64 @ w64, x64.abs() @ w64.abs()
    for extra in (b, r):
        if extra is not None:
            e = extra.double().reshape(-1, n) if extra.dim() > 1 else extra.double()
            p, s = p + e, s + e.abs()
    lead = tuple(x.shape[:-1]) + (n,)
    assert tuple(y.shape) == lead and y.dtype == (out_dtype or x.dtype)
    tol = (k + 4) * E23 * s
    if pre:
        close(p_got.reshape(-1, n), p, tol, 'pre-activation')
    if act:
        tol = 1.13 * tol + 4e-7 * (p.abs() + 1)
    close(y.reshape(-1, n), act64(p, act), tol, 'output')
    return y


def reference_backward(dy, x64, w, act, saved):
    """(dX, dW, db, dP) in 64 bits, and the tolerances of each before the last rounding."""
    t = dy.dtype
    n = dy.shape[-1]
    d = dy.double().reshape(-1, n)
    m, k = x64.shape
    w64 = w.double()
    e_dp = torch.zeros_like(d)
    dp = d
    if act:
        v = saved.double().reshape(-1, n)
        dp = d * act_grad64(v, act)
        if act != 'relu':
            e_dp = d.abs() * 1e-6 * (v.abs() + 1)
    e_in = e_dp if act in (None, 'relu') or t == F32 else e_dp + half_step(t) * dp.abs() * 1.01 + \
        (2.0 ** -25 if t == F16 else 0)
    mag = dp.abs() + e_in
    t_x = e_in @ w64.abs().T + (n + 4) * E23 * (mag @ w64.abs().T)
    t_w = x64.abs().T @ e_in + (m + 4) * E23 * (x64.abs().T @ mag)
    t_b = e_dp.sum(0) + (m + 260) * E23 * dp.abs().sum(0)
    return (dp @ w64.T, x64.T @ dp, dp.sum(0), dp), (t_x, t_w, t_b, e_dp)


def check_backward(dy, x, w, act, saved, grad_dtype=None, residual=True, x64=None):
    from pet_posterior_distribution_amd import dense_backward
    g = dense_backward(dy, x, w, activation=act, saved=saved, need_residual=residual, grad_dtype=grad_dtype)
    n, k = w.shape[1], w.shape[0]
    x64 = x.double().reshape(-1, k) if x64 is None else x64
    ref, tol = reference_backward(dy, x64, w, act, saved)
    assert g.x.dtype == dy.dtype and g.kernel.dtype == g.bias.dtype == (grad_dtype or dy.dtype)
    assert tuple(g.x.shape) == tuple(dy.shape[:-1]) + (k,)
    close(g.x.reshape(-1, k), ref[0], tol[0], 'dx')
    close(g.kernel, ref[1], tol[1], 'dkernel')
    close(g.bias, ref[2], tol[2], 'dbias')
    if residual:
        assert g.residual.dtype == dy.dtype and g.residual.shape == dy.shape
        close(g.residual.reshape(-1, n), ref[3], tol[3], 'dresidual')
    else:
        assert g.residual is None
    return g


def inputs(m, k, n, t, seed=1):
    return (rand((m, k), t, seed), rand((k, n), t, seed + 1, k ** -0.5), rand((n,), t, seed + 2),
            rand((m, n), t, seed + 3), rand((m, n), t, seed + 4))


@pytest.mark.parametrize('t', TYPES, ids=str)
@pytest.mark.parametrize('m,k,n', SHAPES + WIDE)
def test_forward(m, k, n, t):
    x, w, b, r, _ = inputs(m, k, n, t)
    i = SHAPES.index((m, k, n)) if (m, k, n) in SHAPES else 0
    for j, act in enumerate(ACTS):
        # every activation meets every mix of bias and residual over the shapes
        check_forward(x, w, b if (i + j) % 3 else None, act, r if (i + j) % 2 else None, pre=(i + j) % 4 < 2)


@pytest.mark.parametrize('t', TYPES, ids=str)
@pytest.mark.parametrize('m,k,n', [(1, 8000, 16), (2, 5000, 100), (2, 4100, 64), (1, 1024, 4096), (1, 2819, 10),
                                   (2, 1023, 31)])
def test_one_and_two_rows(m, k, n, t):
    """One workgroup's whole contraction, and contractions that several share."""
    x, w, b, r, dy = inputs(m, k, n, t)
    for j, act in enumerate(ACTS):
        check_forward(x, w, b if j % 2 else None, act, r if j < 2 else None, pre=j in (1, 2))
        check_backward(dy, x, w, act, None if act is None else r)


@pytest.mark.parametrize('t', TYPES, ids=str)
def test_tiles_that_one_workgroup_walks(t):
    """297 tiles of 256 x 256, of which the last row and column are cut, on 256 compute units."""
    x, w, b, r, _ = inputs(8200, 2048, 2056, t)
    check_forward(x, w, b, 'gelu', r, pre=True)
    check_forward(x, w, None, 'relu', None, pre=False)
    y = check_forward(x, w, b, None, None, pre=False)
    from pet_posterior_distribution_amd import dense
    for rep in range(3):
        assert torch.equal(dense(x, w, b), y)


@pytest.mark.parametrize('t', [BF16, F16], ids=str)
def test_forward_fp32_outputs_and_bias(t):
    x, w, b, r, _ = inputs(150, 96, 72, t)
    for act in ACTS:
        y = check_forward(x, w, b.float() * 1.001, act, r, True, out_dtype=F32)
        assert y.dtype == F32
    check_forward(x[:3], w, b.float() * 1.001, 'gelu', r[:3], True, out_dtype=F32)


@pytest.mark.parametrize('t', [BF16, F16], ids=str)
def test_the_backward_pass_of_fp32_outputs_is_the_layers(t):
    """A 16-bit layer's backward pass takes dy and saved in its own type, whatever its outputs had."""
    from pet_posterior_distribution_amd import dense, dense_backward
    x, w, b, _, _ = inputs(150, 96, 72, t)
    dy = rand((150, 72), F32, 9)
    _, pre = dense(x, w, b, activation='gelu', return_preactivation=True, out_dtype=F32)
    for bad in (dict(dy=dy, saved=pre), dict(dy=dy.to(t), saved=pre)):
        with pytest.raises(ValueError, match='must be'):
            dense_backward(bad['dy'], x, w, activation='gelu', saved=bad['saved'])
    check_backward(dy.to(t), x, w, 'gelu', pre.to(t), grad_dtype=F32)


@pytest.mark.parametrize('t', TYPES, ids=str)
@pytest.mark.parametrize('m,k,n', SHAPES + WIDE)
def test_backward(m, k, n, t):
    x, w, _, p, dy = inputs(m, k, n, t)
    for act in ACTS:
        saved = None if act is None else (p.clamp(min=0) if act == 'relu' else p)
        check_backward(dy, x, w, act, saved, residual=act in ('relu', 'gelu'))


@pytest.mark.parametrize('act', [None, 'relu'])
@pytest.mark.parametrize('m,k,n', MANY)
def test_backward_of_many_tiles(m, k, n, act):
    x, w, _, p, dy = inputs(m, k, n, BF16)
    check_backward(dy, x, w, act, None if act is None else p, residual=False)


@pytest.mark.parametrize('act', [None, 'relu', 'gelu'])
def test_backward_long_sums_and_fp32_gradients(act):
    """Many rows into few gradients: the rows are split, and the parts joined in fp32."""
    for t in (BF16, F16):
        x, w, _, p, dy = inputs(20011, 48, 56, t)
        check_backward(dy, x, w, act, None if act is None else p, grad_dtype=F32)


def test_gradients_against_differences():
    """dX, dW, db and dR are the derivatives of sum(dense(...) * dy): fp32, central differences of the 64-bit formula
    along random directions (the difference quotient is off by about h^2 = 1e-8 of third derivatives)."""
    from pet_posterior_distribution_amd import dense, dense_backward
    for act in ACTS:
        x, w, b, r, dy = inputs(33, 20, 17, F32, seed=40)
        _, pre = dense(x, w, b, activation=act, residual=r, return_preactivation=True)
        g = dense_backward(dy, x, w, activation=act, saved=pre, need_residual=True)
        args = [v.double() for v in (x, w, b, r)]

        def loss(a):
            return (act64(a[0] @ a[1] + a[2] + a[3], act) * dy.double()).sum()

        for i, gi in enumerate((g.x, g.kernel, g.bias, g.residual)):
            d = rand(tuple(args[i].shape), F32, 50 + i).double()
            h = 1e-4
            if act == 'relu':      # no kink between the two points: only where every |P| is past the step
                base = args[0] @ args[1] + args[2] + args[3]
                step = [torch.zeros_like(a) for a in args]
                step[i] = d * h
                move = step[0] @ args[1] + args[0] @ step[1] + step[2] + step[3]
                h *= min(1.0, 0.5 * (base.abs() / (move.abs() + 1e-30)).min().item())
            up = [a + d * h if j == i else a for j, a in enumerate(args)]
            dn = [a - d * h if j == i else a for j, a in enumerate(args)]
            num = ((loss(up) - loss(dn)) / (2 * h)).item()
            ana = (gi.double() * d).sum().item()
            scale = (gi.double().abs() * d.abs()).sum().item()
            assert abs(num - ana) <= 2e-5 * scale, (act, i, num, ana)


def test_views_strides_and_leading_dimensions():
    """Row strides (aligned and odd), merged and unmergeable leading dimensions, transposed kernels, broadcast
    residuals and gradients: NaN in the gaps stays where it is."""
    for t in (BF16, F32):
        for gap in (8, 3):
            wide = torch.full((66, 64 + gap), float('nan'), dtype=t, device='cuda')
            wide[:, :64] = rand((66, 64), t, 1)
            x = wide[:, :64]
            wk = torch.full((64, 40 + gap), float('nan'), dtype=t, device='cuda')
            wk[:, :40] = rand((64, 40), t, 2, 0.125)
            w = wk[:, :40]
            p = torch.full((66, 40 + gap), float('nan'), dtype=t, device='cuda')
            p[:, :40] = rand((66, 40), t, 3)
            p = p[:, :40]
            check_forward(x, w, None, 'gelu', p, True)
            check_backward(p, x, w, 'silu', p)
            check_forward(x[5:11], w, None, None, p[5:11], False)
        x3 = rand((4, 48, 24), t, 4)
        w = rand((32, 24), t, 5).T
        check_forward(x3, w, None, 'relu', rand((4, 48, 32), t, 6), False)
        check_forward(x3.transpose(0, 1), w, None, 'relu', None, False)
        check_forward(x3[:, 3:20], w, None, 'silu', None, True)
        dy = rand((1, 32), t, 7).expand(4 * 48, 32)                       # the gradient of a sum over rows
        check_backward(dy, x3.reshape(192, 24), w, None, None)
        check_forward(rand((24,), t, 8), w, rand((32,), t, 9), None, None, False)
        check_forward(x3.reshape(192, 24), w, None, None, rand((32,), t, 9).expand(192, 32), False)


def test_a_contraction_longer_than_a_tile_row_reads_no_neighbour():
    """Rows end inside a tile's row of 64 values: what lies behind them (the next row, NaN) must not enter."""
    for t in TYPES:
        for k in (1, 8, 31, 56, 63, 65, 72, 120):
            buf = torch.full((140 * (k + 8),), float('nan'), dtype=t, device='cuda')
            x = buf.view(140, k + 8)[:, :k]
            x.copy_(rand((140, k), t, k))
            w = rand((k, 24), t, k + 1, k ** -0.5)
            check_forward(x, w, None, None, None, False)
            check_backward(rand((140, 24), t, 3), x, w, None, None)


def test_not_finite_values_stay_in_their_rows_and_columns():
    from pet_posterior_distribution_amd import dense, dense_backward
    for t in TYPES:
        for m, k, n in ((200, 64, 72), (5, 33, 17)):
            x, w, b, _, dy = inputs(m, k, n, t)
            x[2, 5] = float('nan')
            x[4, 6] = float('inf')
            y = dense(x, w, b, activation='relu')
            ref = act64(x.double() @ w.double() + b.double(), 'relu')
            assert torch.equal(torch.isnan(y), torch.isnan(ref))
            assert torch.equal(torch.isinf(y), torch.isinf(ref))
            assert torch.isnan(y[2]).all() and torch.isfinite(y[[0, 1, 3]]).all()
            dy[1, 3] = float('nan')
            g = dense_backward(dy, inputs(m, k, n, t)[0], w, need_residual=True)
            assert torch.isnan(g.x[1]).all() and torch.isfinite(g.x[2:]).all() and torch.isfinite(g.x[0]).all()
            bad = torch.zeros(n, dtype=torch.bool, device='cuda')
            bad[3] = True
            assert torch.equal(torch.isnan(g.bias), bad) and torch.isnan(g.kernel[:, 3]).all()
            assert torch.isfinite(g.kernel[:, ~bad]).all()


def test_saved_values_of_relu_may_be_input_or_output():
    from pet_posterior_distribution_amd import dense, dense_backward
    x, w, b, _, dy = inputs(90, 40, 50, BF16)
    y, pre = dense(x, w, b, activation='relu', return_preactivation=True)
    one = dense_backward(dy, x, w, activation='relu', saved=y)
    two = dense_backward(dy, x, w, activation='relu', saved=pre)
    for a, c in zip(one[:3], two[:3]):
        assert torch.equal(a, c)


def test_no_rows():
    from pet_posterior_distribution_amd import checkpoint_activations, dense, dense_backward
    for t in TYPES:
        w = rand((24, 16), t, 1)
        x = torch.empty(0, 24, dtype=t, device='cuda')
        y, p = dense(x, w, activation='gelu', return_preactivation=True)
        assert y.shape == p.shape == (0, 16)
        g = dense_backward(torch.empty(0, 16, dtype=t, device='cuda'), x, w, activation='relu', saved=y,
                           need_residual=True, grad_dtype=F32)
        assert g.x.shape == (0, 24) and g.residual.shape == (0, 16)
        assert not g.kernel.any() and not g.bias.any() and g.kernel.shape == (24, 16)
        c = checkpoint_activations(x)
        assert c.restore().shape == (0, 24) and c.exponents.shape == (0, 1)


def test_only_what_is_asked_for():
    from pet_posterior_distribution_amd import dense_backward
    x, w, _, p, dy = inputs(130, 72, 40, BF16)
    full = dense_backward(dy, x, w, activation='gelu', saved=p, need_residual=True)
    for i in range(4):
        need = [j == i for j in range(4)]
        g = dense_backward(dy, x, w, activation='gelu', saved=p, need_x=need[0], need_kernel=need[1],
                           need_bias=need[2], need_residual=need[3])
        for j in range(4):
            assert (g[j] is not None) == need[j]
        assert torch.equal(g[i], full[i])


def test_gradients_are_refused_where_autograd_would_drop_them():
    from pet_posterior_distribution_amd import dense, dense_backward
    x, w, b, r, dy = inputs(130, 72, 40, BF16)
    plain = dense(x, w, b, activation='gelu', residual=r, return_preactivation=True)
    for i, t in enumerate((x, w, b, r)):
        t.requires_grad_()
        y, pre = dense(x, w, b, activation='gelu', residual=r, return_preactivation=True)
        assert torch.equal(y, plain[0]) and torch.equal(pre, plain[1])
        with pytest.raises(RuntimeError, match='dense_backward'):
            y.float().sum().backward()
        assert t.grad is None
        # the gradient with respect to the output is what dense_backward takes; its own results have no history
        g, = torch.autograd.grad((y.float() * dy.float()).sum(), y)
        got = dense_backward(g, x, w, activation='gelu', saved=pre, need_residual=True)
        assert not any(v.requires_grad for v in got)
        with torch.no_grad():
            assert not dense(x, w, b, residual=r).requires_grad
        t.requires_grad_(False)
    assert not dense(x, w, b, residual=r).requires_grad


def test_rows_between_and_behind_the_outputs_are_left_as_they_were():
    """C entry with output strides wider than the rows, and spare rows behind them."""
    from pet_posterior_distribution_amd import _lib
    from pet_posterior_distribution_amd.layers import _check, _stream
    L = _lib.lib()
    dev = torch.device('cuda', 0)
    for t, code in ((BF16, 1), (F32, 0)):
        for m, k, n in ((37, 40, 56), (130, 24, 30), (5, 24, 30)):
            x, w, _, _, dy = inputs(m, k, n, t)
            y = torch.full((m + 3, n + 5), 7.0, dtype=t, device=dev)
            a = _lib.PetdenseForwardArgs(x.data_ptr(), w.data_ptr(), None, None, y.data_ptr(), None, k, n, 0, n + 5, 0,
                                         m, k, n, code, 0, 0, 0)
            nb = L.petdense_forward_workspace(C.byref(a))
            ws = torch.empty(max(nb, 1), dtype=torch.uint8, device=dev)
            _check(L.petdense_forward(C.byref(a), ws.data_ptr(), nb, _stream(dev)), 'dense')
            assert (y[m:] == 7).all() and (y[:, n:] == 7).all()
            close(y[:m, :n], x.double() @ w.double(), (k + 4) * E23 * (x.double().abs() @ w.double().abs()), 'output')
            gx = torch.full((m + 3, k + 5), 7.0, dtype=t, device=dev)
            gk = torch.full((k + 3, n + 5), 7.0, dtype=t, device=dev)
            gb = torch.full((n + 3,), 7.0, dtype=t, device=dev)
            bw = _lib.PetdenseBackwardArgs(dy.data_ptr(), x.data_ptr(), None, w.data_ptr(), None, gx.data_ptr(),
                                           gk.data_ptr(), gb.data_ptr(), None, n, k, 0, n, 0, k + 5, n + 5, 0, m, k, n,
                                           code, 0, 0)
            nb = L.petdense_backward_workspace(C.byref(bw))
            ws = torch.empty(max(nb, 1), dtype=torch.uint8, device=dev)
            _check(L.petdense_backward(C.byref(bw), ws.data_ptr(), nb, _stream(dev)), 'dense_backward')
            assert (gx[m:] == 7).all() and (gx[:, k:] == 7).all() and (gb[n:] == 7).all()
            assert (gk[k:] == 7).all() and (gk[:, n:] == 7).all()
            ref, tol = reference_backward(dy, x.double(), w, None, None)
            close(gx[:m, :k], ref[0], tol[0], 'dx')
            close(gk[:k, :n], ref[1], tol[1], 'dkernel')
            close(gb[:n], ref[2], tol[2], 'dbias')


@pytest.mark.parametrize('t,out', [(BF16, BF16), (F16, F16), (BF16, F32), (F16, F32), (F32, F32)], ids=str)
def test_the_lower_tail_of_gelu(t, out):
    """x Phi(x) from -3 down to where the type ends, relative to itself.
    fp32: the argument x / sqrt 2 is off by 2^-24 and 2^-25 of itself, which is x^2 times as much of Phi; the
    complementary error function and the two products after it by less than 8 2^-23.
    16-bit layers: Phi is off by 2^-16 of itself (the fit 4e-6, the exponent's two roundings x^2 2^-24, 1e-5 at -13)."""
    from pet_posterior_distribution_amd import dense, dense_backward
    v = torch.linspace(-13, -3, 8000, device='cuda').to(t)
    one = torch.ones(1, 8, dtype=t, device='cuda')
    v6 = v.double()
    cdf = 0.5 * torch.special.erfc(-v6 * 0.5 ** 0.5)             # (torch's ndtr cancels below -7, in 64 bits too)
    ref, pdf = v6 * cdf, torch.exp(-v6 * v6 / 2) / (2 * torch.pi) ** 0.5
    off = (v6 * v6 + 8) * E23 if t == F32 else torch.full_like(v6, 2.0 ** -16)

    def same(got, want, tol, what):
        tol = tol + half_step(got.dtype) * (want.abs() + tol) + (2.0 ** -25 if got.dtype == F16 else 1e-37)
        worst = ((got.double() - want).abs() / tol).max().item()
        assert worst <= 1.0, f'{what}: {worst:.3g} of its tolerance'

    y = dense(v[:, None], one, activation='gelu', out_dtype=out)                        # a tile's epilogue
    for j in (0, 7):
        same(y[:, j], ref, off * ref.abs(), 'tiles')
    y = dense(one[:, :1].expand(2, 1), v[None], activation='gelu', out_dtype=out)        # few rows
    same(y[1], ref, off * ref.abs(), 'rows')
    if out == t:
        g = dense_backward(torch.ones(8000, 1, dtype=t, device='cuda'), v[:, None], one[:, :1], activation='gelu',
                           saved=v[:, None], need_residual=True)
        same(g.residual[:, 0], cdf + v6 * pdf, 2 * off * (cdf + v6.abs() * pdf), 'gradient')


# ---------------------------------------------------------------------------------------------------- checkpoints
def power(e):
    """2^e in 64 bits, exactly (torch.exp2 and torch.ldexp of 64-bit GPU tensors may be off by a bit)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def quantize64(x):
    """(restored values in 64 bits, exponent bytes) by the definition."""
    m, k = x.shape
    nb = -(-k // 32)
    x64 = x.double()
    pad = torch.zeros(m, nb * 32, dtype=torch.float64, device=x.device)
    pad[:, :k] = x64
    b = pad.view(m, nb, 32)
    fin = torch.isfinite(b)
    top = torch.where(fin, b.abs(), torch.zeros_like(b)).amax(-1)
    mant, e = torch.frexp(top)
    big = torch.where(mant <= 0.875, e - 9, e - 8).clamp(min=-117)
    big = torch.where(top == 0, torch.full_like(big, -117), big)
    v = b * power(-big)[..., None]
    step = torch.full_like(v, 2.0 ** -9)
    for e in range(-5, 9):                                    # e4m3's binades
        step = torch.where(v.abs() >= 2.0 ** e, 2.0 ** (e - 3), step)
    q = torch.round(v / step) * step
    lim = torch.where(big == (8 if x.dtype == F16 else 120), 240.0, 448.0)[..., None]
    q = torch.where(fin, q.clamp(-lim, lim), torch.full_like(q, float('nan')))
    return (q * power(big)[..., None]).view(m, -1)[:, :k], (big + 127).to(torch.uint8)


def check_checkpoint(x):
    from pet_posterior_distribution_amd import checkpoint_activations
    c = checkpoint_activations(x)
    ref, e = quantize64(x.reshape(-1, x.shape[-1]))
    assert c.codes.shape == x.shape and c.dtype == x.dtype
    assert torch.equal(c.exponents.reshape(e.shape), e)
    back = c.restore()
    assert back.shape == x.shape and back.dtype == x.dtype
    got = back.double().reshape(ref.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    ok = ~torch.isnan(ref)
    # exact, but for fp16 below its normal range: half of 2^-24
    assert ((got - ref).abs()[ok] <= (2.0 ** -25 if x.dtype == F16 else 0.0)).all()
    assert torch.isfinite(back[torch.isfinite(x)]).all()
    return c


@pytest.mark.parametrize('t', TYPES, ids=str)
@pytest.mark.parametrize('m,k', [(1, 1), (1, 31), (3, 32), (5, 33), (257, 615), (64, 256), (33, 1537), (2, 40000)])
def test_checkpoint(m, k, t):
    x = rand((m, k), F32, k) * torch.exp(rand((m, 1), F32, m) * 3)
    x[0, 0] = 0
    check_checkpoint(x.clamp(-6e4, 6e4).to(t))


@pytest.mark.parametrize('t', TYPES, ids=str)
def test_checkpoint_extremes(t):
    f = torch.finfo(t)
    x = torch.zeros(16, 64, dtype=t, device='cuda')
    x[1, 3], x[1, 4] = f.max, -f.max                                    # restored as finite values
    x[2] = f.tiny
    x[3, :8] = torch.tensor([1, 1.75, 1.7500001, 2, 448, 449, 3.5, -3.5], device='cuda').to(t)
    x[4, 0] = 448
    x[5, 0] = 450 if t != BF16 else 452                                  # just past 448: the next exponent
    x[6, 0], x[6, 1], x[6, 2], x[6, 40] = float('nan'), float('inf'), 1.0, float('-inf')
    x[7] = float('nan')
    x[8, 0], x[8, 1] = f.max, f.smallest_normal
    x[9, :32] = rand((32,), t, 1) * f.max / 8
    x[10, 0], x[10, 1] = f.max / 2, f.max / 4
    x[11] = torch.linspace(-1, 1, 64, device='cuda').to(t)               # ties and subnormal codes
    x[12, :] = torch.exp2(-torch.arange(64, device='cuda').float() / 3).to(t)
    x[13, 0] = f.smallest_normal / 4                                     # a subnormal
    check_checkpoint(x)


def test_checkpoint_views():
    wide = torch.full((40, 80), float('nan'), dtype=BF16, device='cuda')
    wide[:, 3:75] = rand((40, 72), BF16, 1)
    check_checkpoint(wide[:, 3:75])
    check_checkpoint(rand((3, 5, 7, 40), F16, 2))
    check_checkpoint(rand((64, 20), F32, 3).T)


@pytest.mark.parametrize('t', TYPES, ids=str)
# (the last: large enough for its inputs to be restored once)
@pytest.mark.parametrize('m,k,n', SHAPES + [(2048, 2048, 256), (8200, 2056, 2048)])
def test_backward_from_checkpoint(m, k, n, t):
    """dX and db are those of the layer; dW is the product with the restored activations, which it reads as they lie
    (fp16 restores values below 2^-14 to a multiple of 2^-24: half of it times |dP|)."""
    from pet_posterior_distribution_amd import checkpoint_activations, dense_backward
    x, w, _, p, dy = inputs(m, k, n, t)
    x = x * torch.exp2(torch.arange(m, device='cuda') % 9 - 4).to(t)[:, None]
    c = checkpoint_activations(x)
    for act in (None, 'relu', 'silu'):
        saved = None if act is None else p
        g = check_backward(dy, c, w, act, saved, residual=False, x64=c.restore().double(),
                           grad_dtype=F32 if act == 'relu' else None)
        whole = dense_backward(dy, x, w, activation=act, saved=saved, grad_dtype=F32 if act == 'relu' else None)
        assert torch.equal(g.x, whole.x) and torch.equal(g.bias, whole.bias)


def test_offsets_past_32_bits():
    """2.8e9 activations: row offsets pass 2^32 bytes in every operand that has m rows.  Rows and columns are checked
    against 64 bits at both ends and past the border."""
    from pet_posterior_distribution_amd import checkpoint_activations, dense, dense_backward
    m, k, n, t = 70000, 40000, 8, BF16
    x = torch.empty(m, k, dtype=t, device='cuda').normal_(generator=torch.Generator(device='cuda').manual_seed(3))
    w, dy = rand((k, n), t, 1, k ** -0.5), rand((m, n), t, 2)
    rows = torch.tensor([0, 1, 26843, 26844, 53688, 53690, m - 2, m - 1], device='cuda')
    cols = torch.tensor([0, 7, 31, 20000, k - 1], device='cuda')
    x6, w6, d6 = x[rows].double(), w.double(), dy.double()
    y = dense(x, w)
    close(y[rows], x6 @ w6, (k + 4) * E23 * (x6.abs() @ w6.abs()), 'output')
    g = dense_backward(dy, x, w, need_bias=False)
    close(g.x[rows], d6[rows] @ w6.T, (n + 4) * E23 * (d6[rows].abs() @ w6.abs().T), 'dx')
    xc = x[:, cols].double()
    close(g.kernel[cols], xc.T @ d6, (m + 4) * E23 * (xc.abs().T @ d6.abs()), 'dkernel')
    del g, y
    c = checkpoint_activations(x)
    back = c.restore()
    ref, e = quantize64(x[rows])
    assert torch.equal(c.exponents[rows], e) and torch.equal(back[rows].double(), ref)
    g = dense_backward(dy, c, w, need_x=False, need_bias=False)
    xc = back[:, cols].double()
    close(g.kernel[cols], xc.T @ d6, (m + 4) * E23 * (xc.abs().T @ d6.abs()), 'dkernel from 8 bits')


@pytest.mark.parametrize('t', TYPES, ids=str)
@pytest.mark.parametrize('n', [24, 2100])
def test_exponents_of_a_column_slice_of_a_wide_tensor(n, t):
    """Row strides of 70,000,000 exponent bytes: rows 62 and 63 of a step lie past 2^32."""
    from pet_posterior_distribution_amd import ActivationCheckpoint, checkpoint_activations, dense_backward
    m, k = 130, 96
    x, w, _, _, dy = inputs(m, k, n, t)
    x = x * torch.exp2(torch.arange(m, device='cuda') % 9 - 4).to(t)[:, None]
    c = checkpoint_activations(x)
    wide = torch.empty(m, 70_000_000, dtype=torch.uint8, device='cuda')
    wide[:, 5:8] = c.exponents
    s = ActivationCheckpoint(c.codes, wide[:, 5:8], t)
    assert torch.equal(s.restore(), c.restore())
    g, ref = dense_backward(dy, s, w), dense_backward(dy, c, w)
    for a, b in zip(g[:3], ref[:3]):
        assert torch.equal(a, b)


def signs(shape, seed):
    g = torch.Generator(device='cuda').manual_seed(seed)
    return torch.randint(0, 2, shape, device='cuda', generator=g, dtype=torch.int8).mul_(2).sub_(1)


@pytest.mark.parametrize('t,length', [(BF16, 4_300_000), (BF16, 4_300_003), (F16, 6_000_000), (F32, 2_200_000)],
                         ids=str)
def test_rows_longer_than_dma_offsets(t, length):
    """Rows of more than 2^23 bytes, as the contraction and as the layer's width.  Signs, so that every sum is exact in
    fp32 whatever its order."""
    from pet_posterior_distribution_amd import checkpoint_activations, dense, dense_backward
    m, n = 300, 264
    x, w = signs((m, length), 1).to(t), signs((length, n), 2).to(t)
    y = x.float() @ w.float()
    assert torch.equal(dense(x, w, out_dtype=F32), y)
    dy = signs((m, n), 3).to(t)
    for saved_x in (x, checkpoint_activations(x)):
        g = dense_backward(dy, saved_x, w, grad_dtype=F32)
        assert torch.equal(g.kernel, x.float().T @ dy.float()) and torch.equal(g.bias, dy.float().sum(0))
        assert torch.equal(g.x, (dy.float() @ w.float().T).to(t))
    # the same matrices as a layer of `length` units: dP is long
    wide, keep, dz = w.T.contiguous(), x, signs((m, length), 4).to(t)
    small = signs((m, n), 5).to(t)
    dp = torch.where(keep > 0, dz, torch.zeros_like(dz)).float()
    g = dense_backward(dz, small, wide, activation='relu', saved=keep, grad_dtype=F32)
    assert torch.equal(g.x, (dp @ w.float()).to(t))
    assert torch.equal(g.kernel, small.float().T @ dp) and torch.equal(g.bias, dp.sum(0))


@pytest.mark.parametrize('t,n', [(BF16, 16_700_003), (F32, 8_300_000)], ids=str)
def test_layers_as_wide_as_dma_offsets_allow(t, n):
    """A step's 64 rows (32 in fp32) of a kernel or dP of n columns, up to 2^31 bytes.  Signs: sums are exact."""
    from pet_posterior_distribution_amd import dense, dense_backward
    m, k = 130, 72
    x, w, dy, keep = signs((m, k), 1).to(t), signs((k, n), 2).to(t), signs((m, n), 3).to(t), signs((m, n), 4).to(t)
    y = dense(x, w, out_dtype=F32)
    g = dense_backward(dy, x, w, activation='relu', saved=keep, grad_dtype=F32)
    gx = torch.zeros(m, k, device='cuda')
    for i in range(0, n, 1 << 20):              # (the library's own product is wrong past 2^31 outputs)
        c = slice(i, min(n, i + (1 << 20)))
        wc, dp = w[:, c].float(), torch.where(keep[:, c] > 0, dy[:, c], torch.zeros_like(dy[:, c])).float()
        assert torch.equal(y[:, c], x.float() @ wc), i
        assert torch.equal(g.kernel[:, c], x.float().T @ dp) and torch.equal(g.bias[c], dp.sum(0)), i
        gx += dp @ wc.T
    assert torch.equal(g.x, gx.to(t))


def test_one_row_of_more_columns_than_a_launch_has_threads():
    """2^27 columns: more than one launch of a kernel of 1024 threads for 32 columns could take.  Signs and whole
    numbers, so that every sum is exact in fp32 whatever its order."""
    from pet_posterior_distribution_amd import dense, dense_backward
    n = (1 << 27) + 8
    gen = torch.Generator(device='cuda').manual_seed(5)
    w = torch.randint(0, 2, (1, n), device='cuda', generator=gen, dtype=torch.int8).mul_(2).sub_(1).to(BF16)
    dy = torch.randint(-1, 2, (1, n), device='cuda', generator=gen, dtype=torch.int8).to(BF16)
    x = torch.full((1, 1), 3.0, dtype=BF16, device='cuda')
    assert torch.equal(dense(x, w), 3 * w)
    g = dense_backward(dy, x, w)
    assert torch.equal(g.kernel, 3 * dy) and torch.equal(g.bias, dy[0])
    assert torch.equal(g.x, (dy * w).sum(dtype=torch.float64).to(BF16).reshape(1, 1))


def test_column_sums_of_more_columns_than_a_launch_of_their_own_takes():
    """2^28 columns and more: sixteen to a workgroup of 256 threads, they would be 2^32 threads.  Whole numbers, so that
    every sum is exact."""
    from pet_posterior_distribution_amd import dense_backward
    for m in (1, 3):
        n = (1 << 28) + 8
        w, dy = signs((1, n), 6).to(BF16), signs((m, n), 7).to(BF16)
        x = torch.full((m, 1), 3.0, dtype=BF16, device='cuda')
        g = dense_backward(dy, x, w)
        total = dy.float().sum(0)
        assert torch.equal(g.bias, total.to(BF16)) and torch.equal(g.kernel[0], (3 * total).to(BF16))
        assert torch.equal(g.x, (dy.float() * w.float()).sum(1, True, dtype=torch.float64).to(BF16))


def test_a_kernel_gradient_over_more_rows_than_an_input_gradient_may_have():
    """2^29 rows: x's gradient would be more outputs than a call has; it is not asked for.  Signs: sums are exact."""
    from pet_posterior_distribution_amd import checkpoint_activations, dense_backward
    m, k, n = (1 << 29) + 100, 8, 8
    x, dy, w = signs((m, k), 8).to(BF16), signs((m, n), 9).to(BF16), rand((k, n), BF16, 1)
    ref, at = torch.zeros(k, n, dtype=torch.float64, device='cuda'), 1 << 24
    for i in range(0, m, at):
        ref += x[i:i + at].float().T @ dy[i:i + at].float()
    for saved_x in (x, checkpoint_activations(x)):
        g = dense_backward(dy, saved_x, w, need_x=False, grad_dtype=F32)
        assert g.x is None and torch.equal(g.kernel.double(), ref)
        assert torch.equal(g.bias.double(), dy.sum(0, dtype=torch.float64))
    with pytest.raises(ValueError, match='too many'):
        dense_backward(dy, x, w)


# ------------------------------------------------------------------------------------------- streams and graphs
def chain(x, ws, bs, dy):
    """Two layers forward, the first one's input kept in 8 bits, and their backward passes."""
    from pet_posterior_distribution_amd import checkpoint_activations, dense, dense_backward
    c = checkpoint_activations(x)
    h, p1 = dense(x, ws[0], bs[0], activation='gelu', return_preactivation=True)
    y = dense(h, ws[1], bs[1], activation='relu', residual=x)
    g2 = dense_backward(dy, h, ws[1], activation='relu', saved=y, need_residual=True)
    g1 = dense_backward(g2.x, c, ws[0], activation='gelu', saved=p1, grad_dtype=F32)
    return [h, y, g2.x, g2.kernel, g2.bias, g2.residual, g1.x, g1.kernel, g1.bias, c.restore()]


def chain_inputs(seed, m=333, t=BF16):
    x = rand((m, 96), t, seed)
    ws = [rand((96, 200), t, seed + 1, 0.1), rand((200, 96), t, seed + 2, 0.07)]
    bs = [rand((200,), t, seed + 3), rand((96,), F32, seed + 4)]
    return x, ws, bs, rand((m, 96), t, seed + 5)


def test_a_run_of_the_operators_against_64_bits():
    """The chain of two layers as it is used.  Each stage is checked from the stages before it by the tests above; the
    run as a whole by its distance in the 2-norm: about a dozen independent roundings of at most 2^-9 to its inputs,
    sqrt(12) 2^-9 = 0.7 %, and the checkpoint's 2^-4 / sqrt 3 = 3.6 % in the first kernel's gradient alone."""
    x, ws, bs, dy = chain_inputs(7)
    got = chain(x, ws, bs, dy)
    x6, w0, w1, b0, b1, d6 = (v.double() for v in (x, ws[0], ws[1], bs[0], bs[1], dy))
    p1 = x6 @ w0 + b0
    h = act64(p1, 'gelu')
    y = act64(h @ w1 + b1 + x6, 'relu')
    dp2 = d6 * (got[1] > 0)                       # the run's own mask: a pre-activation next to zero may go either way
    gh = dp2 @ w1.T
    dp1 = gh * act_grad64(p1, 'gelu')
    ref = [h, y, gh, h.T @ dp2, dp2.sum(0), dp2, dp1 @ w0.T, x6.T @ dp1, dp1.sum(0), x6]
    for i, (a, r) in enumerate(zip(got, ref)):
        far = ((a.double() - r).norm() / r.norm()).item()
        assert far < (0.036 if i in (7, 9) else 0.007), (i, far)


def test_results_repeat_bit_by_bit_and_on_another_stream():
    x, ws, bs, dy = chain_inputs(11)
    one = chain(x, ws, bs, dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        two = chain(x, ws, bs, dy)
    torch.cuda.current_stream().wait_stream(side)
    three = chain(x, ws, bs, dy)
    torch.cuda.synchronize()
    for a, b, c in zip(one, two, three):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_two_captured_graphs_replay_like_eager_runs():
    sets = [chain_inputs(21), chain_inputs(31, m=40)]
    eager = [chain(*s) for s in sets]
    graphs, outs = [], []
    for s in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(chain(*s))
        graphs.append(g)
    for rep in range(4):
        for o in outs:
            for v in o:
                v.zero_()
        other = chain(*chain_inputs(41 + rep))        # eager work between the replays
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for o, e in zip(outs, eager):
            for a, b in zip(o, e):
                assert torch.equal(a, b), rep
        del other
    # new inputs in the captured tensors' place
    fresh = chain_inputs(61)
    for dst, src in zip([sets[0][0], *sets[0][1], *sets[0][2], sets[0][3]], [fresh[0], *fresh[1], *fresh[2], fresh[3]]):
        dst.copy_(src)
    graphs[0].replay()
    torch.cuda.synchronize()
    for a, b in zip(outs[0], chain(*fresh)):
        assert torch.equal(a, b)


FIRST_CALLS = """
import sys
import torch
from pet_posterior_distribution_amd import checkpoint_activations, dense, dense_backward
t = torch.bfloat16
x, w = torch.randn(300, 256, device='cuda').to(t), (torch.randn(256, 512, device='cuda') / 16).to(t)
big, wide = torch.randn(2048, 512, device='cuda').to(t), (torch.randn(512, 4096, device='cuda') / 16).to(t)
dy, dz = torch.randn(300, 512, device='cuda').to(t), torch.randn(2048, 4096, device='cuda').to(t)
torch.cuda.synchronize()
def run():
    c = checkpoint_activations(x)
    y, p = dense(x, w, activation='gelu', return_preactivation=True)
    return [y, *dense_backward(dy, c, w, activation='gelu', saved=p)[:3], dense(big, wide),
            *dense_backward(dz, big, wide)[:3], dense(x[:1], w), c.restore()]
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    out = run()
for rep in range(3):
    for v in out:
        v.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, run())), rep
print('same')
"""


def test_the_first_calls_of_a_process_may_be_captured():
    """Loading the code and allowing the larger tiles their LDS happen inside the capture."""
    r = subprocess.run([sys.executable, '-c', FIRST_CALLS], capture_output=True, text=True, timeout=100,
                       cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert r.returncode == 0 and 'same' in r.stdout, r.stderr[-2000:]
