"""The dense layer's operators as they are measured: a product with bias, residual and activation in its
epilogue (`dense`), its backward pass (`dense_backward`), the 8-bit activation checkpoint, and the backward
pass that reads it.

    forward      P = X W + b + R,  Y = act(P)            X (m, k), W (k, n), b (n,), R (m, n)
    backward     dP = dY act'(P);  dX = dP W^T,  dW = X^T dP,  db = sum of dP's rows,  dR = dP
    checkpoint   per row, blocks of 32 values share a power of two 2^E, the least with max|x| <= 448 2^E
                 (E >= -117); each value is kept as e4m3 of x 2^-E, rounded to nearest even

A case is measured in its plain form (`own` false: elementary torch operations in 32 bits) or through the
package's entry points (`own` true).
"""
import math

import torch

own = False

BLOCK = 32
TYPES = {'bfloat16': torch.bfloat16, 'float16': torch.float16, 'float32': torch.float32}


def listed():
    return [
        # one row through a wide layer: the smallest call there is, bound by its weights and by latency
        dict(name='fwd one row', op='forward', m=1, k=1024, n=4096, dtype='bfloat16', act='silu', residual=False,
             pre=False),
        # the second layer of the condition encoder (256 -> 128, ReLU) over 49 rows of each of 1024 samples
        dict(name='fwd encoder', op='forward', m=49 * 1024, k=256, n=128, dtype='bfloat16', act='relu',
             residual=False, pre=False),
        # the wide half of a feed-forward block over 8192 rows; its pre-activation is kept for training
        dict(name='fwd wide gelu', op='forward', m=8192, k=4096, n=8192, dtype='bfloat16', act='gelu',
             residual=False, pre=True),
        # odd sizes with a residual, in fp16: no row starts on an aligned address
        dict(name='fwd odd f16', op='forward', m=777, k=1069, n=333, dtype='float16', act='none', residual=True,
             pre=False),
        # the third down level's convolution as a product (6 x 306 -> 512, 12 positions), 512 samples, fp32
        dict(name='fwd conv f32', op='forward', m=12 * 512, k=1836, n=512, dtype='float32', act='relu',
             residual=False, pre=False),
        # the condition encoder's last hidden layer (128 -> 64) for a batch of 32
        dict(name='bwd encoder', op='backward', m=49 * 32, k=128, n=64, dtype='bfloat16', act='relu',
             grad='float32'),
        # the first up level's block (6 x 1024 -> 512, 12 positions), 1024 samples, gradients for fp32 weights
        dict(name='bwd conv', op='backward', m=12 * 1024, k=6144, n=512, dtype='bfloat16', act='relu',
             grad='float32'),
        # a wide layer under a GELU over 8192 rows, gradients in the weights' own type
        dict(name='bwd wide gelu', op='backward', m=8192, k=8192, n=4096, dtype='bfloat16', act='gelu',
             grad='bfloat16'),
        # a short, ragged batch of fp32 activations to 8 bits and back
        dict(name='ckpt ragged', op='checkpoint', m=257, k=615, dtype='float32'),
        # the activations of a long batch to 8 bits and back
        dict(name='ckpt long', op='checkpoint', m=65536, k=4096, dtype='bfloat16'),
        # the last up level's block (6 x 256 -> 128, 48 positions), 512 samples, from 8-bit inputs
        dict(name='bwd ckpt conv', op='backward8', m=48 * 512, k=1536, n=128, dtype='bfloat16', act='relu',
             grad='float32'),
        # odd sizes in fp16, from 8-bit inputs
        dict(name='bwd ckpt odd f16', op='backward8', m=1111, k=1067, n=515, dtype='float16', act='silu',
             grad='float16'),
    ]


def _size(rng, lo, hi):
    s = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return s if rng.random() < 0.5 else max(lo, min(hi, s // 8 * 8))


def draw(rng):
    op = rng.choice(['forward', 'forward', 'backward', 'backward', 'checkpoint', 'backward8'])
    dtype = rng.choice(['bfloat16', 'bfloat16', 'float16', 'float32'])
    m, k, n = _size(rng, 1, 49152), _size(rng, 16, 8192), _size(rng, 8, 8192)
    if op == 'checkpoint':
        return dict(op=op, m=m, k=k, dtype=dtype)
    passes = 1 if op == 'forward' else 2
    m = max(1, min(m, int(2.5e11 / (passes * k * n))))
    act = rng.choice(['none', 'relu', 'gelu', 'silu'])
    if op == 'forward':
        return dict(op=op, m=m, k=k, n=n, dtype=dtype, act=act, residual=rng.random() < 0.3,
                    pre=act in ('gelu', 'silu') and rng.random() < 0.5)
    # fp32 gradients of 16-bit layers are what a ReLU or linear layer's training step asks for
    grad = 'float32' if act in ('none', 'relu') and rng.random() < 0.5 else dtype
    return dict(op=op, m=m, k=k, n=n, dtype=dtype, act=act, grad=grad)


def prepare(case, seed):
    g = torch.Generator(device='cuda').manual_seed(seed)
    t = TYPES[case['dtype']]

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device='cuda').mul_(scale)

    m, k = case['m'], case['k']
    s = dict(case=case)
    if case['op'] == 'checkpoint':
        # rows of unlike size, as tokens and samples are
        s['x'] = (normal(m, k) * torch.exp(normal(m, 1))).to(t)
        return s
    n = case['n']
    s['kernel'] = normal(k, n, scale=k ** -0.5).to(t)
    if case['op'] == 'forward':
        s['x'] = normal(m, k).to(t)
        s['bias'] = normal(n, scale=0.1).to(t)
        s['residual'] = normal(m, n).to(t) if case['residual'] else None
        return s
    s['dy'] = normal(m, n, scale=0.1).to(t)
    p = normal(m, n)
    # what the forward pass saved: ReLU's output, or the pre-activation of GELU and SiLU
    s['saved'] = None if case['act'] == 'none' else (p.clamp_(min=0) if case['act'] == 'relu' else p).to(t)
    x = normal(m, k)
    if case['op'] == 'backward':
        s['x'] = x.to(t)
    else:
        s['codes'], s['exponents'] = _to_8_bits(x.to(t))
    return s


def _blocks(x):
    """x (m, k) as (m, blocks, 32), padded with zeros."""
    m, k = x.shape
    nb = -(-k // BLOCK)
    full = torch.zeros(m, nb * BLOCK, dtype=x.dtype, device=x.device)
    full[:, :k] = x
    return full.view(m, nb, BLOCK)


def _to_8_bits(x):
    """e4m3 codes (m, k) and the bytes E + 127 (m, blocks) of finite activations."""
    b = _blocks(x.float())
    mant, exp = torch.frexp(b.abs().amax(-1))            # max|x| = mant 2^exp, mant in [0.5, 1); 448 = 0.875 2^9
    top = 8 if x.dtype == torch.float16 else 120         # there 256 2^E is past the type's largest value
    e = torch.where(mant <= 0.875, exp - 9, exp - 8).clamp(min=-117)
    y = b * _power(-e)[..., None]
    y = torch.where((e == top)[..., None], y.clamp(-240, 240), y)
    codes = y.to(torch.float8_e4m3fn).view(x.shape[0], -1)[:, :x.shape[1]].contiguous()
    return codes, (e + 127).to(torch.uint8)


def _power(e):
    """2^e in fp32, exactly."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _from_8_bits(codes, exponents):
    scale = _power(exponents.int() - 127)
    return (_blocks(codes.float()) * scale[..., None]).view(codes.shape[0], -1)[:, :codes.shape[1]]


def _act(p, act):
    if act == 'relu':
        return torch.where(p < 0, torch.zeros_like(p), p)
    if act == 'gelu':
        return 0.5 * p * (1 + torch.erf(p * 0.5 ** 0.5))
    if act == 'silu':
        return p / (1 + torch.exp(-p))
    return p


def _act_grad(dy, saved, act):
    if act == 'relu':
        return torch.where(saved <= 0, torch.zeros_like(dy), dy)
    if act == 'gelu':
        cdf = 0.5 * (1 + torch.erf(saved * 0.5 ** 0.5))
        return dy * (cdf + saved * torch.exp(-0.5 * saved * saved) * (2 * math.pi) ** -0.5)
    if act == 'silu':
        sig = 1 / (1 + torch.exp(-saved))
        return dy * sig * (1 + saved * (1 - sig))
    return dy


def _forward(s, case):
    t = TYPES[case['dtype']]
    p = s['x'].float() @ s['kernel'].float() + s['bias'].float()
    if s['residual'] is not None:
        p = p + s['residual'].float()
    y = _act(p, case['act']).to(t)
    return (y, p.to(t)) if case['pre'] else y


def _backward(dy, x, kernel, saved, case):
    t, tg = TYPES[case['dtype']], TYPES[case['grad']]
    dp = _act_grad(dy.float(), None if saved is None else saved.float(), case['act'])
    return {'x': (dp @ kernel.float().T).to(t), 'kernel': (x.T @ dp).to(tg), 'bias': dp.sum(0).to(tg)}


def run(s):
    case = s['case']
    op = case['op']
    if own:
        import pet_posterior_distribution_amd as pet
        act = case.get('act')
        if op == 'forward':
            return pet.dense(s['x'], s['kernel'], s['bias'], activation=act, residual=s['residual'],
                             return_preactivation=case['pre'])
        if op == 'checkpoint':
            c = pet.checkpoint_activations(s['x'])
            return {'restored': c.restore(), 'exponents': c.exponents}
        x = s['x'] if op == 'backward' else pet.ActivationCheckpoint(s['codes'], s['exponents'], s['dy'].dtype)
        g = pet.dense_backward(s['dy'], x, s['kernel'], activation=act, saved=s['saved'],
                               grad_dtype=TYPES[case['grad']])
        return {'x': g.x, 'kernel': g.kernel, 'bias': g.bias}
    if op == 'forward':
        return _forward(s, case)
    if op == 'checkpoint':
        codes, exponents = _to_8_bits(s['x'])
        return {'restored': _from_8_bits(codes, exponents).to(s['x'].dtype), 'exponents': exponents}
    x = s['x'].float() if op == 'backward' else _from_8_bits(s['codes'], s['exponents'])
    return _backward(s['dy'], x, s['kernel'], s['saved'], case)


def work(case):
    m, k = case['m'], case['k']
    size = 4 if case['dtype'] == 'float32' else 2
    if case['op'] == 'checkpoint':
        # activations in, codes and exponents out, restored activations out
        return {'bytes': m * k * (2 * size + 1) + m * -(-k // BLOCK), 'flops': 4 * m * k}
    n = case['n']
    if case['op'] == 'forward':
        mn = 1 + case['residual'] + case['pre']
        return {'bytes': size * (m * k + k * n + n + mn * m * n), 'flops': 2 * m * k * n}
    grad = 4 if case['grad'] == 'float32' else 2
    x_in = size * m * k if case['op'] == 'backward' else m * k + m * -(-k // BLOCK)
    mn = 1 + (case['act'] != 'none')
    return {'bytes': x_in + size * (m * k + k * n + mn * m * n) + grad * (k * n + n), 'flops': 4 * m * k * n}


def exact(case, seed):
    """The definitions in 64 bits."""
    s = prepare(case, seed)
    f64 = torch.float64

    def power(e):
        # torch.exp2 may be off by a bit in 64 bits: an exponent field is not
        return ((e.long() + 1023) << 52).view(f64)

    if case['op'] == 'checkpoint':
        x = s['x'].to(f64)
        m, k = x.shape
        nb = (k + BLOCK - 1) // BLOCK
        index = torch.arange(k, device=x.device) // BLOCK
        peak = torch.zeros(m, nb, dtype=f64, device=x.device)
        peak.scatter_reduce_(1, index.expand(m, k), x.abs(), 'amax')
        e = torch.ceil(torch.log2(peak / 448)).clamp(min=-117)
        # the logarithm is rounded: move to the least exponent that holds the peak
        e = torch.where(448 * power(e - 1) >= peak, e - 1, e).clamp(min=-117)
        e = torch.where(448 * power(e) < peak, e + 1, e)
        scale = power(e)[:, index]
        v = x / scale
        step = torch.ones_like(v) * 2.0 ** -9
        for exponent in range(-5, 9):                    # e4m3's binades
            step = torch.where(v.abs() >= 2.0 ** exponent, 2.0 ** (exponent - 3), step)
        r = torch.round(v / step) * step
        lim = torch.where(scale == 2.0 ** (8 if case['dtype'] == 'float16' else 120), 240.0, 448.0)
        r = torch.minimum(torch.maximum(r, -lim), lim)
        return {'restored': r * scale, 'exponents': None}
    w = s['kernel'].to(f64)
    if case['op'] == 'forward':
        p = torch.addmm(s['bias'].to(f64), s['x'].to(f64), w)
        if s['residual'] is not None:
            p += s['residual'].to(f64)
        y = {'none': lambda v: v, 'relu': torch.relu, 'silu': lambda v: v * torch.sigmoid(v),
             'gelu': lambda v: v * torch.special.ndtr(v)}[case['act']](p)
        return (y, p) if case['pre'] else y
    dp = s['dy'].to(f64)
    if case['act'] != 'none':
        v = s['saved'].to(f64)
        if case['act'] == 'relu':
            dp = dp * (v > 0)
        elif case['act'] == 'silu':
            sg = torch.sigmoid(v)
            dp = dp * (sg + v * sg * (1 - sg))
        else:
            dp = dp * (torch.special.ndtr(v) + v * torch.exp(-v * v / 2) / math.sqrt(2 * math.pi))
    if case['op'] == 'backward':
        x = s['x'].to(f64)
    else:
        index = torch.arange(case['k'], device=dp.device) // BLOCK
        x = s['codes'].to(f64) * power(s['exponents'].long() - 127)[:, index]
    return {'x': torch.mm(dp, w.t()), 'kernel': torch.mm(x.t(), dp), 'bias': torch.sum(dp, 0)}
