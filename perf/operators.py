"""Cases, plain forms and 64-bit definitions of the training operators beside the quantised layers: AdamW over many tensors
(states in 32 or 8 bits, optional clipping by the global norm), group normalisation with an activation (channels last,
forward and backward) and the gated linear recurrence h_t = a_t h_{t-1} + (1 - a_t) x_t, a_t = sigmoid(z_t) (forward, backward,
single token).

``run`` computes an operator in its plain form, or through ``hgq2_b200`` where ``own`` is true.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {'float32': torch.float32, 'bfloat16': torch.bfloat16, 'float16': torch.float16}
BLOCK = 256  # elements that share a scale of the 8-bit optimizer states; every tensor starts at a multiple of it
LR, BETA1, BETA2, EPS, DECAY, CLIP = 1e-3, 0.9, 0.999, 1e-7, 4e-3, 1.0
FIRST_STEP = 1000  # the optimizer cases go on from a state in mid-training


def listed():
    return [
        # the variables of a stack of four small dense layers with their bitwidths: one launch's latency
        dict(name='adamw_small_stack', op='adamw', tensors=28, smallest=5, largest=2048, bits=32, clip=False, grad='float32'),
        # several hundred layers' variables of odd sizes, gradients clipped by their global norm
        dict(name='adamw_many_clipped', op='adamw', tensors=320, smallest=17, largest=1000003, bits=32, clip=True, grad='float32'),
        # 8-bit states, gradients as a mixed-precision backward pass leaves them
        dict(name='adamw_8bit_half_grads', op='adamw', tensors=64, smallest=100, largest=8000001, bits=8, clip=False, grad='bfloat16'),
        # a model whose states would not fit in 32 bits
        dict(name='adamw_8bit_large', op='adamw', tensors=40, smallest=1000, largest=64000000, bits=8, clip=True, grad='float32'),
        # a few feature maps: launch latency of both directions
        dict(name='groupnorm_few_maps', op='groupnorm', batch=8, height=8, width=8, channels=64, groups=8, activation='gelu', dtype='float32', train=True),
        # the first convolution's output of the small convolutional network at its training batch
        dict(name='groupnorm_conv_maps', op='groupnorm', batch=4096, height=30, width=30, channels=16, groups=4, activation='silu', dtype='float32', train=True),
        # [batch, sequence, features] of the attention block at its training batch, evaluation in half precision
        dict(name='groupnorm_sequences', op='groupnorm', batch=8192, height=1, width=64, channels=64, groups=8, activation='relu', dtype='bfloat16', train=False),
        # a few large images, odd extents, three channels to a group
        dict(name='groupnorm_images', op='groupnorm', batch=6, height=255, width=257, channels=96, groups=32, activation='silu', dtype='bfloat16', train=True),
        # serving: one token of 64 streams, the state carried over
        dict(name='recurrence_one_token', op='recurrence', batch=64, length=1, features=256, dtype='float32', padded=False, state=True, train=False),
        # [batch, sequence, features] of the attention block at its training batch
        dict(name='recurrence_sequences', op='recurrence', batch=8192, length=64, features=64, dtype='float32', padded=False, state=False, train=True),
        # two long streams: parallelism has to come from the time axis
        dict(name='recurrence_long', op='recurrence', batch=2, length=65521, features=256, dtype='bfloat16', padded=False, state=True, train=True),
        # a padded batch of sequences of many lengths (zero among them), evaluation
        dict(name='recurrence_padded', op='recurrence', batch=96, length=1999, features=321, dtype='float16', padded=True, state=True, train=False),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(['adamw', 'groupnorm', 'recurrence'])
    if op == 'adamw':
        largest = _spread(rng, 500, 20000000)
        # the sizes are spread over their logarithm: the mean is about largest / ln(largest / smallest)
        tensors = min(_spread(rng, 1, 400), max(1, int(150e6 / (largest / 3))))
        return dict(op='adamw', tensors=tensors, smallest=rng.randint(1, 300), largest=largest, bits=rng.choice([32, 8]),
                    clip=rng.random() < 0.5, grad=rng.choice(list(DTYPES)))
    dtype = rng.choice(list(DTYPES))
    train = rng.random() < 0.6
    if op == 'groupnorm':
        groups = rng.choice([1, 2, 4, 8, 16, 32])
        channels = groups * rng.randint(1, max(1, 256 // groups))
        height, width = _spread(rng, 1, 256), _spread(rng, 4, 256)
        # the slope of a ReLU at its corner is decided by the last bit of a sum: forward only
        activation = rng.choice(['none', 'silu', 'gelu'] if train else ['none', 'relu', 'silu', 'gelu'])
        most = max(1, int(60e6 / (height * width * channels)))
        return dict(op='groupnorm', batch=min(_spread(rng, 1, 8192), most), height=height, width=width, channels=channels,
                    groups=groups, activation=activation, dtype=dtype, train=train)
    length, features = _spread(rng, 1, 60000), _spread(rng, 1, 1024)
    most = max(1, int(30e6 / (length * features)))
    if length * features > 30e6:
        features = max(1, int(30e6 / length))
    return dict(op='recurrence', batch=min(_spread(rng, 1, 8192), most), length=length, features=features, dtype=dtype,
                padded=rng.random() < 0.4, state=rng.random() < 0.5, train=train)


# ---- inputs ---------------------------------------------------------------------------------------------------------------
def _sizes(case):
    """Tensor sizes spread over their logarithm (the fractional parts of multiples of the golden ratio), the largest first."""
    a, b = case['smallest'], max(case['smallest'], case['largest'])
    return [int(round(a * (b / a) ** (1.0 - (i * 0.6180339887498949) % 1.0))) for i in range(case['tensors'])]


def _layout(case):
    sizes = _sizes(case)
    offsets, total = [], 0
    for n in sizes:
        offsets.append(total)
        total += -(-n // BLOCK) * BLOCK
    return sizes, offsets, total


def _decays(case):
    """Every third tensor (biases, bitwidths) takes no weight decay."""
    return [0.0 if i % 3 == 2 else DECAY for i in range(case['tensors'])]


def _inputs(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(int(seed))

    def normal(*shape):
        return torch.randn(shape, device='cuda', generator=gen)

    s = {'case': case}
    if case['op'] == 'adamw':
        sizes, offsets, total = _layout(case)
        s['w'], s['g'] = torch.zeros(total, device='cuda'), torch.zeros(total, device='cuda')
        m, r = torch.zeros(total, device='cuda'), torch.zeros(total, device='cuda')
        for n, o in zip(sizes, offsets):
            scale = 10.0 ** (-1.0 - 2.0 * ((o // BLOCK) % 7) / 6.0)  # gradients of different layers differ by decades
            s['w'][o:o + n] = normal(n) * 0.05
            s['g'][o:o + n] = normal(n) * scale
            m[o:o + n] = normal(n) * (0.3 * scale)
            r[o:o + n] = torch.exp(normal(n) * 0.5) * scale
        s['g'] = s['g'].to(DTYPES[case['grad']])
        per_tensor = torch.tensor(_decays(case), device='cuda', dtype=torch.float64)
        blocks = torch.tensor([-(-n // BLOCK) for n in sizes], device='cuda')
        s['decay'] = torch.repeat_interleave(per_tensor, blocks)
        s['t'] = torch.full((), FIRST_STEP, dtype=torch.int64, device='cuda')
        if case['bits'] == 8:
            for key, x in (('m', m), ('r', r)):
                x = x.view(-1, BLOCK)
                scale = x.abs().amax(1).clamp(min=2.0 ** -100) / 256
                s[key] = (x / scale[:, None]).to(torch.float8_e4m3fn).view(-1)
                s[key + '_scale'] = scale
        else:
            s['m'], s['v'] = m, r * r
        return s
    dtype = DTYPES[case['dtype']]
    if case['op'] == 'groupnorm':
        c = case['channels']
        shape = (case['batch'], case['height'], case['width'], c)
        s['x'] = (normal(*shape) * (0.5 + torch.rand(c, device='cuda', generator=gen)) + normal(c)).to(dtype)
        s['gamma'], s['beta'] = 1 + 0.2 * normal(c), 0.2 * normal(c)
        if case['train']:
            s['gy'] = normal(*shape).to(dtype)
        return s
    b, t, d = case['batch'], case['length'], case['features']
    s['x'], s['z'] = normal(b, t, d).to(dtype), (2.0 + 1.5 * normal(b, t, d)).to(dtype)
    s['h0'] = normal(b, d) if case['state'] else None
    s['lengths'] = torch.randint(0, t + 1, (b,), device='cuda', generator=gen, dtype=torch.int32) if case['padded'] else None
    if case['train']:
        s['gh'] = normal(b, t, d).to(dtype)
        s['g_last'] = normal(b, d) if case['state'] else None
    return s


def _optimizer(s):
    """The optimizer that the program keeps, its states taken over from a checkpoint."""
    from hgq2_b200.train import FusedAdamW

    case = s['case']
    sizes, offsets, _ = _layout(case)
    s['params'] = [s['w'][o:o + n] for n, o in zip(sizes, offsets)]
    s['grads'] = [s['g'][o:o + n] for n, o in zip(sizes, offsets)]
    opt = FusedAdamW(s['params'], learning_rate=LR, beta_1=BETA1, beta_2=BETA2, epsilon=EPS, weight_decay=_decays(case),
                     global_clipnorm=CLIP if case['clip'] else None, state_bits=case['bits'])
    opt.step_count.fill_(FIRST_STEP)
    for key in ('m', 'v') if case['bits'] == 32 else ('m', 'r', 'm_scale', 'r_scale'):
        getattr(opt, key).copy_(s.pop(key))
    return opt


def prepare(case, seed):
    s = _inputs(case, seed)
    if own and case['op'] == 'adamw':
        s['opt'] = _optimizer(s)
    return s


# ---- plain forms ----------------------------------------------------------------------------------------------------------
def _mix(index, t):
    """A 32-bit multiply-xorshift mix of the element's place and the step: the dither of the 8-bit states."""
    low = 0xFFFFFFFF
    h = (index * 0x9E3779B1 + t * 0x6A09E667) & low
    h = h ^ (h >> 16)
    h = (h * 0xBB67AE85) & low
    h = h ^ (h >> 15)
    h = (h * 0x3C6EF373) & low
    return h ^ (h >> 16)


def _dithered(u, dither):
    """u >= 0 on the e4m3 grid, up or down with the odds that keep its mean: 16 dither bits below the third mantissa bit."""
    low = u < 2.0 ** -6
    y = torch.where(low, u + 2.0 ** -6, u)
    y = ((y.view(torch.int32) + (dither.to(torch.int32) << 4)) & -0x100000).view(torch.float32)
    return torch.where(low, y - 2.0 ** -6, y)


def _adamw(s):
    case = s['case']
    s['t'] += 1
    t = s['t'].double()
    alpha = (LR * torch.sqrt(1.0 - BETA2 ** t) / (1.0 - BETA1 ** t)).float()
    g = s['g'].float()
    if case['clip']:
        norm = torch.sqrt(g.double().square().sum())
        g = g * (CLIP / norm).clamp(max=1.0).float()
    if case['bits'] == 8:
        m = (s['m'].float().view(-1, BLOCK) * s['m_scale'][:, None]).view(-1)
        r = (s['r'].float().view(-1, BLOCK) * s['r_scale'][:, None]).view(-1)
        v = r * r
    else:
        m, v = s['m'], s['v']
    m = m * BETA1 + g * (1.0 - BETA1)
    v = v * BETA2 + (g * g) * (1.0 - BETA2)
    root = torch.sqrt(v)
    kept = (1.0 - LR * s['decay']).float()
    w = (s['w'].view(-1, BLOCK) * kept[:, None]).view(-1) - alpha * m / (root + EPS)
    s['w'].copy_(w)
    if case['bits'] == 32:
        s['m'].copy_(m)
        s['v'].copy_(v)
        return {'w': s['w'], 'm': s['m'], 'v': s['v']}
    dither = _mix(torch.arange(m.numel(), device='cuda'), s['t'])
    for key, x, bits in (('m', m, dither & 0xFFFF), ('r', root, dither >> 16)):
        x = x.view(-1, BLOCK)
        size = x.abs()
        top = size.amax(1).clamp(min=2.0 ** -100)
        code = _dithered(size * (256.0 * torch.ones_like(top) / top)[:, None], bits.view(-1, BLOCK))
        if key == 'r':  # a root that is not zero never becomes zero: it divides the step
            code = torch.where((size > 0) & (code == 0), 2.0 ** -9, code)
        s[key].copy_(torch.where(x < 0, -code, code).to(torch.float8_e4m3fn).view(-1))
        s[key + '_scale'].copy_(top / 256)
    return {'w': s['w'], 'm': s['m'], 'r': s['r'], 'm_scale': s['m_scale'], 'r_scale': s['r_scale']}


def _activated(u, name):
    """act(u) and act'(u)."""
    if name == 'relu':
        return torch.where(u > 0, u, torch.zeros_like(u)), (u > 0).to(u.dtype)
    if name == 'silu':
        p = 1 / (1 + torch.exp(-u))
        return u * p, p * (1 + u * (1 - p))
    if name == 'gelu':
        cdf = 0.5 * (1 + torch.erf(u * math.sqrt(0.5)))
        return u * cdf, cdf + u * torch.exp(-0.5 * u * u) / math.sqrt(2 * math.pi)
    return u, torch.ones_like(u)


def _groupnorm(s):
    case = s['case']
    b, c, groups = case['batch'], case['channels'], case['groups']
    x = s['x'].float().view(b, -1, groups, c // groups)
    gamma, beta = s['gamma'].view(groups, -1), s['beta'].view(groups, -1)
    mean = x.mean((1, 3), keepdim=True)
    xhat = x - mean
    rstd = 1 / torch.sqrt(xhat.square().mean((1, 3), keepdim=True) + 1e-3)
    xhat = xhat * rstd
    y, slope = _activated(xhat * gamma + beta, case['activation'])
    out = {'y': y.to(s['x'].dtype).view(s['x'].shape)}
    if case['train']:
        gu = s['gy'].float().view(x.shape) * slope
        out['dbeta'] = gu.sum((0, 1)).view(c)
        out['dgamma'] = (gu * xhat).sum((0, 1)).view(c)
        gx = gu * gamma
        gx = gx - gx.mean((1, 3), keepdim=True) - xhat * (gx * xhat).mean((1, 3), keepdim=True)
        out['dx'] = (gx * rstd).to(s['x'].dtype).view(s['x'].shape)
    return out


def _scan(a, b):
    """h_t = a_t h_{t-1} + b_t along axis 1 from h_{-1} = 0, by doubling the span that each step has taken in."""
    span = 1
    while span < a.shape[1]:
        b = torch.cat([b[:, :span], b[:, span:] + a[:, span:] * b[:, :-span]], 1)
        a = torch.cat([a[:, :span], a[:, span:] * a[:, :-span]], 1)
        span *= 2
    return b


def _recurrence(s):
    x, z = s['x'].float(), s['z'].float()
    length, dtype = x.shape[1], s['x'].dtype
    a, c = 1 / (1 + torch.exp(-z)), 1 / (1 + torch.exp(z))  # the gate and 1 - gate
    live = None
    if s['lengths'] is not None:  # steps behind a sequence's end leave the state as it is
        live = (torch.arange(length, device='cuda') < s['lengths'][:, None])[:, :, None]
        a, c = torch.where(live, a, 1.0), torch.where(live, c, 0.0)
    b = c * x
    h0 = s['h0'] if s['h0'] is not None else torch.zeros_like(x[:, 0])
    h = _scan(a, torch.cat([b[:, :1] + a[:, :1] * h0[:, None], b[:, 1:]], 1))
    shown = h if live is None else torch.where(live, h, 0.0)
    out = {'h': shown.to(dtype), 'h_last': h[:, -1]}
    if s['case']['train']:
        g = s['gh'].float() if live is None else torch.where(live, s['gh'].float(), 0.0)
        if s['g_last'] is not None:
            g = torch.cat([g[:, :-1], g[:, -1:] + s['g_last'][:, None]], 1)
        later = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)  # lambda_t = g_t + a_{t+1} lambda_{t+1}
        lam = _scan(later.flip(1), g.flip(1)).flip(1)
        before = torch.cat([h0[:, None], h[:, :-1]], 1)
        out['dx'] = (lam * c).to(dtype)
        out['dz'] = (lam * a * c * (before - x)).to(dtype)
        if s['h0'] is not None:
            out['dh0'] = a[:, 0] * lam[:, 0]
    return out


# ---- the framework's calls --------------------------------------------------------------------------------------------------
def _run_own(s):
    from hgq2_b200 import kernels

    case = s['case']
    if case['op'] == 'adamw':
        opt = s['opt']
        opt.step(s['grads'])
        if case['bits'] == 32:
            return {'w': s['w'], 'm': opt.m, 'v': opt.v}
        return {'w': s['w'], 'm': opt.m, 'r': opt.r, 'm_scale': opt.m_scale, 'r_scale': opt.r_scale}
    if case['op'] == 'groupnorm':
        act = None if case['activation'] == 'none' else case['activation']
        y, mean, rstd = kernels.group_norm_fwd(s['x'], s['gamma'], s['beta'], case['groups'], 1e-3, act)
        if not case['train']:
            return {'y': y}
        dx, dgamma, dbeta = kernels.group_norm_bwd(s['gy'], s['x'], s['gamma'], s['beta'], mean, rstd, case['groups'], act)
        return {'y': y, 'dx': dx, 'dgamma': dgamma, 'dbeta': dbeta}
    h, h_last, states = kernels.gated_scan_fwd(s['x'], s['z'], s['h0'], s['lengths'], want_states=case['train'])
    out = {'h': h, 'h_last': h_last}
    if case['train']:
        dx, dz, dh0 = kernels.gated_scan_bwd(s['gh'], s['x'], s['z'], s['h0'], s['lengths'], states, s['g_last'],
                                             want_dh0=s['h0'] is not None)
        out.update(dx=dx, dz=dz)
        if dh0 is not None:
            out['dh0'] = dh0
    return out


def run(state):
    if own:
        return _run_own(state)
    return {'adamw': _adamw, 'groupnorm': _groupnorm, 'recurrence': _recurrence}[state['case']['op']](state)


# ---- work and definition ----------------------------------------------------------------------------------------------------
def work(case):
    if case['op'] == 'adamw':
        n = sum(_sizes(case))
        grad = 4 if case['grad'] == 'float32' else 2
        states = 16 if case['bits'] == 32 else 4 + 16 / BLOCK  # both states, read and written
        return {'bytes': n * (8 + grad + states), 'flops': n * 15}
    size = 4 if case['dtype'] == 'float32' else 2
    if case['op'] == 'groupnorm':
        n = case['batch'] * case['height'] * case['width'] * case['channels']
        tensors, params = (4, 4) if case['train'] else (2, 2)
        return {'bytes': tensors * n * size + params * 4 * case['channels'], 'flops': n * (30 if case['train'] else 12)}
    rows = case['batch'] * case['features']
    n = rows * case['length']
    tensors = 6 if case['train'] else 3
    states = 1 + (1 + (2 if case['train'] else 0) if case['state'] else 0)
    return {'bytes': tensors * n * size + states * 4 * rows, 'flops': n * (25 if case['train'] else 10)}


def exact(case, seed):
    s = _inputs(case, seed)
    if case['op'] == 'adamw':
        b1, b2, t = BETA1, BETA2, FIRST_STEP + 1
        g = s['g'].double()
        if case['clip']:
            g = g * min(1.0, CLIP / float(torch.linalg.vector_norm(g)))
        if case['bits'] == 8:
            old_m = s['m'].double() * s['m_scale'].double().repeat_interleave(BLOCK)
            old_v = (s['r'].double() * s['r_scale'].double().repeat_interleave(BLOCK)) ** 2
        else:
            old_m, old_v = s['m'].double(), s['v'].double()
        m, v = torch.lerp(g, old_m, b1), torch.lerp(g * g, old_v, b2)
        step = (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + EPS / math.sqrt(1 - b2 ** t))
        w = s['w'].double() * (1 - LR * s['decay']).repeat_interleave(BLOCK) - LR * step
        if case['bits'] == 32:
            return {'w': w, 'm': m, 'v': v}
        # the codes come of a rounding whose borders 64 bits place elsewhere: they have no value of their own here
        return {'w': w, 'm': None, 'r': None, 'm_scale': m.abs().view(-1, BLOCK).amax(1).clamp(min=2.0 ** -100) / 256,
                'r_scale': v.sqrt().view(-1, BLOCK).amax(1).clamp(min=2.0 ** -100) / 256}
    if case['op'] == 'groupnorm':
        leaves = [s[k].double().requires_grad_(case['train']) for k in ('x', 'gamma', 'beta')]
        x, gamma, beta = leaves
        u = torch.nn.functional.group_norm(x.permute(0, 3, 1, 2), case['groups'], gamma, beta, 1e-3).permute(0, 2, 3, 1)
        act = {'none': lambda v: v, 'relu': torch.relu, 'silu': torch.nn.functional.silu, 'gelu': torch.nn.functional.gelu}
        y = act[case['activation']](u)
        if not case['train']:
            return {'y': y}
        dx, dgamma, dbeta = torch.autograd.grad(y, leaves, s['gy'].double())
        return {'y': y.detach(), 'dx': dx, 'dgamma': dgamma, 'dbeta': dbeta}
    x, z = s['x'].double(), s['z'].double()
    gate, length = torch.sigmoid(z), x.shape[1]
    ends = s['lengths'] if s['lengths'] is not None else torch.full((x.shape[0],), length, device='cuda')
    h = torch.zeros_like(x[:, 0]) if s['h0'] is None else s['h0'].double()
    before, out = torch.empty_like(x), torch.zeros_like(x)
    for t in range(length):
        before[:, t] = h
        h = torch.where((t < ends)[:, None], torch.lerp(x[:, t], h, gate[:, t]), h)
        out[:, t] = h
    live = torch.arange(length, device='cuda')[None, :, None] < ends[:, None, None]
    result = {'h': out * live, 'h_last': h}
    if case['train']:
        lam = torch.zeros_like(h) if s['g_last'] is None else s['g_last'].double()
        dx, dz = torch.zeros_like(x), torch.zeros_like(x)
        gh = s['gh'].double()
        for t in range(length - 1, -1, -1):
            here = (t < ends)[:, None]
            total = lam + gh[:, t]
            dx[:, t] = torch.where(here, total * torch.sigmoid(-z[:, t]), 0.0)
            dz[:, t] = torch.where(here, total * gate[:, t] * torch.sigmoid(-z[:, t]) * (before[:, t] - x[:, t]), 0.0)
            lam = torch.where(here, total * gate[:, t], lam)
        result.update(dx=dx, dz=dz)
        if s['h0'] is not None:
            result['dh0'] = lam
    return result
