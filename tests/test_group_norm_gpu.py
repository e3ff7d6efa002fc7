"""Group normalisation with an activation (``kernels.group_norm_fwd`` / ``_bwd`` and the layer) against its definition in 64 bits."""

import math

import pytest
import torch

gpu = pytest.mark.gpu
U = 2.0 ** -24
HALF_STEP = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}  # half of fp16's smallest subnormal

SHAPES = [  # (batch, spatial, channels, groups)
    (2, (5, 7), 12, 3), (1, (1,), 4, 4), (3, (1,), 8, 2), (2, (64,), 64, 8), (2, (30, 30), 16, 4), (1, (67, 65), 96, 32),
    (4, (3, 3), 37, 1), (2, (9,), 6, 6), (1, (300,), 1, 1), (2, (2, 2), 2048, 4), (1, (40, 40), 1030, 2), (5, (4, 4), 64, 8),
    (1, (129, 127), 24, 24), (300, (2,), 16, 2), (3, (), 128, 4), (1, (700,), 520, 260), (2, (33, 31), 10, 5), (700, (4, 4), 8, 2),
    (2, (200, 100), 64, 1), (1, (3, 1025, 7), 40, 20),
    # channel counts that 16-byte accesses do not divide: rows joined, or not where their number does not allow it
    (3, (8, 8), 37, 37), (2, (16,), 45, 9), (5, (4, 4), 20, 5), (300, (8,), 3, 1), (2, (40, 30), 21, 7), (2, (24,), 255, 5),
    (400, (12,), 45, 3), (3, (30, 30), 44, 11),
]


def act64(u, name):
    if name == 'relu':
        return torch.where(u < 0, torch.zeros_like(u), u), (u > 0).double()
    if name == 'silu':
        p = torch.sigmoid(u)
        return u * p, p * (1 + u * (1 - p))
    if name == 'gelu':
        cdf = 0.5 * (1 + torch.erf(u / math.sqrt(2)))
        return u * cdf, cdf + u * torch.exp(-u * u / 2) / math.sqrt(2 * math.pi)
    return u, torch.ones_like(u)


def reference(x, gamma, beta, groups, eps, act, gy):
    """The definition in fp64, with bounds on an fp32 evaluation's distance."""
    B, C = x.shape[0], x.shape[-1]
    xd = x.double().reshape(B, -1, groups, C // groups)
    ga = (torch.ones(C, device=x.device) if gamma is None else gamma).double().view(groups, -1)
    be = (torch.zeros(C, device=x.device) if beta is None else beta).double().view(groups, -1)
    mean = xd.mean((1, 3), keepdim=True)
    var = (xd - mean).square().mean((1, 3), keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    xh = (xd - mean) * rstd
    u = xh * ga + be
    y, slope = act64(u, act)
    # xhat: the mean is held in fp32 (U |mean| rstd) and comes of sums of numbers near it; the difference, the variance (sums of up
    # to 200 terms a thread, exact across threads), the root and the products add a few dozen roundings of |xhat|
    dxh = U * (250 * xh.abs() + 4 * mean.abs() * rstd + 200 * rstd * (xd - mean).abs().mean((1, 3), keepdim=True) + 4)
    du_ = ga.abs() * dxh + 4 * U * (u.abs() + be.abs())
    dy = 1.2 * du_ + 8 * U * (y.abs() + u.abs())
    out = {'y': (y, dy), 'mean': mean.view(B, groups), 'rstd': rstd.view(B, groups)}
    if gy is not None:
        g = gy.double().reshape(xd.shape)
        du = g * slope
        # slopes bend by at most 1.1 (GELU) per unit of u; their own evaluation is good to a few ulps of 1
        ddu = g.abs() * (1.1 * du_ + 16 * U) if act not in (None, 'relu') else 2 * U * du.abs()
        dxh_, ddxh = du * ga, ddu * ga.abs() + U * (du * ga).abs()
        m1, m2 = dxh_.mean((1, 3), keepdim=True), (dxh_ * xh).mean((1, 3), keepdim=True)
        dm1 = ddxh.mean((1, 3), keepdim=True) + 250 * U * dxh_.abs().mean((1, 3), keepdim=True)
        dm2 = (ddxh * xh.abs() + dxh_.abs() * dxh).mean((1, 3), keepdim=True) + 250 * U * (dxh_ * xh).abs().mean((1, 3), keepdim=True)
        dx = rstd * (dxh_ - m1 - xh * m2)
        ddx = rstd * (ddxh + dm1 + xh.abs() * dm2 + m2.abs() * dxh + 250 * U * (dxh_.abs() + m1.abs() + (xh * m2).abs()))
        out['dx'] = (dx, ddx)
        out['dbeta'] = (du.sum((0, 1)).view(C), (ddu + 400 * U * du.abs()).sum((0, 1)).view(C))
        out['dgamma'] = ((du * xh).sum((0, 1)).view(C),
                         (ddu * xh.abs() + du.abs() * dxh + 400 * U * (du * xh).abs()).sum((0, 1)).view(C))
    return out


def close(got, want, what):
    value, off = want
    value, off = value.reshape(got.shape), off.reshape(got.shape)
    allowed = off + HALF_STEP[got.dtype] * (value.abs() + off) + TINY[got.dtype] + 1e-37
    d = (got.double() - value).abs()
    worst = (d / allowed).max() if d.numel() else torch.zeros(())
    assert bool((d <= allowed).all()), f'{what}: {float(worst):.2f} of the bound'


def inputs(shape, dtype, act, seed=0, offset=True):
    B, spatial, C, G = shape
    gen = torch.Generator(device='cuda').manual_seed(seed)
    x = (torch.randn((B, *spatial, C), device='cuda', generator=gen) * 2 + (1.5 if offset else 0)).to(dtype)
    gamma, beta = torch.randn(C, device='cuda', generator=gen), torch.randn(C, device='cuda', generator=gen)
    gy = torch.randn(x.shape, device='cuda', generator=gen).to(dtype)
    if act == 'relu':  # the slope at the corner is decided by the last bit: no output gradient there
        u = reference(x, gamma, beta, G, 1e-3, None, None)['y'][0].reshape(x.shape)
        gy = torch.where(u.abs() < 1e-3, torch.zeros_like(gy), gy)
    return x, gamma, beta, gy


@gpu
@pytest.mark.parametrize('dtype', list(HALF_STEP), ids=str)
@pytest.mark.parametrize('index', range(len(SHAPES)), ids=lambda i: 'x'.join(map(str, (SHAPES[i][0], *SHAPES[i][1], *SHAPES[i][2:]))))
def test_forward_and_backward(index, dtype):
    from hgq2_b200 import kernels as K

    shape = SHAPES[index]
    act = (None, 'relu', 'silu', 'gelu')[index % 4]
    x, gamma, beta, gy = inputs(shape, dtype, act, index)
    G = shape[3]
    if index % 5 == 1:
        gamma = None
    if index % 5 == 2:
        beta = None
    want = reference(x, gamma, beta, G, 1e-3, act, gy)
    y, mean, rstd = K.group_norm_fwd(x, gamma, beta, G, 1e-3, act)
    assert y.dtype == dtype and y.shape == x.shape
    close(y, want['y'], 'y')
    dx, dgamma, dbeta = K.group_norm_bwd(gy, x, gamma, beta, mean, rstd, G, act)
    close(dx, want['dx'], 'dx')
    close(dgamma, want['dgamma'], 'dgamma')
    close(dbeta, want['dbeta'], 'dbeta')
    # parts of the backward alone, and again: the same bits
    dx2, none, _ = K.group_norm_bwd(gy, x, gamma, beta, mean, rstd, G, act, want_params=False)
    assert none is None and torch.equal(dx, dx2)
    none, dg2, db2 = K.group_norm_bwd(gy, x, gamma, beta, mean, rstd, G, act, want_dx=False)
    assert none is None and torch.equal(dg2, dgamma) and torch.equal(db2, dbeta)


@gpu
@pytest.mark.parametrize('dtype', list(HALF_STEP), ids=str)
def test_misaligned_and_strided_inputs(dtype):
    from hgq2_b200 import kernels as K

    gen = torch.Generator(device='cuda').manual_seed(1)
    base = torch.randn(2 * 50 * 32 + 1, device='cuda', generator=gen).to(dtype)
    x = base[1:].view(2, 50, 32)
    y, mean, rstd = K.group_norm_fwd(x, None, None, 4, 1e-3, 'silu')
    close(y, reference(x, None, None, 4, 1e-3, 'silu', None)['y'], 'misaligned')
    wide = torch.randn(2, 50, 64, device='cuda', generator=gen).to(dtype)
    s = wide[:, ::2, 16:48]
    y, mean, rstd = K.group_norm_fwd(s, None, None, 8)
    close(y, reference(s, None, None, 8, 1e-3, None, None)['y'], 'strided')
    g = torch.ones((), device='cuda', dtype=dtype).expand(s.shape)
    dx, dgamma, dbeta = K.group_norm_bwd(g, s, None, None, mean, rstd, 8)
    want = reference(s, None, None, 8, 1e-3, None, g)
    close(dx, want['dx'], 'dx of a broadcast gradient')
    close(dbeta, want['dbeta'], 'dbeta of a broadcast gradient')


@gpu
def test_large_mean_keeps_its_variance():
    from hgq2_b200 import kernels as K

    gen = torch.Generator(device='cuda').manual_seed(2)
    for shape, G in (((2, 40, 40, 16), 4), ((1, 400, 400, 8), 1), ((64, 16, 64), 8)):
        x = torch.randn(shape, device='cuda', generator=gen) + 4096
        x[:, 0] = 4090  # the first rows lie apart
        y, mean, rstd = K.group_norm_fwd(x, None, None, G)
        want = reference(x, None, None, G, 1e-3, None, None)
        close(y, want['y'], f'{shape}')
        assert bool(((rstd - want['rstd']).abs() <= 1e-4 * want['rstd']).all())


@gpu
def test_not_finite_values_stay_in_their_group():
    from hgq2_b200 import kernels as K

    for big in (False, True):
        x = torch.randn(3, *((200, 150) if big else (6, 5)), 16, device='cuda')
        x[0, 1, 2, 3] = float('nan')
        x[1, 2, 3, 7] = float('inf')
        y, _, _ = K.group_norm_fwd(x, None, None, 4, 1e-3, 'relu')
        bad = torch.isnan(y).view(3, -1, 4, 4).any(3).any(1)
        want = torch.zeros(3, 4, dtype=torch.bool, device='cuda')
        want[0, 0] = want[1, 1] = True
        assert torch.equal(bad, want)


@gpu
def test_offsets_past_32_bits():
    """2.2e9 elements in samples that fit on the chip and in images that do not: the last sample's last group is right."""
    from hgq2_b200 import kernels as K

    for B, S, C, G in ((16500, 2048, 64, 8), (3, 11300, 65536, 64)):
        x = torch.empty(B, S, C, device='cuda', dtype=torch.bfloat16).normal_()
        assert x.numel() > 2 ** 31
        y, mean, rstd = K.group_norm_fwd(x, None, None, G, 1e-3, 'silu')
        dx, _, dbeta = K.group_norm_bwd(x, x, None, None, mean, rstd, G, 'silu')
        gr = slice(C - C // G, C)  # the last group of the last sample
        want = reference(x[-1:, :, gr], None, None, 1, 1e-3, 'silu', x[-1:, :, gr])
        # the bound is for sums of 200 terms a thread; here they are 2048 * 64 / 512 = 256, and for the image, 8 channels a thread
        # and one wave of 148 * 512 threads or more, up to 3 * 11300 * 65536 / (148 * 512) = 29300
        more = 2 if S == 2048 else 150
        close(y[-1:, :, gr], (want['y'][0], want['y'][1] * more), 'y')
        close(dx[-1:, :, gr], (want['dx'][0], want['dx'][1] * more), 'dx')
        assert bool(torch.isfinite(dbeta).all())
        del x, y, dx, want
        torch.cuda.empty_cache()


@gpu
def test_empty_inputs():
    from hgq2_b200 import kernels as K

    for shape in ((0, 5, 8), (3, 0, 8), (2, 4, 0, 8)):
        x = torch.zeros(shape, device='cuda')
        y, mean, rstd = K.group_norm_fwd(x, None, None, 2)
        assert y.shape == x.shape and mean.shape == (shape[0], 2)
        dx, dgamma, dbeta = K.group_norm_bwd(x, x, None, None, mean, rstd, 2)
        assert dx.shape == x.shape and not bool(dgamma.any()) and not bool(dbeta.any())


@gpu
@pytest.mark.parametrize('act', [None, 'silu', 'gelu'])
def test_gradients_against_differences(act):
    """Directional differences of a scalar of the fp64 definition, along random directions, against the kernel's gradients."""
    from hgq2_b200 import kernels as K

    x, gamma, beta, gy = inputs((2, (6, 5), 12, 3), torch.float32, act, 3)
    y, mean, rstd = K.group_norm_fwd(x, gamma, beta, 3, 1e-3, act)
    grads = K.group_norm_bwd(gy, x, gamma, beta, mean, rstd, 3, act)
    leaves = [t.double() for t in (x, gamma, beta)]

    def value(ts):
        return float((reference(ts[0], ts[1], ts[2], 3, 1e-3, act, None)['y'][0].reshape(gy.shape) * gy.double()).sum())

    gen = torch.Generator(device='cuda').manual_seed(4)
    for which in range(3):
        v = torch.randn(leaves[which].shape, device='cuda', generator=gen, dtype=torch.float64)
        h = 1e-5
        up, down = ([t + s * h * v if i == which else t for i, t in enumerate(leaves)] for s in (1, -1))
        diff = (value(up) - value(down)) / (2 * h)
        dot = float((grads[which].double() * v).sum())
        size = float((grads[which].double() * v).abs().sum())
        assert abs(diff - dot) <= 1e-5 * size, (which, diff, dot)


@gpu
def test_captured_on_another_stream_and_two_at_once():
    from hgq2_b200 import kernels as K

    x, gamma, beta, gy = inputs((8, (20, 20), 32, 8), torch.float32, 'silu', 5)
    big, _, _, gbig = inputs((3, (150, 150), 32, 8), torch.float32, 'silu', 6)

    def both(x, gy):
        y, mean, rstd = K.group_norm_fwd(x, gamma, beta, 8, 1e-3, 'silu')
        return (y, *K.group_norm_bwd(gy, x, gamma, beta, mean, rstd, 8, 'silu'))

    want = [t.clone() for t in both(x, gy) + both(big, gbig)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for s, (a, b) in zip(streams, ((x, gy), (big, gbig))):
        with torch.cuda.stream(s):
            for _ in range(5):
                r = both(a, b)
            got += r
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs, outs = [], []
    for a, b in ((x, gy), (big, gbig)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs += both(a, b)
        graphs.append(g)
    for t in outs:
        t.zero_()
    for g in (*graphs, *graphs[::-1]):
        g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))


@gpu
def test_refusals_on_the_device():
    from hgq2_b200 import kernels as K

    x = torch.zeros(2, 3, 8, device='cuda')
    one = torch.ones(8, device='cuda')
    bad = [dict(groups=3), dict(groups=0), dict(groups=-1), dict(gamma=one[:4]), dict(beta=one.double()), dict(activation='tanh'),
           dict(x=x.double()), dict(x=x[0, 0]), dict(gamma=one.bfloat16())]
    for kw in bad:
        args = dict(x=x, gamma=one, beta=one, groups=2)
        args.update(kw)
        with pytest.raises(ValueError):
            K.group_norm_fwd(**args)
    _, mean, rstd = K.group_norm_fwd(x, one, one, 2)
    for gy, m, r, kw in ((x[:1], mean, rstd, {}), (x.bfloat16(), mean, rstd, {}), (x, mean[:1], rstd, {}), (x, mean, rstd.double(), {}),
                         (x, mean, rstd, dict(out_dgamma=one[:4])), (x, mean, rstd, dict(out_dbeta=one.double()))):
        with pytest.raises(ValueError):
            K.group_norm_bwd(gy, x, one, one, m, r, 2, **kw)


def test_refusals_need_no_gpu():
    from hgq2_b200 import _lib, build
    from hgq2_b200 import kernels as K

    with pytest.raises(RuntimeError, match='CUDA tensors only'):
        K.group_norm_fwd(torch.zeros(2, 3, 8), None, None, 2)
    build.build()
    L = _lib.lib()
    p = 4096  # never dereferenced: every call below is refused on the host

    def fwd(x=p, B=2, S=3, C=8, G=2, act=0, kind=0, ws=p, nbytes=1 << 20, gamma=None):
        return L.hgq_group_norm_fwd(x, gamma, None, p, p, p, B, S, C, G, 1e-3, act, kind, ws, nbytes, None)

    def bwd(gy=p, dx=p, dg=p, db=p, B=2, S=3, C=8, G=2, act=0, kind=0, ws=p, nbytes=1 << 20):
        return L.hgq_group_norm_bwd(gy, p, None, None, p, p, dx, dg, db, B, S, C, G, act, kind, ws, nbytes, None)

    assert fwd(x=None) == -1 and bwd(gy=None) == -1
    assert fwd(G=3) == -2 and fwd(C=0) == -2 and fwd(B=-1) == -2 and fwd(S=1 << 62) == -2 and bwd(G=0) == -2
    assert fwd(act=4) == -3 and fwd(kind=3) == -3 and bwd(act=-1) == -3
    assert fwd(x=p + 2) == -4 and fwd(gamma=p + 2) == -4 and bwd(dg=p + 2) == -4
    assert bwd(dg=None) == -1 and bwd(dx=None, dg=None, db=None) == -1
    need = L.hgq_group_norm_workspace(2, 3, 8, 2, 0, 0)
    if need:
        assert fwd(nbytes=need - 1) == -5 and fwd(ws=None) == -5
    assert L.hgq_group_norm_workspace(2, 3, 8, 2, 0, 1) > 0 and bwd(nbytes=4) == -5
    assert fwd(B=0) == 0 and fwd(S=0) == 0
    assert L.hgq_group_norm_workspace(2, 3, 8, 3, 0, 0) == 0


@gpu
@pytest.mark.parametrize('shape', [(16500, 2048, 64, 8), (3, 11300, 65536, 64)], ids=str)
def test_parameter_gradients_past_32_bits(shape):
    """dgamma and dbeta of the last group's channels over more than 2^31 elements."""
    from hgq2_b200 import kernels as K

    B, S, C, G = shape
    x = torch.empty(B, S, C, device='cuda', dtype=torch.bfloat16).normal_()
    assert x.numel() > 2 ** 31
    _, mean, rstd = K.group_norm_fwd(x, None, None, G, 1e-3, 'silu')
    none, dgamma, dbeta = K.group_norm_bwd(x, x, None, None, mean, rstd, G, 'silu', want_dx=False)
    for gr in (slice(0, C // G), slice(C - C // G, C)):
        totals = [torch.zeros(C // G, device='cuda', dtype=torch.float64) for _ in range(4)]
        for part in x[:, :, gr].split(500):
            want = reference(part, None, None, 1, 1e-3, 'silu', part)
            for t, v in zip(totals, (*want['dgamma'], *want['dbeta'])):
                t += v
            del want
        # the bound is for sums of a few hundred terms a thread; an image's thread adds up to 11300 / (148 * 2 / 32) = 1220 rows
        more = 1 if S == 2048 else 4
        for got, value, off in ((dgamma[gr], *totals[:2]), (dbeta[gr], *totals[2:])):
            assert bool(((got.double() - value).abs() <= off * more + U * value.abs()).all())
