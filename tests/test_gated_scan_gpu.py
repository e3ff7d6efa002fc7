"""The gated linear recurrence (``kernels.gated_scan_fwd`` / ``_bwd``) against its definition in 64 bits."""

import pytest
import torch

gpu = pytest.mark.gpu
U = 2.0 ** -24
HALF_STEP = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}

SHAPES = [  # (batch, time, features)
    (1, 1, 1), (64, 1, 256), (3, 2, 33), (2, 15, 7), (2, 16, 32), (2, 17, 64), (5, 31, 100), (700, 64, 64), (3, 255, 40), (2, 256, 32),
    (2, 257, 31), (1, 1000, 5), (1, 4097, 70), (2, 3001, 300), (40, 300, 129), (1, 20000, 3), (0, 5, 8), (3, 0, 8), (4, 9, 0),
]


def reference(x, z, h0, lengths, gh, g_last):
    """The definition step by step in fp64 (on the CPU: long axes are many small steps)."""
    dev = x.device
    x, z = x.double().cpu(), z.double().cpu()
    B, T, D = x.shape
    ends = torch.full((B,), T) if lengths is None else lengths.cpu().clamp(0, T)
    h = torch.zeros(B, D, dtype=torch.float64) if h0 is None else h0.double().cpu()
    a, c = torch.sigmoid(z), torch.sigmoid(-z)
    out, before = torch.zeros_like(x), torch.zeros_like(x)
    size = h.abs()  # the same recurrence on magnitudes: what rounding errors scale with
    sizes = torch.zeros_like(x)
    for t in range(T):
        live = (t < ends)[:, None]
        before[:, t] = h
        h = torch.where(live, a[:, t] * h + c[:, t] * x[:, t], h)
        size = torch.where(live, a[:, t] * size + c[:, t] * x[:, t].abs(), size)
        out[:, t] = torch.where(live, h, 0.0)
        sizes[:, t] = size
    res = {'h': out, 'h_last': h, 'size': sizes, 'size_last': size}
    if gh is not None:
        g = gh.double().cpu()
        mu = torch.zeros(B, D, dtype=torch.float64) if g_last is None else g_last.double().cpu()
        size_mu = mu.abs()
        dx, dz, sdx, sdz = (torch.zeros_like(x) for _ in range(4))
        for t in range(T - 1, -1, -1):
            live = (t < ends)[:, None]
            lam, slam = mu + g[:, t], size_mu + g[:, t].abs()
            dx[:, t] = torch.where(live, c[:, t] * lam, 0.0)
            dz[:, t] = torch.where(live, a[:, t] * c[:, t] * lam * (before[:, t] - x[:, t]), 0.0)
            sdx[:, t] = c[:, t] * slam
            prev = sizes[:, t - 1] if t else (torch.zeros_like(h) if h0 is None else h0.double().cpu().abs())
            sdz[:, t] = a[:, t] * c[:, t] * slam * (prev + x[:, t].abs())
            mu = torch.where(live, a[:, t] * lam, mu)
            size_mu = torch.where(live, a[:, t] * slam, size_mu)
        res.update(dx=dx, dz=dz, dh0=mu, size_dx=sdx, size_dz=sdz, size_dh0=size_mu)
    return {k: v.to(dev) for k, v in res.items()}


def close(got, value, size, dtype, memory, what):
    """A gate and its complement are good to 4 ulps, a step rounds twice more, and errors decay with the state: a step's relative
    error of 6 U is carried for 1 / (1 - a) steps on average (``memory`` bounds that for these gates), folding the runs and
    tiles doubles it."""
    allowed = 2 * 6 * U * memory * size + HALF_STEP[dtype] * (value.abs() + 12 * U * memory * size) + TINY[dtype] + 1e-37
    d = (got.double() - value).abs()
    assert bool((d <= allowed).all()), f'{what}: {float((d / allowed).max()):.2f} of the bound'


def inputs(shape, dtype, seed, spread=1.5, centre=1.0):
    B, T, D = shape
    gen = torch.Generator(device='cuda').manual_seed(seed)
    n = lambda *s: torch.randn(s, device='cuda', generator=gen)  # noqa: E731
    x, z, gh = n(B, T, D).to(dtype), (centre + spread * n(B, T, D)).to(dtype), n(B, T, D).to(dtype)
    return x, z, gh, n(B, D), n(B, D)


@gpu
@pytest.mark.parametrize('dtype', list(HALF_STEP), ids=str)
@pytest.mark.parametrize('index', range(len(SHAPES)), ids=lambda i: 'x'.join(map(str, SHAPES[i])))
@pytest.mark.parametrize('padded', [False, True])
def test_forward_and_backward(index, dtype, padded):
    from hgq2_b200 import kernels as K

    shape = SHAPES[index]
    B, T, D = shape
    x, z, gh, h0, g_last = inputs(shape, dtype, index)
    if index % 3 == 1:
        h0 = None
    if index % 3 == 2:
        g_last = None
    lengths = None
    if padded:
        lengths = torch.randint(0, T + 1, (B,), device='cuda', generator=torch.Generator(device='cuda').manual_seed(index))
        if B > 1:
            lengths[0], lengths[1] = 0, T
        dead = torch.arange(T, device='cuda')[None, :] >= lengths[:, None]
        x[dead], z[dead], gh[dead] = float('nan'), float('inf'), float('nan')  # what stands behind a row's end is not looked at
    want = reference(torch.nan_to_num(x), torch.nan_to_num(z), h0, lengths, torch.nan_to_num(gh), g_last)
    h, h_last, states = K.gated_scan_fwd(x, z, h0, lengths, want_states=True)
    assert h.dtype == dtype and h.shape == shape and h_last.shape == (B, D)
    close(h, want['h'], want['size'], dtype, 40, 'h')
    close(h_last, want['h_last'], want['size_last'], torch.float32, 40, 'h_last')
    dx, dz, dh0 = K.gated_scan_bwd(gh, x, z, h0, lengths, states, g_last, want_dh0=True)
    close(dx, want['dx'], want['size_dx'], dtype, 80, 'dx')
    close(dz, want['dz'], want['size_dz'], dtype, 160, 'dz')
    close(dh0, want['dh0'], want['size_dh0'], torch.float32, 80, 'dh0')
    # without states the forward is the same, and everything repeats bit for bit
    again, last, none = K.gated_scan_fwd(x, z, h0, lengths)
    assert none is None and torch.equal(h, again) and torch.equal(h_last, last)
    assert all(torch.equal(a, b) for a, b in zip((dx, dz), K.gated_scan_bwd(gh, x, z, h0, lengths, states, g_last)))


ROWS = [(5, T, D) for T in (1, 3, 70, 900) for D in (7, 9, 10, 11, 63, 65, 127)]
# as many channels as fill the chip a little more than once with one of them a lane, for each number of warps along time
ROWS += [(B, T, D) for B, T in ((1000, 1), (500, 10), (250, 30), (125, 64), (125, 200)) for D in (130, 131)] + [(100, 200, 254)]


@gpu
@pytest.mark.parametrize('dtype', list(HALF_STEP), ids=str)
@pytest.mark.parametrize('inside', [True, False])
@pytest.mark.parametrize('shape', ROWS, ids=lambda s: 'x'.join(map(str, s)))
def test_rows_that_pairs_do_not_fit(shape, inside, dtype):
    """A row's last feature alone, or (with an odd base, inside a wider tensor) every pair across an access boundary."""
    from hgq2_b200 import kernels as K

    B, T, D = shape
    x, z, gh, h0, g_last = inputs((B, T, D), dtype, D)
    lengths = torch.tensor([T, 0, T // 2, T, 1] * (B // 5), device='cuda')
    out = None
    if inside:
        wide = torch.full((B, T, 2 * D + 3), 7.0, device='cuda', dtype=dtype)
        wide[..., 1:D + 1], wide[..., D + 2:-1] = x, z
        x, z = wide[..., 1:D + 1], wide[..., D + 2:-1]
        out = torch.full_like(wide, 7.0)
    want = reference(x, z, h0, lengths, gh, g_last)
    h, h_last, states = K.gated_scan_fwd(x, z, h0, lengths, want_states=True)
    close(h, want['h'], want['size'], dtype, 40, 'h')
    close(h_last, want['h_last'], want['size_last'], torch.float32, 40, 'h_last')
    into = {'out_dx': out[..., 1:D + 1], 'out_dz': out[..., D + 2:-1]} if inside else {}
    dx, dz, dh0 = K.gated_scan_bwd(gh, x, z, h0, lengths, states, g_last, want_dh0=True, **into)
    close(dx, want['dx'], want['size_dx'], dtype, 80, 'dx')
    close(dz, want['dz'], want['size_dz'], dtype, 160, 'dz')
    close(dh0, want['dh0'], want['size_dh0'], torch.float32, 80, 'dh0')
    if inside:
        assert bool((out[..., [0, D + 1, -1]] == 7).all())


@gpu
@pytest.mark.parametrize('dtype', list(HALF_STEP), ids=str)
def test_tokens_one_by_one_equal_the_sequence(dtype):
    """Serving: the state carried from token to token gives the sequence's outputs."""
    from hgq2_b200 import kernels as K

    x, z, _, h0, _ = inputs((6, 40, 50), dtype, 1)
    h, h_last, _ = K.gated_scan_fwd(x, z, h0)
    state, out = h0, []
    for t in range(40):
        y, state, _ = K.gated_scan_fwd(x[:, t:t + 1], z[:, t:t + 1], state)
        out.append(y)
    want = reference(x, z, h0, None, None, None)
    close(torch.cat(out, 1), want['h'], want['size'], dtype, 40, 'token by token')
    close(state, want['h_last'], want['size_last'], torch.float32, 40, 'state')
    # pieces of a sequence: a prompt of 23, then the rest
    a, s, _ = K.gated_scan_fwd(x[:, :23], z[:, :23], h0)
    b, s, _ = K.gated_scan_fwd(x[:, 23:], z[:, 23:], s)
    close(torch.cat([a, b], 1), want['h'], want['size'], dtype, 40, 'in two pieces')


@gpu
@pytest.mark.parametrize('T', [1, 40, 700, 9000])
def test_slices_of_a_wider_projection_are_read_in_place(T):
    from hgq2_b200 import kernels as K

    gen = torch.Generator(device='cuda').manual_seed(2)
    p = torch.randn(3, T, 100, device='cuda', generator=gen)
    x, z = p[..., :45], p[..., 50:95]
    g = torch.randn(T, 3, 45, device='cuda', generator=gen).transpose(0, 1)  # time-major
    h, last, states = K.gated_scan_fwd(x, z, want_states=True)
    hc, lc, sc = K.gated_scan_fwd(x.contiguous(), z.contiguous(), want_states=True)
    assert torch.equal(h, hc) and torch.equal(last, lc) and torch.equal(states, sc)
    got = K.gated_scan_bwd(g, x, z, None, None, states)
    want = K.gated_scan_bwd(g.contiguous(), x.contiguous(), z.contiguous(), None, None, sc)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    both = torch.full_like(p, 7.0)  # and gradients into the slices of one
    K.gated_scan_bwd(g, x, z, None, None, states, out_dx=both[..., :45], out_dz=both[..., 50:95])
    assert torch.equal(both[..., :45], want[0]) and torch.equal(both[..., 50:95], want[1])
    assert bool((both[..., 45:50] == 7).all() and (both[..., 95:] == 7).all())
    # a broadcast gradient (time stride 0) and features with a stride (copied)
    e = g[:, :1].expand(3, T, 45)
    assert torch.equal(K.gated_scan_bwd(e, x, z, None, None, states)[0], K.gated_scan_bwd(e.contiguous(), x, z, None, None, states)[0])
    q = torch.randn(3, 45, T, device='cuda', generator=gen).transpose(1, 2)
    assert torch.equal(K.gated_scan_fwd(q, z)[0], K.gated_scan_fwd(q.contiguous(), z)[0])


@gpu
@pytest.mark.parametrize('kind', [torch.int8, torch.uint8, torch.int16, torch.int64])
def test_lengths_of_any_whole_type(kind):
    from hgq2_b200 import kernels as K

    x, z, _, h0, _ = inputs((4, 300, 16), torch.float32, 8)
    lengths = torch.tensor([0, 5, 100, 127], device='cuda')
    want = K.gated_scan_fwd(x, z, h0, lengths.to(torch.int32))
    got = K.gated_scan_fwd(x, z, h0, lengths.to(kind))
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
    far = K.gated_scan_fwd(x, z, h0, torch.tensor([-7, 5, 100, 1 << 40], device='cuda'))  # clamped to [0, T]
    assert torch.equal(far[0][:3], want[0][:3]) and torch.equal(far[0][3], K.gated_scan_fwd(x, z, h0)[0][3])


@gpu
def test_long_sequences_with_wide_and_narrow_rows():
    """The same values through 16-byte pieces fetched ahead, pairs and single channels: the access widths agree to the bit."""
    from hgq2_b200 import kernels as K

    for dtype in HALF_STEP:
        x, z, gh, h0, g_last = inputs((3, 1500, 48), dtype, 9)
        h, last, st = K.gated_scan_fwd(x, z, h0, want_states=True)
        grads = K.gated_scan_bwd(gh, x, z, h0, None, st, g_last, want_dh0=True)
        for pad, skip in ((4, 0), (4, 4), (2, 0), (2, 2), (1, 1)):  # strides and offsets that allow four, two, or single channels
            buf = [torch.zeros(3, 1500, 48 + pad + skip, device='cuda', dtype=dtype) for _ in range(3)]
            views = [b[..., skip:skip + 48] for b in buf]
            for v, t in zip(views, (x, z, gh)):
                v.copy_(t)
            h2, last2, st2 = K.gated_scan_fwd(views[0], views[1], h0, want_states=True)
            got = K.gated_scan_bwd(views[2], views[0], views[1], h0, None, st2, g_last, want_dh0=True)
            assert torch.equal(h, h2) and torch.equal(last, last2) and torch.equal(st, st2)
            assert all(torch.equal(a, b) for a, b in zip(grads, got))


@gpu
@pytest.mark.parametrize('T', [1, 50, 5000])
def test_only_the_last_state_has_a_gradient(T):
    from hgq2_b200 import kernels as K

    x, z, _, h0, g_last = inputs((2, T, 33), torch.float32, 7)
    _, _, st = K.gated_scan_fwd(x, z, h0, want_states=True)
    got = K.gated_scan_bwd(None, x, z, h0, None, st, g_last, want_dh0=True)
    want = K.gated_scan_bwd(torch.zeros_like(x), x, z, h0, None, st, g_last, want_dh0=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@gpu
def test_offsets_past_32_bits():
    from hgq2_b200 import kernels as K

    B, T, D = 4200, 4096, 128
    x, z = (torch.empty(B, T, D, device='cuda', dtype=torch.bfloat16).normal_() for _ in range(2))
    assert x.numel() > 2 ** 31
    h, last, st = K.gated_scan_fwd(x, z, want_states=True)
    want = reference(x[-1:], z[-1:], None, None, x[-1:], None)
    close(h[-1:], want['h'], want['size'], torch.bfloat16, 40, 'h')
    del h
    dx, dz, _ = K.gated_scan_bwd(x, x, z, None, None, st)
    close(dx[-1:], want['dx'], want['size_dx'], torch.bfloat16, 80, 'dx')
    close(dz[-1:], want['dz'], want['size_dz'], torch.bfloat16, 160, 'dz')


@gpu
def test_gates_at_their_ends():
    """A gate of exactly 0 forgets, of exactly 1 keeps; very long memory stays accurate."""
    from hgq2_b200 import kernels as K

    x = torch.randn(2, 600, 40, device='cuda')
    z = torch.full_like(x, float('inf'))
    h0 = torch.randn(2, 40, device='cuda')
    assert torch.equal(K.gated_scan_fwd(x, z, h0)[0], h0[:, None].expand_as(x))
    z[:, 300:] = float('-inf')
    h, _, st = K.gated_scan_fwd(x, z, h0, want_states=True)
    assert torch.equal(h[:, 300:], x[:, 300:])
    dx, dz, dh0 = K.gated_scan_bwd(torch.ones_like(x), x, z, h0, None, st, want_dh0=True)
    assert torch.equal(dx[:, 300:], torch.ones_like(dx[:, 300:])) and not bool(dx[:, :300].any()) and not bool(dz.any())
    assert torch.equal(dh0, torch.full_like(dh0, 300.0))
    z = torch.full_like(x, 12.0)  # 1 - a = 6e-6: memory of 160000 steps, longer than the sequence
    want = reference(x, z, h0, None, torch.ones_like(x), None)
    h, _, st = K.gated_scan_fwd(x, z, h0, want_states=True)
    close(h, want['h'], want['size'], torch.float32, 600, 'long memory')
    dx, dz, dh0 = K.gated_scan_bwd(torch.ones_like(x), x, z, h0, None, st, want_dh0=True)
    close(dx, want['dx'], want['size_dx'], torch.float32, 600, 'dx of long memory')
    close(dz, want['dz'], want['size_dz'], torch.float32, 1200, 'dz of long memory')


@gpu
def test_gradients_against_differences():
    from hgq2_b200 import kernels as K

    x, z, gh, h0, g_last = inputs((2, 37, 9), torch.float32, 3)
    _, _, st = K.gated_scan_fwd(x, z, h0, want_states=True)
    grads = K.gated_scan_bwd(gh, x, z, h0, None, st, g_last, want_dh0=True)
    leaves = [t.double() for t in (x, z, h0)]

    def value(ts):
        r = reference(ts[0], ts[1], ts[2], None, None, None)
        return float((r['h'] * gh.double()).sum() + (r['h_last'] * g_last.double()).sum())

    gen = torch.Generator(device='cuda').manual_seed(4)
    for which in range(3):
        v = torch.randn(leaves[which].shape, device='cuda', generator=gen, dtype=torch.float64)
        up, down = ([t + s * 1e-5 * v if i == which else t for i, t in enumerate(leaves)] for s in (1, -1))
        diff = (value(up) - value(down)) / 2e-5
        products = grads[which].double() * v
        assert abs(diff - float(products.sum())) <= 1e-5 * float(products.abs().sum())


@gpu
def test_captured_on_another_stream_and_two_at_once():
    from hgq2_b200 import kernels as K

    cases = [inputs((2, 5000, 64), torch.bfloat16, 5), inputs((300, 70, 64), torch.float32, 6)]

    def both(x, z, gh, h0, g_last):
        h, last, st = K.gated_scan_fwd(x, z, h0, want_states=True)
        return (h, last, *K.gated_scan_bwd(gh, x, z, h0, None, st, g_last, want_dh0=True))

    want = [t.clone() for c in cases for t in both(*c)]
    torch.cuda.synchronize()
    got = []
    for c in cases:
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(5):
                r = both(*c)
            got += r
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs, outs = [], []
    for c in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs += both(*c)
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

    x = torch.zeros(2, 300, 8, device='cuda')
    h0 = torch.zeros(2, 8, device='cuda')
    for kw in (dict(z=x[:1]), dict(z=x.bfloat16()), dict(x=x[0]), dict(x=x.double(), z=x.double()), dict(h0=h0[:1]),
               dict(h0=h0.bfloat16()), dict(lengths=torch.zeros(3, device='cuda', dtype=torch.int32)), dict(lengths=h0[:, 0])):
        args = dict(x=x, z=x)
        args.update(kw)
        with pytest.raises(ValueError):
            K.gated_scan_fwd(**args)
    with pytest.raises(RuntimeError, match='CUDA tensors only'):
        K.gated_scan_fwd(x, x, lengths=torch.zeros(2, dtype=torch.int32))
    _, _, st = K.gated_scan_fwd(x, x, want_states=True)
    assert st.numel() > 0
    for kw in (dict(gh=x[:1]), dict(gh=x.bfloat16()), dict(states=None), dict(states=st[1:]), dict(g_last=h0[:1]), dict(out_dx=x[:1]), dict(out_dz=x.bfloat16())):
        args = dict(gh=x, x=x, z=x, states=st)
        args.update(kw)
        with pytest.raises(ValueError):
            K.gated_scan_bwd(**args)


def test_refusals_need_no_gpu():
    from hgq2_b200 import _lib, build
    from hgq2_b200 import kernels as K

    with pytest.raises(RuntimeError, match='CUDA tensors only'):
        K.gated_scan_fwd(torch.zeros(2, 3, 8), torch.zeros(2, 3, 8))
    build.build()
    L = _lib.lib()
    p = 4096  # never dereferenced: every call below is refused on the host

    def fwd(x=p, last=p, B=1, T=30000, D=8, kind=0, ws=p, nbytes=1 << 30):
        return L.hgq_gated_scan_fwd(x, 1, 1, p, 1, 1, None, None, p, last, None, B, T, D, kind, ws, nbytes, None)

    def bwd(states=p, B=1, T=30000, D=8, kind=0, ws=p, nbytes=1 << 30):
        return L.hgq_gated_scan_bwd(p, 1, 1, p, 1, 1, p, 1, 1, None, None, states, None, p, 1, 1, p, 1, 1, None, B, T, D, kind, ws, nbytes,
                                    None)

    assert fwd(x=None) == -1 and fwd(last=None) == -1 and bwd(states=None) == -1
    assert fwd(B=-1) == -2 and fwd(T=-1) == -2 and fwd(D=-1) == -2 and fwd(T=1 << 62) == -2 and fwd(B=1 << 40) == -2
    assert fwd(kind=3) == -3 and bwd(kind=-1) == -3
    assert fwd(x=p + 2) == -4 and fwd(kind=1, x=p + 1) == -4 and bwd(states=p + 2) == -4
    need = L.hgq_gated_scan_workspace(1, 30000, 8)
    assert need > 0 and fwd(nbytes=need - 1) == -5 and bwd(ws=None) == -5
    assert fwd(B=0) == 0 and bwd(D=0) == 0
    assert L.hgq_gated_scan_workspace(4096, 64, 64) == 0 and L.hgq_gated_scan_states(4096, 64, 64) == 0


@gpu
def test_gates_to_relative_precision():
    """fp32 gates and their complements over the range where both are normal numbers: one step from x = 0, h0 = 1 gives a, one
    from x = 1, h0 = 0 gives c.  Counted in U = 2^-24: 2^x within 2 ulps (5 U), its correction (1), 1 + e (1), the reciprocal within an ulp
    (3), the product (1), and where c = 1 - a another rounding: at most 12 U."""
    from hgq2_b200 import kernels as K

    n = 1 << 20
    z = torch.linspace(-85, 85, n, device='cuda').view(1, 1, n)
    zero, one = torch.zeros_like(z), torch.ones_like(z)
    a = K.gated_scan_fwd(zero, z, one[:, 0])[0].double()
    c = K.gated_scan_fwd(one, z, zero[:, 0])[0].double()
    e = torch.exp(-z.double())
    for got, want, what in ((a, 1 / (1 + e), 'a'), (c, e / (1 + e), 'c')):
        off = ((got - want) / want).abs()
        assert float(off.max()) <= 12 * U, f'{what}: {float(off.max()) / U:.1f} U at z = {float(z.view(-1)[off.argmax()]):.2f}'


@gpu
def test_lengths_that_32_bits_do_not_hold():
    """Lengths travel as int32: an axis longer than that takes no wider ones (they would wrap), but narrower ones and none."""
    from hgq2_b200 import kernels as K

    T = 2 ** 31 + 8
    x = torch.ones(1, 1, 1, device='cuda', dtype=torch.float16).expand(1, T, 1)
    with pytest.raises(ValueError, match='int32'):
        K.gated_scan_fwd(x, x, lengths=torch.tensor([2 ** 31 + 4], device='cuda'))
    h0 = torch.full((1, 1), 3.0, device='cuda')
    h, last, _ = K.gated_scan_fwd(x, x, h0, lengths=torch.zeros(1, dtype=torch.int32, device='cuda'))
    assert torch.equal(last, h0) and not bool(h[:, -1000:].any()) and not bool(h[:, :1000].any())


@gpu
def test_gradients_into_a_tensor_that_overlaps_itself():
    """Steps or rows of an output that share memory would be written in no order: refused."""
    from hgq2_b200 import kernels as K

    x = torch.randn(2, 5, 8, device='cuda')
    row = torch.zeros(2, 5, 8, device='cuda')
    for out in (row[:, :1].expand(2, 5, 8), row[:1].expand(2, 5, 8), row.view(-1).as_strided((2, 5, 8), (40, 4, 1)),
                row.view(-1).as_strided((2, 5, 8), (7, 16, 1)), row.view(-1).as_strided((2, 5, 8), (8, 8, 1)),
                row.view(-1).as_strided((2, 5, 8), (20, 9, 1))):
        for name in ('out_dx', 'out_dz'):
            with pytest.raises(ValueError, match='share memory'):
                K.gated_scan_bwd(x, x, x, **{name: out})
    one = K.gated_scan_bwd(x[:1, :1], x[:1, :1], x[:1, :1], out_dx=row[:1, :1].as_strided((1, 1, 8), (0, 0, 1)))  # nothing to share
    assert torch.equal(one[0], K.gated_scan_bwd(x[:1, :1], x[:1, :1], x[:1, :1])[0])
    turned = torch.zeros(5, 2, 8, device='cuda').transpose(0, 1)  # time-major
    assert torch.equal(K.gated_scan_bwd(x, x, x, out_dx=turned)[0], K.gated_scan_bwd(x, x, x)[0])
    woven = torch.zeros(16, device='cuda').as_strided((2, 3, 2), (6, 4, 1))  # rows at 0, 4, 8 and 6, 10, 14
    y = x[:, :3, :2]
    assert torch.equal(K.gated_scan_bwd(y, y, y, out_dz=woven)[1], K.gated_scan_bwd(y, y, y)[1])


def test_rows_that_meet_are_found():
    """Against the set of places that the rows touch, over all small shapes and strides."""
    import itertools

    from hgq2_b200.kernels import _rows_meet

    buf = torch.empty(200)
    for B, T, D in itertools.product((1, 2, 3, 4), (1, 2, 3), (1, 2, 3)):
        for sb, st in itertools.product(range(11), range(11)):
            places = [b * sb + t * st + d for b in range(B) for t in range(T) for d in range(D)]
            assert _rows_meet(buf.as_strided((B, T, D), (sb, st, 1))) == (len(set(places)) < len(places)), (B, T, D, sb, st)
    assert not _rows_meet(torch.empty(0, 3, 4)) and not _rows_meet(torch.empty(2, 0, 4)) and not _rows_meet(torch.empty(2, 3, 0))
