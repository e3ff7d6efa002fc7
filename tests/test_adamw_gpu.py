"""AdamW over a list of tensors (``train.FusedAdamW``): one step against the formula in 64 bits, the 8-bit codes against the
fp32 formula operation by operation (they are defined to the bit), and the calls around it."""

import math

import pytest
import torch

LR, B1, B2, EPS = 1e-2, 0.9, 0.999, 1e-7
U = 2.0 ** -24  # half a step of fp32

gpu = pytest.mark.gpu


def tensors_of(sizes, dtype, gen, misaligned=False):
    out = []
    for n in sizes:
        base = torch.randn(n + 1, device='cuda', generator=gen).to(dtype)
        out.append(base[1:] if misaligned else base[:n].clone())
    return out


def set_state(opt, gen, scale=1.0):
    """A state in mid-training; returns its (m, v) in fp64, flat."""
    total = opt.m.numel()
    m, r = torch.randn(total, device='cuda', generator=gen) * scale, torch.rand(total, device='cuda', generator=gen) * scale
    if opt.state_bits == 32:
        opt.m.copy_(m)
        opt.v.copy_(r * r)
        return opt.m.double(), opt.v.double()
    for name, x in (('m', m), ('r', r)):
        s = x.view(-1, 256).abs().amax(1) / 256
        getattr(opt, name).copy_((x.view(-1, 256) / s[:, None]).to(torch.float8_e4m3fn).view(-1))
        getattr(opt, name + '_scale').copy_(s)
    return tuple(f(c.double() * s.double().repeat_interleave(256))
                 for c, s, f in ((opt.m, opt.m_scale, lambda x: x), (opt.r, opt.r_scale, lambda x: x * x)))


def want_step(w, g, m, v, t, decay, scale, l1, clip, norm):
    """(w', m', v') in fp64 and bounds on the fp32 kernel's distance from each, from counting roundings: a product or sum is off by
    U relative, a constant held in fp32 too."""
    g = g * scale + l1
    coef = min(1.0, clip / norm) if clip else 1.0
    g = g * coef
    m2, v2 = B1 * m + (1 - B1) * g, B2 * v + (1 - B2) * g * g
    # g' : scale constant, product, l1 constant, sum, coefficient, product (6); then decoding, constant, product, sum
    size_g = (g.abs() + 2 * abs(l1)) * 6 * U
    dm = 4 * U * (B1 * m.abs() + (1 - B1) * g.abs()) + (1 - B1) * size_g
    dv = 5 * U * v2 + 2 * (1 - B2) * g.abs() * size_g + B2 * v * 3 * U  # v itself: read (8 bits: two products) and squared
    alpha = LR * math.sqrt(1 - B2 ** t) / (1 - B1 ** t)
    root = v2.sqrt()
    step = alpha * m2 / (root + EPS)
    w2 = w * (1 - LR * decay) - step
    droot = dv / (2 * root.clamp(min=1e-30)) + U * root
    # a product and a difference on w, its factor; alpha, product, sum, constant, quotient on the step
    dw = 3 * U * (w.abs() + step.abs()) + 5 * U * step.abs() + alpha * dm / (root + EPS) + step.abs() * droot / (root + EPS)
    return (w2, m2, v2), (dw, dm, dv)


@gpu
@pytest.mark.parametrize('bits', [32, 8])
@pytest.mark.parametrize('grad_dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('misaligned', [False, True])
@pytest.mark.parametrize('clip', [None, 0.5, 1e6])
def test_one_step_against_the_formula(bits, grad_dtype, misaligned, clip):
    from hgq2_b200.train import FusedAdamW

    gen = torch.Generator(device='cuda').manual_seed(bits + 7 * misaligned)
    sizes = [1, 5, 255, 256, 257, 1000, 4096, 70001]
    ws = tensors_of(sizes, torch.float32, gen, misaligned)
    gs = tensors_of(sizes, grad_dtype, gen, misaligned)
    decay = [0.1 * (i % 3) for i in range(len(sizes))]
    opt = FusedAdamW(ws, learning_rate=LR, weight_decay=decay, global_clipnorm=clip, state_bits=bits)
    m, v = set_state(opt, gen)
    opt.step_count.fill_(9)
    before = [w.double() for w in ws]
    opt.step(gs, grad_scale=0.25)
    assert int(opt.step_count) == 10 and int(opt._ticket) == 0
    norm = math.sqrt(sum(float((g.double() * 0.25).square().sum()) for g in gs))
    for i, (w, g) in enumerate(zip(ws, gs)):
        o = opt.offsets[i]
        sl = slice(o, o + sizes[i])
        want, off = want_step(before[i], g.double(), m[sl], v[sl], 10, decay[i], 0.25, 0.0, clip, norm)
        assert bool(((w.double() - want[0]).abs() <= off[0] + 1e-30).all()), f'w of size {sizes[i]}'
        got_m, got_v = opt.moments(i)
        if bits == 32:
            assert bool(((got_m.double() - want[1]).abs() <= off[1] + 1e-30).all())
            assert bool(((got_v.double() - want[2]).abs() <= off[2] + 1e-30).all())
        else:  # a dithered code is off by less than one step of its grid: 2^-3 of the value, or 2^-9 of the block's scale
            for got, x, d, scale in ((got_m, want[1], off[1], opt.m_scale), (got_v.sqrt(), want[2].sqrt(), None, opt.r_scale)):
                grid = torch.maximum(x.abs() / 8, scale.double().repeat_interleave(256)[sl] * 2.0 ** -9)
                slack = d if d is not None else 1e-6 * x.abs()
                assert bool(((got.double() - x).abs() <= grid * (1 + 1e-5) + slack).all()), f'state of size {sizes[i]}'


def reference_codes(x, place, step, root):
    """The fp32 definition of the 8-bit states, operation by operation."""
    low32 = 0xFFFFFFFF
    h = (place * 0x9E3779B1 + step * 0x6A09E667) & low32
    h = h ^ (h >> 16)
    h = (h * 0xBB67AE85) & low32
    h = h ^ (h >> 15)
    h = (h * 0x3C6EF373) & low32
    h = h ^ (h >> 16)
    d = (h >> 16) if root else (h & 0xFFFF)
    size = x.abs()
    top = torch.where(size.isfinite(), size, 0.0).amax(1).clamp(min=2.0 ** -100)
    u = size * (torch.full_like(top, 256.0) / top)[:, None]
    low = u < 2.0 ** -6
    y = torch.where(low, u + 2.0 ** -6, u)
    y = ((y.view(torch.int32) + (d.to(torch.int32) << 4)) & -0x100000).view(torch.float32)
    y = torch.where(low, y - 2.0 ** -6, y)
    if root:
        y = torch.where((size > 0) & (y == 0), 2.0 ** -9, y)
    y = torch.where(size.isfinite(), y, float('nan'))
    return torch.where(x < 0, -y, y).to(torch.float8_e4m3fn), top / 256


@gpu
def test_codes_equal_their_definition_over_many_steps():
    from hgq2_b200.train import FusedAdamW

    gen = torch.Generator(device='cuda').manual_seed(3)
    n = 256 * 300
    w = torch.randn(n, device='cuda', generator=gen)
    opt = FusedAdamW([w], learning_rate=LR, state_bits=8)
    m = r = torch.zeros(n // 256, 256, device='cuda')
    sm = sr = torch.zeros(n // 256, device='cuda')
    cm = cr = m.to(torch.float8_e4m3fn)
    place = torch.arange(n, device='cuda').view(-1, 256)
    for t in range(1, 30):
        g = torch.randn(n, device='cuda', generator=gen) * 10.0 ** float(torch.randint(-8, 3, (1,)))
        g[::7] = 0
        opt.step([g])
        g = g.view(-1, 256)
        m = (cm.float() * sm[:, None]) * B1 + g * (1.0 - B1)
        r = cr.float() * sr[:, None]
        r = torch.sqrt((r * r) * B2 + (g * g) * (1.0 - B2))
        (cm, sm), (cr, sr) = reference_codes(m, place, t, False), reference_codes(r, place, t, True)
        assert torch.equal(opt.m.float(), cm.float().view(-1)) and torch.equal(opt.m_scale, sm), t
        assert torch.equal(opt.r.float(), cr.float().view(-1)) and torch.equal(opt.r_scale, sr), t
    assert int(opt.step_count) == 29
    assert not bool(((opt.r.float() == 0) & (r.view(-1) > 0)).any())


@gpu
def test_dithering_keeps_the_mean():
    """A second moment that shrinks by 0.1 % a step follows its formula on average, where rounding to nearest would stay put."""
    from hgq2_b200.train import FusedAdamW

    n = 256 * 2000
    w = torch.zeros(n, device='cuda')
    opt = FusedAdamW([w], state_bits=8)
    r = torch.full((n,), 100.0, device='cuda').view(-1, 256)
    r[:, 0] = 256.0  # the block's largest element holds the scale
    opt.r.copy_(r.view(-1).to(torch.float8_e4m3fn))
    opt.r_scale.fill_(1.0)
    g = torch.zeros(n, device='cuda').view(-1, 256)
    g[:, 0] = 256.0  # keeps the largest element where it is
    for _ in range(20):
        opt.step([g.view(-1)])
    got = (opt.r.float().view(-1, 256) * opt.r_scale[:, None])[:, 1:].double()
    start = float(torch.tensor(100.0).to(torch.float8_e4m3fn))
    want = start * math.sqrt(B2 ** 20)
    # each step moves an element by one grid step (8 at most) with small odds: variance at most 8 * (start - want) over the
    # steps, so the mean of 510000 has a deviation of at most sqrt(8 * 0.97 / 510000) = 0.004; 6 of them.  The root is squared in
    # the recursion: the spread adds at most variance / (2 want) = 0.04 to the mean
    assert abs(float(got.mean()) - want) <= 6 * 0.004 + 0.04, (float(got.mean()), want)


@gpu
@pytest.mark.parametrize('bits', [32, 8])
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
def test_half_precision_tensors_go_through_a_master_copy(bits, dtype):
    from hgq2_b200.train import FusedAdamW

    gen = torch.Generator(device='cuda').manual_seed(5)
    sizes = [3, 256, 777, 2048]
    ws = tensors_of(sizes, dtype, gen)
    ws[2] = torch.randn(778, device='cuda', generator=gen).to(dtype)[1:]  # 2-byte aligned
    fp = [w.float().clone() for w in ws]
    a = FusedAdamW(ws, learning_rate=1e-4, state_bits=bits)
    b = FusedAdamW(fp, learning_rate=1e-4, state_bits=bits)
    for _ in range(5):
        gs = tensors_of(sizes, dtype, gen)
        a.step(gs)
        b.step(gs)
    for w, master, f in zip(ws, a.masters, fp):
        assert torch.equal(master, f)
        assert torch.equal(w, f.to(dtype))
    ws[1].fill_(0.5)
    a.sync_masters()
    assert torch.equal(a.masters[1], torch.full_like(a.masters[1], 0.5))


@gpu
def test_variables_constraints_and_regularizers():
    from hgq2_b200 import backend
    from hgq2_b200.constraints import Max, Min, MinMax
    from hgq2_b200.regularizers import MonoL1
    from hgq2_b200.train import FusedAdamW

    def var(c, r):
        return backend.Variable(torch.linspace(-2, 2, 301, device='cuda'), 'v', True, 'float32', c, r)

    vs = [var(None, None), var(MinMax(-1, 1), None), var(Min(0.5), MonoL1(0.3)), var(Max(0.25), None)]
    gs = [torch.linspace(-1, 1, 301, device='cuda') for _ in vs]
    before = [v.value.detach().double() for v in vs]
    opt = FusedAdamW(vs, learning_rate=LR, weight_decay=0.0)
    opt.step(gs)
    for v, b, g, lo, hi, l1 in zip(vs, before, gs, (-9, -1, 0.5, -9), (9, 1, 9, 0.25), (0, 0, 0.3, 0)):
        zero = torch.zeros_like(b)
        want, off = want_step(b, g.double(), zero, zero, 1, 0.0, 1.0, l1, None, 0.0)
        near = (v.value.detach().double() - want[0].clamp(lo, hi)).abs() <= off[0] + 1e-9
        assert bool(near.all())


@gpu
@pytest.mark.parametrize('bits', [32, 8])
def test_missing_gradients_and_empty_tensors(bits):
    from hgq2_b200.train import FusedAdamW

    gen = torch.Generator(device='cuda').manual_seed(6)
    ws = tensors_of([300, 0, 500, 256], torch.float32, gen)
    opt = FusedAdamW(ws, state_bits=bits, global_clipnorm=1.0)
    set_state(opt, gen)
    kept = {k: a.clone() for k, a in opt.state_dict().items()}
    w2 = ws[2].clone()
    opt.step([torch.ones_like(ws[0]), torch.ones_like(ws[1]), None, torch.ones_like(ws[3])])
    assert torch.equal(ws[2], w2)
    sl = slice(opt.offsets[2], opt.offsets[2] + 512)
    after = opt.state_dict()
    for k in ('m', 'v') if bits == 32 else ('m', 'r'):
        assert torch.equal(after[k][sl], kept[k][sl]) and not torch.equal(after[k], kept[k])
    assert int(opt.step_count) == 1
    with pytest.raises(ValueError, match='no gradients'):
        opt.step([None] * 4)
    assert int(opt.step_count) == 1


@gpu
@pytest.mark.parametrize('bits', [32, 8])
def test_more_tensors_than_one_launch_takes(bits):
    """1200 tensors: three launches share one norm and one step number."""
    from hgq2_b200.train import FusedAdamW

    gen = torch.Generator(device='cuda').manual_seed(7)
    sizes = [1 + (i * 37) % 700 for i in range(1200)]
    ws = tensors_of(sizes, torch.float32, gen)
    gs = tensors_of(sizes, torch.float32, gen)
    flat_w, flat_g = [], []
    for w, g, n in zip(ws, gs, sizes):  # the same blocks as one tensor: padding elements have zero gradients
        pad = -n % 256
        flat_w.append(torch.nn.functional.pad(w, (0, pad)))
        flat_g.append(torch.nn.functional.pad(g, (0, pad)))
    one = [torch.cat(flat_w)]
    a = FusedAdamW(ws, global_clipnorm=0.1, state_bits=bits)
    b = FusedAdamW(one, global_clipnorm=0.1, state_bits=bits)
    for _ in range(3):
        a.step(gs)
        b.step([torch.cat(flat_g)])
    for w, o, n in zip(ws, a.offsets, sizes):
        assert torch.equal(w, one[0][o:o + n])
    assert int(a.step_count) == 3


@gpu
@pytest.mark.parametrize('bits', [32, 8])
def test_offsets_past_32_bits(bits):
    from hgq2_b200.train import FusedAdamW

    n = 2 ** 31 + 777
    w = torch.empty(n, device='cuda').normal_()
    g = torch.empty(n, device='cuda', dtype=torch.bfloat16).normal_()
    tail = w[-2000:].double()
    opt = FusedAdamW([w], learning_rate=LR, weight_decay=0.0, state_bits=bits)
    opt.step([g])
    zero = torch.zeros_like(tail)
    want, off = want_step(tail, g[-2000:].double(), zero, zero, 1, 0.0, 1.0, 0.0, None, 0.0)
    assert bool(((w[-2000:].double() - want[0]).abs() <= off[0] + 1e-30).all())
    assert not bool((opt.m[:n][-2000:].float() == 0).all())


@gpu
def test_not_finite_gradients():
    """Without clipping a NaN or infinite gradient stays in its element; with clipping its norm reaches every weight."""
    from hgq2_b200.train import FusedAdamW

    for bits in (32, 8):
        w = torch.ones(600, device='cuda')
        g = torch.ones(600, device='cuda')
        g[5], g[300] = float('nan'), float('inf')
        opt = FusedAdamW([w], state_bits=bits)
        opt.step([g])
        bad = ~torch.isfinite(w)
        assert bad.nonzero().view(-1).tolist() == ([5, 300] if bits == 32 else [5, 300])
        m, v = opt.moments(0)
        ok = torch.ones(600, dtype=torch.bool, device='cuda')
        ok[5] = ok[300] = False
        assert bool(torch.isfinite(m[ok]).all() and torch.isfinite(v[ok]).all() and (v[ok] > 0).all())
        w = torch.ones(600, device='cuda')
        FusedAdamW([w], state_bits=bits, global_clipnorm=1.0).step([g])
        assert bool(torch.isnan(w).all())


@gpu
@pytest.mark.parametrize('bits', [32, 8])
def test_state_dict_resumes_to_the_bit_and_graphs_replay(bits):
    from hgq2_b200.train import FusedAdamW

    gen = torch.Generator(device='cuda').manual_seed(8)
    sizes = [100, 5000, 257]
    ws = tensors_of(sizes, torch.float32, gen)
    gs = tensors_of(sizes, torch.float32, gen)
    a = FusedAdamW(ws, state_bits=bits, global_clipnorm=1.0)
    a.step(gs)
    ws2 = [w.clone() for w in ws]
    b = FusedAdamW(ws2, state_bits=bits, global_clipnorm=1.0)
    b.load_state_dict(a.state_dict())
    # b's steps run as two captured graphs that take turns
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                b.step(gs)
            graphs.append(g)
    torch.cuda.current_stream().wait_stream(side)
    for i in range(4):
        a.step(gs)
        graphs[i % 2].replay()
    torch.cuda.synchronize()
    for x, y in zip(ws, ws2):
        assert torch.equal(x, y)
    for k, x in a.state_dict().items():
        assert torch.equal(x, b.state_dict()[k]), k
    with pytest.raises(ValueError):
        b.load_state_dict({'m': a.m})


@gpu
def test_refusals_on_the_device():
    from hgq2_b200.train import FusedAdamW

    w = torch.zeros(8, 8, device='cuda')
    with pytest.raises(ValueError, match='contiguous'):
        FusedAdamW([w.t()[1:]])
    with pytest.raises(ValueError, match='share memory'):
        FusedAdamW([w, w])
    with pytest.raises(ValueError, match='share memory'):
        FusedAdamW([w.view(-1)[:33], w.view(-1)[32:]])
    with pytest.raises(ValueError, match='supported'):
        FusedAdamW([w.double()])
    opt = FusedAdamW([w])
    for bad in ([], [w, w], [torch.zeros(8, 7, device='cuda')], [torch.zeros(64, device='cuda')], [w.double()], [torch.zeros(8, 8)]):
        with pytest.raises(ValueError):
            opt.step(bad)
    opt.step([torch.ones(8, 8, device='cuda').t()])  # a strided gradient is laid out, not refused
    assert int(opt.step_count) == 1


def test_refusals_need_no_gpu():
    from hgq2_b200.train import FusedAdamW

    w = torch.zeros(4)
    with pytest.raises(RuntimeError, match='CUDA tensors only'):
        FusedAdamW([w])
    for kw in (dict(state_bits=16), dict(global_clipnorm=0.0), dict(global_clipnorm=-1.0), dict(beta_1=1.0), dict(beta_2=-0.1),
               dict(weight_decay=[0.1, 0.2])):
        with pytest.raises(ValueError):
            FusedAdamW([w], **kw)
    with pytest.raises(ValueError, match='no tensors'):
        FusedAdamW([])


def test_c_entry_refuses_before_any_cuda_call():
    from hgq2_b200 import build

    build.build()
    from hgq2_b200 import _lib

    L = _lib.lib()
    import ctypes

    first = (ctypes.c_int64 * 2)(0, 1)
    grads, kinds = (ctypes.c_uint64 * 1)(0), bytes([0])
    p = 4096  # never dereferenced: every call below is refused on the host

    def call(n=1, bits=32, tensors=p, m=p, scale=p, kinds=kinds, first=first, clip=0.0, ws=None, nbytes=0, grads=grads):
        return L.hgq_adamw_step(tensors, n, p, first, grads, kinds, bits, m, p, scale, scale, 1e-3, 0.9, 0.999, 1e-7, 1.0, clip, p, p,
                                ws, nbytes, None)

    assert call(n=-1) == -2
    assert call(bits=16) == -3
    assert call(tensors=None) == -1
    assert call(bits=8, scale=None) == -1
    assert call(m=p + 4) == -4
    assert call(kinds=bytes([3])) == -3
    assert call(grads=(ctypes.c_uint64 * 1)(p + 2)) == -4
    assert call(first=(ctypes.c_int64 * 2)(1, 0)) == -2
    assert call(clip=1.0) == -5
    assert call(clip=1.0, ws=p, nbytes=8) == -5
    assert call(n=0) == 0
    assert L.hgq_adamw_workspace(0) == 0 and L.hgq_adamw_workspace(1) >= 8


def test_descriptor_matches_the_header(tmp_path):
    import ctypes
    import shutil
    import subprocess
    from pathlib import Path

    from hgq2_b200._lib import AdamWTensor

    gcc = shutil.which('gcc')
    if gcc is None:
        pytest.skip('no C compiler')
    names = [name for name, _ in AdamWTensor._fields_]
    body = 'printf("%zu ", sizeof(hgq_adamw_tensor));' + ''.join(f'printf("%zu ", offsetof(hgq_adamw_tensor, {n}));' for n in names)
    src = tmp_path / 'layout.c'
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "hgq_b200.h"\nint main(void){' + body + 'return 0;}\n')
    root = Path(__file__).resolve().parent.parent
    subprocess.run([gcc, '-I', str(root / 'include'), str(src), '-o', str(tmp_path / 'layout')], check=True)
    got = [int(v) for v in subprocess.run([str(tmp_path / 'layout')], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [ctypes.sizeof(AdamWTensor)] + [getattr(AdamWTensor, n).offset for n in names]


def _mlp_trainer(optimizer):
    from hgq2_b200 import workloads
    from hgq2_b200.train import Trainer, sparse_categorical_crossentropy

    gen = torch.Generator(device='cuda').manual_seed(9)
    x = torch.randn(512, 16, device='cuda', generator=gen)
    y = torch.randint(0, 5, (512,), device='cuda', generator=gen)
    return Trainer(workloads.build(workloads.jet_tagger_mlp()), sparse_categorical_crossentropy, optimizer=optimizer), x, y


@gpu
def test_trainer_takes_it():
    """Without decay and clipping the update rule is the flat bucket's Adam: one step from the same gradients agrees."""
    from hgq2_b200.train import FusedAdamW

    ref, x, y = _mlp_trainer(None)
    tr, _, _ = _mlp_trainer(lambda state: FusedAdamW(state, learning_rate=1e-3, weight_decay=0.0))
    assert torch.equal(ref.state.params, tr.state.params)
    ref.step(x, y)
    tr.step(x, y)
    # the flat bucket's Adam holds 1 - beta_2 as 1 - fp32(0.999), which is 3e-5 off; its root enters the step twice
    d = (ref.state.params - tr.state.params).abs()
    assert bool((d <= 1e-3 * 5e-5 + 4 * U * ref.state.params.abs()).all()), float(d.max())


@gpu
@pytest.mark.parametrize('bits', [32, 8])
def test_trainer_captured_equals_eager(bits):
    from hgq2_b200.train import FusedAdamW

    def make(state):
        return FusedAdamW(state, weight_decay=[0.0] * len(state.variables), global_clipnorm=1.0, state_bits=bits)

    eager, x, y = _mlp_trainer(make)
    cap, _, _ = _mlp_trainer(make)
    cap.capture(x, y, warmup=2)
    for _ in range(5):
        eager.step(x, y)
    for _ in range(3):
        cap.step(x, y)
    torch.cuda.synchronize()
    assert int(cap.opt.step_count) == int(eager.opt.step_count) == 5
    assert torch.equal(eager.state.params, cap.state.params)
    assert bool(torch.isfinite(cap.state.params).all())


@gpu
@pytest.mark.parametrize('bits', [32, 8])
@pytest.mark.parametrize('value,scale', [(float('inf'), 1.0), (-float('inf'), 1.0), (3e38, 4.0)])
def test_infinite_norm_reaches_every_weight(bits, value, scale):
    """One infinite gradient among finite ones, no NaN: Keras adds norm - norm to the clipping factor, which makes it NaN for an
    infinite norm too.  A gradient that overflows only when it is scaled counts as infinite."""
    from hgq2_b200.train import FusedAdamW

    ws = [torch.ones(n, device='cuda') for n in (600, 300, 64)]
    gs = [torch.ones_like(w) for w in ws]
    gs[1][7] = value
    kept = ws[2].clone()
    opt = FusedAdamW(ws, state_bits=bits, global_clipnorm=1.0)
    opt.step([gs[0], gs[1], None], grad_scale=scale)
    for i in range(2):
        assert bool(torch.isnan(ws[i]).all()), i
        m, v = opt.moments(i)
        assert bool(torch.isnan(m).all() and torch.isnan(v).all()), i
    assert torch.equal(ws[2], kept)  # no gradient: left as it is


@gpu
@pytest.mark.parametrize('bits', [32, 8])
def test_large_finite_norm_clips(bits):
    """Gradients whose squares fp32 does not hold: their norm is finite in fp64 and scales them as any other does."""
    from hgq2_b200.train import FusedAdamW

    n = 1000
    w = torch.ones(n, device='cuda')
    g = torch.full((n,), 1e36, device='cuda')
    before = w.double()
    FusedAdamW([w], learning_rate=LR, weight_decay=0.0, global_clipnorm=1.0, state_bits=bits).step([g])
    zero = torch.zeros(n, device='cuda', dtype=torch.float64)
    want, off = want_step(before, g.double(), zero, zero, 1, 0.0, 1.0, 0.0, 1.0, float(torch.linalg.vector_norm(g.double())))
    assert bool(((w.double() - want[0]).abs() <= off[0] + 1e-30).all())


@gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_autograd_sees_the_update(dtype):
    """A backward pass through a graph that was recorded before the step raises, as with torch's optimizers: the weights that it
    saved are gone.  A tensor without a gradient is not touched, and its graph stays usable."""
    from hgq2_b200.backend import Variable
    from hgq2_b200.train import FusedAdamW

    ps = [torch.nn.Parameter(torch.randn(50, device='cuda').to(dtype)) for _ in range(2)]
    items = [*ps, Variable(torch.randn(50, device='cuda'), 'v', True, 'float32', None, None)] if dtype == torch.float32 else ps
    leaves = [v.value if isinstance(v, Variable) else v for v in items]
    opt = FusedAdamW(items)
    values = [(p * p).sum() for p in leaves]
    opt.step([None if i == 1 else torch.ones_like(p) for i, p in enumerate(leaves)])
    values[1].backward()
    for i, v in enumerate(values):
        if i != 1:
            with pytest.raises(RuntimeError, match='modified by an inplace operation'):
                v.backward()


@gpu
@pytest.mark.parametrize('offset', [0, 1, 2, 3])
def test_an_fp32_tensor_beside_an_fp32_master(offset):
    """The C interface allows a master beside a tensor of any type: an fp32 one at an address that 16-byte accesses do not fit
    gets the master's values all the same."""
    from hgq2_b200 import _lib
    from hgq2_b200.train import FusedAdamW

    gen = torch.Generator(device='cuda').manual_seed(12)
    n = 256 * 9 + 5
    base = torch.zeros(n + 4, device='cuda')
    w, g = base[offset:offset + n], torch.randn(n, device='cuda', generator=gen)
    w.copy_(torch.randn(n, device='cuda', generator=gen))
    master, plain = w.clone(), w.clone()
    opt = FusedAdamW([w], learning_rate=LR)
    table = _lib.AdamWTensor.from_buffer_copy(bytes(opt._table.cpu().numpy()))
    table.master = master.data_ptr()
    opt._table.copy_(torch.frombuffer(bytearray(table), dtype=torch.uint8))
    other = FusedAdamW([plain], learning_rate=LR)
    for o in (opt, other):
        o.step([g])
    assert torch.equal(w, plain) and torch.equal(master, plain)
    assert not bool(base[:offset].any()) and not bool(base[offset + n:].any())


def test_c_entry_refuses_misaligned_scales_and_counters():
    import ctypes

    from hgq2_b200 import _lib, build

    build.build()
    L = _lib.lib()
    first, grads = (ctypes.c_int64 * 2)(0, 1), (ctypes.c_uint64 * 1)(0)
    p = 4096  # never dereferenced: every call below is refused on the host

    def call(m_scale=p, v_scale=p, ticket=p, bits=8):
        return L.hgq_adamw_step(p, 1, p, first, grads, bytes([0]), bits, p, p, m_scale, v_scale, 1e-3, 0.9, 0.999, 1e-7, 1.0, 0.0, p,
                                ticket, None, 0, None)

    assert call(m_scale=p + 2) == -4 and call(v_scale=p + 1) == -4
    assert call(ticket=p + 2) == -4 and call(ticket=p + 2, bits=32) == -4


@gpu
@pytest.mark.parametrize('bits,clip', [(32, None), (32, 0.5), (8, None), (8, 0.5)])
def test_states_past_32_bits(bits, clip):
    """More than 2^31 elements: weights, moments, codes and scales at both ends, and the norm over all of them."""
    from hgq2_b200.train import FusedAdamW

    n, ends = 2 ** 31 + 777, 1024 + 9  # whole blocks of 256 from the tail's start, the last of them with 9 elements
    w = torch.empty(n, device='cuda').normal_()
    g = torch.empty(n, device='cuda', dtype=torch.bfloat16).normal_()
    norm = 0.0
    for piece in g.split(1 << 28):
        norm += float(torch.linalg.vector_norm(piece, dtype=torch.float64)) ** 2
    norm = math.sqrt(norm)
    parts = [slice(0, 2048), slice(n - ends, n)]
    assert (n - ends) % 256 == 0
    before = [w[p].double() for p in parts]
    opt = FusedAdamW([w], learning_rate=LR, weight_decay=0.0, state_bits=bits, global_clipnorm=clip)
    opt.step([g])
    for p, old in zip(parts, before):
        zero = torch.zeros_like(old)
        want, off = want_step(old, g[p].double(), zero, zero, 1, 0.0, 1.0, 0.0, clip, norm)
        assert bool(((w[p].double() - want[0]).abs() <= off[0] + 1e-30).all())
        if bits == 32:
            assert bool(((opt.m[p].double() - want[1]).abs() <= off[1] + 1e-30).all())
            assert bool(((opt.v[p].double() - want[2]).abs() <= off[2] + 1e-30).all())
            continue
        blocks = slice(p.start // 256, -(-p.stop // 256))
        for codes, scales, x, root in ((opt.m, opt.m_scale, want[1], False), (opt.r, opt.r_scale, want[2].sqrt(), True)):
            s = scales[blocks]
            got = codes[p].double() * s.double().repeat_interleave(256)[:x.numel()]
            grid = torch.maximum(x.abs() / 8, s.double().repeat_interleave(256)[:x.numel()] * 2.0 ** -9)
            assert bool(((got - x).abs() <= grid * (1 + 1e-5) + 1e-6 * x.abs()).all())
            if clip is None:  # to the bit; clipped moments are a rounded factor of the norm away from that
                pad = torch.nn.functional.pad(g[p].float(), (0, -x.numel() % 256)).view(-1, 256)
                exact = torch.sqrt((pad * pad) * (1.0 - B2)) if root else pad * (1.0 - B1)
                place = torch.arange(blocks.start * 256, blocks.stop * 256, device='cuda').view(-1, 256)
                code, top = reference_codes(exact, place, 1, root)
                assert torch.equal(codes[p].float(), code.float().view(-1)[:x.numel()]) and torch.equal(s, top)


@gpu
def test_codes_are_loaded_as_bytes():
    """e4m3 codes given as e4m3 tensors are the same bytes; as numbers of another type they are refused, and nothing is taken over."""
    from hgq2_b200.train import FusedAdamW

    gen = torch.Generator(device='cuda').manual_seed(13)
    a, b = (FusedAdamW([torch.zeros(700, device='cuda')], state_bits=8) for _ in range(2))
    set_state(a, gen)
    state = a.state_dict()
    with pytest.raises(ValueError, match='codes'):
        b.load_state_dict({**state, 'm': a.m.float()})
    assert not bool(b.m.float().any()) and not bool(b.m_scale.any())
    b.load_state_dict({**state, 'm': a.m.clone(), 'r': a.r.clone()})
    assert all(torch.equal(v, b.state_dict()[k]) for k, v in state.items())
