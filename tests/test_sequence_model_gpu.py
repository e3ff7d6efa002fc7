"""The layers on the group normalisation and recurrence kernels, alone and together in a model that AdamW trains."""

import pytest
import torch

gpu = pytest.mark.gpu


def close(a, b, rtol, what):
    a, b = a.detach().double(), b.detach().double()
    scale = max(float(b.abs().max()), 1e-30)
    err = float((a - b).abs().max()) / scale
    assert err <= rtol, f'{what}: {err:.2e} of the largest value'


def plain_group_norm(x, gamma, beta, groups, eps, activation):
    B, C = x.shape[0], x.shape[-1]
    v = x.reshape(B, -1, groups, C // groups)
    mean = v.mean((1, 3), keepdim=True)
    var = (v - mean).square().mean((1, 3), keepdim=True)
    u = ((v - mean) / torch.sqrt(var + eps)).reshape(x.shape)
    u = u if gamma is None else u * gamma
    u = u if beta is None else u + beta
    return {None: lambda t: t, 'relu': torch.relu, 'silu': torch.nn.functional.silu, 'gelu': torch.nn.functional.gelu}[activation](u)


def plain_scan(p, h0, lengths):
    x, z = p[:, :, 0], p[:, :, 1]
    a = torch.sigmoid(z)
    h = torch.zeros_like(x[:, 0], dtype=torch.promote_types(torch.float32, x.dtype)) if h0 is None else h0
    out = []
    for t in range(x.shape[1]):
        new = a[:, t] * h + (1 - a[:, t]) * x[:, t]
        if lengths is not None:
            live = (t < lengths)[:, None]
            h = torch.where(live, new, h)
            out.append(torch.where(live, h, torch.zeros_like(h)))
        else:
            h = new
            out.append(h)
    return torch.stack(out, 1).to(x.dtype), h


@pytest.fixture
def plain_ops(monkeypatch):
    """Swaps the two kernels for torch expressions that autograd differentiates."""

    def swap():
        from hgq2_b200.layers import gated_recurrence, group_normalization

        class Norm:
            apply = staticmethod(plain_group_norm)

        class Scan:
            apply = staticmethod(plain_scan)

        monkeypatch.setattr(group_normalization, 'GroupNormFn', Norm)
        monkeypatch.setattr(gated_recurrence, 'GatedScanFn', Scan)

    return swap


def sequence_model(T=48, last=True, oq=False):
    from hgq2_b200 import workloads as W
    from hgq2_b200.backend import Sequential
    from hgq2_b200.layers import GroupNormalization, QDense, QEinsumDense, QGatedRecurrence

    w, a, l = W._scopes(4, 8, 1e-5)
    with w, a, l:
        layers = W._seeded([
            QEinsumDense('abc,cd->abd', (T, 32), bias_axes='d'),
            QGatedRecurrence(32, enable_oq=oq),
            GroupNormalization(4, activation='silu'),
            QGatedRecurrence(16, return_sequences=not last),
            *([] if last else [lambda x: x.mean(dim=1)]),
            QDense(5),
        ])
    model = Sequential(layers, name='sequence_model')
    model.input_shape, model.weight_bits = (T, 12), (5, 8)
    return W.build(model)


def conv_model():
    from hgq2_b200 import workloads as W
    from hgq2_b200.backend import Flatten, MaxPooling2D, Sequential
    from hgq2_b200.layers import GroupNormalization, QConv2D, QDense

    w, a, l = W._scopes(3, 6, 1e-5)
    with w, a, l:
        layers = W._seeded([QConv2D(16, 3), GroupNormalization(4, activation='gelu'), MaxPooling2D(2), QConv2D(32, 3),
                            GroupNormalization(8, center=False, activation='silu'), Flatten(), QDense(5)])
    model = Sequential(layers, name='conv_model')
    model.input_shape, model.weight_bits = (12, 12, 3), (5, 8)
    return W.build(model)


def batch(model, n=40, seed=0):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    x = torch.randn((n, *model.input_shape), device='cuda', generator=gen)
    return x, torch.randint(0, 5, (n,), device='cuda', generator=gen)


def trainer(model, engine, **kw):
    from hgq2_b200.train import FusedAdamW, Trainer, sparse_categorical_crossentropy

    return Trainer(model, sparse_categorical_crossentropy, engine=engine,
                   optimizer=lambda state: FusedAdamW(state, weight_decay=[0.0] * len(state.variables), **kw))


MODELS = {'last_state': sequence_model, 'all_steps': lambda: sequence_model(last=False), 'output_quantizer': lambda: sequence_model(oq=True),
          'images': conv_model}


@gpu
@pytest.mark.parametrize('name', list(MODELS))
def test_gradients_equal_those_of_plain_expressions(name, plain_ops):
    """The static step plan, the autograd path and the autograd path on torch expressions: loss, EBOPs, every gradient."""
    runs = []
    for engine, plain in ((True, False), (False, False), (False, True)):
        if plain:
            plain_ops()
        model = MODELS[name]()
        tr = trainer(model, engine)
        x, y = batch(model)
        _, loss = tr.forward_backward(x, y)
        tr.state.check_views()
        runs.append((loss, {v.path.split('/', 1)[-1] + str(i): v.value.grad.clone() for i, v in enumerate(tr.state.variables)},
                     [int(layer.ebops) for layer in model.layers if hasattr(layer, 'ebops')]))
    for loss, grads, ebops in runs[:2]:
        close(loss, runs[2][0], 1e-5, 'loss')
        assert ebops == runs[2][2] and sum(ebops) > 0
        for (k, g), want in zip(grads.items(), runs[2][1].values()):
            # a scalar or tiny bitwidth gradient is a cancelling sum of thousands of signed terms
            close(g, want, 1e-4 if g.numel() > 64 else 2e-3, f'gradient {k}')


@gpu
@pytest.mark.parametrize('bits', [32, 8])
@pytest.mark.parametrize('engine', [True, False])
def test_training_steps_captured_equal_eager(bits, engine):
    a = trainer(sequence_model(), engine, state_bits=bits, global_clipnorm=0.5)
    b = trainer(sequence_model(), engine, state_bits=bits, global_clipnorm=0.5)
    assert torch.equal(a.state.params, b.state.params)
    x, y = batch(a.model)
    b.capture(x, y, warmup=2)
    start = a.state.params.clone()
    for _ in range(5):
        a.step(x, y)
    for _ in range(3):
        b.step(x, y)
    torch.cuda.synchronize()
    assert int(a.opt.step_count) == int(b.opt.step_count) == 5
    assert torch.equal(a.state.params, b.state.params)
    assert bool(torch.isfinite(a.state.params).all()) and not torch.equal(a.state.params, start)


def recurrence(units, T, C, homogeneous, **kw):
    from hgq2_b200.config import QuantizerConfigScope
    from hgq2_b200.layers import QGatedRecurrence
    from hgq2_b200.quantizer import QuantizerConfig

    axes = dict(homogeneous_axis=(0, 1)) if homogeneous else {}
    with QuantizerConfigScope(place='datalane', default_q_type='kif', overflow_mode='WRAP', i0=4, f0=8):
        conf = QuantizerConfig(place='datalane', **axes)
        out = QuantizerConfig(place='datalane', **axes)
    layer = QGatedRecurrence(units, iq_conf=conf, oq_conf=out, **kw)
    layer(torch.zeros(2, T, C, device='cuda'))
    return layer


@gpu
@pytest.mark.parametrize('oq', [False, True])
def test_streaming_equals_the_sequence(oq):
    layer = recurrence(24, 30, 10, True, enable_oq=oq, return_state=True)
    x = torch.randn(3, 30, 10, device='cuda')
    whole, last = layer(x, training=False)
    state, out = None, []
    for t in range(30):
        h, state = layer(x[:, t:t + 1], initial_state=state, training=False)
        out.append(h)
    tol = 1e-5 if not oq else 2.0 ** -8 + 1e-5  # with an output quantizer a last bit may decide between two grid points
    assert float((torch.cat(out, 1) - whole).detach().abs().max()) <= tol and float((state - last).detach().abs().max()) <= 1e-5
    longer, _ = layer(torch.cat([x, x], 1), training=False)
    assert float((longer[:, :30] - whole).detach().abs().max()) <= tol


@gpu
def test_padded_batch_and_initial_state():
    layer = recurrence(24, 30, 10, True, return_state=True)
    gen = torch.Generator(device='cuda').manual_seed(1)
    x = torch.randn(4, 30, 10, device='cuda', generator=gen)
    h0 = torch.randn(4, 24, device='cuda', generator=gen).requires_grad_()
    lengths = torch.tensor([0, 1, 17, 30], device='cuda')
    h, last = layer(x, initial_state=h0, lengths=lengths, training=True)
    w = torch.randn(h.shape, device='cuda', generator=gen)
    kernel = layer.projection.kernel
    grads = torch.autograd.grad((h * w).sum() + (last * last).sum(), (h0, kernel))
    p = layer.projection(x, training=True)
    h2, last2 = plain_scan(p.reshape(4, 30, 2, 24), h0, lengths)
    want = torch.autograd.grad((h2 * w).sum() + (last2 * last2).sum(), (h0, kernel))
    close(h, h2, 1e-6, 'h')
    close(last, last2, 1e-6, 'state')
    assert not bool(h[0].any()) and not bool(h[1, 1:].any()) and torch.equal(last[0], h0[0])
    for g, v in zip(grads, want):
        close(g, v, 1e-5, 'gradient')


@gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
def test_group_normalization_layer(dtype):
    from hgq2_b200.layers import GroupNormalization

    for groups, kw in ((4, {}), (-1, dict(center=False, activation='relu')), (1, dict(scale=False, activation='gelu'))):
        layer = GroupNormalization(groups, **kw)
        x = torch.randn(3, 7, 5, 8, device='cuda').to(dtype).requires_grad_()
        y = layer(x, training=True)
        assert y.dtype == dtype and layer.groups == (8 if groups == -1 else groups)
        assert [v.name for v in layer.variables] == [n for n, on in (('gamma', kw.get('scale', True)), ('beta', kw.get('center', True))) if on]
        want = plain_group_norm(x.float(), layer.gamma, layer.beta, layer.groups, 1e-3, layer.activation)
        close(y, want, {torch.float32: 1e-6, torch.bfloat16: 2 ** -8, torch.float16: 2 ** -11}[dtype] * 1.01, 'y')
        (g,) = torch.autograd.grad(y.float().square().sum(), x)
        assert g.dtype == dtype and bool(torch.isfinite(g).all())
        assert layer.get_config()['groups'] == layer.groups


@gpu
def test_weights_round_trip(tmp_path):
    from hgq2_b200.utils.weights import load_weights, save_weights

    a, b = sequence_model(), sequence_model()
    for p, q in zip(a.layers, b.layers):  # the file addresses layers by name
        q.name = p.name
    x, y = batch(a)
    tr = trainer(a, True)
    for _ in range(2):
        tr.step(x, y)
    save_weights(a, str(tmp_path / 'w.npz'))
    load_weights(b, str(tmp_path / 'w.npz'))
    assert torch.equal(a(x, training=False), b(x, training=False))


@gpu
def test_refusals():
    from hgq2_b200.layers import GroupNormalization, QGatedRecurrence

    x = torch.zeros(2, 6, 8, device='cuda')
    with pytest.raises(ValueError, match='divide'):
        GroupNormalization(3)(x)
    with pytest.raises(NotImplementedError, match='channels last'):
        GroupNormalization(2, axis=1)(x)
    with pytest.raises(ValueError, match='activation'):
        GroupNormalization(2, activation='tanh')
    with pytest.raises(ValueError, match='units'):
        QGatedRecurrence(0)
    with pytest.raises(NotImplementedError, match='batch, time'):
        QGatedRecurrence(4)(x[0])
    layer = recurrence(4, 6, 8, False)
    with pytest.raises(ValueError, match='bitwidth per step'):
        layer(x[:, :3], training=False)
    layer = recurrence(4, 6, 8, True)
    with pytest.raises(ValueError, match='in training'):
        layer(x[:, :3], training=True)
    with pytest.raises(ValueError, match='h0'):
        layer(x, initial_state=torch.zeros(2, 3, device='cuda'), training=False)


@gpu
def test_autograd_of_the_layers_captures():
    """Forward and backward of both layers through autograd, recorded and replayed on new data."""
    from hgq2_b200.layers import GroupNormalization

    norm = GroupNormalization(2, activation='silu')
    scan = recurrence(8, 9, 8, True)
    x = torch.randn(4, 9, 8, device='cuda', requires_grad=True)
    lengths = torch.tensor([9, 0, 4, 9], device='cuda', dtype=torch.int32)
    norm(x)

    def grads():
        return torch.autograd.grad(scan(norm(x), lengths=lengths, training=True).square().sum(),
                                   (x, norm.gamma, norm.beta, scan.projection.kernel))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        grads()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = grads()
    with torch.no_grad():
        x.copy_(torch.randn_like(x))
    graph.replay()
    want = grads()
    for a, b in zip(got, want):
        close(a, b, 1e-6, 'gradient')


@gpu
def test_second_derivatives_are_refused():
    """The backward passes are kernels without a derivative of their own: asking for one is an error, not a zero."""
    from hgq2_b200.layers import GroupNormalization

    x = torch.randn(4, 9, 8, device='cuda', requires_grad=True)
    for layer in (GroupNormalization(2, activation='silu'), recurrence(8, 9, 8, True)):
        (g,) = torch.autograd.grad(layer(x, training=True).square().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError):
            g.square().sum().backward()


def shared_norm_model(T=24):
    """One normalisation that stands in two places of the model."""
    from hgq2_b200 import workloads as W
    from hgq2_b200.backend import Sequential
    from hgq2_b200.layers import GroupNormalization, QDense, QEinsumDense, QGatedRecurrence

    w, a, l = W._scopes(4, 8, 1e-5)
    with w, a, l:
        norm = GroupNormalization(4, activation='silu')
        layers = W._seeded([QEinsumDense('abc,cd->abd', (T, 32), bias_axes='d'), norm, QEinsumDense('abc,cd->abd', (T, 32), bias_axes='d'),
                            norm, QGatedRecurrence(16, return_sequences=False), QDense(5)])
    model = Sequential(layers, name='shared_norm_model')
    model.input_shape, model.weight_bits = (T, 12), (5, 8)
    return W.build(model)


@gpu
def test_a_normalisation_in_two_places_gets_both_gradients():
    """The step plan writes a variable's gradient once; a model that uses it twice takes the autograd path, which adds them up."""
    from hgq2_b200.engine import Unsupported

    runs = []
    for engine in (None, False):
        tr = trainer(shared_norm_model(), engine)
        assert tr.engine is None and (engine is False or 'two places' in tr.engine_refusal)
        x, y = batch(tr.model)
        _, loss = tr.forward_backward(x, y)
        runs.append((loss, [v.value.grad.clone() for v in tr.state.variables], [v.path for v in tr.state.variables]))
    assert sum(p.endswith('gamma') for p in runs[0][2]) == 1
    close(runs[0][0], runs[1][0], 1e-6, 'loss')
    for g, want, path in zip(runs[0][1], runs[1][1], runs[0][2]):
        close(g, want, 1e-5 if g.numel() > 64 else 2e-3, f'gradient {path}')
    with pytest.raises(Unsupported, match='two places'):
        trainer(shared_norm_model(), True)


@gpu
def test_a_layer_of_ones_own_is_not_taken_for_its_parent():
    """A subclass may compute something else: the step plan covers the two layers themselves only."""
    from hgq2_b200 import workloads as W
    from hgq2_b200.backend import Sequential
    from hgq2_b200.layers import GroupNormalization, QDense, QEinsumDense, QGatedRecurrence

    class Shifted(GroupNormalization):
        def call(self, inputs):
            return super().call(inputs) + 1.0

    class Doubled(QGatedRecurrence):
        def call(self, inputs, initial_state=None, lengths=None, training=None):
            return 2.0 * super().call(inputs, initial_state, lengths, training)

    for make in (lambda: Shifted(4), lambda: Doubled(32)):
        runs = []
        for engine in (None, False):
            w, a, l = W._scopes(4, 8, 1e-5)
            with w, a, l:
                layers = W._seeded([QEinsumDense('abc,cd->abd', (24, 32), bias_axes='d'), make(), lambda x: x.mean(dim=1), QDense(5)])
            model = Sequential(layers)
            model.input_shape, model.weight_bits = (24, 12), (5, 8)
            tr = trainer(W.build(model), engine)
            assert tr.engine is None
            x, y = batch(tr.model)
            runs.append(tr.forward_backward(x, y)[0])
        close(runs[0], runs[1], 1e-6, 'loss')
