"""Calls from several host threads at once, on one stream."""

import threading

import pytest
import torch

gpu = pytest.mark.gpu


def in_threads(*functions):
    """Runs the functions at the same time; their results, in order.  An exception of any of them is raised."""
    results, errors = [None] * len(functions), []

    def run(i):
        try:
            results[i] = functions[i]()
        except BaseException as e:  # noqa: BLE001 -- raised below, in the test's own thread
            errors.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(len(functions))]
    for t in threads:
        t.start()
    for t in threads:
        t.join(120)
    assert not any(t.is_alive() for t in threads)
    if errors:
        raise errors[0]
    return results


def test_scratch_is_a_threads_own(monkeypatch):
    """A call's launches meet in its scratch, and the interpreter lock is not held between them: two threads on one stream must
    not get the same buffer.  One thread gets the same one again."""
    from hgq2_b200 import kernels as K

    monkeypatch.setattr(torch.cuda, 'is_current_stream_capturing', lambda: False)
    monkeypatch.setattr(torch._C, '_cuda_getCurrentRawStream', lambda device: 0, raising=False)
    dev = torch.device('cpu', 0)
    ready = threading.Barrier(2)

    def take():
        ws = K.workspace(5000, dev, slot=99)
        ready.wait(60)  # both alive: a freed buffer's address may be used again
        again = K.workspace(4000, dev, slot=99)
        other = K.workspace(4000, dev, slot=98)
        ready.wait(60)
        return ws.data_ptr(), again.data_ptr(), other.data_ptr()

    a, b = in_threads(take, take)
    assert a[0] == a[1] and b[0] == b[1] and a[2] != a[0]
    assert not set(a) & set(b)


@gpu
def test_threads_on_one_stream_do_not_meet():
    """The calls that are several launches, each from two threads that use the default stream."""
    from hgq2_b200 import kernels as K
    from hgq2_b200.train import FusedAdamW

    def scan(seed):
        gen = torch.Generator(device='cuda').manual_seed(seed)
        x, z, g = (torch.randn(2, 6000, 64, device='cuda', generator=gen) for _ in range(3))

        def call():
            h, last, st = K.gated_scan_fwd(x, z, want_states=True)
            return (h, last, *K.gated_scan_bwd(g, x, z, None, None, st)[:2])
        return call

    def norm(seed):
        gen = torch.Generator(device='cuda').manual_seed(seed)
        x, g = (torch.randn(2, 150 * 150, 32, device='cuda', generator=gen) for _ in range(2))

        def call():
            y, mean, rstd = K.group_norm_fwd(x, None, None, 8, 1e-3, 'silu')
            return (y, *K.group_norm_bwd(g, x, None, None, mean, rstd, 8, 'silu'))
        return call

    def adamw(seed):
        gen = torch.Generator(device='cuda').manual_seed(seed)
        start, g = torch.randn(200000, device='cuda', generator=gen), torch.randn(200000, device='cuda', generator=gen) * (1 + seed)

        def call():
            w = start.clone()
            FusedAdamW([w], global_clipnorm=0.1).step([g])
            return (w,)
        return call

    for make in (scan, norm, adamw):
        calls = [make(0), make(1)]
        want = [call() for call in calls]
        torch.cuda.synchronize()

        def often(i):
            return [calls[i]() for _ in range(40)]

        for got, expected in zip(in_threads(lambda: often(0), lambda: often(1)), want):
            torch.cuda.synchronize()
            for outs in got:
                assert all(torch.equal(a, b) for a, b in zip(outs, expected)), make.__name__


@gpu
def test_one_layer_serves_two_lengths_at_once():
    """Two threads inside the projection of one recurrence layer, the first to come leaving before the second: each gets the
    shape of its own call, and the layer keeps the one it is built for."""
    from hgq2_b200.config import QuantizerConfigScope
    from hgq2_b200.layers import QGatedRecurrence
    from hgq2_b200.quantizer import QuantizerConfig

    with QuantizerConfigScope(place='datalane', default_q_type='kif', overflow_mode='WRAP', i0=4, f0=8):
        conf = QuantizerConfig(place='datalane', homogeneous_axis=(0, 1))
    layer = QGatedRecurrence(8, iq_conf=conf, return_state=True)
    x = torch.randn(2, 30, 6, device='cuda')
    layer(x)
    proj = layer.projection
    want = [layer(x[:, :n], training=False)[0] for n in (7, 12, 30)]
    prepare, first_in, second_in, first_out = proj.prepare_params, threading.Event(), threading.Event(), threading.Event()

    def paused():
        if not first_in.is_set():
            first_in.set()
            assert second_in.wait(60)
        elif not second_in.is_set():
            second_in.set()
            assert first_out.wait(60)
        return prepare()

    proj.prepare_params = paused

    def first():
        try:
            return layer(x[:, :7], training=False)[0]
        finally:
            first_out.set()

    def second():
        assert first_in.wait(60)
        try:
            return layer(x[:, :12], training=False)[0]
        finally:
            second_in.set()

    got = in_threads(first, second)
    del proj.prepare_params
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert torch.equal(layer(x, training=False)[0], want[2])


def test_passes_of_different_threads_have_different_numbers():
    """What a quantizer remembers of a pass is for that pass alone: one thread's must not be taken for another's, whose stream may
    not have computed it yet."""
    from hgq2_b200 import backend

    class Probe(backend.Layer):
        def call(self, inputs):
            return backend.current_pass()

    layer, ready = Probe(), threading.Barrier(2)

    def passes():
        ready.wait(60)
        return [layer(torch.zeros(1)) for _ in range(5)]

    a, b = in_threads(passes, passes)
    assert len(set(a)) == len(set(b)) == 5 and not set(a) & set(b)


def two_layers():
    from hgq2_b200.backend import Sequential
    from hgq2_b200.config import QuantizerConfigScope
    from hgq2_b200.layers import QDense

    with QuantizerConfigScope(place='all', default_q_type='kif', f0=6), QuantizerConfigScope(place='datalane', i0=3):
        model = Sequential([QDense(8), QDense(4)])
    x = torch.randn(16, 6, device='cuda')
    model(x)
    return model, x


@gpu
def test_parameters_queued_by_a_pass_that_fails_are_dropped():
    """A training pass that raises in its first layer has queued the second layer's quantised kernel: a later pass must not use it."""
    model, x = two_layers()
    first, second = model.layers
    wrong = torch.randn(16, 7, device='cuda')
    with pytest.raises(Exception):  # noqa: B017 -- whatever the shape mismatch raises
        model(wrong, training=True)
    second._kernel.assign(second.kernel * 0.0)
    y = model(x, training=False)
    assert torch.equal(y, second(first(x, training=False), training=False))
    assert torch.equal(y, model(x, training=False))
