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
