"""Calls of several host threads at once."""
import threading

import pytest
import torch

from shivae_amd import ssm

pytestmark = pytest.mark.gpu


def test_backward_passes_with_different_numbers_of_states():
    """32 states keep 24 KiB in dynamic LDS and 64 keep 48, set by each call for the same kernel: the calls of two threads, each on its own
    stream, give what they give one after the other."""
    gen = torch.Generator(device="cuda").manual_seed(0)
    T, B, D = 40, 2, 64

    def rn(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    inputs = {n: (rn(T, B, D), rn(T, B, D), -rn(n, D).abs(), rn(T, B, 1, n), rn(T, B, 1, n)) for n in (32, 64)}
    dy = rn(T, B, D)

    def gradients(n):  # (what autograd calls, which has one thread of its own for a device)
        y, _, ckpt = ssm._scan_forward(*inputs[n], None, None, None, None, None, 1, False, True)
        return [y] + [g for g in ssm._scan_backward(*inputs[n], None, None, None, None, None, ckpt, 1, dy, None) if g is not None]

    want = {n: gradients(n) for n in inputs}
    torch.cuda.synchronize()
    errors, ready = [], threading.Barrier(2)

    def work(n):
        try:
            stream = torch.cuda.Stream()
            ready.wait(30)
            with torch.cuda.stream(stream):
                for _ in range(100):
                    got = gradients(n)
                    stream.synchronize()
                    assert all(torch.equal(a, b) for a, b in zip(got, want[n]))
        except BaseException as e:  # noqa: B036 (handed to the test's own thread)
            errors.append((n, e))

    threads = [threading.Thread(target=work, args=(n,)) for n in inputs]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not errors, errors
