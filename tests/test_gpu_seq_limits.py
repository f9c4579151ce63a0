"""Sizes past one launch's 2^32 threads: rows that are drawn in several launches, and gradients that a thread has several of."""
import pytest
import torch

import shivae_amd

pytestmark = pytest.mark.gpu


def test_more_rows_than_a_launch_has_threads_for():
    """2^24 rows of more than 4096 categories take 256 threads each.  One row of logits, read by all; tokens repeat with the numbers."""
    V, rows, few = 4097, (1 << 24) + 5, 3000
    gen = torch.Generator(device="cuda").manual_seed(1)
    row, u = torch.randn(1, V, device="cuda", generator=gen).bfloat16(), torch.rand(few, device="cuda", generator=gen)
    k = torch.randint(0, 60, (few,), device="cuda", generator=gen)
    # (as many rows as take the same number of threads)
    want, wantp = shivae_amd.sample_categories(row.expand(few, V), u, top_k=k, top_p=0.9, return_logprob=True)
    at = torch.arange(rows, device="cuda") % few
    got, gotp = shivae_amd.sample_categories(row.expand(rows, V), u[at], top_k=k[at], top_p=0.9, return_logprob=True)
    assert torch.equal(got, want[at]) and torch.equal(gotp, wantp[at])


def test_more_gradients_of_B_and_C_than_a_launch_has_threads():
    """T * B * 2 N = 2^32, one channel; every sequence is the same, and so are its gradients, those of a smaller batch."""
    T, B, Ns = 4096, 8192, 64
    if torch.cuda.mem_get_info()[0] < 60e9:
        pytest.skip("not enough free memory")
    gen = torch.Generator(device="cuda").manual_seed(2)

    def rn(*shape):
        return torch.randn(*shape, device="cuda", generator=gen).bfloat16()

    u, dt, Bm, Cm, dy, A = rn(T, 1, 1), rn(T, 1, 1), rn(T, 1, 1, Ns), rn(T, 1, 1, Ns), rn(T, 1, 1), -torch.rand(Ns, 1, device="cuda", generator=gen)

    def gradients(n):
        leaves = [t.expand(T, n, *t.shape[2:]).requires_grad_(True) for t in (Bm, Cm)]
        y = shivae_amd.selective_scan(u.expand(T, n, 1), dt.expand(T, n, 1), A, *leaves)
        return torch.autograd.grad(y, leaves, dy.expand(T, n, 1))

    want, got = gradients(300), gradients(B)  # (both more workgroups than are split over time)
    for w, g in zip(want, got):
        assert g.abs().amax() > 0 and torch.equal(w, w[:, :1].expand_as(w))
        for b in range(0, B, 1024):  # (a part at a time)
            assert torch.equal(g[:, b:b + 1024], w[:, :1].expand(T, 1024, 1, Ns))
