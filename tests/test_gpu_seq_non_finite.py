"""Selective scan (csrc/ssm.hip) where a parameter is not finite or a decay grows: what the formulas give, in the rows, channels
and states that depend on it, and the same bits as without it everywhere else."""
import numpy as np
import pytest
import torch

import shivae_amd

pytestmark = pytest.mark.gpu


def _inputs(T, B, D, Ns, dtype=torch.float32, seed=0):
    rng = np.random.default_rng(seed)

    def rn(*shape, f=1.0):
        return torch.tensor(rng.standard_normal(shape) * f, dtype=torch.float32).cuda()

    v = dict(u=rn(T, B, D).to(dtype), dt=rn(T, B, D).to(dtype), A=-torch.exp(rn(Ns, D, f=0.5)), B=rn(T, B, 1, Ns).to(dtype),
             C=rn(T, B, 1, Ns).to(dtype), D=rn(D), z=rn(T, B, D).to(dtype), dt_bias=rn(D, f=0.3), initial_state=rn(B, Ns, D))
    return v, rn(T, B, D).to(dtype), rn(B, Ns, D)


def _grads(v, n, dy, dlast):
    leaves = {k: t.clone().requires_grad_(True) for k, t in v.items()}
    y, last = shivae_amd.selective_scan(**leaves, lengths=n, return_state=True)
    return y.detach(), last.detach(), dict(zip(leaves, torch.autograd.grad([y, last], list(leaves.values()), [dy, dlast])))


def _same_where(got, want, where):
    """Equal bits where `where` (broadcast) is false, NaN where it is true."""
    where = where.expand(got.shape)
    assert torch.equal(got[~where], want[~where]) and torch.isnan(got[where]).all()


@pytest.mark.parametrize("T, B, D, Ns, dtype", [(40, 3, 70, 16, torch.float32), (300, 3, 64, 16, torch.bfloat16), (75, 3, 20, 3, torch.float16),
                                                (200, 3, 40, 24, torch.float32), (33, 3, 80, 64, torch.float32), (64, 110, 150, 4, torch.float32)], ids=str)
def test_a_nan_in_A_is_seen(T, B, D, Ns, dtype):
    """One NaN in A: the outputs of its channel are NaN, and so are its state and the gradients that its decay enters."""
    v, dy, dlast = _inputs(T, B, D, Ns, dtype)
    n = torch.full((B,), T, device="cuda", dtype=torch.int32)
    n[1], n[2] = 0, T - 7
    ns, d = Ns - 1, D // 2
    want_y, want_last, want = _grads(v, n, dy, dlast)
    v["A"] = v["A"].clone()
    v["A"][ns, d] = float("nan")
    y, last, got = _grads(v, n, dy, dlast)
    t = torch.arange(T, device="cuda")[:, None]
    live, behind = (t < n), (t + 1 < n)  # a row, and a row that others follow
    some = n > 0
    channel, state = torch.arange(D, device="cuda") == d, torch.arange(Ns, device="cuda") == ns
    both = state[:, None] & channel
    _same_where(y, want_y, live[..., None] & channel)
    _same_where(last, want_last, some[:, None, None] & both)
    _same_where(got["A"], want["A"], both)
    _same_where(got["initial_state"], want["initial_state"], some[:, None, None] & both)
    _same_where(got["u"], want["u"], behind[..., None] & channel)  # (dL/dh of the last row has no decay in it)
    for k in ("dt", "z"):
        _same_where(got[k], want[k], live[..., None] & channel)
    _same_where(got["dt_bias"], want["dt_bias"], channel)
    _same_where(got["B"], want["B"], behind[..., None, None] & state)
    _same_where(got["C"], want["C"], live[..., None, None] & state)
    assert torch.equal(got["D"], want["D"])


def test_a_nan_in_A_is_seen_by_the_step():
    v, _, _ = _inputs(1, 3, 24, 16)
    args = [v["u"][0], v["dt"][0], v["A"].clone(), v["B"][0], v["C"][0]]
    args[2][5, 7] = float("nan")
    for D in (24, 23):  # four channels a thread, and one
        a = [t[..., :D] if t.shape[-1] == 24 else t for t in args]
        state = v["initial_state"][..., :D].contiguous()
        y = shivae_amd.selective_scan_step(*a, state)
        assert torch.isnan(y[:, 7]).all() and torch.isfinite(y).sum() == y.numel() - 3
        assert torch.isnan(state[:, 5, 7]).all() and torch.isfinite(state).sum() == state.numel() - 3


def test_nan_everywhere_else_is_seen():
    """A NaN in any other input reaches the outputs that depend on it."""
    T, B, D, Ns = 70, 2, 33, 16
    v, _, _ = _inputs(T, B, D, Ns)
    for k, at in (("u", (50, 1, 4)), ("dt", (50, 1, 4)), ("B", (50, 1, 0, 3)), ("C", (50, 1, 0, 3)), ("D", (4,)), ("z", (50, 1, 4)),
                  ("dt_bias", (4,)), ("initial_state", (1, 3, 4))):
        w = {**v, k: v[k].clone()}
        w[k][at] = float("nan")
        y, last = shivae_amd.selective_scan(**w, return_state=True)
        assert torch.isnan(y[50, 1, 4]), k
        assert torch.isnan(last[1, 3, 4]) == (k in ("u", "dt", "B", "dt_bias", "initial_state")), k
