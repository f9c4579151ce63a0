"""Selective scan (csrc/ssm.hip) where a parameter is not finite or a decay grows: what the formulas give, in the rows, channels
and states that depend on it, and the same bits as without it everywhere else."""
import numpy as np
import pytest
import torch

import _seq_ref as ref
import shivae_amd
from test_gpu_seq_ops import _near

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


@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("B", [1, 260])
def test_growing_decays_over_a_state_of_zero(B, sign):
    """Decays whose product over a piece of the time axis overflows, while state and adjoint there are 0: the pieces (one sequence) give
    what the unsplit scan (260 sequences fill the card) and the formula give.  A > 0 with positive steps, and A < 0 with negative."""
    T, D, Ns = 200, 40, 16
    v, dy, _ = _inputs(T, B, D, Ns)
    for k in ("D", "z", "dt_bias", "initial_state"):
        v[k] = None
    v["A"] = -v["A"] * sign
    grow = torch.full_like(v["dt"], 3.0 * sign)
    calm = 0.02 * v["dt"].abs() * sign
    # forward: growth in rows 0..129, in front of all input (exp(3 * 0.2) a row at least: past 2^128 within 150 rows)
    v["dt"] = torch.where(torch.arange(T, device="cuda")[:, None, None] < 130, grow, calm)
    v["u"][:130] = 0
    a = {k: None if t is None else t.double().cpu().numpy() for k, t in v.items()}
    want, scale = ref.scan(a["u"], a["dt"], a["A"], a["B"], a["C"], None, None, None, None, None, False)
    assert float(np.abs(a["A"]).max()) * 3 * 64 > 88.8  # past the largest fp32 within a piece
    y, last = shivae_amd.selective_scan(v["u"], v["dt"], v["A"], v["B"], v["C"], softplus=False, return_state=True)
    _near(y, want["y"], scale["y"], 3 * T + 96, "y")
    _near(last, want["last"], scale["last"], 3 * T + 96, "state")
    # backward: growth in rows 70..199, behind all gradient
    v["dt"] = torch.where(torch.arange(T, device="cuda")[:, None, None] < 70, calm, grow)
    v["u"][:] = 0
    dy[70:] = 0
    a = {k: None if t is None else t.double().cpu().numpy() for k, t in v.items()}
    want, scale = ref.scan(a["u"], a["dt"], a["A"], a["B"], a["C"], None, None, None, None, None, False, dy.double().cpu().numpy())
    leaves = [v[k].clone().requires_grad_(True) for k in ("u", "dt", "A", "B", "C")]
    y = shivae_amd.selective_scan(*leaves, softplus=False)
    for k, g in zip(("u", "dt", "A", "B", "C"), torch.autograd.grad(y, leaves, dy)):
        _near(g, want[k], scale[k], 2 * (3 * T + 96) + 8 + np.log2(T * B) + T, "d" + k)


@pytest.mark.parametrize("x", [-240, 240])
def test_states_far_out_of_the_ordinary(x):
    """A large state that decays, and a small one that grows, by 2^x over the second of three pieces: 2^x is out of the range of fp32, the
    states are not.  The exponent is off by a unit for log2(e) and one for A log2(e), relative to |x| log(2) = sum |s A|."""
    T, D, Ns = 192, 8, 4
    rows = torch.arange(T, device="cuda")[:, None, None]
    u, one = torch.zeros(T, 1, D, device="cuda"), torch.ones(T, 1, 1, Ns, device="cuda")
    dt = torch.where((rows >= 64) & (rows < 128), 1.0, 0.0).expand(T, 1, D).contiguous()
    A = torch.full((Ns, D), x * np.log(2.0) / 64, device="cuda")
    s0 = torch.full((1, Ns, D), 2.0 ** (-x // 2), device="cuda")
    y, last = shivae_amd.selective_scan(u, dt, A, one, one, softplus=False, initial_state=s0, return_state=True)
    total = 64 * A.double().cpu().numpy()
    want = s0.double().cpu().numpy() * np.exp(total)
    _near(last, want, want, 3 * T + 96 + 2 * np.abs(total).max(), "state")
    _near(y[128:], np.broadcast_to(want.sum(1), (64, 1, D)), want.sum(), 3 * T + 96 + 2 * np.abs(total).max(), "y")
