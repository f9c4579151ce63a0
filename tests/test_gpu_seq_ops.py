"""Causal convolution and selective scan (csrc/conv.hip, csrc/ssm.hip) against the formulas in 64 bits (_seq_ref.py).

Tolerances.  A stored result is rounded once: half a step, eps/2 of the type, relative to the value.  In front of that
everything is fp32 (unit 2^-24 per operation), so an error is at most a count of operations times 2^-24 times the `scale` of the
result, the same sums over absolute values:
  convolution: W + 1 products and sums, then silu, whose relative error is that of exp(-s), (2 |s| + 6) units, |s| <= scale;
  scan: one decay and two fused operations for every row that still counts, at most 3 T; s = softplus(..) is off by at most
    (2 |dt| + 16) units and enters every decay once, sum |s A| exp(-sum |s A|) < 1; the gate (2 |z| + 6): together 3 T + 96;
  its gradients run forward and back: twice that, and another 8 + log2 of the terms of a sum for those that are summed."""
import numpy as np
import pytest
import torch

import _seq_ref as ref
import shivae_amd

pytestmark = pytest.mark.gpu
UNIT = 2.0 ** -24
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _near(got, want, scale, units, what):
    got64 = got.detach().double().cpu().numpy()
    assert got64.shape == want.shape, (what, got64.shape, want.shape)
    half = torch.finfo(got.dtype).eps / 2
    tiny = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -133, torch.float32: 2.0 ** -126}[got.dtype]  # below the type's range: absolute
    tol = half * np.abs(want) + (1 + half) * units * UNIT * scale + tiny
    bad = ~(np.abs(got64 - want) <= tol)
    assert not bad.any(), "%s: %d of %d off, first at %s: %r for %r, tolerance %r" % (
        what, bad.sum(), bad.size, np.argwhere(bad)[0], got64[bad][0], want[bad][0], tol[bad][0])


class _Maker:
    def __init__(self, seed, dtype):
        self.rng, self.dtype = np.random.default_rng(seed), TYPES[dtype]

    def act(self, *shape, f=1.0):
        return torch.tensor(self.rng.standard_normal(shape) * f, dtype=torch.float32).to(self.dtype).cuda()

    def par(self, *shape, f=1.0, add=0.0):
        return torch.tensor(self.rng.standard_normal(shape) * f + add, dtype=torch.float32).cuda()

    def lengths(self, T, B):
        n = self.rng.integers(0, T + 1, B)
        n[:3] = [0, T, 1][:min(B, 3)]
        return torch.tensor(n, dtype=torch.int32).cuda()


def _np(t):
    return None if t is None else t.detach().double().cpu().numpy()


def _poison(lengths, *tensors):
    """NaN behind every sequence's last row: nothing there may count."""
    T = tensors[0].shape[0]
    dead = torch.arange(T, device="cuda")[:, None] >= lengths[None].long().clamp(0, T)
    for t in tensors:
        if t is not None:
            t[dead] = float("nan")


# ------------------------------------------------------------------------------------------------ convolution
CONV = [  # T, B, D, W, dtype, silu, bias, state, ragged
    (1, 1, 1, 2, "f32", True, True, True, False), (1, 3, 8, 4, "bf16", True, True, True, False),
    (2, 2, 5, 4, "f32", True, False, True, True), (3, 4, 16, 4, "f16", False, True, False, True),
    (17, 3, 24, 3, "bf16", True, True, True, True), (40, 5, 72, 4, "f32", True, True, False, True),
    (33, 2, 7, 2, "f16", True, True, True, True), (130, 4, 264, 4, "bf16", True, False, True, False),
    (64, 1, 520, 3, "f32", False, True, True, False), (200, 6, 64, 4, "f32", True, True, True, True),
]


@pytest.mark.parametrize("case", CONV, ids=lambda c: "-".join(str(v) for v in c))
def test_causal_conv_and_gradients(case):
    T, B, D, W, dtype, silu, has_bias, has_state, ragged = case
    mk = _Maker(T * 131 + D, dtype)
    x, w = mk.act(T, B, D), mk.par(W, D, f=W ** -0.5)
    bias = mk.par(D, f=0.3) if has_bias else None
    state = mk.act(W - 1, B, D) if has_state else None
    n = mk.lengths(T, B) if ragged else None
    dy, dlast = mk.act(T, B, D), mk.act(W - 1, B, D)
    if ragged:
        _poison(n, x, dy)
    act = "silu" if silu else None
    y64, last64, c = ref.conv(_np(x), _np(w), _np(bias), _np(state), _np(n).astype(int) if ragged else None, silu)
    units = W + 1 + (8 + 2 * c["mag"].max() if silu else 0)
    y0, last0 = shivae_amd.causal_conv(x, w, bias, act, state, n, return_state=True)
    _near(y0, y64, c["mag"], units, "y")
    assert torch.equal(last0.double().cpu(), torch.from_numpy(last64))  # moved, not computed
    leaves = {k: v.clone().requires_grad_(True) for k, v in dict(x=x, weight=w, bias=bias, state=state).items() if v is not None}
    y, last = shivae_amd.causal_conv(leaves["x"], leaves["weight"], leaves.get("bias"), act, leaves.get("state"), n, return_state=True)
    assert torch.equal(y, y0) and torch.equal(last, last0)
    grads = dict(zip(leaves, torch.autograd.grad([y, last], list(leaves.values()), [dy, dlast])))
    want, scale = ref.conv_grad(_np(x), _np(w), _np(bias), _np(state), _np(n).astype(int) if ragged else None, silu, _np(dy), _np(dlast))
    for k, g in grads.items():
        more = 8 + np.log2(T * B) if k in ("weight", "bias") else W + 1
        # (a thread adds up to 64 rows one by one in dweight and dbias)
        _near(g, want[k], scale[k], units + more + (64 if k in ("weight", "bias") else 0), "d" + k)


def test_causal_conv_continues_and_steps():
    """A sequence in one call, in two calls joined by the state, and row by row: the same bits."""
    mk = _Maker(5, "bf16")
    T, B, D, W = 23, 3, 40, 4
    x, w, b, s0 = mk.act(T, B, D), mk.par(W, D), mk.par(D), mk.act(W - 1, B, D)
    y, last = shivae_amd.causal_conv(x, w, b, "silu", s0, return_state=True)
    ya, mid = shivae_amd.causal_conv(x[:9], w, b, "silu", s0, return_state=True)
    yb, end = shivae_amd.causal_conv(x[9:], w, b, "silu", mid, return_state=True)
    assert torch.equal(torch.cat([ya, yb]), y) and torch.equal(end, last)
    state, other = s0.clone(), torch.empty_like(s0)
    for t in range(T):
        if t % 2:
            yt = shivae_amd.causal_conv_step(x[t], w, b, state=state, activation="silu")
        else:
            yt = shivae_amd.causal_conv_step(x[t], w, b, state=state, activation="silu", state_out=other)
            state, other = other, state
        assert torch.equal(yt, y[t]), t
    assert torch.equal(state, last)


def test_causal_conv_strides():
    """Batch-major storage, a slice of the channels that is not aligned, a broadcast sequence, strided channels."""
    mk = _Maker(6, "f32")
    T, B, D, W = 12, 3, 16, 3
    w = mk.par(W, D)
    bt = mk.act(B, T, D)
    wide = mk.act(T, B, D + 3)
    forms = [bt.transpose(0, 1), wide[..., 1:1 + D], mk.act(T, 1, D).expand(T, B, D), mk.act(T, B, 2 * D)[..., ::2]]
    for x in forms:
        want = shivae_amd.causal_conv(x.contiguous(), w, None, "silu")
        assert torch.equal(shivae_amd.causal_conv(x, w, None, "silu"), want)
        leaf = x.detach().requires_grad_(True)
        g, = torch.autograd.grad(shivae_amd.causal_conv(leaf, w, None, "silu").sum(), leaf)  # (an expanded gradient)
        leaf2 = x.contiguous().detach().requires_grad_(True)
        g2, = torch.autograd.grad(shivae_amd.causal_conv(leaf2, w, None, "silu"), leaf2, torch.ones(T, B, D, device="cuda"))
        assert torch.equal(g, g2)


# ------------------------------------------------------------------------------------------------ selective scan
SCAN = [  # T, B, D, N, G, dtype, gate, extras (D and dt_bias), softplus, state, ragged
    (1, 1, 1, 1, 1, "f32", False, False, True, False, False), (1, 2, 5, 4, 1, "bf16", True, True, True, True, False),
    (2, 3, 8, 16, 2, "f32", True, True, False, True, True), (15, 2, 64, 16, 1, "f16", True, True, True, False, False),
    (16, 2, 65, 16, 1, "f32", False, True, True, True, True), (17, 4, 70, 5, 1, "bf16", True, False, True, True, True),
    (33, 3, 132, 8, 2, "f32", True, True, True, True, True), (50, 2, 96, 12, 4, "f16", True, True, True, True, False),
    (70, 1, 128, 16, 1, "f32", True, True, True, True, False),       # the time axis in pieces
    (300, 2, 64, 16, 1, "bf16", True, True, True, True, True),       # pieces, some behind a sequence's end
    (150, 1, 40, 17, 1, "f32", False, True, True, False, False), (200, 2, 24, 32, 2, "bf16", True, True, True, True, True),
    (100, 1, 80, 64, 1, "f32", True, True, True, True, False), (40, 3, 66, 40, 1, "f16", False, False, True, False, True),
    (20, 2, 10, 2, 5, "f32", True, True, True, True, True),
]


def _scan_inputs(case, seed=0):
    T, B, D, N, G, dtype, gate, extras, softplus, has_state, ragged = case
    mk = _Maker(T * 17 + D + N + seed, dtype)
    v = dict(u=mk.act(T, B, D), dt=mk.act(T, B, D), A=-torch.exp(mk.par(N, D, f=0.7)), B=mk.act(T, B, G, N), C=mk.act(T, B, G, N),
             D=mk.par(D, f=0.2, add=1.0) if extras else None, z=mk.act(T, B, D) if gate else None,
             dt_bias=mk.par(D, add=-2.0) if extras else None, state=mk.par(B, N, D) if has_state else None)
    if not softplus:  # steps straight from dt: positive, as a model's own activation would make them
        v["dt"] = (v["dt"].abs() * 0.3 + 0.01).to(v["dt"].dtype)
        v["dt_bias"] = None
    n = mk.lengths(T, B) if ragged else None
    dy, dlast = mk.act(T, B, D), mk.par(B, N, D)
    if ragged:
        _poison(n, v["u"], v["dt"], v["z"], v["B"], v["C"], dy)
    return v, n, softplus, dy, dlast


def _scan(v, n, softplus, want):
    return shivae_amd.selective_scan(v["u"], v["dt"], v["A"], v["B"], v["C"], v.get("D"), v.get("z"), v.get("dt_bias"), softplus,
                                     v.get("state"), n, want)


@pytest.mark.parametrize("case", SCAN, ids=lambda c: "-".join(str(v) for v in c))
def test_selective_scan_and_gradients(case):
    T, B, D = case[:3]
    v, n, softplus, dy, dlast = _scan_inputs(case)
    a = {k: _np(t) for k, t in v.items()}
    want, scale = ref.scan(a["u"], a["dt"], a["A"], a["B"], a["C"], a["D"], a["z"], a["dt_bias"], a["state"],
                           _np(n).astype(int) if n is not None else None, softplus, _np(dy), _np(dlast))
    units = 3 * T + 96
    y0, last0 = _scan(v, n, softplus, True)
    _near(y0, want["y"], scale["y"], units, "y")
    _near(last0, want["last"], scale["last"], units, "state")
    leaves = {k: t.clone().requires_grad_(True) for k, t in v.items() if t is not None}
    y, last = _scan({**{k: None for k in v}, **leaves}, n, softplus, True)
    assert torch.equal(y, y0) and torch.equal(last, last0)
    grads = dict(zip(leaves, torch.autograd.grad([y, last], list(leaves.values()), [dy, dlast])))
    for k, g in grads.items():
        terms = {"B": D, "C": D, "A": T * B, "D": T * B, "dt_bias": T * B}.get(k, 1)
        serial = T if k in ("A", "D", "dt_bias") else 0  # a thread adds a piece's rows one by one
        _near(g, want[k], scale[k], 2 * units + 8 + np.log2(terms) + serial, "d" + k)
    again = torch.autograd.grad(list(_scan({**{k: None for k in v}, **leaves}, n, softplus, True)), list(leaves.values()), [dy, dlast])
    for k, g in zip(leaves, again):
        assert torch.equal(g, grads[k]), k  # fixed orders of summation


@pytest.mark.parametrize("case", [(40, 3, 70, 16, 1, "f32"), (33, 2, 64, 24, 2, "bf16"), (21, 2, 6, 3, 3, "f16")], ids=str)
def test_selective_scan_continues_and_steps(case):
    """A sequence in one call, in two joined by the state, row by row in place and out of place."""
    T, B, D, N, G, dtype = case
    v, _, softplus, _, _ = _scan_inputs((T, B, D, N, G, dtype, True, True, True, True, False))
    a = {k: _np(t) for k, t in v.items()}
    want, scale = ref.scan(a["u"], a["dt"], a["A"], a["B"], a["C"], a["D"], a["z"], a["dt_bias"], a["state"], None, True)
    units = 3 * T + 96
    cut = 19

    def part(lo, hi, st):
        return {k: (t[lo:hi] if k in ("u", "dt", "B", "C", "z") else (st if k == "state" else t)) for k, t in v.items()}

    ya, mid = _scan(part(0, cut, v["state"]), None, True, True)
    yb, end = _scan(part(cut, T, mid), None, True, True)
    _near(torch.cat([ya, yb]), want["y"], scale["y"], units, "two calls")
    _near(end, want["last"], scale["last"], units, "two calls' state")
    state, other, ys = v["state"].clone(), torch.empty_like(v["state"]), []
    for t in range(T):
        args = (v["u"][t], v["dt"][t], v["A"], v["B"][t], v["C"][t], state, v["D"], v["z"][t], v["dt_bias"])
        if t % 2:
            ys.append(shivae_amd.selective_scan_step(*args))
        else:
            ys.append(shivae_amd.selective_scan_step(*args, state_out=other))
            state, other = other, state
    _near(torch.stack(ys), want["y"], scale["y"], units, "steps")
    _near(state, want["last"], scale["last"], units, "steps' state")


def test_selective_scan_strides():
    """Batch-major tensors, slices of one wide projection, B and C shared by all sequences (stride 0)."""
    mk = _Maker(9, "bf16")
    T, B, D, N = 37, 2, 72, 16
    wide = mk.act(B, T, 3 * D + 2 * N).transpose(0, 1)
    u, dt, z = wide[..., :D], wide[..., D:2 * D], wide[..., 2 * D:3 * D]
    Bm, Cm = wide[..., 3 * D:3 * D + N].unsqueeze(2), wide[..., 3 * D + N:].unsqueeze(2)
    A = -torch.exp(mk.par(N, D))
    shared = mk.act(T, 1, 1, N).expand(T, B, 1, N)
    for Bx, Cx in ((Bm, Cm), (shared, Cm)):
        x = [t.detach().requires_grad_(True) for t in (u, dt, Bx, Cx, z)]
        xc = [t.detach().contiguous().requires_grad_(True) for t in (u, dt, Bx, Cx, z)]
        y, yc = (shivae_amd.selective_scan(p[0], p[1], A, p[2], p[3], z=p[4]) for p in (x, xc))
        assert torch.equal(y, yc)
        g, gc = torch.autograd.grad(y.float().sum(), x), torch.autograd.grad(yc.float().sum(), xc)
        for a, b in zip(g, gc):
            assert torch.equal(a, b)


def test_non_finite_rows_stay_in_their_sequence():
    """An infinity or NaN inside one sequence reaches no other sequence, and no earlier row's output."""
    mk = _Maker(11, "f32")
    T, B, D, N = 40, 3, 64, 16
    u, dt, Bm, Cm = mk.act(T, B, D), mk.act(T, B, D), mk.act(T, B, 1, N), mk.act(T, B, 1, N)
    A = -torch.exp(mk.par(N, D))
    y = shivae_amd.selective_scan(u, dt, A, Bm, Cm)
    u2 = u.clone()
    u2[20, 1, 5] = float("inf")
    u2[25, 1, 6] = float("nan")
    y2 = shivae_amd.selective_scan(u2, dt, A, Bm, Cm)
    assert torch.equal(y2[:, [0, 2]], y[:, [0, 2]]) and torch.equal(y2[:20, 1], y[:20, 1])
    keep = [i for i in range(D) if i not in (5, 6)]
    assert torch.equal(y2[:, 1][:, keep], y[:, 1][:, keep])
    assert not torch.isfinite(y2[20, 1, 5]) and torch.isnan(y2[25, 1, 6])


def test_streams_and_graph_replay():
    """The whole training pass on a side stream, then captured once and replayed on new inputs, equal to eager every time."""
    case = (90, 2, 64, 16, 1, "bf16", True, True, True, True, True)
    v, n, softplus, dy, _ = _scan_inputs(case)
    mk = _Maker(3, "bf16")
    w = mk.par(4, 64)
    for k in ("u", "dt", "z", "B", "C"):
        v[k] = torch.nan_to_num(v[k])
    dy = torch.nan_to_num(dy)

    def train():
        x = v["u"].detach().requires_grad_(True)
        wl = w.detach().requires_grad_(True)
        c = shivae_amd.causal_conv(x, wl, None, "silu", lengths=n)
        y = _scan({**v, "u": c}, n, softplus, False)
        return [y.detach()] + list(torch.autograd.grad(y, [x, wl], dy))

    want = train()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = train()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    del got
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = train()
    for i in range(4):
        v["u"].copy_(mk.act(*v["u"].shape))
        n.copy_(torch.tensor([i * 30, 90 - i * 7], dtype=torch.int32))
        g.replay()
        eager = train()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager)), i


@pytest.mark.parametrize("only", ["D", "dt_bias"])
def test_selective_scan_with_one_of_its_parameters(only):
    """D without dt_bias and the other way round, with gradients."""
    case = (35, 2, 70, 16, 1, "f32", False, True, True, False, False)
    v, _, softplus, dy, _ = _scan_inputs(case)
    v["dt_bias" if only == "D" else "D"] = None
    a = {k: _np(t) for k, t in v.items()}
    want, scale = ref.scan(a["u"], a["dt"], a["A"], a["B"], a["C"], a["D"], None, a["dt_bias"], None, None, True, _np(dy))
    leaves = {k: t.clone().requires_grad_(True) for k, t in v.items() if t is not None}
    y = _scan({**{k: None for k in v}, **leaves}, None, True, False)
    _near(y, want["y"], scale["y"], 3 * 35 + 96, "y")
    for k, g in zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy)):
        _near(g, want[k], scale[k], 2 * (3 * 35 + 96) + 16 + 35, "d" + k)


def test_selective_scan_without_memory():
    """A = -inf keeps nothing of a state, and rows behind a sequence's end still leave the state as it is."""
    mk = _Maker(21, "f32")
    T, B, D, N = 21, 2, 64, 16
    u, dt, Bm, Cm, s0 = mk.act(T, B, D), mk.act(T, B, D), mk.act(T, B, 1, N), mk.act(T, B, 1, N), mk.par(B, N, D)
    A = torch.full((N, D), -float("inf"), device="cuda", requires_grad=True)
    n = torch.tensor([17, 0], device="cuda")
    y, last = shivae_amd.selective_scan(u, dt, A, Bm, Cm, initial_state=s0, lengths=n, return_state=True)
    step = torch.nn.functional.softplus(dt.double())
    want = (Cm[:, :, 0] * Bm[:, :, 0]).double().sum(-1, keepdim=True) * step * u.double()
    scale = (Cm[:, :, 0] * Bm[:, :, 0]).double().abs().sum(-1, keepdim=True) * (step * u.double()).abs()
    _near(y[:17, 0], want[:17, 0].cpu().numpy(), scale[:17, 0].cpu().numpy(), 64, "y")
    assert torch.equal(last[1], s0[1]) and torch.isfinite(last).all()
    g, = torch.autograd.grad(y.sum(), A)
    assert torch.equal(g, torch.zeros_like(g))


def test_refusals():
    mk = _Maker(22, "f32")
    T, B, D, N = 5, 2, 8, 4
    x, w, A, Bm = mk.act(T, B, D), mk.par(4, D), -torch.exp(mk.par(N, D)), mk.act(T, B, 1, N)
    conv, scan = shivae_amd.causal_conv, shivae_amd.selective_scan
    cs, ss = mk.act(3, B, D), mk.par(B, N, D)
    for f, args, kw, err in (
            (conv, (x, mk.par(5, D)), {}, ValueError), (conv, (x, mk.par(1, D)), {}, ValueError), (conv, (x, mk.par(4, D + 1)), {}, ValueError),
            (conv, (x, w.bfloat16()), {}, TypeError), (conv, (x, w.cpu()), {}, ValueError), (conv, (x, w), dict(activation="relu"), ValueError),
            (conv, (x, w, mk.par(D + 1)), {}, ValueError), (conv, (x, w), dict(initial_state=cs.bfloat16()), TypeError),
            (conv, (x, w), dict(initial_state=cs[:2]), ValueError), (conv, (x, w), dict(lengths=torch.ones(B, device="cuda")), TypeError),
            (conv, (x, w), dict(lengths=torch.ones(B, dtype=torch.int32)), ValueError), (conv, (x, w), dict(lengths=[1, 2]), TypeError),
            (scan, (x, x.bfloat16(), A, Bm, Bm), {}, TypeError), (scan, (x, x[:4], A, Bm, Bm), {}, ValueError),
            (scan, (x, x, mk.par(65, D), mk.act(T, B, 1, 65), mk.act(T, B, 1, 65)), {}, ValueError), (scan, (x, x, A, Bm[:, :, 0], Bm), {}, ValueError),
            (scan, (x, x, A, mk.act(T, B, 3, N), mk.act(T, B, 3, N)), {}, ValueError), (scan, (x, x, A, Bm, Bm[..., :3]), {}, ValueError),
            (scan, (x, x, A.double(), Bm, Bm), {}, TypeError), (scan, (x, x, A, Bm, Bm), dict(initial_state=ss.bfloat16()), TypeError),
            (scan, (x, x, A, Bm, Bm), dict(z=x.cpu()), ValueError),
            (shivae_amd.causal_conv_step, (x[0], w), dict(state=cs, state_out=cs[:2]), ValueError),
            (shivae_amd.causal_conv_step, (x[0], w.requires_grad_(True)), dict(state=cs), RuntimeError),
            (shivae_amd.selective_scan_step, (x[0], x[0], A, Bm[0], Bm[0], ss.transpose(0, 1).contiguous().transpose(0, 1)), {}, ValueError),
            (shivae_amd.selective_scan_step, (x[0], x[0], A, Bm[0], Bm[0], None), {}, TypeError)):
        with pytest.raises(err):
            f(*args, **kw)
    big = mk.par(B + 1, N, D)  # a new state that overlaps the old one by all but one sequence
    with pytest.raises(ValueError, match="overlaps"):
        shivae_amd.selective_scan_step(x[0], x[0], A, Bm[0], Bm[0], big[:B], state_out=big[1:])


def test_a_state_that_a_backward_pass_needs_is_not_changed_unnoticed():
    """The steps write the state behind autograd's back: a graph that holds the old one refuses its backward pass."""
    mk = _Maker(21, "f32")
    x, w, A, B, C = mk.act(5, 2, 8), mk.par(4, 8), -mk.par(4, 8).abs(), mk.act(5, 2, 1, 4), mk.act(5, 2, 1, 4)
    conv_state, scan_state = mk.act(3, 2, 8), mk.par(2, 4, 8)
    leaf = x.clone().requires_grad_(True)
    y = shivae_amd.causal_conv(leaf, w, initial_state=conv_state)
    z = shivae_amd.selective_scan(leaf, x, A, B, C, initial_state=scan_state)
    shivae_amd.causal_conv_step(x[0], w, state=conv_state)
    shivae_amd.selective_scan_step(x[0], x[0], A, B[0], C[0], scan_state)
    for out in (y, z):
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(out, leaf, torch.ones_like(out))
    with torch.inference_mode():
        state = torch.zeros(3, 2, 8, device="cuda")
        shivae_amd.causal_conv_step(x[0], w, state=state)


def test_two_passes_of_states_in_a_graph():
    """More than 16 states: the backward pass keeps adjoints in dynamic LDS, captured and replayed."""
    v, n, softplus, dy, _ = _scan_inputs((50, 2, 40, 40, 1, "bf16", True, True, True, False, False))

    def train():
        u = v["u"].detach().requires_grad_(True)
        y = _scan({**v, "u": u}, None, True, False)
        return [y.detach(), torch.autograd.grad(y, u, dy)[0]]

    train()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = train()
    for i in range(3):
        v["u"].mul_(-0.7)
        g.replay()
        eager = train()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager)), i


def test_state_offsets_past_32_bits():
    """States of more than 2^32 bytes and 2^31 elements apart in one tensor: the last sequence is computed like the first."""
    B, D, N = 33, 1 << 20, 64  # 2^31 + 2^26 fp32 states, 8.6 GB
    if torch.cuda.mem_get_info()[0] < 40e9:
        pytest.skip("not enough free memory")
    mk = _Maker(13, "bf16")
    u1, d1, B1, C1 = mk.act(1, D), mk.act(1, D), mk.act(1, 1, N), mk.act(1, 1, N)
    A = -torch.exp(mk.par(N, D, f=0.3))
    s1 = torch.randn(1, N, D, device="cuda")
    want_state = torch.empty_like(s1)
    want = shivae_amd.selective_scan_step(u1, d1, A, B1, C1, s1, state_out=want_state)
    state = torch.zeros(B, N, D, device="cuda")
    state[-1] = s1[0]
    y = shivae_amd.selective_scan_step(u1.expand(B, D).contiguous(), d1.expand(B, D).contiguous(), A, B1.expand(B, 1, N).contiguous(),
                                       C1.expand(B, 1, N).contiguous(), state)
    assert torch.equal(y[-1], want[0]) and torch.equal(state[-1], want_state[0])
