"""Causal convolution and selective scan at sizes that take the other choices of the host: longer runs of the convolution's backward pass,
grids that fill the card unsplit, many and long pieces of the time axis, and sums of partial gradients in two launches.

Tolerances as in test_gpu_seq_ops.py: operations times 2^-24 times the same sums over absolute values.  What grows here is the number of
additions one after the other: `run` rows by a thread of the convolution (a piece's rows in the scan), then the partial sums, of which a
wave's four accumulators take every 16th, joined by 4 additions, in slices of a 64th where there are more than 64."""
import ctypes

import numpy as np
import pytest
import torch

import _seq_ref as ref
import shivae_amd
from shivae_amd import _native as N
from shivae_amd import ssm
from test_gpu_seq_ops import TYPES, _near, _np, _scan, _scan_inputs

pytestmark = pytest.mark.gpu


def _partial_additions(n):
    """Additions in sequence for n partial sums."""
    if n <= 64:
        return -(-n // 16) + 4
    step = -(-n // 64)
    return -(-step // 16) + 4 + -(-(-(-n // step)) // 16) + 4


# ------------------------------------------------------------------------------------------------ convolution, in 64 bits on the device
def _conv64(x, w, bias, state, live, act, dy, dlast, n, absolute):
    """Gradients (or, over absolute values, their scales) by input name, as in _seq_ref.conv_grad."""
    f = torch.abs if absolute else (lambda t: t)
    T, W = x.shape[0], w.shape[0]
    xs = torch.cat([state, torch.where(live, x, 0.0)])
    pre = bias + sum(w[j] * xs[j:j + T] for j in range(W))
    g = f(torch.where(live, dy, 0.0))
    if act:
        s = torch.sigmoid(pre)
        if absolute:
            g = g * (s + pre.abs() * s * (1 - s) + 0.5 * (bias.abs() + sum((w[j] * xs[j:j + T]).abs() for j in range(W))))
        else:
            g = g * (s + pre * s * (1 - s))
    dxs = torch.zeros_like(xs)
    for j in range(W):
        dxs[j:j + T] += f(w[j]) * g
    b = torch.arange(x.shape[1], device=x.device)
    for j in range(W - 1):
        dxs[n.long() + j, b] += f(dlast[j])
    return dict(x=torch.where(live, dxs[W - 1:], 0.0), state=dxs[:W - 1], bias=g.sum((0, 1)),
                weight=torch.stack([(g * f(xs[j:j + T])).sum((0, 1)) for j in range(W)]))


RUNS = [  # T, B, D, W, dtype, silu, the run that the backward pass takes
    (1000, 64, 256, 4, "f32", True, 32), (300, 64, 257, 4, "f32", True, 32), (260, 256, 512, 4, "bf16", True, 32),
    (300, 64, 1025, 3, "f32", True, 256), (270, 128, 4096, 2, "bf16", False, 256), (130, 200, 1030, 4, "f16", True, 256),
]


@pytest.mark.parametrize("case", RUNS, ids=lambda c: "-".join(str(v) for v in c))
def test_causal_conv_gradients_in_long_runs(case):
    T, B, D, W, dtype, silu, run = case
    vec = {"f32": 4}.get(dtype, 8)
    seqs = B * (-(-D // vec) if D % vec == 0 else D)  # threads of a run: 16-byte groups of channels, or channels
    assert run == 256 or seqs * -(-T // (2 * run)) < 131072
    assert seqs * -(-T // run) >= 131072, "a shorter run"
    gen = torch.Generator(device="cuda").manual_seed(T + D)

    def rn(*shape, f=1.0):
        return torch.randn(*shape, device="cuda", generator=gen) * f

    ty = TYPES[dtype]
    x, state, dy, dlast = rn(T, B, D).to(ty), rn(W - 1, B, D).to(ty), rn(T, B, D).to(ty), rn(W - 1, B, D).to(ty)
    w, bias = rn(W, D, f=W ** -0.5), rn(D, f=0.3)
    n = torch.randint(0, T + 1, (B,), device="cuda", generator=gen, dtype=torch.int32)
    n[:3] = torch.tensor([0, T, 1], dtype=torch.int32)
    live = (torch.arange(T, device="cuda")[:, None] < n)[..., None]
    x, dy = torch.where(live, x, float("nan")), torch.where(live, dy, float("nan"))
    if D % vec == 0 and vec == 8:  # (the workspace is that of the shortest run, by 8 channels a thread)
        args = N.ConvArgs(T, B, D, W, 1, 1, x.data_ptr(), B * D, D, w.data_ptr())
        parts, cols = -(-T // run) * B, (W + 1) * D
        assert N.lib().shivae_causal_conv_bwd_ws(ctypes.byref(args)) == 4 * cols * (parts + (64 if parts > 64 else 0))
    leaves = {k: t.clone().requires_grad_(True) for k, t in dict(x=x, weight=w, bias=bias, state=state).items()}
    y, last = shivae_amd.causal_conv(leaves["x"], leaves["weight"], leaves["bias"], "silu" if silu else None, leaves["state"], n, return_state=True)
    grads = dict(zip(leaves, torch.autograd.grad([y, last], list(leaves.values()), [dy, dlast])))
    a = [t.double() for t in (x, w, bias, state)]
    want, scale = (_conv64(*a, live, silu, dy.double(), dlast.double(), n, absolute) for absolute in (False, True))
    mag = float((bias.abs() + sum((w[j] * torch.cat([state.float(), torch.where(live, x, 0.0).float()])[j:j + T]).abs() for j in range(W))).max())
    units = W + 1 + (8 + 2 * mag if silu else 0)
    for k, g in grads.items():
        more = min(run, T) + _partial_additions(-(-T // run) * B) if k in ("weight", "bias") else W + 1
        half = torch.finfo(g.dtype).eps / 2
        tiny = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -133, torch.float32: 2.0 ** -126}[g.dtype]
        tol = half * want[k].abs() + (1 + half) * (units + more) * 2.0 ** -24 * scale[k] + tiny
        bad = ~((g.double() - want[k]).abs() <= tol)
        assert not bad.any(), (k, int(bad.sum()), bad.nonzero()[0].tolist())


# ------------------------------------------------------------------------------------------------ scan
def _pieces(T, B, D, G):
    groups = -(-(D // G) // 64) * G * B
    np_ = min(1024 // groups, 32, -(-T // 64)) if groups <= 256 else 1
    plen = -(-(-(-T // np_)) // 16) * 16
    return -(-T // plen), plen


SPLITS = [  # T, B, D, N, G, dtype, gate, extras, softplus, state, ragged; pieces, rows of a piece
    ((200, 90, 190, 16, 1, "f32", True, True, True, True, True), 1, 208),       # a full grid, unsplit; more than 64 partial sums
    ((200, 260, 8, 64, 1, "f16", True, True, True, True, True), 1, 208),        # the same with four passes of states
    ((2048, 1, 64, 16, 1, "bf16", True, True, True, True, False), 32, 64),      # the most pieces
    ((3001, 1, 40, 8, 1, "f32", True, True, True, False, False), 32, 96),       # and longer ones
    ((640, 9, 64, 16, 1, "f32", False, True, True, True, True), 10, 64),        # pieces and more than 64 partial sums
    ((700, 4, 72, 40, 1, "bf16", True, True, True, True, True), 11, 64),        # pieces and three passes of states
]


@pytest.mark.parametrize("case, pieces, rows", SPLITS, ids=str)
def test_selective_scan_in_pieces_and_full_grids(case, pieces, rows):
    T, B, D, Ns, G = case[:5]
    assert _pieces(T, B, D, G) == (pieces, rows)
    v, n, softplus, dy, dlast = _scan_inputs(case)
    if pieces > 1 or T > 256:  # (the workspace says how many pieces the library takes)
        args = ssm._scan_args(v["u"], v["dt"], None, v["B"], v["C"], v["A"], None, None, None, None, 1)
        assert N.lib().shivae_selective_scan_fwd_ws(ctypes.byref(args)) == 4 * pieces * B * (Ns + 1) * D
    a = {k: _np(t) for k, t in v.items()}
    want, scale = ref.scan(a["u"], a["dt"], a["A"], a["B"], a["C"], a["D"], a["z"], a["dt_bias"], a["state"],
                           _np(n).astype(int) if n is not None else None, softplus, _np(dy), _np(dlast))
    units = 3 * T + 96
    leaves = {k: t.clone().requires_grad_(True) for k, t in v.items() if t is not None}
    y, last = _scan({**{k: None for k in v}, **leaves}, n, softplus, True)
    _near(y, want["y"], scale["y"], units, "y")
    _near(last, want["last"], scale["last"], units, "state")
    for k, g in zip(leaves, torch.autograd.grad([y, last], list(leaves.values()), [dy, dlast])):
        terms = {"B": D, "C": D}.get(k, 1)
        serial = rows + 2 + _partial_additions(pieces * B) if k in ("A", "D", "dt_bias") else 0
        _near(g, want[k], scale[k], 2 * units + 8 + np.log2(terms) + serial, "d" + k)
