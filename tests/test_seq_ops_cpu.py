"""On the CPU: the 64-bit restatements' gradients against differences, and what the operators refuse."""
import numpy as np
import pytest
import torch

import _seq_ref as ref
import shivae_amd
from shivae_amd import _native as N


def _differences(f, x, g, h=1e-6):
    """Directional derivatives along random directions against <gradient, direction>."""
    rng = np.random.default_rng(1)
    for _ in range(3):
        d = rng.standard_normal(x.shape)
        num = (f(x + h * d) - f(x - h * d)) / (2 * h)
        assert num == pytest.approx(float((g * d).sum()), rel=2e-6, abs=2e-7)


def test_conv_gradients_are_the_differences():
    rng = np.random.default_rng(0)
    T, B, D, W = 7, 3, 4, 4
    v = dict(x=rng.standard_normal((T, B, D)), weight=rng.standard_normal((W, D)), bias=rng.standard_normal(D),
             state=rng.standard_normal((W - 1, B, D)))
    n, dy, dl = np.array([7, 0, 2]), rng.standard_normal((T, B, D)), rng.standard_normal((W - 1, B, D))
    g, _ = ref.conv_grad(v["x"], v["weight"], v["bias"], v["state"], n, True, dy, dl)
    for k in v:
        def f(t):
            a = {**v, k: t}
            y, last, _ = ref.conv(a["x"], a["weight"], a["bias"], a["state"], n, True)
            return (y * dy).sum() + (last * dl).sum()
        _differences(f, v[k], g[k])


@pytest.mark.parametrize("use_softplus", [True, False])
def test_scan_gradients_are_the_differences(use_softplus):
    rng = np.random.default_rng(2)
    T, B, D, Ns, G = 6, 3, 4, 3, 2
    v = dict(u=rng.standard_normal((T, B, D)), dt=rng.standard_normal((T, B, D)) * 0.5, A=-np.exp(rng.standard_normal((Ns, D)) * 0.5),
             B=rng.standard_normal((T, B, G, Ns)), C=rng.standard_normal((T, B, G, Ns)), D=rng.standard_normal(D),
             z=rng.standard_normal((T, B, D)), dt_bias=rng.standard_normal(D) * 0.3, state=rng.standard_normal((B, Ns, D)))
    n, dy, dl = np.array([6, 0, 4]), rng.standard_normal((T, B, D)), rng.standard_normal((B, Ns, D))
    order = ("u", "dt", "A", "B", "C", "D", "z", "dt_bias", "state")
    out, _ = ref.scan(*(v[k] for k in order), n, use_softplus, dy, dl)
    for k in order:
        def f(t):
            o, _ = ref.scan(*({**v, k: t}[q] for q in order), n, use_softplus)
            return (o["y"] * dy).sum() + (o["last"] * dl).sum()
        _differences(f, v[k], out[k])




def test_operators_need_a_gpu():
    x = torch.zeros(2, 1, 4)
    with pytest.raises(N.ShiVAENativeError, match="no CPU fallback"):
        shivae_amd.causal_conv(x, torch.zeros(4, 4))
    with pytest.raises(N.ShiVAENativeError, match="no CPU fallback"):
        shivae_amd.selective_scan(x, x, torch.zeros(2, 4), torch.zeros(2, 1, 1, 2), torch.zeros(2, 1, 1, 2))


def test_wrong_first_arguments():
    with pytest.raises(TypeError, match="float64"):
        shivae_amd.causal_conv(torch.zeros(2, 1, 4, dtype=torch.float64), torch.zeros(4, 4))
    with pytest.raises(ValueError, match="dimensions"):
        shivae_amd.causal_conv(torch.zeros(2, 4), torch.zeros(4, 4))
    with pytest.raises(ValueError, match="no elements"):
        shivae_amd.selective_scan(torch.zeros(0, 1, 4), None, None, None, None)
    with pytest.raises(TypeError, match="tensor"):
        shivae_amd.selective_scan_step(None, None, None, None, None, None)


def _conv(**kw):
    a = N.ConvArgs(4, 2, 8, 4, 0, 1, 64, 16, 8, 64)
    a.y, a.y_st, a.y_sb = 64, 16, 8
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def _ssm(**kw):
    a = N.SsmArgs(4, 2, 8, 4, 1, 0, 1)
    for k in ("u", "dt", "A", "Bm", "Cm", "y"):
        setattr(a, k, 64)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def _refused(f, args, match, *more):
    import ctypes
    rc = f(ctypes.byref(args), *more, None)
    assert rc < 0 and match in N.lib().shivae_last_error().decode(), (rc, N.lib().shivae_last_error())


def test_c_entries_refuse_bad_arguments():
    """Every refusal comes before any GPU call, so it can be seen without one."""
    L = N.lib()
    for kw, match in ((dict(W=1), "filter width"), (dict(W=5), "filter width"), (dict(T=0), "positive"), (dict(B=-1), "positive"),
                      (dict(dtype=3), "dtype"), (dict(x=None), "required"), (dict(y=None), "y is required"),
                      (dict(T=17, state=64, state_out=64), "in place")):
        _refused(L.shivae_causal_conv_fwd, _conv(**kw), match)
    full = dict(dy=64, dx=64, dweight=64)
    for kw, match in ((dict(), "dy, dx and dweight"), (dict(full, state=64), "gradient"), (dict(full, bias=64), "bias"), (full, "workspace")):
        _refused(L.shivae_causal_conv_bwd, _conv(**kw), match, None, 0)
    for kw, match in ((dict(N=0), "states per channel"), (dict(N=65), "states per channel"), (dict(G=3), "do not divide"),
                      (dict(dtype=-1), "dtype"), (dict(u=None), "required"), (dict(y=None), "y is required"),
                      (dict(T=17, state=64, state_out=64), "in place")):
        _refused(L.shivae_selective_scan_fwd, _ssm(**kw), match, None, 0)
    _refused(L.shivae_selective_scan_fwd, _ssm(T=4096), "workspace", None, 0)  # split, and no room for the pieces
    full = {k: 64 for k in ("dy", "du", "ddt", "dB", "dC", "dA", "ckpt")}
    for kw, match in ((dict(), "ckpt are required"), (dict(full, z=64), "gradients"), (dict(full, Dp=64), "gradients"), (full, "workspace")):
        _refused(L.shivae_selective_scan_bwd, _ssm(**kw), match, None, 0)
    assert L.shivae_causal_conv_bwd_ws(None) == 0 and L.shivae_selective_scan_bwd_ws(None) == 0
