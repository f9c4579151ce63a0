"""Derivatives that the sequence operators and the sampler do not have are refused, not dropped."""
import pytest
import torch
from torch.autograd import forward_ad

import shivae_amd

pytestmark = pytest.mark.gpu


def _calls():
    gen = torch.Generator(device="cuda").manual_seed(0)

    def rn(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    T, B, D, Ns = 5, 2, 8, 4
    x, w, b, cs = rn(T, B, D), rn(4, D), rn(D), rn(3, B, D)
    scan = dict(u=rn(T, B, D), dt=rn(T, B, D), A=-rn(Ns, D).abs(), B=rn(T, B, 1, Ns), C=rn(T, B, 1, Ns), D=rn(D), z=rn(T, B, D), dt_bias=rn(D))
    step = {k: t[0] if t.dim() > 2 else t for k, t in scan.items()}
    ss = rn(B, Ns, D)
    return [(shivae_amd.causal_conv, dict(x=x, weight=w, bias=b, initial_state=cs)),
            (shivae_amd.causal_conv_step, dict(x=x[0], weight=w, bias=b, state=cs)),
            (shivae_amd.selective_scan, dict(**scan, initial_state=ss)),
            (shivae_amd.selective_scan_step, dict(**step, state=ss))]


def test_forward_mode_is_refused():
    for f, kw in _calls():
        for k, t in kw.items():
            with forward_ad.dual_level():
                dual = forward_ad.make_dual(t, torch.ones_like(t))
                for grad in (True, False):
                    with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="forward-mode"):
                        f(**{**kw, k: dual})
                f(**kw)  # (no tangent: the call is as ever)


def test_forward_mode_through_a_backward_pass_is_refused():
    for f, kw in _calls()[::2]:
        leaf = next(iter(kw.values())).requires_grad_(True)
        y = f(**kw)
        with forward_ad.dual_level():
            dy = forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y))
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(y, leaf, dy)


def test_second_derivatives_are_refused():
    """A recorded gradient may be used; what differentiates it raises, also where the gradient came from a constant or reaches the leaf by
    another path too."""
    for f, kw in _calls()[::2]:
        for k in kw:
            leaves = {**kw, k: kw[k].detach().clone().requires_grad_(True)}
            for loss in (torch.Tensor.sum, lambda y: y.square().sum()):
                y = f(**leaves)
                want, = torch.autograd.grad(loss(y), leaves[k], retain_graph=True)
                g, = torch.autograd.grad(loss(y), leaves[k], create_graph=True)
                assert torch.equal(g, want)
                total = loss(y) + g.square().sum()
                with pytest.raises(RuntimeError, match="second derivative"):
                    torch.autograd.grad(total, leaves[k], retain_graph=True)
                with pytest.raises(RuntimeError, match="second derivative"):
                    total.backward()


def test_the_log_probability_is_not_differentiable():
    """It is refused where a gradient would be lost; indices have none, as those of argmax."""
    lg, u, t = torch.randn(3, 50, device="cuda"), torch.rand(3, device="cuda"), torch.ones(3, device="cuda")
    f = shivae_amd.sample_categories
    want, logp = f(lg, u, t, return_logprob=True)
    for kw in (dict(logits=lg.clone().requires_grad_(True), temperature=t), dict(logits=lg, temperature=t.clone().requires_grad_(True))):
        with pytest.raises(RuntimeError, match="no derivative"):
            f(u=u, return_logprob=True, **kw)
        assert torch.equal(f(u=u, **kw), want)
        with torch.no_grad():
            assert torch.equal(f(u=u, return_logprob=True, **kw)[1], logp)
        detached = {k: v.detach() for k, v in kw.items()}
        assert torch.equal(f(u=u, return_logprob=True, **detached)[1], logp)
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            f(forward_ad.make_dual(lg, torch.ones_like(lg)), u, t, return_logprob=True)


def test_a_new_state_that_requires_a_gradient_is_refused():
    """As an in-place write to a leaf is; under no_grad it is written."""
    for f, kw in _calls()[1::2]:
        out = torch.zeros_like(kw["state"]).requires_grad_(True)
        with pytest.raises(RuntimeError, match="no backward pass"):
            f(**kw, state_out=out)
        assert not out.any()
        with torch.no_grad():
            f(**kw, state_out=out)
        assert out.any()
