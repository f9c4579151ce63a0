"""Drawing category indices from logits (``csrc/sample.hip``): temperature, top-k, top-p and min-p, from given uniform numbers,
so that a draw is a function of its inputs.  ``ShiVAE.sample_categories`` draws a model's categorical attributes with it."""
from ctypes import byref

import torch

from . import _native as N
from .ssm import _DTYPES, _call, _wants_grad

MAX_CATEGORIES = 1048512  # SHIVAE_SAMPLE_MAX


def _setting(v, name, shape, device, dtype, low, high=None):
    """A number for all rows, or a tensor with one for each -> (pointer owner, number)."""
    if isinstance(v, torch.Tensor):
        if v.device != device:
            raise ValueError("%s is on %s, not on %s" % (name, v.device, device))
        if v.shape != shape:
            raise ValueError("%s has shape %s, expected a number or %s" % (name, tuple(v.shape), tuple(shape)))
        if v.is_floating_point() != dtype.is_floating_point or v.dtype == torch.bool:
            raise TypeError("%s is %s, expected %s" % (name, v.dtype, dtype))
        if v.dtype == torch.int64:
            v = v.clamp(-1, 2 ** 31 - 1)
        return v.to(dtype).contiguous(), 0
    if not dtype.is_floating_point and int(v) != v:
        raise ValueError("%s must be a whole number, not %r" % (name, v))
    if not v >= low or (high is not None and v > high):
        raise ValueError("%s = %r is out of range" % (name, v))
    return None, v


def sample_categories(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, return_logprob=False):
    """Draws one index of the last axis for every row of ``logits`` [..., V] (float32, bfloat16, float16).

    With w = exp((logit - max) / temperature): kept are the top_k largest (equal logits: lowest index first; 0: all), of these the
    shortest lead whose weight reaches top_p of theirs (1: all), of these the ones with w >= min_p; the largest is always kept.
    The index drawn is the first, in index order, at which the running sum of kept weights exceeds ``u`` times their sum;
    temperature 0 takes the largest logit.  ``u`` [...] float32 holds uniform numbers in [0, 1).  Every setting is a number or a
    tensor [...] with one for each row.  NaN logits count as -inf; a row without a logit above -inf gives -1; logits at +inf share
    everything.  A weight is good to 2^-38 of itself and held as a multiple of 2^-43 of the largest (0 below 2^-44); sums of these are exact,
    so the result does not depend on scheduling.

    Returns int64 indices [...], or (indices, log-probability of the index among the kept [...] float32); the log-probability
    is 0 for temperature 0 and -inf where the index is -1.  It has no derivative: with logits or a temperature that require one the call
    is refused, under torch.no_grad() or with detached tensors it is not."""
    if not isinstance(logits, torch.Tensor) or logits.dtype not in _DTYPES:
        raise TypeError("logits must be a float32, bfloat16 or float16 tensor")
    if logits.dim() < 1 or logits.numel() == 0:
        raise ValueError("logits of shape %s have nothing to draw from" % (tuple(logits.shape),))
    if return_logprob and _wants_grad(logits, temperature if isinstance(temperature, torch.Tensor) else None):
        raise RuntimeError("the log-probability has no derivative: call under torch.no_grad(), or detach logits and temperature")
    V = logits.shape[-1]
    if V > MAX_CATEGORIES:
        raise ValueError("%d categories, up to %d are supported" % (V, MAX_CATEGORIES))
    if not logits.is_cuda:
        raise N.ShiVAENativeError("sample_categories runs as a HIP kernel: the logits are on %s and there is no CPU fallback" % logits.device)
    dev, shape = logits.device, logits.shape[:-1]
    if not isinstance(u, torch.Tensor) or u.dtype is not torch.float32:
        raise TypeError("u must be a float32 tensor")
    if u.shape != shape or u.device != dev:
        raise ValueError("u must have shape %s and lie on %s" % (tuple(shape), dev))
    t_rows, t = _setting(temperature, "temperature", shape, dev, torch.float32, 0.0)
    k_rows, k = _setting(top_k, "top_k", shape, dev, torch.int32, 0)
    p_rows, p = _setting(top_p, "top_p", shape, dev, torch.float32, 0.0, 1.0)
    m_rows, m = _setting(min_p, "min_p", shape, dev, torch.float32, 0.0, 1.0)
    rows = logits.detach().reshape(-1, V) if logits.dim() != 2 else logits
    if rows.stride(1) != 1 and V > 1:
        rows = rows.contiguous()
    u = u.contiguous()
    tokens = torch.empty(shape, dtype=torch.int64, device=dev)
    logprob = torch.empty(shape, dtype=torch.float32, device=dev) if return_logprob else None
    args = N.SampleArgs(rows.shape[0], V, _DTYPES[rows.dtype], rows.data_ptr(), rows.stride(0), u.data_ptr(),
                        *[None if r is None else r.data_ptr() for r in (t_rows, k_rows, p_rows, m_rows)], t, min(int(k), 2 ** 31 - 1), p, m,
                        tokens.data_ptr(), None if logprob is None else logprob.data_ptr())
    _call(dev, N.lib().shivae_sample_categories, byref(args))
    return (tokens, logprob) if return_logprob else tokens
