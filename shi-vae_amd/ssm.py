"""Sequence operators beside the recurrent scans: a short causal convolution over time and a selective state-space scan,
as HIP kernels (``csrc/conv.hip``, ``csrc/ssm.hip``) with their backward passes and their single-token steps.

Tensors are time-major, ``[T, B, channels]``, as everywhere in this package; any strides over T and B are read in place
(batch-major storage: pass ``x.transpose(0, 1)``), only the channel axis has to be contiguous and is copied where it is not.
Activations are float32, bfloat16 or float16, all of one call in one type; parameters and scan states are float32, and so is
the arithmetic: every result is rounded once, where it is stored.

``lengths`` ([B], int32 or int64, on the device) gives the number of rows of each sequence (clamped to 0..T); rows behind
it are not read, outputs and gradients are 0 there, and the state that comes out is the one behind the last row.

All calls enqueue on the current stream of the tensors' device and do not synchronise.  There is no CPU fallback.  The sequence forms
have a first derivative in reverse mode; a derivative of it, and dual tensors of forward mode, are refused."""
from ctypes import byref

import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version  # a state written in place that a backward pass still needs is an error there

from . import _native as N

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


# ------------------------------------------------------------------------------------------------ arguments
def _ptr(t):
    return None if t is None else t.data_ptr()


def _rows(t):
    """The tensor with a contiguous last axis."""
    return t if t.stride(-1) == 1 or t.size(-1) == 1 else t.contiguous()


def _activation(t, name, shape, dtype, device):
    if isinstance(t, torch.Tensor) and t.shape == shape and t.dtype is dtype and t.device == device:
        return t if t.stride(-1) == 1 else _rows(t)
    if not isinstance(t, torch.Tensor):
        raise TypeError("%s must be a tensor" % name)
    if t.device != device:
        raise ValueError("%s is on %s, not on %s" % (name, t.device, device))
    if t.dtype != dtype:
        raise TypeError("%s is %s, expected %s" % (name, t.dtype, dtype))
    raise ValueError("%s has shape %s, expected %s" % (name, tuple(t.shape), shape))


def _param(t, name, shape, device, dtype=torch.float32):
    if t is None:
        return None
    t = _activation(t, name, shape, dtype, device)
    return t if t.is_contiguous() else t.contiguous()


def _lengths(t, B, device):
    if t is None:
        return None
    if not isinstance(t, torch.Tensor) or t.dtype not in (torch.int32, torch.int64):
        raise TypeError("lengths must be an int32 or int64 tensor")
    if t.device != device or tuple(t.shape) != (B,):
        raise ValueError("lengths must have shape (%d,) and lie on %s" % (B, device))
    if t.dtype == torch.int64:
        t = t.clamp(0, 2 ** 31 - 1).to(torch.int32)
    return t.contiguous()


def _first(x, name, ndim):
    """Checks the tensor that fixes device, type and sizes."""
    if not isinstance(x, torch.Tensor):
        raise TypeError("%s must be a tensor" % name)
    if x.dtype not in _DTYPES:
        raise TypeError("%s is %s; float32, bfloat16 and float16 are supported" % (name, x.dtype))
    if x.dim() != ndim:
        raise ValueError("%s has %d dimensions, expected %d" % (name, x.dim(), ndim))
    if x.numel() == 0:
        raise ValueError("%s has no elements: %s" % (name, tuple(x.shape)))
    if not x.is_cuda:
        raise N.ShiVAENativeError("the sequence operators run as HIP kernels: %s is on %s and there is no CPU fallback" % (name, x.device))
    return _rows(x)


def _call(device, f, *args):
    """Runs a library call on `device` and its current stream."""
    index = device.index
    if index != torch._C._cuda_getDevice():
        with torch.cuda.device(device):
            return N.check(f(*args, torch._C._cuda_getCurrentRawStream(index)))
    rc = f(*args, torch._C._cuda_getCurrentRawStream(index))  # (a tenth of the time of current_stream(device).cuda_stream)
    if rc:
        N.check(rc)


def _no_tangents(*tensors):
    if forward_ad._current_level >= 0:  # (inside of a dual_level: otherwise no tensor has a tangent)
        for t in tensors:
            if isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError("the sequence operators and the sampler have no forward-mode derivative: unpack the dual tensor, or use the backward pass")


def _wants_grad(*tensors):
    _no_tangents(*tensors)
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def _step_state(state, state_out):
    """The buffer of the new state: `state` itself, or one that does not overlap it."""
    if state_out is None or state_out is state:
        if not state.is_contiguous():
            raise ValueError("the state must be contiguous to be updated in place")
        return state
    if not isinstance(state_out, torch.Tensor) or state_out.dtype != state.dtype or state_out.shape != state.shape or state_out.device != state.device:
        raise ValueError("state_out must be like the state")
    if not state_out.is_contiguous():
        raise ValueError("state_out must be contiguous")
    a, b, n = state.data_ptr(), state_out.data_ptr(), state.numel() * state.element_size()
    if a != b and abs(a - b) < n:
        raise ValueError("state_out overlaps the state")
    return state_out


class _Recorded(torch.autograd.Function):
    """The result of a backward pass that is itself recorded (create_graph), as a function of all that it depends on: a derivative that
    passes through it raises."""
    @staticmethod
    def forward(ctx, grads, *depends_on):
        return grads()

    @staticmethod
    def backward(ctx, *g):
        raise RuntimeError("the sequence operators have no second derivative")


def _first_derivative(grads, *depends_on):
    _no_tangents(*depends_on)
    return _Recorded.apply(grads, *depends_on) if torch.is_grad_enabled() else grads()


def _no_backward(*tensors):
    if _wants_grad(*tensors):
        raise RuntimeError("the single-token steps have no backward pass: call them under torch.no_grad(), or use the sequence form with one row")


# ------------------------------------------------------------------------------------------------ causal convolution
def _conv_args(x, weight, bias, state, lengths, silu, y=None, state_out=None, dy=None, dstate_out=None, dx=None, dweight=None,
               dbias=None, dstate=None):
    T, B, D = x.shape
    return N.ConvArgs(T, B, D, weight.shape[0], _DTYPES[x.dtype], silu, x.data_ptr(), x.stride(0), x.stride(1), weight.data_ptr(),
                      _ptr(bias), _ptr(state), _ptr(lengths), _ptr(y), 0 if y is None else y.stride(0), 0 if y is None else y.stride(1),
                      _ptr(state_out), _ptr(dy), 0 if dy is None else dy.stride(0), 0 if dy is None else dy.stride(1),
                      _ptr(dstate_out), _ptr(dx), _ptr(dweight), _ptr(dbias), _ptr(dstate))


def _conv_forward(x, weight, bias, state, lengths, silu, want_state):
    T, B, D = x.shape
    y = torch.empty((T, B, D), dtype=x.dtype, device=x.device)
    last = torch.empty((weight.shape[0] - 1, B, D), dtype=x.dtype, device=x.device) if want_state else None
    _call(x.device, N.lib().shivae_causal_conv_fwd, byref(_conv_args(x, weight, bias, state, lengths, silu, y, last)))
    return y, last


def _conv_backward(x, weight, bias, state, lengths, silu, dy, dlast):
    dy = torch.zeros_like(x) if dy is None else _rows(dy)
    dlast = None if dlast is None else dlast.contiguous()
    dx, dw = torch.empty(x.shape, dtype=x.dtype, device=x.device), torch.empty_like(weight)
    db = None if bias is None else torch.empty_like(bias)
    ds = None if state is None else torch.empty_like(state)
    args = _conv_args(x, weight, bias, state, lengths, silu, None, None, dy, dlast, dx, dw, db, ds)
    L = N.lib()
    ws = torch.empty(L.shivae_causal_conv_bwd_ws(byref(args)), dtype=torch.uint8, device=x.device)
    _call(x.device, L.shivae_causal_conv_bwd, byref(args), ws.data_ptr(), ws.numel())
    return dx, dw, db, ds


class _CausalConv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, state, lengths, silu, want_state):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, weight, bias, state, lengths)
        ctx.silu = silu
        return _conv_forward(x, weight, bias, state, lengths, silu, want_state)

    @staticmethod
    def backward(ctx, dy, dlast):
        x, weight, bias, state, lengths = ctx.saved_tensors
        grads = _first_derivative(lambda: _conv_backward(x, weight, bias, state, lengths, ctx.silu, dy, dlast), x, weight, bias, state, dy, dlast)
        return (*grads, None, None, None)


def _conv_silu(activation):
    if activation not in (None, "silu"):
        raise ValueError("activation must be None or 'silu', not %r" % (activation,))
    return int(activation == "silu")


def _conv_params(weight, bias, D, device):
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2 or not 2 <= weight.shape[0] <= 4:
        raise ValueError("weight must be a [W, D] tensor with 2, 3 or 4 taps")
    return _param(weight, "weight", (weight.shape[0], D), device), _param(bias, "bias", (D,), device)


def causal_conv(x, weight, bias=None, activation=None, initial_state=None, lengths=None, return_state=False):
    """``y[t] = act(bias + sum_j weight[j] * x[t - W + 1 + j])`` per channel; differentiable.

    x [T, B, D]; weight [W, D] float32 with W = 2, 3 or 4, ``weight[W-1]`` meets the newest row; bias [D] float32;
    activation None or "silu"; initial_state [W-1, B, D] like x: the rows in front of x (None: zeros).
    Returns y, or (y, state) with the last W-1 rows of each sequence, which continue it in the next call."""
    x = _first(x, "x", 3)
    T, B, D = x.shape
    dev = x.device
    weight, bias = _conv_params(weight, bias, D, dev)
    state = _param(initial_state, "initial_state", (weight.shape[0] - 1, B, D), dev, x.dtype)
    lengths = _lengths(lengths, B, dev)
    silu, want = _conv_silu(activation), bool(return_state)
    if _wants_grad(x, weight, bias, state):
        y, last = _CausalConv.apply(x, weight, bias, state, lengths, silu, want)
    else:
        y, last = _conv_forward(x, weight, bias, state, lengths, silu, want)
    return (y, last) if want else y


def causal_conv_step(x, weight, bias=None, *, state, activation=None, state_out=None):
    """One row of :func:`causal_conv`: x [B, D] -> y [B, D].  ``state`` [W-1, B, D] moves on by the row, in place or into
    ``state_out``."""
    x = _first(x, "x", 2)
    B, D = x.shape
    dev = x.device
    weight, bias = _conv_params(weight, bias, D, dev)
    _activation(state, "state", (weight.shape[0] - 1, B, D), x.dtype, dev)
    out, state = _step_state(state, state_out), state.contiguous()
    _no_backward(x, weight, bias, state, out)
    y = torch.empty((B, D), dtype=x.dtype, device=dev)
    args = N.ConvArgs(1, B, D, weight.shape[0], _DTYPES[x.dtype], _conv_silu(activation), x.data_ptr(), 0, x.stride(0), weight.data_ptr(),
                      _ptr(bias), state.data_ptr(), None, y.data_ptr(), 0, D, out.data_ptr())
    _call(dev, N.lib().shivae_causal_conv_fwd, byref(args))
    increment_version(out)
    return y


# ------------------------------------------------------------------------------------------------ selective scan
def _scan_args(u, dt, z, Bm, Cm, A, D, dt_bias, state, lengths, softplus, y=None, state_out=None, ckpt=None, dy=None, dstate_out=None,
               du=None, ddt=None, dz=None, dB=None, dC=None, dA=None, dD=None, dbias=None, dstate=None):
    T, B, Dm = u.shape
    return N.SsmArgs(T, B, Dm, A.shape[0], Bm.shape[2], _DTYPES[u.dtype], softplus, u.data_ptr(), dt.data_ptr(), _ptr(z), u.stride(0),
                     u.stride(1), dt.stride(0), dt.stride(1), 0 if z is None else z.stride(0), 0 if z is None else z.stride(1),
                     Bm.data_ptr(), Cm.data_ptr(), Bm.stride(0), Bm.stride(1), Bm.stride(2), Cm.stride(0), Cm.stride(1), Cm.stride(2),
                     A.data_ptr(), _ptr(D), _ptr(dt_bias), _ptr(state), _ptr(lengths), _ptr(y), 0 if y is None else y.stride(0),
                     0 if y is None else y.stride(1), _ptr(state_out), _ptr(ckpt), _ptr(dy), 0 if dy is None else dy.stride(0),
                     0 if dy is None else dy.stride(1), _ptr(dstate_out), _ptr(du), _ptr(ddt), _ptr(dz), _ptr(dB), _ptr(dC), _ptr(dA),
                     _ptr(dD), _ptr(dbias), _ptr(dstate))


def _scan_forward(u, dt, A, Bm, Cm, D, z, dt_bias, state, lengths, softplus, want_state, keep):
    T, B, Dm = u.shape
    y = torch.empty((T, B, Dm), dtype=u.dtype, device=u.device)
    last = torch.empty((B, A.shape[0], Dm), dtype=torch.float32, device=u.device) if want_state else None
    ckpt = None
    if keep:  # the states in front of every 16th row, from which the backward pass runs the rows again
        ckpt = torch.empty((-(-T // N.SCAN_CKPT), B, A.shape[0], Dm), dtype=torch.float32, device=u.device)
    args = _scan_args(u, dt, z, Bm, Cm, A, D, dt_bias, state, lengths, softplus, y, last, ckpt)
    L = N.lib()
    n = L.shivae_selective_scan_fwd_ws(byref(args))
    ws = torch.empty(n, dtype=torch.uint8, device=u.device) if n else None
    _call(u.device, L.shivae_selective_scan_fwd, byref(args), _ptr(ws), n)
    return y, last, ckpt


def _scan_backward(u, dt, A, Bm, Cm, D, z, dt_bias, state, lengths, ckpt, softplus, dy, dlast):
    dy = torch.zeros_like(u) if dy is None else _rows(dy)
    dlast = None if dlast is None else dlast.contiguous()

    def like(t):
        return None if t is None else torch.empty(t.shape, dtype=t.dtype, device=t.device)

    du, ddt, dz, dB, dC, dA, dD, db, ds = (like(t) for t in (u, dt, z, Bm, Cm, A, D, dt_bias, state))
    args = _scan_args(u, dt, z, Bm, Cm, A, D, dt_bias, state, lengths, softplus, None, None, ckpt, dy, dlast, du, ddt, dz, dB, dC, dA, dD,
                      db, ds)
    L = N.lib()
    ws = torch.empty(L.shivae_selective_scan_bwd_ws(byref(args)), dtype=torch.uint8, device=u.device)
    _call(u.device, L.shivae_selective_scan_bwd, byref(args), ws.data_ptr(), ws.numel())
    return du, ddt, dA, dB, dC, dD, dz, db, ds


class _SelectiveScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, u, dt, A, Bm, Cm, D, z, dt_bias, state, lengths, softplus, want_state):
        ctx.set_materialize_grads(False)
        y, last, ckpt = _scan_forward(u, dt, A, Bm, Cm, D, z, dt_bias, state, lengths, softplus, want_state, True)
        ctx.save_for_backward(u, dt, A, Bm, Cm, D, z, dt_bias, state, lengths, ckpt)
        ctx.softplus = softplus
        return y, last

    @staticmethod
    def backward(ctx, dy, dlast):
        saved = ctx.saved_tensors
        grads = _first_derivative(lambda: _scan_backward(*saved, ctx.softplus, dy, dlast), *saved[:9], dy, dlast)
        return (*grads, None, None, None)


def _scan_inputs(u, dt, A, B, C_, D, z, dt_bias):
    """Checks what the sequence form and the step share; the leading axes are (T, B) or (B,)."""
    lead, Dm = tuple(u.shape[:-1]), u.shape[-1]
    dev, ty = u.device, u.dtype
    if not isinstance(A, torch.Tensor) or A.dim() != 2 or not 1 <= A.shape[0] <= 64:
        raise ValueError("A must be an [N, D] tensor with 1 to 64 states per channel")
    if not isinstance(B, torch.Tensor) or B.dim() != len(lead) + 2:
        raise ValueError("B must have the shape of its rows, then [groups, N]")
    G = B.shape[-2]
    if G < 1 or Dm % G:
        raise ValueError("%d groups do not divide %d channels" % (G, Dm))
    dt = _activation(dt, "dt", lead + (Dm,), ty, dev)
    A = _param(A, "A", (A.shape[0], Dm), dev)
    B = _activation(B, "B", lead + (G, A.shape[0]), ty, dev)
    C_ = _activation(C_, "C", lead + (G, A.shape[0]), ty, dev)
    z = None if z is None else _activation(z, "z", lead + (Dm,), ty, dev)
    return dt, A, B, C_, _param(D, "D", (Dm,), dev), z, _param(dt_bias, "dt_bias", (Dm,), dev)


def selective_scan(u, dt, A, B, C, D=None, z=None, dt_bias=None, softplus=True, initial_state=None, lengths=None, return_state=False):
    """Selective state-space scan, per channel d with its group g and states n; differentiable::

        s    = softplus(dt + dt_bias)                     (softplus=False: dt + dt_bias)
        h[n] = exp(s * A[n]) * h[n] + s * u * B[g, n]
        y    = (sum_n C[g, n] * h[n] + D * u) * silu(z)

    u, dt, z [T, B, D]; B, C [T, B, G, N], groups of D/G neighbouring channels; A [N, D], D and dt_bias [D] float32, N up to 64;
    initial_state [B, N, D] float32 (None: zeros).  Returns y, or (y, state) with the state behind each sequence's last row.
    An A of -inf keeps nothing of a state.  NaN stays NaN; what depends on an infinite u or dy is not finite, but may be NaN where the sum
    above, without the terms that are 0, is an infinity.
    With gradients the states in front of every 16th row are kept (4 N / 16 bytes per element of u) and the rows between are run
    again in the backward pass."""
    u = _first(u, "u", 3)
    T, Bt, Dm = u.shape
    dt, A, B, C, D, z, dt_bias = _scan_inputs(u, dt, A, B, C, D, z, dt_bias)
    state = _param(initial_state, "initial_state", (Bt, A.shape[0], Dm), u.device)
    lengths = _lengths(lengths, Bt, u.device)
    args = (u, dt, A, B, C, D, z, dt_bias, state, lengths, int(bool(softplus)), bool(return_state))
    y, last = _SelectiveScan.apply(*args) if _wants_grad(*args[:9]) else _scan_forward(*args, False)[:2]
    return (y, last) if return_state else y


def selective_scan_step(u, dt, A, B, C, state, D=None, z=None, dt_bias=None, softplus=True, state_out=None):
    """One row of :func:`selective_scan`: u, dt, z [Bt, D], B, C [Bt, G, N] -> y [Bt, D].  ``state`` [Bt, N, D] moves on by the row,
    in place or into ``state_out``."""
    u = _first(u, "u", 2)
    Bt, Dm = u.shape
    dev = u.device
    dt, A, B, C, D, z, dt_bias = _scan_inputs(u, dt, A, B, C, D, z, dt_bias)
    _activation(state, "state", (Bt, A.shape[0], Dm), torch.float32, dev)
    out, state = _step_state(state, state_out), state.contiguous()
    _no_backward(u, dt, A, B, C, D, z, dt_bias, state, out)
    y = torch.empty((Bt, Dm), dtype=u.dtype, device=dev)
    args = N.SsmArgs(1, Bt, Dm, A.shape[0], B.shape[1], _DTYPES[u.dtype], int(bool(softplus)), u.data_ptr(), dt.data_ptr(), _ptr(z), 0,
                     u.stride(0), 0, dt.stride(0), 0, 0 if z is None else z.stride(0), B.data_ptr(), C.data_ptr(), 0, B.stride(0),
                     B.stride(1), 0, C.stride(0), C.stride(1), A.data_ptr(), _ptr(D), _ptr(dt_bias), state.data_ptr(), None,
                     y.data_ptr(), 0, Dm, out.data_ptr())
    _call(dev, N.lib().shivae_selective_scan_fwd, byref(args), None, 0)
    increment_version(out)
    return y

