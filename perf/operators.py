"""The sequence operators and the sampler, measured: the causal convolution and the selective state-space scan
(prompts, training steps, single tokens) and drawing category indices from logits.

Layout everywhere: time-major ``[T, B, channels]``, channels last and contiguous, as in the recurrent scans; parameters,
recurrent states and their gradients are fp32.

  causal convolution  y[t,d] = act(bias[d] + sum_j weight[j,d] x[t-W+1+j, d]); rows before t = 0 come from the state
  selective scan      s = softplus(dt + dt_bias); h[n,d] = exp(s[d] A[n,d]) h[n,d] + s[d] u[d] B[g,n];
                      y[d] = (sum_n C[g,n] h[n,d] + D[d] u[d]) * silu(z[d]);  g = the channel's group
  sampling            kept = top_k largest (ties: lowest index), of these the smallest leading set that holds top_p of
                      their probability, of these weight >= min_p * largest; token = first index i with
                      (sum of kept weights up to i, in index order) > u * (sum of kept weights); temperature 0: arg max;
                      -1 where no logit is above -inf.  Beside it the token's log-probability among the kept
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # a batch of long prompts through the convolution in front of a scan: all traffic
        dict(name="conv_prompt_bf16", op="conv", T=2048, B=16, D=2048, W=4, dtype="bf16", silu=True, state=True, ragged=False),
        # a training step on sequences of unequal length, fp32, at the benchmark's T and width
        dict(name="conv_train_ragged_f32", op="conv_train", T=1000, B=64, D=256, W=4, dtype="f32", silu=True, state=False, ragged=True),
        # one token for each of many sequences: latency
        dict(name="conv_token_bf16", op="conv_token", T=1, B=256, D=2048, W=4, dtype="bf16", silu=True, state=True, ragged=False),
        # a batch of prompts: enough channels to fill the card
        dict(name="scan_prompt_bf16", op="scan", T=2048, B=16, D=2048, N=16, G=1, dtype="bf16", gate=True, state=True, ragged=False),
        # one long prompt: few channels, the time axis has to carry the parallel work
        dict(name="scan_long_one_bf16", op="scan", T=8192, B=1, D=2048, N=16, G=1, dtype="bf16", gate=True, state=False, ragged=False),
        # training steps: sequences of unequal length in fp32 at the benchmark's T and width; and bf16 with a gate
        dict(name="scan_train_ragged_f32", op="scan_train", T=1000, B=64, D=256, N=16, G=1, dtype="f32", gate=False, state=False, ragged=True),
        dict(name="scan_train_bf16", op="scan_train", T=2048, B=4, D=1536, N=16, G=1, dtype="bf16", gate=True, state=False, ragged=False),
        # one token for each of many sequences: the state's traffic
        dict(name="scan_token_bf16", op="scan_token", T=1, B=256, D=2048, N=16, G=1, dtype="bf16", gate=True, state=True, ragged=False),
        # a categorical attribute of the model, drawn for every (t, b): many rows, few categories
        dict(name="sample_attribute_f32", op="sample", rows=102400, V=8, dtype="f32", temperature=0.7, top_k=0, top_p=1.0, min_p=0.0, mixed=False, masked=0.0),
        # one token from a large vocabulary: latency
        dict(name="sample_one_bf16", op="sample", rows=1, V=32768, dtype="bf16", temperature=0.8, top_k=50, top_p=0.9, min_p=0.0, mixed=False, masked=0.0),
        # a batch of tokens from a very large vocabulary, nucleus and min-p
        dict(name="sample_batch_bf16", op="sample", rows=256, V=131072, dtype="bf16", temperature=1.0, top_k=0, top_p=0.95, min_p=0.01, mixed=False, masked=0.0),
        # every request its own settings, odd vocabulary, part of it masked out
        dict(name="sample_mixed_f32", op="sample", rows=37, V=50001, dtype="f32", temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, mixed=True, masked=0.5),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def _shrink(rng, case, sizes):
    """Halve a size at random until the case costs no more than the largest listed ones of its operator."""
    like = [work(c) for c in listed() if c["op"] == case["op"]]
    most = {k: max(w[k] for w in like) for k in ("bytes", "flops")}
    while any(work(case)[k] > most[k] for k in most):
        name = rng.choice([k for k in sizes if case[k] > (case.get("G", 1) if k == "D" else 2 if k == "V" else 1)])
        case[name] = (case[name] + 1) // 2
        if name == "D" and "G" in case:
            case["D"] = -(-case["D"] // case["G"]) * case["G"]
    return case


def draw(rng):
    op = rng.choice(["conv", "conv_train", "conv_token", "scan", "scan_train", "scan_token", "sample", "sample"])
    dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
    if op == "sample":
        return _shrink(rng, dict(op=op, rows=_log_int(rng, 1, 100000), V=_log_int(rng, 2, 131072), dtype=dtype,
                                 temperature=rng.choice([0.0, 0.5, 0.8, 1.0, 1.5]), top_k=rng.choice([0, 0, 1, 40, 200, 3000]),
                                 top_p=rng.choice([1.0, 0.5, 0.9, 0.95]), min_p=rng.choice([0.0, 0.0, 0.05]),
                                 mixed=rng.random() < 0.3, masked=rng.choice([0.0, 0.0, 0.3])), ["rows", "V"])
    token, train = op.endswith("token"), op.endswith("train")
    out = dict(op=op, dtype=dtype, T=1 if token else _log_int(rng, 1, 2048 if train else 8192),
               B=_log_int(rng, 1, 512 if token else 64), D=_log_int(rng, 1, 4096), state=token or rng.random() < 0.5,
               ragged=not token and rng.random() < 0.4)
    if op.startswith("conv"):
        out.update(W=rng.choice([2, 3, 4]), silu=rng.random() < 0.8)
    else:
        G = rng.choice([1, 1, 2, 4])
        out.update(N=rng.choice([16, 16, 8, 32, 64, _log_int(rng, 1, 64)]), G=G, D=-(-out["D"] // G) * G, gate=rng.random() < 0.6)
    return _shrink(rng, out, ["T", "B", "D"])


def work(case):
    if case["op"] == "sample":
        n = case["rows"] * case["V"]
        return {"bytes": n * DTYPES[case["dtype"]].itemsize + case["rows"] * 16, "flops": 4 * n}
    es = DTYPES[case["dtype"]].itemsize
    rows = case["B"] * case["T"]
    n = rows * case["D"]
    train = case["op"].endswith("train")
    if case["op"].startswith("conv"):
        taps = case["W"] - 1
        state = taps * case["B"] * case["D"] * es
        params = (case["W"] + 1) * case["D"] * 4
        if train:  # read x, dy; write y, dx, dweight, dbias
            return {"bytes": 4 * n * es + 2 * params + (2 * state if case["state"] else 0), "flops": (6 * case["W"] + 12) * n}
        return {"bytes": 2 * n * es + params + (2 if case["state"] else 1) * state, "flops": (2 * case["W"] + 4) * n}
    N, G, gate = case["N"], case["G"], int(case["gate"])
    state = case["B"] * N * case["D"] * 4
    params = (N + 2) * case["D"] * 4
    io = (3 + gate) * n * es + 2 * rows * G * N * es  # u, dt, (z), y; B, C
    if train:  # and dy, du, ddt, (dz), dB, dC, the parameters' gradients
        io += (3 + gate) * n * es + 2 * rows * G * N * es
        return {"bytes": io + 2 * params + (2 * state if case["state"] else 0), "flops": 26 * n * N}
    return {"bytes": io + params + (2 if case["state"] else 1) * state, "flops": 7 * n * N}


# ------------------------------------------------------------------------------------------------ inputs
def _lengths(gen, case, dev):
    """Unequal lengths, from an empty sequence to the whole T."""
    if not case["ragged"]:
        return None
    n = torch.randint(0, case["T"] + 1, (case["B"],), generator=gen, device=dev, dtype=torch.int32)
    n[0] = case["T"]
    return n


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(int(seed))

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    s = dict(case=dict(case))
    dt = DTYPES[case["dtype"]]
    if case["op"] == "sample":
        rows, V = case["rows"], case["V"]
        lg = randn(rows, V) * 2.5
        if case["masked"] > 0.0:  # a mask of disallowed categories; the last row allows none
            m = torch.rand(rows, V, generator=gen, device=dev) < case["masked"]
            lg = lg.masked_fill(m, -math.inf)
            if rows > 1:
                lg[-1] = -math.inf
        s["logits"] = lg.to(dt)
        s["u"] = torch.rand(rows, generator=gen, device=dev)
        if case["mixed"]:  # every row its own settings
            def pick(values, t):
                i = torch.randint(0, len(values), (rows,), generator=gen, device=dev)
                return torch.tensor(values, dtype=t, device=dev)[i]
            s.update(temperature=pick([0.0, 0.5, 0.8, 1.0, 1.3], torch.float32), top_k=pick([0, 1, 20, 100, 2000], torch.int32),
                     top_p=pick([0.3, 0.9, 0.98, 1.0], torch.float32), min_p=pick([0.0, 0.02, 0.1], torch.float32))
        else:
            s.update(temperature=case["temperature"], top_k=case["top_k"], top_p=case["top_p"], min_p=case["min_p"])
        return s
    T, B, D = case["T"], case["B"], case["D"]
    train, token = case["op"].endswith("train"), case["op"].endswith("token")
    lead = (B,) if token else (T, B)
    s["lengths"] = None if token else _lengths(gen, case, dev)
    if case["op"].startswith("conv"):
        W = case["W"]
        s.update(x=randn(*lead, D).to(dt), weight=randn(W, D) / math.sqrt(W), bias=randn(D) * 0.2,
                 state=randn(W - 1, B, D).to(dt) if case["state"] else None)
        if token:
            s["next"] = torch.empty_like(s["state"])
        names = ["x", "weight", "bias"] + (["state"] if case["state"] else [])
    else:
        N, G = case["N"], case["G"]
        s.update(u=randn(*lead, D).to(dt), dt=randn(*lead, D).to(dt), B=randn(*lead, G, N).to(dt), C=randn(*lead, G, N).to(dt))
        s["A"] = -torch.exp(torch.log(torch.arange(1, N + 1, device=dev, dtype=torch.float32))[:, None] + 0.1 * randn(N, D))
        s["D"] = 1 + 0.1 * randn(D)
        step = torch.exp(math.log(1e-3) + math.log(100.0) * torch.rand(D, generator=gen, device=dev))  # 1e-3 .. 1e-1
        s["dt_bias"] = step + torch.log(-torch.expm1(-step))
        s["z"] = randn(*lead, D).to(dt) if case["gate"] else None
        s["state"] = randn(B, N, D) if case["state"] else None
        if token:
            s["next"] = torch.empty_like(s["state"])
        names = ["u", "dt", "A", "B", "C", "D", "dt_bias"] + (["z"] if case["gate"] else []) + (["state"] if case["state"] else [])
    if train:
        s["dy"] = randn(T, B, D).to(dt)
        s["leaves"] = names
        for k in names:
            s[k].requires_grad_(True)
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    import shivae_amd
    c = s["case"]
    op = c["op"]
    if op == "sample":
        return list(shivae_amd.sample_categories(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                                                 min_p=s["min_p"], return_logprob=True))
    if op.startswith("conv"):
        act = "silu" if c["silu"] else None
        if op == "conv_token":
            y = shivae_amd.causal_conv_step(s["x"], s["weight"], s["bias"], state=s["state"], activation=act, state_out=s["next"])
            return [y, s["next"]]
        if op == "conv":
            return list(shivae_amd.causal_conv(s["x"], s["weight"], s["bias"], activation=act, initial_state=s["state"],
                                               lengths=s["lengths"], return_state=True))
        y = shivae_amd.causal_conv(s["x"], s["weight"], s["bias"], activation=act, initial_state=s["state"], lengths=s["lengths"])
    else:
        p = dict(D=s["D"], z=s["z"], dt_bias=s["dt_bias"], softplus=True)
        if op == "scan_token":
            y = shivae_amd.selective_scan_step(s["u"], s["dt"], s["A"], s["B"], s["C"], s["state"], state_out=s["next"], **p)
            return [y, s["next"]]
        p.update(initial_state=s["state"], lengths=s["lengths"])
        if op == "scan":
            return list(shivae_amd.selective_scan(s["u"], s["dt"], s["A"], s["B"], s["C"], return_state=True, **p))
        y = shivae_amd.selective_scan(s["u"], s["dt"], s["A"], s["B"], s["C"], **p)
    return [y.detach()] + list(torch.autograd.grad(y, [s[k] for k in s["leaves"]], s["dy"]))


@torch.no_grad()
def _run_plain(s):
    op = s["case"]["op"]
    if op == "sample":
        return _plain_sample(s)
    return _plain_conv(s) if op.startswith("conv") else _plain_scan(s)


def _alive(T, lengths, dev):
    """[T, B, 1]: the rows inside their sequence."""
    return torch.arange(T, device=dev)[:, None, None] < lengths[None, :, None]


def _plain_conv(s):
    c = s["case"]
    token = c["op"] == "conv_token"
    x = (s["x"][None] if token else s["x"]).float()
    T, B, D = x.shape
    W, w, dt = c["W"], s["weight"], s["x"].dtype
    alive = None if s["lengths"] is None else _alive(T, s["lengths"], x.device)
    if alive is not None:
        x = torch.where(alive, x, torch.zeros_like(x))
    before = torch.zeros(W - 1, B, D, device=x.device) if s["state"] is None else s["state"].float()
    xs = torch.cat([before, x])
    pre = s["bias"] + sum(w[j] * xs[j:j + T] for j in range(W))
    sig = torch.sigmoid(pre)
    y = pre * sig if c["silu"] else pre
    if alive is not None:
        y = torch.where(alive, y, torch.zeros_like(y))
    if c["op"] != "conv_train":
        n = torch.full((B,), T, device=x.device) if s["lengths"] is None else s["lengths"].long()
        at = n[None, :] + torch.arange(W - 1, device=x.device)[:, None]
        last = torch.gather(xs, 0, at[:, :, None].expand(W - 1, B, D)).to(dt)
        return [y[0].to(dt) if token else y.to(dt), last]
    g = s["dy"].float()
    if c["silu"]:
        g = g * (sig + pre * sig * (1 - sig))
    if alive is not None:
        g = torch.where(alive, g, torch.zeros_like(g))
    dxs = torch.zeros_like(xs)
    for j in range(W):
        dxs[j:j + T] += w[j] * g
    g64 = g.double()
    dw = torch.stack([(g64 * xs[j:j + T]).sum((0, 1)) for j in range(W)]).float()
    dx = dxs[W - 1:]
    if alive is not None:
        dx = torch.where(alive, dx, torch.zeros_like(dx))
    out = [y.to(dt), dx.to(dt), dw, g64.sum((0, 1)).float()]
    if s["state"] is not None:
        out.append(dxs[:W - 1].to(dt))
    return out


def _plain_scan(s):
    c = s["case"]
    token = c["op"] == "scan_token"
    u, raw, Bm, Cm = ((s[k][None] if token else s[k]).float() for k in ("u", "dt", "B", "C"))
    T, B, D = u.shape
    N, G, dtype = c["N"], c["G"], s["u"].dtype
    E = D // G  # channels of a group; below they are a dimension of their own
    z = None if s["z"] is None else (s["z"][None] if token else s["z"]).float()
    raw = raw + s["dt_bias"]
    step = torch.clamp(raw, min=0) + torch.log1p(torch.exp(-raw.abs()))
    if s["lengths"] is not None:
        alive = _alive(T, s["lengths"], u.device)
        step, u = (torch.where(alive, v, torch.zeros_like(v)) for v in (step, u))
        Bm, Cm = (torch.where(alive[..., None], v, torch.zeros_like(v)) for v in (Bm, Cm))
    A = s["A"].view(N, G, E)
    h = torch.zeros(B, N, G, E, device=u.device) if s["state"] is None else s["state"].clone().view(B, N, G, E)
    step, u = step.view(T, B, 1, G, E), u.view(T, B, 1, G, E)
    Bn, Cn = (v.transpose(2, 3).unsqueeze(-1) for v in (Bm, Cm))  # [T, B, N, G, 1]
    train = c["op"] == "scan_train"
    y = torch.empty(T, B, D, device=u.device)
    hs = torch.empty(T + 1, B, N, G, E, device=u.device) if train else None
    if train:
        hs[0] = h
    for t in range(T):
        h = torch.exp(step[t] * A) * h + step[t] * u[t] * Bn[t]
        y[t] = (Cn[t] * h).sum(1).view(B, D)
        if train:
            hs[t + 1] = h
    flat = u.reshape(T, B, D)
    y = y + s["D"] * flat
    sig = None if z is None else torch.sigmoid(z)
    out = y if z is None else y * z * sig
    if s["lengths"] is not None:
        out = torch.where(alive, out, torch.zeros_like(out))
    if not train:
        return [out[0].to(dtype) if token else out.to(dtype), h.reshape(B, N, D)]
    dy = s["dy"].float()
    if s["lengths"] is not None:
        dy = torch.where(alive, dy, torch.zeros_like(dy))
    dz = None
    if z is not None:
        dz = dy * y * (sig + z * sig * (1 - sig))
        dy = dy * z * sig
        if s["lengths"] is not None:
            dz = torch.where(alive, dz, torch.zeros_like(dz))
    dyg = dy.view(T, B, 1, G, E)
    dA = torch.zeros(N, G, E, device=u.device, dtype=torch.float64)
    dB, dC = torch.empty(T, B, G, N, device=u.device), torch.empty(T, B, G, N, device=u.device)
    du, ds = torch.empty_like(dy), torch.empty_like(dy)
    gh = torch.zeros_like(h)  # the loss's gradient with respect to h[t]
    for t in range(T - 1, -1, -1):
        dC[t] = (dyg[t] * hs[t + 1]).sum(-1).transpose(1, 2)
        gh = gh + Cn[t] * dyg[t]
        dB[t] = (gh * (step[t] * u[t])).sum(-1).transpose(1, 2)
        gb = (gh * Bn[t]).sum(1)
        a = torch.exp(step[t] * A)
        gh = gh * a
        q = gh * hs[t]
        du[t] = (step[t][:, 0] * gb).view(B, D)
        ds[t] = ((q * A).sum(1) + u[t][:, 0] * gb).view(B, D)
        dA += (q * step[t]).double().sum(0)
    du = du + s["D"] * dy
    draw_ = ds * torch.sigmoid(raw)
    if s["lengths"] is not None:
        draw_ = torch.where(alive, draw_, torch.zeros_like(draw_))
    out = [out.to(dtype), du.to(dtype), draw_.to(dtype), dA.float().view(N, D), dB.to(dtype), dC.to(dtype),
           (dy.double() * flat).sum((0, 1)).float(), draw_.double().sum((0, 1)).float()]
    if z is not None:
        out.append(dz.to(dtype))
    if s["state"] is not None:
        out.append(gh.reshape(B, N, D))
    return out


def _plain_sample(s):
    lg = s["logits"].double()
    lg = torch.where(torch.isnan(lg), torch.full_like(lg, -math.inf), lg)
    rows, V = lg.shape

    def column(v, dtype):
        return v.to(dtype)[:, None] if torch.is_tensor(v) else torch.full((rows, 1), v, dtype=dtype, device=lg.device)

    temp, p, mp = (column(s[k], torch.float32).double() for k in ("temperature", "top_p", "min_p"))
    k = column(s["top_k"], torch.long)
    k = torch.where((k <= 0) | (k > V), torch.full_like(k, V), k)
    val, idx = torch.sort(lg, dim=1, descending=True, stable=True)
    top = val[:, :1]
    w = torch.exp(torch.where(val == top, torch.zeros_like(val), (val - top) / torch.where(temp > 0, temp, torch.ones_like(temp))))
    keep = torch.arange(V, device=lg.device)[None, :] < k
    w = torch.where(keep, w, torch.zeros_like(w))
    cum = torch.cumsum(w, 1)
    keep &= (cum - w < p * cum[:, -1:]) | (p >= 1)
    keep &= w >= mp
    w = torch.zeros_like(w).scatter_(1, idx, torch.where(keep, w, torch.zeros_like(w)))
    cum = torch.cumsum(w, 1)
    tok = torch.searchsorted(cum, (s["u"].double()[:, None] * cum[:, -1:]).contiguous(), right=True)
    tok = torch.where(temp > 0, tok, idx[:, :1])
    logp = torch.log(torch.gather(w, 1, tok.clamp(max=V - 1)) / cum[:, -1:])
    logp = torch.where(temp > 0, logp, torch.zeros_like(logp))
    none = top == -math.inf
    return [torch.where(none, torch.full_like(tok, -1), tok)[:, 0], torch.where(none, torch.full_like(logp, -math.inf), logp)[:, 0].float()]


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "sample":
        return _exact_sample(s)
    v = {k: (t.detach().double() if torch.is_tensor(t) and t.is_floating_point() else t) for k, t in s.items()}
    f = _exact_conv if case["op"].startswith("conv") else _exact_scan
    if not case["op"].endswith("train"):
        return f(case, v)
    for k in s["leaves"]:
        v[k].requires_grad_(True)
    y = f(case, v)[0]
    return [y.detach()] + list(torch.autograd.grad(y, [v[k] for k in s["leaves"]], v["dy"]))


def _exact_conv(case, v):
    """Row by row, from a window of the last W rows."""
    token = case["op"] == "conv_token"
    x = v["x"][None] if token else v["x"]
    T, B, D = x.shape
    W = case["W"]
    window = [torch.zeros(B, D, dtype=torch.float64, device=x.device)] * (W - 1) if v["state"] is None else list(v["state"].unbind(0))
    n = torch.full((B,), T, device=x.device) if v["lengths"] is None else v["lengths"]
    ys = []
    for t in range(T):
        live = (t < n)[:, None]
        rows = window + [x[t]]
        pre = v["bias"].expand(B, D)
        for j in range(W):
            pre = pre + v["weight"][j] * rows[j]
        y = torch.nn.functional.silu(pre) if case["silu"] else pre
        ys.append(torch.where(live, y, torch.zeros_like(y)))
        window = [torch.where(live, a, b) for a, b in zip(rows[1:], window)]
    y = torch.stack(ys)
    return [y[0] if token else y, torch.stack(window)]


def _exact_scan(case, v):
    """One state at a time, carried over t; a channel reads its group's column."""
    token = case["op"] == "scan_token"
    u, dt, Bm, Cm = ((v[k][None] if token else v[k]) for k in ("u", "dt", "B", "C"))
    T, B, D = u.shape
    N = case["N"]
    group = torch.arange(D, device=u.device) // (D // case["G"])
    h = torch.zeros(B, N, D, dtype=torch.float64, device=u.device) if v["state"] is None else v["state"]
    n = torch.full((B,), T, device=u.device) if v["lengths"] is None else v["lengths"]
    ys = []
    for t in range(T):
        live = (t < n)[:, None]
        delta = torch.nn.functional.softplus(dt[t] + v["dt_bias"], threshold=200.0)
        new = torch.exp(delta[:, None, :] * v["A"]) * h + (delta * u[t])[:, None, :] * Bm[t].transpose(1, 2)[:, :, group]
        y = torch.einsum("bnd,bnd->bd", Cm[t].transpose(1, 2)[:, :, group], new) + v["D"] * u[t]
        if v["z"] is not None:
            y = y * torch.nn.functional.silu(v["z"] if token else v["z"][t])
        ys.append(torch.where(live, y, torch.zeros_like(y)))
        h = torch.where(live[:, None], new, h)
    y = torch.stack(ys)
    return [y[0] if token else y, h]


def _exact_sample(s):
    """On the host, from ranks: rank r of an element in (value descending, index ascending) order."""
    lg = s["logits"].double().cpu().numpy()
    lg = np.where(np.isnan(lg), -np.inf, lg)
    rows, V = lg.shape
    u = s["u"].cpu().numpy().astype(np.float64)

    def each(v):
        return v.cpu().numpy().astype(np.float64) if torch.is_tensor(v) else np.full(rows, np.float64(np.float32(v)))

    temp, p, mp = each(s["temperature"]), each(s["top_p"]), each(s["min_p"])
    kk = s["top_k"].cpu().numpy().astype(np.int64) if torch.is_tensor(s["top_k"]) else np.full(rows, int(s["top_k"]))
    tok, logp = np.empty(rows, np.int64), np.empty(rows)
    for r0 in range(0, rows, 4096):
        r1 = min(rows, r0 + 4096)
        x = lg[r0:r1]
        order = np.argsort(-x, axis=1, kind="stable")
        top = np.take_along_axis(x, order[:, :1], 1)
        t = np.where(temp[r0:r1] > 0, temp[r0:r1], 1.0)[:, None]
        with np.errstate(invalid="ignore"):
            w = np.where(x == top, 1.0, np.exp((x - top) / t))
        rank = np.empty_like(order)
        np.put_along_axis(rank, order, np.broadcast_to(np.arange(V), order.shape), 1)
        k = kk[r0:r1, None]
        keep = (rank < k) | (k <= 0)
        ws = np.take_along_axis(np.where(keep, w, 0.0), order, 1)
        before = np.concatenate([np.zeros((r1 - r0, 1)), np.cumsum(ws, 1)], 1)
        nucleus = (before[:, :-1] < p[r0:r1, None] * before[:, -1:]) | (p[r0:r1, None] >= 1)
        keep &= np.take_along_axis(nucleus, rank, 1)
        keep &= w >= mp[r0:r1, None]
        cum = np.cumsum(np.where(keep, w, 0.0), 1)
        at = np.minimum((cum <= u[r0:r1, None] * cum[:, -1:]).sum(1), V - 1)
        at = np.where(temp[r0:r1] > 0, at, order[:, 0])
        got = np.take_along_axis(x, at[:, None], 1)
        with np.errstate(invalid="ignore"):
            lp = np.where(got == top, 0.0, (got - top) / t)[:, 0] - np.log(cum[:, -1])
        none = top[:, 0] == -np.inf
        tok[r0:r1] = np.where(none, -1, at)
        logp[r0:r1] = np.where(none, -np.inf, np.where(temp[r0:r1] > 0, lp, 0.0))
    return [torch.from_numpy(tok), torch.from_numpy(logp)]
