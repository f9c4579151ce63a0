"""The sequence operators and the sampler in 64 bits, straight from their formulas (numpy), with hand-derived gradients, and
for every result a `scale`: the same sums over absolute values, which is what rounding errors are relative to."""
import numpy as np


def silu(v):
    return v / (1 + np.exp(-v))


def dsilu(v):
    s = 1 / (1 + np.exp(-v))
    return s + v * s * (1 - s)


def dsilu_scale(v):
    """silu' = s + v s (1 - s) is itself a sum, and its terms cancel at v = -1.278: each carries its own rounding error, a
    few units of |term|, so an error of silu' is relative to s + |v| s (1 - s), not to |silu'|, which is 0 there."""
    s = 1 / (1 + np.exp(-v))
    return s + np.abs(v) * s * (1 - s)


def softplus(v):
    return np.maximum(v, 0) + np.log1p(np.exp(-np.abs(v)))


def clamp_lengths(lengths, T, B):
    return np.full(B, T) if lengths is None else np.clip(np.asarray(lengths), 0, T)


def conv(x, w, bias, state, lengths, act):
    """-> y [T,B,D], last [W-1,B,D], and the arrays the gradient needs."""
    T, B, D = x.shape
    W = w.shape[0]
    n = clamp_lengths(lengths, T, B)
    live = np.arange(T)[:, None, None] < n[None, :, None]
    x = np.where(live, x, 0.0)
    st = np.zeros((W - 1, B, D)) if state is None else state
    xs = np.concatenate([st, x])
    b = np.zeros(D) if bias is None else bias
    pre = b + sum(w[j] * xs[j:j + T] for j in range(W))
    mag = np.abs(b) + sum(np.abs(w[j] * xs[j:j + T]) for j in range(W))
    y = np.where(live, silu(pre) if act else pre, 0.0)
    last = np.stack([np.stack([xs[n[i] + j, i] for i in range(B)]) for j in range(W - 1)])
    return y, last, dict(xs=xs, pre=pre, mag=mag, live=live, n=n)


def conv_grad(x, w, bias, state, lengths, act, dy, dlast=None):
    """-> dict of gradients and dict of scales."""
    T, B, D = x.shape
    W = w.shape[0]
    _, _, c = conv(x, w, bias, state, lengths, act)
    out, scale = {}, {}
    for d, absolute in ((out, False), (scale, True)):
        f = np.abs if absolute else (lambda v: v)
        g = np.where(c["live"], f(np.where(c["live"], dy, 0.0)) * ((dsilu_scale(c["pre"]) + 0.5 * c["mag"] if absolute else dsilu(c["pre"])) if act else 1.0), 0.0)
        dxs = np.zeros_like(c["xs"])
        for j in range(W):
            dxs[j:j + T] += f(w[j]) * g
        if dlast is not None:
            for i in range(B):
                for j in range(W - 1):
                    dxs[c["n"][i] + j, i] += f(dlast[j, i])
        d["x"] = np.where(c["live"], dxs[W - 1:], 0.0)
        d["state"] = dxs[:W - 1]
        d["weight"] = np.stack([(g * f(c["xs"][j:j + T])).sum((0, 1)) for j in range(W)])
        d["bias"] = g.sum((0, 1))
    return out, scale


def scan(u, dt, A, Bm, Cm, D, z, dt_bias, state, lengths, use_softplus, dy=None, dlast=None):
    """u, dt, z [T,B,D], Bm, Cm [T,B,G,N], A [N,D] -> (results, scales): y, last and, with dy, the gradients by input name."""
    T, B, Dm = u.shape
    N, G = A.shape[0], Bm.shape[2]
    grp = np.arange(Dm) // (Dm // G)
    n = clamp_lengths(lengths, T, B)
    live = np.arange(T)[:, None] < n[None, :]
    m3, m4 = live[..., None], live[..., None, None]
    raw = np.where(m3, dt, 0.0) + (0.0 if dt_bias is None else dt_bias)
    s = np.where(m3, softplus(raw) if use_softplus else raw, 0.0)
    slope = 1 / (1 + np.exp(-raw)) if use_softplus else np.ones_like(raw)
    u, Bm, Cm = np.where(m3, u, 0.0), np.where(m4, Bm, 0.0), np.where(m4, Cm, 0.0)
    zz = None if z is None else np.where(m3, z, 0.0)
    gate = np.ones_like(u) if z is None else silu(zz)
    dyl = None if dy is None else np.where(m3, dy, 0.0)
    Dv = np.zeros(Dm) if D is None else D
    out, scale = {}, {}
    for r, absolute in ((out, False), (scale, True)):
        f = np.abs if absolute else (lambda v: v)
        U, Bx, Cx = f(u), f(Bm)[:, :, grp, :].transpose(0, 1, 3, 2), f(Cm)[:, :, grp, :].transpose(0, 1, 3, 2)  # [T,B,N,D]
        S = f(s)
        h = np.zeros((B, N, Dm)) if state is None else f(state)
        hs, y = [h], np.zeros_like(u)
        for t in range(T):
            h = np.exp(s[t][:, None] * A) * h + (S[t] * U[t])[:, None] * Bx[t]
            hs.append(h)
            y[t] = (Cx[t] * h).sum(1) + f(Dv) * U[t]
        gt = f(gate)
        r["y"], r["last"] = np.where(m3, y * gt, 0.0), h
        if dy is None:
            continue
        g = np.zeros_like(h) if dlast is None else f(dlast)
        gy = f(dyl) * gt
        if z is not None:
            r["z"] = np.where(m3, f(dyl) * y * (dsilu_scale(zz) if absolute else dsilu(zz)), 0.0)
        r["D"] = (gy * U).sum((0, 1))
        du, ds, dA = np.zeros_like(u), np.zeros_like(u), np.zeros_like(A)
        dB, dC = np.zeros((T, B, G, N)), np.zeros((T, B, G, N))
        for t in range(T - 1, -1, -1):
            vC = gy[t][:, None] * hs[t + 1]
            g = g + Cx[t] * gy[t][:, None]
            vB = g * (S[t] * U[t])[:, None]
            for k in range(G):
                dB[t, :, k], dC[t, :, k] = vB[:, :, grp == k].sum(2), vC[:, :, grp == k].sum(2)
            gb = (g * Bx[t]).sum(1)
            g = g * np.exp(s[t][:, None] * A)
            q = g * hs[t]
            ds[t] = (q * f(A)).sum(1) + U[t] * gb
            du[t] = S[t] * gb + f(Dv) * gy[t]
            dA += (q * S[t][:, None]).sum(0)
        r["u"], r["dt"] = np.where(m3, du, 0.0), np.where(m3, ds * slope, 0.0)
        r["A"], r["B"], r["C"], r["state"] = dA, dB, dC, g
        r["dt_bias"] = r["dt"].sum((0, 1))
    return out, scale


def sample(logits, u, temperature, top_k, top_p, min_p):
    """One row at a time, on sorted pairs -> (token, log-probability) per row."""
    rows, V = logits.shape
    each = [np.broadcast_to(np.asarray(v, dtype=np.float64), (rows,)) for v in (temperature, top_k, top_p, min_p)]
    tok, logp = np.empty(rows, np.int64), np.empty(rows)
    for r in range(rows):
        t, k, p, m = (a[r] for a in each)
        x = np.where(np.isnan(logits[r]), -np.inf, logits[r].astype(np.float64))
        top = x.max()
        if top == -np.inf:
            tok[r], logp[r] = -1, -np.inf
            continue
        order = sorted(range(V), key=lambda i: (-x[i], i))
        if t <= 0:
            tok[r], logp[r] = order[0], 0.0
            continue
        w = np.array([1.0 if x[i] == top else np.exp((x[i] - top) / t) for i in range(V)])
        kept = order if k <= 0 else order[:int(k)]
        if p < 1:
            total, run, lead = sum(w[i] for i in kept), 0.0, []
            for i in kept:
                if not lead or run < p * total:
                    lead.append(i)
                run += w[i]
            kept = lead
        kept = sorted(i for i in kept if w[i] >= min(m, 1))
        total = sum(w[i] for i in kept)
        goal, run = float(u[r]) * total, 0.0
        for i in kept:
            run += w[i]
            if run > goal:
                break
        tok[r], logp[r] = i, np.log(w[i] / total)
    return tok, logp
