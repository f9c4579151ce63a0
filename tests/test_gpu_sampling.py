"""Drawing categories (csrc/sample.hip) against the definition, row by row in 64 bits (_seq_ref.sample): indices equal, the
log-probability within half a step of fp32 and what 2^-43 of the largest weight, per category, changes in the sum."""
import numpy as np
import pytest
import torch

import _seq_ref as ref
import shivae_amd

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _check(logits, u, **kw):
    tok, logp = shivae_amd.sample_categories(logits, u, return_logprob=True, **kw)
    V = logits.shape[-1]
    a = {k: (v.cpu().numpy().reshape(-1) if torch.is_tensor(v) else np.float32(v) if k != "top_k" else v) for k, v in kw.items()}
    full = dict(temperature=np.float32(1.0), top_k=0, top_p=np.float32(1.0), min_p=np.float32(0.0))
    full.update(a)
    wt, wl = ref.sample(logits.double().cpu().numpy().reshape(-1, V), u.double().cpu().numpy().reshape(-1), **full)
    got, gl = tok.cpu().numpy().reshape(-1), logp.double().cpu().numpy().reshape(-1)
    np.testing.assert_array_equal(got, wt)
    none = wt < 0
    assert np.all(np.isneginf(gl[none]))
    assert np.all(np.abs(gl - wl)[~none] <= 2.0 ** -24 * np.abs(wl[~none]) + V * 2.0 ** -43 + 2.0 ** -45)
    return tok


def _logits(gen, rows, V, dtype, spread=2.0):
    return (torch.randn(rows, V, device="cuda", generator=gen) * spread).to(TYPES[dtype])


SETTINGS = [dict(), dict(temperature=0.0), dict(temperature=0.6), dict(top_k=1), dict(top_k=7), dict(top_p=0.8), dict(top_p=0.0),
            dict(min_p=0.1), dict(min_p=1.0), dict(temperature=1.7, top_k=40, top_p=0.9, min_p=0.02), dict(top_k=300, top_p=0.97)]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("V", [1, 2, 3, 8, 17, 63, 64, 65, 200, 511, 513, 2048, 2051, 5003, 16385, 30011])
def test_settings_and_sizes(V, dtype):
    gen = torch.Generator(device="cuda").manual_seed(V)
    rows = 9 if V < 3000 else 3
    for i, kw in enumerate(SETTINGS):
        u = torch.rand(rows, device="cuda", generator=gen)
        u[0] = 0.0
        u[-1] = 1.0 - 2.0 ** -24
        _check(_logits(gen, rows, V, dtype), u, **kw)


@pytest.mark.parametrize("V", [5, 40, 300, 3001, 20000])
def test_settings_for_each_row(V):
    gen = torch.Generator(device="cuda").manual_seed(7)
    rows = 24

    def pick(values, dtype):
        return torch.tensor(values, dtype=dtype, device="cuda")[torch.randint(0, len(values), (rows,), device="cuda", generator=gen)]

    kw = dict(temperature=pick([0.0, 0.3, 1.0, 2.0], torch.float32), top_k=pick([-1, 0, 1, 5, 1000, 10 ** 9], torch.int64),
              top_p=pick([0.1, 0.9, 0.999, 1.0], torch.float32), min_p=pick([0.0, 0.05, 0.5], torch.float32))
    _check(_logits(gen, rows, V, "bf16"), torch.rand(rows, device="cuda", generator=gen), **kw)


@pytest.mark.parametrize("V", [6, 64, 100, 700, 4099, 9000, 20001])
def test_runs_of_equal_logits(V):
    """Ties go to the lowest index, also where a run of equal values is longer than any list."""
    gen = torch.Generator(device="cuda").manual_seed(V)
    flat = torch.zeros(4, V, device="cuda")
    steps = torch.randint(0, 3, (4, V), device="cuda", generator=gen).float() * 0.01  # three values, all in one bin or two
    signed = torch.where(torch.rand(4, V, device="cuda", generator=gen) < 0.5, -0.0, 0.0)
    few = torch.full((4, V), -50.0, device="cuda")
    few[:, ::3] = 1.0
    for lg in (flat, steps, signed, few):
        for kw in (dict(), dict(temperature=0.0), dict(top_k=3), dict(top_k=V // 2 + 1), dict(top_p=0.37), dict(top_k=V // 2 + 1, top_p=0.5),
                   dict(top_k=max(1, V - 1), top_p=0.99, min_p=0.9)):
            _check(lg.bfloat16(), torch.rand(4, device="cuda", generator=gen), **kw)


@pytest.mark.parametrize("rows, V, dtype", [(2048, 513, "bf16"), (2050, 2049, "f32"), (2048, 4096, "bf16"), (515, 8193, "f16"), (512, 20001, "bf16")])
def test_many_long_rows(rows, V, dtype):
    """The choice of threads goes by rows as well: as many rows as change it, with runs of equal values longer than any list among them."""
    gen = torch.Generator(device="cuda").manual_seed(V)
    lg = _logits(gen, rows, V, dtype)
    lg[1] = 0.0
    lg[2] = (lg[2] > 0).to(lg.dtype)
    lg[3, ::2] = -float("inf")
    lg[4] = torch.randint(0, 3, (V,), device="cuda", generator=gen).to(lg.dtype) * 0.01
    keep = torch.arange(0, rows, max(1, rows // 60), device="cuda")
    keep = torch.cat([torch.arange(5, device="cuda"), keep[1:], torch.tensor([rows - 1], device="cuda")])
    for kw in (dict(), dict(top_k=50, top_p=0.9), dict(top_k=V // 2 + 1, top_p=0.6), dict(top_p=0.95, min_p=0.02), dict(top_k=V - 5)):
        u = torch.rand(rows, device="cuda", generator=gen)
        tok = shivae_amd.sample_categories(lg, u, **kw)
        want = _check(lg[keep], u[keep], **kw)  # (few rows: other threads, and the definition)
        torch.testing.assert_close(tok[keep], want, rtol=0, atol=0)


@pytest.mark.parametrize("V", [1000, 4099, 20001])
def test_top_k_where_the_largest_lie_together(V):
    """Sorted rows, the largest in one stretch, fewer finite logits than top_k, and a +inf among them, for top_k around half the threads."""
    gen = torch.Generator(device="cuda").manual_seed(V)
    lg = _logits(gen, 6, V, "f32")
    lg[0] = lg[0].sort(descending=True).values
    lg[1] = lg[1].sort().values
    lg[2, 100:400] += 9.0
    lg[3] = -float("inf")
    lg[3, 5::V // 9] = 1.0
    lg[4, 77] = float("inf")
    lg[4, 900] = float("inf")
    for k in (2, 20, 32, 33, 128, 129, 512, 513):
        for p in (1.0, 0.9):
            _check(lg, torch.rand(6, device="cuda", generator=gen), top_k=k, top_p=p)


def test_a_lead_that_ends_where_top_k_does():
    """top-k's last element, the lead's last element and min-p's limit in one bin, in rows that start off a 16-byte boundary."""
    gen = torch.Generator(device="cuda").manual_seed(9)
    V = 20001
    lg = _logits(gen, 7, V + 2, "bf16", spread=0.001)[:, 1:V + 1]
    lg[:, ::3] = torch.where(torch.rand(7, V, device="cuda", generator=gen) < 0.5, 1.0, 1.0078125).bfloat16()[:, ::3]
    for kw in (dict(top_k=5000, top_p=0.999), dict(top_k=6000, top_p=0.5, min_p=0.995), dict(top_k=6700, top_p=0.9999, min_p=0.2), dict(top_p=0.8, min_p=0.3)):
        for u in (0.0, 0.5, 1.0 - 2.0 ** -24):
            _check(lg, torch.full((7,), u, device="cuda"), **kw)


@pytest.mark.parametrize("V", [7, 64, 90, 1500, 21000])
def test_masked_and_non_finite_logits(V):
    gen = torch.Generator(device="cuda").manual_seed(3)
    for dtype in ("f32", "bf16", "f16"):
        base = _logits(gen, 8, V, dtype)
        low = torch.finfo(base.dtype).min
        lg = base.clone()
        lg[0] = -float("inf")                       # nothing allowed
        lg[1] = float("nan")
        lg[2, 1:] = -float("inf")                   # one allowed
        lg[3, ::2] = low                            # masked by the type's lowest value
        lg[4, ::2] = float("nan")
        lg[5, V // 2] = float("inf")
        lg[5, V - 1] = float("inf")                 # two share everything
        lg[6] = low                                 # a whole row of the lowest value: all equal
        lg[7, :-1] = -float("inf")
        for kw in (dict(), dict(temperature=0.0), dict(top_k=4), dict(top_p=0.9), dict(temperature=0.8, top_k=50, top_p=0.95, min_p=0.01)):
            tok = _check(lg, torch.rand(8, device="cuda", generator=gen), **kw)
            assert tok[:3].tolist() == [-1, -1, 0] and tok[7] == V - 1


@pytest.mark.parametrize("temperature", [1e-38, 1e-6, 1e-3, 1e4, float("inf")])
@pytest.mark.parametrize("V", [30, 333, 6000, 18000])
def test_extreme_temperatures(V, temperature):
    gen = torch.Generator(device="cuda").manual_seed(2)
    lg = _logits(gen, 3, V, "f32")
    for kw in (dict(), dict(top_k=20), dict(top_p=0.7), dict(top_k=V - 2, top_p=0.5)):
        _check(lg, torch.rand(3, device="cuda", generator=gen), temperature=temperature, **kw)


def test_strides_shapes_and_streams():
    gen = torch.Generator(device="cuda").manual_seed(4)
    wide = _logits(gen, 12, 131, "bf16").view(3, 4, 131)
    u = torch.rand(3, 4, device="cuda", generator=gen)
    for lg in (wide, wide[..., 1:], wide[..., 5:99], wide[:, ::2], wide.transpose(0, 1), wide[..., ::2], wide[:1].expand(3, 4, 131)):
        uu = u[:lg.shape[0], :lg.shape[1]] if lg.shape[0] <= 3 else u.t()
        assert _check(lg, uu, top_k=9, temperature=0.9).shape == lg.shape[:-1]
    one = shivae_amd.sample_categories(wide[0, 0], u[0, 0])
    assert one.shape == () and one == shivae_amd.sample_categories(wide, u)[0, 0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        t = shivae_amd.sample_categories(wide, u, top_p=0.9)
    side.synchronize()
    assert torch.equal(t, shivae_amd.sample_categories(wide, u, top_p=0.9))


def test_many_rows_and_the_largest_row():
    gen = torch.Generator(device="cuda").manual_seed(5)
    lg, u = _logits(gen, 70001, 8, "f32"), torch.rand(70001, device="cuda", generator=gen)
    tok = shivae_amd.sample_categories(lg, u)
    cum = torch.cumsum(torch.exp((lg - lg.max(1, keepdim=True).values).double()), 1)
    assert torch.equal(tok, (cum <= u.double()[:, None] * cum[:, -1:]).sum(1))
    V = shivae_amd.sampling.MAX_CATEGORIES
    row = torch.randn(V, device="cuda", generator=gen)
    for kw in (dict(), dict(top_k=5000), dict(top_p=0.5)):
        _check(row[None], torch.rand(1, device="cuda", generator=gen), **kw)


def test_graph_replay():
    gen = torch.Generator(device="cuda").manual_seed(6)
    lg, u = _logits(gen, 5, 20011, "bf16"), torch.rand(5, device="cuda", generator=gen)
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        tok = shivae_amd.sample_categories(lg, u, top_k=50, top_p=0.9)
    for _ in range(3):
        lg.copy_(_logits(gen, 5, 20011, "bf16"))
        u.copy_(torch.rand(5, device="cuda", generator=gen))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(tok, shivae_amd.sample_categories(lg, u, top_k=50, top_p=0.9))


def test_refusals():
    lg, u = torch.zeros(2, 8, device="cuda"), torch.zeros(2, device="cuda")
    f = shivae_amd.sample_categories
    for args, kw, err in (((lg, u[:1]), {}, ValueError), ((lg, u.double()), {}, TypeError), ((lg, u.cpu()), {}, ValueError),
                          ((lg.double(), u), {}, TypeError), ((lg[:, :0], u), {}, ValueError), ((lg, u), dict(temperature=-1.0), ValueError),
                          ((lg, u), dict(temperature=float("nan")), ValueError), ((lg, u), dict(top_k=-1), ValueError),
                          ((lg, u), dict(top_k=1.5), ValueError), ((lg, u), dict(top_p=1.1), ValueError), ((lg, u), dict(min_p=-0.1), ValueError),
                          ((lg, u), dict(top_k=torch.zeros(2, device="cuda")), TypeError), ((lg, u), dict(top_p=torch.zeros(3, device="cuda")), ValueError),
                          ((lg, u), dict(min_p=torch.zeros(2)), ValueError)):
        with pytest.raises(err):
            f(*args, **kw)


def test_a_models_categorical_attributes():
    """ShiVAE.sample_categories: draws of generated sequences are those of the operator on the likelihoods' logits."""
    tl = shivae_amd.utils.make_types_list(1, 1, 1, [3, 8, 70])
    m = shivae_amd.ShiVAE(16, 4, 3, 1, types_list=tl, learn_std=True).to("cuda")
    torch.manual_seed(0)
    _, _, likes = m.sample_from_prior(6, 11)
    cats = [t["name"] for t in tl if t["type"] == "cat"]
    u = {k: torch.rand(11, 6, device="cuda") for k in cats}
    got = m.sample_categories(likes, u, temperature=0.7, top_p=0.9)
    assert list(got) == cats
    for k in cats:
        assert got[k].shape == (11, 6) and torch.equal(got[k], _check(likes[k].logits, u[k], temperature=0.7, top_p=0.9))
    free = m.sample_categories(likes)
    assert all(int(free[k].min()) >= 0 and int(free[k].max()) < likes[k].logits.shape[-1] for k in cats)


def test_prompt_then_tokens():
    """The operators as they are used together: a prompt through convolution and scan with the states kept, then one drawn category
    at a time; every drawn step equals what the whole sequence, run at once, gives for that row."""
    gen = torch.Generator(device="cuda").manual_seed(8)
    V, D, Ns, B, T, new = 97, 64, 16, 3, 21, 12

    def rn(*s, f=1.0):
        return torch.randn(*s, device="cuda", generator=gen) * f

    table, w, A, head = rn(V, D), rn(4, D, f=0.5), -torch.exp(rn(Ns, D, f=0.5)), rn(D, V, f=D ** -0.5)
    pd, pb, pc, bias = rn(D, D, f=D ** -0.5), rn(D, Ns, f=D ** -0.5), rn(D, Ns, f=D ** -0.5), rn(D) - 2

    def inner(x):
        return x @ pd, (x @ pb).unsqueeze(-2), (x @ pc).unsqueeze(-2)

    def whole(tokens, lengths=None):
        x, cs = shivae_amd.causal_conv(table[tokens], w, None, "silu", lengths=lengths, return_state=True)
        y, ss = shivae_amd.selective_scan(x, *_order(inner(x), A), dt_bias=bias, lengths=lengths, return_state=True)
        return y, cs, ss

    def _order(p, a):
        return p[0], a, p[1], p[2]

    tokens = torch.randint(0, V, (T, B), device="cuda", generator=gen)
    n = torch.tensor([T, 5, 0], device="cuda")  # a full prompt, a short one, none
    y, cs, ss = whole(tokens, n)
    tok = tokens[(n - 1).clamp(min=0), torch.arange(B, device="cuda")]
    seqs = [tokens[:int(n[b]), b].tolist() for b in range(B)]
    outs = [[] for _ in range(B)]
    for _ in range(new):
        x = shivae_amd.causal_conv_step(table[tok], w, state=cs, activation="silu")
        p = inner(x)
        yt = shivae_amd.selective_scan_step(x, p[0], A, p[1], p[2], ss, dt_bias=bias)
        for b in range(B):
            seqs[b].append(int(tok[b]))
            outs[b].append(yt[b])
        tok = shivae_amd.sample_categories(yt @ head, torch.rand(B, device="cuda", generator=gen), temperature=0.9, top_k=20, top_p=0.95)
    for b in range(B):
        yb, _, _ = whole(torch.tensor(seqs[b], device="cuda")[:, None])
        got = torch.stack(outs[b])
        want = yb[-new:, 0]
        # fp32 throughout, at most T + new rows: 3 units a row for the scan and the products' sums over D, of values up to `scale`
        scale = float(want.abs().max())
        assert float((got - want).abs().max()) <= (3 * (T + new) + 96 + 4 * D) * 2.0 ** -24 * 8 * scale
