"""On the CPU: sizes past what a launch can have (2^32 threads) are refused before the first launch."""
from shivae_amd import _native as N

from test_seq_ops_cpu import _conv, _refused, _ssm


def test_grids_past_a_launch_are_refused():
    L = N.lib()
    # 2^30 sequences of four 16-byte groups of channels; of one channel each, where a sequence is not aligned
    for kw in (dict(T=1, B=2 ** 30, D=16, x_sb=16, y_sb=16), dict(T=1, B=2 ** 30, D=4, x=68), dict(T=5, B=2 ** 29, D=9)):
        _refused(L.shivae_causal_conv_fwd, _conv(**kw), "too large")
        _refused(L.shivae_causal_conv_bwd, _conv(**kw, dy=64, dx=64, dweight=64), "too large", None, 0)
    for kw in (dict(T=1, B=2 ** 30, D=16), dict(T=1, B=2 ** 30, D=4, u=68)):
        _refused(L.shivae_selective_scan_fwd, _ssm(**kw), "too large", None, 0)
    full = {k: 64 for k in ("dy", "du", "ddt", "dB", "dC", "dA", "ckpt")}
    for kw in (dict(T=2, B=2 ** 24, D=1), dict(T=1, B=2 ** 23, D=80), dict(T=3, B=2 ** 23, D=2, G=2)):
        _refused(L.shivae_selective_scan_fwd, _ssm(**kw, ckpt=64), "too large", None, 0)
        _refused(L.shivae_selective_scan_bwd, _ssm(**kw, **full), "too large", None, 0)


def test_the_largest_grids_are_not():
    """One sequence fewer, and the next check speaks: the workspace that is missing."""
    L = N.lib()
    full = {k: 64 for k in ("dy", "du", "ddt", "dB", "dC", "dA", "ckpt")}
    _refused(L.shivae_selective_scan_bwd, _ssm(T=2, B=2 ** 24 - 1, D=1, **full), "workspace", None, 0)
    _refused(L.shivae_causal_conv_bwd, _conv(T=1, B=2 ** 30 - 64, D=16, x_sb=16, dy=64, dy_sb=16, dx=64, dweight=64), "workspace", None, 0)
