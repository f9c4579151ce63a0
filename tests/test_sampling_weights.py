"""On the CPU: the polynomial that weighs a category (csrc/sample.hip), from its coefficients in the source, is as good as the interface
says, 2^-38 of the weight."""
import os
import re

import numpy as np

import shivae_amd


def test_the_weights_polynomial():
    path = os.path.join(os.path.dirname(shivae_amd.sampling.__file__), "csrc", "sample.hip")
    body = re.search(r"double exp2_f64\(double y\) \{(.*?)\n\}", open(path).read(), re.S).group(1)
    coefficients = [float(c) for c in re.findall(r"p = (?:fma\(p, f, )?([0-9.e+-]+)\)?;", body)]
    assert len(coefficients) == 9 and coefficients[-1] == 1.0
    f = np.linspace(-0.5, 0.5, 200001).astype(np.longdouble)
    p = np.zeros_like(f)
    for c in coefficients:
        p = p * f + np.longdouble(c)
    off = float(np.abs(p / np.exp2(f) - 1).max())
    # and in 64 bits: nine operations, each within 2^-53 of the result
    assert off + 9 * 2.0 ** -53 <= 2.0 ** -38
    assert off > 2.0 ** -39  # (no better: not the 2^-43 to which weights are held)
