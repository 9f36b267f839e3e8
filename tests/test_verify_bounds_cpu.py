"""The race for the token behind the drafts is run in 32 bits with a bound on the error of every share, and again in 64 bits for the entries
that can win: the bound has to hold for every share that 32 bits have."""
import math
import os
import re

import numpy as np

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mesh-transformer-jax_b200", "csrc", "mtj_verify.cu")
HALF = 2.0 ** -24                         # a rounding to 32 bits


def _constant(name):
    with open(SOURCE) as f:
        value = re.search(rf"\b{name} = ([0-9.e+-]+)f\b", f.read()).group(1)
    return float(np.float32(value))


def test_the_bound_of_a_share_covers_its_roundings():
    # share = ex2((logit - top) * scale) * (1 / sum), scale = log2(e) / temp: the argument reaches 126 before the share leaves the range;
    # its difference, its product and scale's quotient are rounded, and log2(e) is
    log2e = abs(_constant("kLog2e") - math.log2(math.e)) / math.log2(math.e)
    argument = 126 * math.log(2) * (3 * HALF + log2e)
    # ex2.approx.ftz.f32: 2 units in the last place, 2^-22; the sum's reciprocal, the product and p + q (twice: in the slack too)
    bound = argument + 2.0 ** -22 + 4 * HALF
    assert bound < 2.0 ** -15.7
    assert _constant("kSlack") > 1.01 * bound


def test_shares_in_32_bits_are_within_the_bound():
    """The same arithmetic on the host, its exponential exact."""
    rng = np.random.default_rng(3)
    f = np.float32
    worst = 0.0
    for temp in (1e-17, 3.7e-9, 1e-3, 0.3, 1.0, 7.7, 3e5, 1e25):
        distance = (rng.random(20000) * 87 * temp).astype(f)
        for top in (0.0, 12.3, -4567.8):
            top = f(top * temp)
            logit = top - distance
            scale = f(_constant("kLog2e")) / f(temp)
            share = np.exp2(((logit - top) * scale).astype(np.float64))
            exact = np.exp((logit.astype(np.float64) - np.float64(top)) / np.float64(f(temp)))
            worst = max(worst, np.abs(share / exact - 1).max())
    assert 2.0 ** -19 < worst < _constant("kSlack") - 2.0 ** -22 - 4 * HALF
