"""The errors of beam selection's sums in 32 bits, from the constants in its source: two beams whose order they could turn lie closer than BS_NEAR, within which the sums are formed again in 64 bits."""
import math
import os
import re

import numpy as np

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def constants():
    with open(os.path.join(ROOT, "nano-vllm_b200", "csrc", "b2_beam.cu")) as f:
        text = re.sub(r"//[^\n]*", "", f.read())
    return {name: float(re.search(rf"\b{name} = ([0-9.e+-]+?)f?[;,]", text)[1]) for name in ("BS_NEAR", "BS_ABOVE", "BS_VECTORS")}


LOG2E = float(np.float32(math.log2(math.e)))


def largest_exponent(above):
    """The reference is a whole number M; it is raised when a logit is `above` over M / log2(e), a bound that is formed in 32 bits for |M| < 65536 log2(e) + 1: 2^-8 and 2^-7 of rounding at most."""
    return (above + 2.0 ** -7) * math.log2(math.e) + 2.0 ** -6


def test_two_sums_in_32_bits_are_closer_than_what_is_decided_again():
    c = constants()
    top = largest_exponent(c["BS_ABOVE"])
    half_ulp = 2.0 ** (math.ceil(math.log2(top)) - 1 - 24)  # of exponents below the next power of two, rounded to 24 bits
    exponent = half_ulp * math.log(2.0)
    log2e = top * abs(LOG2E / math.log2(math.e) - 1.0) * math.log(2.0)
    exponential = 2.0 ** -22
    additions = (c["BS_VECTORS"] * 8 / 4 + 2) * 2.0 ** -24  # a thread's numbers in four sums, and those together
    assert 2 * (exponent + log2e + exponential + additions) <= c["BS_NEAR"]


def test_an_exponents_error():
    """The multiply-add on the host: the product is exact in 64 bits, and the result is rounded once."""
    c = constants()
    r = np.random.default_rng(1)
    for reference in (-90.0, -3.0, 0.0, 5.0, 1000.0, 94000.0):
        below = reference / math.log2(math.e)
        x = np.float32(below + r.uniform(-1.0, c["BS_ABOVE"], 200000)).astype(np.float64)
        # (the sum's log gives back what log2(e) in 24 bits makes of the reference itself)
        rounded = np.float32(x * LOG2E - reference).astype(np.float64) - reference * (LOG2E / math.log2(math.e) - 1.0)
        error = np.abs(rounded - (x * math.log2(math.e) - reference)) * math.log(2.0)
        assert error.max() <= 1e-6  # 2^-20 log(2) of rounding and 3e-7 of log2(e)
