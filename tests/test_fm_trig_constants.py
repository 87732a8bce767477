"""CPU: where the constants of libm_sinf / libm_cosf / libm_atanf / libm_atan2f (kernels/libm_float.hh) come from.  Each is what
mathematics gives, or lies where the values that sinf and cosf RETURN confine it (tools/fit_fm_trig.py).  Nothing in the file may
rest on the contents of an installed library's binary."""
import importlib.util
import os
import re
from decimal import Decimal

import numpy as np
import pytest

import util

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "cyberether_amd", "csrc", "kernels", "libm_float.hh")


@pytest.fixture(scope="module")
def header():
    return open(HEADER).read()


@pytest.fixture(scope="module")
def fit():
    spec = importlib.util.spec_from_file_location("fit_fm_trig", os.path.join(ROOT, "tools", "fit_fm_trig.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def words(text):
    return [int(v, 16) for v in re.findall(r"0x([0-9a-f]{8})u", text)]


def doubles(header, *names):
    return [float.fromhex(re.search(rf"\b{n} = (-?0x1\.[0-9a-f]+p[+-]?\d+)", header).group(1)) for n in names]


def braces(header, name):
    return words(re.search(rf"{name}\[\d+\] = {{(.*?)}};", header, re.S).group(1))


def test_no_source_rests_on_a_binary(header):
    for phrase in ("objdump", "instruction stream", "stored in libm", "read back from"):
        assert phrase not in header, phrase


def test_multiples_of_pi(header, fit):
    assert doubles(header, "kTwoOverPi", "kHalfPi") == [float(2 / fit.PI), float(fit.PI / 2)]
    assert braces(header, "two_over_pi") == [int(v) for v in fit.two_over_pi_words(8)]
    f32 = lambda d: int(np.float32(float(d)).view(np.uint32))  # noqa: E731
    named = dict(re.findall(r"\b(\w+) = u2f\(0x([0-9a-f]{8})u\)", header[header.index("libm_atan2f(float y"):]))
    pi32 = Decimal(float(np.float32(float(fit.PI))))
    want = {"pi": fit.PI, "pi_lo": fit.PI - pi32, "half_pi": fit.PI / 2, "quarter_pi": fit.PI / 4, "three_quarter_pi": 3 * fit.PI / 4}
    assert {k: int(v, 16) for k, v in named.items()} == {k: f32(v) for k, v in want.items()}


def test_atan_constants_are_chopped_values_and_the_minimax_polynomial(header, fit):
    values = [fit.atan(Decimal(1) / 2), fit.PI / 4, fit.PI / 4 + fit.atan(Decimal(1) / 5), fit.PI / 2]
    hi = [fit.chop(v) for v in values]
    assert braces(header, "atan_hi") == [int(h.view(np.uint32)) for h in hi]
    assert braces(header, "atan_lo") == [int(fit.chop(v - Decimal(float(h))).view(np.uint32)) for v, h in zip(values, hi)]
    a = np.array([int(re.search(rf"\ba{k} = u2f\(0x([0-9a-f]{{8}})u\)", header).group(1), 16) for k in range(11)], np.uint32)
    minimax = np.array([float(v) for v in fit.minimax_atan(10, (Decimal(7) / 16) ** 2)], np.float32).view(np.uint32)
    off = np.abs(a.astype(np.int64) - minimax.astype(np.int64))
    assert (off[:7] <= 1).all() and off.max() <= 1024, off  # the moved ones: ulps of coefficients far below the result's


def test_sine_and_cosine_coefficients_lie_where_the_returned_values_put_them(header, fit):
    if not util.libm_pinned():
        pytest.skip("the values of another libm confine other coefficients")
    lib = fit.compile_scanner()
    hpi, table = float(fit.PI / 2), fit.two_over_pi_words(8)
    for cosine, names in ((0, ("S0", "S1", "S2")), (1, ("C0", "C1", "C2", "C3"))):
        c = np.array(doubles(header, *names))
        zero, buf = np.zeros(len(c)), np.zeros((100000, 4))
        for called in (0, 1):  # every float of [2^-12, 2^20): none may lie outside its rounding interval
            lo, hi = fit.bits(2.0 ** -12), fit.bits(2.0 ** 20)
            n = lib.tightest(called, cosine, lo, 1, hi - lo, fit.ptr(c), fit.ptr(zero), len(c), hpi, fit.ptr(table), 1e-8, fit.ptr(buf),
                             len(buf), fit.THREADS)
            assert 0 < n < len(buf) and buf[:n, 1:3].min() > 0.0, (names, called, n, buf[:n, 1:3].min())
