"""The logarithm that the loss kernels take of a row's sum, compiled here with g++,
against the C library's: within 4e-11, and 2^-51 of the result for the two libraries'
last bits."""
import ctypes
import math
import os
import random
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def logs(tmp_path_factory):
    d = tmp_path_factory.mktemp("log_of")
    src, so = d / "log_of.cpp", d / "log_of.so"
    src.write_text('#include "log_of.hpp"\nextern "C" double log_ratio(double a, double b) { return mc::log_ratio(a, b); }\n'
                   'extern "C" double log_of(double s) { return mc::log_of(s); }\n')
    inc = os.path.join(ROOT, "metal-candle_amd", "csrc")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", "-I", inc, str(src), "-o", str(so)],
                   check=True)
    lib = ctypes.CDLL(str(so))
    lib.log_of.restype, lib.log_of.argtypes = ctypes.c_double, [ctypes.c_double]
    lib.log_ratio.restype, lib.log_ratio.argtypes = ctypes.c_double, [ctypes.c_double] * 2
    return lib


def test_log_of(logs):
    rng = random.Random(0)
    sums = [1.0, 2.0, 0.5, 1.0 + 2.0 ** -40, 1.0 - 2.0 ** -40, math.sqrt(2.0), math.sqrt(0.5), 151936.0, 2.0 ** 31, 1e-300]
    for root in (2.0 ** 0.5, 2.0 ** 1.5):  # either side of where the exponent changes
        sums += [math.nextafter(root, 0.0), math.nextafter(root, 9.0)]
    sums += [math.exp(rng.uniform(0.0, 22.0)) for _ in range(20000)] + [1.0 + rng.random() for _ in range(20000)]
    for s in sums:
        want = math.log(s)
        assert abs(logs.log_of(s) - want) <= 4e-11 + 2.0 ** -51 * abs(want), s


def test_log_ratio(logs):
    """The library's of either number, each with a last bit; sums next to each other, whose logarithm is small."""
    rng = random.Random(1)
    pairs = [(math.exp(rng.uniform(-20.0, 22.0)), math.exp(rng.uniform(-20.0, 22.0))) for _ in range(20000)]
    pairs += [(s, s * (1.0 + d)) for s, d in ((1.0, 2.0 ** -30), (1.999999, 2.0 ** -18), (2.0, -2.0 ** -40), (7.5, 0.0))]
    for a, b in pairs:
        want = math.log(a) - math.log(b)
        assert abs(logs.log_ratio(a, b) - want) <= 4e-11 + 2.0 ** -51 * (abs(math.log(a)) + abs(math.log(b)) + abs(want)), (a, b)
    assert logs.log_ratio(3.0, 3.0) == 0.0


def test_log_of_nan(logs):
    for v in (math.nan, math.inf):
        assert math.isnan(logs.log_of(v)) and math.isnan(logs.log_ratio(v, 2.0)) and math.isnan(logs.log_ratio(2.0, v))
