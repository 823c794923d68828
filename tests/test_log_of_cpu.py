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
def log_of(tmp_path_factory):
    d = tmp_path_factory.mktemp("log_of")
    src, so = d / "log_of.cpp", d / "log_of.so"
    src.write_text('#include "log_of.hpp"\nextern "C" double log_of(double s) { return mc::log_of(s); }\n')
    inc = os.path.join(ROOT, "metal-candle_amd", "csrc")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", "-I", inc, str(src), "-o", str(so)],
                   check=True)
    fn = ctypes.CDLL(str(so)).log_of
    fn.restype, fn.argtypes = ctypes.c_double, [ctypes.c_double]
    return fn


def test_log_of(log_of):
    rng = random.Random(0)
    sums = [1.0, 2.0, 0.5, 1.0 + 2.0 ** -40, 1.0 - 2.0 ** -40, math.sqrt(2.0), math.sqrt(0.5), 151936.0, 2.0 ** 31, 1e-300]
    for root in (2.0 ** 0.5, 2.0 ** 1.5):  # either side of where the exponent changes
        sums += [math.nextafter(root, 0.0), math.nextafter(root, 9.0)]
    sums += [math.exp(rng.uniform(0.0, 22.0)) for _ in range(20000)] + [1.0 + rng.random() for _ in range(20000)]
    for s in sums:
        want = math.log(s)
        assert abs(log_of(s) - want) <= 4e-11 + 2.0 ** -51 * abs(want), s


def test_log_of_nan(log_of):
    assert math.isnan(log_of(math.nan)) and math.isnan(log_of(math.inf))
