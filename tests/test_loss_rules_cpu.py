"""The rules that choose the kernels' shapes for the losses over log-probabilities,
against times measured on an MI355X with either shape: the chosen one is within 5%
of the fastest, or half a microsecond. The rules are the header's own, compiled here
with g++.
"""
import ctypes
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SOURCE = """
#include "rules.hpp"
extern "C" {
int row_threads(int64_t rows, int64_t row_bytes) { return mc::loss_row_threads(rows, row_bytes); }
int row_parts(int64_t rows, int64_t vocab, int elem_size, int both) {
    return mc::loss_row_parts(rows, vocab, elem_size, both != 0);
}
int grad_threads(int64_t rows, int64_t row_bytes) { return mc::loss_grad_grid(rows, row_bytes).threads; }
int grad_parts(int64_t rows, int64_t row_bytes) { return (int)mc::loss_grad_grid(rows, row_bytes).parts; }
}
"""


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    d = tmp_path_factory.mktemp("loss_rules")
    src, so = d / "rules.cpp", d / "rules.so"
    src.write_text(SOURCE)
    inc = os.path.join(ROOT, "metal-candle_amd", "csrc")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", "-I", inc, str(src), "-o", str(so)],
                   check=True)
    return ctypes.CDLL(str(so))


def i64(*values):
    return [ctypes.c_int64(v) for v in values]


def good(times, chosen):
    best = min(times.values())
    return times[chosen] <= 1.05 * best or times[chosen] <= best + 0.5


# KB per row, rows, us by threads
STATISTICS = [
    (4, 400, {64: 5.4, 128: 5.4, 256: 5.6, 512: 6.4, 1024: 8.3}),
    (4, 16384, {64: 17.6, 128: 26.0, 256: 42.8, 512: 67.3, 1024: 132.3}),
    (8, 1000, {64: 6.0, 128: 6.0, 256: 6.8, 512: 9.5, 1024: 13.3}),
    (8, 4096, {64: 11.3, 128: 11.5, 256: 14.7, 512: 24.2, 1024: 40.1}),
    (12, 400, {64: 6.1, 128: 6.3, 256: 5.7, 512: 7.3, 1024: 9.5}),
    (12, 1000, {64: 7.2, 128: 7.5, 256: 7.5, 512: 9.9, 1024: 14.6}),
    (12, 4096, {64: 13.7, 128: 15.3, 256: 15.1, 512: 24.7, 1024: 42.8}),
    (20, 8192, {64: 33.9, 128: 36.4, 256: 40.7, 512: 48.3, 1024: 95.6}),
    (24, 400, {64: 8.6, 128: 7.8, 256: 7.1, 512: 7.5, 1024: 10.5}),
    (24, 1000, {64: 9.8, 128: 9.5, 256: 10.4, 512: 10.5, 1024: 16.5}),
    (24, 4096, {64: 22.0, 128: 21.6, 256: 24.1, 512: 27.4, 1024: 51.4}),
    (32, 400, {64: 10.4, 128: 9.4, 256: 7.7, 512: 8.5, 1024: 10.8}),
    (32, 4096, {64: 30.5, 128: 29.2, 256: 28.1, 512: 30.7, 1024: 52.1}),
    (64, 400, {64: 16.1, 128: 13.8, 256: 10.0, 512: 10.8, 1024: 11.8}),
    (64, 4096, {64: 53.8, 128: 52.7, 256: 53.0, 512: 52.1, 1024: 58.6}),
    (96, 400, {64: 21.5, 128: 18.1, 256: 12.1, 512: 12.7, 1024: 15.4}),
    (96, 4096, {64: 76.0, 128: 75.9, 256: 72.8, 512: 73.2, 1024: 80.1}),
    (128, 4096, {64: 98.0, 128: 98.4, 256: 98.8, 512: 97.3, 1024: 89.2}),
    (192, 400, {64: 37.9, 128: 30.7, 256: 18.9, 512: 18.6, 1024: 20.5}),
    (192, 4096, {64: 146.8, 128: 145.7, 256: 141.7, 512: 142.1, 1024: 131.9}),
    (304, 128, {64: 56.3, 128: 31.8, 256: 19.8, 512: 16.3, 1024: 15.6}),
    (304, 400, {64: 75.8, 128: 48.3, 256: 29.5, 512: 28.9, 1024: 30.5}),
    (304, 1000, {64: 82.4, 128: 58.6, 256: 60.3, 512: 58.7, 1024: 57.1}),
    (608, 1000, {64: 270.8, 256: 224.0, 512: 238.7, 1024: 226.7}),
]
GRADIENTS = [
    (2, 8192, {64: 9.5, 256: 14.5, 512: 22.6, 1024: 38.8}),
    (4, 16384, {64: 24.8, 256: 27.7, 512: 43.6, 1024: 74.3}),
    (4, 1000, {64: 5.1, 256: 5.2, 512: 5.9, 1024: 7.9}),
    (8, 8192, {64: 25.8, 256: 23.8, 512: 28.8, 1024: 43.5}),
    (12, 4096, {64: 19.5, 256: 18.4, 512: 19.9, 1024: 26.9}),
    (16, 8192, {64: 55.0, 256: 50.2, 512: 47.3, 1024: 64.0}),
    (24, 2000, {64: 19.8, 256: 18.3, 512: 18.3, 1024: 20.1}),
    (32, 32, {64: 6.4, 256: 4.9, 512: 4.7, 1024: 5.3}),
    (32, 8192, {64: 106.6, 256: 97.6, 512: 96.7, 1024: 93.1}),
    (64, 256, {64: 18.3, 256: 10.6, 512: 9.7, 1024: 8.8}),
    (96, 32, {64: 6.7, 256: 5.0, 512: 4.8, 1024: 5.5}),
    (96, 128, {64: 11.0, 256: 8.3, 512: 8.2, 1024: 7.8}),
    (304, 32, {64: 9.5, 256: 7.4, 512: 6.8, 1024: 7.4}),
    (304, 256, {64: 68.9, 256: 29.6, 512: 28.1, 1024: 27.6}),
    (608, 128, {64: 42.0, 256: 27.7, 512: 27.1, 1024: 27.5}),
]


@pytest.mark.parametrize("kb,rows,times", STATISTICS)
def test_threads_of_a_row(rules, kb, rows, times):
    assert good(times, rules.row_threads(*i64(rows, kb << 10)))


@pytest.mark.parametrize("kb,rows,times", GRADIENTS)
def test_threads_of_a_gradient(rules, kb, rows, times):
    assert good(times, rules.grad_threads(*i64(rows, kb << 10)))


# rows, vocabulary, bytes per logit, forward and backward in one; us, a workgroup per row / shared rows
@pytest.mark.parametrize("rows,vocab,size,both,one,shared", [
    (1, 151936, 2, 0, 12.0, 7.5), (64, 151936, 2, 0, 13.1, 9.7), (128, 151936, 2, 0, 13.6, 12.3),
    (50, 50257, 4, 0, 7.5, 7.9), (20, 50257, 2, 0, 6.8, 7.2), (4, 151936, 2, 1, 22.1, 9.4), (32, 151936, 2, 1, 23.1, 12.0),
    (64, 151936, 2, 1, 24.2, 15.8), (100, 151936, 2, 1, 24.9, 22.5), (4, 151936, 4, 1, 22.4, 9.1),
    (32, 151936, 4, 1, 25.7, 14.4), (64, 151936, 4, 1, 28.1, 22.7), (100, 151936, 4, 1, 31.2, 33.7),
    (64, 100000, 2, 1, 18.5, 12.8), (16, 50257, 4, 1, 11.5, 8.5), (32, 50257, 4, 1, 12.0, 9.9),
    (32, 50257, 2, 1, 10.7, 8.9), (4, 32000, 2, 1, 7.9, 8.2),
])
def test_rows_shared(rules, rows, vocab, size, both, one, shared):
    parts = rules.row_parts(*i64(rows, vocab), size, both)
    assert good({1: one, 2: shared}, min(parts, 2))


def test_limits(rules):
    most = (1 << 32) - 1
    for rows in (1, 2, 63, 64, 65, 255, 256, 257, 767, 768, 1535, 1536, (1 << 22) - 1, 1 << 22, (1 << 24) - 1):
        for kb in (0, 1, 5, 6, 9, 10, 15, 16, 27, 28, 39, 63, 64, 111, 112, 256, 1 << 20, (1 << 23) - 1):
            b = max(kb << 10, 2)
            for threads, parts in ((rules.row_threads(*i64(rows, b)), 1),
                                   (rules.grad_threads(*i64(rows, b)), rules.grad_parts(*i64(rows, b)))):
                assert threads in (64, 128, 256, 512, 1024) and parts >= 1
                assert rules.grad_threads(*i64(rows, b)) != 128  # not compiled
                assert rows * threads <= most and (parts == 1 or rows < 256) and parts <= 512
            for size in (2, 4):
                for both in (0, 1):
                    parts = rules.row_parts(*i64(rows, b // size), size, both)
                    assert 1 <= parts <= 32 and (parts == 1 or rows <= 128)
