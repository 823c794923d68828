"""The rules that choose how the packed attention reads V and how the embedding's
backward sorts, against times measured on an MI355X with either choice: the chosen one
is within 5% of the faster, or half a microsecond. The rules are the header's own,
compiled here with g++.
"""
import ctypes
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SOURCE = """
#include "rules.hpp"
extern "C" {
int sort_while_clearing(int64_t tokens, int64_t clear) { return mc::embedding_sort_while_clearing(tokens, clear); }
int sort_ids(int64_t vocab) { return mc::embedding_sort_ids(vocab); }
int fwd_from_rows(int64_t seq) { return mc::packed_fwd_from_rows(seq); }
}
"""


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    d = tmp_path_factory.mktemp("packed_rules")
    src, so = d / "rules.cpp", d / "rules.so"
    src.write_text(SOURCE)
    inc = os.path.join(ROOT, "metal-candle_amd", "csrc")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", "-I", inc, str(src), "-o", str(so)],
                   check=True)
    return ctypes.CDLL(str(so))


def good(chosen, other):
    return chosen <= 1.05 * other or chosen <= other + 0.5


# tokens, vocab, dim, us beside the clearing, us after one another
BACKWARD = [
    (256, 2048, 512, 9.3, 11.2),
    (256, 16384, 512, 12.8, 16.4),
    (256, 50257, 512, 20.5, 24.5),
    (256, 32000, 1536, 31.8, 35.9),
    (256, 151936, 896, 89.2, 93.3),
    (1024, 2048, 512, 10.3, 11.9),
    (1024, 16384, 512, 13.3, 17.2),
    (1024, 50257, 512, 20.8, 25.1),
    (1024, 32000, 1536, 32.8, 37.0),
    (1024, 151936, 896, 90.4, 96.0),
    (2048, 2048, 512, 11.6, 12.5),
    (2048, 16384, 512, 14.8, 17.8),
    (2048, 50257, 512, 21.3, 25.9),
    (2048, 32000, 1536, 35.2, 39.9),
    (2048, 151936, 896, 93.6, 98.1),
    (4096, 2048, 512, 14.9, 13.9),
    (4096, 16384, 512, 17.6, 20.0),
    (4096, 50257, 512, 23.6, 28.1),
    (4096, 32000, 1536, 38.7, 44.2),
    (4096, 151936, 896, 98.3, 103.6),
    (8192, 2048, 512, 21.1, 16.8),
    (8192, 16384, 512, 23.2, 23.4),
    (8192, 50257, 512, 29.0, 31.8),
    (8192, 32000, 1536, 44.7, 51.4),
    (8192, 151936, 896, 105.8, 112.1),
    (16384, 2048, 512, 31.3, 22.3),
    (16384, 16384, 512, 34.1, 29.5),
    (16384, 50257, 512, 39.6, 38.8),
    (16384, 32000, 1536, 59.1, 64.2),
    (16384, 151936, 896, 117.7, 127.0),
    (65536, 2048, 512, 95.7, 54.6),
    (65536, 16384, 512, 85.0, 57.5),
    (65536, 50257, 512, 98.1, 72.9),
    (65536, 32000, 1536, 171.2, 146.2),
    (65536, 151936, 896, 210.0, 218.1),
]


@pytest.mark.parametrize("tokens,vocab,dim,beside,after", BACKWARD)
def test_sort_beside_the_clearing(rules, tokens, vocab, dim, beside, after):
    chosen = rules.sort_while_clearing(ctypes.c_int64(tokens), ctypes.c_int64(vocab * dim))
    assert good(beside, after) if chosen else good(after, beside)


def test_sort_into_a_given_gradient(rules):
    """Nothing is cleared: no workgroups to sort beside."""
    assert not rules.sort_while_clearing(ctypes.c_int64(16), ctypes.c_int64(0))


def test_ids_of_a_sorting_workgroup(rules):
    """16 to 512, and 128 to 256 workgroups in between."""
    for vocab in (1, 16, 4096):
        assert rules.sort_ids(ctypes.c_int64(vocab)) == 16
    for vocab in (4097, 16384, 32000, 50257, 131072):
        assert 128 <= -(-vocab // rules.sort_ids(ctypes.c_int64(vocab))) <= 256
    for vocab in (131073, 151936, 2**31 - 1):
        assert rules.sort_ids(ctypes.c_int64(vocab)) == 512


# head dim, batch, heads, length, (rows, V^T) without and with a cap
FORWARD = [
    (64, 1, 14, 65, (6.6, 8.2), (8.0, 9.6)),
    (64, 1, 14, 128, (6.7, 8.3), (8.1, 9.7)),
    (64, 1, 14, 256, (9.4, 9.8), (11.8, 11.9)),
    (64, 1, 14, 384, (12.1, 11.2), (15.7, 14.1)),
    (64, 1, 14, 512, (15.0, 12.7), (19.4, 16.3)),
    (64, 1, 14, 768, (20.4, 15.6), (26.9, 20.7)),
    (64, 1, 14, 1024, (25.8, 18.7), (34.3, 25.0)),
    (64, 1, 14, 2048, (47.5, 30.9), (64.1, 42.4)),
    (64, 8, 12, 65, (6.6, 8.3), (8.1, 9.8)),
    (64, 8, 12, 128, (6.9, 8.7), (8.3, 10.1)),
    (64, 8, 12, 256, (9.9, 10.4), (12.2, 12.5)),
    (64, 8, 12, 384, (12.8, 12.3), (16.3, 15.0)),
    (64, 8, 12, 512, (15.7, 14.3), (20.0, 18.6)),
    (64, 8, 12, 768, (22.2, 20.7), (30.0, 27.1)),
    (64, 8, 12, 1024, (29.6, 27.1), (41.0, 37.6)),
    (64, 8, 12, 2048, (83.6, 72.1), (112.6, 96.4)),
    (128, 1, 14, 65, (8.3, 9.9), (10.0, 11.6)),
    (128, 1, 14, 128, (8.6, 10.2), (10.4, 12.0)),
    (128, 1, 14, 256, (12.6, 12.3), (15.5, 14.9)),
    (128, 1, 14, 384, (16.7, 14.5), (20.3, 17.6)),
    (128, 1, 14, 512, (20.6, 16.5), (25.3, 20.5)),
    (128, 1, 14, 768, (28.6, 20.9), (35.1, 26.1)),
    (128, 1, 14, 1024, (36.4, 25.3), (44.8, 31.7)),
    (128, 1, 14, 2048, (67.6, 43.4), (83.6, 54.5)),
    (128, 8, 12, 65, (8.5, 10.3), (10.4, 12.1)),
    (128, 8, 12, 128, (9.2, 10.8), (10.9, 12.5)),
    (128, 8, 12, 256, (13.6, 13.6), (16.3, 15.7)),
    (128, 8, 12, 384, (18.5, 17.6), (22.3, 20.5)),
    (128, 8, 12, 512, (23.1, 20.7), (27.6, 24.3)),
    (128, 8, 12, 768, (32.1, 30.6), (38.8, 36.2)),
    (128, 8, 12, 1024, (46.6, 44.4), (60.3, 52.5)),
    (128, 8, 12, 2048, (139.0, 121.1), (170.8, 143.7)),
]


@pytest.mark.parametrize("D,B,H,S,plain,capped", FORWARD)
def test_v_from_its_rows(rules, D, B, H, S, plain, capped):
    for rows, transposed in (plain, capped):
        assert good(rows, transposed) if rules.fwd_from_rows(ctypes.c_int64(S)) else good(transposed, rows)
