"""Outputs of the gradients' scaling and clipping that overlap each other or another
tensor's gradient are refused on the host: workgroups of one tensor would overwrite
what those of another have yet to read."""
import ctypes
import random

import pytest

LAYOUT, HIP = 4, 7
FAKE = ctypes.c_void_p(256)
F32, BF16 = 0, 1


def status(mc, rows, which="scale"):
    """The status of a call on (grad, out, numel, dtype, out_dtype) rows of made-up addresses, whose workspace is too
    small: what passes the table's checks ends there."""
    L = mc._lib.lib()
    t = (mc._lib.GradTensor * len(rows))(*[mc._lib.GradTensor(*r) for r in rows])
    if which == "clip":
        return L.mc_clip_gradients(t, len(rows), 1.0, FAKE, FAKE, None, 0, None)
    return L.mc_scale_gradients(t, len(rows), None, None)


PASSES = {"clip": 6, "scale": 1}  # the workspace, the missing scale


@pytest.mark.parametrize("which", ["clip", "scale"])
@pytest.mark.parametrize("name,rows", [
    ("swapped", [(4096, 8192, 64, F32, F32), (8192, 4096, 64, F32, F32)]),
    ("round", [(4096, 8192, 64, F32, F32), (8192, 12288, 64, F32, F32), (12288, 4096, 64, F32, F32)]),
    ("views in place", [(4096, 4096, 100, F32, F32), (4096 + 396, 4096 + 396, 100, F32, F32)]),
    ("views in place, bf16", [(4096 + 198, 4096 + 198, 100, BF16, BF16), (4096, 4096, 100, BF16, BF16)]),
    ("one inside the other", [(4096, 4096, 1000, F32, F32), (4400, 4400, 1, F32, F32), (9000, 9000, 5, F32, F32)]),
    ("outs overlap", [(4096, 65536, 100, BF16, F32), (8192, 65536 + 396, 100, BF16, F32)]),
    ("same out", [(4096, 65536, 10, F32, F32), (8192, 65536, 10, F32, F32)]),
    ("out at another's gradient", [(4096, 65536, 100, F32, F32), (8192, 4096 + 396, 100, F32, BF16)]),
    ("in place beside it", [(4096, 4096, 100, F32, F32), (4096 + 200, 65536, 3, F32, F32)]),
    ("behind an empty one", [(None, None, 0, F32, F32), (4096, 8192, 2, F32, F32), (8196, 16384, 2, F32, F32)]),
])
def test_overlaps_are_refused(mc, which, name, rows):
    for order in (rows, rows[::-1]):
        assert status(mc, order, which) == LAYOUT
        assert "overlap" in mc._lib.last_error()


@pytest.mark.parametrize("which", ["clip", "scale"])
def test_what_lies_apart_passes(mc, which):
    ok = PASSES[which]
    assert status(mc, [(4096, 4096, 100, F32, F32), (4496, 4496, 100, F32, F32)], which) == ok  # one behind the other
    assert status(mc, [(4496, 4496, 100, F32, F32), (4096, 4096, 100, F32, F32)], which) == ok
    assert status(mc, [(4096, 4496, 100, F32, F32), (4896, 5296, 100, F32, F32)], which) == ok  # in turn
    assert status(mc, [(4096, 8192, 10, F32, F32), (4100, 9000, 10, F32, F32)], which) == ok  # gradients may overlap
    assert status(mc, [(4096, 8192, 10, F32, F32), (8200, 8200, 0, F32, F32)], which) == ok


def test_against_every_pair(mc):
    """Drawn tables against the definition, pair by pair."""
    rng = random.Random(5)
    seen = set()
    for _ in range(3000):
        rows, size = [], rng.choice([40, 200, 1000])
        for _ in range(rng.randrange(2, 6)):
            dt, ot, n = rng.randrange(2), rng.randrange(2), rng.randrange(0, 6)
            g, o = 4096 + 4 * rng.randrange(size), 4096 + 4 * rng.randrange(size)
            rows.append((g, g, n, dt, dt) if rng.random() < 0.4 else (g, o, n, dt, ot))
        grads = [(g, g + n * (4, 2)[dt]) for g, o, n, dt, ot in rows]
        outs = [(o, o + n * (4, 2)[ot]) for g, o, n, dt, ot in rows]
        meet = lambda a, b: a[0] < b[1] and b[0] < a[1] and a[0] < a[1] and b[0] < b[1]  # noqa: E731
        bad = False
        for i in range(len(rows)):
            own = rows[i][0] == rows[i][1] and rows[i][3] == rows[i][4]
            bad |= meet(outs[i], grads[i]) and not own
            for j in range(len(rows)):
                if i != j:
                    bad |= meet(outs[i], outs[j]) or meet(outs[i], grads[j])
        assert (status(mc, rows) == LAYOUT) == bad, rows
        seen.add(bad)
    assert seen == {True, False}
