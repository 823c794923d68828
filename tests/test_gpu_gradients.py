"""The gradients' global norm, clipping by it, and AdamW on scaled gradients.

The reference is numpy in 64 bits. The kernels sum squares in 64 bits, so the
norm is off by its rounding to float32, 2^-24 of its value (the 64-bit sums of up
to 1e7 squares add less than 1e7 * 2^-53 = 2^-29), and the scale, a 64-bit
quotient, likewise. A scaled gradient is one float32 product, rounded to the
output's type: compared for equality.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
HALF = 2.0**-24 * (1 + 2.0**-4)


def grads_of(sizes, dtypes, dev, seed=0, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(n, generator=g) * std).to(d).to(dev) for n, d in zip(sizes, dtypes)]


def norm64(grads):
    return math.sqrt(sum(float((g.double().cpu().numpy() ** 2).sum()) for g in grads))


SIZES = {
    "one": [1],
    "scalars": [1] * 7,
    "odd": [3, 257, 8191, 8193, 5],
    "empty_between": [0, 5, 0, 4096, 0],
    "many": [17 + i for i in range(400)],  # more tensors than one launch's table
    "layer": [1536 * 16, 16 * 1536, 1536 * 16, 16 * 256],
    "long": [9_000_001],  # chunks longer than the least
}


@pytest.mark.parametrize("dtype", ["f32", "bf16", "mixed"])
@pytest.mark.parametrize("name", list(SIZES))
def test_norm_and_clip(mc, dev, name, dtype):
    sizes = SIZES[name]
    kinds = {"f32": [torch.float32], "bf16": [torch.bfloat16], "mixed": [torch.bfloat16, torch.float32]}[dtype]
    grads = grads_of(sizes, [kinds[i % len(kinds)] for i in range(len(sizes))], dev)
    want = norm64(grads)
    for max_norm in (0.25 * want, 4.0 * want):
        m = float(np.float32(max_norm))
        scale64 = min(1.0, m / want)
        norm, scale = mc.gradient_norm(grads, m)
        assert abs(norm.item() - want) <= HALF * want
        assert abs(scale.item() - scale64) <= HALF * scale64
        if max_norm > want:
            assert scale.item() == 1.0
        outs = [torch.full((g.numel(),), float("nan"), dtype=d, device=dev)
                for g, d in zip(grads, [torch.float32, torch.bfloat16] * len(grads))]
        n2, s2 = mc.clip_gradients(grads, m, outs=outs)
        assert n2.item() == norm.item() and s2.item() == scale.item()
        for g, o in zip(grads, outs):
            assert torch.equal(o, (g.float() * s2).to(o.dtype))
        mine = [g.clone() for g in grads]
        assert mc.scale_gradients(mine, scale) is mine
        for g, o in zip(grads, mine):
            assert torch.equal(o, (g.float() * scale).to(g.dtype))
        mine = [g.clone() for g in grads]
        n3, _ = mc.clip_gradients(mine, m)
        assert n3.item() == norm.item()
        for g, o in zip(grads, mine):
            assert torch.equal(o, (g.float() * scale).to(g.dtype))
    norm, scale = mc.gradient_norm(grads)
    assert scale is None and abs(norm.item() - want) <= HALF * want


def test_alignments(mc, dev):
    """Gradients and outputs that start at any element of a buffer; what lies between them stays."""
    for td, od in ((torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32),
                   (torch.float32, torch.bfloat16)):
        flat = grads_of([4000], [td], dev, seed=3)[0]
        for a in range(9):
            for b in (0, 1, 3, 8):
                n = 1900 + a
                g = flat[a:a + n]
                back = torch.full((4000,), 7.0, dtype=od, device=dev)
                norm, scale = mc.clip_gradients([g], 1.0, outs=[back[b:b + n]])
                want = norm64([g])
                assert abs(norm.item() - want) <= HALF * want
                assert torch.equal(back[b:b + n], (g.float() * scale).to(od))
                assert (back[:b] == 7.0).all() and (back[b + n:] == 7.0).all()


def test_range_of_values(mc, dev):
    """Squares past float32's range, zeros, infinities and NaN."""
    big = [torch.full((1000,), 1e30, device=dev), torch.full((3,), 1e-30, device=dev)]
    norm, scale = mc.gradient_norm(big, 1.0)
    want = norm64(big)
    assert abs(norm.item() - want) <= HALF * want and abs(scale.item() * want - 1.0) <= HALF
    small = [torch.full((1000,), 1e-30, device=dev)]
    norm, scale = mc.gradient_norm(small, 1.0)
    want = norm64(small)
    assert abs(norm.item() - want) <= HALF * want and scale.item() == 1.0
    # a norm that float32 cannot hold is infinity; its scale is still max_norm / norm
    huge = [torch.full((1 << 20,), 3e38, device=dev)]
    limit = float(np.float32(1e30))
    norm, scale = mc.gradient_norm(huge, limit)
    want = limit / norm64(huge)
    assert norm.item() == math.inf and abs(scale.item() - want) <= HALF * want
    zero = [torch.zeros(5, device=dev), torch.zeros(0, device=dev)]
    norm, scale = mc.clip_gradients(zero, 1.0)
    assert norm.item() == 0.0 and scale.item() == 1.0 and (zero[0] == 0).all()
    for bad, f in ((math.inf, 0.0), (-math.inf, 0.0), (math.nan, math.nan)):
        g = [torch.ones(300, device=dev), torch.ones(70000, device=dev)]
        g[1][69999] = bad
        norm, scale = mc.clip_gradients(g, 1.0)
        assert norm.item() == math.inf or math.isnan(bad) and math.isnan(norm.item())
        assert scale.item() == f or math.isnan(f) and math.isnan(scale.item())
        assert math.isnan(g[1][69999].item())
    # no limit
    norm, scale = mc.gradient_norm(big, math.inf)
    assert scale.item() == 1.0


def test_only_empty_tensors(mc, dev):
    g = [torch.zeros(0, device=dev)]
    norm, scale = mc.clip_gradients(g, 1.0)
    assert norm.item() == 0.0 and scale.item() == 1.0


def test_reproducible_on_streams_and_in_graphs(mc, dev):
    grads = grads_of([70001, 33, 262144], [torch.float32, torch.bfloat16, torch.bfloat16], dev, seed=5)
    outs = [torch.empty(g.numel(), device=dev) for g in grads]
    norm, scale = mc.clip_gradients(grads, 1.0, outs=outs)
    first = [o.clone() for o in outs]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        n2, _ = mc.clip_gradients(grads, 1.0, outs=outs)
    side.synchronize()
    assert n2.item() == norm.item()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        n3, s3 = mc.clip_gradients(grads, 1.0, outs=outs)
        n4, s4 = mc.gradient_norm(grads, 1.0)
    for turn in range(3):
        for o in outs:
            o.fill_(math.nan)
        graph.replay()
        torch.cuda.synchronize()
        assert n3.item() == norm.item() == n4.item() and s3.item() == scale.item() == s4.item()
        assert all(torch.equal(a, b) for a, b in zip(outs, first))
        mc.clip_gradients([torch.ones(5, device=dev)], 1.0)  # another call between the replays


def test_adamw_on_scaled_gradients(mc, dev):
    """Equal bit for bit to scaling first, at ragged sizes and over several launches."""
    sizes = [1, 3, 4, 1025] + [64 + i for i in range(20)]
    make = lambda seed: grads_of(sizes, [torch.float32] * len(sizes), dev, seed=seed)  # noqa: E731
    params, grads, ms = make(0), make(1), [m * 0.1 for m in make(2)]
    vs = [v.abs() * 0.01 for v in make(3)]
    steps = [1 + i for i in range(len(sizes))]
    norm, scale = mc.gradient_norm(grads, 1.0)
    assert scale.item() < 1.0
    a = [[t.clone() for t in g] for g in (params, ms, vs)]
    b = [[t.clone() for t in g] for g in (params, ms, vs)]
    mc.adamw_step(a[0], grads, a[1], a[2], steps, lr=1e-3, grad_scale=scale)
    clipped = [torch.empty_like(g) for g in grads]
    mc.scale_gradients(grads, scale, outs=clipped)
    mc.adamw_step(b[0], clipped, b[1], b[2], steps, lr=1e-3)
    for x, y in zip(a, b):
        assert all(torch.equal(s, t) for s, t in zip(x, y))
    plain = [t.clone() for t in params]
    mc.adamw_step(plain, grads, [m.clone() for m in ms], [v.clone() for v in vs], steps, lr=1e-3)
    assert not torch.equal(plain[3], a[0][3])
