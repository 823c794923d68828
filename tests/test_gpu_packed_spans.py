"""Packed attention on spans that a caller wrote: any intervals on which a query and
a key agree. The first pass of the backward stores dS^T for the second in the
workspace; NaN there before the call must not reach a gradient, and neither must NaN
in rows of q and dout that see nothing and of k and v that nothing sees.

Against 64 bits with the bounds of packed_reference.py."""
import math

import pytest
import torch

import packed_reference as ref

pytestmark = pytest.mark.gpu


def block(S, *parts):
    """Queries [a, b) see keys [c, d) for each (a, b, c, d)."""
    see = torch.zeros(S, S, dtype=torch.bool)
    for a, b, c, d in parts:
        see[a:b, c:d] = True
    return see


def band(S, lo, hi):
    """Query i sees the keys from i + lo up to and without i + hi."""
    far = torch.arange(S) - torch.arange(S)[:, None]
    return (far >= lo) & (far < hi)


LAYOUTS = {
    "second_tile_sees_first": lambda: block(256, (128, 256, 0, 128)),
    "two_far_ranges_in_a_tile": lambda: block(640, (0, 64, 0, 64), (64, 128, 512, 576)),
    "each_other": lambda: block(384, (0, 128, 256, 384), (256, 384, 0, 128)),
    "half_tiles": lambda: block(400, (0, 64, 192, 256), (64, 128, 320, 400), (300, 310, 0, 1)),
    "one_pair": lambda: block(300, (5, 6, 290, 291)),
    "strictly_before_129": lambda: band(129, -129, 0),
    "strictly_before_257": lambda: band(257, -257, 0),
    "strictly_behind_257": lambda: band(257, 1, 257),
    "200_back_and_more": lambda: band(700, -700, -199),
    "200_ahead_and_more": lambda: band(700, 200, 700),
    "window_back": lambda: band(700, -300, -100),
    "window_ahead": lambda: band(900, 256, 512),
    "window_with_itself": lambda: band(500, -70, 1),
    "short_rows": lambda: band(100, -40, -20),
    "nothing": lambda: block(200),
}


@pytest.fixture
def nan_workspace(mc, monkeypatch):
    monkeypatch.setattr(mc.ops, "_workspace",
                        lambda n, device: torch.full((n,), 255, dtype=torch.uint8, device=device) if n else None)


@pytest.mark.parametrize("name", list(LAYOUTS))
@pytest.mark.parametrize("dt,D", [(torch.bfloat16, 64), (torch.bfloat16, 128), (torch.float32, 64), (torch.bfloat16, 40)])
def test_spans_of_a_caller(mc, dev, nan_outputs, nan_workspace, dt, D, name):
    see = LAYOUTS[name]()
    S, B, H, Hkv = see.shape[0], 2, 2, 1
    spans = ref.spans_of(see).expand(B, S, 4).contiguous().to(dev)
    g = torch.Generator().manual_seed(S + D)
    q, k, v = ((torch.randn(B, n, S, D, generator=g) * 1.5).to(dt).to(dev) for n in (H, Hkv, Hkv))
    dout = torch.randn(B, S, H * D, generator=g).to(dt).to(dev)
    blind, unseen = (~see.any(1)).to(dev), (~see.any(0)).to(dev)
    q, dout = q.masked_fill(blind[:, None], math.nan), dout.masked_fill(blind[:, None], math.nan)
    k, v = (x.masked_fill(unseen[:, None], math.nan) for x in (k, v))
    for cap, slopes in ((None, None), (20.0, torch.tensor([0.25, 0.01], device=dev))):
        how = {"spans": spans, "cap": cap, "slopes": slopes}
        o, lse = mc.packed_attention_forward(q, k, v, **how)
        dq, dk, dv = mc.packed_attention_backward(q, k, v, o, lse, dout, **how)
        want = ref.attention(q, k, v, see.expand(B, S, S), D**-0.5, cap, slopes, dout)
        ref.check({"o": o, "lse": lse, "dq": dq, "dk": dk, "dv": dv}, want)
