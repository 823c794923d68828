"""Attention over packed rows, forward and backward, against 64 bits with the bounds
that packed_reference.py derives."""
import math
import random

import pytest
import torch

import packed_reference as ref

pytestmark = pytest.mark.gpu


def layout(kind, B, S, seed=0):
    """(documents, prefix) of a kind of row, or None for either."""
    rng = random.Random(1000 * S + seed)
    ids, flags = torch.zeros(B, S, dtype=torch.int32), torch.zeros(B, S, dtype=torch.uint8)
    for b in range(B):
        t, n = 0, 0
        while t < S:
            size = {"short": rng.randrange(1, 20), "long": rng.randrange(1, S + 1)}.get(kind, rng.randrange(1, S // 2 + 2))
            end = min(S, t + size)
            ids[b, t:end] = -1 if kind == "holes" and rng.random() < 0.4 else n % 3
            if kind == "flags":
                flags[b, t:end] = (torch.rand(end - t, generator=torch.Generator().manual_seed(t)) < 0.8).to(torch.uint8)
            else:
                flags[b, t:t + rng.randrange(0, end - t + 1)] = 1
            t, n = end, n + 1
    if kind == "empty":
        ids[:] = -1
        ids[0, S // 2:] = 4
    if kind == "tail":
        ids[:, S - S // 3:] = -7
    return ids, flags


def inputs(dt, B, H, Hkv, S, D, dev, std=1.5):
    g = torch.Generator().manual_seed(S + D + H)
    make = lambda *s, f=std: (torch.randn(*s, generator=g) * f).to(dt).to(dev)  # noqa: E731
    return make(B, H, S, D), make(B, Hkv, S, D), make(B, Hkv, S, D, f=1.0), make(B, S, H * D, f=1.0)


def slopes_of(H, dev, sign=1.0):
    return torch.tensor([sign * 2.0 ** (-8.0 * (h + 1) / H) for h in range(H)], device=dev)


def run(mc, q, k, v, dout, **how):
    o, lse = mc.packed_attention_forward(q, k, v, **how)
    dq, dk, dv = mc.packed_attention_backward(q, k, v, o, lse, dout, **how)
    return {"o": o, "lse": lse, "dq": dq, "dk": dk, "dv": dv}


def compare(mc, dev, dt, B, H, Hkv, S, D, kind, cap=None, bias=False, causal=True, prefix=False, std=1.5, scale=None):
    q, k, v, dout = inputs(dt, B, H, Hkv, S, D, dev, std)
    slopes = slopes_of(H, dev) if bias else None
    how = {"cap": cap, "slopes": slopes, "scale": scale}
    if kind is None:
        see = ref.visible(S, causal=causal).expand(B, S, S)
        how["causal"] = causal
    else:
        ids, flags = layout(kind, B, S)
        how["spans"] = mc.attention_spans(ids.to(dev), flags.to(dev) if prefix else None, causal=causal)
        see = torch.stack([ref.visible(S, ids[b], flags[b] if prefix else None, causal) for b in range(B)])
    # the bf16 tiles form Delta from P and dP where a tile of queries sees up to 256 keys
    exact = dt == torch.bfloat16 and D in (64, 128) and S <= 256
    want = ref.attention(q, k, v, see, D**-0.5 if scale is None else scale, cap, slopes, dout, exact)
    ref.check(run(mc, q, k, v, dout, **how), want)


def test_packed_documents_of_a_long_row(mc, dev):
    """Tiles of queries on both sides of the 256 keys up to which Delta is formed from P and dP."""
    S, D = 1500, 64
    q, k, v, dout = inputs(torch.bfloat16, 1, 2, 1, S, D, dev)
    ids = torch.zeros(1, S, dtype=torch.int32)
    ids[0, 700:] = 1
    ids[0, 1000:1256] = 2
    for causal in (True, False):
        see = ref.visible(S, ids[0], causal=causal)[None]
        got = run(mc, q, k, v, dout, spans=mc.attention_spans(ids.to(dev), causal=causal), cap=30.0)
        ref.check(got, ref.attention(q, k, v, see, D**-0.5, 30.0, None, dout))
        exact = ref.attention(q, k, v, see, D**-0.5, 30.0, None, dout, True)
        span = {"dq": got["dq"][:, :, 1024:1152]}  # a tile inside the third document
        ref.check(span, {n: (x[:, :, 1024:1152], e[:, :, 1024:1152]) for n, (x, e) in exact.items() if n == "dq"})


@pytest.mark.parametrize("S", [1, 2, 5, 63, 64, 65, 127, 128, 130, 200, 333, 513])
@pytest.mark.parametrize("D", [64, 128])
def test_bf16_lengths(mc, dev, nan_outputs, D, S):
    compare(mc, dev, torch.bfloat16, 2, 4, 2, S, D, None, cap=20.0)
    compare(mc, dev, torch.bfloat16, 2, 4, 2, S, D, "tail", bias=True)


@pytest.mark.parametrize("cap,bias", [(None, False), (5.0, False), (None, True), (50.0, True)])
@pytest.mark.parametrize("kind,causal,prefix", [
    (None, True, False), (None, False, False), ("mid", True, False), ("mid", False, False), ("short", True, False),
    ("short", False, False), ("holes", True, True), ("holes", False, False), ("long", True, True), ("flags", True, True),
    ("empty", True, False), ("empty", False, False), ("tail", True, True)])
@pytest.mark.parametrize("dt,D,S", [(torch.bfloat16, 128, 300), (torch.bfloat16, 64, 261), (torch.float32, 64, 150),
                                    (torch.float32, 36, 77), (torch.bfloat16, 40, 70), (torch.float32, 33, 50)])
def test_masks_and_scores(mc, dev, nan_outputs, dt, D, S, kind, causal, prefix, cap, bias):
    compare(mc, dev, dt, 2, 4, 2, S, D, kind, cap, bias, causal, prefix)


@pytest.mark.parametrize("dt,H,Hkv,S,D", [
    (torch.bfloat16, 6, 1, 200, 128), (torch.bfloat16, 3, 3, 140, 64), (torch.bfloat16, 7, 1, 129, 64),
    (torch.float32, 6, 1, 131, 128), (torch.float32, 3, 3, 70, 32), (torch.float32, 4, 1, 5, 64),
    (torch.float32, 2, 2, 3, 32), (torch.bfloat16, 2, 1, 33, 256), (torch.float32, 2, 1, 40, 160),
    (torch.float32, 4, 4, 1, 128)])
def test_heads_and_dims(mc, dev, nan_outputs, dt, H, Hkv, S, D):
    for cap, bias in ((30.0, False), (None, True)):
        compare(mc, dev, dt, 1, H, Hkv, S, D, "holes", cap, bias, True, True)


@pytest.mark.parametrize("dt,D", [(torch.bfloat16, 128), (torch.bfloat16, 64), (torch.float32, 64), (torch.bfloat16, 24)])
@pytest.mark.parametrize("std,cap,scale", [(0.05, 0.01, None), (6.0, 2.0, None), (6.0, 1000.0, None), (1.5, 50.0, 2.0),
                                           (12.0, None, 0.05), (0.0, 20.0, None)])
def test_ranges_of_scores(mc, dev, dt, D, std, cap, scale):
    """Scores far below and far above the cap, the least and the largest cap, scores of 0."""
    compare(mc, dev, dt, 1, 2, 1, 190, D, "mid", cap=cap, std=std, scale=scale)


@pytest.mark.parametrize("dt,D", [(torch.bfloat16, 64), (torch.float32, 32)])
def test_slopes_of_every_sign(mc, dev, dt, D):
    q, k, v, dout = inputs(dt, 1, 3, 1, 150, D, dev)
    slopes = torch.tensor([0.0, -0.25, 3.0], device=dev)
    see = ref.visible(150, causal=False)[None]
    want = ref.attention(q, k, v, see, D**-0.5, None, slopes, dout)
    ref.check(run(mc, q, k, v, dout, slopes=slopes), want)


def test_plain_rows_agree_with_attention(mc, dev):
    """Without any of it, causal rows are those of attention_forward (to the rounding of both)."""
    for dt, D in ((torch.bfloat16, 128), (torch.float32, 64)):
        q, k, v, dout = inputs(dt, 2, 4, 2, 257, D, dev)
        see = ref.visible(257).expand(2, 257, 257)
        want = ref.attention(q, k, v, see, D**-0.5, None, None, dout)
        o, lse = mc.attention_forward(q, k, v, causal=True)
        ref.check({"o": o, "lse": lse}, want)
        ref.check(run(mc, q, k, v, dout, causal=True), want)
        ones = torch.zeros(2, 257, dtype=torch.int32, device=dev)
        same = run(mc, q, k, v, dout, spans=mc.attention_spans(ones))
        assert all(torch.equal(x, y) for x, y in zip(same.values(), run(mc, q, k, v, dout, causal=True).values()))


def test_gradients_against_differences(mc, dev):
    """The kernels' gradients along a direction against differences of the 64-bit forward: those are off by 1e-16 / h
    of the loss and by h^2 of its third derivatives, far below the gradients' own bounds."""
    B, H, Hkv, S, D = 1, 2, 1, 45, 32
    q, k, v, dout = inputs(torch.float32, B, H, Hkv, S, D, dev, std=0.7)
    ids, flags = layout("mid", B, S)
    see = ref.visible(S, ids[0], flags[0])[None]
    slopes = slopes_of(H, dev)
    got = run(mc, q, k, v, dout, spans=mc.attention_spans(ids.to(dev), flags.to(dev)), cap=3.0, slopes=slopes)
    bounds = ref.attention(q, k, v, see, D**-0.5, 3.0, slopes, dout)
    h = 1e-5
    for name in ("dq", "dk", "dv"):
        x = {"dq": q.double(), "dk": k.double(), "dv": v.double()}
        w = torch.randn(x[name].shape, generator=torch.Generator().manual_seed(9)).to(dev).double()

        def loss(t):
            y = {**x, name: t}
            o = ref.attention(y["dq"], y["dk"], y["dv"], see, D**-0.5, 3.0, slopes)["o"][0]
            return float((o * dout.double()).sum())

        slope = (loss(x[name] + h * w) - loss(x[name] - h * w)) / (2 * h)
        off = abs(slope - float((got[name].double() * w).sum()))
        assert off <= float((bounds[name][1] * w.abs()).sum()) + 1e-6 * abs(slope) + 1e-8, name


SPECIAL = [math.nan, math.inf, -math.inf]


@pytest.mark.parametrize("cap", [5.0, 50.0, 52.5, 1000.0])
@pytest.mark.parametrize("dt,D,S", [(torch.bfloat16, 128, 300), (torch.bfloat16, 64, 70), (torch.float32, 64, 90)])
def test_scores_at_the_cap(mc, dev, dt, D, S, cap):
    """Rows whose scores are all minus the cap, all the cap, and both: no sum leaves float32."""
    q, k, v, dout = inputs(dt, 1, 3, 1, S, D, dev)
    k = torch.full_like(k, 4.0)
    k[:, :, 1::2] *= -1.0
    q = torch.full_like(q, 4.0)
    ids = torch.zeros(1, S, dtype=torch.int32)
    # the second head sees one sign only: tokens of one sign are documents of their own
    ids[0] = torch.arange(S) % 2 if S < 100 else 0
    q[:, 1] *= -1.0
    how = {"spans": mc.attention_spans(ids.to(dev)), "cap": cap, "scale": 50.0}
    got = run(mc, q, k, v, dout, **how)
    want = ref.attention(q, k, v, ref.visible(S, ids[0].tolist())[None], 50.0, cap, None, dout)
    ref.check(got, want)


@pytest.mark.parametrize("cap", [None, 50.0])
@pytest.mark.parametrize("dt,D", [(torch.bfloat16, 64), (torch.bfloat16, 128)])
def test_documents_of_one_token(mc, dev, dt, D, cap):
    """P is 1 and dS nothing but what rounding leaves: with u = 2^-24, P dP / P is off by 2 u of dP, and dP, summed in
    the same products in both kernels but for their order, by D u |dout| |v| each time; dq is scale dS k, rounded."""
    B, H, Hkv, S = 2, 4, 2, 130
    q, k, v, dout = inputs(dt, B, H, Hkv, S, D, dev, std=6.0)
    spans = mc.attention_spans((torch.arange(S, dtype=torch.int32) % 2).repeat(B, 1).to(dev))
    got = run(mc, q, k, v, dout, spans=spans, cap=cap)
    rows = lambda x: x.double().cpu()  # noqa: E731
    do = rows(dout).view(B, S, H, D).transpose(1, 2)
    kk, vv = (rows(x).repeat_interleave(H // Hkv, 1) for x in (k, v))
    most = 2.0**-24 * (2 * D + 8) * (do.abs() * vv.abs()).sum(-1) * D**-0.5  # scale |dS|
    assert torch.equal(got["o"].view(B, S, H, D).transpose(1, 2), v.repeat_interleave(H // Hkv, 1))
    assert (rows(got["dq"]).abs() <= most[..., None] * kk.abs() * 1.01).all()
    sum_of = lambda x: x.view(B, Hkv, H // Hkv, S, -1).sum(2)  # noqa: E731
    assert (rows(got["dk"]).abs() <= sum_of(most[..., None] * rows(q).abs()) * 1.01).all()
    assert (rows(got["dv"]) - sum_of(do)).abs().le(2.0**-8 * sum_of(do.abs()) * 1.01).all()


@pytest.mark.parametrize("cap", [None, 20.0])
@pytest.mark.parametrize("dt,D,S", [(torch.bfloat16, 128, 300), (torch.bfloat16, 64, 200), (torch.float32, 64, 150),
                                    (torch.float32, 128, 70), (torch.bfloat16, 40, 60), (torch.float32, 33, 40),
                                    (torch.bfloat16, 128, 100), (torch.bfloat16, 64, 128)])
def test_what_padding_holds(mc, dev, dt, D, S, cap):
    """Infinities and NaN in every tensor's padding change no bit of any result."""
    B, H, Hkv = 2, 4, 2
    q, k, v, dout = inputs(dt, B, H, Hkv, S, D, dev)
    ids, _ = layout("holes", B, S, seed=1)
    pad = (ids < 0).to(dev)
    assert pad.any() and not pad.all()
    spans = mc.attention_spans(ids.to(dev))
    clean = run(mc, q, k, v, dout, spans=spans, cap=cap)
    junk = torch.tensor(SPECIAL, device=dev)[torch.arange(S * D, device=dev) % 3].view(S, D).to(dt)
    bad = [torch.where(pad[:, None, :, None], junk, x) for x in (q, k, v)]
    bad_dout = torch.where(pad[:, :, None], junk.repeat(1, H), dout)
    dirty = run(mc, *bad, bad_dout, spans=spans, cap=cap)
    for name in clean:
        assert torch.equal(clean[name], dirty[name]), name
    assert (dirty["o"][pad] == 0).all() and (dirty["dq"].transpose(1, 2)[pad] == 0).all()
    assert (dirty["dk"].transpose(1, 2)[pad] == 0).all() and (dirty["dv"].transpose(1, 2)[pad] == 0).all()
    assert (dirty["lse"].transpose(1, 2)[pad] == -math.inf).all()


@pytest.mark.parametrize("which", ["q", "k", "v", "dout"])
@pytest.mark.parametrize("value", SPECIAL)
@pytest.mark.parametrize("dt,D,S", [(torch.bfloat16, 128, 300), (torch.bfloat16, 64, 140), (torch.float32, 64, 130),
                                    (torch.bfloat16, 40, 50), (torch.bfloat16, 128, 128), (torch.bfloat16, 64, 90)])
def test_one_document_that_is_not_finite(mc, dev, dt, D, S, which, value):
    """A NaN or an infinity in one document leaves the others' results as they are, and reaches its own."""
    B, H, Hkv = 1, 2, 1
    q, k, v, dout = inputs(dt, B, H, Hkv, S, D, dev)
    cuts = [0, S // 4 + 3, S // 2 + 1, S]
    ids = torch.zeros(1, S, dtype=torch.int32)
    for n in range(3):
        ids[0, cuts[n]:cuts[n + 1]] = n
    spans = mc.attention_spans(ids.to(dev))
    for cap in (None, 20.0):
        clean = run(mc, q, k, v, dout, spans=spans, cap=cap)
        t = cuts[1] + 2  # in the middle document
        x = {"q": q.clone(), "k": k.clone(), "v": v.clone(), "dout": dout.clone()}
        if which == "dout":
            x[which][0, t, 3] = value
        else:
            x[which][0, 0, t, 3] = value
        dirty = run(mc, x["q"], x["k"], x["v"], x["dout"], spans=spans, cap=cap)
        other = torch.ones(S, dtype=torch.bool, device=dev)
        other[cuts[1]:cuts[2]] = False
        for name in clean:
            a, b = (y[0] if name == "o" else y[0].transpose(0, 1) for y in (clean[name], dirty[name]))
            assert torch.equal(a[other], b[other]), (name, cap)
        # earlier tokens of the document do not see it
        assert torch.equal(clean["o"][0, :t], dirty["o"][0, :t])
        if which == "v":  # only its own column of the rows that see it
            o = dirty["o"].view(S, H, D)
            assert not o[t:cuts[2], :, 3].isfinite().any()
            assert torch.equal(o[..., 4:], clean["o"].view(S, H, D)[..., 4:])
        if value != value:  # NaN reaches everything that depends on it
            if which == "k":
                assert dirty["o"][0, t:cuts[2]].isnan().all()
            if which == "q":
                assert dirty["o"].view(S, H, D)[t, 0].isnan().all() and dirty["dk"][0, 0, cuts[1]:t + 1].isnan().all()
            if which == "dout":
                assert dirty["dq"][0, 0, t].isnan().all() and dirty["dv"][0, 0, cuts[1]:t + 1, 3].isnan().all()


@pytest.mark.parametrize("S", [1, 2, 3, 63, 64, 65, 255, 257, 1000, 4095, 4096, 4097, 9001])
@pytest.mark.parametrize("kind", ["mid", "short", "holes", "flags", "tail", "empty"])
def test_spans(mc, dev, kind, S):
    """Token by token; short rows against the matrix of who sees whom, long ones document by document."""
    ids, flags = layout(kind, 2, S)
    for causal, prefix in ((True, False), (True, True), (False, False)):
        got = mc.attention_spans(ids.to(dev), flags.to(dev) if prefix else None, causal=causal).cpu()
        if S <= 257:
            for b in range(2):
                want = ref.spans_of(ref.visible(S, ids[b], flags[b] if prefix else None, causal))
                assert torch.equal(got[b], want)
            continue
        for b in range(2):
            t = 0
            while t < S:
                rest = (ids[b, t:] != ids[b, t]).nonzero()
                end = t + int(rest[0]) if len(rest) else S
                want = torch.zeros(end - t, 4, dtype=torch.int32)
                if ids[b, t] >= 0:
                    at = torch.arange(t, end, dtype=torch.int32)
                    zeros = (flags[b, t:end] == 0).nonzero()
                    p = (t + int(zeros[0]) if len(zeros) else end) if prefix else t
                    want[:, 0], want[:, 1] = t, at.add(1).clamp(min=p) if causal else end
                    want[:, 2], want[:, 3] = torch.where(at < p, t, at) if causal else t, end
                assert torch.equal(got[b, t:end], want)
                t = end
    only = mc.attention_spans(prefix=flags.to(dev)).cpu()
    if S <= 257:
        assert torch.equal(only[0], ref.spans_of(ref.visible(S, None, flags[0])))
        assert torch.equal(mc.attention_spans(prefix=flags.bool().to(dev)).cpu(), only)


@pytest.mark.parametrize("S", [32640, 32800])
def test_long_row(mc, dev, S):
    """Past 2^31 bytes of one head's dS^T (S > 32640) the dQ pass forms S and dP again; documents keep the reference
    small."""
    D = 64
    for cap, bias in ((20.0, False), (None, True)):
        q, k, v, dout = inputs(torch.bfloat16, 1, 2, 1, S, D, dev)
        slopes = slopes_of(2, dev) if bias else None
        ids = torch.empty(1, S, dtype=torch.int32)
        cuts = list(range(0, S, 410)) + [S]
        for n, (a, b) in enumerate(zip(cuts, cuts[1:])):
            ids[0, a:b] = -1 if n % 9 == 5 else n
        spans = mc.attention_spans(ids.to(dev))
        junk = (ids < 0).to(dev)
        q, k, v = (torch.where(junk[:, None, :, None], math.nan, x) for x in (q, k, v))
        got = run(mc, q, k, v, dout, spans=spans, cap=cap, slopes=slopes)
        for n in (0, 1, 4, 6, 40, len(cuts) - 2):
            a, b = cuts[n], cuts[n + 1]
            part = [x[:, :, a:b].contiguous() for x in (q, k, v)]
            want = ref.attention(*part, ref.visible(b - a)[None], D**-0.5, cap, slopes, dout[:, a:b].contiguous())
            mine = {n: x[:, a:b] if n == "o" else x[:, :, a:b] for n, x in got.items()}
            ref.check(mine, want)
        assert (got["dq"].transpose(1, 2)[junk] == 0).all()


@pytest.mark.parametrize("dt,D", [(torch.bfloat16, 128), (torch.float32, 64), (torch.bfloat16, 40)])
def test_reproducible_on_streams_and_in_graphs(mc, dev, dt, D):
    B, H, Hkv, S = 2, 4, 2, 200
    q, k, v, dout = inputs(dt, B, H, Hkv, S, D, dev)
    ids, flags = (x.to(dev) for x in layout("holes", B, S))

    def all_of_it():
        how = {"spans": mc.attention_spans(ids, flags), "cap": 20.0, "slopes": slopes}
        return run(mc, q, k, v, dout, **how)

    slopes = slopes_of(H, dev)
    first = {n: x.clone() for n, x in all_of_it().items()}
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        again = all_of_it()
    side.synchronize()
    assert all(torch.equal(first[n], again[n]) for n in first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = all_of_it()
    for turn in range(3):
        for x in out.values():
            x.fill_(math.nan)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(first[n], out[n]) for n in first)
        run(mc, q[:1, :, :64].contiguous(), k[:1, :, :64].contiguous(), v[:1, :, :64].contiguous(),
            dout[:1, :64].contiguous(), causal=True)


def test_without_lse(mc, dev):
    q, k, v, _ = inputs(torch.bfloat16, 1, 2, 1, 100, 64, dev)
    o, lse = mc.packed_attention_forward(q, k, v, causal=True, cap=10.0, save_lse=False)
    assert lse is None and torch.equal(o, mc.packed_attention_forward(q, k, v, causal=True, cap=10.0)[0])
