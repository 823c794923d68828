"""Delta = sum_j P_j dP_j of bf16 queries that see few keys, whose gradients would
carry o's rounding if it were formed from o: whatever lies beside them in the row
(the matrix kernels, up to 256 keys a query), and for every head dim (the row
kernels, always).

Against 64 bits with the bounds of packed_reference.py, `exact` for such queries."""
import pytest
import torch

import packed_reference as ref

pytestmark = pytest.mark.gpu
FEW = 256  # keys


def inputs(B, H, Hkv, S, D, dev, std=1.5):
    g = torch.Generator().manual_seed(S + D + H)
    make = lambda *s, f=std: (torch.randn(*s, generator=g) * f).bfloat16().to(dev)  # noqa: E731
    return make(B, H, S, D), make(B, Hkv, S, D), make(B, Hkv, S, D, f=1.0), make(B, S, H * D, f=1.0)


def run(mc, q, k, v, dout, **how):
    o, lse = mc.packed_attention_forward(q, k, v, **how)
    dq, dk, dv = mc.packed_attention_backward(q, k, v, o, lse, dout, **how)
    return {"o": o, "lse": lse, "dq": dq, "dk": dk, "dv": dv}


def want_of(q, k, v, see, cap, dout, few):
    """ref.attention with exact bounds for queries of up to `few` keys. The gradients of the two sorts of queries are
    computed apart: a query's dq has one of them only, dk and dv are their sums, and so are the bounds."""
    B, H, S, D = q.shape
    whole = ref.attention(q, k, v, see, D**-0.5, cap, None, dout)
    sort = see.sum(-1, keepdim=True) <= few
    parts = [ref.attention(q, k, v, see & m, D**-0.5, cap, None, dout, x) for m, x in ((sort, True), (~sort, False))]
    return {**whole, **{n: tuple(a + b for a, b in zip(*(p[n] for p in parts))) for n in ("dq", "dk", "dv")}}


# documents' sizes in a row: short ones behind a long one in its last tile, and some that start inside a tile
ROWS = {"behind_300": [300, 4, 1, 30, 2, 400], "inside_a_tile": [700, 340, 280, 5, 300], "between": [270, 1, 270, 1, 1, 270],
        "many": [257, 255, 256, 1, 3, 258]}


@pytest.mark.parametrize("cap", [None, 20.0])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("name", list(ROWS))
def test_few_keys_beside_many(mc, dev, name, causal, D, cap):
    sizes = ROWS[name]
    S = sum(sizes)
    ids = torch.repeat_interleave(torch.arange(len(sizes), dtype=torch.int32), torch.tensor(sizes))
    q, k, v, dout = inputs(1, 2, 1, S, D, dev)
    see = ref.visible(S, ids, causal=causal)[None]
    got = run(mc, q, k, v, dout, spans=mc.attention_spans(ids[None].to(dev), causal=causal), cap=cap)
    ref.check(got, want_of(q, k, v, see, cap, dout, FEW))


@pytest.mark.parametrize("D", [8, 40, 96, 192, 256])
@pytest.mark.parametrize("cap", [None, 20.0])
def test_other_head_dims(mc, dev, D, cap):
    sizes = [40, 1, 4, 2, 1, 22]
    S = sum(sizes)
    ids = torch.repeat_interleave(torch.arange(len(sizes), dtype=torch.int32), torch.tensor(sizes))
    for causal in (True, False):
        q, k, v, dout = inputs(1, 4, 2, S, D, dev)
        see = ref.visible(S, ids, causal=causal)[None]
        got = run(mc, q, k, v, dout, spans=mc.attention_spans(ids[None].to(dev), causal=causal), cap=cap)
        ref.check(got, want_of(q, k, v, see, cap, dout, S))


@pytest.mark.parametrize("cap", [None, 50.0])
@pytest.mark.parametrize("D,first", [(64, 300), (128, 300), (40, 1), (96, 20), (256, 1)])
def test_documents_of_one_token_behind_a_long_one(mc, dev, D, first, cap):
    """P is 1 and dS nothing but what rounding leaves: dP twice, D u |dout| |v| each, u = 2^-24, P dP / P 2 u of it, and
    where dq is a difference of two sums 3 u more; dq is scale dS k, rounded."""
    B, H, Hkv, S = 1, 4, 2, first + 90
    q, k, v, dout = inputs(B, H, Hkv, S, D, dev, std=6.0)
    ids = torch.zeros(B, S, dtype=torch.int32)
    ids[:, first:] = torch.arange(1, S - first + 1, dtype=torch.int32)
    got = run(mc, q, k, v, dout, spans=mc.attention_spans(ids.to(dev)), cap=cap)
    rows = lambda x: x[:, :, first:].double().cpu()  # noqa: E731
    do = dout.view(B, S, H, D).transpose(1, 2)[:, :, first:].double().cpu()
    kk, vv = (rows(x).repeat_interleave(H // Hkv, 1) for x in (k, v))
    most = 2.0**-24 * (2 * D + 8) * (do.abs() * vv.abs()).sum(-1, keepdim=True) * D**-0.5  # scale |dS|
    assert (rows(got["dq"]).abs() <= most * kk.abs() * 1.01).all()
    sums = (most * rows(q).abs()).view(B, Hkv, H // Hkv, S - first, D).sum(2)
    assert (rows(got["dk"]).abs() <= sums * 1.01).all()
