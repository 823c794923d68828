"""A training step of a small decoder on packed documents, by the operators together:
scaled embedding, attention inside the documents, tied output projection, cross
entropy, back through all of them, the gradients' norm, clipping and AdamW.

In float32 against the same step in 64 bits on the CPU, gradient by autograd. A sum
of n terms is off by at most n u of the sum of their sizes, u = 2^-24, which for the
step's random signs is at most about sqrt(n) times the sum, n <= 512: 23; what later
stages do to an error they do to the value. The sums on the longest way have 160 keys
or queries (four times), 64 features (six), 301 logits (twice) and 480 tokens (once)
and one of 50 rounded functions: 2156 terms, so a gradient is off by at most
2156 * 23 u = 3e-3 of its norm.
"""
import math

import pytest
import torch

import packed_reference as ref

pytestmark = pytest.mark.gpu
OFF = 2156 * 23 * 2.0**-24
B, S, H, HKV, D, V, PAD = 3, 160, 4, 2, 16, 301, 0
E = H * D


def batch():
    g = torch.Generator().manual_seed(7)
    ids = torch.randint(1, V, (B, S), generator=g, dtype=torch.int32)
    ids[:, 5::3] = 11  # a frequent token
    docs = torch.zeros(B, S, dtype=torch.int32)
    prefix = torch.zeros(B, S, dtype=torch.uint8)
    for b, ends in enumerate(((40, 41, 150), (160,), (3, 90))):
        t = 0
        for n, end in enumerate(ends):
            docs[b, t:end] = n % 2
            prefix[b, t:t + (end - t) // 3] = 1
            t = end
        docs[b, t:] = -1
        ids[b, t:] = PAD
    targets = torch.roll(ids, -1, 1)
    targets[:, -1] = PAD
    targets[torch.roll(docs, -1, 1) != docs] = PAD
    return ids, docs, prefix, targets


def weights(dt=torch.float32):
    g = torch.Generator().manual_seed(8)
    make = lambda *s: (torch.randn(*s, generator=g) * s[-1] ** -0.5).to(dt)  # noqa: E731
    return {"table": make(V, E), "wq": make(E, E), "wk": make(HKV * D, E), "wv": make(HKV * D, E), "wo": make(E, E)}


def heads(x, n):
    return x.view(B, S, n, D).transpose(1, 2).contiguous()


def rows(x):
    return x.transpose(1, 2).reshape(B * S, -1)


def step(mc, w, ids, docs, prefix, targets, how):
    """(loss, gradients), every product of an activation with a weight by torch."""
    spans = mc.attention_spans(docs, prefix)
    x = mc.embedding_forward(w["table"], ids, scale=E**0.5, padding_id=PAD)
    flat = x.view(B * S, E)
    q, k, v = heads(flat @ w["wq"].t(), H), heads(flat @ w["wk"].t(), HKV), heads(flat @ w["wv"].t(), HKV)
    o, lse = mc.packed_attention_forward(q, k, v, spans=spans, **how)
    h = flat + o.view(B * S, E) @ w["wo"].t()
    logits = h @ w["table"].t()
    loss, stats = mc.cross_entropy_forward(logits, targets.view(-1), ignore_index=PAD)
    dlogits = mc.cross_entropy_backward(logits, targets.view(-1), stats, ignore_index=PAD)
    dtable, dh = dlogits.t() @ h, dlogits @ w["table"]
    grads = {"wo": dh.t() @ o.view(B * S, E)}
    dq, dk, dv = mc.packed_attention_backward(q, k, v, o, lse, (dh @ w["wo"]).view(B, S, E), spans=spans, **how)
    dx = dh.clone()
    for name, g in (("wq", dq), ("wk", dk), ("wv", dv)):
        grads[name] = rows(g).t() @ flat
        dx += rows(g) @ w[name]
    grads["table"] = mc.embedding_backward(dx.view(B, S, E), ids, V, scale=E**0.5, padding_id=PAD, dtable=dtable)
    return loss, grads


def step64(w, ids, docs, prefix, targets, cap, slopes):
    see = torch.stack([ref.visible(S, docs[b].tolist(), prefix[b].tolist()) for b in range(B)])[:, None]
    w = {n: t.double().requires_grad_() for n, t in w.items()}
    x = (w["table"][ids.long()] * E**0.5).masked_fill((ids == PAD)[..., None], 0.0)
    q, k, v = (((x @ w[n].t()).view(B, S, -1, D)).transpose(1, 2) for n in ("wq", "wk", "wv"))
    k, v = k.repeat_interleave(H // HKV, 1), v.repeat_interleave(H // HKV, 1)
    s = q @ k.transpose(2, 3) * D**-0.5
    if cap:
        s = cap * torch.tanh(s / cap)
    if slopes is not None:
        at = torch.arange(S)
        s = s - slopes.double()[:, None, None] * (at[:, None] - at).abs()
    # a row that sees nothing: any finite softmax, then all of it masked
    p = torch.softmax(s.masked_fill(~see & see.any(-1, keepdim=True), -math.inf), -1) * see
    h = x + (p @ v).transpose(1, 2).reshape(B, S, E) @ w["wo"].t()
    loss = torch.nn.functional.cross_entropy((h @ w["table"].t()).view(-1, V), targets.long().view(-1), ignore_index=PAD)
    loss.backward()
    return loss.item(), {n: t.grad for n, t in w.items()}


@pytest.mark.parametrize("cap,bias", [(None, False), (5.0, False), (None, True), (5.0, True)])
def test_step_against_64_bits(mc, dev, cap, bias):
    ids, docs, prefix, targets = batch()
    w = weights()
    slopes = torch.tensor([0.5, 0.25, 0.125, 0.0625]) if bias else None
    want_loss, want = step64(w, ids, docs, prefix, targets, cap, slopes)
    there = {n: t.to(dev) for n, t in w.items()}
    how = {"cap": cap, "slopes": None if slopes is None else slopes.to(dev)}
    loss, grads = step(mc, there, ids.to(dev), docs.to(dev), prefix.to(dev), targets.to(dev).to(torch.uint32), how)
    assert abs(loss.item() - want_loss) <= OFF * abs(want_loss)
    for n in want:
        off = (grads[n].cpu().double() - want[n]).norm() / want[n].norm()
        assert off <= OFF, n
    total = math.sqrt(sum(float(g.norm()) ** 2 for g in want.values()))
    names = list(w)
    norm, scale = mc.gradient_norm([grads[n] for n in names], 0.5 * total)
    assert abs(norm.item() - total) <= 2 * OFF * total
    # clipped by the optimizer as it reads, or beforehand
    one, two = ([there[n].clone() for n in names] for _ in range(2))
    zeros = lambda: [torch.zeros_like(t) for t in one]  # noqa: E731
    mc.adamw_step(one, [grads[n] for n in names], zeros(), zeros(), 1, lr=1e-2, grad_scale=scale)
    clipped = [torch.empty_like(grads[n]) for n in names]
    mc.clip_gradients([grads[n] for n in names], 0.5 * total, outs=clipped)
    mc.adamw_step(two, clipped, zeros(), zeros(), 1, lr=1e-2)
    for a, b, n in zip(one, two, names):
        assert torch.equal(a, b) and not torch.equal(a, there[n])
    after, _ = step64({n: t.cpu() for n, t in zip(names, one)}, ids, docs, prefix, targets, cap, slopes)
    assert math.isfinite(after)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_step_in_a_graph(mc, dev, dtype):
    """The operators alone, captured together and replayed between eager runs on other weights."""
    ids, docs, prefix, _ = (t.to(dev) for t in batch())
    w = {n: t.to(dev) for n, t in weights(dtype).items()}
    slopes = torch.tensor([0.5, 0.25, 0.125, 0.0625], device=dev)
    dout = torch.randn(B, S, E, generator=torch.Generator().manual_seed(9)).to(dtype).to(dev)
    how = {"cap": 5.0, "slopes": slopes}
    out = [torch.zeros(V, E, device=dev), torch.zeros(B, S, E, dtype=dtype, device=dev)]

    def run(table):
        spans = mc.attention_spans(docs, prefix)
        x = mc.embedding_forward(table, ids, scale=E**0.5, padding_id=PAD)
        q = heads(x, H)
        k, v = q[:, :HKV].contiguous(), q[:, HKV:].contiguous()
        o, lse = mc.packed_attention_forward(q, k, v, spans=spans, **how)
        dq, dk, dv = mc.packed_attention_backward(q, k, v, o, lse, dout, spans=spans, **how)
        dx = rows(dq + torch.cat([dk, dv], 1)).view(B, S, E).contiguous()
        dtable = mc.embedding_backward(dx, ids, V, scale=E**0.5, padding_id=PAD)
        norm, scale = mc.clip_gradients([dtable, dx], 1.0, outs=out)
        return o, dx, dtable, norm, scale

    run(w["table"])
    torch.cuda.synchronize()
    table = w["table"].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run(table)
    for seed in range(3):
        table.copy_(torch.randn(V, E, generator=torch.Generator().manual_seed(seed)).to(dtype))
        want = [t.clone() for t in run(table.clone())] + [t.clone() for t in out]
        for t in out:
            t.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(bool(torch.isfinite(t.float()).all()) for t in want)
        for got, eager in zip([*captured, *out], want):
            assert torch.equal(got, eager)
