"""What a training step on packed documents needs beside the decoder layer's own
operators, as it is measured: the scaled embedding of the tokens and its gradient
summed by token, attention over rows of several documents with capped scores, a
bias by distance and prefixes that see themselves whole, forward and backward, and
the gradients' global norm with the clipping by it.

`run` computes them in elementary torch operations, or, where `own` is true, with
the framework's calls. Sizes: the decoder shapes that the tests and the benchmark
run, and odd and ragged ones of the same ranges.
"""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "bf16": 2}
VOCAB = 151936
PAD = 0  # the padding token's id


def listed():
    return [
        # One short prompt under capped scores: the smallest call, latency.
        {"name": "attention_prompt_bf16", "kind": "attention", "train": False, "dtype": "bf16", "B": 1, "H": 14,
         "Hkv": 2, "S": 65, "D": 64, "cap": 50.0, "bias": False, "documents": False, "prefix": False},
        # Scoring whole rows with capped scores.
        {"name": "attention_capped_bf16", "kind": "attention", "train": False, "dtype": "bf16", "B": 4, "H": 12,
         "Hkv": 2, "S": 2048, "D": 128, "cap": 50.0, "bias": False, "documents": False, "prefix": False},
        # A float32 step on rows of an arbitrary length that hold several documents.
        {"name": "attention_documents_f32", "kind": "attention", "train": True, "dtype": "f32", "B": 4, "H": 12,
         "Hkv": 2, "S": 509, "D": 64, "cap": 30.0, "bias": False, "documents": True, "prefix": False},
        # Prompts that see themselves whole, answers behind them, a bias by distance.
        {"name": "attention_prefix_bf16", "kind": "attention", "train": True, "dtype": "bf16", "B": 3, "H": 14,
         "Hkv": 2, "S": 1021, "D": 64, "cap": 0.0, "bias": True, "documents": True, "prefix": True},
        # A training step on packed documents.
        {"name": "attention_documents_bf16", "kind": "attention", "train": True, "dtype": "bf16", "B": 8, "H": 12,
         "Hkv": 2, "S": 2048, "D": 128, "cap": 0.0, "bias": False, "documents": True, "prefix": False},
        # The largest step: long rows, every head, capped scores, one document a row.
        {"name": "attention_long_bf16", "kind": "attention", "train": True, "dtype": "bf16", "B": 4, "H": 28,
         "Hkv": 4, "S": 4096, "D": 128, "cap": 50.0, "bias": False, "documents": False, "prefix": False},
        # The adapters of one decoder layer.
        {"name": "clip_layer_f32", "kind": "clip", "dtype": "f32", "layers": 1, "hidden": 1536, "mlp": 8960,
         "kv": 256, "rank": 16},
        # The adapters of a whole model: 392 tensors.
        {"name": "clip_adapters_f32", "kind": "clip", "dtype": "f32", "layers": 28, "hidden": 1536, "mlp": 8960,
         "kv": 256, "rank": 16},
        # Whole weights of six layers, bfloat16 gradients to the float32 ones that the optimizer takes.
        {"name": "clip_weights_bf16", "kind": "clip", "dtype": "bf16", "layers": 6, "hidden": 1536, "mlp": 8960,
         "kv": 256, "rank": 0},
        # The embedding of one prompt.
        {"name": "embedding_prompt_bf16", "kind": "embedding", "train": False, "dtype": "bf16", "B": 1, "S": 777,
         "V": VOCAB, "D": 1536, "scaled": True},
        # A float32 table of odd rows and its gradient.
        {"name": "embedding_train_f32", "kind": "embedding", "train": True, "dtype": "f32", "B": 4, "S": 509,
         "V": 50257, "D": 893, "scaled": False},
        # A training step's embedding of 16384 tokens and the gradient of the whole table.
        {"name": "embedding_train_bf16", "kind": "embedding", "train": True, "dtype": "bf16", "B": 8, "S": 2048,
         "V": VOCAB, "D": 1536, "scaled": True},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "clip", "embedding"])
    dtype = rng.choice(["f32", "bf16", "bf16"])
    if kind == "attention":
        H, Hkv = rng.choice([(12, 2), (14, 2), (28, 4), (8, 8), (4, 1), (9, 3)])
        D = rng.choice([64, 128] if dtype == "bf16" else [32, 64, 128])
        S = _log_int(rng, 2, 4096)
        most = 4 * 28 * 4096 * 4096 * 128 // (1 if dtype == "bf16" else 16)
        S = min(S, int(math.sqrt(most / (H * D))))
        B = min(_log_int(rng, 1, 16), max(1, most // (H * D * S * S)))
        return {"kind": kind, "train": rng.random() < 0.7, "dtype": dtype, "B": B, "H": H, "Hkv": Hkv, "S": S, "D": D,
                "cap": rng.choice([0.0, 20.0, 50.0]), "bias": rng.random() < 0.35, "documents": rng.random() < 0.6,
                "prefix": rng.random() < 0.35}
    if kind == "clip":
        rank = rng.choice([0, 8, 16, 64])
        hidden, mlp, kv = rng.choice([(896, 4864, 128), (1536, 8960, 256), (2048, 5632, 256), (1001, 2003, 77)])
        return {"kind": kind, "dtype": dtype, "layers": _log_int(rng, 1, 3 if rank == 0 else 40), "hidden": hidden,
                "mlp": mlp, "kv": kv, "rank": rank}
    B = rng.choice([1, 2, 4, 8])
    V = rng.choice([_log_int(rng, 1000, VOCAB), VOCAB])
    D = rng.choice([512, 768, 896, 1001, 1280, 1536]) if dtype == "bf16" else rng.choice([384, 893, 896])
    return {"kind": kind, "train": rng.random() < 0.6, "dtype": dtype, "B": B, "S": _log_int(rng, 1, 16384 // B),
            "V": V, "D": D, "scaled": rng.random() < 0.5}


# ------------------------------------------------------------------ layouts, alike for every seed
def _documents(case):
    """For each row its documents [(first, end, prompt tokens)] in order; what is behind the last is padding."""
    B, S = case["B"], case["S"]
    rng = random.Random(7919 * B + S)
    rows = []
    for b in range(B):
        # every second row ends in padding; without documents a row is one document to its end
        end = S - (rng.randrange(0, S // 8 + 1) if case["documents"] and b % 2 else 0)
        row, at = [], 0
        while at < end:
            n = min(end - at, _log_int(rng, max(1, S // 32), max(1, S // 2))) if case["documents"] else end
            row.append((at, at + n, rng.randrange(0, n // 2 + 1) if case["prefix"] else 0))
            at += n
        rows.append(row)
    return rows


def _pairs(case):
    """Visible (query, key) pairs of one head over the batch."""
    return sum((e - s) * (e - s + 1) // 2 + p * (p - 1) // 2 for row in _documents(case) for s, e, p in row)


def _shapes(case):
    """The gradients' shapes: A [K, r] and B [r, N] of each projection, or its weight [N, K]."""
    h, m, kv, r = case["hidden"], case["mlp"], case["kv"], case["rank"]
    layer = [(h, h), (h, kv), (h, kv), (h, h), (h, m), (h, m), (m, h)]  # q, k, v, o, gate, up, down as (K, N)
    one = [s for K, N in layer for s in ([(K, r), (r, N)] if r else [(N, K)])]
    return one * case["layers"]


def _spans(lengths, unit):
    """[(start, length)] in a flat buffer in which each tensor starts at a multiple of `unit`; its length."""
    got, at = [], 0
    for n in lengths:
        got.append((at, n))
        at += -(-n // unit) * unit
    return got, at


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, dtype=dtype):
        return torch.empty(shape, dtype=dtype, device="cuda").normal_(0.0, std, generator=g)

    s = {"case": case}
    if case["kind"] == "attention":
        B, H, Hkv, S, D = (case[k] for k in ("B", "H", "Hkv", "S", "D"))
        # scores of a standard deviation of 4: a trained model's rows are far from uniform
        s["q"], s["k"], s["v"] = normal(B, H, S, D, std=2.0), normal(B, Hkv, S, D, std=2.0), normal(B, Hkv, S, D)
        if case["train"]:
            s["dout"] = normal(B, S, H * D, std=0.01)
        rows = _documents(case)
        if case["documents"]:
            ids = torch.full((B, S), -1, dtype=torch.int32)
            for b, row in enumerate(rows):
                for n, (start, end, _) in enumerate(row):
                    ids[b, start:end] = n
            s["documents"] = ids.cuda()
        if case["prefix"]:
            flags = torch.zeros((B, S), dtype=torch.uint8)
            for b, row in enumerate(rows):
                for start, _, prompt in row:
                    flags[b, start:start + prompt] = 1
            s["prefix"] = flags.cuda()
        if case["bias"]:  # a geometric sequence over the heads
            s["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)], device="cuda")
        return s
    if case["kind"] == "clip":
        shapes = _shapes(case)
        n = sum(a * b for a, b in shapes)
        # gradients of a norm around 3, so that clipping to 1 has work to do
        s["grads"] = [normal(*shape, std=3.0 / math.sqrt(n)) for shape in shapes]
        spans, total = _spans([a * b for a, b in shapes], 64)
        s["flat"] = torch.zeros(total, dtype=torch.float32, device="cuda")
        s["outs"] = [s["flat"][at:at + k].view(shape) for (at, k), shape in zip(spans, shapes)]
        return s
    B, S, V, D = (case[k] for k in ("B", "S", "V", "D"))
    s["table"] = normal(V, D, std=0.02)
    # a few tokens make up much of a text: ranks are uniform in their logarithm, ids spread over the table
    rank = torch.rand((B, S), device="cuda", generator=g, dtype=torch.float64).mul_(math.log(V)).exp_().long() - 1
    ids = (rank.clamp_(0, V - 1) * 7919 + 1) % V
    ids = torch.where(ids == PAD, V - 1, ids)
    ids[:, S - S // 8:] = PAD  # the last eighth of a row is padding
    s["ids"] = ids.to(torch.int32)
    s["scale"] = math.sqrt(D) if case["scaled"] else 1.0
    if case["train"]:
        s["dout"] = normal(B, S, D, std=0.01)
    return s


# --------------------------------------------------------------------- run
def run(s):
    return _own(s) if own else _plain(s)


def _own(s):
    import __graft_entry__

    mc = __graft_entry__.load_package()
    c = s["case"]
    if c["kind"] == "attention":
        spans = None
        if c["documents"] or c["prefix"]:
            spans = mc.attention_spans(documents=s.get("documents"), prefix=s.get("prefix"), causal=True)
        how = {"spans": spans, "causal": spans is None, "cap": c["cap"] or None, "slopes": s.get("slopes")}
        o, lse = mc.packed_attention_forward(s["q"], s["k"], s["v"], save_lse=c["train"], **how)
        if not c["train"]:
            return o
        return (o, *mc.packed_attention_backward(s["q"], s["k"], s["v"], o, lse, s["dout"], **how))
    if c["kind"] == "clip":
        norm, scale = mc.clip_gradients(s["grads"], 1.0, outs=s["outs"])
        return norm, scale, s["flat"]
    x = mc.embedding_forward(s["table"], s["ids"], scale=s["scale"], padding_id=PAD)
    if not c["train"]:
        return x
    return x, mc.embedding_backward(s["dout"], s["ids"], c["V"], scale=s["scale"], padding_id=PAD)


def _visible(s, b):
    """[S, S]: may query i see key j in row b of the batch."""
    S = s["q"].shape[2]
    at = torch.arange(S, device="cuda")
    see = at[None, :] <= at[:, None]
    first = torch.ones(S, dtype=torch.bool, device="cuda")
    if "documents" in s:
        ids = s["documents"][b]
        first[1:] = ids[1:] != ids[:-1]
    else:
        first[1:] = False
    run = first.long().cumsum(0) - 1
    if "prefix" in s:  # tokens of a document that nothing but prompt stands before
        answer = (s["prefix"][b] == 0).long()
        before = answer.cumsum(0)
        start = (before - answer)[first]  # answer tokens before the document
        see = see | ((before - start[run]) == 0)[None, :]
    see = see & (run[None, :] == run[:, None])
    if "documents" in s:
        see = see & (ids >= 0)[None, :] & (ids >= 0)[:, None]
    return see


def _plain_attention(s):
    c = s["case"]
    B, H, Hkv, S, D = (c[k] for k in ("B", "H", "Hkv", "S", "D"))
    rep, scale, dtype = H // Hkv, 1.0 / math.sqrt(D), s["q"].dtype
    o = torch.empty((B, S, H * D), dtype=dtype, device="cuda")
    grads = [torch.empty_like(s[n]) for n in "qkv"] if c["train"] else []
    at = torch.arange(S, device="cuda", dtype=torch.float32)
    far = (at[:, None] - at[None, :]).abs()
    for b in range(B):
        q = s["q"][b].float()
        k, v = (s[n][b].float().repeat_interleave(rep, 0) for n in "kv")
        kt = k.transpose(1, 2).contiguous()
        x = torch.matmul(q, kt) * scale
        t = None
        if c["cap"]:
            t = torch.tanh(x / c["cap"])
            x = t * c["cap"]
        if c["bias"]:
            x = x - s["slopes"][:, None, None] * far
        x = torch.where(_visible(s, b), x, -math.inf)
        top = x.amax(-1, keepdim=True)
        p = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
        total = p.sum(-1, keepdim=True)
        p = p / torch.where(total == 0.0, 1.0, total)  # a row that sees nothing gets nothing
        del x
        out = torch.matmul(p, v)
        o[b] = out.transpose(0, 1).reshape(S, H * D).to(dtype)
        if not c["train"]:
            continue
        do = s["dout"][b].float().view(S, H, D).transpose(0, 1).contiguous()
        dp = torch.matmul(do, v.transpose(1, 2).contiguous())
        ds = p * (dp - (do * out).sum(-1, keepdim=True))
        del dp
        if t is not None:
            ds = ds * (1.0 - t * t)
        ds = ds * scale
        grads[0][b] = torch.matmul(ds, k).to(dtype)
        grads[1][b] = torch.matmul(ds.transpose(1, 2).contiguous(), q).view(Hkv, rep, S, D).sum(1).to(dtype)
        grads[2][b] = torch.matmul(p.transpose(1, 2).contiguous(), do).view(Hkv, rep, S, D).sum(1).to(dtype)
    return (o, *grads) if c["train"] else o


def _plain(s):
    c = s["case"]
    if c["kind"] == "attention":
        return _plain_attention(s)
    if c["kind"] == "clip":
        total = sum(g.float().square().sum(dtype=torch.float64) for g in s["grads"])
        norm = total.sqrt().float().view(1)
        scale = (1.0 / norm).clamp(max=1.0)
        for g, out in zip(s["grads"], s["outs"]):
            out.copy_(g.float() * scale)
        return norm, scale, s["flat"]
    ids = s["ids"].long()
    kept = (ids != PAD)[..., None]
    x = torch.where(kept, s["table"][ids].float() * s["scale"], 0.0).to(s["table"].dtype)
    if not c["train"]:
        return x
    d = torch.where(kept, s["dout"].float() * s["scale"], 0.0).flatten(0, 1)
    return x, torch.zeros((c["V"], c["D"]), device="cuda").index_add_(0, ids.flatten(), d)


# -------------------------------------------------------------------- work
def work(case):
    if case["kind"] == "attention":
        B, H, Hkv, S, D = (case[k] for k in ("B", "H", "Hkv", "S", "D"))
        q, kv = B * H * S * D, 2 * B * Hkv * S * D
        inputs = (5 if case["documents"] or case["prefix"] else 0) * B * S
        flops = 4 * H * D * _pairs(case)  # two products, and the backward's four
        size = BYTES[case["dtype"]]
        if not case["train"]:
            return {"bytes": (2 * q + kv) * size + inputs, "flops": flops}
        return {"bytes": (4 * q + 2 * kv) * size + inputs, "flops": flops + 8 * H * D * _pairs(case)}
    if case["kind"] == "clip":
        n = sum(a * b for a, b in _shapes(case))
        return {"bytes": n * (BYTES[case["dtype"]] + 4), "flops": 3 * n}
    T, V, D, size = case["B"] * case["S"], case["V"], case["D"], BYTES[case["dtype"]]
    kept = T - case["B"] * (case["S"] // 8)
    n = {"bytes": 4 * T + (kept + T) * D * size, "flops": T * D}
    if case["train"]:  # the kept tokens' gradients, and the whole table's
        n = {"bytes": n["bytes"] + kept * D * size + 4 * V * D, "flops": n["flops"] + 2 * T * D}
    return n


# ------------------------------------------------------------------- exact
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "attention":
        return _exact_attention(case, s)
    if case["kind"] == "clip":
        norm = torch.sqrt(sum(torch.sum(g.double() ** 2) for g in s["grads"]))
        scale = min(1.0, 1.0 / float(norm))
        flat = torch.zeros(s["flat"].shape, dtype=torch.float64, device="cuda")
        at = 0
        for g in s["grads"]:
            flat[at:at + g.numel()] = g.flatten().double() * scale
            at += (g.numel() + 63) // 64 * 64
        return norm.view(1), torch.tensor([scale], dtype=torch.float64), flat
    ids, table = s["ids"].flatten().to(torch.int64), s["table"].double()
    real = torch.nonzero(ids != PAD)[:, 0]
    x = torch.zeros((ids.numel(), case["D"]), dtype=torch.float64, device="cuda")
    x[real] = table.index_select(0, ids[real]) * s["scale"]
    x = x.view(case["B"], case["S"], case["D"])
    if not case["train"]:
        return x
    del table
    grad = torch.zeros((case["V"], case["D"]), dtype=torch.float64, device="cuda")
    grad.index_put_((ids[real],), s["dout"].flatten(0, 1)[real].double() * s["scale"], accumulate=True)
    return x, grad


def _exact_attention(case, s):
    """By automatic differentiation, one key head of one row at a time, the mask drawn document by document."""
    B, H, Hkv, S, D = (case[k] for k in ("B", "H", "Hkv", "S", "D"))
    rep = H // Hkv
    o = torch.zeros((B, S, H, D), dtype=torch.float64, device="cuda")
    grads = [torch.zeros(s[n].shape, dtype=torch.float64, device="cuda") for n in "qkv"]
    for b, row in enumerate(_documents(case)):
        hidden = torch.ones((S, S), dtype=torch.bool, device="cuda")
        for start, end, prompt in row:
            hidden[start:end, start:end] = torch.ones((end - start,) * 2, device="cuda").tril() == 0
            hidden[start:start + prompt, start:start + prompt] = False
        end = row[-1][1] if row else 0
        for h in range(Hkv):
            heads = slice(h * rep, (h + 1) * rep)
            q = s["q"][b, heads, :end].double().requires_grad_(case["train"])
            k = s["k"][b, h, :end].double().requires_grad_(case["train"])
            v = s["v"][b, h, :end].double().requires_grad_(case["train"])
            x = q @ k.T / math.sqrt(D)
            if case["cap"]:
                x = case["cap"] * torch.tanh(x / case["cap"])
            if case["bias"]:
                i = torch.arange(end, dtype=torch.float64, device="cuda")
                x = x - s["slopes"][heads].double()[:, None, None] * torch.abs(i[:, None] - i)
            x = x.masked_fill(hidden[:end, :end], -math.inf)
            out = torch.softmax(x, -1) @ v
            o[b, :end, heads] = out.detach().transpose(0, 1)
            if case["train"]:
                dout = s["dout"].view(B, S, H, D)[b, :end, heads].double().transpose(0, 1)
                got = torch.autograd.grad(out, (q, k, v), dout)
                grads[0][b, heads, :end], grads[1][b, h, :end], grads[2][b, h, :end] = got
            del x, out
    o = o.view(B, S, H * D)
    return (o, *grads) if case["train"] else o
