"""The losses over a vocabulary's logits that come after supervised fine-tuning,
as they are measured: log-probabilities of given tokens, the preference loss over
pairs of sequences, the clipped policy loss with its KL term, and distillation
from a teacher's top logits, each forward and backward.

`run` computes them in elementary torch operations, or, where `own` is true, with
the framework's calls. Sizes: the vocabularies and token counts that the tests
and the loss's own cases run, and odd and ragged ones of the same ranges.
"""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "bf16": 2}
IGNORE = 0  # the padding token's id: never a counted target
VOCAB = 151936


def listed():
    return [
        # The log-probability of one new token: the smallest call, latency.
        {"name": "logprobs_token", "kind": "logprobs", "train": False, "dtype": "bf16", "B": 1, "S": 1, "V": VOCAB,
         "temperature": 1.0},
        # Scoring a sampled answer of an arbitrary length at the temperature it was sampled with.
        {"name": "logprobs_answer", "kind": "logprobs", "train": False, "dtype": "bf16", "B": 1, "S": 777, "V": VOCAB,
         "temperature": 0.7},
        # A float32 loss of the user's own over log-probabilities, and its gradient.
        {"name": "logprobs_train_f32", "kind": "logprobs", "train": True, "dtype": "f32", "B": 4, "S": 509,
         "V": 50257, "temperature": 1.0},
        # A step on two short pairs, a small vocabulary.
        {"name": "preference_small_f32", "kind": "preference", "dtype": "f32", "B": 4, "S": 65, "V": 32000,
         "loss": "sigmoid", "beta": 0.1, "smoothing": 0.1, "margin": 0.0, "average": False},
        # A training step on four pairs, padded to their longest answer.
        {"name": "preference_train_bf16", "kind": "preference", "dtype": "bf16", "B": 8, "S": 509, "V": VOCAB,
         "loss": "sigmoid", "beta": 0.1, "smoothing": 0.0, "margin": 0.0, "average": False},
        # Means over the answers' tokens, and a vocabulary whose rows start anywhere in a vector.
        {"name": "preference_odd_bf16", "kind": "preference", "dtype": "bf16", "B": 16, "S": 301, "V": 50257,
         "loss": "squared", "beta": 0.25, "smoothing": 0.0, "margin": 0.0, "average": True},
        # A few short answers: a step where latency counts.
        {"name": "policy_small_bf16", "kind": "policy", "dtype": "bf16", "B": 2, "S": 47, "V": 32000,
         "reduction": "sequences", "per_token": False, "kl": 0.04, "temperature": 1.0},
        # A training step on a group of eight answers to one prompt.
        {"name": "policy_train_bf16", "kind": "policy", "dtype": "bf16", "B": 8, "S": 512, "V": VOCAB,
         "reduction": "tokens", "per_token": False, "kl": 0.04, "temperature": 1.0},
        # Float32, an advantage for each token, without a KL term.
        {"name": "policy_train_f32", "kind": "policy", "dtype": "f32", "B": 4, "S": 509, "V": 50257,
         "reduction": "tokens", "per_token": True, "kl": 0.0, "temperature": 0.9},
        # Float32 distillation from the eight best of a teacher.
        {"name": "distill_train_f32", "kind": "distill", "dtype": "f32", "B": 4, "S": 375, "V": 50257, "top": 8,
         "temperature": 1.0, "renormalise": True},
        # A training step towards a teacher's 64 best, softened.
        {"name": "distill_train_bf16", "kind": "distill", "dtype": "bf16", "B": 4, "S": 509, "V": VOCAB, "top": 64,
         "temperature": 2.0, "renormalise": True},
        # The largest batch: 8192 tokens, 128 of the teacher's probabilities as they are.
        {"name": "distill_large_bf16", "kind": "distill", "dtype": "bf16", "B": 16, "S": 512, "V": VOCAB, "top": 128,
         "temperature": 1.0, "renormalise": False},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["logprobs", "preference", "policy", "distill"])
    dtype = rng.choice(["f32", "bf16"])
    V = rng.choice([_log_int(rng, 1000, VOCAB), _log_int(rng, 8000, VOCAB), VOCAB])
    most = 8192 * VOCAB * 2 // (V * BYTES[dtype])  # the largest listed case's bytes
    rows = _log_int(rng, 1 if kind == "logprobs" else 8, min(8192, most))
    B = min(rows, rng.choice([1, 2, 3, 4, 8, 16]))
    if kind == "preference":
        B = max(2, B // 2 * 2)
    c = {"kind": kind, "dtype": dtype, "B": B, "S": max(1, rows // B), "V": V}
    if kind == "logprobs":
        return {**c, "train": rng.random() < 0.5, "temperature": rng.choice([0.7, 1.0, 1.3])}
    if kind == "preference":
        loss = rng.choice(["sigmoid", "sigmoid", "hinge", "squared"])
        return {**c, "loss": loss, "beta": rng.choice([0.05, 0.1, 0.25]),
                "smoothing": rng.choice([0.0, 0.1]) if loss == "sigmoid" else 0.0,
                "margin": rng.choice([0.0, 0.5]) if loss != "squared" else 0.0, "average": rng.random() < 0.3}
    if kind == "policy":
        return {**c, "reduction": rng.choice(["tokens", "sequences"]), "per_token": rng.random() < 0.5,
                "kl": rng.choice([0.0, 0.04, 0.1]), "temperature": rng.choice([0.9, 1.0])}
    return {**c, "top": rng.choice([1, 8, 20, 50, 64, 100, 128, 256]), "temperature": rng.choice([1.0, 2.0]),
            "renormalise": rng.random() < 0.6}


# ------------------------------------------------------------------ inputs
def _spans(case):
    """[(first counted token, first padded one)] of each sequence: a prompt, an answer and padding, alike for
    every seed. A row that is scored, not trained on, counts whole."""
    B, S = case["B"], case["S"]
    if case["kind"] == "logprobs" and not case["train"]:
        return [(0, S)] * B
    rng = random.Random(1009 * B + S)
    ends = [S if i == 0 else S - rng.randrange(0, S // 3 + 1) for i in range(B)]
    return [(rng.randrange(0, e // 4 + 1), e) for e in ends]


def _counted(case):
    spans = torch.tensor(_spans(case), device="cuda")
    at = torch.arange(case["S"], device="cuda")
    return (at >= spans[:, :1]) & (at < spans[:, 1:])


CLIP_LOW, CLIP_HIGH = 0.2, 0.28


def _log_probs(x, targets, T):
    """Of each token under the logits, to make the log-probabilities of nearby policies from."""
    rows = []
    for part, t in zip(x.flatten(0, 1).split(512), targets.flatten().long().split(512)):
        part = part.float() / T
        rows.append(part.gather(1, t[:, None])[:, 0] - torch.logsumexp(part, 1))
    return torch.cat(rows).view(targets.shape)


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    B, S, V, dtype = case["B"], case["S"], case["V"], DTYPES[case["dtype"]]

    def normal(shape, std=1.0, mean=0.0):
        return torch.empty(shape, device="cuda").normal_(mean, std, generator=g)

    # Most of a vocabulary lies far below the tokens in question.
    x = torch.empty((B, S, V), dtype=dtype, device="cuda").normal_(0.0, 2.0, generator=g)
    counted = _counted(case)
    s = {"logits": x}
    if case["kind"] == "distill":
        K = min(case["top"], V)
        first = torch.randint(0, V, (B, S, 1), generator=g, device="cuda")
        step = V // K  # K different tokens
        ids = (first + step * torch.arange(K, device="cuda")) % V
        teacher = 12.0 - 1.5 * torch.arange(1, K + 1, device="cuda").log() + normal((B, S, K), 0.5)
        x.scatter_(2, ids, (teacher + normal((B, S, K))).to(dtype))  # a student that has learnt some of it
        s["ids"], s["teacher"], s["mask"] = ids.to(torch.int32), teacher, counted.to(torch.uint8)
        if not case["renormalise"]:  # the teacher's other tokens hold a tenth
            s["lse"] = torch.logsumexp(teacher / case["temperature"], -1) - math.log(0.9)
        return s
    targets = torch.randint(1, V, (B, S), generator=g, device="cuda")
    x.scatter_(2, targets[..., None], (normal((B, S, 1), 3.0, 12.0)).to(dtype))
    T = case.get("temperature", 1.0)
    if case["kind"] == "logprobs":
        if case["train"]:
            s["dlogps"] = normal((B, S), 1e-2)
    else:
        near = _log_probs(x, targets, T)
        s["ref"] = near + normal((B, S), 0.3)
        if case["kind"] == "preference":
            # training has moved the two answers apart, by up to 12 (where the mean counts, by as much at any length)
            apart = 0.04 if case["average"] else min(0.04, 12.0 / S)
            s["ref"] += torch.where(torch.arange(B, device="cuda") < B // 2, -0.25, 0.75)[:, None] * apart
        if case["kind"] == "policy":
            move = normal((B, S), 0.15)  # what the last updates changed
            for border in (math.log1p(CLIP_HIGH), math.log1p(-CLIP_LOW)):
                move = torch.where((move - border).abs() < 1e-3, move + 2e-3, move)
            s["old"] = near - move
            s["advantages"] = normal((B, S) if case["per_token"] else (B,))
            if case["kl"] == 0.0:
                del s["ref"]
    s["targets"] = torch.where(counted, targets, IGNORE).to(torch.int32)
    return s


def prepare(case, seed):
    return {"case": case, **_inputs(case, seed)}


# --------------------------------------------------------------------- run
def run(s):
    return _own(s) if own else _plain(s)


def _own(s):
    import __graft_entry__

    mc = __graft_entry__.load_package()
    c, x = s["case"], s["logits"]
    if c["kind"] == "logprobs":
        logps, stats = mc.token_logprobs_forward(x, s["targets"], ignore_index=IGNORE, temperature=c["temperature"],
                                                 save_stats=c["train"])
        if not c["train"]:
            return logps
        return logps, mc.token_logprobs_backward(x, s["targets"], stats, s["dlogps"], ignore_index=IGNORE,
                                                 temperature=c["temperature"])
    if c["kind"] == "preference":
        loss, rewards, stats = mc.preference_loss_forward(
            x, s["targets"], ref_logps=s["ref"], beta=c["beta"], kind=c["loss"], label_smoothing=c["smoothing"],
            margin=c["margin"], average=c["average"], ignore_index=IGNORE)
        return loss, rewards, mc.preference_loss_backward(x, s["targets"], stats, ignore_index=IGNORE)
    if c["kind"] == "policy":
        return mc.policy_loss_forward_backward(
            x, s["targets"], s["advantages"], old_logps=s["old"], ref_logps=s.get("ref"), clip_low=CLIP_LOW,
            clip_high=CLIP_HIGH, kl_coef=c["kl"], temperature=c["temperature"], reduction=c["reduction"],
            ignore_index=IGNORE)
    return mc.distillation_loss_forward_backward(x, s["ids"], s["teacher"], temperature=c["temperature"],
                                                 teacher_lse=s.get("lse"), mask=s["mask"])


def _plain(s):
    c = s["case"]
    T = c.get("temperature", 1.0)
    z = s["logits"].float() / T
    z = z - z.amax(-1, keepdim=True)
    e = z.exp()
    if c["kind"] == "distill":
        return _plain_distill(s, z, e, e.sum(-1, keepdim=True))
    # 64 bits where the log-probabilities are summed over whole answers and then subtracted
    total = e.sum(-1, keepdim=True, dtype=torch.float64 if c["kind"] == "preference" else torch.float32)
    targets = s["targets"].long()
    counted = targets != IGNORE
    l = (z.gather(2, targets[..., None]) - total.log())[..., 0]
    l = torch.where(counted, l, 0.0)
    total = total.float()
    del z

    def gradient(dl):  # of the logits, from that of the counted tokens' log-probabilities
        dl = torch.where(counted, dl, 0.0)[..., None] / T
        d = e * (-dl / total)
        return d.scatter_add_(2, targets[..., None], dl).to(s["logits"].dtype)

    if c["kind"] == "logprobs":
        return (l, gradient(s["dlogps"])) if c["train"] else l
    n = counted.sum(1)
    if c["kind"] == "preference":
        score = torch.where(counted, l - s["ref"], 0.0).sum(1)
        if c["average"]:
            score = score / n.clamp(min=1)
        pairs = c["B"] // 2
        d = score[:pairs] - score[pairs:]
        if c["loss"] == "squared":
            off = d - 0.5 / c["beta"]
            loss, dd = off * off, 2.0 * off
        else:
            m = c["beta"] * d - c["margin"]
            if c["loss"] == "hinge":
                loss, dd = (1.0 - m).clamp(min=0.0), torch.where(m < 1.0, -c["beta"], 0.0)
            else:
                tail = torch.log1p(torch.exp(-m.abs()))
                up, down = tail + (-m).clamp(min=0.0), tail + m.clamp(min=0.0)  # -log sigma(m), -log sigma(-m)
                a = c["smoothing"]
                loss = (1.0 - a) * up + a * down
                dd = c["beta"] * (a * torch.exp(-up) - (1.0 - a) * torch.exp(-down))
        dseq = torch.cat([dd, -dd]) / pairs
        if c["average"]:
            dseq = dseq / n.clamp(min=1)
        return (loss.mean().float().reshape(1), (c["beta"] * score).float(),
                gradient(dseq.float()[:, None].expand_as(l)))
    A = s["advantages"] if c["per_token"] else s["advantages"][:, None]
    ratio = torch.exp(l - s["old"])
    weight = counted / (counted.sum() if c["reduction"] == "tokens" else c["B"] * n.clamp(min=1)[:, None])
    held = ratio.clamp(1.0 - CLIP_LOW, 1.0 + CLIP_HIGH) * A
    surrogate = torch.minimum(ratio * A, held)
    clipped = held < ratio * A
    term = -surrogate
    dl = torch.where(clipped, 0.0, -ratio * A)
    kl = torch.zeros_like(l)
    if c["kl"] != 0.0:
        r = s["ref"] - l
        kl = torch.expm1(r) - r
        term = term + c["kl"] * kl
        dl = dl - c["kl"] * torch.expm1(r)
    mean = lambda v: (v * weight).double().sum().float()  # noqa: E731
    return (mean(term).reshape(1), l, torch.stack([mean(kl), mean(clipped.float())]), gradient(dl * weight))


def _plain_distill(s, z, e, total):
    c = s["case"]
    T = c["temperature"]
    t = s["teacher"] / T
    ids = s["ids"].long()
    if "lse" in s:
        log_p = t - s["lse"][..., None]
    else:
        log_p = t - t.amax(-1, keepdim=True)
        log_p = log_p - log_p.exp().sum(-1, keepdim=True).log()
    p = log_p.exp()
    counted = s["mask"] != 0
    kl = (p * (log_p - (z.gather(2, ids) - total.log()))).sum(-1)
    del z
    count = counted.sum()
    loss = T * T * torch.where(counted, kl, 0.0).double().sum() / count
    w = torch.where(counted, T / count, 0.0)[..., None]
    d = e * (w * p.sum(-1, keepdim=True) / total)
    return loss.float().reshape(1), d.scatter_add_(2, ids, -w * p).to(s["logits"].dtype)


# -------------------------------------------------------------------- work
def work(case):
    B, S, V, es = case["B"], case["S"], case["V"], BYTES[case["dtype"]]
    read = sum(end - first for first, end in _spans(case)) * V * es
    small = 4 * 4 * B * S
    if case["kind"] == "logprobs" and not case["train"]:
        return {"bytes": read + small, "flops": 4.0 * read / es}
    if case["kind"] == "distill":
        small = 8 * B * S * min(case["top"], V)
    return {"bytes": read + B * S * V * es + small, "flops": 7.0 * read / es}


# ------------------------------------------------------------------- exact
def exact(case, seed):
    s = _inputs(case, seed)
    T = case.get("temperature", 1.0)
    flat = s["logits"].flatten(0, 1)
    rows, V = flat.shape
    blocks = [slice(i, min(i + 256, rows)) for i in range(0, rows, 256)]
    at = s["ids" if case["kind"] == "distill" else "targets"].long().reshape(rows, -1)
    lq = torch.cat([torch.log_softmax(flat[b].double() / T, -1).gather(1, at[b]) for b in blocks])
    grad = None
    if case["kind"] != "logprobs" or case["train"]:
        grad = torch.empty(rows, V, dtype=torch.float64, device="cuda")

    def backward(dlq):  # sum over the given tokens of dlq d(log q)/dx
        for b in blocks:
            grad[b] = torch.softmax(flat[b].double() / T, -1)
            grad[b] *= -dlq[b].sum(1, keepdim=True) / T
            grad[b] = grad[b].scatter_add(1, at[b], dlq[b] / T)
        return grad.view(s["logits"].shape)

    if case["kind"] == "distill":
        t = s["teacher"].double().reshape(rows, -1) / T
        lp = torch.log_softmax(t, -1) if "lse" not in s else t - s["lse"].double().reshape(rows, 1)
        on = s["mask"].reshape(rows, 1).double()
        p = lp.exp() * on * T * T / on.sum()
        return (p * (lp - lq)).sum().reshape(1), backward(-p)
    on = _counted(case).double()
    l = lq.view(on.shape)
    l = torch.where(on > 0, l, 0.0)
    if case["kind"] == "logprobs":
        if not case["train"]:
            return l
        return l, backward((s["dlogps"].double() * on).reshape(rows, 1))
    l = l.clone().requires_grad_()
    n = on.sum(1)
    if case["kind"] == "preference":
        score = ((l - s["ref"].double()) * on).sum(1)
        if case["average"]:
            score = score / n.clamp(min=1)
        d = score[: case["B"] // 2] - score[case["B"] // 2:]
        m = case["beta"] * d - case["margin"]
        if case["loss"] == "squared":
            each = (d - 1.0 / (2.0 * case["beta"])) ** 2
        elif case["loss"] == "hinge":
            each = torch.relu(1.0 - m)
        else:
            each = -(1.0 - case["smoothing"]) * torch.nn.functional.logsigmoid(m)
            each = each - case["smoothing"] * torch.nn.functional.logsigmoid(-m)
        loss = each.mean()
        outs = (loss.detach().reshape(1), case["beta"] * score.detach())
    else:
        A = s["advantages"].double()
        A = A if case["per_token"] else A[:, None]
        ratio = torch.exp(l - s["old"].double())
        w = on / (on.sum() if case["reduction"] == "tokens" else case["B"] * n.clamp(min=1)[:, None])
        held = torch.clamp(ratio, 1.0 - CLIP_LOW, 1.0 + CLIP_HIGH) * A
        loss = -(torch.minimum(ratio * A, held) * w).sum()
        kl = torch.zeros((), dtype=torch.float64, device="cuda")
        if case["kl"] != 0.0:
            r = s["ref"].double() - l
            kl = ((torch.exp(r) - r - 1.0) * w).sum()
            loss = loss + case["kl"] * kl
        clipped = ((held < ratio * A) * w).sum()
        outs = (loss.detach().reshape(1), l.detach(), torch.stack([kl.detach(), clipped]))
    loss.backward()
    return *outs, backward(l.grad.reshape(rows, 1))
