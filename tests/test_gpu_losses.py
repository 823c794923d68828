"""The losses over log-probabilities (mc_token_logprobs_*, mc_preference_loss_*,
mc_policy_loss_*, mc_distill_loss_*) against a plain implementation in float64.

Tolerances. A token's log-probability is (x_t - m) / T - log(s). Its two parts
are each rounded a few times at their own size, z = (x_t - m) / T and log s, and
s is a sum of exponentials: each is off by 2 ulp of itself and by its argument's
rounding, whose effect e^-a 2^-24 a is below 2^-25, and the sum of a row runs
through chains of at most a few dozen roundings of random sign. So

    |l - l64| <= 2^-20 + 2^-22 (|z| + |log s|)

and a loss's value is off by that of its tokens, times what it multiplies them
with. An element of the gradient is a difference of terms g q and g [j = t]: g
carries the errors of l, q those of (x - m) / T (at most 2^-23 |z| <= 5e-6 where q
is not negligible) and of 1 / s, so it is held to 1e-5 of the sum of its terms'
sizes, plus the rounding of the result, eps / 2 of it (bf16 2^-8, f32 2^-24).
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16]
VOCABS = [1, 2, 7, 9, 17, 255, 1023, 2049, 4096, 8193, 33001]
PAD = 4294967295  # -1 as a uint32


def gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def logits_at(dev, g, shape, dtype, offset=0, std=2.0):
    n = math.prod(shape)
    buf = torch.randn(n + offset, generator=g, device=dev).mul_(std).to(dtype)
    return buf[offset:].view(shape)


def some_targets(dev, g, shape, V, drop=0.3):
    """Random targets, the first and last of the vocabulary among them; a share of the rows padded."""
    t = torch.randint(0, V, shape, generator=g, device=dev)
    t.view(-1)[0], t.view(-1)[-1] = V - 1, 0
    if drop and t.numel() > 1:
        t = torch.where(torch.rand(shape, generator=g, device=dev) < drop, -1, t)
    return t.to(torch.int32)


# ------------------------------------------------------------- plain, 64 bits
def plain_rows(x, T):
    """(x - m) / T, log s, softmax."""
    z = x.double() / T
    z = z - z.amax(-1, keepdim=True)
    e = z.exp()
    s = e.sum(-1, keepdim=True)
    return z, s.log(), e / s


def plain_logps(x, targets, T=1.0):
    """(l, its tolerance, q) of counted tokens; 0 elsewhere."""
    on = targets != -1
    z, ls, q = plain_rows(x, T)
    zt = z.gather(-1, targets.long().clamp(min=0)[..., None])
    tol = 2.0 ** -20 + 2.0 ** -22 * (zt.abs() + ls.abs())
    return torch.where(on, (zt - ls)[..., 0], 0.0), torch.where(on, tol[..., 0], 0.0), q


def plain_grad(q, targets, dl, T=1.0):
    """(gradient, its terms' sizes) from dloss/dl."""
    on = targets != -1
    g = torch.where(on, dl, 0.0)[..., None] / T
    hot = torch.zeros_like(q).scatter_(-1, targets.long().clamp(min=0)[..., None], 1.0)
    return g * (hot - q), g.abs() * (hot + q)


def close(got, want, tol, what=""):
    bad = ~((got.double() - want).abs() <= tol)  # a NaN, too
    assert not bad.any(), f"{what}: {int(bad.sum())} off, the first at {bad.nonzero()[0].tolist()}: " \
        f"{got[bad][0].item()} for {want.expand_as(got)[bad][0].item()}"


def close_grad(d, want, terms, dtype, what="gradient"):
    close(d, want, 1e-5 * terms + torch.finfo(dtype).eps / 2 * want.abs() + 1e-37, what)


def plain_preference(l, targets, ref, beta, kind, eps, margin, average):
    on = (targets != -1).double()
    s = ((l - (0.0 if ref is None else ref.double())) * on).sum(1)
    if average:
        s = s / on.sum(1).clamp(min=1.0)
    P = s.shape[0] // 2
    d = s[:P] - s[P:]
    z = beta * d - margin
    if kind == "sigmoid":
        loss = -(1 - eps) * torch.nn.functional.logsigmoid(z) - eps * torch.nn.functional.logsigmoid(-z)
    elif kind == "hinge":
        loss = (1 - z).clamp(min=0.0)
    else:
        loss = (d - 0.5 / beta) ** 2
    return loss.mean(), beta * s.detach()


def plain_policy(l, targets, A, old, ref, lo, hi, kl_coef, reduction):
    on = (targets != -1).double()
    w = on / on.sum() if reduction == "tokens" else on / (on.shape[0] * on.sum(1, keepdim=True).clamp(min=1.0))
    A = A.double() if A.dim() == 2 else A.double()[:, None]
    r = torch.exp(l - (l.detach() if old is None else old.double()))
    held = r.clamp(1 - lo, 1 + hi) * A
    clipped = held < r * A
    loss = -(torch.where(clipped, held.detach(), r * A) * w).sum()
    kl = torch.zeros((), dtype=torch.float64, device=l.device)
    if ref is not None:
        u = ref.double() - l
        kl = ((torch.exp(u) - u - 1) * w).sum()
        loss = loss + kl_coef * kl
    return loss, torch.stack([kl.detach(), (clipped * w).sum()])


def plain_distill(x, ids, t, T, lse, mask):
    """(loss, its tolerance, gradient, terms)."""
    _, _, q = plain_rows(x, T)
    rows = x.shape[0]
    on = torch.ones(rows, dtype=torch.float64, device=x.device) if mask is None else (mask != 0).double()
    used = (t != -math.inf) & (on != 0)[:, None]
    ids = torch.where(used, ids, 0).long()
    assert int(ids.min()) >= 0 and int(ids.max()) < x.shape[1]  # torch would fault the GPU
    tt = t.double() / T
    z = tt - (torch.logsumexp(tt, 1, keepdim=True).clamp(min=-1e30) if lse is None else lse.double()[:, None])
    p = torch.where(used, z.exp(), 0.0)
    zx, ls, _ = plain_rows(x, T)
    lq = (zx - ls).gather(1, ids)
    kl = torch.where(used, p * (z - lq), 0.0).sum(1)
    # log p carries its own roundings, 2^-23 of the teacher's logits, beside those of l
    tol = torch.where(used, p * (2.0 ** -19 + 2.0 ** -21 * (z.abs() + lq.abs() + tt.abs())), 0.0).sum(1)
    n = on.sum()
    dense = (on * T / n)[:, None] * p.sum(1, keepdim=True) * q
    taken = torch.zeros_like(q).scatter_add_(1, ids, (on * T / n)[:, None] * p)
    return (T * T * kl * on).sum() / n, (T * T * tol * on).sum() / n, dense - taken, dense + taken


# -------------------------------------------------------------- token logprobs
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", VOCABS)
@pytest.mark.parametrize("offset,rows,T", [(0, 5, 1.0), (3, 33, 0.7), (5, 1030, 2.0)])
def test_token_logprobs(mc, dev, nan_outputs, dtype, V, offset, rows, T):
    g = gen(dev, V + offset)
    x = logits_at(dev, g, (rows, V), dtype, offset)
    t = some_targets(dev, g, (rows,), V)
    l, stats = mc.token_logprobs_forward(x, t, ignore_index=PAD, temperature=T)
    dl = torch.randn(rows, generator=g, device=dev)
    dl[1] = 0.0
    d = mc.token_logprobs_backward(x, t, stats, dl, ignore_index=PAD, temperature=T)
    l64, tol, q = plain_logps(x, t, T)
    close(l, l64, tol, "logps")
    close_grad(d, *plain_grad(q, t, dl.double(), T), dtype)
    l2, none = mc.token_logprobs_forward(x, t, ignore_index=PAD, temperature=T, save_stats=False)
    assert none is None and torch.equal(l, l2)


def test_token_logprobs_shapes_and_ids(mc, dev):
    g = gen(dev, 1)
    x = logits_at(dev, g, (2, 3, 101), torch.float32)
    t = torch.randint(0, 101, (2, 3), generator=g, device=dev)
    want, _ = mc.token_logprobs_forward(x, t)
    assert want.shape == (2, 3)
    assert torch.equal(want, mc.token_logprobs_forward(x, t.to(torch.int32))[0])
    assert torch.equal(want.view(-1), mc.token_logprobs_forward(x.view(6, 101), t.to(torch.int32).view(-1))[0])
    one, stats = mc.token_logprobs_forward(x[0, 0], t[0, 0])  # a single row of [V]
    assert one.shape == () and torch.equal(one, want[0, 0]) and stats.shape == (1, 2)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [300, 20001])
def test_rows_are_apart_and_uncounted_rows_unread(mc, dev, nan_outputs, dtype, V):
    """NaN, infinities and the type's lowest value: in uncounted rows they change nothing, in counted ones their own
    row alone."""
    g = gen(dev, V)
    x = logits_at(dev, g, (40, V), dtype)
    t = some_targets(dev, g, (40,), V, drop=0.0)
    low = torch.finfo(dtype).min
    x[2, 1:] = -math.inf                      # one entry left
    t[2] = 0
    x[3, : V // 2] = -math.inf
    t[3] = V - 1
    x[4, V // 3:] = low
    t[4] = 1
    x[5] = low                                # uniform
    x[6, : V - 7] = low
    t[6] = V - 3
    x[8] = -1e30                              # uniform, far down
    t[9] = 0
    x[9, 0] = -math.inf                       # the target itself is masked
    dl = torch.ones(40, device=dev)
    l0, s0 = mc.token_logprobs_forward(x, t)
    d0 = mc.token_logprobs_backward(x, t, s0, dl)
    l64, tol, q = plain_logps(x, t)
    fine = [i for i in range(40) if i != 9]
    close(l0[fine], l64[fine], tol[fine], "logps")
    assert float(l0[9]) == -math.inf
    want, terms = plain_grad(q, t, dl.double())
    close_grad(d0, want, terms, dtype)
    y = x.clone()
    y[10], y[11], y[12, V - 1], y[13, 5] = math.nan, -math.inf, math.inf, math.nan
    l1, s1 = mc.token_logprobs_forward(y, t)
    d1 = mc.token_logprobs_backward(y, t, s1, dl)
    rest = [i for i in range(40) if i not in (10, 11, 12, 13)]
    assert torch.equal(l0[rest], l1[rest]) and torch.equal(d0[rest], d1[rest])
    assert torch.isnan(l1[10:14]).all() and torch.isnan(d1[10]).all() and torch.isnan(d1[13]).all()
    u = t.clone()
    u[10:14] = -1
    l2, s2 = mc.token_logprobs_forward(y, u, ignore_index=PAD)
    d2 = mc.token_logprobs_backward(y, u, s2, torch.full_like(dl, 1.0), ignore_index=PAD)
    assert torch.equal(l0[rest], l2[rest]) and torch.equal(d0[rest], d2[rest])
    assert not l2[10:14].any() and not d2[10:14].any()


def test_token_past_the_vocabulary_is_nan(mc, dev):
    g = gen(dev, 3)
    x = logits_at(dev, g, (4, 50), torch.float32)
    t = torch.tensor([1, 50, 2, -7], device=dev, dtype=torch.int32)
    l, stats = mc.token_logprobs_forward(x, t)
    d = mc.token_logprobs_backward(x, t, stats, torch.ones(4, device=dev))
    assert torch.isnan(l).tolist() == [False, True, False, True]
    assert torch.isnan(d).all(1).tolist() == [False, True, False, True]


def test_offsets_past_32_bits(mc, dev):
    """2.2e9 logits: the last rows lie past 2^31 elements and 2^32 bytes."""
    rows, V = 14500, 151936
    x = torch.zeros(rows, V, dtype=torch.bfloat16, device=dev)
    g = gen(dev, 4)
    t = torch.full((rows,), -1, dtype=torch.int32, device=dev)
    at = [0, 7000, 14134, 14135, rows - 1]
    for i in at:
        x[i] = torch.randn(V, generator=g, device=dev).mul_(3.0).to(torch.bfloat16)
        t[i] = int(torch.randint(0, V, (), generator=g, device=dev))
    l, stats = mc.token_logprobs_forward(x, t, ignore_index=PAD)
    d = mc.token_logprobs_backward(x, t, stats, torch.ones(rows, device=dev), ignore_index=PAD)
    l64, tol, q = plain_logps(x[at], t[at])
    close(l[at], l64, tol, "logps")
    close_grad(d[at], *plain_grad(q, t[at], torch.ones(len(at), device=dev).double()), torch.bfloat16)
    assert int(torch.count_nonzero(l)) == len(at)
    d[at] = 0
    assert not d.view(torch.int16).any()


# ------------------------------------------------------------------ preference
PREFERENCES = [("sigmoid", 0.1, 0.0, 0.0, False), ("sigmoid", 0.3, 0.1, 0.5, False), ("sigmoid", 2.0, 0.0, 1.0, True),
               ("hinge", 0.2, 0.0, 0.3, False), ("hinge", 1.0, 0.0, 0.0, True), ("squared", 0.1, 0.0, 0.0, False),
               ("squared", 0.5, 0.0, 0.0, True)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind,beta,eps,margin,average", PREFERENCES)
@pytest.mark.parametrize("P,S,V,offset,with_ref", [
    (1, 1, 33, 0, True), (3, 37, 1001, 1, True), (2, 300, 4096, 0, False), (300, 2, 65, 0, True)])
def test_preference(mc, dev, nan_outputs, dtype, kind, beta, eps, margin, average, P, S, V, offset, with_ref):
    g = gen(dev, P + V)
    x = logits_at(dev, g, (2 * P, S, V), dtype, offset)
    t = some_targets(dev, g, (2 * P, S), V)
    if P > 1:
        t[1] = -1                       # a preferred answer without a token
    if P > 2:
        t[2], t[2 + P] = -1, -1         # a pair without any
    l64, tol, q = plain_logps(x, t)
    ref = (l64 + 0.3 * torch.randn(l64.shape, generator=g, device=dev)).float() if with_ref else None
    dloss = torch.full((1,), 1.5, device=dev)
    loss, rewards, stats = mc.preference_loss_forward(x, t, ref, beta, kind, eps, margin, average, PAD)
    d = mc.preference_loss_backward(x, t, stats, dloss, PAD)
    l = l64.clone().requires_grad_()
    want, r64 = plain_preference(l, t, ref, beta, kind, eps, margin, average)
    want.backward()
    want = want.detach()
    # a score is off by its tokens' errors (and each l by its rounding to 32 bits, inside tol)
    n = (t != -1).sum(1).clamp(min=1) if average else 1
    stol = (tol.sum(1) / n)
    close(rewards, r64, beta * stol + 2.0 ** -23 * r64.abs() + 1e-30, "rewards")
    dd = (stol[:P] + stol[P:])
    s = r64 / beta
    off = (s[:P] - s[P:] - 0.5 / beta).abs()
    slope = 2 * off + dd if kind == "squared" else beta
    assert abs(float(loss) - float(want)) <= float((slope * dd).mean()) + 2.0 ** -22 * abs(float(want))
    grad, terms = plain_grad(q, t, 1.5 * l.grad)
    # g moves with d: by its second derivative (2, at most beta^2 / 4, none) times the error of d, relative to g
    rel = torch.cat([2 * dd / off.clamp(min=1e-9)] * 2) if kind == "squared" else torch.cat([beta * dd] * 2)
    extra = rel[:, None, None].double() * terms
    close(d, grad, 1e-5 * terms + extra + torch.finfo(dtype).eps / 2 * grad.abs() + 1e-37, "gradient")
    assert not d[t == -1].any()


def test_preference_far_apart(mc, dev):
    """Margins of hundreds: no overflow, and a loss that is all tail."""
    V, S = 64, 200
    x = torch.zeros(2, S, V, device=dev)
    x[0, :, 3], x[1, :, 3] = 30.0, -30.0
    t = torch.full((2, S), 3, device=dev, dtype=torch.int32)
    for flip in (False, True):
        y = x.flip(0).contiguous() if flip else x
        loss, rewards, stats = mc.preference_loss_forward(y, t, None, 1.0)
        l = plain_logps(y, t)[0].requires_grad_()
        want, _ = plain_preference(l, t, None, 1.0, "sigmoid", 0.0, 0.0, False)
        want.backward()
        want = want.detach()
        assert abs(float(loss) - float(want)) <= 1e-5 * float(want)
        d = mc.preference_loss_backward(y, t, stats)
        assert torch.isfinite(d).all()
        if flip:
            close_grad(d, *plain_grad(plain_logps(y, t)[2], t, l.grad), torch.float32)


def test_preference_nothing_counted(mc, dev):
    x = torch.full((4, 3, 20), math.nan, device=dev)
    t = torch.full((4, 3), -1, device=dev, dtype=torch.int32)
    loss, rewards, stats = mc.preference_loss_forward(x, t, ignore_index=PAD)
    assert abs(float(loss) - math.log(2.0)) < 1e-6 and not rewards.any()
    assert not mc.preference_loss_backward(x, t, stats, ignore_index=PAD).any()


def test_preference_bad_token_is_nan(mc, dev):
    x = torch.randn(4, 3, 20, device=dev)
    t = torch.randint(0, 20, (4, 3), device=dev, dtype=torch.int32)
    t[1, 2] = 20
    loss, _, stats = mc.preference_loss_forward(x, t)
    d = mc.preference_loss_backward(x, t, stats)
    assert torch.isnan(loss).all() and torch.isnan(d[1]).all() and torch.isnan(d[3]).all()
    assert torch.isfinite(d[0]).all() and torch.isfinite(d[2]).all()


# ---------------------------------------------------------------------- policy
POLICIES = [dict(), dict(kl_coef=0.1, reduction="sequences"),
            dict(clip_low=0.1, clip_high=0.4, kl_coef=0.02, temperature=0.8),
            dict(reduction="sequences", temperature=1.5), dict(clip_low=0.0, clip_high=0.0)]


def policy_case(dev, B, S, V, dtype, offset, per_token, T, seed):
    g = gen(dev, seed)
    x = logits_at(dev, g, (B, S, V), dtype, offset)
    t = some_targets(dev, g, (B, S), V)
    if B > 2:
        t[1] = -1
    l64, tol, q = plain_logps(x, t, T)
    # ratios on both sides of the clip, none within 1e-3 of a border (steps of 0.02 off the borders' logs)
    u = torch.randint(-30, 31, (B, S), generator=g, device=dev) * 0.02 + 0.0071
    old = (l64 - u).float()
    ref = (l64 + 0.4 * torch.randn(B, S, generator=g, device=dev)).float()
    A = torch.randn((B, S) if per_token else (B,), generator=g, device=dev)
    return x, t, l64, tol, q, old, ref, A


def check_policy(mc, dev, x, t, l64, tol, q, A, old, ref, kw, outs, dloss, dtype):
    """outs: (loss, logps, metrics, dlogits)"""
    lo, hi = kw.get("clip_low", 0.2), kw.get("clip_high", 0.2)
    kc, T = kw.get("kl_coef", 0.0), kw.get("temperature", 1.0)
    loss, logps, metrics, d = outs
    close(logps, l64, tol, "logps")
    l = l64.clone().requires_grad_()
    want, m = plain_policy(l, t, A, old, ref, lo, hi, kc, kw.get("reduction", "tokens"))
    want.backward()
    want = want.detach()
    on = t != -1
    w = on / on.sum() if kw.get("reduction", "tokens") == "tokens" else \
        on / (t.shape[0] * on.sum(1, keepdim=True).clamp(min=1))
    # sizes of a token's terms and of its derivative's
    a = A.double().abs() if A.dim() == 2 else A.double().abs()[:, None]
    r = torch.exp(l64 - (l64 if old is None else old.double()))
    k = torch.exp(ref.double() - l64) if ref is not None else torch.zeros_like(l64)
    u = (ref.double() - l64).abs() if ref is not None else torch.zeros_like(l64)
    size = r * a + kc * (k + 1)
    err = ((size * (tol + 2.0 ** -21) + kc * 2.0 ** -22 * (k + u)) * w).sum()
    assert abs(float(loss) - float(want)) <= float(err) + 2.0 ** -24 * abs(float(want))
    ktol = (((k + 1) * (tol + 2.0 ** -21) + 2.0 ** -22 * u) * w).sum()
    assert abs(float(metrics[0]) - float(m[0])) <= float(ktol)
    assert abs(float(metrics[1]) - float(m[1])) <= 2.0 ** -23
    grad, terms = plain_grad(q, t, dloss * l.grad, T)
    gsize = torch.where(on, dloss * size * w, 0.0)[..., None] / T
    hot = torch.zeros_like(q).scatter_(-1, t.long().clamp(min=0)[..., None], 1.0)
    close_grad(d, grad, terms + gsize * (hot + q), dtype)
    assert not d[~on].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kw", POLICIES)
@pytest.mark.parametrize("B,S,V,offset,per_token", [(1, 1, 50, 0, False), (3, 37, 1001, 1, True),
                                                    (5, 130, 2048, 0, False), (700, 1, 40, 0, True)])
def test_policy(mc, dev, nan_outputs, dtype, kw, B, S, V, offset, per_token):
    T = kw.get("temperature", 1.0)
    x, t, l64, tol, q, old, ref, A = policy_case(dev, B, S, V, dtype, offset, per_token, T, B + V)
    dloss = torch.full((1,), 0.7, device=dev)
    for o, f in [(old, ref), (None, ref)] + ([(old, None), (None, None)] if "kl_coef" not in kw else []):
        loss, logps, metrics, stats = mc.policy_loss_forward(x, t, A, o, f, ignore_index=PAD, **kw)
        d = mc.policy_loss_backward(x, t, stats, dloss, temperature=T, ignore_index=PAD)
        check_policy(mc, dev, x, t, l64, tol, q, A, o, f, kw, (loss, logps, metrics, d), 0.7, dtype)
        outs = mc.policy_loss_forward_backward(x, t, A, o, f, ignore_index=PAD, dloss=dloss, **kw)
        check_policy(mc, dev, x, t, l64, tol, q, A, o, f, kw, outs, 0.7, dtype)


def test_policy_clip_sides(mc, dev):
    """Which side of the minimum holds, token by token: the gradient is there or it is zero."""
    V = 40
    x = torch.randn(1, 6, V, generator=gen(dev, 5), device=dev)
    t = torch.arange(6, device=dev, dtype=torch.int32)[None]
    l = mc.token_logprobs_forward(x, t)[0]
    ratio = torch.tensor([[1.5, 1.5, 0.5, 0.5, 1.0, 1.1]], device=dev)
    A = torch.tensor([[1.0, -1.0, 1.0, -1.0, 0.0, 1.0]], device=dev)
    for outs in (mc.policy_loss_forward_backward(x, t, A, l - ratio.log()),):
        loss, _, metrics, d = outs
        assert (d != 0).any(-1).tolist() == [[False, True, True, False, False, True]]
        want = -(1.2 - 1.5 + 0.5 - 0.8 + 0.0 + 1.1) / 6
        assert abs(float(loss) - want) < 1e-5 and abs(float(metrics[1]) - 2 / 6) < 1e-6
    loss, _, _, stats = mc.policy_loss_forward(x, t, A, l - ratio.log())
    d2 = mc.policy_loss_backward(x, t, stats)
    assert (d2 != 0).any(-1).tolist() == [[False, True, True, False, False, True]]


def test_policy_nothing_counted(mc, dev):
    x = torch.full((2, 3, 20), math.nan, device=dev)
    t = torch.full((2, 3), -1, device=dev, dtype=torch.int32)
    A = torch.full((2,), math.nan, device=dev)
    for reduction in ("tokens", "sequences"):
        loss, logps, metrics, stats = mc.policy_loss_forward(x, t, A, reduction=reduction, ignore_index=PAD)
        d = mc.policy_loss_backward(x, t, stats, ignore_index=PAD)
        loss2, logps2, _, d2 = mc.policy_loss_forward_backward(x, t, A, reduction=reduction, ignore_index=PAD)
        assert not logps.any() and not d.any() and not logps2.any() and not d2.any()
        for v in (loss, loss2):
            assert torch.isnan(v).all() if reduction == "tokens" else not v.any()


def test_policy_bad_token_is_nan(mc, dev):
    x = torch.randn(2, 3, 20, device=dev)
    t = torch.randint(0, 20, (2, 3), device=dev, dtype=torch.int32)
    t[1, 2] = 21
    loss, logps, _, d = mc.policy_loss_forward_backward(x, t, torch.ones(2, device=dev))
    assert torch.isnan(loss).all() and torch.isnan(logps).sum() == 1
    assert torch.isnan(d[1, 2]).all() and torch.isfinite(d[0]).all()


# ---------------------------------------------------------------- distillation
def teacher_case(dev, g, rows, V, K, T, with_lse):
    ids = torch.randint(0, V, (rows, K), generator=g, device=dev, dtype=torch.int32)
    if V >= K:  # distinct but in the first rows
        for i in range(2, rows):
            ids[i] = torch.randperm(V, generator=g, device=dev)[:K].to(torch.int32)
    ids[0, 0], ids[0, -1] = 0, V - 1
    t = 5.0 - torch.arange(K, device=dev).float() * 0.3 + torch.randn(rows, K, generator=g, device=dev)
    if K > 2 and rows > 3:
        t[3, K // 2:] = -math.inf        # fewer entries, with any id
        ids[3, K // 2:] = -5
        ids[3, K // 2 + 1:] = 2**31 - 1
        t[1] = -math.inf                 # none at all
    lse = (torch.logsumexp(t / T, 1).clamp(min=0.0) + 0.2) if with_lse else None
    return ids, t, lse


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [1, 5, 17, 300, 2049, 33001])
@pytest.mark.parametrize("K,rows,offset,T,with_lse,with_mask", [
    (1, 3, 0, 1.0, False, False), (8, 33, 3, 2.0, False, True), (20, 9, 0, 0.7, True, False),
    (64, 600, 0, 1.0, False, True), (256, 5, 1, 1.5, True, True)])
def test_distillation(mc, dev, nan_outputs, dtype, V, K, rows, offset, T, with_lse, with_mask):
    g = gen(dev, V + K)
    x = logits_at(dev, g, (rows, V), dtype, offset)
    ids, t, lse = teacher_case(dev, g, rows, V, K, T, with_lse)
    mask = (torch.rand(rows, generator=g, device=dev) < 0.7).to(torch.uint8) if with_mask else None
    if with_mask:
        mask[0] = 1
        x[mask == 0] = math.nan
        t[mask == 0] = math.nan
    dloss = torch.full((1,), 1.3, device=dev)
    xs, ts = torch.nan_to_num(x, 0.0), torch.nan_to_num(t, 0.0, neginf=-math.inf)
    want, tol, grad, terms = plain_distill(xs, ids, ts, T, lse, mask)
    loss, stats = mc.distillation_loss_forward(x, ids, t, T, lse, mask)
    d = mc.distillation_loss_backward(x, ids, t, stats, dloss, T, lse, mask)
    both = mc.distillation_loss_forward_backward(x, ids, t, T, lse, mask, dloss)
    for v, dv in ((loss, d), both):
        assert abs(float(v) - float(want)) <= float(tol) + 2.0 ** -23 * abs(float(want))
        close_grad(dv, 1.3 * grad, 1.3 * terms, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_distillation_repeated_ids(mc, dev, dtype):
    """An id that comes many times counts as often, in one vector, at the edges of a row and across its vectors."""
    V, K = 1003, 40
    g = gen(dev, 6)
    x = logits_at(dev, g, (6, V), dtype, 1)
    ids = torch.randint(0, V, (6, K), generator=g, device=dev, dtype=torch.int32)
    ids[0], ids[1], ids[2] = 0, V - 1, 500
    ids[3, ::2] = 17
    ids[4] = torch.arange(16, 16 + K, device=dev, dtype=torch.int32) // 2
    t = torch.randn(6, K, generator=g, device=dev)
    want, tol, grad, terms = plain_distill(x, ids, t, 1.0, None, None)
    loss, d = mc.distillation_loss_forward_backward(x, ids, t)
    assert abs(float(loss) - float(want)) <= float(tol) + 2.0 ** -23 * abs(float(want))
    close_grad(d, grad, terms, dtype)
    loss2, d2 = mc.distillation_loss_forward_backward(x, ids.long(), t)
    assert torch.equal(loss, loss2) and torch.equal(d, d2)


def test_distillation_long_row_shares_bits(mc, dev):
    """A row of more than 2^16 vectors."""
    V, K = 4 * 65536 * 2 + 77, 33
    g = gen(dev, 7)
    x = logits_at(dev, g, (2, V), torch.float32)
    ids = torch.randint(0, V, (2, K), generator=g, device=dev, dtype=torch.int32)
    ids[0, :3] = torch.tensor([5, 5 + 4 * 65536, 5 + 8 * 65536], device=dev, dtype=torch.int32)
    t = torch.randn(2, K, generator=g, device=dev)
    want, tol, grad, terms = plain_distill(x, ids, t, 1.0, None, None)
    loss, d = mc.distillation_loss_forward_backward(x, ids, t)
    assert abs(float(loss) - float(want)) <= float(tol) + 2.0 ** -23 * abs(float(want))
    close_grad(d, grad, terms, torch.float32)


def test_distillation_bad_id_and_nothing_counted(mc, dev):
    x = torch.randn(4, 30, device=dev)
    ids = torch.randint(0, 30, (4, 5), device=dev, dtype=torch.int32)
    t = torch.randn(4, 5, device=dev)
    for bad in (30, -1, 2**31 - 1):
        ids[2, 1] = bad
        for loss, d in (mc.distillation_loss_forward_backward(x, ids, t),):
            assert torch.isnan(loss).all() and torch.isnan(d[2]).all() and torch.isfinite(d[[0, 1, 3]]).all()
        loss, stats = mc.distillation_loss_forward(x, ids, t)
        assert torch.isnan(loss).all() and torch.isnan(mc.distillation_loss_backward(x, ids, t, stats)[2]).all()
        mask = torch.tensor([1, 1, 0, 1], device=dev, dtype=torch.uint8)
        loss, d = mc.distillation_loss_forward_backward(x, ids, t, mask=mask)
        assert torch.isfinite(loss).all() and torch.isfinite(d).all() and not d[2].any()
    loss, d = mc.distillation_loss_forward_backward(x, ids, t, mask=torch.zeros(4, device=dev, dtype=torch.uint8))
    assert torch.isnan(loss).all() and not d.any()


# ------------------------------------------------------------------- long rows
# Rows of every way of taking them: shared by workgroups (few long rows), held in
# registers by each number of threads, too long to be held.
LONG = [(torch.bfloat16, 1, 151936), (torch.bfloat16, 7, 60001), (torch.float32, 128, 24577), (torch.float32, 3, 400003),
        (torch.bfloat16, 129, 151936), (torch.float32, 131, 77823), (torch.float32, 129, 77829),
        (torch.float32, 130, 100003), (torch.bfloat16, 129, 155651), (torch.bfloat16, 130, 200003),
        (torch.bfloat16, 300, 20000), (torch.bfloat16, 200, 40007), (torch.bfloat16, 200, 52001),
        (torch.bfloat16, 200, 77001), (torch.float32, 140, 50257), (torch.float32, 140, 65001),
        (torch.float32, 400, 1021), (torch.float32, 400, 4100), (torch.float32, 300, 8193),
        (torch.bfloat16, 1600, 1501), (torch.float32, 1600, 1023), (torch.bfloat16, 1700, 4003),
        (torch.float32, 1536, 2047), (torch.bfloat16, 1600, 8195), (torch.float32, 1600, 4099),
        (torch.bfloat16, 1540, 16387)]


@pytest.mark.parametrize("offset", [0, 3])
@pytest.mark.parametrize("dtype,rows,V", LONG)
def test_rows_of_every_length(mc, dev, nan_outputs, dtype, rows, V, offset):
    g = gen(dev, V)
    x = logits_at(dev, g, (rows, V), dtype, offset)
    t = some_targets(dev, g, (rows,), V, drop=0.2)
    t[0] = min(V - 1, 5)
    dl = torch.randn(rows, generator=g, device=dev)
    l, stats = mc.token_logprobs_forward(x, t, ignore_index=PAD)
    l64, tol, q = plain_logps(x, t)
    close(l, l64, tol, "logps")
    close_grad(mc.token_logprobs_backward(x, t, stats, dl, ignore_index=PAD), *plain_grad(q, t, dl.double()), dtype)
    # an advantage per token: -A r is the whole of dl
    A = torch.randn(rows, 1, generator=g, device=dev)
    outs = mc.policy_loss_forward_backward(x[:, None], t[:, None], A, ignore_index=PAD)
    check_policy(mc, dev, x[:, None], t[:, None], l64[:, None], tol[:, None], q[:, None], A, None, None, {}, outs, 1.0,
                 dtype)
    loss, logps, metrics, pstats = mc.policy_loss_forward(x[:, None], t[:, None], A, ignore_index=PAD)
    d = mc.policy_loss_backward(x[:, None], t[:, None], pstats, ignore_index=PAD)
    check_policy(mc, dev, x[:, None], t[:, None], l64[:, None], tol[:, None], q[:, None], A, None, None, {},
                 (loss, logps, metrics, d), 1.0, dtype)
    ids = torch.randint(0, V, (rows, 40), generator=g, device=dev, dtype=torch.int32)
    ids[:, :4] = torch.tensor([0, V - 1, V // 2, V // 2], device=dev, dtype=torch.int32)
    tl = torch.randn(rows, 40, generator=g, device=dev) * 2
    mask = (torch.rand(rows, generator=g, device=dev) < 0.8).to(torch.uint8)
    mask[0] = 1
    want, tol, grad, terms = plain_distill(x, ids, tl, 1.0, None, mask)
    loss, dstats = mc.distillation_loss_forward(x, ids, tl, mask=mask)
    d = mc.distillation_loss_backward(x, ids, tl, dstats, mask=mask)
    for v, dv in ((loss, d), mc.distillation_loss_forward_backward(x, ids, tl, mask=mask)):
        assert abs(float(v) - float(want)) <= float(tol) + 2.0 ** -23 * abs(float(want))
        close_grad(dv, grad, terms, dtype)
    if rows % 2 == 0:
        P = rows // 2
        ploss, rewards, pst = mc.preference_loss_forward(x[:, None], t[:, None], beta=0.3, ignore_index=PAD)
        l = l64[:, None].clone().requires_grad_()
        want, _ = plain_preference(l, t[:, None], None, 0.3, "sigmoid", 0.0, 0.0, False)
        want.backward()
        assert abs(float(ploss) - float(want.detach())) <= 1e-5 * max(1.0, abs(float(want.detach())))
        grad, terms = plain_grad(q, t, l.grad[:, 0])
        pd = mc.preference_loss_backward(x[:, None], t[:, None], pst, ignore_index=PAD)
        close_grad(pd[:, 0], grad, 1.3 * terms, dtype)


# rows held by each way: alone, shared, with a rest read twice
WAYS = [(16, 300), (40, 1003), (1600, 301), (300, 20001), (14, 100003), (140, 200003)]


@pytest.mark.parametrize("offset", [0, 3])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,V", WAYS)
def test_one_read_with_masked_logits(mc, dev, nan_outputs, dtype, rows, V, offset):
    """-inf, the type's lowest value and NaN in the rows that the policy and distillation losses read once."""
    g = gen(dev, V)
    x = logits_at(dev, g, (rows, V), dtype, offset)
    t = some_targets(dev, g, (rows,), V, drop=0.0)
    low = torch.finfo(dtype).min
    x[2, 1:], t[2] = -math.inf, 0
    x[3, : V // 2], t[3] = -math.inf, V - 1
    x[4, V // 3:], t[4] = low, 1
    x[5] = low
    x[6, : V - 7], t[6] = low, V - 3
    x[8] = -1e30
    x[9], t[9] = math.nan, -1
    x[10], t[10] = -math.inf, -1
    on = t != -1
    l64, tol, q = plain_logps(x, t)
    A = torch.randn(rows, 1, generator=g, device=dev)
    l64, tol, q = torch.where(on, l64, 0.0), torch.where(on, tol, 0.0), torch.where(on[:, None], q, 0.0)
    outs = mc.policy_loss_forward_backward(x[:, None], t[:, None], A, ignore_index=PAD)
    check_policy(mc, dev, x[:, None], t[:, None], l64[:, None], tol[:, None], q[:, None], A, None, None, {}, outs, 1.0,
                 dtype)
    # the teacher's entries where the student's are finite
    ids = torch.randint(0, V, (rows, 6), generator=g, device=dev, dtype=torch.int32)
    ids[2], ids[3], ids[4], ids[6], ids[9:11] = 0, V - 2, ids[4] % (V // 3), V - 1, 2**31 - 1
    tl = torch.randn(rows, 6, generator=g, device=dev)
    tl[9:11] = math.nan
    mask = on.to(torch.uint8)
    clean = torch.where(on[:, None], x, 0.0)
    want, dtol, grad, terms = plain_distill(clean, ids, torch.where(on[:, None], tl, 0.0), 1.0, None, mask)
    for loss, d in (mc.distillation_loss_forward_backward(x, ids, tl, mask=mask),):
        assert abs(float(loss) - float(want)) <= float(dtol) + 2.0 ** -23 * abs(float(want))
        close_grad(d, grad, terms, dtype)
        assert not d[~on].any()
    # NaN and infinities in counted rows stay in them
    z, u = x.clone(), t.clone()
    u[9:11] = 0
    z[11, V // 2], z[12, 0] = math.inf, math.nan
    _, logps, _, d = mc.policy_loss_forward_backward(z[:, None], u[:, None], A, ignore_index=PAD)
    bad = torch.zeros(rows, dtype=torch.bool, device=dev)
    bad[9:13] = True
    assert torch.isnan(logps[bad]).all() and torch.isfinite(logps[~bad]).all()
    assert torch.isnan(d[bad]).all() and torch.isfinite(d[~bad]).all()


@pytest.mark.parametrize("offset", [0, 3])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,V", WAYS)
def test_repeated_ids_in_rows_of_every_way(mc, dev, nan_outputs, dtype, rows, V, offset):
    """256 entries: all the same, all of a few vectors, pairs, the edges; in one call and in two."""
    K, g = 256, gen(dev, rows)
    x = logits_at(dev, g, (rows, V), dtype, offset)
    ids = torch.randint(0, V, (rows, K), generator=g, device=dev, dtype=torch.int32)
    near = torch.arange(K, device=dev, dtype=torch.int32)
    ids[0], ids[1], ids[2] = 0, V - 1, V // 2
    ids[3], ids[4], ids[5], ids[6] = near % 20, V - 1 - near % 17, near // 2, 40 + near // 3
    ids[7, ::2] = 17
    ids[8] = ids[8].sort().values // 4 * 4 % V
    tl = torch.randn(rows, K, generator=g, device=dev) * 2
    want, tol, grad, terms = plain_distill(x, ids, tl, 1.0, None, None)
    loss, stats = mc.distillation_loss_forward(x, ids, tl)
    for v, d in ((loss, mc.distillation_loss_backward(x, ids, tl, stats)),
                 mc.distillation_loss_forward_backward(x, ids, tl)):
        assert abs(float(v) - float(want)) <= float(tol) + 2.0 ** -23 * abs(float(want))
        close_grad(d, grad, terms, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_the_longest_row(mc, dev, dtype):
    """2^31 - 1 logits: 4 or 8 GiB in one row."""
    V, step = 2**31 - 1, 1 << 27
    x = torch.empty(1, V, dtype=dtype, device=dev)
    g = gen(dev, 12)
    for i in range(0, V, step):
        x[0, i: i + step].normal_(0.0, 3.0, generator=g)
    t = torch.tensor([V - 2], device=dev, dtype=torch.int32)
    x[0, V - 2], x[0, 1 << 30] = 20.0, 19.0
    m = float(x.max())
    s = sum(float((x[0, i: i + step].double() - m).exp().sum()) for i in range(0, V, step))
    z = float(x[0, V - 2]) - m
    l, stats = mc.token_logprobs_forward(x, t)
    assert abs(float(l) - (z - math.log(s))) <= 2.0 ** -20 + 2.0 ** -22 * (abs(z) + math.log(s))

    def gradient(d, a, taken):
        """d against a q less what is taken out of single elements."""
        for i in range(0, V, step):
            q = (x[0, i: i + step].double() - m).exp() / s
            want, terms = a * q, abs(a) * q
            for j, p in taken.items():
                if i <= j < i + step:
                    want[j - i] -= p
                    terms[j - i] += abs(p)
            close_grad(d[0, i: i + step], want, terms, dtype)

    one = torch.ones(1, device=dev)
    gradient(mc.token_logprobs_backward(x, t, stats, one), -1.0, {V - 2: -1.0})
    loss, logps, _, d = mc.policy_loss_forward_backward(x[None], t[None], one)
    assert abs(float(logps) - float(l)) <= 2.0 ** -20 + 2.0 ** -22 * (abs(z) + math.log(s))
    gradient(d.view(1, V), 1.0, {V - 2: 1.0})
    del d
    ids = torch.tensor([[0, V - 1, 1 << 30, V - 2]], device=dev, dtype=torch.int32)
    tl = torch.zeros(1, 4, device=dev)
    loss, d = mc.distillation_loss_forward_backward(x, ids, tl)
    lq = [float(x[0, j]) - m - math.log(s) for j in ids[0].tolist()]
    want = sum(0.25 * (math.log(0.25) - v) for v in lq)
    assert abs(float(loss) - want) <= 2.0 ** -19 + 2.0 ** -21 * (2.0 + max(abs(v) for v in lq))
    gradient(d, 1.0, {j: 0.25 for j in ids[0].tolist()})


def test_dloss_and_optional_outputs(mc, dev):
    """A dloss of 0 and of NaN; outputs that may be NULL."""
    import ctypes

    g = gen(dev, 13)
    x = logits_at(dev, g, (4, 5, 77), torch.float32)
    t = some_targets(dev, g, (4, 5), 77)
    A = torch.randn(4, generator=g, device=dev)
    ids = torch.randint(0, 77, (4, 5, 3), generator=g, device=dev, dtype=torch.int32)
    tl = torch.randn(4, 5, 3, generator=g, device=dev)
    ploss, rewards, pstats = mc.preference_loss_forward(x, t, ignore_index=PAD)
    loss, logps, metrics, stats = mc.policy_loss_forward(x, t, A, ignore_index=PAD)
    kl, kstats = mc.distillation_loss_forward(x, ids, tl)
    for v in (0.0, math.nan):
        dloss = torch.full((1,), v, device=dev)
        for d, on in ((mc.preference_loss_backward(x, t, pstats, dloss, ignore_index=PAD), t != -1),
                      (mc.policy_loss_backward(x, t, stats, dloss, ignore_index=PAD), t != -1),
                      (mc.policy_loss_forward_backward(x, t, A, ignore_index=PAD, dloss=dloss)[3], t != -1),
                      (mc.distillation_loss_backward(x, ids, tl, kstats, dloss), None),
                      (mc.distillation_loss_forward_backward(x, ids, tl, dloss=dloss)[1], None)):
            if v == 0.0:
                assert not d.any()
            else:
                assert torch.isnan(d if on is None else d[on]).all() and (on is None or not d[~on].any())
    L, lib = mc.ops._lib, mc.ops.lib()
    s = torch.cuda.current_stream().cuda_stream
    ws = torch.empty(1 << 20, dtype=torch.uint8, device=dev)
    p = lambda v: v.data_ptr()  # noqa: E731
    d = L.PreferenceDesc(2, 5, 77, PAD, L.MC_PREF_SIGMOID, 0, 0.1, 0.0, 0.0, L.MC_F32)
    out = torch.empty(1, device=dev)
    assert lib.mc_preference_loss_fwd(ctypes.byref(d), p(x), p(t), None, p(out), None, None, p(ws), ws.numel(), s) == 0
    assert torch.equal(out, ploss)
    d = L.PolicyDesc(4, 5, 77, PAD, 0, L.MC_MEAN_TOKENS, 0.2, 0.2, 0.0, 1.0, L.MC_F32)
    l = torch.empty(4, 5, device=dev)
    assert lib.mc_policy_loss_fwd(ctypes.byref(d), p(x), p(t), p(A), None, None, p(out), p(l), None, None, p(ws),
                                  ws.numel(), s) == 0
    assert torch.equal(out, loss) and torch.equal(l, logps)
    dx, out2 = torch.empty_like(x), torch.empty(1, device=dev)
    assert lib.mc_policy_loss_fwd_bwd(ctypes.byref(d), p(x), p(t), p(A), None, None, None, p(out2), p(l), None, p(dx),
                                      p(ws), ws.numel(), s) == 0
    got = mc.policy_loss_forward_backward(x, t, A, ignore_index=PAD)
    assert torch.equal(out2, got[0]) and torch.equal(dx, got[3])
    d = L.DistillDesc(20, 77, 3, 1.0, L.MC_F32)
    assert lib.mc_distill_loss_fwd(ctypes.byref(d), p(x), p(ids), p(tl), None, None, p(out), None, p(ws), ws.numel(),
                                   s) == 0
    assert torch.equal(out, kl)


@pytest.mark.parametrize("rows,B", [(20000, 5), (9000, 9000)])
def test_many_rows(mc, dev, rows, B):
    """Sums over more rows than one workgroup takes, counts by a kernel of their own."""
    V, g = 37, gen(dev, rows)
    x, t, l64, tol, q, old, ref, A = policy_case(dev, B, rows // B, V, torch.float32, 0, False, 1.0, rows)
    for kw in (dict(kl_coef=0.1), dict(kl_coef=0.1, reduction="sequences")):
        outs = mc.policy_loss_forward_backward(x, t, A, old, ref, ignore_index=PAD, **kw)
        check_policy(mc, dev, x, t, l64, tol, q, A, old, ref, kw, outs, 1.0, torch.float32)
        loss, logps, metrics, stats = mc.policy_loss_forward(x, t, A, old, ref, ignore_index=PAD, **kw)
        d = mc.policy_loss_backward(x, t, stats, ignore_index=PAD)
        check_policy(mc, dev, x, t, l64, tol, q, A, old, ref, kw, (loss, logps, metrics, d), 1.0, torch.float32)
    ids = torch.randint(0, V, (rows, 3), generator=g, device=dev, dtype=torch.int32)
    tl = torch.randn(rows, 3, generator=g, device=dev)
    for mask in (None, (torch.rand(rows, generator=g, device=dev) < 0.5).to(torch.uint8)):
        want, dtol, grad, terms = plain_distill(x.view(rows, V), ids, tl, 1.0, None, mask)
        for loss, d in (mc.distillation_loss_forward_backward(x.view(rows, V), ids, tl, mask=mask),):
            assert abs(float(loss) - float(want)) <= float(dtol) + 2.0 ** -23 * abs(float(want))
            close_grad(d, grad, terms, torch.float32)
    y, ty = (x[:-1], t[:-1]) if B % 2 else (x, t)
    loss, rewards, _ = mc.preference_loss_forward(y.contiguous(), ty.contiguous(), beta=0.01, ignore_index=PAD)
    want, r64 = plain_preference(l64[: y.shape[0]], ty, None, 0.01, "sigmoid", 0.0, 0.0, False)
    close(rewards, r64, 0.01 * tol[: y.shape[0]].sum(1) + 2.0 ** -23 * r64.abs(), "rewards")
    assert abs(float(loss) - float(want)) <= 1e-5 * float(want)


@pytest.mark.parametrize("rows", [1 << 22, (1 << 24) - 1])
def test_rows_past_a_launch_of_large_workgroups(mc, dev, rows):
    """2^32 work-items: rows that 1024 threads each no longer launch, and the most rows there may be."""
    V = 3
    x, t, l64, tol, q, old, ref, A = policy_case(dev, rows // 5 if rows % 5 == 0 else 1, 5 if rows % 5 == 0 else rows,
                                                 V, torch.bfloat16, 0, True, 1.0, rows)
    kw = dict(kl_coef=0.1, reduction="sequences")
    outs = mc.policy_loss_forward_backward(x, t, A, old, ref, ignore_index=PAD, **kw)
    check_policy(mc, dev, x, t, l64, tol, q, A, old, ref, kw, outs, 1.0, torch.bfloat16)
    del outs, l64, tol, q, old, ref
    flat, g = x.view(rows, V), gen(dev, 1)
    ids = torch.randint(0, V, (rows, 2), generator=g, device=dev, dtype=torch.int32)
    tl = torch.randn(rows, 2, generator=g, device=dev)
    loss, d = mc.distillation_loss_forward_backward(flat, ids, tl)
    want, dtol, grad, terms = plain_distill(flat, ids, tl, 1.0, None, None)
    assert abs(float(loss) - float(want)) <= float(dtol) + 2.0 ** -23 * abs(float(want))
    close_grad(d, grad, terms, torch.bfloat16)


# ------------------------------------------------------- differences, together
def losses_of(mc, name, x, extra):
    """(loss, dlogits) of one of the losses on [4, 5, V]."""
    t, A, old, ref, ids, tl = extra
    if name == "preference":
        loss, _, stats = mc.preference_loss_forward(x, t, ref, 0.5, ignore_index=PAD)
        return loss, mc.preference_loss_backward(x, t, stats, ignore_index=PAD)
    if name == "policy":
        loss, _, _, d = mc.policy_loss_forward_backward(x, t, A, old, ref, clip_high=2.0, clip_low=0.9, kl_coef=0.2,
                                                        temperature=1.2, ignore_index=PAD)
        return loss, d
    if name == "distillation":
        return mc.distillation_loss_forward_backward(x, ids, tl, 1.5)
    l, stats = mc.token_logprobs_forward(x, t, ignore_index=PAD)
    return (l * A).sum().reshape(1), mc.token_logprobs_backward(x, t, stats, A, ignore_index=PAD)


@pytest.mark.parametrize("name", ["logprobs", "preference", "policy", "distillation"])
def test_gradient_against_differences(mc, dev, name):
    """Along random directions v of unit entries: (L(x + h v) - L(x - h v)) / 2h = <g, v> up to h^2 L''' / 6 and the
    loss's own rounding over h. With h = 2^-6 the first is below 2^-12 of the terms' sizes (derivatives of exp are of
    its own size) and the second 2^-20 (|L| + 8) / h."""
    g = gen(dev, 8)
    x = torch.randn(4, 5, 23, generator=g, device=dev)
    t = some_targets(dev, g, (4, 5), 23)
    l64, _, _ = plain_logps(x, t, 1.2 if name == "policy" else 1.0)
    extra = (t, torch.randn(4, 5, generator=g, device=dev), (l64 + 0.05).float(), (l64 - 0.2).float(),
             torch.randint(0, 23, (4, 5, 6), generator=g, device=dev, dtype=torch.int32),
             torch.randn(4, 5, 6, generator=g, device=dev))
    loss, d = losses_of(mc, name, x, extra)
    h = 2.0 ** -6
    for _ in range(4):
        v = torch.randint(0, 2, x.shape, generator=g, device=dev).float() * 2 - 1
        up, down = (float(losses_of(mc, name, x + s * h * v, extra)[0]) for s in (1, -1))
        want = float((d.double() * v).sum())
        size = float(d.double().abs().sum())
        assert abs((up - down) / (2 * h) - want) <= 2.0 ** -10 * size + 2.0 ** -20 * (abs(float(loss)) + 8) / h


def sequence(mc, c):
    """A step as a user runs it: the reference's and the old policy's log-probabilities, every loss, the gradient into
    the adapter that made the logits."""
    x, t, h = c["x"], c["t"], c["hidden"]
    y, saved = mc.lora_forward(h, c["A"], c["B"], 2.0, W=c["W"])
    y = y.view(x.shape)
    ref, _ = mc.token_logprobs_forward(x, t, ignore_index=PAD, save_stats=False)
    loss, rewards, stats = mc.preference_loss_forward(y, t, ref, 0.5, ignore_index=PAD)
    d1 = mc.preference_loss_backward(y, t, stats, ignore_index=PAD)
    ploss, logps, metrics, d2 = mc.policy_loss_forward_backward(y, t, c["adv"], ref, ref, kl_coef=0.1,
                                                                reduction="sequences", ignore_index=PAD)
    ploss2, _, _, pstats = mc.policy_loss_forward(y, t, c["adv"], ref, ref, kl_coef=0.1, ignore_index=PAD)
    d3 = mc.policy_loss_backward(y, t, pstats, c["dloss"], ignore_index=PAD)
    dloss, d4 = mc.distillation_loss_forward_backward(y, c["ids"], c["tl"], 2.0, mask=c["mask"])
    dloss2, dstats = mc.distillation_loss_forward(y, c["ids"], c["tl"], 2.0, mask=c["mask"])
    d5 = mc.distillation_loss_backward(y, c["ids"], c["tl"], dstats, c["dloss"], 2.0, mask=c["mask"])
    dX, dA, dB = mc.lora_backward(h, c["A"], c["B"], d1.view(-1, x.shape[-1]), 2.0, W=c["W"], h_save=saved)
    return [y, ref, loss, rewards, d1, ploss, logps, metrics, d2, ploss2, d3, dloss, d4, dloss2, d5, dX, dA, dB]


def sequence_case(dev, dtype=torch.bfloat16):
    g = gen(dev, 9)
    B, S, V, K, r = 4, 33, 1504, 96, 8
    c = {"x": logits_at(dev, g, (B, S, V), dtype), "t": some_targets(dev, g, (B, S), V)}
    c["hidden"] = torch.randn(B * S, K, generator=g, device=dev).to(dtype)
    c["W"] = (torch.randn(V, K, generator=g, device=dev) * 0.2).to(dtype)
    c["A"] = torch.randn(K, r, generator=g, device=dev) * 0.1
    c["B"] = torch.randn(r, V, generator=g, device=dev) * 0.1
    c["adv"] = torch.randn(B, generator=g, device=dev)
    c["dloss"] = torch.full((1,), 0.5, device=dev)
    c["ids"] = torch.randint(0, V, (B, S, 20), generator=g, device=dev, dtype=torch.int32)
    c["tl"] = torch.randn(B, S, 20, generator=g, device=dev)
    c["mask"] = (torch.rand(B, S, generator=g, device=dev) < 0.8).to(torch.uint8)
    return c


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_step_of_them_together(mc, dev, dtype):
    """Each loss on logits that a LoRA linear made, and the preference gradient back into the adapter."""
    c = sequence_case(dev, dtype)
    y, ref, loss, rewards, d1, _, _, _, _, _, _, dloss, d4, dloss2, d5, _, dA, dB = sequence(mc, c)
    t = c["t"]
    l64, tol, q = plain_logps(y, t)
    l = l64.clone().requires_grad_()
    want, _ = plain_preference(l, t, ref, 0.5, "sigmoid", 0.0, 0.0, False)
    want.backward()
    want = want.detach()
    assert abs(float(loss) - float(want)) <= 0.5 * float(tol.sum())
    close_grad(d1, *[v * 1.0 for v in plain_grad(q, t, l.grad)], dtype)
    # the adapter's gradients from the gradient of the logits, in 64 bits
    d, h, A, Bm = (v.double() for v in (d1.view(-1, y.shape[-1]), c["hidden"], c["A"], c["B"]))
    for got, wanted in ((dA, h.t() @ (2.0 * d @ Bm.t())), (dB, (2.0 * h @ A).t() @ d)):
        tolerance = 1e-5 if dtype == torch.float32 else 2e-2  # the linear's own
        assert float((got.double() - wanted).abs().max()) <= tolerance * float(wanted.abs().max())
    flat = (y.view(-1, y.shape[-1]), c["ids"].view(-1, 20), c["tl"].view(-1, 20), 2.0, None, c["mask"].view(-1))
    dw, dtol, dg, dterms = plain_distill(*flat)
    for v, grad, k in ((dloss, d4, 1.0), (dloss2, d5, 0.5)):
        assert abs(float(v) - float(dw)) <= float(dtol) + 2.0 ** -23 * abs(float(dw))
        close_grad(grad.view_as(dg), k * dg, k * dterms, dtype)


def test_results_repeat_and_replay(mc, dev):
    """Bitwise the same in a second call, on another stream, and in every replay of a captured graph with eager calls
    in between."""
    c = sequence_case(dev)
    eager = [o.clone() for o in sequence(mc, c)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = [o.clone() for o in sequence(mc, c)]
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for i, (a, b) in enumerate(zip(other, eager)):
        assert torch.equal(a, b), f"output {i} on another stream"
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = sequence(mc, c)
    torch.cuda.synchronize()
    for rep in range(3):
        between = sequence(mc, c)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for i, (a, b, e) in enumerate(zip(outs, between, eager)):
            assert torch.equal(a, e), f"replay {rep}: output {i}"
            assert torch.equal(b, e), f"eager call between replays: output {i}"


def test_calls_at_once_on_two_streams(mc, dev):
    """Calls that overlap share nothing."""
    c = sequence_case(dev)
    eager = [o.clone() for o in sequence(mc, c)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(sequence(mc, c))
    torch.cuda.synchronize()
    for n, got in enumerate(outs):
        for i, (a, e) in enumerate(zip(got, eager)):
            assert torch.equal(a, e), f"call {n}: output {i}"
            assert torch.equal(a, e), f"call {n}: output {i}"


# ------------------------------------------------------- small differences
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("with_lse", [False, True])
@pytest.mark.parametrize("T,shift", [(0.7, 0.0), (0.7, 100.0), (1.5, 100.0), (3.0, 0.0), (1.0, 100.0)])
def test_distillation_near_its_teacher(mc, dev, nan_outputs, dtype, with_lse, T, shift):
    """A student within 5e-3 of its teacher's logits, whose own lie anywhere: the KL is about 1e-5 of a log-probability,
    and the loss is held to that.

    The value has two roundings: the float sums of a row's exponentials, at most 32 in a chain, each of at most 2^-24
    of the sum and of either sign, so 2^-24 sqrt(32 / 3) < 2^-22 (rms) for a row and 6 times that over sqrt(rows) for
    their mean; and the mean error of the hardware exponential, below 2^-28. An element of the gradient is
    w (P q - p), in units of 2^-24: q = exp2((x - m) c) / s has three roundings of its argument, 3 |z|, 2 of the
    exponential, 32 of s and at most 6 of the factors; p and w p have 6."""
    rows, V, K = 2000, 4096, 64
    T = float(torch.tensor(T))  # as the call takes it
    g = gen(dev, 21)
    x = torch.randn(rows, V, generator=g, device=dev).mul_(2.0).add_(8.0 - 30.0 * T)
    ids = (torch.randint(0, V, (rows, 1), generator=g, device=dev) + V // K * torch.arange(K, device=dev)) % V
    best = 8.0 - 1.5 * torch.arange(1, K + 1, device=dev).log() + 0.5 * torch.randn(rows, K, generator=g, device=dev)
    x = x.scatter_(1, ids, best).to(dtype)
    t = x.float().gather(1, ids) + shift + 5e-3 * torch.randn(rows, K, generator=g, device=dev)
    lse = torch.logsumexp(t.double() / T, 1).float() if with_lse else None
    want, _, grad, terms = plain_distill(x, ids, t, T, lse, None)
    z = plain_rows(x, T)[0].abs()
    dense, taken = (terms + grad) / 2, (terms - grad) / 2
    gtol = 2.0 ** -24 * ((3 * z + 40) * dense + 6 * taken) + torch.finfo(dtype).eps / 2 * grad.abs() + 1e-37
    ids = ids.to(torch.int32)
    loss, stats = mc.distillation_loss_forward(x, ids, t, T, lse)
    d = mc.distillation_loss_backward(x, ids, t, stats, None, T, lse)
    for name, v, dv in (("two calls", loss, d), ("one call", *mc.distillation_loss_forward_backward(x, ids, t, T, lse))):
        assert abs(float(v) - float(want)) <= T * T * (6 * 2.0 ** -22 / rows ** 0.5 + 2.0 ** -28) + \
            2.0 ** -24 * abs(float(want)), (name, float(v), float(want))
        close(dv, grad, gtol, name)


@pytest.mark.parametrize("B,S,V", [(4, 256, 2000), (2, 16, 60001)])
def test_policy_near_its_reference(mc, dev, nan_outputs, B, S, V):
    """A group without advantages, 1e-3 from its reference: the KL term is the whole gradient, -kl_coef expm1(ref - l),
    and as exact as l is in 64 bits but for the float sums of a row's exponentials, below 2^-22 (rms: 32 roundings of
    at most 2^-24 of the sum and of either sign)."""
    g = gen(dev, 22)
    T, kc = 0.5, 0.1
    x = logits_at(dev, g, (B, S, V), torch.float32, std=4.0)
    t = some_targets(dev, g, (B, S), V)
    l64, _, q = plain_logps(x, t, T)
    ref = (l64 + 1e-3 * torch.randn(B, S, generator=g, device=dev)).float()
    A, on = torch.zeros(B, device=dev), t != -1
    kw = dict(ref_logps=ref, kl_coef=kc, temperature=T, ignore_index=PAD)
    stats = mc.policy_loss_forward(x, t, A, **kw)[3]
    at = t.long().clamp(min=0)[..., None]
    want = torch.expm1(ref.double() - l64) * (1.0 - q.gather(2, at)[..., 0])
    for name, d in (("two calls", mc.policy_loss_backward(x, t, stats, temperature=T, ignore_index=PAD)),
                    ("one call", mc.policy_loss_forward_backward(x, t, A, **kw)[3])):
        got = d.gather(2, at)[..., 0].double() * (-T * float(on.sum()) / kc)
        rms = float((got - want)[on].square().mean().sqrt())
        assert rms <= 2.0 ** -22, (name, rms)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,S,V", [(4, 256, 2000), (2, 16, 60001)])
def test_policy_clips_its_gradient_and_its_value_alike(mc, dev, nan_outputs, dtype, B, S, V):
    """Ratios within a rounding of the borders: the tokens without a gradient are those that the metric counts."""
    g = gen(dev, 23)
    x = logits_at(dev, g, (B, S, V), dtype, std=4.0)
    t = some_targets(dev, g, (B, S), V)
    T, on = 0.5, t != -1
    l64, _, _ = plain_logps(x, t, T)
    up = torch.rand(B, S, generator=g, device=dev) < 0.5
    old = (l64 - torch.where(up, math.log1p(0.2), math.log1p(-0.2))).float()
    A = torch.where(up, 1.0, -1.0)
    kw = dict(old_logps=old, temperature=T, ignore_index=PAD)
    _, _, metrics2, stats = mc.policy_loss_forward(x, t, A, **kw)
    _, _, metrics, d = mc.policy_loss_forward_backward(x, t, A, **kw)
    n = int(on.sum())
    for name, dv, m in (("two calls", mc.policy_loss_backward(x, t, stats, temperature=T, ignore_index=PAD), metrics2),
                        ("one call", d, metrics)):
        held = int((on & ~(dv != 0).any(-1)).sum())
        assert held == round(float(m[1]) * n), (name, held, float(m[1]) * n)
        assert B * S < 64 or 0 < held < n


def test_token_logprobs_of_targets_in_another_shape(mc, dev):
    """Targets may come flat or folded in another way: the log-probabilities have the logits' leading dims."""
    g = gen(dev, 24)
    x = logits_at(dev, g, (2, 3, 101), torch.float32)
    t = torch.randint(0, 101, (2, 3), generator=g, device=dev, dtype=torch.int32)
    want, stats = mc.token_logprobs_forward(x, t)
    dl = torch.randn(2, 3, generator=g, device=dev)
    d = mc.token_logprobs_backward(x, t, stats, dl)
    for shape in ((6,), (3, 2), (1, 6), (6, 1)):
        got, _ = mc.token_logprobs_forward(x, t.view(shape))
        assert got.shape == (2, 3) and torch.equal(got, want), shape
        assert torch.equal(mc.token_logprobs_backward(x, t.view(shape), stats, dl), d), shape


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,V", WAYS)
@pytest.mark.parametrize("K", [1, 64, 65, 256])
def test_near_teachers_of_every_size_and_way(mc, dev, nan_outputs, dtype, rows, V, K):
    """As test_distillation_near_its_teacher, for every way of taking a row, with the teacher's log-sum-exp and
    without. Without it, and of one entry, p is 1 and the value -log q: held to the chain's worst case, 32 roundings of
    2^-24."""
    g = gen(dev, rows + K)
    T, shift = 0.5, -50.0
    x = torch.randn(rows, V, generator=g, device=dev).mul_(2.0).add_(-12.0)
    ids = (torch.randint(0, V, (rows, 1), generator=g, device=dev) + max(1, V // K) * torch.arange(K, device=dev)) % V
    best = 8.0 - 1.5 * torch.arange(1, K + 1, device=dev).log() + 0.5 * torch.randn(rows, K, generator=g, device=dev)
    x = x.scatter_(1, ids, best).to(dtype)
    t = x.float().gather(1, ids) + shift + 5e-3 * torch.randn(rows, K, generator=g, device=dev)
    t[rows // 2, K // 2:] = -math.inf
    full = (torch.logsumexp(t.double() / T, 1)).float()
    full[rows // 2] = 0.0
    z = plain_rows(x, T)[0].abs()
    for lse in (None, full):
        want, _, grad, terms = plain_distill(x, ids, t, T, lse, None)
        dense, taken = (terms + grad) / 2, (terms - grad) / 2
        gtol = 2.0 ** -24 * ((3 * z + 40) * dense + 6 * taken) + torch.finfo(dtype).eps / 2 * grad.abs() + 1e-37
        loss, stats = mc.distillation_loss_forward(x, ids, t, T, lse)
        d = mc.distillation_loss_backward(x, ids, t, stats, None, T, lse)
        for name, v, dv in (("two calls", loss, d),
                            ("one call", *mc.distillation_loss_forward_backward(x, ids, t, T, lse))):
            assert abs(float(v) - float(want)) <= T * T * (32 * 2.0 ** -24 + 2.0 ** -28) + \
                2.0 ** -24 * abs(float(want)), (name, float(v), float(want))
            close(dv, grad, gtol, name)


@pytest.mark.parametrize("dtype", DTYPES)
def test_distillation_entries_of_no_weight(mc, dev, nan_outputs, dtype):
    """Teacher entries at the type's lowest value, whose p underflows to 0: as left out, whatever their id. A teacher
    whose entries are all that low is uniform."""
    V, K, g = 300, 70, gen(dev, 25)
    low = torch.finfo(torch.float32).min
    x = logits_at(dev, g, (5, V), dtype)
    ids = torch.stack([torch.randperm(V, generator=g, device=dev)[:K] for _ in range(5)]).to(torch.int32)
    t = torch.randn(5, K, generator=g, device=dev)
    t[1, 3:], t[2, ::2], t[3] = low, low, low
    clean = torch.where((t == low) & (t != low).any(1, keepdim=True), -math.inf, t)
    want, tol, grad, terms = plain_distill(x, ids, torch.where(clean == low, 0.0, clean), 1.0, None, None)
    bad = ids.clone()
    bad[1, 3:], bad[2, ::2] = 2**31 - 1, -1
    for i in (ids, bad):
        loss, stats = mc.distillation_loss_forward(x, i, t)
        for v, d in ((loss, mc.distillation_loss_backward(x, i, t, stats)),
                     mc.distillation_loss_forward_backward(x, i, t)):
            assert abs(float(v) - float(want)) <= float(tol) + 2.0 ** -23 * abs(float(want))
            close_grad(d, grad, terms, dtype)


@pytest.mark.parametrize("ids", [torch.int32, torch.int64])
def test_padding_of_minus_100(mc, dev, ids):
    """Ids are unsigned: -100 is 2^32 - 100, and an ignore_index below 0 is none. (x_t - m) / T and log s are below 14
    each: 2^-20 + 2^-22 28 = 2^-17."""
    g = gen(dev, 26)
    x = logits_at(dev, g, (2, 5, 33), torch.float32)
    t = torch.randint(0, 33, (2, 5), generator=g, device=dev)
    t[0, :2], t[1, 4] = -100, -100
    l, _ = mc.token_logprobs_forward(x, t.to(ids), ignore_index=2**32 - 100)
    want = torch.log_softmax(x.double(), -1).gather(-1, t.clamp(min=0)[..., None])[..., 0]
    on = t != -100
    assert torch.allclose(l.double()[on], want[on], rtol=0.0, atol=2.0 ** -17) and not l[~on].any()
    l, _ = mc.token_logprobs_forward(x, t.to(ids), ignore_index=-100)
    assert torch.isnan(l[~on]).all() and torch.isfinite(l[on]).all()


@pytest.mark.parametrize("with_lse", [False, True])
@pytest.mark.parametrize("K", [5, 130])
def test_a_teacher_that_is_nan(mc, dev, nan_outputs, K, with_lse):
    """A NaN among a row's teacher logits, or an infinity without their log-sum-exp: the loss and that row are NaN."""
    V, g = 700, gen(dev, 27)
    x = logits_at(dev, g, (4, V), torch.bfloat16)
    ids = torch.stack([torch.randperm(V, generator=g, device=dev)[:K] for _ in range(4)]).to(torch.int32)
    t = torch.randn(4, K, generator=g, device=dev)
    lse = torch.logsumexp(t, 1) + 0.1 if with_lse else None
    t[1, K - 1] = math.nan if with_lse else math.inf
    t[2, 0] = math.nan
    loss, stats = mc.distillation_loss_forward(x, ids, t, teacher_lse=lse)
    for v, d in ((loss, mc.distillation_loss_backward(x, ids, t, stats, teacher_lse=lse)),
                 mc.distillation_loss_forward_backward(x, ids, t, teacher_lse=lse)):
        assert torch.isnan(v).all() and torch.isnan(d[1:3]).all() and torch.isfinite(d[[0, 3]]).all()
