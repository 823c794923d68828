"""Attention over packed rows in 64 bits, with bounds on what the kernels may be off
by, one (batch, head) at a time.

With u = 2^-24 and e half a step of the tensors' type (bf16 2^-8, float32 2^-24), a
score is off by at most
  d = u ((D + 8) max(scale |q| |k|) + 16 max|x| + 16 cap)
(D products summed in float32; the exponent's argument, lse and the bias rounded at
their size; tanh to a few u, times the cap), so a probability by 2 d of its value
(its own and its row's sum), and
  r = 2 d + (S + D) u        for the sums over keys or queries,
  p = e for bf16, whose P and dS are rounded before their products, else 0.
  o    (r + p) sum_j P |v| + e |o|
  dv   (r + p) sum_i P |do| + e |dv|
  dS   (r + p) |dS| + P s (Eo |do| + r |do| |v| + 8 u (|dP| + |Delta|)), s the cap's
       slope (<= 1, itself off by 8 u), Eo the bound of o, from which Delta is formed;
       where Delta is formed from P and dP (exact), r sum_j P |dP| in place of Eo |do|
  dq   scale (sum_j E_dS |k| + (S + D) u sum_j |dS| |k|) + e |dq|, dk alike over the
       queries, summed over the heads that share the key
"""
import math

import torch

U = 2.0**-24


def visible(S, documents=None, prefix=None, causal=True):
    """[S, S] truth values, token by token from the definition."""
    ids = [0] * S if documents is None else [int(x) for x in documents]
    see = torch.zeros(S, S, dtype=torch.bool)
    t = 0
    while t < S:
        end = t
        while end < S and ids[end] == ids[t]:
            end += 1
        if ids[t] >= 0:
            see[t:end, t:end] = True
            if causal:
                see[t:end, t:end] = torch.ones(end - t, end - t, dtype=torch.bool).tril()
            prompt = t
            while prefix is not None and prompt < end and prefix[prompt]:
                prompt += 1
            see[t:prompt, t:prompt] = True
        t = end
    return see


def spans_of(see):
    """[S, 4] of a visibility matrix whose rows and columns are intervals."""
    S = see.shape[0]
    out = torch.zeros(S, 4, dtype=torch.int32)
    for side, m in ((0, see), (2, see.t())):
        for t in range(S):
            at = m[t].nonzero()[:, 0]
            if len(at):
                out[t, side], out[t, side + 1] = int(at[0]), int(at[-1]) + 1
                assert int(at[-1]) + 1 - int(at[0]) == len(at)
    return out


def attention(q, k, v, see, scale, cap=None, slopes=None, dout=None, exact=False):
    """{name: (value, bound)} of o, lse and, with dout, dq, dk, dv; see [B, S, S] truth values."""
    B, H, S, D = q.shape
    Hkv = k.shape[1]
    rep, dt = H // Hkv, q.dtype
    e = 2.0**-8 if dt == torch.bfloat16 else U
    pr = e if dt == torch.bfloat16 else 0.0
    zero = lambda *s: torch.zeros(s, dtype=torch.float64, device=q.device)  # noqa: E731
    o, Eo, lse, El = zero(B, S, H, D), zero(B, S, H, D), zero(B, H, S), zero(B, H, S)
    dq, Eq, dk, Ek, dv, Ev = (zero(*s.shape) for s in (q, q, k, k, k, k))
    at = torch.arange(S, dtype=torch.float64, device=q.device)
    for b in range(B):
        m = see[b].to(q.device)
        row = m.any(-1)
        for h in range(H):
            Q, K, V = (x.double() for x in (q[b, h], k[b, h // rep], v[b, h // rep]))
            # what no pair meets plays no part
            Q = torch.where(row[:, None], Q, 0.0)
            K, V = (torch.where(m.any(0)[:, None], x, 0.0) for x in (K, V))
            x = scale * (Q @ K.t())
            A = float((scale * (Q.abs() @ K.abs().t())).max())
            s = torch.ones_like(x)
            if cap:
                t = torch.tanh(x / cap)
                x, s = cap * t, 1.0 - t * t
            if slopes is not None:
                x = x - slopes[h].double() * (at[:, None] - at).abs()
            X = float(x[m].abs().max()) if m.any() else 0.0
            x = torch.where(m, x, -math.inf)
            top = torch.where(row, x.amax(-1), 0.0)
            p = torch.exp(x - top[:, None])
            total = p.sum(-1)
            p = p / torch.where(row, total, 1.0)[:, None]
            d = U * ((D + 8) * A + 16 * X + 16 * (cap or 0.0))
            r = 2 * d + (S + D) * U
            O = p @ V
            o[b, :, h], Eo[b, :, h] = O, (r + pr) * (p @ V.abs()) + e * O.abs()
            lse[b, h] = torch.where(row, top + torch.log(torch.where(row, total, 1.0)), -math.inf)
            El[b, h] = d + (S + 4) * U + 4 * U * torch.where(row, lse[b, h], 0.0).abs()
            if dout is None:
                continue
            G = torch.where(row[:, None], dout.view(B, S, H, D)[b, :, h].double(), 0.0)
            dP, delta = G @ V.t(), (G * O).sum(-1, keepdim=True)
            dS = p * (dP - delta) * s
            off = r * (p * dP.abs()).sum(-1) if exact else (Eo[b, :, h] * G.abs()).sum(-1)
            EdS = (r + pr) * dS.abs() + p * s * (off[:, None] + r * (G.abs() @ V.abs().t()))
            EdS = EdS + 8 * U * p * (dP.abs() + delta.abs())
            dq[b, h] = scale * (dS @ K)
            Eq[b, h] = scale * ((EdS + (S + D) * U * dS.abs()) @ K.abs()) + e * dq[b, h].abs()
            n = h // rep
            dk[b, n] += scale * (dS.t() @ Q)
            Ek[b, n] += scale * ((EdS + (S + D) * U * dS.abs()).t() @ Q.abs())
            dv[b, n] += p.t() @ G
            Ev[b, n] += (r + pr) * (p.t() @ G.abs())
    got = {"o": (o.view(B, S, H * D), Eo.view(B, S, H * D)), "lse": (lse, El)}
    if dout is not None:
        got.update(dq=(dq, Eq), dk=(dk, Ek + e * dk.abs()), dv=(dv, Ev + e * dv.abs()))
    return got


def check(got, want):
    for name, x in got.items():
        value, bound = want[name]
        x = x.double()
        same = (x == value) | ((x - value).abs() <= bound * 1.01 + 1e-37)
        assert same.all(), (name, int((~same).sum()), float(((x - value).abs() / (bound + 1e-37)).nan_to_num(1e9).max()))
