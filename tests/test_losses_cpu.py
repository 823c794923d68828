"""Refusals of the losses over log-probabilities: the torch front end and the C
ABI check arguments on the host, before anything is enqueued."""
import ctypes

import pytest
import torch

SHAPE, DTYPE, LAYOUT, VALUE, NULL, WORKSPACE = 2, 3, 4, 5, 1, 6


def raises(mc, code, text, fn, *a, **k):
    with pytest.raises(mc.McError) as e:
        fn(*a, **k)
    assert e.value.code == code, e.value
    assert text in str(e.value), e.value


def test_token_logprobs_refusals(mc):
    x, t = torch.zeros(2, 3, 8), torch.zeros(2, 3, dtype=torch.int32)
    f, b = mc.token_logprobs_forward, mc.token_logprobs_backward
    raises(mc, NULL, "logits must be a tensor", f, None, t)
    raises(mc, NULL, "targets must be a tensor", f, x, None)
    raises(mc, DTYPE, "unsupported dtype torch.float16", f, x.half(), t)
    raises(mc, DTYPE, "targets have dtype torch.float32", f, x, t.float())
    raises(mc, SHAPE, "targets have 5 entries, expected 6", f, x, t.view(-1)[:5])
    raises(mc, LAYOUT, "logits must be contiguous", f, x.transpose(0, 1), t.t())
    raises(mc, SHAPE, "logits are empty", f, torch.zeros(0, 8), torch.zeros(0, dtype=torch.int32))
    raises(mc, SHAPE, "logits are empty", f, torch.zeros(3, 0), torch.zeros(3, dtype=torch.int32))
    raises(mc, SHAPE, "Input must have at least 1 dimension", f, torch.zeros(()), torch.zeros((), dtype=torch.int32))
    s, d = torch.zeros(6, 2), torch.zeros(2, 3)
    raises(mc, NULL, "stats and dlogps are required", b, x, t, None, d)
    raises(mc, NULL, "stats and dlogps are required", b, x, t, s, None)
    raises(mc, SHAPE, "stats has shape (6,)", b, x, t, s[:, 0].contiguous(), d)
    raises(mc, SHAPE, "dlogps has shape (6,)", b, x, t, s, d.view(-1))
    raises(mc, DTYPE, "dlogps has dtype torch.bfloat16", b, x, t, s, d.bfloat16())


def test_preference_refusals(mc):
    x, t = torch.zeros(4, 3, 8), torch.zeros(4, 3, dtype=torch.int32)
    f, b = mc.preference_loss_forward, mc.preference_loss_backward
    raises(mc, SHAPE, "logits must be [sequences, tokens, vocab]", f, x.view(12, 8), t.view(-1))
    raises(mc, SHAPE, "3 is odd", f, x[:3], t[:3])
    raises(mc, SHAPE, "targets has shape (12,)", f, x, t.view(-1))
    raises(mc, SHAPE, "ref_logps has shape (4,)", f, x, t, torch.zeros(4))
    raises(mc, DTYPE, "ref_logps has dtype torch.float64", f, x, t, torch.zeros(4, 3, dtype=torch.float64))
    raises(mc, VALUE, "kind must be one of sigmoid, hinge, squared", f, x, t, kind="ipo")
    raises(mc, VALUE, "kind must be one of", f, x, t, kind=["sigmoid"])
    raises(mc, SHAPE, "stats has shape (24,)", b, x, t, torch.zeros(24))
    raises(mc, SHAPE, "dloss has shape ()", b, x, t, torch.zeros(28), torch.zeros(()))
    raises(mc, NULL, "stats from preference_loss_forward", b, x, t, None)


def test_policy_refusals(mc):
    x, t, A = torch.zeros(4, 3, 8), torch.zeros(4, 3, dtype=torch.int32), torch.zeros(4)
    for f in (mc.policy_loss_forward, mc.policy_loss_forward_backward):
        raises(mc, NULL, "advantages must be a tensor", f, x, t, 1.0)
        raises(mc, SHAPE, "advantages has shape (3,), expected (4,)", f, x, t, torch.zeros(3))
        raises(mc, SHAPE, "advantages has shape (4, 1), expected (4, 3)", f, x, t, torch.zeros(4, 1))
        raises(mc, SHAPE, "old_logps has shape (12,)", f, x, t, A, torch.zeros(12))
        raises(mc, LAYOUT, "ref_logps must be contiguous", f, x, t, A, None, torch.zeros(3, 4).t())
        raises(mc, VALUE, "reduction must be one of tokens, sequences", f, x, t, A, reduction="sum")
    raises(mc, SHAPE, "stats has shape (36,)", mc.policy_loss_backward, x, t, torch.zeros(36))


def test_distillation_refusals(mc):
    x, ids, tl = torch.zeros(4, 3, 8), torch.zeros(4, 3, 5, dtype=torch.int32), torch.zeros(4, 3, 5)
    for f in (mc.distillation_loss_forward, mc.distillation_loss_forward_backward):
        raises(mc, NULL, "teacher_ids and teacher_logits must be tensors", f, x, None, tl)
        raises(mc, SHAPE, "teacher_ids has shape (12, 5)", f, x, ids.view(12, 5), tl)
        raises(mc, DTYPE, "teacher_ids has dtype torch.int16", f, x, ids.short(), tl)
        raises(mc, SHAPE, "teacher_logits has shape (4, 3, 4)", f, x, ids, tl[..., :4].contiguous())
        raises(mc, DTYPE, "teacher_logits has dtype torch.bfloat16", f, x, ids, tl.bfloat16())
        raises(mc, SHAPE, "teacher_lse has shape (12,)", f, x, ids, tl, 1.0, torch.zeros(12))
        raises(mc, DTYPE, "mask has dtype torch.bool", f, x, ids, tl, mask=torch.zeros(4, 3, dtype=torch.bool))
    raises(mc, SHAPE, "stats has shape (24,)", mc.distillation_loss_backward, x, ids, tl, torch.zeros(24))


FAKE = ctypes.c_void_p(256)



LIMIT = (2**32 - 1) // 256


@pytest.mark.parametrize("field,value,code,text", [
    ("rows", 0, SHAPE, "rows (0) must be in"), ("rows", LIMIT + 1, SHAPE, "must be in [1, 16777215]"),
    ("vocab", 0, SHAPE, "vocab (0)"), ("vocab", 2**31, SHAPE, "2^31 - 1"), ("dtype", 2, DTYPE, "unsupported dtype code"),
    ("temperature", 0.0, VALUE, "temperature must be in"), ("temperature", float("nan"), VALUE, "temperature"),
    ("temperature", float("inf"), VALUE, "temperature"), ("temperature", -1.0, VALUE, "temperature")])
def test_abi_logprobs(mc, field, value, code, text):
    L = mc._lib.lib()
    d = mc._lib.LogprobDesc(4, 8, -1, 1.0, 0)
    setattr(d, field, value)
    p = ctypes.byref(d)
    assert L.mc_token_logprobs_fwd(p, FAKE, FAKE, FAKE, FAKE, None, 0, None) == code and text in mc._lib.last_error()
    assert L.mc_token_logprobs_bwd(p, FAKE, FAKE, FAKE, FAKE, FAKE, None) == code
    if field in ("rows", "vocab", "dtype", "temperature") and hasattr(mc._lib.DistillDesc, field):
        e = mc._lib.DistillDesc(4, 8, 5, 1.0, 0)
        setattr(e, field, value)
        assert L.mc_distill_loss_workspace_size(ctypes.byref(e)) == 0
        assert L.mc_distill_loss_fwd(ctypes.byref(e), FAKE, FAKE, FAKE, None, None, FAKE, None, FAKE, 1 << 40, None) == code


def test_abi_null_layout_and_workspace(mc):
    L, S = mc._lib.lib(), mc._lib
    odd = ctypes.c_void_p(257)
    lp = ctypes.byref(S.LogprobDesc(4, 8, -1, 1.0, 1))
    assert L.mc_token_logprobs_fwd(None, FAKE, FAKE, FAKE, None, None, 0, None) == NULL
    assert L.mc_token_logprobs_fwd(lp, None, FAKE, FAKE, None, None, 0, None) == NULL
    assert L.mc_token_logprobs_fwd(lp, FAKE, FAKE, None, None, None, 0, None) == NULL
    assert L.mc_token_logprobs_fwd(lp, odd, FAKE, FAKE, None, None, 0, None) == LAYOUT
    few = S.LogprobDesc(1, 1 << 20, -1, 1.0, 1)
    need = L.mc_token_logprobs_workspace_size(ctypes.byref(few))
    assert need > 0 and L.mc_token_logprobs_workspace_size(lp) == 0
    assert L.mc_token_logprobs_fwd(ctypes.byref(few), FAKE, FAKE, FAKE, None, FAKE, need - 1, None) == WORKSPACE
    assert L.mc_token_logprobs_bwd(lp, FAKE, FAKE, None, FAKE, FAKE, None) == NULL
    assert L.mc_token_logprobs_bwd(lp, FAKE, FAKE, FAKE, FAKE, odd, None) == LAYOUT

    pd = S.PreferenceDesc(2, 3, 8, -1, 0, 0, 0.1, 0.0, 0.0, 1)
    p, need = ctypes.byref(pd), L.mc_preference_loss_workspace_size(ctypes.byref(pd))
    assert need > 0
    assert L.mc_preference_loss_fwd(p, FAKE, FAKE, None, None, None, None, FAKE, need, None) == NULL
    assert L.mc_preference_loss_fwd(p, FAKE, FAKE, None, FAKE, None, None, FAKE, need - 1, None) == WORKSPACE
    assert L.mc_preference_loss_fwd(p, FAKE, FAKE, None, FAKE, None, None, None, need, None) == WORKSPACE
    assert L.mc_preference_loss_fwd(p, FAKE, FAKE, None, FAKE, None, None, ctypes.c_void_p(264), need, None) == LAYOUT
    assert L.mc_preference_loss_bwd(p, FAKE, FAKE, None, None, FAKE, None) == NULL

    od = S.PolicyDesc(2, 3, 8, -1, 0, 0, 0.2, 0.2, 0.0, 1.0, 1)
    o = ctypes.byref(od)
    need, both = L.mc_policy_loss_workspace_size(o), L.mc_policy_loss_fwd_bwd_workspace_size(o)
    assert 0 < need <= both
    call = lambda A, loss, ws, n: L.mc_policy_loss_fwd(o, FAKE, FAKE, A, None, None, loss, FAKE, None, None, ws, n, None)  # noqa: E731
    assert call(None, FAKE, FAKE, need) == NULL
    assert call(FAKE, None, FAKE, need) == NULL
    assert call(FAKE, FAKE, FAKE, need - 1) == WORKSPACE
    assert L.mc_policy_loss_fwd_bwd(o, FAKE, FAKE, FAKE, None, None, None, FAKE, FAKE, None, FAKE, FAKE, both - 1, None) == WORKSPACE
    assert L.mc_policy_loss_fwd_bwd(o, FAKE, FAKE, FAKE, None, None, None, FAKE, FAKE, None, None, FAKE, both, None) == NULL
    od.kl_coef = 0.1
    assert call(FAKE, FAKE, FAKE, need) == NULL and "requires ref_logps" in mc._lib.last_error()
    od.kl_coef, od.reduction = 0.0, 1
    assert L.mc_policy_loss_workspace_size(o) > 0

    dd = S.DistillDesc(6, 8, 5, 1.0, 1)
    q = ctypes.byref(dd)
    need, both = L.mc_distill_loss_workspace_size(q), L.mc_distill_loss_fwd_bwd_workspace_size(q)
    assert 0 < need <= both
    assert L.mc_distill_loss_fwd(q, FAKE, None, FAKE, None, None, FAKE, None, FAKE, need, None) == NULL
    assert L.mc_distill_loss_fwd(q, FAKE, FAKE, FAKE, None, None, FAKE, None, FAKE, need - 1, None) == WORKSPACE
    assert L.mc_distill_loss_fwd_bwd(q, FAKE, FAKE, FAKE, None, None, None, FAKE, FAKE, FAKE, both - 1, None) == WORKSPACE
    assert L.mc_distill_loss_bwd(q, FAKE, FAKE, FAKE, None, None, None, None, FAKE, None) == NULL
    for top in (0, 257):
        dd.top = top
        assert L.mc_distill_loss_workspace_size(q) == 0 and "teacher entries per row" in mc._lib.last_error()


@pytest.mark.parametrize("field,value,code,text", [
    ("pairs", 0, SHAPE, "rows (0)"), ("pairs", -(2**63), SHAPE, "rows (0)"), ("pairs", LIMIT, SHAPE, "rows"),
    ("seq", 0, SHAPE, "rows (0)"), ("kind", 3, VALUE, "unknown kind 3"), ("average", 2, VALUE, "average must be 0 or 1"),
    ("beta", 0.0, VALUE, "beta must be positive"), ("beta", float("nan"), VALUE, "beta"),
    ("label_smoothing", 1.0, VALUE, "label_smoothing must be in [0, 1)"), ("margin", float("inf"), VALUE, "margin must be finite")])
def test_abi_preference_values(mc, field, value, code, text):
    L = mc._lib.lib()
    d = mc._lib.PreferenceDesc(2, 3, 8, -1, 0, 0, 0.1, 0.0, 0.0, 1)
    setattr(d, field, value)
    assert L.mc_preference_loss_workspace_size(ctypes.byref(d)) == 0
    assert text in mc._lib.last_error()
    assert L.mc_preference_loss_fwd(ctypes.byref(d), FAKE, FAKE, None, FAKE, None, None, FAKE, 1 << 40, None) == code


def test_abi_preference_kinds(mc):
    L = mc._lib.lib()
    for kind, eps, margin, text in ((1, 0.1, 0.0, "belongs to the sigmoid loss"), (2, 0.0, 0.5, "has no margin")):
        d = mc._lib.PreferenceDesc(2, 3, 8, -1, kind, 0, 0.1, eps, margin, 1)
        assert L.mc_preference_loss_workspace_size(ctypes.byref(d)) == 0
        assert text in mc._lib.last_error()


@pytest.mark.parametrize("field,value,code,text", [
    ("batch", 0, SHAPE, "rows (0)"), ("seq", 2**40, SHAPE, "rows (0)"), ("per_token_advantages", 2, VALUE, "per_token"),
    ("reduction", 2, VALUE, "unknown reduction"), ("clip_low", 1.5, VALUE, "clip_low"), ("clip_low", -0.1, VALUE, "clip_low"),
    ("clip_high", float("inf"), VALUE, "clip_high"), ("kl_coef", -0.1, VALUE, "kl_coef"),
    ("kl_coef", float("nan"), VALUE, "kl_coef"), ("temperature", 0.0, VALUE, "temperature")])
def test_abi_policy_values(mc, field, value, code, text):
    L = mc._lib.lib()
    d = mc._lib.PolicyDesc(2, 3, 8, -1, 0, 0, 0.2, 0.2, 0.0, 1.0, 1)
    setattr(d, field, value)
    assert L.mc_policy_loss_fwd_bwd_workspace_size(ctypes.byref(d)) == 0
    assert text in mc._lib.last_error()
    assert L.mc_policy_loss_bwd(ctypes.byref(d), FAKE, FAKE, FAKE, None, FAKE, None) == code
