"""Refusals of the attention over packed rows: the torch front end and the C ABI
check arguments on the host, before anything is enqueued. The 64-bit reference
of the GPU tests is checked here against automatic differentiation."""
import ctypes
import math

import pytest
import torch

import packed_reference as ref

NULL, SHAPE, DTYPE, LAYOUT, VALUE, WORKSPACE = 1, 2, 3, 4, 5, 6
FAKE = ctypes.c_void_p(256)


def raises(mc, code, text, fn, *a, **k):
    with pytest.raises(mc.McError) as e:
        fn(*a, **k)
    assert e.value.code == code, e.value
    assert text in str(e.value), e.value


def test_spans_refusals(mc):
    ids, flags = torch.zeros(2, 5, dtype=torch.int32), torch.zeros(2, 5, dtype=torch.uint8)
    f = mc.attention_spans
    raises(mc, NULL, "documents or prefix is required", f)
    raises(mc, SHAPE, "must be [batch, seq]", f, ids[0])
    raises(mc, SHAPE, "must be [batch, seq]", f, ids[:, :0])
    raises(mc, DTYPE, "documents has dtype torch.int64", f, ids.long())
    raises(mc, LAYOUT, "documents must be contiguous", f, ids.t())
    raises(mc, SHAPE, "prefix has shape (2, 4)", f, ids, flags[:, :4].contiguous())
    raises(mc, DTYPE, "prefix has dtype torch.int32", f, ids, ids)
    L = mc._lib.lib()
    call = L.mc_attention_spans
    assert call(0, 5, FAKE, None, 1, FAKE, None) == SHAPE and call(2, 0, FAKE, None, 1, FAKE, None) == SHAPE
    assert call(2, 2**31 - 4097, FAKE, None, 1, FAKE, None) == SHAPE
    assert call(4194304, 5, FAKE, None, 1, FAKE, None) == SHAPE
    assert call(2, 5, FAKE, None, 2, FAKE, None) == VALUE
    assert call(2, 5, FAKE, FAKE, 0, FAKE, None) == VALUE and "needs causal" in mc._lib.last_error()
    assert call(2, 5, FAKE, None, 1, None, None) == NULL
    assert call(2, 5, FAKE, None, 1, ctypes.c_void_p(264), None) == LAYOUT
    assert call(2, 5, ctypes.c_void_p(258), None, 1, FAKE, None) == LAYOUT


def test_attention_refusals(mc):
    q, k = torch.zeros(2, 4, 6, 64), torch.zeros(2, 2, 6, 64)
    spans, slopes = torch.zeros(2, 6, 4, dtype=torch.int32), torch.zeros(4)
    o, lse = torch.zeros(2, 6, 256), torch.zeros(2, 4, 6)

    def bwd(q, k, v, **how):
        return mc.packed_attention_backward(q, k, v, o.to(q.dtype), lse, o.to(q.dtype), **how)

    for f in (mc.packed_attention_forward, bwd):
        raises(mc, SHAPE, "q must be [batch, heads, seq, head_dim]", f, q[0], k, k)
        raises(mc, SHAPE, "v has shape (2, 2, 5, 64)", f, q, k, k[:, :, :5].contiguous())
        raises(mc, LAYOUT, "k must be contiguous", f, q, k.transpose(0, 1), k)
        raises(mc, DTYPE, "unsupported dtype torch.float16", f, q.half(), k.half(), k.half())
        raises(mc, DTYPE, "k has dtype torch.float32", f, q.bfloat16(), k, k)
        raises(mc, VALUE, "causal must be False with spans", f, q, k, k, spans=spans, causal=True)
        raises(mc, SHAPE, "spans has shape (2, 6, 2)", f, q, k, k, spans=spans[..., :2].contiguous())
        raises(mc, DTYPE, "spans has dtype torch.int64", f, q, k, k, spans=spans.long())
        raises(mc, SHAPE, "slopes has shape (2,)", f, q, k, k, slopes=slopes[:2])
        raises(mc, DTYPE, "slopes has dtype torch.bfloat16", f, q, k, k, slopes=slopes.bfloat16())
    b = mc.packed_attention_backward
    raises(mc, NULL, "o, lse and dout are required", b, q, k, k, o, None, o)
    raises(mc, SHAPE, "o has shape (2, 6, 128)", b, q, k, k, o[..., :128].contiguous(), lse, o)
    raises(mc, DTYPE, "dout has dtype torch.bfloat16", b, q, k, k, o, lse, o.bfloat16())
    raises(mc, SHAPE, "lse has shape (8, 6)", b, q, k, k, o, lse.view(8, 6), o)


def desc(mc, B=1, S=64, H=2, Hkv=1, D=64, causal=0, scale=0.125, dtype=1, cap=0.0, reserved=0):
    return mc._lib.PackedAttnDesc(mc._lib.AttnDesc(B, S, H, Hkv, D, causal, scale, dtype), cap, reserved)


def test_attention_abi(mc):
    L = mc._lib.lib()

    def fwd(d, q=FAKE, spans=None, slopes=None, o=FAKE, ws=FAKE, have=1 << 40):
        return L.mc_packed_attention_fwd(ctypes.byref(d), q, FAKE, FAKE, spans, slopes, o, None, ws, have, None)

    def bwd(d, q=FAKE, spans=None, slopes=None, o=FAKE, ws=FAKE, have=1 << 40):
        return L.mc_packed_attention_bwd(ctypes.byref(d), q, FAKE, FAKE, spans, slopes, o, FAKE, FAKE, FAKE, FAKE, FAKE,
                                         ws, have, None)

    for call in (fwd, bwd):
        for bad in ({"cap": -1.0}, {"cap": 0.009}, {"cap": 1001.0}, {"cap": math.nan}, {"cap": math.inf}, {"scale": 0.0},
                    {"scale": -0.1}, {"scale": math.nan}, {"scale": 1e31}, {"reserved": 1}, {"causal": 2}):
            assert call(desc(mc, **bad)) == VALUE, bad
        assert call(desc(mc, causal=1), spans=FAKE) == VALUE and "with spans" in mc._lib.last_error()
        for bad in ({"D": 0}, {"D": 257}, {"D": 60}, {"H": 3, "Hkv": 2}, {"S": 0}, {"B": 65536, "H": 1},
                    {"B": 60000, "H": 1, "S": 18000}, {"B": 1100, "H": 32, "S": 2000, "D": 33, "dtype": 0}):
            assert call(desc(mc, **bad)) == SHAPE, bad
        assert call(desc(mc, dtype=2)) == DTYPE
        assert call(desc(mc), q=None) == NULL and call(desc(mc), o=None) == NULL
        assert call(desc(mc), q=ctypes.c_void_p(264)) == LAYOUT
        assert call(desc(mc), spans=ctypes.c_void_p(264)) == LAYOUT
        assert call(desc(mc, S=129), ws=None) == WORKSPACE
    d = desc(mc, S=129)
    need = L.mc_packed_attention_fwd_workspace_size(ctypes.byref(d))
    assert need == 64 * 192 * 2 + 256  # V^T and a flag per 64 keys
    assert fwd(d, have=need - 1) == WORKSPACE
    assert L.mc_packed_attention_fwd_workspace_size(ctypes.byref(desc(mc, S=128))) == 0  # V is read as it is
    d = desc(mc)
    need = L.mc_packed_attention_bwd_workspace_size(ctypes.byref(d), 0)
    # lse and Delta, the flags of Q and of K, two heads' partials, dS^T in blocks of 128 x 128
    assert need == 2 * 512 + 256 + 256 + 2 * (2 * 64 * 64 * 4) + 2 * 128 * 128 * 2
    assert bwd(d, have=need - 1) == WORKSPACE
    # a head's dS^T stays below 2^31 bytes, or none is stored
    size = lambda S: L.mc_packed_attention_bwd_workspace_size(ctypes.byref(desc(mc, H=1, Hkv=1, S=S)), 0)  # noqa: E731
    assert size(32640) > 255 * 255 * 32768 and size(32641) < 2**20
    assert L.mc_packed_attention_fwd_workspace_size(ctypes.byref(desc(mc, dtype=0))) == 0
    assert L.mc_packed_attention_fwd_workspace_size(ctypes.byref(desc(mc, cap=-1.0))) == 0
    assert L.mc_packed_attention_bwd_workspace_size(ctypes.byref(desc(mc, causal=1)), 1) == 0


def test_reference_against_autograd():
    torch.manual_seed(0)
    B, H, Hkv, S, D = 1, 2, 1, 12, 4
    q, k, v, dout = torch.randn(B, H, S, D), torch.randn(B, Hkv, S, D), torch.randn(B, Hkv, S, D), torch.randn(B, S, H * D)
    ids = torch.tensor([0, 0, 0, -1, 1, 1, 1, 1, 0, 0, -2, -2])
    see = ref.visible(S, ids, torch.tensor([1, 1, 0, 0, 1, 0, 1, 0, 1, 1, 1, 1]))
    assert ref.spans_of(see).tolist() == [[0, 2, 0, 3], [0, 2, 0, 3], [0, 3, 2, 3], [0, 0, 0, 0], [4, 5, 4, 8],
                                          [4, 6, 5, 8], [4, 7, 6, 8], [4, 8, 7, 8], [8, 10, 8, 10], [8, 10, 8, 10],
                                          [0, 0, 0, 0], [0, 0, 0, 0]]
    slopes = torch.tensor([0.5, 0.1])
    want = ref.attention(q, k, v, see[None], 0.5, 2.0, slopes, dout)
    x = [t.double().requires_grad_() for t in (q, k, v)]
    i = torch.arange(S).double()
    s = 2 * torch.tanh(0.5 * x[0] @ x[1].transpose(-1, -2) / 2) - slopes.double()[:, None, None] * (i[:, None] - i).abs()
    p = torch.softmax(s.masked_fill(~see, -1e30), -1) * see
    o = (p @ x[2]).transpose(1, 2).reshape(B, S, H * D)
    assert (o - want["o"][0]).abs().max() < 1e-14
    for g, name in zip(torch.autograd.grad(o, x, dout.double()), ("dq", "dk", "dv")):
        assert (g - want[name][0]).abs().max() < 1e-14
