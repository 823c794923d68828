"""Refusals of the gradients' norm and clipping and of the embedding: the torch
front end and the C ABI check arguments on the host, before anything is enqueued."""
import ctypes

import pytest
import torch

NULL, SHAPE, DTYPE, LAYOUT, VALUE, WORKSPACE = 1, 2, 3, 4, 5, 6
FAKE = ctypes.c_void_p(256)


def raises(mc, code, text, fn, *a, **k):
    with pytest.raises(mc.McError) as e:
        fn(*a, **k)
    assert e.value.code == code, e.value
    assert text in str(e.value), e.value


def test_gradient_lists(mc):
    g = [torch.zeros(4, 3), torch.zeros(7)]
    for f in (lambda x, **k: mc.gradient_norm(x, 1.0, **k), lambda x, **k: mc.clip_gradients(x, 1.0, **k)):
        raises(mc, SHAPE, "at least one tensor", f, [])
        raises(mc, SHAPE, "must be a list", f, torch.zeros(3))
        raises(mc, NULL, "must hold tensors only", f, [g[0], None])
        raises(mc, NULL, "must hold tensors only", f, [g[0], 1.0])
        raises(mc, LAYOUT, "must be contiguous", f, [g[0].t(), g[1]])
        raises(mc, DTYPE, "unsupported dtype torch.float16", f, [g[0], g[1].half()])
        raises(mc, LAYOUT, "2 devices", f, [g[0], torch.zeros(3, device="meta")])
    c = mc.clip_gradients
    raises(mc, SHAPE, "outs list has 1 entries, expected 2", c, g, 1.0, outs=[g[0]])
    raises(mc, SHAPE, "outs[1] has 6 elements, expected 7", c, g, 1.0, outs=[g[0].clone(), torch.zeros(6)])
    raises(mc, DTYPE, "unsupported dtype torch.float64", c, g, 1.0, outs=[g[0].double(), g[1].clone()])
    raises(mc, LAYOUT, "expected cpu", c, g, 1.0, outs=[torch.zeros(12, device="meta"), torch.zeros(7, device="meta")])
    s = mc.scale_gradients
    raises(mc, NULL, "scale must be a tensor", s, g, None)
    raises(mc, NULL, "scale must be a tensor", s, g, 0.5)
    raises(mc, SHAPE, "scale has shape ()", s, g, torch.zeros(()))
    raises(mc, DTYPE, "scale has dtype torch.float64", s, g, torch.zeros(1, dtype=torch.float64))
    p = [torch.zeros(4)]
    raises(mc, SHAPE, "grad_scale has shape (2,)", mc.adamw_step, p, p, p, p, 1, grad_scale=torch.zeros(2))
    assert mc.adamw_step([], [], [], [], 1, grad_scale=torch.zeros(1)) == []


def table(mc, *rows):
    return (mc._lib.GradTensor * len(rows))(*[mc._lib.GradTensor(*r) for r in rows])


def test_gradient_table_abi(mc):
    L = mc._lib.lib()
    t = table(mc, (256, 256, 10, 0, 0), (4096, 8192, 9, 1, 0))
    need = L.mc_gradient_norm_workspace_size(t, 2)
    assert need == 2 * 8  # a partial sum per tensor of a chunk or less

    def clip(t, n, max_norm=1.0, norm=FAKE, scale=FAKE, ws=FAKE, have=need):
        return L.mc_clip_gradients(t, n, max_norm, norm, scale, ws, have, None)

    assert clip(t, -1) == SHAPE
    assert clip(None, 1) == NULL
    assert clip(t, 2, norm=None) == NULL and clip(t, 2, scale=None) == NULL
    for bad in (0.0, -1.0, float("nan")):
        assert clip(t, 2, max_norm=bad) == VALUE and "max_norm must be positive" in mc._lib.last_error()
    assert clip(t, 2, have=need - 1) == WORKSPACE and clip(t, 2, ws=None) == WORKSPACE
    assert clip(table(mc, (256, 256, -1, 0, 0)), 1) == SHAPE
    assert clip(table(mc, (256, 256, 1 << 40, 0, 0)), 1) == SHAPE
    assert clip(table(mc, (256, 256, 4, 2, 0)), 1) == DTYPE and clip(table(mc, (256, 512, 4, 0, 7)), 1) == DTYPE
    assert clip(table(mc, (None, 256, 4, 0, 0)), 1) == NULL and clip(table(mc, (256, None, 4, 0, 0)), 1) == NULL
    assert clip(table(mc, (257, 512, 4, 1, 1)), 1) == LAYOUT and clip(table(mc, (258, 512, 4, 0, 0)), 1) == LAYOUT
    assert clip(table(mc, (256, 514, 4, 0, 0)), 1) == LAYOUT
    # an output inside its gradient, or of another dtype in its place
    assert clip(table(mc, (256, 264, 4, 0, 0)), 1) == LAYOUT and "must not overlap" in mc._lib.last_error()
    assert clip(table(mc, (256, 256, 4, 1, 0)), 1) == LAYOUT
    # the norm alone reads no outputs and, without a scale, no max_norm
    assert L.mc_gradient_norm(table(mc, (256, None, 4, 0, 9)), 1, 0.0, None, None, FAKE, 8, None) == NULL
    assert L.mc_gradient_norm(t, 2, 0.0, FAKE, FAKE, FAKE, need, None) == VALUE
    assert L.mc_gradient_norm(t, 2, 0.0, FAKE, None, FAKE, need - 1, None) == WORKSPACE
    assert L.mc_scale_gradients(t, 2, None, None) == NULL
    # nothing to scale, nothing launched
    assert L.mc_scale_gradients(table(mc, (None, None, 0, 0, 0)), 1, FAKE, None) == 0
    assert L.mc_scale_gradients(None, 0, FAKE, None) == 0


def test_same_tensor_twice(mc):
    """It would be scaled twice or once, as the workgroups come; the norm may count it twice."""
    a, b, empty = torch.ones(64), torch.ones(64), torch.ones(0)
    scale = torch.ones(1)
    raises(mc, LAYOUT, "listed twice", mc.clip_gradients, [a, b, a], 1.0)
    raises(mc, LAYOUT, "listed twice", mc.scale_gradients, [a, b, a], scale)
    raises(mc, LAYOUT, "listed twice", mc.clip_gradients, [b, b.clone(), b.clone()], 1.0, outs=[a, torch.ones(64), a])
    # several empty tensors share the address 0: the call goes on to what refuses the CPU
    with pytest.raises(Exception) as e:
        mc.scale_gradients([a, empty, empty], scale)
    assert "twice" not in str(e.value)
    with pytest.raises(Exception) as e:
        mc.gradient_norm([a, a])
    assert "twice" not in str(e.value)


def test_gradient_partials(mc):
    """Chunks of 8192 elements, longer ones where there would be more than about 4096 of them."""
    L = mc._lib.lib()
    size = L.mc_gradient_norm_workspace_size
    assert size(table(mc, (256, 0, 8192, 0, 0)), 1) == 8
    assert size(table(mc, (256, 0, 8193, 1, 0)), 1) == 16
    assert size(table(mc, (256, 0, 4096 * 8192, 0, 0)), 1) == 4096 * 8
    assert size(table(mc, (256, 0, 4096 * 8192 + 1, 0, 0)), 1) == 2049 * 8
    assert size(table(mc, (256, 0, 2**34, 1, 0)), 1) == 4096 * 8
    assert size(table(mc, (None, 0, 0, 0, 0)), 1) == 0


def test_embedding_refusals(mc):
    w, ids = torch.zeros(10, 8), torch.zeros(2, 3, dtype=torch.int32)
    f, b = mc.embedding_forward, mc.embedding_backward
    raises(mc, SHAPE, "table must be [vocab, dim]", f, w[0], ids)
    raises(mc, SHAPE, "table must be [vocab, dim]", f, torch.zeros(0, 8), ids)
    raises(mc, LAYOUT, "table must be contiguous", f, w.t(), ids)
    raises(mc, DTYPE, "unsupported dtype torch.float16", f, w.half(), ids)
    raises(mc, NULL, "ids must be a tensor", f, w, [1, 2])
    raises(mc, DTYPE, "ids has dtype torch.int16", f, w, ids.short())
    raises(mc, LAYOUT, "ids must be contiguous", f, w, ids.t())
    raises(mc, SHAPE, "ids are empty", f, w, ids[:0])
    raises(mc, LAYOUT, "ids is on meta", f, w, ids.to("meta"))
    d = torch.zeros(2, 3, 8)
    raises(mc, SHAPE, "dout must be", b, d[..., :0].contiguous(), ids, 10)
    raises(mc, SHAPE, "ids has shape (6,), expected (2, 3)", b, d, ids.view(-1), 10)
    raises(mc, DTYPE, "unsupported dtype torch.float64", b, d.double(), ids, 10)
    raises(mc, SHAPE, "dtable has shape (10, 8), expected (11, 8)", b, d, ids, 11, dtable=w)
    raises(mc, DTYPE, "dtable has dtype torch.bfloat16", b, d, ids, 10, dtable=w.bfloat16())


def test_embedding_abi(mc):
    L = mc._lib.lib()

    def desc(tokens=8, vocab=100, dim=16, padding=-1, scale=1.0, dtype=0):
        return ctypes.byref(mc._lib.EmbeddingDesc(tokens, vocab, dim, padding, scale, dtype))

    def fwd(d, table=FAKE, ids=FAKE, out=FAKE):
        return L.mc_embedding_fwd(d, table, ids, out, None)

    def bwd(d, ids=FAKE, dout=FAKE, dtable=FAKE, add=0, ws=FAKE, have=1 << 40):
        return L.mc_embedding_bwd(d, ids, dout, dtable, add, ws, have, None)

    for call in (fwd, bwd):
        assert call(None) == NULL
        assert call(desc(dtype=2)) == DTYPE
        for bad in ({"tokens": 0}, {"vocab": 0}, {"dim": 0}, {"tokens": 2**28}, {"vocab": 2**31},
                    {"vocab": 2**30, "dim": 1024}, {"tokens": 2**27, "dim": 8192}):
            assert call(desc(**bad)) == SHAPE, bad
        assert call(desc(scale=float("inf"))) == VALUE
        assert call(desc(), ids=None) == NULL
        assert call(desc(), ids=ctypes.c_void_p(258)) == LAYOUT
    assert fwd(desc(), table=None) == NULL and fwd(desc(), out=None) == NULL
    assert fwd(desc(), table=ctypes.c_void_p(264)) == LAYOUT and fwd(desc(), out=ctypes.c_void_p(264)) == LAYOUT
    assert fwd(desc(tokens=67108861)) == SHAPE
    assert bwd(desc(), dout=None) == NULL and bwd(desc(), dtable=None) == NULL
    assert bwd(desc(), dout=ctypes.c_void_p(264)) == LAYOUT and bwd(desc(), dtable=ctypes.c_void_p(264)) == LAYOUT
    assert bwd(desc(), add=2) == VALUE
    assert bwd(desc(vocab=2**24, dim=1024)) == SHAPE
    assert bwd(desc(vocab=2**31 - 1, dim=1)) == SHAPE
    assert bwd(desc(tokens=2**26, dim=512)) == SHAPE and "too large for a launch" in mc._lib.last_error()
    need = L.mc_embedding_bwd_workspace_size(desc())
    assert need == 256 + 256 + 512  # order, ids and start; no run of 8 tokens is long
    assert L.mc_embedding_bwd_workspace_size(desc(tokens=128)) == 512 + 512 + 512
    # 129 tokens are three units of 64, with two sums of 16 columns each
    assert L.mc_embedding_bwd_workspace_size(desc(tokens=129)) == 768 + 768 + 512 + 512
    assert bwd(desc(), have=need - 1) == WORKSPACE and bwd(desc(), ws=None) == WORKSPACE
    assert L.mc_embedding_bwd_workspace_size(desc(tokens=0)) == 0
