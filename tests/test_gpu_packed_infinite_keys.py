"""An infinite key that a query sees. Its score is an infinity or, under a cap, plus or
minus the cap; P or the cap's slope may then be 0, and dq = scale sum_j dS_ij k_j holds 0
times an infinity, which is NaN, and no finite value, in the infinite column."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cap", [None, 20.0])
@pytest.mark.parametrize("value", [math.inf, -math.inf])
@pytest.mark.parametrize("dt,D,S", [(torch.bfloat16, 64, 140), (torch.bfloat16, 128, 300), (torch.float32, 64, 130),
                                    (torch.bfloat16, 40, 50), (torch.bfloat16, 64, 32800)])
def test_reaches_the_queries_that_see_it(mc, dev, dt, D, S, value, cap):
    g = torch.Generator().manual_seed(S + D)
    q, k, v = (torch.randn(1, n, S, D, generator=g).to(dt).to(dev) for n in (2, 1, 1))
    dout = torch.randn(1, S, 2 * D, generator=g).to(dt).to(dev)
    cuts = [0, 20, 45, S] if S < 1000 else [0, S - 500, S - 300, S]
    ids = torch.zeros(1, S, dtype=torch.int32)
    for n in range(3):
        ids[0, cuts[n]:cuts[n + 1]] = n if n != 0 or S < 1000 else -1
    spans = mc.attention_spans(ids.to(dev))
    t = cuts[1] + 7
    bad = k.clone()
    bad[0, 0, t, 3] = value

    def gradients(k):
        o, lse = mc.packed_attention_forward(q, k, v, spans=spans, cap=cap)
        return mc.packed_attention_backward(q, k, v, o, lse, dout, spans=spans, cap=cap)

    clean, got = gradients(k), gradients(bad)
    assert got[0][0, :, t:cuts[2], 3].isnan().all()
    for a, b in ((cuts[0], t), (cuts[2], S)):  # queries that do not see it
        assert torch.equal(got[0][:, :, a:b], clean[0][:, :, a:b])
