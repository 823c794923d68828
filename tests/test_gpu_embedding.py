"""The scaled embedding and its gradient.

The forward is one float32 product per element, rounded to the table's type:
compared for equality. The gradient of a row is a float32 sum of n terms in some
order, off by at most (n - 1) 2^-24 of the sum of their magnitudes, and one
product (2^-24); with accumulate one sum more (2^-24 of the result).
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0**-24


def check_grad(got, ids, dout, vocab, scale, padding, before=None):
    ids, d = ids.flatten().cpu().numpy().astype(np.int64), dout.reshape(-1, dout.shape[-1]).double().cpu().numpy()
    keep = (ids >= 0) & (ids < vocab) & (ids != (-1 if padding is None else padding))
    want, size = np.zeros((vocab, d.shape[1])), np.zeros((vocab, d.shape[1]))
    np.add.at(want, ids[keep], d[keep])
    np.add.at(size, ids[keep], np.abs(d[keep]))
    n = np.bincount(ids[keep], minlength=vocab)[:, None]
    want, size = want * scale, size * abs(scale)
    bound = (n + 1) * U * size * 1.01
    if before is not None:
        b = before.double().cpu().numpy()
        want = want + b
        bound = bound + np.where(n > 0, U * 1.01 * np.abs(want), 0.0)
    got = got.double().cpu().numpy()
    assert got.shape == want.shape
    off = np.abs(got - want)
    assert (off <= bound).all(), (off - bound).max()  # 0 where no token is


CASES = [  # tokens, vocab, dim
    (1, 1, 1), (1, 7, 4), (5, 3, 7), (64, 512, 8), (65, 513, 256), (130, 511, 257), (63, 1025, 260), (1000, 100, 33),
    (777, 5000, 896), (2036, 50257, 893), (4096, 32000, 128), (300, 151936, 12),
    (40, 16, 6), (90, 17, 6), (3000, 4096, 5), (3000, 4097, 5), (5000, 8193, 3), (2500, 131073, 2),  # ids per workgroup
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,V,D", CASES)
def test_forward_and_backward(mc, dev, nan_outputs, T, V, D, dtype):
    g = torch.Generator().manual_seed(T + V + D)
    table = torch.randn(V, D, generator=g).to(dtype).to(dev)
    ids = torch.randint(0, V, (T,), generator=g, dtype=torch.int32)
    ids[T // 2:] = ids[T // 2:] % 3 % V  # a few frequent tokens
    ids, dout = ids.to(dev), torch.randn(T, D, generator=g).to(dtype).to(dev)
    scale = math.sqrt(D)
    for padding in (None, int(ids[0])):
        out = mc.embedding_forward(table, ids, scale=scale, padding_id=padding)
        want = (table[ids.long()].float() * torch.tensor(scale, dtype=torch.float32)).to(dtype)
        if padding is not None:
            want[ids == padding] = 0
        assert torch.equal(out, want)
        check_grad(mc.embedding_backward(dout, ids, V, scale=scale, padding_id=padding), ids, dout, V,
                   float(np.float32(scale)), padding)
    before = torch.randn(V, D, generator=g).to(dev)
    into = before.clone()
    assert mc.embedding_backward(dout, ids, V, dtable=into) is into
    check_grad(into, ids, dout, V, 1.0, None, before)


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 136), (torch.float32, 37), (torch.bfloat16, 5)])
@pytest.mark.parametrize("name", ["one_token", "two_runs", "unit_borders", "short_units", "long_between", "unsorted_runs", "last_id"])
def test_long_runs(mc, dev, name, dtype, D):
    """Runs past two units of 64 sorted tokens: their units' sums, at every place of a run's ends in a unit."""
    V = 700
    ids = {
        "one_token": [3] * 3001,
        "two_runs": [5] * 129 + [6] * 700,
        "unit_borders": [1] * 64 + [2] * 192 + [3] * 128 + [4] * 129 + [511] * 63 + [512] * 256,
        "short_units": [1] * 16 + [2] * 32 + [3] * 33 + [4] * 31 + [5] * 48 + [6] * 47 + [7] * 49 + [8] * 34,
        "long_between": [0] * 20 + [9] * 500 + [10, 11, 12] + [13] * 300 + [14] * 5,
        "unsorted_runs": [i % 4 * 170 for i in range(2000)],
        "last_id": [V - 1] * 1000 + [V - 2] * 10,
    }[name]
    ids = torch.tensor(ids, dtype=torch.int32)
    if name != "one_token":
        ids = ids[torch.randperm(len(ids), generator=torch.Generator().manual_seed(7))]
    ids = ids.to(dev)
    dout = torch.randn(ids.numel(), D, generator=torch.Generator().manual_seed(1)).to(dtype).to(dev)
    check_grad(mc.embedding_backward(dout, ids, V, scale=0.5), ids, dout, V, 0.5, None)


def test_units_of_many_tokens(mc, dev):
    """Past 65536 tokens the units grow."""
    T, V, D = 70001, 1000, 20
    g = torch.Generator().manual_seed(2)
    ids = torch.randint(0, V, (T,), generator=g, dtype=torch.int32)
    ids[::3] = 17
    ids, dout = ids.to(dev), torch.randn(T, D, generator=g).to(dev)
    check_grad(mc.embedding_backward(dout, ids, V), ids, dout, V, 1.0, None)


def test_ids_outside_the_table_and_padding(mc, dev):
    """Ids past either end give NaN rows and no gradient, padding zeros and none, whatever dout holds there."""
    V, D = 600, 16
    table = torch.randn(V, D, device=dev)
    ids = torch.tensor([[0, -1, 599], [600, 2**31 - 1, 5], [-(2**31), 5, 512]], dtype=torch.int32, device=dev)
    wide = ids.long()
    wide[1, 1] = 2**40 + 3  # not 3
    for i in (ids, wide):
        out = mc.embedding_forward(table, i, padding_id=5)
        real = (i >= 0) & (i < V) & (i != 5)
        assert torch.equal(out[real], table[i[real].long()])
        assert (out[i == 5] == 0).all()
        assert out[~real & (i != 5)].isnan().all()
        dout = torch.randn(3, 3, D, device=dev)
        dout[~real] = math.nan
        grad = mc.embedding_backward(dout, i, V, padding_id=5)
        want = torch.zeros(V, D, device=dev)
        want[i[real].long()] = dout[real]
        assert torch.equal(grad, want)
    # a padding id past the table is still padding
    out = mc.embedding_forward(table, ids, padding_id=600)
    assert (out[1, 0] == 0).all() and torch.equal(out[1, 2], table[5])
    # no token at all has a row
    none = torch.full((200,), -1, dtype=torch.int32, device=dev)
    assert (mc.embedding_backward(torch.full((200, D), math.nan, device=dev), none, V) == 0).all()
    same = torch.full((200,), 5, dtype=torch.int32, device=dev)
    into = torch.ones(V, D, device=dev)
    mc.embedding_backward(torch.full((200, D), math.nan, device=dev), same, V, padding_id=5, dtable=into)
    assert (into == 1).all()


def test_reproducible_on_streams_and_in_graphs(mc, dev):
    T, V, D = 3000, 2000, 96
    g = torch.Generator().manual_seed(4)
    ids = torch.randint(0, 50, (T,), generator=g, dtype=torch.int32).to(dev)
    dout = torch.randn(T, D, generator=g).bfloat16().to(dev)
    table = torch.randn(V, D, generator=g).bfloat16().to(dev)
    first, rows = mc.embedding_backward(dout, ids, V), mc.embedding_forward(table, ids, scale=3.0)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        again = mc.embedding_backward(dout, ids, V)
    side.synchronize()
    assert torch.equal(first, again)
    graph, grad = torch.cuda.CUDAGraph(), torch.zeros(V, D, device=dev)
    with torch.cuda.graph(graph):
        out = mc.embedding_forward(table, ids, scale=3.0)
        new = mc.embedding_backward(dout, ids, V)
        mc.embedding_backward(dout, ids, V, dtable=grad)
    for turn in range(3):
        grad.zero_()
        out.zero_()
        new.fill_(math.nan)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, rows) and torch.equal(new, first) and torch.equal(grad, first)
        mc.embedding_backward(dout[:9], ids[:9], V)
