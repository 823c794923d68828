"""The embedding's gradient where its tokens are sorted beside the clearing in more
steps than a wave keeps in registers: more than 4096 tokens and a table of at least
2048 times as many elements. Against 64 bits; a row's float32 sum of n terms is off by
at most (n + 1) 2^-24 of the sum of their magnitudes, its scaling included."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0**-24


@pytest.mark.parametrize("T,V,D,dtype,frequent", [
    (5000, 32000, 512, torch.bfloat16, 3), (5000, 32000, 511, torch.bfloat16, 3), (4097, 32003, 512, torch.float32, 1),
    (16384, 50257, 893, torch.float32, 5), (16384, 151936, 1536, torch.bfloat16, 4), (20001, 100003, 640, torch.bfloat16, 2),
])
def test_sorted_beside_the_clearing(mc, dev, nan_outputs, T, V, D, dtype, frequent):
    assert T > 4096 and V * D * 4 >= T * 8192
    g = torch.Generator(device=dev).manual_seed(T + D)
    ids = torch.randint(0, V, (T,), generator=g, device=dev, dtype=torch.int32)
    ids[::2] = ids[::2] % frequent  # runs of many units
    ids[5::97], ids[7::101], ids[-1] = -1, V, V - 1
    dout = torch.randn(T, D, generator=g, device=dev).to(dtype)
    for padding in (None, 1):
        keep = (ids >= 0) & (ids < V)
        if padding is not None:
            keep &= ids != padding
        rows = torch.where(keep, ids, 0).long()
        part = torch.where(keep[:, None], dout.double(), 0.0)
        want = torch.zeros(V, D, dtype=torch.float64, device=dev).index_add_(0, rows, part)
        size = torch.zeros(V, D, dtype=torch.float64, device=dev).index_add_(0, rows, part.abs())
        n = torch.bincount(rows[keep], minlength=V)[:, None]
        got = mc.embedding_backward(dout, ids, V, scale=0.5, padding_id=padding)
        assert ((got.double() - 0.5 * want).abs() <= (n + 1) * U * 0.5 * size * 1.01).all()
        before = torch.randn(V, D, generator=g, device=dev)
        into = before.clone()
        mc.embedding_backward(dout, ids, V, scale=0.5, padding_id=padding, dtable=into)
        total = before.double() + 0.5 * want
        assert ((into.double() - total).abs() <= ((n + 1) * U * 0.5 * size + (n > 0) * U * total.abs()) * 1.01).all()
        again = mc.embedding_backward(dout, ids, V, scale=0.5, padding_id=padding)
        assert torch.equal(got, again)
