"""The gradients' norm and clipping where chunks of the norm are longer than the least
(past 4096 * 8192 elements) and where outputs are past the size whose stores go around
the caches (256 MB), and what the host refuses.

The kernels sum squares in 64 bits: the norm is off by its rounding to float32, 2^-24,
and by the sums' 2^-53 for each of at most 1.4e8 terms added in a row, 2^-26. The
reference is a sum in 64 bits, by blocks. A scaled gradient is one float32 product,
rounded to the output's type: compared for equality."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
OFF = 2.0**-24 + 2.0**-26


def norm64(grads):
    return math.sqrt(math.fsum(float(part.double().square().sum()) for g in grads for part in g.split(1 << 22)))


@pytest.mark.parametrize("start", [0, 1, 3])
@pytest.mark.parametrize("td,od", [(torch.bfloat16, torch.float32), (torch.float32, torch.float32),
                                   (torch.float32, torch.bfloat16), (torch.bfloat16, torch.bfloat16)])
def test_long_chunks_and_streamed_stores(mc, dev, td, od, start):
    sizes = [70_000_001, 5, 33, 1_000_003] + ([69_999_990] if od == torch.bfloat16 else [])  # over 256 MB of outputs
    assert sum(sizes) * (4 if od == torch.float32 else 2) > 256 << 20
    g = torch.Generator(device=dev).manual_seed(start)
    grads = [torch.randn(n + start, generator=g, device=dev).to(td)[start:] for n in sizes]
    backs = [torch.full((n + start + 4,), 7.0, dtype=od, device=dev) for n in sizes]
    outs = [b[start:start + n] for b, n in zip(backs, sizes)]
    need = mc._lib.lib().mc_gradient_norm_workspace_size(
        (mc._lib.GradTensor * 1)(mc._lib.GradTensor(grads[0].data_ptr(), None, sizes[0], 0, 0)), 1)
    assert need < 8 * sizes[0] / 8192  # fewer partials than least chunks
    want = norm64(grads)
    norm, scale = mc.clip_gradients(grads, 1.0, outs=outs)
    assert abs(norm.item() - want) <= OFF * want and abs(scale.item() * want - 1.0) <= 2 * OFF
    alone, same = mc.gradient_norm(grads, 1.0)
    assert alone.item() == norm.item() and same.item() == scale.item()
    for x, o, b in zip(grads, outs, backs):
        for xs, os in zip(x.split(1 << 24), o.split(1 << 24)):
            assert torch.equal(os, (xs.float() * scale).to(od))
        assert (b[:start] == 7.0).all() and (b[start + x.numel():] == 7.0).all()


def test_overlapping_tensors(mc, dev):
    """Refused before anything is launched: the gradients stay as they are."""
    a, b = torch.ones(300, device=dev), torch.full((300,), 2.0, device=dev)
    flat = torch.ones(1000, device=dev)
    one = torch.full((1,), 0.5, device=dev)
    for grads, outs in (([a, b], [b, a]), ([flat[:600], flat[400:]], None), ([a, flat[:10]], [flat[5:305], b[:10]])):
        for call in (lambda: mc.clip_gradients(grads, 1.0, outs=outs), lambda: mc.scale_gradients(grads, one, outs=outs)):
            with pytest.raises(mc.McError) as e:
                call()
            assert e.value.code == 4 and "overlap" in str(e.value)
    assert (a == 1).all() and (b == 2).all() and (flat == 1).all()
    mc.scale_gradients([flat[:500], flat[500:]], one)  # one behind the other
    assert (flat == 0.5).all()
