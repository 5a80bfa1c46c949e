"""Softmax loss over the whole catalogue where no kernel takes it (the CPU here; types, widths and compute types that the kernel does not take
on CUDA): inside an autocast region."""
import pytest
import torch

from torchrec_b200.ops.transformer_ops import full_softmax_loss

devices = pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])


def _inputs(P, V, D, device, scale=1.0, seed=1):
    g = torch.Generator().manual_seed(seed)
    h, w, b = torch.randn(P, D, generator=g), torch.randn(V, D, generator=g) * scale, torch.randn(V, generator=g)
    return [x.to(device).requires_grad_(True) for x in (h, w, b)] + [torch.randint(0, V, (P,), generator=g).to(device)]


@devices
@pytest.mark.parametrize("where", ["forward", "both"])
def test_autocast_changes_nothing(device, where):
    """32 bits inside an autocast region too, in both directions."""
    h, w, b, t = _inputs(64, 500, 64, device)
    want = full_softmax_loss(h, w, t, b, reduction="none")
    want_g = torch.autograd.grad(want.sum(), (h, w, b))
    with torch.autocast(device, dtype=torch.bfloat16):
        got = full_softmax_loss(h, w, t, b, reduction="none")
        if where == "both":
            got_g = torch.autograd.grad(got.sum(), (h, w, b))
    if where == "forward":
        got_g = torch.autograd.grad(got.sum(), (h, w, b))
    assert got.dtype == torch.float32 and torch.equal(got, want)
    for x, y in zip(got_g, want_g):
        assert x.dtype == y.dtype and torch.equal(x, y)
    # a row's gradients of the scores add up to zero: 500 terms of at most 1 in fp32, 64 rows
    assert abs(float(got_g[2].sum())) <= 64 * 500 * 2.0**-24
