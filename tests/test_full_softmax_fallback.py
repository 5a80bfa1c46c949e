"""Softmax loss over the whole catalogue where no kernel takes it (the CPU here; types, widths and compute types that the kernel does not take
on CUDA): inside an autocast region, with masks, with confident rows, with targets outside the classes."""
import math

import pytest
import torch

from torchrec_b200.ops import dense_ops
from torchrec_b200.ops.transformer_ops import full_softmax_loss


@pytest.fixture(autouse=True)
def fp32_compute_type():
    """Another test of the process may have left bf16, with which fp32 tensors go to the tensor-core kernels."""
    prev = dense_ops.get_dense_compute_dtype()
    dense_ops.set_dense_compute_dtype(torch.float32)
    yield
    dense_ops.set_dense_compute_dtype(prev)


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


@devices
@pytest.mark.parametrize("mask", [-1e9, -1e20, torch.finfo(torch.float32).min])
def test_rows_whose_mask_leaves_nothing(device, mask):
    """Every class behind the same finite mask, which swallows the products: a uniform softmax, as cross_entropy of these scores."""
    h, w, b, t = _inputs(20, 70, 8, device)
    with torch.no_grad():
        b.fill_(mask)
    loss = full_softmax_loss(h, w, t, b, reduction="none")
    grads = torch.autograd.grad(loss.sum(), (h, w, b))
    want = torch.nn.functional.cross_entropy(h @ w.t() + b, t, reduction="none")
    want_g = torch.autograd.grad(want.sum(), (h, w, b))
    torch.testing.assert_close(loss, want, rtol=1e-6, atol=1e-6)
    assert abs(float(loss[0].detach()) - math.log(70)) < 1e-5
    for x, y in zip(grads, want_g):
        torch.testing.assert_close(x, y, rtol=1e-5, atol=1e-5)


def test_infinite_masks():
    h, w, b, t = _inputs(6, 9, 4, "cpu")
    with torch.no_grad():
        b[:4] = float("-inf")
    t = torch.tensor([4, 5, 6, 7, 8, 0])  # the last target cannot be reached
    rows = full_softmax_loss(h, w, t, b, reduction="none")
    want = torch.nn.functional.cross_entropy(h @ w.t() + b, t, reduction="none")
    torch.testing.assert_close(rows, want)
    assert float(rows[5].detach()) == float("inf")
    one = torch.full((9,), float("-inf"))
    one[5] = 0.5
    loss = full_softmax_loss(h, w, torch.full((6,), 5), one, reduction="sum")
    (dh,) = torch.autograd.grad(loss, h)
    assert float(loss.detach()) == 0 and float(dh.abs().max()) == 0


@devices
def test_confident_rows_keep_their_accuracy(device):
    """1 - p of a target that has almost everything: relative to itself, not to 1.  Scores are off by at most d = D 2^-23 sum |h w|, the rest
    by a dozen roundings, which is the relative error of a loss that small and of its gradient."""
    h, w, b, t = _inputs(60, 200, 32, device)
    with torch.no_grad():
        h.copy_(w[t] * torch.linspace(0.5, 1.5, 60, device=device)[:, None])
    b = None
    loss = full_softmax_loss(h, w, t, b, reduction="none")
    (dh,) = torch.autograd.grad(loss.sum(), h)
    z = h.detach().double() @ w.detach().double().t()
    zt = z.gather(1, t[:, None])[:, 0]
    others = torch.logsumexp(z.scatter(1, t[:, None], float("-inf")), 1) - zt
    want = torch.nn.functional.softplus(others, threshold=1e9)
    want = torch.where(others < -30, torch.exp(others), want)
    d = 32 * 2.0**-23 * float((h.detach().double().abs() @ w.detach().double().abs().t()).max()) + 2.0**-20
    rel = torch.expm1(torch.tensor(2 * d)).item() + 2.0**-20
    assert float(want.min()) < 1e-9  # there are such rows
    assert bool(((loss.detach().double() - want).abs() <= rel * want + 1e-37).all())
    G = torch.exp(z - zt[:, None] - want[:, None])
    G[torch.arange(60, device=device), t] = -torch.sigmoid(others)
    wd = w.detach().double()
    limit = (rel + 200 * 2.0**-23) * (G.abs() @ wd.abs()) + 1e-37
    assert bool(((dh.double() - G @ wd).abs() <= limit).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.float64])
def test_targets_outside_the_classes_are_reported_on_cuda(dtype):
    from torchrec_b200.ops.transformer_ops import full_softmax_error

    h, w, b, t = _inputs(20, 30, 8, "cuda")
    h = h.detach().to(dtype).requires_grad_(True)
    assert full_softmax_error(h.device) == 0
    full_softmax_loss(h, w, t, b, reduction="none")
    assert full_softmax_error(h.device) == 0
    t[3], t[11], t[12] = 30, -1, -100
    rows = full_softmax_loss(h, w, t, b, reduction="none")
    rows.sum().backward()
    assert rows.isnan().nonzero().flatten().tolist() == [3, 11]
    assert float(h.grad[[3, 11, 12]].abs().max()) == 0 and bool(torch.isfinite(h.grad).all())
    assert full_softmax_error(h.device) == 16 and full_softmax_error(h.device) == 0
