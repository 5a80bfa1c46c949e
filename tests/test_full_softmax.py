"""Softmax loss over the whole catalogue on the CPU: the piecewise form against the library's cross entropy in fp64 and against
differences, and the refusals."""
import pytest
import torch

from torchrec_b200.ops import transformer_ops as tops
from torchrec_b200.ops.transformer_ops import full_softmax_loss


@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("piece", [1 << 26, 50])
def test_matches_the_library_in_fp64(reduction, bias, piece, monkeypatch):
    monkeypatch.setattr(tops._FullSoftmaxPieces, "PIECE", piece)
    g = torch.Generator().manual_seed(1)
    h, w, b = (torch.randn(*s, generator=g, dtype=torch.float64).requires_grad_(True) for s in ((9, 5), (13, 5), (13,)))
    t = torch.randint(0, 13, (9,), generator=g)
    t[4] = -100
    want = torch.nn.functional.cross_entropy(h @ w.t() + (b if bias else 0), t, reduction=reduction)
    got = full_softmax_loss(h, w, t, b if bias else None, reduction=reduction)
    torch.testing.assert_close(got, want, rtol=1e-12, atol=1e-12)
    up = torch.rand(want.shape, generator=g, dtype=torch.float64)
    leaves = [h, w] + ([b] if bias else [])
    for x, y in zip(torch.autograd.grad(got, leaves, up), torch.autograd.grad(want, leaves, up)):
        torch.testing.assert_close(x, y, rtol=1e-11, atol=1e-12)
    assert torch.autograd.gradcheck(lambda a, c, d: full_softmax_loss(a, c, t, d, reduction=reduction), (h, w, b))


def test_rows_that_count_nowhere():
    h = torch.randn(4, 3)
    h[1] = float("nan")
    w = torch.randn(6, 3, requires_grad=True)
    t = torch.tensor([0, 7, 5, 7])
    h.requires_grad_(True)
    loss = full_softmax_loss(h, w, t, ignore_index=7)
    loss.backward()
    assert bool(torch.isfinite(loss)) and bool(torch.isfinite(w.grad).all()) and float(h.grad[[1, 3]].abs().max()) == 0
    none = full_softmax_loss(h, w, torch.full((4,), 7), ignore_index=7)
    assert float(none.detach()) == 0
    empty = full_softmax_loss(torch.zeros(0, 3, requires_grad=True), w, torch.zeros(0, dtype=torch.int64))
    empty.backward()
    assert float(empty.detach()) == 0


def test_sixteen_bit_types_on_the_cpu():
    g = torch.Generator().manual_seed(2)
    for dtype in (torch.bfloat16, torch.float16):
        h, w = (torch.randn(*s, generator=g).to(dtype).requires_grad_(True) for s in ((20, 8), (30, 8)))
        t = torch.randint(0, 30, (20,), generator=g)
        loss = full_softmax_loss(h, w, t.int())
        assert loss.dtype == torch.float32
        want = torch.nn.functional.cross_entropy(h.double() @ w.double().t(), t)
        torch.testing.assert_close(loss.double(), want, rtol=1e-5, atol=0)
        got = torch.autograd.grad(loss, (h, w))
        for x, y in zip(got, torch.autograd.grad(want, (h, w))):
            assert x.dtype == dtype
            # one rounding on either side of the comparison
            torch.testing.assert_close(x.double(), y.double(), rtol=torch.finfo(dtype).eps * 1.01, atol=1e-6)


def test_refusals():
    h, w, t = torch.randn(4, 3), torch.randn(6, 3), torch.zeros(4, dtype=torch.int64)
    with pytest.raises(ValueError, match="reduction"):
        full_softmax_loss(h, w, t, reduction="max")
    with pytest.raises(ValueError, match="h \\[P, D\\]"):
        full_softmax_loss(h, w[:, :2], t)
    with pytest.raises(ValueError, match="h \\[P, D\\]"):
        full_softmax_loss(h[0], w, t)
    with pytest.raises(ValueError, match="h \\[P, D\\]"):
        full_softmax_loss(h, w[:0], t)
    with pytest.raises(ValueError, match="targets"):
        full_softmax_loss(h, w, t[:3])
    with pytest.raises(ValueError, match="targets"):
        full_softmax_loss(h, w, t.float())
    with pytest.raises(ValueError, match="bias"):
        full_softmax_loss(h, w, t, torch.zeros(5))
    with pytest.raises(ValueError, match="floating"):
        full_softmax_loss(h, w.int(), t)
    with pytest.raises(IndexError, match="out of bounds"):
        full_softmax_loss(h, w, torch.tensor([0, 6, 0, 0]))
