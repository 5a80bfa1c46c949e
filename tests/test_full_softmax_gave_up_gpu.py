"""A call in which a block of the softmax-loss kernel gave up a wait: the loss and every gradient are NaN.  No wait runs out here: the word that
such a block leaves in the call's state is set from the host."""
import pytest
import torch

from torchrec_b200.ops import _ext

pytestmark = pytest.mark.gpu

IGNORE, GAVE_UP = -100, 4  # the word's place among the state's counters


def _inputs(P, V, D):
    g = torch.Generator().manual_seed(P)
    h, w, b = torch.randn(P, D, generator=g).bfloat16(), torch.randn(V, D, generator=g).bfloat16(), torch.randn(V, generator=g)
    t = torch.randint(0, V, (P,), generator=g)
    t[::5] = IGNORE
    return h.cuda(), w.cuda(), t.cuda(), b.cuda()


@pytest.mark.parametrize("reduction", [0, 1, 2])
@pytest.mark.parametrize("grad", [0, 2])
@pytest.mark.parametrize("P", [3, 300])
def test_forward(P, grad, reduction):
    h, w, t, b = _inputs(P, 500, 64)
    good, _ = _ext.cuda_ops().full_softmax_fwd(h, w, t, b, IGNORE, reduction, grad)
    bad, _ = _ext.cuda_ops().full_softmax_fwd(h, w, t, b, IGNORE, reduction, grad, 1)
    again, _ = _ext.cuda_ops().full_softmax_fwd(h, w, t, b, IGNORE, reduction, grad)
    assert bool(torch.isfinite(good).all()) and torch.equal(good, again)
    if reduction == 0:
        assert torch.equal(bad.isnan(), t != IGNORE) and float(bad[t == IGNORE].abs().max()) == 0
    else:
        assert bool(bad.isnan())


@pytest.mark.parametrize("reduction", [0, 1])
@pytest.mark.parametrize("fp32", [False, True])
@pytest.mark.parametrize("P,V,D", [(3, 500, 64), (300, 500, 64), (300, 20001, 64), (260, 700, 320)])
def test_backward(P, V, D, fp32, reduction):
    h, w, t, b = _inputs(P, V, D)
    _, state = _ext.cuda_ops().full_softmax_fwd(h, w, t, b, IGNORE, reduction, 2)
    up = torch.ones(P, device="cuda") if reduction == 0 else torch.ones((), device="cuda")

    def grads(want_h, want_w, want_b):
        return _ext.cuda_ops().full_softmax_bwd(up, w, state, P, D, True, reduction, True, want_h, want_w, want_b, fp32, fp32, fp32)

    for g in grads(True, True, True):
        assert bool(torch.isfinite(g).all())
    state[:32].view(torch.int32)[GAVE_UP] = 1
    dh, dw, db = grads(True, True, True)
    assert torch.equal(dh.isnan().all(1), t != IGNORE) and float(dh[t == IGNORE].abs().max()) == 0
    assert bool(dw.isnan().all()) and bool(db.isnan().all())
    assert bool(grads(False, True, False)[1].isnan().all())
    assert bool(grads(True, False, False)[0][t != IGNORE].isnan().all())
    assert bool(grads(False, False, True)[2].isnan().all())
