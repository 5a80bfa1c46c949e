"""Softmax loss with more rows than one stretch of the compaction holds: results, and a preparation that grows with the rows."""
import pytest
import torch

pytestmark = pytest.mark.gpu

IGNORE = -100


@pytest.mark.parametrize("P", [65536, 65537, 200001])
@pytest.mark.parametrize("ignored", [0.0, 0.6, "first"])
def test_rows_of_several_stretches(P, ignored):
    """Rows come from few distinct ones, so that a row's loss and gradient are those of its kind.  Tolerances: the same products and the same
    order of sums give the same kind's values but for its part of the classes (fp32 sums of 40 terms in another order, and the bf16 rounding
    of the result)."""
    from torchrec_b200.ops.transformer_ops import full_softmax_error, full_softmax_loss

    g = torch.Generator().manual_seed(P)
    V, D, kinds = 40, 16, 97
    hk, w = torch.randn(kinds, D, generator=g).bfloat16().cuda(), torch.randn(V, D, generator=g).bfloat16().cuda().requires_grad_(True)
    tk = torch.randint(0, V, (kinds,), generator=g).cuda()
    kind = torch.randint(0, kinds, (P,), generator=g).cuda()
    h, t = hk[kind].requires_grad_(True), tk[kind]
    drop = torch.zeros(P, dtype=torch.bool, device="cuda")
    if ignored == "first":
        drop[:65536 - 3] = True
    else:
        drop = torch.rand(P, generator=g).cuda() < ignored
    t = torch.where(drop, IGNORE, t)
    rows = full_softmax_loss(h, w, t, reduction="none")
    z = hk.double() @ w.detach().double().t()
    want = torch.nn.functional.cross_entropy(z, tk, reduction="none")
    limit = 16 * 2.0**-23 * float((hk.double().abs() @ w.detach().double().abs().t()).max()) * 2 + 2.0**-19 * (1 + float(z.abs().max()))
    assert float(rows[drop].detach().abs().sum()) == 0
    assert bool(((rows.detach().double() - want[kind]).abs()[~drop] <= limit).all())
    dh, dw = torch.autograd.grad(rows.sum(), (h, w))
    G = torch.softmax(z, 1)
    G[torch.arange(kinds, device="cuda"), tk] -= 1
    count = torch.bincount(kind[~drop], minlength=kinds).double()
    e, bf = torch.expm1(torch.tensor(2 * limit)).item(), 2.0**-8
    wd = w.detach().double()
    off = (dh.double() - (G @ wd)[kind]).abs() - ((bf + e) * (G.abs() @ wd.abs()) + bf * (G @ wd).abs() + 1e-30)[kind]
    assert float(dh[drop].abs().sum()) == 0 and bool((off[~drop] <= 0).all())
    GW = (G * count[:, None]).t()
    n = int(count.sum())
    assert bool(((dw.double() - GW @ hk.double()).abs() <= (bf + e + n * 2.0**-23) * (GW.abs() @ hk.double().abs()) + bf * (GW @ hk.double()).abs() + 1e-30).all())
    assert full_softmax_error(h.device) == 0


def test_targets_outside_the_classes_far_behind():
    from torchrec_b200.ops.transformer_ops import full_softmax_error, full_softmax_loss

    P = 140000
    h, w = torch.randn(P, 8, device="cuda").bfloat16(), torch.randn(30, 8, device="cuda").bfloat16()
    t = torch.randint(0, 30, (P,), device="cuda")
    t[[5, 70000, 139999]] = 30
    rows = full_softmax_loss(h, w, t, reduction="none")
    assert rows.isnan().nonzero().flatten().tolist() == [5, 70000, 139999]
    assert bool(full_softmax_loss(h, w, t).isnan()) and full_softmax_error(h.device) == 16


def test_the_preparation_grows_with_the_rows():
    """Four times the rows, all of them ignored, take about four times as long; reading all targets in front of every block took 16 times."""
    from torchrec_b200.ops.transformer_ops import full_softmax_loss

    w = torch.randn(30, 8, device="cuda").bfloat16()
    times = []
    for P in (1 << 22, 1 << 24):
        h, t = torch.zeros(1, 8, device="cuda").bfloat16().expand(P, 8), torch.full((P,), IGNORE, device="cuda")
        best = float("inf")
        for _ in range(4):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            loss = full_softmax_loss(h, w, t)
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b))
        assert float(loss) == 0
        times.append(best)
    assert times[1] < 8 * times[0], times
