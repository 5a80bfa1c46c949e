"""Softmax loss over the whole catalogue with scores far from zero: classes masked by a large finite bias, rows whose mask leaves nothing,
and products that are large by themselves; against the definition in fp64 on the scores rounded to fp32.

The scores are ``fp32(h W^T) + bias`` in fp32: a bias of -1e9 swallows the product, and a row in which every class carries it is a uniform
softmax (loss ``log V``).  Tolerances as in the tests beside this one: a score near zero is off by at most ``d = D 2^-23 sum |h w| + 2^-20
(1 + |z|)`` over the scores that no mask swallows; far scores are exact here (the inputs are made so), differ by nothing or by more than an
exponential can hold, and add no error.  A loss is also rounded to fp32, after a few operations on values of its size: ``2^-21 |loss|``."""
import pytest
import torch

pytestmark = pytest.mark.gpu

IGNORE = -100
LOWEST = torch.finfo(torch.float32).min
MASKS = [-1e9, -6.55e9, -1e10, -1e12, -1e18, -1e20, -1e30, LOWEST]


def _inputs(P, V, D, seed=0):
    g = torch.Generator().manual_seed(seed)
    h = torch.randn(P, D, generator=g).bfloat16()
    w = (torch.randn(V, D, generator=g) / D**0.5).bfloat16()
    return h.cuda(), w.cuda(), torch.randint(0, V, (P,), generator=g).cuda(), torch.randn(V, generator=g).cuda()


def _check(h, w, t, b, reduction="none", ignore=IGNORE):
    from torchrec_b200.ops.transformer_ops import full_softmax_error, full_softmax_loss

    P, D = h.shape
    g = torch.Generator().manual_seed(3)
    up = ((torch.rand(P, generator=g) + 0.5) if reduction == "none" else torch.rand((), generator=g) + 0.5).cuda()
    leaves = [x.detach().clone().requires_grad_(True) for x in (h, w, b) if x is not None]
    loss = full_softmax_loss(leaves[0], leaves[1], t, leaves[2] if b is not None else None, ignore, reduction)
    grads = torch.autograd.grad(loss, leaves, up)
    with torch.no_grad():
        again = full_softmax_loss(h, w, t, b, ignore, reduction)
    torch.cuda.synchronize()
    assert full_softmax_error(h.device) == 0

    hd, wd = h.double(), w.double()
    z = (hd @ wd.t()).float()
    z = (z if b is None else z + b.float()).double()
    tt = t[:, None]
    zt = z.gather(1, tt)[:, 0]
    top = z.amax(1)
    rel = z - top[:, None]  # exact: fp32 values in fp64
    others = torch.logsumexp(rel.scatter(1, tt, float("-inf")), 1) - (zt - top)
    rows = torch.logaddexp(others, torch.zeros_like(others))
    n = P
    G = torch.softmax(rel, 1)
    G[torch.arange(P, device=h.device), t] = -torch.sigmoid(others)
    G = G * (up.double() / (n if reduction == "mean" else 1)).reshape(-1, 1)
    want_loss = {"none": rows, "mean": rows.sum() / n, "sum": rows.sum()}[reduction]
    near = z.abs() < 2**20
    mag = torch.where(near, hd.abs() @ wd.abs().t(), 0)
    d = D * 2.0**-23 * float(mag.max()) + 2.0**-20 * (1 + float(torch.where(near, z.abs(), 0).max()))
    e = torch.expm1(torch.tensor(2 * d)).item()
    bf = 2.0**-8
    tol_loss = 2 * d * (P if reduction == "sum" else 1) + 2.0**-21 * want_loss.abs() + (0 if reduction == "none" else P * 2.0**-23 * rows.abs().max())
    for got in (loss.detach(), again):
        off = (got.double() - want_loss).abs() - tol_loss
        assert bool((off <= 0).all()), f"loss: over its tolerance by {float(off.max())}; nan {int(got.isnan().sum())}"
    dh, dw, db = G @ wd, G.t() @ hd, G.sum(0)
    limits = ((bf + e + w.shape[0] * 2.0**-23) * (G.abs() @ wd.abs()) + bf * dh.abs() + 1e-30,
              (bf + e + P * 2.0**-23) * (G.abs().t() @ hd.abs()) + bf * dw.abs() + 1e-30,
              (e + (P + 8) * 2.0**-23) * G.abs().sum(0) + 1e-30)
    for name, got, x, lim in zip(("dh", "dw", "db"), grads, (dh, dw, db), limits):
        off = (got.double() - x).abs() - lim
        assert bool((off <= 0).all()), f"{name}: over its tolerance by {float(off.max())}; nan {int(got.isnan().sum())}"


@pytest.mark.parametrize("mask", MASKS)
def test_finite_masks_over_a_stretch_of_classes(mask):
    """The first columns of the first tile, whole tiles, single classes, all but a few: targets among the classes that are left."""
    for where in (slice(0, 32), slice(0, 300), slice(100, 500), slice(640, 700), slice(1, 699)):
        h, w, t, b = _inputs(150, 700, 64, seed=1)
        masked = torch.zeros(700, dtype=torch.bool, device="cuda")
        masked[where] = True
        masked[7::50] = True
        b[masked] = mask
        left = (~masked).nonzero().flatten()
        _check(h, w, left[t % left.numel()], b)


@pytest.mark.parametrize("mask", MASKS)
def test_rows_whose_mask_leaves_nothing(mask):
    for D in (64, 256):
        h, w, t, b = _inputs(150, 700, D, seed=2)
        b[:] = mask
        _check(h, w, t, b)
        _check(h, w, t, b, "mean")
        b[300] = 2 * mask if mask > -1e37 else float("-inf")  # still further away
        t[t == 300] = 0
        _check(h, w, t, b)


@pytest.mark.parametrize("mask", [-1e9, -1e10, -1e30, LOWEST])
def test_targets_behind_the_mask(mask):
    """The loss is the distance of the target's score, which may be the largest number there is."""
    h, w, t, b = _inputs(90, 700, 64, seed=3)
    b[:200] = mask
    t = t % 200
    _check(h, w, t, b)


@pytest.mark.parametrize("mask", [-1e9, -1e10, -1e20, LOWEST])
def test_whole_parts_behind_the_mask(mask):
    """Few rows against many classes: some blocks see masked classes only, others meet the mask first and a score near zero later."""
    h, w, t, b = _inputs(3, 40001, 64, seed=4)
    b[:20000] = mask
    b[20001:40001:2] = mask
    t = 20000 + 2 * (t % 10000)
    _check(h, w, t, b)
    b[20000:] = mask
    _check(h, w, t, b)


@pytest.mark.parametrize("D", [64, 256, 320, 640])
def test_masks_on_a_long_run_of_tiles(D):
    """Every block streams all classes; the reference of a row goes from far away to near zero and stays, or goes up from far to less far."""
    P, V = 3000, 1500
    h, w, t, b = _inputs(P, V, D, seed=D)
    steps = b.clone()
    b[:300] = -1e10
    b[640:700] = -1e20
    b[1100:1400] = -1e9
    keep = (b > -1e8).nonzero().flatten()
    _check(h, w, keep[t % keep.numel()], b, "sum")
    steps[:] = -1e20
    steps[400:] = -1e12
    steps[900:] = -1e10
    steps[1300:1310] = -1e9
    _check(h, w, t % 10 + 1300, steps, "none")


@pytest.mark.parametrize("shift", [1e6, 1e7, 1e10, 1e20, -1e7])
def test_scores_that_all_lie_far_away(shift):
    """A bias that moves every class alike; scores that survive next to it differ by whole steps of fp32."""
    h, w, t, b = _inputs(130, 600, 64, seed=5)
    h = torch.zeros_like(h)  # the scores are the biases: exact
    b = (torch.full((600,), shift, device="cuda", dtype=torch.float64) + torch.arange(600, device="cuda") % 7).float()
    _check(h, w, t, b)
    _check(h, w, t, b.flip(0), "mean")


@pytest.mark.parametrize("D", [64, 256, 320])
def test_products_that_are_large_by_themselves(D):
    """Scores of 2^34 and multiples of 2^27 below it, exact in fp32, without a bias; ties at the top in some rows."""
    g = torch.Generator().manual_seed(D)
    P, V = 140, 900
    h, w = torch.zeros(P, D), torch.zeros(V, D)
    h[:, 0] = 2.0**17
    w[:, 0] = 2.0**17 - 2.0**10 * torch.randint(0, 5, (V,), generator=g)
    h[::3, 0] *= -1  # the smallest products are the top of these rows
    w[:130, 0] = 2.0**16
    t = torch.randint(0, V, (P,), generator=g).cuda()
    _check(h.bfloat16().cuda(), w.bfloat16().cuda(), t, None)
    _check(h.bfloat16().cuda(), w.bfloat16().cuda(), t, None, "mean")


def test_a_mask_given_in_bf16():
    h, w, t, b = _inputs(80, 500, 64, seed=6)
    b[:200] = -1e9
    b = b.bfloat16()
    from torchrec_b200.ops.transformer_ops import full_softmax_loss

    t = t % 300 + 200
    got = full_softmax_loss(h, w, t, b, reduction="none")
    want = torch.nn.functional.cross_entropy((h.double() @ w.double().t()) + b.double(), t, reduction="none")
    torch.testing.assert_close(got.double(), want, rtol=2.0**-18, atol=2.0**-17)
