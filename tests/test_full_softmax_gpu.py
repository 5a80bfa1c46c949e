"""Softmax loss over the whole catalogue (``full_softmax_kernels.cu``) against the definition in fp64 on the same bf16 operands.

Tolerances.  A rounding to bf16 is off by at most 2^-8 of the value.  A score is a sum of D exact products in fp32: off by at most
``d = D 2^-23 sum_k |h_k w_k| + 2^-20 (1 + |z|)`` (the second part covers the base-2 logarithms and exponentials), which moves a
probability by the factor e^(2 d).  The terms of ``dh = G W`` and ``dW = G^T h`` are rounded to bf16 once, summed in fp32 (off by at
most n 2^-23 of the sum of magnitudes over n terms) and the result is rounded to bf16 once."""
import pytest
import torch

pytestmark = pytest.mark.gpu

IGNORE = -100


def _inputs(P, V, D, bias=True, ignored=0.0, seed=0, scale=1.5):
    g = torch.Generator().manual_seed(seed)
    h = torch.randn(P, D, generator=g).bfloat16()
    w = (torch.randn(V, D, generator=g) * scale / D**0.5).bfloat16()
    t = torch.randint(0, V, (P,), generator=g)
    t[torch.randperm(P, generator=g)[: int(P * ignored)]] = IGNORE
    b = torch.randn(V, generator=g) if bias else None
    return [None if x is None else x.cuda() for x in (h, w, t, b)]


def _oracle(h, w, t, b, dloss, reduction):
    """loss, dh, dw, db in fp64 and their tolerances."""
    h, w = h.detach().double(), w.detach().double()
    P, D = h.shape
    V = w.shape[0]
    keep = t != IGNORE
    h = torch.where(keep[:, None], h, 0)
    z = h @ w.t() + (0 if b is None else b.detach().double())
    tt = torch.where(keep, t, 0)
    # through the sum over the other classes: 1 - p_t would cancel to nothing in fp64 too
    zt = z.gather(1, tt[:, None])[:, 0]
    others = torch.logsumexp(z.scatter(1, tt[:, None], float("-inf")), 1) - zt
    rows = torch.logaddexp(others, torch.zeros_like(others))
    lse = zt + rows
    rows = torch.where(keep, rows, 0)
    n = max(1, int(keep.sum()))
    loss = {"none": rows, "mean": rows.sum() / n, "sum": rows.sum()}[reduction]
    G = torch.exp(z - lse[:, None])
    G[torch.arange(P, device=h.device), tt] = -torch.sigmoid(others)
    up = torch.where(keep, dloss.double() / (n if reduction == "mean" else 1), 0)
    G = torch.where(keep[:, None], G * up.reshape(-1, 1), 0)
    finite = z[torch.isfinite(z)].abs()
    d = D * 2.0**-23 * float((h.abs() @ w.abs().t()).max() if P else 0) + 2.0**-20 * (1 + float(finite.max() if finite.numel() else 0))
    e = torch.expm1(torch.tensor(2 * d)).item()
    bf = 2.0**-8
    # rows are summed in fp32 too; exponentials of far scores are flushed below 2^-126
    tol_loss = 2 * d * (P if reduction == "sum" else 1) + P * 2.0**-23 * float(loss.abs().nan_to_num(posinf=0).max() if P else 0)
    dh, dw, db = G @ w, G.t() @ h, G.sum(0)
    aw, ah = G.abs() @ w.abs(), G.abs().t() @ h.abs()
    tol_h = (bf + e + V * 2.0**-23) * aw + bf * dh.abs() + 1e-30
    tol_w = (bf + e + P * 2.0**-23) * ah + bf * dw.abs() + 1e-30
    tol_b = (e + (P + 8) * 2.0**-23) * G.abs().sum(0) + 1e-30
    return (loss, dh, dw, db), (tol_loss, tol_h, tol_w, tol_b)


def _within(name, got, want, tol):
    got = got.double()
    assert got.shape == want.shape, name
    same = (got == want) | (got.isnan() & want.isnan())
    off = torch.where(same, 0, (got - want).abs()) - tol
    assert bool((off <= 0).all()), f"{name}: over its tolerance by {float(off.max())}, error {float((got - want).abs().max())}"


def _check(h, w, t, b, reduction="mean", seed=3):
    from torchrec_b200.ops.transformer_ops import full_softmax_error, full_softmax_loss

    g = torch.Generator().manual_seed(seed)
    dloss = ((torch.rand(h.shape[0], generator=g) + 0.5) if reduction == "none" else torch.rand((), generator=g) + 0.5).cuda()
    leaves = [x.detach().requires_grad_(True) for x in (h, w, b) if x is not None]
    loss = full_softmax_loss(leaves[0], leaves[1], t, leaves[2] if b is not None else None, IGNORE, reduction)
    grads = torch.autograd.grad(loss, leaves, dloss)
    with torch.no_grad():
        again = full_softmax_loss(h, w, t, b, IGNORE, reduction)
    torch.cuda.synchronize()
    assert full_softmax_error(h.device) == 0
    want, tol = _oracle(h, w, t, b, dloss, reduction)
    _within("loss", loss.detach(), want[0], tol[0])
    _within("loss without gradients", again, want[0], tol[0])
    for name, got, x, lim, leaf in zip(("dh", "dw", "db"), grads, want[1:], tol[1:], leaves):
        assert got.dtype == leaf.dtype
        _within(name, got, x, lim)


@pytest.mark.parametrize("P,V,D", [(1, 1, 8), (1, 130, 64), (5, 127, 16), (129, 128, 72), (300, 1000, 128), (257, 513, 192), (641, 3001, 256)])
@pytest.mark.parametrize("bias", [False, True])
def test_matches_the_definition(P, V, D, bias):
    _check(*_inputs(P, V, D, bias, seed=P + D))


@pytest.mark.parametrize("P,V,D", [(130, 700, 264), (200, 900, 512), (130, 600, 640), (70, 300, 1024)])
def test_wide_rows(P, V, D):
    _check(*_inputs(P, V, D, True, seed=D), reduction="sum")


@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
@pytest.mark.parametrize("ignored", [0.3, 0.85, 1.0])
def test_reductions_and_ignored_rows(reduction, ignored):
    _check(*_inputs(700, 777, 96, True, ignored, seed=7), reduction=reduction)


@pytest.mark.parametrize("D", [1, 3, 33, 100, 250])
def test_widths_that_are_not_a_multiple_of_eight(D):
    _check(*_inputs(150, 301, D, True, 0.2, seed=D), reduction="none")


def test_many_pieces_of_either_axis():
    """Few rows against many classes splits the classes over the blocks, many rows against few classes splits the rows."""
    _check(*_inputs(3, 40001, 64, True, seed=1))
    _check(*_inputs(5000, 60, 64, True, 0.1, seed=2), reduction="none")
    _check(*_inputs(5000, 300, 256, False, 0.5, seed=3))


@pytest.mark.parametrize("D", [64, 128, 200, 256, 320, 640])
def test_long_runs_of_tiles(D):
    """More tiles of rows (classes) than the GPU has SMs: every block streams all classes (rows) past each of its tiles, through many uses
    of its buffers, and takes a second tile.  The maxima rise on the way in some rows."""
    g = torch.Generator().manual_seed(D)
    P, V = 19300, 1500
    level = (torch.arange(V) // 100).float() * 20
    h, w, t, b = _inputs(P, V, D, True, 0.01, seed=D)
    h[:, 0] = torch.where(torch.rand(P, generator=g) < 0.02, 1.0, 0.0).cuda().bfloat16()
    w[:, 0] = level.cuda().bfloat16()
    _check(h, w, t, b, "mean")
    _check(h[:1500].contiguous(), torch.cat([w] * 13)[:19300].contiguous(), t[:1500], None, "none")


def test_maximum_that_keeps_rising():
    """Scores that grow from tile to tile force the rescaling of the accumulator, in some rows more often than in others."""
    h, w, t, b = _inputs(200, 1500, 256, False, seed=5)
    ramp = torch.linspace(0, 1, 1500, device="cuda")[:, None]
    direction = torch.randn(256, generator=torch.Generator().manual_seed(9)).cuda()
    w = (w.float() + 4 * ramp * direction / 16).bfloat16()
    h = (h.float() + torch.linspace(0, 3, 200, device="cuda")[:, None] * direction / 4).bfloat16()
    _check(h, w, t, b)
    _check(-h, w, t, b, reduction="sum")


@pytest.mark.parametrize("D", [64, 256])
def test_maximum_that_rises_by_hundreds(D):
    """Maxima that grow by far more than what one reference can hold, tile after tile, in some rows only, and in one tile of many."""
    g = torch.Generator().manual_seed(D)
    V, P = 2600, 150
    level = (torch.arange(V) // 128).float() * 30  # a tile's scores are 30 above those of the tile before
    level[1000:1010] = 900
    h = torch.zeros(P, D)
    h[:, 0] = torch.linspace(0, 1, P)
    h[:, 1:] = torch.randn(P, D - 1, generator=g) / 8
    w = torch.randn(V, D, generator=g)
    w[:, 0] = level
    t = torch.randint(0, V, (P,), generator=g)
    h, w, t = h.bfloat16().cuda(), w.bfloat16().cuda(), t.cuda()
    _check(h, w, t, None, "none")
    _check(h, w.flip(0), t, None, "sum")
    _check(h, w, t, torch.randn(V, generator=g).cuda(), "mean")


def test_confident_rows_keep_their_accuracy():
    """Rows whose target has almost all of the probability: 1 - p_t must not be the difference of two rounded numbers."""
    h, w, t, b = _inputs(300, 900, 128, False, seed=6)
    h = (w[t].float() * torch.linspace(4, 30, 300, device="cuda")[:, None]).bfloat16()
    _check(h, w, t, b, reduction="none")


def test_classes_that_are_out_of_the_race():
    from torchrec_b200.ops.transformer_ops import full_softmax_loss

    h, w, t, b = _inputs(140, 900, 64, True, seed=8)
    b[:300] = float("-inf")  # more than two whole tiles
    b[650:700] = float("-inf")
    t = t % 350 + 300
    _check(h, w, t, b)
    t[3] = 10  # a target that cannot be reached
    rows = full_softmax_loss(h, w, t, b, reduction="none")
    assert float(rows[3]) == float("inf") and bool(torch.isfinite(rows[4:]).all())
    only = torch.full_like(b, float("-inf"))
    only[5] = 0.5
    t[:] = 5
    hh = h.clone().requires_grad_(True)
    rows = full_softmax_loss(hh, w, t, only, reduction="sum")
    rows.backward()
    assert float(rows.detach()) == 0 and float(hh.grad.abs().max()) == 0


def test_ignored_rows_may_hold_anything():
    from torchrec_b200.ops.transformer_ops import full_softmax_loss

    h, w, t, b = _inputs(300, 500, 64, True, 0.4, seed=10)
    want = full_softmax_loss(h, w, t, b)
    bad = h.clone()
    bad[t == IGNORE] = float("nan")
    bad[(t == IGNORE).nonzero()[0]] = float("inf")
    _check(bad, w, t, b)
    assert torch.equal(want, full_softmax_loss(bad, w, t, b))


def test_targets_outside_the_classes_are_reported():
    from torchrec_b200.ops.transformer_ops import full_softmax_error, full_softmax_loss

    h, w, t, b = _inputs(200, 300, 64, True, seed=11)
    t[7], t[150] = 300, -1
    hh = h.clone().requires_grad_(True)
    rows = full_softmax_loss(hh, w, t, b, reduction="none")
    rows.sum().backward()
    assert rows.isnan().nonzero().flatten().tolist() == [7, 150]
    assert float(hh.grad[[7, 150]].abs().max()) == 0 and bool(torch.isfinite(hh.grad).all())
    assert full_softmax_error(h.device) == 16 and full_softmax_error(h.device) == 0
    assert bool(full_softmax_loss(h, w, t, b).isnan())
    assert full_softmax_error(h.device) == 16


def test_strides_and_types():
    from torchrec_b200.ops import dense_ops
    from torchrec_b200.ops.transformer_ops import full_softmax_loss

    h, w, t, b = _inputs(260, 410, 64, True, 0.1, seed=12)
    wide = torch.zeros(260, 200, device="cuda", dtype=torch.bfloat16)
    wide[:, 3:67] = h  # rows that start off a 16-byte boundary
    wide_w = torch.zeros(410, 136, device="cuda", dtype=torch.bfloat16)
    wide_w[:, 8:72] = w
    t2 = torch.stack([t, t + 1], 1)[:, 0]
    b2 = torch.stack([b, b], 1)[:, 1]
    want = full_softmax_loss(h, w, t, b)
    assert torch.equal(want, full_softmax_loss(wide[:, 3:67], w, t, b))
    assert torch.equal(want, full_softmax_loss(h.t().contiguous().t(), w, t.int(), b))
    assert torch.equal(want, full_softmax_loss(h, wide_w[:, 8:72], t2, b2))
    assert torch.equal(want, full_softmax_loss(h, wide_w[:, 8:72].clone(memory_format=torch.contiguous_format)[:, :], t, b.bfloat16().float() * 0 + b))
    _check(wide[:, 3:67], wide_w[:, 8:72], t2, b2, "none")
    # fp32 parameters are rounded once and get fp32 gradients
    p = torch.nn.Parameter(w.float() * 1.001)
    h32 = (h.float() * 1.001).requires_grad_(True)
    prev = dense_ops.get_dense_compute_dtype()
    dense_ops.set_dense_compute_dtype(torch.bfloat16)
    try:
        loss = full_softmax_loss(h32, p, t, b)
    finally:
        dense_ops.set_dense_compute_dtype(prev)
    one = torch.ones((), device="cuda")
    gh, gw = torch.autograd.grad(loss, (h32, p), one)
    assert gh.dtype == gw.dtype == torch.float32
    want, tol = _oracle(h32.detach().bfloat16(), p.detach().bfloat16(), t, b, one, "mean")
    _within("loss", loss.detach(), want[0], tol[0])
    _within("dh", gh, want[1], tol[1])
    _within("dw", gw, want[2], tol[2])
    dense_ops.bf16_cache.clear()


def test_runs_twice_alike_and_wants_only_what_is_asked_for():
    from torchrec_b200.ops.transformer_ops import full_softmax_loss

    h, w, t, b = _inputs(1000, 2000, 128, True, 0.2, seed=13)
    results = []
    for _ in range(2):
        leaves = [x.detach().clone().requires_grad_(True) for x in (h, w, b)]
        loss = full_softmax_loss(leaves[0], leaves[1], t, leaves[2])
        results.append([loss.detach(), *torch.autograd.grad(loss, leaves)])
    assert all(torch.equal(x, y) for x, y in zip(*results))
    want, tol = _oracle(h, w, t, b, torch.ones((), device="cuda"), "mean")
    for i in range(3):  # one gradient at a time; without dh the log sum is added up in another order
        leaves = [x.detach().clone() for x in (h, w, b)]
        leaves[i].requires_grad_(True)
        (got,) = torch.autograd.grad(full_softmax_loss(leaves[0], leaves[1], t, leaves[2]), [leaves[i]])
        _within(("dh", "dw", "db")[i], got, want[1 + i], tol[1 + i])


def test_other_streams_and_captured_graphs():
    from torchrec_b200.ops.transformer_ops import full_softmax_error, full_softmax_loss

    a = _inputs(400, 900, 64, True, 0.3, seed=14)
    other = _inputs(400, 900, 64, True, 0.6, seed=15)

    def step(h, w, t, b):
        loss = full_softmax_loss(h, w, t, b, reduction="mean")
        return [loss.detach(), *torch.autograd.grad(loss, (h, w, b))]

    def leaves(x):
        return [x[0].clone().requires_grad_(True), x[1].clone().requires_grad_(True), x[2].clone(), x[3].clone().requires_grad_(True)]

    want = [step(*leaves(x)) for x in (a, other)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(*leaves(a))
    side.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want[0]))
    static = leaves(a)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*static)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):  # two graphs over the same inputs, replayed in turn
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(*static)
        graphs.append((g, out))
    for data, expect in ((other, want[1]), (a, want[0])):
        with torch.no_grad():
            for dst, src in zip(static, data):
                dst.copy_(src)
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(x, y) for x, y in zip(out, expect))
    assert full_softmax_error(a[0].device) == 0


def test_refusals_and_modes():
    from torchrec_b200.ops.transformer_ops import full_softmax_loss

    h, w, t, b = _inputs(20, 30, 16, True, seed=16)
    with pytest.raises(ValueError, match="reduction"):
        full_softmax_loss(h, w, t, reduction="max")
    for bad in ((h, w[:, :8]), (h, w[:0])):
        with pytest.raises(ValueError, match="h \\[P, D\\]"):
            full_softmax_loss(*bad, t)
    for bad in (t[:3], t.float(), t[:, None]):
        with pytest.raises(ValueError, match="targets"):
            full_softmax_loss(h, w, bad)
    with pytest.raises(ValueError, match="bias"):
        full_softmax_loss(h, w, t, b[:29])
    for bad in ((h, w.cpu(), t), (h, w, t.cpu()), (h, w, t, b.cpu())):
        with pytest.raises(ValueError, match=" is on "):
            full_softmax_loss(*bad)
    leaves = [x.clone().requires_grad_(True) for x in (h, w, b)]
    loss = full_softmax_loss(leaves[0], leaves[1], t, leaves[2])
    up = torch.ones((), device="cuda", requires_grad=True)
    grads = torch.autograd.grad(loss, leaves, up, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiated again"):
        grads[0].float().sum().backward()
    loss = full_softmax_loss(leaves[0], leaves[1], t, leaves[2])
    with torch.no_grad():
        leaves[1].mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():
        assert not full_softmax_loss(h, w, t, b).requires_grad
    # tensors of more than the kernel's width take the piecewise path
    wide = [x.requires_grad_(True) for x in (torch.randn(5, 1040, device="cuda").bfloat16(), (torch.randn(9, 1040, device="cuda") / 30).bfloat16())]
    target = torch.arange(5, device="cuda")
    want = torch.nn.functional.cross_entropy(wide[0].double() @ wide[1].double().t(), target)
    got = full_softmax_loss(*wide, target)
    assert abs(float(got.detach()) - float(want.detach())) < 1e-5
    for x, y in zip(torch.autograd.grad(got, wide), torch.autograd.grad(want, wide)):
        torch.testing.assert_close(x.double(), y.double(), rtol=2.0**-7, atol=1e-6)  # a bf16 rounding on either side


def test_bias_types_and_gradients_that_come_expanded():
    from torchrec_b200.ops.transformer_ops import full_softmax_loss

    h, w, t, b = _inputs(200, 300, 64, True, 0.2, seed=17)
    b16 = b.bfloat16()
    leaves = [x.clone().requires_grad_(True) for x in (h, w, b16)]
    rows = full_softmax_loss(leaves[0], leaves[1], t, leaves[2], reduction="none")
    rows.sum().backward()  # the upstream gradient is one value, expanded
    want, tol = _oracle(h, w, t, b16.float(), torch.ones(200, device="cuda"), "none")
    for name, leaf, x, lim in zip(("dh", "dw", "db"), leaves, want[1:], tol[1:]):
        assert leaf.grad.dtype == torch.bfloat16
        _within(name, leaf.grad, x, lim + (2.0**-8 * x.abs() if name == "db" else 0))
