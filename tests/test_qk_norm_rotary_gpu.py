"""Norm and rotation of queries and keys (``rotary_kernels.cu``) against complex multiplication in fp64 and its autograd.

Tolerances.  fp32 arithmetic inside: a value passes about a dozen roundings of 2^-24 and a sum of head_dim squares, sine and cosine
are off by 2^-22; with ``u = 2^-19`` for all of that and ``e`` = half a step of the type, an output is off by at most ``(u + e)`` times
the magnitudes that enter it (turned pair), and a weight's gradient, a sum of n fp32 terms, by ``(u + n 2^-24)`` times the sum of theirs."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0**-19


def _oracle(qkv, pos, inv_freq, H, K, qw, kw, eps, sections, interleaved, norm, dout):
    T, half = qkv.shape[0], inv_freq.numel()
    dim = qkv.shape[1] // (H + 2 * K)
    R = 2 * half
    x = qkv.detach().double().requires_grad_(True)
    ws = [torch.ones(dim, dtype=torch.float64, device="cuda") if w is None else w.detach().double() for w in (qw, kw)]
    for w in ws:
        w.requires_grad_(True)
    place = [a for a, n in enumerate(sections) for _ in range(n)]
    angle = (pos.reshape(len(sections), T).double()[place] * inv_freq[:, None]).t()
    spin = torch.polar(torch.ones_like(angle), angle)[:, None]

    def turn(y, magnitude=False):
        rot, rest = y[..., :R], y[..., R:]
        pairs = rot.unflatten(-1, (half, 2)) if interleaved else rot.unflatten(-1, (2, half)).transpose(-1, -2)
        if magnitude:
            pairs = pairs.abs().sum(-1, keepdim=True).expand_as(pairs)
        else:
            pairs = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * spin)
        return torch.cat([pairs.flatten(-2) if interleaved else pairs.transpose(-1, -2).flatten(-2), rest.abs() if magnitude else rest], -1)

    def run(part, w):
        n = torch.sqrt(part.square().mean(-1, keepdim=True) + eps) if norm else 1
        return part / n, part / n * w

    heads = x.reshape(T, H + 2 * K, dim)
    (qx, q), (kx, k) = run(heads[:, :H], ws[0]), run(heads[:, H:H + K], ws[1])
    out = torch.cat([turn(q), turn(k), heads[:, H + K:]], 1).reshape(T, -1)
    dx, dqw, dkw = torch.autograd.grad(out, [x, *ws], dout.double(), allow_unused=True)
    mag = torch.cat([turn(q.detach(), True), turn(k.detach(), True), torch.zeros_like(heads[:, H + K:])], 1).reshape(T, -1)
    # gradient: rstd (|w g| + |x^| mean |w g x^|)
    d = dout.double().reshape(T, H + 2 * K, dim)
    mags, sums = [], []
    for part, xh, w, dd in ((heads[:, :H], qx, ws[0], d[:, :H]), (heads[:, H:H + K], kx, ws[1], d[:, H:H + K])):
        part, xh, w = part.detach(), xh.detach(), w.detach()
        g = turn(dd, True)
        r = 1 / torch.sqrt(part.square().mean(-1, keepdim=True) + eps) if norm else 1
        wg = (w * g).abs()
        mags.append(r * (wg + (xh.abs() * (wg * xh.abs()).mean(-1, keepdim=True) if norm else 0)))
        sums.append((g * xh.abs()).sum((0, 1)))
    gmag = torch.cat([*mags, torch.zeros_like(heads[:, H + K:])], 1).reshape(T, -1)
    return (out.detach(), dx, dqw, dkw), (mag.detach(), gmag.detach(), *sums)


def _within(name, got, want, tol):
    off = (got.double() - want).abs() - tol
    assert got.shape == want.shape and bool((off <= 0).all()), f"{name}: over its tolerance by {float(off.max())}"


def _check(T, H, K, dim, dtype=torch.bfloat16, half=None, sections=None, interleaved=False, weights=True, norm=True, seed=0, far=200, view=lambda t: t, scale=1.0):
    from torchrec_b200.ops.transformer_ops import qk_norm_rotary, rotary_inv_freq

    g = torch.Generator().manual_seed(seed)
    half = dim // 2 if half is None else half
    secs = sections or [half]
    qkv = view((torch.randn(T, (H + 2 * K) * dim, generator=g) * scale).to(dtype).cuda())
    pos = torch.randint(-far, far, (len(secs), T), generator=g).cuda()
    inv = rotary_inv_freq(2 * half, device="cuda")
    qw, kw = ((1 + 0.3 * torch.randn(dim, generator=g)).cuda() for _ in range(2)) if weights else (None, None)
    dout = view(torch.randn(T, (H + 2 * K) * dim, generator=g).to(dtype).cuda())
    leaves = [t.detach().requires_grad_(True) for t in (qkv, qw, kw) if t is not None]
    out = qk_norm_rotary(leaves[0], pos if sections else pos[0], inv, H, K, *(leaves[1:] if weights else (None, None)), eps=1e-6, sections=sections, interleaved=interleaved,
                         norm=norm)
    grads = torch.autograd.grad(out, leaves, dout)
    with torch.no_grad():
        assert torch.equal(out, qk_norm_rotary(qkv, pos.int(), inv, H, K, qw, kw, sections=sections, interleaved=interleaved, norm=norm))
    want, mag = _oracle(qkv, pos, inv, H, K, qw, kw, 1e-6, secs, interleaved, norm, dout)
    e = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).tiny * e  # values below the smallest normal are rounded to multiples of this
    _within("out", out.detach(), want[0], U * mag[0] + e * want[0].abs() * (1 + U) + tiny)
    _within("dqkv", grads[0], want[1], U * mag[1] + e * want[1].abs() * (1 + U) + tiny)
    v = slice((H + K) * dim, None)
    assert torch.equal(out[:, v], qkv[:, v]) and torch.equal(grads[0][:, v], dout[:, v])
    if weights:
        _within("dq_weight", grads[1], want[2], (U + T * H * 2.0**-24) * mag[2])
        _within("dk_weight", grads[2], want[3], (U + T * K * 2.0**-24) * mag[3])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim", [8, 32, 40, 48, 64, 80, 96, 128, 160, 256])
def test_head_dimensions(dtype, interleaved, dim):
    _check(37, 3, 2, dim, dtype, interleaved=interleaved, seed=dim)
    _check(5, 1, 1, dim, dtype, half=max(1, dim // 4), interleaved=interleaved, seed=dim + 1)


@pytest.mark.parametrize("T", [1, 2, 33, 1000, 20011])
def test_token_counts(T):
    _check(T, 4, 4, 64, seed=T)
    _check(T, 13, 1, 32, seed=T + 1, interleaved=True)


def test_odd_numbers_of_frequencies():
    for half in (1, 3, 7, 20, 31, 32):
        for interleaved in (False, True):
            _check(50, 2, 2, 64, half=half, interleaved=interleaved, seed=half)


def test_several_axes_and_far_positions():
    _check(300, 4, 2, 64, sections=[20, 12], far=10**6, seed=1)
    _check(300, 4, 2, 64, torch.float32, sections=[10, 0, 3, 19], far=2**31, seed=2)
    _check(300, 2, 2, 96, torch.float32, sections=[1, 47], interleaved=True, far=2**28, seed=3)


@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("norm", [False, True])
def test_parts_that_may_be_left_out(weights, norm):
    _check(70, 3, 3, 64, weights=weights, norm=norm, seed=4)


def test_strides_and_magnitudes():
    def inside(t):  # rows inside a wider buffer, on 16-byte boundaries
        wide = torch.zeros(t.shape[0], t.shape[1] + 48, dtype=t.dtype, device=t.device)
        wide[:, 16:16 + t.shape[1]] = t
        return wide[:, 16:16 + t.shape[1]]

    def off(t):  # and off them
        wide = torch.zeros(t.shape[0], t.shape[1] + 5, dtype=t.dtype, device=t.device)
        wide[:, 3:3 + t.shape[1]] = t
        return wide[:, 3:3 + t.shape[1]]

    for view in (inside, off, lambda t: t.t().contiguous().t(), lambda t: t[:1].expand_as(t)):
        _check(90, 2, 1, 64, view=view, seed=5)
    _check(90, 2, 1, 64, torch.float32, scale=1e6, seed=6)
    _check(90, 2, 1, 64, torch.float32, scale=1e-4, seed=7)  # eps counts


def test_heads_of_zeros():
    from torchrec_b200.ops.transformer_ops import qk_norm_rotary, rotary_inv_freq

    qkv = torch.zeros(9, 6 * 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    out = qk_norm_rotary(qkv, torch.arange(9, device="cuda"), rotary_inv_freq(64, device="cuda"), 2)
    out.sum().backward()
    assert float(out.detach().abs().max()) == 0 and bool(torch.isfinite(qkv.grad).all())
    none = qk_norm_rotary(qkv[:0], torch.arange(0, device="cuda"), rotary_inv_freq(64, device="cuda"), 2)
    assert none.shape == (0, 384)


def test_runs_twice_alike_on_other_streams_and_in_graphs():
    from torchrec_b200.ops.transformer_ops import qk_norm_rotary, rotary_inv_freq

    T, H, dim = 3000, 4, 64
    g = torch.Generator(device="cuda").manual_seed(8)
    data = [[torch.randn(T, 3 * H * dim, generator=g, device="cuda").bfloat16(), torch.rand(dim, generator=g, device="cuda"), torch.rand(dim, generator=g, device="cuda"),
             torch.randn(T, 3 * H * dim, generator=g, device="cuda").bfloat16(), torch.randint(0, 200, (T,), generator=g, device="cuda")] for _ in range(2)]
    inv = rotary_inv_freq(dim, device="cuda")

    def step(qkv, qw, kw, dout, pos):
        out = qk_norm_rotary(qkv, pos, inv, H, q_weight=qw, k_weight=kw)
        return [out.detach(), *torch.autograd.grad(out, (qkv, qw, kw), dout)]

    def leaves(x):
        return [t.clone().requires_grad_(i < 3) for i, t in enumerate(x)]

    want = [step(*leaves(x)) for x in data]
    assert all(torch.equal(x, y) for x, y in zip(step(*leaves(data[0])), want[0]))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    static = leaves(data[0])
    with torch.cuda.stream(side):
        got = step(*static)
    side.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want[0]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*static)
    for x, expect in ((data[1], want[1]), (data[0], want[0])):
        with torch.no_grad():
            for dst, src in zip(static, x):
                dst.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, expect))


def test_refusals_and_modes():
    from torchrec_b200.ops.transformer_ops import qk_norm_rotary, rotary_inv_freq

    qkv, pos, inv = torch.randn(5, 3 * 8, device="cuda"), torch.arange(5, device="cuda"), rotary_inv_freq(8, device="cuda")
    for bad in (dict(num_heads=0), dict(num_heads=1, num_kv_heads=2), dict(num_heads=2)):  # the last: heads of 4
        with pytest.raises(ValueError, match="qkv is|inv_freq"):
            qk_norm_rotary(qkv, pos, inv, **bad)
    for bad in (rotary_inv_freq(10, device="cuda"), inv[:0], inv[None], inv.int()):
        with pytest.raises(ValueError, match="inv_freq"):
            qk_norm_rotary(qkv, pos, bad, 1, sections=[4] if bad.dim() != 1 else None)
    for bad in (pos[:4], pos.float(), torch.stack([pos, pos])):
        with pytest.raises(ValueError, match="positions"):
            qk_norm_rotary(qkv, bad, inv, 1)
    for bad in ([3, 2], [5, -1], [1] * 9):
        with pytest.raises(ValueError, match="sections|axes"):
            qk_norm_rotary(qkv, torch.stack([pos] * len(bad)), inv, 1, sections=bad)
    with pytest.raises(ValueError, match="k_weight"):
        qk_norm_rotary(qkv, pos, inv, 1, k_weight=torch.ones(7, device="cuda"))
    with pytest.raises(ValueError, match="eps"):
        qk_norm_rotary(qkv, pos, inv, 1, eps=-1.0)
    for bad in (dict(positions=pos.cpu()), dict(inv_freq=inv.cpu()), dict(q_weight=torch.ones(8))):
        with pytest.raises(ValueError, match=" is on "):
            qk_norm_rotary(**{**dict(qkv=qkv, positions=pos, inv_freq=inv, num_heads=1), **bad})
    x = qkv.clone().requires_grad_(True)
    up = torch.ones(5, 24, device="cuda", requires_grad=True)
    (g,) = torch.autograd.grad(qk_norm_rotary(x, pos, inv, 1), x, up, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiated again"):
        g.sum().backward()
    with torch.inference_mode():
        assert not qk_norm_rotary(qkv, pos, inv, 1).requires_grad
    # one weight only, in another type; a head dimension that the kernel does not take
    kw = torch.rand(8, device="cuda").bfloat16().requires_grad_(True)
    qk_norm_rotary(x, pos, inv, 1, k_weight=kw).square().sum().backward()
    assert kw.grad.dtype == torch.bfloat16 and bool((kw.grad != 0).any())
    odd = torch.randn(5, 3 * 6, device="cuda")
    torch.testing.assert_close(qk_norm_rotary(odd, pos, inv[:3], 1).cpu(), qk_norm_rotary(odd.cpu(), pos.cpu(), inv[:3].cpu(), 1), rtol=1e-5, atol=1e-5)
