"""The transformer operators of sequence recommenders that are measured: the softmax loss over all items with its gradient, and
the norm and rotation of queries and keys in packed ``q | k | v`` tokens with its gradient.

``run`` computes a case's operator in plain 32-bit torch operations (``own = False``) or through the package (``own = True``);
``exact`` computes the same values in 64 bits through autograd of the definition."""
from __future__ import annotations

import math

import torch

own = False

IGNORE = -100


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------
def _loss(name, mode, P, V, D, bias=True, ignored=0.0, reduction="mean"):
    return {"name": name, "op": "softmax_loss", "mode": mode, "P": P, "V": V, "D": D, "bias": bias, "ignored": ignored, "reduction": reduction}


def _rotary(name, mode, T, heads, kv_heads, head_dim, dtype="bf16", rotary_dim=None, sections="", interleaved=False, weights=True):
    return {"name": name, "op": "qk_rotary", "mode": mode, "T": T, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype,
            "rotary_dim": rotary_dim or head_dim, "sections": sections, "interleaved": interleaved, "weights": weights}


def listed():
    return [
        # one position scored against the example's catalogue: evaluation of a single request
        _loss("loss one position", "eval", 1, 20000, 64),
        # the masked positions of one batch of the BERT4Rec example (64 sessions of up to 50 items, 15 % masked)
        _loss("loss example step", "step", 260, 20000, 64),
        # all positions of a batch with the unmasked ones ignored, one gradient per row (weighted sessions), odd sizes
        _loss("loss ragged step", "step", 3001, 50021, 128, bias=False, ignored=0.85, reduction="none"),
        # wider hidden size, catalogue of a mid-size shop
        _loss("loss wide step", "step", 4096, 30011, 512, reduction="sum"),
        # validation loss of a large catalogue at the benchmark's hidden size
        _loss("loss catalogue eval", "eval", 8192, 100003, 256, bias=False),
        # training at the benchmark's hidden size over a catalogue of 131 thousand items
        _loss("loss catalogue step", "step", 16384, 131071, 256),
        # one new token of a session
        _rotary("rotary one token", "eval", 1, 4, 4, 64),
        # a batch of sessions with a time axis beside the place in the session
        _rotary("rotary two axes step", "step", 6977, 4, 4, 64, sections="20,12"),
        # shared key heads, adjacent pairs, 32-bit parameters and activations
        _rotary("rotary shared heads step", "step", 20011, 16, 2, 128, dtype="fp32", interleaved=True),
        # half of every head rotated, no learned scale, 16-bit floats, inference over a long batch
        _rotary("rotary partial eval", "eval", 131075, 8, 8, 96, dtype="fp16", rotary_dim=48, weights=False),
        # the sequence benchmark: 4096 sessions of 20 to 200 items, 4 heads of 64
        _rotary("rotary benchmark step", "step", 450563, 4, 4, 64),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.5:
        while True:
            P, V, D = _log_int(rng, 1, 16384), _log_int(rng, 500, 131071), 8 * _log_int(rng, 4, 64)
            if P * V * D <= 16384 * 131071 * 256:
                break
        c = _loss("", rng.choice(["step", "step", "eval"]), P, V, D, rng.random() < 0.5, rng.choice([0.0, 0.0, 0.3, 0.85]), rng.choice(["mean", "sum", "none"]))
    else:
        while True:
            T, heads, kv, dim = _log_int(rng, 1, 450563), rng.randint(1, 16), rng.randint(1, 8), rng.choice([32, 48, 64, 80, 96, 128, 160, 256])
            if kv <= heads and T * (heads + 2 * kv) * dim <= 450563 * 12 * 64:
                break
        rot = rng.choice([dim, dim, dim // 2])
        first = rng.randint(1, rot // 2 - 1)
        sections = rng.choice(["", "", "%d,%d" % (first, rot // 2 - first)])
        c = _rotary("", rng.choice(["step", "step", "eval"]), T, heads, kv, dim, rng.choice(["bf16", "bf16", "fp16", "fp32"]), rot, sections, rng.random() < 0.5,
                    rng.random() < 0.7)
    del c["name"]
    return c


def _valid_rows(case):
    return case["P"] - int(case["P"] * case["ignored"])


def work(case):
    if case["op"] == "softmax_loss":
        P, V, D = _valid_rows(case), case["V"], case["D"]
        operands = 2 * (P * D + V * D) + 8 * case["P"] + 4 * V * case["bias"]
        loss = 4 * (case["P"] if case["reduction"] == "none" else 1)
        if case["mode"] == "eval":
            return {"bytes": operands + loss, "flops": 2.0 * P * V * D}
        return {"bytes": operands + loss + 2 * (case["P"] * D + V * D) + 4 * V * case["bias"], "flops": 6.0 * P * V * D}
    item = 4 if case["dtype"] == "fp32" else 2
    T, turned, all_heads, dim = case["T"], case["heads"] + case["kv_heads"], case["heads"] + 2 * case["kv_heads"], case["head_dim"]
    axes = len(case["sections"].split(",")) if case["sections"] else 1
    fwd = 2 * T * all_heads * dim * item + 8 * T * axes
    if case["mode"] == "eval":
        return {"bytes": fwd, "flops": 8.0 * T * turned * dim}
    return {"bytes": fwd + 2 * T * all_heads * dim * item + T * turned * dim * item, "flops": 24.0 * T * turned * dim}


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    step = case["mode"] == "step"
    if case["op"] == "softmax_loss":
        P, V, D = case["P"], case["V"], case["D"]
        weight = (normal(V, D) * (1.5 / math.sqrt(D))).bfloat16()
        # popular items come first: u ** 3 puts more of the targets on low ids
        targets = (torch.rand(P, generator=g, device="cuda") ** 3 * V).long().clamp_(max=V - 1)
        # a trained model leans towards its targets, from hardly to strongly
        lean = torch.rand(P, 1, generator=g, device="cuda") * 4
        h = (normal(P, D) + lean * weight.index_select(0, targets).float()).bfloat16()
        bias = normal(V) * 0.5 if case["bias"] else None
        drop = torch.randperm(P, generator=g, device="cuda")[: P - _valid_rows(case)]
        targets[drop] = IGNORE
        dloss = torch.rand(P, generator=g, device="cuda") + 0.5 if case["reduction"] == "none" else torch.rand((), generator=g, device="cuda") + 0.5
        if step:
            for t in (h, weight, bias):
                if t is not None:
                    t.requires_grad_(True)
        return {"case": case, "h": h, "weight": weight, "targets": targets, "bias": bias, "dloss": dloss}
    dtype = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}[case["dtype"]]
    T, H, K, dim = case["T"], case["heads"], case["kv_heads"], case["head_dim"]
    qkv = normal(T, (H + 2 * K) * dim).to(dtype)
    sections = [int(s) for s in case["sections"].split(",")] if case["sections"] else None
    positions = torch.randint(0, 200, (T,), generator=g, device="cuda")
    if sections:  # further axes count hours or seconds: far positions
        positions = torch.stack([positions] + [torch.randint(0, 10**6, (T,), generator=g, device="cuda") for _ in sections[1:]])
    j = torch.arange(case["rotary_dim"] // 2, device="cuda", dtype=torch.float64)
    inv_freq = 10000.0 ** (-2 * j / case["rotary_dim"])
    qw, kw = (1 + 0.2 * normal(dim) for _ in range(2)) if case["weights"] else (None, None)
    dout = normal(T, (H + 2 * K) * dim).to(dtype) if step else None
    if step:
        for t in (qkv, qw, kw):
            if t is not None:
                t.requires_grad_(True)
    return {"case": case, "qkv": qkv, "positions": positions, "inv_freq": inv_freq, "sections": sections, "qw": qw, "kw": kw, "dout": dout}


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def _plain_loss(s):
    c, targets, dloss = s["case"], s["targets"], s["dloss"]
    h, w = s["h"].detach().float(), s["weight"].detach().float()
    z = h @ w.t()
    if s["bias"] is not None:
        z += s["bias"].detach()
    keep = targets != IGNORE
    t = targets.clamp(min=0).unsqueeze(1)
    zt = z.gather(1, t)
    m = z.amax(1, keepdim=True)
    e = z.sub_(m).exp_()
    total = e.sum(1, keepdim=True)
    rows = torch.where(keep, (m + total.log() - zt).squeeze(1), 0.0)
    n = keep.sum().clamp(min=1)
    loss = rows if c["reduction"] == "none" else rows.sum() if c["reduction"] == "sum" else rows.sum() / n
    if c["mode"] == "eval":
        return [loss]
    scale = (dloss / n if c["reduction"] == "mean" else dloss) * keep
    p = e.div_(total)
    p.scatter_add_(1, t, torch.full_like(total, -1.0))
    p *= scale.unsqueeze(1)
    return [loss, (p @ w).bfloat16(), (p.t() @ h).bfloat16()] + ([p.sum(0)] if s["bias"] is not None else [])


def _turn(x, cos, sin, interleaved):
    """Rotates the first 2 * len(cos) values of every head; pairs are neighbours, or lie half the rotated part apart."""
    half = cos.shape[-1]
    part, rest = x[..., : 2 * half], x[..., 2 * half :]
    a, b = (part[..., 0::2], part[..., 1::2]) if interleaved else (part[..., :half], part[..., half:])
    u, v = a * cos - b * sin, a * sin + b * cos
    part = torch.stack([u, v], -1).flatten(-2) if interleaved else torch.cat([u, v], -1)
    return torch.cat([part, rest], -1)


def _angles(s):
    pos, f = s["positions"], s["inv_freq"]
    if s["sections"]:
        axis = torch.repeat_interleave(torch.arange(len(s["sections"]), device=f.device), torch.tensor(s["sections"], device=f.device), output_size=f.numel())
        return pos.index_select(0, axis).t().double() * f
    return pos.double().unsqueeze(1) * f


def _plain_rotary(s):
    c, eps = s["case"], 1e-6
    T, H, K, dim = c["T"], c["heads"], c["kv_heads"], c["head_dim"]
    angles = _angles(s)
    cos, sin = angles.cos().float().unsqueeze(1), angles.sin().float().unsqueeze(1)
    x = s["qkv"].detach().float().reshape(T, H + 2 * K, dim)
    qk, v = x[:, : H + K], x[:, H + K :]
    ones = torch.ones(dim, device=x.device)
    qw, kw = (ones, ones) if s["qw"] is None else (s["qw"].detach(), s["kw"].detach())
    w = torch.cat([qw.expand(H, dim), kw.expand(K, dim)])
    rstd = (qk.square().mean(-1, keepdim=True) + eps).rsqrt()
    xhat = qk * rstd
    out = torch.cat([_turn(xhat * w, cos, sin, c["interleaved"]), v], 1).reshape(T, -1).to(s["qkv"].dtype)
    if c["mode"] == "eval":
        return [out]
    d = s["dout"].float().reshape(T, H + 2 * K, dim)
    back = _turn(d[:, : H + K], cos, -sin, c["interleaved"])
    wg = back * w
    dqk = rstd * (wg - xhat * (wg * xhat).mean(-1, keepdim=True))
    dqkv = torch.cat([dqk, d[:, H + K :]], 1).reshape(T, -1).to(s["qkv"].dtype)
    if s["qw"] is None:
        return [out, dqkv]
    dw = back * xhat
    return [out, dqkv, dw[:, :H].sum((0, 1)), dw[:, H:].sum((0, 1))]


def run(state):
    s, c = state, state["case"]
    step = c["mode"] == "step"
    if c["op"] == "softmax_loss":
        if not own:
            return _plain_loss(s)
        from torchrec_b200.ops.transformer_ops import full_softmax_loss

        loss = full_softmax_loss(s["h"], s["weight"], s["targets"], s["bias"], ignore_index=IGNORE, reduction=c["reduction"])
        if not step:
            return [loss]
        leaves = [t for t in (s["h"], s["weight"], s["bias"]) if t is not None]
        return [loss.detach(), *torch.autograd.grad(loss, leaves, s["dloss"])]
    if not own:
        return _plain_rotary(s)
    from torchrec_b200.ops.transformer_ops import qk_norm_rotary

    out = qk_norm_rotary(s["qkv"], s["positions"], s["inv_freq"], c["heads"], c["kv_heads"], s["qw"], s["kw"], eps=1e-6, sections=s["sections"],
                         interleaved=c["interleaved"])
    if not step:
        return [out]
    leaves = [t for t in (s["qkv"], s["qw"], s["kw"]) if t is not None]
    return [out.detach(), *torch.autograd.grad(out, leaves, s["dout"])]


# ---------------------------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def _exact_loss(s):
    c = s["case"]
    P, step = c["P"], c["mode"] == "step"
    h, w = s["h"].detach().double(), s["weight"].detach().double().requires_grad_(step)
    b = None if s["bias"] is None else s["bias"].detach().double().requires_grad_(step)
    keep = s["targets"] != IGNORE
    n = max(1, int(keep.sum()))
    rows, dh = torch.zeros(P, dtype=torch.float64, device=h.device), torch.zeros_like(h)
    index = keep.nonzero().squeeze(1)
    up = s["dloss"].double().expand(P) / (n if c["reduction"] == "mean" else 1)
    piece = max(1, 2**28 // c["V"])  # rows whose scores take two gigabytes
    for lo in range(0, index.numel(), piece):
        i = index[lo : lo + piece]
        x = h[i].requires_grad_(step)
        z = x @ w.t()
        if b is not None:
            z = z + b
        r = torch.logsumexp(z, 1) - z[torch.arange(i.numel(), device=z.device), s["targets"][i]]
        rows[i] = r.detach()
        if step:
            (r * up[i]).sum().backward()
            dh[i] = x.grad
        del x, z, r
    loss = rows if c["reduction"] == "none" else rows.sum() / (n if c["reduction"] == "mean" else 1)
    if not step:
        return [loss]
    return [loss, dh, torch.zeros_like(w) if w.grad is None else w.grad] + ([] if b is None else [torch.zeros_like(b) if b.grad is None else b.grad])


def _exact_rotary(s):
    c = s["case"]
    T, H, K, dim, R = c["T"], c["heads"], c["kv_heads"], c["head_dim"], c["rotary_dim"]
    step = c["mode"] == "step"
    x = s["qkv"].detach().double().requires_grad_(step)
    weights = [torch.ones(dim, dtype=torch.float64, device=x.device) if t is None else t.detach().double().requires_grad_(step) for t in (s["qw"], s["kw"])]
    pos = s["positions"].double().reshape(-1, T)
    place = [a for a, n in enumerate(s["sections"] or [R // 2]) for _ in range(n)]  # the axis of each frequency
    spin = torch.polar(torch.ones((), dtype=torch.float64, device=x.device), (pos[place] * s["inv_freq"].double().unsqueeze(1)).t()).unsqueeze(1)
    heads = x.reshape(T, H + 2 * K, dim)

    def turned(part, w):
        y = part / torch.sqrt((part * part).mean(-1, keepdim=True) + 1e-6) * w
        first, last = y[..., :R], y[..., R:]
        pairs = first.unflatten(-1, (R // 2, 2)) if c["interleaved"] else first.unflatten(-1, (2, R // 2)).transpose(-1, -2)
        pairs = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * spin)
        first = pairs.flatten(-2) if c["interleaved"] else pairs.transpose(-1, -2).flatten(-2)
        return torch.cat([first, last], -1)

    out = torch.cat([turned(heads[:, :H], weights[0]), turned(heads[:, H : H + K], weights[1]), heads[:, H + K :]], 1).reshape(T, -1)
    if not step:
        return [out]
    out.backward(s["dout"].double())
    return [out.detach(), x.grad] + ([w.grad for w in weights] if s["qw"] is not None else [])


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_loss(s) if case["op"] == "softmax_loss" else _exact_rotary(s)
