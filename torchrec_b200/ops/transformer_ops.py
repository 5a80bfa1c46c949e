"""Fused elementwise / normalisation pieces of a transformer block over packed tokens ``[T, D]`` (CUDA: ``transformer_kernels.cu``;
elsewhere plain torch, which is also the oracle of the kernel tests).

``residual_layer_norm(a, r, weight, bias, p)`` returns ``(s, y)`` with ``s = r + dropout(a)`` (the residual stream, ``a`` may be
``None``) and ``y = layer_norm(s)``: one pass instead of dropout + add + layer norm, in bf16 with fp32 statistics.
``gelu_dropout(z, p)`` is ``dropout(gelu(z))``.  Dropout masks are recomputed from a per-call seed in the backward instead of being
stored.  ``packed_attention(qkv, offsets, heads, max_len, p)`` is self-attention inside every sequence of packed tokens
(``varlen_attention.cu``).  ``sampled_softmax_loss(h, positive, negatives)`` is the cross entropy of a sampled softmax with its
gradient produced in the same pass over the scores (``sampled_softmax_kernels.cu``).  ``full_softmax_loss(h, weight, targets, bias)``
is the cross entropy over all rows of ``weight``, with its gradient, without keeping the scores (``full_softmax_kernels.cu``).
``qk_norm_rotary(qkv, positions, inv_freq, heads)`` normalises the queries and keys of every head and turns them by their token's
position, in one pass over the packed tokens in front of the attention (``rotary_kernels.cu``).
"""
from __future__ import annotations

import itertools
from typing import Optional, Sequence, Tuple

import torch
import torch.autograd.forward_ad as fwAD

from torchrec_b200.ops import _ext, dense_ops

_seed_counter = itertools.count(0x5EED)


def _next_seed() -> int:
    """A fresh dropout seed per call, derived from torch's generator so that ``torch.manual_seed`` makes runs repeatable."""
    base = int(torch.initial_seed()) & 0x7FFFFFFF
    return (base * 1_000_003 + next(_seed_counter)) & 0x7FFFFFFFFFFFFFFF


def _kernel_ok(r: torch.Tensor) -> bool:
    return (r.is_cuda and _ext.has_cuda_ext() and r.dtype == torch.bfloat16 and r.dim() == 2 and r.is_contiguous()
            and r.shape[1] % 256 == 0 and r.shape[1] <= 1024)


class _ResidualLayerNorm(torch.autograd.Function):
    """(a, r) -> (s, y): both outputs carry gradient (s feeds the next residual connection, y the next sub-block)."""

    @staticmethod
    def forward(ctx, a, r, weight, bias, p: float, eps: float):
        seed = _next_seed()
        s, y, mean, rstd = torch.ops.trb200.ln_residual_fwd(a, r, weight.float(), bias.float(), p, seed, eps)
        ctx.save_for_backward(s, weight, mean, rstd)
        ctx.cfg = (p, seed)
        return s, y

    @staticmethod
    def backward(ctx, ds_extra, dy):
        s, weight, mean, rstd = ctx.saved_tensors
        p, seed = ctx.cfg
        dy = torch.zeros_like(s) if dy is None else dy.contiguous().to(torch.bfloat16)
        extra = None if ds_extra is None else ds_extra.contiguous().to(torch.bfloat16)
        ds, da, dgamma, dbeta = torch.ops.trb200.ln_residual_bwd(extra, dy, s, weight.float(), mean, rstd, p, seed, True)
        return da, ds, dgamma.to(weight.dtype), dbeta.to(weight.dtype), None, None


class _LayerNorm(torch.autograd.Function):
    """r -> layer_norm(r): the same kernels without the dropout-add half."""

    @staticmethod
    def forward(ctx, r, weight, bias, eps: float):
        _, y, mean, rstd = torch.ops.trb200.ln_residual_fwd(None, r, weight.float(), bias.float(), 0.0, 0, eps)
        ctx.save_for_backward(r, weight, mean, rstd)
        return y

    @staticmethod
    def backward(ctx, dy):
        r, weight, mean, rstd = ctx.saved_tensors
        ds, _, dgamma, dbeta = torch.ops.trb200.ln_residual_bwd(None, dy.contiguous().to(torch.bfloat16), r, weight.float(), mean, rstd, 0.0, 0, False)
        return ds, dgamma.to(weight.dtype), dbeta.to(weight.dtype), None


def residual_layer_norm(a: Optional[torch.Tensor], r: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor, p: float = 0.0,
                        training: bool = True, eps: float = 1e-5) -> Tuple[torch.Tensor, torch.Tensor]:
    """``s = r + dropout(a, p)`` (``a`` may be ``None``), ``y = layer_norm(s) * weight + bias``; returns ``(s, y)``."""
    p = float(p) if training else 0.0
    if _kernel_ok(r) and (a is None or (a.shape == r.shape and a.dtype == r.dtype)):
        if a is None:
            return r, _LayerNorm.apply(r, weight, bias, eps)
        return _ResidualLayerNorm.apply(a.contiguous(), r, weight, bias, p, eps)
    s = r if a is None else r + torch.nn.functional.dropout(a, p, training=p > 0)
    y = torch.nn.functional.layer_norm(s.float(), (s.shape[-1],), weight.float(), bias.float(), eps).to(s.dtype)
    return s, y


class _GeluDropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, z, p: float):
        seed = _next_seed()
        ctx.save_for_backward(z)
        ctx.cfg = (p, seed)
        return torch.ops.trb200.gelu_dropout_fwd(z, p, seed)

    @staticmethod
    def backward(ctx, dh):
        (z,) = ctx.saved_tensors
        p, seed = ctx.cfg
        return torch.ops.trb200.gelu_dropout_bwd(dh.contiguous().to(torch.bfloat16), z, p, seed), None


def gelu_dropout(z: torch.Tensor, p: float = 0.0, training: bool = True) -> torch.Tensor:
    """``dropout(gelu(z), p)`` (exact erf form)."""
    p = float(p) if training else 0.0
    if z.is_cuda and _ext.has_cuda_ext() and z.dtype == torch.bfloat16 and z.is_contiguous() and z.numel() % 8 == 0:
        return _GeluDropout.apply(z, p)
    return torch.nn.functional.dropout(torch.nn.functional.gelu(z), p, training=p > 0)


# --------------------------------------------------------------------------------------
# attention over packed sequences
# --------------------------------------------------------------------------------------
ATTENTION_HEAD_DIM = 64     # the kernel's head dimension
ATTENTION_MAX_LEN = 768     # longest sequence whose K and V (or Q and dO) fit in one CTA's shared memory
_attn_err: dict = {}


def _attention_error_word(device: torch.device) -> torch.Tensor:
    word = _attn_err.get(device)
    if word is None:
        word = _attn_err[device] = torch.zeros(1, dtype=torch.int32, device=device)
    return word


def attention_error(device: torch.device) -> int:
    """Non-zero after a packed-attention launch met a sequence longer than its ``max_len`` (the tail of that sequence got zeros).
    Reading it synchronises with the device."""
    word = _attn_err.get(torch.device(device))
    return 0 if word is None else int(word.item())


def packed_attention_supported(qkv: torch.Tensor, num_heads: int, max_len: int) -> bool:
    return (qkv.is_cuda and _ext.has_cuda_ext() and qkv.dtype == torch.bfloat16 and qkv.dim() == 2 and qkv.shape[1] == 3 * num_heads * ATTENTION_HEAD_DIM
            and 1 <= max_len <= ATTENTION_MAX_LEN)


class _PackedAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, qkv, offsets, num_heads: int, max_len: int, p: float):
        seed = _next_seed() if p > 0 else 0
        err = _attention_error_word(qkv.device)
        out, lse = torch.ops.trb200.varlen_attn_fwd(qkv, offsets, num_heads, max_len, p, seed, err)
        ctx.save_for_backward(qkv, out, lse, offsets)
        ctx.cfg = (num_heads, max_len, p, seed)
        return out

    @staticmethod
    def backward(ctx, dout):
        qkv, out, lse, offsets = ctx.saved_tensors
        num_heads, max_len, p, seed = ctx.cfg
        dqkv = torch.ops.trb200.varlen_attn_bwd(dout.contiguous().to(torch.bfloat16), qkv, out, lse, offsets, num_heads, max_len, p, seed,
                                                _attention_error_word(qkv.device))
        return dqkv, None, None, None, None


def packed_attention(qkv: torch.Tensor, offsets: torch.Tensor, num_heads: int, max_len: int, p: float = 0.0) -> torch.Tensor:
    """Self-attention inside every sequence of the packed ``qkv [T, 3 * D]`` (``q | k | v`` along the columns, head dimension 64,
    bf16); ``offsets [B + 1]`` bounds the sequences, none longer than ``max_len``.  Returns ``[T, D]``; dropout with probability ``p``
    acts on the attention probabilities.  The caller checks ``packed_attention_supported`` first."""
    return _PackedAttention.apply(qkv.contiguous(), offsets.to(torch.int64).contiguous(), int(num_heads), int(max_len), float(p))


# --------------------------------------------------------------------------------------
# norm and rotation of queries and keys
# --------------------------------------------------------------------------------------
ROTARY_MAX_HEAD_DIM = 256  # widest head of the kernel
_ROTARY_TYPES = (torch.bfloat16, torch.float16, torch.float32)


def rotary_inv_freq(rotary_dim: int, base: float = 10000.0, device: Optional[torch.device] = None) -> torch.Tensor:
    """The usual frequencies ``base ** (-2 j / rotary_dim)``, ``j < rotary_dim / 2``, in fp64."""
    if rotary_dim < 2 or rotary_dim % 2 or not base > 0:
        raise ValueError(f"rotary_inv_freq: a positive even dimension and a positive base, got {rotary_dim} and {base}")
    return base ** (torch.arange(rotary_dim // 2, dtype=torch.float64, device=device) * (-2.0 / rotary_dim))


def _has_tangent(*tensors: Optional[torch.Tensor]) -> bool:
    """Whether one of the tensors carries a forward-mode tangent."""
    return fwAD._current_level >= 0 and any(t is not None and fwAD.unpack_dual(t).tangent is not None for t in tensors)


def _qk_norm_rotary_plain(qkv, positions, inv_freq, q_weight, k_weight, cfg):
    """Oracle / fallback in plain torch: fp32 (fp64 for fp64 ``qkv``) with fp64 angles, one rounding at the end."""
    sections, heads, kv_heads, eps, norm, interleaved = cfg
    T, half = qkv.shape[0], inv_freq.shape[0]
    dim = qkv.shape[1] // (heads + 2 * kv_heads)
    x = qkv.to(torch.float64 if qkv.dtype == torch.float64 else torch.float32).reshape(T, heads + 2 * kv_heads, dim)
    place = [a for a, n in enumerate(sections) for _ in range(n)]
    angle = (positions.double()[place] * inv_freq.unsqueeze(1)).t().unsqueeze(1)  # [T, 1, R / 2]
    cos, sin = angle.cos().to(x.dtype), angle.sin().to(x.dtype)
    y = x[:, :heads + kv_heads]
    if norm:
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + eps)
    parts = [p if w is None else p * w.to(p.dtype) for p, w in ((y[:, :heads], q_weight), (y[:, heads:], k_weight))]
    y = torch.cat(parts, 1)
    rot, rest = y[..., :2 * half], y[..., 2 * half:]
    a, b = (rot[..., 0::2], rot[..., 1::2]) if interleaved else (rot[..., :half], rot[..., half:])
    u, v = a * cos - b * sin, a * sin + b * cos
    rot = torch.stack([u, v], -1).flatten(-2) if interleaved else torch.cat([u, v], -1)
    return torch.cat([torch.cat([rot, rest], -1), x[:, heads + kv_heads:]], 1).reshape(qkv.shape).to(qkv.dtype)


def qk_norm_rotary(qkv: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, num_heads: int, num_kv_heads: Optional[int] = None,
                   q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
                   sections: Optional[Sequence[int]] = None, interleaved: bool = False, norm: bool = True) -> torch.Tensor:
    """Queries and keys of the packed ``qkv [T, (num_heads + 2 * num_kv_heads) * head_dim]`` (``q | k | v`` along the columns) with every head
    divided by its root mean square (``norm``), scaled by ``q_weight`` / ``k_weight [head_dim]`` and turned by its token's position; ``v``
    unchanged.  Returns a new tensor of the same shape and type; with equal head counts, heads of 64 and bf16 it is what :func:`packed_attention`
    takes (shared key heads are for an attention of the caller's).

    The first ``2 * len(inv_freq)`` values of a head are turned, pair ``j`` by ``positions[t] * inv_freq[j]`` (:func:`rotary_inv_freq`; the
    angle is formed in fp64): value ``j`` with value ``j + len(inv_freq)``, or neighbours ``2 j, 2 j + 1`` with ``interleaved``.  With several
    axes ``positions`` is ``[axes, T]`` and ``sections`` says how many of the frequencies, in order, take their position from each axis.
    Positions are int32 or int64, below ``2 ** 53`` in magnitude.

    Gradients reach ``qkv`` and the weights.  CUDA tensors in bf16, fp16 or fp32 with a head dimension that is a multiple of 8 up to 256
    run in one kernel; others, and calls that carry forward-mode tangents, in plain torch."""
    kv_heads = num_heads if num_kv_heads is None else num_kv_heads
    sections = [inv_freq.shape[0] if inv_freq.dim() else 0] if sections is None else [int(n) for n in sections]
    if qkv.is_cuda and qkv.dtype in _ROTARY_TYPES and qkv.dim() == 2 and num_heads + 2 * kv_heads > 0 and not _has_tangent(qkv, q_weight, k_weight):
        dim = qkv.shape[1] // (num_heads + 2 * kv_heads)
        if dim % 8 == 0 and dim <= ROTARY_MAX_HEAD_DIM and _ext.use_cuda_kernel(qkv, "qk_norm_rotary"):  # arguments are checked there
            return torch.ops.trb200.qk_norm_rotary(qkv, positions, inv_freq, q_weight, k_weight, sections, num_heads, kv_heads, eps, norm, interleaved)
    if num_heads < 1 or kv_heads < 1 or qkv.dim() != 2 or qkv.shape[1] == 0 or qkv.shape[1] % (num_heads + 2 * kv_heads):
        raise ValueError(f"qk_norm_rotary: qkv is [T, (heads + 2 kv_heads) * head_dim], got {tuple(qkv.shape)} for {num_heads} and {kv_heads} heads")
    T, dim = qkv.shape[0], qkv.shape[1] // (num_heads + 2 * kv_heads)
    if not qkv.is_floating_point():
        raise ValueError(f"qk_norm_rotary: qkv is a floating-point tensor, got {qkv.dtype}")
    if inv_freq.dim() != 1 or not inv_freq.is_floating_point() or not 1 <= inv_freq.shape[0] <= dim // 2:
        raise ValueError(f"qk_norm_rotary: inv_freq holds 1 to head_dim / 2 = {dim // 2} frequencies, got {inv_freq.dtype} {tuple(inv_freq.shape)}")
    if positions.dtype not in (torch.int64, torch.int32) or tuple(positions.shape) not in ({(T,), (1, T)} if len(sections) == 1 else {(len(sections), T)}):
        raise ValueError(f"qk_norm_rotary: positions is an int32 or int64 [T] or [axes, T], got {positions.dtype} {tuple(positions.shape)} for {T} tokens and "
                         f"{len(sections)} axes")
    if not 1 <= len(sections) <= 8 or min(sections) < 0 or sum(sections) != inv_freq.shape[0]:
        raise ValueError(f"qk_norm_rotary: up to 8 sections that add up to the {inv_freq.shape[0]} frequencies, got {sections}")
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None and (w.shape != (dim,) or not w.is_floating_point()):
            raise ValueError(f"qk_norm_rotary: {name} is [head_dim] = [{dim}], got {w.dtype} {tuple(w.shape)}")
    for name, t in (("positions", positions), ("inv_freq", inv_freq), ("q_weight", q_weight), ("k_weight", k_weight)):
        if t is not None and t.device != qkv.device:
            raise ValueError(f"qk_norm_rotary: {name} is on {t.device}, qkv on {qkv.device}")
    if eps < 0:
        raise ValueError(f"qk_norm_rotary: eps is not negative, got {eps}")
    return _qk_norm_rotary_plain(qkv, positions.reshape(len(sections), T), inv_freq.detach().to(torch.float64), q_weight, k_weight,
                                 (sections, int(num_heads), int(kv_heads), float(eps), bool(norm), bool(interleaved)))


# --------------------------------------------------------------------------------------
# sampled softmax
# --------------------------------------------------------------------------------------
class _SampledSoftmaxLoss(torch.autograd.Function):
    """mean_p CE([h_p . pos_p, h_p . neg_0, ..., h_p . neg_{N-1}], class 0).  The scores ``[P, N]`` exist once, in bf16; the kernel
    that reads them for the loss overwrites them with their gradient, which the backward feeds to two GEMMs."""

    @staticmethod
    def forward(ctx, h, positive, negatives):
        from torchrec_b200.ops import dense_ops

        P, D = h.shape
        rows = (P + 7) // 8 * 8  # the weight-gradient GEMM wants a row count that is a multiple of 8: zero rows at the end
        h16 = h.new_zeros(rows, D, dtype=torch.bfloat16)
        h16[:P] = h
        n16 = negatives.to(torch.bfloat16).contiguous()
        scores = dense_ops.gemm_nt(h16, n16)  # [rows, N] bf16
        pos = (h16[:P].float() * positive.float()).sum(-1)
        loss_rows, dpos = torch.ops.trb200.sampled_ce_fwd_bwd(pos, scores, 1.0 / max(P, 1))
        if rows != P:
            scores[P:].zero_()
        ctx.save_for_backward(h16, positive, n16, scores, dpos)
        ctx.P = P
        ctx.dtypes = (h.dtype, positive.dtype, negatives.dtype)
        return loss_rows.sum() / max(P, 1)

    @staticmethod
    def backward(ctx, g):
        from torchrec_b200.ops import dense_ops

        h16, positive, n16, dscores, dpos = ctx.saved_tensors
        P = ctx.P
        dh = dpos_term = dneg = None
        if ctx.needs_input_grad[0]:
            dh = dense_ops.gemm_nt(dscores, n16.t().contiguous())[:P].float() + dpos.unsqueeze(1) * positive.float()
            dh = (dh * g).to(ctx.dtypes[0])
        if ctx.needs_input_grad[1]:
            dpos_term = (dpos.unsqueeze(1) * h16[:P].float() * g).to(ctx.dtypes[1])
        if ctx.needs_input_grad[2]:
            dneg = (dense_ops.gemm_tn(dscores, h16) * g).to(ctx.dtypes[2])
        return dh, dpos_term, dneg


def sampled_softmax_loss(h: torch.Tensor, positive: torch.Tensor, negatives: torch.Tensor) -> torch.Tensor:
    """Mean cross entropy of a sampled softmax: row ``p`` scores its own positive ``positive[p]`` (class 0) and the shared
    ``negatives [N, D]`` against ``h[p]``.  Equal to ``cross_entropy(cat([sum(h * positive, -1, keepdim), h @ negatives.T], 1), 0)``."""
    if (h.is_cuda and _ext.has_cuda_ext() and h.dim() == 2 and h.dtype in (torch.bfloat16, torch.float32) and negatives.shape[0] % 8 == 0
            and negatives.shape[0] >= 8 and h.shape[1] % 8 == 0 and h.shape[0] > 0):
        return _SampledSoftmaxLoss.apply(h, positive, negatives)
    scores = torch.cat([(h * positive.to(h.dtype)).sum(-1, keepdim=True), h @ negatives.to(h.dtype).t()], dim=1).float()
    return torch.nn.functional.cross_entropy(scores, torch.zeros(scores.shape[0], dtype=torch.long, device=scores.device))


# --------------------------------------------------------------------------------------
# softmax over the whole catalogue
# --------------------------------------------------------------------------------------
FULL_SOFTMAX_MAX_DIM = 1024  # widest row of the tensor-core kernel
_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}
_KERNEL_TYPES = (torch.bfloat16, torch.float32)


def full_softmax_error(device: torch.device) -> int:
    """Non-zero after a ``full_softmax_loss`` launch on ``device`` met a target outside ``[0, V)`` that is not ``ignore_index`` (16: the
    loss of that row is NaN, its gradient zero) or gave up waiting for its own copies (1..9: the loss and all gradients of that call are NaN).
    Reading it synchronises and resets it."""
    device = torch.device(device)
    if device.type != "cuda" or not _ext.has_cuda_ext():
        return 0
    with torch.cuda.device(device):
        return int(torch.ops.trb200.full_softmax_status())


class _OnlyOnce(torch.autograd.Function):
    """The gradients of a backward that is itself recorded (``create_graph``), with an error on the way from them to every input."""

    @staticmethod
    def forward(ctx, dh, dw, db, h, weight, bias):
        return tuple(None if x is None else x.view_as(x) for x in (dh, dw, db))

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError("the gradient of full_softmax_loss cannot be differentiated again")


class _FullSoftmaxPieces(torch.autograd.Function):
    """The same loss in plain torch, a piece of the rows at a time (never the whole ``[P, V]`` scores), recomputed in the backward:
    CPU tensors, types and widths the kernel does not take, and the oracle of the small tests."""

    PIECE = 1 << 26  # scores held at a time

    @staticmethod
    def _scores(h, weight, bias, keep, lo, hi, acc):
        x = torch.where(keep[lo:hi, None], h[lo:hi].to(acc), 0)
        z = x @ weight.to(acc).t()
        return x, z if bias is None else z + bias.to(acc)

    @staticmethod
    def forward(ctx, h, weight, bias, targets, ignore_index: int, reduction: int):
        P, V = h.shape[0], weight.shape[0]
        acc = torch.float64 if h.dtype == torch.float64 else torch.float32
        keep = targets != ignore_index
        bad = keep & ((targets < 0) | (targets >= V))
        if not targets.is_cuda and bool(bad.any()):
            raise IndexError(f"full_softmax_loss: target {int(targets[bad][0])} is out of bounds for {V} classes")
        if targets.is_cuda and _ext.has_cuda_ext():
            torch.ops.trb200.full_softmax_check_targets(targets, V, ignore_index)
        keep = keep & ~bad
        t = torch.where(keep, targets, 0)
        step = max(1, _FullSoftmaxPieces.PIECE // V)
        # the log sum is kept as a score of the row and the rest: next to a mask of -1e9 their sum would lose log V; the other classes'
        # distance to the target gives 1 - p of a confident row, which is no difference of two rounded numbers then
        top, lse, gap, rows = (h.new_zeros(P, dtype=acc) for _ in range(4))
        with torch.autocast(h.device.type, enabled=False):  # the products in `acc` in either direction, whatever region the call stands in
            for lo in range(0, P, step):
                hi = min(P, lo + step)
                _, z = _FullSoftmaxPieces._scores(h, weight, bias, keep, lo, hi, acc)
                m = z.amax(1, keepdim=True)
                m = torch.where(m == float("-inf"), 0, m)
                z -= m
                zt = z.gather(1, t[lo:hi, None]).squeeze(1)
                others = torch.logsumexp(z.scatter_(1, t[lo:hi, None], float("-inf")), 1)
                top[lo:hi], lse[lo:hi], gap[lo:hi] = m.squeeze(1), torch.logaddexp(others, zt), others - zt
                rows[lo:hi] = torch.logaddexp(gap[lo:hi], torch.zeros_like(zt))
        rows = torch.where(keep, rows, 0).masked_fill(bad, float("nan"))
        count = keep.sum().clamp(min=1)
        ctx.save_for_backward(h, weight, bias, t, keep, top, lse, gap, count)
        ctx.cfg = (reduction, acc)
        return rows if reduction == 0 else rows.sum() if reduction == 2 else rows.sum() / count

    @staticmethod
    def backward(ctx, g):
        with torch.no_grad():
            grads = _FullSoftmaxPieces._gradients(ctx, g)
        if torch.is_grad_enabled():
            grads = _OnlyOnce.apply(*grads, *ctx.saved_tensors[:3])
        return grads[0], grads[1], grads[2], None, None, None

    @staticmethod
    def _gradients(ctx, g):
        h, weight, bias, t, keep, top, lse, gap, count = ctx.saved_tensors
        reduction, acc = ctx.cfg
        P, V = h.shape[0], weight.shape[0]
        scale = torch.where(keep, (g / count if reduction == 1 else g).to(acc), 0)
        step = max(1, _FullSoftmaxPieces.PIECE // V)
        w = weight.to(acc)
        dh = torch.zeros_like(h)
        dw = weight.new_zeros(weight.shape, dtype=acc)
        db = None if bias is None else bias.new_zeros(bias.shape, dtype=acc)
        with torch.autocast(h.device.type, enabled=False):
            for lo in range(0, P, step):
                hi = min(P, lo + step)
                x, z = _FullSoftmaxPieces._scores(h, weight, bias, keep, lo, hi, acc)
                p = torch.exp((z - top[lo:hi, None]) - lse[lo:hi, None])
                p.scatter_(1, t[lo:hi, None], -torch.sigmoid(gap[lo:hi, None]))
                p = torch.where(keep[lo:hi, None], p * scale[lo:hi, None], 0)
                dh[lo:hi] = (p @ w).to(h.dtype)
                dw += p.t() @ x
                if db is not None:
                    db += p.sum(0)
        return dh, dw.to(weight.dtype), None if db is None else db.to(bias.dtype)


def full_softmax_loss(h: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, bias: Optional[torch.Tensor] = None, ignore_index: int = -100,
                      reduction: str = "mean") -> torch.Tensor:
    """Cross entropy of ``h [P, D]`` against all ``V`` rows of ``weight``: ``cross_entropy(h @ weight.T + bias, targets)`` in fp32, with
    gradients of ``h``, ``weight`` and ``bias``, without ever holding the ``[P, V]`` scores.

    ``targets [P]`` are class indices; a row whose target is ``ignore_index`` counts nowhere, whatever its ``h`` holds.  ``bias [V]`` may
    hold ``-inf`` for classes that are out of the race.  ``reduction`` is ``"mean"`` (over the rows that are not ignored; 0 when there is
    none), ``"sum"`` or ``"none"`` (``[P]``, 0 at ignored rows).

    On CUDA bf16 ``h`` (and fp32 ``h`` while the dense compute type is bf16, ``dense_ops.set_dense_compute_dtype``) with ``D <= 1024`` runs
    on the tensor cores with bf16 operands (the softmax terms of the gradients among them) and fp32 sums; an fp32 ``weight`` is rounded to
    bf16 for the products and gets an fp32 gradient (a parameter once per version, as in the dense layers).  Everything else is computed in fp32 (fp64 for fp64 ``h``), a piece of the rows at a time.  A target outside ``[0, V)``
    raises on the CPU; on CUDA it makes the row's loss NaN and its gradient zero, and ``full_softmax_error`` reports it.  Forward-mode
    and second derivatives are refused."""
    if reduction not in _REDUCTIONS:
        raise ValueError(f"full_softmax_loss: reduction is one of {sorted(_REDUCTIONS)}, got {reduction!r}")
    if h.is_cuda and h.dim() == 2 and h.shape[1] <= FULL_SOFTMAX_MAX_DIM and weight.dtype in _KERNEL_TYPES and (bias is None or bias.dtype in _KERNEL_TYPES):
        if (h.dtype == torch.bfloat16 or (h.dtype == torch.float32 and dense_ops.fused_dense_enabled(h))) and _ext.use_cuda_kernel(h, "full_softmax_loss"):
            # fp32 parameters go through the cache that the dense layers use: rounded once per optimizer step
            rounded = dense_ops.bf16_cache.get(weight) if weight.dtype == torch.float32 and weight.is_cuda and isinstance(weight, torch.nn.Parameter) else None
            return torch.ops.trb200.full_softmax_loss(h, weight, bias, targets, rounded, ignore_index, _REDUCTIONS[reduction])  # arguments are checked there
    if h.dim() != 2 or weight.dim() != 2 or h.shape[1] != weight.shape[1] or weight.shape[0] == 0 or h.shape[1] == 0:
        raise ValueError(f"full_softmax_loss: h [P, D] and weight [V, D] with V, D > 0, got {tuple(h.shape)} and {tuple(weight.shape)}")
    if targets.shape != h.shape[:1] or targets.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"full_softmax_loss: targets is an int32 or int64 [P], got {targets.dtype} {tuple(targets.shape)}")
    if bias is not None and bias.shape != weight.shape[:1]:
        raise ValueError(f"full_softmax_loss: bias is [V], got {tuple(bias.shape)} for {weight.shape[0]} classes")
    for name, t in (("h", h), ("weight", weight), ("bias", bias)):
        if t is not None and not t.is_floating_point():
            raise ValueError(f"full_softmax_loss: {name} is a floating-point tensor, got {t.dtype}")
    for name, t in (("weight", weight), ("targets", targets), ("bias", bias)):
        if t is not None and t.device != h.device:
            raise ValueError(f"full_softmax_loss: {name} is on {t.device}, h on {h.device}")
    return _FullSoftmaxPieces.apply(h, weight, bias, targets.to(torch.int64), int(ignore_index), _REDUCTIONS[reduction])
