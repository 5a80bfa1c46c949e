"""Forward-mode derivatives of the softmax loss over the whole catalogue and of the norm and rotation of queries and keys: computed, or
refused with an error, and never dropped."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

from torchrec_b200.ops.transformer_ops import full_softmax_loss, qk_norm_rotary, rotary_inv_freq

devices = pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])


def _loss_inputs(device, dtype):
    g = torch.Generator().manual_seed(1)
    return [torch.randn(*s, generator=g).to(device, dtype) for s in ((5, 8), (9, 8), (9,))] + [torch.randint(0, 9, (5,), generator=g).to(device)]


def _rotary_inputs(device, dtype):
    g = torch.Generator().manual_seed(2)
    return [torch.randn(6, 3 * 16, generator=g).to(device, dtype), torch.rand(16, generator=g).to(device), torch.rand(16, generator=g).to(device),
            torch.arange(6, device=device), rotary_inv_freq(16, device=device)]


@devices
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("requires_grad", [False, True])
def test_forward_mode_of_the_loss_is_refused(device, dtype, which, requires_grad):
    *x, t = _loss_inputs(device, dtype)
    with fwAD.dual_level():
        x[which] = fwAD.make_dual(x[which].requires_grad_(requires_grad), torch.ones_like(x[which]))
        with pytest.raises((RuntimeError, NotImplementedError), match="[Ff]orward.mode|jvp"):
            full_softmax_loss(x[0], x[1], t, x[2])


@devices
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("requires_grad", [False, True])
def test_forward_mode_of_the_rotation(device, dtype, which, requires_grad):
    """The tangent is the derivative along it: against the same call in fp64 (off by the rounding of its type, and of values as large)."""
    x = _rotary_inputs(device, dtype)
    g = torch.Generator().manual_seed(3)
    tangent = torch.randn(x[which].shape, generator=g).to(x[which])

    def tangent_of(args, tan):
        with fwAD.dual_level():
            args[which] = fwAD.make_dual(args[which].requires_grad_(requires_grad), tan)
            out = qk_norm_rotary(args[0], args[3], args[4], 1, q_weight=args[1], k_weight=args[2])
            return fwAD.unpack_dual(out).tangent.detach()

    got = tangent_of(list(x), tangent)
    want = tangent_of([t.cpu().double() if t.is_floating_point() else t.cpu() for t in x], tangent.cpu().double())
    assert got is not None and got.dtype == dtype
    torch.testing.assert_close(got.cpu().double(), want, rtol=torch.finfo(dtype).eps, atol=16 * torch.finfo(torch.float32).eps * float(want.detach().abs().max()))
