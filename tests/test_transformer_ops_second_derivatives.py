"""Second derivatives of the softmax loss over the whole catalogue and of the norm and rotation of queries and keys: computed, or refused with
an error, and never dropped."""
import pytest
import torch

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
def test_second_derivatives_of_the_loss_are_refused(device, dtype):
    """A gradient penalty: the upstream gradient is the constant one, and the gradient is still no constant."""
    *x, t = _loss_inputs(device, dtype)
    leaves = [v.requires_grad_(True) for v in x]
    grads = torch.autograd.grad(full_softmax_loss(leaves[0], leaves[1], t, leaves[2]), leaves, create_graph=True)
    for g in grads:
        assert g.requires_grad
        with pytest.raises(RuntimeError, match="differentiated again"):
            (g.float().square().sum() + leaves[0].float().sum()).backward(retain_graph=True)


@devices
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_second_derivatives_of_the_rotation_are_never_dropped(device, dtype):
    x = _rotary_inputs(device, dtype)
    leaves = [v.requires_grad_(True) for v in x[:3]]
    out = qk_norm_rotary(leaves[0], x[3], x[4], 1, q_weight=leaves[1], k_weight=leaves[2])
    (g,) = torch.autograd.grad(out.float().sum(), leaves[:1], create_graph=True)
    assert g.requires_grad
    if device == "cpu":  # plain torch: differentiable
        (second,) = torch.autograd.grad(g.float().square().sum(), leaves[:1])
        assert bool((second != 0).any())
    else:
        with pytest.raises(RuntimeError, match="differentiated again"):
            (g.float().square().sum() + leaves[0].float().sum()).backward()


@devices
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("which", [0, 1, 2])
def test_second_derivatives_of_the_loss_along_another_path(device, dtype, which):
    """torch.autograd.grad walks only the paths to the inputs that it is asked for: the gradient has to lie on one."""
    *x, t = _loss_inputs(device, dtype)
    leaves = [v.requires_grad_(True) for v in x]
    grads = torch.autograd.grad(full_softmax_loss(leaves[0], leaves[1], t, leaves[2]), leaves, create_graph=True)
    for g in grads:
        with pytest.raises(RuntimeError, match="differentiated again"):
            torch.autograd.grad(g.float().square().sum() + leaves[which].float().sum(), leaves[which], retain_graph=True)
    with pytest.raises(RuntimeError, match="differentiated again"):
        torch.autograd.functional.hessian(lambda v: full_softmax_loss(v, leaves[1].detach(), t), leaves[0].detach())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("which", [0, 1, 2])
def test_second_derivatives_of_the_rotation_along_another_path(dtype, which):
    x = _rotary_inputs("cuda", dtype)
    leaves = [v.requires_grad_(True) for v in x[:3]]
    out = qk_norm_rotary(leaves[0], x[3], x[4], 1, q_weight=leaves[1], k_weight=leaves[2])
    grads = torch.autograd.grad(out.float().square().sum(), leaves, create_graph=True)
    for g in grads:
        with pytest.raises(RuntimeError, match="differentiated again"):
            torch.autograd.grad(g.float().square().sum() + leaves[which].float().sum(), leaves[which], retain_graph=True)
