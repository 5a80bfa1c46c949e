"""Norm and rotation of queries and keys on the CPU: properties of a rotation, gradients against differences, and the refusals."""
import pytest
import torch

from torchrec_b200.ops.transformer_ops import qk_norm_rotary, rotary_inv_freq


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [False, True])
def test_gradients_against_differences(interleaved, norm):
    g = torch.Generator().manual_seed(1)
    qkv, qw, kw = (torch.randn(*s, generator=g, dtype=torch.float64).requires_grad_(True) for s in ((3, 4 * 6), (6,), (6,)))
    pos = torch.tensor([[0, 3, 7], [5, 1, 9]])
    fn = lambda x, a, b: qk_norm_rotary(x, pos, rotary_inv_freq(6), 2, 1, a, b, sections=[2, 1], interleaved=interleaved, norm=norm)  # noqa: E731
    assert torch.autograd.gradcheck(fn, (qkv, qw, kw))


@pytest.mark.parametrize("interleaved", [False, True])
def test_scores_depend_on_the_distance_alone(interleaved):
    g = torch.Generator().manual_seed(2)
    qkv = torch.randn(1, 3 * 16, generator=g, dtype=torch.float64).expand(9, -1)
    pos = torch.arange(9)
    a, b = (qk_norm_rotary(qkv, pos + shift, rotary_inv_freq(16), 1, interleaved=interleaved) for shift in (0, 10**6))
    score = [(x[:, :16] @ x[:, 16:32].t()) for x in (a, b)]
    torch.testing.assert_close(score[0], score[1], rtol=0, atol=1e-8)  # angles of a million radians are off by 1e-10
    assert torch.equal(a[:, 32:], qkv[:, 32:])
    torch.testing.assert_close(a[:, :16].square().mean(1), torch.ones(9, dtype=torch.float64), rtol=1e-4, atol=0)
    torch.testing.assert_close(a[0], torch.cat([qkv[0, :32].reshape(2, 16) / (qkv[0, :32].reshape(2, 16).square().mean(1, keepdim=True) + 1e-6).sqrt(),
                                                qkv[:1, 32:]]).flatten())


def test_values_by_hand():
    qkv = torch.tensor([[1.0, 2.0, 3.0, 4.0, 5.0, 6.0]])
    quarter = torch.tensor([torch.pi / 2], dtype=torch.float64)
    out = qk_norm_rotary(qkv, torch.tensor([1]), quarter, 1, norm=False)
    torch.testing.assert_close(out, torch.tensor([[-2.0, 1.0, -4.0, 3.0, 5.0, 6.0]]))
    out = qk_norm_rotary(qkv, torch.tensor([-1]), quarter, 1, q_weight=torch.tensor([1.0, 2.0]), norm=False)
    torch.testing.assert_close(out, torch.tensor([[4.0, -1.0, 4.0, -3.0, 5.0, 6.0]]))


def test_refusals():
    qkv, pos, inv = torch.randn(5, 3 * 8), torch.arange(5), rotary_inv_freq(8)
    for bad in (dict(num_heads=5), dict(num_heads=0), dict(num_heads=1, num_kv_heads=2)):
        with pytest.raises(ValueError, match="qkv is"):
            qk_norm_rotary(qkv, pos, inv, **bad)
    with pytest.raises(ValueError, match="qkv is"):
        qk_norm_rotary(qkv[0], pos, inv, 1)
    with pytest.raises(ValueError, match="floating"):
        qk_norm_rotary(qkv.int(), pos, inv, 1)
    for bad in (rotary_inv_freq(10), inv[:0], inv[None], inv.int()):
        with pytest.raises(ValueError, match="inv_freq"):
            qk_norm_rotary(qkv, pos, bad, 1)
    for bad in (pos[:4], pos.float(), torch.stack([pos, pos])):
        with pytest.raises(ValueError, match="positions"):
            qk_norm_rotary(qkv, bad, inv, 1)
    for bad in ([3, 2], [5, -1], [1] * 9):
        with pytest.raises(ValueError, match="sections|axes"):
            qk_norm_rotary(qkv, torch.stack([pos] * len(bad)), inv, 1, sections=bad)
    with pytest.raises(ValueError, match="q_weight"):
        qk_norm_rotary(qkv, pos, inv, 1, q_weight=torch.ones(7))
    with pytest.raises(ValueError, match="eps"):
        qk_norm_rotary(qkv, pos, inv, 1, eps=-1.0)
    with pytest.raises(ValueError, match="even"):
        rotary_inv_freq(7)
