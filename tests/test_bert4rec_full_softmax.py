"""BERT4Rec with the softmax loss over the whole vocabulary and with normalised, position-rotated queries and keys."""
import os
import subprocess
import sys

import pytest
import torch

from torchrec_b200.models.bert4rec import BERT4Rec, BERT4RecSampled
from torchrec_b200.modules.jagged_transformer import QKNormRotary, jagged_encoder_forward, packed_token_positions
from torchrec_b200.ops import dense_ops
from torchrec_b200.sparse.jagged_tensor import KeyedJaggedTensor


def _batch(B, max_len, vocab, count, seed=3):
    g = torch.Generator().manual_seed(seed)
    lengths = torch.randint(1, max_len + 1, (B,), generator=g)
    lengths[1] = max_len
    items = torch.randint(1, vocab - 1, (int(lengths.sum()),), generator=g)
    off = torch.cat([torch.zeros(1, dtype=torch.long), lengths.cumsum(0)])
    row = torch.repeat_interleave(torch.arange(B), lengths)
    col = torch.arange(items.numel()) - off[:-1][row]
    sel = torch.randperm(items.numel(), generator=g)[:count]
    return KeyedJaggedTensor(keys=["item"], values=items, lengths=lengths, stride=B), (row * max_len + col)[sel], items[sel], (items, lengths)


@pytest.mark.parametrize("rotary", [False, True])
def test_full_loss_is_the_cross_entropy_of_the_logits(rotary):
    torch.manual_seed(0)
    model = BERT4Rec(200, 12, 32, nhead=2, num_layers=2, dropout=0.0, rotary=rotary)
    kjt, pos, targets, _ = _batch(7, 12, 200, 15)
    targets[4] = -100
    loss = model(kjt, pos, targets)
    loss.backward()
    got = {n: p.grad.clone() for n, p in model.named_parameters()}
    model.zero_grad()
    logits = model(kjt)
    assert logits.shape == (7, 12, 200)
    want = torch.nn.functional.cross_entropy(logits.reshape(-1, 200)[pos], targets)
    want.backward()
    torch.testing.assert_close(loss, want, rtol=1e-5, atol=1e-6)
    for n, p in model.named_parameters():
        torch.testing.assert_close(got[n], p.grad, rtol=1e-3, atol=1e-6, msg=n)
    assert any("rotary" in n for n in got) == rotary and any("positional" in n for n in got) != rotary


def test_rotary_module_and_positions():
    assert packed_token_positions(torch.tensor([0, 3, 3, 5]), 5).tolist() == [0, 1, 2, 0, 1]
    m = QKNormRotary(16, sections=[3, 5]).to(torch.bfloat16)
    assert m.q_weight.dtype == torch.bfloat16 and m.inv_freq.dtype == torch.float64 and float(m.inv_freq[0]) == 1.0
    assert list(m.state_dict()) == ["q_weight", "k_weight"]
    meta = QKNormRotary(16, device=torch.device("meta")).to_empty(device="cpu")
    torch.testing.assert_close(meta.inv_freq, QKNormRotary(16).inv_freq, rtol=0, atol=0)
    enc = BERT4Rec(50, 8, 32, nhead=2, num_layers=2, rotary=True)
    with pytest.raises(ValueError, match="layers"):
        jagged_encoder_forward(enc.encoder, torch.zeros(3, 32), torch.tensor([0, 3]), 8, rotary=enc.rotary[:1])


def test_order_of_the_items_matters_only_with_positions():
    """Without positions the encoder cannot tell a history from its reverse; turned queries and keys can."""
    torch.manual_seed(1)
    model = BERT4Rec(100, 6, 32, nhead=2, num_layers=1, dropout=0.0, rotary=True).eval()
    for i, items in enumerate(([5, 6, 7, 8], [8, 7, 6, 5])):
        kjt = KeyedJaggedTensor(keys=["item"], values=torch.tensor(items), lengths=torch.tensor([4]), stride=1)
        h, _ = model.encode_packed(kjt)
        first = h if i == 0 else first
    assert float((first - h.flip(0)).detach().abs().max()) > 1e-4
    model.rotary = None
    plain = [model.encode_packed(KeyedJaggedTensor(keys=["item"], values=torch.tensor(v), lengths=torch.tensor([4]), stride=1))[0] for v in ([5, 6, 7, 8], [8, 7, 6, 5])]
    torch.testing.assert_close(plain[0], plain[1].flip(0), rtol=1e-4, atol=1e-5)


def test_example_runs_with_both():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    cmd = [sys.executable, "examples/bert4rec/bert4rec_main.py", "--vocab_size", "300", "--max_len", "8", "--emb_dim", "16", "--nhead", "2", "--num_layers", "1",
           "--batch_size", "8", "--num_iterations", "2", "--full_softmax", "--rotary"]
    out = subprocess.run(cmd, cwd=root, capture_output=True, text=True, timeout=300, env=dict(os.environ, MASTER_PORT="29563", CUDA_VISIBLE_DEVICES=""))
    assert out.returncode == 0 and "iter 2" in out.stdout, out.stdout + out.stderr


@pytest.mark.gpu
def test_kernels_together_in_a_training_step():
    """Norm and rotation -> packed attention -> softmax loss over all items, bf16 on the tensor cores, against the same model in fp32
    through plain torch.  Both sides share the weights; activations of the first are rounded to bf16 some twenty times on the way,
    each by at most 2^-8 of the value, so that a gradient's direction agrees to about sqrt(20) 2^-8 = 2 % and 6 % leaves room for their
    growth through two layers."""
    from torchrec_b200.ops.transformer_ops import attention_error, full_softmax_error

    torch.manual_seed(0)
    dev = torch.device("cuda")
    model = BERT4Rec(3001, 40, 256, nhead=4, num_layers=2, dim_feedforward=512, dropout=0.0, device=dev, rotary=True)
    with torch.no_grad():
        for m in model.rotary:
            m.q_weight.uniform_(0.5, 1.5)
            m.k_weight.uniform_(0.5, 1.5)
    kjt, pos, targets, _ = _batch(33, 40, 3001, 90)
    kjt, pos, targets = kjt.to(dev), pos.to(dev), targets.to(dev)
    targets[::7] = -100

    def step():
        model.zero_grad()
        loss = model(kjt, pos, targets)
        loss.backward()
        return float(loss.detach()), {n: p.grad.detach().double().clone() for n, p in model.named_parameters()}

    want, want_g = step()  # fp32 compute type: plain torch (and the fp32 rotary kernel)
    prev = dense_ops.get_dense_compute_dtype()
    dense_ops.set_dense_compute_dtype(torch.bfloat16)
    try:
        got, got_g = step()
    finally:
        dense_ops.set_dense_compute_dtype(prev)
        dense_ops.bf16_cache.clear()
    assert abs(got - want) <= 2e-2 * want
    for n, g in want_g.items():
        off = float((got_g[n] - g).norm() / g.norm().clamp(min=1e-12))
        # gradients that are zero in exact arithmetic (the key bias moves every score of a query alike) are rounding noise on both sides
        assert off < 6e-2 or float(g.norm()) < 1e-3 * max(float(x.norm()) for x in want_g.values()), (n, off, float(g.norm()))
    assert full_softmax_error(dev) == 0 and attention_error(dev) == 0


@pytest.mark.gpu
def test_sampled_model_with_rotary_trains():
    dev = torch.device("cuda")
    torch.manual_seed(0)
    model = BERT4RecSampled(2000, 40, 256, nhead=4, num_layers=2, dim_feedforward=512, dropout=0.1, device=dev, rotary=True)
    _, pos, targets, (items, lengths) = _batch(33, 40, 2000, 50)
    kjt = BERT4RecSampled.make_input(items, lengths, targets, torch.randint(1, 1999, (64,))).to(dev)
    prev = dense_ops.get_dense_compute_dtype()
    dense_ops.set_dense_compute_dtype(torch.bfloat16)
    try:
        loss = model(kjt, pos.to(dev), loss=True)
        loss.backward()
    finally:
        dense_ops.set_dense_compute_dtype(prev)
        dense_ops.bf16_cache.clear()
    for n, p in model.named_parameters():
        assert p.grad is not None and bool(torch.isfinite(p.grad).all()), n
