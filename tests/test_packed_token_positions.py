"""Places of packed tokens, also where the buffer holds more rows than the sequences have tokens."""
import pytest
import torch

from torchrec_b200.models.bert4rec import BERT4Rec
from torchrec_b200.modules.jagged_transformer import jagged_encoder_forward, packed_token_positions
from torchrec_b200.ops import dense_ops


@pytest.fixture(autouse=True)
def fp32_compute_type():
    """Another test of the process may have left bf16, with which fp32 tensors go to the tensor-core kernels."""
    prev = dense_ops.get_dense_compute_dtype()
    dense_ops.set_dense_compute_dtype(torch.float32)
    yield
    dense_ops.set_dense_compute_dtype(prev)


devices = pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])


@devices
@pytest.mark.parametrize("offsets,count,want", [
    ([0, 3, 3, 5], 5, [0, 1, 2, 0, 1]),
    ([0, 3, 5], 8, [0, 1, 2, 0, 1, 0, 1, 2]),  # three rows behind the last sequence
    ([0, 0, 0], 2, [0, 1]),
    ([0], 3, [0, 1, 2]),
    ([0], 0, []),
    ([0, 4], 4, [0, 1, 2, 3]),
])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_positions(offsets, count, want, dtype, device):
    assert packed_token_positions(torch.tensor(offsets, dtype=dtype, device=device), count).tolist() == want


@devices
def test_rows_behind_the_last_sequence_change_nothing(device):
    torch.manual_seed(0)
    model = BERT4Rec(50, 8, 32, nhead=2, num_layers=2, dropout=0.0, rotary=True).eval().to(device)
    x, offsets = torch.randn(16, 32, device=device), torch.tensor([0, 3, 3, 8], device=device)
    want = jagged_encoder_forward(model.encoder, x[:8], offsets, 8, rotary=model.rotary)
    got = jagged_encoder_forward(model.encoder, x, offsets, 8, rotary=model.rotary)
    assert got.shape == (16, 32)
    torch.testing.assert_close(got[:8], want, rtol=1e-4, atol=1e-5)  # products of another number of rows, fp32
