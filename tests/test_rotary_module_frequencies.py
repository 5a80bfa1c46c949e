"""Frequencies of the rotary module through casts and moves: in fp64, and those that were set."""
import copy

import pytest
import torch

from torchrec_b200.modules.jagged_transformer import QKNormRotary


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_frequencies_that_were_set_stay(device):
    m = QKNormRotary(16)
    scaled = m.inv_freq / 3  # stretched to longer histories
    m.inv_freq.copy_(scaled)
    for moved in (m, copy.deepcopy(m).to(torch.bfloat16), copy.deepcopy(m).half().to(device).float()):
        assert moved.inv_freq.dtype == torch.float64 and torch.equal(moved.inv_freq.cpu(), scaled)
        assert moved.inv_freq.device == moved.q_weight.device
    m.inv_freq = scaled / 2
    assert torch.equal(m.to(device).inv_freq.cpu(), scaled / 2)


def test_frequencies_off_the_meta_device():
    m = QKNormRotary(16, rotary_dim=8, base=500.0, device=torch.device("meta"))
    assert m.inv_freq.is_meta
    assert torch.equal(m.to_empty(device="cpu").inv_freq, QKNormRotary(16, rotary_dim=8, base=500.0).inv_freq)
    assert QKNormRotary(16).to("meta").inv_freq.is_meta
