"""The BERT4Rec example with its options for the softmax over the whole vocabulary reaches the loss kernel on a GPU."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
# the piecewise form is taken away: a step that needs it fails
RUN = """
import runpy, sys
from torchrec_b200.ops import transformer_ops
if {kernel}:
    transformer_ops._FullSoftmaxPieces.apply = None
sys.argv = ["bert4rec_main.py"] + sys.argv[1:]
runpy.run_path("examples/bert4rec/bert4rec_main.py", run_name="__main__")
"""


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_example_in_bf16(device):
    args = ["--vocab_size", "300", "--max_len", "8", "--emb_dim", "64", "--nhead", "2", "--num_layers", "1", "--batch_size", "8", "--num_iterations", "2",
            "--full_softmax", "--rotary", "--bf16"]
    env = dict(os.environ, MASTER_PORT="29567", PYTHONPATH=ROOT)
    if device == "cpu":
        env["CUDA_VISIBLE_DEVICES"] = ""
    out = subprocess.run([sys.executable, "-c", RUN.format(kernel=device == "cuda"), *args], cwd=ROOT, capture_output=True, text=True, timeout=300, env=env)
    assert out.returncode == 0 and "iter 2" in out.stdout, out.stdout + out.stderr
    assert "nan" not in out.stdout
