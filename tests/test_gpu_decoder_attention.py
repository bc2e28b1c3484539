"""The example of a decoder layer's attention half: its operators together, by calls and by graph replay."""
import importlib.util
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    path = Path(__file__).resolve().parent.parent / "examples" / "decoder_attention.py"
    spec = importlib.util.spec_from_file_location("decoder_attention", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("prompts,q_heads,kv_heads,head_dim", [((300, 17, 1), 8, 2, 128), ((40,), 4, 4, 64), ((1, 2, 1500), 12, 4, 64)])
def test_layer(cuda, example, prompts, q_heads, kv_heads, head_dim):
    """Against float32: 4 bits hold a group of normal numbers, five to six sigma wide, to a fifteenth of that over
    sqrt(12), 0.1 sigma.  In the values that is 0.1 of a single token's output (less of an average's, as the output is); in the
    keys 0.1 of a score of about one sigma, and so 0.1 of a weight.  The 8-bit roundings of the products' operands are
    0.02 to 0.03 each, four of them.  Together 0.15: twice that is not exceeded."""
    called, replayed, plain, _ = example.run(prompts, 6, 512, q_heads, kv_heads, head_dim)
    assert example.distance(called, plain) < 0.3
    for a, b in zip(called, replayed):
        assert torch.equal(a, b)
