"""The example model: it trains, and token by token it says what it says of whole sequences."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "grid_transformer.py")
    spec = importlib.util.spec_from_file_location("grid_transformer", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_example_learns(example, dtype):
    torch.manual_seed(0)
    model = example.Describer().cuda()
    losses = example.train(model, 80, dtype=dtype)
    # words are uniform: knowing nothing is worth ln 16 = 2.77
    assert all(x == x for x in losses)
    assert sum(losses[-10:]) / 10 < min(2.6, sum(losses[:10]) / 10)
    for name, p in model.named_parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all(), name


def test_one_token_at_a_time_is_the_whole_sequence(example):
    """In 32 bits: a few hundred terms a sum and about ten sums in a row keep relative errors below 1e-5 of values of order one."""
    torch.manual_seed(0)
    model = example.Describer().cuda()
    tables = model.tables("cuda")
    pictures, words, _ = example.make_pictures(5, model, torch.Generator().manual_seed(3), "cuda")
    lengths = torch.tensor([12, 1, 7, 12, 3], device="cuda")
    with torch.no_grad():
        whole = model(pictures, words, tables)
    got, said = model.describe(pictures, tables, lengths, words)
    assert torch.equal(said, words)
    for b, n in enumerate(lengths.tolist()):
        assert (got[b, :n] - whole[b, :n]).abs().max() < 1e-4, b
