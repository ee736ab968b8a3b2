"""The example model with several descriptions of a picture: searched for with beams, and trained on."""
import importlib.util
import itertools
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


def made(example, B, seed=3):
    torch.manual_seed(0)
    model = example.Describer().cuda()
    pictures, words, lengths = example.make_pictures(B, model, torch.Generator().manual_seed(seed), "cuda")
    return model, model.tables("cuda"), pictures, words, lengths


def test_one_beam_describes(example):
    model, tables, pictures, _, _ = made(example, 5)
    lengths = torch.tensor([12, 1, 7, 12, 3], device="cuda")
    _, said = model.describe(pictures, tables, lengths)
    found, scores = model.search(pictures, tables, lengths, beams=1)
    assert torch.isfinite(scores).all()
    for b, n in enumerate(lengths.tolist()):
        assert torch.equal(found[b, 0, :n], said[b, :n])


def test_as_many_beams_as_words_find_the_best_pair(example):
    """Sixteen beams keep every first word, so that two words are searched in full."""
    model, tables, pictures, _, _ = made(example, 3)
    pairs = torch.tensor(list(itertools.product(range(model.words), repeat=2)), device="cuda")
    found, scores = model.search(pictures, tables, torch.tensor([2, 2, 1], device="cuda"), beams=16)
    with torch.no_grad():
        # every pair of every picture, behind its one picture's keys
        logits = model(pictures, pairs.repeat(3, 1), tables).double().log_softmax(-1)
    each = logits.gather(-1, pairs.repeat(3, 1).unsqueeze(-1)).squeeze(-1).view(3, -1, 2)
    for b in range(2):
        best = each[b].sum(-1).topk(16)
        # ten sums in a row in 32 bits: 1e-5 of values of order one
        assert (scores[b].double() - best.values).abs().max() < 1e-4
        assert torch.equal(found[b], pairs[best.indices])
    single = each[2, ::model.words, 0].topk(16)          # one word each
    assert torch.equal(found[2, :, 0], single.indices) and (scores[2].double() - single.values).abs().max() < 1e-4


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_descriptions_that_share_a_picture_train_as_if_each_had_its_own(example, dtype):
    model, tables, pictures, words, lengths = made(example, 2)
    each = 3
    many = torch.randint(model.words, (2 * each, model.most_tokens), generator=torch.Generator().manual_seed(5)).cuda()
    weight = torch.randn(2 * each, model.most_tokens, model.words, generator=torch.Generator().manual_seed(6)).cuda()

    def step(pictures):
        with torch.autocast("cuda", dtype, enabled=dtype != torch.float32):
            logits = model(pictures, many, tables)
        grads = torch.autograd.grad((logits.float() * weight).sum(), list(model.parameters()))
        return logits.detach(), grads
    got, want = step(pictures), step(pictures.repeat_interleave(each, 0))
    # 32 bits: about ten sums in a row; bf16: as many roundings of 2^-8, and gradients go through them twice
    near = 1e-4 if dtype == torch.float32 else 0.1
    assert (got[0] - want[0]).abs().max() < near * want[0].abs().max()
    for (name, _), a, b in zip(model.named_parameters(), got[1], want[1]):
        assert torch.isfinite(a).all() and (a - b).norm() <= near * b.norm() + 1e-6, name
