"""The oracle of top alternatives and distillation against values computed by hand."""
import math

import pytest
import torch

import oracle as O
from oracle.topk import order_of_alternatives

INF, NAN = math.inf, math.nan


def test_order_of_alternatives():
    z = torch.tensor([[1.0, 3.0, 3.0, -0.0, 0.0, -INF], [NAN, -INF, 2.0, NAN, -INF, 2.0]], dtype=torch.float64)
    assert order_of_alternatives(z, 6).tolist() == [[1, 2, 0, 3, 4, 5], [2, 5, 1, 4, 0, 3]]


def test_logprobs_entropy_and_alternatives_of_known_probabilities():
    q = torch.tensor([[0.5, 0.125, 0.25, 0.125], [0.5, 0.0, 0.5, 0.0]], dtype=torch.float64)
    labels = torch.tensor([3, -100])
    lp, ent, top, index = O.topk_logprobs(2 * q.log() + 1.25, labels, 3, 2.0)
    assert torch.allclose(lp, torch.tensor([math.log(0.125), 0.0], dtype=torch.float64))
    assert torch.allclose(ent, torch.tensor([1.75 * math.log(2), math.log(2)], dtype=torch.float64))
    assert index.tolist() == [[0, 2, 1], [0, 2, 1]]
    assert torch.allclose(top, torch.tensor([[0.5, 0.25, 0.125], [0.5, 0.5, 0.0]], dtype=torch.float64).log())


@pytest.mark.parametrize("kind", ["forward_kl", "reverse_kl", "jsd"])
def test_divergences_of_known_probabilities(kind):
    q = torch.tensor([[0.5, 0.125, 0.25, 0.125]], dtype=torch.float64)
    t = torch.tensor([[0.25, 0.5, 1.0, 1.0, 0.0]], dtype=torch.float64).log()
    index = torch.tensor([[0, 2, -1, 4, 1]])   # two entries count: p = (1/4, 1/2) against q = (1/2, 1/4)
    m = (0.3 * 0.25 + 0.7 * 0.5, 0.3 * 0.5 + 0.7 * 0.25)
    want = {"forward_kl": 0.25 * math.log(0.25 / 0.5) + 0.5 * math.log(0.5 / 0.25),
            "reverse_kl": 0.5 * math.log(0.5 / 0.25) + 0.25 * math.log(0.25 / 0.5),
            "jsd": 0.3 * (0.25 * math.log(0.25 / m[0]) + 0.5 * math.log(0.5 / m[1]))
            + 0.7 * (0.5 * math.log(0.5 / m[0]) + 0.25 * math.log(0.25 / m[1]))}[kind]
    got = O.topk_distillation(q.log(), t, index, kind, 0.3)
    assert torch.allclose(got, torch.tensor([want], dtype=torch.float64))
    assert O.topk_distillation(q.log(), t, torch.full_like(index, -1), kind, 0.3).item() == 0.0
