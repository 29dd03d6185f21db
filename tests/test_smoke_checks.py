"""What smoke() accepts as results of routing and of the experts."""

import math

import pytest
import torch

from __graft_entry__ import check_experts, check_routing

IDS = torch.tensor([[1, 3], [0, 2]], dtype=torch.int32)
WEIGHTS = torch.tensor([[math.e / (math.e + 1), 1 / (math.e + 1)], [0.5, 0.5]])


def test_right_results_pass():
    check_routing(WEIGHTS, IDS)
    v = torch.arange(3000).remainder(29).sub(14).div(8).view(3, 1000)
    check_experts(v, v * v * torch.sigmoid(v) * 1.01)


@pytest.mark.parametrize("weights", [WEIGHTS * 0, -WEIGHTS, WEIGHTS * 0.9, WEIGHTS * 1.1, WEIGHTS.flip(1), WEIGHTS * math.nan])
def test_wrong_weights_do_not(weights):
    with pytest.raises(AssertionError):
        check_routing(weights, IDS)


def test_a_wrong_choice_does_not():
    with pytest.raises(AssertionError):
        check_routing(WEIGHTS, IDS.flip(1))


@pytest.mark.parametrize("wrong", [lambda h: h * 0, lambda h: h * 0.9, lambda h: -h, lambda h: h.flip(1), lambda h: h * math.nan])
def test_wrong_experts_do_not(wrong):
    v = torch.arange(3000).remainder(29).sub(14).div(8).view(3, 1000)
    with pytest.raises(AssertionError):
        check_experts(v, wrong(v * v * torch.sigmoid(v)))
