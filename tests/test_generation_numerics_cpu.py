"""Sampling on the CPU path: random numbers that are none, and gradients."""

from __future__ import annotations

import math

import pytest
import torch

import hybrid_training.ops as ops
from hybrid_training.errors import UnsupportedFeatureError


def test_sampling_names_a_token_whatever_the_random_numbers() -> None:
    noise = torch.full((3, 7), math.nan)
    noise[1, 4] = 2.0
    for filters in ({}, {"temperature": 1e30}, {"min_p": 0.5}, {"top_p": 0.9, "top_k": 6}):
        token, _ = ops.sample_tokens(torch.zeros(3, 7), noise, **filters)
        assert token.tolist() == [0, 4, 0]


def test_sampling_refuses_logits_that_need_a_gradient() -> None:
    logits = torch.randn(2, 9, requires_grad=True)
    with pytest.raises(UnsupportedFeatureError):
        ops.sample_tokens(logits, torch.ones(2, 9))
    with torch.no_grad():
        token, logprob = ops.sample_tokens(logits, torch.ones(2, 9))
    assert token.shape == (2,) and not logprob.requires_grad
    ops.sample_tokens(logits.detach(), torch.ones(2, 9))
