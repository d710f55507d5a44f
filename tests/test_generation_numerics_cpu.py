"""Sampling of the CPU path where random numbers or filters are not numbers."""

from __future__ import annotations

import math

import torch

import hybrid_training.ops as ops


def test_sampling_names_a_token_whatever_the_random_numbers() -> None:
    noise = torch.full((3, 7), math.nan)
    noise[1, 4] = 2.0
    for filters in ({}, {"temperature": 1e30}, {"min_p": 0.5}, {"top_p": 0.9, "top_k": 6}):
        token, _ = ops.sample_tokens(torch.zeros(3, 7), noise, **filters)
        assert token.tolist() == [0, 4, 0]
