"""Rank functions of the generation tests on several ranks."""

from __future__ import annotations

from typing import Any

import torch
import torch.distributed as dist

from hybrid_training.config import ExperimentConfig, TopologyConfig
from hybrid_training.distributed import init_distributed
from hybrid_training.models import ParallelPlan, TinyTransformer, generate

from .generation_workers import PROMPTS, llama_config


def _gathered(value: Any, group: Any) -> list[Any]:
    got: list[Any] = [None] * group.size
    dist.all_gather_object(got, value, group=group.process_group)
    return got


def sampling_worker(rank: int, world: int) -> dict[str, Any]:
    """Drawn tokens with generators that differ from rank to rank, without and with a stop token."""
    cfg = ExperimentConfig(backend="gloo", device="cpu", topology=TopologyConfig(tensor_parallel_size=world), model=llama_config())
    ctx = init_distributed(cfg)
    try:
        group = ctx.group("tensor")
        model = TinyTransformer(llama_config(), ParallelPlan(tensor_group=group, sequence_group=group), seed=11)
        own = generate(model, PROMPTS, 12, generator=torch.Generator().manual_seed(rank))
        texts = [[t.tolist() for t in own.tokens]]
        scores = [p.tolist() for p in own.logprobs]
        if len({tuple(map(tuple, t)) for t in _gathered(texts[0], group)}) > 1:
            return {"texts": texts, "scores": scores}  # ranks that disagree would wait for one another for good behind a stop token
        torch.manual_seed(100 + rank)
        texts.append([t.tolist() for t in generate(model, PROMPTS, 12).tokens])
        stop = texts[0][0][3]
        texts.append([t.tolist() for t in generate(model, PROMPTS, 12, stop_token=stop, generator=torch.Generator().manual_seed(rank)).tokens])
        return {"texts": texts, "scores": scores}
    finally:
        ctx.shutdown()
