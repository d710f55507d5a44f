"""Rank functions of the generation tests."""

from __future__ import annotations

from typing import Any

from hybrid_training.config import ExperimentConfig, ModelConfig, TopologyConfig
from hybrid_training.distributed import init_distributed

PROMPTS = [[1, 2, 3, 4], [50], list(range(30))]


def llama_config(**over: Any) -> ModelConfig:
    base = dict(kind="transformer", hidden_size=32, num_layers=2, num_heads=4, num_kv_heads=2, ffn_hidden_size=48, vocab_size=62,
                max_sequence_length=320, activation="swiglu", norm="rmsnorm", position_embedding="rope", bias=False)
    base.update(over)
    return ModelConfig(**base)


def tensor_parallel_worker(rank: int, world: int) -> dict[str, Any]:
    """Greedy generation with heads, vocabulary and features over the ranks; refusals of what cannot generate."""
    from hybrid_training.errors import UnsupportedFeatureError
    from hybrid_training.models import ParallelPlan, TinyTransformer, generate
    from hybrid_training.parallel import FullyShardedDataParallel

    cfg = ExperimentConfig(backend="gloo", device="cpu", topology=TopologyConfig(tensor_parallel_size=world), model=llama_config())
    ctx = init_distributed(cfg)
    try:
        group = ctx.group("tensor")
        model = TinyTransformer(llama_config(), ParallelPlan(tensor_group=group, sequence_group=group), seed=11)
        out = generate(model, PROMPTS, 5, temperature=0.0)

        def refused(model: Any) -> str:
            try:
                generate(model, [[1]], 1)
            except UnsupportedFeatureError as e:
                return type(e).__name__
            return "nothing"

        sharded = TinyTransformer(llama_config(), seed=11)
        sharded.blocks[0] = FullyShardedDataParallel(sharded.blocks[0], group)
        split = TinyTransformer(llama_config(), ParallelPlan(tensor_group=group, sequence_group=group, sequence_parallel=True), seed=11)
        return {"tokens": [t.tolist() for t in out.tokens], "logprobs": [p.tolist() for p in out.logprobs],
                "sequence_parallel": refused(split), "fsdp": refused(sharded)}
    finally:
        ctx.shutdown()
