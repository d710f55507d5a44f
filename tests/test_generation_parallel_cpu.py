"""Generation on several ranks and in several chunks: who draws, and who computes."""

from __future__ import annotations

import pytest
import torch

from hybrid_training.distributed import launch_workers
from hybrid_training.models import TinyTransformer, generate

from . import generation_parallel_workers as P
from . import generation_workers as G


@pytest.mark.distributed
def test_tensor_parallel_ranks_draw_the_same_tokens_whatever_their_generators() -> None:
    """The first rank's draws are everyone's: those of one process with that generator; a stop token ends all ranks together."""
    single = generate(TinyTransformer(G.llama_config(), seed=11), G.PROMPTS, 12, generator=torch.Generator().manual_seed(0))
    first, second = (r.value for r in launch_workers(P.sampling_worker, 2, timeout_seconds=300))
    assert first["texts"] == second["texts"] and len(first["texts"]) == 3
    assert first["scores"] == second["scores"]
    assert first["texts"][0] == [t.tolist() for t in single.tokens]
    for a, b in zip(first["scores"], single.logprobs):
        assert torch.allclose(torch.tensor(a), b, atol=1e-5)
    stop = first["texts"][0][0][3]
    for cut, whole in zip(first["texts"][2], first["texts"][0]):
        assert cut == (whole[: whole.index(stop) + 1] if stop in whole else whole)
