"""Generation on several ranks and in several chunks: who draws, and who computes."""

from __future__ import annotations

import pytest
import torch

import hybrid_training.ops as ops
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


def test_prompts_that_have_ended_leave_the_prefill(monkeypatch) -> None:
    """One long prompt among short ones: later chunks run and read back that one alone, and every text is that of its prompt alone."""
    model = TinyTransformer(G.llama_config(), seed=4)
    gen = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, 62, (n,), generator=gen) for n in (5, 300, 128, 129, 1)]
    rows, reads = [], []
    project, read = model.blocks[0].attention.qkv.forward, ops.kv_cache_read
    monkeypatch.setattr(model.blocks[0].attention.qkv, "forward", lambda x: rows.append(tuple(x.shape[:2])) or project(x))
    monkeypatch.setattr(ops, "kv_cache_read", lambda pages, slots, out=None: reads.append(slots.shape[0]) or read(pages, slots, out))
    out = generate(model, prompts, 3, temperature=0.0, prefill_chunk=128)
    assert rows[:3] == [(5, 128), (2, 128), (1, 44)]
    assert reads == [128, 128, 128, 128, 256, 256]  # two layers
    for p, tokens, logprobs in zip(prompts, out.tokens, out.logprobs):
        alone = generate(model, [p], 3, temperature=0.0)
        assert torch.equal(tokens, alone.tokens[0]) and torch.allclose(logprobs, alone.logprobs[0], atol=1e-5)
