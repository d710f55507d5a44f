"""What the host does while text is generated on a GPU."""

from __future__ import annotations

import pytest
import torch

from hybrid_training.config import ModelConfig
from hybrid_training.models import TinyTransformer, generate

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("stop_token", [None, 3])
def test_the_host_waits_only_for_stop_tokens(stop_token) -> None:
    """The whole generation is queued behind what the stream has to do, prompts of several chunks and filters included."""
    cfg = ModelConfig.gpt2_124m(hidden_size=128, num_layers=2, num_heads=2, vocab_size=500, max_sequence_length=512)
    model = TinyTransformer(cfg, seed=5, device=torch.device("cuda"), compute_dtype=torch.bfloat16)
    prompts = [list(range(n)) for n in (3, 300, 129)]
    run = lambda: generate(model, prompts, 6, top_k=40, top_p=0.9, cache_dtype=torch.int8, prefill_chunk=128, stop_token=stop_token,  # noqa: E731
                           generator=torch.Generator(device="cuda").manual_seed(1))
    first = run()
    torch.cuda.set_sync_debug_mode("error")
    try:
        if stop_token is None:
            again = run()
        else:
            with pytest.raises(RuntimeError, match="synchroniz"):
                run()
    finally:
        torch.cuda.set_sync_debug_mode("default")
    if stop_token is None:
        assert all(torch.equal(a, b) for a, b in zip(first.tokens + first.logprobs, again.tokens + again.logprobs))
