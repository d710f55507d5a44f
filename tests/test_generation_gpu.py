"""Generation on the GPU: the decoder with its paged cache against its own whole-sequence forward pass."""

from __future__ import annotations

import subprocess
import sys
from pathlib import Path

import pytest
import torch

from hybrid_training.config import ModelConfig
from hybrid_training.models import TinyTransformer, generate

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parents[1]


def _model(kind: str) -> TinyTransformer:
    if kind == "gpt2":
        cfg = ModelConfig.gpt2_124m(hidden_size=128, num_layers=2, num_heads=2, vocab_size=500, max_sequence_length=512)
    else:
        cfg = ModelConfig.llama_1b3(hidden_size=512, num_layers=2, num_heads=4, num_kv_heads=1, ffn_hidden_size=256, vocab_size=512,
                                    max_sequence_length=512)
    return TinyTransformer(cfg, seed=5, device=torch.device("cuda"), compute_dtype=torch.bfloat16)


@pytest.mark.parametrize("kind", ["gpt2", "llama"])
@pytest.mark.parametrize("cache", [torch.bfloat16, torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("chunk", [2048, 128])
def test_log_probabilities_equal_the_forward_pass(kind, cache, chunk) -> None:
    """Each drawn token's log-probability against the model run over the whole sequence.

    bf16 activations through two layers leave a few hundredths in a log-probability; an 8-bit cache adds the
    effect of its rounding (1/16 of a value at most) on one attention of several.
    """
    model = _model(kind)
    gen = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, 500, (n,), generator=gen) for n in (3, 300, 129, 1)]
    noise = torch.Generator(device="cuda").manual_seed(2)
    out = generate(model, prompts, 12, temperature=0.9, top_p=0.95, generator=noise, cache_dtype=cache, prefill_chunk=chunk, page_size=16)
    tolerance = 0.06 if cache == torch.bfloat16 else 0.15
    for prompt, tokens, logprobs in zip(prompts, out.tokens, out.logprobs):
        ids = torch.cat([prompt.cuda(), tokens])[None]
        with torch.no_grad():
            logp = torch.log_softmax(model(ids[:, :-1].contiguous()).float()[0] / 0.9, -1)[len(prompt) - 1:]
        want = logp.gather(1, tokens[:, None])[:, 0]
        assert float((want - logprobs).abs().max()) < tolerance


def test_generation_repeats() -> None:
    model = _model("llama")
    runs = [generate(model, [[1, 2, 3], [4] * 70], 20, top_k=50, generator=torch.Generator(device="cuda").manual_seed(3), cache_dtype=torch.int8)
            for _ in range(2)]
    for a, b in zip(runs[0].tokens + runs[0].logprobs, runs[1].tokens + runs[1].logprobs):
        assert torch.equal(a, b)


def test_example_runs() -> None:
    done = subprocess.run([sys.executable, str(ROOT / "examples" / "generate_text.py"), "--tiny", "--steps", "20", "--tokens", "8", "--cache", "int8"],
                          capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]
    assert "32 tokens in" in done.stdout
