"""Train a GPT-2-124M-shape decoder for a few steps on a repeating sequence of tokens, then let it go on.

Shows the generation path: prompts of unequal lengths into a paged key/value cache (bf16, int8 or fp8), one token
per sequence and step with paged attention, and sampling with temperature, top-k, top-p and min-p.  Runs in one
process on a GPU or, with ``--tiny``, in seconds on a CPU.

Run, e.g.: `python examples/generate_text.py --cache int8 --top-p 0.9`
"""

from __future__ import annotations

import argparse
import sys
import time
from pathlib import Path

import torch

ROOT = Path(__file__).resolve().parent.parent
if str(ROOT) not in sys.path:
    sys.path.insert(0, str(ROOT))

from hybrid_training.config import ModelConfig  # noqa: E402
from hybrid_training.models import TinyTransformer, generate  # noqa: E402

CACHES = {"default": None, "bf16": torch.bfloat16, "int8": torch.int8, "fp8": torch.float8_e4m3fn}


def main() -> None:
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.ArgumentDefaultsHelpFormatter)
    p.add_argument("--tiny", action="store_true", help="a small model (also on CPU)")
    p.add_argument("--steps", type=int, default=60, help="training steps before generating")
    p.add_argument("--tokens", type=int, default=32, help="tokens to generate per prompt")
    p.add_argument("--batch", type=int, default=4, help="number of prompts")
    p.add_argument("--cache", choices=CACHES, default="default", help="type of the key/value cache")
    p.add_argument("--temperature", type=float, default=0.8)
    p.add_argument("--top-k", type=int, default=0)
    p.add_argument("--top-p", type=float, default=0.95)
    p.add_argument("--min-p", type=float, default=0.0)
    p.add_argument("--seed", type=int, default=0)
    args = p.parse_args()

    device = torch.device("cuda", 0) if torch.cuda.is_available() else torch.device("cpu")
    shape = dict(hidden_size=128, num_layers=2, num_heads=2, vocab_size=512, max_sequence_length=256) if args.tiny else {}
    config = ModelConfig.gpt2_124m(**shape)
    torch.manual_seed(args.seed)
    model = TinyTransformer(config, device=device, compute_dtype=torch.bfloat16 if device.type == "cuda" else None)

    # a cycle of 23 tokens, started anywhere
    cycle = torch.randperm(config.vocab_size, generator=torch.Generator().manual_seed(7))[:23]

    def sequence(start: int, length: int) -> torch.Tensor:
        return cycle[(torch.arange(length) + start) % len(cycle)]

    optimizer = torch.optim.AdamW(model.parameters(), lr=1e-3 if args.tiny else 3e-4)
    for step in range(args.steps):
        batch = torch.stack([sequence(step * 8 + i, 65) for i in range(8)]).to(device)
        loss = model(batch[:, :-1].contiguous(), targets=batch[:, 1:].contiguous())
        loss.backward()
        optimizer.step()
        optimizer.zero_grad(set_to_none=True)
    if args.steps:
        print(f"loss after {args.steps} steps: {float(loss.detach()):.4f}")

    prompts = [sequence(3 * i, 5 + 7 * i) for i in range(args.batch)]
    generator = torch.Generator(device=device).manual_seed(args.seed)
    begin = time.perf_counter()
    answer = generate(model, prompts, args.tokens, temperature=args.temperature, top_k=args.top_k, top_p=args.top_p, min_p=args.min_p,
                      generator=generator, cache_dtype=CACHES[args.cache])
    right = 0
    for i, tokens in enumerate(answer.tokens):
        expected = sequence(3 * i + len(prompts[i]), args.tokens)
        right += int((tokens.cpu() == expected).sum())
        print(f"prompt {i} ({len(prompts[i])} tokens) -> {tokens.tolist()}  mean log-probability {float(answer.logprobs[i].mean()):.3f}")
    seconds = time.perf_counter() - begin
    print(f"{args.batch * args.tokens} tokens in {seconds:.2f} s, {right} of them the cycle's")


if __name__ == "__main__":
    main()
