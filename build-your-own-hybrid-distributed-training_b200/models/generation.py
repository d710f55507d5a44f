"""Text from a trained decoder: prompts into a paged cache, then one token per sequence and step.

:func:`generate` answers a batch of prompts of any lengths with a
:class:`~hybrid_training.models.TinyTransformer`.  The keys and values of every layer live in
:class:`GenerationCache`, pages of :class:`~hybrid_training.ops.KVPages` (bf16, int8 or fp8):

* the prompts run through the flash kernels, in chunks of ``prefill_chunk`` positions (which bounds the
  activations; those that have ended leave the batch); each chunk's keys and values are written to the cache, and a later chunk reads the earlier
  ones back next to its own and attends with a query window;
* each further token is embedded, projected and written for all sequences at once, attends through
  :func:`~hybrid_training.ops.paged_attention`, and the next one is drawn by
  :func:`~hybrid_training.ops.sample_tokens`.

Every step is stream-ordered; the host waits only where a stop token is asked for.  Tensor parallelism
works as in training: each rank caches its own key/value heads, and the tokens that the tensor group's
first rank draws are everyone's, whatever the other ranks' generators say.  The reference has no generation; its model recomputes whole sequences
(``src/hybrid_training/models/transformer.py:427-512``).
"""

from __future__ import annotations

from collections.abc import Callable, Sequence
from dataclasses import dataclass

import torch

from .. import ops
from ..distributed.collectives import broadcast
from ..errors import ConfigurationError, UnsupportedFeatureError, format_error
from ..ops.attention import attention_window_forward
from .transformer import TinyTransformer

__all__ = ["GenerationCache", "GenerationOutput", "generate"]

# One layer's attention: (layer index, packed QKV [B, S, W]) -> context [B, S, H * D]
Attend = Callable[[int, torch.Tensor], torch.Tensor]


@dataclass(frozen=True)
class GenerationOutput:
    """Per prompt: the tokens that followed it and their log-probabilities under the model at the sampling temperature."""

    tokens: list[torch.Tensor]
    logprobs: list[torch.Tensor]


def _to_device(x: torch.Tensor, device: torch.device) -> torch.Tensor:
    """A copy on ``device`` that the host does not wait for."""
    return x.pin_memory().to(device, non_blocking=True) if device.type == "cuda" else x.to(device)


class GenerationCache:
    """Keys and values of every layer for a batch of sequences, in pages that are handed out up front.

    ``capacities[b]`` tokens are reserved for sequence ``b``: its row of ``block_table`` lists the pages, and
    ``lengths[b]`` counts the tokens that are cached.
    """

    def __init__(self, model: TinyTransformer, capacities: Sequence[int], *, dtype: torch.dtype | None = None, page_size: int = 32,
                 device: torch.device | None = None) -> None:
        attention = model.blocks[0].attention
        if device is None:
            device = model.token_embedding.weight.device
        if dtype is None:
            dtype = torch.bfloat16 if device.type == "cuda" else model.compute_dtype or torch.float32
        counts = [-(-c // page_size) for c in capacities]
        # one page more than is handed out, so that an empty batch still has a pool
        self.layers = [ops.KVPages.allocate(sum(counts) + 1, attention.kv_heads_per_partition, page_size, attention.head_dim, dtype=dtype,
                                            device=device) for _ in model.blocks]
        table = torch.full((len(counts), max(counts, default=0)), -1, dtype=torch.int32)
        start = 0
        for b, n in enumerate(counts):
            table[b, :n] = torch.arange(start, start + n, dtype=torch.int32)
            start += n
        self.page_size = page_size
        self.block_table = _to_device(table, device)
        self.lengths = torch.zeros(len(counts), dtype=torch.int32, device=device)

    def slots(self, positions: torch.Tensor, valid: torch.Tensor, rows: torch.Tensor | None = None) -> torch.Tensor:
        """Slots ``[B, S]`` of each sequence's (or those of ``rows``) tokens at ``positions`` ``[B, S]``; -1 where ``valid`` is false."""
        table = self.block_table if rows is None else self.block_table[rows]
        page = torch.div(positions, self.page_size, rounding_mode="floor").clamp(max=max(self.block_table.shape[1] - 1, 0))
        at = torch.gather(table.long(), 1, page)
        return torch.where(valid, at * self.page_size + positions % self.page_size, -1)


def _check_model(model: TinyTransformer) -> None:
    from ..parallel.fsdp import FullyShardedDataParallel

    if not isinstance(model, TinyTransformer):
        raise ConfigurationError(format_error("models.generate", "only the decoder model generates text", expected="TinyTransformer",
                                              observed=type(model).__name__, resolution="pass the unwrapped model"))
    if model.plan.sequence_parallel:
        raise UnsupportedFeatureError(format_error("models.generate", "a sequence of one token cannot be split over ranks",
                                                   expected="a plan without sequence parallelism", observed="sequence_parallel=True",
                                                   resolution="build the model for generation without sequence parallelism"))
    if any(isinstance(m, FullyShardedDataParallel) for m in model.modules()):
        raise UnsupportedFeatureError(format_error("models.generate", "parameters sharded by FSDP are not gathered for generation",
                                                   expected="whole parameters", observed="FSDP units",
                                                   resolution="load the full state dict into a plain model"))
    if not model.config.num_layers:
        raise ConfigurationError(format_error("models.generate", "a model without layers has nothing to cache", expected=">= 1 layer",
                                              observed=0, resolution="use a model with layers"))


def _embed(model: TinyTransformer, tokens: torch.Tensor, positions: torch.Tensor) -> torch.Tensor:
    """Embedded ``tokens`` ``[B, S]``, token ``s`` of every row at ``positions[s]``."""
    if model.position_embedding is None:
        return model.token_embedding(tokens)
    rows = model.position_embedding.weight[positions]
    if model.token_embedding.group.size == 1:
        return model.token_embedding(tokens, rows)
    hidden = model.token_embedding(tokens)
    return hidden + rows[None].to(hidden.dtype)


def _run_layers(model: TinyTransformer, hidden: torch.Tensor, attend: Attend) -> torch.Tensor:
    """The model's blocks and final norm with ``attend`` in place of attention."""
    residual, delta = hidden, None
    for i, block in enumerate(model.blocks):
        if delta is None:
            h = block.input_norm(residual, out_dtype=block.compute_dtype)
        else:
            residual, h = block.input_norm(residual, delta, out_dtype=block.compute_dtype)
        a = block.attention.output(attend(i, block.attention.qkv(h)))
        residual, h = block.post_attention_norm(residual, a, out_dtype=block.compute_dtype)
        delta = block.feed_forward(h)
    return model.final_norm(residual, delta, out_dtype=model.compute_dtype)[1]


def _prefill(model: TinyTransformer, cache: GenerationCache, tokens: torch.Tensor, counts: torch.Tensor, begin: int,
             tables: tuple[torch.Tensor, torch.Tensor] | None, sequences: torch.Tensor | None) -> torch.Tensor:
    """Runs positions ``[begin, begin + S)`` of right-padded prompts ``tokens`` ``[B, S]`` of the cache's ``sequences`` (``None``: of
    all) and caches them; returns the hidden states."""
    b, s = tokens.shape
    attention = model.blocks[0].attention
    h, hkv, d = attention.heads_per_partition, attention.kv_heads_per_partition, attention.head_dim
    positions = torch.arange(begin, begin + s, device=tokens.device)
    slots = cache.slots(positions.expand(b, s), positions[None] < counts[:, None], sequences).reshape(-1)
    before = torch.arange(begin, device=tokens.device)
    earlier = cache.slots(before.expand(b, begin), before[None] < counts[:, None], sequences).reshape(-1)
    if tables is not None:
        cos, sin = (t[begin:begin + s].contiguous() for t in tables)

    def attend(layer: int, qkv: torch.Tensor) -> torch.Tensor:
        if tables is not None:
            qkv = ops.apply_rope(qkv, cos, sin, h, hkv, d)
        rows = qkv.reshape(b * s, h + 2 * hkv, d)
        ops.kv_cache_write(cache.layers[layer], rows[:, h:h + hkv], rows[:, h + hkv:], slots)
        if begin == 0:
            return ops.attention(qkv, h, hkv, d)
        # the cached positions next to this chunk's, in the packed layout that the flash kernels read
        full = torch.zeros(b, begin + s, qkv.shape[-1], dtype=qkv.dtype, device=qkv.device)
        full[:, begin:] = qkv
        heads = full.view(b, begin + s, h + 2 * hkv, d)
        for i in range(b):
            ops.kv_cache_read(cache.layers[layer], earlier[i * begin:(i + 1) * begin], (heads[i, :begin, h:h + hkv], heads[i, :begin, h + hkv:]))
        if qkv.is_cuda:
            return attention_window_forward(full, h, hkv, d, begin, s, True)[0][:, begin:]
        return ops.attention(full, h, hkv, d)[:, begin:]

    return _run_layers(model, _embed(model, tokens, positions), attend)


def _decode(model: TinyTransformer, cache: GenerationCache, tokens: torch.Tensor, active: torch.Tensor, tables: tuple[torch.Tensor, torch.Tensor] | None) -> torch.Tensor:
    """Feeds one token ``tokens`` ``[B]`` to every active sequence; returns the hidden states ``[B, hidden]``."""
    attention = model.blocks[0].attention
    h, hkv, d = attention.heads_per_partition, attention.kv_heads_per_partition, attention.head_dim
    positions = cache.lengths.long()
    slots = cache.slots(positions[:, None], active[:, None])[:, 0]
    cache.lengths += active.to(torch.int32)
    if tables is not None:
        cos, sin = (t[positions] for t in tables)

    def attend(layer: int, qkv: torch.Tensor) -> torch.Tensor:
        # the batch lies along the sequence dimension, so the rotation's tables have a row per sequence
        if tables is not None:
            qkv = ops.apply_rope(qkv, cos, sin, h, hkv, d)
        rows = qkv[0].reshape(-1, h + 2 * hkv, d)
        ops.kv_cache_write(cache.layers[layer], rows[:, h:h + hkv], rows[:, h + hkv:], slots)
        return ops.paged_attention(rows[:, :h], cache.layers[layer], cache.block_table, cache.lengths).reshape(1, -1, h * d)

    return _run_layers(model, _embed(model, tokens[None], positions), attend)[0]


def _agree(token: torch.Tensor, logprob: torch.Tensor, model: TinyTransformer) -> tuple[torch.Tensor, torch.Tensor]:
    """The first tensor rank's draws on every rank: one token that differed would mix two texts in every later step."""
    group = model.plan.tensor_group
    if group.size == 1:
        return token, logprob
    both = torch.stack((token, logprob.view(torch.int32).long()))
    broadcast(both, group).wait()
    return both[0], both[1].int().view(torch.float32)


@torch.no_grad()
def generate(model: TinyTransformer, prompts: Sequence[Sequence[int] | torch.Tensor], max_new_tokens: int, *,
             temperature: float | torch.Tensor = 1.0, top_k: int | torch.Tensor = 0, top_p: float | torch.Tensor = 1.0,
             min_p: float | torch.Tensor = 0.0, generator: torch.Generator | None = None, stop_token: int | None = None,
             cache_dtype: torch.dtype | None = None, page_size: int = 32, prefill_chunk: int = 2048) -> GenerationOutput:
    """``max_new_tokens`` tokens after each of ``prompts`` (token ids), fewer where ``stop_token`` comes first (it is kept).

    ``temperature``, ``top_k``, ``top_p`` and ``min_p`` are those of :func:`~hybrid_training.ops.sample_tokens`, numbers or one value
    per prompt; ``generator`` (on the model's device) makes a run repeatable (with tensor parallelism the first rank's).  ``cache_dtype`` is ``torch.bfloat16`` (default on CUDA),
    ``torch.int8`` or ``torch.float8_e4m3fn``.  ``prefill_chunk`` is a multiple of 128.
    """
    _check_model(model)
    device = model.token_embedding.weight.device
    ids = [torch.as_tensor(p, dtype=torch.int64).reshape(-1) for p in prompts]
    counts = [int(p.numel()) for p in ids]
    if max_new_tokens < 1 or prefill_chunk < 128 or prefill_chunk % 128:
        raise ConfigurationError(format_error("models.generate", "max_new_tokens or prefill_chunk is out of range",
                                              expected=">= 1 token, chunks of a multiple of 128", observed=(max_new_tokens, prefill_chunk),
                                              resolution="choose values in range"))
    if not ids or min(counts) < 1 or max(counts) + max_new_tokens > model.config.max_sequence_length:
        raise ConfigurationError(format_error(
            "models.generate", "a prompt is empty or leaves no room for the answer",
            expected=f"1 to {model.config.max_sequence_length - max_new_tokens} tokens", observed=counts,
            resolution="shorten the prompt or the answer, or raise max_sequence_length"))
    attention = model.blocks[0].attention
    longest = max(counts) + max_new_tokens
    tables = None
    if attention.rope_theta is not None:
        tables = ops.rope_tables(longest, attention.head_dim, float(attention.rope_theta), device)
    cache = GenerationCache(model, [n + max_new_tokens for n in counts], dtype=cache_dtype, page_size=page_size, device=device)
    batch = len(ids)
    prompt = torch.zeros(batch, max(counts), dtype=torch.int64)
    for b, p in enumerate(ids):
        prompt[b, :counts[b]] = p
    prompt = _to_device(prompt, device)
    length = _to_device(torch.tensor(counts), device)

    # hidden state of every prompt's last token, from the chunk that it falls into
    ends, order = [], []
    for begin in range(0, max(counts), prefill_chunk):
        mine = [b for b in range(batch) if counts[b] > begin]
        sequences = None if len(mine) == batch else _to_device(torch.tensor(mine), device)
        chunk, of = (prompt, length) if sequences is None else (prompt[sequences], length[sequences])
        hidden = _prefill(model, cache, chunk[:, begin:begin + prefill_chunk].contiguous(), of, begin, tables, sequences)
        ending = [i for i, b in enumerate(mine) if counts[b] <= begin + prefill_chunk]
        if ending:
            order += [mine[i] for i in ending]
            at = torch.tensor([[i, counts[mine[i]] - 1 - begin] for i in ending])
            ends.append(hidden[tuple(_to_device(at, device).T)])
    last = torch.cat(ends)[_to_device(torch.tensor(order).argsort(), device)]
    cache.lengths.copy_(length)

    active = torch.ones(batch, dtype=torch.bool, device=device)
    tokens, logprobs, kept = [], [], []  # kept: with a stop token, who had not met it yet
    for step in range(max_new_tokens):
        logits = model.output_projection(last)
        noise = torch.empty(logits.shape, dtype=torch.float32, device=device).exponential_(generator=generator)
        token, logprob = _agree(*ops.sample_tokens(logits, noise, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p), model)
        tokens.append(token)
        logprobs.append(logprob)
        if stop_token is not None:
            kept.append(active)
            active = active & (token != stop_token)
            if not bool(active.any()):
                break
        if step + 1 < max_new_tokens:
            # a sequence that has stopped stays in the batch; what it computes is not kept
            last = _decode(model, cache, token.clamp(min=0), active, tables)
    keep = torch.stack(kept).sum(0).tolist() if kept else [max_new_tokens] * batch
    rows, scores = torch.stack(tokens, 1), torch.stack(logprobs, 1)
    return GenerationOutput([rows[b, :n] for b, n in enumerate(keep)], [scores[b, :n] for b, n in enumerate(keep)])
