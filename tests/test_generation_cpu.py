"""Generation on the CPU path: the paged cache, paged attention and sampling against plain statements, and the decoder end to end."""

from __future__ import annotations

import math

import pytest
import torch

import hybrid_training.ops as ops
from hybrid_training.config import ModelConfig
from hybrid_training.distributed import launch_workers
from hybrid_training.errors import ConfigurationError, UnsupportedFeatureError
from hybrid_training.models import GenerationCache, TinyTransformer, generate

from . import generation_workers as G


def _gpt2(**over) -> TinyTransformer:
    cfg = ModelConfig.gpt2_124m(**{**dict(hidden_size=32, num_layers=2, num_heads=4, vocab_size=61, max_sequence_length=320), **over})
    return TinyTransformer(cfg, seed=3)


def _llama(**over) -> TinyTransformer:
    return TinyTransformer(G.llama_config(**over), seed=4)


def _greedy_by_recomputing(model: TinyTransformer, prompt: torch.Tensor, count: int) -> tuple[list[int], list[float]]:
    ids, scores = prompt[None], []
    with torch.no_grad():
        for _ in range(count):
            logp = torch.log_softmax(model(ids)[0, -1].double(), -1)
            nxt = int(logp.argmax())
            scores.append(float(logp[nxt]))
            ids = torch.cat([ids, torch.tensor([[nxt]])], 1)
    return ids[0, len(prompt):].tolist(), scores


@pytest.mark.parametrize("build", [_gpt2, _llama])
@pytest.mark.parametrize("page_size,chunk", [(16, 2048), (64, 128)])
def test_greedy_generation_equals_recomputing(build, page_size, chunk) -> None:
    """Ragged prompts (one longer than a prefill chunk) continue as the whole-sequence forward pass says."""
    model = build()
    gen = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, 61, (n,), generator=gen) for n in (1, 17, 200, 129)]
    out = generate(model, prompts, 6, temperature=0.0, page_size=page_size, prefill_chunk=chunk)
    for p, tokens, logprobs in zip(prompts, out.tokens, out.logprobs):
        want, scores = _greedy_by_recomputing(model, p, 6)
        assert tokens.tolist() == want
        assert torch.allclose(logprobs.double(), torch.tensor(scores, dtype=torch.float64), atol=1e-5)


@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn])
def test_quantised_cache_changes_little(dtype) -> None:
    """Log-probabilities of the first drawn tokens stay within what a quantisation of a per cent or a few can move."""
    model = _llama()
    prompts = [torch.arange(n) % 61 for n in (9, 40)]
    noise = torch.Generator().manual_seed(5)
    exact = generate(model, prompts, 1, generator=noise)
    noise.manual_seed(5)
    held = generate(model, prompts, 3, generator=noise, cache_dtype=dtype)
    for a, b in zip(exact.logprobs, held.logprobs):
        assert abs(float(a[0]) - float(b[0])) < 1e-5  # the prompt's attention does not read the cache
        assert bool(torch.isfinite(b).all()) and len(b) == 3


def test_sampling_repeats_with_a_generator_and_follows_the_filters() -> None:
    model = _gpt2()
    gen = torch.Generator()
    runs = [generate(model, [[1, 2, 3], [4]], 8, temperature=0.9, top_k=torch.tensor([1, 40], dtype=torch.int32), generator=gen.manual_seed(s))
            for s in (1, 1, 2)]
    assert all(torch.equal(a, b) for a, b in zip(runs[0].tokens, runs[1].tokens))
    greedy = generate(model, [[1, 2, 3]], 8, temperature=0.0)
    assert torch.equal(runs[2].tokens[0], greedy.tokens[0])  # top_k = 1
    assert not torch.equal(runs[0].tokens[1], runs[2].tokens[1])


def test_stop_token_ends_a_sequence() -> None:
    model = _gpt2()
    free = generate(model, [[1, 2, 3], [7, 8]], 8, temperature=0.0)
    stop = int(free.tokens[0][2])
    out = generate(model, [[1, 2, 3], [7, 8]], 8, temperature=0.0, stop_token=stop)
    for a, b in zip(out.tokens, free.tokens):
        hits = (b == stop).nonzero().flatten().tolist()
        n = hits[0] + 1 if hits else 8
        assert torch.equal(a, b[:n])


def test_generation_refusals() -> None:
    model = _gpt2()
    for bad in (dict(prompts=[]), dict(prompts=[[]]), dict(prompts=[[1] * 316]), dict(max_new_tokens=0), dict(prefill_chunk=100)):
        with pytest.raises(ConfigurationError):
            generate(model, **{**dict(prompts=[[1, 2]], max_new_tokens=8), **bad})
    with pytest.raises(ConfigurationError):
        generate(torch.nn.Linear(2, 2), [[1]], 1)  # type: ignore[arg-type]


@pytest.mark.distributed
def test_sequence_parallel_plans_and_fsdp_are_refused_and_tensor_parallel_agrees() -> None:
    single = generate(TinyTransformer(G.llama_config(), seed=11), G.PROMPTS, 5, temperature=0.0)
    results = launch_workers(G.tensor_parallel_worker, 2, timeout_seconds=300)
    for r in results:
        assert r.value["tokens"] == [t.tolist() for t in single.tokens]
        for a, b in zip(r.value["logprobs"], single.logprobs):
            assert torch.allclose(torch.tensor(a), b, atol=1e-5)
        assert r.value["sequence_parallel"] == "UnsupportedFeatureError" and r.value["fsdp"] == "UnsupportedFeatureError"


def test_cache_hands_out_pages_and_slots() -> None:
    cache = GenerationCache(_gpt2(), [1, 40, 0, 16], page_size=16)
    assert cache.block_table.tolist() == [[0, -1, -1], [1, 2, 3], [-1, -1, -1], [4, -1, -1]]
    positions = torch.tensor([[0, 1], [17, 39], [0, 0], [15, 0]])
    valid = torch.tensor([[True, False], [True, True], [False, False], [True, True]])
    assert cache.slots(positions, valid).tolist() == [[0, -1], [33, 55], [-1, -1], [79, 64]]
    assert cache.layers[0].k.dtype == torch.float32 and cache.layers[0].k.shape == (6, 4, 16, 8)


# --------------------------------------------------------------------------- the operators' CPU path


def test_paged_attention_equals_packed_attention() -> None:
    """The last row of causal attention over a packed sequence, from pages in any order."""
    h, hkv, d, n, page = 6, 2, 8, 37, 16
    qkv = torch.randn(1, n, (h + 2 * hkv) * d)
    want = ops.reference_attention(qkv, h, hkv, d)[0, -1].view(h, d)
    pages = ops.KVPages.allocate(5, hkv, page, d, dtype=torch.float32)
    pages.k.fill_(math.nan)
    pages.v.fill_(math.nan)
    table = torch.tensor([[4, 0, 2]], dtype=torch.int32)
    t = torch.arange(n)
    rows = qkv[0].view(n, h + 2 * hkv, d)
    ops.kv_cache_write(pages, rows[:, h:h + hkv], rows[:, h + hkv:], table[0].long()[t // page] * page + t % page)
    out, lse = ops.paged_attention(rows[-1:, :h], pages, table, torch.tensor([n], dtype=torch.int32), return_lse=True)
    assert torch.allclose(out[0], want, atol=1e-6)
    k = rows[:, h:h + hkv].repeat_interleave(h // hkv, 1)
    scores = torch.einsum("hd,nhd->hn", rows[-1, :h], k) / math.sqrt(d)
    assert torch.allclose(lse[0], torch.logsumexp(scores, -1), atol=1e-6)


@pytest.mark.parametrize("dtype,top", [(torch.int8, 127.0), (torch.float8_e4m3fn, 448.0)])
def test_cache_round_trip(dtype, top) -> None:
    pages = ops.KVPages.allocate(4, 3, 16, 32, dtype=dtype)
    k, v = torch.randn(20, 3, 32), torch.randn(20, 3, 32)
    k[3, 1], v[5, 0, 2] = 0.0, math.inf
    slots = torch.randperm(64)[:20]
    slots[7] = -1
    ops.kv_cache_write(pages, k, v, slots)
    rk, rv = ops.kv_cache_read(pages, slots)
    assert rk.dtype == torch.bfloat16 and bool((rk[7] == 0).all()) and bool(torch.isnan(rv[5, 0]).all()) and bool((rk[3, 1] == 0).all())
    stored = torch.ones(20, dtype=torch.bool)
    stored[7] = False
    amax = k[stored].abs().amax(-1, keepdim=True)
    step = amax / 254 if dtype == torch.int8 else k[stored].abs() / 16 + amax / 448 * 2.0**-10
    assert bool(((rk[stored].float() - k[stored]).abs() <= 1.001 * step + 2.0**-8 * k[stored].abs()).all())
    out = (torch.zeros(20, 3, 32), torch.zeros(20, 3, 32))
    assert ops.kv_cache_read(pages, slots, out=out)[0] is out[0] and torch.equal(out[0].bfloat16(), rk)


def test_sampling_is_a_draw_from_what_the_filters_leave() -> None:
    row = torch.tensor([1.0, 0.0, 2.0, -1.0, 1.0, 0.5])
    b = 20000
    noise = torch.empty(b, 6).exponential_(generator=torch.Generator().manual_seed(2))
    token, logprob = ops.sample_tokens(row.expand(b, 6), noise, top_p=0.7)
    p = torch.softmax(row.double(), 0)
    kept = torch.tensor([True, False, True, False, False, False])  # 0.42, then 0.155 (the lower index first): 0.42 + 0.155 < 0.7
    kept[4] = True
    q = torch.where(kept, p, 0.0) / p[kept].sum()
    share = torch.bincount(token, minlength=6).double() / b
    assert bool(((share - q).abs() <= 5 * torch.sqrt(q * (1 - q) / b)).all())
    assert torch.allclose(logprob, torch.log(p)[token].float(), atol=1e-6)


def test_sampling_edges() -> None:
    inf = math.inf
    logits = torch.tensor([[-inf, -inf, -inf], [math.nan, 1.0, -inf], [2.0, 2.0, 2.0], [inf, 0.0, inf]])
    token, logprob = ops.sample_tokens(logits, torch.ones(4, 3), temperature=0.0)
    assert token.tolist() == [-1, 1, 0, 0]
    assert torch.allclose(logprob, torch.tensor([-inf, 0.0, -math.log(3), -math.log(2)]))
    token, _ = ops.sample_tokens(logits, torch.tensor([[1.0, 1.0, 1.0]] * 3 + [[3.0, 1e-9, 2.0]]))
    assert token.tolist() == [-1, 1, 0, 2]


def test_operator_refusals() -> None:
    pages = ops.KVPages.allocate(2, 2, 16, 8, dtype=torch.float32)
    rows, slots = torch.zeros(3, 2, 8), torch.arange(3)
    for bad in ((rows[:, :1], rows, slots), (rows, rows, slots[:2]), (rows, rows, slots.float()), (rows.long(), rows.long(), slots)):
        with pytest.raises(ConfigurationError):
            ops.kv_cache_write(pages, *bad)
    with pytest.raises(UnsupportedFeatureError):
        ops.kv_cache_write(pages, rows.clone().requires_grad_(), rows, slots)
    q, table, n = torch.zeros(1, 4, 8), torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    for bad in ((q[:, :3], table, n), (q, table.long(), n), (q, table, n.long()), (q, table[:0], n), (q[0], table, n)):
        with pytest.raises(ConfigurationError):
            ops.paged_attention(bad[0], pages, *bad[1:])
    for shape, kind in (((2, 2, 20, 8), torch.float32), ((2, 2, 16, 8), torch.int16)):
        with pytest.raises(ConfigurationError):
            ops.KVPages.allocate(*shape, dtype=kind)
    logits, noise = torch.randn(2, 5), torch.ones(2, 5)
    for bad in ({"temperature": -0.5}, {"top_p": 2.0}, {"min_p": math.nan}, {"top_k": -3}, {"top_k": torch.ones(2)}, {"top_p": torch.ones(1)}):
        with pytest.raises(ConfigurationError):
            ops.sample_tokens(logits, noise, **bad)
    with pytest.raises(ConfigurationError):
        ops.sample_tokens(logits, noise[:1])
