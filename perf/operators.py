"""Workloads of the text-generation operators, for timing and for comparing outputs.

A trained decoder answers with four operators of ``hybrid_training.ops``: the keys and values of
new tokens are written into a paged cache (``kv_cache_write``, held as bf16, int8 or fp8 with one
scale per token and head), read back (``kv_cache_read``), attended to by one new token of every
sequence (``paged_attention``), and the logits that follow are turned into a token
(``sample_tokens``).  Each case below is one pass through one of them (writing and reading back
form one pass: what a cache holds in 8 bits is seen as the values that are read from it).

``own`` selects who computes: ``False`` is the plain form, elementary torch operations in fp32 with
one rounding at the end; ``True`` makes the calls a user makes of ``hybrid_training.ops``.
"""

from __future__ import annotations

import math
import random
from typing import Any

import torch

own = False

_CACHE_DTYPES = {"bf16": torch.bfloat16, "int8": torch.int8, "fp8": torch.float8_e4m3fn}
_LARGEST = {"bf16": 127.0, "int8": 127.0, "fp8": 448.0}  # the value a row's largest magnitude is stored as
_SMALLEST_SCALE = 2.0**-64

# (query heads, key/value heads, head size): the GPT-2 124M shape, a 2048-wide Llama shape, the Llama-3-8B
# shape whole and as the slices that 2, 4 and 8 tensor-parallel ranks hold.
_HEADS = [(12, 12, 64), (16, 16, 128), (32, 8, 128), (16, 4, 128), (8, 2, 128), (4, 1, 128)]
_VOCABULARIES = [32000, 50257, 128256]


def listed() -> list[dict[str, Any]]:
    return [
        # Attention of one new token per sequence over the paged cache.
        # One GPT-2 answer at the end of its context, alone on the GPU: latency counts.
        {"name": "decode_gpt2_one", "op": "decode", "batch": 1, "heads": 12, "kv_heads": 12, "dim": 64, "page": 16,
         "shortest": 1024, "longest": 1024, "cache": "bf16"},
        # Samples drawn from GPT-2 during its training: a batch of very unequal lengths.
        {"name": "decode_gpt2_batch", "op": "decode", "batch": 48, "heads": 12, "kv_heads": 12, "dim": 64, "page": 16,
         "shortest": 1, "longest": 1024, "cache": "bf16"},
        # The Llama-3-8B shape, an ordinary batch within its 4096 tokens, unquantised.
        {"name": "decode_llama_bf16", "op": "decode", "batch": 32, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16,
         "shortest": 257, "longest": 4096, "cache": "bf16"},
        # One of eight tensor-parallel ranks: one key/value head, fp8 cache, an odd batch.
        {"name": "decode_llama_tp8_fp8", "op": "decode", "batch": 61, "heads": 4, "kv_heads": 1, "dim": 128, "page": 64,
         "shortest": 100, "longest": 4096, "cache": "fp8"},
        # Two long documents: few rows, so the work has to be split over the length.
        {"name": "decode_long_int8", "op": "decode", "batch": 2, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64,
         "shortest": 100003, "longest": 100003, "cache": "int8"},
        # The largest: a full rollout batch on an int8 cache.
        {"name": "decode_rollout_int8", "op": "decode", "batch": 128, "heads": 32, "kv_heads": 8, "dim": 128, "page": 32,
         "shortest": 4097, "longest": 8192, "cache": "int8"},
        # Quantising keys and values as they are written, and reading them back.
        # One decoding step of 32 sequences: latency counts.
        {"name": "cache_step_int8", "op": "cache", "tokens": 32, "kv_heads": 8, "dim": 128, "page": 16, "cache": "int8"},
        # A ragged GPT-2 prompt batch in fp8.
        {"name": "cache_prompt_fp8", "op": "cache", "tokens": 8191, "kv_heads": 12, "dim": 64, "page": 16, "cache": "fp8"},
        # Four full prompts of the Llama-3-8B shape in int8.
        {"name": "cache_prompt_int8", "op": "cache", "tokens": 16384, "kv_heads": 8, "dim": 128, "page": 32, "cache": "int8"},
        # Choosing the next token from logits and given random numbers.
        # One GPT-2 answer with every filter on: latency counts.
        {"name": "sample_gpt2_one", "op": "sample", "batch": 1, "vocab": 50257, "logits": "bf16", "temperature": 0.8,
         "top_k": 50, "top_p": 0.95, "min_p": 0.02},
        # An ordinary batch with a nucleus over the Llama-3 vocabulary.
        {"name": "sample_llama_top_p", "op": "sample", "batch": 64, "vocab": 128256, "logits": "bf16", "temperature": 0.7,
         "top_k": 0, "top_p": 0.9, "min_p": 0.0},
        # The largest: a rollout batch drawn from the whole distribution of fp32 logits.
        {"name": "sample_rollout_all", "op": "sample", "batch": 256, "vocab": 128256, "logits": "fp32", "temperature": 1.0,
         "top_k": 0, "top_p": 1.0, "min_p": 0.0},
    ]


def _log_uniform(rng: random.Random, low: int, high: int) -> int:
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng: random.Random) -> dict[str, Any]:
    op = rng.choice(["decode", "decode", "cache", "sample"])
    if op == "sample":
        return {"op": op, "batch": _log_uniform(rng, 1, 256), "vocab": rng.choice(_VOCABULARIES), "logits": rng.choice(["bf16", "fp32"]),
                "temperature": rng.choice([0.0, 0.6, 0.8, 1.0, 1.3]), "top_k": rng.choice([0, 0, 1, 20, 50, 1000]),
                "top_p": rng.choice([1.0, 1.0, 0.5, 0.9, 0.95]), "min_p": rng.choice([0.0, 0.0, 0.02, 0.1])}
    heads, kv_heads, dim = rng.choice(_HEADS)
    page, cache = rng.choice([16, 32, 64, 128]), rng.choice(["bf16", "int8", "fp8"])
    if op == "cache":
        most = 16384 * 8 * 128 // (kv_heads * dim)
        return {"op": op, "tokens": _log_uniform(rng, 1, min(most, 32768)), "kv_heads": kv_heads, "dim": dim, "page": page, "cache": cache}
    longest = _log_uniform(rng, 1, 100000)
    # tokens x heads x head size stay within half of the largest listed case (bf16 holds twice the bytes)
    most = max(1, 128 * 8192 * 8 * 128 // 2 // (longest * kv_heads * dim))
    batch = _log_uniform(rng, 1, min(256, most))
    shortest = rng.choice([1, max(1, longest // 2), longest])
    return {"op": op, "batch": batch, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "shortest": shortest,
            "longest": longest, "cache": cache}


# --------------------------------------------------------------------------- inputs


def _lengths(case: dict[str, Any], seed: int) -> list[int]:
    rng = random.Random(seed * 7919 + 13)
    lengths = [rng.randint(case["shortest"], case["longest"]) for _ in range(case["batch"])]
    lengths[rng.randrange(case["batch"])] = case["longest"]  # the table is as wide as the longest sequence
    return lengths


def _filled(shape: tuple[int, ...], cache: str, gen: torch.Generator) -> tuple[torch.Tensor, torch.Tensor | None]:
    """A pool of normal keys or values as the cache holds them, and its scales."""
    x = torch.randn(shape, device="cuda", generator=gen, dtype=torch.bfloat16 if cache == "bf16" else torch.float16)
    if cache == "bf16":
        return x, None
    # a head's largest magnitude is 2.5 to 4 of its standard deviations, at the magnitude the token happens to have
    scale = torch.rand(shape[:-1], device="cuda", generator=gen).mul_(0.02).add_(0.01)
    if cache == "int8":
        return x.mul_(40).round_().clamp_(-127, 127).to(torch.int8), scale
    return x.mul_(140).clamp_(-448, 448).to(torch.float8_e4m3fn), scale.mul_(0.28)


def _pages(case: dict[str, Any], k: torch.Tensor, v: torch.Tensor, ks: torch.Tensor | None, vs: torch.Tensor | None) -> Any:
    from hybrid_training.ops import KVPages

    return KVPages(k, v, ks, vs)


def prepare(case: dict[str, Any], seed: int) -> dict[str, Any]:
    gen = torch.Generator(device="cuda").manual_seed(seed * 1000003 + 17)
    state: dict[str, Any] = {"case": case}
    if case["op"] == "sample":
        b, v = case["batch"], case["vocab"]
        logits = torch.randn(b, v, device="cuda", generator=gen).mul_(2.0)
        # a language model's logits: a broad bulk, and a few dozen plausible tokens well above it
        apart = v // 48
        likely = torch.randint(0, apart, (b, 48), device="cuda", generator=gen) + apart * torch.arange(48, device="cuda")
        logits.scatter_(1, likely, 6.0 + 8.0 * torch.rand(b, 48, device="cuda", generator=gen))
        state["logits"] = logits.bfloat16() if case["logits"] == "bf16" else logits
        state["noise"] = torch.empty(b, v, device="cuda").exponential_(1.0, generator=gen).clamp_(min=1e-30)
        fill = {"temperature": torch.float32, "top_p": torch.float32, "min_p": torch.float32, "top_k": torch.int32}
        state.update({n: torch.full((b,), case[n], dtype=t, device="cuda") for n, t in fill.items()})
        return state
    page, kvh, dim = case["page"], case["kv_heads"], case["dim"]
    if case["op"] == "cache":
        t = case["tokens"]
        pool = t // page + 8
        x = torch.randn(t, 2 * kvh, dim, device="cuda", generator=gen)
        x.mul_(torch.rand(t, 2 * kvh, 1, device="cuda", generator=gen).add_(0.5))
        # keys and values lie side by side in the projection's output, as the fused projection writes them
        state["kv"] = x.bfloat16()
        order = torch.randperm(pool, device="cuda", generator=gen)
        at = torch.arange(t, device="cuda")
        state["slots"] = order[at // page] * page + at % page
        dtype = _CACHE_DTYPES[case["cache"]]
        k, v = (torch.zeros(pool, kvh, page, dim, dtype=dtype, device="cuda") for _ in range(2))
        ks, vs = (None if case["cache"] == "bf16" else torch.zeros(pool, kvh, page, device="cuda") for _ in range(2))
    else:
        b, width = case["batch"], -(-case["longest"] // page)
        lengths = _lengths(case, seed)
        used = [-(-n // page) for n in lengths]
        pool = sum(used) + 1
        order = torch.randperm(pool - 1, device="cuda", generator=gen).to(torch.int32) + 1  # page 0 is nobody's
        table = torch.zeros(b, width, dtype=torch.int32)
        table = table.cuda()
        count = torch.tensor(used, device="cuda")
        held = torch.arange(width, device="cuda")[None, :] < count[:, None]
        table[held] = order
        state["table"] = table
        state["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        state["q"] = (1.5 * torch.randn(b, case["heads"], dim, device="cuda", generator=gen)).bfloat16()
        k, ks = _filled((pool, kvh, page, dim), case["cache"], gen)
        v, vs = _filled((pool, kvh, page, dim), case["cache"], gen)
    state.update(k=k, v=v, k_scale=ks, v_scale=vs)
    if own:
        state["pages"] = _pages(case, k, v, ks, vs)
    return state


# --------------------------------------------------------------------------- one pass


def run(state: dict[str, Any]) -> dict[str, torch.Tensor]:
    case = state["case"]
    if case["op"] == "decode":
        return _run_decode(state)
    return _run_cache(state) if case["op"] == "cache" else _run_sample(state)


def _bytes(pool: torch.Tensor) -> torch.Tensor:
    """fp8 values as the bytes they are, since indexing need not know the type."""
    return pool.view(torch.uint8) if pool.dtype == torch.float8_e4m3fn else pool


def _run_decode(s: dict[str, Any]) -> dict[str, torch.Tensor]:
    if own:
        from hybrid_training import ops

        out, lse = ops.paged_attention(s["q"], s["pages"], s["table"], s["lengths"], return_lse=True)
        return {"out": out, "lse": lse}
    q, table = s["q"].float(), s["table"].long()
    b, h, d = q.shape
    kvh, page = s["k"].shape[1:3]
    n = table.shape[1] * page
    valid = (torch.arange(n, device=q.device)[None, :] < s["lengths"][:, None])[:, None, :, None]

    def gathered(pool: torch.Tensor, scale: torch.Tensor | None) -> torch.Tensor:
        x = _bytes(pool)[table].view(pool.dtype).float()
        if scale is not None:
            x = x * scale[table][..., None]
        x = x.transpose(1, 2).reshape(b, kvh, n, d)
        return torch.where(valid, x, 0.0)

    scores = q.view(b, kvh, h // kvh, d) @ gathered(s["k"], s["k_scale"]).transpose(-1, -2) * (1.0 / math.sqrt(d))
    scores = torch.where(valid.transpose(-1, -2), scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    out = (p @ gathered(s["v"], s["v_scale"])) / total
    return {"out": out.reshape(b, h, d).to(s["q"].dtype), "lse": (top + torch.log(total)).reshape(b, h)}


def _run_cache(s: dict[str, Any]) -> dict[str, torch.Tensor]:
    kvh = s["case"]["kv_heads"]
    k, v = s["kv"][:, :kvh], s["kv"][:, kvh:]
    if own:
        from hybrid_training import ops

        ops.kv_cache_write(s["pages"], k, v, s["slots"])
        k, v = ops.kv_cache_read(s["pages"], s["slots"])
    else:
        k = _plain_round_trip(s, k, s["k"], s["k_scale"])
        v = _plain_round_trip(s, v, s["v"], s["v_scale"])
    out = {"k": k, "v": v}
    if s["k_scale"] is not None:
        out.update(k_scale=s["k_scale"], v_scale=s["v_scale"])
    return out


def _plain_round_trip(s: dict[str, Any], x: torch.Tensor, pool: torch.Tensor, scales: torch.Tensor | None) -> torch.Tensor:
    page = pool.shape[2]
    at, row = s["slots"] // page, s["slots"] % page
    if scales is None:
        pool[at, :, row] = x
        return pool[at, :, row]
    top, cache = _LARGEST[s["case"]["cache"]], s["case"]["cache"]
    xf = x.float()
    scale = (xf.abs().amax(-1) * (1.0 / top)).clamp(min=_SMALLEST_SCALE)
    y = xf * (1.0 / scale)[..., None]
    y = torch.round(y) if cache == "int8" else y
    _bytes(pool)[at, :, row] = _bytes(y.clamp(-top, top).to(pool.dtype))
    scales[at, :, row] = scale
    return (_bytes(pool)[at, :, row].view(pool.dtype).float() * scales[at, :, row][..., None]).to(x.dtype)


def _run_sample(s: dict[str, Any]) -> dict[str, torch.Tensor]:
    if own:
        from hybrid_training import ops

        tokens, logprobs = ops.sample_tokens(s["logits"], s["noise"], temperature=s["temperature"], top_k=s["top_k"],
                                             top_p=s["top_p"], min_p=s["min_p"])
        return {"tokens": tokens, "logprobs": logprobs}
    logits, noise = s["logits"].float(), s["noise"]
    b, v = logits.shape
    greedy = (s["temperature"] <= 0)[:, None]
    t = torch.where(greedy, 1.0, s["temperature"][:, None])
    best = logits.amax(-1, keepdim=True)
    x = (logits - best) / t
    w = torch.exp(x)
    # tokens in falling order of their logit, the lower index first among equals
    ranked, order = torch.sort(logits, dim=-1, descending=True, stable=True)
    rank = torch.arange(v, device=logits.device)[None, :]
    top_k = s["top_k"][:, None]
    keep = (rank < top_k) | (top_k <= 0)
    ws = torch.gather(w, 1, order)
    mass = torch.where(keep, ws, 0.0)
    before = torch.cumsum(mass, -1) - mass
    top_p = s["top_p"][:, None]
    keep &= (before < top_p * mass.sum(-1, keepdim=True)) | (top_p >= 1.0)
    keep &= ws >= s["min_p"][:, None]
    keep &= (rank == 0) | ~greedy
    keep |= rank == 0
    score = torch.where(keep, ws / torch.gather(noise, 1, order), -1.0)
    tied = score == score.amax(-1, keepdim=True)
    token = torch.where(tied, order, v).amin(-1)
    logprob = torch.gather(x, 1, token[:, None])[:, 0] - torch.log(w.sum(-1))
    return {"tokens": token, "logprobs": logprob}


# --------------------------------------------------------------------------- what a pass cannot do without


def work(case: dict[str, Any]) -> dict[str, float]:
    if case["op"] == "sample":
        rows = case["batch"] * case["vocab"]
        filtered = case["top_k"] > 0 or case["top_p"] < 1.0 or case["min_p"] > 0.0 or case["temperature"] <= 0.0
        # logits once; the random numbers only of tokens that can be drawn (a filter leaves a handful)
        return {"bytes": rows * (2.0 if case["logits"] == "bf16" else 4.0) + (0.0 if filtered else rows * 4.0), "flops": 4.0 * rows}
    size = 2.0 if case["cache"] == "bf16" else 1.0
    scale = 0.0 if case["cache"] == "bf16" else 4.0
    if case["op"] == "cache":
        rows = 2.0 * case["tokens"] * case["kv_heads"]
        # read the new rows, write them as held, write them as read back
        return {"bytes": rows * (4.0 * case["dim"] + size * case["dim"] + scale), "flops": 4.0 * rows * case["dim"]}
    # lengths are uniform between the shortest and the longest, and one sequence is the longest
    tokens = case["longest"] + (case["batch"] - 1) * 0.5 * (case["shortest"] + case["longest"])
    held = tokens * case["kv_heads"] * 2.0 * (size * case["dim"] + scale)
    rows = case["batch"] * case["heads"]
    return {"bytes": held + rows * (4.0 * case["dim"] + 4.0), "flops": 4.0 * tokens * case["heads"] * case["dim"]}


# --------------------------------------------------------------------------- the definitions in 64 bits


def exact(case: dict[str, Any], seed: int) -> dict[str, torch.Tensor | None] | None:
    s = prepare(case, seed)
    if case["op"] == "decode":
        return _exact_decode(s)
    return _exact_cache(s) if case["op"] == "cache" else _exact_sample(s)


def _exact_decode(s: dict[str, Any]) -> dict[str, torch.Tensor | None]:
    q = s["q"].double()
    kvh, page, d = s["k"].shape[1:]
    group = q.shape[1] // kvh
    out = torch.empty(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.empty(q.shape[:2], dtype=torch.float64, device=q.device)
    for b, n in enumerate(s["lengths"].tolist()):
        mine = s["table"][b, : -(-n // page)].long()
        for g in range(kvh):
            k, v = (_bytes(p)[mine, g].view(p.dtype).double().reshape(-1, d)[:n] for p in (s["k"], s["v"]))
            if s["k_scale"] is not None:
                k = k * s["k_scale"][mine, g].double().reshape(-1, 1)[:n]
                v = v * s["v_scale"][mine, g].double().reshape(-1, 1)[:n]
            heads = slice(g * group, (g + 1) * group)
            scores = q[b, heads] @ k.T / math.sqrt(d)
            lse[b, heads] = torch.logsumexp(scores, -1)
            out[b, heads] = torch.softmax(scores, -1) @ v
    return {"out": out, "lse": lse}


def _exact_cache(s: dict[str, Any]) -> dict[str, torch.Tensor | None]:
    kvh, cache = s["case"]["kv_heads"], s["case"]["cache"]
    x = s["kv"].double()
    if cache == "bf16":
        return {"k": x[:, :kvh], "v": x[:, kvh:]}
    scale = (x.abs().max(-1, keepdim=True).values / _LARGEST[cache]).clamp_min(_SMALLEST_SCALE)
    y = x / scale
    if cache == "int8":
        y = torch.round(y)
    else:
        # steps of 1/8 of the power of two below, and of 2^-9 below 2^-6
        step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0**-6))) - 3.0)
        y = torch.round(y / step) * step
    back = y * scale
    page = s["k"].shape[2]
    pools = []
    for one in (scale[:, :kvh, 0], scale[:, kvh:, 0]):
        pool = torch.zeros(s["k"].shape[:3], dtype=torch.float64, device=x.device)
        pool[torch.div(s["slots"], page, rounding_mode="floor"), :, s["slots"] % page] = one
        pools.append(pool)
    return {"k": back[:, :kvh], "v": back[:, kvh:], "k_scale": pools[0], "v_scale": pools[1]}


def _exact_sample(s: dict[str, Any]) -> dict[str, torch.Tensor | None]:
    """The log-probability of the drawn token; the token itself is a whole number and has no value in 64 bits."""
    case = s["case"]
    temperature = case["temperature"] if case["temperature"] > 0 else 1.0
    z = s["logits"].double() / temperature
    logp = torch.log_softmax(z, -1)
    if case["temperature"] <= 0:
        return {"tokens": None, "logprobs": logp.max(-1).values}
    p = torch.softmax(z, -1)
    sorted_p, order = torch.sort(p, dim=-1, descending=True, stable=True)
    k = case["top_k"] if case["top_k"] > 0 else p.shape[1]
    sorted_p[:, k:] = 0.0
    if case["top_p"] < 1.0:
        share = sorted_p / sorted_p.sum(-1, keepdim=True)
        sorted_p[torch.cumsum(share, -1) - share >= case["top_p"]] = 0.0
    sorted_p[sorted_p < case["min_p"] * sorted_p[:, :1]] = 0.0
    race = sorted_p / s["noise"].double().gather(1, order)
    token = order.gather(1, race.argmax(-1, keepdim=True))
    return {"tokens": None, "logprobs": logp.gather(1, token)[:, 0]}
