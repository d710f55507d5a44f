"""How many bits the text-generation kernels carry, and over which magnitudes, against plain statements in 64 bits.

Outputs are bf16, whose rounding hides what a kernel keeps of its weights.  The inputs here cancel, so that the result is small
next to what was summed and its rounding small as well.
"""

from __future__ import annotations

import math

import pytest
import torch

import hybrid_training.ops as ops
from hybrid_training.errors import UnsupportedFeatureError

pytestmark = pytest.mark.gpu


def _one_page_each(b: int, kvh: int, d: int, dtype: torch.dtype) -> tuple[ops.KVPages, torch.Tensor]:
    """A pool of zeros with one page of 16 tokens for each of ``b`` sequences, and its block table."""
    pages = ops.KVPages.allocate(b, kvh, 16, d, dtype=dtype, device="cuda")
    for x in (pages.k, pages.v):
        x.view(torch.uint8).zero_()
    return pages, torch.arange(b, dtype=torch.int32, device="cuda")[:, None].contiguous()


def _check(q, pages, table, n, scale, relative: float) -> None:
    """Each output within one rounding to bf16 and ``relative`` of the average magnitude that was summed for it."""
    got = ops.paged_attention(q, pages, table, n, scale=scale)
    want = ops.reference_paged_attention(q, pages, table, n, scale=scale, compute_dtype=torch.float64)[0]
    v = pages.v if pages.v_scale is not None else pages.v.abs()
    magnitudes = ops.KVPages(pages.k, v if v.dtype == torch.bfloat16 else v.float().abs().to(v.dtype), pages.k_scale, pages.v_scale)
    summed = ops.reference_paged_attention(q, magnitudes, table, n, scale=scale, compute_dtype=torch.float64)[0]
    excess = (got.double() - want).abs() - 2.0**-8 * want.abs() - relative * summed
    assert bool((excess <= 0).all()), float((excess / summed).max())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.int8])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads,kvh", [(1, 1), (8, 2), (10, 2), (8, 1), (12, 1)])
def test_paged_attention_carries_weights_in_full(dtype, d, heads, kvh) -> None:
    """A token of weight 1 against fifteen of weight 2^-a, whose values cancel it.

    The exponential is right to 2^-22 and a, up to 8, to 2^-24 of itself: 2^-21 of the weight, on half of what is summed.
    Weights of 16 bits (relative to the largest: 2^-17, to their own magnitude: 2^-18) show at several times the 2^-20 allowed.
    """
    b = 64
    pages, table = _one_page_each(b, kvh, d, dtype)
    a = 4.0 + 4.0 * torch.rand(b, kvh, device="cuda", generator=torch.Generator(device="cuda").manual_seed(d + heads))
    if dtype == torch.bfloat16:
        a = a.bfloat16().float()
        pages.k[:, :, 1:, 0] = -a[..., None].bfloat16()
    else:
        pages.k[:, :, 1:, 0] = -1
        pages.k_scale.copy_(a[..., None].expand(b, kvh, 16))
        pages.v_scale.fill_(1.0)
    c = 127.0 - torch.arange(d, device="cuda") % 64
    pages.v[:, :, 1:] = -c.to(dtype)
    pages.v[:, :, 0] = torch.round(15.0 * c * torch.exp2(-a)[..., None]).to(dtype)
    q = torch.zeros(b, heads, d, device="cuda", dtype=torch.bfloat16)
    q[..., 0] = 1.0
    n = torch.full((b,), 16, dtype=torch.int32, device="cuda")
    _check(q, pages, table, n, math.log(2.0), 2.0**-20)


@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("heads,kvh", [(4, 1), (8, 1)])
def test_paged_attention_value_scales_round_nothing(dtype, heads, kvh) -> None:
    """Two tokens of equal scores, whose values cancel through unequal scales.

    Equal scores have weights that are powers of two times a scale: two terms of fp16 or digits leave 2^-22 of one of them, so
    2^-21 allows for twice that.  A logarithm of the scale that joins the exponent would leave 2^-22 of its own magnitude, five
    times that.
    """
    b, d = 512, 64
    pages, table = _one_page_each(b, kvh, d, dtype)
    gen = torch.Generator(device="cuda").manual_seed(heads)
    first = torch.exp2(-3.0 - 20.0 * torch.rand(b, kvh, device="cuda", generator=gen))
    c = torch.tensor([64.0, 96.0, 112.0, 72.0], device="cuda").repeat(d // 4)
    pages.v[:, :, 0] = c.to(dtype)
    pages.v[:, :, 1] = (-(c / 2)).to(dtype)
    pages.k_scale.fill_(1.0)
    pages.v_scale[:, :, 0] = first
    pages.v_scale[:, :, 1] = 2.0 * first * (1.0 + 1e-6 * torch.randn(b, kvh, device="cuda", generator=gen))
    # the cancelling partner at another power of two and mantissa: a third token takes part of the second's share
    part = torch.rand(b, kvh, device="cuda", generator=gen)
    pages.v[:, :, 2] = pages.v[:, :, 1]
    pages.v_scale[:, :, 2] = pages.v_scale[:, :, 1] * part
    pages.v_scale[:, :, 1] = pages.v_scale[:, :, 1] * (1.0 - part)
    q = torch.zeros(b, heads, d, device="cuda", dtype=torch.bfloat16)
    n = torch.full((b,), 3, dtype=torch.int32, device="cuda")
    _check(q, pages, table, n, 1.0, 2.0**-21)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("length", [5, 900])
def test_paged_attention_what_is_not_a_number_stays_so(dtype, length) -> None:
    """A NaN in a query, a key or a value reaches that head's output, and in a query or a key its log-sum-exp; no other head's."""
    pages = ops.KVPages.allocate(64, 3, 16, 64, dtype=dtype, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(1)
    k, v = (torch.randn(1024, 3, 64, device="cuda", generator=gen).bfloat16() for _ in range(2))
    k[3, 1, 5] = math.nan
    v[4, 2, 7] = math.nan
    ops.kv_cache_write(pages, k, v, torch.arange(1024, device="cuda"))
    q = torch.randn(1, 6, 64, device="cuda", generator=gen).bfloat16()
    q[0, 1, 9] = math.nan
    table, n = torch.arange(64, dtype=torch.int32, device="cuda")[None].contiguous(), torch.tensor([length], dtype=torch.int32, device="cuda")
    out, lse = ops.paged_attention(q, pages, table, n, return_lse=True)
    assert torch.isnan(out[0]).any(-1).tolist() == [False, True, True, True, True, True]
    assert torch.isnan(lse[0, :4]).tolist() == [False, True, True, True]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("factor", [1e-36, 1e-33, 1e-30, 1e-20, 1.0, 1e20, 1e30, 5e30, 1e33, 1e36, 1e37])
def test_paged_attention_query_magnitudes(dtype, factor) -> None:
    """Queries of every magnitude that bf16 has, whose scores the scale brings back to a few units.

    One rounding to bf16, and the error of the weights: scores up to 30 in fp32 (2^-19) and, of 8-bit caches, queries to 2^-22
    (int8) or all of their 8 bits (e4m3).
    """
    pages = ops.KVPages.allocate(16, 2, 16, 64, dtype=dtype, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(2)
    k, v = (torch.randn(256, 2, 64, device="cuda", generator=gen).bfloat16() for _ in range(2))
    ops.kv_cache_write(pages, 0.25 * k, v, torch.arange(256, device="cuda"))
    table = torch.arange(16, dtype=torch.int32, device="cuda").view(2, 8)
    n = torch.tensor([128, 77], dtype=torch.int32, device="cuda")
    q = (factor * torch.randn(2, 8, 64, device="cuda", generator=gen)).bfloat16()
    assert bool(torch.isfinite(q).all())
    _check(q, pages, table, n, 0.5 / factor, 2.0**-18)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("exponent", [-100, -60, 0, 40, 62, 64, 70, 90, 120])
@pytest.mark.parametrize("order", ["mixed", "falling", "rising"])
@pytest.mark.parametrize("lengths", [[200, 37], [9001]])
def test_paged_attention_value_magnitudes(dtype, exponent, order, lengths) -> None:
    """Values of every magnitude next to rows of zeros and of small values, whose weights count as much; in any order.

    One rounding to bf16, and the error of the weights: scores up to 10 in fp32 (2^-21), twice.
    """
    total = sum(-(-n // 16) * 16 for n in lengths)
    pages = ops.KVPages.allocate(total // 16, 2, 16, 64, dtype=dtype, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(exponent + 200)
    k, v = (torch.randn(total, 2, 64, device="cuda", generator=gen) for _ in range(2))
    kind = torch.randint(0, 3, (total, 1, 1), device="cuda", generator=gen) if order == "mixed" else torch.arange(total, device="cuda")[:, None, None] * 3 // total
    if order == "falling":
        kind = 2 - kind
    v = torch.where(kind == 0, 0.0, torch.where(kind == 1, v, v * 2.0**exponent))
    ops.kv_cache_write(pages, (0.25 * k).bfloat16(), v.bfloat16(), torch.arange(total, device="cuda"))
    table = torch.full((len(lengths), -(-max(lengths) // 16)), -1, dtype=torch.int32, device="cuda")
    start = 0
    for i, n in enumerate(lengths):
        used = -(-n // 16)
        table[i, :used] = torch.arange(start, start + used, device="cuda")
        start += used
    q = torch.randn(len(lengths), 8, 64, device="cuda", generator=gen).bfloat16()
    _check(q, pages, table, torch.tensor(lengths, dtype=torch.int32, device="cuda"), 0.5, 2.0**-20)


# --------------------------------------------------------------------------- sampling


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("filters", [{}, {"top_p": 0.9}, {"top_k": 700}, {"temperature": 0.0}])
def test_sample_tokens_while_the_gpu_is_busy(dtype, filters) -> None:
    """Clusters whose blocks start when another stream's blocks leave room, with short stretches of a row per block."""
    gen = torch.Generator(device="cuda").manual_seed(4)
    b, v = 9, 33000
    logits = (2.0 * torch.randn(b, v, device="cuda", generator=gen)).to(dtype)
    noise = torch.empty(b, v, device="cuda").exponential_(generator=gen).clamp_(min=1e-30)
    want = ops.reference_sample_tokens(logits, noise, **filters, compute_dtype=torch.float64)[0]
    x = torch.randn(4096, 4096, device="cuda", generator=gen).bfloat16()
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(20):
        with torch.cuda.stream(other):
            torch.mm(x, x)
        got += [ops.sample_tokens(logits, noise, **filters)[0] for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("skew", [1, 3])
@pytest.mark.parametrize("filters", [{"temperature": 1e30}, {"temperature": 1e-4}, {"min_p": 0.5, "temperature": 1e30}, {}])
def test_sample_tokens_names_a_token_whatever_the_random_numbers(dtype, skew, filters) -> None:
    """Rows at odd offsets without a usable random number: the lowest index of those that may be drawn, never one outside the row."""
    b, v = 5, 3001
    room = torch.zeros(b, v + 8, device="cuda", dtype=dtype)
    logits, noise = room[:, skew : skew + v], torch.full((b, v), math.nan, device="cuda")
    noise[3, 2000] = 1.0
    token, logprob = ops.sample_tokens(logits, noise, **filters)
    assert token.tolist() == [0, 0, 0, 2000, 0]
    assert bool(((logprob + math.log(v)).abs() <= 1e-5 * math.log(v)).all())


@pytest.mark.parametrize("v", [32769, 33320, 33321, 35000, 36800, 36864, 36865])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("filters", [{"top_p": 0.9}, {"top_k": 900}])
def test_sample_tokens_vocabularies_between_powers_of_two(v, dtype, filters) -> None:
    """Many rows of vocabularies that are a little more than what a block holds of half as many."""
    gen = torch.Generator(device="cuda").manual_seed(v)
    b = 150
    logits = (2.0 * torch.randn(b, v + 1, device="cuda", generator=gen)).to(dtype)[:, 1:]
    noise = torch.empty(b, v, device="cuda").exponential_(generator=gen).clamp_(min=1e-30)
    want, want_logprob = ops.reference_sample_tokens(logits, noise, **filters, compute_dtype=torch.float64)
    token, logprob = ops.sample_tokens(logits, noise, **filters)
    assert torch.equal(token, want)
    assert bool(((logprob.double() - want_logprob).abs() <= 4e-6 * (1.0 + want_logprob.abs())).all())


@pytest.mark.parametrize("b, v", [(6, 50), (6, 40001), (160, 40001), (40, 128256)])
@pytest.mark.parametrize("name", ["temperature", "top_p", "min_p"])
@pytest.mark.parametrize("filters", [{}, {"top_k": 700}])
def test_sample_tokens_filters_that_are_not_numbers(b, v, name, filters) -> None:
    """A row whose value is NaN yields its most probable token, in batches of any size and with any other filter."""
    gen = torch.Generator(device="cuda").manual_seed(b)
    logits = 2.0 * torch.randn(b, v, device="cuda", generator=gen)
    noise = torch.empty(b, v, device="cuda").exponential_(generator=gen).clamp_(min=1e-30)
    values = torch.full((b,), 0.0 if name == "min_p" else 1.0, device="cuda")
    values[::2] = math.nan
    filters = {**filters, name: values}
    token, logprob = ops.sample_tokens(logits, noise, **filters)
    want, want_logprob = ops.reference_sample_tokens(logits, noise, **filters, compute_dtype=torch.float64)
    assert torch.equal(token, want) and torch.equal(token[::2], logits[::2].argmax(-1))
    assert bool(((logprob.double() - want_logprob).abs() <= 4e-6 * (1.0 + want_logprob.abs())).all())


def test_sample_tokens_refuses_logits_that_need_a_gradient() -> None:
    logits, noise = torch.randn(2, 9, device="cuda", requires_grad=True), torch.ones(2, 9, device="cuda")
    with pytest.raises(UnsupportedFeatureError):
        ops.sample_tokens(logits, noise)
    with torch.no_grad():
        token, logprob = ops.sample_tokens(logits, noise)
    assert token.shape == (2,) and not logprob.requires_grad


@pytest.mark.parametrize("v,b", [(128256, 2), (128256, 40), (50257, 6), (20011, 100), (3001, 4)])
@pytest.mark.parametrize("depth", [10.0, 24.0, 28.0, 30.5, 33.5, 45.0])
@pytest.mark.parametrize("top_k", [0, 2999])
def test_sample_tokens_cuts_long_tails_where_their_sum_says(v, b, depth, top_k) -> None:
    """One likely token and a tail of weights 2^-depth, of which top_p keeps half.

    Row after row, the one token that would win the draw lies a thirtieth of the tail's mass within the cut, or beyond it.  Weights
    are right to 2^-22 and add up as multiples of 2^-44 or finer, far closer than that; multiples of 2^-31 would keep the
    whole tail, or none.  top_p is an fp32 number, so the tail has to weigh a few hundred of its last places.
    """
    kept_of = v - 1 if top_k == 0 else top_k - 1
    tail = kept_of * 2.0**-depth
    if tail < 300 * 2.0**-24:
        pytest.skip("the tail is lost among top_p's last places")
    gen = torch.Generator(device="cuda").manual_seed(v)
    z = -math.log(2.0) * depth + 0.01 * torch.randn(b, v, device="cuda", generator=gen)
    z.scatter_(1, torch.randint(0, v, (b, 1), device="cuda", generator=gen), 0.0)
    top_p = (1.0 + 0.5 * tail) / (1.0 + tail)
    order = torch.sort(z, dim=-1, descending=True, stable=True).indices
    w = torch.softmax(torch.gather(z, 1, order).double(), -1)
    if top_k:
        w[:, top_k:] = 0.0
    w /= w.sum(-1, keepdim=True)
    before = torch.cumsum(w, -1) - w
    edge = float(torch.tensor(top_p, dtype=torch.float32)) + torch.where(torch.arange(b, device="cuda") % 2 == 0, -1.0, 1.0)[:, None] * (1.0 - 1.0 / (1.0 + tail)) / 30.0
    favourite = torch.gather(order, 1, (before < edge).sum(-1, keepdim=True) - 1)
    noise = torch.ones(b, v, device="cuda").scatter_(1, favourite, 1e-20)
    token, _ = ops.sample_tokens(z, noise, top_p=top_p, top_k=top_k)
    inside = torch.arange(b, device="cuda") % 2 == 0
    assert torch.equal(token, torch.where(inside, favourite[:, 0], z.argmax(-1)))
    assert torch.equal(token, ops.reference_sample_tokens(z, noise, top_p=top_p, top_k=top_k, compute_dtype=torch.float64)[0])
