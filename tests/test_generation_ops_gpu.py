"""Paged KV cache, paged attention and token sampling on the GPU, against plain statements in 64 bits."""

from __future__ import annotations

import math

import pytest
import torch

import hybrid_training.ops as ops
from hybrid_training.errors import ConfigurationError, UnsupportedFeatureError

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.int8, torch.float8_e4m3fn]


def _pool(num_pages: int, kvh: int, page: int, d: int, dtype: torch.dtype, seed: int = 0) -> ops.KVPages:
    """A pool whose every slot was written through the op under test's plain statement."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    pages = ops.KVPages.allocate(num_pages, kvh, page, d, dtype=dtype, device="cuda")
    t = num_pages * page
    k = torch.randn(t, kvh, d, device="cuda", generator=gen) * (0.5 + torch.rand(t, kvh, 1, device="cuda", generator=gen))
    v = torch.randn(t, kvh, d, device="cuda", generator=gen) * (0.5 + torch.rand(t, kvh, 1, device="cuda", generator=gen))
    ops.reference_kv_cache_write(pages, k.bfloat16(), v.bfloat16(), torch.arange(t, device="cuda"))
    return pages


def _tables(lengths: list[int], page: int, num_pages: int, seed: int = 0) -> torch.Tensor:
    """Block tables over distinct pages in random order; entries behind a sequence's end are -1."""
    gen = torch.Generator().manual_seed(seed)
    order = torch.randperm(num_pages, generator=gen).to(torch.int32)
    width = max(1, max(-(-n // page) for n in lengths))
    table = torch.full((len(lengths), width), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(lengths):
        w = -(-n // page)
        table[i, :w] = order[at:at + w]
        at += w
    assert at <= num_pages
    return table.cuda()


def _check_attention(q, pages, table, lengths, scale=None) -> None:
    out, lse = ops.paged_attention(q, pages, table, lengths, scale=scale, return_lse=True)
    want, want_lse = ops.reference_paged_attention(q, pages, table, lengths, scale=scale, compute_dtype=torch.float64)
    torch.cuda.synchronize()
    assert out.dtype == q.dtype and out.shape == q.shape
    # One rounding to bf16 (half an ulp, 2^-8 of the value); weights carried to 16 bits or more and sums in fp32 leave
    # less than 2^-14 of the largest value that was averaged.
    v = pages.v.to(torch.float32) if pages.v_scale is None else pages.v.to(torch.float32) * pages.v_scale[..., None]
    largest = float(torch.nan_to_num(v, 0.0, 0.0, 0.0).abs().max())
    err = (out.double() - want).abs()
    assert bool((err <= 1.01 * 2.0**-8 * want.abs() + 2.0**-14 * largest).all()), float(err.max())
    # lse: an fp32 rounding of the scores (their magnitude times 2^-22 or so) and of a sum
    empty = want_lse == -math.inf
    assert torch.equal(lse == -math.inf, empty)
    gap = (lse.double() - want_lse)[~empty].abs()
    assert bool((gap <= 1e-5 * (1.0 + want_lse[~empty].abs())).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads,kvh", [(12, 12), (32, 8), (6, 2), (8, 1), (24, 2), (40, 1), (1, 1)])
def test_paged_attention_matches_plain(dtype, d, heads, kvh) -> None:
    page = 16 if d == 64 else 32
    lengths = [0, 1, 15, 16, 17, 31, 32, 33, 64, 65, 100, 127, 129, 300, 511]
    num = sum(-(-n // page) for n in lengths) + 3
    pages = _pool(num, kvh, page, d, dtype)
    table = _tables(lengths, page, num)
    q = (2.0 * torch.randn(len(lengths), heads, d, device="cuda")).bfloat16()
    _check_attention(q, pages, table, torch.tensor(lengths, dtype=torch.int32, device="cuda"))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_paged_attention_page_sizes_and_long_rows(dtype, page) -> None:
    """One or two long rows are split over the GPU and joined; pages end inside every kind of tile."""
    lengths = [20011, 1, 4099]
    num = sum(-(-n // page) for n in lengths)
    pages = _pool(num, 2, page, 128, dtype, seed=1)
    q = (1.5 * torch.randn(3, 16, 128, device="cuda")).bfloat16()
    _check_attention(q, pages, _tables(lengths, page, num), torch.tensor(lengths, dtype=torch.int32, device="cuda"))


@pytest.mark.parametrize("batch", [1, 7, 148, 300, 1100])
def test_paged_attention_batches(batch) -> None:
    gen = torch.Generator().manual_seed(batch)
    lengths = torch.randint(0, 200, (batch,), generator=gen).tolist()
    num = sum(-(-n // 16) for n in lengths) + 1
    pages = _pool(num, 3, 16, 64, torch.int8, seed=2)
    q = torch.randn(batch, 9, 64, device="cuda").bfloat16()
    _check_attention(q, pages, _tables(lengths, 16, num), torch.tensor(lengths, dtype=torch.int32, device="cuda"))


@pytest.mark.parametrize("dtype", DTYPES)
def test_paged_attention_ignores_what_lies_behind_a_sequence(dtype) -> None:
    """NaN and infinity in unused slots, and scales of NaN there, reach no output."""
    lengths = [1, 17, 45, 0, 80]
    page, num = 16, 20
    pages = _pool(num, 2, page, 64, dtype, seed=3)
    table = _tables(lengths, page, num)
    used = torch.zeros(num, page, dtype=torch.bool, device="cuda")
    for i, n in enumerate(lengths):
        for t in range(n):
            used[table[i, t // page], t % page] = True
    unused = ~used[:, None, :].expand(num, 2, page)
    if dtype == torch.bfloat16:
        pages.k[unused] = math.nan
        pages.v[unused] = math.inf
    else:
        pages.k_scale[unused] = math.nan
        pages.v_scale[unused] = math.inf
        if dtype == torch.float8_e4m3fn:
            pages.v.view(torch.uint8)[unused] = 0x7F
    q = torch.randn(5, 4, 64, device="cuda").bfloat16()
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    out, lse = ops.paged_attention(q, pages, table, n, return_lse=True)
    want, want_lse = ops.reference_paged_attention(q, pages, table, n, compute_dtype=torch.float64)
    assert bool(torch.isfinite(out).all()) and bool((out[3] == 0).all()) and bool((lse[3] == -math.inf).all())
    assert bool(((out.double() - want).abs() <= 1.01 * 2.0**-8 * want.abs() + 2.0**-14 * 8.0).all())


def test_paged_attention_masks_pages_outside_the_pool() -> None:
    pages = _pool(8, 2, 16, 128, torch.int8)
    table = torch.tensor([[0, -1, 2, 3], [4, 1 << 30, 5, 8], [-5, 9, -1, 77]], dtype=torch.int32, device="cuda")
    n = torch.tensor([60, 64, 64], dtype=torch.int32, device="cuda")
    _check_attention(torch.randn(3, 8, 128, device="cuda").bfloat16(), pages, table, n)


def test_paged_attention_cuts_lengths_to_the_table() -> None:
    pages = _pool(8, 1, 16, 64, torch.bfloat16)
    table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device="cuda")
    q = torch.randn(2, 4, 64, device="cuda").bfloat16()
    n = torch.tensor([1000, -7], dtype=torch.int32, device="cuda")
    got = ops.paged_attention(q, pages, table, n)
    same = ops.paged_attention(q, pages, table, torch.tensor([32, 0], dtype=torch.int32, device="cuda"))
    assert torch.equal(got, same)
    none = ops.paged_attention(q, pages, table[:, :0], n)
    assert bool((none == 0).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_paged_attention_extreme_scores_and_scales(dtype) -> None:
    """Scores of hundreds (one token takes all), equal scores, and value magnitudes 2^40 apart."""
    page, lengths = 16, [333, 333, 333]
    num = 3 * -(-333 // page)
    pages = _pool(num, 2, page, 128, dtype, seed=5)
    table, n = _tables(lengths, page, num), torch.tensor(lengths, dtype=torch.int32, device="cuda")
    q = torch.randn(3, 8, 128, device="cuda")
    q[0] *= 60.0
    q[1] = 0.0
    _check_attention(q.bfloat16(), pages, table, n)
    _check_attention(q.bfloat16(), pages, table, n, scale=3.7)
    if dtype != torch.bfloat16:
        exponent = torch.randint(-20, 21, pages.v_scale.shape, device="cuda").float()
        pages.v_scale.mul_(torch.exp2(exponent))
        pages.v_scale[3] = 0.0
        _check_attention(q.bfloat16(), pages, table, n)


def test_paged_attention_tiny_queries() -> None:
    """Query magnitudes far below and above fp16's range keep their scores."""
    pages = _pool(16, 2, 16, 64, torch.int8, seed=6)
    table, n = _tables([200, 10], 16, 16), torch.tensor([200, 10], dtype=torch.int32, device="cuda")
    q = torch.randn(2, 4, 64, device="cuda")
    for factor in (1e-20, 1e-6, 1e6):
        _check_attention((q * factor).bfloat16(), pages, table, n, scale=0.125 / factor)


def test_paged_attention_strides_and_packed_queries() -> None:
    pages = _pool(32, 2, 16, 64, torch.bfloat16, seed=7)
    lengths = [100, 37, 260]
    table = _tables(lengths, 16, 32)
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    packed = torch.randn(3, (8 + 4) * 64, device="cuda").bfloat16()
    q = packed[:, :8 * 64].view(3, 8, 64)
    want = ops.paged_attention(q.contiguous(), pages, table, n)
    assert torch.equal(ops.paged_attention(q, pages, table, n), want)
    assert torch.equal(ops.paged_attention(q.transpose(1, 2).contiguous().transpose(1, 2), pages, table, n), want)
    odd = torch.empty(3 * 8 * 64 + 1, device="cuda", dtype=torch.bfloat16)[1:].view(3, 8, 64).copy_(q)
    assert torch.equal(ops.paged_attention(odd, pages, table, n), want)
    wide = torch.full((3, table.shape[1] + 5), -1, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    assert torch.equal(ops.paged_attention(q, pages, wide[:, :table.shape[1]], n), want)


def test_paged_attention_repeats_bit_for_bit_and_in_graphs() -> None:
    lengths = [9000, 3, 700]
    num = sum(-(-n // 32) for n in lengths)
    pages = _pool(num, 4, 32, 128, torch.int8, seed=8)
    table, n = _tables(lengths, 32, num), torch.tensor(lengths, dtype=torch.int32, device="cuda")
    q = torch.randn(3, 16, 128, device="cuda").bfloat16()
    first = ops.paged_attention(q, pages, table, n)
    for _ in range(5):
        assert torch.equal(ops.paged_attention(q, pages, table, n), first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = ops.paged_attention(q, pages, table, n)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(again, first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = ops.paged_attention(q, pages, table, n)
    n.copy_(torch.tensor([8000, 0, 100], dtype=torch.int32))
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(captured, ops.paged_attention(q, pages, table, n))


def test_paged_attention_streams_side_by_side() -> None:
    """Calls that overlap on two streams do not share scratch memory."""
    lengths = [30000, 12000]
    num = sum(-(-n // 64) for n in lengths)
    pages = _pool(num, 2, 64, 128, torch.int8, seed=9)
    table, n = _tables(lengths, 64, num), torch.tensor(lengths, dtype=torch.int32, device="cuda")
    qs = [torch.randn(2, 8, 128, device="cuda").bfloat16() for _ in range(2)]
    want = [ops.paged_attention(q, pages, table, n) for q in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got: list[list[torch.Tensor]] = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ops.paged_attention(qs[i], pages, table, n))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


@pytest.mark.parametrize("dtype", [torch.int8, torch.bfloat16])
def test_offsets_beyond_32_bits(dtype) -> None:
    """Pages whose elements start behind 2^31 (and, in bf16, bytes behind 2^32)."""
    kvh, page, d = 8, 256, 128
    num = (1 << 31) // (kvh * page * d) + 6
    pages = ops.KVPages.allocate(num, kvh, page, d, dtype=dtype, device="cuda")
    far = [num - 1, num - 3, 0, num - 2]
    slots = torch.cat([torch.arange(page, device="cuda") + p * page for p in far])
    k, v = (torch.randn(len(far) * page, kvh, d, device="cuda").bfloat16() for _ in range(2))
    ops.kv_cache_write(pages, k, v, slots)
    small = ops.KVPages.allocate(len(far), kvh, page, d, dtype=dtype, device="cuda")
    ops.kv_cache_write(small, k, v, torch.arange(len(far) * page, device="cuda"))
    for a, b in zip(ops.kv_cache_read(pages, slots), ops.kv_cache_read(small, torch.arange(len(far) * page, device="cuda"))):
        assert torch.equal(a, b)
    q = torch.randn(1, 32, d, device="cuda").bfloat16()
    n = torch.tensor([len(far) * page - 3], dtype=torch.int32, device="cuda")
    got = ops.paged_attention(q, pages, torch.tensor([far], dtype=torch.int32, device="cuda"), n)
    want = ops.paged_attention(q, small, torch.arange(len(far), dtype=torch.int32, device="cuda")[None], n)
    assert torch.equal(got, want)


# --------------------------------------------------------------------------- writing and reading back


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("tokens,kvh,page", [(1, 1, 16), (5, 3, 16), (333, 12, 32), (1000, 8, 256)])
def test_cache_write_and_read_are_exact(dtype, d, tokens, kvh, page) -> None:
    """Every step is one IEEE operation, so bytes, scales and values equal the plain statement's."""
    num = tokens // page + 3
    got, want = (ops.KVPages.allocate(num, kvh, page, d, dtype=dtype, device="cuda") for _ in range(2))
    for p in (got, want):
        for t in (p.k, p.v):
            t.view(torch.uint8).zero_()
        if p.k_scale is not None:
            p.k_scale.zero_()
            p.v_scale.zero_()
    x = torch.randn(tokens, 2 * kvh + 1, d, device="cuda") * torch.exp2(torch.randint(-30, 30, (tokens, 2 * kvh + 1, 1), device="cuda").float())
    x[0, 0] = 0.0
    x[tokens // 2, kvh] = 1e-38
    packed = x.bfloat16()
    k, v = packed[:, :kvh], packed[:, kvh:2 * kvh]
    slots = torch.randperm(num * page, device="cuda")[:tokens]
    if tokens > 3:
        slots[1] = -1
        slots[2] = num * page
    ops.kv_cache_write(got, k, v, slots)
    ops.reference_kv_cache_write(want, k, v, slots)
    for a, b in ((got.k, want.k), (got.v, want.v)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    if dtype != torch.bfloat16:
        assert torch.equal(got.k_scale, want.k_scale) and torch.equal(got.v_scale, want.v_scale)
    for kind in (torch.int64, torch.int32):
        for a, b in zip(ops.kv_cache_read(got, slots.to(kind)), ops.reference_kv_cache_read(want, slots)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES[1:])
def test_cache_error_is_that_of_the_format(dtype) -> None:
    """int8: at most half a step of amax / 127 away; e4m3: at most 2^-4 of the value (2^-10 of a step below 2^-6)."""
    pages = ops.KVPages.allocate(16, 4, 16, 128, dtype=dtype, device="cuda")
    k, v = (torch.randn(256, 4, 128, device="cuda").bfloat16() for _ in range(2))
    slots = torch.arange(256, device="cuda")
    ops.kv_cache_write(pages, k, v, slots)
    for x, y in zip((k, v), ops.kv_cache_read(pages, slots)):
        x, y = x.double(), y.double()
        amax = x.abs().amax(-1, keepdim=True)
        bound = amax / 254 if dtype == torch.int8 else x.abs() / 16 + amax / 448 * 2.0**-10
        assert bool(((x - y).abs() <= 1.001 * bound + 2.0**-8 * x.abs()).all())


@pytest.mark.parametrize("dtype", DTYPES[1:])
def test_cache_rows_that_are_not_finite_read_back_as_nan(dtype) -> None:
    pages = ops.KVPages.allocate(2, 2, 16, 64, dtype=dtype, device="cuda")
    k, v = (torch.randn(4, 2, 64, device="cuda").bfloat16() for _ in range(2))
    k[1, 0, 3], k[2, 1, 60], v[3, 0, 0] = math.inf, math.nan, -math.inf
    slots = torch.arange(4, device="cuda")
    ops.kv_cache_write(pages, k, v, slots)
    rk, rv = ops.kv_cache_read(pages, slots)
    bad_k, bad_v = torch.zeros(4, 2, dtype=torch.bool, device="cuda"), torch.zeros(4, 2, dtype=torch.bool, device="cuda")
    bad_k[1, 0] = bad_k[2, 1] = bad_v[3, 0] = True
    assert torch.equal(torch.isnan(rk).all(-1), bad_k) and torch.equal(torch.isnan(rk).any(-1), bad_k)
    assert torch.equal(torch.isnan(rv).all(-1), bad_v) and torch.equal(torch.isnan(rv).any(-1), bad_v)


def test_cache_rows_of_other_orders_and_alignments() -> None:
    pages = ops.KVPages.allocate(4, 3, 16, 64, dtype=torch.int8, device="cuda")
    slots = torch.randperm(64, device="cuda")[:40]
    k, v = (torch.randn(40, 3, 64, device="cuda").bfloat16() for _ in range(2))
    ops.kv_cache_write(pages, k, v, slots)
    want = ops.kv_cache_read(pages, slots)
    for reorder in (lambda x: x.transpose(1, 2).contiguous().transpose(1, 2), lambda x: x.transpose(0, 1).contiguous().transpose(0, 1),
                    lambda x: torch.empty(x.numel() + 1, dtype=x.dtype, device="cuda")[1:].view(x.shape).copy_(x)):
        pages.k.zero_()
        ops.kv_cache_write(pages, reorder(k), reorder(v), torch.stack([slots, slots], 1)[:, 0])
        assert all(torch.equal(a, b) for a, b in zip(ops.kv_cache_read(pages, slots), want))
    packed = torch.zeros(40, (4 + 6) * 64, device="cuda", dtype=torch.bfloat16)
    columns = (packed[:, 4 * 64:7 * 64].view(40, 3, 64), packed[:, 7 * 64:].view(40, 3, 64))
    ops.kv_cache_read(pages, slots, out=columns)
    assert torch.equal(columns[0], want[0]) and torch.equal(columns[1], want[1]) and bool((packed[:, :4 * 64] == 0).all())


def test_empty_calls() -> None:
    pages = ops.KVPages.allocate(2, 2, 16, 64, dtype=torch.int8, device="cuda")
    none = torch.empty(0, 2, 64, device="cuda", dtype=torch.bfloat16)
    ops.kv_cache_write(pages, none, none, torch.empty(0, dtype=torch.int64, device="cuda"))
    assert ops.kv_cache_read(pages, torch.empty(0, dtype=torch.int64, device="cuda"))[0].shape == (0, 2, 64)
    q, n = torch.empty(0, 4, 64, device="cuda", dtype=torch.bfloat16), torch.empty(0, dtype=torch.int32, device="cuda")
    assert ops.paged_attention(q, pages, torch.empty(0, 3, dtype=torch.int32, device="cuda"), n).shape == (0, 4, 64)
    token, logprob = ops.sample_tokens(torch.empty(0, 50, device="cuda"), torch.empty(0, 50, device="cuda"))
    assert token.shape == (0,) and logprob.shape == (0,)


# --------------------------------------------------------------------------- sampling


def _logits(b: int, v: int, dtype: torch.dtype, seed: int) -> tuple[torch.Tensor, torch.Tensor]:
    gen = torch.Generator(device="cuda").manual_seed(seed)
    logits = 2.0 * torch.randn(b, v, device="cuda", generator=gen)
    if v > 64:
        apart = v // 32
        at = torch.randint(0, apart, (b, 32), device="cuda", generator=gen) + apart * torch.arange(32, device="cuda")
        logits.scatter_(1, at, 5.0 + 6.0 * torch.rand(b, 32, device="cuda", generator=gen))
    return logits.to(dtype), torch.empty(b, v, device="cuda").exponential_(generator=gen).clamp_(min=1e-30)


def _check_sample(logits, noise, **filters) -> torch.Tensor:
    token, logprob = ops.sample_tokens(logits, noise, **filters)
    want, want_logprob = ops.reference_sample_tokens(logits, noise, **filters, compute_dtype=torch.float64)
    assert torch.equal(token, want), (token != want).nonzero()
    some = want_logprob > -math.inf
    assert torch.equal(logprob > -math.inf, some)
    # an exponent of up to some hundreds and a sum of up to 2^18 terms in fp32: a few 2^-22 of their magnitude
    assert bool(((logprob.double() - want_logprob)[some].abs() <= 4e-6 * (1.0 + want_logprob[some].abs())).all())
    return token


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("v", [1, 2, 31, 1000, 4097, 32000, 50257, 128256])
@pytest.mark.parametrize("filters", [
    {}, {"temperature": 0.0}, {"temperature": 0.7}, {"top_k": 1}, {"top_k": 50, "temperature": 1.3}, {"top_p": 0.9}, {"top_p": 0.0},
    {"min_p": 0.05}, {"top_k": 40, "top_p": 0.8, "min_p": 0.02, "temperature": 0.9}, {"top_k": 1 << 20, "top_p": 0.999}, {"min_p": 1.0}])
def test_sample_tokens_matches_plain(dtype, v, filters) -> None:
    logits, noise = _logits(9, v, dtype, seed=v)
    _check_sample(logits, noise, **filters)


@pytest.mark.parametrize("b", [1, 3, 150, 700])
def test_sample_tokens_batches_with_values_per_row(b) -> None:
    logits, noise = _logits(b, 5003, torch.float32, seed=b)
    gen = torch.Generator(device="cuda").manual_seed(b)
    pick = lambda values: torch.tensor(values, device="cuda")[torch.randint(0, len(values), (b,), device="cuda", generator=gen)]  # noqa: E731
    _check_sample(logits, noise, temperature=pick([0.0, 0.5, 1.0, 2.0]), top_k=pick([0, 1, 7, 5003, 9999]).to(torch.int32),
                  top_p=pick([0.1, 0.5, 0.95, 1.0]), min_p=pick([0.0, 0.1]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("v", [8, 1003, 40000, 128256])
@pytest.mark.parametrize("filters", [{}, {"top_k": 5}, {"top_k": 700}, {"top_p": 0.5}, {"top_k": 1000, "top_p": 0.25}, {"temperature": 0.0}])
def test_sample_tokens_ties(dtype, v, filters) -> None:
    """Equal logits stay in the order of their index; half of them sit at each of two values."""
    noise = torch.empty(4, v, device="cuda").exponential_().clamp_(min=1e-30)
    logits = torch.zeros(4, v, device="cuda", dtype=dtype)
    _check_sample(logits, noise, **filters)
    logits[:, ::2] = -1.0
    _check_sample(logits, noise, **filters)
    logits[1::2, -1] = 3.0
    _check_sample(logits, noise, **filters)


@pytest.mark.parametrize("filters", [{}, {"top_k": 3}, {"top_p": 0.7}, {"min_p": 0.2}, {"temperature": 0.0}, {"temperature": 1e-30},
                                     {"temperature": 1e30, "top_p": 0.5}])
def test_sample_tokens_masked_infinite_and_nan_logits(filters) -> None:
    v = 3001
    logits, noise = _logits(8, v, torch.float32, seed=11)
    logits[0] = -math.inf  # nothing to draw
    logits[1] = -math.inf
    logits[1, 1234] = -5.0  # one token
    logits[2, 1:] = -math.inf
    logits[3, ::3] = math.nan
    logits[4] = math.nan
    logits[5, 7] = math.inf  # takes all
    logits[6, 5:] = torch.finfo(torch.float32).min  # a mask of the type's lowest value
    logits[7] = torch.finfo(torch.float32).min
    token = _check_sample(logits, noise, **filters)
    assert token[0] == -1 and token[4] == -1 and token[1] == 1234 and token[2] == 0 and token[5] == 7 and token[6] < 5


def test_sample_tokens_strides() -> None:
    logits, noise = _logits(6, 777, torch.bfloat16, seed=12)
    want = ops.sample_tokens(logits, noise, top_p=0.9)
    padded = torch.zeros(6, 800, device="cuda", dtype=torch.bfloat16)
    padded[:, 3:780] = logits
    turned = logits.t().contiguous().t()
    for x, e in ((padded[:, 3:780], noise), (turned, noise), (logits, noise.t().contiguous().t())):
        got = ops.sample_tokens(x, e, top_p=0.9)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    last = torch.randn(6, 3, 777, device="cuda").bfloat16()
    last[:, -1] = logits
    assert torch.equal(ops.sample_tokens(last[:, -1], noise, top_p=0.9)[0], want[0])


def test_sample_tokens_follows_the_distribution() -> None:
    """20000 draws of one row: every token's share is within five standard deviations of its probability."""
    b, v = 20000, 12
    row = torch.tensor([1.0, 0.0, -1.0, 2.0, 0.5, -2.0, 1.5, 0.0, -0.5, 0.25, -3.0, 1.0], device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(3)
    noise = torch.empty(b, v, device="cuda").exponential_(generator=gen)
    token, _ = ops.sample_tokens(row.expand(b, v), noise, temperature=0.8, top_k=6)
    p = torch.softmax((row / 0.8).double(), 0)
    p[torch.sort(row, descending=True, stable=True).indices[6:]] = 0.0
    p = p / p.sum()
    share = torch.bincount(token, minlength=v).double() / b
    assert bool(((share - p).abs() <= 5.0 * torch.sqrt(p * (1 - p) / b)).all())


# Batches whose rows are streamed by persistent blocks (more than one wave of clusters): shared rows, odd sizes, the largest vocabulary.
_MANY = [(151, 18500, torch.float32), (77, 50257, torch.float32), (39, 128256, torch.float32), (38, 262144, torch.float32),
         (75, 128256, torch.bfloat16), (160, 50257, torch.bfloat16), (38, 262143, torch.bfloat16), (700, 20011, torch.float32)]


@pytest.mark.parametrize("b, v, dtype", _MANY)
@pytest.mark.parametrize("filters", [{}, {"temperature": 0.0}, {"temperature": 0.6}, {"temperature": 40.0}, {"temperature": 0.01, "top_k": 1 << 20},
                                     {"temperature": 0.0, "top_k": 3, "top_p": 0.5}])
def test_sample_tokens_many_rows(b, v, dtype, filters) -> None:
    logits, noise = _logits(b, v, dtype, seed=b + v)
    token = _check_sample(logits, noise, **filters)
    per_row = torch.full((b,), filters.get("temperature", 1.0), device="cuda")
    assert torch.equal(token, ops.sample_tokens(logits, noise, **{**filters, "temperature": per_row})[0])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("filters", [{}, {"temperature": 0.0}, {"temperature": 500.0}])
def test_sample_tokens_many_rows_masked_infinite_and_nan(dtype, filters) -> None:
    b, v = 160, 40001
    logits, noise = _logits(b, v, dtype, seed=21)
    lowest = torch.finfo(dtype).min
    logits[0] = -math.inf
    logits[1] = -math.inf
    logits[1, 12345] = -5.0
    logits[2, 1:] = -math.inf
    logits[3, ::3] = math.nan
    logits[4] = math.nan
    logits[5, 7] = math.inf
    logits[6, 5:] = lowest
    logits[7] = lowest
    logits[8] = 3e6 * logits[8]  # too far apart for exponents without a reference
    logits[9] = logits[9] - 2.0**40
    logits[10, : v // 2] = -math.inf
    logits[11, v // 2 :] = lowest
    logits[12] = lowest
    logits[12, v - 1] = -1e4
    logits[b - 1] = -math.inf
    logits[b - 2, :-1] = -math.inf
    token = _check_sample(logits, noise, **filters)
    assert token[0] == -1 and token[4] == -1 and token[b - 1] == -1
    assert token[1] == 12345 and token[2] == 0 and token[5] == 7 and token[6] < 5 and token[12] == v - 1 and token[b - 2] == v - 1


@pytest.mark.parametrize("b, v, dtype", [(151, 50257, torch.float32), (150, 128256, torch.bfloat16), (1500, 36999, torch.float32), (2049, 36999, torch.float32)])
@pytest.mark.parametrize("share", [0.0, 0.02, 0.5, 1.0])
def test_sample_tokens_many_rows_with_values_per_row(b, v, dtype, share) -> None:
    """Rows that are cut, greedy rows and rows of which nothing is cut, of different temperatures, in one batch."""
    logits, noise = _logits(b, v, dtype, seed=b + 7)
    gen = torch.Generator(device="cuda").manual_seed(b)
    plain = torch.rand(b, device="cuda", generator=gen) < share
    pick = lambda values: torch.tensor(values, device="cuda")[torch.randint(0, len(values), (b,), device="cuda", generator=gen)]  # noqa: E731
    choose = lambda values, otherwise: torch.where(plain, torch.full_like(pick(values), otherwise), pick(values))  # noqa: E731
    _check_sample(logits, noise, temperature=torch.where(plain, pick([0.3, 1.0, 2.0, 9.0]), pick([0.0, 0.5, 1.0, 1e-4])),
                  top_k=choose([0, 7, 900], 0).to(torch.int32), top_p=choose([0.5, 0.95], 1.0), min_p=choose([0.0, 0.1], 0.0))
    if share == 1.0:
        temperature = pick([0.3, 1.0, 2.0, 9.0])
        _check_sample(logits, noise, temperature=temperature)
        _check_sample(logits, noise, temperature=0.7, top_p=torch.ones(b, device="cuda"), min_p=torch.zeros(b, device="cuda"))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("filters", [{}, {"temperature": 0.0}])
def test_sample_tokens_many_rows_ties_and_strides(dtype, filters) -> None:
    b, v = 160, 40001
    logits, noise = torch.zeros(b, v + 8, device="cuda", dtype=dtype)[:, 3 : v + 3], torch.ones(b, v + 6, device="cuda")[:, 1 : v + 1]
    assert torch.equal(_check_sample(logits, noise, **filters), torch.zeros(b, dtype=torch.int64, device="cuda"))  # the first among equals
    at = torch.randint(1, v - 1, (b,), device="cuda")
    logits.scatter_(1, at[:, None], 1.0)
    logits.scatter_(1, at[:, None] + 1, 1.0)
    assert torch.equal(_check_sample(logits, noise, **filters), at)
    values, luck = _logits(b, v, dtype, seed=22)
    want = ops.sample_tokens(values, luck, **filters)
    logits.copy_(values)
    noise.copy_(luck)
    for x, e in ((logits, noise), (values, noise), (logits, luck), (values.t().contiguous().t(), luck)):
        got = ops.sample_tokens(x, e, **filters)
        assert torch.equal(got[0], want[0])
        assert bool(((got[1] - want[1]).abs() <= 4e-6 * (1.0 + want[1].abs())).all())


def test_sample_tokens_many_rows_on_streams_and_in_graphs() -> None:
    inputs = [_logits(b, v, torch.float32, seed=b) for b, v in ((77, 50257), (151, 18500))]
    want = [ops.sample_tokens(*x) for x in inputs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        got = []
        for stream, x in zip(streams, inputs, strict=True):
            with torch.cuda.stream(stream):
                got.append(ops.sample_tokens(*x))
        torch.cuda.synchronize()
        assert all(torch.equal(g, w) for gs, ws in zip(got, want, strict=True) for g, w in zip(gs, ws, strict=True))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = [ops.sample_tokens(*x) for x in inputs]
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(g, w) for gs, ws in zip(got, want, strict=True) for g, w in zip(gs, ws, strict=True))


def test_sample_tokens_many_rows_with_values_per_row_in_stream_order() -> None:
    """Two launches share such a batch: what follows them on the stream, or in a graph, finds both ended."""
    b, v = 160, 50257
    logits, noise = _logits(b, v, torch.float32, seed=31)
    rows = torch.arange(b, device="cuda")
    for cut in (rows < 0, rows % 2 == 0, rows == b - 1, rows == 0, rows < b - 1, rows >= 0):
        top_k = torch.where(cut, 40, 0).to(torch.int32)
        want = [x.clone() for x in ops.sample_tokens(logits, noise, top_k=top_k)]
        assert torch.equal(want[0], ops.reference_sample_tokens(logits, noise, 1.0, top_k, 1.0, 0.0, compute_dtype=torch.float64)[0])
        values = torch.empty_like(logits)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            values.copy_(logits)
            got = ops.sample_tokens(values, noise, top_k=top_k)
            copies = [x.clone() for x in got]
            values.fill_(-math.inf)
        for _ in range(3):
            graph.replay()
        assert all(torch.equal(x, y) for x, y in zip(copies, want, strict=True))
        for _ in range(3):
            values.copy_(logits)
            got = ops.sample_tokens(values, noise, top_k=top_k)
            values.fill_(math.nan)
            assert all(torch.equal(x, y) for x, y in zip(got, want, strict=True))


# --------------------------------------------------------------------------- refusals


def test_refusals() -> None:
    pages = ops.KVPages.allocate(4, 2, 16, 64, dtype=torch.int8, device="cuda")
    q = torch.randn(2, 4, 64, device="cuda").bfloat16()
    table, n = torch.zeros(2, 3, dtype=torch.int32, device="cuda"), torch.ones(2, dtype=torch.int32, device="cuda")
    for bad in ((q[..., :32], pages, table, n), (q[:, :3], pages, table, n), (q.float(), pages, table, n), (q, pages, table.long(), n),
                (q, pages, table, n.long()), (q, pages, table[:1], n), (q, pages, table, n[:1]), (q, pages, table.cpu(), n), (q[0], pages, table, n)):
        with pytest.raises(ConfigurationError):
            ops.paged_attention(*bad)
    with pytest.raises(UnsupportedFeatureError):
        ops.paged_attention(q.clone().requires_grad_(), pages, table, n)
    rows, slots = torch.zeros(3, 2, 64, device="cuda", dtype=torch.bfloat16), torch.arange(3, device="cuda")
    for bad in ((rows[:, :1], rows, slots), (rows, rows[:2], slots), (rows, rows, slots[:2]), (rows, rows, slots.float()),
                (rows.float(), rows, slots), (rows, rows, slots.cpu()), (rows, rows, slots[None])):
        with pytest.raises(ConfigurationError):
            ops.kv_cache_write(pages, *bad)
    with pytest.raises(UnsupportedFeatureError):
        ops.kv_cache_write(pages, rows.clone().requires_grad_(), rows, slots)
    with pytest.raises(ConfigurationError):
        ops.kv_cache_read(pages, slots[None])
    with pytest.raises(RuntimeError):  # rows that no 16-byte store can take
        ops.kv_cache_read(pages, slots, out=(rows.transpose(1, 2).contiguous().transpose(1, 2), rows))
    for shape, kind in (((4, 2, 15, 64), torch.int8), ((4, 2, 24, 64), torch.int8), ((4, 2, 512, 64), torch.int8), ((4, 2, 16, 80), torch.int8),
                        ((4, 2, 16, 64), torch.float16)):
        with pytest.raises(ConfigurationError):
            ops.KVPages.allocate(*shape, dtype=kind, device="cuda")
    with pytest.raises(ConfigurationError):
        ops.KVPages(pages.k, pages.v)
    with pytest.raises(ConfigurationError):
        ops.KVPages(pages.k, pages.v, pages.k_scale[:2], pages.v_scale)
    logits, noise = torch.randn(2, 9, device="cuda"), torch.ones(2, 9, device="cuda")
    for bad in ((logits[0], noise[0]), (logits, noise[:, :8]), (logits.half(), noise), (logits, noise.double()), (logits, noise.cpu()),
                (logits[:, :0], noise[:, :0])):
        with pytest.raises(ConfigurationError):
            ops.sample_tokens(*bad)
    for bad in ({"temperature": -1.0}, {"top_p": 1.5}, {"min_p": -0.1}, {"top_k": -1}, {"temperature": math.nan},
                {"top_k": torch.ones(2, device="cuda")}, {"top_p": torch.ones(3, device="cuda")}, {"min_p": torch.ones(2)}):
        with pytest.raises(ConfigurationError):
            ops.sample_tokens(logits, noise, **bad)
