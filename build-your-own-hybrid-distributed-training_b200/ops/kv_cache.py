"""A paged key/value cache and attention of new tokens over it: what answering with a trained decoder reads and writes.

A layer's cache is a pool of pages (:class:`KVPages`), each holding ``page_size`` consecutive tokens of
one sequence for every key/value head: ``[pages, Hkv, page_size, D]`` for the keys and the same for the
values, so the rows that one head's attention reads from a page lie next to each other.  A token's
place is its *slot*, ``page * page_size + row``.  The pool holds bf16, or 8 bits per element (``int8`` or
``float8_e4m3fn``) with one fp32 scale per token and head:

* ``kv_cache_write(pages, k, v, slots)`` quantises rows as it stores them,
* ``kv_cache_read(pages, slots)`` gives them back as bf16,
* ``paged_attention(q, pages, block_table, lengths)`` attends with one query token per sequence
  to the sequence's cached tokens; row ``i`` of a block table lists the pages of sequence ``i``.

These ops have no gradient: they serve a model that has been trained (training runs
:func:`~hybrid_training.ops.attention`).  The kernels are ``csrc/kv_cache.cu`` and
``csrc/paged_attention.cu``; the reference has no counterpart (its model recomputes the whole
sequence, ``src/hybrid_training/models/transformer.py:253-295``).
"""

from __future__ import annotations

import math
from dataclasses import dataclass

import torch

from ..errors import ConfigurationError, UnsupportedFeatureError, format_error
from ._ext import extension

__all__ = ["KVPages", "kv_cache_read", "kv_cache_write", "paged_attention", "reference_kv_cache_read", "reference_kv_cache_write",
           "reference_paged_attention"]

_LARGEST = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
_SMALLEST_SCALE = 2.0**-64


def _refuse(op: str, problem: str, expected: object, observed: object, resolution: str) -> ConfigurationError:
    return ConfigurationError(format_error(f"ops.{op}", problem, expected=expected, observed=observed, resolution=resolution))


@dataclass(frozen=True)
class KVPages:
    """The key/value pool of one layer; see the module docstring for the layout."""

    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor | None = None
    v_scale: torch.Tensor | None = None

    def __post_init__(self) -> None:
        k, v = self.k, self.v
        if k.dim() != 4 or v.shape != k.shape or v.dtype != k.dtype or v.device != k.device or not (k.is_contiguous() and v.is_contiguous()):
            raise _refuse("KVPages", "the key and value pools must be alike", "two contiguous [pages, Hkv, page_size, D] tensors of one type",
                          f"{tuple(k.shape)} {k.dtype} and {tuple(v.shape)} {v.dtype}", "allocate them with KVPages.allocate")
        page = k.shape[2]
        if page < 16 or page > 256 or page & (page - 1):
            raise _refuse("KVPages", "unsupported page size", "16, 32, 64, 128 or 256 tokens", page, "choose one of these page sizes")
        if k.is_cuda and k.shape[3] not in (64, 128):
            raise _refuse("KVPages", "unsupported head size on CUDA", "64 or 128", k.shape[3], "use a model with one of these head sizes")
        quantised = k.dtype in _LARGEST
        if not quantised and k.dtype != torch.bfloat16 and (k.is_cuda or not k.is_floating_point()):
            raise _refuse("KVPages", "unsupported cache type", "bfloat16, int8 or float8_e4m3fn", k.dtype, "choose one of these types")
        for s in (self.k_scale, self.v_scale):
            if quantised != (s is not None):
                raise _refuse("KVPages", "scales go with 8-bit pools", "scales" if quantised else "no scales",
                              "none" if s is None else "scales", "pass one scale tensor each for keys and values of an 8-bit pool")
            if s is not None and (s.shape != k.shape[:3] or s.dtype != torch.float32 or s.device != k.device or not s.is_contiguous()):
                raise _refuse("KVPages", "a scale tensor does not fit the pool", f"contiguous float32 {tuple(k.shape[:3])}",
                              f"{s.dtype} {tuple(s.shape)}", "allocate it with KVPages.allocate")

    @classmethod
    def allocate(cls, num_pages: int, num_kv_heads: int, page_size: int, head_dim: int, *, dtype: torch.dtype = torch.bfloat16,
                 device: torch.device | str | None = None) -> KVPages:
        """An empty pool (its contents are undefined until written)."""
        shape = (num_pages, num_kv_heads, page_size, head_dim)
        k, v = (torch.empty(shape, dtype=dtype, device=device) for _ in range(2))
        if dtype not in _LARGEST:
            return cls(k, v)
        ks, vs = (torch.empty(shape[:3], dtype=torch.float32, device=device) for _ in range(2))
        return cls(k, v, ks, vs)

    @property
    def num_pages(self) -> int:
        return self.k.shape[0]

    @property
    def num_kv_heads(self) -> int:
        return self.k.shape[1]

    @property
    def page_size(self) -> int:
        return self.k.shape[2]

    @property
    def head_dim(self) -> int:
        return self.k.shape[3]


def _check_rows(op: str, pages: KVPages, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
    want = (slots.shape[0] if slots.dim() == 1 else -1, *pages.k.shape[1::2])
    if k.shape != want or v.shape != want:
        raise _refuse(op, "the rows do not fit the pool and the slots", f"k and v of shape {want}, one slot per token",
                      f"{tuple(k.shape)}, {tuple(v.shape)} and slots {tuple(slots.shape)}", "pass [T, Hkv, D] rows and [T] slots")
    if slots.dtype not in (torch.int64, torch.int32) or not (slots.device == k.device == v.device == pages.k.device):
        raise _refuse(op, "slots must be integers, and everything on the pool's device", f"int32 or int64 on {pages.k.device}",
                      f"{slots.dtype} on {slots.device}, rows on {k.device}", "convert or move them")
    wanted = torch.bfloat16 if k.is_cuda else k.dtype
    if k.dtype != wanted or v.dtype != wanted or not k.is_floating_point():
        raise _refuse(op, "unsupported row type", "bfloat16 keys and values", f"{k.dtype} and {v.dtype}", "cast them to bfloat16")


def _no_gradient(op: str, *tensors: torch.Tensor) -> None:
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise UnsupportedFeatureError(format_error(f"ops.{op}", "this op has no gradient", expected="inputs that need no gradient",
                                                   observed="requires_grad=True", resolution="call it under torch.no_grad()"))


def _flat(pool: torch.Tensor) -> torch.Tensor:
    """fp8 pools as bytes: indexing does not need the type."""
    return pool.view(torch.uint8) if pool.dtype == torch.float8_e4m3fn else pool


def reference_kv_cache_write(pages: KVPages, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
    """Plain PyTorch statement of :func:`kv_cache_write` (the CPU path)."""
    page = pages.page_size
    stored = (slots >= 0) & (slots < pages.num_pages * page)
    slots = slots[stored].long()
    at, row = torch.div(slots, page, rounding_mode="floor"), slots % page
    for x, pool, scales in ((k, pages.k, pages.k_scale), (v, pages.v, pages.v_scale)):
        x = x[stored]
        if scales is None:
            pool[at, :, row] = x.to(pool.dtype)
            continue
        xf = x.float()
        top = xf.abs().amax(-1)
        scale = torch.where(top < math.inf, (top * (1.0 / _LARGEST[pool.dtype])).clamp(min=_SMALLEST_SCALE), math.nan)
        y = xf * (1.0 / scale)[..., None]
        y = torch.round(y) if pool.dtype == torch.int8 else y
        y = torch.where(torch.isnan(scale)[..., None], 0.0, y.clamp(-_LARGEST[pool.dtype], _LARGEST[pool.dtype]))
        _flat(pool)[at, :, row] = _flat(y.to(pool.dtype))
        scales[at, :, row] = scale


def reference_kv_cache_read(pages: KVPages, slots: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> tuple[torch.Tensor, torch.Tensor]:
    """Plain PyTorch statement of :func:`kv_cache_read` (the CPU path)."""
    page = pages.page_size
    stored = (slots >= 0) & (slots < pages.num_pages * page)
    safe = torch.where(stored, slots, 0).long()
    at, row = torch.div(safe, page, rounding_mode="floor"), safe % page
    out = []
    for pool, scales in ((pages.k, pages.k_scale), (pages.v, pages.v_scale)):
        x = _flat(pool)[at, :, row].view(pool.dtype)
        if scales is not None:
            x = x.float() * scales[at, :, row][..., None]
        out.append(torch.where(stored[:, None, None], x.to(dtype), 0.0))
    return out[0], out[1]


def reference_paged_attention(q: torch.Tensor, pages: KVPages, block_table: torch.Tensor, lengths: torch.Tensor, *,
                              scale: float | None = None, compute_dtype: torch.dtype = torch.float32) -> tuple[torch.Tensor, torch.Tensor]:
    """Plain PyTorch statement of :func:`paged_attention` (the CPU path); returns ``(out, lse)``."""
    b, h, d = q.shape
    kvh, page = pages.num_kv_heads, pages.page_size
    n = block_table.shape[1] * page
    held = (block_table >= 0) & (block_table < pages.num_pages)
    valid = (torch.arange(n, device=q.device)[None] < lengths[:, None]) & held.repeat_interleave(page, 1)
    table = torch.where(held, block_table, 0).long()

    def rows(pool: torch.Tensor, scales: torch.Tensor | None) -> torch.Tensor:
        x = _flat(pool)[table].view(pool.dtype).to(compute_dtype)
        if scales is not None:
            x = x * scales[table][..., None].to(compute_dtype)
        x = x.transpose(1, 2).reshape(b, kvh, n, d)
        return torch.where(valid[:, None, :, None], x, 0.0)

    scale = 1.0 / math.sqrt(d) if scale is None else scale
    qg = q.to(compute_dtype).reshape(b, kvh, h // kvh, d)
    scores = torch.where(valid[:, None, None, :], qg @ rows(pages.k, pages.k_scale).transpose(-1, -2) * scale, -math.inf)
    empty = ~valid.any(-1)[:, None, None, None]
    top = torch.where(empty, 0.0, scores.amax(-1, keepdim=True)) if n else scores.new_zeros(b, kvh, h // kvh, 1)
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    out = torch.where(empty, 0.0, (p @ rows(pages.v, pages.v_scale)) / total)
    lse = top + torch.log(total)
    return out.reshape(b, h, d).to(q.dtype if compute_dtype == torch.float32 else compute_dtype), lse.reshape(b, h)


def _check_attention(q: torch.Tensor, pages: KVPages, block_table: torch.Tensor, lengths: torch.Tensor) -> None:
    kvh = pages.num_kv_heads
    if q.dim() != 3 or q.shape[2] != pages.head_dim or q.shape[1] % kvh or q.shape[1] == 0:
        raise _refuse("paged_attention", "the queries do not fit the pool", f"[B, a multiple of {kvh}, {pages.head_dim}]", tuple(q.shape),
                      "pass one token per sequence with the pool's head layout")
    b = q.shape[0]
    if block_table.dim() != 2 or block_table.shape[0] != b or lengths.shape != (b,):
        raise _refuse("paged_attention", "every query needs a row of the block table and a length", f"[{b}, W] and [{b}]",
                      f"{tuple(block_table.shape)} and {tuple(lengths.shape)}", "pass one row and one length per sequence")
    if block_table.dtype != torch.int32 or lengths.dtype != torch.int32 or not (q.device == block_table.device == lengths.device == pages.k.device):
        raise _refuse("paged_attention", "the block table and the lengths must be int32, and everything on one device", f"int32 on {pages.k.device}",
                      f"{block_table.dtype} and {lengths.dtype} on {block_table.device} and {lengths.device}, q on {q.device}", "convert or move them")
    if q.is_cuda and q.dtype != torch.bfloat16:
        raise _refuse("paged_attention", "unsupported query type", "bfloat16", q.dtype, "cast q to bfloat16")
    _no_gradient("paged_attention", q)


# On CUDA the native entry points check every argument themselves, in the time that a check or two takes here.  Where
# one of them refuses, the checks of this module say why in the framework's words.


def kv_cache_write(pages: KVPages, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
    """Store the rows ``k``, ``v`` ``[T, Hkv, D]`` (any strides) at ``slots`` ``[T]``, quantised as the pool holds them.

    The slots of one call are distinct.  A slot outside the pool stores nothing: ``-1`` marks a row of padding.
    A row with an infinity or a NaN in an 8-bit pool reads back as NaN.
    """
    if pages.k.is_cuda:
        try:
            return extension().kv_cache_write(pages.k, pages.v, pages.k_scale, pages.v_scale, k, v, slots)
        except RuntimeError:
            _check_rows("kv_cache_write", pages, k, v, slots)
            _no_gradient("kv_cache_write", k, v)
            raise
    _check_rows("kv_cache_write", pages, k, v, slots)
    _no_gradient("kv_cache_write", k, v)
    reference_kv_cache_write(pages, k, v, slots)


def kv_cache_read(pages: KVPages, slots: torch.Tensor, out: tuple[torch.Tensor, torch.Tensor] | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """The rows at ``slots`` ``[T]`` as bf16 keys and values ``[T, Hkv, D]``; zeros for slots outside the pool.

    ``out`` takes a pair of tensors to write into, whose rows may be strided (the key and value columns of a
    packed QKV tensor, for one).
    """
    k, v = (None, None) if out is None else out
    if pages.k.is_cuda:
        try:
            return extension().kv_cache_read(pages.k, pages.v, pages.k_scale, pages.v_scale, slots, k, v)
        except RuntimeError:
            if slots.dim() != 1:
                raise _refuse("kv_cache_read", "slots must be a vector", "[T]", tuple(slots.shape), "flatten them") from None
            if k is not None and v is not None:
                _check_rows("kv_cache_read", pages, k, v, slots)
            raise
    if slots.dim() != 1:
        raise _refuse("kv_cache_read", "slots must be a vector", "[T]", tuple(slots.shape), "flatten them")
    if k is None or v is None:
        return reference_kv_cache_read(pages, slots)
    _check_rows("kv_cache_read", pages, k, v, slots)
    for o, x in zip((k, v), reference_kv_cache_read(pages, slots, k.dtype)):
        o.copy_(x)
    return k, v


def paged_attention(q: torch.Tensor, pages: KVPages, block_table: torch.Tensor, lengths: torch.Tensor, *, scale: float | None = None,
                    return_lse: bool = False) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """Attention of one query token per sequence, ``q`` ``[B, H, D]``, over its ``lengths[b]`` cached tokens.

    ``block_table`` ``[B, W]`` (int32) lists each sequence's pages in order; token ``t`` is row ``t % page_size`` of
    page ``block_table[b, t // page_size]``.  ``H`` is a multiple of the pool's ``Hkv`` heads: query head ``h`` reads
    key/value head ``h // (H / Hkv)``.  ``scale`` defaults to ``1 / sqrt(D)``.  Returns ``[B, H, D]`` in the type of
    ``q``, and with ``return_lse`` the fp32 log-sum-exp of the scores ``[B, H]`` as well.  A sequence of length 0
    gives zeros and ``-inf``; lengths beyond the table are cut to it, and tokens of pages outside the pool count as
    masked, as do whatever values lie behind a sequence's length.
    """
    if q.is_cuda:
        try:
            out, lse = extension().paged_attention(q, pages.k, pages.v, pages.k_scale, pages.v_scale, block_table, lengths, scale, return_lse)
        except RuntimeError:
            _check_attention(q, pages, block_table, lengths)
            raise
    else:
        _check_attention(q, pages, block_table, lengths)
        out, lse = reference_paged_attention(q, pages, block_table, lengths, scale=scale)
    return (out, lse) if return_lse else out
