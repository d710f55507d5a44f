"""Choosing the next token from logits and given random numbers (temperature, top-k, top-p, min-p).

``sample_tokens`` draws by an exponential race: with ``noise`` independent and exponentially
distributed (``torch.empty(B, V).exponential_()``), the token with the largest ``weight / noise`` among
those that the filters leave is a draw from their softmax.  The random numbers are the caller's, so a
draw can be repeated, and no rounding of a long cumulative sum decides it.  The kernels are
``csrc/sampling.cu`` and ``csrc/sampling_stream.cu``; the reference has no counterpart.
"""

from __future__ import annotations

import math

import torch

from ..errors import ConfigurationError, UnsupportedFeatureError, format_error
from ._ext import extension

__all__ = ["reference_sample_tokens", "sample_tokens"]

Number = float | int | torch.Tensor
_MOST_TOKENS = 1 << 18  # vocabulary of the kernel


def _refuse(problem: str, expected: object, observed: object, resolution: str) -> ConfigurationError:
    return ConfigurationError(format_error("ops.sample_tokens", problem, expected=expected, observed=observed, resolution=resolution))


def _no_gradient(logits: torch.Tensor) -> None:
    if torch.is_grad_enabled() and logits.requires_grad:
        raise UnsupportedFeatureError(format_error("ops.sample_tokens", "a drawn token has no gradient, and its log-probability here none either",
                                                   expected="logits that need no gradient", observed="requires_grad=True",
                                                   resolution="call it under torch.no_grad(); for a log-probability with a gradient take "
                                                              "torch.log_softmax of the logits at the tokens that it returns"))


def _check(logits: torch.Tensor, noise: torch.Tensor, filters: dict[str, Number]) -> None:
    if logits.dim() != 2 or logits.shape[1] == 0 or noise.shape != logits.shape or noise.dtype != torch.float32 or noise.device != logits.device:
        raise _refuse("logits and noise must be alike", "[B, V] logits and fp32 noise of the same shape and device",
                      f"{tuple(logits.shape)} and {noise.dtype} {tuple(noise.shape)} on {noise.device}", "draw one Exp(1) number per logit")
    if logits.dtype not in (torch.bfloat16, torch.float32):
        raise _refuse("unsupported logit type", "bfloat16 or float32", logits.dtype, "cast the logits")
    if logits.is_cuda and logits.shape[1] > _MOST_TOKENS:
        raise _refuse("the vocabulary is too large", f"at most {_MOST_TOKENS} tokens", logits.shape[1], "sample from slices of it")
    for name, value in filters.items():
        if isinstance(value, torch.Tensor):
            dtype = torch.int32 if name == "top_k" else torch.float32
            if value.shape != logits.shape[:1] or value.dtype != dtype or value.device != logits.device or not value.is_contiguous():
                raise _refuse(f"{name} does not fit the logits", f"a number or a contiguous {dtype} tensor [{logits.shape[0]}] on {logits.device}",
                              f"{value.dtype} {tuple(value.shape)} on {value.device}", "pass one value per row, or one number")
        elif not value >= 0 or (name in ("top_p", "min_p") and value > 1):
            raise _refuse(f"{name} is out of range", "0 to 1" if name in ("top_p", "min_p") else "0 or more", value, "choose a value in range")


def reference_sample_tokens(logits: torch.Tensor, noise: torch.Tensor, temperature: Number = 1.0, top_k: Number = 0, top_p: Number = 1.0,
                            min_p: Number = 0.0, *, compute_dtype: torch.dtype = torch.float32) -> tuple[torch.Tensor, torch.Tensor]:
    """Plain PyTorch statement of :func:`sample_tokens` (the CPU path)."""
    b, v = logits.shape
    col = lambda x: (x if isinstance(x, torch.Tensor) else torch.full((b,), x, device=logits.device))[:, None]  # noqa: E731
    temperature, top_k, top_p, min_p = (col(x) for x in (temperature, top_k, top_p, min_p))
    z = logits.to(compute_dtype)
    z = torch.where(torch.isnan(z), -math.inf, z)
    best = z.amax(-1, keepdim=True)
    empty = best[:, 0] == -math.inf
    greedy = ~(temperature > 0)
    x = torch.where(z == best, 0.0, torch.where(z == -math.inf, -math.inf, (z - best) / torch.where(greedy, 1.0, temperature.to(compute_dtype))))
    w = torch.exp(x)
    ranked, order = torch.sort(z, dim=-1, descending=True, stable=True)
    rank = torch.arange(v, device=logits.device)[None]
    keep = (rank < top_k) | (top_k <= 0)
    ws = torch.gather(w, 1, order)
    mass = torch.where(keep, ws, 0.0)
    before = torch.cumsum(mass, -1) - mass
    keep &= (before < top_p.to(compute_dtype) * mass.sum(-1, keepdim=True)) | (top_p >= 1)
    keep &= (ws >= min_p) & ~greedy & (ranked > -math.inf)
    keep |= rank == 0
    # a random number that is none loses to every other, but still names a token
    score = torch.where(keep, torch.nan_to_num(ws / torch.gather(noise.to(compute_dtype), 1, order), nan=-0.5, posinf=math.inf), -1.0)
    token = torch.where(score == score.amax(-1, keepdim=True), order, v).amin(-1)
    logprob = torch.gather(x, 1, token.clamp(max=v - 1)[:, None])[:, 0] - torch.log(w.sum(-1))
    return torch.where(empty, -1, token), torch.where(empty, -math.inf, logprob)


def sample_tokens(logits: torch.Tensor, noise: torch.Tensor, *, temperature: Number = 1.0, top_k: Number = 0, top_p: Number = 1.0,
                  min_p: Number = 0.0) -> tuple[torch.Tensor, torch.Tensor]:
    """One token per row of ``logits`` ``[B, V]`` (bf16 or fp32), drawn with ``noise`` ``[B, V]`` (fp32, positive, Exp(1)).

    The filters apply in this order: ``top_k`` keeps that many tokens of the largest logits (0: all), ``top_p`` the
    smallest prefix of those that holds this share of their probability (1: all), ``min_p`` drops tokens less
    probable than this share of the most probable one.  The most probable token always stays, the lower index wins
    ties, and ``temperature`` 0 takes it without drawing.  Each of the four is a number or one value per row
    (fp32; ``top_k`` int32); a NaN among a tensor's values leaves the most probable token.  Returns ``(tokens int64 [B], logprobs fp32 [B])``; the log-probability is that of the whole
    row at this temperature (at 1 where the temperature is 0), before any filter.  Logits of ``-inf`` or NaN cannot
    be drawn; a row without any other gives ``-1`` and ``-inf``.  Neither result has a gradient: logits that need one are
    refused outside ``torch.no_grad()``.
    """
    if logits.is_cuda:
        try:
            # a filter is a tensor with a value per row, or a number
            t = (temperature, 1.0) if isinstance(temperature, torch.Tensor) else (None, temperature)
            k = (top_k, 0) if isinstance(top_k, torch.Tensor) else (None, top_k)
            p = (top_p, 1.0) if isinstance(top_p, torch.Tensor) else (None, top_p)
            m = (min_p, 0.0) if isinstance(min_p, torch.Tensor) else (None, min_p)
            return extension().sample_tokens(logits, noise, *t, *k, *p, *m)
        except RuntimeError:
            _check(logits, noise, {"temperature": temperature, "top_k": top_k, "top_p": top_p, "min_p": min_p})
            _no_gradient(logits)
            raise
    _check(logits, noise, {"temperature": temperature, "top_k": top_k, "top_p": top_p, "min_p": min_p})
    _no_gradient(logits)
    return reference_sample_tokens(logits, noise, temperature, top_k, top_p, min_p)
