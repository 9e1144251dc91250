"""Sampling of the next token from logits: temperature, top-k, top-p and min-p from given uniform numbers (sm_100a).

The decode step ends in a greedy argmax; this draws from the logits it returns.  For each row, with
``w_i = exp((l_i - max l) / temperature)`` and tokens ordered by logit (equal ones by index):

1. the first ``top_k`` tokens stay,
2. of those the shortest prefix that holds ``top_p`` of their weight,
3. of those the ones with ``w_i >= min_p`` (as likely as ``min_p`` times the most likely token),

and the token drawn is the lowest index at which the running sum of kept weights, in index order, exceeds ``uniform``
times their sum.  The most likely token always stays.  NaN and ``-inf`` are never drawn; a row of nothing else gives
id 0 (logprob NaN).  Weights are 64-bit integers relative to the row's largest, with at least 44 fractional bits: the
same call gives the same ids whatever else runs.  A token keeps at least one unit unless its weight underflows a
double (below ``e**-707``), so masks of a type's lowest value are never drawn either.
"""
from __future__ import annotations

import torch

from .._cabi import load_ops

load_ops()

__all__ = ["MAX_VOCAB", "sample", "Sampler"]

MAX_VOCAB = 262144


@torch.library.register_fake("prime_sampling::sample")
def _sample_fake(logits, uniform, temperature, temperature_value, top_k, top_k_value, top_p, top_p_value, min_p, min_p_value):
    return torch.empty((logits.shape[0],), dtype=torch.int64, device=logits.device)


@torch.library.register_fake("prime_sampling::sample_out")
def _sample_out_fake(logits, uniform, temperature, temperature_value, top_k, top_k_value, top_p, top_p_value, min_p,
                     min_p_value, ids, logprobs):
    return None


_sample = torch.ops.prime_sampling.sample.default
_sample_out = torch.ops.prime_sampling.sample_out.default


def _check(temperature, top_k, top_p, min_p):
    if not 0 <= temperature < float("inf"):
        raise ValueError(f"temperature must be finite and not negative, got {temperature}")
    if top_k < 0:
        raise ValueError(f"top_k must not be negative (0: off), got {top_k}")
    if not 0 < top_p <= 1:
        raise ValueError(f"top_p must be in (0, 1], got {top_p}")
    if not 0 <= min_p <= 1:
        raise ValueError(f"min_p must be in [0, 1], got {min_p}")


def sample(logits, uniform, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, out=None, return_logprobs: bool = False):
    """Draw one id per row of ``logits`` (bf16, fp16 or fp32 ``[rows, vocab]``, unit last stride) with the uniform numbers
    ``uniform`` (fp32 ``[rows]`` in [0, 1)).

    Each setting is a number for all rows or a tensor ``[rows]`` on the device (``top_k`` int32, the others fp32).
    ``temperature`` 0 takes the largest logit (lowest index among equals); ``top_k`` 0, ``top_p`` 1 and ``min_p`` 0 are
    off.  In a tensor, values outside those ranges mean: temperature negative or NaN 0, top_k negative off, top_p above 1
    off and below 0 the most likely token only, min_p negative off.  Returns int64 ids ``[rows]`` (written to ``out``
    where given), with ``return_logprobs`` ``(ids, logprobs)``: the log of each drawn id's share of the kept weight."""
    t = k = p = m = None
    if isinstance(temperature, torch.Tensor):
        t, temperature = temperature, 1.0
    if isinstance(top_k, torch.Tensor):
        k, top_k = top_k, 0
    if isinstance(top_p, torch.Tensor):
        p, top_p = top_p, 1.0
    if isinstance(min_p, torch.Tensor):
        m, min_p = min_p, 0.0
    _check(temperature, top_k, top_p, min_p)
    if out is None:
        if not return_logprobs:
            return _sample(logits, uniform, t, temperature, k, top_k, p, top_p, m, min_p)
        out = torch.empty((logits.shape[0],), dtype=torch.int64, device=logits.device)
    lp = torch.empty((logits.shape[0],), dtype=torch.float32, device=logits.device) if return_logprobs else None
    _sample_out(logits, uniform, t, temperature, k, top_k, p, top_p, m, min_p, out, lp)
    return (out, lp) if return_logprobs else out


class Sampler:
    """Settings of :func:`sample` with a generator for its uniform numbers, as ``decode.DecodeSession`` takes them."""

    def __init__(self, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, generator: torch.Generator | None = None):
        self.settings = {"temperature": temperature, "top_k": top_k, "top_p": top_p, "min_p": min_p}
        _check(*(0 if isinstance(v, torch.Tensor) and n != "top_p" else (1 if isinstance(v, torch.Tensor) else v)
                 for n, v in self.settings.items()))
        self.generator = generator

    def __call__(self, logits, out=None, return_logprobs: bool = False):
        uniform = torch.rand((logits.shape[0],), generator=self.generator, device=logits.device)
        return sample(logits, uniform, out=out, return_logprobs=return_logprobs, **self.settings)
