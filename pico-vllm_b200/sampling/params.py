"""Sampling options, with the reference's names and meanings: ``max_new_tokens``,
``temperature`` (0 = greedy argmax) and ``top_p`` (>= 1 = off) are the arguments of its
``Engine.submit`` (pico_vllm/engine.py:243-247) and of ``sampler.sample``
(pico_vllm/sampler.py:91-107).  ``seed`` and ``ignore_eos`` are additions: the reference draws
from torch's global generator and always stops at the tokenizer's end token."""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Optional

from ..errors import ConfigError


@dataclass
class SamplingParams:
    max_new_tokens: int = 16
    temperature: float = 1.0
    top_p: float = 1.0
    seed: Optional[int] = None
    ignore_eos: bool = False
    max_tokens: Optional[int] = None     # another name for max_new_tokens

    def __post_init__(self):
        if self.max_tokens is not None:
            self.max_new_tokens = self.max_tokens
        if self.max_new_tokens < 1:
            raise ConfigError("max_new_tokens must be at least 1")
        if self.temperature < 0:
            raise ConfigError("temperature must be >= 0 (0 means greedy)")
        if not self.top_p > 0:
            raise ConfigError("top_p must be > 0")


@dataclass
class BeamParams:
    """Options of beam search: the ``beams`` best continuations are kept at every token.  A hypothesis is worth the sum of its tokens'
    log-probabilities divided by its length to the power ``length_penalty`` (its end token counted; 0: the sum itself;
    max_new_tokens ** length_penalty is at most 2 ** 873).  The reference has no beam search."""
    beams: int = 4
    max_new_tokens: int = 16
    length_penalty: float = 1.0
    ignore_eos: bool = False
    num_return: Optional[int] = None     # hypotheses to return, best first; None = as many as beams

    def __post_init__(self):
        if not 1 <= self.beams <= 32:
            raise ConfigError("beams must lie in 1 .. 32")
        if self.max_new_tokens < 1:
            raise ConfigError("max_new_tokens must be at least 1")
        if not 0 <= self.length_penalty < float("inf"):
            raise ConfigError("length_penalty must be a number >= 0")
        # the value of a hypothesis is to be a number of full precision: a sum of log-probabilities as small as a float32 holds (2^-149), divided, is
        # not below the smallest such float64 (2^-1022)
        if self.max_new_tokens > 1 and self.length_penalty > 873 / math.log2(self.max_new_tokens):
            raise ConfigError(f"length_penalty {self.length_penalty} with max_new_tokens {self.max_new_tokens}: a length to that power is beyond the "
                              f"numbers that hypotheses can be ranked by (at most {873 / math.log2(self.max_new_tokens):.1f})")
        if self.num_return is None:
            self.num_return = self.beams
        if not 1 <= self.num_return <= self.beams:
            raise ConfigError("num_return must lie in 1 .. beams")
