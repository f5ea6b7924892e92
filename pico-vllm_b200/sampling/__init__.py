from .params import BeamParams, SamplingParams
from .sampler import Sampler, PendingTokens, uniform_for

__all__ = ["SamplingParams", "BeamParams", "Sampler", "PendingTokens", "uniform_for"]
