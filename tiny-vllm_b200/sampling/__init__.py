from .params import SamplingParams
from .rules import LogitRules
from .sampler import Sampler

__all__ = ["LogitRules", "Sampler", "SamplingParams"]
