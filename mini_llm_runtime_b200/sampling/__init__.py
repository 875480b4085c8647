from .params import GREEDY, SamplingParams
from .rules import LogitRules

__all__ = ["GREEDY", "LogitRules", "SamplingParams"]
