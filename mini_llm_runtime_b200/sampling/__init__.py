from .limits import RequestLimits
from .params import GREEDY, SamplingParams
from .rules import LogitRules

__all__ = ["GREEDY", "LogitRules", "RequestLimits", "SamplingParams"]
