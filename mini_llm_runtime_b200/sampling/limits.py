"""The limits of the requests on what is drawn for them, resident on the device and read by slot.

An engine made with ``sampling_limits=True`` holds one set of tables (``ops.SamplingLimits``): top-k, top-p and min-p of every slot.  Each
step then draws its tokens under them; temperature, seed and counter stay in the slot records.  The host writes a slot's entries when
its request is admitted, so a captured step finds whatever requests its rows belong to.
"""

from __future__ import annotations

import torch

from .. import ops
from .params import SamplingParams


class RequestLimits:
    """The tables of ``max_requests`` slots (12 bytes each)."""

    def __init__(self, max_requests: int, device: torch.device | str) -> None:
        if max_requests <= 0:
            raise ValueError("max_requests must be > 0")
        self.device = torch.device(device)
        self.tables = ops.SamplingLimits(top_k=torch.zeros(max_requests, dtype=torch.int32, device=self.device),
                                         top_p=torch.ones(max_requests, device=self.device), min_p=torch.zeros(max_requests, device=self.device))

    def admit(self, slot: int, sampling: SamplingParams) -> None:
        """A new request owns the slot."""
        tables = self.tables
        tables.top_k[slot].fill_(sampling.top_k)
        tables.top_p[slot].fill_(sampling.top_p)
        tables.min_p[slot].fill_(sampling.min_p)
