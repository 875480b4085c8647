"""Attention behind shared prefixes at the edges of what a call may bring."""

from __future__ import annotations

import pytest
import torch

from mini_llm_runtime_b200 import ops
from test_shared_prefix_gpu import Step

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def every_prefix_by_itself(monkeypatch):
    monkeypatch.setattr(ops.current(), "shared_prefix_least", 0)


@pytest.mark.parametrize("dim", [1, 7, 33, 127, 255])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 1), (9, 3)])
@pytest.mark.parametrize("groups,alone,own", [([(3, 40)], 0, (1,)), ([(2, 300)], 1, (5, 300)), ([], 1, (9,))])
def test_odd_heads_of_odd_sizes(dim, heads, kv_heads, groups, alone, own):
    """Three, one or five requests: the numbers of states are odd too."""
    for dtype in (torch.float32, torch.bfloat16):
        step = Step(groups, alone, own, heads, kv_heads, dim, 8, dtype, seed=dim)
        step.check(step.run())


@pytest.mark.parametrize("heads,kv_heads,dim,dtype", [(14, 2, 64, torch.bfloat16), (28, 4, 128, torch.bfloat16), (16, 1, 64, torch.bfloat16),
                                                      (6, 2, 64, torch.float32), (6, 2, 80, torch.bfloat16)])
def test_members_with_fewer_keys_than_their_group(heads, kv_heads, dim, dtype):
    """A request attends to its own context, whatever number of keys its group was planned with."""
    step = Step([(6, 320), (3, 700)], 1, (5, 90, 33), heads, kv_heads, dim, 16, dtype, seed=dim)
    for member, context in ((0, 1), (3, 64), (5, 65), (7, 319), (8, 200)):
        step.contexts[member] = min(context, step.contexts[member])
        step.batch.seg_pos0[member] = step.contexts[member] - 1
    step.check(step.run())


@pytest.mark.parametrize("heads,kv_heads,dim,dtype", [(14, 2, 64, torch.bfloat16), (8, 2, 128, torch.bfloat16), (6, 2, 48, torch.float32)])
@pytest.mark.parametrize("scale", [0.0, -0.125, -4.0])
def test_scales_of_zero_and_below(heads, kv_heads, dim, dtype, scale):
    """softmax(q k scale) of a negative scale is that of -q with its magnitude; of zero, the mean of the values."""
    step = Step([(6, 300)], 1, (5, 90), heads, kv_heads, dim, 16, dtype, seed=dim)
    step.scale = scale
    got = step.run()
    step.scale = abs(scale)
    step.q = -step.q
    step.check(got)


@pytest.mark.parametrize("least", [0, 1 << 40])
@pytest.mark.parametrize("name", ["q", "k", "v"])
@pytest.mark.parametrize("dim", [64, 128])
def test_tensors_on_no_16_byte_boundary(monkeypatch, dim, name, least):
    """They go through the general kernels, also where sharing saves too little; ``paged_attention``'s kernels refuse them."""
    monkeypatch.setattr(ops.current(), "shared_prefix_least", least)
    step = Step([(6, 320)], 1, (5, 90, 33), 14, 2, dim, 16, torch.bfloat16, seed=dim)
    tensor = getattr(step, name)
    view = torch.empty(tensor.numel() + 8, dtype=tensor.dtype, device=tensor.device)[1:tensor.numel() + 1].view(tensor.shape)
    setattr(step, name, view.copy_(tensor))
    step.check(step.run())
    kernels = ops.current()
    for use_tma in (True, False):
        monkeypatch.setattr(kernels, "use_tma_attention", use_tma)
        with pytest.raises(ops.KernelError, match="aligned"):
            kernels.paged_attention(step.q, step.k, step.v, step.batch, 14, 2, dim, step.scale, None)
