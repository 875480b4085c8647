"""What ``shared_prefix_attention`` hands to its kernels: the arguments of the launch, with a library that records them."""

from __future__ import annotations

import pytest
import torch

from mini_llm_runtime_b200.ops import CudaOps, cuda_ops
from test_request_operators_cpu import decoded, shared


class Recorder:
    def __init__(self):
        self.calls = []

    def mlr_attention_prefix(self, *arguments):
        names = ("q k_pool v_pool out q_row pos0 seg_slot block_table seg_keys members tile_first tile_count tile_keys acc state segments tiles "
                 "heads kv_heads dim page_size pages table_width chunk prefix_parts own_parts units scale dtype fast error_word stream").split()
        self.calls.append(dict(zip(names, arguments, strict=True)))
        return 0


@pytest.fixture
def library(monkeypatch):
    recorder = Recorder()
    recorder.allocated = []
    empty = torch.empty

    def recorded(*args, **named):
        tensor = empty(*args, **named)
        recorder.allocated.append(tensor)
        return tensor

    monkeypatch.setattr(cuda_ops, "_need", lambda *args, **named: None)
    monkeypatch.setattr(cuda_ops, "_need_here", lambda **tensors: None)
    monkeypatch.setattr(cuda_ops, "_raw_stream", lambda: 0)
    monkeypatch.setattr(cuda_ops, "_declared_library", lambda name: recorder)
    monkeypatch.setattr(CudaOps, "sm_count", lambda self, device: 148)
    monkeypatch.setattr(CudaOps, "_error_word", lambda self, device: torch.zeros(1, dtype=torch.int32))
    monkeypatch.setattr(cuda_ops.torch, "empty", recorded)
    return recorder


@pytest.mark.parametrize("dim", [1, 7, 33, 64, 80, 127, 255, 256])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 1), (9, 3), (4, 2)])
@pytest.mark.parametrize("segments,longest", [(1, 50), (3, 900), (5, 50)])
def test_states_lie_on_their_boundaries(library, dim, heads, kv_heads, segments, longest):
    """Outputs on 16 bytes, the pairs behind them on 8, both inside the memory they were given, whatever is odd."""
    prefix = shared([(range(segments), 16)] if segments > 1 else [], segments, heads // kv_heads)
    batch = decoded(segments, longest, pages=60)
    kernels = CudaOps()
    kernels.shared_prefix_least = 0
    pool = torch.zeros((9, kv_heads, 16, dim))
    kernels.shared_prefix_attention(torch.zeros((segments, heads * dim)), pool, pool, batch, prefix, heads, kv_heads, dim, 0.3)
    call = library.calls[-1]
    states = (call["prefix_parts"] + call["own_parts"]) * segments * heads
    scratch = next(t for t in library.allocated if t.data_ptr() == call["acc"])
    assert (call["acc"] % 16, call["state"] % 8) == (0, 0)
    assert call["acc"] + 4 * states * dim <= call["state"]
    assert call["state"] + 8 * states <= scratch.data_ptr() + 4 * scratch.numel()


@pytest.mark.parametrize("least", [0, 1 << 40])
@pytest.mark.parametrize("moved", ["q", "k", "v"])
def test_tensors_on_no_16_byte_boundary_take_the_general_kernels(monkeypatch, library, moved, least):
    kernels = CudaOps()
    kernels.shared_prefix_least = least
    decoding = []
    monkeypatch.setattr(kernels, "_decode_attention", lambda *args, **named: decoding.append(args))
    tensors = {"q": torch.zeros((3, 4 * 64), dtype=torch.bfloat16), "k": torch.zeros((9, 2, 16, 64), dtype=torch.bfloat16),
               "v": torch.zeros((9, 2, 16, 64), dtype=torch.bfloat16)}
    place = tensors[moved]
    tensors[moved] = torch.zeros(place.numel() + 8, dtype=torch.bfloat16)[1:place.numel() + 1].view(place.shape)
    kernels.shared_prefix_attention(tensors["q"], tensors["k"], tensors["v"], decoded(3, 900, pages=60), shared([(range(3), 16)], 3, 2), 4, 2, 64, 0.3)
    assert not decoding and library.calls[-1]["fast"] == 0
