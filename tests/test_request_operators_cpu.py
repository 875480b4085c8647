"""What the operators of requests refuse, before anything reaches a kernel: argument checks run here without a GPU, with the
question whether a tensor lies on the device left out and a library that must not be reached."""

from __future__ import annotations

import pytest
import torch

from mini_llm_runtime_b200.ops import AdapterStack, CudaOps, KernelError, LogitTables, cuda_ops


@pytest.fixture
def kernels(monkeypatch):
    def need(tensor, name, dtype=None, dims=None):
        if not isinstance(tensor, torch.Tensor):
            raise KernelError(f"{name} must be a tensor")
        if not tensor.is_contiguous():
            raise KernelError(f"{name} must be contiguous")
        if dtype is not None and tensor.dtype != dtype:
            raise KernelError(f"{name} must be {dtype}")
        if dims is not None and tensor.dim() != dims:
            raise KernelError(f"{name} must have {dims} dimensions")

    def library(name):
        raise AssertionError("a refused call reached the library")

    monkeypatch.setattr(cuda_ops, "_need", need)
    monkeypatch.setattr(cuda_ops, "_need_here", lambda **tensors: None)
    monkeypatch.setattr(cuda_ops, "_declared_library", library)
    monkeypatch.setattr(cuda_ops.build, "load_library", library)
    return CudaOps()


def history(slots=2, vocab=40):
    return dict(penalties=torch.ones((slots, 3)), counts=torch.zeros((slots, vocab), dtype=torch.int32),
                seen=torch.zeros((slots, -(-vocab // 32)), dtype=torch.int32))


@pytest.mark.parametrize("change", [
    {"counts": None}, {"penalties": None}, {"seen": None},
    {"counts": torch.zeros((2, 65), dtype=torch.int32)}, {"seen": torch.zeros((2, 1), dtype=torch.int32)},
    {"penalties": torch.ones((2, 2))}, {"penalties": torch.ones((3, 3))}, {"counts": torch.zeros((2, 40))},
    {"bias_tokens": torch.zeros((2, 4), dtype=torch.int32)}, {"bias_values": torch.zeros((2, 4))},
    {"bias_tokens": torch.zeros((2, 4), dtype=torch.int32), "bias_values": torch.zeros((2, 5))},
    {"bias_tokens": torch.zeros((2, 4), dtype=torch.int64), "bias_values": torch.zeros((2, 4))},
    {"allowed": torch.zeros((2, 3), dtype=torch.int32)}, {"allowed": torch.zeros((1, 2), dtype=torch.int32)},
    {"seen": torch.zeros((2, 4), dtype=torch.int32)[:, ::2]},
])
def test_tables_that_do_not_fit(kernels, change):
    with pytest.raises(KernelError):
        LogitTables(**{**history(), **change})


@pytest.mark.parametrize("logits,row_slot", [
    (torch.zeros((1, 40), dtype=torch.bfloat16), torch.zeros(1, dtype=torch.int32)),
    (torch.zeros((2, 40)), torch.zeros(1, dtype=torch.int32)),
    (torch.zeros((1, 40)), torch.zeros(1, dtype=torch.int64)),
    (torch.zeros((1, 80))[:, ::2], torch.zeros(1, dtype=torch.int32)),
    (torch.zeros(40), torch.zeros(1, dtype=torch.int32)),
])
def test_logits_that_do_not_fit(kernels, logits, row_slot):
    for call in (kernels.shape_logits, kernels.shape_logits_):
        with pytest.raises(KernelError):
            call(logits, row_slot, LogitTables(**history()))


def test_tables_without_a_rule_or_slot(kernels):
    for tables in ({}, {"allowed": torch.zeros((0, 2), dtype=torch.int32)}):
        with pytest.raises(KernelError):
            LogitTables(**tables)


@pytest.mark.parametrize("tables", [history(vocab=41), {"allowed": torch.zeros((2, 3), dtype=torch.int32)}])
def test_tables_of_another_vocabulary(kernels, tables):
    with pytest.raises(KernelError):
        kernels.shape_logits(torch.zeros((1, 40)), torch.zeros(1, dtype=torch.int32), LogitTables(**tables))


@pytest.mark.parametrize("tokens,slots,tables", [
    (torch.zeros(3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), history()),
    (torch.zeros(3, dtype=torch.int64), torch.zeros(3, dtype=torch.int32), history()),
    (torch.zeros(3, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), {"allowed": torch.zeros((2, 2), dtype=torch.int32)}),
])
def test_histories_that_do_not_fit(kernels, tokens, slots, tables):
    with pytest.raises(KernelError):
        kernels.count_tokens(tokens, slots, LogitTables(**tables))


def stack(**change):
    return AdapterStack(**{**dict(down=torch.zeros((3, 4, 16)), up=torch.zeros((3, 24, 4)), scales=torch.ones(3)), **change})


@pytest.mark.parametrize("change", [
    {"down": torch.zeros((3, 4, 16), dtype=torch.float16)}, {"down": torch.zeros((3, 4, 16), dtype=torch.bfloat16)},
    {"down": torch.zeros((2, 4, 16))}, {"down": torch.zeros((3, 5, 16))}, {"down": torch.zeros((4, 16))},
    {"down": torch.zeros((3, 0, 16)), "up": torch.zeros((3, 24, 0))}, {"scales": torch.ones(2)},
    {"scales": torch.ones(3, dtype=torch.float64)}, {"down": torch.zeros((3, 129, 16)), "up": torch.zeros((3, 24, 129))},
    {"down": torch.zeros((0, 4, 16)), "up": torch.zeros((0, 24, 4)), "scales": torch.ones(0)},
    {"down": torch.zeros((3, 4, 32))[:, :, ::2]}, {"down": torch.zeros(3 * 4 * 16 + 1)[1:].view(3, 4, 16)},
])
def test_stacks_that_do_not_fit(kernels, change):
    with pytest.raises(KernelError):
        stack(**change)


@pytest.mark.parametrize("change", [
    {"x": torch.zeros((5, 17))}, {"x": torch.zeros((5, 16), dtype=torch.bfloat16)}, {"x": torch.zeros((5, 32))[:, ::2]},
    {"weight": torch.zeros((25, 16))}, {"weight": torch.zeros((24, 17))}, {"row_adapter": torch.zeros(4, dtype=torch.int32)},
    {"row_adapter": torch.zeros(5, dtype=torch.int64)}, {"out_dtype": torch.bfloat16}, {"bias": torch.zeros(23)},
    {"x": torch.zeros(5 * 16 + 1)[1:].view(5, 16)},
])
def test_projections_that_do_not_fit(kernels, change):
    call = dict(x=torch.zeros((5, 16)), weight=torch.zeros((24, 16)), adapters=stack(), row_adapter=torch.zeros(5, dtype=torch.int32))
    with pytest.raises(KernelError):
        kernels.linear_adapters(**{**call, **change})


def test_tensors_of_another_device_are_refused(monkeypatch):
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)

    class Elsewhere:
        device = torch.device("cuda", 1)

    with pytest.raises(KernelError, match="current device"):
        cuda_ops._need_here(x=None, weight=Elsewhere())
