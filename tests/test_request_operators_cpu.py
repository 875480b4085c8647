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


# ------------------------------------------------------------------ shared prefixes
def test_plan_of_shared_prefixes():
    arrays, counts = cuda_ops.plan_shared_prefix([((4, 0, 2), 100), ((), 50), ((1,), 0), ((3,), 7)], 6, 50)
    assert arrays["seg_keys"].tolist() == [100, 0, 100, 7, 100, 0]
    assert arrays["members"].tolist() == [4, 0, 2, 3]
    assert arrays["tile_first"].tolist() == [0, 2, 3] and arrays["tile_count"].tolist() == [2, 1, 1]
    assert arrays["tile_keys"].tolist() == [100, 100, 7] and counts["tile_keys"] == (100, 100, 7)
    assert counts["tiles"] == 3 and counts["least_shared"] == 0 and counts["segments"] == 6
    assert all(array.dtype.name == "int32" for array in arrays.values())
    empty, counts = cuda_ops.plan_shared_prefix([], 0, 7)
    assert counts["tiles"] == 0 and empty["seg_keys"].shape == (0,)


@pytest.mark.parametrize("groups,segments,per", [
    ([((0, 6), 5)], 6, 1), ([((-1,), 5)], 6, 1), ([((1, 1), 5)], 6, 1), ([((0, 1), 5), ((1, 2), 5)], 6, 1), ([((0,), -1)], 6, 1),
    ([((0, 1), 0), ((1,), 5)], 6, 1), ([], 6, 0), ([], 6, 129),
])
def test_groups_that_do_not_fit(groups, segments, per):
    with pytest.raises(KernelError):
        cuda_ops.plan_shared_prefix(groups, segments, per)


def decoded(count, longest=50, pages=8):
    arrays, counts = cuda_ops.plan_attention([1] * count, [longest - 1] * count)
    index = torch.arange(count, dtype=torch.int32)
    return cuda_ops.AttentionBatch(index, torch.ones_like(index), torch.full((count,), longest - 1, dtype=torch.int32), index,
                                   torch.zeros((count, pages), dtype=torch.int32), count, 1, longest,
                                   {name: torch.from_numpy(a) for name, a in arrays.items()}, counts)


def shared(groups, count, per):
    arrays, counts = cuda_ops.plan_shared_prefix(groups, count, per)
    return cuda_ops.SharedPrefix({name: torch.from_numpy(a) for name, a in arrays.items()}, counts)


@pytest.mark.parametrize("change", [
    {"q": torch.zeros((3, 31))}, {"q": torch.zeros((2, 32))}, {"q": torch.zeros((3, 64))[:, ::2]}, {"k_pool": torch.zeros((9, 3, 16, 8))},
    {"v_pool": torch.zeros((9, 2, 16, 16))}, {"v_pool": torch.zeros((8, 2, 16, 8))}, {"k_pool": torch.zeros((9, 2, 16, 8), dtype=torch.bfloat16)},
    {"batch": decoded(4)}, {"prefix": ([((0, 1), 16)], 4, 2)}, {"prefix": ([((0, 1), 16)], 3, 4)},
    {"prefix": ([((0, 1), 51)], 3, 2)}, {"num_heads": 5}, {"num_kv_heads": 0}, {"head_dim": 0},
])
def test_attention_that_does_not_fit(kernels, change):
    call = dict(q=torch.zeros((3, 32)), k_pool=torch.zeros((9, 2, 16, 8)), v_pool=torch.zeros((9, 2, 16, 8)), batch=decoded(3),
                prefix=([((0, 1), 16)], 3, 2), num_heads=4, num_kv_heads=2, head_dim=8, scale=0.3)
    call.update(change)
    call["prefix"] = shared(*call["prefix"])
    with pytest.raises(KernelError):
        kernels.shared_prefix_attention(**call)


@pytest.mark.parametrize("name,value", [
    ("tile_keys", torch.zeros(2, dtype=torch.int32)), ("seg_keys", torch.zeros(2, dtype=torch.int32)), ("members", torch.zeros(3, dtype=torch.int32)),
    ("tile_first", torch.zeros(1, dtype=torch.int64)), ("tile_count", torch.zeros((1, 1), dtype=torch.int32)),
])
def test_a_prefix_whose_arrays_do_not_belong_together(kernels, name, value):
    whole = shared([((0, 1), 16)], 3, 2)
    with pytest.raises(KernelError):
        cuda_ops.SharedPrefix({**whole.plan, name: value}, whole.counts)


def test_parts_of_prefixes():
    """Every key has its part, whatever the sizes; the parts fit their bounds."""
    for keys in ((), (1,), (300,), (16384,) * 3 + (9001,) * 2 + (4100,), (131072,), tuple(range(1, 40))):
        for segments, heads, kv_heads, dim, longest in ((2, 14, 2, 64, 400), (64, 28, 4, 128, 9000), (256, 64, 8, 128, 131072), (1, 1, 1, 16, 1)):
            chunk, parts, units, own = cuda_ops.prefix_parts(keys, 0, segments, max((longest,) + keys), heads, kv_heads, dim, 148)
            assert 1 <= own <= 64 and parts <= 64
            if keys:
                assert chunk % 64 == 0 and chunk * parts >= max(keys) > chunk * (parts - 1)
                assert units == sum(-(-n // chunk) for n in keys) >= len(keys)
            else:
                assert chunk == parts == units == 0


def test_a_prompt_portion_is_refused(kernels):
    arrays, counts = cuda_ops.plan_attention([1, 2, 1], [5, 5, 5])
    batch = decoded(3)
    batch.counts = counts
    with pytest.raises(KernelError, match="decoded token"):
        kernels.shared_prefix_attention(torch.zeros((3, 32)), torch.zeros((9, 2, 16, 8)), torch.zeros((9, 2, 16, 8)), batch,
                                        shared([], 3, 2), 4, 2, 8, 0.3)
