"""Attention of decoded tokens behind shared prefixes (``shared_prefix_attention``) against softmax attention in 64 bits, request by
request through its row of the block table: prefixes that end inside pages and tiles, requests of no group, one key, long ones."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from mini_llm_runtime_b200 import ops
from mini_llm_runtime_b200.ops import AttentionBatch, SharedPrefix

pytestmark = pytest.mark.gpu

DEVICE = "cuda:0"


@pytest.fixture(autouse=True)
def every_prefix_by_itself(monkeypatch):
    """Small steps too; the rule that sends them through ``paged_attention`` has a test of its own."""
    monkeypatch.setattr(ops.current(), "shared_prefix_least", 0)


class Step:
    """A step of decoded tokens: groups of (number of requests, shared keys), requests alone, own keys of each in turn."""

    def __init__(self, groups, alone, own, heads, kv_heads, dim, page, dtype, seed, spare_slots=2, limit=None, share=None):
        rng = np.random.default_rng(seed)
        g = torch.Generator(device=DEVICE).manual_seed(seed)
        owners = [i for i, (count, _) in enumerate(groups) for _ in range(count)] + [-1] * alone
        rng.shuffle(owners)
        count = len(owners)
        self.contexts = [(groups[o][1] if o >= 0 else 0) + own[i % len(own)] for i, o in enumerate(owners)]
        width = -(-max(self.contexts) // page) + 1
        # whole pages of the prefix are one for all; the page it ends in is copied for each request
        need = sum(keys // page for _, keys in groups) + sum(-(-c // page) for c in self.contexts)
        ids = rng.permutation(need + 3).astype(np.int32).tolist()
        lead = [[ids.pop() for _ in range(keys // page)] for _, keys in groups]
        slots = rng.permutation(count + spare_slots)[:count].astype(np.int32)
        table = np.full((count + spare_slots, width), -1, dtype=np.int32)
        for i, o in enumerate(owners):
            row = list(lead[o]) if o >= 0 else []
            row += [ids.pop() for _ in range(-(-self.contexts[i] // page) - len(row))]
            table[slots[i], :len(row)] = row
        self.heads, self.kv_heads, self.dim, self.page, self.scale = heads, kv_heads, dim, page, dim ** -0.5
        self.q = torch.randn((count, heads * dim), generator=g, device=DEVICE).to(dtype)
        pool = (need + 3, kv_heads, page, dim)
        self.k = torch.randn(pool, generator=g, device=DEVICE).to(dtype)
        self.v = torch.randn(pool, generator=g, device=DEVICE).to(dtype)
        self.table, self.slots = torch.from_numpy(table).to(DEVICE), slots
        position = np.asarray(self.contexts, dtype=np.int32) - 1
        arrays, counts = ops.current().plan_attention(np.ones(count, dtype=np.int32), position)
        self.batch = AttentionBatch(
            seg_q_start=torch.arange(count, dtype=torch.int32, device=DEVICE), seg_q_len=torch.ones(count, dtype=torch.int32, device=DEVICE),
            seg_pos0=torch.from_numpy(position).to(DEVICE), seg_slot=torch.from_numpy(slots).to(DEVICE), block_table=self.table,
            num_segments=count, max_q_len=1, max_kv_len=limit or max(self.contexts),
            plan={name: torch.from_numpy(a).to(DEVICE) for name, a in arrays.items()}, counts=counts)
        sharing = [([i for i in range(count) if owners[i] == o], keys // page * page if share is None else share)
                   for o, (_, keys) in enumerate(groups)]
        self.prefix = self.planned(sharing)

    def planned(self, sharing):
        arrays, counts = ops.current().plan_shared_prefix(sharing, len(self.contexts), self.heads // self.kv_heads)
        return SharedPrefix({name: torch.from_numpy(a).to(DEVICE) for name, a in arrays.items()}, counts)

    def run(self, prefix=None):
        return ops.current().shared_prefix_attention(self.q, self.k, self.v, self.batch, prefix or self.prefix, self.heads, self.kv_heads,
                                                     self.dim, self.scale)

    def check(self, got):
        """|error| of o = sum p v, p the normalised weights, sum p |v| = A, n keys: half a step of the result; A times the relative
        error of a weight: one rounding of p to the tensor cores' type, e^x off by 2^-20, twice the score's error, which is at most
        (dim + 4) 2^-24 of sum |q||k| scale, and n sums in 32 bits, 4 sqrt(n) 2^-24."""
        dtype, per = self.q.dtype, self.heads // self.kv_heads
        u = torch.finfo(dtype).eps / 2
        in_p = u if dtype == torch.bfloat16 else 2.0 ** -24
        for i, context in enumerate(self.contexts):
            place = torch.arange(context, device=DEVICE)
            page = self.table[int(self.slots[i])].long()[place // self.page]
            k = self.k[page, :, place % self.page].double().permute(1, 0, 2)
            v = self.v[page, :, place % self.page].double().permute(1, 0, 2)
            q = self.q[i].double().view(self.kv_heads, per, self.dim)
            p = torch.softmax(q @ k.transpose(1, 2) * self.scale, dim=-1)
            want, mass = (p @ v).reshape(-1), (p @ v.abs()).reshape(-1)
            reach = float((q.abs() @ k.abs().transpose(1, 2)).max()) * self.scale
            relative = in_p + 2.0 ** -20 + 2 * (self.dim + 4) * 2.0 ** -24 * reach + 4 * context ** 0.5 * 2.0 ** -24
            bound = u * want.abs() + 1.02 * relative * (mass + want.abs())
            error = (got[i].double() - want).abs()
            assert bool((error <= bound).all()), (i, context, float((error - bound).max()), float(error.max()))


KINDS = [(14, 2, 64, torch.bfloat16), (28, 4, 128, torch.bfloat16), (3, 1, 32, torch.float32), (12, 3, 96, torch.float32), (8, 8, 64, torch.bfloat16),
         (16, 1, 128, torch.bfloat16), (6, 2, 80, torch.bfloat16), (4, 2, 256, torch.float32), (20, 1, 64, torch.bfloat16), (2, 2, 16, torch.bfloat16)]


@pytest.mark.parametrize("heads,kv_heads,dim,dtype", KINDS)
@pytest.mark.parametrize("groups,alone,own,page", [
    ([(3, 40)], 1, (1, 17, 5), 16),                      # a prefix of two and a half pages
    ([(2, 64), (5, 300), (1, 129)], 2, (1, 64, 65, 200), 8),
    ([(19, 513)], 0, (3, 700, 64), 16),                  # more members than one work item holds
    ([], 4, (1, 2, 90, 300), 16),                        # nobody shares
    ([(4, 7)], 0, (30,), 16),                            # a prefix shorter than a page: nothing to share
    ([(2, 96), (2, 96)], 1, (33,), 32),
])
def test_against_softmax_attention(heads, kv_heads, dim, dtype, groups, alone, own, page):
    step = Step(groups, alone, own, heads, kv_heads, dim, page, dtype, seed=heads + page)
    step.check(step.run())


@pytest.mark.parametrize("heads,kv_heads,dim", [(14, 2, 64), (28, 4, 128), (40, 8, 128), (16, 1, 64)])
def test_long_prefixes(heads, kv_heads, dim):
    step = Step([(33, 5000), (2, 1111), (12, 9001)], 2, (1, 300, 1500, 64), heads, kv_heads, dim, 16, torch.bfloat16, seed=dim)
    step.check(step.run())


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page", [1, 4, 8, 12, 16, 64, 128])
def test_page_sizes(dim, page):
    step = Step([(6, 260)], 1, (1, 70, 130), 8, 2, dim, page, torch.bfloat16, seed=page)
    step.check(step.run())


@pytest.mark.parametrize("dim", [64, 128])
def test_shared_keys_that_end_inside_a_page(dim):
    """The plan may share fewer keys than the pages hold: any number up to the shared ones."""
    for share in (1, 15, 63, 64, 65, 100, 127, 128):
        step = Step([(5, 128)], 0, (9, 40), 14, 2, dim, 16, torch.bfloat16, seed=share, share=share)
        step.check(step.run())


@pytest.mark.parametrize("dim", [64, 128])
def test_what_lies_behind_the_keys_does_not_matter(dim):
    """NaN and infinities in the pools, in every place that no key of the step uses."""
    step = Step([(5, 100)], 1, (9, 40, 1), 14, 2, dim, 16, torch.bfloat16, seed=3)
    want = step.run()
    used = torch.zeros(step.k.shape[0] * step.page, dtype=torch.bool, device=DEVICE)
    for i, context in enumerate(step.contexts):
        place = torch.arange(context, device=DEVICE)
        used[step.table[int(step.slots[i])].long()[place // step.page] * step.page + place % step.page] = True
    used = used.view(step.k.shape[0], 1, step.page, 1)
    step.k = torch.where(used, step.k, torch.tensor(float("nan"), dtype=step.k.dtype, device=DEVICE))
    step.v = torch.where(used, step.v, torch.tensor(float("inf"), dtype=step.v.dtype, device=DEVICE))
    assert torch.equal(step.run(), want)


@pytest.mark.parametrize("dim,dtype", [(64, torch.bfloat16), (128, torch.bfloat16), (48, torch.float32)])
def test_a_far_key_that_dominates(dim, dtype):
    """One key of the prefix, then one of the own keys, outweighs all others by far: both parts' states must carry it."""
    for place in (3, 130, 421, 430):
        step = Step([(4, 421)], 0, (30,), 4, 2, dim, 16, dtype, seed=place)
        for i in range(4):
            page = int(step.table[int(step.slots[i]), place // 16])
            step.k[page, :, place % 16] = step.q[i].view(2, 2, dim)[:, 0] * 6
        step.check(step.run())


def test_groups_in_any_split_give_the_same_numbers():
    """The same step as one group, as two, and with nobody sharing."""
    step = Step([(6, 640)], 0, (20, 90), 14, 2, 64, 16, torch.bfloat16, seed=4)
    for sharing in ([(range(6), 640)], [((0, 2, 4), 640), ((5, 3, 1), 320)], [((2,), 640)], [(range(6), 0)], []):
        step.check(step.run(step.planned(sharing)))


@pytest.mark.parametrize("dim,dtype", [(64, torch.bfloat16), (128, torch.bfloat16), (64, torch.float32)])
def test_a_captured_step_follows_positions_and_tables(dim, dtype):
    """Captured against a context limit and replayed while contexts grow into further pages."""
    step = Step([(5, 200), (4, 333)], 1, (9, 40, 1), 8, 2, dim, 16, dtype, seed=5, limit=1024)
    step.run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step.run()
    for grown in (0, 5, 6):
        step.contexts = [c + grown for c in step.contexts]
        step.batch.seg_pos0 += grown
        spare = torch.arange(len(step.contexts), device=DEVICE, dtype=torch.int32)       # a page that others use too: only reads
        for i, context in enumerate(step.contexts):
            held = -(-context // 16)
            row = step.table[int(step.slots[i])]
            if held <= row.shape[0] and int(row[held - 1]) < 0:
                row[held - 1] = spare[i]
        graph.replay()
        torch.cuda.synchronize()
        step.check(out)


def test_repeated_calls_give_the_same_bits():
    step = Step([(9, 2000)], 2, (500, 20), 28, 4, 128, 16, torch.bfloat16, seed=6)
    first = step.run()
    for _ in range(5):
        assert torch.equal(step.run(), first)


def test_on_another_stream_and_beside_paged_attention():
    step = Step([(9, 700)], 2, (200, 20), 14, 2, 64, 16, torch.bfloat16, seed=7)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = step.run()
    stream.synchronize()
    step.check(got)
    step.check(ops.current().paged_attention(step.q, step.k, step.v, step.batch, 14, 2, 64, step.scale, None))


def test_pages_beyond_32_bit_offsets():
    """A pool of more than 2^31 elements whose last pages are the ones in use."""
    step = Step([(3, 160)], 1, (20, 90), 8, 4, 128, 16, torch.bfloat16, seed=8)
    pages = (1 << 31) // (4 * 16 * 128) + 50
    shift = pages - step.k.shape[0]
    for name in ("k", "v"):
        pool = torch.zeros((pages, 4, 16, 128), dtype=torch.bfloat16, device=DEVICE)
        pool[shift:] = getattr(step, name)
        setattr(step, name, pool)
    step.table[step.table >= 0] += shift
    step.check(step.run())


@pytest.mark.parametrize("dim", [64, 128])
def test_the_rule_of_small_savings(monkeypatch, dim):
    """On both sides of the bytes from which a prefix is walked by itself: the same numbers, and ``paged_attention`` just below."""
    kernels = ops.current()
    saved = 4 * 3 * 512 * 2 * dim              # three of four requests spared 512 keys of two kv heads
    calls = []
    decode = kernels._decode_attention
    monkeypatch.setattr(kernels, "_decode_attention", lambda *args, **named: calls.append(1) or decode(*args, **named))
    for least, expected in ((saved, 0), (saved + 1, 1)):
        monkeypatch.setattr(kernels, "shared_prefix_least", least)
        step = Step([(4, 512)], 1, (9, 200, 1), 8, 2, dim, 16, torch.bfloat16, seed=dim)
        step.check(step.run())
        assert len(calls) == expected
