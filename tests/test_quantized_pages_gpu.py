"""Keys and values stored in 8 bits (``quantize_kv_write``), read back (``dequantize_pages``), and pages copied (``copy_pages``): codes,
scales and pages have to be equal to the last bit."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from mini_llm_runtime_b200 import ops
from quantized_support import stored, values

pytestmark = pytest.mark.gpu

DEVICE = "cuda:0"


class Cache:
    """A pool with random contents and its copy on the host."""

    def __init__(self, pages, kv_heads, page, dim, block, seed, offset=0):
        rng = np.random.default_rng(seed)
        self.page, self.dim, self.kv_heads, self.block, self.pages = page, dim, kv_heads, block, pages
        self.codes = [rng.integers(-127, 128, (pages, kv_heads, page, dim)).astype(np.int8) for _ in range(2)]
        self.scales = [(rng.random((pages, kv_heads, page // block)) * 0.02 + 0.001).astype(np.float32) for _ in range(2)]

        def placed(array):      # on a boundary of its own
            flat = torch.empty(array.size + offset, dtype=torch.from_numpy(array).dtype, device=DEVICE)[offset:]
            return flat.copy_(torch.from_numpy(array).flatten()).view(array.shape)

        self.pool = ops.QuantizedPool(placed(self.codes[0]), placed(self.codes[1]), placed(self.scales[0]), placed(self.scales[1]))

    def write(self, rows, slots):
        """``rows`` [n, 2 * kv_heads * dim]: keys and values side by side; slots on the host."""
        width = self.kv_heads * self.dim
        ops.current().quantize_kv_write(rows[:, :width], rows[:, width:], torch.tensor(slots, dtype=torch.int64, device=DEVICE), self.pool)
        exact = rows.double().cpu().numpy()
        for i in range(2):
            stored(self.codes[i], self.scales[i], exact[:, i * width:(i + 1) * width].reshape(-1, self.kv_heads, self.dim), slots, self.block)

    def check(self):
        for got, want in zip((self.pool.key, self.pool.value), self.codes):
            assert np.array_equal(got.cpu().numpy(), want)
        for got, want in zip((self.pool.key_scales, self.pool.value_scales), self.scales):
            assert np.array_equal(got.cpu().numpy(), want, equal_nan=True)


def rows_of(count, width, dtype, seed, spare=0):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    rows = torch.randn((count, width + spare), generator=g, device=DEVICE) * (torch.rand((count, 1), generator=g, device=DEVICE) * 3 + 0.01)
    return rows.to(dtype)[:, :width]


SHAPES = [
    # kv_heads, dim, page, block, dtype
    (2, 64, 16, 16, torch.bfloat16), (4, 128, 16, 16, torch.bfloat16), (8, 128, 16, 1, torch.bfloat16), (3, 96, 16, 4, torch.float32),
    (1, 80, 8, 8, torch.bfloat16), (2, 17, 5, 5, torch.float32), (2, 256, 128, 64, torch.bfloat16), (1, 1, 1, 1, torch.float32),
    (3, 20, 6, 3, torch.bfloat16)]


@pytest.mark.parametrize("kv_heads,dim,page,block,dtype", SHAPES)
def test_tokens_of_prompts_and_decode_steps(kv_heads, dim, page, block, dtype):
    """A prompt in portions that end inside blocks and pages, then token by token, two requests in each step."""
    cache = Cache(60, kv_heads, page, dim, block, 1)
    tables = np.random.default_rng(2).permutation(60).reshape(2, 30)
    done = [0, 0]
    for step, counts in enumerate([(page * 2 + 3, 1), (1, page + 1), (5, 2), (1, 1), (1, 1), (1, 1), (block, 1), (1, 1)]):
        slots = []
        for request, count in enumerate(counts):
            for position in range(done[request], min(done[request] + count, 30 * page)):
                slots.append(int(tables[request, position // page]) * page + position % page)
            done[request] = min(done[request] + count, 30 * page)
        if slots:
            cache.write(rows_of(len(slots), 2 * kv_heads * dim, dtype, 10 + step, spare=step % 3), slots)
        cache.check()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_ties_and_neighbours_of_ties(dtype):
    """Halves of a step go to the even code; numbers one rounding beside them do not.  A scale that is no power of two: the quotient
    of x = amax / 2 lies at 63.5 or next to it, by the scale's own rounding."""
    cache = Cache(64, 1, 16, 64, 1, 3)
    rows = torch.zeros((64, 128), dtype=torch.float64)
    for r in range(64):
        top = 127.0 * 2.0 ** (r % 5 - 2) if r < 32 else float(129 + r)
        rows[r, 0] = rows[r, 64] = top
        steps = torch.arange(63, dtype=torch.float64) + (0.5 if r % 2 else 0.25)
        rows[r, 1:64] = steps * (2.0 ** (r % 5 - 2)) if r < 32 else top / 2 * (2.0 ** -(steps.floor() % 7))
        rows[r, 65:] = -rows[r, 1:64]
    cache.write(rows.to(dtype).to(DEVICE), list(range(0, 1024, 16)))
    cache.check()


def test_scales_that_grow_by_halves_round_held_codes_to_even():
    cache = Cache(1, 1, 8, 8, 8, 4)
    first = torch.zeros((1, 16))
    first[0, :8] = torch.tensor([127.0, 1.0, 3.0, 5.0, 7.0, -1.0, -3.0, 63.0])
    first[0, 8:] = first[0, :8]
    cache.write(first.to(DEVICE), [0])
    cache.check()
    later = torch.zeros((2, 16))
    later[:, 0], later[:, 8] = 254.0, 381.0        # twice and three times the scale
    cache.write(later.to(DEVICE), [1, 2])
    cache.check()
    assert cache.codes[0][0, 0, 0].tolist() == [64, 0, 2, 2, 4, 0, -2, 32]      # 63.5, 0.5, 1.5, 2.5 ..


def test_zeros_tiny_and_not_finite_numbers():
    cache = Cache(8, 2, 4, 16, 2, 5)
    rows = torch.randn((6, 64), generator=torch.Generator().manual_seed(6))
    rows[0] = 0.0
    rows[1] *= 2.0 ** -130                  # scales of few bits
    rows[2, 3] = float("inf")               # a key of head 0
    rows[3, 40] = float("nan")              # a value of head 0
    rows[4] *= 2.0 ** 120
    rows[5] = 2.0 ** -149
    cache.write(rows.to(DEVICE), [0, 4, 8, 12, 16, 20])
    cache.check()
    assert np.isnan(cache.scales[0][2, 0, 0]) and not np.isnan(cache.scales[0][2, 1, 0])
    # the next token of those blocks: NaN stays, zeros grow
    cache.write(torch.randn((6, 64), generator=torch.Generator().manual_seed(7)).to(DEVICE), [1, 5, 9, 13, 17, 21])
    cache.check()


def test_slots_outside_the_pool_are_passed_over_and_none_is_no_work():
    cache = Cache(4, 2, 8, 32, 4, 8)
    rows = rows_of(7, 128, torch.bfloat16, 9)
    cache.write(rows, [-1, 0, 1, 4 * 8, 1 << 40, -5, 9])
    cache.check()
    cache.write(rows[:0], [])
    cache.check()


def test_pools_and_rows_on_any_boundary():
    cache = Cache(6, 2, 8, 32, 8, 10, offset=3)
    wide = rows_of(20, 129, torch.bfloat16, 11)
    cache.write(wide[:, 1:], list(range(20)))
    cache.check()


def test_a_long_prompt():
    cache = Cache(300, 8, 16, 128, 16, 12)
    pages = np.random.default_rng(13).permutation(300)
    slots = [int(pages[position // 16]) * 16 + position % 16 for position in range(7, 4500)]
    cache.write(rows_of(len(slots), 2 * 8 * 128, torch.bfloat16, 14), slots)
    cache.check()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kv_heads,dim,page,block", [(4, 128, 16, 16), (3, 96, 16, 4), (2, 17, 5, 1)])
def test_pages_read_back(kv_heads, dim, page, block, dtype):
    cache = Cache(9, kv_heads, page, dim, block, 15)
    pages = [3, 0, 8, -1, 3, 9]
    got = ops.current().dequantize_pages(cache.pool, torch.tensor(pages, dtype=torch.int32, device=DEVICE), dtype)
    for mine, codes, scales in zip(got, (cache.pool.key, cache.pool.value), (cache.pool.key_scales, cache.pool.value_scales)):
        want = values(codes, scales).float().to(dtype)
        for i, at in enumerate(pages):
            assert torch.equal(mine[i], want[at] if 0 <= at < 9 else torch.zeros_like(mine[i]))
    assert ops.current().dequantize_pages(cache.pool, torch.zeros(0, dtype=torch.int32, device=DEVICE))[0].shape == (0, kv_heads, page, dim)


# ------------------------------------------------------------------ pages copied
@pytest.mark.parametrize("shape,dtype,moves", [
    ((24, 40, 2, 16, 64), torch.bfloat16, 1), ((3, 1000, 4, 16, 128), torch.int8, 450), ((2, 50, 3, 4), torch.float32, 20),
    ((5, 30, 7), torch.int8, 13), ((1, 2, 1), torch.bfloat16, 1), ((2, 9, 8, 128, 256), torch.bfloat16, 4), ((4, 30, 1, 1), torch.int64, 9)])
def test_pages_within_their_pools(shape, dtype, moves):
    g = torch.Generator(device=DEVICE).manual_seed(20)
    pools = [torch.randint(-100, 100, shape, generator=g, device=DEVICE, dtype=torch.int32).to(dtype) for _ in range(2)]
    # a pool of other pages beside them, as scales lie beside codes
    pools.append(torch.randint(0, 9, (2, shape[1], 3), generator=g, device=DEVICE, dtype=torch.int32).float())
    order = np.random.default_rng(21).permutation(shape[1])
    source, target = order[:moves].tolist(), order[-moves:].tolist() if 2 * moves <= shape[1] else order[moves:].tolist()
    source = source[:len(target)]
    source[-1] = source[0]                       # a page may go to several places
    want = [pool.clone() for pool in pools]
    for pool in want:
        for a, b in zip(source, target):
            pool[:, b] = pool[:, a]
    ops.current().copy_pages(pools, source, target)
    for pool, expected in zip(pools, want):
        assert torch.equal(pool, expected)


def test_pages_into_other_pools_and_more_pools_than_a_launch_takes():
    pools = [torch.arange(4 * 10 * 33, device=DEVICE, dtype=torch.float32).view(4, 10, 33) + i for i in range(11)]
    into = [torch.full((4, 25, 33), -1.0, device=DEVICE) for _ in range(11)]
    ops.current().copy_pages(pools, range(10), [24, 3, 5, 7, 9, 11, 0, 1, 2, 23], into=into)
    for pool, other in zip(pools, into):
        assert torch.equal(other[:, [24, 3, 5, 7, 9, 11, 0, 1, 2, 23]], pool)
        assert int((other == -1.0).all(-1).all(0).sum()) == 15
    ops.current().copy_pages([], [0], [1])
    ops.current().copy_pages(pools, [], [])


def test_pools_on_odd_boundaries():
    flat = torch.arange(2 * 6 * 12 + 1, device=DEVICE, dtype=torch.int32).to(torch.int8)[1:]
    pool = flat.view(2, 6, 12)
    want = pool.clone()
    want[:, 5] = want[:, 2]
    ops.current().copy_pages([pool], [2], [5])
    assert torch.equal(pool, want)


def test_what_is_refused():
    k = ops.current()
    pool = torch.zeros((2, 8, 4), device=DEVICE)
    for source, target, message in (([0], [0], "source and target"), ([0, 1], [2, 2], "one copy"), ([8], [1], "lie in"), ([0], [-1], "lie in"),
                                    ([0, 1], [2], "one page number each"), ([0, 1], [1, 2], "source and target")):
        with pytest.raises(ops.KernelError, match=message):
            k.copy_pages([pool], source, target)
    with pytest.raises(ops.KernelError, match="number of pages"):
        k.copy_pages([pool, torch.zeros((2, 9, 4), device=DEVICE)], [0], [1])
    with pytest.raises(ops.KernelError, match="do not fit"):
        k.copy_pages([pool], [0], [1], into=[torch.zeros((2, 8, 5), device=DEVICE)])
    with pytest.raises(ops.KernelError, match="must not be those"):
        k.copy_pages([pool], [0], [1], into=[pool])
    with pytest.raises(ops.KernelError, match="contiguous"):
        k.copy_pages([torch.zeros((8, 2, 4), device=DEVICE).transpose(0, 1)], [0], [1])
    cache = Cache(4, 2, 8, 32, 4, 8)
    rows = rows_of(3, 128, torch.bfloat16, 9)
    slots = torch.arange(3, device=DEVICE)
    for key, value, at in ((rows[:, :64], rows[:, 64:].float(), slots), (rows[:, :63], rows[:, 64:], slots), (rows[:, :64], rows[:, 64:], slots[:2]),
                           (rows[:, :64].half(), rows[:, 64:].half(), slots), (rows[:, :64], rows[:, 64:], slots.int()),
                           (rows[:, :64].t().contiguous().t(), rows[:, 64:], slots)):
        with pytest.raises(ops.KernelError):
            k.quantize_kv_write(key, value, at, cache.pool)
    with pytest.raises(ops.KernelError):
        ops.QuantizedPool(cache.pool.key, cache.pool.value, cache.pool.key_scales[:, :1].contiguous(), cache.pool.value_scales)
    with pytest.raises(ops.KernelError):
        ops.QuantizedPool(cache.pool.key.to(torch.uint8), cache.pool.value, cache.pool.key_scales, cache.pool.value_scales)
