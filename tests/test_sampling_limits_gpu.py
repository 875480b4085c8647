"""Tokens drawn under top-k, top-p and min-p from given random numbers (``sample_limited``) against the definition in 64 bits: equal tokens,
but for a draw or a limit that lies nearer to a border than 64-bit sums can tell (1e-11 of the whole; 2^18 terms are off by 2^18 2^-53 at most)."""

from __future__ import annotations

import pytest
import torch

from limits_support import chosen
from mini_llm_runtime_b200 import ops

pytestmark = pytest.mark.gpu

DEVICE = "cuda:0"
NEAR = 1e-11


def limits_of(rows):
    """Rows of (temperature, k, p, min p) on the device."""
    columns = list(zip(*rows))
    return ops.SamplingLimits(*(torch.tensor(c, dtype=d, device=DEVICE) for c, d in zip(columns, (torch.float32, torch.int32, torch.float32, torch.float32))))


def check(logits, uniforms, rows):
    got = ops.current().sample_limited(logits, uniforms, limits_of(rows)).tolist()
    for row, (token, (temperature, k, p, least)) in enumerate(zip(got, rows)):
        f32 = [float(torch.tensor(x, dtype=torch.float32)) for x in (temperature, p, least)]
        want, near = chosen(logits[row], float(uniforms[row]), f32[0], k, f32[1], f32[2])
        assert token == want or near < NEAR, f"row {row} {rows[row]}: token {token}, expected {want} (nearest border {near:.1e})"


def case(rows, vocab, spread, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    return torch.randn((rows, vocab), generator=g, device=DEVICE) * spread, torch.rand(rows, generator=g, device=DEVICE)


LIMITS = [(1.0, 0, 1.0, 0.0), (0.7, 50, 1.0, 0.0), (0.7, 0, 0.9, 0.0), (1.2, 0, 1.0, 0.05), (0.8, 40, 0.95, 0.0), (0.8, 40, 0.95, 0.02),
          (1.0, 0, 0.5, 0.001), (0.0, 40, 0.9, 0.0), (1.0, 1, 1.0, 0.0), (1.0, 5000, 0.99, 0.0), (1.5, 3000, 1.0, 0.0), (1.0, 0, 0.999, 0.0),
          (0.1, 0, 0.9, 0.0), (5.0, 0, 0.9, 0.0), (1.0, 1 << 30, 2.0, 0.0), (2.0, 100000, 0.7, 1e-6)]


@pytest.mark.parametrize("vocab", [1, 2, 31, 32, 33, 1000, 2047, 4099, 16384, 32003, 151936, 152064])
@pytest.mark.parametrize("spread", [0.3, 1.0, 3.0])
def test_all_limits(vocab, spread):
    logits, uniforms = case(len(LIMITS), vocab, spread, vocab)
    check(logits, uniforms, LIMITS)


@pytest.mark.parametrize("rows", [1, 2, 9, 37, 75, 200])
def test_rows(rows):
    logits, uniforms = case(rows, 20011, 2.0, rows)
    check(logits, uniforms, [LIMITS[i % len(LIMITS)] for i in range(rows)])


def test_a_vocabulary_that_no_cluster_holds():
    logits, uniforms = case(3, 300007, 2.0, 5)
    check(logits, uniforms, [LIMITS[4], LIMITS[2], LIMITS[0]])


def test_many_draws_of_one_row():
    logits, _ = case(1, 5003, 2.0, 6)
    uniforms = torch.rand(400, generator=torch.Generator(device=DEVICE).manual_seed(7), device=DEVICE)
    for limits in ((0.9, 20, 0.9, 0.0), (0.9, 0, 0.97, 0.0), (0.9, 0, 1.0, 0.0), (0.9, 0, 1.0, 0.01)):
        check(logits.expand(400, -1).contiguous(), uniforms, [limits] * 400)


@pytest.mark.parametrize("vocab", [50, 5000, 152064])
def test_ties(vocab):
    """Few different logits, all equal ones: of a tie the lowest indexes stay."""
    g = torch.Generator(device=DEVICE).manual_seed(8)
    logits = torch.randint(-3, 4, (len(LIMITS) + 8, vocab), generator=g, device=DEVICE).float()
    logits[len(LIMITS):] = 1.25
    logits[len(LIMITS) + 4:, ::2] = 1.5
    uniforms = torch.rand(len(logits), generator=g, device=DEVICE)
    equal = [(1.0, 7, 1.0, 0.0), (1.0, 0, 0.501, 0.0), (1.0, vocab // 2 + 1, 0.33, 0.0), (0.5, 0, 1.0, 0.9)]
    check(logits, uniforms, LIMITS + equal + equal)


def test_zeros_of_both_signs_tie():
    logits = torch.zeros((4, 3000), device=DEVICE)
    logits[:, ::2] = -0.0
    check(logits, torch.tensor([0.0, 0.3, 0.6, 0.9999], device=DEVICE), [(1.0, 5, 1.0, 0.0)] * 4)
    check(logits, torch.tensor([0.0, 0.3, 0.6, 0.9999], device=DEVICE), [(0.0, 5, 1.0, 0.0)] * 4)


@pytest.mark.parametrize("vocab", [7, 3001, 151936])
def test_forbidden_tokens_and_numbers_that_are_none(vocab):
    logits, uniforms = case(8, vocab, 2.0, 9)
    logits[0] = -torch.inf
    logits[1] = -torch.inf
    logits[1, vocab // 2] = 3.0                       # one token is allowed
    logits[2, 1:] = torch.nan
    logits[3, ::3] = torch.nan
    logits[4, ::2] = -torch.inf
    logits[5, [1, 5]] = torch.inf                     # infinite ones share the whole
    logits[6] = torch.nan
    logits[7] = 3.4e38
    logits[7, 3:] = -3.4e38
    for limits in ((1.0, 0, 1.0, 0.0), (1.0, 3, 1.0, 0.0), (1.0, 0, 0.8, 0.0), (0.3, 1000, 0.8, 0.1), (1e-30, 0, 0.8, 0.0), (1e30, 0, 0.8, 0.0)):
        check(logits, uniforms, [limits] * 8)
        got = ops.current().sample_limited(logits, uniforms, limits_of([limits] * 8)).tolist()
        assert got[0] == 0 and got[1] == vocab // 2 and got[2] == 0 and got[3] % 3 and got[4] % 2 and got[5] in (1, 5) and got[6] == 0 and got[7] < 3


def test_ends_of_the_ranges():
    """Random numbers of 0 and next to 1 and beyond, limits of zero, above one, negative and NaN."""
    logits, _ = case(1, 9001, 1.0, 10)
    logits = logits.expand(6, -1).contiguous()
    uniforms = torch.tensor([0.0, 1.0 - 2.0 ** -24, 1.0, 7.0, -1.0, float("nan")], device=DEVICE)
    ordinary = torch.tensor([0.0, 1.0 - 2.0 ** -24, 1.0, 1.0, 0.0, 0.0], device=DEVICE)
    k = ops.current()
    for limits in ((1.0, 0, 1.0, 0.0), (1.0, 30, 0.9, 0.0), (1.0, 0, 0.9, 0.0), (1.0, 0, 1.0, 0.1)):
        assert torch.equal(k.sample_limited(logits, uniforms, limits_of([limits] * 6)), k.sample_limited(logits, ordinary, limits_of([limits] * 6)))
    best = int(logits[0].argmax())
    for limits in ((1.0, 0, 0.0, 0.0), (1.0, 0, -1.0, 0.0), (1.0, 0, 1e-30, 0.0), (1.0, 0, 1.0, 1.0), (1.0, 0, 1.0, 9.0), (-1.0, 0, 1.0, 0.0),
                   (float("nan"), 0, 1.0, 0.0)):
        assert k.sample_limited(logits, uniforms, limits_of([limits] * 6)).tolist() == [best] * 6
    free = k.sample_limited(logits, ordinary, limits_of([(1.0, 0, 1.0, 0.0)] * 6))
    for limits in ((1.0, -5, 1.0, 0.0), (1.0, 0, float("nan"), 0.0), (1.0, 0, 1.0, float("nan")), (1.0, 9001, 3.0, -1.0)):
        assert torch.equal(k.sample_limited(logits, ordinary, limits_of([limits] * 6)), free)


def test_limits_by_slot_views_and_rows_of_no_slot():
    logits, uniforms = case(5, 3001, 2.0, 11)
    limits = limits_of([LIMITS[i] for i in (1, 2, 3, 4, 5, 6)])
    slots = torch.tensor([4, 0, 9, -1, 2], dtype=torch.int32, device=DEVICE)
    odd = torch.empty(5 * 3001 + 3, device=DEVICE)[3:].view(5, 3001).copy_(logits)          # on no 16-byte boundary
    got = ops.current().sample_limited(odd, uniforms, limits, slots).tolist()
    for row, slot in enumerate(slots.tolist()):
        if 0 <= slot < 6:
            t, k, p, least = LIMITS[slot + 1]
            want, near = chosen(logits[row], float(uniforms[row]), *(float(torch.tensor(x)) if x is not k else x for x in (t, k, p, least)))
            assert got[row] == want or near < NEAR
        else:
            assert got[row] == int(logits[row].argmax())
    assert ops.current().sample_limited(logits[:0], uniforms[:0], limits, slots[:0]).shape == (0,)


def test_a_row_does_not_depend_on_the_others_nor_on_a_replay():
    logits, uniforms = case(120, 30011, 2.0, 12)
    rows = [LIMITS[i % len(LIMITS)] for i in range(120)]
    k = ops.current()
    whole = k.sample_limited(logits, uniforms, limits_of(rows))
    for i in range(0, 120, 7):
        assert int(k.sample_limited(logits[i:i + 1], uniforms[i:i + 1], limits_of(rows[i:i + 1]))) == int(whole[i])
    limits = limits_of(rows)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        k.sample_limited(logits, uniforms, limits)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = k.sample_limited(logits, uniforms, limits)
        logits.copy_(logits.roll(1, 0))
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, k.sample_limited(logits, uniforms, limits))


def test_what_is_refused():
    k = ops.current()
    logits, uniforms = case(3, 100, 1.0, 13)
    limits = limits_of(LIMITS[:3])
    slots = torch.zeros(3, dtype=torch.int32, device=DEVICE)
    for call in (lambda: k.sample_limited(logits, uniforms[:2], limits), lambda: k.sample_limited(logits[:2], uniforms[:2], limits),
                 lambda: k.sample_limited(logits.double(), uniforms, limits), lambda: k.sample_limited(logits, uniforms.double(), limits),
                 lambda: k.sample_limited(logits.t(), uniforms, limits), lambda: k.sample_limited(logits, uniforms, limits, slots[:2]),
                 lambda: k.sample_limited(logits, uniforms, limits, slots.long()), lambda: k.sample_limited(logits.cpu(), uniforms, limits),
                 lambda: k.sample_limited(logits, uniforms, ops.SamplingLimits(top_k=limits.top_k)), lambda: ops.SamplingLimits(),
                 lambda: ops.SamplingLimits(limits.temperatures, limits.top_k[:2]), lambda: ops.SamplingLimits(top_p=limits.top_k),
                 lambda: k.sample_slots(logits, slots, torch.zeros((5, 8), dtype=torch.int32, device=DEVICE), limits=limits)):
        with pytest.raises(ops.KernelError):
            call()


@pytest.mark.parametrize("rows,vocab", [(300, 50257), (280, 8191), (70, 152065), (20, 1400001)])
def test_many_rows_on_odd_boundaries(rows, vocab):
    """One to four CTAs a row, slices that stay in shared memory and such that are read again, rows that begin on no 16-byte boundary."""
    logits, uniforms = case(rows, vocab, 2.5, rows)
    limits = [LIMITS[i % len(LIMITS)] for i in range(rows)]
    got = ops.current().sample_limited(logits, uniforms, limits_of(limits)).tolist()
    for row in range(0, rows, 3):
        t, k, p, least = limits[row]
        want, near = chosen(logits[row], float(uniforms[row]), *(float(torch.tensor(x)) if x is not k else x for x in (t, k, p, least)))
        assert got[row] == want or near < NEAR, (row, limits[row])


@pytest.mark.parametrize("rows", [1, 60])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_logits_rounded_to_16_bits(rows, dtype):
    """Many equal logits in every place, more than a thousand at a cut."""
    logits, uniforms = case(rows, 151936, 2.0, 13)
    logits = logits.to(dtype).float()
    check(logits, uniforms, [[(1.0, 0, 0.9, 0.0), (1.0, 0, 0.5, 0.0), (0.6, 0, 0.95, 0.0), (1.0, 9000, 0.99, 0.0), (1.0, 0, 0.97, 1e-4)][i % 5] for i in range(rows)])


@pytest.mark.parametrize("rows", [1, 40])
def test_the_likely_tokens_side_by_side(rows):
    """All in one warp's stretch, in falling and in rising order, and a few far above the rest."""
    vocab = 100352
    logits, uniforms = case(rows, vocab, 1.0, 14)
    falling = torch.sort(logits, dim=1, descending=True).values
    for kind in (falling, falling.flip(1), torch.cat([falling[:, :6] + 9.0, logits[:, 6:]], 1)):
        for limits in ((0.8, 1000, 1.0, 0.0), (0.8, 1200, 0.95, 0.0), (0.4, 0, 0.9, 0.0), (0.25, 0, 0.8, 0.0), (0.5, 0, 1.0, 0.05), (1.0, 0, 1.0, 0.0)):
            check(kind.contiguous(), uniforms, [limits] * rows)


def test_long_rows_in_an_order_of_their_own():
    """More rows than are taken at once, read by slot: the order in which they are taken changes none of them."""
    rows, vocab = 110, 81931
    logits, uniforms = case(rows, vocab, 2.5, 15)
    limits = [LIMITS[i % len(LIMITS)] for i in range(rows + 7)]
    slots = torch.randperm(rows + 7, generator=torch.Generator().manual_seed(16))[:rows].to(torch.int32)
    slots[[3, 50]] = torch.tensor([-1, rows + 7], dtype=torch.int32)
    tables, k = limits_of(limits), ops.current()
    got = k.sample_limited(logits, uniforms, tables, slots.to(DEVICE)).tolist()
    for row, slot in enumerate(slots.tolist()):
        alone = k.sample_limited(logits[row:row + 1], uniforms[row:row + 1], tables, slots[row:row + 1].to(DEVICE))
        assert got[row] == int(alone), (row, slot)
        if row in (3, 50):
            assert got[row] == int(logits[row].argmax())
