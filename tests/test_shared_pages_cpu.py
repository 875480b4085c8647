"""Requests that start with another's pages, on the CPU: the cache manager under random orders, what it refuses, and the engine with
stand-ins for the kernels (which tokens run through the model, which steps take the shared attention, what a prefix outlives)."""

from __future__ import annotations

import random

import numpy as np
import pytest
import torch

import plain_qwen2 as plain
from fake_ops import FakeOps
from harness import TinyEngine, random_prompt
from mini_llm_runtime_b200 import ops
from mini_llm_runtime_b200.cache import OutOfPages
from mini_llm_runtime_b200.engine import ContinuousBatchEngine, StepEntry
from mini_llm_runtime_b200.ops import KernelError, cuda_ops
from mini_llm_runtime_b200.parts import StateNeed
from test_cache_manager import FULL, WINDOW, manager
from tiny_configs import TINY


class SharedFakeOps(FakeOps):
    """The stand-ins with shared prefixes: the plan is the real one, the attention is the one of every request by itself."""

    def __init__(self):
        self.shared_calls = []

    def plan_shared_prefix(self, groups, num_segments, heads_per_kv):
        return cuda_ops.plan_shared_prefix(groups, num_segments, heads_per_kv)

    def shares_prefix(self, dtype, counts, num_kv_heads, head_dim):
        return True

    def shared_prefix_attention(self, q, k_pool, v_pool, batch, prefix, heads, kv_heads, dim, scale):
        plan, counts = prefix.plan, prefix.counts
        assert counts["segments"] == batch.num_segments == q.shape[0]
        for first, count, keys in zip(plan["tile_first"].tolist(), plan["tile_count"].tolist(), plan["tile_keys"].tolist()):
            rows = [batch.block_table[int(batch.seg_slot[m])][:keys // k_pool.shape[2]].tolist()
                    for m in plan["members"][first:first + count].tolist()]
            assert all(row == rows[0] and min(row) >= 0 for row in rows), "the members' tables start with the same pages"
        self.shared_calls.append(plan["seg_keys"].tolist())
        return self.paged_attention(q, k_pool, v_pool, batch, heads, kv_heads, dim, scale, None)


@pytest.fixture
def kernels(monkeypatch):
    monkeypatch.setattr(cuda_ops, "_need", lambda *args, **kwargs: None)
    stand_in = SharedFakeOps()
    with ops.use(stand_in):
        yield stand_in


# ------------------------------------------------------------------ the cache manager
def test_a_request_starts_with_anothers_pages():
    m = manager(pages=8, page=4)
    m.create_request("source")
    m.begin_step([("source", 10)])
    m.commit_step()
    request = m.create_request("a", prefix=("source", 8))
    assert request.committed == 8 and request.shared_pages == 2 and m.get("source").sharers == 1
    assert int(m.slot_mirror[request.slot, 0]) == 8, "the device record starts behind the shared tokens"
    m.check_consistency()
    m.begin_step([("a", 5), ("source", 1)])
    m.commit_step()
    for group in m.groups:
        row = group.table[request.slot]
        assert list(row[:2]) == m.get("source").pages[group.index][:2] and len(set(row[:4])) == 4
    m.check_consistency()
    with pytest.raises(RuntimeError, match="start with"):
        m.release("source")
    freed = m.release("a")
    assert all(len(ids) == 2 for ids in freed.values()), "its own pages only"
    m.release("source")
    m.check_consistency()
    assert m.stats().free_pages == (8,) and m.stats().live_requests == 0


def test_an_aborted_step_leaves_shared_pages():
    m = manager(pages=8, page=4)
    m.create_request("source")
    m.adopt("source", 8)
    request = m.create_request("a", prefix=("source", 8))
    m.begin_step([("a", 6)])
    m.abort_step()
    m.check_consistency()
    assert request.committed == 8 and [len(p) for p in request.pages] == [2] * len(m.groups)


def test_a_promise_counts_own_pages_only():
    m = manager(needs=(FULL,), pages=6, page=4)
    m.create_request("source", lifetime_tokens=12)          # 3 pages
    m.adopt("source", 12)
    assert m.create_request("a", lifetime_tokens=24) is None, "six pages do not fit beside three"
    first = m.create_request("a", lifetime_tokens=20, prefix=("source", 12))     # two of its own
    assert first is not None and m.create_request("b", lifetime_tokens=20, prefix=("source", 12)) is None
    assert m.create_request("b", lifetime_tokens=16, prefix=("source", 12)) is not None
    m.begin_step([("a", 8), ("b", 4)])
    m.commit_step()
    m.check_consistency()
    with pytest.raises(OutOfPages):
        m.begin_step([("a", 1)])
    for name in ("a", "b", "source"):
        m.release(name)
    assert m.stats().promised_pages == (0,) and m.stats().free_pages == (6,)


@pytest.mark.parametrize("prefix", [("source", 0), ("source", 6), ("source", 12), ("source", -4)])
def test_tokens_that_cannot_be_shared(prefix):
    m = manager(pages=8, page=4)
    m.create_request("source")
    m.adopt("source", 10)
    with pytest.raises(ValueError):
        m.create_request("a", prefix=prefix)
    with pytest.raises(KeyError):
        m.create_request("a", prefix=("nobody", 4))
    with pytest.raises(ValueError, match="of its own"):
        m.create_request("a", lifetime_tokens=8, prefix=("source", 8))
    assert m.stats().live_requests == 1 and m.get("source").sharers == 0
    m.check_consistency()


@pytest.mark.parametrize("needs", [(FULL, WINDOW), (FULL, StateNeed((3,), torch.float32)), (WINDOW,)])
def test_windows_and_states_share_nothing(needs):
    m = manager(needs=needs, pages=8, page=4)
    assert not m.can_share_pages
    m.create_request("source")
    m.adopt("source", 8)
    with pytest.raises(ValueError, match="every key"):
        m.create_request("a", prefix=("source", 4))


@pytest.mark.parametrize("seed", range(4))
def test_random_orders_with_sharing(seed):
    rng = random.Random(seed)
    m = manager(pages=40, page=4, requests=7, tokens=64)
    names = 0
    for _ in range(400):
        live = list(m.requests.values())
        action = rng.random()
        if action < 0.3 and m.slots.free_count:
            names += 1
            sources = [r for r in live if r.committed >= 4]
            prefix = None
            if sources and rng.random() < 0.7:
                source = rng.choice(sources)                # one that shares itself, too
                prefix = (source.request_id, 4 * rng.randint(1, source.committed // 4))
            if prefix is None or prefix[1] < 60:
                m.create_request(f"r{names}", prefix=prefix)
        elif action < 0.8 and live:
            chosen = [r for r in rng.sample(live, rng.randint(1, len(live))) if r.committed + 9 <= 64]
            try:
                if chosen:
                    m.begin_step([(r.request_id, rng.randint(1, 9)) for r in chosen])
                    m.commit_step() if rng.random() < 0.8 else m.abort_step()
            except OutOfPages:
                pass
        elif live:
            request = rng.choice(live)
            if request.sharers:
                with pytest.raises(RuntimeError):
                    m.release(request.request_id)
            else:
                m.release(request.request_id)
        m.check_consistency()
    while m.requests:
        for request in list(m.requests.values()):
            if not request.sharers:
                m.release(request.request_id)
    m.check_consistency()
    assert all(free == 40 for free in m.stats().free_pages)


# ------------------------------------------------------------------ the engine
def engine_of(tiny, name="A", **options):
    return ContinuousBatchEngine.from_model(tiny.model, block_size=TINY[name][1], max_running_requests=3, max_batch_tokens=24, max_model_len=160,
                                            **{"max_prefixes": 2, **options})


@pytest.fixture
def tiny():
    return TinyEngine(*TINY["A"], torch.float32, "cpu")


def plain_tokens(tiny, prompt, count):
    return plain.greedy_tokens(tiny.tensors, tiny.config_dict, prompt, count)


def test_prompts_behind_a_shared_prefix(tiny, kernels):
    """Five requests over three places behind two prefixes and none: the plain loop's tokens; what is shared is computed once."""
    vocab = tiny.config.vocab_size
    engine = engine_of(tiny)
    long, short = random_prompt(vocab, 70, 1), random_prompt(vocab, 16, 2)
    assert engine.add_prefix("long", long) == 64 and engine.add_prefix("short", short) == 16
    rows = []
    forward = tiny.model.forward
    tiny.model.forward = lambda ctx: (rows.append(ctx.num_rows), forward(ctx))[1]
    prompts = {"a": long + [5, 6, 7], "b": long + random_prompt(vocab, 9, 3), "c": random_prompt(vocab, 20, 4), "d": short + [9], "e": long[:65]}
    named = {"a": "long", "b": "long", "d": "short", "e": "long"}
    for name, prompt in prompts.items():
        engine.submit(name, prompt, max_new_tokens=5, prefix=named.get(name))
    engine.run()
    for name, prompt in prompts.items():
        assert list(engine.scheduler.get_request(name).generated_token_ids) == plain_tokens(tiny, prompt, 5), name
    prompt_rows = 3 + 6 + 9 + 6 + 20 + 1 + 1          # behind the whole pages: 73, 79 and 65 less 64, 20, 17 less 16
    assert sum(rows) == prompt_rows + 5 * 4, "each further token is one row"
    assert any(sorted(call) == [0, 64, 64] for call in kernels.shared_calls), "two of three decoded together share"
    engine.manager.check_consistency()
    for name in ("long", "short"):
        engine.drop_prefix(name)
    assert engine.manager.stats().live_requests == 0
    assert engine.manager.stats().free_pages == engine.manager.stats().total_pages


def test_a_prefix_outlives_its_requests(tiny, kernels):
    engine = engine_of(tiny)
    prefix = random_prompt(tiny.config.vocab_size, 32, 1)
    engine.add_prefix("p", prefix)
    engine.submit("a", prefix + [3], max_new_tokens=4, prefix="p")
    with pytest.raises(RuntimeError, match="shared by"):
        engine.drop_prefix("p")                       # waiting
    engine.step()
    with pytest.raises(RuntimeError, match="shared by"):
        engine.drop_prefix("p")                       # running
    engine.run()
    engine.drop_prefix("p")
    with pytest.raises(KeyError):
        engine.drop_prefix("p")
    with pytest.raises(ValueError, match="no prefix"):
        engine.submit("b", prefix + [3], max_new_tokens=4, prefix="p")
    engine.add_prefix("p", prefix)                    # the name is free again
    engine.submit("b", prefix + [3], max_new_tokens=4, prefix="p")
    engine.run()
    assert list(engine.scheduler.get_request("b").generated_token_ids) == plain_tokens(tiny, prefix + [3], 4)


def test_a_step_that_fails_leaves_the_prefix(tiny, kernels, monkeypatch):
    engine = engine_of(tiny)
    prefix = random_prompt(tiny.config.vocab_size, 32, 1)
    engine.add_prefix("p", prefix)
    engine.submit("a", prefix + [3, 4], max_new_tokens=3, prefix="p")
    forward, failures = tiny.model.forward, [1]

    def once(ctx):
        if failures:
            failures.pop()
            raise RuntimeError("made by the test")
        return forward(ctx)

    monkeypatch.setattr(tiny.model, "forward", once)
    with pytest.raises(RuntimeError, match="made by the test"):
        engine.step()
    engine.manager.check_consistency()
    engine.run()
    assert list(engine.scheduler.get_request("a").generated_token_ids) == plain_tokens(tiny, prefix + [3, 4], 3)


def test_a_prefix_that_fails_gives_its_pages_back(tiny, kernels, monkeypatch):
    engine = engine_of(tiny)
    monkeypatch.setattr(tiny.model, "forward", lambda ctx: (_ for _ in ()).throw(RuntimeError("made by the test")))
    with pytest.raises(RuntimeError, match="made by the test"):
        engine.add_prefix("p", random_prompt(tiny.config.vocab_size, 40, 1))
    assert engine.manager.stats().live_requests == 0 and engine.manager.stats().free_pages == engine.manager.stats().total_pages


def test_a_device_error_while_a_prefix_is_computed(tiny, kernels):
    """Found at the end of ``add_prefix``, not by the requests that would start with it."""
    engine = engine_of(tiny)
    tokens = random_prompt(tiny.config.vocab_size, 40, 1)
    engine.submit("a", tokens[:9], max_new_tokens=3)
    engine.step()
    kernels.error_code = 3
    with pytest.raises(KernelError, match="bounded wait"):
        engine.add_prefix("p", tokens)
    assert list(engine.manager.requests) == ["a"]
    engine.run()
    assert list(engine.scheduler.get_request("a").generated_token_ids) == plain_tokens(tiny, tokens[:9], 3)
    engine.add_prefix("p", tokens)
    engine.submit("b", tokens, max_new_tokens=3, prefix="p")
    engine.run()
    assert list(engine.scheduler.get_request("b").generated_token_ids) == plain_tokens(tiny, tokens, 3)


def test_prefixes_that_are_refused(tiny, kernels):
    engine = engine_of(tiny, max_prefixes=1)
    vocab = tiny.config.vocab_size
    tokens = random_prompt(vocab, 40, 1)
    for bad in (tokens[:15], [], [-1] * 20, [vocab] * 20):
        with pytest.raises(ValueError):
            engine.add_prefix("p", bad)
    engine.add_prefix("p", tokens)
    with pytest.raises(ValueError, match="exists"):
        engine.add_prefix("p", tokens)
    with pytest.raises(ValueError, match="made for 1"):
        engine.add_prefix("q", tokens)
    for prompt in ([1] + tokens, tokens[:20] + [tokens[20] ^ 1] + tokens[21:] + [4]):
        with pytest.raises(ValueError, match="does not start"):
            engine.submit("a", prompt, max_new_tokens=2, prefix="p")
    engine.submit("short", tokens[:10], max_new_tokens=2, prefix="p")     # fewer tokens than a page: nothing to share, nothing wrong
    engine.run()
    assert list(engine.scheduler.get_request("short").generated_token_ids) == plain_tokens(tiny, tokens[:10], 2)
    none = ContinuousBatchEngine.from_model(tiny.model, block_size=TINY["A"][1], max_running_requests=1, max_model_len=96)
    with pytest.raises(ValueError, match="made for 0"):
        none.add_prefix("p", tokens)


def test_requests_and_prefixes_do_not_share_names(tiny, kernels):
    engine = engine_of(tiny)
    tokens = random_prompt(tiny.config.vocab_size, 40, 1)
    engine.submit("prefix p", tokens, max_new_tokens=2)
    with pytest.raises(ValueError, match="is called"):
        engine.add_prefix("p", tokens)
    engine.run()
    engine.add_prefix("p", tokens)
    engine.add_prefix("q", tokens)
    with pytest.raises(ValueError, match="holds a prefix"):
        engine.submit("prefix q", tokens, max_new_tokens=2)
    engine.submit("b", tokens, max_new_tokens=2, prefix="p")
    engine.run()
    assert list(engine.scheduler.get_request("b").generated_token_ids) == plain_tokens(tiny, tokens, 2)


def test_groups_too_small_for_lists_need_no_step_of_their_own(tiny, kernels, monkeypatch):
    cache, runner = tiny.cache, tiny.runner
    page = TINY["A"][1]
    cache.create_request("p")
    runner.step([StepEntry("p", random_prompt(tiny.config.vocab_size, 2 * page, 1))])
    requests = [cache.create_request(name, prefix=("p", 2 * page)) for name in "abc"]
    cache.begin_step([(request.request_id, 1) for request in requests])
    assert runner._graph_key(requests, True, False)[4:] == ((3, 2 * page),)
    monkeypatch.setattr(kernels, "shares_prefix", lambda dtype, counts, kv_heads, dim: counts["members"] > 2)
    assert runner._graph_key(requests[:2], True, False)[4:] == ()
    assert runner._graph_key(requests, True, False)[4:] == ((3, 2 * page),)
    cache.abort_step()


def test_pages_of_odd_sizes_take_no_shared_attention(kernels):
    odd = TinyEngine(TINY["A"][0], 12, torch.float32, "cpu")
    cache, runner = odd.cache, odd.runner
    prefix = random_prompt(odd.config.vocab_size, 24, 1)
    cache.create_request("p")
    runner.step([StepEntry("p", prefix)])
    for name in "ab":
        cache.create_request(name, prefix=("p", 24))
    got = runner.step([StepEntry(name, [token], [0]) for name, token in (("a", 3), ("b", 4))])
    assert not kernels.shared_calls
    for row, token in enumerate((3, 4)):
        assert torch.allclose(got[row], odd.plain_logits(prefix + [token])[-1], atol=1e-4)


def test_a_model_with_windows_has_no_prefixes(kernels):
    windowed = TinyEngine(*TINY["C"], torch.float32, "cpu")
    engine = engine_of(windowed, "C")
    with pytest.raises(ValueError, match="every key"):
        engine.add_prefix("p", random_prompt(windowed.config.vocab_size, 40, 1))


def test_prompt_portions_and_mixed_steps_take_no_shared_plan(tiny, kernels):
    """A step that holds a prompt portion attends request by request; logits through the runner are the plain ones either way."""
    cache, runner = tiny.cache, tiny.runner
    vocab, page = tiny.config.vocab_size, TINY["A"][1]
    prefix = random_prompt(vocab, 2 * page, 1)
    cache.create_request("p")
    runner.step([StepEntry("p", prefix)])
    tails = {name: random_prompt(vocab, 4, seed) for name, seed in (("a", 2), ("b", 3))}
    for name in tails:
        cache.create_request(name, prefix=("p", 2 * page))
    got = [runner.step([StepEntry("a", tails["a"][:3], [2]), StepEntry("b", tails["b"][:1], [0])])]
    assert not kernels.shared_calls
    got.append(runner.step([StepEntry("a", tails["a"][3:4], [0]), StepEntry("b", tails["b"][1:2], [0])]))
    assert kernels.shared_calls == [[2 * page, 2 * page]] * len(tiny.model.blocks)
    for row, (name, upto) in enumerate((("a", 3), ("b", 1), ("a", 4), ("b", 2))):
        want = tiny.plain_logits(prefix + tails[name][:upto])[-1]
        assert torch.allclose(torch.cat(got)[row], want, atol=1e-4)


def test_lists_of_a_model_with_equal_plan_keys_and_other_heads():
    """Lists made for other heads per kv head are left alone: the layer attends request by request."""
    arrays, counts = cuda_ops.plan_shared_prefix([((0, 1), 32)], 2, 4)
    assert counts["heads_per_kv"] == 4 and np.array_equal(arrays["seg_keys"], [32, 32])
    with pytest.raises(KernelError):
        cuda_ops.plan_shared_prefix([((0, 1), 32)], 2, 200)
