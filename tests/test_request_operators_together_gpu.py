"""A decode step of requests that share a system prompt, each with an adapter and rules of its own: projections with adapters, cache
write, attention behind the shared prefix, output projection with adapters, head, rules, choice, history; eager and captured, against
the same in 64 bits, while adapters and rules change between replays."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from mini_llm_runtime_b200 import ops
from mini_llm_runtime_b200.ops import AdapterStack, AttentionBatch, LogitTables, SharedPrefix

pytestmark = pytest.mark.gpu

DEVICE = "cuda:0"
HIDDEN, HEADS, KV, DIM, VOCAB, PAGE, RANK = 256, 8, 2, 64, 1003, 16, 16


class Layer:
    def __init__(self, count, prefix, own, seed):
        g = torch.Generator(device=DEVICE).manual_seed(seed)

        def normal(*shape, scale=1.0):
            return (torch.randn(shape, generator=g, device=DEVICE) * scale).to(torch.bfloat16)

        self.count, self.prefix = count, prefix
        self.contexts = [prefix + 1 + (own * i) // count for i in range(count)]          # the new token included
        rows = (HEADS + 2 * KV) * DIM
        self.x, self.w_qkv, self.b_qkv = normal(count, HIDDEN), normal(rows, HIDDEN, scale=HIDDEN ** -0.5), normal(rows, scale=0.1)
        self.w_o, self.head = normal(HIDDEN, HEADS * DIM, scale=(HEADS * DIM) ** -0.5), normal(VOCAB, HIDDEN, scale=3 * HIDDEN ** -0.5)
        self.stacks = [AdapterStack(normal(5, RANK, k, scale=k ** -0.5), normal(5, n, RANK, scale=RANK ** -0.5),
                                    torch.rand(5, generator=g, device=DEVICE) + 0.5) for n, k in ((rows, HIDDEN), (HIDDEN, HEADS * DIM))]
        self.row_adapter = torch.tensor([i % 6 - 1 for i in range(count)], dtype=torch.int32, device=DEVICE)
        self.inv_freq = 10000.0 ** (-torch.arange(0, DIM, 2, device=DEVICE).float() / DIM)
        # pages: the prefix's are shared
        lead, width = prefix // PAGE, -(-max(self.contexts) // PAGE)
        need = lead + sum(-(-c // PAGE) - lead for c in self.contexts)
        pages = np.random.default_rng(seed).permutation(need).astype(np.int32)
        table = np.full((count, width), -1, dtype=np.int32)
        used = lead
        for i, context in enumerate(self.contexts):
            more = -(-context // PAGE) - lead
            table[i, :lead], table[i, lead:lead + more] = pages[:lead], pages[used:used + more]
            used += more
        self.k, self.v = normal(need, KV, PAGE, DIM), normal(need, KV, PAGE, DIM)
        position = np.asarray(self.contexts, dtype=np.int32) - 1
        self.places = torch.tensor([int(table[i, p // PAGE]) * PAGE + p % PAGE for i, p in enumerate(position.tolist())], device=DEVICE)
        self.positions, self.table = torch.from_numpy(position).to(DEVICE), torch.from_numpy(table).to(DEVICE)
        kernels = ops.current()
        arrays, counts = kernels.plan_attention(np.ones(count, dtype=np.int32), position)
        self.rows = torch.arange(count, dtype=torch.int32, device=DEVICE)
        self.batch = AttentionBatch(self.rows, torch.ones_like(self.rows), self.positions, self.rows, self.table, count, 1, max(self.contexts),
                                    {name: torch.from_numpy(a).to(DEVICE) for name, a in arrays.items()}, counts)
        arrays, counts = kernels.plan_shared_prefix([(range(count), prefix)], count, HEADS // KV)
        self.shared = SharedPrefix({name: torch.from_numpy(a).to(DEVICE) for name, a in arrays.items()}, counts)
        words = -(-VOCAB // 32)
        self.tables = LogitTables(
            penalties=torch.tensor([[1.0 + 0.1 * i, 0.2, 0.3] for i in range(count)], device=DEVICE),
            counts=torch.zeros((count, VOCAB), dtype=torch.int32, device=DEVICE), seen=torch.zeros((count, words), dtype=torch.int32, device=DEVICE),
            bias_tokens=torch.tensor([[i, 500 + i] for i in range(count)], dtype=torch.int32, device=DEVICE),
            bias_values=torch.full((count, 2), 1.5, device=DEVICE),
            allowed=torch.randint(-(1 << 31), 1 << 31, (count, words), generator=g, device=DEVICE).to(torch.int32))
        history = torch.randint(0, VOCAB, (count, 40), generator=g, device=DEVICE, dtype=torch.int32)
        kernels.count_tokens(history.flatten(), self.rows.repeat_interleave(40), self.tables, prompt=True)
        self.cold = torch.zeros(count, device=DEVICE), torch.zeros(count, dtype=torch.int64, device=DEVICE)

    def step(self):
        k = ops.current()
        qkv = k.linear_adapters(self.x, self.w_qkv, self.stacks[0], self.row_adapter, bias=self.b_qkv)
        q = k.rope_kv_write(qkv, self.positions, self.inv_freq, self.places, self.k, self.v, HEADS, KV, DIM)
        mixed = k.shared_prefix_attention(q, self.k, self.v, self.batch, self.shared, HEADS, KV, DIM, DIM ** -0.5)
        out = k.linear_adapters(mixed, self.w_o, self.stacks[1], self.row_adapter)
        logits = k.shape_logits_(k.linear(out, self.head, out_dtype=torch.float32), self.rows, self.tables)
        tokens = k.sample(logits, self.cold[0], self.cold[1], self.cold[1])
        k.count_tokens(tokens, self.rows, self.tables)
        return out, logits, tokens

    def projected(self, x, weight, bias, stack):
        y = x @ weight.double().T + (0 if bias is None else bias.double())
        for row, adapter in enumerate(self.row_adapter.tolist()):
            if 0 <= adapter < 5:
                y[row] += float(stack.scales[adapter]) * (stack.up[adapter].double() @ (stack.down[adapter].double() @ x[row]))
        return y

    def exact(self, counts):
        """``out`` and the ruled logits in 64 bits; the cache as the kernels left it (the new keys are rounded where they are stored)."""
        qkv = self.projected(self.x.double(), self.w_qkv, self.b_qkv, self.stacks[0])
        q = qkv[:, :HEADS * DIM].view(self.count, HEADS, DIM)
        angle = self.positions.double()[:, None] * self.inv_freq.double()
        sine, cosine = torch.sin(angle)[:, None], torch.cos(angle)[:, None]
        a, b = q[..., :DIM // 2], q[..., DIM // 2:]
        q = torch.cat([a * cosine - b * sine, b * cosine + a * sine], dim=-1)
        mixed = []
        for i, context in enumerate(self.contexts):
            place = torch.arange(context, device=DEVICE)
            page = self.table[i].long()[place // PAGE]
            keys, values = self.k[page, :, place % PAGE].double(), self.v[page, :, place % PAGE].double()
            query = q[i].view(KV, HEADS // KV, DIM)
            p = torch.softmax(query @ keys.permute(1, 2, 0) * DIM ** -0.5, dim=-1)
            mixed.append((p @ values.permute(1, 0, 2)).reshape(-1))
        out = self.projected(torch.stack(mixed), self.w_o, None, self.stacks[1])
        x = out @ self.head.double().T
        for i in range(self.count):
            repetition, presence, frequency = self.tables.penalties[i].double()
            known, n = counts[i] != 0, (counts[i] & (LogitTables.IN_PROMPT - 1)).double()
            x[i] = torch.where(known, torch.where(x[i] > 0, x[i] / repetition, x[i] * repetition), x[i]) - frequency * n - presence * (n > 0)
            x[i].index_add_(0, self.tables.bias_tokens[i].long(), self.tables.bias_values[i].double())
            index = torch.arange(VOCAB, device=DEVICE)
            x[i][(self.tables.allowed[i].long()[index // 32] >> (index % 32)) & 1 == 0] = -float("inf")
        return out, x

    def check(self, out, logits, tokens, counts):
        """Four roundings to bfloat16 lie between the 64-bit chain and ``out`` (qkv, q turned, weights and the attention's result, out
        itself), each half a step of 2^-8 of its operand, carried on by products that keep the size of a row: of its norm at most
        6 * 2^-8 with the stored keys being taken as they are; the logits are a product of the rounded row."""
        want, ruled = self.exact(counts)
        error = (out.double() - want).norm(dim=1) / want.norm(dim=1)
        assert float(error.max()) < 6 * 2 ** -8, float(error.max())
        open_ = torch.isfinite(ruled)
        assert torch.equal(torch.isfinite(logits), open_)
        size = (self.head.double().norm(dim=1)[None, :] * want.norm(dim=1)[:, None])
        # a penalty multiplies by up to 1.1 + 0.1 * count
        assert bool(((logits.double() - ruled).abs() <= 6 * 2 ** -8 * size * (1 + 0.1 * self.count))[open_].all())
        assert torch.equal(tokens.long(), logits.argmax(dim=1))
        grown = counts.clone()
        grown[torch.arange(self.count, device=DEVICE), tokens.long()] += 1
        assert torch.equal(self.tables.counts, grown)


@pytest.mark.parametrize("count", [2, 9, 40, 150])
@pytest.mark.parametrize("least", [0, None])
def test_a_step_of_tenants(monkeypatch, count, least):
    if least is not None:
        monkeypatch.setattr(ops.current(), "shared_prefix_least", least)
    layer = Layer(count, 208, 60, seed=count)
    counts = layer.tables.counts.clone()
    layer.check(*layer.step(), counts)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out, logits, tokens = layer.step()
    for turn in range(3):
        layer.row_adapter.copy_(layer.row_adapter.roll(turn + 1))
        layer.x.copy_(layer.x.roll(1, dims=0))
        layer.tables.allowed.copy_(layer.tables.allowed.roll(1, dims=1))
        counts = layer.tables.counts.clone()
        graph.replay()
        torch.cuda.synchronize()
        layer.check(out, logits, tokens, counts)
    ops.current().raise_if_device_error()


def test_two_captured_steps_of_their_own():
    """Two graphs, replayed in turn in either order: neither holds memory of the other's."""
    layers = [Layer(6, 208, 60, seed=1), Layer(30, 208, 90, seed=2)]
    ops.current().shared_prefix_least, least = 0, ops.current().shared_prefix_least
    try:
        graphs, results = [], []
        for layer in layers:
            layer.tables.penalties.copy_(torch.tensor([1.0, 0.0, 0.0], device=DEVICE))      # a history that grows then changes nothing
            layer.step()
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                results.append(layer.step())
            graphs.append(graph)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        want = [[t.clone() for t in result] for result in results]
        for result in results:
            for t in result:
                t.zero_()
        torch.cuda.synchronize()
        for graph in reversed(graphs):
            graph.replay()
        torch.cuda.synchronize()
        for result, expected in zip(results, want):
            assert all(torch.equal(a, b) for a, b in zip(result, expected))
    finally:
        ops.current().shared_prefix_least = least
