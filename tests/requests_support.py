"""The stand-ins of the kernels with a cache in 8 bits, page copies and limits on what is drawn, for tests without a GPU."""

from __future__ import annotations

import torch

from fake_ops import FakeOps
from limits_support import chosen
from mini_llm_runtime_b200.cache.slots import COUNTER, LAST_TOKEN, LENGTH, read_record
from plain_qwen2 import uniform_from_seed
from quantized_support import stored


class RequestFakeOps(FakeOps):
    def __init__(self):
        self.copied = []          # (source, target) pages, call by call

    def copy_pages(self, pools, source, target, into=None):
        pools, source, target = list(pools), list(source), list(target)
        assert into is not None or not set(source) & set(target)
        assert len(set(target)) == len(target)
        self.copied.append((source, target))
        for pool, other in zip(pools, pools if into is None else into):
            for a, b in zip(source, target):
                other[:, b] = pool[:, a]

    def sample_slots(self, logits, row_slot, slot_state, advance=False, limits=None):
        if limits is None:
            return super().sample_slots(logits, row_slot, slot_state, advance)
        tokens = torch.empty(logits.shape[0], dtype=torch.int32)
        for row, slot in enumerate(row_slot.tolist()):
            record = read_record(slot_state[slot].numpy())
            u = uniform_from_seed(record["seed"], record["counter"])
            token, _ = chosen(logits[row], u, record["temperature"], int(limits.top_k[slot]), float(limits.top_p[slot]), float(limits.min_p[slot]))
            tokens[row] = token
            slot_state[slot, LAST_TOKEN] = token
            slot_state[slot, COUNTER] += 1
            if advance:
                slot_state[slot, LENGTH] += 1
        return tokens

    def rope_quantize_kv_write(self, qkv, positions, inv_freq, slots, pool, num_heads, num_kv_heads, head_dim, write_kv=True):
        turned = [torch.zeros((qkv.shape[0], num_kv_heads, 1, head_dim), dtype=qkv.dtype) for _ in range(2)]
        q = self.rope_kv_write(qkv, positions, inv_freq, torch.arange(qkv.shape[0]), *turned, num_heads, num_kv_heads, head_dim)
        if write_kv:
            for rows, codes, scales in zip(turned, (pool.key, pool.value), (pool.key_scales, pool.value_scales)):
                stored(codes.numpy(), scales.numpy(), rows[:, :, 0].double().numpy(), slots.tolist(), pool.block)
        return q

    def quantized_attention(self, q, pool, batch, num_heads, num_kv_heads, head_dim, scale, window=None):
        each = pool.key_scales.shape[2]
        key, value = (codes.float() * scales.repeat_interleave(codes.shape[2] // each, dim=2)[..., None]
                      for codes, scales in ((pool.key, pool.key_scales), (pool.value, pool.value_scales)))
        return self.paged_attention(q, key, value, batch, num_heads, num_kv_heads, head_dim, scale, window)
