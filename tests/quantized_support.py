"""A cache in 8 bits in plain numpy and torch, 64 bits, block by block: what the kernels are compared with."""

from __future__ import annotations

import numpy as np
import torch

from mini_llm_runtime_b200 import ops
from mini_llm_runtime_b200.ops import AttentionBatch


def stored(codes, scales, rows, slots, block):
    """``codes`` int8 [pages, kv_heads, page, dim] and ``scales`` float32 [pages, kv_heads, page / block] (numpy, changed in place) after
    the rows [n, kv_heads, dim] (64 bits, exact) went to ``slots``: one call's rows, block after block."""
    pages, kv_heads, page, _ = codes.shape
    done = 0
    while done < len(slots):
        slot = int(slots[done])
        if not 0 <= slot < pages * page:
            done += 1
            continue
        at, offset = divmod(slot, page)
        held = offset % block
        count = 1
        while done + count < len(slots) and held + count < block and int(slots[done + count]) == slot + count:
            count += 1
        cell, first = offset // block, offset - held
        for head in range(kv_heads):
            new = rows[done:done + count, head].astype(np.float64)
            top = np.abs(new).max()
            need = np.float32(np.float32(top) / np.float32(127.0)) if np.isfinite(top) else np.float32(np.nan)
            older = scales[at, head, cell] if held else np.float32(0.0)
            grown = np.float32(np.nan) if held and (np.isnan(older) or np.isnan(need)) else max(older, need) if held else need
            if held and not grown == older:
                before = codes[at, head, first:offset].astype(np.float64)
                codes[at, head, first:offset] = nearest(before * np.float64(older), grown)
            codes[at, head, offset:offset + count] = nearest(new, grown)
            scales[at, head, cell] = grown
        done += count


def nearest(x, scale):
    if not scale > 0:
        return np.zeros(x.shape, dtype=np.int8)
    return np.clip(np.rint(x / np.float64(scale)), -127, 127).astype(np.int8)


def values(codes, scales):
    """What codes [pages, kv_heads, page, dim] stand for, in 64 bits."""
    return codes.double() * scales.double().repeat_interleave(codes.shape[2] // scales.shape[2], dim=2)[..., None]


class Step:
    """A step over a cache in 8 bits with random contents: ``lengths`` rows of each request behind ``first`` cached tokens."""

    def __init__(self, lengths, first, heads, kv_heads, dim, page, block, dtype, seed, device="cuda:0", spare_slots=2, spare_pages=3):
        rng = np.random.default_rng(seed)
        g = torch.Generator(device=device).manual_seed(seed)
        self.lengths, self.first = np.asarray(lengths, dtype=np.int32), np.asarray(first, dtype=np.int32)
        self.heads, self.kv_heads, self.dim, self.page, self.block, self.scale = heads, kv_heads, dim, page, block, dim ** -0.5
        ends = self.first + self.lengths
        counts = [-(-int(end) // page) for end in ends]
        pages = sum(counts) + spare_pages
        ids = rng.permutation(pages).astype(np.int32).tolist()
        slots = rng.permutation(len(lengths) + spare_slots)[:len(lengths)].astype(np.int32)
        table = np.full((len(lengths) + spare_slots, max(counts) + 1), -1, dtype=np.int32)
        for i, count in enumerate(counts):
            table[slots[i], :count] = [ids.pop() for _ in range(count)]
        self.slots, self.table, self.device = slots, torch.from_numpy(table).to(device), device
        self.start = np.concatenate([[0], np.cumsum(self.lengths)[:-1]]).astype(np.int32)
        self.q = torch.randn((int(self.lengths.sum()), heads * dim), generator=g, device=device).to(dtype)

        def held():
            codes = torch.randint(-127, 128, (pages, kv_heads, page, dim), generator=g, device=device, dtype=torch.int16).to(torch.int8)
            return codes, (torch.rand((pages, kv_heads, page // block), generator=g, device=device) * 2.0 + 0.1) / 127.0

        (key, key_scales), (value, value_scales) = held(), held()
        self.pool = ops.QuantizedPool(key, value, key_scales, value_scales)

    def batch(self, limit=None):
        arrays, counts = ops.current().plan_attention(self.lengths, self.first)
        return AttentionBatch(
            seg_q_start=torch.from_numpy(self.start).to(self.device), seg_q_len=torch.from_numpy(self.lengths).to(self.device),
            seg_pos0=torch.from_numpy(self.first).to(self.device), seg_slot=torch.from_numpy(self.slots).to(self.device), block_table=self.table,
            num_segments=len(self.lengths), max_q_len=int(self.lengths.max()), max_kv_len=limit or int((self.first + self.lengths).max()),
            plan={name: torch.from_numpy(a).to(self.device) for name, a in arrays.items()}, counts=counts)

    def run(self, window=None, limit=None):
        return ops.current().quantized_attention(self.q, self.pool, self.batch(limit), self.heads, self.kv_heads, self.dim, self.scale, window)

    def place(self, i, keys):
        """Pages and offsets of the first ``keys`` keys of request i."""
        at = torch.arange(keys, device=self.device)
        return self.table[int(self.slots[i])].long()[at // self.page], at % self.page

    def check(self, got, window=None):
        """|error| of o = sum p v, p the normalised weights, A = sum p |v|, n keys.  Half a step of the result's type.  A times the relative
        errors of a weight and of its place in the sum: twice the score's error (a dot product of dim terms in 32 bits, the scales'
        products and the sum with a value's exponent, |log2 vs| < 16: (dim + 8) 2^-24 sum |q||k| scale + 16 2^-23), e^x off by 2^-20, sums
        of n terms 4 sqrt(n) 2^-24.  On the tensor cores weights times the values' scales are held in float16 relative to the row's
        largest: half a step 2^-11 of each, and 2^-25 of the largest for those too small to have all bits.  A prompt's keys and values
        are there in float16 themselves, code times scale rounded by half a step 2^-11 relative to each (beside powers of two, exact): the
        values' rounding moves o by 2^-11 A at most, the keys' a score by 2^-11 sum |q||k| scale, and a weight, which has its own score
        in it and the others' in the sum that divides it, by twice that; 2^-25 of the tile's largest scale for values too small to have
        all bits, weighed by p, sum p = 1."""
        assert got.dtype == self.q.dtype and bool(torch.isfinite(got).all())
        u = torch.finfo(got.dtype).eps / 2
        cores = got.dtype == torch.bfloat16
        per = self.heads // self.kv_heads
        keys_of, values_of = values(self.pool.key, self.pool.key_scales), values(self.pool.value, self.pool.value_scales)
        for i, (rows, first) in enumerate(zip(self.lengths.tolist(), self.first.tolist())):
            n = first + rows
            page, offset = self.place(i, n)
            k, v = keys_of[page, :, offset].permute(1, 0, 2), values_of[page, :, offset].permute(1, 0, 2)
            vs = self.pool.value_scales[page, :, offset // self.block].double().T
            at = int(self.start[i])
            q = self.q[at:at + rows].double().view(rows, self.kv_heads, per, self.dim).permute(1, 2, 0, 3)
            position = first + torch.arange(rows, device=self.device)[:, None]
            key = torch.arange(n, device=self.device)[None, :]
            hidden = (key > position) | ((key <= position - window) if window else torch.zeros_like(key > position))
            scores = torch.matmul(q, k.transpose(1, 2)[:, None]) * self.scale
            p = torch.softmax(scores.masked_fill(hidden, -torch.inf), dim=-1)
            want = torch.matmul(p, v[:, None])
            a = torch.matmul(p, v.abs()[:, None])
            size = (torch.matmul(q.abs(), k.abs().transpose(1, 2)[:, None]) * self.scale).masked_fill(hidden, 0.0).amax(-1, keepdim=True)
            relative = 2 * ((self.dim + 8) * 2.0 ** -24 * size + 16 * 2.0 ** -23) + 2.0 ** -20 + 4 * n ** 0.5 * 2.0 ** -24
            bound = u * want.abs() + a * relative
            if cores:
                bound = bound + a * 2.0 ** -11 + n * 2.0 ** -25 * 127 * (p * vs[:, None, None, :]).amax(-1, keepdim=True)
                if rows > 1 and self.dim in (64, 128):
                    bound = bound + a * (2.0 ** -11 + 2 * 2.0 ** -11 * size) + 2.0 ** -25 * 127 * vs.amax(-1)[:, None, None, None]
            mine = got[at:at + rows].double().view(rows, self.kv_heads, per, self.dim).permute(1, 2, 0, 3)
            worst = ((mine - want).abs() / bound.clamp_min(1e-300)).max()
            assert float(worst) <= 1.0, f"request {i} of {rows} rows behind {first}: {float(worst):.3f} of what is allowed"
