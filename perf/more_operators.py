"""A cache in 8 bits, its pages, and answers drawn under limits, as cases that can be timed and compared.

Four operators of serving: attention over keys and values held in 8 bits with a scale for each block of tokens and head
(``attend``: decoded tokens, prompt portions, both in one step), storing new keys and values there (``store``), copying
pages of a cache, as forked requests and moved pages need (``pages``), and the choice of tokens under a temperature, top-k,
top-p and min-p from given random numbers (``choose``).  ``run`` computes them in their plain form by elementary torch
operations, or, with ``own`` true, through the framework's entry points on the same inputs.  ``exact`` is the definition in
64 bits, request by request and row by row.

Sizes are those of the benchmarked Qwen2.5 models: 0.5B (14 query and 2 key heads of 64, 24 layers, 151,936 tokens), 7B (28
and 4 heads of 128, 28 layers, 152,064 tokens), 14B (40 and 8 heads of 128).
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

PAGE = 16
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


def listed():
    return [
        # ---- attend: an interactive session, one token of one request, 0.5B
        {"name": "attend 1 x 700", "kind": "attend", "portions": "", "history": 0, "decodes": 1, "context": 700, "block": 16, "heads": 14,
         "kv_heads": 2, "dim": 64, "dtype": "bfloat16"},
        # 24 decoded tokens in 32 bits, heads of no power of two, blocks smaller than a page
        {"name": "attend 24 x 2500 f32", "kind": "attend", "portions": "", "history": 0, "decodes": 24, "context": 2500, "block": 4, "heads": 12,
         "kv_heads": 3, "dim": 96, "dtype": "float32"},
        # the benchmark's 64 requests with long contexts, 7B
        {"name": "attend 64 x 8192", "kind": "attend", "portions": "", "history": 0, "decodes": 64, "context": 8192, "block": 16, "heads": 28,
         "kv_heads": 4, "dim": 128, "dtype": "bfloat16"},
        # 100 requests with longer ones, 14B, a scale for each token
        {"name": "attend 100 x 16384", "kind": "attend", "portions": "", "history": 0, "decodes": 100, "context": 16384, "block": 1, "heads": 40,
         "kv_heads": 8, "dim": 128, "dtype": "bfloat16"},
        # a mixed step: portions of three prompts beside twenty decoded tokens, 0.5B
        {"name": "attend 713 + 20", "kind": "attend", "portions": "513 191 9", "history": 800, "decodes": 20, "context": 1500, "block": 16,
         "heads": 14, "kv_heads": 2, "dim": 64, "dtype": "bfloat16"},
        # a prompt's portion of a full step behind 6,000 tokens, 7B
        {"name": "attend 2048 behind 6000", "kind": "attend", "portions": "2048", "history": 6000, "decodes": 0, "context": 0, "block": 16,
         "heads": 28, "kv_heads": 4, "dim": 128, "dtype": "bfloat16"},
        # ---- store: a decode step of 64 requests, whose blocks are under way, 7B
        {"name": "store 64", "kind": "store", "portions": "", "decodes": 64, "block": 16, "kv_heads": 4, "dim": 128, "dtype": "bfloat16"},
        # a full prompt step of two portions beside eight decoded tokens, 14B
        {"name": "store 2048 + 8", "kind": "store", "portions": "1301 747", "decodes": 8, "block": 16, "kv_heads": 8, "dim": 128,
         "dtype": "bfloat16"},
        # ---- pages: one request forks inside a page, 0.5B
        {"name": "pages 1 x 24", "kind": "pages", "moves": 1, "entries": 24, "pages": 96, "kv_heads": 2, "dim": 64, "dtype": "bfloat16"},
        # pages of requests that ended leave holes, into which 300 of the others move, 7B
        {"name": "pages 300 x 28", "kind": "pages", "moves": 300, "entries": 28, "pages": 700, "kv_heads": 4, "dim": 128, "dtype": "bfloat16"},
        # ---- choose: an interactive session under the usual limits
        {"name": "choose 1 x 151936", "kind": "choose", "rows": 1, "vocab": 151936, "limits": "k p", "spread": 3.0},
        # as many requests as a captured step may hold, each under limits of its own, some under none, some greedy
        {"name": "choose 256 x 152064", "kind": "choose", "rows": 256, "vocab": 152064, "limits": "mixed", "spread": 3.0},
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over the logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def _several(numbers):
    """A case holds numbers and texts: several numbers are a text."""
    return " ".join(str(n) for n in numbers)


def _numbers(text):
    return [int(n) for n in text.split()]


def draw(rng):
    kind = rng.choice(["attend", "attend", "store", "pages", "choose"])
    if kind == "choose":
        return {"kind": kind, "rows": _spread(rng, 1, 200), "vocab": _spread(rng, 2000, 152064),
                "limits": rng.choice(["k p", "k", "p", "min", "k min", "none", "mixed", "mixed"]), "spread": round(rng.uniform(1.0, 5.0), 2)}
    if kind == "pages":
        entries, moves = rng.choice([24, 28, 48]), _spread(rng, 1, 200)
        return {"kind": kind, "moves": moves, "entries": entries, "pages": 2 * moves + _spread(rng, 1, 100), "kv_heads": rng.choice([1, 2, 4]),
                "dim": rng.choice([64, 96, 128]), "dtype": rng.choice(["bfloat16", "bfloat16", "float32"])}
    heads, kv_heads, dim = rng.choice([(14, 2, 64), (28, 4, 128), (40, 8, 128), (16, 16, 64), (16, 1, 128), (12, 3, 96)])
    small = dim == 96
    block = rng.choice([1, 4, 16, 16])
    if kind == "store":
        portions = [_spread(rng, 2, 700) for _ in range(rng.randrange(0, 4))]
        return {"kind": kind, "portions": _several(portions), "decodes": _spread(rng, 1, 200), "block": block, "kv_heads": kv_heads, "dim": dim,
                "dtype": "float32" if small else "bfloat16"}
    portions = [_spread(rng, 2, 100 if small else 700) for _ in range(rng.choice([0, 0, 1, 2]))]
    return {"kind": kind, "portions": _several(portions), "history": _spread(rng, 1, 800 if small else 5000) if portions else 0,
            "decodes": _spread(rng, 1, 12 if small else 80) if not portions or rng.random() < 0.5 else 0,
            "context": _spread(rng, 1, 1500 if small else 12000), "block": block, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "dtype": "float32" if small else "bfloat16"}


# ------------------------------------------------------------------ inputs
def _generator(seed):
    generator = torch.Generator(device="cuda")
    generator.manual_seed(int(seed))
    return generator


def _portions(case):
    """(rows, first position) of every request of a step, the prompts' portions first."""
    out = [(rows, case["history"]) for rows in _numbers(case["portions"])]
    spread = (np.arange(case["decodes"]) * 0.61803398875 + 0.9) % 1.0
    return out + [(1, int(case["context"] * share)) for share in spread]


def _place(requests, seed):
    """Pages of the requests in a pool in no order: (block table [requests, widest], pages of the pool)."""
    counts = [-(-(first + rows) // PAGE) for rows, first in requests]
    total = sum(counts) + 5
    order = np.random.default_rng(seed).permutation(total).astype(np.int32)
    table = np.full((len(requests), max(counts)), -1, dtype=np.int32)
    used = 0
    for i, count in enumerate(counts):
        table[i, :count] = order[used:used + count]
        used += count
    return table, total


def _held(pages, kv_heads, dim, block, g):
    """Keys or values in 8 bits as a cache holds them, and their scales."""
    codes = torch.empty((pages, kv_heads, PAGE, dim), dtype=torch.int8, device="cuda")
    scales = torch.empty((pages, kv_heads, PAGE // block), dtype=torch.float32, device="cuda")
    for first in range(0, pages, 4096):
        x = torch.randn((min(4096, pages - first), kv_heads, PAGE // block, block * dim), generator=g, device="cuda")
        x *= torch.rand((*x.shape[:3], 1), generator=g, device="cuda") + 0.5
        scale = x.abs().amax(-1) / 127.0
        codes[first:first + 4096] = torch.round(x / scale[..., None]).to(torch.int8).view(-1, kv_heads, PAGE, dim)
        scales[first:first + 4096] = scale
    return codes, scales


def _pool(state):
    from mini_llm_runtime_b200 import ops
    return ops.QuantizedPool(key=state["key"], value=state["value"], key_scales=state["key_scales"], value_scales=state["value_scales"])


def _prepare_attend(case, seed):
    g = _generator(seed)
    requests = _portions(case)
    table, pages = _place(requests, seed)
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    state = {"requests": requests, "heads": heads, "kv_heads": kv_heads, "dim": dim, "block": case["block"], "scale": dim ** -0.5,
             "q": torch.randn((sum(rows for rows, _ in requests), heads * dim), generator=g, device="cuda").to(DTYPES[case["dtype"]]),
             "table": torch.from_numpy(table).cuda()}
    state["key"], state["key_scales"] = _held(pages, kv_heads, dim, case["block"], g)
    state["value"], state["value_scales"] = _held(pages, kv_heads, dim, case["block"], g)
    if own:
        from mini_llm_runtime_b200 import ops
        lengths, first = (np.asarray(column, dtype=np.int32) for column in zip(*requests))
        arrays, counts = ops.current().plan_attention(lengths, first)
        start = np.concatenate([[0], np.cumsum(lengths)[:-1]]).astype(np.int32)
        state["batch"] = ops.AttentionBatch(
            seg_q_start=torch.from_numpy(start).cuda(), seg_q_len=torch.from_numpy(lengths).cuda(), seg_pos0=torch.from_numpy(first).cuda(),
            seg_slot=torch.arange(len(requests), dtype=torch.int32, device="cuda"), block_table=state["table"], num_segments=len(requests),
            max_q_len=int(lengths.max()), max_kv_len=int((first + lengths).max()),
            plan={name: torch.from_numpy(array).cuda() for name, array in arrays.items()}, counts=counts)
        state["pool"] = _pool(state)
    return state


def _prepare_store(case, seed):
    g = _generator(seed)
    # a portion begins where the last step's ended, inside a page or a block; a decoded token anywhere in its page
    offsets = [int(n) for n in np.random.default_rng(seed).integers(0, PAGE, len(_numbers(case["portions"])) + case["decodes"])]
    requests = list(zip(_numbers(case["portions"]) + [1] * case["decodes"], offsets))
    table, pages = _place(requests, seed)
    kv_heads, dim, block = case["kv_heads"], case["dim"], case["block"]
    places = np.concatenate([table[i, (first + np.arange(rows)) // PAGE].astype(np.int64) * PAGE + (first + np.arange(rows)) % PAGE
                             for i, (rows, first) in enumerate(requests)])
    # keys and values lie side by side in the rows of a projection, as the layer's product leaves them
    rows = torch.randn((len(places), 2 * kv_heads * dim), generator=g, device="cuda")
    rows *= torch.rand((len(places), 1), generator=g, device="cuda") + 0.5
    state = {"rows": rows.to(DTYPES[case["dtype"]]), "slots": torch.from_numpy(places).cuda(), "places": places, "requests": requests,
             "kv_heads": kv_heads, "dim": dim, "block": block}
    state["key"], state["key_scales"] = _held(pages, kv_heads, dim, block, g)
    state["value"], state["value_scales"] = _held(pages, kv_heads, dim, block, g)
    state["all"] = torch.arange(pages, dtype=torch.int32, device="cuda")
    if own:
        state["pool"] = _pool(state)
    return state


def _prepare_pages(case, seed):
    g = _generator(seed)
    shape = (case["entries"], case["pages"], case["kv_heads"], PAGE, case["dim"])
    order = np.random.default_rng(seed).permutation(case["pages"])[:2 * case["moves"]]
    return {"pools": [torch.randn(shape, generator=g, device="cuda").to(DTYPES[case["dtype"]]) for _ in range(2)],
            "source": [int(n) for n in order[:case["moves"]]], "target": [int(n) for n in order[case["moves"]:]]}


def _prepare_choose(case, seed):
    g = _generator(seed)
    rows, vocab = case["rows"], case["vocab"]
    logits = torch.randn((rows, vocab), generator=g, device="cuda") * case["spread"]
    # a few tokens stand out, as a model's favourites do
    favourites = torch.randint(0, vocab, (rows, 12), generator=g, device="cuda")
    logits.scatter_add_(1, favourites, torch.rand((rows, 12), generator=g, device="cuda") * 4.0 * case["spread"])

    def some(values):
        return torch.tensor(values, device="cuda")[torch.randint(0, len(values), (rows,), generator=g, device="cuda")]

    limits = {"temperatures": torch.rand(rows, generator=g, device="cuda") * 0.8 + 0.4,
              "top_k": torch.zeros(rows, dtype=torch.int32, device="cuda"), "top_p": torch.ones(rows, device="cuda"),
              "min_p": torch.zeros(rows, device="cuda")}
    named = case["limits"].split()
    if "k" in named or "mixed" in named:
        limits["top_k"] = some([20, 40, 50, 100, 1000] + ([0, 0, 0, 1] if "mixed" in named else [])).to(torch.int32)
    if "p" in named or "mixed" in named:
        limits["top_p"] = some([0.8, 0.9, 0.95, 0.99] + ([1.0, 1.0] if "mixed" in named else []))
    if "min" in named or "mixed" in named:
        limits["min_p"] = some([0.02, 0.05, 0.1] + ([0.0, 0.0, 0.0] if "mixed" in named else []))
    if "mixed" in named:
        limits["temperatures"] *= torch.rand(rows, generator=g, device="cuda") < 0.9
    state = {"logits": logits, "uniforms": torch.rand(rows, generator=g, device="cuda"), **limits}
    if own:
        from mini_llm_runtime_b200 import ops
        state["limits"] = ops.SamplingLimits(**limits)
    return state


def prepare(case, seed):
    return {"kind": case["kind"],
            **{"attend": _prepare_attend, "store": _prepare_store, "pages": _prepare_pages, "choose": _prepare_choose}[case["kind"]](case, seed)}


# ------------------------------------------------------------------ one pass
def _values(codes, scales):
    """What codes [.., kv_heads, tokens, dim] with scales [.., kv_heads, blocks] stand for, in 32 bits."""
    return codes.float() * scales.repeat_interleave(codes.shape[-2] // scales.shape[-1], dim=-1)[..., None]


def _plain_attend(state):
    heads, kv_heads, dim = state["heads"], state["kv_heads"], state["dim"]
    per = heads // kv_heads
    out = torch.empty_like(state["q"])
    row = 0
    for i, (rows, first) in enumerate(state["requests"]):
        last = first + rows
        pages = state["table"][i, :-(-last // PAGE)].long()
        keys, values = (_values(state[name][pages], state[name + "_scales"][pages]).permute(1, 0, 2, 3).flatten(1, 2)[:, :last]
                        for name in ("key", "value"))
        q = state["q"][row:row + rows].float().view(rows, kv_heads, per, dim)
        hidden = torch.arange(last, device=q.device) > first + torch.arange(rows, device=q.device)[:, None]
        mixed = torch.empty_like(q)
        for h in range(kv_heads):
            scores = (q[:, h].flatten(0, 1) @ keys[h].T).view(rows, per, last) * state["scale"]
            scores.masked_fill_(hidden[:, None], -math.inf)
            weights = torch.exp(scores - scores.amax(-1, keepdim=True))
            mixed[:, h] = (weights.flatten(0, 1) @ values[h]).view(rows, per, dim) / weights.sum(-1, keepdim=True)
        out[row:row + rows] = mixed.view(rows, heads * dim).to(out.dtype)
        row += rows
    return out


def _plain_store_one(codes, scales, rows, slots, block):
    """The rows [rows, kv_heads, dim] into one pool: a block's scale grows to what its new numbers need, and the tokens that it
    held are rounded to the new scale.  A quotient next to half a step is told apart in 64 bits."""
    per_page = scales.shape[-1]
    x = rows.double()
    page, offset = slots // PAGE, slots % PAGE
    where, which = torch.unique(page * per_page + offset // block, return_inverse=True)
    first = torch.full_like(where, PAGE).scatter_reduce_(0, which, offset, "amin")      # the first new token of each block
    top = torch.zeros((len(where), x.shape[1]), device=x.device)
    top.scatter_reduce_(0, which[:, None].expand(-1, x.shape[1]), rows.float().abs().amax(-1), "amax")
    blocks = scales.permute(0, 2, 1).flatten(0, 1)[where]
    older = torch.where((first % block == 0)[:, None], torch.zeros_like(blocks), blocks)
    newer = torch.maximum(older, top / torch.full_like(top, 127.0))
    cells = codes.view(codes.shape[0], codes.shape[1], per_page, block, -1)
    held = cells[where // per_page, :, where % per_page]
    rounded = torch.round(held.double() * older[:, :, None, None].double() / newer.clamp(min=1e-30)[:, :, None, None].double())
    before = torch.arange(block, device=x.device) < (first % block)[:, None]
    cells[where // per_page, :, where % per_page] = torch.where(before[:, None, :, None], rounded.to(torch.int8), held)
    codes[page, :, offset] = torch.round(x / newer[which].clamp(min=1e-30)[:, :, None].double()).to(torch.int8)
    scales[where // per_page, :, where % per_page] = newer


def _plain_store(state):
    width = state["kv_heads"] * state["dim"]
    for name, at in (("key", 0), ("value", width)):
        rows = state["rows"][:, at:at + width].reshape(-1, state["kv_heads"], state["dim"])
        _plain_store_one(state[name], state[name + "_scales"], rows, state["slots"], state["block"])
    # whole pages, as the values they stand for; behind a block's last token lies what lay there
    return [_values(state[name], state[name + "_scales"]) for name in ("key", "value")]


def _plain_pages(state):
    source, target = (torch.tensor(state[name], device="cuda") for name in ("source", "target"))
    for pool in state["pools"]:
        pool[:, target] = pool[:, source]
    return state["pools"]


def _plain_choose(state):
    logits = state["logits"].double()
    vocab = logits.shape[1]
    temperature = state["temperatures"].double()[:, None]
    greedy = (temperature <= 0).flatten()
    order = torch.sort(logits, dim=1, descending=True, stable=True)
    scaled = order.values / torch.where(temperature > 0, temperature, torch.ones_like(temperature))
    weights = torch.exp(scaled - scaled[:, :1])
    rank = torch.arange(vocab, device=logits.device)
    k = state["top_k"].long()[:, None]
    keep = ((k <= 0) | (rank < k)) & (weights >= state["min_p"].double()[:, None])
    weights = torch.where(keep, weights, torch.zeros_like(weights))
    p = state["top_p"].double()[:, None]
    before = torch.cumsum(weights, dim=1) - weights
    weights = torch.where((p >= 1) | (before < p * weights.sum(1, keepdim=True)), weights, torch.zeros_like(weights))
    # the draw walks the tokens in the order of the vocabulary
    spread = torch.zeros_like(weights).scatter_(1, order.indices, weights)
    until = torch.cumsum(spread, dim=1)
    tokens = (until <= state["uniforms"].double()[:, None] * until[:, -1:]).sum(1)
    return torch.where(greedy, order.indices[:, 0], tokens.clamp(max=vocab - 1)).to(torch.int32)


def run(state):
    kind = state["kind"]
    if not own:
        return {"attend": _plain_attend, "store": _plain_store, "pages": _plain_pages, "choose": _plain_choose}[kind](state)
    from mini_llm_runtime_b200 import ops
    kernels = ops.current()
    if kind == "attend":
        return kernels.quantized_attention(state["q"], state["pool"], state["batch"], state["heads"], state["kv_heads"], state["dim"],
                                           state["scale"])
    if kind == "store":
        width = state["kv_heads"] * state["dim"]
        kernels.quantize_kv_write(state["rows"][:, :width], state["rows"][:, width:], state["slots"], state["pool"])
        return list(kernels.dequantize_pages(state["pool"], state["all"], torch.float32))
    if kind == "pages":
        kernels.copy_pages(state["pools"], state["source"], state["target"])
        return state["pools"]
    return kernels.sample_limited(state["logits"], state["uniforms"], state["limits"])


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    if case["kind"] == "choose":
        return {"bytes": case["rows"] * (4 * case["vocab"] + 24), "flops": 2 * case["rows"] * case["vocab"]}
    size = 2 if case["dtype"] == "bfloat16" else 4
    kv_heads, dim = case["kv_heads"], case["dim"]
    if case["kind"] == "pages":
        return {"bytes": 2 * 2 * case["moves"] * case["entries"] * kv_heads * PAGE * dim * size, "flops": 0}
    if case["kind"] == "store":
        rows = sum(_numbers(case["portions"])) + case["decodes"]
        blocks = -(-rows // case["block"])
        # the rows in, their codes and scales out, and what the codes stand for read and written once
        pages = -(-rows // PAGE)
        return {"bytes": 2 * kv_heads * (rows * dim * (size + 1) + 4 * blocks + pages * PAGE * (dim * 5 + 4 // case["block"])),
                "flops": 2 * 3 * rows * kv_heads * dim}
    requests = _portions(case)
    keys = sum(first + rows for rows, first in requests)
    seen = sum(rows * first + rows * (rows + 1) // 2 for rows, first in requests)
    rows = sum(rows for rows, _ in requests)
    return {"bytes": 2 * kv_heads * keys * dim + 2 * 4 * kv_heads * -(-keys // case["block"]) + 2 * size * rows * case["heads"] * dim,
            "flops": 4 * case["heads"] * dim * seen}


# ------------------------------------------------------------------ the definition in 64 bits
def _exact_attend(case, state):
    heads, kv_heads, dim, block = case["heads"], case["kv_heads"], case["dim"], case["block"]
    out, row = [], 0
    for i, (rows, first) in enumerate(state["requests"]):
        place = torch.arange(first + rows, device="cuda")
        page = state["table"][i].long()[place // PAGE]
        keys, values = (state[name][page, :, place % PAGE].double() * state[name + "_scales"][page, :, place % PAGE // block].double()[:, :, None]
                        for name in ("key", "value"))
        for start in range(0, rows, 128):       # a part of the rows at a time
            count = min(128, rows - start)
            at = row + start
            query = state["q"][at:at + count].double().view(count, kv_heads, heads // kv_heads, dim).permute(1, 2, 0, 3)
            scores = torch.matmul(query, keys.permute(1, 2, 0)[:, None]) * state["scale"]
            late = place[None, :] > first + start + torch.arange(count, device="cuda")[:, None]
            weights = torch.softmax(scores.masked_fill(late, -math.inf), dim=-1)
            out.append(torch.matmul(weights, values.permute(1, 0, 2)[:, None]).permute(2, 0, 1, 3).reshape(count, -1))
        row += rows
    return torch.cat(out)


def _exact_store(case, state):
    """Token by token of each request's step: the blocks one behind the other."""
    kv_heads, dim, block = case["kv_heads"], case["dim"], case["block"]
    out = []
    for name, at in (("key", 0), ("value", kv_heads * dim)):
        codes, scales = state[name].double(), state[name + "_scales"].clone()
        rows = state["rows"][:, at:at + kv_heads * dim].double().view(-1, kv_heads, dim)
        begin = 0
        for length, first in state["requests"]:
            position = first
            while position < first + length:
                end = min(first + length, position // block * block + block)
                mine = rows[begin + position - first:begin + end - first]
                slot = int(state["places"][begin + position - first])
                page, offset, cell = slot // PAGE, slot % PAGE, slot % PAGE // block
                need = (mine.abs().amax(dim=(0, 2)) / torch.full((kv_heads,), 127.0, dtype=torch.float64, device="cuda")).float()
                if position % block:
                    grown = torch.maximum(scales[page, :, cell], need)
                    held = slice(cell * block, offset)
                    codes[page, :, held] = torch.round(codes[page, :, held] * scales[page, :, cell].double()[:, None, None] / grown.double()[:, None, None])
                    need = grown
                codes[page, :, offset:offset + end - position] = torch.round(mine.permute(1, 0, 2) / need.double()[:, None, None])
                scales[page, :, cell] = need
                position = end
            begin += length
        out.append(codes * scales.double().repeat_interleave(block, dim=-1)[..., None])
    return out


def _exact_choose(case, state):
    tokens = []
    for row in range(case["rows"]):
        x = state["logits"][row].double()
        temperature = float(state["temperatures"][row])
        best = int((x == x.max()).nonzero()[0])
        if temperature <= 0:
            tokens.append(best)
            continue
        weight = torch.exp((x - x[best]) / temperature)
        down = torch.argsort(x, descending=True, stable=True)
        count, k = case["vocab"], int(state["top_k"][row])
        if k > 0:
            count = min(count, k)
        count = min(count, int((weight >= float(state["min_p"][row])).sum()))
        p = float(state["top_p"][row])
        if p < 1:
            sums = torch.cumsum(weight[down[:count]], 0)
            count = min(count, 1 + int((sums < p * sums[-1]).sum()))
        kept = torch.sort(down[:count]).values
        sums = torch.cumsum(weight[kept], 0)
        passed = int((sums <= float(state["uniforms"][row]) * sums[-1]).sum())
        tokens.append(int(kept[min(passed, count - 1)]))
    return torch.tensor(tokens, dtype=torch.int32, device="cuda")


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "pages":
        out = []
        for pool in state["pools"]:
            moved = pool.clone()
            for source, target in zip(state["source"], state["target"]):
                moved[:, target].copy_(pool[:, source])
            out.append(moved)
        return out
    if case["kind"] == "attend":
        return _exact_attend(case, state)
    return _exact_store(case, state) if case["kind"] == "store" else _exact_choose(case, state)
