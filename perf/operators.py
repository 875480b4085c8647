"""What requests of one batch bring of their own and have in common, as cases that can be timed and compared.

Three operators of a serving step: attention of decoded tokens whose requests share a long prefix (``prefix``), a
projection with low-rank adapters of many requests beside its shared weight (``adapters``), and the rules of each
request on its logits before a token is chosen (``logits``).  ``run`` computes them in their plain form by elementary
torch operations, or, with ``own`` true, through the framework's entry points on the same inputs.  ``exact`` is the
definition in 64 bits, row by row.

Sizes are those of the benchmarked Qwen2.5 models: 0.5B (896 wide, 14 query and 2 key heads of 64, 4,864 inner,
151,936 tokens), 7B (3,584 wide, 28 and 4 heads of 128, 18,944 inner, 152,064 tokens), 14B (5,120 wide, 40 and 8 heads of 128).
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

PAGE = 16
IN_PROMPT = 1 << 30            # history words: this bit for a token of the prompt, below it how often it was generated
NO_TOKEN = (1 << 31) - 1       # fills the unused end of a list of biased tokens
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


def listed():
    return [
        # ---- logits: one request with penalties only, as an interactive session decodes
        {"name": "logits 1 x 151936", "kind": "logits", "rows": 1, "vocab": 151936, "slots": 8, "history": 700, "biases": 0, "grammar": False},
        # a small batch under every rule, with a vocabulary that is no multiple of anything
        {"name": "logits 8 x 32003", "kind": "logits", "rows": 8, "vocab": 32003, "slots": 16, "history": 1500, "biases": 40, "grammar": True},
        # the benchmark's largest batch with every rule
        {"name": "logits 64 x 152064", "kind": "logits", "rows": 64, "vocab": 152064, "slots": 64, "history": 4000, "biases": 300, "grammar": True},
        # four times that: as many requests as a captured step may hold
        {"name": "logits 256 x 151936", "kind": "logits", "rows": 256, "vocab": 151936, "slots": 256, "history": 2000, "biases": 16, "grammar": True},
        # ---- adapters: a single decoded token, 0.5B q|k|v
        {"name": "adapters 1 x 896 x 1152 r8", "kind": "adapters", "rows": "1", "each": False, "inner": 896, "outer": 1152, "rank": 8, "adapters": 4,
         "bare": 0, "bias": True, "dtype": "bfloat16"},
        # 24 decoded tokens in 32 bits
        {"name": "adapters 24 x 896 x 896 r12 f32", "kind": "adapters", "rows": "24", "each": True, "inner": 896, "outer": 896, "rank": 12,
         "adapters": 8, "bare": 3, "bias": False, "dtype": "float32"},
        # 64 decoded tokens of 40 tenants (some requests without an adapter), 7B down projection
        {"name": "adapters 64 x 18944 x 3584 r16", "kind": "adapters", "rows": "64", "each": True, "inner": 18944, "outer": 3584, "rank": 16,
         "adapters": 40, "bare": 6, "bias": False, "dtype": "bfloat16"},
        # a prompt step of four portions, one of them bare, beside the others' adapters, 7B gate|up
        {"name": "adapters 2048 x 3584 x 37888 r64", "kind": "adapters", "rows": "1000 513 311 224", "each": False, "inner": 3584, "outer": 37888,
         "rank": 64, "adapters": 16, "bare": 1, "bias": False, "dtype": "bfloat16"},
        # ---- prefix: two requests behind a short system prompt that ends inside a page, 0.5B
        {"name": "prefix 2 x 300", "kind": "prefix", "prefixes": "300", "members": "2", "alone": 0, "own": 60, "heads": 14, "kv_heads": 2, "dim": 64,
         "dtype": "bfloat16"},
        # sixteen requests behind two prompts and one request by itself, 0.5B
        {"name": "prefix 17 x 2048", "kind": "prefix", "prefixes": "2048 1111", "members": "9 7", "alone": 1, "own": 500, "heads": 14, "kv_heads": 2,
         "dim": 64, "dtype": "bfloat16"},
        # the benchmark's 64 requests behind one prompt of 8,192 tokens, 7B
        {"name": "prefix 64 x 8192", "kind": "prefix", "prefixes": "8192", "members": "64", "alone": 0, "own": 1024, "heads": 28, "kv_heads": 4,
         "dim": 128, "dtype": "bfloat16"},
        # 128 requests behind three long documents, 14B
        {"name": "prefix 128 x 16384", "kind": "prefix", "prefixes": "16384 9001 4100", "members": "70 33 25", "alone": 0, "own": 800, "heads": 40,
         "kv_heads": 8, "dim": 128, "dtype": "bfloat16"},
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
    kind = rng.choice(["logits", "adapters", "prefix"])
    if kind == "logits":
        rows = _spread(rng, 1, 200)
        return {"kind": kind, "rows": rows, "vocab": _spread(rng, 2000, 152064), "slots": rows + rng.randrange(0, 20),
                "history": _spread(rng, 1, 8000), "biases": rng.choice([0, 1, _spread(rng, 2, 500)]), "grammar": rng.random() < 0.6}
    if kind == "adapters":
        dtype = rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"])
        inner, outer = 8 * _spread(rng, 32, 1200), 8 * _spread(rng, 32, 1200)
        each = rng.random() < 0.6
        if each:      # decoded tokens, each of a request of its own
            rows = _several([_spread(rng, 1, 256)])
        else:         # portions of prompts
            rows = _several(_spread(rng, 2, 700 if dtype == "bfloat16" else 200) for _ in range(rng.randrange(1, 5)))
        adapters = _spread(rng, 1, 64)
        return {"kind": kind, "rows": rows, "each": each, "inner": inner, "outer": outer, "rank": rng.choice([4, 8, 12, 16, 24, 32, 64, 128]),
                "adapters": adapters, "bare": rng.randrange(0, 1 + (_numbers(rows)[0] if each else len(_numbers(rows))) // 2), "bias": rng.random() < 0.5,
                "dtype": dtype}
    heads, kv_heads, dim = rng.choice([(14, 2, 64), (28, 4, 128), (40, 8, 128), (16, 16, 64), (16, 1, 128), (12, 3, 96)])
    count = rng.randrange(1, 4)
    small = dim == 96
    return {"kind": kind, "prefixes": _several(_spread(rng, 20, 1500 if small else 12000) for _ in range(count)),
            "members": _several(_spread(rng, 1, 12 if small else 40) for _ in range(count)), "alone": rng.randrange(0, 4), "own": _spread(rng, 1, 600), "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "dtype": "float32" if small else "bfloat16"}


# ------------------------------------------------------------------ inputs
def _generator(seed):
    generator = torch.Generator(device="cuda")
    generator.manual_seed(int(seed))
    return generator


def _pack_bits(flags):
    """Truth values [n, width] as int32 words, token t in bit t % 32 of word t // 32."""
    n, width = flags.shape
    words = -(-width // 32)
    padded = torch.zeros((n, words * 32), dtype=torch.int64, device=flags.device)
    padded[:, :width] = flags
    packed = (padded.view(n, words, 32) << torch.arange(32, device=flags.device)).sum(-1)
    return torch.where(packed >= 1 << 31, packed - (1 << 32), packed).to(torch.int32)


def _prepare_logits(case, seed):
    g = _generator(seed)
    rows, vocab, slots = case["rows"], case["vocab"], case["slots"]
    logits = torch.randn((rows, vocab), generator=g, device="cuda") * 3.0
    row_slot = torch.randperm(slots, generator=g, device="cuda")[:rows].to(torch.int32)
    # a history: tokens of a prompt and generated ones, common tokens far more often than rare ones
    length = case["history"]
    ranks = torch.rand((slots, length), generator=g, device="cuda")
    tokens = (vocab * ranks ** 4).long().clamp_(max=vocab - 1)
    prompt = length // 3
    counts = torch.zeros((slots, vocab), dtype=torch.int32, device="cuda")
    counts.scatter_add_(1, tokens[:, prompt:], torch.ones_like(tokens[:, prompt:], dtype=torch.int32))
    in_prompt = torch.zeros((slots, vocab), dtype=torch.bool, device="cuda")
    in_prompt.scatter_(1, tokens[:, :prompt], True)
    counts += in_prompt.to(torch.int32) * IN_PROMPT
    penalties = torch.stack([1.0 + torch.rand(slots, generator=g, device="cuda") * 0.5,
                             torch.rand(slots, generator=g, device="cuda") * 1.5,
                             torch.rand(slots, generator=g, device="cuda") * 0.8], dim=1).contiguous()
    state = {"logits": logits, "row_slot": row_slot, "counts": counts, "seen": _pack_bits(counts != 0), "penalties": penalties,
             "bias_tokens": None, "bias_values": None, "allowed": None}
    if case["biases"]:
        width = case["biases"]
        # ascending, each token once: a random start, then steps of at least one
        steps = torch.randint(1, max(2, vocab // width), (slots, width), generator=g, device="cuda")
        tokens = torch.cumsum(steps, dim=1) - 1
        state["bias_tokens"] = torch.where(tokens < vocab, tokens, torch.full_like(tokens, NO_TOKEN)).to(torch.int32)
        state["bias_values"] = torch.randn((slots, width), generator=g, device="cuda") * 4.0
    if case["grammar"]:
        # a third of the requests under a narrow grammar, a third under a wide one, a third under none
        chance = torch.tensor([0.003, 0.7, 1.1], device="cuda")[torch.arange(slots, device="cuda") % 3]
        allowed = torch.rand((slots, vocab), generator=g, device="cuda") < chance[:, None]
        allowed[:, 0] = True
        state["allowed"] = _pack_bits(allowed)
    if own:
        from mini_llm_runtime_b200 import ops
        state["tables"] = ops.LogitTables(penalties=state["penalties"], counts=state["counts"], seen=state["seen"],
                                          bias_tokens=state["bias_tokens"], bias_values=state["bias_values"], allowed=state["allowed"])
    return state


def _adapter_rows(case):
    """Which adapter the rows take, before they are shuffled: -1 for none."""
    if case["each"]:
        rows = _numbers(case["rows"])[0]
        return [-1 if i < case["bare"] else i % case["adapters"] for i in range(rows)]
    out = []
    for i, length in enumerate(_numbers(case["rows"])):
        out += [-1 if i < case["bare"] else i % case["adapters"]] * length
    return out


def _prepare_adapters(case, seed):
    g = _generator(seed)
    dtype = DTYPES[case["dtype"]]
    rows, inner, outer, rank, count = sum(_numbers(case["rows"])), case["inner"], case["outer"], case["rank"], case["adapters"]

    def normal(*shape, scale=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)

    ids = torch.tensor(_adapter_rows(case), dtype=torch.int32, device="cuda")
    if case["each"]:
        ids = ids[torch.randperm(rows, generator=g, device="cuda")].contiguous()
    state = {"x": normal(rows, inner), "weight": normal(outer, inner, scale=inner ** -0.5),
             "bias": normal(outer) if case["bias"] else None,
             "down": normal(count, rank, inner, scale=inner ** -0.5), "up": normal(count, outer, rank, scale=rank ** -0.5),
             "scales": torch.rand(count, generator=g, device="cuda") + 0.5, "row_adapter": ids}
    if own:
        from mini_llm_runtime_b200 import ops
        state["adapters"] = ops.AdapterStack(down=state["down"], up=state["up"], scales=state["scales"])
    return state


def _contexts(case, seed):
    """Requests in the order of the batch: (group or -1, keys of its own), shuffled by the seed."""
    order = np.random.default_rng(seed)
    groups = [g for g, count in enumerate(_numbers(case["members"])) for _ in range(count)] + [-1] * case["alone"]
    lengths = 1 + (case["own"] * (np.arange(len(groups)) * 0.61803398875 % 1.0)).astype(int)
    order.shuffle(groups)
    return groups, [int(n) for n in lengths]


def _prepare_prefix(case, seed):
    g = _generator(seed)
    dtype = DTYPES[case["dtype"]]
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    groups, own_keys = _contexts(case, seed)
    count = len(groups)
    prefixes = _numbers(case["prefixes"])
    prefix_keys = [prefixes[group] if group >= 0 else 0 for group in groups]
    contexts = [a + b for a, b in zip(prefix_keys, own_keys)]
    width = -(-max(contexts) // PAGE)
    # whole pages of a prefix are shared; a page in which it ends is every request's own copy
    shared = [length // PAGE for length in prefixes]
    need = sum(shared) + sum(-(-contexts[i] // PAGE) - (shared[groups[i]] if groups[i] >= 0 else 0) for i in range(count))
    pages = np.random.default_rng(seed + 1).permutation(need + 7).astype(np.int32)
    table = np.full((count, width), -1, dtype=np.int32)
    used = 0
    lead = []
    for length in shared:
        lead.append(pages[used:used + length])
        used += length
    for i in range(count):
        held = 0
        if groups[i] >= 0:
            held = shared[groups[i]]
            table[i, :held] = lead[groups[i]]
        rest = -(-contexts[i] // PAGE) - held
        table[i, held:held + rest] = pages[used:used + rest]
        used += rest
    pool = (need + 7, kv_heads, PAGE, dim)
    state = {"q": torch.randn((count, heads * dim), generator=g, device="cuda").to(dtype),
             "k_pool": torch.randn(pool, generator=g, device="cuda").to(dtype), "v_pool": torch.randn(pool, generator=g, device="cuda").to(dtype),
             "table": torch.from_numpy(table).cuda(), "contexts": contexts, "groups": groups,
             # of a prefix the whole pages are common, and only they are shared
             "shared": [length * PAGE for length in shared], "heads": heads, "kv_heads": kv_heads, "dim": dim, "scale": dim ** -0.5}
    if own:
        from mini_llm_runtime_b200 import ops
        lengths, position = np.ones(count, dtype=np.int32), np.asarray(contexts, dtype=np.int32) - 1
        arrays, counts = ops.current().plan_attention(lengths, position)
        index = torch.arange(count, dtype=torch.int32, device="cuda")
        state["batch"] = ops.AttentionBatch(
            seg_q_start=index, seg_q_len=torch.ones_like(index), seg_pos0=torch.from_numpy(position).cuda(), seg_slot=index,
            block_table=state["table"], num_segments=count, max_q_len=1, max_kv_len=max(contexts),
            plan={name: torch.from_numpy(array).cuda() for name, array in arrays.items()}, counts=counts)
        sharing = [([i for i in range(count) if groups[i] == group], state["shared"][group]) for group in range(len(shared))]
        arrays, counts = ops.current().plan_shared_prefix(sharing, count, heads // kv_heads)
        state["prefix"] = ops.SharedPrefix(plan={name: torch.from_numpy(array).cuda() for name, array in arrays.items()}, counts=counts)
    return state


def prepare(case, seed):
    return {"kind": case["kind"],
            **{"logits": _prepare_logits, "adapters": _prepare_adapters, "prefix": _prepare_prefix}[case["kind"]](case, seed)}


# ------------------------------------------------------------------ one pass
def _unpack_bits(words, width):
    return ((words[:, :, None] >> torch.arange(32, device=words.device, dtype=torch.int32)) & 1).bool().flatten(1)[:, :width]


def _plain_logits(state):
    slot = state["row_slot"].long()
    x = state["logits"].float()
    counts = state["counts"][slot]
    repetition, presence, frequency = state["penalties"][slot].unbind(1)
    x = torch.where(counts != 0, torch.where(x > 0, x / repetition[:, None], x * repetition[:, None]), x)
    made = (counts & (IN_PROMPT - 1)).float()
    x = x - made * frequency[:, None] - (made > 0) * presence[:, None]
    if state["bias_tokens"] is not None:
        tokens, values = state["bias_tokens"][slot].long(), state["bias_values"][slot]
        padded = torch.cat([x, torch.zeros_like(x[:, :1])], dim=1)
        x = padded.scatter_add(1, tokens.clamp(max=x.shape[1]), values)[:, :-1]
    if state["allowed"] is not None:
        x = torch.where(_unpack_bits(state["allowed"][slot], x.shape[1]), x, torch.full_like(x, -math.inf))
    return x


def _plain_adapters(state):
    x = state["x"].float()
    out = x @ state["weight"].float().T
    if state["bias"] is not None:
        out = out + state["bias"].float()
    # every adapter for every row, and only the row's own one kept
    count, rank = state["down"].shape[:2]
    low = (x @ state["down"].float().flatten(0, 1).T).view(-1, count, rank)
    mine = state["row_adapter"][:, None] == torch.arange(count, device=x.device)
    low = torch.where(mine[:, :, None], low * state["scales"][:, None], torch.zeros_like(low))
    out = out + low.flatten(1) @ state["up"].float().permute(0, 2, 1).flatten(0, 1)
    return out.to(state["x"].dtype)


def _gathered(pool, table, first, last):
    """Keys or values first .. last - 1 of a request, [kv_heads, keys, dim] in 32 bits."""
    pages = table[first // PAGE:-(-last // PAGE)].long()
    rows = pool[pages].float().permute(1, 0, 2, 3).flatten(1, 2)
    start = first // PAGE * PAGE
    return rows[:, first - start:last - start]


def _plain_prefix(state):
    heads, kv_heads, dim = state["heads"], state["kv_heads"], state["dim"]
    per = heads // kv_heads
    q = state["q"].float().view(-1, kv_heads, per, dim)
    out = torch.empty_like(q)
    members = {}
    for i, group in enumerate(state["groups"]):
        members.setdefault(group if group >= 0 else -1 - i, []).append(i)
    for group, mine in members.items():
        shared = state["shared"][group] if group >= 0 else 0
        table = state["table"][mine[0]]
        keys, values = _gathered(state["k_pool"], table, 0, shared), _gathered(state["v_pool"], table, 0, shared)
        # scores of every member over the prefix, once for all
        together = torch.einsum("bkgd,ktd->bkgt", q[mine], keys) * state["scale"]
        for place, i in enumerate(mine):
            own_keys = _gathered(state["k_pool"], state["table"][i], shared, state["contexts"][i])
            own_values = _gathered(state["v_pool"], state["table"][i], shared, state["contexts"][i])
            alone = torch.einsum("kgd,ktd->kgt", q[i], own_keys) * state["scale"]
            top = alone.amax(-1, keepdim=True)
            if shared:
                top = torch.maximum(top, together[place].amax(-1, keepdim=True))
            a, b = torch.exp(together[place] - top), torch.exp(alone - top)
            total = a.sum(-1, keepdim=True) + b.sum(-1, keepdim=True)
            out[i] = (torch.einsum("kgt,ktd->kgd", a, values) + torch.einsum("kgt,ktd->kgd", b, own_values)) / total
    return out.reshape(-1, heads * dim).to(state["q"].dtype)


def run(state):
    kind = state["kind"]
    if not own:
        return {"logits": _plain_logits, "adapters": _plain_adapters, "prefix": _plain_prefix}[kind](state)
    from mini_llm_runtime_b200 import ops
    kernels = ops.current()
    if kind == "logits":
        return kernels.shape_logits(state["logits"], state["row_slot"], state["tables"])
    if kind == "adapters":
        return kernels.linear_adapters(state["x"], state["weight"], state["adapters"], state["row_adapter"], bias=state["bias"])
    return kernels.shared_prefix_attention(state["q"], state["k_pool"], state["v_pool"], state["batch"], state["prefix"],
                                           state["heads"], state["kv_heads"], state["dim"], state["scale"])


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    if case["kind"] == "logits":
        rows, vocab = case["rows"], case["vocab"]
        words = 4 * -(-vocab // 32)
        # logits in and out, the plane of seen tokens, their counts, the biases, the plane of allowed tokens
        each = 8 * vocab + words + 4 * min(case["history"], vocab) + 8 * case["biases"] + (words if case["grammar"] else 0) + 16
        return {"bytes": rows * each, "flops": rows * (3 * min(case["history"], vocab) + case["biases"])}
    if case["kind"] == "adapters":
        size = 2 if case["dtype"] == "bfloat16" else 4
        rows, inner, outer, rank = sum(_numbers(case["rows"])), case["inner"], case["outer"], case["rank"]
        ids = _adapter_rows(case)
        used, adapted = len(set(ids) - {-1}), sum(i >= 0 for i in ids)
        entries = rows * (inner + outer) + inner * outer + used * rank * (inner + outer) + (outer if case["bias"] else 0)
        return {"bytes": size * entries + 4 * rows, "flops": 2 * rows * inner * outer + 2 * adapted * rank * (inner + outer)}
    size = 2 if case["dtype"] == "bfloat16" else 4
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    groups, own_keys = _contexts(case, 0)
    prefixes, members = _numbers(case["prefixes"]), _numbers(case["members"])
    # (the prefix's last keys, on a page that it does not fill, are each request's own)
    held = sum(length // PAGE * PAGE for length in prefixes)
    tails = sum(count * (length % PAGE) for length, count in zip(prefixes, members))
    total = sum(count * length for length, count in zip(prefixes, members)) + sum(own_keys)
    return {"bytes": size * (2 * kv_heads * dim * (held + tails + sum(own_keys)) + 2 * len(groups) * heads * dim),
            "flops": 4 * heads * dim * total}


# ------------------------------------------------------------------ the definition in 64 bits
def _exact_logits(case, state):
    rows = []
    for row in range(case["rows"]):
        slot = int(state["row_slot"][row])
        x = state["logits"][row].double()
        words = state["counts"][slot]
        repetition, presence, frequency = (float(p) for p in state["penalties"][slot])
        known = torch.nonzero(words).flatten()
        value, made = x[known], (words[known] % IN_PROMPT).double()
        value = torch.where(value > 0, value / repetition, value * repetition)
        x[known] = value - frequency * made - presence * made.clamp(max=1.0)
        if state["bias_tokens"] is not None:
            tokens = state["bias_tokens"][slot].long()
            live = tokens < case["vocab"]
            x.index_add_(0, tokens[live], state["bias_values"][slot][live].double())
        if state["allowed"] is not None:
            index = torch.arange(case["vocab"], device=x.device)
            bits = torch.bitwise_right_shift(state["allowed"][slot][index // 32].long(), index % 32) % 2
            x[bits == 0] = -math.inf
        rows.append(x)
    return torch.stack(rows)


def _exact_adapters(state):
    x = state["x"].double()
    out = torch.mm(x, state["weight"].double().t())
    if state["bias"] is not None:
        out += state["bias"].double()
    for adapter in torch.unique(state["row_adapter"]).tolist():
        if adapter >= 0:
            rows = torch.nonzero(state["row_adapter"] == adapter).flatten()
            delta = state["up"][adapter].double() @ (state["down"][adapter].double() @ x[rows].t())
            out[rows] += float(state["scales"][adapter]) * delta.t()
    return out


def _exact_prefix(state):
    heads, kv_heads, dim = state["heads"], state["kv_heads"], state["dim"]
    rows = []
    for i, length in enumerate(state["contexts"]):
        place = torch.arange(length, device="cuda")
        page = state["table"][i].long()[place // PAGE]
        keys, values = state["k_pool"][page, :, place % PAGE].double(), state["v_pool"][page, :, place % PAGE].double()
        query = state["q"][i].double().view(kv_heads, heads // kv_heads, dim)
        weights = torch.softmax(torch.matmul(query, keys.permute(1, 2, 0)) * state["scale"], dim=-1)
        rows.append(torch.matmul(weights, values.permute(1, 0, 2)).reshape(-1))
    return torch.stack(rows)


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "logits":
        return _exact_logits(case, state)
    return _exact_adapters(state) if case["kind"] == "adapters" else _exact_prefix(state)
