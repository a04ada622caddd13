"""The operators of a drafted decoding step over the paged 4-bit KV cache, and what their speed is measured on.

A drafted step: for every sequence the target model runs its last token and some drafted ones together, in one pass
over the weights; the drafts that the target agrees with are kept. Four kinds of call, each through
``texelator_amd.layers``, over the head layouts of the 3B- and 27B-class decoders of ``texelator_amd.modeling`` and
generic ones:

* ``rotate``  ``kv4_append_rope``: the tokens' queries and keys turned by their positions (rotary embedding, half or
              interleaved layout, all of a head or its first part, tables scaled for long contexts or not), keys and
              values stored in the cache; and ``kv4_read``: the stored rows read back as the values they stand for.
* ``tree``    ``kv4_tree_attention``: attention of the drafted tokens over the cached positions, each seeing the context
              and the drafts that lead to it.
* ``verify``  ``verify_drafts``: which drafts the target accepts, and the token behind them, from given random numbers.
* ``keep``    ``kv4_keep_path``: the accepted drafts' rows moved together in every layer's cache.

A sequence's rows: row 0 is its last token, already decided; the rows behind it are drafts. Row i follows row
parents[i] of its sequence (-1: nothing before it but the context; without parents each row follows the one before it).
The cache's format is that of ``perf/operators.py``: pages ``[pages, kv_heads, 2 (k, v), page_size * head_dim * 17 / 32]``
uint8, the packed E2M1 codes of ``page_size`` rows first (even element in the low nibble), then an E8M0 scale for each 32
elements: 2^(floor(log2(amax)) - 2), codes v / scale rounded to the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6, ties to the
even code, saturated at 6.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
MOST_ROWS = 64                       # of one sequence
MOST_TURNED = 16384 * 8              # tokens times KV heads of the largest rotate case
MOST_KEYS = 262144 * 8               # cached positions times KV heads of the largest tree case
MOST_PAIRS = 16 * 40 * 262144        # rows times heads times positions of the largest tree case
MOST_LOGITS = 24 * 64 * 32003        # rows times vocabulary of the largest verify case
MOST_POOL = 600 << 20                # bytes of the pools of the largest keep case


def listed() -> list[dict]:
    return [
        # a small tree of drafts for each of four conversations: 3B class
        {"name": "rotate_tree_3b", "kind": "rotate", "heads": 16, "kv_heads": 2, "dim": 128, "dtype": "bf16", "sequences": 4,
         "longest": 8, "prefix": 700, "page": 16, "rotary": 128, "interleaved": False, "tree": True, "ahead": 0, "mix": 1},
        # prompts of different lengths, pages entered in the middle: 27B class
        {"name": "rotate_prompts_27b", "kind": "rotate", "heads": 40, "kv_heads": 8, "dim": 128, "dtype": "bf16",
         "sequences": 7, "longest": 8192, "prefix": 500, "page": 64, "rotary": 128, "interleaved": False, "tree": False,
         "ahead": 0, "mix": 2},
        # turns of long fp16 conversations whose oldest positions were dropped, half of each head of 64 turned in pairs
        {"name": "rotate_partial_fp16", "kind": "rotate", "heads": 28, "kv_heads": 4, "dim": 64, "dtype": "fp16",
         "sequences": 9, "longest": 777, "prefix": 2500, "page": 32, "rotary": 32, "interleaved": True, "tree": False,
         "ahead": 100003, "mix": 3},
        # a few drafts of one conversation of 700 tokens: 3B class
        {"name": "tree_one_3b", "kind": "tree", "heads": 16, "kv_heads": 2, "dim": 128, "dtype": "bf16", "sequences": 1,
         "longest": 700, "rows": 6, "page": 16, "tree": True, "mix": 4},
        # trees of up to 26 rows for a batch of ordinary conversations: 27B class
        {"name": "tree_batch_27b", "kind": "tree", "heads": 40, "kv_heads": 8, "dim": 128, "dtype": "bf16", "sequences": 24,
         "longest": 8191, "rows": 26, "page": 64, "tree": True, "mix": 5},
        # wide trees in fp16, one KV head for each query head, heads of 64
        {"name": "tree_wide_fp16", "kind": "tree", "heads": 16, "kv_heads": 16, "dim": 64, "dtype": "fp16", "sequences": 48,
         "longest": 2500, "rows": 64, "page": 32, "tree": True, "mix": 6},
        # a chain of drafts behind one very long context: 27B class
        {"name": "chain_long_27b", "kind": "tree", "heads": 40, "kv_heads": 8, "dim": 128, "dtype": "bf16", "sequences": 1,
         "longest": 262144, "rows": 16, "page": 128, "tree": False, "mix": 7},
        # one conversation's tree, sampled: the vocabulary of both decoders
        {"name": "verify_one", "kind": "verify", "vocab": 151936, "dtype": "bf16", "sequences": 1, "rows": 6, "drafted": "tree",
         "greedy": 0.0, "mix": 8},
        # a batch of chains sampled from a draft model's own probabilities
        {"name": "verify_chains", "kind": "verify", "vocab": 151936, "dtype": "bf16", "sequences": 16, "rows": 8,
         "drafted": "sampled", "greedy": 0.0, "mix": 9},
        # wide trees over an odd vocabulary in fp32, every third conversation greedy
        {"name": "verify_trees_fp32", "kind": "verify", "vocab": 32003, "dtype": "fp32", "sequences": 24, "rows": 64,
         "drafted": "tree", "greedy": 0.33, "mix": 10},
        # the accepted rows of a few small trees: 3B class
        {"name": "keep_3b", "kind": "keep", "layers": 36, "kv_heads": 2, "dim": 128, "sequences": 4, "rows": 8, "longest": 700,
         "page": 16, "mix": 11},
        # a batch of trees: 27B class
        {"name": "keep_27b", "kind": "keep", "layers": 64, "kv_heads": 8, "dim": 128, "sequences": 32, "rows": 26, "longest": 600,
         "page": 64, "mix": 12},
    ]


def _spread(rng, low: float, high: float) -> int:
    """An integer spread evenly over the logarithm of [low, high]."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(max(low, high))))))


def draw(rng) -> dict:
    kind = rng.choices(["rotate", "tree", "verify", "keep"], [2, 4, 3, 1])[0]
    mix = rng.randrange(1 << 20)
    if kind == "verify":
        vocab = _spread(rng, 500, 152000)
        sequences = _spread(rng, 1, 48)
        return {"kind": kind, "vocab": vocab, "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "sequences": sequences,
                "rows": _spread(rng, 1, min(MOST_ROWS, MOST_LOGITS / 2 / vocab / sequences)),
                "drafted": rng.choice(["tree", "tree", "chain", "sampled"]), "greedy": rng.choice([0.0, 0.0, 0.5, 1.0]), "mix": mix}
    dim, page = rng.choice([128, 128, 64]), rng.choice([16, 32, 64, 128, 256])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    heads, kv_heads = rng.choice([(40, 8), (16, 2), (32, 8), (28, 4), (8, 8), (16, 16), (12, 1)])
    if kind == "rotate":
        sequences = _spread(rng, 1, 64)
        tree = rng.random() < 0.5
        most = MOST_ROWS if tree else MOST_TURNED / kv_heads / sequences / (heads // kv_heads)
        return {"kind": kind, "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "sequences": sequences,
                "longest": _spread(rng, 1, most), "prefix": _spread(rng, 1, 2500), "page": page,
                "rotary": rng.choice([dim, dim, dim // 2, dim // 4, 48]), "interleaved": rng.random() < 0.4, "tree": tree,
                "ahead": rng.choice([0, 0, _spread(rng, 1000, 200000)]), "mix": mix}
    if kind == "keep":
        layers = rng.randint(1, 64)
        row_bytes = layers * kv_heads * 2 * dim * 17 // 32
        sequences = _spread(rng, 1, min(64, MOST_POOL / row_bytes / 600))
        return {"kind": kind, "layers": layers, "kv_heads": kv_heads, "dim": dim, "sequences": sequences,
                "rows": _spread(rng, 1, MOST_ROWS), "longest": rng.randint(1, 500), "page": page, "mix": mix}
    sequences = _spread(rng, 1, 64)
    rows = _spread(rng, 1, MOST_ROWS)
    longest = _spread(rng, 1, min(MOST_KEYS / kv_heads / sequences, MOST_PAIRS / heads / sequences / rows))
    return {"kind": kind, "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "sequences": sequences,
            "longest": longest, "rows": rows, "page": page, "tree": rng.random() < 0.7, "mix": mix}


# ---------------------------------------------------------------------------------------------
# Sizes of a case: from the case alone


def _rows(case: dict) -> list[int]:
    """Rows of each sequence: ragged, the most of them occurs; prompts are spread over the logarithm."""
    rng = random.Random(case["mix"])
    most = case["longest"] if case["kind"] == "rotate" else case["rows"]
    low = 1 if case["kind"] == "rotate" and not case["tree"] else max(1, most // 2)
    rows = [most] + [_spread(rng, low, most) for _ in range(case["sequences"] - 1)]
    rng.shuffle(rows)
    return rows


def _contexts(case: dict) -> list[int]:
    """Positions of each sequence before its rows, ragged; rows and context together stay within ``longest`` for the
    attention, whose longest occurs."""
    rng = random.Random(case["mix"] + 1)
    if case["kind"] == "rotate":
        return [rng.randint(0, case["prefix"]) for _ in range(case["sequences"])]
    lengths = [case["longest"]] + [_spread(rng, 1, case["longest"]) for _ in range(case["sequences"] - 1)]
    return [max(0, n - r) for n, r in zip(lengths, _rows(case))]


def _parents(case: dict, rows: list[int]) -> list[list[int]]:
    """Every sequence's tree: a row follows one of the rows shortly before it, so that trees are a few rows wide."""
    rng = random.Random(case["mix"] + 2)
    return [[-1] + [rng.randint(max(0, i - 1 - i // 2), i - 1) for i in range(1, n)] for n in rows]


def _chains(rows: list[int]) -> list[list[int]]:
    return [list(range(-1, n - 1)) for n in rows]


def _depths(parents: list[list[int]]) -> list[list[int]]:
    depths = []
    for tree in parents:
        depth = []
        for parent in tree:
            depth.append(0 if parent < 0 else depth[parent] + 1)
        depths.append(depth)
    return depths


def _row_bytes(case: dict) -> int:
    """Bytes of one cached key or value of one head."""
    return case["dim"] * 17 // 32


def _inner(parents: list[list[int]]) -> int:
    """Rows that some row follows."""
    return sum(len({p for p in tree if p >= 0}) for tree in parents)


def work(case: dict) -> dict:
    rows = _rows(case)
    if case["kind"] == "verify":
        size = torch.finfo(DTYPES[case["dtype"]]).bits // 8
        logits = sum(rows) * case["vocab"]
        if case["drafted"] == "sampled":
            logits += _inner(_chains(rows)) * case["vocab"]
        return {"bytes": logits * size, "flops": 3 * logits}  # a difference, an exponential, a sum
    if case["kind"] == "keep":
        moved = sum(len(path) - 1 for path in _paths(case, rows, random.Random(case["mix"] + 3)))
        return {"bytes": 2 * moved * case["layers"] * case["kv_heads"] * 2 * _row_bytes(case) + 4 * sum(rows), "flops": 0}
    dim, heads, kv_heads = case["dim"], case["heads"], case["kv_heads"]
    if case["kind"] == "rotate":
        tokens = sum(rows)
        values = tokens * dim * 2 * (2 * heads + 2 * kv_heads + 2 * kv_heads)  # q in and out, k and v in, read back
        cache = 2 * tokens * kv_heads * 2 * _row_bytes(case)
        return {"bytes": values + cache + tokens * case["rotary"] * 4, "flops": 3 * tokens * (heads + kv_heads) * case["rotary"]}
    contexts = _contexts(case)
    depths = _depths(_parents(case, rows) if case["tree"] else _chains(rows))
    pairs = sum(n * c + sum(depth) + n for n, c, depth in zip(rows, contexts, depths))
    cache = sum(n + c for n, c in zip(rows, contexts)) * kv_heads * 2 * _row_bytes(case)
    return {"bytes": cache + 2 * sum(rows) * heads * dim * 2, "flops": 4 * dim * heads * pairs}


# ---------------------------------------------------------------------------------------------
# Inputs (from the seed alone)


def _normal(g: torch.Generator, *shape: int) -> torch.Tensor:
    return torch.randn(shape, device="cuda", generator=g)


def _i32(values) -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _flat(lists: list[list[int]]) -> list[int]:
    return [x for part in lists for x in part]


def _cumulative(lengths: list[int]) -> torch.Tensor:
    return _i32([sum(lengths[:i]) for i in range(len(lengths) + 1)])


def _block_table(lengths: list[int], page: int, g: torch.Generator) -> tuple[torch.Tensor, int]:
    """Pages of every sequence, scattered over the pool as an allocator leaves them; -1 past a sequence's last page."""
    counts = [-(-n // page) for n in lengths]
    pool = max(1, sum(counts))
    order = torch.randperm(pool, device="cuda", generator=g).to(torch.int32)
    table = torch.full((len(lengths), max(1, max(counts))), -1, dtype=torch.int32, device="cuda")
    at = 0
    for s, n in enumerate(counts):
        table[s, :n] = order[at:at + n]
        at += n
    return table, pool


def _rope_tables(rows: int, rotary: int, stretch: float) -> tuple[torch.Tensor, torch.Tensor]:
    """cos and sin float32 [rows, rotary / 2] of theta 1e6; with ``stretch``, frequencies whose wave is longer than 4096
    positions are slowed down by it, as for contexts longer than the model was trained on."""
    frequency = 1e6 ** (-torch.arange(0, rotary, 2, device="cuda", dtype=torch.float64) / rotary)
    frequency = torch.where(2 * math.pi / frequency > 4096, frequency / stretch, frequency)
    angles = torch.arange(rows, device="cuda", dtype=torch.float64)[:, None] * frequency
    return angles.cos().float(), angles.sin().float()


def _paths(case: dict, rows: list[int], rng) -> list[list[int]]:
    """An accepted path from row 0 on in every sequence's tree: it goes on with probability 0.8, to a child by chance."""
    paths = []
    for tree in _parents(case, rows):
        path = [0]
        while rng.random() < 0.8:
            children = [i for i, p in enumerate(tree) if p == path[-1]]
            if not children:
                break
            path.append(rng.choice(children))
        paths.append(path)
    return paths


def _stored_cache(case: dict, pool: int, seed: int, g: torch.Generator) -> torch.Tensor:
    """A pool of pages that hold normal keys and values under a gain for each channel, as projections give them."""
    dim, kv_heads = case["dim"], case["kv_heads"]
    pages = torch.empty((pool, kv_heads, 2, case["page"] * _row_bytes(case)), dtype=torch.uint8, device="cuda")
    gain = torch.exp(0.5 * _normal(g, 2, kv_heads, dim))
    step = max(1, (1 << 26) // (case["page"] * kv_heads * 2 * dim))
    for first in range(0, pool, step):
        count = min(step, pool - first)
        kv = (_normal(g, count, case["page"], 2, kv_heads, dim) * gain).to(DTYPES[case["dtype"]]).float()
        codes, scales = _quantise(kv.permute(0, 3, 2, 1, 4))  # [count, kv_heads, 2, page, dim]
        pages[first:first + count] = torch.cat([codes.flatten(3), scales.flatten(3)], dim=3)
    return pages


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    rows = _rows(case)
    state = {"case": case, "most": max(rows), "cu": _cumulative(rows), "tokens": sum(rows)}
    if case["kind"] == "verify":
        return _prepare_verify(state, rows, g)
    contexts = _contexts(case)
    lengths = [n + c for n, c in zip(rows, contexts)]
    state["table"], pool = _block_table(lengths, case["page"], g)
    state["lengths"], state["longest"] = _i32(lengths), max(lengths)
    if case["kind"] == "keep":
        shape = (case["layers"], pool, case["kv_heads"], 2, case["page"] * _row_bytes(case))
        state["pages"] = torch.randint(0, 256, shape, dtype=torch.uint8, device="cuda", generator=g)
        paths = _paths(case, rows, random.Random(case["mix"] * 1009 + int(seed)))
        state["path"] = _i32(_flat([path + [-1] * (n - len(path)) for path, n in zip(paths, rows)]))
        state["accepted"] = _i32([len(path) - 1 for path in paths])
        return state
    dim, heads, kv_heads, dtype = case["dim"], case["heads"], case["kv_heads"], DTYPES[case["dtype"]]
    state["parents"] = _i32(_flat(_parents(case, rows))) if case["tree"] else None
    if case["kind"] == "tree":
        state["pages"] = _stored_cache(case, pool, seed, g)
        state["q"] = _normal(g, sum(rows), heads, dim).to(dtype)
        return state
    gain = torch.exp(0.5 * _normal(g, heads + 2 * kv_heads, dim))
    qkv = (_normal(g, sum(rows), heads + 2 * kv_heads, dim) * gain).to(dtype)  # rows of one [q | k | v] projection
    state["q"], state["k"], state["v"] = qkv.split([heads, kv_heads, kv_heads], dim=1)
    shape = (pool, kv_heads, 2, case["page"] * _row_bytes(case))
    state["pages"] = torch.randint(0, 250, shape, dtype=torch.uint8, device="cuda", generator=g)
    depths = _depths(_parents(case, rows)) if case["tree"] else [list(range(n)) for n in rows]
    positions = [c + case["ahead"] + d for c, depth in zip(contexts, depths) for d in depth]
    plain = not case["tree"] and case["ahead"] == 0  # every token's position is its place in the cache
    state["positions"] = None if plain else _i32(positions)
    state["cos"], state["sin"] = _rope_tables(max(positions) + 1, case["rotary"], 4.0 if case["ahead"] else 1.0)
    return state


def _prepare_verify(state: dict, rows: list[int], g: torch.Generator) -> dict:
    """Target logits with a few likely tokens a row, as models give them; drafts from a model that mostly agrees."""
    case, total = state["case"], sum(rows)
    vocab, dtype = case["vocab"], DTYPES[case["dtype"]]
    parents = _parents(case, rows) if case["drafted"] == "tree" else _chains(rows)
    state["parents"] = _i32(_flat(parents)) if case["drafted"] == "tree" else None
    target = 2.5 * _normal(g, total, vocab)
    likely = torch.randint(0, vocab, (total, 8), device="cuda", generator=g)
    target.scatter_add_(1, likely, 9.0 + 2.0 * _normal(g, total, 8))
    draft = target + 0.5 * _normal(g, total, vocab)
    state["logits"] = target.to(dtype)
    rng = random.Random(case["mix"] + 4)
    temperature = [0.0 if rng.random() < case["greedy"] else rng.choice([0.6, 0.8, 1.0, 1.3]) for _ in rows]
    state["temperature"] = torch.tensor(temperature, dtype=torch.float32, device="cuda")
    state["uniforms"] = torch.rand(total, device="cuda", generator=g)
    # where each draft comes from, and as which of its row's drafts
    source, rank, at = [0] * total, [0] * total, 0
    for tree in parents:
        seen = {}
        for i, parent in enumerate(tree):
            source[at + i] = at + max(parent, 0)
            rank[at + i] = seen.get(parent, 0)
            seen[parent] = rank[at + i] + 1
        at += len(tree)
    source, rank = torch.tensor(source, device="cuda"), torch.tensor(rank, device="cuda")
    if case["drafted"] == "sampled":
        draft = draft.to(dtype)
        state["draft_logits"] = draft
        warm = state["temperature"].repeat_interleave(_i32(rows).long(), output_size=total).clamp(min=1e-3)[:, None]
        weights = torch.exp((draft.float() - draft.float().amax(1, keepdim=True)) / warm)
        state["ids"] = torch.multinomial(weights, 1, generator=g)[source, 0]
    else:
        state["draft_logits"] = None
        most = int(rank.max()) + 1
        state["ids"] = draft.topk(min(most, vocab), dim=1).indices[source, rank]
    return state


# ---------------------------------------------------------------------------------------------
# The plain forms: all sequences at once, padded to the longest


_MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _quantise(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """[..., dim] to packed E2M1 codes uint8 [..., dim / 2] and E8M0 scales uint8 [..., dim / 32]."""
    groups = x.unflatten(-1, (-1, 32))
    amax = groups.abs().amax(-1, keepdim=True)
    _, exponent = torch.frexp(amax)  # amax = m * 2^exponent, m in [0.5, 1)
    scale = torch.where(amax > 0, exponent - 3 + 127, torch.zeros_like(exponent)).clamp(0, 254)
    y = torch.ldexp(groups, 127 - scale)
    magnitude = y.abs()
    step = torch.where(magnitude < 2, 0.5, torch.where(magnitude < 4, 1.0, 2.0))
    doubled = (torch.round(magnitude / step) * step).clamp(max=6.0) * 2  # 0 1 2 3 4 6 8 12
    code = torch.where(doubled <= 4, doubled, torch.where(doubled == 6, 5.0, torch.where(doubled == 8, 6.0, 7.0)))
    code = (code.to(torch.uint8) | (torch.signbit(y).to(torch.uint8) << 3)).flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), scale.squeeze(-1).to(torch.uint8)


def _dequantise(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    table = torch.tensor(_MAGNITUDES + tuple(-m for m in _MAGNITUDES), device=codes.device)
    nibbles = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2)
    values = table[nibbles.int()].unflatten(-1, (-1, 32))
    return torch.ldexp(values, scales.int().unsqueeze(-1) - 127).flatten(-2)


def _split_pages(state: dict) -> tuple[torch.Tensor, torch.Tensor]:
    """Views of a pool: codes [..., page, dim / 2] and scales [..., page, dim / 32]."""
    page, dim = state["case"]["page"], state["case"]["dim"]
    return (state["pages"][..., :page * dim // 2].unflatten(-1, (page, dim // 2)),
            state["pages"][..., page * dim // 2:].unflatten(-1, (page, dim // 32)))


def _counts(state: dict) -> torch.Tensor:
    return (state["cu"][1:] - state["cu"][:-1]).long()


def _tokens(state: dict) -> tuple[torch.Tensor, torch.Tensor]:
    """The sequence of every row, and its number in it."""
    counts = _counts(state)
    sequence = torch.repeat_interleave(torch.arange(len(counts), device="cuda"), counts, output_size=state["tokens"])
    return sequence, torch.arange(state["tokens"], device="cuda") - state["cu"].long()[sequence]


def _ancestors(state: dict) -> tuple[torch.Tensor, torch.Tensor]:
    """Padded to the most rows n: each row's parent [sequences, n] (-1 where there is none), and in float64
    [sequences, n, n] a value above zero where row j leads to row i, itself included."""
    n = state["most"]
    sequence, local = _tokens(state)
    parent = torch.full((len(state["cu"]) - 1, n), -1, dtype=torch.int64, device="cuda")
    parent[sequence, local] = local - 1 if state["parents"] is None else state["parents"].long()
    above = torch.eye(n, dtype=torch.float64, device="cuda") + (parent[:, :, None] == torch.arange(n, device="cuda"))
    return parent, torch.linalg.matrix_power(above, 64)


def _turn(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, interleaved: bool) -> torch.Tensor:
    """float64 [tokens, heads, dim] with the first 2 * cos.shape[1] dimensions of every head turned: slowly turning pairs
    of 16-bit values stay next to where they were, which is often midway between two codes."""
    rotary = 2 * cos.shape[1]
    x = x.double()
    a, b = (x[..., 0:rotary:2], x[..., 1:rotary:2]) if interleaved else (x[..., :rotary // 2], x[..., rotary // 2:rotary])
    cos, sin = cos.double()[:, None], sin.double()[:, None]
    turned = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack(turned, dim=-1).flatten(-2) if interleaved else torch.cat(turned, dim=-1)
    return torch.cat([turned, x[..., rotary:]], dim=-1)


def _rotate(state: dict):
    case = state["case"]
    dtype = DTYPES[case["dtype"]]
    codes, scales = _split_pages(state)
    sequence, local = _tokens(state)
    place = state["lengths"].long()[sequence] - _counts(state)[sequence] + local
    page, offset = state["table"].long()[sequence, place // case["page"]], place % case["page"]
    at = place if state["positions"] is None else state["positions"].long()
    cos, sin = state["cos"][at], state["sin"][at]
    q = _turn(state["q"], cos, sin, case["interleaved"]).to(dtype)
    k = _turn(state["k"], cos, sin, case["interleaved"])
    new_codes, new_scales = _quantise(torch.stack([k, state["v"].double()], dim=2))
    codes[page, :, :, offset] = new_codes
    scales[page, :, :, offset] = new_scales
    kept = _dequantise(codes[page, :, :, offset], scales[page, :, :, offset]).to(dtype)
    return q, kept[:, :, 0], kept[:, :, 1]


def _tree(state: dict) -> torch.Tensor:
    case, n = state["case"], state["most"]
    dim, kv_heads = case["dim"], case["kv_heads"]
    group = case["heads"] // kv_heads
    codes, scales = _split_pages(state)
    sequence, local = _tokens(state)
    counts = _counts(state)
    _, above = _ancestors(state)
    columns = -(-state["longest"] // case["page"])
    ids = state["table"][:, :columns].long().clamp(min=0)
    # [sequences, kv_heads, 2, positions, dim]
    kv = _dequantise(codes[ids], scales[ids]).permute(0, 2, 3, 1, 4, 5).flatten(3, 4)
    position = torch.arange(kv.shape[3], device="cuda")
    draft = position - (state["lengths"].long() - counts)[:, None]  # a position's row, below 0 in the context
    own_rows = torch.gather(above > 0, 2, draft.clamp(0, n - 1)[:, None].expand(-1, n, -1))
    seen = ((draft < 0)[:, None] | own_rows) & (position < state["lengths"][:, None])[:, None]
    q = torch.zeros(len(counts), n, case["heads"], dim, device="cuda")
    q[sequence, local] = state["q"].float()
    # columns: row, then query head of the KV head
    q = q.unflatten(2, (kv_heads, group)).permute(0, 2, 1, 3, 4).reshape(len(counts), kv_heads, n * group, dim)
    scores = (q @ kv[:, :, 0].transpose(2, 3).contiguous()) * dim ** -0.5
    scores = scores.masked_fill(~seen.repeat_interleave(group, dim=1)[:, None], float("-inf"))
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - torch.where(top == float("-inf"), 0.0, top))
    total = weights.sum(-1, keepdim=True)
    out = (weights @ kv[:, :, 1]) / torch.where(total == 0, 1.0, total)
    out = out.view(len(counts), kv_heads, n, group, dim).permute(0, 2, 1, 3, 4).flatten(2, 3)
    return out[sequence, local].to(DTYPES[case["dtype"]])


def _verify(state: dict):
    """In 64 bits: sums over the vocabulary, and random numbers next to a border."""
    n, vocab = state["most"], state["case"]["vocab"]
    sequence, local = _tokens(state)
    counts = _counts(state)
    first = state["cu"][:-1].long()
    slots = torch.arange(n, device="cuda")
    valid = slots < counts[:, None]
    row = torch.where(valid, first[:, None] + slots, 0)  # [sequences, n] into the packed rows
    parent, above = _ancestors(state)
    leads = above > 0
    greedy = state["temperature"] <= 0
    warm = torch.where(greedy, 1.0, state["temperature"].double())
    best = state["logits"].float().argmax(1)  # of equal ones the first below
    best = torch.where(state["logits"] == state["logits"].gather(1, best[:, None]), torch.arange(vocab, device="cuda"), vocab).amin(1)

    def weights_of(logits, rows, sequences):
        x = logits[rows].double()
        return torch.exp((x - x.amax(1, keepdim=True)) / warm[sequences][:, None])

    def probability(logits):
        w = weights_of(logits, torch.arange(state["tokens"], device="cuda"), sequence)
        return w / w.sum(1, keepdim=True)

    ids, source = state["ids"][row], torch.gather(row, 1, parent.clamp(min=0))
    p_all = probability(state["logits"])
    p = torch.where(greedy[:, None], (best[source] == ids).double(), p_all[source, ids])
    child = valid & (parent >= 0)
    sibling = (parent[:, :, None] == parent[:, None, :]) & child[:, :, None] & child[:, None, :]
    earlier = sibling & (slots[None, :] < slots[:, None])  # [s, i, j]: j is tried before i
    repeated = (earlier & (ids[:, :, None] == ids[:, None, :])).any(2)
    p = torch.where(child & ~repeated, p, 0.0)
    u = state["uniforms"].double()[row]
    if state["draft_logits"] is None:
        against = u * (1.0 - (earlier * p[:, None, :]).sum(2))
    else:
        q_all = probability(state["draft_logits"])
        against = torch.where(greedy[:, None], 0.0, u * q_all[source, ids])
    accept = (p > 0) & torch.where(greedy[:, None], p > 0, against < p)
    taken = accept & ~(earlier & accept[:, None, :]).any(2)
    fine = taken | (slots == 0)
    visited = valid & leads[:, :, 0] & (~leads | fine[:, None, :]).all(2)
    depth = leads.sum(2) - 1
    accepted = visited.sum(1) - 1
    last = torch.where(visited, depth, -1).argmax(1)
    # the token behind the last accepted row
    at = row.gather(1, last[:, None])[:, 0]
    every = torch.arange(len(counts), device="cuda")
    w = weights_of(state["logits"], at, every)
    follows = child & (parent == last[:, None])
    if state["draft_logits"] is None:
        rest = w.clone()
        rest.scatter_(1, torch.where(follows, ids, ids.gather(1, follows.long().argmax(1, keepdim=True))),
                      torch.where(follows.any(1, keepdim=True), 0.0, w.gather(1, ids[:, :1])).expand(-1, n).contiguous())
    else:
        v = weights_of(state["draft_logits"], at, every)
        residual = (w / w.sum(1, keepdim=True) - v / v.sum(1, keepdim=True)).clamp(min=0)
        rest = torch.where(follows.any(1, keepdim=True), residual, w)
    rest = torch.where(rest.sum(1, keepdim=True) > 0, rest, w)
    summed = rest.cumsum(1)
    chosen = (summed <= state["uniforms"].double()[first][:, None] * summed[:, -1:]).sum(1)
    most = torch.where(rest > 0, torch.arange(vocab, device="cuda"), -1).amax(1)
    chosen = torch.where(greedy, best[at], torch.minimum(chosen, most))
    # path and tokens, packed like the rows
    path = torch.full((len(counts), n + 1), -1, dtype=torch.int64, device="cuda")
    path.scatter_(1, torch.where(visited, depth, n), slots.expand(len(counts), -1))
    path = path[:, :n]
    new = torch.full_like(path, -1)
    new[:, :-1] = torch.where(path[:, 1:] >= 0, ids.gather(1, path[:, 1:].clamp(min=0)), -1)
    new.scatter_(1, accepted[:, None], chosen[:, None])
    path = torch.where(slots <= accepted[:, None], path, -1)
    return accepted.to(torch.int32), path[sequence, local].to(torch.int32), new[sequence, local]


def _keep(state: dict):
    case = state["case"]
    sequence, local = _tokens(state)
    context = (state["lengths"].long() - _counts(state))[sequence]
    # a row behind the accepted ones moves to its own place
    source = context + torch.where(local <= state["accepted"].long()[sequence], state["path"].long(), local)
    target = context + local
    size = case["page"]
    pages = state["table"].long()
    for part in _split_pages(state):
        moved = part[:, pages[sequence, source // size], :, :, source % size]
        part[:, pages[sequence, target // size], :, :, target % size] = moved
    return state["pages"], (state["lengths"] - _counts(state) + state["accepted"] + 1).to(torch.int32)


def run(state: dict):
    if own:
        return _run_own(state)
    return {"rotate": _rotate, "tree": _tree, "verify": _verify, "keep": _keep}[state["case"]["kind"]](state)


def _run_own(state: dict):
    from texelator_amd import layers

    case = state["case"]
    if case["kind"] == "verify":
        return layers.verify_drafts(state["logits"], state["ids"], state["uniforms"], state["cu"], parents=state["parents"],
                                    draft_logits=state["draft_logits"], temperature=state["temperature"])
    if case["kind"] == "keep":
        return state["pages"], layers.kv4_keep_path(state["pages"], state["table"], state["lengths"], state["cu"], state["path"],
                                                    state["accepted"], case["dim"])
    if case["kind"] == "tree":
        return layers.kv4_tree_attention(state["q"], state["pages"], state["table"], state["lengths"], state["cu"],
                                         case["dim"] ** -0.5, parents=state["parents"])
    q = layers.kv4_append_rope(state["q"], state["k"], state["v"], state["cos"], state["sin"], state["pages"], state["table"],
                               state["lengths"], cu=state["cu"], positions=state["positions"], interleaved=case["interleaved"])
    k, v = layers.kv4_read(state["pages"], state["table"], state["lengths"], case["dim"], cu=state["cu"], tokens=state["tokens"],
                           dtype=DTYPES[case["dtype"]])
    return q, k, v


# ---------------------------------------------------------------------------------------------
# The definitions in 64 bits


def _exact_values(raw: torch.Tensor, page: int, dim: int) -> torch.Tensor:
    """float64 [..., page, dim] of pages uint8 [..., page * dim * 17 / 32]."""
    codes = raw[..., :page * dim // 2].reshape(*raw.shape[:-1], page, dim // 2).int()
    scales = raw[..., page * dim // 2:].reshape(*raw.shape[:-1], page, dim // 32).double()
    nibbles = torch.empty(*codes.shape[:-1], dim, dtype=torch.int32, device=raw.device)
    nibbles[..., 0::2], nibbles[..., 1::2] = codes % 16, codes // 16
    exponent, mantissa = (nibbles % 8) // 2, nibbles % 2
    magnitude = torch.where(exponent == 0, mantissa * 0.5, (1 + mantissa * 0.5) * torch.exp2(exponent.double() - 1))
    signed = torch.where(nibbles >= 8, -magnitude, magnitude).double()
    return signed * torch.exp2(scales - 127).repeat_interleave(32, dim=-1)


def _exact_round_trip(x: torch.Tensor) -> torch.Tensor:
    """What a value stands for once it is stored: float64 of the same shape, found by distance to every level."""
    y = x.unflatten(-1, (-1, 32))
    amax = y.abs().amax(-1, keepdim=True)
    scale = torch.exp2(torch.floor(torch.log2(amax.clamp(min=2.0 ** -125))) - 2)
    levels = torch.tensor(_MAGNITUDES, dtype=torch.float64, device=x.device)
    best = torch.zeros_like(y)
    distance = (y.abs() / scale - best).abs()
    for index in range(1, 8):
        d = (y.abs() / scale - levels[index]).abs()
        nearer = (d < distance) | ((d == distance) & (index % 2 == 0))
        best, distance = torch.where(nearer, levels[index], best), torch.where(nearer, d, distance)
    return (torch.sign(y) * best * scale).flatten(-2)


def _exact_rotate(case: dict, state: dict):
    """The rotation as a product with a complex number for each pair."""
    rows, contexts = _rows(case), _contexts(case)
    depths = _depths(_parents(case, rows)) if case["tree"] else [list(range(n)) for n in rows]
    positions = torch.tensor([c + case["ahead"] + d for c, depth in zip(contexts, depths) for d in depth], device="cuda")
    factor = torch.complex(state["cos"].double(), state["sin"].double())[positions][:, None]
    half = case["rotary"] // 2
    first = torch.arange(half, device="cuda") * (2 if case["interleaved"] else 1)
    second = first + (1 if case["interleaved"] else half)

    def turned(x):
        x = x.double().clone()
        pair = torch.complex(x[..., first], x[..., second]) * factor
        x[..., first], x[..., second] = pair.real, pair.imag
        return x

    return turned(state["q"]), _exact_round_trip(turned(state["k"])), _exact_round_trip(state["v"].double())


def _exact_tree(case: dict, state: dict) -> torch.Tensor:
    """One sequence and KV head after the other, the rows seen as a list for each row."""
    rows, contexts = _rows(case), _contexts(case)
    parents = _parents(case, rows) if case["tree"] else _chains(rows)
    group = case["heads"] // case["kv_heads"]
    out = torch.empty(state["q"].shape, dtype=torch.float64, device="cuda")
    at = 0
    for s, (n, context, tree) in enumerate(zip(rows, contexts, parents)):
        seen = torch.zeros(n, n, dtype=torch.bool)
        for i in range(n):
            j = i
            while j >= 0:
                seen[i, j] = True
                j = tree[j]
        ids = state["table"][s, :-(-(n + context) // case["page"])].long()
        hidden = torch.cat([torch.zeros(n, context, dtype=torch.bool), ~seen], dim=1).cuda()
        for head in range(case["kv_heads"]):
            k, v = _exact_values(state["pages"][ids, head], case["page"], case["dim"]).transpose(0, 1).flatten(1, 2)[:, :n + context]
            for h in range(head * group, (head + 1) * group):
                scores = (state["q"][at:at + n, h].double() @ k.t()) / math.sqrt(case["dim"])
                out[at:at + n, h] = torch.softmax(scores.masked_fill(hidden, float("-inf")), dim=-1) @ v
        at += n
    return out


def exact(case: dict, seed: int):
    if case["kind"] in ("verify", "keep"):
        return None  # whole numbers, which the plain form finds in 64 bits, and bytes moved
    state = prepare(case, seed)
    return _exact_rotate(case, state) if case["kind"] == "rotate" else _exact_tree(case, state)
