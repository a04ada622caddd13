"""The operators that serve many conversations at once from a paged KV cache held in 4 bits, and what
their speed is measured on.

Five kinds of call, each through ``texelator_amd.layers``, over the head layouts of the 3B- and
27B-class decoders of ``texelator_amd.modeling`` and generic ones:

* ``packed``  ``packed_attention``: causal attention of several prompts of different lengths packed one
              behind the other, grouped heads, with or without keys of earlier turns before them.
* ``append``  ``kv4_append`` and ``kv4_read``: new keys and values into the cache (one token for each
              sequence, or whole prompts), and the same rows read back as the values they stand for.
* ``read``    ``kv4_read``: the whole cached prefix of every sequence, as a prompt's later part needs it.
* ``attend``  ``kv4_attention``: one query token for each sequence over its cached positions.
* ``copy``    ``kv4_copy_pages``: pages of every layer's cache to other pages (a fork, a compaction).

The cache: a pool of pages ``[pages, kv_heads, 2 (k, v), page_size * head_dim * 17 / 32]`` uint8. A page
holds, for each KV head, ``page_size`` keys and as many values: first the packed E2M1 codes
``[page_size][head_dim / 2]`` (even element in the low nibble), then one E8M0 scale for each 32 elements,
``[page_size][head_dim / 32]``. A group's scale is 2^(floor(log2(amax)) - 2), its codes are v / scale
rounded to the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 with ties to the even code, saturated at 6. Position
p of sequence s lies at offset p % page_size of page block_table[s][p // page_size].
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
MOST_KEYS = 262144 * 8          # cached positions times KV heads of the largest read or attend case
MOST_PAIRS = 16 * 9000 * 9000   # heads times longest length squared, of a drawn packed case
MOST_ROWS = 16384 * 8           # tokens times KV heads of the largest append case
MOST_COPY = 800 << 20           # bytes of the pool of the largest copy case


def listed() -> list[dict]:
    return [
        # a handful of short chat prompts of ragged lengths arriving together: 3B class
        {"name": "packed_short_3b", "kind": "packed", "heads": 16, "kv_heads": 2, "dim": 128, "dtype": "bf16",
         "sequences": 5, "longest": 93, "prefix": 0, "mix": 1},
        # long documents of different lengths in one prefill: 27B class
        {"name": "packed_documents_27b", "kind": "packed", "heads": 40, "kv_heads": 8, "dim": 128, "dtype": "bf16",
         "sequences": 6, "longest": 8190, "prefix": 0, "mix": 2},
        # the next turn of several fp16 conversations: new tokens behind keys of earlier turns, heads of 64
        {"name": "packed_turns_fp16", "kind": "packed", "heads": 28, "kv_heads": 4, "dim": 64, "dtype": "fp16",
         "sequences": 9, "longest": 777, "prefix": 2500, "mix": 3},
        # one decoded token for each of a few sequences into their last pages
        {"name": "append_tokens", "kind": "append", "kv_heads": 2, "dim": 128, "dtype": "bf16", "sequences": 5,
         "longest": 1, "prefix": 700, "page": 16, "mix": 4},
        # prompts of different lengths into the cache, pages entered in the middle: 27B class
        {"name": "append_prompts_27b", "kind": "append", "kv_heads": 8, "dim": 128, "dtype": "bf16", "sequences": 7,
         "longest": 8192, "prefix": 500, "page": 64, "mix": 5},
        # the prefix of one conversation in fp16, heads of 64, read back for its next prompt
        {"name": "read_prefix_fp16", "kind": "read", "kv_heads": 4, "dim": 64, "dtype": "fp16", "sequences": 3,
         "longest": 20011, "page": 32, "mix": 6},
        # one conversation of 700 tokens: the smallest decode step, 3B class
        {"name": "attend_one_3b", "kind": "attend", "heads": 16, "kv_heads": 2, "dim": 128, "dtype": "bf16",
         "sequences": 1, "longest": 700, "page": 16, "idle": False, "mix": 7},
        # a batch of ordinary conversations, some slots idle: 27B class
        {"name": "attend_batch_27b", "kind": "attend", "heads": 40, "kv_heads": 8, "dim": 128, "dtype": "bf16",
         "sequences": 32, "longest": 8191, "page": 64, "idle": True, "mix": 8},
        # many fp16 conversations of very different lengths, one KV head for each query head, heads of 64
        {"name": "attend_many_fp16", "kind": "attend", "heads": 16, "kv_heads": 16, "dim": 64, "dtype": "fp16",
         "sequences": 96, "longest": 16384, "page": 32, "idle": False, "mix": 9},
        # one very long context: 27B class
        {"name": "attend_long_27b", "kind": "attend", "heads": 40, "kv_heads": 8, "dim": 128, "dtype": "bf16",
         "sequences": 1, "longest": 262144, "page": 128, "idle": False, "mix": 10},
        # a conversation forked four ways: the last, partly filled page of every layer copied
        {"name": "copy_fork", "kind": "copy", "layers": 36, "pages": 96, "copies": 4, "kv_heads": 2, "dim": 128,
         "page": 64, "mix": 11},
        # a pool compacted after long conversations ended
        {"name": "copy_compact", "kind": "copy", "layers": 12, "pages": 900, "copies": 400, "kv_heads": 8, "dim": 128,
         "page": 64, "mix": 12},
    ]


def _spread(rng, low: float, high: float) -> int:
    """An integer spread evenly over the logarithm of [low, high]."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng) -> dict:
    kind = rng.choices(["packed", "append", "read", "attend", "copy"], [4, 2, 1, 4, 1])[0]
    mix = rng.randrange(1 << 20)
    dtype, dim = rng.choice(["bf16", "bf16", "fp16"]), rng.choice([128, 128, 64])
    if kind == "packed":
        heads, kv_heads = rng.choice([(40, 8), (16, 2), (32, 8), (28, 4), (8, 8), (12, 1)])
        return {"kind": kind, "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype,
                "sequences": _spread(rng, 1, 12), "longest": _spread(rng, 1, math.sqrt(MOST_PAIRS / heads)),
                "prefix": rng.choice([0, 0, _spread(rng, 1, 3000)]), "mix": mix}
    page = rng.choice([16, 32, 64, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8, 16])
    if kind == "append":
        sequences = _spread(rng, 1, 64)
        longest = rng.choice([1, _spread(rng, 2, max(2, MOST_ROWS / kv_heads / sequences))])
        return {"kind": kind, "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "sequences": sequences,
                "longest": longest, "prefix": _spread(rng, 1, 1000), "page": page, "mix": mix}
    if kind == "copy":
        page_bytes = kv_heads * 2 * page * dim * 17 // 32
        layers = rng.randint(1, 36)
        pages = _spread(rng, 8, max(8, min(4000, MOST_COPY / layers / page_bytes)))
        return {"kind": kind, "layers": layers, "pages": pages, "copies": rng.randint(1, pages // 2), "kv_heads": kv_heads,
                "dim": dim, "page": page, "mix": mix}
    sequences = _spread(rng, 1, 128)
    longest = _spread(rng, 1, max(1, MOST_KEYS / kv_heads / sequences / (8 if kind == "read" else 1)))
    case = {"kind": kind, "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "sequences": sequences, "longest": longest,
            "page": page, "mix": mix}
    if kind == "attend":
        case["heads"] = kv_heads * rng.choice([1, 2, 5, 7, 8, 12] if kv_heads < 8 else [1, 4, 5])
        case["idle"] = rng.random() < 0.3
    return case


# ---------------------------------------------------------------------------------------------
# Sizes of a case


def _new_lengths(case: dict) -> list[int]:
    """New tokens of each sequence (packed, append) or cached positions (read, attend): ragged, spread over
    the logarithm up to ``longest``, which occurs; of ``idle`` batches every fourth is empty."""
    rng = random.Random(case["mix"])
    lengths = [case["longest"]] + [_spread(rng, 1, case["longest"]) for _ in range(case["sequences"] - 1)]
    if case.get("idle"):
        lengths[3::4] = [0] * len(lengths[3::4])
    rng.shuffle(lengths)
    return lengths


def _prefix_lengths(case: dict) -> list[int]:
    """Positions of each sequence before its new tokens."""
    rng = random.Random(case["mix"] + 1)
    prefix = case.get("prefix", 0)
    return [rng.randint(0, prefix) if prefix else 0 for _ in range(case["sequences"])]


def _row_bytes(case: dict) -> int:
    """Bytes of one cached key or value of one head."""
    return case["dim"] * 17 // 32


def work(case: dict) -> dict:
    if case["kind"] == "copy":
        return {"bytes": 2 * case["layers"] * case["copies"] * case["kv_heads"] * 2 * case["page"] * _row_bytes(case),
                "flops": 0}
    new, old = _new_lengths(case), _prefix_lengths(case)
    tokens, dim, kv_heads = sum(new), case["dim"], case["kv_heads"]
    if case["kind"] == "packed":
        pairs = sum(n * o + n * (n + 1) // 2 for n, o in zip(new, old))
        rows = 2 * tokens * case["heads"] + 2 * (tokens + sum(old)) * kv_heads
        return {"bytes": 2 * dim * rows, "flops": 4 * dim * case["heads"] * pairs}
    cache = tokens * kv_heads * 2 * _row_bytes(case)
    values = tokens * kv_heads * 2 * dim * 2
    if case["kind"] == "append":  # written from 16 bits, read back to 16 bits
        return {"bytes": 2 * (cache + values), "flops": 0}
    if case["kind"] == "read":
        return {"bytes": cache + values, "flops": 0}
    return {"bytes": cache + 2 * case["sequences"] * case["heads"] * dim * 2,
            "flops": 4 * dim * case["heads"] * tokens}


# ---------------------------------------------------------------------------------------------
# Inputs (from the seed alone)


def _normal(g: torch.Generator, *shape: int) -> torch.Tensor:
    return torch.randn(shape, device="cuda", generator=g)


def _keys_values(g: torch.Generator, rows: int, kv_heads: int, dim: int) -> torch.Tensor:
    """float32 [rows, 2, kv_heads, dim]: normal values under a gain for each channel, as projections give
    them: a few channels of the keys are much larger than the rest."""
    gain = torch.exp(0.5 * _normal(g, 2, kv_heads, dim))
    return _normal(g, rows, 2, kv_heads, dim) * gain


def _i32(values: list[int]) -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _cumulative(lengths: list[int]) -> torch.Tensor:
    return _i32([sum(lengths[:i]) for i in range(len(lengths) + 1)])


def _block_table(lengths: list[int], page: int, g: torch.Generator) -> tuple[torch.Tensor, int]:
    """Pages of every sequence, scattered over the pool as an allocator leaves them; -1 past a sequence's
    last page."""
    counts = [-(-n // page) for n in lengths]
    pool = max(1, sum(counts))
    order = torch.randperm(pool, device="cuda", generator=g).to(torch.int32)
    table = torch.full((len(lengths), max(1, max(counts))), -1, dtype=torch.int32, device="cuda")
    at = 0
    for s, n in enumerate(counts):
        table[s, :n] = order[at:at + n]
        at += n
    return table, pool


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    state = {"case": case}
    if case["kind"] == "copy":
        shape = (case["layers"], case["pages"], case["kv_heads"], 2, case["page"] * _row_bytes(case))
        state["pages"] = torch.randint(0, 256, shape, dtype=torch.uint8, device="cuda", generator=g)
        rng = random.Random(case["mix"] * 1009 + int(seed))
        chosen = rng.sample(range(case["pages"]), 2 * case["copies"])
        state["src"], state["dst"] = chosen[:case["copies"]], chosen[case["copies"]:]
        return state
    new, old = _new_lengths(case), _prefix_lengths(case)
    dtype, dim, kv_heads = DTYPES[case["dtype"]], case["dim"], case["kv_heads"]
    state["new"], state["old"] = new, old
    if case["kind"] == "packed":
        total = sum(new) + sum(old)
        kv = _keys_values(g, total, kv_heads, dim).to(dtype)
        state["q"] = _normal(g, sum(new), case["heads"], dim).to(dtype)
        state["k"], state["v"] = kv[:, 0], kv[:, 1]  # rows of one [k | v] projection
        state["cu_q"] = _cumulative(new)
        state["cu_k"] = _cumulative([n + o for n, o in zip(new, old)])
        return state
    lengths = [n + o for n, o in zip(new, old)]
    state["table"], pool = _block_table(lengths, case["page"], g)
    state["lengths"], state["cu"] = _i32(lengths), _cumulative(new)
    if case["kind"] == "append":
        shape = (pool, kv_heads, 2, case["page"] * _row_bytes(case))
        state["pages"] = torch.randint(0, 250, shape, dtype=torch.uint8, device="cuda", generator=g)
        kv = _keys_values(g, sum(new), kv_heads, dim).to(dtype)
        state["k"], state["v"] = kv[:, 0], kv[:, 1]
        return state
    state["pages"] = torch.empty((pool, kv_heads, 2, case["page"] * _row_bytes(case)), dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 26) // (case["page"] * kv_heads * 2 * dim))
    gain_seed = int(torch.randint(0, 1 << 30, (1,), generator=torch.Generator().manual_seed(int(seed))))
    for first in range(0, pool, step):
        count = min(step, pool - first)
        gains = torch.Generator(device="cuda").manual_seed(gain_seed)  # the channels' gains are the cache's own
        gain = torch.exp(0.5 * _normal(gains, 2, kv_heads, dim))
        kv = (_normal(g, count, case["page"], 2, kv_heads, dim) * gain).to(dtype).float()
        codes, scales = _quantise(kv.permute(0, 3, 2, 1, 4))  # [count, kv_heads, 2, page, dim]
        state["pages"][first:first + count] = torch.cat([codes.flatten(3), scales.flatten(3)], dim=3)
    if case["kind"] == "attend":
        state["q"] = _normal(g, case["sequences"], case["heads"], dim).to(dtype)
    return state


# ---------------------------------------------------------------------------------------------
# The plain forms


_MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _quantise(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """float32 [..., dim] to packed E2M1 codes uint8 [..., dim / 2] and E8M0 scales uint8 [..., dim / 32]."""
    groups = x.unflatten(-1, (-1, 32))
    _, exponent = torch.frexp(groups.abs().amax(-1, keepdim=True))  # amax = m * 2^exponent, m in [0.5, 1)
    scale = torch.where(groups.abs().amax(-1, keepdim=True) > 0, exponent - 3 + 127, torch.zeros_like(exponent)).clamp(0, 254)
    y = torch.ldexp(groups, 127 - scale)
    magnitude = y.abs()
    step = torch.where(magnitude < 2, 0.5, torch.where(magnitude < 4, 1.0, 2.0))
    doubled = (torch.round(magnitude / step) * step).clamp(max=6.0) * 2  # 0 1 2 3 4 6 8 12
    code = torch.where(doubled <= 4, doubled, torch.where(doubled == 6, 5.0, torch.where(doubled == 8, 6.0, 7.0)))
    code = code.to(torch.uint8) | (torch.signbit(y).to(torch.uint8) << 3)
    code = code.flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), scale.squeeze(-1).to(torch.uint8)


def _dequantise(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    table = torch.tensor(_MAGNITUDES + tuple(-m for m in _MAGNITUDES), device=codes.device)
    nibbles = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2)
    values = table[nibbles.long()].unflatten(-1, (-1, 32))
    return torch.ldexp(values, scales.int().unsqueeze(-1) - 127).flatten(-2)


def _positions(state: dict) -> tuple[torch.Tensor, torch.Tensor]:
    """Page and offset of every row that ``cu`` names: the last new[s] positions before lengths[s]."""
    page = state["case"]["page"]
    tokens = sum(state["new"])
    new, cu = _i32(state["new"]).long(), state["cu"].long()
    sequence = torch.repeat_interleave(torch.arange(len(new), device="cuda"), new, output_size=tokens)
    position = torch.arange(tokens, device="cuda") - cu[sequence] + state["lengths"].long()[sequence] - new[sequence]
    return state["table"].long()[sequence, position // page], position % page


def _split_pages(state: dict) -> tuple[torch.Tensor, torch.Tensor]:
    """Views of the pool: codes [pages, kv_heads, 2, page, dim / 2] and scales [pages, kv_heads, 2, page, dim / 32]."""
    page, dim = state["case"]["page"], state["case"]["dim"]
    codes = state["pages"][..., :page * dim // 2].unflatten(-1, (page, dim // 2))
    return codes, state["pages"][..., page * dim // 2:].unflatten(-1, (page, dim // 32))


def _read(state: dict) -> tuple[torch.Tensor, torch.Tensor]:
    codes, scales = _split_pages(state)
    page, offset = _positions(state)
    rows = _dequantise(codes[page, :, :, offset], scales[page, :, :, offset]).to(DTYPES[state["case"]["dtype"]])
    return rows[:, :, 0], rows[:, :, 1]


def _append(state: dict) -> None:
    codes, scales = _split_pages(state)
    page, offset = _positions(state)
    new_codes, new_scales = _quantise(torch.stack([state["k"], state["v"]], dim=2).float())
    codes[page, :, :, offset] = new_codes
    scales[page, :, :, offset] = new_scales


def _attend(state: dict) -> torch.Tensor:
    case = state["case"]
    codes, scales = _split_pages(state)
    group = case["heads"] // case["kv_heads"]
    out = torch.zeros(state["q"].shape, dtype=torch.float32, device="cuda")
    for s, n in enumerate(state["new"]):
        if n == 0:
            continue
        pages = state["table"][s, :-(-n // case["page"])].long()
        # [kv_heads, 2, positions, dim]
        kv = _dequantise(codes[pages], scales[pages]).permute(1, 2, 0, 3, 4).flatten(2, 3)[:, :, :n]
        q = state["q"][s].float().view(case["kv_heads"], group, case["dim"])
        scores = (q @ kv[:, 0].transpose(1, 2)) * case["dim"] ** -0.5
        weights = torch.exp(scores - scores.amax(-1, keepdim=True))
        out[s] = ((weights / weights.sum(-1, keepdim=True)) @ kv[:, 1]).flatten(0, 1)
    return out.to(DTYPES[case["dtype"]])


def _packed(state: dict) -> torch.Tensor:
    case = state["case"]
    group = case["heads"] // case["kv_heads"]
    out = torch.empty(state["q"].shape, dtype=DTYPES[case["dtype"]], device="cuda")
    q0 = k0 = 0
    for n, o in zip(state["new"], state["old"]):
        hidden = torch.ones(n, n + o, dtype=torch.bool, device="cuda").triu(o + 1)
        for head in range(case["heads"]):
            q = state["q"][q0:q0 + n, head].float()
            k = state["k"][k0:k0 + n + o, head // group].float()
            scores = (q @ k.t()) * case["dim"] ** -0.5
            scores = scores.masked_fill(hidden, float("-inf"))
            weights = torch.exp(scores - scores.amax(-1, keepdim=True))
            rows = (weights / weights.sum(-1, keepdim=True)) @ state["v"][k0:k0 + n + o, head // group].float()
            out[q0:q0 + n, head] = rows.to(out.dtype)
        q0, k0 = q0 + n, k0 + n + o
    return out


def run(state: dict):
    kind = state["case"]["kind"]
    if own:
        return _run_own(state)
    if kind == "packed":
        return _packed(state)
    if kind == "append":
        _append(state)
        return _read(state)
    if kind == "read":
        return _read(state)
    if kind == "attend":
        return _attend(state)
    dst, src = (torch.tensor(state[name], device="cuda") for name in ("dst", "src"))
    state["pages"][:, dst] = state["pages"][:, src]
    return state["pages"]


def _run_own(state: dict):
    from texelator_amd import layers

    case = state["case"]
    if case["kind"] == "packed":
        return layers.packed_attention(state["q"], state["k"], state["v"], state["cu_q"], case["dim"] ** -0.5,
                                       cu_k=state["cu_k"])
    if case["kind"] == "copy":
        layers.kv4_copy_pages(state["pages"], state["src"], state["dst"])
        return state["pages"]
    if case["kind"] == "attend":
        return layers.kv4_attention(state["q"], state["pages"], state["table"], state["lengths"], case["dim"] ** -0.5)
    if case["kind"] == "append":
        layers.kv4_append(state["k"], state["v"], state["pages"], state["table"], state["lengths"], cu=state["cu"])
    return layers.kv4_read(state["pages"], state["table"], state["lengths"], case["dim"], cu=state["cu"],
                           tokens=sum(state["new"]), dtype=DTYPES[case["dtype"]])


# ---------------------------------------------------------------------------------------------
# The definition in 64 bits


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
    y = x.double().unflatten(-1, (-1, 32))
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


def _exact_softmax_rows(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, first: int) -> torch.Tensor:
    """Rows of softmax(q k^T / sqrt(dim)) v in float64, row i over keys 0 .. first + i."""
    scores = (q.double() @ k.double().t()) / math.sqrt(q.shape[-1])
    rows = torch.arange(q.shape[0], device=q.device)[:, None]
    scores[torch.arange(k.shape[0], device=q.device)[None, :] > rows + first] = float("-inf")
    return torch.softmax(scores, dim=-1) @ v.double()


def exact(case: dict, seed: int):
    if case["kind"] == "copy":
        return None  # bytes moved, nothing computed
    state = prepare(case, seed)
    new, old = state["new"], state["old"]
    if case["kind"] == "append":
        return _exact_round_trip(state["k"]), _exact_round_trip(state["v"])
    if case["kind"] == "packed":
        group = case["heads"] // case["kv_heads"]
        out = torch.empty(state["q"].shape, dtype=torch.float64, device="cuda")
        q0 = k0 = 0
        for n, o in zip(new, old):
            for head in range(case["heads"]):
                k, v = (state[name][k0:k0 + n + o, head // group] for name in ("k", "v"))
                for i in range(0, n, 2048):
                    j = min(n, i + 2048)
                    out[q0 + i:q0 + j, head] = _exact_softmax_rows(state["q"][q0 + i:q0 + j, head], k, v, o + i)
            q0, k0 = q0 + n, k0 + n + o
        return out
    values = []  # per sequence [kv_heads, 2, length, dim]
    for s, n in enumerate(new):
        ids = state["table"][s, :-(-n // case["page"])].long()
        rows = _exact_values(state["pages"][ids], case["page"], case["dim"])
        values.append(rows.permute(1, 2, 0, 3, 4).reshape(case["kv_heads"], 2, -1, case["dim"])[:, :, :n])
    if case["kind"] == "read":
        return tuple(torch.cat([x[:, i].transpose(0, 1) for x in values]) for i in (0, 1))
    out = torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda")
    group = case["heads"] // case["kv_heads"]
    for s, n in enumerate(new):
        for head in range(case["heads"] if n else 0):
            k, v = values[s][head // group]
            out[s, head] = _exact_softmax_rows(state["q"][s, head][None], k, v, n - 1)[0]
    return out
