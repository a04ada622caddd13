"""Batches for the tests of packed attention and of the paged 4-bit cache, with 64-bit results and error bounds."""
from __future__ import annotations

import numpy as np
import torch

from oracle import mxfp4

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def i32(values, device="cuda"):
    return torch.tensor(list(values), dtype=torch.int32, device=device)


def cumulative(lengths, device="cuda"):
    return i32([0, *np.cumsum(lengths)], device)


def attention64(q, k, v, scale, first):
    """Row i of q [n, dim] over the keys 0 .. first + i of k [m, dim]: softmax(scale q k^T) v in 64 bits (zeros where there is
    no key), and the bound of a 16-bit kernel's error, element by element.

    Let u be half a step of the rows' type, A = sum p |v| / sum p and S the largest sum |scale q_d k_d|. Rounding the
    probabilities changes numerator and denominator by a factor in 1 +- u each: 2 u A. The fp32 scores are off by at most (dim
    + 4) 2^-24 S (sums, the two factors), which changes a probability by that share, again in both: twice; the same for the
    exponential's own 2^-22 and for fp32 sums over m keys and a few joins, (m + 64) 2^-24. The output is rounded once: u |out|, or
    half of the smallest subnormal. In fp16 probabilities are held times 2^11 at least, and below 2^-25 (subnormals then, half
    a step being 2^-25) they are off by up to 2^-36, in numerator and denominator."""
    u = HALF_STEP[q.dtype]
    q, k, v = q.double(), k.double(), v.double()
    n, m, dim = q.shape[0], k.shape[0], q.shape[1]
    out, bound = torch.zeros(n, dim, dtype=torch.float64, device=q.device), torch.zeros(n, dim, dtype=torch.float64, device=q.device)
    if n == 0 or m == 0:
        return out, bound
    scores = (q @ k.t()) * scale
    hidden = torch.arange(m, device=q.device)[None, :] > torch.arange(n, device=q.device)[:, None] + first
    seen = ~hidden.all(dim=1)
    scores = scores.masked_fill(hidden, float("-inf"))
    p = torch.softmax(scores[seen], dim=1)
    out[seen] = p @ v
    spread = ((q.abs() @ k.abs().t()) * abs(scale)).masked_fill(hidden, 0).amax(dim=1, keepdim=True)[seen]
    loss = 2 * u + 2 * ((dim + 4) * 2.0 ** -24 * spread + 2.0 ** -22 + (m + 64) * 2.0 ** -24)
    bound[seen] = loss * (p @ v.abs()) + u * out[seen].abs() * (1 + loss)
    if u == HALF_STEP[torch.float16]:
        bound[seen] += 2.0 ** -25 + m * 2.0 ** -35 * v.abs().max()
    return out, bound


def assert_within(got, want, bound):
    got = got.double()
    assert torch.isfinite(got).all()
    over = (got - want).abs() - bound
    assert float(over.max()) <= 0, (float((got - want).abs().max()), float(bound.max()), int(over.argmax()))


def halves_from_rows(rows, page_size, dim):
    """Rows uint8/float [page_size, dim] of 32-bit values as one head's half of a page, by the oracle's quantiser."""
    codes, exponents = mxfp4.quantize(rows)
    return np.concatenate([mxfp4.pack(codes).reshape(-1), exponents.reshape(-1)])


def half_values(half, page_size, dim):
    """A half page uint8 [..., bytes] as float64 [..., page_size, dim]; scale 255 is NaN."""
    half = np.asarray(half)
    codes = mxfp4.unpack(half[..., :page_size * dim // 2].reshape(*half.shape[:-1], page_size, dim // 2))
    exponents = half[..., page_size * dim // 2:].reshape(*half.shape[:-1], page_size, dim // 32)
    values = mxfp4.dequantize(codes, exponents)
    return np.where(np.repeat(exponents == 255, 32, axis=-1), np.nan, values)


class Cache:
    """A pool whose pages are scattered over the sequences; pages of no sequence and rows past the lengths hold noise with
    NaN scales among it. values[s] float64 [kv_heads, 2, length, dim]."""

    def __init__(self, lengths, kv_heads, dim, page_size, seed, dtype=torch.bfloat16, spare=3, extra_columns=2, spread=None):
        rng = np.random.default_rng(seed)
        self.lengths_host, self.page_size, self.dim, self.kv_heads = list(lengths), page_size, dim, kv_heads
        counts = [-(-n // page_size) for n in lengths]
        total = sum(counts) + spare
        half = page_size * dim * 17 // 32
        pages = rng.integers(0, 256, size=(total, kv_heads, 2, half), dtype=np.uint8)
        pages[..., page_size * dim // 2:][rng.random((total, kv_heads, 2, page_size * dim // 32)) < 0.5] = 255
        order = rng.permutation(total)
        table = np.full((len(lengths), max(1, max(counts, default=1)) + extra_columns), -1, dtype=np.int32)
        self.values, at = [], 0
        for s, n in enumerate(lengths):
            ids = order[at:at + counts[s]]
            at += counts[s]
            table[s, :counts[s]] = ids
            rows = rng.standard_normal((kv_heads, 2, n, dim)).astype(np.float32)
            if spread is not None:
                rows[:, 0] *= spread(n)[None, :, None]
            rows = torch.from_numpy(rows).to(dtype).float().numpy()
            codes, exponents = mxfp4.quantize(rows)
            self.values.append(torch.from_numpy(mxfp4.dequantize(codes, exponents)))
            packed = mxfp4.pack(codes)
            for i, page in enumerate(ids):
                take = min(page_size, n - i * page_size)
                part = slice(i * page_size, i * page_size + take)
                pages[page, :, :, :take * dim // 2] = packed[:, :, part].reshape(kv_heads, 2, -1)
                start = page_size * dim // 2
                pages[page, :, :, start:start + take * dim // 32] = exponents[:, :, part].reshape(kv_heads, 2, -1)
        self.pages, self.table, self.lengths = torch.from_numpy(pages).cuda(), torch.from_numpy(table).cuda(), i32(lengths)

    def attention(self, q, scale):
        """64-bit results and bounds [sequences, heads, dim] of one query per sequence."""
        group = q.shape[1] // self.kv_heads
        results = [[attention64(q[s, h][None], values[h // group, 0].cuda(), values[h // group, 1].cuda(), scale, n - 1)
                    for h in range(q.shape[1])] for s, (n, values) in enumerate(zip(self.lengths_host, self.values))]
        return tuple(torch.stack([torch.stack([r[i][0] for r in row]) for row in results]) for i in (0, 1))
