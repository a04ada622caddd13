"""Trees of drafted rows for the tests of a drafted step, with 64-bit results and error bounds."""
from __future__ import annotations

import numpy as np
import torch

from oracle import mxfp4
from tests.serving import HALF_STEP, Cache


def random_parents(rng, rows, spread=3):
    """Every row behind one of the `spread` rows before it."""
    return [int(rng.integers(max(0, i - spread), i)) if i else -1 for i in range(rows)]


def seen_rows(parents, rows):
    """bool [rows, rows]: row i sees row j; parents outside the rows end a walk, and so does a row seen already."""
    seen = np.zeros((rows, rows), dtype=bool)
    for i in range(rows):
        j = i
        while 0 <= j < rows and not seen[i, j]:
            seen[i, j] = True
            j = parents[j]
    return seen


def masked_attention64(q, k, v, scale, hidden):
    """Rows of softmax(scale q k^T) v in 64 bits over the keys that hidden [n, m] leaves (zeros where it leaves none), and the bound of a
    16-bit kernel's error, as tests.serving.attention64 derives it; hidden keys and values take no part in either."""
    u = HALF_STEP[q.dtype]
    q, k, v = q.double(), k.double(), v.double()
    (n, dim), m = q.shape, k.shape[0]
    out, bound = (torch.zeros(n, dim, dtype=torch.float64, device=q.device) for _ in range(2))
    if m == 0:
        return out, bound
    seen = ~hidden.all(dim=1)
    products = (q @ k.t()) * scale
    scores = torch.where(hidden, float("-inf"), products)
    p = torch.softmax(scores[seen], dim=1)
    used = torch.where(hidden.all(dim=0)[:, None], 0.0, v)
    out[seen] = p @ used
    spread = torch.where(hidden, 0.0, (q.abs() @ k.abs().t()) * abs(scale)).amax(dim=1, keepdim=True)[seen]
    loss = 2 * u + 2 * ((dim + 4) * 2.0 ** -24 * spread + 2.0 ** -22 + (m + 64) * 2.0 ** -24)
    bound[seen] = loss * (p @ used.abs()) + u * out[seen].abs() * (1 + loss)
    if u == HALF_STEP[torch.float16]:
        bound[seen] += 2.0 ** -25 + m * 2.0 ** -35 * used.abs().max()
    return out, bound


class Trees(Cache):
    """A cache whose sequences end in drafted rows: rows[s] of lengths[s] positions, which may be fewer than the rows."""

    def __init__(self, lengths, rows, kv_heads, dim, page_size, seed, dtype=torch.bfloat16, chain=False, **more):
        super().__init__(lengths, kv_heads, dim, page_size, seed, dtype, **more)
        rng = np.random.default_rng(seed + 1)
        self.rows = list(rows)
        self.trees = [list(range(-1, n - 1)) if chain else random_parents(rng, n) for n in rows]
        self.cu = torch.tensor([0, *np.cumsum(rows)], dtype=torch.int32, device="cuda")
        flat = [p for tree in self.trees for p in tree]
        self.parents = None if chain else torch.tensor(flat, dtype=torch.int32, device="cuda")

    def tree_attention(self, q, scale):
        """64-bit results and bounds [tokens, heads, dim]."""
        group, at = q.shape[1] // self.kv_heads, 0
        out, bound = (torch.zeros(q.shape, dtype=torch.float64, device="cuda") for _ in range(2))
        for n, rows, tree, values in zip(self.lengths_host, self.rows, self.trees, self.values):
            hidden = torch.from_numpy(~seen_rows(tree, rows))
            context = n - rows
            hidden = torch.cat([torch.zeros(rows, max(context, 0), dtype=torch.bool), hidden[:, max(-context, 0):]], dim=1).cuda()
            values = values.cuda()
            for h in range(q.shape[1]):
                k, v = values[h // group]
                out[at:at + rows, h], bound[at:at + rows, h] = masked_attention64(q[at:at + rows, h], k, v, scale, hidden)
            at += rows
        return out, bound


def turned64(x, cos, sin, interleaved):
    """float64 [tokens, heads, dim] of x with its first 2 * cos.shape[1] dimensions turned, one pair after the other; cos and sin
    [tokens, rotary / 2]."""
    x = x.double().clone()
    half = cos.shape[1]
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        c, s = cos[:, None, i].double(), sin[:, None, i].double()
        x[..., a], x[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    return x


def rounded64(x, dtype):
    """float64 x rounded once to a 16-bit type, ties to even, as float64 (torch's own cast of float64 rounds to float32 on the way)."""
    digits, least = (8, -126) if dtype == torch.bfloat16 else (11, -14)
    _, exponent = torch.frexp(x)
    step = torch.ldexp(torch.ones_like(x), (exponent - 1).clamp(min=least) - (digits - 1))
    return torch.round(x / step) * step


def quantise64(x):
    """MXFP4 codes and exponents of float64 [..., dim], without a rounding on the way."""
    groups = x.reshape(*x.shape[:-1], -1, mxfp4.GROUP)
    amax = np.abs(groups).max(axis=-1)
    _, exponent = np.frexp(amax)
    e = np.clip(np.where(amax > 0, exponent - 3 + 127, 0), 0, 254)
    return mxfp4.e2m1_codes(x * np.ldexp(1.0, 127 - np.repeat(e, mxfp4.GROUP, axis=-1))), e.astype(np.uint8)


def verify64(logits, ids, uniforms, trees, temperatures, draft_logits=None):
    """(accepted, path, next) as lists, one sequence and one draft after the other, in 64 bits."""
    accepted, path, following, at = [], [], [], 0
    vocab = logits.shape[1]
    for tree, temperature in zip(trees, temperatures):
        n = len(tree)
        token = ids[at:at + n].tolist()
        u = uniforms[at:at + n].double().tolist()

        def weights(source, row):
            x = source[at + row].double()
            if torch.isnan(x).any() or x.max() == float("-inf") or (temperature > 0 and x.max() == float("inf")):
                return None
            if temperature <= 0:
                p = torch.zeros(vocab, dtype=torch.float64)
                p[int((x == x.max()).nonzero()[0])] = 1.0
                return p
            p = torch.exp(((x - x.max()) / float(torch.tensor(temperature, dtype=torch.float32))).masked_fill(x == float("-inf"), float("-inf")))
            return p

        row, steps, closing = 0, [0], -1
        while n:
            raw = weights(logits, row)
            p = None if raw is None else raw / raw.sum()
            children = [i for i in range(1, n) if tree[i] == row]
            if p is None:
                break
            rest, taken = raw.clone(), None  # the closing token is drawn from weights as they are: their sums round least
            if draft_logits is not None and temperature > 0:
                q = weights(draft_logits, row) if children else None
                if children and q is None:
                    break
                q = q / q.sum() if children else None
                for i in children:
                    x = token[i]
                    if 0 <= x < vocab and p[x] > 0 and u[i] * q[x] < p[x]:
                        taken = i
                    else:
                        rest = (p - q).clamp(min=0)
            else:
                before, tried = 0.0, set()
                for i in children:
                    x = token[i]
                    if 0 <= x < vocab and x not in tried:
                        if p[x] > 0 and (temperature <= 0 or u[i] * (1 - before) < p[x]):
                            taken = i
                            break
                        before += float(p[x])
                        rest[x] = 0.0
                    tried.add(x)
            if taken is not None:
                row = taken
                steps.append(row)
                continue
            if temperature <= 0 or not rest.sum() > 0:
                rest = raw
            summed = rest.cumsum(0)
            closing = min(int((summed <= u[0] * summed[-1]).sum()), int(rest.nonzero().max()))
            break
        if n:
            following += [token[i] for i in steps[1:]] + [closing] + [-1] * (n - len(steps))
            path += steps + [-1] * (n - len(steps))
        accepted.append(len(steps) - 1 if n else -1)
        at += n
    return accepted, path, following
