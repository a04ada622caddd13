"""The operators for several sequences as a program uses them together: prompts in, tokens out, turns, forks and a
compaction, over one pool of pages for two layers, against the same computed in 64 bits from the cached values."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import mxfp4
from tests.serving import assert_within, attention64, cumulative, i32
from texelator_amd import layers

pytestmark = pytest.mark.gpu
LAYERS, HEADS, KV_HEADS, PAGE = 2, 10, 2, 16


class Conversations:
    """What a serving program keeps: pools, page lists on the host, block table and lengths on the device; and, for the
    check, every sequence's cached values in 64 bits."""

    def __init__(self, slots, dim, dtype, num_pages=120, columns=20):
        self.dim, self.dtype, self.scale = dim, dtype, dim ** -0.5
        self.pools = layers.kv4_pages(num_pages, KV_HEADS, dim, PAGE, layers=LAYERS)
        self.free = list(np.random.default_rng(3).permutation(num_pages))
        self.held = [[] for _ in range(slots)]
        self.table = torch.full((slots, columns), -1, dtype=torch.int32, device="cuda")
        self.count = [0] * slots
        self.lengths = torch.zeros(slots, dtype=torch.int32, device="cuda")
        self.cached = [[torch.zeros(2, 0, KV_HEADS, dim, dtype=torch.float64) for _ in range(slots)] for _ in range(LAYERS)]
        self.g = torch.Generator().manual_seed(5)

    def rows(self, tokens, heads):
        return torch.randn(tokens, heads, self.dim, generator=self.g).to(self.dtype).cuda()

    def grow(self, new):
        """Room for new[s] more tokens, and lengths that count them: once for all layers."""
        for s, n in enumerate(new):
            self.count[s] += n
            while len(self.held[s]) * PAGE < self.count[s]:
                self.held[s].append(int(self.free.pop()))
            self.table[s, :len(self.held[s])] = i32(self.held[s])
        self.lengths += i32(new)

    def store(self, layer, k, v, new, cu=None):
        layers.kv4_append(k, v, self.pools[layer], self.table, self.lengths, cu=cu)
        at = 0
        for s, n in enumerate(new):
            rows = torch.stack([k[at:at + n], v[at:at + n]]).float().cpu().numpy()
            values = torch.from_numpy(mxfp4.dequantize(*mxfp4.quantize(rows)))
            self.cached[layer][s] = torch.cat([self.cached[layer][s], values], dim=1)
            at += n

    def prompt(self, new):
        """Prompts of new[s] tokens: their attention sees earlier turns as the cache holds them and their own keys unrounded."""
        before = list(self.count)
        cu_q, cu_old = cumulative(new), cumulative(before)
        old_lengths = self.lengths.clone()
        old_table = self.table.clone()
        self.grow(new)
        for layer in range(LAYERS):
            q, k, v = self.rows(sum(new), HEADS), self.rows(sum(new), KV_HEADS), self.rows(sum(new), KV_HEADS)
            old_k, old_v = layers.kv4_read(self.pools[layer], old_table, old_lengths, self.dim, cu=cu_old, tokens=sum(before),
                                           dtype=self.dtype)
            for s, n in enumerate(before):
                at = sum(before[:s])
                for rows, values in zip((old_k, old_v), self.cached[layer][s]):
                    assert torch.equal(rows[at:at + n].cpu(), values.to(self.dtype))
            keys, values = (torch.cat([part for s in range(len(new)) for part in
                                       (o[sum(before[:s]):sum(before[:s + 1])], x[sum(new[:s]):sum(new[:s + 1])])])
                            for o, x in ((old_k, k), (old_v, v)))
            both = [n + o for n, o in zip(new, before)]
            out = layers.packed_attention(q, keys, values, cu_q, self.scale, cu_k=cumulative(both))
            for s, n in enumerate(new):
                rows = slice(sum(new[:s]), sum(new[:s + 1]))
                seen = slice(sum(both[:s]), sum(both[:s + 1]))
                for h in range(HEADS):
                    kv = h // (HEADS // KV_HEADS)
                    want, bound = attention64(q[rows, h], keys[seen, kv], values[seen, kv], self.scale, before[s])
                    assert_within(out[rows, h], want, bound) if n else None
            self.store(layer, k, v, new, cu=cu_q)

    def check_token(self, layer, q, out):
        for s, n in enumerate(self.count):
            for h in range(HEADS):
                k, v = (x[:, h // (HEADS // KV_HEADS)].cuda() for x in self.cached[layer][s])
                want, bound = attention64(q[s, h][None], k, v, self.scale, n - 1)
                assert_within(out[s, h][None], want, bound)

    def token(self):
        """One decoded token of every sequence."""
        new = [1] * len(self.count)
        self.grow(new)
        for layer in range(LAYERS):
            q, k, v = self.rows(len(new), HEADS), self.rows(len(new), KV_HEADS), self.rows(len(new), KV_HEADS)
            self.store(layer, k, v, new)
            self.check_token(layer, q, layers.kv4_attention(q, self.pools[layer], self.table, self.lengths, self.scale))

    def fork(self, source, target):
        """Slot `target` continues as a copy of `source`: full pages shared, the last, partly filled one copied."""
        self.free += self.held[target]
        self.held[target] = list(self.held[source])
        if self.count[source] % PAGE:
            last = int(self.free.pop())
            layers.kv4_copy_pages(self.pools, [self.held[source][-1]], [last])
            self.held[target][-1] = last
        self.count[target] = self.count[source]
        self.lengths[target] = self.lengths[source]
        self.table[target].fill_(-1)
        self.table[target, :len(self.held[target])] = i32(self.held[target])
        for layer in self.cached:
            layer[target] = layer[source]

    def compact(self):
        """The pages in use move to the front of the pool."""
        used = sorted({p for pages in self.held for p in pages})
        holes = [p for p in range(len(used)) if p not in used]
        src = [p for p in used if p >= len(used)]
        layers.kv4_copy_pages(self.pools, src, holes)
        moved = dict(zip(src, holes))
        self.held = [[moved.get(p, p) for p in pages] for pages in self.held]
        self.free = list(range(len(used), self.pools.shape[1]))
        for s, pages in enumerate(self.held):
            self.table[s, :len(pages)] = i32(pages)
        self.pools[:, len(used):] = 255  # what was left behind


@pytest.mark.parametrize("dim,dtype", [(128, torch.bfloat16), (64, torch.float16)])
def test_conversations(ext, dim, dtype):
    c = Conversations(4, dim, dtype)
    c.prompt([37, 0, 5, 64])
    for _ in range(3):
        c.token()
    c.prompt([10, 33, 0, 1])  # the next turn of some
    c.token()
    c.fork(0, 2)
    for _ in range(2):
        c.token()             # the fork's pages are its own from here on
    c.compact()
    c.token()
    c.prompt([1, 2, 3, 4])


def test_decode_step_in_a_graph(ext):
    """Both layers' append and attention of one token captured once, replayed while lengths and pages grow."""
    c = Conversations(3, 128, torch.bfloat16)
    c.prompt([20, 3, 50])
    static = [tuple(torch.zeros(3, h, 128, dtype=torch.bfloat16, device="cuda") for h in (HEADS, KV_HEADS, KV_HEADS)) for _ in range(LAYERS)]
    outs = [torch.zeros(3, HEADS, 128, dtype=torch.bfloat16, device="cuda") for _ in range(LAYERS)]

    def step():
        for layer, (q, k, v) in enumerate(static):
            layers.kv4_append(k, v, c.pools[layer], c.table, c.lengths)
            layers.kv4_attention(q, c.pools[layer], c.table, c.lengths, c.scale, out=outs[layer])

    c.grow([1] * 3)  # so that the rows the capture's warm-up writes are the first token's
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step()
        for turn in range(18):
            if turn:
                c.grow([1] * 3)
            for layer, (q, k, v) in enumerate(static):
                for t in (q, k, v):
                    t.copy_(torch.randn(t.shape, generator=c.g))
            graph.replay()
            stream.synchronize()
            for layer, (q, k, v) in enumerate(static):
                rows = torch.stack([k, v]).float().cpu().numpy()
                values = torch.from_numpy(mxfp4.dequantize(*mxfp4.quantize(rows)))
                for s in range(3):
                    c.cached[layer][s] = torch.cat([c.cached[layer][s], values[:, s:s + 1]], dim=1)
                c.check_token(layer, q, outs[layer])
